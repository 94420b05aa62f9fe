"""Argument checks of the rotary and paged-cache binding that fire before any launch (no GPU), and the numbers behind a
`Rope`."""
import itertools
import math
import struct
from fractions import Fraction

import pytest
import torch

from triton_ext_b200 import backend as B
from triton_ext_b200 import paged as P
from triton_ext_b200 import rotary as R

bf16, f16, i32 = torch.bfloat16, torch.float16, torch.int32


def turns_of(rope):
    return struct.unpack(f"iifi{R.MAX_PAIRS}Q", rope._packed)[4:]


# ---- Rope ------------------------------------------------------------------------------------------------------------
def test_turns_are_the_frequencies_to_64_bits():
    rope = R.Rope(64)
    for w, t in zip(rope.frequencies, turns_of(rope)):
        assert abs(t / 2 ** 64 - w / (2 * math.pi)) <= w * 2.0 ** -52
    assert turns_of(rope)[32:] == (0,) * (R.MAX_PAIRS - 32)
    assert turns_of(R.Rope(2, frequencies=[-0.25]))[0] == (1 << 64) - turns_of(R.Rope(2, frequencies=[0.25]))[0]
    # one radian in 2^-64 turns, from the digits of 1 / (2 pi)
    assert turns_of(R.Rope(2))[0] == round(2 ** 64 * Fraction("0.15915494309189533576888376337251436203445964574046"))


def test_scalings():
    plain = R.Rope(64).frequencies
    assert R.Rope(64, scaling="linear", factor=4.0).frequencies == tuple(w / 4 for w in plain)
    base = R.Rope(64, scaling="base", factor=4.0).frequencies
    assert base[0] == 1.0 and math.isclose(base[-1], plain[-1] / 4, rel_tol=1e-12)
    rope = R.Rope(64, scaling="parts", factor=8.0, original_len=4096)
    for w, p in zip(rope.frequencies, plain):
        n = 4096 * p / (2 * math.pi)
        want = p if n >= 32 else p / 8 if n <= 1 else p * ((n - 1) / 31 + (1 - (n - 1) / 31) / 8)
        assert math.isclose(w, want, rel_tol=1e-12)
    assert math.isclose(rope.magnitude, 0.1 * math.log(8.0) + 1)
    assert R.Rope(64, scaling="parts", factor=8.0, original_len=4096, magnitude=1.0).magnitude == 1.0


@pytest.mark.parametrize("args,kw", [((7,), {}), ((0,), {}), ((258,), {}), ((64,), dict(scaling="other")),
                                     ((64,), dict(scaling="parts", factor=2.0)), ((64,), dict(base=0.0)),
                                     ((64,), dict(factor=math.inf)), ((2,), dict(scaling="base", factor=2.0)),
                                     ((64,), dict(frequencies=[1.0])), ((4,), dict(frequencies=[1.0, math.nan])),
                                     ((4,), dict(frequencies=[1.0, 0.5], scaling="linear")),
                                     ((64,), dict(scaling="parts", factor=2.0, original_len=9, low=3.0, high=3.0))])
def test_rope_refuses(args, kw):
    with pytest.raises(ValueError):
        R.Rope(*args, **kw)


# ---- C entry points (the library is built; there is no device) ---------------------------------------------------------
class Built:
    """CPU tensors behind which the checks up to the device check can be reached."""

    def __init__(self):
        self.k = torch.zeros(4, 16, 2, 64, dtype=bf16)
        self.v = torch.zeros_like(self.k)
        self.table = torch.zeros(3, 2, dtype=i32)
        self.lens = torch.ones(3, dtype=i32)

    def view(self, **kw):
        a = dict(k=self.k, v=self.v, table=self.table, lens=self.lens, cu=None)
        a.update(kw)
        return P._view(a["k"], a["v"], a["table"], a["lens"], a["cu"], -1)[0]


def status_of(call):
    with pytest.raises(B.DotError) as e:
        call()
    return e.value.status, str(e.value)


@pytest.mark.parametrize("kw,text", [
    (dict(v=torch.zeros(4, 16, 2, 32, dtype=bf16)), "one shape and type"),
    (dict(v=torch.zeros(4, 16, 2, 64, dtype=f16)), "one shape and type"),
    (dict(k=torch.zeros(4, 16, 64, 2, dtype=bf16).transpose(2, 3)), "contiguous dimension"),
    (dict(table=torch.zeros(3, 2, dtype=torch.int64)), "page_table must be int32"),
    (dict(table=torch.zeros(2, 3, dtype=i32).t()), "unit column stride"),
    (dict(lens=torch.ones(2, dtype=i32)), "kv_lens"),
    (dict(lens=torch.ones(6, dtype=i32)[::2]), "kv_lens"),
    (dict(cu=torch.zeros(3, dtype=i32)), "cu_q"),
    (dict(cu=torch.zeros(4, dtype=torch.int64)), "cu_q"),
])
def test_view_refuses(built_libs, kw, text):
    status, message = status_of(lambda: Built().view(**kw))
    assert status == B.TXD_ERR_INVALID and text in message


def c_append(view, tokens=3, q_heads=0, rope=None, k=1 << 20, v=1 << 20):
    lib = P._lib()
    rc = lib.tx_paged_append(view, rope, P._APPEND.pack(0, k, v, 0, 0, 0, 128, 64, 128, 64, 0, 0, tokens, q_heads), None)
    return rc, lib.tx_paged_last_error().decode()


@pytest.mark.parametrize("change,text,code", [
    (dict(page_size=8), "page_size 8", B.TXD_ERR_UNSUPPORTED), (dict(page_size=48), "page_size 48", B.TXD_ERR_UNSUPPORTED),
    (dict(head_dim=48), "head_dim 48", B.TXD_ERR_UNSUPPORTED), (dict(dtype=B.TXD_F32), "dtype", B.TXD_ERR_UNSUPPORTED),
    (dict(k=0), "null cache pointer", B.TXD_ERR_INVALID), (dict(k=(1 << 20) + 2), "aligned", B.TXD_ERR_INVALID),
    (dict(ks2=65), "multiples of 16 bytes", B.TXD_ERR_UNSUPPORTED), (dict(table=0), "null table", B.TXD_ERR_INVALID),
    (dict(pages=0), "num_pages", B.TXD_ERR_INVALID)])
def test_c_view_checks(built_libs, change, text, code):
    a = dict(k=1 << 20, v=1 << 20, ks0=2048, ks1=128, ks2=64, table=1 << 20, lens=1 << 20, batch=3, width=2, pages=4,
             page_size=16, heads=2, head_dim=64, dtype=B.TXD_BF16)
    a.update(change)
    view = P._VIEW.pack(a["k"], a["v"], a["ks0"], a["ks1"], a["ks2"], a["ks0"], a["ks1"], a["ks2"], a["table"], 2, a["lens"], 0,
                        a["batch"], a["width"], a["pages"], a["page_size"], a["heads"], a["head_dim"], a["dtype"], 0)
    rc, message = c_append(view)
    assert rc == code and text in message


def c_attention(view, pointers=(1 << 20, 1 << 20, 0), strides=(128, 64, 128, 64), tokens=3, heads=2, max_q=1, causal=1,
                window=0, scale=0.125, ws=1 << 20, size=1 << 40):
    lib = P._lib()
    problem = P._ATTN.pack(*pointers, *strides, tokens, heads, max_q, causal, window, scale)
    return lib.tx_paged_attention(view, problem, ws, size, None), lib.tx_paged_last_error().decode()


def test_c_attention_checks(built_libs):
    view = Built().view()
    for kw, text in ((dict(tokens=-1), "tokens"), (dict(heads=3), "multiple of kv_heads"), (dict(heads=0), "q_heads"),
                     (dict(heads=130), "at most 64"), (dict(max_q=0), "max_q"), (dict(window=-1), "window"),
                     (dict(window=3, causal=0), "window"), (dict(scale=0.0), "sm_scale"), (dict(scale=math.nan), "sm_scale"),
                     (dict(scale=math.inf), "sm_scale"), (dict(tokens=2), "one new token"), (dict(pointers=(0, 1 << 20, 0)), "null tensor"),
                     (dict(pointers=(1 << 20, (1 << 20) + 8, 0)), "16-byte aligned"), (dict(strides=(124, 64, 128, 64)), "multiples of 16 bytes"),
                     (dict(strides=(128, 0, 128, 64)), "positive")):
        rc, message = c_attention(view, **kw)
        assert rc in (B.TXD_ERR_INVALID, B.TXD_ERR_UNSUPPORTED) and text in message, (kw, rc, message)
    if not torch.cuda.is_available():
        assert c_attention(view)[0] == B.TXD_ERR_NO_DEVICE
    none = Built().view(table=torch.zeros(0, 2, dtype=i32), lens=torch.ones(0, dtype=i32))
    assert c_attention(none, tokens=0)[0] == B.TXD_OK
    # the workspace grows with the rows of a tile, and is asked for without a device
    lib = P._lib()
    sizes = [lib.tx_paged_attention_workspace(view, P._ATTN.pack(1 << 20, 1 << 20, 0, 128, 64, 128, 64, 3, 2, q, 1, 0, 0.1))
             for q in (1,)]
    assert sizes[0] > 0


def test_c_append_checks(built_libs):
    view = Built().view()
    assert c_append(view, tokens=-1)[0] == B.TXD_ERR_INVALID
    assert c_append(view, k=0)[0] == B.TXD_ERR_INVALID
    assert c_append(view, q_heads=2)[0] == B.TXD_ERR_INVALID                      # q and its output are null
    assert c_append(view, rope=R.Rope(128)._packed)[0] == B.TXD_ERR_INVALID        # more columns than head_dim
    assert c_append(view, tokens=0)[0] == B.TXD_OK                                 # nothing to do


def test_c_pages_checks(built_libs):
    lib = P._lib()
    good = dict(k=1 << 20, v=1 << 20, page_bytes=64, table=1 << 20, lens=1 << 20, refs=1 << 20, layers=1, pages=8, page=16, rows=4, width=4)

    def state(**kw):
        a = dict(good, **kw)
        return P._STATE.pack(a["k"], a["v"], a["page_bytes"], a["table"], a["lens"], a["refs"], a["layers"], a["pages"], a["page"], a["rows"], a["width"], 0)

    for bad in (dict(page_bytes=24), dict(page=24), dict(layers=0), dict(k=0), dict(refs=(1 << 20) + 4), dict(rows=0), dict(rows=1 << 21)):
        assert lib.tx_pages_free(state(**bad), 1 << 20, 1, None) in (B.TXD_ERR_INVALID, B.TXD_ERR_UNSUPPORTED), bad
    assert lib.tx_pages_free(state(), None, 1, None) == B.TXD_ERR_INVALID
    assert lib.tx_pages_free(state(), None, 0, None) == B.TXD_OK
    assert lib.tx_pages_reserve(state(), 1 << 20, 1 << 20, P.MAX_LIST + 1, 1 << 20, None) == B.TXD_ERR_UNSUPPORTED
    assert lib.tx_pages_reserve(state(width=1 << 20), 1 << 20, 1 << 20, P.MAX_LIST, 1 << 20, None) == B.TXD_ERR_UNSUPPORTED
    assert lib.tx_pages_reserve(state(), 1 << 20, 1 << 20, 1, (1 << 20) + 8, None) == B.TXD_ERR_INVALID  # workspace
    assert lib.tx_pages_fork(state(), 1 << 20, 1 << 20, 1, None, None) == B.TXD_ERR_INVALID

    def copy(src, dst):
        import ctypes
        n = len(src)
        rc = lib.tx_pages_copy(state(), (ctypes.c_int32 * n)(*src), (ctypes.c_int32 * n)(*dst), n, None)
        return rc, lib.tx_paged_last_error().decode()

    assert copy([0, 8], [1, 2])[0] == B.TXD_ERR_INVALID and copy([0], [-1])[0] == B.TXD_ERR_INVALID
    assert "page 3" in copy([0, 1], [3, 3])[1] and "page 1" in copy([0, 1], [1, 2])[1]
    if not torch.cuda.is_available():
        assert copy([0, 0], [3, 4])[0] == B.TXD_ERR_NO_DEVICE


# ---- Python entry points -----------------------------------------------------------------------------------------------
def test_cpu_tensors_are_refused_not_computed(built_libs):
    c = Built()
    x = torch.zeros(3, 2, 64, dtype=bf16)
    assert status_of(lambda: P.append(None, x, x, c.k, c.v, c.table, c.lens))[0] == B.TXD_ERR_NO_DEVICE
    assert status_of(lambda: P.paged_attention(x, c.k, c.v, c.table, c.lens, 0.1))[0] == B.TXD_ERR_NO_DEVICE
    q = torch.zeros(1, 2, 3, 64, dtype=bf16)
    assert status_of(lambda: R.rotary_forward(q, None, torch.arange(3), R.Rope(64)))[0] == B.TXD_ERR_NO_DEVICE
    cache = P.PagedCache.create(4, 16, 2, 64, rows=3, width=2, device="cpu")
    rows = torch.zeros(1, dtype=i32)
    for call in (lambda: cache.free(rows), lambda: cache.fork(rows, rows), lambda: cache.reserve(rows, rows), cache.compact,
                 lambda: cache.copy_pages([0], [1])):
        assert status_of(call)[0] == B.TXD_ERR_NO_DEVICE


def test_cache_refuses():
    k = torch.zeros(2, 4, 16, 2, 64, dtype=bf16)
    table, lens, refs = torch.zeros(3, 2, dtype=i32), torch.zeros(3, dtype=i32), torch.zeros(4, dtype=i32)
    P.PagedCache(k, k.clone(), table, lens, refs)
    for args in ((k, k[:1], table, lens, refs), (k.float(), k.float(), table, lens, refs), (k, k, table.long(), lens, refs),
                 (k, k, table, lens[:2], refs), (k, k, table, lens, refs[:3]), (k, k, table.t().contiguous().t(), lens, refs),
                 (k[:, :, :, :, ::2], k[:, :, :, :, ::2], table, lens, refs)):
        with pytest.raises(B.DotError):
            P.PagedCache(*args)


def test_truncate_refuses(built_libs):
    lib = P._lib()
    state = P._STATE.pack(1 << 20, 1 << 20, 64, 1 << 20, 1 << 20, 1 << 20, 1, 8, 16, 4, 4, 0)
    assert lib.tx_pages_truncate(state, None, 1 << 20, 1, None) == B.TXD_ERR_INVALID
    assert lib.tx_pages_truncate(state, 1 << 20, None, 1, None) == B.TXD_ERR_INVALID
    assert lib.tx_pages_truncate(state, 1 << 20, 1 << 20, -1, None) == B.TXD_ERR_INVALID
    assert lib.tx_pages_truncate(state, None, None, 0, None) == B.TXD_OK
    cache = P.PagedCache.create(4, 16, 2, 64, rows=3, width=2, device="cpu")
    rows = torch.zeros(1, dtype=i32)
    assert status_of(lambda: cache.truncate(rows, rows))[0] == B.TXD_ERR_NO_DEVICE


def test_reserve_with_lengths_refuses(built_libs):
    """The checks of a plain reserve, and nothing to do for an empty list."""
    lib = P._lib()
    state = P._STATE.pack(1 << 20, 1 << 20, 64, 1 << 20, 1 << 20, 1 << 20, 1, 8, 16, 4, 4, 0)
    call = lib.tx_pages_reserve_lens
    assert call(None, 1 << 20, 1 << 20, 1, 1 << 20, 1 << 20, None) == B.TXD_ERR_INVALID
    assert call(state, None, 1 << 20, 1, 1 << 20, 1 << 20, None) == B.TXD_ERR_INVALID
    assert call(state, 1 << 20, 1 << 20, P.MAX_LIST + 1, 1 << 20, 1 << 20, None) == B.TXD_ERR_UNSUPPORTED
    assert call(state, 1 << 20, 1 << 20, 1, 1 << 20, None, None) == B.TXD_ERR_INVALID  # workspace
    assert call(state, None, None, 0, None, None, None) == B.TXD_OK


@pytest.mark.parametrize("shape,strides,want", [
    ((4, 3, 8), (24, 8, 1), False), ((4, 3, 8), (8, 32, 1), False), ((4, 3, 8), (100, 10, 1), False), ((1, 3, 8), (0, 8, 1), False),
    ((4, 1, 8), (8, 0, 1), False), ((4, 3, 8), (0, 8, 1), True), ((4, 3, 8), (24, 0, 1), True), ((4, 3, 8), (8, 8, 1), True),
    ((4, 1, 8), (1, 8, 1), True), ((4, 1, 8), (7, 8, 1), True), ((2, 4, 3, 8), (23, 8, 8, 1), True), ((1, 1, 1), (0, 0, 1), False),
    ((0, 3, 8), (24, 8, 1), False)])
def test_overlaps(shape, strides, want):
    x = torch.zeros(500).as_strided(shape, strides)
    assert R._overlaps(x) == want
    if x.numel():
        places = {sum(i * s for i, s in zip(at, strides)) for at in itertools.product(*(range(n) for n in shape))}
        assert (len(places) < x.numel()) == want


def test_outputs_that_overlap_themselves_are_refused():
    """Windows of one vector, a column apart: rows would overwrite one another. Refused before there is a device to ask for."""
    x = torch.zeros(2, 3, 10, 64)
    with pytest.raises(B.DotError, match="overlap itself"):
        R._part(x, torch.zeros(700).as_strided(x.shape, (300, 100, 1, 1)), 3, "out_q")
    R._part(x, torch.zeros(2, 10, 3, 64).transpose(1, 2), 3, "out_q")


@pytest.mark.parametrize("head_dim,tokens,rows,per_sm", [(16, 1, 16, 2), (64, 8, 16, 2), (128, 8, 16, 2), (64, 9, 32, 1), (128, 16, 32, 1),
                                                         (32, 17, 256, 1), (64, 400, 256, 1), (128, 17, 256, 1), (256, 8, 16, 1),
                                                         (256, 16, 32, 1), (256, 17, 64, 1), (256, 400, 64, 1)])
def test_workspace_holds_the_parts_of_every_kernel(built_libs, head_dim, tokens, rows, per_sm):
    """Two parts of a tile for each CTA: rows of fp32 columns, a maximum and a sum; and 16 bytes of border. Two query heads to a key
    head; `rows` is the tile of the kernel that takes `tokens` of one sequence."""
    lib = P._lib()
    a = 1 << 20
    view = P._VIEW.pack(a, a, 16 * 2 * head_dim, 2 * head_dim, head_dim, 16 * 2 * head_dim, 2 * head_dim, head_dim, a, 600, a, a, 1, 600,
                        700, 16, 2, head_dim, B.TXD_BF16, 0)

    def size(max_q):
        return lib.tx_paged_attention_workspace(view, P._ATTN.pack(a, a, 0, 4 * head_dim, head_dim, 4 * head_dim, head_dim, tokens, 4, max_q,
                                                                   1, 0, 0.1))

    ctas = (torch.cuda.get_device_properties(0).multi_processor_count if torch.cuda.is_available() else 148) * per_sm
    least = ctas * 2 * rows * (max(head_dim, 64) * 4 + 8) + 16 * ctas
    assert least <= size(tokens) < least + 256
    assert size(2 ** 31 - 1) == size(tokens)                       # the bound is cut to the tokens that there are
    refused = lib.tx_paged_attention(view, P._ATTN.pack(a, a, 0, 4 * head_dim, head_dim, 4 * head_dim, head_dim, tokens, 4, tokens, 1, 0, 0.1),
                                     a, size(tokens) - 1, None)
    if torch.cuda.is_available():
        assert refused == B.TXD_ERR_INVALID and f"of {size(tokens)} bytes" in lib.tx_paged_last_error().decode()
    else:
        assert refused == B.TXD_ERR_NO_DEVICE
