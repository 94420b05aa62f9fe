"""Paged attention on the GPU against its definition in 64 bits.

Tolerance, per element of the output, with u the half step of the type (2^-8 bf16, 2^-11 f16) and A = sum_j p_j |v_j| (the
softmax-weighted magnitudes, p summing to 1):
  * the output's own rounding: u |o|
  * every P is rounded to the type before its product with V: u A; for f16, P below 2^-14 rounds among the subnormals, off by
    2^-25 of a reference that is at most 2^8 below the row's maximum: 2^-17 per key against a sum of at least 2^-8, counted
    as keys * 2^-25 * 2^8 * max |v| / 2^-0 only where it can happen: covered by `keys * 2^-24 * max|v|` at a lazily moved
    reference that is never above the maximum (the largest P is then >= 1)
  * scores are fp32 sums of D exact products (the 16-bit inputs' products are exact in fp32): D 2^-24 sum|q||k|, times the scale;
    the exponent's argument is rounded (2^-24 of its size, |argument| <= the largest score), ex2.approx is within 2^-22;
    dp / p <= that: with E = D 2^-24 (|q|.|k|) scale + 2^-23 max|score| + 2^-21, o moves by at most 2 E A (numerator and sum)
  * fp32 accumulation of the P V sums and of l: keys 2^-24 each: 2 keys 2^-24 A
m = max + log2(sum): E / ln 2 + keys 2^-24 / ln 2 + 2^-22 |m|."""
import math
import random

import pytest
import torch

pytestmark = pytest.mark.gpu

f16, bf16, i32 = torch.float16, torch.bfloat16, torch.int32


@pytest.fixture(scope="module")
def P(built_libs, cuda_device):
    from triton_ext_b200 import paged
    return paged


def ints(x):
    return torch.tensor(list(x), dtype=i32, device="cuda")


class Batch:
    """A batch over a paged cache. Slots that no sequence has written hold NaN, unused table cells garbage."""

    def __init__(self, q_lens, kv_lens, h, hk, d, page, dtype, seed=0, heads_first=False, std=1.0, behind=0):
        g = torch.Generator().manual_seed(seed)
        self.q_lens, self.kv_lens_host, self.page, self.group = list(q_lens), list(kv_lens), page, h // hk
        used = [-(-n // page) for n in kv_lens]
        pages, width = sum(used) + 2, max(max(used, default=0), 1) + 2
        order = torch.randperm(pages, generator=g).tolist()
        table, at = [], 0
        for n in used:
            table.append(order[at:at + n] + [-7, 1 << 30, 5][: width - n] + [-1] * max(0, width - n - 3))
            at += n
        self.table = torch.tensor(table, dtype=i32).view(len(used), width).cuda()
        self.kv_lens = ints(kv_lens)
        self.single = all(n == 1 for n in q_lens) and not behind
        self.cu_q = None if self.single else torch.tensor([0] + self.q_lens).cumsum(0).to(i32).cuda()
        self.max_q = max(max(q_lens, default=1), 1)
        total = sum(q_lens) + behind
        self.q = (torch.randn(total, h, d, generator=g) * std).to(dtype).cuda()
        self.kv = [(torch.randn(sum(kv_lens), hk, d, generator=g) * std).to(dtype).cuda() for _ in range(2)]
        shape = (pages, hk, page, d) if heads_first else (pages, page, hk, d)
        self.pools = [torch.full(shape, math.nan, dtype=dtype, device="cuda") for _ in range(2)]
        if heads_first:
            self.pools = [x.transpose(1, 2) for x in self.pools]
        at = 0
        for i, n in enumerate(kv_lens):
            pos = torch.arange(n, device="cuda")
            for pool, new in zip(self.pools, self.kv):
                pool[self.table[i].long()[pos // page], pos % page] = new[at:at + n]
            at += n

    def run(self, P, scale, **kw):
        if not self.single:
            kw.setdefault("max_q", self.max_q)
        return P.paged_attention(self.q, *self.pools, self.table, self.kv_lens, scale, cu_q=self.cu_q, **kw)

    def reference(self, scale, causal=True, window=0):
        """Per sequence: (output, m, tolerance of the output, tolerance of m) in double, [tokens, heads, ...]."""
        out, at_q, at_k = [], 0, 0
        eps = torch.finfo(self.q.dtype).eps / 2
        for n, m in zip(self.q_lens, self.kv_lens_host):
            q = self.q[at_q:at_q + n].double().transpose(0, 1)
            k, v = (x[at_k:at_k + m].double().transpose(0, 1).repeat_interleave(self.group, 0) for x in self.kv)
            pos = torch.arange(m - n, m, device="cuda")[:, None]
            key = torch.arange(m, device="cuda")
            seen = (key <= pos) if causal else torch.ones(n, m, dtype=torch.bool, device="cuda")
            if window:
                seen = seen & (key > pos - window)
            s = (q @ k.transpose(1, 2) * scale).masked_fill(~seen, -math.inf)
            empty = ~seen.any(-1)
            p = torch.where(empty[None, :, None], 0.0, s.softmax(-1))
            o = p @ v
            lse2 = torch.logsumexp(s, -1) / math.log(2.0)
            d, size = q.shape[-1], torch.where(seen, q.abs() @ k.abs().transpose(1, 2), 0.0)
            most = size.amax(-1, keepdim=True) if m else torch.zeros(*q.shape[:2], 1, device="cuda")
            e = most * scale * (d * 2.0 ** -24 + 2.0 ** -23) + 2.0 ** -21
            a = p @ v.abs()
            vmax = v.abs().amax((-1, -2), keepdim=True) if m else torch.zeros(q.shape[0], 1, 1, device="cuda")
            tiny = m * 2.0 ** -24 * vmax if self.q.dtype == f16 else 0.0
            tol = eps * o.abs() + eps * a * 1.01 + 2 * e * a + 2 * m * 2.0 ** -24 * a + tiny + 2.0 ** -24 * (self.q.dtype == f16)
            tol_m = (e[..., 0] + m * 2.0 ** -24) / math.log(2.0) + 2.0 ** -22 * lse2.abs().nan_to_num(posinf=0.0)
            out.append([x.transpose(0, 1) for x in (o, lse2, tol, tol_m)])
            at_q, at_k = at_q + n, at_k + m
        return [torch.cat(x) for x in zip(*out)]

    def compare(self, P, scale, **kw):
        got, m = self.run(P, scale, return_m=True, **kw)
        P.check()
        o, lse2, tol, tol_m = self.reference(scale, kw.get("causal", True), kw.get("window", 0))
        n = sum(self.q_lens)
        err = (got[:n].double() - o).abs()
        assert not bool(err.isnan().any())
        worst = float((err / tol.clamp(min=1e-30)).max())
        assert worst <= 1.0, f"output: {worst} of the tolerance"
        none = lse2.isinf()
        assert torch.equal(m[:n].isinf() & (m[:n] < 0), none)
        err = torch.where(none, 0.0, (m[:n].double() - lse2).abs())
        assert bool((err <= tol_m).all()), f"m: {float((err / tol_m).max())} of the tolerance"
        return got, m


SCALE = {16: 0.25, 32: 0.2, 64: 0.125, 128: 0.09, 256: 0.0625}

DECODE = [
    # kv lengths, h, hk, d, page, dtype
    ([1], 1, 1, 64, 16, bf16),
    ([777], 16, 4, 64, 16, f16),
    ([0, 1, 15, 16, 17, 63, 64, 65, 1000], 8, 2, 128, 16, bf16),
    ([5000, 3, 128], 6, 2, 64, 32, bf16),
    ([2049], 8, 1, 128, 64, f16),
    ([300, 301], 5, 5, 128, 128, bf16),
    ([300, 90], 64, 1, 64, 256, bf16),
    ([130, 4097], 12, 2, 256, 16, f16),
    ([70, 20], 4, 2, 16, 16, bf16),
    ([70, 200], 3, 1, 32, 64, f16),
    ([33] * 300, 4, 2, 64, 16, bf16),           # more sequences than threads of a CTA
    ([20000], 20, 1, 128, 16, bf16),
]


@pytest.mark.parametrize("kv,h,hk,d,page,dtype", DECODE)
@pytest.mark.parametrize("heads_first", [False, True])
def test_single_tokens(P, kv, h, hk, d, page, dtype, heads_first):
    Batch([1] * len(kv), kv, h, hk, d, page, dtype, seed=len(kv), heads_first=heads_first).compare(P, SCALE[d])


CHUNKS = [
    # q lengths, kv lengths, h, hk, d, page, dtype, window
    ([5] * 4, [5, 90, 1000, 64], 8, 2, 128, 32, f16, 0),
    ([3, 0, 1, 8], [50, 20, 700, 8], 6, 2, 64, 16, bf16, 0),
    ([16], [1200], 4, 1, 128, 16, bf16, 0),                       # 64 rows
    ([4, 4], [300, 2000], 8, 2, 128, 64, bf16, 100),
    ([70], [70], 3, 3, 64, 16, f16, 0),
    ([129, 1, 64], [129, 500, 900], 4, 2, 64, 16, bf16, 0),
    ([256], [4000], 8, 2, 128, 16, bf16, 0),
    ([500, 300], [500, 1500], 4, 1, 128, 128, f16, 0),
    ([333], [900], 7, 1, 128, 32, bf16, 0),                       # 128 rows are 18 tokens of 7 heads and two rows over
    ([100, 700], [800, 700], 2, 2, 64, 64, bf16, 130),
    ([300], [1000], 4, 2, 128, 256, bf16, 1),                     # every row sees one key
    ([200], [600], 2, 1, 256, 16, bf16, 0),
    ([150, 20], [200, 20], 2, 1, 32, 16, f16, 0),
    ([40], [300], 2, 2, 16, 32, bf16, 60),
    ([64, 2], [10, 1], 4, 2, 64, 16, bf16, 0),                    # more new tokens than cached ones: the first rows see nothing
    ([130], [0], 2, 1, 128, 16, f16, 0),
    ([100], [513], 64, 1, 64, 16, bf16, 0),
    ([1] * 30 + [400], list(range(1, 31)) + [3000], 8, 8, 64, 16, bf16, 0),
]


@pytest.mark.parametrize("q,kv,h,hk,d,page,dtype,window", CHUNKS)
def test_chunks(P, q, kv, h, hk, d, page, dtype, window):
    Batch(q, kv, h, hk, d, page, dtype, seed=sum(q)).compare(P, SCALE[d], window=window)


@pytest.mark.parametrize("q,kv,h,hk,d,page,dtype,window", CHUNKS[:9])
def test_chunks_without_causal(P, q, kv, h, hk, d, page, dtype, window):
    Batch(q, kv, h, hk, d, page, dtype, seed=sum(q)).compare(P, SCALE[d], causal=False)


@pytest.mark.parametrize("q", [1, 4, 200])
def test_large_scores_move_the_reference(P, q):
    """Scores of standard deviation 60 and more: the running maximum moves often and by much."""
    Batch([q] * 2, [700, 1500], 4, 2, 64, 16, bf16, seed=5, std=2.7).compare(P, 1.0)
    b = Batch([q] * 2, [700, 1500], 4, 2, 64, 16, f16, seed=6)
    b.compare(P, 3.0)


@pytest.mark.parametrize("q,kv,page,window", [(1, 700, 16, 65), (200, 900, 16, 65), (5, 700, 64, 200)])
def test_pages_behind_the_window_may_be_gone(P, q, kv, page, window):
    """Positions that no row sees are not read: their pages may be given away and hold NaN, their table cells -1."""
    b = Batch([q], [kv], 4, 2, 64, page, bf16, seed=8)
    want, m = b.compare(P, 0.125, window=window)
    first = kv - q + 1 - window                                   # the first position that is seen
    gone = first // page
    for pool in b.pools:
        pool[b.table[0, :gone].long()] = math.nan
        pool[b.table[0, gone].long(), : first % page] = math.inf
    b.table[0, :gone] = -1
    got, m2 = b.run(P, 0.125, window=window, return_m=True)
    P.check()
    assert torch.equal(got, want) and torch.equal(m, m2)


def test_strided_q_and_out_and_rows_behind(P):
    b = Batch([3, 40], [30, 300], 4, 2, 64, 16, bf16, seed=9, behind=5)
    want, _ = b.compare(P, 0.125)
    wide = torch.zeros(48, 3, 4, 64, dtype=bf16, device="cuda")
    wide[:, 1] = b.q
    b.q = wide[:, 1]
    out = torch.full((48, 2, 4, 64), 3.0, dtype=bf16, device="cuda")
    got = b.run(P, 0.125, out=out[:, 0])
    assert torch.equal(got[:43], want[:43]) and bool((out[43:] == 3.0).all()) and bool((out[:, 1] == 3.0).all())


def test_many_sequences_in_tiles(P):
    """More sequences than a CTA has threads, prompts and single tokens mixed, on the kernel for many rows."""
    rng = random.Random(3)
    q = [rng.choice([0, 1, 1, 2, 40, 130]) for _ in range(400)]
    kv = [n + rng.choice([0, 0, 5, 200]) for n in q]
    Batch(q, kv, 2, 1, 64, 16, bf16, seed=20).compare(P, 0.125)


def test_waves_of_whole_tiles(P):
    """Several tiles for every SM, of unequal lengths: dealt out whole, the rest cut."""
    Batch([700, 1300, 90, 2000], [700, 2500, 4000, 2000], 16, 4, 64, 32, bf16, seed=21).compare(P, 0.125)
    Batch([512] * 10, [512] * 10, 32, 32, 64, 64, f16, seed=22).compare(P, 0.125)


def test_table_and_lengths_that_are_views(P):
    b = Batch([1, 1, 1], [300, 20, 77], 4, 2, 64, 16, bf16, seed=23)
    want = b.run(P, 0.125)
    wide = torch.full((6, b.table.shape[1] + 9), -5, dtype=i32, device="cuda")
    wide[::2, 4:4 + b.table.shape[1]] = b.table
    b.table = wide[::2, 4:4 + b.table.shape[1]]
    assert torch.equal(b.run(P, 0.125), want)
    e = b.q[:, :1].expand(3, 4, 64)                               # one query for all heads
    b.q = e.contiguous()
    want = b.run(P, 0.125)
    b.q = e
    assert torch.equal(b.run(P, 0.125), want)


def test_tokens_before_and_behind_the_sequences(P):
    """cu_q may start above zero and end before the last row: rows outside are left alone, by append too."""
    b = Batch([4, 40], [30, 300], 4, 2, 64, 16, bf16, seed=24)
    want = b.run(P, 0.125)
    q = torch.cat((b.q[:3], b.q, b.q[:2]))
    out = torch.full_like(q, 9.0)
    P.paged_attention(q, *b.pools, b.table, b.kv_lens, 0.125, cu_q=b.cu_q + 3, max_q=40, out=out)
    assert torch.equal(out[3:47], want) and bool((out[:3] == 9.0).all()) and bool((out[47:] == 9.0).all())
    pools = [x.clone() for x in b.pools]
    k, v = (torch.full((49, 2, 64), x, dtype=bf16, device="cuda") for x in (2.0, 3.0))
    got = torch.full_like(q, 9.0)
    P.append(q, k, v, *pools, b.table, b.kv_lens, cu_q=b.cu_q + 3, out=got)
    P.check()
    assert torch.equal(got[3:47], b.q) and bool((got[:3] == 9.0).all()) and bool((got[47:] == 9.0).all())
    expected = [x.clone() for x in b.pools]
    for i, (n, m) in enumerate(zip(b.q_lens, b.kv_lens_host)):
        pos = torch.arange(m - n, m, device="cuda")
        for pool, value in zip(expected, (2.0, 3.0)):
            pool[b.table[i].long()[pos // 16], pos % 16] = value
    assert all(torch.equal(x.view(torch.int16), y.view(torch.int16)) for x, y in zip(pools, expected))


def test_in_place(P):
    for q, kv in (([1] * 4, [3000, 5, 64, 900]), ([300, 70], [900, 70])):
        b = Batch(q, kv, 8, 2, 128, 16, bf16, seed=25)
        want = b.run(P, 0.09)
        got = b.run(P, 0.09, out=b.q)
        assert got.data_ptr() == b.q.data_ptr() and torch.equal(got, want)


def test_pools_past_2_to_the_32_bytes_and_elements(P):
    """Pages whose offsets pass 2^31 elements: append writes them, both kernels read them, a fork's copy moves them."""
    page, hk, d = 256, 8, 128
    pages = (1 << 31) // (page * hk * d) + 40                     # 8232 pages: 2.16e9 elements a pool
    cache = P.PagedCache.create(pages, page, hk, d, rows=3, width=4)
    cache.refs[: pages - 12] = 1                                  # only the last pages are free
    g = torch.Generator().manual_seed(26)
    lens = [600, 300]
    cache.reserve(ints([0, 1]), ints(lens))
    assert int(cache.table[0, 0]) == pages - 12
    total = sum(lens)
    q, k, v = (torch.randn(total, n, d, generator=g).to(bf16).cuda() for n in (16, hk, hk))
    cu = ints([0, 600, 900])
    table, kv = cache.table[:2], cache.lens[:2]
    P.append(None, k, v, cache.k[0], cache.v[0], table, kv, cu_q=cu)
    cache.fork(ints([2]), ints([0]))
    cache.reserve(ints([2]), ints([1]))
    P.check()
    kk, vv = (torch.cat((x[:600], x[:1])) for x in (k, v))
    P.append(None, kk[600:], vv[600:], cache.k[0], cache.v[0], cache.table[2:], cache.lens[2:])
    many = P.paged_attention(q, cache.k[0], cache.v[0], table, kv, 0.09, cu_q=cu, max_q=600)
    one = P.paged_attention(q[:1], cache.k[0], cache.v[0], cache.table[2:], cache.lens[2:], 0.09)
    P.check()

    def dense(q, k, v, causal):
        s = torch.einsum("thd,khd->htk", q.double(), k.double().repeat_interleave(2, 1)) * 0.09
        if causal:
            s = s.masked_fill(torch.ones(s.shape[1:], device="cuda").triu(1).bool(), -math.inf)
        return torch.einsum("htk,khd->thd", s.softmax(-1), v.double().repeat_interleave(2, 1))

    # values of standard deviation 1, |o| and the weighted magnitudes below 5: 2^-8 * 5 for the output's rounding and as
    # much for P's
    for got, want in ((many[:600], dense(q[:600], k[:600], v[:600], True)), (many[600:], dense(q[600:], k[600:], v[600:], True)),
                      (one, dense(q[:1], kk, vv, False))):
        assert float((got.double() - want).abs().max()) <= 2 * 5 * 2.0 ** -8


@pytest.mark.parametrize("max_q", [1, 5, 4096])
def test_max_q_only_chooses_the_kernel(P, max_q):
    Batch([5, 77], [300, 900], 8, 2, 128, 16, bf16, seed=10).compare(P, 0.09, max_q=max_q)


def test_same_bits_every_time_and_on_two_streams(P):
    for q, kv in (([1] * 7, [9000, 5, 300, 4000, 64, 1, 2500]), ([300, 20], [5000, 900])):
        b = Batch(q, kv, 8, 2, 128, 16, bf16, seed=11)
        want = b.run(P, 0.09)
        streams = [torch.cuda.Stream() for _ in range(2)]
        torch.cuda.synchronize()
        got = []
        for _ in range(10):
            for s in streams:                                     # two calls at once
                with torch.cuda.stream(s):
                    got.append(b.run(P, 0.09))
        torch.cuda.synchronize()
        assert all(torch.equal(want, x) for x in got)
        P.check()


def test_graph_replays_follow_the_lengths(P):
    """Captured once, replayed while the sequences grow: lengths, table and queries are read at replay."""
    b = Batch([1] * 4, [500, 60, 1000, 3], 8, 2, 128, 16, bf16, seed=12)
    lens = b.kv_lens.clone()
    b.kv_lens.copy_(ints([100, 1, 5, 2]))
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = b.run(P, 0.09)
    with torch.cuda.graph(other):                                 # a second graph next to it, replayed in between
        out2 = b.run(P, 0.09)
    for step in (lens, lens - 2, ints([0, 0, 1, 3])):
        b.kv_lens.copy_(step)
        graph.replay()
        other.replay()
        want = b.run(P, 0.09)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(out2, want)
    P.check()


def test_bad_pages_and_lengths_are_reported(P):
    from triton_ext_b200 import backend as B
    for q in (1, 100):
        for bad in (-1, 1 << 20):
            b = Batch([q], [300], 4, 2, 64, 16, bf16, seed=13)
            b.table[0, 3] = bad
            b.run(P, 0.125)
            with pytest.raises(B.DotError, match="outside the cache"):
                P.check()
        b = Batch([q], [300], 4, 2, 64, 16, bf16, seed=13)
        b.table = b.table[:, :10].contiguous()                    # 160 positions
        b.run(P, 0.125)
        with pytest.raises(B.DotError, match="width"):
            P.check()


@pytest.mark.parametrize("q", [1, 100])
def test_a_wait_that_runs_out_is_reported_and_the_next_call_is_right(P, q, monkeypatch):
    from triton_ext_b200 import backend as B
    b = Batch([q] * 2, [300, 900], 4, 2, 64, 16, bf16, seed=14)
    monkeypatch.setenv("TXD_INJECT_STALL", "1")
    monkeypatch.setenv("TXD_WAIT_LIMIT_MS", "50")
    b.run(P, 0.125)
    with pytest.raises(B.DotError) as e:
        P.check()
    assert e.value.status == B.TXD_ERR_DEVICE_TIMEOUT
    monkeypatch.delenv("TXD_INJECT_STALL")
    monkeypatch.delenv("TXD_WAIT_LIMIT_MS")
    b.compare(P, 0.125)


def test_empty_calls(P):
    b = Batch([1], [40], 4, 2, 64, 16, bf16)
    none = torch.empty(0, 4, 64, dtype=bf16, device="cuda")
    assert P.paged_attention(none, *b.pools, b.table[:0], b.kv_lens[:0], 0.1).shape == none.shape
    assert P.paged_attention(none, *b.pools, b.table, b.kv_lens, 0.1, cu_q=ints([0, 0]), max_q=4).shape == none.shape


def test_refusals(P):
    from triton_ext_b200 import backend as B
    b = Batch([2], [40], 4, 2, 64, 16, bf16)
    for kw in (dict(max_q=0), dict(window=-1), dict(window=5, causal=False), dict(out=b.q[:1]), dict(out=b.q[:, :1].expand(2, 4, 64))):
        with pytest.raises(B.DotError):
            b.run(P, 0.1, **kw)
    for scale in (0.0, -1.0, math.nan, math.inf):
        with pytest.raises(B.DotError):
            b.run(P, scale)
    with pytest.raises(B.DotError, match="needs max_q"):
        P.paged_attention(b.q, *b.pools, b.table, b.kv_lens, 0.1, cu_q=b.cu_q)
    with pytest.raises(B.DotError, match="one new token"):
        P.paged_attention(b.q, *b.pools, b.table, b.kv_lens, 0.1)
    with pytest.raises(B.DotError, match="multiple of kv_heads"):
        P.paged_attention(b.q[:, :3].contiguous(), *b.pools, b.table, b.kv_lens, 0.1, cu_q=b.cu_q, max_q=2)
    with pytest.raises(B.DotError, match="head_dim"):
        P.paged_attention(b.q[:, :, :32].contiguous(), *b.pools, b.table, b.kv_lens, 0.1, cu_q=b.cu_q, max_q=2)
    with pytest.raises(B.DotError, match="multiples of 16 bytes"):
        odd = torch.zeros(2, 4, 65, dtype=bf16, device="cuda")[:, :, :64]
        P.paged_attention(odd, *b.pools, b.table, b.kv_lens, 0.1, cu_q=b.cu_q, max_q=2)
    P.check()


def test_bounds_past_32_bits(P):
    """A window or a bound on the new tokens beyond every length is as good as none."""
    from triton_ext_b200 import backend as B
    b = Batch([3, 40], [30, 70], 4, 2, 64, 16, bf16)
    want = b.run(P, 0.1)
    assert torch.equal(b.run(P, 0.1, window=2 ** 40, max_q=2 ** 40), want)
    assert torch.equal(b.run(P, 0.1, window=2 ** 31 - 1, max_q=2 ** 31 - 1), want)
    for kw in (dict(window=-2 ** 40), dict(max_q=-2 ** 40)):
        with pytest.raises(B.DotError):
            b.run(P, 0.1, **kw)


# ---- a run of the operators together ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("page,d,dtype", [(16, 64, bf16), (64, 128, f16)])
def test_a_serving_run(P, page, d, dtype):
    """Prompts in chunks, samples forked from them, tokens, a reordering, a compaction: every step's attention against the
    dense one over the tokens that each row has seen, turned by their positions in double precision."""
    from test_rotary_gpu import turned64
    from triton_ext_b200.rotary import Rope
    g = torch.Generator().manual_seed(page)
    rng = random.Random(page)
    rope, h, hk, rows = Rope(d, scaling="linear", factor=2.0), 6, 2, 6
    cache = P.PagedCache.create(200, page, hk, d, rows=rows, width=600 // page + 1, layers=2, dtype=dtype)
    cache.k.fill_(math.nan)
    cache.v.fill_(math.nan)
    history = [[([], []) for _ in range(rows)] for _ in range(2)]       # [layer][row]: turned keys as stored, values

    def step(active, new):
        cache.reserve(ints(active), ints(new))
        table, lens = cache.table[torch.tensor(active)], cache.lens[torch.tensor(active)]
        cu = torch.tensor([0] + new).cumsum(0).to(i32).cuda() if max(new) > 1 else None
        for layer in range(2):
            q, k, v = ((torch.randn(sum(new), n, d, generator=g)).to(dtype).cuda() for n in (h, hk, hk))
            tq = P.append(q, k, v, cache.k[layer], cache.v[layer], table, lens, rope=rope, cu_q=cu)
            got = P.paged_attention(tq, cache.k[layer], cache.v[layer], table, lens, d ** -0.5, cu_q=cu, max_q=max(new))
            at = 0
            for r, n in zip(active, new):
                keys, values = history[layer][r]
                pos = torch.arange(len(keys), len(keys) + n, device="cuda")
                tk, _ = turned64(k[at:at + n].transpose(0, 1)[None], pos, rope)
                keys += list(tk[0].transpose(0, 1).to(dtype))
                values += list(v[at:at + n])
                kk, vv = (torch.stack(x).double().repeat_interleave(h // hk, 1).transpose(0, 1) for x in (keys, values))
                qq, _ = turned64(q[at:at + n].transpose(0, 1)[None], pos, rope)
                s = qq[0].to(dtype).double() @ kk.transpose(1, 2) * d ** -0.5
                hidden = torch.arange(len(keys), device="cuda") > pos[:, None]
                want = (s.masked_fill(hidden, -math.inf).softmax(-1) @ vv).transpose(0, 1)
                # against values of standard deviation 1: u for the output, u for P, and a step of the type in a turned
                # q or k (u |q||k| scale in a score, twice): 8 u of the largest |v| (below 5) is beyond all of it
                assert float((got[at:at + n].double() - want).abs().max()) <= 8 * 5 * torch.finfo(dtype).eps / 2
                at += n

    def copy_rows(dst, src):
        cache.fork(ints(dst), ints(src))
        for layer in history:
            old = [(list(a), list(b)) for a, b in layer]
            for a, b in zip(dst, src):
                layer[a] = (list(old[b][0]), list(old[b][1]))

    step([0, 3], [70, 200])                # first chunks
    step([3, 0], [33, 1])                  # a second chunk, next to a token
    copy_rows([1, 2, 4, 5], [0, 0, 3, 3])
    for _ in range(3):
        step([0, 1, 2, 3, 4, 5], [1] * 6)
    copy_rows([0, 1, 2, 3, 4, 5], [rng.randrange(6) for _ in range(6)])
    step([5, 4, 3, 2, 1, 0], [3, 1, 4, 1, 5, 2])
    cache.free(ints([1, 3]))
    for layer in history:
        layer[1], layer[3] = ([], []), ([], [])
    cache.compact()
    used = int((cache.refs > 0).sum())
    assert bool((cache.refs[:used] > 0).all())
    step([0, 1, 2, 3, 4, 5], [1, 40, 1, 17, 1, 1])
    P.check()


@pytest.mark.parametrize("page,window,captured", [(16, 0, False), (32, 40, True)])
def test_drafts_that_are_not_accepted(P, page, window, captured):
    """Five drafted tokens for each row, of which as many are kept as a device tensor says: the step is reserve, append,
    attention, truncate, eager or captured once and replayed. No page is lost, and every step's attention is that over the
    kept tokens and the drafts."""
    from triton_ext_b200.rotary import Rope
    g = torch.Generator().manual_seed(page)
    rng = random.Random(page)
    d, h, hk, rows, drafts = 64, 4, 2, 3, 5
    cache = P.PagedCache.create(30, page, hk, d, rows=rows, width=128 // page, dtype=bf16)
    every, count, kept = ints(range(rows)), ints([drafts] * rows), ints([drafts] * rows)
    cu = ints(range(0, drafts * rows + 1, drafts))
    q, k, v = (torch.zeros(drafts * rows, n, d, dtype=bf16, device="cuda") for n in (h, hk, hk))

    def step():
        cache.reserve(every, count)
        P.append(None, k, v, cache.k[0], cache.v[0], cache.table, cache.lens, cu_q=cu)
        out = P.paged_attention(q, cache.k[0], cache.v[0], cache.table, cache.lens, 0.125, cu_q=cu, max_q=drafts, window=window)
        cache.truncate(every, cache.lens - drafts + kept)
        return out

    if captured:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
    keys, values = [[] for _ in range(rows)], [[] for _ in range(rows)]
    for _ in range(12):
        for x in (q, k, v):
            x.copy_(torch.randn(x.shape, generator=g).bfloat16())
        keep = [rng.randint(0, drafts) for _ in range(rows)]
        kept.copy_(ints(keep))
        if captured:
            graph.replay()
        else:
            out = step()
        for r in range(rows):
            new = slice(r * drafts, (r + 1) * drafts)
            kk, vv = (torch.stack(a + list(b[new])).double().repeat_interleave(h // hk, 1).transpose(0, 1)
                      for a, b in ((keys[r], k.clone()), (values[r], v.clone())))
            s = q[new].double().transpose(0, 1) @ kk.transpose(1, 2) * 0.125
            pos = torch.arange(len(keys[r]), len(keys[r]) + drafts, device="cuda")[:, None]
            key = torch.arange(kk.shape[1], device="cuda")
            hidden = (key > pos) | (key <= pos - window if window else key < 0)
            want = (s.masked_fill(hidden, -math.inf).softmax(-1) @ vv).transpose(0, 1)
            # u for the output and u for P, of at most the largest |v| (below 5); a third for all the rest (2^-11 and less)
            assert float((out[new].double() - want).abs().max()) <= 3 * 5 * 2.0 ** -8
            keys[r] += list(k[new].clone()[: keep[r]])
            values[r] += list(v[new].clone()[: keep[r]])
    P.check()
    lens = [len(x) for x in keys]
    assert cache.lens.tolist() == lens
    assert [sum(p >= 0 for p in r) for r in cache.table.tolist()] == [-(-n // page) for n in lens]
    assert int(cache.refs.sum()) == sum(-(-n // page) for n in lens)
