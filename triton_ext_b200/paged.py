"""A cache of keys and values in pages, and what a serving step does with it (include/b200_paged.h):

  append            the new tokens' k (turned by their positions) and v into their pages, and the turned q
  paged_attention   the new tokens' attention over their sequences' pages: chunks of a prompt, drafted tokens, single tokens
  PagedCache        who holds which page, on the device: reserve, truncate, fork, free, compact, copy_pages

A step is `lens = cache.reserve(rows, counts)`, then for every layer `append` and `paged_attention` with those lengths. Nothing
in a step synchronises, reads the device or depends on the host knowing a length, so a step can be captured in a CUDA graph
and replayed while the sequences grow. What kernels find wrong (a bad page, no free pages) is reported by `check`; a step whose
`reserve` was refused leaves the cache as it was.

torch is used for device memory and streams only. There is no fallback: if the shared library is missing or no B200 is
present the calls raise.
"""
from __future__ import annotations

import ctypes
import struct
from typing import Optional, Sequence

import torch

from . import backend as B
from .rotary import Rope, _call, _overlaps, check  # noqa: F401  (check: part of this module's interface)

_DTYPES = {torch.float16: B.TXD_F16, torch.bfloat16: B.TXD_BF16}
MAX_LIST = 4096  # rows in one reserve
_INT_MAX = 2 ** 31 - 1

_lib_cache = None


def _lib() -> ctypes.CDLL:
    global _lib_cache
    if _lib_cache is None:
        lib = B.load_library()
        vp, i32, i64 = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64
        for name, args, res in (
                ("tx_paged_append", [vp, vp, vp, vp], ctypes.c_int),
                ("tx_paged_attention", [vp, vp, vp, i64, vp], ctypes.c_int),
                ("tx_paged_attention_workspace", [vp, vp], i64),
                ("tx_pages_workspace", [vp, i32], i64),
                ("tx_pages_free", [vp, vp, i32, vp], ctypes.c_int),
                ("tx_pages_truncate", [vp, vp, vp, i32, vp], ctypes.c_int),
                ("tx_pages_fork", [vp, vp, vp, i32, vp, vp], ctypes.c_int),
                ("tx_pages_reserve", [vp, vp, vp, i32, vp, vp], ctypes.c_int),
                ("tx_pages_reserve_lens", [vp, vp, vp, i32, vp, vp, vp], ctypes.c_int),
                ("tx_pages_compact", [vp, vp, vp], ctypes.c_int),
                ("tx_pages_copy", [vp, vp, vp, i32, vp], ctypes.c_int)):
            f = getattr(lib, name)
            f.argtypes, f.restype = args, res
        lib.tx_paged_last_error.restype = ctypes.c_char_p
        lib.tx_paged_kernel_launches.restype = ctypes.c_uint64
        _lib_cache = lib
    return _lib_cache


def _invalid(text: str):
    raise B.DotError(B.TXD_ERR_INVALID, text)


def kernel_launches() -> int:
    return int(_lib().tx_paged_kernel_launches())


_VIEW = struct.Struct("2P6qPq2P8i")
_APPEND = struct.Struct("4P8q2i")
_ATTN = struct.Struct("3P4q5if")
_STATE = struct.Struct("2Pq3P6i")


def _view(k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor, kv_lens: torch.Tensor,
          cu_q: Optional[torch.Tensor], device: int) -> tuple[bytes, int, int, int]:
    """(the packed tx_paged_view, batch, kv_heads, head_dim); `device` as `Tensor.get_device` numbers it."""
    dtype, code = k_pages.dtype, _DTYPES.get(k_pages.dtype)
    shape = k_pages.shape
    if len(shape) != 4 or v_pages.shape != shape or v_pages.dtype != dtype:
        _invalid("k_pages and v_pages must be [pages, page_size, kv_heads, head_dim] of one shape and type")
    if code is None:
        raise B.DotError(B.TXD_ERR_UNSUPPORTED, f"cache dtype {dtype}: f16 and bf16 are built")
    if (k_pages.get_device() != device or v_pages.get_device() != device or page_table.get_device() != device or
            kv_lens.get_device() != device):
        _invalid("the cache, page_table and kv_lens must be on the device of the new tokens")
    pages, page_size, heads, d = shape
    k0, k1, k2, k3 = k_pages.stride()
    v0, v1, v2, v3 = v_pages.stride()
    if k3 != 1 or v3 != 1:
        _invalid("head_dim must be the contiguous dimension of k_pages and v_pages")
    table_shape, table_stride = page_table.shape, page_table.stride()
    if page_table.dtype != torch.int32 or len(table_shape) != 2 or (table_stride[1] != 1 and table_shape[1] > 1):
        _invalid("page_table must be int32 [batch, pages of a sequence] with unit column stride")
    batch, width = table_shape
    if kv_lens.dtype != torch.int32 or kv_lens.shape != (batch,) or (batch > 1 and kv_lens.stride(0) != 1):
        _invalid(f"kv_lens must be a contiguous int32 vector of {batch} lengths")
    cu = 0
    if cu_q is not None:
        if (cu_q.dtype != torch.int32 or cu_q.shape != (batch + 1,) or (batch > 0 and cu_q.stride(0) != 1) or
                cu_q.get_device() != device):
            _invalid(f"cu_q must be a contiguous int32 vector of {batch + 1} offsets on the device of the new tokens")
        cu = cu_q.data_ptr()
    return _VIEW.pack(k_pages.data_ptr(), v_pages.data_ptr(), k0, k1, k2, v0, v1, v2, page_table.data_ptr(), table_stride[0],
                      kv_lens.data_ptr(), cu, batch, width, pages, page_size, heads, d, code, 0), batch, heads, d


def _token_strides(x: torch.Tensor, name: str, tokens: int, head_dim: int, like: torch.Tensor, device: int) -> tuple[int, int]:
    shape, s = x.shape, x.stride()
    if len(shape) != 3 or shape[0] != tokens or shape[2] != head_dim or x.dtype != like.dtype or x.get_device() != device:
        _invalid(f"{name} must be [tokens, heads, head_dim] = [{tokens}, *, {head_dim}] of the cache's type and device")
    if s[2] != 1 and head_dim > 1:
        _invalid(f"head_dim must be the contiguous dimension of {name}")
    return s[0], s[1]


def _not_cuda(q: torch.Tensor):
    raise B.DotError(B.TXD_ERR_NO_DEVICE, f"CUDA tensors are wanted, got {q.device}: there is no CPU path")


class _Forward(torch.autograd.Function):
    """The result of an operator that has no gradient, for inputs that want one: a backward that reaches it raises."""

    @staticmethod
    def forward(ctx, name, out, m, *inputs):
        ctx.name = name
        return out, m

    @staticmethod
    def backward(ctx, *grads):
        raise B.DotError(B.TXD_ERR_UNSUPPORTED, f"{ctx.name} has no gradient: it is for serving (use it under torch.no_grad)")


def _without_gradient(name: str, out: torch.Tensor, m: Optional[torch.Tensor], *inputs: torch.Tensor):
    if out.requires_grad:  # an input that was written in place: what a backward has kept of it is gone
        torch.autograd.graph.increment_version(out)
    return _Forward.apply(name, out, m, *inputs)


def append(q: Optional[torch.Tensor], k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
           page_table: torch.Tensor, kv_lens: torch.Tensor, *, rope: Optional[Rope] = None, cu_q: Optional[torch.Tensor] = None,
           out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """Write the new tokens' k and v to their places in the cache and return q, q and k turned by their positions if a `rope`
    is given. One launch on the current CUDA stream.

    q, k, v: [tokens, heads, head_dim], any strides with head_dim contiguous (parts of one projection's output, say); q may
    be None. k_pages, v_pages: [pages, page_size, kv_heads, head_dim]. page_table: int32 [batch, width]. kv_lens: int32
    [batch], the sequences' lengths WITH the new tokens. cu_q: int32 [batch + 1], where each sequence's new tokens start
    (None: one token for each sequence, in order). Sequence b's new tokens take its last positions. out: where the turned q
    goes (q itself is allowed). Tokens behind cu_q[-1] are left alone: their rows of `out` are not written.
    There is no gradient: a backward through the result raises, and the cache carries none."""
    lib = _lib_cache or _lib()
    device = k.get_device()
    if device < 0:
        _not_cuda(k)
    view, batch, kv_heads, d = _view(k_pages, v_pages, page_table, kv_lens, cu_q, device)
    shape = k.shape
    if len(shape) != 3 or shape[1] != kv_heads or v.shape != shape or shape[2] != d:
        _invalid("k and v must be [tokens, kv_heads, head_dim] with the cache's heads and head_dim")
    tokens = shape[0]
    if cu_q is None and tokens != batch:
        _invalid(f"without cu_q there is one new token for each of the {batch} sequences, got {tokens}")
    ks, vs = _token_strides(k, "k", tokens, d, k_pages, device), _token_strides(v, "v", tokens, d, k_pages, device)
    q_ptr, o_ptr, q_heads, qs, os_ = 0, 0, 0, (0, 0), (0, 0)
    if q is not None:
        qs, q_heads = _token_strides(q, "q", tokens, d, k_pages, device), q.shape[1]
        if out is None:
            out = torch.empty_like(q)
            os_ = out.stride()
            if os_[2] != 1:  # q is made of overlapping windows: its layout is none to follow
                out = torch.empty_like(q, memory_format=torch.contiguous_format)
                os_ = out.stride()
        else:
            os_ = _token_strides(out, "out", tokens, d, k_pages, device)
            if out.shape != q.shape or _overlaps(out):
                _invalid("out must have the shape of q and not be an expanded tensor, nor overlap itself in another way")
        q_ptr, o_ptr = q.data_ptr(), out.data_ptr()
    elif out is not None:
        _invalid("out is for the turned q: there is none")
    if rope is not None and rope.rotary_dim > d:
        _invalid(f"rotary_dim {rope.rotary_dim} exceeds head_dim {d}")
    problem = _APPEND.pack(q_ptr, k.data_ptr(), v.data_ptr(), o_ptr, qs[0], qs[1], ks[0], ks[1], vs[0], vs[1], os_[0], os_[1],
                           tokens, q_heads)
    _call(device, lib.tx_paged_append, view, rope._packed if rope is not None else None, problem)
    if q is not None and (q.requires_grad or k.requires_grad or v.requires_grad) and torch.is_grad_enabled():
        out, _ = _without_gradient("append", out, None, q, k, v)
    return out


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                    kv_lens: torch.Tensor, sm_scale: float, *, cu_q: Optional[torch.Tensor] = None,
                    max_q: Optional[int] = None, causal: bool = True, window: int = 0, out: Optional[torch.Tensor] = None,
                    return_m: bool = False):
    """Attention of new tokens over their sequences' pages, on the current CUDA stream; see `append` for the arguments that
    describe the cache and the batch.

    q: [tokens, heads, head_dim], heads a multiple of kv_heads (query head h reads key head h // (heads // kv_heads)). A new
    token sees the keys up to its own position (all keys of its sequence if not `causal`), with `window` > 0 the last `window`
    of them. max_q: a bound on the new tokens of one sequence, needed with cu_q. A row that sees nothing gives zeros.
    Returns the output, with `return_m` also [tokens, heads] fp32 of max + log2(sum) (base 2), -inf where nothing is seen.
    Rows behind cu_q[-1] are left alone. There is no gradient: a backward through the result raises."""
    lib = _lib_cache or _lib()
    device = q.get_device()
    if device < 0:
        _not_cuda(q)
    view, batch, _, head_dim = _view(k_pages, v_pages, page_table, kv_lens, cu_q, device)
    shape = q.shape
    if len(shape) != 3 or shape[2] != head_dim:
        _invalid(f"q must be [tokens, heads, head_dim] with the cache's head_dim {head_dim}, got {tuple(shape)}")
    tokens, heads, d = shape
    qs = _token_strides(q, "q", tokens, d, k_pages, device)
    if 0 in qs:  # expanded heads or tokens
        q = q.contiguous()
        qs = q.stride()
    if cu_q is None:
        if tokens != batch:
            _invalid(f"without cu_q there is one new token for each of the {batch} sequences, got {tokens}")
        max_q = 1
    elif max_q is None:
        _invalid("cu_q needs max_q, a bound on the new tokens of one sequence")
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        os_ = out.stride()
    else:
        os_ = _token_strides(out, "out", tokens, d, k_pages, device)
        if out.shape != shape or _overlaps(out):
            _invalid("out must have the shape of q and not be an expanded tensor, nor overlap itself in another way")
    m = torch.empty((tokens, heads), dtype=torch.float32, device=q.device) if return_m else None
    problem = _ATTN.pack(q.data_ptr(), out.data_ptr(), m.data_ptr() if return_m else 0, qs[0], qs[1], os_[0], os_[1], tokens,
                         heads, min(max(max_q, -1), _INT_MAX), 1 if causal else 0, min(max(window, -1), _INT_MAX), sm_scale)
    size = lib.tx_paged_attention_workspace(view, problem)
    ws = q.new_empty((size + 1) // 2)  # 16-bit values
    _call(device, lib.tx_paged_attention, view, problem, ws.data_ptr(), size)
    if (q.requires_grad or k_pages.requires_grad or v_pages.requires_grad) and torch.is_grad_enabled():
        out, m = _without_gradient("paged_attention", out, m, q, k_pages, v_pages)
    return (out, m) if return_m else out


class PagedCache:
    """A cache of `layers` pools of pages and the device-side record of who holds them.

    k, v    [layers, pages, page_size, kv_heads, head_dim], contiguous, f16 or bf16; `k[layer]` is what `append` and
            `paged_attention` take
    table   int32 [rows, width]: the pages of each row (a sequence), -1 where there is none
    lens    int32 [rows]: its tokens (to be read; the operations change it). A step takes its lengths from `reserve` instead
    refs    int32 [pages]: in how many table cells a page stands; 0: free

    The operations take rows as int32 CUDA vectors, run in stream order and never synchronise; a row outside the table is
    passed over (by `reserve`: nothing is done at all) and reported by `check`."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, lens: torch.Tensor, refs: torch.Tensor):
        if k.dim() != 5 or v.shape != k.shape or v.dtype != k.dtype or k.dtype not in _DTYPES:
            _invalid("k and v must be [layers, pages, page_size, kv_heads, head_dim] of one shape and type, f16 or bf16")
        for name, t, dims in (("table", table, 2), ("lens", lens, 1), ("refs", refs, 1)):
            if t.dtype != torch.int32 or t.dim() != dims:
                _invalid(f"{name} must be int32 with {dims} dimension(s)")
        if lens.shape[0] != table.shape[0] or refs.shape[0] != k.shape[1]:
            _invalid("lens must have one entry for each row of table, refs one for each page")
        for name, t in (("k", k), ("v", v), ("table", table), ("lens", lens), ("refs", refs)):
            if not t.is_contiguous():
                _invalid(f"{name} must be contiguous")
            if t.device != k.device:
                _invalid("k, v, table, lens and refs must be on one device")
        self.k, self.v, self.table, self.lens, self.refs = k, v, table, lens, refs
        layers, pages, page_size, heads, d = k.shape
        self.page_size = page_size
        self._workspaces = {}  # their sizes, by the length of a list
        self._device = k.get_device()  # below zero: not a CUDA device
        self._own = tuple(x for t in (table, lens, refs) for x in (t.data_ptr(), t.data_ptr() + 4 * t.numel()))
        self._state = _STATE.pack(k.data_ptr(), v.data_ptr(), page_size * heads * d * k.element_size(), table.data_ptr(),
                                  lens.data_ptr(), refs.data_ptr(), layers, pages, page_size, table.shape[0], table.shape[1], 0)

    @classmethod
    def create(cls, pages: int, page_size: int, kv_heads: int, head_dim: int, *, rows: int, width: int, layers: int = 1,
               dtype: torch.dtype = torch.bfloat16, device="cuda") -> "PagedCache":
        """An empty cache; the pools are not initialised."""
        k, v = (torch.empty((layers, pages, page_size, kv_heads, head_dim), dtype=dtype, device=device) for _ in range(2))
        table = torch.full((rows, width), -1, dtype=torch.int32, device=k.device)
        return cls(k, v, table, torch.zeros(rows, dtype=torch.int32, device=k.device),
                   torch.zeros(pages, dtype=torch.int32, device=k.device))

    def _list(self, x: torch.Tensor, name: str, n: Optional[int] = None) -> torch.Tensor:
        if self._device < 0:
            _not_cuda(self.k)
        shape = x.shape
        if x.dtype != torch.int32 or len(shape) != 1 or x.get_device() != self._device or (n is not None and shape[0] != n):
            _invalid(f"{name} must be an int32 vector{f' of {n}' if n is not None else ''} on the device of the cache")
        # a part of the state (lengths as counts, say) would change under the kernel that reads it
        at, (t0, t1, l0, l1, r0, r1) = x.data_ptr(), self._own
        end = at + 4 * shape[0]
        if not x.is_contiguous() or l0 < end and at < l1 or t0 < end and at < t1 or r0 < end and at < r1:
            return x.clone(memory_format=torch.contiguous_format)
        return x

    def _workspace(self, lib, n: int) -> torch.Tensor:
        ints = self._workspaces.get(n)
        if ints is None:
            ints = self._workspaces[n] = (lib.tx_pages_workspace(self._state, n) + 3) // 4
        return self.refs.new_empty(ints)

    def free(self, rows: torch.Tensor) -> None:
        """Give the pages of the listed rows back (those that no other row holds become free) and empty the rows."""
        lib, rows = _lib_cache or _lib(), self._list(rows, "rows")
        _call(self._device, lib.tx_pages_free, self._state, rows.data_ptr(), rows.shape[0])

    def truncate(self, rows: torch.Tensor, keep: torch.Tensor) -> None:
        """Cut row rows[i] to keep[i] tokens (drafted tokens that were not accepted) and give the pages behind them back; a row
        that is no longer keeps its length. Rows are shortened by this, not by writing to `lens`."""
        lib, rows = _lib_cache or _lib(), self._list(rows, "rows")
        keep = self._list(keep, "keep", rows.shape[0])
        _call(self._device, lib.tx_pages_truncate, self._state, rows.data_ptr(), keep.data_ptr(), rows.shape[0])

    def fork(self, dst: torch.Tensor, src: torch.Tensor) -> None:
        """Row dst[i] becomes what row src[i] was before the call, sharing its pages. Rows may be both (the reordering of a
        beam search); what a destination held is given back; of a destination listed twice the last one holds."""
        lib, dst = _lib_cache or _lib(), self._list(dst, "dst")
        n = dst.shape[0]
        src = self._list(src, "src", n)
        ws = self._workspace(lib, n)
        _call(self._device, lib.tx_pages_fork, self._state, dst.data_ptr(), src.data_ptr(), n, ws.data_ptr())

    def reserve(self, rows: torch.Tensor, counts: torch.Tensor) -> torch.Tensor:
        """Make room for counts[i] more tokens in row rows[i] and add them to its length, before they are appended. New pages
        are the lowest free ones in list order. A partly filled last page that other rows share is copied first (all layers);
        of the listed rows that alone share one, the last keeps it.

        Returns the rows' new lengths, int32 [n], for the step that follows: `kv_lens` of `append` and `paged_attention`, and
        less the drafts that were not accepted, `keep` of `truncate`. Where there is no room nothing is done for any row, and
        they are far below zero: append then writes nothing to the cache, attention gives zeros, truncate cuts nothing, and
        `check` reports it. (`lens` stays as it was: an append with it would overwrite the rows' last tokens.)"""
        lib, rows = _lib_cache or _lib(), self._list(rows, "rows")
        n = rows.shape[0]
        counts = self._list(counts, "counts", n)
        ws, lens = self._workspace(lib, n), rows.new_empty(n)
        _call(self._device, lib.tx_pages_reserve_lens, self._state, rows.data_ptr(), counts.data_ptr(), n, lens.data_ptr(),
              ws.data_ptr())
        return lens

    def compact(self) -> None:
        """Move pages (all layers) so that the used ones are the lowest, the fewest that do it; the table follows."""
        lib = _lib_cache or _lib()
        if self._device < 0:
            _not_cuda(self.k)
        ws = self._workspace(lib, 0)
        _call(self._device, lib.tx_pages_compact, self._state, ws.data_ptr())

    def copy_pages(self, src: Sequence[int], dst: Sequence[int]) -> None:
        """Copy the contents of pages src[i] to dst[i] in every layer. Host lists; no page may be a destination twice, or
        source and destination."""
        lib, n = _lib(), len(src)
        if self._device < 0:
            _not_cuda(self.k)
        if len(dst) != n:
            _invalid("src and dst must be of one length")
        pages = self.k.shape[1]
        for x in (*src, *dst):
            if not 0 <= int(x) < pages:
                _invalid(f"page {x} is outside the {pages} pages")
        _call(self._device, lib.tx_pages_copy, self._state, (ctypes.c_int32 * n)(*src), (ctypes.c_int32 * n)(*dst), n)
