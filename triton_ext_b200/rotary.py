"""Rotary positions on the GPU (include/b200_paged.h, `tx_rotary`): q and k turned by their positions before
`attention.attention`, with the gradient (the same turn backwards).

`Rope` describes the rotation: how many columns of a head turn, how they pair up, and the angle a pair turns by per
position. Angles are kept as 64-bit fractions of a whole turn, so position 2^31 is as exact as position 1 (2^40: to 2^-25 of a
turn; each doubling from there loses a bit).

torch is used for device memory, streams and autograd only. There is no fallback: if the shared library is missing or no
B200 is present the calls raise.
"""
from __future__ import annotations

import ctypes
import math
import struct
from fractions import Fraction
from typing import Optional, Sequence

import torch

from . import backend as B

MAX_PAIRS = 128
_DTYPES = {torch.float16: B.TXD_F16, torch.bfloat16: B.TXD_BF16, torch.float32: B.TXD_F32}
# 1 / (2 pi) to 100 binary digits: a product with an exact double gives all 64 bits of a turn's fraction
_INV_2PI_BITS = 201752859139730814931732094791
_INV_2PI = Fraction(_INV_2PI_BITS, 1 << 100)


def _turns(w: float) -> int:
    """w / (2 pi) as a 64-bit fraction of a turn, rounded to nearest."""
    n, d = w.as_integer_ratio()  # d is a power of two
    return (((n * _INV_2PI_BITS >> (d.bit_length() + 34)) + 1) >> 1) & 0xFFFFFFFFFFFFFFFF

_lib_cache = None


def _lib() -> ctypes.CDLL:
    global _lib_cache
    if _lib_cache is None:
        lib = B.load_library()
        vp = ctypes.c_void_p
        lib.tx_rotary.argtypes = [vp, vp, vp, vp]
        lib.tx_rotary.restype = ctypes.c_int
        lib.tx_paged_last_error.restype = ctypes.c_char_p
        lib.tx_paged_kernel_launches.restype = ctypes.c_uint64
        lib.tx_paged_check.argtypes = [vp]
        lib.tx_paged_check.restype = ctypes.c_int
        _lib_cache = lib
    return _lib_cache


def kernel_launches() -> int:
    return int(_lib().tx_paged_kernel_launches())


class Rope:
    """Rotary positions of the first `rotary_dim` columns of a head: pair i turns by `position * w_i` radians,
    w_i = base ** (-2 i / rotary_dim). Pairs are columns (i, i + rotary_dim / 2), or (2 i, 2 i + 1) if `interleaved`.

    scaling, for contexts `factor` times longer than a model was trained on:
      None      as above
      "linear"  positions divided by `factor`: w_i / factor
      "base"    the base stretched by factor ** (rotary_dim / (rotary_dim - 2)): the slowest pair ends up at w / factor, the
                fastest keeps its speed
      "parts"   pairs that turn more than `high` times within `original_len` positions keep w_i, those that turn less than
                `low` times get w_i / factor, and those between a mixture, linear in the number of turns

    `magnitude` multiplies the turned columns; None: 0.1 ln(factor) + 1 for "parts", else 1.
    `frequencies` (radians per position, one for each pair) replaces the formula.
    """

    def __init__(self, rotary_dim: int, *, base: float = 10000.0, interleaved: bool = False, scaling: Optional[str] = None,
                 factor: float = 1.0, original_len: int = 0, low: float = 1.0, high: float = 32.0,
                 magnitude: Optional[float] = None, frequencies: Optional[Sequence[float]] = None):
        if rotary_dim < 2 or rotary_dim % 2 or rotary_dim > 2 * MAX_PAIRS:
            raise ValueError(f"rotary_dim must be even and 2 .. {2 * MAX_PAIRS}, got {rotary_dim}")
        if scaling not in (None, "linear", "base", "parts"):
            raise ValueError(f"scaling must be None, 'linear', 'base' or 'parts', got {scaling!r}")
        if not (base > 0 and factor > 0 and math.isfinite(base) and math.isfinite(factor)):
            raise ValueError("base and factor must be positive and finite")
        pairs = rotary_dim // 2
        if frequencies is not None:
            if scaling is not None:
                raise ValueError("frequencies are given as they are: no scaling with them")
            freq = [float(w) for w in frequencies]
            if len(freq) != pairs or not all(math.isfinite(w) for w in freq):
                raise ValueError(f"{pairs} finite frequencies are wanted")
        else:
            if scaling == "base":
                if rotary_dim == 2:
                    raise ValueError("scaling 'base' needs rotary_dim > 2")
                base = base * factor ** (rotary_dim / (rotary_dim - 2))
            freq = [base ** (-2.0 * i / rotary_dim) for i in range(pairs)]
            if scaling == "linear":
                freq = [w / factor for w in freq]
            elif scaling == "parts":
                if original_len < 1 or not low < high:
                    raise ValueError("scaling 'parts' needs original_len >= 1 and low < high")
                kept = [min(1.0, max(0.0, (original_len * w / (2 * math.pi) - low) / (high - low))) for w in freq]
                freq = [w * (g + (1.0 - g) / factor) for w, g in zip(freq, kept)]
        if magnitude is None:
            magnitude = 0.1 * math.log(factor) + 1.0 if scaling == "parts" else 1.0
        self.rotary_dim, self.interleaved, self.frequencies, self.magnitude = rotary_dim, interleaved, tuple(freq), magnitude
        turns = [_turns(w) for w in freq]
        self._packed = struct.pack(f"iifi{MAX_PAIRS}Q", rotary_dim, int(interleaved), magnitude, 0,
                                   *(turns + [0] * (MAX_PAIRS - pairs)))


_HEAD = struct.Struct("6i2q2i")
_PART = struct.Struct("2P6q2i")
_NO_PART = _PART.pack(0, 0, 0, 0, 0, 0, 0, 0, 0, 0)


def _overlaps(x: torch.Tensor) -> bool:
    """Whether elements of x may share their memory (expanded tensors, overlapping windows): no result can stand there."""
    end = 0
    for s, n in sorted((s, n) for n, s in zip(x.shape, x.stride()) if n > 1):
        if s <= end:
            return True
        end += s * (n - 1)
    return False


def _check_out(out: torch.Tensor, x: torch.Tensor, name: str) -> None:
    if out.shape != x.shape or out.dtype != x.dtype or out.device != x.device or out.stride(-1) != 1:
        raise B.DotError(B.TXD_ERR_INVALID, f"{name} must have its input's shape, type and device, HEAD_DIM contiguous")
    if _overlaps(out):
        raise B.DotError(B.TXD_ERR_INVALID, f"{name} must not be an expanded tensor, nor overlap itself in another way")


def _part(x: torch.Tensor, out: Optional[torch.Tensor], heads: int, name: str):
    """The packed tx_rotary_part of x, where its result goes, and what it is read from (x or a copy of it): to be kept until
    the launch, or its memory may be the next copy's."""
    if out is not None:
        _check_out(out, x, name)
    a = x.stride()
    if a[3] != 1:
        x = x.contiguous()
        a = x.stride()
    if out is None:
        out = torch.empty_like(x)
        if out.stride(3) != 1:  # x is made of overlapping windows: its layout is none to follow
            out = torch.empty_like(x, memory_format=torch.contiguous_format)
    b = out.stride()
    return _PART.pack(x.data_ptr(), out.data_ptr(), a[0], a[1], a[2], b[0], b[1], b[2], heads, 0), out, x


def rotary_forward(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, rope: Rope, *, inverse: bool = False,
                   out_q: Optional[torch.Tensor] = None, out_k: Optional[torch.Tensor] = None):
    """(q, k) turned by their positions, on the current CUDA stream; `k` may be None (the second result then is, too).

    q, k: [Z, H, N_CTX, HEAD_DIM] of one 16-bit type or float32 and any strides with HEAD_DIM contiguous (others are
    copied); k may have its own number of heads. positions: int32 or int64, [N_CTX] or [Z, N_CTX]. out_q, out_k: where the
    results go (the inputs themselves are allowed: in place). inverse: turn backwards. No gradient is recorded: `rotary` is the
    differentiable form."""
    lib = _lib_cache or _lib()
    shape = q.shape
    device = q.get_device()
    if len(shape) != 4:
        raise B.DotError(B.TXD_ERR_INVALID, "q must be [Z, H, N_CTX, HEAD_DIM]")
    if device < 0:
        raise B.DotError(B.TXD_ERR_NO_DEVICE, "q must be a CUDA tensor: there is no CPU path")
    z, heads, n, d = shape
    dtype = _DTYPES.get(q.dtype)
    if dtype is None:
        raise B.DotError(B.TXD_ERR_UNSUPPORTED, f"rotary dtype {q.dtype}: f16, bf16 and f32 are built")
    if rope.rotary_dim > d:
        raise B.DotError(B.TXD_ERR_INVALID, f"rotary_dim {rope.rotary_dim} exceeds HEAD_DIM {d}")
    wide = positions.dtype == torch.int64
    if not (wide or positions.dtype == torch.int32) or positions.get_device() != device:
        raise B.DotError(B.TXD_ERR_INVALID, "positions must be int32 or int64 on the device of q")
    pos_shape, pos_stride = positions.shape, positions.stride()
    if pos_shape == (n,):
        pos_stride = (0, pos_stride[0])
    elif pos_shape != (z, n):
        raise B.DotError(B.TXD_ERR_INVALID, f"positions must be [{n}] or [{z}, {n}], got {tuple(pos_shape)}")
    first, out_q, q = _part(q, out_q, heads, "out_q")
    if k is None:
        parts, second, out_k = 1, _NO_PART, None
    else:
        ks = k.shape
        if len(ks) != 4 or ks[0] != z or ks[2] != n or ks[3] != d or k.dtype != q.dtype or k.get_device() != device:
            raise B.DotError(B.TXD_ERR_INVALID, "q and k must agree in all but their heads, and in type and device")
        parts = 2
        second, out_k, k = _part(k, out_k, ks[1], "out_k")
    packed = _HEAD.pack(z, n, d, dtype, 1 if inverse else 0, 1 if wide else 0, pos_stride[0], pos_stride[1], parts, 0) + first + second
    _call(device, lib.tx_rotary, rope._packed, packed, positions.data_ptr())
    return out_q, out_k


def _call(index: int, function, *args) -> None:
    """One C entry point on the current stream of device `index` (made the current device meanwhile); raises if it fails. The
    stream is the entry point's last argument."""
    if torch.cuda.current_device() == index:
        rc = function(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            rc = function(*args, torch._C._cuda_getCurrentRawStream(index))
    if rc:
        raise B.DotError(rc, _lib().tx_paged_last_error().decode())


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, rope, inverse):
        ctx.save_for_backward(positions)
        ctx.rope, ctx.inverse = rope, inverse
        ctx.set_materialize_grads(False)
        return rotary_forward(q, k, positions, rope, inverse=inverse)

    @staticmethod
    def backward(ctx, gq, gk):
        (positions,) = ctx.saved_tensors
        rope, inverse = ctx.rope, not ctx.inverse
        # the gradient of a turn is the turn backwards; where it is to be differentiated again, as a function itself
        again = torch.is_grad_enabled()

        def turn(a, b):
            return _Rotary.apply(a, b, positions, rope, inverse) if again else rotary_forward(a, b, positions, rope, inverse=inverse)

        if gq is not None:
            gq, gk = turn(gq, gk)
        elif gk is not None:
            gk = turn(gk, None)[0]
        return gq, gk, None, None, None


def rotary(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, rope: Rope):
    """The differentiable `rotary_forward`: (q, k) turned by their positions, for `attention.attention`.

    A backward may be captured in a CUDA graph. As for every autograd function, no eager graph of the same leaves may be
    alive then: PyTorch would order the capture with that graph's stream, and the capture fails."""
    return _Rotary.apply(q, k, positions, rope, False)


def check(device=None) -> None:
    """Synchronise the current stream and raise for what the rotary, append, paged attention and page kernels found wrong
    on the device since the last check, on this stream and, as far as they have run, on others. Nothing goes unreported, but
    where several threads check one device, any of them may be the one that is told."""
    index = None if device is None else device if isinstance(device, int) else torch.device(device).index
    lib = _lib()
    _call(torch.cuda.current_device() if index is None else index, lib.tx_paged_check)
