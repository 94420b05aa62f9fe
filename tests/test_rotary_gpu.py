"""Rotary positions on the GPU against their definition in 64 bits (complex numbers, angles in double).

Tolerance, per element: half a step of the output type, plus what the kernel's fp32 arithmetic may be off. The angle is an
integer product, cut to 32 bits (2^-32 of a turn) and rounded to 24 (2^-25 half turns: 9.4e-8 rad); sincospi is within 2
steps (2 * 2^-24); the magnitude's product and the two products and the sum round once each (4 * 2^-24). Together under
6.0e-7 of magnitude * (|x1| + |x2|); 2^-20 is used."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

f16, bf16, f32 = torch.float16, torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def R(built_libs, cuda_device):
    from triton_ext_b200 import rotary
    return rotary


def turned64(x, pos, rope, inverse=False):
    """x [Z, H, N, D] in double, turned as complex numbers; and |x1| + |x2| per element for the tolerance."""
    x = x.double()
    rd = rope.rotary_dim
    w = torch.tensor(rope.frequencies, dtype=torch.float64, device=x.device)
    pos = pos.double()
    pos = pos[None, None, :, None] if pos.dim() == 1 else pos[:, None, :, None]
    phase = pos * w * (-1 if inverse else 1)
    unit = torch.polar(torch.full_like(phase, rope.magnitude), phase)
    pairs = (slice(0, rd, 2), slice(1, rd, 2)) if rope.interleaved else (slice(0, rd // 2), slice(rd // 2, rd))
    z = torch.complex(x[..., pairs[0]], x[..., pairs[1]]) * unit
    out, size = x.clone(), torch.zeros_like(x)
    out[..., pairs[0]], out[..., pairs[1]] = z.real, z.imag
    both = (x[..., pairs[0]].abs() + x[..., pairs[1]].abs()) * rope.magnitude
    size[..., pairs[0]], size[..., pairs[1]] = both, both
    return out, size


def close(got, want, size):
    eps = torch.finfo(got.dtype).eps / 2
    tiny = torch.finfo(got.dtype).smallest_normal * eps  # half a step among the subnormals
    err = (got.double() - want).abs()
    tol = want.abs() * eps + size * 2.0 ** -20 * (1 + eps) + tiny
    assert bool((err <= tol).all()), f"worst {float((err / tol.clamp(min=1e-300)).max())} of the tolerance"


def tensor(shape, dtype, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


CASES = [
    # z, h, hk, n, d, rotary_dim, interleaved, dtype, first position
    (1, 1, 1, 1, 64, 64, False, bf16, 0),
    (2, 4, 2, 33, 128, 128, False, bf16, 7),
    (3, 5, 1, 77, 64, 32, True, f16, 120000),
    (1, 3, 3, 130, 128, 96, True, bf16, 1 << 20),
    (2, 2, 1, 9, 64, 20, False, f16, 3),          # 10 pairs: vectors of 2
    (2, 2, 1, 9, 66, 6, True, f16, 3),            # 3 pairs: single values
    (1, 2, 2, 11, 33, 2, False, f32, 2),          # odd head dimension
    (1, 8, 2, 600, 128, 128, True, f32, 2_000_000_000),
    (1, 1, 1, 5, 256, 256, False, f16, 1),
    (1, 1, 1, 5, 512, 256, False, bf16, 1),
]


@pytest.mark.parametrize("z,h,hk,n,d,rd,inter,dtype,first", CASES)
@pytest.mark.parametrize("inverse", [False, True])
def test_against_the_definition(R, z, h, hk, n, d, rd, inter, dtype, first, inverse):
    rope = R.Rope(rd, interleaved=inter)
    q, k = tensor((z, h, n, d), dtype, 1), tensor((z, hk, n, d), dtype, 2)
    pos = torch.arange(first, first + n, device="cuda")
    for p in (pos, pos.to(torch.int32), pos[None].repeat(z, 1)):
        oq, ok = R.rotary_forward(q, k, p, rope, inverse=inverse)
        close(oq, *turned64(q, p, rope, inverse))
        close(ok, *turned64(k, p, rope, inverse))


@pytest.mark.parametrize("kw", [dict(scaling="linear", factor=4.0), dict(scaling="base", factor=8.0),
                                dict(scaling="parts", factor=8.0, original_len=4096),
                                dict(scaling="parts", factor=8.0, original_len=8192, low=1.0, high=4.0, magnitude=1.0),
                                dict(frequencies=[0.5 / (i + 1) for i in range(32)])])
def test_scalings_against_the_definition(R, kw):
    rope = R.Rope(64, **kw)
    q = tensor((1, 4, 50, 64), bf16, 3)
    pos = torch.arange(50, device="cuda") * 4099
    oq, none = R.rotary_forward(q, None, pos, rope)
    assert none is None
    close(oq, *turned64(q, pos, rope))


def test_negative_and_repeated_positions(R):
    rope = R.Rope(64)
    q = tensor((2, 2, 6, 64), f16, 4)
    pos = torch.tensor([[0, 0, -1, -70000, 5, 5], [1, 2, 3, 2 ** 40, -2 ** 40, 0]], device="cuda")
    close(R.rotary_forward(q, None, pos, rope)[0], *turned64(q, pos, rope))


def test_far_positions_agree_with_exact_fractions(R):
    """At 2^40 the product position * frequency in double has lost 2^-13 rad: the angle from whole numbers instead."""
    from fractions import Fraction
    rope = R.Rope(2, frequencies=[0.7316888])
    p = 2 ** 40 + 12345
    x = torch.zeros(1, 1, 1, 2, device="cuda")
    x[..., 0] = 1
    got = R.rotary_forward(x, None, torch.tensor([p], device="cuda"), rope)[0].flatten().tolist()
    turns = Fraction(0.7316888) * p * R._INV_2PI
    a = 2 * math.pi * float(turns - int(turns))
    assert abs(got[0] - math.cos(a)) < 2.0 ** -20 and abs(got[1] - math.sin(a)) < 2.0 ** -20


def test_strides_in_place_and_outputs(R):
    rope = R.Rope(32, interleaved=True)
    buf = tensor((2, 19, 6, 64), bf16, 5)                      # [Z, N, H, D] as a projection leaves it
    q, k = buf[:, :, :4].transpose(1, 2), buf[:, :, 4:5].transpose(1, 2)
    pos = torch.arange(19, device="cuda")
    want_q, want_k = turned64(q, pos, rope), turned64(k, pos, rope)
    rest = buf[:, :, 5:].clone()
    oq, ok = R.rotary_forward(q, k, pos, rope)
    close(oq, *want_q)
    close(ok, *want_k)
    assert oq.shape == q.shape and ok.shape == k.shape
    iq, ik = R.rotary_forward(q, k, pos, rope, out_q=q, out_k=k)  # in place
    assert iq.data_ptr() == q.data_ptr() and torch.equal(q, oq) and torch.equal(k, ok)
    assert torch.equal(buf[:, :, 5:], rest)
    # an expanded input, and one whose last dimension is strided
    e = tensor((1, 1, 19, 64), bf16, 6).expand(3, 4, 19, 64)
    close(R.rotary_forward(e, None, pos, rope)[0], *turned64(e, pos, rope))
    s = tensor((2, 3, 64, 19), bf16, 7).transpose(2, 3)
    close(R.rotary_forward(s, None, pos, rope)[0], *turned64(s, pos, rope))
    # a misaligned start
    m = tensor((2 * 3 * 19 * 64 + 1,), f16, 8)[1:].view(2, 3, 19, 64)
    close(R.rotary_forward(m, None, pos, rope)[0], *turned64(m, pos, rope))


def test_both_tensors_have_to_be_copied(R):
    """Neither head dimension is contiguous: both copies have to live until the launch. The gradient of a sum is such a tensor
    (its strides are zero)."""
    rope, pos = R.Rope(64), torch.arange(50, device="cuda")
    q, k = (torch.randn(2, 3, 64, 50, device="cuda").bfloat16().transpose(2, 3) for _ in range(2))
    want = R.rotary_forward(q.contiguous(), None, pos, rope)[0], R.rotary_forward(k.contiguous(), None, pos, rope)[0]
    got = R.rotary_forward(q, k, pos, rope)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    q, k = (x.contiguous().requires_grad_() for x in (q, k))
    a, b = R.rotary(q, k, pos, rope)
    gq, gk = torch.autograd.grad(a.sum() + 2 * b.sum(), (q, k))
    one = R.rotary_forward(torch.ones_like(q), None, pos, rope, inverse=True)[0]
    assert torch.equal(gq, one) and torch.equal(gk, 2 * one)


def test_overlapping_windows(R):
    """Rows that are windows of one vector, a column apart: empty_like lays such a tensor out with its columns not contiguous."""
    rope = R.Rope(64)
    x = torch.randn(200, device="cuda").unfold(0, 64, 1)[:10]          # strides (1, 1)
    for q in (x[None, None], x[:, None][None], x[None, None].bfloat16().as_strided((1, 1, 10, 64), (640, 640, 1, 1))):
        pos = torch.arange(q.shape[2], device="cuda")
        got, _ = R.rotary_forward(q, None, pos, rope)
        want, _ = R.rotary_forward(q.clone(memory_format=torch.contiguous_format), None, pos, rope)
        assert torch.equal(got, want) and got.is_contiguous()


def test_empty(R):
    rope = R.Rope(32)
    q, k = tensor((2, 3, 0, 64), bf16, 1), tensor((2, 1, 0, 64), bf16, 1)
    oq, ok = R.rotary_forward(q, k, torch.zeros(0, dtype=torch.int64, device="cuda"), rope)
    assert oq.shape == q.shape and ok.shape == k.shape


@pytest.mark.parametrize("inter", [False, True])
def test_gradient_is_the_formulas_and_the_differences(R, inter):
    rope = R.Rope(16, interleaved=inter, scaling="parts", factor=4.0, original_len=64)
    q = tensor((2, 3, 7, 24), f32, 9).requires_grad_()
    k = tensor((2, 1, 7, 24), f32, 10).requires_grad_()
    pos = torch.arange(100, 107, device="cuda")
    gq, gk = tensor((2, 3, 7, 24), f32, 11), tensor((2, 1, 7, 24), f32, 12)
    oq, ok = R.rotary(q, k, pos, rope)
    dq, dk = torch.autograd.grad((oq, ok), (q, k), (gq, gk))
    close(dq, *turned64(gq, pos, rope, inverse=True))
    close(dk, *turned64(gk, pos, rope, inverse=True))
    # The map is linear: the difference along any direction, with any step, is the derivative but for rounding. Sums of
    # n = 1008 products of fp32 values: n * 2^-23 relative to the sum of magnitudes.
    dirq = tensor((2, 3, 7, 24), f32, 13)
    plus, _ = R.rotary_forward(q.detach() + dirq, None, pos, rope)
    minus, _ = R.rotary_forward(q.detach() - dirq, None, pos, rope)
    by_difference = (gq.double() * (plus.double() - minus.double()) / 2).sum()
    by_gradient = (dq.double() * dirq.double()).sum()
    size = (gq.abs().double() * (plus.abs() + minus.abs()).double()).sum()
    assert abs(float(by_difference - by_gradient)) <= 2.0 ** -20 * float(size)


def test_gradient_of_shared_heads_one_result_and_twice(R):
    rope = R.Rope(64)
    pos = torch.arange(5, device="cuda")
    x = tensor((1, 1, 5, 64), f32, 14).requires_grad_()
    oq, ok = R.rotary(x.expand(2, 4, 5, 64), x.expand(2, 1, 5, 64), pos, rope)     # one leaf behind all heads and k
    oq.sum().backward(retain_graph=True)                       # k's gradient is absent
    want = turned64(torch.ones(2, 4, 5, 64, device="cuda"), pos, rope, inverse=True)
    # sum of 8 fp32 terms of magnitude <= 2: 8 roundings of at most 16 * 2^-24, and the terms' own
    assert bool(((x.grad.double() - want[0].sum((0, 1), keepdim=True)).abs() <= 8 * 16 * 2.0 ** -24 + 8 * 2 * 2.0 ** -20).all())
    x.grad = None
    ok.sum().backward()
    want = turned64(torch.ones(2, 1, 5, 64, device="cuda"), pos, rope, inverse=True)
    assert bool(((x.grad.double() - want[0].sum((0, 1), keepdim=True)).abs() <= 2 * 4 * 2.0 ** -24 + 2 * 2 * 2.0 ** -20).all())
    only_k = R.rotary(x, None, pos, rope)
    assert only_k[1] is None
    # the gradient's gradient is the turn again
    g = tensor((1, 1, 5, 64), f32, 15).requires_grad_()
    (dx,) = torch.autograd.grad(R.rotary(x, None, pos, rope)[0], x, g, create_graph=True)
    h = tensor((1, 1, 5, 64), f32, 16)
    (dg,) = torch.autograd.grad(dx, g, h)
    close(dg, *turned64(h, pos, rope))


def test_before_attention_with_gradients(R):
    """rotary next to the attention it is for: forward and backward through both against double precision."""
    from triton_ext_b200.attention import attention
    rope, z, h, n, d = R.Rope(64), 1, 2, 128, 64
    q, k, v, go = (tensor((z, h, n, d), f16, s) * 0.5 for s in (20, 21, 22, 23))
    pos = torch.arange(n, device="cuda")
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    oq, ok = R.rotary(leaves[0], leaves[1], pos, rope)
    o = attention(oq, ok, leaves[2], True, 0.125)
    o.backward(go)
    ref = [t.double().requires_grad_() for t in (q, k, v)]
    rq, rk = (turned64(t, pos, rope)[0] for t in ref[:2])
    s = (rq @ rk.transpose(2, 3)) * 0.125
    s = s.masked_fill(torch.ones(n, n, device="cuda").triu(1).bool(), -math.inf)
    ro = s.softmax(-1) @ ref[2]
    ro.backward(go.double())
    assert float((o.double() - ro).detach().abs().max()) < 1e-2          # the bound the attention's own tests use
    for a, b in zip(leaves, ref):
        assert float((a.grad.double() - b.grad).abs().max()) < 1e-2


def test_other_stream_graph_and_two_calls(R):
    rope = R.Rope(128)
    q, k = tensor((1, 4, 40, 128), bf16, 30), tensor((1, 2, 40, 128), bf16, 31)
    pos = torch.arange(40, device="cuda")
    want = R.rotary_forward(q, k, pos, rope)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = R.rotary_forward(q, k, pos, rope)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        g = R.rotary_forward(q, k, pos, rope)
    pos += 1
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(g, R.rotary_forward(q, k, pos, rope)))


def test_training_step_in_a_graph(R):
    """Forward and backward captured together; the eager graphs of the same leaf are gone by then, as `rotary` asks."""
    rope = R.Rope(64)
    q = tensor((1, 2, 16, 64), bf16, 32).requires_grad_()
    pos, go = torch.arange(16, device="cuda"), tensor((1, 2, 16, 64), bf16, 33)
    (want,) = torch.autograd.grad(R.rotary(q, None, pos, rope)[0], q, go)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        (got,) = torch.autograd.grad(R.rotary(q, None, pos, rope)[0], q, go)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)
