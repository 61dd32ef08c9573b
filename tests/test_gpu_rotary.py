"""Rotary positions on the GPU against the formula in 64 bits."""
import pytest
import torch

from _sequence import half_step, rotary_ref
from _util import ensure_built

pytestmark = pytest.mark.gpu
BF16, F16, F32, F64 = torch.bfloat16, torch.float16, torch.float32, torch.float64


def _bound(y, size, dtype):
    """One rounding to the type, after float32 arithmetic: sine and cosine are off by up to 2^-22 (their
    argument, a half turn at most, is rounded to float32, and their own error), the products and the sum
    by 2^-23 of their size.  float64: the same with 2^-51; the angle is the same product."""
    return half_step(dtype) * y.abs() + size * (2.0 ** -49 if dtype == F64 else 2.0 ** -21)


def _inputs(B, N, Nk, T, d, dtype, layout, seed):
    g = torch.Generator().manual_seed(seed)
    if layout == "proj":
        x = torch.randn((B, T, N + 2 * Nk, d), generator=g, dtype=F64).to(dtype).cuda()
        return x[:, :, :N].transpose(1, 2), x[:, :, N:N + Nk].transpose(1, 2)
    if layout == "odd":   # rows on no particular address, unit stride kept
        x = torch.randn((B, N + Nk, T + 1, d + 3), generator=g, dtype=F64).to(dtype).cuda()
        return x[:, :N, 1:, 1:d + 1], x[:, N:, 1:, 1:d + 1]
    return (torch.randn((B, N, T, d), generator=g, dtype=F64).to(dtype).cuda(),
            torch.randn((B, Nk, T, d), generator=g, dtype=F64).to(dtype).cuda())


@pytest.mark.parametrize("B,N,Nk,T,d,R,dtype,interleaved,layout,first", [
    (1, 16, 16, 1, 128, 128, BF16, False, "plain", 5000),     # one token
    (1, 1, 1, 1, 2, 2, F32, False, "plain", 0),               # the smallest
    (1, 1, 1, 1, 2, 2, F32, True, "plain", 3),
    (2, 8, 2, 100, 64, 64, BF16, False, "proj", 0),
    (2, 8, 2, 100, 64, 64, F16, True, "proj", 100000),
    (3, 5, 1, 33, 80, 40, BF16, False, "proj", 7),            # half of 20 pairs: no whole packs
    (3, 5, 1, 33, 80, 40, F16, True, "proj", 7),
    (1, 3, 3, 17, 25, 6, F32, False, "odd", 1 << 20),         # odd head_dim, odd addresses
    (1, 3, 3, 17, 25, 6, BF16, True, "odd", -40),             # positions of both signs
    (2, 4, 4, 50, 96, 96, F32, True, "plain", 999983),
    (1, 2, 2, 130, 256, 64, F64, False, "proj", 31),
    (1, 2, 2, 13, 32, 32, F64, True, "plain", 12345),
    (1, 1, 1, 3, 1024, 1024, F64, False, "plain", 5),         # the widest table
    (1, 40, 8, 3, 128, 128, BF16, False, "plain", 1000),      # few tokens, many heads: cut by heads
    (2, 3, 2, 4100, 32, 8, BF16, False, "proj", 2),           # many tokens: sixteen to a workgroup
])
def test_rotary(B, N, Nk, T, d, R, dtype, interleaved, layout, first):
    ensure_built()
    from e_natten_amd import rotary, rotary_frequencies
    print("case rotary", B, N, Nk, T, d, R, dtype, interleaved, layout, flush=True)
    f, _ = rotary_frequencies(R, device="cuda")
    scale = 1.25
    q, k = _inputs(B, N, Nk, T, d, dtype, layout, seed=T)
    positions = first + torch.arange(T).flip(0) + 11 * torch.arange(B)[:, None]
    p = positions.cuda()
    qo, ko = rotary(q, k, p, f, interleaved, scale)
    for x, y in ((q, qo), (k, ko)):
        ref, size = rotary_ref(x, positions, f, interleaved, scale)
        assert y.shape == x.shape and y.dtype == dtype and y.stride(-1) == 1
        assert ((y.cpu().double() - ref).abs() <= _bound(ref, size, dtype)).all()
        # the channels behind the rotated ones are the same bits
        assert torch.equal(y[..., R:], x[..., R:])
    # one tensor alone, 32-bit positions, and a row of positions for all: the same bits
    assert torch.equal(rotary(q, None, p.int(), f, interleaved, scale)[0], qo)
    one = rotary(q[:1], k[:1], p[0], f, interleaved, scale)
    assert torch.equal(one[0], qo[:1]) and torch.equal(one[1], ko[:1])
    assert rotary(q, None, p, f)[1] is None


@pytest.mark.parametrize("dtype,interleaved", [(BF16, False), (F16, True), (F32, False), (F64, True)])
def test_gradients(dtype, interleaved):
    ensure_built()
    from e_natten_amd import rotary, rotary_frequencies
    print("case rotary gradients", dtype, interleaved, flush=True)
    B, N, Nk, T, d, R = 2, 6, 2, 37, 48, 32
    f, scale = rotary_frequencies(R, scaling="yarn", factor=4.0, original_length=64, device="cuda")
    p = torch.arange(50, 50 + T, device="cuda")
    q, k = (x.detach().requires_grad_(True) for x in _inputs(B, N, Nk, T, d, dtype, "proj", 1))
    gq, gk = _inputs(B, N, Nk, T, d, dtype, "proj", 2)
    qo, ko = rotary(q, k, p, f, interleaved, scale)
    got = torch.autograd.grad((qo, ko), (q, k), (gq, gk), retain_graph=True)
    for g, x in zip((gq, gk), got):
        ref, size = rotary_ref(g, p, f, interleaved, scale, inverse=True)
        assert ((x.cpu().double() - ref).abs() <= _bound(ref, size, dtype)).all()
    # one of the two alone (the other has no gradient then), and a broadcast upstream gradient
    (dk,) = torch.autograd.grad(ko, k, gk, retain_graph=True)
    assert torch.equal(dk, got[1])
    (dq,) = torch.autograd.grad(qo, q, gq, retain_graph=True)
    assert torch.equal(dq, got[0])
    (dq,) = torch.autograd.grad(qo.sum(), q)
    ref, size = rotary_ref(torch.ones_like(qo), p, f, interleaved, scale, inverse=True)
    assert ((dq.cpu().double() - ref).abs() <= _bound(ref, size, dtype)).all()


@pytest.mark.parametrize("interleaved", [False, True])
def test_against_differences(interleaved):
    ensure_built()
    from e_natten_amd import rotary, rotary_frequencies
    f, _ = rotary_frequencies(6, device="cuda")
    p = torch.tensor([[3, 900000, -2], [0, 1, 2]], device="cuda")
    g = torch.Generator().manual_seed(4)
    q = torch.randn((2, 2, 3, 8), generator=g, dtype=F64).cuda().requires_grad_(True)
    k = torch.randn((2, 1, 3, 8), generator=g, dtype=F64).cuda().requires_grad_(True)
    call = lambda q, k: rotary(q, k, p, f, interleaved, 1.5)
    assert torch.autograd.gradcheck(call, (q, k))
    assert torch.autograd.gradgradcheck(call, (q, k))


def test_both_bindings_agree():
    ensure_built()
    from e_natten_amd import rotary, rotary_frequencies
    from e_natten_amd.sequence import Rotary
    f, _ = rotary_frequencies(64, device="cuda")
    p = torch.arange(9, device="cuda")
    q, k = (x.detach().requires_grad_(True) for x in _inputs(2, 4, 2, 9, 64, BF16, "proj", 3))
    a, b = rotary(q, k, p, f, True, 0.5), Rotary.apply(q, k, p, f, True, 0.5, False)
    ga, gb = (torch.autograd.grad(o, (q, k), o) for o in (a, b))
    assert all(torch.equal(x, y) for x, y in zip((*a, *ga), (*b, *gb)))


def test_far_positions_and_large_values():
    ensure_built()
    from e_natten_amd import rotary
    # a position near 2^31 with an angle of one radian each: the angle is exact to 2^-22
    f = torch.ones(1, dtype=F64, device="cuda")
    x = torch.tensor([1.0, 0.0], device="cuda").view(1, 1, 1, 2)
    p = torch.tensor([2 ** 31 - 1], device="cuda")
    y = rotary(x, None, p, f)[0].cpu().double().flatten()
    ref, _ = rotary_ref(x, p, f)
    assert (y - ref.flatten()).abs().max() < 2.0 ** -20
    # infinities stay in their pair, NaN too
    x = torch.ones((1, 1, 1, 8), device="cuda")
    x[..., 0], x[..., 1] = float("inf"), float("nan")
    y = rotary(x, None, p * 0 + 1, torch.tensor([0.5, 0.25], device="cuda"))[0].flatten()
    assert not torch.isfinite(y[[0, 2, 1, 3]]).any() and torch.equal(y[4:], x.flatten()[4:])
