"""Rotary positions with several axes on the GPU, against the formula in 64 bits; gradients against it and
against differences."""
import pytest
import torch

from _sequence import half_step
from _util import ensure_built

pytestmark = pytest.mark.gpu
BF16, F16, F32, F64 = torch.bfloat16, torch.float16, torch.float32, torch.float64


def _ref(x, positions, frequencies, axes, interleaved=False, scale=1.0, inverse=False):
    """(y, |x1| + |x2| of every channel's pair): pair by pair, in float64 on the CPU.  x: [B, heads, T, d];
    positions: [axes, B or 1, T]."""
    x = x.detach().cpu().double()
    y, size = x.clone(), torch.zeros_like(x)
    half = len(axes)
    for i, a in enumerate(axes):
        lo, hi = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        angle = positions[a].cpu().double()[:, None] * float(frequencies[i])
        c, s = angle.cos() * scale, angle.sin() * scale * (-1 if inverse else 1)
        y[..., lo] = x[..., lo] * c - x[..., hi] * s
        y[..., hi] = x[..., hi] * c + x[..., lo] * s
        size[..., lo] = size[..., hi] = (x[..., lo].abs() + x[..., hi].abs()) * abs(scale)
    return y, size


def _near(got, ref, size, dtype):
    """Angles in double; sines and cosines of float32 are off by 2 of their last places (2^-22), products and
    the sum by half a place each, then one rounding to the type.  float64: the angle, 2^-53 of its size (up
    to 2^20 here), and as many places."""
    few = 2.0 ** -30 if dtype == F64 else 2.0 ** -21
    off = (got.detach().cpu().double() - ref).abs()
    assert (off <= size * few + half_step(dtype) * (ref.abs() + size * few)).all()


def _make(B, N, T, d, dtype, layout, seed, grid=None):
    g = torch.Generator().manual_seed(seed)
    if layout == "plain":
        return torch.randn((B, N, T, d), generator=g).to(dtype).cuda()
    if layout == "odd":
        return torch.randn((B, N, T, d + 3), generator=g).to(dtype).cuda()[..., 1:d + 1]
    if layout == "proj":
        return torch.randn((B, T, N + 2, d), generator=g).to(dtype).cuda()[:, :, 1:N + 1].transpose(1, 2)
    x = torch.randn((B, *grid, N + 2, d), generator=g).to(dtype).cuda()[..., 1:N + 1, :].movedim(-2, 1)
    return x if layout == "grid" else x.transpose(2, 3).contiguous().transpose(2, 3)   # rows inside columns


@pytest.mark.parametrize("B,N,Nk,T,d,R,axes,order,dtype,interleaved,layout,grid", [
    (1, 1, 1, 1, 2, 2, 1, "blocks", BF16, False, "plain", None),
    (3, 4, 2, 1, 64, 64, 3, "blocks", BF16, False, "plain", None),
    (2, 4, 1, 37, 128, 96, 3, "cyclic", F16, True, "proj", None),
    (2, 3, 3, 130, 80, 40, [7, 0, 13], "cyclic", BF16, False, "proj", None),
    (1, 2, 0, 50, 22, 14, [1, 6], "blocks", F32, True, "odd", None),
    (2, 2, 1, 9, 256, 256, 4, "blocks", F64, False, "plain", None),
    (2, 4, 4, 0, 128, 128, 2, "blocks", BF16, False, "grid", (13, 9)),
    (1, 3, 1, 0, 32, 16, 2, "cyclic", F16, True, "grid", (1, 70)),
    (2, 2, 2, 0, 64, 64, 2, "blocks", F32, False, "turned", (6, 11)),
    (40, 8, 8, 0, 64, 64, 2, "blocks", BF16, False, "grid", (16, 16)),
])
def test_axes(B, N, Nk, T, d, R, axes, order, dtype, interleaved, layout, grid):
    ensure_built()
    from e_natten_amd import rotary, rotary_axes, rotary_frequencies
    print("case axes", B, N, Nk, T, d, R, axes, order, dtype, interleaved, layout, grid, flush=True)
    T = T or grid[0] * grid[1]
    which = rotary_axes(R, axes, order, "cuda")
    count = axes if isinstance(axes, int) else len(axes)
    f, _ = rotary_frequencies(R, 1000.0, device="cuda")
    g = torch.Generator().manual_seed(1)
    q = _make(B, N, T, d, dtype, layout, 2, grid)
    k = _make(B, Nk, T, d, dtype, layout, 3, grid) if Nk else None
    for shape in ((count, T), (count, 1, T), (count, B, T)):
        p = torch.randint(-1000, 1 << 20, shape, generator=g)
        p = p.int() if len(shape) == 2 else p
        given = (p.unflatten(-1, grid) if grid else p).cuda()
        if len(shape) == 3 and shape[1] == B:   # (no particular strides)
            given = given.movedim(0, -1).contiguous().movedim(-1, 0)
        out = rotary(q, k, given, f, interleaved, 0.75, which)
        assert (out[1] is None) == (k is None)
        for x, y in zip((q, k), out):
            if x is None:
                continue
            assert y.shape == x.shape and y.dtype == x.dtype
            x, y = (x.flatten(2, 3), y.flatten(2, 3)) if grid else (x, y)
            _near(y, *_ref(x, p if p.dim() == 3 else p[:, None], f, which.tolist(), interleaved, 0.75), dtype)


def test_one_axis_for_all_is_what_rotary_without_axes_gives():
    """Text among images: equal positions on every axis."""
    ensure_built()
    from e_natten_amd import rotary, rotary_axes, rotary_frequencies
    f, _ = rotary_frequencies(64, device="cuda")
    q, k = _make(2, 4, 33, 64, BF16, "proj", 1), _make(2, 2, 33, 64, BF16, "proj", 2)
    p = torch.arange(33, device="cuda") + torch.tensor([[5], [1000]], device="cuda")
    want = rotary(q, k, p, f)
    for order in ("blocks", "cyclic"):
        got = rotary(q, k, p.expand(3, 2, 33), f, axes=rotary_axes(64, 3, order, "cuda"))
        assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_an_axis_that_is_not_there_makes_its_pair_nan():
    ensure_built()
    from e_natten_amd import rotary, rotary_frequencies
    f, _ = rotary_frequencies(16, device="cuda")
    q = _make(1, 2, 5, 20, F32, "plain", 1)
    which = torch.tensor([0, 1, 2, -1, 0, 2 ** 31 - 1, 1, -2 ** 31], dtype=torch.int32, device="cuda")
    p = torch.arange(10, device="cuda").view(2, 5)
    y, _ = rotary(q, None, p, f, axes=which)
    bad = torch.tensor([2, 3, 5, 7], device="cuda")
    gone = torch.zeros(20, dtype=torch.bool, device="cuda")
    gone[bad] = gone[bad + 8] = True
    assert torch.isnan(y[..., gone]).all() and torch.isfinite(y[..., ~gone]).all()
    good = which.clone()
    good[bad] = 0
    assert torch.equal(y[..., ~gone], rotary(q, None, p, f, axes=good)[0][..., ~gone])


@pytest.mark.parametrize("dtype,layout,grid", [(F32, "proj", None), (BF16, "grid", (7, 5)), (F16, "turned", (4, 6))])
def test_gradients(dtype, layout, grid):
    """The turn the other way round; of q alone, of k alone, of both, and twice."""
    ensure_built()
    from e_natten_amd import rotary, rotary_axes, rotary_frequencies
    T = grid[0] * grid[1] if grid else 19
    which = rotary_axes(32, 2, "cyclic", "cuda")
    f, _ = rotary_frequencies(32, device="cuda")
    p = torch.randint(0, 5000, (2, 2, T), generator=torch.Generator().manual_seed(4))
    given = (p.unflatten(-1, grid) if grid else p).cuda()
    q, k = _make(2, 4, T, 48, dtype, layout, 5, grid), _make(2, 2, T, 48, dtype, layout, 6, grid)
    dq, dk = _make(2, 4, T, 48, dtype, layout, 7, grid), _make(2, 2, T, 48, dtype, layout, 8, grid)
    flat = (lambda x: x.flatten(2, 3)) if grid else (lambda x: x)
    want = [_ref(flat(g), p, f, which.tolist(), True, 1.5, True) for g in (dq, dk)]
    for wants_q, wants_k in ((True, True), (True, False), (False, True)):
        x, y = q.detach().requires_grad_(wants_q), k.detach().requires_grad_(wants_k)
        out = rotary(x, y, given, f, True, 1.5, which)
        wanted = [(t, o, g, w) for t, o, g, w in ((x, out[0], dq, want[0]), (y, out[1], dk, want[1])) if t.requires_grad]
        got = torch.autograd.grad([o for _, o, _, _ in wanted], [t for t, _, _, _ in wanted], [g for _, _, g, _ in wanted])
        for got_one, (_, _, _, w) in zip(got, wanted):
            _near(flat(got_one), *w, dtype)
    # a shared head's gradient is the sum over those that read it; the operator's own gradient has one again
    x = q[:, :1].detach().requires_grad_(True)
    out, _ = rotary(x.expand(q.shape), None, given, f, True, 1.5, which)
    g, = torch.autograd.grad(out, x, dq, create_graph=True)
    ref, size = want[0]
    few = 4 * half_step(dtype)
    limit = (size * 2.0 ** -21 + few * (ref.abs() + size)).sum(1, keepdim=True)
    assert ((flat(g).detach().cpu().double() - ref.sum(1, keepdim=True)).abs() <= limit).all()


def test_against_differences():
    ensure_built()
    from e_natten_amd import rotary, rotary_axes, rotary_frequencies
    which = rotary_axes(8, 3, "blocks", "cuda")
    f, _ = rotary_frequencies(8, device="cuda")
    p = torch.randint(0, 100, (3, 2, 3), generator=torch.Generator().manual_seed(1)).cuda()
    q = _make(1, 2, 6, 10, F64, "plain", 1).unflatten(2, (2, 3)).requires_grad_(True)
    k = _make(1, 1, 6, 10, F64, "plain", 2).unflatten(2, (2, 3)).requires_grad_(True)

    def call(q, k):
        return rotary(q, k, p, f, False, 1.25, which)

    assert torch.autograd.gradcheck(call, (q, k))
    assert torch.autograd.gradgradcheck(call, (q, k))


def test_both_bindings_agree():
    ensure_built()
    import e_natten_amd as E
    from e_natten_amd import sequence as S
    which = E.rotary_axes(64, 3, "cyclic", "cuda")
    f, _ = E.rotary_frequencies(64, device="cuda")
    q, k = _make(2, 4, 33, 64, BF16, "proj", 1), _make(2, 2, 33, 64, BF16, "proj", 2)
    p = torch.randint(0, 5000, (3, 2, 33), generator=torch.Generator().manual_seed(4)).cuda()
    want = E.rotary(q, k, p, f, True, 1.5, which)
    a, b = q.detach().requires_grad_(True), k.detach().requires_grad_(True)
    got = S.Rotary.apply(a, b, p, f, True, 1.5, False, which)
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    back = torch.autograd.grad(got, (a, b), (q, k))
    c, d = q.detach().requires_grad_(True), k.detach().requires_grad_(True)
    assert all(torch.equal(x, y) for x, y in zip(back, torch.autograd.grad(E.rotary(c, d, p, f, True, 1.5, which), (c, d), (q, k))))


def test_another_stream_and_a_graph():
    ensure_built()
    from e_natten_amd import rotary, rotary_axes, rotary_frequencies
    which = rotary_axes(64, 2, device="cuda")
    f, _ = rotary_frequencies(64, device="cuda")
    q = _make(2, 4, 0, 64, BF16, "grid", 1, (8, 9))
    p = torch.stack(torch.meshgrid(torch.arange(8), torch.arange(9), indexing="ij")).cuda()
    want = rotary(q, None, p, f, axes=which)[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = rotary(q, None, p, f, axes=which)[0]
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    x = q.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = rotary(x, None, p, f, axes=which)[0]
    for i in range(4):
        x.copy_(q * (i + 1))
        p.add_(3)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, rotary(x, None, p, f, axes=which)[0])
