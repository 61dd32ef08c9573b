"""rotary of sequences that have the same positions, on the GPU: one row of positions for all of them is what the
same row for each gives, bit by bit, whether or not their sines and cosines are formed together."""
import pytest
import torch

from _util import ensure_built

pytestmark = pytest.mark.gpu
BF16, F16, F32, F64 = torch.bfloat16, torch.float16, torch.float32, torch.float64


# B, heads of q and of k, T, d, R, type, interleaved, axes: few heads and many sequences, an odd number of them; the last
# ones with too many heads, or too few tokens, to share anything
@pytest.mark.parametrize("B,N,Nk,T,d,R,dtype,interleaved,axes", [
    (8191, 1, 1, 1, 64, 64, BF16, False, 0), (8191, 1, 1, 1, 64, 64, BF16, False, 3), (4099, 1, 0, 1, 32, 30, F32, True, 0),
    (4098, 2, 1, 3, 48, 32, F16, True, 2), (5000, 3, 4, 2, 16, 16, F64, False, 0), (17, 1, 1, 5003, 24, 10, F32, False, 2),
    (3, 2, 0, 30011, 16, 16, BF16, False, 0), (5000, 4, 4, 1, 32, 32, BF16, False, 0), (5000, 4, 4, 1, 32, 32, F32, False, 2),
    (2048, 1, 0, 1, 128, 128, BF16, False, 0), (3, 2, 2, 70, 64, 64, F32, True, 2),
])
def test_one_row_of_positions_is_the_same_row_for_each(B, N, Nk, T, d, R, dtype, interleaved, axes):
    ensure_built()
    from e_natten_amd import rotary, rotary_axes, rotary_frequencies
    print("case same positions", B, N, Nk, T, d, R, dtype, interleaved, axes, flush=True)
    g = torch.Generator(device="cuda").manual_seed(B + T)
    q = torch.randn(B, T, N, d, generator=g, device="cuda", dtype=F32).to(dtype).transpose(1, 2)
    k = torch.randn(B, Nk, T, d, generator=g, device="cuda", dtype=F32).to(dtype) if Nk else None
    frequencies, _ = rotary_frequencies(R, device="cuda")
    positions = torch.randint(-9000, 9000, (axes, T) if axes else (T,), generator=g, device="cuda")
    each = positions.unsqueeze(-2).expand(*positions.shape[:-1], B, T).contiguous()
    kw = dict(interleaved=interleaved, scale=0.7, axes=rotary_axes(R, axes, device="cuda") if axes else None)
    want = rotary(q, k, each, frequencies, **kw)
    for p in (positions, positions.unsqueeze(-2)):
        for x, y in zip(rotary(q, k, p, frequencies, **kw), want):
            assert (x is None and y is None) or torch.equal(x, y)
    # ... and the definition, of a sequence at either end and of one in the middle
    which = [0, B // 2, B - 1]
    at = positions.double()[kw["axes"].long()].t() if axes else positions.double().unsqueeze(1)
    turn = at * frequencies.double()
    c, s = 0.7 * torch.cos(turn), 0.7 * torch.sin(turn)
    x = q[which].double()
    half = R // 2
    x1, x2 = (x[..., :R:2], x[..., 1:R:2]) if interleaved else (x[..., :half], x[..., half:R])
    y = want[0][which].double()
    y1, y2 = (y[..., :R:2], y[..., 1:R:2]) if interleaved else (y[..., :half], y[..., half:R])
    # each of c, s, two products and their sum in float32 (double for float64), then one rounding of the result
    eps = torch.finfo(dtype).eps / 2
    inner = 2.0 ** -21 if dtype != F64 else 2.0 ** -37      # (angles of up to 9000: their own last bits in double)
    for got, ref in ((y1, c * x1 - s * x2), (y2, c * x2 + s * x1)):
        assert ((got - ref).abs() <= eps * ref.abs() + inner * (x1.abs() + x2.abs())).all()
    assert torch.equal(want[0][which][..., R:], q[which][..., R:])
