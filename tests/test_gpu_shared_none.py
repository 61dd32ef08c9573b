"""cache_attention of runs that share nothing, and of tables that are passed as wide as their sequences need, on the
GPU.  Memory that the allocator gives out holds NaN, so that a part nobody left would show."""
import pytest
import torch

from _pages import ints
from _sequence import Cache, attention_ref
from _util import ensure_built
from test_gpu_shared import _check, _columns, _q, _share, _shares

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
I8, E4M3 = torch.int8, torch.float8_e4m3fn


def _poison():
    """Blocks of many sizes that held NaN, left to the allocator."""
    blocks = [torch.full((1 << n,), float("nan"), device="cuda") for n in range(8, 25) for _ in range(2)]
    torch.cuda.synchronize()
    del blocks


# sequences, runs, shared, heads of q and of the cache, T, d, page, type, cache, window
@pytest.mark.parametrize("B,runs,shared,N,heads,T,d,page,dtype,cache_dtype,window", [
    (6, 2, [0, 0], 4, 2, 1, 64, 16, BF16, I8, None), (6, 2, [0, 224], 4, 2, 1, 64, 16, BF16, E4M3, None),
    (6, 3, [-7, 15, 224], 4, 2, 2, 80, 16, F32, I8, None), (6, 2, [0, 0], 4, 2, 1, 256, 32, F16, I8, None),
    (12, 2, [0, 0], 16, 2, 1, 128, 32, BF16, I8, None), (12, 2, [0, 192], 16, 2, 1, 128, 32, F16, E4M3, None),
    (12, 4, [224, 31, 0, 192], 32, 2, 1, 64, 32, F32, I8, None), (24, 3, [0, 0, 0], 16, 2, 3, 128, 32, BF16, E4M3, None),
    (24, 3, [0, 192, 0], 16, 2, 3, 256, 32, BF16, I8, None), (24, 2, [0, 0], 12, 2, 1, 192, 16, F16, E4M3, None),
    (140, 70, [16 * (i % 3) for i in range(70)], 20, 1, 1, 64, 16, BF16, I8, None),
    (1200, 600, [0] * 600, 1, 1, 1, 32, 16, F16, E4M3, None), (6, 2, [0, 0], 4, 2, 1, 64, 16, BF16, I8, 1 << 20),
])
def test_runs_that_share_nothing(B, runs, shared, N, heads, T, d, page, dtype, cache_dtype, window):
    ensure_built()
    from e_natten_amd import cache_attention
    print("case nothing shared", B, runs, shared[:6], N, heads, T, d, page, dtype, cache_dtype, window, flush=True)
    lengths = [240 + 3 * (b % 7) for b in range(B)]
    size = B // runs
    columns = max(_columns(B, heads, page, d, size * T * N // heads), 20)
    cache = _share(Cache(lengths, heads, page, d, cache_dtype, seed=d + B, columns=columns), runs, shared)
    q = _q(B, N, T, d, dtype, 5)
    assert _shares(q, cache, runs, window)
    ref, bound = attention_ref(q, cache, None, window, d ** -0.5)
    args = (q.cuda(), *cache.on("cuda"), ints(lengths), window, d ** -0.5, None, ints(shared))
    first = None
    for _ in range(2):
        _poison()
        o = cache_attention(*args)
        _check(o, ref, bound, dtype, "nothing shared")
        assert first is None or torch.equal(o, first)
        first = o
    # captured, with tokens to share in every other replay
    x = args[-1].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = cache_attention(*args[:-1], x)
    for i in range(4):
        x.copy_(args[-1] if i % 2 else args[-1].clamp(max=0))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, cache_attention(*args[:-1], x))
        _check(o, ref, bound, dtype, "replayed")


@pytest.mark.parametrize("N", [2, 16])
def test_columns_in_use_of_a_wider_table(N):
    """A view of the columns that the sequences need gives what a table of that width gives; the rule goes by it."""
    ensure_built()
    from e_natten_amd import cache_attention
    lengths = [240 + b for b in range(8)]
    cache = _share(Cache(lengths, 2, 16, 64, I8, seed=3, columns=_columns(8, 2, 16, 64, 4 * N)), 2, [224, 224])
    q = _q(8, 2 * N, 1, 64, BF16, 3)
    assert _shares(q, cache, 2)
    kc, vc, ks, vs, pages = cache.on("cuda")
    n = -(-max(lengths) // 16)
    rest = (ints(lengths), None, 0.125, None)
    want = cache_attention(q.cuda(), kc, vc, ks, vs, pages[:, :n].contiguous(), *rest)
    assert torch.equal(cache_attention(q.cuda(), kc, vc, ks, vs, pages[:, :n], *rest, ints([224, 224])), want)
