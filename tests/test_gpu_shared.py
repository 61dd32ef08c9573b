"""Attention of sequences that continue one prompt, whose shared tokens are read once, on the GPU: against the
definition in 64 bits, which knows nothing of sharing."""
import math

import pytest
import torch

from _pages import ints
from _sequence import Cache, attention_ref, half_step
from _util import ensure_built

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
I8, E4M3 = torch.int8, torch.float8_e4m3fn


def _share(cache, runs, shared):
    """The pages of whole shared tokens are those of the run's first sequence that has them."""
    size = len(cache.lengths) // runs
    for r, n in enumerate(shared):
        first = None
        for b in range(r * size, (r + 1) * size):
            m = max(min(n, cache.lengths[b]), 0) // cache.page
            if first is None and 0 < n <= cache.lengths[b]:
                first = b
            if first is not None and b != first:
                cache.pages[b, :m] = cache.pages[first, :m]
    return cache


def _padded(d):
    return 64 if d <= 64 else 128 if d <= 128 else 256


def _columns(B, heads, page, d, rows):
    """A table so wide that its sequences could have the codes from which on a run's tokens are read together: 16 MB
    with up to 16 rows, else 160, or 320 above 128 channels."""
    return ((16 if rows <= 16 else 160 if d <= 128 else 320) << 20) // (2 * _padded(d) * page * heads * B) + 2


def _pays(B, runs, N, heads, T, d, dtype, tokens):
    """The rule: by the codes that all sequences could have, sequences in a run, and rows of a sequence."""
    size, rows, mb = B // runs, T * N // heads, 2 * _padded(d) * tokens * heads * B / 2 ** 20
    if size == 1:
        return False
    if size * rows <= 16 or d > 128 and dtype == F32:
        return mb >= 16 and 4 * -(-size * rows // 16) <= 3 * size * -(-rows // 16)
    if rows > 96:
        return False
    if d > 128:
        return mb >= 64 if rows > 16 else mb >= 320 and size >= 6
    return mb >= 160 and (size > 2 or rows > 16)


def _shares(q, cache, runs, window=0):
    """Whether a call's sizes make it one (else each sequence reads for itself): its workspace is another."""
    from e_natten_amd import _lib
    lib = ensure_built()
    sizes = (*q.shape[:2], cache.heads, *q.shape[2:], cache.page, cache.pages.shape[1], window or 0,
             {BF16: _lib.BF16, F16: _lib.F16, F32: _lib.F32}[q.dtype])
    return lib.enatten_cache_attention_shared_workspace_bytes(*sizes, runs) != lib.enatten_cache_attention_workspace_bytes(*sizes)


def _check(o, ref, bound, dtype, what):
    off = (o.detach().cpu().double() - ref).abs()
    limit = bound + half_step(dtype) * (ref.abs() + bound)
    worst = (off / limit.clamp(min=1e-300)).max().item()
    print("   %s: worst element at %.3f of its bound, 2-norm %.2e"
          % (what, worst, (off.norm() / ref.norm().clamp(min=1e-300)).item()), flush=True)
    assert torch.isfinite(o.float()).all(), what
    assert (off <= limit).all(), what


def _q(B, N, T, d, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn((B, T, N, d), generator=g) * 2).to(dtype).transpose(1, 2)


# lengths, counts, runs, shared, heads of q and of the cache, T, d, page, type, cache, window
_CASES = [
    ([40, 37], None, 1, [32], 2, 2, 1, 64, 16, BF16, I8, None),
    ([17, 17, 17], None, 1, [16], 1, 1, 1, 16, 16, F32, I8, None),                    # one token behind the shared ones
    ([100, 140, 99, 90], None, 2, [64, 80], 8, 2, 1, 128, 16, BF16, E4M3, None),
    ([100, 140, 99, 90], None, 2, [70, 95], 8, 2, 1, 128, 16, F16, I8, None),         # the end within a page
    ([300, 310, 320, 290, 301, 305], None, 3, [256, 0, 288], 4, 4, 1, 64, 32, BF16, I8, None),   # a run without
    ([300, 310, 320, 290], None, 2, [-5, 2 ** 31 - 1], 4, 4, 1, 64, 32, BF16, I8, None),         # numbers out of any range
    ([300, 200, 320, 290], None, 1, [256], 8, 2, 1, 128, 64, BF16, E4M3, None),       # one is shorter: by itself
    ([200, 300, 320, 290], None, 1, [256], 8, 2, 1, 128, 64, BF16, E4M3, None),       # ... the first one
    ([300, 400, 330], None, 3, [256, 399, 0], 8, 2, 1, 128, 64, BF16, E4M3, None),    # a sequence for itself in each run
    ([300, 400], None, 2, [256, 384], 40, 2, 1, 64, 16, F16, I8, None),
    ([500], None, 1, [448], 8, 2, 1, 128, 64, BF16, I8, None), ([500], None, 1, [448], 8, 2, 3, 80, 16, F32, E4M3, 100),
    ([0, 300, 0, 290], [0, 1, 0, 1], 1, [256], 8, 2, 1, 128, 64, BF16, I8, None),     # some without tokens
    ([300] * 4, [0, 2, 1, 2], 1, [256], 4, 2, 2, 80, 16, F32, E4M3, None),            # ... without new ones
    ([5000, 5050, 5020], None, 1, [4928], 4, 1, 1, 128, 64, BF16, I8, None),          # split along the tokens
    ([5000, 4500, 5020, 9000, 8900, 8999], None, 2, [4480, 8896], 8, 2, 1, 64, 32, F16, E4M3, None),
    ([2000 + i for i in range(12)], None, 1, [1984], 4, 1, 1, 128, 64, BF16, I8, None),    # 48 rows
    ([2000 + i for i in range(16)], None, 1, [1984], 4, 1, 1, 64, 64, BF16, E4M3, None),   # 64
    ([700 + i for i in range(9)], None, 1, [640], 8, 1, 1, 96, 32, F16, I8, None),         # 72: wide tiles
    ([3000 + i for i in range(40)], None, 1, [2944], 8, 1, 1, 128, 64, BF16, E4M3, None),  # 320: two of them
    ([3000 + i for i in range(40)], None, 2, [2944, 2000], 8, 2, 1, 128, 64, BF16, I8, None),
    ([300 + i for i in range(70)], None, 1, [256], 2, 1, 1, 64, 32, BF16, I8, None),       # more sequences than lanes
    ([100] * 64 + [300 + i for i in range(6)], None, 1, [256], 2, 1, 1, 64, 32, BF16, I8, None),  # readers behind them
    ([600, 609, 650], [5, 3, 0], 1, [512], 8, 2, 5, 64, 128, BF16, E4M3, None),       # drafted tokens
    ([600, 609, 650, 700], [5, 3, 1, 4], 2, [500, 640], 15, 5, 5, 80, 48, F32, I8, None),
    ([600, 609, 650, 700], [5, 3, 1, 4], 1, [500], 15, 5, 5, 80, 48, F32, I8, None),
    ([620, 609, 650, 700], [5, 13, 1, 7], 2, [500, 640], 15, 5, 13, 80, 48, F32, I8, None),
    # more rows than a sequence's tiles of 16 to 64, which it has several of: 64 of 80, 48 of 84 and 64, 16 of 96, 50, 20
    ([700, 690, 800, 790], [20, 14, 1, 13], 2, [512, 700], 8, 2, 20, 64, 64, BF16, I8, None),
    ([700, 690, 800, 790], [20, 14, 1, 13], 1, [512], 8, 2, 20, 48, 64, F32, E4M3, None),
    ([700, 690, 800, 790], [21, 14, 1, 0], 2, [512, 700], 8, 2, 21, 128, 64, F16, E4M3, None),
    ([700, 690, 800, 790], [16, 14, 1, 0], 1, [512], 8, 2, 16, 96, 32, F32, I8, None),
    ([700, 690, 800, 790], [24, 14, 1, 0], 2, [512, 700], 8, 2, 24, 256, 64, BF16, I8, None),
    ([700, 690, 800], [25, 14, 1], 1, [512], 4, 2, 25, 192, 16, F16, E4M3, None),
    ([700, 690, 800], [5, 4, 1], 1, [512], 8, 2, 5, 256, 48, BF16, E4M3, None),
    ([700, 690, 800, 790], [70, 64, 1, 33], 2, [512, 700], 8, 2, 70, 128, 64, BF16, I8, None),  # chunks behind a prompt
    ([700, 690, 800, 790], [70, 64, 1, 33], 2, [512, 700], 8, 2, 70, 64, 64, F32, E4M3, None),
    ([520, 530], [257, 200], 1, [256], 4, 1, 257, 64, 16, BF16, I8, None),            # tiles of rows in both passes
    ([900, 910, 930], None, 1, [768], 8, 2, 1, 256, 64, BF16, I8, None),
    ([900 + i for i in range(12)], None, 2, [768, 800], 8, 2, 1, 256, 32, F16, E4M3, None),   # wide tiles of 256 channels
    ([900, 910, 930, 905], None, 1, [768], 8, 2, 3, 192, 64, F32, I8, None),          # ... in tiles of 16, three for four
    ([900, 910, 930], None, 1, [768], 8, 2, 3, 192, 64, F32, I8, None),               # (three for three: by themselves)
    # more runs than lanes, and than workgroups that start at once; in tiles of many rows
    ([200 + i % 90 for i in range(140)], None, 70, [160 + 16 * (i % 3) if i % 5 else 0 for i in range(70)], 2, 1, 1, 64, 16, BF16, I8, None),
    ([60 + i % 40 for i in range(1200)], None, 600, [16 * (i % 4) for i in range(600)], 1, 1, 1, 32, 16, F16, E4M3, None),
    ([200 + i % 90 for i in range(140)], None, 70, [160 + 16 * (i % 3) if i % 5 else 0 for i in range(70)], 20, 1, 1, 64, 16, BF16, E4M3, None),
    ([90 + i % 40 for i in range(600)], [2 - i % 2 for i in range(600)], 300, [16 * (i % 5) for i in range(300)], 9, 1, 2, 128, 16, F16, I8, None),
    # windows (by themselves where these are short): as long as the own tokens, into the shared ones, one token
    ([1000, 990, 1020], None, 1, [960], 8, 2, 1, 128, 64, BF16, I8, 20),
    ([1000, 990, 1020, 980], None, 2, [960, 500], 8, 2, 1, 128, 64, F16, E4M3, 300),
    ([1000, 990, 1020], None, 1, [960], 8, 2, 1, 64, 64, BF16, E4M3, 1),
    ([1000, 990], None, 1, [960], 8, 2, 1, 128, 64, F32, I8, 20000),
    ([1000 + 7 * i for i in range(20)], None, 1, [960], 8, 1, 1, 128, 16, BF16, E4M3, 100),   # wide tiles
    ([1000 + 7 * i for i in range(20)], None, 1, [960], 8, 1, 1, 64, 16, F32, I8, 200),
    ([800, 790, 780], [100, 9, 30], 1, [600], 4, 2, 100, 96, 48, BF16, I8, 150),
    # ... long enough for runs to be read together: one launch, tiles of 32, 64 and 128 rows
    ([6000 + 7 * i for i in range(16)], None, 1, [5984], 1, 1, 1, 128, 32, BF16, I8, 4200),
    ([6000 + 7 * i for i in range(8)], [2, 1] * 4, 2, [5984, 5900], 4, 4, 2, 64, 16, F32, E4M3, 4200),
    ([5500 + 7 * i for i in range(60)], None, 2, [5400, 5440], 2, 2, 1, 128, 32, BF16, E4M3, 5480),
    ([5500 + 7 * i for i in range(60)], None, 1, [5440], 2, 2, 1, 128, 32, F16, I8, 5480),
    ([9000 + 7 * i for i in range(72)], None, 1, [8960], 2, 2, 1, 64, 64, BF16, I8, 9110),
]


@pytest.mark.parametrize("lengths,counts,runs,shared,N,heads,T,d,page,dtype,cache_dtype,window", _CASES)
def test_shared(lengths, counts, runs, shared, N, heads, T, d, page, dtype, cache_dtype, window):
    ensure_built()
    from e_natten_amd import cache_attention
    B = len(lengths)
    print("case shared", lengths[:6], counts, runs, shared, N, heads, T, d, page, dtype, cache_dtype, window, flush=True)
    starts = [n - (T if counts is None else counts[b]) for b, n in enumerate(lengths)]
    size = B // runs
    rows = size * T * N // heads
    columns = max(_columns(B, heads, page, d, rows), -(-max(lengths) // page) + 2)
    cache = Cache(lengths, heads, page, d, cache_dtype, seed=B + d, columns=columns)
    _share(cache, runs, [min([s for s in starts[r * size:(r + 1) * size] if s // page * page >= n // page * page] or [0])
                         if n > 0 else 0 for r, n in enumerate(shared)])
    q = _q(B, N, T, d, dtype, 7)
    pays = _pays(B, runs, N, heads, T, d, dtype, min(cache.pages.shape[1] * page, window + T if window else 1 << 31))
    assert _shares(q, cache, runs, window) == pays
    assert pays or size == 1 or window and window < 4000 or T * N // heads > 96 or T == 5 or (size, d) == (3, 192)
    ref, bound = attention_ref(q, cache, counts, window, d ** -0.5)
    args = (q.cuda(), *cache.on("cuda"), ints(lengths), window, d ** -0.5, None if counts is None else ints(counts))
    o = cache_attention(*args, ints(shared))
    _check(o, ref, bound, dtype, "shared")
    assert torch.equal(o, cache_attention(*args, ints(shared)))
    _check(cache_attention(*args), ref, bound, dtype, "not shared")
    few = cache.pages[:, :max(-(-n // page) for n in lengths)].contiguous().cuda()   # a narrow table
    _check(cache_attention(*args[:5], few, *args[6:], ints(shared)), ref, bound, dtype, "narrow")
    for b in range(B):
        assert (o[b, :, T if counts is None else counts[b]:] == 0).all()


def test_first_rows_of_a_run_that_ended():
    """Rows that cache_fork has emptied name no page: the run's next sequence is asked for its pages."""
    ensure_built()
    from e_natten_amd import cache_attention, cache_fork
    for size in (4, 80):
        lengths = [300 + i for i in range(size)]
        cache = _share(Cache(lengths, 2, 16, 64, I8, seed=1, columns=_columns(size, 2, 16, 64, 2 * size)), 1, [288])
        cache.pages[cache.pages == 2 ** 31 - 1] = -1
        kc, vc, ks, vs, pages = cache.on("cuda")
        holders = torch.zeros(kc.shape[0], dtype=torch.int32, device="cuda")
        entries = pages[pages >= 0].long()
        holders.index_add_(0, entries, torch.ones_like(entries, dtype=torch.int32))
        n, gone = ints(lengths), size - 1 if size == 4 else 70
        cache_fork(pages, n, holders, ints([-1] * gone + list(range(gone, size))), 16)
        counts = ints([0] * gone + [1] * (size - gone))
        q = _q(size, 4, 1, 64, BF16, 3)
        assert _shares(q, cache, 1)
        cache.lengths = [0] * gone + lengths[gone:]
        ref, bound = attention_ref(q, cache, counts.tolist(), None, 0.125)
        o = cache_attention(q.cuda(), kc, vc, ks, vs, pages, n, None, 0.125, counts, ints([288]))
        _check(o, ref, bound, BF16, "ended rows")
        assert (o[:gone] == 0).all()


@pytest.mark.parametrize("rows", [1, 20])
def test_numbers_and_pages_that_do_not_fit(rows):
    """A sequence whose numbers contradict each other is NaN, a page outside the cache makes NaN of who sees it: of
    all that share it, and of nobody else."""
    ensure_built()
    from e_natten_amd import cache_attention
    size = 4
    lengths = [400 + i for i in range(2 * size)]
    cache = Cache(lengths, 2, 16, 64, I8, seed=2, columns=_columns(2 * size, 2, 16, 64, size * rows))
    _share(cache, 2, [384, 384])
    kc, vc, ks, vs, pages = cache.on("cuda")
    q = _q(2 * size, 2 * rows, 1, 64, BF16, 3).cuda()
    assert _shares(q, cache, 2)
    good = cache_attention(q, kc, vc, ks, vs, pages, ints(lengths), None, 0.125, None, ints([384, 384]))
    bad = list(lengths)
    bad[0], bad[5] = -3, 2 ** 31 - 1
    o = cache_attention(q, kc, vc, ks, vs, pages, ints(bad), None, 0.125, None, ints([384, 384]))
    assert torch.isnan(o[[0, 5]]).all()
    rest = [1, 2, 3, 4, 6, 7]
    # (the split goes by the lengths of all: bfloat16 results of the same sums but for float32 roundings)
    assert torch.isfinite(o[rest]).all() and (o[rest].float() - good[rest].float()).abs().max() <= 2 * 2.0 ** -8 * good.abs().max()
    for entry in (-1, kc.shape[0], -2 ** 31):
        p = pages.clone()
        p[:size, 5] = entry
        o = cache_attention(q, kc, vc, ks, vs, p, ints(lengths), None, 0.125, None, ints([384, 384]))
        assert torch.isnan(o[:size]).all() and torch.equal(o[size:], good[size:])
        # own tokens
        p = pages.clone()
        p[2, 25] = entry
        o = cache_attention(q, kc, vc, ks, vs, p, ints([*lengths[:2], 410, *lengths[3:]]), None, 0.125, None, ints([384, 384]))
        assert torch.isnan(o[2]).all() and torch.isfinite(o[[0, 1, 3, 4, 5, 6, 7]]).all()


@pytest.mark.parametrize("rows", [1, 12])
def test_values_that_are_not_finite(rows):
    """A row of q with one is NaN, the others of its run are not; a scale that is none makes NaN of the run."""
    ensure_built()
    from e_natten_amd import cache_attention
    lengths = [400 + i for i in range(8)]
    cache = Cache(lengths, 2, 16, 128, E4M3, seed=2, columns=_columns(8, 2, 16, 128, 4 * rows))
    _share(cache, 2, [384, 384])
    kc, vc, ks, vs, pages = cache.on("cuda")
    q = _q(8, 2 * rows, 1, 128, F16, 3).cuda()
    assert _shares(q, cache, 2)
    args = (kc, vc, ks, vs, pages, ints(lengths), None, 0.125, None, ints([384, 384]))
    good = cache_attention(q, *args)
    for value in (math.inf, -math.inf, math.nan):
        x = q.clone()
        x[3, rows, 0, 17] = value
        o = cache_attention(x, *args)
        assert torch.isnan(o[3, rows]).all()
        o[3, rows] = good[3, rows]
        assert torch.equal(o, good)
    page = int(cache.pages[1, 3])
    for z in (ks, vs):
        for value in (math.inf, math.nan):
            was = z[page, 1].clone()
            z[page, 1] = value
            o = cache_attention(q, *args)
            z[page, 1] = was
            assert torch.isnan(o[:4, rows:]).all()
            assert torch.equal(o[4:], good[4:]) and torch.equal(o[:4, :rows], good[:4, :rows])
    assert torch.isnan(cache_attention(q, *args[:7], math.inf, *args[8:])).all()
    tiny = cache_attention(q, *args[:7], 0.0, *args[8:])      # all tokens alike
    assert torch.isfinite(tiny).all()


def test_large_logits_in_one_part_only():
    """All weight on a shared token, all on an own one, logits of some ten thousands."""
    ensure_built()
    from e_natten_amd import cache_attention
    lengths = [140, 139]
    for where in (5, 136):
        cache = Cache(lengths, 1, 16, 32, I8, seed=4, scale_spread=(1.0, 1.001), columns=_columns(2, 1, 16, 32, 4))
        _share(cache, 1, [128])
        for b in range(2):
            p = int(cache.pages[b, where // 16])
            cache.codes[0].view(I8)[p, 0, where % 16] = 127
        q = torch.full((2, 2, 1, 32), 40.0, dtype=F32)
        assert _shares(q, cache, 1)
        ref, bound = attention_ref(q, cache, None, None, 1.0)
        o = cache_attention(q.cuda(), *cache.on("cuda"), ints(lengths), None, 1.0, None, ints([128]))
        _check(o, ref, bound, F32, "token %d" % where)


@pytest.mark.parametrize("T,N", [(1, 8), (1, 16), (4, 16), (70, 8)])
def test_streams_graphs_bindings_and_layouts(T, N):
    ensure_built()
    import e_natten_amd as E
    from e_natten_amd import sequence as S
    lengths = [700, 690, 720, 715]
    columns = _columns(4, 2, 32, 128, T * N)
    cache = _share(Cache(lengths, 2, 32, 128, E4M3, seed=5, columns=columns), 2, [512, 608])
    assert _shares(_q(4, N, T, 128, BF16, 6), cache, 2) == (T < 70)
    where = cache.on("cuda")
    q, n, shared = _q(4, N, T, 128, BF16, 6).cuda(), ints(lengths), ints([512, 608])
    want = E.cache_attention(q, *where, n, None, 0.1, None, shared)
    assert torch.equal(S._attention_impl(q, *where, n, None, 0, 0.1, shared), want)
    odd = torch.zeros(4, N, T, 131, dtype=BF16, device="cuda")
    odd[..., 1:129] = q
    assert torch.equal(E.cache_attention(odd[..., 1:129], *where, n, None, 0.1, None, shared), want)
    twice = torch.stack((shared, shared), 1)[:, 0]
    assert torch.equal(E.cache_attention(q, *where, n, None, 0.1, None, twice), want)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    out = []
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            out.append(E.cache_attention(q, *where, n, None, 0.1, None, shared))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in out)
    # captured: lengths and shared tokens change between the replays
    x, m, c = q.clone(), n.clone(), shared.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = E.cache_attention(x, *where, m, None, 0.1, None, c)
    for i in range(4):
        x.copy_(q * (1 + i))
        m.copy_(n - 2 * i)
        c.copy_(shared - 40 * i)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, E.cache_attention(x, *where, m, None, 0.1, None, c))
    if E.ops.NATIVE_BINDING:   # (the check multiplies its inputs, which torch does not do with float8)
        where = _share(Cache(lengths, 2, 32, 128, I8, seed=5, columns=columns), 2, [512, 608]).on("cuda")
        where = [x.nan_to_num(nan=1.0) if x.dtype == F32 else x for x in where]
        torch.library.opcheck(torch.ops.enatten.cache_attention.default, (q, *where, n, None, 0, 0.1, shared),
                              test_utils=("test_schema", "test_faketensor"))


@pytest.mark.parametrize("T,N", [(1, 4), (3, 32)])
def test_offsets_past_32_bits(T, N):
    """Pages, heads and tokens whose places are beyond 2^31 and 2^32 codes."""
    ensure_built()
    from e_natten_amd import cache_attention
    heads, page, d, pages = 2, 64, 128, 5
    far = (1 << 32) // (pages - 1) // 16 * 16 + (1 << 20)
    pool = torch.zeros(far * (pages - 1) + heads * page * d, dtype=torch.int8, device="cuda")
    view = pool.as_strided((pages, heads, page, d), (far, page * d, d, 1))
    columns = _columns(2, heads, page, d, T * N)
    lengths, table = [64 * 3 + 5, 64 * 3 + 60], [[4, 1, 3, n] + [-1] * columns for n in (0, 2)]
    g = torch.Generator().manual_seed(1)
    small = [torch.randint(-127, 128, (pages, heads, page, d), generator=g, dtype=torch.int8) for _ in range(2)]
    scales = [torch.rand(pages, heads, generator=g) * 0.02 + 0.01 for _ in range(2)]
    view.copy_(small[0])
    q = _q(2, N, T, d, BF16, 3).cuda()
    rest = (scales[0].cuda(), scales[1].cuda(), ints(table), ints(lengths), None, 0.1, None, ints([192]))
    want = cache_attention(q, small[0].cuda(), small[1].cuda(), *rest)
    assert torch.equal(cache_attention(q, view, small[1].cuda(), *rest), want)
    view.copy_(small[1])
    assert torch.equal(cache_attention(q, small[0].cuda(), view, *rest), want)
