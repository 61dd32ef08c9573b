"""The cache of 8 bits on the GPU: new tokens written into it, and attention over it, against their
definitions (the codes bit for bit, the attention in 64 bits)."""
import pytest
import torch

from _sequence import Cache, append_ref, attention_ref, half_step
from _util import ensure_built

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
I8, E4M3 = torch.int8, torch.float8_e4m3fn


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _new_tokens(B, heads, T, d, dtype, seed, layout="proj", spread=1.0):
    g = torch.Generator().manual_seed(seed)
    k, v = (torch.randn((B, T, heads, d), generator=g) * spread for _ in range(2))
    if layout == "odd":   # rows on no particular address
        x = torch.zeros((2, B, heads, T, d + 3), dtype=dtype)
        x[0, ..., 1:d + 1], x[1, ..., 1:d + 1] = k.transpose(1, 2).to(dtype), v.transpose(1, 2).to(dtype)
        return x[0, ..., 1:d + 1], x[1, ..., 1:d + 1]
    return k.to(dtype).transpose(1, 2), v.to(dtype).transpose(1, 2)


@pytest.mark.parametrize("lengths,counts,heads,T,d,page,dtype,cache_dtype,layout", [
    ([1], None, 1, 1, 16, 16, BF16, I8, "proj"),                       # the first token
    ([17, 40, 1], None, 2, 1, 128, 16, BF16, E4M3, "proj"),            # first of a page, inside one, first of all
    ([33, 64, 65], None, 3, 1, 80, 32, F32, I8, "odd"),
    ([300, 129], None, 2, 100, 64, 64, F16, I8, "proj"),               # several pages, old tokens before them
    ([300, 129, 50, 7], [100, 0, 33, 7], 2, 100, 64, 48, BF16, E4M3, "proj"),   # ragged; one brings none
    ([1030], None, 1, 1030, 256, 256, BF16, I8, "proj"),               # blocks of more than a workgroup holds
    ([1500], [1100], 1, 1101, 256, 1024, F32, E4M3, "proj"),
    ([70, 31], None, 2, 31, 48, 16, F16, E4M3, "odd"),
])
def test_append(lengths, counts, heads, T, d, page, dtype, cache_dtype, layout):
    ensure_built()
    from e_natten_amd import cache_append
    print("case append", lengths, counts, heads, T, d, page, dtype, cache_dtype, layout, flush=True)
    cache = Cache(lengths, heads, page, d, cache_dtype, seed=T, scale_spread=(0.1, 1.0))
    k, v = _new_tokens(len(lengths), heads, T, d, dtype, 5, layout)
    want = append_ref(cache, k, v, counts)
    kc, vc, ks, vs, pages = cache.on("cuda")
    cache_append(k.cuda(), v.cuda(), kc, vc, ks, vs, pages, _ints(lengths), None if counts is None else _ints(counts))
    for (codes, scales), c, s in zip(want, (kc, vc), (ks, vs)):
        # -0 of float8 and NaN scales: compared as bits
        assert torch.equal(c.view(torch.uint8).cpu(), codes)
        assert torch.equal(s.cpu().nan_to_num(nan=-1.0), scales.nan_to_num(nan=-1.0))


@pytest.mark.parametrize("cache_dtype", [I8, E4M3])
def test_append_corner_values(cache_dtype):
    """Zeros, values that are not finite, values too small for a scale, and a scale that grows."""
    ensure_built()
    from e_natten_amd import cache_append
    heads, d, page = 6, 32, 16
    cache = Cache([20, 20], heads, page, d, cache_dtype, seed=3, scale_spread=(0.5, 0.6))
    k, v = _new_tokens(2, heads, 2, d, F32, 6)
    k[0, 0], v[0, 0] = 0.0, 1e-39
    k[0, 1, 1, 3] = float("inf")
    v[0, 1, 0, 31] = float("nan")
    k[0, 2] *= 1e4          # older tokens of the page lose nearly all their bits
    v[0, 3] *= 3.4e38 / v[0, 3].abs().max()
    k[1, 4, 0, 0] = float("-inf")
    want = append_ref(cache, k, v)
    kc, vc, ks, vs, pages = cache.on("cuda")
    cache_append(k.cuda(), v.cuda(), kc, vc, ks, vs, pages, _ints([20, 20]))
    for (codes, scales), c, s in zip(want, (kc, vc), (ks, vs)):
        assert torch.equal(c.view(torch.uint8).cpu(), codes)
        assert torch.equal(s.cpu().nan_to_num(nan=-1.0), scales.nan_to_num(nan=-1.0))
    # a block that is NaN stays so, another token of the sequence's next page starts afresh
    page_at = int(cache.pages[0, 1])
    assert torch.isnan(ks[page_at, 1]) and torch.isnan(vs[page_at, 1])


def test_append_leaves_out_what_does_not_fit():
    """Counts and lengths that contradict each other or the table, and pages outside the cache: nothing
    of the cache changes for them, the other sequences get their tokens."""
    ensure_built()
    from e_natten_amd import cache_append
    cache = Cache([20, 20, 20, 20, 20, 20], 2, 16, 32, I8, seed=8, extra_columns=0)
    k, v = _new_tokens(6, 2, 4, 32, BF16, 9)
    lengths, counts = [20, 2, 33, -5, 20, 20], [4, 4, 4, 0, -1, 5]
    cache.lengths = [20, 0, 0, 0, 0, 0]
    want = append_ref(cache, k, v, [4, 0, 0, 0, 0, 0])
    kc, vc, ks, vs, pages = cache.on("cuda")
    cache_append(k.cuda(), v.cuda(), kc, vc, ks, vs, pages, _ints(lengths), _ints(counts))
    for bad in (-1, kc.shape[0], 2 ** 31 - 1, -2 ** 31):
        pages[1:, 1] = bad
        cache_append(k.cuda(), v.cuda(), kc, vc, ks, vs, pages, _ints([20] * 6), _ints([4] * 6))
    for (codes, scales), c, s in zip(want, (kc, vc), (ks, vs)):
        assert torch.equal(c.view(torch.uint8).cpu(), codes)
        assert torch.equal(s.cpu().nan_to_num(nan=-1.0), scales.nan_to_num(nan=-1.0))


def _check(o, ref, bound, dtype, what):
    off = (o.detach().cpu().double() - ref).abs()
    limit = bound + half_step(dtype) * (ref.abs() + bound)
    worst = (off / limit.clamp(min=1e-300)).max().item()
    print("   %s: worst element at %.3f of its bound, 2-norm %.2e"
          % (what, worst, (off.norm() / ref.norm().clamp(min=1e-300)).item()), flush=True)
    assert torch.isfinite(o.float()).all(), what
    assert (off <= limit).all(), what


@pytest.mark.parametrize("lengths,counts,N,heads,T,d,page,dtype,cache_dtype,window", [
    ([1], None, 1, 1, 1, 16, 16, BF16, I8, None),                    # a single token sees itself
    ([5], None, 4, 4, 1, 128, 16, BF16, E4M3, None),
    ([16, 17, 31, 32, 33], None, 4, 2, 1, 64, 16, F16, I8, None),    # around the groups and steps of tokens
    ([100, 1000, 257], None, 8, 2, 1, 128, 64, BF16, I8, None),
    ([3000], None, 8, 1, 1, 128, 16, BF16, E4M3, None),              # split along the tokens
    ([5000, 0, 12, 2500], None, 16, 2, 1, 64, 48, F16, E4M3, None),  # one sequence without tokens
    ([700, 33], None, 32, 1, 1, 256, 32, BF16, I8, None),            # two tiles of rows
    ([700, 300], None, 6, 3, 1, 80, 48, F32, I8, None),
    ([4000], None, 15, 5, 1, 96, 16, F32, E4M3, 1000),
    ([900, 128, 127, 1], None, 4, 4, 1, 128, 32, BF16, I8, 128),     # sliding window
    ([900, 40], None, 4, 4, 1, 128, 32, F16, I8, 1),                 # ... of the token itself
    ([900, 40], None, 4, 4, 1, 32, 1024, BF16, E4M3, 33),
    ([600, 9, 250], [5, 3, 0], 8, 2, 5, 64, 128, BF16, E4M3, None),  # drafted tokens, ragged
    ([600, 9, 250], [5, 3, 1], 8, 2, 5, 64, 128, F16, I8, 7),
    ([7, 50], None, 15, 5, 7, 80, 48, F32, I8, None),                # the whole sequence at once
    ([600, 9, 1250], [5, 3, 1], 16, 2, 5, 64, 128, F16, E4M3, None),  # 40 rows
    ([600, 8], None, 16, 2, 8, 64, 16, BF16, I8, 77),                # 64
    ([600, 8], None, 16, 2, 8, 128, 16, F32, E4M3, None),
    ([300, 6], None, 16, 2, 6, 128, 64, BF16, I8, None),
    ([2000], None, 9, 1, 8, 96, 64, F16, I8, None),                  # 72 rows
    ([3000, 2500, 64], None, 8, 4, 64, 128, 64, BF16, E4M3, 1500),   # 128 rows, split along the tokens
    ([1500], None, 4, 1, 40, 64, 48, F32, I8, None),
    ([300, 200], [70, 33], 8, 2, 70, 128, 64, BF16, I8, None),       # chunks: several tiles of rows
    ([300, 200], [70, 33], 8, 2, 70, 128, 64, F16, E4M3, 50),
    ([260], None, 2, 2, 130, 192, 16, BF16, E4M3, 20),
    ([513, 400], [257, 1], 4, 1, 257, 64, 16, BF16, I8, None),
    ([200, 130], [129, 130], 6, 2, 130, 256, 32, F32, E4M3, 70),
    ([200, 130], [129, 130], 6, 2, 130, 112, 80, F32, I8, None),
    ([900, 130, 200], None, 3, 1, 1, 256, 64, BF16, I8, None),       # up to 16 rows of more than 128 channels
    ([900, 130, 200], None, 6, 2, 3, 256, 16, F16, I8, None),
    ([900, 130, 200], None, 4, 2, 1, 192, 16, BF16, E4M3, 100),
    ([900, 130, 200], None, 5, 1, 3, 240, 32, F32, I8, None),
    ([900, 130, 200], None, 4, 4, 4, 144, 16, F32, E4M3, 77),
    ([900, 130, 200], None, 12, 2, 3, 256, 16, BF16, E4M3, None),    # 18
    ([900, 130, 200], None, 8, 2, 5, 160, 48, F32, I8, None),
    ([900, 130, 200], None, 8, 1, 5, 128, 16, BF16, I8, None),       # 40 rows of 128
    ([900, 130, 200], None, 8, 1, 6, 128, 16, F16, E4M3, 55),
    ([900, 130, 200], None, 8, 1, 6, 112, 16, F32, I8, 55),
    ([900, 130, 200], None, 8, 1, 5, 80, 16, F32, E4M3, None),
])
def test_attention(lengths, counts, N, heads, T, d, page, dtype, cache_dtype, window):
    ensure_built()
    from e_natten_amd import cache_attention
    print("case attention", lengths, counts, N, heads, T, d, page, dtype, cache_dtype, window, flush=True)
    cache = Cache(lengths, heads, page, d, cache_dtype, seed=sum(lengths))
    g = torch.Generator().manual_seed(T)
    q = (torch.randn((len(lengths), T, N, d), generator=g) * 2).to(dtype).transpose(1, 2)
    if 0 in lengths:
        counts = [min(n, T) for n in lengths]
    scale = d ** -0.5
    kc, vc, ks, vs, pages = cache.on("cuda")
    args = (kc, vc, ks, vs, pages, _ints(lengths), window, scale, None if counts is None else _ints(counts))
    o = cache_attention(q.cuda(), *args)
    assert o.shape == q.shape and o.dtype == dtype
    ref, bound = attention_ref(q, cache, counts, window, scale)
    _check(o, ref, bound, dtype, "o")
    if counts is not None:
        for b, c in enumerate(counts):
            assert not o[b, :, c:].any()
    # the same call again, and rows that lie elsewhere: the same bits
    assert torch.equal(o, cache_attention(q.cuda(), *args))
    x = torch.zeros((len(lengths), N, T, d + 5), dtype=dtype, device="cuda")
    x[..., 3:d + 3] = q.cuda()
    assert torch.equal(o, cache_attention(x[..., 3:d + 3], *args))


@pytest.mark.parametrize("T,d,window,dtype,cache_dtype", [
    (1, 64, 40, BF16, I8), (1, 128, 40, F32, E4M3), (6, 64, 24, BF16, E4M3), (6, 128, None, F32, I8),
    (40, 64, 24, F16, I8), (40, 64, 24, F32, E4M3), (70, 128, 33, BF16, E4M3), (70, 128, None, F16, I8),
    (70, 64, 100, F32, I8), (70, 256, 33, BF16, E4M3), (20, 256, 33, F32, I8),
])
def test_masked_places_do_not_matter(T, d, window, dtype, cache_dtype):
    """Blocks whose scale is NaN or infinite, and codes of E4M3 that are no numbers: queries that do not
    see them get what they get without them; those that see a NaN block get NaN.

    Bit for bit where keys change: rows do not know of each other.  A value scale has a part in the power
    of two that the value scales of a step are taken relative to.  Another power of two scales the weights
    and all sums exactly, but for float16's subnormals and the rounding of a sum of two logarithms; both
    results are then within the bound of one, and twice that apart at most."""
    ensure_built()
    from e_natten_amd import cache_attention
    n, page, group = 200, 16, 4
    cache = Cache([n, n], 2, page, d, cache_dtype, seed=d + T)
    g = torch.Generator().manual_seed(1)
    q = torch.randn((2, 2 * group, T, d), generator=g).to(dtype).cuda()
    kc, vc, ks, vs, pages = cache.on("cuda")
    call = lambda: cache_attention(q, kc, vc, ks, vs, pages, _ints([n, n]), window, d ** -0.5)
    clean = call()
    ref, bound = attention_ref(q, cache, None, window, d ** -0.5)
    apart = (2 * (bound + half_step(dtype) * (ref.abs() + bound)))[0]
    place = torch.arange(n - T, n)
    first = torch.zeros(T, dtype=torch.long) if window is None else (place - window + 1).clamp(min=0)
    for which, value, block in (("k", float("nan"), 10), ("v", float("nan"), 12), ("k", float("inf"), 11),
                                ("v", float("inf"), 9), ("codes", None, 11)):
        at = int(pages[0, block])
        cache_now = {"k": ks, "v": vs}.get(which)
        if which == "codes":
            if cache_dtype == I8:
                continue
            keep = kc[at].clone(), vc[at].clone()
            kc.view(torch.uint8)[at], vc.view(torch.uint8)[at] = 0x7f, 0xff
        else:
            keep = cache_now[at].clone()
            cache_now[at] = value
        o = call()
        sees = (first < (block + 1) * page) & (place >= block * page)
        assert torch.equal(o[1], clean[1])
        if which == "v":
            off = (o[0].double() - clean[0].double()).abs().cpu()
            assert (off <= apart)[:, ~sees].all(), (which, value)
        else:
            assert torch.equal(o[0][:, ~sees], clean[0][:, ~sees]), (which, value)
        if value != value:
            assert torch.isnan(o[0][:, sees]).all()
        if which == "codes":
            kc[at], vc[at] = keep
        else:
            cache_now[at] = keep
    assert torch.equal(call(), clean)


def test_numbers_that_do_not_fit_give_nan():
    """Counts and lengths that contradict each other or the table: NaN for that sequence, for no other;
    pages outside the cache: NaN for the queries that see them.

    The work of a call is cut by the lengths of all its sequences, and where a sequence is cut its sums
    are rounded elsewhere: two results that are each within the bound of the exact one are at most twice
    that apart.  With the same lengths they are the same bits."""
    ensure_built()
    from e_natten_amd import cache_attention
    for T in (1, 4, 80):
        cache = Cache([200] * 6, 2, 16, 64, I8, seed=8, extra_columns=0)
        q = torch.randn((6, 4, T, 64), generator=torch.Generator().manual_seed(2)).to(BF16).cuda()
        kc, vc, ks, vs, pages = cache.on("cuda")
        full = cache_attention(q, kc, vc, ks, vs, pages, _ints([200] * 6), None, 0.1, _ints([T] * 6))
        lengths, counts = [200, T - 1, 209, -5, 200, 200], [T, T, T, 0, -1, T + 1]
        o = cache_attention(q, kc, vc, ks, vs, pages, _ints(lengths), None, 0.1, _ints(counts))
        ref, bound = attention_ref(q, cache, [T] * 6, None, 0.1)
        apart = (2 * (bound + half_step(BF16) * (ref.abs() + bound)))[0]
        assert ((o[0].double() - full[0].double()).abs().cpu() <= apart).all() and torch.isnan(o[1:]).all()
        for bad in (-1, kc.shape[0], 2 ** 31 - 1, -2 ** 31):
            broken = pages.clone()
            broken[1, 12] = bad      # tokens 192 ..
            broken[2, 3] = bad       # not in the window
            o = cache_attention(q, kc, vc, ks, vs, broken, _ints([200] * 6), 30, 0.1)
            want = cache_attention(q, kc, vc, ks, vs, pages, _ints([200] * 6), 30, 0.1)
            sees = torch.arange(200 - T, 200) >= 192
            assert torch.isnan(o[1][:, sees]).all() and torch.equal(o[1][:, ~sees], want[1][:, ~sees])
            inner = torch.arange(200 - T, 200) >= 64 + 29
            assert torch.equal(o[2][:, inner], want[2][:, inner]) and torch.equal(o[3:], want[3:])


def test_queries_that_are_not_finite_stay_in_their_rows():
    ensure_built()
    from e_natten_amd import cache_attention
    for T, dtype in ((1, BF16), (5, F32), (40, F16), (90, BF16)):
        cache = Cache([150], 2, 32, 64, E4M3, seed=T)
        q = torch.randn((1, 4, T, 64), generator=torch.Generator().manual_seed(3)).to(dtype).cuda()
        args = (*cache.on("cuda"), _ints([150]))
        want = cache_attention(q, *args)
        q[0, 1, 0, 5], q[0, 2, T - 1, 63] = float("nan"), float("inf")
        o = cache_attention(q, *args)
        bad = torch.zeros((4, T), dtype=torch.bool)
        bad[1, 0] = bad[2, T - 1] = True
        assert torch.isnan(o[0][bad]).all() and torch.equal(o[0][~bad], want[0][~bad])


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_extreme_scales(dtype):
    """Logits of hundreds, a maximum that comes late, a negative and a zero factor, value scales many
    powers of two apart (zero among them)."""
    ensure_built()
    from e_natten_amd import cache_attention
    for T, scale, spread in ((1, 3.0, (1e-12, 1e12)), (6, -2.0, (1e-3, 1e3)), (80, 0.0, (1e-30, 1e30)),
                             (80, 1.5, (1e-6, 1e2))):
        cache = Cache([500, 90], 2, 16, 64, I8, seed=T, scale_spread=spread)
        cache.scales[0] = torch.where(torch.isnan(cache.scales[0]), cache.scales[0], torch.full_like(cache.scales[0], 0.03))
        cache.scales[1][int(cache.pages[0, 2])] = 0.0
        q = (torch.randn((2, 4, T, 64), generator=torch.Generator().manual_seed(5)) * 3).to(dtype)
        o = cache_attention(q.cuda(), *cache.on("cuda"), _ints([500, 90]), None, scale)
        ref, bound = attention_ref(q, cache, None, None, scale)
        # tokens whose value scale is far below the largest: their weights go in as float16 of the
        # product of probability and scale, off by at most 2^-31 (2^-41) of the largest value
        top = torch.stack([cache.values(1, b).abs().amax((1, 2)) for b in range(2)]).view(2, 2, 1, 1)
        n = torch.tensor([500.0, 90.0]).view(2, 1, 1, 1)
        bound = bound + (n * top * 2.0 ** -31).repeat_interleave(2, 1)
        _check(o, ref, bound, dtype, "o, factor %g" % scale)


@pytest.mark.parametrize("T,dtype,cache_dtype", [(1, BF16, I8), (1, F32, E4M3), (6, F16, E4M3), (40, BF16, I8),
                                                 (90, BF16, E4M3), (90, F32, I8)])
def test_a_factor_that_is_not_finite(T, dtype, cache_dtype):
    """Logits are no numbers then: NaN for every row that a sequence has, whatever the tile; 0 behind."""
    ensure_built()
    from e_natten_amd import cache_attention
    cache = Cache([150, 100], 2, 32, 64, cache_dtype, seed=T)
    q = torch.randn((2, 4, T, 64), generator=torch.Generator().manual_seed(3)).to(dtype).cuda()
    counts = [T, T // 2]
    for scale in (float("nan"), float("inf"), float("-inf")):
        o = cache_attention(q, *cache.on("cuda"), _ints([150, 100]), None, scale, _ints(counts))
        assert torch.isnan(o[0]).all() and torch.isnan(o[1, :, :T // 2]).all(), scale
        assert not o[1, :, T // 2:].any()


@pytest.mark.parametrize("T,dtype,cache_dtype", [(1, BF16, I8), (1, F32, E4M3), (6, F32, I8), (90, BF16, I8),
                                                 (90, F32, E4M3), (90, BF16, E4M3), (300, F32, I8)])
def test_values_next_to_the_smallest(T, dtype, cache_dtype):
    """Value scales from 2^-126, the smallest that cache_append writes, to 2^-119: nothing of them is lost on the
    way.  Results under 2^-126 are whole multiples of 2^-149 (bfloat16: 2^-133), a rounding there is off by half
    of that; so are the sums of up to 8 parts and of 4 waves each, in float32."""
    ensure_built()
    from e_natten_amd import cache_attention
    lengths = [1500, 301]
    cache = Cache(lengths, 2, 32, 64, cache_dtype, seed=T)
    g = torch.Generator().manual_seed(7)
    tiny = torch.exp2(-126 + 7 * torch.rand(cache.scales[1].shape, generator=g)).clamp(min=2.0 ** -126)
    cache.scales[1] = torch.where(torch.isnan(cache.scales[1]), cache.scales[1], tiny)
    q = torch.randn((2, 4, T, 64), generator=g).to(dtype)
    o = cache_attention(q.cuda(), *cache.on("cuda"), _ints(lengths), None, 0.2)
    ref, bound = attention_ref(q, cache, None, None, 0.2)
    _check(o, ref, bound + 64 * 2.0 ** -150 + (2.0 ** -134 if dtype == BF16 else 0.0), dtype, "o")


@pytest.mark.parametrize("N,heads,d,page,dtype,cache_dtype,window", [
    (4, 2, 256, 32, BF16, I8, None), (4, 2, 256, 32, F16, E4M3, 40), (4, 4, 128, 64, F16, E4M3, None),
    (6, 2, 64, 16, F32, I8, 90), (2, 2, 128, 48, F32, E4M3, None), (4, 2, 160, 16, F32, I8, None),
])
def test_whole_prompts_at_once(N, heads, d, page, dtype, cache_dtype, window):
    """Nothing stands before the new tokens: the causal triangle alone, over several tiles of 256 rows (16 for
    float32 above 128 channels) whose first ones see next to nothing; prompts of different lengths, one token."""
    ensure_built()
    from e_natten_amd import cache_attention
    lengths = [600, 257, 1]
    cache = Cache(lengths, heads, page, d, cache_dtype, seed=d + N)
    q = (torch.randn((3, N, 600, d), generator=torch.Generator().manual_seed(4)) * 2).to(dtype)
    o = cache_attention(q.cuda(), *cache.on("cuda"), _ints(lengths), window, d ** -0.5, _ints(lengths))
    ref, bound = attention_ref(q, cache, lengths, window, d ** -0.5)
    _check(o, ref, bound, dtype, "o")
    assert not o[1, :, 257:].any() and not o[2, :, 1:].any()
