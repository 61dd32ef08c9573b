"""The operators of growing sequences as they are used: rotary, append and attention step after step,
in graphs, on other streams, over strided, shared and large caches."""
import pytest
import torch

from _sequence import Cache, append_ref, attention_ref, half_step, rotary_ref
from _util import FP32_MAX_ABS, ensure_built

pytestmark = pytest.mark.gpu
BF16, F16, F32, F64 = torch.bfloat16, torch.float16, torch.float32, torch.float64
I8, E4M3 = torch.int8, torch.float8_e4m3fn


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _within(o, ref, bound, dtype):
    """The bound before rounding, and one rounding: half a step relative to the value, but for float16
    values under 2^-14, which are whole multiples of 2^-24: a rounding there is off by up to 2^-25."""
    more = 2.0 ** -25 if dtype == F16 else 0.0
    off = (o.detach().cpu().double() - ref).abs()
    limit = bound + half_step(dtype) * (ref.abs() + bound) + more
    assert torch.isfinite(o.float()).all()
    print("   worst element at %.3f of its bound" % (off / limit.clamp(min=1e-300)).max().item(), flush=True)
    assert (off <= limit).all()


def _empty_cache(final, heads, page, d, dtype, seed):
    """A cache with room for the sequences' final lengths, which hold nothing yet."""
    cache = Cache(final, heads, page, d, dtype, seed=seed)
    for raw, z in zip(cache.codes, cache.scales):
        raw.fill_(0x7f)
        z.fill_(float("nan"))
    return cache


@pytest.mark.parametrize("dtype,cache_dtype,window,d,R,interleaved", [
    (BF16, I8, None, 64, 64, False), (F16, E4M3, 50, 128, 64, True), (F32, I8, 33, 80, 80, False),
    (BF16, E4M3, None, 256, 128, False), (F32, E4M3, None, 64, 32, True),
])
def test_a_run_of_steps(dtype, cache_dtype, window, d, R, interleaved):
    """Prompts of different lengths, single tokens, drafted ones, another chunk, over one layer of a pool
    that keeps keys and values of a page together.  Every step's codes bit for bit, its attention against
    64 bits over what the cache then holds, and at the end against natten1d over the whole sequence."""
    ensure_built()
    from e_natten_amd import cache_append, cache_attention, natten1d, rotary, rotary_frequencies
    print("case steps", dtype, cache_dtype, window, d, flush=True)
    B, N, heads, page = 3, 6, 2, 32
    steps = [(90, [90, 17, 64]), (1, None), (1, None), (5, [5, 2, 0]), (1, [1, 1, 1]), (70, [3, 70, 0]), (1, [0, 1, 1])]
    final = [sum(T if c is None else c[b] for T, c in steps) for b in range(B)]
    cache = _empty_cache(final, heads, page, d, cache_dtype, seed=d)
    total = cache.codes[0].shape[0]
    pool = torch.full((3, total, 2, heads, page, d), 0x55, dtype=torch.uint8, device="cuda")
    scales = torch.full((3, total, 2, heads), 7.0, device="cuda")
    pool[1] = 0x7f
    kc, vc = pool[1, :, 0].view(cache_dtype), pool[1, :, 1].view(cache_dtype)
    ks, vs = scales[1, :, 0], scales[1, :, 1]
    ks.fill_(float("nan")), vs.fill_(float("nan"))
    # page table and lengths as columns of larger tables
    pages = torch.zeros((B, 2 * cache.pages.shape[1]), dtype=torch.int32, device="cuda")[:, ::2]
    pages.copy_(cache.pages)
    lengths = torch.zeros((B, 2), dtype=torch.int32, device="cuda")[:, 1]
    f, factor = rotary_frequencies(R, scaling="yarn", factor=4.0, original_length=32, device="cuda")
    g = torch.Generator().manual_seed(R)
    now, seen_q, scale = [0] * B, [[] for _ in range(B)], d ** -0.5
    for T, counts in steps:
        x = torch.randn((B, T, N + 2 * heads, d), generator=g).to(dtype).cuda().transpose(1, 2)
        c = [T] * B if counts is None else counts
        c_dev = None if counts is None else _ints(counts)
        now = [a + b for a, b in zip(now, c)]
        lengths += _ints(c)
        positions = (lengths - _ints(c))[:, None] + torch.arange(T, device="cuda", dtype=torch.int32)
        q, k = rotary(x[:, :N], x[:, N:N + heads], positions, f, interleaved, factor)
        ref, size = rotary_ref(x[:, N:N + heads], positions, f, interleaved, factor)
        assert ((k.cpu().double() - ref).abs() <= half_step(dtype) * ref.abs() + size * 2.0 ** -21).all()
        v = x[:, N + heads:]
        cache.lengths = list(now)
        want = append_ref(cache, k.cpu(), v.cpu(), c)
        cache_append(k, v, kc, vc, ks, vs, pages, lengths, c_dev)
        for which, (codes, z) in enumerate(want):
            got, got_z = ((kc, ks), (vc, vs))[which]
            assert torch.equal(got.view(torch.uint8).cpu(), codes)
            assert torch.equal(got_z.cpu().nan_to_num(nan=-1.0), z.nan_to_num(nan=-1.0))
            cache.codes[which], cache.scales[which] = codes, z
        o = cache_attention(q, kc, vc, ks, vs, pages, lengths, window, scale, c_dev)
        _within(o, *attention_ref(q, cache, c, window, scale), dtype)
        for b in range(B):
            seen_q[b].append(q[b, :, :c[b]])
    # nothing else of the pool was touched
    assert (pool[::2] == 0x55).all() and (scales[::2] == 7.0).all()
    # the last token once more, as natten1d has it over the sequence that the cache stands for
    for b in range(B):
        last = torch.cat(seen_q[b], 1)
        n = last.shape[1]
        assert n == final[b]
        kk, vv = (cache.values(i, b).float().cuda().repeat_interleave(N // heads, 0)[None] for i in range(2))
        whole = natten1d(last[None].float(), kk, vv, window or n, scale, is_causal=True)[:, :, -1:]
        one = Cache([n], heads, page, d, cache_dtype)
        one.pages, one.codes, one.scales, one.lengths = cache.pages[b:b + 1], cache.codes, cache.scales, [n]
        ref, bound = attention_ref(last[None, :, -1:], one, None, window, scale)
        o = cache_attention(last[None, :, -1:], kc, vc, ks, vs, pages[b:b + 1], lengths[b:b + 1], window, scale)
        limit = bound + half_step(dtype) * (ref.abs() + bound) + FP32_MAX_ABS
        assert ((o.double() - whole.double()).abs().cpu() <= limit).all()


def test_steps_in_graphs():
    """Two graphs of one memory pool, for single and for drafted tokens, which advance the sequences by
    themselves, replayed in turn with eager work between: the same bits as the eager steps each time."""
    ensure_built()
    from e_natten_amd import cache_append, cache_attention, rotary, rotary_frequencies
    B, N, heads, page, d = 4, 8, 2, 16, 128
    start, columns = [700, 33, 1500, 64], 110
    cache = Cache(start, heads, page, d, I8, seed=4, spare=40, columns=columns)
    # every sequence's next tokens go to pages of its own
    pages = cache.pages.clone()
    free = [p for p in range(cache.codes[0].shape[0]) if not cache.owned[p].any()]
    for b, n in enumerate(start):
        have = -(-n // page)
        for i in range(8):
            pages[b, have + i] = free.pop()
    f, _ = rotary_frequencies(d, device="cuda")

    def state():
        kc, vc, ks, vs, _ = cache.on("cuda")
        return dict(kc=kc, vc=vc, ks=ks, vs=vs, pages=pages.cuda(), lengths=_ints(start))

    def step(s, x, counts):
        T = x.shape[1]
        x = x.transpose(1, 2)
        s["lengths"] += counts
        positions = (s["lengths"] - counts)[:, None] + torch.arange(T, device="cuda", dtype=torch.int32)
        q, k = rotary(x[:, :N], x[:, N:N + heads], positions, f)
        cache_append(k, x[:, N + heads:], s["kc"], s["vc"], s["ks"], s["vs"], s["pages"], s["lengths"], counts)
        return cache_attention(q, s["kc"], s["vc"], s["ks"], s["vs"], s["pages"], s["lengths"], None, d ** -0.5, counts)

    g = torch.Generator().manual_seed(9)
    eager, graphed = state(), state()
    kinds = []
    pool = None
    for T in (1, 6):
        x = torch.zeros((B, T, N + 2 * heads, d), dtype=BF16, device="cuda")
        counts = _ints([0] * B)   # warms up without writing anything
        step(graphed, x, counts)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool):
            o = step(graphed, x, counts)
        pool = pool or graph.pool()
        kinds.append((graph, x, counts, o))
    for i in range(6):
        graph, x, counts, o = kinds[i % 2]
        now = torch.randn(x.shape, generator=g).to(BF16).cuda()
        c = _ints([1] * B if i % 2 == 0 else [6, 0, 3, 5])
        want = step(eager, now, c)
        x.copy_(now), counts.copy_(c)
        o.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, want), i
        for name in eager:
            a, b = eager[name], graphed[name]
            if a.dtype == F32:
                a, b = a.nan_to_num(nan=-1.0), b.nan_to_num(nan=-1.0)
            assert torch.equal(a.view(torch.uint8) if a.dtype == E4M3 else a, b.view(torch.uint8) if b.dtype == E4M3 else b), (i, name)
        _ = (want.float() @ want.float().transpose(-1, -2).contiguous()).sum().item()   # unrelated eager work


def test_rotary_with_its_gradient_in_a_graph():
    ensure_built()
    from e_natten_amd import rotary, rotary_frequencies
    f, _ = rotary_frequencies(64, device="cuda")
    p = torch.arange(300, device="cuda")
    x = torch.randn(2, 300, 12, 64, device="cuda", dtype=BF16)
    go = torch.randn(2, 8, 300, 64, device="cuda", dtype=BF16)

    def both(x):
        leaf = x.detach().requires_grad_(True)
        y = leaf.transpose(1, 2)
        q, k = rotary(y[:, :8], y[:, 8:10], p, f, True, 1.5)
        return (q, k, *torch.autograd.grad((q, k), leaf, (go, go[:, :2])))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both(x)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both(x)
    for i in range(4):
        x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(i)))
        want = both(x)
        for t in out:
            t.detach().fill_(float("nan"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


@pytest.mark.parametrize("T", [1, 5, 100])
def test_other_stream_and_both_bindings(T):
    ensure_built()
    from e_natten_amd import cache_append, cache_attention, sequence as S
    cache = Cache([900, 400, 100], 2, 64, 64, E4M3, seed=T)
    g = torch.Generator().manual_seed(T)
    q = torch.randn((3, 6, T, 64), generator=g).to(F16).cuda()
    k, v = (torch.randn((3, 2, T, 64), generator=g).to(F16).cuda() for _ in range(2))
    n, c = _ints([900, 400, 100]), _ints([T, T // 2, 0])
    first, second, third = (list(cache.on("cuda")) for _ in range(3))
    cache_append(k, v, *first, n, c)
    o = cache_attention(q, *first, n, 300, 0.125, c)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cache_append(k, v, *second, n, c)
        o2 = cache_attention(q, *second, n, 300, 0.125, c)
    side.synchronize()
    S._append_impl(k, v, *third, n, c)
    o3 = S._attention_impl(q, *third, n, c, 300, 0.125)
    assert torch.equal(o, o2) and torch.equal(o, o3)
    for a, b, d in zip(first, second, third):
        a, b, d = (x.view(torch.uint8) if x.dtype == E4M3 else x.nan_to_num(nan=-1.0) if x.dtype == F32 else x for x in (a, b, d))
        assert torch.equal(a, b) and torch.equal(a, d)


@pytest.mark.parametrize("T", [1, 4, 90])
def test_offsets_past_32_bits(T):
    """Pages behind the first 2^31 codes, and rows of q, k and v 2^31 elements apart."""
    ensure_built()
    from e_natten_amd import cache_append, cache_attention, rotary
    d, page, far = 256, 1024, 8200
    g = torch.Generator().manual_seed(T)
    big = torch.empty((2 ** 31 + 2 ** 22,), dtype=BF16, device="cuda")
    rows = big.as_strided((2, 5, T, d), (2 ** 31, T * d, d, 1))
    rows.copy_(torch.randn((2, 5, T, d), generator=g))
    q, k, v = rows[:, :3], rows[:, 3:4], rows[:, 4:]
    p, f = torch.arange(T, device="cuda"), torch.ones(d // 2, device="cuda")
    assert all(torch.equal(a, b) for a, b in zip(rotary(q, k, p, f), rotary(q.contiguous(), k.contiguous(), p, f)))
    lengths = _ints([1500, 200])
    small = [torch.randint(-127, 128, (3, 1, page, d), generator=g).to(I8).cuda() for _ in range(2)]
    scales = [torch.rand((3, 1), generator=g).cuda() * 0.02 for _ in range(2)]
    large, large_scales = [], []
    where = torch.tensor([far - 1, 3, 8192], device="cuda")
    for c, z in zip(small, scales):
        large.append(torch.empty((far, 1, page, d), dtype=I8, device="cuda"))
        large_scales.append(torch.full((far, 1), float("nan"), device="cuda"))
        for i, at in enumerate(where.tolist()):
            large[-1][at], large_scales[-1][at] = c[i], z[i]
    pages, far_pages = _ints([[0, 1], [2, -1]]), _ints([[far - 1, 3], [8192, -1]])
    cache_append(k, v, *small, *scales, pages, lengths)
    cache_append(k, v, *large, *large_scales, far_pages, lengths)
    for a, b in zip((*small, *scales), (*large, *large_scales)):
        assert all(torch.equal(a[i], b[at]) for i, at in enumerate(where.tolist()))
    o = cache_attention(q.contiguous(), *small, *scales, pages, lengths, None, 0.1)
    assert torch.equal(o, cache_attention(q, *large, *large_scales, far_pages, lengths, None, 0.1))
    assert torch.isfinite(o.float()).all()


@pytest.mark.parametrize("T", [1, 6, 70])
def test_shared_pages(T):
    """Sequences that share the pages of what they begin with, and one row of pages for all."""
    ensure_built()
    from e_natten_amd import cache_attention
    cache = Cache([400], 2, 16, 64, I8, seed=2)
    kc, vc, ks, vs, pages = cache.on("cuda")
    q = torch.randn((3, 4, T, 64), generator=torch.Generator().manual_seed(T)).to(BF16).cuda()
    lengths = [400, 333, 200]
    o = cache_attention(q, kc, vc, ks, vs, pages.expand(3, -1), _ints(lengths), None, 0.125)
    assert torch.equal(o, cache_attention(q, kc, vc, ks, vs, pages.repeat(3, 1), _ints(lengths), None, 0.125))
    shared = Cache([400], 2, 16, 64, I8, seed=2)
    shared.pages, shared.lengths = cache.pages.expand(3, -1), lengths
    _within(o, *attention_ref(q, shared, None, None, 0.125), BF16)


@pytest.mark.parametrize("B,T,N,heads,longest,window,dtype", [
    (300, 1, 4, 2, 70, None, BF16),       # a workgroup for every sequence and head
    (100, 1, 3, 1, 900, None, F16),       # more sequences than lanes, split along the tokens
    (70, 3, 4, 1, 500, 40, F32),
    (80, 70, 4, 1, 200, None, BF16),      # two tiles of 256 rows each
    (300, 66, 4, 1, 80, 30, F16),         # ... more than workgroups
])
def test_many_sequences(B, T, N, heads, longest, window, dtype):
    ensure_built()
    from e_natten_amd import cache_attention
    g = torch.Generator().manual_seed(B)
    lengths = torch.randint(0, longest + 1, (B,), generator=g).tolist()
    counts = [min(n, int(c)) for n, c in zip(lengths, torch.randint(0, T + 1, (B,), generator=g))] if T > 1 else [min(n, 1) for n in lengths]
    cache = Cache(lengths, heads, 16, 32, I8, seed=T)
    q = torch.randn((B, N, T, 32), generator=g).to(dtype)
    o = cache_attention(q.cuda(), *cache.on("cuda"), _ints(lengths), window, 0.2, _ints(counts))
    _within(o, *attention_ref(q, cache, counts, window, 0.2), dtype)


def test_broadcast_inputs():
    """Heads, tokens and batches that are one row seen several times, and rows of other strides."""
    ensure_built()
    from e_natten_amd import cache_append, cache_attention, rotary, rotary_frequencies
    g = torch.Generator().manual_seed(3)
    f, _ = rotary_frequencies(32, device="cuda")
    p = torch.arange(40, device="cuda")[::4].expand(3, 10)
    x = torch.randn((1, 1, 1, 32), generator=g).to(BF16).cuda().expand(3, 4, 10, 32)
    y = torch.randn((3, 32, 10, 2), generator=g).to(BF16).cuda().permute(0, 3, 2, 1)   # channels apart
    a, b = rotary(x, y, p, f), rotary(x.contiguous(), y.contiguous(), p.contiguous(), f)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    one, other = Cache([50, 12, 10], 2, 16, 32, I8, seed=1), Cache([50, 12, 10], 2, 16, 32, I8, seed=1)
    n = _ints([50, 12, 10])
    first, second = list(one.on("cuda")), list(other.on("cuda"))
    cache_append(x[:, :2], y, *first, n)
    cache_append(x[:, :2].contiguous(), y.contiguous(), *second, n)
    assert all(torch.equal(s.nan_to_num(nan=-1.0) if s.dtype == F32 else s, t.nan_to_num(nan=-1.0) if t.dtype == F32 else t)
               for s, t in zip(first, second))
    assert torch.equal(cache_attention(x, *first, n), cache_attention(x.contiguous(), *second, n))
    # a broadcast input's gradient is the sum over its places, of the rounded rows
    leaf = torch.randn((1, 1, 10, 32), generator=g, dtype=F64).cuda().requires_grad_(True)
    go = torch.randn((3, 4, 10, 32), generator=g, dtype=F64).cuda()
    (dx,) = torch.autograd.grad(rotary(leaf.expand(3, 4, 10, 32), None, p, f)[0], leaf, go)
    ref, size = rotary_ref(go, p, f, inverse=True)
    assert ((dx.cpu() - ref.sum((0, 1), keepdim=True)).abs() <= 2.0 ** -48 * size.sum((0, 1), keepdim=True)).all()


def test_operators_agree_with_their_schemas():
    """What tracing relies on: which arguments are written, and the shapes and strides without data."""
    ensure_built()
    import e_natten_amd as E
    if not E.ops.NATIVE_BINDING:
        pytest.skip("needs the native binding")
    f, _ = E.rotary_frequencies(32, device="cuda")
    p = torch.arange(7, device="cuda")
    x = torch.randn(2, 7, 8, 64, device="cuda", dtype=BF16).transpose(1, 2)
    cache = list(Cache([100, 60], 2, 16, 64, I8).on("cuda"))
    n = _ints([100, 60])
    ops, utils = torch.ops.enatten, ("test_schema", "test_faketensor")
    torch.library.opcheck(ops.rotary.default, (x[:, :4], x[:, 4:6], p, f, False, 1.0, False), test_utils=utils)
    torch.library.opcheck(ops.cache_append.default, (x[:, :2], x[:, 2:4], *cache, n, None), test_utils=utils)
    odd = torch.randn(2, 7, 4, 67, device="cuda", dtype=BF16).transpose(1, 2)[..., 1:65]
    for q in (x[:, :4], odd):
        torch.library.opcheck(ops.cache_attention.default, (q, *cache, n, None, 0, 1.0), test_utils=utils)


def test_calls_on_two_streams_at_once():
    ensure_built()
    from e_natten_amd import cache_attention
    cases = []
    for T, length in ((1, 6000), (70, 3000)):
        cache = Cache([length, length // 2], 2, 32, 128, E4M3, seed=T)
        q = torch.randn((2, 8, T, 128), generator=torch.Generator().manual_seed(T)).to(BF16).cuda()
        args = (q, *cache.on("cuda"), _ints([length, length // 2]), None, 0.1)
        cases.append((args, cache_attention(*args), torch.cuda.Stream()))
    torch.cuda.synchronize()
    out = [[], []]
    for _ in range(10):
        for i, (args, _, stream) in enumerate(cases):
            with torch.cuda.stream(stream):
                out[i].append(cache_attention(*args))
    torch.cuda.synchronize()
    for (_, want, _), got in zip(cases, out):
        assert all(torch.equal(o, want) for o in got)


def test_compiled_steps():
    """Traced as a whole, a training step and an answering step give the same bits."""
    ensure_built()
    import e_natten_amd as E
    if not E.ops.NATIVE_BINDING:
        pytest.skip("needs the native binding")
    f, _ = E.rotary_frequencies(64, device="cuda")
    p = torch.arange(7, device="cuda")
    x = torch.randn(2, 7, 8, 64, device="cuda", dtype=BF16)

    def train(x):
        y = x.transpose(1, 2)
        q, k = E.rotary(y[:, :4], y[:, 4:], p, f)
        return E.natten1d(q, k, y[:, :4], 5, 0.125, is_causal=True)

    def serve(x, kc, vc, ks, vs, pages, n):
        y = x.transpose(1, 2)
        q, k = E.rotary(y[:, :4], y[:, 4:6], p, f)
        E.cache_append(k, y[:, 6:], kc, vc, ks, vs, pages, n)
        return E.cache_attention(q, kc, vc, ks, vs, pages, n, None, 0.125)

    a, b = (x.detach().requires_grad_(True) for _ in range(2))
    o, want = torch.compile(train, backend="aot_eager", fullgraph=True)(a), train(b)
    assert torch.equal(o, want)
    assert torch.equal(torch.autograd.grad(o, a, want.detach())[0], torch.autograd.grad(want, b, want.detach())[0])
    first, second = (list(Cache([100, 60], 2, 16, 64, I8).on("cuda")) for _ in range(2))
    n = _ints([100, 60])
    with torch.no_grad():
        o = torch.compile(serve, backend="aot_eager", fullgraph=True)(x, *first, n)
        assert torch.equal(o, serve(x, *second, n))
    for s, t in zip(first, second):
        assert torch.equal(s.nan_to_num(nan=-1.0), t.nan_to_num(nan=-1.0)) if s.dtype == F32 else torch.equal(s, t)
