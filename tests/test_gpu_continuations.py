"""Sequences that continue prompts, the operators together as a program uses them on the GPU: positions with several
axes, rows that fork, pages that are reserved, copied, appended to and read together, and moved."""
import pytest
import torch

from _pages import compact_ref, fork_ref, ints, random_state, reserve_ref
from _sequence import Cache, append_ref, attention_ref, half_step
from _util import ensure_built

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
I8, E4M3 = torch.int8, torch.float8_e4m3fn


def _places(lengths, counts, T):
    """[3, B, T]: a token's place, and that as row and column of a picture seven wide."""
    p = (lengths - counts)[:, None] + torch.arange(T, device="cuda", dtype=torch.int32)
    return torch.stack((p, p // 7, p % 7))


def _turned(x, places, f, axes):
    """(y, |x1| + |x2| of every channel's pair) in float64 on the CPU"""
    x, half = x.cpu().double(), len(axes)
    y, size = x.clone(), torch.zeros_like(x)
    for i, a in enumerate(axes.tolist()):
        angle = places[a].cpu().double()[:, None] * float(f[i])
        u, v = x[..., i], x[..., i + half]
        y[..., i], y[..., i + half] = u * angle.cos() - v * angle.sin(), v * angle.cos() + u * angle.sin()
        size[..., i] = size[..., i + half] = u.abs() + v.abs()
    return y, size


def _bits(t):
    return t.view(torch.uint8) if t.dtype == E4M3 else t.nan_to_num(nan=-1.0) if t.dtype == F32 else t


def _columns(B, heads, page, d, rows):
    """A table so wide that its sequences could have the codes from which on a run's tokens are read together."""
    return ((16 if rows <= 16 else 160 if d <= 128 else 320) << 20) // (2 * max(d, 64) * page * heads * B) + 2


@pytest.mark.parametrize("dtype,cache_dtype,d,page,size,N,heads,window,wide", [
    (BF16, I8, 64, 16, 3, 4, 2, None, False), (BF16, E4M3, 128, 32, 4, 4, 1, None, True), (F16, I8, 80, 16, 2, 6, 2, None, True),
    (F32, E4M3, 64, 48, 3, 2, 2, None, True), (BF16, I8, 256, 16, 5, 8, 2, 70, True), (F16, E4M3, 96, 64, 2, 3, 1, 50, False),
])
def test_a_run_of_steps(dtype, cache_dtype, d, page, size, N, heads, window, wide):
    """Two prompts in two layers, their samples, beams that leave each other, sequences that end, drafted tokens,
    pages moved to the low end: codes and table exactly, attention against 64 bits over what the cache holds."""
    ensure_built()
    from e_natten_amd import (cache_append, cache_attention, cache_compact, cache_copy, cache_fork, cache_reserve, rotary,
                              rotary_axes, rotary_frequencies)
    print("case steps", dtype, cache_dtype, d, page, size, N, window, wide, flush=True)
    B, layers, prompts, scale = 2 * size, 2, [2 * page + 5, 5 * page], d ** -0.5
    total = 14 + 6 * B
    columns = max(9, _columns(B, heads, page, d, size * 4 * N // heads) if wide else 0)
    held = [Cache([0] * B, heads, page, d, cache_dtype, seed=i, spare=total, columns=columns) for i in range(layers)]
    assert held[0].codes[0].shape[0] == total
    at = [c.on("cuda")[:4] for c in held]
    kc, vc, ks, vs = (torch.stack([x[i].view(torch.uint8) if i < 2 else x[i] for x in at]) for i in range(4))
    kc, vc = kc.view(cache_dtype), vc.view(cache_dtype)
    pages, lengths, holders = torch.full((B, columns), -1, dtype=torch.int32, device="cuda"), ints([0] * B), ints([0] * total)
    rows, now, holds = pages.tolist(), [0] * B, [0] * total
    f, _ = rotary_frequencies(d, device="cuda")
    axes = rotary_axes(d, 3, "cyclic", device="cuda")
    g = torch.Generator().manual_seed(d + page)
    first = [size * (b // size) for b in range(B)]
    again = [first[b] + b % size // 2 for b in range(B)]
    ended = list(range(B))
    ended[1] = ended[size] = -1
    back = [first[b] if b in (1,) else size + 1 if b == size else b for b in range(B)]
    # what comes before the tokens (parents, or whether pages move), and the tokens of each row
    steps = [(None, [prompts[b // size] if b % size == 0 else 0 for b in range(B)]), (first, [1] * B), (None, [1] * B),
             (again, [1] * B), (None, [b % 4 + 1 if b != 1 else 0 for b in range(B)]), (ended, [0 if b in (1, size) else 1 for b in range(B)]),
             ("compact", [0 if b in (1, size) else 4 for b in range(B)]), (back, [1] * B), (again, [3] * B), ("compact", [1] * B)]

    def copied(copies):
        cache_copy(kc, vc, ks, vs, copies)
        for s, t, n in copies.tolist():
            if s < 0:
                continue
            for c in held:
                for which in range(2):
                    c.codes[which][t, :, :n] = c.codes[which][s, :, :n]
                    c.scales[which][t] = c.scales[which][s]

    copies_seen = 0
    for before, counts in steps:
        if before == "compact":
            want = compact_ref(rows, holds, page)
            got = cache_compact(pages, holders, page)
            rows, holds = want[:2]
            assert got.tolist() == [list(x) for x in want[2]]
            copied(got)
        elif before is not None:
            cache_fork(pages, lengths, holders, ints(before), page)
            rows, now, holds = fork_ref(rows, now, holds, before, page)
            assert lengths.tolist() == now
        T = max(counts)
        single = counts == [1] * B
        c = ints(counts)
        lengths += c
        now = [a + b for a, b in zip(now, counts)]
        want = reserve_ref(rows, now, holds, page, counts)
        got = cache_reserve(pages, lengths, holders, page, 1 if single else c)
        rows, holds = want[:2]
        assert pages.tolist() == rows and holders.tolist() == holds and got.tolist() == [list(x) for x in want[2]]
        assert all(rows[b][i] >= 0 for b in range(B) for i in range(-(-now[b] // page)))
        copies_seen += sum(x[0] >= 0 for x in want[2])
        copied(got)
        places = _places(lengths, c, T)
        for layer, cache in enumerate(held):
            cache.pages, cache.lengths = pages.cpu(), list(now)
            x = torch.randn((B, T, N + 2 * heads, d), generator=g).to(dtype).cuda().transpose(1, 2)
            q, k = rotary(x[:, :N], x[:, N:N + heads], places, f, axes=axes)
            v = x[:, N + heads:]
            # sines and cosines of float32, products and a sum: 2^-21 of the pair, and the rounding
            ref, pair = _turned(x[:, N:N + heads], places, f, axes)
            assert ((k.cpu().double() - ref).abs() <= half_step(dtype) * (ref.abs() + pair * 2.0 ** -21) + pair * 2.0 ** -21).all()
            want = append_ref(cache, k.cpu(), v.cpu(), counts)
            where = (kc[layer], vc[layer], ks[layer], vs[layer])
            cache_append(k, v, *where, pages, lengths, c)
            for which, (codes, z) in enumerate(want):
                cache.codes[which], cache.scales[which] = codes, z
                assert torch.equal(where[which].view(torch.uint8).cpu(), codes)
                assert torch.equal(where[2 + which].cpu().nan_to_num(nan=-1.0), z.nan_to_num(nan=-1.0))
            o = cache_attention(q, *where, pages, lengths, window, scale, None if single else c, ints(prompts))
            ref, bound = attention_ref(q, cache, counts, window, scale)
            limit = bound + half_step(dtype) * (ref.abs() + bound)
            assert ((o.cpu().double() - ref).abs() <= limit).all()
    assert copies_seen >= size - 1 + 2 * (size // 2)


def _state(B, size, heads, page, d, columns, prompts, seed):
    """A cache of one layer whose runs' first rows hold their prompts, and the numbers beside it."""
    cache = Cache([prompts[b // size] if b % size == 0 else 0 for b in range(B)], heads, page, d, I8, seed=seed, spare=8 * B,
                  columns=columns)
    kc, vc, ks, vs, pages = cache.on("cuda")
    pages = torch.where((pages >= 0) & (pages < kc.shape[0]), pages, -1)
    holders = torch.zeros(kc.shape[0], dtype=torch.int32)
    for e in pages.flatten().tolist():
        if e >= 0:
            holders[e] += 1
    return dict(kc=kc, vc=vc, ks=ks, vs=vs, pages=pages, holders=holders.cuda(), lengths=ints(cache.lengths))


def _step(s, x, parents, counts, shared, f, axes, N, page):
    from e_natten_amd import cache_append, cache_attention, cache_copy, cache_fork, cache_reserve, rotary
    heads, T = s["kc"].shape[1], x.shape[1]
    cache_fork(s["pages"], s["lengths"], s["holders"], parents, page)
    s["lengths"] += counts
    copies = cache_reserve(s["pages"], s["lengths"], s["holders"], page, counts)
    cache_copy(s["kc"], s["vc"], s["ks"], s["vs"], copies)
    x = x.transpose(1, 2)
    p = (s["lengths"] - counts)[:, None] + torch.arange(T, device="cuda", dtype=torch.int32)
    q, k = rotary(x[:, :N], x[:, N:N + heads], torch.stack((p, p // 7, p % 7)), f, axes=axes)
    cache_append(k, x[:, N + heads:], s["kc"], s["vc"], s["ks"], s["vs"], s["pages"], s["lengths"], counts)
    return cache_attention(q, s["kc"], s["vc"], s["ks"], s["vs"], s["pages"], s["lengths"], None, 0.1, counts, shared)


@pytest.mark.parametrize("size,N", [(4, 2), (8, 8)])
def test_steps_in_graphs(size, N):
    """Two graphs of one memory pool, for single and for drafted tokens, replayed in turn with eager work between:
    the same bits as the eager steps, in every number and code."""
    ensure_built()
    from e_natten_amd import cache_compact, cache_copy, rotary_axes, rotary_frequencies
    heads, page, d, prompts = 2, 16, 128, [700, 333]
    B = 2 * size
    columns = _columns(B, heads, page, d, 5 * size * N // heads)
    f, _ = rotary_frequencies(d, device="cuda")
    axes = rotary_axes(d, 3, device="cuda")
    eager, graphed = (_state(B, size, heads, page, d, columns, prompts, 3) for _ in range(2))
    shared = ints(prompts)
    stay = ints(list(range(B)))
    kinds, pool = [], None
    for T in (1, 5):
        x = torch.zeros((B, T, N + 2 * heads, d), dtype=BF16, device="cuda")
        parents, counts = stay.clone(), ints([0] * B)   # warms up without writing anything
        _step(graphed, x, parents, counts, shared, f, axes, N, page)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool):
            o = _step(graphed, x, parents, counts, shared, f, axes, N, page)
        pool = pool or graph.pool()
        kinds.append((graph, x, parents, counts, o))
    for name in eager:
        assert torch.equal(_bits(eager[name]), _bits(graphed[name])), name
    g = torch.Generator().manual_seed(9)
    for i in range(8):
        graph, x, parents, counts, o = kinds[i % 2]
        now = torch.randn(x.shape, generator=g).to(BF16).cuda()
        who = [size * (b // size) + (0 if i == 0 else (b * 5 + i) % size) for b in range(B)] if i % 3 == 0 else list(range(B))
        if i == 4:
            who[1] = -1
        some = [1] * B if i % 2 == 0 else [(b + i) % 6 for b in range(B)]
        if i == 5:
            some[1] = 0   # (the sequence that ended)
        want = _step(eager, now, ints(who), ints(some), shared, f, axes, N, page)
        x.copy_(now), parents.copy_(ints(who)), counts.copy_(ints(some))
        o.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, want), i
        for name in eager:
            assert torch.equal(_bits(eager[name]), _bits(graphed[name])), (i, name)
        if i == 3:   # pages move between the replays
            for s in (eager, graphed):
                cache_copy(s["kc"], s["vc"], s["ks"], s["vs"], cache_compact(s["pages"], s["holders"], page))
        _ = (want.float() @ want.float().transpose(-1, -2).contiguous()).sum().item()   # unrelated eager work


@pytest.mark.parametrize("B,columns,total", [(5, 40, 300), (300, 9, 4000), (2100, 12, 32000)])
def test_pages_on_streams_in_graphs_and_both_bindings(B, columns, total):
    ensure_built()
    import e_natten_amd as E
    from e_natten_amd import pages as P
    page = 16
    states = [random_state(B, columns, page, 50, seed) for seed in (1, 2)]
    parents = [ints([(b * 7 + 3) % (B + 3) - 1 for b in range(B)]), ints([0] * B)]
    counts = ints([b % 5 for b in range(B)])

    def run(state, parents, fork, reserve, compact):
        p, n, h = state
        fork(p, n, h, parents, page)
        n += counts
        a = reserve(p, n, h, page, counts)
        return a, compact(p, h, page)

    def fresh():
        out = []
        for pages, lengths, holders in states:
            out.append([ints(pages), ints(lengths), ints(holders + [0] * (total - len(holders)))])
        return out

    public = (E.cache_fork, E.cache_reserve, E.cache_compact)
    want = []
    for s, who in zip(fresh(), parents):
        out = run(s, who, *public)
        want.append([*s, *out])
    ctyped = (P._fork_impl, lambda p, n, h, page, c: P._reserve_impl(p, n, h, page, c, 0), P._compact_impl)
    for s, who, w in zip(fresh(), parents, want):
        out = run(s, who, *ctyped)
        assert all(torch.equal(x, y) for x, y in zip((*s, *out), w))
    # two streams at once, a state each
    streams = [torch.cuda.Stream() for _ in range(2)]
    rounds = [fresh() for _ in range(4)]
    torch.cuda.synchronize()
    outs = []
    for s in rounds:
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                outs.append((i, s[i], run(s[i], parents[i], *public)))
    torch.cuda.synchronize()
    for i, s, out in outs:
        assert all(torch.equal(x, y) for x, y in zip((*s, *out), want[i]))
    # captured, replayed on other numbers each time
    s, who = fresh()[0], parents[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(s, who, *public)
    for i in (0, 1, 0, 1):
        for t, x in zip(s, fresh()[i]):
            t.copy_(x)
        who.copy_(parents[i])
        for t in out:
            t.fill_(77)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip((*s, *out), want[i])), i
        _ = torch.randn(300, 300, device="cuda").sum().item()


def test_operators_agree_with_their_schemas():
    ensure_built()
    import e_natten_amd as E
    if not E.ops.NATIVE_BINDING:
        pytest.skip("needs the native binding")
    s = _state(4, 2, 2, 16, 64, 30, [100, 60], 1)
    for x in (s["ks"], s["vs"]):
        x.nan_to_num_(nan=1.0)
    ops, utils = torch.ops.enatten, ("test_schema", "test_faketensor")
    table = (s["pages"], s["lengths"], s["holders"])
    torch.library.opcheck(ops.cache_fork.default, (*table, ints([0, 0, 2, 2]), 16), test_utils=utils)
    torch.library.opcheck(ops.cache_reserve.default, (*table, 16, None, 1), test_utils=utils)
    torch.library.opcheck(ops.cache_reserve.default, (*table, 16, ints([1, 0, 2, 3]), 0), test_utils=utils)
    torch.library.opcheck(ops.cache_compact.default, (s["pages"], s["holders"], 16), test_utils=utils)
    cache = (s["kc"], s["vc"], s["ks"], s["vs"])
    copies = ints([[0, 1, 5], [2, 3, 16], [-1, -1, 0]])
    torch.library.opcheck(ops.cache_copy.default, (*cache, copies), test_utils=utils)
    x = torch.randn(2, 7, 8, 64, device="cuda", dtype=BF16).transpose(1, 2)
    f, _ = E.rotary_frequencies(32, device="cuda")
    p = torch.randint(0, 50, (3, 2, 7), device="cuda")
    axes = E.rotary_axes(32, 3, device="cuda")
    torch.library.opcheck(ops.rotary.default, (x[:, :4], x[:, 4:6], p, f, False, 1.0, False, axes), test_utils=utils)


def test_compiled_steps():
    """Traced as a whole, a step gives the same bits; so does a training step of an image's attention."""
    ensure_built()
    import e_natten_amd as E
    if not E.ops.NATIVE_BINDING:
        pytest.skip("needs the native binding")
    f, _ = E.rotary_frequencies(64, device="cuda")
    axes = E.rotary_axes(64, 3, device="cuda")
    first, second = (_state(4, 2, 2, 16, 64, 30, [100, 60], 1) for _ in range(2))
    x = torch.randn(4, 1, 8, 64, device="cuda", dtype=BF16)
    args = (x, ints([0, 0, 2, 2]), ints([1, 1, 1, 0]), ints([100, 60]), f, axes, 4, 16)
    with torch.no_grad():
        o = torch.compile(_step, backend="aot_eager", fullgraph=True)(first, *args)
        assert torch.equal(o, _step(second, *args))
    for name in first:
        assert torch.equal(_bits(first[name]), _bits(second[name])), name
    grid = torch.stack(torch.meshgrid(torch.arange(9, device="cuda"), torch.arange(6, device="cuda"), indexing="ij"))
    two = E.rotary_axes(64, 2, device="cuda")

    def train(x):
        y = x.movedim(-2, 1)
        q, k = E.rotary(y[:, :4], y[:, 4:8], grid, f, axes=two)
        return E.natten2d(q, k, y[:, 8:], 3, 0.125)

    x = torch.randn(2, 9, 6, 12, 64, device="cuda", dtype=BF16)
    a, b = (x.detach().requires_grad_(True) for _ in range(2))
    o, want = torch.compile(train, backend="aot_eager", fullgraph=True)(a), train(b)
    assert torch.equal(o, want)
    assert torch.equal(torch.autograd.grad(o, a, want.detach())[0], torch.autograd.grad(want, b, want.detach())[0])


def test_copies_past_32_bits():
    """Pages, heads and layers whose places are beyond 2^31 and 2^32 codes."""
    ensure_built()
    from e_natten_amd import cache_copy
    heads, page, d = 2, 16, 32
    far = (1 << 32) + (1 << 20)
    pool = torch.zeros(far + (1 << 20), dtype=I8, device="cuda")
    g = torch.Generator().manual_seed(1)
    copies = ints([[0, 1, 7], [3, 2, 16]])
    # layers, pages, heads, page, d with one axis after the other as the far one
    for strides in ((1 << 14, far // 3 // 16 * 16, 1 << 10, d, 1), (far, 1 << 13, 1 << 10, d, 1), (1 << 14, 1 << 12, far, d, 1)):
        view = pool.as_strided((2, 4, heads, page, d), strides)
        small = torch.randint(-127, 128, view.shape, generator=g, dtype=I8).cuda()
        other = torch.randint(-127, 128, view.shape, generator=g, dtype=I8).cuda()
        z = torch.rand(2, 2, 4, heads, generator=g).cuda()
        view.copy_(small)
        mine, z2 = (small.clone(), other.clone()), z.clone()
        cache_copy(view, other, *z, copies)
        for x in mine:
            x[:, 2], x[:, 1, :, :7] = x[:, 3], x[:, 0, :, :7]
        z2[:, :, 1], z2[:, :, 2] = z2[:, :, 0], z2[:, :, 3]
        assert torch.equal(view, mine[0]) and torch.equal(other, mine[1]) and torch.equal(z, z2)
