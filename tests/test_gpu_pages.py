"""Pages of a cache that sequences share, leave and get, on the GPU: whole numbers, against their definitions
entry by entry, and copies bit by bit."""
import random

import pytest
import torch

from _pages import compact_ref, fork_ref, ints, random_state, reserve_ref
from _util import ensure_built

pytestmark = pytest.mark.gpu
I8, E4M3 = torch.int8, torch.float8_e4m3fn


def _table(pages, layout):
    """The rows as they are, or as part of a wider table."""
    if layout == "plain":
        return ints(pages)
    x = torch.full((len(pages), len(pages[0]) + 5), 7, dtype=torch.int32, device="cuda")
    x[:, 2:-3] = ints(pages)
    return x[:, 2:-3]


_SIZES = [
    # rows, columns, tokens of a page, free pages besides
    (1, 1, 16, 0), (2, 1, 16, 3), (4, 6, 16, 40), (5, 67, 64, 9), (32, 9, 48, 100), (70, 33, 128, 500),
    (300, 5, 16, 700), (1100, 3, 64, 900), (9, 1000, 16, 3000), (4096, 1, 16, 50), (2100, 12, 32, 20),
]


@pytest.mark.parametrize("B,columns,page,spare", _SIZES)
@pytest.mark.parametrize("layout", ["plain", "wide"])
def test_fork(B, columns, page, spare, layout):
    ensure_built()
    from e_natten_amd import cache_fork
    print("case fork", B, columns, page, spare, layout, flush=True)
    for seed in range(3):
        pages, lengths, holders = random_state(B, columns, page, spare, seed)
        r = random.Random(seed + 10)
        parents = [r.choice((b, r.randint(-1, B - 1), r.randint(0, B - 1), -1, -2, B, 2 ** 31 - 1)) for b in range(B)]
        if seed == 1:   # all continue one
            parents = [r.randint(0, B - 1)] * B
        if seed == 2:   # entries and lengths that nobody should have written
            for b in range(0, B, 3):
                pages[b][r.randint(0, columns - 1)] = r.choice((-7, len(holders), 2 ** 31 - 1, -2 ** 31))
                lengths[b] = r.choice((-5, 10 * columns * page, 2 ** 31 - 1, lengths[b]))
        want = fork_ref(pages, list(lengths), holders, parents, page)
        p, n, h = _table(pages, layout), ints(lengths), ints(holders)
        cache_fork(p, n, h, ints(parents), page)
        for got, ref in zip((p, n, h), want):
            assert got.tolist() == ref, seed
        if layout == "wide":
            assert (p._base[:, :2] == 7).all() and (p._base[:, -3:] == 7).all()


@pytest.mark.parametrize("B,columns,page,spare", _SIZES)
@pytest.mark.parametrize("layout", ["plain", "wide"])
def test_reserve(B, columns, page, spare, layout):
    """Single tokens, several, whole prompts; more than there are pages for; numbers that do not fit together."""
    ensure_built()
    from e_natten_amd import cache_reserve
    print("case reserve", B, columns, page, spare, layout, flush=True)
    for seed in range(4):
        pages, lengths, holders = random_state(B, columns, page, spare, seed, longest=max(1, (columns - 1) * page))
        r = random.Random(seed + 20)
        most = (1, 17, columns * page, page)[seed]
        counts = [r.choice((r.randint(0, most), 1, 0)) for _ in range(B)]
        if seed == 0:
            counts = [1] * B
        lengths = [n + c for n, c in zip(lengths, counts)]
        if seed == 3:
            for b in range(0, B, 4):
                pages[b][r.randint(0, columns - 1)] = r.choice((-7, len(holders), 2 ** 31 - 1, -1))
                lengths[b], counts[b] = r.choice(((-5, 3), (4, 5), (columns * page + 1, 2), (2 ** 31 - 1, 9), (5, -1),
                                                  (lengths[b], counts[b])))
        want = reserve_ref(pages, lengths, holders, page, counts)
        p, h = _table(pages, layout), ints(holders)
        if layout == "wide":   # (not at a multiple of 16 bytes)
            h = torch.cat((ints([3]), h))[1:]
        n = ints(lengths)
        copies = cache_reserve(p, n, h, page, 1 if seed == 0 else ints(counts))
        assert p.tolist() == want[0] and h.tolist() == want[1], seed
        assert copies.tolist() == [list(c) for c in want[2]], seed
        assert n.tolist() == lengths


def test_lengths_and_holders_between_the_rows_of_a_wider_table():
    """One allocation for all of a program's numbers: refused only where elements are the same."""
    ensure_built()
    from e_natten_amd import cache_fork, cache_reserve
    pages, lengths, holders = random_state(3, 4, 16, 5, 1)
    n = len(holders)
    state = torch.full((3, 4 + 3 + n), 7, dtype=torch.int32, device="cuda")
    p, m, h = state[:, :4], state[0, 4:7], state[1, 7:]
    p.copy_(ints(pages)), m.copy_(ints(lengths)), h.copy_(ints(holders))
    want = fork_ref(pages, lengths, holders, [1, 1, 0], 16)
    cache_fork(p, m, h, ints([1, 1, 0]), 16)
    assert [x.tolist() for x in (p, m, h)] == list(want)
    with pytest.raises(ValueError, match="share memory"):
        cache_fork(p, m, h, m, 16)
    with pytest.raises(ValueError, match="share memory"):
        cache_reserve(state[:, :8], m, h, 16)
    count = ints([5, 5, 5])
    cache_reserve(p, count, h, 16, count)   # whole prompts: lengths and counts may be one tensor


def test_reserve_gives_every_holder_of_a_page_its_own():
    """All rows that hold a page write to it: the last one keeps it.  A row that only reads it holds it on."""
    ensure_built()
    from e_natten_amd import cache_reserve
    for reader in (False, True):
        rows = 5
        pages = [[9, 4, -1]] * rows
        holders = [0] * 12
        holders[9] = holders[4] = rows
        counts = [1] * (rows - 1) + [0 if reader else 1]
        lengths = [16 + 3 + c for c in counts]
        p, h = ints(pages), ints(holders)
        copies = cache_reserve(p, ints(lengths), h, 16, ints(counts)).tolist()
        taken = [0, 1, 2, 3]
        assert copies[:4] == [[4, t, 3] for t in taken] and copies[4] == [-1, -1, 0]
        assert p.tolist() == [[9, t, -1] for t in taken] + [[9, 4, -1]]
        assert h.tolist() == [1, 1, 1, 1, 1, 0, 0, 0, 0, 5, 0, 0]


@pytest.mark.parametrize("B,columns,page,spare", _SIZES)
def test_lengths_that_went_back(B, columns, page, spare):
    """Rows whose length went back behind tokens that they share, or have on pages of their own: new tokens never go to a
    page that others hold."""
    ensure_built()
    from e_natten_amd import cache_reserve
    print("case back", B, columns, page, spare, flush=True)
    replaced = 0
    for seed in range(4):
        pages, lengths, holders = random_state(B, columns, page, spare, seed, sharing=0.8)
        r = random.Random(seed)
        for b in range(1, B):   # whole rows that others hold, as forks leave them
            if r.random() < 0.4:
                for e in pages[b]:
                    holders[e] -= e >= 0
                pages[b], lengths[b] = list(pages[b - 1]), lengths[b - 1]
                for e in pages[b]:
                    holders[e] += e >= 0
        kept = [r.choice((n, n // page * page, r.randint(0, n), max(n - 3, 0))) for n in lengths]
        # (few new tokens where all of a row have few columns, many else)
        counts = [min(r.choice((0, 1, 2, page, 2 * page if seed % 2 else columns * page)), columns * page - k) for k in kept]
        now = [k + c for k, c in zip(kept, counts)]
        want = reserve_ref(pages, now, holders, page, counts)
        p, h = ints(pages), ints(holders)
        copies = cache_reserve(p, ints(now), h, page, ints(counts))
        assert p.tolist() == want[0] and h.tolist() == want[1] and copies.tolist() == [list(x) for x in want[2]], seed
        for b in range(B):
            for c in range(kept[b] // page, -(-now[b] // page)):
                e = want[0][b][c]
                if counts[b] and e >= 0:
                    assert want[1][e] == 1
                    replaced += 0 <= pages[b][c] != e
    assert replaced or B == 1


def test_a_pool_that_runs_out():
    """The first rows get what there is; the others' entries are no pages, and stay none while they should hold
    older tokens."""
    ensure_built()
    from e_natten_amd import cache_reserve
    pages, holders = [[0, -1], [1, -1], [1, -1]], [1, 2, 0]
    p, h = ints(pages), ints(holders)
    copies = cache_reserve(p, ints([17, 6, 6]), h, 16, 1)
    assert p.tolist() == [[0, 2], [-1, -1], [1, -1]] and h.tolist() == [1, 1, 1]
    assert copies.tolist() == [[-1, -1, 0]] * 3
    h[2] = 0
    copies = cache_reserve(p, ints([18, 7, 7]), h, 16, 1)
    assert p.tolist() == [[0, 2], [-1, -1], [1, -1]] and copies.tolist() == [[-1, -1, 0]] * 3


@pytest.mark.parametrize("B,columns,page,spare", _SIZES)
@pytest.mark.parametrize("layout", ["plain", "wide"])
def test_compact(B, columns, page, spare, layout):
    ensure_built()
    from e_natten_amd import cache_compact
    print("case compact", B, columns, page, spare, layout, flush=True)
    for seed in range(3):
        pages, lengths, holders = random_state(B, columns, page, spare, seed)
        r = random.Random(seed)
        if seed == 1:   # held by no row; entries that are none
            for i in r.sample(range(len(holders)), len(holders) // 3):
                holders[i] += 1
            pages[0][0], pages[-1][-1] = 2 ** 31 - 1, -9
        if seed == 2:
            holders = [int(h > 0 and r.random() < 0.5) for h in holders]
        want = compact_ref(pages, holders, page)
        p, h = _table(pages, layout), ints(holders)
        if layout == "wide":
            h = torch.cat((ints([3]), h))[1:]
        copies = cache_compact(p, h, page)
        assert p.tolist() == want[0] and h.tolist() == want[1], seed
        assert copies.tolist() == [list(c) for c in want[2]], seed


@pytest.mark.parametrize("total", [1, 2, 3, 2047, 2048, 2049, 4096, 10000, 300000])
def test_compact_of_whole_pools(total):
    """Nothing held, everything, only the last page, only the second half."""
    ensure_built()
    from e_natten_amd import cache_compact
    at = torch.arange(total)
    for which in (at < 0, at >= 0, at == total - 1, at >= total // 2, at % 2 == 1):
        holders = which.int()
        n = int(which.sum())
        h, p = holders.cuda(), at[which][-1:].int().repeat(2, 1).cuda() if n else ints([[-1], [-1]])
        copies = cache_compact(p, h, 16).cpu()
        assert torch.equal(h.cpu(), (at < n).int())
        high, low = at[which & (at >= n)], at[~which & (at < n)]
        k = len(high)
        assert torch.equal(copies[:k, 0].long(), high) and torch.equal(copies[:k, 1].long(), low)
        assert (copies[:k, 2] == 16).all() and (copies[k:] == torch.tensor([-1, -1, 0])).all()
        last = int(at[which][-1]) if n else -1
        assert p.tolist() == [[int(low[-1]) if last >= n else last]] * 2


def _pool(layers, total, heads, page, d, dtype, layout, seed):
    """(k, v, ks, vs) on the GPU, 5-D, or 4-D without layers."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    shape = ((layers,) if layers else ()) + (total, heads, page, d)

    def some(*s):
        return torch.randint(-128, 128, s, dtype=torch.int8, generator=g, device="cuda")

    if layout == "plain":
        k, v = some(*shape), some(*shape)
    elif layout == "tokens":   # [.., pages, page, heads, d + 16]
        k, v = (some(*shape[:-3], page, heads, d + 16)[..., 16:].transpose(-2, -3) for _ in range(2))
    else:                      # keys and values side by side in one pool, layers inside the pages
        x = some(total, max(layers, 1), 2, heads, page, d)
        k, v = (x[:, :, i].transpose(0, 1) for i in range(2))
        k, v = (k, v) if layers else (k[0], v[0])
    z = torch.rand(2, *shape[:-2], generator=g, device="cuda")
    return k.view(dtype) if k.dtype != dtype else k, v.view(dtype) if v.dtype != dtype else v, z[0], z[1]


@pytest.mark.parametrize("layers,total,heads,page,d,n,dtype,layout", [
    (0, 3, 1, 16, 16, 1, I8, "plain"), (0, 40, 2, 16, 64, 11, E4M3, "plain"), (3, 60, 5, 48, 80, 20, I8, "plain"),
    (2, 50, 3, 64, 128, 17, E4M3, "tokens"), (4, 30, 8, 128, 256, 10, I8, "pairs"), (0, 300, 4, 32, 96, 100, I8, "pairs"),
    (1, 9, 1, 1024, 48, 3, E4M3, "plain"), (2, 5000, 1, 16, 16, 2400, I8, "plain"), (33, 12, 16, 16, 32, 4, I8, "tokens"),
])
def test_copy(layers, total, heads, page, d, n, dtype, layout):
    ensure_built()
    from e_natten_amd import cache_copy
    print("case copy", layers, total, heads, page, d, n, dtype, layout, flush=True)
    r = random.Random(n)
    order = r.sample(range(total), min(total, 2 * n))
    copies = [[order[2 * i], order[2 * i + 1], r.choice((page, 1, r.randint(1, page), page + 5, 2 ** 31 - 1))]
              for i in range(len(order) // 2)]
    copies += [[-1, -1, 0], [0, total, 4], [total, 0, 4], [2, 2, 7], [1, 0, 0], [1, 0, -3], [-2 ** 31, 1, 9], [0, -1, page]]
    copies += [[-1, -1, 0]] * 3 * n
    r.shuffle(copies)
    pool = _pool(layers, total, heads, page, d, dtype, layout, 3)
    bits = [x.view(torch.uint8) if x.dtype != torch.float32 else x for x in pool]
    want = [x.clone() for x in bits]
    for s, t, m in copies:
        if s == t or m < 1 or not 0 <= s < total or not 0 <= t < total:
            continue
        for x in want:
            x = x if layers else x[None]
            if x.dtype == torch.float32:
                x[:, t] = x[:, s]
            else:
                x[:, t, :, :m] = x[:, s, :, :m]
    cache_copy(*pool, ints(copies))
    assert all(torch.equal(x, y) for x, y in zip(bits, want))
    cache_copy(*pool, ints(copies)[:0])
    assert all(torch.equal(x, y) for x, y in zip(bits, want))
