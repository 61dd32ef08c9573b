"""What the operators on pages of a cache do, entry by entry on lists of numbers, and inputs for their tests."""
from __future__ import annotations

import random

import torch


def fork_ref(pages, lengths, holders, parents, page):
    """The lists as the call leaves them."""
    B, n = len(pages), len(holders)
    before, tokens = [list(r) for r in pages], list(lengths)
    pages, holders = [list(r) for r in pages], list(holders)
    for b, p in enumerate(parents):
        if p == b or not -1 <= p < B:
            continue
        row = [-1] * len(before[b])
        if p >= 0:
            for c in range(len(row)):
                if c * page < tokens[p]:
                    row[c] = before[p][c]
        for e in before[b]:
            if 0 <= e < n:
                holders[e] -= 1
        for e in row:
            if 0 <= e < n:
                holders[e] += 1
        pages[b] = row
        lengths[b] = tokens[p] if p >= 0 else 0
    return pages, lengths, holders


def reserve_ref(pages, lengths, holders, page, counts):
    """(pages, holders, copies) as the call leaves them: row by row, each page by itself."""
    n, columns = len(holders), len(pages[0])
    pages, holders = [list(r) for r in pages], list(holders)
    free = [p for p in range(n) if holders[p] == 0]
    copies, dropped, places = [(-1, -1, 0)] * len(pages), [], []
    for b, (length, count) in enumerate(zip(lengths, counts)):
        if 0 < count <= length <= columns * page:
            start = length - count
            places += [(b, c, max(start - c * page, 0)) for c in range(start // page, -(-length // page))]
    leave = set()
    for b, c, older in places:
        e = pages[b][c]
        if older and 0 <= e < n and holders[e] > 1:
            holders[e] -= 1
            leave.add(b)
    held = list(holders)
    for b, c, older in places:
        e = pages[b][c]
        there = 0 <= e < n
        if older and b not in leave:
            continue            # its own, or tokens that are not there
        if not older and there:
            if held[e] < 2:
                continue
            dropped.append(e)   # (free when the call is over)
        got = free.pop(0) if free else -1
        if older and got >= 0:
            copies[b] = (e, got, older)
        if got >= 0:
            holders[got] = 1
        pages[b][c] = got
    for e in dropped:
        holders[e] -= 1
    return pages, holders, copies


def compact_ref(pages, holders, page):
    """(pages, holders, copies) as the call leaves them."""
    held = [p for p, h in enumerate(holders) if h]
    n = len(held)
    moves = dict(zip([p for p in held if p >= n], [p for p in range(n) if not holders[p]]))
    holders = list(holders)
    for p, to in moves.items():
        holders[to], holders[p] = holders[p], 0
    copies = [(p, to, page) for p, to in moves.items()]
    copies += [(-1, -1, 0)] * (max(len(holders) // 2, 1) - len(copies))
    return [[moves.get(e, e) for e in r] for r in pages], holders, copies


def random_state(B, columns, page, spare, seed, sharing=0.5, longest=None):
    """(pages, lengths, holders) of sequences as earlier calls leave them: runs of rows that share their first
    pages, at times a page that is partly filled too; free pages between the held ones."""
    r = random.Random(seed)
    lengths = [r.choice((0, r.randint(0, longest or columns * page), r.randint(0, page))) for _ in range(B)]
    need = sum(-(-n // page) for n in lengths)
    total = max(1, need + spare)
    order = list(range(total))
    r.shuffle(order)
    pages = []
    for b in range(B):
        used = -(-lengths[b] // page)
        row = [order.pop() for _ in range(used)]
        if b and r.random() < sharing:
            other, m = pages[b - 1], r.randint(0, used)
            for c in range(m):
                if other[c] < 0:
                    break
                order.append(row[c])
                row[c] = other[c]
        pages.append(row + [-1] * (columns - used))
    holders = [0] * total
    for row in pages:
        for e in row:
            if e >= 0:
                holders[e] += 1
    return pages, lengths, holders


def ints(x, device="cuda"):
    return torch.tensor(x, dtype=torch.int32, device=device)
