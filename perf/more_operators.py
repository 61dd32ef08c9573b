"""What a model needs that gives many answers to one prompt, as cases that can be timed.

The prompt may hold images or video, is read once, and is continued by several sequences: positions
with several axes (``rotary`` with ``axes``), pages of the cache that sequences share, leave and get
(``cache_fork``, ``cache_reserve``, ``cache_copy``, ``cache_compact``), and attention that reads a shared
prompt once for all of its sequences (``cache_attention`` with ``shared``).  With ``own`` false the
same is computed in elementary torch operations.

Fields of a case
    op        "rotary", "step", "compact" or "attend"
    dtype     of q and k: "bf16", "fp16" or "fp32"
    B, Nq, Nk, T, d   sequences, heads of q, heads of k and v, new tokens of each sequence, head_dim
    rotary:   R, channels that are rotated; axes, how many; order, whether an axis has a run of
              neighbouring pairs ("blocks") or every axes-th pair ("cyclic"); interleaved; mode "train"
              (forward and backward) or "infer"; layout "plain" ([B, heads, T, d]), "proj" (views of one
              projection [B, T, heads of q, k and v, d]) or "grid" (views [B, heads, H, W, d] of one
              projection [B, H, W, heads, d], T = H W); H, W, rows and columns of an image
    step, compact:   cache, "int8" or "e4m3"; page, tokens of a page; layers of the pool; longest,
              tokens of the longest sequence (the shortest has about half); spare, free pages of the
              pool for every sequence
              step: what happens between two steps of a model: sequences go on, are continued by others
              or end, get pages for T new tokens each, and what they wrote into shared pages is copied.
              group, neighbouring sequences of which one in `group` is continued by all (beams,
              samples); incoming, prompts of up to so many tokens that take every other row (0: none)
              compact: every other sequence has ended since; held pages move to the low end
    attend:   cache, page; runs, into which the B sequences fall; shared, tokens that the sequences of
              the longest run share (those of the last have about half); longest, own tokens of the
              longest sequence behind these, its new ones included; ragged, whether the sequences bring
              different numbers of new tokens; window, how many tokens a query sees, its own the last
              (0: all)
"""
import math

import torch

own = False

_DTYPE = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_CACHE = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
_TOP = {"int8": 127.0, "e4m3": 448.0}


def _rotary(**fields):
    return dict({"op": "rotary", "dtype": "bf16", "B": 1, "interleaved": False, "order": "blocks", "axes": 3,
                 "mode": "infer", "layout": "plain", "H": 0, "W": 0}, **fields)


def _step(**fields):
    return dict({"op": "step", "cache": "int8", "T": 1, "group": 1, "incoming": 0, "layers": 1, "spare": 2},
                **fields)


def _compact(**fields):
    return dict({"op": "compact", "cache": "int8", "layers": 1, "spare": 2}, **fields)


def _attend(**fields):
    return dict({"op": "attend", "dtype": "bf16", "T": 1, "runs": 1, "ragged": False, "window": 0}, **fields)


def listed():
    return [
        # one token for each of eight sequences, three axes: the smallest call, only latency counts
        _rotary(name="axes_token", B=8, Nq=16, Nk=16, T=1, d=128, R=128),
        # a layer of neighborhood attention over images in training: rows and columns, the image of
        # natten2d's own benchmark as its attention takes it
        _rotary(name="axes_image", mode="train", layout="grid", axes=2, B=4, Nq=4, Nk=4, T=16384, H=128, W=128,
                d=128, R=128),
        # reading a prompt of video: time, rows and columns over every third pair, shared heads of k,
        # pairs side by side, half precision
        _rotary(name="axes_video", dtype="fp16", layout="proj", order="cyclic", interleaved=True, B=2, Nq=16,
                Nk=4, T=8192, H=28, W=28, d=128, R=96),
        # four beams of one prompt: only latency counts
        _step(name="step_beams", B=4, Nk=4, d=64, page=16, longest=60, group=4),
        # many prompts with several samples each, a pool of several layers: the copies count
        _step(name="step_samples", cache="e4m3", B=128, Nk=8, d=128, page=64, longest=480, group=4, layers=4),
        # prompts come in where sequences have ended, a large pool of small pages: the tables count
        _step(name="step_prompts", B=64, Nk=1, d=32, page=16, longest=8192, incoming=8192, spare=256),
        # a small pool after half of its sequences have ended
        _compact(name="compact_small", B=8, Nk=2, d=64, page=16, longest=500),
        # a large one, several layers
        _compact(name="compact_large", cache="e4m3", B=32, Nk=8, d=128, page=32, longest=2000, layers=2),
        # eight samples of a short prompt, one token each: only latency counts
        _attend(name="shared_small", cache="int8", B=8, Nq=16, Nk=16, d=128, page=32, shared=500, longest=40),
        # many samples of one long prompt
        _attend(name="shared_long", cache="e4m3", B=64, Nq=32, Nk=8, d=128, page=64, shared=16384, longest=500),
        # beams of many prompts of different lengths
        _attend(name="shared_beams", cache="int8", B=64, Nq=32, Nk=4, d=128, page=64, runs=16, shared=8192,
                longest=300),
        # a few drafted tokens each, odd sizes throughout, a window that cuts the prompt, float32
        _attend(name="shared_odd_fp32", dtype="fp32", cache="int8", B=9, Nq=15, Nk=5, T=5, d=80, page=48, runs=3,
                shared=1500, longest=211, ragged=True, window=1000),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


# no drawn case has more of either than the largest listed ones, nor a larger pool or larger products in between
_MAX_BYTES, _MAX_FLOPS, _MAX_POOL, _MAX_PAIRS = 5.5e8, 1.8e10, 7e8, 3.5e7


def _pool_bytes(case):
    tokens = case["B"] * (case["longest"] + case["page"] * case["spare"])
    return 2 * case["layers"] * case["Nk"] * case["d"] * tokens


def _fit(case):
    def large():
        w = work(case)
        return (w["bytes"] > _MAX_BYTES or w["flops"] > _MAX_FLOPS
                or case["op"] in ("step", "compact") and _pool_bytes(case) > _MAX_POOL
                or case["op"] == "attend" and case["B"] * case["Nq"] * case["T"]
                * (case["shared"] + case["longest"]) > _MAX_PAIRS)

    while large():
        runs = case.get("runs", 1)
        size = case["B"] // runs  # sequences of a run
        if case.get("layers", 1) > 1:
            case["layers"] //= 2
        elif size > 2:
            case["B"] = (size + 1) // 2 * runs
        elif case["op"] == "rotary" and case["layout"] == "grid" and case["H"] > 1:
            case["H"] = (case["H"] + 1) // 2
            case["T"] = case["H"] * case["W"]
        elif case["op"] == "rotary" and case["layout"] != "grid" and case["T"] > 1:
            case["T"] = (case["T"] + 1) // 2
        elif case["op"] == "attend" and runs > 1:
            case.update(runs=runs // 2, B=runs // 2 * size)
        elif case["op"] == "attend":
            case["T"] = (case["T"] + 1) // 2
            case["shared"] = (case["shared"] + 1) // 2
            case["longest"] = case["T"] + case["longest"] // 2
        else:
            case["longest"] = (case["longest"] + 1) // 2
            case["spare"] = 2 + (case["spare"] - 2) // 2
            if case.get("incoming"):
                case["incoming"] = max(1, min(case["incoming"] // 2, case["page"] * (case["spare"] - 2)))
    return case


def draw(rng):
    """One more case: an operator, then sizes over its whole range."""
    op = rng.choice(("rotary", "step", "step", "compact", "attend", "attend", "attend"))
    dtype = rng.choice(("bf16", "bf16", "bf16", "fp16", "fp16", "fp32"))
    Nk, cache = rng.choice((1, 2, 3, 4, 8, 8, 16)), rng.choice(("int8", "e4m3"))
    page = rng.choice((16, 32, 48, 64, 64, 128))
    if op == "rotary":
        d, layout = rng.choice((32, 64, 80, 96, 128, 128, 192, 256)), rng.choice(("plain", "proj", "grid"))
        axes, H, W = rng.choice((2, 3, 3, 4)), _log_int(rng, 1, 128), _log_int(rng, 1, 128)
        return _fit(_rotary(
            dtype=dtype, mode=rng.choice(("train", "infer")), layout=layout, B=_log_int(rng, 1, 64),
            Nq=Nk * rng.choice((1, 1, 2, 4, 7)), Nk=Nk, H=H, W=W,
            T=H * W if layout == "grid" else _log_int(rng, 1, 16384), d=d, R=rng.choice((d, d, d // 2, d // 4)),
            axes=axes, order=rng.choice(("blocks", "cyclic")), interleaved=rng.random() < 0.4))
    d = rng.choice((32, 64, 64, 80, 96, 128, 128, 128, 192, 256))
    if op == "attend":
        runs = rng.choice((1, 1, 2, 3, _log_int(rng, 1, 32)))
        T = rng.choice((1, 1, 1, rng.randint(2, 8), _log_int(rng, 8, 64)))
        return _fit(_attend(
            dtype=dtype, cache=cache, B=runs * _log_int(rng, 2, 64), Nq=Nk * rng.choice((1, 2, 4, 4, 6, 8)), Nk=Nk,
            T=T, d=d, page=page, runs=runs, shared=_log_int(rng, 1, 32768), longest=T + _log_int(rng, 1, 2048),
            ragged=rng.random() < 0.5, window=rng.choice((0, 0, 0, _log_int(rng, 1, 8192)))))
    fields = dict(cache=cache, B=_log_int(rng, 2, 256), Nk=Nk, d=d, page=page, layers=rng.choice((1, 2, 4, 8)),
                  longest=_log_int(rng, 1, 4096), spare=rng.randint(2, 8))
    if op == "compact":
        return _fit(_compact(**fields))
    T = rng.choice((1, 1, rng.randint(2, 16)))
    incoming = rng.choice((0, _log_int(rng, 1, 4096)))
    return _fit(_step(T=T, group=rng.choice((1, 2, 4, 4, 5, 16)), incoming=incoming,
                      **dict(fields, spare=-(-incoming // page) + fields["spare"])))


def _lengths(case):
    """Tokens of each sequence: from the longest down to about half.  (attend: those behind the shared
    ones, the new ones included)"""
    counts = _counts(case) if case["op"] == "attend" else [0] * case["B"]
    return [max(c, case["longest"] - b * case["longest"] // (2 * case["B"])) for b, c in enumerate(counts)]


def _counts(case):
    """attend: new tokens of each sequence."""
    T = case["T"]
    return [T - (b * T // (2 * case["B"]) if case["ragged"] else 0) for b in range(case["B"])]


def _shared(case):
    """attend: tokens that the sequences of each run share."""
    return [case["shared"] - r * case["shared"] // (2 * case["runs"]) for r in range(case["runs"])]


def _frequencies(case):
    """One angle per position and pair of channels, base 10000: each axis has the whole range if it has its
    own run of pairs, else the axes take turns along one range.  Also the axis of every pair."""
    half, axes = case["R"] // 2, case["axes"]
    if case["order"] == "cyclic":
        return [10000.0 ** (-i / half) for i in range(half)], [i % axes for i in range(half)]
    sizes = [half // axes + (a < half % axes) for a in range(axes)]
    return ([10000.0 ** (-i / n) for n in sizes for i in range(n)],
            [a for a, n in enumerate(sizes) for _ in range(n)])


def _normal(gen, *shape, dtype=torch.float32):
    return torch.randn(shape, generator=gen, device="cuda", dtype=dtype)


def _qk(gen, case):
    B, Nq, Nk, T, d = (case[k] for k in ("B", "Nq", "Nk", "T", "d"))
    dtype = _DTYPE[case["dtype"]]
    if case["layout"] == "plain":
        return [_normal(gen, B, Nq, T, d, dtype=dtype), _normal(gen, B, Nk, T, d, dtype=dtype)]
    sizes = (case["H"], case["W"]) if case["layout"] == "grid" else (T,)
    x = _normal(gen, B, *sizes, Nq + 2 * Nk, d, dtype=dtype)
    return [y.movedim(-2, 1) for y in (x[..., :Nq, :], x[..., Nq:Nq + Nk, :])]


def _positions(gen, case):
    """Rows and columns of an image, or with more axes frames of images in a row behind some text; a fourth
    axis counts the tokens.  [axes, B, T], or [axes, H, W] for one grid."""
    H, W, T, axes = max(case["H"], 1), max(case["W"], 1), case["T"], case["axes"]
    t = torch.arange(T, device="cuda")
    frame = [t // W % H, t % W] if axes == 2 else [t // (H * W), t // W % H, t % W, t][:axes]
    p = torch.stack(frame)
    if case["layout"] == "grid":
        return p.view(axes, case["H"], case["W"])
    first = torch.randint(0, 1000, (case["B"], 1), generator=gen, device="cuda")
    return p[:, None] + first


def _blocks(gen, case, count):
    """Pages as earlier calls left them: codes of normal values, scales for maxima of about 4 sigma."""
    top = _TOP[case["cache"]]
    shape = (case.get("layers", 1), count, case["Nk"], case["page"], case["d"])
    codes = torch.empty(shape, dtype=_CACHE[case["cache"]], device="cuda")
    for layer in codes:
        x = (_normal(gen, *shape[1:], dtype=torch.bfloat16) * (top / 4)).clamp(-top, top)
        layer.copy_(x.round() if case["cache"] == "int8" else x)
    scale = torch.rand(shape[:3], generator=gen, device="cuda") * 0.5 + 0.75
    return codes, scale * (4 / top)


def _table(gen, lengths, page, columns, total):
    """Pages of the sequences in a random order over the pool, -1 behind the last, on the host."""
    order = torch.randperm(total, generator=gen, device="cuda").tolist()
    rows, at = [], 0
    for n in lengths:
        need = -(-n // page)
        rows.append(order[at:at + need] + [-1] * (columns - need))
        at += need
    return rows


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _parents(gen, case):
    """Row by row which sequence it continues: one of the group for all of it, now and then itself; where
    prompts come in, every other row ends."""
    B, group = case["B"], case["group"]
    rows = torch.arange(B, device="cuda")
    base = rows // group * group
    chosen = torch.randint(0, group, (B,), generator=gen, device="cuda")[base]
    parents = torch.minimum(base + chosen, torch.tensor(B - 1, device="cuda"))
    stays = torch.rand(B, generator=gen, device="cuda") < 0.125
    parents = torch.where(stays, rows, parents)
    if case["incoming"]:
        parents = torch.where(rows % 2 == 1, -1, torch.where(parents % 2 == 1, rows, parents))
    return parents.to(torch.int32)


def _prepare_pages(gen, case):
    B, page, lengths = case["B"], case["page"], _lengths(case)
    columns = -(-(max(lengths) + max(case.get("T", 1), case.get("incoming", 0))) // page) + 1
    need = sum(-(-n // page) for n in lengths)
    total = need + case["B"] * case["spare"]
    table = _table(gen, lengths, page, columns, total)
    if case["op"] == "compact":
        table = [r if b % 2 == 0 else [-1] * columns for b, r in enumerate(table)]
    holders = [0] * total
    for r in table:
        for p in r:
            if p >= 0:
                holders[p] += 1
    k, ks = _blocks(gen, case, total)
    v, vs = _blocks(gen, case, total)
    state = {"case": case, "pages": _ints(table), "holders": _ints(holders), "k": k, "v": v, "ks": ks, "vs": vs}
    if case["op"] == "compact":
        return dict(state, pages_then=state["pages"].clone(), holders_then=state["holders"].clone())
    counts = torch.full((B,), case["T"], dtype=torch.int32, device="cuda")
    parents = _parents(gen, case)
    if case["incoming"]:
        new = torch.randint(1, case["incoming"] + 1, (B,), generator=gen, device="cuda", dtype=torch.int32)
        counts = torch.where(parents < 0, new, counts)
    return dict(state, lengths=_ints(lengths), parents=parents, counts=counts)


def _prepare_attend(gen, case):
    B, page, T, runs = (case[k] for k in ("B", "page", "T", "runs"))
    shared, counts, behind = _shared(case), _counts(case), _lengths(case)
    size = B // runs
    lengths = [shared[b // size] + n for b, n in enumerate(behind)]
    columns = -(-max(lengths) // page) + 1
    common = [n // page for n in shared]  # whole pages
    need = [-(-n // page) - common[b // size] for b, n in enumerate(lengths)]
    total = sum(common) + sum(need)
    order = torch.randperm(total, generator=gen, device="cuda").tolist()
    table, at = [], sum(common)
    for b, n in enumerate(need):
        r = b // size
        first = sum(common[:r])
        row = order[first:first + common[r]] + order[at:at + n]
        at += n
        table.append(row + [-1] * (columns - len(row)))
    state = {"case": case, "pages": _ints(table), "lengths": _ints(lengths), "shared": _ints(shared),
             "counts": _ints(counts) if case["ragged"] else None}
    for x in ("k", "v"):
        codes, scale = _blocks(gen, case, total)
        state[x], state[x + "s"] = codes[0], scale[0]
    # logits of a standard deviation of 2
    state["q"] = (_normal(gen, B, T, case["Nq"], case["d"]) * 2).to(_DTYPE[case["dtype"]]).transpose(1, 2)
    return state


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "attend":
        return _prepare_attend(gen, case)
    if case["op"] != "rotary":
        return _prepare_pages(gen, case)
    train = case["mode"] == "train"
    frequencies, axes = _frequencies(case)
    return {"case": case, "qk": [x.requires_grad_(train) for x in _qk(gen, case)],
            "positions": _positions(gen, case), "axes": _ints(axes),
            "frequencies": torch.tensor(frequencies, device="cuda", dtype=torch.float64),
            "grads": _qk(gen, case) if train else None}


# --- the plain forms ---

def _turn(x, cos, sin, R, interleaved):
    """x with the pairs of its first R channels turned, in 32 bits."""
    part = x[..., :R].float()
    if interleaved:
        a, b = part[..., 0::2], part[..., 1::2]
        y = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
    else:
        a, b = part[..., :R // 2], part[..., R // 2:]
        y = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
    return torch.cat((y.to(x.dtype), x[..., R:]), dim=-1)


def _plain_rotary(s):
    case, (q, k) = s["case"], s["qk"]
    p = s["positions"][:, None] if case["layout"] == "grid" else s["positions"]
    angle = p.double()[s["axes"].long()].movedim(0, -1) * s["frequencies"]  # [B, T or H, W, pairs]
    angle = angle[:, None]
    cos, sin = angle.cos().float(), angle.sin().float()
    return (_turn(q, cos, sin, case["R"], case["interleaved"]), _turn(k, cos, sin, case["R"], case["interleaved"]))


def _add(holders, entries, by):
    """holders[e] += by for every entry that is a page."""
    n = holders.numel()
    entries = entries.flatten().long()
    there = (entries >= 0) & (entries < n)
    holders.index_add_(0, entries.clamp(0, n - 1), there.to(holders.dtype) * by)


def _plain_fork(pages, lengths, holders, parents, page):
    B, columns = pages.shape
    rows = torch.arange(B, device=pages.device)
    moved = (parents >= -1) & (parents < B) & (parents != rows)
    source = parents.clamp(0, B - 1).long()
    used = (-(-lengths // page)).clamp(0, columns)[source]
    kept = (moved & (parents >= 0))[:, None] & (torch.arange(columns, device=pages.device) < used[:, None])
    now = torch.where(moved[:, None], torch.where(kept, pages[source], -1), pages)
    _add(holders, pages, -1)
    _add(holders, now, 1)
    lengths.copy_(torch.where(moved, torch.where(parents >= 0, lengths[source], 0), lengths))
    pages.copy_(now)


def _ranked(which, most):
    """The places where `which` is true, in order, then -1: `most` of them."""
    place = torch.where(which, which.cumsum(0) - 1, most)
    at = torch.arange(which.numel(), device=which.device, dtype=torch.int32)
    return torch.full((most + 1,), -1, dtype=torch.int32, device=which.device).scatter_(0, place, at)[:most]


def _plain_reserve(pages, lengths, holders, page, counts):
    (B, columns), n = pages.shape, holders.numel()
    column, rows = torch.arange(columns, device=pages.device), torch.arange(B, device=pages.device)
    there = (pages >= 0) & (pages < n)
    start = lengths - counts
    some = (counts > 0) & (start >= 0) & (lengths <= columns * page)
    begun = some & (start % page != 0)  # the first page holds older tokens
    first = (start // page).clamp(0, columns - 1).long()[:, None]
    write = some[:, None] & (column >= first) & (column < -(-lengths // page)[:, None])
    at = pages.gather(1, first)[:, 0].clamp(0, n - 1).long()
    common = begun & there.gather(1, first)[:, 0] & (holders[at] > 1)
    writers = torch.zeros_like(holders).index_add_(0, at, common.to(holders.dtype))
    last = torch.full((n,), -1, device=pages.device).scatter_reduce_(0, at, torch.where(common, rows, -1), "amax")
    leaves = common & ~((writers[at] == holders[at]) & (last[at] == rows))
    wanted = write & ~there & ~(begun[:, None] & (column == first)) | leaves[:, None] & (column == first)
    free = _ranked(holders == 0, n)
    rank = wanted.flatten().cumsum(0).view(B, columns) - 1
    fresh = torch.where(rank < n, free[rank.clamp(0, n - 1)], -1)
    _add(holders, torch.where(leaves, at, -1), -1)
    _add(holders, torch.where(wanted, fresh, -1), 1)
    target = torch.where(leaves, fresh.gather(1, first)[:, 0], -1)
    pages.copy_(torch.where(wanted, fresh, pages))
    copied = target >= 0
    return torch.stack((torch.where(copied, at, -1), target, torch.where(copied, start % page, 0)), 1).to(torch.int32)


def _plain_compact(pages, holders, page):
    n = holders.numel()
    held, at = holders != 0, torch.arange(n, device=pages.device, dtype=torch.int32)
    count = held.sum()
    high, low, most = held & (at >= count), ~held & (at < count), max(1, n // 2)
    source, target = _ranked(high, most), _ranked(low, most)
    to = torch.where(high, target[(high.cumsum(0) - 1).clamp(0, most - 1)], at)
    inside = (pages >= 0) & (pages < n)
    pages.copy_(torch.where(inside, to[pages.clamp(0, n - 1).long()], pages))
    moved = torch.zeros_like(holders).index_add_(0, to.long(), holders)
    holders.copy_(moved)
    return torch.stack((source, target, torch.where(source >= 0, page, 0).to(torch.int32)), 1)


def _plain_copy(caches, scales, copies):
    source, target, tokens = copies.long()[copies[:, 0] >= 0].unbind(1)
    for x in caches:
        x = x.view(torch.int8)
        some = (torch.arange(x.shape[3], device=x.device) < tokens[:, None])[:, None, :, None]
        x[:, target] = torch.where(some, x[:, source], x[:, target])
    for z in scales:
        z[:, target] = z[:, source]


def _plain_attend(s):
    """The shared tokens turned into values once for every run, then each sequence's own."""
    case, q = s["case"], s["q"]
    B, Nq, Nk, T, d, page, runs = (case[k] for k in ("B", "Nq", "Nk", "T", "d", "page", "runs"))
    size, group = B // runs, Nq // Nk
    most = max(_shared(case)) // page
    behind = max(_lengths(case)) + page
    first = (s["shared"] // page).long()  # pages that are shared

    def values(x, table):  # [rows of the table, Nk, tokens, d]
        at = table.long().clamp(min=0)
        v = s[x][at].float() * s[x + "s"][at][..., None, None]
        return v.transpose(1, 2).reshape(table.shape[0], Nk, -1, d)

    column = first.repeat_interleave(size)[:, None] + torch.arange(-(-behind // page), device=q.device)
    own_table = s["pages"].gather(1, column.clamp(max=s["pages"].shape[1] - 1))
    counts = torch.full_like(s["lengths"], T) if s["counts"] is None else s["counts"]
    t = torch.arange(T, device=q.device)
    place = (s["lengths"] - counts)[:, None] + t
    live = (t < counts[:, None])[..., None]

    def logits(x, k, token, stop):  # x: rows by heads of the cache; token [B, tokens], stop [B]
        seen = live & (token[:, None] <= place[..., None]) & (token < stop[:, None])[:, None]
        if case["window"]:
            seen = seen & (token[:, None] > place[..., None] - case["window"])
        return x @ k.transpose(-1, -2), seen[:, None, None]

    x = q.float().reshape(B, Nk, group, T, d) * d ** -0.5
    token = column.repeat_interleave(page, 1) * page + torch.arange(column.shape[1] * page, device=q.device) % page
    own_k, own_v = values("k", own_table), values("v", own_table)
    y, seen = logits(x.flatten(2, 3), own_k, token, s["lengths"])
    parts = [y.unflatten(2, (group, T)).masked_fill(~seen, -math.inf)]
    if most:
        table = s["pages"][::size, :most]
        k, v = values("k", table), values("v", table)
        token = torch.arange(most * page, device=q.device).expand(B, -1)
        rows = x.unflatten(0, (runs, size)).transpose(1, 2).flatten(2, 4)
        y, seen = logits(rows, k, token, (first * page).repeat_interleave(size))
        y = y.unflatten(2, (size, group, T)).transpose(1, 2).flatten(0, 1)
        parts.append(y.masked_fill(~seen, -math.inf))
    top = torch.stack([p.amax(-1) for p in parts]).amax(0)[..., None]
    p = [(y - torch.where(top == -math.inf, 0.0, top)).exp() for y in parts]
    o = (p[0].flatten(2, 3) @ own_v).unflatten(2, (group, T))
    total = p[0].sum(-1, keepdim=True)
    if most:
        rows = p[1].unflatten(0, (runs, size)).transpose(1, 2).flatten(2, 4)
        y = (rows @ v).unflatten(2, (size, group, T)).transpose(1, 2).flatten(0, 1)
        o, total = o + y, total + p[1].sum(-1, keepdim=True)
    return (o / total.clamp(min=1e-30)).to(q.dtype).reshape(B, Nq, T, d)


def _readable(s, copies, lengths=None):
    """The tables, and the pool.  Codes are moved bit by bit, so they are whole numbers here."""
    out = {"pages": s["pages"], "holders": s["holders"], "copies": copies, "k_scale": s["ks"], "v_scale": s["vs"],
           "k": s["k"].view(torch.int8), "v": s["v"].view(torch.int8)}
    return out if lengths is None else dict(out, lengths=lengths)


def run(state):
    """One call: (q, k) with positions, and in training their gradients; what happens to the pages between
    two steps of a model; or what the new tokens read from the cache."""
    case = state["case"]
    if own:
        import e_natten_amd
    if case["op"] == "rotary":
        if own:
            out = e_natten_amd.rotary(*state["qk"], state["positions"], state["frequencies"], case["interleaved"],
                                      axes=state["axes"])
        else:
            out = _plain_rotary(state)
        if case["mode"] == "infer":
            return tuple(out)
        return (*out, *torch.autograd.grad(out, state["qk"], state["grads"]))
    if case["op"] == "attend":
        if own:
            return e_natten_amd.cache_attention(
                state["q"], state["k"], state["v"], state["ks"], state["vs"], state["pages"], state["lengths"],
                case["window"] or None, case["d"] ** -0.5, state["counts"], state["shared"])
        return _plain_attend(state)
    pages, holders, page, lengths = state["pages"], state["holders"], case["page"], None
    if case["op"] == "compact":
        # the pool as it was when the sequences had ended
        pages.copy_(state["pages_then"])
        holders.copy_(state["holders_then"])
        copies = e_natten_amd.cache_compact(pages, holders, page) if own else _plain_compact(pages, holders, page)
    else:
        fork, reserve = ((e_natten_amd.cache_fork, e_natten_amd.cache_reserve) if own
                         else (_plain_fork, _plain_reserve))
        fork(pages, state["lengths"], holders, state["parents"], page)
        lengths = state["lengths"] + state["counts"]
        copies = reserve(pages, lengths, holders, page, state["counts"])
    if own:
        e_natten_amd.cache_copy(state["k"], state["v"], state["ks"], state["vs"], copies)
    else:
        _plain_copy((state["k"], state["v"]), (state["ks"], state["vs"]), copies)
    return _readable(state, copies, lengths)


def work(case):
    """Bytes and operations that the call cannot do without.  rotary: q and k read and written (twice in
    training) and the positions, three operations a channel.  step and compact: the table read and written,
    the counts of holders read, the codes of the copied tokens read and written (about half a page for all
    but one sequence of a group; half of the held pages).  attend: the codes of the tokens that any query
    sees, the shared ones once, with their scales, q and the output; two products of length d per (query,
    token) pair."""
    if case["op"] == "rotary":
        passes, size = 2 if case["mode"] == "train" else 1, 4 if case["dtype"] == "fp32" else 2
        rows = case["B"] * case["T"] * (case["Nq"] + case["Nk"]) * passes
        positions = case["T"] * case["axes"] * (1 if case["layout"] == "grid" else case["B"]) * 8 * passes
        return {"bytes": rows * case["d"] * size * 2 + positions, "flops": rows * case["R"] * 3}
    B, page, lengths = case["B"], case["page"], _lengths(case)
    if case["op"] in ("step", "compact"):
        more = max(case.get("T", 1), case.get("incoming", 0))
        columns = -(-(max(lengths) + more) // page) + 1
        held = sum(-(-n // page) for n in lengths)
        total = held + B * case["spare"]
        token = 2 * case["layers"] * case["Nk"] * case["d"]
        if case["op"] == "compact":
            copied = held // 4 * page
        else:
            copied = (B - B // case["group"]) * page // 2 // (2 if case["incoming"] else 1)
        return {"bytes": 2 * 4 * B * columns + 4 * total + 2 * copied * token, "flops": 0}
    shared, counts, Nk, d = _shared(case), _counts(case), case["Nk"], case["d"]
    size, byte = B // case["runs"], 4 if case["dtype"] == "fp32" else 2
    tokens = pairs = 0
    for r, n in enumerate(shared):
        least = min(lengths[r * size:(r + 1) * size])
        tokens += max(0, min(n, (case["window"] or n + least) - least))
    for b, (n, c) in enumerate(zip(lengths, counts)):
        total = n + shared[b // size]
        w = case["window"] or total
        tokens += min(n, w + c - 1)
        pairs += sum(min(w, total - c + 1 + t) for t in range(c))
    rows = B * case["T"] * case["Nq"] * d * byte * 2
    return {"bytes": 2 * tokens * Nk * (d + 4 / page) + rows, "flops": 4 * pairs * case["Nq"] * d}


# --- the definitions, in 64 bits, and step by step on the host for what is whole ---

def _exact_rotary(s):
    case, half = s["case"], s["case"]["R"] // 2
    p, f = s["positions"].double(), s["frequencies"]
    if case["layout"] == "grid":
        p = p.flatten(1)[:, None]
    angle = torch.stack([p[a] * f[i] for i, a in enumerate(s["axes"].tolist())], -1)[:, None]  # [B or 1, 1, T, pairs]
    wheel = torch.polar(torch.ones_like(angle), angle)

    def turned(x, w):
        shape, x = x.shape, x.detach().double().flatten(2, -2)
        if case["interleaved"]:
            z = torch.view_as_complex(x[..., :2 * half].unflatten(-1, (half, 2)).contiguous()) * w
            y = torch.view_as_real(z).flatten(-2)
        else:
            z = torch.complex(x[..., :half].contiguous(), x[..., half:2 * half].contiguous()) * w
            y = torch.cat((z.real, z.imag), -1)
        return torch.cat((y, x[..., 2 * half:]), -1).view(shape)

    out = [turned(x, wheel) for x in s["qk"]]
    if s["grads"] is not None:
        out += [turned(g, wheel.conj()) for g in s["grads"]]
    return tuple(out)


def _exact_step(case, pages, lengths, holders, parents, counts):
    """Row by row: the copies; the lists hold what the call leaves."""
    page, columns = case["page"], len(pages[0])
    before, tokens = [list(r) for r in pages], list(lengths)
    for b, p in enumerate(parents):
        if p == b:
            continue
        for e in before[b]:
            if e >= 0:
                holders[e] -= 1
        used = -(-tokens[p] // page) if p >= 0 else 0
        pages[b] = (before[p][:used] if p >= 0 else []) + [-1] * (columns - used)
        lengths[b] = tokens[p] if p >= 0 else 0
        for e in pages[b]:
            if e >= 0:
                holders[e] += 1
    free = iter([p for p, h in enumerate(holders) if h == 0])
    copies = []
    for b, c in enumerate(counts):
        start, end, copy = lengths[b], lengths[b] + c, [-1, -1, 0]
        lengths[b] = end
        for column in range(start // page, -(-end // page)):
            e, older = pages[b][column], start - column * page
            if older > 0 and (e < 0 or holders[e] == 1):
                continue
            if older <= 0 and e >= 0:
                continue
            to = next(free, -1)
            if older > 0:
                holders[e] -= 1
                if to >= 0:
                    copy = [e, to, older]
            if to >= 0:
                holders[to] += 1
            pages[b][column] = to
        copies.append(copy)
    return copies


def _exact_pages(s):
    case = s["case"]
    pages, holders = s["pages"].tolist(), s["holders"].tolist()
    if case["op"] == "step":
        lengths = s["lengths"].tolist()
        copies = _exact_step(case, pages, lengths, holders, s["parents"].tolist(), s["counts"].tolist())
    else:
        lengths, n = None, sum(h > 0 for h in holders)
        high = [p for p, h in enumerate(holders) if h and p >= n]
        low = [p for p, h in enumerate(holders) if not h and p < n]
        for p, to in zip(high, low):
            holders[to], holders[p] = holders[p], 0
        moves = dict(zip(high, low))
        pages = [[moves.get(e, e) for e in r] for r in pages]
        copies = [[p, to, case["page"]] for p, to in moves.items()]
        copies += [[-1, -1, 0]] * (max(1, len(holders) // 2) - len(copies))
    for p, to, n in copies:
        if p >= 0:
            for x, z in (("k", "ks"), ("v", "vs")):
                s[x].view(torch.int8)[:, to, :, :n] = s[x].view(torch.int8)[:, p, :, :n]
                s[z][:, to] = s[z][:, p]
    out = {"pages": _ints(pages), "holders": _ints(holders), "copies": _ints(copies), "k_scale": s["ks"],
           "v_scale": s["vs"], "k": s["k"].view(torch.int8), "v": s["v"].view(torch.int8)}
    return out if lengths is None else dict(out, lengths=_ints(lengths))


def _exact_attend(s):
    case, q = s["case"], s["q"].double()
    group, size, page = case["Nq"] // case["Nk"], case["B"] // case["runs"], case["page"]
    out = torch.zeros_like(q)
    for b, (n, c) in enumerate(zip(_lengths(case), _counts(case))):
        n += _shared(case)[b // size]
        columns = s["pages"][b, :-(-n // page)].long()
        places, tokens = torch.arange(n - c, n, device="cuda")[:, None], torch.arange(n, device="cuda")[None]
        hidden = tokens > places
        if case["window"]:
            hidden = hidden | (tokens <= places - case["window"])
        for h in range(case["Nk"]):
            k, v = ((s[x][columns, h].double() * s[x + "s"][columns, h].double()[:, None, None]).flatten(0, 1)[:n]
                    for x in ("k", "v"))
            for g in range(h * group, (h + 1) * group):
                logits = q[b, g, :c] @ k.t().contiguous() / math.sqrt(case["d"])
                out[b, g, :c] = torch.softmax(logits.masked_fill(hidden, -math.inf), -1) @ v
    return out


def exact(case, seed):
    state = prepare(case, seed)
    return {"rotary": _exact_rotary, "step": _exact_pages, "compact": _exact_pages, "attend": _exact_attend}[case["op"]](state)
