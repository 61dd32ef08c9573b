"""The operators around natten1d that a language model trains and answers with, as cases that can be timed.

natten1d(is_causal=True) is the attention of a sequence that is there as a whole.  A case here is one
call of what stands beside it: rotary positions for q and k (``rotary``), tokens written into a paged
cache of 8 bits (``cache_append``), and attention over that cache for the tokens that come next
(``cache_attention``).  With ``own`` false the same is computed in elementary torch operations.

Fields of a case
    op        "rotary", "append" or "attend"
    dtype     of q, k and v: "bf16", "fp16" or "fp32"
    B, Nq, Nk, T, d   sequences, heads of q, heads of k and v, new tokens of each sequence, head_dim
    rotary:   R, channels that are rotated; interleaved; factor, how far the context is stretched
              beyond `first_context` positions (1: not at all); first, the first position;
              mode "train" (forward and backward) or "infer"; layout "plain" ([B, heads, T, d]) or
              "proj" (views of one projection [B, T, heads of q, k and v, d])
    append, attend:   cache, "int8" or "e4m3"; page, tokens of a page; longest, tokens of the longest
              sequence with its new ones (the shortest has about half); ragged, whether the
              sequences bring different numbers of new tokens
    attend:   window, how many tokens a query sees, its own the last (0: all)
"""
import math

import torch

own = False

_DTYPE = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_CACHE = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
_TOP = {"int8": 127.0, "e4m3": 448.0}
_TINY = 2.0 ** -126


def _rotary(**fields):
    return dict({"op": "rotary", "dtype": "bf16", "B": 1, "interleaved": False, "factor": 1.0,
                 "first": 0, "mode": "infer", "layout": "plain"}, **fields)


def _append(**fields):
    return dict({"op": "append", "dtype": "bf16", "ragged": False}, **fields)


def _attend(**fields):
    return dict({"op": "attend", "dtype": "bf16", "ragged": False, "window": 0}, **fields)


def listed():
    return [
        # one token of one sequence: the smallest call, only latency counts
        _rotary(name="rotary_token", Nq=16, Nk=16, T=1, d=128, R=128, first=5000),
        # a layer of a sequence model in training, the sizes of natten1d's own benchmark
        _rotary(name="rotary_train", mode="train", layout="proj", B=4, Nq=8, Nk=8, T=16384, d=64,
                R=64),
        # reading a long prompt far behind the trained context: part of the head, pairs side by
        # side, shared heads of k
        _rotary(name="rotary_far", dtype="fp16", B=2, Nq=16, Nk=4, T=8192, d=128, R=64,
                interleaved=True, factor=8.0, first=100000, layout="proj"),
        # one token for each of many sequences: pages that hold tokens already
        _append(name="append_token", cache="e4m3", B=32, Nk=8, T=1, d=128, page=16, longest=60),
        # prompts of different lengths read into the cache, behind what the last turn left there
        _append(name="append_prompt", cache="int8", B=2, Nk=16, T=8192, d=128, page=64,
                longest=8300, ragged=True),
        # one token with a sliding window, as natten1d's causal windows have it: a short stretch at
        # the end of a long cache, only latency counts
        _attend(name="attend_window", cache="int8", B=1, Nq=16, Nk=16, T=1, d=128, page=32,
                longest=8192, window=128),
        # serving: one token for each of many sequences of different lengths
        _attend(name="attend_batch", cache="e4m3", B=64, Nq=32, Nk=8, T=1, d=128, page=64,
                longest=8192),
        # one token of a single sequence that is very long
        _attend(name="attend_long", cache="int8", B=1, Nq=32, Nk=4, T=1, d=128, page=16,
                longest=131072),
        # a few drafted tokens of each sequence at once, narrow heads, half precision
        _attend(name="attend_draft", dtype="fp16", cache="e4m3", B=8, Nq=16, Nk=2, T=5, d=64,
                page=128, longest=16384, ragged=True),
        # the next piece of long prompts: the most arithmetic
        _attend(name="attend_chunk", cache="int8", B=2, Nq=16, Nk=4, T=2048, d=128, page=64,
                longest=16384),
        # odd sizes throughout, in float32: a head_dim between the powers of two, pages of 48
        _attend(name="attend_odd_fp32", dtype="fp32", cache="int8", B=3, Nq=15, Nk=5, T=7, d=80,
                page=48, longest=1031, ragged=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


# no drawn case has more of either than the largest listed ones, nor larger products in between
_MAX_BYTES, _MAX_FLOPS, _MAX_PAIRS = 8e8, 3.7e11, 6e8


def _fit(case):
    while (work(case)["bytes"] > _MAX_BYTES or work(case)["flops"] > _MAX_FLOPS
           or (case["op"] == "attend" and case["B"] * case["Nq"] * case["T"] * case["longest"] > _MAX_PAIRS)):
        if case["B"] > 1:
            case["B"] //= 2
        elif case["T"] > 1:
            case["T"] = (case["T"] + 1) // 2
        else:
            case["longest"] = (case["longest"] + 1) // 2
    return case


def draw(rng):
    """One more case: an operator, then sizes over its whole range."""
    op = rng.choice(("rotary", "append", "attend", "attend", "attend"))
    dtype = rng.choice(("bf16", "bf16", "bf16", "fp16", "fp16", "fp32"))
    Nk = rng.choice((1, 2, 3, 4, 8, 8, 16))
    if op == "rotary":
        d = rng.choice((32, 64, 80, 96, 128, 128, 192, 256))
        return _fit(_rotary(
            dtype=dtype, mode=rng.choice(("train", "infer")), layout=rng.choice(("plain", "proj")),
            B=_log_int(rng, 1, 64), Nq=Nk * rng.choice((1, 1, 2, 4, 7)), Nk=Nk,
            T=_log_int(rng, 1, 16384), d=d, R=rng.choice((d, d, d // 2, d // 4)),
            interleaved=rng.random() < 0.4, factor=rng.choice((1.0, 1.0, 4.0, 16.0)),
            first=rng.choice((0, rng.randint(1, 1000), _log_int(rng, 1000, 1000000)))))
    cache, page = rng.choice(("int8", "e4m3")), rng.choice((16, 32, 48, 64, 64, 128, 256))
    d, ragged = rng.choice((32, 64, 64, 80, 96, 128, 128, 128, 192, 256)), rng.random() < 0.5
    if op == "append":
        T = rng.choice((1, rng.randint(2, 16), _log_int(rng, 16, 8192)))
        return _fit(_append(dtype=dtype, cache=cache, B=_log_int(rng, 1, 64), Nk=Nk, T=T, d=d,
                            page=page, longest=2 * T + rng.randint(0, 300), ragged=ragged))
    T = rng.choice((1, 1, 1, rng.randint(2, 8), _log_int(rng, 8, 2048)))
    longest = max(2 * T, _log_int(rng, 1, 131072 if T < 9 else 16384))
    return _fit(_attend(dtype=dtype, cache=cache, B=_log_int(rng, 1, 64),
                        Nq=Nk * rng.choice((1, 2, 4, 4, 6, 8)), Nk=Nk, T=T, d=d, page=page,
                        longest=longest, ragged=ragged,
                        window=rng.choice((0, 0, _log_int(rng, 1, 8192)))))


def _counts(case):
    """New tokens of each sequence."""
    T = case["T"]
    return [T - (b * T // (2 * case["B"]) if case["ragged"] else 0) for b in range(case["B"])]


def _lengths(case):
    """Tokens of each sequence, the new ones included: from the longest down to about half."""
    return [max(c, case["longest"] - b * case["longest"] // (2 * case["B"]))
            for b, c in enumerate(_counts(case))]


def _frequencies(case):
    """One angle per position and pair of channels: base 10000, and for a longer context the slow
    pairs stretched by the factor, the fast ones kept, a ramp between (those that turn 1 to 32
    times in a context of 4096).  Also the factor that q and k are multiplied by then."""
    half = case["R"] // 2
    f = [10000.0 ** (-i / half) for i in range(half)]
    if case["factor"] == 1.0:
        return f, 1.0
    turns = [4096 * x / (2 * math.pi) for x in f]
    keep = [min(1.0, max(0.0, (t - 1.0) / 31.0)) for t in turns]
    return ([x * (w + (1.0 - w) / case["factor"]) for x, w in zip(f, keep)],
            0.1 * math.log(case["factor"]) + 1.0)


def _normal(gen, *shape, dtype=torch.float32):
    return torch.randn(shape, generator=gen, device="cuda", dtype=dtype)


def _qk(gen, case):
    B, Nq, Nk, T, d = (case[k] for k in ("B", "Nq", "Nk", "T", "d"))
    dtype = _DTYPE[case["dtype"]]
    if case["layout"] == "plain":
        return [_normal(gen, B, Nq, T, d, dtype=dtype), _normal(gen, B, Nk, T, d, dtype=dtype)]
    x = _normal(gen, B, T, Nq + 2 * Nk, d, dtype=dtype)
    return [x[:, :, :Nq].transpose(1, 2), x[:, :, Nq:Nq + Nk].transpose(1, 2)]


def _blocks(gen, case, count, low, high):
    """Pages as earlier calls left them: codes of normal values, scales for maxima of 4 sigma
    (times low to high, another for every block)."""
    shape = (count, case["Nk"], case["page"], case["d"])
    top = _TOP[case["cache"]]
    codes = (_normal(gen, *shape, dtype=torch.bfloat16) * (top / 4)).clamp(-top, top)
    if case["cache"] == "int8":
        codes = codes.round()
    scale = torch.rand(shape[:2], generator=gen, device="cuda") * (high - low) + low
    return codes.to(_CACHE[case["cache"]]), scale * (4 / top)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "rotary":
        train = case["mode"] == "train"
        frequencies, factor = _frequencies(case)
        first = case["first"] + torch.randint(0, 64, (case["B"], 1), generator=gen, device="cuda")
        return {"case": case, "qk": [x.requires_grad_(train) for x in _qk(gen, case)],
                "positions": first + torch.arange(case["T"], device="cuda"),
                "frequencies": torch.tensor(frequencies, device="cuda", dtype=torch.float64),
                "factor": factor, "grads": _qk(gen, case) if train else None}
    B, T, page, dtype = case["B"], case["T"], case["page"], _DTYPE[case["dtype"]]
    lengths, counts = _lengths(case), _counts(case)
    if case["op"] == "append":
        # the pages that new tokens go to, and one more, are there for every sequence
        columns = max(n - c for n, c in zip(lengths, counts)) // page + -(-T // page) + 1
        total = B * columns
    else:
        columns = -(-max(lengths) // page) + 1
        total = sum(-(-n // page) for n in lengths)
    order = torch.randperm(total, generator=gen, device="cuda").to(torch.int32)
    if case["op"] == "append":
        pages = order.view(B, columns)
    else:
        pages = torch.full((B, columns), -1, dtype=torch.int32, device="cuda")
        at = 0
        for b, n in enumerate(lengths):
            pages[b, :-(-n // page)] = order[at:at - (-n // page)]
            at += -(-n // page)
    state = {"case": case, "pages": pages,
             "lengths": torch.tensor(lengths, dtype=torch.int32, device="cuda"),
             "counts": torch.tensor(counts, dtype=torch.int32, device="cuda") if case["ragged"] else None}
    low, high = (0.4, 1.2) if case["op"] == "append" else (0.75, 1.25)
    for x in ("k", "v"):
        state[x + "_cache"], state[x + "_scale"] = _blocks(gen, case, total, low, high)
        if case["op"] == "append":
            # tokens in rows, heads side by side, as a projection leaves them
            state[x] = _normal(gen, B, T, case["Nk"], case["d"], dtype=dtype).transpose(1, 2)
    if case["op"] == "attend":
        # logits of a standard deviation of 2
        state["q"] = (_normal(gen, B, T, case["Nq"], case["d"]) * 2).to(dtype).transpose(1, 2)
    return state


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
    angle = (s["positions"].double()[..., None] * s["frequencies"])[:, None]
    cos, sin = (angle.cos() * s["factor"]).float(), (angle.sin() * s["factor"]).float()
    return (_turn(q, cos, sin, case["R"], case["interleaved"]),
            _turn(k, cos, sin, case["R"], case["interleaved"]))


def _codes(x, cache):
    top = _TOP[cache]
    x = x.clamp(-top, top)
    return (x.round() if cache == "int8" else x).to(_CACHE[cache])


def _plain_append_one(s, x, cache, scales):
    case, pages = s["case"], s["pages"].long()
    B, Nk, T, d, page, top = *(case[k] for k in ("B", "Nk", "T", "d", "page")), _TOP[case["cache"]]
    end = s["lengths"].long()
    start = end - (T if s["counts"] is None else s["counts"].long())
    columns = -(-T // page) + 1  # pages that the new tokens of one sequence may lie on
    column = (start // page)[:, None] + torch.arange(columns, device=x.device)
    at = pages.gather(1, column)
    place = column[..., None] * page + torch.arange(page, device=x.device)  # [B, columns, page]
    new = (place >= start[:, None, None]) & (place < end[:, None, None])
    old = (place < start[:, None, None])[:, :, None, :, None]
    row = (place - start[:, None, None]).clamp(0, T - 1).view(B, 1, -1, 1).expand(B, Nk, -1, d)
    val = x.gather(2, row).float().view(B, Nk, columns, page, d).transpose(1, 2)
    new = new[:, :, None, :, None]
    most = val.abs().masked_fill(~new, 0).amax((-2, -1))
    before = torch.where((column * page < start[:, None])[..., None], scales[at], torch.zeros_like(most))
    after = torch.maximum(before, most / top)
    after = torch.where(torch.isfinite(after), torch.where(after < _TINY, 0.0, after), math.nan)
    inverse = torch.where(after > 0, 1.0 / after, 0.0)
    was = cache[at]
    again = _codes(was.float() * (before * inverse)[..., None, None], case["cache"])
    fresh = _codes(val * inverse[..., None, None], case["cache"])
    changed = (old & (after > before)[..., None, None]).expand(was.shape)
    now = torch.where(new, fresh.float(), torch.where(changed, again.float(), was.float()))
    cache[at] = now.to(cache.dtype)
    scales[at] = torch.where(new.flatten(2).any(-1, keepdim=True), after, scales[at])


def _plain_attend(s):
    case, q = s["case"], s["q"]
    B, Nk, T, d, page = (case[k] for k in ("B", "Nk", "T", "d", "page"))
    at = s["pages"].long().clamp(min=0)

    def values(x):  # [B, Nk, tokens, d]
        v = s[x + "_cache"][at].float() * s[x + "_scale"][at][..., None, None]
        return v.transpose(1, 2).reshape(B, Nk, -1, d)

    k, v = values("k"), values("v")
    counts = torch.full_like(s["lengths"], T) if s["counts"] is None else s["counts"]
    t, j = torch.arange(T, device=q.device), torch.arange(k.shape[2], device=q.device)
    place = (s["lengths"] - counts)[:, None] + t
    seen = (j <= place[..., None]) & (t < counts[:, None])[..., None]
    if case["window"]:
        seen = seen & (j > place[..., None] - case["window"])
    x = q.float().reshape(B, Nk, -1, d) * d ** -0.5  # rows: the heads of a group, then tokens
    logits = (x @ k.transpose(-1, -2)).view(B, case["Nq"], T, -1).masked_fill(~seen[:, None], -math.inf)
    most = logits.amax(-1, keepdim=True)
    p = (logits - torch.where(most == -math.inf, 0.0, most)).exp()
    o = (p.view(B, Nk, -1, p.shape[-1]) @ v).view(B, case["Nq"], T, d)
    return (o / p.sum(-1, keepdim=True).clamp(min=1e-30)).to(q.dtype)


def _readable(s):
    """What a cache holds, as the values that its codes stand for."""
    dtype = _DTYPE[s["case"]["dtype"]]
    out = {x: (s[x + "_cache"].float() * s[x + "_scale"][..., None, None]).to(dtype) for x in ("k", "v")}
    return dict(out, k_scale=s["k_scale"], v_scale=s["v_scale"])


def run(state):
    """One call: (q, k) with positions, and in training their gradients; the cache with its new
    tokens; or what the new tokens read from it."""
    case = state["case"]
    if own:
        import e_natten_amd
    if case["op"] == "rotary":
        if own:
            out = e_natten_amd.rotary(*state["qk"], state["positions"], state["frequencies"],
                                      case["interleaved"], state["factor"])
        else:
            out = _plain_rotary(state)
        if case["mode"] == "infer":
            return tuple(out)
        return (*out, *torch.autograd.grad(out, state["qk"], state["grads"]))
    if case["op"] == "append":
        if own:
            e_natten_amd.cache_append(state["k"], state["v"], state["k_cache"], state["v_cache"],
                                      state["k_scale"], state["v_scale"], state["pages"],
                                      state["lengths"], state["counts"])
        else:
            _plain_append_one(state, state["k"], state["k_cache"], state["k_scale"])
            _plain_append_one(state, state["v"], state["v_cache"], state["v_scale"])
        return _readable(state)
    if own:
        return e_natten_amd.cache_attention(
            state["q"], state["k_cache"], state["v_cache"], state["k_scale"], state["v_scale"],
            state["pages"], state["lengths"], case["window"] or None, case["d"] ** -0.5,
            state["counts"])
    return _plain_attend(state)


def work(case):
    """Bytes and operations that the call cannot do without.  rotary: q and k read and written
    (twice in training), three operations a channel.  append: k and v read, a byte written for each
    value, and what the pass does besides, the pages read and written as values.  attend: the codes
    of the tokens that any query sees, with their scales, q and the output; two products of length
    d per (query, token) pair."""
    B, T, d = case["B"], case["T"], case["d"]
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "rotary":
        passes = 2 if case["mode"] == "train" else 1
        rows = B * T * (case["Nq"] + case["Nk"]) * passes
        return {"bytes": rows * d * size * 2 + B * T * 8 * passes, "flops": rows * case["R"] * 3}
    counts, lengths, Nk, page = _counts(case), _lengths(case), case["Nk"], case["page"]
    if case["op"] == "append":
        columns = max(n - c for n, c in zip(lengths, counts)) // page + -(-T // page) + 1
        held = B * columns * page * Nk * d
        values = 2 * sum(counts) * Nk * d
        return {"bytes": values * (size + 1) + 2 * held * (1 + size), "flops": 2 * values + 2 * held}
    tokens = pairs = 0
    for n, c in zip(lengths, counts):
        w = case["window"] or n
        tokens += min(n, w + c - 1)
        full = max(0, min(c, n - w + 1))  # queries with the whole window, the others one less each
        first = n - c + 1                 # tokens that the first of the others sees
        pairs += full * w + (c - full) * first + (c - full) * (c - full - 1) // 2
    rows = B * T * case["Nq"] * d * size * 2
    scales = 2 * 4 * Nk * sum(-(-n // page) for n in lengths) if not case["window"] else 0
    return {"bytes": 2 * tokens * Nk * d + scales + rows, "flops": 4 * pairs * case["Nq"] * d}


# --- the definitions, in 64 bits ---

def _exact_rotary(s):
    case, factor = s["case"], s["factor"]
    wheel = torch.polar(torch.full((), float(factor), device="cuda", dtype=torch.float64),
                        (s["positions"].double().unsqueeze(-1) * s["frequencies"]).unsqueeze(1))
    half = case["R"] // 2

    def turned(x, w):
        x = x.detach().double()
        if case["interleaved"]:
            z = torch.view_as_complex(x[..., :2 * half].unflatten(-1, (half, 2)).contiguous()) * w
            y = torch.view_as_real(z).flatten(-2)
        else:
            z = torch.complex(x[..., :half].contiguous(), x[..., half:2 * half].contiguous()) * w
            y = torch.cat((z.real, z.imag), -1)
        return torch.cat((y, x[..., 2 * half:]), -1)

    out = [turned(x, wheel) for x in s["qk"]]
    if s["grads"] is not None:
        out += [turned(g, wheel.conj()) for g in s["grads"]]
    return tuple(out)


def _exact_append(s):
    case, out = s["case"], {}
    page, top = case["page"], _TOP[case["cache"]]
    table = s["pages"].tolist()
    for x in ("k", "v"):
        codes, scales = s[x + "_cache"].double(), s[x + "_scale"].double()
        for b, (n, c) in enumerate(zip(_lengths(case), _counts(case))):
            for column in range((n - c) // page, (n - 1) // page + 1):
                at, lo, hi = table[b][column], max(n - c, column * page), min(n, (column + 1) * page)
                r = lo - column * page  # rows of the page that hold tokens already
                new = s[x][b, :, lo - (n - c):hi - (n - c)].double()
                most = new.abs().amax((1, 2)) / top
                scale = torch.maximum(scales[at], most) if r else most
                grown = scale > scales[at]
                for rows, values in ((slice(0, r), codes[at, :, :r] * scales[at][:, None, None]),
                                     (slice(r, r + hi - lo), new)):
                    y = (values / scale[:, None, None]).clamp(-top, top)
                    y = y.round() if case["cache"] == "int8" else y.float().to(torch.float8_e4m3fn).double()
                    keep = codes[at, :, rows] if rows.start == 0 and r else y
                    codes[at, :, rows] = torch.where((grown | (rows.start > 0 or not r))[:, None, None], y, keep)
                scales[at] = scale
        out[x], out[x + "_scale"] = codes * scales[..., None, None], scales
    return out


def _exact_attend(s):
    case, q = s["case"], s["q"].double()
    group, page = case["Nq"] // case["Nk"], case["page"]
    out = torch.zeros_like(q)
    for b, (n, c) in enumerate(zip(_lengths(case), _counts(case))):
        first = max(0, n - c - case["window"] + 1) if case["window"] else 0
        columns = s["pages"][b, first // page:-(-n // page)].long()
        skip = first - first // page * page
        places = torch.arange(n - c, n, device="cuda")[:, None]
        tokens = torch.arange(first, n, device="cuda")[None]
        hidden = tokens > places
        if case["window"]:
            hidden = hidden | (tokens <= places - case["window"])
        for h in range(case["Nk"]):
            k, v = ((s[x + "_cache"][columns, h].double() * s[x + "_scale"][columns, h].double()[:, None, None])
                    .flatten(0, 1)[skip:skip + n - first] for x in ("k", "v"))
            for g in range(h * group, (h + 1) * group):
                logits = q[b, g, :c] @ k.t().contiguous() / math.sqrt(case["d"])
                out[b, g, :c] = torch.softmax(logits.masked_fill(hidden, -math.inf), -1) @ v
    return out


def exact(case, seed):
    state = prepare(case, seed)
    return {"rotary": _exact_rotary, "append": _exact_append, "attend": _exact_attend}[case["op"]](state)
