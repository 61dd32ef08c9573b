"""Plain 64-bit forms of the operators of growing sequences, and inputs for their tests."""
from __future__ import annotations

import math

import torch

TOP = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}


def half_step(dtype):
    """A rounding is off by at most half a step: eps / 2 of the value."""
    return torch.finfo(dtype).eps / 2


def rotary_ref(x, positions, frequencies, interleaved=False, scale=1.0, inverse=False):
    """(y, |x1| + |x2| of every channel's pair) in float64 on the CPU."""
    x = x.detach().cpu().double()
    angle = positions.cpu().double().reshape(-1, 1, x.shape[2], 1) * frequencies.cpu().double()
    w = torch.polar(torch.full_like(angle, float(scale)), -angle if inverse else angle)
    half = frequencies.numel()
    part, rest = x[..., :2 * half], x[..., 2 * half:]
    a, b = (part[..., 0::2], part[..., 1::2]) if interleaved else (part[..., :half], part[..., half:])
    z = torch.complex(a, b) * w
    size = (a.abs() + b.abs()) * abs(scale)

    def join(u, v):
        return torch.stack((u, v), -1).flatten(-2) if interleaved else torch.cat((u, v), -1)

    return torch.cat((join(z.real, z.imag), rest), -1), torch.cat((join(size, size), torch.zeros_like(rest)), -1)


class Cache:
    """A pool of pages on the CPU, of which every sequence has some in a random order.  Pages that no
    sequence has, and rows behind a sequence's end, hold codes and scales that must not matter."""

    def __init__(self, lengths, heads, page, d, dtype, seed=0, spare=3, columns=None, extra_columns=2,
                 scale_spread=(0.2, 2.0)):
        g = torch.Generator().manual_seed(seed)
        need = [-(-n // page) for n in lengths]
        columns = columns or max(max(need), 1) + extra_columns
        total = sum(need) + spare
        self.page, self.heads, self.d, self.dtype, self.lengths = page, heads, d, dtype, list(lengths)
        order = torch.randperm(total, generator=g)
        # entries behind the last page: not read, whatever they are
        self.pages = torch.full((len(lengths), columns), -1, dtype=torch.int32)
        self.pages[:, 1::2] = 2 ** 31 - 1
        self.codes, self.scales = [], []
        for _ in range(2):
            x = torch.randn((total, heads, page, d), generator=g) * (TOP[dtype] / 4)
            x = x.clamp(-TOP[dtype], TOP[dtype])
            raw = (x.round() if dtype == torch.int8 else x).to(dtype).view(torch.uint8)
            lo, hi = scale_spread
            z = torch.exp(torch.rand((total, heads), generator=g) * math.log(hi / lo) + math.log(lo)) * (4 / TOP[dtype])
            self.codes.append(raw)
            self.scales.append(z)
        owned = torch.zeros((total, page), dtype=torch.bool)
        at = 0
        for b, n in enumerate(lengths):
            mine = order[at:at + need[b]]
            at += need[b]
            self.pages[b, :need[b]] = mine.to(torch.int32)
            for i, p in enumerate(mine.tolist()):
                owned[p, :min(page, n - i * page)] = True
        for raw, z in zip(self.codes, self.scales):
            raw.masked_fill_(~owned[:, None, :, None], 0x7f)   # NaN as E4M3
            z.masked_fill_(~owned.any(-1)[:, None], math.nan)
        self.owned = owned

    def on(self, device):
        """(k_cache, v_cache, k_scale, v_scale, pages) there"""
        k, v = (c.to(device).view(self.dtype) for c in self.codes)
        return k, v, self.scales[0].to(device), self.scales[1].to(device), self.pages.to(device)

    def values(self, which, b, n=None):
        """[heads, tokens, d] in float64: what the first n tokens of sequence b stand for."""
        n = self.lengths[b] if n is None else n
        if n == 0:
            return torch.zeros((self.heads, 0, self.d), dtype=torch.float64)
        p = self.pages[b, :-(-n // self.page)].long()
        v = self.codes[which][p].view(self.dtype).float().double() * self.scales[which][p].double()[..., None, None]
        return v.transpose(0, 1).reshape(self.heads, -1, self.d)[:, :n]


def attention_ref(q, cache, counts=None, kernel_size=None, scale=1.0):
    """(o, bound) in float64 on the CPU.  The bound, for results in q's type before their rounding:
    probabilities go into the second product with 11 bits (float32: 22), so A = sum p |v| times 2^-11
    (2^-21, products and sums in float32 included); the logits are sums of products in float32, off by
    at most 2^-21 of L = scale sum |q| |k|, and an error of a logit by e moves the result by at most
    2 e A.  Probabilities under 2^-28 of the largest lose up to 2^-38 of the largest |v| each."""
    single = q.dtype == torch.float32
    q = q.detach().cpu().double()
    B, N, T, d = q.shape
    group = N // cache.heads
    o, bound = torch.zeros_like(q), torch.zeros_like(q)
    few = 2.0 ** (-21 if single else -11)
    for b, n in enumerate(cache.lengths):
        c = T if counts is None else int(counts[b])
        if c == 0 or n == 0:
            continue
        k, v = cache.values(0, b), cache.values(1, b)
        place = torch.arange(n - c, n)[:, None]
        token = torch.arange(n)[None]
        hidden = token > place
        if kernel_size is not None:
            hidden = hidden | (token <= place - kernel_size)
        for h in range(N):
            kh, vh = k[h // group], v[h // group]
            s = (q[b, h, :c] @ kh.t()) * scale
            size = (q[b, h, :c].abs() @ kh.abs().t() * abs(scale)).masked_fill(hidden, 0).amax(-1, keepdim=True)
            p = torch.softmax(s.masked_fill(hidden, -math.inf), -1)
            o[b, h, :c] = p @ vh
            A = p @ vh.abs()
            bound[b, h, :c] = A * (few + 2 * 2.0 ** -21 * size) + n * 2.0 ** -38 * vh.abs().max()
    return o, bound


def append_ref(cache, k, v, counts=None):
    """The append's definition in float32 on the CPU, step for step: (codes, scales) of k and v, as the
    cache holds them after `counts` of the T rows of k and v became its sequences' last tokens."""
    B, heads, T, d = k.shape
    top, page = TOP[cache.dtype], cache.page

    def code(y):
        y = y.clamp(-top, top)
        return (y.round() if cache.dtype == torch.int8 else y).to(cache.dtype).view(torch.uint8)

    out = []
    for which, x in enumerate((k, v)):
        codes, scales = cache.codes[which].clone(), cache.scales[which].clone()
        for b, n in enumerate(cache.lengths):
            c = T if counts is None else int(counts[b])
            start = n - c
            for col in range(start // page, -(-n // page)):
                lo, hi = max(start, col * page), min(n, (col + 1) * page)
                if lo >= hi:
                    continue
                at, old = int(cache.pages[b, col]), lo - col * page
                for h in range(heads):
                    new = x[b, h, lo - start:hi - start].float()
                    before = scales[at, h] if old else torch.zeros(())
                    most = new.abs().max()
                    if not torch.isfinite(new).all() or not torch.isfinite(before):
                        after, inverse = torch.tensor(math.nan), torch.zeros(())
                    else:
                        after = torch.maximum(before, most / torch.tensor(top))
                        inverse = torch.ones(()) / after
                        if after < 2.0 ** -126:
                            after, inverse = torch.zeros(()), torch.zeros(())
                    if old and after > before:
                        was = codes[at, h, :old].view(cache.dtype).float()
                        codes[at, h, :old] = code(was * (before * inverse))
                    fresh = code(new * inverse) if inverse > 0 else torch.zeros_like(new, dtype=torch.uint8)
                    codes[at, h, old:old + hi - lo] = fresh
                    scales[at, h] = after
        out.append((codes, scales))
    return out
