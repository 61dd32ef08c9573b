"""Operators of sequences that grow, beside ``natten1d(..., is_causal=True)``, which takes a sequence
as a whole: rotary positions for q and k, a cache of 8 bits for the keys and values that were read
before, and the attention of the next tokens over it.

They have no counterpart in the reference, whose 1D operator (e_natten/triton.py:425-485) has neither
positions nor a cache.  A model trains with ``rotary`` in front of ``natten1d``, and answers with

    q, k = rotary(q, k, positions, frequencies)
    lengths += counts                     # the tokens of this step included
    cache_append(k, v, k_cache, v_cache, k_scale, v_scale, pages, lengths, counts)
    o = cache_attention(q, k_cache, v_cache, k_scale, v_scale, pages, lengths, kernel_size, scale, counts)

All tensors are ``[B, heads, T, d]``, strided views as everywhere in this package.  No call waits for
the GPU or reads a length on the host, so a step can be captured into a graph and replayed.

Like ``natten1d`` they run through the native torch binding where it is built (operators
``enatten::rotary``, ``enatten::cache_append``, ``enatten::cache_attention``), else through ctypes.
"""
from __future__ import annotations

import math

import torch
from torch.autograd import forward_ad

from . import _lib
from .ops import NATIVE_BINDING, _DTYPES, _check, _kernel_layout, _require_gpu, _stream_of

# the operators themselves: a call by overload costs two microseconds less than one by name
_OPS = tuple(getattr(torch.ops.enatten, name).default for name in ("rotary", "cache_append", "cache_attention")
             ) if NATIVE_BINDING else None
_CACHE_DTYPES = {torch.int8: _lib.I8, torch.float8_e4m3fn: _lib.E4M3}


def rotary_frequencies(rotary_dim, base=10000.0, scaling=None, factor=1.0, original_length=None,
                       fast_turns=32.0, slow_turns=1.0, device=None):
    """Angles per position of the ``rotary_dim / 2`` pairs, float64, and the factor for q and k:
    ``(frequencies, scale)`` for :func:`rotary`.

    Pair i turns by ``base ** (-2 i / rotary_dim)`` a position.  ``scaling`` stretches that for
    contexts ``factor`` times as long as the trained one:

    ``"linear"``  all angles divided by the factor (position interpolation, Chen et al. 2023)
    ``"ntk"``     the base times ``factor ** (rotary_dim / (rotary_dim - 2))``, which divides the
                  slowest pair's angle by the factor and leaves the fastest one's
    ``"yarn"``    by pair (Peng et al. 2023): pairs that make at least ``fast_turns`` turns in
                  ``original_length`` positions are kept, those with at most ``slow_turns`` divided by
                  the factor, a linear ramp between; q and k are multiplied by 0.1 ln(factor) + 1
    """
    if not isinstance(rotary_dim, int) or isinstance(rotary_dim, bool):
        raise TypeError("rotary_dim must be an int")
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError("rotary_dim must be even and >= 2, got %d" % rotary_dim)
    if scaling not in (None, "linear", "ntk", "yarn"):
        raise ValueError("scaling must be None, 'linear', 'ntk' or 'yarn', got %r" % (scaling,))
    if not base > 0 or not factor >= 1:
        raise ValueError("base must be positive and factor at least 1")
    scale = 1.0
    if scaling == "ntk":
        if rotary_dim == 2:
            raise ValueError("'ntk' scaling needs a rotary_dim of at least 4")
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    pairs = torch.arange(0, rotary_dim, 2, dtype=torch.float64)
    frequencies = torch.pow(torch.tensor(float(base), dtype=torch.float64), -pairs / rotary_dim)
    if scaling == "linear":
        frequencies = frequencies / factor
    if scaling == "yarn":
        if original_length is None or original_length < 1 or not fast_turns > slow_turns:
            raise ValueError("'yarn' scaling needs original_length, and fast_turns above slow_turns")
        turns = original_length * frequencies / (2 * math.pi)
        keep = ((turns - slow_turns) / (fast_turns - slow_turns)).clamp(0, 1)
        frequencies = frequencies * (keep + (1 - keep) / factor)
        scale = 0.1 * math.log(factor) + 1.0
    return frequencies.to(device), scale


def _tensors(**named):
    for name, t in named.items():
        if not isinstance(t, torch.Tensor):
            raise TypeError("%s must be a tensor" % name)


def _rows(name, x, dtypes):
    if x.dim() != 4:
        raise ValueError("expected [B, heads, T, head_dim] tensors, got %d-D %s" % (x.dim(), name))
    if x.dtype not in dtypes:
        raise ValueError("dtype %s is not supported (%s)"
                         % (x.dtype, ", ".join(str(d).replace("torch.", "") for d in dtypes)))
    if x.numel() == 0:
        raise ValueError("empty tensors are not supported")
    if max(x.shape) > 0x7fffffff or x.shape[1] > 1 << 20:
        raise ValueError("tensor too large")


# --- rotary ---

def _validate_rotary(q, k, positions, frequencies, axes) -> None:
    _rows("q", q, _DTYPES)
    if k is not None:
        if k.dim() != 4 or k.shape[1] < 1 or k.shape[::2] != q.shape[::2] or k.shape[3] != q.shape[3]:
            raise ValueError("q and k must differ in their heads only, got %s, %s" % (tuple(q.shape), tuple(k.shape)))
        if k.shape[1] > 1 << 20:
            raise ValueError("tensor too large")
        if k.dtype != q.dtype:
            raise ValueError("q and k must share a dtype")
        if k.device != q.device:
            raise ValueError("q and k must be on the same device")
    if positions.dtype not in (torch.int32, torch.int64):
        raise ValueError("positions must be int32 or int64, got %s" % positions.dtype)
    shape = tuple(positions.shape) if axes is None else tuple(positions.shape[1:])
    if shape not in ((q.shape[2],), (1, q.shape[2]), (q.shape[0], q.shape[2])) or positions.shape[0] < 1:
        raise ValueError("positions must have shape [T] or [B, T]%s, got %s"
                         % ("" if axes is None else " for every axis", tuple(positions.shape)))
    if frequencies.dtype not in (torch.float32, torch.float64):
        raise ValueError("frequencies must be float32 or float64, got %s" % frequencies.dtype)
    if frequencies.dim() != 1 or not 0 < 2 * frequencies.shape[0] <= q.shape[3]:
        raise ValueError("frequencies must be one for every rotated pair, at most head_dim / 2, got %s"
                         % (tuple(frequencies.shape),))
    if axes is not None and (axes.dtype != torch.int32 or axes.shape != frequencies.shape):
        raise ValueError("axes must be int32, one for every frequency, got %s %s" % (axes.dtype, tuple(axes.shape)))
    if axes is not None and positions.shape[0] > 0x7fffffff:
        raise ValueError("tensor too large")
    if q.shape[3] > 1024:
        raise ValueError("head_dim %d exceeds the supported maximum of 1024" % q.shape[3])
    if positions.device != q.device or frequencies.device != q.device:
        raise ValueError("positions and frequencies must be on the device of q")
    if axes is not None and axes.device != q.device:
        raise ValueError("axes must be on the device of q")


def _rotary_impl(q, k, positions, frequencies, interleaved: bool, scale: float, inverse: bool, axes=None):
    _validate_rotary(q, k, positions, frequencies, axes)
    _require_gpu(q, "rotary")
    lib = _lib.load()
    xs = [_kernel_layout(t) for t in ((q,) if k is None else (q, k))]
    if positions.stride(-1) != 1 and positions.shape[-1] != 1:
        positions = positions.contiguous()
    frequencies = frequencies.contiguous()
    with torch.cuda.device(q.device):
        ys = [_kernel_layout(torch.empty_like(x)) for x in xs]
        x2, y2 = (xs[1], ys[1]) if k is not None else (None, None)
        B, N, T, D = q.shape
        each = positions if axes is None else positions[0]
        data = (xs[0].data_ptr(), x2 if x2 is None else x2.data_ptr(), ys[0].data_ptr(),
                y2 if y2 is None else y2.data_ptr(), positions.data_ptr(), frequencies.data_ptr())
        sizes = (B, N, 0 if k is None else k.shape[1], T, D, 2 * frequencies.shape[0], _DTYPES[q.dtype],
                 _lib.I32 if positions.dtype == torch.int32 else _lib.I64, _DTYPES[frequencies.dtype],
                 int(interleaved), int(inverse), _lib.strides3(xs[0]), None if x2 is None else _lib.strides3(x2),
                 _lib.strides3(ys[0]), None if y2 is None else _lib.strides3(y2),
                 each.stride(0) if each.dim() == 2 and each.shape[0] > 1 else 0)
        if axes is None:
            _check(lib.enatten_rotary(*data, *sizes, float(scale), _stream_of(q)))
        else:
            axes = axes.contiguous()
            _check(lib.enatten_rotary_axes(*data, axes.data_ptr(), positions.shape[0], *sizes, positions.stride(0),
                                           float(scale), _stream_of(q)))
    return ys


class Rotary(torch.autograd.Function):
    """(q, k) -> (q', k') with k None or a tensor; the gradient is the turn the other way round."""

    @staticmethod
    def forward(ctx, q, k, positions, frequencies, interleaved, scale, inverse, axes=None):
        ctx.save_for_backward(positions, frequencies, axes)
        ctx.args = (interleaved, scale, inverse)
        ctx.set_materialize_grads(False)
        return tuple(_rotary_impl(q, k, positions, frequencies, interleaved, scale, inverse, axes))

    @staticmethod
    def backward(ctx, *grads):
        interleaved, scale, inverse = ctx.args
        there = [g for g in grads if g is not None]
        out = iter(())
        if there:
            positions, frequencies, axes = ctx.saved_tensors
            out = iter(Rotary.apply(there[0], there[1] if len(there) > 1 else None, positions, frequencies,
                                    interleaved, scale, not inverse, axes))
        dq, dk = (next(out) if i < len(grads) and grads[i] is not None else None for i in range(2))
        return dq, dk, None, None, None, None, None, None


def rotary_axes(rotary_dim, axes, order="blocks", device=None):
    """Which of a token's ``axes`` positions turns each of the ``rotary_dim / 2`` pairs, for :func:`rotary`.

    ``axes``  how many there are, or a list with the number of pairs of each.  With a number the pairs are
              shared out evenly, the first axes taking one more where that leaves a rest.
    ``order``  ``"blocks"``: the pairs of an axis are neighbours, in the order of the axes; ``"cyclic"``: the
              axes take turns, 0, 1, ..., 0, 1, ..., and one whose pairs are used up is passed over.
    """
    if not isinstance(rotary_dim, int) or isinstance(rotary_dim, bool):
        raise TypeError("rotary_dim must be an int")
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError("rotary_dim must be even and >= 2, got %d" % rotary_dim)
    if order not in ("blocks", "cyclic"):
        raise ValueError("order must be 'blocks' or 'cyclic', got %r" % (order,))
    pairs = rotary_dim // 2
    if isinstance(axes, int) and not isinstance(axes, bool):
        if axes < 1:
            raise ValueError("there must be one axis at least, got %d" % axes)
        sizes = [pairs // axes + (a < pairs % axes) for a in range(axes)]
    else:
        sizes = list(axes)
        if any(not isinstance(n, int) or isinstance(n, bool) for n in sizes):
            raise TypeError("axes must be an int, or the number of pairs of each axis")
    if not sizes or min(sizes) < 0 or sum(sizes) != pairs:
        raise ValueError("the axes' pairs must add up to %d, got %r" % (pairs, sizes))
    if order == "blocks":
        which = [a for a, n in enumerate(sizes) for _ in range(n)]
    else:
        which = [a for i in range(max(sizes)) for a, n in enumerate(sizes) if i < n]
    return torch.tensor(which, dtype=torch.int32, device=device)


def rotary(q, k, positions, frequencies, interleaved=False, scale=1.0, axes=None):
    """Rotary positions: ``(q', k')`` of ``q [B, heads, T, d]`` and ``k [B, heads_k, T, d]`` (or None,
    which comes back as None).  Differentiable in q and k, any number of times, by the backward pass
    (forward mode is refused).

    The first ``R = 2 len(frequencies)`` channels form pairs, ``(i, i + R / 2)``, or ``(2 i, 2 i + 1)``
    if ``interleaved``; the pair of the token at position p turns by the angle ``p * frequencies[i]``
    and is multiplied by ``scale``.  The other channels are copied.  ``positions`` are int32 or int64,
    ``[T]`` or ``[B, T]``, of any sign and size: angles are formed in double.  ``frequencies`` are
    float32 or float64, on the tensors' device (:func:`rotary_frequencies`); neither has a gradient.
    float32, bfloat16, float16 and float64; computed in float32 (float64 in double), rounded once.

    Tokens with several positions, as pixels of an image (row, column) or a video (time, row, column):
    ``axes``, int32, names for every pair the position that turns it (:func:`rotary_axes`), and
    ``positions`` are ``[axes, T]`` or ``[axes, B, T]``.  A pair whose axis is not there becomes NaN.
    Then q and k may also be images as :func:`natten2d` takes them, ``[B, heads, H, W, d]``, with
    positions ``[axes, H, W]`` or ``[axes, B, H, W]``; ones whose rows do not follow each other at an
    even distance are copied first.
    """
    _tensors(q=q, positions=positions, frequencies=frequencies)
    if k is not None:
        _tensors(k=k)
    if torch.is_grad_enabled() and frequencies.requires_grad:
        raise RuntimeError("frequencies have no gradient; call it on detached ones")
    call = _OPS[0] if NATIVE_BINDING else Rotary.apply
    if axes is None:
        out = call(q, k, positions, frequencies, bool(interleaved), float(scale), False)
        return out[0], out[1] if k is not None else None
    _tensors(axes=axes)
    image = q.shape[2:4] if q.dim() == 5 else None
    if image is not None:
        if k is not None and (k.dim() != 5 or k.shape[2:4] != image):
            raise ValueError("q and k must differ in their heads only, got %s, %s" % (tuple(q.shape), tuple(k.shape)))
        if positions.dim() < 3 or positions.shape[-2:] != image:
            raise ValueError("positions must have shape [H, W] or [B, H, W] for every axis, got %s"
                             % (tuple(positions.shape),))
        q, positions = q.flatten(2, 3), positions.flatten(-2, -1)
        k = None if k is None else k.flatten(2, 3)
    out = call(q, k, positions, frequencies, bool(interleaved), float(scale), False, axes)
    if image is not None:
        out = [x.unflatten(2, image) for x in out]
    return out[0], out[1] if k is not None else None


# --- the cache ---

def _validate_cache(name, x, k_cache, v_cache, k_scale, v_scale, pages, lengths, counts) -> None:
    _rows(name, x, (torch.float32, torch.bfloat16, torch.float16))
    B, _, _, D = x.shape
    if k_cache.dim() != 4 or k_cache.shape != v_cache.shape or k_cache.shape[3] != D or k_cache.numel() == 0:
        raise ValueError("k_cache and v_cache must be [pages, heads, tokens, %d], got %s, %s"
                         % (D, tuple(k_cache.shape), tuple(v_cache.shape)))
    if k_cache.dtype not in _CACHE_DTYPES or v_cache.dtype != k_cache.dtype:
        raise ValueError("k_cache and v_cache must both be int8 or float8_e4m3fn, got %s, %s"
                         % (k_cache.dtype, v_cache.dtype))
    if k_cache.stride(3) != 1 or v_cache.stride(3) != 1:
        raise ValueError("the cache needs unit stride on the channels")
    for t in (k_scale, v_scale):
        if t.shape != k_cache.shape[:2]:
            raise ValueError("k_scale and v_scale must be [pages, heads] = %s, got %s"
                             % (list(k_cache.shape[:2]), list(t.shape)))
        if t.dtype != torch.float32:
            raise ValueError("k_scale and v_scale must be float32")
    if pages.dim() != 2 or pages.shape[0] != B or pages.shape[1] < 1 or pages.dtype != torch.int32:
        raise ValueError("pages must be int32 [B, columns], got %s %s" % (pages.dtype, list(pages.shape)))
    if pages.shape[1] > 0x7fffffff or k_cache.shape[0] > 0x7fffffff or k_cache.shape[2] > 1024:
        raise ValueError("too many pages, or more than 1024 tokens in one")
    for what, t in (("lengths", lengths), ("counts", counts)):
        if t is not None and (t.dim() != 1 or t.shape[0] != B or t.dtype != torch.int32):
            raise ValueError("%s must be int32 [B], got %s %s" % (what, t.dtype, list(t.shape)))
    for t in (k_cache, v_cache, k_scale, v_scale, pages, lengths, counts):
        if t is not None and t.device != x.device:
            raise ValueError("all tensors must be on the same device")


def _no_gradient(what, *inputs) -> None:
    mode = torch.is_grad_enabled()
    if any(mode and t.requires_grad or forward_ad.unpack_dual(t).tangent is not None for t in inputs):
        raise RuntimeError("%s: a cache of 8 bits has no gradient; call it under torch.no_grad() or on "
                           "detached tensors, which have no tangent" % what)


def _page_rows(t):
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


def _aligned_rows(t):
    """Rows at multiples of 16 bytes (head dims are multiples of 16): nearly always the tensor itself."""
    pack = 16 // t.element_size()
    if t.stride(3) == 1 and not any(s % pack for s in t.stride()[:3]) and t.data_ptr() % 16 == 0:
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _is_distance(distance, axes):
    """Whether a distance is a sum of whole numbers of the strides; axes: (stride, size), longest stride first."""
    if not axes:
        return distance == 0
    (stride, size), rest = axes[0], axes[1:]
    inner = sum(s * (n - 1) for s, n in rest)
    if stride <= inner:
        return False
    near = distance // stride
    return any(abs(k) < size and abs(distance - k * stride) <= inner and _is_distance(distance - k * stride, rest)
               for k in (near, near + 1))


def _share_memory(a, b):
    """Whether two tensors of the same shape share an element.  Exact where both are dense, and where they have
    the same strides and these are nested (each longer than all that lies within it), as views of one pool have:
    the distance of the addresses is then a whole number of each stride, with two choices at most.  Other views
    whose ranges cross are let pass."""
    size = a.element_size()
    extents = [(1 + sum(s * (n - 1) for s, n in zip(t.stride(), t.shape))) * size for t in (a, b)]
    distance = b.data_ptr() - a.data_ptr()
    if distance >= extents[0] or -distance >= extents[1]:
        return False
    if all(torch.ops.aten.is_non_overlapping_and_dense(t) for t in (a, b)):
        return True
    axes = [(s, r, n) for s, r, n in zip(a.stride(), b.stride(), a.shape) if n > 1]
    if any(s != r for s, r, _ in axes):
        return False
    return distance % size == 0 and _is_distance(distance // size, sorted(((s, n) for s, _, n in axes), reverse=True))


def _append_impl(k, v, k_cache, v_cache, k_scale, v_scale, pages, lengths, counts) -> None:
    _validate_cache("k", k, k_cache, v_cache, k_scale, v_scale, pages, lengths, counts)
    if v.shape != k.shape:
        raise ValueError("k and v must have the same shape, got %s, %s" % (tuple(k.shape), tuple(v.shape)))
    if v.dtype != k.dtype or v.device != k.device:
        raise ValueError("k and v must share a dtype and a device")
    if k_cache.shape[1] != k.shape[1]:
        raise ValueError("k has %d heads, the cache %d" % (k.shape[1], k_cache.shape[1]))
    for t in (k_cache, v_cache, k_scale, v_scale):
        if any(n > 1 and s == 0 for n, s in zip(t.shape, t.stride())):
            raise RuntimeError("the cache must not share memory between its elements")
    if _share_memory(k_cache, v_cache) or _share_memory(k_scale, v_scale):
        raise ValueError("keys and values must not share a cache")
    _require_gpu(k, "cache_append")
    _no_gradient("cache_append", k, v, k_cache, v_cache, k_scale, v_scale)
    lib = _lib.load()
    k, v, pages = _kernel_layout(k), _kernel_layout(v), _page_rows(pages)
    lengths, counts = lengths.contiguous(), None if counts is None else counts.contiguous()
    B, N, T, D = k.shape
    with torch.cuda.device(k.device):
        _check(lib.enatten_cache_append(
            k.data_ptr(), v.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(),
            v_scale.data_ptr(), pages.data_ptr(), lengths.data_ptr(), None if counts is None else counts.data_ptr(),
            B, N, T, D, k_cache.shape[0], k_cache.shape[2], pages.shape[1], _DTYPES[k.dtype],
            _CACHE_DTYPES[k_cache.dtype], _lib.strides3(k), _lib.strides3(v), _lib.strides3(k_cache),
            _lib.strides3(v_cache), _lib.strides2(k_scale), _lib.strides2(v_scale), pages.stride(0),
            _stream_of(k)))
    for t in (k_cache, v_cache, k_scale, v_scale):
        if not t.is_inference():
            torch.autograd.graph.increment_version(t)


def _attention_impl(q, k_cache, v_cache, k_scale, v_scale, pages, lengths, counts, kernel_size: int, scale: float,
                    shared=None):
    _validate_cache("q", q, k_cache, v_cache, k_scale, v_scale, pages, lengths, counts)
    if q.shape[1] % k_cache.shape[1]:
        raise ValueError("%d heads are no multiple of the cache's %d" % (q.shape[1], k_cache.shape[1]))
    if shared is not None:
        if shared.dim() != 1 or shared.dtype != torch.int32 or shared.shape[0] < 1 or q.shape[0] % shared.shape[0]:
            raise ValueError("shared must be int32 [runs], runs a divisor of %d sequences, got %s %s"
                             % (q.shape[0], shared.dtype, list(shared.shape)))
        if shared.device != q.device:
            raise ValueError("all tensors must be on the same device")
    _require_gpu(q, "cache_attention")
    _no_gradient("cache_attention", q, k_cache, v_cache, k_scale, v_scale)
    lib = _lib.load()
    rows, pages = _kernel_layout(q), _page_rows(pages)
    q = _aligned_rows(rows)
    lengths, counts = lengths.contiguous(), None if counts is None else counts.contiguous()
    B, N, T, D = q.shape
    heads, page, columns, window = k_cache.shape[1], k_cache.shape[2], pages.shape[1], min(kernel_size, 0x7fffffff)
    with torch.cuda.device(q.device):
        o = _aligned_rows(_kernel_layout(torch.empty_like(rows)))
        sizes = (B, N, heads, T, D, page, columns, window, _DTYPES[q.dtype])
        data = (q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(),
                pages.data_ptr(), lengths.data_ptr(), None if counts is None else counts.data_ptr())
        rest = (B, N, heads, T, D, k_cache.shape[0], page, columns, window,
                _DTYPES[q.dtype], _CACHE_DTYPES[k_cache.dtype], _lib.strides3(q), _lib.strides3(o),
                _lib.strides3(k_cache), _lib.strides3(v_cache), _lib.strides2(k_scale), _lib.strides2(v_scale),
                pages.stride(0), float(scale), _stream_of(q))

        def run(entry, need, *extra):
            ws = torch.empty(need, dtype=torch.uint8, device=q.device)
            return entry(*data, *extra, o.data_ptr(), ws.data_ptr() if need else None, *rest)

        rc = _lib.EUNSUPPORTED
        if shared is not None:
            shared = shared.contiguous()
            rc = run(lib.enatten_cache_attention_shared,
                     lib.enatten_cache_attention_shared_workspace_bytes(*sizes, shared.shape[0]), shared.data_ptr(), shared.shape[0])
        if rc == _lib.EUNSUPPORTED:   # (too many rows for sharing, and nothing queued: every sequence reads for itself)
            rc = run(lib.enatten_cache_attention, lib.enatten_cache_attention_workspace_bytes(*sizes))
        _check(rc)
    return o


def cache_append(k, v, k_cache, v_cache, k_scale, v_scale, pages, lengths, counts=None):
    """Write the new tokens ``k, v [B, heads, T, d]`` of each sequence into a paged cache of 8 bits,
    in place.

    ``k_cache, v_cache``  ``[pages, heads, page, d]``, int8 or float8_e4m3fn; d a multiple of 16 up to
        256, page a multiple of 16 up to 1024.  Strided views with unit stride on d, such as one
        layer of a larger pool, if strides and address are multiples of 16.
    ``k_scale, v_scale``  float32 ``[pages, heads]``, not negative: a code stands for code * scale of
        its block (page, head).
    ``pages``  int32 ``[B, columns]``: token j of sequence b is row j % page of page pages[b, j // page].
        A page that tokens are written to belongs to one sequence.
    ``lengths``  int32 ``[B]``: tokens of each sequence, the new ones included.
    ``counts``  int32 ``[B]``: how many of T each sequence brings (its first rows of k and v); None: T.

    A block's scale is the largest magnitude over 127 (448 for float8) of what it holds.  It grows with
    new tokens, and the codes of older ones are rounded anew then; it does not shrink, but a page that
    starts with a new token starts with a new scale.  A value that is not finite makes its block NaN.
    A sequence whose numbers do not fit together (a count outside 0 .. T or above the length, a length
    beyond the columns) is left out, as are pages outside the cache; :func:`cache_attention` returns
    NaN for both.  No gradient.
    """
    _tensors(k=k, v=v, k_cache=k_cache, v_cache=v_cache, k_scale=k_scale, v_scale=v_scale, pages=pages,
             lengths=lengths)
    if counts is not None:
        _tensors(counts=counts)
    call = _OPS[1] if NATIVE_BINDING else _append_impl
    call(k, v, k_cache, v_cache, k_scale, v_scale, pages, lengths, counts)


def cache_attention(q, k_cache, v_cache, k_scale, v_scale, pages, lengths, kernel_size=None, scale=1.0,
                    counts=None, shared=None):
    """Attention of the last tokens of each sequence over its cache: ``q [B, heads, T, d] -> o`` of the
    same shape, what ``natten1d(..., is_causal=True)`` gives for these tokens of a whole sequence.

    The cache, ``pages``, ``lengths`` and ``counts`` are those of :func:`cache_append`, whose call for
    the same tokens comes first.  Query t stands at position p = lengths[b] - counts[b] + t and sees the
    last ``kernel_size`` tokens up to and including its own, or all of them (None).  Logits are
    q.k * scale.  ``heads`` is a multiple of the cache's heads; head h reads head h // (heads / cache
    heads).  Rows from counts[b] on are 0.  float32, bfloat16 and float16.  No gradient.

    The products are those of float16 terms, two each for float32, with sums and statistics in float32.
    Weighted values are summed up before the division: one times 256 times the number of tokens has to
    stay within float32.  A call's work is cut by the lengths of all its sequences, so that another
    sequence's length may change where a result is rounded; the same call gives the same bits.  A token
    whose logit is below -6e14 counts for nothing.  A ``scale`` that is not finite gives NaN.

    A float8 cache that :func:`cache_append` wrote holds finite codes only.  The two codes that are no
    numbers, written there by other means, read as +-480 or as NaN by the queries that see them, by the
    sizes of the call; queries that do not see them never notice.

    ``shared``, int32 ``[runs]``, is for sequences that continue one prompt: they come in that many runs of
    neighbours, B / runs each, and those of run r have their first ``shared[r]`` tokens on the same pages
    (:func:`cache_fork`).  These are read once for all rows of the run; whole pages of them count.  A sequence
    whose new tokens start before their end is computed by itself, and numbers below 1 share nothing, so
    that the result is the same but for its rounding.  Where that would not pay, by the sizes of the call (few
    codes in all that its columns could name or its window holds, many new tokens), every sequence reads for itself.
    These sizes are the table's, as lengths are not known here: with a table much wider than the sequences are long,
    a call takes some 20 us more than without ``shared``.  So pass the columns that the longest sequence needs,
    ``pages[:, :n]``, or leave ``shared`` out.  Where only the device knows, numbers of 0 take most of that back: 4 to
    8 us are left for single tokens.  Reading together pays from 16 MB of codes that the sequences have in all, shared
    ones counted for each of them, with up to 16 rows in a run (new tokens times heads of q for one of the cache),
    160 MB beyond.
    """
    _tensors(q=q, k_cache=k_cache, v_cache=v_cache, k_scale=k_scale, v_scale=v_scale, pages=pages,
             lengths=lengths)
    if counts is not None:
        _tensors(counts=counts)
    if shared is not None:
        _tensors(shared=shared)
    if kernel_size is None:
        kernel_size = 0
    elif not isinstance(kernel_size, int) or isinstance(kernel_size, bool):
        raise TypeError("kernel_size must be an int or None")
    elif kernel_size < 1:
        raise ValueError("kernel_size must be >= 1, got %d" % kernel_size)
    call = _OPS[2] if NATIVE_BINDING else _attention_impl
    if shared is None:
        return call(q, k_cache, v_cache, k_scale, v_scale, pages, lengths, counts, kernel_size, float(scale))
    return call(q, k_cache, v_cache, k_scale, v_scale, pages, lengths, counts, kernel_size, float(scale), shared)
