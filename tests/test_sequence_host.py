"""Host side of the operators of growing sequences, without a GPU: frequencies against their formulas,
what the entry points refuse (in Python, in the native binding and at the C boundary), shapes without data."""
import ctypes
import math

import pytest
import torch

from _util import ensure_built

BF16, F16, F32, F64 = torch.bfloat16, torch.float16, torch.float32, torch.float64
I8, E4M3 = torch.int8, torch.float8_e4m3fn


# --- frequencies ---

@pytest.mark.parametrize("dim,base", [(2, 10000.0), (64, 10000.0), (128, 500000.0), (6, 10.0)])
def test_frequencies(dim, base):
    ensure_built()
    from e_natten_amd import rotary_frequencies
    plain = [base ** (-2 * i / dim) for i in range(dim // 2)]
    f, scale = rotary_frequencies(dim, base)
    assert f.dtype == F64 and scale == 1.0
    # a power in double is off by a few units of its last place
    near = lambda x, y: all(abs(a - b) <= 2.0 ** -48 * abs(b) for a, b in zip(x.tolist(), y)) and len(x) == len(y)
    assert near(f, plain)
    f, scale = rotary_frequencies(dim, base, "linear", 4.0)
    assert near(f, [x / 4 for x in plain]) and scale == 1.0
    if dim > 2:
        f, scale = rotary_frequencies(dim, base, "ntk", 4.0)
        wide = base * 4.0 ** (dim / (dim - 2))
        assert near(f, [wide ** (-2 * i / dim) for i in range(dim // 2)]) and scale == 1.0
        assert abs(f[-1].item() / (plain[-1] / 4) - 1) < 2.0 ** -45 and f[0] == 1.0
    f, scale = rotary_frequencies(dim, base, "yarn", 8.0, original_length=2048, fast_turns=32.0, slow_turns=1.0)
    want = []
    for x in plain:
        turns = 2048 * x / (2 * math.pi)
        keep = min(max((turns - 1.0) / 31.0, 0.0), 1.0)
        want.append(x * keep + x / 8 * (1 - keep))
    assert near(f, want) and scale == 0.1 * math.log(8.0) + 1.0
    assert torch.equal(rotary_frequencies(dim, base, "linear", 1.0)[0], rotary_frequencies(dim, base)[0])


@pytest.mark.parametrize("error,args", [
    (TypeError, dict(rotary_dim=8.0)), (TypeError, dict(rotary_dim=True)), (ValueError, dict(rotary_dim=7)),
    (ValueError, dict(rotary_dim=0)), (ValueError, dict(rotary_dim=-2)), (ValueError, dict(rotary_dim=8, base=0.0)),
    (ValueError, dict(rotary_dim=8, base=math.nan)), (ValueError, dict(rotary_dim=8, factor=0.5)),
    (ValueError, dict(rotary_dim=8, scaling="other")), (ValueError, dict(rotary_dim=2, scaling="ntk", factor=2.0)),
    (ValueError, dict(rotary_dim=8, scaling="yarn", factor=2.0)),
    (ValueError, dict(rotary_dim=8, scaling="yarn", factor=2.0, original_length=0)),
    (ValueError, dict(rotary_dim=8, scaling="yarn", factor=2.0, original_length=64, fast_turns=1.0, slow_turns=1.0)),
])
def test_frequencies_refuse(error, args):
    from e_natten_amd import rotary_frequencies
    with pytest.raises(error):
        rotary_frequencies(**args)


# --- refusals, through both host sides ---

def _impls(name):
    """(the public function, the same call through ctypes)"""
    import e_natten_amd as E
    from e_natten_amd import sequence as S
    if name == "rotary":
        ctyped = lambda q, k, p, f, interleaved=False, scale=1.0: S.Rotary.apply(q, k, p, f, interleaved, scale, False)
    elif name == "cache_append":
        def ctyped(*a, counts=None):
            S._append_impl(*a, counts)
    else:
        def ctyped(*a, kernel_size=None, counts=None):
            return S._attention_impl(*a, counts, kernel_size or 0, 1.0)
    return getattr(E, name), ctyped


def _rotary_args(device="cpu", **change):
    a = dict(q=torch.zeros(2, 4, 5, 16, device=device), k=torch.zeros(2, 2, 5, 16, device=device),
             positions=torch.arange(5, device=device), frequencies=torch.ones(8, dtype=F64, device=device))
    a.update(change)
    return a["q"], a["k"], a["positions"], a["frequencies"]


def _z(*shape, dtype=F32):
    return torch.zeros(shape, dtype=dtype)


@pytest.mark.parametrize("change,text", [
    (dict(q=_z(2, 4, 16)), "4-D|heads, T"), (dict(q=_z(2, 4, 5, 16, dtype=torch.int32)), "not supported"),
    (dict(q=_z(2, 0, 5, 16)), "empty"), (dict(k=_z(2, 2, 6, 16)), "differ in their heads"),
    (dict(k=_z(2, 0, 5, 16)), "differ in their heads"), (dict(k=_z(1, 2, 5, 16)), "differ in their heads"),
    (dict(k=_z(2, 2, 5, 16, dtype=BF16)), "share a dtype"), (dict(positions=_z(5)), "int32 or int64"),
    (dict(positions=torch.arange(4)), "shape"), (dict(positions=torch.arange(15).view(3, 5)), "shape"),
    (dict(positions=torch.arange(5).view(1, 1, 5)), "shape"), (dict(frequencies=_z(8, dtype=F16)), "float32 or float64"),
    (dict(frequencies=_z(9)), "at most head_dim"), (dict(frequencies=_z(0)), "at most head_dim"),
    (dict(frequencies=_z(8, 1)), "at most head_dim"),
    (dict(q=_z(2, 4, 5, 1026), k=None), "1024"),
    (dict(positions=torch.arange(5, device="meta")), "device"), (dict(frequencies=torch.ones(8, device="meta")), "device"),
    (dict(k=torch.zeros(2, 2, 5, 16, device="meta")), "same device"),
    (dict(q=_z(1, 1, 1, 16).expand(1, 1, 1 << 32, 16), k=None, positions=torch.zeros(1, dtype=torch.int64).expand(1 << 32)),
     "too large"),
    (dict(q=_z(1, 1, 5, 16).expand(1, 1 << 21, 5, 16), k=None), "too large"),
    (dict(), "GPU"),
])
def test_rotary_refuses(change, text):
    ensure_built()
    for call in _impls("rotary"):
        with pytest.raises((ValueError, RuntimeError), match=text):
            call(*_rotary_args(**change))


def test_rotary_refuses_what_is_no_tensor_and_frequencies_that_want_a_gradient():
    ensure_built()
    from e_natten_amd import rotary
    for change in (dict(q=[1.0]), dict(k=3), dict(positions=[0, 1, 2, 3, 4]), dict(frequencies=None)):
        with pytest.raises(TypeError, match="tensor"):
            rotary(*_rotary_args(**change))
    for q in (_z(2, 4, 5, 16), _z(2, 4, 5, 16).requires_grad_(True)):
        with pytest.raises(RuntimeError, match="no gradient"):
            rotary(*_rotary_args(q=q, frequencies=torch.ones(8, dtype=F64, requires_grad=True)))


def _cache_args(name, device="cpu", T=3, d=32, page=16, heads=2, N=4, dtype=BF16, cache=I8, **change):
    make = lambda *s, dtype: torch.zeros(s, dtype=dtype, device=device)
    a = dict(q=make(2, N, T, d, dtype=dtype), k=make(2, heads, T, d, dtype=dtype), v=make(2, heads, T, d, dtype=dtype),
             k_cache=make(6, heads, page, d, dtype=cache), v_cache=make(6, heads, page, d, dtype=cache),
             k_scale=make(6, heads, dtype=F32), v_scale=make(6, heads, dtype=F32),
             pages=make(2, 3, dtype=torch.int32), lengths=make(2, dtype=torch.int32))
    extra = {n: change.pop(n) for n in ("counts", "kernel_size") if n in change}
    a.update(change)
    rows = (a["q"],) if name == "cache_attention" else (a["k"], a["v"])
    return (*rows, a["k_cache"], a["v_cache"], a["k_scale"], a["v_scale"], a["pages"], a["lengths"]), extra


_I32 = torch.int32
_SHARED = _z(6, 2, 16, 32, dtype=I8)


@pytest.mark.parametrize("change,text", [
    (dict(q=_z(2, 4, 32, dtype=BF16), k=_z(2, 2, 32, dtype=BF16)), "heads, T"),
    (dict(dtype=F64), "not supported"), (dict(T=0), "empty"),
    (dict(k_cache=_z(6, 2, 16, 16, dtype=I8)), "must be \\[pages"),
    (dict(k_cache=_z(6, 2, 16, dtype=I8)), "must be \\[pages"),
    (dict(v_cache=_z(5, 2, 16, 32, dtype=I8)), "must be \\[pages"),
    (dict(cache=torch.uint8), "int8 or float8"), (dict(v_cache=_z(6, 2, 16, 32, dtype=E4M3)), "int8 or float8"),
    (dict(k_cache=_z(6, 2, 32, 16, dtype=I8).transpose(2, 3)), "unit stride"),
    (dict(v_scale=_z(6, 3)), "must be \\[pages, heads\\]"), (dict(k_scale=_z(6, 2, dtype=F16)), "float32"),
    (dict(pages=_z(2, 3, dtype=torch.int64)), "int32"), (dict(pages=_z(3, 3, dtype=_I32)), "int32"),
    (dict(pages=_z(2, 0, dtype=_I32)), "int32"), (dict(lengths=_z(3, dtype=_I32)), "int32"),
    (dict(lengths=_z(2, dtype=torch.int64)), "int32"), (dict(counts=_z(2)), "int32"), (dict(counts=_z(1, dtype=_I32)), "int32"),
    (dict(page=1040), "1024"), (dict(lengths=torch.zeros(2, dtype=_I32, device="meta")), "same device"),
    (dict(counts=torch.zeros(2, dtype=_I32, device="meta")), "same device"), (dict(), "GPU"),
    (dict(heads=3, N=3, k_cache=_z(6, 2, 16, 32, dtype=I8), v_cache=_z(6, 2, 16, 32, dtype=I8), k_scale=_z(6, 2),
          v_scale=_z(6, 2)), "heads"),
])
def test_cache_refuses(change, text):
    ensure_built()
    for name in ("cache_append", "cache_attention"):
        args, extra = _cache_args(name, **change)
        for call in _impls(name):
            with pytest.raises((ValueError, RuntimeError), match=text):
                call(*args, **extra)


@pytest.mark.parametrize("change,text", [
    (dict(v=_z(2, 2, 4, 32, dtype=BF16)), "same shape"), (dict(v=_z(2, 2, 3, 32, dtype=F16)), "share a dtype"),
    (dict(v_cache=_z(1, 2, 16, 32, dtype=I8).expand(6, 2, 16, 32)), "memory"),
    (dict(k_scale=_z(6, 1).expand(6, 2)), "memory"),
    (dict(k_cache=_SHARED, v_cache=_SHARED), "must not share"),
])
def test_append_refuses(change, text):
    ensure_built()
    args, extra = _cache_args("cache_append", **change)
    for call in _impls("cache_append"):
        with pytest.raises((ValueError, RuntimeError), match=text):
            call(*args, **extra)


def _pool(*shape, dtype=I8):
    return torch.zeros(shape, dtype=dtype)


_LAYERS = _pool(9, 3, 2, 16, 32)            # pages, layers, heads, tokens, channels
_PAIRS = _pool(6, 2, 2, 16, 32)             # pages, keys and values, heads, ...
_TOKENS = _pool(6, 16, 2, 2, 32)            # pages, tokens, keys and values, heads, ...
_Z = _pool(6, 2, 2, dtype=F32)


@pytest.mark.parametrize("shared,change", [
    (True, dict(k_cache=_LAYERS[:6, 0], v_cache=_LAYERS[3:, 0])),              # some pages of both
    (False, dict(k_cache=_LAYERS[:6, 0], v_cache=_LAYERS[3:, 1])),             # those of two layers
    (True, dict(k_cache=_LAYERS[3:, 1], v_cache=_LAYERS[:6, 1])),
    (True, dict(k_cache=_pool(9, 2, 16, 32)[:6], v_cache=None)),               # (v_cache: the same pool, from page 3)
    (False, dict(k_cache=_PAIRS[:, 0], v_cache=_PAIRS[:, 1])),
    (True, dict(k_cache=_pool(6, 3, 16, 32)[:, :2], v_cache=1)),               # (... from head 1)
    (False, dict(k_cache=_TOKENS[:, :, 0].transpose(1, 2), v_cache=_TOKENS[:, :, 1].transpose(1, 2))),
    (True, dict(k_cache=_TOKENS[:, :, 0].transpose(1, 2), v_cache=_TOKENS[:, :, 0].transpose(1, 2))),
    (False, dict(k_cache=_pool(6, 2, 16, 64)[..., :32], v_cache=32)),          # (... from channel 32)
    (True, dict(k_cache=_pool(6, 2, 16, 64)[..., :32], v_cache=16)),
    (True, dict(k_scale=_Z[:, 0], v_scale=_Z[:, 0])),
    (False, dict(k_scale=_Z[:, 0], v_scale=_Z[:, 1])),
    (True, dict(k_scale=_Z.view(12, 2)[:6], v_scale=_Z.view(12, 2)[5:11])),
    (False, dict(k_scale=_Z.view(12, 2)[:6], v_scale=_Z.view(12, 2)[6:])),
    (False, dict(k_scale=_Z[..., 0], v_scale=_Z[..., 1])),
])
def test_append_refuses_keys_and_values_that_share_some_memory(shared, change):
    """Not only the same tensor twice: any element in common; views that lie between each other are fine."""
    ensure_built()
    start = change.get("v_cache", 0)
    if "v_cache" in change and not isinstance(start, torch.Tensor):
        k = change["k_cache"]
        offset = {None: 3 * k.stride(0), 1: k.stride(1)}.get(start, start)
        change = dict(change, v_cache=k.as_strided(k.shape, k.stride(), offset))
    k, v = (change.get(n) for n in (("k_cache", "v_cache") if "k_cache" in change else ("k_scale", "v_scale")))
    places = [set((t.storage_offset() + sum((torch.arange(n) * s).view([-1] + [1] * (3 - i)) for i, (n, s) in enumerate(
        zip((1,) * (4 - t.dim()) + tuple(t.shape), (0,) * (4 - t.dim()) + t.stride())))).flatten().tolist()) for t in (k, v)]
    assert bool(places[0] & places[1]) == shared and k.untyped_storage().data_ptr() == v.untyped_storage().data_ptr()
    args, _ = _cache_args("cache_append", **change)
    for call in _impls("cache_append"):
        with pytest.raises((ValueError, RuntimeError), match="must not share" if shared else "GPU"):
            call(*args)


def test_kernel_sizes_and_what_is_no_tensor():
    ensure_built()
    from e_natten_amd import cache_append, cache_attention
    args, _ = _cache_args("cache_attention")
    for bad, error in ((0, ValueError), (-3, ValueError), (2.0, TypeError), (True, TypeError), ("5", TypeError)):
        with pytest.raises(error, match="kernel_size"):
            cache_attention(*args, kernel_size=bad)
    with pytest.raises(TypeError, match="lengths must be a tensor"):
        cache_attention(*args[:-1], [1, 2])
    with pytest.raises(TypeError, match="counts must be a tensor"):
        cache_attention(*args, counts=[1, 2])
    args, _ = _cache_args("cache_append")
    with pytest.raises(TypeError, match="v must be a tensor"):
        cache_append(args[0], None, *args[2:])
    with pytest.raises(TypeError, match="counts must be a tensor"):
        cache_append(*args, counts=3)


def test_nothing_of_a_cache_has_a_gradient():
    """A caller that would silently get none is told (on tensors without data, which pass the other checks)."""
    ensure_built()
    import e_natten_amd as E
    if not E.ops.NATIVE_BINDING:
        pytest.skip("needs the native binding")
    for name, wants in (("cache_append", ("k", "v", "k_scale")), ("cache_attention", ("q", "v_scale"))):
        for what in wants:
            shape = {"q": (2, 4, 3, 32), "k": (2, 2, 3, 32), "v": (2, 2, 3, 32)}.get(what, (6, 2))
            x = torch.zeros(shape, dtype=F32 if "scale" in what else BF16, device="meta", requires_grad=True)
            args, _ = _cache_args(name, "meta", **{what: x})
            with pytest.raises(RuntimeError, match="no gradient"):
                getattr(E, name)(*args)
            with torch.no_grad():
                getattr(E, name)(*args)


def test_tangents_are_not_dropped():
    """A dual tensor has its tangent without requires_grad, in every grad mode; none of the operators has a
    derivative of forward mode, and a caller that would silently get zeros is told (tensors without data)."""
    ensure_built()
    import e_natten_amd as E
    from torch.autograd import forward_ad
    if not E.ops.NATIVE_BINDING:
        pytest.skip("needs the native binding")
    q, k, p, f = _rotary_args("meta")
    calls = [(q, lambda x: E.rotary(x, k, p, f)), (q, lambda x: E.rotary(x, None, p, f)),
             (k, lambda x: E.rotary(q, x, p, f)), (f, lambda x: E.rotary(q, k, p, x))]
    for name, which in (("cache_attention", (0, 3, 4)), ("cache_append", (0, 1, 4, 5))):
        args, _ = _cache_args(name, "meta")
        for i in which:
            calls.append((args[i], lambda x, name=name, args=args, i=i: getattr(E, name)(*args[:i], x, *args[i + 1:])))
    for x, call in calls:
        for mode in (torch.enable_grad, torch.no_grad):
            with forward_ad.dual_level(), mode():
                with pytest.raises(RuntimeError, match="forward-mode|no gradient"):
                    call(forward_ad.make_dual(x, torch.ones_like(x)))
                call(x)     # within the level, without a tangent
            with mode(), pytest.raises(RuntimeError, match="forward-mode|no gradient"):
                torch.func.jvp(lambda y: (call(y), y)[1], (x,), (torch.ones_like(x),))
    with pytest.raises(RuntimeError):
        torch.func.jacfwd(lambda y: E.rotary(y, None, p, f)[0].sum())(q)


def test_tangents_are_not_dropped_through_ctypes(monkeypatch):
    ensure_built()
    from e_natten_amd import sequence as S
    from torch.autograd import forward_ad
    monkeypatch.setattr(S, "_rotary_impl", lambda q, k, *rest: [q * 2.0] if k is None else [q * 2.0, k * 2.0])
    q, k, p, f = _rotary_args()
    call = lambda q, k, f: S.Rotary.apply(q, k, p, f, False, 1.0, False)
    for mode in (torch.enable_grad, torch.no_grad):
        with forward_ad.dual_level(), mode():
            dual = lambda x: forward_ad.make_dual(x, torch.ones_like(x))
            for args in ((dual(q), k, f), (dual(q), None, f), (q, dual(k), f), (q, k, dual(f))):
                with pytest.raises(RuntimeError):
                    call(*args)
                with pytest.raises(RuntimeError, match="no gradient"):
                    S._no_gradient("cache_append", *(x for x in args if x is not None))
            S._no_gradient("cache_append", q, k, f)


def test_append_counts_versions_in_every_mode():
    """A graph that saved a cache or its scales notices an append under torch.inference_mode() too."""
    ensure_built()
    import e_natten_amd as E
    if not E.ops.NATIVE_BINDING:
        pytest.skip("needs the native binding")
    x = torch.ones(6, 2, device="meta", requires_grad=True)
    for mode in (torch.enable_grad, torch.no_grad, torch.inference_mode):
        args, _ = _cache_args("cache_append", "meta")
        written = args[2:6]
        saved = x * args[4]
        before = [t._version for t in written]
        with mode():
            E.cache_append(*args)
        assert [t._version for t in written] == [n + 1 for n in before], mode
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            saved.sum().backward()
    with torch.inference_mode():
        args, _ = _cache_args("cache_append", "meta")   # inference tensors have no versions
        E.cache_append(*args)
    args, _ = _cache_args("cache_append", "meta")
    with torch.inference_mode():
        rows, _ = _cache_args("cache_append", "meta")
        E.cache_append(*rows[:2], *args[2:])            # new tokens of that mode, a cache that is older
    assert [t._version for t in args[2:6]] == [1] * 4


def test_shapes_without_data():
    ensure_built()
    import e_natten_amd as E
    if not E.ops.NATIVE_BINDING:
        pytest.skip("needs the native binding")
    q, k, p, f = _rotary_args("meta")
    a, b = E.rotary(q, k, p, f)
    assert (a.shape, b.shape, a.device.type) == (q.shape, k.shape, "meta") and E.rotary(q, None, p, f)[1] is None
    x = torch.zeros(2, 5, 6, 16, device="meta", requires_grad=True)
    a, b = E.rotary(x.transpose(1, 2)[:, :4], x.transpose(1, 2)[:, 4:], p, f)
    (g,) = torch.autograd.grad((a.sum() + b.sum()), x)
    assert g.shape == x.shape
    for cache in (I8, E4M3):
        args, _ = _cache_args("cache_append", "meta", cache=cache)
        before = args[2]._version, args[5]._version
        assert E.cache_append(*args) is None
        assert args[2]._version > before[0] and args[5]._version > before[1]
        args, _ = _cache_args("cache_attention", "meta", cache=cache, dtype=F16)
        o = E.cache_attention(*args)
        assert o.shape == args[0].shape and o.dtype == F16


# --- the C boundary ---

def _i64(*x):
    return (ctypes.c_int64 * len(x))(*x)


def test_c_rotary_validates_before_launch():
    lib = ensure_built()
    from e_natten_amd import _lib
    good = dict(q=16, k=16, qo=16, ko=16, p=16, f=16, B=1, hq=2, hk=1, T=3, D=16, R=8, dt=0, pd=_lib.I64, fd=_lib.F64,
                qs=None, ks=None, qos=None, kos=None, ps=0)

    def call(**change):
        a = dict(good, **change)
        return lib.enatten_rotary(a["q"], a["k"], a["qo"], a["ko"], a["p"], a["f"], a["B"], a["hq"], a["hk"], a["T"], a["D"],
                                  a["R"], a["dt"], a["pd"], a["fd"], 0, 0, a["qs"], a["ks"], a["qos"], a["kos"], a["ps"], 1.0,
                                  None)
    for change, text in ((dict(dt=9), "dtype"), (dict(pd=0), "positions"), (dict(fd=_lib.BF16), "frequencies"),
                         (dict(B=0), "dimension"), (dict(hk=0), "dimension"), (dict(T=-1), "dimension"), (dict(R=7), "even"),
                         (dict(R=18), "fit"), (dict(R=0), "even"), (dict(D=1040), "1024"), (dict(p=None), "NULL"),
                         (dict(f=None), "NULL"), (dict(ko=None), "together"), (dict(k=None), "together"), (dict(q=None), "q is NULL"),
                         (dict(qo=None), "q_out is NULL"), (dict(ps=-1), "negative"), (dict(qs=_i64(1, -1, 1)), "negative stride for q"),
                         (dict(kos=_i64(1, 1, -16)), "negative stride for k_out")):
        assert call(**change) == 1 and text in _lib.last_error(), change
    assert call(B=1 << 20, T=1 << 20, hq=16) == 2 and call(T=0x7fffffff, hq=1, hk=1) == 2 and call(hq=1 << 20, D=1024, R=8) == 2


def test_c_cache_validates_before_launch():
    lib = ensure_built()
    from e_natten_amd import _lib
    good = dict(x=16, y=16, kc=16, vc=16, ks=16, vs=16, pg=16, ln=16, ws=16, B=2, N=4, hk=2, T=3, D=32, np=6, page=16, cols=3,
                win=0, dt=1, cd=_lib.I8, xs=None, ys=None, kcs=None, vcs=None, kss=None, vss=None, pst=3)

    def append(**change):
        a = dict(good, **change)
        return lib.enatten_cache_append(a["x"], a["y"], a["kc"], a["vc"], a["ks"], a["vs"], a["pg"], a["ln"], None, a["B"],
                                        a["hk"], a["T"], a["D"], a["np"], a["page"], a["cols"], a["dt"], a["cd"], a["xs"],
                                        a["ys"], a["kcs"], a["vcs"], a["kss"], a["vss"], a["pst"], None)

    def attend(**change):
        a = dict(good, **change)
        return lib.enatten_cache_attention(a["x"], a["kc"], a["vc"], a["ks"], a["vs"], a["pg"], a["ln"], None, a["y"], a["ws"],
                                           a["B"], a["N"], a["hk"], a["T"], a["D"], a["np"], a["page"], a["cols"], a["win"],
                                           a["dt"], a["cd"], a["xs"], a["ys"], a["kcs"], a["vcs"], a["kss"], a["vss"], a["pst"],
                                           1.0, None)
    for change, text in ((dict(dt=3), "dtype"), (dict(cd=0), "cache dtype"), (dict(B=0), "dimension"), (dict(np=0), "dimension"),
                         (dict(cols=0), "dimension"), (dict(D=24), "head_dim"), (dict(D=272), "head_dim"), (dict(D=0), "head_dim"),
                         (dict(page=8), "pages must"), (dict(page=24), "pages must"), (dict(page=1040), "pages must"),
                         (dict(pst=-3), "pages"), (dict(x=None), "NULL"), (dict(y=None), "NULL"), (dict(kc=None), "NULL"),
                         (dict(vs=None), "NULL"), (dict(pg=None), "NULL"), (dict(ln=None), "NULL"),
                         (dict(xs=_i64(1, -16, 16)), "negative stride"), (dict(kcs=_i64(1024, 512, 16)), "to 2^20 between"),
                         (dict(vcs=_i64(1024, 512, 1 << 21)), "to 2^20 between"), (dict(kss=_i64(-1, 1)), "not be negative"),
                         (dict(kc=4), "multiples"), (dict(vcs=_i64(1028, 512, 32)), "multiples")):
        for f in (append, attend):
            assert f(**change) == 1 and text in _lib.last_error(), (f, change, _lib.last_error())
    for f in (append, attend):
        assert f(cols=1 << 27) == 2 and f(B=1 << 20, T=1 << 20) == 2 and f(T=0x7fffffff) == 2
    for change, text in ((dict(N=3), "multiple"), (dict(N=1), "multiple"), (dict(win=-1), "kernel_size"),
                         (dict(x=8), "16 bytes"), (dict(ys=_i64(4 * 3 * 32, 3 * 32 + 4, 32)), "16 bytes"),
                         (dict(kcs=_i64(1032, 512, 32)), "multiples of 16"), (dict(cols=100, ws=None), "workspace"),
                         (dict(cols=100, ws=8), "workspace")):
        assert attend(**change) == 1 and text in _lib.last_error(), (change, _lib.last_error())


def test_workspace_sizes():
    """None where one workgroup goes over a row tile; else for every possible part of rows x (D + 2) floats."""
    lib = ensure_built()
    need = lambda B=1, N=4, hk=2, T=1, D=64, page=16, cols=4, win=0, dt=1: lib.enatten_cache_attention_workspace_bytes(
        B, N, hk, T, D, page, cols, win, dt)
    assert need() == 0                                        # too short to be split
    assert need(B=4096, cols=4096) == 0                       # enough sequences
    assert need(cols=4096, win=100) == 0                      # the window is what counts
    parts = 16 * 4096 // 256 + 1                              # parts of at least 256 tokens, one for 16 tokens before
    assert need(cols=4096) == 4 * (4 + (min(parts, 256) + 1) * 2 * 16 * 66)
    assert need(T=40, N=16) == need(T=400, N=16) == 4 * (256 + 2 * 256 * 256 * 66)
    for bad in (dict(B=0), dict(N=3), dict(hk=0), dict(T=0), dict(D=0), dict(page=0), dict(cols=0), dict(win=-1)):
        assert need(**bad) == 0


def test_attention_kernels_do_not_spill():
    """A spilled operand of a matrix instruction came back incomplete where the compiler kept a part of it in
    an accumulation register: kernels that use these must not spill (cache_attention.hip).  What the
    compiler notes of every kernel is in the built library, its keys in alphabetical order."""
    ensure_built()
    import re
    from e_natten_amd import _lib
    text = open(_lib.LIB_PATH, "rb").read()
    entry = re.compile(rb"\.symbol.{1,3}?(_ZN7enatten12_GLOBAL__N_1\d+(?:attend|attend_join)I\w+)\.kd"
                       rb".{0,200}?\.vgpr_spill_count(.)", re.S)
    spills = {m.group(1): m.group(2)[0] for m in entry.finditer(text)}
    assert len(spills) > 40
    assert not any(spills.values()), [k for k, n in spills.items() if n]


def _registers():
    """{kernel: (accumulation registers, spilled registers)} of the built library, as the compiler notes them:
    maps with their keys in alphabetical order, .agpr_count first, numbers of up to two bytes."""
    import re
    from e_natten_amd import _lib

    def number(b):
        return b[0] if b[0] < 0x80 else b[1] if b[0] == 0xcc else int.from_bytes(b[1:3], "big")

    found = {}
    for part in open(_lib.LIB_PATH, "rb").read().split(b".agpr_count")[1:]:
        name = re.search(rb"\.symbol.{1,3}?(_Z\w+)\.kd", part[:40000], re.S)
        spilled = re.search(rb"\.vgpr_spill_count(.{3})", part[:40000], re.S)
        if name and spilled and name.start() < spilled.start():
            found[name.group(1).decode()] = number(part), number(spilled.group(1))
    return found


def test_kernels_that_spill_have_no_accumulation_registers():
    """The other half of the rule above: attend_rows spills above 128 channels (about 50 registers), which is
    sound as long as every spilled register goes to memory, that is as long as the kernel has no accumulation
    registers.  Every instantiation of the four kernels has to be there."""
    ensure_built()
    import re
    found = _registers()
    ours = {kind: {n: v for n, v in found.items() if re.match(r"_ZN7enatten12_GLOBAL__N_1%d%sI" % (len(kind), kind), n)}
            for kind in ("attend", "attend_join", "attend_rows", "join_rows")}
    # 4 + 3 + 1 numbers of row tiles by head dim, 2 caches, 3 types; float32 above 128 channels has no wide tile
    assert {kind: len(v) for kind, v in ours.items()} == {"attend": 48, "attend_join": 12, "attend_rows": 16, "join_rows": 8}
    bad = {n: v for kind in ours.values() for n, v in kind.items() if v[0] and v[1]}
    assert not bad, bad
    assert not any(v[0] for v in ours["attend_rows"].values())


def test_no_other_kernel_spills_beside_accumulation_registers():
    """Three builds of the dQ pass with a bias at head_dim 128, 11x11 and 13x13 windows, do: what they spill are
    single words and pairs, each back in ordinary registers before its use.  A further one has to be read first."""
    ensure_built()
    import re
    beside = {n: v for n, v in _registers().items() if v[0] and v[1]}
    known = re.compile(r"_ZN7enatten12_GLOBAL__N_112bwd_dq2_mfmaILb[01]ELi128ELi1[13]ELi4ELb0ELb0EEEv")
    assert len(beside) <= 3 and all(known.match(n) for n in beside), beside
