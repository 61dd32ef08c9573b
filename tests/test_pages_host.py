"""Host side of the operators on pages of a cache and of rotary positions with several axes, without a GPU:
what the entry points refuse (in Python, in the native binding and at the C boundary), shapes without data."""
import ctypes

import pytest
import torch

from _util import ensure_built

BF16, F16, F32, F64 = torch.bfloat16, torch.float16, torch.float32, torch.float64
I8, E4M3, I32, I64 = torch.int8, torch.float8_e4m3fn, torch.int32, torch.int64


def _z(*shape, dtype=I32):
    return torch.zeros(shape, dtype=dtype)


# --- axes ---

def test_axes_of_pairs():
    ensure_built()
    from e_natten_amd import rotary_axes
    assert rotary_axes(12, 2).tolist() == [0, 0, 0, 1, 1, 1]
    assert rotary_axes(14, 3).tolist() == [0, 0, 0, 1, 1, 2, 2]
    assert rotary_axes(14, 3, "cyclic").tolist() == [0, 1, 2, 0, 1, 2, 0]
    assert rotary_axes(12, [1, 0, 5]).tolist() == [0, 2, 2, 2, 2, 2]
    assert rotary_axes(12, [3, 2, 1], "cyclic").tolist() == [0, 1, 2, 0, 1, 0]
    assert rotary_axes(2, 1).tolist() == [0] and rotary_axes(4, 2).dtype == I32
    assert rotary_axes(4, 5).tolist() == [0, 1]


@pytest.mark.parametrize("error,args", [
    (TypeError, (8.0, 2)), (TypeError, (True, 2)), (ValueError, (7, 2)), (ValueError, (0, 2)), (ValueError, (8, 0)),
    (ValueError, (8, -1)), (ValueError, (8, [1, 2])), (ValueError, (8, [5, -1])), (TypeError, (8, [2.0, 2])),
    (TypeError, (8, True)), (ValueError, (8, [])), (ValueError, (8, 2, "other")),
])
def test_axes_of_pairs_refuse(error, args):
    from e_natten_amd import rotary_axes
    with pytest.raises(error):
        rotary_axes(*args)


def _rotary_args(**change):
    a = dict(q=_z(2, 4, 6, 16, dtype=F32), k=_z(2, 2, 6, 16, dtype=F32), positions=torch.arange(12).view(2, 6),
             frequencies=torch.ones(8, dtype=F64), axes=_z(8))
    a.update(change)
    return a


_IMAGE = dict(q=_z(2, 4, 2, 3, 16, dtype=F32), k=_z(2, 2, 2, 3, 16, dtype=F32), positions=torch.arange(12).view(2, 2, 3))


@pytest.mark.parametrize("change,text", [
    (dict(axes=_z(7)), "one for every frequency"), (dict(axes=_z(8, dtype=I64)), "int32"), (dict(axes=_z(8, 1)), "every frequency"),
    (dict(positions=torch.arange(6)), "shape"), (dict(positions=_z(2, 3, 6)), "shape"), (dict(positions=_z(0, 6)), "shape"),
    (dict(positions=_z(2, 1, 1, 6)), "shape"), (dict(positions=_z(2, 5)), "shape"), (dict(positions=_z()), "shape"),
    (dict(axes=torch.zeros(8, dtype=I32, device="meta")), "device"),
    (dict(q=_z(2, 4, 16, dtype=F32), k=None), "heads, T"), (dict(), "GPU"),
])
def test_rotary_with_axes_refuses(change, text):
    ensure_built()
    import e_natten_amd as E
    from e_natten_amd import sequence as S
    a = _rotary_args(**change)
    for call in (lambda: E.rotary(a["q"], a["k"], a["positions"], a["frequencies"], axes=a["axes"]),
                 lambda: S.Rotary.apply(a["q"], a["k"], a["positions"], a["frequencies"], False, 1.0, False, a["axes"])):
        with pytest.raises((ValueError, RuntimeError), match=text):
            call()


@pytest.mark.parametrize("change,text", [
    (dict(k=_z(2, 2, 6, 16, dtype=F32)), "differ in their heads"), (dict(k=_z(2, 2, 3, 2, 16, dtype=F32)), "differ in their heads"),
    (dict(positions=_z(2, 6)), "H, W"), (dict(positions=_z(2, 3, 2)), "H, W"), (dict(positions=_z(2, 3, 2, 3)), "shape"),
    (dict(), "GPU"),
])
def test_rotary_of_images_refuses(change, text):
    ensure_built()
    from e_natten_amd import rotary
    a = _rotary_args(**dict(_IMAGE, **change))
    with pytest.raises((ValueError, RuntimeError), match=text):
        rotary(a["q"], a["k"], a["positions"], a["frequencies"], axes=a["axes"])


def test_rotary_without_axes_takes_no_images():
    ensure_built()
    from e_natten_amd import rotary
    a = _rotary_args(**_IMAGE)
    with pytest.raises(ValueError, match="5-D"):
        rotary(a["q"], a["k"], torch.arange(6), a["frequencies"])
    with pytest.raises(TypeError, match="tensor"):
        rotary(a["q"], a["k"], a["positions"], a["frequencies"], axes=[0] * 8)


# --- pages ---

def _args(name, **change):
    a = dict(pages=_z(3, 5), lengths=_z(3), holders=_z(20), parents=_z(3), page=16, counts=1,
             k_cache=_z(4, 2, 16, 32, dtype=I8), v_cache=_z(4, 2, 16, 32, dtype=I8), k_scale=_z(4, 2, dtype=F32),
             v_scale=_z(4, 2, dtype=F32), copies=_z(6, 3))
    a.update(change)
    keys = {"cache_fork": ("pages", "lengths", "holders", "parents", "page"),
            "cache_reserve": ("pages", "lengths", "holders", "page", "counts"),
            "cache_compact": ("pages", "holders", "page"),
            "cache_copy": ("k_cache", "v_cache", "k_scale", "v_scale", "copies")}[name]
    return tuple(a[k] for k in keys)


def _impls(name):
    """(the public function, the same call through ctypes)"""
    import e_natten_amd as E
    from e_natten_amd import pages as P
    ctyped = {"cache_fork": P._fork_impl, "cache_compact": P._compact_impl, "cache_copy": P._copy_impl}.get(name)
    if name == "cache_reserve":
        def ctyped(pages, lengths, holders, page, counts):
            none = isinstance(counts, int)
            return P._reserve_impl(pages, lengths, holders, page, None if none else counts, counts if none else 0)
    return getattr(E, name), ctyped


@pytest.mark.parametrize("change,text", [
    (dict(pages=_z(3)), "B, columns"), (dict(pages=_z(3, 5, dtype=I64)), "int32"), (dict(pages=_z(3, 0)), "B, columns"),
    (dict(pages=_z(5, 3).t()), "unit stride"), (dict(pages=_z(1, 5).expand(3, 5)), "overlap"),
    (dict(page=0), "multiple of 16"), (dict(page=24), "multiple of 16"), (dict(page=1040), "multiple of 16"),
    (dict(page=-16), "multiple of 16"), (dict(holders=_z(0)), "holders"), (dict(holders=_z(4, 5)), "holders"),
    (dict(holders=_z(20, dtype=I64)), "holders"), (dict(holders=_z(40)[::2]), "contiguous"),
    (dict(holders=torch.zeros(20, dtype=I32, device="meta")), "same device"), (dict(), "GPU"),
])
def test_tables_refuse(change, text):
    ensure_built()
    for name in ("cache_fork", "cache_reserve", "cache_compact"):
        for call in _impls(name):
            with pytest.raises((ValueError, RuntimeError), match=text):
                call(*_args(name, **change))


@pytest.mark.parametrize("name,change,text", [
    ("cache_fork", dict(lengths=_z(4)), "lengths"), ("cache_fork", dict(lengths=_z(3, dtype=I64)), "lengths"),
    ("cache_fork", dict(lengths=_z(6)[::2]), "contiguous"), ("cache_fork", dict(parents=_z(2)), "parents"),
    ("cache_fork", dict(parents=_z(3, dtype=I64)), "parents"),
    ("cache_fork", dict(parents=torch.zeros(3, dtype=I32, device="meta")), "same device"),
    ("cache_reserve", dict(lengths=_z(4)), "lengths"), ("cache_reserve", dict(counts=_z(2)), "counts"),
    ("cache_reserve", dict(counts=_z(3, dtype=I64)), "counts"), ("cache_reserve", dict(counts=-1), "negative"),
    ("cache_reserve", dict(counts=torch.zeros(3, dtype=I32, device="meta")), "same device"),
    ("cache_copy", dict(k_cache=_z(2, 16, 32, dtype=I8), v_cache=_z(2, 16, 32, dtype=I8)), "must be \\[pages"),
    ("cache_copy", dict(v_cache=_z(5, 2, 16, 32, dtype=I8)), "must be \\[pages"),
    ("cache_copy", dict(k_cache=_z(0, 2, 16, 32, dtype=I8), v_cache=_z(0, 2, 16, 32, dtype=I8)), "must be \\[pages"),
    ("cache_copy", dict(v_cache=_z(4, 2, 16, 32, dtype=E4M3)), "int8 or float8"),
    ("cache_copy", dict(k_cache=_z(4, 2, 16, 32, dtype=BF16), v_cache=_z(4, 2, 16, 32, dtype=BF16)), "int8 or float8"),
    ("cache_copy", dict(k_cache=_z(4, 2, 32, 16, dtype=I8).transpose(2, 3)), "unit stride"),
    ("cache_copy", dict(k_scale=_z(4, 3, dtype=F32)), "k_scale"), ("cache_copy", dict(v_scale=_z(4, 2, dtype=F16)), "float32"),
    ("cache_copy", dict(k_cache=_z(3, 4, 2, 16, 32, dtype=I8), v_cache=_z(3, 4, 2, 16, 32, dtype=I8)), "k_scale"),
    ("cache_copy", dict(copies=_z(6)), "copies"), ("cache_copy", dict(copies=_z(6, 2)), "copies"),
    ("cache_copy", dict(copies=_z(6, 3, dtype=I64)), "copies"), ("cache_copy", dict(k_scale=_z(4, 1, dtype=F32).expand(4, 2)), "memory"),
    ("cache_copy", dict(k_cache=_z(1, 2, 16, 32, dtype=I8).expand(4, 2, 16, 32)), "memory"),
    ("cache_copy", dict(copies=torch.zeros(6, 3, dtype=I32, device="meta")), "same device"),
    ("cache_copy", dict(k_cache=_z(1, 1, 1040, 16, dtype=I8), v_cache=_z(1, 1, 1040, 16, dtype=I8), k_scale=_z(1, 1, dtype=F32),
                        v_scale=_z(1, 1, dtype=F32)), "1024"),
    ("cache_copy", dict(), "GPU"),
])
def test_pages_refuse(name, change, text):
    ensure_built()
    for call in _impls(name):
        with pytest.raises((ValueError, RuntimeError), match=text):
            call(*_args(name, **change))


_LAYERS = _z(4, 3, 2, 16, 32, dtype=I8).transpose(0, 1)     # layers, pages, heads, tokens, channels
_POOL = _z(6, 2, 2, 16, 32, dtype=I8)                       # pages, keys and values, ...


@pytest.mark.parametrize("shared,change", [
    (True, dict(k_cache=_POOL[:4, 0], v_cache=_POOL[:4, 0])), (True, dict(k_cache=_POOL[:4, 0], v_cache=_POOL[2:, 0])),
    (False, dict(k_cache=_POOL[:4, 0], v_cache=_POOL[:4, 1])),
    (True, dict(k_cache=_LAYERS[:2], v_cache=_LAYERS[1:], k_scale=_z(2, 4, 2, dtype=F32), v_scale=_z(2, 4, 2, dtype=F32))),
    (False, dict(k_cache=_LAYERS[:1], v_cache=_LAYERS[1:2], k_scale=_z(1, 4, 2, dtype=F32), v_scale=_z(1, 4, 2, dtype=F32))),
    (True, dict(k_scale=_z(6, 2, dtype=F32)[:4], v_scale=0)),   # (v_scale: the same from page 2 on)
])
def test_copy_refuses_keys_and_values_that_share_some_memory(shared, change):
    ensure_built()
    if isinstance(change.get("v_scale"), int):
        change = dict(change, v_scale=change["k_scale"]._base[2:])
    for call in _impls("cache_copy"):
        with pytest.raises((ValueError, RuntimeError), match="must not share a cache" if shared else "GPU"):
            call(*_args("cache_copy", **change))


def test_what_is_no_tensor_or_no_int():
    ensure_built()
    import e_natten_amd as E
    for name, key in (("cache_fork", "pages"), ("cache_fork", "parents"), ("cache_reserve", "holders"), ("cache_reserve", "counts"),
                      ("cache_compact", "holders"), ("cache_copy", "copies"), ("cache_copy", "v_scale")):
        with pytest.raises(TypeError, match="tensor"):
            getattr(E, name)(*_args(name, **{key: [1, 2, 3]}))
    for name in ("cache_fork", "cache_reserve", "cache_compact"):
        for page in (16.0, True, None):
            with pytest.raises(TypeError, match="page"):
                getattr(E, name)(*_args(name, page=page))
    with pytest.raises(TypeError, match="tensor"):
        E.cache_reserve(*_args("cache_reserve", counts=True))


def test_scales_that_want_a_gradient():
    ensure_built()
    import e_natten_amd as E
    from e_natten_amd import pages as P
    for call in (E.cache_copy, P._copy_impl):
        if call is P._copy_impl and not torch.cuda.is_available():
            continue    # (the device is looked at first)
        with pytest.raises(RuntimeError, match="no gradient|GPU"):
            call(*_args("cache_copy", k_scale=torch.zeros(4, 2, requires_grad=True)))
    with pytest.raises(RuntimeError, match="no gradient"):
        E.cache_copy(*(x.to("meta") for x in _args("cache_copy", k_scale=torch.zeros(4, 2, requires_grad=True))))


def test_shapes_without_data():
    ensure_built()
    import e_natten_amd as E
    if not E.ops.NATIVE_BINDING:
        pytest.skip("needs the native binding")
    there = lambda name, **c: [x.to("meta") if isinstance(x, torch.Tensor) else x for x in _args(name, **c)]
    assert E.cache_fork(*there("cache_fork")) is None and E.cache_copy(*there("cache_copy")) is None
    copies = E.cache_reserve(*there("cache_reserve"))
    assert copies.shape == (3, 3) and copies.dtype == I32 and copies.device.type == "meta"
    assert E.cache_compact(*there("cache_compact")).shape == (10, 3)
    assert E.cache_compact(*there("cache_compact", holders=_z(1))).shape == (1, 3)
    a = _rotary_args(**_IMAGE)
    m = {k: v.to("meta") for k, v in a.items()}
    q, k = E.rotary(m["q"], m["k"], m["positions"], m["frequencies"], axes=m["axes"])
    assert q.shape == a["q"].shape and k.shape == a["k"].shape


def test_versions_are_counted_in_every_mode():
    """A graph made before may have saved what the calls write."""
    ensure_built()
    import e_natten_amd as E
    if not E.ops.NATIVE_BINDING:
        pytest.skip("needs the native binding")
    written = {"cache_fork": (0, 1, 2), "cache_reserve": (0, 2), "cache_compact": (0, 1), "cache_copy": (0, 1, 2, 3)}
    for name, which in written.items():
        args = [x.to("meta") if isinstance(x, torch.Tensor) else x for x in _args(name)]
        before = [x._version for x in args if isinstance(x, torch.Tensor)]
        getattr(E, name)(*args)
        with torch.no_grad():
            getattr(E, name)(*args)
        with torch.inference_mode():
            getattr(E, name)(*args)
        tensors = [x for x in args if isinstance(x, torch.Tensor)]
        grown = [x._version - b for x, b in zip(tensors, before)]
        places = [i for i, x in enumerate(args) if isinstance(x, torch.Tensor)]
        assert grown == [3 if p in which else 0 for p in places], name


# --- the C boundary ---

def _lib():
    ensure_built()
    from e_natten_amd import _lib
    return _lib.load(), _lib


def _text(lib):
    return lib.enatten_last_error().decode()


def test_c_rotary_axes_validates_before_launch():
    lib, L = _lib()
    at, none = ctypes.c_void_p(16), None

    def call(axes=at, count=2, stride=5, R=16, D=16):
        return lib.enatten_rotary_axes(at, none, at, none, at, at, axes, count, 1, 1, 0, 5, D, R, L.F32, L.I32, L.F64, 0, 0, none,
                                       none, none, none, 0, stride, 1.0, none)

    for bad in (dict(axes=none), dict(count=0), dict(stride=-1), dict(R=18), dict(R=3)):
        assert call(**bad) == 1 and "enatten_rotary_axes" in _text(lib)


def test_c_pages_validate_before_launch():
    lib, _ = _lib()
    at, none = ctypes.c_void_p(16), None

    def fork(pages=at, lengths=at, holders=at, parents=at, B=2, columns=3, total=4, page=16, stride=3):
        return lib.enatten_cache_fork(pages, lengths, holders, parents, B, columns, total, page, stride, none)

    def reserve(pages=at, lengths=at, holders=at, copies=at, ws=at, B=2, columns=3, total=4, page=16, stride=3):
        return lib.enatten_cache_reserve(pages, lengths, none, 1, holders, copies, ws, B, columns, total, page, stride, none)

    def compact(pages=at, holders=at, copies=at, ws=at, B=2, columns=3, total=4, page=16, stride=3):
        return lib.enatten_cache_compact(pages, holders, copies, ws, B, columns, total, page, stride, none)

    for call in (fork, reserve, compact):
        for bad in (dict(pages=none), dict(holders=none), dict(B=0), dict(columns=0), dict(total=0), dict(page=8),
                    dict(page=2048), dict(stride=2), dict(stride=-3)):
            assert call(**bad) == 1 and "enatten_cache" in _text(lib), (call, bad)
        for bad in (dict(B=4097), dict(columns=1 << 30, stride=1 << 30), dict(columns=1 << 27, stride=1 << 27)):
            assert call(**bad) not in (0, 1), (call, bad)
    for bad in (dict(lengths=none), dict(parents=none)):
        assert fork(**bad) == 1
    for call, bads in ((reserve, (dict(lengths=none), dict(copies=none), dict(ws=none), dict(ws=ctypes.c_void_p(8)))),
                       (compact, (dict(copies=none), dict(ws=none), dict(ws=ctypes.c_void_p(20))))):
        for bad in bads:
            assert call(**bad) == 1, (call, bad)
    assert lib.enatten_cache_reserve_workspace_bytes(2, 3, 4) == 2 * 4 * 4
    assert lib.enatten_cache_compact_workspace_bytes(4096) == 4 * (4096 + 2)
    assert lib.enatten_cache_compact_workspace_bytes(2 ** 31 - 1) == 4 * (2 ** 31 - 1 + 2 ** 20)
    for bad in ((0, 3, 4), (2, 0, 4), (2, 3, 0)):
        assert lib.enatten_cache_reserve_workspace_bytes(*bad) == 0
    assert lib.enatten_cache_compact_workspace_bytes(0) == 0


def test_c_pages_refuse_memory_that_is_written_twice():
    """Addresses that nothing is read from: a table [3, 4] of rows 10 entries apart, 20 pages."""
    lib, _ = _lib()
    none, base = ctypes.c_void_p(None), 1 << 20

    def at(entry, byte=0):
        return ctypes.c_void_p(base + 4 * entry + byte)

    far = dict(lengths=at(100), holders=at(200), parents=at(300), copies=at(400), ws=at(500), counts=at(600))
    sizes = (3, 4, 20, 16, 10, none)

    def fork(lengths, holders, parents, **_):
        return lib.enatten_cache_fork(at(0), lengths, holders, parents, *sizes)

    def reserve(lengths, holders, copies, ws, counts, **_):
        return lib.enatten_cache_reserve(at(0), lengths, counts, 1, holders, copies, ws, *sizes)

    def compact(holders, copies, ws, **_):
        return lib.enatten_cache_compact(at(0), holders, copies, ws, *sizes)

    for call, bads in (
            (fork, (dict(lengths=at(0)), dict(lengths=at(-2)), dict(lengths=at(3)), dict(lengths=at(8)), dict(lengths=at(23)),
                    dict(holders=at(4)), dict(holders=at(-19)), dict(parents=at(11)), dict(parents=far["lengths"]),
                    dict(parents=at(302), lengths=at(300)), dict(lengths=at(219)), dict(holders=at(300, -76)),
                    dict(lengths=at(4, -1)), dict(lengths=at(7, 1)))),
            (reserve, (dict(lengths=at(12)), dict(counts=at(23)), dict(counts=at(200)), dict(lengths=at(408)), dict(copies=at(0)),
                       dict(copies=at(219)), dict(ws=at(400)), dict(ws=at(8)), dict(ws=at(596), counts=at(600)))),
            (compact, (dict(holders=at(0)), dict(copies=at(20)), dict(copies=far["holders"]), dict(ws=at(180)),
                       dict(copies=at(371), ws=at(400))))):
        for bad in bads:
            assert call(**dict(far, **bad)) == 1 and "must not share memory" in _text(lib), (call, bad)


def test_c_copy_validates_before_launch():
    lib, _ = _lib()
    at, none = ctypes.c_void_p(16), None
    s4 = lambda *x: (ctypes.c_int64 * 4)(*x)

    def call(k=at, v=at, ks=at, vs=at, copies=at, n=3, layers=1, heads=2, D=32, total=4, page=16, st=None, zst=None):
        return lib.enatten_cache_copy(k, v, ks, vs, copies, n, layers, heads, D, total, page, st, none, zst, none, none)

    for bad in (dict(k=none), dict(v=none), dict(ks=none), dict(vs=none), dict(copies=none), dict(n=-1), dict(layers=0),
                dict(heads=0), dict(D=24), dict(D=272), dict(total=0), dict(page=20), dict(page=2048), dict(k=ctypes.c_void_p(8)),
                dict(st=s4(0, 1024, 512, 40)), dict(st=s4(0, 1024, 512, 16)), dict(st=s4(0, -1024, 512, 32)),
                dict(st=s4(8, 1024, 512, 32)), dict(st=s4(0, 1024, 512, 1 << 21)), dict(zst=(ctypes.c_int64 * 3)(0, -1, 1))):
        assert call(**bad) == 1 and "enatten_cache_copy" in _text(lib), bad
    assert call(layers=1 << 10, heads=64) not in (0, 1)
    assert call(n=0) == 0 and call(n=0, copies=none) == 0
