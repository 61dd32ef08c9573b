"""Host side of cache_attention over runs that share their first tokens, without a GPU: what the entry points
refuse, workspaces, and the built kernels' registers."""
import ctypes
import re

import pytest
import torch

from _util import ensure_built

BF16, F32, I8, I32 = torch.bfloat16, torch.float32, torch.int8, torch.int32


def _z(*shape, dtype=I32):
    return torch.zeros(shape, dtype=dtype)


def _args(**change):
    a = dict(q=_z(6, 4, 1, 32, dtype=BF16), k=_z(8, 2, 16, 32, dtype=I8), v=_z(8, 2, 16, 32, dtype=I8),
             ks=_z(8, 2, dtype=F32), vs=_z(8, 2, dtype=F32), pages=_z(6, 3), lengths=_z(6), counts=None, shared=_z(2))
    a.update(change)
    return a


@pytest.mark.parametrize("change,text", [
    (dict(shared=_z(4)), "divisor of 6"), (dict(shared=_z(0)), "divisor"), (dict(shared=_z(12)), "divisor"),
    (dict(shared=_z(2, 1)), "shared must be"), (dict(shared=_z(2, dtype=torch.int64)), "int32"), (dict(shared=_z(2, dtype=F32)), "int32"),
    (dict(shared=torch.zeros(2, dtype=I32, device="meta")), "same device"), (dict(lengths=_z(5)), "lengths"), (dict(), "GPU"),
])
def test_shared_refuses(change, text):
    ensure_built()
    import e_natten_amd as E
    from e_natten_amd import sequence as S
    a = _args(**change)
    front = (a["q"], a["k"], a["v"], a["ks"], a["vs"], a["pages"], a["lengths"])
    for call in (lambda: E.cache_attention(*front, None, 1.0, a["counts"], a["shared"]),
                 lambda: S._attention_impl(*front, a["counts"], 0, 1.0, a["shared"])):
        with pytest.raises((ValueError, RuntimeError), match=text):
            call()


def test_shared_is_a_tensor_and_has_shapes_without_data():
    ensure_built()
    import e_natten_amd as E
    a = _args()
    front = [a["q"], a["k"], a["v"], a["ks"], a["vs"], a["pages"], a["lengths"]]
    for bad in (3, [0, 0], 1.5):
        with pytest.raises(TypeError, match="tensor"):
            E.cache_attention(*front, None, 1.0, None, bad)
    if E.ops.NATIVE_BINDING:
        o = E.cache_attention(*(x.to("meta") for x in front), None, 1.0, None, a["shared"].to("meta"))
        assert o.shape == a["q"].shape and o.dtype == BF16


def test_c_shared_validates_before_launch():
    ensure_built()
    from e_natten_amd import _lib
    lib = _lib.load()
    at, none = ctypes.c_void_p(16), None

    wide = 1 << 16   # columns: so many that the sequences' codes could be 16 MB and more

    def call(shared=at, runs=2, B=6, heads=4, ws=at, o=at, D=32, lengths=at):
        return lib.enatten_cache_attention_shared(at, at, at, at, at, at, lengths, none, shared, runs, o, ws, B, heads, 2, 1, D,
                                                  8, 16, wide, 0, _lib.BF16, _lib.I8, none, none, none, none, none, none, wide, 1.0, none)

    for bad in (dict(shared=none), dict(runs=0), dict(runs=-1), dict(runs=4), dict(runs=12), dict(ws=none),
                dict(ws=ctypes.c_void_p(8)), dict(heads=3), dict(o=none), dict(D=24), dict(lengths=none), dict(B=0)):
        assert call(**bad) == 1 and "enatten_cache_attention_shared" in lib.enatten_last_error().decode(), bad
    # rows of runs with up to 16 have a workgroup each that joins their parts: fewer than 2^24
    assert call(B=1 << 22, runs=1 << 21) not in (0, 1)
    assert "too many rows" in lib.enatten_last_error().decode()

    def need(B=6, runs=2, T=1, cols=wide, heads=4, D=32, window=0, call=lib.enatten_cache_attention_shared_workspace_bytes):
        return call(B, heads, 2, T, D, 16, cols, window, _lib.BF16, *((runs,) if call is not plain else ()))

    plain = lib.enatten_cache_attention_workspace_bytes
    rows = lambda B, T: B * 4 * T * 34 * 4   # a row's sums of values, maximum and sum, once for the run and once for itself
    assert need() >= 2 * rows(6, 1) and need(T=3) >= 2 * rows(6, 3) and need(T=16) >= 2 * rows(6, 16)
    # by themselves: few codes, short windows, tiles of 256 rows for every sequence
    for alone in (dict(cols=3), dict(cols=682), dict(window=10921), dict(T=100), dict(T=49), dict(T=7, cols=6826),
                  dict(T=16, cols=6826), dict(runs=6), dict(runs=3, T=7), dict(runs=2, T=3, D=256), dict(runs=1, T=3, D=256, cols=3413),
                  dict(runs=2, T=9, D=256, cols=682)):
        assert need(**alone) == need(**alone, call=plain), alone
    for together in (dict(cols=683), dict(window=10922), dict(T=7, cols=6827), dict(T=16, cols=6827), dict(T=48), dict(runs=3, T=16),
                     dict(runs=3), dict(runs=1, T=3, D=256, cols=3414), dict(runs=2, T=9, D=256, cols=683)):
        assert need(**together) != need(**together, call=plain), together
    for bad in (dict(B=0), dict(runs=0), dict(runs=4), dict(T=0), dict(cols=0), dict(heads=3), dict(T=1 << 28)):
        assert need(**bad) == 0


def test_kernels_do_not_spill_beside_accumulation_registers():
    """As those for sequences by themselves: a spilled operand of a matrix instruction is sound only where every
    spilled register goes to memory, that is in kernels without accumulation registers.  Every instantiation of
    the two passes has to be there."""
    ensure_built()
    from test_sequence_host import _registers
    found = _registers()
    ours = {kind: {n: v for n, v in found.items() if re.match(r"_ZN7enatten12_GLOBAL__N_1%d%sI" % (len(kind), kind), n)}
            for kind in ("run_attend", "run_rows", "run_join", "run_join_tiles")}
    assert {kind: len(v) for kind, v in ours.items()} == {"run_attend": 48, "run_rows": 40, "run_join": 8, "run_join_tiles": 3}
    for kind, kernels in ours.items():
        assert not {n: v for n, v in kernels.items() if v[1] and (v[0] or kind != "run_rows")}
