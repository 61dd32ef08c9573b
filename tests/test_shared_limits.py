"""cache_attention of runs with more rows than a launch joins: refused at the C boundary before anything is queued
(without a GPU a launch would say that it failed), answered by the public function, where every sequence reads for
itself."""
import ctypes

import pytest
import torch

from _util import ensure_built

BF16, I8, I32 = torch.bfloat16, torch.int8, torch.int32
# B, heads, heads of the cache, sequences of a run: up to 16 rows in a run, and more
_SIZES = [((1 << 21) + 2, 8, 1, 2), (1 << 22, 17, 1, 2)]


@pytest.mark.parametrize("B,heads,heads_kv,size", _SIZES)
def test_c_refuses_before_launch(B, heads, heads_kv, size):
    ensure_built()
    from e_natten_amd import _lib
    lib, at, none = _lib.load(), ctypes.c_void_p(16), None
    D, page, columns = 16, 16, 2
    sizes = (B, heads, heads_kv, 1, D, page, columns, 0, _lib.BF16)
    rc = lib.enatten_cache_attention_shared(at, at, at, at, at, at, at, none, at, B // size, at, at, B, heads, heads_kv, 1, D, 8, page,
                                            columns, 0, _lib.BF16, _lib.I8, none, none, none, none, none, none, columns, 1.0, none)
    assert rc == _lib.EUNSUPPORTED and "too many rows" in lib.enatten_last_error().decode()
    assert lib.enatten_cache_attention_shared_workspace_bytes(*sizes, B // size) == 0
    fewer = (B // 2 // size * size, *sizes[1:])
    assert lib.enatten_cache_attention_shared_workspace_bytes(*fewer, fewer[0] // size) > 0


@pytest.mark.gpu
@pytest.mark.parametrize("B,heads,heads_kv,size", _SIZES)
def test_every_sequence_reads_for_itself(B, heads, heads_kv, size):
    ensure_built()
    from e_natten_amd import cache_attention
    from e_natten_amd import sequence as S
    print("case many rows", B, heads, heads_kv, size, flush=True)
    g = torch.Generator(device="cuda").manual_seed(1)
    pages, page, d = 64, 16, 16
    codes = [torch.randint(-127, 128, (pages, heads_kv, page, d), generator=g, device="cuda", dtype=I8) for _ in range(2)]
    scales = [torch.rand(pages, heads_kv, generator=g, device="cuda") * 0.02 + 0.01 for _ in range(2)]
    q = torch.randn(B, heads, 1, d, generator=g, device="cuda", dtype=BF16)
    table = torch.randint(0, pages, (B, 2), generator=g, device="cuda", dtype=I32)
    table.view(B // size, size, 2)[:, :, 0] = table[::size, :1]
    lengths = torch.randint(17, 33, (B,), generator=g, device="cuda", dtype=I32)
    shared = torch.full((B // size,), 16, device="cuda", dtype=I32)
    args = (q, *codes, *scales, table, lengths)
    want = cache_attention(*args, None, 0.25)
    assert torch.equal(cache_attention(*args, None, 0.25, None, shared), want)
    assert torch.equal(S._attention_impl(*args, None, 0, 0.25, shared), want)
    # the definition, for some of them
    some = torch.tensor([0, 1, B // 2, B - 1], device="cuda")
    kv = [(c.double() * s.double()[:, :, None, None])[table[some].long(), 0].flatten(1, 2) for c, s in zip(codes, scales)]
    logits = (q[some, :, 0].double() * 0.25) @ kv[0].transpose(1, 2)
    p = torch.where(torch.arange(32, device="cuda") < lengths[some, None, None], logits, -torch.inf).softmax(-1)
    ref, most = p @ kv[1], (p @ kv[1].abs())
    # a rounding of the result, and of each weight to 11 bits
    assert ((want[some, :, 0].double() - ref).abs() <= 2.0 ** -8 * ref.abs() + 2.0 ** -9 * most).all()
