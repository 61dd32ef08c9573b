"""How many pages a table may speak of, without a GPU: places in the list of moves are numbers of 32 bits, three for
each of up to half of the pages."""
import ctypes

import pytest
import torch

from _util import ensure_built

MOST = 1 << 30


def test_moves_of_the_most_pages_have_places_of_32_bits():
    assert 3 * (MOST // 2) + 2 < 2 ** 31 <= 3 * ((2 ** 31 - 1) // 2)


@pytest.mark.parametrize("total,refused", [(MOST, False), (MOST + 1, True), (2 ** 31 - 1, True)])
def test_c_pages_of_a_table(total, refused):
    """Addresses that nothing is read from; calls that are not refused for their size are for a NULL argument."""
    ensure_built()
    from e_natten_amd import _lib
    lib, none = _lib.load(), ctypes.c_void_p(None)
    at = lambda i: ctypes.c_void_p((i + 1) << 36)
    text = lambda: lib.enatten_last_error().decode()
    for call in (lambda: lib.enatten_cache_fork(at(0), none, at(1), at(2), 2, 3, total, 16, 3, none),
                 lambda: lib.enatten_cache_reserve(at(0), none, none, 1, at(1), at(2), at(3), 2, 3, total, 16, 3, none),
                 lambda: lib.enatten_cache_compact(at(0), at(1), none, at(3), 2, 3, total, 16, 3, none)):
        rc = call()
        assert (rc not in (0, 1) and "2^30 pages" in text()) if refused else (rc == 1 and "NULL" in text())


def test_host_sides_refuse_more_pages():
    ensure_built()
    import e_natten_amd as E
    from e_natten_amd import pages as P
    there = lambda n: torch.empty(n, dtype=torch.int32, device="meta")
    table = there(6).view(2, 3)
    few, many = there(MOST), there(MOST + 1)
    for call in (E.cache_compact, P._compact_impl):
        with pytest.raises(ValueError, match="too large"):
            call(table, many, 16)
    for call in (lambda: E.cache_reserve(table, there(2), many, 16), lambda: E.cache_fork(table, there(2), many, there(2), 16)):
        with pytest.raises(ValueError, match="too large"):
            call()
    if E.ops.NATIVE_BINDING:     # (the other host side has no shapes without data)
        assert E.cache_compact(table, few, 16).shape == (MOST // 2, 3)
        E.cache_fork(table, there(2), few, there(2), 16)
