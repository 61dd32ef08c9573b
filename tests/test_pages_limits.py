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
    for holders, error in ((there(MOST + 1), ValueError), (there(MOST), None)):
        for call in (lambda: E.cache_compact(table, holders, 16), lambda: P._compact_impl(table, holders, 16),
                     lambda: E.cache_reserve(table, there(2), holders, 16), lambda: E.cache_fork(table, there(2), holders, there(2), 16)):
            if error:
                with pytest.raises(error, match="too large"):
                    call()
            elif E.ops.NATIVE_BINDING:
                try:
                    call()
                except RuntimeError as e:     # (the ctypes side has no shapes without data)
                    assert "GPU" in str(e)
