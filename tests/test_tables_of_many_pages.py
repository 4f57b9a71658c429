"""Block tables that are as long as 32-bit counting allows: what lies beyond is refused before anything is launched."""
import ctypes as C

from tests.test_decode_arguments import P

MOST = (1 << 31) - 512  # pages of a sequence: a wave's steps over its entries, and the entries rounded up for the waves, stay below 2^31


def test_longer_tables_are_refused(et):
    size = C.c_size_t()
    for pages, status in ((MOST, 0), (MOST + 1, -2), ((1 << 31) - 128, -2), ((1 << 31) - 1, -2)):
        assert et.lib().et_kv_tables_workspace(pages, 1, C.byref(size)) == status, pages
    for pages in (MOST + 1, (1 << 31) - 128):
        assert et.lib().et_kv_tables(P, P, pages, 1, 8, None, None, None, 1, 1, 0, 0, P, P, P, None, P, 1 << 30, None) == -2
        assert b"max_pages" in et.lib().et_last_error()
