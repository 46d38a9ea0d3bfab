"""The longest text that the attention counts in 32 bits: tiles of 128 keys, the last one's end included.  Without a device."""
import ctypes as C

import pytest

from test_cache_refusals import CTX, NOMEM, P, UNSUPPORTED, lib, paged   # noqa: F401 (a fixture)


@pytest.mark.parametrize("page", [8, 16, 64, 128])
def test_tables_up_to_it(lib, page):   # noqa: F811
    def call(entries):
        cache = paged(page_size=page, table_n=entries, table_ld=entries)
        return lib.q38b_attention(CTX, C.byref(cache), P + 4096, 2, 256, 64, 4, 0.125, P, 2, 256, 64, None, 5, P, 15, None)
    longest = (2 ** 31 - 128) // page
    assert call(longest) == NOMEM and call(longest // 2) == NOMEM      # (counted; refused for its work area)
    if (longest + 1) * page < 2 ** 31:
        assert call(longest + 1) == UNSUPPORTED and call((2 ** 31 - 1) // page) == UNSUPPORTED


def test_what_is_counted():
    """The kernel's own sums at that length, in wrapping 32-bit arithmetic: tiles of keys, and the end of the last one.  128 more and both are wrong."""
    wrap = lambda x: (x + 2 ** 31) % 2 ** 32 - 2 ** 31   # noqa: E731
    for seen, right in ((2 ** 31 - 128, True), (2 ** 31 - 127, False), (2 ** 31 - 8, False)):
        units = max(1, wrap(seen + 127) // 128)
        last = (units - 1) * 128
        assert (units == -(-seen // 128) and last < seen <= wrap(last + 128)) == right
