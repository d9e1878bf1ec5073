"""Sizes next to the limit of 32-bit positions, without a GPU: refused before any kernel is launched."""
import ctypes

import pytest

from test_attention import _arguments

LIMIT = 0x7fffff00


@pytest.mark.parametrize("kw", [dict(tokens=LIMIT), dict(keys=LIMIT), dict(tokens=0x7fffffff), dict(keys=0x7fffffff),
                                dict(page_table=4096, key_lengths=4096, pages=1, page=1, max_pages=LIMIT)])
def test_more_rows_than_a_tile_can_end_at(kw):
    from sapa_b200 import _lib
    h = _lib.lib()
    for dtype in (0, 1, 2):
        ref = ctypes.byref(_arguments(**kw))
        assert h.sapa_attention_forward(ref, None, 0, dtype, None) == -5 and b"2^31" in h.sapa_last_error()
        assert h.sapa_attention_workspace(ref, dtype) == 0 and h.sapa_attention_backward_workspace(ref, dtype) == 0
        assert h.sapa_attention_backward(ref, 4096, 64, 16, 4096, 4096, 4096, 4096, 1 << 40, dtype, None) == -5


def test_one_fewer_is_taken():
    from sapa_b200 import _lib
    h = _lib.lib()
    assert h.sapa_attention_backward_workspace(ctypes.byref(_arguments(tokens=LIMIT - 1, keys=LIMIT - 1)), 1) > 3 * 4 * 4 * (LIMIT - 1)
