"""Paged caches whose tables are wrong in more than one place."""
import pytest
import torch

import attention_oracle as oracle
import sapa_b200
from attention_oracle import Cache, check, offsets_of

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("page", [16, 24])
@pytest.mark.parametrize("new", [1, 30, 200])
def test_a_bad_page_and_a_table_that_ends_early(new, page, dtype):
    """A page outside the cache in the first tile, and a length beyond the table's end: every token that sees either is NaN, the sequences beside it are whole."""
    t, keys = TYPES[dtype], [240, 240, 240]
    g = torch.Generator(device="cuda").manual_seed(3)
    q, k, v = (torch.randn(n, h, 64, generator=g, device="cuda").to(t) for n, h in ((3 * new, 4), (720, 2), (720, 2)))
    c = Cache(k, v, keys, page, table_extra=0)
    want = oracle.packed(q, k, v, [new] * 3, keys, True, 0.125)
    c.table[1, 1] = c.key.shape[0] + 5
    lengths = c.lengths.clone()
    lengths[1] += 7                                      # the last 7 positions have no entry
    for _ in range(10):
        out = sapa_b200.paged_attention(q, c.key, c.value, c.table, lengths, offsets_of([new] * 3))
        for b in (0, 2):
            rows = slice(b * new, (b + 1) * new)
            check(out[rows], want["out"][rows], want["out_tol"][rows])
        assert bool(out[new:2 * new].isnan().all())      # each sees position `page` at least


def test_no_wait_gave_up():
    from sapa_b200 import _lib
    assert _lib.wait_timeout_flags("cuda") == 0
