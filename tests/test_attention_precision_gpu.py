"""What the forward of a training step hands to its gradients beyond the outputs' own type, and what that is worth."""
import math

import pytest
import torch

from attention_oracle import offsets_of

pytestmark = pytest.mark.gpu


def _forward(q, k, v, lengths, key_lengths, causal):
    from sapa_b200 import _lib
    return _lib.load_host().packed_attention_forward(q, k, v, offsets_of(lengths), offsets_of(key_lengths), causal, None)


@pytest.mark.parametrize("tokens, keys, causal", [(5000, 5000, True), (1, 7919, False), (3, 30011, False), (40, 257, False)])
def test_logarithms_of_sums(tokens, keys, causal):
    """Queries of zero: all weights are 1, sums are whole numbers and exact, and lse with what its rounding left out is their logarithm: log2 and the product with
    log(2) in float64, and half a step of the float32 number that holds the rest of a number below 16, 2^-24 * 2^-24 * 16 in all."""
    q = torch.zeros(tokens, 2, 64, device="cuda")
    k, v = (torch.randn(keys, 1, 64, device="cuda") for _ in range(2))
    out, lse, low, _ = _forward(q, k, v, [tokens], [keys], causal)
    count = (torch.arange(tokens, device="cuda", dtype=torch.float64) + 1 if causal else torch.full((tokens,), float(keys), device="cuda", dtype=torch.float64))[:, None]
    assert float((lse.double() + low.double() - count.log()).abs().max()) <= 2.0 ** -44
