"""float16 gradients of attention over sequences at gradients far from 1: as exact as at 1, and finite where the formula's are.

The bound on an error's norm comes from the roundings that the kernels make, each taken as even over half a step u = 2^-11 (u^2 / 3 of a value's square): of the
result itself (computed exactly here, float16's smallest numbers among it), of dS, of P for the gradient of values, and of the weights that make the
outputs, which reach dS through delta.  1.5 of their root sum is allowed."""
import math

import pytest
import torch

import attention_oracle as oracle
import sapa_b200
from attention_oracle import check, offsets_of

pytestmark = pytest.mark.gpu
U = 2.0 ** -11


def _made(shape, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).half()


def _grads(q, k, v, go, off, **kw):
    q, k, v = (x.detach().clone().requires_grad_() for x in (q, k, v))
    return torch.autograd.grad(sapa_b200.packed_attention(q, k, v, off, **kw), (q, k, v), go)


def _squares(q, k, v, go, scale):
    """(exact gradient, square of the error's norm to expect) of q, k, v of one causal sequence in one group."""
    q, k, v, go = (x.double() for x in (q, k, v, go))
    hidden = ~oracle.visible(q.shape[0], k.shape[0], True, q.device)
    gq, gk, gv = torch.zeros_like(q), torch.zeros_like(k[:, 0]), torch.zeros_like(k[:, 0])
    eq = ek = ev = 0.0
    for h in range(q.shape[1]):
        p = torch.softmax((q[:, h] @ k[:, 0].T * scale).masked_fill(hidden, -math.inf), 1)
        dp = go[:, h] @ v[:, 0].T
        ds = p * (dp - (p * dp).sum(1, keepdim=True))
        gq[:, h] = scale * (ds @ k[:, 0])
        gk += scale * (ds.T @ q[:, h])
        gv += p.T @ go[:, h]
        delta = U ** 2 / 3 * (p * dp).square().sum(1)
        eq += scale ** 2 * float(U ** 2 / 3 * (ds.square() @ k[:, 0].square()).sum() + (delta * (p @ k[:, 0]).square().sum(1)).sum())
        both = U ** 2 / 3 * ds.square() + p.square() * delta[:, None]
        ek += scale ** 2 * float((both.T @ q[:, h].square()).sum())
        ev += float(((U * p).clamp(min=2.0 ** -25).masked_fill(hidden, 0).square().T / 3 @ go[:, h].square()).sum())
    return [(x, e + float((x.half().double() - x).square().sum())) for x, e in ((gq, eq), (gk[:, None], ek), (gv[:, None], ev))]


@pytest.mark.parametrize("size", [1e-4, 1e-3, 1.0, 300.0])
@pytest.mark.parametrize("dim", [64, 128])
def test_gradients_of_any_size(dim, size):
    T, share = 3000, 2
    q, k, v = _made((T, share, dim), 0, 1.5), _made((T, 1, dim), 1), _made((T, 1, dim), 2)
    go = _made((T, share, dim), 9, size)
    for name, got, (want, square) in zip(("gq", "gk", "gv"), _grads(q, k, v, go, offsets_of([T])), _squares(q, k, v, go, dim ** -0.5)):
        assert float((got.double() - want).norm()) <= 1.5 * math.sqrt(square), name


@pytest.mark.parametrize("dim", [64, 128])
def test_large_gradients_and_values(dim):
    """dS beyond float16's largest number where the gradients are not."""
    lengths, scale = [5, 3, 40, 2, 1, 100], 0.02
    T = sum(lengths)
    q, k = _made((T, 4, dim), 0), _made((T, 2, dim), 1)
    v, go = _made((T, 2, dim), 2, 8.0), _made((T, 4, dim), 9, 6000.0)
    want = oracle.packed(q, k, v, lengths, lengths, True, scale, go)
    for name, g in zip(("gq", "gk", "gv"), _grads(q, k, v, go, offsets_of(lengths), scale=scale)):
        assert float(want[name].abs().max()) < 65504
        check(g, want[name], want[name + "_tol"])


@pytest.mark.parametrize("dim", [64, 128])
def test_sequences_do_not_see_each_others_sizes(dim):
    """A sequence's gradients have the same bits beside sequences, groups and padding with gradients and values of any size."""
    lengths = [300, 70, 500]
    T = sum(lengths) + 11
    q, k, v = _made((T, 4, dim), 0), _made((T, 2, dim), 1), _made((T, 2, dim), 2)
    go = _made((T, 4, dim), 9, 1e-4)
    off = offsets_of(lengths)
    alone = [x.clone() for x in _grads(q, k, v, go, off)]
    go[300:370] *= 2.0 ** 20
    v[300:370] *= 2.0 ** 6
    go[:300, 2:] = 0
    go[870:] = 60000.0
    v[870:] = -60000.0
    for a, b in zip(_grads(q, k, v, go, off), alone):
        heads = a.shape[1] // 2
        assert torch.equal(a[:300, :heads], b[:300, :heads]) and torch.equal(a[370:], b[370:])
        assert bool((a[870:] == 0).all())
