"""float16 gradients of attention over sequences at gradients far from 1: as exact as at 1, and finite where the formula's are.  An
error's norm may be 1.5 of what the roundings to float16 lead to (attention_rounding)."""
import math

import pytest
import torch

import attention_oracle as oracle
import attention_rounding as rounding
import sapa_b200
from attention_oracle import check, offsets_of

pytestmark = pytest.mark.gpu


def _made(shape, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).half()


def _grads(q, k, v, go, off, **kw):
    q, k, v = (x.detach().clone().requires_grad_() for x in (q, k, v))
    return torch.autograd.grad(sapa_b200.packed_attention(q, k, v, off, **kw), (q, k, v), go)


@pytest.mark.parametrize("size", [1e-4, 1e-3, 1.0, 300.0])
@pytest.mark.parametrize("dim", [64, 128])
def test_gradients_of_any_size(dim, size):
    T, share = 3000, 2
    q, k, v = _made((T, share, dim), 0, 1.5), _made((T, 1, dim), 1), _made((T, 1, dim), 2)
    go = _made((T, share, dim), 9, size)
    for name, got, (want, square) in zip(("gq", "gk", "gv"), _grads(q, k, v, go, offsets_of([T])), rounding.gradients(q, k, v, go, torch.float16, True)):
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


def test_captured_and_replayed_with_other_sizes():
    """The factor of dS is found anew in every replay: other lengths, gradients and values a thousand times as large and as small."""
    T = 400
    q, k, v = (x.requires_grad_() for x in (_made((T, 4, 64), 0), _made((T, 2, 64), 1), _made((T, 2, 64), 2)))
    go, off = _made((T, 4, 64), 9), offsets_of([250, 100, 50])

    def step():
        return torch.autograd.grad(sapa_b200.packed_attention(q, k, v, off), (q, k, v), go)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i, (size, lengths) in enumerate(((1e-3, [30, 300, 70]), (1e3, [1, 2, 397]), (1.0, [0, 0, 17]))):
        go.copy_(_made((T, 4, 64), 10 + i, size))
        off.copy_(offsets_of(lengths))
        graph.replay()
        for a, b in zip(held, step()):
            assert torch.equal(a, b)


@pytest.mark.parametrize("size", [1e-4, 3000.0])
def test_many_sequences(size):
    """Hundreds of sequences, some empty, whose factors are found by warps: the bits of calls on few of them, whose factors are found by blocks."""
    lengths = [(7 * i) % 23 for i in range(900)]
    T = sum(lengths)
    q, k, v, go = _made((T, 2, 64), 0), _made((T, 1, 64), 1), _made((T, 1, 64), 2), _made((T, 2, 64), 9, size)
    off = offsets_of(lengths)
    together = _grads(q, k, v, go, off)
    for first in (0, 300, 820):
        some = off[first:first + 81].contiguous()
        rows = slice(int(some[0]), int(some[-1]))
        for a, b in zip(_grads(q, k, v, go, some), together):
            assert bool(b[rows].isfinite().all()) and torch.equal(a[rows], b[rows])


def test_no_wait_gave_up():
    from sapa_b200 import _lib
    assert _lib.wait_timeout_flags("cuda") == 0
