"""Attention over sequences under traces, forward-mode differentiation and torch.func: recorded as itself, or refused, as the other operators are."""
import pytest
import torch

import sapa_b200
from attention_oracle import Cache, offsets_of

pytestmark = pytest.mark.gpu


def _inputs(seed=0, T=40, S=40):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.randn(n, h, 64, generator=g, device="cuda") for n, h in ((T, 4), (S, 2), (S, 2))]


def _transforms(op, x):
    """What torch.func and forward mode do with `op` of one tensor."""
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda t: op(t).sum())(x)
    with pytest.raises(RuntimeError):
        torch.func.vmap(op)(x[None])
    with torch.autograd.forward_ad.dual_level(), pytest.raises((RuntimeError, NotImplementedError)):
        op(torch.autograd.forward_ad.make_dual(x, torch.ones_like(x)))


@pytest.mark.parametrize("own_keys", [False, True])
def test_packed(own_keys):
    off, koff = offsets_of([25, 15]), offsets_of([10, 30]) if own_keys else None

    def op(q, k, v, off, *koff):
        return sapa_b200.packed_attention(q, k, v, off, *koff)
    rest = (off,) if koff is None else (off, koff)
    x = [t.requires_grad_() for t in _inputs()]
    want = torch.autograd.grad(op(*x, *rest).square().sum(), x)
    traced = torch.jit.trace(op, (*[t.detach().clone().requires_grad_() for t in x], *rest), check_trace=False)
    other, turned = [t.requires_grad_() for t in _inputs(5)], (offsets_of([5, 35]), *rest[1:])
    assert torch.equal(traced(*other, *turned), op(*other, *turned))
    for a, b in zip(torch.autograd.grad(traced(*x, *rest).square().sum(), x), want):
        assert torch.equal(a, b)
    q, k, v = (t.detach() for t in x)
    _transforms(lambda t: op(t, k, v, *rest), q)
    _transforms(lambda t: op(q, k, t, *rest), v)


def _step(q, k, v, key_pages, value_pages, table, lengths, off):
    sapa_b200.paged_write(k, v, key_pages, value_pages, table, lengths, off)
    return sapa_b200.paged_attention(q, key_pages, value_pages, table, lengths, off)


def _cache(seed):
    _, k, v = _inputs(seed, S=130)
    return Cache(k, v, [100, 30], 16)


def test_paged_steps_are_recorded():
    """A traced step writes into the cache it is called with and reads that: other tokens, another cache, other lengths."""
    new = offsets_of([3, 1])

    def write_alone(k, v, *rest):
        sapa_b200.paged_write(k, v, *rest)
        return k + 1
    for fn, tensors in ((_step, _inputs(1, 4, 4)), (write_alone, _inputs(1, 4, 4)[1:])):
        c = _cache(2)
        traced = torch.jit.trace(fn, (*tensors, c.key, c.value, c.table, c.lengths, new), check_trace=False)
        for seed in (3, 4, 5):
            other = _inputs(seed, 4, 4)[-len(tensors):]
            here, there = _cache(seed), _cache(seed)
            lengths = here.lengths - seed
            want = fn(*other, here.key, here.value, here.table, lengths, new)
            assert torch.equal(traced(*other, there.key, there.value, there.table, lengths, new), want)
            for a, b in ((here.key, there.key), (here.value, there.value)):
                assert torch.equal(a.nan_to_num(9.0), b.nan_to_num(9.0))


def test_paged_refusals():
    q, k, v = _inputs(1, 4, 4)
    new, c = offsets_of([3, 1]), _cache(2)
    rest = (c.table, c.lengths, new)
    kept = c.key.clone()
    _transforms(lambda t: sapa_b200.paged_attention(t, c.key, c.value, *rest), q)
    _transforms(lambda t: sapa_b200.paged_attention(q, c.key, t, *rest), c.value)

    def write(t):
        sapa_b200.paged_write(t, v, c.key, c.value, *rest)
        return t
    _transforms(write, k)
    assert torch.equal(c.key.nan_to_num(9.0), kept.nan_to_num(9.0))
    with pytest.raises(NotImplementedError):
        torch.jit.trace(_step, (q.requires_grad_(), k, v, c.key, c.value, *rest), check_trace=False)
    with pytest.raises(NotImplementedError):
        torch.jit.trace(lambda k, v: sapa_b200.paged_write(k, v, c.key, c.value, *rest), (k.requires_grad_(), v), check_trace=False)


def test_no_wait_gave_up():
    from sapa_b200 import _lib
    assert _lib.wait_timeout_flags("cuda") == 0
