"""What lies beside the tokens of a sequence - padding of one tensor alone, heads of the next group, the rest of a tile - has no part in its
gradients, whatever it holds."""
import math

import pytest
import torch

import attention_oracle as oracle
import sapa_b200
from attention_oracle import check, offsets_of

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _made(shape, dtype, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def _step(q, k, v, go, off, koff=None, **kw):
    q, k, v = (x.detach().clone().requires_grad_() for x in (q, k, v))
    out = sapa_b200.packed_attention(q, k, v, off, koff, **kw)
    return (out.detach(), *torch.autograd.grad(out, (q, k, v), go))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("which", ["query", "grad_out", "both"])
def test_padding_of_one_tensor(which, dim, dtype):
    """Rows of no sequence in the query alone, in its gradient alone (zeros or numbers in the other) and in both."""
    lengths, start, t = [150, 37], 5, TYPES[dtype]
    T = start + sum(lengths) + 30
    q, go = (_made((T, 4, dim), t, s) for s in (0, 9))
    k, v = (_made((T, 2, dim), t, s) for s in (1, 2))
    off = offsets_of(lengths, start)
    outside = torch.ones(T, dtype=torch.bool, device="cuda")
    outside[start:start + sum(lengths)] = False
    want = oracle.packed(q, k, v, lengths, lengths, True, dim ** -0.5, go, start, start)
    clean = _step(q, k, v, go, off)
    for name, x in zip(("out", "gq", "gk", "gv"), clean):
        check(x, want[name], want[name + "_tol"])
    for rest in (0.0, 1.0):
        for what in (math.nan, math.inf, -math.inf):
            qq, gg = q.clone(), go.clone()
            qq[outside] = what if which != "grad_out" else rest
            gg[outside] = what if which != "query" else rest
            for a, b in zip(_step(qq, k, v, gg, off), clean):
                assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("dim", [40, 64])
@pytest.mark.parametrize("which", ["query", "grad_out"])
def test_heads_of_the_next_group(which, dim, dtype):
    """More query heads to a key head than a tile has rows: the last tile of a token reaches into the heads of the next key head."""
    T, share, t = 30, 70, TYPES[dtype]
    q, go = (_made((T, 2 * share, dim), t, s) for s in (0, 9))
    k, v = (_made((T, 2, dim), t, s) for s in (1, 2))
    off = offsets_of([18, 12])
    clean = _step(q, k, v, go, off)
    for what in (math.nan, math.inf):
        qq, gg = q.clone(), go.clone()
        (qq if which == "query" else gg)[7, share + 5, 3] = what
        out, gq, gk, gv = _step(qq, k, v, gg, off)
        assert torch.equal(gk[:, 0], clean[2][:, 0]) and torch.equal(gv[:, 0], clean[3][:, 0])
        assert torch.equal(gk[18:], clean[2][18:]) and torch.equal(gv[18:], clean[3][18:])
        assert not bool(gv[:8, 1, 3].isfinite().any())


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads, groups", [(3, 1), (12, 2), (5, 1), (7, 1), (70, 1)])
def test_key_without_weight(heads, groups, dim, dtype):
    """A key whose scores are all -infinity has gradients of zero, also where the query heads that share it do not divide a tile."""
    T, t = 200, TYPES[dtype]
    q = _made((T, heads, dim), t, 0).abs()
    k, v = (_made((T, groups, dim), t, s).abs() for s in (1, 2))
    go = _made((T, heads, dim), t, 9)
    keep = [j for j in range(T) if j != 50]
    want = oracle.packed(q, k[keep], v[keep], [T], [T - 1], False, dim ** -0.5, go)
    k[50, :, 5] = -math.inf
    out, gq, gk, gv = _step(q, k, v, go, offsets_of([T]), causal=False)
    check(out, want["out"], want["out_tol"])
    for name, x in (("gk", gk), ("gv", gv)):
        assert bool((x[50] == 0).all())
        check(x[keep], want[name], want[name + "_tol"])
    rest = [c for c in range(dim) if c != 5]             # there 0 * infinity
    check(gq[..., rest], want["gq"][..., rest], want["gq_tol"][..., rest])


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("T", [90, 3000])
def test_no_sequence(T, dtype):
    """Offsets of one entry: every row is of no sequence, however many there are."""
    q, go = (_made((T, 8, 64), TYPES[dtype], s) for s in (0, 9))
    k, v = (_made((T, 2, 64), TYPES[dtype], s) for s in (1, 2))
    with torch.no_grad():
        assert bool((sapa_b200.packed_attention(q, k, v, offsets_of([])) == 0).all())
    for x in _step(q, k, v, go, offsets_of([])):
        assert bool((x == 0).all())


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
def test_infinite_values_at_the_diagonal_of_two_row_tiles(dim, dtype):
    """Tiles that both row tiles of a block clean: the tokens from an infinite value on have it, the others not a bit of it, each time."""
    T, t = 700, TYPES[dtype]
    q = _made((T, 4, dim), t, 0)
    k, v = (_made((T, 2, dim), t, s) for s in (1, 2))
    off = offsets_of([T])
    with torch.no_grad():
        clean = sapa_b200.packed_attention(q, k, v, off)
        at = [63, 64, 127, 130, 255, 300, 500, 639, 699]
        for i, j in enumerate(at):
            v[j, 1, i] = math.inf if i % 2 == 0 else -math.inf
        for _ in range(50):
            out = sapa_b200.packed_attention(q, k, v, off)
            assert torch.equal(out[:, :2], clean[:, :2]) and torch.equal(out[:, 2:, len(at):], clean[:, 2:, len(at):])
            for i, j in enumerate(at):
                assert torch.equal(out[:j, 2:, i], clean[:j, 2:, i]) and bool((out[j:, 2:, i] == v[j, 1, i]).all())


def test_no_wait_gave_up():
    from sapa_b200 import _lib
    assert _lib.wait_timeout_flags("cuda") == 0
