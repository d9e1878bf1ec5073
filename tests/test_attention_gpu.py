"""Attention over packed sequences and over paged caches against float64, at the sizes and masks where it can go wrong."""
import math

import pytest
import torch

import attention_oracle as oracle
import sapa_b200
from attention_oracle import Cache, check, offsets_of

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _made(shape, dtype, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def _inputs(T, S, heads, groups, dim, dtype, seed=0):
    return _made((T, heads, dim), dtype, seed, 1.5), _made((S, groups, dim), dtype, seed + 1), _made((S, groups, dim), dtype, seed + 2)


SHAPES = [  # lengths, heads, groups, dim
    ([1], 1, 1, 8), ([1, 1, 1], 4, 2, 64), ([7, 0, 1, 130], 4, 2, 64), ([64, 65, 63], 6, 2, 40), ([128, 127, 129, 1], 2, 2, 128), ([257], 5, 1, 96),
    ([300, 2, 0, 0, 77], 8, 8, 32), ([513], 16, 2, 80), ([33] * 40, 3, 3, 16), ([5, 250], 70, 1, 64), ([4, 9], 128, 1, 128), ([700, 20], 12, 4, 128)]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lengths, heads, groups, dim", SHAPES)
def test_packed(lengths, heads, groups, dim, causal, dtype):
    T = sum(lengths)
    q, k, v = (t.requires_grad_() for t in _inputs(T, T, heads, groups, dim, TYPES[dtype]))
    go = _made((T, heads, dim), TYPES[dtype], 9)
    scale = 1 / math.sqrt(dim)
    out = sapa_b200.packed_attention(q, k, v, offsets_of(lengths), causal=causal)
    want = oracle.packed(q.detach(), k.detach(), v.detach(), lengths, lengths, causal, scale, go)
    check(out.detach(), want["out"], want["out_tol"])
    with torch.no_grad():
        assert torch.equal(sapa_b200.packed_attention(q, k, v, offsets_of(lengths), causal=causal), out)
    for name, g in zip(("gq", "gk", "gv"), torch.autograd.grad(out, (q, k, v), go)):
        check(g, want[name], want[name + "_tol"])


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lengths, keys", [([3, 200], [200, 3]), ([5, 0, 130, 1], [0, 4, 131, 500]), ([260], [129]), ([1], [1000])])
def test_keys_of_other_lengths(lengths, keys, causal, dtype):
    """Tokens that see no key get 0 and give no gradient; rows in front of the first and behind the last sequence are 0."""
    T, S, start, key_start = sum(lengths) + 9, sum(keys) + 7, 4, 3
    q, k, v = (t.requires_grad_() for t in _inputs(T, S, 4, 2, 64, TYPES[dtype]))
    go = _made((T, 4, 64), TYPES[dtype], 9)
    out = sapa_b200.packed_attention(q, k, v, offsets_of(lengths, start), offsets_of(keys, key_start), causal=causal, scale=0.2)
    want = oracle.packed(q.detach(), k.detach(), v.detach(), lengths, keys, causal, 0.2, go, start, key_start)
    check(out.detach(), want["out"], want["out_tol"])
    for name, g in zip(("gq", "gk", "gv"), torch.autograd.grad(out, (q, k, v), go)):
        check(g, want[name], want[name + "_tol"])


@pytest.mark.parametrize("dtype", list(TYPES))
def test_mostly_padding(dtype):
    """Two short sequences somewhere in a large padded tensor full of NaN: zeros around them, in the outputs and in every gradient."""
    T, start, lengths = 3001, 700, [5, 40]
    q, k, v = (x.requires_grad_() for x in _inputs(T, T, 6, 3, 40, TYPES[dtype]))
    go = _made((T, 6, 40), TYPES[dtype], 9)
    with torch.no_grad():
        for x in (q, k, v, go):
            x[:start] = x[start + 45:] = math.nan
    out = sapa_b200.packed_attention(q, k, v, offsets_of(lengths, start))
    want = oracle.packed(q.detach(), k.detach(), v.detach(), lengths, lengths, True, 40 ** -0.5, go, start, start)
    check(out.detach(), want["out"], want["out_tol"])
    for name, g in zip(("gq", "gk", "gv"), torch.autograd.grad(out, (q, k, v), go)):
        check(g, want[name], want[name + "_tol"])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_strides(dtype):
    """Parts of one projection's output, heads before tokens, an unaligned view, and broadcast heads: the numbers of dense tensors."""
    lengths, T, t = [70, 131], 201, TYPES[dtype]
    off = offsets_of(lengths)
    together = _made((T, 4 + 2 + 2, 64), t, 0)
    q, k, v = together.split((4, 2, 2), 1)
    want = sapa_b200.packed_attention(q.contiguous(), k.contiguous(), v.contiguous(), off)
    assert torch.equal(sapa_b200.packed_attention(q, k, v, off), want)
    turned = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v)]
    assert torch.equal(sapa_b200.packed_attention(*turned, off), want)
    odd = torch.empty(T * 4 * 64 + 1, dtype=t, device="cuda")[1:].view(T, 4, 64).copy_(q)
    assert torch.equal(sapa_b200.packed_attention(odd, k, v, off), want)
    one_k, one_v = (x[:, :1].contiguous().requires_grad_() for x in (k, v))
    go = _made((T, 4, 64), t, 3).transpose(0, 1).contiguous().transpose(0, 1)
    wide = sapa_b200.packed_attention(q, one_k.expand(-1, 4, -1), one_v.expand(-1, 4, -1), off)
    shared = sapa_b200.packed_attention(q, one_k, one_v, off)
    w = oracle.packed(q, one_k.detach(), one_v.detach(), lengths, lengths, True, 0.125, go)
    for out in (wide, shared):
        check(out.detach(), w["out"], w["out_tol"])
    for name, g in zip(("gk", "gv"), torch.autograd.grad(shared, (one_k, one_v), go)):
        check(g, w[name], w[name + "_tol"])
    # of a broadcast input the four heads' gradients are rounded and then added: half a step of each, of their sums, and of the shared form
    apart = oracle.packed(q, one_k.detach().expand(-1, 4, -1), one_v.detach().expand(-1, 4, -1), lengths, lengths, True, 0.125, go)
    u = oracle.HALF_STEP[t]
    for name, g in zip(("gk", "gv"), torch.autograd.grad(wide, (one_k, one_v), go)):
        tol = apart[name + "_tol"].sum(1, keepdim=True) + 4 * u * apart[name].abs().sum(1, keepdim=True)
        check(g, w[name], tol)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("dim", [64, 128])
def test_what_is_not_seen_has_no_part(dim, dtype):
    """Infinities and NaN in later tokens, in other sequences and behind the last one change no bit of what does not see them, forward and backward."""
    lengths, t = [150, 40, 300], TYPES[dtype]
    T = sum(lengths) + 20
    off = offsets_of(lengths)
    q, k, v = _inputs(T, T, 4, 2, dim, t)
    go = _made((T, 4, dim), t, 9)

    def run(q, k, v, go):
        q, k, v = (x.clone().requires_grad_() for x in (q, k, v))
        out = sapa_b200.packed_attention(q, k, v, off)
        return (out.detach(), *torch.autograd.grad(out, (q, k, v), go))
    clean = run(q, k, v, go)
    for x in (q, k, v, go):
        x[sum(lengths):] = math.nan                      # of no sequence
    bad = (100, 190 + 130)                               # tokens of the first and third sequence
    for i, (x, what) in enumerate([(k, math.nan), (v, math.nan), (v, math.inf), (v, -math.inf), (k, math.inf), (q, math.nan), (q, math.inf), (go, math.nan), (go, math.inf)]):
        for token in bad:
            y = [z.clone() for z in (q, k, v, go)]
            j = [z is x for z in (q, k, v, go)].index(True)
            y[j][token, 1, 3] = what
            got = run(*y)
            begin, end = (0, 150) if token == 100 else (190, 490)
            before, behind = slice(begin, token), slice(token, end)
            others = [r for r in ((0, 150), (150, 190), (190, 490), (490, T)) if r[0] != begin]
            for a, c in zip(got, clean):
                for lo, hi in others:
                    assert torch.equal(a[lo:hi], c[lo:hi])
            out, gq, gk, gv = got
            if x is k or x is v:                         # key head 1: query heads 2, 3 from the token on
                assert torch.equal(out[before], clean[0][before]) and torch.equal(gq[before], clean[1][before])
                assert torch.equal(out[behind, :2], clean[0][behind, :2])
                assert torch.equal(gk[begin:end, :1], clean[2][begin:end, :1]) and torch.equal(gv[begin:end, :1], clean[3][begin:end, :1])
                if math.isnan(what):
                    seen = out[behind, 2:] if x is k else out[behind, 2:, 3]
                    assert bool(seen.isnan().all())
                elif x is v:
                    assert bool((out[behind, 2:, 3] == what).all())
                    rest = [c for c in range(dim) if c != 3]
                    assert torch.equal(out[behind][:, :, rest], clean[0][behind][:, :, rest])
            else:                                        # query head 1: key head 0 up to the token
                after = slice(token + 1, end)
                assert torch.equal(gk[after], clean[2][after]) and torch.equal(gv[after], clean[3][after])
                assert torch.equal(gk[begin:end, 1:], clean[2][begin:end, 1:]) and torch.equal(gv[begin:end, 1:], clean[3][begin:end, 1:])
                rows = torch.arange(begin, end) != token
                for a, c in ((out, clean[0]), (gq, clean[1])):
                    assert torch.equal(a[begin:end][rows], c[begin:end][rows])
                reached = gv[begin:token + 1, 0] if x is q else gv[begin:token + 1, 0, 3]
                assert not bool(reached.isfinite().any())


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_far_scores(dtype):
    """Scores hundreds apart, the largest last, and rows of equal scores."""
    t, T = TYPES[dtype], 400
    q, k, v = _inputs(T, T, 2, 1, 64, t)
    k = (k.float() * torch.linspace(0.1, 12, T, device="cuda")[:, None, None]).to(t)
    q[50:60] = 0
    want = oracle.packed(q, k, v, [T], [T], True, 1.0)
    check(sapa_b200.packed_attention(q, k, v, offsets_of([T]), scale=1.0), want["out"], want["out_tol"])
    want = oracle.packed(q, k, v, [T], [T], True, -0.3)
    check(sapa_b200.packed_attention(q, k, v, offsets_of([T]), scale=-0.3), want["out"], want["out_tol"])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_gradients_against_differences(dtype):
    """<gradient, direction> against the difference of the oracle's outputs along it."""
    lengths, t = [37, 5], TYPES[dtype]
    q, k, v = (x.requires_grad_() for x in _inputs(42, 42, 4, 2, 32, t))
    go = _made((42, 4, 32), t, 5)
    grads = torch.autograd.grad(sapa_b200.packed_attention(q, k, v, offsets_of(lengths)), (q, k, v), go)
    w = oracle.packed(q.detach(), k.detach(), v.detach(), lengths, lengths, True, 32 ** -0.5, go)
    step = 1e-5
    for i, name in enumerate(("gq", "gk", "gv")):
        d = _made(grads[i].shape, torch.float32, 20 + i).double()
        sides = []
        for s in (step, -step):
            x = [a.detach().double() for a in (q, k, v)]
            x[i] = x[i] + s * d
            out = _plain64(*x, lengths, 32 ** -0.5)
            sides.append((out * go.double()).sum())
        numeric = (sides[0] - sides[1]) / (2 * step)
        # the third derivative is of the order of the sums' magnitudes: 1e-8 of them
        tol = (w[name + "_tol"] * d.abs()).sum() + 1e-8 * (w[name].abs() * d.abs()).sum() + 1e-6
        assert abs(float((grads[i].double() * d).sum() - numeric)) <= float(tol)


def _plain64(q, k, v, lengths, scale):
    outs, at = [], 0
    share = q.shape[1] // k.shape[1]
    for n in lengths:
        kk, vv = (x[at:at + n].repeat_interleave(share, 1) for x in (k, v))
        s = torch.einsum("ihd,jhd->hij", q[at:at + n], kk) * scale
        s = s.masked_fill(~oracle.visible(n, n, True, q.device), -math.inf)
        outs.append(torch.einsum("hij,jhd->ihd", torch.softmax(s, -1), vv))
        at += n
    return torch.cat(outs)


# ---------------------------------------------------------------------------------- paged caches
PAGED = [  # new tokens, keys, heads, groups, dim, page
    ([1], [1], 1, 1, 8, 16), ([1, 1, 1, 1], [5, 0, 300, 1025], 8, 2, 64, 16), ([1] * 9, [700, 1, 16, 17, 15, 128, 129, 64, 2000], 32, 8, 128, 64),
    ([5, 1, 0, 130], [5, 77, 40, 400], 4, 2, 64, 32), ([257, 3], [300, 1000], 5, 1, 96, 128), ([40], [33], 4, 4, 128, 8), ([2, 2], [600, 3], 12, 4, 40, 1),
    ([1, 7], [100, 100], 4, 2, 64, 24), ([3, 200], [500, 201], 6, 2, 80, 256), ([1, 1], [4000, 3000], 16, 1, 128, 100), ([20, 1], [900, 30], 128, 1, 64, 16)]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("layout", ["slots", "heads", "both"])
@pytest.mark.parametrize("new, keys, heads, groups, dim, page", PAGED)
def test_paged(new, keys, heads, groups, dim, page, layout, dtype):
    q, k, v = _inputs(sum(new), sum(keys), heads, groups, dim, TYPES[dtype])
    c = Cache(k, v, keys, page, layout=layout)
    want = oracle.packed(q, k, v, new, keys, True, 1 / math.sqrt(dim))
    out = sapa_b200.paged_attention(q, c.key, c.value, c.table, c.lengths, offsets_of(new))
    check(out, want["out"], want["out_tol"])
    if layout == "slots":
        want = oracle.packed(q, k, v, new, keys, False, 0.1)
        check(sapa_b200.paged_attention(q, c.key, c.value, c.table, c.lengths, offsets_of(new), causal=False, scale=0.1), want["out"], want["out_tol"])


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("dim", [64, 128])
def test_many_items_to_a_block(dim, dtype):
    """More sequences than SMs, of one to eight tiles of keys, and few sequences whose keys are split into parts of that many: every
    block goes through several items of every length."""
    for new, keys, groups in (([1] * 160, [1 + 7 * i % 1000 for i in range(160)], 4), ([3 + i % 40 for i in range(90)], [60 + 11 * i % 900 for i in range(90)], 4),
                              ([300 + 13 * i for i in range(20)], [300 + 13 * i for i in range(20)], 4), ([1], [8192], 8), ([2, 1], [6000, 800], 2), ([200], [5000], 4)):
        q, k, v = _inputs(sum(new), sum(keys), 2 * groups, groups, dim, TYPES[dtype])
        c = Cache(k, v, keys, 16)
        want = oracle.packed(q, k, v, new, keys, True, dim ** -0.5)
        for _ in range(2):
            check(sapa_b200.paged_attention(q, c.key, c.value, c.table, c.lengths, offsets_of(new)), want["out"], want["out_tol"])
            check(sapa_b200.packed_attention(q, k, v, offsets_of(new), offsets_of(keys)), want["out"], want["out_tol"])
    from sapa_b200 import _lib
    assert _lib.wait_timeout_flags("cuda") == 0


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("page", [16, 24, 128])
def test_pages_outside_the_cache(page, dtype):
    """Tokens that see a position without a page get NaN, the others their numbers; rows of no sequence are 0."""
    new, keys = [1, 60, 1, 1], [300, 300, 400, 90]
    q, k, v = _inputs(sum(new) + 5, sum(keys), 4, 2, 64, TYPES[dtype])
    c = Cache(k, v, keys, page, table_extra=0)
    want = oracle.packed(q, k, v, new, keys, True, 0.125)
    off = offsets_of(new)
    first = 270 // page                                  # the page of position 270 of the second sequence
    c.table[1, first] = c.key.shape[0]
    c.table[2, 0] = -1
    lengths = c.lengths.clone()
    lengths[3] = c.table.shape[1] * page + 1             # longer than the table
    out = sapa_b200.paged_attention(q, c.key, c.value, c.table, lengths, off)
    clear = max(0, first * page - 240)                   # tokens of the second sequence that do not see it
    check(out[:1 + clear], want["out"][:1 + clear], want["out_tol"][:1 + clear])
    assert bool(out[1 + clear:63].isnan().all())
    assert bool((out[63:] == 0).all())


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_write(dtype):
    new, keys, page = [1, 0, 70, 5, 3], [40, 9, 70, 300, 2], 16
    T = sum(new) + 4
    k, v = (_made((T, 2, 40), TYPES[dtype], s) for s in (0, 1))
    old = _made((sum(keys), 2, 40), TYPES[dtype], 3)
    for layout in ("slots", "heads", "both"):
        c = Cache(old, old, keys, page, layout=layout, fill=3.0)
        want_k, want_v = c.key.clone(), c.value.clone()
        table = c.table.clone()
        table[3, 18] = c.key.shape[0]                    # positions 288 on, where its new tokens go, have no page
        at = 0
        for b, (n, m) in enumerate(zip(new, keys)):
            for i in range(n):
                p = m - n + i
                page_of = int(table[b, p // page]) if p >= 0 else -1
                if 0 <= page_of < c.key.shape[0]:
                    want_k[page_of, p % page], want_v[page_of, p % page] = k[at + i], v[at + i]
            at += n
        sapa_b200.paged_write(k, v, c.key, c.value, table, c.lengths, offsets_of(new))
        assert torch.equal(c.key, want_k) and torch.equal(c.value, want_v)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_prompt_then_tokens(dtype):
    """As a program uses them: prompts through the packed form, their keys into the cache, then a chunk and single tokens over it."""
    t, page, dim = TYPES[dtype], 16, 64
    lengths = [50, 129]
    T = sum(lengths)
    total = [60, 135]
    q, k, v = _inputs(sum(total), sum(total), 4, 2, dim, t)
    seq = [slice(0, 60), slice(60, 195)]
    full = oracle.packed(q, k, v, total, total, True, dim ** -0.5)
    pages = 30
    kc, vc = (torch.full((pages, page, 2, dim), math.nan, dtype=t, device="cuda") for _ in range(2))
    table = torch.randperm(pages, generator=torch.Generator().manual_seed(1))[:2 * 9].view(2, 9).to("cuda", torch.int32)

    def part(x, lo, hi):
        return torch.cat([x[s][a:b] for s, a, b in zip(seq, lo, hi)])

    def step(lo, hi):
        off, have = offsets_of([b - a for a, b in zip(lo, hi)]), torch.tensor(hi, dtype=torch.int32, device="cuda")
        sapa_b200.paged_write(part(k, lo, hi), part(v, lo, hi), kc, vc, table, have, off)
        return sapa_b200.paged_attention(part(q, lo, hi), kc, vc, table, have, off)
    lo, hi = [0, 0], lengths
    prompt = sapa_b200.packed_attention(part(q, lo, hi), part(k, lo, hi), part(v, lo, hi), offsets_of(lengths))
    check(prompt, part(full["out"], lo, hi), part(full["out_tol"], lo, hi))
    assert step(lo, hi).shape == prompt.shape            # the prompt's keys are in the cache now
    lo, hi = hi, [55, 131]
    while lo != total:
        check(step(lo, hi), part(full["out"], lo, hi), part(full["out_tol"], lo, hi))
        lo, hi = hi, [min(n, h + 1) for n, h in zip(total, hi)]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("tokens, keys, heads, groups, dim", [(1000, 1000, 4, 4, 128), (385, 385, 4, 2, 64), (150, 611, 2, 1, 72), (611, 129, 3, 1, 24), (40, 9000, 1, 1, 64), (9000, 40, 1, 1, 64)])
def test_gradients_of_few_long_sequences(tokens, keys, heads, groups, dim, causal):
    """float32: blocks in clusters share the tiles of one item, so there are several sums to join; twice the same bits."""
    q, k, v = (t.requires_grad_() for t in _inputs(tokens, keys, heads, groups, dim, torch.float32))
    go = _made((tokens, heads, dim), torch.float32, 9)
    out = sapa_b200.packed_attention(q, k, v, offsets_of([tokens]), offsets_of([keys]), causal=causal)
    want = oracle.packed(q.detach(), k.detach(), v.detach(), [tokens], [keys], causal, 1 / math.sqrt(dim), go)
    first = torch.autograd.grad(out, (q, k, v), go, retain_graph=True)
    for name, g, again in zip(("gq", "gk", "gv"), first, torch.autograd.grad(out, (q, k, v), go)):
        check(g, want[name], want[name + "_tol"])
        assert torch.equal(g, again)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_more_sequences_than_are_sorted(dtype):
    """Hundreds of sequences, some empty, forward, backward and over a cache."""
    lengths = [(7 * i) % 23 for i in range(700)]
    T = sum(lengths)
    q, k, v = (x.requires_grad_() for x in _inputs(T, T, 4, 2, 32, TYPES[dtype]))
    go = _made((T, 4, 32), TYPES[dtype], 9)
    want = oracle.packed(q.detach(), k.detach(), v.detach(), lengths, lengths, True, 32 ** -0.5, go)
    out = sapa_b200.packed_attention(q, k, v, offsets_of(lengths))
    check(out.detach(), want["out"], want["out_tol"])
    for name, g in zip(("gq", "gk", "gv"), torch.autograd.grad(out, (q, k, v), go)):
        check(g, want[name], want[name + "_tol"])
    c = Cache(k.detach(), v.detach(), lengths, 16)
    with torch.no_grad():
        check(sapa_b200.paged_attention(q, c.key, c.value, c.table, c.lengths, offsets_of(lengths)), want["out"], want["out_tol"])


@pytest.mark.parametrize("dtype", list(TYPES))
def test_scale_of_zero_is_the_mean(dtype):
    q, k, v = _inputs(300, 300, 4, 2, 64, TYPES[dtype])
    want = oracle.packed(q, k, v, [300], [300], True, 0.0)
    check(sapa_b200.packed_attention(q, k, v, offsets_of([300]), scale=0.0), want["out"], want["out_tol"])
    k[100, 0, 0] = math.inf                              # 0 * infinity is not a number
    assert bool(sapa_b200.packed_attention(q, k, v, offsets_of([300]), scale=0.0)[100:, :2].isnan().all())


@pytest.mark.parametrize("dtype", list(TYPES))
def test_infinite_scores(dtype):
    """A score of -infinity has no weight, one of +infinity, or nothing but -infinity, makes a row NaN, as the formula does; gradients of the rest stay finite."""
    q, k, v = (x.abs() for x in _inputs(200, 200, 2, 1, 64, TYPES[dtype]))
    k = k.clone()
    k[50, 0, 5] = -math.inf
    out = sapa_b200.packed_attention(q, k, v, offsets_of([200]))
    keep = [j for j in range(200) if j != 50]
    assert bool(out.isfinite().all())
    without = oracle.packed(q[150:], k[keep], v[keep], [50], [199], True, 0.125)      # rows from 150 on see all of the 199 up to their own
    check(out[150:], without["out"], without["out_tol"])
    qq, kk, vv = (x.clone().requires_grad_() for x in (q, k, v))
    gq, gk, gv = torch.autograd.grad(sapa_b200.packed_attention(qq, kk, vv, offsets_of([200])).sum(), (qq, kk, vv))
    assert bool(gq[:50].isfinite().all()) and bool(gk.isfinite().all()) and bool(gv.isfinite().all())
    assert bool(gq[50:, :, 5].isnan().all()) and bool(gq[50:, :, 6].isfinite().all())      # 0 * infinity
    k[50, 0, 5] = math.inf
    out = sapa_b200.packed_attention(q, k, v, offsets_of([200]))
    assert bool(out[:50].isfinite().all()) and bool(out[50:].isnan().all())
    k[:, 0, 5] = -math.inf
    assert bool(sapa_b200.packed_attention(q, k, v, offsets_of([200])).isnan().all())


def test_which_kernels_serve():
    from sapa_b200 import _lib
    q, k, v = (x.requires_grad_() for x in _inputs(4000, 4000, 8, 2, 64, torch.bfloat16))
    off = offsets_of([4000])
    out = sapa_b200.packed_attention(q, k, v, off)
    assert _lib.last_kernels()[0] == "sapa_attention_umma_kernel<wide>"
    torch.autograd.grad(out.sum(), (q, k, v))
    assert _lib.last_kernels() == ["sapa_attention_delta_kernel", "sapa_attention_umma_grad_kernel<keys>", "sapa_attention_umma_grad_kernel<queries>"]
    with torch.no_grad():
        for page, kernel in ((16, "sapa_attention_umma_kernel<narrow>"), (256, "sapa_attention_umma_kernel<narrow>"), (24, "sapa_attention_rows_kernel"),
                             (4, "sapa_attention_rows_kernel")):
            c = Cache(k, v, [4000], page)
            sapa_b200.paged_attention(q[:1], c.key, c.value, c.table, c.lengths, offsets_of([1]))
            assert _lib.last_kernels() == [kernel, "sapa_attention_join_kernel"]
            sapa_b200.paged_write(k[:3], v[:3], c.key, c.value, c.table, c.lengths, offsets_of([3]))
            assert _lib.last_kernels() == ["sapa_paged_write_kernel"]
    f = [x.detach().float().requires_grad_() for x in (q, k, v)]
    out = sapa_b200.packed_attention(*f, off)
    assert _lib.last_kernels()[0] == "sapa_attention_rows_kernel"
    torch.autograd.grad(out.sum(), f)
    assert _lib.last_kernels() == ["sapa_attention_delta_kernel", "sapa_attention_rows_grad_kernel<keys>", "sapa_attention_rows_grad_kernel<queries>"]


def test_captured_and_replayed_with_other_lengths():
    q, k, v = _inputs(64, 600, 8, 2, 64, torch.bfloat16)
    off, koff = offsets_of([1] * 4), offsets_of([100, 20, 5, 300])
    off = torch.cat([off, off[-1:].expand(60)])          # room for 64 sequences
    c = Cache(k, v, [100, 20, 5, 300], 16)
    table = torch.full((64, 40), -1, dtype=torch.int32, device="cuda")
    table[:4, :c.table.shape[1]] = c.table
    have = torch.zeros(64, dtype=torch.int32, device="cuda")
    have[:4] = c.lengths

    def both():
        return (sapa_b200.paged_attention(q, c.key, c.value, table, have, off),
                sapa_b200.packed_attention(q, k, v, off[:5], koff))
    eager = both()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = both()
    graph.replay()
    for a, b in zip(held, eager):
        assert torch.equal(a, b)
    want = oracle.packed(q, k, v, [1] * 4, [100, 20, 5, 300], True, 0.125)
    for a in held:
        check(a, want["out"], want["out_tol"])
    have[3] = 170
    koff[4] = 295
    off[1:] = 4
    off[1], off[2], off[3] = 2, 3, 3
    graph.replay()
    want = oracle.packed(q, k, v, [2, 1, 0, 1], [100, 20, 5, 170], True, 0.125)
    for a in held:
        check(a, want["out"], want["out_tol"])


def test_training_step_captured():
    q, k, v = (x.requires_grad_() for x in _inputs(200, 200, 4, 2, 64, torch.bfloat16))
    go, off = _made((200, 4, 64), torch.bfloat16, 4), offsets_of([150, 50])

    def step():
        out = sapa_b200.packed_attention(q, k, v, off)
        return (out, *torch.autograd.grad(out, (q, k, v), go))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eager = [x.detach().clone() for x in step()]
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for _ in range(2):
        graph.replay()
        for a, b in zip(held, eager):
            assert torch.equal(a, b)


def test_streams_threads_and_no_sequence():
    q, k, v = _inputs(90, 90, 4, 2, 64, torch.float16)
    off = offsets_of([60, 30])
    want = sapa_b200.packed_attention(q, k, v, off)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append([sapa_b200.packed_attention(q, k, v, off) for _ in range(8)])
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for g in got for x in g)
    assert sapa_b200.packed_attention(q[:0], k[:0], v[:0], off[:1]).shape == (0, 4, 64)
    assert bool((sapa_b200.packed_attention(q, k, v, off[:1]) == 0).all())
    assert bool((sapa_b200.packed_attention(q, k[:0], v[:0], off, off * 0) == 0).all())
    qq, kk = q[:0].clone().requires_grad_(), k.clone().requires_grad_()
    out = sapa_b200.packed_attention(qq, kk, kk, off * 0, off)
    out.sum().backward()
    assert bool((kk.grad == 0).all())


def test_offsets_out_of_order_stay_inside():
    """Numbers that no program should pass are taken within bounds: the call returns, and sequences that are well formed have their values."""
    q, k, v = _inputs(90, 90, 4, 2, 64, torch.bfloat16)
    bad = torch.tensor([-5, 40, 20, 1 << 30], dtype=torch.int32, device="cuda")
    out = sapa_b200.packed_attention(q, k, v, bad)
    want = oracle.packed(q, k, v, [20], [20], True, 0.125)      # tokens 20 on are of two sequences
    check(out[:20], want["out"][:20], want["out_tol"][:20])
    c = Cache(k, v, [90], 16)
    out = sapa_b200.paged_attention(q, c.key, c.value, c.table, torch.tensor([-3], dtype=torch.int32, device="cuda"), offsets_of([90]))
    assert bool((out == 0).all())
    torch.cuda.synchronize()


def test_cache_beyond_32_bits():
    """A cache of more than 2^32 elements: pages behind that are read and written."""
    page, G, D = 64, 8, 128
    pages = (1 << 32) // (page * G * D) + 40
    kc = torch.zeros(pages, page, G, D, dtype=torch.bfloat16, device="cuda")
    vc = torch.zeros(pages, page, G, D, dtype=torch.bfloat16, device="cuda")
    keys, new = [150, 90], [150, 90]
    q, k, v = _inputs(240, 240, 16, G, D, torch.bfloat16)
    table = torch.tensor([[pages - 1, pages - 7, pages - 3], [pages - 20, 0, -1]], dtype=torch.int32, device="cuda")
    have, off = torch.tensor(keys, dtype=torch.int32, device="cuda"), offsets_of(new)
    sapa_b200.paged_write(k, v, kc, vc, table, have, off)
    want = oracle.packed(q, k, v, new, keys, True, D ** -0.5)
    check(sapa_b200.paged_attention(q, kc, vc, table, have, off), want["out"], want["out_tol"])
    last = torch.stack([q[149], q[239]])
    check(sapa_b200.paged_attention(last, kc, vc, table, have, offsets_of([1, 1])), torch.stack([want["out"][149], want["out"][239]]),
          torch.stack([want["out_tol"][149], want["out_tol"][239]]))


def test_transforms_and_refusals():
    q, k, v = (x.requires_grad_() for x in _inputs(30, 30, 4, 2, 64, torch.float32))
    off = offsets_of([30])
    out = sapa_b200.packed_attention(q, k, v, off)
    g = torch.autograd.grad(out.sum(), (q, k, v))
    made = sapa_b200.PackedAttentionFunction.apply(q, k, v, off, None, True, None)
    assert torch.equal(out, made)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(made.sum(), (q, k, v)), g))
    with torch.autocast("cuda", dtype=torch.bfloat16):
        assert torch.equal(sapa_b200.packed_attention(q, k, v, off), out)
    with pytest.raises(RuntimeError, match="Int"):
        sapa_b200.packed_attention(q, k, v, off.long())
    with pytest.raises(RuntimeError, match="CUDA"):
        sapa_b200.packed_attention(q, k, v, off.cpu())
    with pytest.raises(RuntimeError, match="dtype"):
        sapa_b200.packed_attention(q, k.half(), v, off)
    c = Cache(k.detach(), v.detach(), [30], 16)
    with pytest.raises(NotImplementedError):
        sapa_b200.paged_attention(q, c.key, c.value, c.table, c.lengths, off)
    with pytest.raises(NotImplementedError):
        sapa_b200.paged_write(k, v, c.key, c.value, c.table, c.lengths, off)
    with pytest.raises(RuntimeError, match="dense rows"):
        sapa_b200.paged_attention(q.detach(), c.key.transpose(2, 3).contiguous().transpose(2, 3), c.value, c.table, c.lengths, off)
    with pytest.raises(RuntimeError, match="the cache holds"):
        sapa_b200.paged_attention(q.detach().half(), c.key, c.value, c.table, c.lengths, off)


def test_no_wait_gave_up():
    from sapa_b200 import _lib
    assert _lib.wait_timeout_flags("cuda") == 0
