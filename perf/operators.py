"""Attention over sequences of tokens, as cases to time: whole sequences packed one behind the other, with and without their gradients; new
tokens over a paged cache of keys and values, from one token a sequence to chunks; and the writing of new keys and values into that cache.

A case is a dict of plain values:

    op       "packed" (packed_attention), "paged" (paged_attention) or "write" (paged_write)
    train    packed: the output and the gradients of query, key and value instead of the output alone
    dtype    "f32", "f16", "bf16"
    causal   packed: a token sees the tokens up to itself; otherwise it sees its whole sequence (the paged operator is always causal)
    B        sequences; "longest" the keys of the longest one, "mix" the number from which the lengths of the others come
    heads, groups, dim   query heads, key / value heads (a divisor of heads), channels of a head
    new, page            paged, write: the most new tokens of a sequence, tokens of a page
"""
import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # a handful of short prompts: the time of a call counts
        {"name": "packed_small_bf16", "op": "packed", "train": False, "dtype": "bf16", "causal": True, "B": 4, "longest": 100, "mix": 1,
         "heads": 8, "groups": 2, "dim": 64},
        # prompts of very different lengths in one batch, grouped heads
        {"name": "packed_mixed_bf16", "op": "packed", "train": False, "dtype": "bf16", "causal": True, "B": 8, "longest": 2047, "mix": 2,
         "heads": 32, "groups": 8, "dim": 128},
        # one long prompt
        {"name": "packed_long_f16", "op": "packed", "train": False, "dtype": "f16", "causal": True, "B": 1, "longest": 8192, "mix": 3,
         "heads": 32, "groups": 8, "dim": 128},
        # a training step over packed documents
        {"name": "packed_train_bf16", "op": "packed", "train": True, "dtype": "bf16", "causal": True, "B": 4, "longest": 4096, "mix": 4,
         "heads": 16, "groups": 4, "dim": 128},
        # feature maps of 512 x 512 images at stride 16 as bidirectional tokens, with a few more of another size, one key head to a query head
        {"name": "packed_train_both_f16", "op": "packed", "train": True, "dtype": "f16", "causal": False, "B": 8, "longest": 1024, "mix": 5,
         "heads": 12, "groups": 12, "dim": 64},
        # the same in full precision, as a check run or a small model trains
        {"name": "packed_train_f32", "op": "packed", "train": True, "dtype": "f32", "causal": True, "B": 3, "longest": 515, "mix": 6,
         "heads": 8, "groups": 4, "dim": 64},
        # a few requests that answer token by token: latency
        {"name": "paged_one_small_f16", "op": "paged", "dtype": "f16", "B": 3, "longest": 301, "mix": 7, "heads": 8, "groups": 2, "dim": 64,
         "new": 1, "page": 16},
        # many requests that answer token by token over long caches: reading the cache counts
        {"name": "paged_one_bf16", "op": "paged", "dtype": "bf16", "B": 48, "longest": 8190, "mix": 8, "heads": 32, "groups": 8, "dim": 128,
         "new": 1, "page": 16},
        # chunks of long prompts, next to requests that add few tokens
        {"name": "paged_chunks_bf16", "op": "paged", "dtype": "bf16", "B": 6, "longest": 6000, "mix": 9, "heads": 32, "groups": 8, "dim": 128,
         "new": 512, "page": 64},
        # one sequence, one token, full precision
        {"name": "paged_one_f32", "op": "paged", "dtype": "f32", "B": 2, "longest": 2500, "mix": 10, "heads": 16, "groups": 4, "dim": 64,
         "new": 1, "page": 32},
        # what goes with them before each: a token of every request, and the chunks of prompts
        {"name": "write_one_bf16", "op": "write", "dtype": "bf16", "B": 48, "longest": 1000, "mix": 11, "heads": 32, "groups": 8, "dim": 128,
         "new": 1, "page": 16},
        {"name": "write_chunks_bf16", "op": "write", "dtype": "bf16", "B": 8, "longest": 3000, "mix": 12, "heads": 32, "groups": 8, "dim": 128,
         "new": 2048, "page": 64},
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, spread evenly over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op, train = rng.choice([("packed", False)] * 3 + [("packed", True)] * 3 + [("paged", False)] * 4 + [("write", False)])
    case = {"op": op, "dtype": rng.choice(("bf16", "bf16", "f16", "f32")), "mix": rng.randrange(1 << 20)}
    groups, share = rng.choice((1, 2, 3, 4, 8)), rng.choice((1, 1, 2, 3, 4, 5, 7, 8))
    case["heads"], case["groups"], case["dim"] = groups * share, groups, rng.choice((32, 40, 64, 64, 80, 96, 128, 128))
    full = case["dtype"] == "f32"
    if op == "packed":
        case["train"], case["causal"] = train, rng.random() < 0.75
        case["B"] = _spread(rng, 1, 24)
        # scores of all sequences, each as long as the longest
        room = (1 << 26 if full else 1 << 28) if train else (1 << 28 if full else 1 << 30)
        most = math.isqrt(room // (case["B"] * case["heads"]))
        # the gradient of a lone token's query is zero: a longest sequence of two at least where it is compared
        case["longest"] = _spread(rng, 2 if train else 1, max(2, min(8192 if not train else 4096, most)))
    elif op == "paged":
        case["B"], case["page"] = _spread(rng, 1, 64), rng.choice((16, 16, 32, 64, 128))
        case["new"] = rng.choice((1, 1, _spread(rng, 2, 16), _spread(rng, 17, 512)))
        most = min(8192, (1 << 23) // (case["B"] * groups), (1 << 28) // (case["B"] * case["heads"] * case["new"]) if not full else
                   (1 << 26) // (case["B"] * case["heads"] * case["new"]))
        case["longest"] = _spread(rng, case["new"], max(case["new"], most))
    else:
        case["B"], case["page"], case["new"] = _spread(rng, 1, 64), rng.choice((16, 32, 64)), _spread(rng, 1, 512)
        case["longest"] = _spread(rng, case["new"], 2048 if case["B"] <= 16 else 1024)
        case["new"] = min(case["new"], case["longest"])
    return case


def _lengths(case):
    """(new tokens, keys) of every sequence, as two lists."""
    rng = random.Random(case["mix"])
    keys = [case["longest"]] + [rng.randint(max(1, case["longest"] // 8), case["longest"]) for _ in range(case["B"] - 1)]
    rng.shuffle(keys)
    if case["op"] == "packed":
        return list(keys), keys
    most = case["new"]
    return [min(k, rng.choice((most, most, rng.randint(1, most)))) for k in keys], keys


def _offsets(lengths):
    total = [0]
    for n in lengths:
        total.append(total[-1] + n)
    return torch.tensor(total, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t, H, G, D = DTYPES[case["dtype"]], case["heads"], case["groups"], case["dim"]
    new, keys = _lengths(case)
    T = sum(new)

    def made(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(t)
    state = {"case": case, "offsets": _offsets(new), "most_new": max(new), "most_keys": max(keys)}
    if case["op"] == "packed":
        if case["train"]:
            state["query"], state["key"], state["value"] = (made(T, n, D, scale=s).requires_grad_() for n, s in ((H, 1.5), (G, 1.0), (G, 1.0)))
            state["grad"] = made(T, H, D)
        else:      # the parts of one projection's output
            together = made(T, H + 2 * G, D)
            together[:, :H] *= 1.5
            state["query"], state["key"], state["value"] = together.split((H, G, G), dim=1)
        return state
    page = case["page"]
    need = [-(-k // page) for k in keys]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((case["B"], max(need) + 1), -1, dtype=torch.int32, device="cuda")      # no page where no key is
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    state["key_pages"], state["value_pages"] = made(pages, page, G, D), made(pages, page, G, D)
    state["table"], state["key_lengths"] = table, torch.tensor(keys, dtype=torch.int32, device="cuda")
    if case["op"] == "paged":
        state["query"] = made(T, H, D, scale=1.5)
    else:
        state["key"], state["value"] = made(T, G, D), made(T, G, D)
    return state


# ---------------------------------------------------------------------------------- the framework's calls
def _own(state):
    import sapa_b200

    case = state["case"]
    if case["op"] == "packed":
        out = sapa_b200.packed_attention(state["query"], state["key"], state["value"], state["offsets"], causal=case["causal"])
        if not case["train"]:
            return out
        return (out.detach(), *torch.autograd.grad(out, (state["query"], state["key"], state["value"]), state["grad"]))
    if case["op"] == "paged":
        return sapa_b200.paged_attention(state["query"], state["key_pages"], state["value_pages"], state["table"], state["key_lengths"],
                                         state["offsets"])
    sapa_b200.paged_write(state["key"], state["value"], state["key_pages"], state["value_pages"], state["table"], state["key_lengths"],
                          state["offsets"])
    return state["key_pages"], state["value_pages"]


# ---------------------------------------------------------------------------------- the plain form
def _padded(x, offsets, most):
    """[T, n, D] -> [B, most, n, D] in 32 bits, and which rows are tokens."""
    begin, end = offsets[:-1].long(), offsets[1:].long()
    at = begin[:, None] + torch.arange(most, device=x.device)
    there = at < end[:, None]
    return torch.where(there[:, :, None, None], x.float()[at.clamp(max=x.shape[0] - 1)], 0.0), there


def _rows(x, groups):
    """[B, L, heads, D] -> [B, groups, L * heads of a group, D]"""
    B, L, H, D = x.shape
    return x.view(B, L, groups, H // groups, D).transpose(1, 2).reshape(B, groups, L * (H // groups), D)


def _tokens(x, there, share):
    """The way back, without the padding: [B, groups, L * share, D] -> [T, heads, D]"""
    B, G, R, D = x.shape
    return x.view(B, G, R // share, share, D).transpose(1, 2).reshape(B, R // share, G * share, D)[there]


def _weights(q, k, sees, share, scale):
    """softmax(scale q k^T) over what a row sees; zeros where it sees nothing.  sees: [B, L, keys]"""
    sees = sees[:, None, :, None].expand(-1, 1, -1, share, -1).flatten(2, 3)
    s = torch.where(sees, (q @ k.transpose(-1, -2)) * scale, -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-3e38))
    return p / p.sum(-1, keepdim=True).clamp(min=1e-37)


def _plain_packed(state):
    case = state["case"]
    G, share, scale, t = case["groups"], case["heads"] // case["groups"], 1 / math.sqrt(case["dim"]), DTYPES[case["dtype"]]
    q, there = _padded(state["query"].detach(), state["offsets"], state["most_new"])
    k, v = (_padded(state[x].detach(), state["offsets"], state["most_new"])[0].transpose(1, 2) for x in ("key", "value"))
    q = _rows(q, G)
    sees = there[:, None, :] & there[:, :, None]
    if case["causal"]:
        sees = sees.tril()
    p = _weights(q, k, sees, share, scale)
    out = _tokens(p @ v, there, share).to(t)
    if not case["train"]:
        return out
    go = _rows(_padded(state["grad"], state["offsets"], state["most_new"])[0], G)
    gv = p.transpose(-1, -2) @ go
    gp = go @ v.transpose(-1, -2)
    gs = p * (gp - (p * gp).sum(-1, keepdim=True))
    del p, gp
    gq, gk = (gs @ k) * scale, (gs.transpose(-1, -2) @ q) * scale
    return out, _tokens(gq, there, share).to(t), _tokens(gk, there, 1).to(t), _tokens(gv, there, 1).to(t)


def _plain_paged(state):
    case = state["case"]
    G, share, page, most = case["groups"], case["heads"] // case["groups"], case["page"], state["most_keys"]
    q, there = _padded(state["query"], state["offsets"], state["most_new"])
    new = state["offsets"][1:] - state["offsets"][:-1]
    at = torch.arange(most, device=q.device)
    where = state["table"].long()[:, at // page].clamp(min=0)
    k, v = (state[x][where, at % page].float().transpose(1, 2) for x in ("key_pages", "value_pages"))      # [B, groups, keys, D]
    last = (state["key_lengths"] - new)[:, None] + torch.arange(state["most_new"], device=q.device)        # the last key that a token sees
    sees = (at <= last[:, :, None]) & there[:, :, None]
    full = at < state["key_lengths"][:, None]
    v = torch.where(full[:, None, :, None], v, 0.0)
    p = _weights(_rows(q, G), k, sees & full[:, None, :], share, 1 / math.sqrt(case["dim"]))
    return _tokens(p @ v, there, share).to(DTYPES[case["dtype"]])


def _plain_write(state):
    page, offsets = state["case"]["page"], state["offsets"].long()
    token = torch.arange(state["key"].shape[0], device=offsets.device)
    b = torch.searchsorted(offsets, token, right=True) - 1
    at = state["key_lengths"].long()[b] - offsets[b + 1] + token
    where, slot = state["table"].long()[b, at // page], at % page
    state["key_pages"][where, slot] = state["key"]
    state["value_pages"][where, slot] = state["value"]
    return state["key_pages"], state["value_pages"]


def run(state):
    if own:
        return _own(state)
    return {"packed": _plain_packed, "paged": _plain_paged, "write": _plain_write}[state["case"]["op"]](state)


# ---------------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    new, keys = _lengths(case)
    e, H, G, D = DTYPES[case["dtype"]].itemsize, case["heads"], case["groups"], case["dim"]
    T = sum(new)
    if case["op"] == "write":
        return {"bytes": 4 * T * G * D * e, "flops": 0}
    causal = case.get("causal", True)
    pairs = sum(n * k - (n * (n - 1) // 2 if causal else 0) for n, k in zip(new, keys))      # a token and a key that it sees
    cells = H * D * T * 2 + 2 * G * D * sum(keys)
    products = 2
    if case.get("train"):      # the gradients, and what they come from, once more
        cells, products = cells + 2 * H * D * T + 2 * G * D * T, 7
    return {"bytes": cells * e, "flops": 2 * products * pairs * H * D}


# ---------------------------------------------------------------------------------- in 64 bits, a sequence and a group of heads at a time
def _exact_rows(q, k, v, first, go):
    """Output rows of one head, and the gradients of q, k, v where go is there.  Row i sees the keys below first + i (all, if None)."""
    s = torch.einsum("id,jd->ij", q, k) / math.sqrt(q.shape[1])
    if first is not None:
        hidden = torch.arange(k.shape[0], device=q.device)[None, :] >= first + torch.arange(q.shape[0], device=q.device)[:, None]
        s.masked_fill_(hidden, -math.inf)
    p = torch.softmax(s, dim=1)
    out = torch.einsum("ij,jd->id", p, v)
    if go is None:
        return out, None, None, None
    gs = p * (torch.einsum("id,jd->ij", go, v) - (go * out).sum(1)[:, None]) / math.sqrt(q.shape[1])
    return out, torch.einsum("ij,jd->id", gs, k), torch.einsum("ij,id->jd", gs, q), torch.einsum("ij,id->jd", p, go)


def exact(case, seed):
    state = prepare(case, seed)
    new, keys = _lengths(case)
    H, G, D = case["heads"], case["groups"], case["dim"]
    if case["op"] == "write":
        pages = [state["key_pages"].double(), state["value_pages"].double()]
        token = 0
        for b, (n, k) in enumerate(zip(new, keys)):
            at = torch.arange(k - n, k, device="cuda")
            rows = state["table"][b].long()[at // case["page"]] * case["page"] + at % case["page"]
            for p, x in zip(pages, (state["key"], state["value"])):
                p.view(-1, G, D).index_copy_(0, rows, x[token:token + n].double())
            token += n
        return tuple(pages)
    T = sum(new)
    train = bool(case.get("train"))
    out = torch.zeros(T, H, D, dtype=torch.float64, device="cuda")
    if train:
        grads = [torch.zeros(T, n, D, dtype=torch.float64, device="cuda") for n in (H, G, G)]
    at = 0
    for b, (n, k) in enumerate(zip(new, keys)):
        here = slice(at, at + n)
        if case["op"] == "packed":
            kk, vv = state["key"].detach()[here].double(), state["value"].detach()[here].double()
            first = 1 if case["causal"] else None
        else:
            used = state["table"][b, :-(-k // case["page"])].long()
            kk, vv = (state[x][used].flatten(0, 1)[:k].double() for x in ("key_pages", "value_pages"))
            first = k - n + 1
        for h in range(H):
            j = h // (H // G)
            go = state["grad"][here, h].double() if train else None
            o, gq, gk, gv = _exact_rows(state["query"].detach()[here, h].double(), kk[:, j], vv[:, j], first, go)
            out[here, h] = o
            if train:
                grads[0][here, h] = gq
                grads[1][here, j] += gk
                grads[2][here, j] += gv
        at += n
    return (out, *grads) if train else out
