"""Attention over sequences in float64 on the tensors' device, a sequence at a time, with how far a kernel may be off.

u = half a step of the 16-bit or 32-bit type.  An output is rounded once (u |o|); the 16-bit kernels round the softmax's weights to the type before the
second product (u sum p |v|).  What float32 arithmetic adds to a weight is e = 2 ((dim + 4) 2^-24 max sum |q k| scale + keys 2^-24 + 2^-20): the scores'
sums, the sum of the weights, and the exponential."""
import math

import torch

HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def visible(nq, nk, causal, device):
    i, j = torch.arange(nq, device=device)[:, None], torch.arange(nk, device=device)[None, :]
    return j <= i + nk - nq if causal else torch.ones(nq, nk, dtype=torch.bool, device=device)


def sequence(q, k, v, causal, scale, go=None):
    """q [nq, H, D], k, v [nk, G, D] of one sequence -> a dict of outputs and their tolerances (gradients with go)."""
    dtype, (nq, H, D), (nk, G) = q.dtype, q.shape, k.shape[:2]
    u = HALF_STEP[dtype]
    up = 0.0 if dtype == torch.float32 else u
    least = 2.0 ** -25 if dtype == torch.float16 else 0.0             # half a step of the smallest float16 numbers
    q, k, v = q.double(), k.double(), v.double()
    r = {"out": torch.zeros(nq, H, D, dtype=torch.float64, device=q.device)}
    r["out_tol"] = torch.zeros_like(r["out"])
    if go is not None:
        go = go.double()
        for name, like in (("gq", q), ("gk", k), ("gv", v)):
            r[name], r[name + "_tol"] = torch.zeros_like(like), torch.zeros_like(like)
    if nk == 0 or nq == 0:
        return r
    sees = visible(nq, nk, causal, q.device)
    some = sees.any(1)
    for h in range(H):
        g = h // (H // G)
        s = (q[:, h] @ k[:, g].T) * scale
        reach = float(((q[:, h].abs() @ k[:, g].abs().T) * abs(scale))[sees].max()) if bool(sees.any()) else 0.0
        e = 2 * ((D + 4) * 2.0 ** -24 * reach + nk * 2.0 ** -24 + 2.0 ** -20)
        p = torch.softmax(s.masked_fill(~sees, -math.inf), 1)
        p = torch.where(some[:, None], p, torch.zeros_like(p))
        o = p @ v[:, g]
        r["out"][:, h] = o
        off = u * o.abs() + (up + e) * (p @ v[:, g].abs()) + least * (1 + sees.double() @ v[:, g].abs())
        r["out_tol"][:, h] = off
        if go is None:
            continue
        dp = go[:, h] @ v[:, g].T
        delta = (go[:, h] * o).sum(1, keepdim=True)
        ds = p * (dp - delta)
        r["gq"][:, h] = scale * (ds @ k[:, g])
        r["gk"][:, g] += scale * (ds.T @ q[:, h])
        r["gv"][:, g] += p.T @ go[:, h]
        # dP and delta in float32, delta from the rounded output
        mag = go[:, h].abs() @ v[:, g].abs().T
        e_ds = p * ((up + e) * (dp - delta).abs() + (D + 4) * 2.0 ** -24 * 2 * mag + (go[:, h].abs() * off).sum(1, keepdim=True)) + least * sees
        long = (nq * (H // G) + nk) * 2.0 ** -24
        e_ds = e_ds + long * ds.abs()
        r["gq_tol"][:, h] += abs(scale) * (e_ds @ k[:, g].abs())
        r["gk_tol"][:, g] += abs(scale) * (e_ds.T @ q[:, h].abs())
        r["gv_tol"][:, g] += ((up + e + long) * p + least * sees).T @ go[:, h].abs()
    if go is not None:
        for name in ("gq", "gk", "gv"):
            r[name + "_tol"] += u * r[name].abs() + least
    return r


def packed(q, k, v, lengths, key_lengths, causal, scale, go=None, start=0, key_start=0):
    """All sequences of packed tensors: {"out", "out_tol", ...}, zeros where no sequence is."""
    r = None
    a, b = start, key_start
    for nq, nk in zip(lengths, key_lengths):
        one = sequence(q[a:a + nq], k[b:b + nk], v[b:b + nk], causal, scale, None if go is None else go[a:a + nq])
        if r is None:
            r = {}
            for name in one:
                like = q if name.startswith(("out", "gq")) else k
                r[name] = torch.zeros(like.shape, dtype=torch.float64, device=q.device)
        for name, t in one.items():
            at = a if name.startswith(("out", "gq")) else b
            r[name][at:at + t.shape[0]] = t
        a, b = a + nq, b + nk
    return r


def check(got, want, tol):
    assert got.shape == want.shape
    off = (got.double() - want).abs()
    bad = ~(off <= tol * (1 + 1e-6))
    assert not bool(bad.any()), (f"{int(bad.sum())} of {bad.numel()} beyond the tolerance, first at {tuple(bad.nonzero()[0].tolist())}: "
                                 f"got {got[bad][0].item()}, want {want[bad][0].item()}, tolerance {tol[bad][0].item()}")


def offsets_of(lengths, start=0, device="cuda"):
    total = [start]
    for n in lengths:
        total.append(total[-1] + n)
    return torch.tensor(total, dtype=torch.int32, device=device)


class Cache:
    """A paged cache filled with packed keys and values: pages in an order of their own, entries of the table behind a sequence's last page
    outside the cache."""

    def __init__(self, keys, values, lengths, page, spare=2, layout="slots", seed=0, table_extra=1, fill=float("nan")):
        G, D = keys.shape[1:]
        need = [-(-n // page) for n in lengths]
        pages = sum(need) + spare
        shape = {"slots": (pages, page, G, D), "heads": (pages, G, page, D), "both": (pages, 2, page, G, D)}[layout]
        made = [torch.full(shape, fill, dtype=keys.dtype, device=keys.device) for _ in range(1 if layout == "both" else 2)]
        if layout == "both":
            self.key, self.value = made[0][:, 0], made[0][:, 1]
        elif layout == "heads":
            self.key, self.value = (m.transpose(1, 2) for m in made)
        else:
            self.key, self.value = made
        order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
        table = torch.full((len(lengths), max(need + [0]) + table_extra), -7, dtype=torch.int32)
        at = token = 0
        for b, n in enumerate(lengths):
            for i in range(need[b]):
                table[b, i] = order[at]
                m = min(page, n - i * page)
                self.key[order[at], :m] = keys[token:token + m]
                self.value[order[at], :m] = values[token:token + m]
                token += m
                at += 1
        self.table = table.to(keys.device)
        self.lengths = torch.tensor(lengths, dtype=torch.int32, device=keys.device)
