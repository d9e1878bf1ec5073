"""How far the 16-bit gradients of attention over sequences are off, from the roundings that the kernels make."""
import math

import torch

import attention_oracle as oracle


def gradients(q, k, v, go, dtype, rounded_dscores):
    """(exact gradient, square of the error's norm) of q, k, v of one causal sequence, key heads by themselves.  Every rounding to the type is taken as even over half
    a step u (u^2 / 3 of a value's square): the weights that make the outputs (they reach dS through delta), P for the gradient of values, the result
    (computed exactly here), and dS where it is rounded.  float16's smallest numbers are half of 2^-24 off at most."""
    var = oracle.HALF_STEP[dtype] ** 2 / 3
    least = 2.0 ** -50 / 3 if dtype == torch.float16 else 0.0
    q, k, v, go = (x.double() for x in (q, k, v, go))
    D, share, hidden = q.shape[2], q.shape[1] // k.shape[1], ~oracle.visible(q.shape[0], k.shape[0], True, q.device)
    want = [torch.zeros_like(x) for x in (q, k, v)]
    square = [0.0, 0.0, 0.0]
    for h in range(q.shape[1]):
        kk, vv, scale = k[:, h // share], v[:, h // share], D ** -0.5
        p = torch.softmax((q[:, h] @ kk.T * scale).masked_fill(hidden, -math.inf), 1)
        dp = go[:, h] @ vv.T
        ds = p * (dp - (p * dp).sum(1, keepdim=True))
        want[0][:, h] = scale * (ds @ kk)
        want[1][:, h // share] += scale * (ds.T @ q[:, h])
        want[2][:, h // share] += p.T @ go[:, h]
        delta = var * (p * dp).square().sum(1)
        own = var * ds.square() if rounded_dscores else torch.zeros_like(ds)
        square[0] += scale ** 2 * float((own @ kk.square()).sum() + (delta * (p @ kk).square().sum(1)).sum())
        square[1] += scale ** 2 * float(((own + p.square() * delta[:, None]).T @ q[:, h].square()).sum())
        square[2] += float(((var * p.square()).clamp(min=least).masked_fill(hidden, 0).T @ go[:, h].square()).sum())
    return [(x, e + float((x.to(dtype).double() - x).square().sum())) for x, e in zip(want, square)]
