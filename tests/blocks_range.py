"""Long caches over the 8-bit block cache in 64 bits: inputs whose every block matters, or whose first row takes most of the weight, and a bound on one
output's error that follows each key's own rounding."""
import math

import torch

import blocks_util as U

F64 = torch.float64
LIFT = 7  # the kernel's largest weight stands at 2^LIFT at least when it becomes fp16


def held_rows(x):
    """Rows [n, dim] -> (what the cache holds for them [n, dim], scale exponent of every row [n]), block by block as append rounds them."""
    n, dim = x.shape
    y = torch.nn.functional.pad(x.double(), (0, 0, 0, -n % U.BLOCK)).view(-1, U.BLOCK, dim)
    e = torch.tensor([U.exponent(float(t)) for t in y.abs().amax((1, 2))])
    scale = torch.exp2(e.double())[:, None, None]
    return (U.e4m3(y / scale) * scale).view(-1, dim)[:n], e.repeat_interleave(U.BLOCK)[:n]


def one_head(q, k, v, v_exp, scale, pos0=None):
    """q [tokens, dim]; k, v [n, dim] as the cache holds them, v_exp [n]: softmax weights [tokens, n], scaled weights p 2^v_exp, outputs, tolerance.

    A key's weight enters the product with the bare codes as fp16, in units in which the largest p 2^v_exp of the column is 2^LIFT at least: half a step is 2^-11
    relative, or 2^-25 where fp16 is subnormal, 2^-(25 + LIFT) of the largest; a weight that is lost altogether is off by itself.  The scores are ``dim`` products summed in
    fp32, the exponent is rounded in units of log2: a relative error d of every weight, twice in the quotient.  Sums over keys: n * 2^-23.  Output: bf16, 2^-8."""
    n, dim = k.shape
    t = q.double() @ k.T * scale
    if pos0 is not None:
        t = t.masked_fill(torch.arange(n)[None] > (pos0 + torch.arange(len(q)))[:, None], -math.inf)
    p = torch.softmax(t, -1)
    most = float(t[torch.isfinite(t)].abs().max())
    mass = float((q.double().abs() @ k.abs().T * scale).max())
    d = dim * 2.0**-24 * mass + (most + 50) * 1.45 * 2.0**-23 + 2.0**-21
    unit = torch.exp2(v_exp.double())
    y = p * unit
    lost = torch.maximum(y * 2.0**-11, torch.minimum(y, y.amax(-1, keepdim=True) * 2.0 ** -(25 + LIFT)))
    o, size = p @ v, p @ v.abs()
    tol = o.abs() * 2.0**-8 + ((lost / unit) @ v.abs() + size * (2 * d + n * 2.0**-23)) * (1 + 2.0**-8)
    return p, y, o, tol


def sink(n, dim, share, size, outlier, seed):
    """One head's keys and values: the first row takes ``share`` of every query's weight and has values of ``size``, another row of its block one of ``outlier``; all
    other values lie between 0.5 and 1.5, so that what the many others have together shows in every coordinate.  Queries have an 8 in coordinate 0."""
    g = torch.Generator().manual_seed(seed)
    k, v = torch.randn(n, dim, generator=g), torch.rand(n, dim, generator=g) + 0.5
    spread = (dim - 1) / dim  # of the other rows' scores, at queries of standard normals and scale dim^-0.5
    k[:, 0] = 0.0
    k[0] = 0.0
    k[0, 0] = round((math.log(share / (1 - share)) + math.log(n) + spread / 2) * math.sqrt(dim) / 8, 1)
    v[0] *= size
    v[1, 5] = outlier
    return k.to(torch.bfloat16), v.to(torch.bfloat16)


def marked(n, dim, seed):
    """Small values, and one of 8 in every block, in another row and coordinate of each: an output that lacks a block, or takes its row or coordinate for another, is off by far more than its tolerance."""
    g = torch.Generator().manual_seed(seed)
    k, v = torch.randn(n, dim, generator=g), torch.randn(n, dim, generator=g) * 0.02
    for b in range((n + U.BLOCK - 1) // U.BLOCK):
        v[min(b * U.BLOCK + 7 * b % U.BLOCK, n - 1), b % dim] = 8.0
    return k.to(torch.bfloat16), v.to(torch.bfloat16)


SINKS = [(0.994, 0.02, 16.0), (0.994, 0.02, 64.0), (0.957, 0.02, 64.0), (0.9992, 0.001, 1.0)]  # (share, size, outlier)
LENGTHS = [5003, 9001, 7777]
