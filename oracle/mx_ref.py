"""The 8-bit KV cache and attention over a paged cache in 64 bits, from their definitions (CPU, numpy-free torch)."""
import math

import torch

BLOCK = 32


def quantise(x):
    """x [..., D] -> (values [..., D] float64, scale bytes [..., D / 32] uint8)."""
    b = x.double().unflatten(-1, (-1, BLOCK))
    finite = torch.where(b.isfinite(), b.abs(), torch.zeros_like(b))
    a = finite.amax(-1, keepdim=True)
    e = torch.full_like(a, -117.0)
    for k in range(-117, 122):  # the least e with a 2^-e <= 448
        e = torch.where((a > 448 * 2.0 ** (k - 1)) & (e == k - 1), torch.full_like(e, float(k)), e)
    scale = torch.exp2(e)
    y = b / scale
    # a code's step: 2^-3 of its power of two, 2^-9 below 2^-6
    _, exp = torch.frexp(torch.where(y.isfinite(), y, torch.ones_like(y)))
    step = torch.exp2(torch.clamp(exp.double() - 1, min=-6.0) - 3)
    value = torch.round(y / step) * step * scale   # torch.round: ties to even
    value = torch.where(b.isfinite(), value, torch.full_like(value, math.nan))
    return value.flatten(-2), (e.squeeze(-1) + 127).to(torch.uint8)


def code_values():
    """The numbers of the 256 e4m3 codes."""
    out = []
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        v = math.nan if (e, m) == (15, 7) else m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10)
        out.append(-v if c & 128 else v)
    return torch.tensor(out, dtype=torch.float64)


def dequantise(codes, scales):
    """What codes [..., D] (any 8-bit type) and scales [..., D / 32] stand for, float64."""
    factor = torch.exp2(scales.double() - 127)
    return code_values()[codes.view(torch.uint8).long()] * factor.repeat_interleave(BLOCK, dim=-1)


def rows_of(cache, table, n, block_dim):
    """Tokens 0 .. n - 1 of a sequence with block table `table` (list) of a cache [pages, ...] whose dim block_dim is the
    page's rows: ([n, Hkv, D], which of them lie in a valid page)."""
    bs = cache.shape[block_dim]
    out, ok = [], []
    for t in range(n):
        page = int(table[t // bs]) if t // bs < len(table) else -1
        good = 0 <= page < cache.shape[0]
        row = cache[page if good else 0]
        out.append(row[:, t % bs] if block_dim == 2 else row[t % bs])
        ok.append(good)
    return torch.stack(out), torch.tensor(ok)


def attention(q, k, v, visible, scale):
    """One sequence: q [n, Hq, D], k, v [L, Hkv, D], visible [n, L] -> (o, sum of p |v|, largest sum of scale |q_d k_d|
    over a row's keys) in float64, [n, Hq, D], [n, Hq, D] and [n, Hq]; a row that sees nothing is 0."""
    q, k, v = q.double(), k.double(), v.double()
    n, Hq, D = q.shape
    G = Hq // k.shape[1]
    o, bound, reach = torch.zeros(n, Hq, D, dtype=torch.float64), torch.zeros(n, Hq, D, dtype=torch.float64), \
        torch.zeros(n, Hq, dtype=torch.float64)
    for h in range(Hq):
        for i in range(n):
            see = visible[i]
            if not bool(see.any()):
                continue
            kk, vv = k[see, h // G], v[see, h // G]
            s = (kk @ q[i, h]) * scale
            p = torch.softmax(s, 0)
            o[i, h], bound[i, h] = p @ vv, p @ vv.abs()
            reach[i, h] = ((kk.abs() @ q[i, h].abs()) * scale).max()
    return o, bound, reach
