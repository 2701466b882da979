"""FP64 / integer restatement of batched decoding on a paged key-value cache: the step's maps, the
rotary append, and attention over a request's pages (numpy and plain torch, one request at a time)."""
import math

import numpy as np
import torch


def ceil_div(a, b):
    return -(-a // b)


def plan(cached, added, page, free, table, rows):
    """(table, lengths, request, position, slot, summary) of a step; `free` is the free stack, its top last."""
    cached, added = [int(x) for x in cached], [int(x) for x in added]
    table = np.array(table, dtype=np.int64)
    out = [np.full(rows, -1, dtype=np.int64) for _ in range(3)]
    need = [ceil_div(c + max(n, 0), page) for c, n in zip(cached, added)]
    taken = sum(m - ceil_div(c, page) for m, c in zip(need, cached))
    status = 0
    if any(c < 0 or n < 0 for c, n in zip(cached, added)):
        status = 4
    elif sum(added) > rows:
        status = 1
    elif max(need) > table.shape[1]:
        status = 3
    elif taken > len(free):
        status = 2
    if status:
        return table, np.array(cached), *out, np.array([0, 0, status, len(free)])
    stack = [int(x) for x in free]
    r = 0
    for b, (c, n) in enumerate(zip(cached, added)):
        for at in range(ceil_div(c, page), need[b]):
            table[b, at] = stack.pop()
        for pos in range(c, c + n):
            out[0][r], out[1][r], out[2][r] = b, pos, table[b, pos // page] * page + pos % page
            r += 1
    return table, np.array(cached) + np.array(added), *out, np.array([r, taken, 0, len(stack)])


def frequencies(rope_dim, theta, scaling="plain", factor=1.0, original=0, fast=32.0, slow=1.0):
    """The angular frequencies and the amplitude of a scaled rotary table."""
    i = np.arange(rope_dim // 2, dtype=np.float64)
    if scaling == "base" and rope_dim > 2:
        theta = theta * factor ** (rope_dim / (rope_dim - 2))
    f = theta ** (-2.0 * i / rope_dim)
    if scaling == "linear":
        return f / factor, 1.0
    if scaling == "ramp":
        w = np.clip((original * f / (2 * math.pi) - slow) / (fast - slow), 0.0, 1.0)
        return w * f + (1 - w) * f / factor, 0.1 * math.log(factor) + 1.0
    return f, 1.0


def rope_table(t, rope_dim, theta, offset=0, **scaling):
    f, amplitude = frequencies(rope_dim, theta, **scaling)
    angle = (np.arange(t, dtype=np.float64) + offset)[:, None] * f
    return np.stack((np.cos(angle), np.sin(angle)), axis=-1) * amplitude


def rotate(x, table, position, rope_dim, half):
    """x f64 [rows, heads, dim]; table f64 [positions, rope_dim / 2, 2]."""
    y = x.clone()
    cos, sin = table[position][:, None, :, 0], table[position][:, None, :, 1]
    i = torch.arange(rope_dim)
    first, second = (i[:rope_dim // 2], i[rope_dim // 2:]) if half else (i[0::2], i[1::2])
    a, b = x[:, :, first], x[:, :, second]
    y[:, :, first], y[:, :, second] = a * cos - b * sin, a * sin + b * cos
    return y


def attention(q, k, v, table, request, position, page, window=0):
    """q [rows, hq, dim], k and v [pages, hk, page, dim], all f64.  Returns o, lse, the weighted mean of
    |v| and the largest sum of |q_i k_i| / sqrt(dim) of each row and head (for error bounds)."""
    rows, hq, dim = q.shape
    hk = k.shape[1]
    o, size = torch.zeros_like(q), torch.zeros_like(q)
    lse = torch.full((rows, hq), -math.inf, dtype=torch.float64)
    reach = torch.zeros(rows, hq, dtype=torch.float64)
    for r in range(rows):
        n = int(position[r]) + 1
        if int(request[r]) < 0 or n <= 0:
            continue
        at = torch.arange(max(0, n - window) if window else 0, n)
        ids = table[int(request[r])][at // page]
        for h in range(hq):
            g = h // (hq // hk)
            kk, vv = k[ids, g, at % page], v[ids, g, at % page]
            s = kk @ q[r, h] / math.sqrt(dim)
            p = torch.softmax(s, 0)
            o[r, h], size[r, h] = p @ vv, p @ vv.abs()
            lse[r, h] = torch.logsumexp(s, 0)
            reach[r, h] = (kk.abs() @ q[r, h].abs()).max() / math.sqrt(dim)
    return o, lse, size, reach
