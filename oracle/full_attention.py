"""Full-attention operators of a serving step in 64 bits, token by token: block tables, rotary positions with the per-head
norm, and attention of one new token over a paged cache."""
from __future__ import annotations

import math

import torch


def block_tables(block_table, context_lens, offsets, free, block_size, num_tokens, start=0):
    """Lists in, ``(table, slots, positions, seq_lens, free_next, status)`` out; status bits as the kernel reports them."""
    table = [list(row) for row in block_table]
    columns, rows = len(table[0]) if table else 0, min(max(offsets[-1], 0), num_tokens)
    slots, positions, lens, status, at = [-1] * num_tokens, [0] * num_tokens, [], 0, start
    for n, (c, lo, hi) in enumerate(zip(context_lens, offsets, offsets[1:])):
        if c < 0 or hi < lo or lo < max([0] + offsets[:n]) or c + hi - lo >= 1 << 31:
            status |= 1
            lens.append(max(c, 0))
            continue
        if hi > rows:                             # what has no row is left out
            status |= 1
        m = min(hi, rows) - min(lo, rows)
        lens.append(c + m)
        held, wanted = -(-c // block_size), -(-(c + m) // block_size)
        if wanted > columns:
            status |= 64
        for col in range(held, min(wanted, columns)):
            if at < len(free):
                table[n][col] = free[at]
            else:
                table[n][col] = -1
                status |= 32
            at += 1
        for t in range(lo, min(hi, rows)):
            p = c + t - lo
            positions[t] = p
            if p // block_size < columns and table[n][p // block_size] >= 0:
                slots[t] = table[n][p // block_size] * block_size + p % block_size
    return table, slots, positions, lens, min(at, len(free)), status


def rms_norm(x, weight, eps=1e-6, unit_offset=False):
    x = x.double()
    w = weight.double() + (1.0 if unit_offset else 0.0)
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * w


def rotate(x, positions, inv_freq, interleaved=False, factor=1.0):
    """``(y, size)``: the rotated rows and, for error bounds, the length of the pair each channel comes from."""
    x = x.double()
    R = 2 * inv_freq.numel()
    angle = positions.double()[:, None] * inv_freq.double()
    cos, sin = (factor * angle.cos())[:, None], (factor * angle.sin())[:, None]
    first, second = (slice(0, R, 2), slice(1, R, 2)) if interleaved else (slice(0, R // 2), slice(R // 2, R))
    y, size = x.clone(), x.abs()
    a, b = x[..., first], x[..., second]
    y[..., first], y[..., second] = a * cos - b * sin, b * cos + a * sin
    size[..., first] = size[..., second] = abs(factor) * torch.hypot(a, b)
    return y, size


def paged_attention(q, k_cache, v_cache, block_table, seq_lens, scale=None):
    """``(out, lse, spread, reach)``; for error bounds also sum p |v| per output and the largest scale * sum |q| |k| per row.
    Pages outside the pool are left out."""
    B, Hq, D = q.shape
    bs, Hk = k_cache.shape[1], k_cache.shape[2]
    scale = D ** -0.5 if scale is None else scale
    out = torch.zeros(B, Hq, D, dtype=torch.float64)
    spread, lse = torch.zeros_like(out), torch.full((B, Hq), -math.inf, dtype=torch.float64)
    reach = torch.zeros(B, Hq, dtype=torch.float64)
    for b in range(B):
        n = min(max(int(seq_lens[b]), 0), block_table.shape[1] * bs)
        at = [(int(block_table[b, j // bs]), j % bs) for j in range(n)]
        at = [(page, i) for page, i in at if 0 <= page < k_cache.shape[0]]
        if not at:
            continue
        pages, inside = torch.tensor([x for x, _ in at]), torch.tensor([x for _, x in at])
        k, v = k_cache[pages, inside].double(), v_cache[pages, inside].double()
        for h in range(Hq):
            kh, vh = k[:, h // (Hq // Hk)], v[:, h // (Hq // Hk)]
            s = scale * (kh @ q[b, h].double())
            p = torch.softmax(s, 0)
            out[b, h], spread[b, h] = p @ vh, p @ vh.abs()
            lse[b, h] = torch.logsumexp(s, 0)
            reach[b, h] = abs(scale) * (kh.abs() @ q[b, h].double().abs()).max()
    return out, lse, spread, reach
