"""Plain 64-bit forms of the paged-cache operators, for their tests."""
from __future__ import annotations

import numpy as np
import torch

NO_SLOT = 0xFFFFFFFF


def tables(context, new, free, page_size, block_tables, num_tokens):
    """query_start, seq_lens, positions, slots, block tables and status, request
    by request.  `free` is the stack, its top last."""
    max_blocks = block_tables.shape[1]
    block_tables = block_tables.copy()
    start, seq, pos, slot, claimed, taken, refused = [0], [], [], [], 0, 0, 0
    for b, (c, n) in enumerate(zip(context, new)):
        old, end = -(-c // page_size), -(-(c + n) // page_size)
        need = end - old if end <= max_blocks else 0
        ok = end <= max_blocks and start[-1] + n <= num_tokens
        ok = ok and (need == 0 or claimed + need <= len(free))
        if ok:
            for j in range(need):
                block_tables[b, old + j] = free[len(free) - 1 - claimed - j]
            taken = max(taken, claimed + need if need else 0)
        claimed += need
        refused += not ok
        seq.append(c + n if ok else c)
        for i in range(min(n, max(0, num_tokens - start[-1]))):  # rows past num_tokens: not there
            p = c + i
            pos.append(p)
            slot.append(int(block_tables[b, p // page_size]) * page_size + p % page_size
                        if ok else NO_SLOT)
        start.append(start[-1] + n)
    pos = (pos + [0] * num_tokens)[:num_tokens]
    slot = (slot + [NO_SLOT] * num_tokens)[:num_tokens]
    start = [min(x, 0xFFFFFFFF) for x in start]
    return start, seq, pos, slot, block_tables, [len(free) - taken, refused]


def rms_rope(x, w, cos_sin, eps):
    """x [T][H][D], cos_sin [T][D/2][2], all float64."""
    d = x.shape[-1]
    y = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w
    c, s = cos_sin[:, None, :, 0], cos_sin[:, None, :, 1]
    a, b = y[..., :d // 2], y[..., d // 2:]
    return np.concatenate([a * c - b * s, b * c + a * s], -1)


def visible(n, length, window, sinks):
    """[n][length] mask of a request with n new tokens."""
    p = length - n + np.arange(n)[:, None]
    j = np.arange(length)[None, :]
    seen = j <= p
    if window:
        seen &= (p - j < window) | (j < sinks)
    return seen


def attention(q, k, v, window, sinks):
    """One request: q [n][Hq][D], k and v [length][Hkv][D] float64 tensors.
    Returns o, the weights' mean distance of v from o (sum_j w_j |v_j - o|) and
    their mean |v|, each [n][Hq][D]: what a rounding of each weight can move."""
    n, hq, d = q.shape
    length, hkv, _ = k.shape
    seen = torch.from_numpy(visible(n, length, window, sinks)).to(q.device)
    o, away, size = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(q)
    for h in range(hq if length else 0):
        kh, vh = k[:, h // (hq // hkv)], v[:, h // (hq // hkv)]
        s = (q[:, h] @ kh.t().contiguous()) / d ** 0.5
        s = torch.where(seen, s, torch.full_like(s, -float("inf")))
        m = s.amax(-1, keepdim=True)
        w = torch.where(seen, torch.exp(s - m), torch.zeros_like(s))
        total = w.sum(-1, keepdim=True)
        w = torch.where(total > 0, w / total, torch.zeros_like(w))
        for i in range(n):
            live = seen[i].nonzero()[:, 0]
            wi, vi = w[i, live][:, None], vh[live]
            o[i, h] = (wi * vi).sum(0)
            away[i, h] = (wi * (vi - o[i, h]).abs()).sum(0)
            size[i, h] = (wi * vi.abs()).sum(0)
    return o, away, size
