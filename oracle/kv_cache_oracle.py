"""CPU oracle of the paged key-value cache and the one-token attention over it
-- TEST INFRASTRUCTURE ONLY.

Plain restatements in 64 bits, token by token, of what include/ma_api.h says
of ma_cache_write, ma_cache_read and ma_decode.  Codes and scales are computed
in 32 bits, which is part of their definition (numpy rounds fp32 divisions
correctly).
"""
from __future__ import annotations

import math

import numpy as np
import torch

TOP = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}


def quantise(x: torch.Tensor, dtype: torch.dtype) -> tuple[torch.Tensor, torch.Tensor]:
    """Codes and scales of rows (..., D) of values."""
    y = x.float().numpy()
    amax = np.maximum(np.abs(y).max(-1), np.float32(1e-12))
    scale = (amax * (np.float32(1) / np.float32(TOP[dtype]))).astype(np.float32)
    z = (y / scale[..., None]).astype(np.float32)
    if dtype == torch.int8:
        return torch.from_numpy(np.clip(np.rint(z), -127, 127).astype(np.int8)), torch.from_numpy(scale)
    return torch.from_numpy(z).to(dtype), torch.from_numpy(scale)


def write(x, pages, scale, table, start, count):
    """x (E, Hk, T, D) into pages (P, Hk, page, D) and scale (P, Hk, page), in place."""
    page = pages.shape[2]
    for e in range(x.shape[0]):
        for t in range(int(count[e])):
            pos = int(start[e]) + t
            p, s = int(table[e, pos // page]), pos % page
            row = x[e, :, t]
            if scale is not None:
                row, sc = quantise(row, pages.dtype)
                scale[p, :, s] = sc
            pages[p, :, s] = row.to(pages.dtype)


def token(pages, scale, table, e, pos):
    """Keys or values (Hk, D) of one position, in 64 bits."""
    page = pages.shape[2]
    p, s = int(table[e, pos // page]), pos % page
    x = pages[p, :, s].double()
    return x if scale is None else x * scale[p, :, s].double()[:, None]


def sequence(pages, scale, table, e, positions):
    """(Hk, len(positions), D) in 64 bits."""
    if not positions:
        return torch.zeros(pages.shape[1], 0, pages.shape[3], dtype=torch.float64)
    return torch.stack([token(pages, scale, table, e, p) for p in positions], 1)


def read(pages, scale, table, lengths, N):
    E, Hk, D = table.shape[0], pages.shape[1], pages.shape[3]
    out = torch.zeros(E, Hk, N, D, dtype=torch.float64)
    for e in range(E):
        n = min(int(lengths[e]), N)
        out[e, :, :n] = sequence(pages, scale, table, e, list(range(n)))
    return out


def attend(q, k_pages, v_pages, k_scale, v_scale, table, lengths, mask=None, sm_scale=None):
    """out (E, H, 1, D), lse (E, H) in 64 bits, and what errors go by (see
    sizes()), each (E, H)."""
    E, H, _, D = q.shape
    Hk = k_pages.shape[1]
    G = H // Hk
    sm_scale = 1.0 / math.sqrt(D) if sm_scale is None else sm_scale
    out = torch.zeros(E, H, 1, D, dtype=torch.float64)
    lse = torch.full((E, H), -math.inf, dtype=torch.float64)
    size = torch.zeros(4, E, H, dtype=torch.float64)
    for e in range(E):
        pos = [j for j in range(int(lengths[e]))
               if mask is None or (j < mask.shape[1] and bool(mask[e, j] != 0))]
        if not pos:
            continue
        k = sequence(k_pages, k_scale, table, e, pos).repeat_interleave(G, 0)  # (H, n, D)
        v = sequence(v_pages, v_scale, table, e, pos).repeat_interleave(G, 0)
        qe = q[e].double()  # (H, 1, D)
        out[e, :, 0], lse[e], size[:, e] = attend_dense(qe, k, v, sm_scale)
    return out, lse, size


def attend_dense(q, k, v, sm_scale):
    """One sequence: q (H, 1, D), k, v (H, n, D) in 64 bits -> out (H, D),
    lse (H), and four sizes (4, H) that errors go by: the largest sm_scale *
    sum_d |q_d k_d|, the largest weighted sum of |v|, the largest weight times
    |v| of one token, and the largest weight times the largest |v|."""
    s = (k * q).sum(-1) * sm_scale
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - m)
    total = p.sum(-1, keepdim=True)
    w = p / total
    va = v.abs()
    size = torch.stack([(k.abs() * q.abs()).sum(-1).amax(-1) * sm_scale,
                        (w[..., None] * va).sum(1).amax(-1), (w * va.amax(-1)).amax(-1),
                        w.amax(-1) * va.amax((1, 2))])
    return (w[..., None] * v).sum(1), (m + torch.log(total))[:, 0], size
