"""Rotation, append and attention over a paged cache from their definitions, in 64 bits and one sequence at a time."""
from __future__ import annotations

import math

import torch


def rotate(x, positions, rotary, weight=None, eps=1e-6, pairs="halves"):
    """x [T, H, D] -> the normalised and rotated rows in f64."""
    y = x.double()
    if weight is not None:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) * weight.double()
    R = rotary.shape[1]
    out = y.clone()
    known = (positions >= 0) & (positions < rotary.shape[0])
    angles = rotary.double()[torch.where(known, positions, 0).long()] if known.any() else rotary.new_zeros((len(y), R)).double()
    for i in range(R // 2):
        a, b = (i, i + R // 2) if pairs == "halves" else (2 * i, 2 * i + 1)
        cos, sin = angles[:, None, i], angles[:, None, R // 2 + i]
        out[..., a] = y[..., a] * cos - y[..., b] * sin
        out[..., b] = y[..., b] * cos + y[..., a] * sin
    if R:
        out[~known] = math.nan
    return out


def append(cache, rows, slots):
    """The cache [PAGES, HK, PAGE, D] with rows [T, HK, D] at their slots (those outside it are left out)."""
    out, page = cache.clone(), cache.shape[2]
    for t, slot in enumerate(slots.tolist()):
        if 0 <= slot < cache.shape[0] * page:
            out[slot // page, :, slot % page] = rows[t]
    return out


def paged_attention(q, k_cache, v_cache, page_table, query_offsets, kv_lengths, scale=None, window=0):
    """(out, weight): the result in f64 and, per element, sum_j softmax_j * |v_j|, the scale of its rounding errors."""
    T, HQ, D = q.shape
    pages, HK, page, _ = k_cache.shape
    group = HQ // HK
    scale = 1 / math.sqrt(D) if scale is None else scale
    out = torch.zeros(T, HQ, D, dtype=torch.float64)
    weight = torch.zeros(T, HQ, D, dtype=torch.float64)
    for b, length in enumerate(kv_lengths.tolist()):
        start, stop = int(query_offsets[b]), int(query_offsets[b + 1])
        for i in range(stop - start):
            position = length - (stop - start) + i
            tokens = [j for j in range(max(0, position - window + 1) if window else 0, position + 1)
                      if 0 <= int(page_table[b, j // page]) < pages]
            if not tokens:
                continue
            j = torch.tensor(tokens)
            where = page_table[b, j // page].long()
            keys = k_cache[where, :, j % page].double()          # [n, HK, D]
            values = v_cache[where, :, j % page].double()
            x = q[start + i].double().view(HK, group, D)
            scores = torch.einsum("hgd,nhd->hgn", x, keys) * scale
            w = torch.softmax(scores, -1)
            out[start + i] = torch.einsum("hgn,nhd->hgd", w, values).reshape(HQ, D)
            weight[start + i] = torch.einsum("hgn,nhd->hgd", w, values.abs()).reshape(HQ, D)
    return out, weight
