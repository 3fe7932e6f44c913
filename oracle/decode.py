"""New rows of a step and beam search, in 64 bits.

No counterpart in the reference. Restates the definitions of
include/daric_cache_ops.h (daric_rotate_rows, daric_append_tokens,
daric_select_beams, daric_reorder_beams) row by row.
"""
from __future__ import annotations

import numpy as np
import torch

from .attend import _f64
from .select import k_rows_view, v_view

E = 2.0 ** -24
LEAST = 2.0 ** 103 - 2.0 ** 128      # rounds to -inf in fp32, as all below does


def rotate(x, positions, inv_freq, rotary_dim, neox=True, m=1.0):
    """(rotated rows in 64 bits, what fp32 arithmetic may be off by before the last
    rounding) of x [T, H, D]. The bound: cosine and sine off by 4 e each (the reduced
    angle's conversion, the series' last roundings, the factor m), the angle itself by
    8 * 2^-53 of its size (three fp64 roundings here and in the kernel), and two roundings
    of the sum."""
    x = _f64(x) if isinstance(x, torch.Tensor) else np.asarray(x, np.float64)
    p = np.asarray(positions, np.int64).astype(np.float64)
    a = p[:, None] * np.asarray(inv_freq, np.float32).astype(np.float64)[None, : rotary_dim // 2]
    c, s = (m * np.cos(a))[:, None], (m * np.sin(a))[:, None]
    i = np.arange(rotary_dim // 2)
    i1, i2 = (i, i + rotary_dim // 2) if neox else (2 * i, 2 * i + 1)
    out, off = x.copy(), np.zeros_like(x)
    x1, x2 = x[..., i1], x[..., i2]
    out[..., i1] = x1 * c - x2 * s
    out[..., i2] = x2 * c + x1 * s
    err = (6 * E + 8 * 2.0 ** -53 * np.abs(a))[:, None] * abs(m) * (np.abs(x1) + np.abs(x2))
    off[..., i1] = off[..., i2] = err
    return out, off


def append(layer, page_first, bt, k, v, seqs, positions=None, rope=None, k_scale=None, v_scale=None):
    """(row of k, page, slot) of every token that is written, and (K values, V values,
    what K's fp32 arithmetic may be off by) of all rows, in units of the cache's codes.
    rope: (inv_freq, rotary_dim, neox, m) or None."""
    rows = k_rows_view(layer, page_first)
    nb, ps = rows.shape[0], rows.shape[1]
    where, pos = [], np.zeros(k.shape[0], np.int64)
    for s in seqs:
        bo, r0, n, ctx = (int(x) for x in s[:4])
        for i in range(n):
            t = ctx + i
            page = int(bt[bo + t // ps])
            pos[r0 + i] = t
            if 0 < page < nb:
                where.append((r0 + i, page, t % ps))
    if positions is not None:
        pos = np.asarray(positions)
    kk, off = rotate(k, pos, *rope) if rope is not None else (_f64(k), np.zeros(k.shape))
    vv = _f64(v) if v is not None else None
    if k_scale is not None:
        sc = np.asarray(k_scale, np.float64)[None, :, None]
        kk, off = kk / sc, off / sc
    if v_scale is not None and vv is not None:
        vv = vv / np.asarray(v_scale, np.float64)[None, :, None]
    return where, pos, kk, vv, off


def select(logits, scores, k, ended=None, end_token=-1):
    """(scores, parents, tokens) [B, k] of the best candidates, in 64 bits, by a sort of
    all of a request's: by score, then beam, then logit, then token."""
    x = _f64(logits)
    B, W, V = x.shape
    out = np.full((B, k), -np.inf), np.full((B, k), -1, np.int32), np.full((B, k), -1, np.int32)
    for b in range(B):
        s = np.full((W, V), -np.inf)
        for w in range(W):
            base = float(scores[b][w])
            if ended is not None and ended[b][w]:
                s[w, end_token] = base
                continue
            with np.errstate(all="ignore"):
                d = x[b, w] - np.max(x[b, w])        # before the sum's logarithm: logits may be huge
                s[w] = base + (d - np.log(np.sum(np.exp(d))))
        s[np.isnan(s)] = -np.inf
        flat = s.reshape(-1)
        logit = np.where(np.isneginf(flat), 0.0, x[b].reshape(-1))
        if ended is not None:
            logit.reshape(W, V)[np.asarray(ended[b], bool)] = 0.0          # not looked at
        best = np.lexsort((np.arange(W * V), -logit, np.arange(W * V) // V, -flat))[:k]
        for i, c in enumerate(best):
            if flat[c] > LEAST:
                out[0][b, i], out[1][b, i], out[2][b, i] = flat[c], c // V, c % V
    return out


def reorder(layers, page_first, bt, parents, beams):
    """In place: block lists and the rows of last pages, beam by beam from copies of
    what stood there before."""
    for (bo, stride, W, n), row in zip(beams, np.asarray(parents)):
        ps = k_rows_view(layers[0], page_first).shape[1]
        nb = k_rows_view(layers[0], page_first).shape[0]
        full, rest = n // ps, n % ps
        lists = [np.array(bt[bo + w * stride: bo + w * stride + -(-n // ps)]) for w in range(W)]
        for layer in layers:
            planes = [k_rows_view(layer, page_first)] + ([v_view(layer, page_first)] if layer.dim() != 3 else [])
            for rows in planes:
                before = rows.clone()
                for w in range(W):
                    p = int(row[w])
                    if rest == 0 or not 0 <= p < W or p == w:
                        continue
                    src, dst = int(lists[p][full]), int(lists[w][full])
                    if 0 < src < nb and 0 < dst < nb:
                        rows[dst, :rest] = before[src, :rest]
        for w in range(W):
            p = int(row[w])
            if 0 <= p < W:
                bt[bo + w * stride: bo + w * stride + full] = lists[p][:full]
