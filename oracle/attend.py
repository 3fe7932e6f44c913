"""Attention over the paged cache, token weights and eviction, in 64 bits.

No counterpart in the reference. Restates the definitions of
include/daric_cache_ops.h (daric_attend_pages, daric_weigh_tokens,
daric_evict_tokens) row by row.
"""
from __future__ import annotations

import numpy as np
import torch

from . import fp8
from .select import k_rows_view, v_view


def _f64(x: torch.Tensor) -> np.ndarray:
    if x.dtype in (torch.uint8, torch.float8_e4m3fn):
        return fp8.decode(x.contiguous().view(torch.uint8).numpy()).astype(np.float64)
    return x.to(torch.float64).numpy()


def gather(rows: torch.Tensor, bt, bt_offset: int, n: int):
    """(rows of tokens 0..n-1 [n, H, D] in 64 bits, which of them are there)."""
    nb, ps = rows.shape[0], rows.shape[1]
    j = np.arange(n)
    page = np.asarray(bt)[bt_offset + j // ps].astype(np.int64)
    there = (page > 0) & (page < nb)
    x = _f64(rows[torch.as_tensor(np.where(there, page, 0)), torch.as_tensor(j % ps)])
    return np.where(there[:, None, None], x, 0.0), there


def sees(i: int, n_ctx: int, n_rows: int, words) -> np.ndarray:
    """Which tokens row i of a sequence sees, if they are there."""
    v = np.zeros(n_ctx + n_rows, bool)
    v[:n_ctx] = True
    for b in range(n_rows):
        v[n_ctx + b] = (b <= i) if words is None else bool((int(words[b // 64]) >> (b % 64)) & 1)
    return v


def _rows(layer, page_first, bt, q, seqs, mask, scale, k_scale):
    """Per (sequence, row, head): (sequence, global row, head, KV head, tokens
    seen, their scores, sum over d of |q k| times the scale)."""
    k_all = k_rows_view(layer, page_first)
    H = k_all.shape[2]
    qn = _f64(q)
    G = q.shape[1] // H
    for s in seqs:
        bo, r0, n_rows, n_ctx = (int(x) for x in s[:4])
        k, there = gather(k_all, bt, bo, n_ctx + n_rows)
        for i in range(n_rows):
            words = None if mask is None else mask[r0 + i].numpy().view(np.uint64)
            seen = np.nonzero(sees(i, n_ctx, n_rows, words) & there)[0]
            for h in range(q.shape[1]):
                g = h // G
                c = scale * (1.0 if k_scale is None else float(k_scale[g]))
                kk = k[seen, g]
                with np.errstate(all="ignore"):
                    yield s, r0 + i, h, g, seen, kk @ qn[r0 + i, h] * c, np.abs(kk) @ np.abs(qn[r0 + i, h]) * abs(c)


def attend(layer, page_first, bt, q, seqs, mask=None, scale=1.0, k_scale=None, v_scale=None):
    """(out, lse, sum of P |V|, largest sum of |q k| of a row, largest |V|, and
    tokens seen), 64 bits; rows of no sequence NaN."""
    v_all = v_view(layer, page_first)
    T, Hq, D = q.shape
    out, mag = np.full((T, Hq, D), np.nan), np.zeros((T, Hq, D))
    lse, amax, vmax, n_seen = np.full((T, Hq), np.nan), np.zeros((T, Hq)), np.zeros((T, Hq)), np.zeros((T, Hq))
    cache = {}
    for s, r, h, g, seen, x, a in _rows(layer, page_first, bt, q, seqs, mask, scale, k_scale):
        if id(s) not in cache:
            cache = {id(s): gather(v_all, bt, int(s[0]), int(s[2]) + int(s[3]))[0]}
        v = cache[id(s)][seen, g] * (1.0 if v_scale is None else float(v_scale[g]))
        with np.errstate(all="ignore"):
            m = x.max() if len(x) else -np.inf
            p = np.exp(x - (0.0 if m == -np.inf else m))
            l = p.sum()
            if l == 0:
                out[r, h], lse[r, h] = 0, -np.inf
                continue
            out[r, h] = (p[:, None] * v).sum(0) / l
            mag[r, h] = (p[:, None] * np.abs(v)).sum(0) / l
            lse[r, h] = m + np.log(l)
            amax[r, h], vmax[r, h], n_seen[r, h] = a.max(), np.abs(v).max(), len(seen)
    return out, lse, mag, amax, vmax, n_seen


def weigh(layer, page_first, bt, q, lse, seqs, weights, mask=None, scale=1.0, k_scale=None):
    """(weights after the call, largest |score| and |lse| met by a token, largest
    sum of |q k|, rows that saw it), 64 bits."""
    w = np.array(weights, dtype=np.float64)
    size, amax, rows = np.zeros_like(w), np.zeros_like(w), np.zeros_like(w)
    for s, r, h, g, seen, x, a in _rows(layer, page_first, bt, q, seqs, mask, scale, k_scale):
        l = float(lse[r, h])
        if l == -np.inf:
            continue
        at = int(s[4]) + seen
        with np.errstate(all="ignore"):
            w[g, at] += np.exp(x - l)
        size[g, at] = np.maximum(size[g, at], np.abs(x) + abs(l))
        amax[g, at] = np.maximum(amax[g, at], a)
        rows[g, at] += 1
    return w, size, amax, rows


def order_key(x: np.ndarray) -> np.ndarray:
    """Rank of fp32 weights: the total order of their bits, NaN above +inf."""
    b = x.astype(np.float32).view(np.uint32).copy()
    b[(b & 0x7FFFFFFF) > 0x7F800000] = 0x7FC00000
    return np.where(b & 0x80000000, ~b, b | np.uint32(0x80000000))


def evict(layers, page_first, bt, weights, evictions, kmax):
    """kept [L, H or 1, n, kmax]; layers and weights (numpy fp32) change in place."""
    L, hw, _ = weights.shape
    kept = np.full((L, hw, len(evictions), kmax), -1, np.int32)
    for l in range(L):
        views = [v for v in (k_rows_view(layers[l], page_first), v_view(layers[l], page_first)) if v is not None]
        if views[0].element_size() == 1:
            views = [v.view(torch.uint8) for v in views]
        nb, ps, H = views[0].shape[0], views[0].shape[1], views[0].shape[2]
        for h in range(hw):
            heads = [h] if hw == H else range(H)
            for i, (bo, c0, n, keep, first, recent) in enumerate(evictions):
                if n <= keep:
                    kept[l, h, i, :n] = np.arange(n)
                    continue
                w = weights[l, h, c0:c0 + n].copy()
                mid = order_key(w[first:n - recent])
                best = np.argsort(-mid.astype(np.int64), kind="stable")[:keep - first - recent] + first
                stay = np.zeros(n, bool)
                stay[:first] = True
                stay[n - recent:] = True
                stay[best] = True
                src = np.arange(keep)
                src[~stay[:keep]] = np.nonzero(stay)[0][np.nonzero(stay)[0] >= keep]
                kept[l, h, i, :keep] = src
                weights[l, h, c0:c0 + n] = 0
                weights[l, h, c0:c0 + keep] = w[src]
                for dst in np.nonzero(src != np.arange(keep))[0]:
                    a, b = int(bt[bo + src[dst] // ps]), int(bt[bo + dst // ps])
                    if not (0 < a < nb and 0 < b < nb):
                        continue
                    for v in views:
                        for hh in heads:
                            v[b, dst % ps, hh] = v[a, src[dst] % ps, hh].clone()
    return kept


# The same definitions over whole matrices, a sequence and KV head at a time: for
# cases of many rows or tokens, where row by row takes minutes.
def _matrices(layer, page_first, bt, q, seqs, mask, scale, k_scale):
    """Per (sequence, KV head): (sequence, KV head, tokens that rows see
    [rows, n], scores [rows, G, n] with -inf where unseen, sums of |q k| times
    the scale, -inf where unseen)."""
    k_all = k_rows_view(layer, page_first)
    H = k_all.shape[2]
    G = q.shape[1] // H
    qn = _f64(q)
    for s in seqs:
        bo, r0, n_rows, n_ctx = (int(x) for x in s[:4])
        if n_rows == 0:
            continue
        k, there = gather(k_all, bt, bo, n_ctx + n_rows)
        see = np.ones((n_rows, n_ctx + n_rows), bool)
        if mask is None:
            see[:, n_ctx:] = np.tri(n_rows, dtype=bool)
        else:
            words = mask[r0:r0 + n_rows].numpy().view(np.uint64)
            b = np.arange(n_rows)
            see[:, n_ctx:] = (words[:, b // 64] >> (b % 64).astype(np.uint64)) & np.uint64(1) != 0
        see &= there
        for g in range(H):
            c = scale * (1.0 if k_scale is None else float(k_scale[g]))
            rows = torch.from_numpy(qn[r0:r0 + n_rows, g * G:(g + 1) * G].reshape(n_rows * G, -1))
            kg = torch.from_numpy(np.ascontiguousarray(k[:, g]).T.copy())
            x = (rows @ kg).numpy().reshape(n_rows, G, -1) * c
            a = (rows.abs() @ kg.abs()).numpy().reshape(n_rows, G, -1) * abs(c)
            hidden = ~see[:, None, :] & np.ones((1, G, 1), bool)
            x[hidden] = -np.inf
            a[hidden] = -np.inf
            yield s, g, see, x, a


def attend_matrix(layer, page_first, bt, q, seqs, mask=None, scale=1.0, k_scale=None, v_scale=None):
    """What attend returns; finite K, V and q."""
    v_all = v_view(layer, page_first)
    T, Hq, D = q.shape
    G = Hq // k_rows_view(layer, page_first).shape[2]
    out, mag = np.full((T, Hq, D), np.nan), np.zeros((T, Hq, D))
    lse, amax, vmax, n_seen = np.full((T, Hq), np.nan), np.zeros((T, Hq)), np.zeros((T, Hq)), np.zeros((T, Hq))
    for s, g, see, x, a in _matrices(layer, page_first, bt, q, seqs, mask, scale, k_scale):
        bo, r0, n_rows, n_ctx = (int(i) for i in s[:4])
        v = gather(v_all, bt, bo, n_ctx + n_rows)[0][:, g] * (1.0 if v_scale is None else float(v_scale[g]))
        m = x.max(-1, keepdims=True)
        p = np.exp(x - np.where(m == -np.inf, 0.0, m))
        total = p.sum(-1)
        p /= np.where(total == 0, 1.0, total)[..., None]
        at = np.s_[r0:r0 + n_rows, g * G:(g + 1) * G]
        pt, vt = torch.from_numpy(p.reshape(-1, p.shape[-1])), torch.from_numpy(np.ascontiguousarray(v))
        out[at] = (pt @ vt).numpy().reshape(n_rows, G, D)
        mag[at] = (pt @ vt.abs()).numpy().reshape(n_rows, G, D)
        with np.errstate(divide="ignore"):
            lse[at] = np.where(total == 0, -np.inf, m[..., 0] + np.log(total))
        amax[at] = np.maximum(a.max(-1), 0.0)
        big = np.where(see, np.abs(v).max(-1)[None, :], 0.0).max(-1)
        vmax[at] = big[:, None]
        n_seen[at] = see.sum(-1)[:, None]
    return out, lse, mag, amax, vmax, n_seen


def weigh_matrix(layer, page_first, bt, q, lse, seqs, weights, mask=None, scale=1.0, k_scale=None):
    """What weigh returns; finite K and q."""
    w = np.array(weights, dtype=np.float64)
    size, amax, rows = np.zeros_like(w), np.zeros_like(w), np.zeros_like(w)
    G = q.shape[1] // w.shape[0]
    for s, g, see, x, a in _matrices(layer, page_first, bt, q, seqs, mask, scale, k_scale):
        l = lse[int(s[1]):int(s[1]) + int(s[2]), g * G:(g + 1) * G].double().numpy()[..., None]
        live = see[:, None, :] & (l > -np.inf)
        at = np.s_[g, int(s[4]):int(s[4]) + see.shape[1]]
        w[at] += np.exp(np.where(live, x - np.where(live, l, 0.0), -np.inf)).sum((0, 1))
        size[at] = np.where(live, np.abs(x) + np.where(live, np.abs(l), 0.0), 0.0).max((0, 1))
        amax[at] = np.where(live, a, 0.0).max((0, 1))
        rows[at] = live.sum((0, 1))
    return w, size, amax, rows


def evict_matrix(layers, page_first, bt, weights, evictions, kmax):
    """What evict returns and does; the rows that move are copied together."""
    L, hw, _ = weights.shape
    kept = np.full((L, hw, len(evictions), kmax), -1, np.int32)
    bt = np.asarray(bt)
    for l in range(L):
        views = [v for v in (k_rows_view(layers[l], page_first), v_view(layers[l], page_first)) if v is not None]
        if views[0].element_size() == 1:
            views = [v.view(torch.uint8) for v in views]
        nb, ps, H = views[0].shape[0], views[0].shape[1], views[0].shape[2]
        for h in range(hw):
            heads = slice(h, h + 1) if hw == H else slice(None)
            for i, (bo, c0, n, keep, first, recent) in enumerate(evictions):
                if n <= keep:
                    kept[l, h, i, :n] = np.arange(n)
                    continue
                w = weights[l, h, c0:c0 + n].copy()
                best = np.argsort(-order_key(w[first:n - recent]).astype(np.int64), kind="stable")[:keep - first - recent]
                stay = np.zeros(n, bool)
                stay[:first] = stay[n - recent:] = stay[best + first] = True
                src = np.arange(keep)
                src[~stay[:keep]] = keep + np.nonzero(stay[keep:])[0]
                kept[l, h, i, :keep] = src
                weights[l, h, c0:c0 + n] = 0
                weights[l, h, c0:c0 + keep] = w[src]
                dst = np.nonzero(src != np.arange(keep))[0]
                a, b = bt[bo + src[dst] // ps].astype(np.int64), bt[bo + dst // ps].astype(np.int64)
                ok = (a > 0) & (a < nb) & (b > 0) & (b < nb)
                a, b, sa, sb = (torch.from_numpy(np.ascontiguousarray(y[ok])) for y in (a, b, src[dst] % ps, dst % ps))
                for v in views:
                    v[b, sb, heads] = v[a, sa, heads]
    return kept
