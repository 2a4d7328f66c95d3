"""float64 restatement of the paged key-value cache's operators (test infrastructure).

Written from their definition, one sequence and one row at a time: the append
(head norm, rotation, cache slots) and attention over what a row sees. Tables
as the C ABI's: row_start [nseq + 1], length [nseq], pages [nseq, max_pages];
pools [n_pages, kv_heads, page_size, dim].
"""
import numpy as np


def new_rows(row_start, length, b):
    """(row, position) of each new row of sequence b."""
    r0, r1 = int(row_start[b]), int(row_start[b + 1])
    return [(r, max(int(length[b]), 0) - (r1 - r0) + r - r0) for r in range(r0, r1)]


def slot(pages, b, j, n_pages, page_size):
    """(page, slot) of key j of sequence b, or None where the table names no page."""
    if j < 0 or j // page_size >= pages.shape[1]:
        return None
    pg = int(pages[b, j // page_size])
    return (pg, j % page_size) if 0 <= pg < n_pages else None


def prepare_head(x, w, eps, p, rot, interleaved, freq):
    """A head of q or k, normed (w or None) and its first `rot` features rotated by p * freq."""
    x = np.array(x, np.float64)
    if w is not None:
        x = x / np.sqrt(np.mean(x * x) + eps) * np.asarray(w, np.float64)
    for i in range(rot // 2):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
        c, s = np.cos(p * freq[i]), np.sin(p * freq[i])
        x[a], x[b] = x[a] * c - x[b] * s, x[a] * s + x[b] * c
    return x


def append(k_pool, v_pool, row_start, length, pages, q, k, v, q_norm=None, k_norm=None, eps=0.0, rot=0,
           interleaved=False, freq=None):
    """(q_out, k_pool, v_pool) in float64: q_out NaN and the pools as they were where nothing is written.
    q [rows, heads, dim], k and v [rows, kv_heads, dim]."""
    n_pages, _, page_size, _ = k_pool.shape
    q_out = np.full(q.shape, np.nan)
    kp, vp = k_pool.astype(np.float64), v_pool.astype(np.float64)
    for b in range(len(length)):
        for r, p in new_rows(row_start, length, b):
            for h in range(q.shape[1]):
                q_out[r, h] = prepare_head(q[r, h], q_norm, eps, p, rot, interleaved, freq)
            at = slot(pages, b, p, n_pages, page_size)
            if at is None:
                continue
            for h in range(k.shape[1]):
                kp[at[0], h, at[1]] = prepare_head(k[r, h], k_norm, eps, p, rot, interleaved, freq)
                vp[at[0], h, at[1]] = v[r, h]
    return q_out, kp, vp


def sees(p, length, max_len, causal, window, sinks):
    """The keys a row at position p sees, before the pages are asked."""
    top = min(length, max_len)
    return [j for j in range(max(top, 0))
            if (not causal or j <= p) and (not window or j > p - window or j < sinks)]


def attention(k_pool, v_pool, row_start, length, pages, q, scale, causal=True, window=0, sinks=0, max_len=1 << 30):
    """(out, terms, count, vmax): out [rows, heads, dim] in float64, NaN for rows of no sequence; per row and head the
    largest sum of |scale q_f k_f| over the keys it sees, their number and the largest |v| among them."""
    n_pages, hk, page_size, dim = k_pool.shape
    g = q.shape[1] // hk
    out = np.full(q.shape, np.nan)
    terms, count, vmax = (np.zeros(q.shape[:2]) for _ in range(3))
    kp, vp = k_pool.astype(np.float64), v_pool.astype(np.float64)
    for b in range(len(length)):
        for r, p in new_rows(row_start, length, b):
            keys = sees(p, int(length[b]), max_len, causal, window, sinks)
            at = [s for s in (slot(pages, b, j, n_pages, page_size) for j in keys) if s is not None]
            if not at:
                out[r] = 0.0
                continue
            pg, sl = np.array(at).T
            for h in range(q.shape[1]):
                k, v, x = kp[pg, h // g, sl], vp[pg, h // g, sl], q[r, h].astype(np.float64)
                with np.errstate(invalid="ignore", over="ignore"):
                    s = scale * (k @ x)
                    w = np.exp(s - s.max())
                    out[r, h] = (w / w.sum()) @ v
                    terms[r, h] = abs(scale) * (np.abs(k) @ np.abs(x)).max()
                count[r, h], vmax[r, h] = len(at), np.abs(v).max()
    return out, terms, count, vmax
