"""64-bit references of the serving operators (plain numpy and Python, nothing of the library)."""

from __future__ import annotations

import numpy as np


def batch_tables_ref(computed, new, tables, free, start, block_size, tokens):
    """build_batch_tables by its definition, one token at a time."""
    lim = 2**31 - 1
    c = [min(max(int(v), 0), lim) for v in computed]
    n = [min(max(int(v), 0), lim) for v in new]
    tables = np.array(tables, dtype=np.int64, copy=True)
    width = tables.shape[1]
    starts, seq, pos, slot, req = [0], [], [], [], []
    head = start
    for r, (cr, nr) in enumerate(zip(c, n)):
        nr = min(nr, tokens - starts[-1])
        have = min(width, -(-cr // block_size))
        need = min(width, -(-(cr + nr) // block_size))
        for j in range(have, need):
            tables[r, j] = free[head] if 0 <= head < len(free) else -1
            head += 1
        for i in range(nr):
            p = cr + i
            block = tables[r, p // block_size] if p // block_size < width else -1
            pos.append(p)
            slot.append(block * block_size + p % block_size if block >= 0 else -1)
            req.append(r)
        starts.append(starts[-1] + nr)
        seq.append(min(cr + nr, lim))
    pad = tokens - len(pos)
    return dict(tables=tables, query_starts=np.array(starts), seq_lens=np.array(seq, dtype=np.int64),
                positions=np.array(pos + [0] * pad, dtype=np.int64),
                slot_mapping=np.array(slot + [-1] * pad, dtype=np.int64),
                token_requests=np.array(req + [-1] * pad, dtype=np.int64), free_end=head)


def sample_ref(v, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """One row's token by the definition of sample_tokens, in 64 bits.  Returns (token, kept)."""
    v = np.asarray(v, np.float64)
    v = np.where(np.isnan(v), -np.inf, v)
    top = v.max()
    if not temperature > 0 or top == -np.inf:
        return int(np.argmax(v)), None
    w = np.zeros_like(v)
    w[v == top] = 1.0
    rest = (v < top) & (v > -np.inf)
    w[rest] = np.exp((v[rest] - top) / np.float64(temperature))
    order = np.argsort(-v, kind="stable")
    ws = w[order]
    n = int(top_k) if 0 < top_k < len(v) else len(v)
    s = np.concatenate([[0.0], np.cumsum(ws)])
    limit = n
    if top_p < 1:
        limit = max(1, int((s[:n] < np.float64(top_p) * s[n]).sum()))
    if min_p > 0:
        limit = min(limit, max(1, int((ws >= np.float64(min_p)).sum())))
    kept = np.sort(order[:limit])
    mass = np.cumsum(w[kept])
    u = 0.0 if not u > 0 else min(float(u), 1 - 2.0**-53)
    return int(kept[np.searchsorted(mass, u * mass[-1], side="right")]), kept


def lora_ref(base, x, a, b, ids, scales):
    """(out, bound) of lora_add in 64 bits: the result and how far an implementation with fp32
    sums, a rank-wide vector of 15 bits or more and one rounding to bf16 may be off."""
    base, x, a, b = (np.asarray(t, np.float64) for t in (base, x, a, b))
    out, err = base.copy(), np.zeros_like(base)
    rank, k = a.shape[1], a.shape[2]
    f = 2.0**-24  # half a step of fp32
    for t, i in enumerate(ids):
        if not 0 <= i < a.shape[0]:
            continue
        h = a[i] @ x[t]
        # k fp32 additions of exact products, each off by at most f of the sum of magnitudes
        eh = (k + 16) * f * (np.abs(a[i]) @ np.abs(x[t]))
        mag = np.abs(b[i]) @ np.abs(h)
        # the two bf16 parts drop at most 2^-15 of h; 2 rank additions follow
        ed = np.abs(b[i]) @ eh * (1 + 2.0**-14) + mag * (2.0**-15 + (2 * rank + 16) * f)
        delta = scales[i] * (b[i] @ h)
        out[t] += delta
        err[t] = abs(scales[i]) * ed + 4 * f * (np.abs(base[t]) + abs(scales[i]) * mag)
    return out, err + 2.0**-8 * (np.abs(out) + err) * (err > 0)
