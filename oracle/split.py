"""Decode attention in 64 bits over cache values that are given as such (bf16 rows or oracle/mx.py's values).  Test
infrastructure only.  Also returns what the derivation of a tolerance needs: sum_j w_j |v_j| for every output element."""
from __future__ import annotations

import torch


def attention(q, k_new, v_new, k_values, v_values, block_tables, context_lens, cu_q, cu_new, scale, block_causal=False, dbs=32):
    """q [T, H_q, hd], k_new / v_new [N, H_kv, hd], k_values / v_values fp64 [pages, page, H_kv, hd] (CPU).  Returns (out, spread,
    written): fp64 [T, H_q, hd] twice, and which token rows have a key to attend to at all.  Pages with an id outside the cache
    are skipped (their keys take no part); a row whose keys are all skipped is zero."""
    T, hq, hd = q.shape
    hkv = k_new.shape[1]
    g = hq // hkv
    pages, page = k_values.shape[:2] if k_values is not None else (0, 1)
    out, spread, written = torch.zeros(T, hq, hd, dtype=torch.float64), torch.zeros(T, hq, hd, dtype=torch.float64), torch.zeros(T, dtype=torch.bool)
    for s in range(len(cu_q) - 1):
        a, b = int(cu_q[s]), int(cu_q[s + 1])
        n0, n1 = int(cu_new[s]), int(cu_new[s + 1])
        ctx = int(context_lens[s]) if k_values is not None else 0
        if a == b or ctx + n1 - n0 == 0:
            continue
        written[a:b] = True
        pos = torch.arange(ctx)
        ids = block_tables[s].long()[pos // page] if ctx else pos
        ok = (ids >= 0) & (ids < pages)
        kk = [k_values[ids[ok], pos[ok] % page]] if ctx else []
        vv = [v_values[ids[ok], pos[ok] % page]] if ctx else []
        kk, vv = torch.cat(kk + [k_new[n0:n1].double()]), torch.cat(vv + [v_new[n0:n1].double()])
        n_ctx = int(ok.sum())
        i, j = torch.arange(b - a), torch.arange(kk.shape[0])
        seen = torch.ones(b - a, kk.shape[0], dtype=torch.bool)
        if block_causal:
            seen = (j[None] < n_ctx) | (j[None] - n_ctx < (i[:, None] // dbs + 1) * dbs)
        if kk.shape[0] == 0:
            continue
        for h in range(hq):
            dots = (q[a:b, h].double() @ kk[:, h // g].T) * scale
            dots = dots.masked_fill(~seen, float("-inf"))
            top = dots.max(-1, keepdim=True).values
            w = torch.exp(dots - torch.where(torch.isfinite(top), top, 0.0))
            l = w.sum(-1, keepdim=True)
            w = torch.where(l > 0, w / l, 0.0)
            out[a:b, h], spread[a:b, h] = w @ vv[:, h // g], w @ vv[:, h // g].abs()
    return out, spread, written
