"""Microscaled KV-cache elements in 64-bit numpy.  Test infrastructure only.

A block is 32 consecutive elements of a head row.  Definition (include/diffulex_amd.h, ``dfx_kv_store_mx``): scale exponent
e = the smallest integer >= -127 with A <= M 2^e for the block's largest magnitude A, codes nearest to x 2^-e with ties to
the even code, among those whose magnitude times 2^e is below 2^128; element = code value * 2^e.  A block with an infinity or NaN
has scale byte 255 and codes 0.  Pinned in
tests/test_oracle_mx.py against library casts, a brute-force search over all code values and the grids written out.
"""
from __future__ import annotations

import numpy as np
import torch

BLOCK = 32
LARGEST = {"e4m3": 448.0, "e2m1": 6.0}


def code_values(fmt: str) -> np.ndarray:
    """fp64 value of every code (E4M3: 256 codes, two NaN; E2M1: 16 codes)."""
    bits, m, bias = (7, 3, 7) if fmt == "e4m3" else (3, 1, 1)
    c = np.arange(1 << bits)
    ex, frac = c >> m, (c & ((1 << m) - 1)) / (1 << m)
    v = np.where(ex == 0, frac * 2.0 ** (1 - bias), (1 + frac) * 2.0 ** (ex - bias))
    if fmt == "e4m3":
        v[127] = np.nan
    return np.concatenate([v, -v])


def scale_bytes(x: np.ndarray, fmt: str) -> np.ndarray:
    """x: fp64 [..., 32 k] -> uint8 [..., k]."""
    a = np.abs(x.reshape(*x.shape[:-1], -1, BLOCK))
    bad = ~np.isfinite(a).all(-1)
    top = np.where(bad, 0.0, a.max(-1, initial=0.0, where=np.isfinite(a)))
    m, p = np.frexp(top / LARGEST[fmt])            # exact: the quotient by 7 * 2^n or 3 * 2^n is compared below
    e = p.astype(np.int64)                          # top / M = m 2^p with m in [0.5, 1): e = p, or p - 1 where m == 0.5
    e = np.where(m == 0.5, e - 1, e)
    # (division rounds: settle the two neighbours by comparing products, which are exact)
    e = np.where(top > LARGEST[fmt] * np.exp2(e.astype(float)), e + 1, e)
    e = np.where(top <= LARGEST[fmt] * np.exp2(e - 1.0), e - 1, e)
    e = np.where(top == 0, -127, np.maximum(e, -127))
    return np.where(bad, 255, e + 127).astype(np.uint8)


def quantise(x: torch.Tensor, fmt: str):
    """bf16 [..., hd] -> (codes uint8 [..., hd], one code each; scale bytes uint8 [..., hd / 32])."""
    xd = x.double().numpy()
    b = scale_bytes(xd, fmt)
    s = np.where(b == 255, 0.0, np.exp2(b.astype(float) - 127))[..., None]
    blocks = xd.reshape(*xd.shape[:-1], -1, BLOCK)
    y = np.divide(blocks, s, out=np.zeros_like(blocks), where=s > 0)
    grid = code_values(fmt)
    half = len(grid) // 2
    pos = grid[:half][np.isfinite(grid[:half])]
    mid = (pos[1:] + pos[:-1]) / 2
    a = np.abs(y)
    code = np.searchsorted(mid, a, side="left")      # number of midpoints below a: a tie stays at the lower code
    tie = (code < len(mid)) & (a == mid[np.minimum(code, len(mid) - 1)])
    code = np.where(tie & (code % 2 == 1), code + 1, code)
    last = np.searchsorted(pos, np.where(s > 0, 2.0 ** 128 / np.where(s > 0, s, 1.0), np.inf), side="left") - 1  # the largest below 2^128 / s
    code = np.minimum(code, last)
    code = np.where(np.signbit(y), code + half, code)
    code = np.where((b == 255)[..., None], 0, code)
    return torch.from_numpy(code.reshape(xd.shape).astype(np.uint8)), torch.from_numpy(b)


def pack(codes: torch.Tensor, fmt: str) -> torch.Tensor:
    """One code per element -> the cache's bytes."""
    if fmt == "e4m3":
        return codes
    c = codes.reshape(*codes.shape[:-1], -1, 2)
    return c[..., 0] | (c[..., 1] << 4)


def values(packed: torch.Tensor, scales: torch.Tensor, fmt: str) -> torch.Tensor:
    """fp64 element values of a cache's bytes."""
    c = packed.cpu().view(torch.uint8).numpy()
    if fmt == "e2m1":
        c = np.stack([c & 15, c >> 4], -1).reshape(*c.shape[:-1], -1)
    b = scales.cpu().view(torch.uint8).numpy().astype(np.int64)
    s = np.where(b == 255, np.nan, np.exp2(b - 127.0))
    v = code_values(fmt)[c].reshape(*c.shape[:-1], -1, BLOCK) * s[..., None]
    return torch.from_numpy(v.reshape(c.shape))
