"""Plain 64-bit (or bit-exact) restatements of the row, adapter and AdamW operators for their tests."""
from __future__ import annotations

import math

import numpy as np
import torch


def route_reference(index: np.ndarray, groups: int):
    """(order, slot, offsets); an out-of-range index has ~pair and ~place"""
    flat = index.reshape(-1)
    bad = (flat < -1) | (flat >= groups)
    key = np.where((flat < 0) | bad, groups, flat)
    order = np.argsort(key, kind="stable")
    slot = np.empty_like(order)
    slot[order] = np.arange(len(order))
    offsets = np.array([int((key < e).sum()) for e in range(groups + 1)])
    return np.where(bad[order], ~order, order), np.where(bad, ~slot, slot).reshape(index.shape), offsets


def adapter_reference(x, weight, bias, down, up, offsets, scale, relu, gy=None):
    """In 64 bits on the CPU: (y, sum of magnitudes behind each y, dx, its magnitudes, ddown, .., dup, ..) of the products' terms"""
    d = lambda t: t.detach().cpu().double()  # noqa: E731
    x, W, A, B = d(x), d(weight), d(down), d(up)
    s = d(scale) if isinstance(scale, torch.Tensor) else torch.full((A.shape[0],), float(scale), dtype=torch.float64)
    b = d(bias) if bias is not None else torch.zeros(W.shape[0], dtype=torch.float64)
    off = offsets.cpu().tolist()
    y, big = x @ W.t() + b, x.abs() @ W.t().abs() + b.abs()
    low = torch.zeros_like(y)  # the low-rank part's magnitudes
    for e in range(A.shape[0]):
        r = slice(off[e], off[e + 1])
        y[r] += s[e] * (x[r] @ A[e].t()) @ B[e].t()
        low[r] = s[e].abs() * (x[r].abs() @ A[e].t().abs()) @ B[e].t().abs()
    out = {"y": y, "y_terms": big, "y_low": low}
    if relu:
        out["y"] = torch.relu(y)
    if gy is not None:
        g = d(gy) * (y > 0) if relu else d(gy)
        dx, dxt, dxl = g @ W, g.abs() @ W.abs(), torch.zeros_like(x)
        dA, dAt, dB, dBt = (torch.zeros_like(t) for t in (A, A, B, B))
        for e in range(A.shape[0]):
            r = slice(off[e], off[e + 1])
            t, ta = s[e] * (g[r] @ B[e]), s[e].abs() * (g[r].abs() @ B[e].abs())
            u, ua = s[e] * (x[r] @ A[e].t()), s[e].abs() * (x[r].abs() @ A[e].t().abs())
            dx[r] += t @ A[e]
            dxl[r] = ta @ A[e].abs()
            dA[e], dAt[e] = t.t() @ x[r], ta.t() @ x[r].abs()
            dB[e], dBt[e] = g[r].t() @ u, g[r].abs().t() @ ua
        out |= {"dx": dx, "dx_terms": dxt, "dx_low": dxl, "ddown": dA, "ddown_terms": dAt, "dup": dB, "dup_terms": dBt}
    return out


def dither_codes(value: np.ndarray, scale: float, place: np.ndarray, step: int, mult: int, lowest: float) -> np.ndarray:
    """The e4m3 code value (as a float) each value of a block goes to: exact arithmetic in 64 bits."""
    y = np.abs(value.astype(np.float64)) / scale
    u = (((place.astype(object) * mult + step * 0x9E3779B1) % 2**32) // 2**12).astype(np.float64) / 2**20
    with np.errstate(divide="ignore"):
        ex = np.where(y > 0, np.floor(np.log2(np.where(y > 0, y, 1.0))), -6)
    ex = np.where(2.0**ex > y, ex - 1, ex)
    unit = 2.0 ** (np.maximum(ex, -6) - 3)
    q = np.minimum(np.floor(y / unit + u) * unit, 448.0)
    q = np.where(y > 0, np.maximum(q, lowest), q)
    return np.copysign(q, value)


def block_scale(value: np.ndarray) -> float:
    big = float(np.max(np.abs(value[np.isfinite(value)]), initial=0.0))
    if big == 0.0:
        return 1.0
    k = math.ceil(math.log2(big / 448.0) - 1e-12)
    while big / 2.0**k > 448.0:
        k += 1
    while k > -126 and big / 2.0 ** (k - 1) <= 448.0:
        k -= 1
    return 2.0 ** max(k, -126)


def adamw8_reference(p, g, m, ms, r, rs, step, lr=1e-3, b1=0.9, b2=0.999, eps=1e-8, wd=1e-2):
    """One step of the 8-bit form in the operator's own fp32 operations: code values (as floats) in and out, scales per 256."""
    f = np.float32
    n = len(p)
    rep = lambda s: np.repeat(s, 256)[:n].astype(f)  # noqa: E731
    mv, rv = m.astype(f) * rep(ms), r.astype(f) * rep(rs)
    vv = rv * rv
    mv = f(b1) * mv + f(1 - b1) * g
    vv = f(b2) * vv + f(1 - b2) * (g * g)
    rv = np.sqrt(vv)
    inv = f(1) / f(math.sqrt(1 - b2**step))
    p = p * f(1 - lr * wd) - f(lr / (1 - b1**step)) * (mv / (rv * inv + f(eps)))
    out_m, out_r, out_ms, out_rs = np.empty(n), np.empty(n), [], []
    for a in range(0, n, 256):
        b = slice(a, min(a + 256, n))
        place = np.arange(a, min(a + 256, n))
        sm, sr = block_scale(mv[b]), block_scale(rv[b])
        out_ms.append(sm)
        out_rs.append(sr)
        out_m[b] = dither_codes(mv[b], sm, place, step, 0x6A09E667, 0.0)
        out_r[b] = dither_codes(rv[b], sr, place, step, 0xBB67AE85, 2.0**-9)
    return p, out_m, np.array(out_ms), out_r, np.array(out_rs)
