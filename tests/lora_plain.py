"""Low-rank adapters in 64 bits, row by row, with the error that 24-bit sums and the kernels' roundings may add."""
from __future__ import annotations

import numpy as np
import torch

HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}   # half a step, relative
TINY = {torch.float32: 0.0, torch.float16: 2.0 ** -25, torch.bfloat16: 0.0}                # half of the smallest fp16 step


def group_list(ids, slots, experts, G, E, T):
    """group of every entry, -1: none."""
    out = []
    for t in range(T):
        g = 0 if ids is None else int(ids[t])
        for j in range(slots):
            e = 0 if experts is None else int(experts[t][j])
            out.append(g * E + e if 0 <= g < G and 0 <= e < E else -1)
    return np.array(out)


def plain(y, x, a, b, group, scaling, slots=1, shared=False, dy=None):
    """{name: (value, largest error)} as float64 arrays: y, and with dy also dx, da, db.
    y [n, N], x [n or n / slots, K], a [groups, r, K], b [groups, N, r], scaling per group.

    A float32 sum of n products is off by at most (n + 64) 2^-23 of the sum of their sizes, whatever the order (the tensor cores
    cut off where floats round). u and v enter the next product as two 16-bit terms: 2^-16; float32 parameters as two terms there,
    2^-16 more. Gradients kept in float32 take three terms (2^-23), those rounded to 16 bits two."""
    out_half, out_tiny, p_half, p_tiny = HALF[y.dtype], TINY[y.dtype], HALF[a.dtype], TINY[a.dtype]
    f32 = a.dtype == torch.float32
    y, x, a, b = (t.detach().double().cpu().numpy() for t in (y, x, a, b))
    n, N = y.shape
    K, r = x.shape[1], a.shape[1]
    s = np.asarray(scaling, np.float64)
    bits = lambda m: (m + 64) * 2.0 ** -23  # noqa: E731
    vals, errs = y.copy(), np.zeros_like(y)
    dy = None if dy is None else dy.detach().double().cpu().numpy()
    dx, dxe = np.zeros_like(x), np.zeros_like(x)
    da, dae, db, dbe = np.zeros_like(a), np.zeros_like(a), np.zeros_like(b), np.zeros_like(b)
    two = 2.0 ** -16 * (2 if f32 else 1)
    last = 2.0 ** -22 if f32 else 2.0 ** -16
    for g in np.unique(group[group >= 0]):
        e = np.nonzero(group == g)[0]
        src = e // slots if shared else e
        u = x[src] @ a[g].T
        ue = (bits(K) + (2.0 ** -22 if f32 else 0)) * (np.abs(x[src]) @ np.abs(a[g]).T)
        vals[e] += s[g] * (u @ b[g].T)
        errs[e] += s[g] * (ue @ np.abs(b[g]).T + (two + bits(r)) * (np.abs(u) @ np.abs(b[g]).T))
        if dy is None:
            continue
        v = s[g] * (dy[e] @ b[g])
        ve = s[g] * (bits(N) + (2.0 ** -22 if f32 else 0)) * (np.abs(dy[e]) @ np.abs(b[g]))
        np.add.at(dx, src, v @ a[g])
        np.add.at(dxe, src, ve @ np.abs(a[g]) + (two + bits(r + slots)) * (np.abs(v) @ np.abs(a[g])))
        da[g] = v.T @ x[src]
        dae[g] = ve.T @ np.abs(x[src]) + (last + bits(len(e))) * (np.abs(v).T @ np.abs(x[src]))
        db[g] = s[g] * (dy[e].T @ u)
        dbe[g] = s[g] * (np.abs(dy[e]).T @ ue + (last + bits(len(e))) * (np.abs(dy[e]).T @ np.abs(u)))
    done = lambda v, err, half, tiny: (v, err * (1 + half) + half * np.abs(v) + tiny + 1e-30)  # noqa: E731
    res = {"y": done(vals, errs, out_half, out_tiny)}
    if dy is not None:
        res["dx"] = done(dx, dxe, out_half, out_tiny)
        res["da"], res["db"] = done(da, dae, p_half, p_tiny), done(db, dbe, p_half, p_tiny)
    return res


def check(got: torch.Tensor, want, name=""):
    """Every element within its bound; and the whole as near as roundings that point nowhere in particular leave it: half a step
    for 16 bits, 4e-6 for float32 (sqrt(n) 2^-24 with n up to 4200)."""
    value, bound = want
    v = got.detach().double().cpu().numpy().reshape(value.shape)
    off = np.abs(v - value)
    worst = np.unravel_index(np.argmax(off - bound), off.shape) if off.size else None
    assert (off <= bound).all(), f"{name}: {v[worst]} at {worst}, wanted {value[worst]} +- {bound[worst]:.3g}"
    norm = np.linalg.norm(value)
    if norm > 0:
        most = max(4e-6, HALF[got.dtype])
        assert np.linalg.norm(v - value) <= most * norm, f"{name}: {np.linalg.norm(v - value) / norm:.3g} of the norm"
