"""Test helper: paged caches with chosen contents and the attention with modified scores in 64 bits."""
from __future__ import annotations

import math

import numpy as np

from paged_fixture import load_b200

BT = 16


class Caches:
    """Slots of (prefix length, ring tokens, ring cursor) on one paged layer; logical K/V of every slot in fp64.

    Everything the slots do not hold (other blocks, block tails, unused ring tokens) is NaN in the pool, and so are the
    tokens of `hidden` (slot -> list of fixed-region tokens that no row sees)."""

    def __init__(self, slots, kvh, hd, dtype, window, seed, hidden=None, slot_count=None):
        import torch
        self.b, self.torch = load_b200(), torch
        self.kvh, self.hd, self.W = kvh, hd, window
        self.slots = slots
        rng = np.random.default_rng(seed)
        rb = (window + BT - 1) // BT
        nb = [(p + BT - 1) // BT for p, _, _ in slots]
        total = sum(nb) + rb * len(slots) + 2
        ids = rng.permutation(total).astype(np.int32)
        stride = max(nb) + rb + 1
        table = np.full((len(slots), stride), -1, np.int32)
        at = 0
        tdt = torch.bfloat16 if dtype == self.b.BF16 else torch.float32
        pool = [np.full((total, kvh, BT, hd), np.nan, np.float32) for _ in range(2)]
        self.k, self.v = [], []
        for s, (p, ring, _) in enumerate(slots):
            table[s, :nb[s] + rb] = ids[at:at + nb[s] + rb]
            at += nb[s] + rb
            kv = [torch.tensor(rng.standard_normal((p + ring, kvh, hd)), dtype=torch.float32).to(tdt).double().numpy() for _ in range(2)]
            for x in kv:
                for t in (hidden or {}).get(s, []):
                    x[t] = np.nan
            for x, pl in zip(kv, pool):
                for t in range(p + ring):
                    e = t // BT if t < p else nb[s] + (t - p) // BT
                    o = t % BT if t < p else (t - p) % BT
                    pl[table[s, e], :, o] = x[t]
            self.k.append(kv[0])
            self.v.append(kv[1])
        self.table_np = table
        self.table = torch.tensor(table, device="cuda")
        self.layer = self.b.PagedLayer(total, kvh, hd, dtype, self.table, pools=tuple(torch.tensor(x, device="cuda").to(tdt) for x in pool))
        ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
        self.d_prefill = ints([p for p, _, _ in slots])
        self.d_len = ints([p + r for p, r, _ in slots])
        self.d_ring = ints([c for _, _, c in slots])

    def ring_age(self, slot):
        p, ring, cursor = self.slots[slot]
        r = np.arange(ring)
        newest = ring - 1 if ring < self.W else (cursor - 1) % self.W
        return (newest - r) % self.W


def attend(q, k, v, dist, heads, kvh, hd, scale=0.0, cap=0.0, slopes=None):
    """One row in 64 bits: q [heads * hd], visible keys k, v [n, kvh, hd], dist [n].
    Returns out [heads, hd], weights [heads, n], a bound on the kernel's fp32 error of out and of the weights."""
    out, tol = np.zeros((heads, hd)), np.zeros((heads, hd))
    n = len(k)
    w_all, w_tol = np.zeros((heads, n)), np.zeros((heads, n))
    s = scale or 1.0 / math.sqrt(hd)
    for h in range(heads if n else 0):
        kk, vv, qq = k[:, h * kvh // heads], v[:, h * kvh // heads], q[h * hd:(h + 1) * hd]
        x = kk @ qq * s
        size = np.abs(kk) @ np.abs(qq) * abs(s)
        if cap:
            x = cap * np.tanh(x / cap)
        far = np.zeros(n)
        if slopes is not None:
            far = slopes[h] * np.abs(dist)
            x = x - far
        e = np.exp(x - x.max())
        w = e / e.sum()
        out[h] = w @ vv
        # Relative error of a weight before the normalisation.  The dot product is summed by lanes of 8 terms and
        # a tree of at most 5 levels, q is scaled first: at most 16 roundings on the way of any term.  tanh 2 ulp, cap,
        # slope * distance and the differences: one rounding of 2^-24 each of their own size.  ex2: 2^-22.
        eps = 2.0 ** -24 * (16 * size.max() + 4 * (cap + far[w > 0].max(initial=0.0) + np.abs(x[w > 0]).max(initial=0.0))) + 2.0 ** -22
        # numerator and denominator each off by eps, plus the roundings of the sums (n terms, a rescale per 16 of them)
        rel = 2 * eps + (1.2 * n + 40) * 2.0 ** -24
        tol[h] = rel * (w @ np.abs(vv))
        w_all[h], w_tol[h] = w, rel * w + 2.0 ** -126
    return out, w_all, tol, w_tol


def check_out(torch, got, want, tol, what=""):
    g = got.double().cpu().numpy().reshape(want.shape)
    half = torch.finfo(got.dtype).eps / 2
    bound = tol + half * np.abs(want) * 1.001 + 1e-30
    assert np.isfinite(g).all(), what
    worst = (np.abs(g - want) / bound).max()
    assert worst <= 1.0, (what, worst)
