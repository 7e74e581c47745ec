"""Statements in 64 bits of the operators over a paged cache and of the draw, for the tests (no code of the package)."""

import math

import numpy as np
import torch


def attention(q, k_pages, v_pages, q_start, kv_len, table, scale, window=0):
    """Host float64: out [N, Hq, D], its spread sum(p |v|) / sum(p) and sum(|v|) / sum(exp(s - max)) for tolerances."""
    q, kp, vp = (t.detach().cpu() for t in (q, k_pages, v_pages))
    N, Hq, D = q.shape
    n_pages, Hkv, page, _ = kp.shape
    out, spread, flat = (torch.zeros(N, Hq, D, dtype=torch.float64) for _ in range(3))
    for b, n in enumerate(kv_len):
        first, T = q_start[b], q_start[b + 1] - q_start[b]
        lo_all = max(0, n - T - window + 1) if window else 0
        j = torch.arange(lo_all, n)
        if T == 0 or n <= 0:
            continue
        ids = torch.tensor([table[b][int(x) // page] for x in j], dtype=torch.int64)
        there = (ids >= 0) & (ids < n_pages)
        at = torch.where(there, ids, torch.zeros_like(ids))
        k, v = (torch.where(there[:, None, None], p[at, :, j % page].double(), torch.zeros((), dtype=torch.float64)) for p in (kp, vp))   # [keys, Hkv, D]
        k, v = (x.repeat_interleave(Hq // Hkv, 1) for x in (k, v))
        s = torch.einsum("thd,jhd->thj", q[first:first + T].double(), k) * scale
        pos = torch.arange(n - T, n)[:, None]
        seen = j[None] <= pos
        if window:
            seen &= j[None] > pos - window
        s = s.masked_fill(~seen[:, None], -math.inf)
        top = s.amax(-1, keepdim=True)
        e = torch.where(seen[:, None], torch.exp(s - torch.where(top.isinf(), torch.zeros_like(top), top)), torch.zeros_like(s))
        l = e.sum(-1, keepdim=True)
        live = l > 0
        p = torch.where(live, e / torch.where(live, l, torch.ones_like(l)), torch.zeros_like(e))
        out[first:first + T] = torch.einsum("thj,jhd->thd", p, v)
        spread[first:first + T] = torch.einsum("thj,jhd->thd", p, v.abs())
        flat[first:first + T] = torch.einsum("thj,jhd->thd", seen[:, None].double().expand_as(e) / torch.where(live, l, torch.ones_like(l)), v.abs())
    return out, spread, flat


def draw(x, u, temperature=None, top_k=None, top_p=None, min_p=None):
    """Token ids of rows x [rows, cols] (float64 numpy)."""
    tokens = []
    for r in range(len(x)):
        z = x[r]
        T = 1.0 if temperature is None else float(temperature[r])
        if np.isnan(z).any() or z.max() == -np.inf:   # nothing to draw from
            tokens.append(0)
            continue
        if not T > 0:
            tokens.append(int(z.argmax()))
            continue
        rank = np.argsort(-z, kind="stable")
        if top_k is not None and top_k[r] > 0:
            rank = rank[:int(top_k[r])]
        with np.errstate(invalid="ignore"):
            w = np.where(z[rank] == z.max(), 1.0, np.exp((z[rank] - z.max()) / T))
        if top_p is not None and top_p[r] < 1:
            before = np.cumsum(w) - w
            keep = before < float(top_p[r]) * w.sum()
            keep[0] = True
            rank, w = rank[keep], w[keep]
        if min_p is not None and min_p[r] > 0:
            keep = w >= min(float(min_p[r]), 1.0)
            rank, w = rank[keep], w[keep]
        w = np.where(w < 2.0 ** -41, 0.0, w)   # by definition nothing that weighs less is drawn (it matters where u is 0)
        o = np.argsort(rank)
        rank, sums = rank[o], np.cumsum(w[o])
        tokens.append(int(rank[min(len(rank) - 1, np.searchsorted(sums, float(u[r]) * sums[-1], side="right"))]))
    return tokens
