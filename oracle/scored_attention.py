"""Paged attention with capped, biased, windowed and tree-masked scores, in 64
bits on the CPU, and bounds on what a kernel with 16-bit weights may differ by."""

from __future__ import annotations

import math

import torch


def gather_keys(cache, scales, table, kv_len, page_size, kv_layout):
    """(K, V) [kv_len, Hkv, D] in float64 of one request; scales: [pages, 2, Hkv] or None."""
    pos = torch.arange(kv_len)
    pages = torch.as_tensor(table, dtype=torch.long)[pos // page_size] if kv_len else torch.zeros(0, dtype=torch.long)
    c = cache.double()
    if kv_layout == "HND":
        c = c.transpose(-2, -3)
    kv = c[pages, :, pos % page_size]  # [keys, 2, Hkv, D]
    if scales is not None:
        kv = kv * scales.double()[pages][..., None]
    return kv[:, 0], kv[:, 1]


def scored_attention(q, cache, qo_indptr, kv_indptr, kv_indices, kv_lens, *, page_size, kv_layout="NHD", scales=None,
                     causal=False, visible=None, window_left=-1, prefix_lens=None, soft_cap=0.0, slopes=None,
                     sm_scale=None, weight_eps=2.0 ** -8):
    """(out, lse, bound on |out' - out|, bound on |lse' - lse|).  ``visible``: per
    request a [queries, keys] bool mask (a draft tree's), or None.

    The bounds: a weight rounded to 16 bits is off by weight_eps of itself, so the
    output by weight_eps * sum p |v|; a weight that falls below fp16's range by 2^-24 of the
    largest V; a score summed in fp32 over D products by (D + 8) 2^-24 of the sum of
    their magnitudes (doubled for the exponent's own error), a cap c computed as
    c - 2 c / (1 + e) by c 2^-21 (e is off by 2^-22 of itself, which moves the quotient by c / 2 of
    that, and the reciprocal by 2^-23 of up to 2 c), which changes every weight by as much; the result is rounded once to q's type."""
    hq, d = q.shape[1], q.shape[2]
    sm = d ** -0.5 if sm_scale is None else sm_scale
    outs, lses, tols, ltols = [], [], [], []
    half = torch.finfo(q.dtype).eps / 2
    for b, n_keys in enumerate(kv_lens):
        qs = q[qo_indptr[b]:qo_indptr[b + 1]].double()
        n = qs.shape[0]
        k, v = gather_keys(cache, scales, kv_indices[kv_indptr[b]:kv_indptr[b + 1]], n_keys, page_size, kv_layout)
        g = hq // k.shape[1]
        k, v = k.repeat_interleave(g, 1), v.repeat_interleave(g, 1)
        s = torch.einsum("qhd,khd->hqk", qs, k) * sm
        mag = torch.einsum("qhd,khd->hqk", qs.abs(), k.abs()) * abs(sm)
        at, me = torch.arange(n_keys), n_keys - n + torch.arange(n)[:, None]
        if soft_cap:
            s = soft_cap * torch.tanh(s / soft_cap)
        if slopes is not None:
            bias = slopes.double()[:, None, None] * (me - at).abs().double()
            s, mag = s - bias, mag + bias
        vis = torch.ones((n, n_keys), dtype=torch.bool)
        if visible is not None:
            vis = visible[b]
        elif causal:
            vis = at <= me
            if window_left >= 0:
                vis = vis & (at >= me - window_left)
            if prefix_lens is not None:
                vis = vis | (at < prefix_lens[b])
        # what no query may see must not matter, whatever it is
        s = torch.where(vis, s, torch.full_like(s, -math.inf))
        mag = torch.where(vis, mag, torch.zeros_like(mag))
        lse = torch.logsumexp(s, -1) if n_keys else torch.full((hq, n), -math.inf, dtype=torch.float64)
        p = torch.where(lse[..., None] == -math.inf, torch.zeros_like(s), torch.exp(s - lse[..., None]))
        o = torch.zeros((hq, n, d), dtype=torch.float64)
        a = torch.zeros_like(o)
        for h in range(hq):
            for i in range(n):
                seen = vis[i].nonzero()[:, 0]
                o[h, i] = p[h, i, seen] @ v[seen, h]
                a[h, i] = p[h, i, seen] @ v[seen, h].abs()
        ds = 2 * (d + 8) * 2.0 ** -24 * (mag.amax(-1) if n_keys else torch.zeros((hq, n))) + 2.0 ** -20 + soft_cap * 2.0 ** -21
        vmax = v[torch.isfinite(v)].abs().max() if n_keys else 0.0
        outs.append(o.transpose(0, 1))
        lses.append(lse.transpose(0, 1))
        tol = (weight_eps + 4 * ds[..., None]) * a + half * o.abs() + n_keys * 2.0 ** -24 * vmax + 1e-7
        tols.append(tol.transpose(0, 1))
        ltols.append((ds + (n_keys + 64) * 2.0 ** -24 + 2.0 ** -22 * lse.abs().nan_to_num(posinf=0)).transpose(0, 1))
    return torch.cat(outs), torch.cat(lses), torch.cat(tols), torch.cat(ltols)
