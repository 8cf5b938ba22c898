"""Float64 restatement of the operators around attention in a decoder layer.

`attention` is softmax attention of grouped heads over the keys each query
sees, with its gradients, one (batch, head) pair at a time; `norm_rope` is the
RMS norm of head vectors and their rotation, element by element. Used by the
tests only. Both also return what error bounds are stated against.
"""

from __future__ import annotations

import math

import torch


def attention(Q, K, V, scale, seen=None, dO=None):
    """Q (B, H, N, D); K, V (B, Hk, L, D); seen (B, N, L) bool or None.

    Returns a dict in float64: O; lse; A = P |V| (the error scale of O); W (B, Hk,
    L), the weight P of every key summed over its heads and queries; smax =
    largest sum_d scale |q_d k_d| of a seen pair; with dO also dQ, dK, dV and
    their scales aQ = (P W) |K| scale, aK = (P W)^T |Q| scale, aV = P^T |dO|, W
    = |dO| |V|^T + rowsum |dO| A.
    """
    Q, K, V = (t.detach().double().cpu() for t in (Q, K, V))
    B, H, N, D = Q.shape
    Hk, L = K.shape[1], K.shape[2]
    G = H // Hk
    f = dict(dtype=torch.float64)
    r = {"O": torch.zeros(B, H, N, D, **f), "A": torch.zeros(B, H, N, D, **f), "lse": torch.zeros(B, H, N, **f), "smax": 0.0}
    r["W"] = torch.zeros(B, Hk, L, **f)
    if dO is not None:
        dO = dO.detach().double().cpu()
        for k, t in (("dQ", Q), ("aQ", Q), ("dK", K), ("aK", K), ("dV", K), ("aV", K)):
            r[k] = torch.zeros(t.shape, **f)
    for b in range(B):
        ok = torch.ones(N, L, dtype=torch.bool) if seen is None else seen[b].cpu()
        cols = ok.any(0)  # what stands in keys that no query sees is never used
        for h in range(H):
            q = Q[b, h]
            k, v = (torch.where(cols[:, None], t[b, h // G], torch.zeros((), **f)) for t in (K, V))
            s = torch.where(ok, q @ k.t() * scale, torch.full((), -math.inf, **f))
            if L == 0:
                r["lse"][b, h] = -math.inf
                continue
            m = s.amax(1, keepdim=True)
            p = torch.exp(s - torch.where(m == -math.inf, torch.zeros_like(m), m))
            tot = p.sum(1, keepdim=True)
            r["lse"][b, h] = (m + tot.log()).squeeze(1)
            p = p / torch.where(tot == 0, torch.ones_like(tot), tot)
            r["O"][b, h], r["A"][b, h] = p @ v, p @ v.abs()
            r["W"][b, h // G] += p.sum(0)
            mag = torch.where(ok, q.abs() @ k.abs().t() * scale, torch.zeros((), **f))
            if mag.numel():
                r["smax"] = max(r["smax"], float(mag.max()))
            if dO is None:
                continue
            g = dO[b, h]
            ds = p * (g @ v.t() - (g * r["O"][b, h]).sum(1, keepdim=True)) * scale
            w = p * (g.abs() @ v.abs().t() + (g.abs() * r["A"][b, h]).sum(1, keepdim=True)) * scale
            r["dQ"][b, h], r["aQ"][b, h] = ds @ k, w @ k.abs()
            r["dK"][b, h // G] += ds.t() @ q
            r["aK"][b, h // G] += w.t() @ q.abs()
            r["dV"][b, h // G] += p.t() @ g
            r["aV"][b, h // G] += p.t() @ g.abs()
    return r


def lengths_seen(lengths, N, L, causal=False):
    """seen (B, N, L) of key counts (B,); causal: query i sees N - 1 - i fewer."""
    n = lengths.cpu().clamp(0, L).view(-1, 1, 1)
    if causal:
        n = n - (N - 1 - torch.arange(N)).view(1, N, 1)
    return (torch.arange(L) < n).expand(-1, N, -1)


def paged_rows(pages, table):
    """Every sequence's rows in order, (B, Hk, columns * page_size, D), row by row
    from pages (P, Hk, page_size, D) and table (B, columns); zeros where a table
    entry names no page."""
    pages, table = pages.detach().cpu(), table.cpu()
    count, Hk, size, D = pages.shape
    B, cols = table.shape
    out = torch.zeros(B, Hk, cols * size, D, dtype=pages.dtype)
    for b in range(B):
        for c in range(cols):
            if 0 <= int(table[b, c]) < count:
                out[b, :, c * size : (c + 1) * size] = pages[int(table[b, c])]
    return out


def chunk_seen(lengths, new_lengths, N, L):
    """seen (B, N, L) of the last m of n cached rows' queries, query i with the
    rows up to its own: j <= n - m + i. Queries i >= m see nothing."""
    B = lengths.numel()
    seen = torch.zeros(B, N, L, dtype=torch.bool)
    for b in range(B):
        n = min(max(int(lengths[b]), 0), L)
        m = N if new_lengths is None else min(max(int(new_lengths[b]), 0), N)
        for i in range(m):
            seen[b, i, : max(n - m + i + 1, 0)] = True
    return seen


def paged_append(K, V, K_pages, V_pages, table, lengths, new_lengths=None, weights=None):
    """New copies of (K_pages, V_pages, weights) with the new rows written one at
    a time, and the new lengths."""
    K, V, table = K.detach().cpu(), V.detach().cpu(), table.cpu()
    kp, vp = K_pages.detach().cpu().clone(), V_pages.detach().cpu().clone()
    w = None if weights is None else weights.cpu().clone()
    count, _, size, _ = kp.shape
    L, after = table.shape[1] * size, []
    for b in range(table.shape[0]):
        n = min(max(int(lengths[b]), 0), L)
        m = K.shape[2] if new_lengths is None else min(max(int(new_lengths[b]), 0), K.shape[2])
        after.append(min(n + m, L))
        for i in range(after[-1] - n):
            j = n + i
            if w is not None:
                w[b, :, j] = 0
            p = int(table[b, j // size])
            if 0 <= p < count:
                kp[p, :, j % size], vp[p, :, j % size] = K[b, :, i], V[b, :, i]
    return kp, vp, w, torch.tensor(after, dtype=lengths.dtype)


def paged_evict(K_pages, V_pages, weights, table, lengths, budget, recent):
    """New copies of (K_pages, V_pages, weights) after the eviction, and the new
    lengths: rows ranked by (NaN, weight, first place) with Python's sort."""
    kp, vp, w, table = K_pages.detach().cpu().clone(), V_pages.detach().cpu().clone(), weights.cpu().clone(), table.cpu()
    count, Hk, size, D = kp.shape
    L, after = table.shape[1] * size, []
    for b in range(table.shape[0]):
        n = min(max(int(lengths[b]), 0), L)
        after.append(min(n, budget))
        if n <= budget:
            continue
        ids = [int(p) for p in table[b]]
        for h in range(Hk):
            old = w[b, h].tolist()
            order = sorted(range(n - recent), key=lambda j: (0, 0.0, j) if math.isnan(old[j]) else (1, -old[j], j))  # noqa: B023
            kept = sorted(order[: budget - recent]) + list(range(n - recent, n))
            for pages in (kp, vp):
                rows = [pages[ids[j // size], h, j % size].clone() if 0 <= ids[j // size] < count
                        else torch.zeros(D, dtype=pages.dtype) for j in kept]
                for d, row in enumerate(rows):
                    if 0 <= ids[d // size] < count:
                        pages[ids[d // size], h, d % size] = row
            for d, j in enumerate(kept):
                w[b, h, d] = old[j]
    return kp, vp, w, torch.tensor(after, dtype=lengths.dtype)


def norm_rope(x, w, positions, inv_freq, eps, interleaved, dy=None):
    """x (B, H, S, D), w (D,), positions (S,) or (B, S). Returns a dict in
    float64: y; ay = |n_a| + |n_b| of each element's pair (its error scale);
    with dy also dx, dw, and the scales adx = r (|w dn| + |x| r^2 / D sum |x w
    dn|), adw = sum_rows |dn x r|, |dn| being |dy_a| + |dy_b|.
    """
    x, w = x.detach().double().cpu(), w.detach().double().cpu()
    B, H, S, D = x.shape
    pos = positions.cpu().double().expand(B, S)
    f = inv_freq.detach().double().cpu()
    half = f.numel()
    idx = torch.arange(half)
    a, b = (2 * idx, 2 * idx + 1) if interleaved else (idx, idx + half)
    cos, sin = (fn(pos[:, None, :, None] * f) for fn in (torch.cos, torch.sin))
    r = ((x * x).mean(-1, keepdim=True) + eps) ** -0.5
    n = x * r * w

    def turn(t, sgn):
        y, ab = t.clone(), t.abs()
        y[..., a] = t[..., a] * cos - sgn * t[..., b] * sin
        y[..., b] = t[..., b] * cos + sgn * t[..., a] * sin
        ab[..., a] = ab[..., b] = t[..., a].abs() + t[..., b].abs()
        return y, ab

    out = {}
    out["y"], out["ay"] = turn(n, 1.0)
    if dy is not None:
        dn, adn = turn(dy.detach().double().cpu(), -1.0)
        out["dw"] = (dn * x * r).sum((0, 1, 2))
        out["adw"] = (adn * (x * r).abs()).sum((0, 1, 2))
        out["dx"] = r * (w * dn) - x * r**3 * (x * w * dn).mean(-1, keepdim=True)
        out["adx"] = r * ((w * adn).abs() + x.abs() * r**2 * (x * w * adn).abs().mean(-1, keepdim=True))
    return out
