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

    Returns a dict in float64: O; lse; A = P |V| (the error scale of O); smax =
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
