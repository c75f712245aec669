"""Head-wise norm + rotation, masked attention and the bucketed relative bias in fp64 (CPU torch), gradients by autograd: the oracle of
mgld_vsr_amd.hip's transformer operators.  Written from the formulas, without the product's code."""
import math

import torch


def qk_norm_rope(x, pos, freqs, gamma, eps, interleaved):
    """x [rows, heads, d] fp64 -> the same, normed and turned"""
    d = x.shape[-1]
    y = x / torch.sqrt((x * x).sum(-1, keepdim=True) / d + eps)
    if gamma is not None:
        y = y * gamma
    n = 0 if freqs is None else len(freqs)
    if n == 0:
        return y
    ang = pos.double()[:, None, None] * freqs
    c, s = torch.cos(ang), torch.sin(ang)
    if interleaved:
        a, b = y[..., 0:2 * n:2], y[..., 1:2 * n:2]
        t = torch.stack([a * c - b * s, a * s + b * c], -1).flatten(-2)
    else:
        a, b = y[..., :n], y[..., n:2 * n]
        t = torch.cat([a * c - b * s, a * s + b * c], -1)
    return torch.cat([t, y[..., 2 * n:]], -1)


def visible(B, Nq, Nk, causal=False, docs=None, prefix=None, kv_len=None, q_pos0=None):
    """(bool [B, Nq, Nk], distance key - query [B, Nq, Nk])"""
    vis = torch.zeros(B, Nq, Nk, dtype=torch.bool)
    dist = torch.zeros(B, Nq, Nk, dtype=torch.long)
    for b in range(B):
        n = Nk if kv_len is None else min(max(int(kv_len[b]), 0), Nk)
        p0 = n - Nq if q_pos0 is None else q_pos0
        i, j = torch.arange(Nq)[:, None] + p0, torch.arange(Nk)[None, :]
        dist[b] = j - i
        v = (j < n).expand(Nq, Nk)
        if causal:
            v = v & ((j <= i) | (j < (0 if prefix is None else int(prefix[b]))))
        if docs is not None:
            v = v & (docs[0][b][:, None] == docs[1][b][None, :]) & (docs[1][b] >= 0)[None, :]
        vis[b] = v
    return vis, dist


def attention(q, k, v, vis, dist, scale, softcap=0.0, slopes=None, rel=None):
    """fp64 q [B, Nq, H, d], k / v [B, Nk, Hk, d] -> dict o, lse, and per query head P, score parts (for error bounds)"""
    B, Nq, H, d = q.shape
    G = H // k.shape[2]
    kk, vv = k.repeat_interleave(G, 2), v.repeat_interleave(G, 2)
    t = torch.matmul(q.permute(0, 2, 1, 3), kk.permute(0, 2, 3, 1)) * scale
    u = softcap * torch.tanh(t / softcap) if softcap else t
    s = u
    if slopes is not None:
        s = s - slopes[None, :, None, None] * dist.abs()[:, None]
    if rel is not None:
        R = rel.shape[1] // 2
        s = s + rel[:, dist.clamp(-R, R) + R].permute(1, 0, 2, 3)
    m = vis[:, None].expand_as(s)
    s = torch.where(m, s, torch.full_like(s, -math.inf))
    top = s.amax(-1, keepdim=True) if s.shape[-1] else torch.full(s.shape[:-1] + (1,), -math.inf, dtype=s.dtype)
    some = m.any(-1, keepdim=True)
    e = torch.where(m, torch.exp(torch.where(m, s, torch.zeros_like(s)) - torch.where(some, top, torch.zeros_like(top))), torch.zeros_like(s))
    tot = e.sum(-1, keepdim=True)
    P = e / torch.where(some, tot, torch.ones_like(tot))
    lse = torch.where(some, torch.where(some, top, torch.zeros_like(top)) + torch.log(torch.where(some, tot, torch.ones_like(tot))),
                      torch.full_like(tot, -math.inf))[..., 0]
    vm = vv.permute(0, 2, 1, 3)
    o = torch.matmul(P, vm).permute(0, 2, 1, 3)
    return {"o": o, "lse": lse, "P": P, "t": t, "u": u, "k": kk, "v": vv, "vis": m}


def rel_bucket(distance, num_buckets, max_distance, bidirectional):
    nb, first, n = num_buckets, 0, -distance
    if bidirectional:
        nb //= 2
        first, n = (nb if distance > 0 else 0), abs(distance)
    n = max(n, 0)
    exact = nb // 2
    if n < exact:
        return first + n
    # 1e-9: a distance on a border opens its bucket
    return first + min(nb - 1, exact + math.floor(math.log(n / exact) / math.log(max_distance / exact) * (nb - exact) + 1e-9))
