"""mgld_vsr_amd.hip's transformer operators against the fp64 oracle (oracle/transformer.py).

Tolerances are error bounds, element by element.  With u half a step of the type (eps / 2) and E the relative error of a probability from its
fp32 score (E = 2 (scale sum|q k| (d + 4) 2^-24 + 2^-20 softcap + 2^-20), two of them: numerator and normaliser):
  o   : u |o| + (u + E) sum P |v|                       (one rounding of the result, one of every probability)
  dv  : u |dv| + (u + E) sum P |do|
  dS  : P (d 2^-24 sum|do v| + tol(D)) + E |dS|,  tol(D) = sum P (d 2^-24 sum|do v| + E |dP|)
  dq  : u |dq| + scale sum (u |dT| + tol(dS)) |k|;  dk likewise with |q|;  drel: sum tol(dS) + 2^-14 sum |dS|
and for fp16 what the smallest step of the scaled operands leaves.
"""
import math

import pytest
import torch

from oracle import transformer as tr

pytestmark = pytest.mark.gpu
DEV = "cuda"
F16, BF16 = torch.float16, torch.bfloat16


def gen(seed):
    return torch.Generator().manual_seed(seed)


def randn(g, *shape, scale=1.0):
    return torch.randn(*shape, generator=g) * scale


def half_step(dt):
    return torch.finfo(dt).eps / 2


def check(name, got, ref, tol):
    got = got.detach().double().cpu()
    assert got.shape == ref.shape, (name, got.shape, ref.shape)
    bad = ~((got - ref).abs() <= tol)
    assert not bad.any(), (name, int(bad.sum()), float((got - ref).abs()[bad].max()), float(tol[bad].min() if isinstance(tol, torch.Tensor) else tol),
                           bad.nonzero()[0].tolist())


# ---- norm + rotation ---------------------------------------------------------------------------------------------------------------------------
ROPE = [  # rows, heads, kv heads, d, rot, interleaved, type, gammas
    (1, 32, 8, 128, 128, False, BF16, True), (1, 1, 1, 8, 8, False, F16, True), (7, 3, 0, 64, 32, True, F16, True), (33, 2, 2, 80, 40, False, BF16, False),
    (5, 4, 2, 72, 8, True, BF16, True), (130, 5, 1, 256, 256, False, F16, True), (4099, 3, 2, 64, 64, True, BF16, True), (4100, 16, 4, 128, 64, False, F16, True),
    (19, 2, 1, 96, 0, False, F16, True), (64, 0, 3, 40, 40, True, BF16, True), (2, 70, 70, 16, 16, False, BF16, True)]


def rope_case(rows, H, Hk, d, rot, dt, gammas, seed=1, cols=0):
    """q and k as column blocks of one buffer, with `cols` more columns between them"""
    g = gen(seed)
    buf = randn(g, rows, (H + Hk) * d + cols, scale=1.7).to(dt)
    q = buf[:, :H * d].unflatten(1, (H, d)) if H else None
    k = buf[:, H * d + cols:].unflatten(1, (Hk, d)) if Hk else None
    pos = torch.randint(0, 1 << 20, (rows,), generator=g)
    freqs = None if rot == 0 else 10000.0 ** (-2.0 * torch.arange(rot // 2, dtype=torch.float64) / rot)
    gq = 1 + 0.3 * randn(g, d) if gammas and H else None
    gk = 1 + 0.3 * randn(g, d) if gammas and Hk else None
    return buf, q, k, pos, freqs, gq, gk


def dev(x):
    return None if x is None else x.to(DEV)


@pytest.mark.parametrize("rows,H,Hk,d,rot,il,dt,gammas", ROPE)
def test_qk_norm_rope(hip, rows, H, Hk, d, rot, il, dt, gammas):
    buf, q, k, pos, freqs, gq, gk = rope_case(rows, H, Hk, d, rot, dt, gammas, cols=16)
    b = buf.to(DEV)
    dq = b[:, :H * d].unflatten(1, (H, d)) if H else None
    dk = b[:, H * d + 16:].unflatten(1, (Hk, d)) if Hk else None
    for p in (pos, pos.int()):
        out = hip.qk_norm_rope(dq, dk, p.to(DEV), dev(freqs), q_gamma=dev(gq), k_gamma=dev(gk), eps=1e-6, interleaved=il)
        for n, x, gm, y in (("q", q, gq, out[0]), ("k", k, gk, out[1])):
            if x is None:
                assert y is None
                continue
            ref = tr.qk_norm_rope(x.double(), pos, freqs, None if gm is None else gm.double(), 1e-6, il)
            # fp32: norm (d / 2 additions in tree order, rsqrt) 2^-20 relative; sines 2^-22 absolute; each element mixes two of its pair
            pair = tr.qk_norm_rope(x.double(), pos, None, None if gm is None else gm.double(), 1e-6, il).abs().amax(-1, keepdim=True)
            check(n, y, ref, half_step(dt) * ref.abs() + 2.0 ** -19 * pair + torch.finfo(dt).smallest_normal * torch.finfo(dt).eps)
    assert torch.equal(b.cpu(), buf), "inputs stay"


@pytest.mark.parametrize("rows,H,Hk,d,rot,il,dt,gammas", ROPE)
def test_qk_norm_rope_grad(hip, rows, H, Hk, d, rot, il, dt, gammas):
    buf, q, k, pos, freqs, gq, gk = rope_case(rows, H, Hk, d, rot, dt, gammas, seed=2)
    g = gen(3)
    b = buf.to(DEV)
    qd = b[:, :H * d].unflatten(1, (H, d)) if H else None
    kd = b[:, H * d:].unflatten(1, (Hk, d)) if Hk else None
    gqo = randn(g, rows, H, d).to(dt) if H else None
    gko = randn(g, rows, Hk, d).to(dt) if Hk else None
    kw = dict(q_gamma=dev(gq), k_gamma=dev(gk), eps=1e-6, interleaved=il)
    a = hip.qk_norm_rope_grad(qd, kd, pos.to(DEV), dev(freqs), dev(gqo), dev(gko), **kw)
    again = hip.qk_norm_rope_grad(qd, kd, pos.to(DEV), dev(freqs), dev(gqo), dev(gko), **kw)
    for n, x, gm, go, dx, dg, dx2, dg2 in (("q", q, gq, gqo, a[0], a[2], again[0], again[2]), ("k", k, gk, gko, a[1], a[3], again[1], again[3])):
        if x is None:
            assert dx is None and dg is None
            continue
        x64 = x.double().requires_grad_()
        g64 = None if gm is None else gm.double().requires_grad_()
        y = tr.qk_norm_rope(x64, pos, freqs, g64, 1e-6, il)
        grads = torch.autograd.grad(y, [x64] + ([g64] if g64 is not None else []), go.double())
        # every term of dx is at most r (|g z| + |x r| mean|g z x r|): bounded by its largest over the head
        r = 1 / torch.sqrt((x.double() ** 2).mean(-1, keepdim=True) + 1e-6)
        z = (go.double().abs().amax(-1, keepdim=True) * 1.4143) * (1 if gm is None else gm.double().abs().max())
        big = r * z * (1 + (x.double() * r).abs().amax(-1, keepdim=True))
        check("d" + n, dx, grads[0], half_step(dt) * grads[0].abs() + 2.0 ** -18 * big + torch.finfo(dt).smallest_normal * torch.finfo(dt).eps)
        if gm is None:
            assert dg is None
        else:
            xr = (x.double() * r).abs()
            heads = x.shape[1]
            # a block's fp32 sums: at most rows / (blocks) * heads + 64 additions of terms |z x r|
            terms = (go.double().abs().amax(-1, keepdim=True) * 1.4143 * xr).sum((0, 1))
            check("d" + n + "_gamma", dg, grads[1], 2.0 ** -24 * (rows / 256 * heads + 72) * terms + 1e-30)
            assert torch.equal(dg, dg2)
        assert torch.equal(dx, dx2)


def test_qk_norm_rope_in_place_and_zero_rows(hip):
    buf, q, k, pos, freqs, gq, gk = rope_case(50, 4, 2, 64, 64, F16, True)
    b = buf.to(DEV)
    qd, kd = b[:, :256].unflatten(1, (4, 64)), b[:, 256:].unflatten(1, (2, 64))
    kw = dict(q_gamma=gq.to(DEV), k_gamma=gk.to(DEV))
    ref = hip.qk_norm_rope(qd, kd, pos.to(DEV), freqs.to(DEV), **kw)
    go = torch.randn(50, 4, 64, device=DEV).half()
    gko = torch.randn(50, 2, 64, device=DEV).half()
    gref = hip.qk_norm_rope_grad(qd, kd, pos.to(DEV), freqs.to(DEV), go, gko, **kw)
    ga, gb = go.clone(), gko.clone()
    got = hip.qk_norm_rope_grad(qd, kd, pos.to(DEV), freqs.to(DEV), ga, gb, dq=ga, dk=gb, **kw)
    assert all(torch.equal(x, y) for x, y in zip(got, gref)) and got[0] is ga
    hip.qk_norm_rope(qd, kd, pos.to(DEV), freqs.to(DEV), q_out=qd, k_out=kd, **kw)
    assert torch.equal(qd, ref[0]) and torch.equal(kd, ref[1])
    # 4-D tensors in another order: [heads, rows, d]
    t = torch.randn(4, 50, 64, device=DEV).half()
    a = hip.qk_norm_rope(t.transpose(0, 1), None, pos.to(DEV), freqs.to(DEV))[0]
    c = hip.qk_norm_rope(t.transpose(0, 1).contiguous(), None, pos.to(DEV), freqs.to(DEV))[0]
    assert torch.equal(a, c)
    e = torch.empty(0, 4, 64, device=DEV, dtype=F16)
    p0 = torch.empty(0, dtype=torch.int64, device=DEV)
    assert hip.qk_norm_rope(e, None, p0, freqs.to(DEV))[0].shape == (0, 4, 64)
    z = hip.qk_norm_rope_grad(e, None, p0, freqs.to(DEV), e, None, q_gamma=gq.to(DEV))
    assert z[0].shape == (0, 4, 64) and float(z[2].abs().max()) == 0


# ---- attention -----------------------------------------------------------------------------------------------------------------------------------
def docs_of(g, B, N, pad=0, sort=True):
    ids = torch.randint(0, max(2, N // 40 + 2), (B, N), generator=g, dtype=torch.int32)
    if sort:
        ids = ids.sort(1).values
    if pad:
        ids[:, N - pad:] = -1
    return ids


ATT = {  # name: B, Nq, Nk, H, Hk, d, options
    "one": (1, 1, 1, 1, 1, 64, {}),
    "text": (3, 77, 77, 4, 4, 64, dict(causal=True)),
    "plain": (2, 130, 200, 2, 2, 64, {}),
    "d128": (1, 129, 257, 2, 1, 128, dict(causal=True)),
    "d8": (2, 40, 70, 2, 2, 8, {}),
    "d72": (1, 65, 131, 3, 1, 72, dict(causal=True, softcap=20.0)),
    "d40_slopes": (1, 100, 100, 2, 2, 40, dict(slopes=True, causal=True)),
    "cap": (2, 191, 191, 4, 2, 128, dict(causal=True, softcap=30.0, loud=4.0)),
    "cap_d64": (1, 150, 300, 2, 2, 64, dict(softcap=5.0, loud=6.0)),
    "docs": (2, 333, 333, 2, 1, 64, dict(docs=13)),
    "docs_causal_cap": (2, 300, 300, 2, 2, 128, dict(docs=70, causal=True, softcap=15.0, loud=3.0)),
    "docs_unsorted": (1, 200, 200, 2, 2, 64, dict(docs=5, unsorted=True)),
    "docs_cross": (2, 90, 170, 2, 2, 64, dict(docs=9, slopes=True)),
    "all_padding": (1, 70, 70, 2, 2, 64, dict(docs=70)),
    "prefix": (3, 160, 160, 4, 2, 64, dict(causal=True, prefix=[0, 50, 160])),
    "prefix_d128": (2, 140, 140, 2, 1, 128, dict(causal=True, prefix=[-5, 500])),
    "lens": (4, 100, 100, 2, 2, 64, dict(kv_len=[100, 0, 1, 65], q_pos0=0, causal=True)),
    "lens_end": (3, 20, 150, 2, 2, 128, dict(kv_len=[150, 7, 200], causal=True)),
    "behind": (1, 30, 50, 2, 2, 64, dict(causal=True, q_pos0=-12)),
    "ahead": (1, 30, 50, 2, 2, 64, dict(causal=True, q_pos0=1000, slopes=True)),
    "rel": (2, 100, 100, 3, 3, 64, dict(rel=20, q_pos0=0)),
    "rel_causal_cap": (2, 140, 140, 4, 2, 128, dict(rel=33, causal=True, softcap=12.0, loud=3.0)),
    "rel_wide": (1, 70, 200, 2, 2, 64, dict(rel=1024)),
    "rel0": (1, 70, 70, 2, 1, 128, dict(rel=0, causal=True)),
    "rel_docs": (2, 200, 200, 2, 2, 64, dict(rel=17, docs=11)),
    "token": (3, 1, 300, 8, 2, 128, dict(causal=True, kv_len=[300, 129, 1], softcap=25.0, loud=3.0)),
    "tokens": (2, 5, 700, 8, 1, 64, dict(causal=True, slopes=True)),
    "token_long": (1, 1, 5000, 4, 4, 64, {}),
    "token_long128": (1, 2, 4100, 6, 2, 128, dict(causal=True)),
    "token_rel": (2, 3, 900, 4, 2, 64, dict(rel=40, causal=True, kv_len=[900, 100])),
    "token_docs": (2, 2, 600, 4, 2, 64, dict(docs=20)),
    "token_empty": (2, 1, 200, 4, 4, 64, dict(kv_len=[0, 200], causal=True)),
    "rows60_long": (1, 60, 2300, 2, 1, 128, dict(causal=True, prefix=[1000])),
    "many_heads": (1, 33, 33, 24, 3, 64, dict(causal=True)),
    "long": (1, 1100, 1100, 1, 1, 64, dict(causal=True)),
}


def problem(name, dt, seed=0):
    B, Nq, Nk, H, Hk, d, opt = ATT[name]
    opt = dict(opt)
    g = gen(seed + 17)
    loud = opt.pop("loud", 1.0)
    q, k, v, do = randn(g, B, Nq, H, d, scale=loud).to(dt), randn(g, B, Nk, Hk, d).to(dt), randn(g, B, Nk, Hk, d).to(dt), randn(g, B, Nq, H, d).to(dt)
    kw = dict(scale=d ** -0.5, causal=opt.get("causal", False), softcap=opt.get("softcap", 0.0), q_pos0=opt.get("q_pos0"))
    unsorted = opt.pop("unsorted", False)
    if "docs" in opt:
        dk = docs_of(g, B, Nk, opt["docs"], not unsorted)
        dq = dk if Nq == Nk else dk[:, Nk - Nq:].contiguous()
        kw["docs"] = (dq, dk)
    if "prefix" in opt:
        kw["prefix"] = torch.tensor(opt["prefix"], dtype=torch.int32)
    if "kv_len" in opt:
        kw["kv_len"] = torch.tensor(opt["kv_len"], dtype=torch.int32)
    if opt.get("slopes"):
        kw["slopes"] = 2.0 ** -torch.arange(1, H + 1).float()
    if "rel" in opt:
        kw["rel"] = randn(g, H, 2 * opt["rel"] + 1)
    return q, k, v, do, kw


def on_gpu(kw):
    def mv(x):
        return tuple(mv(y) for y in x) if isinstance(x, tuple) else x.to(DEV) if isinstance(x, torch.Tensor) else x
    return {n: mv(x) for n, x in kw.items()}


def reference(q, k, v, do, kw, grads=True):
    """fp64 results and their bounds"""
    dt, u = q.dtype, half_step(q.dtype)
    B, Nq, H, d = q.shape
    Nk, Hk = k.shape[1], k.shape[2]
    vis, dist = tr.visible(B, Nq, Nk, kw["causal"], kw.get("docs"), kw.get("prefix"), kw.get("kv_len"), kw.get("q_pos0"))
    leaves = [x.double().requires_grad_(grads) for x in (q, k, v)]
    rel = kw["rel"].double().requires_grad_(grads) if "rel" in kw else None
    cap, scale = kw["softcap"], kw["scale"]
    r = tr.attention(*leaves, vis, dist, scale, cap, kw["slopes"].double() if "slopes" in kw else None, rel)
    res, tol = {"o": r["o"], "lse": r["lse"]}, {}
    with torch.no_grad():
        tiny = torch.finfo(dt).smallest_normal * torch.finfo(dt).eps
        P, kk, vv = r["P"], r["k"], r["v"]
        big = torch.matmul(q.double().abs().permute(0, 2, 1, 3), kk.abs().permute(0, 2, 3, 1)) * scale
        bias = 0.0
        if "slopes" in kw:
            bias = float((kw["slopes"].max() * (dist * vis).abs().max()).item())
        if rel is not None:
            bias = float(rel.abs().max())
        es = float(big.max() if big.numel() else 0) * (d + 4) * 2.0 ** -24 + cap * 2.0 ** -20 + (bias + 1) * 2.0 ** -20
        E = 2 * es
        to = u * r["o"].abs() + (u + E) * torch.matmul(P, vv.abs().permute(0, 2, 1, 3)).permute(0, 2, 1, 3) * 1.02 + tiny
        tol["o"], tol["lse"] = to, es + r["lse"].abs().nan_to_num(posinf=0) * 2.0 ** -21 + 2.0 ** -20
    if not grads:
        return res, tol
    do64 = do.double()
    out = torch.autograd.grad(r["o"], leaves + ([rel] if rel is not None else []), do64, allow_unused=True)
    out = [torch.zeros_like(x) if gx is None else gx for x, gx in zip(leaves + [rel], out)]
    res.update(dq=out[0], dk=out[1], dv=out[2])
    with torch.no_grad():
        dob = do64.permute(0, 2, 1, 3)
        dP = torch.matmul(dob, vv.permute(0, 2, 3, 1))
        D = (do64 * r["o"]).sum(-1).permute(0, 2, 1)[..., None]
        dS = P * (dP - D)
        tdP = torch.matmul(dob.abs(), vv.abs().permute(0, 2, 3, 1)) * (d + 4) * 2.0 ** -24
        tD = (P * (tdP + E * dP.abs())).sum(-1, keepdim=True) * 1.02
        tS = P * (tdP + tD) + E * (dS.abs() + P * tD)
        f = 1 - (r["u"] / cap) ** 2 if cap else torch.ones_like(dS)
        dT = dS * f
        tT = (tS * f + dS.abs() * 2.0 ** -20) * 1.02 + u * dT.abs()
        amax = float(do64.abs().max()) if do64.numel() else 0.0
        seen = r["vis"].double()
        fl = dict(q=amax * 2.0 ** -29, k=amax * 2.0 ** -24, v=2.0 ** -34) if dt == F16 else dict(q=0, k=0, v=0)      # half a smallest step over the scale

        def fold(x):                                   # the heads that share a key head
            return x.permute(0, 2, 1, 3).unflatten(2, (Hk, H // Hk)).sum(3)

        tol["dq"] = (u * res["dq"].abs() + scale * torch.matmul(tT + fl["q"] * seen, kk.abs().permute(0, 2, 1, 3)).permute(0, 2, 1, 3) * 1.02 + tiny)
        tol["dk"] = u * res["dk"].abs() + scale * fold(torch.matmul((tT + fl["k"] * seen).transpose(2, 3), q.double().abs().permute(0, 2, 1, 3))) * 1.02 + tiny
        tol["dv"] = u * res["dv"].abs() + fold(torch.matmul(((u + E) * P + fl["v"] * seen).transpose(2, 3), dob.abs())) * 1.02 + tiny
        if rel is not None:
            res["drel"] = out[3]
            R = rel.shape[1] // 2
            idx = (dist.clamp(-R, R) + R)
            t = torch.zeros_like(out[3])
            for b in range(B):
                for h in range(H):
                    t[h].index_add_(0, idx[b].flatten(), (tS[b, h] * 1.02 + 2.0 ** -14 * dS[b, h].abs()).flatten())
            tol["drel"] = t + 1e-30
    return {n: x.detach() for n, x in res.items()}, tol


def check_lse(got, ref, tol):
    got = got.double().cpu()
    none = torch.isinf(ref)
    assert torch.equal(torch.isinf(got) & (got < 0), none)
    check("lse", torch.where(none, torch.zeros_like(got), got), torch.where(none, torch.zeros_like(ref), ref), tol)


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("name", list(ATT))
def test_masked_attention(hip, name, dt):
    q, k, v, do, kw = problem(name, dt)
    res, tol = reference(q, k, v, do, kw, grads=False)
    o, lse = hip.masked_attention(q.to(DEV), k.to(DEV), v.to(DEV), **on_gpu(kw))
    check("o", o, res["o"], tol["o"])
    check_lse(lse, res["lse"], tol["lse"])


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("name", list(ATT))
def test_masked_attention_grad(hip, name, dt):
    q, k, v, do, kw = problem(name, dt, seed=5)
    res, tol = reference(q, k, v, do, kw)
    g = [x.to(DEV) for x in (q, k, v)]
    kg = on_gpu(kw)
    o, lse = hip.masked_attention(*g, **kg)
    out = hip.masked_attention_grad(*g, o, lse, do.to(DEV), **kg)
    again = hip.masked_attention_grad(*g, o, lse, do.to(DEV), **kg)
    for n, x, y in zip(("dq", "dk", "dv", "drel"), out, again):
        if n not in res:
            assert x is None
            continue
        check(n, x, res[n], tol[n])
        assert torch.equal(x, y), n


@pytest.mark.parametrize("name", ["text", "d128", "cap", "docs", "token", "tokens", "rel", "lens_end"])
def test_masked_attention_strides(hip, name):
    """column blocks of one buffer, [B, heads, N, d] tensors, results into slices of wider buffers: the bits of contiguous tensors"""
    q, k, v, do, kw = problem(name, BF16, seed=9)
    kg = on_gpu(kw)
    B, Nq, H, d = q.shape
    Nk, Hk = k.shape[1:3]
    c = [x.to(DEV) for x in (q, k, v, do)]
    o, lse = hip.masked_attention(*c[:3], **kg)
    grads = hip.masked_attention_grad(*c[:3], o, lse, c[3], **kg)
    kv = torch.empty(B, Nk, 2 * Hk * d + 8, dtype=BF16, device=DEV)
    ks, vs = kv[..., :Hk * d].unflatten(2, (Hk, d)), kv[..., Hk * d + 8:].unflatten(2, (Hk, d))
    ks.copy_(c[1]), vs.copy_(c[2])
    qs = c[0].transpose(1, 2).contiguous().transpose(1, 2)
    wide = torch.full((B, Nq, H * d + 24), 7.0, dtype=BF16, device=DEV)
    os_ = wide[..., 16:16 + H * d].unflatten(2, (H, d))
    o2, lse2 = hip.masked_attention(qs, ks, vs, o=os_, **kg)
    assert o2 is os_ and torch.equal(o2, o) and torch.equal(lse2, lse)
    assert float((wide[..., :16] - 7).abs().max()) == 0 and float((wide[..., 16 + H * d:] - 7).abs().max()) == 0
    dkv = torch.full_like(kv, 7.0)
    dks, dvs = dkv[..., :Hk * d].unflatten(2, (Hk, d)), dkv[..., Hk * d + 8:].unflatten(2, (Hk, d))
    out = hip.masked_attention_grad(qs, ks, vs, o2, lse2, c[3].transpose(1, 2).contiguous().transpose(1, 2), dk=dks, dv=dvs, **kg)
    for x, y in zip(out, grads):
        assert (x is None and y is None) or torch.equal(x, y)
    assert float((dkv[..., Hk * d:Hk * d + 8] - 7).abs().max()) == 0
    # one key / value row for the whole batch (batch stride 0)
    if "kv_len" not in kw:
        ke, ve = c[1][:1].expand(B, -1, -1, -1), c[2][:1].expand(B, -1, -1, -1)
        x, _ = hip.masked_attention(c[0], ke, ve, **kg)
        y, _ = hip.masked_attention(c[0], ke.contiguous(), ve.contiguous(), **kg)
        assert torch.equal(x, y)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf"), "max"])
@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("Nq,Nk,H,Hk,d", [(150, 150, 4, 2, 64), (130, 130, 2, 2, 128), (1, 200, 4, 1, 64), (3, 900, 4, 4, 128)])
def test_masked_places_hold_anything(hip, Nq, Nk, H, Hk, d, dt, bad):
    """values that a query does not see: past the length, ahead of it, in padding, in another document"""
    if bad == "max":
        bad = torch.finfo(dt).min
    g = gen(3)
    q, k, v = randn(g, 2, Nq, H, d).to(dt), randn(g, 2, Nk, Hk, d).to(dt), randn(g, 2, Nk, Hk, d).to(dt)
    n = Nk - 30
    lens = torch.tensor([n, Nk], dtype=torch.int32)
    docs = torch.zeros(2, Nk, dtype=torch.int32)
    docs[1, 20:60] = 1
    docs[1, Nk - 10:] = -1
    dq = docs[:, Nk - Nq:].clone()
    if Nq <= 3:
        dq[:] = 0
    kw = dict(causal=True, kv_len=lens, docs=(dq, docs), scale=d ** -0.5, softcap=0.0, q_pos0=Nk - Nq)
    res, tol = reference(q, k, v, torch.zeros_like(q), kw, grads=False)
    kb, vb = k.clone(), v.clone()
    for x in (kb, vb):
        x[0, n:] = bad
        x[1, Nk - 10:] = bad
    o, lse = hip.masked_attention(q.to(DEV), kb.to(DEV), vb.to(DEV), **on_gpu(kw))
    check("o", o, res["o"], tol["o"])
    check_lse(lse, res["lse"], tol["lse"])
    # document 1's values are seen by its own queries alone; a future value by later queries alone
    v2 = vb.clone()
    v2[1, 40] = bad
    o2, _ = hip.masked_attention(q.to(DEV), kb.to(DEV), v2.to(DEV), **on_gpu(kw))
    vis, _ = tr.visible(2, Nq, Nk, True, kw["docs"], None, lens, Nk - Nq)
    blind = ~vis[:, :, 40]
    blind[0] = True
    m = blind[:, :, None, None].expand_as(res["o"])
    check("o blind", torch.where(m, o2.cpu().double(), res["o"]), res["o"], tol["o"])
    if bad != torch.finfo(dt).min and bool((~blind).any()):
        assert not torch.isfinite(o2.cpu()[~m]).all()


def test_masked_gradient_ignores_padding(hip):
    """keys and values past the length or in padding may hold anything; their gradients are zeros"""
    g = gen(4)
    q, k, v, do = (randn(g, 2, 100, 2, 64).half() for _ in range(4))
    docs = torch.zeros(2, 100, dtype=torch.int32)
    docs[1, 70:] = -1
    kw = dict(causal=True, kv_len=torch.tensor([64, 100], dtype=torch.int32), docs=(docs, docs), scale=0.125, softcap=0.0, q_pos0=0)
    res, tol = reference(q, k, v, do, kw)
    for x in (k, v):
        x[0, 64:] = float("nan")
        x[1, 70:] = float("inf")
    q[1, 70:], do[1, 70:] = float("nan"), float("nan")
    c = [x.to(DEV) for x in (q, k, v)]
    kg = on_gpu(kw)
    o, lse = hip.masked_attention(*c, **kg)
    check("o", o, res["o"], tol["o"])
    dq, dk, dv, _ = hip.masked_attention_grad(*c, o, lse, do.to(DEV), **kg)
    for n, x in (("dq", dq), ("dk", dk), ("dv", dv)):
        check(n, x, res[n], tol[n])
    assert float(dk[0, 64:].abs().max()) == 0 and float(dv[1, 70:].abs().max()) == 0 and float(dq[1, 70:].abs().max()) == 0


@pytest.mark.parametrize("what", ["before the first key", "a document without keys", "keys ahead of every query"])
@pytest.mark.parametrize("dt,d", [(F16, 64), (BF16, 128)])
def test_masked_gradient_ignores_what_nothing_sees(hip, dt, d, what):
    """queries that see no key, and keys that no query sees, may hold anything; their gradients are zeros"""
    g = gen(14)
    q, k, v, do = (randn(g, 2, 150, 2, d).to(dt) for _ in range(4))
    kw = dict(causal=True, scale=d ** -0.5, softcap=0.0, q_pos0=0)
    gone_q, gone_k = torch.zeros(2, 150, dtype=torch.bool), torch.zeros(2, 150, dtype=torch.bool)
    if what == "before the first key":                       # the queries are the last ones of a shorter sequence
        kw.update(q_pos0=None, kv_len=torch.tensor([70, 150], dtype=torch.int32))
        gone_q[0, :80] = True
        gone_k[0, 70:] = True
    elif what == "a document without keys":
        dq = torch.zeros(2, 150, dtype=torch.int32)
        dk = dq.clone()
        dq[1, 40:71] = 9
        kw.update(docs=(dq, dk))
        gone_q[1, 40:71] = True
    else:
        kw.update(q_pos0=-45)
        gone_q[:, :45] = True
        gone_k[:, 105:] = True
    res, tol = reference(q, k, v, do, kw)
    for x, m in ((q, gone_q), (do, gone_q), (k, gone_k), (v, gone_k)):
        x[m] = float("nan")
    c = [x.to(DEV) for x in (q, k, v)]
    kg = on_gpu(kw)
    o, lse = hip.masked_attention(*c, **kg)
    check("o", o, res["o"], tol["o"])
    dq, dk, dv, _ = hip.masked_attention_grad(*c, o, lse, do.to(DEV), **kg)
    for n, x in (("dq", dq), ("dk", dk), ("dv", dv)):
        check(n, x, res[n], tol[n])
    assert not dq.cpu()[gone_q].any() and not dk.cpu()[gone_k].any() and not dv.cpu()[gone_k].any()


@pytest.mark.parametrize("mag", [1e-4, 3e3])
def test_fp16_gradient_at_other_magnitudes(hip, mag):
    """the gradient of a small or large loss: dS is scaled before its rounding to fp16"""
    q, k, v, do, kw = problem("long", F16, seed=6)
    do = (do.float() * mag).half()
    res, tol = reference(q, k, v, do, kw)
    c = [x.to(DEV) for x in (q, k, v)]
    o, lse = hip.masked_attention(*c, **on_gpu(kw))
    for n, x in zip(("dq", "dk", "dv"), hip.masked_attention_grad(*c, o, lse, do.to(DEV), **on_gpu(kw))):
        ref = res[n].clamp(-65504, 65504)
        check(n, x.float().clamp(-65504, 65504), ref, tol[n])


def test_no_queries_or_keys(hip):
    q, k = torch.randn(2, 5, 4, 64, device=DEV).half(), torch.randn(2, 0, 2, 64, device=DEV).half()
    for causal in (False, True):
        o, lse = hip.masked_attention(q, k, k, causal=causal)
        assert float(o.abs().max()) == 0 and bool(torch.isinf(lse).all())
        dq, dk, dv, _ = hip.masked_attention_grad(q, k, k, o, lse, q, causal=causal)
        assert float(dq.abs().max()) == 0 and dk.shape == k.shape
    o, lse = hip.masked_attention(q[:, :0], q, q)
    assert o.shape == (2, 0, 4, 64)
    rel = torch.randn(4, 9, device=DEV)
    o, lse = hip.masked_attention(q[:, :0], q, q, rel=rel)
    dq, dk, dv, drel = hip.masked_attention_grad(q[:, :0], q, q, o, lse, q[:, :0], rel=rel)
    assert float(dk.abs().max()) == 0 and float(dv.abs().max()) == 0 and float(drel.abs().max()) == 0
    o, lse = hip.masked_attention(q[:0], q[:0], q[:0], rel=rel)
    out = hip.masked_attention_grad(q[:0], q[:0], q[:0], o, lse, q[:0], rel=rel)
    assert o.shape[0] == 0 and float(out[3].abs().max()) == 0


def test_cache_past_32_bit_offsets(hip):
    """a cache whose rows lie 2^22 elements apart: offsets of several GiB inside one head"""
    N, step = 1100, 1 << 22
    big = torch.empty(N * step + 128, dtype=F16, device=DEV)
    k, v = (big.as_strided((1, N, 1, 64), (N * step, step, 64, 1), off) for off in (0, 64))
    g = gen(8)
    kc, vc, q = randn(g, 1, N, 1, 64).half(), randn(g, 1, N, 1, 64).half(), randn(g, 1, 200, 1, 64).half()
    k.copy_(kc.to(DEV)), v.copy_(vc.to(DEV))
    for nq in (1, 200):
        a = hip.masked_attention(q[:, :nq].to(DEV), k, v, causal=True)
        b = hip.masked_attention(q[:, :nq].to(DEV), kc.to(DEV), vc.to(DEV), causal=True)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


# ---- relative bias ---------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("nb,maxd,both,H", [(32, 128, True, 16), (32, 128, False, 3), (16, 20, True, 1), (4, 1024, True, 7), (2, 2, False, 2)])
def test_rel_bias(hip, nb, maxd, both, H):
    plan = hip.rel_buckets(nb, maxd, bidirectional=both)
    index = [tr.rel_bucket(i, nb, maxd, both) for i in range(-maxd, maxd + 1)]
    assert plan.index.tolist() == index
    g = gen(1)
    table = randn(g, nb, H)
    rel = hip.rel_bias(table.to(DEV), plan)
    assert torch.equal(rel.cpu(), table[torch.tensor(index)].t())
    drel = randn(g, H, 2 * maxd + 1)
    ref = torch.zeros(nb, H, dtype=torch.float64).index_add_(0, torch.tensor(index), drel.double().t())
    got = hip.rel_bias_grad(drel.to(DEV), plan)
    check("dtable", got, ref, 2.0 ** -24 * ref.abs() + 1e-12 * drel.abs().sum().double())
    assert torch.equal(got, hip.rel_bias_grad(drel.to(DEV), plan))


# ---- the operators together ---------------------------------------------------------------------------------------------------------------------------
def block(hip, x, wq, wk, wv, gq, gk, pos, freqs, table, plan, do, kw):
    """q / k / v projections (fp32 torch here), norm + rotation, attention with the bucket bias, and the way back to x's projections"""
    H, Hk, d = wq.shape[0], wk.shape[0], wq.shape[1]
    B, N, _ = x.shape
    q, k, v = (torch.matmul(x.float(), w.reshape(-1, w.shape[2]).t()).to(x.dtype).view(B, N, -1, d) for w in (wq, wk, wv))
    rel = hip.rel_bias(table, plan)
    args = dict(q_gamma=gq, k_gamma=gk)
    qn, kn = hip.qk_norm_rope(q.flatten(0, 1), k.flatten(0, 1), pos, freqs, **args)
    qn, kn = qn.view(B, N, H, d), kn.view(B, N, Hk, d)
    o, lse = hip.masked_attention(qn, kn, v, rel=rel, **kw)
    dqn, dkn, dv, drel = hip.masked_attention_grad(qn, kn, v, o, lse, do, rel=rel, **kw)
    dq, dk, dgq, dgk = hip.qk_norm_rope_grad(q.flatten(0, 1), k.flatten(0, 1), pos, freqs, dqn.flatten(0, 1), dkn.flatten(0, 1), **args)
    return q, k, v, o, dq.view_as(q), dk.view_as(k), dv, dgq, dgk, hip.rel_bias_grad(drel, plan)


def test_operators_together(hip):
    g = gen(21)
    B, N, C, H, Hk, d = 2, 150, 96, 4, 2, 64
    x = randn(g, B, N, C).half()
    wq, wk, wv = (randn(g, n, d, C, scale=C ** -0.5) for n in (H, Hk, Hk))
    gq, gk = 1 + 0.2 * randn(g, d), 1 + 0.2 * randn(g, d)
    table, do = randn(g, 32, H), randn(g, B, N, H, d).half()
    pos = torch.arange(N).repeat(B)
    freqs = 10000.0 ** (-torch.arange(32, dtype=torch.float64) / 32)
    docs = docs_of(g, B, N, 7)
    plan = hip.rel_buckets(32, 40, bidirectional=False)
    kw = dict(causal=True, softcap=20.0, docs=docs.to(DEV))
    out = block(hip, x.to(DEV), wq.to(DEV), wk.to(DEV), wv.to(DEV), gq.to(DEV), gk.to(DEV), pos.to(DEV), freqs.to(DEV), table.to(DEV), plan, do.to(DEV), kw)
    q, k, v = (t.cpu().double().requires_grad_() for t in out[:3])
    g64 = [gq.double().requires_grad_(), gk.double().requires_grad_()]
    t64 = table.double().requires_grad_()
    qn = tr.qk_norm_rope(q.flatten(0, 1), pos, freqs, g64[0], 1e-6, False).view(B, N, H, d)
    kn = tr.qk_norm_rope(k.flatten(0, 1), pos, freqs, g64[1], 1e-6, False).view(B, N, Hk, d)
    index = torch.tensor([tr.rel_bucket(i, 32, 40, False) for i in range(-40, 41)])
    vis, dist = tr.visible(B, N, N, True, (docs, docs))
    r = tr.attention(qn, kn, v, vis, dist, d ** -0.5, 20.0, None, t64[index].t())
    ref = [r["o"]] + list(torch.autograd.grad(r["o"], [q, k, v] + g64 + [t64], do.double()))
    # each tensor passes at most three fp16 roundings (norm, probabilities / dS, result) besides those of its neighbours: relative L2, 8 half steps
    for n, a, b in zip(("o", "dq", "dk", "dv", "dgq", "dgk", "dtable"), out[3:], ref):
        err = float((a.cpu().double() - b.detach()).norm() / b.detach().norm())
        assert err < 8 * half_step(F16), (n, err)


def test_difference_quotient(hip):
    """the gradient against the kernel's own forward: a step of h along a direction changes sum(o do) by h <grad, direction>"""
    g = gen(31)
    B, N, H, d = 1, 60, 2, 64
    q, k, v = (randn(g, B, N, H, d).half() for _ in range(3))
    do = randn(g, B, N, H, d).half()
    kw = dict(causal=True, softcap=10.0, scale=0.125)
    c = [x.to(DEV) for x in (q, k, v)]
    o, lse = hip.masked_attention(*c, **kw)
    grads = hip.masked_attention_grad(*c, o, lse, do.to(DEV), **kw)
    for n, (x, gx) in enumerate(zip(c, grads)):
        # along the gradient's own sign pattern, in steps fp16 holds exactly: x +- 2^-5 sign
        s = torch.sign(gx.float())
        h = 2.0 ** -5
        lo, hi = (x.float() - h * s).half(), (x.float() + h * s).half()
        val = []
        for y in (lo, hi):
            a = list(c)
            a[n] = y
            val.append((hip.masked_attention(*a, **kw)[0].double() * do.to(DEV).double()).sum())
        step = (hi.double() - lo.double())
        quot, want = float(val[1] - val[0]), float((gx.double() * step).sum())
        # o's roundings: 2 x sum |o do| u, random signs: at most 6 sigma of u |o do| over all elements; curvature: third order, h^2 / 6 of the change
        sigma = float(((o.double() * do.to(DEV).double()) ** 2).sum().sqrt()) * half_step(F16) * 2
        assert abs(quot - want) < 6 * sigma + 0.02 * abs(want), (n, quot, want, sigma)


# ---- streams, graphs --------------------------------------------------------------------------------------------------------------------------------------
def test_other_stream_and_two_calls_at_once(hip):
    q, k, v, do, kw = problem("token_long128", F16, seed=3)
    c = [x.to(DEV) for x in (q, k, v)]
    kg = on_gpu(kw)
    ref = hip.masked_attention(*c, **kg)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    outs = []
    for _ in range(4):
        for s in (s1, s2):
            with torch.cuda.stream(s):
                outs.append(hip.masked_attention(*c, **kg))
    torch.cuda.synchronize()
    assert all(torch.equal(a, ref[0]) and torch.equal(b, ref[1]) for a, b in outs)


@pytest.mark.parametrize("name", ["token_long128", "docs_causal_cap", "rel"])
def test_captured_graph(hip, name):
    """forward and gradient captured once, replayed on new inputs with eager work in between: the bits of eager calls"""
    q, k, v, do, kw = problem(name, F16, seed=1)
    c = [x.to(DEV) for x in (q, k, v)]
    dd = do.to(DEV)
    kg = on_gpu(kw)
    o, lse = hip.masked_attention(*c, **kg)
    first = hip.masked_attention_grad(*c, o, lse, dd, **kg)
    wk, wg = (torch.empty(64 << 20, dtype=torch.uint8, device=DEV) for _ in range(2))
    bufs = [torch.empty_like(x) if x is not None else None for x in (o, lse) + first]
    gk = dict(kg, work=wk)
    gg = dict(kg, work=wg, dq=bufs[2], dk=bufs[3], dv=bufs[4], **({"drel": bufs[5]} if bufs[5] is not None else {}))
    s = torch.cuda.Stream()
    gr = hip.Graph()
    with torch.cuda.stream(s):
        gr.begin()
        hip.masked_attention(*c, o=bufs[0], lse=bufs[1], **gk)
        hip.masked_attention_grad(*c, bufs[0], bufs[1], dd, **gg)
        gr.end()
        for rep in range(4):
            for x in (*c, dd):
                x.copy_(torch.randn(x.shape, generator=gen(100 + rep)).to(x.dtype))
            gr.launch()
            s.synchronize()
            a, b = hip.masked_attention(*c, **kg)
            e = (a, b) + hip.masked_attention_grad(*c, a, b, dd, **kg)
            assert all(x is None or torch.equal(x, y) for x, y in zip(e, bufs)), rep
            s.synchronize()


def test_capture_needs_the_callers_buffers(hip):
    q = torch.randn(1, 1, 4, 64, device=DEV).half()
    k = torch.randn(1, 4000, 4, 64, device=DEV).half()
    o, lse = hip.masked_attention(q, k, k)
    count = torch.zeros(1, dtype=torch.int32, device=DEV)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        gr = hip.Graph()
        gr.begin()
        try:
            with pytest.raises(ValueError, match="o="):
                hip.masked_attention(q, k, k)
            with pytest.raises(ValueError, match="work="):
                hip.masked_attention(q, k, k, o=o, lse=lse)
        finally:
            hip.step_advance(count, 1)                 # a graph of one node
            gr.end()
        gr.launch()
        s.synchronize()
    assert int(count) == 1


# ---- the text tower -------------------------------------------------------------------------------------------------------------------------------------------
def test_text_tower_on_the_masked_attention(hip, monkeypatch):
    from mgld_vsr_amd import synth
    from mgld_vsr_amd.text import FrozenOpenCLIPEmbedder
    e = FrozenOpenCLIPEmbedder(context_dim=128, heads=2, layers=3, vocab_size=100, build_tower=True)
    synth.fill_module_(e.model, "text")
    toks = torch.randint(0, 100, (3, 77), generator=gen(2))
    ref = e.encode_with_transformer(toks).clone()
    monkeypatch.setenv("MGLD_TEXT_ATTN", "1")
    got = e.encode_with_transformer(toks)
    err = float((got - ref).double().norm() / ref.double().norm())
    assert err < 2e-3, err           # two evaluations that round their probabilities and activations to fp16 in different places: 3 layers x 2^-11 each way
