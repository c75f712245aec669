"""Timed cases of the transformer operators: head-wise norms of queries and keys with the position rotation, attention with capped
scores, distance biases and document / prefix masks, and the learned relative bias by buckets, each with its gradient.

`own` chooses between the plain form (elementary torch operations in fp32, one rounding at the end) and the framework's kernels.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ---- cases ------------------------------------------------------------------------------------------------------------------------
def _rotate(name, tokens, heads, kv_heads, d, dtype, rot=None, start=0, interleaved=False, train=False):
    return {"name": name, "op": "rotate", "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "d": d, "dtype": dtype,
            "rot": d if rot is None else rot, "start": start, "interleaved": interleaved, "train": train}


def _attend(name, batch, nq, nk, heads, kv_heads, d, dtype, causal=True, softcap=0.0, slopes=False, docs="", prefix="", lens="",
            buckets=0, train=False):
    """docs: lengths of the documents of every packed row (what they leave of a row is padding); prefix / lens: one number per row"""
    return {"name": name, "op": "attend", "batch": batch, "nq": nq, "nk": nk, "heads": heads, "kv_heads": kv_heads, "d": d,
            "dtype": dtype, "causal": causal, "softcap": softcap, "slopes": slopes, "docs": docs, "prefix": prefix, "lens": lens,
            "buckets": buckets, "train": train}


def _ragged(total, weights, rows=1):
    """lengths in the proportion of `weights` that fill `total` but for a few tokens of padding, another order in every row"""
    s = sum(weights)
    cut = [max(1, total * w // s - (i % 3)) for i, w in enumerate(weights)]
    return ";".join(",".join(str(cut[(i + r) % len(cut)]) for i in range(len(cut))) for r in range(rows))


def listed():
    return [
        # one new token of a served sequence: latency
        _rotate("rotate_one_token", 1, 32, 8, 128, "bf16", start=1000),
        # a long prompt at far positions, keys and values shared by four query heads
        _rotate("rotate_prompt", 16384, 32, 8, 128, "bf16", start=120000),
        # a training step: half of every head rotated in interleaved pairs, an odd number of tokens
        _rotate("rotate_train", 8195, 16, 16, 64, "fp16", rot=32, interleaved=True, train=True),
        # the text tower's attention on a batch of prompts (77 tokens, 16 heads of 64)
        _attend("text_prompts", 16, 77, 77, 16, 16, 64, "fp16"),
        # a long prompt with capped scores
        _attend("capped_prompt", 1, 8192, 8192, 32, 8, 128, "bf16", softcap=50.0),
        # documents packed into rows, with a linear distance bias and padding at the end of every row
        _attend("packed_documents", 2, 6001, 6001, 16, 16, 64, "fp16", slopes=True,
                docs=_ragged(5980, [7, 1, 19, 3, 11, 40, 5, 2], 2)),
        # a training step with a prefix that every token sees
        _attend("prefix_train", 2, 2048, 2048, 16, 4, 128, "bf16", prefix="300,77", train=True),
        # a training step on packed documents with capped scores
        _attend("capped_documents_train", 1, 4096, 4096, 16, 8, 128, "bf16", softcap=30.0,
                docs=_ragged(4090, [9, 2, 30, 1, 14], 1), train=True),
        # one new token for each of 16 served sequences over their caches of ragged lengths
        _attend("token_long_cache", 16, 1, 32768, 32, 8, 128, "bf16", softcap=50.0,
                lens=",".join(str(32768 - 1531 * i) for i in range(16))),
        # one new token of one short sequence: latency
        _attend("token_short_cache", 1, 1, 500, 16, 16, 64, "fp16", slopes=True, lens="413"),
        # an encoder whose attention has the learned bias by buckets and no mask
        _attend("bucket_encoder", 8, 512, 512, 16, 16, 64, "fp16", causal=False, buckets=32),
        # its training step, on more and longer rows of ragged lengths
        _attend("bucket_train", 4, 1024, 1024, 16, 16, 64, "bf16", causal=False, buckets=32, lens="1024,1000,517,129", train=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rotate", "rotate_train", "prompt", "documents", "prefix_train", "documents_train", "token", "bucket", "bucket_train"])
    dtype = rng.choice(["bf16", "fp16"])
    d = rng.choice([64, 128])
    kv = rng.choice([2, 4, 8])
    heads = kv * rng.choice([1, 2, 4])
    cap = rng.choice([0.0, 30.0, 50.0])
    if kind.startswith("rotate"):
        train = kind == "rotate_train"
        return _rotate("", _log(rng, 1, 6000 if train else 16000), heads, kv, d, dtype, rot=rng.choice([d, d // 2]), start=_log(rng, 1, 200000),
                       interleaved=rng.random() < 0.5, train=train)
    if kind == "prompt":
        n = _log(rng, 17, 6000)
        b = max(1, min(16, 3000 // n))
        return _attend("", b, n, n, heads, kv, d, dtype, softcap=cap, slopes=rng.random() < 0.5)
    if kind.startswith("documents"):
        train = kind == "documents_train"
        n = _log(rng, 300, 2100 if train else 4000)
        b = rng.choice([1, 2])
        w = [rng.randint(1, 30) for _ in range(rng.randint(2, 9))]
        return _attend("", b, n, n, heads, kv, d, dtype, causal=rng.random() < 0.7, softcap=cap, slopes=rng.random() < 0.5,
                       docs=_ragged(n - rng.randint(0, 20), w, b), train=train)
    if kind == "prefix_train":
        n = _log(rng, 64, 2100)
        return _attend("", 2, n, n, heads, kv, d, dtype, softcap=cap, prefix=f"{rng.randint(0, n)},{rng.randint(0, n)}", train=True)
    if kind == "token":
        n = _log(rng, 60, 21000)
        b = rng.choice([1, 2, 5, 16])
        return _attend("", b, rng.choice([1, 1, 2, 4]), n, heads, kv, d, dtype, softcap=cap, slopes=rng.random() < 0.5,
                       lens=",".join(str(rng.randint(max(4, n // 2), n)) for _ in range(b)))
    train = kind == "bucket_train"
    n = _log(rng, 33, 1100 if train else 2200)
    b = max(1, min(8, 4000 // n))
    lens = ",".join(str(rng.randint(max(1, n // 3), n)) for _ in range(b))
    return _attend("", b, n, n, heads, kv, d, dtype, causal=rng.random() < 0.3, buckets=rng.choice([16, 32]), lens=lens, train=train)


# ---- inputs -----------------------------------------------------------------------------------------------------------------------
MAX_DISTANCE = 128
EPS = 1e-6


def _ints(text):
    return [int(x) for x in text.split(",")] if text else []


def _document_ids(case):
    """int32 [batch, nk]: the number of its document for each token, -1 for padding"""
    rows = []
    for text in case["docs"].split(";"):
        ids = []
        for i, n in enumerate(_ints(text)):
            ids += [i] * n
        rows.append((ids + [-1] * case["nk"])[:case["nk"]])
    return torch.tensor(rows, dtype=torch.int32)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def randn(*shape, scale=1.0, dtype=dt):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)

    st = dict(case)
    hq, hk, d = case["heads"], case["kv_heads"], case["d"]
    if case["op"] == "rotate":
        n = case["tokens"]
        # a token's key and value lie side by side, as one projection writes them
        st["q"] = randn(n, hq, d)
        st["k"] = randn(n, 2 * hk * d)[:, :hk * d].unflatten(1, (hk, d))
        st["pos"] = torch.arange(n, device="cuda", dtype=torch.int64) + case["start"]
        st["q_gamma"] = 1.0 + 0.2 * torch.randn(d, generator=g, device="cuda")
        st["k_gamma"] = 1.0 + 0.2 * torch.randn(d, generator=g, device="cuda")
        j = torch.arange(case["rot"] // 2, device="cuda", dtype=torch.float64)
        st["freqs"] = 10000.0 ** (-2.0 * j / case["rot"])
        if case["train"]:
            st["dq_out"], st["dk_out"] = randn(n, hq, d), randn(n, hk, d)
        return st
    b, nq, nk = case["batch"], case["nq"], case["nk"]
    loud = 3.0 if case["softcap"] else 1.0          # scores that reach the cap's curved part
    if nq == nk:
        kv = randn(b, nk, 2 * hk * d)
        st["k"], st["v"] = kv[..., :hk * d].unflatten(2, (hk, d)), kv[..., hk * d:].unflatten(2, (hk, d))
    else:                                           # a cache [batch, position, head, d] and the newest tokens' queries
        st["k"], st["v"] = randn(b, nk, hk, d), randn(b, nk, hk, d)
    st["q"] = randn(b, nq, hq, d, scale=loud)
    st["docs_t"] = _document_ids(case).cuda() if case["docs"] else None
    st["prefix_t"] = torch.tensor(_ints(case["prefix"]), dtype=torch.int32, device="cuda") if case["prefix"] else None
    st["lens_t"] = torch.tensor(_ints(case["lens"]), dtype=torch.int32, device="cuda") if case["lens"] else None
    # of a padded batch the queries stand at 0, 1, ..; a cache's newest tokens at its end
    st["q_pos0"] = 0 if nq == nk else None
    st["slopes_t"] = 2.0 ** (-8.0 * torch.arange(1, hq + 1, device="cuda", dtype=torch.float32) / hq) if case["slopes"] else None
    st["table"] = torch.randn(case["buckets"], hq, generator=g, device="cuda") if case["buckets"] else None
    if case["train"]:
        st["do"] = randn(b, nq, hq, d)
    if own and case["buckets"]:
        from mgld_vsr_amd import hip
        st["plan"] = hip.rel_buckets(case["buckets"], MAX_DISTANCE, bidirectional=not case["causal"])
    return st


# ---- the passes -------------------------------------------------------------------------------------------------------------------
def run(st):
    if st["op"] == "rotate":
        return _own_rotate(st) if own else _plain_rotate(st)
    return _own_attend(st) if own else _plain_attend(st)


def _own_rotate(st):
    from mgld_vsr_amd import hip
    kw = dict(q_gamma=st["q_gamma"], k_gamma=st["k_gamma"], eps=EPS, interleaved=st["interleaved"])
    out = list(hip.qk_norm_rope(st["q"], st["k"], st["pos"], st["freqs"], **kw))
    if st["train"]:
        out += hip.qk_norm_rope_grad(st["q"], st["k"], st["pos"], st["freqs"], st["dq_out"], st["dk_out"], **kw)
    return out


def _own_attend(st):
    from mgld_vsr_amd import hip
    rel = hip.rel_bias(st["table"], st["plan"]) if st["table"] is not None else None
    kw = dict(causal=st["causal"], softcap=st["softcap"], slopes=st["slopes_t"], rel=rel, docs=st["docs_t"], prefix=st["prefix_t"],
              kv_len=st["lens_t"], q_pos0=st["q_pos0"])
    o, lse = hip.masked_attention(st["q"], st["k"], st["v"], **kw)
    if not st["train"]:
        return o
    dq, dk, dv, drel = hip.masked_attention_grad(st["q"], st["k"], st["v"], o, lse, st["do"], **kw)
    out = [o, dq, dk, dv]
    if rel is not None:
        out.append(hip.rel_bias_grad(drel, st["plan"]))
    return out


def _plain_rotate(st):
    ang = st["pos"].double()[:, None] * st["freqs"][None]               # fp64: far positions
    c, s = ang.cos().float()[:, None], ang.sin().float()[:, None]
    rot = st["rot"]

    def split(y):
        t = y[..., :rot]
        if st["interleaved"]:
            return t[..., 0::2], t[..., 1::2], y[..., rot:]
        return t[..., :rot // 2], t[..., rot // 2:], y[..., rot:]

    def join(a, b, rest):
        t = torch.stack([a, b], -1).flatten(-2) if st["interleaved"] else torch.cat([a, b], -1)
        return torch.cat([t, rest], -1)

    def forward(x, gamma):
        x = x.float()
        a, b, rest = split(x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * gamma)
        return join(a * c - b * s, a * s + b * c, rest)

    def gradient(x, gamma, dy):
        x = x.float()
        r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
        a, b, rest = split(dy.float())
        z = join(a * c + b * s, b * c - a * s, rest)
        xh = x * r
        dgamma = (z * xh).double().sum((0, 1)).float()
        w = z * gamma
        return r * (w - xh * (w * xh).mean(-1, keepdim=True)), dgamma

    dt = st["q"].dtype
    out = [forward(st["q"], st["q_gamma"]).to(dt), forward(st["k"], st["k_gamma"]).to(dt)]
    if st["train"]:
        dq, dgq = gradient(st["q"], st["q_gamma"], st["dq_out"])
        dk, dgk = gradient(st["k"], st["k_gamma"], st["dk_out"])
        out += [dq.to(dt), dk.to(dt), dgq, dgk]
    return out


def _bucket_borders(buckets, bidirectional):
    """distances at which the next bucket begins, by whole numbers: n is in bucket >= exact + j where
    log(n / exact) / log(MAX_DISTANCE / exact) * (nb - exact) >= j"""
    nb = buckets // 2 if bidirectional else buckets
    exact = nb // 2
    m = nb - exact
    borders = list(range(1, exact + 1))
    for j in range(1, m):
        n = exact
        while n ** m * exact ** j < MAX_DISTANCE ** j * exact ** m:
            n += 1
        borders.append(n)
    return nb, borders


def _plain_bias(st, delta):
    """(bucket of every pair [nq, nk], bias [heads, nq, nk])"""
    both = not st["causal"]
    nb, borders = _bucket_borders(st["buckets"], both)
    n = delta.abs() if both else (-delta).clamp(min=0)
    bucket = torch.zeros_like(n)
    for x in borders:
        bucket += n >= x
    if both:
        bucket += nb * (delta > 0)
    return bucket, st["table"].float()[bucket].movedim(-1, -3)


def _plain_attend(st):
    q, k, v = st["q"], st["k"], st["v"]
    b, nq, hq, d = q.shape
    nk, hk = k.shape[1], k.shape[2]
    grp = hq // hk
    dev, dt = q.device, q.dtype
    # [b, shared head, query head of it x query, d]
    qf = q.float().unflatten(2, (hk, grp)).permute(0, 2, 3, 1, 4).reshape(b, hk, grp * nq, d)
    kf, vf = k.float().transpose(1, 2).contiguous(), v.float().transpose(1, 2).contiguous()
    scale, cap = d ** -0.5, st["softcap"]
    u = torch.matmul(qf, kf.transpose(2, 3).contiguous()) * scale
    if cap:
        u = torch.tanh(u / cap) * cap
    u = u.view(b, hq, nq, nk)
    lens = st["lens_t"].long() if st["lens_t"] is not None else torch.full((b,), nk, device=dev)
    j = torch.arange(nk, device=dev)
    pos0 = torch.zeros_like(lens) if st["q_pos0"] == 0 else lens - nq
    qpos = pos0[:, None] + torch.arange(nq, device=dev)                   # [b, nq]
    delta = j[None, None, :] - qpos[:, :, None]                           # [b, nq, nk]
    s, bucket = u, None
    if st["slopes_t"] is not None:
        s = s - st["slopes_t"][None, :, None, None] * delta.abs()[:, None]
    if st["table"] is not None:
        bucket, bias = _plain_bias(st, delta[0])                          # every row of these cases has the same positions
        s = s + bias
    seen = (j[None, :] < lens[:, None])[:, None, :].expand(b, nq, nk)
    if st["causal"]:
        past = delta <= 0
        if st["prefix_t"] is not None:
            past = past | (j[None, None, :] < st["prefix_t"].long()[:, None, None])
        seen = seen & past
    if st["docs_t"] is not None:
        ids = st["docs_t"]
        seen = seen & (ids[:, :, None] == ids[:, None, :]) & (ids[:, None, :] >= 0)
    s = s.masked_fill(~seen[:, None], float("-inf"))
    top = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = e.sum(-1, keepdim=True)
    p = torch.where(total > 0, e / total, torch.zeros_like(e))
    del s, e

    def heads_last(x):
        return x.view(b, hk, grp, nq, d).permute(0, 3, 1, 2, 4).reshape(b, nq, hq, d)

    pg = p.view(b, hk, grp * nq, nk)
    o = heads_last(torch.matmul(pg, vf)).to(dt)
    if not st["train"]:
        return o
    dof = st["do"].float().unflatten(2, (hk, grp)).permute(0, 2, 3, 1, 4).reshape(b, hk, grp * nq, d)
    dv = torch.matmul(pg.transpose(2, 3).contiguous(), dof).transpose(1, 2)
    dp = torch.matmul(dof, vf.transpose(2, 3).contiguous()).view(b, hq, nq, nk)
    ds = p * (dp - (p * dp).sum(-1, keepdim=True))
    del dp
    dtab = None
    if bucket is not None:
        # pairs of one distance lie on one diagonal: the sheared matrix has them in one column
        by = ds.double().sum(0).flip(1)                                   # [hq, nq, nk], last query first
        by = torch.cat([by, torch.zeros(hq, nq, nq, device=dev, dtype=by.dtype)], 2).flatten(1)[:, :nq * (nk + nq) - nq]
        diag = by.view(hq, nq, nk + nq - 1).sum(1)                        # column c: distance c - (nq - 1)
        first = torch.cat([bucket[:, 0].flip(0), bucket[0, 1:]])          # the bucket of every distance
        dtab = torch.zeros(st["buckets"], hq, device=dev, dtype=torch.float64)
        for i in range(st["buckets"]):
            dtab[i] = diag[:, first == i].sum(1)
        dtab = dtab.float()
    if cap:
        ds = ds * (1.0 - (u / cap) ** 2)
    dsg = ds.view(b, hk, grp * nq, nk) * scale
    dq = heads_last(torch.matmul(dsg, kf))
    dk = torch.matmul(dsg.transpose(2, 3).contiguous(), qf).transpose(1, 2)
    out = [o, dq.to(dt), dk.to(dt), dv.to(dt)]
    if dtab is not None:
        out.append(dtab)
    return out


# ---- what a pass cannot do without -----------------------------------------------------------------------------------------------------
def _pairs(case):
    """visible (query, key) pairs of one query head, over the batch; keys that are seen at all"""
    b, nq, nk = case["batch"], case["nq"], case["nk"]
    pairs = keys = 0
    lens = _ints(case["lens"]) or [nk] * b
    prefix = _ints(case["prefix"]) or [0] * b
    docs = [_ints(t) for t in case["docs"].split(";")] if case["docs"] else None
    for r in range(b):
        if docs is not None:
            for n in docs[r]:
                pairs += n * (n + 1) // 2 if case["causal"] else n * n
                keys += n
            continue
        n = lens[r]
        keys += n
        if not case["causal"]:
            pairs += nq * n
            continue
        first = 0 if nq == nk else n - nq
        for i in range(nq):
            pairs += min(n, max(first + i + 1, prefix[r]))
    return pairs, keys


def work(case):
    hq, hk, d = case["heads"], case["kv_heads"], case["d"]
    if case["op"] == "rotate":
        el = case["tokens"] * (hq + hk) * d
        bytes_ = 2 * el * (5 if case["train"] else 2) + 8 * case["tokens"]
        return {"bytes": bytes_, "flops": el * (20 if case["train"] else 7)}
    pairs, keys = _pairs(case)
    b, nq = case["batch"], case["nq"]
    q_bytes, kv_bytes = 2 * b * nq * hq * d, 2 * 2 * keys * hk * d
    if not case["train"]:
        return {"bytes": 2 * q_bytes + kv_bytes, "flops": 4 * pairs * hq * d}
    return {"bytes": 4 * q_bytes + 2 * kv_bytes, "flops": 14 * pairs * hq * d}


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------------------------
def exact(case, seed):
    global own
    keep, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = keep
    return _exact_rotate(st) if case["op"] == "rotate" else _exact_attend(st)


def _exact_rotate(st):
    turn = torch.exp(1j * (st["pos"].double()[:, None] * st["freqs"][None]))          # the rotation as a complex factor
    half = st["rot"] // 2
    idx = torch.arange(half, device="cuda")
    re, im = (2 * idx, 2 * idx + 1) if st["interleaved"] else (idx, idx + half)

    def turned(y, factor):
        out = y.clone()
        z = torch.complex(y[:, re], y[:, im]) * factor
        out[:, re], out[:, im] = z.real, z.imag
        return out

    res, grads, gammas = [], [], []
    for x, gamma, dy in ((st["q"], st["q_gamma"], st.get("dq_out")), (st["k"], st["k_gamma"], st.get("dk_out"))):
        gm = gamma.double()
        y, dx, dg = [], [], torch.zeros_like(gm)
        for h in range(x.shape[1]):
            xh = x[:, h].double()
            rms = (xh.square().sum(1, keepdim=True) / xh.shape[1] + EPS).sqrt()
            y.append(turned(xh / rms * gm, turn))
            if dy is not None:
                z = turned(dy[:, h].double(), turn.conj())
                dg += (z * xh / rms).sum(0)
                w = z * gm
                dx.append(w / rms - xh * (w * xh).sum(1, keepdim=True) / (xh.shape[1] * rms ** 3))
        res.append(torch.stack(y, 1))
        if dy is not None:
            grads.append(torch.stack(dx, 1))
            gammas.append(dg)
    return res + grads + gammas


def _exact_attend(st):
    q, k, v = st["q"], st["k"], st["v"]
    b, nq, hq, d = q.shape
    nk, hk = k.shape[1], k.shape[2]
    cap, scale = st["softcap"], 1.0 / math.sqrt(d)
    o = torch.zeros(b, nq, hq, d, dtype=torch.float64, device="cuda")
    dq = torch.zeros_like(o)
    dk = torch.zeros(b, nk, hk, d, dtype=torch.float64, device="cuda")
    dv = torch.zeros_like(dk)
    dtab = torch.zeros(max(1, st["buckets"]), hq, dtype=torch.float64, device="cuda")
    kpos = torch.arange(nk, device="cuda")
    for r in range(b):
        n = int(st["lens_t"][r]) if st["lens_t"] is not None else nk
        qpos = torch.arange(nq, device="cuda") + (0 if st["q_pos0"] == 0 else n - nq)
        diff = kpos[None, :] - qpos[:, None]
        hidden = (kpos >= n)[None, :].expand(nq, nk)
        if st["causal"]:
            ahead = diff > 0
            if st["prefix_t"] is not None:
                ahead = ahead & (kpos >= int(st["prefix_t"][r]))[None, :]
            hidden = hidden | ahead
        if st["docs_t"] is not None:
            ids = st["docs_t"][r]
            hidden = hidden | (ids[:, None] != ids[None, :]) | (ids[None, :] < 0)
        group = None
        if st["buckets"]:
            both = not st["causal"]
            nb = st["buckets"] // 2 if both else st["buckets"]
            ex = nb // 2
            far = diff.abs().double() if both else (-diff).clamp(min=0).double()
            # 1e-9: a distance on a border belongs to the bucket that begins there
            grow = torch.log(far.clamp(min=1) / ex) / math.log(MAX_DISTANCE / ex) * (nb - ex) + 1e-9
            group = torch.where(far < ex, far, (ex + grow.floor()).clamp(max=nb - 1)).long()
            if both:
                group = group + nb * (diff > 0)
        for h in range(hq):
            g = h // (hq // hk)
            qd, kd, vd = q[r, :, h].double(), k[r, :, g].double(), v[r, :, g].double()
            t = qd @ kd.t() * scale
            th = torch.tanh(t / cap) if cap else None
            s = cap * th if cap else t
            if st["slopes_t"] is not None:
                s = s - st["slopes_t"][h].double() * diff.abs()
            if group is not None:
                s = s + st["table"][:, h].double()[group]
            s[hidden] = float("-inf")
            lse = torch.logsumexp(s, 1, keepdim=True)
            p = torch.where(torch.isinf(lse), torch.zeros_like(s), torch.exp(s - lse))
            o[r, :, h] = p @ vd
            if not st["train"]:
                continue
            dod = st["do"][r, :, h].double()
            dv[r, :, g] += p.t() @ dod
            ds = p * (dod @ vd.t() - (dod * o[r, :, h]).sum(1, keepdim=True))
            if group is not None:
                dtab[:, h] += torch.zeros_like(dtab[:, h]).index_add_(0, group.flatten(), ds.flatten())
            if cap:
                ds = ds * (1 - th * th)
            dq[r, :, h] = ds @ kd * scale
            dk[r, :, g] += ds.t() @ qd * scale
    if not st["train"]:
        return o
    return [o, dq, dk, dv] + ([dtab] if st["buckets"] else [])
