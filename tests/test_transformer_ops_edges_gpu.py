"""mgld_vsr_amd.hip's transformer operators at the edges of their ranges: padding numbers, magnitudes, caps, masked places.  Oracle, problems and
error bounds are those of test_transformer_ops_gpu.py; a bound that a case adds is derived where it stands."""
import math

import pytest
import torch

from oracle import transformer as tr
from test_transformer_ops_gpu import ATT, BF16, DEV, F16, check, check_lse, gen, half_step, on_gpu, problem, randn, reference

pytestmark = pytest.mark.gpu


def run(hip, q, k, v, do, kw):
    c, kg = [x.to(DEV) for x in (q, k, v)], on_gpu(kw)
    o, lse = hip.masked_attention(*c, **kg)
    return o, lse, hip.masked_attention_grad(*c, o, lse, do.to(DEV), **kg)

# ---- padding ----------------------------------------------------------------------------------------------------------------------------------
PADS = {"-2": lambda ids: torch.full_like(ids, -2), "mixed": lambda ids: -1 - torch.arange(ids.numel(), dtype=torch.int32).view_as(ids) % 4,
        "lowest": lambda ids: torch.full_like(ids, -1 << 31)}


def padded(docs, pad):
    return tuple(torch.where(ids < 0, PADS[pad](ids), ids) for ids in docs)


@pytest.mark.parametrize("pad", list(PADS))
@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("name", [n for n in ATT if "docs" in ATT[n][6]])
def test_any_negative_document_is_padding(hip, name, dt, pad):
    q, k, v, do, kw = problem(name, dt, seed=11)
    kw["docs"] = padded(kw["docs"], pad)
    res, tol = reference(q, k, v, do, kw)
    o, lse, grads = run(hip, q, k, v, do, kw)
    check("o", o, res["o"], tol["o"])
    check_lse(lse, res["lse"], tol["lse"])
    for n, x in zip(("dq", "dk", "dv", "drel"), grads):
        if n in res:
            check(n, x, res[n], tol[n])


@pytest.mark.parametrize("pad", list(PADS))
@pytest.mark.parametrize("Nq,N", [(100, 100), (2, 100)])
def test_padding_rows_of_any_number_hold_anything(hip, Nq, N, pad):
    """a mixed tile of two real documents and padding, whose rows and keys hold NaN"""
    g = gen(41)
    q, do = (randn(g, 2, Nq, 4, 64).half() for _ in range(2))
    k, v = (randn(g, 2, N, 2, 64).half() for _ in range(2))
    dk = torch.full((2, N), 3, dtype=torch.int32)
    dk[:, 40:70] = 5
    dk[0, 20:40], dk[1, 80:] = -1, -1
    dq = dk[:, [3, 30]].clone() if Nq == 2 else dk.clone()
    if Nq == 2:
        dq[1, 1] = -1
    dq, dk = padded((dq, dk), pad)
    kw = dict(causal=False, scale=0.125, softcap=0.0, q_pos0=0, docs=(dq, dk))
    res, tol = reference(q, k, v, do, kw)
    for x in (q, do):
        x[dq < 0] = float("nan")
    for x in (k, v):
        x[dk < 0] = float("nan")
    o, lse, grads = run(hip, q, k, v, do, kw)
    check("o", o, res["o"], tol["o"])
    check_lse(lse, res["lse"], tol["lse"])
    for n, x in zip(("dq", "dk", "dv"), grads):
        check(n, x, res[n], tol[n])
    assert not o.cpu()[dq < 0].any() and not grads[0].cpu()[dq < 0].any() and not grads[1].cpu()[dk < 0].any()

# ---- fp16 gradients where the values are large ----------------------------------------------------------------------------------------------------
def check_fp16_grads(hip, q, k, v, do, kw):
    """reference()'s bounds, with what the smallest step of the scaled dT leaves: a row's (dQ) or the call's (dK) largest |dS| bound, at most
    2 max|dP|, is brought to 2^13 or more, half a smallest step is 2^-25"""
    res, tol = reference(q, k, v, do, kw)
    d, G = q.shape[3], q.shape[2] // k.shape[2]
    fl = 2 * d * float(do.double().abs().max()) * float(v.double().abs().max()) * 2.0 ** -38
    keys = k.double().abs().sum(1).repeat_interleave(G, 1)[:, None]
    rows = q.double().abs().sum(1).unflatten(1, (k.shape[2], G)).sum(2)[:, None]
    tol["dq"], tol["dk"] = tol["dq"] + kw["scale"] * fl * keys, tol["dk"] + kw["scale"] * fl * rows
    o, lse, grads = run(hip, q, k, v, do, kw)
    check("o", o, res["o"], tol["o"])
    for n, x in zip(("dq", "dk", "dv"), grads):
        assert not torch.isnan(x).any(), n
        check(n, x.float().clamp(-65504, 65504), res[n].clamp(-65504, 65504), tol[n])
    return res


@pytest.mark.parametrize("mag,back", [(30.0, 1.0), (1000.0, 1.0), (8000.0, 1e-3), (8000.0, 30.0)])
@pytest.mark.parametrize("name", ["long", "cap_d64", "d128", "docs", "rel_causal_cap", "tokens"])
def test_fp16_gradient_of_large_values(hip, name, mag, back):
    q, k, v, do, kw = problem(name, F16, seed=12)
    check_fp16_grads(hip, q, k, (v.float() * mag).clamp(-65504, 65504).half(), (do.float() * back).half(), kw)


@pytest.mark.parametrize("val,back,chan", [(32.0, 1.0, 128), (40.0, 1.0, 128), (8000.0, 1e-3, 1), (512.0, 1.0, 128), (60000.0, 1.0, 1)])
def test_fp16_gradient_of_two_keys(hip, val, back, chan):
    """two keys at P = 1/2 with values +-val in `chan` channels and a constant gradient: dS = +-val back chan / 2, dT is the same; its rounding must not pass
    fp16's range where dQ = scale dS (k1 - k2) and dK = scale sum dS q stay inside it"""
    g = gen(43)
    N = 40
    q, k = torch.zeros(1, N, 2, 128), torch.zeros(1, 2, 2, 128)
    q[..., 0], k[..., 0] = 2.0 ** -9 * randn(g, 1, N, 2), 1.0            # the only channel q has is the one the keys share: equal scores
    k[..., 1:] = 2.0 ** -4 * randn(g, 1, 2, 2, 127)
    v = torch.zeros(1, 2, 2, 128)
    v[:, 0, :, :chan], v[:, 1, :, :chan] = val, -val
    kw = dict(causal=False, scale=128 ** -0.5, softcap=0.0, q_pos0=0)
    res = check_fp16_grads(hip, q.half(), k.half(), v.half(), torch.full((1, N, 2, 128), back).half(), kw)
    assert float(res["dq"].abs().max()) < 65504 and float(res["dk"].abs().max()) < 65504


def test_fp16_gradient_of_a_quiet_document(hip):
    """two documents whose losses differ by 2^14: the quiet one's dK and dV keep their bits (bounds of a call of its own, and the smallest step that
    the loud one leaves)"""
    q, k, v, do, kw = problem("docs", F16, seed=13)
    ids = torch.zeros(q.shape[0], q.shape[1], dtype=torch.int32)
    ids[:, 150:] = 1
    do[:, 150:] *= 2.0 ** -14
    kw["docs"] = (ids, ids)
    check_fp16_grads(hip, q, k, v, do, kw)
    quiet = [x[:, 150:].contiguous() for x in (q, k, v, do)]
    alone = dict(kw, docs=None)
    res, tol = reference(*quiet, {n: x for n, x in alone.items() if x is not None})
    fl = 2 * q.shape[3] * float(do.double().abs().max()) * float(v.double().abs().max()) * 2.0 ** -38
    rows = quiet[0].double().abs().sum(1).unflatten(1, (k.shape[2], -1)).sum(2)[:, None]
    _, _, grads = run(hip, q, k, v, do, kw)
    check("dk", grads[1][:, 150:], res["dk"], tol["dk"] + kw["scale"] * fl * rows)

# ---- caps ------------------------------------------------------------------------------------------------------------------------------------------
def cap_bounds(q, k, v, do, kw):
    """fp64 results and bounds that do not grow with the cap.  A score's error: the product's, scale sum|q k| (d + 4) 2^-24 (the cap's slope is at most 1),
    and the cap's own, at most 2^-20 |u| (below a quarter of the cap the odd series ends 2^-26 short and rounds six times, above it 1 - 2 / (1 + e^2x)
    is off by 2^-23 of the cap <= 4.1 |u|).  A probability below fp32's smallest normal, 2^-126, may come out as zero."""
    u, d, cap, scale = half_step(q.dtype), q.shape[3], kw["softcap"], kw["scale"]
    Hk, G = k.shape[2], q.shape[2] // k.shape[2]
    vis, dist = tr.visible(q.shape[0], q.shape[1], k.shape[1], kw["causal"], kw.get("docs"), None, None, kw.get("q_pos0"))
    leaves = [x.double().requires_grad_() for x in (q, k, v)]
    r = tr.attention(*leaves, vis, dist, scale, cap, kw["slopes"].double() if "slopes" in kw else None, kw["rel"].double() if "rel" in kw else None)
    grads = torch.autograd.grad(r["o"], leaves, do.double())
    with torch.no_grad():
        tiny = torch.finfo(q.dtype).smallest_normal * torch.finfo(q.dtype).eps
        P, kk, vv, dob = r["P"], r["k"].permute(0, 2, 1, 3), r["v"].permute(0, 2, 1, 3), do.double().permute(0, 2, 1, 3)
        qa = q.double().abs().permute(0, 2, 1, 3)
        es = float(torch.matmul(qa, kk.abs().transpose(2, 3)).max()) * scale * (d + 4) * 2.0 ** -24 + float(r["u"].abs().max()) * 2.0 ** -20 + 2.0 ** -18
        E = 2 * es

        def rows(x):
            return x.permute(0, 2, 1, 3)

        def fold(x):
            return rows(x).unflatten(2, (Hk, G)).sum(3)

        dP = torch.matmul(dob, vv.transpose(2, 3))
        D = (P * dP).sum(-1, keepdim=True)
        dS = P * (dP - D)
        tdP = torch.matmul(dob.abs(), vv.abs().transpose(2, 3)) * (d + 4) * 2.0 ** -24
        tD = (P * (tdP + E * dP.abs())).sum(-1, keepdim=True) * 1.02
        dT = dS * (1 - (r["u"] / cap) ** 2)
        tT = (P * (tdP + tD) + E * (dS.abs() + P * tD) + dS.abs() * 2.0 ** -20 + 2.0 ** -126 * r["vis"] * (dP - D).abs()) * 1.02 + u * dT.abs()
        if q.dtype is F16:
            tT = tT + r["vis"] * float(dP.abs().max()) * 2.0 ** -37          # (check_fp16_grads)
        tol = {"o": u * r["o"].abs() + (u + E) * rows(torch.matmul(P, vv.abs())) * 1.02 + tiny, "lse": es + r["lse"].abs().nan_to_num(posinf=0) * 2.0 ** -21 + 2.0 ** -20,
               "dq": u * grads[0].abs() + scale * rows(torch.matmul(tT, kk.abs())) * 1.02 + tiny,
               "dk": u * grads[1].abs() + scale * fold(torch.matmul(tT.transpose(2, 3), qa)) * 1.02 + tiny,
               "dv": u * grads[2].abs() + fold(torch.matmul(((u + E) * P + (2.0 ** -34 if q.dtype is F16 else 2.0 ** -126)).transpose(2, 3), dob.abs())) * 1.02 + tiny}
    return {"o": r["o"].detach(), "lse": r["lse"].detach(), "dq": grads[0], "dk": grads[1], "dv": grads[2]}, tol


@pytest.mark.parametrize("cap", [100.0, 150.0, 1e4, 1e6, 1e9, 1e30])
@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("name", ["cap", "cap_d64", "docs_causal_cap", "rel_causal_cap", "token", "d40_slopes", "rel_docs"])
def test_caps_far_above_the_scores(hip, name, dt, cap):
    q, k, v, do, kw = problem(name, dt, seed=15)
    kw.pop("kv_len", None)
    kw["softcap"] = cap
    res, tol = cap_bounds(q, k, v, do, kw)
    o, lse, grads = run(hip, q, k, v, do, kw)
    check("o", o, res["o"], tol["o"])
    check_lse(lse, res["lse"], tol["lse"])
    for n, x in zip(("dq", "dk", "dv"), grads):
        check(n, x, res[n], tol[n])


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("name", ["cap", "cap_d64", "token"])
def test_a_large_cap_that_bends(hip, name, dt):
    """scores of several hundred under a cap of 200: both of the cap's forms, and the border between them (t / cap = 1/4) inside one tile"""
    q, k, v, do, kw = problem(name, dt, seed=16)
    kw.pop("kv_len", None)
    q = (q.float() * 32).to(dt)
    kw["softcap"] = 200.0
    res, tol = cap_bounds(q, k, v, do, kw)
    o, lse, grads = run(hip, q, k, v, do, kw)
    check("o", o, res["o"], tol["o"])
    check_lse(lse, res["lse"], tol["lse"])
    for n, x in zip(("dq", "dk", "dv"), grads):
        check(n, x, res[n], tol[n])


@pytest.mark.parametrize("cap", [1e-3, 1e-36, 1e-38, 1e-40])
@pytest.mark.parametrize("name", ["cap", "cap_d64", "token"])
def test_caps_far_below_the_scores(hip, name, cap):
    """every score becomes +-cap: equal weights.  A zero query row has score 0 and the cap's full slope there; rows of zeros are the only ones with a gradient
    for q.  (cap 1e-3: reference()'s bounds, the slope of small scores included)"""
    q, k, v, do, kw = problem(name, BF16, seed=17)
    kw.pop("kv_len", None)
    q[:, 0] = 0
    kw["softcap"] = cap
    res, tol = reference(q, k, v, do, kw)
    o, lse, grads = run(hip, q, k, v, do, kw)
    check("o", o, res["o"], tol["o"])
    check_lse(lse, res["lse"], tol["lse"])
    for n, x in zip(("dq", "dk", "dv"), grads):
        assert torch.isfinite(x).all(), n
    check("dv", grads[2], res["dv"], tol["dv"])
    check("dq", grads[0][:, :1], res["dq"][:, :1], tol["dq"][:, :1])

# ---- what a mask hides, gradient ---------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("what", ["a document without queries", "documents in between", "ahead of its document's queries", "two documents' tiles"])
@pytest.mark.parametrize("dt,d", [(F16, 64), (BF16, 128)])
def test_keys_that_no_query_sees_hold_anything(hip, dt, d, what, bad):
    g = gen(44)
    q, k, v, do = (randn(g, 2, 150, 2, d).to(dt) for _ in range(4))
    kw = dict(causal=False, scale=d ** -0.5, softcap=0.0, q_pos0=0)
    dq = torch.zeros(2, 150, dtype=torch.int32)
    dk, gone = dq.clone(), torch.zeros(2, 150, dtype=torch.bool)
    if what == "a document without queries":
        dk[1, 40:71] = 9
        gone[1, 40:71] = True
    elif what == "documents in between":                                  # the missing number lies between two that the block has
        dq[:, 70:] = dk[:, 70:] = 12
        dk[:, 60:90] = 9
        gone[:, 60:90] = True
    elif what == "ahead of its document's queries":                       # document 1's queries end before its last keys begin
        kw["causal"] = True
        dq[:, 30:50] = 1
        dk[:, 20:50] = 1
        dk[:, 100:110] = 1
        gone[:, 100:110] = True
    else:
        kw["causal"] = True
        dq[0, 64:] = dk[0, 64:] = 1
        dk[0, 120:130], dk[1, 3:5] = 4, 4
        gone[0, 120:130], gone[1, 3:5] = True, True
    kw["docs"] = (dq, dk)
    vis, _ = tr.visible(2, 150, 150, kw["causal"], kw["docs"], None, None, 0)
    assert torch.equal(gone, ~vis.any(1))
    res, tol = reference(q, k, v, do, kw)
    k[gone], v[gone] = bad, bad
    o, lse, grads = run(hip, q, k, v, do, kw)
    check("o", o, res["o"], tol["o"])
    check_lse(lse, res["lse"], tol["lse"])
    for n, x in zip(("dq", "dk", "dv"), grads):
        check(n, x, res[n], tol[n])
    assert not grads[1].cpu()[gone].any() and not grads[2].cpu()[gone].any()


@pytest.mark.parametrize("name,dt,key", [("docs", F16, 100), ("docs_causal_cap", BF16, 60), ("prefix", F16, 155), ("d40_slopes", BF16, 50), ("rel_causal_cap", F16, 130),
                                         ("tokens", BF16, 698)])
def test_dq_depends_on_what_its_row_sees_alone(hip, name, dt, key):
    """a NaN or infinity in a key or value reaches dQ of the rows that see it, and no other row's"""
    q, k, v, do, kw = problem(name, dt, seed=18)
    res, tol = reference(q, k, v, do, kw)
    vis, _ = tr.visible(q.shape[0], q.shape[1], k.shape[1], kw["causal"], kw.get("docs"), kw.get("prefix"), kw.get("kv_len"), kw.get("q_pos0"))
    for x, bad, cols in ((k, float("nan"), slice(None)), (v, float("inf"), slice(None)), (k, float("inf"), [2]), (k, float("nan"), [0, 5]), (v, float("nan"), [1])):
        kb, vb = k.clone(), v.clone()
        (kb if x is k else vb)[:, key, :, cols] = bad
        _, _, grads = run(hip, q, kb, vb, do, kw)
        blind = ~vis[:, :, key]
        m = blind[:, :, None, None].expand_as(res["dq"])
        check("dq blind", torch.where(m, grads[0].cpu().double(), res["dq"]), res["dq"], tol["dq"])
        assert bool(blind.any()) and bool((~blind).any())
        assert not torch.isfinite(grads[0].cpu()[~m]).all()

@pytest.mark.parametrize("cap", [40.0, 300.0, 1e5])
@pytest.mark.parametrize("name,dt", [("docs_causal_cap", F16), ("cap_d64", BF16)])
def test_row_by_row_forms_under_any_cap(hip, name, dt, cap):
    """one row's NaN key and value leave the other rows of its tile to their visible keys, one by one: o and dq there keep the cap's bounds"""
    q, k, v, do, kw = problem(name, dt, seed=19)
    q = (q.float() * 8).to(dt)
    if "docs" not in kw:                                    # key 30 is seen by the rows of its document alone
        ids_q, ids_k = torch.zeros(q.shape[:2], dtype=torch.int32), torch.zeros(k.shape[:2], dtype=torch.int32)
        ids_q[:, 7], ids_k[:, 25:33] = 1, 1
        kw["docs"] = (ids_q, ids_k)
    key = 60 if name == "docs_causal_cap" else 30
    kw["softcap"] = cap
    res, tol = cap_bounds(q, k, v, do, kw)
    blind = ~tr.visible(q.shape[0], q.shape[1], k.shape[1], kw["causal"], kw["docs"], None, None, kw.get("q_pos0"))[0][:, :, key]
    k[:, key], v[:, key] = float("nan"), float("nan")
    o, _, grads = run(hip, q, k, v, do, kw)
    m = blind[:, :, None, None].expand_as(res["o"])
    assert bool(m.any()) and not bool(m.all())
    for n, x in (("o", o), ("dq", grads[0])):
        check(n, torch.where(m, x.cpu().double(), res[n]), res[n], tol[n])


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf"), "row"])
@pytest.mark.parametrize("name,dt,key", [("docs", F16, 100), ("text", F16, 40), ("d128", BF16, 70), ("cap", BF16, 64), ("tokens", BF16, 690), ("token_long", F16, 3000), ("d72", F16, 66)])
def test_a_bad_value_that_rows_see(hip, name, dt, key, bad):
    """an infinity or NaN in some columns of one value shows in those columns of the rows that see it, and nowhere else; a value row of NaN makes them NaN"""
    q, k, v, do, kw = problem(name, dt, seed=20)
    res, tol = reference(q, k, v, do, kw, grads=False)
    vis, _ = tr.visible(q.shape[0], q.shape[1], k.shape[1], kw["causal"], kw.get("docs"), kw.get("prefix"), kw.get("kv_len"), kw.get("q_pos0"))
    cols = slice(None) if bad == "row" else [1, q.shape[3] - 1]
    v[:, key, :, cols] = float("nan") if bad == "row" else bad
    o, lse = hip.masked_attention(q.to(DEV), k.to(DEV), v.to(DEV), **on_gpu(kw))
    check_lse(lse, res["lse"], tol["lse"])
    o, hit = o.cpu(), torch.zeros(res["o"].shape, dtype=torch.bool)
    hit[:, :, :, cols] = vis[:, :, key, None, None]
    assert bool(hit.any())
    check("o", torch.where(hit, res["o"], o.double()), res["o"], tol["o"])
    assert torch.isnan(o[hit]).all() if bad == "row" or bad != bad else (o[hit] == bad).all()


# ---- many small probabilities ------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("Nq,H", [(1, 1), (130, 40)])
@pytest.mark.parametrize("below", [17.0, 20.4, 24.6])
def test_many_small_probabilities_beside_a_large_one(hip, below, Nq, H, dt):
    """2^17 keys whose probabilities are 2^-below of the first one's: their sum counts.  Rounded to fp16 as P 2^9, each is off by at most 2^-34 of the largest
    (half a smallest step, 2^-25, over 2^9; the running maximum is at most 2^6 below the largest score) beside its relative half step"""
    N, d = 1 << 17, 64
    q, k, v = torch.zeros(1, Nq, H, d), torch.zeros(1, N, 1, d), torch.ones(1, N, 1, d)
    q[..., 0], k[:, 0, :, 0], v[:, 0] = 8.0, below * math.log(2.0), 0.0
    v[:, 1:, :, 1] = 0.5
    q, k, v = (x.to(dt) for x in (q, k, v))
    kw = dict(scale=0.125, causal=False, softcap=0.0, q_pos0=0)
    s = float(k[0, 0, 0, 0].double()) * 8.0 * 0.125
    P = math.exp(-s) / (1 + (N - 1) * math.exp(-s))
    ref = torch.full((1, Nq, H, d), (N - 1) * P, dtype=torch.float64)
    ref[..., 1] *= 0.5
    E = 2 * (s * (d + 4) * 2.0 ** -24 + 2.0 ** -20)
    o, lse = hip.masked_attention(q.to(DEV), k.to(DEV), v.to(DEV), **kw)
    # (the sum of N fp32 terms of one size: 2^-24 of it a step, at most N / 64 steps in a lane's chain)
    check("o", o, ref, (2 * half_step(dt) + E + N / 64 * 2.0 ** -24) * ref + (N * 2.0 ** -34 if dt is F16 else 0.0))
