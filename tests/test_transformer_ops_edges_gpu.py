"""mgld_vsr_amd.hip's transformer operators at the edges of their ranges: padding numbers, magnitudes, caps, masked places.  Oracle, problems and
error bounds are those of test_transformer_ops_gpu.py; a bound that a case adds is derived where it stands."""
import math

import pytest
import torch

from oracle import transformer as tr
from test_transformer_ops_gpu import ATT, BF16, DEV, F16, check, check_lse, docs_of, gen, half_step, on_gpu, problem, randn, reference

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
