"""The transformer operators' host side (no GPU): refusals of the C entry points and of the wrappers, work sizes, bucket borders, the oracle's
gradient against differences."""
import ctypes as C

import pytest
import torch

from mgld_vsr_amd import build, hip
from oracle import transformer as tr


@pytest.fixture(scope="module")
def lib():
    build.build(verbose=False)
    return hip.lib()


def attn(**kw):
    p = hip.MgldMaskAttn()
    p.batch, p.heads, p.kv_heads, p.Nq, p.Nkv, p.head_dim, p.scale = 2, 4, 2, 100, 200, 64, 0.125
    for n in ("Q", "K", "V", "O", "lse", "dO", "dQ", "dK", "dV"):
        setattr(p, n, 0x10000)             # never read: every call here is refused
    for n in ("q", "o", "do", "dq"):
        setattr(p, n + "_sb", 25600), setattr(p, n + "_si", 256), setattr(p, n + "_sh", 64)
    for n in ("k", "v", "dk", "dv"):
        setattr(p, n + "_sb", 25600), setattr(p, n + "_si", 128), setattr(p, n + "_sh", 64)
    for n, x in kw.items():
        setattr(p, n, x)
    return p


BAD = [dict(kv_heads=3), dict(heads=0), dict(kv_heads=0), dict(batch=-1), dict(Nq=-1), dict(Nkv=-1), dict(head_dim=0), dict(head_dim=60), dict(head_dim=136),
       dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(softcap=-1.0), dict(softcap=float("nan")), dict(Q=None), dict(K=None), dict(V=None),
       dict(O=None), dict(Q=0x10008), dict(k_si=130), dict(v_sh=63), dict(o_sb=4), dict(k_si=-128), dict(k_si=1 << 23), dict(prefix=0x1000),
       dict(doc_q=0x1000), dict(doc_k=0x1000), dict(rel=0x1000, reach=1025), dict(rel=0x1000, reach=-1), dict(rel=0x1000, reach=4, slopes=0x1000),
       dict(q_pos0=(1 << 30) + 1), dict(Nkv=(1 << 30) + 1)]


@pytest.mark.parametrize("bad", BAD, ids=lambda b: ",".join(f"{n}={x}" for n, x in b.items()))
def test_c_entry_refuses(lib, bad):
    p = attn(**bad)
    assert lib.mgld_masked_attention(C.byref(p), None) == -1
    if bad not in (dict(O=None), dict(o_sb=4)):          # (the gradient does not read O; without a work buffer it is refused all the same)
        assert lib.mgld_masked_attention_grad_work(C.byref(p)) == 0
    assert lib.mgld_masked_attention_grad(C.byref(p), None) == -1
    assert lib.mgld_masked_attention_work(C.byref(p)) == 0


@pytest.mark.parametrize("bad", [dict(dO=None), dict(dQ=None), dict(dK=None), dict(dV=0x10008), dict(lse=None), dict(dk_si=1), dict(work=0x10000, work_bytes=16),
                                 dict(), dict(heads=32, rel=0x1000, reach=1024, work=0x10000, work_bytes=1 << 40), dict(dRel=0x1000, work=0x10000, work_bytes=1 << 40)])
def test_c_gradient_refuses(lib, bad):
    p = attn(**bad)
    assert lib.mgld_masked_attention_grad(C.byref(p), None) == -1


def test_c_entry_work_buffer(lib):
    """documents and split keys need a work buffer of the size the library names"""
    p = attn(Nq=1, Nkv=50000)
    need = lib.mgld_masked_attention_work(C.byref(p))
    assert need > 0 and lib.mgld_masked_attention(C.byref(p), None) == -1
    p.work, p.work_bytes = 0x10000, need - 1
    assert lib.mgld_masked_attention(C.byref(p), None) == -1
    p.work, p.work_bytes = 0x10004, need
    assert lib.mgld_masked_attention(C.byref(p), None) == -1
    d = attn(doc_q=0x1000, doc_k=0x1000)
    assert lib.mgld_masked_attention_work(C.byref(d)) >= 16 * 2 * (2 + 4)
    assert lib.mgld_masked_attention_work(C.byref(attn())) == 0
    assert lib.mgld_masked_attention(None, None) == -1 and lib.mgld_masked_attention_work(None) == 0
    # empty problems: nothing to do, nothing launched
    assert lib.mgld_masked_attention(C.byref(attn(batch=0)), None) == 0 and lib.mgld_masked_attention(C.byref(attn(Nq=0)), None) == 0
    assert lib.mgld_masked_attention_grad(C.byref(attn(batch=0)), None) == 0


def test_c_qk_norm_rope_refuses(lib):
    def p(**kw):
        s = hip.MgldQkRope()
        s.rows, s.head_dim, s.rot_dim, s.eps, s.pos, s.freqs = 5, 64, 64, 1e-6, 0x1000, 0x1000
        for h in (s.q, s.k):
            h.x = h.y = h.dy = 0x10000
            h.heads, h.x_sr, h.x_sh, h.y_sr, h.y_sh, h.dy_sr, h.dy_sh = 2, 128, 64, 128, 64, 128, 64
        for n, x in kw.items():
            o, n = (getattr(s, n[0]), n[2:]) if n[1] == "_" else (s, n)
            setattr(o, n, x)
        return s
    for bad in (dict(rows=-1), dict(head_dim=60), dict(head_dim=264), dict(rot_dim=12), dict(rot_dim=72), dict(rot_dim=-8), dict(eps=-1.0), dict(pos=None), dict(freqs=None),
                dict(q_x=None), dict(k_y=None), dict(q_x=0x10004), dict(k_x_sr=66), dict(q_y_sh=2), dict(q_heads=0, k_heads=0), dict(q_heads=-1)):
        s = p(**bad)
        assert lib.mgld_qk_norm_rope(C.byref(s), None) == -1, bad
        assert lib.mgld_qk_norm_rope_grad(C.byref(s), None) == -1, bad
    assert lib.mgld_qk_norm_rope_grad(C.byref(p(q_dy=None)), None) == -1
    assert lib.mgld_qk_norm_rope_grad(C.byref(p(q_dgamma=0x1000)), None) == -1                    # needs work
    assert lib.mgld_qk_norm_rope(C.byref(p(rows=0)), None) == 0
    assert lib.mgld_qk_norm_rope_grad_work(C.byref(p())) >= 2 * 64 * 4
    for args in ((0, 0x1000, 0x1000, 4, 2, 9), (0x1000, 0x1000, 0x1000, 0, 2, 9), (0x1000, 0x1000, 0x1000, 4, 0, 9), (0x1000, 0x1000, 0x1000, 4, 2, 0)):
        a = [C.c_void_p(x) for x in args[:3]] + list(args[3:]) + [None]
        assert lib.mgld_rel_bias(*a) == -1 and lib.mgld_rel_bias_grad(*a) == -1


class _Quiet:
    """a library whose entry points succeed without doing anything, and which records that they were reached"""

    def __init__(self, real):
        self.real, self.calls = real, []

    def __getattr__(self, n):
        if n.endswith("_work"):
            return getattr(self.real, n)

        def call(*a):
            self.calls.append(n)
            return 0
        return call


@pytest.fixture
def quiet(lib, monkeypatch):
    q = _Quiet(lib)
    monkeypatch.setattr(hip, "lib", lambda: q)
    monkeypatch.setattr(hip, "_req_cuda", lambda *t: None)
    monkeypatch.setattr(hip, "_capturing", lambda: False)
    monkeypatch.setattr(hip, "stream_ptr", lambda: None)
    return q


def h(*s):
    return torch.zeros(*s, dtype=torch.float16)


def test_wrappers_refuse(quiet, monkeypatch):
    q, k = h(2, 10, 4, 64), h(2, 20, 2, 64)
    f, i32 = torch.zeros, torch.int32
    hip.masked_attention(q, k, k, causal=True, softcap=3.0, slopes=f(4), kv_len=f(2, dtype=i32), prefix=f(2, dtype=i32),
                         docs=(f(2, 10, dtype=i32), f(2, 20, dtype=i32)), q_pos0=3)
    assert quiet.calls == ["mgld_masked_attention"]
    quiet.calls.clear()
    buf = h(2, 10, 4 * 64 + 4 * 64)
    bad = [dict(q=q.float()), dict(k=k.bfloat16()), dict(q=h(10, 4, 64)), dict(q=h(2, 10, 3, 64)), dict(k=h(3, 20, 2, 64), v=h(3, 20, 2, 64)), dict(v=h(2, 21, 2, 64)),
           dict(q=h(2, 10, 4, 60), k=h(2, 20, 2, 60), v=h(2, 20, 2, 60)), dict(q=h(2, 10, 4, 136), k=h(2, 20, 2, 136), v=h(2, 20, 2, 136)), dict(q=h(2, 10, 64, 4).transpose(2, 3)),
           dict(scale=0.0), dict(scale=-1.0), dict(softcap=-2.0), dict(scale=float("nan")), dict(slopes=f(3)), dict(slopes=f(4).double()), dict(slopes=f(8)[::2]),
           dict(rel=f(4, 8)), dict(rel=f(3, 9)), dict(rel=f(4, 2051)), dict(rel=f(4, 9), slopes=f(4)), dict(docs=f(2, 10, dtype=i32)), dict(docs=(f(2, 10), f(2, 20))),
           dict(docs=(f(2, 10, dtype=i32), f(2, 10, dtype=i32))), dict(prefix=f(2, dtype=i32)), dict(prefix=f(3, dtype=i32), causal=True), dict(kv_len=f(2, dtype=torch.int64)),
           dict(kv_len=f(1, dtype=i32)), dict(q_pos0=1 << 31), dict(o=h(2, 10, 4, 32)), dict(o=q), dict(o=h(2, 10, 4, 64).bfloat16()), dict(o=h(2, 1, 4, 64).expand(2, 10, 4, 64)),
           dict(o=h(4000).as_strided((2, 10, 4, 64), (1000, 64, 32, 1))), dict(o=h(4000).as_strided((2, 10, 4, 64), (640, 256, 64, 1))),
           dict(lse=f(2, 10, 4)), dict(lse=f(2, 4, 10).double()), dict(lse=f(2, 10, 4).transpose(1, 2)),
           dict(q=buf[..., :256].unflatten(2, (4, 64)), o=buf[..., 64:320].unflatten(2, (4, 64)))]
    for b in bad:
        a = dict(q=q, k=k, v=b.get("v", b.get("k", k)))
        a.update(b)
        with pytest.raises((ValueError, RuntimeError)):
            hip.masked_attention(a.pop("q"), a.pop("k"), a.pop("v"), **a)
        assert not quiet.calls, b
    # column blocks of one buffer do not overlap
    hip.masked_attention(buf[..., :256].unflatten(2, (4, 64)), k, k, o=buf[..., 256:].unflatten(2, (4, 64)))
    assert quiet.calls == ["mgld_masked_attention"]
    quiet.calls.clear()
    long = h(2, 9000, 2, 64)
    with pytest.raises(ValueError, match="work"):
        hip.masked_attention(q[:, :1], long, long, work=torch.zeros(64, dtype=torch.uint8))
    o, lse = h(2, 10, 4, 64), f(2, 4, 10)
    for b in (dict(do=h(2, 10, 4, 32)), dict(lse=f(2, 10, 4)), dict(o=h(2, 10, 4, 64).bfloat16()), dict(dq=q), dict(dk=k), dict(dq=h(2, 10, 4, 32)), dict(dv=h(2, 20, 1, 64).expand(2, 20, 2, 64)),
              dict(rel=f(4, 9), drel=f(4, 7)), dict(work=torch.zeros(64, dtype=torch.uint8))):
        a = dict(o=o, lse=lse, do=h(2, 10, 4, 64))
        a.update(b)
        with pytest.raises(ValueError):
            hip.masked_attention_grad(q, k, k, a.pop("o"), a.pop("lse"), a.pop("do"), **a)
        assert not quiet.calls, b
    monkeypatch.setattr(hip, "_capturing", lambda: True)
    with pytest.raises(ValueError, match="captured"):
        hip.masked_attention(q, k, k)
    with pytest.raises(ValueError, match="captured"):
        hip.rel_bias(f(4, 3), hip.rel_buckets(4, 8, device="cpu"))
    with pytest.raises(ValueError, match="captured"):
        hip.qk_norm_rope(h(4, 2, 64), None, f(4, dtype=i32), hip.rope_freqs(64, device="cpu"))


def test_rope_wrapper_refuses(quiet):
    q, k, pos, fr = h(6, 4, 64), h(6, 2, 64), torch.zeros(6, dtype=torch.int32), hip.rope_freqs(64, device="cpu")
    hip.qk_norm_rope(q, k, pos, fr, q_gamma=torch.zeros(64), q_out=q, k_out=k)
    hip.qk_norm_rope(q, None, None, None)
    assert len(quiet.calls) == 2
    quiet.calls.clear()
    big = h(6, 8, 64)
    for a, b in (((None, None, pos, fr), {}), ((q.float(), k, pos, fr), {}), ((q, k.bfloat16(), pos, fr), {}), ((q, h(5, 2, 64), pos, fr), {}), ((q, h(6, 2, 32), pos, fr), {}), ((q, k, pos[:5], fr), {}),
                 ((q, k, pos.float(), fr), {}), ((q, k, None, fr), {}), ((q, k, pos, fr.float()), {}), ((q, k, pos, torch.zeros(6, dtype=torch.float64)), {}),
                 ((q, k, pos, torch.zeros(64, dtype=torch.float64)), {}), ((q, k, pos, fr), dict(q_gamma=torch.zeros(32))), ((q, k, pos, fr), dict(eps=-1.0)), ((h(6, 4, 60), None, None, None), {}),
                 ((h(6, 4, 264), None, None, None), {}), ((big[:, :4], None, pos, fr), dict(q_out=big[:, 1:5])), ((q, k, pos, fr), dict(q_out=h(6, 4, 64).bfloat16())),
                 ((q, k, pos, fr), dict(k_out=h(6, 1, 64).expand(6, 2, 64))), ((big[:, :4], big[:, 4:6], pos, fr), dict(q_out=big[:, 4:8]))):
        with pytest.raises(ValueError):
            hip.qk_norm_rope(*a, **b)
        assert not quiet.calls, (a, b)
    for a, b in (((q, k, pos, fr, q, None), {}), ((q, None, pos, fr, h(6, 4, 32), None), {}), ((q, k, pos, fr, q, k), dict(dq=h(6, 4, 32))),
                 ((q, None, pos, fr, h(6, 4, 64), None), dict(q_gamma=torch.zeros(64), dq_gamma=torch.zeros(32))), ((big[:, :4], None, pos, fr, h(6, 4, 64), None), dict(dq=big[:, 2:6]))):
        with pytest.raises(ValueError):
            hip.qk_norm_rope_grad(*a, **b)
        assert not quiet.calls, (a, b)


def test_rel_wrappers_refuse(quiet):
    for a in ((7, 20), (2, 20), (32, 8), (32, 1025)):
        with pytest.raises(ValueError):
            hip.rel_buckets(*a, device="cpu")
    plan = hip.rel_buckets(8, 20, device="cpu")
    for t in (torch.zeros(7, 3), torch.zeros(8, 3).half(), torch.zeros(3, 8).t(), torch.zeros(24)):
        with pytest.raises(ValueError):
            hip.rel_bias(t, plan)
    for t in (torch.zeros(3, 40), torch.zeros(3, 41).double()):
        with pytest.raises(ValueError):
            hip.rel_bias_grad(t, plan)
    with pytest.raises(ValueError):
        hip.rel_bias(torch.zeros(8, 3), plan, out=torch.zeros(3, 39))
    assert not quiet.calls


def test_cpu_tensors_are_refused(lib):
    with pytest.raises(RuntimeError, match="device tensors"):
        hip.masked_attention(h(1, 1, 1, 64), h(1, 1, 1, 64), h(1, 1, 1, 64))
    with pytest.raises(RuntimeError, match="device tensors"):
        hip.qk_norm_rope(h(1, 1, 64), None, torch.zeros(1, dtype=torch.int32), hip.rope_freqs(64, device="cpu"))


@pytest.mark.parametrize("nb,maxd,both", [(32, 128, True), (32, 128, False), (16, 20, True), (4, 1024, True), (2, 2, False), (10, 500, True), (7, 100, False)])
def test_bucket_borders(nb, maxd, both):
    for n in range(-maxd - 3, maxd + 4):
        assert hip.rel_bucket(n, nb, maxd, both) == tr.rel_bucket(n, nb, maxd, both), n
    assert hip.rel_bucket(-maxd, nb, maxd, both) == hip.rel_bucket(-10 * maxd, nb, maxd, both) == (nb // 2 if both else nb) - 1


def test_kernel_structs_match_the_header(tmp_path):
    import shutil
    import subprocess
    gcc = shutil.which("gcc")
    if gcc is None:
        pytest.skip("no C compiler on this box")
    root = __file__.rsplit("/tests/", 1)[0]
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "mgld_hip.h"', "int main(void) {"]
    structs = (("MgldHeads", hip.MgldHeads), ("MgldQkRope", hip.MgldQkRope), ("MgldMaskAttn", hip.MgldMaskAttn))
    want = []
    for name, cls in structs:
        lines.append(f'  printf("%zu\\n", sizeof({name}));')
        want.append(C.sizeof(cls))
        for f, _ in cls._fields_:
            lines.append(f'  printf("%zu\\n", offsetof({name}, {f}));')
            want.append(getattr(cls, f).offset)
    (tmp_path / "p.c").write_text("\n".join(lines + ["  return 0;", "}"]))
    subprocess.check_call([gcc, "-I", root + "/include", str(tmp_path / "p.c"), "-o", str(tmp_path / "p")])
    assert [int(x) for x in subprocess.check_output([str(tmp_path / "p")]).split()] == want


def test_oracle_gradient_against_differences():
    """autograd of the fp64 oracle = difference quotients, mask, cap, bias and all"""
    g = torch.Generator().manual_seed(1)
    B, N, H, d = 1, 9, 2, 8
    q, k, v, do = (torch.randn(B, N, H, d, generator=g, dtype=torch.float64) for _ in range(4))
    rel = torch.randn(H, 7, generator=g, dtype=torch.float64)
    docs = torch.tensor([[0, 0, 0, 1, 1, 1, 1, -1, -1]])
    vis, dist = tr.visible(B, N, N, True, (docs, docs), None, None, 0)
    leaves = [x.requires_grad_() for x in (q, k, v, rel)]

    def f(q, k, v, rel):
        return (tr.attention(q, k, v, vis, dist, 0.3, 2.0, None, rel)["o"] * do).sum()
    grads = torch.autograd.grad(f(*leaves), leaves)
    with torch.no_grad():
        for i, x in enumerate(leaves):
            e = torch.randn(x.shape, generator=g, dtype=torch.float64)
            a = [y.clone() for y in leaves]
            b = [y.clone() for y in leaves]
            a[i] += 1e-5 * e
            b[i] -= 1e-5 * e
            quot = float((f(*a) - f(*b)) / 2e-5)
            assert abs(quot - float((grads[i] * e).sum())) < 1e-7 * (1 + abs(quot))
    y = torch.randn(3, 2, 16, generator=g, dtype=torch.float64, requires_grad=True)
    gm = torch.randn(16, generator=g, dtype=torch.float64, requires_grad=True)
    pos, fr = torch.tensor([0, 5, 1000]), torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64)
    for il in (False, True):
        assert torch.autograd.gradcheck(lambda a, b: tr.qk_norm_rope(a, pos, fr, b, 1e-6, il), (y, gm))


def test_work_sizes(quiet):
    """the sizes the helper names are the ones the calls ask for"""
    i32 = torch.int32
    q, k = h(2, 300, 4, 64), h(2, 300, 2, 64)
    docs = torch.zeros(2, 300, dtype=i32)
    rel = torch.zeros(4, 65)
    for qq, kw in ((q, {}), (q, dict(causal=True, docs=docs)), (q, dict(rel=rel)), (h(2, 2, 4, 64), dict(kv_len=torch.zeros(2, dtype=i32)))):
        for grad in (False, True):
            n = hip.masked_attention_work_bytes(qq, k, k, grad=grad, **kw)
            o, lse = torch.zeros_like(qq), torch.zeros(2, 4, qq.shape[1])
            run = (lambda w: hip.masked_attention_grad(qq, k, k, o, lse, o.clone(), work=w, **kw)) if grad else (lambda w: hip.masked_attention(qq, k, k, work=w, **kw))
            if n == 0:
                continue
            room = torch.zeros(n + 16, dtype=torch.uint8)
            room = room[-room.data_ptr() % 16:][:n]
            run(room)
            with pytest.raises(ValueError, match=str(n)):
                run(room[:-1])
