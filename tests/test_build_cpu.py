"""What the library is compiled to (no GPU): no packed fp32 arithmetic in any kernel, the normalisations' roundings as their source writes them."""
import os
import re
import subprocess

import pytest

import codeobj
from mgld_vsr_amd import build

OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"


def test_every_source_is_compiled_without_packed_fp32():
    for s in build.SOURCES:
        f = build.flags(s)
        assert any(f[i:i + 4] == ["-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"] for i in range(len(f))), s
    assert build.flags("norm.hip")[-1] == "-ffp-contract=off"


@pytest.fixture(scope="module")
def listings(tmp_path_factory):
    """{kernel: its instructions' names}, of every kernel of the built library"""
    if not os.path.exists(OBJDUMP):
        pytest.skip("no llvm-objdump")
    path = build.build(verbose=False)
    out, tmp = {}, tmp_path_factory.mktemp("co")
    for i, (triple, code) in enumerate(codeobj._bundles(open(path, "rb").read())):
        if "gfx950" not in triple or not code:
            continue
        f = tmp / f"{i}.co"
        f.write_bytes(code)
        text = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", str(f)], check=True, stdout=subprocess.PIPE, text=True).stdout
        for part in re.split(r"^[0-9a-f]+ <", text, flags=re.M)[1:]:
            name, body = part.split(">:", 1)
            out[name] = re.findall(r"^\s+([vs]_\w+)", body, flags=re.M)
    assert len(out) > 200
    return out


def test_no_packed_fp32_arithmetic(listings):
    bad = {n: sorted({x for x in ins if re.match(r"v_pk_(add|mul|fma)_f32", x)}) for n, ins in listings.items()}
    assert not {n: x for n, x in bad.items() if x}


def test_squares_round_by_themselves(listings):
    """gn_fused's and layernorm's squared sums are product and sum (their source's roundings), not fused: 128 and 8 products that only they make"""
    def count(frag, *ops):
        n = [k for k in listings if frag in k]
        assert len(n) == 1, n
        return sum(re.sub(r"_e32$|_e64$", "", x) in ops for x in listings[n[0]])
    assert count("gn_fused_kernelILb1ELb0E", "v_mul_f32") >= 128
    assert count("layernorm_kernelILi1ELb0E", "v_mul_f32") >= 8 + 8
