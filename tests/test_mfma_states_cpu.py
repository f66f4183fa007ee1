"""tools/mfma_hazards.py on gfx950 listings: the states a product needs there, accumulation registers, the GEMM kernels."""
import os
import shutil
import subprocess

import pytest

from test_mfma_hazards_cpu import ROOT, _load

HEAD = '\t.amdgcn_target "amdgcn-amd-amdhsa--{target}"\n_Z4testv:\n'
TAIL = "\ts_endpgm\n.end_amdhsa_kernel\n"


def _count(tmp_path, body, target="gfx950"):
    tool = _load("tools/mfma_hazards.py", "mfma_hazards")
    f = tmp_path / "a.s"
    f.write_text(HEAD.format(target=target) + "".join(f"\t{line}\n" for line in body) + TAIL)
    return sum(len(tool.early_reads(c)) for c in tool.kernels(str(f)).values())


@pytest.mark.parametrize("product,states", [("v_mfma_f32_16x16x32_f16", 8), ("v_mfma_f32_16x16x32_bf16", 8), ("v_mfma_f32_32x32x16_f16", 12)])
@pytest.mark.parametrize("result,read", [("v[2:5]", "v_add_f32_e32 v20, v2, v2"), ("a[2:5]", "v_accvgpr_read_b32 v20, a5"),
                                         ("v[2:5]", "ds_write_b64 v9, v[4:5]"), ("a[2:5]", "global_store_dwordx4 v[8:9], a[2:5], off")])
def test_states_between_a_product_and_its_reader(tmp_path, product, states, result, read):
    code = lambda n: [f"{product} {result}, v[6:9], v[10:13], 0", f"s_nop {n - 1}", read]
    assert _count(tmp_path, code(states)) == 0 and _count(tmp_path, code(states - 1)) == 1
    assert _count(tmp_path, code(states - 1), "gfx942") == 0 and _count(tmp_path, code(states - 2), "gfx942") == 1


def test_registers_of_either_kind_are_told_apart(tmp_path):
    code = ["v_mfma_f32_16x16x32_f16 a[2:5], v[6:9], v[10:13], 0", "v_add_f32_e32 v20, v2, v2", "v_accvgpr_read_b32 v21, a6"]
    assert _count(tmp_path, code) == 0
    assert _count(tmp_path, code + ["v_accvgpr_read_b32 v21, a2"]) == 1


def test_a_branch_counts_as_one_state(tmp_path):
    code = lambda n: ["v_mfma_f32_16x16x32_f16 v[2:5], v[6:9], v[10:13], 0", "s_branch .LBB0_2", f"s_nop {n}", "v_mov_b32_e32 v2, v2"]
    tool = _load("tools/mfma_hazards.py", "mfma_hazards")
    for n, want in ((6, 0), (5, 1)):
        f = tmp_path / "b.s"
        lines = code(n)
        f.write_text(HEAD.format(target="gfx950") + f"\t{lines[0]}\n\t{lines[1]}\n.LBB0_2:\n\t{lines[2]}\n\t{lines[3]}\n" + TAIL)
        assert sum(len(tool.early_reads(c)) for c in tool.kernels(str(f)).values()) == want


@pytest.mark.parametrize("source", ["gemm_nt.hip", "gemm_nn.hip", "gemm_tn.hip"])
def test_gemm_kernels_wait_for_their_products(source, tmp_path):
    hipcc = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
    if not shutil.which(hipcc):
        pytest.skip("no hipcc")
    tool, build = _load("tools/mfma_hazards.py", "mfma_hazards"), _load("build_ext.py", "build_ext")
    out = str(tmp_path / "k.s")
    subprocess.run([hipcc] + build.kernel_flags(source) + ["--cuda-device-only", "-S", os.path.join(ROOT, "csrc", "kernels", source),
                                                           "-o", out], check=True, capture_output=True)
    kernels = tool.kernels(out)
    assert all(code[0] == ("target", "gfx950") for code in kernels.values())
    assert any("mfma" in ins for code in kernels.values() for _, ins in code)
    bad = [(name, *b) for name, code in kernels.items() for b in tool.early_reads(code)]
    assert not bad, bad[:3]
