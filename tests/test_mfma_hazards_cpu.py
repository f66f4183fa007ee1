"""The generated code of the attention kernels reads no matrix result before it is there (tools/mfma_hazards.py)."""
import importlib.util
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _load(path, name):
    spec = importlib.util.spec_from_file_location(name, os.path.join(ROOT, path))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


LISTING = """
_Z4testv:
\tv_mfma_f32_16x16x32_f16 v[2:5], v[6:9], v[10:13], 0
\ts_cbranch_scc1 .LBB0_2
; %bb.1:
\ts_nop 6
\tv_add_f32_e32 v20, v2, v2
.LBB0_2:
\t{gap}
\tv_fma_f32 v25, v5, v27, v25
\ts_endpgm
.end_amdhsa_kernel
"""


def test_scan_follows_branches(tmp_path):
    tool = _load("tools/mfma_hazards.py", "mfma_hazards")
    for gap, want in (("s_nop 5", 0), ("s_nop 4", 1), ("v_mov_b32_e32 v30, 0", 1)):
        f = tmp_path / "a.s"
        f.write_text(LISTING.format(gap=gap))
        assert sum(len(tool.early_reads(c)) for c in tool.kernels(str(f)).values()) == want


@pytest.mark.parametrize("source", ["rel_attention.hip", "attention.hip"])
def test_attention_kernels_wait_for_their_products(source, tmp_path):
    hipcc = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
    if not shutil.which(hipcc):
        pytest.skip("no hipcc")
    tool, build = _load("tools/mfma_hazards.py", "mfma_hazards"), _load("build_ext.py", "build_ext")
    out = str(tmp_path / "k.s")
    subprocess.run([hipcc] + build.kernel_flags(source) + ["--cuda-device-only", "-S", os.path.join(ROOT, "csrc", "kernels", source),
                                                           "-o", out], check=True, capture_output=True)
    kernels = tool.kernels(out)
    assert any("mfma" in ins for code in kernels.values() for _, ins in code)
    bad = [(name, *b) for name, code in kernels.items() for b in tool.early_reads(code)]
    assert not bad, bad[:3]
