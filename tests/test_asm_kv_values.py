"""Cached attention: a page's codes are still in their registers when they are
widened (CPU only: hipcc -S).

The compiler once kept V's codes and the probabilities' terms in the same
registers.  V's tail mask sat in a branch, vr[t][w] &= mask; behind it,

    v_cvt_pk_bf16_f32 v46, v35, s0                 a term of the probabilities
    ...
    v_cvt_scalef32_pk_bf16_fp8 v116, v46, 1.0      V's codes, which v46 held

so rows of head_dim 64 came out wrong (ROCm 7.2.0, clang 22.0.0git 7b800a19).
The source said nothing of the kind: V is written by its load and the mask alone.
Since then every page is masked without a branch.  The scan reads the compiled
kernels: within a basic block, the last writer of a register that is widened is a
load, the mask, or the select that drops what lies past head_dim.
"""
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "lightining-core_amd", "csrc")
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")

_FINE = ("global_load_dwordx4", "v_and_b32_e32", "v_and_b32_e64", "v_cndmask_b32_e32", "v_cndmask_b32_e64")


def _regs(operand):
    m = re.match(r"v\[(\d+):(\d+)\]$", operand)
    if m:
        return range(int(m.group(1)), int(m.group(2)) + 1)
    m = re.match(r"v(\d+)$", operand)
    return [int(m.group(1))] if m else []


def scan(text):
    """(registers widened whose last writer the block shows, those written by something else)."""
    writer, seen, wrong = {}, 0, []
    for line in text.split("\n"):
        t = line.split(";")[0].strip()
        if t.endswith(":"):
            writer = {}  # what came before is not known here
            continue
        parts = t.split(None, 1)
        if len(parts) < 2 or t.startswith("."):
            continue
        name, operands = parts[0], [x.strip() for x in parts[1].split(",")]
        if name.startswith("v_cvt_scalef32_pk_bf16_fp8"):
            for r in _regs(operands[1].split()[0]):
                if r in writer:
                    seen += 1
                    if not writer[r].startswith(_FINE):
                        wrong.append(f"[{writer[r]}] -> [{t}]")
        if name.startswith(("v_", "global_load", "ds_read", "buffer_load", "scratch_load")) and \
                not name.startswith(("v_cmp", "v_nop", "v_readlane", "v_readfirstlane")):
            for op in operands[:2] if name.startswith(("v_swap", "v_permlane")) else operands[:1]:
                for r in _regs(op):
                    writer[r] = t
    return seen, wrong


def test_scan_catches_the_miscompiled_sequence():
    planted = "\n".join([
        "\tglobal_load_dwordx4 v[46:49], v0, s[40:41] nt",
        "\tv_and_b32_e32 v46, v46, v59",
        "\tv_cvt_pk_bf16_f32 v46, v35, s0",
        "\tv_cvt_pk_bf16_f32 v108, v35, v36",
        "\tv_cvt_scalef32_pk_bf16_fp8 v116, v46, 1.0",
        "\tv_cvt_scalef32_pk_bf16_fp8 v118, v47, 1.0 op_sel:[1,0,0]",
    ])
    seen, wrong = scan(planted)
    assert seen == 2 and wrong == ["[v_cvt_pk_bf16_f32 v46, v35, s0] -> [v_cvt_scalef32_pk_bf16_fp8 v116, v46, 1.0]"]
    assert scan(planted.replace("v_cvt_pk_bf16_f32 v46", "v_cvt_pk_bf16_f32 v45")) == (2, [])
    # a block's start forgets: the value may come from any of the blocks before it
    assert scan(planted.replace("\tv_cvt_scalef32_pk_bf16_fp8 v116", ".LBB0_1:\n\tv_cvt_scalef32_pk_bf16_fp8 v116")) \
        == (0, [])
    assert len(scan(planted.replace("v_cvt_pk_bf16_f32 v46, v35, s0", "v_permlane32_swap_b32_e32 v9, v46"))[1]) == 1


@pytest.mark.skipif(shutil.which(HIPCC) is None and not os.path.exists(HIPCC), reason="needs hipcc")
def test_built_kernels_widen_what_they_loaded(tmp_path):
    out = tmp_path / "k.s"
    cmd = [HIPCC, "-x", "hip", "--offload-arch=gfx950", "-O3", "-std=c++17", "-Xclang", "-target-feature", "-Xclang",
           "-packed-fp32-ops", "-I" + os.path.join(ROOT, "include"), "-I" + CSRC, "-S", "--cuda-device-only",
           os.path.join(CSRC, "kernels", "kv_cache.hip"), "-o", str(out)]
    r = subprocess.run(cmd, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    kernels = re.findall(r"^(_Z\S*kv_attn_kernel\S*):(.*?)\.end_amdhsa_kernel", out.read_text(), re.S | re.M)
    assert len(kernels) == 24
    for name, body in kernels:
        seen, wrong = scan(body)
        # V's codes, if not more: each of the 4 (head_dim 64) or 8 loads' dwords twice
        assert seen >= (32 if "Li1E" in name else 64) and not wrong, (name, seen, wrong[:3])
