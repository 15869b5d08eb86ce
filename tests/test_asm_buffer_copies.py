"""Hardware hazards of the buffer LDS copies (CPU only: hipcc -S).

load_lds16_buffer (csrc/kernels/elements.hpp) is inline asm, whose inside the
compiler does not pad.  A VMEM instruction may read an SGPR five wait states
after a VALU wrote it at the earliest, and an LDS copy may read M0 one after an
SALU wrote it, so each copy begins with s_nop 4.  The scan finds every copy in
the built kernel and the s_nop right before it, and shows that it catches one
without.
"""
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "lightining-core_amd", "csrc")
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")


def _bare_copies(text):
    """(copies, those without five wait states before them)."""
    ins = [t for t in (line.split(";")[0].strip() for line in text.split("\n")) if t and not t.startswith(".")]
    copies, bare = 0, []
    for i, t in enumerate(ins):
        if re.match(r"buffer_load_dwordx4\b.*\blds\b", t):
            copies += 1
            m = re.match(r"s_nop (\d+)$", ins[i - 1]) if i else None
            if m is None or int(m.group(1)) < 4:
                bare.append(ins[max(0, i - 3):i + 1])
    return copies, bare


def test_scan_catches_a_bare_copy():
    good = "v_readfirstlane_b32 s4, v1\ns_mov_b32 m0, s9\ns_nop 4\nbuffer_load_dwordx4 v2, s[4:7], 0 offen lds\n"
    assert _bare_copies(good) == (1, [])
    assert len(_bare_copies(good.replace("s_nop 4\n", ""))[1]) == 1
    assert len(_bare_copies(good.replace("s_nop 4", "s_nop 1"))[1]) == 1
    assert _bare_copies("buffer_load_dwordx4 v[2:5], v1, s[4:7], 0 offen\n") == (0, [])


@pytest.mark.skipif(shutil.which(HIPCC) is None and not os.path.exists(HIPCC), reason="needs hipcc")
def test_built_kernel_has_no_bare_copy(tmp_path):
    out = tmp_path / "k.s"
    cmd = [HIPCC, "-x", "hip", "--offload-arch=gfx950", "-O3", "-std=c++17", "-Xclang", "-target-feature", "-Xclang",
           "-packed-fp32-ops", "-I" + os.path.join(ROOT, "include"), "-I" + CSRC, "-S", "--cuda-device-only",
           os.path.join(CSRC, "kernels", "cross_attention.hip"), "-o", str(out)]
    r = subprocess.run(cmd, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    copies, bare = _bare_copies(out.read_text())
    assert copies > 100 and not bare, bare[:2]
