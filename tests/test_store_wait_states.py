"""A 16-byte store written in assembly is followed by the wait states that its data registers need before they may be written again (the
compiler keeps them for its own stores only)."""
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HIPCC = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"

SOURCE = """
#include "common.hpp"
using namespace onellm;
template <bool NT> __global__ void k(float* out, const stream_f32x4* in, int n) {
    for (int i = threadIdx.x; i < n; i += 64) store16_write_through<NT>(out + 4 * i, in[i] * 2.f);
}
template __global__ void k<true>(float*, const stream_f32x4*, int);
template __global__ void k<false>(float*, const stream_f32x4*, int);
"""


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="no compiler")
def test_write_through_stores_keep_their_data(tmp_path):
    src, asm = tmp_path / "k.hip", tmp_path / "k.s"
    src.write_text(SOURCE)
    subprocess.run([HIPCC, "-S", "--cuda-device-only", str(src), "-o", str(asm), "-O3", "-std=c++17", "--offload-arch=gfx950",
                    "-I" + os.path.join(ROOT, "include"), "-I" + os.path.join(ROOT, "onellm_amd", "csrc"),
                    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"], check=True, capture_output=True)
    lines = [x.strip() for x in asm.read_text().splitlines()]
    stores = [i for i, x in enumerate(lines) if re.match(r"global_store_dwordx4 .* sc1", x)]
    assert len(stores) >= 2
    for i in stores:
        m = re.match(r"s_nop (\d+)", lines[i + 1])
        assert m and int(m.group(1)) >= 1, lines[i:i + 3]
