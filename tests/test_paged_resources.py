"""Register and occupancy budgets of the paged-cache kernels, from the remarks hipcc leaves during the build (no GPU needed)."""
import os
import re

import pytest

from onellm_amd import build

SOURCES = ["paged_store.hip", "paged_prompt.hip", "paged_decode.hip", "logprobs.hip"]


@pytest.fixture(scope="module")
def resources():
    if not all(os.path.exists(build.resources_file(s)) for s in SOURCES):
        build.build(force=True)
    return {s: build.kernel_resources(s) for s in SOURCES}


def test_no_kernel_spills_but_the_widest_fp32_prompt(resources):
    for src, res in resources.items():
        assert res, src
        for name, r in res.items():
            limit = 256 if "paged_prompt_attn_kernelIfLi256E" in name else 0     # 128 rows x 256 fp32 columns of Q and of O per workgroup
            assert r["scratch"] <= limit, "%s: %s uses %d bytes of scratch per lane" % (src, name, r["scratch"])


@pytest.mark.parametrize("src,pattern,occupancy", [
    ("paged_prompt.hip", r"prompt_attn_kernelI(6__half|f)Li(64|128)E", 2),
    ("paged_decode.hip", r"decode_attn_kernelI(6__half|f)Li(64|128)E", 2),
    ("paged_store.hip", r"qkv_store_kernel", 4),
    ("logprobs.hip", r"logprobs_kernel", 5),
    ("logprobs.hip", r"logprobs_join_kernel", 8),
])
def test_occupancy(resources, src, pattern, occupancy):
    hits = {k: v for k, v in resources[src].items() if re.search(pattern, k)}
    assert hits
    for name, r in hits.items():
        assert r["occupancy"] >= occupancy, "%s: %d waves per SIMD (VGPRs %d, AGPRs %d)" % (name, r["occupancy"], r["vgprs"], r["agprs"])
