"""Prompt attention whose rows are cut into pieces although its tiles alone would fill the chip once, against the definition in 64 bits: each rule that
decides on the cut, pieces without a row, rows without a page, and q written over."""
import pytest
import torch

import paged_model as pm
from test_gpu_paged import check_prompt

pytestmark = pytest.mark.gpu

F16, F32 = torch.float16, torch.float32


def pieces(capi, c, max_rows=None):
    """at least this many fit into the workspace of the call"""
    n = capi.paged_prompt_attn_workspace_bytes(len(c.lens), c.tokens, c.hq, c.hkv, c.d, c.max_rows if max_rows is None else max_rows)
    return n // (c.tokens * c.hq * (c.d + 2) * 4)


@pytest.mark.parametrize("dtype,lens,hist,hq,hkv,d", [
    (F16, [700, 300, 150], [1400, 0, 3000], 32, 32, 64),       # 352 workgroups, sequences of different lengths
    (F16, [2100], [0], 16, 2, 40),                             # 264, one sequence from its start
    (F32, [300, 200], [100, 900], 8, 8, 64),                   # 40
    (F32, [900, 130], [0, 700], 32, 8, 48),                    # 272
    (F32, [700], [400], 8, 8, 160),                            # 48, heads above 128
])
def test_cut(capi, dev, dtype, lens, hist, hq, hkv, d):
    c = pm.Case(dtype, lens, hist, hq, hkv, d, 32, seed=41)
    assert pieces(capi, c) >= 2
    got = check_prompt(capi, c)
    assert torch.equal(got, check_prompt(capi, c))
    # with a bound of one row nothing is cut
    assert pieces(capi, c, 1) == 0
    check_prompt(capi, c, max_rows=1)


@pytest.mark.parametrize("dtype", [F16, F32])
def test_cut_over_q_with_rows_that_have_no_page(capi, dev, dtype):
    c = pm.Case(dtype, [700, 300, 150, 1, 40], [1400, 0, 3000, 20, -1], 32, 32, 16, 16, extra_tokens=3, seed=42)
    assert pieces(capi, c) >= 2
    # whole pieces of a sequence, its last rows, and all of another's
    c.table[0, 40:110] = -1
    c.table[1, 10:] = c.num_pages
    c.table[3, :] = -1
    plain = check_prompt(capi, c)
    buf = c.q.clone()
    capi.paged_prompt_attn(buf, c.kp, c.vp, buf, c.cu, c.hist, c.table, c.max_rows)
    assert torch.equal(buf[:1151], plain[:1151]) and torch.equal(buf[1151:], c.q[1151:])
    assert (plain[1150] == 0).all()
