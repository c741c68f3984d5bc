"""Prompt attention cut into pieces, each type by its own rule: heads of several column rounds, pieces without a row, q written over."""
import pytest
import torch

import paged_model as pm
from paged_calls import is_cut
from test_gpu_paged import check_prompt

pytestmark = pytest.mark.gpu

F16, F32 = torch.float16, torch.float32


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("lens,hist,hq,hkv,d", [
    ([3, 1, 8], [5000, 7000, 40], 8, 2, 128),
    ([64], [800], 8, 8, 64),
    ([20, 5], [1500, 3000], 6, 2, 256),                        # heads above 128: a wave's rows leave in two rounds of columns
    ([130], [900], 4, 1, 160),
    ([9], [2100], 2, 2, 24),
])
def test_cut(capi, dev, dtype, lens, hist, hq, hkv, d):
    c = pm.Case(dtype, lens, hist, hq, hkv, d, 32, seed=101)
    assert is_cut(capi, c) and not is_cut(capi, c, 1)
    got = check_prompt(capi, c)
    assert torch.equal(got, check_prompt(capi, c))


@pytest.mark.parametrize("lens,hist,hq,hkv,d", [
    ([700, 300, 150], [1400, 0, 3000], 32, 32, 64),            # 257 to 384 workgroups, sequences of different lengths
    ([2100], [0], 16, 2, 40),                                  # one sequence from its start
])
def test_cut_fp16_for_evenness(capi, dev, lens, hist, hq, hkv, d):
    c = pm.Case(F16, lens, hist, hq, hkv, d, 32, seed=102)
    assert is_cut(capi, c)
    check_prompt(capi, c)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("d", [16, 136])
def test_cut_over_q_with_rows_that_have_no_page(capi, dev, dtype, d):
    c = pm.Case(dtype, [700, 300, 150, 1, 40], [1400, 0, 3000, 20, -1], 24, 24, d, 16, extra_tokens=3, seed=103)
    assert is_cut(capi, c)
    # whole pieces of a sequence, its last rows, and all of another's
    c.table[0, 40:110] = -1
    c.table[1, 10:] = c.num_pages
    c.table[3, :] = -1
    plain = check_prompt(capi, c)
    buf = c.q.clone()
    capi.paged_prompt_attn(buf, c.kp, c.vp, buf, c.cu, c.hist, c.table, c.max_rows)
    torch.cuda.synchronize()
    assert torch.equal(buf[:1151], plain[:1151]) and torch.equal(buf[1151:], c.q[1151:])
    assert (plain[1150] == 0).all()


@pytest.mark.parametrize("dtype", [F16, F32])
def test_few_tokens_behind_many_rows_without_pages(capi, dev, dtype):
    c = pm.Case(dtype, [5, 2, 1], [6000, 3000, 100], 8, 2, 128, 16, seed=104)
    assert is_cut(capi, c)
    c.table[0, 100:340] = -1                                   # most of its pieces
    c.table[1, :] = -1
    c.table[1, 150:] = c.num_pages
    out = check_prompt(capi, c)
    assert (out[5:7] == 0).all()
