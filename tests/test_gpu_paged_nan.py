"""NaNs in queries and keys reach the outputs that see them, and no others, however the rows are cut into pieces."""
import math

import pytest
import torch

import paged_model as pm
from paged_calls import decode, decode_case, is_cut, prompt, row

pytestmark = pytest.mark.gpu

F16, F32 = torch.float16, torch.float32


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("cut", [False, True])
def test_prompt_nan_in_a_query(capi, dev, dtype, cut):
    c = pm.Case(dtype, [3, 40, 130], [900, 300, 20], 8, 2, 64, 16, seed=61)
    top = c.max_rows if cut else 1
    assert is_cut(capi, c, top) == cut
    clean = prompt(capi, c, top)
    assert torch.isfinite(clean).all()
    for token, head in ((1, 0), (20, 5), (100, 7), (172, 3)):
        c.q[token, head, (7 * head) % 64] = math.nan
    got = prompt(capi, c, top)
    hit = torch.zeros(173, 8, dtype=torch.bool, device=dev)
    for token, head in ((1, 0), (20, 5), (100, 7), (172, 3)):
        hit[token, head] = True
    assert torch.isnan(got[hit]).all()
    assert torch.equal(got[~hit], clean[~hit])


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("cut", [False, True])
def test_prompt_nan_in_the_only_key_of_a_piece(capi, dev, dtype, cut):
    """the last row of the sequence stands alone on its page, behind pages that are none"""
    c = pm.Case(dtype, [1, 2], [1008, 500], 4, 2, 64, 16, seed=62)
    c.table[0, 20:63] = -1
    top = c.max_rows if cut else 1
    assert is_cut(capi, c, top) == cut
    clean = prompt(capi, c, top)
    row(c, c.kp, 0, 1008)[1, 9] = math.nan
    got = prompt(capi, c, top)
    assert torch.isnan(got[0, 2:]).all()                      # the heads of kv head 1
    assert torch.equal(got[0, :2], clean[0, :2]) and torch.equal(got[1:], clean[1:])


@pytest.mark.parametrize("dtype", [F16, F32])
def test_decode_nan_in_queries_and_keys(capi, dev, dtype):
    c = decode_case(dtype, [5000, 40, 1], 8, 2, 64, 16, seed=63)
    clean = decode(capi, c)
    assert torch.isfinite(clean).all()
    c.qkv[0, 2, 5] = math.nan                                 # a query head
    c.qkv[2, 8 + 1, 5] = math.nan                             # the new key of kv head 1
    row(c, c.kp, 1, 38)[0, 3] = math.nan                      # a key of the cache
    got = decode(capi, c)
    hit = torch.zeros(3, 8, dtype=torch.bool, device=dev)
    hit[0, 2] = hit[2, 4] = hit[2, 5] = hit[2, 6] = hit[2, 7] = True
    hit[1, :4] = True
    assert torch.isnan(got[hit]).all()
    assert torch.equal(got[~hit], clean[~hit])
