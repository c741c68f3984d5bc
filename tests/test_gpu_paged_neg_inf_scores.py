"""Keys whose score is -inf have no weight; a token that sees nothing else has no distribution, and its output is NaN, not the zeros of a
token that sees no row."""
import math

import pytest
import torch

import paged_model as pm
from paged_calls import decode, decode_case, is_cut, prompt, row

pytestmark = pytest.mark.gpu

F16, F32 = torch.float16, torch.float32


@pytest.mark.parametrize("dtype", [F16, F32])
def test_prompt_first_key(capi, dev, dtype):
    c = pm.Case(dtype, [40, 1], [0, 30], 4, 2, 64, 16, seed=64)
    c.q[:, :, 5] = 1.0
    row(c, c.kp, 0, 0)[0, 5] = -60000.0                       # scores of -7500 and below: no weight beside any other
    clean = prompt(capi, c)
    assert torch.isfinite(clean).all()
    row(c, c.kp, 0, 0)[0, 5] = -math.inf
    got = prompt(capi, c)
    assert torch.isnan(got[0, :2]).all()
    assert torch.equal(got[0, 2:], clean[0, 2:]) and torch.equal(got[1:], clean[1:])


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("cut", [False, True])
def test_prompt_long_stretches(capi, dev, dtype, cut):
    c = pm.Case(dtype, [1, 2, 1], [1008, 900, 700], 4, 2, 64, 16, seed=65)
    c.q[:, :, 5] = 1.0
    top = c.max_rows if cut else 1
    assert is_cut(capi, c, top) == cut
    for r in range(701):                                      # all that sequence 2 sees; whole pieces of sequence 1
        row(c, c.kp, 2, r)[:, 5] = -60000.0
    for r in range(100, 800):
        row(c, c.kp, 1, r)[:, 5] = -60000.0
    clean = prompt(capi, c, top)
    assert torch.isfinite(clean).all()
    for r in range(701):
        row(c, c.kp, 2, r)[:, 5] = -math.inf
    for r in range(100, 800):
        row(c, c.kp, 1, r)[:, 5] = -math.inf
    got = prompt(capi, c, top)
    assert torch.isnan(got[3]).all()
    assert torch.equal(got[:3], clean[:3])
    c.table[2] = -1                                           # now it sees no row
    assert (prompt(capi, c, top)[3] == 0).all()


@pytest.mark.parametrize("dtype", [F16, F32])
def test_decode(capi, dev, dtype):
    c = decode_case(dtype, [900, 300, 1], 4, 2, 64, 16, seed=66)
    c.qkv[:, :4, 5] = 1.0
    for r in range(299):
        row(c, c.kp, 1, r)[:, 5] = -60000.0
    clean = decode(capi, c)
    assert torch.isfinite(clean).all()
    for r in range(299):
        row(c, c.kp, 1, r)[:, 5] = -math.inf
    got = decode(capi, c)
    assert torch.equal(got, clean)
    c.qkv[1:, 4:6, 5] = -math.inf                             # the new token's key too
    got = decode(capi, c)
    assert torch.isnan(got[1:]).all() and torch.equal(got[0], clean[0])


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("cut", [False, True])
def test_prompt_behind_rows_that_have_no_page(capi, dev, dtype, cut):
    """The first tokens see only pages that are none, the next ones one page of scores of -inf, the last ones another key as well"""
    c = pm.Case(dtype, [100], [2200], 2, 1, 64, 16, seed=67)
    c.q[:, :, 5] = 1.0
    c.table[0, :140] = -1                                     # rows 0 .. 2239: tokens 0 .. 39 see nothing
    for r in range(2240, 2256):
        row(c, c.kp, 0, r)[0, 5] = -math.inf
    top = c.max_rows if cut else 1
    assert is_cut(capi, c, top) == cut
    got = prompt(capi, c, top)
    assert (got[:40] == 0).all()
    assert torch.isnan(got[40:56]).all()
    assert torch.isfinite(got[56:]).all()
    c.table[0, 140] = -1
    clean = prompt(capi, c, top)
    assert (clean[:56] == 0).all() and torch.equal(clean[56:], got[56:])
