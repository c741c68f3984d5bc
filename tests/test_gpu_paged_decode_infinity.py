"""NaNs and infinities in V, decode steps: the rule of test_gpu_paged_infinity.py."""
import math

import pytest
import torch

from paged_calls import bits, decode, decode_case, row
from test_gpu_paged_infinity import SPECIALS, expected, same

pytestmark = pytest.mark.gpu

F16, F32 = torch.float16, torch.float32
INF, NAN = math.inf, math.nan


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("d", [64, 128, 200])
@pytest.mark.parametrize("scale", [1.0, 60.0])
def test_decode(capi, dev, dtype, d, scale):
    c = decode_case(dtype, [701, 5000, 40, 1], 20, 1, d, 16, seed=84)
    c.qkv[:, :20] *= scale
    clean = decode(capi, c)
    assert torch.isfinite(clean).all()
    for col, values in SPECIALS.items():
        for r, v in values:
            for b in range(2):
                row(c, c.vp, b, r)[0, col] = v
    got = decode(capi, c)
    for b in range(2):
        assert same(got[b], expected(clean[b], 701)), b
    assert torch.equal(got[2:], clean[2:])
    # the new token's own value
    c.qkv[:, 21, 33] = -INF
    c.qkv[:, 21, 3] = NAN
    got = decode(capi, c)
    for b in range(4):
        want = expected(clean[b], 701) if b < 2 else clean[b].clone()
        want[:, 33], want[:, 3] = -INF, NAN
        assert same(got[b], want), b


@pytest.mark.parametrize("dtype", [F16, F32])
def test_decode_scores_that_are_nan_win(capi, dev, dtype):
    c = decode_case(dtype, [700, 6000], 2, 1, 64, 16, seed=85)
    for b in range(2):
        row(c, c.vp, b, 10)[0, 3] = INF
    c.qkv[:, 0, 0] = NAN
    got = decode(capi, c)
    assert torch.isnan(got[:, 0]).all() and (got[:, 1, 3] == INF).all()


@pytest.mark.parametrize("dtype", [F16, F32])
def test_rows_without_a_page_while_the_first_page_is_not_finite(capi, dev, dtype):
    c = decode_case(dtype, [700, 33, 18, 2, 100], 4, 2, 64, 16, seed=86)
    spare = sorted(set(range(c.num_pages)) - set(c.table.flatten().tolist()))[0]
    for p in (c.kp, c.vp):                                    # page 0 becomes one that no sequence has
        p[:, spare] = p[:, 0]
        p[:, 0] = NAN
    c.table[c.table == 0] = spare
    c.table[0, 5:30] = -1
    c.table[4, 1] = c.num_pages
    got = decode(capi, c)
    assert torch.isfinite(got).all()
    for p in (c.kp, c.vp):
        p[:, 0] = 0.0
    assert torch.equal(bits(decode(capi, c)), bits(got))
