"""NaNs and infinities in V.  A weight is above zero in the definition, however small, so a component whose column holds such values in rows
that the token sees is their sum: the infinity, or NaN.  Columns without one, and tokens that do not see one, are as without it."""
import math

import pytest
import torch

import paged_model as pm
from paged_calls import is_cut, prompt, row

pytestmark = pytest.mark.gpu

F16, F32 = torch.float16, torch.float32
INF, NAN = math.inf, math.nan
# column -> [(row, value)]: one infinity, both signs, a NaN, one of each
SPECIALS = {3: [(10, INF)], 5: [(200, -INF), (650, INF)], 9: [(100, NAN)], 12: [(300, -INF)], 17: [(0, INF), (63, INF), (64, INF), (640, INF)],
            21: [(20, -INF), (640, NAN)], 50: [(511, -INF), (512, -INF)]}


def expected(clean, seen):
    """clean [heads, D]: with the columns of SPECIALS that hold values in rows below `seen`"""
    out = clean.clone()
    for col, values in SPECIALS.items():
        s = [v for r, v in values if r < seen]
        if s:
            out[:, col] = sum(s)
    return out


def same(got, want):
    return torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(torch.nan_to_num(got, nan=1.0), torch.nan_to_num(want, nan=1.0))


# (with q times 60 the weights span hundreds of powers of two: most are zero in the type, or in fp32)
@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("d", [64, 128, 200])
@pytest.mark.parametrize("scale", [1.0, 60.0])
@pytest.mark.parametrize("cut", [False, True])
def test_prompt(capi, dev, dtype, d, scale, cut):
    c = pm.Case(dtype, [70, 3], [620, 900], 4, 2, d, 16, seed=81)
    c.q *= scale
    top = c.max_rows if cut else 1
    assert is_cut(capi, c, top) == cut
    clean = prompt(capi, c, top)
    assert torch.isfinite(clean).all()
    for col, values in SPECIALS.items():
        for r, v in values:
            row(c, c.vp, 0, r)[1, col] = v                    # kv head 1 of sequence 0
    got = prompt(capi, c, top)
    assert torch.equal(got[:, :2], clean[:, :2]) and torch.equal(got[70:], clean[70:])
    for i in range(70):
        assert same(got[i, 2:], expected(clean[i, 2:], 620 + i + 1)), i


@pytest.mark.parametrize("dtype", [F16, F32])
def test_prompt_at_every_step_boundary(capi, dev, dtype):
    """one infinity, in turn behind and in front of where plain steps, the diagonal and pieces begin"""
    c = pm.Case(dtype, [40], [400], 2, 1, 64, 16, seed=82)
    c.q *= 60.0
    for top in (1, 440):
        clean = prompt(capi, c, top)
        for r in (0, 31, 32, 63, 64, 127, 128, 191, 192, 255, 256, 383, 384, 399, 400, 415, 416, 438, 439):
            was = row(c, c.vp, 0, r)[0, 7].clone()
            row(c, c.vp, 0, r)[0, 7] = INF
            got = prompt(capi, c, top)
            want = clean.clone()
            want[max(0, r - 400):, :, 7] = INF
            assert torch.equal(got, want), (top, r)
            row(c, c.vp, 0, r)[0, 7] = was


@pytest.mark.parametrize("dtype", [F16, F32])
def test_prompt_scores_that_are_nan_win(capi, dev, dtype):
    c = pm.Case(dtype, [2], [700], 2, 1, 64, 16, seed=83)
    row(c, c.vp, 0, 10)[0, 3] = INF
    c.q[1, 0, 0] = NAN
    for top in (1, 702):
        got = prompt(capi, c, top)
        assert torch.isnan(got[1, 0]).all() and got[1, 1, 3] == INF and (got[0, :, 3] == INF).all()
