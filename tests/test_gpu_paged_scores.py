"""Scores far from zero that are still inside fp32, as q and k entries of some thousands make them.  All scores here are exact in fp32
(products and sums of powers of two), so the weights, which depend on their differences, are those of the definition."""
import pytest
import torch

import paged_model as pm
from paged_calls import is_cut, prompt, row

pytestmark = pytest.mark.gpu

F16, F32 = torch.float16, torch.float32


def within(got, want, mean, dtype, rows, vmax):
    # scores exact; the scaling of a difference of up to 40 that still counts and exp2: 2 * 2^-22 * 40; the sums: 2^-24 a row; fp16: a weight,
    # times 2^7 at least, rounded by half a step or half a subnormal one; the result rounded once
    rel = 2 * 2.0 ** -22 * 40 + (rows + 8) * 2.0 ** -24 + (pm.EPS[dtype] if dtype == F16 else 0.0)
    tol = pm.EPS[dtype] * want.abs() + rel * mean + (rows * 2.0 ** -32 * vmax if dtype == F16 else 0.0) + pm.TINY[dtype]
    assert torch.isfinite(got).all(), "%d values are not finite" % int((~torch.isfinite(got)).sum())
    assert float(((got.double() - want).abs() / tol).max()) <= 1.0


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("cut", [False, True])
@pytest.mark.parametrize("a,b", [(2.0 ** 10, 2.0 ** 10), (2.0 ** 13, 2.0 ** 13), (2.0 ** 14, 2.0 ** 14), (2.0 ** 14, 2.0 ** 15),
                                 (-2.0 ** 14, 2.0 ** 15), (1.5 * 2.0 ** 13, 2.0 ** 15)])
@pytest.mark.parametrize("growing", [False, True])
def test_prompt(capi, dev, dtype, cut, a, b, growing):
    rows, tokens, d = 640, 40, 64
    c = pm.Case(dtype, [tokens], [rows - tokens], 1, 1, d, 16, seed=71)
    top = rows if cut else 1
    assert is_cut(capi, c, top) == cut
    # score a b + 64 m, m = 0, 1 or 2: up to 8 m in units of 1 / sqrt(d)
    if growing:
        m = (torch.arange(rows) >= 100).double() + (torch.arange(rows) >= 420).double()
    else:
        m = torch.randint(0, 3, (rows,), generator=torch.Generator().manual_seed(72)).double()
    c.q.zero_()
    c.q[:, :, 0], c.q[:, :, 1] = a, 8.0
    for r in range(rows):
        k = row(c, c.kp, 0, r)
        k.zero_()
        k[0, 0], k[0, 1] = b, 8.0 * float(m[r])
    v = torch.stack([row(c, c.vp, 0, r)[0] for r in range(rows)]).double().cpu()
    got = prompt(capi, c, top).cpu()
    want, mean = torch.zeros(tokens, 1, d, dtype=torch.float64), torch.zeros(tokens, 1, d, dtype=torch.float64)
    for i in range(tokens):
        n = rows - tokens + i + 1
        w = torch.softmax(8.0 * m[:n], dim=0)
        want[i, 0], mean[i, 0] = w @ v[:n], w @ v[:n].abs()
    within(got, want, mean, dtype, rows, float(v.abs().max()))


@pytest.mark.parametrize("dtype", [F16, F32])
def test_prompt_rows_of_one_wave_do_not_touch_each_other(capi, dev, dtype):
    """a token whose scores are far from zero, beside tokens whose are not: these come out bit for bit as without it"""
    c = pm.Case(dtype, [8], [300], 1, 1, 64, 16, seed=75)
    clean = prompt(capi, c)
    c.q[3] *= 2.0 ** 10
    got = prompt(capi, c)
    others = [0, 1, 2, 4, 5, 6, 7]
    assert torch.equal(got[others], clean[others])
