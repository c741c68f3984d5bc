"""Rows of one score far from zero among rows far below it: the mean of their values, in a decode step and in a prompt."""
import pytest
import torch

from paged_calls import decode, decode_case, prompt, row
from test_gpu_paged_scores import within

pytestmark = pytest.mark.gpu

F16, F32 = torch.float16, torch.float32


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("n,a,b", [(1, 2.0 ** 12, 2.0 ** 13), (1, 2.0 ** 13, 2.0 ** 13), (1, 2.0 ** 15, 2.0 ** 14), (8, 2.0 ** 15, 2.0 ** 15),
                                   (8, -2.0 ** 15, 2.0 ** 15), (3, 1.25 * 2.0 ** 13, 1.75 * 2.0 ** 13)])
def test_equal_scores(capi, dev, dtype, d, n, a, b):
    """Some rows of one score, the others - the new token of the decode step among them - far below it: the mean of those rows' values"""
    rows = 700
    c = decode_case(dtype, [rows], 2, 1, d, 16, seed=73)
    chosen = torch.randint(0, 5, (rows,), generator=torch.Generator().manual_seed(74)) == 0
    chosen[rows - 1] = False
    other = 0.0 if a > 0 else 2 * b
    c.qkv.zero_()
    c.qkv[:, :2, :n] = a
    c.qkv[:, 2, :n] = other if other < 65504 else 65504.0
    for r in range(rows):
        k = row(c, c.kp, 0, r)
        k.zero_()
        k[:, :n] = b if chosen[r] else (other if other < 65504 else 65504.0)
    for r in (0, rows - 2):
        row(c, c.kp, 0, r)[:, :n] = b
        chosen[r] = True
    c.qkv[:, 3] = 1.0
    row(c, c.vp, 0, rows - 1).fill_(1.0)
    v = torch.stack([row(c, c.vp, 0, r)[0] for r in range(rows)]).double().cpu()
    want, mean = v[chosen].mean(dim=0), v[chosen].abs().mean(dim=0)
    got = decode(capi, c).cpu()
    for h in range(2):
        within(got[0, h], want, mean, dtype, rows, float(v.abs().max()))
    # the same as one prompt token behind them
    c.q = c.qkv[:, :2].contiguous()
    c.cu = torch.tensor([0, 1], dtype=torch.int32, device=dev)
    c.hist = torch.tensor([rows - 1], dtype=torch.int32, device=dev)
    c.tokens = 1
    for top in (1, rows):
        got = prompt(capi, c, top).cpu()
        for h in range(2):
            within(got[0, h], want, mean, dtype, rows, float(v.abs().max()))
