"""Rows written by the store and by a decode step hold the same bits: signs of zeros, columns that are not rotated, with and without a bias."""
import pytest
import torch

import paged_model as pm
from conftest import announce
from paged_calls import bits

pytestmark = pytest.mark.gpu

F16, F32 = torch.float16, torch.float32


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("d,rotary_dim", [(64, 64), (128, 32), (80, 0), (256, 256)])
def test_store_and_decode_write_the_same_bits(capi, dev, dtype, bias, d, rotary_dim):
    ts = [1, 18, 700, 33]
    announce("paged bits", dtype, bias, d, rotary_dim)
    c = pm.Case(dtype, [1] * 4, [t - 1 for t in ts], 4, 2, d, 16, seed=91)
    g = torch.Generator(device=dev).manual_seed(92)
    kind = torch.randint(0, 6, c.qkv.shape, generator=g, device=dev)
    c.qkv[kind == 0] = 0.0
    c.qkv[kind == 1] = -0.0
    assert ((c.qkv == 0) & (bits(c.qkv) < 0)).any()
    c.bias[::3] = -0.0
    b = c.bias if bias else None
    kp, vp = c.kp.clone(), c.vp.clone()
    q = torch.empty(4, 4, d, dtype=dtype, device=dev)
    capi.paged_qkv_store(q, kp, vp, c.qkv, b, c.cu, c.hist, c.table, rotary_dim, 10000.0)
    kd, vd = c.kp.clone(), c.vp.clone()
    t = torch.tensor(ts, dtype=torch.int32, device=dev)
    capi.paged_decode_attn(c.qkv, b, kd, vd, torch.empty_like(q), c.table, t, max(ts), rotary_dim, 10000.0)
    torch.cuda.synchronize()
    assert torch.equal(bits(kd), bits(kp)) and torch.equal(bits(vd), bits(vp))
