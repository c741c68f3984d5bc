"""Attention over paged caches of fp16 where the type's narrow range could show: many rows of tiny weight, queries far smaller or larger than the
keys."""
import math

import pytest
import torch

import paged_model as pm
from test_gpu_paged import check_decode, decode_case

pytestmark = pytest.mark.gpu

F16, F32 = torch.float16, torch.float32
ROWS, D, HKV, SEQS = 20000, 64, 8, 64


def one_row_that_stands_out(dev, dtype):
    """Row 0 has the score 9 * 16 / sqrt(64) = 18 and a value of 0, all others 0 and 1; the sequences share their pages but the last"""
    ps = 16
    pages = ROWS // ps
    kp = torch.zeros(1, pages + SEQS, HKV, ps, D, dtype=dtype, device=dev)
    vp = torch.ones_like(kp)
    kp[0, 0, :, 0, 0] = 9.0
    vp[0, 0, :, 0] = 0.0
    table = torch.arange(pages + 1, dtype=torch.int32, device=dev).repeat(SEQS, 1)
    table[:, pages] = torch.arange(pages, pages + SEQS, dtype=torch.int32, device=dev)
    return kp, vp, table


@pytest.mark.parametrize("dtype", [F16, F32])
def test_decode_many_rows_of_tiny_weight(capi, dev, dtype):
    kp, vp, table = one_row_that_stands_out(dev, dtype)
    qkv = torch.zeros(SEQS, 3 * HKV, D, dtype=dtype, device=dev)
    qkv[:, :HKV, 0] = 16.0
    qkv[:, 2 * HKV:] = 1.0
    out = torch.empty(SEQS, HKV, D, dtype=dtype, device=dev)
    t = torch.full((SEQS,), ROWS + 1, dtype=torch.int32, device=dev)
    capi.paged_decode_attn(qkv, None, kp, vp, out, table, t, ROWS + 1, 0, 10000.0)
    torch.cuda.synchronize()
    w = ROWS * math.exp(-18.0)                             # ROWS - 1 of the cache and the new one
    want = w / (1.0 + w)
    # the scores are exact; scaling and exp2 2^-22 (1 + 18 log2 e) twice, the sums ROWS 2^-24, a weight in two halves 2^-22
    rel = 2 * 2.0 ** -22 * 27 + (ROWS + 8) * 2.0 ** -24 + 2.0 ** -22
    assert (out.double() - want).abs().max().item() <= want * (rel + pm.EPS[dtype]) + pm.TINY[dtype]


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("tokens", [1, 130])
def test_prompt_many_rows_of_tiny_weight(capi, dev, dtype, tokens):
    """one token per sequence (rows in pieces), and many of one"""
    kp, vp, table = one_row_that_stands_out(dev, dtype)
    table[:, -1] = -1
    B = SEQS if tokens == 1 else 1
    q = torch.zeros(B * tokens, HKV, D, dtype=dtype, device=dev)
    q[:, :, 0] = 16.0
    out = torch.empty_like(q)
    cu = torch.arange(B + 1, dtype=torch.int32, device=dev) * tokens
    hist = torch.full((B,), ROWS - tokens, dtype=torch.int32, device=dev)
    capi.paged_prompt_attn(q, kp, vp, out, cu, hist, table[:B].contiguous(), ROWS)
    torch.cuda.synchronize()
    seen = torch.arange(ROWS - tokens + 1, ROWS + 1, dtype=torch.float64, device=dev)
    w = (seen - 1) * math.exp(-18.0)
    want = (w / (1.0 + w)).repeat(B)[:, None, None]
    # as above; fp16: a weight times 2^7 is rounded by half a subnormal step, 2^-25, at most, and there are ROWS of them
    rel = 2 * 2.0 ** -22 * 27 + (ROWS + 8) * 2.0 ** -24
    tol = want * (rel + pm.EPS[dtype]) + pm.TINY[dtype] + (ROWS * 2.0 ** -32 if dtype == F16 else 0.0)
    assert ((out.double() - want).abs() / tol).max().item() <= 1.0


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("q_scale,k_scale", [(2.0 ** -13, 2.0 ** 13), (2.0 ** 12, 2.0 ** -13)])
def test_decode_queries_far_from_the_keys(capi, dev, dtype, q_scale, k_scale):
    c = decode_case(dtype, [700, 33, 200], 6, 2, 64, 16, seed=51)
    c.qkv[:, :c.hq] = (c.qkv[:, :c.hq].float() * q_scale).to(dtype)
    c.qkv[:, c.hq:c.hq + c.hkv] = (c.qkv[:, c.hq:c.hq + c.hkv].float() * k_scale).to(dtype)
    c.kp.copy_((c.kp.float() * k_scale).to(dtype))
    # (no rotation: the bound on a stored k row is absolute, for rows of size 1)
    check_decode(capi, c, 0, bias=False)


def test_decode_queries_beyond_the_type(capi, dev):
    """the type's largest value plus a bias of that size, in heads of 8: 2 * 65504 log2(e) / sqrt(8) leaves fp16"""
    c = decode_case(F16, [300, 5], 4, 2, 8, 16, seed=52)
    c.qkv[:, :4] = 65504.0
    c.bias.zero_()
    c.bias.view(8, 8)[:4] = 65504.0
    c.qkv[:, 4:6] = (c.qkv[:, 4:6].float() * 2.0 ** -17).to(F16)
    c.kp.copy_((c.kp.float() * 2.0 ** -17).to(F16))
    check_decode(capi, c, 0)
