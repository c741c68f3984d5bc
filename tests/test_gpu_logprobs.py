"""onellm_token_logprobs against its definition in 64 bits."""
import math

import pytest
import torch

from conftest import announce

pytestmark = pytest.mark.gpu

F16, F32 = torch.float16, torch.float32


def model(x, targets, K):
    """(logprob, entropy, top ids, top logprobs) in float64, ids exact; rows of nothing but -inf as the header defines them"""
    y = x.double()
    V = y.shape[1]
    # (against the row's maximum: next to the lowest value of fp32 the logarithm of the sum vanishes even in 64 bits)
    top = y.amax(dim=1, keepdim=True)
    empty = torch.isneginf(y).all(dim=1)
    lp = torch.where(empty[:, None], torch.full_like(y, -math.inf), (y - top) - torch.logsumexp(y - top, dim=1, keepdim=True))
    ok = (targets >= 0) & (targets < V)
    logprob = lp.gather(1, targets.clamp(0, V - 1).long()[:, None])[:, 0]
    logprob = torch.where(ok, logprob, torch.zeros_like(logprob))
    p = lp.exp()
    entropy = -(p * lp.masked_fill(p == 0, 0)).sum(dim=1)
    ids = torch.sort(y, dim=1, descending=True, stable=True)[1][:, :K]
    tops = lp.gather(1, ids)
    none = torch.isneginf(y.gather(1, ids))
    ids = ids.masked_fill(none, -1).int()
    if K > V:
        ids = torch.cat([ids, torch.full((len(ids), K - V), -1, dtype=torch.int32, device=ids.device)], dim=1)
        tops = torch.cat([tops, torch.full((len(tops), K - V), -math.inf, dtype=tops.dtype, device=tops.device)], dim=1)
    return logprob, entropy, ids, tops, (p * lp.masked_fill(p == 0, 0).abs()).sum(dim=1)


def run(capi, x, targets, K, workspace=None):
    N = x.shape[0]
    out = (torch.full((N,), 7.0, device=x.device), torch.full((N,), 7.0, device=x.device),
           torch.full((N, K), 7, dtype=torch.int32, device=x.device), torch.full((N, K), 7.0, device=x.device))
    capi.token_logprobs(x, targets, K, *out, workspace=workspace)
    torch.cuda.synchronize()
    return out


def check(capi, x, targets, K):
    announce("logprobs", x.dtype, tuple(x.shape), x.stride(), K)
    got = run(capi, x, targets, K)
    lp, ent, ids, tops, spread = model(x, targets, K)
    # a thread's sum of ceil(V / 256) terms and the joins (64): 2^-24 each; an exponent's rounding, 2^-24 of up to 150 that
    # still count; the logarithm and its scale: 2^-22 of it
    rel = (x.shape[1] / 256 + 64 + 150) * 2.0 ** -24 + 2.0 ** -22
    def close(a, b, tol):
        a = a.double()
        inf = torch.isinf(b)
        assert torch.equal(a[inf], b[inf])
        err = (a - b).abs()[~inf] / tol.expand_as(b)[~inf]
        assert not torch.isnan(err).any() and (err.numel() == 0 or err.max() <= 1), float(err.max())
    close(got[0], lp, rel + 2.0 ** -21 * lp.abs().clamp_max(1e30) + 2.0 ** -21)
    close(got[1], ent, 2 * rel * (1 + spread) + 2.0 ** -20)
    assert torch.equal(got[2], ids)
    close(got[3], tops, rel + 2.0 ** -21 * tops.abs().clamp_max(1e30) + 2.0 ** -21)
    return got


def logits(N, V, dtype, dev, seed, scale=3.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    return (torch.randn(N, V, generator=g, device=dev) * scale).to(dtype), torch.randint(0, V, (N,), generator=g, device=dev).int()


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("N,V,K", [
    (1, 1, 1), (3, 7, 5), (2, 33, 32), (5, 1000, 0), (4, 8191, 1), (1, 16384, 8), (2, 16385, 8), (1, 150001, 20), (7, 32000, 32), (600, 999, 3),
    (130, 40001, 5),
])
def test_shapes(capi, dev, dtype, N, V, K):
    x, t = logits(N, V, dtype, dev, seed=N + V)
    check(capi, x, t, K)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("offset", [0, 1, 3, 5])
def test_strides_and_alignments(capi, dev, dtype, offset):
    for N, V, ld in ((5, 20000, 20011), (5, 257, 300), (600, 777, 783)):
        big, t = logits(N, ld, dtype, dev, seed=offset)
        big[:, :offset] = 1000.0                             # neighbours that would win
        big[:, offset + V:] = 1000.0
        check(capi, big[:, offset:offset + V], t % V, 6)


@pytest.mark.parametrize("dtype", [F16, F32])
def test_ties_sorted_rows_and_signed_zeros(capi, dev, dtype):
    V = 20000
    x = torch.zeros(6, V, dtype=dtype, device=dev)
    x[0] = 1.5                                               # all equal
    x[1] = torch.linspace(-20, 20, V, device=dev).to(dtype)  # ascending, with ties after rounding
    x[2] = x[1].flip(0)
    x[3, 1::2] = -0.0                                        # zeros of both signs tie
    x[4] = (torch.arange(V, device=dev) % 7).to(dtype)
    x[5] = (torch.arange(V, device=dev) // 4000).to(dtype)
    t = torch.tensor([0, V - 1, 5, 17, 6, 19999], dtype=torch.int32, device=dev)
    for K in (1, 4, 32):
        check(capi, x, t, K)


@pytest.mark.parametrize("dtype", [F16, F32])
def test_banned_tokens_and_empty_rows(capi, dev, dtype):
    x, t = logits(5, 30000, dtype, dev, seed=9)
    x[0] = -math.inf                                         # nothing left
    x[1] = -math.inf
    x[1, 12345] = 2.0                                        # one token left
    x[2] = -math.inf
    x[2, 100:29000:3000] = torch.arange(10, device=dev).to(dtype)
    x[3, ::2] = -math.inf
    x[4] = torch.finfo(dtype).min                            # masked with the lowest value throughout: all equal
    t[1], t[2] = 12345, 101
    got = check(capi, x, t, 16)
    assert got[0][0] == -math.inf and got[1][0] == 0 and (got[2][0] == -1).all() and (got[3][0] == -math.inf).all()
    assert got[2][1].tolist() == [12345] + [-1] * 15 and got[0][1] == 0
    x[4, 7], x[4, 29999] = 3.0, 2.0                          # lowest values beside ordinary ones
    t[4] = 29999
    check(capi, x, t, 16)


@pytest.mark.parametrize("dtype", [F16, F32])
def test_large_magnitudes(capi, dev, dtype):
    x, t = logits(3, 5000, dtype, dev, seed=10, scale=2000.0)
    check(capi, x, t, 5)
    x, t = logits(3, 5000, F32, dev, seed=11, scale=1.0)
    x += torch.tensor([30000.0, -30000.0, 1e6], device=dev)[:, None]
    check(capi, x, t, 5)


def test_targets_outside_the_vocabulary(capi, dev):
    x, t = logits(5, 3001, F16, dev, seed=12)
    t = torch.tensor([-1, 3001, -100, 2 ** 31 - 1, 3000], dtype=torch.int32, device=dev)
    got = check(capi, x, t, 2)
    assert (got[0][:4] == 0).all() and got[0][4] < 0


@pytest.mark.parametrize("dtype", [F16, F32])
def test_nan_and_infinity(capi, dev, dtype):
    x, t = logits(3, 30000, dtype, dev, seed=13)
    clean = run(capi, x, t, 5)
    y = x.clone()
    y[0, 777] = math.nan
    y[1, 29998] = math.inf
    got = run(capi, y, t, 5)
    for a in got[:2]:
        assert torch.isnan(a[0]) and torch.isnan(a[1])
    assert got[2][1, 0] == 29998
    order = torch.sort(torch.where(torch.isnan(y[0]), -math.inf, y[0].double()), descending=True, stable=True)[1][:5].int()
    assert torch.equal(got[2][0], order)
    for a, b in zip(got, clean):
        assert torch.equal(a[2], b[2])


def test_outputs_left_out(capi, dev):
    x, t = logits(4, 40000, F16, dev, seed=14)
    full = check(capi, x, t, 5)
    lp = torch.empty(4, device=dev)
    capi.token_logprobs(x, t, 0, lp, None, None, None)
    assert torch.equal(lp, full[0])
    ent = torch.empty(4, device=dev)
    capi.token_logprobs(x, None, 0, None, ent, None, None)
    torch.testing.assert_close(ent, full[1], rtol=1e-6, atol=1e-6)
    ids, tops = torch.empty(4, 5, dtype=torch.int32, device=dev), torch.empty(4, 5, device=dev)
    capi.token_logprobs(x, None, 5, None, None, ids, tops)
    assert torch.equal(ids, full[2]) and torch.equal(tops, full[3])


def test_rows_beyond_four_gigabytes(capi, dev):
    N, V = 70000, 32000                                      # 4.5 GB in fp16
    x = torch.zeros(N, V, dtype=F16, device=dev)
    last, t = logits(3, V, F16, dev, seed=15)
    x[-3:] = last
    targets = torch.zeros(N, dtype=torch.int32, device=dev)
    targets[-3:] = t
    out = run(capi, x, targets, 4)
    ref = check(capi, last, t, 4)
    for a, b in zip(out, ref):
        torch.testing.assert_close(a[-3:], b, rtol=1e-5, atol=1e-5)
    assert (out[2][:-3] == torch.arange(4, device=dev, dtype=torch.int32)).all()


def test_streams_and_graphs(capi, dev):
    cases = [logits(3, 90000, F16, dev, seed=16 + i) for i in range(2)]
    want = [check(capi, x, t, 8) for x, t in cases]
    torch.cuda.synchronize()
    got = []
    for x, t in cases:
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            out = (torch.empty(3, device=dev), torch.empty(3, device=dev), torch.empty(3, 8, dtype=torch.int32, device=dev),
                   torch.empty(3, 8, device=dev))
            ws = torch.empty(capi.token_logprobs_workspace_bytes(3, 90000, 8), dtype=torch.uint8, device=dev)
            got.append((capi.token_logprobs(x, t, 8, *out, workspace=ws), ws))
    torch.cuda.synchronize()
    for (a, _), b in zip(got, want):
        assert all(torch.equal(p, q) for p, q in zip(a, b))
    x, t = cases[0]
    ws = torch.empty(capi.token_logprobs_workspace_bytes(3, 90000, 8), dtype=torch.uint8, device=dev)
    out = tuple(torch.empty_like(w) for w in want[0])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        capi.token_logprobs(x, t, 8, *out, workspace=ws)
    for _ in range(3):
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, want[0]))
        x.copy_(x.roll(1, dims=1))
        t.add_(1)
        t.remainder_(90000)
        want[0] = check(capi, x, t, 8)
