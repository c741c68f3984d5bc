"""Log-probabilities of logits far below the largest are rounded once, in fp16 calls too."""
import pytest
import torch

from conftest import announce

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("scale,offset", [(500.0, 0.0), (100.0, -1500.0), (3.0, 50.0)])
@pytest.mark.parametrize("N,V,K", [(2000, 1000, 8), (40, 20000, 32)])
def test_far_below_the_largest(capi, dev, dtype, scale, offset, N, V, K):
    announce("logprobs", dtype, N, V, scale, offset)
    g = torch.Generator(device=dev).manual_seed(95)
    x = (torch.randn(N, V, generator=g, device=dev) * scale + offset).round().clamp(-2048, 2048).to(dtype)      # whole numbers: x - max is exact
    t = torch.randint(0, V, (N,), generator=g, device=dev).int()
    lp, ids, tops = torch.empty(N, device=dev), torch.empty(N, K, dtype=torch.int32, device=dev), torch.empty(N, K, device=dev)
    capi.token_logprobs(x, t, K, lp, None, ids, tops)
    torch.cuda.synchronize()
    y = x.double()
    below = y - y.amax(dim=1, keepdim=True)
    logz = torch.logsumexp(below, dim=1, keepdim=True)
    want = below - logz
    # the last difference is rounded by half a step of its result.  log Z, up to log V: its terms' exponents, up to 30 where they count, are
    # off by 2^-23 of themselves, a thread's sum and the joins by (V / 256 + 64) 2^-24, the logarithm and its scale by 2^-22 of it
    half_step = 2.0 ** (torch.floor(torch.log2(want.abs().clamp_min(1e-9))) - 24)
    tol = half_step + 30 * 2.0 ** -23 + (V / 256 + 64) * 2.0 ** -24 + 2.0 ** -22 * logz.abs()
    for got, at in ((lp[:, None], t[:, None].long()), (tops, ids.long())):
        err = ((got.double() - want.gather(1, at)).abs() / tol.gather(1, at)).max().item()
        assert err <= 1.0, err
