"""The paged operators together, as a server uses them: prompts into pages and attended in pieces, a prefix shared between two
sequences, decode steps, the answers' log-probabilities - against a model that keeps no cache and computes in 64 bits."""
import math

import pytest
import torch

import paged_model as pm
from conftest import announce

pytestmark = pytest.mark.gpu

LAYERS, HQ, HKV, D, PS, VOCAB, BASE = 2, 6, 2, 64, 16, 997, 10000.0
HID = HQ * D


class Model:
    def __init__(self, dtype, device):
        g = torch.Generator().manual_seed(51)
        r = lambda *s, scale: (torch.randn(*s, generator=g) * scale).to(dtype).to(device)
        self.emb = r(VOCAB, HID, scale=1.0)
        self.wqkv = [r(HID, (HQ + 2 * HKV) * D, scale=HID ** -0.5) for _ in range(LAYERS)]
        self.bqkv = [r((HQ + 2 * HKV) * D, scale=0.1) for _ in range(LAYERS)]
        self.wo = [r(HID, HID, scale=HID ** -0.5) for _ in range(LAYERS)]
        self.wout = r(HID, VOCAB, scale=2.0 * HID ** -0.5)


def reference_logits(m, ids):
    """logits of every position of one sequence, float64, no cache"""
    n = len(ids)
    x = m.emb.double()[ids]
    pos = torch.arange(n, device=x.device)
    for l in range(LAYERS):
        qkv = (x @ m.wqkv[l].double() + m.bqkv[l].double()).view(n, HQ + 2 * HKV, D)
        qk = pm.rotate(qkv[:, :HQ + HKV], pos, D, BASE)
        o, _, _ = pm.attend(qk[:, :HQ], qk[:, HQ:], qkv[:, HQ + HKV:], torch.ones(n, dtype=torch.bool, device=x.device), 0)
        x = x + o.reshape(n, HID) @ m.wo[l].double()
    return x @ m.wout.double()


class Server:
    def __init__(self, capi, m, tables, dtype, device):
        self.capi, self.m = capi, m
        num_pages = int(tables.max()) + 1
        self.kp, self.vp = (torch.full((LAYERS, num_pages, HKV, PS, D), float("nan"), dtype=dtype, device=device) for _ in range(2))
        self.tables = tables.to(device)
        self.dtype, self.dev = dtype, device
        self.ws = torch.zeros(capi.paged_decode_attn_workspace_bytes(8, HQ, HKV, D, 400), dtype=torch.uint8, device=device)

    def prefill(self, seqs, ids, hist):
        """ids: one tensor per sequence; logits [tokens, VOCAB] of the packed tokens"""
        cu = torch.tensor([0] + [len(i) for i in ids]).cumsum(0).int().to(self.dev)
        h = torch.tensor(hist, dtype=torch.int32, device=self.dev)
        table = self.tables[seqs].contiguous()
        x = self.m.emb[torch.cat(ids)]
        top = max(a + len(i) for a, i in zip(hist, ids))
        for l in range(LAYERS):
            qkv = (x @ self.m.wqkv[l]).view(len(x), HQ + 2 * HKV, D)
            self.capi.paged_qkv_store(qkv[:, :HQ], self.kp, self.vp, qkv, self.m.bqkv[l], cu, h, table, D, BASE, layer=l)
            o = torch.empty(len(x), HQ, D, dtype=self.dtype, device=self.dev)
            self.capi.paged_prompt_attn(qkv[:, :HQ], self.kp, self.vp, o, cu, h, table, top, layer=l)
            x = x + o.view(len(x), HID) @ self.m.wo[l]
        return x @ self.m.wout

    def step(self, ids, t):
        """one token per sequence; t int32: lengths with it"""
        x = self.m.emb[ids]
        for l in range(LAYERS):
            qkv = (x @ self.m.wqkv[l]).view(len(x), HQ + 2 * HKV, D)
            o = torch.empty(len(x), HQ, D, dtype=self.dtype, device=self.dev)
            self.capi.paged_decode_attn(qkv, self.m.bqkv[l], self.kp, self.vp, o, self.tables, t, 400, D, BASE, layer=l,
                                        flags=self.capi.ATTN_ZEROED_WORKSPACE, workspace=self.ws)
            x = x + o.view(len(x), HID) @ self.m.wo[l]
        return x @ self.m.wout

    def score(self, logits, targets, K):
        n = len(logits)
        out = (torch.empty(n, device=self.dev), torch.empty(n, device=self.dev),
               torch.empty(n, K, dtype=torch.int32, device=self.dev), torch.empty(n, K, device=self.dev))
        return self.capi.token_logprobs(logits, targets, K, *out)


# fp32: a dozen chained sums of up to 384 terms, each off by at most 384 * 2^-24 of its absolute terms (2.3e-5), which are about 4 of
# the logits' scale of 2: 1e-3 covers all of them lined up.  fp16: every activation is rounded (2^-11) some ten times on the way to a
# logit of scale 2, the sums over them grow that like a walk over 384 terms of a scale below 1: 0.05 covers five deviations.
@pytest.mark.parametrize("dtype,bound", [(torch.float32, 1e-3), (torch.float16, 0.05)])
def test_serving(capi, dev, dtype, bound):
    announce("paged serving", dtype)
    m = Model(dtype, dev)
    g = torch.Generator().manual_seed(52)
    prompts = [torch.randint(0, VOCAB, (n,), generator=g).to(dev) for n in (70, 1, 133)]
    # sequence 3 begins with the first 64 tokens of sequence 2 and shares their four pages
    prompts.append(torch.cat([prompts[2][:64], torch.randint(0, VOCAB, (21,), generator=g).to(dev)]))
    pages = torch.randperm(60, generator=g).int()
    tables = torch.full((4, 12), -1, dtype=torch.int32)
    for b in range(4):
        tables[b] = pages[12 * b:12 * b + 12]
    tables[3, :4] = tables[2, :4]
    server = Server(capi, m, tables, dtype, dev)

    # sequences 0 and 1 whole, 2 in two pieces, then 3 behind the shared rows
    a = server.prefill([0, 1, 2], [prompts[0], prompts[1], prompts[2][:50]], [0, 0, 0])
    b = server.prefill([2], [prompts[2][50:]], [50])
    c = server.prefill([3], [prompts[3][64:]], [64])
    got = [a[:70], a[70:71], torch.cat([a[71:], b]), torch.cat([torch.cat([a[71:], b])[:64], c])]
    for logits, ids in zip(got, prompts):
        want = reference_logits(m, ids)
        assert (logits.double() - want).abs().max() <= bound
        # the prompt's own tokens, scored
        lp, entropy, top, top_lp = server.score(logits[:-1], ids[1:].int(), 3) if len(ids) > 1 else server.score(logits, ids.int(), 3)
        ref = torch.log_softmax(want, dim=1)
        if len(ids) > 1:
            assert (lp.double() - ref[:-1].gather(1, ids[1:, None])[:, 0]).abs().max() <= 2 * bound + 1e-5
            assert (entropy.double() + (ref.exp() * ref).sum(dim=1)[:-1]).abs().max() <= 20 * bound
        assert (torch.sort(top_lp, dim=1, descending=True)[0] == top_lp).all()

    # five steps, all sequences at once, each answering with its likeliest token
    seqs = [list(p.tolist()) for p in prompts]
    logits = torch.stack([x[-1] for x in got])
    for _ in range(5):
        _, _, top, top_lp = server.score(logits.contiguous(), torch.zeros(4, dtype=torch.int32, device=dev), 2)
        chosen = top[:, 0].long()
        for b in range(4):
            seqs[b].append(int(chosen[b]))
        t = torch.tensor([len(s) for s in seqs], dtype=torch.int32, device=dev)
        logits = server.step(chosen, t)
        for b in range(4):
            want = reference_logits(m, torch.tensor(seqs[b], device=dev))[-1]
            assert (logits[b].double() - want).abs().max() <= bound
        lp, _, _, _ = server.score(logits, top[:, 0].contiguous(), 2)
        ref = torch.log_softmax(logits.double(), dim=1).gather(1, chosen[:, None])[:, 0]
        assert (lp.double() - ref).abs().max() <= 1e-4


def test_a_prompt_token_and_a_decode_step_agree(capi, dev):
    """the last token of a prompt computed as part of it and as a decode step behind it"""
    for dtype in (torch.float16, torch.float32):
        c = pm.Case(dtype, [90, 33], [0, 0], 8, 2, 128, 16, seed=53)
        q = torch.empty(123, 8, 128, dtype=dtype, device=dev)
        capi.paged_qkv_store(q, c.kp, c.vp, c.qkv, c.bias, c.cu, c.hist, c.table, 128, BASE)
        out = torch.empty_like(q)
        capi.paged_prompt_attn(q, c.kp, c.vp, out, c.cu, c.hist, c.table, 90)
        kp, vp = c.kp.clone(), c.vp.clone()
        last = torch.tensor([89, 122], device=dev)
        for b, row in ((0, 89), (1, 32)):
            page = int(c.table[b, row // 16])
            kp[0, page, :, row % 16] = vp[0, page, :, row % 16] = math.nan
        step = torch.empty(2, 8, 128, dtype=dtype, device=dev)
        capi.paged_decode_attn(c.qkv[last].contiguous(), c.bias, kp, vp, step, c.table, torch.tensor([90, 33], dtype=torch.int32, device=dev),
                               90, 128, BASE)
        # the rows themselves are the same bits; the outputs differ by a rounding of q (and of the weights) to fp16
        assert torch.equal(torch.nan_to_num(kp), torch.nan_to_num(c.kp)) and torch.equal(torch.nan_to_num(vp), torch.nan_to_num(c.vp))
        want, tol, _ = pm.prompt(q, c.kp, c.vp, c.cu, [0, 0], c.table, 0)
        err = (step.double() - want[last]).abs()
        # q rounded to the type moves a score by 2^-11 (2^-24) of its absolute products, at most 2^-11 * 12 for these rows
        slack = tol[last] + pm.EPS[dtype] * 24 * 4
        assert (err <= slack).all(), float((err / slack).max())
