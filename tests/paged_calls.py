"""Calls of the paged attention that its tests of special values share."""
import torch

import paged_model as pm
from conftest import announce

MARK = 7.0                                     # what outputs hold before a call


def prompt(capi, c, max_rows=None, out=None, workspace=None):
    """attention of case c's packed tokens; tokens of no sequence keep MARK"""
    announce("paged prompt", c.dtype, c.lens, c.hist_host, c.hq, c.hkv, c.d, c.ps, max_rows)
    if out is None:
        out = torch.full((c.tokens, c.hq, c.d), MARK, dtype=c.dtype, device=c.q.device)
    capi.paged_prompt_attn(c.q, c.kp, c.vp, out, c.cu, c.hist, c.table, c.max_rows if max_rows is None else max_rows, layer=c.layer,
                           workspace=workspace)
    torch.cuda.synchronize()
    return out


def is_cut(capi, c, max_rows=None):
    """whether the call cuts its rows into pieces, in its own type: only then does it ask for a workspace"""
    try:
        prompt(capi, c, max_rows, workspace=torch.empty(0, dtype=torch.uint8, device=c.q.device))
    except capi.OnellmError:
        return True
    return False


def row(c, pages, b, r, layer=0):
    """[Hkv, D] view of row r of sequence b in k_pages or v_pages"""
    return pages[layer, int(c.table[b, r // c.ps]), :, r % c.ps]


def bits(t):
    return t.view(torch.int16 if t.dtype == torch.float16 else torch.int32)


def decode_case(dtype, ts, hq, hkv, d, ps, seed):
    """sequences of ts[b] rows with the new token, whose own row holds NaN in the cache yet"""
    c = pm.Case(dtype, ts, [0] * len(ts), hq, hkv, d, ps, seed=seed)
    c.ts = ts
    c.qkv = c.qkv[:len(ts)].contiguous()
    c.t_dev = torch.tensor(ts, dtype=torch.int32, device=c.q.device)
    for b, t in enumerate(ts):
        row(c, c.kp, b, t - 1).fill_(float("nan"))
        row(c, c.vp, b, t - 1).fill_(float("nan"))
    return c


def decode(capi, c, rotary_dim=0, bias=None, kp=None, vp=None):
    announce("paged decode", c.dtype, c.ts, c.hq, c.hkv, c.d, c.ps, rotary_dim)
    out = torch.full((len(c.ts), c.hq, c.d), MARK, dtype=c.dtype, device=c.q.device)
    capi.paged_decode_attn(c.qkv, bias, c.kp.clone() if kp is None else kp, c.vp.clone() if vp is None else vp, out, c.table, c.t_dev,
                           max(c.ts), rotary_dim, 10000.0, layer=c.layer)
    torch.cuda.synchronize()
    return out
