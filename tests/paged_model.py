"""Serving from a paged key-value cache in 64 bits, straight from the definitions (torch float64, any device), with the
bounds its tests compare by."""
import math

import torch

EPS = {torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}        # half a step, relative
TINY = {torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}      # half a step of the subnormals


def rotate(x, pos, rotary_dim, base):
    """x [tokens, heads, D] float64, pos [tokens]: adjacent pairs (2i, 2i + 1), 2i < rotary_dim, by pos / base^(2i / rotary_dim)"""
    y = x.clone()
    D = x.shape[-1]
    for i in range(min(rotary_dim, D) // 2):
        ang = pos.double() / base ** (2 * i / rotary_dim)
        c, s = torch.cos(ang)[:, None], torch.sin(ang)[:, None]
        y[..., 2 * i] = x[..., 2 * i] * c - x[..., 2 * i + 1] * s
        y[..., 2 * i + 1] = x[..., 2 * i + 1] * c + x[..., 2 * i] * s
    return y


def page_of(table, b, row, num_pages, page_size):
    p = row // page_size
    if p >= table.shape[1]:
        return -1
    i = int(table[b, p])
    return i if 0 <= i < num_pages else -1


def rows_of(pages, layer, table, b, n):
    """(rows [n, Hkv, D] float64, has_page bool [n]) of sequence b; rows without a page are zeros"""
    _, num_pages, hkv, ps, d = pages.shape
    out = torch.zeros(n, hkv, d, dtype=torch.float64, device=pages.device)
    there = torch.zeros(n, dtype=torch.bool, device=pages.device)
    for p in range(-(-n // ps)):
        i = page_of(table, b, p * ps, num_pages, ps)
        if i < 0:
            continue
        m = min(ps, n - p * ps)
        out[p * ps:p * ps + m] = pages[layer, i, :, :m].transpose(0, 1).double()
        there[p * ps:p * ps + m] = True
    return out, there


def store(qkv, bias, k_pages, v_pages, cu, hist, table, layer, rotary_dim, base):
    """(q [tokens, Hq, D], {(page, row): (k, v)}, covered token list) in float64"""
    hkv, ps, num_pages = k_pages.shape[2], k_pages.shape[3], k_pages.shape[1]
    tokens, heads, d = qkv.shape
    hq = heads - 2 * hkv
    x = qkv.double()
    if bias is not None:
        x = x + bias.double().view(heads, d)
    q = torch.zeros(tokens, hq, d, dtype=torch.float64, device=qkv.device)
    written, covered = {}, []
    for b in range(len(hist)):
        lo, hi = int(cu[b]), int(cu[b + 1])
        if hi <= lo or int(hist[b]) < 0:
            continue
        pos = torch.arange(hi - lo, device=qkv.device) + int(hist[b])
        qk = rotate(x[lo:hi, :hq + hkv], pos, rotary_dim, base)
        q[lo:hi] = qk[:, :hq]
        covered += range(lo, hi)
        for i in range(hi - lo):
            row = int(hist[b]) + i
            page = page_of(table, b, row, num_pages, ps)
            if page >= 0:
                written[(page, row % ps)] = (qk[i, hq:], x[lo + i, hq + hkv:])
    return q, written, covered


def attend(q, rows_k, rows_v, there, first_limit):
    """q [n, Hq, D]; rows [t, Hkv, D]; row i of q sees rows <= first_limit + i that are `there`.  Returns (out, bound_mean,
    bound_score): out; sum_j w_j |v_j|, what errors of the weights scale; the largest sum_d |q_d k_jd| / sqrt(D) of a row"""
    n, hq, d = q.shape
    t, hkv, _ = rows_k.shape
    g = hq // hkv
    out = torch.zeros(n, hq, d, dtype=torch.float64, device=q.device)
    mean = torch.zeros_like(out)
    size = torch.zeros(n, hq, 1, dtype=torch.float64, device=q.device)
    seen = (torch.arange(t, device=q.device)[None, :] <= first_limit + torch.arange(n, device=q.device)[:, None]) & there[None, :]
    for h in range(hq):
        k, v = rows_k[:, h // g], rows_v[:, h // g]
        kt = k.t().contiguous()
        s = (q[:, h] @ kt / math.sqrt(d)).masked_fill(~seen, -math.inf)
        size[:, h, 0] = (q[:, h].abs() @ kt.abs() / math.sqrt(d)).masked_fill(~seen, 0).amax(dim=1)
        w = torch.exp(s - s.amax(dim=1, keepdim=True)).masked_fill(~seen, 0)
        z = w.sum(dim=1, keepdim=True)
        w = torch.where(z > 0, w / z.clamp_min(1e-300), torch.zeros_like(w))
        out[:, h] = w @ v
        mean[:, h] = w @ v.abs()
    return out, mean, size


def attention_tolerance(dtype, d, rows, out, mean, size, vmax):
    """How far an output may be off (see attend()).  A score is a sum of d products in fp32 plus a scaling: off by at
    most (d + 4) 2^-24 of the sum of its absolute products; exp2 and its argument add 2^-22 (1 + size); a weight's relative
    error is twice that (numerator and sum), plus `rows` 2^-24 for the sums over the rows, plus half a step of the type for
    a weight rounded to it, or half a subnormal step of it, each row.  The result is rounded once."""
    rel = 2 * ((d + 4) * 2.0 ** -24 * size + 2.0 ** -22 * (1 + size)) + (rows + 8) * 2.0 ** -24
    if dtype == torch.float16:
        rel = rel + EPS[dtype]
        extra = rows * TINY[dtype] * vmax
    else:
        extra = 0.0
    return EPS[dtype] * out.abs() + rel * mean + extra + TINY[dtype]


def prompt(q, k_pages, v_pages, cu, hist, table, layer):
    """(out, tolerance, covered tokens)"""
    tokens, hq, d = q.shape
    out = torch.zeros(tokens, hq, d, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    covered = []
    for b in range(len(hist)):
        lo, hi = int(cu[b]), int(cu[b + 1])
        if hi <= lo or int(hist[b]) < 0:
            continue
        covered += range(lo, hi)
        t = int(hist[b]) + hi - lo
        k, there = rows_of(k_pages, layer, table, b, t)
        v, _ = rows_of(v_pages, layer, table, b, t)
        o, mean, size = attend(q[lo:hi].double(), k, v, there, int(hist[b]))
        out[lo:hi] = o
        tol[lo:hi] = attention_tolerance(q.dtype, d, t, o, mean, size, float(v.abs().max()))
    return out, tol, covered


def decode(c, t_host, k_rows, v_rows, rotary_dim, base, bias=True):
    """One new token per sequence of case c (its qkv's first rows).  k_rows, v_rows [B, Hkv, D]: the new rows as the cache holds
    them.  Returns (out, tolerance) [B, Hq, D]; sequences of length 0 or less are left at zero."""
    B = len(t_host)
    x = c.qkv[:B].double()
    if bias:
        x = x + c.bias.double().view(c.hq + 2 * c.hkv, c.d)
    out = torch.zeros(B, c.hq, c.d, dtype=torch.float64, device=c.q.device)
    tol = torch.zeros_like(out)
    for b, t in enumerate(t_host):
        if t < 1:
            continue
        q = rotate(x[b:b + 1, :c.hq], torch.tensor([t - 1], device=c.q.device), rotary_dim, base)
        k, there = rows_of(c.kp, c.layer, c.table, b, t)
        v, _ = rows_of(c.vp, c.layer, c.table, b, t)
        k[t - 1], v[t - 1], there[t - 1] = k_rows[b].double(), v_rows[b].double(), True
        o, mean, size = attend(q, k, v, there, t - 1)
        # on top of attention's: q is rotated in fp32 (2^-21 of a pair) and enters as two halves (2^-22)
        out[b] = o[0]
        tol[b] = (attention_tolerance(c.dtype, c.d, t, o, mean, size, float(v.abs().max())) + 2.0 ** -18 * size * mean)[0]
    return out, tol


class Case:
    """Random inputs of a packed batch over shuffled pages; rows no sequence has hold NaN"""

    def __init__(self, dtype, lens, hist, hq, hkv, d, page_size=16, layers=1, layer=0, seed=0, device="cuda", extra_tokens=0, spare_pages=2):
        g = torch.Generator().manual_seed(seed)
        self.dtype, self.lens, self.hist_host, self.hq, self.hkv, self.d, self.ps = dtype, lens, hist, hq, hkv, d, page_size
        self.layer = layer
        B = len(lens)
        rows = [max(0, h) + n for n, h in zip(lens, hist)]
        need = [-(-r // page_size) for r in rows]
        self.max_pages = max(1, max(need)) + 1
        self.num_pages = max(1, sum(need)) + spare_pages
        ids = torch.randperm(self.num_pages, generator=g).to(torch.int32)
        table = torch.full((B, self.max_pages), -1, dtype=torch.int32)
        kp = torch.full((layers, self.num_pages, hkv, page_size, d), float("nan"))
        vp = kp.clone()
        at = 0
        for b, n in enumerate(need):
            table[b, :n] = ids[at:at + n]
            for p in range(n):
                m = min(page_size, rows[b] - p * page_size)
                page = int(ids[at + p])
                kp[layer, page, :, :m] = torch.randn(hkv, m, d, generator=g)
                vp[layer, page, :, :m] = torch.randn(hkv, m, d, generator=g)
            at += n
        self.tokens = sum(lens) + extra_tokens
        self.rows = rows
        self.table = table.to(device)
        self.kp, self.vp = kp.to(dtype).to(device), vp.to(dtype).to(device)
        self.cu = torch.tensor([sum(lens[:i]) for i in range(B + 1)], dtype=torch.int32, device=device)
        self.hist = torch.tensor(hist, dtype=torch.int32, device=device)
        self.q = torch.randn(self.tokens, hq, d, generator=g).to(dtype).to(device)
        self.qkv = torch.randn(self.tokens, hq + 2 * hkv, d, generator=g).to(dtype).to(device)
        self.bias = (torch.randn((hq + 2 * hkv) * d, generator=g) * 0.3).to(dtype).to(device)
        self.max_rows = max(1, max(rows))
