"""Measured cases of serving from a paged key-value cache: rows into pages, a packed prompt's attention over them, one new
token's attention over them, and the log-probabilities of an answer's tokens.

`own` chooses between the operators' plain form (elementary torch operations in 32 bits, angles in 64) and the calls a
program makes of this library.  Shapes follow bench.py: 32 x 128 heads over 32 or 8 kv heads, contexts of up to 8192 rows,
4 x 2048 prompt tokens, 32000-token vocabularies.
"""
import math

import torch

own = False

DEV = "cuda:0"
TYPES = {"fp16": torch.float16, "fp32": torch.float32}
ROPE_BASE = 10000.0


# ---------------------------------------------------------------- cases

def listed():
    return [
        # a few tokens of each running sequence go into the cache between two steps (a drafted continuation)
        dict(name="store_few_tokens", op="store", dtype="fp16", hq=32, hkv=8, d=128, page=16, lens="4*8", hist="200..1800"),
        # the prefill line of bench.py: 4 prompts of 2048 tokens, 96 heads in all
        dict(name="store_prompts", op="store", dtype="fp16", hq=32, hkv=32, d=128, page=64, lens="2048*4", hist="0..0"),
        # short prompts of a chat service's first turn, one of them a single token
        dict(name="prompt_short", op="prompt", dtype="fp16", hq=32, hkv=8, d=128, page=16, lens="1,37,100,64", hist="0..0"),
        # a packed batch of uneven prompts
        dict(name="prompt_packed", op="prompt", dtype="fp16", hq=32, hkv=8, d=128, page=16, lens="1,1500,77,2048,513,1024,300,7",
             hist="0..0"),
        # one long document
        dict(name="prompt_long", op="prompt", dtype="fp16", hq=32, hkv=8, d=128, page=64, lens="8192", hist="0..0"),
        # the next piece of two long documents, and a few drafted tokens behind a third
        dict(name="prompt_chunk", op="prompt", dtype="fp16", hq=32, hkv=8, d=128, page=16, lens="200,256,5", hist="15000..20000"),
        # full-precision caches with small heads
        dict(name="prompt_fp32", op="prompt", dtype="fp32", hq=16, hkv=2, d=64, page=32, lens="700,1,333,1024", hist="0..300"),
        # one conversation alone: latency
        dict(name="decode_single", op="decode", dtype="fp16", hq=32, hkv=8, d=128, page=16, t="900..900", batch=1),
        # the headline step of bench.py on pages: 16 sequences of 4096 rows, one kv head per query head
        dict(name="decode_full_heads", op="decode", dtype="fp16", hq=32, hkv=32, d=128, page=16, t="4096..4096", batch=16),
        # a grouped-query batch of uneven lengths
        dict(name="decode_uneven", op="decode", dtype="fp16", hq=32, hkv=8, d=128, page=32, t="1024..8192", batch=32),
        # the tokens of one decode step, with the alternatives a service reports
        dict(name="logprobs_step", op="logprobs", dtype="fp32", rows=16, vocab=32000, k=5),
        # scoring a prompt's tokens
        dict(name="logprobs_prompt", op="logprobs", dtype="fp16", rows=4096, vocab=32000, k=8),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.999)))))))


def draw(rng):
    op = rng.choice(["store", "prompt", "prompt", "decode", "decode", "logprobs"])
    if op == "logprobs":
        dtype = rng.choice(["fp16", "fp32"])
        vocab = _log_int(rng, 1000, 150000)
        rows = _log_int(rng, 1, max(1, min(4096, 60_000_000 // vocab)))
        return dict(op=op, dtype=dtype, rows=rows, vocab=vocab, k=rng.choice([0, 1, 2, 5, 8, 20]))
    hkv = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 3, 4, 7, 8])
    d = rng.choice([64, 64, 80, 96, 128, 128, 128, 256])
    case = dict(op=op, dtype=rng.choice(["fp16", "fp16", "fp32"]), hq=hkv * group, hkv=hkv, d=d, page=rng.choice([16, 32, 64, 256]))
    hq = case["hq"]
    if op == "decode":
        batch = _log_int(rng, 1, 48)
        top = _log_int(rng, 16, max(17, min(16384, 130_000_000 // (batch * hkv * d), 500_000_000 // (batch * hq * d))))
        low = max(1, int(top * rng.choice([0.1, 0.5, 1.0])))
        return dict(case, t=f"{low}..{top}", batch=batch)
    if op == "store":
        total, hist = _log_int(rng, 1, min(8192, 100_000_000 // ((hq + 2 * hkv) * d))), rng.choice([0, 0, 100, 5000])
    else:
        pairs = 1_000_000_000_000 // (4 * d * hq) // (2 if case["dtype"] == "fp16" else 40)
        total = _log_int(rng, 1, min(8192, math.isqrt(pairs)))
        hist = _log_int(rng, 1, max(1, min(20000, pairs // total, 60_000_000 // (hkv * d * 8)))) if rng.random() < 0.5 else 0
    n = min(total, rng.choice([1, 1, 2, 3, 5, 8]))
    cuts = sorted(rng.sample(range(1, total), n - 1)) if n > 1 else []
    lens = [b - a for a, b in zip([0] + cuts, cuts + [total])]
    return dict(case, lens=",".join(map(str, lens)), hist=f"{hist // 2}..{hist}")


def _lens(text):
    if "*" in text:
        length, count = text.split("*")
        return [int(length)] * int(count)
    return [int(x) for x in text.split(",")]


def _span(text, n):
    """n lengths spread evenly over the span, in an order that is not sorted"""
    lo, hi = (int(x) for x in text.split(".."))
    vals = [lo + (hi - lo) * i // max(1, n - 1) for i in range(n)] if n > 1 else [hi]
    step = 7
    while math.gcd(step, n) != 1:
        step += 1
    return [vals[(i * step) % n] for i in range(n)]


def _geometry(case):
    """(tokens per sequence, rows before them, rows behind them)"""
    if case["op"] == "decode":
        t = _span(case["t"], case["batch"])
        return [1] * len(t), [x - 1 for x in t], t
    lens = _lens(case["lens"])
    hist = _span(case["hist"], len(lens))
    return lens, hist, [a + b for a, b in zip(lens, hist)]


# ---------------------------------------------------------------- inputs

def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    dt = TYPES[case["dtype"]]
    if case["op"] == "logprobs":
        n, v, k = case["rows"], case["vocab"], case["k"]
        # logits of a trained model: a broad bulk, a few tokens far above it, some tokens banned
        x = torch.randn(n, v, generator=g, device=DEV) * 2.0
        hot = torch.randint(0, v, (n, 12), generator=g, device=DEV)
        x.scatter_add_(1, hot, torch.rand(n, 12, generator=g, device=DEV) * 12.0)
        x[:, torch.randint(0, v, (5,), generator=g, device=DEV)] = -math.inf
        targets = hot[:, 0].to(torch.int32).contiguous()
        st = dict(case=case, x=x.to(dt), targets=targets)
        if own:
            from onellm_amd import capi
            st.update(logprob=torch.empty(n, device=DEV), entropy=torch.empty(n, device=DEV),
                      top_ids=torch.empty(n, k, dtype=torch.int32, device=DEV), top_logprobs=torch.empty(n, k, device=DEV),
                      ws=torch.zeros(capi.token_logprobs_workspace_bytes(n, v, k), dtype=torch.uint8, device=DEV))
        return st
    hq, hkv, d, ps = case["hq"], case["hkv"], case["d"], case["page"]
    new, hist, rows = _geometry(case)
    batch, tokens = len(new), sum(new)
    per_seq = [-(-r // ps) for r in rows]
    max_pages = max(per_seq) + 1
    num_pages = sum(per_seq) + 3
    ids = torch.randperm(num_pages, generator=g, device=DEV).to(torch.int32)
    table = torch.full((batch, max_pages), -1, dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(per_seq):
        table[b, :n] = ids[at:at + n]
        at += n
    kp = torch.randn(1, num_pages, hkv, ps, d, generator=g, device=DEV).to(dt)
    vp = torch.randn(1, num_pages, hkv, ps, d, generator=g, device=DEV).to(dt)
    cu = torch.tensor([sum(new[:i]) for i in range(batch + 1)], dtype=torch.int32, device=DEV)
    st = dict(case=case, kp=kp, vp=vp, table=table, cu=cu, hist=torch.tensor(hist, dtype=torch.int32, device=DEV),
              new=new, hist_host=hist, rows=rows, tokens=tokens, max_rows=max(rows))
    if case["op"] == "prompt":
        st["q"] = torch.randn(tokens, hq, d, generator=g, device=DEV).to(dt)
    else:
        st["qkv"] = torch.randn(tokens, hq + 2 * hkv, d, generator=g, device=DEV).to(dt)
        st["bias"] = (torch.randn((hq + 2 * hkv) * d, generator=g, device=DEV) * 0.1).to(dt)
        st["t"] = torch.tensor(rows, dtype=torch.int32, device=DEV)
    if own:
        from onellm_amd import capi
        st["out"] = torch.empty(tokens, hq, d, dtype=dt, device=DEV)
        if case["op"] == "prompt":
            nbytes = capi.paged_prompt_attn_workspace_bytes(batch, tokens, hq, hkv, d, max(rows))
            st["ws"] = torch.zeros(nbytes, dtype=torch.uint8, device=DEV)
        elif case["op"] == "decode":
            nbytes = capi.paged_decode_attn_workspace_bytes(batch, hq, hkv, d, max(rows))
            st["ws"] = torch.zeros(nbytes, dtype=torch.uint8, device=DEV)
    return st


# ---------------------------------------------------------------- one pass

def run(st):
    case = st["case"]
    if own:
        return _run_own(st, case["op"])
    return {"store": _plain_store, "prompt": _plain_prompt, "decode": _plain_decode, "logprobs": _plain_logprobs}[case["op"]](st)


def _run_own(st, op):
    from onellm_amd import capi
    if op == "store":
        capi.paged_qkv_store(st["out"], st["kp"], st["vp"], st["qkv"], st["bias"], st["cu"], st["hist"], st["table"],
                             st["case"]["d"], ROPE_BASE)
        return st["out"], st["kp"], st["vp"]
    if op == "prompt":
        capi.paged_prompt_attn(st["q"], st["kp"], st["vp"], st["out"], st["cu"], st["hist"], st["table"], st["max_rows"],
                               workspace=st["ws"])
        return st["out"]
    if op == "decode":
        capi.paged_decode_attn(st["qkv"], st["bias"], st["kp"], st["vp"], st["out"], st["table"], st["t"], st["max_rows"],
                               st["case"]["d"], ROPE_BASE, flags=capi.ATTN_ZEROED_WORKSPACE, workspace=st["ws"])
        return st["out"], st["kp"], st["vp"]
    capi.token_logprobs(st["x"], st["targets"], st["case"]["k"], st["logprob"], st["entropy"], st["top_ids"], st["top_logprobs"],
                        workspace=st["ws"])
    return st["logprob"], st["entropy"], st["top_ids"], st["top_logprobs"]


def _rotate(x, pos, dim):
    """x [tokens, heads, d] in 32 bits, pos int64 [tokens]; angles in 64 bits, adjacent pairs"""
    freq = ROPE_BASE ** (-torch.arange(0, dim, 2, dtype=torch.float64, device=DEV) / dim)
    ang = pos.to(torch.float64)[:, None] * freq[None, :]
    c, s = torch.cos(ang).float()[:, None, :], torch.sin(ang).float()[:, None, :]
    x0, x1 = x[..., 0::2], x[..., 1::2]
    return torch.stack((x0 * c - x1 * s, x1 * c + x0 * s), dim=-1).flatten(-2)


def _split_rotated(st):
    """(q, k, v) of the new tokens in 32 bits, and where their rows go: (page, row inside the page)"""
    case = st["case"]
    hq, hkv, d, ps = case["hq"], case["hkv"], case["d"], case["page"]
    x = st["qkv"].float() + st["bias"].float().view(1, hq + 2 * hkv, d)
    cu, hist = st["cu"].long(), st["hist"].long()
    token = torch.arange(st["tokens"], device=DEV)
    seq = torch.searchsorted(cu, token, right=True) - 1
    pos = hist[seq] + token - cu[seq]
    qk = _rotate(x[:, :hq + hkv], pos, d)
    page = st["table"].long()[seq, pos // ps]
    return qk[:, :hq], qk[:, hq:], x[:, hq + hkv:], page, pos % ps


def _write_rows(st, k, v, page, row):
    st["kp"][0][page, :, row] = k.to(st["kp"].dtype)
    st["vp"][0][page, :, row] = v.to(st["vp"].dtype)


def _plain_store(st):
    q, k, v, page, row = _split_rotated(st)
    _write_rows(st, k, v, page, row)
    return q.to(st["kp"].dtype), st["kp"], st["vp"]


def _rows_of(pages, table, b, n, ps):
    """the first n rows of sequence b: [hkv, n, d] in 32 bits"""
    picked = pages[0][table[b, :-(-n // ps)].long()]                     # [pages, hkv, ps, d]
    return picked.transpose(0, 1).reshape(picked.shape[1], -1, picked.shape[3])[:, :n].float().contiguous()


def _plain_prompt(st):
    case = st["case"]
    hq, hkv, d, ps = case["hq"], case["hkv"], case["d"], case["page"]
    group = hq // hkv
    out = torch.empty(st["tokens"], hq, d, dtype=st["q"].dtype, device=DEV)
    first = 0
    for b, (n, h) in enumerate(zip(st["new"], st["hist_host"])):
        k = _rows_of(st["kp"], st["table"], b, h + n, ps)
        v = _rows_of(st["vp"], st["table"], b, h + n, ps)
        for i in range(0, n, 2048):
            m = min(2048, n - i)
            end = h + i + m
            q = st["q"][first + i:first + i + m].float().view(m, hkv, group, d)
            hidden = torch.arange(end, device=DEV)[None, :] > torch.arange(h + i, end, device=DEV)[:, None]
            for kvh in range(hkv):
                s = torch.matmul(q[:, kvh].transpose(0, 1).reshape(group * m, d), k[kvh, :end].t().contiguous()) * d ** -0.5
                s.view(group, m, end).masked_fill_(hidden, -math.inf)
                s = torch.exp_(s.sub_(s.amax(dim=1, keepdim=True)))
                o = torch.matmul(s, v[kvh, :end]) / s.sum(dim=1, keepdim=True)
                out[first + i:first + i + m, kvh * group:(kvh + 1) * group] = o.view(group, m, d).transpose(0, 1).to(out.dtype)
        first += n
    return out


def _plain_decode(st):
    case = st["case"]
    hq, hkv, d, ps = case["hq"], case["hkv"], case["d"], case["page"]
    q, k, v, page, row = _split_rotated(st)
    _write_rows(st, k, v, page, row)
    out = torch.empty(st["tokens"], hq, d, dtype=st["qkv"].dtype, device=DEV)
    for b, t in enumerate(st["rows"]):
        kb, vb = _rows_of(st["kp"], st["table"], b, t, ps), _rows_of(st["vp"], st["table"], b, t, ps)
        s = torch.matmul(q[b].reshape(hkv, hq // hkv, d), kb.transpose(1, 2).contiguous()) * d ** -0.5
        s = torch.exp(s - s.amax(dim=2, keepdim=True))
        out[b] = (torch.matmul(s, vb) / s.sum(dim=2, keepdim=True)).view(hq, d).to(out.dtype)
    return out, st["kp"], st["vp"]


def _plain_logprobs(st):
    k = st["case"]["k"]
    x = st["x"].float()
    m = x.amax(dim=1, keepdim=True)
    e = torch.exp(x - m)
    z = e.sum(dim=1, keepdim=True)
    logz = torch.log(z)
    logprob = (x.gather(1, st["targets"].long()[:, None]) - m - logz)[:, 0]
    moment = torch.where(e > 0, e * (x - m), torch.zeros((), device=DEV)).sum(dim=1, keepdim=True)
    entropy = (logz - moment / z)[:, 0]
    vals, ids = torch.sort(x, dim=1, descending=True, stable=True)
    return logprob, entropy, ids[:, :k].to(torch.int32), vals[:, :k] - m - logz


# ---------------------------------------------------------------- the definition in 64 bits

def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "logprobs":
        return _exact_logprobs(st, case["k"])
    hq, hkv, d, ps = case["hq"], case["hkv"], case["d"], case["page"]
    new, hist, rows = _geometry(case)
    kp, vp = st["kp"].double(), st["vp"].double()
    table = st["table"].tolist()
    if case["op"] == "prompt":
        q_all = st["q"].double()
    else:
        x = st["qkv"].double() + st["bias"].double().reshape(hq + 2 * hkv, d)
        pos = torch.cat([torch.arange(h, h + n, device=DEV) for n, h in zip(new, hist)]).double()
        turn = torch.polar(torch.ones((), dtype=torch.float64, device=DEV),
                           pos[:, None] / ROPE_BASE ** (torch.arange(d // 2, device=DEV).double() * 2 / d))
        pairs = torch.view_as_complex(x[:, :hq + hkv].reshape(len(pos), hq + hkv, d // 2, 2).contiguous())
        qk = torch.view_as_real(pairs * turn[:, None, :]).reshape(len(pos), hq + hkv, d)
        q_all, k_new, v_new = qk[:, :hq], qk[:, hq:], x[:, hq + hkv:]
        first = 0
        # rows as the cache holds them: attention reads the stored values
        kr, vr = k_new.to(st["kp"].dtype).double(), v_new.to(st["vp"].dtype).double()
        kp_new, vp_new = kp.clone(), vp.clone()
        for b, (n, h) in enumerate(zip(new, hist)):
            p = torch.arange(h, h + n, device=DEV)
            pg = torch.tensor(table[b], device=DEV)[p // ps]
            kp_new[0][pg, :, p % ps], vp_new[0][pg, :, p % ps] = k_new[first:first + n], v_new[first:first + n]
            kp[0][pg, :, p % ps], vp[0][pg, :, p % ps] = kr[first:first + n], vr[first:first + n]
            first += n
        if case["op"] == "store":
            return q_all, kp_new, vp_new
    out = torch.empty(sum(new), hq, d, dtype=torch.float64, device=DEV)
    first = 0
    for b, (n, h) in enumerate(zip(new, hist)):
        pages = torch.tensor(table[b][:-(-rows[b] // ps)], device=DEV)
        for head in range(hq):
            kvh = head // (hq // hkv)
            k = kp[0, pages, kvh].reshape(-1, d)[:rows[b]]
            v = vp[0, pages, kvh].reshape(-1, d)[:rows[b]]
            for i in range(0, n, 4096):
                m = min(4096, n - i)
                s = q_all[first + i:first + i + m, head] @ k[:h + i + m].t().contiguous() / math.sqrt(d)
                s = s.masked_fill(torch.ones_like(s, dtype=torch.bool).triu(h + i + 1), -math.inf)
                out[first + i:first + i + m, head] = torch.softmax(s, dim=1) @ v[:h + i + m]
        first += n
    return out if case["op"] == "prompt" else (out, kp_new, vp_new)


def _exact_logprobs(st, k):
    x = st["x"]
    logprob, entropy, tops = [], [], []
    for i in range(0, x.shape[0], 512):
        y = x[i:i + 512].double()
        lp = y - torch.logsumexp(y, dim=1, keepdim=True)
        p = lp.exp()
        logprob.append(lp.gather(1, st["targets"][i:i + 512].long()[:, None])[:, 0])
        entropy.append(-(p * lp.masked_fill(p == 0, 0.0)).sum(dim=1))
        order = torch.sort(y, dim=1, descending=True, stable=True)[1][:, :k]
        tops.append((order.to(torch.int32), lp.gather(1, order)))
    return torch.cat(logprob), torch.cat(entropy), torch.cat([a for a, _ in tops]), torch.cat([b for _, b in tops])


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    size = 2 if case["dtype"] == "fp16" else 4
    if case["op"] == "logprobs":
        n, v, k = case["rows"], case["vocab"], case["k"]
        return {"bytes": n * v * size + n * (4 + 8 + 8 * k), "flops": 5 * n * v}
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    new, hist, rows = _geometry(case)
    tokens, heads = sum(new), hq + 2 * hkv
    meta = 4 * sum(-(-r // case["page"]) for r in rows) + 8 * len(rows)
    if case["op"] == "store":
        return {"bytes": 2 * tokens * heads * d * size + heads * d * size + meta, "flops": tokens * (heads + 3 * (hq + hkv)) * d}
    pairs = sum(n * h + n * (n + 1) // 2 for n, h in zip(new, hist))
    moved = 2 * tokens * hq * d + 2 * sum(rows) * hkv * d
    if case["op"] == "decode":
        moved += 2 * tokens * hkv * d + heads * d        # the new rows come with qkv and go to the cache; the bias
    return {"bytes": moved * size + meta, "flops": 4 * d * hq * pairs}
