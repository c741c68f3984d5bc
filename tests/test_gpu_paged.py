"""The operators over a paged key-value cache against their definitions in 64 bits (tests/paged_model.py), at the sizes, strides,
tables and values where they can go wrong."""
import pytest
import torch

import paged_model as pm
from conftest import announce

pytestmark = pytest.mark.gpu

F16, F32 = torch.float16, torch.float32
MARK = 7.0                                     # what outputs hold before a call


def assert_within(got, want, tol):
    got = got.double()
    assert torch.isfinite(got).all(), "%d values are not finite" % int((~torch.isfinite(got)).sum())
    worst = ((got - want).abs() / tol).max().item() if got.numel() else 0.0
    assert worst <= 1.0, "off by %.3f of the tolerance" % worst


# ---------------------------------------------------------------- rows into pages

def check_store(capi, c, rotary_dim, base=10000.0, bias=True, in_place=False):
    announce("paged store", c.dtype, c.lens, c.hist_host, c.hq, c.hkv, c.d, c.ps, rotary_dim)
    q64, written, covered = pm.store(c.qkv, c.bias if bias else None, c.kp, c.vp, c.cu, c.hist_host, c.table, c.layer, rotary_dim, base)
    kp, vp = c.kp.clone(), c.vp.clone()
    if in_place:
        buf = c.qkv.clone()
        q_out = buf[:, :c.hq]
        before = c.qkv[:, :c.hq].clone()
    else:
        buf = c.qkv
        q_out = torch.full((c.tokens, c.hq, c.d), MARK, dtype=c.dtype, device=c.qkv.device)
        before = q_out.clone()
    capi.paged_qkv_store(q_out, kp, vp, buf, c.bias if bias else None, c.cu, c.hist, c.table, rotary_dim, base, layer=c.layer)
    torch.cuda.synchronize()
    x = c.qkv.double().abs() + (c.bias.double().abs().view(c.hq + 2 * c.hkv, c.d) if bias else 0)
    pair = x + x.view(*x.shape[:-1], -1, 2).flip(-1).view(x.shape)
    # the sum with the bias (2^-24), the two rotation products (2^-24 each) and a sine or cosine good to 2^-22
    tol = pm.EPS[c.dtype] * (q64.abs() + 0) + 2.0 ** -21 * pair[:, :c.hq] + pm.TINY[c.dtype]
    assert_within(q_out[covered], q64[covered], tol[covered])
    rest = sorted(set(range(c.tokens)) - set(covered))
    assert torch.equal(q_out[rest], before[rest])
    if in_place:
        assert torch.equal(buf[:, c.hq:], c.qkv[:, c.hq:])
    scale = float(pair.max())
    for (page, row), (k, v) in written.items():
        assert_within(kp[c.layer, page, :, row], k, pm.EPS[c.dtype] * k.abs() + 2.0 ** -21 * scale)
        assert_within(vp[c.layer, page, :, row], v, pm.EPS[c.dtype] * v.abs() + 2.0 ** -23 * scale)
        kp[c.layer, page, :, row] = c.kp[c.layer, page, :, row]
        vp[c.layer, page, :, row] = c.vp[c.layer, page, :, row]
    bits = torch.int16 if c.dtype == F16 else torch.int32
    assert torch.equal(kp.view(bits), c.kp.view(bits)) and torch.equal(vp.view(bits), c.vp.view(bits))      # nothing else


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("lens,hist,hq,hkv,d,ps", [
    ([1], [0], 1, 1, 8, 16),
    ([5, 0, 1, 17], [0, 3, 31, 15], 4, 2, 64, 16),
    ([33, 2], [100, 63], 6, 3, 80, 64),
    ([9, 9, 9], [0, 5, 250], 7, 1, 128, 256),
    ([3, 30], [40000, 7], 8, 8, 256, 32),
])
def test_store(capi, dev, dtype, lens, hist, hq, hkv, d, ps):
    check_store(capi, pm.Case(dtype, lens, hist, hq, hkv, d, ps, seed=3), d)


def test_store_many_sequences_layers_and_leftover_tokens(capi, dev):
    lens = [(i * 7) % 4 for i in range(150)]
    hist = [(i * 13) % 50 for i in range(150)]
    check_store(capi, pm.Case(F16, lens, hist, 4, 2, 64, 16, layers=3, layer=1, extra_tokens=5, seed=4), 64)


def test_store_partial_rotation_no_bias_negative_history(capi, dev):
    check_store(capi, pm.Case(F16, [4, 6, 3], [2, -1, 0], 2, 1, 64, 16, seed=5), 32)
    check_store(capi, pm.Case(F32, [4, 6], [2, 9], 2, 2, 64, 16, seed=6), 128, base=500000.0, bias=False)
    check_store(capi, pm.Case(F16, [4, 6], [2, 9], 2, 2, 64, 16, seed=6), 0, bias=False)


@pytest.mark.parametrize("dtype", [F16, F32])
def test_store_in_place(capi, dev, dtype):
    check_store(capi, pm.Case(dtype, [40, 1, 7], [0, 9, 100], 6, 2, 96, 32, extra_tokens=2, seed=7), 96, in_place=True)
    check_store(capi, pm.Case(dtype, [1], [9], 6, 2, 96, 32, seed=7), 96, in_place=True)


def test_store_drops_rows_without_a_page(capi, dev):
    c = pm.Case(F16, [40, 20], [0, 10], 2, 2, 64, 16, seed=8)
    for b, p, value in ((0, 1, -1), (0, 2, c.num_pages), (1, 1, 2 ** 31 - 1), (1, 0, -2 ** 31)):
        c.table[b, p] = value
    check_store(capi, c, 64)
    c.hist_host = [100000, 2 ** 31 - 21]            # past the table, and to the end of the positions
    c.hist = torch.tensor(c.hist_host, dtype=torch.int32, device=c.q.device)
    check_store(capi, c, 64)


# ---------------------------------------------------------------- attention of packed prompts

def check_prompt(capi, c, out=None, q=None, max_rows=None, workspace=None):
    q = c.q if q is None else q
    announce("paged prompt", c.dtype, c.lens, c.hist_host, c.hq, c.hkv, c.d, c.ps, max_rows)
    want, tol, covered = pm.prompt(q, c.kp, c.vp, c.cu, c.hist_host, c.table, c.layer)
    if out is None:
        out = torch.full((c.tokens, c.hq, c.d), MARK, dtype=c.dtype, device=c.q.device)
    before = out.clone()
    capi.paged_prompt_attn(q, c.kp, c.vp, out, c.cu, c.hist, c.table, c.max_rows if max_rows is None else max_rows, layer=c.layer,
                           workspace=workspace)
    torch.cuda.synchronize()
    assert_within(out[covered], want[covered], tol[covered])
    rest = sorted(set(range(c.tokens)) - set(covered))
    assert torch.equal(out[rest], before[rest])
    return out


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("lens,hist,hq,hkv,d,ps", [
    ([1], [0], 1, 1, 8, 16),
    ([1, 0, 2], [0, 5, 31], 4, 2, 64, 16),
    ([130], [0], 1, 1, 64, 16),
    ([200], [0], 4, 4, 128, 64),
    ([64, 65, 1, 31], [0, 0, 64, 7], 8, 2, 128, 16),
    ([63, 129], [1, 200], 7, 1, 96, 32),
    ([37, 300], [0, 11], 6, 2, 80, 256),
    ([70, 5], [3, 130], 4, 2, 256, 16),
    ([19, 40], [0, 50], 12, 4, 160, 32),
    ([90], [10], 3, 1, 24, 16),
])
def test_prompt(capi, dev, dtype, lens, hist, hq, hkv, d, ps):
    check_prompt(capi, pm.Case(dtype, lens, hist, hq, hkv, d, ps, seed=11))


def test_prompt_many_sequences_layers_and_leftover_tokens(capi, dev):
    lens = [(i * 11) % 9 for i in range(140)]
    hist = [(i * 17) % 70 for i in range(140)]
    check_prompt(capi, pm.Case(F16, lens, hist, 4, 2, 64, 16, layers=3, layer=2, extra_tokens=6, seed=12))


def test_prompt_long(capi, dev):
    check_prompt(capi, pm.Case(F16, [1500, 600], [0, 700], 8, 2, 128, 16, seed=13))


@pytest.mark.parametrize("dtype", [F16, F32])
def test_prompt_few_tokens_behind_many_rows(capi, dev, dtype):
    """the rows are cut into pieces and joined"""
    c = pm.Case(dtype, [3, 1, 8], [5000, 7000, 40], 8, 2, 128, 16, seed=14)
    assert capi.paged_prompt_attn_workspace_bytes(3, 12, 8, 2, 128, c.max_rows) > 256
    full = check_prompt(capi, c)
    # bounds that are too small or far too large change the cut, not the result
    check_prompt(capi, c, max_rows=1)
    check_prompt(capi, c, max_rows=2000)
    check_prompt(capi, c, max_rows=100000)
    assert torch.equal(full, check_prompt(capi, c))


def test_prompt_strided_tokens_and_in_place(capi, dev):
    c = pm.Case(F16, [50, 9], [0, 33], 6, 2, 64, 16, extra_tokens=1, seed=15)
    c.qkv[:, :6] = c.q
    wide = torch.full((c.tokens, 10, c.d), MARK, dtype=F16, device=c.q.device)
    check_prompt(capi, c, q=c.qkv[:, :6], out=wide[:, 2:8])
    assert (wide[:, :2] == MARK).all() and (wide[:, 8:] == MARK).all()
    plain = check_prompt(capi, c)
    buf = c.q.clone()
    capi.paged_prompt_attn(buf, c.kp, c.vp, buf, c.cu, c.hist, c.table, c.max_rows)
    assert torch.equal(buf[:59], plain[:59])


def test_prompt_rows_without_a_page_take_no_part(capi, dev):
    for dtype in (F16, F32):
        c = pm.Case(dtype, [40, 150, 20], [0, 10, 300], 4, 2, 64, 16, seed=16)
        for b, p, value in ((0, 0, -1), (1, 0, c.num_pages), (1, 3, 2 ** 31 - 1), (1, 6, -2 ** 31), (2, 19, -5)):
            c.table[b, p] = value
        out = check_prompt(capi, c)
        assert (out[:16] == 0).all()                      # the first page of sequence 0 is none: its first rows see nothing
        c.table[1] = -1
        out = check_prompt(capi, c)
        assert (out[40:190] == 0).all()
        c = pm.Case(dtype, [40, 150, 20], [0, 10, 300], 4, 2, 64, 16, seed=16)
        outs = []
        for far in (1000, 10 ** 8, 2 ** 31 - 1):              # left alone; rows past the table are none
            c.hist_host = [-3, 1000, 300]
            c.hist = torch.tensor([-3, far, 300], dtype=torch.int32, device=c.q.device)
            outs.append(check_prompt(capi, c))
            assert (outs[-1][:40] == MARK).all() and torch.equal(outs[-1], outs[0])


@pytest.mark.parametrize("dtype", [F16, F32])
def test_prompt_values_a_row_does_not_see_do_not_reach_it(capi, dev, dtype):
    c = pm.Case(dtype, [100, 90], [20, 0], 4, 2, 64, 16, seed=17)
    clean = check_prompt(capi, c)
    kp, vp = c.kp.clone(), c.vp.clone()
    for row, what in ((77, float("nan")), (90, float("inf")), (101, float("-inf"))):       # rows of sequence 0: tokens 57, 70, 81
        page = int(c.table[0, row // 16])
        c.vp[0, page, 0, row % 16, 3] = what
        c.kp[0, page, 1, row % 16, 5] = what
    got = torch.full_like(clean, MARK)
    capi.paged_prompt_attn(c.q, c.kp, c.vp, got, c.cu, c.hist, c.table, c.max_rows)
    assert torch.equal(got[:57], clean[:57]) and torch.equal(got[100:], clean[100:])
    heads0 = got[57:100, :2]
    assert torch.isnan(heads0[:, :, 3]).all()                                              # a NaN that is seen stays one
    others = [d for d in range(64) if d != 3]
    assert torch.equal(heads0[:, :, others], clean[57:100, :2][:, :, others])
    assert torch.isnan(got[57:100, 2:]).all()
    c.kp, c.vp = kp, vp.clone()
    page = int(c.table[0, 90 // 16])
    c.vp[0, page, 0, 90 % 16, 3] = float("inf")
    capi.paged_prompt_attn(c.q, c.kp, c.vp, got, c.cu, c.hist, c.table, c.max_rows)
    assert torch.equal(got[:70], clean[:70])
    assert (got[70:100, :2, 3] == float("inf")).all()
    assert torch.equal(got[70:100, :2][:, :, others], clean[70:100, :2][:, :, others])


def test_prompt_extreme_scores(capi, dev):
    c = pm.Case(F32, [70], [30], 2, 1, 64, 16, seed=18)
    c.q *= 300.0                                            # weights of exactly one key, scores in the thousands
    check_prompt(capi, c)
    c = pm.Case(F16, [70], [30], 2, 1, 64, 16, seed=18)
    c.q.zero_()                                             # all scores equal
    check_prompt(capi, c)


def test_prompt_and_store_beyond_four_gigabytes(capi, dev):
    """pages whose offsets pass 2^32 bytes and 2^31 elements"""
    c = pm.Case(F16, [70], [90], 4, 2, 128, 16, seed=19)
    big = 2 ** 32 // (2 * 16 * 128 * 2) * 5 // 4
    kp, vp = (torch.zeros(1, big, 2, 16, 128, dtype=F16, device=dev) for _ in range(2))
    far = c.table.clone()
    for p in range(10):
        page = big - 1 - 3 * p
        kp[0, page], vp[0, page] = c.kp[0, int(c.table[0, p])], c.vp[0, int(c.table[0, p])]
        far[0, p] = page
    want = check_prompt(capi, c)
    out = torch.full_like(want, MARK)
    capi.paged_prompt_attn(c.q, kp, vp, out, c.cu, c.hist, far, c.max_rows)
    assert torch.equal(out, want)
    capi.paged_qkv_store(out, kp, vp, c.qkv, c.bias, c.cu, c.hist, far, 128, 10000.0)
    ref = torch.full_like(want, MARK)
    capi.paged_qkv_store(ref, c.kp, c.vp, c.qkv, c.bias, c.cu, c.hist, c.table, 128, 10000.0)
    assert torch.equal(out, ref)
    for p in range(10):
        assert torch.equal(kp[0, int(far[0, p])], c.kp[0, int(c.table[0, p])])


def test_prompt_on_other_streams_and_in_graphs(capi, dev):
    """two calls at once with a workspace each; one call captured and replayed on changing inputs"""
    cases = [pm.Case(F16, [3, 2], [5000, 4000], 8, 2, 128, 16, seed=20 + i) for i in range(2)]
    want = [check_prompt(capi, c) for c in cases]
    outs = [torch.full_like(w, MARK) for w in want]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for c, o, s in zip(cases, outs, streams):
        with torch.cuda.stream(s):
            capi.paged_prompt_attn(c.q, c.kp, c.vp, o, c.cu, c.hist, c.table, c.max_rows)
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert torch.equal(o, w)
    c = cases[0]
    n = capi.paged_prompt_attn_workspace_bytes(2, 5, 8, 2, 128, c.max_rows)
    ws = torch.empty(n, dtype=torch.uint8, device=dev)
    out = torch.full_like(want[0], MARK)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        capi.paged_prompt_attn(c.q, c.kp, c.vp, out, c.cu, c.hist, c.table, c.max_rows, workspace=ws)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[0])
        c.q.mul_(1.25)
        c.hist[0] -= 100
        c.hist_host[0] -= 100
        want[0] = check_prompt(capi, c)


# ---------------------------------------------------------------- one new token per sequence

def decode_case(dtype, ts, hq, hkv, d, ps, seed, **kw):
    """sequences of ts[b] rows with the new token; its own row is not in the cache yet"""
    c = pm.Case(dtype, [max(t, 1) for t in ts], [0] * len(ts), hq, hkv, d, ps, seed=seed, **kw)
    c.ts = ts
    c.qkv = c.qkv[:len(ts)].contiguous()
    c.t_dev = torch.tensor(ts, dtype=torch.int32, device=c.q.device)
    for b, t in enumerate(ts):
        if t >= 1:
            page = pm.page_of(c.table, b, t - 1, c.num_pages, ps)
            c.kp[c.layer, page, :, (t - 1) % ps] = float("nan")
            c.vp[c.layer, page, :, (t - 1) % ps] = float("nan")
    return c


def run_decode(capi, c, kp, vp, rotary_dim, base=10000.0, bias=True, max_t=None, flags=0, workspace=None, out=None):
    announce("paged decode", c.dtype, c.ts, c.hq, c.hkv, c.d, c.ps, max_t, flags)
    if out is None:
        out = torch.full((len(c.ts), c.hq, c.d), MARK, dtype=c.dtype, device=c.q.device)
    capi.paged_decode_attn(c.qkv, c.bias if bias else None, kp, vp, out, c.table, c.t_dev, max(1, max(c.ts)) if max_t is None else max_t,
                           rotary_dim, base, layer=c.layer, flags=flags, workspace=workspace)
    torch.cuda.synchronize()
    return out


def check_decode(capi, c, rotary_dim, base=10000.0, bias=True, skip=(), **kw):
    """skip: sequences that have to be left alone"""
    B = len(c.ts)
    ts = [0 if b in skip else t for b, t in enumerate(c.ts)]
    # the new rows, within a rounding of their definition
    lens, hist = [1 if t >= 1 else 0 for t in ts], [max(0, t - 1) for t in ts]
    cu = [sum(lens[:i]) for i in range(B + 1)]
    keep = [b for b in range(B) if lens[b]]
    _, written, _ = pm.store(c.qkv[keep], c.bias if bias else None, c.kp, c.vp, cu, hist, c.table, c.layer, rotary_dim, base)
    kp, vp = c.kp.clone(), c.vp.clone()
    out = run_decode(capi, c, kp, vp, rotary_dim, base, bias, **kw)
    k_rows = torch.zeros(B, c.hkv, c.d, dtype=c.dtype, device=c.q.device)
    v_rows = k_rows.clone()
    for b in keep:
        page = pm.page_of(c.table, b, c.ts[b] - 1, c.num_pages, c.ps)
        row = (c.ts[b] - 1) % c.ps
        if page < 0:                                        # not stored: what the same call stores where there is a page
            other = pm.Case(c.dtype, [c.ts[b]], [0], c.hq, c.hkv, c.d, c.ps, device=c.q.device, seed=1)
            other.qkv, other.bias, other.ts, other.layer = c.qkv[b:b + 1].contiguous(), c.bias, [c.ts[b]], 0
            other.t_dev = c.t_dev[b:b + 1].contiguous()
            run_decode(capi, other, other.kp, other.vp, rotary_dim, base, bias)
            k_rows[b], v_rows[b] = (x[0, int(other.table[0, (c.ts[b] - 1) // c.ps]), :, row] for x in (other.kp, other.vp))
            continue
        k_rows[b], v_rows[b] = kp[c.layer, page, :, row], vp[c.layer, page, :, row]
        k, v = written[(page, row)]
        assert_within(k_rows[b], k, pm.EPS[c.dtype] * k.abs() + 2.0 ** -18)
        assert_within(v_rows[b], v, pm.EPS[c.dtype] * v.abs() + 2.0 ** -21)
        kp[c.layer, page, :, row], vp[c.layer, page, :, row] = c.kp[c.layer, page, :, row], c.vp[c.layer, page, :, row]
    bits = torch.int16 if c.dtype == F16 else torch.int32
    assert torch.equal(kp.view(bits), c.kp.view(bits)) and torch.equal(vp.view(bits), c.vp.view(bits))      # nothing else
    want, tol = pm.decode(c, ts, k_rows, v_rows, rotary_dim, base, bias)
    assert_within(out[keep], want[keep], tol[keep])
    rest = [b for b in range(B) if b not in keep]
    assert (out[rest] == MARK).all()
    return out


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("ts,hq,hkv,d,ps", [
    ([1], 1, 1, 8, 16),
    ([2, 1, 16, 17], 4, 2, 64, 16),
    ([33, 64, 65, 129], 7, 1, 128, 64),
    ([900], 32, 8, 128, 16),
    ([257, 3000, 1, 511], 8, 8, 128, 32),
    ([100, 700], 6, 2, 80, 16),
    ([100, 1300], 16, 1, 96, 256),
    ([77, 640], 20, 1, 64, 16),
    ([40, 500], 34, 2, 128, 16),
    ([90, 1000], 4, 2, 256, 16),
    ([50, 200], 6, 2, 160, 32),
])
def test_decode(capi, dev, dtype, ts, hq, hkv, d, ps):
    check_decode(capi, decode_case(dtype, ts, hq, hkv, d, ps, seed=31), d)


def test_decode_many_sequences_and_layers(capi, dev):
    ts = [1 + (i * 37) % 400 for i in range(200)]
    check_decode(capi, decode_case(F16, ts, 8, 2, 64, 16, seed=32, layers=3, layer=1), 64)


@pytest.mark.parametrize("dtype", [F16, F32])
def test_decode_one_long_sequence(capi, dev, dtype):
    """many pieces per unit; positions far out"""
    check_decode(capi, decode_case(dtype, [20000], 8, 1, 128, 64, seed=33), 128)
    check_decode(capi, decode_case(dtype, [30011, 5], 3, 1, 64, 16, seed=34), 64, base=500000.0)


def test_decode_partial_rotation_and_no_bias(capi, dev):
    check_decode(capi, decode_case(F16, [70, 5], 4, 2, 64, 16, seed=35), 32, bias=False)
    check_decode(capi, decode_case(F32, [70, 5], 4, 2, 64, 16, seed=35), 0)
    check_decode(capi, decode_case(F16, [70, 5], 4, 2, 64, 16, seed=35), 128)


@pytest.mark.parametrize("dtype", [F16, F32])
def test_decode_lengths_out_of_range_are_left_alone(capi, dev, dtype):
    c = decode_case(dtype, [40, 100, 7, 90, 33], 4, 2, 64, 16, seed=36)
    c.ts = [0, 100, -7, 101, 33]
    c.t_dev = torch.tensor(c.ts, dtype=torch.int32, device=c.q.device)
    check_decode(capi, c, 64, max_t=100, skip=(0, 2, 3))
    c.ts = [0, 100, -7, 1000, 33]                            # past the table
    c.t_dev = torch.tensor(c.ts, dtype=torch.int32, device=c.q.device)
    check_decode(capi, c, 64, max_t=5000, skip=(0, 2, 3))
    c.t_dev.fill_(0)
    c.ts = [0] * 5
    check_decode(capi, c, 64, max_t=100, skip=range(5))


@pytest.mark.parametrize("dtype", [F16, F32])
def test_decode_rows_without_a_page_take_no_part(capi, dev, dtype):
    c = decode_case(dtype, [400, 150, 3000, 20], 6, 2, 64, 16, seed=37)
    for b, p, value in ((0, 0, -1), (0, 7, c.num_pages), (0, 24, -9), (1, 4, 2 ** 31 - 1), (1, 9, -2 ** 31)):
        c.table[b, p] = value
    c.table[2, 10:180] = -1                                  # whole pieces without a row
    c.table[3] = -1                                          # nothing but the new token
    check_decode(capi, c, 64)


def test_decode_workspace_with_and_without_the_flag(capi, dev):
    cases = [decode_case(F16, [5000, 300], 8, 2, 128, 16, seed=38), decode_case(F32, [1, 900, 4000], 4, 1, 64, 32, seed=39)]
    size = max(capi.paged_decode_attn_workspace_bytes(len(c.ts), c.hq, c.hkv, c.d, max(c.ts)) for c in cases)
    ws = torch.zeros(size, dtype=torch.uint8, device=dev)
    plain = [check_decode(capi, c, c.d) for c in cases]
    for _ in range(20):                                      # shapes in turn on one zero-filled workspace
        for c, want in zip(cases, plain):
            out = run_decode(capi, c, c.kp.clone(), c.vp.clone(), c.d, flags=capi.ATTN_ZEROED_WORKSPACE, workspace=ws)
            assert torch.equal(out, want)
    dirty = torch.full((size,), 0x5A, dtype=torch.uint8, device=dev)
    for c, want in zip(cases, plain):
        assert torch.equal(run_decode(capi, c, c.kp.clone(), c.vp.clone(), c.d, workspace=dirty), want)


def test_decode_on_other_streams_and_in_graphs(capi, dev):
    cases = [decode_case(F16, [3000, 800], 8, 2, 128, 16, seed=40 + i) for i in range(2)]
    want = [check_decode(capi, c, 128) for c in cases]
    outs = [torch.full_like(w, MARK) for w in want]
    torch.cuda.synchronize()
    for c, o in zip(cases, outs):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            capi.paged_decode_attn(c.qkv, c.bias, c.kp, c.vp, o, c.table, c.t_dev, 3000, 128, 10000.0)
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert torch.equal(o, w)
    # two captured calls share a zero-filled workspace; the lengths grow between replays
    c = cases[0]
    ws = torch.zeros(capi.paged_decode_attn_workspace_bytes(2, 8, 2, 128, 3000), dtype=torch.uint8, device=dev)
    outs = [torch.full_like(want[0], MARK) for _ in range(2)]
    graphs = []
    for o in outs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            capi.paged_decode_attn(c.qkv, c.bias, c.kp, c.vp, o, c.table, c.t_dev, 3000, 128, 10000.0,
                                   flags=capi.ATTN_ZEROED_WORKSPACE, workspace=ws)
        graphs.append(g)
    for _ in range(3):
        for g, o in zip(graphs, outs):
            o.fill_(MARK)
            g.replay()
        torch.cuda.synchronize()
        for o in outs:
            assert torch.equal(o, want[0])
        c.ts = [c.ts[0] - 700, c.ts[1] + 1]
        c.t_dev.copy_(torch.tensor(c.ts, dtype=torch.int32))
        want[0] = check_decode(capi, c, 128, max_t=3000)


def test_decode_beyond_four_gigabytes(capi, dev):
    c = decode_case(F16, [150], 4, 2, 128, 16, seed=43)
    want = check_decode(capi, c, 128)
    big = 2 ** 32 // (2 * 16 * 128 * 2) * 5 // 4
    kp, vp = (torch.zeros(1, big, 2, 16, 128, dtype=F16, device=dev) for _ in range(2))
    near = c.table.clone()
    for p in range(10):
        page = big - 1 - 3 * p
        kp[0, page], vp[0, page] = c.kp[0, int(near[0, p])], c.vp[0, int(near[0, p])]
        c.table[0, p] = page
    assert torch.equal(run_decode(capi, c, kp, vp, 128), want)


def test_decode_agrees_with_the_contiguous_cache(capi, dev):
    """the same step on onellm_decode_attn's cache, positions from 0 as prompts write them"""
    c = decode_case(F16, [700, 700, 700], 8, 2, 128, 16, seed=44)
    out = check_decode(capi, c, 128)
    kc = torch.zeros(1, 3, 2, 704, 128, dtype=F16, device=dev)
    vc = torch.zeros_like(kc)
    for b in range(3):
        for p in range(44):
            kc[0, b, :, 16 * p:16 * p + 16] = c.kp[0, int(c.table[b, p])]
            vc[0, b, :, 16 * p:16 * p + 16] = c.vp[0, int(c.table[b, p])]
    flat = torch.empty(3, 8 * 128, dtype=F16, device=dev)
    capi.decode_attn(c.qkv, c.bias, kc, vc, flat, 8, 700, 128, 10000.0, rope_pos_offset=-1)
    torch.testing.assert_close(out.view(3, -1), flat, rtol=1e-2, atol=2e-3)


# ---------------------------------------------------------------- what the Python bindings refuse

def test_bindings_refuse_other_devices_types_and_layouts(capi, dev):
    c = pm.Case(F16, [20, 9], [0, 33], 4, 2, 64, 16, seed=45)
    out = torch.empty_like(c.q)
    good = dict(q=c.q, kp=c.kp, vp=c.vp, out=out, cu=c.cu, hist=c.hist, table=c.table)

    def prompt(**kw):
        a = dict(good, **kw)
        capi.paged_prompt_attn(a["q"], a["kp"], a["vp"], a["out"], a["cu"], a["hist"], a["table"], c.max_rows)

    prompt()
    for name in good:
        with pytest.raises(ValueError):
            prompt(**{name: good[name].cpu()})
    for name in ("cu", "hist", "table"):
        with pytest.raises(TypeError):
            prompt(**{name: good[name].long()})
    for bad in (dict(q=c.q.float()), dict(out=out.float()), dict(out=out[:, :2]), dict(kp=c.kp[0]), dict(vp=c.vp.float()), dict(cu=c.cu[:-1]),
                dict(hist=c.hist[:1]), dict(table=c.table[:, ::2]), dict(q=c.q.transpose(1, 2).contiguous().transpose(1, 2))):
        with pytest.raises((ValueError, TypeError)):
            prompt(**bad)
    with pytest.raises(ValueError):
        capi.paged_qkv_store(out, c.kp, c.vp, c.qkv.cpu(), c.bias, c.cu, c.hist, c.table, 64, 10000.0)
    with pytest.raises(ValueError):
        capi.paged_qkv_store(out, c.kp, c.vp, c.qkv, c.bias[:-1], c.cu, c.hist, c.table, 64, 10000.0)
    with pytest.raises(capi.OnellmError):
        capi.paged_qkv_store(out, c.kp, c.vp, c.qkv, c.bias, c.cu, c.hist, c.table, 63, 10000.0)
    t = torch.tensor([5, 5], dtype=torch.int32, device=dev)
    for bad in (dict(t=t.cpu()), dict(t=t[:1]), dict(out=out[:1])):
        with pytest.raises(ValueError):
            capi.paged_decode_attn(c.qkv[:2].contiguous(), c.bias, c.kp, c.vp, bad.get("out", out[:2]), c.table, bad.get("t", t), 64, 64, 10000.0)
    torch.cuda.synchronize()
