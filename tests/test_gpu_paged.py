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
