"""What the entry points over a paged cache refuse, before anything is launched (no GPU needed: no pointer is dereferenced)."""
import ctypes

import pytest

FAKE = 0x10000


def ptr(v):
    return None if v is None else ctypes.c_void_p(v)


GEOMETRY_REFUSALS = [
    (dict(dtype=2), "EINVAL"), (dict(dtype=-1), "EINVAL"),
    (dict(kp=None), "EINVAL"), (dict(vp=None), "EINVAL"), (dict(table=None), "EINVAL"),
    (dict(B=0), "EINVAL"), (dict(B=-3), "EINVAL"), (dict(Hq=0), "EINVAL"), (dict(Hkv=0), "EINVAL"), (dict(Hq=5), "EINVAL"), (dict(D=0), "EINVAL"),
    (dict(page=0), "EINVAL"), (dict(page=-16), "EINVAL"), (dict(num_pages=0), "EINVAL"), (dict(max_pages=0), "EINVAL"),
    (dict(layer=-1), "EINVAL"), (dict(layer=2), "EINVAL"), (dict(L=0), "EINVAL"),
    (dict(page=8), "EUNSUPPORTED"), (dict(page=24), "EUNSUPPORTED"), (dict(page=48), "EUNSUPPORTED"),
    (dict(D=264), "EUNSUPPORTED"), (dict(D=68), "EUNSUPPORTED"), (dict(dtype=0, D=66), "EUNSUPPORTED"),
    (dict(B=65536), "EUNSUPPORTED"), (dict(Hq=4098, Hkv=2), "EUNSUPPORTED"), (dict(max_pages=2 ** 26), "EUNSUPPORTED"),
    (dict(page=2 ** 22, max_pages=1), "EUNSUPPORTED"),
    (dict(kp=FAKE + 8), "EUNSUPPORTED"), (dict(vp=FAKE + 2), "EUNSUPPORTED"),
]


def store(capi, **kw):
    a = dict(dtype=1, q_out=FAKE, q_stride=512, kp=FAKE, vp=FAKE, qkv=2 * FAKE, bias=None, cu=FAKE, hist=FAKE, table=FAKE, B=2, tokens=3, Hq=4,
             Hkv=2, D=128, page=16, num_pages=9, max_pages=4, layer=1, L=2, rot=128, base=10000.0)
    a.update(kw)
    return capi.lib().onellm_paged_qkv_store(a["dtype"], ptr(a["q_out"]), a["q_stride"], ptr(a["kp"]), ptr(a["vp"]), ptr(a["qkv"]),
                                             ptr(a["bias"]), ptr(a["cu"]), ptr(a["hist"]), ptr(a["table"]), a["B"], a["tokens"], a["Hq"],
                                             a["Hkv"], a["D"], a["page"], a["num_pages"], a["max_pages"], a["layer"], a["L"], a["rot"],
                                             a["base"], None)


def prompt(capi, **kw):
    a = dict(dtype=1, q=FAKE, q_stride=512, kp=FAKE, vp=FAKE, out=FAKE, out_stride=512, cu=FAKE, hist=FAKE, table=FAKE, B=2, tokens=3, Hq=4,
             Hkv=2, D=128, page=16, num_pages=9, max_pages=400, layer=1, L=2, max_rows=64, ws=FAKE, ws_bytes=2 ** 40)
    a.update(kw)
    return capi.lib().onellm_paged_prompt_attn(a["dtype"], ptr(a["q"]), a["q_stride"], ptr(a["kp"]), ptr(a["vp"]), ptr(a["out"]),
                                               a["out_stride"], ptr(a["cu"]), ptr(a["hist"]), ptr(a["table"]), a["B"], a["tokens"],
                                               a["Hq"], a["Hkv"], a["D"], a["page"], a["num_pages"], a["max_pages"], a["layer"], a["L"],
                                               a["max_rows"], ptr(a["ws"]), a["ws_bytes"], None)


def decode(capi, **kw):
    a = dict(dtype=1, qkv=FAKE, bias=None, kp=FAKE, vp=FAKE, out=FAKE, table=FAKE, t=FAKE, B=2, Hq=4, Hkv=2, D=128, page=16, num_pages=9,
             max_pages=4, layer=1, L=2, max_t=64, rot=128, base=10000.0, flags=0, ws=FAKE, ws_bytes=2 ** 40)
    a.update(kw)
    return capi.lib().onellm_paged_decode_attn(a["dtype"], ptr(a["qkv"]), ptr(a["bias"]), ptr(a["kp"]), ptr(a["vp"]), ptr(a["out"]),
                                               ptr(a["table"]), ptr(a["t"]), a["B"], a["Hq"], a["Hkv"], a["D"], a["page"],
                                               a["num_pages"], a["max_pages"], a["layer"], a["L"], a["max_t"], a["rot"], a["base"],
                                               a["flags"], ptr(a["ws"]), a["ws_bytes"], None)


@pytest.mark.parametrize("call", [store, prompt, decode])
@pytest.mark.parametrize("kw,code", GEOMETRY_REFUSALS)
def test_geometry(capi, call, kw, code):
    assert call(capi, **kw) == getattr(capi, code)


@pytest.mark.parametrize("kw,code", [
    (dict(q_out=None), "EINVAL"), (dict(qkv=None), "EINVAL"), (dict(cu=None), "EINVAL"), (dict(hist=None), "EINVAL"), (dict(tokens=-1), "EINVAL"),
    (dict(rot=-2), "EINVAL"), (dict(rot=63), "EINVAL"), (dict(base=0.0), "EINVAL"), (dict(base=-1.0), "EINVAL"),
    (dict(base=float("nan")), "EINVAL"), (dict(base=float("inf")), "EINVAL"), (dict(q_stride=511), "EINVAL"), (dict(q_stride=-512), "EINVAL"),
    (dict(q_stride=516), "EUNSUPPORTED"), (dict(q_out=FAKE + 8), "EUNSUPPORTED"), (dict(qkv=2 * FAKE + 4), "EUNSUPPORTED"), (dict(bias=FAKE + 2), "EUNSUPPORTED"),
    # q over a part of qkv that is not its own place
    (dict(qkv=FAKE), "EINVAL"), (dict(qkv=FAKE, q_stride=1032), "EINVAL"), (dict(qkv=FAKE + 1024, q_stride=1024), "EINVAL"),
    (dict(q_out=2 * FAKE + 3 * 8 * 128 * 2 - 16), "EINVAL"), (dict(tokens=2 ** 28 + 1), "EUNSUPPORTED"), (dict(tokens=2 ** 31 - 1), "EUNSUPPORTED"),
])
def test_store_refusals(capi, kw, code):
    assert store(capi, **kw) == getattr(capi, code)


@pytest.mark.parametrize("kw,code", [
    (dict(q=None), "EINVAL"), (dict(out=None), "EINVAL"), (dict(cu=None), "EINVAL"), (dict(hist=None), "EINVAL"), (dict(tokens=-1), "EINVAL"),
    (dict(max_rows=0), "EINVAL"), (dict(max_rows=-1), "EINVAL"), (dict(q_stride=508), "EINVAL"), (dict(out_stride=0), "EINVAL"),
    (dict(q_stride=514), "EUNSUPPORTED"), (dict(out_stride=516), "EUNSUPPORTED"), (dict(q=FAKE + 4), "EUNSUPPORTED"), (dict(out=FAKE + 8), "EUNSUPPORTED"),
    (dict(tokens=2 ** 28 + 1), "EUNSUPPORTED"),
    (dict(max_rows=5000, ws=None), "EWORKSPACE"), (dict(max_rows=5000, ws_bytes=1000), "EWORKSPACE"), (dict(max_rows=5000, ws=FAKE + 8), "EWORKSPACE"),
])
def test_prompt_refusals(capi, kw, code):
    assert prompt(capi, **kw) == getattr(capi, code)


@pytest.mark.parametrize("kw,code", [
    (dict(qkv=None), "EINVAL"), (dict(out=None), "EINVAL"), (dict(t=None), "EINVAL"), (dict(max_t=0), "EINVAL"), (dict(max_t=-4), "EINVAL"),
    (dict(flags=1), "EINVAL"), (dict(flags=2), "EINVAL"), (dict(flags=12), "EINVAL"), (dict(rot=-2), "EINVAL"), (dict(rot=7), "EINVAL"),
    (dict(base=0.0), "EINVAL"), (dict(base=float("nan")), "EINVAL"),
    (dict(qkv=FAKE + 4), "EUNSUPPORTED"), (dict(out=FAKE + 8), "EUNSUPPORTED"), (dict(bias=FAKE + 2), "EUNSUPPORTED"),
    (dict(ws=None), "EWORKSPACE"), (dict(ws=FAKE + 4), "EWORKSPACE"), (dict(ws_bytes=4096), "EWORKSPACE"),
    # more work than the schedule can number, however coarse its items
    (dict(B=65535, Hq=4096, Hkv=4096, max_t=64), "EUNSUPPORTED"),
])
def test_decode_refusals(capi, kw, code):
    assert decode(capi, **kw) == getattr(capi, code)


def logprobs(capi, **kw):
    a = dict(dtype=1, x=FAKE, ld=100000, targets=FAKE, N=3, V=100000, K=5, lp=FAKE, ent=FAKE, ids=FAKE, tops=FAKE, ws=FAKE, ws_bytes=2 ** 40)
    a.update(kw)
    return capi.lib().onellm_token_logprobs(a["dtype"], ptr(a["x"]), a["ld"], ptr(a["targets"]), a["N"], a["V"], a["K"], ptr(a["lp"]),
                                            ptr(a["ent"]), ptr(a["ids"]), ptr(a["tops"]), ptr(a["ws"]), a["ws_bytes"], None)


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=2), "EINVAL"), (dict(x=None), "EINVAL"), (dict(x=FAKE + 1), "EINVAL"), (dict(dtype=0, x=FAKE + 2), "EINVAL"),
    (dict(targets=None), "EINVAL"), (dict(N=-1), "EINVAL"), (dict(V=0), "EINVAL"), (dict(ld=99999), "EINVAL"), (dict(K=-1), "EINVAL"),
    (dict(ids=None), "EINVAL"), (dict(tops=None), "EINVAL"), (dict(lp=None, ent=None, K=0), "EINVAL"),
    (dict(K=33), "EUNSUPPORTED"), (dict(V=2 ** 28 + 1, ld=2 ** 29), "EUNSUPPORTED"), (dict(N=2 ** 26 + 1), "EUNSUPPORTED"),
    (dict(ws=None), "EWORKSPACE"), (dict(ws=FAKE + 8), "EWORKSPACE"), (dict(ws_bytes=200), "EWORKSPACE"),
])
def test_logprobs_refusals(capi, kw, code):
    assert logprobs(capi, **kw) == getattr(capi, code)


def test_no_tokens_is_no_work(capi):
    assert logprobs(capi, N=0, x=None, targets=None, ids=None, tops=None, ws=None, ws_bytes=0) == 0
    assert store(capi, tokens=0, q_out=None, qkv=None) == 0
    assert prompt(capi, tokens=0, q=None, out=None, ws=None, ws_bytes=0) == 0


def test_workspace_sizes(capi):
    size = capi.paged_prompt_attn_workspace_bytes
    assert size(1, 8192, 32, 8, 128, 8192) == 256                     # enough tiles: nothing is cut in either type
    n = size(1, 8, 32, 8, 128, 32768)
    assert n % 256 == 0 and n >= 2 * 8 * 32 * 130 * 4
    assert size(0, 8, 32, 8, 128, 32768) == 256 and size(1, 8, 32, 7, 128, 100) == 256
