"""The far ends of what the paged entry points and the log-probabilities take, and buffers that share memory (no GPU needed: every call
here is refused before anything is launched)."""
import pytest

from test_paged_refusals import FAKE, decode, logprobs, prompt, store

E = 2                                                       # bytes of an element (fp16)


def test_a_launch_has_to_hold_the_tokens(capi):
    # one head of 8 elements: 8 tokens per workgroup of 256 threads, so 2^28 tokens would be 2^33 threads
    small = dict(Hq=1, Hkv=1, D=8, rot=8, q_stride=8, qkv=2 ** 44)
    assert store(capi, tokens=2 ** 25 + 1, **small) == capi.EUNSUPPORTED
    assert logprobs(capi, N=2 ** 23 + 1) == capi.EUNSUPPORTED


def test_prompt_tiles(capi):
    far = dict(out=2 ** 45, Hq=32, Hkv=8, q_stride=4096, out_stride=4096)
    assert prompt(capi, tokens=2 ** 21 + 128, **far) == capi.EUNSUPPORTED          # 65540 tiles of 128 rows
    assert prompt(capi, tokens=2 ** 25, **far) == capi.EUNSUPPORTED                # 2^30 rows


@pytest.mark.parametrize("kw", [
    dict(out=FAKE + 16), dict(out=FAKE - 16), dict(out_stride=1024), dict(q_stride=520),
    dict(out=FAKE + 512 * E), dict(out=FAKE + 2 * 512 * E),                        # a row of q each
    # rows a stride apart that reach into the next one's
    dict(q_stride=1016, out_stride=1016, out=FAKE + 512 * E), dict(q_stride=1024, out_stride=1024, out=FAKE + 504 * E),
    dict(q_stride=1024, out_stride=1024, out=FAKE + 520 * E), dict(q_stride=1024, out_stride=1024, out=FAKE - 504 * E),
])
def test_prompt_out_over_q(capi, kw):
    assert prompt(capi, **kw) == capi.EINVAL


@pytest.mark.parametrize("kw", [
    dict(), dict(out=FAKE + 3 * 512 * E), dict(out=FAKE - 3 * 512 * E), dict(tokens=1, out_stride=1024),
    dict(q_stride=1024, out_stride=1024, out=FAKE + 512 * E), dict(q_stride=1024, out_stride=1024, out=FAKE - 512 * E),
])
def test_prompt_out_beside_q_is_taken(capi, kw):
    # (past the check of the buffers: a workspace that is too small is found behind it)
    assert prompt(capi, max_rows=5000, ws=None, **kw) == capi.EWORKSPACE


@pytest.mark.parametrize("out", [FAKE, FAKE + 2 * 8 * 128 * E - 16, FAKE - 2 * 4 * 128 * E + 16, FAKE + 1024])
def test_decode_out_over_qkv(capi, out):
    assert decode(capi, out=out) == capi.EINVAL


def test_prompt_workspace_never_grows_past_its_bound(capi):
    for hkv in (1, 2, 8, 32, 40):
        for g in (1, 3, 8):
            for d in (8, 64, 128, 136, 256):
                for tokens in (1, 2, 63, 64, 129, 500, 1100, 4000, 12000, 50000):
                    for B in (1, 7, 300):
                        n = capi.paged_prompt_attn_workspace_bytes(B, tokens, g * hkv, hkv, d, 2 ** 29)
                        assert n <= 786432 * (d + 2) + 256, (B, tokens, g, hkv, d, n)
