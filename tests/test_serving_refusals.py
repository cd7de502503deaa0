"""Batched serving over a paged cache: argument checks of the C entry points.  Every refusal comes
before any HIP call, so these run without a GPU (pointers are addresses that are never read)."""
import pytest

P = 4096  # an aligned address


def _check(rc):
    from camelid_amd._native import check
    check(rc)


ROPE = dict(qkv=P, n_seqs=2, n_new=1, new_lens=None, n_heads=8, n_kv=2, hd=64, rope_dim=64, split_half=0, cos=P, sin=P,
            q_norm=None, k_norm=None, eps=1e-5, q_out=P, q_type=0, kc=P, vc=P, kv_type=1, n_pages=4, page_size=16,
            table=P, stride=2, lens=P, status=None, stream=None)
ATTN = dict(q=P, q_type=0, q_stride=512, n_seqs=2, n_new=1, new_lens=None, n_heads=8, n_kv=2, hd=64, kc=P, vc=P,
            kv_type=1, n_pages=4, page_size=16, table=P, stride=2, lens=P, scale=0.125, out=P, out_stride=512,
            weights=None, ws=P, ws_bytes=1 << 30, status=None, stream=None)
EVICT = dict(kc=P, vc=P, n_pages=4, page_size=16, n_kv=2, hd=64, table=P, stride=2, lens=P, n_seqs=2, weights=P,
             keep=16, recent=4, lens_out=P, kept=None, ws=P, ws_bytes=1 << 30, status=None, stream=None)
VERIFY = dict(target=P, draft=P, type=0, tokens=P, draft_lens=None, n_seqs=2, n_draft=3, vocab=100, temperature=P,
              uniforms=P, accepted=P, out=P, logprobs=None, ws=P, ws_bytes=1 << 30, stream=None)

GEOMETRY = [(dict(hd=96), "head_dim"), (dict(n_kv=0), "n_kv"), (dict(page_size=24), "power of two"),
            (dict(page_size=4), "power of two"), (dict(page_size=8192), "power of two"), (dict(n_pages=0), "nonzero"),
            (dict(stride=0), "nonzero"), (dict(stride=1 << 21), "2\\^24"), (dict(table=P + 2), "aligned"),
            (dict(kc=P + 8), "aligned"), (dict(vc=P + 8), "aligned"), (dict(kc=None), "null"),
            (dict(table=None), "null"), (dict(lens=None), "null"), (dict(n_seqs=1 << 20), "2\\^20")]


@pytest.mark.parametrize("change,match", GEOMETRY + [
    (dict(n_heads=7), "multiple of n_kv"), (dict(n_heads=0), "multiple of n_kv"), (dict(rope_dim=66), "rope_dim"),
    (dict(rope_dim=63), "rope_dim"), (dict(cos=None), "null"), (dict(qkv=None), "null"), (dict(q_type=3), "type"),
    (dict(kv_type=0), "type"), (dict(q_type=2), "cache's type"), (dict(qkv=P + 4), "aligned"),
    (dict(q_out=P + 8), "aligned"), (dict(n_new=1 << 30), "too many rows"),
    (dict(n_new=1 << 23), "too many rows"), (dict(n_new=1 << 23, rope_dim=32), "too many rows")])
def test_rope_kv_refuses(native, change, match):
    from camelid_amd._native import HipError
    with pytest.raises(HipError, match="paged_rope_kv: .*" + match):
        _check(native.camelid_hip_paged_rope_kv(*{**ROPE, **change}.values()))


@pytest.mark.parametrize("change,match", GEOMETRY + [
    (dict(n_heads=7), "multiple of n_kv"), (dict(n_new=9), "at most 8"), (dict(q_type=3), "type"),
    (dict(kv_type=0), "type"), (dict(q_type=2), "cache's type"), (dict(scale=float("nan")), "finite"),
    (dict(scale=float("inf")), "finite"), (dict(q_stride=508), "q_stride"), (dict(out_stride=514), "q_stride"),
    (dict(q=P + 4), "aligned"), (dict(ws=None), "null"), (dict(ws=P + 4), "aligned"), (dict(out=None), "null"),
    (dict(ws_bytes=0), "workspace too small"), (dict(weights=P + 1), "aligned"),
    (dict(n_seqs=1 << 19, n_new=8), "too many rows"), (dict(n_seqs=1 << 18, stride=1 << 19, weights=P), "too many rows"),
    (dict(n_seqs=1 << 18, stride=1 << 20, ws_bytes=1 << 60), "too large for one call")])
def test_attention_refuses(native, change, match):
    from camelid_amd._native import HipError
    with pytest.raises(HipError, match="paged_attention: .*" + match):
        _check(native.camelid_hip_paged_attention(*{**ATTN, **change}.values()))


@pytest.mark.parametrize("change,match", GEOMETRY + [
    (dict(keep=0), "keep"), (dict(recent=17), "recent"), (dict(weights=None), "null"), (dict(lens_out=None), "null"),
    (dict(ws_bytes=0), "workspace too small"), (dict(ws=P + 4), "aligned"), (dict(kept=P + 2), "aligned"),
    (dict(n_seqs=1 << 19, keep=1 << 12, ws_bytes=1 << 60), "too large for one call")])
def test_evict_refuses(native, change, match):
    from camelid_amd._native import HipError
    with pytest.raises(HipError, match="paged_evict: .*" + match):
        _check(native.camelid_hip_paged_evict(*{**EVICT, **change}.values()))


@pytest.mark.parametrize("change,match", [
    (dict(target=None), "null"), (dict(tokens=None), "null"), (dict(n_draft=32), "at most 31"),
    (dict(vocab=0), "vocab"), (dict(vocab=1 << 25), "vocab"), (dict(type=5), "type"), (dict(target=P + 2), "aligned"),
    (dict(draft=P + 1, type=1), "aligned"), (dict(ws_bytes=0), "workspace too small"), (dict(ws=P + 4), "aligned"),
    (dict(n_seqs=70000), "65535")])
def test_verify_refuses(native, change, match):
    from camelid_amd._native import HipError
    with pytest.raises(HipError, match="verify_drafts: .*" + match):
        _check(native.camelid_hip_verify_drafts(*{**VERIFY, **change}.values()))


@pytest.mark.parametrize("scale", [2.4e38, -3.4e38])
@pytest.mark.parametrize("kind", [1, 2])
def test_attention_refuses_scales_beyond_the_exponent_of_16_bit_rows(native, scale, kind):
    """Scores are taken in powers of two: for 16-bit q scale times log2(e) has to be an f32 too."""
    from camelid_amd._native import HipError
    change = {"scale": scale, "q_type": kind, "kv_type": kind}
    with pytest.raises(HipError, match="paged_attention: .*log2"):
        _check(native.camelid_hip_paged_attention(*{**ATTN, **change}.values()))


def test_attention_refuses_batches_that_its_plan_cannot_serve(native):
    """Every workgroup reads all lengths: batches whose plan alone takes seconds are refused."""
    from camelid_amd._native import HipError
    with pytest.raises(HipError, match="paged_attention: .*65535 sequences"):
        _check(native.camelid_hip_paged_attention(*{**ATTN, "n_seqs": 65536}.values()))


def test_empty_calls_do_nothing(native):
    """No sequences, or no new tokens: success without a launch."""
    _check(native.camelid_hip_paged_rope_kv(*{**ROPE, "n_seqs": 0}.values()))
    _check(native.camelid_hip_paged_rope_kv(*{**ROPE, "n_new": 0}.values()))
    _check(native.camelid_hip_paged_attention(*{**ATTN, "n_seqs": 0}.values()))
    _check(native.camelid_hip_paged_attention(*{**ATTN, "n_new": 0}.values()))
    _check(native.camelid_hip_paged_evict(*{**EVICT, "n_seqs": 0}.values()))
    _check(native.camelid_hip_verify_drafts(*{**VERIFY, "n_seqs": 0}.values()))


def test_workspaces_grow_with_the_call(native):
    """A workspace for the largest call serves every smaller one."""
    at = native.camelid_hip_paged_attention_workspace
    big = at(8, 8, 32, 8, 128, 16, 100, 1)
    for s, n, stride, w in [(1, 1, 100, 0), (8, 8, 3, 1), (8, 1, 100, 1), (3, 5, 50, 0), (8, 8, 100, 0)]:
        assert 0 < at(s, n, 32, 8, 128, 16, stride, w) <= big
    ev = native.camelid_hip_paged_evict_workspace
    assert 0 < ev(1, 8, 16, 10, 7) <= ev(4, 8, 16, 100, 64)
    vd = native.camelid_hip_verify_drafts_workspace
    assert 0 < vd(1, 0, 10) <= vd(4, 5, 1000) <= vd(9, 31, 200000)
