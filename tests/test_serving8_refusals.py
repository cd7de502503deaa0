"""The 8-bit cache, its pages and logits: argument checks of the C entry points.  Every refusal comes before any HIP
call, so these run without a GPU (pointers are addresses that are never read)."""
import ctypes as C

import pytest

P = 4096  # an aligned address


def _check(rc):
    from camelid_amd._native import check
    check(rc)


ROPE = dict(qkv=P, n_seqs=2, n_new=1, new_lens=None, n_heads=8, n_kv=2, hd=64, rope_dim=64, split_half=0, cos=P, sin=P,
            q_norm=None, k_norm=None, eps=1e-5, q_out=P, q_type=0, kc=P, vc=P, k_exp=P + 1, v_exp=P + 3, kv_type=3,
            n_pages=4, page_size=16, table=P, stride=2, lens=P, status=None, stream=None)
READ = dict(kc=P, vc=P, k_exp=P, v_exp=P, kv_type=4, n_pages=4, page_size=16, n_kv=2, hd=64, table=P, stride=2, lens=P,
            n_seqs=2, k_out=P, v_out=P, out_type=0, out_positions=20, status=None, stream=None)
ATTN = dict(q=P, q_type=0, q_stride=512, n_seqs=2, n_new=1, new_lens=None, n_heads=8, n_kv=2, hd=64, kc=P, vc=P, k_exp=P,
            v_exp=P, kv_type=3, n_pages=4, page_size=16, table=P, stride=2, lens=P, scale=0.125, out=P, out_stride=512,
            ws=P, ws_bytes=1 << 30, status=None, stream=None)
RESERVE = dict(table=P, stride=4, held=P, n_seqs=2, first=P, lens=P, page_size=16, refs=P, n_pages=8, pairs=P, max_pairs=2,
               n_pairs=P, granted=None, ws=P, ws_bytes=1 << 20, status=None, stream=None)
FORK = dict(table=P, stride=4, held=P, n_seqs=2, parents=P, children=P, n_forks=1, lens=None, page_size=16, refs=P, n_pages=8,
            status=None, stream=None)
COMPACT = dict(table=P, stride=4, held=P, n_seqs=2, refs=P, n_pages=8, table_out=P, refs_out=P, pairs=P, max_pairs=2, n_pairs=P,
               extent=None, ws=P, ws_bytes=1 << 20, status=None, stream=None)
LOGITS = dict(logits=P, in_stride=100, out=P, out_stride=100, type=0, n_seqs=2, n_rows=3, vocab=100, history=P, history_stride=9,
              history_lens=None, prompt_lens=None, drafts=P, draft_lens=None, rep=P, freq=P, pres=P, bias_tokens=P,
              bias_values=P, bias_stride=4, bias_lens=None, mask=P, mask_stride=4, stream=None)

GEOMETRY = [(dict(hd=96), "head_dim"), (dict(n_kv=0), "n_kv"), (dict(page_size=24), "16..=4096"),
            (dict(page_size=8), "16..=4096"), (dict(page_size=8192), "16..=4096"), (dict(n_pages=0), "nonzero"),
            (dict(stride=0), "nonzero"), (dict(stride=1 << 21), "2\\^24"), (dict(table=P + 2), "aligned"),
            (dict(kc=P + 8), "aligned"), (dict(vc=P + 8), "aligned"), (dict(kc=None), "null"), (dict(k_exp=None), "null"),
            (dict(v_exp=None), "null"), (dict(table=None), "null"), (dict(lens=None), "null"), (dict(n_seqs=1 << 20), "2\\^20"),
            (dict(kv_type=1), "type"), (dict(kv_type=5), "type")]


def _refuses(call, base, change, match):
    from camelid_amd._native import HipError
    with pytest.raises(HipError, match=match):
        _check(call(*{**base, **change}.values()))


@pytest.mark.parametrize("change,match", GEOMETRY + [
    (dict(n_heads=7), "multiple of n_kv"), (dict(n_heads=0), "multiple of n_kv"), (dict(rope_dim=66), "rope_dim"),
    (dict(rope_dim=63), "rope_dim"), (dict(cos=None), "null"), (dict(qkv=None), "null"), (dict(q_type=3), "type"),
    (dict(qkv=P + 4), "aligned"), (dict(q_out=P + 8), "aligned"), (dict(k_norm=P + 2), "aligned"),
    (dict(n_new=1 << 28), "too many rows"), (dict(n_new=1 << 27, rope_dim=32), "too many rows")])
def test_store_refuses(native, change, match):
    _refuses(native.camelid_hip_paged8_rope_kv, ROPE, change, "paged8_rope_kv: .*" + match)


@pytest.mark.parametrize("change,match", GEOMETRY + [
    (dict(k_out=None), "null"), (dict(v_out=P + 8), "aligned"), (dict(out_type=3), "type"),
    (dict(n_seqs=1 << 19, stride=1 << 19, out_positions=1 << 23), "too many positions")])
def test_read_refuses(native, change, match):
    _refuses(native.camelid_hip_paged8_read, READ, change, "paged8_read: .*" + match)


@pytest.mark.parametrize("change,match", GEOMETRY + [
    (dict(n_heads=7), "multiple of n_kv"), (dict(q_type=3), "type"), (dict(scale=float("nan")), "finite"),
    (dict(scale=float("inf")), "finite"), (dict(q_stride=508), "q_stride"), (dict(out_stride=514), "q_stride"),
    (dict(q_type=2, q_stride=516), "q_stride"), (dict(q=P + 4), "aligned"), (dict(ws=None), "null"), (dict(ws=P + 4), "aligned"),
    (dict(out=None), "null"), (dict(ws_bytes=0), "workspace too small"), (dict(new_lens=P + 1), "aligned"),
    (dict(n_seqs=1 << 19, n_new=1 << 6, ws_bytes=1 << 60), "too many rows"),
    (dict(n_heads=4096, n_kv=1, q_stride=1 << 18, out_stride=1 << 18, n_new=300, ws_bytes=1 << 60), "too many rows"),
    (dict(n_seqs=1 << 18, stride=1 << 20, ws_bytes=1 << 60), "too large for one call"),
    (dict(n_seqs=65536, ws_bytes=1 << 60), "65535")])
def test_attention_refuses(native, change, match):
    _refuses(native.camelid_hip_paged8_attention, ATTN, change, "paged8_attention: .*" + match)


PAGES = [(dict(table=None), "null"), (dict(held=None), "null"), (dict(refs=None), "null"), (dict(stride=0), "nonzero"),
         (dict(n_pages=0), "nonzero"), (dict(n_pages=1 << 31), "below 2\\^31"), (dict(stride=1 << 31), "below 2\\^31"),
         (dict(n_seqs=(1 << 20) + 1, stride=1), "2\\^20"), (dict(table=P + 2), "aligned"), (dict(status=P + 1), "aligned")]


@pytest.mark.parametrize("change,match", PAGES + [
    (dict(lens=None), "null"), (dict(ws=None), "null"), (dict(n_pairs=None), "null"), (dict(pairs=None), "null"),
    (dict(page_size=4), "page_size"), (dict(page_size=48), "page_size"), (dict(ws=P + 8), "aligned"),
    (dict(granted=P + 2), "aligned"), (dict(ws_bytes=100), "workspace too small")])
def test_reserve_refuses(native, change, match):
    _refuses(native.camelid_hip_pages_reserve, RESERVE, change, "pages_reserve: .*" + match)


@pytest.mark.parametrize("change,match", PAGES + [
    (dict(parents=None), "null"), (dict(children=None), "null"), (dict(n_forks=3), "more forks"), (dict(page_size=0), "page_size"),
    (dict(children=P + 2), "aligned")])
def test_fork_refuses(native, change, match):
    _refuses(native.camelid_hip_pages_fork, FORK, change, "pages_fork: .*" + match)


@pytest.mark.parametrize("change,match", PAGES + [
    (dict(table_out=None), "null"), (dict(n_pairs=None), "null"), (dict(pairs=None), "null"), (dict(extent=P + 1), "aligned"),
    (dict(ws_bytes=100), "workspace too small")])
def test_compact_refuses(native, change, match):
    _refuses(native.camelid_hip_pages_compact, COMPACT, change, "pages_compact: .*" + match)


@pytest.mark.parametrize("change,match", [
    (dict(buffers=None), "null"), (dict(sizes=None), "null"), (dict(pairs=None), "null"), (dict(n_pages=0), "n_pages"),
    (dict(n_pages=1 << 31), "n_pages"), (dict(pairs=P + 2), "aligned"), (dict(hole=True), "null")])
def test_copy_refuses(native, change, match):
    from camelid_amd._native import HipError
    where = (C.c_void_p * 2)(P, None if change.pop("hole", False) else P)
    a = {**dict(buffers=where, sizes=(C.c_size_t * 2)(64, 64), n=2, n_pages=4, pairs=P, max_pairs=2, n_pairs=None, status=None,
                stream=None), **change}
    with pytest.raises(HipError, match="pages_copy: .*" + match):
        _check(native.camelid_hip_pages_copy(*a.values()))


@pytest.mark.parametrize("change,match", [
    (dict(logits=None), "null"), (dict(out=None), "null"), (dict(bias_values=None), "null"), (dict(n_rows=33), "32 rows"),
    (dict(vocab=0), "vocab"), (dict(vocab=(1 << 24) + 1, in_stride=1 << 25, out_stride=1 << 25), "vocab"), (dict(type=3), "type"),
    (dict(in_stride=99), "strides"), (dict(out=2 * P, out_stride=99), "strides"), (dict(out_stride=101), "in place"),
    (dict(mask_stride=3), "mask_stride"), (dict(history_stride=(1 << 28) + 1), "history_stride"),
    (dict(bias_stride=16385), "bias_stride"), (dict(logits=P + 2, out=P + 2), "aligned"), (dict(type=1, logits=P + 1, out=P + 1), "aligned"),
    (dict(mask=P + 1), "aligned"), (dict(drafts=P + 2), "aligned"),
    (dict(n_seqs=1 << 20, vocab=1 << 24, in_stride=1 << 24, out_stride=1 << 24, mask_stride=1 << 20), "too many rows")])
def test_adjust_logits_refuses(native, change, match):
    _refuses(native.camelid_hip_adjust_logits, LOGITS, change, "adjust_logits: .*" + match)


def test_empty_calls_do_nothing(native):
    for call, base, change in ((native.camelid_hip_paged8_rope_kv, ROPE, dict(n_seqs=0)),
                               (native.camelid_hip_paged8_rope_kv, ROPE, dict(n_new=0)),
                               (native.camelid_hip_paged8_read, READ, dict(out_positions=0)),
                               (native.camelid_hip_paged8_attention, ATTN, dict(n_seqs=0)),
                               (native.camelid_hip_paged8_attention, ATTN, dict(n_new=0)),
                               (native.camelid_hip_pages_reserve, RESERVE, dict(n_seqs=0)),
                               (native.camelid_hip_pages_fork, FORK, dict(n_forks=0)),
                               (native.camelid_hip_adjust_logits, LOGITS, dict(n_rows=0))):
        _check(call(*{**base, **change}.values()))
    _check(native.camelid_hip_pages_copy(None, None, 0, 4, None, 2, None, None, None))
