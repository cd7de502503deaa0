"""Calls so large that the number of their threads passes 64 bits are refused like any that is too large, before any HIP call
(pointers are addresses that are never read)."""
import pytest

from test_serving8_refusals import ROPE as ROPE8, _refuses
from test_serving_refusals import ROPE


# (threads: powers of two from 2^64 on, which leave nothing in 64 bits)
@pytest.mark.parametrize("change", [dict(n_seqs=1 << 20, n_kv=1, n_heads=4088, n_new=(1 << 32) - 16),
                                    dict(n_seqs=1 << 20, n_kv=1, n_heads=4094, n_new=(1 << 32) - 16, rope_dim=32)])
def test_8_bit_store_refuses(native, change):
    _refuses(native.camelid_hip_paged8_rope_kv, ROPE8, change, "paged8_rope_kv: .*too many rows")


@pytest.mark.parametrize("change", [dict(n_seqs=1 << 20, n_kv=1, n_heads=4095, n_new=1 << 26),
                                    dict(n_seqs=1 << 20, n_kv=1, n_heads=4095, n_new=1 << 26, rope_dim=32)])
def test_16_bit_store_refuses(native, change):
    _refuses(native.camelid_hip_paged_rope_kv, ROPE, change, "paged_rope_kv: .*too many rows")
