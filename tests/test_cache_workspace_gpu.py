"""GPU test of the attention's workspace: it does not grow with the queries of a call without bound."""
import ctypes

import pytest

pytestmark = pytest.mark.gpu


def workspace(batch, max_q, q_heads, kv_heads, table_pages, head_dim=128, page_size=64, q_tokens=None):
    from w4a16_opt import capi
    lib = capi.load()
    c = capi.Cache(data=None, num_pages=1 << 20, page_size=page_size, kv_heads=kv_heads, head_dim=head_dim, group_size=head_dim)
    a = capi.CacheAttentionArgs(q_tokens=batch * max_q if q_tokens is None else q_tokens, scale=0.1, dtype=0, q_heads=q_heads,
                                batch=batch, table_pages=table_pages, max_q=max_q, causal=1, window=0)
    n = ctypes.c_uint64()
    capi.check(lib.w4a16_cache_attention_workspace(ctypes.byref(c), ctypes.byref(a), ctypes.byref(n)), lib)
    return n.value


@pytest.mark.parametrize("batch,max_q,q_heads,kv_heads,tokens", [
    (1024, 16, 64, 8, 4096), (1024, 16, 64, 8, 16), (256, 128, 32, 32, 128), (256, 128, 32, 32, 8192), (60000, 33, 32, 32, 4096),
    (64, 16, 64, 8, 131072), (1, 40, 8, 1, 131072), (1, 30000, 64, 8, 131072), (8, 4096, 32, 8, 4096)])
def test_workspace_is_bounded(cuda_device, batch, max_q, q_heads, kv_heads, tokens):
    assert workspace(batch, max_q, q_heads, kv_heads, tokens // 16, page_size=16) <= 256 << 20


def test_a_call_whose_sequences_have_up_to_128_rows_each_needs_none(cuda_device):
    """Enough sequences for every SM: nothing is split over CTAs, so nothing passes through memory."""
    assert workspace(256, 128, 32, 32, 8) == 0
