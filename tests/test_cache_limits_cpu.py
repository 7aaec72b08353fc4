"""CPU tests of the sizes at which the cache's entry points refuse a call: those whose index arithmetic would not
hold.  No call here reaches a device: what is not refused by its sizes ends at the check for one."""
import pytest

from test_cache_cpu import append, attention, cache, rotary

DIM_RANGE, DEVICE, CUDA = 4, 13, 14


@pytest.fixture(autouse=True)
def _no_device():
    """The addresses of these calls are not real: with a device they would be used."""
    import torch
    if torch.cuda.is_available():
        pytest.skip("for machines without a GPU")


@pytest.mark.parametrize("page_size", [16, 32, 64, 128, 256])
def test_a_table_is_refused_where_its_tokens_rounded_up_pass_32_bits(page_size):
    most = ((1 << 31) - 1024) // page_size
    for pages, refused in ((most, False), (most + 1, True), ((1 << 31) // page_size - 1, True), ((1 << 31) // page_size, True)):
        st, err = attention(cache(page_size=page_size), table_pages=pages)
        if refused:
            assert st == DIM_RANGE and "table_pages * page_size" in err, (pages, st, err)
        else:
            assert st in (DEVICE, CUDA), (pages, st, err)


@pytest.mark.parametrize("tokens", [1 << 31, 1 << 61, 1 << 62, (1 << 63) - 1])
def test_counts_whose_product_wraps_around_are_refused(tokens):
    """tokens * heads in 64 bits may come out small, or negative, for counts of this size."""
    from w4a16_opt import capi
    import ctypes
    for heads in (1, 2, 4, 8, 1024):
        st, err = append(cache(kv_heads=heads), tokens=tokens)
        assert st == DIM_RANGE and "fit in int32" in err
        st, err = append(cache(kv_heads=heads), tokens=tokens, rot=rotary(q_heads=3 * heads))
        assert st == DIM_RANGE and "fit in int32" in err
        st, err = attention(cache(kv_heads=heads), q_tokens=tokens, q_heads=4 * heads)
        assert st == DIM_RANGE and "fit in int32" in err
        lib = capi.load()
        c = cache(kv_heads=heads)
        assert lib.w4a16_cache_read(ctypes.byref(c), 0x10000, tokens, 0x10000, 0x10000, 0, None) == DIM_RANGE


def test_a_negative_number_of_query_heads_does_not_widen_the_limit():
    """tokens * (kv_heads + q_heads) with q_heads < 0 came out small before q_heads was looked at."""
    st, err = append(tokens=1 << 40, rot=rotary(q_heads=-2))
    assert st in (DIM_RANGE, 19), (st, err)
