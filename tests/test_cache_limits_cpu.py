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
