"""Sizes of a paged cache whose products do not fit 64 bits are refused like others that are too large (nothing is launched: the pointers are made up)."""
import pytest

import capi
import capi_paged as cp
from test_paged_host import append, attend, pages


@pytest.mark.parametrize("page_type", [None, cp.FP8_E4M3], ids=["16", "e4m3"])
@pytest.mark.parametrize("change", [dict(stride_row=1 << 60), dict(stride_row=1 << 62), dict(stride_row=(1 << 60) + 128), dict(page_size=1024, stride_row=1 << 54),
                                    dict(pages_per_seq=1 << 60), dict(pages_per_seq=(1 << 60) + 4), dict(page_size=1024, pages_per_seq=1 << 54)])
def test_products_beyond_64_bits(change, page_type):
    for call in (attend, append):
        assert call(page_type=page_type, pg=pages(**change)) == capi.EINVAL
        assert "2^30" in capi.last_error()


@pytest.mark.parametrize("page_size", [16, 1024])
def test_the_largest_are_taken(page_size):
    """No sequences: the checks alone."""
    pg = pages(page_size=page_size, stride_row=(1 << 30) // page_size - 16, pages_per_seq=(1 << 30) // page_size, stride_head=1 << 30, stride_page=1 << 31)
    for page_type in (None, cp.FP8_E4M3):
        assert attend(page_type=page_type, pg=pg, n_seqs=0) == capi.OK and append(page_type=page_type, pg=pg, n_seqs=0) == capi.OK
