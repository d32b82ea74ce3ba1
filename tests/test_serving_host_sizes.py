"""Host side of the operators of a serving step, without a GPU: calls whose worst case is past what the kernels for groups count, which are flash_attn_paged's."""
import pytest

import capi
import capi_serving as cs
from test_serving_host import P, shared, wide


def sizes(n_seqs, n_groups, T, Hq, Hkv, D, rows, max_q):
    """Workspaces of the call with groups, of the call without."""
    lib = cs.lib()
    return (lib.minfer_flash_attn_paged_shared_workspace_bytes(n_seqs, n_groups, T, Hq, Hkv, D, rows, max_q),
            lib.minfer_flash_attn_paged_workspace_bytes(n_seqs, T, Hq, Hkv, D, rows, max_q))


@pytest.mark.parametrize("n_seqs,n_groups,T,Hq,Hkv,D,rows,max_q", [
    (4096, 8, 4096 * 6, 32, 8, 128, 1 << 20, 6),         # drafts in tables of a million rows: a line of 2^31 places for their own rows
    (4096, 1024, 4096 * 4, 24, 8, 64, 1 << 20, 8),
    (2048, 2, 2048, 32, 8, 128, (1 << 21) - 16, 1),      # single tokens, in the few places between the two operators' bounds
])
def test_lines_past_31_bits_are_flash_attn_pageds(n_seqs, n_groups, T, Hq, Hkv, D, rows, max_q):
    with_groups, without = sizes(n_seqs, n_groups, T, Hq, Hkv, D, rows, max_q)
    assert with_groups == without
    # (half as many sequences are the kernels for groups' own)
    with_groups, without = sizes(n_seqs // 2, n_groups // 2, T // 2, Hq, Hkv, D, rows, max_q)
    assert with_groups > without


def test_what_flash_attn_paged_takes_is_not_refused():
    """The call between the bounds gets as far as its workspace; beyond both of them it is too large."""
    pages = lambda rows: wide(page_size=16, pages_per_seq=rows // 16, table_stride=rows // 16)
    big = dict(n_seqs=2048, n_groups=2, T=2048, Hq=32, Hkv=8, max_q=1, st=capi.Strides(0, 128, 4096, 0, 0, 0, 0, 128, 4096))
    assert shared(**big, pg=pages((1 << 21) - 16), ws=None) == capi.EWORKSPACE and "workspace" in capi.last_error()
    assert shared(**big, pg=pages(1 << 22), ws=P, ws_bytes=1 << 50) == capi.EINVAL and "too large" in capi.last_error()


@pytest.mark.parametrize("n_seqs,T,Hq,Hkv,D,max_q", [(4096, 4096, 32, 8, 128, 1), (4096, 4096, 8, 2, 64, 1), (1000, 4000, 32, 8, 128, 6), (600, 2400, 24, 4, 64, 4)])
def test_the_workspace_does_not_grow_with_the_groups(n_seqs, T, Hq, Hkv, D, max_q):
    """Partial results of prefixes: a row for every (token, head) and a block for each of 256 or 512 shares, whatever the number of groups; the rest is a few words a group."""
    most = n_seqs // 4
    one, many = (sizes(n_seqs, n, T, Hq, Hkv, D, 1 << 13, max_q)[0] for n in (1, most))
    assert one > sizes(n_seqs, 0, T, Hq, Hkv, D, 1 << 13, max_q)[0]
    assert many - one <= 16 * most + 256
    own = n_seqs * max_q * Hq + (2048 + 16) * min(max_q * Hq // Hkv, 32) + T * Hq + (512 // Hkv) * 128 * Hkv * (D // 64)
    assert many <= own * (D + 2) * 4 + 16 * (n_seqs + most) + 4096


@pytest.mark.parametrize("D,codes", [(64, 70), (128, 25)])
@pytest.mark.parametrize("Hq,max_q", [(32, 6), (48, 8), (64, 8)])
def test_more_columns_ask_for_longer_tables(D, codes, Hq, max_q):
    """24 to 64 columns of a KV head: partial results of each, and own rows read twice past 32, are paid for by so many rows a column of a table; below that the call is flash_attn_paged's.
    (Codes, of which fewer rows are enough: the workspace is that of either kind.)"""
    n, columns = 1500, Hq // 8 * max_q
    takes = lambda rows: (lambda x: x[0] > x[1])(sizes(n, 1, n * max_q, Hq, 8, D, rows, max_q))
    least = max(codes * columns, 600)
    assert [takes(rows) for rows in (least - 16, least)] == [False, True]


@pytest.mark.parametrize("D,rows_per_column", [(64, 100), (128, 70)])
def test_more_columns_ask_for_longer_tables_of_16_bit_rows(D, rows_per_column):
    """Which of the two operators asks for its workspace (20 sequences, whose blocks flash_attn_paged cuts, so that it asks, too)."""
    least = 48 * rows_per_column
    for rows, op in ((least - 16, "flash_attn_paged:"), (least, "flash_attn_paged_shared:")):
        pg = wide(page_size=16, pages_per_seq=rows // 16, table_stride=rows // 16)
        assert shared(pg=pg, n_seqs=20, n_groups=1, T=160, Hq=48, Hkv=8, D=D, max_q=8, st=capi.Strides(0, D, 48 * D, 0, 0, 0, 0, D, 48 * D), ws=None) == capi.EWORKSPACE
        assert capi.last_error().startswith(op)
