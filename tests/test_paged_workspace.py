"""Workspace of the attention over a paged cache, without a GPU (256 units are assumed there): it goes by the partial results that a launch can
leave, not by the most that every row could have."""
import pytest

import capi_paged as cp

WAVES, UNITS = 2048, 256


@pytest.mark.parametrize("n,Hq,Hkv,D,tokens", [(65, 32, 8, 128, 1), (256, 64, 8, 128, 1), (256, 64, 8, 128, 2), (512, 64, 8, 128, 1), (1024, 32, 8, 128, 1),
                                               (4096, 32, 8, 128, 1), (4096, 32, 8, 64, 4), (300, 48, 1, 128, 1), (70, 40, 2, 64, 1)])
def test_line(n, Hq, Hkv, D, tokens):
    """A share and a pair are one partial result more, each; a partial result is the columns of a group, D sums and two numbers for each."""
    columns = Hq // Hkv * tokens
    groups, per_part = (columns + 15) // 16, min(columns, 16)
    need = (WAVES + n * Hkv * groups) * per_part * (D + 2) * 4 + (n + 2) * 4
    got = {cp.lib().minfer_flash_attn_paged_workspace_bytes(n, n * tokens, Hq, Hkv, D, rows, tokens) for rows in (4096, 1 << 17, 1 << 20)}
    assert len(got) == 1 and need <= got.pop() <= need + 3 * 256


@pytest.mark.parametrize("n,Hq,Hkv,D,rows", [(1, 8, 2, 64, 1 << 20), (4, 32, 8, 128, 1 << 17), (64, 32, 8, 128, 512), (16, 48, 1, 128, 4096)])
def test_chunks(n, Hq, Hkv, D, rows):
    """A workgroup of one or two rounds is a partial result at most."""
    per_part = min(Hq // Hkv, 16)
    rounds = 1 if n * Hkv * ((Hq // Hkv + 15) // 16) <= UNITS else 2
    assert cp.lib().minfer_flash_attn_paged_workspace_bytes(n, n, Hq, Hkv, D, rows, 1) <= rounds * UNITS * per_part * (D + 2) * 4 + 3 * 256
