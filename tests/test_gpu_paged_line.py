"""Few rows per KV head over a paged cache: the line of all sequences' rows, cut into equal shares, at the lengths that its indices are made for."""
import pytest
import torch

import paged_ref as ref
from test_gpu_paged import DEV, QT, make_q

pytestmark = pytest.mark.gpu


def test_line_of_almost_2_31_groups(kerns):
    """The longest line that is not refused, 2048 pairs of up to 16.8 million rows: positions and shares that together pass 31 bits.  Of each
    context the last one or two pages are there, the same few for all sequences."""
    n, H, S, D, P = 64, 32, 1024, 64, 16383
    g = torch.Generator().manual_seed(3)
    pools = [torch.randn(4, H, S, D, generator=g).half() for _ in range(2)]
    ctx = [P * S - 300 * (s % 3) for s in range(n)]
    groups = sum((x + 15) // 16 for x in ctx) * H
    assert groups + groups // 2048 > 2 ** 31 - 1   # (2048 waves on 256 units)
    table = torch.full((n, P), -1, dtype=torch.int32)
    for s in range(n):
        table[s, P - 1] = s % 4
        if s % 5 == 0:
            table[s, P - 2] = (s + 1) % 4
    q = make_q(n, H, D, torch.float16)
    out = torch.full_like(q, 7.0)
    cu = torch.arange(n + 1, dtype=torch.int32, device=DEV)
    kerns.flash_attn_paged(*QT[q.dtype], q.transpose(1, 2), pools[0].to(DEV), pools[1].to(DEV), table.to(DEV), cu,
                           torch.tensor(ctx, dtype=torch.int32, device=DEV), 1, out.transpose(1, 2))
    torch.cuda.synchronize()
    # the same tokens behind the pages that are there alone
    short = ref.Paged([(1, 0)], S, H, D, torch.float16, "cpu")
    ids = [table[s][table[s] >= 0].tolist() for s in range(n)]
    held = [len(ids[s]) * S - (P * S - ctx[s]) for s in range(n)]
    short.seqs, short.cu_list, short.table_list = [(1, x - 1) for x in held], list(range(n)), ids
    short.k_dense, short.v_dense = ([pool[i].double().transpose(0, 1).flatten(1, 2)[:, :x] for i, x in zip(ids, held)] for pool in pools)
    want, bound = ref.attend(short, q[0].transpose(0, 1))
    ok = bool(((out[0].transpose(0, 1).double().cpu() - want).abs() <= bound).all())
    assert ok
