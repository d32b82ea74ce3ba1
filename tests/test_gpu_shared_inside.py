"""Attention of groups that share a prefix where some tokens stand inside it: found by their place in cu_seqlens, whatever the number of sequences beside them."""
import pytest
import torch

from test_gpu_shared import DEV, QT, Shared, check, queries
from test_gpu_shared_depth import for_groups

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("D", [64, 128])
def test_sequences_inside_and_without_tokens(kerns, eight, D):
    """Tokens inside the prefix, behind it and none at all in any order, in the second of three groups; the batch padded behind them, with entries that fall."""
    r = torch.Generator().manual_seed(D)
    new = torch.randint(0, 4, (150,), generator=r).tolist()
    past = [int(x) if i % 3 else 384 + int(x) // 8 for i, x in enumerate(torch.randint(0, 380, (150,), generator=r))]
    lens = [(2, 300), (1, 70)] + [(3, 420)] + list(zip(new, past)) + [(0, 200), (1, 200), (2, 210)] + [(0, 0)] * 5
    groups = [(0, 2, 64), (2, 153, 384), (153, 161, 192)]
    c = Shared(lens, [(0, 2, 64), (2, 153, 384), (154, 156, 192)], 16, 2, D, torch.float16, eight=eight, told=[64, 384, 192])
    c.cu_groups = [0, 2, 154, 161]   # the one sequence without tokens in the second group, those behind the last token in the third
    for_groups(c, 8, 3)
    want = check(kerns, c, 8, torch.float16)
    q, n = queries(c, 8, torch.float16), len(lens)
    for tail in ([0] * 5, [c.T, c.T, 3, 0, 0], [c.T + 9] * 5, [7, 5, 4, 2, 1]):
        assert torch.equal(c.call(kerns, q, cu=c.cu_list[:n - 4] + tail), want)
    # the second group reaches to the end: what is behind its last token says nothing
    lens = lens[:-8] + [(0, 0)] * 5
    c = Shared(lens, groups[:2], 16, 2, D, torch.float16, eight=eight)
    c.cu_groups, n = [0, 2, len(lens)], len(lens)
    want = check(kerns, c, 8, torch.float16)
    q = queries(c, 8, torch.float16)
    for tail in ([0] * 5, [c.T, c.T, 3, 0, 0], [7, 5, 4, 2, 1]):
        assert torch.equal(c.call(kerns, q, cu=c.cu_list[:n - 4] + tail), want)


def time_of(f):
    f()
    times = []
    for _ in range(7):
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        start.record()
        f()
        end.record()
        end.synchronize()
        times.append(start.elapsed_time(end))
    return sorted(times)[3]


def test_one_sequence_inside_beside_thousands(kerns):
    """A search along the sequences for every token was 2.0 ms where the call without it took 0.13."""
    n, page, rows, Hq, Hkv, D = 4000, 64, 1024, 8, 1, 128
    width = rows // page + 2
    g = torch.Generator(device=DEV).manual_seed(0)
    table = rows // page + torch.arange(2 * n, device=DEV, dtype=torch.int32).view(n, 2)
    table = torch.cat((torch.arange(rows // page, device=DEV, dtype=torch.int32).expand(n, -1), table), 1).contiguous()
    k, v = (torch.randn(rows // page + 2 * n, Hkv, page, D, generator=g, device=DEV).half() for _ in range(2))
    q = torch.randn(1, n, Hq, D, generator=g, device=DEV).half().transpose(1, 2)
    cu, ctx = torch.arange(n + 1, dtype=torch.int32, device=DEV), torch.full((n,), rows + 65, dtype=torch.int32, device=DEV)
    groups, told = torch.tensor([0, n], dtype=torch.int32, device=DEV), torch.tensor([rows], dtype=torch.int32, device=DEV)
    assert table.shape[1] == width
    times, outs = [], []
    for inside in (0, 1):
        ctx[n // 2] = rows - 300 if inside else rows + 65
        out, plain = torch.empty_like(q), torch.empty_like(q)
        times.append(time_of(lambda: kerns.flash_attn_paged_shared(*QT[q.dtype], q, k, v, table, cu, ctx, groups, told, 1, out)))
        kerns.flash_attn_paged(*QT[q.dtype], q, k, v, table, cu, ctx, 1, plain)
        # (two kernels whose weights are rounded by 2^-11 each: 2 x 2 x 2^-11 of sums of w |v|, which are 0.8)
        torch.testing.assert_close(out, plain, atol=2e-3, rtol=2e-3)
        outs.append(out)
    assert not torch.allclose(outs[0][:, :, n // 2], outs[1][:, :, n // 2], atol=2e-3)
    assert times[1] < 4 * times[0]
