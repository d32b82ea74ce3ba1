"""Attention of groups that share a prefix where a workgroup's or a wave's share is long: the rings of tiles and of groups of rows go round several times, with
pages that are missing and rows that are no numbers deep inside; and combinations of columns, groups, layouts and captured calls."""
import pytest
import torch

import capi_serving as cs
import paged_ref as ref
from test_gpu_shared import DEV, QT, Shared, check, queries

pytestmark = pytest.mark.gpu
PARTS = 61   # a row has no more than 64 partial results, of which three are ends: a share is longer than what there is of a block or a sequence divided by this


def for_groups(c, Hq, most):
    """The kernels that know of groups take the call: their workspace is not the other ones'."""
    lib, rows = cs.lib(), c.width * c.page
    args = (c.T, Hq, c.Hkv, c.D, rows, most)
    assert lib.minfer_flash_attn_paged_shared_workspace_bytes(len(c.seqs), len(c.told), *args) > lib.minfer_flash_attn_paged_workspace_bytes(len(c.seqs), *args)


# (sequences, tokens of each at most, query heads of the one KV head): 4 columns and, for groups of 16 columns in pairs, 24 and 40
COLUMNS = [(3, 1, 4), (4, 3, 8), (4, 5, 8)]


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n,most,Hq", COLUMNS[:2])
@pytest.mark.parametrize("holes", [False, True])
def test_long_prefixes(kerns, eight, D, n, most, Hq, holes):
    rows, page = 24000, 16 if holes else 64
    assert rows // 64 // PARTS + 1 >= 7   # tiles of a share, of which four are on their way
    # (pages of tiles here and there and of whole tiles, beside each other and at every distance from a share's first)
    gone = {(0, i) for t in (0, 1, 9, 52, 101, 102, 103, 147, 201, 262, 317, 374) for i in range(4 * t + t % 3, 4 * t + 4)} if holes else ()
    c = Shared([(1 + i % most, rows + 7 * i) for i in range(n)], [(0, n, rows)], page, 1, D, torch.bfloat16 if holes else torch.float16, eight=eight, gone=gone, seed=D)
    for_groups(c, Hq, max(q for q, _ in c.seqs))
    check(kerns, c, Hq, c.dtype)


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n,most,Hq", COLUMNS)
def test_long_own_rows(kerns, eight, D, n, most, Hq):
    group = 32 if eight else 16
    own = 8 * PARTS * group
    assert own // group // PARTS + 1 >= 9   # groups of a share, of which two are on their way
    lens = [(1 + (i * 3) % most, 128 + own - 400 * i) for i in range(n - 1)] + [(most, 140)]
    gone = {(1, i) for i in (40, 41, 200, 201, 202, 203, 204, 205, 206, 207, 208)} | {(0, 8 + 5 * i) for i in range(30)}
    c = Shared(lens, [(0, n, 128)], 16, 1, D, torch.float16 if D == 64 else torch.bfloat16, eight=eight, gone=gone, seed=most)
    for_groups(c, Hq, most)
    check(kerns, c, Hq, c.dtype)


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("row", [12345, 20031, 23999])
def test_a_row_of_no_numbers_deep_inside_a_prefix(kerns, eight, D, row):
    """A NaN of V inside the prefix, which some sequences' tokens stand behind, some in front of and some around."""
    rows = 24000
    lens = [(1, rows + 5), (3, row - 1), (2, 300), (1, row - 64 if row < 23999 else 16001), (2, row + 40 if row < 23900 else row)]
    make = lambda: Shared(lens, [(0, 5, rows)], 32, 2, D, torch.float16, eight=eight, seed=7)
    c, clean = make(), make()
    for_groups(c, 4, 3)
    q = queries(clean, 4, torch.float16)
    want, bound = ref.attend(clean, q[0].cpu())
    raw = c.v_pages.view(torch.uint8) if eight else c.v_pages
    raw[c.table_list[0][row // 32], 1, row % 32, 9] = 0x7F if eight else float("nan")
    out = c.call(kerns, q)[0].cpu().double()
    position = torch.tensor([past + i for n, past in lens for i in range(n)])
    hit = torch.zeros(4, c.T, D, dtype=torch.bool)
    hit[2:, position >= row, 9] = True
    assert 0 < int(hit.any(0).any(-1).sum()) < c.T
    assert torch.equal(torch.isnan(out), hit)
    assert ((out - want).abs() <= bound)[~hit].all()


@pytest.mark.parametrize("order", ["heads", "rows"])
@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("D", [64, 128])
def test_drafts_of_several_groups(kerns, order, eight, D):
    """More than 16 columns with groups of different prefixes, sequences without a group, tokens inside the prefix and holes in it, in both layouts of a pool."""
    lens = [(2, 30), (3, 0)] + [(1 + i % 6, 300 + 50 * i) for i in range(9)] + [(6, 100), (5, 640), (1, 900), (6, 3), (4, 639), (6, 1500), (2, 700), (3, 650), (6, 64)] + [(6, 500)]
    gone = {(2, 3), (2, 4), (11, 4), (12, 5), (12, 6), (4, 20), (16, 60)}
    groups = [(2, 11, 288), (11, 12, 0), (12, 20, 640)]   # (a group begins where the one in front of it ends: a sequence between two that shares nothing is one without a prefix)
    c = Shared(lens, groups, 16, 2, D, torch.float16, order=order, eight=eight, gone=gone, gap=3)
    for_groups(c, 8, 6)
    check(kerns, c, 8, torch.float16)


@pytest.mark.parametrize("most", [1, 6])
def test_many_groups_over_codes(kerns, most):
    """More groups than are looked up at once, of three sequences each."""
    lens = [(1 + (s * 5) % most, 128 + (11 * s) % 50) for s in range(213)]
    c = Shared(lens, [(3 * i, 3 * i + 3, 128 - 64 * (i % 2)) for i in range(70)], 16, 2, 64, torch.bfloat16, eight=True)
    for_groups(c, 8, most)
    check(kerns, c, 8, torch.bfloat16)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("most", [2, 5])
def test_a_captured_call_over_codes(kerns, D, most):
    lens = [(1 + i % most, 700 + 31 * i) for i in range(20)]
    c = Shared(lens, [(0, 12, 640), (12, 18, 300)], 32, 2, D, torch.bfloat16, eight=True)
    for_groups(c, 8, most)
    q = queries(c, 8, torch.bfloat16)
    want = check(kerns, c, 8, torch.bfloat16)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    groups, told, out = i32(c.cu_groups), i32(c.told), torch.zeros_like(q)

    def step():
        kerns.flash_attn_paged_shared_fp8(*QT[q.dtype], q, c.k_pages, c.v_pages, c.k_scales, c.v_scales, c.table, c.cu, c.ctx, groups, told, most, out)

    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    for k in range(4):
        told.copy_(i32([640, 300] if k % 2 == 0 else [128, 0]))
        out.zero_()
        g.replay()
        got = out.clone()
        step()
        assert torch.equal(got, out)
        if k % 2 == 0:
            assert torch.equal(got, want)


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("most", [1, 3])
def test_several_blocks_of_several_groups(kerns, eight, D, most):
    """Groups of more rows than a block has, one that fills its last block to the row, one without a prefix between them: partial results of blocks, shares and groups lie side by side."""
    n = [75, 3, 64, 50] if most == 1 else [40, 3, 32, 26]
    lens = [(1 + s % most, 1000 + 3 * s) for s in range(sum(n))]
    at = [sum(n[:i]) for i in range(5)]
    c = Shared(lens, [(at[0], at[1], 960), (at[1], at[2], 0), (at[2], at[3], 512), (at[3], at[4], 768)], 64, 2, D, torch.bfloat16, eight=eight)
    for_groups(c, 16, most)
    check(kerns, c, 16, torch.bfloat16)
