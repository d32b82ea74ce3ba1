"""torch.library.opcheck on the operators of a serving step: what their schemas say is written, their fakes, dispatch under tracing."""
import pytest
import torch

from test_gpu_reference_recipes import OPCHECKS
from test_gpu_shared import DEV, QT, Shared, queries
from test_gpu_tables import Pool, i32
from test_gpu_verify import Case

pytestmark = pytest.mark.gpu


def test_opcheck_tables_and_release(kerns):
    c = Pool(70, 16, 100, 5, 12, 200, 3)
    n, past, held, ring, state = c.n, i32(c.past), i32(c.held), i32(c.ring), i32(c.state)
    slots = torch.full((sum(c.new),), -77, dtype=torch.int64, device=DEV)
    torch.library.opcheck(torch.ops.minfer.paged_tables.default, (16, past, i32(c.new), held, ring, state, c.tensors(), i32([0] * (n + 1)), i32([0] * n), slots, i32([0] * n), i32([0] * 3)),
                          test_utils=OPCHECKS)
    torch.library.opcheck(torch.ops.minfer.paged_release.default, (16, i32([p // 2 for p in c.past]), held, c.tensors(), ring, state, i32([0] * n), i32([0] * 3)), test_utils=OPCHECKS)


@pytest.mark.parametrize("drafter", [True, False])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_opcheck_verify_drafts(kerns, drafter, dtype):
    c = Case(5, 3, 9001, dtype, drafter)
    T = c.tokens.numel()
    torch.library.opcheck(torch.ops.minfer.verify_drafts.default,
                          (c.tokens.to(DEV), i32(c.cu), c.target.to(DEV), c.draft.to(DEV) if drafter else None, c.accept_u.to(DEV), c.sample_u.to(DEV),
                           torch.zeros(T, dtype=torch.int64, device=DEV), i32([0] * 5)), test_utils=OPCHECKS)


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("wide", [False, True])
def test_opcheck_shared(kerns, eight, wide):
    c = Shared([(1, 128 + i) for i in range(4)], [(0, 4, 128)], 16, 2, 64, torch.float16, wide=wide, eight=eight)
    q = queries(c, 8, torch.float16)
    pools = [c.k_pages, c.v_pages] if eight else [c.k_pages.nan_to_num(0), c.v_pages.nan_to_num(0)]
    op = torch.ops.minfer.flash_attn_paged_shared_fp8 if eight else torch.ops.minfer.flash_attn_paged_shared
    torch.library.opcheck(op.default, (*QT[q.dtype], q, *pools, *c.scales(), c.table, c.cu, c.ctx, i32(c.cu_groups), i32(c.told), 1, torch.zeros_like(q)),
                          test_utils=("test_faketensor",) if eight else OPCHECKS)
