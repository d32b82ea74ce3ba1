"""Calls of the operators of a serving step at the edges that their documentation allows: nothing to do, no entries, an unknown bound of tokens."""
import pytest
import torch

import serving_ref as ref
from test_gpu_shared import Shared, check, queries
from test_gpu_tables import DEV, LEFT, i32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("drafter", [True, False])
@pytest.mark.parametrize("V", [7, 50000])
@pytest.mark.parametrize("n", [1, 40])
def test_verify_no_tokens(kerns, drafter, V, n):
    none = torch.empty(0, dtype=torch.int64, device=DEV)
    probs, kept = torch.empty(0, V, device=DEV), i32([LEFT] * n)
    kerns.verify_drafts(none, i32([0] * (n + 1)), probs, probs.clone() if drafter else None, torch.empty(0, device=DEV), torch.rand(n, device=DEV), none.clone(), kept)
    assert kept.tolist() == [0] * n
    kerns.verify_drafts(none, i32([5] * n + [9]), probs, None, torch.empty(0, device=DEV), torch.rand(n, device=DEV), none.clone(), kept.fill_(LEFT))
    assert kept.tolist() == [0] * n
    kerns.verify_drafts(none, i32([0]), probs, None, torch.empty(0, device=DEV), torch.empty(0, device=DEV), none.clone(), i32([]))


@pytest.mark.parametrize("n", [1, 3, 70])
def test_tables_without_entries(kerns, n):
    table = torch.empty(n, 0, dtype=torch.int32, device=DEV)
    cu, ctx, after, state = i32([LEFT] * (n + 1)), i32([LEFT] * n), i32([LEFT] * n), i32([LEFT] * 3)
    slots = torch.full((2 * n + 1,), LEFT, dtype=torch.int64, device=DEV)
    kerns.paged_tables(16, i32([1] * n), i32([2] * n), i32([4] * n), i32([3, 1, 2]), i32([1, 2, 0]), table, cu, ctx, slots, after, state)
    assert cu.tolist() == list(range(0, 2 * n + 1, 2)) and ctx.tolist() == [3] * n and slots.tolist() == [-1] * 2 * n + [LEFT]
    assert after.tolist() == [0] * n and state.tolist() == [1, 2, 0]
    ring = i32([3, 1, 2])
    kerns.paged_release(16, i32([0] * n), i32([4] * n), table, ring, i32([1, 2, 0]), after.fill_(LEFT), state)
    assert ring.tolist() == [3, 1, 2] and after.tolist() == [0] * n and state.tolist() == [1, 2, 0]


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("lens", [[(1, 200), (1, 300), (1, 260)], [(2, 200), (1, 300), (3, 260), (2, 400)], [(9, 200), (1, 300), (30, 260)]])
def test_tokens_of_no_known_bound(kerns, eight, lens):
    """max_q_len 0: a sequence may have all of the tokens, which for a few of them is a call for groups still."""
    c = Shared(lens, [(0, len(lens), 192)], 16, 2, 64, torch.float16, eight=eight)
    out = check(kerns, c, 8, torch.float16, max_q=0)
    if sum(n for n, _ in lens) > 16:   # more than 64 rows
        assert torch.equal(out, c.unshared(kerns, queries(c, 8, torch.float16)))


@pytest.mark.parametrize("n", [64, 65, 300])
def test_pages_of_a_shared_prefix(kerns, n):
    """Sequences that name one prefix's pages: all but one keep its rows, and every page comes back once."""
    rest = [s % 3 for s in range(n)]
    N = 4 + sum(rest)
    names = iter(range(4, N))
    table = [[0, 1, 2, 3] + [next(names) for _ in range(r)] + [-1] * (2 - r) for r in rest]
    keep, held, ring, state = [64] * (n - 1) + [0], [4 + r for r in rest], [-1] * N, [5 % N, 0, 0]
    ring_t, after, state_after = i32(ring), i32([LEFT] * n), i32([LEFT] * 3)
    kerns.paged_release(16, i32(keep), i32(held), i32(table), ring_t, i32(state), after, state_after)
    want = ref.release(16, keep, held, table, ring, state)
    assert (ring_t.tolist(), after.tolist(), state_after.tolist()) == tuple(want)
    assert sorted(ring_t.tolist()) == list(range(N))
