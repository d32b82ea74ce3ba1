"""Pages given back where sums over the sequences in front are large: counts past 31 bits, more sequences than there are workgroups for."""
import random

import pytest
import torch

import serving_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def test_more_entries_than_31_bits_count(kerns):
    """32 sequences of 2^26 entries, which name pages over and over, in front of one: its pages find no room, and the number of those that did not is whole."""
    N, wide, free, head = 100, 1 << 26, 90, 7
    table = torch.full((33, wide), 5, dtype=torch.int32, device=DEV)   # 8.3 GiB
    table[0, :12] = torch.arange(30, 42, device=DEV)
    table[32, :3] = i32([20, 21, 22])
    guard = torch.full((3 * N,), -77, dtype=torch.int32, device=DEV)
    guard[N:2 * N] = torch.arange(N, device=DEV)
    want = guard.clone()
    for i in range(N - free):
        want[N + (head + free + i) % N] = 30 + i
    held, state = i32([-77] * 33), i32([-77] * 3)
    kerns.paged_release(16, i32([0] * 33), i32([wide] * 32 + [3]), table, guard[N:2 * N], i32([head, free, 0]), held, state)
    assert torch.equal(guard, want)
    assert held.tolist() == [0] * 33 and state.tolist() == [head, N, 32 * wide + 3 - (N - free)]
