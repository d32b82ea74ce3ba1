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


def sequences(n, seed):
    """n sequences with up to three pages of a shuffled pool, some entries naming none; what each keeps; a ring without free pages."""
    r = random.Random(seed)
    held = [r.randint(0, 3) for _ in range(n)]
    names = list(range(sum(held) + 5))
    r.shuffle(names)
    table = [[(names.pop() if r.random() < 0.9 else -1) if i < h else -1 for i in range(4)] for h in held]
    keep = [r.choice((0, 16, 17, 1 << 30)) for _ in range(n)]
    return held, table, keep, [-1] * (sum(held) + 5), [r.randrange(sum(held) + 5), 0, 0]


@pytest.mark.parametrize("n", [4095, 4096, 4097, 4101, 8193, 50003])
def test_more_sequences_than_workgroups_of_four(kerns, n):
    held, table, keep, ring, state = sequences(n, n)
    ring_t, after, state_after = i32(ring), i32([-77] * n), i32([-77] * 3)
    kerns.paged_release(16, i32(keep), i32(held), i32(table), ring_t, i32(state), after, state_after)
    for got, want, name in zip((ring_t, after, state_after), ref.release(16, keep, held, table, ring, state), ("ring", "held_after", "state_after")):
        assert got.tolist() == want, name


def test_millions_of_sequences(kerns):
    """The sums over what lies in front do not make the work grow with the square of the sequences: 2^22 of them end, with a page each.  (Where every four of
    them have a workgroup that sums the counts in front this takes half a second and, at 2^24, eight; 1024 workgroups take 6 ms.)"""
    n = 1 << 22
    g = torch.Generator(device=DEV).manual_seed(1)
    pages = torch.randperm(n, generator=g, device=DEV).to(torch.int32)
    ring, after, state = torch.full((n,), -1, dtype=torch.int32, device=DEV), torch.full((n,), -77, dtype=torch.int32, device=DEV), i32([-77] * 3)
    zeros, ones, before = torch.zeros(n, dtype=torch.int32, device=DEV), torch.ones(n, dtype=torch.int32, device=DEV), i32([9, 0, 0])
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    kerns.paged_release(16, zeros[:65], ones[:65], pages[:65].view(65, 1), ring.clone(), before, after[:65].clone(), state.clone())   # (the kernels are loaded)
    start.record()
    kerns.paged_release(16, zeros, ones, pages.view(n, 1), ring, before, after, state)
    end.record()
    assert torch.equal(ring, pages.roll(9)) and not after.any() and state.tolist() == [9, n, 0]
    assert start.elapsed_time(end) < 100.0
