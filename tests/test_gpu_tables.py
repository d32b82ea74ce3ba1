"""Block tables, slots and the ring of free pages on the GPU, number for number against their definition."""
import random

import pytest
import torch

import serving_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
LEFT = -77   # what nothing was written over


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


class Pool:
    """n sequences with pages out of a shuffled pool, some of its pages free in a ring that goes on around its end."""

    def __init__(self, n, page, past_hi, new_hi, width, free, seed, surplus=0.3, gone=0.0):
        r = random.Random(seed)
        self.page, self.n = page, n
        self.past = [r.randint(0, past_hi) for _ in range(n)]
        self.new = [r.randint(0, new_hi) for _ in range(n)]
        self.held = [min(-(-p // page) + (r.random() < surplus), width) for p in self.past]
        used = sum(self.held)
        self.N = used + free + 3
        names = list(range(self.N))
        r.shuffle(names)
        self.table = [[-1] * width for _ in range(n)]
        for row, h in zip(self.table, self.held):
            for i in range(h):
                row[i] = names.pop()
                if r.random() < gone:
                    row[i] = -1
        head = r.randrange(self.N)
        self.ring = [-1] * self.N
        for i in range(free):
            self.ring[(head + i) % self.N] = names.pop()
        self.state = [head, free, 5]

    def tensors(self, gap=0):
        t = torch.full((self.n, len(self.table[0]) + gap), LEFT, dtype=torch.int32, device=DEV)
        t[:, :len(self.table[0])] = i32(self.table)
        return t[:, :len(self.table[0])] if gap else t


def run_tables(kerns, c, n_slots, gap=0):
    table, ring = c.tensors(gap), i32(c.ring)
    cu, ctx, held, state = i32([LEFT] * (c.n + 1)), i32([LEFT] * c.n), i32([LEFT] * c.n), i32([LEFT] * 3)
    slots = torch.full((n_slots,), LEFT, dtype=torch.int64, device=DEV)
    kerns.paged_tables(c.page, i32(c.past), i32(c.new), i32(c.held), ring, i32(c.state), table, cu, ctx, slots, held, state)
    return [x.tolist() for x in (cu, ctx, slots, table, held, state)], table


def check_tables(kerns, c, n_slots, gap=0):
    got, table = run_tables(kerns, c, n_slots, gap)
    want = ref.tables(c.page, c.past, c.new, c.held, c.ring, c.state, c.table, n_slots)
    want = [[LEFT if x is None else x for x in w] if i == 2 else w for i, w in enumerate(want)]
    for g, w, name in zip(got, want, ("cu", "ctx", "slots", "table", "held_after", "state_after")):
        assert g == list(w), name
    if gap:
        assert (table.as_strided((c.n, gap), (table.stride(0), 1), len(c.table[0])) == LEFT).all()


@pytest.mark.parametrize("n,page,past_hi,new_hi,free", [
    (1, 16, 0, 1, 4), (1, 16, 700, 3000, 300), (5, 32, 100, 1, 9), (64, 16, 800, 1, 80), (256, 16, 900, 9, 300), (23, 64, 500, 2000, 900), (257, 128, 3000, 40, 600),
    (1025, 16, 60, 3, 2000), (3000, 1024, 5000, 5, 4000), (7, 16, 0, 0, 10)])
def test_tables(kerns, n, page, past_hi, new_hi, free):
    width = -(-(past_hi + new_hi) // page) + 2
    c = Pool(n, page, past_hi, new_hi, width, free, n)
    check_tables(kerns, c, sum(c.new))


def test_tables_strided_and_slots_of_another_length(kerns):
    c = Pool(40, 16, 300, 50, 30, 200, 3)
    check_tables(kerns, c, sum(c.new), gap=5)
    check_tables(kerns, c, sum(c.new) + 70)    # entries behind the last token stay
    check_tables(kerns, c, sum(c.new) - 333)   # tokens behind the last entry have none
    check_tables(kerns, c, 0)


@pytest.mark.parametrize("free", [0, 1, 37])
def test_tables_where_pages_are_lacking(kerns, free):
    check_tables(kerns, Pool(60, 16, 200, 40, 20, free, 5), 2000)


def test_tables_wider_than_the_table(kerns):
    check_tables(kerns, Pool(30, 16, 300, 300, 12, 500, 6), 5000)


def test_tables_over_data_that_nobody_checked(kerns):
    c = Pool(8, 16, 100, 30, 10, 40, 8)
    c.past[1], c.new[2], c.held[3], c.held[4] = -5, -9, -1, 1000
    c.table[5][0], c.table[6][0] = c.N, -1
    check_tables(kerns, c, 400)
    for state in ([c.N + 3, 40, 0], [-1, 40, 0], [3, c.N + 50, 0], [3, -4, 0]):
        c.state = state
        check_tables(kerns, c, 400)


def test_tables_saturate(kerns):
    big = 2 ** 31 - 1
    c = Pool(4, 16, 10, 3, 4, 9, 1)
    c.new = [1 << 30, 1 << 30, 1 << 30, 2]
    got, _ = run_tables(kerns, c, 100)
    assert got[0] == [0, 1 << 30, big, big, big]
    assert got[1][:3] == [min(p + (1 << 30), big) for p in c.past[:3]]


def test_no_sequences_and_no_pages(kerns):
    cu, state = i32([LEFT]), i32([LEFT] * 3)
    none, slots = i32([]), torch.full((3,), LEFT, dtype=torch.int64, device=DEV)
    kerns.paged_tables(16, none, none, none, i32([4, 5]), i32([1, 2, 0]), torch.empty(0, 3, dtype=torch.int32, device=DEV), cu, none, slots, none, state)
    assert cu.tolist() == [0] and state.tolist() == [1, 2, 0] and slots.tolist() == [LEFT] * 3
    held = i32([LEFT])
    kerns.paged_release(16, none, none, torch.empty(0, 3, dtype=torch.int32, device=DEV), i32([4, 5]), i32([1, 2, 0]), none, state)
    assert state.tolist() == [1, 2, 0]
    table = torch.full((1, 2), -1, dtype=torch.int32, device=DEV)
    cu = i32([LEFT] * 2)
    kerns.paged_tables(16, i32([0]), i32([2]), i32([0]), none, i32([0, 0, 0]), table, cu, i32([0]), slots, held, state)
    assert cu.tolist() == [0, 2] and slots.tolist() == [-1, -1, LEFT] and held.tolist() == [0] and state.tolist() == [0, 0, 1] and table.tolist() == [[-1, -1]]


def check_release(kerns, c, keep, gap=0):
    table, ring, held, state = c.tensors(gap), i32(c.ring), i32([LEFT] * c.n), i32([LEFT] * 3)
    before = table.clone()
    kerns.paged_release(c.page, i32(keep), i32(c.held), table, ring, i32(c.state), held, state)
    want = ref.release(c.page, keep, c.held, c.table, c.ring, c.state)
    for g, w, name in zip((ring, held, state), want, ("ring", "held_after", "state_after")):
        assert g.tolist() == w, name
    assert torch.equal(table, before)


@pytest.mark.parametrize("n,page,past_hi,free,ends,gone", [(1, 16, 500, 3, 1.0, 0.0), (9, 16, 4000, 50, 0.5, 0.2), (64, 16, 900, 10, 0.1, 0.0), (300, 32, 3000, 0, 0.4, 0.3), (63, 16, 20000, 40, 1.0, 0.1), (65, 16, 20000, 40, 1.0, 0.1),
                                                           (1030, 64, 700, 9, 1.0, 0.05), (5, 16, 100, 7, 0.0, 0.0)])
def test_release(kerns, n, page, past_hi, free, ends, gone):
    c = Pool(n, page, past_hi, 0, -(-past_hi // page) + 1, free, n + 1, gone=gone)
    r = random.Random(n)
    keep = [0 if r.random() < ends else p if r.random() < 0.5 else 2 ** 31 - 1 for p in c.past]
    check_release(kerns, c, keep, gap=3)


def test_release_over_data_that_nobody_checked(kerns):
    c = Pool(6, 16, 200, 0, 14, 12, 4)
    c.held[0], c.held[1] = -3, 500
    c.table[2][0] = c.N + 7
    check_release(kerns, c, [0, 0, 0, -8, 1, 17])
    c.state = [c.N * 2 + 1, c.N - 2, 0]   # a ring that has no room for all of them
    check_release(kerns, c, [0] * 6)


def test_steps_one_after_the_other(kerns):
    """Pages go round: what ends gives its pages back, what grows takes them, and no page is ever in two places."""
    r, S, n, N = random.Random(7), 16, 12, 60
    table = torch.full((n, 10), -1, dtype=torch.int32, device=DEV)
    ring = torch.randperm(N, device=DEV).to(torch.int32)
    states, helds = [i32([0, N, 0]), i32([0] * 3)], [i32([0] * n), i32([0] * n)]
    lens = [0] * n
    for _ in range(40):
        new = [min(r.choice((0, 1, 1, 3, 30)), 160 - x) for x in lens]
        cu, ctx, slots = i32([0] * (n + 1)), i32([0] * n), torch.full((sum(new),), LEFT, dtype=torch.int64, device=DEV)
        kerns.paged_tables(S, i32(lens), i32(new), helds[0], ring, states[0], table, cu, ctx, slots, helds[1], states[1])
        lens = [min(a + b, 16 * h) for a, b, h in zip(lens, new, helds[1].tolist())]   # (rows without a page are not there)
        keep = [0 if r.random() < 0.2 else x for x in lens]
        kerns.paged_release(S, i32(keep), helds[1], table, ring, states[1], helds[0], states[0])
        lens = keep
        head, count, _ = states[0].tolist()
        names = [p for row, h in zip(table.tolist(), helds[0].tolist()) for p in row[:h]] + [int(ring[(head + i) % N]) for i in range(count)]
        assert sorted(names) == list(range(N))


def test_replayed(kerns):
    """A captured step, replayed over new lengths, gives what the same calls give outside."""
    c = Pool(50, 16, 400, 6, 40, 300, 9)
    past, new, held, ring, state = i32(c.past), i32(c.new), i32(c.held), i32(c.ring), i32(c.state)
    table, cu, ctx = c.tensors(), i32([0] * 51), i32([0] * 50)
    slots, after, state_after = torch.zeros(400, dtype=torch.int64, device=DEV), i32([0] * 50), i32([0] * 3)
    keep, after2, state2 = i32([0] * 50), i32([0] * 50), i32([0] * 3)

    def step():
        kerns.paged_tables(16, past, new, held, ring, state, table, cu, ctx, slots, after, state_after)
        kerns.paged_release(16, keep, after, table, ring, state_after, after2, state2)

    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    for k in range(3):
        table.copy_(i32(c.table)); ring.copy_(i32(c.ring))
        past.copy_(i32(c.past)); keep.copy_(i32([0 if i % 3 == k else 2 ** 31 - 1 for i in range(50)]))
        new.copy_(torch.roll(i32(c.new), k))
        g.replay()
        got = [x.clone() for x in (cu, ctx, table, ring, after, after2, state2)]
        table.copy_(i32(c.table)); ring.copy_(i32(c.ring))
        step()
        assert all(torch.equal(a, b) for a, b in zip(got, (cu, ctx, table, ring, after, after2, state2)))


def test_refusals(kerns):
    c = Pool(4, 16, 50, 3, 6, 9, 1)
    past, new, held, ring, state, table = i32(c.past), i32(c.new), i32(c.held), i32(c.ring), i32(c.state), c.tensors()
    cu, ctx, slots, after, state2 = i32([0] * 5), i32([0] * 4), torch.zeros(20, dtype=torch.int64, device=DEV), i32([0] * 4), i32([0] * 3)
    good = [16, past, new, held, ring, state, table, cu, ctx, slots, after, state2]
    for at, x, text in ((0, 24, "page_size"), (2, new[:3], "new_lens"), (3, held.long(), "pages_held"), (4, ring.view(1, -1), "free_ring"), (5, state[:2], "ring_state"),
                        (6, table.t(), "block_table"), (7, cu[:4], "cu_seqlens"), (9, slots.int(), "slots"), (10, held, "must not be inputs"), (11, state, "must not be state")):
        with pytest.raises(RuntimeError, match=text):
            kerns.paged_tables(*good[:at], x, *good[at + 1:])
    good = [16, past, held, table, ring, state, after, state2]
    for at, x, text in ((0, 0, "page_size"), (2, held[1:], "pages_held"), (3, table[:3], "block_table"), (6, past, "must not be inputs"), (7, state, "must not be state")):
        with pytest.raises(RuntimeError, match=text):
            kerns.paged_release(*good[:at], x, *good[at + 1:])
