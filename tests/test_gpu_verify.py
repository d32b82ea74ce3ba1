"""Verification of drafted tokens on the GPU, token for token against its definition in 64 bits."""
import pytest
import torch

import serving_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
LEFT = -77


class Case:
    """Drafts drawn from distributions near the target's; every sequence with up to `most` of them."""

    def __init__(self, n, most, V, dtype=torch.float32, drafter=True, seed=0, lens=None, sharp=3.0, ids=torch.int64):
        g = torch.Generator().manual_seed(seed)
        lens = torch.randint(1, most + 2, (n,), generator=g).tolist() if lens is None else lens
        self.cu = [sum(lens[:i]) for i in range(len(lens) + 1)]
        T = self.cu[-1]
        logits = sharp * torch.randn(T, V, generator=g)
        q = torch.softmax(logits + 0.7 * torch.randn(T, V, generator=g), -1)
        self.target, self.draft = torch.softmax(logits, -1).to(dtype), q.to(dtype) if drafter else None
        self.tokens = torch.randint(0, V, (T,), generator=g).to(ids)
        if T > 1:
            self.tokens[1:] = torch.multinomial(q[:-1], 1, generator=g)[:, 0].to(ids)
        self.accept_u, self.sample_u = torch.rand(T, generator=g), torch.rand(len(lens), generator=g)

    def call(self, kerns, views=False):
        T, V = self.target.shape
        target, draft = self.target.to(DEV), None if self.draft is None else self.draft.to(DEV)
        if views:   # rows that lie apart and start anywhere
            target = torch.nn.functional.pad(target, (3, 4), value=9.0)[:, 3:3 + V]
            draft = None if draft is None else torch.nn.functional.pad(draft, (1, 2), value=9.0)[:, 1:1 + V]
        out = torch.full((T,), LEFT, dtype=self.tokens.dtype, device=DEV)
        kept = torch.full((len(self.cu) - 1,), LEFT, dtype=torch.int32, device=DEV)
        kerns.verify_drafts(self.tokens.to(DEV), torch.tensor(self.cu, dtype=torch.int32, device=DEV), target, draft, self.accept_u.to(DEV), self.sample_u.to(DEV), out, kept)
        return out.tolist(), kept.tolist()

    def check(self, kerns, views=False):
        want, kept = ref.verify(self.tokens, self.cu, self.target, self.draft, self.accept_u, self.sample_u)
        got = self.call(kerns, views)
        assert got[1] == kept
        assert got[0] == [LEFT if x is None else x for x in want]
        return kept


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("drafter", [True, False])
@pytest.mark.parametrize("n,most,V", [(1, 4, 32000), (3, 0, 7), (17, 5, 2047), (5, 2, 2049), (40, 8, 1), (9, 3, 100003), (70, 2, 4096)])
def test_verify(kerns, dtype, drafter, n, most, V):
    Case(n, most, V, dtype, drafter, seed=n + V).check(kerns)


@pytest.mark.parametrize("V", [33, 5001, 20000])
def test_rows_apart_and_32_bit_tokens(kerns, V):
    for dtype in (torch.float32, torch.bfloat16):
        Case(12, 4, V, dtype, ids=torch.int32, seed=V).check(kerns, views=True)


def test_all_and_none_kept(kerns):
    c = Case(8, 6, 3000, lens=[7] * 8)
    c.accept_u.fill_(0.0)
    assert c.check(kerns) == [6] * 8
    c.accept_u.fill_(0.9999)
    c.target, c.draft = c.draft.flip(1), c.draft
    assert sum(c.check(kerns)) < 8
    assert Case(200, 0, 500, lens=[1] * 200).check(kerns) == [0] * 200


def test_more_drafts_than_lanes(kerns):
    c = Case(2, 0, 400, lens=[150, 66])
    c.accept_u.fill_(0.0)
    c.accept_u[100] = 1.0 - 2.0 ** -24
    c.tokens[101] = int(c.target[100].argmin())
    c.draft[100, c.tokens[101]] = 0.9
    assert c.check(kerns)[0] == 100


def test_many_sequences(kerns):
    Case(2500, 1, 300, seed=3).check(kerns)       # more than there are counters
    Case(2500, 1, 4100, torch.float16, seed=4).check(kerns)


@pytest.mark.parametrize("n,V", [(20, 16001), (100, 4100), (128, 4097), (129, 4097)])
def test_calls_one_after_the_other(kerns, n, V):
    """Several chunks to a row, whether or not the last workgroup of a sequence ends it, sequences without tokens among them; what one call counted is not the next one's."""
    lens = [(0, 1, 3, 2)[(s * 7 + s // 4) % 4] for s in range(n)]
    c = Case(n, 0, V, seed=n, lens=lens)
    want = (lambda r: ([LEFT if x is None else x for x in r[0]], r[1]))(ref.verify(c.tokens, c.cu, c.target, c.draft, c.accept_u, c.sample_u))
    for _ in range(3):
        assert c.call(kerns) == want


def test_marks_on_borders(kerns):
    """Equal weights of a power of two: every sum is exact, and a mark on a border belongs to the token behind it."""
    V = 4096
    c = Case(64, 0, V, lens=[1] * 64)
    c.target.fill_(1.0 / V)
    c.sample_u = torch.arange(64) / 64.0
    out, _ = c.call(kerns)
    assert out == [64 * i for i in range(64)]
    c.check(kerns)
    c.sample_u.fill_(1.0 - 2.0 ** -24)
    assert c.call(kerns)[0] == [V - 1] * 64
    c.sample_u.fill_(1.0)                          # no sum is larger: the last with a weight
    c.target[:, -9:] = 0
    assert c.call(kerns)[0] == [V - 10] * 64


@pytest.mark.parametrize("V", [50, 9000])
def test_rows_without_weight(kerns, V):
    c = Case(6, 0, V, lens=[3] * 6)
    c.accept_u.fill_(1.0 - 2.0 ** -24)
    c.target, c.draft = c.draft.clone(), c.draft
    x = c.tokens.roll(-1)
    c.draft[torch.arange(18), x] *= 1.5            # refused, and nowhere is there more of p than of q: p itself
    c.target[6:9] = 0                              # no probability at all
    c.target[9:12] = float("nan")
    c.target[12, ::2] = float("nan")
    c.target[13, 1::2] *= -1
    c.draft[15, ::3] = float("nan")
    c.check(kerns)
    assert c.call(kerns)[0][6] == -1


def test_drafts_that_are_no_tokens(kerns):
    for drafter in (True, False):
        c = Case(5, 0, 1000, drafter=drafter, lens=[4] * 5)
        c.accept_u.fill_(0.0)
        c.tokens[2], c.tokens[5], c.tokens[11] = -1, 1000, 1 << 40
        assert c.check(kerns)[:3] == [1, 0, 2]


def test_cu_seqlens_that_nobody_checked(kerns):
    c = Case(6, 0, 700, lens=[3] * 6)
    c.cu = [0, 3, 3, 9, 40, 0, 0]
    c.check(kerns)
    # tokens 0 and 1, none, 1 to 4, ..: token 1 is in two sequences, and gets what either of them says
    c.cu = [-4, 2, 1, 5, 18, 19, 30]
    want, kept = ref.verify(c.tokens, c.cu, c.target, c.draft, c.accept_u, c.sample_u)
    first, _ = ref.verify(c.tokens, c.cu[:2], c.target, c.draft, c.accept_u, c.sample_u[:1])
    got = c.call(kerns)
    assert got[1] == kept and got[0][1] in (first[1], want[1])
    assert [x for i, x in enumerate(got[0]) if i != 1] == [LEFT if x is None else x for i, x in enumerate(want) if i != 1]


def test_another_stream_and_a_graph(kerns):
    """Off the null stream there are no counters, and a second launch ends the rows: the same tokens."""
    c = Case(20, 5, 40000, seed=9)
    want = c.call(kerns)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        assert c.call(kerns) == want
    dev = [x.to(DEV) for x in (c.tokens, torch.tensor(c.cu, dtype=torch.int32), c.target, c.draft, c.accept_u, c.sample_u)]
    out, kept = torch.zeros_like(dev[0]), torch.zeros(20, dtype=torch.int32, device=DEV)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        kerns.verify_drafts(*dev, out, kept)
    for k in range(3):
        dev[4].copy_(torch.rand(dev[4].shape, device=DEV) if k else c.accept_u)
        out.fill_(LEFT)
        g.replay()
        got = out.tolist(), kept.tolist()
        kerns.verify_drafts(*dev, out, kept)
        assert got == (out.tolist(), kept.tolist())
        if k == 0:
            assert got == want


def test_refusals(kerns):
    c = Case(3, 2, 100)
    T = c.tokens.numel()
    good = [c.tokens.to(DEV), torch.tensor(c.cu, dtype=torch.int32, device=DEV), c.target.to(DEV), c.draft.to(DEV), c.accept_u.to(DEV), c.sample_u.to(DEV),
            torch.zeros(T, dtype=torch.int64, device=DEV), torch.zeros(3, dtype=torch.int32, device=DEV)]
    for at, x, text in ((0, good[0].float(), "tokens"), (1, good[1].long(), "cu_seqlens"), (2, good[2].double(), "target_probs"), (2, good[2][:-1], "target_probs"),
                        (2, good[2].t().contiguous().t(), "contiguous"), (3, good[3].half(), "draft_probs"), (3, good[3][:, :-1], "draft_probs"), (4, good[4].double(), "accept_u"),
                        (4, good[4][1:], "accept_u"), (5, good[5][1:], "sample_u"), (6, good[6].int(), "out_tokens"), (6, good[0], "must not be tokens"), (7, good[7][1:], "n_accepted")):
        with pytest.raises(RuntimeError, match=text):
            kerns.verify_drafts(*good[:at], x, *good[at + 1:])
