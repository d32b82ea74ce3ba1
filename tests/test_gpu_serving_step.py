"""The operators of a serving step together, as a server calls them: pages for new tokens, the append, attention of a batch behind one prompt, drafts checked,
lengths of the next step, pages given back; everything on the device but the random numbers."""
import pytest
import torch

import paged_ref
import serving_ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
LEFT = -77


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


class Server:
    def __init__(self, kerns, n, dtype, seed, S=16, Hq=8, Hkv=2, D=64, prompt=150, pool=400):
        self.kerns, self.n, self.dtype, self.S, self.Hq, self.Hkv, self.D, self.N = kerns, n, dtype, S, Hq, Hkv, D, pool
        self.g = torch.Generator().manual_seed(seed)
        # a table so wide that the attention is one of those that know of groups
        self.width = max(64, 230000000 // ((n + 1) * Hkv * D * 4 * S))
        self.table = torch.full((n + 1, self.width), -1, dtype=torch.int32, device=DEV)
        self.ring = torch.randperm(pool, generator=self.g).to(torch.int32).to(DEV)
        self.state, self.held = [i32([0, pool, 0]), i32([0] * 3)], [i32([0] * (n + 1)), i32([0] * (n + 1))]
        self.past = i32([0] * (n + 1))
        nan = torch.full((pool, Hkv, S, D), float("nan"), dtype=dtype, device=DEV)
        self.k, self.v = nan, nan.clone()
        self.rows = [[] for _ in range(n + 1)]      # of every sequence, the rows of the pool that hold it
        self.prefix = 0
        # the prompt, by a sequence of its own (the last one); the others then name its whole pages
        self.step([0] * n + [prompt])
        self.past = i32([0] * n + [prompt])
        self.prefix = prompt // S * S
        for s in range(n):
            self.table[s, :self.prefix // S] = self.table[n, :self.prefix // S]
            self.rows[s] = self.rows[n][:self.prefix]
        self.held[0][:n] = self.prefix // S
        self.past[:n] = self.prefix

    def step(self, new, qtype=(1, 1, 2)):
        """One step's index tensors, append and attention; (the attention's output, its definition, its bound)."""
        T, n = sum(new), self.n + 1
        cu, ctx, slots = i32([LEFT] * (n + 1)), i32([LEFT] * n), torch.full((T,), LEFT, dtype=torch.int64, device=DEV)
        self.kerns.paged_tables(self.S, self.past, i32(new), self.held[0], self.ring, self.state[0], self.table, cu, ctx, slots, self.held[1], self.state[1])
        self.held.reverse(), self.state.reverse()
        q, k, v = (torch.randn(1, T, h, self.D, generator=self.g).to(self.dtype).to(DEV) for h in (self.Hq, self.Hkv, self.Hkv))
        self.kerns.rope_kv_append_paged(1, self.D, 1e4, q, k, v, cu, self.past, self.table, self.k, self.v)
        out = torch.full_like(q, float("nan"))
        groups = i32([0, self.n]) if self.prefix else i32([0, 0])
        self.kerns.flash_attn_paged_shared(*qtype, q.transpose(1, 2), self.k, self.v, self.table, cu, ctx, groups, i32([self.prefix]), max(new), out.transpose(1, 2))
        # the same from the pool's rows by the slots, which nobody but paged_tables made
        at, flat = 0, [x.transpose(1, 2).reshape(-1, self.Hkv, self.D).cpu() for x in (self.k, self.v)]
        past = self.past.tolist()
        for s, w in enumerate(new):
            self.rows[s] = self.rows[s][:past[s]] + slots[at:at + w].tolist()
            at += w

        class Dense:
            Hkv, seqs, cu_list = self.Hkv, [(w, p) for w, p in zip(new, past)], cu.tolist()
            k_dense, v_dense = ([x[r].double().transpose(0, 1) for r in self.rows] for x in flat)

            @staticmethod
            def row_there(s):
                return torch.ones(len(self.rows[s]), dtype=torch.bool)

        want, bound = paged_ref.attend(Dense, q[0].transpose(0, 1).cpu())
        err = (out[0].transpose(0, 1).cpu().double() - want).abs()
        assert (err <= bound).all()
        return cu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("drafter", [True, False])
def test_steps_with_drafts(kerns, dtype, drafter):
    qtype = (1, 1, 2) if dtype == torch.float16 else (30, 256, 512)
    n, V, sv = 5, 3001, None
    sv = Server(kerns, n, dtype, 3)
    g = torch.Generator().manual_seed(9)
    moved = []
    for step in range(8):
        new = [1 + (step + s) % 4 for s in range(n)] + [0]     # (the prompt's own sequence has no tokens any more)
        cu = sv.step(new, qtype)
        T = sum(new)
        logits = 2.0 * torch.randn(T, V, generator=g)
        p, q = torch.softmax(logits, -1), torch.softmax(logits + torch.randn(T, V, generator=g), -1)
        tokens = torch.randint(0, V, (T,), generator=g)
        tokens[1:] = torch.multinomial(q[:-1], 1, generator=g)[:, 0]
        au, su = torch.rand(T, generator=g), torch.rand(n + 1, generator=g)
        out, kept = torch.full((T,), LEFT, dtype=torch.int64, device=DEV), i32([LEFT] * (n + 1))
        kerns.verify_drafts(tokens.to(DEV), cu, p.to(DEV), q.to(DEV) if drafter else None, au.to(DEV), su.to(DEV), out, kept)
        want, n_kept = serving_ref.verify(tokens, cu.tolist(), p, q if drafter else None, au, su)
        assert out.tolist() == want and kept.tolist() == n_kept
        moved += n_kept[:n]
        # a sequence goes on behind its kept drafts, whose rows are there; the row of the token that was drawn is the next step's first
        sv.past = (sv.past + kept + (i32(new) > 0)).to(torch.int32)
    assert len(set(moved)) > 1
    # three sequences end and keep the prompt's pages only, then everything ends, the prompt last
    total = sv.prefix // sv.S
    keep = torch.where(i32([1, 0, 1, 0, 1, 0]) > 0, sv.prefix, sv.past)
    for k in (keep, i32([sv.prefix] * n + [0])):
        before = sum(sv.held[0].tolist())
        kerns.paged_release(sv.S, k.to(torch.int32), sv.held[0], sv.table, sv.ring, sv.state[0], sv.held[1], sv.state[1])
        given = before - sum(sv.held[1].tolist())
        assert sv.state[1].tolist()[1] == sv.state[0].tolist()[1] + given and sv.state[1].tolist()[2] == 0
        sv.held.reverse(), sv.state.reverse()
    head, count, _ = sv.state[0].tolist()
    assert count == sv.N and sorted(int(sv.ring[(head + i) % sv.N]) for i in range(count)) == list(range(sv.N))
    assert sv.held[0].tolist() == [total] * n + [0]


def test_a_captured_step(kerns):
    """Tables, append, attention and verification recorded once and replayed with other lengths, each replay against the same calls made eagerly on copies."""
    n, V = 4, 800
    sv = Server(kerns, n, torch.float16, 5)
    T = 2 * n
    names = dict(past=sv.past.clone(), new=i32([2] * n + [0]), held=sv.held[0].clone(), state=sv.state[0].clone(), ring=sv.ring.clone(), table=sv.table.clone(), k=sv.k.clone(), v=sv.v.clone())
    g = torch.Generator().manual_seed(1)
    fixed = [torch.randn(1, T, h, 64, generator=g).half().to(DEV) for h in (8, 2, 2)]
    groups, prefix = i32([0, n]), i32([sv.prefix])
    p = torch.softmax(torch.randn(T, V, generator=g), -1).to(DEV)
    tokens, au, su = torch.randint(0, V, (T,), generator=g).to(DEV), torch.rand(T, generator=g).to(DEV), torch.rand(n + 1, generator=g).to(DEV)

    def outputs():
        return dict(cu=i32([0] * (n + 2)), ctx=i32([0] * (n + 1)), slots=torch.zeros(T, dtype=torch.int64, device=DEV), held2=i32([0] * (n + 1)), state2=i32([0] * 3),
                    q=torch.zeros(1, T, 8, 64, dtype=torch.float16, device=DEV), out=torch.zeros(1, T, 8, 64, dtype=torch.float16, device=DEV),
                    tok=torch.zeros(T, dtype=torch.int64, device=DEV), kept=i32([0] * (n + 1)))

    def step(a, o):
        kerns.paged_tables(16, a["past"], a["new"], a["held"], a["ring"], a["state"], a["table"], o["cu"], o["ctx"], o["slots"], o["held2"], o["state2"])
        o["q"].copy_(fixed[0])
        kerns.rope_kv_append_paged(1, 64, 1e4, o["q"], fixed[1], fixed[2], o["cu"], a["past"], a["table"], a["k"], a["v"])
        kerns.flash_attn_paged_shared(1, 1, 2, o["q"].transpose(1, 2), a["k"], a["v"], a["table"], o["cu"], o["ctx"], groups, prefix, 4, o["out"].transpose(1, 2))
        kerns.verify_drafts(tokens, o["cu"], p, None, au, su, o["tok"], o["kept"])

    o = outputs()
    step({k: x.clone() for k, x in names.items()}, o)
    torch.cuda.synchronize()
    live, graph = {k: x.clone() for k, x in names.items()}, torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(live, o)
    for new in ([2, 2, 2, 2, 0], [1, 4, 0, 3, 0], [4, 4, 0, 0, 0]):
        for k, x in names.items():
            live[k].copy_(x)
        live["new"].copy_(i32(new))
        graph.replay()
        got = {k: x.clone() for k, x in o.items()}
        again, e = {k: x.clone() for k, x in names.items()}, outputs()
        again["new"].copy_(i32(new))
        step(again, e)
        torch.cuda.synchronize()
        for k in got:
            assert torch.equal(got[k], e[k]), k
        # (rows that nothing was written to hold NaN)
        assert torch.equal(live["k"].view(torch.int16), again["k"].view(torch.int16)) and torch.equal(live["table"], again["table"])


def test_opcheck(kerns):
    from test_gpu_shared import QT, Shared, queries
    ops = torch.ops.minfer
    utils = ("test_schema", "test_faketensor")
    z = lambda *n: torch.zeros(*n, dtype=torch.int32, device=DEV)
    long = lambda n: torch.zeros(n, dtype=torch.int64, device=DEV)
    torch.library.opcheck(ops.paged_tables.default, (16, i32([3, 0]), i32([2, 1]), i32([1, 0]), i32([3, 2, 0, 1]), i32([0, 3, 0]), z(2, 3), z(3), z(2), long(3), z(2), z(3)), test_utils=utils)
    torch.library.opcheck(ops.paged_release.default, (16, i32([0, 9]), i32([1, 1]), i32([[2, 0], [1, 0]]), z(4), i32([0, 2, 0]), z(2), z(3)), test_utils=utils)
    p = torch.softmax(torch.randn(4, 9, device=DEV), -1)
    for draft in (None, p.flip(0).contiguous()):
        torch.library.opcheck(ops.verify_drafts.default, (torch.arange(4, device=DEV), i32([0, 3, 4]), p, draft, torch.rand(4, device=DEV), torch.rand(2, device=DEV), long(4), z(2)), test_utils=utils)
    for eight in (False, True):
        c = Shared([(1, 70), (2, 90)], [(0, 2, 64)], 16, 2, 64, torch.float16, eight=eight)
        q = queries(c, 4, torch.float16)
        op = ops.flash_attn_paged_shared_fp8 if eight else ops.flash_attn_paged_shared
        torch.library.opcheck(op.default, (*QT[q.dtype], q, c.k_pages, c.v_pages, *c.scales(), c.table, c.cu, c.ctx, i32([0, 2]), i32([64]), 2, torch.zeros_like(q)), test_utils=("test_faketensor",))
