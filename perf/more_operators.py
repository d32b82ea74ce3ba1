"""One step of a serving batch around its paged KV cache, as cases that can be timed and compared.

A serving program goes through the same four things every step.  It gives the sequences the pages that their new rows need and maps
the new tokens to rows of the pool (`tables`); it gives the pages of sequences that ended back (`release`); it lets the new tokens
attend the cache, in which groups of sequences share the pages of a long prompt (`shared`); and it checks tokens that a
cheaper model drafted against the model's own probabilities, with random numbers that it drew before (`verify`).

The tokens of a step are packed: sequence s has tokens cu_seqlens[s] .. cu_seqlens[s + 1] - 1.  Pages lie in the pool in no order.
"""
import math
import os
import random
import sys

import torch

own = False

_DEV = "cuda"

# (query heads, KV heads) of the models' layers
_HEADS = ((8, 2), (16, 16), (24, 8), (32, 8), (48, 8), (64, 8))
_VOCABS = (32000, 50257, 100003, 128256)


def listed():
    return [
        # the tables of one decode step of a full serving batch; latency only
        {"name": "tables_step", "kind": "tables", "n": 256, "new_lo": 1, "new_hi": 1, "past_lo": 0, "past_hi": 8000, "page": 16, "lens": 1, "short": False},
        # prompts of no round length that come in together, in a pool that does not hold them all
        {"name": "tables_prompts", "kind": "tables", "n": 23, "new_lo": 300, "new_hi": 4095, "past_lo": 0, "past_hi": 700, "page": 32, "lens": 2, "short": True},
        # a few conversations that ended
        {"name": "release_few", "kind": "release", "n": 64, "past_lo": 20, "past_hi": 8000, "page": 16, "ends": 0.1, "lens": 3, "gone": False},
        # a third of a large batch that ended, behind windows that had given first pages back before
        {"name": "release_batch", "kind": "release", "n": 500, "past_lo": 1000, "past_hi": 16000, "page": 32, "ends": 0.33, "lens": 4, "gone": True},
        # a few users of a small model behind one instruction
        {"name": "shared_few", "kind": "shared", "n": 8, "groups": 1, "alone": 0, "pre_lo": 1500, "pre_hi": 1500, "q_lo": 1, "q_hi": 1,
         "past_lo": 30, "past_hi": 400, "Hq": 8, "Hkv": 2, "D": 64, "page": 16, "dtype": "f16", "cache": "16", "lens": 5},
        # one decode step of a full serving batch behind one long instruction
        {"name": "shared_step", "kind": "shared", "n": 64, "groups": 1, "alone": 0, "pre_lo": 6000, "pre_hi": 6000, "q_lo": 1, "q_hi": 1,
         "past_lo": 50, "past_hi": 1500, "Hq": 32, "Hkv": 8, "D": 128, "page": 16, "dtype": "bf16", "cache": "16", "lens": 6},
        # several documents that different numbers of users ask about, and users without one
        {"name": "shared_groups", "kind": "shared", "n": 90, "groups": 7, "alone": 9, "pre_lo": 500, "pre_hi": 9000, "q_lo": 1, "q_hi": 1,
         "past_lo": 20, "past_hi": 2000, "Hq": 24, "Hkv": 8, "D": 128, "page": 32, "dtype": "f16", "cache": "16", "lens": 7},
        # drafts of three to six tokens checked together, behind one document
        {"name": "shared_drafts", "kind": "shared", "n": 24, "groups": 1, "alone": 0, "pre_lo": 12000, "pre_hi": 12000, "q_lo": 3, "q_hi": 6,
         "past_lo": 10, "past_hi": 900, "Hq": 32, "Hkv": 8, "D": 128, "page": 64, "dtype": "bf16", "cache": "16", "lens": 8},
        # a large batch behind a very long shared document in 8-bit pages; the largest case
        {"name": "shared8_step", "kind": "shared", "n": 192, "groups": 2, "alone": 0, "pre_lo": 16000, "pre_hi": 24000, "q_lo": 1, "q_hi": 1,
         "past_lo": 100, "past_hi": 2500, "Hq": 32, "Hkv": 8, "D": 128, "page": 32, "dtype": "f16", "cache": "fp8", "lens": 9},
        # one user's drafts
        {"name": "verify_one", "kind": "verify", "n": 1, "d_lo": 4, "d_hi": 4, "V": 32000, "dtype": "f32", "drafter": True, "lens": 10},
        # a serving batch's drafts, some sequences without any
        {"name": "verify_batch", "kind": "verify", "n": 64, "d_lo": 0, "d_hi": 5, "V": 128256, "dtype": "f32", "drafter": True, "lens": 11},
        # drafts that were looked up in the prompt, and so have no probabilities; 16-bit probabilities over an odd vocabulary
        {"name": "verify_lookup", "kind": "verify", "n": 150, "d_lo": 1, "d_hi": 8, "V": 50257, "dtype": "bf16", "drafter": False, "lens": 12},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(("tables", "release", "shared", "shared", "shared", "verify", "verify"))
    c = {"kind": kind, "lens": rng.randrange(1 << 20)}
    if kind == "tables":
        form = rng.choice(("one", "few", "prompt"))
        c["new_hi"] = 1 if form == "one" else rng.randint(2, 9) if form == "few" else _log_int(rng, 16, 8192)
        c["n"] = _log_int(rng, 1, max(1, min(2048, 65536 // c["new_hi"])))
        c["new_lo"] = rng.choice((0 if c["n"] > 9 else 1, 1, max(1, c["new_hi"] // 2)))
        c["past_hi"] = rng.choice((0, _log_int(rng, 1, 60000)))
        c["past_lo"] = c["past_hi"] // rng.choice((1, 3, 20))
        c["page"] = rng.choice((16, 16, 32, 64, 128, 256))
        c["short"] = rng.random() < 0.25
        return c
    if kind == "release":
        c["n"] = _log_int(rng, 1, 1024)
        c["past_hi"] = _log_int(rng, 1, 30000)
        c["past_lo"] = c["past_hi"] // rng.choice((1, 3, 20))
        c["page"] = rng.choice((16, 16, 32, 64, 128, 256))
        c["ends"] = rng.choice((0.02, 0.2, 0.5, 1.0))
        c["gone"] = rng.random() < 0.3
        return c
    if kind == "verify":
        c["V"] = rng.choice(_VOCABS + (_log_int(rng, 100, 160000) | 1,))
        c["d_hi"] = rng.choice((1, 3, 5, 8))
        c["d_lo"] = rng.choice((0, 1, c["d_hi"]))
        c["dtype"] = rng.choice(("f32", "f32", "bf16", "f16"))
        c["drafter"] = rng.random() < 0.7
        c["n"] = _log_int(rng, 1, max(1, min(512, 64 * 128256 * 6 // (c["V"] * (c["d_hi"] + 1)))))
        return c
    c["Hq"], c["Hkv"] = rng.choice(_HEADS)
    c["D"] = rng.choice((64, 128, 128))
    c["page"] = rng.choice((16, 16, 32, 64, 128, 256))
    c["dtype"] = rng.choice(("f16", "bf16"))
    c["cache"] = rng.choice(("16", "16", "fp8"))
    c["n"] = _log_int(rng, 2, 192)
    c["groups"] = min(rng.choice((1, 1, 2, 3, 8)), c["n"] // 2)
    c["alone"] = rng.randint(0, (c["n"] - 2 * c["groups"]) // 4)
    c["q_hi"] = rng.choice((1, 1, 1, rng.randint(2, 8)))
    c["q_lo"] = max(1, c["q_hi"] // rng.choice((1, 2)))
    # bytes of the sequences' own rows and of the prefixes, and (query, key) pairs of all heads, within those of the largest listed case
    row = 4 * c["Hkv"] * c["D"]
    c["past_hi"] = _log_int(rng, 1, max(1, min(8192, 400000000 // (c["n"] * row))))
    c["past_lo"] = c["past_hi"] // rng.choice((1, 4, 16))
    c["pre_hi"] = _log_int(rng, 100, max(100, min(40000, 150000000 // (c["groups"] * row), 192 * 20000 * 32 // (c["n"] * c["q_hi"] * c["Hq"]))))
    c["pre_lo"] = max(1, c["pre_hi"] // rng.choice((1, 4)))
    return c


def _dtype(case):
    return {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}[case["dtype"]]


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=_DEV)


def _cu(lens):
    return [sum(lens[:i]) for i in range(len(lens) + 1)]


def _gen(seed):
    return torch.Generator(device=_DEV).manual_seed(seed)


# ---- lengths, all from the case alone -----------------------------------------------------------------------------------------
def _table_lens(case):
    """(rows held, new tokens, pages held) of every sequence; some hold pages for rows that a check of drafts took back."""
    r, S = random.Random(case["lens"]), case["page"]
    out = []
    for _ in range(case["n"]):
        past, new = r.randint(case["past_lo"], case["past_hi"]), r.randint(case["new_lo"], case["new_hi"])
        out.append((past, new, -(-past // S) + (past > 0 and r.random() < 0.2)))
    return out


def _ended(case):
    """(rows held, rows kept, first pages that a window gave back) of every sequence."""
    r = random.Random(case["lens"])
    out = []
    for _ in range(case["n"]):
        past = r.randint(case["past_lo"], case["past_hi"])
        gone = past // 2 // case["page"] if case["gone"] and r.random() < 0.5 else 0
        out.append((past, 0 if r.random() < case["ends"] else past, gone))
    return out


def _members(case):
    """Sequences of every group, the ones without a group left out: the first so many of each size; sizes of two at least."""
    r = random.Random(case["lens"] + 1)
    left = case["n"] - case["alone"] - 2 * case["groups"]
    cuts = sorted(r.randint(0, left) for _ in range(case["groups"] - 1))
    return [2 + b - a for a, b in zip([0] + cuts, cuts + [left])]


def _shared_lens(case):
    """(rows of the shared prefix, own rows held, new tokens) of every sequence; a prefix is whole pages."""
    r, S = random.Random(case["lens"]), case["page"]
    out = []
    for m in _members(case):
        pre = max(1, r.randint(case["pre_lo"], case["pre_hi"]) // S) * S
        out += [(pre, r.randint(case["past_lo"], case["past_hi"]), r.randint(case["q_lo"], case["q_hi"])) for _ in range(m)]
    return out + [(0, r.randint(case["past_lo"], case["past_hi"]), r.randint(case["q_lo"], case["q_hi"])) for _ in range(case["alone"])]


def _drafts(case):
    r = random.Random(case["lens"])
    return [r.randint(case["d_lo"], case["d_hi"]) for _ in range(case["n"])]


# ---- inputs -------------------------------------------------------------------------------------------------------------------
def _prepare_tables(case, gen):
    lens, S, n = _table_lens(case), case["page"], case["n"]
    need = [max(-(-(past + new) // S), held) for past, new, held in lens]
    used, more = sum(h for _, _, h in lens), sum(w - h for w, (_, _, h) in zip(need, lens))
    free = more * 2 // 3 if case["short"] else more + 100
    n_pages = used + free
    order = torch.randperm(max(n_pages, 1), generator=gen, device=_DEV).to(torch.int32)
    table = torch.full((n, max(need + [1])), -1, dtype=torch.int32, device=_DEV)
    held = _i32([h for _, _, h in lens])
    there = torch.arange(table.shape[1], device=_DEV)[None, :] < held[:, None]
    table[there] = order[:used]
    # the ring of free pages goes on from its end to its start
    head = int(torch.randint(0, max(n_pages, 1), (1,), generator=gen, device=_DEV))
    ring = torch.full_like(order, -1)
    ring[(head + torch.arange(free, device=_DEV)) % max(n_pages, 1)] = order[used:used + free]
    T = sum(new for _, new, _ in lens)
    return {"table": table, "held": held, "ring": ring, "state": _i32([head, free, 0]), "past": _i32([p for p, _, _ in lens]),
            "new": _i32([w for _, w, _ in lens]), "cu": _i32([0] * (n + 1)), "ctx": _i32([0] * n), "held_after": _i32([0] * n),
            "state_after": _i32([0] * 3), "slots": torch.zeros(T, dtype=torch.int64, device=_DEV)}


def _prepare_release(case, gen):
    lens, S, n = _ended(case), case["page"], case["n"]
    held = [-(-past // S) for past, _, _ in lens]
    used = sum(h - g for h, (_, _, g) in zip(held, lens))
    free = max(16, used // 3)
    n_pages = used + free
    order = torch.randperm(n_pages, generator=gen, device=_DEV).to(torch.int32)
    at = torch.arange(max(held), device=_DEV)[None, :]
    there = (at < _i32(held)[:, None]) & (at >= _i32([g for _, _, g in lens])[:, None])
    table = torch.full((n, max(held)), -1, dtype=torch.int32, device=_DEV)
    table[there] = order[:used]
    head = int(torch.randint(0, n_pages, (1,), generator=gen, device=_DEV))
    ring = torch.full_like(order, -1)
    ring[(head + torch.arange(free, device=_DEV)) % n_pages] = order[used:]
    return {"table": table, "held": _i32(held), "ring": ring, "state": _i32([head, free, 0]), "keep": _i32([k for _, k, _ in lens]),
            "held_after": _i32([0] * n), "state_after": _i32([0] * 3)}


def _needed(amax):
    """The least e with amax <= 448 * 2^e, as a whole number; -100 for no value at all."""
    m, e = torch.frexp(amax)
    e = torch.where(m <= 0.875, e - 9, e - 8).clamp(-100, 119)
    return torch.where(amax > 0, e, torch.full_like(e, -100))


def _prepare_shared(case, gen):
    n, Hq, Hkv, D, S, dtype = case["n"], case["Hq"], case["Hkv"], case["D"], case["page"], _dtype(case)
    lens, members = _shared_lens(case), _members(case)
    first = _cu(members)
    ends = [-(-(pre + past + q) // S) for pre, past, q in lens]
    prefixes = [lens[f][0] for f in first[:-1]]
    n_pages = sum(p // S for p in prefixes) + sum(e - pre // S for e, (pre, _, _) in zip(ends, lens))
    order = torch.randperm(n_pages, generator=gen, device=_DEV).to(torch.int32)
    table = torch.full((n, max(ends)), -1, dtype=torch.int32, device=_DEV)
    taken = 0
    for f, m, p in zip(first, members, prefixes):
        table[f:f + m, :p // S] = order[taken:taken + p // S]
        taken += p // S
    for s, (e, (pre, _, _)) in enumerate(zip(ends, lens)):
        table[s, pre // S:e] = order[taken:taken + e - pre // S]
        taken += e - pre // S

    def rnd(*shape):
        return torch.randn(*shape, generator=gen, device=_DEV, dtype=dtype)

    # a model's keys have a few channels that are far larger than the others
    loud = 1.0 + 7.0 * (torch.rand(Hkv, 1, D, generator=gen, device=_DEV) < 0.02).to(dtype)
    T = sum(q for _, _, q in lens)
    s = {"table": table, "cu": _i32(_cu([q for _, _, q in lens])), "ctx": _i32([sum(x) for x in lens]), "max_q": max(q for _, _, q in lens),
         "cu_groups": _i32(first), "prefix": _i32(prefixes), "k_pages": rnd(n_pages, Hkv, S, D) * loud.to(dtype), "v_pages": rnd(n_pages, Hkv, S, D),
         "q": rnd(1, T, Hq, D), "out": torch.empty(1, T, Hq, D, dtype=dtype, device=_DEV)}
    if case["cache"] == "fp8":
        for name in ("k", "v"):
            x = s[name + "_pages"]
            e = _needed(x.abs().amax(dim=(2, 3)).float())
            s[name + "_scales"] = (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)
            s[name + "_pages"] = (x.float() * torch.exp2(-e.float())[:, :, None, None]).clamp(-448, 448).to(torch.float8_e4m3fn)
    # rows that nothing was written to: behind the last one in its page
    page = table.gather(1, (s["ctx"].long()[:, None] // S).clamp(max=table.shape[1] - 1)).flatten()
    behind = (torch.arange(S, device=_DEV)[None, :] >= (s["ctx"] % S)[:, None]) & (s["ctx"] % S > 0)[:, None]
    at, row = behind.nonzero(as_tuple=True)
    for name in ("k_pages", "v_pages"):
        raw = s[name].view(torch.uint8 if case["cache"] == "fp8" else torch.int16)
        raw[page[at].long(), :, row] = 0x7F if case["cache"] == "fp8" else 0x7FFF   # a NaN in all three types
    return s


def _prepare_verify(case, gen):
    drafts, V, dtype = _drafts(case), case["V"], _dtype(case)
    cu = _cu([d + 1 for d in drafts])
    T = cu[-1]
    # a model's next token is mostly one of a few; its drafter agrees with it more or less
    logits = 3.0 * torch.randn(T, V, generator=gen, device=_DEV)
    s = {"cu": _i32(cu), "target": torch.softmax(logits, -1).to(dtype), "draft": None,
         "accept_u": torch.rand(T, generator=gen, device=_DEV), "sample_u": torch.rand(case["n"], generator=gen, device=_DEV),
         "out": torch.zeros(T, dtype=torch.int64, device=_DEV), "accepted": _i32([0] * case["n"])}
    logits += (1.5 if case["drafter"] else 0.0) * torch.randn(T, V, generator=gen, device=_DEV)
    q = torch.softmax(logits, -1)
    if case["drafter"]:
        s["draft"] = q.to(dtype)
    pick = (torch.rand(T, 1, generator=gen, device=_DEV, dtype=torch.float64) * 0.999999 < torch.cumsum(q.double(), -1)).int().argmax(-1)
    s["tokens"] = torch.randint(0, V, (T,), generator=gen, device=_DEV)
    s["tokens"][1:] = pick[:-1]
    return s


def prepare(case, seed):
    make = {"tables": _prepare_tables, "release": _prepare_release, "shared": _prepare_shared, "verify": _prepare_verify}[case["kind"]]
    return {"case": case, **make(case, _gen(seed))}


# ---- the framework's kernels ------------------------------------------------------------------------------------------------
def _kernels():
    pkg = os.path.abspath("minfer-python_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from minfer.const import GGML_QUANT_SIZES, GGMLQuantizationType
    from minfer.kernels import KernelBackend
    return KernelBackend("torch_ext"), {d: (int(t), *GGML_QUANT_SIZES[t]) for d, t in (("f16", GGMLQuantizationType.F16), ("bf16", GGMLQuantizationType.BF16))}


_made = []


def _own(s):
    if not _made:
        _made.append(_kernels())
    kerns, types = _made[0]
    case = s["case"]
    if case["kind"] == "tables":
        kerns.paged_tables(case["page"], s["past"], s["new"], s["held"], s["ring"], s["state"], s["table"], s["cu"], s["ctx"], s["slots"],
                           s["held_after"], s["state_after"])
    elif case["kind"] == "release":
        kerns.paged_release(case["page"], s["keep"], s["held"], s["table"], s["ring"], s["state"], s["held_after"], s["state_after"])
    elif case["kind"] == "verify":
        kerns.verify_drafts(s["tokens"], s["cu"], s["target"], s["draft"], s["accept_u"], s["sample_u"], s["out"], s["accepted"])
    else:
        eight = case["cache"] == "fp8"
        call = kerns.flash_attn_paged_shared_fp8 if eight else kerns.flash_attn_paged_shared
        call(*types[case["dtype"]], s["q"].transpose(1, 2), s["k_pages"], s["v_pages"], *((s["k_scales"], s["v_scales"]) if eight else ()), s["table"],
             s["cu"], s["ctx"], s["cu_groups"], s["prefix"], s["max_q"], s["out"].transpose(1, 2))


# ---- the plain forms --------------------------------------------------------------------------------------------------------
def _exclusive(x):
    return torch.cumsum(x, 0) - x


def _places(cu, T):
    """Sequence of every packed token and its number inside the sequence."""
    t = torch.arange(T, device=_DEV)
    seq = torch.searchsorted(cu, t, right=True) - 1
    return seq, t - cu[seq]


def _plain_tables(s):
    S, (n, W) = s["case"]["page"], s["table"].shape
    past, new, held = s["past"].long(), s["new"].long(), s["held"].long()
    head, count, N = s["state"][0].long(), s["state"][1].long(), s["ring"].numel()
    need = torch.clamp((past + new + S - 1) // S, max=W)
    take = torch.clamp(need - held, min=0)
    off = _exclusive(take)
    cu = torch.cat((torch.zeros(1, dtype=torch.long, device=_DEV), torch.cumsum(new, 0)))
    s["cu"].copy_(cu)
    s["ctx"].copy_(past + new)
    at = torch.arange(W, device=_DEV)[None, :] - held[:, None]
    number = off[:, None] + at
    fresh = (at >= 0) & (at < take[:, None])
    page = torch.where(number < count, s["ring"][(head + number) % N], -1)
    s["table"].copy_(torch.where(fresh, page, s["table"]))
    total = take.sum()
    taken = torch.minimum(total, count)
    s["held_after"].copy_(held + torch.minimum(take, torch.clamp(count - off, min=0)))
    s["state_after"].copy_(torch.stack(((head + taken) % N, count - taken, total - taken)))
    seq, i = _places(cu, s["slots"].numel())
    row = past[seq] + i
    page = torch.where(row < W * S, s["table"][seq, torch.clamp(row // S, max=W - 1)].long(), -1)
    s["slots"].copy_(torch.where(page >= 0, page * S + row % S, -1))


def _plain_release(s):
    S, W = s["case"]["page"], s["table"].shape[1]
    held = s["held"].long()
    head, count, N = s["state"][0].long(), s["state"][1].long(), s["ring"].numel()
    stay = torch.minimum((s["keep"].long() + S - 1) // S, held)
    at = torch.arange(W, device=_DEV)[None, :]
    given = (at >= stay[:, None]) & (at < held[:, None]) & (s["table"] >= 0) & (s["table"] < N)
    number = torch.cumsum(given.flatten(), 0) - 1
    pages = s["table"].flatten()
    place = (head + count + number) % N
    at = given.flatten().nonzero().flatten()
    s["ring"][place[at]] = pages[at]
    s["held_after"].copy_(stay)
    s["state_after"].copy_(torch.stack((head, count + given.sum(), torch.zeros_like(count))))


def _rows(s, name, table, lo, hi):
    """Rows lo .. hi - 1 (whole pages) of a table's sequences, [sequences, Hkv, rows, D] in 32 bits."""
    pages, S = s[name + "_pages"], s["case"]["page"]
    ids = table[:, lo // S:hi // S].long().clamp(min=0)
    if s["case"]["cache"] == "fp8":
        x = pages.view(torch.uint8)[ids].view(torch.float8_e4m3fn).float() * s[name + "_scales"].float()[ids][..., None, None]
    else:
        x = pages[ids].float()
    return x.permute(0, 2, 1, 3, 4).flatten(2, 3)


def _plain_shared(s):
    """Group by group: the prefix's scores with all the group's tokens in one product, the sequences' own rows one sequence beside the other."""
    case = s["case"]
    Hq, Hkv, D, S = case["Hq"], case["Hkv"], case["D"], case["page"]
    lens, members = _shared_lens(case), _members(case)
    rep, at, t0 = Hq // Hkv, 0, 0
    for m in members + ([case["alone"]] if case["alone"] else []):
        part = lens[at:at + m]
        pre, most, width = part[0][0], max(q for _, _, q in part), max(-(-sum(x) // S) * S for x in part)
        count = sum(q for _, _, q in part)
        table, ctx = s["table"][at:at + m], s["ctx"][at:at + m].long()
        seq, i = _places(s["cu"][at:at + m + 1].long() - t0, count)
        q = torch.zeros(m, most, Hkv, rep, D, device=_DEV)
        q[seq, i] = s["q"][0, t0:t0 + count].float().view(count, Hkv, rep, D) * D ** -0.5
        q = q.permute(2, 0, 1, 3, 4).reshape(Hkv, m, most * rep, D)
        rows = torch.arange(pre, width, device=_DEV)
        k, v = (torch.where((rows < ctx[:, None])[:, None, :, None], _rows(s, name, table, pre, width), 0.0) for name in ("k", "v"))
        ends = ctx - (s["cu"][at + 1:at + m + 1] - s["cu"][at:at + m]).long()
        pos = (ends[:, None] + torch.arange(most, device=_DEV)).repeat_interleave(rep, 1)                         # [m, most * rep]
        score = torch.matmul(q, k.transpose(0, 1).transpose(-1, -2))                                              # [Hkv, m, most * rep, own rows]
        score = torch.where(rows <= pos[..., None], score, -math.inf)
        top = score.amax(-1, keepdim=True)
        if pre:
            k0, v0 = (_rows(s, name, table[:1], 0, pre)[0] for name in ("k", "v"))
            score0 = torch.matmul(q.flatten(1, 2), k0.transpose(-1, -2)).view(*q.shape[:3], pre)
            top = torch.maximum(top, score0.amax(-1, keepdim=True))
        weight = torch.exp(score - top)
        y, total = torch.matmul(weight, v.transpose(0, 1)), weight.sum(-1, keepdim=True)
        if pre:
            weight = torch.exp(score0 - top)
            y = y + torch.matmul(weight.flatten(1, 2), v0).view_as(y)
            total = total + weight.sum(-1, keepdim=True)
        y = (y / total).view(Hkv, m, most, rep, D).permute(1, 2, 0, 3, 4).reshape(m, most, Hq, D)
        s["out"][0, t0:t0 + count] = y[seq, i].to(s["out"].dtype)
        at, t0 = at + m, t0 + count


def _plain_verify(s):
    cu, T = s["cu"].long(), s["tokens"].numel()
    n, V = cu.numel() - 1, s["target"].shape[1]
    seq, i = _places(cu, T)
    last = cu[1:] - 1
    checked = torch.cat((s["tokens"][1:], s["tokens"][:1]))                 # the draft that row t decides about
    p = s["target"].gather(1, checked[:, None])[:, 0].double()
    q = s["draft"].gather(1, checked[:, None])[:, 0].double() if s["draft"] is not None else torch.ones_like(p)
    yes = (s["accept_u"].double() * q < p) & (torch.arange(T, device=_DEV) < last[seq])
    refused = torch.where(yes, T, i)
    accepted = torch.full((n,), T, device=_DEV).scatter_reduce(0, seq, refused, "amin")
    row = cu[:-1] + accepted
    p = s["target"][row].double()
    q = s["draft"][row].double() if s["draft"] is not None else torch.zeros_like(p).scatter_(1, checked[row][:, None], 1.0)
    some = accepted < last - cu[:-1]
    weight = torch.where(some[:, None], torch.clamp(p - q, min=0.0), p)
    weight = torch.where(weight.sum(-1, keepdim=True) > 0, weight, p)
    upto = torch.cumsum(weight, -1)
    over = upto > s["sample_u"].double()[:, None] * upto[:, -1:]
    picked = over.int().argmax(-1)
    a = accepted[seq]
    s["out"].copy_(torch.where(i < a, checked, torch.where(i == a, picked[seq], -1)))
    s["accepted"].copy_(accepted)


def run(s):
    kind = s["case"]["kind"]
    if own:
        _own(s)
    else:
        {"tables": _plain_tables, "release": _plain_release, "shared": _plain_shared, "verify": _plain_verify}[kind](s)
    if kind == "shared":
        return s["out"]
    names = {"tables": ("cu", "ctx", "slots", "table", "held_after", "state_after"), "release": ("ring", "held_after", "state_after"),
             "verify": ("out", "accepted")}[kind]
    return {name: s[name] for name in names}


def work(case):
    n = case["n"]
    if case["kind"] == "tables":
        lens = _table_lens(case)
        fresh = sum(max(-(-(past + new) // case["page"]) - held, 0) for past, new, held in lens)
        return {"bytes": 20 * n + 8 * fresh + 8 * sum(new for _, new, _ in lens), "flops": 10 * n + 5 * sum(new for _, new, _ in lens)}
    if case["kind"] == "release":
        given = sum(-(-past // case["page"]) for past, keep, _ in _ended(case) if keep == 0)
        return {"bytes": 12 * n + 8 * given, "flops": 5 * n + 3 * given}
    if case["kind"] == "verify":
        drafts, width = _drafts(case), 4 if case["dtype"] == "f32" else 2
        return {"bytes": n * case["V"] * width * (2 if case["drafter"] else 1) + 40 * sum(d + 1 for d in drafts), "flops": 4 * n * case["V"]}
    lens, width = _shared_lens(case), 1 if case["cache"] == "fp8" else 2
    rows = sum(past + q for _, past, q in lens) + sum(lens[f][0] for f in _cu(_members(case))[:-1])
    pairs = sum(q * (pre + past) + q * (q + 1) // 2 for pre, past, q in lens)
    return {"bytes": 2 * rows * case["Hkv"] * case["D"] * width + 2 * sum(q for _, _, q in lens) * case["Hq"] * case["D"] * 2,
            "flops": 4 * case["D"] * case["Hq"] * pairs}


# ---- the definitions, one sequence after the other ----------------------------------------------------------------------------
def _exact_tables(s):
    S, lens = s["case"]["page"], list(zip(s["past"].tolist(), s["new"].tolist(), s["held"].tolist()))
    table, ring = s["table"].tolist(), s["ring"].tolist()
    head, count, _ = s["state"].tolist()
    at, lacking, cu, ctx, slots, held_after = 0, 0, [0], [], [], []
    for row, (past, new, held) in zip(table, lens):
        for p in range(held, min(-(-(past + new) // S), len(row))):
            if at < count:
                row[p] = ring[(head + at) % len(ring)]
                at, held = at + 1, held + 1
            else:
                row[p] = -1
                lacking += 1
        held_after.append(held)
        cu.append(cu[-1] + new)
        ctx.append(past + new)
        slots += [row[r // S] * S + r % S if r // S < len(row) and row[r // S] >= 0 else -1 for r in range(past, past + new)]
    return {"cu": _i32(cu), "ctx": _i32(ctx), "slots": torch.tensor(slots, dtype=torch.int64, device=_DEV), "table": _i32(table),
            "held_after": _i32(held_after), "state_after": _i32([(head + at) % len(ring), count - at, lacking])}


def _exact_release(s):
    S, ring, held_after = s["case"]["page"], s["ring"].tolist(), []
    head, count, _ = s["state"].tolist()
    for row, keep, held in zip(s["table"].tolist(), s["keep"].tolist(), s["held"].tolist()):
        stay = min(-(-keep // S), held)
        for page in row[stay:held]:
            if 0 <= page < len(ring):
                ring[(head + count) % len(ring)] = page
                count += 1
        held_after.append(stay)
    return {"ring": _i32(ring), "held_after": _i32(held_after), "state_after": _i32([head, count, 0])}


def _exact_shared(s):
    case = s["case"]
    Hkv, D, S = case["Hkv"], case["D"], case["page"]
    table, ctx, cu = s["table"].tolist(), s["ctx"].tolist(), s["cu"].tolist()
    out = torch.empty(1, cu[-1], case["Hq"], D, dtype=torch.float64, device=_DEV)
    for n, (row, c) in enumerate(zip(table, ctx)):
        ids = torch.tensor(row[:-(-c // S)], device=_DEV)
        both = []
        for name in ("k", "v"):
            x = s[name + "_pages"].view(torch.uint8)[ids].view(torch.float8_e4m3fn).double() if case["cache"] == "fp8" else s[name + "_pages"][ids].double()
            if case["cache"] == "fp8":
                x = x * torch.exp2(s[name + "_scales"].view(torch.uint8)[ids].double() - 127)[:, :, None, None]
            both.append(x.transpose(0, 1).flatten(1, 2)[:, :c].contiguous())
        q = s["q"][0, cu[n]:cu[n + 1]].double().unflatten(1, (Hkv, -1)).permute(1, 2, 0, 3)                      # [Hkv, heads, tokens, D]
        score = torch.matmul(q.flatten(1, 2), both[0].transpose(1, 2).contiguous()).unflatten(1, q.shape[1:3]) / math.sqrt(D)
        position = torch.arange(c - q.shape[2], c, device=_DEV)
        weight = torch.softmax(score.masked_fill(torch.arange(c, device=_DEV)[None, :] > position[:, None], -math.inf), -1)
        out[0, cu[n]:cu[n + 1]] = torch.matmul(weight.flatten(1, 2), both[1]).unflatten(1, q.shape[1:3]).permute(2, 0, 1, 3).flatten(1, 2)
    return out


def _exact_verify(s):
    cu, tokens, u = s["cu"].tolist(), s["tokens"].tolist(), s["accept_u"].tolist()
    out, accepted = [], []
    for n, (lo, hi) in enumerate(zip(cu, cu[1:])):
        a = 0
        while lo + a < hi - 1:
            x = tokens[lo + a + 1]
            q = float(s["draft"][lo + a, x]) if s["draft"] is not None else 1.0
            if not u[lo + a] * q < float(s["target"][lo + a, x]):
                break
            a += 1
        weight = s["target"][lo + a].double()
        if lo + a < hi - 1:
            q = s["draft"][lo + a].double() if s["draft"] is not None else torch.nn.functional.one_hot(torch.tensor(tokens[lo + a + 1], device=_DEV), weight.numel())
            left = (weight - q).clamp(min=0)
            weight = left if float(left.sum()) > 0 else weight
        sums = weight.cumsum(0)
        chosen = int(torch.searchsorted(sums, sums[-1:] * float(s["sample_u"][n]), right=True)[0])
        out += tokens[lo + 1:lo + a + 1] + [chosen] + [-1] * (hi - lo - a - 1)
        accepted.append(a)
    return {"out": torch.tensor(out, dtype=torch.int64, device=_DEV), "accepted": _i32(accepted)}


def exact(case, seed):
    s = prepare(case, seed)
    return {"tables": _exact_tables, "release": _exact_release, "shared": _exact_shared, "verify": _exact_verify}[case["kind"]](s)
