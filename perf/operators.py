"""Attention over a paged KV cache and the steps that fill it, as cases that can be timed and compared.

A serving program keeps the keys and values of many sequences in pages of `page` rows and a table of pages per sequence.  The
tokens of a step are packed, [1, T, heads, head_dim] with `cu_seqlens`: one new token of every sequence, a few (drafts that are
checked together), or a chunk of a prompt.  The append rotates q in place and writes the rotated k and the v into the pages; the
attention lets every new token see the cached rows up to itself.  Pages hold 16-bit rows, or 8-bit ones (e4m3) with a power of two
as the scale of each page and head.

Pages lie in the pool in no order.  Rows behind a sequence's last one were never written: they hold NaN here.  With `evicted`, the
first pages of long sequences are gone (a window that moved on): their entries in the table are -1 and nothing attends them.
"""
import math
import os
import random
import sys

import torch

own = False

_DEV = "cuda"
_BASE = 5e5      # rotary frequency base
_E4M3 = 448.0    # largest e4m3 number, 1.75 * 2^8

# (query heads, KV heads) of the models' layers
_HEADS = ((8, 2), (16, 16), (24, 8), (32, 8), (48, 8), (64, 8))


def listed():
    return [
        # one decode step of a serving batch
        {"name": "append_step", "kind": "append", "n": 64, "q_lo": 1, "q_hi": 1, "past_lo": 512, "past_hi": 8191, "lens": 1, "Hq": 32, "Hkv": 8,
         "D": 128, "rd": 128, "style": 1, "page": 16, "dtype": "bf16", "cache": "16"},
        # prompts of no round length, at the head count and rotary width of the repository's own rope benchmark
        {"name": "append_prompts", "kind": "append", "n": 6, "q_lo": 200, "q_hi": 2048, "past_lo": 0, "past_hi": 0, "lens": 2, "Hq": 48, "Hkv": 8,
         "D": 128, "rd": 64, "style": 0, "page": 64, "dtype": "f16", "cache": "16"},
        # one decode step into 8-bit pages
        {"name": "append8_step", "kind": "append", "n": 40, "q_lo": 1, "q_hi": 1, "past_lo": 20, "past_hi": 1100, "lens": 3, "Hq": 32, "Hkv": 8,
         "D": 128, "rd": 128, "style": 1, "page": 32, "dtype": "f16", "cache": "fp8"},
        # chunks of prompts that go on in pages others began
        {"name": "append8_chunks", "kind": "append", "n": 5, "q_lo": 300, "q_hi": 1500, "past_lo": 0, "past_hi": 700, "lens": 4, "Hq": 64, "Hkv": 8,
         "D": 128, "rd": 128, "style": 1, "page": 16, "dtype": "bf16", "cache": "fp8"},
        # one user of a small model; the smallest call, latency only
        {"name": "attend_single", "kind": "attend", "n": 1, "q_lo": 1, "q_hi": 1, "past_lo": 1500, "past_hi": 1500, "lens": 5, "Hq": 8, "Hkv": 2,
         "D": 64, "page": 16, "dtype": "f16", "cache": "16", "evicted": False},
        # one decode step's attention of a full serving batch
        {"name": "attend_batch", "kind": "attend", "n": 64, "q_lo": 1, "q_hi": 1, "past_lo": 511, "past_hi": 8191, "lens": 6, "Hq": 32, "Hkv": 8,
         "D": 128, "page": 16, "dtype": "bf16", "cache": "16", "evicted": False},
        # drafts of three and four tokens checked together
        {"name": "attend_drafts", "kind": "attend", "n": 12, "q_lo": 3, "q_hi": 4, "past_lo": 200, "past_hi": 6000, "lens": 7, "Hq": 32, "Hkv": 8,
         "D": 128, "page": 32, "dtype": "f16", "cache": "16", "evicted": False},
        # chunks of prompts behind cached rows, three query heads to a KV head
        {"name": "attend_chunks", "kind": "attend", "n": 4, "q_lo": 100, "q_hi": 777, "past_lo": 500, "past_hi": 8000, "lens": 8, "Hq": 24, "Hkv": 8,
         "D": 128, "page": 64, "dtype": "bf16", "cache": "16", "evicted": False},
        # a whole long prompt; the largest case
        {"name": "attend_prompt", "kind": "attend", "n": 1, "q_lo": 8192, "q_hi": 8192, "past_lo": 0, "past_hi": 0, "lens": 9, "Hq": 32, "Hkv": 8,
         "D": 128, "page": 128, "dtype": "f16", "cache": "16", "evicted": False},
        # a few conversations over 8-bit pages
        {"name": "attend8_few", "kind": "attend", "n": 3, "q_lo": 1, "q_hi": 1, "past_lo": 200, "past_hi": 2999, "lens": 10, "Hq": 32, "Hkv": 8,
         "D": 128, "page": 64, "dtype": "f16", "cache": "fp8", "evicted": False},
        # the serving batch's step over 8-bit pages
        {"name": "attend8_batch", "kind": "attend", "n": 64, "q_lo": 1, "q_hi": 1, "past_lo": 511, "past_hi": 8191, "lens": 6, "Hq": 32, "Hkv": 8,
         "D": 128, "page": 32, "dtype": "f16", "cache": "fp8", "evicted": False},
        # chunks of long prompts whose first pages a window has left behind
        {"name": "attend8_chunks", "kind": "attend", "n": 2, "q_lo": 600, "q_hi": 1024, "past_lo": 2000, "past_hi": 8000, "lens": 12, "Hq": 64, "Hkv": 8,
         "D": 128, "page": 16, "dtype": "bf16", "cache": "fp8", "evicted": True},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    Hq, Hkv = rng.choice(_HEADS)
    D = rng.choice((64, 128, 128))
    c = {"kind": rng.choice(("append", "attend", "attend")), "n": _log_int(rng, 1, 64)}
    form = rng.choice(("one", "one", "few", "chunk"))
    c["q_hi"] = 1 if form == "one" else rng.randint(2, 9) if form == "few" else _log_int(rng, 16, 4096)
    if form == "chunk":
        c["n"] = max(1, min(c["n"], 8192 // c["q_hi"]))
    c["q_lo"] = max(1, c["q_hi"] // rng.choice((1, 2, 8)))
    c["lens"] = rng.randrange(1 << 20)
    c.update(Hq=Hq, Hkv=Hkv, D=D, page=rng.choice((16, 16, 32, 64, 128, 256)), dtype=rng.choice(("f16", "bf16")), cache=rng.choice(("16", "fp8")))
    if c["kind"] == "append":
        c["past_hi"] = rng.choice((0, _log_int(rng, 1, 100000)))
        c["past_lo"] = c["past_hi"] // rng.choice((1, 3, 20))
        c["rd"] = rng.choice((D, D, D // 2))
        c["style"] = rng.choice((0, 1))
        return c
    # rows of all sequences, and (query, key) pairs of all heads, within those of the largest listed cases
    most = min(65536, 64 * 8192 * 8 * 128 // (c["n"] * Hkv * D), 32 * 8192 * 8192 // (c["n"] * Hq * c["q_hi"])) - c["q_hi"]
    c["past_hi"] = _log_int(rng, 1, max(1, most))
    c["past_lo"] = c["past_hi"] // rng.choice((1, 4, 16))
    c["evicted"] = rng.random() < 0.25
    return c


def _dtype(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float16


def _lens(case):
    """(new tokens, cached rows before them) of every sequence."""
    r = random.Random(case["lens"])
    return [(r.randint(case["q_lo"], case["q_hi"]), r.randint(case["past_lo"], case["past_hi"])) for _ in range(case["n"])]


def _first_page(case, past):
    """The first page of a sequence that is in the pool: an append's call looks at no page in front of the one that it goes on
    in, and a window of half the rows has left the others behind."""
    if case["kind"] == "append":
        return past // case["page"]
    return past // 2 // case["page"] if case["evicted"] else 0


def _table(case, gen):
    """Block table [n, most pages] with -1 where no page is, and the number of pages in the pool."""
    S, at, width, used = case["page"], [], 0, 0
    for q, past in _lens(case):
        last = (past + q + S - 1) // S
        at.append((_first_page(case, past), last))
        width = max(width, last)
        used += last - at[-1][0]
    order = torch.randperm(used, generator=gen, device=_DEV).to(torch.int32)
    table = torch.full((case["n"], width), -1, dtype=torch.int32, device=_DEV)
    taken = 0
    for s, (first, last) in enumerate(at):
        table[s, first:last] = order[taken:taken + last - first]
        taken += last - first
    return table, used


def _needed(amax):
    """The least e with amax <= 448 * 2^e, as a whole number; -100 for no value at all."""
    m, e = torch.frexp(amax)
    e = torch.where(m <= 0.875, e - 9, e - 8).clamp(-100, 119)
    return torch.where(amax > 0, e, torch.full_like(e, -100))


def _codes(x, e):
    """x as e4m3 codes of the scale 2^e."""
    return (x.float() * torch.exp2(-e.float())).clamp(-_E4M3, _E4M3).to(torch.float8_e4m3fn)


def _to_e8m0(e):
    return (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def _exponents(scales):
    return scales.view(torch.uint8).to(torch.int32) - 127


def _values(pages, scales, dtype):
    """What 8-bit pages stand for."""
    return pages.to(dtype) * scales.to(dtype)[:, :, None, None]


def prepare(case, seed):
    n, Hq, Hkv, D, S, dtype = case["n"], case["Hq"], case["Hkv"], case["D"], case["page"], _dtype(case)
    gen = torch.Generator(device=_DEV).manual_seed(seed)

    def rnd(*shape):
        return torch.randn(*shape, generator=gen, device=_DEV, dtype=dtype)

    lens = _lens(case)
    T = sum(q for q, _ in lens)
    cu = [sum(q for q, _ in lens[:i]) for i in range(n + 1)]
    table, n_pages = _table(case, gen)
    # a model's keys have a few channels that are far larger than the others
    loud = 1.0 + 7.0 * (torch.rand(Hkv, 1, D, generator=gen, device=_DEV) < 0.02).to(dtype)
    k_pages, v_pages = rnd(n_pages, Hkv, S, D) * loud.to(dtype), rnd(n_pages, Hkv, S, D)
    s = {"case": case, "table": table, "max_q": max(q for q, _ in lens),
         "cu": torch.tensor(cu, dtype=torch.int32, device=_DEV),
         "past": torch.tensor([p for _, p in lens], dtype=torch.int32, device=_DEV),
         "ctx": torch.tensor([q + p for q, p in lens], dtype=torch.int32, device=_DEV)}
    if case["cache"] == "fp8":
        for name, pages in (("k", k_pages), ("v", v_pages)):
            e = _needed(pages.abs().amax(dim=(2, 3)).float())
            s[name + "_scales"] = _to_e8m0(e)
            pages = _codes(pages, e[:, :, None, None])
            s[name + "_pages"] = pages
    else:
        s["k_pages"], s["v_pages"] = k_pages, v_pages
    # rows that nothing was written to: behind the last one in its page
    held = s["past"] if case["kind"] == "append" else s["ctx"]
    page = table.gather(1, (held.long()[:, None] // S).clamp(max=table.shape[1] - 1)).flatten()
    behind = torch.arange(S, device=_DEV)[None, :] >= (held % S)[:, None]
    behind &= (held % S > 0)[:, None]
    at, row = (behind & (page >= 0)[:, None]).nonzero(as_tuple=True)
    for name in ("k_pages", "v_pages"):
        raw = s[name].view(torch.uint8 if case["cache"] == "fp8" else torch.int16)
        raw[page[at].long(), :, row] = 0x7F if case["cache"] == "fp8" else 0x7FFF   # a NaN in all three types
    s["q"] = rnd(1, T, Hq * D).view(1, T, Hq, D)
    if case["kind"] == "append":
        s["k"] = (rnd(1, T, Hkv, D) * loud.view(Hkv, D)).contiguous()
        s["v"] = rnd(1, T, Hkv, D)
    else:
        s["out"] = torch.empty(1, T, Hq, D, dtype=dtype, device=_DEV)
    return s


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
    eight = case["cache"] == "fp8"
    scales = (s["k_scales"], s["v_scales"]) if eight else ()
    if case["kind"] == "append":
        call = kerns.rope_kv_append_paged_fp8 if eight else kerns.rope_kv_append_paged
        call(case["style"], case["rd"], _BASE, s["q"], s["k"], s["v"], s["cu"], s["past"], s["table"], s["k_pages"], s["v_pages"], *scales)
    else:
        call = kerns.flash_attn_paged_fp8 if eight else kerns.flash_attn_paged
        call(*types[case["dtype"]], s["q"].transpose(1, 2), s["k_pages"], s["v_pages"], *scales, s["table"], s["cu"], s["ctx"], s["max_q"],
             s["out"].transpose(1, 2))


# ---- the plain forms --------------------------------------------------------------------------------------------------------
def _places(s, T):
    """Sequence of every packed token and its number inside the sequence."""
    t = torch.arange(T, device=_DEV)
    seq = torch.searchsorted(s["cu"].long(), t, right=True) - 1
    return seq, t - s["cu"].long()[seq]


def _rotated(x, pos, case):
    """x [T, H, D] in 32 bits, rotated to the positions; the angles in 64."""
    rd = case["rd"]
    freq = _BASE ** (-2.0 * torch.arange(rd // 2, device=_DEV, dtype=torch.float64) / rd)
    angle = pos.double()[:, None] * freq
    c, n = torch.cos(angle).float()[:, None, :], torch.sin(angle).float()[:, None, :]
    x = x.float()
    a, b = (x[..., 0:rd:2], x[..., 1:rd:2]) if case["style"] == 0 else (x[..., :rd // 2], x[..., rd // 2:rd])
    lo, hi = c * a - n * b, n * a + c * b
    both = torch.stack((lo, hi), dim=-1).flatten(-2) if case["style"] == 0 else torch.cat((lo, hi), dim=-1)
    return torch.cat((both, x[..., rd:]), dim=-1)


def _plain_append(s):
    case, S = s["case"], s["case"]["page"]
    T = s["q"].shape[1]
    seq, i = _places(s, T)
    pos = s["past"].long()[seq] + i
    page, row = s["table"][seq, pos // S].long(), pos % S
    s["q"].copy_(_rotated(s["q"][0], pos, case)[None])
    new = {"k": _rotated(s["k"][0], pos, case).to(_dtype(case)), "v": s["v"][0]}
    if case["cache"] != "fp8":
        s["k_pages"][page, :, row] = new["k"]
        s["v_pages"][page, :, row] = new["v"]
        return
    n_pages, Hkv = s["k_pages"].shape[:2]
    # rows that a page held before the call: those of the page that a sequence goes on in
    held = torch.zeros(n_pages, dtype=torch.long, device=_DEV)
    held.index_put_((page,), torch.where(pos // S == s["past"].long()[seq] // S, s["past"].long()[seq] % S, 0))
    written = torch.zeros(n_pages, dtype=torch.bool, device=_DEV).index_fill_(0, page, True)
    older = (torch.arange(S, device=_DEV)[None, :] < held[:, None])[:, None, :, None]
    for name in ("k", "v"):
        pages, scales = s[name + "_pages"], s[name + "_scales"]
        amax = torch.zeros(n_pages, Hkv, device=_DEV).index_reduce_(0, page, new[name].float().abs().amax(-1), "amax")
        e_old, e_new = _exponents(scales), _needed(amax)
        e_new = torch.where((held > 0)[:, None], torch.maximum(e_old, e_new), e_new)
        e_new = torch.where(written[:, None], e_new, e_old)
        moved = (pages.float() * torch.exp2((e_old - e_new).float())[:, :, None, None]).to(torch.float8_e4m3fn)
        raw = torch.where(older, moved.view(torch.uint8), pages.view(torch.uint8))
        raw[page, :, row] = _codes(new[name], e_new[page][:, :, None]).view(torch.uint8)
        pages.view(torch.uint8).copy_(raw)
        scales.view(torch.uint8).copy_(_to_e8m0(e_new).view(torch.uint8))


def _gathered(s, name, kept):
    """Rows of every sequence, [n, Hkv, rows, D] in 32 bits; zero where a sequence has none."""
    pages, table = s[name + "_pages"], s["table"].long().clamp(min=0)
    n, P = table.shape
    _, Hkv, S, D = pages.shape
    if s["case"]["cache"] == "fp8":
        x = pages.view(torch.uint8)[table].view(torch.float8_e4m3fn).float() * s[name + "_scales"].float()[table][..., None, None]
    else:
        x = pages[table].float()
    x = x.permute(0, 2, 1, 3, 4).reshape(n, Hkv, P * S, D)
    return torch.where(kept[:, None, :, None], x, 0.0)


def _plain_attend(s):
    case = s["case"]
    n, Hq, Hkv, D, S, m = case["n"], case["Hq"], case["Hkv"], case["D"], case["page"], s["max_q"]
    cu, ctx = s["cu"].long(), s["ctx"].long()
    rows = s["table"].shape[1] * S
    key = torch.arange(rows, device=_DEV)
    kept = (s["table"] >= 0).repeat_interleave(S, dim=1) & (key < ctx[:, None])
    k, v = _gathered(s, "k", kept), _gathered(s, "v", kept)
    T = s["q"].shape[1]
    at = (cu[:-1, None] + torch.arange(m, device=_DEV)).clamp(max=T - 1)                        # [n, m]
    q = s["q"][0][at].float().view(n, m, Hkv, Hq // Hkv, D).permute(0, 2, 3, 1, 4).reshape(n, Hkv, -1, D)
    pos = (ctx - (cu[1:] - cu[:-1]))[:, None] + torch.arange(m, device=_DEV)                    # [n, m]
    seen = kept[:, None, :] & (key <= pos[..., None])                                           # [n, m, rows]
    score = torch.matmul(q * D ** -0.5, k.transpose(-1, -2)).view(n, Hkv, Hq // Hkv, m, rows)
    score = torch.where(seen[:, None, None], score, -math.inf)
    top = score.amax(-1, keepdim=True)
    weight = torch.exp(score - torch.where(top > -math.inf, top, 0.0))
    total = weight.sum(-1, keepdim=True)
    y = torch.matmul(weight.view(n, Hkv, -1, rows), v).view(n, Hkv, Hq // Hkv, m, D)
    y = torch.where(total > 0, y / total, 0.0).permute(0, 3, 1, 2, 4).reshape(n, m, Hq, D)
    seq, i = _places(s, T)
    s["out"].copy_(y[seq, i][None])


def run(s):
    case = s["case"]
    if own:
        _own(s)
    elif case["kind"] == "append":
        _plain_append(s)
    else:
        _plain_attend(s)
    if case["kind"] == "attend":
        return s["out"]
    if case["cache"] == "fp8":
        return {"q": s["q"], **{n: _values(s[n + "_pages"], s[n + "_scales"], _dtype(case)) for n in ("k", "v")}}
    return {"q": s["q"], "k": s["k_pages"], "v": s["v_pages"]}


def work(case):
    Hq, Hkv, D = case["Hq"], case["Hkv"], case["D"]
    lens = _lens(case)
    T = sum(q for q, _ in lens)
    width = 1 if case["cache"] == "fp8" else 2   # bytes of a cached value
    if case["kind"] == "append":
        return {"bytes": T * (2 * Hq * case["rd"] * 2 + 2 * Hkv * D * (2 + width)), "flops": T * (Hq + Hkv) * case["rd"] * 3}
    gone = [_first_page(case, past) * case["page"] for _, past in lens]
    rows = sum(q + past - g for (q, past), g in zip(lens, gone))
    pairs = sum(q * (past - g) + q * (q + 1) // 2 for (q, past), g in zip(lens, gone))
    return {"bytes": 2 * rows * Hkv * D * width + 2 * T * Hq * D * 2, "flops": 4 * D * Hq * pairs}


# ---- the definitions, in 64 bits, one sequence after the other ----------------------------------------------------------------
def _turned(x, first, case):
    """x [tokens, heads, D], token i at position first + i, as complex numbers times e^(i angle)."""
    rd, x = case["rd"], x.double()
    p = torch.arange(first, first + x.shape[0], device=_DEV, dtype=torch.float64)
    angle = torch.outer(p, torch.tensor([_BASE ** (-2.0 * j / rd) for j in range(rd // 2)], device=_DEV, dtype=torch.float64))
    part = x[..., :rd]
    pairs = part.unflatten(-1, (rd // 2, 2)) if case["style"] == 0 else part.unflatten(-1, (2, rd // 2)).transpose(-1, -2)
    z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * torch.polar(torch.ones_like(angle), angle)[:, None])
    z = z.flatten(-2) if case["style"] == 0 else z.transpose(-1, -2).flatten(-2)
    return torch.cat((z, x[..., rd:]), -1)


def _nearest_e4m3(x):
    """x (|x| <= 448) to the nearest number of three fraction bits and exponents from -6, ties to even."""
    step = torch.exp2((torch.frexp(x)[1] - 1).clamp(min=-6).double() - 3)
    return torch.round(x / step) * step


def exact(case, seed):
    s = prepare(case, seed)
    S, lens = case["page"], _lens(case)
    table = s["table"].tolist()
    pools = {}
    for name in ("k", "v"):
        pools[name] = s[name + "_pages"].double()
        if case["cache"] == "fp8":
            pools[name + "_e"] = _exponents(s[name + "_scales"]).double()
            pools[name] = pools[name] * torch.exp2(pools[name + "_e"])[:, :, None, None]
    t0, out = 0, []
    for n, (count, past) in enumerate(lens):
        q = s["q"][0, t0:t0 + count]
        if case["kind"] == "append":
            out.append(_turned(q, past, case))
            new = {"k": _turned(s["k"][0, t0:t0 + count], past, case), "v": s["v"][0, t0:t0 + count].double()}
            new["k"] = new["k"].to(_dtype(case)).double() if case["cache"] == "fp8" else new["k"]   # what a 16-bit cache would hold is what is rounded
            for p in range(past // S, (past + count - 1) // S + 1):
                lo, hi = max(past, p * S), min(past + count, (p + 1) * S)
                at, old = table[n][p], lo - p * S
                for name in ("k", "v"):
                    rows = new[name][lo - past:hi - past].transpose(0, 1)           # [Hkv, rows, D]
                    if case["cache"] == "fp8":
                        most = rows.abs().amax((1, 2))
                        e = torch.ceil(torch.log2(most / _E4M3)).clamp(-100, 119)
                        if old:
                            e = torch.maximum(e, pools[name + "_e"][at])
                        unit = torch.exp2(e)[:, None, None]
                        rows = _nearest_e4m3(rows / unit) * unit
                        pools[name][at, :, :old] = _nearest_e4m3(pools[name][at, :, :old] / unit) * unit
                        pools[name][at, :, hi - p * S:] *= (unit / torch.exp2(pools[name + "_e"][at])[:, None, None])
                    pools[name][at, :, old:hi - p * S] = rows
        else:
            ids = torch.tensor([p for p in table[n] if p >= 0], device=_DEV)
            gone = _first_page(case, past) * S
            k, v = (pools[name][ids].transpose(0, 1).flatten(1, 2)[:, :past + count - gone] for name in ("k", "v"))
            Hkv, D = case["Hkv"], case["D"]
            y = torch.empty(count, case["Hq"], D, dtype=torch.float64, device=_DEV)
            per = max(1, (1 << 27) // (case["Hq"] * k.shape[1]))
            for i0 in range(0, count, per):
                part = q[i0:i0 + per].double().unflatten(1, (Hkv, -1)).permute(1, 2, 0, 3)            # [Hkv, heads, tokens, D]
                score = torch.matmul(part.flatten(1, 2), k.transpose(1, 2).contiguous()).unflatten(1, part.shape[1:3]) / math.sqrt(D)
                position = torch.arange(past + i0, past + i0 + part.shape[2], device=_DEV)
                hidden = torch.arange(gone, past + count, device=_DEV)[None, :] > position[:, None]
                weight = torch.softmax(score.masked_fill(hidden, -math.inf), -1)
                y[i0:i0 + per] = torch.matmul(weight.flatten(1, 2), v).unflatten(1, part.shape[1:3]).permute(2, 0, 1, 3).flatten(1, 2)
            out.append(y)
        t0 += count
    whole = torch.cat(out)[None]
    return whole if case["kind"] == "attend" else {"q": whole, "k": pools["k"], "v": pools["v"]}
