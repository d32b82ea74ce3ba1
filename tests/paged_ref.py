"""A paged KV cache built from a list of sequences, and the definitions of the operators over it in float64: what the tests of
these operators compare with.  Written sequence by sequence, from dense rows; nothing here is shared with the kernels."""
import math

import torch

E4M3_MAX = 448.0


def e4m3(x):
    """float64 x (|x| <= 448) to the nearest e4m3 number, ties to even; NaN stays."""
    step = torch.exp2(torch.frexp(x)[1].sub(1).clamp(min=-6).double() - 3)
    return torch.round(x / step) * step


def needed_exponent(rows, max_e):
    """Exponent of the scale that float64 rows need: the least e in [-100, max_e] with max |finite| <= 448 * 2^e."""
    a = rows.abs()
    a = a[torch.isfinite(a)]
    top = float(a.max()) if a.numel() else 0.0
    if top == 0.0:
        return -100
    m, e = math.frexp(top)
    return min(max(e - 9 if m <= 0.875 else e - 8, -100), max_e)


class Paged:
    """Pools and a table for `seqs`, a list of (new tokens, rows held before them).

    order: how a pool lies in memory, "heads" [page, head, row, D] or "rows" [page, row, head, D] (head_dim innermost either way).
    extra: pages in the pool that belong to nobody.  gone: {(sequence, page)} whose table entry is no page.  Rows behind a
    sequence's last one hold NaN, and so do the pages that belong to nobody."""

    def __init__(self, seqs, page, Hkv, D, dtype, device, seed=0, order="heads", extra=3, gone=(), width=None, eight=False, held_only=False, gap=0):
        g = torch.Generator().manual_seed(seed)
        self.seqs, self.page, self.Hkv, self.D, self.dtype, self.device, self.eight = seqs, page, Hkv, D, dtype, device, eight
        need = [(q + past + page - 1) // page for q, past in seqs]
        self.width = max(need + [1]) if width is None else width
        self.n_pages = sum(need) + extra
        ids = torch.randperm(self.n_pages, generator=g)
        table = torch.full((len(seqs), self.width + gap), -1, dtype=torch.int32)
        self.table_list, at = [], 0
        for s, n in enumerate(need):
            row = ids[at:at + n].tolist()
            at += n
            row = [-1 if (s, i) in gone else p for i, p in enumerate(row)]
            self.table_list.append(row)
            table[s, :len(row)] = torch.tensor(row, dtype=torch.int32)
        self.table = table.to(device)[:, :self.width] if gap else table.to(device)
        self.k_scales = self.v_scales = None
        self.dense = []    # float64 rows [Hkv, rows, D] of every sequence, k and v, as the cache holds them
        rows = [(past if held_only else q + past) for q, past in seqs]
        pools = []
        for what in range(2):
            pool = torch.full((self.n_pages, Hkv, page, D), float("nan"), dtype=torch.float64)
            exps = torch.full((self.n_pages, Hkv), -3, dtype=torch.int64)
            for s, n in enumerate(rows):
                x = torch.randn(Hkv, n, D, generator=g, dtype=torch.float64)
                if what == 0:
                    x[:, :, 0] *= 6.0
                x = x.to(dtype).double()
                if eight:
                    for i in range(0, n, page):
                        p = self.table_list[s][i // page]
                        for h in range(Hkv):
                            e = needed_exponent(x[h, i:i + page], 7)
                            x[h, i:i + page] = e4m3((x[h, i:i + page] / 2.0 ** e).clamp(-E4M3_MAX, E4M3_MAX)) * 2.0 ** e
                            if p >= 0:
                                exps[p, h] = e
                for i in range(n):
                    p = self.table_list[s][i // page]
                    if p >= 0:
                        pool[p, :, i % page] = x[:, i]
                self.dense.append(x)
            if eight:
                codes = (pool / torch.exp2(exps.double())[:, :, None, None]).to(torch.float8_e4m3fn)
                pools.append(self._laid_out(codes, order, device))
                scales = (exps + 127).to(torch.uint8).view(torch.float8_e8m0fnu).to(device)
                if what == 0:
                    self.k_scales = scales
                else:
                    self.v_scales = scales
            else:
                pools.append(self._laid_out(pool.to(dtype), order, device))
        self.k_pages, self.v_pages = pools
        self.k_dense, self.v_dense = self.dense[:len(seqs)], self.dense[len(seqs):]
        lens = [q for q, _ in seqs]
        self.T = sum(lens)
        self.cu_list = [sum(lens[:i]) for i in range(len(lens) + 1)]
        self.cu = torch.tensor(self.cu_list, dtype=torch.int32, device=device)
        self.past = torch.tensor([p for _, p in seqs], dtype=torch.int32, device=device)
        self.ctx = torch.tensor([q + p for q, p in seqs], dtype=torch.int32, device=device)

    @staticmethod
    def _laid_out(pool, order, device):
        if order == "rows":
            return pool.view(torch.uint8 if pool.element_size() == 1 else torch.int16).transpose(1, 2).contiguous().view(pool.dtype).to(device).transpose(1, 2)
        return pool.to(device)

    def scales(self):
        return (self.k_scales, self.v_scales) if self.eight else ()

    def row_there(self, s):
        """Which rows 0 .. of sequence s lie in pages that are there."""
        n = sum(self.seqs[s])
        return torch.tensor([self.table_list[s][i // self.page] >= 0 for i in range(n)], dtype=torch.bool)


def attend(cache, q, scale=None):
    """out [Hq, T, D] in float64 over `cache` for q [Hq, T, D], and the bound of a 16-bit kernel's error for each element.

    The bound: a weight is off by the rounding of the scaled query (half a step of each of its D values: ds = eps / 2 * sum
    |q k| / sqrt(D) in the exponent, the largest over the row's keys) and of the weight itself (eps / 2).  With weights
    off by at most R relatively, numerator and denominator together move the output by at most 2 R / (1 - R) * sum(w |v|); the
    output is rounded once more.  fp32 sums and the exponential's error stand far below (1e-5 of sum(w |v|))."""
    Hq, T, D = q.shape
    eps = torch.finfo(q.dtype).eps
    q = q.double().cpu()
    out = torch.zeros(Hq, T, D, dtype=torch.float64)
    bound = torch.zeros(Hq, T, D, dtype=torch.float64)
    n_rep = Hq // cache.Hkv
    for s, (n, past) in enumerate(cache.seqs):
        if n == 0:
            continue
        there = cache.row_there(s)
        lo = cache.cu_list[s]
        for h in range(Hq):
            k, v = cache.k_dense[s][h // n_rep], cache.v_dense[s][h // n_rep]
            x = q[h, lo:lo + n]
            score = x @ k.T / math.sqrt(D)
            seen = (torch.arange(n + past)[None, :] <= (past + torch.arange(n))[:, None]) & there[None, :]
            score = torch.where(seen, score, -math.inf)
            top = score.amax(1, keepdim=True)
            w = torch.exp(score - torch.where(top > -math.inf, top, 0.0))
            total = w.sum(1, keepdim=True)
            w = torch.where(total > 0, w / total, 0.0)
            out[h, lo:lo + n] = w @ v
            size = (x.abs() @ k.abs().T) / math.sqrt(D)
            ds = eps / 2 * torch.where(seen, size, 0.0).amax(1, keepdim=True)
            R = eps / 2 + torch.expm1(ds)
            bound[h, lo:lo + n] = (2 * R / (1 - R) + 1e-5) * (w @ v.abs())
    return out, bound * (1 + eps) + eps / 2 * out.abs() + 1e-12


def rotated(x, first, style, rd, base):
    """x [tokens, heads, D] in float64, token i at position first + i."""
    n, half = x.shape[0], rd // 2
    angle = (first + torch.arange(n, dtype=torch.float64))[:, None] * base ** (-2.0 * torch.arange(half, dtype=torch.float64) / rd)
    c, s = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
    y = x.clone()
    a, b = (slice(0, rd, 2), slice(1, rd, 2)) if style == 0 else (slice(0, half), slice(half, rd))
    y[..., a] = c * x[..., a] - s * x[..., b]
    y[..., b] = s * x[..., a] + c * x[..., b]
    return y
