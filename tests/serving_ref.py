"""Definitions of the operators of a serving step around the paged cache, on the host, one sequence after the other, in whole numbers and
float64: what their tests compare with."""
import torch


def tables(page, past, new, held, ring, state, table, n_slots):
    """(cu_seqlens, ctx_lens, slots, table, held_after, state_after) as lists; slots and table with None where nothing is written."""
    N, width = len(ring), len(table[0]) if table else 0
    head, count = (state[0] % N if N and state[0] >= 0 else 0), min(max(state[1], 0), N)
    table = [list(row) for row in table]
    cu, ctx, slots, held_after, at, lacking = [0], [], [None] * n_slots, [], 0, 0
    for row, p, w, h in zip(table, past, new, held):
        p, w, h = max(p, 0), max(w, 0), min(max(h, 0), width)
        own = h
        for i in range(h, min(-(-(p + w) // page), width)):
            if at < count:
                row[i] = ring[(head + at) % N]
                at, own = at + 1, own + 1
            else:
                row[i] = -1
                lacking += 1
        end = max(h, min(-(-(p + w) // page), width))
        held_after.append(own)
        for i in range(w):
            if cu[-1] + i < n_slots:
                r = p + i
                name = row[r // page] if r // page < end else -1
                slots[cu[-1] + i] = name * page + r % page if 0 <= name < N else -1
        cu.append(cu[-1] + w)
        ctx.append(p + w)
    return cu, ctx, slots, table, held_after, [(head + at) % N if N else 0, count - at, lacking]


def release(page, keep, held, table, ring, state):
    """(ring, held_after, state_after)."""
    ring, N = list(ring), len(ring)
    width = len(table[0]) if table else 0
    head, count = (state[0] % N if N and state[0] >= 0 else 0), min(max(state[1], 0), N)
    held_after, dropped = [], 0
    for row, k, h in zip(table, keep, held):
        h = min(max(h, 0), width)
        stay = min(-(-max(k, 0) // page), h)
        for name in row[stay:h]:
            if 0 <= name < N:
                if count < N:
                    ring[(head + count) % N] = name
                    count += 1
                else:
                    dropped += 1
        held_after.append(stay)
    return ring, held_after, [head, count, dropped]


def verify(tokens, cu, target, draft, accept_u, sample_u):
    """(out_tokens with None where nothing is written, n_accepted).  Tensors on the host; probabilities of any float type."""
    T, V = target.shape
    out, accepted = [None] * T, []
    for s, (lo, hi) in enumerate(zip(cu, cu[1:])):
        lo = min(max(lo, 0), T)
        hi = min(max(hi, lo), T)
        if lo == hi:
            accepted.append(0)
            continue
        a = 0
        while lo + a < hi - 1:
            x = int(tokens[lo + a + 1])
            if not 0 <= x < V:
                break
            q = float(draft[lo + a, x]) if draft is not None else 1.0
            if not float(accept_u[lo + a]) * q < float(target[lo + a, x]):
                break
            a += 1
        p = torch.nan_to_num(target[lo + a].double(), nan=0.0).clamp(min=0)
        w = p
        if lo + a < hi - 1:
            x = int(tokens[lo + a + 1])
            q = draft[lo + a].double() if draft is not None else (torch.arange(V) == x).double()
            left = torch.nan_to_num(target[lo + a].double() - q, nan=0.0).clamp(min=0)
            w = left if float(left.sum()) > 0 else p
        sums = torch.cumsum(w, 0)
        over = (sums > float(sample_u[s]) * sums[-1]) & (w > 0)
        some = w > 0
        chosen = int(over.int().argmax()) if over.any() else int(some.nonzero()[-1]) if some.any() else -1
        for i in range(lo, hi):
            out[i] = int(tokens[i + 1]) if i - lo < a else chosen if i - lo == a else -1
        accepted.append(a)
    return out, accepted
