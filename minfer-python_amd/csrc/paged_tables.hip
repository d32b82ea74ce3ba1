// Block tables, slot maps and the pool's free pages of a paged KV cache from the lengths of its sequences, on the device: what a serving loop does
// between two steps, without a copy to the host.
//
// The free pages are a ring: the first `count` entries from `head` on, around its end.  Pages are taken from the front and given back behind
// the last, so what a launch reads and what it writes never meet, and a page that was given back is the last to be handed out again.
//
// Which page goes where follows from sums over the sequences in front (pages that they take or give back), so the result does not depend on the
// order in which anything runs.  Every workgroup makes the sum that it needs itself, from lengths that lie in the L2: one launch, no workspace, no
// waiting for one another.  Only pages that are given back have to be looked at (a window that moved on may have left no page), so paged_release
// counts in one launch and moves in a second.
//
// Bound by latency: a launch and, for tables, two or three loads that depend on one another; for pages given back up to eight loads a sequence one after the other, twice.
#include <algorithm>

#include "attn_common.h"
#include "attn_host.h"

namespace minfer_attn {

constexpr int kTableThreads = 256;
constexpr int kMaxLen = 1 << 30;   // rows and pages of a sequence; what is given beyond is cut, so that sums of two fit 32 bits

struct Ring { int head, count; };
struct TableParams {
    const int32_t* past; const int32_t* fresh; const int32_t* held;   // rows held, new tokens, pages held
    int32_t* ring; const int32_t* state;
    int32_t* table;
    int32_t* cu; int32_t* ctx; int64_t* slots;
    int32_t* held_after; int32_t* state_after;
    int32_t* counts;     // release: pages that every sequence gives back
    int64_t table_stride, n_slots;
    int n_seqs, width, page_log2, n_pages;
    int per_wg;          // consecutive sequences of a workgroup
};

MA_DEV int cut(int x, int most) { return min(max(x, 0), most); }
// The ring's state, whatever the memory holds: indexes made from it stay inside.
MA_DEV Ring ring_of(const TableParams& p) {
    int head = p.state[0];
    if ((unsigned)head >= (unsigned)p.n_pages) head = p.n_pages > 0 && head >= 0 ? head % p.n_pages : 0;
    return Ring{head, cut(p.state[1], p.n_pages)};
}
// Entry i from the head on, i at most n_pages.
MA_DEV int ring_at(const TableParams& p, const Ring& r, int64_t i) {
    const uint32_t at = (uint32_t)r.head + (uint32_t)i;
    return (int)(at >= (uint32_t)p.n_pages ? at - (uint32_t)p.n_pages : at);
}
MA_DEV int saturated(int64_t x) { return (int)min(x, (int64_t)0x7fffffff); }

// x of another lane, as row_exchange; the sum over a wave is lane 63's of a prefix sum.
template <int CTRL, int ROW_MASK = 0xf> MA_DEV int64_t row_exchange64(int64_t x) {
    const uint32_t lo = row_exchange<CTRL, ROW_MASK>((uint32_t)x), hi = row_exchange<CTRL, ROW_MASK>((uint32_t)(x >> 32));
    return (int64_t)((uint64_t)hi << 32 | lo);
}
MA_DEV int64_t wave_scan(int64_t x) {
    x += row_exchange64<0x111>(x);
    x += row_exchange64<0x112>(x);
    x += row_exchange64<0x114>(x);
    x += row_exchange64<0x118>(x);
    x += row_exchange64<0x142, 0xa>(x);
    x += row_exchange64<0x143, 0xc>(x);
    return x;
}
MA_DEV int64_t lane_value(int64_t x, int lane) {
    return (int64_t)((uint64_t)(uint32_t)lane_value((int)(x >> 32), lane) << 32 | (uint32_t)lane_value((int)x, lane));
}
MA_DEV int64_t wave_sum(int64_t x) { return lane_value(wave_scan(x), 63); }
// x summed over the workgroup, in every thread; `part` is the caller's, one entry a wave.
MA_DEV int64_t block_sum(int64_t x, int64_t* part) {
    x = wave_sum(x);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = x;
    __syncthreads();
    int64_t all = 0;
#pragma unroll
    for (int i = 0; i < kTableThreads / 64; ++i) all += part[i];
    return all;
}

// ---- new pages and slots -------------------------------------------------------------------------------------------
struct Grown { int past, fresh, held, need; };   // need: pages of the rows with the new ones, or those that it holds if they are more
MA_DEV Grown grown(const TableParams& p, int s) {
    Grown r{cut(p.past[s], kMaxLen), cut(p.fresh[s], kMaxLen), cut(p.held[s], p.width), 0};
    const int64_t rows = (int64_t)r.past + r.fresh + (1 << p.page_log2) - 1;
    r.need = max((int)min(rows >> p.page_log2, (int64_t)p.width), r.held);
    return r;
}

// grid (workgroups of per_wg sequences, parts of their tokens).  256 sequences of a token each 3.3 us, 23 prompts of 300 to 4095 3.4; a call 6.0, which is what issuing it takes.
__global__ __launch_bounds__(kTableThreads) void paged_tables_kernel(const TableParams p) {
    __shared__ int64_t parts[2][kTableThreads / 64];
    const int tid = threadIdx.x, s0 = (int)blockIdx.x * p.per_wg, s1 = min(s0 + p.per_wg, p.n_seqs);
    const bool writes = blockIdx.y == 0;   // the part that leaves what a sequence has once
    const Ring ring = ring_of(p);
    int64_t tokens = 0, taken = 0;   // of the sequences in front
    for (int s = tid; s < s0; s += kTableThreads) {
        const Grown q = grown(p, s);
        tokens += q.fresh;
        taken += q.need - q.held;
    }
    tokens = block_sum(tokens, parts[0]);
    taken = block_sum(taken, parts[1]);
    const int step = kTableThreads * (int)gridDim.y, i0 = (int)blockIdx.y * kTableThreads + tid;
    auto page_of = [&](int64_t number) { return number < ring.count ? p.ring[ring_at(p, ring, number)] : -1; };
    for (int s = s0; s < s1; ++s) {
        const Grown q = grown(p, s);
        int32_t* const row = p.table + (int64_t)s * p.table_stride;
        for (int i = i0; i < q.need - q.held; i += step) row[q.held + i] = page_of(taken + i);
        const int here = (int)max(min((int64_t)q.fresh, p.n_slots - tokens), (int64_t)0);   // (tokens behind the last slot have none)
        for (int i = i0; i < here; i += step) {
            const int at = q.past + i, page_no = at >> p.page_log2;
            int page = -1;
            if (page_no < q.held) page = row[page_no];
            else if (page_no < q.need) page = page_of(taken + page_no - q.held);
            p.slots[tokens + i] = (unsigned)page < (unsigned)p.n_pages ? ((int64_t)page << p.page_log2) + (at & ((1 << p.page_log2) - 1)) : -1;
        }
        if (writes && tid == 0) {
            p.cu[s] = saturated(tokens);
            p.ctx[s] = saturated((int64_t)q.past + q.fresh);
            p.held_after[s] = q.held + (int)min(max((int64_t)ring.count - taken, (int64_t)0), (int64_t)(q.need - q.held));
        }
        tokens += q.fresh;
        taken += q.need - q.held;
    }
    if (writes && tid == 0 && s1 >= p.n_seqs) {   // the last workgroup (the only one of no sequences)
        const int given = (int)min(taken, (int64_t)ring.count);
        p.cu[p.n_seqs] = saturated(tokens);
        p.state_after[0] = p.n_pages > 0 ? ring_at(p, ring, given) : 0;
        p.state_after[1] = ring.count - given;
        p.state_after[2] = saturated(taken - given);
    }
}

// ---- pages that are given back -------------------------------------------------------------------------------------
struct Shrunk { int stay, held; };
MA_DEV Shrunk shrunk(const TableParams& p, int s) {
    const int held = cut(p.held[s], p.width), keep = cut(p.past[s], kMaxLen);
    return Shrunk{min((keep + (1 << p.page_log2) - 1) >> p.page_log2, held), held};
}

// f(entries, lane's is a page, the pages in front of it), 64 entries of a sequence's surplus at a time, eight times 64 a round; the number of pages.  The whole wave.  (Each of a round's loads
// stands behind the condition that its entry is the sequence's, and the built code waits for it in front of the next one.)
template <class F> MA_DEV int each_page(const TableParams& p, int s, int stay, int held, F f) {
    const int lane = threadIdx.x & 63;
    const int32_t* const row = p.table + (int64_t)s * p.table_stride;
    constexpr int UN = 8;
    int n = 0;
    for (int base = stay; base < held; base += 64 * UN) {
        int page[UN];
#pragma unroll
        for (int u = 0; u < UN; ++u) page[u] = base + 64 * u + lane < held ? row[base + 64 * u + lane] : -1;
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            const bool on = (unsigned)page[u] < (unsigned)p.n_pages;
            const uint64_t all = __ballot(on);
            f(page[u], on, n + __popcll(all & (((uint64_t)1 << lane) - 1)));
            n += __popcll(all);
        }
    }
    return n;
}
// A sequence's pages to the ring, behind `front` pages of the sequences in front of it.
MA_DEV int give_back(const TableParams& p, const Ring& ring, int s, const Shrunk& q, int64_t front) {
    const int64_t room = p.n_pages - ring.count;   // (more pages than the ring has room for are there only if some were named twice)
    return each_page(p, s, q.stay, q.held, [&](int page, bool on, int before) __attribute__((always_inline)) {
        if (on && front + before < room) p.ring[ring_at(p, ring, ring.count + front + before)] = page;
    });
}
MA_DEV void leave_state(const TableParams& p, const Ring& ring, int64_t given) {
    const int took = (int)min(given, (int64_t)(p.n_pages - ring.count));
    p.state_after[0] = ring.head;
    p.state_after[1] = ring.count + took;
    p.state_after[2] = saturated(given - took);
}

// Up to 64 sequences: one workgroup counts and moves, a wave every sixteenth sequence.  64 sequences, a tenth of them ended, 5.4 us where two launches take 9.1.
constexpr int kFewSeqs = 64, kFewWaves = 16;
__global__ __launch_bounds__(kFewWaves * 64) void paged_release_few_kernel(const TableParams p) {
    __shared__ int counts[kFewSeqs];
    const int lane = threadIdx.x & 63, w = wave_id();
    const Ring ring = ring_of(p);
    const Shrunk mine = lane < p.n_seqs ? shrunk(p, lane) : Shrunk{0, 0};   // a sequence to a lane
    for (int s = w; s < p.n_seqs; s += kFewWaves) {
        const int n = each_page(p, s, lane_value(mine.stay, s), lane_value(mine.held, s), [](int, bool, int) {});
        if (lane == 0) { counts[s] = n; p.held_after[s] = lane_value(mine.stay, s); }
    }
    __syncthreads();
    const int n = lane < p.n_seqs ? counts[lane] : 0;
    const int64_t incl = wave_scan((int64_t)n);   // (64 times 2^26 pages, which a table may name, are 2^32)
    for (int s = w; s < p.n_seqs; s += kFewWaves) {
        const Shrunk q{lane_value(mine.stay, s), lane_value(mine.held, s)};
        if (lane_value(n, s) > 0) give_back(p, ring, s, q, lane_value(incl - n, s));
    }
    if (threadIdx.x == 0) leave_state(p, ring, lane_value(incl, 63));
}

// More of them.  A wave per sequence: its entries that name a page.
__global__ __launch_bounds__(kTableThreads) void paged_release_count_kernel(const TableParams p) {
    const int s = (int)blockIdx.x * (kTableThreads / 64) + wave_id(), lane = threadIdx.x & 63;
    if (s >= p.n_seqs) return;
    const Shrunk q = shrunk(p, s);
    const int n = each_page(p, s, q.stay, q.held, [](int, bool, int) {});
    if (lane == 0) { p.counts[s] = n; p.held_after[s] = q.stay; }
}

// A wave per sequence again: its pages behind those of the sequences in front.  Up to kReleaseWgs workgroups of per_wg consecutive sequences, four at a time: every workgroup sums all counts in front of
// its first sequence, so that more of them would cost sequences times sequences (2^18 that end 2.0 ms with a workgroup for every four of them, 0.36 so; 2^24 27 ms).
constexpr int64_t kReleaseWgs = 1024;
__global__ __launch_bounds__(kTableThreads) void paged_release_kernel(const TableParams p) {
    __shared__ int64_t parts[kTableThreads / 64];
    constexpr int NW = kTableThreads / 64;
    const int tid = threadIdx.x, lane = tid & 63, w = wave_id();
    const int first = (int)blockIdx.x * p.per_wg, last = min(first + p.per_wg, p.n_seqs);
    const Ring ring = ring_of(p);
    int64_t front = 0;
    for (int i = tid; i < first; i += kTableThreads) front += p.counts[i];
    front = block_sum(front, parts);
    for (int s0 = first; s0 < last; s0 += NW) {
        int count[NW];   // of the four
#pragma unroll
        for (int i = 0; i < NW; ++i) count[i] = s0 + i < last ? p.counts[s0 + i] : 0;
        int64_t mine = front;
#pragma unroll
        for (int i = 0; i < NW; ++i) {
            mine += i < w ? count[i] : 0;
            front += count[i];
        }
        const int s = s0 + w;
        if (s >= last) continue;
        give_back(p, ring, s, shrunk(p, s), mine);
        if (lane == 0 && s == p.n_seqs - 1) leave_state(p, ring, front);
    }
}

static bool overlap(const void* a, int64_t na, const void* b, int64_t nb) {
    const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
    return na > 0 && nb > 0 && x < y + (uintptr_t)nb && y < x + (uintptr_t)na;
}

// Checks that both operators share.
static int check_tables(const char* op, const minfer_page_ring* ring, int64_t page_size, int64_t n_seqs, int64_t pages_per_seq, int64_t table_stride, TableParams& p) {
    char msg[256];
    auto bad = [&](const char* what) { snprintf(msg, sizeof msg, "%s: %s", op, what); return fail(MINFER_ATTN_EINVAL, msg); };
    if (page_size < 16 || page_size > 1024 || (page_size & (page_size - 1)) != 0) return bad("page_size must be a power of two in 16..1024");
    if (n_seqs < 0 || n_seqs > (1 << 24)) return bad("n_seqs must be in 0..2^24");
    if (pages_per_seq < 0 || pages_per_seq > ((int64_t)1 << 30) / page_size) return bad("pages_per_seq * page_size must be in 0..2^30");
    if (table_stride < 0 || (n_seqs > 1 && table_stride < pages_per_seq)) return bad("table_stride must not be smaller than pages_per_seq");
    if (!ring) return bad("ring is null");
    if (ring->n_pages < 0 || ring->n_pages > 0x7fffffffLL) return bad("bad number of pages");
    if (!ring->state || !ring->state_after || (ring->n_pages > 0 && !ring->pages)) return bad("the ring's pages, state and state_after must be non-null");
    if (overlap(ring->state, 12, ring->state_after, 12)) return bad("state_after must not be state: workgroups read the one while others write the other");
    p.ring = ring->pages; p.state = ring->state; p.state_after = ring->state_after;
    p.n_pages = (int)ring->n_pages;
    p.table_stride = table_stride;
    p.n_seqs = (int)n_seqs; p.width = (int)pages_per_seq;
    p.page_log2 = __builtin_ctzll((unsigned long long)page_size);
    return MINFER_ATTN_OK;
}

}  // namespace minfer_attn

using namespace minfer_attn;

MINFER_ATTN_EXPORT int minfer_paged_tables(int64_t page_size, const int32_t* past_lens, const int32_t* new_lens, const int32_t* pages_held,
                                           const minfer_page_ring* ring, int32_t* block_table, int64_t table_stride, int64_t pages_per_seq,
                                           int32_t* cu_seqlens, int32_t* ctx_lens, int64_t* slots, int64_t n_slots, int32_t* held_after,
                                           int64_t n_seqs, void* stream) {
    clear_error();
    TableParams p{};
    if (int rc = check_tables("paged_tables", ring, page_size, n_seqs, pages_per_seq, table_stride, p)) return rc;
    auto bad = [&](const char* what) { return fail(MINFER_ATTN_EINVAL, what); };
    if (n_slots < 0 || n_slots > 0x7fffffffLL) return bad("paged_tables: n_slots must be in 0..2^31-1");
    if (!cu_seqlens || (n_slots > 0 && !slots)) return bad("paged_tables: cu_seqlens and slots must be non-null");
    if (n_seqs > 0 && (!past_lens || !new_lens || !pages_held || !ctx_lens || !held_after || (pages_per_seq > 0 && !block_table)))
        return bad("paged_tables: past_lens, new_lens, pages_held, block_table, ctx_lens and held_after must be non-null");
    const int32_t* const in[3] = {past_lens, new_lens, pages_held};
    int32_t* const out[3] = {cu_seqlens, ctx_lens, held_after};
    for (const int32_t* i : in)
        for (int32_t* o : out)
            if (overlap(i, 4 * n_seqs, o, 4 * (o == cu_seqlens ? n_seqs + 1 : n_seqs))) return bad("paged_tables: outputs must not be inputs: workgroups read the ones while others write the others");
    p.past = past_lens; p.fresh = new_lens; p.held = pages_held;
    p.table = block_table;
    p.cu = cu_seqlens; p.ctx = ctx_lens; p.slots = slots; p.held_after = held_after;
    p.n_slots = n_slots;
    // up to 1024 workgroups with a sequence each; long sequences' tokens to several workgroups, 256 at a time
    p.per_wg = (int)std::max<int64_t>((n_seqs + 1023) / 1024, 1);
    const int64_t wgs = std::max<int64_t>((n_seqs + p.per_wg - 1) / p.per_wg, 1);
    const int64_t parts = std::max<int64_t>(std::min<int64_t>((n_slots / wgs + kTableThreads - 1) / kTableThreads, 1024 / wgs), 1);
    hipLaunchKernelGGL(paged_tables_kernel, dim3((unsigned)wgs, (unsigned)parts), dim3(kTableThreads), 0, (hipStream_t)stream, p);
    return check_launch("paged_tables_kernel");
}

MINFER_ATTN_EXPORT size_t minfer_paged_release_workspace_bytes(int64_t n_seqs) { return n_seqs > kFewSeqs ? ((size_t)n_seqs * 4 + 255) / 256 * 256 : 0; }

MINFER_ATTN_EXPORT int minfer_paged_release(int64_t page_size, const int32_t* keep_lens, const int32_t* pages_held, const minfer_page_ring* ring,
                                            const int32_t* block_table, int64_t table_stride, int64_t pages_per_seq, int32_t* held_after, int64_t n_seqs,
                                            void* workspace, size_t workspace_bytes, void* stream_v) {
    clear_error();
    TableParams p{};
    if (int rc = check_tables("paged_release", ring, page_size, n_seqs, pages_per_seq, table_stride, p)) return rc;
    auto bad = [&](const char* what) { return fail(MINFER_ATTN_EINVAL, what); };
    if (n_seqs > 0 && (!keep_lens || !pages_held || !held_after || (pages_per_seq > 0 && !block_table)))
        return bad("paged_release: keep_lens, pages_held, block_table and held_after must be non-null");
    if (overlap(keep_lens, 4 * n_seqs, held_after, 4 * n_seqs) || overlap(pages_held, 4 * n_seqs, held_after, 4 * n_seqs))
        return bad("paged_release: outputs must not be inputs: the second launch reads them again");
    if (n_seqs > kFewSeqs && (!workspace || ((uintptr_t)workspace & 3) || workspace_bytes < minfer_paged_release_workspace_bytes(n_seqs)))
        return fail(MINFER_ATTN_EWORKSPACE, "paged_release: workspace too small or misaligned (see minfer_paged_release_workspace_bytes)");
    p.past = keep_lens; p.held = pages_held;
    p.table = const_cast<int32_t*>(block_table);
    p.held_after = held_after;
    p.counts = (int32_t*)workspace;
    hipStream_t stream = (hipStream_t)stream_v;
    if (n_seqs <= kFewSeqs) {
        hipLaunchKernelGGL(paged_release_few_kernel, dim3(1), dim3(kFewWaves * 64), 0, stream, p);
        return check_launch("paged_release_few_kernel");
    }
    constexpr int64_t NW = kTableThreads / 64;
    const int64_t wgs = (n_seqs + NW - 1) / NW;
    p.per_wg = (int)((wgs + kReleaseWgs - 1) / kReleaseWgs * NW);
    hipLaunchKernelGGL(paged_release_count_kernel, dim3((unsigned)wgs), dim3(kTableThreads), 0, stream, p);
    if (int rc = check_launch("paged_release_count_kernel")) return rc;
    hipLaunchKernelGGL(paged_release_kernel, dim3((unsigned)((n_seqs + p.per_wg - 1) / p.per_wg)), dim3(kTableThreads), 0, stream, p);
    return check_launch("paged_release_kernel");
}
