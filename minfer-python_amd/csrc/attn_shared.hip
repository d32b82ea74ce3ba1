// Attention of few query rows per sequence over a paged cache where groups of sequences share their first pages, for gfx950: a batch behind one instruction or
// document, whose pages every table names.  The prefix's rows are read once for all of a group's tokens instead of once for each sequence.
//
// out = softmax over [prefix, own rows] is made of two softmaxes with references and sums of their own:
// * the prefix: the tokens of a group times the query heads of a KV head are a list of rows, 128 of which walk the prefix's 64-key tiles together (attend_tiles),
//   cut into pieces that fill the chip: matrix work, a group's K and V read once for every 128 rows and from the L2 where several blocks of rows meet;
// * the own rows: streamed by single waves over a line of equal shares (stream_pages): bound by memory.
// Both are one launch, which the workgroups divide between them by what each part is estimated to take, so that matrix units and memory work side by side
// and both end together.  Everything is a partial result, and shared_merge_kernel puts a row's together.
//
// How the work is cut follows from device data (lengths, contexts, groups) that every wave looks up for itself, a sequence or a group to a lane.
#include <algorithm>

#include "attn_paged_stream.h"
#include "attn_paged_tile.h"

namespace minfer_attn {

typedef int i32x4 __attribute__((ext_vector_type(4)));

constexpr int kSharedWaves = 4, kBlockRows = kSharedWaves * 32;
constexpr int kSharedUnits = 256, kSharedWgs = 2 * kSharedUnits;   // workgroups of the launch: what the chip holds at once
constexpr int kMaxSharedHeads = 128;                               // KV heads: each has workgroups of its own for the prefix

struct SharedWork {
    DecodeWork d;                    // of the own rows; part_o / part_ml of d.p are theirs
    const int32_t* cu_groups; const int32_t* prefix;
    int n_groups;
    float* tile_o; float* tile_ml;   // partial results of the prefixes: [piece][KV head][128][D] and their references and sums
    int max_pieces;                  // that there is room for
    int32_t* seq_tab;                // [n_seqs][2]: a sequence's place on the line, its group (-1: none); then the quota
    i32x4* group_tab;                 // [n_groups]: first token, (token, head) rows, first piece, pieces of a block of rows
};

// Rows of group i's prefix that are computed for all its tokens together: whole tiles.
MA_DEV int shared_rows(const SharedWork& w, int i) { return min(max(w.prefix[i], 0), w.d.p.c.width << w.d.p.c.page_log2) & ~63; }

// The group of sequence s (-1: none): cu_groups is a list of increasing starts.
MA_DEV int group_of(const SharedWork& w, int s) {
    int lo = 0, hi = w.n_groups;   // the last entry that is <= s, of n_groups + 1
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (w.cu_groups[mid] <= s) lo = mid; else hi = mid - 1;
    }
    return lo < w.n_groups && w.cu_groups[lo] <= s ? lo : -1;
}

struct OwnSeq { SeqInfo info; int group, g0, groups; };   // g0: the first group of rows behind the prefix; groups: how many there are
template <int GR> MA_DEV OwnSeq own_seq(const SharedWork& w, int s) {   // (per lane)
    OwnSeq r{{0, 0, 0}, -1, 0, 0};
    if (s < w.d.p.n_seqs) {
        const LineSeq q = line_seq<GR>(w.d, s);
        r.info = q.info;
        r.group = group_of(w, s);
        r.g0 = r.group >= 0 ? shared_rows(w, r.group) / GR : 0;
        r.groups = max(q.groups - r.g0, 0);
    }
    return r;
}

struct Group { int first, last, lo, rows, tiles; };   // sequences, first token, (token, head) rows, tiles of the prefix
// The whole wave, a group to a lane.
MA_DEV Group group_at(const SharedWork& w, int i) {
    const PagedParams& p = w.d.p;
    Group r{0, 0, 0, 0, 0};
    int hi = 0;
    if (i < w.n_groups) {
        r.first = min(max(w.cu_groups[i], 0), p.n_seqs);
        r.last = min(max(w.cu_groups[i + 1], r.first), p.n_seqs);
        r.tiles = shared_rows(w, i) >> 6;
        r.lo = min(max(p.cu[r.first], 0), p.T);
        hi = min(max(p.cu[r.last], 0), p.T);
    }
    // (a group with sequences and no tokens, or one whose last sequences have none and entries of zero: looked at one by one)
    uint64_t odd = __ballot(r.last > r.first && r.tiles > 0 && hi <= r.lo);
    while (odd) {
        const int lane = threadIdx.x & 63, at = __ffsll((unsigned long long)odd) - 1, last = lane_value(r.last, at);
        int top = 0, low = p.T;
        for (int s = lane_value(r.first, at); s < last; ++s) {
            const TokenRange t = token_range(const_load(p.cu + s), const_load(p.cu + s + 1), p.T);
            if (t.len > 0) { top = max(top, t.lo + t.len); low = min(low, t.lo); }
        }
        if (lane == at) { r.lo = min(low, top); hi = top; }
        odd &= odd - 1;
    }
    r.rows = r.last > r.first ? max(hi - r.lo, 0) * p.n_rep : 0;
    return r;
}

// How the launch is laid out, worked out by every wave.
struct SharedPlan {
    int n_tile;         // workgroups for the prefixes, the launch's first ones
    int size;           // tiles of a piece
    int pieces;         // per KV head
    int total, quota;   // of the line
    OwnSeq kept;        // per lane: the first 64 sequences
    Group group;        // per lane: the first 64 groups
};
MA_DEV int blocks_of(const Group& g) { return g.tiles > 0 ? (g.rows + kBlockRows - 1) / kBlockRows : 0; }
MA_DEV int parts_of(const Group& g, int size) { return (g.tiles + size - 1) / size; }

template <int D, int GR> MA_DEV SharedPlan plan_shared(const SharedWork& w, bool writes) {
    const PagedParams& p = w.d.p;
    const int lane = threadIdx.x & 63, pairs = p.Hkv * w.d.n_hg;
    SharedPlan r;
    // ---- the groups: blocks of rows and tiles ----
    int blocks = 0;
    float units = 0.f;   // tiles of all blocks
    for (int base = 0; base < w.n_groups; base += 64) {
        const Group q = group_at(w, base + lane);
        if (base == 0) r.group = q;
        blocks += lane_value(wave_inclusive_scan(blocks_of(q)), 63);
        units += lane_sum<64>((float)blocks_of(q) * (float)q.tiles);
    }
    // ---- the line ----
    int total = 0, longest = 0;
    for (int base = 0; base < p.n_seqs; base += 64) {
        const OwnSeq q = own_seq<GR>(w, base + lane);
        if (base == 0) r.kept = q;
        const int incl = wave_inclusive_scan(q.groups * pairs);
        if (writes && base + lane < p.n_seqs) {
            w.seq_tab[2 * (base + lane)] = total + incl - q.groups * pairs;
            w.seq_tab[2 * (base + lane) + 1] = q.group;
        }
        total += lane_value(incl, 63);
        longest = max(longest, q.groups);
    }
    longest = __builtin_amdgcn_readfirstlane((int)wave_max((float)longest));
    r.total = total;
    // ---- who does what: a tile of a block takes a workgroup about twice as long as 64 rows of the line (16-bit rows; four groups of them) ----
    constexpr float kTileCost = 2.f;
    const float tile_work = units * (float)p.Hkv * kTileCost, line_work = (float)total / (float)(64 / GR) ;
    const int G = (int)gridDim.x;
    int ranks = 0;
    if (__any(tile_work > 0.f)) {
        const int least_line = total > 0 ? G / 8 : 0;
        ranks = (int)((float)G * tile_work / (tile_work + line_work) / (float)p.Hkv + 0.5f);
        ranks = __builtin_amdgcn_readfirstlane(min(max(ranks, 1), (G - least_line) / p.Hkv));
    }
    r.n_tile = ranks * p.Hkv;
    // ---- pieces: equal to within a tile, no more of them than workgroups where blocks may be cut; more than 64 groups are not cut ----
    r.size = 0x3fffffff;
    r.pieces = blocks;
    if (ranks > 0 && w.n_groups <= 64) {
        constexpr int kLeastTiles = 2;
        const int most = max(ranks, blocks), tiles = (int)wave_max((float)r.group.tiles);
        int size = __builtin_amdgcn_readfirstlane(max(max((int)(units / (float)most), kLeastTiles), tiles / kMaxParts + 1));
        for (;; size += 1 + size / 8) {   // (ends: with the most tiles of a group as the size there is a piece for every block)
            r.pieces = lane_value(wave_inclusive_scan(blocks_of(r.group) * parts_of(r.group, size)), 63);
            if (r.pieces <= most) break;
        }
        r.size = size;
    }
    r.pieces = min(r.pieces, w.max_pieces);   // (of groups that overlap, which no valid call has, there may be more than there is room for)
    const int n_waves = (G - r.n_tile) * kLineWaves;
    r.quota = max(max((total + n_waves - 1) / max(n_waves, 1), kLeastShare / GR), longest / (kMaxParts - 3) + 1);
    if (writes) {
        if (lane == 0) w.seq_tab[2 * p.n_seqs] = r.quota;
        int first = 0;
        for (int base = 0; base < w.n_groups; base += 64) {
            const Group q = base == 0 ? r.group : group_at(w, base + lane);
            const int parts = parts_of(q, r.size), incl = wave_inclusive_scan(blocks_of(q) * parts);
            if (base + lane < w.n_groups) w.group_tab[base + lane] = i32x4{q.lo, q.rows, first + incl - blocks_of(q) * parts, parts};
            first += lane_value(incl, 63);
        }
    }
    return r;
}

// Pieces rank, rank + ranks, .. of KV head g.
template <class T, int D, bool FP8> MA_DEV void shared_tiles(const SharedWork& w, const SharedPlan& plan, PagedParams p, char* lds) {
    const int lane = threadIdx.x & 63, ranks = plan.n_tile / p.Hkv;
    int g, rank;
    if ((p.Hkv & 7) == 0) {   // a KV head's workgroups on one XCD (ids go round-robin)
        const int per = p.Hkv >> 3, m = (int)blockIdx.x >> 3;
        g = (m % per) * 8 + ((int)blockIdx.x & 7);
        rank = m / per;
    } else {
        g = (int)blockIdx.x % p.Hkv;
        rank = (int)blockIdx.x / p.Hkv;
    }
    p.part_o = w.tile_o;
    p.part_ml = w.tile_ml;
    for (int x = rank; x < plan.pieces; x += ranks) {
        TileJob job{};
        job.g = g;
        job.slot = x;
        int left = x;
        for (int base = 0; base < w.n_groups; base += 64) {
            const Group q = base == 0 ? plan.group : group_at(w, base + lane);
            const int parts = parts_of(q, plan.size), n = blocks_of(q) * parts, incl = wave_inclusive_scan(n), sum = lane_value(incl, 63);
            if (left < sum) {
                const int src = __builtin_amdgcn_readfirstlane(__ffsll((unsigned long long)__ballot(left < incl)) - 1);
                job.first = lane_value(q.first, src);
                job.last = lane_value(q.last, src);
                job.lo = lane_value(q.lo, src);
                job.rows = lane_value(q.rows, src);
                job.ctx = lane_value(q.tiles, src) * 64;
                job.parts = lane_value(parts, src);
                left -= lane_value(incl - n, src);
                break;
            }
            left -= sum;
        }
        if (job.parts <= 0) break;   // (groups that overlap, and sums of them past 31 bits: there is no such piece)
        job.seq = job.first;
        job.block = left / job.parts;
        job.part = left - job.block * job.parts;
        bool inside = false;   // sequences whose first new token stands inside the prefix
        for (int base = job.first; base < job.last; base += 64) {
            const int s = base + lane;
            if (s < job.last) {
                const TokenRange t = token_range(p.cu[s], p.cu[s + 1], p.T);
                inside = inside || (t.len > 0 && context_of(p.c, p.ctx[s], t) - t.len < job.ctx - 1);
            }
        }
        job.inside = __any(inside) != 0;
        if (x != rank) {   // every wave is done with the stages, and its results are on their way no more
            wait_vmcnt<0>();
            __syncthreads();
        }
        attend_tiles<T, D, FP8, kSharedWaves, true>(p, job, lds);
    }
}

// The line, as in paged_line_kernel, of the rows behind the prefixes.
template <class T, int D, bool FP8> MA_DEV void shared_line(const SharedWork& w, const SharedPlan& plan, char* lds) {
    constexpr int GR = kRows<FP8>;
    const DecodeWork& d = w.d;
    const PagedParams& p = d.p;
    const int lane = threadIdx.x & 63, wid = wave_id(), pairs = p.Hkv * d.n_hg;
    const int n_wg = (int)gridDim.x - plan.n_tile, wg = (int)blockIdx.x - plan.n_tile, quota = plan.quota, total = plan.total;
    const int n_shares = total > 0 ? (total - 1) / quota + 1 : 0;
    const int wave = n_shares <= n_wg ? wid * n_wg + wg : wg * kLineWaves + wid;
    if (wave >= n_shares) return;
    int x = wave * quota;
    const int x_end = x + min(quota, total - x);
    int s = 0, off = 0, groups = 0, first = 0;
    for (int base = 0, start = 0; base < p.n_seqs; base += 64) {
        const OwnSeq q = base == 0 ? plan.kept : own_seq<GR>(w, base + lane);
        const int incl = wave_inclusive_scan(q.groups * pairs), sum = lane_value(incl, 63);
        if (x < start + sum) {
            const int src = __builtin_amdgcn_readfirstlane(__ffsll((unsigned long long)__ballot(x < start + incl)) - 1);
            s = base + src;
            groups = lane_value(q.groups, src);
            first = lane_value(q.g0, src);
            off = start + lane_value(incl, src) - groups * pairs;
            break;
        }
        start += sum;
    }
    SeqInfo info = seq_info(p, s);
    while (x < x_end) {
        if (x >= off + pairs * groups) {   // the sequence is done: on to the next that has rows
            off += pairs * groups;
            do {
                info = seq_info(p, ++s);
                const int i = __builtin_amdgcn_readfirstlane(group_of(w, s));
                first = i >= 0 ? __builtin_amdgcn_readfirstlane(shared_rows(w, i)) / GR : 0;
                groups = info.len > 0 ? max((info.ctx + GR - 1) / GR - first, 0) : 0;
            } while (groups == 0);
        }
        const int y = x - off, pair = y / groups, g0 = y - pair * groups, g1 = min(groups, g0 + (x_end - x));
        const int hg = d.n_hg == 1 ? 0 : pair / p.Hkv, g = pair - hg * p.Hkv;
        ColumnAcc<D> acc;
        stream_pages<T, D, FP8>(d, s, info, g, hg, first + g0, first + g1, lds + wid * kWaveLds<D, FP8>, acc);
        store_part<D>(d, hg, (int64_t)s * pairs + pair + wave, acc);
        x += g1 - g0;
    }
}

template <class T, int D, bool FP8>
__global__ __launch_bounds__(kSharedWaves * 64, 2) void shared_kernel(const SharedWork w) {
    static_assert(kSharedWaves == kLineWaves && kLineWaves * kWaveLds<D, FP8> <= TileLds<D, FP8, kSharedWaves>::BYTES, "one size of workgroup, one area");
    __shared__ __attribute__((aligned(1024))) char lds[TileLds<D, FP8, kSharedWaves>::BYTES];
    const SharedPlan plan = plan_shared<D, kRows<FP8>>(w, blockIdx.x == 0 && wave_id() == 0);
    if ((int)blockIdx.x < plan.n_tile) shared_tiles<T, D, FP8>(w, plan, w.d.p, lds);
    else shared_line<T, D, FP8>(w, plan, lds);
}

// out = sum_i O_i w_i / sum_i l_i w_i, w_i = 2^(m_i - max m), over the parts of a row, those of the line and those of its group's prefix; a wave per row (sequence,
// token, head), lane i holding the references and sums of both parts i.
template <class T, int D, int GR>
__global__ __launch_bounds__(256) void shared_merge_kernel(const SharedWork w) {
    const DecodeWork& work = w.d;
    const PagedParams& p = work.p;
    constexpr int EPL = D / 64;
    const int lane = threadIdx.x & 63;
    const int64_t row = (int64_t)blockIdx.x * 4 + wave_id();
    const int per_seq = p.Hkv * work.n_col;
    if (row >= (int64_t)p.n_seqs * per_seq) return;
    const int s = (int)(row / per_seq), in = (int)(row - (int64_t)s * per_seq), g = in / work.n_col, col = in - g * work.n_col;
    const SeqInfo info = seq_info(p, s);
    const int tok = col / p.n_rep, head = col - tok * p.n_rep;
    if (tok >= info.len) return;
    const int group = const_load(w.seq_tab + 2 * s + 1), quota = const_load(w.seq_tab + 2 * p.n_seqs), pair = (col / 16) * p.Hkv + g;
    // the parts of the group's prefix
    int n_pre = 0, skip = 0;
    int64_t pre0 = 0;
    const int64_t pre_step = (int64_t)p.Hkv * kBlockRows;
    if (group >= 0) {
        skip = shared_rows(w, group);
        const i32x4 t = const_load(w.group_tab + group);   // as written by plan_shared
        const int r = (info.lo + tok - t[0]) * p.n_rep + head;
        if (skip > 0 && r >= 0 && r < t[1]) {
            const int64_t piece = t[2] + (int64_t)(r / kBlockRows) * t[3];
            if (piece >= 0 && piece < w.max_pieces) {
                n_pre = min(min(t[3], kMaxParts), (int)(w.max_pieces - piece));
                pre0 = (piece * p.Hkv + g) * kBlockRows + r % kBlockRows;
            }
        }
    }
    // those of the line
    const int groups = max((info.ctx + GR - 1) / GR - skip / GR, 0);
    const int start = const_load(w.seq_tab + 2 * s) + pair * groups, first = start / quota;
    const int ns = groups > 0 ? min((start + groups - 1) / quota - first + 1, kMaxParts) : 0;
    const int64_t at0 = part_row(work, (int64_t)s * p.Hkv * work.n_hg + pair + first, col % 16);
    f32x2 ml = {-INFINITY, 0.f}, pre = {-INFINITY, 0.f};
    if (lane < ns) ml = *reinterpret_cast<const f32x2*>(p.part_ml + (at0 + (int64_t)lane * work.per_part) * 2);
    if (lane < n_pre) pre = *reinterpret_cast<const f32x2*>(w.tile_ml + (pre0 + lane * pre_step) * 2);
    auto load_o = [&](const float* at, float (&x)[EPL]) __attribute__((always_inline)) {
        if (EPL == 2) { const f32x2 v = *reinterpret_cast<const f32x2*>(at); x[0] = v[0]; x[EPL - 1] = v[1]; }
        else x[0] = at[0];
    };
    const float top = wave_max(max2(ml[0], pre[0]));
    const float w_own = ml[0] > -INFINITY ? fast_exp2(ml[0] - top) : 0.f, w_pre = pre[0] > -INFINITY ? fast_exp2(pre[0] - top) : 0.f;
    const float all = lane_sum<64>(ml[1] * w_own + pre[1] * w_pre);
    float acc[EPL];
#pragma unroll
    for (int e = 0; e < EPL; ++e) acc[e] = 0.f;
    auto add = [&](const float* src, int64_t step, int n, float weight) __attribute__((always_inline)) {
        for (int i0 = 0; i0 < n; i0 += 8) {
            float x[8][EPL];
#pragma unroll
            for (int u = 0; u < 8; ++u) load_o(src + min(i0 + u, n - 1) * step, x[u]);
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const float wi = lane_value(weight, min(i0 + u, 63));
#pragma unroll
                for (int e = 0; e < EPL; ++e) acc[e] += i0 + u < n ? x[u][e] * wi : 0.f;
            }
        }
    };
    add(w.tile_o + pre0 * D + EPL * lane, pre_step * D, n_pre, w_pre);
    add(p.part_o + at0 * D + EPL * lane, (int64_t)work.per_part * D, ns, w_own);
    const float inv = all > 0.f ? 1.f / all : 0.f;
    uint16_t* dst = reinterpret_cast<uint16_t*>(p.out) + (int64_t)(info.lo + tok) * p.o2 + (int64_t)(g * p.n_rep + head) * p.o1 + EPL * lane;
    if (EPL == 2) *reinterpret_cast<uint32_t*>(dst) = T::pack2(acc[0] * inv, acc[EPL - 1] * inv);
    else dst[0] = (uint16_t)(T::pack2(acc[0] * inv, 0.f) & 0xffffu);
}

// Whether a call is one for these kernels; others go to flash_attn_paged, whose blocks of rows fill up with a single sequence's tokens.
static bool shared_takes(int64_t n_groups, int64_t Hq, int64_t Hkv, int64_t max_q) {
    const int64_t n_rep = Hq / Hkv;
    return n_groups > 0 && Hkv <= kMaxSharedHeads && (max_q == 1 || (n_rep <= 16 && max_q * n_rep <= 64));
}

// How a call is laid out, from its sizes alone.
struct SharedSizes { int64_t n_col, n_hg, per_part, parts, pieces; size_t o_bytes, ml_bytes, tile_o_bytes, tile_ml_bytes, seq_bytes, bytes; };
static size_t lines(int64_t bytes) { return ((size_t)bytes + 255) / 256 * 256; }
static SharedSizes shared_sizes(int64_t n_seqs, int64_t n_groups, int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int64_t max_q) {
    SharedSizes r{};
    const int64_t n_rep = Hq / Hkv;
    r.n_col = max_q * n_rep;
    r.n_hg = (r.n_col + 15) / 16;
    r.per_part = std::min<int64_t>(r.n_col, 16);
    r.parts = (int64_t)kSharedWgs * kLineWaves + n_seqs * Hkv * r.n_hg;
    r.pieces = std::max<int64_t>(kSharedWgs / Hkv, T * n_rep / kBlockRows + n_groups);
    r.o_bytes = lines(r.parts * r.per_part * D * 4);
    r.ml_bytes = lines(r.parts * r.per_part * 2 * 4);
    r.tile_o_bytes = lines(r.pieces * Hkv * kBlockRows * D * 4);
    r.tile_ml_bytes = lines(r.pieces * Hkv * kBlockRows * 2 * 4);
    r.seq_bytes = lines((2 * n_seqs + 1) * 4);
    r.bytes = r.o_bytes + r.ml_bytes + r.tile_o_bytes + r.tile_ml_bytes + r.seq_bytes + lines(n_groups * 16);
    return r;
}

template <class T, int D, bool FP8> static int launch_shared(const SharedWork& w, hipStream_t stream) {
    hipLaunchKernelGGL((shared_kernel<T, D, FP8>), dim3(kSharedWgs), dim3(kSharedWaves * 64), 0, stream, w);
    if (int rc = check_launch("shared_kernel")) return rc;
    const int64_t rows = (int64_t)w.d.p.n_seqs * w.d.p.Hkv * w.d.n_col;
    hipLaunchKernelGGL((shared_merge_kernel<T, D, kRows<FP8>>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, stream, w);
    return check_launch("shared_merge_kernel");
}
template <class T> static int launch_shared_as(const SharedWork& w, int64_t D, bool eight, hipStream_t stream) {
    if (eight) return D == 128 ? launch_shared<T, 128, true>(w, stream) : launch_shared<T, 64, true>(w, stream);
    return D == 128 ? launch_shared<T, 128, false>(w, stream) : launch_shared<T, 64, false>(w, stream);
}

static int64_t bounded_tokens(int64_t T, int64_t max_q_len) { return max_q_len > 0 && max_q_len < T ? max_q_len : T; }

}  // namespace minfer_attn

using namespace minfer_attn;

MINFER_ATTN_EXPORT size_t minfer_flash_attn_paged_shared_workspace_bytes(int64_t n_seqs, int64_t n_groups, int64_t T, int64_t Hq, int64_t Hkv, int64_t D,
                                                                         int64_t max_context, int64_t max_q_len) {
    if (n_seqs <= 0 || n_groups < 0 || T <= 0 || Hq <= 0 || Hkv <= 0 || D <= 0 || max_context < 0 || Hq % Hkv != 0) return 0;
    const int64_t max_q = bounded_tokens(T, max_q_len);
    if (!shared_takes(n_groups, Hq, Hkv, max_q)) return minfer_flash_attn_paged_workspace_bytes(n_seqs, T, Hq, Hkv, D, max_context, max_q_len);
    return shared_sizes(n_seqs, n_groups, T, Hq, Hkv, D, max_q).bytes;
}

MINFER_ATTN_EXPORT int minfer_flash_attn_paged_shared(int dtype, int page_type, const void* q, const minfer_kv_pages* pages, const int32_t* cu_seqlens,
                                                      const int32_t* ctx_lens, const int32_t* cu_groups, const int32_t* prefix_lens, void* out, int64_t n_seqs,
                                                      int64_t n_groups, int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int64_t max_q_len,
                                                      const minfer_attn_strides* st, void* workspace, size_t workspace_bytes, void* stream_v) {
    clear_error();
    SharedWork w{};
    PagedParams& p = w.d.p;
    if (int rc = check_pages("flash_attn_paged_shared", dtype, page_type, pages, n_seqs, Hkv, D, p.c)) return rc;
    auto bad = [&](const char* what) { return fail(MINFER_ATTN_EINVAL, what); };
    if (Hq <= 0 || Hq % Hkv != 0) return bad("flash_attn_paged_shared: n_heads must be a positive multiple of n_kv_heads");
    if (Hq > 65535) return bad("flash_attn_paged_shared: n_heads > 65535 unsupported");
    if (!st) return bad("flash_attn_paged_shared: strides is null");
    if (n_seqs < 0 || T < 0 || max_q_len < 0 || n_groups < 0) return bad("flash_attn_paged_shared: negative size");
    if (n_groups > n_seqs) return bad("flash_attn_paged_shared: more groups than sequences");
    if (n_seqs == 0 || T == 0) return MINFER_ATTN_OK;
    if (!q || !out || !cu_seqlens || !ctx_lens) return bad("flash_attn_paged_shared: q, out, cu_seqlens and ctx_lens must be non-null");
    if (n_groups > 0 && (!cu_groups || !prefix_lens)) return bad("flash_attn_paged_shared: cu_groups and prefix_lens must be non-null");
    const int64_t max_q = bounded_tokens(T, max_q_len);
    if (!shared_takes(n_groups, Hq, Hkv, max_q))
        return minfer_flash_attn_paged(dtype, page_type, q, pages, cu_seqlens, ctx_lens, out, n_seqs, T, Hq, Hkv, D, max_q_len, st, workspace, workspace_bytes, stream_v);
    if (!aligned16(q) || !aligned16(out)) return bad("flash_attn_paged_shared: q and out must be 16-byte aligned");
    const int64_t s[4] = {st->q1, st->q2, st->o1, st->o2};
    for (int i = 0; i < 4; ++i)
        if (s[i] < 0 || s[i] % 8 != 0) return bad("flash_attn_paged_shared: strides of q and out must be non-negative multiples of 8 elements");
    const int64_t max_context = (int64_t)p.c.width << p.c.page_log2;
    if (T > (1 << 30) || T * Hq > 0x7fffffffLL - 4096 || n_seqs > (1 << 24)) return bad("flash_attn_paged_shared: problem too large for one launch");
    const SharedSizes z = shared_sizes(n_seqs, n_groups, T, Hq, Hkv, D, max_q);
    if (n_seqs * Hkv * z.n_col > 0x7fffffffLL || n_seqs * Hkv * z.n_hg * ((max_context + 15) / 16 + 1) > 0x7fffffffLL - 65536)
        return bad("flash_attn_paged_shared: problem too large for one launch");
    if (!workspace || !aligned16(workspace) || workspace_bytes < z.bytes)
        return fail(MINFER_ATTN_EWORKSPACE, "flash_attn_paged_shared: workspace too small or misaligned (see minfer_flash_attn_paged_shared_workspace_bytes)");
    p.q = q; p.out = out; p.cu = cu_seqlens; p.ctx = ctx_lens;
    p.q1 = st->q1; p.q2 = st->q2; p.o1 = st->o1; p.o2 = st->o2;
    p.n_seqs = (int)n_seqs; p.T = (int)T; p.Hq = (int)Hq; p.Hkv = (int)Hkv; p.n_rep = (int)(Hq / Hkv);
    p.max_q = (int)max_q;
    p.scale_log2 = (float)(1.4426950408889634 / sqrt((double)D));
    p.inv_scale_log2 = (float)(sqrt((double)D) / 1.4426950408889634);
    char* at = (char*)workspace;
    p.part_o = (float*)at; at += z.o_bytes;
    p.part_ml = (float*)at; at += z.ml_bytes;
    w.tile_o = (float*)at; at += z.tile_o_bytes;
    w.tile_ml = (float*)at; at += z.tile_ml_bytes;
    w.seq_tab = (int32_t*)at; at += z.seq_bytes;
    w.group_tab = (i32x4*)at;
    w.d.n_col = (int)z.n_col; w.d.n_hg = (int)z.n_hg; w.d.per_part = (int)z.per_part;
    w.cu_groups = cu_groups; w.prefix = prefix_lens; w.n_groups = (int)n_groups;
    w.max_pieces = (int)z.pieces;
    const bool eight = page_type == MINFER_FP8_E4M3;
    return dtype == MINFER_ATTN_F16 ? launch_shared_as<F16>(w, D, eight, (hipStream_t)stream_v) : launch_shared_as<BF16>(w, D, eight, (hipStream_t)stream_v);
}
