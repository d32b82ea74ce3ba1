// Attention of few query rows per KV head over a paged cache for gfx950: single tokens of many sequences, drafts of a few tokens.
//
// HBM-bound: each cached row is used by at most 16 columns (a token and head each) at a time, so what counts is bytes in flight.  The columns of a
// KV head are its group's query heads for every new token of the sequence, token by token; up to 16 of them are the columns of one
// 16-wide matrix product, each with a limit of its own (the row of its token), so a few drafts read the cache once.
//
// How a wave streams rows is csrc/attn_paged_stream.h's.
//
// Two ways to share the work out:
// * the line: all rows to be read, sequence by sequence, KV head by KV head, cut into as many equal shares as the launch has waves; a
//   wave's share covers parts of a few (sequence, KV head) pairs, each of which leaves a partial result that
//   paged_merge_kernel puts together.  Whatever the mix of contexts, all waves end together.  64 sequences of 512 to 8192 rows, 32 query
//   heads on 8 of 128: 179 us, 6.1 TB/s, of which the merge 5; over codes 98 us, 5.6 TB/s.
// * chunks, for few pairs: eight waves of a workgroup share one chunk of a pair and merge in LDS, and the last workgroup of a pair merges its
//   chunks (on the null stream; elsewhere paged_chunk_merge_kernel does).  A sequence is cut by its own context, which the host does not know.
//   12 sequences of 3 or 4 drafts, 28964 rows: 27 us, 4.4 TB/s; one token, 8 heads on 2 of 64, against 1501 rows 8 us, three against 5570 rows of
//   codes 10 us, which is latency: a launch, two dependent loads of tables, the first rows, the merge in LDS.
#include <algorithm>
#include <atomic>

#include "attn_paged_stream.h"

namespace minfer_attn {

constexpr int kLineWgPerCu = 2;
constexpr int kChunkWaves = 8;

template <class T, int D, bool FP8>
__global__ __launch_bounds__(kLineWaves * 64, 2) void paged_line_kernel(const DecodeWork work) {
    __shared__ __attribute__((aligned(1024))) char lds[kLineWaves][kWaveLds<D, FP8>];
    constexpr int GR = kRows<FP8>;
    const PagedParams& p = work.p;
    const int lane = threadIdx.x & 63, w = wave_id();
    const int pairs = p.Hkv * work.n_hg, n_waves = work.n_wg * kLineWaves;
    const bool first = blockIdx.x == 0 && w == 0;   // the wave that leaves the sequences' places for the merge
    // 64 sequences at a time, 256 requested together; the first 64 are kept
    constexpr int UN = 4;
    LineSeq kept{{0, 0, 0}, 0};
    int total = 0, longest = 0;
    for (int base = 0; base < p.n_seqs; base += 64 * UN) {
        LineSeq q[UN];
#pragma unroll
        for (int u = 0; u < UN; ++u) q[u] = line_seq<GR>(work, base + 64 * u + lane);
        if (base == 0) kept = q[0];
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            const int b = base + 64 * u;
            if (b >= p.n_seqs) break;
            const int incl = wave_inclusive_scan(q[u].groups * pairs);
            if (first && b + lane < p.n_seqs) work.seq_off[b + lane] = total + incl - q[u].groups * pairs;
            total += lane_value(incl, 63);
            longest = max(longest, q[u].groups);
        }
    }
    longest = (int)wave_max((float)longest);   // (below 2^24 exactly, and above rounded up or down by less than the parts to spare)
    const int quota = max(max((total + n_waves - 1) / n_waves, kLeastShare / GR), longest / (kMaxParts - 3) + 1);
    if (first && lane == 0) { work.seq_off[p.n_seqs] = total; work.seq_off[p.n_seqs + 1] = quota; }
    // shares to the waves of a workgroup in turn; where there are no more shares than workgroups, one to each
    // (the line's length and a share of it may together pass 31 bits)
    const int n_shares = total > 0 ? (total - 1) / quota + 1 : 0;
    const int wave = n_shares <= (int)gridDim.x ? w * (int)gridDim.x + (int)blockIdx.x : (int)blockIdx.x * kLineWaves + w;
    if (wave >= n_shares) return;
    int x = wave * quota;
    const int x_end = x + min(quota, total - x);
    // the sequence that holds position x
    int s = 0, off = 0, groups = 0;
    for (int base = 0, start = 0; base < p.n_seqs; base += 64) {
        const LineSeq q = base == 0 ? kept : line_seq<GR>(work, base + lane);
        const int incl = wave_inclusive_scan(q.groups * pairs), sum = lane_value(incl, 63);
        if (x < start + sum) {
            const int src = __builtin_amdgcn_readfirstlane(__ffsll((unsigned long long)__ballot(x < start + incl)) - 1);
            s = base + src;
            groups = lane_value(q.groups, src);
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
                groups = info.len > 0 ? (info.ctx + GR - 1) / GR : 0;
            } while (groups == 0);
        }
        const int y = x - off, pair = y / groups, g0 = y - pair * groups, g1 = min(groups, g0 + (x_end - x));
        const int hg = work.n_hg == 1 ? 0 : pair / p.Hkv, g = pair - hg * p.Hkv;
        ColumnAcc<D> acc;
        stream_pages<T, D, FP8>(work, s, info, g, hg, g0, g1, lds[w], acc);
        store_part<D>(work, hg, (int64_t)s * pairs + pair + wave, acc);
        x += g1 - g0;
    }
}

// out = sum_i O_i w_i / sum_i l_i w_i, w_i = 2^(m_i - max m), over the parts of a row; a wave per row (sequence, token, head), lane i holding part i's
// reference and sum.
template <class T, int D, int GR>
__global__ __launch_bounds__(256) void paged_merge_kernel(const DecodeWork work) {
    const PagedParams& p = work.p;
    constexpr int EPL = D / 64;
    const int lane = threadIdx.x & 63;
    const int64_t row = (int64_t)blockIdx.x * 4 + wave_id();
    const int per_seq = p.Hkv * work.n_col;
    if (row >= (int64_t)p.n_seqs * per_seq) return;
    const int s = (int)(row / per_seq), in = (int)(row - (int64_t)s * per_seq), g = in / work.n_col, col = in - g * work.n_col;
    const SeqInfo info = seq_info(p, s);
    const int tok = col / p.n_rep;
    if (tok >= info.len) return;
    const int groups = (info.ctx + GR - 1) / GR, quota = const_load(work.seq_off + p.n_seqs + 1), pair = (col / 16) * p.Hkv + g;
    const int start = const_load(work.seq_off + s) + pair * groups, first = start / quota;   // the pair's first group and its share
    const int ns = groups > 0 ? min((start + groups - 1) / quota - first + 1, kMaxParts) : 0;
    const int64_t at0 = part_row(work, (int64_t)s * p.Hkv * work.n_hg + pair + first, col % 16);
    const float* src = p.part_o + at0 * D + EPL * lane;
    auto load_o = [&](int part, float (&x)[EPL]) __attribute__((always_inline)) {
        const float* at = src + (int64_t)part * work.per_part * D;
        if (EPL == 2) { const f32x2 v = *reinterpret_cast<const f32x2*>(at); x[0] = v[0]; x[EPL - 1] = v[1]; }
        else x[0] = at[0];
    };
    // the first parts' rows beside their references and sums
    f32x2 ml = {-INFINITY, 0.f};
    if (lane < ns) ml = *reinterpret_cast<const f32x2*>(p.part_ml + (at0 + (int64_t)lane * work.per_part) * 2);
    constexpr int kEarly = 4;
    float x[8][EPL];
#pragma unroll
    for (int u = 0; u < kEarly; ++u) {
#pragma unroll
        for (int e = 0; e < EPL; ++e) x[u][e] = 0.f;
        if (ns > 0) load_o(min(u, ns - 1), x[u]);
    }
    const PartWeights pw = part_weights(ml[0], ml[1]);
    float acc[EPL];
#pragma unroll
    for (int e = 0; e < EPL; ++e) acc[e] = 0.f;
    for (int s0 = 0; s0 < ns; s0 += 8) {
#pragma unroll
        for (int u = 0; u < 8; ++u)
            if (s0 > 0 || u >= kEarly) load_o(min(s0 + u, ns - 1), x[u]);
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const float wi = lane_value(pw.w, min(s0 + u, 63));
#pragma unroll
            for (int e = 0; e < EPL; ++e) acc[e] += s0 + u < ns ? x[u][e] * wi : 0.f;
        }
    }
    const float inv = pw.total > 0.f ? 1.f / pw.total : 0.f;
    uint16_t* dst = reinterpret_cast<uint16_t*>(p.out) + (int64_t)(info.lo + tok) * p.o2 + (int64_t)(g * p.n_rep + col - tok * p.n_rep) * p.o1 + EPL * lane;
    if (EPL == 2) *reinterpret_cast<uint32_t*>(dst) = T::pack2(acc[0] * inv, acc[EPL - 1] * inv);
    else dst[0] = (uint16_t)(T::pack2(acc[0] * inv, 0.f) & 0xffffu);
}

// ---- chunks ----------------------------------------------------------------------------------------------------------
// What the line costs a small problem is latency: a wave streams its rows one group after the other, and a second launch merges.  Here the eight waves of
// a workgroup share a chunk and merge in LDS.  A pair that is one chunk long is done with that; otherwise the chunk's result goes to
// the workspace, and the workgroup that comes last (a counter per pair) merges the pair's.  Results cross from one XCD's L2 to
// another's: they are written and read with device-scope accesses, which go past the L2s on both sides, and a workgroup counts itself
// only when its own have arrived; the reader's loads stand behind a barrier that thread 0 reaches with the count's value in hand.
MA_DEV void store_shared(float* p, float x) { __hip_atomic_store(p, x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
MA_DEV float load_shared(const float* p) { return __hip_atomic_load(const_cast<float*>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
MA_DEV void store_shared2(float* p, f32x2 x) {
    __hip_atomic_store(reinterpret_cast<uint64_t*>(p), __builtin_bit_cast(uint64_t, x), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
MA_DEV f32x2 load_shared2(const float* p) {
    return __builtin_bit_cast(f32x2, __hip_atomic_load(reinterpret_cast<uint64_t*>(const_cast<float*>(p)), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
}

// Every pair of a sequence is cut into the same number of chunks, equal to within a group; the chunk's size, the same for all sequences, is the
// smallest (256 rows at least) that leaves no more chunks than workgroups.  Up to 64 sequences, one to a lane; all waves
// work it out for themselves.
template <int GR> struct ChunkPlan {
    LineSeq q;        // per lane: the sequence
    int each, incl;   // per lane: chunks of each of its pairs; chunks of the sequences up to and with it
    int total;
    MA_DEV ChunkPlan(const DecodeWork& w, int n_wg) {
        const int lane = threadIdx.x & 63, pairs = w.p.Hkv * w.n_hg;
        q = line_seq<GR>(w, lane);
        const bool on = lane < w.p.n_seqs && q.info.len > 0;
        const int sum = lane_value(wave_inclusive_scan(q.groups * pairs), 63), active = __popcll(__ballot(on));
        const int longest = (int)wave_max((float)q.groups);
        // a pair's last chunk is half full on average: that many workgroups are as good as not there
        int size = max(max((sum + n_wg - 1) / max(n_wg - active * pairs / 2, 1), 256 / GR), longest / kMaxParts + 1);
        for (;; size += 1 + size / 16) {   // (ends: with the longest context as the size there is one chunk a pair, and no more pairs than workgroups)
            each = on ? max((q.groups + size - 1) / size, 1) : 0;
            incl = wave_inclusive_scan(each * pairs);
            total = lane_value(incl, 63);
            if (total <= n_wg) break;
        }
    }
};

// Merges the n chunks, from number `first` of the launch on, of the columns of (s, g, hg) from the workspace and stores the output rows; all threads of the workgroup, a wave 64
// elements of a column at a time, without LDS and barriers (with the weights made by 16 threads in LDS it took twice the time).  The order of
// the sums depends on nothing but n.
template <class T, int D>
MA_DEV void merge_chunks(const DecodeWork& w, const SeqInfo& info, int g, int hg, int first, int n) {
    const PagedParams& p = w.p;
    const int lane = threadIdx.x & 63, wave = wave_id(), cols = min(16, w.n_col - hg * 16);
    const int64_t at0 = part_row(w, first, 0), step = (int64_t)w.per_part * D;
    constexpr int PER = 16 * D / (kChunkWaves * 64);
    float x[PER][8];
    f32x2 ml[PER];
#pragma unroll
    for (int e = 0; e < PER; ++e) {
        const int idx = (wave + e * kChunkWaves) * 64;
        if (idx < cols * D) {
            const int64_t at = at0 + idx / D;
            ml[e] = load_shared2(p.part_ml + (at + (int64_t)min(lane, n - 1) * w.per_part) * 2);
            const float* src = p.part_o + at * D + idx % D + lane;
#pragma unroll
            for (int u = 0; u < 8; ++u) x[e][u] = load_shared(src + min(u, n - 1) * step);
        }
    }
#pragma unroll
    for (int e = 0; e < PER; ++e) {
        const int idx = (wave + e * kChunkWaves) * 64;
        if (idx >= cols * D) break;
        const int c = idx / D, d = idx % D + lane, col = hg * 16 + c, tok = col / p.n_rep;
        const PartWeights pw = part_weights(lane < n ? ml[e][0] : -INFINITY, lane < n ? ml[e][1] : 0.f);
        const float* src = p.part_o + (at0 + c) * D + d;
        float sum = 0.f;
        for (int s0 = 0; s0 < n; s0 += 8) {
            if (s0 > 0) {
#pragma unroll
                for (int u = 0; u < 8; ++u) x[e][u] = load_shared(src + min(s0 + u, n - 1) * step);
            }
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const float wi = lane_value(pw.w, min(s0 + u, 63));
                sum += s0 + u < n ? x[e][u] * wi : 0.f;
            }
        }
        if (tok < info.len)
            reinterpret_cast<uint16_t*>(p.out)[(int64_t)(info.lo + tok) * p.o2 + (int64_t)(g * p.n_rep + col - tok * p.n_rep) * p.o1 + d] = (uint16_t)(T::pack2(sum * (pw.total > 0.f ? 1.f / pw.total : 0.f), 0.f) & 0xffffu);
    }
}

template <class T, int D, bool FP8>
__global__ __launch_bounds__(kChunkWaves * 64, 2) void paged_chunk_kernel(const DecodeWork work) {
    const PagedParams& p = work.p;
    constexpr int NW = kChunkWaves, DB = D / 16, GR = kRows<FP8>, WAVE_LDS = kWaveLds<D, FP8>;
    constexpr int ORS = D + 4;   // floats between two columns of a wave's result: their 16-byte pieces start in different banks
    constexpr int LDS = NW * WAVE_LDS > NW * 16 * ORS * 4 ? NW * WAVE_LDS : NW * 16 * ORS * 4;
    __shared__ __attribute__((aligned(1024))) char lds[LDS];   // the waves' row areas, then their results
    __shared__ float ml_s[2 * NW * 16];
    __shared__ int last_s;
    const int tid = threadIdx.x, lane = tid & 63, w = wave_id(), l16 = lane & 15, quad = lane >> 4;
    const int pairs = p.Hkv * work.n_hg;
    const ChunkPlan<GR> plan(work, (int)gridDim.x);
    const int x = (int)blockIdx.x;
    if (x >= plan.total) return;
    const int s = __builtin_amdgcn_readfirstlane(__ffsll((unsigned long long)__ballot(x < plan.incl)) - 1);
    const SeqInfo info{lane_value(plan.q.info.lo, s), lane_value(plan.q.info.len, s), lane_value(plan.q.info.ctx, s)};
    const int n = lane_value(plan.each, s), all = lane_value(plan.q.groups, s);   // chunks and groups of the pair
    const int local = x - (lane_value(plan.incl, s) - n * pairs), pair = local / n, split = local - pair * n;
    const int hg = work.n_hg == 1 ? 0 : pair / p.Hkv, g = pair - hg * p.Hkv;
    const int size = all / n, longer = all - size * n;   // the first `longer` chunks are a group longer
    const int first = split * size + min(split, longer), groups = size + (split < longer ? 1 : 0);
    const int per = (groups + NW - 1) / NW;
    const int g_lo = min(w * per, groups), g_hi = min(g_lo + per, groups);
    ColumnAcc<D> acc;
    acc.m = -INFINITY; acc.l = 0.f;
#pragma unroll
    for (int db = 0; db < DB; ++db) acc.o[db] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (g_hi > g_lo) stream_pages<T, D, FP8>(work, s, info, g, hg, first + g_lo, first + g_hi, lds + w * WAVE_LDS, acc);
    __syncthreads();   // every wave is done with its row area
    const int cols = min(16, work.n_col - hg * 16);
    float* o_s = reinterpret_cast<float*>(lds);   // [wave][column][ORS]
    if (l16 < cols) {
        float* dst = o_s + (w * 16 + l16) * ORS + 4 * quad;
#pragma unroll
        for (int db = 0; db < DB; ++db) *reinterpret_cast<f32x4*>(dst + 16 * db) = acc.o[db];
        if (quad == 0) { ml_s[w * 16 + l16] = acc.m; ml_s[(NW + w) * 16 + l16] = acc.l; }
    }
    __syncthreads();
    const bool whole = n <= 1;   // the chunk is the whole context: its result is the output
    const int64_t at0 = part_row(work, x, 0);
    for (int idx = w * 64; idx < cols * D; idx += NW * 64) {   // a wave 64 elements of a column
        const int c = idx / D, d = idx % D + lane;
        const PartWeights pw = part_weights(lane < NW ? ml_s[lane * 16 + c] : -INFINITY, lane < NW ? ml_s[(NW + lane) * 16 + c] : 0.f);
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < NW; ++i) sum += o_s[(i * 16 + c) * ORS + d] * lane_value(pw.w, i);
        if (whole) {
            const int col = hg * 16 + c, tok = col / p.n_rep;
            if (tok < info.len)
                reinterpret_cast<uint16_t*>(p.out)[(int64_t)(info.lo + tok) * p.o2 + (int64_t)(g * p.n_rep + col - tok * p.n_rep) * p.o1 + d] = (uint16_t)(T::pack2(sum * (pw.total > 0.f ? 1.f / pw.total : 0.f), 0.f) & 0xffffu);
        } else {
            store_shared(p.part_o + (at0 + c) * D + d, sum);
            if (idx % D == 0 && lane == 0) store_shared2(p.part_ml + (at0 + c) * 2, f32x2{pw.top, pw.total});
        }
    }
    if (whole || !work.done) return;
    wait_vmcnt<0>();   // the thread's stores have arrived
    __syncthreads();
    if (tid == 0) {
        uint32_t* done = work.done + s * pairs + pair;
        const uint32_t before = __hip_atomic_fetch_add(done, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        last_s = before == (uint32_t)(n - 1);
        if (last_s) __hip_atomic_store(done, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (last_s) merge_chunks<T, D>(work, info, g, hg, x - split, n);
}

// (where there are no counters) grid (column groups x KV heads, sequences)
template <class T, int D, int GR>
__global__ __launch_bounds__(kChunkWaves * 64) void paged_chunk_merge_kernel(const DecodeWork work, int n_wg) {
    const PagedParams& p = work.p;
    const int s = blockIdx.y, hg = (int)blockIdx.x / p.Hkv, g = (int)blockIdx.x - hg * p.Hkv;
    const ChunkPlan<GR> plan(work, n_wg);
    const int n = lane_value(plan.each, s), pairs = p.Hkv * work.n_hg;
    if (n > 1) merge_chunks<T, D>(work, seq_info(p, s), g, hg, lane_value(plan.incl, s) - n * (pairs - (int)blockIdx.x), n);
}

// Workgroups of the line: as many as the chip holds at once.
static int compute_units() {
    static std::atomic<int> cached[64];
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) dev = 0;
    int n = cached[dev].load(std::memory_order_relaxed);
    if (n == 0) {
        if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0) n = 256;
        cached[dev].store(n, std::memory_order_relaxed);
    }
    return n;
}

bool paged_decode_takes(int64_t Hq, int64_t Hkv, int64_t max_q) { return max_q == 1 || max_q * (Hq / Hkv) <= 16; }

template <class T, int D, bool FP8> static int launch_line(DecodeWork w, hipStream_t stream) {
    hipLaunchKernelGGL((paged_line_kernel<T, D, FP8>), dim3((unsigned)w.n_wg), dim3(kLineWaves * 64), 0, stream, w);
    if (int rc = check_launch("paged_line_kernel")) return rc;
    const int64_t rows = (int64_t)w.p.n_seqs * w.p.Hkv * w.n_col;
    hipLaunchKernelGGL((paged_merge_kernel<T, D, kRows<FP8>>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, stream, w);
    return check_launch("paged_merge_kernel");
}
// Whether a call is one for chunks.  Up to a pair for every unit always (us, chunks / line, contexts alike and from a sixteenth up, 32 heads on 8 of 128: one of 4000
// 10.0 / 14.0, 8.2 / 10.6; 4 of 30000 78 / 87, 43 / 62; 16 of 4000 44 / 48, 26 / 31, of 20000 e4m3 109 / 114, 87 / 76; 32 of 300 8.4 / 15.9, 7.2 / 12.3, of 1500
// e4m3 21 / 28, 18 / 21; where every unit has one long context, contexts that differ leave units idle: 32 of 6000 123 / 131, 79 / 72, e4m3 66 / 73, 55 / 45).
// Two rounds of whole contexts where the table has no room for long ones: 64 of 100 11.5 / 13.2, 10.7 / 14.0, of 400 23.0 / 24.6, 17.0 / 17.6, of 1000
// 44.5 / 48.8, 30.2 / 30.4, of 2000 82 / 88, 55 / 53, of 6000 242 / 251, 148 / 141; e4m3 of 100 11.4 / 11.4, 10.9 / 12.5, of 400 18.1 / 21.1, 16.8 / 15.6, of 700 23.4 /
// 27.1, 20.7 / 20.8, of 1000 32.0 / 31.0, 27.9 / 24.4.
static int chunk_rounds(int64_t n_seqs, int64_t pairs, int64_t max_context, bool eight) {
    const int64_t units = compute_units();
    if (n_seqs > 64 || pairs > kStreamCounters) return 0;
    return pairs <= units ? 1 : pairs <= 2 * units && max_context <= (eight ? 768 : 2048) ? 2 : 0;
}

// How a call is laid out, from its sizes alone.
struct DecodePlan {
    int64_t n_col, n_hg, per_part;   // as in DecodeWork
    int rounds;                      // chunk_rounds
    int64_t parts;                   // partial results: chunks, a workgroup each; of the line, shares and pairs
    size_t o_bytes, ml_bytes, bytes;
};
static size_t whole_lines(int64_t bytes) { return ((size_t)bytes + 255) / 256 * 256; }
static DecodePlan plan_decode(bool eight, int64_t n_seqs, int64_t Hq, int64_t Hkv, int64_t D, int64_t max_context, int64_t max_q) {
    DecodePlan r{};
    r.n_col = max_q * (Hq / Hkv);
    r.n_hg = (r.n_col + 15) / 16;
    r.per_part = std::min<int64_t>(r.n_col, 16);
    const int64_t pairs = n_seqs * Hkv * r.n_hg, units = compute_units();
    r.rounds = chunk_rounds(n_seqs, pairs, max_context, eight);
    r.parts = r.rounds > 0 ? r.rounds * units : units * kLineWgPerCu * kLineWaves + pairs;
    r.o_bytes = whole_lines(r.parts * r.per_part * D * 4);
    r.ml_bytes = whole_lines(r.parts * r.per_part * 2 * 4);
    r.bytes = r.o_bytes + r.ml_bytes + (r.rounds > 0 ? 0 : whole_lines((n_seqs + 2) * 4));
    return r;
}
size_t paged_decode_workspace_bytes(int64_t n_seqs, int64_t Hq, int64_t Hkv, int64_t D, int64_t max_context, int64_t max_q) {
    return std::max(plan_decode(false, n_seqs, Hq, Hkv, D, max_context, max_q).bytes, plan_decode(true, n_seqs, Hq, Hkv, D, max_context, max_q).bytes);
}

template <class T, int D, bool FP8> static int launch_chunks(DecodeWork w, int rounds, hipStream_t stream) {
    const int n_wg = rounds * compute_units();
    w.done = stream_counters(stream);
    hipLaunchKernelGGL((paged_chunk_kernel<T, D, FP8>), dim3((unsigned)n_wg), dim3(kChunkWaves * 64), 0, stream, w);
    if (int rc = check_launch("paged_chunk_kernel")) return rc;
    if (w.done) return MINFER_ATTN_OK;
    hipLaunchKernelGGL((paged_chunk_merge_kernel<T, D, kRows<FP8>>), dim3((unsigned)(w.p.Hkv * w.n_hg), (unsigned)w.p.n_seqs), dim3(kChunkWaves * 64), 0, stream, w, n_wg);
    return check_launch("paged_chunk_merge_kernel");
}
template <class T, int D, bool FP8> static int launch_rows(const DecodeWork& w, int rounds, hipStream_t stream) {
    return rounds > 0 ? launch_chunks<T, D, FP8>(w, rounds, stream) : launch_line<T, D, FP8>(w, stream);
}
template <class T> static int launch_decode_as(const DecodeWork& w, int64_t D, bool eight, int rounds, hipStream_t stream) {
    if (eight) return D == 128 ? launch_rows<T, 128, true>(w, rounds, stream) : launch_rows<T, 64, true>(w, rounds, stream);
    return D == 128 ? launch_rows<T, 128, false>(w, rounds, stream) : launch_rows<T, 64, false>(w, rounds, stream);
}

int launch_paged_decode(PagedParams p, int dtype, int64_t D, bool eight, int64_t max_context, void* workspace, hipStream_t stream) {
    DecodeWork w{};
    const DecodePlan plan = plan_decode(eight, p.n_seqs, p.Hq, p.Hkv, D, max_context, p.max_q);
    w.n_col = (int)plan.n_col;
    w.n_hg = (int)plan.n_hg;
    w.per_part = (int)plan.per_part;
    w.n_wg = compute_units() * kLineWgPerCu;
    const int64_t rows = (int64_t)p.n_seqs * p.Hkv * w.n_col;
    if (rows > 0x7fffffffLL || (int64_t)p.n_seqs * p.Hkv * w.n_hg * ((max_context + 15) / 16 + 1) > 0x7fffffffLL - 65536)
        return fail(MINFER_ATTN_EINVAL, "flash_attn_paged: problem too large for one launch");
    p.part_o = (float*)workspace;
    p.part_ml = (float*)((char*)workspace + plan.o_bytes);
    w.seq_off = plan.rounds > 0 ? nullptr : (int32_t*)((char*)p.part_ml + plan.ml_bytes);
    w.p = p;
    return dtype == MINFER_ATTN_F16 ? launch_decode_as<F16>(w, D, eight, plan.rounds, stream) : launch_decode_as<BF16>(w, D, eight, plan.rounds, stream);
}

}  // namespace minfer_attn
