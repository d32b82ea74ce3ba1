// Verification of drafted tokens against the target's probabilities, from random numbers given by the caller.
//
// Row i of a sequence is the target's distribution p_i after its token i, and token i + 1, drawn from q_i by whoever drafted it, is kept while
// u_i q_i(x) < p_i(x).  The next token comes from the row of the first one that is not kept, from what p has more than q there, or from the
// last row's p where all are kept: the least j with w_0 + .. + w_j > r * (w_0 + w_1 + ..).  A kept or drawn token is then distributed as p says, whatever q is.
//
// One row of p and q per sequence is read, whatever the number of drafts: a row is cut into chunks with a workgroup each, whose sums decide which chunk
// holds the token, and that chunk alone is read again.  Memory is the floor of a batch (64 rows of 128256 with a drafter 12.6 us).  What bounds it as built is the latency of a workgroup's loads, each of
// which is waited for in front of the next (RowReader::share), and of the second launch: 17.7 us; 150 rows of 50257 bf16 13.8, floor 2.9.
//
// Which token is drawn is a comparison of sums of up to V numbers: sums are held in 64 bits.  (In 32 each of V borders between two tokens would be off by
// about 1e-7 of the total, so that of 1e5 tokens one draw in a hundred were the neighbour's; in 64 one in 1e11.)  w = p - q is a single subtraction in 64 bits.
#include <algorithm>

#include "attn_common.h"
#include "attn_host.h"
#include "attn_paged.h"

namespace minfer_attn {

constexpr int kVerifyThreads = 256, kVerifyWaves = kVerifyThreads / 64;
constexpr int kMaxChunks = kVerifyThreads;   // of a row: a thread each where they are put together
constexpr int kLeastChunk = 2048;            // elements, eight to a thread: two of its loads of fp32, one of 16 bits
constexpr int64_t kVerifyWgs = 2048;         // that the chip holds at once
// Workgroups, and bytes that each of them reads, up to which the last one of a sequence goes on (a counter per sequence, each in 64 bytes of its own: side by side, 2048 arrivals
// wait 3 us longer for one another).  Beyond, where workgroups hold their places on the chip for an answer that comes behind all those loads (one after the other, as they are), a second launch is shorter
// (us, one launch / two: 16 workgroups of 16 KiB 6.9 / 8.1, 1008 9.7 / 10.8, 1512 10.7 / 11.8, 1600 11.0 / 11.9, 2048 20.6 / 18.3; 1300 of 8 KiB 11.4 / 12.5, 1560 13.1 / 13.2,
// 1950 14.2 / 13.9; 1536 of 32 KiB 16.7 / 15.8).
constexpr int64_t kCountedWgs = 1600, kCountedBytes = 16384;
constexpr int kCounterStep = 16;
constexpr int kMostChunk = 8192;             // what is read again by one workgroup (longer only where a row would have more than kMaxChunks)

struct VerifyParams {
    const void* tokens; const int32_t* cu;
    const void* target; const void* draft;   // [T, V]; draft null: every draft has the probability one
    const float* accept_u; const float* sample_u;
    void* out; int32_t* n_accepted;
    double* sums;        // [n_seqs][chunks]
    int32_t* kept;       // [n_seqs] for the second launch
    uint32_t* done;      // zeroed counters, one per sequence, kCounterStep apart, left zero; or null: a second launch
    int64_t target_stride, draft_stride;
    int n_seqs, T, V, chunks, chunk_len;
    bool wide;           // tokens and out are 64-bit numbers
};

struct F32 {
    typedef float elem;
    static MA_DEV float value(float x) { return x; }
};
struct H16 {
    typedef _Float16 elem;
    static MA_DEV float value(_Float16 x) { return (float)x; }
};
struct B16 {
    typedef uint16_t elem;
    static MA_DEV float value(uint16_t x) { return __builtin_bit_cast(float, (uint32_t)x << 16); }
};

MA_DEV int64_t token_at(const VerifyParams& p, int64_t i) { return p.wide ? ((const int64_t*)p.tokens)[i] : (int64_t)((const int32_t*)p.tokens)[i]; }
MA_DEV void put_token(const VerifyParams& p, int64_t i, int64_t x) {
    if (p.wide) ((int64_t*)p.out)[i] = x; else ((int32_t*)p.out)[i] = (int32_t)x;
}

// The row that the next token is drawn from.
struct Row { int lo, len, kept; bool refused; int64_t draft; };   // draft: the token that was not kept
// Drafts of the sequence that are kept, a draft to a lane; every wave works it out for itself.
template <class E> MA_DEV Row row_of(const VerifyParams& p, int s) {
    const TokenRange r = token_range(const_load(p.cu + s), const_load(p.cu + s + 1), p.T);
    const int lane = threadIdx.x & 63, drafts = r.len - 1;
    Row out{r.lo, r.len, max(drafts, 0), false, 0};
    for (int base = 0; base < drafts; base += 64) {
        const int i = base + lane, at = r.lo + i;
        bool no = false;
        int64_t x = 0;
        if (i < drafts) {
            x = token_at(p, at + 1);
            no = true;
            if (x >= 0 && x < p.V) {   // (no token: nothing that the target would say)
                const double pt = (double)E::value(((const typename E::elem*)p.target)[(int64_t)at * p.target_stride + x]);
                const double qd = p.draft ? (double)E::value(((const typename E::elem*)p.draft)[(int64_t)at * p.draft_stride + x]) : 1.0;
                no = !((double)p.accept_u[at] * qd < pt);   // (exact: a product of two 24-bit numbers)
            }
        }
        const uint64_t hit = __ballot(no);
        if (hit) {
            const int first = __builtin_amdgcn_readfirstlane(__ffsll((unsigned long long)hit) - 1);
            out.kept = base + first;
            out.refused = true;
            out.draft = (int64_t)(((uint64_t)(uint32_t)lane_value((int)(uint32_t)((uint64_t)x >> 32), first) << 32) | (uint32_t)lane_value((int)(uint32_t)(uint64_t)x, first));
            break;
        }
    }
    return out;
}

// Weight of an element: what p has more than q; what is negative or no number weighs nothing.
MA_DEV double weight_of(float pt, float qd) { return fmax((double)pt - (double)qd, 0.0); }   // (fmax of NaN and 0 is 0)

// The row and what is taken from it: the draft's probabilities where a draft was not kept (of drafts without: one at the draft), nothing where all were, or where
// p has nothing more than q (whole).  Rows start anywhere; loads of 16 bytes do not mind.
template <class E> struct RowReader {
    typedef typename E::elem elem;
    static constexpr int N = 16 / (int)sizeof(elem);
    struct Piece { elem x[N]; };
    const elem* p; const elem* q;
    int64_t draft; bool refused;
    MA_DEV RowReader(const VerifyParams& v, const Row& r, bool whole = false) {
        const int64_t at = r.lo + r.kept;
        p = (const elem*)v.target + at * v.target_stride;
        refused = r.refused && !whole;
        q = v.draft && refused ? (const elem*)v.draft + at * v.draft_stride : nullptr;
        draft = r.draft;
    }
    static MA_DEV Piece load(const elem* at) {
        Piece r;
        __builtin_memcpy(&r, at, 16);
        return r;
    }
    MA_DEV float other(int i, float qd) const { return q ? qd : (refused && i == draft ? 1.f : 0.f); }
    MA_DEV double one(int i) const { return weight_of(E::value(p[i]), other(i, q ? E::value(q[i]) : 0.f)); }
    MA_DEV double of(const Piece& a, const Piece& b, int at) const {
        double sum = 0.0;
#pragma unroll
        for (int e = 0; e < N; ++e) sum += weight_of(E::value(a.x[e]), other(at + e, E::value(b.x[e])));
        return sum;
    }
    // elements lo .. hi - 1 of the row, this thread's share of them.  (Unrolled by four, but q's loads stand behind a branch, and the built code waits for p's in front of it: a round is four
    // pairs of loads one after the other.  A thread of 2048 fp32 or 4096 16-bit elements has two loads and never enters the unrolled rounds.)
    MA_DEV double share(int lo, int hi) const {
        double sum = 0.0;
        constexpr int UN = 4, STEP = kVerifyThreads * N;
        int i = lo + (int)threadIdx.x * N;
        for (; i + (UN - 1) * STEP + N <= hi; i += UN * STEP) {
            Piece a[UN], b[UN];
#pragma unroll
            for (int u = 0; u < UN; ++u) {
                a[u] = load(p + i + u * STEP);
                b[u] = q ? load(q + i + u * STEP) : a[u];
            }
#pragma unroll
            for (int u = 0; u < UN; ++u) sum += of(a[u], b[u], i + u * STEP);
        }
        for (; i + N <= hi; i += STEP) {
            const Piece a = load(p + i), b = q ? load(q + i) : a;
            sum += of(a, b, i);
        }
        for (; i < hi; ++i) sum += one(i);   // the one thread whose piece the end cuts
        return sum;
    }
};

// Inclusive prefix sum over a wave, as wave_inclusive_scan: through vector instructions, a tenth of the latency of exchanges through the LDS.
template <int CTRL, int ROW_MASK = 0xf> MA_DEV double row_exchange64(double x) {
    const uint64_t u = __builtin_bit_cast(uint64_t, x);
    const uint32_t lo = row_exchange<CTRL, ROW_MASK>((uint32_t)u), hi = row_exchange<CTRL, ROW_MASK>((uint32_t)(u >> 32));
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
MA_DEV double wave_scan(double x) {
    x += row_exchange64<0x111>(x);
    x += row_exchange64<0x112>(x);
    x += row_exchange64<0x114>(x);
    x += row_exchange64<0x118>(x);
    x += row_exchange64<0x142, 0xa>(x);
    x += row_exchange64<0x143, 0xc>(x);
    return x;
}
MA_DEV double lane_value(double x, int lane) {
    const uint64_t u = __builtin_bit_cast(uint64_t, x);
    return __builtin_bit_cast(double, (uint64_t)(uint32_t)lane_value((int)(u >> 32), lane) << 32 | (uint32_t)lane_value((int)u, lane));
}

// x over the workgroup: the sum of the threads in front, and of all.  `part` holds one entry a wave; a barrier stands in front of its next use.
struct Scan { double front, all; };
MA_DEV Scan block_scan(double x, double* part) {
    const int lane = threadIdx.x & 63, w = wave_id();
    const double incl = wave_scan(x);
    if (lane == 63) part[w] = incl;
    __syncthreads();
    Scan r{0.0, 0.0};
#pragma unroll
    for (int i = 0; i < kVerifyWaves; ++i) {
        if (i < w) r.front += part[i];
        r.all += part[i];
    }
    __syncthreads();
    const double before = __shfl_up(incl, 1);
    r.front += lane > 0 ? before : 0.0;
    return r;
}
// The least thread for which `hit`, or the greatest for which `some` where there is none (-1: neither); in every thread.
MA_DEV int first_thread(bool hit, bool some, int* part) {
    const int w = wave_id();
    const uint64_t h = __ballot(hit), o = __ballot(some);
    if ((threadIdx.x & 63) == 0) {
        part[w] = h ? w * 64 + __ffsll((unsigned long long)h) - 1 : kVerifyThreads;
        part[kVerifyWaves + w] = o ? w * 64 + 63 - __clzll((long long)o) : -1;
    }
    __syncthreads();
    int first = kVerifyThreads, last = -1;
#pragma unroll
    for (int i = 0; i < kVerifyWaves; ++i) {
        first = min(first, part[i]);
        last = max(last, part[kVerifyWaves + i]);
    }
    __syncthreads();
    return first < kVerifyThreads ? first : last;
}

MA_DEV double load_sum(const double* p) {
    return __builtin_bit_cast(double, __hip_atomic_load(reinterpret_cast<uint64_t*>(const_cast<double*>(p)), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
}
MA_DEV void store_sum(double* p, double x) {
    __hip_atomic_store(reinterpret_cast<uint64_t*>(p), __builtin_bit_cast(uint64_t, x), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// The token, from the chunks' sums (one to a thread), and what the sequence gets; the whole workgroup.
template <class E> MA_DEV void finish_row(const VerifyParams& p, int s, const Row& r, double mine, double* part, int* ipart) {
    __shared__ double front_s;
    typedef RowReader<E> Reader;
    const int tid = threadIdx.x;
    Scan of = block_scan(mine, part);
    bool whole = false;
    if (r.refused && !(of.all > 0.0)) {   // p has nothing more than q: p itself (one workgroup for all of the row; sums of probabilities that are off by their roundings)
        whole = true;
        const Reader row(p, r, true);
        for (int c = 0; c < p.chunks; ++c) {
            const double sum = block_scan(row.share(c * p.chunk_len, min((c + 1) * p.chunk_len, p.V)), part).all;
            if (tid == c) mine = sum;
        }
        of = block_scan(mine, part);
    }
    const double mark = (double)p.sample_u[s] * of.all;
    // (a thread that weighs nothing is not a hit: sums to its front and to the end of the one before are added in different orders, and a mark may lie between them)
    const int chunk = first_thread(mine > 0.0 && of.front + mine > mark, mine > 0.0, ipart);
    int64_t token = -1;   // a row that holds no probability
    if (chunk >= 0) {
        // the sum in front of the chunk, from the thread that has it
        if (tid == chunk) front_s = of.front;
        __syncthreads();
        const double front = front_s;
        const Reader row(p, r, whole);
        const int lo = chunk * p.chunk_len, hi = min(lo + p.chunk_len, p.V), per = p.chunk_len / kVerifyThreads;
        const int i0 = min(lo + tid * per, hi), i1 = min(i0 + per, hi);
        double sum = 0.0;
        int i = i0;
#pragma unroll 4
        for (; i + Reader::N <= i1; i += Reader::N) {
            const typename Reader::Piece a = Reader::load(row.p + i), b = row.q ? Reader::load(row.q + i) : a;
            sum += row.of(a, b, i);
        }
        for (; i < i1; ++i) sum += row.one(i);
        const Scan in = block_scan(sum, part);
        const int owner = first_thread(sum > 0.0 && front + in.front + sum > mark, sum > 0.0, ipart);
        if (tid == owner) front_s = front + in.front;
        __syncthreads();
        if (wave_id() == 0 && owner >= 0) {   // the owner's elements, one to a lane
            double before = front_s;
            const int lane = tid & 63, o0 = lo + owner * per, o1 = min(o0 + per, hi);
            for (int at = o0; at < o1; at += 64) {
                const double w = at + lane < o1 ? row.one(at + lane) : 0.0;
                const double incl = wave_scan(w);
                const uint64_t over = __ballot(w > 0.0 && before + incl > mark), some = __ballot(w > 0.0);
                if (some) token = at + 63 - __clzll((long long)some);
                if (over) { token = at + __ffsll((unsigned long long)over) - 1; break; }
                before += lane_value(incl, 63);
            }
        }
    }
    if (tid == 0) put_token(p, (int64_t)r.lo + r.kept, token);
    for (int i = tid; i < r.len; i += kVerifyThreads)
        if (i != r.kept) put_token(p, r.lo + i, i < r.kept ? token_at(p, r.lo + i + 1) : -1);
    if (tid == 0) p.n_accepted[s] = r.kept;
}

// grid (chunks, sequences)
template <class E> __global__ __launch_bounds__(kVerifyThreads) void verify_kernel(const VerifyParams p) {
    __shared__ double part[kVerifyWaves];
    __shared__ int ipart[2 * kVerifyWaves];
    __shared__ int last_s;
    typedef RowReader<E> Reader;
    const int tid = threadIdx.x, c = blockIdx.x, s = blockIdx.y;
    const Row r = row_of<E>(p, s);
    if (r.len == 0) {
        if (c == 0 && tid == 0) p.n_accepted[s] = 0;
        return;
    }
    const Reader row(p, r);
    const double sum = block_scan(row.share(c * p.chunk_len, min((c + 1) * p.chunk_len, p.V)), part).all;
    if (p.chunks == 1) {
        finish_row<E>(p, s, r, tid == 0 ? sum : 0.0, part, ipart);
        return;
    }
    double* const sums = p.sums + (int64_t)s * p.chunks;
    if (tid == 0) store_sum(sums + c, sum);
    if (!p.done) {
        if (c == 0 && tid == 0) p.kept[s] = r.kept;
        return;
    }
    // the sequence's last workgroup goes on (as in the attention's chunks: what crosses from one L2 to another goes past both, and a workgroup
    // counts itself when its sums have arrived)
    if (tid == 0) {
        wait_vmcnt<0>();
        const uint32_t before = __hip_atomic_fetch_add(p.done + s * kCounterStep, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        last_s = before == (uint32_t)(p.chunks - 1);
        if (last_s) __hip_atomic_store(p.done + s * kCounterStep, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (!last_s) return;
    finish_row<E>(p, s, r, tid < p.chunks ? load_sum(sums + tid) : 0.0, part, ipart);
}

// (where there are no counters) a workgroup per sequence
template <class E> __global__ __launch_bounds__(kVerifyThreads) void verify_finish_kernel(const VerifyParams p) {
    __shared__ double part[kVerifyWaves];
    __shared__ int ipart[2 * kVerifyWaves];
    const int tid = threadIdx.x, s = blockIdx.x;
    const double sum = tid < p.chunks ? p.sums[(int64_t)s * p.chunks + tid] : 0.0;   // (of a sequence without tokens nobody wrote it, and it is not used)
    const TokenRange t = token_range(const_load(p.cu + s), const_load(p.cu + s + 1), p.T);
    if (t.len == 0) return;
    Row r{t.lo, t.len, const_load(p.kept + s), false, 0};
    r.refused = r.kept < r.len - 1;
    if (r.refused) r.draft = token_at(p, (int64_t)r.lo + r.kept + 1);
    finish_row<E>(p, s, r, sum, part, ipart);
}

// Chunks of a row: as many as make kVerifyWgs workgroups, of whole rounds of loads, 2048 to 8192 elements; from the sizes alone.
struct VerifyPlan { int64_t chunks, chunk_len; size_t bytes; };
static VerifyPlan plan_verify(int64_t n_seqs, int64_t V) {
    VerifyPlan r{};
    const int64_t want = std::min<int64_t>(std::max<int64_t>((kVerifyWgs + n_seqs - 1) / n_seqs, (V + kMostChunk - 1) / kMostChunk), kMaxChunks);
    r.chunk_len = std::max<int64_t>(((V + want - 1) / want + kLeastChunk - 1) / kLeastChunk * kLeastChunk, kLeastChunk);
    r.chunks = std::max<int64_t>((V + r.chunk_len - 1) / r.chunk_len, 1);
    if (r.chunks > 1) r.bytes = (size_t)(n_seqs * r.chunks * 8 + (n_seqs * 4 + 255) / 256 * 256);
    return r;
}

template <class E> static int launch_verify(const VerifyParams& p, hipStream_t stream) {
    hipLaunchKernelGGL((verify_kernel<E>), dim3((unsigned)p.chunks, (unsigned)p.n_seqs), dim3(kVerifyThreads), 0, stream, p);
    if (int rc = check_launch("verify_kernel")) return rc;
    if (p.chunks == 1 || p.done) return MINFER_ATTN_OK;
    hipLaunchKernelGGL((verify_finish_kernel<E>), dim3((unsigned)p.n_seqs), dim3(kVerifyThreads), 0, stream, p);
    return check_launch("verify_finish_kernel");
}

}  // namespace minfer_attn

using namespace minfer_attn;

MINFER_ATTN_EXPORT size_t minfer_verify_drafts_workspace_bytes(int64_t n_seqs, int64_t V) { return n_seqs > 0 && V > 0 ? plan_verify(n_seqs, V).bytes : 0; }

MINFER_ATTN_EXPORT int minfer_verify_drafts(int prob_dtype, int token_bits, const void* tokens, const int32_t* cu_seqlens, const void* target_probs,
                                            const void* draft_probs, const float* accept_u, const float* sample_u, void* out_tokens, int32_t* n_accepted,
                                            int64_t n_seqs, int64_t T, int64_t V, int64_t target_stride, int64_t draft_stride, void* workspace,
                                            size_t workspace_bytes, void* stream_v) {
    clear_error();
    auto bad = [&](const char* what) { return fail(MINFER_ATTN_EINVAL, what); };
    if (prob_dtype != MINFER_ATTN_F32 && prob_dtype != MINFER_ATTN_F16 && prob_dtype != MINFER_ATTN_BF16)
        return bad("verify_drafts: prob_dtype must be MINFER_ATTN_F32, MINFER_ATTN_F16 or MINFER_ATTN_BF16");
    if (token_bits != 32 && token_bits != 64) return bad("verify_drafts: token_bits must be 32 or 64");
    if (n_seqs < 0 || n_seqs > 65535) return bad("verify_drafts: n_seqs must be in 0..65535");
    if (T < 0 || T > (1 << 30)) return bad("verify_drafts: T must be in 0..2^30");
    if (V <= 0 || V > (1 << 28)) return bad("verify_drafts: V must be in 1..2^28");
    if (target_stride < V || (draft_probs && draft_stride < V)) return bad("verify_drafts: rows must not overlap");
    if (n_seqs == 0) return MINFER_ATTN_OK;
    if (!cu_seqlens || !n_accepted || !sample_u) return bad("verify_drafts: cu_seqlens, sample_u and n_accepted must be non-null");
    if (T > 0 && (!tokens || !target_probs || !accept_u || !out_tokens)) return bad("verify_drafts: tokens, target_probs, accept_u and out_tokens must be non-null");
    const uintptr_t a = (uintptr_t)tokens, b = (uintptr_t)out_tokens, bytes = (uintptr_t)(T * token_bits / 8);
    if (a < b + bytes && b < a + bytes) return bad("verify_drafts: out_tokens must not be tokens: workgroups read the one while others write the other");
    const VerifyPlan plan = plan_verify(n_seqs, V);
    if (plan.bytes > 0 && (!workspace || !aligned16(workspace) || workspace_bytes < plan.bytes))
        return fail(MINFER_ATTN_EWORKSPACE, "verify_drafts: workspace too small or misaligned (see minfer_verify_drafts_workspace_bytes)");
    VerifyParams p{};
    p.tokens = tokens; p.cu = cu_seqlens; p.target = target_probs; p.draft = draft_probs;
    p.accept_u = accept_u; p.sample_u = sample_u; p.out = out_tokens; p.n_accepted = n_accepted;
    p.target_stride = target_stride; p.draft_stride = draft_stride;
    p.n_seqs = (int)n_seqs; p.T = (int)T; p.V = (int)V; p.chunks = (int)plan.chunks; p.chunk_len = (int)plan.chunk_len;
    p.wide = token_bits == 64;
    p.sums = (double*)workspace;
    p.kept = (int32_t*)((char*)workspace + n_seqs * plan.chunks * 8);
    hipStream_t stream = (hipStream_t)stream_v;
    const int64_t chunk_bytes = plan.chunk_len * (prob_dtype == MINFER_ATTN_F32 ? 4 : 2) * (draft_probs ? 2 : 1);
    if (plan.chunks > 1 && n_seqs * plan.chunks <= kCountedWgs && n_seqs * kCounterStep <= kStreamCounters && chunk_bytes <= kCountedBytes) p.done = stream_counters(stream);
    if (prob_dtype == MINFER_ATTN_F32) return launch_verify<F32>(p, stream);
    return prob_dtype == MINFER_ATTN_F16 ? launch_verify<H16>(p, stream) : launch_verify<B16>(p, stream);
}
