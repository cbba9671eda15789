// kv4_step_kernel.cuh -- attention of a few rows per sequence over the
// block-scaled FP4 cache (a generation step, a draft that is checked).
//
// For row r (a token's head) of a KV head's group, over the tokens j it sees:
//   s_rj = softmax_scale g_k q_r . k_j,   o_r = g_v sum_j e^{s_rj} v_j / sum_j e^{s_rj}
// with k_j = e2m1 * e4m3, an FP16 value, and FP32 sums.  One pass over the
// cache with a running maximum m and sum l.
//
// What bounds it: 18 D / 16 bytes a token and KV head come from memory, and
// an SM has about six cycles for the 144 bytes of D = 128.  In those it must
// turn 256 codes into FP16 and multiply them, so instructions count (issue slots
// are 60% full, and the conversions and half-precision products, two cycles
// each, are what the warps wait for beside fixed latencies):
//   - S^T = K Q^T and O^T = V^T P^T put tokens (d) on the 16-row side of
//     mma.m16n8k16 and the rows r on its 8 columns: eight rows, the usual size
//     of a group, cost half of what padding them to 16 would.  (tcgen05.mma
//     has the rate to spare, but wants the codes decoded into shared or tensor
//     memory first, which costs more than the product here.)
//   - operands are decoded in registers, in fragment order: the order of d in
//     K Q^T is free as long as Q follows, so a lane reads a whole 32 (D = 64:
//     16) values of a token with one load and each byte is one fragment
//     register.  V^T wants two tokens in a register, so the nibbles of two
//     tokens are interleaved before they are converted (two operations for
//     eight values), not the FP16 values after (four).
//   - P^T's fragment is S^T's, transposed in 8 x 8 blocks: movmatrix.
//   - the maximum is moved only when a score passes it by almost 2^16, and is
//     then set 2^6 below the largest score: P stays inside FP16, and the
//     reductions over lanes are rare.
// P is rounded to FP16: by 2^-11 of itself down to 2^-20 of the row's largest
// (P's largest is 2^6 at least), below that, where FP16 is subnormal, by up to
// 2^-31 of the largest.  So where a row's weight lies on a few tokens of no value
// the sum of the others is good to 1% while they are above 2^-24; with P at 1 at
// most it was off by 13% at 2^-22 and all of it was lost at 2^-26.
// l is summed from the FP32 values.
//
// BF16 queries are scaled per row by a power of two to at most 2^15 and taken
// as FP16: exact for values within 2^-28 of the row's largest, and off by at
// most 2^-39 of it below.  FP32 sums do not resolve that where the largest meets
// a key that is not zero; where it meets only zeros, queries below 2^-40 of it
// are lost from the scores.
//
// Split: the (sequence, KV head) units' chunks are laid end to end, and each
// CTA takes an equal run of them, so a batch of any lengths loads all SMs
// alike.  A run's ends inside a unit leave partial results (o, m, l) in the
// workspace for k_kv4_join.  Short sequences need no such plan: a cluster of
// up to eight CTAs shares a unit and joins through distributed shared memory,
// in one launch.  Within a CTA one warp looks pages up and issues
// the bulk copies, a whole tile of 256 or 384 tokens by its lanes at once, and
// goes on into the next unit while the other warps compute, each on its own 32
// tokens of a tile with its own o, m, l, merged once per unit in a fixed order.
//
// Measured in a CUDA graph, 8 KV heads of 128, one row: 4 sequences of 65536
// tokens, 64 heads, 68.0 us (4.44 TB/s, 0.68 of a copy; about 10 us of it are the
// start and the ends of the runs, the rest goes at 0.72); 32 of 4000, 32 heads,
// 42 us; 1 of 1000 7.5 us.  20 packed rows (three tiles of 8), 8 of 10000: 48 us.
#pragma once

#include "kv4_cache_kernel.cuh"

namespace tb {

struct Kv4Attn {
    Kv4Cache cache;
    Kv4Rows rows;
    const void* q;
    void* out;
    float* lse;                    // may be null
    long long q_stride, out_stride;
    int q_heads, group;
    float scale_log2;              // softmax_scale * k_scale * log2(e)
    int window, sinks;
    float* ws;                     // partial results
    int cluster;                   // step kernel: CTAs of a cluster that shares a unit; 0: runs of chunks
    int runs;                      // CTAs that share all chunks (cluster 0)
    int min_run;                   // chunks a CTA should have at least
    int step_rows;                 // packed rows that the step kernel takes; sequences with more are the prompt kernel's
    float* prompt_ws;
    int* ticket;                   // counter of the prompt kernel's items, set to 0 by the step kernel
    int prompt_tiles;              // tiles of 256 packed rows of a sequence at most
    int prompt_splits;             // CTAs that share a prompt unit's tokens
    int prompt_units;              // sequences * KV heads * prompt_tiles
};

// Bit of the device error word: a sequence has more rows than max_rows.
enum : int { kErrRows = 4 };

constexpr int kStepChunk = 32;     // tokens of a warp's share of a tile
// A row's maximum before it has seen a score: finite, so that a hidden score less
// it is -inf and not NaN, and so low that every score passes it (a difference that
// overflows does too).
constexpr float kNoMax = -3.402823466e38f;
// In log2 units: a score that passes the row's m by more than kPMost moves it, to
// kPSet below the largest score.  P is at most 2^15.9, below FP16's 65504, and its
// largest at 2^6 when m has moved: higher, small weights keep more bits, but m
// moves more often.  The prompt kernel's windowed chunks of 1500 rows (32 heads of
// 64, window 2048) and prompt of 4096 tokens, a call: kPSet 4 151, 177 us; 5 160,
// 177; 6 171, 178; 7 190, 181; 7 with kPMost 15 212, 190.
constexpr float kPMost = 15.9f, kPSet = 6.0f;
constexpr int kStepRowsMost = 32;  // packed rows of a (sequence, KV head)

// NT tiles of eight rows.  Eight computing warps, and twelve for two tiles,
// where one CTA is all that an SM holds and eight leave its pipes idle (16 rows,
// 8 sequences of 10000 tokens, 8 KV heads of 128: 39.4 us with twelve, 41.9 with
// eight).
template <int D_, int NT_>
struct StepCfg {
    static constexpr int D = D_, NT = NT_;
    static constexpr int WARPS = NT == 2 ? 12 : 8;        // that compute
    static constexpr int THREADS = 32 * (WARPS + 4);      // the loading warp's group of four: three of them idle
    static constexpr int TILE = kStepChunk * WARPS;       // tokens
    static constexpr int GRAN_MOST = WARPS == 8 ? 8 : 7;  // log2 of a power of two that divides the tile
    static constexpr int ROWS = 8 * NT;
    static constexpr int TOKEN_BYTES = D / 2 + D / 16;  // of K or of V
    static constexpr int STAGE = TILE * TOKEN_BYTES * 2;
    static constexpr int ST = D == 64 ? 3 : 2;
    static constexpr int OFF_MERGE = ST * STAGE;
    static constexpr int OFF_Q = OFF_MERGE + WARPS * ROWS * (D + 4) * 4;
    static constexpr int OFF_ML = OFF_Q + NT * (D / 16) * 32 * 8;
    static constexpr int OFF_SCALE = OFF_ML + WARPS * ROWS * 2 * 4;
    static constexpr int OFF_INFO = OFF_SCALE + ROWS * 4;
    static constexpr int OFF_BAR = OFF_INFO + ST * WARPS * 8;
    static constexpr int OFF_SUMS = OFF_BAR + 2 * ST * 8;
    static constexpr int SMEM = OFF_SUMS + (THREADS / 32 + 3) * 8;
    // Registers a thread: at launch, then of the loading group and of the
    // computing warps.  The split never asks for more than the launch held.
    static constexpr int CTAS = NT == 1 ? 2 : 1;
    static constexpr int REGS = NT == 1 ? 80 : NT == 2 ? 128 : 168;
    static constexpr int REGS_LOAD = NT >= 3 ? 40 : 32, REGS_COMPUTE = NT == 1 ? 104 : NT == 2 ? 160 : 232;
    static_assert(128 * REGS_LOAD + 32 * WARPS * REGS_COMPUTE <= THREADS * REGS, "registers of the launch");
    static_assert(SMEM <= 227 * 1024 / CTAS - 1024 * (CTAS - 1), "shared memory");
    static constexpr int SLOT = ROWS * (D + 2);  // floats of a partial result: o [ROWS x D], m, l
};

// A partial result belongs to CTA `run`: slot 0 for the unit that began in an
// earlier CTA's run, slot 1 for one that begins here and goes on.  The slots
// follow a StepLink of each run.
template <class C>
__device__ __forceinline__ float* step_slot(const Kv4Attn& a, int run, int slot) {
    return a.ws + static_cast<size_t>(a.runs) * 4 + (static_cast<size_t>(run) * 2 + slot) * C::SLOT;
}

// What a run leaves for k_kv4_join: the last run of the unit that begins in it
// and goes on (-1: none does), and where the unit's rows belong.
struct alignas(16) StepLink {
    int last, first, rows, head;
};
__device__ __forceinline__ StepLink* step_link(const Kv4Attn& a, int run) {
    return reinterpret_cast<StepLink*>(a.ws) + run;
}

__device__ __forceinline__ void bulk_load(void* smem_dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
            smem_addr(smem_dst)),
        "l"(reinterpret_cast<uint64_t>(src)), "r"(bytes), "r"(smem_addr(bar))
        : "memory");
}

// Four floats of a CTA's shared memory, by shared::cluster address.
__device__ __forceinline__ float4 ld_cluster4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}

// Hand registers back to the CTA's pool, or take more of them (whole groups
// of four warps; taking waits until the pool has them).
template <int N>
__device__ __forceinline__ void reg_dec() {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void reg_inc() {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}

__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                          uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t movmatrix(uint32_t x) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}

// 2^k for -126 <= k <= 127.
__device__ __forceinline__ float exp2i(int k) { return __uint_as_float(static_cast<uint32_t>(k + 127) << 23); }

__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
    const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
}

__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
    const __half2 r = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&r);
}

// A row's factor from products to scores, last of all steps: not zero, which
// would make NaN of a hidden score's -inf, and not infinite, which would of a
// product that is zero.
__device__ __forceinline__ float kv4_row_factor(float scale) { return fminf(fmaxf(scale, 1e-37f), 3e38f); }

// log2 of the tokens of a chunk, in which sequences are split: a page's, but 32
// at least (a warp's share) and `most` at most (it divides a tile).
TB_KV4_HD int step_gran(int page_shift, int most) {
    return page_shift < 5 ? 5 : page_shift > most ? most : page_shift;
}

// Adds a partial result (u, li, mi) to (v, l, top).  A part that saw nothing
// of the row has kNoMax, l = 0 and o = 0, or NaN, which stays.
__device__ __forceinline__ void kv4_merge(float& top, float& l, float4& v, float mi, float li, float4 u) {
    const float mt = fmaxf(top, mi);
    const float f = ex2(top - mt), fi = ex2(mi - mt);
    l = l * f + li * fi;
    v.x = v.x * f + u.x * fi;
    v.y = v.y * f + u.y * fi;
    v.z = v.z * f + u.z * fi;
    v.w = v.w * f + u.w * fi;
    top = mt;
}

// Chunks of sequence b's tokens for each KV head; 0 where it has no rows or
// is not the step kernel's.
struct StepSeq {
    Kv4Seq q;
    Kv4Span span;
    int chunks;
    __device__ __forceinline__ long long total(int heads) const { return static_cast<long long>(heads) * chunks; }
};

template <class C>
__device__ __forceinline__ StepSeq step_seq(const Kv4Attn& a, int b) {
    StepSeq s;
    s.q = kv4_rows_seq(a.rows, a.cache.page_shift, a.rows.cu[b], a.rows.cu[b + 1], a.rows.lens[b]);
    s.span = kv4_span(s.q.pos0, s.q.pos0 + s.q.n - 1, s.q.len, a.window, a.sinks, step_gran(a.cache.page_shift, C::GRAN_MOST));
    const long long rows = static_cast<long long>(s.q.n) * a.group;
    s.chunks = rows > 0 && rows <= a.step_rows ? kv4_span_chunks(s.span) : 0;
    return s;
}

// Reports a sequence with rows outside the caller's, and one that neither
// kernel takes: more rows than max_rows said.
__device__ __forceinline__ void step_report(const Kv4Attn& a, const StepSeq& s) {
    if (s.q.cut) atomicOr(&g_tb_device_error, kErrPage);
    if (a.prompt_tiles == 0 && static_cast<long long>(s.q.n) * a.group > a.step_rows)
        atomicOr(&g_tb_device_error, kErrRows);
}

// Sum of `v` over the CTA's threads, in every thread; `sums` has a slot per warp.
__device__ __forceinline__ long long block_sum(long long v, long long* sums) {
    for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, off);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sums[threadIdx.x / 32] = v;
    __syncthreads();
    long long t = 0;
    for (int w = 0; w < static_cast<int>(blockDim.x / 32); ++w) t += sums[w];
    return t;
}

// How many CTAs share `total` chunks.
__device__ __forceinline__ int step_runs(const Kv4Attn& a, long long total) {
    const long long most = total / a.min_run;
    return static_cast<int>(most < 1 ? 1 : most < a.runs ? most : a.runs);
}

__device__ __forceinline__ long long run_start(long long total, int runs, int i) { return total * i / runs; }

// Four values d..d+3 of packed row `row` (token row / group of the sequence,
// head row % group of the KV head's group) from its unnormalised sums, with
// the maximum `top` (log2 units) and sum l; d = 0 also writes the row's lse.
template <bool BF16, int D>
__device__ __forceinline__ void kv4_store_row(const Kv4Attn& a, int first, int row, int head, int d, float4 v,
                                              float top, float l) {
    const int i = row / a.group, h = head * a.group + row - i * a.group;
    const float f = l == 0.0f ? 0.0f : a.cache.v_scale / l;
    const float x[4] = {l == 0.0f ? 0.0f : v.x * f, l == 0.0f ? 0.0f : v.y * f, l == 0.0f ? 0.0f : v.z * f,
                        l == 0.0f ? 0.0f : v.w * f};
    uint2 u;
    if constexpr (BF16) {
        const __nv_bfloat162 p = __floats2bfloat162_rn(x[0], x[1]), q = __floats2bfloat162_rn(x[2], x[3]);
        u = make_uint2(*reinterpret_cast<const uint32_t*>(&p), *reinterpret_cast<const uint32_t*>(&q));
    } else {
        u = make_uint2(pack_half2(x[0], x[1]), pack_half2(x[2], x[3]));
    }
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + static_cast<long long>(first + i) * a.out_stride +
                              static_cast<long long>(h) * D + d) = u;
    if (d == 0 && a.lse != nullptr)
        a.lse[static_cast<long long>(first + i) * a.q_heads + h] =
            l == 0.0f ? -INFINITY : (top + log2f(l)) * 0.6931471805599453f;
}

template <class C, bool BF16>
__global__ void __launch_bounds__(C::THREADS, C::CTAS) k_kv4_step(const Kv4Attn a) {
    constexpr int D = C::D, NT = C::NT, ROWS = C::ROWS, ST = C::ST, WARPS = C::WARPS;
    constexpr int KS = D / 16;   // k-steps of K Q^T
    constexpr int MT = D / 16;   // 16-row tiles of V^T
    extern __shared__ __align__(128) uint8_t smem[];
    float* merge = reinterpret_cast<float*>(smem + C::OFF_MERGE);
    uint2* qfrag = reinterpret_cast<uint2*>(smem + C::OFF_Q);
    float* sm_m = reinterpret_cast<float*>(smem + C::OFF_ML);
    float* sm_l = sm_m + WARPS * ROWS;
    float* sm_scale = reinterpret_cast<float*>(smem + C::OFF_SCALE);
    int2* info = reinterpret_cast<int2*>(smem + C::OFF_INFO);  // per stage and warp: first token, flags
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);
    uint64_t* empty = full + ST;
    long long* sums = reinterpret_cast<long long*>(smem + C::OFF_SUMS);  // one per warp, then the result
    volatile int* abort = reinterpret_cast<volatile int*>(sums + C::THREADS / 32 + 2);

    volatile int* failed = abort + 1;  // by a computing warp, before its second barrier of a unit

    if (blockIdx.x == 0 && threadIdx.x == 0 && a.prompt_tiles > 0) *a.ticket = 0;
    grid_dep_launch_dependents();  // what comes next waits for this grid's end
    const int tid = threadIdx.x, warp = tid / 32, lane = tid & 31;
    const int g = lane >> 2, c = lane & 3;
    if (tid == 0) {
        for (int i = 0; i < ST; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], WARPS);
        }
        fence_barrier_init();
        *abort = 0;
        *failed = 0;
    }
    __syncthreads();

    // This CTA's run of chunks: sequence b, offset `off` in it, `left` chunks.
    int b = 0;
    long long off = 0, left = 0;
    long long end = 0, all_chunks = 0;  // of this run in all chunks laid end to end; their number
    int all_runs = 0;
    const int my_run = blockIdx.x;
    if (a.cluster) {
        const int unit = blockIdx.x / a.cluster, rank = blockIdx.x - unit * a.cluster;
        b = unit / a.cache.heads;
        const StepSeq s = step_seq<C>(a, b);
        if (tid == 0) step_report(a, s);
        if (s.chunks == 0) return;  // every CTA of the cluster
        const int from = static_cast<int>(run_start(s.chunks, a.cluster, rank));
        off = static_cast<long long>(unit - b * a.cache.heads) * s.chunks + from;
        left = run_start(s.chunks, a.cluster, rank + 1) - from;
    } else {
        // The chunks of all sequences and of those before each one: a thread
        // takes the sequences tid, tid + 384, ...
        constexpr int kWarps = C::THREADS / 32;
        long long mine = 0, sum = 0;
        for (int i = tid; i < a.rows.batch; i += C::THREADS) {
            const StepSeq s = step_seq<C>(a, i);
            if (my_run == 0) step_report(a, s);
            const long long w = s.total(a.cache.heads);
            if (i == tid) mine = w;
            sum += w;
        }
        const long long total = block_sum(sum, sums);
        const int runs = step_runs(a, total);
        const long long from = run_start(total, runs, my_run);
        left = my_run < runs ? run_start(total, runs, my_run + 1) - from : 0;
        if (tid == 0) {
            // The unit that the run ends in, if it goes on, is the next run's too.
            *step_link(a, my_run) = StepLink{-1, 0, 0, 0};
        }
        if (left <= 0) return;
        end = from + left;
        all_chunks = total;
        all_runs = runs;
        long long before = 0;
        for (int b0 = 0; b0 < a.rows.batch && before <= from; b0 += C::THREADS) {
            const int i = b0 + tid;
            const long long w = b0 == 0 ? mine : i < a.rows.batch ? step_seq<C>(a, i).total(a.cache.heads) : 0;
            long long upto = w;  // inclusive sum over the CTA's threads
            for (int d = 1; d < 32; d <<= 1) {
                const long long o = __shfl_up_sync(0xFFFFFFFFu, upto, d);
                if (lane >= d) upto += o;
            }
            __syncthreads();
            if (lane == 31) sums[warp] = upto;
            __syncthreads();
            long long all = 0;
            for (int k = 0; k < kWarps; ++k) {
                if (k < warp) upto += sums[k];
                all += sums[k];
            }
            const long long lo = before + upto - w;
            if (w > 0 && from >= lo && from < lo + w) {
                sums[kWarps] = i;
                sums[kWarps + 1] = from - lo;
            }
            before += all;
        }
        __syncthreads();
        b = static_cast<int>(sums[kWarps]);
        off = sums[kWarps + 1];
    }

    // Chunk geometry.  A stage holds a tile of tokens as whole chunks; a chunk
    // is a page's block of this head as it lies in the cache, two of them for
    // 16-token pages, or some tokens of a larger page.
    const int shift = a.cache.page_shift, gs = step_gran(shift, C::GRAN_MOST);
    const uint32_t gran = 1u << gs;
    const int per_tile = C::TILE >> gs;
    const uint32_t codes = kv4_codes_bytes(a.cache), scales = kv4_scales_bytes(a.cache);
    const uint32_t block_tokens = shift == 4 ? 16u : gran;  // contiguous in the stage: Kc, Ks, Vc, Vs
    const uint32_t at_ks = block_tokens * (D / 2), at_vc = at_ks + block_tokens * (D / 16),
                   at_vs = at_vc + block_tokens * (D / 2), block_bytes = block_tokens * C::TOKEN_BYTES * 2;

    int stage = 0;
    uint32_t phase = 0;
    if (warp >= WARPS) {
        reg_dec<C::REGS_LOAD>();
        if (warp > WARPS) return;
        // ---- the loading warp: lane i looks after tokens 16 i .. + 15 of a tile ----
        const int sub = lane * 16;                       // place in the tile
        const int entry = sub >> gs;                     // its chunk of the tile
        const bool leads = lane < 2 * WARPS && (sub & static_cast<int>(block_tokens - 1)) == 0;  // first of a block
        uint32_t filled = 0;
        while (left > 0 && b < a.rows.batch) {
            const StepSeq s = step_seq<C>(a, b);
            if (off >= s.total(a.cache.heads)) {
                off -= s.total(a.cache.heads);
                ++b;
                continue;
            }
            const int head = static_cast<int>(off / s.chunks);
            const int c0 = static_cast<int>(off - static_cast<long long>(head) * s.chunks);
            const int c1 = left < s.chunks - c0 ? c0 + static_cast<int>(left) : s.chunks;
            left -= c1 - c0;
            off += c1 - c0;
            if (lane == 0 && s.q.bad) atomicOr(&g_tb_device_error, kErrPage);
            const int* table = a.rows.table + static_cast<size_t>(b) * a.rows.width;
            const uint8_t* blocks = a.cache.data + static_cast<size_t>(head) * kv4_head_bytes(a.cache);
            // A chunk at token tok0 is open (every row sees all of it) if it ends
            // by `open_end` and starts by `open_low` or ends in the sinks.
            const int last_pos = s.q.pos0 + s.q.n - 1;
            const int open_end = min(s.q.pos0 + 1, s.q.len);
            // Pages out of every row's sight may be gone.
            const int oldest = a.window > 0 && s.q.pos0 >= a.window ? s.q.pos0 - a.window + 1 : 0;
            const int open_low = a.window > 0 && last_pos >= a.window ? last_pos - a.window + 1 : 0;
            // Token and page number of this lane's granule of the tile at chunk q.
            auto look = [&](int q, int& tok, int& page) {
                tok = -1;
                page = -1;
                if (lane < 2 * WARPS && q + entry < c1) {
                    tok = (kv4_span_chunk(s.span, q + entry) << gs) + (sub & static_cast<int>(gran - 1));
                    if (tok < s.q.len) page = table[tok >> shift];
                }
            };
            int tok, page;
            look(c0, tok, page);
            for (int q = c0; q < c1; q += per_tile) {
                if (!__all_sync(0xFFFFFFFFu, filled < ST || mbar_wait(&empty[stage], phase ^ 1u, abort))) break;
                const bool inside = tok >= 0 && tok < s.q.len;
                const bool ok = inside && kv4_page_ok(a.cache, page);
                if (inside && !ok && (tok + 16 > oldest || tok < a.sinks)) atomicOr(&g_tb_device_error, kErrPage);
                const uint32_t have = __ballot_sync(0xFFFFFFFFu, ok);
                const uint32_t copies = __ballot_sync(0xFFFFFFFFu, ok && leads);
                if (lane < 2 * WARPS && (lane & 1) == 0) {
                    const uint32_t two = (have >> lane) & 3u;
                    const bool open = two == 3u && tok + kStepChunk <= open_end &&
                                      (tok >= open_low || tok + kStepChunk <= a.sinks);
                    info[stage * WARPS + lane / 2] = make_int2(tok, static_cast<int>(two | (open ? 4u : 0u)));
                }
                __syncwarp();
                if (lane == 0) mbar_arrive_expect_tx(&full[stage], __popc(copies) * block_bytes);
                __syncwarp();
                uint8_t* dst = smem + stage * C::STAGE + (sub / static_cast<int>(block_tokens)) * block_bytes;
                if (shift <= gs) {
                    if (ok && leads)
                        bulk_load(dst, blocks + static_cast<unsigned long long>(static_cast<uint32_t>(page)) * a.cache.page_stride,
                                  block_bytes, &full[stage]);
                } else if (ok && leads) {  // a chunk of a larger page, part by part
                    const uint32_t place = static_cast<uint32_t>(tok) & ((1u << shift) - 1u);
                    const uint8_t* src =
                        blocks + static_cast<unsigned long long>(static_cast<uint32_t>(page)) * a.cache.page_stride;
                    bulk_load(dst, src + place * (D / 2), at_ks, &full[stage]);
                    bulk_load(dst + at_ks, src + codes + place * (D / 16), at_vc - at_ks, &full[stage]);
                    src += codes + scales;
                    bulk_load(dst + at_vc, src + place * (D / 2), at_ks, &full[stage]);
                    bulk_load(dst + at_vs, src + codes + place * (D / 16), at_vc - at_ks, &full[stage]);
                }
                __syncwarp();
                ++filled;
                if (++stage == ST) stage = 0, phase ^= 1u;
                if (q + per_tile < c1) look(q + per_tile, tok, page);
            }
            if (__any_sync(0xFFFFFFFFu, *abort)) break;
        }
        if (*abort)  // copies in flight end before the CTA does
            for (int i = 0; i < ST && filled > 0; ++i, --filled) {
                if (--stage < 0) stage = ST - 1, phase ^= 1u;
                mbar_wait_drain(&full[stage], phase);
            }
        return;
    }

    // ---- the computing warps: 32 tokens of a tile each ------------------------------------
    reg_inc<C::REGS_COMPUTE>();
    // Where the warp's tokens lie in a stage; tokens 16..31 follow 16 places on, or in the next block.
    const uint32_t in_block = (warp * kStepChunk) & (block_tokens - 1u);
    const uint32_t block0 = (warp * kStepChunk) / block_tokens * block_bytes;
    const uint32_t half_step = shift == 4 ? block_bytes : 16u * (D / 2), half_step_s = shift == 4 ? block_bytes : 16u * (D / 16);
    const int tg = g ^ ((g >> 1) & 1);
    // Row g of a 16-token tile is token g ^ (g >> 1 & 1): neighbouring lanes of
    // the loads of K and of V then fall into different banks.
    const uint32_t k_codes = block0 + in_block * (D / 2) + tg * (D / 2) + c * (D / 8);
    const uint32_t k_scales = block0 + at_ks + in_block * (D / 16) + tg * (D / 16) + c * (D / 64);
    const uint32_t ta = static_cast<uint32_t>((2 * c) ^ (c & 1));  // V: tokens ta, ta ^ 1, and 8 on
    const uint32_t v_codes = block0 + at_vc + (in_block + ta) * (D / 2) + g * (D / 16);
    const uint32_t v_scales = block0 + at_vs + (in_block + ta) * (D / 16) + (g * (D / 16)) / 8;
    const int v_pair = ta & 1u ? -1 : 1;  // from token ta to ta ^ 1

    // A CTA of a cluster has one pass, with or without chunks.
    for (bool once = a.cluster != 0; (once || left > 0) && b < a.rows.batch; once = false) {
        const StepSeq s = step_seq<C>(a, b);
        if (off >= s.total(a.cache.heads) && left > 0) {
            off -= s.total(a.cache.heads);
            ++b;
            continue;
        }
        const int head = a.cluster ? blockIdx.x / a.cluster - b * a.cache.heads : static_cast<int>(off / s.chunks);
        const int c0 = static_cast<int>(off - static_cast<long long>(head) * s.chunks);
        const int c1 = left < s.chunks - c0 ? c0 + static_cast<int>(left) : s.chunks;
        const int row_count = s.q.n * a.group;  // at most ROWS
        left -= c1 - c0;
        off += c1 - c0;

        // Queries in fragment order: lane (g, c) of k-step ks holds, for row
        // g, the values d = (D/4) c + 4 ks .. + 3, each pair swapped as the
        // converter leaves a byte's two codes.
        for (int r = warp; r < ROWS; r += WARPS) {
            uint2 v = make_uint2(0u, 0u);
            // The factor is taken positive, its sign into q: the largest product
            // is the largest score.
            float scale = fabsf(a.scale_log2);
            const uint32_t sign = a.scale_log2 < 0.0f ? 0x80008000u : 0u;
            if (r < row_count) {
                const int i = r / a.group;
                const long long at = (s.q.first + i) * a.q_stride +
                                     static_cast<long long>(head * a.group + r - i * a.group) * D + 4 * lane;
                if (lane < D / 4) v = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(a.q) + at);
                if constexpr (BF16) {
                    // Exponent of the row's largest value -> 2^k that brings it to [2^14, 2^15),
                    // in two factors (k passes 127 for the smallest rows).  Where it is infinity or
                    // NaN all scores are, whatever the others are: they only have to stay finite.
                    uint32_t e = max(max((v.x >> 7) & 0xFFu, (v.x >> 23) & 0xFFu),
                                     max((v.y >> 7) & 0xFFu, (v.y >> 23) & 0xFFu));
                    e = __reduce_max_sync(0xFFFFFFFFu, e);
                    const int k = e == 255u ? -113 : 141 - static_cast<int>(e), k1 = k > 120 ? 120 : k, k2 = k - k1;
                    const float up = exp2i(k1), up2 = exp2i(k2);
                    scale = (scale * exp2i(-k1)) * exp2i(-k2);
                    v.x = pack_half2(__uint_as_float(v.x << 16) * up * up2, __uint_as_float(v.x & 0xFFFF0000u) * up * up2);
                    v.y = pack_half2(__uint_as_float(v.y << 16) * up * up2, __uint_as_float(v.y & 0xFFFF0000u) * up * up2);
                }
            }
            v.x ^= sign;
            v.y ^= sign;
            if (lane < D / 4) {
                const int ks = lane % KS, cc = lane / KS;
                qfrag[((r / 8) * KS + ks) * 32 + (r % 8) * 4 + cc] =
                    make_uint2(prmt(v.x, 0u, 0x1032u), prmt(v.y, 0u, 0x1032u));
            }
            if (lane == 0) sm_scale[r] = kv4_row_factor(scale);
        }
        named_bar_sync(1, 32 * WARPS);

        float sf[NT][2];  // score -> log2 units, of rows 8 nt + 2c, + 1
        float m[NT][2], l[NT][2];
        float o[MT][NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                sf[nt][e] = sm_scale[8 * nt + 2 * c + e];
                m[nt][e] = kNoMax;
                l[nt][e] = 0.0f;
            }
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[mt][nt][e] = 0.0f;

        for (int q = c0; q < c1; q += per_tile) {
            if (!__all_sync(0xFFFFFFFFu, mbar_wait(&full[stage], phase, abort))) {
                *failed = 1;
                break;
            }
            const int2 what = info[stage * WARPS + warp];
            const int tok0 = what.x;
            const uint32_t have = what.y & 3u;
            const bool open = what.y & 4;
            const uint32_t base = smem_addr(smem) + stage * C::STAGE;
            uint64_t* done = &empty[stage];
            if (++stage == ST) stage = 0, phase ^= 1u;
            if (have == 0u) {  // nothing of this warp's share exists
                __syncwarp();
                if (lane == 0) mbar_arrive(done);
                continue;
            }

            // S^T = K Q^T of two times 16 tokens.
            float sc[2][NT][4];
            {
                uint32_t ka[2][D / 32], kc[2][D / 32];  // codes of rows g and g + 8
                uint32_t sa[2][D / 64], sd[2][D / 64];  // their scales, doubled
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    const uint32_t kb = base + k_codes + t * half_step, sb = base + k_scales + t * half_step_s;
                    if constexpr (D == 128) {
                        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                                     : "=r"(ka[t][0]), "=r"(ka[t][1]), "=r"(ka[t][2]), "=r"(ka[t][3]) : "r"(kb));
                        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                                     : "=r"(kc[t][0]), "=r"(kc[t][1]), "=r"(kc[t][2]), "=r"(kc[t][3])
                                     : "r"(kb + 8 * (D / 2)));
                        uint16_t x, y;
                        asm volatile("ld.shared.u16 %0, [%1];" : "=h"(x) : "r"(sb));
                        asm volatile("ld.shared.u16 %0, [%1];" : "=h"(y) : "r"(sb + 8 * (D / 16)));
                        const uint32_t xx = cvt_e4m3x2(x), yy = cvt_e4m3x2(y);
                        sa[t][0] = prmt(xx, 0u, 0x1010u); sa[t][1] = prmt(xx, 0u, 0x3232u);
                        sd[t][0] = prmt(yy, 0u, 0x1010u); sd[t][1] = prmt(yy, 0u, 0x3232u);
                    } else {
                        asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(ka[t][0]), "=r"(ka[t][1]) : "r"(kb));
                        asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];"
                                     : "=r"(kc[t][0]), "=r"(kc[t][1]) : "r"(kb + 8 * (D / 2)));
                        uint32_t x, y;
                        asm volatile("ld.shared.u8 %0, [%1];" : "=r"(x) : "r"(sb));
                        asm volatile("ld.shared.u8 %0, [%1];" : "=r"(y) : "r"(sb + 8 * (D / 16)));
                        sa[t][0] = cvt_e4m3x2(static_cast<uint16_t>(x | (x << 8)));
                        sd[t][0] = cvt_e4m3x2(static_cast<uint16_t>(y | (y << 8)));
                    }
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int e = 0; e < 4; ++e) sc[t][nt][e] = 0.0f;
                }
#pragma unroll
                for (int w = 0; w < D / 32; ++w) {
                    uint32_t fa[2][4], fc[2][4];
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        cvt_e2m1x2_x4(ka[t][w], fa[t]);
                        cvt_e2m1x2_x4(kc[t][w], fc[t]);
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            fa[t][j] = hmul2(fa[t][j], sa[t][w / 2]);
                            fc[t][j] = hmul2(fc[t][j], sd[t][w / 2]);
                        }
                    }
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            const uint2 qf = qfrag[(nt * KS + 2 * w + h) * 32 + lane];
#pragma unroll
                            for (int t = 0; t < 2; ++t)
                                mma_16816(sc[t][nt], fa[t][2 * h], fc[t][2 * h], fa[t][2 * h + 1], fc[t][2 * h + 1], qf.x,
                                          qf.y);
                        }
                }
            }

            if (__builtin_expect(!open, 0)) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int pos = s.q.pos0 + (8 * nt + 2 * c + e) / a.group;
#pragma unroll
                        for (int t = 0; t < 2; ++t)
#pragma unroll
                            for (int hi = 0; hi < 2; ++hi) {
                                const int tok = tok0 + 16 * t + 8 * hi + tg;
                                if (!((have >> t) & 1u) || tok >= s.q.len || !kv4_sees(pos, tok, a.window, a.sinks))
                                    sc[t][nt][2 * hi + e] = -INFINITY;
                            }
                    }
            }
            // In log2 units a score is s f - m; a row whose largest passes kPMost moves its m.
            bool past = false;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    past |= fmaf(fmaxf(fmaxf(sc[0][nt][e], sc[0][nt][e + 2]), fmaxf(sc[1][nt][e], sc[1][nt][e + 2])),
                                 sf[nt][e], -m[nt][e]) > kPMost;
            if (__builtin_expect(__any_sync(0xFFFFFFFFu, past), 0)) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float y = fmaxf(fmaxf(sc[0][nt][e], sc[0][nt][e + 2]), fmaxf(sc[1][nt][e], sc[1][nt][e + 2]));
#pragma unroll
                        for (int d = 4; d < 32; d <<= 1) y = fmaxf(y, __shfl_xor_sync(0xFFFFFFFFu, y, d));
                        y = fmaxf(fmaf(y, sf[nt][e], -kPSet), m[nt][e]);
                        const float r = ex2(m[nt][e] - y);
                        m[nt][e] = y;
                        l[nt][e] *= r;
#pragma unroll
                        for (int mt = 0; mt < MT; ++mt) {
                            o[mt][nt][e] *= r;
                            o[mt][nt][e + 2] *= r;
                        }
                    }
            }
            uint32_t pf[2][NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    float p[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) p[e] = ex2(fmaf(sc[t][nt][e], sf[nt][e & 1], -m[nt][e & 1]));
                    l[nt][0] += p[0] + p[2];
                    l[nt][1] += p[1] + p[3];
                    pf[t][nt][0] = movmatrix(pack_half2(p[0], p[1]));
                    pf[t][nt][1] = movmatrix(pack_half2(p[2], p[3]));
                }

            // O^T += V^T P^T.  The lane's tokens 2c, 2c+1, 2c+8, 2c+9 of the
            // 16, and its D/8 values d of each.
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const uint32_t vb = base + v_codes + t * half_step, sb = base + v_scales + t * half_step_s;
                constexpr int VW = D / 64;  // words of a token
                uint32_t v[4][VW], sv[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const uint32_t at = vb + ((k & 1) * v_pair + (k >> 1) * 8) * (D / 2);
                    if constexpr (VW == 2)
                        asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v[k][0]), "=r"(v[k][VW - 1]) : "r"(at));
                    else
                        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v[k][0]) : "r"(at));
                    asm volatile("ld.shared.u8 %0, [%1];"
                                 : "=r"(sv[k]) : "r"(sb + ((k & 1) * v_pair + (k >> 1) * 8) * (D / 16)));
                }
                if (__builtin_expect(!open, 0)) {
                    // A token that a row does not see adds nothing to it, NaN
                    // or not: 0 * NaN is avoided by zeroing the scale, and a
                    // NaN block is put into the rows that do see its token.
                    uint32_t nan = 0;
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const int tok = tok0 + 16 * t + static_cast<int>(ta) + (k & 1) * v_pair + 8 * (k >> 1);
                        const bool there = ((have >> t) & 1u) && tok < s.q.len;
                        if (!there) sv[k] = 0u;
                        if ((sv[k] & 0x7Fu) == 0x7Fu) {
                            nan |= 1u << k;
                            sv[k] = 0u;
                        }
                    }
                    if (__any_sync(0xFFFFFFFFu, nan != 0u)) {
                        for (int k = 0; k < 16; ++k) {  // token k of the 16 belongs to lane (g, k / 4)'s k % 4
                            const uint32_t theirs = __shfl_sync(0xFFFFFFFFu, nan, (lane & ~3) | (k >> 2));
                            if (!((theirs >> (k & 3)) & 1u)) continue;
                            const int cc = k >> 2, x = (2 * cc) ^ (cc & 1);
                            const int tok = tok0 + 16 * t + (x ^ (k & 1)) + 8 * ((k >> 1) & 1);
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                                for (int e = 0; e < 2; ++e) {
                                    const int pos = s.q.pos0 + (8 * nt + 2 * c + e) / a.group;
                                    if (kv4_sees(pos, tok, a.window, a.sinks))
#pragma unroll
                                        for (int mt = 0; mt < MT; ++mt)
                                            o[mt][nt][e] = o[mt][nt][e + 2] = __uint_as_float(0x7FC00000u);
                                }
                        }
                    }
                }
                const uint32_t s01 = cvt_e4m3x2(static_cast<uint16_t>(sv[0] | (sv[1] << 8)));
                const uint32_t s23 = cvt_e4m3x2(static_cast<uint16_t>(sv[2] | (sv[3] << 8)));
#pragma unroll
                for (int w = 0; w < VW; ++w) {
                    constexpr uint32_t kLow = 0x0F0F0F0Fu;
                    uint32_t e01[4], d01[4], e23[4], d23[4];  // even and odd d of the two pairs of tokens
                    cvt_e2m1x2_x4(((v[0][w] >> 4) & kLow) | (v[1][w] & ~kLow), e01);
                    cvt_e2m1x2_x4((v[0][w] & kLow) | ((v[1][w] << 4) & ~kLow), d01);
                    cvt_e2m1x2_x4(((v[2][w] >> 4) & kLow) | (v[3][w] & ~kLow), e23);
                    cvt_e2m1x2_x4((v[2][w] & kLow) | ((v[3][w] << 4) & ~kLow), d23);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint32_t a0 = hmul2(e01[j], s01), a1 = hmul2(d01[j], s01);
                        const uint32_t a2 = hmul2(e23[j], s23), a3 = hmul2(d23[j], s23);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
                            mma_16816(o[4 * w + j][nt], a0, a1, a2, a3, pf[t][nt][0], pf[t][nt][1]);
                    }
                }
            }

            __syncwarp();
            if (lane == 0) mbar_arrive(done);
        }

        // Merge the warps: m and l first, then o scaled to the common maximum.
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) l[nt][e] += __shfl_xor_sync(0xFFFFFFFFu, l[nt][e], d);
                if (g == 0) {
                    sm_m[warp * ROWS + 8 * nt + 2 * c + e] = m[nt][e];
                    sm_l[warp * ROWS + 8 * nt + 2 * c + e] = l[nt][e];
                }
            }
        named_bar_sync(1, 32 * WARPS);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int r = 8 * nt + 2 * c + e;
                float top = kNoMax;
#pragma unroll
                for (int w = 0; w < WARPS; ++w) top = fmaxf(top, sm_m[w * ROWS + r]);
                const float f = ex2(m[nt][e] - top);
                float* at = merge + (warp * ROWS + r) * (D + 4) + g * (D / 8);
#pragma unroll
                for (int k = 0; k < MT / 2; ++k) {
                    *reinterpret_cast<float4*>(at + 4 * k) =
                        make_float4(o[2 * k][nt][e] * f, o[2 * k][nt][e + 2] * f, o[2 * k + 1][nt][e] * f,
                                    o[2 * k + 1][nt][e + 2] * f);
                }
            }
        named_bar_sync(1, 32 * WARPS);
        if (*failed && a.cluster == 0) return;  // all of them
        const bool partial = !(c0 == 0 && c1 == s.chunks) && a.cluster == 0;
        float* slot = partial ? step_slot<C>(a, my_run, c0 == 0 ? 1 : 0) : nullptr;
        if (partial && c0 == 0 && tid == 0)  // the run's last unit: it ends s.chunks - c1 chunks behind the run
            *step_link(a, my_run) = StepLink{
                static_cast<int>(((end + s.chunks - c1) * all_runs - 1) / all_chunks), s.q.first, row_count, head};
        for (int x = tid; x < row_count * (D / 4); x += WARPS * 32) {
            const int r = x / (D / 4), d = 4 * (x % (D / 4));
            float top = kNoMax;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) top = fmaxf(top, sm_m[w * ROWS + r]);
            float sum = 0.0f;
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < WARPS; ++w) {
                sum += sm_l[w * ROWS + r] * ex2(sm_m[w * ROWS + r] - top);
                const float4 u = *reinterpret_cast<const float4*>(merge + (w * ROWS + r) * (D + 4) + d);
                v.x += u.x; v.y += u.y; v.z += u.z; v.w += u.w;
            }
            if (a.cluster > 1) {  // into the ring, which is idle: o [row][D + 4] with m and l behind
                float* part = reinterpret_cast<float*>(smem) + r * (D + 4);
                *reinterpret_cast<float4*>(part + d) = v;
                if (d == 0) *reinterpret_cast<float2*>(part + D) = make_float2(top, sum);
            } else if (partial) {
                *reinterpret_cast<float4*>(slot + r * D + d) = v;
                if (d == 0) {
                    slot[ROWS * D + r] = top;
                    slot[ROWS * D + ROWS + r] = sum;
                }
            } else {
                kv4_store_row<BF16, D>(a, s.q.first, r, head, d, v, top, sum);
            }
        }
        if (a.cluster > 1) {
            // The CTAs of the cluster join their results through distributed
            // shared memory, each some of the values.
            __syncwarp();
            cluster_sync();
            const int rank = static_cast<int>(cluster_ctarank());
            for (int x = tid * a.cluster + rank; x < row_count * (D / 4); x += 32 * WARPS * a.cluster) {
                const int r = x / (D / 4), d = 4 * (x % (D / 4));
                float top = kNoMax, l = 0.0f;
                float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
                for (int k = 0; k < a.cluster; ++k) {
                    const uint32_t part = cluster_addr(smem, k) + r * (D + 4) * 4;
                    const float4 u = ld_cluster4(part + 4 * d), ml = ld_cluster4(part + 4 * D);
                    kv4_merge(top, l, v, ml.x, ml.y, u);
                }
                kv4_store_row<BF16, D>(a, s.q.first, r, head, d, v, top, l);
            }
            __syncwarp();
            cluster_sync();  // nobody leaves while its part is read
        }
    }
}

// Joins the partial results that the four threads of a value hold (every
// fourth each, in order) and stores the rows' values; the CTA's 256 threads
// have 256 / D rows.
template <bool BF16, int D>
__device__ __forceinline__ void join_and_store(const Kv4Attn& a, bool valid, int first, int row, int head, int d,
                                               float top, float l, float4 v) {
    __shared__ float4 part_v[4][64];
    __shared__ float2 part_ml[4][64];
    const int quarter = threadIdx.x / 64, item = threadIdx.x % 64;
    part_v[quarter][item] = v;
    part_ml[quarter][item] = make_float2(top, l);
    __syncthreads();
    if (quarter == 0 && valid) {
#pragma unroll
        for (int k = 1; k < 4; ++k) kv4_merge(top, l, v, part_ml[k][item].x, part_ml[k][item].y, part_v[k][item]);
        kv4_store_row<BF16, D>(a, first, row, head, d, v, top, l);
    }
}

// Joins the partial results of the units that more than one run shares.  The
// CTA of the run that a unit begins in follows the link that the run left;
// blockIdx.y takes 256 / D rows.
template <class C, bool BF16>
__global__ void __launch_bounds__(256) k_kv4_join(const Kv4Attn a) {
    constexpr int D = C::D, ROWS = C::ROWS, LANES = D / 4;
    grid_dep_wait();
    const int run = blockIdx.x;
    const StepLink link = *step_link(a, run);
    const int quarter = threadIdx.x / 64, item = threadIdx.x % 64;
    const int r = blockIdx.y * (64 / LANES) + item / LANES, d = 4 * (item % LANES);
    if (link.last < 0 || static_cast<int>(blockIdx.y) * (64 / LANES) >= link.rows) return;
    const bool valid = r < link.rows;
    float top = kNoMax, l = 0.0f;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (valid) {
#pragma unroll 4
        for (int i = run + quarter; i <= link.last; i += 4) {
            const float* slot = step_slot<C>(a, i, i == run ? 1 : 0);
            kv4_merge(top, l, v, slot[ROWS * D + r], slot[ROWS * D + ROWS + r],
                      *reinterpret_cast<const float4*>(slot + r * D + d));
        }
    }
    join_and_store<BF16, D>(a, valid, link.first, r, link.head, d, top, l, v);
}

}  // namespace tb
