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
// turn 256 codes into FP16 and multiply them, so instructions count:
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
//   - the maximum is moved only when a score passes it by 2^8: P stays below
//     2^8, far inside FP16, and the reductions over lanes are rare.
// P is rounded to FP16 (2^-11), finer than either output type is to a sum's
// terms; l is summed from the FP32 values.
//
// BF16 queries are scaled per row by a power of two to at most 2^15 and taken
// as FP16: exact for values within 2^-28 of the row's largest, and off by at
// most 2^-39 of it below, which FP32 sums do not resolve.
//
// Split: the (sequence, row tile, KV head) units' 32-token chunks are laid end
// to end, and each CTA takes an equal run of them, so a batch of any lengths
// loads all SMs alike.  A run's ends inside a unit leave partial results
// (o, m, l) in the workspace for k_kv4_join.  Within a CTA the warps take
// chunks in turn, each with its own ring of bulk copies and its own o, m, l,
// merged once per unit in a fixed order.
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
    int whole;                     // step kernel: one CTA per unit, no partial results
    int runs;                      // CTAs that share the chunks (not `whole`)
    int min_run;                   // chunks a CTA should have at least
    int step_rows;                 // packed rows that the step kernel takes; sequences with more are the prompt kernel's
    float* prompt_ws;
    int prompt_tiles;              // tiles of 256 packed rows of a sequence at most
    int prompt_splits;             // CTAs that share a prompt unit's tokens
};

// Bit of the device error word: a sequence has more rows than max_rows.
enum : int { kErrRows = 4 };

constexpr int kStepWarps = 8;
constexpr int kStepChunk = 32;  // tokens
constexpr int kStepRowsMost = 32;  // packed rows of a (sequence, KV head)

template <int D_, int NT_>
struct StepCfg {
    static constexpr int D = D_, NT = NT_;
    static constexpr int ROWS = 8 * NT;
    static constexpr int TOKEN_BYTES = D / 2 + D / 16;  // of K or of V
    static constexpr int STAGE = kStepChunk * TOKEN_BYTES * 2;
    static constexpr int ST = 3;
    static constexpr int RING = kStepWarps * ST * STAGE;
    static constexpr int MERGE = kStepWarps * ROWS * (D + 4) * 4;
    static constexpr int QFRAG = NT * (D / 16) * 32 * 8;
    static constexpr int UNION = RING > MERGE ? RING : MERGE;
    static constexpr int ML = kStepWarps * ROWS * 2 * 4;
    static constexpr int SMEM = UNION + QFRAG + ML + ROWS * 4 + kStepWarps * ST * 8 + 256;
    static constexpr int SLOT = ROWS * (D + 2);  // floats of a partial result: o [ROWS x D], m, l
};

// A partial result belongs to CTA `run`: slot 0 for the unit that began in an
// earlier CTA's run, slot 1 for one that begins here and goes on.
template <class C>
__device__ __forceinline__ float* step_slot(float* ws, int run, int slot) {
    return ws + (static_cast<size_t>(run) * 2 + slot) * C::SLOT;
}

__device__ __forceinline__ void bulk_load(void* smem_dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
            smem_addr(smem_dst)),
        "l"(reinterpret_cast<uint64_t>(src)), "r"(bytes), "r"(smem_addr(bar))
        : "memory");
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

// Adds a partial result (u, li, mi) to (v, l, top); a part that saw nothing of
// the row has mi = -inf, li = 0 and u = 0, or NaN that stays.
__device__ __forceinline__ void kv4_merge(float& top, float& l, float4& v, float mi, float li, float4 u) {
    const float mt = fmaxf(top, mi);
    const float f = top == -INFINITY ? 0.0f : ex2(top - mt), fi = mi == -INFINITY ? 0.0f : ex2(mi - mt);
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

__device__ __forceinline__ StepSeq step_seq(const Kv4Attn& a, int b) {
    StepSeq s;
    s.q = kv4_seq(a.rows, a.cache.page_shift, a.rows.cu[b], a.rows.cu[b + 1], a.rows.lens[b]);
    s.span = kv4_span(s.q.pos0, s.q.pos0 + s.q.n - 1, s.q.len, a.window, a.sinks, 5);
    const long long rows = static_cast<long long>(s.q.n) * a.group;
    s.chunks = rows > 0 && rows <= a.step_rows ? kv4_span_chunks(s.span) : 0;
    return s;
}

// Reports a sequence that neither kernel takes: more rows than max_rows said.
__device__ __forceinline__ void step_report(const Kv4Attn& a, const StepSeq& s) {
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
__global__ void __launch_bounds__(kStepWarps * 32, C::NT == 1 ? 2 : 1) k_kv4_step(const Kv4Attn a) {
    constexpr int D = C::D, NT = C::NT, ROWS = C::ROWS, ST = C::ST;
    constexpr int KS = D / 16;   // k-steps of K Q^T
    constexpr int MT = D / 16;   // 16-row tiles of V^T
    extern __shared__ __align__(128) uint8_t smem[];
    uint8_t* ring = smem;
    float* merge = reinterpret_cast<float*>(smem);
    uint2* qfrag = reinterpret_cast<uint2*>(smem + C::UNION);
    float* sm_m = reinterpret_cast<float*>(smem + C::UNION + C::QFRAG);
    float* sm_l = sm_m + kStepWarps * ROWS;
    float* sm_scale = sm_l + kStepWarps * ROWS;
    uint64_t* bars = reinterpret_cast<uint64_t*>(sm_scale + ROWS);
    long long* sums = reinterpret_cast<long long*>(bars + kStepWarps * ST);  // one per warp, then the result
    volatile int* abort = reinterpret_cast<volatile int*>(sums + kStepWarps + 2);

    grid_dep_launch_dependents();  // k_kv4_join waits for this grid's end
    const int tid = threadIdx.x, warp = tid / 32, lane = tid & 31;
    const int g = lane >> 2, c = lane & 3;
    uint64_t* bar = bars + warp * ST;
    if (lane == 0) {
        for (int i = 0; i < ST; ++i) mbar_init(&bar[i], 1);
        fence_barrier_init();
    }
    if (tid == 0) *abort = 0;
    __syncthreads();

    // This CTA's run of chunks: sequence b, offset `off` in it, `left` chunks.
    int b = 0;
    long long off = 0, left = 0;
    int my_run = blockIdx.x;
    if (a.whole) {
        b = blockIdx.x / a.cache.heads;
        const StepSeq s = step_seq(a, b);
        step_report(a, s);
        if (s.chunks == 0) return;
        off = static_cast<long long>(blockIdx.x - b * a.cache.heads) * s.chunks;
        left = s.chunks;
    } else {
        long long sum = 0;
        for (int i = tid; i < a.rows.batch; i += blockDim.x) {
            const StepSeq s = step_seq(a, i);
            step_report(a, s);
            sum += s.total(a.cache.heads);
        }
        const long long total = block_sum(sum, sums);
        const int runs = step_runs(a, total);
        if (my_run >= runs) return;
        const long long from = run_start(total, runs, my_run);
        left = run_start(total, runs, my_run + 1) - from;
        if (left <= 0) return;
        long long before = 0;
        for (int b0 = 0; b0 < a.rows.batch; b0 += blockDim.x) {
            const int i = b0 + tid;
            const long long w = i < a.rows.batch ? step_seq(a, i).total(a.cache.heads) : 0;
            long long upto = w;  // inclusive sum over the CTA's threads
            for (int d = 1; d < 32; d <<= 1) {
                const long long o = __shfl_up_sync(0xFFFFFFFFu, upto, d);
                if (lane >= d) upto += o;
            }
            __syncthreads();
            if (lane == 31) sums[warp] = upto;
            __syncthreads();
            long long all = 0;
            for (int k = 0; k < kStepWarps; ++k) {
                if (k < warp) upto += sums[k];
                all += sums[k];
            }
            const long long lo = before + upto - w;
            if (w > 0 && from >= lo && from < lo + w) {
                sums[kStepWarps] = i;
                sums[kStepWarps + 1] = from - lo;
            }
            before += all;
            if (before > from) break;
        }
        __syncthreads();
        b = static_cast<int>(sums[kStepWarps]);
        off = sums[kStepWarps + 1];
    }

    uint32_t used = 0;  // chunks this warp has taken through its ring
    const float thr = 8.0f;
    while (left > 0 && b < a.rows.batch) {
        const StepSeq s = step_seq(a, b);
        if (off >= s.total(a.cache.heads)) {
            off -= s.total(a.cache.heads);
            ++b;
            continue;
        }
        const int head = static_cast<int>(off / s.chunks);
        const int c0 = static_cast<int>(off - static_cast<long long>(head) * s.chunks);
        const int c1 = left < s.chunks - c0 ? c0 + static_cast<int>(left) : s.chunks;
        const int row_count = s.q.n * a.group;  // at most ROWS
        left -= c1 - c0;
        off += c1 - c0;
        if (tid == 0 && s.q.bad) atomicOr(&g_tb_device_error, kErrPage);

        // Queries in fragment order: lane (g, c) of k-step ks holds, for row
        // g, the values d = (D/4) c + 4 ks .. + 3, each pair swapped as the
        // converter leaves a byte's two codes.
        for (int r = warp; r < ROWS; r += kStepWarps) {
            uint2 v = make_uint2(0u, 0u);
            float scale = a.scale_log2;
            if (r < row_count) {
                const int i = r / a.group;
                const long long at = (s.q.first + i) * a.q_stride +
                                     static_cast<long long>(head * a.group + r - i * a.group) * D + 4 * lane;
                if (lane < D / 4) v = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(a.q) + at);
                if constexpr (BF16) {
                    // Exponent of the row's largest value -> 2^k that brings it to [2^14, 2^15),
                    // in two factors (k passes 127 for the smallest rows); not for infinity and NaN.
                    uint32_t e = max(max((v.x >> 7) & 0xFFu, (v.x >> 23) & 0xFFu),
                                     max((v.y >> 7) & 0xFFu, (v.y >> 23) & 0xFFu));
                    e = __reduce_max_sync(0xFFFFFFFFu, e);
                    const int k = e == 255u ? 0 : 141 - static_cast<int>(e), k1 = k > 120 ? 120 : k, k2 = k - k1;
                    const float up = exp2i(k1), up2 = exp2i(k2);
                    scale = (scale * exp2i(-k1)) * exp2i(-k2);
                    v.x = pack_half2(__uint_as_float(v.x << 16) * up * up2, __uint_as_float(v.x & 0xFFFF0000u) * up * up2);
                    v.y = pack_half2(__uint_as_float(v.y << 16) * up * up2, __uint_as_float(v.y & 0xFFFF0000u) * up * up2);
                }
            }
            if (lane < D / 4) {
                const int ks = lane % KS, cc = lane / KS;
                qfrag[((r / 8) * KS + ks) * 32 + (r % 8) * 4 + cc] =
                    make_uint2(prmt(v.x, 0u, 0x1032u), prmt(v.y, 0u, 0x1032u));
            }
            if (lane == 0) sm_scale[r] = scale;
        }
        __syncthreads();

        float sf[NT][2];  // score -> log2 units, of rows 8 nt + 2c, + 1
        float m[NT][2], l[NT][2];
        float o[MT][NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                sf[nt][e] = sm_scale[8 * nt + 2 * c + e];
                m[nt][e] = -INFINITY;
                l[nt][e] = 0.0f;
            }
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[mt][nt][e] = 0.0f;

        // Chunk geometry: pages of 16 and of 32 tokens come with all four
        // parts of a page's head block in one copy; larger pages part by part.
        const int shift = a.cache.page_shift;
        const uint32_t codes = kv4_codes_bytes(a.cache), scales = kv4_scales_bytes(a.cache);
        const uint32_t unit_tokens = shift == 4 ? 16u : 32u;
        const uint32_t half_step = shift == 4 ? 16u * C::TOKEN_BYTES * 2 : 16u * (D / 2);  // codes of tokens 16..31
        const uint32_t half_step_s = shift == 4 ? half_step : 16u * (D / 16);              // scales of tokens 16..31
        const uint32_t at_ks = unit_tokens * (D / 2), at_vc = at_ks + unit_tokens * (D / 16),
                       at_vs = at_vc + unit_tokens * (D / 2);
        const int* table = a.rows.table + static_cast<size_t>(b) * a.rows.width;
        const int first_pos = s.q.pos0, last_pos = s.q.pos0 + s.q.n - 1;  // of the rows

        // Page numbers of a chunk: two for 16-token pages.
        auto look = [&](int q, int& p0, int& p1) {
            p0 = p1 = -1;
            if (q >= c1) return;
            const int tok = kv4_span_chunk(s.span, q) * kStepChunk;
            if (tok < s.q.len) p0 = table[tok >> shift];
            if (shift == 4 && tok + 16 < s.q.len) p1 = table[(tok >> shift) + 1];
        };
        // Start the copies of chunk q into `stage`; returns which halves hold tokens.
        auto issue = [&](int q, int p0, int p1, int stage) -> uint32_t {
            const int tok = kv4_span_chunk(s.span, q) * kStepChunk;
            uint32_t have = 0;
            const bool ok0 = tok < s.q.len && kv4_page_ok(a.cache, p0);
            const bool ok1 = shift == 4 ? tok + 16 < s.q.len && kv4_page_ok(a.cache, p1) : ok0;
            have = (ok0 ? 1u : 0u) | (ok1 ? 2u : 0u);
            if (lane == 0) {
                uint8_t* dst = ring + (warp * ST + stage) * C::STAGE;
                if ((tok < s.q.len && !ok0) || (shift == 4 && tok + 16 < s.q.len && !ok1))
                    atomicOr(&g_tb_device_error, kErrPage);
                const uint32_t bytes = shift == 4 ? (ok0 + ok1) * (C::STAGE / 2) : ok0 ? C::STAGE : 0u;
                mbar_arrive_expect_tx(&bar[stage], bytes);
                if (shift <= 5) {
                    if (ok0)
                        bulk_load(dst, a.cache.data + kv4_block_offset(a.cache, p0, head),
                                  shift == 4 ? C::STAGE / 2 : C::STAGE, &bar[stage]);
                    if (shift == 4 && ok1)
                        bulk_load(dst + C::STAGE / 2, a.cache.data + kv4_block_offset(a.cache, p1, head), C::STAGE / 2,
                                  &bar[stage]);
                } else if (ok0) {
                    const uint32_t place = static_cast<uint32_t>(tok) & ((1u << shift) - 1u);
                    const uint8_t* src = a.cache.data + kv4_block_offset(a.cache, p0, head);
                    bulk_load(dst, src + place * (D / 2), kStepChunk * (D / 2), &bar[stage]);
                    bulk_load(dst + at_ks, src + codes + place * (D / 16), kStepChunk * (D / 16), &bar[stage]);
                    src += codes + scales;
                    bulk_load(dst + at_vc, src + place * (D / 2), kStepChunk * (D / 2), &bar[stage]);
                    bulk_load(dst + at_vs, src + codes + place * (D / 16), kStepChunk * (D / 16), &bar[stage]);
                }
            }
            return have;
        };

        uint32_t halves = 0;  // which halves of the chunks in flight hold tokens: two bits a stage
        int next = c0 + warp, p0, p1;
        const int mine = next < c1 ? (c1 - next + kStepWarps - 1) / kStepWarps : 0;
#pragma unroll
        for (int i = 0; i < ST; ++i) {
            if (i < mine) {
                look(next, p0, p1);
                const int stage = (used + i) % ST;
                halves = (halves & ~(3u << (2 * stage))) | (issue(next, p0, p1, stage) << (2 * stage));
                next += kStepWarps;
            }
        }
        look(next, p0, p1);

        for (int it = 0; it < mine; ++it) {
            const int stage = used % ST;
            const uint32_t parity = (used / ST) & 1u;
            ++used;
            const int tok0 = kv4_span_chunk(s.span, c0 + warp + it * kStepWarps) * kStepChunk;
            if (!mbar_wait(&bar[stage], parity, abort)) {
                // Let the copies in flight end before the ring is given up.
                const int flying = min(ST, mine - it);
                for (int i = 0; i < flying; ++i)
                    mbar_wait_drain(&bar[(used - 1 + i) % ST], ((used - 1 + i) / ST) & 1u);
                break;
            }
            const uint32_t base = smem_addr(ring + (warp * ST + stage) * C::STAGE);
            const uint32_t have = (halves >> (2 * stage)) & 3u;
            // Every row sees the whole chunk, and all of it is there.
            const bool open = have == 3u && tok0 + kStepChunk - 1 <= first_pos &&
                              tok0 + kStepChunk <= s.q.len &&
                              (a.window <= 0 || last_pos - tok0 < a.window || tok0 + kStepChunk <= a.sinks);

            float sc[2][NT][4];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) sc[t][nt][e] = 0.0f;
                // Row g of the tile is token g ^ (g >> 1 & 1): neighbouring
                // lanes of the loads below then fall into different banks.
                const uint32_t tok = static_cast<uint32_t>(g ^ ((g >> 1) & 1));
                const uint32_t kb = base + t * half_step + tok * (D / 2) + c * (D / 8);
                const uint32_t sb = base + at_ks + t * half_step_s + tok * (D / 16) + c * (D / 64);
                uint32_t ka[D / 32], kc[D / 32];  // codes of tokens g and g + 8
                uint32_t sa[D / 64], sd[D / 64];  // their scales, doubled
                if constexpr (D == 128) {
                    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                                 : "=r"(ka[0]), "=r"(ka[1]), "=r"(ka[2]), "=r"(ka[3]) : "r"(kb));
                    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                                 : "=r"(kc[0]), "=r"(kc[1]), "=r"(kc[2]), "=r"(kc[3]) : "r"(kb + 8 * (D / 2)));
                    uint16_t x, y;
                    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(x) : "r"(sb));
                    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(y) : "r"(sb + 8 * (D / 16)));
                    const uint32_t xx = cvt_e4m3x2(x), yy = cvt_e4m3x2(y);
                    sa[0] = prmt(xx, 0u, 0x1010u); sa[1] = prmt(xx, 0u, 0x3232u);
                    sd[0] = prmt(yy, 0u, 0x1010u); sd[1] = prmt(yy, 0u, 0x3232u);
                } else {
                    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(ka[0]), "=r"(ka[1]) : "r"(kb));
                    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(kc[0]), "=r"(kc[1]) : "r"(kb + 8 * (D / 2)));
                    uint32_t x, y;
                    asm volatile("ld.shared.u8 %0, [%1];" : "=r"(x) : "r"(sb));
                    asm volatile("ld.shared.u8 %0, [%1];" : "=r"(y) : "r"(sb + 8 * (D / 16)));
                    sa[0] = cvt_e4m3x2(static_cast<uint16_t>(x | (x << 8)));
                    sd[0] = cvt_e4m3x2(static_cast<uint16_t>(y | (y << 8)));
                }
#pragma unroll
                for (int w = 0; w < D / 32; ++w) {
                    uint32_t fa[4], fc[4];
                    cvt_e2m1x2_x4(ka[w], fa);
                    cvt_e2m1x2_x4(kc[w], fc);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        fa[j] = hmul2(fa[j], sa[w / 2]);
                        fc[j] = hmul2(fc[j], sd[w / 2]);
                    }
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            const uint2 qf = qfrag[(nt * KS + 2 * w + h) * 32 + lane];
                            mma_16816(sc[t][nt], fa[2 * h], fc[2 * h], fa[2 * h + 1], fc[2 * h + 1], qf.x, qf.y);
                        }
                }
            }

            // Scores in log2 units; hidden ones are -inf.
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) sc[t][nt][e] *= sf[nt][e & 1];
            const int tg = g ^ ((g >> 1) & 1);
            if (!open) {
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
            bool past = false;
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) past |= sc[t][nt][e] > m[nt][e & 1] + thr;
            if (__any_sync(0xFFFFFFFFu, past)) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float x = fmaxf(fmaxf(sc[0][nt][e], sc[0][nt][e + 2]), fmaxf(sc[1][nt][e], sc[1][nt][e + 2]));
#pragma unroll
                        for (int d = 4; d < 32; d <<= 1) x = fmaxf(x, __shfl_xor_sync(0xFFFFFFFFu, x, d));
                        x = fmaxf(x, m[nt][e]);
                        const float f = x == -INFINITY ? 1.0f : ex2(m[nt][e] - x);
                        m[nt][e] = x;
                        l[nt][e] *= f;
#pragma unroll
                        for (int mt = 0; mt < MT; ++mt) {
                            o[mt][nt][e] *= f;
                            o[mt][nt][e + 2] *= f;
                        }
                    }
            }
            uint32_t pf[2][NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const float m0 = m[nt][0] == -INFINITY ? 0.0f : m[nt][0];
                const float m1 = m[nt][1] == -INFINITY ? 0.0f : m[nt][1];
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    float x[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[e] = ex2(sc[t][nt][e] - (e & 1 ? m1 : m0));
                    l[nt][0] += x[0] + x[2];
                    l[nt][1] += x[1] + x[3];
                    pf[t][nt][0] = movmatrix(pack_half2(x[0], x[1]));
                    pf[t][nt][1] = movmatrix(pack_half2(x[2], x[3]));
                }
            }

            // O^T += V^T P^T.  The lane's tokens 2c, 2c+1, 2c+8, 2c+9 of the
            // 16, and its D/8 values d of each.
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const uint32_t ta = static_cast<uint32_t>((2 * c) ^ (c & 1)), tb2 = ta ^ 1u;
                const uint32_t vb = base + at_vc + t * half_step + g * (D / 16);
                const uint32_t sb = base + at_vs + t * half_step_s + (g * (D / 16)) / 8;
                constexpr int VW = D / 64;  // words of a token
                uint32_t v[4][VW], sv[4];
                const uint32_t tk[4] = {ta, tb2, ta + 8, tb2 + 8};
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    if constexpr (VW == 2)
                        asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];"
                                     : "=r"(v[k][0]), "=r"(v[k][VW - 1]) : "r"(vb + tk[k] * (D / 2)));
                    else
                        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v[k][0]) : "r"(vb + tk[k] * (D / 2)));
                    asm volatile("ld.shared.u8 %0, [%1];" : "=r"(sv[k]) : "r"(sb + tk[k] * (D / 16)));
                }
                if (!open) {
                    // A token that a row does not see adds nothing to it, NaN
                    // or not: 0 * NaN is avoided by zeroing the scale, and a
                    // NaN block is put into the rows that do see its token.
                    uint32_t nan = 0;
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const int tok = tok0 + 16 * t + static_cast<int>(tk[k]);
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
            if (it + ST < mine) {
                halves = (halves & ~(3u << (2 * stage))) | (issue(next, p0, p1, stage) << (2 * stage));
                next += kStepWarps;
                look(next, p0, p1);
            }
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
        __syncthreads();  // also: nobody reads the ring any more
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int r = 8 * nt + 2 * c + e;
                float top = -INFINITY;
#pragma unroll
                for (int w = 0; w < kStepWarps; ++w) top = fmaxf(top, sm_m[w * ROWS + r]);
                const float f = m[nt][e] == -INFINITY ? 0.0f : ex2(m[nt][e] - top);
                float* at = merge + (warp * ROWS + r) * (D + 4) + g * (D / 8);
#pragma unroll
                for (int k = 0; k < MT / 2; ++k) {
                    *reinterpret_cast<float4*>(at + 4 * k) =
                        make_float4(o[2 * k][nt][e] * f, o[2 * k][nt][e + 2] * f, o[2 * k + 1][nt][e] * f,
                                    o[2 * k + 1][nt][e + 2] * f);
                }
            }
        __syncthreads();
        const bool partial = !(c0 == 0 && c1 == s.chunks);
        float* slot = partial ? step_slot<C>(a.ws, my_run, c0 == 0 ? 1 : 0) : nullptr;
        for (int x = tid; x < row_count * (D / 4); x += kStepWarps * 32) {
            const int r = x / (D / 4), d = 4 * (x % (D / 4));
            float top = -INFINITY;
#pragma unroll
            for (int w = 0; w < kStepWarps; ++w) top = fmaxf(top, sm_m[w * ROWS + r]);
            float sum = 0.0f;
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < kStepWarps; ++w) {
                const float mw = sm_m[w * ROWS + r];
                sum += sm_l[w * ROWS + r] * (mw == -INFINITY ? 0.0f : ex2(mw - top));  // NaN stays NaN
                const float4 u = *reinterpret_cast<const float4*>(merge + (w * ROWS + r) * (D + 4) + d);
                v.x += u.x; v.y += u.y; v.z += u.z; v.w += u.w;
            }
            if (partial) {
                *reinterpret_cast<float4*>(slot + r * D + d) = v;
                if (d == 0) {
                    slot[ROWS * D + r] = top;
                    slot[ROWS * D + ROWS + r] = sum;
                }
            } else {
                kv4_store_row<BF16, D>(a, s.q.first, r, head, d, v, top, sum);
            }
        }
        // The merge area becomes the ring again: generic accesses first.
        fence_proxy_async_smem();
        __syncthreads();
        if (*abort) return;
    }
}

// Joins the partial results of the units that more than one run shares, in the
// order of the runs.  One CTA per unit that may exist.
template <class C, bool BF16>
__global__ void __launch_bounds__(256) k_kv4_join(const Kv4Attn a) {
    constexpr int D = C::D, ROWS = C::ROWS;
    __shared__ long long sums[8];
    grid_dep_wait();
    const int b = blockIdx.x / a.cache.heads, head = blockIdx.x - b * a.cache.heads;
    const StepSeq s = step_seq(a, b);
    if (s.chunks == 0) return;
    long long sum = 0, sum_before = 0;
    for (int i = threadIdx.x; i < a.rows.batch; i += blockDim.x) {
        const long long w = step_seq(a, i).total(a.cache.heads);
        sum += w;
        if (i < b) sum_before += w;
    }
    const long long total = block_sum(sum, sums), before = block_sum(sum_before, sums);
    const int runs = step_runs(a, total);
    const long long u0 = before + static_cast<long long>(head) * s.chunks, u1 = u0 + s.chunks;
    const int r0 = static_cast<int>(((u0 + 1) * runs - 1) / total), r1 = static_cast<int>((u1 * runs - 1) / total);
    if (r0 == r1) return;  // one run had all of it
    const int row_count = s.q.n * a.group;
    for (int x = threadIdx.x; x < row_count * (D / 4); x += blockDim.x) {
        const int r = x / (D / 4), d = 4 * (x % (D / 4));
        float top = -INFINITY, l = 0.0f;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int i = r0; i <= r1; ++i) {
            const float* slot = step_slot<C>(a.ws, i, i == r0 ? 1 : 0);
            kv4_merge(top, l, v, slot[ROWS * D + r], slot[ROWS * D + ROWS + r],
                      *reinterpret_cast<const float4*>(slot + r * D + d));
        }
        kv4_store_row<BF16, D>(a, s.q.first, r, head, d, v, top, l);
    }
}

}  // namespace tb
