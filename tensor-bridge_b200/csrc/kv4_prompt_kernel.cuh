// kv4_prompt_kernel.cuh -- attention of many rows per sequence (a prompt, or a
// chunk of one) over the block-scaled FP4 cache, on tcgen05.
//
// The kernel is persistent, and what loads and decodes goes on into the next
// item while the last one's rows are finished.  Where the sequences have like
// numbers of rows a CTA takes an item of each round.  Else (DRAWN) the loading
// warp draws items from a counter that all CTAs share and hands their numbers
// on through a ring.
// An item is 256 packed rows (token, head of one KV head's group) as two tiles
// of 128 and runs over their visible tokens in tiles of 128:
//   S_t = Q_t K^T     tcgen05.mma, both operands in shared memory, S_t in TMEM
//   P_t = 2^(S_t - m) one thread per row, S_t read from and P_t (FP16) written
//                     to the same TMEM columns
//   O_t += P_t V      tcgen05.mma, P_t from TMEM, V from shared memory
// While one tile's rows take their exponentials the tensor core works for the
// other: P_0 V, the next S_0, P_1 V, the next S_1.  K and V arrive as codes
// (bulk copies, one per page where a page is at most a tile) and eight warps turn
// them into FP16 operand tiles once per 256 rows, K's and V's in turn; a thread
// owns half of a token of the tile.
//
// Layout: K, V and Q tiles are [row][64 d] panels of 128-byte rows under the
// 128-byte swizzle.  The same picture is K-major for Q K^T and, as [token][d],
// N-major for P V, so one decoder serves both.  A byte's two codes come out of
// the converter second value first; Q is stored in the same order, and the
// output's columns are swapped back when they are read.
//
// The maximum m of a row is moved only when a score passes it by almost 2^16, to
// 2^6 below that score, so the usual tile takes one pass: exponentials with the old
// m, the largest score found along the way, and a second pass (with O scaled in
// TMEM) only if it passed.  S_t of a tile is issued behind
// P_t V of the tile before, so a thread that sees S_t finds O_t at rest.
//
// What bounds it: a row tile and token tile (128 x 128, D = 128) needs 1024
// cycles of an SM's exponentials and 1024 of its tensor core, and takes about
// 2300: S_t waits for P_t V and P_t for S_t, so that the two tiles' phases
// overlap only in part, and what the softmax warps issue beside the exponentials
// (scale, maximum, sum, packing) shares its slots with the decoding warps.  At
// D = 64 a tile takes hardly less, though its products are half: the softmax
// warps' chain (wait, load, scale, maximum, exponential, pack, store) is what
// remains, and each move of m, two passes more and O scaled, adds to it.
// P is rounded to FP16 as in the step kernel (m is a whole number here, so P's
// largest may lie at 2^5), l is summed in FP32.
// Measured, 32 heads of 128, 8 KV heads, in a CUDA graph with the cache in L2: a
// prompt of 4096 tokens 162 us (848 TFLOP/s, 0.52 of a bf16 GEMM; a call with L2
// cold 176 us, 781 TFLOP/s), 2048 rows behind 14336 tokens 542 us (951 TFLOP/s;
// with a CTA an item instead of persistent ones it took 493 us, the prompt as
// long); ends of items cost ~14000 cycles each, hence whole rounds of large items
// first.
//
// TMEM (512 columns): S_0, S_1 (128 each, P in the first 64), O_0, O_1 (D each).
#pragma once

#include "kv4_step_kernel.cuh"

namespace tb {

constexpr int kPromptRows = 256;
constexpr int kPromptTile = 128;                    // tokens
constexpr int kPromptBatch = 2048;                  // sequences that a list of those with rows here holds
constexpr int kPromptThreads = 640;                 // warps: 8 softmax, 8 decode, MMA, loader, 2 idle

template <int D_>
struct PromptCfg {
    static constexpr int D = D_;
    static constexpr int PANELS = D / 64;
    static constexpr int PANEL = 128 * 128;         // bytes: 128 rows of 64 FP16 values
    static constexpr int OPERAND = PANELS * PANEL;  // a K, V or Q tile
    static constexpr int SLOTS = 3;
    static constexpr int TOKEN_BYTES = D / 2 + D / 16;
    static constexpr int RAW = kPromptTile * TOKEN_BYTES * 2;
    static constexpr int NR = 3;
    static constexpr int OFF_SLOT = 2 * OPERAND;
    static constexpr int OFF_RAW = OFF_SLOT + SLOTS * OPERAND;
    static constexpr int OFF_BAR = OFF_RAW + NR * RAW;
    static constexpr int OFF_QSCALE = OFF_BAR + 512;
    static constexpr int OFF_LIST = OFF_QSCALE + kPromptRows * 4;
    static constexpr int SMEM = OFF_LIST + kPromptBatch * 4 + 1024;  // + alignment of the base
    static_assert(SMEM <= 227 * 1024, "shared memory");
    static constexpr int S_COLS = 128;
    static constexpr int O_COL = 256;
    // Registers a thread: at launch, then by role.
    static constexpr int REGS = 96, REGS_SOFTMAX = 152, REGS_DECODE = 64, REGS_REST = 40;
    static_assert(256 * (REGS_SOFTMAX + REGS_DECODE) + 128 * REGS_REST <= kPromptThreads * REGS, "registers of the launch");
};

// Low word of the descriptor of an N-major operand tile (V as [token][d]): 64
// values of N are a 128-byte row, 8 rows of K an atom of 1024 bytes (the stride
// byte offset, in the high word), 64 more values of N a panel (the leading byte
// offset).
template <class C>
__device__ __forceinline__ uint32_t sdesc_v_lo(uint32_t addr) {
    return ((addr >> 4) & 0x3FFFu) | (static_cast<uint32_t>(C::PANEL >> 4) << 16);
}

// Whether the prompt kernel takes a sequence: more packed rows than the step
// kernel's largest tile.
__device__ __forceinline__ bool prompt_takes(const Kv4Attn& a, const Kv4Seq& q) {
    return static_cast<long long>(q.n) * a.group > kStepRowsMost;
}

// An item of work: some rows of a sequence and head, and a share of their
// tiles of tokens (t0 == t1: nothing to do).
struct PromptUnit {
    Kv4Seq q;
    Kv4Span span;
    int b, head, row_base, row_count;
    int first_pos, last_pos;
    int t0, t1;  // tiles of the span
    bool any;
    int split;  // share of its tokens
};

// Row tile `tile` of KV head `head` of sequence b, with all its tokens.
__device__ __forceinline__ PromptUnit prompt_rows(const Kv4Attn& a, int b, int head, int tile) {
    PromptUnit u;
    u.b = b;
    u.head = head;
    u.split = 0;
    u.q = kv4_rows_seq(a.rows, a.cache.page_shift, a.rows.cu[u.b], a.rows.cu[u.b + 1], a.rows.lens[u.b]);
    u.row_base = tile * kPromptRows;
    u.row_count = min(kPromptRows, u.q.n * a.group - u.row_base);
    u.t0 = u.t1 = 0;
    u.any = prompt_takes(a, u.q) && u.row_count > 0;
    if (!u.any) return u;
    u.first_pos = u.q.pos0 + u.row_base / a.group;
    u.last_pos = u.q.pos0 + (u.row_base + u.row_count - 1) / a.group;
    u.span = kv4_span(u.first_pos, u.last_pos, u.q.len, a.window, a.sinks, 7);
    u.t1 = kv4_span_chunks(u.span);
    return u;
}

// Partial results lie by share, KV head and packed row of the whole call: all
// o, then all m, then all l.  The number of a unit's first row among them: tiles
// of 256 rows of the call * heads * splits are no more than the SMs, so it is
// small; a 64-bit address cost registers (a prompt of 4096 tokens 165 us for 162).
__device__ __forceinline__ uint32_t prompt_slot(const Kv4Attn& a, const PromptUnit& u, int split) {
    return static_cast<uint32_t>(((split * a.cache.heads + u.head) * a.rows.rows + u.q.first) * a.group + u.row_base);
}
template <class C>
__device__ __forceinline__ float* prompt_m(const Kv4Attn& a) {
    return a.prompt_ws + static_cast<size_t>(a.prompt_splits) * a.cache.heads * a.rows.rows * a.group * C::D;
}
__device__ __forceinline__ size_t prompt_m_to_l(const Kv4Attn& a) {
    return static_cast<size_t>(a.prompt_splits) * a.cache.heads * a.rows.rows * a.group;
}

// Item number `item`: share (item % splits) of unit item / splits.  A unit is a
// KV head of a row tile; a sequence's last row tiles see the most tokens, so all
// sequences' last ones come first.  `list` holds the `seqs` sequences that have
// row tiles here; nullptr: all of them.
__device__ __forceinline__ PromptUnit prompt_unit(const Kv4Attn& a, const int* list, int seqs, int item) {
    PromptUnit u;
    int unit = item, split = 0;
    if (a.prompt_splits > 1) {
        unit = item / a.prompt_splits;
        split = item - unit * a.prompt_splits;
    }
    const int per_tile = seqs * a.cache.heads;
    const int tile = a.prompt_tiles - 1 - unit / per_tile;
    const int rest = unit % per_tile;
    u.b = rest / a.cache.heads;
    u.head = rest - u.b * a.cache.heads;
    if (list != nullptr) u.b = list[u.b];
    u = prompt_rows(a, u.b, u.head, tile);
    if (a.prompt_splits > 1) {
        const long long tiles = u.t1;
        u.split = split;
        u.t0 = static_cast<int>(tiles * split / a.prompt_splits);
        u.t1 = static_cast<int>(tiles * (split + 1) / a.prompt_splits);
    }
    return u;
}

// A tile's pages.  Granule g is 16 tokens, or a page's share of the tile if
// that is more; lane g looks it up.  prompt_look only loads the lane's page
// number (-2 behind the sequence), so that a tile's can be on its way while the
// tile before is worked on; prompt_pages then gives the word in which bit g is
// set where granule g has a page of the cache.  The whole warp calls them.
__device__ __forceinline__ int prompt_look(const Kv4Attn& a, const PromptUnit& u, int j) {
    if (j >= u.t1) return -2;
    const int lane = threadIdx.x & 31;
    const int shift = a.cache.page_shift, gshift = shift < 7 ? shift : 7;
    const int tok = kv4_span_chunk(u.span, j) * kPromptTile + (lane << gshift);
    if ((lane << gshift) >= kPromptTile || tok >= u.q.len) return -2;
    return a.rows.table[static_cast<size_t>(u.b) * a.rows.width + (tok >> shift)];
}
__device__ __forceinline__ uint32_t prompt_pages(const Kv4Attn& a, int page) {
    return __ballot_sync(0xFFFFFFFFu, kv4_page_ok(a.cache, page));
}

// Whether every row of the unit sees the whole tile and all of it has pages.
__device__ __forceinline__ bool prompt_open(const Kv4Attn& a, const PromptUnit& u, int tok0, uint32_t pages) {
    const int gshift = a.cache.page_shift < 7 ? a.cache.page_shift : 7;
    const uint32_t all = (1u << (kPromptTile >> gshift)) - 1u;
    return pages == all && tok0 + kPromptTile <= u.q.len && tok0 + kPromptTile - 1 <= u.first_pos &&
           (a.window <= 0 || u.last_pos - tok0 < a.window || tok0 + kPromptTile <= a.sinks);
}

// Bits [lo, hi) of a word; lo and hi are any integers.
__device__ __forceinline__ uint32_t bit_range(int lo, int hi) {
    lo = max(lo, 0);
    hi = min(hi, 32);
    if (lo >= hi) return 0u;
    return (0xFFFFFFFFu >> (32 - (hi - lo))) << lo;
}

// Two FP32 operations in one instruction.
__device__ __forceinline__ uint64_t pack_f32x2(float lo, float hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ void fma_f32x2(float& x0, float& x1, float s0, float s1, uint64_t f, uint64_t c) {
    asm("{\n\t.reg .b64 s, r;\n\tmov.b64 s, {%2, %3};\n\tfma.rn.f32x2 r, s, %4, %5;\n\tmov.b64 {%0, %1}, r;\n\t}"
        : "=f"(x0), "=f"(x1) : "f"(s0), "f"(s1), "l"(f), "l"(c));
}
__device__ __forceinline__ void add_f32x2(float& a0, float& a1, float b0, float b1) {
    asm("{\n\t.reg .b64 a, b;\n\tmov.b64 a, {%0, %1};\n\tmov.b64 b, {%2, %3};\n\tadd.rn.f32x2 a, a, b;\n\t"
        "mov.b64 {%0, %1}, a;\n\t}"
        : "+f"(a0), "+f"(a1) : "f"(b0), "f"(b1));
}

// One pass over the thread's 64 scores: p = 2^(s f - m), hidden ones 0.
// Returns the largest s f - m; *sum gets the sum of p.
template <bool MASKED>
__device__ __forceinline__ float prompt_pass(uint32_t s_tmem, float f, float m, uint32_t mask0, uint32_t mask1,
                                             uint32_t (&p)[32], float* sum) {
    uint32_t s[2][32];
    tmem_ld_32x32b_x32(s_tmem, s[0]);
    tmem_ld_32x32b_x32(s_tmem + 32, s[1]);
    tmem_wait_ld();
    float top = -INFINITY, t0 = 0.0f, t1 = 0.0f;
    const uint64_t ff = pack_f32x2(f, f), mm = pack_f32x2(-m, -m);
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
            float x0, x1;
            fma_f32x2(x0, x1, __uint_as_float(s[c][i]), __uint_as_float(s[c][i + 1]), ff, mm);
            if constexpr (MASKED) {
                x0 = ((c ? mask1 : mask0) >> i) & 1u ? x0 : -INFINITY;
                x1 = ((c ? mask1 : mask0) >> (i + 1)) & 1u ? x1 : -INFINITY;
            }
            top = fmaxf(top, fmaxf(x0, x1));
            x0 = ex2(x0);
            x1 = ex2(x1);
            add_f32x2(t0, t1, x0, x1);
            p[16 * c + i / 2] = pack_half2(x0, x1);
        }
    *sum = t0 + t1;
    return top;
}

// The largest s f of the thread's row that is not hidden.
__device__ __noinline__ float prompt_top(uint32_t s_tmem, float f, uint32_t mask0, uint32_t mask1) {
    float top = -INFINITY;
#pragma unroll 1
    for (int c = 0; c < 4; ++c) {
        uint32_t s[16];
        tmem_ld_32x32b_x16(s_tmem + 16 * c, s);
        tmem_wait_ld();
        const uint32_t w = (c < 2 ? mask0 : mask1) >> (16 * (c & 1));
#pragma unroll
        for (int i = 0; i < 16; ++i) top = fmaxf(top, (w >> i) & 1u ? __uint_as_float(s[i]) * f : -INFINITY);
    }
    return top;
}

// Queries of a warp's 32 rows of tile t on their way: D / 8 lanes load a row.
template <class C>
struct PromptQ {
    static constexpr int LANES = C::D / 8, AT_ONCE = 32 / LANES, N = 32 / AT_ONCE;
    uint4 v[N];
};

template <class C>
__device__ __forceinline__ void prompt_q_load(const Kv4Attn& a, const PromptUnit& u, int r0, PromptQ<C>& q) {
    using Q = PromptQ<C>;
    const int lane = threadIdx.x & 31, k = lane % Q::LANES;  // 16-byte chunk of the row
    r0 += lane / Q::LANES;
    int to = (u.row_base + r0) / a.group, head = (u.row_base + r0) - to * a.group;  // of the lane's row
    const int to_step = Q::AT_ONCE / a.group, head_step = Q::AT_ONCE - to_step * a.group;
    const uint16_t* src = static_cast<const uint16_t*>(a.q) + u.q.first * a.q_stride +
                          static_cast<long long>(u.head) * a.group * C::D + 8 * k;
#pragma unroll
    for (int x = 0; x < Q::N; ++x) {
        q.v[x] = make_uint4(0u, 0u, 0u, 0u);
        if (r0 + x * Q::AT_ONCE < u.row_count)
            q.v[x] = *reinterpret_cast<const uint4*>(src + to * a.q_stride + head * C::D);
        to += to_step;
        head += head_step;
        if (head >= a.group) head -= a.group, ++to;
    }
}

// ... and into the tile, pairs swapped; BF16 scaled and the sign of the factor
// moved as in the step kernel.  `scale` gets the rows' factors.
template <class C, bool BF16>
__device__ __forceinline__ void prompt_q_store(const Kv4Attn& a, const PromptQ<C>& q, uint8_t* tile, int r0,
                                               float* scale) {
    using Q = PromptQ<C>;
    const int lane = threadIdx.x & 31, k = lane % Q::LANES;
    const uint32_t sign = a.scale_log2 < 0.0f ? 0x80008000u : 0u;
#pragma unroll
    for (int x = 0; x < Q::N; ++x) {
        const int rr = r0 + x * Q::AT_ONCE + lane / Q::LANES;
        uint32_t w[4] = {q.v[x].x, q.v[x].y, q.v[x].z, q.v[x].w};
        float f = fabsf(a.scale_log2);
        if constexpr (BF16) {
            uint32_t e = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) e = max(e, max((w[j] >> 7) & 0xFFu, (w[j] >> 23) & 0xFFu));
#pragma unroll
            for (int d = 1; d < Q::LANES; d <<= 1) e = max(e, __shfl_xor_sync(0xFFFFFFFFu, e, d));
            const int kk = e == 255u ? -113 : 141 - static_cast<int>(e), k1 = kk > 120 ? 120 : kk, k2 = kk - k1;
            const float up = exp2i(k1), up2 = exp2i(k2);
            f = (f * exp2i(-k1)) * exp2i(-k2);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                w[j] = pack_half2(__uint_as_float(w[j] & 0xFFFF0000u) * up * up2, __uint_as_float(w[j] << 16) * up * up2);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = prmt(w[j], 0u, 0x1032u);
        }
        if (k == 0) scale[rr] = kv4_row_factor(f);
        *reinterpret_cast<uint4*>(tile + (k / 8) * C::PANEL + rr * 128 + (((k & 7) ^ (rr & 7)) << 4)) =
            make_uint4(w[0] ^ sign, w[1] ^ sign, w[2] ^ sign, w[3] ^ sign);
    }
}

// Where tile t's thread r of an item belongs.
struct PromptRow {
    bool valid;
    int pos, at, head;  // position; row of the caller's arrays; query head
};
__device__ __forceinline__ PromptRow prompt_row(const Kv4Attn& a, const PromptUnit& u, int r) {
    PromptRow p;
    const int row = u.row_base + r, i = row / a.group;
    p.valid = r < u.row_count;
    p.pos = u.q.pos0 + i;
    p.at = u.q.first + i;
    p.head = u.head * a.group + row - i * a.group;
    return p;
}

// Rare: the blocks of 16 values d in which a row at position pos sees a NaN of V
// that was left out of the products: those of tiles that the unit's rows do not
// all see whole.  (All tiles looked through, a chunk of 8192 packed rows behind
// 262144 tokens took 58.6 ms with one NaN at its end, 8.0 ms like this, as without it.)
template <int D>
__device__ __noinline__ uint32_t prompt_nan_blocks(const Kv4Attn& a, const int* list, int seqs, int item, int pos) {
    const PromptUnit u = prompt_unit(a, list, seqs, item);
    const int shift = a.cache.page_shift, gshift = shift < 7 ? shift : 7;
    const int* table = a.rows.table + static_cast<size_t>(u.b) * a.rows.width;
    uint32_t found = 0;
    for (int j = u.t0; j < u.t1; ++j) {
        const int tok0 = kv4_span_chunk(u.span, j) * kPromptTile;
        uint32_t pages = 0;  // as prompt_pages gives them
        for (int k = 0; k < (kPromptTile >> gshift); ++k) {
            const int tok = tok0 + (k << gshift);
            if (tok < u.q.len && kv4_page_ok(a.cache, table[tok >> shift])) pages |= 1u << k;
        }
        if (prompt_open(a, u, tok0, pages)) continue;
        for (int k = 0; k < kPromptTile; ++k) {
            const int tok = tok0 + k;
            if (!((pages >> (k >> gshift)) & 1u) || tok >= u.q.len || !kv4_sees(pos, tok, a.window, a.sinks)) continue;
            const uint8_t* sc = a.cache.data + kv4_block_offset(a.cache, table[tok >> shift], u.head) +
                                2 * kv4_codes_bytes(a.cache) + kv4_scales_bytes(a.cache) +
                                (tok & ((1 << shift) - 1)) * (D / 16);
            for (int x = 0; x < D / 16; ++x)
                if ((sc[x] & 0x7F) == 0x7F) found |= 1u << x;
        }
    }
    return found;
}

template <class C, bool BF16, bool DRAWN>
__global__ void __launch_bounds__(kPromptThreads, 1) k_kv4_prompt(const __grid_constant__ Kv4Attn a) {
    constexpr int D = C::D;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (smem_addr(smem_raw) & 1023u)) & 1023u);
    uint64_t* raw_full = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);
    uint64_t* raw_empty = raw_full + C::NR;
    uint64_t* op_full = raw_empty + C::NR;
    uint64_t* op_empty = op_full + C::SLOTS;
    uint64_t* s_full = op_empty + C::SLOTS;
    uint64_t* p_full = s_full + 2;           // [tile of rows][half of the tokens]
    uint64_t* pv_half = p_full + 4;          // P V of the first half has ended
    uint64_t* o_full = pv_half + 2;
    uint64_t* q_full = o_full + 2;
    uint64_t* drain = q_full + 2;
    uint64_t* item_full = drain + 1;         // a ring of four item numbers
    uint64_t* item_empty = item_full + 4;
    uint32_t* tmem_ptr = reinterpret_cast<uint32_t*>(item_empty + 4);
    volatile int* abort = reinterpret_cast<volatile int*>(tmem_ptr + 1);
    volatile int* nan_seen = abort + 1;  // some item's V had a NaN block left out
    volatile int* ring = nan_seen + 1;   // items by round & 3, -1 behind the last
    int* warp_sums = const_cast<int*>(ring) + 4;  // 20
    float* q_scale = reinterpret_cast<float*>(smem + C::OFF_QSCALE);  // score -> log2 units, per row

    // A value that a shuffle or a vote gives is the same in the whole warp for
    // the compiler too, which then keeps what follows from it in uniform
    // registers: MMAs are issued from those.
    const int tid = threadIdx.x, warp = __shfl_sync(0xFFFFFFFFu, tid / 32, 0), lane = tid & 31;
    if (tid == 0) {
        for (int i = 0; i < C::NR; ++i) {
            mbar_init(&raw_full[i], 1);
            mbar_init(&raw_empty[i], 8);
        }
        for (int i = 0; i < C::SLOTS; ++i) {
            mbar_init(&op_full[i], 8);
            mbar_init(&op_empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[2 * i], 4);
            mbar_init(&p_full[2 * i + 1], 4);
            mbar_init(&pv_half[i], 1);
            mbar_init(&o_full[i], 1);
            mbar_init(&q_full[i], 4);
        }
        mbar_init(drain, 1);
        for (int i = 0; i < 4; ++i) {
            mbar_init(&item_full[i], 1);
            mbar_init(&item_empty[i], 17);
        }
        fence_barrier_init();
        *abort = 0;
        *nan_seen = 0;
    }
    if (warp == 16) tmem_alloc(tmem_ptr, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_ptr;

    int seqs = a.rows.batch;
    int* list = nullptr;
    if (DRAWN && a.rows.batch <= kPromptBatch) {  // more do not fit: then all are gone through
        list = reinterpret_cast<int*>(smem + C::OFF_LIST);
        seqs = 0;
        for (int b0 = 0; b0 < a.rows.batch; b0 += kPromptThreads) {
            const int b = b0 + tid;
            const bool here = b < a.rows.batch && prompt_takes(a, kv4_rows_seq(a.rows, a.cache.page_shift, a.rows.cu[b],
                                                                          a.rows.cu[b + 1], a.rows.lens[b]));
            const uint32_t some = __ballot_sync(0xFFFFFFFFu, here);
            if (lane == 0) warp_sums[warp] = __popc(some);
            __syncthreads();
            int before = seqs + __popc(some & ((1u << lane) - 1u));
            for (int k = 0; k < kPromptThreads / 32; ++k) {
                if (k < warp) before += warp_sums[k];
                seqs += warp_sums[k];
            }
            if (here) list[before] = b;
            __syncthreads();
        }
    }
    const int items = seqs * a.cache.heads * a.prompt_tiles * a.prompt_splits;
    // The next item (-1: none); `round` counts those that the warp has had.
    uint32_t round = 0;
    auto take_item = [&]() {
        int item = -1;
        if constexpr (DRAWN) {
            if (__all_sync(0xFFFFFFFFu, mbar_wait(&item_full[round & 3], (round >> 2) & 1, abort))) {
                item = ring[round & 3];
                __syncwarp();
                if (lane == 0) mbar_arrive(&item_empty[round & 3]);
            }
        } else {  // there and back through the items, so that the CTAs' sums are alike
            item = static_cast<int>(round * gridDim.x + (round & 1 ? gridDim.x - 1 - blockIdx.x : blockIdx.x));
            if (item >= items) item = -1;
        }
        ++round;
        return item;
    };

    const int gshift = a.cache.page_shift < 7 ? a.cache.page_shift : 7;
    const uint32_t gtok = 1u << gshift;
    const uint32_t at_ks = gtok * (D / 2), at_vc = at_ks + gtok * (D / 16), at_vs = at_vc + gtok * (D / 2);
    const uint32_t gbytes = gtok * C::TOKEN_BYTES * 2;

    if (warp < 8) {
        reg_inc<C::REGS_SOFTMAX>();
        // ---- softmax: thread = row ----------------------------------------------------
        const int t = warp / 4, r = tid & 127;
        const uint32_t quarter = static_cast<uint32_t>(warp & 3) << 21;  // lane offset 32 * (warp % 4)
        const uint32_t s_tmem = tmem + quarter + t * C::S_COLS;
        const uint32_t o_tmem = tmem + quarter + C::O_COL + t * D;
        uint32_t s_phase = 0, o_phase = 0;
        bool ok = true;
        const int warp_row = (warp & 3) * 32;  // first of the warp's rows in the tile
        uint8_t* q_tile = smem + t * C::OPERAND;
        // The next item with rows for this tile; -1: none.
        auto find = [&](PromptUnit& u) {
            for (;;) {
                const int item = take_item();
                if (item < 0) return -1;
                u = prompt_unit(a, list, seqs, item);
                if (u.t0 < u.t1 && u.row_count > t * 128) return item;
            }
        };
        auto give_q = [&](const PromptQ<C>& q) {
            prompt_q_store<C, BF16>(a, q, q_tile, warp_row, q_scale + t * 128);
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&q_full[t]);
        };
        PromptUnit u;
        int item = find(u);
        if (item >= 0) {
            PromptQ<C> q;
            prompt_q_load<C>(a, u, t * 128 + warp_row, q);
            give_q(q);
        }
        while (item >= 0 && ok) {
            const PromptRow row = prompt_row(a, u, t * 128 + r);
            const int pos = row.pos;
            const float f = q_scale[t * 128 + r];  // written by this warp
            float m = kNoMax, l = 0.0f;
            int page = prompt_look(a, u, u.t0);
            for (int j = u.t0; j < u.t1; ++j) {
                const int tok0 = kv4_span_chunk(u.span, j) * kPromptTile;
                const uint32_t pages = prompt_pages(a, page);
                const bool open = prompt_open(a, u, tok0, pages);
                page = prompt_look(a, u, j + 1);
                uint32_t mask[4];
                if (!open) {
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const int base = tok0 + 32 * c;
                        uint32_t w = bit_range(0, min(pos + 1, u.q.len) - base);
                        if (a.window > 0) {
                            const int oldest = pos >= a.window ? pos - a.window + 1 : 0;
                            w &= bit_range(oldest - base, 32) | bit_range(0, a.sinks - base);
                        }
                        uint32_t there = 0;
#pragma unroll
                        for (int k = 0; k < 2; ++k)
                            if ((pages >> ((32 * c + 16 * k) >> gshift)) & 1u) there |= 0xFFFFu << (16 * k);
                        mask[c] = w & there;
                    }
                }
                ok = __all_sync(0xFFFFFFFFu, mbar_wait(&s_full[t], s_phase, abort));
                if (!ok) break;
                s_phase ^= 1u;
                tc_fence_after();  // S_t is there, and O_t at rest: its last P V came before
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const uint32_t s_half = s_tmem + 64 * half;
                    const uint32_t m0 = open ? 0xFFFFFFFFu : mask[2 * half], m1 = open ? 0xFFFFFFFFu : mask[2 * half + 1];
                    uint32_t p[32];
                    float sum;
                    float top = INFINITY;  // the item's first scores only set m
                    if (half == 1 || j > u.t0)
                        top = open ? prompt_pass<false>(s_half, f, m, m0, m1, p, &sum)
                                   : prompt_pass<true>(s_half, f, m, m0, m1, p, &sum);
                    const bool move = top > kPMost;
                    if (__any_sync(0xFFFFFFFFu, move)) {
                        // The row's largest score, found anew: s f - m has lost
                        // it where m was kNoMax.  m stays a whole number, so
                        // that what is scaled by its steps is not rounded.
                        const float y = ceilf(prompt_top(s_half, f, m0, m1)) - kPSet;
                        const float m_new = move ? fmaxf(m, y) : m;  // the warp's other rows go through the same values again
                        const float step = m_new - m;
                        const float scale = step < 126.0f ? exp2i(-static_cast<int>(step)) : 0.0f;
                        m = m_new;
                        l *= scale;
                        if (open) prompt_pass<false>(s_half, f, m, m0, m1, p, &sum);
                        else prompt_pass<true>(s_half, f, m, m0, m1, p, &sum);
                        if (half == 1) {  // O at rest again: P V of the first half has ended
                            ok = __all_sync(0xFFFFFFFFu, mbar_wait(&pv_half[t], s_phase ^ 1u, abort));
                            tc_fence_after();
                        }
                        if (half == 1 || j > u.t0) {
#pragma unroll 1
                            for (int c = 0; c < D; c += 16) {
                                uint32_t o[16];
                                tmem_ld_32x32b_x16(o_tmem + c, o);
                                tmem_wait_ld();
#pragma unroll
                                for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * scale);
                                tmem_st_32x32b_x16(o_tmem + c, o);
                            }
                        }
                    }
                    l += sum;
                    tmem_st_32x32b_x32(s_tmem + 32 * half, p);  // over scores that have been read
                    tmem_wait_st();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&p_full[2 * t + half]);
                }
            }

            // ---- the rows' result ----------------------------------------------------------
            PromptUnit un;
            const int item_next = find(un);
            ok = __all_sync(0xFFFFFFFFu, ok && mbar_wait(&o_full[t], o_phase, abort));
            o_phase ^= 1u;
            if (!ok) break;
            tc_fence_after();
            uint32_t nan_blocks = 0;
            if (*nan_seen && row.valid) nan_blocks = prompt_nan_blocks<D>(a, list, seqs, item, pos);
            const bool partial = a.prompt_splits > 1;
            const float g = partial ? 1.0f : l == 0.0f ? 0.0f : a.cache.v_scale / l;
            // The warp's 32 rows go through its part of the query tile (whose
            // products have ended), D / 8 chunks of 16 bytes of a row at a time,
            // chunk x at x ^ (row & 7) of its panel, so that they leave in whole
            // lines: with a row a thread this took 5 us an item.
            const uint32_t slot = partial ? prompt_slot(a, u, u.split) : 0u;
            uint8_t* stage = q_tile + warp_row * 128;
            uint16_t* out = static_cast<uint16_t*>(a.out) + static_cast<long long>(u.head) * a.group * D +
                            8 * (lane % PromptQ<C>::LANES);
            const int width = partial ? D / 2 : D;  // columns of a pass
            for (int col = 0; col < D; col += width) {
                auto put = [&](int x, uint4 v) {
                    *reinterpret_cast<uint4*>(stage + (x >> 3) * C::PANEL + lane * 128 + (((x & 7) ^ (lane & 7)) << 4)) = v;
                };
#pragma unroll 1
                for (int c = 0; c < width; c += 32) {
                    uint32_t o[32];  // columns come in swapped pairs
                    tmem_ld_32x32b_x32(o_tmem + col + c, o);
                    tmem_wait_ld();
                    if (nan_blocks) {
#pragma unroll
                        for (int k = 0; k < 32; ++k)
                            if ((nan_blocks >> ((col + c + k) / 16)) & 1u) o[k] = 0x7FC00000u;
                    }
                    if (partial) {
#pragma unroll
                        for (int k = 0; k < 8; ++k)
                            put(c / 4 + k, make_uint4(o[4 * k + 1], o[4 * k], o[4 * k + 3], o[4 * k + 2]));
                    } else {
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            uint32_t w[4];
#pragma unroll
                            for (int y = 0; y < 4; ++y) {
                                float lo = __uint_as_float(o[8 * k + 2 * y + 1]) * g;
                                float hi = __uint_as_float(o[8 * k + 2 * y]) * g;
                                if (l == 0.0f) lo = hi = 0.0f;
                                if constexpr (BF16) {
                                    const __nv_bfloat162 z = __floats2bfloat162_rn(lo, hi);
                                    w[y] = *reinterpret_cast<const uint32_t*>(&z);
                                } else {
                                    w[y] = pack_half2(lo, hi);
                                }
                            }
                            put(c / 8 + k, make_uint4(w[0], w[1], w[2], w[3]));
                        }
                    }
                }
                __syncwarp();
                using Q = PromptQ<C>;
                const int x = lane % Q::LANES;
                int rr = lane / Q::LANES;
                const PromptRow first = prompt_row(a, u, t * 128 + warp_row + rr);
                int at = first.at, head = first.head - u.head * a.group;
                const int at_step = Q::AT_ONCE / a.group, head_step = Q::AT_ONCE - at_step * a.group;
#pragma unroll 1
                for (int part = 0; part < 2; ++part) {
                    uint4 v[Q::N / 2];
#pragma unroll
                    for (int k = 0; k < Q::N / 2; ++k)
                        v[k] = *reinterpret_cast<const uint4*>(stage + (x >> 3) * C::PANEL + (rr + k * Q::AT_ONCE) * 128 +
                                                               (((x & 7) ^ ((rr + k * Q::AT_ONCE) & 7)) << 4));
#pragma unroll
                    for (int k = 0; k < Q::N / 2; ++k) {
                        const int tr = t * 128 + warp_row + rr;
                        if (tr < u.row_count) {
                            if (partial)
                                *reinterpret_cast<uint4*>(a.prompt_ws + static_cast<size_t>(slot + tr) * D + col + 4 * x) = v[k];
                            else
                                *reinterpret_cast<uint4*>(out + at * a.out_stride + head * D) = v[k];
                        }
                        rr += Q::AT_ONCE;
                        at += at_step;
                        head += head_step;
                        if (head >= a.group) head -= a.group, ++at;
                    }
                }
                __syncwarp();
            }
            PromptQ<C> q;
            if (item_next >= 0) prompt_q_load<C>(a, un, t * 128 + warp_row, q);
            if (row.valid && partial) {
                float* at = prompt_m<C>(a) + slot + t * 128 + r;
                at[0] = m;
                at[prompt_m_to_l(a)] = l;
            } else if (row.valid && a.lse != nullptr) {
                a.lse[static_cast<long long>(row.at) * a.q_heads + row.head] =
                    l == 0.0f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
            }
            tc_fence_before();  // O has been read before the next item's P is announced
            if (item_next >= 0) give_q(q);
            u = un;
            item = item_next;
        }
    } else if (warp < 16) {
        reg_dec<C::REGS_DECODE>();
        // ---- decode: thread = half of a token's values, K tile and V tile in turn ---------
        const uint32_t tok = static_cast<uint32_t>(tid & 127), half = (warp - 8) / 4;
        const uint32_t g0 = (tok >> gshift) * gbytes, place = tok & (gtok - 1u);
        constexpr int PARTS = D / 64;  // 16-byte parts of the thread's codes: 32 values, two scales each
        int rs = 0, slot = 0;
        uint32_t r_phase = 0, op_phase = 1;  // of the empty slot: the first round passes at once
        bool ok = true;
        for (int item = take_item(); item >= 0 && ok; item = take_item()) {
            const PromptUnit u = prompt_unit(a, list, seqs, item);
            int page = prompt_look(a, u, u.t0);
            for (int j = u.t0; j < u.t1; ++j) {
                const int tok0 = kv4_span_chunk(u.span, j) * kPromptTile;
                const uint32_t pages = prompt_pages(a, page);
                const bool open = prompt_open(a, u, tok0, pages);
                page = prompt_look(a, u, j + 1);
                const bool there = ((pages >> (tok >> gshift)) & 1u) && tok0 + static_cast<int>(tok) < u.q.len;
                ok = __all_sync(0xFFFFFFFFu, mbar_wait(&raw_full[rs], r_phase, abort));
                if (!ok) break;
                const uint8_t* raw = smem + C::OFF_RAW + rs * C::RAW + g0;
#pragma unroll 1
                for (int kv = 0; kv < 2; ++kv) {
                    const uint8_t* codes = raw + (kv ? at_vc : 0u) + place * (D / 2) + half * (D / 4);
                    const uint8_t* scales = raw + (kv ? at_vs : at_ks) + place * (D / 16) + half * (D / 32);
                    uint4 v[PARTS];
                    // Lanes start at different parts, so that the writes of a
                    // quarter warp fall into different banks.
#pragma unroll
                    for (int x = 0; x < PARTS; ++x)
                        v[x] = *reinterpret_cast<const uint4*>(codes + 16 * ((x + (tok >> 1)) & (PARTS - 1)));
                    uint32_t sc;
                    if constexpr (D == 128) sc = *reinterpret_cast<const uint32_t*>(scales);
                    else sc = *reinterpret_cast<const uint16_t*>(scales);
                    if (!there) sc = 0u;
                    if (kv && !open && e4m3_nan_bits(sc)) {
                        // A NaN block that some row may not see: out of the
                        // product, and into the rows that see it at the end.
                        *nan_seen = 1;
                        __threadfence_block();
                        sc &= ~((e4m3_nan_bits(sc) >> 7) * 0xFFu);
                    }
                    ok = __all_sync(0xFFFFFFFFu, mbar_wait(&op_empty[slot], op_phase, abort));
                    if (!ok) break;
                    uint8_t* dst = smem + C::OFF_SLOT + slot * C::OPERAND + tok * 128;
#pragma unroll
                    for (int x = 0; x < PARTS; ++x) {
                        const uint32_t part = (x + (tok >> 1)) & (PARTS - 1);
                        const uint32_t w[4] = {v[x].x, v[x].y, v[x].z, v[x].w};
                        const uint32_t ss = cvt_e4m3x2(static_cast<uint16_t>(sc >> (16 * part)));
                        const uint32_t sa = prmt(ss, 0u, 0x1010u), sb = prmt(ss, 0u, 0x3232u);
#pragma unroll
                        for (int y = 0; y < 4; ++y) {
                            uint32_t o[4];
                            cvt_e2m1x2_x4(w[y], o);
#pragma unroll
                            for (int z = 0; z < 4; ++z) o[z] = hmul2(o[z], y < 2 ? sa : sb);
                            const uint32_t chunk = (D / 16) * half + 4 * part + y;  // 16-byte chunk of the decoded row
                            *reinterpret_cast<uint4*>(dst + (chunk >> 3) * C::PANEL + (((chunk & 7u) ^ (tok & 7u)) << 4)) =
                                make_uint4(o[0], o[1], o[2], o[3]);
                        }
                    }
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) {
                        mbar_arrive(&op_full[slot]);
                        if (kv) mbar_arrive(&raw_empty[rs]);
                    }
                    if (++slot == C::SLOTS) slot = 0, op_phase ^= 1u;
                }
                if (!ok) break;
                if (++rs == C::NR) rs = 0, r_phase ^= 1u;
            }
        }
    } else {
      reg_dec<C::REGS_REST>();
      if (warp == 16) {
        // ---- tensor core: the warp waits, one lane issues ---------------------------------
        // All 512 columns are this CTA's, so its tensor memory starts at column 0.
        constexpr uint32_t idesc_s = idesc_make(0, 0, 128, 128);
        constexpr uint32_t idesc_o = idesc_make(0, 0, 128, D) | (1u << 16);  // V is N-major
        const uint32_t q_lo = sdesc_lo(smem_addr(smem));
        const uint32_t k_lo = sdesc_lo(smem_addr(smem + C::OFF_SLOT)), v_lo = sdesc_v_lo<C>(smem_addr(smem + C::OFF_SLOT));
        bool ok = __all_sync(0xFFFFFFFFu, tmem == 0u);
        if (!ok && lane == 0) {
            atomicOr(&g_tb_device_error, kErrTimeout);
            *abort = 1;
        }
        auto wait = [&](uint64_t* bar, uint32_t parity) {
            ok = __all_sync(0xFFFFFFFFu, ok && mbar_wait(bar, parity, abort));
            tc_fence_after();
            return ok;
        };
        // S_t = Q_t K^T with the K tile in `slot`.
        auto scores = [&](int t, uint32_t slot) {
            const uint32_t ql = q_lo + t * (C::OPERAND >> 4), kl = k_lo + slot * (C::OPERAND >> 4);
#pragma unroll
            for (int k = 0; k < D / 16; ++k) {
                const uint32_t at = ((k / 4) * C::PANEL + (k % 4) * 32) >> 4;
                mma_f16_ss(t * C::S_COLS, sdesc_make(ql + at), sdesc_make(kl + at), idesc_s, k > 0);
            }
            mma_commit(&s_full[t]);
        };
        // O_t += P_t V of half the tokens.
        auto values = [&](int t, uint32_t slot, int half, uint32_t accumulate) {
            const uint32_t vl = v_lo + slot * (C::OPERAND >> 4);
#pragma unroll
            for (int x = 0; x < kPromptTile / 32; ++x) {
                const int k = half * (kPromptTile / 32) + x;
                mma_f16_ts(C::O_COL + t * D, t * C::S_COLS + 8 * k, sdesc_make(vl + k * (2048 >> 4)), idesc_o,
                           x > 0 ? 1u : accumulate);
            }
        };
        int slot = 0;  // operands take the slots in turn: K_0, V_0, K_1, V_1, ...
        uint32_t op_phase = 0, p_phase0 = 0, p_phase1 = 0, q_phase0 = 0, q_phase1 = 0;
        auto next = [&]() {
            if (++slot == C::SLOTS) slot = 0, op_phase ^= 1u;
        };
        for (int item = take_item(); item >= 0 && ok; item = take_item()) {
            const PromptUnit u = prompt_unit(a, list, seqs, item);
            const int n = __reduce_max_sync(0xFFFFFFFFu, u.t1 - u.t0);
            if (n == 0) continue;
            const bool two = __any_sync(0xFFFFFFFFu, u.row_count > 128);
            if (!wait(&q_full[0], q_phase0)) break;
            q_phase0 ^= 1u;
            if (two) {
                if (!wait(&q_full[1], q_phase1)) break;
                q_phase1 ^= 1u;
            }
            if (!wait(&op_full[slot], op_phase)) break;
            if (elect_one()) {
                scores(0, slot);
                if (two) scores(1, slot);
                mma_commit(&op_empty[slot]);
            }
            __syncwarp();
            next();
            for (int j = 0; j < n; ++j) {
                const bool more = j + 1 < n;
                const int v_slot = slot;
                if (!wait(&op_full[slot], op_phase)) break;
                next();
                if (!wait(&p_full[0], p_phase0)) break;
                if (elect_one()) {
                    values(0, v_slot, 0, j > 0);
                    mma_commit(&pv_half[0]);
                }
                __syncwarp();
                if (!wait(&p_full[1], p_phase0)) break;
                p_phase0 ^= 1u;
                if (elect_one()) {
                    values(0, v_slot, 1, 1u);
                    if (!two) mma_commit(&op_empty[v_slot]);
                    if (!more) mma_commit(&o_full[0]);
                }
                __syncwarp();
                if (more) {
                    if (!wait(&op_full[slot], op_phase)) break;
                    if (elect_one()) {
                        scores(0, slot);
                        if (!two) mma_commit(&op_empty[slot]);
                    }
                    __syncwarp();
                }
                if (two) {
                    if (!wait(&p_full[2], p_phase1)) break;
                    if (elect_one()) {
                        values(1, v_slot, 0, j > 0);
                        mma_commit(&pv_half[1]);
                    }
                    __syncwarp();
                    if (!wait(&p_full[3], p_phase1)) break;
                    p_phase1 ^= 1u;
                    if (elect_one()) {
                        values(1, v_slot, 1, 1u);
                        mma_commit(&op_empty[v_slot]);
                        if (more) {
                            scores(1, slot);
                            mma_commit(&op_empty[slot]);
                        } else {
                            mma_commit(&o_full[1]);
                        }
                    }
                    __syncwarp();
                }
                if (more) next();
            }
        }
        if (!ok && lane == 0) {  // let what was issued end before the tensor memory is given up
            mma_commit(drain);
            mbar_wait_drain(drain, 0);
        }
        __syncwarp();
      } else if (warp == 17) {
        // ---- loader ---------------------------------------------------------------------------
        int rs = 0;
        uint32_t r_phase = 1, filled = 0;  // of the empty stage: the first round passes at once
        bool ok = true;
        // The first item is the CTA's own, later ones are drawn from the
        // counter, which the step kernel set to 0.
        auto draw = [&](int item) {
            if constexpr (DRAWN) {
                if (item < 0) {
                    item = blockIdx.x;
                } else {
                    if (round < 2) grid_dep_wait();
                    if (lane == 0) item = static_cast<int>(gridDim.x) + atomicAdd(a.ticket, 1);
                    item = __shfl_sync(0xFFFFFFFFu, item, 0);
                }
                return item < items ? item : -1;
            } else {
                return take_item();
            }
        };
        auto publish = [&](int item) {
            if constexpr (DRAWN) {
                ok = __all_sync(0xFFFFFFFFu, ok && mbar_wait(&item_empty[round & 3], ((round >> 2) & 1) ^ 1u, abort));
                if (lane == 0 && ok) {
                    ring[round & 3] = item;
                    mbar_arrive(&item_full[round & 3]);
                }
                __syncwarp();
                ++round;
            }
        };
        for (int item = draw(-1); item >= 0 && ok; item = draw(item)) {
            const PromptUnit u = prompt_unit(a, list, seqs, item);
            if (lane == 0 && u.any) {
                if (u.q.bad) atomicOr(&g_tb_device_error, kErrPage);
                if (static_cast<long long>(u.q.n) * a.group > static_cast<long long>(a.prompt_tiles) * kPromptRows)
                    atomicOr(&g_tb_device_error, kErrRows);
            }
            if (u.t0 == u.t1) continue;
            publish(item);
            const int oldest = a.window > 0 && u.first_pos >= a.window ? u.first_pos - a.window + 1 : 0;
            int after = prompt_look(a, u, u.t0);
            for (int j = u.t0; j < u.t1; ++j) {
                const int tok0 = kv4_span_chunk(u.span, j) * kPromptTile;
                const int page = after;
                const uint32_t pages = prompt_pages(a, page);
                after = prompt_look(a, u, j + 1);
                ok = __all_sync(0xFFFFFFFFu, mbar_wait(&raw_empty[rs], r_phase, abort));
                if (!ok) break;
                uint8_t* dst = smem + C::OFF_RAW + rs * C::RAW;
                const int want = min(kPromptTile, u.q.len - tok0);  // tokens that should have pages
                const bool mine = (pages >> lane) & 1u;
                // Pages out of every row's sight may be gone.
                const int upto = tok0 + ((lane + 1) << gshift);
                const bool seen = upto > oldest || upto - static_cast<int>(gtok) < a.sinks;
                if ((lane << gshift) < want && !mine && seen) atomicOr(&g_tb_device_error, kErrPage);
                if (lane == 0) mbar_arrive_expect_tx(&raw_full[rs], __popc(pages) * gbytes);
                __syncwarp();
                if (mine) {
                    const uint8_t* src = a.cache.data + kv4_block_offset(a.cache, page, u.head);
                    uint8_t* to = dst + lane * gbytes;
                    if (a.cache.page_shift <= 7) {
                        bulk_load(to, src, gbytes, &raw_full[rs]);
                    } else {  // a tile of a larger page, part by part (lane 0 alone)
                        const uint32_t place_in_page = static_cast<uint32_t>(tok0) & ((1u << a.cache.page_shift) - 1u);
                        const uint32_t codes = kv4_codes_bytes(a.cache), scales = kv4_scales_bytes(a.cache);
                        bulk_load(to, src + place_in_page * (D / 2), at_ks, &raw_full[rs]);
                        bulk_load(to + at_ks, src + codes + place_in_page * (D / 16), gtok * (D / 16), &raw_full[rs]);
                        src += codes + scales;
                        bulk_load(to + at_vc, src + place_in_page * (D / 2), at_ks, &raw_full[rs]);
                        bulk_load(to + at_vs, src + codes + place_in_page * (D / 16), gtok * (D / 16), &raw_full[rs]);
                    }
                }
                __syncwarp();
                ++filled;
                if (++rs == C::NR) rs = 0, r_phase ^= 1u;
            }
        }
        publish(-1);
        if (!ok && lane == 0)  // copies in flight end before the memory is given up
            for (int k = 0; k < C::NR && filled > 0; ++k, --filled) {
                if (--rs < 0) rs = C::NR - 1, r_phase ^= 1u;
                mbar_wait_drain(&raw_full[rs], r_phase ^ 1u);
            }
      }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 16) {
        tc_fence_after();
        tmem_relinquish();
        tmem_dealloc(tmem, 512);
    }
    grid_dep_wait();
}

// Joins the splits of the prompt kernel's rows, in their order: 256 / D packed
// rows of KV head blockIdx.y to a CTA.
template <class C, bool BF16>
__global__ void __launch_bounds__(256) k_kv4_prompt_join(const Kv4Attn a) {
    constexpr int D = C::D, LANES = D / 4, ROWS = 64 / LANES;
    __shared__ int seq[ROWS];
    const int row0 = blockIdx.x * ROWS;
    if (a.rows.batch > 1) {  // one needs no search, a trip to memory less
        if (threadIdx.x < ROWS) seq[threadIdx.x] = -1;
        __syncthreads();
        for (int b = threadIdx.x; b < a.rows.batch; b += blockDim.x) {
            const int c0 = a.rows.cu[b], c1 = a.rows.cu[b + 1];
            for (int i = 0; i < ROWS; ++i) {
                const int at = (row0 + i) / a.group;
                if (c0 <= at && at < c1) seq[i] = b;
            }
        }
        __syncthreads();
    }
    const int quarter = threadIdx.x / 64, item = threadIdx.x % 64, d = 4 * (item % LANES);
    const int b = a.rows.batch > 1 ? seq[item / LANES] : 0, row = row0 + item / LANES;
    PromptUnit u;
    int r = 0;  // row of the unit
    u.any = false;
    if (b >= 0 && row < a.rows.rows * a.group) {
        const Kv4Seq q = kv4_rows_seq(a.rows, a.cache.page_shift, a.rows.cu[b], a.rows.cu[b + 1], a.rows.lens[b]);
        const int packed = row - q.first * a.group, tile = packed / kPromptRows;
        r = packed - tile * kPromptRows;
        u.any = packed >= 0 && packed < q.n * a.group && tile < a.prompt_tiles;
        if (u.any) u = prompt_rows(a, b, blockIdx.y, tile);
    }
    if (!__syncthreads_or(u.any)) return;
    float top = kNoMax, l = 0.0f;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (u.any) {
        const long long tiles = u.t1;
        const float* ml = prompt_m<C>(a);
        const size_t to_l = prompt_m_to_l(a);
#pragma unroll 4
        for (int s = quarter; s < a.prompt_splits; s += 4) {
            if (tiles * s / a.prompt_splits == tiles * (s + 1) / a.prompt_splits) continue;  // no tiles, no result
            const size_t at = prompt_slot(a, u, s) + static_cast<uint32_t>(r);
            kv4_merge(top, l, v, ml[at], ml[at + to_l], *reinterpret_cast<const float4*>(a.prompt_ws + at * D + d));
        }
    }
    join_and_store<BF16, D>(a, u.any, u.q.first, u.row_base + r, u.head, d, top, l, v);
}

}  // namespace tb
