// kv4_cache_kernel.cuh -- rows of keys and values into a paged cache of
// block-scaled FP4, and back.
//
//   append  per (row, head) and block of 16 values x, with g the tensor's
//           scale:  s = the E4M3 value nearest to max|x| / (6 g), ties to the
//           smaller, 448 at most;  code = the E2M1 value nearest to
//           x / (g s), ties to the smaller magnitude, 6 at most, with x's sign
//           bit; a block whose s is 0 has zero codes, and one that holds a NaN
//           has the scale byte 0x7F (NaN) and zero codes.
//   read    x = e2m1(code) * e4m3(s) * g.
//
// Both are bound by memory: append reads 2 bytes and writes 9/16 a value, read
// the other way round.  A CTA takes ROWS consecutive rows.  Its threads look
// the rows' sequences up together (each takes some sequences and compares all
// the CTA's rows against them: one trip to memory however many sequences there
// are, where a search per row would be a chain of them), then a warp takes a
// (K or V, head) pair and runs over the CTA's rows, so that tokens which are
// neighbours in a page are read and written by neighbouring lanes.
// Measured, 131072 rows of 8 KV heads of 128: append 139 us (4.96 TB/s, 0.76 of
// a copy; with every border compared, 213 us), read 124 us (5.57 TB/s, 0.85).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include "kv4_layout.h"
#include "tb_decode.cuh"
#include "tb_ptx.cuh"

namespace tb {

// Bit of the device error word: a row's token has no page in the table, or
// the table names a page outside the cache.
enum : int { kErrPage = 2 };

struct Kv4Copy {
    Kv4Cache cache;
    Kv4Rows rows;
    void* k;                       // rows of K and V; append reads them, read writes them
    void* v;
    long long k_stride, v_stride;  // elements from one row to the next
    uint32_t lanes_per_row;        // items of a (row, head)
    uint32_t magic;                // ceil(65536 / lanes_per_row)
    float rk, rv, r6k, r6v;        // append: 1 / g and 1 / (6 g) of K and V
};

constexpr int kKv4CopyThreads = 256;

// Where each of the CTA's rows lies: offset of its page (or ~0 where the row
// belongs to no sequence or its token has no page) and its place in the page.
template <int ROWS>
struct Kv4Places {
    unsigned long long page[ROWS];
    int place[ROWS];
    int seq[ROWS];
};

template <int ROWS>
__device__ __forceinline__ void kv4_find_rows(const Kv4Copy& a, int row0, Kv4Places<ROWS>& s) {
    if (threadIdx.x < ROWS) s.seq[threadIdx.x] = -1;
    __syncthreads();
    for (int b = threadIdx.x; b < a.rows.batch; b += kKv4CopyThreads) {
        const int c0 = a.rows.cu[b], c1 = a.rows.cu[b + 1];
        for (int i = 0; i < ROWS; ++i)
            if (c0 <= row0 + i && row0 + i < c1) s.seq[i] = b;
        if (row0 == 0 && blockIdx.y == 0 && (c0 < 0 || c1 < c0 || c1 > a.rows.rows)) atomicOr(&g_tb_device_error, kErrPage);
    }
    __syncthreads();
    if (threadIdx.x < ROWS) {
        const int i = threadIdx.x, b = s.seq[i];
        unsigned long long page = ~0ull;
        int place = 0;
        if (b >= 0 && row0 + i < a.rows.rows) {
            const int shift = a.cache.page_shift;
            const Kv4Seq q = kv4_rows_seq(a.rows, shift, a.rows.cu[b], a.rows.cu[b + 1], a.rows.lens[b]);
            const int pos = q.pos0 + (row0 + i - q.first);
            const int slot = pos >> shift;
            bool ok = pos >= 0 && kv4_slot_ok(a.rows, slot);
            const int p = ok ? a.rows.table[static_cast<size_t>(b) * a.rows.width + slot] : -1;
            ok = ok && kv4_page_ok(a.cache, p);
            if (ok) page = static_cast<unsigned long long>(p) * a.cache.page_stride;
            else atomicOr(&g_tb_device_error, kErrPage);
            place = pos & ((1 << shift) - 1);
        }
        s.page[i] = page;
        s.place[i] = place;
    }
    __syncthreads();
}

// The E4M3 value of a scale byte 0x00-0x7E as FP32 (exact).
__device__ __forceinline__ float e4m3_value(uint32_t byte) {
    return __half2float(__ushort_as_half(static_cast<unsigned short>(cvt_e4m3x2(static_cast<uint16_t>(byte)))));
}

// Scale byte of a block whose largest magnitude is `amax` (not NaN); r6g is
// 1 / (6 g).  The borders between two E4M3 values lie at 6 g times their mean,
// m; 6 m has at most 7 significant bits, so `__fmul_rd(6 m, g)` is the exact
// border rounded down to FP32, and the FP32 number amax exceeds the border
// exactly when it exceeds that.  The product with r6g only finds the value
// below: where its rounding picks a neighbour, the border compared against
// still decides.
__device__ __forceinline__ uint32_t kv4_scale_byte(float amax, float g, float r6g) {
    const float q = fminf(amax * r6g, 448.0f);
    // largest E4M3 value not above q
    uint32_t c;
    if (q < 0.015625f) c = static_cast<uint32_t>(q * 512.0f);  // subnormal: multiples of 2^-9
    else c = (__float_as_uint(q) >> 20) - (120u << 3);         // exponent bias 127 -> 7, three mantissa bits
    if (c >= 126u) return 126u;
    const uint32_t two = cvt_e4m3x2(static_cast<uint16_t>(c * 0x101u + 0x100u));
    const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&two));
    return amax > __fmul_rd(3.0f * (v.x + v.y), g) ? c + 1 : c;
}

// Eight values to codes by the converter, first value in the high nibble of
// the first byte.
__device__ __forceinline__ uint32_t cvt_e2m1_x8(const float (&x)[8], float by) {
    uint32_t r;
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b0, %1, %2;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b1, %3, %4;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b2, %5, %6;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b3, %7, %8;\n\t"
        "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
        : "=r"(r)
        : "f"(x[0] * by), "f"(x[1] * by), "f"(x[2] * by), "f"(x[3] * by), "f"(x[4] * by), "f"(x[5] * by),
          "f"(x[6] * by), "f"(x[7] * by));
    return r;
}

// Codes of eight values for the scale value s > 0; rg is 1 / g.  The border
// above magnitude i lies at t_i s g with t_i s exact in FP32, so x passes it
// exactly when |x| > __fmul_rd(t_i s, g).  The converter rounds x / (s g) to
// the nearest E2M1 value; here that quotient is off by less than 2^-21 of
// itself (the reciprocal of s 2^-23, three products and rg 2^-24 each), so
// where it converts alike 2^-20 below and above no border lies between and the
// code is right; else the borders are compared.
__device__ __forceinline__ uint32_t kv4_codes(const float (&x)[8], float s, float g, float rg) {
    float inv;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(s));
    inv *= rg;
    const uint32_t lo = cvt_e2m1_x8(x, inv * (1.0f - 0x1p-20f)), hi = cvt_e2m1_x8(x, inv * (1.0f + 0x1p-20f));
    if (lo == hi) return lo;
    uint32_t word = 0;
#pragma unroll 1
    for (int i = 0; i < 7; ++i) {
        const float mids[7] = {0.25f, 0.75f, 1.25f, 1.75f, 2.5f, 3.5f, 5.0f};
        const float border = __fmul_rd(mids[i] * s, g);
#pragma unroll
        for (int j = 0; j < 8; ++j) word += static_cast<uint32_t>(fabsf(x[j]) > border) << (8 * (j / 2) + (j & 1 ? 0 : 4));
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) word |= ((__float_as_uint(x[j]) >> 31) << 3) << (8 * (j / 2) + (j & 1 ? 0 : 4));
    return word;
}

template <bool BF16>
__device__ __forceinline__ void unpack8(const uint4& u, float* x) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (BF16) {
            x[2 * i] = __uint_as_float(w[i] << 16);
            x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        } else {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
            x[2 * i] = f.x;
            x[2 * i + 1] = f.y;
        }
    }
}

// One lane quantises one block of 16 values; the values of UNROLL blocks are on
// their way before the first is worked on.
template <bool BF16, int ROWS, int UNROLL>
__global__ void __launch_bounds__(kKv4CopyThreads) k_kv4_append(const Kv4Copy a) {
    __shared__ Kv4Places<ROWS> s;
    const int row0 = blockIdx.x * ROWS;
    kv4_find_rows<ROWS>(a, row0, s);
    const int warps = kKv4CopyThreads / 32;
    const uint32_t items = ROWS * a.lanes_per_row;
    const uint32_t codes = kv4_codes_bytes(a.cache), scales = kv4_scales_bytes(a.cache);
    for (int pair = blockIdx.y * warps + threadIdx.x / 32; pair < 2 * a.cache.heads; pair += gridDim.y * warps) {
        const bool is_v = pair >= a.cache.heads;
        const int head = is_v ? pair - a.cache.heads : pair;
        const float g = is_v ? a.cache.v_scale : a.cache.k_scale, rg = is_v ? a.rv : a.rk, r6g = is_v ? a.r6v : a.r6k;
        const uint16_t* src = static_cast<const uint16_t*>(is_v ? a.v : a.k) + static_cast<size_t>(head) * a.cache.dim;
        const long long stride = is_v ? a.v_stride : a.k_stride;
        uint8_t* block = a.cache.data + static_cast<size_t>(head) * kv4_head_bytes(a.cache) +
                         (is_v ? codes + scales : 0u);
        for (uint32_t t0 = threadIdx.x & 31; t0 < items; t0 += 32 * UNROLL) {
            uint4 u[UNROLL][2];
            bool on[UNROLL];
#pragma unroll
            for (int k = 0; k < UNROLL; ++k) {
                const uint32_t t = t0 + 32 * k;
                const uint32_t r = (t * a.magic) >> 16, i = t - r * a.lanes_per_row;
                on[k] = t < items && s.page[t < items ? r : 0] != ~0ull;
                if (on[k]) {
                    const uint4* p = reinterpret_cast<const uint4*>(src + static_cast<long long>(row0 + r) * stride + 16 * i);
                    u[k][0] = p[0];
                    u[k][1] = p[1];
                }
            }
#pragma unroll
            for (int k = 0; k < UNROLL; ++k) {
                if (!on[k]) continue;
                const uint32_t t = t0 + 32 * k;
                const uint32_t r = (t * a.magic) >> 16, i = t - r * a.lanes_per_row;
                // The largest magnitude: without their signs the values order
                // like their bits, NaN above all.
                constexpr uint32_t kAbs = 0x7FFF7FFFu;
                uint32_t m = __vmaxu2(__vmaxu2(__vmaxu2(u[k][0].x & kAbs, u[k][0].y & kAbs),
                                               __vmaxu2(u[k][0].z & kAbs, u[k][0].w & kAbs)),
                                      __vmaxu2(__vmaxu2(u[k][1].x & kAbs, u[k][1].y & kAbs),
                                               __vmaxu2(u[k][1].z & kAbs, u[k][1].w & kAbs)));
                m = max(m & 0xFFFFu, m >> 16);
                const bool nan = m > (BF16 ? 0x7F80u : 0x7C00u);
                const float amax = BF16 ? __uint_as_float(m << 16)
                                        : __half2float(__ushort_as_half(static_cast<unsigned short>(m)));
                const uint32_t sb = nan ? 0x7Fu : kv4_scale_byte(amax, g, r6g);
                uint2 w = make_uint2(0u, 0u);
                if (sb != 0u && !nan) {
                    const float sv = e4m3_value(sb);
                    float x[8];
                    unpack8<BF16>(u[k][0], x);
                    w.x = kv4_codes(x, sv, g, rg);
                    unpack8<BF16>(u[k][1], x);
                    w.y = kv4_codes(x, sv, g, rg);
                }
                uint8_t* at = block + s.page[r];
                const uint32_t tok = static_cast<uint32_t>(s.place[r]);
                *reinterpret_cast<uint2*>(at + tok * (a.cache.dim / 2) + 8 * i) = w;
                at[codes + tok * (a.cache.dim / 16) + i] = static_cast<uint8_t>(sb);
            }
        }
    }
}

// One lane reads back eight values; UNROLL of them are loaded before the first
// is stored, to keep enough of the memory's latency in flight.
template <bool BF16, int ROWS, int UNROLL>
__global__ void __launch_bounds__(kKv4CopyThreads, 4) k_kv4_read(const Kv4Copy a) {
    __shared__ Kv4Places<ROWS> s;
    const int row0 = blockIdx.x * ROWS;
    kv4_find_rows<ROWS>(a, row0, s);
    const int warps = kKv4CopyThreads / 32;
    const uint32_t items = ROWS * a.lanes_per_row;
    const uint32_t codes = kv4_codes_bytes(a.cache), scales = kv4_scales_bytes(a.cache);
    for (int pair = blockIdx.y * warps + threadIdx.x / 32; pair < 2 * a.cache.heads; pair += gridDim.y * warps) {
        const bool is_v = pair >= a.cache.heads;
        const int head = is_v ? pair - a.cache.heads : pair;
        const float g = is_v ? a.cache.v_scale : a.cache.k_scale;
        uint16_t* dst = static_cast<uint16_t*>(is_v ? a.v : a.k) + static_cast<size_t>(head) * a.cache.dim;
        const long long stride = is_v ? a.v_stride : a.k_stride;
        const uint8_t* block = a.cache.data + static_cast<size_t>(head) * kv4_head_bytes(a.cache) +
                               (is_v ? codes + scales : 0u);
        for (uint32_t t0 = threadIdx.x & 31; t0 < items; t0 += 32 * UNROLL) {
            uint32_t w[UNROLL];
            uint32_t sb[UNROLL];
            bool on[UNROLL];
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) {
                const uint32_t t = t0 + 32 * u;
                const uint32_t r = (t * a.magic) >> 16, i = t - r * a.lanes_per_row;
                on[u] = t < items && s.page[t < items ? r : 0] != ~0ull;
                if (on[u]) {
                    const uint8_t* at = block + s.page[r];
                    const uint32_t tok = static_cast<uint32_t>(s.place[r]);
                    w[u] = *reinterpret_cast<const uint32_t*>(at + tok * (a.cache.dim / 2) + 4 * i);
                    sb[u] = at[codes + tok * (a.cache.dim / 16) + i / 2];
                }
            }
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) {
                if (!on[u]) continue;
                const uint32_t t = t0 + 32 * u;
                const uint32_t r = (t * a.magic) >> 16, i = t - r * a.lanes_per_row;
                // e2m1 * e4m3 is an FP16 value; the tensor's scale is applied in
                // FP32 and the product rounded once to the output type.
                const uint32_t sc = cvt_e4m3x2(static_cast<uint16_t>(sb[u] | (sb[u] << 8)));
                uint32_t v[4], o[4];
                decode_e2m1_packed_x8(w[u], v);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const __half2 h = __hmul2(*reinterpret_cast<const __half2*>(&v[j]),
                                              *reinterpret_cast<const __half2*>(&sc));
                    const float2 f = __half22float2(h);
                    if constexpr (BF16) {
                        const __nv_bfloat162 b = __floats2bfloat162_rn(f.x * g, f.y * g);
                        o[j] = *reinterpret_cast<const uint32_t*>(&b);
                    } else {
                        const __half2 b = __floats2half2_rn(f.x * g, f.y * g);
                        o[j] = *reinterpret_cast<const uint32_t*>(&b);
                    }
                }
                *reinterpret_cast<uint4*>(dst + static_cast<long long>(row0 + r) * stride + 8 * i) =
                    make_uint4(o[0], o[1], o[2], o[3]);
            }
        }
    }
}

}  // namespace tb
