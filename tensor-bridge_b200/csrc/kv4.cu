// kv4.cu -- the key/value cache in block-scaled FP4: argument checks and
// launches of tb_kv4_append, tb_kv4_read and tb_kv4_attention.
#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdio>
#include <cuda_runtime.h>
#include "tensor_bridge_b200.h"
#include "tb_host.h"
#include "kv4_prompt_kernel.cuh"

namespace {

using namespace tb;

tb_status refuse(tb_status s, const char* what) { return set_last_error(s, "kv4", what); }

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

size_t head_bytes(const tb_kv4_cache* c) {
    return static_cast<size_t>(c->page_size) * static_cast<size_t>(c->head_dim) * 9 / 8;
}

// The cache's description, checked.
tb_status check_cache(const tb_kv4_cache* c, Kv4Cache* out) {
    if (!c) return refuse(TB_ERR_INVALID_ARGUMENT, "cache is NULL");
    if (c->page_size < 16 || c->page_size > 1024 || (c->page_size & (c->page_size - 1)))
        return refuse(TB_ERR_SHAPE, "page_size must be a power of two from 16 to 1024");
    if (c->head_dim < 16 || c->head_dim > 256 || c->head_dim % 16)
        return refuse(TB_ERR_SHAPE, "head_dim must be a multiple of 16 up to 256");
    if (c->kv_heads < 1 || c->kv_heads > 65535 || c->num_pages < 0)
        return refuse(TB_ERR_SHAPE, "kv_heads must be 1 to 65535 and num_pages not negative");
    const size_t least = head_bytes(c) * static_cast<size_t>(c->kv_heads);
    const size_t stride = c->page_stride ? c->page_stride : least;
    if (stride < least) return refuse(TB_ERR_SHAPE, "page_stride is less than the page's bytes");
    if (stride % 16) return refuse(TB_ERR_ALIGNMENT, "page_stride must be a multiple of 16 bytes");
    // Also keeps every border of the quantiser an ordinary FP32 number.
    const float least_scale = 0x1p-100f, most_scale = 0x1p100f;
    if (!(c->k_scale >= least_scale && c->k_scale <= most_scale && c->v_scale >= least_scale &&
          c->v_scale <= most_scale))
        return refuse(TB_ERR_INVALID_ARGUMENT, "k_scale and v_scale must lie between 2^-100 and 2^100");
    if (!c->data && c->num_pages) return refuse(TB_ERR_INVALID_ARGUMENT, "cache data is NULL");
    if (!aligned16(c->data)) return refuse(TB_ERR_ALIGNMENT, "cache data must be 16-byte aligned");
    out->data = static_cast<uint8_t*>(c->data);
    out->page_stride = stride;
    out->num_pages = c->num_pages;
    out->page_shift = __builtin_ctz(static_cast<unsigned>(c->page_size));
    out->heads = c->kv_heads;
    out->dim = c->head_dim;
    out->k_scale = c->k_scale;
    out->v_scale = c->v_scale;
    return TB_OK;
}

tb_status check_rows(const tb_kv4_rows* r, int page_shift, Kv4Rows* out) {
    if (!r) return refuse(TB_ERR_INVALID_ARGUMENT, "rows is NULL");
    if (r->batch < 0 || r->rows < 0 || r->table_width < 0) return refuse(TB_ERR_SHAPE, "negative batch, rows or table_width");
    // Kernels step over rows and sequences in 32 bits, by less than 4096 at a time.
    if (r->batch > 0x7FFFFFFF - 4096 || r->rows > 0x7FFFFFFF - 4096)
        return refuse(TB_ERR_SHAPE, "batch and rows must not pass 2^31 - 4097");
    if ((static_cast<long long>(r->table_width) << page_shift) > 0x7FFFFFFFll - 4096)
        return refuse(TB_ERR_SHAPE, "table_width * page_size must stay below 2^31 - 4096");
    if (r->batch && r->rows && (!r->cu_rows || !r->seq_lens || (!r->block_table && r->table_width)))
        return refuse(TB_ERR_INVALID_ARGUMENT, "cu_rows, seq_lens or block_table is NULL");
    out->cu = r->cu_rows;
    out->lens = r->seq_lens;
    out->table = r->block_table;
    out->batch = r->batch;
    out->width = r->table_width;
    out->rows = r->rows;
    return TB_OK;
}

tb_status check_type(tb_format fmt) {
    return fmt == TB_FMT_F16 || fmt == TB_FMT_BF16 ? TB_OK : refuse(TB_ERR_INVALID_ARGUMENT, "rows must be F16 or BF16");
}

// Row stride in elements: 0 stands for dense rows.
tb_status check_stride(long long* stride, long long least) {
    if (*stride == 0) *stride = least;
    if (*stride < least) return refuse(TB_ERR_SHAPE, "a row stride is less than a row");
    if (*stride % 8) return refuse(TB_ERR_ALIGNMENT, "a row stride must be a multiple of 8 elements");
    return TB_OK;
}

tb_status check_gpu(int* sms) {
    int dev = 0;
    const cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return refuse(TB_ERR_CUDA, cudaGetErrorString(e));
    const DeviceInfo& d = device_info(dev);
    if (d.major != 10 || d.minor != 0) return refuse(TB_ERR_UNSUPPORTED, "the current device is not sm_100");
    *sms = d.sms;
    return TB_OK;
}

tb_status launched(cudaError_t e) {
    return e == cudaSuccess ? TB_OK : refuse(TB_ERR_LAUNCH, cudaGetErrorString(e));
}

tb_status check_copy(const tb_kv4_cache* cache, const tb_kv4_rows* rows, tb_format fmt, const void* k,
                     long long k_stride, const void* v, long long v_stride, Kv4Copy* a, int* sms) {
    tb_status s = check_cache(cache, &a->cache);
    if (s == TB_OK) s = check_rows(rows, a->cache.page_shift, &a->rows);
    if (s == TB_OK) s = check_type(fmt);
    const long long width = static_cast<long long>(cache && s == TB_OK ? cache->kv_heads : 0) * a->cache.dim;
    if (s == TB_OK) s = check_stride(&k_stride, width);
    if (s == TB_OK) s = check_stride(&v_stride, width);
    if (s != TB_OK) return s;
    if (a->rows.batch == 0 || a->rows.rows == 0) return TB_OK;
    if (!k || !v) return refuse(TB_ERR_INVALID_ARGUMENT, "null pointer");
    if (!aligned16(k) || !aligned16(v)) return refuse(TB_ERR_ALIGNMENT, "rows must be 16-byte aligned");
    a->k = const_cast<void*>(k);
    a->v = const_cast<void*>(v);
    a->k_stride = k_stride;
    a->v_stride = v_stride;
    return check_gpu(sms);
}

// A CTA of few rows starts fastest and spreads a step's rows over the SMs; one
// of many rows has enough loads in flight.  The change is made where the small
// CTAs would come in more than `per_sm` an SM (8 are there at once).  8 KV heads
// of 128, few against many: append 592 rows 3.1, 6.8 us, 2400 rows 6.2, 8.9, 16384
// rows 29.3, 22.1; read 592 rows 2.9, 5.2 us, 2400 rows 6.7, 6.9, 16384 rows
// 32.4, 19.4.
bool many_rows(const Kv4Copy& a, int per_cta, int per_sm, int sms, unsigned* y) {
    const int pairs = 2 * a.cache.heads;
    *y = static_cast<unsigned>((pairs + kKv4CopyThreads / 32 - 1) / (kKv4CopyThreads / 32));
    return static_cast<long long>((a.rows.rows + per_cta - 1) / per_cta) * *y > static_cast<long long>(per_sm) * sms;
}

dim3 copy_grid(const Kv4Copy& a, int per_cta, unsigned y) {
    return dim3(static_cast<unsigned>((a.rows.rows + per_cta - 1) / per_cta), y);
}

template <bool BF16>
cudaError_t run_append(const Kv4Copy& a, cudaStream_t st, int sms) {
    unsigned y;
    if (many_rows(a, 4, 20, sms, &y)) k_kv4_append<BF16, 32, 2><<<copy_grid(a, 32, y), kKv4CopyThreads, 0, st>>>(a);
    else k_kv4_append<BF16, 4, 1><<<copy_grid(a, 4, y), kKv4CopyThreads, 0, st>>>(a);
    return cudaGetLastError();
}

template <bool BF16>
cudaError_t run_read(const Kv4Copy& a, cudaStream_t st, int sms) {
    unsigned y;
    if (many_rows(a, 4, 9, sms, &y)) k_kv4_read<BF16, 32, 8><<<copy_grid(a, 32, y), kKv4CopyThreads, 0, st>>>(a);
    else k_kv4_read<BF16, 4, 2><<<copy_grid(a, 4, y), kKv4CopyThreads, 0, st>>>(a);
    return cudaGetLastError();
}

// ---- attention -----------------------------------------------------------------------

// What a call's sizes alone decide.
struct AttnPlan {
    int nt;             // step kernel: tiles of 8 rows
    int cluster, runs, min_run;
    size_t step_bytes;  // of its partial results
    int prompt_tiles;   // 0: no sequence has more rows than the step kernel takes
    bool drawn;         // its items are drawn from a counter
    int splits;
    size_t bytes;       // of both kernels' partial results
};

AttnPlan plan_attention(int batch, int heads, int dim, int page_shift, int group, int call_rows, int max_rows,
                        int max_len, int window, int sinks, int sms) {
    AttnPlan p{};
    const long long rows = static_cast<long long>(max_rows) * group;
    // Tokens that a sequence's rows see at most.  A window can only lower it,
    // and with it the bytes: tb_kv4_attention_workspace, which is told of none,
    // asks for enough.
    if (window > 0)
        max_len = static_cast<int>(std::min<long long>(max_len, static_cast<long long>(window) + sinks + max_rows));
    p.nt = rows <= 8 ? 1 : rows <= 16 ? 2 : rows <= 24 ? 3 : 4;
    p.runs = sms * (p.nt == 1 ? 2 : 1);
    // Clusters where they all fit on the GPU at once, a tile of tokens or more
    // to a CTA and not many (a cluster waits for its longest sequence, runs of
    // chunks share it): up to 1024 tokens, or 2560 where the clusters fill most
    // of the GPU.  One row, 8 KV heads of 128, clusters against runs: 1 sequence
    // of 1000 tokens 7.4, 10.6 us; 1 of 16384 17.3, 15.3 us; 4 of 16384 24.5,
    // 28.5 us; 32 of 2000 23.5, 28.3 us; 1 of 32768 28.3, 19.7 us.
    const long long units = static_cast<long long>(batch) * heads, room = p.runs / std::max(1ll, units);
    const long long share = std::min(std::min(8ll, room), std::max(1ll, (max_len + 255ll) / 256));
    if (share > 0 && max_len <= share * (units * share * 4 >= p.runs * 3ll ? 2560 : 1024))
        p.cluster = static_cast<int>(share);
    // A run has 512 tokens at least: one row at 16384 tokens 15.3 us, 15.9 with
    // 256, 17.3 with 1024.
    p.min_run = std::max(1, 512 >> step_gran(page_shift, p.nt == 2 ? 7 : 8));
    p.step_bytes = p.cluster ? 0 : static_cast<size_t>(p.runs) * (sizeof(StepLink) + 2 * (8 * p.nt) * (dim + 2) * sizeof(float));
    p.splits = 1;
    p.bytes = p.step_bytes;
    if (rows > kStepRowsMost) {
        p.prompt_tiles = static_cast<int>((rows + kPromptRows - 1) / kPromptRows);
        // Items drawn from a counter where fewer than three quarters of batch *
        // max_rows rows are there, so that sequences are unlike; else a fixed share
        // each.  32 heads of 128, 8 KV heads, drawn against fixed: 3 prompts of 2048
        // and 13 single rows 209, 279 us; 2048 rows behind 2048 tokens and 63 single
        // rows 304, 351 us; but 8 prompts of 2000 468, 445 us, one of 4096 171, 162 us.
        p.drawn = call_rows * 4ll < static_cast<long long>(batch) * max_rows * 3;
        // Fewer units than SMs: a unit's tokens are shared, 512 at least to each
        // (128 rows behind 3968 tokens, 8 KV heads: 35.2 us, 36.5 with 256, 39.2
        // with 1024).
        // Unlike sequences have about as many units as their rows fill tiles: 128
        // rows behind 32640 tokens and 31 single rows 594 us, 1032 without shares.
        // Rows of a padded batch count too: the partial results have their place.
        long long tiles = (static_cast<long long>(call_rows) * group + kPromptRows - 1) / kPromptRows;
        if (!p.drawn) tiles = std::max(tiles, static_cast<long long>(batch) * p.prompt_tiles);
        p.splits = static_cast<int>(std::max(1ll, std::min(sms / std::max(tiles * heads, 1ll), max_len / 512ll)));
        p.bytes += 16;  // the items' counter
        if (p.splits > 1)
            p.bytes += static_cast<size_t>(p.splits) * heads * call_rows * group * (dim + 2) * sizeof(float);
    }
    return p;
}

// Once per device and kernel: allow its shared memory, and make sure that it
// was built to launch with the registers that its warps divide later (a build
// with fewer would wait for ever, so it is not launched).
template <class K>
cudaError_t prepare_kernel(K kernel, int smem, int regs, std::atomic<uint64_t>& done) {
    const uint64_t bit = 1ull << (current_device() & 63);
    if (done.load() & bit) return cudaSuccess;
    cudaFuncAttributes attr{};
    cudaError_t e = cudaFuncGetAttributes(&attr, kernel);
    if (e == cudaSuccess && attr.numRegs < regs) e = cudaErrorInvalidDeviceFunction;
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e == cudaSuccess) done.fetch_or(bit);
    return e;
}

// Launch that may begin while the kernel before it ends.
template <class K>
cudaError_t launch_early(K kernel, dim3 grid, int threads, int smem, cudaStream_t st, const Kv4Attn& a) {
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(static_cast<unsigned>(threads));
    cfg.dynamicSmemBytes = static_cast<size_t>(smem);
    cfg.stream = st;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, a);
}

// Launch of `units` clusters.
template <class K>
cudaError_t launch_cluster(K kernel, unsigned units, int cluster, int threads, int smem, cudaStream_t st,
                           const Kv4Attn& a) {
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = static_cast<unsigned>(cluster);
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(units * static_cast<unsigned>(cluster));
    cfg.blockDim = dim3(static_cast<unsigned>(threads));
    cfg.dynamicSmemBytes = static_cast<size_t>(smem);
    cfg.stream = st;
    cfg.attrs = &attr;
    cfg.numAttrs = cluster > 1 ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kernel, a);
}

template <int D, int NT, bool BF16>
cudaError_t run_step(const Kv4Attn& a, cudaStream_t st) {
    using C = StepCfg<D, NT>;
    static std::atomic<uint64_t> done{0};
    cudaError_t e = prepare_kernel(k_kv4_step<C, BF16>, C::SMEM, C::REGS, done);
    if (e != cudaSuccess) return e;
    const unsigned units = static_cast<unsigned>(a.rows.batch) * a.cache.heads;
    if (a.cluster) return launch_cluster(k_kv4_step<C, BF16>, units, a.cluster, C::THREADS, C::SMEM, st, a);
    k_kv4_step<C, BF16><<<a.runs, C::THREADS, C::SMEM, st>>>(a);
    e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    constexpr int kJoinRows = 256 / D;  // rows of a CTA of k_kv4_join
    return launch_early(k_kv4_join<C, BF16>, dim3(a.runs, (C::ROWS + kJoinRows - 1) / kJoinRows), 256, 0, st, a);
}

template <int D, bool BF16>
cudaError_t run_prompt(const Kv4Attn& a, bool drawn, int sms, cudaStream_t st) {
    using C = PromptCfg<D>;
    const auto kernel = drawn ? k_kv4_prompt<C, BF16, true> : k_kv4_prompt<C, BF16, false>;
    static std::atomic<uint64_t> done[2] = {};
    cudaError_t e = prepare_kernel(kernel, C::SMEM, C::REGS, done[drawn]);
    if (e != cudaSuccess) return e;
    const int ctas = std::min(a.prompt_units * a.prompt_splits, sms);
    e = launch_early(kernel, dim3(ctas), kPromptThreads, C::SMEM, st, a);
    if (e != cudaSuccess || a.prompt_splits == 1) return e;
    constexpr int kJoinRows = 256 / D;  // rows of a CTA of k_kv4_prompt_join
    const unsigned x = static_cast<unsigned>((a.rows.rows * a.group + kJoinRows - 1) / kJoinRows);
    k_kv4_prompt_join<C, BF16><<<dim3(x, a.cache.heads), 256, 0, st>>>(a);
    return cudaGetLastError();
}

template <int D, bool BF16>
cudaError_t run_attention(const Kv4Attn& a, int nt, bool drawn, int sms, cudaStream_t st) {
    if (nt == 1) return run_step<D, 1, BF16>(a, st);
    if (nt == 2) return run_step<D, 2, BF16>(a, st);
    if (nt == 3) return run_step<D, 3, BF16>(a, st);
    const cudaError_t e = run_step<D, 4, BF16>(a, st);
    return e == cudaSuccess && a.prompt_tiles ? run_prompt<D, BF16>(a, drawn, sms, st) : e;
}

tb_status check_heads(const tb_kv4_cache* c, int q_heads, int max_rows, int max_len) {
    if (c->head_dim != 64 && c->head_dim != 128)
        return refuse(TB_ERR_SHAPE, "attention needs a head_dim of 64 or 128");
    if (q_heads < 1 || q_heads % c->kv_heads) return refuse(TB_ERR_SHAPE, "q_heads must be a multiple of kv_heads");
    // A query's place within its KV head's group is a 32-bit number of elements.
    if (static_cast<long long>(q_heads / c->kv_heads) * c->head_dim > 0x7FFFFFFFll)
        return refuse(TB_ERR_SHAPE, "q_heads / kv_heads * head_dim must stay below 2^31");
    if (max_rows < 0 || max_len < 0) return refuse(TB_ERR_SHAPE, "negative max_rows or max_len");
    return TB_OK;
}

}  // namespace

cudaError_t tb::kv4_device_error_read(int* v) { return cudaMemcpyFromSymbol(v, g_tb_device_error, sizeof(int)); }

cudaError_t tb::kv4_device_error_clear() {
    const int zero = 0;
    return cudaMemcpyToSymbol(g_tb_device_error, &zero, sizeof zero);
}

extern "C" {

size_t tb_kv4_page_bytes(int page_size, int kv_heads, int head_dim) {
    if (page_size < 1 || kv_heads < 1 || head_dim < 1) return 0;
    return static_cast<size_t>(page_size) * head_dim * 9 / 8 * kv_heads;
}

tb_status tb_kv4_append(const tb_kv4_cache* cache, const tb_kv4_rows* rows, tb_format fmt, const void* k,
                        long long k_stride, const void* v, long long v_stride, tb_stream_t stream) {
    Kv4Copy a{};
    int sms = 0;
    const tb_status s = check_copy(cache, rows, fmt, k, k_stride, v, v_stride, &a, &sms);
    if (s != TB_OK || a.rows.batch == 0 || a.rows.rows == 0) return s;
    a.rk = 1.0f / a.cache.k_scale;
    a.rv = 1.0f / a.cache.v_scale;
    a.r6k = 1.0f / (6.0f * a.cache.k_scale);
    a.r6v = 1.0f / (6.0f * a.cache.v_scale);
    a.lanes_per_row = static_cast<uint32_t>(a.cache.dim) / 16;
    a.magic = (65536u + a.lanes_per_row - 1) / a.lanes_per_row;
    return launched(fmt == TB_FMT_BF16 ? run_append<true>(a, stream, sms) : run_append<false>(a, stream, sms));
}

tb_status tb_kv4_read(const tb_kv4_cache* cache, const tb_kv4_rows* rows, tb_format fmt, void* k, long long k_stride,
                      void* v, long long v_stride, tb_stream_t stream) {
    Kv4Copy a{};
    int sms = 0;
    const tb_status s = check_copy(cache, rows, fmt, k, k_stride, v, v_stride, &a, &sms);
    if (s != TB_OK || a.rows.batch == 0 || a.rows.rows == 0) return s;
    a.lanes_per_row = static_cast<uint32_t>(a.cache.dim) / 8;
    a.magic = (65536u + a.lanes_per_row - 1) / a.lanes_per_row;
    return launched(fmt == TB_FMT_BF16 ? run_read<true>(a, stream, sms) : run_read<false>(a, stream, sms));
}

size_t tb_kv4_attention_workspace(const tb_kv4_cache* cache, const tb_kv4_rows* rows, int q_heads, int max_rows,
                                  int max_len) {
    Kv4Cache c{};
    Kv4Rows r{};
    if (check_cache(cache, &c) != TB_OK || check_rows(rows, c.page_shift, &r) != TB_OK) return 0;
    if (check_heads(cache, q_heads, max_rows, max_len) != TB_OK) return 0;
    return plan_attention(r.batch, c.heads, c.dim, c.page_shift, q_heads / c.heads, r.rows,
                          std::min(max_rows, r.rows), max_len, 0, 0, device_info(current_device()).sms)
        .bytes;
}

tb_status tb_kv4_attention(const tb_kv4_cache* cache, const tb_kv4_rows* rows, tb_format fmt, const void* q,
                           long long q_stride, void* out, long long out_stride, float* lse, int q_heads, int max_rows,
                           int max_len, float softmax_scale, int window, int sinks, void* workspace,
                           size_t workspace_bytes, tb_stream_t stream) {
    Kv4Attn a{};
    tb_status s = check_cache(cache, &a.cache);
    if (s == TB_OK) s = check_rows(rows, a.cache.page_shift, &a.rows);
    if (s == TB_OK) s = check_type(fmt);
    if (s == TB_OK) s = check_heads(cache, q_heads, max_rows, max_len);
    if (s != TB_OK) return s;
    if (static_cast<long long>(a.rows.rows) * q_heads > 0x7FFFFFFFll / 2)
        return refuse(TB_ERR_SHAPE, "rows * q_heads must stay below 2^30");
    if (window < 0 || sinks < 0) return refuse(TB_ERR_INVALID_ARGUMENT, "window and sinks must not be negative");
    if (!std::isfinite(softmax_scale)) return refuse(TB_ERR_INVALID_ARGUMENT, "softmax_scale must be finite");
    a.scale_log2 = softmax_scale * a.cache.k_scale * 1.4426950408889634f;
    if (!std::isfinite(a.scale_log2))
        return refuse(TB_ERR_INVALID_ARGUMENT, "softmax_scale * k_scale * log2(e) must be an FP32 number");
    const long long width = static_cast<long long>(q_heads) * a.cache.dim;
    s = check_stride(&q_stride, width);
    if (s == TB_OK) s = check_stride(&out_stride, width);
    if (s != TB_OK) return s;
    if (a.rows.batch == 0 || a.rows.rows == 0 || max_rows == 0) return TB_OK;
    if (!q || !out) return refuse(TB_ERR_INVALID_ARGUMENT, "null pointer");
    if (!aligned16(q) || !aligned16(out)) return refuse(TB_ERR_ALIGNMENT, "q and out must be 16-byte aligned");
    a.q = q;
    a.out = out;
    a.lse = lse;
    a.q_stride = q_stride;
    a.out_stride = out_stride;
    a.q_heads = q_heads;
    a.group = q_heads / a.cache.heads;
    a.window = window;
    a.sinks = sinks;
    int sms = 0;
    s = check_gpu(&sms);
    if (s != TB_OK) return s;
    max_rows = std::min(max_rows, a.rows.rows);
    const AttnPlan p = plan_attention(a.rows.batch, a.cache.heads, a.cache.dim, a.cache.page_shift, a.group, a.rows.rows,
                                      max_rows, max_len, window, sinks, sms);
    if (p.bytes) {
        if (!workspace || workspace_bytes < p.bytes) return refuse(TB_ERR_WORKSPACE, "workspace missing or too small");
        if (!aligned16(workspace)) return refuse(TB_ERR_ALIGNMENT, "workspace must be 16-byte aligned");
    }
    a.ws = static_cast<float*>(workspace);
    a.cluster = p.cluster;
    a.runs = p.runs;
    a.min_run = p.min_run;
    a.step_rows = 8 * p.nt;
    a.ticket = reinterpret_cast<int*>(static_cast<uint8_t*>(workspace) + p.step_bytes);
    a.prompt_ws = reinterpret_cast<float*>(a.ticket + 4);
    a.prompt_tiles = p.prompt_tiles;
    a.prompt_splits = p.splits;
    const long long units = static_cast<long long>(a.rows.batch) * a.cache.heads * std::max(p.prompt_tiles, 1);
    if (units * p.splits > 0x3FFFFFFFll)
        return refuse(TB_ERR_SHAPE, "batch * kv_heads * row tiles must stay below 2^30");
    a.prompt_units = static_cast<int>(units);
    const bool bf16 = fmt == TB_FMT_BF16;
    cudaError_t e;
    if (a.cache.dim == 128)
        e = bf16 ? run_attention<128, true>(a, p.nt, p.drawn, sms, stream) : run_attention<128, false>(a, p.nt, p.drawn, sms, stream);
    else
        e = bf16 ? run_attention<64, true>(a, p.nt, p.drawn, sms, stream) : run_attention<64, false>(a, p.nt, p.drawn, sms, stream);
    return launched(e);
}

}  // extern "C"
