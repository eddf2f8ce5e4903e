// Attention over the 4-bit cache (sx_kv4_attention): one warp a (row, query head), 32 keys at a time.
#include <cuda_runtime.h>
#include <math_constants.h>

#include <algorithm>
#include <cmath>

#include "sx_kv4_attn.cuh"

namespace sx {

constexpr int kAttnWarps = 4;

template <int D>
__global__ void __launch_bounds__(kAttnWarps * 32) kv4_attn_rows_kernel(Kv4AttnArgs a) {
    __shared__ float qs[kAttnWarps][D];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const long long item = (long long)blockIdx.x * kAttnWarps + warp;
    if (item >= (long long)a.tokens * a.heads) return;
    const int row = (int)(item / a.heads), head = (int)(item % a.heads);
    const int h = head / (a.heads / a.kv_heads);
    constexpr int E = D / 32;
    float o[E] = {};
    float m = -CUDART_INF_F, l = 0.0f;
    int b = -1;
    for (int i = 0; i < a.requests; i++)
        if (row >= a.cu_q[i] && row < a.cu_q[i + 1]) b = i;
    if (b < 0 || (a.cu_q[b + 1] - a.cu_q[b]) * (long long)a.group <= a.max_cols) return;  // the streaming kernel's
    {
        for (int c = lane; c < D; c += 32)
            qs[warp][c] = load_act(a.q, row * a.qts + head * a.qhs + c, a.dt) * a.scale_log2;
        __syncwarp();
        const int kv = min(a.kv_lens[b], a.width * a.page_size);
        const int pos = a.kv_lens[b] - (a.cu_q[b + 1] - a.cu_q[b]) + row - a.cu_q[b];
        const int first = a.window > 0 ? max(0, pos - a.window + 1) : 0;
        const int end = min(kv, pos + 1);
        for (int k0 = first; k0 < end; k0 += 32) {
            const int key = k0 + lane;
            float s = -CUDART_INF_F;
            const uint8_t* gran = nullptr;
            if (key < end) {
                const int page = a.table[b * a.tstride + (key >> a.shift)];
                if (page >= 0 && page < a.pages) {
                    gran = a.pool + kv4_granule<D>(page, a.kv_heads, h, a.page_size, key & (a.page_size - 1));
                    s = 0.0f;
                    for (int gr = 0; gr < D / kKvGroup; gr++) {
                        const uint32_t par = *reinterpret_cast<const uint32_t*>(gran + kv4_kpar_off(D) +
                                                                                ((key & 15) * (D / kKvGroup) + gr) * 4);
                        const float st = h2f((uint16_t)par), mn = h2f((uint16_t)(par >> 16));
                        for (int w = 0; w < 8; w++) {
                            const uint32_t word =
                                *reinterpret_cast<const uint32_t*>(gran + kv4_key_word<D>(key & 15, gr, w));
#pragma unroll
                            for (int j = 0; j < 8; j++)
                                s = fmaf(qs[warp][gr * 64 + w * 8 + j], fmaf((float)((word >> (4 * j)) & 15u), st, mn), s);
                        }
                    }
                }
            }
            float top = s;
#pragma unroll
            for (int x = 16; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
            if (!__any_sync(0xffffffffu, gran != nullptr)) continue;
            // A NaN score is passed over by fmaxf and lands in the sums.
            const float mnew = fmaxf(m, top), mref = mnew == -CUDART_INF_F ? 0.0f : mnew;
            const float corr = m == -CUDART_INF_F ? 0.0f : ex2(m - mref);
            const float p = gran ? ex2(s - mref) : 0.0f;
            float sum = p;
#pragma unroll
            for (int x = 16; x > 0; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
            l = l * corr + sum;
            m = mnew;
#pragma unroll
            for (int e = 0; e < E; e++) o[e] *= corr;
            const unsigned long long gp = reinterpret_cast<unsigned long long>(gran);
            for (int j = 0; j < 32; j++) {
                const float pj = __shfl_sync(0xffffffffu, p, j);
                const uint8_t* gj = reinterpret_cast<const uint8_t*>(__shfl_sync(0xffffffffu, gp, j));
                if (!gj) continue;
                const int tok = (k0 + j) & 15;
#pragma unroll
                for (int e = 0; e < E; e++) {
                    const int c = lane + 32 * e, gr = c >> 6, w = (c & 63) >> 3;
                    const uint32_t word = *reinterpret_cast<const uint32_t*>(gj + kv4_value_word<D>(tok, gr, w));
                    const uint32_t par = *reinterpret_cast<const uint32_t*>(gj + kv4_vpar_off(D) + (tok * (D / kKvGroup) + gr) * 4);
                    o[e] = fmaf(pj, fmaf((float)((word >> (4 * (c & 7))) & 15u), h2f((uint16_t)par), h2f((uint16_t)(par >> 16))), o[e]);
                }
            }
        }
    }
#pragma unroll
    for (int e = 0; e < E; e++)
        store_act(a.out, ((size_t)row * a.heads + head) * D + lane + 32 * e, a.dt, l == 0.0f ? 0.0f : o[e] / l);
}

}  // namespace sx

using namespace sx;

namespace {

// The workspace: a counter a CTA, then two partial slots a CTA of 16 columns.
size_t counters_bytes() { return (size_t)kv4_max_ctas() * sizeof(int); }
size_t part_bytes(int D) { return (size_t)kv4_max_ctas() * 2 * 16 * (D + 2) * sizeof(float); }

}  // namespace

extern "C" {

size_t sx_kv4_attention_workspace_bytes(const sx_kv4* cache, int32_t requests, int32_t tokens, int32_t heads,
                                        int32_t max_q) {
    (void)requests, (void)tokens, (void)heads, (void)max_q;
    if (!cache || !kv4_dim_ok(cache->head_dim)) return 0;
    return counters_bytes() + part_bytes(cache->head_dim);
}

sx_status sx_kv4_attention(sx_stream stream, const sx_kv4* cache, const void* q, int64_t q_token_stride,
                           int64_t q_head_stride, sx_dtype dtype, int32_t tokens, int32_t heads, const int32_t* cu_q,
                           const int32_t* kv_lens, const int32_t* table, int32_t requests, int32_t table_width,
                           int64_t table_stride, int32_t max_q, float scale, int32_t window, void* out, void* workspace,
                           size_t workspace_bytes) {
    sx_status st = kv4_check(cache);
    if (st) return st;
    if (dtype != SX_DT_F16 && dtype != SX_DT_BF16) return SX_ERR_BAD_DTYPE;
    if (tokens < 0 || heads < 1 || heads % cache->kv_heads || requests < 1 || table_width < 1 ||
        table_stride < table_width || max_q < 1 || window < 0 || !std::isfinite(scale))
        return SX_ERR_BAD_SHAPE;
    if (tokens == 0) return SX_OK;
    if (!q || !cu_q || !kv_lens || !table || !out || !workspace) return SX_ERR_NULL_POINTER;
    if (reinterpret_cast<uintptr_t>(workspace) % 16 || reinterpret_cast<uintptr_t>(out) % 16) return SX_ERR_BAD_SHAPE;
    if (workspace_bytes < sx_kv4_attention_workspace_bytes(cache, requests, tokens, heads, max_q))
        return SX_ERR_WORKSPACE_TOO_SMALL;
    Kv4AttnArgs a = {};
    a.pool = static_cast<const uint8_t*>(cache->pool);
    a.pages = cache->pages, a.kv_heads = cache->kv_heads, a.page_size = cache->page_size;
    while ((1 << a.shift) < a.page_size) a.shift++;
    a.q = q, a.qts = q_token_stride, a.qhs = q_head_stride;
    a.out = out, a.dt = dtype, a.tokens = tokens, a.heads = heads;
    a.cu_q = cu_q, a.kv_lens = kv_lens, a.table = table;
    a.requests = requests, a.width = table_width, a.tstride = table_stride;
    a.group = heads / cache->kv_heads;
    a.qvec = reinterpret_cast<uintptr_t>(q) % 16 == 0 && q_token_stride % 8 == 0 && q_head_stride % 8 == 0;
    a.scale_log2 = (float)(scale * 1.4426950408889634), a.window = window;
    const long long most = (long long)max_q * a.group;  // columns a key head, of any request
    a.max_cols = a.group > 8 || (most > 8 && most <= 16) ? 16 : 8;
    a.count = static_cast<int*>(workspace);
    a.part = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + counters_bytes());
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    cudaError_t e = kv4_stream_launch(a, cache->head_dim, s);
    if (e != cudaSuccess) return cuda_status(e, "kv4_attention stream launch");
    if (most <= a.max_cols) return SX_OK;
    const long long items = (long long)tokens * heads;
    const unsigned grid = (unsigned)((items + kAttnWarps - 1) / kAttnWarps);
    if (cache->head_dim == 64) kv4_attn_rows_kernel<64><<<grid, kAttnWarps * 32, 0, s>>>(a);
    else if (cache->head_dim == 128) kv4_attn_rows_kernel<128><<<grid, kAttnWarps * 32, 0, s>>>(a);
    else kv4_attn_rows_kernel<256><<<grid, kAttnWarps * 32, 0, s>>>(a);
    return cuda_status(cudaGetLastError(), "kv4_attention launch");
}

}  // extern "C"
