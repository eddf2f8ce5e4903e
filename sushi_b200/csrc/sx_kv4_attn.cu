// sx_kv4_attention: admission, and the choice between its two kernels, request by request on the
// device: at most max_cols (row, query head) pairs a key head go to the streaming kernel, whose MMAs
// carry 8 or 16 columns, the rest to the tile kernel, whose carry 128 rows.
#include <cuda_runtime.h>
#include <algorithm>
#include <cmath>

#include "sx_kv4_attn.cuh"

using namespace sx;

namespace {

// The widest request of a call, and the pairs up to which its requests are the streaming kernel's.
long long most_pairs(const sx_kv4* c, int heads, int max_q) { return (long long)max_q * (heads / c->kv_heads); }
int stream_cols(const sx_kv4* c, int heads, int max_q) {
    const long long most = most_pairs(c, heads, max_q);
    return heads / c->kv_heads > 8 || (most > 8 && most <= 16) ? 16 : 8;
}

// The workspace: a counter a CTA, then two partial slots a CTA, of 16 columns (streaming kernel) or of
// a block of rows (tile kernel, which runs after it on the stream and takes the same space).
size_t counters_bytes() { return ((size_t)kv4_max_ctas() * sizeof(int) + 15) / 16 * 16; }
size_t part_bytes(int D, bool tile) {
    const size_t stream = (size_t)kv4_max_ctas() * 2 * 16 * (D + 2) * sizeof(float);
    return std::max(stream, tile ? (size_t)sm_count() * 2 * kv4_tile_part_floats(D) * sizeof(float) : 0);
}

}  // namespace

extern "C" {

size_t sx_kv4_attention_workspace_bytes(const sx_kv4* cache, int32_t requests, int32_t tokens, int32_t heads,
                                        int32_t max_q) {
    (void)requests, (void)tokens;
    if (!cache || !kv4_dim_ok(cache->head_dim) || cache->kv_heads < 1 || heads < cache->kv_heads || max_q < 1) return 0;
    return counters_bytes() +
           part_bytes(cache->head_dim, most_pairs(cache, heads, max_q) > stream_cols(cache, heads, max_q));
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
    a.max_cols = stream_cols(cache, heads, max_q);
    a.count = static_cast<int*>(workspace);
    a.part = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + counters_bytes());
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    cudaError_t e = kv4_stream_launch(a, cache->head_dim, s);
    if (e != cudaSuccess) return cuda_status(e, "kv4_attention stream launch");
    if (most_pairs(cache, heads, max_q) <= a.max_cols) return SX_OK;
    return cuda_status(kv4_tile_launch(a, cache->head_dim, s), "kv4_attention tile launch");
}

}  // extern "C"
