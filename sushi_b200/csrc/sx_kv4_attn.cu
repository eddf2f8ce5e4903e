// sx_kv4_attention: admission, and the choice between its two kernels, request by request on the
// device: few (row, query head) pairs a key head go to the streaming kernel, whose units carry 8 or 16 of
// them, the rest to the tile kernel, whose carry 256 (128 at D = 256).
#include <cuda_runtime.h>
#include <algorithm>
#include <climits>
#include <cmath>

#include "sx_kv4_attn.cuh"

using namespace sx;

namespace {

// A request of at most this many pairs a key head goes to the streaming kernel.  Measured on both sides, us a
// call, streaming / tile kernel, bf16, 2 key heads of 8 query heads:
//   pairs                         48           64           96          128
//   D = 64,  1 x 16384 keys    19 / 74      21 / 75      21 / 76      26 / 77
//            2 x 32768         29 / 65      37 / 65      43 / 66      53 / 66
//            16 x 8192         50 / 65      57 / 66      69 / 66      84 / 67
//            64 x 1024         34 / 55      39 / 55      53 / 57      64 / 58
//   D = 128, 1 x 16384         21 / 105     29 / 129     30 / 129     38 / 131
//            2 x 32768         38 / 79      49 / 90      62 / 91      78 / 92
//            16 x 8192         68 / 72      81 / 74     104 / 76     127 / 78
//            64 x 1024         39 / 61      48 / 63      64 / 65      81 / 67
//   D = 256, 1 x 16384         33 / 134     44 / 137     45 / 140     58 / 142
//            2 x 32768         66 / 114     90 / 118    111 / 122    146 / 127
//            16 x 8192        120 / 123    146 / 126    202 / 132    256 / 138
//            64 x 1024         70 / 97      84 / 105    118 / 102    151 / 116
// (F16: the streaming kernel 5 to 20% slower, the tile kernel, with its second parts, 5 to 50%; the same choice, a
// little early: 64 / 96 pairs at D = 128, 16 x 8192 keys, 88 / 101 and 115 / 103.)  Many long requests would turn to
// the tile kernel earlier, few requests later; the host does not know the lengths.
constexpr int stream_pairs(int D) { return D == 64 ? 96 : 64; }

// The widest request of a call, in pairs a key head.
long long most_pairs(const sx_kv4* c, int heads, int max_q) { return (long long)max_q * (heads / c->kv_heads); }
// The columns of a streaming unit: 16 where a single row has more than 8 pairs or where every request is
// the streaming kernel's and some have more than 8; 8 otherwise (a column tile less to multiply by).
int stream_cols(const sx_kv4* c, int heads, int max_q) {
    const long long most = most_pairs(c, heads, max_q);
    return heads / c->kv_heads > 8 || (most > 8 && most <= stream_pairs(c->head_dim)) ? 16 : 8;
}

// The workspace: the two partial slots of every CTA, the streaming kernel's (16 columns), then the
// tile kernel's (a block of rows) where the call can reach it.  Nothing in it outlives the call.
size_t stream_bytes(int D, int cols) { return (size_t)kv4_stream_grid(D, cols) * 2 * kStRows * (D + 2) * sizeof(float); }
size_t tile_bytes(int D) { return (size_t)sm_count() * 2 * kv4_tile_rows(D) * (D + 2) * sizeof(float); }

}  // namespace

extern "C" {

size_t sx_kv4_attention_workspace_bytes(const sx_kv4* cache, int32_t requests, int32_t tokens, int32_t heads,
                                        int32_t max_q) {
    (void)requests, (void)tokens;  // partial slots are the CTAs', two each, whatever the requests
    if (!cache || !kv4_dim_ok(cache->head_dim) || cache->kv_heads < 1 || heads < cache->kv_heads || max_q < 1) return 0;
    const int D = cache->head_dim, cols = stream_cols(cache, heads, max_q);
    return stream_bytes(D, cols) + (most_pairs(cache, heads, max_q) > stream_pairs(D) ? tile_bytes(D) : 0);
}

sx_status sx_kv4_attention(sx_stream stream, const sx_kv4* cache, const void* q, int64_t q_token_stride,
                           int64_t q_head_stride, sx_dtype dtype, int32_t tokens, int32_t heads, const int32_t* cu_q,
                           const int32_t* kv_lens, const int32_t* table, int32_t requests, int32_t table_width,
                           int64_t table_stride, int32_t max_q, float scale, int32_t window, void* out, void* workspace,
                           size_t workspace_bytes) {
    sx_status st = kv4_check(cache);
    if (st) return st;
    if (dtype != SX_DT_F16 && dtype != SX_DT_BF16) return SX_ERR_BAD_DTYPE;
    if (tokens < 0 || heads < 1 || heads % cache->kv_heads || requests < 1 || requests > kKvMostRequests || table_width < 1 ||
        table_stride < table_width || max_q < 1 || window < 0 || !(std::fabs(scale) < 0x1p100f))
        return SX_ERR_BAD_SHAPE;
    // the work lists count steps and tiles of keys in 32 bits
    const int D = cache->head_dim, few = stream_pairs(D);
    const long long most = most_pairs(cache, heads, max_q);
    const int cols = stream_cols(cache, heads, max_q);
    const long long units = (long long)requests * cache->kv_heads * ((std::min<long long>(most, few) + cols - 1) / cols);
    const long long steps = (long long)table_width * cache->page_size / (kKvGranule * (256 / D)) + 1 + kStPad;
    if ((double)units * (double)steps > INT_MAX) return SX_ERR_BAD_SHAPE;
    const long long blocks = (long long)tokens * (heads / cache->kv_heads) / kv4_tile_rows(D) + requests;
    const long long tiles = (long long)table_width * cache->page_size / kv4_tile_keys(D) + 1 + kv4_tile_pad(D);
    if (most > few && (double)blocks * (double)tiles * cache->kv_heads > INT_MAX)
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
    a.scale_log2 = (float)(scale * 1.4426950408889634);
    a.window = window > (1 << 30) ? 0 : window;  // wider than any cache: none (and positions less it stay in 32 bits)
    a.max_cols = few;
    a.alone = most <= few;
    a.cols = cols;
    a.part = static_cast<float*>(workspace);
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    cudaError_t e = kv4_stream_launch(a, D, s);
    if (e != cudaSuccess) return cuda_status(e, "kv4_attention stream launch");
    if (a.alone)
        return cuda_status(kv4_join_launch(a, nullptr, D, s), "kv4_attention join launch");
    Kv4AttnArgs t = a;
    t.part = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + stream_bytes(D, a.cols));
    e = kv4_tile_launch(t, D, s);
    if (e != cudaSuccess) return cuda_status(e, "kv4_attention tile launch");
    return cuda_status(kv4_join_launch(a, &t, D, s), "kv4_attention join launch");
}

}  // extern "C"
