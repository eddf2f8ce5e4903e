// The 4-bit key/value cache's bookkeeping and storage: the block tables of a step, writing keys and
// values, reading them back.
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>

#include "sx_kv4.cuh"

namespace sx {

// ------------------------------------------------------------------ block tables
// Prefix sums over the requests (new tokens; new pages), then two flat lists: the step's tokens and
// the new table entries, each item finding its request by a binary search of the sums.  Every CTA
// makes the sums for itself (8 bytes a request from L2), so the step is one launch in which no CTA
// waits for another; a token on a new page takes the page from the stack itself rather than from the
// table entry another CTA writes.  Bound by launch and load latency (8 requests 2.7 us; 1024 requests with
// 13 thousand new tokens 6.7 us).
constexpr int kTablesThreads = 256;
constexpr int kTablesItems = 4;           // tokens a thread

__device__ __forceinline__ int kv4_pages_of(int tokens, int shift) {
    return (int)(((unsigned)tokens + (1u << shift) - 1) >> shift);
}

// The last b of n requests with sum[b] <= i (sum[0] = 0 <= i < sum[n]): requests without items are passed over.
__device__ __forceinline__ int request_of(const int* sum, int n, int i) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (sum[mid] <= i) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

__global__ void __launch_bounds__(kTablesThreads) block_tables_kernel(
    const int* __restrict__ ctx_lens, const int* __restrict__ new_lens, int B, int shift, int* table, int width,
    long long tstride, const int* __restrict__ free_pages, const int* __restrict__ free_count, int tokens,
    int* __restrict__ kv_lens, int* __restrict__ cu_q, long long* __restrict__ slots, int* __restrict__ positions,
    int* __restrict__ free_left) {
    extern __shared__ int sums[];
    int* tok = sums;           // [B + 1] running sum of new tokens
    int* grow = sums + B + 1;  // [B + 1] running sum of new pages
    __shared__ int2 part[kTablesThreads / 32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int nfree = free_count[0];

    int2 base = make_int2(0, 0);
    for (int b0 = 0; b0 < B; b0 += kTablesThreads) {
        const int b = b0 + tid;
        int c = 0, n = 0, g = 0;
        if (b < B) {
            c = max(ctx_lens[b], 0);
            n = max(new_lens[b], 0);
            g = max(min(kv4_pages_of(c + n, shift), width) - kv4_pages_of(c, shift), 0);
        }
        int2 s = make_int2(n, g);
#pragma unroll
        for (int m = 1; m < 32; m <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, s.x, m), y = __shfl_up_sync(0xffffffffu, s.y, m);
            if (lane >= m) s.x += x, s.y += y;
        }
        if (lane == 31) part[warp] = s;
        __syncthreads();
        int2 all = make_int2(0, 0);
#pragma unroll
        for (int w = 0; w < kTablesThreads / 32; w++) {
            if (w < warp) s.x += part[w].x, s.y += part[w].y;
            all.x += part[w].x, all.y += part[w].y;
        }
        if (b < B) {
            tok[b] = base.x + s.x - n;
            grow[b] = base.y + s.y - g;
            if (blockIdx.x == 0) {
                kv_lens[b] = c + n;
                cu_q[b] = base.x + s.x - n;
            }
        }
        base.x += all.x, base.y += all.y;
        __syncthreads();
    }
    if (tid == 0) {
        tok[B] = base.x;
        grow[B] = base.y;
        if (blockIdx.x == 0) {
            cu_q[B] = base.x;
            free_left[0] = nfree - base.y;
        }
    }
    __syncthreads();

    const int stride = gridDim.x * kTablesThreads;
    for (int i = blockIdx.x * kTablesThreads + tid; i < base.y; i += stride) {
        const int b = request_of(grow, B, i);
        const int at = nfree - 1 - i;
        table[b * tstride + kv4_pages_of(max(ctx_lens[b], 0), shift) + i - grow[b]] = at >= 0 ? free_pages[at] : -1;
    }
    const int mask = (1 << shift) - 1;
    for (long long i = blockIdx.x * kTablesThreads + tid; i < tokens; i += stride) {
        long long slot = -1;
        int pos = 0;
        if (i < base.x) {
            const int b = request_of(tok, B, (int)i);
            const int c = max(ctx_lens[b], 0);
            pos = c + (int)i - tok[b];
            const int col = pos >> shift, have = kv4_pages_of(c, shift);
            int page = -1;
            if (col < width) {
                if (col < have) {
                    page = table[b * tstride + col];
                } else {
                    const int at = nfree - 1 - grow[b] - (col - have);
                    if (at >= 0) page = free_pages[at];
                }
            }
            if (page >= 0) slot = ((long long)page << shift) + (pos & mask);
        }
        slots[i] = slot;
        positions[i] = pos;
    }
}

// ------------------------------------------------------------------ write and read
// A thread takes eight consecutive channels of a token's key AND value: two 16-byte loads in flight
// (16-bit types), each group's minimum and maximum over its eight lanes by shuffles, one 32-bit word of
// codes each; one pass over the data.  The grid's x walks the tokens, so an item's head and piece come from 32-bit
// arithmetic (a 64-bit division an item took most of the time: 8192 tokens of 8 heads of 128, written and read
// back, 76 us with it, 37 us now).  Each alone, over more data than L2 holds (43 MB a call, bf16): the write 27 us,
// 1.6 TB/s, bound by the encoding's instructions, its one item in flight a thread and stores of 4 bytes; the read
// 13.4 us, 3.2 TB/s, by instructions and loads of 4 bytes.  f32: 25 and 22 us for 77 MB.
constexpr int kKvThreads = 256;
constexpr int kKvMostHeads = 65536;  // a token's items, and a CTA's, stay in 32 bits

struct KvIoArgs {
    uint8_t* pool;
    long long places;  // pages * page_size
    int kv_heads, page_size, shift;
    int row_items;  // kv_heads * D / 8: a token's items
    const void* src[2];  // write: k, v
    long long ts[2], hs[2];
    void* dst[2];  // read: k, v
    const long long* slots;
    int tokens;
    int per_cta;  // tokens a CTA
    int dt;
    int vec;  // every row of eight channels starts 16-byte aligned
};

__device__ __forceinline__ void load8(const void* p, long long i, int dt, bool vec, float (&x)[8]) {
    if (!vec) {
#pragma unroll
        for (int j = 0; j < 8; j++) x[j] = load_act(p, (size_t)(i + j), dt);
        return;
    }
    if (dt == 0) {
        const float4 a = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + i);
        const float4 b = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + i + 4);
        x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
        return;
    }
    const uint4 u = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + i);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const uint16_t h = (uint16_t)(w[j >> 1] >> (16 * (j & 1)));
        x[j] = dt == 1 ? __half2float(__ushort_as_half(h)) : __bfloat162float(__ushort_as_bfloat16(h));
    }
}

// A group's codes and parameters; the eight lanes of `lanes` hold its 64 channels, eight each.
__device__ __forceinline__ uint32_t encode8(float (&x)[8], unsigned lanes, uint32_t& par) {
    bool bad = false;
    float lo = kKvLargest, hi = -kKvLargest;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        bad |= !(fabsf(x[j]) <= 3.402823466e38f);
        x[j] = fminf(fmaxf(x[j], -kKvLargest), kKvLargest);
        lo = fminf(lo, x[j]);
        hi = fmaxf(hi, x[j]);
    }
#pragma unroll
    for (int m = 1; m < 8; m <<= 1) {
        lo = fminf(lo, __shfl_xor_sync(lanes, lo, m));
        hi = fmaxf(hi, __shfl_xor_sync(lanes, hi, m));
    }
    bad = __any_sync(lanes, bad);
    __half mh = __float2half_rn(lo), sh = __float2half_rn((hi - lo) * (1.0f / 15.0f));
    const float mf = __half2float(mh), s = __half2float(sh);
    uint32_t word = 0;
    if (bad) {
        mh = sh = __ushort_as_half((unsigned short)0x7fff);
    } else if (s > 0.0f) {
        // (x - m) / s: one correction of the product with the reciprocal by its remainder (Markstein
        // 1990) gives the rounded quotient, so a value half way between two codes goes the same way
        // as under a division.
        const float inv = __frcp_rn(s);
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float d = x[j] - mf;
            const float q0 = d * inv;
            const float q = fmaf(fmaf(-q0, s, d), inv, q0);
            word |= (uint32_t)min(max(__float2int_rn(q), 0), 15) << (4 * j);
        }
    }
    par = (uint32_t)__half_as_ushort(sh) | ((uint32_t)__half_as_ushort(mh) << 16);
    return word;
}

// Item i of a CTA's tokens [t0, t0 + n): token, head and piece.
struct KvItem {
    int t, h, piece;
};
template <int D>
__device__ __forceinline__ KvItem kv_item(const KvIoArgs& a, int t0, int i) {
    const unsigned t = (unsigned)i / (unsigned)a.row_items, rest = i - t * a.row_items;
    return {t0 + (int)t, (int)(rest / (D / 8)), (int)(rest % (D / 8))};
}

template <int D>
__global__ void __launch_bounds__(kKvThreads) kv4_write_kernel(KvIoArgs a) {
    const int t0 = blockIdx.x * a.per_cta;
    const int items = min(a.per_cta, a.tokens - t0) * a.row_items;
    const unsigned lanes = 0xffu << (threadIdx.x & 24);
    // The eight lanes of a group share a token and head, so they leave and skip together and the shuffles
    // name only lanes that are there.
    for (int i = blockIdx.y * kKvThreads + threadIdx.x; i < items; i += gridDim.y * kKvThreads) {
        const KvItem it = kv_item<D>(a, t0, i);
        const long long slot = a.slots[it.t];
        if (slot < 0 || slot >= a.places) continue;
        float k[8], v[8];
        load8(a.src[0], it.t * a.ts[0] + it.h * a.hs[0] + it.piece * 8, a.dt, a.vec, k);
        load8(a.src[1], it.t * a.ts[1] + it.h * a.hs[1] + it.piece * 8, a.dt, a.vec, v);
        uint32_t kp, vp;
        const uint32_t kw = encode8(k, lanes, kp), vw = encode8(v, lanes, vp);
        const int tok = (int)(slot & (a.page_size - 1));
        uint8_t* gran = a.pool + kv4_granule<D>(slot >> a.shift, a.kv_heads, it.h, a.page_size, tok);
        const int gt = tok & (kKvGranule - 1), gr = it.piece >> 3, w = it.piece & 7;
        *reinterpret_cast<uint32_t*>(gran + kv4_key_word<D>(gt, gr, w)) = kw;
        *reinterpret_cast<uint32_t*>(gran + kv4_value_word<D>(gt, gr, w)) = vw;
        if (w == 0) *reinterpret_cast<uint32_t*>(gran + kv4_kpar_off(D) + (gt * (D / kKvGroup) + gr) * 4) = kp;
        if (w == 1) *reinterpret_cast<uint32_t*>(gran + kv4_vpar_off(D) + (gt * (D / kKvGroup) + gr) * 4) = vp;
    }
}

__device__ __forceinline__ void store8(void* p, long long o, int dt, bool vec, const float (&x)[8]) {
    if (!vec) {
#pragma unroll
        for (int j = 0; j < 8; j++) store_act(p, (size_t)(o + j), dt, x[j]);
    } else if (dt == 0) {
        float4* y = reinterpret_cast<float4*>(static_cast<float*>(p) + o);
        y[0] = make_float4(x[0], x[1], x[2], x[3]);
        y[1] = make_float4(x[4], x[5], x[6], x[7]);
    } else {
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const uint16_t e0 = dt == 1 ? f2h(x[2 * j]) : __bfloat16_as_ushort(__float2bfloat16_rn(x[2 * j]));
            const uint16_t e1 = dt == 1 ? f2h(x[2 * j + 1]) : __bfloat16_as_ushort(__float2bfloat16_rn(x[2 * j + 1]));
            w[j] = (uint32_t)e0 | ((uint32_t)e1 << 16);
        }
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + o) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

template <int D>
__global__ void __launch_bounds__(kKvThreads) kv4_read_kernel(KvIoArgs a) {
    const int t0 = blockIdx.x * a.per_cta;
    const int items = min(a.per_cta, a.tokens - t0) * a.row_items;
    for (int i = blockIdx.y * kKvThreads + threadIdx.x; i < items; i += gridDim.y * kKvThreads) {
        const KvItem it = kv_item<D>(a, t0, i);
        const long long slot = a.slots[it.t];
        uint32_t word[2] = {0, 0}, par[2] = {0, 0};  // 0 0: a place outside the pool reads 0
        if (slot >= 0 && slot < a.places) {
            const int tok = (int)(slot & (a.page_size - 1));
            const uint8_t* gran = a.pool + kv4_granule<D>(slot >> a.shift, a.kv_heads, it.h, a.page_size, tok);
            const int gt = tok & (kKvGranule - 1), gr = it.piece >> 3, w = it.piece & 7;
            word[0] = *reinterpret_cast<const uint32_t*>(gran + kv4_key_word<D>(gt, gr, w));
            word[1] = *reinterpret_cast<const uint32_t*>(gran + kv4_value_word<D>(gt, gr, w));
            par[0] = *reinterpret_cast<const uint32_t*>(gran + kv4_kpar_off(D) + (gt * (D / kKvGroup) + gr) * 4);
            par[1] = *reinterpret_cast<const uint32_t*>(gran + kv4_vpar_off(D) + (gt * (D / kKvGroup) + gr) * 4);
        }
        const long long o = ((long long)it.t * a.kv_heads + it.h) * D + it.piece * 8;
#pragma unroll
        for (int kv = 0; kv < 2; kv++) {
            const float s = h2f((uint16_t)par[kv]), m = h2f((uint16_t)(par[kv] >> 16));
            float x[8];
#pragma unroll
            for (int j = 0; j < 8; j++) x[j] = fmaf((float)((word[kv] >> (4 * j)) & 15u), s, m);
            store8(a.dst[kv], o, a.dt, a.vec, x);
        }
    }
}

}  // namespace sx

using namespace sx;

namespace {

int log2_of(int p) {
    int s = 0;
    while ((1 << s) < p) s++;
    return s;
}

KvIoArgs io_args(const sx_kv4* c, const int64_t* slots, int32_t tokens, sx_dtype dtype) {
    KvIoArgs a = {};
    a.pool = static_cast<uint8_t*>(c->pool);
    a.places = (long long)c->pages * c->page_size;
    a.kv_heads = c->kv_heads;
    a.page_size = c->page_size;
    a.shift = log2_of(c->page_size);
    a.slots = reinterpret_cast<const long long*>(slots);
    a.tokens = tokens;
    a.dt = dtype;
    a.row_items = c->kv_heads * (c->head_dim / 8);
    return a;
}

// The launch of one thread an item.  x: tokens, as many a CTA as make about 1024 items (long rows are
// spread over y instead).
dim3 io_grid(KvIoArgs& a) {
    a.per_cta = std::max(1, 4 * kKvThreads / a.row_items);
    const int y = std::min(std::max(1, a.row_items / (4 * kKvThreads)), 64);
    // few tokens: one pass a thread
    const int ctas = (a.tokens + a.per_cta - 1) / a.per_cta;
    const int passes = (a.per_cta * a.row_items / y + kKvThreads - 1) / kKvThreads;
    return dim3(ctas, std::min(64, ctas * y < 2 * sm_count() ? y * passes : y));
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

}  // namespace

extern "C" {

size_t sx_kv4_block_bytes(int32_t head_dim, int32_t page_size) {
    if (!kv4_dim_ok(head_dim) || !kv4_page_ok(page_size)) return 0;
    return (size_t)(page_size / kKvGranule) * kv4_granule_bytes(head_dim);
}

sx_status sx_block_tables(sx_stream stream, const int32_t* ctx_lens, const int32_t* new_lens, int32_t requests,
                          int32_t page_size, int32_t* table, int32_t table_width, int64_t table_stride,
                          const int32_t* free_pages, const int32_t* free_count, int32_t tokens, int32_t* kv_lens,
                          int32_t* cu_q, int64_t* slots, int32_t* positions, int32_t* free_left) {
    if (!ctx_lens || !new_lens || !table || !free_pages || !free_count || !kv_lens || !cu_q || !free_left)
        return SX_ERR_NULL_POINTER;
    if (tokens > 0 && (!slots || !positions)) return SX_ERR_NULL_POINTER;
    if (requests < 1 || requests > kKvMostRequests || !kv4_page_ok(page_size) || table_width < 1 ||
        table_stride < table_width || tokens < 0)
        return SX_ERR_BAD_SHAPE;
    const int smem = 2 * (requests + 1) * (int)sizeof(int);
    if (smem > 48 * 1024) {
        cudaError_t e = func_attrs(reinterpret_cast<const void*>(block_tables_kernel), smem, false);
        if (e != cudaSuccess) return cuda_status(e, "block_tables attributes");
    }
    // Tokens, and at most a page a request more than the tokens' pages, spread over the CTAs.
    const long long items = std::max<long long>(tokens, requests);
    const int per = kTablesThreads * kTablesItems;
    const int grid = (int)std::min<long long>((items + per - 1) / per, 4 * sm_count());
    block_tables_kernel<<<grid, kTablesThreads, smem, reinterpret_cast<cudaStream_t>(stream)>>>(
        ctx_lens, new_lens, requests, log2_of(page_size), table, table_width, table_stride, free_pages, free_count, tokens,
        kv_lens, cu_q, reinterpret_cast<long long*>(slots), positions, free_left);
    return cuda_status(cudaGetLastError(), "block_tables launch");
}

sx_status sx_kv4_write(sx_stream stream, const sx_kv4* cache, const void* k, int64_t k_token_stride,
                       int64_t k_head_stride, const void* v, int64_t v_token_stride, int64_t v_head_stride,
                       sx_dtype dtype, int32_t tokens, const int64_t* slots) {
    sx_status st = kv4_check(cache);
    if (st) return st;
    if (!dtype_ok(dtype)) return SX_ERR_BAD_DTYPE;
    if (tokens < 0 || cache->kv_heads > kKvMostHeads) return SX_ERR_BAD_SHAPE;
    if (tokens == 0) return SX_OK;
    if (!k || !v || !slots) return SX_ERR_NULL_POINTER;
    KvIoArgs a = io_args(cache, slots, tokens, dtype);
    const dim3 grid = io_grid(a);
    const int esz = dtype == SX_DT_F32 ? 4 : 2;
    a.src[0] = k, a.src[1] = v;
    a.ts[0] = k_token_stride, a.ts[1] = v_token_stride;
    a.hs[0] = k_head_stride, a.hs[1] = v_head_stride;
    a.vec = aligned16(k) && aligned16(v);
    for (int i = 0; i < 2; i++) a.vec = a.vec && (a.ts[i] * esz) % 16 == 0 && (a.hs[i] * esz) % 16 == 0;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    if (cache->head_dim == 64) kv4_write_kernel<64><<<grid, kKvThreads, 0, s>>>(a);
    else if (cache->head_dim == 128) kv4_write_kernel<128><<<grid, kKvThreads, 0, s>>>(a);
    else kv4_write_kernel<256><<<grid, kKvThreads, 0, s>>>(a);
    return cuda_status(cudaGetLastError(), "kv4_write launch");
}

sx_status sx_kv4_read(sx_stream stream, const sx_kv4* cache, const int64_t* slots, int32_t tokens, sx_dtype dtype,
                      void* k, void* v) {
    sx_status st = kv4_check(cache);
    if (st) return st;
    if (!dtype_ok(dtype)) return SX_ERR_BAD_DTYPE;
    if (tokens < 0 || cache->kv_heads > kKvMostHeads) return SX_ERR_BAD_SHAPE;
    if (tokens == 0) return SX_OK;
    if (!k || !v || !slots) return SX_ERR_NULL_POINTER;
    KvIoArgs a = io_args(cache, slots, tokens, dtype);
    const dim3 grid = io_grid(a);
    a.dst[0] = k, a.dst[1] = v;
    a.vec = aligned16(k) && aligned16(v);
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    if (cache->head_dim == 64) kv4_read_kernel<64><<<grid, kKvThreads, 0, s>>>(a);
    else if (cache->head_dim == 128) kv4_read_kernel<128><<<grid, kKvThreads, 0, s>>>(a);
    else kv4_read_kernel<256><<<grid, kKvThreads, 0, s>>>(a);
    return cuda_status(cudaGetLastError(), "kv4_read launch");
}

}  // extern "C"
