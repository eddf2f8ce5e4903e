// What the attention kernels over the 4-bit cache share: arguments, a request's geometry, the store
// of an output row.
#pragma once

#include "sx_kv4.cuh"

namespace sx {

struct Kv4AttnArgs {
    const uint8_t* pool;
    int pages, kv_heads, page_size, shift;
    const void* q;
    long long qts, qhs;  // elements between tokens and heads
    int qvec;            // every row starts 16-byte aligned
    void* out;
    int dt, tokens, heads, group;  // group: query heads a key head
    const int* cu_q;
    const int* kv_lens;
    const int* table;
    int requests, width;
    long long tstride;
    float scale_log2;  // scale * log2(e)
    int window;
    int max_cols;      // requests of at most this many (row, head) pairs a key head are the streaming kernel's
    float* part;       // partial sums of units that several CTAs share
    int* count;        // arrivals, zero between calls
};

// One request of a call: its rows, and the positions its keys occupy.
struct Kv4Request {
    int q0, qn;  // rows [q0, q0 + qn)
    int pos0;    // position of row 0 (negative when rows outnumber the keys)
    int lo, hi;  // positions [lo, hi) that any row may see; lo a multiple of 16
};

__device__ __forceinline__ Kv4Request kv4_request(const Kv4AttnArgs& a, int b) {
    Kv4Request r;
    const int c0 = a.cu_q[b], c1 = a.cu_q[b + 1], kv = a.kv_lens[b];
    r.q0 = min(max(c0, 0), a.tokens);
    r.qn = min(max(c1, r.q0), a.tokens) - r.q0;
    r.pos0 = kv - r.qn;
    const long long held = (long long)a.width << a.shift;
    r.hi = r.qn > 0 ? (int)max(0ll, min((long long)kv, held)) : 0;
    r.lo = a.window > 0 ? max(0, min(r.pos0 - a.window + 1, r.hi)) & ~(kKvGranule - 1) : 0;
    return r;
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ uint32_t pack_act2(float a, float b, int dt) {
    if (dt == 1) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// The streaming kernel (sx_kv4_stream.cu).  kv4_max_ctas: CTAs no launch of it passes.
inline int kv4_max_ctas() { return 4 * sm_count(); }
cudaError_t kv4_stream_launch(const Kv4AttnArgs& a, int D, cudaStream_t stream);
// The tile kernel (sx_kv4_tile.cu), one CTA an SM; floats of one of its two partial slots a CTA.
size_t kv4_tile_part_floats(int D);
cudaError_t kv4_tile_launch(const Kv4AttnArgs& a, int D, cudaStream_t stream);

}  // namespace sx
