// What the attention kernels over the 4-bit cache share: arguments, a request's geometry, scales of the
// scores, the work lists.
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
    int alone;         // the tile kernel does not run: no request is said to be wider
    int cols;          // the pairs its units take: 8 or 16
    float* part;       // the kernel's partial slots, two a CTA (units that several CTAs share)
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

// A softmax reference before any score; below every score (|score| log2(e) <= 2^126, see kv4_most_scale).
constexpr float kNoScore = -3.0e38f;

// The factor from a product of prepared operands (below 2^`bits`) to a score, kept so that scores are finite: a
// score's 24 bits then stand for differences of 2^40 and more, so the softmax is its limit already.
__device__ __forceinline__ float kv4_most_scale(float c, int bits) {
    const float most = __uint_as_float((uint32_t)(127 + 126 - bits) << 23);
    return fminf(fmaxf(c, -most), most);
}

// 2^k that brings a query row's largest entry into [2^13, 2^14); 1 for a row of zeros or without a finite largest.
__device__ __forceinline__ int query_scale(float top) {
    return top > 0.0f && top <= 3.402823466e38f ? min(max(13 - ((int)(__float_as_uint(top) >> 23) - 127), -120), 120) : 0;
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

// ------------------------------------------------------------------ the work lists
// Both kernels lay their units' steps end to end and cut the list into equal runs, one a CTA: run c is
// steps [start(c), start(c + 1)).
struct RunCut {
    int ctas, per, rem;  // the first rem runs have per + 1 steps
    __device__ __forceinline__ RunCut(int total, int most) {
        ctas = max(1, min(most, total));
        per = (int)((unsigned)total / (unsigned)ctas);
        rem = total - per * ctas;
    }
    __device__ __forceinline__ int start(int c) const { return c * per + min(c, rem); }
    __device__ __forceinline__ int owner(int step) const {
        const int head = rem * (per + 1);
        return step < head ? step / (per + 1) : rem + (step - head) / per;
    }
};

// Streaming kernel: a step is 256/D granules of one unit = (request, key head, block of `cols` pairs; the
// blocks of a key head follow one another, so all but the first find its cache in L2).  A unit that has steps
// begins with kStPad empty ones, which stand for the time a CTA needs to begin and merge it (3 to 4 us, a
// step of its four warps 0.4 us): without them the CTAs of short requests finished last (64 requests of
// 1024 to 16384 keys: from 83 to 110 us).  Measured with 4 / 8 / 16, us: 64 requests of 1024 to 16384 keys, 8 key heads
// of 64, 71 / 66 / 69, of 128, 118 / 111 / 114; 4 of 256 to 8192 keys, 72 / 69 / 67.
constexpr int kStWarps = 4;
constexpr int kStRows = 16;  // columns of a partial slot
constexpr int kStPad = 8;
template <int D>
__device__ __forceinline__ int stream_steps(const Kv4AttnArgs& a, const Kv4Request& r) {
    constexpr int T = kKvGranule * (256 / D);
    if (r.qn * (long long)a.group > a.max_cols) return 0;
    return (r.hi - r.lo + T - 1) / T;
}
__device__ __forceinline__ int stream_blocks(const Kv4AttnArgs& a, const Kv4Request& r) {
    return (r.qn * a.group + a.cols - 1) / a.cols;
}
__device__ __forceinline__ int stream_list(int steps) { return steps > 0 ? steps + kStPad : 0; }  // a unit's share of the list
// Every warp of a CTA that runs has a step to take.
__device__ __forceinline__ int stream_most(int total, int grid) { return min(grid, (total + kStWarps - 1) / kStWarps); }

// Tile kernel: a step is a tile of kv4_tile_keys(D) keys of one unit = (request, key head, block of
// kv4_tile_rows(D) (row, query head) pairs).
// A unit that has tiles begins with kv4_tile_pad(D) empty ones in the list, which stand for the time a CTA
// needs to begin and end it (about 8 us, a tile of D = 128 3.6): without them the CTAs of short units finished last.
// Measured with 2 / 3 / 6, us: 3 chunks of 400 to 777 rows beside 29 single tokens, window 2048, D = 64
// 126 / 126 / 133, D = 128 187 / 176 / 177, D = 256 268 / 260 / 241; 8 chunks of 150 to 300 rows, D = 64 76 / 76 / 81, D = 256
// 267 / 245 / 221.
__host__ __device__ constexpr int kv4_tile_pad(int D) { return D == 256 ? 6 : 3; }
__host__ __device__ constexpr int kv4_tile_rows(int D) { return D == 256 ? 128 : 256; }
__host__ __device__ constexpr int kv4_tile_keys(int D) { return D == 256 ? 64 : 128; }

struct TileUnit {
    int e0, rows;  // pairs [e0, e0 + rows)
    int lo, n;     // n tiles of keys from position lo
};

template <int D>
__device__ __forceinline__ TileUnit tile_unit(const Kv4AttnArgs& a, const Kv4Request& r, int u) {
    TileUnit t;
    t.e0 = u * kv4_tile_rows(D);
    t.rows = (int)min((long long)kv4_tile_rows(D), r.qn * (long long)a.group - t.e0);
    const int first = r.pos0 + t.e0 / a.group, last = r.pos0 + (t.e0 + t.rows - 1) / a.group;
    const int hi = min(r.hi, last + 1);
    t.lo = a.window > 0 ? max(0, min(first - a.window + 1, hi)) & ~(kKvGranule - 1) : 0;
    t.n = hi > t.lo ? (hi - t.lo + kv4_tile_keys(D) - 1) / kv4_tile_keys(D) : 0;
    return t;
}

template <int D>
__device__ __forceinline__ int tile_list(int tiles) { return tiles > 0 ? tiles + kv4_tile_pad(D) : 0; }  // a unit's share of the list

// A request's blocks; 0 for the streaming kernel's requests.
template <int D>
__device__ __forceinline__ int tile_blocks(const Kv4AttnArgs& a, const Kv4Request& r) {
    const long long pairs = r.qn * (long long)a.group;
    return pairs <= a.max_cols ? 0 : (int)((pairs + kv4_tile_rows(D) - 1) / kv4_tile_rows(D));
}

// Sum of v over the block's W warps, and the running sum before this thread (both in thread order).
template <int W>
__device__ __forceinline__ int block_scan(int v, int* red, int& before) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int s = v;
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, s, m);
        if (lane >= m) s += x;
    }
    __syncthreads();
    if (lane == 31) red[warp] = s;
    __syncthreads();
    int all = 0;
    before = s - v;
#pragma unroll
    for (int w = 0; w < W; w++) {
        if (w < warp) before += red[w];
        all += red[w];
    }
    return all;
}

// The list's length by steps(b) of every request, W warps together; n0 is steps(threadIdx.x).  `mark`, which
// steps() may set, is then true for every thread if it was for one.
template <int W, typename F>
__device__ __forceinline__ int list_total(int requests, int* red, int& n0, bool& mark, F steps) {
    n0 = (int)threadIdx.x < requests ? steps((int)threadIdx.x) : 0;
    int v = n0;
    for (int b = threadIdx.x + W * 32; b < requests; b += W * 32) v += steps(b);
    v = __reduce_add_sync(0xffffffffu, v);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    mark = __syncthreads_or(mark);
    int all = 0;
#pragma unroll
    for (int w = 0; w < W; w++) all += red[w];
    return all;
}

// The request that holds step `at` of the list, and the list position of its first step (in `pick`).
template <int W, typename F>
__device__ __forceinline__ void list_find(int requests, int* red, int* pick, int n0, int at, F steps) {
    int base = 0;
    for (int b0 = 0; b0 < requests; b0 += W * 32) {
        const int b = b0 + threadIdx.x;
        const int n = b0 == 0 ? n0 : (b < requests ? steps(b) : 0);
        int before;
        const int all = block_scan<W>(n, red, before);
        before += base;
        if (n > 0 && at >= before && at < before + n) pick[0] = b, pick[1] = before;
        base += all;
        if (at < base) break;
    }
    __syncthreads();
}

// The tile kernel's list, W warps together: every request's tiles (over one key head), by a warp a request
// where requests are few (their blocks are many then), else by a thread; `each` sees every unit once, and may set
// `mark` (as list_total's steps).
constexpr int kTlFew = 64;
template <int D, int W, typename F>
__device__ __forceinline__ int tile_list_total(const Kv4AttnArgs& a, int* red, int* few, int& n0, bool& mark, F each) {
    auto request = [&](int b, int u0, int du) {
        const Kv4Request r = kv4_request(a, b);
        const int blocks = tile_blocks<D>(a, r);
        int n = 0;
        for (int u = u0; u < blocks; u += du) {
            const TileUnit t = tile_unit<D>(a, r, u);
            each(b, r, t, u);
            n += tile_list<D>(t.n);
        }
        return n;
    };
    if (a.requests <= kTlFew) {
        for (int b = threadIdx.x >> 5; b < a.requests; b += W) {
            const int n = __reduce_add_sync(0xffffffffu, request(b, threadIdx.x & 31, 32));
            if ((threadIdx.x & 31) == 0) few[b] = n * a.kv_heads;
        }
        __syncthreads();
        return list_total<W>(a.requests, red, n0, mark, [&](int b) { return few[b]; });
    }
    return list_total<W>(a.requests, red, n0, mark, [&](int b) { return request(b, 0, 1) * a.kv_heads; });
}

// The unit that holds step `at` of the list: request pick[0], block pick[2], key head pick[4]; its first
// step is list position pick[3] (pick[1]: the request's).
template <int D, int W>
__device__ __forceinline__ void tile_list_find(const Kv4AttnArgs& a, int* red, int* pick, int n0, int at) {
    list_find<W>(a.requests, red, pick, n0, at, [&](int b) {
        const Kv4Request r = kv4_request(a, b);
        const int blocks = tile_blocks<D>(a, r);
        int n = 0;
        for (int u = 0; u < blocks; u++) n += tile_list<D>(tile_unit<D>(a, r, u).n);
        return n * a.kv_heads;
    });
    const Kv4Request r = kv4_request(a, pick[0]);
    const int blocks = tile_blocks<D>(a, r);
    auto unit = [&](int u) { return u < blocks ? tile_list<D>(tile_unit<D>(a, r, u).n) : 0; };
    int head = 0, before;
    for (int u0 = 0; u0 < blocks; u0 += W * 32) head += block_scan<W>(unit(u0 + threadIdx.x), red, before);
    const int h = (at - pick[1]) / head, first = pick[1] + h * head;
    int base = first;
    for (int u0 = 0; u0 < blocks; u0 += W * 32) {
        const int n = unit(u0 + threadIdx.x);
        const int all = block_scan<W>(n, red, before);
        before += base;
        if (n > 0 && at >= before && at < before + n) pick[2] = u0 + threadIdx.x, pick[3] = before, pick[4] = h;
        base += all;
        if (at < base) break;
    }
    __syncthreads();
}

// Programmatic dependent launch: the next kernel of the call may start; this one's predecessors done.
__device__ __forceinline__ void pdl_release() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// The streaming kernel (sx_kv4_stream.cu); its grid.
int kv4_stream_grid(int D, int cols);
cudaError_t kv4_stream_launch(const Kv4AttnArgs& a, int D, cudaStream_t stream);
// The tile kernel (sx_kv4_tile.cu): one CTA an SM.
cudaError_t kv4_tile_launch(const Kv4AttnArgs& a, int D, cudaStream_t stream);
// The join of the units that several CTAs of either kernel shared (sx_kv4_join.cu): `tile` null
// where that kernel did not run.
cudaError_t kv4_join_launch(const Kv4AttnArgs& stream_args, const Kv4AttnArgs* tile, int D, cudaStream_t stream);

}  // namespace sx
