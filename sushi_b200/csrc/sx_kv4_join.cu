// The join of attention units that several CTAs shared: out = sum_k 2^(m_k - M) O_k / sum_k 2^(m_k - M) l_k
// over the shares k in CTA order, M = max m_k.
//
// The first cut of a kernel's list inside a unit stands for the unit's join; its other cuts, and cuts
// between units, have nothing to do.  Everything but the shares themselves is known while the attention
// kernels still run (programmatic dependent launch), so the units are found first and what is left after the
// last attention CTA is two dependent loads: for one request of 131071 keys and 8 key heads (55 shares a
// head) a join inside the attention kernel by the last CTA to arrive took 12 us of fence, counter and one
// SM's loads.  Streaming kernel: a warp, or four, takes one column of a unit.  Tile kernel: a CTA takes 64 rows.
// Bound by load latency.
#include <cuda_runtime.h>

#include <algorithm>

#include "sx_kv4_attn.cuh"

namespace sx {

constexpr int kJoinWarps = 16;
constexpr int kJoinThreads = kJoinWarps * 32;
constexpr int kJoinShares = 64;  // shares whose weights are held at a time

// One column of a unit the streaming kernel's CTAs shared, by one warp, or by `parts` warps of a group that
// take the shares in turn and add up in `sums` (parts > 1; the group's barrier id).
template <int D>
__device__ __forceinline__ void join_column(const Kv4AttnArgs& a, const Kv4Request& r, int h, int pair, int c, const float* s0,
                                            const float* s1, int shares, int part, int parts, float* sums, int barrier) {
    constexpr int E = D / 32;  // channels a lane
    constexpr size_t STRIDE = (size_t)kStRows * (D + 2);
    const int lane = threadIdx.x & 31;
    auto share = [&](int k) { return k == 0 ? s0 : s1 + (size_t)(2 * k) * STRIDE; };
    // J shares' values and references are asked for before anything is worked out
    constexpr int J = 64 / E < 16 ? 64 / E : 16;
    float y[J][E], mw;
    auto fetch = [&](int k0) {
        mw = lane < J && k0 + lane * parts < shares ? __ldcg(share(k0 + lane * parts) + kStRows * D + 2 * c) : kNoScore;
#pragma unroll
        for (int j = 0; j < J; j++) {
#pragma unroll
            for (int e = 0; e < E; e++) y[j][e] = 0.0f;
            if (k0 + j * parts < shares) {
                const float* p = share(k0 + j * parts) + c * D + lane * E;
                if constexpr (E == 2) {
                    const float2 t = __ldcg(reinterpret_cast<const float2*>(p));
                    y[j][0] = t.x, y[j][1] = t.y;
                } else {
#pragma unroll
                    for (int e = 0; e < E; e += 4) {
                        const float4 t = __ldcg(reinterpret_cast<const float4*>(p + e));
                        y[j][e] = t.x, y[j][e + 1] = t.y, y[j][e + 2] = t.z, y[j][e + 3] = t.w;
                    }
                }
            }
        }
    };
    fetch(part);
    float top = kNoScore, ls = 0.0f;
#pragma unroll 2
    for (int k = lane; k < shares; k += 32) {
        const float2 ml = __ldcg(reinterpret_cast<const float2*>(share(k) + kStRows * D + 2 * c));
        const float up = fmaxf(top, ml.x);
        ls = fmaf(ls, ex2(top - up), ml.y * ex2(ml.x - up));
        top = up;
    }
    float all = top;
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) all = fmaxf(all, __shfl_xor_sync(0xffffffffu, all, m));
    ls *= ex2(top - all);
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) ls += __shfl_xor_sync(0xffffffffu, ls, m);
    float v[E];
#pragma unroll
    for (int e = 0; e < E; e++) v[e] = 0.0f;
    for (int k0 = part; k0 < shares;) {
        const float w = ex2(mw - all);
#pragma unroll
        for (int j = 0; j < J; j++) {
            const float f = __shfl_sync(0xffffffffu, w, j);
#pragma unroll
            for (int e = 0; e < E; e++) v[e] = k0 + j * parts < shares ? fmaf(f, y[j][e], v[e]) : v[e];
        }
        k0 += J * parts;
        if (k0 < shares) fetch(k0);
    }
    if (parts > 1) {
        if (part > 0) {
#pragma unroll
            for (int e = 0; e < E; e++) sums[part * D + lane * E + e] = v[e];
        }
        asm volatile("bar.sync %0, %1;" ::"r"(barrier), "r"(parts * 32) : "memory");
        if (part == 0)
            for (int p = 1; p < parts; p++)
#pragma unroll
                for (int e = 0; e < E; e++) v[e] += sums[p * D + lane * E + e];
        asm volatile("bar.sync %0, %1;" ::"r"(barrier), "r"(parts * 32) : "memory");
        if (part > 0) return;
    }
    const float inv = ls == 0.0f ? 0.0f : 1.0f / ls;
    uint32_t* o = reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(a.out) +
                                              ((size_t)(r.q0 + pair / a.group) * a.heads + h * a.group + pair % a.group) * D + lane * E);
#pragma unroll
    for (int e = 0; e < E; e += 2) o[e / 2] = pack_act2(v[e] * inv, v[e + 1] * inv, a.dt);
}

template <int D>
__global__ void __launch_bounds__(kJoinThreads) kv4_join_kernel(Kv4AttnArgs a, int stream_grid) {
    extern __shared__ int starts[];  // [requests + 1] the first step of each request in the list
    __shared__ int red[kJoinWarps];
    const int tid = threadIdx.x, warp = tid >> 5;
    int total = 0;
    for (int b0 = 0; b0 < a.requests; b0 += kJoinThreads) {
        const int b = b0 + tid;
        int n = 0;
        if (b < a.requests) {
            const Kv4Request r = kv4_request(a, b);
            n = stream_list(stream_steps<D>(a, r));
            if (n > 0) n *= a.kv_heads * stream_blocks(a, r);
        }
        int before;
        const int all = block_scan<kJoinWarps>(n, red, before);
        if (b < a.requests) starts[b] = total + before;
        total += all;
    }
    if (tid == 0) starts[a.requests] = total;
    __syncthreads();
    const RunCut run(total, stream_most(total, stream_grid));
    const int items = total ? (run.ctas - 1) * a.cols : 0;
    // few units: many shares each, which four warps take in turn
    const int parts = a.requests * a.kv_heads * 4 <= run.ctas ? 4 : 1;
    __shared__ float sums[kJoinWarps * D];
    bool waited = false;
    for (int i = blockIdx.x + (int)gridDim.x * (warp / parts); i < items; i += (int)gridDim.x * (kJoinWarps / parts)) {
        const int cut = i / a.cols + 1, c = i % a.cols, at = run.start(cut);
        int lo = 0, hi = a.requests - 1;  // the last request that starts at or before `at`
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (starts[mid] <= at) lo = mid;
            else hi = mid - 1;
        }
        const Kv4Request r = kv4_request(a, lo);
        const int n = stream_list(stream_steps<D>(a, r)), u = (at - starts[lo]) / n, u0 = starts[lo] + u * n;
        const int blocks = stream_blocks(a, r), h = u / blocks, pair = (u - h * blocks) * a.cols + c;
        if (pair >= r.qn * a.group) continue;
        const int first = run.owner(u0 + kStPad);  // of the unit's steps
        if (at <= u0 + kStPad || first != cut - 1) continue;
        // a CTA's slots: its first segment, its last; the unit is the first CTA's last, unless its run began in it
        const float* s1 = a.part + (size_t)(2 * first) * ((size_t)kStRows * (D + 2));
        const float* s0 = s1 + (run.start(first) < u0 ? (size_t)kStRows * (D + 2) : 0);
        const int shares = run.owner(u0 + n - 1) - first + 1;
        if (!waited) pdl_wait();
        waited = true;
        join_column<D>(a, r, h, pair, c, s0, s1, shares, warp % parts, parts, sums + warp / parts * parts * D, 1 + warp / parts);
    }
    if (!waited) pdl_wait();  // a warp with nothing to join waits too: this grid's end stands for the whole call's
}

// 64 rows of a unit that the tile kernel's CTAs shared (32 at D = 256: eight channels of a row a lane's worth
// of loads either way).
template <int D>
constexpr int join_rows() {
    return D == 256 ? 32 : 64;
}

template <int D>
__global__ void __launch_bounds__(kJoinThreads, 2) kv4_join_tile_kernel(Kv4AttnArgs a, int tile_grid) {
    constexpr int ROWS = join_rows<D>(), PARTS = kJoinThreads / ROWS;  // threads a row
    constexpr int TG = kv4_tile_rows(D) / ROWS;                        // CTAs a cut
    constexpr int ITEMS = ROWS * (D / 4) / kJoinThreads;               // four channels each, a thread's
    __shared__ int red[kJoinWarps], pick[5], few[kTlFew];
    __shared__ float top_sm[ROWS], inv_sm[ROWS];
    __shared__ float wt[ROWS * kJoinShares];
    const int cut = (int)blockIdx.x / TG + 1, row0 = (int)blockIdx.x % TG * ROWS, tid = threadIdx.x;
    pdl_release();
    int n0;
    bool mark = false;
    const int total = tile_list_total<D, kJoinWarps>(a, red, few, n0, mark, [](int, const Kv4Request&, const TileUnit&, int) {});
    const RunCut run(total, tile_grid);
    if (total == 0 || cut >= run.ctas) {  // a CTA with nothing to join waits too: this grid's end stands for the whole call's
        pdl_wait();
        return;
    }
    const int at = run.start(cut);
    tile_list_find<D, kJoinWarps>(a, red, pick, n0, at);
    const Kv4Request r = kv4_request(a, pick[0]);
    const TileUnit t = tile_unit<D>(a, r, pick[2]);
    const int u0 = pick[3], h = pick[4];
    const int first = run.owner(u0 + kv4_tile_pad(D));  // of the unit's tiles
    if (at <= u0 + kv4_tile_pad(D) || first != cut - 1 || row0 >= t.rows) {
        pdl_wait();
        return;
    }
    const int shares = run.owner(u0 + kv4_tile_pad(D) + t.n - 1) - first + 1, rows = min(t.rows - row0, ROWS);
    constexpr size_t STRIDE = (size_t)kv4_tile_rows(D) * (D + 2);
    // a CTA's slots: its first segment, its last; the unit is the first CTA's last, unless its run began in it
    const float* s1 = a.part + (size_t)(2 * first) * STRIDE;
    const float* s0 = s1 + (run.start(first) < u0 ? STRIDE : 0);
    auto share = [&](int k) { return k == 0 ? s0 : s1 + (size_t)(2 * k) * STRIDE; };
    const int ml_at = kv4_tile_rows(D) * D + 2 * row0;

    pdl_wait();

    {   // the shares' references and sums of a row, by the row's PARTS threads (neighbouring lanes)
        const int c = tid / PARTS, part = tid % PARTS;
        constexpr int H = kJoinShares / PARTS;
        float held[H];
        float top = kNoScore, ls = 0.0f;
        auto take = [&](const float2& ml) {
            const float up = fmaxf(top, ml.x);
            ls = fmaf(ls, ex2(top - up), ml.y * ex2(ml.x - up));
            top = up;
        };
        float2 ml[H];
#pragma unroll
        for (int i = 0; i < H; i++) {
            const int k = part + i * PARTS;
            ml[i] = c < rows && k < shares ? __ldcg(reinterpret_cast<const float2*>(share(k) + ml_at + 2 * c)) : make_float2(kNoScore, 0.0f);
        }
#pragma unroll
        for (int i = 0; i < H; i++) {
            take(ml[i]);
            held[i] = ml[i].x;
        }
        for (int k = part + kJoinShares; k < shares; k += PARTS)
            if (c < rows) take(__ldcg(reinterpret_cast<const float2*>(share(k) + ml_at + 2 * c)));
        float all = top;
#pragma unroll
        for (int m = PARTS / 2; m > 0; m >>= 1) all = fmaxf(all, __shfl_xor_sync(0xffffffffu, all, m));
        ls *= ex2(top - all);
#pragma unroll
        for (int m = PARTS / 2; m > 0; m >>= 1) ls += __shfl_xor_sync(0xffffffffu, ls, m);
#pragma unroll
        for (int i = 0; i < H; i++) wt[c * kJoinShares + part + i * PARTS] = ex2(held[i] - all);
        if (part == 0) {
            top_sm[c] = all;
            inv_sm[c] = ls == 0.0f ? 0.0f : 1.0f / ls;
        }
    }
    __syncthreads();

    float4 v[ITEMS];
#pragma unroll
    for (int i = 0; i < ITEMS; i++) v[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 2
    for (int k = 0; k < shares; k++) {
        const float* s = share(k) + row0 * D;
#pragma unroll
        for (int i = 0; i < ITEMS; i++) {
            const int it = tid + i * kJoinThreads, c = it / (D / 4);
            if (c >= rows) continue;
            const float f = k < kJoinShares ? wt[c * kJoinShares + k] : ex2(__ldcg(share(k) + ml_at + 2 * c) - top_sm[c]);
            const float4 y = __ldcg(reinterpret_cast<const float4*>(s + it * 4));
            v[i].x = fmaf(f, y.x, v[i].x), v[i].y = fmaf(f, y.y, v[i].y);
            v[i].z = fmaf(f, y.z, v[i].z), v[i].w = fmaf(f, y.w, v[i].w);
        }
    }
#pragma unroll
    for (int i = 0; i < ITEMS; i++) {
        const int it = tid + i * kJoinThreads, c = it / (D / 4), ch = (it % (D / 4)) * 4;
        if (c >= rows) continue;
        const float inv = inv_sm[c];
        const int pair = t.e0 + row0 + c;
        const size_t o = ((size_t)(r.q0 + pair / a.group) * a.heads + h * a.group + pair % a.group) * D + ch;
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + o) =
            make_uint2(pack_act2(v[i].x * inv, v[i].y * inv, a.dt), pack_act2(v[i].z * inv, v[i].w * inv, a.dt));
    }
}

namespace {

template <typename F, typename... Args>
cudaError_t join_launch_one(F kern, int grid, int smem, cudaStream_t stream, Args... args) {
    cudaError_t e = func_attrs(reinterpret_cast<const void*>(kern), smem, false);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid, 1, 1);
    cfg.blockDim = dim3(kJoinThreads, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kern, args...);
}

template <int D>
cudaError_t join_launch(const Kv4AttnArgs& s, const Kv4AttnArgs* t, cudaStream_t stream) {
    if (t) {
        const int tg = sm_count();
        cudaError_t e = join_launch_one(kv4_join_tile_kernel<D>, std::max(1, (tg - 1) * (kv4_tile_rows(D) / join_rows<D>())), 0,
                                        stream, *t, tg);
        if (e != cudaSuccess) return e;
    }
    return join_launch_one(kv4_join_kernel<D>, sm_count(), (s.requests + 1) * (int)sizeof(int), stream, s,
                           kv4_stream_grid(D, s.cols));
}

}  // namespace

cudaError_t kv4_join_launch(const Kv4AttnArgs& s, const Kv4AttnArgs* t, int D, cudaStream_t stream) {
    if (D == 64) return join_launch<64>(s, t, stream);
    if (D == 128) return join_launch<128>(s, t, stream);
    return join_launch<256>(s, t, stream);
}

}  // namespace sx
