// The join of attention units that several CTAs shared: out = sum_k 2^(m_k - M) O_k / sum_k 2^(m_k - M) l_k
// over the shares k in CTA order, M = max m_k.
//
// The first cut of a kernel's list inside a unit stands for the unit's join; its other cuts, and cuts
// between units, have nothing to do.  Everything but the shares themselves is known while the attention
// kernels still run (programmatic dependent launch), so the units are found first and what is left after the
// last attention CTA is two dependent loads: for one request of 131071 keys and 8 key heads (55 shares a
// head) a join inside the attention kernel by the last CTA to arrive took 12 us of fence, counter and one
// SM's loads.  Streaming kernel: a warp takes one column of a unit.  Tile kernel: a CTA takes 64 rows.
// Bound by load latency.
#include <cuda_runtime.h>

#include "sx_kv4_attn.cuh"

namespace sx {

constexpr int kJoinWarps = 16;
constexpr int kJoinThreads = kJoinWarps * 32;
constexpr int kJoinRows = 64;    // rows of a unit a CTA joins
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
        mw = lane < J && k0 + lane * parts < shares ? __ldcg(share(k0 + lane * parts) + kStRows * D + 2 * c) : -1.0e30f;
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
    float top = -1.0e30f, ls = 0.0f;
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
__global__ void __launch_bounds__(kJoinThreads) kv4_join_kernel(Kv4AttnArgs sa, Kv4AttnArgs ta, int stream_grid, int tile_grid,
                                                                int column_ctas) {
    extern __shared__ int starts[];  // [requests + 1] the first step of each request in the streaming kernel's list
    __shared__ int red[kJoinWarps], pick[5], few[kTlFew];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const bool tile = (int)blockIdx.x >= column_ctas;
    const Kv4AttnArgs& a = tile ? ta : sa;
    if (!tile) {
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
        for (int i = blockIdx.x + column_ctas * (warp / parts); i < items; i += column_ctas * (kJoinWarps / parts)) {
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
        return;
    }

    __shared__ float top_sm[kJoinRows], inv_sm[kJoinRows];
    __shared__ float wt[kJoinRows * kJoinShares];
    __shared__ float4 part_sm[kJoinThreads];
    constexpr int TG = kv4_tile_rows(D) / kJoinRows;  // CTAs a cut
    const int cut = ((int)blockIdx.x - column_ctas) / TG + 1, row0 = ((int)blockIdx.x - column_ctas) % TG * kJoinRows;
    int n0;
    const int total = tile_list_total<D, kJoinWarps>(a, red, few, n0, [](int, const Kv4Request&, const TileUnit&, int) {});
    const RunCut run(total, tile_grid);
    if (total == 0 || cut >= run.ctas) {
        pdl_wait();
        return;
    }
    const int at = run.start(cut);
    tile_list_find<D, kJoinWarps>(a, red, pick, n0, at);
    const Kv4Request r = kv4_request(a, pick[0]);
    const TileUnit t = tile_unit<D>(a, r, pick[2]);
    const int u0 = pick[3], h = pick[4], n = t.n, e0 = t.e0;
    int rows = t.rows;
    const int first = run.owner(u0);
    if (u0 == at || first != cut - 1 || row0 >= rows) {
        pdl_wait();
        return;
    }
    const int shares = run.owner(u0 + n - 1) - first + 1;
    rows = min(rows - row0, kJoinRows);
    constexpr int slot_rows = kv4_tile_rows(D);
    const size_t stride = (size_t)slot_rows * (D + 2);
    // a CTA's slots: its first segment, its last; the unit is the first CTA's last, unless it fills the run
    const float* s0 = a.part + (size_t)(2 * first + (run.start(first) != u0 ? 1 : 0)) * stride;
    const float* s1 = a.part + (size_t)(2 * first) * stride;
    auto share = [&](int k) { return k == 0 ? s0 : s1 + (size_t)(2 * k) * stride; };
    const int ml_at = slot_rows * D + 2 * row0;

    pdl_wait();

    // a warp a row: the reference and the sum over the shares; the first shares' weights
    for (int c = warp; c < rows; c += kJoinWarps) {
        float top = -1.0e30f, ls = 0.0f;
        for (int k = lane; k < shares; k += 32) {
            const float2 ml = __ldcg(reinterpret_cast<const float2*>(share(k) + ml_at + 2 * c));
            if (k < kJoinShares) wt[c * kJoinShares + k] = ml.x;
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
        for (int k = lane; k < min(shares, kJoinShares); k += 32) wt[c * kJoinShares + k] = ex2(wt[c * kJoinShares + k] - all);
        if (lane == 0) {
            top_sm[c] = all;
            inv_sm[c] = ls == 0.0f ? 0.0f : 1.0f / ls;
        }
    }
    __syncthreads();

    // a thread four channels of a row; where the items are few, groups of threads take every G-th share
    const int items = rows * (D / 4);
    int groups = 1;
    while (groups < 16 && items * groups * 2 <= kJoinThreads) groups *= 2;
    const int width = kJoinThreads / groups;
    const int gi = tid / width;
    for (int i0 = 0; i0 < items; i0 += width) {
        const int i = i0 + tid % width;
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        const int c = i / (D / 4), ch = (i % (D / 4)) * 4;
        if (i < items) {
            const int off = (row0 + c) * D + ch;
            auto add = [&](int k, float f) {
                const float4 y = __ldcg(reinterpret_cast<const float4*>(share(k) + off));
                v.x = fmaf(f, y.x, v.x), v.y = fmaf(f, y.y, v.y), v.z = fmaf(f, y.z, v.z), v.w = fmaf(f, y.w, v.w);
            };
            const int held = min(shares, kJoinShares);
#pragma unroll 8
            for (int k = gi; k < held; k += groups) add(k, wt[c * kJoinShares + k]);
            for (int k = kJoinShares + gi; k < shares; k += groups)
                add(k, ex2(__ldcg(share(k) + ml_at + 2 * c) - top_sm[c]));
        }
        if (groups > 1) {  // i0 == 0: every item is in this pass
            part_sm[tid] = v;
            __syncthreads();
            if (gi == 0)
                for (int g = 1; g < groups; g++) {
                    const float4 y = part_sm[g * width + tid];
                    v.x += y.x, v.y += y.y, v.z += y.z, v.w += y.w;
                }
        }
        if (gi == 0 && i < items) {
            const float inv = inv_sm[c];
            const int pair = e0 + row0 + c;
            const size_t o = ((size_t)(r.q0 + pair / a.group) * a.heads + h * a.group + pair % a.group) * D + ch;
            *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + o) =
                make_uint2(pack_act2(v.x * inv, v.y * inv, a.dt), pack_act2(v.z * inv, v.w * inv, a.dt));
        }
    }
}

namespace {

template <int D>
cudaError_t join_launch(const Kv4AttnArgs& s, const Kv4AttnArgs* t, cudaStream_t stream) {
    const int sg = kv4_stream_grid(D, s.cols), tg = t ? sm_count() : 1, blocks = sm_count();
    const int smem = (s.requests + 1) * (int)sizeof(int);
    cudaError_t e = func_attrs(reinterpret_cast<const void*>(kv4_join_kernel<D>), smem, false);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(blocks + (tg - 1) * (kv4_tile_rows(D) / kJoinRows), 1, 1);
    cfg.blockDim = dim3(kJoinThreads, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kv4_join_kernel<D>, s, t ? *t : s, sg, tg, blocks);
}

}  // namespace

cudaError_t kv4_join_launch(const Kv4AttnArgs& s, const Kv4AttnArgs* t, int D, cudaStream_t stream) {
    if (D == 64) return join_launch<64>(s, t, stream);
    if (D == 128) return join_launch<128>(s, t, stream);
    return join_launch<256>(s, t, stream);
}

}  // namespace sx
