// The join of attention units that several CTAs shared: out = sum_k 2^(m_k - M) O_k / sum_k 2^(m_k - M) l_k
// over the shares k in CTA order, M = max m_k.
//
// Every place where the list of steps is cut gets CTAs of its own here (the first cut inside a unit
// joins it, the unit's other cuts and cuts between units have nothing to do).  They find their unit
// while the attention kernels still run (programmatic dependent launch) and wait only before reading the
// shares, so what is left after the last attention CTA is a few dependent loads: for one request of 131071
// keys and 8 key heads (55 shares a head) the in-kernel join by the last CTA to arrive took 12 us of
// fence, counter and one SM's loads.  Bound by load latency.
#include <cuda_runtime.h>

#include "sx_kv4_attn.cuh"

namespace sx {

constexpr int kJoinWarps = 16;
constexpr int kJoinThreads = kJoinWarps * 32;
constexpr int kJoinRows = 64;    // rows of a unit a CTA joins
constexpr int kJoinShares = 64;  // shares whose weights are held at a time

template <int D>
__global__ void __launch_bounds__(kJoinThreads) kv4_join_kernel(Kv4AttnArgs sa, Kv4AttnArgs ta, int stream_grid, int tile_grid) {
    __shared__ int red[kJoinWarps], pick[5], few[kTlFew];
    __shared__ float top_sm[kJoinRows], inv_sm[kJoinRows];
    __shared__ float wt[kJoinRows * kJoinShares];
    __shared__ float4 part_sm[kJoinThreads];
    constexpr int TG = kv4_tile_rows(D) / kJoinRows;  // CTAs a tile cut
    const bool tile = (int)blockIdx.x >= stream_grid - 1;
    const Kv4AttnArgs& a = tile ? ta : sa;
    const int cut = tile ? ((int)blockIdx.x - (stream_grid - 1)) / TG + 1 : (int)blockIdx.x + 1;
    const int row0 = tile ? ((int)blockIdx.x - (stream_grid - 1)) % TG * kJoinRows : 0;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

    auto steps = [&](int b) { return stream_steps<D>(a, kv4_request(a, b)) * a.kv_heads; };
    int n0;
    const int total = tile ? tile_list_total<D, kJoinWarps>(a, red, few, n0, [](int, const Kv4Request&, const TileUnit&, int) {})
                           : list_total<kJoinWarps>(a.requests, red, n0, steps);
    const RunCut run(total, tile ? tile_grid : stream_most(total, stream_grid));
    // A CTA with nothing to join waits too: this grid's end stands for the whole call's.
    if (total == 0 || cut >= run.ctas) {
        pdl_wait();
        return;
    }
    const int at = run.start(cut);
    if (tile) tile_list_find<D, kJoinWarps>(a, red, pick, n0, at);
    else list_find<kJoinWarps>(a.requests, red, pick, n0, at, steps);
    const Kv4Request r = kv4_request(a, pick[0]);
    int h, u0, n, e0 = 0, rows;
    if (!tile) {
        n = stream_steps<D>(a, r);
        h = (at - pick[1]) / n;
        u0 = pick[1] + h * n;
        rows = r.qn * a.group;
    } else {
        const TileUnit t = tile_unit<D>(a, r, pick[2]);
        u0 = pick[3], h = pick[4];
        n = t.n, e0 = t.e0, rows = t.rows;
    }
    const int first = run.owner(u0);
    if (u0 == at || first != cut - 1 || row0 >= rows) {
        pdl_wait();
        return;
    }
    const int shares = run.owner(u0 + n - 1) - first + 1;
    rows = min(rows - row0, kJoinRows);
    const int slot_rows = tile ? kv4_tile_rows(D) : kStRows;
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
    const int sg = kv4_stream_grid(D, s.max_cols), tg = t ? sm_count() : 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(sg - 1 + (tg - 1) * (kv4_tile_rows(D) / kJoinRows), 1, 1);
    cfg.blockDim = dim3(kJoinThreads, 1, 1);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kv4_join_kernel<D>, s, t ? *t : s, sg, tg);
}

}  // namespace

cudaError_t kv4_join_launch(const Kv4AttnArgs& s, const Kv4AttnArgs* t, int D, cudaStream_t stream) {
    if (D == 64) return join_launch<64>(s, t, stream);
    if (D == 128) return join_launch<128>(s, t, stream);
    return join_launch<256>(s, t, stream);
}

}  // namespace sx
