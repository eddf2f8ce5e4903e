// Attention over the 4-bit cache for requests of few rows: one token, a few drafted ones.
//
// A unit is one request and key head; its columns are the (row, query head) pairs that read that key
// head, at most 8 NT.  With 16 keys on the M axis and the columns on the N axis of m16n8k16:
//   S^T[key][col] = sum over groups g of  s_kg * (codes . q) + m_kg * (sum of q in g)
//   O^T[channel][col] = codes^T . (P * s_g) + sum over keys of P * m_g
// so the products take the codes themselves: a code masked out of its word is the F16 subnormal
// code * 2^-24 (or code * 2^-20 for every second nibble), exact, with no conversion.  The query is
// scaled by a power of two per column (its largest entry to [2^13, 2^14)) and by 1/16 where the
// nibble brings 16, and rounded to F16 (exact for bf16 and f16 entries within 2^24 of the largest).
// P * s is rounded to F16 once; m, sums and accumulators are f32.
//
// The softmax reference of a column is kept so that P * s <= 2^15, whatever the values' magnitude:
// it moves (one vote a step) only when a score or a step would pass that, with 2^4 to spare.
//
// Work: the units' steps (4.5 KB of one head: 256/D granules of 16 tokens) laid end to end and cut
// into equal runs, one a CTA, so ragged lengths balance; a CTA's warps take its steps in turn, each
// with its own ring of bulk copies.  A unit that several CTAs share is joined by the last of them to
// arrive, in CTA order (a counter, no CTA waits), so results do not depend on the arrival order.
#include <cuda_runtime.h>
#include <math_constants.h>

#include <algorithm>

#include "sx_kv4_attn.cuh"

namespace sx {

constexpr int kStWarps = 4;
constexpr int kStThreads = kStWarps * 32;
constexpr int kStStages = 3;

template <int D, int NT>
struct StreamLayout {
    static constexpr int G = D / kKvGroup;
    static constexpr int GS = 256 / D;  // granules a step
    static constexpr int GB = kv4_granule_bytes(D);
    static constexpr int STEP = GS * GB;  // 4608
    static constexpr int COLS = 8 * NT;
    static constexpr int ROW = D + 4;  // floats of a merge row
    static constexpr int RING = 0;
    static constexpr int Q = RING + kStWarps * kStStages * STEP;  // [COLS][D] f16, fragment order
    static constexpr int MERGE = Q + COLS * D * 2;                // [warps][8][ROW] f32
    static constexpr int QS = MERGE + kStWarps * 8 * ROW * 4;     // [COLS][G] f32
    static constexpr int CH = QS + COLS * G * 4;                  // [COLS] f32
    static constexpr int ML = CH + COLS * 4;                      // [warps][COLS] m, then l
    static constexpr int BAR = (ML + 2 * kStWarps * COLS * 4 + 15) / 16 * 16;
    static constexpr int TOTAL = BAR + kStWarps * kStStages * 8;
};

// A walk over the units' steps: request b, key head h, steps [u0, u0 + n) of the whole list.
struct StreamCursor {
    Kv4Request r;
    int b, h, n;
    long long u0;
};

template <int D>
__device__ __forceinline__ int stream_steps(const Kv4AttnArgs& a, const Kv4Request& r) {
    constexpr int T = kKvGranule * (256 / D);
    if (r.qn * (long long)a.group > a.max_cols) return 0;
    return (r.hi - r.lo + T - 1) / T;
}

// Moves the cursor forward to the unit that holds step i of the list.
template <int D>
__device__ __forceinline__ void stream_seek(const Kv4AttnArgs& a, StreamCursor& c, long long i) {
    while (i >= c.u0 + c.n) {
        c.u0 += c.n;
        if (++c.h == a.kv_heads || c.n == 0) {
            c.h = 0;
            c.b++;
            c.r = kv4_request(a, c.b);
            c.n = stream_steps<D>(a, c.r);
        }
    }
}

__device__ __forceinline__ uint32_t movmatrix(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// The token of a granule that sits in row r of the 16-row fragments (rows 2t and 2t+1 of a lane's
// four are tokens t and 4 + (t ^ 1), which the block's word order spreads over the banks).
__device__ __forceinline__ int row_token(int r) { return (r & 8) + ((r & 1) ? 4 + (((r & 7) >> 1) ^ 1) : ((r & 7) >> 1)); }

template <int D, int NT>
__global__ void __launch_bounds__(kStThreads, NT == 1 && D <= 128 ? 3 : 2) kv4_stream_kernel(Kv4AttnArgs a) {
    using L = StreamLayout<D, NT>;
    constexpr int G = L::G, GS = L::GS, COLS = L::COLS;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ long long red[kStWarps];
    __shared__ int pick_b, arrived;
    __shared__ long long pick_u0;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int g = lane >> 2, t = lane & 3;
    uint64_t* bar = reinterpret_cast<uint64_t*>(smem + L::BAR) + warp * kStStages;
    uint8_t* ring = smem + L::RING + warp * kStStages * L::STEP;
    if (lane == 0)
        for (int i = 0; i < kStStages; i++) mbar_init(&bar[i], 1);
    fence_mbar_init();

    // ---------------- the list: its length, then the unit of this CTA's first step
    long long total = 0;
    for (int b0 = 0; b0 < a.requests; b0 += kStThreads) {
        const int b = b0 + tid;
        total += b < a.requests ? (long long)stream_steps<D>(a, kv4_request(a, b)) * a.kv_heads : 0;
    }
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) total += __shfl_xor_sync(0xffffffffu, total, m);
    if (lane == 0) red[warp] = total;
    __syncthreads();
    total = 0;
#pragma unroll
    for (int w = 0; w < kStWarps; w++) total += red[w];
    // every warp of a CTA that runs has a step to take
    const long long ctas = min((long long)gridDim.x, (total + kStWarps - 1) / kStWarps);
    const int cta = blockIdx.x;

    // Rows that no unit writes: requests without a visible position, rows past the last request.
    const size_t row_units = (size_t)a.heads * D / 8;
    for (int b = cta; b <= a.requests; b += gridDim.x) {
        int r0, rn;
        if (b < a.requests) {
            const Kv4Request r = kv4_request(a, b);
            r0 = r.q0;
            rn = r.hi <= r.lo && r.qn * (long long)a.group <= a.max_cols ? r.qn : 0;
        } else {
            r0 = min(max(a.cu_q[a.requests], 0), a.tokens);
            rn = a.tokens - r0;
        }
        uint4* o = reinterpret_cast<uint4*>(a.out) + r0 * row_units;
        for (size_t i = tid; i < rn * row_units; i += kStThreads) o[i] = make_uint4(0, 0, 0, 0);
    }
    if (cta >= ctas) return;
    const long long start = total * cta / ctas, end = total * (cta + 1) / ctas;

    long long base = 0;
    for (int b0 = 0; b0 < a.requests; b0 += kStThreads) {
        const int b = b0 + tid;
        const long long n = b < a.requests ? (long long)stream_steps<D>(a, kv4_request(a, b)) * a.kv_heads : 0;
        long long s = n;
#pragma unroll
        for (int m = 1; m < 32; m <<= 1) {
            const long long x = __shfl_up_sync(0xffffffffu, s, m);
            if (lane >= m) s += x;
        }
        __syncthreads();
        if (lane == 31) red[warp] = s;
        __syncthreads();
        long long all = 0;
#pragma unroll
        for (int w = 0; w < kStWarps; w++) {
            if (w < warp) s += red[w];
            all += red[w];
        }
        if (n > 0 && start >= base + s - n && start < base + s) {
            pick_b = b;
            pick_u0 = base + s - n;
        }
        base += all;
        if (start < base) break;
    }
    __syncthreads();
    StreamCursor cur;
    cur.b = pick_b;
    cur.r = kv4_request(a, cur.b);
    cur.n = stream_steps<D>(a, cur.r);
    cur.h = (int)((start - pick_u0) / cur.n);
    cur.u0 = pick_u0 + (long long)cur.h * cur.n;
    StreamCursor ahead = cur;

    // ---------------- this warp's ring: step start + warp + 4 k in stage k % S
    uint32_t valid = 0;  // 4 bits a stage: the granules that were copied
    long long next = start + warp;
    auto issue = [&](int st) {
        if (next < end) {
            stream_seek<D>(a, ahead, next);
            const int pos = ahead.r.lo + ((int)(next - ahead.u0) * GS + (lane < GS ? lane : 0)) * kKvGranule;
            int page = -1;
            if (lane < GS && pos < ahead.r.hi) page = a.table[ahead.b * a.tstride + (pos >> a.shift)];
            const bool ok = page >= 0 && page < a.pages;
            const uint32_t m = __ballot_sync(0xffffffffu, ok);
            if (lane == 0) mbar_arrive_expect_tx(&bar[st], __popc(m) * L::GB);
            __syncwarp();
            if (ok)
                bulk_g2s(ring + st * L::STEP + lane * L::GB,
                         a.pool + kv4_granule<D>(page, a.kv_heads, ahead.h, a.page_size, pos & (a.page_size - 1)), L::GB,
                         &bar[st]);
            valid = (valid & ~(15u << (4 * st))) | (m << (4 * st));
        }
        next += kStWarps;
    };
#pragma unroll
    for (int i = 0; i < kStStages; i++) issue(i);

    float* qs_sm = reinterpret_cast<float*>(smem + L::QS);
    float* ch_sm = reinterpret_cast<float*>(smem + L::CH);
    float* m_sm = reinterpret_cast<float*>(smem + L::ML);
    float* l_sm = m_sm + kStWarps * COLS;
    float* merge = reinterpret_cast<float*>(smem + L::MERGE);
    const int tok0 = row_token(g);                   // fragment row g; row g + 8 is token tok0 + 8
    const int vt[4] = {t, 4 + (t ^ 1), 8 + t, 12 + (t ^ 1)};  // rows 2t, 2t+1, 2t+8, 2t+9

    long long mine = start + warp;  // this warp's next step
    int stage = 0;
    uint32_t parity = 0;
    bool alive = true;
    for (long long pos = start; pos < end;) {
        stream_seek<D>(a, cur, pos);
        const long long seg_end = min(end, cur.u0 + cur.n);
        const Kv4Request r = cur.r;
        const int ncols = r.qn * a.group;

        // ---------------- the unit's query columns: power-of-two scale, F16, fragment order
        __syncthreads();
        for (int c = warp; c < COLS; c += kStWarps) {
            constexpr int E = D / 32;
            float x[E];
            const int qi = c / a.group, hh = cur.h * a.group + c % a.group;
            float top = 0.0f;
#pragma unroll
            for (int e = 0; e < E; e++) x[e] = 0.0f;
            if (c < ncols) {
                const long long at = (r.q0 + qi) * a.qts + hh * a.qhs + lane * E;
                if (a.qvec && E >= 4) {
#pragma unroll
                    for (int e = 0; e < E; e += 4) {
                        float v4[4];
                        load_act4(a.q, (size_t)(at + e), a.dt, v4);
#pragma unroll
                        for (int j = 0; j < 4 && e + j < E; j++) x[e + j] = v4[j];
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < E; e++) x[e] = load_act(a.q, (size_t)(at + e), a.dt);
                }
            }
#pragma unroll
            for (int e = 0; e < E; e++) top = fmaxf(top, fabsf(x[e]));
#pragma unroll
            for (int m = 16; m > 0; m >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, m));
            // 2^k with top * 2^k in [2^13, 2^14); 1 for a column of zeros or without a finite maximum
            int k = 0;
            if (top > 0.0f && top < 3.0e38f) k = min(max(13 - ((int)(__float_as_uint(top) >> 23) - 127), -120), 120);
            const float up = __uint_as_float((uint32_t)(k + 127) << 23);
            float sum = 0.0f;
#pragma unroll
            for (int e = 0; e < E; e++) {
                const int ch = lane * E + e, n = ch & 7;
                const bool odd = n & 1;
                const __half hq = __float2half_rn(odd ? x[e] * up * 0.0625f : x[e] * up);
                sum += odd ? __half2float(hq) * 16.0f : __half2float(hq);
                // fragment order of a word: nibbles 0 4 2 6 1 5 3 7
                const int place = ((n & 1) << 2) | (n & 2) | (n >> 2);
                reinterpret_cast<__half*>(smem + L::Q)[c * D + (ch & ~7) + place] = hq;
            }
            // the group's sum: 64 / E lanes hold it
#pragma unroll
            for (int m = 32 / G / 2; m > 0; m >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, m);
            if (lane % (32 / G) == 0) qs_sm[c * G + lane / (32 / G)] = sum * 5.9604644775390625e-08f;  // 2^-24
            if (lane == 0) ch_sm[c] = a.scale_log2 * 16777216.0f * __uint_as_float((uint32_t)(127 - k) << 23);
        }
        __syncthreads();
        float qs[NT][2][G], chs[NT][2];
        int qpos[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const int c = nt * 8 + 2 * t + j;
                chs[nt][j] = ch_sm[c];
                qpos[nt][j] = r.pos0 + (c < ncols ? c / a.group : 0);
#pragma unroll
                for (int gr = 0; gr < G; gr++) qs[nt][j][gr] = qs_sm[c * G + gr];
            }

        // ---------------- this warp's steps of the segment
        float o[G][4][NT][4], mn[G][NT][2], l[NT][2], mref[NT][2];
        float se = -26.0f, sthr = 0.0f;  // steps seen so far are at most sthr = 2^se
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int j = 0; j < 2; j++) {
                l[nt][j] = 0.0f;
                mref[nt][j] = -1.0e30f;
#pragma unroll
                for (int gr = 0; gr < G; gr++) mn[gr][nt][j] = 0.0f;
            }
#pragma unroll
        for (int gr = 0; gr < G; gr++)
#pragma unroll
            for (int mt = 0; mt < 4; mt++)
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int j = 0; j < 4; j++) o[gr][mt][nt][j] = 0.0f;

        for (; mine < seg_end; mine += kStWarps) {
            if (alive) alive = mbar_wait(&bar[stage], parity, DEV_TIMEOUT_FULL);
            const uint8_t* st = ring + stage * L::STEP;
            const int p0 = r.lo + (int)(mine - cur.u0) * GS * kKvGranule;
            const uint32_t vm = (valid >> (4 * stage)) & 15u;
            // every key of the step seen by every row?
            const bool full = vm == (1u << GS) - 1 && p0 + GS * kKvGranule <= min(r.hi, r.pos0 + 1) &&
                              (a.window == 0 || p0 > r.pos0 + r.qn - 1 - a.window);

            // scores
            float s[GS][NT][4];
#pragma unroll
            for (int gi = 0; gi < GS; gi++) {
                const uint8_t* gran = st + gi * L::GB;
                float acc[G][NT][4];
                uint32_t kw[2][G][2];
#pragma unroll
                for (int rr = 0; rr < 2; rr++) {
                    const int tok = tok0 + 8 * rr;
                    if constexpr (D == 64) {
                        const uint2 u = *reinterpret_cast<const uint2*>(gran + kv4_key_word<D>(tok, 0, 2 * t));
                        kw[rr][0][0] = u.x, kw[rr][0][1] = u.y;
                    } else {
#pragma unroll
                        for (int gr = 0; gr < G; gr += 2) {
                            const uint4 u = *reinterpret_cast<const uint4*>(gran + kv4_key_word<D>(tok, gr, 2 * t));
                            kw[rr][gr][0] = u.x, kw[rr][gr][1] = u.y, kw[rr][gr + 1][0] = u.z, kw[rr][gr + 1][1] = u.w;
                        }
                    }
                }
#pragma unroll
                for (int gr = 0; gr < G; gr++) {
#pragma unroll
                    for (int nt = 0; nt < NT; nt++)
#pragma unroll
                        for (int j = 0; j < 4; j++) acc[gr][nt][j] = 0.0f;
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        const uint32_t x0 = kw[0][gr][i], x1 = kw[1][gr][i], y0 = x0 >> 8, y1 = x1 >> 8;
#pragma unroll
                        for (int nt = 0; nt < NT; nt++) {
                            const uint4 qb = *reinterpret_cast<const uint4*>(smem + L::Q +
                                                                             ((nt * 8 + g) * D + gr * 64 + (2 * t + i) * 8) * 2);
                            mma16816(acc[gr][nt], x0 & 0x000f000fu, x1 & 0x000f000fu, y0 & 0x000f000fu, y1 & 0x000f000fu, qb.x, qb.y);
                            mma16816(acc[gr][nt], x0 & 0x00f000f0u, x1 & 0x00f000f0u, y0 & 0x00f000f0u, y1 & 0x00f000f0u, qb.z, qb.w);
                        }
                    }
                }
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int j = 0; j < 4; j++) s[gi][nt][j] = 0.0f;
#pragma unroll
                for (int gr = 0; gr < G; gr++)
#pragma unroll
                    for (int rr = 0; rr < 2; rr++) {
                        const __half2 par = *reinterpret_cast<const __half2*>(gran + kv4_kpar_off(D) + ((tok0 + 8 * rr) * G + gr) * 4);
                        const float2 f = __half22float2(par);
#pragma unroll
                        for (int nt = 0; nt < NT; nt++)
#pragma unroll
                            for (int j = 0; j < 2; j++)
                                s[gi][nt][2 * rr + j] = fmaf(f.y, qs[nt][j][gr], fmaf(f.x, acc[gr][nt][2 * rr + j], s[gi][nt][2 * rr + j]));
                    }
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int j = 0; j < 4; j++) s[gi][nt][j] *= chs[nt][j & 1];
            }
            if (!full) {
#pragma unroll
                for (int gi = 0; gi < GS; gi++)
#pragma unroll
                    for (int rr = 0; rr < 2; rr++) {
                        const int key = p0 + gi * kKvGranule + tok0 + 8 * rr;
#pragma unroll
                        for (int nt = 0; nt < NT; nt++)
#pragma unroll
                            for (int j = 0; j < 2; j++)
                                if (!((vm >> gi) & 1u) || key >= r.hi || key > qpos[nt][j] ||
                                    (a.window > 0 && key <= qpos[nt][j] - a.window))
                                    s[gi][nt][2 * rr + j] = -CUDART_INF_F;
                    }
            }

            // the values' steps and minima of this lane's keys (0 for keys that no row sees)
            float vs[GS][2][G], vmn[GS][2][G];
            float smax = 0.0f;
#pragma unroll
            for (int gi = 0; gi < GS; gi++)
#pragma unroll
                for (int rr = 0; rr < 2; rr++) {
                    const int key = p0 + gi * kKvGranule + tok0 + 8 * rr;
                    const bool seen = full || (((vm >> gi) & 1u) && key < r.hi);
#pragma unroll
                    for (int gr = 0; gr < G; gr++) {
                        const __half2 par =
                            *reinterpret_cast<const __half2*>(st + gi * L::GB + kv4_vpar_off(D) + ((tok0 + 8 * rr) * G + gr) * 4);
                        const float2 f = __half22float2(par);
                        vs[gi][rr][gr] = seen ? f.x : 0.0f;
                        vmn[gi][rr][gr] = seen ? f.y : 0.0f;
                        smax = fmaxf(smax, vs[gi][rr][gr]);
                    }
                }
            float over = -CUDART_INF_F;
#pragma unroll
            for (int gi = 0; gi < GS; gi++)
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int j = 0; j < 4; j++) over = fmaxf(over, s[gi][nt][j] - mref[nt][j & 1]);
            if (__any_sync(0xffffffffu, over > 15.0f - se || smax > sthr)) {
                // move the references: each column's best score at 2^(11 - se)
#pragma unroll
                for (int m = 16; m > 0; m >>= 1) smax = fmaxf(smax, __shfl_xor_sync(0xffffffffu, smax, m));
                float se_new = se;
                if (smax > sthr) {
                    const int e = min(max((int)(__float_as_uint(smax) >> 23) - 126, -24), 17);
                    se_new = (float)e;
                    sthr = __uint_as_float((uint32_t)(e + 127) << 23);
                }
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        float best = -CUDART_INF_F;
#pragma unroll
                        for (int gi = 0; gi < GS; gi++) best = fmaxf(best, fmaxf(s[gi][nt][j], s[gi][nt][j + 2]));
#pragma unroll
                        for (int m = 4; m < 32; m <<= 1) best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, m));
                        const float moved = fmaxf(mref[nt][j] + (se_new - se), best - (11.0f - se_new));
                        const float f = ex2(mref[nt][j] - moved);
                        mref[nt][j] = moved;
                        l[nt][j] *= f;
#pragma unroll
                        for (int gr = 0; gr < G; gr++) {
                            mn[gr][nt][j] *= f;
#pragma unroll
                            for (int mt = 0; mt < 4; mt++) {
                                o[gr][mt][nt][j] *= f;
                                o[gr][mt][nt][j + 2] *= f;
                            }
                        }
                    }
                se = se_new;
            }

            // probabilities and values
#pragma unroll
            for (int gi = 0; gi < GS; gi++) {
                const uint8_t* gran = st + gi * L::GB;
                uint32_t pb[G][NT][2];
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    float p[4];
#pragma unroll
                    for (int j = 0; j < 4; j++) p[j] = ex2(s[gi][nt][j] - mref[nt][j & 1]);
                    l[nt][0] += p[0] + p[2];
                    l[nt][1] += p[1] + p[3];
#pragma unroll
                    for (int gr = 0; gr < G; gr++)
#pragma unroll
                        for (int rr = 0; rr < 2; rr++) {
                            float a0 = p[2 * rr] * vs[gi][rr][gr], a1 = p[2 * rr + 1] * vs[gi][rr][gr];
                            float b0 = p[2 * rr] * vmn[gi][rr][gr], b1 = p[2 * rr + 1] * vmn[gi][rr][gr];
                            if (!full) {  // a key one row sees and another does not may hold NaN
                                if (p[2 * rr] == 0.0f) a0 = b0 = 0.0f;
                                if (p[2 * rr + 1] == 0.0f) a1 = b1 = 0.0f;
                            }
                            mn[gr][nt][0] += b0;
                            mn[gr][nt][1] += b1;
                            const __half2 h2 = __floats2half2_rn(a0, a1);
                            pb[gr][nt][rr] = movmatrix(*reinterpret_cast<const uint32_t*>(&h2));
                        }
                }
                uint32_t vw[4][G];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const uint8_t* w = gran + kv4_value_word<D>(vt[j], 0, g);
                    if constexpr (D == 64) {
                        vw[j][0] = *reinterpret_cast<const uint32_t*>(w);
                    } else if constexpr (D == 128) {
                        const uint2 u = *reinterpret_cast<const uint2*>(w);
                        vw[j][0] = u.x, vw[j][1] = u.y;
                    } else {
                        const uint4 u = *reinterpret_cast<const uint4*>(w);
                        vw[j][0] = u.x, vw[j][1] = u.y, vw[j][2] = u.z, vw[j][3] = u.w;
                    }
                }
#pragma unroll
                for (int gr = 0; gr < G; gr++) {
                    const uint32_t w01[2] = {__byte_perm(vw[0][gr], vw[1][gr], 0x5410), __byte_perm(vw[0][gr], vw[1][gr], 0x7632)};
                    const uint32_t w23[2] = {__byte_perm(vw[2][gr], vw[3][gr], 0x5410), __byte_perm(vw[2][gr], vw[3][gr], 0x7632)};
#pragma unroll
                    for (int mt = 0; mt < 4; mt++) {
                        const uint32_t x = w01[mt >> 1] >> (8 * (mt & 1)), y = w23[mt >> 1] >> (8 * (mt & 1));
#pragma unroll
                        for (int nt = 0; nt < NT; nt++)
                            mma16816(o[gr][mt][nt], x & 0x000f000fu, x & 0x00f000f0u, y & 0x000f000fu, y & 0x00f000f0u,
                                     pb[gr][nt][0], pb[gr][nt][1]);
                    }
                }
            }
            __syncwarp();
            issue(stage);
            if (++stage == kStStages) stage = 0, parity ^= 1u;
        }

        // ---------------- the warps' sums into one: common reference, then f32 adds in warp order
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int j = 0; j < 2; j++) {
#pragma unroll
                for (int m = 4; m < 32; m <<= 1) {
                    l[nt][j] += __shfl_xor_sync(0xffffffffu, l[nt][j], m);
#pragma unroll
                    for (int gr = 0; gr < G; gr++) mn[gr][nt][j] += __shfl_xor_sync(0xffffffffu, mn[gr][nt][j], m);
                }
                if (g == 0) {
                    m_sm[warp * COLS + nt * 8 + 2 * t + j] = mref[nt][j];
                    l_sm[warp * COLS + nt * 8 + 2 * t + j] = l[nt][j];
                }
            }
        __syncthreads();
        const bool whole = pos == cur.u0 && seg_end == cur.u0 + cur.n;
        float* slot = a.part + (size_t)(2 * cta + (pos == start ? 0 : 1)) * (16 * (D + 2));
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const int c = nt * 8 + 2 * t + j;
                float top = m_sm[c];
#pragma unroll
                for (int w = 1; w < kStWarps; w++) top = fmaxf(top, m_sm[w * COLS + c]);
                const float f = ex2(mref[nt][j] - top);
#pragma unroll
                for (int gr = 0; gr < G; gr++) {
                    float v[8];
#pragma unroll
                    for (int mt = 0; mt < 4; mt++) {
                        v[2 * mt] = f * fmaf(o[gr][mt][nt][j], 16777216.0f, mn[gr][nt][j]);
                        v[2 * mt + 1] = f * fmaf(o[gr][mt][nt][j + 2], 1048576.0f, mn[gr][nt][j]);
                    }
                    float4* dst = reinterpret_cast<float4*>(merge + (warp * 8 + 2 * t + j) * L::ROW + gr * 64 + g * 8);
                    dst[0] = make_float4(v[0], v[1], v[2], v[3]);
                    dst[1] = make_float4(v[4], v[5], v[6], v[7]);
                }
            }
            __syncthreads();
            for (int i = tid; i < 8 * (D / 8); i += kStThreads) {
                const int cc = i / (D / 8), ch = (i % (D / 8)) * 8, c = nt * 8 + cc;
                if (c >= ncols) continue;
                float top = m_sm[c], ls = 0.0f;
#pragma unroll
                for (int w = 1; w < kStWarps; w++) top = fmaxf(top, m_sm[w * COLS + c]);
#pragma unroll
                for (int w = 0; w < kStWarps; w++) ls += ex2(m_sm[w * COLS + c] - top) * l_sm[w * COLS + c];
                float v[8] = {};
#pragma unroll
                for (int w = 0; w < kStWarps; w++) {
                    const float4* src = reinterpret_cast<const float4*>(merge + (w * 8 + cc) * L::ROW + ch);
                    const float4 x = src[0], y = src[1];
                    v[0] += x.x, v[1] += x.y, v[2] += x.z, v[3] += x.w, v[4] += y.x, v[5] += y.y, v[6] += y.z, v[7] += y.w;
                }
                if (whole) {
                    const float inv = ls == 0.0f ? 0.0f : 1.0f / ls;
                    const size_t at = ((size_t)(r.q0 + c / a.group) * a.heads + cur.h * a.group + c % a.group) * D + ch;
                    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + at) =
                        make_uint4(pack_act2(v[0] * inv, v[1] * inv, a.dt), pack_act2(v[2] * inv, v[3] * inv, a.dt),
                                   pack_act2(v[4] * inv, v[5] * inv, a.dt), pack_act2(v[6] * inv, v[7] * inv, a.dt));
                } else {
                    float4* dst = reinterpret_cast<float4*>(slot + c * D + ch);
                    __stcg(dst, make_float4(v[0], v[1], v[2], v[3]));
                    __stcg(dst + 1, make_float4(v[4], v[5], v[6], v[7]));
                    if (ch == 0) {
                        __stcg(slot + 16 * D + 2 * c, top);
                        __stcg(slot + 16 * D + 2 * c + 1, ls);
                    }
                }
            }
            __syncthreads();
        }

        if (!whole) {
            // CTAs first .. last share the unit; the first's counter counts them in
            const int first = (int)(((cur.u0 + 1) * ctas - 1) / total);
            const int last = (int)(((cur.u0 + cur.n) * ctas - 1) / total);
            if (tid == 0) {
                __threadfence();
                arrived = atomicAdd(&a.count[first], 1);
            }
            __syncthreads();
            if (arrived == last - first) {
                __threadfence();
                if (tid == 0) a.count[first] = 0;
                const size_t stride = 16 * (D + 2);
                auto slot_of = [&](int c) {
                    return a.part + (size_t)(2 * c + (c == first && total * c / ctas != cur.u0 ? 1 : 0)) * stride;
                };
                for (int i = tid; i < ncols * (D / 4); i += kStThreads) {
                    const int c = i / (D / 4), ch = (i % (D / 4)) * 4;
                    float top = -1.0e30f;
#pragma unroll 4
                    for (int k = first; k <= last; k++) top = fmaxf(top, __ldcg(slot_of(k) + 16 * D + 2 * c));
                    float ls = 0.0f;
                    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
                    for (int k = first; k <= last; k++) {
                        const float* sl = slot_of(k);
                        const float2 ml = __ldcg(reinterpret_cast<const float2*>(sl + 16 * D + 2 * c));
                        const float4 x = __ldcg(reinterpret_cast<const float4*>(sl + c * D + ch));
                        const float f = ex2(ml.x - top);
                        ls += f * ml.y;
                        v.x += f * x.x, v.y += f * x.y, v.z += f * x.z, v.w += f * x.w;
                    }
                    const float inv = ls == 0.0f ? 0.0f : 1.0f / ls;
                    const size_t at = ((size_t)(r.q0 + c / a.group) * a.heads + cur.h * a.group + c % a.group) * D + ch;
                    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + at) =
                        make_uint2(pack_act2(v.x * inv, v.y * inv, a.dt), pack_act2(v.z * inv, v.w * inv, a.dt));
                }
            }
        }
        pos = seg_end;
    }
}

namespace {

template <int D, int NT>
int stream_ctas() {
    // CTAs an SM holds by shared memory (registers allow as many)
    return std::min(4, (227 * 1024) / (StreamLayout<D, NT>::TOTAL + 1024)) * sm_count();
}

template <int D, int NT>
cudaError_t stream_launch(const Kv4AttnArgs& a, cudaStream_t stream) {
    using L = StreamLayout<D, NT>;
    auto kern = kv4_stream_kernel<D, NT>;
    cudaError_t e = func_attrs(reinterpret_cast<const void*>(kern), L::TOTAL, false);
    if (e != cudaSuccess) return e;
    kern<<<stream_ctas<D, NT>(), kStThreads, L::TOTAL, stream>>>(a);
    return cudaGetLastError();
}

}  // namespace

cudaError_t kv4_stream_launch(const Kv4AttnArgs& a, int D, cudaStream_t stream) {
    const bool one = a.max_cols <= 8;
    if (D == 64) return one ? stream_launch<64, 1>(a, stream) : stream_launch<64, 2>(a, stream);
    if (D == 128) return one ? stream_launch<128, 1>(a, stream) : stream_launch<128, 2>(a, stream);
    return one ? stream_launch<256, 1>(a, stream) : stream_launch<256, 2>(a, stream);
}

}  // namespace sx
