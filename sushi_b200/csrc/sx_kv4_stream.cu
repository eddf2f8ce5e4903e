// Attention over the 4-bit cache for requests of few rows: one token, a few drafted ones.
//
// A unit is one request and key head; its columns are (row, query head) pairs that read that key head, 8 NT
// at most (more pairs make more units).  With 16 keys on the M axis and the columns on the N axis of m16n8k16:
//   S^T[key][col] = sum over groups g of  s_kg * (codes . q) + m_kg * (sum of q in g)
//   O^T[channel][col] = codes^T . (P * s_g) + sum over keys of P * m_g
// so the products take the codes themselves: a code masked out of its word is the F16 subnormal
// code * 2^-24 (or code * 2^-20 for every second nibble), exact, with no conversion.  The query is
// scaled by a power of two per column (its largest entry to [2^13, 2^14)) and by 1/16 where the
// nibble brings 16, and rounded to F16 (exact for bf16 and f16 entries within 2^24 of the largest).
// P * s is rounded to F16 (h), once for bf16 calls.  Against the whole code that rounding would count
// up to three times the value it stands for, since code * s and m nearly cancel; so the minima's sum takes
// P (m + 7.5 s) - 7.5 h, and what h lost counts against code - 7.5, which is of the value's size: 1.68e-3 off where
// the bf16 output's own rounding is 1.67e-3 (1.74e-3 without; 114 -> 117 us for 64 requests).  F16 calls keep P * s
// in two F16 parts with a second product (FINE; 2.09e-4 off of 2.08e-4).  m, sums and accumulators are f32.
//
// The MMA's f32 sums, and the products within one, are cut, not rounded.  Codes are 0 to 15, so over a long cache
// the codes' part and the minima's are hundreds of times their sum, the output, and what is cut of the one always has
// its sign: at 131072 keys a CTA outputs were 5% off.  So every second granule is turned over: 15 - code (the
// complement of the word, which costs nothing beside the masks) times -P * s, and P (m + 15 s) among the minima (bf16:
// the 7.5 of above already does that).  The sums then stay near 0 and the cuts cancel; and every 16 steps the minima's
// part moves into them, so that what is left does not depend on the length (131072 keys a CTA, relative: bf16 1.64e-3,
// of which the output's own rounding is 1.63e-3; F16 2.2e-4 of 2.1e-4).
//
// The softmax reference of a column is kept so that P * s <= 2^15, whatever the values' magnitude:
// it moves (one vote a step) only when a score or a step would pass that, with 2^4 to spare.
//
// Work: the units' steps (4.5 KB of one head: 256/D granules of 16 tokens) laid end to end and cut
// into equal runs, one a CTA, so ragged lengths balance; a CTA's warps take its steps in turn, each
// with its own ring of bulk copies.  A unit that several CTAs share is joined by sx_kv4_join.cu.
//
// Bound by instructions (633 a step of 32 keys, 56% of the issue slots, ALU pipe 50% busy), by HBM close behind (5 TB/s
// while all CTAs stream).  With the join: 64 requests of 1024 to 16384 keys and 8 key heads of 128 (480 MB) 117 us, one
// of 131071 keys (151 MB) 51 us, one of 517 keys and 2 key heads 9.1 us.  D = 256 with two column tiles runs at 255
// registers and spills (208 bytes a thread, 280 in F16): 16 requests of 4 drafted tokens, 8 query heads a key head, 51 us.
#include <cuda_runtime.h>
#include <math_constants.h>

#include <algorithm>
#include <type_traits>

#include "sx_kv4_attn.cuh"

namespace sx {

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

// A walk over the units' steps: request b, key head h, block k of its blocks; the unit's n steps (n = 0, or the empty ones among
// them) begin at step `beg` of this CTA's run (negative where the unit began in an earlier CTA's).
struct StreamCursor {
    Kv4Request r;
    int b, h, k, blocks, n, beg;
};

template <int D>
__device__ __forceinline__ void stream_load(const Kv4AttnArgs& a, StreamCursor& c) {
    c.r = kv4_request(a, c.b);
    c.n = stream_list(stream_steps<D>(a, c.r));
    c.blocks = stream_blocks(a, c.r);
}

// Moves the cursor forward to the unit that holds step i of the run.
template <int D>
__device__ __forceinline__ void stream_seek(const Kv4AttnArgs& a, StreamCursor& c, int i) {
    while (i >= c.beg + c.n) {
        c.beg += c.n;
        if (++c.k >= c.blocks || c.n == 0) {
            c.k = 0;
            if (++c.h >= a.kv_heads || c.n == 0) {
                c.h = 0;
                c.b++;
                stream_load<D>(a, c);
            }
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

// A token's parameters (step, minimum) of every group.
template <int G>
__device__ __forceinline__ void load_params(const uint8_t* p, float2 (&f)[G]) {
    uint32_t w[G];
    if constexpr (G == 1) {
        w[0] = *reinterpret_cast<const uint32_t*>(p);
    } else if constexpr (G == 2) {
        const uint2 u = *reinterpret_cast<const uint2*>(p);
        w[0] = u.x, w[1] = u.y;
    } else {
        const uint4 u = *reinterpret_cast<const uint4*>(p);
        w[0] = u.x, w[1] = u.y, w[2] = u.z, w[3] = u.w;
    }
#pragma unroll
    for (int gr = 0; gr < G; gr++) f[gr] = __half22float2(*reinterpret_cast<const __half2*>(&w[gr]));
}

template <int D, int NT>
__host__ __device__ constexpr int stream_resident() {
    return NT == 1 && D <= 128 ? 3 : 2;
}

template <int D, int NT, bool FINE>
__global__ void __launch_bounds__(kStThreads, stream_resident<D, NT>()) kv4_stream_kernel(Kv4AttnArgs a) {
    using L = StreamLayout<D, NT>;
    constexpr int G = L::G, GS = L::GS, COLS = L::COLS;
    constexpr int MOVE = 16;  // steps between two moves of the minima's part
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ int red[kStWarps], pick[2];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int g = lane >> 2, t = lane & 3;
    uint64_t* bar = reinterpret_cast<uint64_t*>(smem + L::BAR) + warp * kStStages;
    uint8_t* ring = smem + L::RING + warp * kStStages * L::STEP;
    if (lane == 0)
        for (int i = 0; i < kStStages; i++) mbar_init(&bar[i], 1);
    fence_mbar_init();

    // ---------------- the list: its length, then the unit of this CTA's first step
    pdl_release();
    const int cta = blockIdx.x;
    const int past = min(max(a.cu_q[a.requests], 0), a.tokens);  // rows from here on belong to no request
    // no unit writes the rows of a request without a key to see (0), nor of one past the call's max_q that only the
    // tile kernel could take (NaN): CTA b % grid does
    auto wide = [&](const Kv4Request& r) { return r.qn * (long long)a.group > a.max_cols; };
    auto keyless = [&](const Kv4Request& r) { return r.qn > 0 && r.hi <= r.lo && !wide(r); };
    bool zeros = false;
    auto steps = [&](int b) {
        const Kv4Request r = kv4_request(a, b);
        const int n = stream_steps<D>(a, r);
        if ((keyless(r) || (a.alone && wide(r))) && b % (int)gridDim.x == cta) zeros = true;
        return n > 0 ? stream_list(n) * a.kv_heads * stream_blocks(a, r) : 0;
    };
    int n0;
    const int total = list_total<kStWarps>(a.requests, red, n0, zeros, steps);
    for (int b = cta; zeros && b < a.requests; b += gridDim.x) {
        const Kv4Request r = kv4_request(a, b);
        if (!keyless(r) && !(a.alone && wide(r))) continue;
        const uint32_t fill = wide(r) ? 0x7fff7fffu : 0u;  // NaN in both types
        uint4* o = reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + (size_t)r.q0 * a.heads * D);
        for (size_t i = tid; i < (size_t)r.qn * a.heads * D / 8; i += kStThreads) o[i] = make_uint4(fill, fill, fill, fill);
    }
    const RunCut run(total, stream_most(total, gridDim.x));
    if (past < a.tokens) {
        uint4* o = reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + (size_t)past * a.heads * D);
        const size_t n = (size_t)(a.tokens - past) * a.heads * D / 8;
        for (size_t i = (size_t)cta * kStThreads + tid; i < n; i += (size_t)gridDim.x * kStThreads) o[i] = make_uint4(0, 0, 0, 0);
    }
    if (total == 0 || cta >= run.ctas) return;
    const int start = run.start(cta);
    const int len = run.start(cta + 1) - start;  // this CTA's run
    list_find<kStWarps>(a.requests, red, pick, n0, start, steps);
    StreamCursor cur;
    cur.b = pick[0];
    stream_load<D>(a, cur);
    const int into = start - pick[1];
    const int unit = into / cur.n;
    cur.h = unit / cur.blocks;
    cur.k = unit - cur.h * cur.blocks;
    cur.beg = unit * cur.n - into;
    StreamCursor ahead = cur;

    // ---------------- this warp's ring: step warp + 4 k of the run in stage k % S.  A step's page ids (a
    // load of their own, lane by lane) and places are looked up a step ahead of its copies.
    uint32_t valid = 0;  // 4 bits a stage: the granules that were copied
    int next = warp, page = -1;
    size_t place = 0;
    auto look = [&]() {
        page = -1;
        while (next < len) {  // past the empty steps
            stream_seek<D>(a, ahead, next);
            const int skip = ahead.beg + kStPad - next;
            if (skip <= 0) break;
            next += (skip + kStWarps - 1) / kStWarps * kStWarps;
        }
        if (next < len) {
            const int pos = ahead.r.lo + ((next - ahead.beg - kStPad) * GS + lane) * kKvGranule;
            if (lane < GS && pos < ahead.r.hi) page = a.table[ahead.b * a.tstride + (pos >> a.shift)];
            place = kv4_granule<D>(0, a.kv_heads, ahead.h, a.page_size, pos & (a.page_size - 1));
        }
    };
    const size_t page_bytes = kv4_granule<D>(1, a.kv_heads, 0, a.page_size, 0);
    auto issue = [&](int st) {
        if (next < len) {
            const bool ok = page >= 0 && page < a.pages;
            const uint32_t m = __ballot_sync(0xffffffffu, ok);
            if (lane == 0) mbar_arrive_expect_tx(&bar[st], __popc(m) * L::GB);
            __syncwarp();
            if (ok) bulk_g2s(ring + st * L::STEP + lane * L::GB, a.pool + page * page_bytes + place, L::GB, &bar[st]);
            valid = (valid & ~(15u << (4 * st))) | (m << (4 * st));
            next += kStWarps;
            look();
        }
    };
    // a unit's query entries of this warp's columns, loaded while the unit before is merged (where the
    // registers allow)
    constexpr int E = D / 32, CW = COLS / kStWarps;  // entries a lane, columns a warp
    constexpr bool EARLY = E * CW <= 8;
    float x[CW][E];
    auto load_columns = [&]() {
        const int n = cur.r.qn * a.group, h = cur.h, e0 = cur.k * a.cols;
#pragma unroll
        for (int w = 0; w < CW; w++) {
            const int c = e0 + warp + w * kStWarps;
#pragma unroll
            for (int e = 0; e < E; e++) x[w][e] = 0.0f;
            if (c < n && warp + w * kStWarps < a.cols) {
                const int qi = c / a.group, hh = h * a.group + c - qi * a.group;
                const long long at = (cur.r.q0 + qi) * a.qts + hh * a.qhs + lane * E;
                if (a.qvec && E >= 4) {
#pragma unroll
                    for (int e = 0; e < E; e += 4) {
                        float v4[4];
                        load_act4(a.q, (size_t)(at + e), a.dt, v4);
#pragma unroll
                        for (int j = 0; j < 4 && e + j < E; j++) x[w][e + j] = v4[j];
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < E; e++) x[w][e] = load_act(a.q, (size_t)(at + e), a.dt);
                }
            }
        }
    };
    if (EARLY) load_columns();
    look();
#pragma unroll
    for (int i = 0; i < kStStages; i++) issue(i);

    float* qs_sm = reinterpret_cast<float*>(smem + L::QS);
    float* ch_sm = reinterpret_cast<float*>(smem + L::CH);
    float* m_sm = reinterpret_cast<float*>(smem + L::ML);
    float* l_sm = m_sm + kStWarps * COLS;
    float* merge = reinterpret_cast<float*>(smem + L::MERGE);
    const int tok0 = row_token(g);                   // fragment row g; row g + 8 is token tok0 + 8
    const uint8_t* q_lane = smem + L::Q + (g * D + 2 * t * 8) * 2;
    const int vt[4] = {t, 4 + (t ^ 1), 8 + t, 12 + (t ^ 1)};  // rows 2t, 2t+1, 2t+8, 2t+9

    int mine = warp;  // this warp's next step of the run
    int stage = 0;
    uint32_t parity = 0;
    bool alive = true;
    for (int pos = 0; pos < len;) {
        const int seg_end = min(len, cur.beg + cur.n);
        const Kv4Request r = cur.r;
        const int beg = cur.beg + kStPad, n = cur.n - kStPad, head = cur.h;
        const int e0 = cur.k * a.cols;  // the unit's first pair
        const int ncols = min(a.cols, r.qn * a.group - e0);
        const int from = max(pos, beg);  // steps [from, seg_end) are this CTA's
        if (from >= seg_end) break;      // the run ends among the unit's empty steps
        if (mine < from) mine += (from - mine + kStWarps - 1) / kStWarps * kStWarps;

        // ---------------- the unit's query columns: power-of-two scale, F16, fragment order
        if (!EARLY) load_columns();
        __syncthreads();
#pragma unroll
        for (int w = 0; w < CW; w++) {
            const int c = warp + w * kStWarps;
            float top = 0.0f;
#pragma unroll
            for (int e = 0; e < E; e++) top = fmaxf(top, fabsf(x[w][e]));
            top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top)));  // entries of no sign order as integers
            const int k = query_scale(top);
            const float up = __uint_as_float((uint32_t)(k + 127) << 23);
            float sum = 0.0f;
#pragma unroll
            for (int e = 0; e < E; e++) {
                const int ch = lane * E + e, n = ch & 7;
                const bool odd = n & 1;
                const __half hq = __float2half_rn(odd ? x[w][e] * up * 0.0625f : x[w][e] * up);
                sum += odd ? __half2float(hq) * 16.0f : __half2float(hq);
                // fragment order of a word: nibbles 0 4 2 6 1 5 3 7
                const int place = ((n & 1) << 2) | (n & 2) | (n >> 2);
                reinterpret_cast<__half*>(smem + L::Q)[c * D + (ch & ~7) + place] = hq;
            }
            // the group's sum: 64 / E lanes hold it
#pragma unroll
            for (int m = 32 / G / 2; m > 0; m >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, m);
            if (lane % (32 / G) == 0) qs_sm[c * G + lane / (32 / G)] = sum * 5.9604644775390625e-08f;  // 2^-24
            // (codes * s and m below 2^16, the query below 2^14, 2^8 channels, 2^-24)
            if (lane == 0) ch_sm[c] = kv4_most_scale(a.scale_log2 * 16777216.0f * __uint_as_float((uint32_t)(127 - k) << 23), 16);
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
                qpos[nt][j] = r.pos0 + (e0 + (c < ncols ? c : 0)) / a.group;
#pragma unroll
                for (int gr = 0; gr < G; gr++) qs[nt][j][gr] = qs_sm[c * G + gr];
            }

        // ---------------- this warp's steps of the segment
        float o[G][4][NT][4], mn[G][NT][2], l[NT][2], mref[NT][2], thr[NT][2];
        float sthr = 0.0f, lim = 41.0f;  // steps so far are at most sthr; a score may pass its reference by lim
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int j = 0; j < 2; j++) {
                l[nt][j] = 0.0f;
                mref[nt][j] = thr[nt][j] = kNoScore;
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

        // steps at positions [full_lo, full_hi) are seen whole by every row
        const int full_hi = min(r.hi, r.pos0 + 1) - GS * kKvGranule;
        const int full_lo = a.window > 0 ? r.pos0 + r.qn - a.window : 0;
        auto step = [&](const uint8_t* st, int p0, uint32_t vm, auto whole_step) {
            constexpr bool FULL = decltype(whole_step)::value;
            const bool odd_step = mine / kStWarps & 1;
            // scores
            float x[GS][NT][4];
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
                            const uint4 qb = *reinterpret_cast<const uint4*>(q_lane + nt * 8 * D * 2 + (gr * 64 + i * 8) * 2);
                            mma16816(acc[gr][nt], x0 & 0x000f000fu, x1 & 0x000f000fu, y0 & 0x000f000fu, y1 & 0x000f000fu, qb.x, qb.y);
                            mma16816(acc[gr][nt], x0 & 0x00f000f0u, x1 & 0x00f000f0u, y0 & 0x00f000f0u, y1 & 0x00f000f0u, qb.z, qb.w);
                        }
                    }
                }
                float2 par[2][G];
#pragma unroll
                for (int rr = 0; rr < 2; rr++) load_params<G>(gran + kv4_kpar_off(D) + (tok0 + 8 * rr) * G * 4, par[rr]);
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        float v = par[j >> 1][0].y * qs[nt][j & 1][0];
                        v = fmaf(par[j >> 1][0].x, acc[0][nt][j], v);
#pragma unroll
                        for (int gr = 1; gr < G; gr++)
                            v = fmaf(par[j >> 1][gr].x, acc[gr][nt][j], fmaf(par[j >> 1][gr].y, qs[nt][j & 1][gr], v));
                        x[gi][nt][j] = v * chs[nt][j & 1];
                    }
            }
            // the values' steps and minima of this lane's keys
            float2 vpar[GS][2][G];
            float smax = 0.0f;
#pragma unroll
            for (int gi = 0; gi < GS; gi++)
#pragma unroll
                for (int rr = 0; rr < 2; rr++) {
                    load_params<G>(st + gi * L::GB + kv4_vpar_off(D) + (tok0 + 8 * rr) * G * 4, vpar[gi][rr]);
                    if constexpr (!FULL) {
                        // keys a column does not see score -inf; keys no row sees weigh 0 whatever they hold
                        const int key = p0 + gi * kKvGranule + tok0 + 8 * rr;
                        const bool here = ((vm >> gi) & 1u) && key < r.hi;
#pragma unroll
                        for (int nt = 0; nt < NT; nt++)
#pragma unroll
                            for (int j = 0; j < 2; j++)
                                if (!here || key > qpos[nt][j] || (a.window > 0 && key <= qpos[nt][j] - a.window))
                                    x[gi][nt][2 * rr + j] = -CUDART_INF_F;
#pragma unroll
                        for (int gr = 0; gr < G; gr++)
                            if (!here) vpar[gi][rr][gr] = make_float2(0.0f, 0.0f);
                    }
#pragma unroll
                    for (int gr = 0; gr < G; gr++) smax = fmaxf(smax, vpar[gi][rr][gr].x);
                }
            float best[NT][2];
            bool move = smax > sthr;
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    best[nt][j] = fmaxf(x[0][nt][j], x[0][nt][j + 2]);
#pragma unroll
                    for (int gi = 1; gi < GS; gi++) best[nt][j] = fmaxf(best[nt][j], fmaxf(x[gi][nt][j], x[gi][nt][j + 2]));
                    move |= best[nt][j] > thr[nt][j];
                }
            if (__any_sync(0xffffffffu, move)) {
                // move the references: each column's best score at 2^(11 - se)
#pragma unroll
                for (int m = 16; m > 0; m >>= 1) smax = fmaxf(smax, __shfl_xor_sync(0xffffffffu, smax, m));
                float grow = 0.0f;
                if (smax > sthr) {
                    const int e = min(max((int)(__float_as_uint(smax) >> 23) - 126, -24), 17);
                    grow = lim - (15.0f - (float)e);
                    lim = 15.0f - (float)e;
                    sthr = __uint_as_float((uint32_t)(e + 127) << 23);
                }
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        float top = best[nt][j];
#pragma unroll
                        for (int m = 4; m < 32; m <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, m));
                        const float moved = fmaxf(mref[nt][j] + grow, top - (lim - 4.0f));
                        const float f = ex2(mref[nt][j] - moved);
                        mref[nt][j] = moved;
                        thr[nt][j] = moved + lim;
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
            }

            // probabilities and values
#pragma unroll
            for (int gi = 0; gi < GS; gi++) {
                const uint8_t* gran = st + gi * L::GB;
                const bool turned = GS == 1 ? odd_step : gi & 1;
                const uint32_t over = turned ? 0xffffffffu : 0u;
                uint32_t pb[G][NT][2];                  // P * s, or -P * s
                [[maybe_unused]] uint32_t pl[G][NT][2];  // FINE: what its rounding left
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    float p[4];
#pragma unroll
                    for (int j = 0; j < 4; j++) p[j] = ex2(x[gi][nt][j] - mref[nt][j & 1]);
                    l[nt][0] += p[0] + p[2];
                    l[nt][1] += p[1] + p[3];
#pragma unroll
                    for (int gr = 0; gr < G; gr++)
#pragma unroll
                        for (int rr = 0; rr < 2; rr++) {
                            const float2 vp = vpar[gi][rr][gr];
                            const float by = turned ? -vp.x : vp.x;
                            float a0 = p[2 * rr] * by, a1 = p[2 * rr + 1] * by;
                            const float mid = FINE ? (turned ? fmaf(15.0f, vp.x, vp.y) : vp.y) : fmaf(7.5f, vp.x, vp.y);
                            float b0 = p[2 * rr], b1 = p[2 * rr + 1], m0 = mid, m1 = mid;
                            if constexpr (!FULL) {  // a key one row sees and another does not may hold NaN
                                if (x[gi][nt][2 * rr] == -CUDART_INF_F) a0 = m0 = 0.0f;
                                if (x[gi][nt][2 * rr + 1] == -CUDART_INF_F) a1 = m1 = 0.0f;
                            }
                            mn[gr][nt][0] = fmaf(b0, m0, mn[gr][nt][0]);
                            mn[gr][nt][1] = fmaf(b1, m1, mn[gr][nt][1]);
                            const __half2 h2 = __floats2half2_rn(a0, a1);
                            const float2 r2 = __half22float2(h2);
                            pb[gr][nt][rr] = movmatrix(*reinterpret_cast<const uint32_t*>(&h2));
                            if constexpr (FINE) {
                                const __half2 l2 = __floats2half2_rn(a0 - r2.x, a1 - r2.y);
                                pl[gr][nt][rr] = movmatrix(*reinterpret_cast<const uint32_t*>(&l2));
                            } else {
                                mn[gr][nt][0] = fmaf(-7.5f, r2.x, mn[gr][nt][0]);
                                mn[gr][nt][1] = fmaf(-7.5f, r2.y, mn[gr][nt][1]);
                            }
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
                        const uint32_t xx = (w01[mt >> 1] >> (8 * (mt & 1))) ^ over, yy = (w23[mt >> 1] >> (8 * (mt & 1))) ^ over;
#pragma unroll
                        for (int nt = 0; nt < NT; nt++) {
                            mma16816(o[gr][mt][nt], xx & 0x000f000fu, xx & 0x00f000f0u, yy & 0x000f000fu, yy & 0x00f000f0u,
                                     pb[gr][nt][0], pb[gr][nt][1]);
                            if constexpr (FINE)
                                mma16816(o[gr][mt][nt], xx & 0x000f000fu, xx & 0x00f000f0u, yy & 0x000f000fu, yy & 0x00f000f0u,
                                         pl[gr][nt][0], pl[gr][nt][1]);
                        }
                    }
                }
            }
        };
        while (mine < seg_end) {
            const int stop = min(seg_end, mine + MOVE * kStWarps);
            for (; mine < stop; mine += kStWarps) {
                if (alive) alive = mbar_wait(&bar[stage], parity, DEV_TIMEOUT_FULL);
                const int p0 = r.lo + (mine - beg) * GS * kKvGranule;
                const uint32_t vm = (valid >> (4 * stage)) & 15u;
                if (p0 >= full_lo && p0 <= full_hi && vm == (1u << GS) - 1) step(ring + stage * L::STEP, p0, vm, std::true_type());
                else step(ring + stage * L::STEP, p0, vm, std::false_type());
                __syncwarp();
                issue(stage);
                if (++stage == kStStages) stage = 0, parity ^= 1u;
            }
            if (mine >= seg_end) break;
            // the minima's part into the sums of codes
#pragma unroll
            for (int gr = 0; gr < G; gr++)
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        float y = mn[gr][nt][j];
                        mn[gr][nt][j] = 0.0f;
#pragma unroll
                        for (int m = 4; m < 32; m <<= 1) y += __shfl_xor_sync(0xffffffffu, y, m);
#pragma unroll
                        for (int mt = 0; mt < 4; mt++) {
                            o[gr][mt][nt][j] = fmaf(y, 5.9604644775390625e-08f, o[gr][mt][nt][j]);          // 2^-24
                            o[gr][mt][nt][j + 2] = fmaf(y, 9.5367431640625e-07f, o[gr][mt][nt][j + 2]);  // 2^-20
                        }
                    }
        }

        if (seg_end < len) {
            stream_seek<D>(a, cur, seg_end);
            if (EARLY) load_columns();
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
        const bool whole = from == beg && seg_end == beg + n;
        float* slot = a.part + (size_t)(2 * cta + (pos == 0 ? 0 : 1)) * (kStRows * (D + 2));
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
                    const int pair = e0 + c;
                    const size_t at = ((size_t)(r.q0 + pair / a.group) * a.heads + head * a.group + pair % a.group) * D + ch;
                    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + at) =
                        make_uint4(pack_act2(v[0] * inv, v[1] * inv, a.dt), pack_act2(v[2] * inv, v[3] * inv, a.dt),
                                   pack_act2(v[4] * inv, v[5] * inv, a.dt), pack_act2(v[6] * inv, v[7] * inv, a.dt));
                } else {
                    float4* dst = reinterpret_cast<float4*>(slot + c * D + ch);
                    __stcg(dst, make_float4(v[0], v[1], v[2], v[3]));
                    __stcg(dst + 1, make_float4(v[4], v[5], v[6], v[7]));
                    if (ch == 0) {
                        __stcg(reinterpret_cast<float2*>(slot + kStRows * D + 2 * c), make_float2(top, ls));
                    }
                }
            }
            __syncthreads();
        }

        pos = seg_end;
    }
}

namespace {

template <int D, int NT>
int stream_ctas() {
    // CTAs an SM holds, by its shared memory and the kernel's launch bounds
    return std::min(stream_resident<D, NT>(), (227 * 1024) / (StreamLayout<D, NT>::TOTAL + 1024)) * sm_count();
}

template <int D, int NT>
cudaError_t stream_launch(const Kv4AttnArgs& a, cudaStream_t stream) {
    using L = StreamLayout<D, NT>;
    auto kern = a.dt == SX_DT_F16 ? kv4_stream_kernel<D, NT, true> : kv4_stream_kernel<D, NT, false>;
    cudaError_t e = func_attrs(reinterpret_cast<const void*>(kern), L::TOTAL, false);
    if (e != cudaSuccess) return e;
    kern<<<stream_ctas<D, NT>(), kStThreads, L::TOTAL, stream>>>(a);
    return cudaGetLastError();
}

}  // namespace

int kv4_stream_grid(int D, int cols) {
    const bool one = cols <= 8;
    if (D == 64) return one ? stream_ctas<64, 1>() : stream_ctas<64, 2>();
    if (D == 128) return one ? stream_ctas<128, 1>() : stream_ctas<128, 2>();
    return one ? stream_ctas<256, 1>() : stream_ctas<256, 2>();
}

cudaError_t kv4_stream_launch(const Kv4AttnArgs& a, int D, cudaStream_t stream) {
    const bool one = a.cols <= 8;
    if (D == 64) return one ? stream_launch<64, 1>(a, stream) : stream_launch<64, 2>(a, stream);
    if (D == 128) return one ? stream_launch<128, 1>(a, stream) : stream_launch<128, 2>(a, stream);
    return one ? stream_launch<256, 1>(a, stream) : stream_launch<256, 2>(a, stream);
}

}  // namespace sx
