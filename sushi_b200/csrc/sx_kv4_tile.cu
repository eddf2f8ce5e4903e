// Attention over the 4-bit cache for requests of many rows (prompt chunks, long drafts, many query
// heads a key head) on the tensor cores.
//
// A unit is one request, key head and block of 128 MT (row, query head) pairs, MT = 2 (1 at D = 256,
// whose output accumulator takes half the tensor memory).  Per tile of NK keys:
//   S = Q K^T  (tcgen05, M = 128, N = NK, both from shared memory, f32 in tensor memory)
//   P = exp2(c S - ref) by one thread a row, F16, over S's columns in tensor memory
//   O += P V   (tcgen05, A = P from tensor memory, B = V from shared memory)
// Other warps widen the codes to F16 tiles (code * s + m, rounded once: one word of eight codes is one
// 16-byte chunk): a task is the keys or the values of one granule; the warps take them in turn, each from
// its own ring of bulk copies.  Eight consecutive channels lie in the order of a word's nibble pairs
// (0 4 1 5 2 6 3 7), in Q and K alike, and in O's columns.  Keys are K-major (rows of 64 channels,
// 128-byte swizzle); values have the same image, read as the N-major operand.  The two row tiles take
// turns: one's softmax runs under the other's products.  The reference moves only when a score passes
// it by 2^8 (P's best at 2^7, at most 2^15).
//
// Precision.  bf16 calls round held keys and values, and P, to F16 once (11 bits): outputs are 4.6e-4 off beyond
// their own rounding of 1.66e-3 (1.72e-3 in all).  F16 outputs would show it (4.0e-4 to 5.7e-4 in all, of 2.1e-4
// of their own), so F16 calls (FINE) keep each in two F16 parts, with a second product for the scores and two more
// for the values: 2.08e-4 in all, for 1.1 to 1.7 times the time (4096 rows over 8192 keys 1100 us, 650 in bf16).
// Sums are f32, cut (not rounded) at each of the MMA's additions, so outputs come short with the tiles summed, in
// bf16 calls by 1.1e-4 over 131072 keys of a CTA.  F16 calls, with three additions for one, sum at most MOST tiles
// in tensor memory and add them up in the CTA's partial slot.
//
// Work: the units' tiles laid end to end and cut into equal runs, one a CTA (one CTA an SM), so
// causal lengths balance and few long rows are split; a unit of several CTAs is joined by
// sx_kv4_join.cu.  Every wait is bounded (sx_common.cuh).
//
// Bound by the chain of a row tile: its softmax (2900 clocks a tile of 128 keys), then both row tiles'
// products (3300), with the widening warps 4650 clocks busy beside them; 4096 rows over 8192 keys, 32 query and
// 8 key heads of 128: 651 us with the join, 633 TFLOP/s.
#include <cuda_runtime.h>
#include <math_constants.h>

#include "sx_gemm_impl.cuh"
#include "sx_kv4_attn.cuh"

namespace sx {

template <int D, bool FINE>
struct TileLayout {
    static constexpr int G = D / kKvGroup;
    static constexpr int MT = kv4_tile_rows(D) / 128;
    static constexpr int NK = kv4_tile_keys(D);
    static constexpr int NG = NK / kKvGranule;  // granules a tile
    static constexpr int PARTS = FINE ? 2 : 1;  // of a key or value tile: leading, then trailing
    static constexpr int KST = FINE && D >= 128 ? 1 : 2, VST = D == 256 || (FINE && D == 128) ? 1 : 2;
    // Widening warps.  7 beside 8 softmax warps and the MMA warp: 16, so 128 registers a thread.  Every
    // warp must have a task among a tile's keys (and among its values) in every tile or in none: a wait by
    // parity tells only neighbouring phases of a stage apart.
    static constexpr int WIDEN = D == 256 ? 8 : 7;
    static_assert(WIDEN <= NG || WIDEN == 2 * NG, "no warp passes over a tile's stage");
    static constexpr int SM_WARPS = 4 * MT;
    static constexpr int MMA_WARP = SM_WARPS + WIDEN;
    static constexpr int THREADS = (MMA_WARP + 1) * 32;
    static constexpr int HB = kv4_granule_bytes(D) / 2;  // a granule's keys, or its values
    static constexpr int RING = D == 128 ? 3 : (D == 64 ? 6 : (FINE ? 1 : 2));
    static constexpr int Q_TILE = 128 * D * 2;
    static constexpr int KV_TILE = NK * D * 2;  // one part
    static constexpr int SUB = NK * 128;  // bytes of 64 channels of a key tile
    static constexpr int Q = 0;
    static constexpr int K = Q + MT * Q_TILE;
    static constexpr int V = K + KST * PARTS * KV_TILE;
    static constexpr int RAW = V + VST * PARTS * KV_TILE;
    static constexpr int BAD = RAW + WIDEN * RING * HB;  // [VST][G][NG] u16: keys whose value group holds NaN
    static constexpr int GONE = BAD + VST * G * NG * 2;     // [4][NG] u8: granules without a page
    static constexpr int BAR = (GONE + 4 * NG + 15) / 16 * 16;
    static constexpr int NBAR = WIDEN * RING + 2 * KST + 2 * VST + 2 + 2 + 2 + 1;
    static constexpr int TOTAL = BAR + NBAR * 8;
    static constexpr int ALLOC = TOTAL + 1024;
    static constexpr int MOST = FINE ? 64 : 1 << 30;  // tiles summed in tensor memory at a time
    static constexpr int S_COL = 0;  // two S tiles of NK columns
    static constexpr int O_COL = 256;
    static_assert(ALLOC <= 227 * 1024, "fits a CTA");
};

// A walk over the units' tiles: the unit's first tile is tile `beg` of this CTA's (negative where an earlier
// CTA has it).
struct TileCursor {
    Kv4Request r;
    TileUnit t;
    int b, h, u, blocks, beg;
};

template <int D>
__device__ __forceinline__ void tile_load(const Kv4AttnArgs& a, TileCursor& c) {
    c.r = kv4_request(a, c.b);
    c.blocks = tile_blocks<D>(a, c.r);
    c.h = c.u = 0;
    c.t.n = 0;
    if (c.blocks) c.t = tile_unit<D>(a, c.r, 0);
}

// Moves the cursor forward to the unit that holds this CTA's tile i.
template <int D>
__device__ __forceinline__ void tile_seek(const Kv4AttnArgs& a, TileCursor& c, int i) {
    while (i >= c.beg + c.t.n) {
        c.beg += c.t.n;
        if (++c.u >= c.blocks) {
            c.u = 0;
            if (++c.h >= a.kv_heads || c.blocks == 0) {
                c.b++;
                tile_load<D>(a, c);
                continue;
            }
        }
        c.t = tile_unit<D>(a, c.r, c.u);
    }
}

// Zeros for the blocks of this CTA that see no key, a warp a block: its lanes look for them in 32 requests at a time.
template <int D, int W>
__device__ __forceinline__ void tile_zeros(const Kv4AttnArgs& a) {
    const int lane = threadIdx.x & 31, grid = gridDim.x;
    for (int b0 = (int)(threadIdx.x >> 5) * 32; b0 < a.requests; b0 += W * 32) {
        const int b = b0 + lane;
        Kv4Request r = {};
        int blocks = 0;
        if (b < a.requests) {
            r = kv4_request(a, b);
            blocks = tile_blocks<D>(a, r);
        }
        // the first block u with (b + u) % grid this CTA
        for (int u = ((int)blockIdx.x - b % grid + grid) % grid; __any_sync(0xffffffffu, u < blocks); u += grid) {
            TileUnit t = {};
            t.n = 1;
            if (u < blocks) t = tile_unit<D>(a, r, u);
            for (unsigned m = __ballot_sync(0xffffffffu, t.n == 0); m; m &= m - 1) {
                const int from = __ffs(m) - 1;
                const int q0 = __shfl_sync(0xffffffffu, r.q0, from), e0 = __shfl_sync(0xffffffffu, t.e0, from),
                          rows = __shfl_sync(0xffffffffu, t.rows, from);
                // whole tokens [t0, t1) are one piece; of the tokens at the ends, pairs [e0, t0 group) and [t1 group, e1)
                const int e1 = e0 + rows, t1 = e1 / a.group, t0 = min((e0 + a.group - 1) / a.group, t1);
                uint4* o = reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + (size_t)q0 * a.heads * D);
                const size_t row = (size_t)a.heads * (D / 8);
                for (size_t i = t0 * row + lane; i < t1 * row; i += 32) o[i] = make_uint4(0, 0, 0, 0);
                auto pairs = [&](int first, int last) {
                    for (int h = 0; h < a.kv_heads; h++)
                        for (int e = first; e < last; e++)
                            if (lane < D / 8) o[e / a.group * row + (h * a.group + e % a.group) * (D / 8) + lane] = make_uint4(0, 0, 0, 0);
                };
                pairs(e0, min(e1, max(t0 * a.group, e0)));
                pairs(max(t1 * a.group, e0), e1);
            }
        }
    }
}

__device__ __forceinline__ void tc_mma_ts_f16(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                              uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}

// N-major operand, 128-byte swizzle: 64-channel blocks `lead` bytes apart, 8-key groups 1024.
__device__ __forceinline__ uint64_t smem_desc_sw128_n(uint32_t saddr, uint32_t lead) {
    return (uint64_t)((saddr >> 4) & 0x3FFFu) | (uint64_t)(lead >> 4) << 16 | (uint64_t)(1024u >> 4) << 32 |
           (uint64_t)1u << 46 | (uint64_t)2u << 61;
}

// 32 columns of this warp's 32 lanes, in two parts: a load is in flight while the one before is worked on.
__device__ __forceinline__ void tmem_ld32_start(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {"
        "%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,"
        "%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_ld32_wait(uint32_t (&r)[32]) {  // names the registers: nothing reads them earlier
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]),
                   "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]),
                   "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]),
                   "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
                 :
                 : "memory");
}

__device__ __forceinline__ void tmem_st32u(uint32_t taddr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {"
        "%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,"
        "%28,%29,%30,%31,%32};" ::"r"(taddr),
          "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
          "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]),
          "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]),
          "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}

__device__ __forceinline__ void tmem_st32(uint32_t taddr, const float (&v)[32]) {
    uint32_t r[32];
#pragma unroll
    for (int i = 0; i < 32; i++) r[i] = __float_as_uint(v[i]);
    tmem_st32u(taddr, r);
}

__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ uint32_t dup_lo(uint32_t p) { return __byte_perm(p, p, 0x1010); }
__device__ __forceinline__ uint32_t dup_hi(uint32_t p) { return __byte_perm(p, p, 0x3232); }
__device__ __forceinline__ __half2 as_half2(uint32_t p) { return *reinterpret_cast<const __half2*>(&p); }

// Eight codes as F16 pairs (0 4, 1 5, 2 6, 3 7), times the step plus the minimum of each of PARTS parameters.
// A code under 1024's exponent is 1024 + code (or 1024 + 16 code), made the code itself exactly before the one rounding.
template <int PARTS>
__device__ __forceinline__ void widen8(uint32_t x, const uint32_t (&par)[PARTS], uint4 (&out)[PARTS]) {
    const __half2 k1024 = __half2half2(__ushort_as_half((unsigned short)0x6400));
    const __half2 k16 = __half2half2(__ushort_as_half((unsigned short)0x2c00));  // 1/16
    const __half2 k64 = __half2half2(__ushort_as_half((unsigned short)0xd400));  // -64
    const uint32_t y = x >> 8;
    const uint32_t w[4] = {(x & 0x000f000fu) | 0x64006400u, (x & 0x00f000f0u) | 0x64006400u,
                           (y & 0x000f000fu) | 0x64006400u, (y & 0x00f000f0u) | 0x64006400u};
    uint32_t o[PARTS][4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const __half2 h = as_half2(w[i]);
        const __half2 c = i & 1 ? __hfma2(h, k16, k64) : __hsub2(h, k1024);
#pragma unroll
        for (int k = 0; k < PARTS; k++) {
            const __half2 v = __hfma2(c, as_half2(dup_lo(par[k])), as_half2(dup_hi(par[k])));
            o[k][i] = *reinterpret_cast<const uint32_t*>(&v);
        }
    }
#pragma unroll
    for (int k = 0; k < PARTS; k++) out[k] = make_uint4(o[k][0], o[k][1], o[k][2], o[k][3]);
}

// A step and minimum p as the sum of two: `lead` multiples of 2^-8 of the group's largest power of two, so that
// code * s + m is exact in F16, `trail` what is left (code * s + m of it below 2^-4 of that power, rounded once).
__device__ __forceinline__ void split_params(uint32_t p, uint32_t& lead, uint32_t& trail) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&p));
    const float most = fmaxf(fabsf(f.y), fabsf(fmaf(15.0f, f.x, f.y)));
    // 1.5 * 2^15 times that power: its last bit is 2^-8 of the power
    const float grid = __uint_as_float(((__float_as_uint(most) & 0x7f800000u) + (15u << 23)) | 0x00400000u);
    const float s = (f.x + grid) - grid, m = (f.y + grid) - grid;
    const __half2 a = __floats2half2_rn(s, m), b = __floats2half2_rn(f.x - s, f.y - m);
    lead = *reinterpret_cast<const uint32_t*>(&a);
    trail = *reinterpret_cast<const uint32_t*>(&b);
}

// A word's eight values to one 16-byte chunk, or their two parts to chunks TRAIL bytes apart.
template <int PARTS, int TRAIL>
__device__ __forceinline__ void widen_store(uint32_t x, const uint32_t (&par)[PARTS], uint8_t* out) {
    uint4 v[PARTS];
    widen8(x, par, v);
#pragma unroll
    for (int k = 0; k < PARTS; k++) *reinterpret_cast<uint4*>(out + k * TRAIL) = v[k];
}

// The channel of eight that sits at place p of a chunk.
__host__ __device__ constexpr int chunk_channel(int p) { return (p >> 1) + 4 * (p & 1); }

// The keys of a granule as rows row0 .. row0 + 15 of a tile; tokens from `live` on become 0.  Lanes: words
// 2t and 2t + 1 of every group of one token, eight tokens at a time.
template <int D, bool FINE>
__device__ __forceinline__ void widen_keys(const uint8_t* gran, int live, int row0, uint8_t* out) {
    using L = TileLayout<D, FINE>;
    constexpr int G = L::G;
    const int lane = threadIdx.x & 31, t = lane & 3;
    uint32_t x[2][G][2], p[2][G];
#pragma unroll
    for (int hf = 0; hf < 2; hf++) {
        const int tok = hf * 8 + (lane >> 2);
        if constexpr (D == 64) {
            const uint2 u = *reinterpret_cast<const uint2*>(gran + kv4_key_word<D>(tok, 0, 2 * t));
            x[hf][0][0] = u.x, x[hf][0][1] = u.y;
        } else {
#pragma unroll
            for (int gr = 0; gr < G; gr += 2) {
                const uint4 u = *reinterpret_cast<const uint4*>(gran + kv4_key_word<D>(tok, gr, 2 * t));
                x[hf][gr][0] = u.x, x[hf][gr][1] = u.y, x[hf][gr + 1][0] = u.z, x[hf][gr + 1][1] = u.w;
            }
        }
#pragma unroll
        for (int gr = 0; gr < G; gr++) {
            p[hf][gr] = *reinterpret_cast<const uint32_t*>(gran + kv4_kpar_off(D) + (tok * G + gr) * 4);
            if (tok >= live) p[hf][gr] = 0u;
        }
    }
#pragma unroll
    for (int hf = 0; hf < 2; hf++)
#pragma unroll
        for (int gr = 0; gr < G; gr++) {
            uint32_t par[L::PARTS] = {p[hf][gr]};
            if constexpr (FINE) split_params(p[hf][gr], par[0], par[1]);
#pragma unroll
            for (int i = 0; i < 2; i++)
                widen_store<L::PARTS, L::KV_TILE>(x[hf][gr][i], par, out + gr * L::SUB + sw128_offset(row0 + hf * 8 + (lane >> 2), (2 * t + i) * 8));
        }
}

// The values of a granule (`gran`: the granule's start, of which only the values' half is there).  NaN
// groups become 0 (a key some row does not see must not reach it) and are named in bad[group] for the rows
// that do see them; the writer gives both parameters NaN or neither.  Lanes: word lane % 8 of every group of
// one token, four tokens at a time.
template <int D, bool FINE>
__device__ __forceinline__ void widen_values(const uint8_t* gran, int live, int row0, uint8_t* out, uint16_t* bad) {
    using L = TileLayout<D, FINE>;
    constexpr int G = L::G;
    const int lane = threadIdx.x & 31, pc = lane & 7;
    uint32_t x[4][G], p[4][G], nan[G];
#pragma unroll
    for (int gr = 0; gr < G; gr++)
        nan[gr] = *reinterpret_cast<const uint32_t*>(gran + kv4_vpar_off(D) + ((lane & 15) * G + gr) * 4);
#pragma unroll
    for (int q4 = 0; q4 < 4; q4++) {
        const int tok = q4 * 4 + (lane >> 3);
        const uint8_t* src = gran + kv4_value_word<D>(tok, 0, pc);
        if constexpr (D == 64) {
            x[q4][0] = *reinterpret_cast<const uint32_t*>(src);
        } else if constexpr (D == 128) {
            const uint2 u = *reinterpret_cast<const uint2*>(src);
            x[q4][0] = u.x, x[q4][1] = u.y;
        } else {
            const uint4 u = *reinterpret_cast<const uint4*>(src);
            x[q4][0] = u.x, x[q4][1] = u.y, x[q4][2] = u.z, x[q4][3] = u.w;
        }
#pragma unroll
        for (int gr = 0; gr < G; gr++) {
            p[q4][gr] = *reinterpret_cast<const uint32_t*>(gran + kv4_vpar_off(D) + (tok * G + gr) * 4);
            if (tok >= live) p[q4][gr] = 0u;
        }
    }
    uint32_t any = 0;
#pragma unroll
    for (int gr = 0; gr < G; gr++) {
        nan[gr] = __ballot_sync(0xffffffffu, (lane & 15) < live && (nan[gr] & 0x7c00u) == 0x7c00u) & 0xffffu;
        if (lane == 0) bad[gr * L::NG] = (uint16_t)nan[gr];
        any |= nan[gr];
    }
    if (any) {
#pragma unroll
        for (int q4 = 0; q4 < 4; q4++)
#pragma unroll
            for (int gr = 0; gr < G; gr++)
                if ((p[q4][gr] & 0x7c00u) == 0x7c00u) p[q4][gr] = 0u;
    }
#pragma unroll
    for (int q4 = 0; q4 < 4; q4++)
#pragma unroll
        for (int gr = 0; gr < G; gr++) {
            uint32_t par[L::PARTS] = {p[q4][gr]};
            if constexpr (FINE) split_params(p[q4][gr], par[0], par[1]);
            widen_store<L::PARTS, L::KV_TILE>(x[q4][gr], par, out + gr * L::SUB + sw128_offset(row0 + q4 * 4 + (lane >> 3), pc * 8));
        }
}

template <int D, bool FINE>
__global__ void __launch_bounds__(TileLayout<D, FINE>::THREADS, 1) kv4_tile_kernel(const __grid_constant__ Kv4AttnArgs a) {
    using L = TileLayout<D, FINE>;
    constexpr int G = L::G, MT = L::MT, NK = L::NK, NG = L::NG;
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint32_t tmem_slot;
    __shared__ int red[L::THREADS / 32], pick[5], few[kTlFew], run_tiles;
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    uint64_t* raw_full = reinterpret_cast<uint64_t*>(smem + L::BAR);  // [widening warps][RING]
    uint64_t* kfull = raw_full + L::WIDEN * L::RING;
    uint64_t* kempty = kfull + L::KST;
    uint64_t* vfull = kempty + L::KST;
    uint64_t* vempty = vfull + L::VST;
    uint64_t* sfull = vempty + L::VST;  // [2]: MT = 2 by row tile, MT = 1 by turn
    uint64_t* pfull = sfull + 2;        // [2]
    uint64_t* odone = pfull + 2;        // [2] (MT = 1: the first)
    uint64_t* qfull = odone + 2;
    if (tid == 0) {
        for (int i = 0; i < L::WIDEN * L::RING; i++) mbar_init(&raw_full[i], 1);
        for (int i = 0; i < L::KST; i++) mbar_init(&kfull[i], NG), mbar_init(&kempty[i], 1);
        for (int i = 0; i < L::VST; i++) mbar_init(&vfull[i], NG), mbar_init(&vempty[i], 1);
        for (int i = 0; i < 2; i++) mbar_init(&sfull[i], 1), mbar_init(&pfull[i], 4), mbar_init(&odone[i], 1);
        mbar_init(qfull, L::SM_WARPS);
        fence_mbar_init();
    }

    // ---------------- the list's length; blocks that see no key are zeroed here, by CTA (request + block) % grid
    const size_t head_row = (size_t)a.heads * D;
    pdl_release();
    constexpr int W = L::THREADS / 32;
    const int cta = blockIdx.x;
    int n0;
    bool zeros = false;
    const int total = tile_list_total<D, W>(a, red, few, n0, zeros, [&](int b, const Kv4Request&, const TileUnit& t, int u) {
        if (t.n == 0 && (b + u) % (int)gridDim.x == cta) zeros = true;
    });
    if (zeros) tile_zeros<D, W>(a);
    const RunCut run(total, gridDim.x);
    if (total == 0 || cta >= run.ctas) {
        pdl_wait();  // the join that follows waits for this grid: the streaming kernel's end is part of it
        return;
    }
    const int start = run.start(cta);
    tile_list_find<D, W>(a, red, pick, n0, start);
    TileCursor cur;
    cur.b = pick[0];
    tile_load<D>(a, cur);
    cur.u = pick[2], cur.h = pick[4];
    cur.beg = min(0, pick[3] + kv4_tile_pad(D) - start);
    cur.t = tile_unit<D>(a, cur.r, cur.u);
    if (tid == 0) {
        // the run's tiles, less the units' empty ones
        const int end = run.start(cta + 1);
        TileCursor c = cur;
        int n = 0;
        for (int p = pick[3]; p < end; p += tile_list<D>(c.t.n)) {
            if (p > pick[3]) tile_seek<D>(a, c, c.beg + c.t.n);
            n += max(0, min(end, p + tile_list<D>(c.t.n)) - max(start, p + kv4_tile_pad(D)));
        }
        run_tiles = n;
    }
    if (warp == L::MMA_WARP) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "n"(512)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    const int len = run_tiles;  // this CTA's tiles

    if (warp < L::SM_WARPS) {
        // ---------------- softmax: one thread a (row, head) pair of row tile `mt`
        const int mt = warp >> 2, row = tid & 127;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t o_tm = tmem + lanes + L::O_COL + mt * D;
        uint32_t turns = 0;  // tiles this row tile has taken
        uint32_t tiles = 0;  // tiles the CTA has taken (the key and value rings' turn)
        bool ok = true;
        for (int pos = 0; pos < len;) {
            // both row tiles start a unit together: one that sits a unit out must not count for the next
            asm volatile("bar.sync 2, %0;" ::"n"(L::SM_WARPS * 32) : "memory");
            tile_seek<D>(a, cur, pos);
            const Kv4Request r = cur.r;
            const TileUnit un = cur.t;
            const int unit_end = min(len, cur.beg + un.n), seg_end = min(unit_end, pos + min(L::MOST, len));
            const int j0 = pos - cur.beg, n = seg_end - pos;
            const int e = mt * 128 + row;
            const bool live = e < un.rows;              // this thread has a pair
            const bool tile_live = mt * 128 < un.rows;  // the row tile takes part
            const int pair = un.e0 + (live ? e : 0);
            const int qi = pair / a.group, head = cur.h * a.group + pair % a.group;
            const int qpos = r.pos0 + qi;

            // the query row: scaled by a power of two (largest entry to [2^13, 2^14)), F16, chunk order
            // (a thread without a pair reads the block's first and takes 0 of it; 16 loads in flight)
            const long long at = (r.q0 + qi) * a.qts + head * a.qhs;
            const uint16_t* qrow = static_cast<const uint16_t*>(a.q) + at;
            auto load_q = [&](int c0, uint4 (&w)[8]) {
                if (a.qvec) {
#pragma unroll
                    for (int i = 0; i < 8; i++) w[i] = *reinterpret_cast<const uint4*>(qrow + c0 + i * 8);
                } else {
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const uint16_t* p = qrow + c0 + i * 8;
                        w[i] = make_uint4(p[0] | (uint32_t)p[1] << 16, p[2] | (uint32_t)p[3] << 16,
                                          p[4] | (uint32_t)p[5] << 16, p[6] | (uint32_t)p[7] << 16);
                    }
                }
            };
            auto widen = [&](const uint4& w, float (&x)[8]) {
                const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const uint16_t h = (uint16_t)(ww[i >> 1] >> (16 * (i & 1)));
                    x[i] = a.dt == 1 ? __half2float(__ushort_as_half(h)) : __bfloat162float(__ushort_as_bfloat16(h));
                }
            };
            constexpr bool HOLD = D <= 128;  // the whole row in registers between the two passes
            uint4 qw[HOLD ? D / 64 : 1][8];
            float top = 0.0f;
#pragma unroll
            for (int b = 0; HOLD && b < D / 64; b++) load_q(b * 64, qw[HOLD ? b : 0]);
#pragma unroll
            for (int b = 0; b < D / 64; b++) {
                if (!HOLD) load_q(b * 64, qw[0]);
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    float x[8];
                    widen(qw[HOLD ? b : 0][i], x);
#pragma unroll
                    for (int k = 0; k < 8; k++) top = fmaxf(top, fabsf(x[k]));
                }
            }
            const int k2 = query_scale(top);
            // a negative scale goes into the query's sign, so that c >= 0 below
            const float up = copysignf(__uint_as_float((uint32_t)(k2 + 127) << 23), a.scale_log2);
            // (a scale of 0 keeps c above 0: -inf c is then -inf, and what is left of the scores adds nothing; keys below
            // 2^16, the query below 2^14, 2^8 channels)
            float c = fmaxf(kv4_most_scale(fabsf(a.scale_log2) * __uint_as_float((uint32_t)(127 - k2) << 23), 38), 1.0e-30f);
            volatile float c_first = c;  // not worth a register: read once, after the tiles
#pragma unroll
            for (int b = 0; b < D / 64; b++) {
                if (!HOLD) load_q(b * 64, qw[0]);
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    float x[8];
                    widen(qw[HOLD ? b : 0][i], x);
                    uint32_t w[4];
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const __half2 h = __floats2half2_rn(x[k] * up, x[k + 4] * up);
                        w[k] = live ? *reinterpret_cast<const uint32_t*>(&h) : 0u;
                    }
                    *reinterpret_cast<uint4*>(smem + L::Q + mt * L::Q_TILE + b * 16384 + sw128_offset(row, i * 8)) =
                        make_uint4(w[0], w[1], w[2], w[3]);
                }
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(qfull);

            const int lowest = a.window > 0 ? qpos - a.window + 1 : 0, highest = min(r.hi - 1, qpos);
            // tiles of keys that start at or after full_lo and end by full_hi are seen whole by every pair
            const int full_hi = min(r.hi, r.pos0 + un.e0 / a.group + 1) - NK;
            const int full_lo = a.window > 0 ? r.pos0 + (un.e0 + un.rows - 1) / a.group - a.window + 1 : 0;
            float mref = kNoScore, l = 0.0f;
            uint32_t bad = 0;  // groups in which the row sees a NaN value
            for (int j = 0; tile_live && j < n; j++, turns++) {
                const int bi = MT == 2 ? mt : (int)(turns & 1);
                const uint32_t par = MT == 2 ? turns & 1 : (turns >> 1) & 1;
                const uint32_t s_tm = tmem + lanes + L::S_COL + bi * NK;
                const int k0 = un.lo + (j0 + j) * NK;
                if (ok) ok = mbar_wait(&sfull[bi], par, DEV_TIMEOUT_FULL);
                tc_fence_after();
                bool full = k0 >= full_lo && k0 <= full_hi;
                uint32_t gone = 0;  // granules without a page
                {
                    const uint32_t* gm = reinterpret_cast<const uint32_t*>(smem + L::GONE + ((tiles + j) & 3) * NG);
                    uint32_t any = 0;
#pragma unroll
                    for (int i = 0; i < NG / 4; i++) any |= gm[i];
                    if (any) {
                        for (int i = 0; i < NG; i++) gone |= ((gm[i >> 2] >> (8 * (i & 3))) & 1u) << i;
                        full = false;
                    }
                }
                if (!full) {
                    // keys this row does not see score -inf from here on
#pragma unroll 1
                    for (int q = 0; q < NK; q += 32) {
                        const int from = max(lowest - k0 - q, 0), to = min(highest - k0 - q, 31);  // the row's keys among the 32
                        uint32_t seen = from > 31 || to < from ? 0u : (0xffffffffu << from) & (0xffffffffu >> (31 - to));
                        if ((gone >> (q >> 4)) & 1u) seen &= 0xffff0000u;
                        if ((gone >> (q >> 4)) & 2u) seen &= 0x0000ffffu;
                        uint32_t v[32];
                        __syncwarp();
                        tmem_ld32_start(s_tm + q, v);
                        tmem_ld32_wait(v);
#pragma unroll
                        for (int i = 0; i < 32; i++) v[i] = (seen >> i) & 1u ? v[i] : 0xff800000u;
                        tmem_st32u(s_tm + q, v);
                    }
                    tmem_st_wait();
                }
                float m4[4] = {-CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F};
                uint32_t va[32], vb[32];
                auto top_of = [&](uint32_t (&v)[32]) {
#pragma unroll
                    for (int i = 0; i < 32; i++) m4[i & 3] = fmaxf(m4[i & 3], __uint_as_float(v[i]));
                };
                __syncwarp();
                tmem_ld32_start(s_tm, va);
#pragma unroll 1
                for (int q = 0; q < NK; q += 64) {
                    tmem_ld32_wait(va);
                    tmem_ld32_start(s_tm + q + 32, vb);
                    top_of(va);
                    __syncwarp();
                    tmem_ld32_wait(vb);
                    tmem_ld32_start(s_tm + (q + 64 < NK ? q + 64 : 0), va);  // the last: the first for the second pass
                    top_of(vb);
                    __syncwarp();
                }
                const float mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * c;
                if (__any_sync(0xffffffffu, mx > mref + 15.0f)) {
                    // c S - mref, in one rounding, is off by mref's own: past 2^22 the row's c shrinks by a power of two.
                    // Two scores of 11-bit operands that differ at all then still differ by 2^10.
                    float size = 1.0f;
                    if (fabsf(mx) > 4194304.0f && mx > kNoScore) size = __uint_as_float((275u << 23) - (__float_as_uint(mx) & 0x7f800000u));
                    c *= size;
                    mref *= size;
                    const float moved = fmaxf(mref, mx * size - 7.0f);
                    const float f = ex2(mref - moved);
                    mref = moved;
                    l *= f;
                    if (j > 0) {
                        // the product of the tile before is in
                        if (ok) ok = mbar_wait(&odone[MT == 2 ? mt : 0], (turns - 1) & 1, DEV_TIMEOUT_FULL);
                        tc_fence_after();
                        tmem_ld32_wait(va);
#pragma unroll 1
                        for (int q = 0; q < D; q += 32) {
                            float v[32];
                            tmem_ld32(o_tm + q, v);
#pragma unroll
                            for (int i = 0; i < 32; i++) v[i] *= f;
                            tmem_st32(o_tm + q, v);
                        }
                    }
                }
                float l4[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                auto weights = [&](uint32_t (&v)[32], uint32_t* w) {
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        const float p0 = ex2(fmaf(__uint_as_float(v[2 * i]), c, -mref));
                        const float p1 = ex2(fmaf(__uint_as_float(v[2 * i + 1]), c, -mref));
                        if constexpr (FINE) v[2 * i] = __float_as_uint(p0), v[2 * i + 1] = __float_as_uint(p1);
                        l4[i & 3] += p0 + p1;
                        const __half2 h = __floats2half2_rn(p0, p1);
                        w[i] = *reinterpret_cast<const uint32_t*>(&h);
                    }
                };
                // FINE: the weights of 32 columns go over them, in two parts of 16 columns
                auto both = [&](uint32_t (&v)[32], uint32_t (&w)[32]) {
                    weights(v, w);
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        const float2 r = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
                        const __half2 h = __floats2half2_rn(__uint_as_float(v[2 * i]) - r.x, __uint_as_float(v[2 * i + 1]) - r.y);
                        w[16 + i] = *reinterpret_cast<const uint32_t*>(&h);
                    }
                };
#pragma unroll 1
                for (int q = 0; FINE && q < NK; q += 64) {
                    uint32_t w[32];
                    tmem_ld32_wait(va);
                    tmem_ld32_start(s_tm + q + 32, vb);
                    both(va, w);
                    __syncwarp();
                    tmem_ld32_wait(vb);
                    tmem_st32u(s_tm + q, w);
                    if (q + 64 < NK) tmem_ld32_start(s_tm + q + 64, va);
                    both(vb, w);
                    __syncwarp();
                    tmem_st32u(s_tm + q + 32, w);
                }
                // the weights of columns q go over columns q / 2, which are in registers by then; 64 at a
                // time, since a store holds up the warp's later loads while the products run
#pragma unroll 1
                for (int q = 0; !FINE && q < NK; q += 64) {
                    uint32_t w[32];
                    tmem_ld32_wait(va);
                    tmem_ld32_start(s_tm + q + 32, vb);
                    weights(va, w);
                    __syncwarp();
                    tmem_ld32_wait(vb);
                    if (q + 64 < NK) tmem_ld32_start(s_tm + q + 64, va);
                    weights(vb, w + 16);
                    __syncwarp();
                    tmem_st32u(s_tm + q / 2, w);
                }
                l += (l4[0] + l4[1]) + (l4[2] + l4[3]);
                {
                    // value groups with NaN (widened to 0): named for the rows that see them
                    const uint32_t vt = tiles + j;
                    if (ok) ok = mbar_wait(&vfull[vt % L::VST], (vt / L::VST) & 1, DEV_TIMEOUT_FULL);
                    const uint32_t* bm = reinterpret_cast<const uint32_t*>(smem + L::BAD + (vt % L::VST) * (G * NG * 2));
                    uint32_t any = 0;
#pragma unroll
                    for (int i = 0; i < G * NG / 2; i++) any |= bm[i];
                    if (any)
                        for (int i = 0; i < G * NK; i++) {
                            const int key = k0 + i % NK;
                            if (((bm[i >> 5] >> (i & 31)) & 1u) && key >= lowest && key <= highest) bad |= 1u << (i / NK);
                        }
                    __syncwarp();
                }
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&pfull[bi]);
            }
            tiles += n;

            // ---------------- the rows out, or this CTA's share of them into its slot
            const int begun = max(cur.beg, 0);  // the unit's first tile here
            const bool whole = begun == cur.beg && seg_end == cur.beg + un.n;
            float* slot = a.part + (size_t)(2 * cta + (begun == 0 ? 0 : 1)) * (kv4_tile_rows(D) * (D + 2));
            if (tile_live) {
                if (ok) ok = mbar_wait(&odone[MT == 2 ? mt : 0], (turns - 1) & 1, DEV_TIMEOUT_FULL);
                tc_fence_after();
                float* ml = slot + kv4_tile_rows(D) * D + 2 * e;
                float m = mref * (c_first / c), now = 1.0f;
                [[maybe_unused]] float before = 0.0f;  // the weight of what this unit's tiles left in the slot before
                const bool more = FINE && pos > begun;
                if (more && live) {
                    const float2 held = __ldcg(reinterpret_cast<const float2*>(ml));
                    const float up = fmaxf(held.x, m);
                    before = ex2(held.x - up), now = ex2(m - up);
                    l = fmaf(l, now, held.y * before);
                    m = up;
                }
                const float inv = whole ? (l == 0.0f ? 0.0f : now / l) : now;
                if (whole) before = l == 0.0f ? 0.0f : before / l;
#pragma unroll 1
                for (int q = 0; q < D; q += 32) {
                    float v[32];
                    __syncwarp();
                    tmem_ld32(o_tm + q, v);
                    if (live) {
                        const float by = (bad >> (q >> 6)) & 1u ? CUDART_NAN_F : inv;
#pragma unroll
                        for (int i = 0; i < 32; i++) v[i] *= by;
#pragma unroll
                        for (int w = 0; w < 32; w += 8) {
                            float x[8];
#pragma unroll
                            for (int i = 0; i < 8; i++) x[chunk_channel(i)] = v[w + i];
                            float4* at = reinterpret_cast<float4*>(slot + e * D + q + w);
                            if (more) {
                                const float4 y = __ldcg(at), z = __ldcg(at + 1);
                                x[0] = fmaf(before, y.x, x[0]), x[1] = fmaf(before, y.y, x[1]);
                                x[2] = fmaf(before, y.z, x[2]), x[3] = fmaf(before, y.w, x[3]);
                                x[4] = fmaf(before, z.x, x[4]), x[5] = fmaf(before, z.y, x[5]);
                                x[6] = fmaf(before, z.z, x[6]), x[7] = fmaf(before, z.w, x[7]);
                            }
                            if (whole) {
                                *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + (r.q0 + qi) * head_row +
                                                          (size_t)head * D + q + w) =
                                    make_uint4(pack_act2(x[0], x[1], a.dt), pack_act2(x[2], x[3], a.dt),
                                               pack_act2(x[4], x[5], a.dt), pack_act2(x[6], x[7], a.dt));
                            } else {
                                __stcg(at, make_float4(x[0], x[1], x[2], x[3]));
                                __stcg(at + 1, make_float4(x[4], x[5], x[6], x[7]));
                            }
                        }
                    }
                }
                __syncwarp();
                tc_fence_before();  // the next unit's first product overwrites O after the next arrival
                if (!whole && live) __stcg(reinterpret_cast<float2*>(ml), make_float2(m, l));
            }
            pos = seg_end;
        }
    } else if (warp < L::MMA_WARP) {
        // ---------------- widening: task q of the CTA's is granule q % NG of tile q / (2 NG), its keys, then its values
        const int w = warp - L::SM_WARPS;
        uint8_t* ring = smem + L::RAW + w * L::RING * L::HB;
        uint64_t* bar = raw_full + w * L::RING;
        uint32_t there = 0;  // a bit a ring place: the granule was copied
        bool ok = true;
        TileCursor ahead = cur;
        const int tasks = len * 2 * NG;
        int in_q = w, in_place = 0;
        // the next copy's place in the cache, looked up a copy ahead (its page id is a load of its own)
        const uint8_t* next = nullptr;
        int next_page = -1;
        auto look = [&]() {
            next_page = -1;
            if (in_q >= tasks) return;
            const int tile = in_q / (2 * NG), part = in_q % (2 * NG);
            tile_seek<D>(a, ahead, tile);
            const int key = ahead.t.lo + (tile - ahead.beg) * NK + (part % NG) * kKvGranule;
            if (key < ahead.r.hi) next_page = a.table[ahead.b * a.tstride + (key >> a.shift)];
            next = a.pool + (part >= NG ? kv4_value_off(D) : 0) +
                   kv4_granule<D>(0, a.kv_heads, ahead.h, a.page_size, key & (a.page_size - 1));
        };
        const size_t page_bytes = kv4_granule<D>(1, a.kv_heads, 0, a.page_size, 0);
        auto issue = [&]() {  // the warp's next copy into its next ring place
            if (in_q < tasks) {
                const bool got = next_page >= 0 && next_page < a.pages;
                if (lane == 0) {
                    mbar_arrive_expect_tx(&bar[in_place], got ? L::HB : 0);
                    if (got) bulk_g2s(ring + in_place * L::HB, next + next_page * page_bytes, L::HB, &bar[in_place]);
                }
                there = (there & ~(1u << in_place)) | ((got ? 1u : 0u) << in_place);
            }
            in_q += L::WIDEN;
            if (++in_place == L::RING) in_place = 0;
            look();
        };
        look();
        for (int i = 0; i < L::RING; i++) issue();
        int place = 0;
        uint32_t parity = 0;
        for (int task = w; task < tasks; task += L::WIDEN) {
            const uint32_t tile = task / (2 * NG);
            const int part = task % (2 * NG), gi = part % NG;
            tile_seek<D>(a, cur, (int)tile);
            const int first = cur.t.lo + ((int)tile - cur.beg) * NK + gi * kKvGranule;  // the granule's first key
            const bool got = (there >> place) & 1u;
            const int live = got ? min(cur.r.hi - first, kKvGranule) : 0;  // tokens that are there
            const uint8_t* raw = ring + place * L::HB;
            uint64_t* full;
            if (part < NG) {
                const int stage = (int)(tile % L::KST);
                full = &kfull[stage];
                if (ok && tile >= L::KST) ok = mbar_wait(&kempty[stage], (tile / L::KST - 1) & 1, DEV_TIMEOUT_EMPTY);
                if (ok) ok = mbar_wait(&bar[place], parity, DEV_TIMEOUT_FULL);
                if (lane == 0) smem[L::GONE + (tile & 3) * NG + gi] = !got && first < cur.r.hi;
                widen_keys<D, FINE>(raw, live, gi * kKvGranule, smem + L::K + stage * L::PARTS * L::KV_TILE);
            } else {
                const int stage = (int)(tile % L::VST);
                full = &vfull[stage];
                if (ok && tile >= L::VST) ok = mbar_wait(&vempty[stage], (tile / L::VST - 1) & 1, DEV_TIMEOUT_EMPTY);
                if (ok) ok = mbar_wait(&bar[place], parity, DEV_TIMEOUT_FULL);
                widen_values<D, FINE>(raw - kv4_value_off(D), live, gi * kKvGranule, smem + L::V + stage * L::PARTS * L::KV_TILE,
                                reinterpret_cast<uint16_t*>(smem + L::BAD) + stage * (G * NG) + gi);
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(full);
            issue();
            if (++place == L::RING) place = 0, parity ^= 1u;
        }
    } else if (lane == 0) {
        // ---------------- the products
        constexpr uint32_t id_s = idesc_f16_m128(NK);
        constexpr uint32_t id_o = idesc_f16_m128(D) | (1u << 16);  // B is N-major
        uint32_t tiles = 0, segs = 0;
        uint32_t turn[2] = {0, 0};
        bool ok = true;
        auto scores = [&](int mt, int bi, uint32_t tile) {
            const uint32_t q = smem_u32(smem + L::Q + mt * L::Q_TILE), k = smem_u32(smem + L::K + (tile % L::KST) * L::PARTS * L::KV_TILE);
            if (ok) {
#pragma unroll
                for (int kk = 0; kk < L::PARTS * (D / 16); kk++) {
                    const int part = kk / (D / 16), k16 = kk % (D / 16);
                    tc_mma_f16(tmem + L::S_COL + bi * NK, smem_desc_sw128(q + (k16 >> 2) * 16384 + (k16 & 3) * 32),
                               smem_desc_sw128(k + part * L::KV_TILE + (k16 >> 2) * L::SUB + (k16 & 3) * 32), id_s, kk > 0 ? 1u : 0u);
                }
            }
            tc_commit(&sfull[bi]);
        };
        auto values = [&](int mt, int bi, uint32_t tile, bool first) {
            const uint32_t v = smem_u32(smem + L::V + (tile % L::VST) * L::PARTS * L::KV_TILE);
            const uint32_t o = tmem + L::O_COL + mt * D, p = tmem + L::S_COL + bi * NK;
            if (ok) {
#pragma unroll
                for (int kk = 0; kk < NK / 16; kk++) {
                    const uint64_t lead = smem_desc_sw128_n(v + kk * 2048, L::SUB);
                    if constexpr (FINE) {  // all but the two trailing parts' product
                        const uint32_t at = p + (kk >> 1) * 32 + (kk & 1) * 8;
                        tc_mma_ts_f16(o, at, lead, id_o, (!first || kk > 0) ? 1u : 0u);
                        tc_mma_ts_f16(o, at, smem_desc_sw128_n(v + L::KV_TILE + kk * 2048, L::SUB), id_o, 1u);
                        tc_mma_ts_f16(o, at + 16, lead, id_o, 1u);
                    } else {
                        tc_mma_ts_f16(o, p + kk * 8, lead, id_o, (!first || kk > 0) ? 1u : 0u);
                    }
                }
            }
            tc_commit(&odone[MT == 2 ? mt : 0]);
        };
        for (int pos = 0; pos < len;) {
            tile_seek<D>(a, cur, pos);
            const int seg_end = min(min(len, cur.beg + cur.t.n), pos + min(L::MOST, len));
            const int n = seg_end - pos;
            const int live = MT == 2 && cur.t.rows > 128 ? 2 : 1;
            if (ok) ok = mbar_wait(qfull, segs & 1, DEV_TIMEOUT_FULL);
            if (ok) ok = mbar_wait(&kfull[tiles % L::KST], (tiles / L::KST) & 1, DEV_TIMEOUT_FULL);
            tc_fence_after();
            for (int s = 0; s < live; s++) scores(s, MT == 2 ? s : (int)(turn[0] & 1), tiles);
            tc_commit(&kempty[tiles % L::KST]);
            for (int j = 0; j < n; j++, tiles++) {
                const uint32_t nx = tiles + 1;
                if (MT == 1 && j + 1 < n) {
                    if (ok) ok = mbar_wait(&kfull[nx % L::KST], (nx / L::KST) & 1, DEV_TIMEOUT_FULL);
                    tc_fence_after();
                    scores(0, (int)((turn[0] + 1) & 1), nx);
                    tc_commit(&kempty[nx % L::KST]);
                }
                if (ok) ok = mbar_wait(&vfull[tiles % L::VST], (tiles / L::VST) & 1, DEV_TIMEOUT_FULL);
                for (int s = 0; s < live; s++) {
                    const int bi = MT == 2 ? s : (int)(turn[0] & 1);
                    if (ok) ok = mbar_wait(&pfull[bi], MT == 2 ? turn[s] & 1 : (turn[0] >> 1) & 1, DEV_TIMEOUT_FULL);
                    tc_fence_after();
                    values(s, bi, tiles, j == 0);
                    if (MT == 2 && j + 1 < n) {
                        if (s == 0) {
                            if (ok) ok = mbar_wait(&kfull[nx % L::KST], (nx / L::KST) & 1, DEV_TIMEOUT_FULL);
                            tc_fence_after();
                        }
                        scores(s, s, nx);
                    }
                    turn[s]++;
                }
                tc_commit(&vempty[tiles % L::VST]);
                if (MT == 2 && j + 1 < n) tc_commit(&kempty[nx % L::KST]);
            }
            segs++;
            pos = seg_end;
        }
        // the last commit of all: nothing of this CTA's is in flight when it frees its tensor memory
        if (ok && tiles > 0) mbar_wait(&vempty[(tiles - 1) % L::VST], ((tiles - 1) / L::VST) & 1, DEV_TIMEOUT_EMPTY);
    }
    pdl_wait();  // the join that follows waits for this grid: the streaming kernel's end is part of it
    tc_fence_before();
    __syncthreads();
    if (warp == L::MMA_WARP) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(512) : "memory");
    }
}

namespace {

template <int D, bool FINE>
cudaError_t tile_launch(const Kv4AttnArgs& a, cudaStream_t stream) {
    using L = TileLayout<D, FINE>;
    auto kern = kv4_tile_kernel<D, FINE>;
    cudaError_t e = func_attrs(reinterpret_cast<const void*>(kern), L::ALLOC, false);
    if (e != cudaSuccess) return e;
    // starts as the streaming kernel drains: neither reads what the other writes
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(sm_count(), 1, 1);
    cfg.blockDim = dim3(L::THREADS, 1, 1);
    cfg.dynamicSmemBytes = L::ALLOC;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kern, a);
}

}  // namespace

cudaError_t kv4_tile_launch(const Kv4AttnArgs& a, int D, cudaStream_t stream) {
    const bool fine = a.dt == SX_DT_F16;
    if (D == 64) return fine ? tile_launch<64, true>(a, stream) : tile_launch<64, false>(a, stream);
    if (D == 128) return fine ? tile_launch<128, true>(a, stream) : tile_launch<128, false>(a, stream);
    return fine ? tile_launch<256, true>(a, stream) : tile_launch<256, false>(a, stream);
}

}  // namespace sx
