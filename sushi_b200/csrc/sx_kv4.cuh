// The 4-bit key/value cache: where a block keeps each code and parameter.
//
// A block (one page of one head) is page_size/16 granules of 16 tokens, each contiguous:
//   [16 x D/2 key codes][16 x G key parameters][16 x D/2 value codes][16 x G value parameters]
// (G = D/64 groups; a parameter is the F16 step in the low half and the F16 minimum in the high
// half of a 32-bit word), so one bulk copy brings a granule, or its keys or values alone, into shared
// memory.
// A code row is D/8 words of eight consecutive channels, channel c in nibble c % 8 of its word.
// The words of a row are ordered for the attention kernel's shared-memory reads:
//   keys:   a lane (token row g, t = 0..3) of an m16n8k16 A fragment takes words 2t and 2t+1 of every
//           group; they are stored together, 16 bytes at a time (D >= 128), and at D = 256 the two
//           halves of a row change places in odd tokens (two rows of 128 bytes read in one phase).
//   values: a lane takes word g of every group; stored together, with the position rotated by the
//           token so that the four rows read in one phase fall into different banks.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/sushi_exl3.h"
#include "sx_common.cuh"
#include "sx_internal.h"

namespace sx {

constexpr int kKvGroup = 64;    // channels that share a step and a minimum
// Inputs past this count as it: 15 s + m, with s and m rounded to F16, then stays within F16.
constexpr float kKvLargest = 57344.0f;
constexpr int kKvGranule = 16;  // tokens of one contiguous piece of a block

__host__ __device__ constexpr int kv4_granule_bytes(int D) { return kKvGranule * (D + 8 * (D / kKvGroup)); }
__host__ __device__ constexpr int kv4_kpar_off(int D) { return kKvGranule * D / 2; }
__host__ __device__ constexpr int kv4_value_off(int D) { return kv4_granule_bytes(D) / 2; }
__host__ __device__ constexpr int kv4_vpar_off(int D) { return kv4_value_off(D) + kKvGranule * D / 2; }

// Byte offset in a granule of the key word (group gr, word w of 8) of token tok (0..15).
template <int D>
__device__ __forceinline__ int kv4_key_word(int tok, int gr, int w) {
    const int row = tok * (D / 2);
    if (D == 64) return row + w * 4;
    if (D == 128) return row + (w >> 1) * 16 + gr * 8 + (w & 1) * 4;
    return row + (((gr >> 1) ^ (tok & 1)) * 4 + (w >> 1)) * 16 + (gr & 1) * 8 + (w & 1) * 4;
}

// Byte offset in a granule of the value word (group gr, word w of 8) of token tok.
template <int D>
__device__ __forceinline__ int kv4_value_word(int tok, int gr, int w) {
    const int row = kv4_value_off(D) + tok * (D / 2);
    if (D == 64) return row + w * 4;
    if (D == 128) return row + (w ^ (((tok >> 1) & 1) * 4)) * 8 + gr * 4;
    return row + (w ^ ((tok & 3) * 2)) * 16 + gr * 4;
}

// The granule of token `tok` (0 .. page_size - 1) of head h in page `page`.
template <int D>
__device__ __forceinline__ size_t kv4_granule(long long page, int kv_heads, int h, int page_size, int tok) {
    return ((size_t)page * kv_heads + h) * (size_t)(page_size / kKvGranule) * kv4_granule_bytes(D) +
           (size_t)(tok / kKvGranule) * kv4_granule_bytes(D);
}

constexpr int kKvMostRequests = 16384;  // a call's: two words each in shared memory

inline bool kv4_page_ok(int p) { return p == 16 || p == 32 || p == 64 || p == 128 || p == 256; }
inline bool kv4_dim_ok(int d) { return d == 64 || d == 128 || d == 256; }

// The admission every entry point of the cache shares.
inline sx_status kv4_check(const sx_kv4* c) {
    if (!c || !c->pool) return SX_ERR_NULL_POINTER;
    if (c->pages < 1 || c->kv_heads < 1 || !kv4_dim_ok(c->head_dim) || !kv4_page_ok(c->page_size)) return SX_ERR_BAD_SHAPE;
    if (reinterpret_cast<uintptr_t>(c->pool) % 16) return SX_ERR_BAD_SHAPE;
    return SX_OK;
}

}  // namespace sx
