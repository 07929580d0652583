// The 4-bit KV cache's format on the device (minisgl/quant/kv4.py states it).
//
// A group of 32 dims of one token and head has the scale s = (8 + m) 2^(e - 24),
// byte 8 e + m; an element is s (c - 8) with a code c in 0..15. The byte is the
// top of a float's bits: the fp32 number s is (byte << 20) + (106 << 23) and the
// bf16 number (byte << 4) + (106 << 7), since (8 + m) 2^(e - 24) =
// (1 + m / 8) 2^(e - 21) and 106 = 127 - 21. s (c - 8) has at most 4 + 4
// significant bits, so products in bf16 are exact.
#pragma once

#include "common.cuh"

namespace minisgl {
namespace kv4 {

constexpr int kGroup = 32;               // dims under one scale
constexpr uint32_t kScaleF32 = 106u << 23;
constexpr uint32_t kScaleBf16x2 = (106u << 7) | (106u << 23);

__host__ __device__ constexpr int row_code_bytes(int d) { return d / 2; }
__host__ __device__ constexpr int row_scale_bytes(int d) { return d / kGroup; }
__host__ __device__ constexpr int row_bytes(int d) { return d / 2 + d / kGroup; }

// Place of the word of dims 8 u .. 8 u + 7 in a row of K codes.
template <int D>
__device__ __forceinline__ int k_word(int u) {
  return (u & 3) * (D / kGroup) + (u >> 2);
}
// Byte of a V word (and of a V scale word) that belongs to token 4 a + b.
__device__ __forceinline__ int v_byte(int b) { return ((b & 1) << 1) | (b >> 1); }
// Place of 16-byte chunk x (dims 8 x .. 8 x + 7 of four tokens) in row a of V codes.
__device__ __forceinline__ int v_chunk(int a, int x) { return x ^ (2 * (a & 3)); }

__device__ __forceinline__ float scale_f32(uint32_t byte) { return __uint_as_float((byte << 20) + kScaleF32); }

}  // namespace kv4

// Query tokens of request b; offsets outside q make none.
__device__ __forceinline__ int kv4_query_tokens(const int32_t* cu_q, int b, int T) {
  const int from = cu_q[b], to = cu_q[b + 1];
  return from >= 0 && to <= T && to > from ? to - from : 0;
}
// Whether request b's offsets fall. One that does leaves the whole call without work:
// rows counted twice would take the sums of tiles out of 32 bits.
__device__ __forceinline__ bool kv4_offsets_fall(const int32_t* cu_q, int b) { return cu_q[b + 1] < cu_q[b]; }
// Keys of request b, of no more positions than the page table has.
__device__ __forceinline__ int kv4_keys(const int32_t* seq_lens, int b, int ld_pt) { return min(max(seq_lens[b], 0), ld_pt); }

}  // namespace minisgl
