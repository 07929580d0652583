// Rows of the 4-bit paged KV cache: store (with the per-head norms and the
// rotation of queries and keys in the same pass), read-back as bf16 rows or as
// tile images for the attention of many query rows, and copies of whole pages.
//
// The 16-bit counterpart of the store is rope_store.cu; the reference stores
// 16-bit rows only (python/minisgl/kernel/csrc/jit/store.cu:25-53).
#include <algorithm>
#include <stdexcept>

#include "kv4.cuh"
#include "launch.h"
#include "ops.h"

namespace minisgl {
namespace {

using bf16 = __nv_bfloat16;

__device__ __forceinline__ void unpack8(const uint4& raw, float (&x)[8]) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}

// Maximum that keeps a NaN.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Codes of eight dims of one row, four lanes to a group of 32 (whole warps call):
// the scale byte and the word of nibbles (dim i in bits 4 i .. 4 i + 3).
//
// top / 7.5 is rounded up to four significant bits by adding all but one unit of
// the 20 bits that go. x / s is a product with the reciprocal and one correction
// by its remainder (Markstein, IBM J. Res. Dev. 34, 1990): exact where the
// quotient is a float, so that halves between codes, which rows of 8 bits meet
// often, go to the even one as the format says. Adding 1.5 2^23 + 8 rounds it and
// leaves the code in the low bits; words add up with the constants' bits and
// lose those at the end.
__device__ __forceinline__ uint32_t quantize8(const float (&x)[8], uint32_t& word) {
  float top = fabsf(x[0]);
#pragma unroll
  for (int i = 1; i < 8; ++i) top = max_nan(top, fabsf(x[i]));
  top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, 1));
  top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, 2));
  if (top <= 7.5f * 1920.f) {
    const int r = static_cast<int>((__float_as_uint(__fdiv_rn(top, 7.5f)) + 0xfffffu) >> 20);
    const uint32_t byte = static_cast<uint32_t>(max(r - (106 << 3), 0));
    const float s = kv4::scale_f32(byte), inv = __frcp_rn(s);
    constexpr uint32_t kBits = 0x4b400000u;  // of 1.5 2^23
    word = 0u - (kBits * 0x11111111u);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float q = x[i] * inv;
      q = fmaf(fmaf(-q, s, x[i]), inv, q);
      word += __float_as_uint(fminf(q, 7.25f) + 12582920.f) << (4 * i);  // 7.5 would go to 8
    }
    return byte;
  }
  // beyond the range: an infinity's side, NaN as zero
  float most = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) most = fmaxf(most, fabsf(x[i]));  // drops NaN
  const uint32_t four = 0xfu << (threadIdx.x & 28);
  most = fmaxf(most, __shfl_xor_sync(four, most, 1));
  most = fmaxf(most, __shfl_xor_sync(four, most, 2));
  const int r = static_cast<int>((__float_as_uint(__fdiv_rn(most, 7.5f)) + 0xfffffu) >> 20);
  const uint32_t byte = static_cast<uint32_t>(min(max(r - (106 << 3), 0), 255));
  const float s = kv4::scale_f32(byte);
  word = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float q = __fdiv_rn(x[i], s);
    const int c = __float2int_rn(fminf(fmaxf(q, -8.f), 7.f));
    word |= static_cast<uint32_t>(q == q ? c + 8 : 8) << (4 * i);
  }
  return byte;
}

// ================================================================ store ====
// One role a block: queries and keys, kHeads of one token a thread, or values.
//
// A thread has dims 8 x .. 8 x + 7 and those that they turn with, D / 2 on, of its
// heads: no lane waits for another in the rotation, one read of the token's
// cosines and sines (as many bytes as a head) serves 16 dims of each, and all its
// rows are on the way before the first is worked on. Values, four tokens of eight
// dims a thread, so that a run of tokens whose slots fill whole rows of V codes is
// written in 16-byte chunks; other tokens' codes are bytes between those of their
// neighbours. q is rounded once, to bf16 at the end, k and v once, to codes.
//
// Bound by memory where there are many rows, but for the work on each: 8189 rows
// of 64 + 2 x 8 heads, 315 MB read and written, take 65.5 us, 4.8 TB/s (74 % of the
// copy rate). With eight dims a thread and a shuffle for each partner 73, with IEEE
// division calls for the codes 113. A few rows: by the launch and one round of
// loads, 2.3 us for one.
template <int D, int kHeads, bool kQuery>
__device__ __forceinline__ void store_turned(const Kv4StoreArgs& a, int unit, int x, const ErrorSink& err) {
  constexpr int kLanes = D / 16;  // threads of a head
  const int heads = kQuery ? a.hq : a.hk;
  const int per = (heads + kHeads - 1) / kHeads;
  const bool live = unit < a.T * per;  // the others go along for the shuffles
  const int t = live ? unit / per : 0;
  const int h0 = live ? (unit - t * per) * kHeads : 0;
  const bf16* src = static_cast<const bf16*>(kQuery ? a.q : a.k) + static_cast<int64_t>(t) * (kQuery ? a.ld_q : a.ld_k);
  uint4 raw[kHeads][2];
#pragma unroll
  for (int i = 0; i < kHeads; ++i) {
    const uint4* head = reinterpret_cast<const uint4*>(src + min(h0 + i, heads - 1) * D) + x;
    raw[i][0] = head[0], raw[i][1] = head[kLanes];
  }
  float c[8], s[8];
  if (a.cos_sin != nullptr) {
    int pos = a.positions[t];
    if (pos < 0 || pos >= a.max_pos) {
      if (live && x == 0) err.report(kErrBadIndex, 951);
      pos = 0;
    }
    const float4* cs = reinterpret_cast<const float4*>(a.cos_sin + static_cast<int64_t>(pos) * D) + 2 * x;
    *reinterpret_cast<float4*>(c) = cs[0], *reinterpret_cast<float4*>(c + 4) = cs[1];
    *reinterpret_cast<float4*>(s) = cs[D / 8], *reinterpret_cast<float4*>(s + 4) = cs[D / 8 + 1];
  }
  bool stored = false;
  int page = 0, tok = 0;
  if constexpr (!kQuery) {
    const int slot = a.out_loc[t];
    stored = live && slot >= 0 && slot < a.kv_slots;
    if (live && !stored && x == 0) err.report(kErrBadIndex, 952);
    page = slot >> a.page_shift, tok = slot & (a.page_size - 1);
  }
  const bf16* nw = static_cast<const bf16*>(kQuery ? a.q_norm_w : a.k_norm_w);
  uint4 raw_w[2];
  if (nw != nullptr) raw_w[0] = *(reinterpret_cast<const uint4*>(nw) + x), raw_w[1] = *(reinterpret_cast<const uint4*>(nw) + kLanes + x);
#pragma unroll
  for (int i = 0; i < kHeads; ++i) {
    const int h = h0 + i;
    float y[2][8];
    unpack8(raw[i][0], y[0]), unpack8(raw[i][1], y[1]);
    if (nw != nullptr) {
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) sum += y[0][j] * y[0][j] + y[1][j] * y[1][j];
#pragma unroll
      for (int o = 1; o < kLanes; o *= 2) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      const float inv = rsqrtf(sum / D + a.eps);
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        float w[8];
        unpack8(raw_w[u], w);
#pragma unroll
        for (int j = 0; j < 8; ++j) y[u][j] = y[u][j] * inv * w[j];
      }
    }
    if (a.cos_sin != nullptr) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float lo = y[0][j], hi = y[1][j];
        y[0][j] = lo * c[j] - hi * s[j], y[1][j] = hi * c[j] + lo * s[j];
      }
    }
    if constexpr (kQuery) {
      uint4* dst = reinterpret_cast<uint4*>(static_cast<bf16*>(a.q_out) + static_cast<int64_t>(t) * a.ld_qo + h * D) + x;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        uint4 o;
        o.x = pack_bf16x2(y[u][0], y[u][1]), o.y = pack_bf16x2(y[u][2], y[u][3]);
        o.z = pack_bf16x2(y[u][4], y[u][5]), o.w = pack_bf16x2(y[u][6], y[u][7]);
        if (live && h < heads) dst[u * kLanes] = o;
      }
    } else {
      uint8_t* dst = a.k_pool + (static_cast<int64_t>(page) * a.hk + h) * a.page_size * kv4::row_bytes(D);
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        uint32_t word;
        const uint32_t byte = quantize8(y[u], word);
        if (stored && h < heads) {
          reinterpret_cast<uint32_t*>(dst + tok * (D / 2))[kv4::k_word<D>(u * kLanes + x)] = word;
          if (x % 4 == 0)
            dst[a.page_size * (D / 2) + tok * (D / kv4::kGroup) + (u * kLanes + x) / 4] = static_cast<uint8_t>(byte);
        }
      }
    }
  }
}

// Tokens 4 g - shift .. of one head's values, with shift the place of the first
// token in its row of codes.
template <int D>
__device__ __forceinline__ void store_values(const Kv4StoreArgs& a, int unit, int x, const ErrorSink& err) {
  constexpr int kNG = D / kv4::kGroup;
  const int shift = a.out_loc[0] & 3;
  const int g = unit / a.hk, h = unit - g * a.hk;
  const int t0 = g * 4 - shift;
  uint4 raw[4];
  int slot[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int t = t0 + i;
    const bool live = t >= 0 && t < a.T;
    raw[i] = *(reinterpret_cast<const uint4*>(static_cast<const bf16*>(a.v) +
                                              static_cast<int64_t>(min(max(t, 0), a.T - 1)) * a.ld_v + h * D) + x);
    slot[i] = live ? a.out_loc[t] : -1;
    if (live && (slot[i] < 0 || slot[i] >= a.kv_slots)) {
      if (x == 0) err.report(kErrBadIndex, 953);
      slot[i] = -1;
    }
  }
  uint32_t word[4], byte[4];
  bool run = slot[0] >= 0 && (slot[0] & 3) == 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float y[8];
    unpack8(raw[i], y);
    byte[i] = quantize8(y, word[i]);
    run = run && slot[i] == slot[0] + i;
  }
  const int64_t block = static_cast<int64_t>(a.page_size) * kv4::row_bytes(D);
  if (run) {
    const int page = slot[0] >> a.page_shift, row = (slot[0] & (a.page_size - 1)) / 4;
    uint8_t* dst = a.v_pool + (static_cast<int64_t>(page) * a.hk + h) * block;
    // byte j of token i's word to byte v_byte(i) of word j
    const uint32_t e0 = __byte_perm(word[0], word[2], 0x5140), e1 = __byte_perm(word[0], word[2], 0x7362);
    const uint32_t o0 = __byte_perm(word[1], word[3], 0x5140), o1 = __byte_perm(word[1], word[3], 0x7362);
    uint4 q;  // tokens 0, 2, 1, 3 from the low byte up
    q.x = __byte_perm(e0, o0, 0x5410), q.y = __byte_perm(e0, o0, 0x7632);
    q.z = __byte_perm(e1, o1, 0x5410), q.w = __byte_perm(e1, o1, 0x7632);
    *(reinterpret_cast<uint4*>(dst + row * (2 * D)) + kv4::v_chunk(row, x)) = q;
    if (x % 4 == 0)
      reinterpret_cast<uint32_t*>(dst + a.page_size * (D / 2))[row * kNG + x / 4] =
          byte[0] | byte[2] << 8 | byte[1] << 16 | byte[3] << 24;
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (slot[i] < 0) continue;
    const int page = slot[i] >> a.page_shift, tok = slot[i] & (a.page_size - 1);
    const int row = tok / 4, b = kv4::v_byte(tok & 3);
    uint8_t* dst = a.v_pool + (static_cast<int64_t>(page) * a.hk + h) * block;
    uint8_t* codes = dst + row * (2 * D) + kv4::v_chunk(row, x) * 16 + b;
#pragma unroll
    for (int j = 0; j < 4; ++j) codes[4 * j] = static_cast<uint8_t>(word[i] >> (8 * j));
    if (x % 4 == 0) dst[a.page_size * (D / 2) + (row * kNG + x / 4) * 4 + b] = static_cast<uint8_t>(byte[i]);
  }
}

template <int D, int kHeads, int kMin>
__global__ void __launch_bounds__(256, kMin) kv4_store_kernel(const __grid_constant__ Kv4StoreArgs a, int q_blocks,
                                                        int k_blocks) {
  pdl_launch_dependents();
  pdl_wait();
  constexpr int kLanes = D / 16, kUnits = 256 / kLanes;
  const ErrorSink err{a.err};
  const int x = threadIdx.x % kLanes, in = threadIdx.x / kLanes;
  const int block = blockIdx.x, thread = threadIdx.x;
  if (block < q_blocks) store_turned<D, kHeads, true>(a, block * kUnits + in, x, err);
  else if (block < q_blocks + k_blocks) store_turned<D, kHeads, false>(a, (block - q_blocks) * kUnits + in, x, err);
  else store_values<D>(a, (block - q_blocks - k_blocks) * (kUnits / 2) + thread / (D / 8), thread % (D / 8), err);
}

// ================================================================= load ====
// Eight dims of K and of V of one row and head a thread. Values are s (c - 8),
// exact in bf16: 128 + c has the bits 0x4300 | c, and s (128 + c) - 136 s is one
// fused multiply-add (136 s = 17 s 8 has at most 8 significant bits). Bound by
// what it writes, 512 bytes for 136 read of a row of 128 dims.
__device__ __forceinline__ uint4 values8(uint32_t word, uint32_t byte) {
  const uint32_t s2 = byte * 0x00100010u + kv4::kScaleBf16x2;
  const __nv_bfloat162 s = *reinterpret_cast<const __nv_bfloat162*>(&s2);
  const __nv_bfloat162 off = __hmul2(s, __float2bfloat162_rn(-136.f));
  uint32_t p[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    // dims 2 i and 2 i + 1: nibbles 2 i and 2 i + 1 to the halves
    const uint32_t n = word >> (8 * i);
    const uint32_t c2 = (n & 0xfu) | ((n & 0xf0u) << 12) | 0x43004300u;
    const __nv_bfloat162 v = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&c2), s, off);
    p[i] = *reinterpret_cast<const uint32_t*>(&v);
  }
  return make_uint4(p[0], p[1], p[2], p[3]);
}

template <int D>
__device__ __forceinline__ void load_row(const Kv4LoadArgs& a, int slot, int h, int x, uint4& k, uint4& v) {
  constexpr int kNG = D / kv4::kGroup;
  const int page = slot >> a.page_shift, tok = slot & (a.page_size - 1), row = tok / 4, b = kv4::v_byte(tok & 3);
  const int64_t at = (static_cast<int64_t>(page) * a.hk + h) * a.page_size * kv4::row_bytes(D);
  const uint8_t* kb = a.k_pool + at;
  const uint8_t* vb = a.v_pool + at;
  const int codes = a.page_size * (D / 2);
  const uint32_t kw = reinterpret_cast<const uint32_t*>(kb + tok * (D / 2))[kv4::k_word<D>(x)];
  const uint4 vq = *(reinterpret_cast<const uint4*>(vb + row * (2 * D)) + kv4::v_chunk(row, x));
  const uint32_t ks = kb[codes + tok * kNG + x / 4], vs = vb[codes + (row * kNG + x / 4) * 4 + b];
  const uint32_t lo = __byte_perm(vq.x, vq.y, (4 + b) << 4 | b), hi = __byte_perm(vq.z, vq.w, (4 + b) << 4 | b);
  k = values8(kw, ks);
  v = values8(__byte_perm(lo, hi, 0x5410), vs);
}

// Splits the key tiles of all (request, pair of row tiles, KV head) of a prefill
// into runs of equal cost; one block. A row tile has 128 / group tokens. In the
// sequence that is split a pair has kKv4PairCost places before its tiles, for
// what a piece costs beside them (queries in, output out); a pair without any key
// counts as one tile, so that somebody writes its zeros. Runs have four places at
// least: a record costs about as much as a tile.
__device__ void plan_runs(const Kv4LoadArgs& a, const ErrorSink& err) {
  __shared__ int pre[kKv4MaxBatch + 1], units[kKv4MaxBatch + 1];  // sums over the requests: places, pairs x heads
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int W = 2 * (kKv4TileKeys / a.group);  // tokens of a pair
  auto tiles = [&](int b, int q_len, int pair) {
    const int keys = kv4_keys(a.seq_lens, b, a.ld_pt);
    return max(1, (keys - q_len + min(q_len, (pair + 1) * W) + kKv4TileKeys - 1) / kKv4TileKeys);
  };
  // where each request's images begin; a plan that does not hold all of its keys,
  // from its first to its last, has none of them
  for (int b = threadIdx.x; b < a.B; b += 256) {
    const int keys = kv4_keys(a.seq_lens, b, a.ld_pt), row = a.first_row[b];
    auto holds = [&](int at, int pos) { return a.row_req[at] == b && a.row_pos[at] == pos; };
    const bool all = keys == 0 || (row >= 0 && row % kKv4TileKeys == 0 && row <= a.T - keys && holds(row, 0) &&
                                   holds(row + keys - 1, keys - 1));
    if (!all) err.report(kErrBadIndex, 957);
    a.starts[b] = all ? row / kKv4TileKeys : -1;
  }
  bool falls = false;
  for (int b = warp; b < a.B; b += 8) {
    const int q_len = kv4_query_tokens(a.cu_q, b, a.q_rows);
    falls = falls || kv4_offsets_fall(a.cu_q, b);
    if (lane == 0 && (a.cu_q[b] < 0 || a.cu_q[b + 1] > a.q_rows || a.cu_q[b + 1] < a.cu_q[b] || a.seq_lens[b] > a.ld_pt))
      err.report(kErrBadIndex, 956);
    int sum = 0;
    for (int p = lane; p * W < q_len; p += 32) sum += kKv4PairCost + tiles(b, q_len, p);
#pragma unroll
    for (int o = 16; o > 0; o /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) pre[b + 1] = sum * a.hk, units[b + 1] = (q_len + W - 1) / W * a.hk;
  }
  const bool none = __syncthreads_or(falls) != 0;
  if (warp < 2) {
    int* x = warp == 0 ? pre : units;
    int carry = 0;
    for (int b0 = 0; b0 < a.B; b0 += 32) {
      int v = b0 + lane < a.B ? x[b0 + lane + 1] : 0;
#pragma unroll
      for (int o = 1; o < 32; o *= 2) {
        const int u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
      }
      if (b0 + lane < a.B) x[b0 + lane + 1] = carry + v;
      carry += __shfl_sync(0xffffffffu, v, 31);
    }
    if (lane == 0) x[0] = 0;
  }
  __syncthreads();
  const int64_t total = none ? 0 : pre[a.B];
  const int n = static_cast<int>(min(static_cast<int64_t>(a.ctas), max(total / 4, static_cast<int64_t>(1))));
  struct Place {
    int b, pair, h, kt, at, real;  // at: of the pair; real: tiles before
  };
  auto find = [&](int v) {
    Place p{0, 0, 0, 0, 0, 0};
    if (v >= total) {
      p.real = static_cast<int>(total) - kKv4PairCost * units[a.B];
      return p;
    }
    int hi = a.B;  // the last b with pre[b] <= v
    while (hi - p.b > 1) {
      const int mid = (p.b + hi) / 2;
      if (pre[mid] <= v) p.b = mid; else hi = mid;
    }
    const int q_len = kv4_query_tokens(a.cu_q, p.b, a.q_rows);
    int in = v - pre[p.b], t = kKv4PairCost + tiles(p.b, q_len, 0);
    while (in >= t * a.hk) in -= t * a.hk, t = kKv4PairCost + tiles(p.b, q_len, ++p.pair);
    p.h = in / t;
    p.kt = max(0, in - p.h * t - kKv4PairCost);
    p.at = v - (in - p.h * t);
    p.real = p.at - kKv4PairCost * (units[p.b] + p.pair * a.hk + p.h) + p.kt;
    return p;
  };
  for (int i = threadIdx.x; i < a.ctas; i += 256) {
    int4* run = reinterpret_cast<int4*>(a.runs) + 2 * i;
    if (total == 0 || i >= n) {
      run[0] = run[1] = make_int4(0, 0, 1, 1);
      run[1].x = 0;
      continue;
    }
    const Place p = find(static_cast<int>(total * i / n)), q = find(static_cast<int>(total * (i + 1) / n));
    run[0] = make_int4(p.b, p.pair, p.h, p.kt);
    run[1] = make_int4(q.real - p.real, p.at, static_cast<int>(total), n);
  }
}

// Rows of a.slots to k_out / v_out [T, hk, D], or (kImages) rows of a prefill plan
// to tile images: row r is key row_pos[r] of request row_req[r] (none: zeros);
// 128 rows of a head are one K and one V image of D / 64 halves, 128 bytes a row
// and half, whose 16-byte chunks are swizzled as the tcgen05 descriptors read
// them (chunk c of row r at c ^ (r mod 8)).
template <int D, bool kImages>
__global__ void __launch_bounds__(256) kv4_load_kernel(const __grid_constant__ Kv4LoadArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  constexpr int kLanes = D / 8;
  const ErrorSink err{a.err};
  const int x = threadIdx.x % kLanes;
  int64_t block = blockIdx.x;
  if constexpr (kImages) {
    if (block == 0) return plan_runs(a, err);
    --block;
  }
  const int64_t unit = block * (256 / kLanes) + threadIdx.x / kLanes;
  if (unit >= static_cast<int64_t>(a.T) * a.hk) return;
  int h, slot;
  uint4 *k_to, *v_to;
  if constexpr (kImages) {
    const int tile = static_cast<int>(unit / (kKv4TileKeys * a.hk)), in = static_cast<int>(unit % (kKv4TileKeys * a.hk));
    h = in / kKv4TileKeys;
    const int row = in % kKv4TileKeys, r = tile * kKv4TileKeys + row;
    k_to = static_cast<uint4*>(a.k_out) + (static_cast<int64_t>(tile) * a.hk + h) * (2 * kKv4TileKeys * kLanes) +
           (x / 8) * (kKv4TileKeys * 8) + row * 8 + ((x ^ row) & 7);
    v_to = k_to + kKv4TileKeys * kLanes;
    const int req = a.row_req[r], pos = a.row_pos[r];
    slot = -1;
    if (req >= 0 && req < a.B && pos < a.seq_lens[req]) {  // a plan may hold more keys than there are now
      const int table_row = a.req_rows[req];
      if (table_row >= 0 && table_row < a.pt_rows && pos >= 0 && pos < a.ld_pt)
        slot = a.page_table[static_cast<int64_t>(table_row) * a.ld_pt + pos];
      if (slot < 0 || slot >= a.kv_slots) {
        if (x == 0) err.report(kErrBadIndex, 955);
        slot = -1;
      }
    }
  } else {
    const int r = static_cast<int>(unit / a.hk);
    h = static_cast<int>(unit - static_cast<int64_t>(r) * a.hk);
    k_to = static_cast<uint4*>(a.k_out) + unit * kLanes + x;
    v_to = static_cast<uint4*>(a.v_out) + unit * kLanes + x;
    slot = a.slots[r];
    if (slot < 0 || slot >= a.kv_slots) {
      if (x == 0) err.report(kErrBadIndex, 954);
      slot = -1;
    }
  }
  uint4 k = make_uint4(0, 0, 0, 0), v = k;
  if (slot >= 0) load_row<D>(a, slot, h, x, k, v);
  *k_to = k;
  *v_to = v;
}

// ================================================================= copy ====
// Pages of every plane (K / V and layer) of a pool, pair by pair; the pairs
// travel as a kernel argument (32 of them, or 480 where there are more: 256 bytes
// or 4 KB to send with a launch), so a call of up to 480 is one launch and leaves
// nothing behind on the device. grid (chunks of a page, pairs, planes in turn).
// Bound by memory: 500 pages of 64 layers x 8 heads (4-bit, 4.46 GB read and
// written) 659 us, 6.8 TB/s, 103 % of the copy rate; one page 3.1 us.
template <int N>
struct PagePairs {
  int src[N], dst[N];
};
constexpr int kCopyVecs = 4;  // 16-byte vectors a thread

template <int N>
__global__ void __launch_bounds__(256) copy_pages_kernel(uint4* pool, int64_t plane_vecs, int page_vecs, int planes,
                                                         const __grid_constant__ PagePairs<N> pairs) {
  pdl_launch_dependents();
  pdl_wait();
  const int i0 = blockIdx.x * (256 * kCopyVecs) + threadIdx.x;
  const int64_t src = static_cast<int64_t>(pairs.src[blockIdx.y]) * page_vecs;
  const int64_t dst = static_cast<int64_t>(pairs.dst[blockIdx.y]) * page_vecs;
  for (int p = blockIdx.z; p < planes; p += gridDim.z) {
    uint4* base = pool + p * plane_vecs;
    uint4 v[kCopyVecs];
#pragma unroll
    for (int i = 0; i < kCopyVecs; ++i)
      if (i0 + i * 256 < page_vecs) v[i] = __ldcs(base + src + i0 + i * 256);
#pragma unroll
    for (int i = 0; i < kCopyVecs; ++i)
      if (i0 + i * 256 < page_vecs) __stcs(base + dst + i0 + i * 256, v[i]);
  }
}

template <int N>
void copy_pairs(const CopyPagesArgs& a, int from, int n, cudaStream_t s) {
  PagePairs<N> pairs;
  for (int i = 0; i < n; ++i) pairs.src[i] = a.src[from + i], pairs.dst[i] = a.dst[from + i];
  const int page_vecs = static_cast<int>(a.page_bytes / 16);
  const int chunks = (page_vecs + 256 * kCopyVecs - 1) / (256 * kCopyVecs);
  dim3 grid(chunks, n, std::min(a.planes, 65535));
  launch_pdl(copy_pages_kernel<N>, grid, dim3(256), 0, s, static_cast<uint4*>(a.pool), a.plane_bytes / 16, page_vecs,
             a.planes, pairs);
}

}  // namespace

namespace {
template <int D>
void store_typed(const Kv4StoreArgs& a, cudaStream_t s) {
  constexpr int kUnits = 256 / (D / 16);  // of queries and keys in a block; of values half as many
  // One head a thread while they all fit the GPU at once, two up to four times as
  // many, then four. us with 1, 2 and 4 for rows of 64 + 2 x 8 heads of 128 dims:
  // 256 rows 4.3, 4.5, 6.4; 512 7.3, 7.0, 7.5; 1024 12.1, 10.8, 11.4; 2048 19.9,
  // 19.6, 17.1; 8189 74.2, 77.9, 65.5.
  const int64_t wave = int64_t{148} * 5 * kUnits, all = static_cast<int64_t>(a.T) * (a.hq + a.hk);
  const int heads = all <= wave ? 1 : all <= 4 * wave ? 2 : 4;
  auto blocks = [](int64_t units, int per) { return (units + per - 1) / per; };
  const int64_t q = blocks(static_cast<int64_t>(a.T) * ((a.hq + heads - 1) / heads), kUnits);
  const int64_t k = blocks(static_cast<int64_t>(a.T) * ((a.hk + heads - 1) / heads), kUnits);
  const int64_t v = blocks(static_cast<int64_t>((a.T + 6) / 4) * a.hk, kUnits / 2);
  if (q + k + v > 0x7fffffff / kUnits) throw std::runtime_error("minisgl.rope_store_kv4: too many rows");
  auto kern = heads == 1 ? kv4_store_kernel<D, 1, 5> : heads == 2 ? kv4_store_kernel<D, 2, 2> : kv4_store_kernel<D, 4, 3>;
  launch_pdl(kern, dim3(static_cast<unsigned>(q + k + v)), dim3(256), 0, s, a, static_cast<int>(q), static_cast<int>(k));
}
}  // namespace

void launch_kv4_store(const Kv4StoreArgs& a, cudaStream_t s) {
  if (a.T <= 0) return;
  if (a.d == 128) store_typed<128>(a, s);
  else if (a.d == 64) store_typed<64>(a, s);
  else throw std::runtime_error("minisgl.rope_store_kv4: head_dim must be 64 or 128");
}

void launch_kv4_load(const Kv4LoadArgs& a, cudaStream_t s) {
  const bool images = a.runs != nullptr;  // (a plan without keys has no rows)
  if (a.T <= 0 && !images) return;
  if (a.d != 64 && a.d != 128) throw std::runtime_error("minisgl.load_kv4: head_dim must be 64 or 128");
  const int per_block = 256 / (a.d / 8);
  const int64_t blocks = (static_cast<int64_t>(a.T) * a.hk + per_block - 1) / per_block + (images ? 1 : 0);
  if (blocks > 0x7fffffff) throw std::runtime_error("minisgl.load_kv4: too many rows");
  if (images && a.T % kKv4TileKeys != 0)
    throw std::runtime_error("minisgl.prefill_attention_kv4: tile images are of 128 keys");
  auto kern = a.d == 128 ? (images ? kv4_load_kernel<128, true> : kv4_load_kernel<128, false>)
                         : (images ? kv4_load_kernel<64, true> : kv4_load_kernel<64, false>);
  launch_pdl(kern, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, s, a);
}

int launch_copy_pages(const CopyPagesArgs& a, cudaStream_t s) {
  int launches = 0;
  for (int from = 0; from < a.n; ++launches) {
    const int left = a.n - from;
    if (left <= 32) {
      copy_pairs<32>(a, from, left, s);
      from += left;
    } else {
      const int n = std::min(left, 480);  // pairs that fit 4 KB of arguments
      copy_pairs<480>(a, from, n, s);
      from += n;
    }
  }
  return launches;
}

}  // namespace minisgl
