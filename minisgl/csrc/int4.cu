// Products with 4-bit weights under group scales:
//   out[m, n] = sum_k x[m, k] (c[n, k] - z[n, k / G]) s[n, k / G] (+ bias[n])
// for few rows x (decode batches). Weight layout: minisgl/quant/int4.py.
//
// The weights are read once and dominate the bytes: 16 bytes per lane are 16
// rows x 64 columns per warp, already in the order of the first operand of the
// warp-level 16 x 8 x 32 integer product; x (up to 8 rows) is the second.
#include <cuda_fp8.h>

#include <algorithm>
#include <atomic>
#include <stdexcept>
#include <string>

#include "common.cuh"
#include "launch.h"
#include "ops.h"

namespace minisgl {
namespace {

__device__ __forceinline__ float half_bits_to_f32(uint32_t bits, int is_half) {
  return is_half ? __half2float(__ushort_as_half(static_cast<unsigned short>(bits)))
                 : __uint_as_float(bits << 16);
}
__device__ __forceinline__ float load_as_f32(const void* p, int64_t i, int type) {
  if (type == static_cast<int>(DType::kF32)) return static_cast<const float*>(p)[i];
  if (type == static_cast<int>(DType::kF16)) return __half2float(static_cast<const __half*>(p)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}
__device__ __forceinline__ void store_from_f32(void* p, int64_t i, int type, float v) {
  if (type == static_cast<int>(DType::kF32))
    static_cast<float*>(p)[i] = v;
  else if (type == static_cast<int>(DType::kF16))
    static_cast<__half*>(p)[i] = __float2half_rn(v);
  else
    static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}

// 2^(byte - 127); 255 is NaN
__device__ __forceinline__ float e8m0(uint32_t byte) {
  return __uint_as_float(byte == 0 ? 0x00400000u : byte == 255 ? 0x7FC00000u : byte << 23);
}


// ---------------------------------------------------------------------------
// Few rows (up to 8, one operand of a warp-level product): the weight stream.
//
// A unit is kR tiles (1 or 2) of 16 rows x 128 columns: kR KB of codes and their
// scales. Whole tiles are dealt to clusters of S = 1 to 8 CTAs, whose CTAs share
// the columns; the units of a CTA, tile after tile, are cut into one contiguous
// range per warp. Each warp copies its own units into its own ring of shared
// memory (cp.async, kDepth ahead), waits for them alone and multiplies them;
// nothing else synchronises the warps while they stream.
//
// The products are integer: a value of x under a power of two common to its
// row's 128 columns is three 8-bit digits, a code minus 8 is a signed byte after
// one mask, and the tensor cores sum 8-bit products exactly in 32 bits. That
// takes 3 operations for 8 codes, where unpacking them to 16-bit floats takes 9
// (B200, 1 x 51200 x 5120: 39 us with bf16 products, 30 so; at 6.5 TB/s an SM
// has about 44 cycles for the 2048 codes of a KB). A group's scale (and z - 8
// times the sum of x) is applied to its finished sum.
//
// A tile whose units lie in one warp's range is finished there. Where a range
// starts or ends inside a tile, the warp parks its partial sums; after the one
// block barrier the warp that started the tile adds them in warp order. With
// S > 1 finished tiles go to the shared memory of the CTA that owns them and
// are added in rank order after a cluster barrier. Every sum has a fixed order:
// the same inputs give the same bits.
//
// Measured (B200, cold weights, bf16): 1 x 51200 x 5120 in groups of 128 29.9 us
// (4.5 TB/s; a plain read of the bytes 20.6), 1 x 5120 x 25600 19.6, 8 x 5120 x
// 25600 with zero points 24.9, 1 x 5120 x 5120 7.3. What bounds it is latency, not
// the issue of instructions (117 a KB of codes, 2.0 a cycle of the 4 that an SM
// can): with four warps to a scheduler each issues once in 7.4 cycles, of which it
// waits 1.6 for the instruction before, 1.3 for the pipe of its product or
// conversion, 1.1 for its turn and 0.8 for loads of x. In small calls it is some
// 4 us of launch, staging of x and the joins. Deeper rings, 20 or 24 warps and two
// batches of x in flight measured no better.
// ---------------------------------------------------------------------------
constexpr int kDepth = 3;
constexpr int kMaxSmem = 227 * 1024;
// of a CTA of W warps, 16 of which share an SM: the SM's 228 KB less 1 KB of the system's a CTA
template <int W>
constexpr int kCtaSmem = 228 * 1024 * W / 16 - 1024;
static_assert(kCtaSmem<16> == kMaxSmem);
constexpr int kBatch = 4;  // runs of 8 values of x that a thread converts side by side

enum { kXBf16 = 0, kXHalf = 1, kXMx8 = 2 };
struct VecArgs {
  const void* x;
  const uint8_t* x_scales;
  const uint8_t* packed;
  const uint32_t* scales;  // [16-row tiles, groups, 8] pairs
  const uint8_t* zeros;    // [16-row tiles, groups rounded up to even, 8]
  const void* bias;
  void* out;
  int M, N, K, tiles, steps, S;  // tiles of 16 kR rows, steps of 128 columns
  int tiles_each, tiles_more, steps_each, steps_more;
  uint32_t inv_each, inv_more;  // 2^31 / steps_each and / (steps_each + 1), rounded up
  int64_t ldx, ld_xs, ldo;
  int ld_z;  // bytes of a 16-row tile's zero points
  int scale_half, bias_type, out_type;
  int x_kind;
  int x_bytes;     // of the x area
  int recv_slots;  // tiles that a CTA owns at most (S > 1)
};

template <int W, int kR, int G, bool ZERO>
struct VecSmem {
  static constexpr int kGroups = 128 / G;
  static constexpr int kScaleB = kGroups * 32;  // of one tile
  static constexpr int kZeroB = kGroups * 8;
  static constexpr int kUnit = (kR * (1024 + kScaleB + kZeroB) + 15) / 16 * 16;  // 16-byte copies into every slot
  static constexpr int kRing = W * kDepth * kUnit;
  // per step: each row's power of two and, with zero points, each group's sum in two parts
  static constexpr int kSide = 32 + (ZERO ? 64 * kGroups : 0);
};
// bytes between x's rows (three digits of 128 columns a step): an odd
// multiple of 64, so that the eight 16-byte reads of a quarter warp (two rows
// x four lanes) fall into distinct banks
__host__ __device__ inline int vec_x_pitch(int steps) { return steps * 384 + 64; }

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t lds8(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.u8 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}

// 8 values x[m, k .. k + 7] as they lie in memory (zeros past K; K % 8 == 0); MXFP8 rows: two words and the scale
__device__ __forceinline__ uint4 x_raw(const VecArgs& a, int m, int k) {
  if (k >= a.K) return make_uint4(0, 0, 0, 0);
  if (a.x_kind == kXMx8) {  // K % 32 == 0: the 8 values lie under one scale
    const uint2 q = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(a.x) + m * a.ldx + k);
    return make_uint4(q.x, q.y, a.x_scales[m * a.ld_xs + k / 32], 0);
  }
  return *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.x) + m * a.ldx + k);
}
__device__ __forceinline__ void x_values(float (&v)[8], const uint4 raw, int kind) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
  if (kind == kXMx8) {
    const float s = e8m0(raw.z);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w[i >> 1] >> (16 * (i & 1))), __NV_E4M3);
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
      v[2 * i] = f.x * s, v[2 * i + 1] = f.y * s;
    }
  } else if (kind == kXHalf) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      v[2 * i] = f.x, v[2 * i + 1] = f.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[2 * i] = __uint_as_float(w[i] << 16), v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
}

// D (+)= A B on 8-bit integers, 16 x 8 x 32: codes times a digit of x (the top digit signed, the others not)
template <bool TOP, bool FIRST>
__device__ __forceinline__ void mma_i8(int (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
#define MINISGL_MMA(TYPE)                                                                                         \
  if constexpr (FIRST)                                                                                            \
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8." TYPE ".s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};" \
        : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])                                                          \
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "r"(0));                                  \
  else                                                                                                            \
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8." TYPE ".s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};" \
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])                                                          \
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1))
  if constexpr (TOP) {
    MINISGL_MMA("s8");
  } else {
    MINISGL_MMA("u8");
  }
#undef MINISGL_MMA
}

// What the infinities and NaN of x add to an output: sum over columns [k, k_end) with x not finite of x * W
// (the digits of such values are zero). Never on the path of finite inputs.
__device__ __noinline__ float not_finite_part(const VecArgs& a, int64_t tile, int r, int m, int group, int k, int k_end) {
  const int64_t n = tile * 16 + r;
  if (n >= a.N || m >= a.M) return 0.f;
  float sum = 0.f;
  for (; k < k_end; k += 8) {
    float v[8];
    x_values(v, x_raw(a, m, k), a.x_kind);
    for (int j = 0; j < 8; ++j) {
      if (fabsf(v[j]) <= 3.4028234e38f) continue;
      const int c = (k + j) % 64, t = c % 16 / 4, q = c % 4 / 2, e = c % 2;
      const uint32_t word = reinterpret_cast<const uint32_t*>(
          a.packed)[((tile * a.steps * 2 + (k + j) / 64) * 32 + 4 * (r & 7) + t) * 4 + c / 16];
      const int code = (word >> (4 * (4 * e + 2 * q + (r >> 3))) & 15) ^ 8;
      const int64_t gi = tile * (a.steps * 128 / group) + (k + j) / group;
      const uint32_t zz = a.zeros != nullptr ? a.zeros[tile * a.ld_z + (k + j) / group * 8 + (r & 7)] : 0x88u;
      const uint32_t sw = a.scales[gi * 8 + (r & 7)];
      const float s = half_bits_to_f32(r >> 3 ? sw >> 16 : sw & 0xFFFFu, a.scale_half);
      sum += v[j] * (static_cast<float>(code - static_cast<int>(r >> 3 ? zz >> 4 : zz & 15u)) * s);
    }
  }
  return sum;
}

__device__ __forceinline__ void store_sum(const VecArgs& a, int64_t tile, int r, int m, float v) {
  const int64_t n = tile * 16 + r;
  if (n >= a.N || m >= a.M) return;
  if (a.bias != nullptr) v += load_as_f32(a.bias, n, a.bias_type);
  store_from_f32(a.out, m * a.ldo + n, a.out_type, v);
}

template <int W, int kR, int G, bool ZERO>
__global__ void __launch_bounds__(W * 32, 16 / W) int4_vec_kernel(const VecArgs a) {
  using L = VecSmem<W, kR, G, ZERO>;
  constexpr int P = L::kGroups;  // groups of a unit
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  pdl_launch_dependents();
  // whole tiles are dealt to clusters, 128-column steps to the CTAs of a cluster, units to warps; each as even as
  // can be, the first ones taking one more
  const int S = a.S;
  int rank = 0, cluster = blockIdx.x;
  if (S > 1) cluster = blockIdx.x / S, rank = blockIdx.x - cluster * S;
  const int t0 = cluster * a.tiles_each + min(cluster, a.tiles_more);
  const int t1 = t0 + a.tiles_each + (cluster < a.tiles_more ? 1 : 0);
  const int k0 = rank * a.steps_each + min(rank, a.steps_more);
  const int ks = a.steps_each + (rank < a.steps_more ? 1 : 0);
  const int units = (t1 - t0) * ks;
  auto warp_start = [&](int w) { return units / W * w + (units % W * w) / W; };
  const int u0 = warp_start(warp), u1 = warp_start(warp + 1);
  float4* park = reinterpret_cast<float4*>(smem + L::kRing);  // [warp][2: head, tail][R][lane]
  uint8_t* xs = smem + L::kRing + W * 2 * 512 * kR;
  const int pitch = vec_x_pitch(ks);
  uint8_t* side = xs + a.M * pitch;                          // [step][power of two | P sums of two parts][8]
  float4* recv = reinterpret_cast<float4*>(xs + a.x_bytes);  // [slot][rank][R][lane]
  const uint32_t inv = rank < a.steps_more ? a.inv_more : a.inv_each;
  auto by_ks = [&](int n) { return static_cast<int>(static_cast<uint64_t>(static_cast<uint32_t>(n)) * inv >> 31); };  // n / ks
  const int u0_tile = by_ks(u0);
  int tile = t0 + u0_tile, k = u0 - u0_tile * ks;

  // the codes of the warp's first units, on their way to L2 while the kernel before this one ends (a prefetch
  // carries no value: the copies below read memory after griddepcontrol.wait)
  {
    constexpr int kLanes = 8 * kR;  // of a unit: a 128-byte line each
    const int ahead = k + lane / kLanes;  // the units run on through the tile, then in the next
    if (u0 + lane / kLanes < u1) {
      const int on = ahead >= ks ? by_ks(ahead) : 0;
      const int64_t row16 = static_cast<int64_t>(tile + on) * kR + (lane >> 3 & (kR - 1));
      asm volatile("prefetch.global.L2 [%0];" ::"l"(a.packed + (row16 * a.steps + k0 + ahead - on * ks) * 1024 + (lane & 7) * 128));
    }
  }
  pdl_wait();

  const uint32_t ring = smem_u32(smem) + warp * (kDepth * L::kUnit);
  // a unit's second tile lies a.steps units of memory behind its first
  const int64_t first = static_cast<int64_t>(tile) * kR * a.steps + k0 + k;
  const uint8_t* src_w = a.packed + first * 1024 + lane * 16;
  constexpr int SW = 8 * P, ZW = 2 * P;  // scale and zero words of a tile
  const uint32_t* src_s = a.scales + (first + (P < 4 && lane >= SW ? a.steps : 0)) * SW + (P < 4 ? lane % SW : lane);
  const uint8_t* src_z =
      ZERO ? a.zeros + (static_cast<int64_t>(tile) * kR + (lane >= ZW ? 1 : 0)) * a.ld_z + (k0 + k) * SW + lane % ZW * 4 : nullptr;
  int left = u1 - u0, pk = k;
  // from the end of a pair's columns to the start of the next pair's
  const int64_t skip = kR * a.steps - ks;
  const int skip_z = kR * a.ld_z - ks * SW;
  const int64_t second = static_cast<int64_t>(a.steps) * 1024;
  auto fetch = [&](uint32_t dst) {
    if (left > 0) {
      --left;
#pragma unroll
      for (int r = 0; r < kR; ++r) {
        cp_async16(dst + r * 1024 + lane * 16, src_w + r * second);
        cp_async16(dst + r * 1024 + 512 + lane * 16, src_w + r * second + 512);
      }
      if constexpr (P < 4) {
        if (lane < kR * SW) cp_async4(dst + kR * 1024 + lane * 4, src_s);
      } else {
#pragma unroll
        for (int r = 0; r < kR; ++r) cp_async4(dst + kR * 1024 + (r * SW + lane) * 4, src_s + r * a.steps * SW);
      }
      if (ZERO && lane < kR * ZW) cp_async4(dst + kR * (1024 + L::kScaleB) + lane * 4, src_z);
      src_w += 1024;
      src_s += SW;
      if (ZERO) src_z += SW;
      if (++pk == ks) {
        pk = 0;
        src_w += skip * 1024;
        src_s += skip * SW;
        if (ZERO) src_z += skip_z;
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  // the first of x's loads go ahead of the weights', which they would else queue behind
  uint4 ahead[kBatch];
  // run c of row m: a warp's 32 runs are of one row or (ks odd) of two neighbours
  const int per_row = ks * 16;
  int xm = 0, xc = threadIdx.x;
  while (xc >= per_row) xc -= per_row, ++xm;
  int lm = xm, lc = xc;
  auto next_run = [&](int& m, int& c) {
    c += W * 32;
    while (c >= per_row) c -= per_row, ++m;
  };
  auto load_x = [&]() {
#pragma unroll
    for (int q = 0; q < kBatch; ++q) {
      if (lm < a.M) ahead[q] = x_raw(a, lm, k0 * 128 + lc * 8);
      next_run(lm, lc);
    }
  };
  load_x();
#pragma unroll
  for (int d = 0; d < kDepth; ++d) fetch(ring + d * L::kUnit);

  // x as 24-bit integers [row][step][digit][columns]: a row's 128 columns under a power of two that puts their
  // largest value into [2^21, 2^22), rounded to nearest: exact for what lies above 2^-14 of it (bf16; fp16
  // 2^-11, E4M3 2^-18), else at most 2^-22 of it off: what one rounding of a float32 sum that holds the largest
  // value costs. The power stops at 2^122: a block below 2^-101 keeps an absolute 2^-123. Two digits would do for
  // bf16 results beside moderate outliers, three keep float32 results right.
  bool odd = false;  // met an infinity or NaN
  const int batches = (a.M * per_row + kBatch * W * 32 - 1) / (kBatch * W * 32);
#pragma unroll 1
  for (int batch = 0; batch < batches; ++batch) {
    // kBatch runs a thread side by side: their shuffles and conversions do not wait for one another
    float v[kBatch][8];
    uint32_t top[kBatch];
    int m[kBatch], c[kBatch];
#pragma unroll
    for (int q = 0; q < kBatch; ++q) {
      m[q] = xm, c[q] = xc;
      next_run(xm, xc);
      x_values(v[q], m[q] < a.M ? ahead[q] : make_uint4(0, 0, 0, 0), a.x_kind);
    }
    if (batch + 1 < batches) load_x();  // the next batch is on its way while this one is converted
#pragma unroll
    for (int q = 0; q < kBatch; ++q) {
      auto largest = [&]() {
        uint32_t b[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) b[j] = __float_as_uint(v[q][j]) & 0x7FFFFFFFu;
        return max(__vimax3_u32(b[0], b[1], b[2]), __vimax3_u32(max(b[3], b[4]), b[5], max(b[6], b[7])));
      };
      top[q] = largest();
      if (top[q] >= 0x7F800000u) {
        odd = true;
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (!(fabsf(v[q][j]) <= 3.4028234e38f)) v[q][j] = 0.f;
        top[q] = largest();
      }
    }
    // 16 lanes share a row's 128 columns
#pragma unroll
    for (int o = 1; o < 16; o <<= 1)
#pragma unroll
      for (int q = 0; q < kBatch; ++q) top[q] = max(top[q], __shfl_xor_sync(0xffffffffu, top[q], o));
    int sum[kBatch];
#pragma unroll
    for (int q = 0; q < kBatch; ++q) {
      const int step = c[q] >> 4;
      const uint32_t e = max(top[q] >> 23, 26u);
      const float up = __uint_as_float((275u - e) << 23);
      uint32_t xi[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) xi[j] = __float_as_uint(fmaf(v[q][j], up, 12582912.f)) - 0x4B400000u;  // 1.5 * 2^23
      sum[q] = 0;
      if constexpr (ZERO) {
#pragma unroll
        for (int j = 0; j < 8; ++j) sum[q] += static_cast<int>(xi[j]);
      }
      if (m[q] >= a.M) continue;
      // lane 4 g + t reads columns 4 t .. 4 t + 3 of each 16: this run is two lanes' words
      uint8_t* dst = xs + m[q] * pitch + step * 384 + (c[q] >> 3 & 1) * 64 + (c[q] & 1) * 32 + (c[q] >> 1 & 3) * 4;
#pragma unroll
      for (int l = 0; l < 2; ++l) {  // columns 0, 2, 1, 3: the order of a code word's bytes
        const uint32_t t0 = __byte_perm(xi[4 * l], xi[4 * l + 2], 0x5140), t1 = __byte_perm(xi[4 * l + 1], xi[4 * l + 3], 0x5140);
        const uint32_t t2 = __byte_perm(xi[4 * l], xi[4 * l + 2], 0x0062), t3 = __byte_perm(xi[4 * l + 1], xi[4 * l + 3], 0x0062);
        *reinterpret_cast<uint32_t*>(dst + l * 16) = __byte_perm(t0, t1, 0x5410);
        *reinterpret_cast<uint32_t*>(dst + l * 16 + 128) = __byte_perm(t0, t1, 0x7632);
        *reinterpret_cast<uint32_t*>(dst + l * 16 + 256) = __byte_perm(t2, t3, 0x5410);
      }
      // codes count in sixteenths (they sit in a byte's upper half): 2^-4 goes with the power of two
      if ((c[q] & 15) == 0)
        *reinterpret_cast<float*>(side + step * L::kSide + m[q] * 4) = __uint_as_float((e - 25u) << 23);
    }
    if constexpr (ZERO) {
#pragma unroll
      for (int o = 1; o < G / 8; o <<= 1)
#pragma unroll
        for (int q = 0; q < kBatch; ++q) sum[q] += __shfl_xor_sync(0xffffffffu, sum[q], o);
#pragma unroll
      for (int q = 0; q < kBatch; ++q)
        if (m[q] < a.M && (c[q] & (G / 8 - 1)) == 0)
          *reinterpret_cast<int2*>(side + (c[q] >> 4) * L::kSide + 32 + (c[q] & 15) / (G / 8) * 64 + m[q] * 8) =
              make_int2(sum[q] & 0xFFFF, sum[q] >> 16);
    }
  }
  odd = __syncthreads_or(odd);
  if (S > 1) cluster_sync();  // the peers have started: their shared memory may be written

  // a finished pair of tiles, this CTA's columns
  auto emit = [&](int tile, float (&acc)[kR][4]) {
    if (odd) {
#pragma unroll
      for (int r = 0; r < kR; ++r)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          acc[r][j] += not_finite_part(a, static_cast<int64_t>(tile) * kR + r, g + (j >> 1) * 8, 2 * t + (j & 1), G,
                                       k0 * 128, min(a.K, (k0 + ks) * 128));
    }
    if (S == 1) {
#pragma unroll
      for (int r = 0; r < kR; ++r)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          store_sum(a, static_cast<int64_t>(tile) * kR + r, g + (j >> 1) * 8, 2 * t + (j & 1), acc[r][j]);
    } else {
      const int local = tile - t0;
      const uint32_t base = map_shared_rank(smem_u32(recv + (local / S * S + rank) * (kR * 32) + lane), local % S);
#pragma unroll
      for (int r = 0; r < kR; ++r)
        asm volatile("st.shared::cluster.v4.f32 [%0], {%1,%2,%3,%4};" ::"r"(base + r * 512), "f"(acc[r][0]),
                     "f"(acc[r][1]), "f"(acc[r][2]), "f"(acc[r][3])
                     : "memory");
    }
  };

  float acc[kR][4];
#pragma unroll
  for (int r = 0; r < kR; ++r)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[r][j] = 0.f;
  bool head = k != 0;  // the pair was started by the warp before
  const uint32_t x_row = smem_u32(xs) + g * pitch + t * 16;
  uint32_t side_at = smem_u32(side) + t * 8;
  uint32_t src = ring;
  // rows past M stay zero: their lanes never load
  uint4 xv[3][2];
#pragma unroll
  for (int d = 0; d < 3; ++d) xv[d][0] = xv[d][1] = make_uint4(0, 0, 0, 0);
#pragma unroll 1
  for (int u = u0; u < u1;) {
    const int run = min(ks - k, u1 - u);  // this warp's units of the pair
    uint32_t x_at = x_row + k * 384, sd = side_at + k * L::kSide;
#pragma unroll 1
    for (int i = 0; i < run; ++i, x_at += 384, sd += L::kSide) {
      asm volatile("cp.async.wait_group %0;" ::"n"(kDepth - 1) : "memory");
      __syncwarp();
      uint32_t sc[kR][P], zz[kR][P];
      uint32_t f[kR][4][4];  // the first operand
#pragma unroll
      for (int r = 0; r < kR; ++r) {
#pragma unroll
        for (int p = 0; p < P; ++p) {
          sc[r][p] = lds32(src + kR * 1024 + (SW * r + 8 * p + g) * 4);
          zz[r][p] = ZERO ? lds8(src + kR * (1024 + L::kScaleB) + SW * r + 8 * p + g) : 0x88u;
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint4 w = lds128(src + r * 1024 + h * 512 + lane * 16);
          // bytes whose upper halves are the signed codes c - 8: row g's are the low nibbles, row g + 8's the high
          f[r][2 * h][0] = w.x << 4 & 0xF0F0F0F0u, f[r][2 * h][1] = w.x & 0xF0F0F0F0u;
          f[r][2 * h][2] = w.y << 4 & 0xF0F0F0F0u, f[r][2 * h][3] = w.y & 0xF0F0F0F0u;
          f[r][2 * h + 1][0] = w.z << 4 & 0xF0F0F0F0u, f[r][2 * h + 1][1] = w.z & 0xF0F0F0F0u;
          f[r][2 * h + 1][2] = w.w << 4 & 0xF0F0F0F0u, f[r][2 * h + 1][3] = w.w & 0xF0F0F0F0u;
        }
      }
      __syncwarp();  // every lane has read the slot
      fetch(src);
      src = src + L::kUnit == ring + kDepth * L::kUnit ? ring : src + L::kUnit;
      if (g < a.M) {
#pragma unroll
        for (int d = 0; d < 3; ++d) {
          xv[d][0] = lds128(x_at + d * 128);
          xv[d][1] = lds128(x_at + d * 128 + 64);
        }
      }
      const uint2 pw = lds64(sd);
#pragma unroll
      for (int p = 0; p < P; ++p) {
        int c[kR][3][4];
        // products of one digit and tile wait for one another; the 3 R chains run side by side
#pragma unroll
        for (int j = p * 4 / P; j < (p + 1) * 4 / P; ++j) {
#pragma unroll
          for (int r = 0; r < kR; ++r) {
#pragma unroll
            for (int d = 0; d < 3; ++d) {
              const uint4 v = xv[d][j >> 1];
              const uint32_t b0 = j & 1 ? v.z : v.x, b1 = j & 1 ? v.w : v.y;
              if (j == p * 4 / P) {
                if (d == 2)
                  mma_i8<true, true>(c[r][d], f[r][j], b0, b1);
                else
                  mma_i8<false, true>(c[r][d], f[r][j], b0, b1);
              } else {
                if (d == 2)
                  mma_i8<true, false>(c[r][d], f[r][j], b0, b1);
                else
                  mma_i8<false, false>(c[r][d], f[r][j], b0, b1);
              }
            }
          }
        }
        uint4 sums;
        if constexpr (ZERO) sums = lds128(sd + 32 + p * 64 + t * 8);
#pragma unroll
        for (int r = 0; r < kR; ++r) {
          float s0, s1;
          if (a.scale_half) {
            const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&sc[r][p]));
            s0 = h.x, s1 = h.y;
          } else {
            s0 = __uint_as_float(sc[r][p] << 16), s1 = __uint_as_float(sc[r][p] & 0xFFFF0000u);
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            // at most 2^22 (256 + 1) in the lower part, 2^20 in the upper: exact integers, one rounding to float32
            // each and one where they meet
            int lo = c[r][1][j] * 256 + c[r][0][j], hi = c[r][2][j];
            if constexpr (ZERO) {
              const int z = 16 * static_cast<int>(j < 2 ? zz[r][p] & 15u : zz[r][p] >> 4) - 128;  // 16 (z - 8)
              lo -= z * static_cast<int>(j & 1 ? sums.z : sums.x);
              hi -= z * static_cast<int>(j & 1 ? sums.w : sums.y);
            }
            const float v = fmaf(static_cast<float>(hi), 65536.f, static_cast<float>(lo));
            acc[r][j] = fmaf(v * (j < 2 ? s0 : s1), __uint_as_float(j & 1 ? pw.y : pw.x), acc[r][j]);
          }
        }
      }
    }
    u += run;
    k += run;
    if (!head && k == ks) {
      emit(tile, acc);
    } else {
      float4* dst = park + (warp * 2 + (head ? 0 : 1)) * (kR * 32) + lane;
#pragma unroll
      for (int r = 0; r < kR; ++r) dst[r * 32] = make_float4(acc[r][0], acc[r][1], acc[r][2], acc[r][3]);
    }
    head = false;
    ++tile;
    k = 0;
#pragma unroll
    for (int r = 0; r < kR; ++r)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[r][j] = 0.f;
  }
  __syncthreads();
  // the pair that this warp started and did not finish: its own part, then the heads of the warps after it
  if (u1 > u0) {
    const int last = by_ks(u1 - 1);   // pair of the last unit, from t0
    const int end = (last + 1) * ks;  // one past the pair's units
    if (end > u1 && last * ks >= u0) {
      for (int w = warp; w < W; ++w) {
        const int b = warp_start(w);
        if (b >= end) break;
        if (warp_start(w + 1) == b) continue;
        const float4* part = park + (w * 2 + (w == warp ? 1 : 0)) * (kR * 32) + lane;
#pragma unroll
        for (int r = 0; r < kR; ++r) {
          const float4 v = part[r * 32];
          acc[r][0] += v.x, acc[r][1] += v.y, acc[r][2] += v.z, acc[r][3] += v.w;
        }
      }
      emit(t0 + last, acc);
    }
  }
  if (S > 1) {
    cluster_sync();
    // a row's 16 R outputs of a tile by neighbouring threads
    for (int i = threadIdx.x; i < a.recv_slots * 16 * kR * a.M; i += W * 32) {
      const int n = i % (16 * kR), rest = i / (16 * kR), sl = rest / a.M, m = rest - sl * a.M;
      const int tl = t0 + sl * S + rank;
      if (tl >= t1) break;
      // where the owning lane put it: lane 4 (n % 8) + m / 2, value 2 (n / 8) + m % 2
      const int at = (n >> 4) * 128 + ((n & 7) * 4 + m / 2) * 4 + (n >> 3 & 1) * 2 + (m & 1);
      const float* part = reinterpret_cast<const float*>(recv) + sl * S * (kR * 128) + at;
      float v = 0.f;
      for (int r = 0; r < S; ++r) v += part[r * (kR * 128)];
      store_sum(a, static_cast<int64_t>(tl) * kR + (n >> 4), n & 15, m, v);
    }
  }
}

// Codes two per byte, row after row, into the tile layout (minisgl/quant/int4.py): one thread makes the 16 bytes of
// one lane. Words are 4 columns of rows g and g + 8, two bytes of each.
__global__ void __launch_bounds__(256) int4_pack_kernel(uint4* out, const uint8_t* codes, int64_t n, int64_t row_bytes,
                                                        int64_t ld, int blocks, int64_t total) {
  pdl_wait();  // no early launch of the kernels after it: they may read the layout at once
  const int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (i >= total) return;
  const int lane = static_cast<int>(i & 31), g = lane >> 2, t = lane & 3;
  const int64_t unit = i >> 5, tile = unit / blocks, block = unit - tile * blocks;
  uint32_t w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int64_t at = block * 32 + 8 * j + 2 * t;  // columns 2 at .. of the row
    uint32_t b[2][2] = {};
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int64_t row = tile * 16 + g + 8 * h;
      if (row < n && at < row_bytes) {  // whole runs of 4 columns: K is a multiple of 8
        b[h][0] = codes[row * ld + at];
        b[h][1] = codes[row * ld + at + 1];
      }
    }
    // bytes (e, p): the low nibble is row g's column 2 p + e, the high one row g + 8's
    w[j] = 0;
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      w[j] |= ((b[0][p] & 15u) | (b[1][p] & 15u) << 4) << (8 * p);
      w[j] |= (b[0][p] >> 4 | (b[1][p] >> 4) << 4) << (16 + 8 * p);
    }
    w[j] ^= 0x88888888u;  // c - 8, two's complement
  }
  out[i] = make_uint4(w[0], w[1], w[2], w[3]);
}

// How a call is cut up: warps of a CTA, tiles of 16 rows that a unit holds, CTAs that share a tile's columns.
struct VecPlan {
  int W, R, S, clusters, tiles, x_bytes, recv_slots, smem;
  int64_t cost;
};

// Per device and kernel: its shared-memory limit raised, and how many clusters of each size fit at once.
template <auto kern, int W>
int resident_clusters(int S) {
  constexpr int kDevices = 64;
  static std::atomic<int> known[kDevices][8];
  int dev = 0;
  cudaGetDevice(&dev);
  const int at = S - 1;
  int n = dev < kDevices ? known[dev][at].load() : 0;
  if (n > 0) return n;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem);
  if (e != cudaSuccess) throw std::runtime_error(std::string("minisgl.int4_linear: ") + cudaGetErrorString(e));
  if (S == 1) {
    cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    n *= 16 / W;
  } else {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(S);
    cfg.blockDim = dim3(W * 32);
    cfg.dynamicSmemBytes = kCtaSmem<W>;
    cudaLaunchAttribute at2;
    at2.id = cudaLaunchAttributeClusterDimension;
    at2.val.clusterDim.x = S;
    at2.val.clusterDim.y = at2.val.clusterDim.z = 1;
    cfg.attrs = &at2;
    cfg.numAttrs = 1;
    e = cudaOccupancyMaxActiveClusters(&n, kern, &cfg);
    if (e != cudaSuccess) throw std::runtime_error(std::string("minisgl.int4_linear: ") + cudaGetErrorString(e));
  }
  if (n < 1) throw std::runtime_error("minisgl.int4_linear: the kernel does not fit this device");
  if (dev < kDevices) known[dev][at].store(n);
  return n;
}

// Estimated time of a call under each plan, in hundredths of what a CTA of 16 warps takes to stream a KB of codes
// (about 0.035 us); fitted to 68 sizes under every plan (B200, cold weights), where the chosen plan is 2.4% slower
// than the best one in the geometric mean and at worst 27%. Both sides of each choice, one of its sizes:
//  - 8 warps, two CTAs to an SM (the next kernel's start overlaps this one's end, few tiles spread further)
//    against 16 (x is staged once per SM): 1 x 2048 x 1024 3.9 against 5.7 us; 8 x 25600 x 5120 27.9 against 24.3.
//  - one 16-row tile to a unit (finer shares of the work) against two (x is read once for both): 1 x 10240 x 5120
//    9.9 against 11.0 us; 2 x 28672 x 4096 with zero points, whose sums are x's too, 19.9 against 17.8.
//  - columns shared by a cluster (less of x to stage, even shares of few tiles) against whole tiles: 6 x 7168 x 7168
//    12.5 (4 CTAs) against 14.6 us; 1 x 28672 x 640 8.1 (2 CTAs) against 6.7. Clusters of 3, 5, 6 and 7 CTAs lost
//    against their neighbours (8 x 14336 x 5120: 5 CTAs 20.7, 4 CTAs 16.2, 8 CTAs 18.1): only powers of two.
constexpr int64_t kCostKb = 100, kCostOneTile = 5, kCostOneTileZeros = 20, kCostXStep = 40, kCostXBatch = 3000,
                  kCostCluster = 8000, kCostClusterCta = 400, kCostWide = 1000, kCostTwoTiles = 3200;
template <int W, int kR, int G, bool ZERO>
void vec_plan(const VecArgs& a, VecPlan& best) {
  using L = VecSmem<W, kR, G, ZERO>;
  constexpr int kPerSm = 16 / W;
  VecPlan p;
  p.W = W, p.R = kR;
  p.tiles = (a.N + 16 * kR - 1) / (16 * kR);
  for (p.S = 1; p.S <= std::min(8, a.steps); p.S *= 2) {
    const int slots = resident_clusters<int4_vec_kernel<W, kR, G, ZERO>, W>(p.S);
    p.clusters = std::min(slots, p.tiles);
    const int64_t per = (p.tiles + p.clusters - 1) / p.clusters, ks = (a.steps + p.S - 1) / p.S;
    const int64_t x_bytes = a.M * static_cast<int64_t>(vec_x_pitch(static_cast<int>(ks))) + ks * L::kSide;
    const int64_t recv_slots = p.S > 1 ? (per + p.S - 1) / p.S : 0;
    const int64_t smem = L::kRing + (W * 2 + recv_slots * p.S) * 512 * kR + x_bytes;
    // n * ks stays below 2^31: the reciprocals are exact
    if (smem > kCtaSmem<W> || per * ks > (1 << 30) / a.steps) continue;
    p.x_bytes = static_cast<int>(x_bytes), p.recv_slots = static_cast<int>(recv_slots), p.smem = static_cast<int>(smem);
    const int sms = std::max(1, slots / kPerSm);  // clusters side by side with one CTA to an SM
    const int64_t on_sm = std::min(kPerSm, (p.clusters + sms - 1) / sms);
    int64_t kb = (per * ks + W - 1) / W * W * kR;  // of a CTA whose warps all take the longest share
    if (kPerSm > 1) kb = std::max(kb, (p.tiles + sms - 1) / sms * ks * kR);
    const int64_t x_batches = (a.M * ks * 16 + kBatch * W * 32 - 1) / (kBatch * W * 32);
    p.cost = kb * (kCostKb + (kR == 1 ? kCostOneTile + (ZERO ? kCostOneTileZeros : 0) : 0)) +
             on_sm * (a.M * ks * kCostXStep + x_batches * kCostXBatch / kPerSm) +
             (p.S > 1 ? kCostCluster + p.S * kCostClusterCta : 0) + (W == 16 ? kCostWide : 0) + (kR == 2 ? kCostTwoTiles : 0);
    if (best.S == 0 || p.cost < best.cost) best = p;
  }
}

template <int W, int kR, int G, bool ZERO>
void launch_vec(VecArgs a, const VecPlan& p, cudaStream_t s) {
  a.tiles = p.tiles;
  a.S = p.S;
  a.tiles_each = a.tiles / p.clusters, a.tiles_more = a.tiles % p.clusters;
  a.steps_each = a.steps / p.S, a.steps_more = a.steps % p.S;
  a.inv_each = static_cast<uint32_t>(((1ull << 31) + a.steps_each - 1) / a.steps_each);
  a.inv_more = static_cast<uint32_t>(((1ull << 31) + a.steps_each) / (a.steps_each + 1));
  a.x_bytes = p.x_bytes;
  a.recv_slots = p.recv_slots;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(p.clusters * p.S));
  cfg.blockDim = dim3(W * 32);
  cfg.dynamicSmemBytes = p.smem;
  cfg.stream = s;
  cudaLaunchAttribute attrs[2];
  int n = 0;
  if (pdl_enabled()) {
    attrs[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (p.S > 1) {
    attrs[n].id = cudaLaunchAttributeClusterDimension;
    attrs[n].val.clusterDim.x = p.S;
    attrs[n].val.clusterDim.y = attrs[n].val.clusterDim.z = 1;
    ++n;
  }
  cfg.attrs = attrs;
  cfg.numAttrs = n;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, int4_vec_kernel<W, kR, G, ZERO>, a);
  if (e != cudaSuccess) throw std::runtime_error(std::string("minisgl: kernel launch failed: ") + cudaGetErrorString(e));
}

// false: x does not fit shared memory under any plan
template <int G, bool ZERO>
bool launch_vec_group(const VecArgs& a, cudaStream_t s) {
  // the sixteen estimates cost a small call's launch some 15% of its time: a decode loop's next sizes are mostly the
  // last layer's, so a thread keeps a few
  struct Known {
    int M = 0, N, K, dev;
    VecPlan p;
  };
  constexpr int kKnown = 64;
  static thread_local Known known[kKnown];
  int dev = 0;
  cudaGetDevice(&dev);
  Known& e = known[(static_cast<unsigned>(a.N) * 2654435761u + static_cast<unsigned>(a.K) * 40503u + a.M) >> 16 & (kKnown - 1)];
  if (e.M != a.M || e.N != a.N || e.K != a.K || e.dev != dev) {
    VecPlan p{};
    vec_plan<8, 1, G, ZERO>(a, p);
    vec_plan<8, 2, G, ZERO>(a, p);
    vec_plan<16, 1, G, ZERO>(a, p);
    vec_plan<16, 2, G, ZERO>(a, p);
    e = Known{a.M, a.N, a.K, dev, p};
  }
  const VecPlan& p = e.p;
  if (p.S == 0) return false;
  if (p.W == 8)
    p.R == 1 ? launch_vec<8, 1, G, ZERO>(a, p, s) : launch_vec<8, 2, G, ZERO>(a, p, s);
  else
    p.R == 1 ? launch_vec<16, 1, G, ZERO>(a, p, s) : launch_vec<16, 2, G, ZERO>(a, p, s);
  return true;
}

}  // namespace

void launch_int4_pack(void* out, const uint8_t* codes, int64_t n, int64_t k, int64_t ld, cudaStream_t s) {
  const int blocks = static_cast<int>(2 * ((k + 127) / 128));
  const int64_t total = 2 * ((n + 31) / 32) * blocks * 32;
  launch_pdl(int4_pack_kernel, dim3(static_cast<unsigned>((total + 255) / 256)), dim3(256), 0, s, static_cast<uint4*>(out),
             codes, n, k / 2, ld, blocks, total);
}

bool launch_int4_stream(const Int4LinearArgs& r, cudaStream_t s) {
  if (r.M > kInt4FewRows) return false;
  VecArgs v{};
  v.x = r.x, v.x_scales = r.x_scales, v.packed = r.packed;
  v.scales = static_cast<const uint32_t*>(r.scales), v.zeros = r.zeros, v.bias = r.bias, v.out = r.out;
  v.M = static_cast<int>(r.M), v.N = static_cast<int>(r.N), v.K = static_cast<int>(r.K);
  v.steps = (v.K + 127) / 128;
  v.ldx = r.ldx, v.ld_xs = r.ld_xs, v.ldo = r.ldo;
  v.ld_z = static_cast<int>((v.steps * (128 / r.group) + 1) / 2 * 16);
  v.scale_half = r.scale_type == DType::kF16;
  v.bias_type = static_cast<int>(r.bias_type), v.out_type = static_cast<int>(r.out_type);
  v.x_kind = r.x_scales != nullptr ? kXMx8 : r.x_type == DType::kF16 ? kXHalf : kXBf16;
  const bool z = v.zeros != nullptr;
  switch (r.group) {
    case 32: return z ? launch_vec_group<32, true>(v, s) : launch_vec_group<32, false>(v, s);
    case 64: return z ? launch_vec_group<64, true>(v, s) : launch_vec_group<64, false>(v, s);
    default: return z ? launch_vec_group<128, true>(v, s) : launch_vec_group<128, false>(v, s);
  }
}

}  // namespace minisgl
