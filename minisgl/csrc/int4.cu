// Products with 4-bit weights under group scales:
//   out[m, n] = sum_k x[m, k] (c[n, k] - z[n, k / G]) s[n, k / G] (+ bias[n])
// for few rows x (decode batches). Weight layout: minisgl/quant/int4.py.
//
// The weights are read once and dominate the bytes, so a tile of them goes
// straight from memory to the registers of the lane that multiplies it: 16
// bytes per lane are 16 rows x 64 columns per warp, already in the order of
// the first operand of the warp-level 16 x 8 x 16 product. x is the second
// operand (8 rows of x per product). Codes become exact bf16 / fp16 integers
// (a nibble under the exponent of 128 / 1024, minus 128 / 1024 + z), are
// multiplied exactly and summed in float32 over at most 64 columns; only then
// is the group's scale applied, in float32.
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

constexpr int kWarps = 8;

struct LinArgs {
  const void* x;
  const uint8_t* x_scales;
  const uint8_t* packed;
  const uint16_t* scales;
  const uint8_t* zeros;
  const void* bias;
  void* out;
  int M, N, K, blocks, groups;
  int64_t ldx, ld_xs, ldo;
  int scale_half, bias_type, out_type;
};

template <typename T>
struct Num;
template <>
struct Num<__nv_bfloat16> {
  static constexpr uint32_t kMagic = 0x43004300u;  // 128 | 128
  __device__ static uint32_t offset(uint32_t z) { return (0x4300u + z) * 0x10001u; }
  __device__ static uint32_t sub(uint32_t a, uint32_t b) {
    const __nv_bfloat162 r = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  __device__ static void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};
template <>
struct Num<__half> {
  static constexpr uint32_t kMagic = 0x64006400u;  // 1024 | 1024
  __device__ static uint32_t offset(uint32_t z) { return (0x6400u + z) * 0x10001u; }
  __device__ static uint32_t sub(uint32_t a, uint32_t b) {
    const __half2 r = __hsub2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  __device__ static void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};

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

// The lane's two runs of 8 values x[m, k .. k + 7] and x[m, k + 32 .. k + 39] as 8 words of pairs
// (zeros past M and K; K % 8 == 0)
template <typename T, bool MX8>
__device__ __forceinline__ void load_x(uint32_t (&r)[8], const LinArgs& a, int m, int k) {
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = 0;
  if (m >= a.M) return;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int kk = k + 32 * h;
    if (kk >= a.K) break;
    if constexpr (!MX8) {
      const uint4 v = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.x) + m * a.ldx + kk);
      r[4 * h] = v.x, r[4 * h + 1] = v.y, r[4 * h + 2] = v.z, r[4 * h + 3] = v.w;
    } else {  // K % 32 == 0: the 8 values lie under one scale
      const uint2 q = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(a.x) + m * a.ldx + kk);
      const float s = e8m0(a.x_scales[m * a.ld_xs + kk / 32]);
      const uint32_t w[2] = {q.x, q.y};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const __half2_raw raw =
            __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w[i >> 1] >> (16 * (i & 1))), __NV_E4M3);
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&raw));
        // four significant bits and a power of two: exact in bf16
        r[4 * h + i] = pack_bf16x2(f.x * s, f.y * s);
      }
    }
  }
}

// One CTA: 16 weight rows, 8 NT rows of x; its warps share the columns.
template <typename T, bool MX8, int NT, int G>
__global__ void __launch_bounds__(kWarps * 32) int4_linear_kernel(const LinArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  __shared__ float red[kWarps][16][8 * NT + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int64_t tile = blockIdx.x;
  const int m0 = blockIdx.y * 8 * NT;
  const int b0 = static_cast<int>(static_cast<int64_t>(a.blocks) * warp / kWarps);
  const int b1 = static_cast<int>(static_cast<int64_t>(a.blocks) * (warp + 1) / kWarps);
  const uint4* wp = reinterpret_cast<const uint4*>(a.packed + tile * a.blocks * 512) + lane;
  const uint16_t* sp = a.scales + tile * a.groups * 16 + 2 * g;
  const uint8_t* zp = a.zeros != nullptr ? a.zeros + tile * a.groups * 8 + g : nullptr;
  float acc[NT][4];
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = 0.f;
#pragma unroll 2
  for (int b = b0; b < b1; ++b) {
    const uint4 w = wp[static_cast<int64_t>(b) * 32];
    const uint32_t words[4] = {w.x, w.y, w.z, w.w};
    uint32_t xr[NT][8];
#pragma unroll
    for (int i = 0; i < NT; ++i) load_x<T, MX8>(xr[i], a, m0 + 8 * i + g, b * 64 + t * 8);
    constexpr int PER = G < 64 ? 64 / G : 1;  // groups inside a block
#pragma unroll
    for (int p = 0; p < PER; ++p) {
      const int64_t gi = b * 64 / G + p;
      const float s0 = half_bits_to_f32(sp[gi * 16], a.scale_half), s1 = half_bits_to_f32(sp[gi * 16 + 1], a.scale_half);
      const uint32_t zz = zp != nullptr ? zp[gi * 8] : 0x88u;
      const uint32_t z0 = Num<T>::offset(zz & 15u), z1 = Num<T>::offset(zz >> 4);
      float part[NT][4];
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) part[i][j] = 0.f;
#pragma unroll
      for (int j = p * 4 / PER; j < (p + 1) * 4 / PER; ++j) {
        uint32_t f[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          f[i] = Num<T>::sub(((words[j] >> (4 * i)) & 0x000F000Fu) | Num<T>::kMagic, (i & 1) ? z1 : z0);
#pragma unroll
        for (int i = 0; i < NT; ++i) Num<T>::mma(part[i], f, xr[i][2 * j], xr[i][2 * j + 1]);
      }
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        acc[i][0] += part[i][0] * s0, acc[i][1] += part[i][1] * s0;
        acc[i][2] += part[i][2] * s1, acc[i][3] += part[i][3] * s1;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    red[warp][g][8 * i + 2 * t] = acc[i][0];
    red[warp][g][8 * i + 2 * t + 1] = acc[i][1];
    red[warp][g + 8][8 * i + 2 * t] = acc[i][2];
    red[warp][g + 8][8 * i + 2 * t + 1] = acc[i][3];
  }
  __syncthreads();
  for (int e = threadIdx.x; e < 16 * 8 * NT; e += kWarps * 32) {
    const int r = e & 15, c = e >> 4;
    const int64_t n = tile * 16 + r;
    const int m = m0 + c;
    if (n >= a.N || m >= a.M) continue;
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) v += red[w][r][c];  // warp order: the same sum every time
    if (a.bias != nullptr) v += load_as_f32(a.bias, n, a.bias_type);
    store_from_f32(a.out, m * a.ldo + n, a.out_type, v);
  }
}

template <typename T, bool MX8, int NT>
void launch_nt(const LinArgs& a, int group, cudaStream_t s) {
  const dim3 grid((a.N + 15) / 16, (a.M + 8 * NT - 1) / (8 * NT));
  switch (group) {
    case 32: launch_pdl(int4_linear_kernel<T, MX8, NT, 32>, grid, dim3(kWarps * 32), 0, s, a); break;
    case 64: launch_pdl(int4_linear_kernel<T, MX8, NT, 64>, grid, dim3(kWarps * 32), 0, s, a); break;
    default: launch_pdl(int4_linear_kernel<T, MX8, NT, 128>, grid, dim3(kWarps * 32), 0, s, a); break;
  }
}

template <typename T, bool MX8>
void launch_type(const LinArgs& a, int group, cudaStream_t s) {
  if (a.M <= 8)
    launch_nt<T, MX8, 1>(a, group, s);
  else if (a.M <= 16)
    launch_nt<T, MX8, 2>(a, group, s);
  else
    launch_nt<T, MX8, 4>(a, group, s);
}

// ---------------------------------------------------------------------------
// Few rows (up to 16): the weight stream.
//
// One CTA of 16 warps per SM, alone or in a cluster of S = 2, 4 or 8 whose
// CTAs share the columns of the cluster's tiles. A unit is 16 rows x 128
// columns (1 KB of codes and its scales); the units of a CTA, tile after tile,
// are cut into one contiguous range per warp. Each warp copies its own units
// into its own ring of shared memory (cp.async, kDepth units ahead), waits for
// them alone and multiplies them; nothing else synchronises the warps while
// they stream. x lies in shared memory for the CTA's columns, once, as 16-bit
// values.
//
// A tile whose units lie in one warp's range is finished there. Where a range
// starts or ends inside a tile, the warp parks its partial sums; after the one
// block barrier the warp that started the tile adds them in warp order. With
// S > 1 finished tiles go to the shared memory of the CTA that owns them and
// are added in rank order after a cluster barrier. Every sum has a fixed order:
// the same inputs give the same bits.
// ---------------------------------------------------------------------------
constexpr int kVecWarps = 16;
constexpr int kDepth = 4;
constexpr int kMaxSmem = 227 * 1024;

struct VecArgs {
  const void* x;
  const uint8_t* x_scales;
  const uint8_t* packed;
  const uint32_t* scales;  // [tiles, groups, 8] pairs
  const uint8_t* zeros;    // [tiles, groups, 8]
  const void* bias;
  void* out;
  int M, N, K, tiles, steps, S;  // steps of 128 columns
  int64_t ldx, ld_xs, ldo;
  int scale_half, bias_type, out_type;
  int x_bytes;     // of the x area
  int recv_slots;  // tiles that a CTA owns at most (S > 1)
};

template <int G>
struct VecSmem {
  static constexpr int kGroups = 128 / G;
  static constexpr int kScaleB = kGroups * 32;
  static constexpr int kZeroB = kGroups * 8 < 16 ? 16 : kGroups * 8;
  static constexpr int kUnit = 1024 + kScaleB + kZeroB;
  static constexpr int kRing = kVecWarps * kDepth * kUnit;
  static int total(int NT, int x_bytes, int recv_slots, int S) {
    return kRing + kVecWarps * 2 * 512 * NT + x_bytes + recv_slots * S * 512 * NT;
  }
};
// bytes between x's rows: an odd multiple of 64, so that the eight 16-byte
// reads of a quarter warp (two rows x four lanes) fall into distinct banks
__host__ __device__ inline int vec_x_pitch(int steps) { return steps * 256 + 64; }

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async8(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
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

// 8 values x[m, k .. k + 7] as 16-bit pairs (zeros past K; K % 8 == 0)
template <typename T, bool MX8>
__device__ __forceinline__ uint4 x_run(const VecArgs& a, int m, int k) {
  if (k >= a.K) return make_uint4(0, 0, 0, 0);
  if constexpr (!MX8) {
    return *reinterpret_cast<const uint4*>(static_cast<const T*>(a.x) + m * a.ldx + k);
  } else {  // K % 32 == 0: the 8 values lie under one scale
    const uint2 q = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(a.x) + m * a.ldx + k);
    const float s = e8m0(a.x_scales[m * a.ld_xs + k / 32]);
    uint32_t r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t w = i < 2 ? q.x : q.y;
      const __half2_raw raw = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w >> (16 * (i & 1))), __NV_E4M3);
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&raw));
      r[i] = pack_bf16x2(f.x * s, f.y * s);  // four significant bits and a power of two: exact in bf16
    }
    return make_uint4(r[0], r[1], r[2], r[3]);
  }
}

__device__ __forceinline__ void store_sum(const VecArgs& a, int64_t tile, int r, int m, float v) {
  const int64_t n = tile * 16 + r;
  if (n >= a.N || m >= a.M) return;
  if (a.bias != nullptr) v += load_as_f32(a.bias, n, a.bias_type);
  store_from_f32(a.out, m * a.ldo + n, a.out_type, v);
}

template <typename T, bool MX8, int NT, int G, bool ZERO>
__global__ void __launch_bounds__(kVecWarps * 32, 1) int4_vec_kernel(const VecArgs a) {
  using L = VecSmem<G>;
  constexpr int P = L::kGroups;  // groups of a unit
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  pdl_launch_dependents();
  const int S = a.S, rank = blockIdx.x % S, cluster = blockIdx.x / S, clusters = gridDim.x / S;
  const int t0 = static_cast<int>(static_cast<int64_t>(a.tiles) * cluster / clusters);
  const int t1 = static_cast<int>(static_cast<int64_t>(a.tiles) * (cluster + 1) / clusters);
  const int k0 = a.steps * rank / S, ks = a.steps * (rank + 1) / S - k0;
  const int64_t units = static_cast<int64_t>(t1 - t0) * ks;
  const int u0 = static_cast<int>(units * warp / kVecWarps), u1 = static_cast<int>(units * (warp + 1) / kVecWarps);
  uint8_t* ring = smem + warp * (kDepth * L::kUnit);
  float4* park = reinterpret_cast<float4*>(smem + L::kRing);  // [warp][2: head, tail][NT][lane]
  uint8_t* xs = smem + L::kRing + kVecWarps * 2 * 512 * NT;
  float4* recv = reinterpret_cast<float4*>(xs + a.x_bytes);  // [slot][rank][NT][lane]
  const int pitch = vec_x_pitch(ks);

  // the codes of the ring's first fill, on their way to L2 while the kernel before this one ends (a prefetch
  // carries no value: the copies below read memory after griddepcontrol.wait)
  {
    const int u = u0 + (lane >> 3);
    if (u < u1) {
      const int64_t tile = t0 + u / ks;
      const uint8_t* p = a.packed + (tile * a.steps + k0 + u % ks) * 1024 + (lane & 7) * 128;
      asm volatile("prefetch.global.L2 [%0];" ::"l"(p));
    }
    static_assert(kDepth == 4, "eight lanes prefetch one unit");
  }
  pdl_wait();

  int pu = u0, ptile = t0 + (ks > 0 ? u0 / ks : 0), pk = ks > 0 ? u0 % ks : 0;
  const uint32_t ring_a = smem_u32(ring);
  auto fetch = [&](int slot) {
    if (pu < u1) {
      const int64_t unit = static_cast<int64_t>(ptile) * a.steps + k0 + pk;
      const uint32_t dst = ring_a + slot * L::kUnit;
      const uint8_t* src = a.packed + unit * 1024 + lane * 16;
      cp_async16(dst + lane * 16, src);
      cp_async16(dst + 512 + lane * 16, src + 512);
      if (lane < 8 * P) cp_async4(dst + 1024 + lane * 4, a.scales + unit * (8 * P) + lane);
      if (ZERO && lane < P) cp_async8(dst + 1024 + L::kScaleB + lane * 8, a.zeros + unit * (8 * P) + lane * 8);
      if (++pk == ks) pk = 0, ++ptile;
    }
    ++pu;
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int d = 0; d < kDepth; ++d) fetch(d);

  // x, 16-bit, [row][the CTA's columns]
  {
    const int runs = ks * 16;
    for (int i = threadIdx.x; i < a.M * runs; i += kVecWarps * 32) {
      const int m = i / runs, c = i - m * runs;
      *reinterpret_cast<uint4*>(xs + m * pitch + c * 16) = x_run<T, MX8>(a, m, k0 * 128 + c * 8);
    }
  }
  if (S > 1)
    cluster_sync();  // and the peers have started: their shared memory may be written
  else
    __syncthreads();

  // a finished tile of this CTA's columns
  auto emit = [&](int tile, const float (&acc)[NT][4]) {
    if (S == 1) {
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) store_sum(a, tile, g + (j >> 1) * 8, 8 * i + 2 * t + (j & 1), acc[i][j]);
    } else {
      const int local = tile - t0;
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        const uint32_t dst = map_shared_rank(smem_u32(recv + ((local / S * S + rank) * NT + i) * 32 + lane), local % S);
        asm volatile("st.shared::cluster.v4.f32 [%0], {%1,%2,%3,%4};" ::"r"(dst), "f"(acc[i][0]), "f"(acc[i][1]),
                     "f"(acc[i][2]), "f"(acc[i][3])
                     : "memory");
      }
    }
  };

  float acc[NT][4];
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = 0.f;
  int tile = t0 + (ks > 0 ? u0 / ks : 0), k = ks > 0 ? u0 % ks : 0;
  bool head = k != 0;  // the tile was started by the warp before
  const uint32_t xa = smem_u32(xs) + g * pitch + t * 16;
  const bool row_in[2] = {g < a.M, 8 + g < a.M};
  int slot = 0;
  for (int u = u0; u < u1; ++u) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kDepth - 1) : "memory");
    __syncwarp();
    const uint32_t src = ring_a + slot * L::kUnit;
    uint4 w[2];
    w[0] = lds128(src + lane * 16);
    w[1] = lds128(src + 512 + lane * 16);
    uint32_t sc[P], zz[P];
#pragma unroll
    for (int p = 0; p < P; ++p) {
      sc[p] = lds32(src + 1024 + (8 * p + g) * 4);
      zz[p] = ZERO ? lds8(src + 1024 + L::kScaleB + 8 * p + g) : 0x88u;
    }
    __syncwarp();  // every lane has read the slot
    fetch(slot);
    slot = slot + 1 == kDepth ? 0 : slot + 1;
    uint4 xv[NT][4];
    const uint32_t xk = xa + k * 256;
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        xv[i][q] = row_in[i] ? lds128(xk + i * 8 * pitch + q * 64) : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const uint32_t z0 = Num<T>::offset(zz[p] & 15u), z1 = Num<T>::offset(zz[p] >> 4);
      float part[NT][4];
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) part[i][j] = 0.f;
#pragma unroll
      for (int j = p * 8 / P; j < (p + 1) * 8 / P; ++j) {
        const uint4 wv = w[j >> 2];
        const uint32_t word = (j & 3) == 0 ? wv.x : (j & 3) == 1 ? wv.y : (j & 3) == 2 ? wv.z : wv.w;
        uint32_t f[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          f[i] = Num<T>::sub(((word >> (4 * i)) & 0x000F000Fu) | Num<T>::kMagic, (i & 1) ? z1 : z0);
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          const uint4 v = xv[i][j >> 1];
          Num<T>::mma(part[i], f, (j & 1) ? v.z : v.x, (j & 1) ? v.w : v.y);
        }
      }
      const float s0 = half_bits_to_f32(sc[p] & 0xFFFFu, a.scale_half), s1 = half_bits_to_f32(sc[p] >> 16, a.scale_half);
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        acc[i][0] += part[i][0] * s0, acc[i][1] += part[i][1] * s0;
        acc[i][2] += part[i][2] * s1, acc[i][3] += part[i][3] * s1;
      }
    }
    if (++k == ks || u + 1 == u1) {
      if (!head && k == ks) {
        emit(tile, acc);
      } else {
        float4* dst = park + (warp * 2 + (head ? 0 : 1)) * NT * 32 + lane;
#pragma unroll
        for (int i = 0; i < NT; ++i) dst[i * 32] = make_float4(acc[i][0], acc[i][1], acc[i][2], acc[i][3]);
      }
      head = false;
      ++tile;
      k = 0;
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = 0.f;
    }
  }
  __syncthreads();
  // the tile that this warp started and did not finish: its own part, then the heads of the warps after it
  if (u1 > u0) {
    const int last = (u1 - 1) / ks;                         // tile of the last unit, from t0
    const int64_t end = static_cast<int64_t>(last + 1) * ks;  // one past the tile's units
    if (end > u1 && static_cast<int64_t>(last) * ks >= u0) {
      float4 sum[NT];
#pragma unroll
      for (int i = 0; i < NT; ++i) sum[i] = park[((warp * 2 + 1) * NT + i) * 32 + lane];
      for (int w = warp + 1; w < kVecWarps; ++w) {
        const int b = static_cast<int>(units * w / kVecWarps), e = static_cast<int>(units * (w + 1) / kVecWarps);
        if (b >= end) break;
        if (e == b) continue;
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          const float4 v = park[(w * 2 * NT + i) * 32 + lane];
          sum[i].x += v.x, sum[i].y += v.y, sum[i].z += v.z, sum[i].w += v.w;
        }
      }
#pragma unroll
      for (int i = 0; i < NT; ++i) acc[i][0] = sum[i].x, acc[i][1] = sum[i].y, acc[i][2] = sum[i].z, acc[i][3] = sum[i].w;
      emit(t0 + last, acc);
    }
  }
  if (S > 1) {
    cluster_sync();
    for (int64_t i = threadIdx.x; i < static_cast<int64_t>(a.recv_slots) * NT * 128; i += kVecWarps * 32) {
      const int e = static_cast<int>(i % 128), nt = static_cast<int>(i / 128 % NT), sl = static_cast<int>(i / (128 * NT));
      const int64_t tl = t0 + static_cast<int64_t>(sl) * S + rank;
      if (tl >= t1) break;
      float v = 0.f;
      for (int r = 0; r < S; ++r) v += reinterpret_cast<const float*>(recv)[((sl * S + r) * NT + nt) * 128 + e];
      const int ln = e >> 2, j = e & 3;
      store_sum(a, tl, (ln >> 2) + (j >> 1) * 8, 8 * nt + 2 * (ln & 3) + (j & 1), v);
    }
  }
}

struct VecPlan {
  int S, clusters, x_bytes, recv_slots, smem;
};

// Per device and kernel: its shared-memory limit raised, and how many clusters of each size fit at once.
template <auto kern>
int resident_clusters(int S) {
  constexpr int kDevices = 64;
  static std::atomic<int> known[kDevices][4];
  int dev = 0;
  cudaGetDevice(&dev);
  const int at = S == 1 ? 0 : S == 2 ? 1 : S == 4 ? 2 : 3;
  int n = dev < kDevices ? known[dev][at].load() : 0;
  if (n > 0) return n;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem);
  if (e != cudaSuccess) throw std::runtime_error(std::string("minisgl.int4_linear: ") + cudaGetErrorString(e));
  if (S == 1) {
    cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
  } else {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(S);
    cfg.blockDim = dim3(kVecWarps * 32);
    cfg.dynamicSmemBytes = kMaxSmem;
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

// The cluster size whose busiest CTA has the least to stream: whole tiles
// are dealt to clusters, so many tiles balance alone (S = 1) and few tiles only
// when their columns are shared. A cluster's two barriers and exchange cost
// about as much as kClusterCost units. False: x does not fit shared memory.
constexpr int kClusterCost = 30;
template <int G, auto kern>
bool vec_plan(int NT, const VecArgs& a, VecPlan& best) {
  int64_t best_cost = -1;
  for (int S = 1; S <= 8; S *= 2) {
    if (S > a.steps) break;
    VecPlan p;
    p.S = S;
    p.clusters = std::min(resident_clusters<kern>(S), a.tiles);
    const int per = (a.tiles + p.clusters - 1) / p.clusters, ks = (a.steps + S - 1) / S;
    if (static_cast<int64_t>(a.M) * vec_x_pitch(ks) > kMaxSmem) continue;
    p.x_bytes = a.M * vec_x_pitch(ks);
    p.recv_slots = S > 1 ? (per + S - 1) / S : 0;
    if (p.recv_slots > 4096) continue;
    p.smem = VecSmem<G>::total(NT, p.x_bytes, p.recv_slots, S);
    if (p.smem > kMaxSmem) continue;
    const int64_t cost = static_cast<int64_t>(per) * ks + (S > 1 ? kClusterCost : 0);
    if (best_cost < 0 || cost < best_cost) best_cost = cost, best = p;
  }
  return best_cost >= 0;
}

template <typename T, bool MX8, int NT, int G, bool ZERO>
bool launch_vec(VecArgs a, cudaStream_t s) {
  constexpr auto kern = int4_vec_kernel<T, MX8, NT, G, ZERO>;
  VecPlan p;
  if (!vec_plan<G, kern>(NT, a, p)) return false;
  a.S = p.S;
  a.x_bytes = p.x_bytes;
  a.recv_slots = p.recv_slots;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(p.clusters * p.S));
  cfg.blockDim = dim3(kVecWarps * 32);
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
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, a);
  if (e != cudaSuccess) throw std::runtime_error(std::string("minisgl: kernel launch failed: ") + cudaGetErrorString(e));
  return true;
}

template <typename T, bool MX8, int NT>
bool launch_vec_group(const VecArgs& a, int group, cudaStream_t s) {
  const bool z = a.zeros != nullptr;
  switch (group) {
    case 32: return z ? launch_vec<T, MX8, NT, 32, true>(a, s) : launch_vec<T, MX8, NT, 32, false>(a, s);
    case 64: return z ? launch_vec<T, MX8, NT, 64, true>(a, s) : launch_vec<T, MX8, NT, 64, false>(a, s);
    default: return z ? launch_vec<T, MX8, NT, 128, true>(a, s) : launch_vec<T, MX8, NT, 128, false>(a, s);
  }
}
template <typename T, bool MX8>
bool launch_vec_type(const VecArgs& a, int group, cudaStream_t s) {
  return a.M <= 8 ? launch_vec_group<T, MX8, 1>(a, group, s) : launch_vec_group<T, MX8, 2>(a, group, s);
}

}  // namespace

void launch_int4_linear(const Int4LinearArgs& r, cudaStream_t s) {
  if (r.M <= 0) return;
  if (r.M > 65535 * 32 || r.N > (1ll << 30) || r.K > (1ll << 30))
    throw std::runtime_error("minisgl.int4_linear: size out of range");
  if (r.M <= 16) {
    VecArgs v{};
    v.x = r.x, v.x_scales = r.x_scales, v.packed = r.packed;
    v.scales = static_cast<const uint32_t*>(r.scales), v.zeros = r.zeros, v.bias = r.bias, v.out = r.out;
    v.M = static_cast<int>(r.M), v.N = static_cast<int>(r.N), v.K = static_cast<int>(r.K);
    v.tiles = (v.N + 15) / 16, v.steps = (v.K + 127) / 128;
    v.ldx = r.ldx, v.ld_xs = r.ld_xs, v.ldo = r.ldo;
    v.scale_half = r.scale_type == DType::kF16;
    v.bias_type = static_cast<int>(r.bias_type), v.out_type = static_cast<int>(r.out_type);
    const bool done = r.x_scales != nullptr         ? launch_vec_type<__nv_bfloat16, true>(v, r.group, s)
                      : r.x_type == DType::kF16 ? launch_vec_type<__half, false>(v, r.group, s)
                                                : launch_vec_type<__nv_bfloat16, false>(v, r.group, s);
    if (done) return;
  }
  LinArgs a{};
  a.x = r.x, a.x_scales = r.x_scales, a.packed = r.packed;
  a.scales = static_cast<const uint16_t*>(r.scales), a.zeros = r.zeros, a.bias = r.bias, a.out = r.out;
  a.M = static_cast<int>(r.M), a.N = static_cast<int>(r.N), a.K = static_cast<int>(r.K);
  a.blocks = 2 * ((a.K + 127) / 128);
  a.groups = a.blocks * 64 / r.group;
  a.ldx = r.ldx, a.ld_xs = r.ld_xs, a.ldo = r.ldo;
  a.scale_half = r.scale_type == DType::kF16;
  a.bias_type = static_cast<int>(r.bias_type), a.out_type = static_cast<int>(r.out_type);
  if (r.x_scales != nullptr)
    launch_type<__nv_bfloat16, true>(a, r.group, s);
  else if (r.x_type == DType::kF16)
    launch_type<__half, false>(a, r.group, s);
  else
    launch_type<__nv_bfloat16, false>(a, r.group, s);
}

}  // namespace minisgl
