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

#include <stdexcept>

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
  const uint16_t* sp = a.scales + tile * a.groups * 16 + g;
  const uint8_t* zp = a.zeros != nullptr ? a.zeros + tile * a.groups * 16 + g : nullptr;
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
      const int64_t gi = static_cast<int64_t>(b * 64 / G + p) * 16;
      const float s0 = half_bits_to_f32(sp[gi], a.scale_half), s1 = half_bits_to_f32(sp[gi + 8], a.scale_half);
      const uint32_t z0 = Num<T>::offset(zp != nullptr ? zp[gi] : 8), z1 = Num<T>::offset(zp != nullptr ? zp[gi + 8] : 8);
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

}  // namespace

void launch_int4_linear(const Int4LinearArgs& r, cudaStream_t s) {
  if (r.M <= 0) return;
  if (r.M > 65535 * 32 || r.N > (1ll << 30) || r.K > (1ll << 30))
    throw std::runtime_error("minisgl.int4_linear: size out of range");
  LinArgs a{};
  a.x = r.x, a.x_scales = r.x_scales, a.packed = r.packed;
  a.scales = static_cast<const uint16_t*>(r.scales), a.zeros = r.zeros, a.bias = r.bias, a.out = r.out;
  a.M = static_cast<int>(r.M), a.N = static_cast<int>(r.N), a.K = static_cast<int>(r.K);
  a.blocks = (a.K + 63) / 64;
  a.groups = (a.blocks * 64 + r.group - 1) / r.group;
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
