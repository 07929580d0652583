// Row kernels whose output is MXFP8: residual addition + RMSNorm, and the
// gated activations (SiLU / GELU times the up projection). They stand beside
// the bf16 / fp16 / fp32 forms of elementwise.cu and feed products that take
// 8-bit rows (int4.cu).
//
// MXFP8 rows (OCP microscaling v1.0), scales row-major:
//   q  uint8 [rows, cols]       E4M3 elements
//   sf uint8 [rows, cols / 32]  E8M0: one power of two 2^(byte - 127) per 32 columns
// For a block of values y: byte - 127 is the smallest e >= -126 with
// max |y| <= 448 * 2^e (448 is E4M3's largest), the elements are y / 2^e
// rounded to nearest even; an all-zero block has byte 0 and zero elements; a
// block that holds an infinity, a NaN or a magnitude beyond float32 has byte
// 255 and NaN elements.
//
// The stored bits are those of the formula in exact arithmetic (64 bits):
// y is computed in float32 with a bound on its error, and where a value
// lies closer to a rounding border than that bound (about one element in
// 10^5) it is computed again in double and rounded to odd on the way to
// E4M3, so that the second rounding cannot move it. Results then do not
// depend on how an exponential or a sum of squares is rounded on the way.
#include <cuda_fp8.h>

#include <algorithm>
#include <atomic>
#include <stdexcept>
#include <string>
#include <type_traits>

#include "common.cuh"
#include "launch.h"
#include "ops.h"

namespace minisgl {
namespace {

constexpr int kBlock = 32;  // columns under one scale

// A lane's share of a row is two 16-byte vectors: 16 values of a 16-bit type (two lanes share a scale), 8 of float32
// (four lanes). With one vector a lane the shuffles, the scale and the addresses cost as much as the values.
struct Pair {
  uint4 v[2];
};
template <typename T>
__device__ __forceinline__ Pair load_pair(const T* p) {
  return Pair{{reinterpret_cast<const uint4*>(p)[0], reinterpret_cast<const uint4*>(p)[1]}};
}
template <typename T>
__device__ __forceinline__ void store_pair(T* p, const Pair& r) {
  reinterpret_cast<uint4*>(p)[0] = r.v[0];
  reinterpret_cast<uint4*>(p)[1] = r.v[1];
}
// whole words at a time: a 16-bit value taken out alone costs one more instruction
template <typename T, int V>
__device__ __forceinline__ void unpack(const Pair& raw, float (&v)[V]) {
  static_assert(V * sizeof(T) == 32, "two vectors");
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint4& q = raw.v[i >> 2];
    const uint32_t w = (i & 3) == 0 ? q.x : (i & 3) == 1 ? q.y : (i & 3) == 2 ? q.z : q.w;
    if constexpr (sizeof(T) == 4) {
      v[i] = __uint_as_float(w);
    } else if constexpr (std::is_same_v<T, __half>) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
      v[2 * i] = f.x, v[2 * i + 1] = f.y;
    } else {
      v[2 * i] = __uint_as_float(w << 16), v[2 * i + 1] = __uint_as_float(w & 0xFFFF0000u);
    }
  }
}
// v rounded to T, as stored and as floats again
template <typename T, int V>
__device__ __forceinline__ Pair round_to(float (&v)[V]) {
  Pair r;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    uint32_t w;
    if constexpr (sizeof(T) == 4) {
      w = __float_as_uint(v[i]);
    } else if constexpr (std::is_same_v<T, __half>) {
      const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
      w = *reinterpret_cast<const uint32_t*>(&h);
    } else {
      const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
      w = *reinterpret_cast<const uint32_t*>(&h);
    }
    uint4& q = r.v[i >> 2];
    ((i & 3) == 0 ? q.x : (i & 3) == 1 ? q.y : (i & 3) == 2 ? q.z : q.w) = w;
  }
  unpack<T, V>(r, v);
  return r;
}

// E4M3 bits of a double: truncated to float32 with a sticky last bit
// (round to odd), then rounded to nearest even once.
__device__ __forceinline__ uint32_t e4m3_of(double t) {
  float f = __double2float_rz(t);
  if (static_cast<double>(f) != t) f = __uint_as_float(__float_as_uint(f) | 1u);
  return __nv_cvt_float_to_fp8(f, __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ double pow2(int e) {  // 2^e, |e| <= 1000
  return __longlong_as_double(static_cast<long long>(1023 + e) << 52);
}

// max |.| of three with NaN above everything
__device__ __forceinline__ float max_abs3(float a, float b, float c) {
  float d;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float min3(float a, float b, float c) {
  float d;
  asm("min.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// two products or sums in one instruction
__device__ __forceinline__ float2 mul2(float a, float b, float c, float d) {
  float2 r;
  asm("{\n.reg .b64 v, w;\nmov.b64 v, {%2, %3};\nmov.b64 w, {%4, %5};\nmul.rn.f32x2 v, v, w;\nmov.b64 {%0, %1}, v;\n}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a), "f"(b), "f"(c), "f"(d));
  return r;
}
__device__ __forceinline__ float2 add2(float a, float b, float c, float d) {
  float2 r;
  asm("{\n.reg .b64 v, w;\nmov.b64 v, {%2, %3};\nmov.b64 w, {%4, %5};\nadd.rn.f32x2 v, v, w;\nmov.b64 {%0, %1}, v;\n}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a), "f"(b), "f"(c), "f"(d));
  return r;
}
__device__ __forceinline__ uint32_t e4m3x4(const float* t, float s) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(mul2(t[0], t[1], s, s), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(mul2(t[2], t[3], s, s), __NV_SATFINITE, __NV_E4M3);
  return lo | hi << 16;
}

// The V elements y = v * factor of this lane, quantised. The 32 / V neighbouring lanes
// that share a block call it together with the rest of their warp (`active`
// may differ between blocks, not inside one). `slack`: bound on y's relative
// error in units of 2^-24; bit i of `doubt` marks an element whose error may be
// larger but not twofold, and at most `edge` such units where |y| is above 1e-20 (below, no such element decides a
// scale: those blocks are done in double). An element that float32 cannot tell is NaN: its block is done in double. exact(i): element i in double;
// zero(): whether all of the lane's inputs make zeros (asked only where y is too small for float32).
//
// Rounding is monotonic: where y (1 - slack) and y (1 + slack) round to the
// same E4M3 value, so does the exact one.
template <int V, typename Exact, typename Zero>
__device__ __forceinline__ void mx8_block(const float (&v)[V], float factor, uint32_t slack, uint32_t edge, uint32_t doubt,
                                          Exact exact, Zero zero, uint8_t* q, uint8_t* sf, bool active) {
  constexpr int G = kBlock / V;  // lanes of a block
  const int lane = threadIdx.x & 31;
  float top_v = max_abs3(v[0], v[1], v[2]);
#pragma unroll
  for (int i = 3; i < V; i += 2) top_v = max_abs3(top_v, v[i], v[i + 1 < V ? i + 1 : i]);
  uint32_t mv = __float_as_uint(top_v);  // as bits: NaN above infinity above every number
#pragma unroll
  for (int o = 1; o < G; o <<= 1) mv = max(mv, __shfl_xor_sync(0xffffffffu, mv, o));
  const uint32_t m = __float_as_uint(__uint_as_float(mv) * factor);
  if (!active) return;
  const uint32_t group = ((1u << G) - 1u) << (lane & ~(G - 1));
  uint32_t words[V / 4];
  uint32_t sbyte;
  // magnitudes far inside float32's range (v's down to 2^-118, of which more could not be seen)
  if (m - (64u << 23) < (186u << 23) && mv - (27u << 23) < (220u << 23)) {
    // exponent of the largest, one up where the fraction is above 448's 1.75
    sbyte = ((m + 0x1FFFFFu) >> 23) - 8;
    if ((m & 0x7FFFFFu) + edge - 0x600000u <= 2 * edge) {
      // closer to 1.75 than its error (a fraction has units of 2^-23): what may be the largest, in double
      const float least = __uint_as_float(mv) * (1.f - static_cast<float>(edge) * 2.3841858e-7f);
      double top = 0.0;
#pragma unroll 1
      for (int i = 0; i < V; ++i) {
        float vi = 0.f;
#pragma unroll
        for (int k = 0; k < V; ++k)
          if (k == i) vi = v[k];
        if (fabsf(vi) >= least) top = fmax(top, fabs(exact(i)));
      }
#pragma unroll
      for (int o = 1; o < G; o <<= 1) top = fmax(top, __shfl_xor_sync(group, top, o));
      sbyte = (m >> 23) - 8 + (top > 1.75 * pow2(static_cast<int>(m >> 23) - 127) ? 1 : 0);
    }
    const float inv = factor * __uint_as_float((254u - sbyte) << 23);  // about 448 / top_v: no overflow
    const float eps = static_cast<float>(slack + 2) * 5.9604645e-8f;  // two more: this factor and the products are rounded
    uint32_t apart[V / 4], any = doubt;
#pragma unroll
    for (int w = 0; w < V / 4; ++w) {
      words[w] = e4m3x4(v + 4 * w, inv + inv * eps);
      apart[w] = words[w] ^ e4m3x4(v + 4 * w, inv - inv * eps);
      any |= apart[w];
    }
    if (any != 0) {
      uint32_t near = 0;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        if ((apart[i >> 2] >> (8 * (i & 3)) & 0xFFu) != 0) near |= 1u << i;
        // an element in doubt matters unless it is far below half of the smallest step
        if (fabsf(v[i] * inv) > 0.00048828125f) near |= doubt & (1u << i);
      }
      const double s = pow2(127 - static_cast<int>(sbyte));
#pragma unroll 1
      for (int i = 0; i < V; ++i) {
        if ((near >> i & 1u) == 0) continue;
        const uint32_t b = e4m3_of(exact(i) * s) << (8 * (i & 3)), keep = ~(0xFFu << (8 * (i & 3)));
#pragma unroll
        for (int w = 0; w < V / 4; ++w)
          if (w == (i >> 2)) words[w] = (words[w] & keep) | b;
      }
    }
  } else {
    // the whole block in double
    double top = 0.0;
    bool nan = false;
    const bool zeros = m == 0 && __all_sync(group, zero());
    if (!zeros) {
#pragma unroll 1
      for (int i = 0; i < V; ++i) {
        const double a = fabs(exact(i));
        nan |= !(a <= 3.4028234663852886e38);
        top = fmax(top, a);
      }
#pragma unroll
      for (int o = 1; o < G; o <<= 1) top = fmax(top, __shfl_xor_sync(group, top, o));
      nan = __any_sync(group, nan);
    }
    if (nan) {
      sbyte = 255;
#pragma unroll
      for (int w = 0; w < V / 4; ++w) words[w] = 0x7F7F7F7Fu;
    } else if (top == 0.0) {
      sbyte = 0;
#pragma unroll
      for (int w = 0; w < V / 4; ++w) words[w] = 0;
    } else {
      const long long bits = __double_as_longlong(top);
      int e = static_cast<int>(bits >> 52) - 1023 - 8;  // 448 = 1.75 * 2^8
      if ((bits & 0xFFFFFFFFFFFFFll) > 0xC000000000000ll) ++e;
      e = max(e, -126);
      sbyte = static_cast<uint32_t>(e + 127);
      const double s = pow2(-e);
#pragma unroll
      for (int w = 0; w < V / 4; ++w) words[w] = 0;
#pragma unroll 1
      for (int i = 0; i < V; ++i) {
        const uint32_t b = e4m3_of(exact(i) * s) << (8 * (i & 3));
#pragma unroll
        for (int w = 0; w < V / 4; ++w)
          if (w == (i >> 2)) words[w] |= b;
      }
    }
  }
  if constexpr (V == 16) {
    *reinterpret_cast<uint4*>(q) = make_uint4(words[0], words[1], words[2], words[3]);
  } else {
    *reinterpret_cast<uint2*>(q) = make_uint2(words[0], words[1]);
  }
  if ((lane & (G - 1)) == 0) *sf = static_cast<uint8_t>(sbyte);
}

// --------------------------------------------------------------- RMSNorm ----
struct NormArgs {
  const void* x;
  const void* res;   // nullptr: no residual
  void* res_out;
  const void* w;     // nullptr: no weight
  uint8_t* q;
  uint8_t* sf;
  int cols;
  int64_t ld_x, ld_res, ld_res_out, ld_q, ld_sf;
  double eps, inv_cols;
  int64_t rows;
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

// A CTA walks rows; a row stays in registers between its two passes, and the next one is on its way to shared memory
// meanwhile: each warp copies what it will read itself, so that only its own copies' arrival is waited for. Held in
// registers (two vectors a lane, so that each load takes half sectors) the row ahead cost the occupancy that hides the
// barrier and the conversions: B200, 8192 x 7168 bf16 with residual 98 us, now 73 (5.7 TB/s, 87% of a copy's rate); two
// rows ahead cost it again (83). Short rows are bound by the instructions, some 30 an element (72% of the issue slots):
// 8192 x 2048 without residual 18.4 us, 2.8 TB/s. The sum of squares is held in double: the squares of 16-bit inputs are
// exact there, so the statistic is exact but for the final additions.
template <typename T, int NP, int THREADS>
__global__ void __launch_bounds__(THREADS) rmsnorm_mx8_kernel(const NormArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  constexpr int V = 32 / sizeof(T);
  extern __shared__ __align__(16) uint4 ahead[];  // [x, residual][NP][warp][64]
  __shared__ double red[2][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nw = blockDim.x >> 5;
  const bool has_res = a.res != nullptr, has_w = a.w != nullptr;
  const int tensor = NP * 2 * blockDim.x;
  // A warp's 64 vectors of a part are copied in memory's order (an instruction takes whole sectors) and read in pairs:
  // the lowest bit of a vector's place is flipped in every other 8, so that eight lanes' reads meet 8 banks of 16 bytes.
  auto load = [&](int64_t row) {
    if (row < a.rows) {
      const T* x = static_cast<const T*>(a.x) + row * a.ld_x;
      const T* res = static_cast<const T*>(a.res) + row * a.ld_res;
      const uint32_t dst = smem_u32(ahead + warp * 64 + (lane ^ (lane >> 3 & 1)));
#pragma unroll
      for (int k = 0; k < NP; ++k) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int at = 2 * k * blockDim.x + h * 32, c = (at + warp * 64 + lane) * (V / 2);
          if (c < a.cols) {
            cp_async16(dst + at * 16, x + c);
            if (has_res) cp_async16(dst + (tensor + at) * 16, res + c);
          }
        }
      }
    }
  };
  load(blockIdx.x);
  int turn = 0;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, turn ^= 1) {
    T* res_out = static_cast<T*>(a.res_out) + row * a.ld_res_out;
    Pair raw[NP];  // what is normalised, in its type
    double part[4] = {0.0, 0.0, 0.0, 0.0};  // four short chains
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncwarp();
    const uint4* mine = ahead + warp * 64 + 2 * lane;
    const int flip = lane >> 2 & 1;
#pragma unroll
    for (int k = 0; k < NP; ++k) {
      const int c = (k * blockDim.x + threadIdx.x) * V;
      if (c < a.cols) {
        float v[V];
        raw[k] = Pair{{mine[2 * k * blockDim.x + flip], mine[2 * k * blockDim.x + 1 - flip]}};
        unpack<T, V>(raw[k], v);
        if (has_res) {
          float r[V];
          unpack<T, V>(Pair{{mine[tensor + 2 * k * blockDim.x + flip], mine[tensor + 2 * k * blockDim.x + 1 - flip]}}, r);
          // the residual stream is kept in the activation's type: the sum is rounded before it is normalised
#pragma unroll
          for (int i = 0; i < V; i += 2) {
            const float2 t = add2(v[i], v[i + 1], r[i], r[i + 1]);
            v[i] = t.x, v[i + 1] = t.y;
          }
          raw[k] = round_to<T, V>(v);
          store_pair(res_out + c, raw[k]);
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const double d = v[i];
          part[i & 3] = fma(d, d, part[i & 3]);
        }
      }
    }
    double ss = (part[0] + part[1]) + (part[2] + part[3]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    // the two halves of red alternate: a warp that writes one again has passed the barrier after everybody read it
    if (lane == 0) red[turn][warp] = ss;
    __syncthreads();
    load(row + gridDim.x);  // every read of this row's copy lies before the barrier
    ss = red[turn][0];  // the same order in every thread
    for (int w = 1; w < nw; ++w) ss += red[turn][w];
    // 1 / sqrt: two Newton steps in double on the float32 estimate leave some units of 2^-53
    const double mean = ss * a.inv_cols + a.eps;
    double inv_d;
    if (mean > 1e-30 && mean < 1e30) {
      inv_d = rsqrtf(static_cast<float>(mean));
      const double half = 0.5 * mean;
      inv_d = fma(inv_d, fma(-half * inv_d, inv_d, 0.5), inv_d);
      inv_d = fma(inv_d, fma(-half * inv_d, inv_d, 0.5), inv_d);
    } else {
      inv_d = 1.0 / sqrt(mean);
    }
    // a row whose factor is at the ends of float32's range is computed in double as a whole (NaN sends it there)
    const bool tame = inv_d > 1e-30 && inv_d < 1e30;
    const float inv = tame ? static_cast<float>(inv_d) : __uint_as_float(0x7FC00000u);
#pragma unroll
    for (int k = 0; k < NP; ++k) {
      const int c = (k * blockDim.x + threadIdx.x) * V;
      const bool active = c < a.cols;
      float v[V];
      if (active) {
        unpack<T, V>(raw[k], v);
        if (has_w) {  // exact for 16-bit types
          float w[V];
          unpack<T, V>(load_pair(static_cast<const T*>(a.w) + c), w);
#pragma unroll
          for (int i = 0; i < V; i += 2) {
            const float2 t = mul2(v[i], v[i + 1], w[i], w[i + 1]);
            v[i] = t.x, v[i + 1] = t.y;
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = 0.f;
      }
      const T* src = (has_res ? res_out : static_cast<const T*>(a.x) + row * a.ld_x) + c;  // the normalised row's input, as stored
      const T* wc = static_cast<const T*>(a.w) + c;
      mx8_block<V>(
          v, inv, 3u, 4u, 0u,  // two roundings, inv and v w, with room for the bounds' own; for the scale their product
          [=](int i) {
            const double d = static_cast<double>(to_f32<T>(src[i])) * inv_d;
            return has_w ? d * static_cast<double>(to_f32<T>(wc[i])) : d;
          },
          [=]() {
            bool z = true;
#pragma unroll 1
            for (int i = 0; i < V; ++i) z &= to_f32<T>(src[i]) == 0.f;
            return z;
          },
          a.q + row * a.ld_q + c, a.sf + row * a.ld_sf + c / kBlock, active);
    }
  }
}

// ------------------------------------------------------ gated activation ----
struct ActArgs {
  const void* x;  // [rows, 2 d], row stride ld_x
  uint8_t* q;
  uint8_t* sf;
  int64_t rows, ld_x, ld_q, ld_sf;
  int d;
  int interleaved;  // gate|up in alternating blocks of 64 columns
};

// exact forms, in double
template <int ACT>
__device__ __noinline__ double act_exact(double g, double u) {
  if (ACT == 0) return g / (1.0 + exp(-g)) * u;
  return 0.5 * g * erfc(-g * 0.70710678118654752440) * u;
}

__device__ __forceinline__ float rcp_approx(float x) {  // 1 unit of the last place
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float ex2_approx(float x) {  // 2 units
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// P(X < -a) of a standard normal X, a >= 0: e^(-a^2 / 2) times a polynomial in t = 1 / (1 + a / 4), fitted to
// erfcx(a / sqrt 2) / 2 on [0, 13.4] by iteratively reweighted least squares (relative error 2^-26). a^2 and its
// product with log2(e) / 2 are carried with their rounding errors, which e^-85 would magnify. Compared with double
// for every float32 a up to 12.5: at most 9.5 * 2^-24 off.
__device__ __forceinline__ float normal_tail(float a) {
  const float t = rcp_approx(fmaf(a, 0.25f, 1.f));
  float r = 3.4584614e-2f;
  r = fmaf(r, t, -1.9962448e-1f);
  r = fmaf(r, t, 4.0307708e-1f);
  r = fmaf(r, t, -3.4421673e-1f);
  r = fmaf(r, t, 3.1342766e-1f);
  r = fmaf(r, t, -2.5198551e-2f);
  r = fmaf(r, t, 1.2324397e-1f);
  r = fmaf(r, t, 9.4456886e-2f);
  r = fmaf(r, t, 1.0027349e-1f);
  r = fmaf(r, t, -2.3943172e-5f);
  constexpr float kHi = -0.72134752f, kLo = -0.72134752044448170 - static_cast<double>(kHi);
  const float a2 = a * a, e = a2 * kHi;
  const float low = fmaf(a2, kLo, fmaf(fmaf(a, a, -a2), kHi, fmaf(a2, kHi, -e)));  // of the exponent
  return r * fmaf(ex2_approx(e), low * 0.69314718f, ex2_approx(e));
}

// A CTA takes a part of a row at a time, and the loads of its next row are on their way while it works; as many CTAs
// as fit the SMs. B200: SiLU of 4096 x 25600 bf16 90 us (5.9 TB/s, 90% of a copy's rate), of 2048 x 12288 float32
// 35 us (6.5 TB/s): memory. GELU of 2048 x 12288 fp16 34 us (3.7 TB/s) is bound by its instructions, some 40 an element
// at two CTAs to an SM; held to three, its registers spill (37 us). 64 x 25600 4.4 us: launch and one row's latency.
template <typename T, int ACT>
__global__ void __launch_bounds__(256) act_mx8_kernel(const ActArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  constexpr int V = 32 / sizeof(T);
  const int c0 = (blockIdx.x * blockDim.x + threadIdx.x) * V;
  const bool active = c0 < a.d;  // the same for the lanes of a block: d is a multiple of 32
  const int c = active ? c0 : 0;
  const T* gp = static_cast<const T*>(a.x) + blockIdx.y * a.ld_x + (a.interleaved ? (c / 64) * 128 + c % 64 : c);
  const int to_up = a.interleaved ? 64 : a.d;
  const int64_t step = gridDim.y * a.ld_x;
  Pair next_g = load_pair(gp), next_u = load_pair(gp + to_up);
  uint8_t* q = a.q + blockIdx.y * a.ld_q + c;
  uint8_t* sf = a.sf + blockIdx.y * a.ld_sf + c / kBlock;
  const int64_t step_q = gridDim.y * a.ld_q, step_sf = gridDim.y * a.ld_sf;
  const int rows = static_cast<int>(a.rows), rows_step = static_cast<int>(gridDim.y);
  for (int r = blockIdx.y; r < rows; r += rows_step, gp += step, q += step_q, sf += step_sf) {
    float g[V], u[V], y[V];
    unpack<T, V>(next_g, g);
    unpack<T, V>(next_u, u);
    const T* up = gp + to_up;
    if (r < rows - rows_step) {
      next_g = load_pair(gp + step);
      next_u = load_pair(up + step);
    }
    constexpr float kTail = ACT == 0 ? -16.f : -12.5f;
    float low = g[0];
#pragma unroll
    for (int k = 1; k < V; k += 2) low = min3(low, g[k], g[k + 1 < V ? k + 1 : k]);
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const float p = g[k] * u[k];  // exact for 16-bit types
      if (ACT == 0)
        // p / (1 + e^-g): for g >= -16 the exponential's argument (16 * 2^-24) and value, the sum, the reciprocal
        // and the products leave at most 26 * 2^-24
        y[k] = p * rcp_approx(1.f + ex2_approx(-1.44269504f * g[k]));
      else {
        // with the tail's error, the difference's and the product's: at most 13 * 2^-24 for g >= -12.5
        const float h = normal_tail(fabsf(g[k]));
        y[k] = p * (g[k] < 0.f ? h : 1.f - h);
      }
    }
    uint32_t doubt = 0;
    if (low < kTail) {
      // the tail; where e^g leaves float32 only a vast product could matter beside a block's ordinary values
#pragma unroll
      for (int k = 0; k < V; ++k) {
        if (g[k] < kTail) {
          doubt |= 1u << k;
          if (fabsf(g[k] * u[k]) > 1e12f) y[k] = __uint_as_float(0x7FC00000u);
        }
      }
    }
    mx8_block<V>(
        // edge: SiLU's exponent of up to 128 is off by 2^-17 and its value by 180 * 2^-24 in the tail, until y < 1e-20
        y, 1.f, ACT == 0 ? 32u : 16u, ACT == 0 ? 256u : 16u, doubt,
        [=](int k) { return act_exact<ACT>(to_f32<T>(gp[k]), to_f32<T>(up[k])); },
        [=]() {
          bool z = true;
#pragma unroll 1
          for (int k = 0; k < V; ++k) z &= to_f32<T>(gp[k]) == 0.f || to_f32<T>(up[k]) == 0.f;
          return z;
        },
        q, sf, active);
  }
}

template <typename F>
void by_dtype(DType dt, F&& f) {
  switch (dt) {
    case DType::kBF16: f(__nv_bfloat16{}); break;
    case DType::kF16: f(__half{}); break;
    default: f(float{}); break;
  }
}

// CTAs of so many threads and bytes of shared memory that fit the SMs at once
template <auto kern>
int64_t resident_ctas(int threads, int smem, bool residual) {
  constexpr int kDevices = 64;
  static std::atomic<int> fit[kDevices][33][2];  // of an SM
  int dev = 0;
  cudaGetDevice(&dev);
  int n = dev < kDevices ? fit[dev][threads / 32][residual].load() : 0;
  if (n == 0) {
    if (smem > 0) {
      const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024);
      if (e != cudaSuccess) throw std::runtime_error(std::string("minisgl.rmsnorm_mx8: ") + cudaGetErrorString(e));
    }
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kern, threads, smem) != cudaSuccess || n < 1) n = 1;
    if (dev < kDevices) fit[dev][threads / 32][residual].store(n);
  }
  return 148 * n;
}

// each CTA walks its rows
template <typename T, int NP, int THREADS>
void launch_norm(const NormArgs& a, int pairs, cudaStream_t s) {
  constexpr auto kern = rmsnorm_mx8_kernel<T, NP, THREADS>;
  const bool residual = a.res != nullptr;
  const int threads = (pairs + NP * 32 - 1) / (NP * 32) * 32, smem = threads * NP * 32 * (residual ? 2 : 1);
  const int64_t ctas = std::min<int64_t>(a.rows, resident_ctas<kern>(threads, smem, residual));
  launch_pdl(kern, dim3(static_cast<unsigned>(ctas)), dim3(threads), smem, s, a);
}

// CTAs of up to 256 threads for each part of the columns, which share its rows
template <auto kern, int V>
void launch_act(const ActArgs& a, cudaStream_t s) {
  const int lanes = a.d / V, threads = std::min(256, (lanes + 31) / 32 * 32);
  const int64_t parts = (lanes + threads - 1) / threads;
  const int64_t walkers = std::min<int64_t>({a.rows, std::max<int64_t>(1, resident_ctas<kern>(threads, 0, false) / parts), 65535});
  launch_pdl(kern, dim3(static_cast<unsigned>(parts), static_cast<unsigned>(walkers)), dim3(threads), 0, s, a);
}

}  // namespace

void launch_rmsnorm_mx8(const RmsnormMx8Args& r, cudaStream_t s) {
  if (r.rows <= 0) return;
  by_dtype(r.dtype, [&](auto tag) {
    using T = decltype(tag);
    constexpr int V = 32 / sizeof(T);
    const int pairs = r.cols / V;
    if (r.cols % kBlock != 0 || pairs > 2 * 1024) throw std::runtime_error("minisgl.rmsnorm_mx8: unsupported width");
    const NormArgs a{r.x, r.residual, r.residual_out, r.w, r.q, r.sf, r.cols, r.ld_x, r.ld_res, r.ld_res_out,
                     r.ld_q, r.ld_sf, r.eps, 1.0 / r.cols, r.rows};
    // One pair a thread: shorter chains (B200, bf16 with residual: 1 x 5120 2.8 us against 3.6 with two pairs,
    // 2048 x 5120 16.1 against 17.4). Two: many rows whose CTAs of one pair a thread leave an SM's registers unused
    // (8192 x 7168 73.0 against 77.2), and wide ones (4096 x 16384 82 against 100).
    if (pairs <= 384 || (pairs <= 512 && r.rows <= 2 * 148))
      launch_norm<T, 1, 512>(a, pairs, s);
    else
      launch_norm<T, 2, 1024>(a, pairs, s);
  });
}

void launch_act_mx8(const ActMx8Args& r, cudaStream_t s) {
  if (r.rows <= 0) return;
  by_dtype(r.dtype, [&](auto tag) {
    using T = decltype(tag);
    if (r.d % kBlock != 0) throw std::runtime_error("minisgl.act_mx8: width must be a multiple of 32");
    if (r.interleaved && r.d % 64 != 0)
      throw std::runtime_error("minisgl.act_mx8: interleaved width must be a multiple of 64");
    const ActArgs a{r.x, r.q, r.sf, r.rows, r.ld_x, r.ld_q, r.ld_sf, r.d, r.interleaved ? 1 : 0};
    if (r.act == 0)
      launch_act<act_mx8_kernel<T, 0>, 32 / sizeof(T)>(a, s);
    else
      launch_act<act_mx8_kernel<T, 1>, 32 / sizeof(T)>(a, s);
  });
}

}  // namespace minisgl
