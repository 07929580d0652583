// Products of many rows with 4-bit weights under group scales (int4.cu has
// few rows): out[m, n] = sum_k x[m, k] W[n, k] (+ bias[n]) on the 5th-generation
// tensor cores. Weight layout: minisgl/quant/int4.py.
//
// One persistent CTA per SM walks tiles of 128 weight rows x BN rows of x
// (weights are the 128-row first operand, so that the 4-bit side is unpacked
// as rarely as possible: once per BN rows of x). Per step of 128 columns eight
// converter warps turn 128 x 128 codes into bf16 (fp16) values in tensor
// memory, where the MMAs take their first operand from: shared memory, whose
// bandwidth bounds the large tiles (x is written and read there once per step),
// sees nothing of the unpacked weights. The sums stay in tensor memory; four
// epilogue warps store them.
//
//   warp 0      x by TMA, a ring of kXs steps
//   warp 1      issues the MMAs
//   warp 2      codes by TMA, a ring of kPs steps (8 KB)
//   warps 4-7   epilogue (tensor-memory lanes 32 (w % 4) ..)
//   warps 8-23  two sets of converters, which take the steps in turn; a warp has 32 rows x 64 columns of a step
//
// W = (c - z) s is rounded once to bf16 (fp16): the one rounding besides those
// of the float32 sums. fp16 weights are formed under each row's own power of
// two, which puts the row's largest scale into [2^11, 2^12): 15 of it fit fp16,
// and scales down to 2^-25 of it stay normal (smaller ones lose bits).
//
// Few tiles (N small, M small): S CTAs of a cluster share a tile's columns and
// add their sums through shared memory in rank order.
//
// Measured (B200, bf16, groups of 128): 2000 x 8192 x 7168 187 to 193 us (1.22 to
// 1.26 PFLOP/s; 212 where power holds the clock down, as it does a library
// product: 1.38 of 1.63 PFLOP/s), 512 x 8192 x 7168 49, 128 x 8192 x 7168 22.5,
// 24 x 7168 x 8192 (groups of 64, MXFP8 rows) 19.6. Large tiles are bound by x on
// its way from L2 and by power. Small ones take some 730 cycles a step, most of
// them in the converters (two thirds of the 2200 instructions a step of 16384
// codes); the SM issues 2.0 of the 4 instructions a cycle that it can, so latency
// between them counts more than their number. More steps in tensor memory or a
// third set of converters measured no better.
//
// Every wait is bounded: a timeout records an error, raises an abort flag that
// the other roles check, and the CTA drains its copies and returns.
#include <cuda_fp8.h>

#include <algorithm>
#include <atomic>
#include <stdexcept>
#include <string>
#include <type_traits>

#include "common.cuh"
#include "launch.h"
#include "ops.h"
#include "tma_host.h"

namespace minisgl {
namespace {

constexpr int kRows = 128;       // weight rows of a tile
constexpr int kConverters = 8;
constexpr int kACols = 64;       // tensor-memory columns of one step of weights: 128 values of 16 bits a row
constexpr int kCodes = 8 * 1024;  // 128 rows x 128 columns

template <int BN>
struct GSmem {
  static constexpr int kX = BN * 256;  // one step of x, as two 64-column tiles
  // 192 rows: 3 steps of x and 4 of codes 193 us at 2000 x 8192 x 7168 and 384 at 1536 x 5120 x 25600 (B200), 4 and 2 191
  // and 398
  static constexpr int kXs = BN >= 128 ? 3 : 6;
  static constexpr int kPs = BN == 256 ? 2 : BN == 192 ? 4 : 6;
  static constexpr int kAs = BN == 192 ? 2 : BN == 32 ? 3 : 4;  // steps of weights in tensor memory
  // Converter sets of 8 warps, which take the steps in turn. A wait by parity is sure only for a waiter that knows the
  // phase before the awaited one to have ended: while that is open it passes too. So each slot of codes belongs to one
  // set, which has then waited for every earlier fill of it (copies may land in any order; with three slots a set could
  // read one whose last but one fill, the other set's, was still on its way). Slots in tensor memory change sets, but
  // MMAs end in order, and the set's step before waited for step n - kAs - kSets, which is no earlier than n - 2 kAs.
  // Three sets were no faster than two.
  static constexpr int kSets = 2;
  static_assert(kPs % kSets == 0 && kSets <= kAs, "turns");
  static constexpr int kThreads = 256 + kSets * 256;
  static constexpr int kAcc = BN == 256 ? 1 : 2;  // sums in tensor memory; 256 columns leave room for one (one tile a CTA)
  static constexpr int kPt = kXs * kX;
  static constexpr int kSt = kPt + kPs * kCodes;   // the steps' scales, 1 KB apart
  static constexpr int kZt = kSt + kPs * 1024;     // and zero points, 256 bytes apart
  static constexpr int kOut = kZt + kPs * 256;
  static constexpr int kRing = kOut + 4 * 1024;  // the epilogue's 1 KB a warp
  static constexpr int kBars = 8 * (2 * kXs + 2 * kPs + 2 * kAs + 4) + 16;
  static constexpr int bytes(int S) { return 1024 + kRing + (kBars + 127) / 128 * 128 + (S > 1 ? kRows * BN * 4 : 0); }
  static_assert(bytes(BN <= 128 ? 2 : 1) <= 227 * 1024, "shared memory");
  static constexpr uint32_t kCols = BN == 32 ? 256 : 512;
  static_assert(kAcc * BN + kAs * kACols <= kCols, "tensor memory");
};

struct GArgs {
  const uint8_t* packed;
  const uint8_t* zeros;  // nullptr: 8 everywhere
  const float* row_pow;  // fp16: power of two taken out of a row's scales
  const void* bias;
  void* out;
  int M, N, steps, tiles16;
  int m_tiles, n_tiles, S;
  int vec_out;   // 16-bit outputs whose rows lie at multiples of 16 bytes, N % 8 == 0
  int x_blocks;  // x by 64-column blocks (K % 64 == 0): one copy a step
  int64_t ldo;
  int scale_half, bias_type, out_type;
  ErrorSink err;
};

__device__ __forceinline__ float scale_f32(uint32_t bits, int is_half) {
  return is_half ? __half2float(__ushort_as_half(static_cast<unsigned short>(bits))) : __uint_as_float(bits << 16);
}
__device__ __forceinline__ float any_f32(const void* p, int64_t i, int type) {
  if (type == static_cast<int>(DType::kF32)) return static_cast<const float*>(p)[i];
  if (type == static_cast<int>(DType::kF16)) return __half2float(static_cast<const __half*>(p)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}
__device__ __forceinline__ void store_any(void* p, int64_t i, int type, float v) {
  if (type == static_cast<int>(DType::kF32))
    static_cast<float*>(p)[i] = v;
  else if (type == static_cast<int>(DType::kF16))
    static_cast<__half*>(p)[i] = __float2half_rn(v);
  else
    static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}

// 16 rows x 64 values of 16 bits (32 columns) of tensor memory: lane 4 g + t holds of each 8 columns (16 values)
// columns 2 t, 2 t + 1 of row g, then of row g + 8
__device__ __forceinline__ void tmem_st_16x256b_x4(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.16x256b.x4.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

// One thread of a converged warp. The asynchronous instructions take their operands from uniform registers: under
// an elected predicate the compiler keeps them there, under lane == 0 it moves each operand of each instruction
// over (about 100 cycles an MMA).
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}

// Pairs of 16-bit floats: a code under an exponent, exactly code - zero, times the scale.
template <bool HALF>
struct Pair {
  static constexpr uint32_t kBase = HALF ? 0x64086408u : 0x43084308u;  // 1024 | 8 or 128 | 8: codes are stored as c ^ 8
  __device__ static uint32_t zero(uint32_t z) { return ((HALF ? 0x6400u : 0x4300u) + z) * 0x10001u; }
  __device__ static uint32_t code(uint32_t w) {  // (w & 0x000F000F) ^ base
    uint32_t d;
    asm("lop3.b32 %0, %1, %2, %3, 0x6A;" : "=r"(d) : "r"(w), "r"(0x000F000Fu), "r"(kBase));
    return d;
  }
  __device__ static uint32_t sub(uint32_t a, uint32_t b) {
    uint32_t d;
    if constexpr (HALF)
      asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    else
      asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
  }
  __device__ static uint32_t mul(uint32_t a, uint32_t b) {
    uint32_t d;
    if constexpr (HALF)
      asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    else
      asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
  }
};

template <int BN, int G, bool HALF>
__global__ void __launch_bounds__(GSmem<BN>::kThreads, 1)
    int4_gemm_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_s,
                     const __grid_constant__ CUtensorMap tm_z, const __grid_constant__ CUtensorMap tm_x, const GArgs a) {
  using L = GSmem<BN>;
  constexpr int P = 128 / G, kSets = L::kSets;
  constexpr int kZeroRow = P == 1 ? 16 : 8 * P, kZeroB = 8 * kZeroRow;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint64_t* xfull = reinterpret_cast<uint64_t*>(smem + L::kRing);
  uint64_t* xempty = xfull + L::kXs;
  uint64_t* pfull = xempty + L::kXs;
  uint64_t* pempty = pfull + L::kPs;
  uint64_t* afull = pempty + L::kPs;
  uint64_t* aempty = afull + L::kAs;
  uint64_t* acc_full = aempty + L::kAs;  // [2]
  uint64_t* acc_empty = acc_full + 2;  // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
  int* s_abort = reinterpret_cast<int*>(tmem_slot + 1);
  float* part = reinterpret_cast<float*>(smem + L::kRing + (L::kBars + 127) / 128 * 128);  // S > 1: [BN][128] sums

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int S = a.S, rank = S > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int first = static_cast<int>(blockIdx.x) / S, stride = static_cast<int>(gridDim.x) / S;
  const int num_tiles = a.m_tiles * a.n_tiles;
  const int k0 = static_cast<int>(static_cast<int64_t>(a.steps) * rank / S);
  const int k1 = static_cast<int>(static_cast<int64_t>(a.steps) * (rank + 1) / S);
  pdl_launch_dependents();
  if (threadIdx.x == 0) {
    for (int s = 0; s < L::kXs; ++s) mbar_init(&xfull[s], 1), mbar_init(&xempty[s], 1);
    for (int s = 0; s < L::kPs; ++s) mbar_init(&pfull[s], 1), mbar_init(&pempty[s], kConverters);
    for (int s = 0; s < L::kAs; ++s) mbar_init(&afull[s], kConverters), mbar_init(&aempty[s], 1);
    for (int i = 0; i < 2; ++i) mbar_init(&acc_full[i], 1), mbar_init(&acc_empty[i], 4);
    *s_abort = 0;
    fence_barrier_init();
    prefetch_tmap(&tm_w);
    prefetch_tmap(&tm_s);
    prefetch_tmap(&tm_x);
  }
  // the first codes, on their way to L2 while the kernel before this one ends (a prefetch carries no value)
  if (warp >= 8 && warp < 16 && first < num_tiles) {
    const int tile16 = first / a.m_tiles * 8 + warp - 8;
    if (tile16 < a.tiles16 && k0 + (lane >> 3) < k1)
      asm volatile("prefetch.global.L2 [%0];" ::"l"(
          a.packed + (static_cast<int64_t>(tile16) * a.steps + k0 + (lane >> 3)) * 1024 + (lane & 7) * 128));
  }
  pdl_wait();
  if (warp == 1) {
    tmem_alloc(tmem_slot, L::kCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  if (S > 1) cluster_sync();  // the peers have started: their shared memory may be written
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  volatile int* abort_flag = s_abort;
  int issued = 0;  // copies this thread has started (warps 0 and 2)

  if (warp == 0) {
    // -------------------------------------------------------------- x ----
    int it = 0;
    bool ok = true;
    for (int tile = first; ok && tile < num_tiles && !*abort_flag; tile += stride) {
      const int m0 = tile % a.m_tiles * BN;
      for (int k = k0; k < k1; ++k, ++it) {
        const int s = it % L::kXs;
        if (it >= L::kXs) ok = __all_sync(0xffffffffu, mbar_wait(&xempty[s], ((it / L::kXs) - 1) & 1, a.err, 421));
        if (!ok) break;
        if (elect_one()) {
          mbar_arrive_expect_tx(&xfull[s], L::kX);
          uint8_t* dst = smem + s * L::kX;
          if (a.x_blocks) {  // both tiles in one copy
            tma_load_3d(dst, &tm_x, &xfull[s], 0, m0, 2 * k);
          } else {
            tma_load_2d(dst, &tm_x, &xfull[s], k * 128, m0);
            tma_load_2d(dst + L::kX / 2, &tm_x, &xfull[s], k * 128 + 64, m0);
          }
        }
        __syncwarp();
        issued = it + 1;
      }
    }
    if (!ok && lane == 0) *abort_flag = 1;
    __syncwarp();
  } else if (warp == 2) {
    // ---------------------------------------------------------- codes ----
    int it = 0;
    bool ok = true;
    for (int tile = first; ok && tile < num_tiles && !*abort_flag; tile += stride) {
      const int t16 = tile / a.m_tiles * 8;
      for (int k = k0; k < k1; ++k, ++it) {
        const int s = it % L::kPs;
        if (it >= L::kPs) ok = __all_sync(0xffffffffu, mbar_wait(&pempty[s], ((it / L::kPs) - 1) & 1, a.err, 422));
        if (!ok) break;
        if (elect_one()) {
          // eight tiles x 1 KB in one copy (eight bulk copies took 130 cycles each to issue)
          mbar_arrive_expect_tx(&pfull[s], kCodes + 256 * P + (a.zeros ? kZeroB : 0));
          tma_load_2d(smem + L::kPt + s * kCodes, &tm_w, &pfull[s], k * 256, t16);
          tma_load_2d(smem + L::kSt + s * 1024, &tm_s, &pfull[s], k * (8 * P), t16);
          // zero points by 16 bytes a tile: with one group a step those of an even step and the next
          if (a.zeros) tma_load_2d(smem + L::kZt + s * 256, &tm_z, &pfull[s], P == 1 ? (k & ~1) * 8 : k * (8 * P), t16);
        }
        __syncwarp();
        issued = it + 1;
      }
    }
    if (!ok && lane == 0) *abort_flag = 1;
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA ----
    // instruction descriptor: float32 sums, 128 x BN, both operands K-major and of one 16-bit type
    constexpr uint32_t idesc = HALF ? make_idesc_bf16(kRows, BN) & ~((1u << 7) | (1u << 10)) : make_idesc_bf16(kRows, BN);
    const uint64_t x_desc = make_sdesc_k_sw128(smem_u32(smem));  // start addresses add up in its low bits
    int it = 0, lt = 0;
    bool ok = true;
    for (int tile = first; ok && tile < num_tiles; tile += stride, ++lt) {
      const int acc = lt % L::kAcc;
      if (lt >= L::kAcc) ok = __all_sync(0xffffffffu, mbar_wait(&acc_empty[acc], (lt / L::kAcc - 1) & 1, a.err, 423));
      if (!ok) break;
      tc_fence_after();
      for (int k = k0; k < k1 && ok; ++k, ++it) {
        const int as = it % L::kAs, xs = it % L::kXs;
        ok = __all_sync(0xffffffffu, mbar_wait(&afull[as], (it / L::kAs) & 1, a.err, 425) &&
                                         mbar_wait(&xfull[xs], (it / L::kXs) & 1, a.err, 424));
        if (!ok) break;
        tc_fence_after();
        const uint32_t d = tmem + acc * BN, wa = tmem + L::kAcc * BN + as * kACols;
        const uint64_t xd = x_desc + static_cast<uint32_t>(xs * L::kX >> 4);
        if (elect_one()) {
#pragma unroll
          for (int q = 0; q < 8; ++q)  // 16 columns: 8 of tensor memory, 32 bytes of a 64-column tile of x
            tc_mma_f16_ta(d, wa + q * 8, xd + static_cast<uint32_t>((q >> 2) * (L::kX / 2) + (q & 3) * 32 >> 4), idesc,
                          k > k0 || q > 0 ? 1u : 0u);
          tc_commit(&xempty[xs]);
          tc_commit(&aempty[as]);
        }
        __syncwarp();
      }
      if (ok && elect_one()) tc_commit(&acc_full[acc]);
      __syncwarp();
    }
    if (!ok && lane == 0) *abort_flag = 1;
    __syncwarp();
  } else if (warp >= 8) {
    // ----------------------------------------------------- converters ----
    // warp q + 4 h of a set: rows 32 q .. 32 q + 31 (the tensor-memory lanes it reaches), columns 64 h .. of a step
    const int set = (warp - 8) / 8, quad = warp & 3, half = (warp >> 2) & 1, g = lane >> 2;
    const uint32_t a_base = tmem + L::kAcc * BN + half * (kACols / 2) + (static_cast<uint32_t>(32 * quad) << 16);
    constexpr int H = P == 4 ? 2 : 1;  // groups of 64 columns
    // own steps lie kSets apart, over the ends of tiles too: slots and phases are carried along
    int ps = set, as = set, turn = set;
    uint32_t ps_phase = 0, as_phase = 1;  // the first use of a slot in tensor memory finds it empty
    const uint32_t codes_at = L::kPt + quad * 2048 + half * 512 + lane * 16;
    const uint32_t scales_at = L::kSt + (2 * quad * P + (P == 1 ? 0 : half * H)) * 32 + g * 4;
    uint32_t zero[2][H][2];  // as the pairs that are subtracted; 8 without zero points
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int p = 0; p < H; ++p) zero[c][p][0] = zero[c][p][1] = Pair<HALF>::zero(8);
    bool ok = true;
    for (int tile = first; ok && tile < num_tiles; tile += stride) {
      float down[2][2];  // 1 / the rows' power of two
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int tile16 = min(tile / a.m_tiles * 8 + 2 * quad + c, a.tiles16 - 1);  // rows past N are never stored
#pragma unroll
        for (int r = 0; r < 2; ++r) down[c][r] = HALF ? 1.f / a.row_pow[tile16 * 16 + g + 8 * r] : 1.f;
      }
      int k = k0 + turn;
      for (; k < k1; k += kSets) {
        if (!__all_sync(0xffffffffu, mbar_try_wait(&pfull[ps], ps_phase)))
          ok = __all_sync(0xffffffffu, mbar_wait(&pfull[ps], ps_phase, a.err, 426));
        if (!ok) break;
        const uint8_t* codes = smem + codes_at + ps * kCodes;
        const uint4 w[2] = {*reinterpret_cast<const uint4*>(codes), *reinterpret_cast<const uint4*>(codes + 1024)};
        uint32_t sc[2][H];
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int p = 0; p < H; ++p)
            sc[c][p] = *reinterpret_cast<const uint32_t*>(smem + scales_at + ps * 1024 + (c * P + p) * 32);
        if (a.zeros != nullptr) {
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int p = 0; p < H; ++p) {
              const uint32_t zz = smem[L::kZt + ps * 256 + (2 * quad + c) * kZeroRow + (P == 1 ? (k & 1) * 8 : (half * H + p) * 8) + g];
              zero[c][p][0] = Pair<HALF>::zero(zz & 15u), zero[c][p][1] = Pair<HALF>::zero(zz >> 4);
            }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&pempty[ps]);  // the codes are in registers
        ps += kSets;
        if (ps >= L::kPs) ps -= L::kPs, ps_phase ^= 1;
        uint32_t o[2][16];  // per tile and word (16 columns): two pairs of row g, two of row g + 8
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const uint32_t words[4] = {w[c].x, w[c].y, w[c].z, w[c].w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t sw = sc[c][j * H / 4];
            uint32_t d[4];
#pragma unroll
            for (int r = 0; r < 4; ++r)  // r: bit 0 the row half, bit 1 the column pair
              d[2 * (r & 1) + (r >> 1)] = Pair<HALF>::sub(Pair<HALF>::code(words[j] >> (4 * r)), zero[c][j * H / 4][r & 1]);
            if (HALF || !a.scale_half) {
              uint32_t s[2];
              if constexpr (HALF) {
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                  const __half q = __float2half_rn(scale_f32(r ? sw >> 16 : sw & 0xFFFFu, a.scale_half) * down[c][r]);
                  s[r] = static_cast<uint32_t>(__half_as_ushort(q)) * 0x10001u;
                }
              } else {
                s[0] = __byte_perm(sw, 0, 0x1010), s[1] = __byte_perm(sw, 0, 0x3232);
              }
#pragma unroll
              for (int i = 0; i < 4; ++i) o[c][4 * j + i] = Pair<HALF>::mul(d[i], s[i >> 1]);
            } else {
              // fp16 scales do not fit bf16: the product is formed in float32 and rounded once
              const float f[2] = {scale_f32(sw & 0xFFFFu, 1), scale_f32(sw >> 16, 1)};
#pragma unroll
              for (int i = 0; i < 4; ++i)
                o[c][4 * j + i] = pack_bf16x2(__uint_as_float(d[i] << 16) * f[i >> 1], __uint_as_float(d[i] & 0xFFFF0000u) * f[i >> 1]);
            }
          }
        }
        // only the store waits for the MMAs that read the slot before
        if (!__all_sync(0xffffffffu, mbar_try_wait(&aempty[as], as_phase)))
          ok = __all_sync(0xffffffffu, mbar_wait(&aempty[as], as_phase, a.err, 427));
        if (!ok) break;
        tc_fence_after();
#pragma unroll
        for (int c = 0; c < 2; ++c)
          tmem_st_16x256b_x4(a_base + as * kACols + (static_cast<uint32_t>(16 * c) << 16), o[c]);
        tc_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&afull[as]);
        as += kSets;
        if (as >= L::kAs) as -= L::kAs, as_phase ^= 1;
      }
      turn = k - k1;  // of the next tile's steps
    }
    if (!ok && lane == 0) *abort_flag = 1;
    __syncwarp();
  } else if (warp >= 4) {
    // ------------------------------------------------------- epilogue ----
    const int quad = warp & 3, row = 32 * quad + lane;
    const uint32_t lane_base = tmem + (static_cast<uint32_t>(32 * quad) << 16);
    int lt = 0;
    bool ok = true;
    for (int tile = first; tile < num_tiles; tile += stride, ++lt) {
      const int acc = lt % L::kAcc;
      ok = __all_sync(0xffffffffu, mbar_wait(&acc_full[acc], (lt / L::kAcc) & 1, a.err, 428));
      if (!ok) break;
      tc_fence_after();
      const int m0 = tile % a.m_tiles * BN;
      const int64_t n = static_cast<int64_t>(tile / a.m_tiles) * kRows + row;
      const bool in = n < a.N;
      const float bias = in && a.bias != nullptr ? any_f32(a.bias, n, a.bias_type) : 0.f;
      const float pow = HALF && in ? a.row_pow[n] : 1.f;
      constexpr int CH = 32;
#pragma unroll 1
      for (int c = 0; c < BN; c += CH) {
        uint32_t r[32];
        tmem_ld_32x32b_x32(lane_base + acc * BN + c, r);
        tc_wait_ld();
        if (c + CH >= BN) {  // the accumulator is read out: the MMAs may reuse it
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&acc_empty[acc]);
        }
        if (S > 1) {
#pragma unroll
          for (int j = 0; j < CH; ++j) part[(c + j) * kRows + row] = __uint_as_float(r[j]);
        } else if (a.vec_out) {
          // 16 rows of x by 32 outputs at a time, turned in shared memory into 16-byte pieces of a row
          uint16_t* turn = reinterpret_cast<uint16_t*>(smem + L::kOut + quad * 1024);
#pragma unroll
          for (int b = 0; b < 32; b += 16) {
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              const float v = __uint_as_float(r[b + j]) * pow + bias;
              turn[j * 32 + lane] = a.out_type == static_cast<int>(DType::kF16) ? __half_as_ushort(__float2half_rn(v))
                                                                               : __bfloat16_as_ushort(__float2bfloat16_rn(v));
            }
            __syncwarp();
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              const int i = q * 32 + lane, m = m0 + c + b + i / 4;
              const int64_t n8 = n - lane + i % 4 * 8;
              if (m < a.M && n8 < a.N)  // N is a multiple of 8 here
                *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + m * a.ldo + n8) =
                    *reinterpret_cast<const uint4*>(turn + i * 8);
            }
            __syncwarp();
          }
        } else if (in) {
          // neighbouring lanes are neighbouring outputs of one row
#pragma unroll
          for (int j = 0; j < CH; ++j)
            if (m0 + c + j < a.M)
              store_any(a.out, static_cast<int64_t>(m0 + c + j) * a.ldo + n, a.out_type, __uint_as_float(r[j]) * pow + bias);
        }
      }
    }
    if (!ok && lane == 0) *abort_flag = 1;
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  if (*abort_flag && lane == 0) {
    // after an abort, let the copies still in flight land (bounded)
    if (warp == 0)
      for (int it = max(0, issued - L::kXs); it < issued; ++it) mbar_wait(&xfull[it % L::kXs], (it / L::kXs) & 1, a.err, 429);
    if (warp == 2)
      for (int it = max(0, issued - L::kPs); it < issued; ++it) mbar_wait(&pfull[it % L::kPs], (it / L::kPs) & 1, a.err, 430);
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, L::kCols);
  }
  if (S > 1) {
    // one tile per cluster: this CTA adds its share of the rows of x, the S partial sums in rank order
    __syncwarp();
    cluster_sync();
    const int x0 = BN * rank / S, x1 = BN * (rank + 1) / S;
    const int64_t n0 = static_cast<int64_t>(first / a.m_tiles) * kRows;
    for (int i = threadIdx.x; i < (x1 - x0) * (kRows / 4); i += L::kThreads) {
      const int at = x0 + i / (kRows / 4), q = i % (kRows / 4) * 4;
      const int m = first % a.m_tiles * BN + at;
      if (m >= a.M) continue;
      const uint32_t local = smem_u32(part + at * kRows + q);
      float v[4] = {0.f, 0.f, 0.f, 0.f};
      for (int r = 0; r < S; ++r) {
        const float4 p = ld_shared_cluster_v4(map_shared_rank(local, r));
        v[0] += p.x, v[1] += p.y, v[2] += p.z, v[3] += p.w;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int64_t n = n0 + q + j;
        if (n >= a.N || *abort_flag) continue;
        if (HALF) v[j] *= a.row_pow[n];
        if (a.bias != nullptr) v[j] += any_f32(a.bias, n, a.bias_type);
        store_any(a.out, static_cast<int64_t>(m) * a.ldo + n, a.out_type, v[j]);
      }
    }
    cluster_sync();  // no CTA leaves while a peer reads its sums
  }
}

// MXFP8 rows as bf16: four significant bits times a power of two are exact down to bf16's smallest subnormal, 2^-133
// (scale bytes of 3 and more; under 0 to 2 the smallest elements are rounded to it)
__global__ void __launch_bounds__(256) mx8_rows_bf16_kernel(uint4* out, const uint8_t* q, const uint8_t* sf, int64_t rows,
                                                          int K, int64_t ldq, int64_t ldsf) {
  pdl_launch_dependents();
  pdl_wait();
  const int runs = K / 8;
  const int64_t total = rows * runs;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int64_t m = i / runs;
    const int c = static_cast<int>(i - m * runs) * 8;
    const uint2 v = *reinterpret_cast<const uint2*>(q + m * ldq + c);
    const uint32_t byte = sf[m * ldsf + c / 32];
    const float s = __uint_as_float(byte == 0 ? 0x00400000u : byte == 255 ? 0x7FC00000u : byte << 23);
    uint32_t r[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(
          static_cast<__nv_fp8x2_storage_t>((j < 2 ? v.x : v.y) >> (16 * (j & 1))), __NV_E4M3);
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
      r[j] = pack_bf16x2(f.x * s, f.y * s);
    }
    out[i] = make_uint4(r[0], r[1], r[2], r[3]);
  }
}

template <auto kern>
int resident(int S, int smem, int threads) {
  constexpr int kDevices = 64;
  static std::atomic<int> known[kDevices][8];
  int dev = 0;
  cudaGetDevice(&dev);
  const int at = S - 1;
  int n = dev < kDevices ? known[dev][at].load() : 0;
  if (n > 0) return n;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024);
  if (e == cudaSuccess && S == 1) {
    e = cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
  } else if (e == cudaSuccess) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(S);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = S;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    e = cudaOccupancyMaxActiveClusters(&n, kern, &cfg);
  }
  if (e != cudaSuccess || n < 1)
    throw std::runtime_error(std::string("minisgl.int4_linear: ") + (e != cudaSuccess ? cudaGetErrorString(e) : "the kernel does not fit this device"));
  if (dev < kDevices) known[dev][at].store(n);
  return n;
}

struct GPlan {
  int bn, S, grid;
  int64_t cost;
};

// The rows of x per tile and the CTAs per tile with the least estimated cycles in the busiest CTA. A step costs what
// its slowest part does: x from L2 (256 BN bytes at about 55 a cycle and SM) or the unpacking of 128 x 128 codes
// (730 cycles); a tile about kTile more (start, end of its sums), a cluster's exchange kExchange. Measured on a B200
// (us): 512 x 8192 x 7168 in tiles of 256 56, of 192 75; 2000 x 8192 x 7168 of 192 196, of 256 (with the end of
// each tile's sums exposed) 287.
constexpr int64_t kUnpack = 730, kTile = 3000, kExchange = 2500;
template <int BN, int G, bool HALF>
void plan_bn(const GArgs& a, GPlan& best) {
  constexpr auto kern = int4_gemm_kernel<BN, G, HALF>;
  using L = GSmem<BN>;
  const int64_t tiles = static_cast<int64_t>((a.M + BN - 1) / BN) * a.n_tiles;
  const int64_t step = std::max<int64_t>(BN * 256 / 55, kUnpack);
  for (int S = 1; S <= 8 && S <= a.steps; ++S) {
    if (S > 1 && BN > 128) break;  // no room for the partial sums
    const int fit = resident<kern>(S, L::bytes(S), L::kThreads);
    if (S > 1 && tiles > fit) break;  // a cluster has one tile
    const int64_t waves = (tiles + fit - 1) / fit;
    if (BN == 256 && waves > 1) break;
    const int64_t cost = waves * ((a.steps + S - 1) / S * step + kTile) + (S > 1 ? kExchange : 0);
    if (best.cost < 0 || cost < best.cost)
      best = GPlan{BN, S, static_cast<int>(S > 1 ? tiles * S : std::min<int64_t>(tiles, fit)), cost};
  }
}

template <int BN, int G, bool HALF>
void launch_bn(GArgs a, const GPlan& p, const CUtensorMap* tw, const CUtensorMap& tm, cudaStream_t s) {
  constexpr auto kern = int4_gemm_kernel<BN, G, HALF>;
  using L = GSmem<BN>;
  a.m_tiles = (a.M + BN - 1) / BN;
  a.S = p.S;
  const int grid = p.grid;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(L::kThreads);
  cfg.dynamicSmemBytes = L::bytes(a.S);
  cfg.stream = s;
  cudaLaunchAttribute attrs[2];
  int n = 0;
  if (pdl_enabled()) {
    attrs[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (a.S > 1) {
    attrs[n].id = cudaLaunchAttributeClusterDimension;
    attrs[n].val.clusterDim.x = a.S;
    attrs[n].val.clusterDim.y = attrs[n].val.clusterDim.z = 1;
    ++n;
  }
  cfg.attrs = attrs;
  cfg.numAttrs = n;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, tw[0], tw[1], tw[2], tm, a);
  if (e != cudaSuccess) throw std::runtime_error(std::string("minisgl: kernel launch failed: ") + cudaGetErrorString(e));
}

template <int G, bool HALF>
GPlan plan_type(const GArgs& a) {
  GPlan p{0, 1, 0, -1};
  plan_bn<32, G, HALF>(a, p);
  plan_bn<64, G, HALF>(a, p);
  plan_bn<128, G, HALF>(a, p);
  plan_bn<192, G, HALF>(a, p);
  plan_bn<256, G, HALF>(a, p);
  return p;
}

template <int G, bool HALF>
void launch_type(GArgs a, const void* scales, const void* x, int64_t ldx, int64_t K, cudaStream_t s) {
  constexpr int group = G;
  const GPlan p = plan_type<G, HALF>(a);
  const int best = p.bn;
  a.x_blocks = K % 64 == 0;
  const CUtensorMap tm = a.x_blocks ? make_tmap_bf16_kblocks(x, a.M, K, ldx, best, 2) : make_tmap_bf16_2d_sw128(x, a.M, K, ldx, best);
  // codes, scales, zero points: a row of a map is a tile of 16 rows, its columns the tile's 128-column units
  const uint64_t tiles = static_cast<uint64_t>(a.tiles16), steps = static_cast<uint64_t>(a.steps), per = 128 / group;
  const auto words = [&](const void* p, CUtensorMapDataType type, int size, uint64_t cols, uint32_t box_cols) {
    const uint64_t dims[2] = {cols, tiles}, strides[1] = {cols * size};
    const uint32_t box[2] = {box_cols, 8};
    return make_tmap(p, type, size, 2, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_NONE);
  };
  const uint32_t pairs = static_cast<uint32_t>(8 * per);
  CUtensorMap tw[3];
  tw[0] = words(a.packed, CU_TENSOR_MAP_DATA_TYPE_INT32, 4, steps * 256, 256);
  tw[1] = words(scales, CU_TENSOR_MAP_DATA_TYPE_INT32, 4, steps * pairs, pairs);
  tw[2] = a.zeros == nullptr ? tw[1]
                             : words(a.zeros, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, (steps * per + 1) / 2 * 16, std::max(16u, pairs));
  switch (best) {
    case 32: launch_bn<32, G, HALF>(a, p, tw, tm, s); break;
    case 64: launch_bn<64, G, HALF>(a, p, tw, tm, s); break;
    case 128: launch_bn<128, G, HALF>(a, p, tw, tm, s); break;
    case 192: launch_bn<192, G, HALF>(a, p, tw, tm, s); break;
    default: launch_bn<256, G, HALF>(a, p, tw, tm, s); break;
  }
}

template <bool HALF>
void launch_group(const GArgs& a, const void* scales, const void* x, int64_t ldx, int64_t K, int group, cudaStream_t s) {
  switch (group) {
    case 32: launch_type<32, HALF>(a, scales, x, ldx, K, s); break;
    case 64: launch_type<64, HALF>(a, scales, x, ldx, K, s); break;
    default: launch_type<128, HALF>(a, scales, x, ldx, K, s); break;
  }
}

template <int BN>
std::array<int, 5> ring_of() {
  using L = GSmem<BN>;
  return {BN, L::kXs, L::kPs, L::kAs, L::kSets};
}

}  // namespace

std::vector<std::array<int, 5>> int4_rings() {
  return {ring_of<32>(), ring_of<64>(), ring_of<128>(), ring_of<192>(), ring_of<256>()};
}

std::pair<int, int> int4_tiles(int64_t M, int64_t N, int64_t K, int group, bool half) {
  GArgs a{};
  a.M = static_cast<int>(M), a.N = static_cast<int>(N);
  a.steps = static_cast<int>((K + 127) / 128), a.n_tiles = static_cast<int>((N + kRows - 1) / kRows);
  const auto plan = [&](auto h) {
    constexpr bool H = decltype(h)::value;
    return group == 32 ? plan_type<32, H>(a) : group == 64 ? plan_type<64, H>(a) : plan_type<128, H>(a);
  };
  const GPlan p = half ? plan(std::true_type{}) : plan(std::false_type{});
  return {p.bn, p.S};
}

void launch_int4_gemm(const Int4LinearArgs& r, cudaStream_t s) {
  if (r.M <= 0) return;
  if ((r.M + 31) / 32 * ((r.N + kRows - 1) / kRows) >= (1ll << 31) || r.M >= (1ll << 31) || r.N > (1ll << 30) ||
      r.K > (1ll << 30))
    throw std::runtime_error("minisgl.int4_linear: size out of range");
  if (r.x_scales != nullptr && r.x_wide == nullptr)
    throw std::runtime_error("minisgl.int4_linear: scratch for the widened rows is missing");
  GArgs a{};
  a.packed = r.packed, a.zeros = r.zeros, a.row_pow = r.row_pow;
  a.bias = r.bias, a.out = r.out;
  a.M = static_cast<int>(r.M), a.N = static_cast<int>(r.N);
  a.steps = static_cast<int>((r.K + 127) / 128), a.tiles16 = static_cast<int>(2 * ((r.N + 31) / 32));
  a.n_tiles = static_cast<int>((r.N + kRows - 1) / kRows);
  a.ldo = r.ldo;
  a.scale_half = r.scale_type == DType::kF16;
  a.bias_type = static_cast<int>(r.bias_type), a.out_type = static_cast<int>(r.out_type);
  a.err = ErrorSink{r.err};
  a.vec_out = r.out_type != DType::kF32 && r.N % 8 == 0 && (r.M == 1 || r.ldo % 8 == 0) &&
              reinterpret_cast<uintptr_t>(r.out) % 16 == 0;
  const void* x = r.x;
  int64_t ldx = r.M > 1 ? r.ldx : r.K;
  if (r.x_scales != nullptr) {
    const int64_t runs = r.M * (r.K / 8);
    const unsigned blocks = static_cast<unsigned>(std::min<int64_t>((runs + 255) / 256, 148 * 8));
    launch_pdl(mx8_rows_bf16_kernel, dim3(blocks), dim3(256), 0, s, static_cast<uint4*>(r.x_wide),
               static_cast<const uint8_t*>(r.x), r.x_scales, r.M, static_cast<int>(r.K), r.ldx, r.ld_xs);
    x = r.x_wide;
    ldx = r.K;
  }
  if (r.x_scales == nullptr && r.x_type == DType::kF16)
    launch_group<true>(a, r.scales, x, ldx, r.K, r.group, s);
  else
    launch_group<false>(a, r.scales, x, ldx, r.K, r.group, s);
}

}  // namespace minisgl
