// Attention of few query rows over the 4-bit paged KV cache: one token per
// request (decode) or a few at its end (drafted tokens, short extends).
//
//   o_r = sum_j p_rj v_j / sum_j p_rj,  p_rj = 2^((q_r . k_j - m_r) c),  c = scale log2 e,
//
// with k_j and v_j in 4-bit codes, 136 bytes of cache per token and 128-dim
// head. Bound by what a warp has to do per code, not by the tensor pipe, so
// everything is laid out to keep that small:
//
// * The products are taken the other way round, S^T = K q^T and O^T = V^T P^T
//   (warp-level m16n8k16 bf16 MMA): keys and dims fill the 16 rows of A, and
//   the query rows, 8 at a time, are the 8 columns of B, so nothing is wasted
//   on padding for groups of up to 8 heads. tcgen05 would need 128 rows.
// * The cache's byte order is the A fragments' order: a lane's 16 bytes from
//   shared memory are the codes of two MMAs (K) or four (V), and a code pair
//   becomes two bf16 numbers by one mask: 128 + c has the bits 0x4300 | c.
// * K: the product starts at -136 sum(q) instead of 0, which turns 128 + c into
//   c - 8, and a group's scale multiplies its four sums. V: s (128 + c) - 136 s
//   in one packed fused multiply-add, exact in bf16.
// * The running maximum moves only when a score exceeds it by 8 (in powers of
//   two); other tiles neither reduce over lanes nor rescale the output.
//
// Work is split evenly whatever the lengths are: all key tiles of all requests,
// heads and row tiles form one sequence, of which each CTA takes an equal run.
// A run's first and last pieces may be parts of a longer one: those write
// (m, l, O) records, which a second small kernel joins.
#include <stdexcept>

#include "kv4.cuh"
#include "launch.h"
#include "ops.h"

namespace minisgl {
namespace {

using bf16 = __nv_bfloat16;

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kWarps = 8;                          // consumers; each takes 16 keys of a tile
constexpr int kTile = 16 * kWarps;                 // keys per tile
constexpr int kRows = 8;                           // query rows per tile
constexpr int kThreads = (kWarps + 1) * 32;        // and one producer warp
constexpr int kStages = 4;
constexpr float kFloor = -1e30f;                   // maximum of a row that has seen no key

__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// nibbles 0 and 4 of w as the bf16 pair (128 + c, 128 + c)
__device__ __forceinline__ uint32_t code_pair(uint32_t w) {
  uint32_t r;
  asm("lop3.b32 %0, %1, 0x000f000f, 0x43004300, 0xea;" : "=r"(r) : "r"(w));
  return r;
}
__device__ __forceinline__ uint32_t fma_pair(uint32_t x, uint32_t s, uint32_t o) {
  uint32_t r;
  asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(x), "r"(s), "r"(o));
  return r;
}
__device__ __forceinline__ uint32_t mul_pair(uint32_t x, uint32_t y) {
  const __nv_bfloat162 v =
      __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&x), *reinterpret_cast<const __nv_bfloat162*>(&y));
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ void consumers_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kWarps * 32) : "memory"); }

// Bytes of one stage: the K blocks of a tile, then its V blocks.
template <int D>
constexpr int half_bytes() { return kTile * kv4::row_bytes(D); }

// One request's place in the sequence of tiles.
struct Piece {
  int b, h, rt;       // request, KV head, row tile
  int kt0, kt1, kts;  // key tiles [kt0, kt1) of kts
};

__device__ __forceinline__ int rows_of(const Kv4AttnArgs& a, int b) {
  const int n = a.cu_q == nullptr ? 1 : max(0, a.cu_q[b + 1] - a.cu_q[b]);
  return n * (a.hq / a.hk);
}
__device__ __forceinline__ int keys_of(const Kv4AttnArgs& a, int b) { return min(max(a.seq_lens[b], 0), a.ld_pt); }
__device__ __forceinline__ int key_tiles(int keys) { return max(1, (keys + kTile - 1) / kTile); }

// The run [at, end) of this CTA as pieces, request by request (pre: sums of the
// requests' tiles, in shared memory).
struct Walk {
  int at, end, b;
  __device__ __forceinline__ bool next(const Kv4AttnArgs& a, const int* pre, Piece& p) {
    if (at >= end) return false;
    while (pre[b + 1] <= at) ++b;
    const int kts = key_tiles(keys_of(a, b));
    const int in = at - pre[b];
    const int tile_rows = (rows_of(a, b) + kRows - 1) / kRows;
    p.b = b, p.kts = kts;
    p.kt0 = in % kts;
    const int unit = in / kts;
    p.rt = unit % tile_rows, p.h = unit / tile_rows;
    p.kt1 = min(kts, p.kt0 + end - at);
    at += p.kt1 - p.kt0;
    return true;
  }
};

template <int D>
__global__ void __launch_bounds__(kThreads, 2) kv4_attn_kernel(Kv4AttnArgs a) {
  extern __shared__ uint8_t smem_raw[];
  constexpr int kNG = D / kv4::kGroup;    // scale groups of a row
  constexpr int kHalf = half_bytes<D>();
  constexpr int kStage = 2 * kHalf;
  constexpr int kLd = D + 4;              // padded row of the merge buffer (floats)
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 127) & ~static_cast<uintptr_t>(127));
  float* so = reinterpret_cast<float*>(ring + kStages * kStage);  // [warps][rows][kLd]
  float* sm = so + kWarps * kRows * kLd;                          // [warps][rows]
  float* sl = sm + kWarps * kRows;
  uint64_t* full = reinterpret_cast<uint64_t*>(sl + kWarps * kRows);
  uint64_t* empty = full + kStages;
  int* pre = reinterpret_cast<int*>(empty + kStages);  // [B + 1]
  const ErrorSink err{a.err};
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  pdl_launch_dependents();
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], kWarps);
    }
    fence_barrier_init();
  }
  pdl_wait();
  // sums of the requests' tiles
  for (int b = threadIdx.x; b < a.B; b += kThreads) {
    const int rows = rows_of(a, b);
    pre[b + 1] = key_tiles(keys_of(a, b)) * ((rows + kRows - 1) / kRows) * a.hk;
  }
  __syncthreads();
  if (warp == 0) {
    int carry = 0;
    for (int b0 = 0; b0 < a.B; b0 += 32) {
      int v = b0 + lane < a.B ? pre[b0 + lane + 1] : 0;
#pragma unroll
      for (int o = 1; o < 32; o *= 2) {
        const int u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
      }
      if (b0 + lane < a.B) pre[b0 + lane + 1] = carry + v;
      carry += __shfl_sync(0xffffffffu, v, 31);
    }
    if (lane == 0) pre[0] = 0;
  }
  __syncthreads();
  const int64_t total = pre[a.B];
  // no run is empty among the first n CTAs, so the records of a chain are all written
  const int n = min(static_cast<int>(gridDim.x), pre[a.B]), me = blockIdx.x;
  Walk walk;
  walk.at = me < n ? static_cast<int>(total * me / n) : 0;
  walk.end = me < n ? static_cast<int>(total * (me + 1) / n) : 0;
  {
    int lo = 0, hi = a.B;  // last b with pre[b] <= at
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (pre[mid] <= walk.at) lo = mid; else hi = mid;
    }
    walk.b = lo;
  }
  int4* desc = reinterpret_cast<int4*>(a.desc) + me;
  if (threadIdx.x == 0) *desc = make_int4(-1, 0, 0, 0);
  const int page_size = a.page_size, shift = a.page_shift;
  const int seg = min(page_size, kTile);       // keys that are side by side in the cache
  const int segs = kTile / seg;
  const int seg_bytes = seg * kv4::row_bytes(D);
  Piece p;

  if (warp == kWarps) {
    // ------------------------------------------------------------ producer ----
    const int64_t block = static_cast<int64_t>(page_size) * kv4::row_bytes(D);
    int it = 0;
    bool ok = true;
    while (ok && walk.next(a, pre, p)) {
      const int row = a.req_rows[p.b];
      const bool row_ok = row >= 0 && row < a.pt_rows;
      if (!row_ok && lane == 0) err.report(kErrBadIndex, 961);
      const int32_t* pt = a.page_table + static_cast<int64_t>(row_ok ? row : 0) * a.ld_pt;
      const int keys = row_ok ? keys_of(a, p.b) : 0;
      if (a.seq_lens[p.b] > a.ld_pt && lane == 0) err.report(kErrBadIndex, 962);
      auto slot_of = [&](int kt) {
        const int pos = kt * kTile + lane * seg;
        return lane < segs && pos < keys ? pt[pos] : -1;
      };
      int slot = slot_of(p.kt0);
      for (int kt = p.kt0; kt < p.kt1; ++kt, ++it) {
        const int next = kt + 1 < p.kt1 ? slot_of(kt + 1) : -1;  // a tile ahead
        const int s = it % kStages;
        if (it >= kStages && !mbar_wait(&empty[s], ((it / kStages) & 1u) ^ 1u, err, 260)) {
          ok = false;
          break;
        }
        const bool wanted = lane < segs && kt * kTile + lane * seg < keys;
        const bool good = wanted && slot >= 0 && slot < a.kv_slots;
        if (wanted && !good) err.report(kErrBadIndex, 963);
        const int count = __popc(__ballot_sync(0xffffffffu, good));
        if (lane == 0) mbar_arrive_expect_tx(&full[s], 2 * count * seg_bytes);
        __syncwarp();
        if (good) {
          const int off = slot & (page_size - 1);
          const int64_t at = (static_cast<int64_t>(slot >> shift) * a.hk + p.h) * block;
          uint8_t* dst = ring + s * kStage + lane * seg_bytes;
          if (seg == page_size) {
            bulk_load(dst, a.k_pool + at, seg_bytes, &full[s]);
            bulk_load(dst + kHalf, a.v_pool + at, seg_bytes, &full[s]);
          } else {  // part of a larger page: its codes and its scales
            const int64_t codes = at + (off & ~(kTile - 1)) * (D / 2);
            const int64_t scales = at + page_size * (D / 2) + (off & ~(kTile - 1)) * kNG;
            bulk_load(dst, a.k_pool + codes, kTile * (D / 2), &full[s]);
            bulk_load(dst + kTile * (D / 2), a.k_pool + scales, kTile * kNG, &full[s]);
            bulk_load(dst + kHalf, a.v_pool + codes, kTile * (D / 2), &full[s]);
            bulk_load(dst + kHalf + kTile * (D / 2), a.v_pool + scales, kTile * kNG, &full[s]);
          }
        }
        slot = next;
      }
    }
    // copies in flight land before the CTA's shared memory is given back
    for (int j = max(0, it - kStages); j < it; ++j)
      if (!mbar_wait(&full[j % kStages], (j / kStages) & 1u, err, 261)) break;
    return;
  }

  // ------------------------------------------------------------- consumers ----
  const int g = lane >> 2, t = lane & 3;
  const int G = a.hq / a.hk;
  const float c = a.scale * kLog2e;
  // this lane's keys of the warp's 16 (rows g and g + 8 of S^T), the segment
  // they lie in and the places of its codes and scales there
  const int key0 = warp * 16 + 4 * (g >> 1) + (g & 1);
  const int seg_at = (warp * 16 / seg) * seg_bytes;
  const int in_seg = (warp * 16) & (seg - 1);
  const int key_in = in_seg + 4 * (g >> 1) + (g & 1);
  const int quad_in = in_seg / 4 + t;
  const int k_at = seg_at + key_in * (D / 2) + t * (D / 8);
  const int ks_at = seg_at + seg * (D / 2) + key_in * kNG;
  const int v_at = kHalf + seg_at + quad_in * (2 * D) + ((g ^ (2 * t)) * 16);
  const int vs_at = kHalf + seg_at + seg * (D / 2) + (quad_in * kNG + (g >> 2)) * 4;
  constexpr int kHalves = D / 64;  // 64-dim halves of V
  int it = 0;
  bool ok = true;

  while (walk.next(a, pre, p)) {
    const int keys = keys_of(a, p.b);
    const int q0 = a.cu_q == nullptr ? p.b : a.cu_q[p.b];
    const int rows = rows_of(a, p.b);
    const int q_len = rows / G;
    // query fragments of row 8 rt + g, and the starts of its groups' sums
    uint32_t qb[kNG][4];
    float init[kNG][2];
    {
      const int r = p.rt * kRows + g;
      const bool live = r < rows;
      const bf16* src = static_cast<const bf16*>(a.q) + static_cast<int64_t>(q0 + (live ? r / G : 0)) * a.ld_q +
                        (p.h * G + (live ? r % G : 0)) * D + 8 * t;
#pragma unroll
      for (int i = 0; i < kNG; ++i) {
        uint4 v = make_uint4(0, 0, 0, 0);
        if (live) v = *reinterpret_cast<const uint4*>(src + 32 * i);
        // dims 0..7 of the word -> (0, 4), (1, 5), (2, 6), (3, 7)
        qb[i][0] = __byte_perm(v.x, v.z, 0x5410), qb[i][1] = __byte_perm(v.x, v.z, 0x7632);
        qb[i][2] = __byte_perm(v.y, v.w, 0x5410), qb[i][3] = __byte_perm(v.y, v.w, 0x7632);
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) sum += __uint_as_float(qb[i][j] << 16) + __uint_as_float(qb[i][j] & 0xffff0000u);
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        sum *= -136.f;
        init[i][0] = __shfl_sync(0xffffffffu, sum, 8 * t);      // of row 2 t
        init[i][1] = __shfl_sync(0xffffffffu, sum, 8 * t + 4);  // of row 2 t + 1
      }
    }
    // keys that rows 2 t and 2 t + 1 see, and that every row of the tile sees
    const int r0 = p.rt * kRows + 2 * t;
    const int see0 = r0 < rows ? keys - q_len + r0 / G + 1 : 0;
    const int see1 = r0 + 1 < rows ? keys - q_len + (r0 + 1) / G + 1 : 0;
    const int see_all = keys - q_len + p.rt * kRows / G + 1;
    float o[2 * kNG][4];
#pragma unroll
    for (int i = 0; i < 2 * kNG; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    float m0 = kFloor, m1 = kFloor, l0 = 0.f, l1 = 0.f;
    float mc0 = kFloor * c, mc1 = kFloor * c;

    for (int kt = p.kt0; kt < p.kt1; ++kt, ++it) {
      const int s = it % kStages;
      if (ok) ok = mbar_wait(&full[s], (it / kStages) & 1u, err, 262);
      const uint8_t* st = ring + s * kStage;
      // ---- S^T of 16 keys x 8 rows
      float sc[4] = {0.f, 0.f, 0.f, 0.f};
      {
        uint32_t w0[kNG], w1[kNG];  // words of rows key0 and key0 + 2
        if constexpr (D == 128) {
          *reinterpret_cast<uint4*>(w0) = *reinterpret_cast<const uint4*>(st + k_at);
          *reinterpret_cast<uint4*>(w1) = *reinterpret_cast<const uint4*>(st + k_at + D);
        } else {
          *reinterpret_cast<uint2*>(w0) = *reinterpret_cast<const uint2*>(st + k_at);
          *reinterpret_cast<uint2*>(w1) = *reinterpret_cast<const uint2*>(st + k_at + D);
        }
        uint32_t s0, s1;  // the rows' scale bytes
        if constexpr (D == 128) {
          s0 = *reinterpret_cast<const uint32_t*>(st + ks_at);
          s1 = *reinterpret_cast<const uint32_t*>(st + ks_at + 2 * kNG);
        } else {
          s0 = *reinterpret_cast<const uint16_t*>(st + ks_at);
          s1 = *reinterpret_cast<const uint16_t*>(st + ks_at + 2 * kNG);
        }
#pragma unroll
        for (int i = 0; i < kNG; ++i) {
          float acc[4] = {init[i][0], init[i][1], init[i][0], init[i][1]};
          const uint32_t x[4] = {code_pair(w0[i]), code_pair(w1[i]), code_pair(w0[i] >> 4), code_pair(w1[i] >> 4)};
          mma_bf16(acc, x, qb[i][0], qb[i][1]);
          const uint32_t y[4] = {code_pair(w0[i] >> 8), code_pair(w1[i] >> 8), code_pair(w0[i] >> 12),
                                 code_pair(w1[i] >> 12)};
          mma_bf16(acc, y, qb[i][2], qb[i][3]);
          const float f0 = kv4::scale_f32(__byte_perm(s0, 0, 0x4440 + i));
          const float f1 = kv4::scale_f32(__byte_perm(s1, 0, 0x4440 + i));
          sc[0] += acc[0] * f0, sc[1] += acc[1] * f0;
          sc[2] += acc[2] * f1, sc[3] += acc[3] * f1;
        }
      }
      const int pos = kt * kTile + key0;
      if ((kt + 1) * kTile > see_all) {  // uniform over the CTA
        if (pos >= see0) sc[0] = -INFINITY;
        if (pos >= see1) sc[1] = -INFINITY;
        if (pos + 2 >= see0) sc[2] = -INFINITY;
        if (pos + 2 >= see1) sc[3] = -INFINITY;
      }
      // ---- running maximum
      {
        float x0 = fmaxf(sc[0], sc[2]), x1 = fmaxf(sc[1], sc[3]);
        if (__any_sync(0xffffffffu, fmaxf(fmaf(x0, c, -mc0), fmaf(x1, c, -mc1)) > 8.f)) {
#pragma unroll
          for (int sh = 4; sh < 32; sh *= 2) {
            x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, sh));
            x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, sh));
          }
          const float n0 = fmaxf(m0, x0), n1 = fmaxf(m1, x1);
          const float f0 = exp2_approx((m0 - n0) * c), f1 = exp2_approx((m1 - n1) * c);
          m0 = n0, m1 = n1, mc0 = m0 * c, mc1 = m1 * c;
          l0 *= f0, l1 *= f1;
#pragma unroll
          for (int i = 0; i < 2 * kNG; ++i) o[i][0] *= f0, o[i][1] *= f1, o[i][2] *= f0, o[i][3] *= f1;
        }
      }
      const float p0 = exp2_approx(fmaf(sc[0], c, -mc0)), p1 = exp2_approx(fmaf(sc[1], c, -mc1));
      const float p2 = exp2_approx(fmaf(sc[2], c, -mc0)), p3 = exp2_approx(fmaf(sc[3], c, -mc1));
      l0 += p0 + p2, l1 += p1 + p3;
      const uint32_t b0 = transpose8x8(pack_bf16x2(p0, p1));
      const uint32_t b1 = transpose8x8(pack_bf16x2(p2, p3));
      // ---- O^T += V^T P^T
#pragma unroll
      for (int hf = 0; hf < kHalves; ++hf) {
        const uint4 v4 = *reinterpret_cast<const uint4*>(st + v_at + hf * 128);
        const uint32_t w[4] = {v4.x, v4.y, v4.z, v4.w};
        const uint32_t sv = *reinterpret_cast<const uint32_t*>(st + vs_at + hf * 8);
        const uint32_t sa = (sv & 0x00ff00ffu) * 16 + kv4::kScaleBf16x2;                        // tokens 0 and 1
        const uint32_t sb = __byte_perm(sv, 0, 0x4341) * 16 + kv4::kScaleBf16x2;  // tokens 2 and 3
        const uint32_t oa = mul_pair(sa, 0xc308c308u), ob = mul_pair(sb, 0xc308c308u);          // times -136
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t x[4] = {fma_pair(code_pair(w[j]), sa, oa), fma_pair(code_pair(w[j] >> 4), sa, oa),
                                 fma_pair(code_pair(w[j] >> 8), sb, ob), fma_pair(code_pair(w[j] >> 12), sb, ob)};
          mma_bf16(o[4 * hf + j], x, b0, b1);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[s]);
    }

    // ---- the warps' states of the piece, joined
#pragma unroll
    for (int sh = 4; sh < 32; sh *= 2) {
      l0 += __shfl_xor_sync(0xffffffffu, l0, sh);
      l1 += __shfl_xor_sync(0xffffffffu, l1, sh);
    }
    consumers_sync();  // the previous piece's states have been read
    {
      float* d0 = so + (warp * kRows + 2 * t) * kLd + 8 * g;
      float* d1 = d0 + kLd;
#pragma unroll
      for (int hf = 0; hf < kHalves; ++hf) {
        const float(*v)[4] = o + 4 * hf;
        *reinterpret_cast<float4*>(d0 + 64 * hf) = make_float4(v[0][0], v[0][2], v[1][0], v[1][2]);
        *reinterpret_cast<float4*>(d0 + 64 * hf + 4) = make_float4(v[2][0], v[2][2], v[3][0], v[3][2]);
        *reinterpret_cast<float4*>(d1 + 64 * hf) = make_float4(v[0][1], v[0][3], v[1][1], v[1][3]);
        *reinterpret_cast<float4*>(d1 + 64 * hf + 4) = make_float4(v[2][1], v[2][3], v[3][1], v[3][3]);
      }
      if (g == 0) {
        sm[warp * kRows + 2 * t] = m0, sm[warp * kRows + 2 * t + 1] = m1;
        sl[warp * kRows + 2 * t] = l0, sl[warp * kRows + 2 * t + 1] = l1;
      }
    }
    consumers_sync();
    {
      constexpr int kE = D / 32;  // dims of a lane; row = warp
      float top = kFloor;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) top = fmaxf(top, sm[w * kRows + warp]);
      float acc[kE] = {}, l = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float f = exp2_approx((sm[w * kRows + warp] - top) * c);
        l += f * sl[w * kRows + warp];
        const float* v = so + (w * kRows + warp) * kLd + lane * kE;
#pragma unroll
        for (int e = 0; e < kE; ++e) acc[e] += f * v[e];
      }
      const int r = p.rt * kRows + warp;
      if (p.kt0 == 0 && p.kt1 == p.kts) {
        if (r < rows) {
          const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);  // no key: zeros; NaN stays
          uint32_t* dst = reinterpret_cast<uint32_t*>(static_cast<bf16*>(a.out) +
                                                      (static_cast<int64_t>(q0 + r / G) * a.hq + p.h * G + r % G) * D + lane * kE);
#pragma unroll
          for (int e = 0; e < kE / 2; ++e) dst[e] = pack_bf16x2(acc[2 * e] * inv, acc[2 * e + 1] * inv);
        }
      } else {
        const int rec = (2 * me + (p.kt0 == 0 ? 1 : 0)) * kRows + warp;
        float* dst = a.part_o + static_cast<int64_t>(rec) * D + lane * kE;
#pragma unroll
        for (int e = 0; e < kE; ++e) dst[e] = acc[e];
        if (lane == 0) a.part_ml[2 * rec] = top, a.part_ml[2 * rec + 1] = l;
        if (p.kt0 == 0 && threadIdx.x == 0) {
          // the CTA whose run holds the piece's last tile
          const int64_t last = walk.at - 1 + p.kts - p.kt1;
          *desc = make_int4(static_cast<int>(((last + 1) * n - 1) / total), p.b, p.h, p.rt);
        }
      }
    }
  }
}

// Joins the records of the piece that CTA blockIdx.x began and others went on
// with. Warp w: row w % 8, records w / 8 modulo 4 of the chain.
template <int D>
__global__ void __launch_bounds__(1024) kv4_join_kernel(Kv4AttnArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  constexpr int kE = D / 32;
  __shared__ float so[3][kRows][D];
  __shared__ float sml[3][kRows][2];
  const int4 d = reinterpret_cast<const int4*>(a.desc)[blockIdx.x];
  if (d.x < 0) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int row = warp % kRows, part = warp / kRows;
  const float c = a.scale * kLog2e;
  float m = kFloor, l = 0.f, acc[kE] = {};
#pragma unroll 4
  for (int i = static_cast<int>(blockIdx.x) + part; i <= d.x; i += 4) {
    const int rec = (2 * i + (i == static_cast<int>(blockIdx.x) ? 1 : 0)) * kRows + row;
    const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + 2 * rec);
    const float top = fmaxf(m, ml.x);
    const float f = exp2_approx((m - top) * c), e = exp2_approx((ml.x - top) * c);
    const float* v = a.part_o + static_cast<int64_t>(rec) * D + lane * kE;
    m = top, l = l * f + ml.y * e;
#pragma unroll
    for (int k = 0; k < kE; ++k) acc[k] = acc[k] * f + v[k] * e;
  }
  if (part > 0) {
#pragma unroll
    for (int k = 0; k < kE; ++k) so[part - 1][row][lane * kE + k] = acc[k];
    if (lane == 0) sml[part - 1][row][0] = m, sml[part - 1][row][1] = l;
  }
  __syncthreads();
  if (part > 0) return;
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    const float top = fmaxf(m, sml[i][row][0]);
    const float f = exp2_approx((m - top) * c), e = exp2_approx((sml[i][row][0] - top) * c);
    m = top, l = l * f + sml[i][row][1] * e;
#pragma unroll
    for (int k = 0; k < kE; ++k) acc[k] = acc[k] * f + so[i][row][lane * kE + k] * e;
  }
  const int G = a.hq / a.hk;
  const int r = d.w * kRows + row;
  if (r >= rows_of(a, d.y)) return;
  const int q0 = a.cu_q == nullptr ? d.y : a.cu_q[d.y];
  const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
  uint32_t* dst = reinterpret_cast<uint32_t*>(static_cast<bf16*>(a.out) +
                                              (static_cast<int64_t>(q0 + r / G) * a.hq + d.z * G + r % G) * D + lane * kE);
#pragma unroll
  for (int e = 0; e < kE / 2; ++e) dst[e] = pack_bf16x2(acc[2 * e] * inv, acc[2 * e + 1] * inv);
}

template <int D>
int attn_smem(int B) {
  return 128 + kStages * 2 * half_bytes<D>() + kWarps * kRows * (D + 4 + 2) * 4 + 2 * kStages * 8 + (B + 1) * 4;
}

template <int D>
void launch_typed(const Kv4AttnArgs& a, cudaStream_t s) {
  static bool done[64] = {};  // per device
  int dev = 0;
  cudaGetDevice(&dev);
  const int most = attn_smem<D>(kKv4MaxBatch);
  if (!done[dev & 63]) {
    if (cudaFuncSetAttribute(kv4_attn_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, most) != cudaSuccess)
      throw std::runtime_error("minisgl.attention_kv4: shared memory limit");
    done[dev & 63] = true;
  }
  launch_pdl(kv4_attn_kernel<D>, dim3(a.ctas), dim3(kThreads), attn_smem<D>(a.B), s, a);
  launch_pdl(kv4_join_kernel<D>, dim3(a.ctas), dim3(1024), 0, s, a);
}

}  // namespace

int kv4_attn_ctas(int sms) { return 2 * sms; }

void launch_kv4_attention(const Kv4AttnArgs& a, cudaStream_t s) {
  if (a.B <= 0) return;
  if (a.d == 128) launch_typed<128>(a, s);
  else if (a.d == 64) launch_typed<64>(a, s);
  else throw std::runtime_error("minisgl.attention_kv4: head_dim must be 64 or 128");
}

}  // namespace minisgl
