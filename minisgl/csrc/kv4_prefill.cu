// Causal attention of many query rows over keys of the 4-bit cache, expanded
// once to bf16 tiles (kv4_load_kernel writes them; their values are exact).
//
//   S = Q K^T,  P = 2^(S scale log2 e - m),  O += P V,  out = O / sum P
//
// on tcgen05. Bound by the tensor pipe (4 d flops per query row and key) and,
// close behind, by the exponentials: 128 x 128 scores of 128 dims take 1024 cycles
// of MMA for both products and 1024 of the special-function unit (64 dims: 640).
// 2048 queries of 64 heads over 16384 keys, with the expansion: 935 us in a stream
// of calls, where the power limit takes the clock down, 1100 TFLOP/s, 80 % of what
// cuBLAS sustains; 811 us in bursts (a graph of 20 calls, the best of five), 1270
// TFLOP/s, 78 % of cuBLAS's own burst. 4 prompts of 2048 tokens, 32 heads of 64
// dims: 147 us (burst).
//
// Query rows are (token, head of the group): TT = 128 / G tokens are a tile, so
// every group size fills its 128 rows (G = 7: 126 of them) and all heads of a
// group share each key tile. A CTA has two row tiles, whose softmax warps take
// turns with the tensor pipe: while one tile's scores become weights, the other
// tile's products run. 128-key tiles: an MMA of 128 x 128 x 16 takes 64 cycles,
// of 128 x 64 x 16 48 (measured), so 64-key tiles would leave a quarter unused.
//
// Weights are rounded to bf16 for the second product; their sums are of fp32
// ones, and a row's maximum is fp32: it is taken off scores of any size, where a
// rounding of its own would take the weights out of fp32's range.
//
// Work is split evenly: the key tiles of all row-tile pairs form one sequence, of
// which each CTA (one an SM) takes an equal run; a pair whose tiles fall to
// several CTAs leaves (m, l, O) records, joined by a second kernel. 2048 queries
// of 8 KV heads are 512 pairs, 3.46 a CTA: as whole pairs they took 4 turns.
//
// Keys come as shared-memory images: 128 rows of K (or V) of a head are 64-dim
// halves of 128-byte rows, swizzled as the MMA descriptors expect, so one plain
// bulk copy of 32 KB (64 dims: 16) brings each. Tensor memory: O of tile X at
// columns 128 X, S of it at 256 + 128 X with P (bf16 pairs) over its first 64.
#include <algorithm>
#include <stdexcept>

#include "exp2.cuh"
#include "kv4.cuh"
#include "launch.h"
#include "ops.h"
#include "tma_host.h"

namespace minisgl {
namespace {

constexpr int kRows = 128;                 // query rows of a tile
constexpr int kKeys = kKv4TileKeys;        // keys of a tile
constexpr int kHalf = kRows * 128;         // 64 dims of 128 rows (16 KB)
constexpr int kSlots = 5;                  // images in flight: K_0, V_0, K_1, ...
constexpr int kLoader = 16, kIssuer = 17;  // after eight softmax warps a tile
constexpr int kThreads = 576;
constexpr int kSCol = 256;
constexpr int kPolyPairs = 2;              // of 8 pairs of exponentials, on the FMA pipe
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kRescale = 8.f;            // the running maximum moves by more than this or not at all
constexpr int kAhead = 4;                  // pieces whose descriptions are kept
static_assert(kKeys == 128, "tiles of 128 keys");
template <int kD>
constexpr int image_bytes() { return kD / 64 * kHalf; }  // K or V of a tile (32 KB, 16 KB)
template <int kD>
constexpr int smem_bytes() { return (2 + kSlots) * image_bytes<kD>() + 256 + 2 * 4 * 256 + kAhead * 48; }
static_assert(smem_bytes<128>() <= 227 * 1024, "shared memory of a CTA");

// Waits that sleep: a first try that may suspend the thread for 20 us leaves the
// issue slots of its scheduler to the softmax warps (spinning waits took a third
// of them). The bounded loop follows.
__device__ __forceinline__ bool wait_asleep(uint64_t* bar, uint32_t parity, const ErrorSink& err, int where,
                                            const volatile int* s_abort) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, 20000;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0 || (mbar_wait(bar, parity, err, where) && !*s_abort);
}

// Whether this thread is the one that the warp elects (always the same one). Under
// it the compiler keeps the operands of tcgen05 instructions in uniform registers;
// under a test of the lane number it checks every lane's, and an MMA took 115
// cycles to issue, nearly twice its own 64.
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(r));
  return r != 0;
}

// One piece of a CTA's run: key tiles [kt0, kt1) of a pair of row tiles of one
// request and KV head. The loader walks the run and leaves descriptions in shared
// memory a piece ahead of the others (each of them walking took 5000 cycles of
// dependent loads a piece).
struct alignas(16) Piece {
  int q_begin, q_len, keys, tok0;
  int n0, n1, kt0, kt1;  // n0, n1: key tiles that row tile 0 / 1 sees anything of; kt1 < 0: no more pieces
  int h, whole, pad[2];  // whole: all tiles of the pair
};
static_assert(sizeof(Piece) == 48, "piece descriptions");

// The run of a CTA, piece by piece.
struct Walk {
  int b, pair, h, kt, left;
  int64_t at;  // place of the pair in the sequence that is split (kPairCost, then its tiles)
  int first;   // of the piece: image tile of the request's key 0
  __device__ __forceinline__ bool next(const Kv4PrefillArgs& a, Piece& p) {
    if (left <= 0 || b >= a.B) return false;
    const int TT = kRows / a.group;
    p.h = h;
    p.q_begin = a.cu_q[b], p.q_len = kv4_query_tokens(a.cu_q, b, a.T);
    p.keys = kv4_keys(a.seq_lens, b, a.ld_pt);
    first = a.starts[b];
    p.tok0 = pair * 2 * TT;
    const int cached = p.keys - p.q_len;
    auto tiles = [&](int t) { return t >= p.q_len ? 0 : max(0, (cached + min(p.q_len, t + TT) + kKeys - 1) / kKeys); };
    p.n0 = tiles(p.tok0), p.n1 = tiles(p.tok0 + TT);
    const int n = max(1, max(p.n0, p.n1));
    p.kt0 = kt, p.kt1 = min(n, kt + left);
    p.whole = kt == 0 && p.kt1 == n;
    left -= p.kt1 - p.kt0;
    if (kt == 0 && p.kt1 < n) {  // others go on with the pair
      const int4 more = reinterpret_cast<const int4*>(a.runs)[2 * blockIdx.x + 1];  // tiles, place, total, runs
      reinterpret_cast<int4*>(a.desc)[blockIdx.x] =
          make_int4(static_cast<int>(((at + kKv4PairCost + n) * more.w - 1) / more.z), b, pair, h);
    }
    if (first < 0) p.n0 = p.n1 = 0;  // keys that the plan does not have: none (the planning block has reported it)
    if (p.kt1 < n) {
      kt = p.kt1;
    } else {
      kt = 0, at += kKv4PairCost + n;
      if (++h == a.hk) {
        h = 0, ++pair;
        if (pair * 2 * TT >= p.q_len && left > 0) {
          pair = 0, ++b;
          while (b < a.B && kv4_query_tokens(a.cu_q, b, a.T) == 0) ++b;  // there is more to do, so there is one
        }
      }
    }
    return true;
  }
};

// 4 x 4 transpose of 16-byte vectors among four neighbouring lanes: lane i's vector
// j becomes lane j's vector i.
__device__ __forceinline__ void swap_vec(uint4& a, uint4& b, int mask, bool upper) {
  // the lower lane of a pair keeps a and gives b for the other's a
  uint4 give = upper ? a : b;
  give.x = __shfl_xor_sync(0xffffffffu, give.x, mask), give.y = __shfl_xor_sync(0xffffffffu, give.y, mask);
  give.z = __shfl_xor_sync(0xffffffffu, give.z, mask), give.w = __shfl_xor_sync(0xffffffffu, give.w, mask);
  if (upper) a = give; else b = give;
}
__device__ __forceinline__ void transpose4(uint4 (&v)[4], int lane) {
  swap_vec(v[0], v[1], 1, lane & 1), swap_vec(v[2], v[3], 1, lane & 1);
  swap_vec(v[0], v[2], 2, lane & 2), swap_vec(v[1], v[3], 2, lane & 2);
}

// Maxima that keep a NaN.
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// Tiles of row tile x in the piece.
__device__ __forceinline__ int tiles_in(const Piece& p, int x) { return max(0, min(p.kt1, x == 0 ? p.n0 : p.n1) - p.kt0); }

template <int kD>
__global__ void __launch_bounds__(kThreads, 1)
    kv4_prefill_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ Kv4PrefillArgs a) {
  extern __shared__ __align__(1024) uint8_t smem[];
  constexpr int kHalves = kD / 64;
  constexpr int kImage = image_bytes<kD>();
  uint8_t* sQ = smem;  // [tile][64-dim half]
  uint8_t* sKV = sQ + 2 * kImage;
  uint64_t* full = reinterpret_cast<uint64_t*>(sKV + kSlots * kImage);  // [kSlots]
  uint64_t* empty = full + kSlots;                                      // [kSlots]
  uint64_t* s_full = empty + kSlots;                                    // [2 tiles]
  uint64_t* p_full = s_full + 2;                                        // [2 tiles][2 chunks]
  uint64_t* o_done = p_full + 4;                                        // [2]
  uint64_t* o_free = o_done + 2;                                        // [2]
  uint64_t* q_full = o_free + 2;
  uint64_t* q_empty = q_full + 1;
  uint64_t* d_full = q_empty + 1;                                       // [kAhead] descriptions
  uint64_t* d_empty = d_full + kAhead;                                  // [kAhead]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(d_empty + kAhead);
  int* s_abort = reinterpret_cast<int*>(tmem_slot + 1);
  float* s_swap = reinterpret_cast<float*>(full + 32);          // [2 tiles][4 quadrants][2 halves][32 rows]
  Piece* s_piece = reinterpret_cast<Piece*>(s_swap + 2 * 4 * 64);  // [kAhead]
  const ErrorSink err{a.err};
  if ((smem_u32(smem) & 1023) != 0) {  // the swizzled tiles' alignment, as declared: nothing runs without it
    pdl_wait();
    if (threadIdx.x == 0) {
      err.report(kErrBadIndex, 285);
      reinterpret_cast<int4*>(a.desc)[blockIdx.x] = make_int4(-1, 0, 0, 0);
    }
    return;
  }
  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x) >> 5, 0), lane = threadIdx.x & 31;
  const int G = a.group, TT = kRows / G;  // tokens of a row tile

  pdl_launch_dependents();
  if (threadIdx.x == 0) {
    for (int i = 0; i < kSlots; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[2 * i], 8);
      mbar_init(&p_full[2 * i + 1], 8);
      mbar_init(&o_done[i], 1);
      mbar_init(&o_free[i], 8);
    }
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    for (int i = 0; i < kAhead; ++i) {
      mbar_init(&d_full[i], 1);
      mbar_init(&d_empty[i], 17);
    }
    *s_abort = 0;
    fence_barrier_init();
    prefetch_tmap(&tm_q);
  }
  if (warp == kIssuer) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  // rows that no query fills are zeros
  for (int i = threadIdx.x; i < 2 * kHalves * (kRows - TT * G) * 8; i += kThreads) {
    const int part = i / ((kRows - TT * G) * 8), at = i % ((kRows - TT * G) * 8);
    reinterpret_cast<uint4*>(sQ + part * kHalf + TT * G * 128)[at] = make_uint4(0, 0, 0, 0);
  }
  fence_proxy_async_smem();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  constexpr uint32_t tmem = 0;  // all 512 columns: the allocation's only place
  pdl_wait();
  Piece p;
  int issued = 0, pieces = 0;
  // the next piece, for all but the loader
  auto describe = [&](int k) {
    bool ok = wait_asleep(&d_full[k % kAhead], (k / kAhead) & 1, err, 283, s_abort);
    const int4* src = reinterpret_cast<const int4*>(s_piece + k % kAhead);
    int4* dst = reinterpret_cast<int4*>(&p);
    dst[0] = src[0], dst[1] = src[1], dst[2] = src[2];
    return ok && p.kt1 >= 0;
  };

  if (warp == kLoader) {
    // ------------------------------------------------------------- copies ----
    if (lane == 0) {
      Walk walk;
      const int4 run = reinterpret_cast<const int4*>(a.runs)[2 * blockIdx.x];
      walk.b = run.x, walk.pair = run.y, walk.h = run.z, walk.kt = run.w;
      walk.left = a.runs[8 * blockIdx.x + 4], walk.at = a.runs[8 * blockIdx.x + 5];
      reinterpret_cast<int4*>(a.desc)[blockIdx.x] = make_int4(-1, 0, 0, 0);
      bool ok = true;
      auto image = [&](const uint8_t* src) {
        const int s = issued % kSlots;
        if (issued >= kSlots) ok = wait_asleep(&empty[s], (issued / kSlots - 1) & 1, err, 271, s_abort);
        if (!ok) return;
        mbar_arrive_expect_tx(&full[s], kImage);
        bulk_load(sKV + s * kImage, src, kImage, &full[s]);
        ++issued;
      };
      for (int k = 0; ok; ++k) {
        const bool more = walk.next(a, p);
        if (!more) p.kt1 = -1;
        if (k >= kAhead) ok = wait_asleep(&d_empty[k % kAhead], (k / kAhead - 1) & 1, err, 284, s_abort);
        if (!ok) break;
        s_piece[k % kAhead] = p;
        mbar_arrive(&d_full[k % kAhead]);
        if (!more) break;
        const int count = max(tiles_in(p, 0), tiles_in(p, 1));
        if (count == 0) continue;
        // images of this head: K of a tile, then its V
        const uint8_t* src = static_cast<const uint8_t*>(a.images) + (static_cast<int64_t>(walk.first + p.kt0) * a.hk + p.h) * (2 * kImage);
        const int64_t step = static_cast<int64_t>(a.hk) * (2 * kImage);
        image(src);
        if (ok && pieces > 0) ok = wait_asleep(q_empty, (pieces - 1) & 1, err, 270, s_abort);
        if (!ok) break;
        mbar_arrive_expect_tx(q_full, 2 * kHalves * TT * G * 128);
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int c = 0; c < kHalves; ++c)
            tma_load_3d(sQ + x * kImage + c * kHalf, &tm_q, q_full, 64 * c, p.h * G, p.q_begin + p.tok0 + x * TT);
        ++pieces;
        image(src + kImage);
        for (int j = 1; ok && j < count; ++j) {
          image(src + j * step);
          if (ok) image(src + j * step + kImage);
        }
      }
      if (!ok) atomicExch(s_abort, 1);
    }
    __syncwarp();
  } else if (warp == kIssuer) {
    // ---------------------------------------------------------------- MMA ----
    constexpr uint32_t idesc_qk = make_idesc_bf16(kRows, kKeys);
    constexpr uint32_t idesc_pv = make_idesc_bf16(kRows, kD, false, true);
    const uint64_t q_desc = make_sdesc_k_sw128(smem_u32(sQ));
    const uint64_t k_desc = make_sdesc_k_sw128(smem_u32(sKV));
    const uint64_t v_desc = make_sdesc_mn_sw128(smem_u32(sKV), kHalf);
    auto qk = [&](int x, int e) {  // S_x = Q_x K^T of entry e
      const uint64_t k = k_desc + static_cast<uint64_t>((e % kSlots) * (kImage >> 4));
#pragma unroll
      for (int c = 0; c < kHalves; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          tc_mma_f16(tmem + kSCol + 128 * x, q_desc + static_cast<uint64_t>((x * kImage + c * kHalf + i * 32) >> 4),
                 k + static_cast<uint64_t>((c * kHalf + i * 32) >> 4), idesc_qk, (c | i) != 0 ? 1u : 0u);
      tc_commit(&s_full[x]);
    };
    // O_x += P_x V of entry e, chunk: keys 32 chunk .. + 31 of both halves
    auto pv = [&](int x, int e, int chunk, bool add) {
      const uint64_t v = v_desc + static_cast<uint64_t>((e % kSlots) * (kImage >> 4));
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int i = 4 * (k >> 1) + 2 * chunk + (k & 1);  // 16 keys = 8 columns of P
        tc_mma_f16_ta(tmem + 128 * x, tmem + kSCol + 128 * x + i * 8, v + static_cast<uint64_t>(i * (2048 >> 4)), idesc_pv,
                      add || chunk > 0 || k > 0 ? 1u : 0u);
      }
    };
    auto wait = [&](uint64_t* bar, uint32_t parity, int where) { return wait_asleep(bar, parity, err, where, s_abort); };
    bool ok = true;
    int e = 0;                // images used
    int done[2] = {0, 0};     // tiles of each row tile
    int outs[2] = {0, 0};     // pieces of each row tile
    const bool leader = elect_one();
    for (int k = 0; leader && ok && describe(k); ++k) {
      const int nx[2] = {tiles_in(p, 0), tiles_in(p, 1)}, count = max(nx[0], nx[1]);
      mbar_arrive(&d_empty[k % kAhead]);
      if (count == 0) continue;
      ok = wait(q_full, pieces & 1, 272) && wait(&full[e % kSlots], (e / kSlots) & 1, 273);
      ++pieces;
      tc_fence_after();
      if (ok) {
#pragma unroll
        for (int x = 0; x < 2; ++x)
          if (nx[x] > 0) qk(x, e);
        tc_commit(&empty[e % kSlots]);
        if (count == 1) tc_commit(q_empty);
      }
      for (int j = 0; ok && j < count; ++j, e += 2) {
        const int ev = e + 1, ek = e + 2;
        // both images of this turn first: they are here long before the weights
        ok = wait(&full[ev % kSlots], (ev / kSlots) & 1, 275);
        if (j + 1 < count) ok = ok && wait(&full[ek % kSlots], (ek / kSlots) & 1, 276);
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          if (ok && j < nx[x]) {
            // the piece before has left O
            if (j == 0 && outs[x] > 0) ok = wait(&o_free[x], (outs[x] - 1) & 1, 281);
            ok = ok && wait(&p_full[2 * x], done[x] & 1, 274);
            tc_fence_after();
            if (ok) pv(x, ev, 0, j > 0);
            ok = ok && wait(&p_full[2 * x + 1], done[x] & 1, 282);
            tc_fence_after();
            if (ok) {
              pv(x, ev, 1, true);
              tc_commit(&o_done[x]);
              if (j + 1 < nx[x]) qk(x, ek);
            }
            ++done[x];
          }
        }
        if (ok) {
          tc_commit(&empty[ev % kSlots]);
          if (j + 1 < count) tc_commit(&empty[ek % kSlots]);
          if (j + 2 == count) tc_commit(q_empty);
        }
      }
#pragma unroll
      for (int x = 0; x < 2; ++x)
        if (nx[x] > 0) ++outs[x];
    }
    if (!ok) atomicExch(s_abort, 1);
    __syncwarp();
  } else {
    // ------------------------------------------------------------- softmax ----
    // Two warps a quadrant of 32 rows, 64 keys of a tile each; a row's two threads
    // swap their maxima, which also tells that both have read their scores before
    // weights are written over them. (Neither is at the next tile's maximum before
    // the other has read this one's: its scores come after products of both threads'
    // weights.)
    const int x = warp >> 3, part = (warp >> 2) & 1, quad = warp & 3;
    const int r = 32 * quad + lane;  // this thread's row (TMEM lane)
    const uint32_t lane_base = tmem + (static_cast<uint32_t>(32 * quad) << 16);
    const uint32_t s_col = lane_base + kSCol + 128 * x, o_col = lane_base + 128 * x + kD / 2 * part;
    volatile float* mine = s_swap + ((4 * x + quad) * 2 + part) * 32 + lane;
    const volatile float* other = s_swap + ((4 * x + quad) * 2 + 1 - part) * 32 + lane;
    // Meetings of the two warps have no time limit, so both come to as many whichever
    // wait runs out for one of them: they go on to a piece together or not at all, and
    // a failed wait (ok) leaves out later waits, never a tile or a meeting.
    auto pair_sync = [&] { asm volatile("bar.sync %0, 64;" ::"r"(1 + 4 * x + quad) : "memory"); };
    auto agree = [&](bool yes) {  // a meeting that tells whether every lane of both says so
      uint32_t both;
      asm volatile(
          "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.and.pred q, %2, 64, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
          : "=r"(both)
          : "r"(static_cast<uint32_t>(yes)), "r"(1 + 4 * x + quad)
          : "memory");
      return both != 0;
    };
    const float c = a.scale * kLog2e;
    bool ok = true;
    int done = 0;
    for (int k = 0; agree(ok && __all_sync(0xffffffffu, describe(k))); ++k) {
      if (lane == 0) mbar_arrive(&d_empty[k % kAhead]);
      const int t = p.tok0 + x * TT + r / G;
      const bool live = r < TT * G && t < p.q_len;
      const int see = live ? p.keys - p.q_len + t + 1 : 1 << 30;  // keys that this row sees
      const int nx = tiles_in(p, x);
      float m = -INFINITY, l = 0.f;
      for (int j = 0; j < nx; ++j, ++done) {
        if (ok) ok = __all_sync(0xffffffffu, wait_asleep(&s_full[x], done & 1, err, 277, s_abort));
        tc_fence_after();
        uint32_t sv[64];
#pragma unroll
        for (int q = 0; q < 2; ++q)
          tmem_ld_32x32b_x32(s_col + 64 * part + 32 * q, *reinterpret_cast<uint32_t(*)[32]>(sv + 32 * q));
        tc_wait_ld();
        const int lim = see - (p.kt0 + j) * kKeys - 64 * part;
        const bool cut = __any_sync(0xffffffffu, lim < 64);  // some row does not see all of the tile
        if (cut) {
#pragma unroll
          for (int i = 0; i < 64; ++i)
            if (i >= lim) sv[i] = __float_as_uint(-INFINITY);
        }
        float m4[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) m4[q] = max_nan(__uint_as_float(sv[2 * q]), __uint_as_float(sv[2 * q + 1]));
#pragma unroll
        for (int i = 8; i < 64; i += 8) {
#pragma unroll
          for (int q = 0; q < 4; ++q)
            m4[q] = max3_nan(m4[q], __uint_as_float(sv[i + 2 * q]), __uint_as_float(sv[i + 2 * q + 1]));
        }
        const float top = max3_nan(m4[0], m4[1], max_nan(m4[2], m4[3])) * c;
        *mine = top;
        pair_sync();
        float mt = max_nan(top, *other);
        // scores that are not finite (queries are not) make the row NaN, as in the formula;
        // the weights alone would not: the polynomial takes NaN for its least argument
        if (lim + 64 * part > 0 && !(fabsf(mt) < INFINITY)) mt = NAN;
        const bool grow = !(mt <= m + kRescale);
        float alpha = 1.f;
        if (grow) {
          alpha = ex2_fast(m - mt);  // 0 on the first tile (m = -inf)
          l *= alpha;
          m = mt;
        }
        // S of this tile is there, so the products before it are complete: O may be
        // read and written (tcgen05.ld / st take whole warps)
        if (__any_sync(0xffffffffu, grow) && j > 0) {
#pragma unroll 1
          for (int q = 0; q < kD / 32; ++q) {
            uint32_t ov[16];
            tmem_ld_32x32b_x16(o_col + 16 * q, ov);
            tc_wait_ld();
#pragma unroll
            for (int i = 0; i < 16; ++i) ov[i] = __float_as_uint(__uint_as_float(ov[i]) * alpha);
            tmem_st_32x32b_x16(o_col + 16 * q, ov);
          }
        }
        // a row that has seen no key yet has m = -inf and weights of 0
        const float base = m == -INFINITY ? 0.f : m;
        const uint64_t c2 = f2_pack(c, c), neg = f2_pack(-base, -base);
        uint64_t sum[2] = {f2_pack(0.f, 0.f), f2_pack(0.f, 0.f)};
#pragma unroll
        for (int chunk = 0; chunk < 2; ++chunk) {
          uint32_t pk[16];
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            const int i = 16 * chunk + k;
            const uint64_t x2 = f2_fma(f2_pack(__uint_as_float(sv[2 * i]), __uint_as_float(sv[2 * i + 1])), c2, neg);
            float lo, hi;
            if ((i % 8) < kPolyPairs) {
              exp2_poly_pair(x2, lo, hi);
              // its least weight is 2^-126; a hidden key's is 0
              if (cut) lo = 2 * i < lim ? lo : 0.f, hi = 2 * i + 1 < lim ? hi : 0.f;
            } else {
              float y0, y1;
              f2_unpack(x2, y0, y1);
              lo = ex2_fast(y0), hi = ex2_fast(y1);
            }
            sum[i & 1] = f2_add(sum[i & 1], f2_pack(lo, hi));
            pk[k] = pack_bf16x2(lo, hi);
          }
          tmem_st_32x32b_x16(s_col + 32 * part + 16 * chunk, pk);
          tc_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_full[2 * x + chunk]);
        }
        float s0, s1;
        f2_unpack(f2_add(sum[0], sum[1]), s0, s1);
        l += s0 + s1;
      }
      // ---------------------------------------------------------- epilogue ----
      if (ok && nx > 0) ok = __all_sync(0xffffffffu, wait_asleep(&o_done[x], (done - 1) & 1, err, 278, s_abort));
      tc_fence_after();
      // the row's sum over both halves of the keys
      pair_sync();
      *mine = l;
      pair_sync();
      l += *other;
      uint32_t ov[kD / 2] = {};
      if (ok && nx > 0) {
#pragma unroll
        for (int q = 0; q < kHalves; ++q) tmem_ld_32x32b_x32(o_col + 32 * q, *reinterpret_cast<uint32_t(*)[32]>(ov + 32 * q));
        tc_wait_ld();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&o_free[x]);  // the next piece's products may begin
      }
      if (p.whole) {
        const float inv = l > 0.f ? 1.f / l : l;  // no key: zeros; NaN stays
        // four lanes swap vectors, so that a store has 64 bytes of a row side by
        // side (of 16 bytes a row each they took the load-store unit 4000 cycles a piece)
        const int64_t row = live ? static_cast<int64_t>(p.q_begin + t) * a.hq + p.h * G + r % G : -1;
#pragma unroll
        for (int q = 0; q < kHalves; ++q) {
          uint4 v[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t* o = ov + 32 * q + 8 * i;
            v[i].x = pack_bf16x2(__uint_as_float(o[0]) * inv, __uint_as_float(o[1]) * inv);
            v[i].y = pack_bf16x2(__uint_as_float(o[2]) * inv, __uint_as_float(o[3]) * inv);
            v[i].z = pack_bf16x2(__uint_as_float(o[4]) * inv, __uint_as_float(o[5]) * inv);
            v[i].w = pack_bf16x2(__uint_as_float(o[6]) * inv, __uint_as_float(o[7]) * inv);
          }
          transpose4(v, lane);
#pragma unroll
          for (int i = 0; i < 4; ++i) {  // of the row of lane (lane & ~3) + i
            const int64_t to = __shfl_sync(0xffffffffu, row, (lane & ~3) + i);
            if (to >= 0)
              reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(a.out) + to * kD + kD / 2 * part + 32 * q)[lane & 3] = v[i];
          }
        }
      } else {
        // a record of the part: the run's first piece in slot 0 unless the pair begins with it
        // (vectors of four dims, a warp's rows side by side)
        const int64_t rec = 2 * static_cast<int>(blockIdx.x) + (p.kt0 == 0 ? 1 : 0);
        if (part == 0) *reinterpret_cast<float2*>(a.part_ml + 2 * (rec * (2 * kRows) + x * kRows + r)) = make_float2(m, l);
        uint4* dst = reinterpret_cast<uint4*>(a.part_o + rec * (2 * kRows) * kD) + ((4 * x + quad) * (kD / 4) + kD / 8 * part) * 32 + lane;
#pragma unroll
        for (int i = 0; i < kD / 8; ++i) dst[32 * i] = make_uint4(ov[4 * i], ov[4 * i + 1], ov[4 * i + 2], ov[4 * i + 3]);
      }
    }
    if (!ok && lane == 0) atomicExch(s_abort, 1);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kLoader && lane == 0 && *reinterpret_cast<volatile int*>(s_abort)) {
    // after an abort, copies still in flight land before the CTA leaves
    if (pieces > 0) mbar_wait(q_full, (pieces - 1) & 1, err, 279);
    for (int i = max(0, issued - kSlots); i < issued; ++i) mbar_wait(&full[i % kSlots], (i / kSlots) & 1, err, 280);
  }
  if (warp == kIssuer) {
    tc_fence_after();
    tmem_dealloc(*tmem_slot, 512);
  }
}

// Joins the records of the pair that CTA blockIdx.x began and others went on
// with: a lane a row, four dims of 32 rows a warp.
template <int kD>
__global__ void __launch_bounds__(256) kv4_prefill_join_kernel(const __grid_constant__ Kv4PrefillArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  const int4 d = reinterpret_cast<const int4*>(a.desc)[blockIdx.x];
  if (d.x < 0) return;
  const int lane = threadIdx.x & 31;
  const int block = blockIdx.y / (kD / 32), vec = blockIdx.y % (kD / 32) * 8 + (threadIdx.x >> 5);  // 32 rows, 4 dims
  const int G = a.group, TT = kRows / G, row = 32 * block + lane, r = row % kRows;
  const int t = d.z * 2 * TT + row / kRows * TT + r / G;
  if (r >= TT * G || t >= kv4_query_tokens(a.cu_q, d.y, a.T)) return;
  const int begin = blockIdx.x;
  auto rec_of = [&](int i) { return static_cast<int64_t>(2 * i + (i == begin ? 1 : 0)) * (2 * kRows); };
  float top = -INFINITY;
  for (int i = begin; i <= d.x; ++i) top = fmaxf(top, a.part_ml[2 * (rec_of(i) + row)]);
  float l = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int i = begin; i <= d.x; ++i) {
    const int64_t rec = rec_of(i);
    const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + 2 * (rec + row));
    const float4 v = reinterpret_cast<const float4*>(a.part_o + rec * kD)[(block * (kD / 4) + vec) * 32 + lane];
    const float f = ml.x == -INFINITY ? 0.f : ex2_fast(ml.x - top);  // no key of the row there
    l += ml.y * f;
    acc[0] += v.x * f, acc[1] += v.y * f, acc[2] += v.z * f, acc[3] += v.w * f;
  }
  const float inv = l > 0.f ? 1.f / l : l;
  uint2* dst = reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(a.out) +
                                        (static_cast<int64_t>(a.cu_q[d.y] + t) * a.hq + d.w * G + r % G) * kD);
  dst[vec] = make_uint2(pack_bf16x2(acc[0] * inv, acc[1] * inv), pack_bf16x2(acc[2] * inv, acc[3] * inv));
}

template <int kD>
void launch_typed(const Kv4PrefillArgs& a, cudaStream_t s) {
  constexpr int kSmem = smem_bytes<kD>();
  static bool done[64] = {};  // per device
  int dev = 0;
  cudaGetDevice(&dev);
  if (!done[dev & 63]) {
    if (cudaFuncSetAttribute(kv4_prefill_kernel<kD>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem) != cudaSuccess)
      throw std::runtime_error("minisgl.prefill_attention_kv4: shared memory limit");
    done[dev & 63] = true;
  }
  const int TT = kRows / a.group;
  // query rows of one token tile: [token, head of a group, 64 dims]
  const uint64_t dims[3] = {kD, static_cast<uint64_t>(a.hq), static_cast<uint64_t>(a.T)};
  const uint64_t strides[2] = {kD * 2, static_cast<uint64_t>(a.ld_q) * 2};
  const uint32_t box[3] = {64, static_cast<uint32_t>(a.group), static_cast<uint32_t>(TT)};
  const CUtensorMap tq = make_tmap(a.q, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, 3, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
  launch_pdl(kv4_prefill_kernel<kD>, dim3(a.ctas), dim3(kThreads), kSmem, s, tq, a);
  launch_pdl(kv4_prefill_join_kernel<kD>, dim3(a.ctas, 2 * kRows / 32 * (kD / 32)), dim3(256), 0, s, a);
}

}  // namespace

bool kv4_prefill_takes(int d, int group) { return (d == 64 || d == 128) && group >= 1 && group <= kRows; }

void launch_kv4_prefill(const Kv4PrefillArgs& a, cudaStream_t s) {
  if (a.B <= 0 || a.T <= 0) return;
  if (a.d == 128) launch_typed<128>(a, s);
  else if (a.d == 64) launch_typed<64>(a, s);
  else throw std::runtime_error("minisgl.prefill_attention_kv4: head_dim must be 64 or 128");
}

}  // namespace minisgl
