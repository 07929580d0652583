// Attention of few query rows over the 4-bit paged KV cache: one token per
// request (decode) or a few at its end (drafted tokens, short extends).
//
//   o_r = sum_j p_rj v_j / sum_j p_rj,  p_rj = 2^((q_r . k_j - m_r) c),  c = scale log2 e,
//
// with k_j and v_j in 4-bit codes, 136 bytes of cache per token and 128-dim
// head. Bound by what a warp has to do per code, on the integer and half2 pipes:
// 256 requests of up to 4096 keys and 8 KV heads take 139 us in bursts (a graph of
// 20 calls, the best of five), 4.2 TB/s (64 % of the copy rate), and 150 in a stream
// of calls (59 %), one of 131072 keys 46 us. Everything is laid out to keep that
// small:
//
// * The products are taken the other way round, S^T = K q^T and O^T = V^T P^T
//   (warp-level m16n8k16 MMA): keys and dims fill the 16 rows of A, and the query
//   rows, 8 at a time, are the 8 columns of B, so nothing is wasted on padding for
//   groups of up to 8 heads. tcgen05 would need 128 rows, and the codes written
//   out to shared memory.
// * The cache's byte order is the A fragments' order: a lane's 16 bytes from
//   shared memory are the codes of two MMAs (K) or four (V).
// * K: the bits of a code c, where they stand, are the fp16 number c 2^-24 (or
//   16 c 2^-24 four bits up): a mask makes a pair, with no exponent to set. q is
//   taken to fp16 by a power of two for each row, odd dims with 1/16 of it. The 8
//   that codes are above their values is a product of its own: a group's scale
//   with -8 sum(q) of its dims, in three bf16 parts. A group's scale multiplies
//   its four sums. (256 requests took 172 us at that stage; with bf16 numbers
//   128 + c, whose exponents have to be set, 173; with 8-bit floats, which the
//   warp-level MMA converts first, 205.)
// * V: 128 + c has the bf16 bits 0x4300 | c, and s (128 + c) - 136 s is one packed
//   fused multiply-add, exact in bf16.
// * The running maximum moves only when a score exceeds it by 8 (in powers of
//   two); other tiles neither reduce over lanes nor rescale the output.
// * Weights p are rounded to bf16, as V is held; their sum is of fp32 weights.
//
// A CTA, one an SM, is three groups of four warps, 32 keys of a tile each, and a
// warp for each group that fetches its tiles by bulk copies, page numbers a tile
// ahead: those take few registers, so the launch's 128 a thread are dealt anew
// (152 and 56). Without the split, eight warps at a time: 164 us instead of 140;
// sixteen of 112 registers: 144. Four CTAs of one group, which fetches for
// itself: 188.
//
// Work is split evenly whatever the lengths are: all key tiles of all requests,
// heads and row tiles form one sequence, with two places more for each unit of them
// (what a piece costs beside its tiles), of which each group of warps takes an
// equal run. A run's first and last pieces may be parts of a longer one: those
// write (m, l, O) records, which a second small kernel joins.
#include <stdexcept>

#include "kv4.cuh"
#include "launch.h"
#include "ops.h"

namespace minisgl {
namespace {

using bf16 = __nv_bfloat16;

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kWarps = 4;                          // each takes 32 keys of a tile
constexpr int kTile = 32 * kWarps;                 // keys per tile
constexpr int kRows = 8;                           // query rows per tile
constexpr int kGroups = 3;                         // of kWarps warps in a CTA, one CTA per SM
constexpr int kThreads = (kGroups + 1) * kWarps * 32;  // and a warp that fetches for each of them
constexpr int kStages = 3;
// registers: 16 warps are launched with 128; the last four, of which three fetch,
// give up theirs to the others
constexpr int kRegs = 152, kFetchRegs = 56;
static_assert(kGroups == 3 && kWarps == 4 && 12 * kRegs + 4 * kFetchRegs == 16 * 128, "register split");
constexpr float kFloor = -1e30f;                   // maximum of a row that has seen no key

__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// d = a b
__device__ __forceinline__ void mma_bf16_zero(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void mma_f16_zero(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
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
// Bytes of one stage: the K blocks of a tile, its V blocks and, where a piece
// begins, the query rows (16 bytes apart from multiples of 128: no bank twice).
template <int D>
constexpr int half_bytes() { return kTile * kv4::row_bytes(D); }
template <int D>
constexpr int q_pitch() { return 2 * D + 16; }
template <int D>
constexpr int stage_bytes() { return 2 * half_bytes<D>() + kRows * q_pitch<D>(); }
constexpr int kLd = 64 + 4;  // padded row of the merge buffer (floats): 64 dims at a time

template <int D>
constexpr int group_bytes() {
  return (kStages * stage_bytes<D>() + kWarps * kRows * (kLd + 2) * 4 + 16 * D + D + 2 * kStages * 8 + 127) / 128 * 128;
}

// Query rows (tokens x heads of a group) and keys of a request.
template <bool kSingle>
__device__ __forceinline__ int rows_of(const Kv4AttnArgs& a, int b) {
  return kSingle ? a.group : kv4_query_tokens(a.cu_q, b, a.T) * a.group;
}
__device__ __forceinline__ int key_tiles(int keys) { return max(1, (keys + kTile - 1) / kTile); }

constexpr int kUnitCost = kKv4UnitCost;

// A place in the work: request, unit of it (KV head x row tile) and key tile.
struct Place {
  int b, unit, kt;
};

__device__ __forceinline__ void group_sync(int group) {
  asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "n"(kWarps * 32) : "memory");
}
// A wait that sleeps: the first try may suspend the thread for 20 us, so that it
// leaves the issue slots to the others. The bounded loop follows.
__device__ __forceinline__ bool wait_slow(uint64_t* bar, uint32_t parity, int* flag, int where) {
  return mbar_wait(bar, parity, ErrorSink{flag}, where);
}
__device__ __forceinline__ bool wait_for(uint64_t* bar, uint32_t parity, int* flag, int where) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, 20000;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0 || wait_slow(bar, parity, flag, where);
}

// kSingle: one query token per request (row r of a KV head is its head r).
template <int D, bool kSingle>
__global__ void __launch_bounds__(kThreads, 1) kv4_attn_kernel(const __grid_constant__ Kv4AttnArgs a) {
  extern __shared__ __align__(128) uint8_t smem[];
  constexpr int kNG = D / kv4::kGroup;    // scale groups of a row
  constexpr int kHalves = D / 64;         // 64-dim halves of V
  constexpr int kHalf = half_bytes<D>();
  constexpr int kStage = stage_bytes<D>();
  constexpr int kPitch = q_pitch<D>();
  const ErrorSink err{a.err};
  const int warp = (threadIdx.x >> 5) % kWarps, lane = threadIdx.x & 31;
  const bool fetches = threadIdx.x >= kGroups * kWarps * 32;
  const int group = fetches ? min((static_cast<int>(threadIdx.x) >> 5) - kGroups * kWarps, kGroups - 1) : (threadIdx.x >> 5) / kWarps;
  const bool idle = threadIdx.x >= kGroups * (kWarps + 1) * 32;
  uint8_t* ring = smem + group * group_bytes<D>();
  float* so = reinterpret_cast<float*>(ring + kStages * kStage);  // [warps][rows][kLd]
  float* sm = so + kWarps * kRows * kLd;                          // [warps][rows]
  float* sl = sm + kWarps * kRows;
  uint4* sq = reinterpret_cast<uint4*>(sl + kWarps * kRows);  // [kNG][32 lanes] query fragments of the piece
  float* ssum = reinterpret_cast<float*>(sq + kNG * 32);        // [kNG][rows] -8 times their groups' sums
  uint64_t* full = reinterpret_cast<uint64_t*>(ssum + kNG * kRows);
  uint64_t* empty = full + kStages;
  int* pre = reinterpret_cast<int*>(smem + kGroups * group_bytes<D>());  // [B + 1] sums of places
  int* units = pre + a.B + 1;                                            // [B + 1] sums of units
  int* len = units + a.B + 1;                                            // [B] keys
  int* pt_row = len + a.B;                                               // [B] page-table rows (-1: outside)

  pdl_launch_dependents();
  if (fetches && !idle && lane == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], kWarps);
    }
    fence_barrier_init();
  }
  pdl_wait();
  bool falls = false;
  for (int b = threadIdx.x; b < a.B; b += kThreads) {
    const int keys = kv4_keys(a.seq_lens, b, a.ld_pt);
    if constexpr (!kSingle) falls = falls || kv4_offsets_fall(a.cu_q, b);
    len[b] = keys;
    const int row = a.req_rows[b];
    const bool row_ok = row >= 0 && row < a.pt_rows;
    pt_row[b] = row_ok ? row : -1;
    if (blockIdx.x == 0 && (!row_ok || a.seq_lens[b] > a.ld_pt)) err.report(kErrBadIndex, row_ok ? 962 : 961);
    const int n = (rows_of<kSingle>(a, b) + kRows - 1) / kRows * a.hk;
    units[b + 1] = n, pre[b + 1] = n * (kUnitCost + key_tiles(keys));
    if (!kSingle && blockIdx.x == 0 && (a.cu_q[b] < 0 || a.cu_q[b + 1] > a.T || a.cu_q[b + 1] < a.cu_q[b]))
      err.report(kErrBadIndex, 964);
  }
  const bool none = __syncthreads_or(falls) != 0;
  if (threadIdx.x < 64) {
    int* x = threadIdx.x < 32 ? pre : units;
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
  // equal runs for the groups of all CTAs (CTA by CTA in the last place, so that
  // few runs use every SM). Each has a place at least, so the runs that a unit's
  // tiles span all have some of them, and their records are all written.
  const int total = none ? 0 : pre[a.B];
  const int n = max(1, min(kGroups * static_cast<int>(gridDim.x), total)), me = group * gridDim.x + blockIdx.x;
  const int each = total / n, more = total - each * n;  // places of a run; the runs share `more` others
  auto start_of = [&](int i) { return each * i + more * i / n; };  // of run i: total i / n without 64 bits
  auto find = [&](int v, Place& p) {  // the place and how many tiles are before it
    if (v >= total) return pre[a.B] - kUnitCost * units[a.B];
    p.b = 0;  // the last request with pre[b] <= v
    for (int step = a.pow2; step > 0; step /= 2)
      if (p.b + step < a.B && pre[p.b + step] <= v) p.b += step;
    const int per = kUnitCost + key_tiles(len[p.b]), in = v - pre[p.b];
    p.unit = in / per;
    p.kt = max(0, in - p.unit * per - kUnitCost);
    return pre[p.b] - kUnitCost * units[p.b] + p.unit * (per - kUnitCost) + p.kt;
  };
  Place at{0, 0, 0};
  int count = 0;  // tiles of this run
  if (me < n && total > 0) {
    Place end;
    count = find(start_of(me + 1), end);
    count -= find(start_of(me), at);
  }

  const int seg = min(a.page_size, kTile);  // keys that are side by side in the cache
  const int segs = kTile / seg;
  const int seg_bytes = seg * kv4::row_bytes(D);

  if (fetches) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kFetchRegs));
    if (idle) return;
    // ---- tiles of the run into the ring, page numbers read a tile ahead
    if (lane == 0) reinterpret_cast<int4*>(a.desc)[me] = make_int4(-1, 0, 0, 0);
    int b = at.b, kt = at.kt, kts = 0, unit = at.unit, left = 0, keys = 0, rows = 0, tile_rows = 1, h = 0;
    const int32_t* pt = a.page_table;
    bool row_ok = true;
    auto begin = [&] {  // request b
      keys = len[b], kts = key_tiles(keys);
      rows = rows_of<kSingle>(a, b);
      tile_rows = (rows + kRows - 1) / kRows;
      left = units[b + 1] - units[b];
      const int row = pt_row[b];
      row_ok = row >= 0;
      pt = a.page_table + static_cast<int64_t>(max(row, 0)) * a.ld_pt;
    };
    auto page_of = [&] { return lane < segs && kt * kTile + lane * seg < keys && row_ok ? pt[kt * kTile + lane * seg] : -1; };
    int slot = -1, issued = -1;
    if (count > 0) begin(), h = unit / tile_rows, slot = page_of();
    for (int j = 0; j < count; ++j) {
      // this tile's copies, from what was looked up
      const bool wanted = lane < segs && kt * kTile + lane * seg < keys && row_ok;
      const bool good = wanted && slot >= 0 && slot < a.kv_slots;
      const int64_t block = (static_cast<int64_t>(slot >> a.page_shift) * a.hk + h) * a.page_size * kv4::row_bytes(D);
      const int off = slot & (a.page_size - 1) & ~(kTile - 1);
      const bf16* q = nullptr;
      if (kt == 0 || j == 0) {  // the piece's query rows
        const int r = (unit - h * tile_rows) * kRows + lane;
        if (lane < kRows && r < rows) {
          const int tok = kSingle ? 0 : r / a.group;
          q = static_cast<const bf16*>(a.q) + static_cast<int64_t>((kSingle ? b : a.cu_q[b]) + tok) * a.ld_q +
              (h * a.group + r - tok * a.group) * D;
        }
      }
      // the next tile's page numbers
      if (++kt == kts && j + 1 < count) {
        kt = 0;
        if (++unit == left) {
          unit = 0;
          do ++b; while (units[b + 1] == units[b]);  // past requests without queries: there is more to do
          begin();
        }
        h = tile_rows == 1 ? unit : unit / tile_rows;
      }
      slot = j + 1 < count ? page_of() : -1;

      if (wanted && !good) err.report(kErrBadIndex, 963);
      const int bytes = 2 * __popc(__ballot_sync(0xffffffffu, good)) * seg_bytes +
                        __popc(__ballot_sync(0xffffffffu, q != nullptr)) * 2 * D;
      const int s = j % kStages;
      if (j >= kStages && !wait_for(&empty[s], (j / kStages - 1) & 1u, a.err, 260)) break;
      if (lane == 0) mbar_arrive_expect_tx(&full[s], bytes);
      __syncwarp();
      uint8_t* st = ring + s * kStage;
      if (good) {
        uint8_t* dst = st + lane * seg_bytes;
        if (seg == a.page_size) {
          bulk_load(dst, a.k_pool + block, seg_bytes, &full[s]);
          bulk_load(dst + kHalf, a.v_pool + block, seg_bytes, &full[s]);
        } else {  // part of a larger page: its codes and its scales
          const int64_t codes = block + off * (D / 2);
          const int64_t scales = block + a.page_size * (D / 2) + off * kNG;
          bulk_load(dst, a.k_pool + codes, kTile * (D / 2), &full[s]);
          bulk_load(dst + kTile * (D / 2), a.k_pool + scales, kTile * kNG, &full[s]);
          bulk_load(dst + kHalf, a.v_pool + codes, kTile * (D / 2), &full[s]);
          bulk_load(dst + kHalf + kTile * (D / 2), a.v_pool + scales, kTile * kNG, &full[s]);
        }
      }
      if (q != nullptr) bulk_load(st + 2 * kHalf + lane * kPitch, q, 2 * D, &full[s]);
      issued = j;
    }
    // copies in flight land before the CTA's shared memory is given back
    for (int j = max(0, issued - kStages + 1); j <= issued; ++j)
      if (!wait_for(&full[j % kStages], (j / kStages) & 1u, a.err, 261)) break;
    return;
  }

  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegs));
  const int g = lane >> 2, t = lane & 3;
  const float c = a.scale * kLog2e;
  // this lane's keys of the warp's first 16 (rows g and g + 8 of S^T are keys
  // key0 and key0 + 2), the segment they lie in and the places of its codes and
  // scales there; the second 16 keys are a constant distance away
  const int key0 = warp * 32 + 4 * (g >> 1) + (g & 1);
  int k_at[2], ks_at[2], v_at[2], vs_at[2];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int base = warp * 32 + u * 16;
    const int seg_at = base / seg * seg_bytes, in_seg = base & (seg - 1);
    const int key_in = in_seg + 4 * (g >> 1) + (g & 1), quad_in = in_seg / 4 + t;
    k_at[u] = seg_at + key_in * (D / 2) + t * (D / 8);
    ks_at[u] = seg_at + seg * (D / 2) + key_in * kNG;
    v_at[u] = kHalf + seg_at + quad_in * (2 * D) + ((g ^ (2 * t)) * 16);
    vs_at[u] = kHalf + seg_at + seg * (D / 2) + (quad_in * kNG + (g >> 2)) * 4;
  }
  int left = count, s = 0;
  uint32_t phase = 0;
  bool ok = true;

  while (left > 0) {
    // ---- the next piece: key tiles [kt0, kt1) of kts of the unit `at`
    while (at.unit == units[at.b + 1] - units[at.b]) at.unit = 0, ++at.b;
    const int keys = len[at.b], kts = key_tiles(keys);
    const int kt0 = at.kt, kt1 = min(kts, kt0 + left);
    const int rows = rows_of<kSingle>(a, at.b), tile_rows = (rows + kRows - 1) / kRows;
    const int h = tile_rows == 1 ? at.unit : at.unit / tile_rows, rt = at.unit - h * tile_rows;
    left -= kt1 - kt0;
    // keys that rows 2 t and 2 t + 1 see, and that every row of the tile sees
    int see0 = keys, see1 = keys, see_all = keys;
    if constexpr (!kSingle) {
      const int q_len = rows / a.group, r0 = rt * kRows + 2 * t;
      see0 = keys - q_len + r0 / a.group + 1;
      see1 = keys - q_len + (r0 + 1) / a.group + 1;
      see_all = keys - q_len + rt * kRows / a.group + 1;
    }
    uint32_t off0, off1;
    float o[2 * kNG][4];
#pragma unroll
    for (int i = 0; i < 2 * kNG; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    float m0 = kFloor, m1 = kFloor, l0 = 0.f, l1 = 0.f, c0 = 0.f, c1 = 0.f;

    for (int kt = kt0; kt < kt1; ++kt) {
      const uint8_t* st = ring + s * kStage;
      if (ok) ok = wait_for(&full[s], phase, a.err, 262);
      if (kt == kt0) {
        // Query fragments in fp16, row g by the lanes g: q 2^-x, 2^x the power of two
        // that takes the row's largest to 2^14..2^15, which keeps the 8 bits of every
        // element within 2^-18 of it; odd dims are divided by 16, because their codes
        // are taken from where they stand, 4 bits up. And -8 times the groups' sums.
        // Warp i writes group i for all four.
        const bool live = rt * kRows + g < rows;
        uint4 v[kNG];
        float top = 0.f;
        bool finite = true;
#pragma unroll
        for (int i = 0; i < kNG; ++i) {
          v[i] = *reinterpret_cast<const uint4*>(st + 2 * kHalf + g * kPitch + 64 * i + 16 * t);
          if (!live) v[i] = make_uint4(0, 0, 0, 0);
          const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float x = __uint_as_float(w[j] << 16), y = __uint_as_float(w[j] & 0xffff0000u);
            top = fmaxf(top, fmaxf(fabsf(x), fabsf(y)));
            finite = finite && x == x && y == y;
          }
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int ex = max(static_cast<int>(__float_as_uint(top) >> 23), 24);
        // an infinity or a NaN makes the row NaN, as it does in the formula
        const float down = finite && ex < 255 ? __uint_as_float((268 - ex) << 23) : NAN;
        const float up = c * 16777216.f * __uint_as_float((min(ex, 254) - 14) << 23);
        c0 = __shfl_sync(0xffffffffu, up, 8 * t);      // of row 2 t
        c1 = __shfl_sync(0xffffffffu, up, 8 * t + 4);  // of row 2 t + 1
        if (warp < kNG) {
          uint4 mine = v[0];
#pragma unroll
          for (int i = 1; i < kNG; ++i)
            if (warp == i) mine = v[i];
          const uint32_t w[4] = {mine.x, mine.y, mine.z, mine.w};
          // dims 0..7 of the word -> (0, 4), (1, 5), (2, 6), (3, 7)
          float z[8], sum = 0.f;
          uint32_t q[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            z[2 * j] = __uint_as_float(w[j] << 16) * down, z[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u) * down;
            sum += z[2 * j] + z[2 * j + 1];
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float f = j & 1 ? 0.0625f : 1.f;
            const __half2 hh = __floats2half2_rn(z[j] * f, z[j + 4] * f);
            q[j] = *reinterpret_cast<const uint32_t*>(&hh);
          }
          sum += __shfl_xor_sync(0xffffffffu, sum, 1);
          sum += __shfl_xor_sync(0xffffffffu, sum, 2);
          sq[warp * 32 + lane] = make_uint4(q[0], q[1], q[2], q[3]);
          if (t == 0) ssum[warp * kRows + g] = sum * (-8.f / 16777216.f);  // codes are c 2^-24
        }
        group_sync(group);
        // the sums in three bf16 parts: D = 128: lanes t take groups t % 2 and t % 2 + 2
        const float x = ssum[(D == 128 ? t & 1 : 0) * kRows + g], y = ssum[(D == 128 ? 2 + (t & 1) : 1) * kRows + g];
        const uint32_t hi = pack_bf16x2(x, y);
        const float x1 = x - __uint_as_float(hi << 16), y1 = y - __uint_as_float(hi & 0xffff0000u);
        const uint32_t mid = pack_bf16x2(x1, y1);
        const uint32_t lo = pack_bf16x2(x1 - __uint_as_float(mid << 16), y1 - __uint_as_float(mid & 0xffff0000u));
        if constexpr (D == 128) {
          off0 = t < 2 ? hi : mid, off1 = t < 2 ? lo : 0u;
        } else {
          off0 = t == 0 ? hi : t == 1 ? mid : t == 2 ? lo : 0u, off1 = 0u;
        }
      }
      if (kt * kTile + warp * 32 < keys) {  // some key of the warp's is there
        // ---- S^T of 2 x 16 keys x 8 rows
        float sc[2][4];
        uint32_t w0[2][kNG], w1[2][kNG];  // words of keys key0 and key0 + 2
        float f0[2][kNG], f1[2][kNG];     // and their scales
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          uint32_t s0, s1;
          if constexpr (D == 128) {
            *reinterpret_cast<uint4*>(w0[u]) = *reinterpret_cast<const uint4*>(st + k_at[u]);
            *reinterpret_cast<uint4*>(w1[u]) = *reinterpret_cast<const uint4*>(st + k_at[u] + D);
            s0 = *reinterpret_cast<const uint32_t*>(st + ks_at[u]);
            s1 = *reinterpret_cast<const uint32_t*>(st + ks_at[u] + 2 * kNG);
          } else {
            *reinterpret_cast<uint2*>(w0[u]) = *reinterpret_cast<const uint2*>(st + k_at[u]);
            *reinterpret_cast<uint2*>(w1[u]) = *reinterpret_cast<const uint2*>(st + k_at[u] + D);
            s0 = *reinterpret_cast<const uint16_t*>(st + ks_at[u]);
            s1 = *reinterpret_cast<const uint16_t*>(st + ks_at[u] + 2 * kNG);
          }
          // the scales as bf16 pairs (groups 0 and 2, 1 and 3; D = 64: 0 and 1)
          uint32_t e0, e1, d0, d1;
          if constexpr (D == 128) {
            e0 = (s0 & 0x00ff00ffu) * 16 + kv4::kScaleBf16x2, d0 = __byte_perm(s0, 0, 0x4341) * 16 + kv4::kScaleBf16x2;
            e1 = (s1 & 0x00ff00ffu) * 16 + kv4::kScaleBf16x2, d1 = __byte_perm(s1, 0, 0x4341) * 16 + kv4::kScaleBf16x2;
            f0[u][0] = __uint_as_float(e0 << 16), f0[u][2] = __uint_as_float(e0 & 0xffff0000u);
            f0[u][1] = __uint_as_float(d0 << 16), f0[u][3] = __uint_as_float(d0 & 0xffff0000u);
            f1[u][0] = __uint_as_float(e1 << 16), f1[u][2] = __uint_as_float(e1 & 0xffff0000u);
            f1[u][1] = __uint_as_float(d1 << 16), f1[u][3] = __uint_as_float(d1 & 0xffff0000u);
            if (t & 1) e0 = d0, e1 = d1;
          } else {
            e0 = __byte_perm(s0, 0, 0x4140) * 16 + kv4::kScaleBf16x2;
            e1 = __byte_perm(s1, 0, 0x4140) * 16 + kv4::kScaleBf16x2;
            f0[u][0] = __uint_as_float(e0 << 16), f0[u][1] = __uint_as_float(e0 & 0xffff0000u);
            f1[u][0] = __uint_as_float(e1 << 16), f1[u][1] = __uint_as_float(e1 & 0xffff0000u);
          }
          const uint32_t po[4] = {e0, e1, e0, e1};
          mma_bf16_zero(sc[u], po, off0, off1);
        }
#pragma unroll
        for (int i = 0; i < kNG; ++i) {
          const uint4 q = sq[i * 32 + lane];
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            float acc[4];
            // codes as they stand, c or 16 c, are fp16 numbers c 2^-24 and c 2^-20
            const uint32_t x[4] = {w0[u][i] & 0x000f000fu, w1[u][i] & 0x000f000fu, w0[u][i] & 0x00f000f0u, w1[u][i] & 0x00f000f0u};
            mma_f16_zero(acc, x, q.x, q.y);
            const uint32_t z0 = w0[u][i] >> 8, z1 = w1[u][i] >> 8;
            const uint32_t y[4] = {z0 & 0x000f000fu, z1 & 0x000f000fu, z0 & 0x00f000f0u, z1 & 0x00f000f0u};
            mma_f16(acc, y, q.z, q.w);
            sc[u][0] += acc[0] * f0[u][i], sc[u][1] += acc[1] * f0[u][i];
            sc[u][2] += acc[2] * f1[u][i], sc[u][3] += acc[3] * f1[u][i];
          }
        }
        if ((kt + 1) * kTile > see_all) {  // uniform over the CTA
          const int pos = kt * kTile + key0;
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            if (pos + 16 * u >= see0) sc[u][0] = -INFINITY;
            if (pos + 16 * u >= see1) sc[u][1] = -INFINITY;
            if (pos + 16 * u + 2 >= see0) sc[u][2] = -INFINITY;
            if (pos + 16 * u + 2 >= see1) sc[u][3] = -INFINITY;
          }
        }
        // ---- running maximum (of the scores in powers of two)
        {
          float x0 = fmaxf(fmaxf(sc[0][0], sc[0][2]), fmaxf(sc[1][0], sc[1][2])) * c0;
          float x1 = fmaxf(fmaxf(sc[0][1], sc[0][3]), fmaxf(sc[1][1], sc[1][3])) * c1;
          if (__any_sync(0xffffffffu, x0 > m0 + 8.f || x1 > m1 + 8.f)) {
#pragma unroll
            for (int sh = 4; sh < 32; sh *= 2) {
              x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, sh));
              x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, sh));
            }
            const float n0 = fmaxf(m0, x0), n1 = fmaxf(m1, x1);
            const float f0 = exp2_approx(m0 - n0), f1 = exp2_approx(m1 - n1);
            m0 = n0, m1 = n1;
            l0 *= f0, l1 *= f1;
#pragma unroll
            for (int i = 0; i < 2 * kNG; ++i) o[i][0] *= f0, o[i][1] *= f1, o[i][2] *= f0, o[i][3] *= f1;
          }
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const float p0 = exp2_approx(fmaf(sc[u][0], c0, -m0)), p1 = exp2_approx(fmaf(sc[u][1], c1, -m1));
          const float p2 = exp2_approx(fmaf(sc[u][2], c0, -m0)), p3 = exp2_approx(fmaf(sc[u][3], c1, -m1));
          l0 += p0 + p2, l1 += p1 + p3;
          const uint32_t b0 = transpose8x8(pack_bf16x2(p0, p1));
          const uint32_t b1 = transpose8x8(pack_bf16x2(p2, p3));
          // ---- O^T += V^T P^T
#pragma unroll
          for (int hf = 0; hf < kHalves; ++hf) {
            const uint4 v4 = *reinterpret_cast<const uint4*>(st + v_at[u] + hf * 128);
            const uint32_t w[4] = {v4.x, v4.y, v4.z, v4.w};
            const uint32_t sv = *reinterpret_cast<const uint32_t*>(st + vs_at[u] + hf * 8);
            const uint32_t sa = (sv & 0x00ff00ffu) * 16 + kv4::kScaleBf16x2;         // tokens 0 and 1
            const uint32_t sb = __byte_perm(sv, 0, 0x4341) * 16 + kv4::kScaleBf16x2;  // tokens 2 and 3
            const uint32_t oa = mul_pair(sa, 0xc308c308u), ob = mul_pair(sb, 0xc308c308u);  // times -136
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const uint32_t x[4] = {fma_pair(code_pair(w[j]), sa, oa), fma_pair(code_pair(w[j] >> 4), sa, oa),
                                     fma_pair(code_pair(w[j] >> 8), sb, ob), fma_pair(code_pair(w[j] >> 12), sb, ob)};
              mma_bf16(o[4 * hf + j], x, b0, b1);
            }
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[s]);
      if (++s == kStages) s = 0, phase ^= 1u;
    }

    // ---- the warps' states of the piece, joined 64 dims at a time: row
    // 2 warp + lane / 16, four dims a lane
#pragma unroll
    for (int sh = 4; sh < 32; sh *= 2) {
      l0 += __shfl_xor_sync(0xffffffffu, l0, sh);
      l1 += __shfl_xor_sync(0xffffffffu, l1, sh);
    }
    const int jr = 2 * warp + lane / 16, jd = lane % 16 * 4;
    const int r = rt * kRows + jr;
    const bool whole = kt0 == 0 && kt1 == kts;
    const int rec = (2 * me + (kt0 == 0 ? 1 : 0)) * kRows + jr;
    float f[kWarps], inv = 0.f;
#pragma unroll
    for (int hf = 0; hf < kHalves; ++hf) {
      group_sync(group);  // what was here has been read
      float* d0 = so + (warp * kRows + 2 * t) * kLd + 8 * g;
      float* d1 = d0 + kLd;
      const float(*v)[4] = o + 4 * hf;
      *reinterpret_cast<float4*>(d0) = make_float4(v[0][0], v[0][2], v[1][0], v[1][2]);
      *reinterpret_cast<float4*>(d0 + 4) = make_float4(v[2][0], v[2][2], v[3][0], v[3][2]);
      *reinterpret_cast<float4*>(d1) = make_float4(v[0][1], v[0][3], v[1][1], v[1][3]);
      *reinterpret_cast<float4*>(d1 + 4) = make_float4(v[2][1], v[2][3], v[3][1], v[3][3]);
      if (hf == 0 && g == 0) {
        *reinterpret_cast<float2*>(sm + warp * kRows + 2 * t) = make_float2(m0, m1);
        *reinterpret_cast<float2*>(sl + warp * kRows + 2 * t) = make_float2(l0, l1);
      }
      group_sync(group);
      if (hf == 0) {
        float top = kFloor, l = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) top = fmaxf(top, sm[w * kRows + jr]);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          f[w] = exp2_approx(sm[w * kRows + jr] - top);
          l += f[w] * sl[w * kRows + jr];
        }
        if (whole) {
          inv = l > 0.f ? 1.f / l : l;  // no key: zeros; NaN stays
        } else if (lane % 16 == 0) {
          *reinterpret_cast<float2*>(a.part_ml + 2 * rec) = make_float2(top, l);
        }
      }
      float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float4 x = *reinterpret_cast<const float4*>(so + (w * kRows + jr) * kLd + jd);
        acc[0] += f[w] * x.x, acc[1] += f[w] * x.y, acc[2] += f[w] * x.z, acc[3] += f[w] * x.w;
      }
      if (!whole) {
        *reinterpret_cast<float4*>(a.part_o + static_cast<int64_t>(rec) * D + 64 * hf + jd) =
            make_float4(acc[0], acc[1], acc[2], acc[3]);
      } else if (r < rows) {
        const int tok = kSingle ? 0 : r / a.group;
        bf16* dst = static_cast<bf16*>(a.out) +
                    (static_cast<int64_t>((kSingle ? at.b : a.cu_q[at.b]) + tok) * a.hq + h * a.group + r - tok * a.group) * D;
        *reinterpret_cast<uint2*>(dst + 64 * hf + jd) =
            make_uint2(pack_bf16x2(acc[0] * inv, acc[1] * inv), pack_bf16x2(acc[2] * inv, acc[3] * inv));
      }
    }
    if (!whole && kt0 == 0 && warp == 0 && lane == 0) {
      // the run that has the unit's last place
      const int last = pre[at.b] + (at.unit + 1) * (kUnitCost + kts) - 1;
      int i = min(n - 1, static_cast<int>(static_cast<float>(last) / static_cast<float>(total) * n));
      while (i > me && start_of(i) > last) --i;
      while (i + 1 < n && start_of(i + 1) <= last) ++i;
      reinterpret_cast<int4*>(a.desc)[me] = make_int4(i, at.b, h, rt);
    }
    at.kt = 0, ++at.unit;  // if this was not its end, the run is over
  }
}

// Joins the records of the unit that run blockIdx.x began and others went on
// with. Warp w: row w % 8, records w / 8 modulo 4 of the chain. Bound by latency:
// with a warp for all records of a row a chain of 55 (one request of 131072 keys)
// took 55 us in all instead of 45.
template <int D, bool kSingle>
__global__ void __launch_bounds__(1024) kv4_join_kernel(const __grid_constant__ Kv4AttnArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  constexpr int kE = D / 32;
  __shared__ float so[3][kRows][D], sl[3][kRows];
  const int4 d = reinterpret_cast<const int4*>(a.desc)[blockIdx.x];
  if (d.x < 0) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int row = warp % kRows, part = warp / kRows, begin = blockIdx.x, count = d.x - begin + 1;
  auto rec_of = [&](int i) { return (2 * (begin + i) + (i == 0 ? 1 : 0)) * kRows + row; };
  float top = kFloor;
  for (int i = lane; i < count; i += 32) top = fmaxf(top, a.part_ml[2 * rec_of(i)]);
  top = warp_max(top);
  float l = 0.f, acc[kE] = {};
#pragma unroll 8
  for (int i = part; i < count; i += 4) {
    const int rec = rec_of(i);
    const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + 2 * rec);
    const float f = exp2_approx(ml.x - top);
    const float* v = a.part_o + static_cast<int64_t>(rec) * D + lane * kE;
    l += ml.y * f;
#pragma unroll
    for (int k = 0; k < kE; ++k) acc[k] += v[k] * f;
  }
  if (part > 0) {
#pragma unroll
    for (int k = 0; k < kE; ++k) so[part - 1][row][lane * kE + k] = acc[k];
    if (lane == 0) sl[part - 1][row] = l;
  }
  __syncthreads();
  const int G = a.group, r = d.w * kRows + row;
  if (part > 0 || r >= rows_of<kSingle>(a, d.y)) return;
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    l += sl[i][row];
#pragma unroll
    for (int k = 0; k < kE; ++k) acc[k] += so[i][row][lane * kE + k];
  }
  const float inv = l > 0.f ? 1.f / l : l;
  const int tok = kSingle ? 0 : r / G;
  uint32_t* dst = reinterpret_cast<uint32_t*>(
      static_cast<bf16*>(a.out) +
      (static_cast<int64_t>((kSingle ? d.y : a.cu_q[d.y]) + tok) * a.hq + d.z * G + r - tok * G) * D + lane * kE);
#pragma unroll
  for (int k = 0; k < kE / 2; ++k) dst[k] = pack_bf16x2(acc[2 * k] * inv, acc[2 * k + 1] * inv);
}

template <int D>
int attn_smem(int B) {
  return kGroups * group_bytes<D>() + (4 * B + 2) * 4;
}

template <int D, bool kSingle>
void launch_typed(const Kv4AttnArgs& a, cudaStream_t s) {
  static bool done[64] = {};  // per device
  int dev = 0;
  cudaGetDevice(&dev);
  if (!done[dev & 63]) {
    if (cudaFuncSetAttribute(kv4_attn_kernel<D, kSingle>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             attn_smem<D>(kKv4MaxBatch)) != cudaSuccess)
      throw std::runtime_error("minisgl.attention_kv4: shared memory limit");
    done[dev & 63] = true;
  }
  launch_pdl(kv4_attn_kernel<D, kSingle>, dim3(a.runs / kGroups), dim3(kThreads), attn_smem<D>(a.B), s, a);
  launch_pdl(kv4_join_kernel<D, kSingle>, dim3(a.runs), dim3(1024), 0, s, a);
}

}  // namespace

int kv4_attn_runs(int sms) { return kGroups * sms; }

void launch_kv4_attention(const Kv4AttnArgs& a, cudaStream_t s) {
  if (a.B <= 0) return;
  const bool single = a.cu_q == nullptr;
  if (a.d == 128) single ? launch_typed<128, true>(a, s) : launch_typed<128, false>(a, s);
  else if (a.d == 64) single ? launch_typed<64, true>(a, s) : launch_typed<64, false>(a, s);
  else throw std::runtime_error("minisgl.attention_kv4: head_dim must be 64 or 128");
}

}  // namespace minisgl
