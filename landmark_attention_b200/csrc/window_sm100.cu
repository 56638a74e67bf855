// Sliding-window attention with sinks on the tensor cores (sm_100a): bf16 / fp16, head dims up to 128, TMA-fed tcgen05 products with
// accumulators in TMEM.  Query tiles of 128 rows meet key tiles of 64 (forward, dQ) or pairs of them (dK, dV); only the tiles that
// the window or the sinks make visible are visited (window_params.h), and only those on an edge are masked.
//
// Forward: unit = (query tile, head), persistent; key tiles newest first, the sinks' last.
//   S = Q K^T -> a softmax thread owns one row (= one TMEM lane): p = 2^(s c - m), l += sum p, P written in 16 bits over the TMEM
//   columns its S came from -> O += P V with A = P from TMEM.  m is the running maximum, but is only moved when a tile exceeds it by more
//   than 2^8: O then has to be read, scaled and written back (TMEM), which with the first tile's maximum as m happens to a few rows of
//   a long sequence.  p <= 2^8 costs no precision: p, l and O are floating point, and O / l does not depend on m.
// Backward: recomputed from lse = m + log2 l, in three launches and a join of the sinks' sums (window.cu).
//   delta = rowsum(O dO).
//   dQ: unit = (query tile, head), persistent.  Q and dO rows go to TMEM as A operands; per key tile S, dP -> dS in 16 bits over
//   the TMEM columns of dP -> dQ += dS K with A = dS from TMEM.
//   dK/dV: unit = (pair of key tiles, key head, run of query tiles), persistent; Q and dO tiles of all heads that share the keys
//   stream through, and their contributions are summed in the accumulators.  The query tiles of a pair with sinks are dealt out to several
//   units (SinkSplit): one unit would be as long as the sequence.
// Rows behind a sequence's end (lengths) are hidden by selects and, where a product would multiply them with a zero, overwritten with zeros in
// shared memory by the loading warp, so that NaN there stays there.
// B1 H32 L2048 D128, window 512, sinks 4, bf16: forward 34 us (37 with the rest for the backward pass), delta 6 to 10, dQ 43, dK/dV 54, join 4.
// L32768 on 8 key heads, window 4096, where starts and boundaries do not count: 1850, 95, 2950, 3370, at 69, 65 and 75 % of the measured rate of
// products in the three that have some (S and dP are formed twice in the backward pass).
// All waits are bounded (sm100_ptx.cuh).
#include <mutex>
#include "common.cuh"
#include "attn_params.h"
#include "window_params.h"
#include "sm100_ptx.cuh"
#include "sm100_tiles.cuh"

namespace lmk {
namespace {

using namespace ptx;

constexpr int kBlk = 64;
constexpr int kQTile = 128;
constexpr uint32_t kTileBytes = 16384;   // one [128 x 64] or two [64 x 64] 16-bit tiles
constexpr uint32_t kHalfTile = 8192;
constexpr float kLog2e = 1.4426950408889634f;
enum { kErrFwdProducer = 711, kErrFwdMma = 712, kErrFwdSoftmax = 713, kErrFwdEpilogue = 714, kErrDkvProducer = 721, kErrDkvMma = 722,
       kErrDkvSoftmax = 723, kErrDkvEpilogue = 724, kErrDqProducer = 731, kErrDqMma = 732, kErrDqSoftmax = 733, kErrDqEpilogue = 734 };

__device__ __forceinline__ int length_of(const int* lengths, int b, int Lk) {
  return lengths == nullptr ? Lk : min(max(ld_behind_wait(lengths + b), 0), Lk);
}
// rows [from, rows) of a tile of 64-feature sub-tiles become zeros, ahead of products that read the tile; one warp (one thread took 6000 clk)
__device__ __forceinline__ void zero_rows(uint32_t tile, uint32_t subtile_bytes, int subtiles, int from, int rows, int lane) {
  from = max(from, 0);
  for (int c = 0; c < subtiles; ++c)
    for (uint32_t a = tile + c * subtile_bytes + from * 128u + lane * 16u; a < tile + c * subtile_bytes + rows * 128u; a += 512)
      asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(a), "r"(0) : "memory");
  fence_proxy_async_smem();
  __syncwarp();
}

// A row's visible columns among 32 keys from key0 on, a bit each: j <= pos - key0 and (j > pos - key0 - window or j < sinks - key0).  (With
// the comparisons at each column an item at an edge took twice the time of a full one.)
__device__ __forceinline__ uint32_t low_bits(int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1u; }
__device__ __forceinline__ uint32_t columns_seen(int pos, int key0, int window, int sinks) {
  return low_bits(pos - key0 + 1) & (~low_bits(pos - window + 1 - key0) | low_bits(sinks - key0));
}
// Every one of the rows at positions p0 .. p1 sees every one of the keys k0 .. k1 / none sees one.
__device__ __forceinline__ bool all_seen(int p0, int p1, int k0, int k1, int window, int sinks) {
  return k1 <= p0 && (p1 - k0 < window || k1 < sinks);
}
__device__ __forceinline__ bool none_seen(int p0, int p1, int k0, int k1, int window, int sinks) {
  return k0 > p1 || (p0 - k1 >= window && k0 >= sinks);
}

// n 16-byte pieces from `to` on become zeros, by `threads` threads side by side (a row a thread took 15 000 clk for 128 rows)
__device__ __forceinline__ void zero_fill(void* to, int n, int thread, int threads) {
#pragma unroll 1
  for (int i = thread; i < n; i += threads) reinterpret_cast<uint4*>(to)[i] = make_uint4(0u, 0u, 0u, 0u);
}

// two numbers in the 16-bit type, as fp32
template <bool kBf16> __device__ __forceinline__ float2 unpack2(uint32_t x) {
  if (kBf16) return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&x));
  return __half22float2(*reinterpret_cast<const __half2*>(&x));
}

// What rounding x to 16 bits left, a byte a number: in steps of 1 / 128 of the rounded number's last place, so at most 64 of them either way,
// whatever the number's size, and 64 added.  (Below 2^-112 in bf16 the step stays that of 2^-112: 2^-126.)
constexpr uint32_t kRestZero = 64;
// two exponent fields of rounded numbers, in bf16's place, and not below the least one a step is made from
template <bool kBf16> __device__ __forceinline__ uint32_t exponents2(uint32_t rounded) {
  return kBf16 ? __vmaxu2(rounded & 0x7f807f80u, 0x07800780u) : __vmaxu2((rounded & 0x7c007c00u) >> 3, 0x00800080u);
}
template <bool kBf16> __device__ __forceinline__ uint32_t rest4(const float (&x)[4]) {
  uint32_t r[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const uint32_t rounded = pack2<kBf16>(x[2 * e], x[2 * e + 1]);
    const float2 back = unpack2<kBf16>(rounded);
    const __nv_bfloat162 left = __floats2bfloat162_rn(x[2 * e] - back.x, x[2 * e + 1] - back.y);
    // 1 / step = 2^(134 - field + 7) or 2^(25 - field + 7), by its exponent field
    const uint32_t per_step = (kBf16 ? 0x86008600u : 0x4f804f80u) - exponents2<kBf16>(rounded);
    // bf16 numbers between 128 and 256 are whole: 192 + steps, rounded, whose low byte is 64 + steps
    const __nv_bfloat162 n = __hfma2(left, *reinterpret_cast<const __nv_bfloat162*>(&per_step), __floats2bfloat162_rn(192.f, 192.f));
    r[e] = *reinterpret_cast<const uint32_t*>(&n);
  }
  return __byte_perm(r[0], r[1], 0x6420);
}
// the two numbers, as they were, of a pair of rounded ones and bytes first, first + 1 of the rest
template <bool kBf16> __device__ __forceinline__ float2 restored2(uint32_t rounded, uint32_t rest, int first) {
  const float2 x = unpack2<kBf16>(rounded);
  const uint32_t step = exponents2<kBf16>(rounded) + (kBf16 ? 0u - 0x07000700u : 0x2f802f80u);      // 14 fields down; fp16: 112 up, 17 down
  const float2 s = unpack2<true>(step);
  const float a = __uint_as_float(__byte_perm(rest, 0x4b000000u, 0x7440u + first)) - (8388608.f + kRestZero);      // 2^23 + byte
  const float b = __uint_as_float(__byte_perm(rest, 0x4b000000u, 0x7441u + first)) - (8388608.f + kRestZero);
  return make_float2(fmaf(a, s.x, x.x), fmaf(b, s.y, x.y));
}

struct WindowTensors {
  void* o;
  uint8_t* rest;
  float* lse;
  const int* lengths;
  int BH, H, G, Lq, Lk, D, window, sinks;
  float scale_log2;
};

// ---------------------------------------------------------------------------------------------- forward
// Persistent, two CTAs an SM whose gaps fill each other; a unit is a query tile of 128 rows of a head.  The loads run on into the next unit
// and its first scores are there when the last one's output has been written: with a CTA a unit, setting up, fetching Q and ending took
// 7000 of a unit's 17 000 clk (B1 H32 L2048, window 512).
// One warp issues all products: S of item i + 2 right behind P V of item i, which reads the P that stands in its place (the tensor core works
// through what one thread issues in order).  TMEM: 2 x 64 S / P + kD O.  Shared memory: Q, and a ring of K and V tiles.
constexpr int kFwdThreads = (4 + 2) * 32;
template <int kD> constexpr int kFwdSlots = kD == 128 ? 5 : 10;      // 64-row K and V tiles, in turn
constexpr int kFwdPolyEvery = 4;         // one pair of exponentials in this many is a polynomial on the FMA pipe
constexpr float kLazy = 8.f;             // the maximum moves when it is exceeded by this much (log2)

template <int kSlots> struct FwdSmem {
  uint64_t q_full, q_empty, patch;
  uint64_t full[kSlots], empty[kSlots];
  uint64_t s_full[2], p_ready[2];        // [S / P buffer]
  uint64_t o_full, o_empty;
  uint32_t tmem_base;
};

__device__ __forceinline__ float max_of_64(const float (&v)[64]) {      // NaN where one is
  float m[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
  for (int j = 0; j < 64; j += 2) m[j / 2 % 4] = max3_nan(m[j / 2 % 4], v[j], v[j + 1]);
  return max3_nan(max3_nan(m[0], m[1], m[2]), m[3], m[3]);
}

// a query tile of 128 rows of a head, and the key tiles it meets: the newest first, the sinks' last
struct RowUnit {
  int t, bh, b, h, len, n_win, total;
  KeyTiles k;
  __device__ int tile_of(int i) const { return i < n_win ? k.last - i : k.sink_tiles - 1 - (i - n_win); }
};
__device__ __forceinline__ RowUnit row_unit(int w, int n_tiles, int BH, int H, const int* lengths, int Lq, int Lk, int window, int sinks) {
  RowUnit u;
  u.t = n_tiles - 1 - w / BH;                // longest tiles first, across all heads
  u.bh = w % BH;
  u.b = u.bh / H;
  u.h = u.bh - u.b * H;
  u.len = length_of(lengths, u.b, Lk);
  u.k = keys_of_queries(u.t, kQTile, kBlk, Lq, Lk - Lq, u.len, window, sinks);
  u.n_win = u.k.last - u.k.first + 1;        // 0: nothing but padding
  u.total = u.n_win + u.k.sink_tiles;
  return u;
}
// units are dealt to the CTAs in rounds, in alternating direction
__device__ __forceinline__ int unit_at(int r) { return r * (int)gridDim.x + ((r & 1) ? (int)(gridDim.x - 1 - blockIdx.x) : (int)blockIdx.x); }

template <bool kBf16, int kD>
__global__ void __launch_bounds__(kFwdThreads, 2)
window_fwd_sm100_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                        const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ WindowTensors p, int* status) {
  constexpr int kSlots = kFwdSlots<kD>;
  constexpr uint32_t kQBytes = (kD / 64) * kTileBytes, kKvBytes = kQBytes / 2;
  extern __shared__ __align__(1024) uint8_t smem_aligned[];      // (a kilobyte of slack would not fit twice)
  const uint32_t base = smem_u32(smem_aligned);
  if ((base & 1023u) != 0) {                                     // the swizzle needs it
    if (threadIdx.x == 0) atomicCAS(status, 0, kErrFwdProducer);
    return;
  }
  auto slot = [&](int m) { return base + kQBytes + (uint32_t)(m % kSlots) * kKvBytes; };
  FwdSmem<kSlots>* sm = reinterpret_cast<FwdSmem<kSlots>*>(smem_aligned + kQBytes + kSlots * kKvBytes);

  const int tid = threadIdx.x, warp = warp_uniform(tid >> 5), lane = tid & 31;
  const int off = p.Lk - p.Lq, n_tiles = (p.Lq + kQTile - 1) / kQTile, n_units = n_tiles * p.BH;
  auto unit_of = [&](int w) { return row_unit(w, n_tiles, p.BH, p.H, p.lengths, p.Lq, p.Lk, p.window, p.sinks); };

  if (tid == 0) {
    for (const CUtensorMap* tm : {&tm_q, &tm_k, &tm_v}) prefetch_tensormap(tm);
    for (uint64_t* bar : {&sm->q_full, &sm->q_empty, &sm->patch, &sm->o_full, &sm->s_full[0], &sm->s_full[1]}) mbar_init(smem_u32(bar), 1);
    for (uint64_t* bar : {&sm->o_empty, &sm->p_ready[0], &sm->p_ready[1]}) mbar_init(smem_u32(bar), 128);
    for (int s = 0; s < kSlots; ++s) {
      mbar_init(smem_u32(&sm->full[s]), 1);
      mbar_init(smem_u32(&sm->empty[s]), 1);
    }
    mbar_init_fence();
  }
  if (warp == 5) tmem_alloc(smem_u32(&sm->tmem_base), 256);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = (uint32_t)warp_uniform((int)sm->tmem_base);
  const uint32_t tmem_s = tmem, tmem_o = tmem + 128u;
  grid_dep_wait();
  grid_dep_launch();

  if (warp == 4) {
    // ------------------------------------------------------------------ loads
    int m = 0, uq = 0, patches = 0;
    for (int r = 0, w = unit_at(0); w < n_units; w = unit_at(++r)) {
      const RowUnit u = unit_of(w);
      if (u.total == 0) continue;
      const int hk = u.h / p.G;
      auto load_kv = [&](const CUtensorMap* tm, int key0, bool patch) {
        mbar_wait(smem_u32(&sm->empty[m % kSlots]), ((m / kSlots) & 1) ^ 1, status, kErrFwdProducer);
        const uint32_t bar = smem_u32(patch ? &sm->patch : &sm->full[m % kSlots]);
        if (lane == 0) {
          mbar_arrive_expect_tx(bar, kKvBytes);
          for (int c = 0; c < kD / 64; ++c) tma_load_4d(slot(m) + c * kHalfTile, tm, bar, 64 * c, key0, hk, u.b);
        }
        __syncwarp();
        if (patch) {
          mbar_wait(bar, patches++ & 1, status, kErrFwdProducer);
          zero_rows(slot(m), kHalfTile, kD / 64, u.len - key0, kBlk, lane);
          if (lane == 0) mbar_arrive(smem_u32(&sm->full[m % kSlots]));
        }
        ++m;
      };
      mbar_wait(smem_u32(&sm->q_empty), (uq++ & 1) ^ 1, status, kErrFwdProducer);
      if (lane == 0) {
        mbar_arrive_expect_tx(smem_u32(&sm->q_full), kQBytes);
        for (int c = 0; c < kD / 64; ++c) tma_load_4d(base + c * kTileBytes, &tm_q, smem_u32(&sm->q_full), 64 * c, u.t * kQTile, u.h, u.b);
      }
      __syncwarp();
      for (int i = 0; i < u.total; ++i) {
        const int key0 = u.tile_of(i) * kBlk;
        load_kv(&tm_k, key0, false);
        load_kv(&tm_v, key0, key0 + kBlk > u.len && u.len < p.Lk);      // values of the tile the sequence ends in
      }
    }
  } else if (warp == 5) {
    // ------------------------------------------------------------------ products
    constexpr uint32_t fmt = kBf16 ? 1u : 0u;
    constexpr uint32_t idesc_s = instr_desc_f16(fmt, 128, 64, 0, 0), idesc_o = instr_desc_f16(fmt, 128, kD, 0, 1);
    const uint64_t dq = smem_desc_sw128(base, 16, 1024), dk0 = smem_desc_sw128(slot(0), 16, 1024), dv0 = smem_desc_sw128(slot(0), kHalfTile, 1024);
    int r = -1, u = -1, it = 0;                      // it: items of all units
    auto next_unit = [&]() {                         // items of the next unit that has any, 0: no more
      for (;;) {
        const int w = unit_at(++r);
        if (w >= n_units) return 0;
        const int n = warp_uniform(unit_of(w).total);
        if (n > 0) {
          ++u;
          return n;
        }
      }
    };
    auto arrived = [&](int m) {
      mbar_wait(smem_u32(&sm->full[m % kSlots]), (m / kSlots) & 1, status, kErrFwdMma);
      tc_fence_after();
    };
    auto issue_s = [&](int i, int n, int j) {        // item i of n, the j-th of all
      if (i == 0) mbar_wait(smem_u32(&sm->q_full), u & 1, status, kErrFwdMma);
      arrived(2 * j);
      const uint64_t dk = desc_advance(dk0, (uint32_t)((2 * j) % kSlots) * kKvBytes);
      if (elect_one()) {
#pragma unroll
        for (int kk = 0; kk < kD / 16; ++kk)
          mma_f16_ss(tmem_s + (j & 1) * 64, desc_advance(dq, kmajor_step(kk, kTileBytes)), desc_advance(dk, kmajor_step(kk, kHalfTile)), idesc_s, kk > 0);
        mma_commit(smem_u32(&sm->s_full[j & 1]));
        mma_commit(smem_u32(&sm->empty[(2 * j) % kSlots]));
        if (i == n - 1) mma_commit(smem_u32(&sm->q_empty));
      }
    };
    for (int n = next_unit(); n > 0; n = next_unit()) {
      for (int i = 0; i < min(n, 2); ++i) issue_s(i, n, it + i);
      for (int i = 0; i < n; ++i, ++it) {
        arrived(2 * it + 1);
        if (i == 0) mbar_wait(smem_u32(&sm->o_empty), (u & 1) ^ 1, status, kErrFwdMma);
        mbar_wait(smem_u32(&sm->p_ready[it & 1]), (it >> 1) & 1, status, kErrFwdMma);
        tc_fence_after();
        const uint64_t dv = desc_advance(dv0, (uint32_t)((2 * it + 1) % kSlots) * kKvBytes);
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < kBlk / 16; ++kk)     // P: 8 columns = 16 keys per K-step
            mma_f16_ts(tmem_o, tmem_s + (it & 1) * 64 + kk * 8, desc_advance(dv, kk * 2048), idesc_o, (i > 0 || kk > 0) ? 1u : 0u);
          mma_commit(smem_u32(&sm->empty[(2 * it + 1) % kSlots]));
          if (i == n - 1) mma_commit(smem_u32(&sm->o_full));
        }
        if (i + 2 < n) issue_s(i + 2, n, it + 2);
      }
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------------ softmax
    const int row = tid;
    const uint32_t lane_base = (uint32_t)(warp * 32) << 16;
    const float c = p.scale_log2;
    int it = 0, units = 0;
    for (int r = 0, x = unit_at(0); x < n_units; x = unit_at(++r)) {
      const RowUnit u = unit_of(x);
      const int pos = off + u.t * kQTile + row, grow = u.t * kQTile + row;
      const bool stored = grow < p.Lq;
      if (u.total == 0) {                            // nothing but padding
        const int64_t at = ((int64_t)u.bh * p.Lq + u.t * kQTile) * p.D;
        const int n = min(kQTile, p.Lq - u.t * kQTile) * p.D / 8;
        zero_fill(reinterpret_cast<uint16_t*>(p.o) + at, n, tid, 128);      // (its rest is not read)
        if (stored && p.lse != nullptr) p.lse[(int64_t)u.bh * p.Lq + grow] = INFINITY;
        __syncwarp();
        continue;
      }
      const int warp_p0 = warp_uniform(off + u.t * kQTile + warp * 32), warp_p1 = warp_p0 + 31;
      float m2 = -INFINITY, l = 0.f;
      for (int i = 0; i < u.total; ++i, ++it) {
        const int key0 = u.tile_of(i) * kBlk;
        const uint32_t ts = tmem_s + (uint32_t)(it & 1) * 64u + lane_base;
        const bool none = none_seen(warp_p0, warp_p1, key0, key0 + kBlk - 1, p.window, p.sinks);
        const bool full = all_seen(warp_p0, warp_p1, key0, key0 + kBlk - 1, p.window, p.sinks);
        mbar_wait(smem_u32(&sm->s_full[it & 1]), (it >> 1) & 1, status, kErrFwdSoftmax);
        tc_fence_after();
        uint32_t wgt[32];
        if (none) {
#pragma unroll
          for (int j = 0; j < 32; ++j) wgt[j] = 0u;
        } else {
          float sv[64];
          {
            uint32_t ra[32], rb[32];
            tmem_ld_32x32b_x32(ts, ra);
            tmem_ld_32x32b_x32(ts + 32, rb);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 32; ++j) {
              sv[j] = __uint_as_float(ra[j]);
              sv[32 + j] = __uint_as_float(rb[j]);
            }
          }
          if (!full) {
            const uint32_t lo = columns_seen(pos, key0, p.window, p.sinks), hi = columns_seen(pos, key0 + 32, p.window, p.sinks);
#pragma unroll
            for (int j = 0; j < 32; ++j) {
              sv[j] = lo & (1u << j) ? sv[j] : -INFINITY;
              sv[32 + j] = hi & (1u << j) ? sv[32 + j] : -INFINITY;
            }
          }
          const float mx = max_of_64(sv);
          const float mc = mx * c;                                     // -inf: nothing visible
          const bool move = mc > m2 + kLazy;                           // from -inf on too
          if (__any_sync(0xffffffffu, move && m2 != -INFINITY)) {
            // O is rescaled behind P V of the item before.  That came behind S of this one: its end is that of the item's V tile, or
            // of the unit; the next S of its buffer would tell as well, but is not due before this item's P.
            mbar_wait(smem_u32(&sm->empty[(2 * it - 1) % kSlots]), ((2 * it - 1) / kSlots) & 1, status, kErrFwdSoftmax);
            tc_fence_after();
            const float f = move ? ex2(m2 - mc) : 1.f;                 // from -inf: 0, where O is 0
            l *= f;
            for (int cc = 0; cc < kD / 16; ++cc) {
              uint32_t o[16];
              tmem_ld_32x32b_x16(tmem_o + cc * 16 + lane_base, o);
              tmem_ld_wait();
#pragma unroll
              for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * f);
              tmem_st_32x32b_x16(tmem_o + cc * 16 + lane_base, o);
            }
            tmem_st_wait();
          }
          if (move) m2 = mc;
          uint64_t sp[32];
          if (!full) {
            const float shift = m2 == -INFINITY ? 0.f : m2;
#pragma unroll
            for (int j = 0; j < 32; ++j) sp[j] = pk2(ex2(fmaf(sv[2 * j], c, -shift)), ex2(fmaf(sv[2 * j + 1], c, -shift)));
          } else {
            // polynomials make finite numbers of NaN and infinities: a maximum that is one makes NaN of the shift of all
            const float n = fmaf(mx, 0.f, -m2);
            const uint64_t c2 = pk2(c, c), n2 = pk2(n, n);
#pragma unroll
            for (int j = 0; j < 32; ++j) {
              const uint64_t e = fma2(pk2(sv[2 * j], sv[2 * j + 1]), c2, n2);
              if (j % kFwdPolyEvery == 1) {
                sp[j] = ex2_poly2<4>(e);
              } else {
                float e0, e1;
                upk2(e, e0, e1);
                sp[j] = pk2(ex2(e0), ex2(e1));
              }
            }
          }
          uint64_t s0 = sp[0], s1 = sp[1], s2 = sp[2], s3 = sp[3];
#pragma unroll
          for (int j = 4; j < 32; j += 4) {
            s0 = add2(s0, sp[j]);
            s1 = add2(s1, sp[j + 1]);
            s2 = add2(s2, sp[j + 2]);
            s3 = add2(s3, sp[j + 3]);
          }
          float dl, dh;
          upk2(add2(add2(s0, s1), add2(s2, s3)), dl, dh);
          l += dl + dh;
          // P enters the product in 16 bits: half a step of relative error a weight; l sums the unrounded ones
#pragma unroll
          for (int j = 0; j < 32; ++j) wgt[j] = pack2p<kBf16>(sp[j]);
        }
        tmem_st_32x32b_x32(ts, wgt);                 // P replaces S in place; the P V product reads it there
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(smem_u32(&sm->p_ready[it & 1]));
      }
      // epilogue
      mbar_wait(smem_u32(&sm->o_full), units & 1, status, kErrFwdEpilogue);
      ++units;
      tc_fence_after();
      const bool valid = pos < u.len;                // sees its own key at least; l = 0 where every score is -inf: NaN, as by the formula
      const float inv = valid ? 1.f / l : 0.f;
      int64_t row_off[4];                            // of the four rows that four lanes write together
      {
        const int64_t at = stored ? ((int64_t)u.bh * p.Lq + grow) * p.D : -1;
#pragma unroll
        for (int j = 0; j < 4; ++j) row_off[j] = __shfl_sync(0xffffffffu, at, (lane & ~3) + j);
      }
#pragma unroll
      for (int cc = 0; cc < kD / 32; ++cc) {
        uint32_t o[32];
        tmem_ld_32x32b_x32(tmem_o + cc * 32 + lane_base, o);
        tmem_ld_wait();
        if (cc == kD / 32 - 1) {
          tc_fence_before();
          mbar_arrive(smem_u32(&sm->o_empty));       // the next unit may start accumulating
        }
#pragma unroll
        for (int e = 0; e < 32; ++e) o[e] = valid ? __float_as_uint(__uint_as_float(o[e]) * inv) : 0u;      // (not 0 * what padding left there)
        store_acc_cols<kBf16>(p.o, row_off, o, cc * 32, p.D, lane);
        if (p.rest != nullptr && stored) {
#pragma unroll
          for (int e = 0; e < 32; e += 8) {
            const float x[4] = {__uint_as_float(o[e]), __uint_as_float(o[e + 1]), __uint_as_float(o[e + 2]), __uint_as_float(o[e + 3])};
            const float y[4] = {__uint_as_float(o[e + 4]), __uint_as_float(o[e + 5]), __uint_as_float(o[e + 6]), __uint_as_float(o[e + 7])};
            if (cc * 32 + e < p.D)
              *reinterpret_cast<uint2*>(p.rest + ((int64_t)u.bh * p.Lq + grow) * p.D + cc * 32 + e) = make_uint2(rest4<kBf16>(x), rest4<kBf16>(y));
          }
        }
        __syncwarp();
      }
      if (stored && p.lse != nullptr) p.lse[(int64_t)u.bh * p.Lq + grow] = valid ? m2 + __log2f(l) : INFINITY;
      __syncwarp();
    }
    tc_fence_before();
  }
  __syncthreads();
  if (warp == 5) {
    tc_fence_after();
    tmem_dealloc(tmem, 256);
  }
}

// ---------------------------------------------------------------------------------------------- backward
// Four softmax warpgroups in both kernels: with the normaliser known there are no sums over a row, so a row's columns can belong to
// several threads, and 32 columns a thread fit 96 registers.  (Two warpgroups of 64 columns each: training size 176 us, four 156.)
constexpr int kBwdWarps = 16;
constexpr int kCols = 32;                           // columns of a score tile that one thread holds
// one pair of exponentials in this many is a cubic (7.5e-5, below half a step of either type); full tiles only
constexpr int kBwdPolyEvery = 4;

// 32 TMEM columns of the thread's lane -> 16 packed pairs
__device__ __forceinline__ void load_pairs(uint64_t (&x)[kCols / 2], uint32_t taddr) {
  uint32_t r[kCols];
  tmem_ld_32x32b_x32(taddr, r);
  tmem_ld_wait();
#pragma unroll
  for (int j = 0; j < kCols / 2; ++j) x[j] = pk2u(r[2 * j], r[2 * j + 1]);
}
// The same 32 x 32 part of a score tile as fragments: x[h][2 j + e] is row 16 h + 8 e + lane / 4, columns 8 j + 2 (lane % 4) and the next.
__device__ __forceinline__ void load_fragments(uint64_t (&x)[2][8], uint32_t taddr) {
  uint32_t a[16], b[16];
  tmem_ld_16x256b_x4(taddr, a);
  tmem_ld_16x256b_x4(taddr + (16u << 16), b);
  tmem_ld_wait();
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    x[0][k] = pk2u(a[2 * k], a[2 * k + 1]);
    x[1][k] = pk2u(b[2 * k], b[2 * k + 1]);
  }
}
__device__ __forceinline__ void store_fragments(const uint32_t (&w)[2][8], uint32_t taddr) {
  tmem_st_16x128b_x4(taddr, w[0]);
  tmem_st_16x128b_x4(taddr + (16u << 16), w[1]);
  tmem_st_wait();
}
__device__ __forceinline__ uint64_t ex2_pair(uint64_t x) {
  float a, b;
  upk2(x, a, b);
  return pk2(ex2(a), ex2(b));
}
// x: scores -> weights 2^(s c + nl), nl = -lse; hidden columns become 0 (kind 1)
__device__ __forceinline__ void weights_of(uint64_t (&x)[kCols / 2], int kind, uint32_t seen, float c, uint64_t nl) {
  const uint64_t c2 = pk2(c, c);
#pragma unroll
  for (int j = 0; j < kCols / 2; ++j) {
    const uint64_t e = fma2(x[j], c2, nl);
    if (kind == 1) {
      float a, b;
      upk2(e, a, b);
      x[j] = pk2(seen & (1u << 2 * j) ? ex2(a) : 0.f, seen & (2u << 2 * j) ? ex2(b) : 0.f);
    } else if (j % kBwdPolyEvery == 1) {
      x[j] = ex2_poly2<3>(e);
    } else {
      float a, b;
      upk2(e, a, b);
      x[j] = pk2(ex2(a), ex2(b));
    }
  }
}
// dS = p (dP - delta) scale in 16 bits; nd = -delta scale.  What a hidden value or a padded row brought along is dropped by
// a select, not multiplied by 0 (kind 1).
template <bool kBf16>
__device__ __forceinline__ void dscores_of(uint32_t (&w)[kCols / 2], const uint64_t (&p)[kCols / 2], const uint64_t (&dp)[kCols / 2], int kind,
                                           uint32_t seen, float scale, uint64_t nd) {
  const uint64_t s2 = pk2(scale, scale);
#pragma unroll
  for (int j = 0; j < kCols / 2; ++j) {
    float a, b;
    upk2(mul2(p[j], fma2(dp[j], s2, nd)), a, b);
    if (kind == 1) {
      a = seen & (1u << 2 * j) ? a : 0.f;
      b = seen & (2u << 2 * j) ? b : 0.f;
    }
    w[j] = pack2<kBf16>(a, b);
  }
}

// ---------------------------------------------------------------------------------------------- backward: dK, dV
// Transposed scores: S^T = K Q^T and dP^T = V dO^T, 128 keys on the TMEM lanes and 128 queries on the columns, so that P^T and dS^T, written
// in 16 bits over the columns they came from, are the A operands of dV += P^T dO and dK += dS^T Q straight from TMEM: no
// shared-memory tiles for them, and all four products run at the tensor cores' rate.  Shared memory still moves 256 KB an
// item (K and V as A operands, Q and dO twice as B, their loads), as long as the products take, 2048 clk each, and an item takes 3000.
// TMEM: 128 S + 128 dP + kD dV + kD dK columns.  The softmax threads and the products take turns: while P^T of an item is made, dK of the
// item before and dP of this one run; while dS^T is made, dV and the next S.  Row statistics are per column here: the loading
// warp lays them out in shared memory, and the score tiles are read as fragments, whose threads need eight columns' values and not 32: with a
// column a register 128 KB of broadcasts an item competed with the operands (3550 -> 3300 us at B1 H32 Hkv8 L32768, window 4096).
constexpr int kPair = 128;                          // keys of a unit
constexpr int kDkvThreads = (kBwdWarps + 2) * 32;
constexpr int kDkvStages = 2;
constexpr int kDealt = 4;                           // unit numbers on their way from the loading warp to the others

struct DkvSmem {
  uint64_t k_full, k_empty, v_full, v_empty, patch;
  uint64_t q_full[kDkvStages], q_empty[kDkvStages];       // Q and the statistics: until dK has been formed
  uint64_t do_full[kDkvStages], do_empty[kDkvStages];     // dO: until dV has been formed
  uint64_t stat_full[kDkvStages];
  uint64_t s_full, dp_full;                               // the products' results are there
  uint64_t p_ready, ds_ready;                             // P and dS have taken their places
  uint64_t acc_full[2], acc_empty[2];                     // [0] dV, [1] dK
  uint64_t dealt_full[kDealt], dealt_empty[kDealt];
  int dealt[kDealt];
  uint32_t tmem_base;
  alignas(16) float nlse[kDkvStages][kQTile];             // -lse
  alignas(16) float ndelta[kDkvStages][kQTile];           // -delta scale
};

struct DkvArgs {
  const float *lse, *delta;
  void *dk, *dv;
  const int* lengths;
  int* next;                                        // units given out beyond the first of each CTA; set to 0 by the delta kernel
  int H, Hkv, G, B, Lq, Lk, D, window, sinks, n_pairs;
  float scale, scale_log2;
  SinkSplit split;
};
// a unit: query tiles first .. last of every head of the group against a pair of key tiles
struct DkvUnit {
  int b, hk, pair, first, n_q, len;      // n_q: query tiles of one head
  int run;                               // -1: the window's share, else the run of the sinks' share
  __device__ bool base() const { return run < 0; }
};

template <bool kBf16, int kD>
__global__ void __launch_bounds__(kDkvThreads, 1)
window_dkv_sm100_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                        const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_do,
                        const __grid_constant__ DkvArgs p, int* status) {
  constexpr int kStages = kDkvStages;
  constexpr uint32_t kOperand = (kD / 64) * kTileBytes;     // [128 rows x kD] as 64-feature sub-tiles of 16 KB
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  const uint32_t k_pair = base, v_pair = base + kOperand;
  auto q_slot = [&](int s) { return base + 2 * kOperand + (uint32_t)s * 2 * kOperand; };
  auto do_slot = [&](int s) { return base + 3 * kOperand + (uint32_t)s * 2 * kOperand; };
  DkvSmem* sm = reinterpret_cast<DkvSmem*>(smem_raw + (base - raw) + (2 + 2 * kStages) * kOperand);

  const int tid = threadIdx.x, warp = warp_uniform(tid >> 5), lane = tid & 31;
  const int off = p.Lk - p.Lq, heads = p.B * p.Hkv;
  const int n_runs = p.split.tiles * p.split.runs * heads, n_units = n_runs + p.n_pairs * heads;
  // Units differ by the number of query tiles, with ragged sequences many times over: each CTA asks for its next one (dealt out in turn, the
  // busiest had 93 000 clk and the idlest 59 000 at the training size).  The runs come first: they are as long as the longest of the others.
  auto unit_of = [&](int w) {
    DkvUnit u;
    int bk;
    if (w < n_runs) {
      const int x = w / heads;
      bk = w - x * heads;
      u.pair = x / p.split.runs;
      u.run = x - u.pair * p.split.runs;
    } else {
      u.pair = (w - n_runs) / heads;
      bk = (w - n_runs) - u.pair * heads;
      u.run = -1;
    }
    u.b = bk / p.Hkv;
    u.hk = bk - u.b * p.Hkv;
    u.len = length_of(p.lengths, u.b, p.Lk);
    const QueryTiles q = queries_of_keys(u.pair, kQTile, kPair, p.Lq, off, u.len, p.window, p.sinks);
    u.first = q.first;
    int last = u.pair < p.split.tiles ? q.last : q.end;
    if (u.run >= 0) {
      u.first = q.last + 1 + u.run * p.split.run;
      last = min(q.end, u.first + p.split.run - 1);
    }
    u.n_q = max(last - u.first + 1, 0);
    return u;
  };

  if (tid == 0) {
    for (const CUtensorMap* tm : {&tm_q, &tm_k, &tm_v, &tm_do}) prefetch_tensormap(tm);
    for (uint64_t* bar : {&sm->k_full, &sm->k_empty, &sm->v_full, &sm->v_empty, &sm->patch, &sm->s_full, &sm->dp_full})
      mbar_init(smem_u32(bar), 1);
    for (int s = 0; s < kStages; ++s) {
      mbar_init(smem_u32(&sm->q_full[s]), 1);
      mbar_init(smem_u32(&sm->q_empty[s]), 1);
      mbar_init(smem_u32(&sm->do_full[s]), 1);
      mbar_init(smem_u32(&sm->do_empty[s]), 1);
      mbar_init(smem_u32(&sm->stat_full[s]), 32);
    }
    for (uint64_t* bar : {&sm->p_ready, &sm->ds_ready}) mbar_init(smem_u32(bar), kBwdWarps * 32);
    for (int g = 0; g < 2; ++g) {
      mbar_init(smem_u32(&sm->acc_full[g]), 1);
      mbar_init(smem_u32(&sm->acc_empty[g]), kBwdWarps * 16);
    }
    for (int s = 0; s < kDealt; ++s) {
      sm->dealt[s] = INT32_MAX;                    // no unit: what a reader finds whose wait ran out before a number came
      mbar_init(smem_u32(&sm->dealt_full[s]), 1);
      mbar_init(smem_u32(&sm->dealt_empty[s]), kBwdWarps + 1);
    }
    mbar_init_fence();
  }
  if (warp == kBwdWarps + 1) tmem_alloc(smem_u32(&sm->tmem_base), 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = (uint32_t)warp_uniform((int)sm->tmem_base);
  const uint32_t tmem_s = tmem, tmem_dp = tmem + 128u, tmem_dv = tmem + 256u, tmem_dk = tmem + 256u + kD;
  auto dealt = [&](int r, int where) {             // number of the CTA's r-th unit
    mbar_wait(smem_u32(&sm->dealt_full[r % kDealt]), (r / kDealt) & 1, status, where);
    const int w = warp_uniform(sm->dealt[r % kDealt]);
    __syncwarp();
    if (lane == 0) mbar_arrive(smem_u32(&sm->dealt_empty[r % kDealt]));
    return w;
  };
  // A operand of K-step kk (16 queries) of P^T / dS^T: a warpgroup's 32 queries sit in the first 16 of their 32 columns
  auto a_step = [](int kk) { return (uint32_t)((kk >> 1) * kCols + (kk & 1) * 8); };

  if (warp == kBwdWarps) {
    // ------------------------------------------------------------------ loads: lane 0 issues TMA, all lanes bring the statistics
    int it = 0, u = 0, patches = 0;
    auto deal = [&](int r, int w) {
      mbar_wait(smem_u32(&sm->dealt_empty[r % kDealt]), ((r / kDealt) & 1) ^ 1, status, kErrDkvProducer);
      if (lane == 0) {
        sm->dealt[r % kDealt] = w;
        mbar_arrive(smem_u32(&sm->dealt_full[r % kDealt]));
      }
      __syncwarp();
    };
    auto ask_unit = [&]() {
      int w = 0;
      if (lane == 0) w = gridDim.x + atomicAdd(p.next, 1);
      return __shfl_sync(0xffffffffu, w, 0);
    };
    // the others get no unit without items: their keys' gradients, zeros, come from the dQ kernel
    auto with_items = [&](int w) {
      while (w < n_units && unit_of(w).n_q == 0) w = ask_unit();
      return w;
    };
    int w_next = with_items(blockIdx.x);
    deal(0, w_next);
    for (int r = 0, w = w_next; w < n_units; w = w_next, ++r) {
      const DkvUnit un = unit_of(w);
      const int n_items = un.n_q * p.G;
      auto load_pair = [&](uint32_t dst, const CUtensorMap* tm, uint64_t* full, uint64_t* empty) {
        const uint32_t fb = smem_u32(full);
        mbar_wait(smem_u32(empty), (u & 1) ^ 1, status, kErrDkvProducer);
        if (lane == 0) {
          mbar_arrive_expect_tx(fb, kOperand);
          for (int g = 0; g < 2; ++g)
            for (int c = 0; c < kD / 64; ++c)
              tma_load_4d(dst + c * kTileBytes + g * kHalfTile, tm, fb, 64 * c, un.pair * kPair + g * kBlk, un.hk, un.b);
        }
        __syncwarp();
      };
      auto load_rows = [&](uint32_t dst, const CUtensorMap* tm, uint64_t* full, uint64_t* empty, int h, int tile) {
        mbar_wait(smem_u32(empty), ((it / kStages) & 1) ^ 1, status, kErrDkvProducer);
        const int rows = un.len - off - tile * kQTile;            // rows of the tile that the sequence has
        const bool ends = rows < kQTile && un.len < p.Lk;
        const uint32_t fb = smem_u32(ends ? &sm->patch : full);
        if (lane == 0) {
          mbar_arrive_expect_tx(fb, kOperand);
          for (int c = 0; c < kD / 64; ++c) tma_load_4d(dst + c * kTileBytes, tm, fb, 64 * c, tile * kQTile, h, un.b);
        }
        __syncwarp();
        if (ends) {
          mbar_wait(fb, patches++ & 1, status, kErrDkvProducer);
          zero_rows(dst, kTileBytes, kD / 64, rows, kQTile, lane);
          if (lane == 0) mbar_arrive(smem_u32(full));
        }
      };
      float4 nl, nd;
      auto ask = [&](int i) {                      // statistics of an item's rows 4 lane .. 4 lane + 3, one item ahead
        const int g = i / un.n_q, tile = un.first + i - g * un.n_q, row = tile * kQTile + lane * 4;
        const int64_t at = ((int64_t)un.b * p.H + un.hk * p.G + g) * p.Lq + row;
        float l[4], d[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const bool valid = off + row + e < un.len;
          l[e] = valid ? -ld_behind_wait(p.lse + at + e) : -INFINITY;
          d[e] = valid ? -p.scale * ld_behind_wait(p.delta + at + e) : 0.f;
        }
        nl = make_float4(l[0], l[1], l[2], l[3]);
        nd = make_float4(d[0], d[1], d[2], d[3]);
      };
      load_pair(k_pair, &tm_k, &sm->k_full, &sm->k_empty);
      for (int i = 0; i < n_items; ++i, ++it) {
        const int s = it % kStages, g = i / un.n_q, h = un.hk * p.G + g, tile = un.first + i - g * un.n_q;
        load_rows(q_slot(s), &tm_q, &sm->q_full[s], &sm->q_empty[s], h, tile);
        if (i == 0) load_pair(v_pair, &tm_v, &sm->v_full, &sm->v_empty);
        if (i == 0) {
          w_next = with_items(ask_unit());
          deal(r + 1, w_next);
          ask(0);
        }
        *reinterpret_cast<float4*>(&sm->nlse[s][lane * 4]) = nl;
        *reinterpret_cast<float4*>(&sm->ndelta[s][lane * 4]) = nd;
        mbar_arrive(smem_u32(&sm->stat_full[s]));
        if (i + 1 < n_items) ask(i + 1);
        load_rows(do_slot(s), &tm_do, &sm->do_full[s], &sm->do_empty[s], h, tile);
      }
      ++u;
    }
    __syncwarp();
  } else if (warp == kBwdWarps + 1) {
    // ------------------------------------------------------------------ all four products, A of dV and dK from TMEM
    // One warp issues them: S of the next item right behind dV, which reads the P that stands in its place, and dP right behind dK.
    // The tensor core works through what one thread issues in order, so neither waits for the other's end; with two issuing
    // warps and barriers between them an item's time was mostly the way from a product's end to the next one's start.
    constexpr uint32_t fmt = kBf16 ? 1u : 0u;
    constexpr uint32_t idesc_s = instr_desc_f16(fmt, 128, 128, 0, 0), idesc_t = instr_desc_f16(fmt, 128, kD, 0, 1);
    const uint64_t dk0 = smem_desc_sw128(k_pair, 16, 1024), dv0 = smem_desc_sw128(v_pair, 16, 1024);
    const uint64_t dq0 = smem_desc_sw128(q_slot(0), 16, 1024), ddo0 = smem_desc_sw128(do_slot(0), 16, 1024);
    const uint64_t dq0t = smem_desc_sw128(q_slot(0), kTileBytes, 1024), ddo0t = smem_desc_sw128(do_slot(0), kTileBytes, 1024);
    struct Cursor { int i, n, u; };                // item i of n in the u-th unit; n = 0: no more
    auto advance = [&](Cursor& c) {
      if (++c.i < c.n) return;
      c.i = 0;
      const int w = dealt(++c.u, kErrDkvMma);
      c.n = w < n_units ? warp_uniform(unit_of(w).n_q) * p.G : 0;
    };
    auto slot = [&](uint64_t d, int it) { return desc_advance(d, (uint32_t)(it % kStages) * 2 * kOperand); };
    auto issue_s = [&](const Cursor& c, int it) {
      if (c.i == 0) mbar_wait(smem_u32(&sm->k_full), c.u & 1, status, kErrDkvMma);
      mbar_wait(smem_u32(&sm->q_full[it % kStages]), (it / kStages) & 1, status, kErrDkvMma);
      tc_fence_after();
      const uint64_t dq = slot(dq0, it);
      if (elect_one()) {
#pragma unroll
        for (int kk = 0; kk < kD / 16; ++kk)
          mma_f16_ss(tmem_s, desc_advance(dk0, kmajor_step(kk, kTileBytes)), desc_advance(dq, kmajor_step(kk, kTileBytes)), idesc_s, kk > 0);
        mma_commit(smem_u32(&sm->s_full));
        if (c.i == c.n - 1) mma_commit(smem_u32(&sm->k_empty));
      }
    };
    auto issue_dp = [&](const Cursor& c, int it) {
      if (c.i == 0) mbar_wait(smem_u32(&sm->v_full), c.u & 1, status, kErrDkvMma);
      mbar_wait(smem_u32(&sm->do_full[it % kStages]), (it / kStages) & 1, status, kErrDkvMma);
      tc_fence_after();
      const uint64_t ddo = slot(ddo0, it);
      if (elect_one()) {
#pragma unroll
        for (int kk = 0; kk < kD / 16; ++kk)
          mma_f16_ss(tmem_dp, desc_advance(dv0, kmajor_step(kk, kTileBytes)), desc_advance(ddo, kmajor_step(kk, kTileBytes)), idesc_s, kk > 0);
        mma_commit(smem_u32(&sm->dp_full));
        if (c.i == c.n - 1) mma_commit(smem_u32(&sm->v_empty));
      }
    };
    Cursor now = {0, 0, -1};
    advance(now);
    if (now.n > 0) {
      issue_s(now, 0);
      issue_dp(now, 0);
    }
    for (int it = 0; now.n > 0; ++it) {
      const int s = it % kStages;
      Cursor next = now;
      advance(next);
      if (now.i == 0) mbar_wait(smem_u32(&sm->acc_empty[0]), (now.u & 1) ^ 1, status, kErrDkvMma);
      mbar_wait(smem_u32(&sm->p_ready), it & 1, status, kErrDkvMma);
      tc_fence_after();
      const uint64_t ddot = slot(ddo0t, it), dqt = slot(dq0t, it);
      if (elect_one()) {
#pragma unroll
        for (int kk = 0; kk < kQTile / 16; ++kk)
          mma_f16_ts(tmem_dv, tmem_s + a_step(kk), desc_advance(ddot, kk * 2048), idesc_t, (now.i > 0 || kk > 0) ? 1u : 0u);
        mma_commit(smem_u32(&sm->do_empty[s]));
        if (now.i == now.n - 1) mma_commit(smem_u32(&sm->acc_full[0]));
      }
      if (next.n > 0) issue_s(next, it + 1);
      if (now.i == 0) mbar_wait(smem_u32(&sm->acc_empty[1]), (now.u & 1) ^ 1, status, kErrDkvMma);
      mbar_wait(smem_u32(&sm->ds_ready), it & 1, status, kErrDkvMma);
      tc_fence_after();
      if (elect_one()) {
#pragma unroll
        for (int kk = 0; kk < kQTile / 16; ++kk)
          mma_f16_ts(tmem_dk, tmem_dp + a_step(kk), desc_advance(dqt, kk * 2048), idesc_t, (now.i > 0 || kk > 0) ? 1u : 0u);
        mma_commit(smem_u32(&sm->q_empty[s]));
        if (now.i == now.n - 1) mma_commit(smem_u32(&sm->acc_full[1]));
      }
      if (next.n > 0) issue_dp(next, it + 1);
      now = next;
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------------ softmax: lane = key of the pair, warpgroup = 32 queries of the tile
    const int g = warp >> 2;
    const int row = tid & 127;
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t ts = tmem_s + (uint32_t)g * kCols + lane_base, tdp = tmem_dp + (uint32_t)g * kCols + lane_base;
    int it = 0, u = 0;
    for (int w = dealt(0, kErrDkvSoftmax); w < n_units; w = dealt(++u, kErrDkvSoftmax)) {
      const DkvUnit un = unit_of(w);
      const int n_items = un.n_q * p.G, bk = un.b * p.Hkv + un.hk, key = un.pair * kPair + row;
      const bool split = un.pair < p.split.tiles;
      float* const part = split ? p.split.part + (((int64_t)bk * p.split.tiles + un.pair) * (1 + p.split.runs) + 1 + un.run) * 2 * kPair * p.D : nullptr;
      // this thread's part of the results: warpgroups 0, 1 the halves of dV's features, 2, 3 of dK's
      constexpr int kOut = kD / 2;
      const bool is_dv = g < 2;
      const int col0 = (g & 1) * kOut;
      const int kmin = warp_uniform(un.pair * kPair + (warp & 3) * 32), kmax = kmin + 31;
      const int frow = kmin + (lane >> 2), fcol = 2 * (lane & 3);      // fragments: keys frow + 8 e, queries fcol + 8 j and the next
      for (int i = 0, tq = un.first; i < n_items; ++i, ++it) {
        const int s = it % kStages, p0 = off + tq * kQTile + g * kCols, p1 = p0 + kCols - 1;      // positions of the columns
        if (++tq == un.first + un.n_q) tq = un.first;
        const int kind = p0 >= un.len || none_seen(p0, p1, kmin, kmax, p.window, p.sinks) ? 0
                         : p1 < un.len && all_seen(p0, p1, kmin, kmax, p.window, p.sinks) ? 2 : 1;
        const uint64_t* const nl = reinterpret_cast<const uint64_t*>(&sm->nlse[s][g * kCols + fcol]);
        const uint64_t* const nd = reinterpret_cast<const uint64_t*>(&sm->ndelta[s][g * kCols + fcol]);
        mbar_wait(smem_u32(&sm->stat_full[s]), (it / kStages) & 1, status, kErrDkvSoftmax);
        mbar_wait(smem_u32(&sm->s_full), it & 1, status, kErrDkvSoftmax);
        tc_fence_after();
        uint64_t sp[2][8];                         // [16 lanes][pair 2 j + e]
        uint32_t wd[2][8];
        if (kind != 0) {
          load_fragments(sp, ts);
          uint64_t l2[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) l2[j] = nl[4 * j];
          const uint64_t c2 = pk2(p.scale_log2, p.scale_log2);
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int k = 0; k < 8; ++k) sp[h][k] = fma2(sp[h][k], c2, l2[k >> 1]);
          if (kind == 2) {
            // polynomials make finite numbers of NaN: a row that has one has it in its lse too, from where it reaches the weight
            const uint64_t zero = pk2(0.f, 0.f);
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int k = 0; k < 8; ++k)
                sp[h][k] = k % kBwdPolyEvery == 1 ? fma2(l2[k >> 1], zero, ex2_poly2<3>(sp[h][k])) : ex2_pair(sp[h][k]);
          } else {
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const int key_r = frow + 16 * h + 8 * e, first = key_r - p0 - fcol;       // the key is seen from columns first .. end - 1
                const int end = min(key_r < p.sinks ? INT32_MAX / 2 : key_r + p.window, un.len) - p0 - fcol;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                  float x, y;
                  upk2(sp[h][2 * j + e], x, y);
                  sp[h][2 * j + e] = pk2(8 * j >= first && 8 * j < end ? ex2(x) : 0.f, 8 * j + 1 >= first && 8 * j + 1 < end ? ex2(y) : 0.f);
                }
              }
          }
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int k = 0; k < 8; ++k) wd[h][k] = pack2p<kBf16>(sp[h][k]);
        } else {
#pragma unroll
          for (int k = 0; k < 8; ++k) wd[0][k] = wd[1][k] = 0u;
        }
        store_fragments(wd, ts);
        tc_fence_before();
        mbar_arrive(smem_u32(&sm->p_ready));
        mbar_wait(smem_u32(&sm->dp_full), it & 1, status, kErrDkvSoftmax);
        tc_fence_after();
        if (kind != 0) {
          uint64_t dp[2][8];
          load_fragments(dp, tdp);
          uint64_t d2[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) d2[j] = nd[4 * j];
          const uint64_t s2 = pk2(p.scale, p.scale);
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              uint64_t x = mul2(sp[h][k], fma2(dp[h][k], s2, d2[k >> 1]));
              if (kind == 1) {                     // a key behind the end may hold anything: dropped, not multiplied by 0
                float x0, x1, w0, w1;
                upk2(x, x0, x1);
                upk2(sp[h][k], w0, w1);
                x = pk2(w0 == 0.f ? 0.f : x0, w1 == 0.f ? 0.f : x1);
              }
              wd[h][k] = pack2p<kBf16>(x);
            }
        }
        store_fragments(wd, tdp);                  // (kind 0: still zeros)
        tc_fence_before();
        mbar_arrive(smem_u32(&sm->ds_ready));
      }
      // epilogue
      // a run's rows see the sinks alone, and the sinks' sums are joined later
      const bool sink = split && key < p.sinks;
      const int64_t off_r = key < p.Lk && !sink ? ((int64_t)bk * p.Lk + key) * p.D : -1;
      int64_t row_off[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) row_off[j] = __shfl_sync(0xffffffffu, off_r, (lane & ~3) + j);
      const int acc = is_dv ? 0 : 1;
      mbar_wait(smem_u32(&sm->acc_full[acc]), u & 1, status, kErrDkvEpilogue);
      tc_fence_after();
      const uint32_t t_acc = (is_dv ? tmem_dv : tmem_dk) + col0 + lane_base;
      float* const prow = split ? part + ((is_dv ? kPair : 0) + row) * p.D : nullptr;
#pragma unroll
      for (int c = 0; c < kOut / 32; ++c) {
        uint32_t ra[32];
        tmem_ld_32x32b_x32(t_acc + c * 32, ra);
        tmem_ld_wait();
        if (c == kOut / 32 - 1) {
          tc_fence_before();
          mbar_arrive(smem_u32(&sm->acc_empty[acc]));     // the next unit may start accumulating
        }
        if (sink) {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (col0 + c * 32 + e * 4 < p.D)
              *reinterpret_cast<uint4*>(prow + col0 + c * 32 + e * 4) = make_uint4(ra[4 * e], ra[4 * e + 1], ra[4 * e + 2], ra[4 * e + 3]);
        }
        __syncwarp();
        if (un.base()) store_acc_cols<kBf16>(is_dv ? p.dv : p.dk, row_off, ra, col0 + c * 32, p.D, lane);
        __syncwarp();
      }
    }
    grid_dep_wait();                               // a CTA without units, too, ends behind the kernel in front
    tc_fence_before();
  }
  __syncthreads();
  if (warp == kBwdWarps + 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ---------------------------------------------------------------------------------------------- backward: delta = rowsum(O dO)
// with what the rounding of O left: without it a row of dS would miss its sum of 0 by as much as dS's own rounding is off, and dQ and dK
// had 1.46 to 1.53 instead of 1.43 to 1.46 times the error of their own rounding (lengths of 700 and 2048, both types).  Bound by memory; in the dQ kernel the tiles of O and of the rest took
// the places of key tiles on their way (training size 46 -> 53 us), and the dK/dV kernel had to wait for the last of its CTAs.
struct DeltaArgs {
  const void *o, *dO;
  const uint8_t* rest;
  float* delta;
  int* next;                // set to 0 for the dK/dV kernel
  const int* lengths;
  int BH, H, Lq, Lk, D;
  int64_t dos[3];
};
constexpr int kDeltaThreads = 256, kDeltaSteps = 4;

template <bool kBf16, int kD>
__global__ void __launch_bounds__(kDeltaThreads, 4) window_delta_kernel(const __grid_constant__ DeltaArgs p) {
  constexpr int kLanes = kD / 8, kRows = kDeltaThreads / kLanes;      // lanes of a row, rows a step
  grid_dep_wait();
  grid_dep_launch();
  if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) *p.next = 0;
  const int bh = blockIdx.y, b = bh / p.H, h = bh - b * p.H, f = threadIdx.x % kLanes * 8;
  const int len = length_of(p.lengths, b, p.Lk) - (p.Lk - p.Lq);      // rows that are some
  const int row0 = blockIdx.x * kRows * kDeltaSteps + threadIdx.x / kLanes;
  const uint16_t* const dO = reinterpret_cast<const uint16_t*>(p.dO) + b * p.dos[0] + h * p.dos[1] + f;
  uint4 x[kDeltaSteps], g[kDeltaSteps];
  uint2 y[kDeltaSteps];
#pragma unroll
  for (int e = 0; e < kDeltaSteps; ++e) {
    const int row = row0 + e * kRows;
    x[e] = g[e] = make_uint4(0u, 0u, 0u, 0u);
    y[e] = make_uint2(0u, 0u);
    if (row < min(len, p.Lq) && f < p.D) {
      const int64_t at = ((int64_t)bh * p.Lq + row) * p.D + f;
      x[e] = ld_behind_wait(reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(p.o) + at));
      y[e] = ld_behind_wait(reinterpret_cast<const uint2*>(p.rest + at));
      g[e] = ld_behind_wait(reinterpret_cast<const uint4*>(dO + row * p.dos[2]));
    }
  }
#pragma unroll
  for (int e = 0; e < kDeltaSteps; ++e) {
    const uint32_t xs[4] = {x[e].x, x[e].y, x[e].z, x[e].w}, ys[2] = {y[e].x, y[e].y}, gs[4] = {g[e].x, g[e].y, g[e].z, g[e].w};
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float2 fx = restored2<kBf16>(xs[w], ys[w / 2], 2 * (w & 1)), fg = unpack2<kBf16>(gs[w]);
      sum = fmaf(fx.x, fg.x, sum);
      sum = fmaf(fx.y, fg.y, sum);
    }
#pragma unroll
    for (int d = kLanes / 2; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    const int row = row0 + e * kRows;
    if (f == 0 && row < p.Lq) p.delta[(int64_t)bh * p.Lq + row] = sum;
  }
}

// ---------------------------------------------------------------------------------------------- backward: dQ
// One persistent CTA an SM; a unit is 128 query rows of a head, an item 64 keys.  A comes from TMEM in all three products (Q and dO rows are brought
// there once a unit, dS stands over dP), so shared memory feeds the B side alone.  Two pairs of warpgroups take the items in turn; the pair
// that a unit's last item leaves free brings the next unit's rows, whose first S and dP are under way before this one's dQ is written out
// (training size 53 -> 46 us with it and with masks as words, 43 with delta elsewhere).  A full item takes 1300 clk against 768 of
// products: the softmax warps' way from S to dS.  (Two CTAs an SM with operands in shared memory: 78 us; three stages of K and V: 52.)
constexpr int kDqK = 6, kDqV = 4;                   // tiles of keys (kept until dQ has been formed) and of values (until dP has)
constexpr int kSdpBufs = 2;                         // S / dP buffers in TMEM
constexpr int kDqThreads = (kBwdWarps + 2) * 32;

struct DqSmem {
  // [2]: units in turn.  A pair of warpgroups that has no item of a unit sees nothing of it, and a parity tells only neighbouring phases
  // apart: with one barrier the pair took rows for its next unit's that had not arrived.  Of the unit two before, it always had a part.
  uint64_t qdo_full[2], patch;
  uint64_t ops_ready;       // the unit's Q and dO rows sit in TMEM (written by the pair of warpgroups that takes its first item)
  uint64_t ops_free[2];     // the S / dP products of the unit have read them
  uint64_t rows_read;       // and are no longer needed in shared memory
  uint64_t k_full[kDqK], k_empty[kDqK], v_full[kDqV], v_empty[kDqV];
  uint64_t s_full[kSdpBufs], s_free[kSdpBufs], dp_full[kSdpBufs];
  uint64_t ds_ready[kSdpBufs];                         // dS has taken dP's place
  uint64_t acc_full[2];     // per draining pair of warpgroups (the one that took the unit's last item)
  uint64_t acc_empty;
  uint32_t tmem_base;
};
struct DqArgs {
  const float *lse, *delta;
  void *dq, *dk, *dv;       // dk, dv: rows that no query sees
  const int* lengths;
  int H, Hkv, G, BH, Lq, Lk, D, window, sinks, n_pairs;
  float scale, scale_log2;
  SinkSplit split;
};

template <bool kBf16, int kD>
__global__ void __launch_bounds__(kDqThreads, 1)
window_dq_sm100_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                       const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_do,
                       const __grid_constant__ DqArgs p, int* status) {
  extern __shared__ __align__(1024) uint8_t smem_aligned[];
  const uint32_t base = smem_u32(smem_aligned);
  if ((base & 1023u) != 0) {                         // the swizzle needs it
    if (threadIdx.x == 0) atomicCAS(status, 0, kErrDqProducer);
    return;
  }
  const uint32_t q_tile = base, do_tile = base + 32768u;
  auto k_slot = [&](int s) { return base + 65536u + (uint32_t)s * 16384u; };
  auto v_slot = [&](int s) { return base + 65536u + (uint32_t)(kDqK + s) * 16384u; };
  DqSmem* sm = reinterpret_cast<DqSmem*>(smem_aligned + 65536u + (kDqK + kDqV) * 16384u);

  const int tid = threadIdx.x, warp = warp_uniform(tid >> 5), lane = tid & 31;
  const int n_tiles = (p.Lq + kQTile - 1) / kQTile, off = p.Lk - p.Lq, n_units = n_tiles * p.BH;
  auto unit_of = [&](int w) { return row_unit(w, n_tiles, p.BH, p.H, p.lengths, p.Lq, p.Lk, p.window, p.sinks); };

  if (tid == 0) {
    for (const CUtensorMap* tm : {&tm_q, &tm_k, &tm_v, &tm_do}) prefetch_tensormap(tm);
    for (uint64_t* bar : {&sm->qdo_full[0], &sm->qdo_full[1], &sm->ops_free[0], &sm->ops_free[1], &sm->patch}) mbar_init(smem_u32(bar), 1);
    mbar_init(smem_u32(&sm->ops_ready), 256);
    mbar_init(smem_u32(&sm->rows_read), 256);
    for (int s = 0; s < kDqK; ++s) {
      mbar_init(smem_u32(&sm->k_full[s]), 1);
      mbar_init(smem_u32(&sm->k_empty[s]), 1);
    }
    for (int s = 0; s < kDqV; ++s) {
      mbar_init(smem_u32(&sm->v_full[s]), 1);
      mbar_init(smem_u32(&sm->v_empty[s]), 1);
    }
    for (int s = 0; s < kSdpBufs; ++s) {
      mbar_init(smem_u32(&sm->ds_ready[s]), 256);
      mbar_init(smem_u32(&sm->s_full[s]), 1);
      mbar_init(smem_u32(&sm->s_free[s]), 256);
      mbar_init(smem_u32(&sm->dp_full[s]), 1);
    }
    mbar_init(smem_u32(&sm->acc_full[0]), 1);
    mbar_init(smem_u32(&sm->acc_full[1]), 1);
    mbar_init(smem_u32(&sm->acc_empty), 256);
    mbar_init_fence();
  }
  if (warp == kBwdWarps + 1) tmem_alloc(smem_u32(&sm->tmem_base), 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = (uint32_t)warp_uniform((int)sm->tmem_base);
  // TMEM: S buffers [0,128), dP buffers [128,256), dQ [256,384), Q rows [384,448), dO rows [448,512)
  const uint32_t tmem_s = tmem, tmem_dp = tmem + 128, tmem_dq = tmem + 256, tmem_q = tmem + 384, tmem_do = tmem + 448;

  if (warp == kBwdWarps) {
    // ------------------------------------------------------------------ TMA producer
    int it = 0, u = 0, patches = 0;
    for (int r = 0, w = unit_at(0); w < n_units; w = unit_at(++r)) {
      const RowUnit un = unit_of(w);
      if (un.total == 0) continue;
      const int hk = un.h / p.G;
      const uint32_t qb = smem_u32(&sm->qdo_full[u & 1]);
      mbar_wait(smem_u32(&sm->rows_read), (u & 1) ^ 1, status, kErrDqProducer);
      if (lane == 0) {
        mbar_arrive_expect_tx(qb, 2 * (kD / 64) * kTileBytes);
        for (int c = 0; c < kD / 64; ++c) {
          tma_load_4d(q_tile + c * kTileBytes, &tm_q, qb, 64 * c, un.t * kQTile, un.h, un.b);
          tma_load_4d(do_tile + c * kTileBytes, &tm_do, qb, 64 * c, un.t * kQTile, un.h, un.b);
        }
      }
      __syncwarp();
      for (int i = 0; i < un.total; ++i, ++it) {
        const int sk = it % kDqK, sv = it % kDqV, key0 = un.tile_of(i) * kBlk;
        const bool ends = key0 + kBlk > un.len && un.len < p.Lk;
        const uint32_t kb = smem_u32(ends ? &sm->patch : &sm->k_full[sk]), vb = smem_u32(&sm->v_full[sv]);
        mbar_wait(smem_u32(&sm->k_empty[sk]), ((it / kDqK) & 1) ^ 1, status, kErrDqProducer);
        if (lane == 0) {
          mbar_arrive_expect_tx(kb, (kD / 64) * kHalfTile);
          for (int c = 0; c < kD / 64; ++c) tma_load_4d(k_slot(sk) + c * kHalfTile, &tm_k, kb, 64 * c, key0, hk, un.b);
        }
        __syncwarp();
        if (ends) {                                // dS is 0 there, and dQ += dS K
          mbar_wait(kb, patches++ & 1, status, kErrDqProducer);
          zero_rows(k_slot(sk), kHalfTile, kD / 64, un.len - key0, kBlk, lane);
          if (lane == 0) mbar_arrive(smem_u32(&sm->k_full[sk]));
        }
        mbar_wait(smem_u32(&sm->v_empty[sv]), ((it / kDqV) & 1) ^ 1, status, kErrDqProducer);
        if (lane == 0) {
          mbar_arrive_expect_tx(vb, (kD / 64) * kHalfTile);
          for (int c = 0; c < kD / 64; ++c) tma_load_4d(v_slot(sv) + c * kHalfTile, &tm_v, vb, 64 * c, key0, hk, un.b);
        }
        __syncwarp();
      }
      ++u;
    }
    __syncwarp();
  } else if (warp == kBwdWarps + 1) {
    // ------------------------------------------------------------------ all three products, two items ahead with S and dP
    // One warp issues them: dP of item i + 2 right behind dQ of item i, which reads the dS that stands in its place (see the dK/dV kernel).
    constexpr uint32_t fmt = kBf16 ? 1u : 0u;
    constexpr uint32_t idesc_s = instr_desc_f16(fmt, 128, 64, 0, 0), idesc_q = instr_desc_f16(fmt, 128, kD, 0, 1);
    const uint64_t dk0 = smem_desc_sw128(k_slot(0), 16, 1024), dv0 = smem_desc_sw128(v_slot(0), 16, 1024);
    const uint64_t dk0t = smem_desc_sw128(k_slot(0), kHalfTile, 1024);
    struct Cursor { int r, i, n, u; };             // item i of n in the u-th unit that has any; n = 0: no more
    auto advance = [&](Cursor& c) {
      if (++c.i < c.n) return;
      c.i = 0;
      c.n = 0;
      ++c.u;
      for (;;) {
        const int w = unit_at(++c.r);
        if (w >= n_units) return;
        c.n = warp_uniform(unit_of(w).total);
        if (c.n > 0) return;
      }
    };
    auto k_of = [&](uint64_t d, int it) { return desc_advance(d, (uint32_t)(it % kDqK) * 16384u); };
    auto issue_s = [&](const Cursor& c, int it) {
      const int sb = it % kSdpBufs;
      mbar_wait(smem_u32(&sm->k_full[it % kDqK]), (it / kDqK) & 1, status, kErrDqMma);
      if (it >= kSdpBufs) mbar_wait(smem_u32(&sm->s_free[sb]), ((it / kSdpBufs) & 1) ^ 1, status, kErrDqMma);
      if (c.i == 0) mbar_wait(smem_u32(&sm->ops_ready), c.u & 1, status, kErrDqMma);
      tc_fence_after();
      const uint64_t db = k_of(dk0, it);
      if (elect_one()) {
#pragma unroll
        for (int kk = 0; kk < kD / 16; ++kk)      // A from TMEM: 8 columns = 16 features per K-step
          mma_f16_ts(tmem_s + sb * 64, tmem_q + kk * 8, desc_advance(db, kmajor_step(kk, kHalfTile)), idesc_s, kk > 0);
        mma_commit(smem_u32(&sm->s_full[sb]));
      }
    };
    auto issue_dp = [&](const Cursor& c, int it) {
      const int sb = it % kSdpBufs;
      mbar_wait(smem_u32(&sm->v_full[it % kDqV]), (it / kDqV) & 1, status, kErrDqMma);
      tc_fence_after();
      const uint64_t db = desc_advance(dv0, (uint32_t)(it % kDqV) * 16384u);
      if (elect_one()) {
#pragma unroll
        for (int kk = 0; kk < kD / 16; ++kk)
          mma_f16_ts(tmem_dp + sb * 64, tmem_do + kk * 8, desc_advance(db, kmajor_step(kk, kHalfTile)), idesc_s, kk > 0);
        mma_commit(smem_u32(&sm->dp_full[sb]));
        mma_commit(smem_u32(&sm->v_empty[it % kDqV]));
        if (c.i == c.n - 1) mma_commit(smem_u32(&sm->ops_free[c.u & 1]));        // the next unit's Q / dO rows may be written
      }
    };
    Cursor now = {-1, 0, 0, -1};
    advance(now);
    Cursor ahead = now;
    for (int j = 0; j < kSdpBufs && ahead.n > 0; ++j) {
      issue_s(ahead, j);
      issue_dp(ahead, j);
      advance(ahead);
    }
    for (int it = 0; now.n > 0; ++it) {
      const int sb = it % kSdpBufs, next = it + kSdpBufs;
      // S goes ahead of dQ but for a unit's first item: its rows come behind this item's dS, from the same warpgroups
      const bool early = ahead.n > 0 && ahead.i > 0;
      if (early) issue_s(ahead, next);
      if (now.i == 0) mbar_wait(smem_u32(&sm->acc_empty), (now.u & 1) ^ 1, status, kErrDqMma);
      mbar_wait(smem_u32(&sm->ds_ready[sb]), (it / kSdpBufs) & 1, status, kErrDqMma);
      tc_fence_after();
      const uint64_t dkt = k_of(dk0t, it);
      if (elect_one()) {
#pragma unroll
        for (int kk = 0; kk < kBlk / 16; ++kk)
          mma_f16_ts(tmem_dq, tmem_dp + sb * 64 + (kk >> 1) * kCols + (kk & 1) * 8, desc_advance(dkt, kk * 2048), idesc_q,
                     (now.i > 0 || kk > 0) ? 1u : 0u);
        mma_commit(smem_u32(&sm->k_empty[it % kDqK]));
        if (now.i == now.n - 1) mma_commit(smem_u32(&sm->acc_full[it & 1]));     // drained by the pair that took the last item
      }
      if (ahead.n > 0) {
        if (!early) issue_s(ahead, next);
        issue_dp(ahead, next);
        advance(ahead);
      }
      advance(now);
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------------ softmax: warpgroups 2 e, 2 e + 1 take the items with (running count) % 2 == e,
    // 32 columns each
    const int g = warp >> 2, pair = g >> 1, half = g & 1;
    const int row = tid & 127;
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    int it0 = 0, u = 0, drains = 0;
    // dQ of a unit is drained by the pair that took its last item, half of the features each; the other pair has brought the next unit's
    // rows to TMEM meanwhile
    constexpr int kOut = kD / 2;
    int64_t drain_row = -1;
    bool drain_stored = false, drain_valid = false;
    auto drain = [&]() {
      mbar_wait(smem_u32(&sm->acc_full[pair]), drains & 1, status, kErrDqEpilogue);
      ++drains;
      tc_fence_after();
      int64_t row_off[4];
      {
        const int64_t at = drain_stored ? drain_row * p.D : -1;
#pragma unroll
        for (int j = 0; j < 4; ++j) row_off[j] = __shfl_sync(0xffffffffu, at, (lane & ~3) + j);
      }
#pragma unroll
      for (int c = 0; c < kOut / 32; ++c) {
        const int col = half * kOut + c * 32;
        uint32_t r[32];
        tmem_ld_32x32b_x32(tmem_dq + col + lane_base, r);
        tmem_ld_wait();
        if (c == kOut / 32 - 1) {
          tc_fence_before();
          mbar_arrive(smem_u32(&sm->acc_empty));     // the next unit may start accumulating
        }
#pragma unroll
        for (int e = 0; e < 32; ++e) r[e] = drain_valid ? r[e] : 0u;
        store_acc_cols<kBf16>(p.dq, row_off, r, col, p.D, lane);
        __syncwarp();
      }
      drain_row = -1;
    };
    // row statistics of the next unit are asked for while the current one runs
    float n_lse = 0.f, n_delta = 0.f;
    auto fetch_rows = [&](int w) {
      if (w >= n_units) return;
      const int rr = min((n_tiles - 1 - w / p.BH) * kQTile + row, p.Lq - 1);
      n_lse = ld_behind_wait(p.lse + (int64_t)(w % p.BH) * p.Lq + rr);
      n_delta = ld_behind_wait(p.delta + (int64_t)(w % p.BH) * p.Lq + rr);
    };
    // delta comes from the kernel in front, what else is read was complete before that one's first CTA was behind its wait
    grid_dep_wait();
    grid_dep_launch();
    fetch_rows(unit_at(0));
    for (int r = 0, w = unit_at(0); w < n_units; w = unit_at(++r)) {
      const RowUnit un = unit_of(w);
      const int64_t grow = (int64_t)un.bh * p.Lq + un.t * kQTile + row;
      const int pos = off + un.t * kQTile + row;
      const bool stored = un.t * kQTile + row < p.Lq, valid = stored && pos < un.len;
      const float lse = n_lse, delta = n_delta;
      fetch_rows(unit_at(r + 1));
      if (un.total == 0) {                         // nothing but padding
        zero_fill(reinterpret_cast<uint16_t*>(p.dq) + ((int64_t)un.bh * p.Lq + un.t * kQTile) * p.D, min(kQTile, p.Lq - un.t * kQTile) * p.D / 8, tid,
                  kBwdWarps * 32);
        __syncwarp();
        continue;
      }
      const int warp_p0 = warp_uniform(off + un.t * kQTile + (warp & 3) * 32), warp_p1 = warp_p0 + 31;
      auto chunk_at = [&](int c) { return (uint32_t)(c >> 3) * kTileBytes + (uint32_t)row * 128u + (uint32_t)(((c & 7) ^ (row & 7)) << 4); };
      // The pair that takes the unit's first item moves its rows to TMEM, a warpgroup Q and the other dO: row -> lane, 32-bit word j (two
      // features) -> column j, the layout of a K-major A operand
      if (pair == (it0 & 1)) {
        mbar_wait(smem_u32(&sm->qdo_full[u & 1]), (u >> 1) & 1, status, kErrDqSoftmax);
        if (u > 0) mbar_wait(smem_u32(&sm->ops_free[(u - 1) & 1]), ((u - 1) >> 1) & 1, status, kErrDqSoftmax);
        tc_fence_after();
#pragma unroll 1
        for (int c0 = 0; c0 < kD / 8; c0 += 8) {
          uint32_t x[32];
#pragma unroll
          for (int c = 0; c < 8; ++c)
            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(x[4 * c]), "=r"(x[4 * c + 1]), "=r"(x[4 * c + 2]), "=r"(x[4 * c + 3])
                         : "r"((half == 0 ? q_tile : do_tile) + chunk_at(c0 + c)));
          tmem_st_32x32b_x32((half == 0 ? tmem_q : tmem_do) + c0 * 4 + lane_base, x);
        }
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(smem_u32(&sm->ops_ready));
        fence_proxy_async_smem();                  // TMA writes the next unit's rows through another proxy than these reads went through
        mbar_arrive(smem_u32(&sm->rows_read));
      }
      if (warp_uniform(drain_row >= 0)) drain();
      const uint64_t nl = pk2(-lse, -lse);
      const float nds = -delta * p.scale;
      const uint64_t nd = pk2(nds, nds);
      for (int i = (it0 + pair) & 1; i < un.total; i += 2) {
        const int it = it0 + i, sb = it % kSdpBufs, key0 = un.tile_of(i) * kBlk + half * kCols;
        const uint32_t seen = columns_seen(pos, key0, p.window, p.sinks);
        // a row of padding spoils its own row of dQ alone, which is not stored
        const int kind = warp_uniform(none_seen(warp_p0, warp_p1, key0, key0 + kCols - 1, p.window, p.sinks) ? 0
                                      : all_seen(warp_p0, warp_p1, key0, key0 + kCols - 1, p.window, p.sinks) ? 2 : 1);
        const uint32_t ts = tmem_s + sb * 64 + half * kCols + lane_base, tdp = tmem_dp + sb * 64 + half * kCols + lane_base;
        mbar_wait(smem_u32(&sm->s_full[sb]), (it / kSdpBufs) & 1, status, kErrDqSoftmax);
        tc_fence_after();
        uint64_t sp[kCols / 2];
        if (kind != 0) load_pairs(sp, ts);
        tc_fence_before();
        mbar_arrive(smem_u32(&sm->s_free[sb]));      // S is in registers: its buffer may take the next product
        if (kind != 0) weights_of(sp, kind, seen, p.scale_log2, nl);
        mbar_wait(smem_u32(&sm->dp_full[sb]), (it / kSdpBufs) & 1, status, kErrDqSoftmax);
        tc_fence_after();
        uint32_t wd[kCols / 2];
        if (kind != 0) {
          uint64_t dp[kCols / 2];
          load_pairs(dp, tdp);
          dscores_of<kBf16>(wd, sp, dp, kind, seen, p.scale, nd);
        } else {
#pragma unroll
          for (int j = 0; j < kCols / 2; ++j) wd[j] = 0u;
        }
        tmem_st_32x32b_x16(tdp, wd);      // dS takes the place of dP; dQ takes it from there as its A operand
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(smem_u32(&sm->ds_ready[sb]));
      }
      it0 += un.total;
      if (pair == ((it0 - 1) & 1)) {
        drain_row = grow;
        drain_stored = stored;
        drain_valid = valid;
      }
      ++u;
    }
    if (warp_uniform(drain_row >= 0)) drain();
    // Gradients of keys that nobody sees, in the time in which other CTAs have a unit more.  (In the dK/dV kernel the softmax warps reach such
    // a unit only when the one before is done, and the loading warp alone took 7000 clk for each.)
    for (int w = blockIdx.x; w < p.n_pairs * (p.BH / p.G); w += gridDim.x) {
      const int bk = w / p.n_pairs, tile = w - bk * p.n_pairs;
      const QueryTiles q = queries_of_keys(tile, kQTile, kPair, p.Lq, off, length_of(p.lengths, bk / p.Hkv, p.Lk), p.window, p.sinks);
      if ((tile < p.split.tiles ? q.last : q.end) >= q.first) continue;
      const int64_t at = ((int64_t)bk * p.Lk + tile * kPair) * p.D;
      const int n = min(kPair, p.Lk - tile * kPair) * p.D / 8;
      zero_fill(reinterpret_cast<uint16_t*>(p.dk) + at, n, tid, kBwdWarps * 32);
      zero_fill(reinterpret_cast<uint16_t*>(p.dv) + at, n, tid, kBwdWarps * 32);
      if (tile < p.split.tiles) {                    // (whose sinks' sums are joined over these rows)
        float* const part = p.split.part + ((int64_t)bk * p.split.tiles + tile) * (1 + p.split.runs) * 2 * kPair * p.D;
        zero_fill(part, 2 * kPair * p.D / 4, tid, kBwdWarps * 32);
      }
    }
    tc_fence_before();
  }
  __syncthreads();
  if (warp == kBwdWarps + 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ---------------------------------------------------------------------------------------------- host side
template <int kD> constexpr size_t kSmemFwd = (kD / 64) * (kTileBytes + kFwdSlots<kD> * kHalfTile) + sizeof(FwdSmem<kFwdSlots<kD>>);
template <int kD> constexpr size_t kSmemDkv = 1024 + (2 + 2 * kDkvStages) * (kD / 64) * kTileBytes + sizeof(DkvSmem);
constexpr size_t kSmemDq = 65536 + (kDqK + kDqV) * 16384 + sizeof(DqSmem);
static_assert(kSmemFwd<128> <= 233472 / 2 - 1024 && kSmemFwd<64> <= 233472 / 2 - 1024 && kSmemDkv<128> <= 232448 && kSmemDkv<64> <= 232448 && kSmemDq <= 232448,
              "shared memory of one SM");

struct Facts {
  bool ready = false;
  int n_sm = 0;
  int* status = nullptr;
};
// SM count, status word and the opt-in to large shared memory, once per device
int facts_of(const Facts** out) {
  static std::mutex mu;
  static Facts facts[64];
  int dev = 0, rc;
  LMK_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64) return fail(LMK_ERR_UNSUPPORTED, "device index %d out of range", dev);
  std::lock_guard<std::mutex> lock(mu);
  Facts& f = facts[dev];
  if (!f.ready) {
    if ((rc = sm_count(&f.n_sm)) != LMK_OK) return rc;
    f.status = device_status_word();
    if (f.status == nullptr) return fail(LMK_ERR_CUDA, "no device status word");
    const auto attr = cudaFuncAttributeMaxDynamicSharedMemorySize;
#define LMK_ATTRS(BF, DIM)                                                                         \
    LMK_CUDA(cudaFuncSetAttribute(window_fwd_sm100_kernel<BF, DIM>, attr, (int)kSmemFwd<DIM>));    \
    LMK_CUDA(cudaFuncSetAttribute(window_dq_sm100_kernel<BF, DIM>, attr, (int)kSmemDq));           \
    LMK_CUDA(cudaFuncSetAttribute(window_dkv_sm100_kernel<BF, DIM>, attr, (int)kSmemDkv<DIM>));
    LMK_ATTRS(true, 128) LMK_ATTRS(true, 64) LMK_ATTRS(false, 128) LMK_ATTRS(false, 64)
#undef LMK_ATTRS
    f.ready = true;
  }
  *out = &f;
  return LMK_OK;
}

int maps(const WindowParams& p, int dtype, CUtensorMap* q, CUtensorMap* k, CUtensorMap* v) {
  int rc = tensor_map_4d_now(q, p.q, dtype, p.B, p.H, p.Lq, p.D, p.qs, kQTile);
  if (rc == LMK_OK) rc = tensor_map_4d_now(k, p.k, dtype, p.B, p.Hkv, p.Lk, p.D, p.ks, kBlk);
  if (rc == LMK_OK) rc = tensor_map_4d_now(v, p.v, dtype, p.B, p.Hkv, p.Lk, p.D, p.vs, kBlk);
  return rc;
}

}  // namespace

bool window_sm100_operand_ok(const void* p, const int64_t st[3], int D) {
  return ((uintptr_t)p & 15) == 0 && st[0] > 0 && st[1] > 0 && st[0] % 8 == 0 && st[1] % 8 == 0 && st[2] % 8 == 0 && st[2] >= D;
}

int window_sm100_fwd(const WindowParams& p, int dtype, cudaStream_t st) {
  const Facts* f;
  CUtensorMap tq, tk, tv;
  int rc = facts_of(&f);
  if (rc != LMK_OK || (rc = maps(p, dtype, &tq, &tk, &tv)) != LMK_OK) return rc;
  const WindowTensors a = {p.o, static_cast<uint8_t*>(p.rest), p.lse, p.lengths, p.B * p.H, p.H, p.H / p.Hkv, p.Lq, p.Lk, p.D, p.window, p.sinks, p.scale * kLog2e};
  const int64_t units = (int64_t)((p.Lq + kQTile - 1) / kQTile) * p.B * p.H;
  int most = 2 * f->n_sm;
  const int cap = attn_sm100_max_ctas();
  if (cap >= 1 && cap < most) most = cap;
  const dim3 grid((unsigned)(units < most ? units : most));
#define LMK_FWD(BF, DIM) \
  LMK_CUDA(launch_overlapped(window_fwd_sm100_kernel<BF, DIM>, grid, dim3(kFwdThreads), kSmemFwd<DIM>, st, tq, tk, tv, a, f->status))
  if (dtype == LMK_BF16) {
    if (p.D <= 64) LMK_FWD(true, 64); else LMK_FWD(true, 128);
  } else {
    if (p.D <= 64) LMK_FWD(false, 64); else LMK_FWD(false, 128);
  }
#undef LMK_FWD
  return LMK_OK;
}

int window_sm100_bwd(const WindowParams& p, int dtype, cudaStream_t st) {
  const Facts* f;
  CUtensorMap tq, tk, tv, tdo;
  int rc = facts_of(&f);
  if (rc != LMK_OK || (rc = maps(p, dtype, &tq, &tk, &tv)) != LMK_OK) return rc;
  if ((rc = tensor_map_4d_now(&tdo, p.dO, dtype, p.B, p.H, p.Lq, p.D, p.dos, kQTile)) != LMK_OK) return rc;
  int n_sm = f->n_sm;
  const int cap = attn_sm100_max_ctas();
  if (cap >= 1 && cap < n_sm) n_sm = cap;
  const int n_pairs = (p.Lk + kPair - 1) / kPair, G = p.H / p.Hkv;
  const int64_t dq_units = (int64_t)((p.Lq + kQTile - 1) / kQTile) * p.B * p.H;
  const int64_t dkv_units = ((int64_t)n_pairs + (int64_t)p.split.tiles * p.split.runs) * p.B * p.Hkv;
  const DqArgs aq = {p.lse, p.delta, p.dq, p.dk, p.dv, p.lengths, p.H, p.Hkv, G, p.B * p.H, p.Lq, p.Lk, p.D, p.window, p.sinks, n_pairs, p.scale,
                     p.scale * kLog2e, p.split};
  const DkvArgs ak = {p.lse, p.delta, p.dk, p.dv, p.lengths, p.next, p.H, p.Hkv, G, p.B, p.Lq, p.Lk, p.D, p.window, p.sinks, n_pairs, p.scale, p.scale * kLog2e,
                      p.split};
  const dim3 grid_q((unsigned)(dq_units < n_sm ? dq_units : n_sm)), grid_k((unsigned)(dkv_units < n_sm ? dkv_units : n_sm));
  const DeltaArgs ad = {p.o, p.dO, static_cast<const uint8_t*>(p.rest), p.delta, p.next, p.lengths, p.B * p.H, p.H, p.Lq, p.Lk, p.D, {p.dos[0], p.dos[1], p.dos[2]}};
  const int delta_rows = kDeltaSteps * kDeltaThreads / ((p.D <= 64 ? 64 : 128) / 8);
  const dim3 grid_d((p.Lq + delta_rows - 1) / delta_rows, p.B * p.H);
  // The dK/dV kernel starts on every SM that the dQ kernel has left and waits for nothing: what it reads, delta included, was complete before
  // any CTA of the dQ kernel was behind its wait.  It ends behind the dQ kernel.
#define LMK_BWD(BF, DIM)                                                                                                                    \
  do {                                                                                                                                      \
    LMK_CUDA(launch_overlapped(window_delta_kernel<BF, DIM>, grid_d, dim3(kDeltaThreads), 0, st, ad));                                      \
    LMK_CUDA(launch_overlapped(window_dq_sm100_kernel<BF, DIM>, grid_q, dim3(kDqThreads), kSmemDq, st, tq, tk, tv, tdo, aq, f->status));     \
    LMK_CUDA(launch_overlapped(window_dkv_sm100_kernel<BF, DIM>, grid_k, dim3(kDkvThreads), kSmemDkv<DIM>, st, tq, tk, tv, tdo, ak, f->status)); \
  } while (0)
  if (dtype == LMK_BF16) {
    if (p.D <= 64) LMK_BWD(true, 64); else LMK_BWD(true, 128);
  } else {
    if (p.D <= 64) LMK_BWD(false, 64); else LMK_BWD(false, 128);
  }
#undef LMK_BWD
  return p.split.tiles > 0 ? window_join_parts(p, kQTile, kPair, dtype, st) : LMK_OK;
}

}  // namespace lmk
