// Sliding-window attention with sinks in fp32, on the CUDA cores: 64 x 64 tiles of scores, 8 rows a warp, 8 x 2 results a thread.
//
//   S = scale Q K^T over the visible keys, P = e^{S - lse}, O = P V (running maximum and sum, one pass over the keys)
//   dV = P^T dO,  dP = dO V^T,  delta = rowsum(O dO),  dS = scale P (dP - delta),  dQ = dS K,  dK = dS^T Q
// Only the key tiles that a query tile sees are visited (window_params.h).  dK and dV of heads that share keys are summed in the
// unit that owns the keys; no atomics.  Rows behind a sequence's end are read as zeros, whatever they hold.
// A 16-byte read of 32 different places takes the shared memory 4 cycles, of one place 1.  A warp's eight rows are the same for all its lanes,
// which hold the columns: 64 multiply-adds a lane, issued as 32 pairs, cost 16 cycles of reads (with 4 x 4 results a thread 32, and
// the reads were the bound: B2 H16 Hkv8 L2048 D128, window 512, forward and backward 3040 -> 2195 us, 24 of 74 TFLOP/s).  The tiles lie as
// in memory, two of each on their way; P and dS go to the second product through a buffer of the warp's own.  The products are unrolled
// whole (by two: 2360 us), so that reads run ahead of their multiply-adds.  What is left is latency: two to four warps a scheduler, with
// two fifths of the cycles issuing.  (Sixteen warps of four rows 2650 us; tiles that need no mask told apart: no difference.)
#include "common.cuh"
#include "window_params.h"
#include "sm100_ptx.cuh"

namespace lmk {
namespace {

using namespace ptx;

constexpr int kTile = 64, kThreads = 256, kRows = 8;      // kRows: rows of a warp
constexpr float kLog2e = 1.4426950408889634f;
template <int kD> constexpr int kStride = kD + 4;          // of a row in shared memory: eight rows' 16 bytes meet in no bank
template <int kD> constexpr int kTileFloats = kTile * kStride<kD>;

// a 64-row tile on its way to shared memory; rows from `valid` on and features from D on become zeros
template <int kD>
__device__ __forceinline__ void copy_tile(float* to, const float* from, int64_t stride, int valid, int D) {
#pragma unroll
  for (int e = 0; e < kTile * kD / 4 / kThreads; ++e) {
    const int i = e * kThreads + threadIdx.x, r = i / (kD / 4), c = i % (kD / 4) * 4;
    const bool is = r < valid && c < D;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(to + r * kStride<kD> + c)), "l"(is ? from + r * stride + c : from),
                 "r"(is ? 16 : 0) : "memory");
  }
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group 0;" ::: "memory"); }

__device__ __forceinline__ void read4(uint64_t (&x)[2], const float* from) {      // two pairs
  const ulonglong2 t = *reinterpret_cast<const ulonglong2*>(from);
  x[0] = t.x;
  x[1] = t.y;
}
// d[r][j] = a's row r times b's row lane + 32 j; a: the warp's rows.  Multiply-adds in pairs: even and odd features.
template <int kD>
__device__ __forceinline__ void product(float (&d)[kRows][2], const float* a, const float* b, int lane) {
  uint64_t sum[kRows][2];
#pragma unroll
  for (int r = 0; r < kRows; ++r) sum[r][0] = sum[r][1] = 0ull;
#pragma unroll 16
  for (int c = 0; c < kD; c += 4) {
    uint64_t x[kRows][2], y[2][2];
    read4(y[0], b + lane * kStride<kD> + c);
    read4(y[1], b + (lane + 32) * kStride<kD> + c);
#pragma unroll
    for (int r = 0; r < kRows; ++r) read4(x[r], a + r * kStride<kD> + c);
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        sum[r][0] = fma2(x[r][e], y[0][e], sum[r][0]);
        sum[r][1] = fma2(x[r][e], y[1][e], sum[r][1]);
      }
  }
#pragma unroll
  for (int r = 0; r < kRows; ++r)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      float even, odd;
      upk2(sum[r][j], even, odd);
      d[r][j] = even + odd;
    }
}
// d[r][f] += sum over 64 n of w[n][2 r ..] b[n][lane kF + f], r a pair of rows; w [64][kRows]: the warp's weights
template <int kD>
__device__ __forceinline__ void accumulate(uint64_t (&d)[kRows / 2][kD / 32], const float* w, const float* b, int lane) {
  constexpr int kF = kD / 32;
#pragma unroll
  for (int n = 0; n < kTile; n += 2) {
    uint64_t x[2][kRows / 2];
    float y[2][kF];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const float* const from = b + (n + e) * kStride<kD> + lane * kF;
      if constexpr (kF == 2) {
        const float2 t = *reinterpret_cast<const float2*>(from);
        y[e][0] = t.x;
        y[e][1] = t.y;
      } else {
        const float4 t = *reinterpret_cast<const float4*>(from);
        y[e][0] = t.x;
        y[e][1] = t.y;
        y[e][2] = t.z;
        y[e][3] = t.w;
      }
      const ulonglong2 lo = *reinterpret_cast<const ulonglong2*>(w + (n + e) * kRows), hi = *reinterpret_cast<const ulonglong2*>(w + (n + e) * kRows + 4);
      x[e][0] = lo.x;
      x[e][1] = lo.y;
      x[e][2] = hi.x;
      x[e][3] = hi.y;
    }
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int f = 0; f < kF; ++f) {
        const uint64_t y2 = pk2(y[e][f], y[e][f]);
#pragma unroll
        for (int r = 0; r < kRows / 2; ++r) d[r][f] = fma2(x[e][r], y2, d[r][f]);
      }
  }
}
// the warp's weights take the places that the last product has read
__device__ __forceinline__ void share(float* w, const float (&x)[kRows][2], int lane) {
  __syncwarp();
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int r = 0; r < kRows; r += 4)
      *reinterpret_cast<float4*>(w + (lane + 32 * j) * kRows + r) = make_float4(x[r][j], x[r + 1][j], x[r + 2][j], x[r + 3][j]);
  __syncwarp();
}
// row r of a pair-wise sum
template <int kF> __device__ __forceinline__ void row_of(float (&x)[kF], const uint64_t (&d)[kRows / 2][kF], int r) {
#pragma unroll
  for (int f = 0; f < kF; ++f) {
    float a, b;
    upk2(d[r / 2][f], a, b);
    x[f] = r & 1 ? b : a;
  }
}
template <int kF> __device__ __forceinline__ void write_row(float* to, const float (&x)[kF], bool nonzero) {
  if constexpr (kF == 2) *reinterpret_cast<float2*>(to) = nonzero ? make_float2(x[0], x[1]) : make_float2(0.f, 0.f);
  else *reinterpret_cast<float4*>(to) = nonzero ? make_float4(x[0], x[1], x[2], x[3]) : make_float4(0.f, 0.f, 0.f, 0.f);
}
__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
  for (int w = 16; w > 0; w >>= 1) x += __shfl_xor_sync(0xffffffffu, x, w);
  return x;
}
__device__ __forceinline__ float warp_max_nan(float x) {      // NaN where a lane has one
  asm volatile("redux.sync.max.NaN.f32 %0, %0, 0xffffffff;" : "+f"(x));
  return x;
}
__device__ __forceinline__ int length_of(const WindowParams& p, int b) {
  return p.lengths == nullptr ? p.Lk : min(max(ld_behind_wait(p.lengths + b), 0), p.Lk);
}

template <int kD>
__global__ void __launch_bounds__(kThreads, kD == 64 ? 2 : 1) window_fwd_f32_kernel(const __grid_constant__ WindowParams p, float scale_log2) {
  constexpr int kF = kD / 32, kT = kTileFloats<kD>;
  extern __shared__ __align__(16) float smem[];
  float *const qt = smem, *const kv = qt + kT, *const wts = kv + 4 * kT + threadIdx.x / 32 * (kRows * kTile);      // kv: 2 x (K, V)
  grid_dep_wait();
  grid_dep_launch();
  const int lane = threadIdx.x % 32, r0 = threadIdx.x / 32 * kRows;
  const int tiles = gridDim.x, tile = tiles - 1 - (int)blockIdx.x, bh = blockIdx.y, b = bh / p.H, h = bh - b * p.H;
  const int hk = h / (p.H / p.Hkv), off = p.Lk - p.Lq, len = length_of(p, b);
  const int rows = min(kTile, p.Lq - tile * kTile), p0 = off + tile * kTile;
  const float* k = (const float*)p.k + b * p.ks[0] + hk * p.ks[1];
  const float* v = (const float*)p.v + b * p.vs[0] + hk * p.vs[1];
  const KeyTiles kts = keys_of_queries(tile, kTile, kTile, p.Lq, off, len, p.window, p.sinks);
  const int n = kts.sink_tiles + kts.last - kts.first + 1;
  auto key_of = [&](int i) { return (i < kts.sink_tiles ? i : kts.first + i - kts.sink_tiles) * kTile; };
  auto ask = [&](int i) {
    float* const to = kv + (i & 1) * 2 * kT;
    copy_tile<kD>(to, k + key_of(i) * p.ks[2], p.ks[2], len - key_of(i), p.D);
    copy_tile<kD>(to + kT, v + key_of(i) * p.vs[2], p.vs[2], len - key_of(i), p.D);
    copy_commit();
  };
  if (n > 0) {
    copy_tile<kD>(qt, (const float*)p.q + b * p.qs[0] + h * p.qs[1] + (int64_t)tile * kTile * p.qs[2], p.qs[2], min(rows, len - p0), p.D);
    ask(0);
  }
  float m[kRows], l[kRows];                    // l: the lane's share
  uint64_t o[kRows / 2][kF] = {};
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    m[r] = -INFINITY;
    l[r] = 0.f;
  }
  for (int i = 0; i < n; ++i) {
    const float* const kt = kv + (i & 1) * 2 * kT;
    const int key0 = key_of(i) + lane;
    copy_wait();
    __syncthreads();                           // tile i is there, and nobody reads tile i - 1 any more
    if (i + 1 < n) ask(i + 1);
    float s[kRows][2], turn[kRows];
    product<kD>(s, qt + r0 * kStride<kD>, kt, lane);
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const int pos = p0 + r0 + r;
#pragma unroll
      for (int j = 0; j < 2; ++j) s[r][j] = pos < len && window_sees(pos, key0 + 32 * j, p.window, p.sinks) ? s[r][j] * scale_log2 : -INFINITY;
      const float mx = warp_max_nan(max3_nan(m[r], s[r][0], s[r][1]));
      const float shift = mx == -INFINITY ? 0.f : mx;
      turn[r] = exp2f(m[r] - shift);
      m[r] = mx;
      s[r][0] = exp2f(s[r][0] - shift);
      s[r][1] = exp2f(s[r][1] - shift);
      l[r] = fmaf(l[r], turn[r], s[r][0] + s[r][1]);
    }
#pragma unroll
    for (int r = 0; r < kRows / 2; ++r)
#pragma unroll
      for (int f = 0; f < kF; ++f) o[r][f] = mul2(o[r][f], pk2(turn[2 * r], turn[2 * r + 1]));
    share(wts, s, lane);
    accumulate<kD>(o, wts, kt + kT, lane);
  }
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const float sum = warp_sum(l[r]);
    if (r0 + r >= rows) continue;
    const int64_t at = (int64_t)bh * p.Lq + tile * kTile + r0 + r;
    const bool is = p0 + r0 + r < len;           // sees its own key at least; the sum is 0 where every score is -inf: NaN, as by the formula
    const float inv = is ? 1.f / sum : 0.f;
    float x[kF];
    row_of<kF>(x, o, r);
#pragma unroll
    for (int f = 0; f < kF; ++f) x[f] *= inv;
    if (lane * kF < p.D) write_row<kF>((float*)p.o + at * p.D + lane * kF, x, is);
    if (lane == 0 && p.lse != nullptr) p.lse[at] = is ? m[r] + log2f(sum) : INFINITY;
  }
}

// dQ of a tile of 64 query rows, and delta for the dK/dV kernel
template <int kD>
__global__ void __launch_bounds__(kThreads, 1) window_dq_f32_kernel(const __grid_constant__ WindowParams p, float scale_log2) {
  constexpr int kF = kD / 32, kT = kTileFloats<kD>;
  extern __shared__ __align__(16) float smem[];
  float *const qt = smem, *const gt = qt + kT, *const kv = gt + kT, *const wts = kv + 4 * kT + threadIdx.x / 32 * (kRows * kTile);
  grid_dep_wait();
  grid_dep_launch();
  const int lane = threadIdx.x % 32, r0 = threadIdx.x / 32 * kRows;
  const int tiles = gridDim.x, tile = tiles - 1 - (int)blockIdx.x, bh = blockIdx.y, b = bh / p.H, h = bh - b * p.H;
  const int hk = h / (p.H / p.Hkv), off = p.Lk - p.Lq, len = length_of(p, b);
  const int rows = min(kTile, p.Lq - tile * kTile), p0 = off + tile * kTile, valid = min(rows, len - p0);
  const int64_t row0 = (int64_t)bh * p.Lq + tile * kTile;
  const float* k = (const float*)p.k + b * p.ks[0] + hk * p.ks[1];
  const float* v = (const float*)p.v + b * p.vs[0] + hk * p.vs[1];
  const KeyTiles kts = keys_of_queries(tile, kTile, kTile, p.Lq, off, len, p.window, p.sinks);
  const int n = kts.sink_tiles + kts.last - kts.first + 1;
  auto key_of = [&](int i) { return (i < kts.sink_tiles ? i : kts.first + i - kts.sink_tiles) * kTile; };
  auto ask = [&](int i) {
    float* const to = kv + (i & 1) * 2 * kT;
    copy_tile<kD>(to, k + key_of(i) * p.ks[2], p.ks[2], len - key_of(i), p.D);
    copy_tile<kD>(to + kT, v + key_of(i) * p.vs[2], p.vs[2], len - key_of(i), p.D);
    copy_commit();
  };
  if (n > 0) {
    copy_tile<kD>(qt, (const float*)p.q + b * p.qs[0] + h * p.qs[1] + (int64_t)tile * kTile * p.qs[2], p.qs[2], valid, p.D);
    copy_tile<kD>(gt, (const float*)p.dO + b * p.dos[0] + h * p.dos[1] + (int64_t)tile * kTile * p.dos[2], p.dos[2], valid, p.D);
    ask(0);
    copy_wait();
    __syncthreads();
  }
  float delta[kRows], lse[kRows];
  uint64_t dq[kRows / 2][kF] = {};
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const bool is = r0 + r < valid;
    float sum = 0.f;
    if (is && lane * kF < p.D) {
#pragma unroll
      for (int f = 0; f < kF; ++f)
        sum = fmaf(ld_behind_wait((const float*)p.o + (row0 + r0 + r) * p.D + lane * kF + f), gt[(r0 + r) * kStride<kD> + lane * kF + f], sum);
    }
    delta[r] = warp_sum(sum);
    lse[r] = is ? ld_behind_wait(p.lse + row0 + r0 + r) : INFINITY;
    if (r0 + r < rows && lane == 0) p.delta[row0 + r0 + r] = delta[r];
  }
  for (int i = 0; i < n; ++i) {
    const float* const kt = kv + (i & 1) * 2 * kT;
    const int key0 = key_of(i) + lane;
    copy_wait();
    __syncthreads();
    if (i + 1 < n) ask(i + 1);
    float s[kRows][2], dp[kRows][2];
    product<kD>(s, qt + r0 * kStride<kD>, kt, lane);
    product<kD>(dp, gt + r0 * kStride<kD>, kt + kT, lane);
#pragma unroll
    for (int r = 0; r < kRows; ++r)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float w = window_sees(p0 + r0 + r, key0 + 32 * j, p.window, p.sinks) ? exp2f(fmaf(s[r][j], scale_log2, -lse[r])) : 0.f;
        s[r][j] = w * (dp[r][j] - delta[r]) * p.scale;
      }
    share(wts, s, lane);
    accumulate<kD>(dq, wts, kt, lane);
  }
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    float x[kF];
    row_of<kF>(x, dq, r);
    if (r0 + r < rows && lane * kF < p.D) write_row<kF>((float*)p.dq + (row0 + r0 + r) * p.D + lane * kF, x, r0 + r < valid);
  }
}

// dK and dV of a tile of 64 keys of one key head from a run of query tiles of all heads that share it; a warp has eight keys
template <int kD>
__global__ void __launch_bounds__(kThreads, 1) window_dkv_f32_kernel(const __grid_constant__ WindowParams p, float scale_log2) {
  constexpr int kF = kD / 32, kT = kTileFloats<kD>;
  extern __shared__ __align__(16) float smem[];
  float *const kt = smem, *const vt = kt + kT, *const qg = vt + kT, *const wts = qg + 4 * kT + threadIdx.x / 32 * (kRows * kTile);
  grid_dep_wait();
  grid_dep_launch();
  const int lane = threadIdx.x % 32, r0 = threadIdx.x / 32 * kRows;
  const int key_tiles = (p.Lk + kTile - 1) / kTile, bk = blockIdx.y, b = bk / p.Hkv, hk = bk - b * p.Hkv, G = p.H / p.Hkv;
  const int off = p.Lk - p.Lq, len = length_of(p, b);
  const int extra = (int)blockIdx.x - key_tiles;                         // >= 0: a run of a split tile
  const int tile = extra < 0 ? (int)blockIdx.x : extra / p.split.runs, run = extra < 0 ? -1 : extra % p.split.runs;
  const QueryTiles qts = queries_of_keys(tile, kTile, kTile, p.Lq, off, len, p.window, p.sinks);
  const bool split = tile < p.split.tiles;
  int first = qts.first, last = split ? qts.last : qts.end;
  if (run >= 0) {
    first = qts.last + 1 + run * p.split.run;
    last = min(qts.end, first + p.split.run - 1);
    if (first > last) return;
  }
  const int key0 = tile * kTile + r0, valid_k = min(kTile, len - tile * kTile);
  uint64_t dk[kRows / 2][kF] = {}, dv[kRows / 2][kF] = {};
  const int per_head = last - first + 1, n = per_head > 0 ? per_head * G : 0;
  auto rows_of = [&](int t) { return min(min(kTile, p.Lq - t * kTile), len - off - t * kTile); };
  auto ask = [&](int i) {
    const int g = i / per_head, t = first + i - g * per_head, h = hk * G + g;
    float* const to = qg + (i & 1) * 2 * kT;
    copy_tile<kD>(to, (const float*)p.q + b * p.qs[0] + h * p.qs[1] + (int64_t)t * kTile * p.qs[2], p.qs[2], rows_of(t), p.D);
    copy_tile<kD>(to + kT, (const float*)p.dO + b * p.dos[0] + h * p.dos[1] + (int64_t)t * kTile * p.dos[2], p.dos[2], rows_of(t), p.D);
    copy_commit();
  };
  if (n > 0) {
    copy_tile<kD>(kt, (const float*)p.k + b * p.ks[0] + hk * p.ks[1] + (int64_t)tile * kTile * p.ks[2], p.ks[2], valid_k, p.D);
    copy_tile<kD>(vt, (const float*)p.v + b * p.vs[0] + hk * p.vs[1] + (int64_t)tile * kTile * p.vs[2], p.vs[2], valid_k, p.D);
    ask(0);
  }
  for (int i = 0; i < n; ++i) {
    const float* const qt = qg + (i & 1) * 2 * kT;
    const int g = i / per_head, t = first + i - g * per_head, valid_q = rows_of(t);
    const int64_t row0 = ((int64_t)b * p.H + hk * G + g) * p.Lq + t * kTile + lane;
    float lse[2], delta[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const bool is = lane + 32 * j < valid_q;
      lse[j] = is ? ld_behind_wait(p.lse + row0 + 32 * j) : INFINITY;
      delta[j] = is ? ld_behind_wait(p.delta + row0 + 32 * j) : 0.f;
    }
    copy_wait();
    __syncthreads();
    if (i + 1 < n) ask(i + 1);
    float s[kRows][2];                         // [key][query lane + 32 j]
    product<kD>(s, kt + r0 * kStride<kD>, qt, lane);
    const int pos = off + t * kTile + lane;
#pragma unroll
    for (int r = 0; r < kRows; ++r)
#pragma unroll
      for (int j = 0; j < 2; ++j)
        s[r][j] = window_sees(pos + 32 * j, key0 + r, p.window, p.sinks) ? exp2f(fmaf(s[r][j], scale_log2, -lse[j])) : 0.f;
    share(wts, s, lane);
    accumulate<kD>(dv, wts, qt + kT, lane);
    float dp[kRows][2];
    product<kD>(dp, vt + r0 * kStride<kD>, qt + kT, lane);
#pragma unroll
    for (int r = 0; r < kRows; ++r)
#pragma unroll
      for (int j = 0; j < 2; ++j) dp[r][j] = s[r][j] * (dp[r][j] - delta[j]) * p.scale;
    share(wts, dp, lane);
    accumulate<kD>(dk, wts, qt, lane);
  }
  if (lane * kF >= p.D) return;
  float* const part = split ? p.split.part + (((int64_t)bk * p.split.tiles + tile) * (1 + p.split.runs) + 1 + run) * 2 * kTile * p.D : nullptr;
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    if (key0 + r >= (run >= 0 ? p.sinks : p.Lk)) continue;               // a run's rows see the sinks alone
    const bool sink = split && key0 + r < p.sinks;
    const int64_t at = sink ? (int64_t)(r0 + r) * p.D : ((int64_t)bk * p.Lk + key0 + r) * p.D;
    float x[kF];
    row_of<kF>(x, dk, r);
    write_row<kF>((sink ? part : (float*)p.dk) + at + lane * kF, x, true);
    row_of<kF>(x, dv, r);
    write_row<kF>((sink ? part + kTile * p.D : (float*)p.dv) + at + lane * kF, x, true);
  }
}

template <int kD> constexpr size_t kSmemFwd = sizeof(float) * (5 * kTileFloats<kD> + kTile * kTile);
template <int kD> constexpr size_t kSmemBwd = sizeof(float) * (6 * kTileFloats<kD> + kTile * kTile);
static_assert(kSmemBwd<128> <= 232448, "shared memory of one SM");

template <typename F> int allow(F* kernel, size_t smem) {
  LMK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  return LMK_OK;
}
template <int kD> int fwd(const WindowParams& p, cudaStream_t st) {
  int rc = allow(window_fwd_f32_kernel<kD>, kSmemFwd<kD>);
  if (rc != LMK_OK) return rc;
  const dim3 grid((p.Lq + kTile - 1) / kTile, p.B * p.H);
  LMK_CUDA(launch_overlapped(window_fwd_f32_kernel<kD>, grid, dim3(kThreads), kSmemFwd<kD>, st, p, p.scale * kLog2e));
  return LMK_OK;
}
template <int kD> int bwd(const WindowParams& p, cudaStream_t st) {
  int rc = allow(window_dq_f32_kernel<kD>, kSmemBwd<kD>);
  if (rc == LMK_OK) rc = allow(window_dkv_f32_kernel<kD>, kSmemBwd<kD>);
  if (rc != LMK_OK) return rc;
  const dim3 grid_q((p.Lq + kTile - 1) / kTile, p.B * p.H);
  const dim3 grid_k((p.Lk + kTile - 1) / kTile + p.split.tiles * p.split.runs, p.B * p.Hkv);
  LMK_CUDA(launch_overlapped(window_dq_f32_kernel<kD>, grid_q, dim3(kThreads), kSmemBwd<kD>, st, p, p.scale * kLog2e));
  LMK_CUDA(launch_overlapped(window_dkv_f32_kernel<kD>, grid_k, dim3(kThreads), kSmemBwd<kD>, st, p, p.scale * kLog2e));
  return p.split.tiles > 0 ? window_join_parts(p, kTile, kTile, LMK_F32, st) : LMK_OK;
}

}  // namespace

int window_f32_fwd(const WindowParams& p, cudaStream_t st) { return p.D <= 64 ? fwd<64>(p, st) : fwd<128>(p, st); }
int window_f32_bwd(const WindowParams& p, cudaStream_t st) { return p.D <= 64 ? bwd<64>(p, st) : bwd<128>(p, st); }

}  // namespace lmk
