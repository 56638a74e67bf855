// Sliding-window attention with sinks in fp32, on the CUDA cores: 64 x 64 tiles of scores, 4 x 4 results a thread.
//
//   S = scale Q K^T over the visible keys, P = e^{S - lse}, O = P V (running maximum and sum, one pass over the keys)
//   dV = P^T dO,  dP = dO V^T,  delta = rowsum(O dO),  dS = scale P (dP - delta),  dQ = dS K,  dK = dS^T Q
// Only the key tiles that a query tile sees are visited (window_params.h).  dK and dV of heads that share keys are summed in the
// unit that owns the keys; no atomics.  Rows behind a sequence's end are read as zeros, whatever they hold.
// Operands of the products lie in shared memory with the contracted index outermost, so that a thread reads its four rows and its four
// columns as one 16-byte vector each: two reads for 16 multiply-adds, which keeps the FMA units the bound and not the shared memory.
#include "common.cuh"
#include "window_params.h"
#include "sm100_ptx.cuh"

namespace lmk {
namespace {

using namespace ptx;

constexpr int kTile = 64, kPad = 68, kThreads = 256;
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float4 load4(const float* p) { return *reinterpret_cast<const float4*>(p); }

// A 64-row tile on its way to shared memory: asked for while the tile in front is worked on, stored as [kD][kPad].  A warp takes 32 rows of
// one 16-byte chunk: the stores of a feature lie next to each other (along the features they met in two banks).
template <int kD> struct Tile {
  float4 x[kTile * kD / 4 / kThreads];
  __device__ __forceinline__ void ask(const float* from, int64_t stride, int valid, int D) {
#pragma unroll
    for (int e = 0; e < kTile * kD / 4 / kThreads; ++e) {
      const int i = e * kThreads + threadIdx.x, r = i % kTile, c = i / kTile * 4;
      x[e] = r < valid && c < D ? load4(from + r * stride + c) : make_float4(0.f, 0.f, 0.f, 0.f);      // (rows behind the end: zeros)
    }
  }
  __device__ __forceinline__ void store(float* to) const {
#pragma unroll
    for (int e = 0; e < kTile * kD / 4 / kThreads; ++e) {
      const int i = e * kThreads + threadIdx.x, r = i % kTile, c = i / kTile * 4;
      to[c * kPad + r] = x[e].x;
      to[(c + 1) * kPad + r] = x[e].y;
      to[(c + 2) * kPad + r] = x[e].z;
      to[(c + 3) * kPad + r] = x[e].w;
    }
  }
};
// d[4][4] = sum over n of a[n][row ..] b[n][col ..]
template <int kN>
__device__ __forceinline__ void product(float (&d)[4][4], const float* a, const float* b, int ty, int tx) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) d[i][j] = 0.f;
#pragma unroll 8
  for (int n = 0; n < kN; ++n) {
    const float4 x = *reinterpret_cast<const float4*>(a + n * kPad + ty * 4);
    const float4 y = *reinterpret_cast<const float4*>(b + n * kPad + tx * 4);
    const float xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) d[i][j] = fmaf(xs[i], ys[j], d[i][j]);
  }
}
// d[4][kD / 16] += sum over 64 n of a[n][row ..] b[feature tx + 16 c][n], four n at a time
template <int kD>
__device__ __forceinline__ void accumulate(float (&d)[4][kD / 16], const float* a, const float* b, int ty, int tx) {
#pragma unroll 2
  for (int n = 0; n < kTile; n += 4) {
    float4 x[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = *reinterpret_cast<const float4*>(a + (n + e) * kPad + ty * 4);
#pragma unroll
    for (int c = 0; c < kD / 16; ++c) {
      const float4 y = *reinterpret_cast<const float4*>(b + (c * 16 + tx) * kPad + n);
      const float ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        d[0][c] = fmaf(x[e].x, ys[e], d[0][c]);
        d[1][c] = fmaf(x[e].y, ys[e], d[1][c]);
        d[2][c] = fmaf(x[e].z, ys[e], d[2][c]);
        d[3][c] = fmaf(x[e].w, ys[e], d[3][c]);
      }
    }
  }
}
__device__ __forceinline__ int length_of(const WindowParams& p, int b) {
  return p.lengths == nullptr ? p.Lk : min(max(ld_behind_wait(p.lengths + b), 0), p.Lk);
}

template <int kD>
__global__ void __launch_bounds__(kThreads) window_fwd_f32_kernel(const __grid_constant__ WindowParams p, float scale_log2) {
  extern __shared__ float smem[];
  float *qt = smem, *kt = qt + kD * kPad, *vt = kt + kD * kPad, *pt = vt + kD * kPad;      // pt [key][row]
  grid_dep_wait();
  grid_dep_launch();
  const int tid = threadIdx.x, ty = tid / 16, tx = tid % 16;
  const int tiles = gridDim.x, tile = tiles - 1 - (int)blockIdx.x, bh = blockIdx.y, b = bh / p.H, h = bh - b * p.H;
  const int hk = h / (p.H / p.Hkv), off = p.Lk - p.Lq, len = length_of(p, b);
  const int rows = min(kTile, p.Lq - tile * kTile), p0 = off + tile * kTile;
  const float* q = (const float*)p.q + b * p.qs[0] + h * p.qs[1] + (int64_t)tile * kTile * p.qs[2];
  const float* k = (const float*)p.k + b * p.ks[0] + hk * p.ks[1];
  const float* v = (const float*)p.v + b * p.vs[0] + hk * p.vs[1];
  Tile<kD> tk, tv;
  tk.ask(q, p.qs[2], min(rows, len - p0), p.D);
  tk.store(qt);
  float m[4], l[4], o[4][kD / 16];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.f;
#pragma unroll
    for (int c = 0; c < kD / 16; ++c) o[i][c] = 0.f;
  }
  const KeyTiles kts = keys_of_queries(tile, kTile, kTile, p.Lq, off, len, p.window, p.sinks);
  const int n = kts.sink_tiles + kts.last - kts.first + 1;
  auto key_of = [&](int i) { return (i < kts.sink_tiles ? i : kts.first + i - kts.sink_tiles) * kTile; };
  auto ask = [&](int i) {
    tk.ask(k + key_of(i) * p.ks[2], p.ks[2], len - key_of(i), p.D);
    tv.ask(v + key_of(i) * p.vs[2], p.vs[2], len - key_of(i), p.D);
  };
  if (n > 0) ask(0);
  for (int i = 0; i < n; ++i) {
    const int key0 = key_of(i);
    __syncthreads();
    tk.store(kt);
    tv.store(vt);
    __syncthreads();
    if (i + 1 < n) ask(i + 1);
    float s[4][4];
    product<kD>(s, qt, kt, ty, tx);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int pos = p0 + ty * 4 + r;
      float mx = m[r];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[r][j] = pos < len && window_sees(pos, key0 + tx * 4 + j, p.window, p.sinks) ? s[r][j] * scale_log2 : -INFINITY;
        mx = max3_nan(mx, s[r][j], s[r][j]);
      }
#pragma unroll
      for (int w = 8; w > 0; w >>= 1) {
        const float y = __shfl_xor_sync(0xffffffffu, mx, w);
        mx = max3_nan(mx, y, y);
      }
      const float shift = mx == -INFINITY ? 0.f : mx, f = exp2f(m[r] - shift);
      m[r] = mx;
      l[r] *= f;
#pragma unroll
      for (int c = 0; c < kD / 16; ++c) o[r][c] *= f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[r][j] = exp2f(s[r][j] - shift);
        l[r] += s[r][j];
        pt[(tx * 4 + j) * kPad + ty * 4 + r] = s[r][j];
      }
    }
    __syncthreads();
    accumulate<kD>(o, pt, vt, ty, tx);
  }
#pragma unroll
  for (int r = 0; r < 4; ++r) {
#pragma unroll
    for (int w = 8; w > 0; w >>= 1) l[r] += __shfl_xor_sync(0xffffffffu, l[r], w);
    const int row = ty * 4 + r;
    if (row >= rows) continue;
    const int64_t at = (int64_t)bh * p.Lq + tile * kTile + row;
    const float inv = l[r] == 0.f ? 0.f : 1.f / l[r];
#pragma unroll
    for (int c = 0; c < kD / 16; ++c)
      if (c * 16 + tx < p.D) ((float*)p.o)[at * p.D + c * 16 + tx] = o[r][c] * inv;
    if (tx == 0) p.lse[at] = l[r] == 0.f ? INFINITY : m[r] + log2f(l[r]);
  }
}

// dQ of a tile of 64 query rows, and delta for the dK/dV kernel
template <int kD>
__global__ void __launch_bounds__(kThreads) window_dq_f32_kernel(const __grid_constant__ WindowParams p, float scale_log2) {
  extern __shared__ float smem[];
  float *qt = smem, *gt = qt + kD * kPad, *kt = gt + kD * kPad, *vt = kt + kD * kPad, *dst = vt + kD * kPad;      // dst [key][row]
  grid_dep_wait();
  grid_dep_launch();
  const int tid = threadIdx.x, ty = tid / 16, tx = tid % 16;
  const int tiles = gridDim.x, tile = tiles - 1 - (int)blockIdx.x, bh = blockIdx.y, b = bh / p.H, h = bh - b * p.H;
  const int hk = h / (p.H / p.Hkv), off = p.Lk - p.Lq, len = length_of(p, b);
  const int rows = min(kTile, p.Lq - tile * kTile), p0 = off + tile * kTile, valid = min(rows, len - p0);
  const int64_t row0 = (int64_t)bh * p.Lq + tile * kTile;
  const float* k = (const float*)p.k + b * p.ks[0] + hk * p.ks[1];
  const float* v = (const float*)p.v + b * p.vs[0] + hk * p.vs[1];
  Tile<kD> tk, tv;
  tk.ask((const float*)p.q + b * p.qs[0] + h * p.qs[1] + (int64_t)tile * kTile * p.qs[2], p.qs[2], valid, p.D);
  tv.ask((const float*)p.dO + b * p.dos[0] + h * p.dos[1] + (int64_t)tile * kTile * p.dos[2], p.dos[2], valid, p.D);
  tk.store(qt);
  tv.store(gt);
  __syncthreads();
  float delta[4], lse[4], dq[4][kD / 16];
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int row = ty * 4 + r;
    float sum = 0.f;
    if (row < valid)
      for (int c = tx; c < p.D; c += 16) sum = fmaf(((const float*)p.o)[(row0 + row) * p.D + c], gt[c * kPad + row], sum);
#pragma unroll
    for (int w = 8; w > 0; w >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
    delta[r] = sum;
    lse[r] = row < valid ? ld_behind_wait(p.lse + row0 + row) : INFINITY;
    if (row < rows && tx == 0) p.delta[row0 + row] = sum;
#pragma unroll
    for (int c = 0; c < kD / 16; ++c) dq[r][c] = 0.f;
  }
  const KeyTiles kts = keys_of_queries(tile, kTile, kTile, p.Lq, off, len, p.window, p.sinks);
  const int n = kts.sink_tiles + kts.last - kts.first + 1;
  auto key_of = [&](int i) { return (i < kts.sink_tiles ? i : kts.first + i - kts.sink_tiles) * kTile; };
  auto ask = [&](int i) {
    tk.ask(k + key_of(i) * p.ks[2], p.ks[2], len - key_of(i), p.D);
    tv.ask(v + key_of(i) * p.vs[2], p.vs[2], len - key_of(i), p.D);
  };
  if (n > 0) ask(0);
  for (int i = 0; i < n; ++i) {
    const int key0 = key_of(i);
    __syncthreads();
    tk.store(kt);
    tv.store(vt);
    __syncthreads();
    if (i + 1 < n) ask(i + 1);
    float s[4][4], dp[4][4];
    product<kD>(s, qt, kt, ty, tx);
    product<kD>(dp, gt, vt, ty, tx);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int pos = p0 + ty * 4 + r;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const bool seen = window_sees(pos, key0 + tx * 4 + j, p.window, p.sinks);
        const float w = seen ? exp2f(fmaf(s[r][j], scale_log2, -lse[r])) : 0.f;
        dst[(tx * 4 + j) * kPad + ty * 4 + r] = w * (dp[r][j] - delta[r]) * p.scale;
      }
    }
    __syncthreads();
    accumulate<kD>(dq, dst, kt, ty, tx);
  }
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int row = ty * 4 + r;
    if (row >= rows) continue;
#pragma unroll
    for (int c = 0; c < kD / 16; ++c)
      if (c * 16 + tx < p.D) ((float*)p.dq)[(row0 + row) * p.D + c * 16 + tx] = row < valid ? dq[r][c] : 0.f;
  }
}

// dK and dV of a tile of 64 keys of one key head from a run of query tiles of all heads that share it
template <int kD>
__global__ void __launch_bounds__(kThreads) window_dkv_f32_kernel(const __grid_constant__ WindowParams p, float scale_log2) {
  extern __shared__ float smem[];
  float *kt = smem, *vt = kt + kD * kPad, *qt = vt + kD * kPad, *gt = qt + kD * kPad;
  float *pr = gt + kD * kPad, *dsr = pr + kTile * kPad;                  // [query][key]
  grid_dep_wait();
  grid_dep_launch();
  const int tid = threadIdx.x, ty = tid / 16, tx = tid % 16;
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
  const int key0 = tile * kTile, valid_k = min(kTile, len - key0);
  Tile<kD> tq, tg;
  tq.ask((const float*)p.k + b * p.ks[0] + hk * p.ks[1] + key0 * p.ks[2], p.ks[2], valid_k, p.D);
  tg.ask((const float*)p.v + b * p.vs[0] + hk * p.vs[1] + key0 * p.vs[2], p.vs[2], valid_k, p.D);
  tq.store(kt);
  tg.store(vt);
  float dk[4][kD / 16], dv[4][kD / 16];                                  // keys 4 ty .., features tx + 16 c
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int c = 0; c < kD / 16; ++c) dk[r][c] = dv[r][c] = 0.f;
  const int per_head = last - first + 1, n = per_head > 0 ? per_head * G : 0;
  auto rows_of = [&](int t) { return min(min(kTile, p.Lq - t * kTile), len - off - t * kTile); };
  auto ask = [&](int i) {
    const int g = i / per_head, t = first + i - g * per_head, h = hk * G + g;
    tq.ask((const float*)p.q + b * p.qs[0] + h * p.qs[1] + (int64_t)t * kTile * p.qs[2], p.qs[2], rows_of(t), p.D);
    tg.ask((const float*)p.dO + b * p.dos[0] + h * p.dos[1] + (int64_t)t * kTile * p.dos[2], p.dos[2], rows_of(t), p.D);
  };
  if (n > 0) ask(0);
  for (int i = 0; i < n; ++i) {
    const int g = i / per_head, t = first + i - g * per_head, valid_q = rows_of(t);
    const int64_t row0 = ((int64_t)b * p.H + hk * G + g) * p.Lq + t * kTile;
    __syncthreads();
    tq.store(qt);
    tg.store(gt);
    __syncthreads();
    if (i + 1 < n) ask(i + 1);
    float s[4][4], dp[4][4];
    product<kD>(s, qt, kt, ty, tx);
    product<kD>(dp, gt, vt, ty, tx);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int row = ty * 4 + r, pos = off + t * kTile + row;
      const float lse = row < valid_q ? ld_behind_wait(p.lse + row0 + row) : INFINITY;
      const float delta = row < valid_q ? ld_behind_wait(p.delta + row0 + row) : 0.f;
      float w[4], d[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        w[j] = window_sees(pos, key0 + tx * 4 + j, p.window, p.sinks) ? exp2f(fmaf(s[r][j], scale_log2, -lse)) : 0.f;
        d[j] = w[j] * (dp[r][j] - delta) * p.scale;
      }
      *reinterpret_cast<float4*>(pr + row * kPad + tx * 4) = make_float4(w[0], w[1], w[2], w[3]);
      *reinterpret_cast<float4*>(dsr + row * kPad + tx * 4) = make_float4(d[0], d[1], d[2], d[3]);
    }
    __syncthreads();
    accumulate<kD>(dv, pr, gt, ty, tx);
    accumulate<kD>(dk, dsr, qt, ty, tx);
  }
  float* const part = split ? p.split.part + (((int64_t)bk * p.split.tiles + tile) * (1 + p.split.runs) + 1 + run) * 2 * kTile * p.D : nullptr;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int key = ty * 4 + r;
    if (key0 + key >= (run >= 0 ? p.sinks : p.Lk)) continue;      // a run's rows see the sinks alone
    const int64_t at = ((int64_t)bk * p.Lk + key0 + key) * p.D;
#pragma unroll
    for (int c = 0; c < kD / 16; ++c) {
      const int f = c * 16 + tx;
      if (f >= p.D) continue;
      if (split) {
        part[key * p.D + f] = dk[r][c];
        part[(kTile + key) * p.D + f] = dv[r][c];
      } else {
        ((float*)p.dk)[at + f] = dk[r][c];
        ((float*)p.dv)[at + f] = dv[r][c];
      }
    }
  }
}

template <int kD> constexpr size_t kSmemFwd = sizeof(float) * (3 * kD * kPad + kTile * kPad);
template <int kD> constexpr size_t kSmemDq = sizeof(float) * (4 * kD * kPad + kTile * kPad);
template <int kD> constexpr size_t kSmemDkv = sizeof(float) * (4 * kD * kPad + 2 * kTile * kPad);

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
  int rc = allow(window_dq_f32_kernel<kD>, kSmemDq<kD>);
  if (rc == LMK_OK) rc = allow(window_dkv_f32_kernel<kD>, kSmemDkv<kD>);
  if (rc != LMK_OK) return rc;
  const dim3 grid_q((p.Lq + kTile - 1) / kTile, p.B * p.H);
  const dim3 grid_k((p.Lk + kTile - 1) / kTile + p.split.tiles * p.split.runs, p.B * p.Hkv);
  LMK_CUDA(launch_overlapped(window_dq_f32_kernel<kD>, grid_q, dim3(kThreads), kSmemDq<kD>, st, p, p.scale * kLog2e));
  LMK_CUDA(launch_overlapped(window_dkv_f32_kernel<kD>, grid_k, dim3(kThreads), kSmemDkv<kD>, st, p, p.scale * kLog2e));
  return p.split.tiles > 0 ? window_join_parts(p, kTile, kTile, LMK_F32, st) : LMK_OK;
}

}  // namespace

int window_f32_fwd(const WindowParams& p, cudaStream_t st) { return p.D <= 64 ? fwd<64>(p, st) : fwd<128>(p, st); }
int window_f32_bwd(const WindowParams& p, cudaStream_t st) { return p.D <= 64 ? bwd<64>(p, st) : bwd<128>(p, st); }

}  // namespace lmk
