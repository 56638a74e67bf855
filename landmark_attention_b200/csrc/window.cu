// extern "C" entry points of sliding-window attention: argument checks, the division of the sinks' gradient, the choice of kernels.
#include "common.cuh"
#include "window_params.h"
#include "sm100_ptx.cuh"

namespace lmk {
namespace {

constexpr size_t kNextBytes = 256;
constexpr size_t up256(size_t x) { return (x + 255) / 256 * 256; }

int check_window(const void* q, const void* k, const void* v, int B, int H, int Hkv, int Lq, int Lk, int D,
                 const int64_t* qs, const int64_t* ks, const int64_t* vs, int window, int sinks, float scale, int dtype) {
  LMK_CHECK_ARG(q && k && v, "window attention: q, k or v is null");
  LMK_CHECK_ARG(qs && ks && vs, "window attention: stride arrays are required");
  LMK_CHECK_ARG(B >= 1 && H >= 1 && Hkv >= 1 && Lq >= 1 && Lk >= 1, "window attention: empty problem (B=%d H=%d Hkv=%d Lq=%d Lk=%d)", B, H, Hkv, Lq, Lk);
  LMK_CHECK_ARG(H % Hkv == 0, "window attention: %d query heads are not a multiple of %d key heads", H, Hkv);
  LMK_CHECK_ARG((int64_t)B * H <= 65535, "window attention: B*H = %lld exceeds 65535", (long long)B * H);
  LMK_CHECK_ARG(Lk >= Lq, "window attention: %d queries are more than %d keys", Lq, Lk);
  LMK_CHECK_ARG(Lk <= (1 << 22), "window attention: %d keys exceed 2^22", Lk);
  LMK_CHECK_ARG((int64_t)B * H * ((Lk + 63) / 64) <= INT32_MAX / 4, "window attention: %d heads of %d keys are too many", B * H, Lk);
  LMK_CHECK_ARG(D >= 8 && D <= 128 && D % 8 == 0, "window attention: head dim %d must be a multiple of 8 up to 128", D);
  LMK_CHECK_ARG(dtype == LMK_F32 || dtype == LMK_F16 || dtype == LMK_BF16, "window attention: bad dtype %d", dtype);
  LMK_CHECK_ARG(window >= 1, "window attention: window %d must be at least 1", window);
  LMK_CHECK_ARG(sinks >= 0, "window attention: sinks %d must not be negative", sinks);
  LMK_CHECK_ARG(scale > 0.f && isfinite(scale), "window attention: scale must be positive and finite");
  return LMK_OK;
}

void fill(WindowParams& p, const void* q, const void* k, const void* v, const int32_t* lengths, int B, int H, int Hkv, int Lq, int Lk, int D,
          const int64_t* qs, const int64_t* ks, const int64_t* vs, int window, int sinks, float scale) {
  p.q = q; p.k = k; p.v = v; p.lengths = lengths;
  p.B = B; p.H = H; p.Hkv = Hkv; p.Lq = Lq; p.Lk = Lk; p.D = D; p.scale = scale;
  p.window = window < Lk ? window : Lk;
  p.sinks = sinks < Lk ? sinks : Lk;
  for (int i = 0; i < 3; ++i) { p.qs[i] = qs[i]; p.ks[i] = ks[i]; p.vs[i] = vs[i]; }
}
// fp32 rows are read as 16-byte vectors, 16-bit tensors by TMA
bool rows_ok(const void* p, const int64_t* st, int D, int dtype) {
  if (dtype != LMK_F32) return window_sm100_operand_ok(p, st, D);
  return ((uintptr_t)p & 15) == 0 && st[0] % 4 == 0 && st[1] % 4 == 0 && st[2] % 4 == 0;
}

// How the query tiles of the sinks' key tiles are dealt out (SinkSplit): runs as long as the window's share of an ordinary key tile, or
// longer where the units are enough to fill the device anyway.
int plan_split(SinkSplit* s, int B, int Hkv, int Lq, int Lk, int window, int sinks, int qt, int kk) {
  *s = SinkSplit{};
  if (sinks == 0 || Lk - 1 <= kk + window - 2) return LMK_OK;      // every query sees the first tile through the window
  int n_sm = 0, rc;
  if ((rc = sm_count(&n_sm)) != LMK_OK) return rc;
  const int q_tiles = (Lq + qt - 1) / qt;
  s->tiles = (sinks + kk - 1) / kk;
  const int share = (window + kk) / qt + 1, run = share < 4 ? 4 : share;
  int runs = (q_tiles + run - 1) / run;
  const int64_t enough = (2 * (int64_t)n_sm + (int64_t)B * Hkv * s->tiles - 1) / ((int64_t)B * Hkv * s->tiles);
  if (runs > enough) runs = (int)enough;
  s->run = (q_tiles + runs - 1) / runs;
  s->runs = (q_tiles + s->run - 1) / s->run;
  return LMK_OK;
}
size_t part_bytes(const SinkSplit& s, int B, int Hkv, int D, int kk) {
  return sizeof(float) * (size_t)B * Hkv * s.tiles * (1 + s.runs) * 2 * kk * D;
}
void tile_sizes(int dtype, int* qt, int* kk) { *qt = *kk = dtype == LMK_F32 ? 64 : 128; }      // of the dK/dV kernels

// The parts of the sinks, added up in the order of their runs.
template <typename T>
__global__ void __launch_bounds__(256) window_join_kernel(const __grid_constant__ WindowParams p, int qt, int kk) {
  ptx::grid_dep_wait();
  ptx::grid_dep_launch();
  const int tile = blockIdx.x % p.split.tiles, bk = blockIdx.x / p.split.tiles, b = bk / p.Hkv;
  const int len = p.lengths == nullptr ? p.Lk : min(max(ptx::ld_behind_wait(p.lengths + b), 0), p.Lk);
  const QueryTiles qts = queries_of_keys(tile, qt, kk, p.Lq, p.Lk - p.Lq, len, p.window, p.sinks);
  const int runs = (qts.end - qts.last + p.split.run - 1) / p.split.run;
  const int e = (blockIdx.y * 256 + threadIdx.x) * 4, key = e / p.D, f = e - key * p.D;
  if (key >= kk || tile * kk + key >= p.sinks) return;
  const int64_t slot = 2ll * kk * p.D;
  const float* part = p.split.part + ((int64_t)bk * p.split.tiles + tile) * (1 + p.split.runs) * slot + e;
  const int64_t at = ((int64_t)bk * p.Lk + tile * kk + key) * p.D + f;
#pragma unroll
  for (int g = 0; g < 2; ++g) {                     // dK, dV
    float4 sum = *reinterpret_cast<const float4*>(part + g * (slot / 2));
    for (int r = 1; r <= runs; ++r) {
      const float4 x = *reinterpret_cast<const float4*>(part + r * slot + g * (slot / 2));
      sum = make_float4(sum.x + x.x, sum.y + x.y, sum.z + x.z, sum.w + x.w);
    }
    T* const to = (T*)(g == 0 ? p.dk : p.dv) + at;
    to[0] = from_f32<T>(sum.x);
    to[1] = from_f32<T>(sum.y);
    to[2] = from_f32<T>(sum.z);
    to[3] = from_f32<T>(sum.w);
  }
}

}  // namespace

int window_join_parts(const WindowParams& p, int qt, int kk, int dtype, cudaStream_t st) {
  // the tiles in x: there may be more of them than y has room for
  const dim3 grid((unsigned)(p.B * p.Hkv * p.split.tiles), ((p.sinks < kk ? p.sinks : kk) * p.D / 4 + 255) / 256);
  if (dtype == LMK_F32) LMK_CUDA(launch_overlapped(window_join_kernel<float>, grid, dim3(256), 0, st, p, qt, kk));
  else if (dtype == LMK_F16) LMK_CUDA(launch_overlapped(window_join_kernel<__half>, grid, dim3(256), 0, st, p, qt, kk));
  else LMK_CUDA(launch_overlapped(window_join_kernel<__nv_bfloat16>, grid, dim3(256), 0, st, p, qt, kk));
  return LMK_OK;
}

}  // namespace lmk

using namespace lmk;

extern "C" int lmk_window_fwd(const void* q, const void* k, const void* v, void* o, void* o_rest, float* lse, const int32_t* lengths, int B,
                              int H, int Hkv, int Lq, int Lk, int D, const int64_t q_strides[3], const int64_t k_strides[3],
                              const int64_t v_strides[3], int window, int sinks, float sm_scale, int dtype, void* stream) {
  int rc = check_window(q, k, v, B, H, Hkv, Lq, Lk, D, q_strides, k_strides, v_strides, window, sinks, sm_scale, dtype);
  if (rc != LMK_OK) return rc;
  LMK_CHECK_ARG(o != nullptr, "window attention: o is null");
  LMK_CHECK_ARG(o_rest == nullptr || (dtype != LMK_F32 && lse != nullptr), "window attention: o_rest is for 16-bit types, beside lse");
  LMK_CHECK_ARG((((uintptr_t)o | (uintptr_t)o_rest) & 15) == 0, "window attention: o and o_rest must start on 16-byte boundaries");
  WindowParams p = {};
  fill(p, q, k, v, lengths, B, H, Hkv, Lq, Lk, D, q_strides, k_strides, v_strides, window, sinks, sm_scale);
  p.o = o;
  p.rest = o_rest;
  p.lse = lse;
  LMK_CHECK_ARG(rows_ok(q, q_strides, D, dtype) && rows_ok(k, k_strides, D, dtype) && rows_ok(v, v_strides, D, dtype),
                "window attention: tensors must start on 16-byte boundaries, strides be multiples of 16 bytes (16-bit types: positive, rows not overlapping)");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == LMK_F32 ? window_f32_fwd(p, st) : window_sm100_fwd(p, dtype, st);
}

extern "C" size_t lmk_window_bwd_workspace(int B, int H, int Hkv, int Lq, int Lk, int D, int window, int sinks, int dtype) {
  if (B < 1 || H < 1 || Hkv < 1 || Lq < 1 || Lk < Lq || D < 1 || window < 1 || sinks < 0) return 0;
  SinkSplit s;
  int qt, kk;
  tile_sizes(dtype, &qt, &kk);
  if (plan_split(&s, B, Hkv, Lq, Lk, window < Lk ? window : Lk, sinks < Lk ? sinks : Lk, qt, kk) != LMK_OK) return 0;
  return kNextBytes + up256(sizeof(float) * (size_t)B * H * Lq) + up256(part_bytes(s, B, Hkv, D, kk));
}

extern "C" int lmk_window_bwd(const void* q, const void* k, const void* v, const void* o, const void* o_rest, const void* dO, const float* lse,
                              const int32_t* lengths, void* dQ, void* dK, void* dV, void* workspace, size_t workspace_bytes, int B, int H,
                              int Hkv, int Lq, int Lk, int D, const int64_t q_strides[3], const int64_t k_strides[3],
                              const int64_t v_strides[3], const int64_t do_strides[3], int window, int sinks, float sm_scale, int dtype,
                              void* stream) {
  int rc = check_window(q, k, v, B, H, Hkv, Lq, Lk, D, q_strides, k_strides, v_strides, window, sinks, sm_scale, dtype);
  if (rc != LMK_OK) return rc;
  LMK_CHECK_ARG(o && lse && dO && dQ && dK && dV && do_strides, "window attention backward: o, lse, dO or a gradient is null");
  LMK_CHECK_ARG((o_rest != nullptr) == (dtype != LMK_F32), "window attention backward: 16-bit types need o_rest, fp32 has none");
  LMK_CHECK_ARG((((uintptr_t)o | (uintptr_t)o_rest | (uintptr_t)dQ | (uintptr_t)dK | (uintptr_t)dV) & 15) == 0,
                "window attention backward: o, o_rest and the gradients must start on 16-byte boundaries");
  WindowParams p = {};
  fill(p, q, k, v, lengths, B, H, Hkv, Lq, Lk, D, q_strides, k_strides, v_strides, window, sinks, sm_scale);
  p.o = const_cast<void*>(o);
  p.rest = const_cast<void*>(o_rest);
  p.dO = dO;
  p.lse = const_cast<float*>(lse);
  p.dq = dQ; p.dk = dK; p.dv = dV;
  for (int i = 0; i < 3; ++i) p.dos[i] = do_strides[i];
  LMK_CHECK_ARG(rows_ok(q, q_strides, D, dtype) && rows_ok(k, k_strides, D, dtype) && rows_ok(v, v_strides, D, dtype) && rows_ok(dO, do_strides, D, dtype),
                "window attention: tensors must start on 16-byte boundaries, strides be multiples of 16 bytes (16-bit types: positive, rows not overlapping)");
  int qt, kk;
  tile_sizes(dtype, &qt, &kk);
  if ((rc = plan_split(&p.split, B, Hkv, Lq, Lk, p.window, p.sinks, qt, kk)) != LMK_OK) return rc;
  const size_t delta_bytes = up256(sizeof(float) * (size_t)B * H * Lq), need = kNextBytes + delta_bytes + up256(part_bytes(p.split, B, Hkv, D, kk));
  if (workspace == nullptr || workspace_bytes < need || ((uintptr_t)workspace & 255) != 0)
    return fail(LMK_ERR_WORKSPACE, "window attention backward: workspace of %zu bytes on a 256-byte boundary needed", need);
  p.next = static_cast<int*>(workspace);
  p.delta = reinterpret_cast<float*>(static_cast<char*>(workspace) + kNextBytes);
  p.split.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + kNextBytes + delta_bytes);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == LMK_F32 ? window_f32_bwd(p, st) : window_sm100_bwd(p, dtype, st);
}
