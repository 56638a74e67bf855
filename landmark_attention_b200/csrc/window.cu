// extern "C" entry points of sliding-window attention: argument checks, the division of the sinks' gradient, the choice of kernels.
#include "common.cuh"
#include "window_params.h"

namespace lmk {
namespace {

constexpr size_t up256(size_t x) { return (x + 255) / 256 * 256; }

int check_window(const void* q, const void* k, const void* v, const float* lse, int B, int H, int Hkv, int Lq, int Lk, int D,
                 const int64_t* qs, const int64_t* ks, const int64_t* vs, int window, int sinks, float scale, int dtype) {
  LMK_CHECK_ARG(q && k && v && lse, "window attention: q, k, v or lse is null");
  LMK_CHECK_ARG(qs && ks && vs, "window attention: stride arrays are required");
  LMK_CHECK_ARG(B >= 1 && H >= 1 && Hkv >= 1 && Lq >= 1 && Lk >= 1, "window attention: empty problem (B=%d H=%d Hkv=%d Lq=%d Lk=%d)", B, H, Hkv, Lq, Lk);
  LMK_CHECK_ARG(H % Hkv == 0, "window attention: %d query heads are not a multiple of %d key heads", H, Hkv);
  LMK_CHECK_ARG((int64_t)B * H <= 65535, "window attention: B*H = %lld exceeds 65535", (long long)B * H);
  LMK_CHECK_ARG(Lk >= Lq, "window attention: %d queries are more than %d keys", Lq, Lk);
  LMK_CHECK_ARG(Lk <= (1 << 28), "window attention: %d keys exceed 2^28", Lk);
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
// fp32 rows are read as 16-byte vectors
bool rows_ok(const void* p, const int64_t* st, int dtype) {
  return dtype != LMK_F32 || (((uintptr_t)p & 15) == 0 && st[0] % 4 == 0 && st[1] % 4 == 0 && st[2] % 4 == 0);
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
void tile_sizes(int dtype, int* qt, int* kk) {
  (void)dtype;
  *qt = 64;
  *kk = 64;
}

}  // namespace
}  // namespace lmk

using namespace lmk;

extern "C" int lmk_window_fwd(const void* q, const void* k, const void* v, void* o, float* lse, const int32_t* lengths, int B, int H,
                              int Hkv, int Lq, int Lk, int D, const int64_t q_strides[3], const int64_t k_strides[3],
                              const int64_t v_strides[3], int window, int sinks, float sm_scale, int dtype, void* stream) {
  int rc = check_window(q, k, v, lse, B, H, Hkv, Lq, Lk, D, q_strides, k_strides, v_strides, window, sinks, sm_scale, dtype);
  if (rc != LMK_OK) return rc;
  LMK_CHECK_ARG(o != nullptr, "window attention: o is null");
  WindowParams p = {};
  fill(p, q, k, v, lengths, B, H, Hkv, Lq, Lk, D, q_strides, k_strides, v_strides, window, sinks, sm_scale);
  p.o = o;
  p.lse = lse;
  LMK_CHECK_ARG(rows_ok(q, q_strides, dtype) && rows_ok(k, k_strides, dtype) && rows_ok(v, v_strides, dtype),
                "window attention: fp32 rows must start on 16-byte boundaries");
  return window_general_fwd(p, dtype, static_cast<cudaStream_t>(stream));
}

extern "C" size_t lmk_window_bwd_workspace(int B, int H, int Hkv, int Lq, int Lk, int D, int window, int sinks, int dtype) {
  if (B < 1 || H < 1 || Hkv < 1 || Lq < 1 || Lk < Lq || D < 1 || window < 1 || sinks < 0) return 0;
  SinkSplit s;
  int qt, kk;
  tile_sizes(dtype, &qt, &kk);
  if (plan_split(&s, B, Hkv, Lq, Lk, window < Lk ? window : Lk, sinks < Lk ? sinks : Lk, qt, kk) != LMK_OK) return 0;
  return up256(sizeof(float) * (size_t)B * H * Lq) + up256(part_bytes(s, B, Hkv, D, kk));
}

extern "C" int lmk_window_bwd(const void* q, const void* k, const void* v, const void* o, const void* dO, const float* lse,
                              const int32_t* lengths, void* dQ, void* dK, void* dV, void* workspace, size_t workspace_bytes, int B, int H,
                              int Hkv, int Lq, int Lk, int D, const int64_t q_strides[3], const int64_t k_strides[3],
                              const int64_t v_strides[3], const int64_t do_strides[3], int window, int sinks, float sm_scale, int dtype,
                              void* stream) {
  int rc = check_window(q, k, v, lse, B, H, Hkv, Lq, Lk, D, q_strides, k_strides, v_strides, window, sinks, sm_scale, dtype);
  if (rc != LMK_OK) return rc;
  LMK_CHECK_ARG(o && dO && dQ && dK && dV && do_strides, "window attention backward: o, dO or a gradient is null");
  WindowParams p = {};
  fill(p, q, k, v, lengths, B, H, Hkv, Lq, Lk, D, q_strides, k_strides, v_strides, window, sinks, sm_scale);
  p.o = const_cast<void*>(o);
  p.dO = dO;
  p.lse = const_cast<float*>(lse);
  p.dq = dQ; p.dk = dK; p.dv = dV;
  for (int i = 0; i < 3; ++i) p.dos[i] = do_strides[i];
  LMK_CHECK_ARG(rows_ok(q, q_strides, dtype) && rows_ok(k, k_strides, dtype) && rows_ok(v, v_strides, dtype) && rows_ok(dO, do_strides, dtype),
                "window attention: fp32 rows must start on 16-byte boundaries");
  int qt, kk;
  tile_sizes(dtype, &qt, &kk);
  if ((rc = plan_split(&p.split, B, Hkv, Lq, Lk, p.window, p.sinks, qt, kk)) != LMK_OK) return rc;
  LMK_CHECK_ARG((int64_t)B * Hkv * (p.split.tiles > 0 ? p.split.tiles : 1) <= 65535, "window attention backward: %d sinks of %d key heads are too many",
                sinks, B * Hkv);
  const size_t delta_bytes = up256(sizeof(float) * (size_t)B * H * Lq), need = delta_bytes + up256(part_bytes(p.split, B, Hkv, D, kk));
  if (workspace == nullptr || workspace_bytes < need || ((uintptr_t)workspace & 255) != 0)
    return fail(LMK_ERR_WORKSPACE, "window attention backward: workspace of %zu bytes on a 256-byte boundary needed", need);
  p.delta = static_cast<float*>(workspace);
  p.split.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + delta_bytes);
  return window_general_bwd(p, dtype, static_cast<cudaStream_t>(stream));
}
