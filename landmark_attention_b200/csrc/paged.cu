// Paged key-value cache: append, attention of a sequence's newest tokens over its pages, eviction by accumulated attention weight.
//
// Pages are [n_pages, Hkv, page, D] (any page, head and row strides); table [B, max_pages] names a sequence's pages in order, lengths [B]
// say how many of their rows are tokens.  Nothing here trusts either: lengths are held between 0 and the table's capacity, a table
// entry outside of the pool is never followed (its keys count as hidden, and the device status says 601).
//
// Attention.  Query t of T stands at position p = length - T + t and sees key j if j <= p and (no window, p - j < window or j < sinks).
//   o = sum_j e^{s_j - m} v_j / sum_j e^{s_j - m}, m = max_j s_j, s_j = scale q . k_j  over the visible j; 0 where nothing is visible.
// Every visible row of K and V is read once for up to 16 query rows of its key head, 512 bytes a key and head at D = 128 in 16 bits against
// 4 D multiply-adds a query row: bound by HBM (5.8 TB/s with one row, 5.5 with 16).  What decides is how evenly the rows are dealt out and
// how many loads are in flight.
//   - The work of all sequences is one line of steps of 16 keys (sequence, key head, tile of 16 query rows, step).  Every CTA takes the same
//     length of it, so neither short sequences nor a large capacity leave SMs idle, whatever the lengths are; they are read on the
//     device, so a captured graph serves them as they grow.  A piece that holds all of its keys is written out at once; pieces of a
//     longer row leave their maximum, sum and unnormalised output, which a second kernel joins.
//   - A warp streams its own steps (every fourth of the CTA's) through its own ring in shared memory: no barrier of the CTA in the loop.  One
//     lane asks TMA for a step's rows (with 16-byte cp.async the addresses alone took 1200 clk a step, as long as the arithmetic, and
//     the warps could not keep up with the memory).  Rows that nobody sees are overwritten with zeros before the values are used, so
//     what they hold does not matter.
//   - Up to 16 of the G T query rows of a key head are the rows of an mma.sync tile (fp32: FMAs), and K and V are read once for them.  More rows
//     are further tiles, items of the line of their own that stream the history again: B8 Hkv8 D128, 16384 keys, 16 rows a key head 97 us,
//     20 or 32 rows 180, 64 rows 343.
//   - fp32 does the products of a row on the FMA units, a run-time number of rows a warp: 284 us with one row (3.8 TB/s), 1790 with 16.  Its
//     exponentials for rescaling and for the sums of weights are ex2.approx, off by 2^-22 of the value at most.
// Weights (for eviction): the scores are kept, 4 bytes a key and query row of the table's whole capacity, and the second kernel, which knows
// every row's maximum and sum, adds e^{s - m} / l of a group's rows to the key's weight.  One thread adds up one key: no atomics,
// bit-reproducible.
#include <atomic>
#include <type_traits>
#include "common.cuh"
#include "attn_params.h"
#include "mma16.cuh"
#include "sm100_ptx.cuh"

namespace lmk {
namespace {

using namespace ptx;

constexpr int kStep = 16;              // keys a warp takes at a time; pages are whole steps
constexpr int kRowTile = 16;           // query rows of one key head at a time
constexpr int kStages = 3;
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kBadPage = 601, kFull = 602, kErrRing = 611;

struct Pages {
  const void *k, *v;
  int64_t ks[3], vs[3];                // element strides {page, head, row}
  const int* table;
  const int* lengths;
  int B, Hkv, D, page, shift, n_pages, max_pages;      // page = 1 << shift
  int* status;
  __device__ int length(int b) const { return min(max(ld_behind_wait(lengths + b), 0), max_pages << shift); }
  __device__ int id(int b, int page_no) const { return ld_behind_wait(table + (int64_t)b * max_pages + page_no); }
};

// The steps of one sequence: `first` of them cover the sinks that lie in front of the window, the rest run from key `lo` (a multiple
// of 16) to the end.
struct Span {
  int len, lo, first, steps;
  __device__ int key(int step) const { return step < first ? step * kStep : lo + (step - first) * kStep; }
};
__device__ __forceinline__ Span span_of(int len, int T, int window, int sinks) {
  Span s;
  s.len = len;
  const int p0 = max(len - T, 0);
  const int lo = window > 0 && p0 >= window ? p0 - window + 1 : 0;
  s.lo = lo & ~(kStep - 1);
  s.first = min((min(sinks, lo) + kStep - 1) / kStep, s.lo / kStep);
  s.steps = s.first + (len - s.lo + kStep - 1) / kStep;
  return s;
}

struct AttendArgs {
  Pages pg;
  const void* q;
  int64_t qs[3];
  void* o;
  float* weights;                      // [B, Hkv, capacity] or null
  float decay;
  float* acc;                          // [2 grid][16][kD] unnormalised outputs of pieces
  float2* stat;                        // [2 grid][16] their (maximum, sum)
  float2* whole;                       // [items][16] of items in one piece (weights only)
  float* scores;                       // [B, Hkv, rows, capacity] in units of log2 (weights only)
  int H, T, G, rows, tiles, window, sinks, grid, least;
  bool one_piece;                      // every row is one CTA's: CTAs take items instead of lengths of the line
  float scale_log2;
  // query row of a key head -> head of its group, token
  __device__ int head(int r) const { return T == 1 ? r : r / T; }
  __device__ int token(int r) const { return T == 1 ? 0 : r % T; }
};

// All sequences' steps lie in one line; a CTA takes `piece` of them.  The sums over the sequences are worked out by whole warps.
template <typename F>
__device__ __forceinline__ int warp_total(int B, F f) {      // sum of f(b) over b < B
  int sum = 0;
  for (int b = threadIdx.x & 31; b < B; b += 32) sum += f(b);
  return __reduce_add_sync(0xffffffffu, sum);
}
struct Found { int b, before; };
template <typename F>
__device__ __forceinline__ Found warp_find(int B, int at, F f) {      // the sequence that holds step `at`, and the steps in front of it
  const int lane = threadIdx.x & 31;
  int before = 0;
  for (int b0 = 0; b0 < B; b0 += 32) {
    const int n = b0 + lane < B ? f(b0 + lane) : 0;
    int inc = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += v;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, n > 0 && before + inc > at);
    if (hit) {
      const int src = __ffs((int)hit) - 1;
      return {b0 + src, __shfl_sync(0xffffffffu, before + inc - n, src)};
    }
    before += __shfl_sync(0xffffffffu, inc, 31);
  }
  return {B, before};
}
__device__ __forceinline__ int piece_of(const AttendArgs& a, int total) { return max((total + a.grid - 1) / a.grid, a.least); }

// A stage of a warp's ring: the step's keys, then its values, as sub-tiles of 16 rows of 128 bytes in TMA's 128-byte swizzle.
constexpr int kSubTile = kStep * 128;
template <typename T, int kD> constexpr int kSubTiles = kD * (int)sizeof(T) / 128;
template <typename T, int kD> constexpr int kStageBytes = 2 * kSubTiles<T, kD> * kSubTile;
template <typename T, int kD, int kWarps> constexpr int kAttendSmem = kWarps * kStages * kStageBytes<T, kD>;
// byte offset of the 16-byte chunk c of row r
__device__ __forceinline__ uint32_t chunk_at(int r, int c) { return (uint32_t)((c >> 3) * kSubTile + r * 128 + (((c & 7) ^ (r & 7)) << 4)); }

// One warp's state over its steps of a piece: 16 query rows, of which a thread of the mma.sync form holds rows g and g + 8 (g = lane / 4).
template <typename T, int kD> struct Rows16 {
  uint32_t q[kD / 16][4];
  float o[kD / 8][4];
  float m[2], l[2];
};

template <typename T, int kD>
__device__ __forceinline__ void load_queries(Rows16<T, kD>& w, const AttendArgs& a, int b, int h, int row0) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
  const T* base[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int r = row0 + g + 8 * e;
    base[e] = r < a.rows ? reinterpret_cast<const T*>(a.q) + b * a.qs[0] + (int64_t)(h * a.G + a.head(r)) * a.qs[1] + (int64_t)a.token(r) * a.qs[2]
                         : nullptr;
  }
#pragma unroll
  for (int kk = 0; kk < kD / 16; ++kk)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int col = kk * 16 + (e >> 1) * 8 + 2 * t4;
      const T* p = base[e & 1];
      w.q[kk][e] = p != nullptr && col < a.pg.D ? *reinterpret_cast<const uint32_t*>(p + col) : 0u;
    }
#pragma unroll
  for (int n = 0; n < kD / 8; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) w.o[n][e] = 0.f;
  w.m[0] = w.m[1] = -INFINITY;
  w.l[0] = w.l[1] = 0.f;
}

template <typename T>
__device__ __forceinline__ uint32_t pack16(float a, float b) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    __nv_bfloat162 t = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&t);
  } else {
    __half2 t = __floats2half2_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&t);
  }
}

// visible(row e of the thread, key): see the head of the file
template <typename T, int kD, typename Seen, typename Keep>
__device__ __forceinline__ void take_step(Rows16<T, kD>& w, const uint8_t* stage, float scale_log2, bool all, Seen seen, Keep keep) {
  const int lane = threadIdx.x & 31, t4 = lane & 3;
  float s[2][4] = {}, s1[2][4] = {};                 // even and odd features: two shorter chains of products
  const int kr = (lane >> 4) * 8 + (lane & 7), kc = (lane >> 3) & 1;
#pragma unroll
  for (int kk = 0; kk < kD / 16; ++kk) {
    uint32_t f[4];
    ldmatrix_x4(f, stage + chunk_at(kr, kk * 2 + kc));
    mma16<T>(kk & 1 ? s1[0] : s[0], w.q[kk][0], w.q[kk][1], w.q[kk][2], w.q[kk][3], f[0], f[1]);
    mma16<T>(kk & 1 ? s1[1] : s[1], w.q[kk][0], w.q[kk][1], w.q[kk][2], w.q[kk][3], f[2], f[3]);
  }
  // element (n, e): row g + 8 (e / 2), key 8 n + 2 t + e % 2
  float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
  for (int n = 0; n < 2; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float x = (s[n][e] + s1[n][e]) * scale_log2;
      if (!all && !seen(e >> 1, 8 * n + 2 * t4 + (e & 1))) x = -INFINITY;
      s[n][e] = x;
      mx[e >> 1] = max3_nan(mx[e >> 1], x, x);
    }
  keep(s);
  bool grew = false;
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    mx[e] = max3_nan(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 1), w.m[e]);
    const float other = __shfl_xor_sync(0xffffffffu, mx[e], 2);
    mx[e] = max3_nan(mx[e], other, other);
    grew |= !(mx[e] == w.m[e]);
  }
  float shift[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) shift[e] = mx[e] == -INFINITY ? 0.f : mx[e];
  if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const float f = ex2(w.m[e] - shift[e]);        // 0 from -inf
      w.l[e] *= f;
      w.m[e] = mx[e];
#pragma unroll
      for (int n = 0; n < kD / 8; ++n) {
        w.o[n][2 * e] *= f;
        w.o[n][2 * e + 1] *= f;
      }
    }
  }
#pragma unroll
  for (int n = 0; n < 2; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      s[n][e] = ex2(s[n][e] - shift[e >> 1]);
      w.l[e >> 1] += s[n][e];                        // a thread's own keys; joined at the end of the piece
    }
  // the weights enter the product in 16 bits (half a step of relative error each, as in every kernel here); their sum l does not
  const uint32_t p0 = pack16<T>(s[0][0], s[0][1]), p1 = pack16<T>(s[0][2], s[0][3]);
  const uint32_t p2 = pack16<T>(s[1][0], s[1][1]), p3 = pack16<T>(s[1][2], s[1][3]);
  const uint8_t* vs = stage + kSubTiles<T, kD> * kSubTile;
  const int vr = ((lane >> 3) & 1) * 8 + (lane & 7), vc = lane >> 4;
#pragma unroll
  for (int n = 0; n < kD / 16; ++n) {
    uint32_t f[4];
    ldmatrix_x4_trans(f, vs + chunk_at(vr, n * 2 + vc));
    mma16<T>(w.o[2 * n], p0, p1, p2, p3, f[0], f[1]);
    mma16<T>(w.o[2 * n + 1], p0, p1, p2, p3, f[2], f[3]);
  }
}

// A warp's unnormalised outputs as [16][kD] floats, and its maxima and sums
template <typename T, int kD>
__device__ __forceinline__ void leave_result(Rows16<T, kD>& w, float* to, float2* stat) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    w.l[e] += __shfl_xor_sync(0xffffffffu, w.l[e], 1);
    w.l[e] += __shfl_xor_sync(0xffffffffu, w.l[e], 2);
    if (t4 == 0) stat[g + 8 * e] = make_float2(w.m[e], w.l[e]);
#pragma unroll
    for (int n = 0; n < kD / 8; ++n)
      *reinterpret_cast<float2*>(to + (g + 8 * e) * kD + n * 8 + 2 * t4) = make_float2(w.o[n][2 * e], w.o[n][2 * e + 1]);
  }
}

// fp32: a lane holds the keys' scores as (key, half of the features), then the outputs of the features 4 lane .. 4 lane + 3
template <int kD> struct Rows32 {
  float o[kRowTile][kD / 32];
  float m[kRowTile], l[kRowTile];
};

// kWarps: 4, with two CTAs an SM or four for 64 features; 8 on whole rows where there are no more of them than SMs, and the latency of a
// warp's steps counts (us: 32 rows of 300 keys 10.1 with 4, 8.8 with 8; 512 rows 23.5 / 34.6).
// (registers are only held down where four CTAs are to fit; 128 features then leave room for the next kernel's first CTAs)
template <typename T, int kD, int kWarps> constexpr int kAttendPerSm = kWarps == 4 && kD == 64 && sizeof(T) == 2 ? 4 : 1;
template <typename T, int kD, int kWarps>
__global__ void __launch_bounds__(kWarps * 32, kAttendPerSm<T, kD, kWarps>)
paged_attend_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ AttendArgs a) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ float2 s_stat[kWarps][kRowTile];
  __shared__ int s_free[kWarps];
  __shared__ uint64_t s_full[kWarps][kStages];
  constexpr bool kF32 = std::is_same<T, float>::value;
  constexpr int kSub = kSubTiles<T, kD>;
  uint8_t* const smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const int tid = threadIdx.x, warp = warp_uniform(tid >> 5), lane = tid & 31;
  if (lane == 0) {
    for (int k = 0; k < kStages; ++k) mbar_init(smem_u32(&s_full[warp][k]), 1);
    mbar_init_fence();
    prefetch_tensormap(&tm_k);
    prefetch_tensormap(&tm_v);
  }
  __syncwarp();
  grid_dep_wait();
  grid_dep_launch();
  const Pages& pg = a.pg;
  const int per_seq = pg.Hkv * a.tiles;
  const int len_lane = lane < pg.B ? pg.length(lane) : 0;      // the first 32 lengths stay at hand
  auto length = [&](int b) { return b < 32 ? __shfl_sync(0xffffffffu, len_lane, b) : pg.length(b); };      // (the same b in all lanes)
  auto steps_of = [&](int b) { return per_seq * span_of(b < 32 ? len_lane : pg.length(b), a.T, a.window, a.sinks).steps; };
  // sequences without keys: their outputs are zeros (a share of the sequences for every CTA)
  for (int b = blockIdx.x; b < pg.B; b += gridDim.x)
    if (length(b) == 0)
      for (int64_t i = tid; i < (int64_t)a.H * a.T * pg.D; i += kWarps * 32) reinterpret_cast<T*>(a.o)[b * (int64_t)a.H * a.T * pg.D + i] = from_f32<T>(0.f);
  uint8_t* const ring = smem + warp * kStages * kStageBytes<T, kD>;
  const uint32_t ring_at = (uint32_t)warp_uniform((int)smem_u32(ring)), bar_at = (uint32_t)warp_uniform((int)smem_u32(&s_full[warp][0]));
  static_assert(kRowTile * kD * 4 <= kStageBytes<T, kD>, "a warp's outputs fit a stage");

  // A place in the line, moved on by whole warps.
  struct Place {
    int b, item, step;
    Span sp;
  };
  auto settle = [&](Place& p) {                      // `step` may lie behind the item's end
    while (p.step >= p.sp.steps) {
      p.step -= p.sp.steps;
      if (++p.item < per_seq) continue;
      p.item = 0;
      do {                                           // the next sequence that has keys
        if (++p.b >= pg.B) return;                   // behind the last one: nothing is taken from there
        p.sp = span_of(length(p.b), a.T, a.window, a.sinks);
      } while (p.sp.steps == 0);
    }
  };
  const int64_t cap = (int64_t)pg.max_pages << pg.shift;
  int i = 0;                                         // this warp's steps that are done; stage (i + kStages - 1) % kStages is free

  // The steps begin .. end - 1 of the line, of which `now` is the first.
  auto take = [&](int begin, int end, Place now) {
    // Loads run ahead of the steps that use them, also into the next item: first the page's number, then its rows.
    const int last = i + (end - begin - warp + kWarps - 1) / kWarps;       // this warp's steps: begin + warp, + kWarps, ...
    Place ask = now;
    ask.step += warp;
    settle(ask);
    struct Asked { int h, key0, id; };
    unsigned bad = 0;                                // bit n % kStages: step n, in that stage, has no page
    auto ask_page = [&](int n) {
      Asked x = {0, 0, 0};
      if (n >= last) return x;
      x.h = a.tiles == 1 ? ask.item : ask.item / a.tiles;
      x.key0 = ask.sp.key(ask.step);
      x.id = pg.id(ask.b, x.key0 >> pg.shift);
      ask.step += kWarps;
      settle(ask);
      return x;
    };
    auto issue = [&](int n, const Asked& x) {
      if (n >= last) return;
      // one elected lane issues; what it needs is made warp-uniform, or the compiler moves it to uniform registers copy by copy
      const int asked = warp_uniform(x.id), row = warp_uniform(x.key0 & (pg.page - 1)), h = warp_uniform(x.h);
      const bool ok = asked >= 0 && asked < pg.n_pages;
      const unsigned bit = 1u << (n % kStages);
      bad = ok ? bad & ~bit : bad | bit;
      const uint32_t to = ring_at + (uint32_t)(n % kStages) * kStageBytes<T, kD>, bar = bar_at + (uint32_t)(n % kStages) * 8u;
      const int id = ok ? asked : pg.n_pages;        // behind the pool: zeros
      if (elect_one()) {
        if (!ok) note_condition(pg.status, kBadPage);
        mbar_arrive_expect_tx(bar, kStageBytes<T, kD>);
#pragma unroll
        for (int c = 0; c < kSub; ++c) {
          tma_load_4d(to + c * kSubTile, &tm_k, bar, c * (128 / (int)sizeof(T)), row, h, id);
          tma_load_4d(to + (kSub + c) * kSubTile, &tm_v, bar, c * (128 / (int)sizeof(T)), row, h, id);
        }
      }
    };
    Asked next;
    {
      Asked first[kStages];
#pragma unroll
      for (int k = 0; k < kStages; ++k) first[k] = ask_page(i + k);
#pragma unroll
      for (int k = 0; k < kStages - 1; ++k) issue(i + k, first[k]);
      next = first[kStages - 1];
    }
    for (int at = begin; at < end;) {
      const Span sp = now.sp;
      const int b = now.b, step0 = now.step, h = now.item / a.tiles, row0 = (now.item - h * a.tiles) * kRowTile;
      const int count = min(sp.steps - step0, end - at);
      const int p0 = sp.len - a.T;                               // position of the first token's queries
      const int first = (warp - (at - begin)) & (kWarps - 1);
      const int64_t score_row = ((int64_t)b * pg.Hkv + h) * a.rows;
      const int lo = a.window > 0 && p0 >= a.window ? p0 - a.window + 1 : 0;      // the first key that the first token's window holds
      // The step's rows are there; those that nobody sees are made zeros (scores are hidden by a select, values would be multiplied).
      auto arrive = [&](int key0) {
        mbar_wait(bar_at + (uint32_t)(i % kStages) * 8u, (i / kStages) & 1, pg.status, kErrRing);
        if (key0 + kStep <= sp.len && (key0 >= lo || key0 + kStep <= a.sinks)) return;
        const uint32_t at_v = ring_at + (uint32_t)(i % kStages) * kStageBytes<T, kD> + kSub * kSubTile;
        for (int r = 0; r < kStep; ++r) {
          const int key = key0 + r;
          if (key < sp.len && (key >= lo || key < a.sinks)) continue;
          for (int c = lane; c < kSub * 8; c += 32)
            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(at_v + (c >> 3) * kSubTile + r * 128 + (c & 7) * 16), "r"(0) : "memory");
        }
        __syncwarp();
      };
      // every row that exists sees all 16 keys (the last token's window is the one that has moved on furthest)
      auto all_see = [&](int key0, bool no_page) {
        return !no_page && p0 >= 0 && key0 + kStep - 1 <= p0 && (a.window == 0 || p0 + a.T - 1 - key0 < a.window);
      };

      if constexpr (!kF32) {
        Rows16<T, kD> w;
        load_queries<T, kD>(w, a, b, h, row0);
        int pos[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int r = row0 + (lane >> 2) + 8 * e;
          pos[e] = r < a.rows ? p0 + a.token(r) : -1;
        }
        for (int k = first; k < count; k += kWarps, ++i) {
          const bool no_page = bad >> (i % kStages) & 1u;
          issue(i + kStages - 1, next);
          next = ask_page(i + kStages);
          const int key0 = sp.key(step0 + k);
          arrive(key0);
          take_step<T, kD>(w, ring + (i % kStages) * kStageBytes<T, kD>, a.scale_log2, all_see(key0, no_page),
              [&](int e, int j) {
                const int key = key0 + j;
                return !no_page && key <= pos[e] && (a.window == 0 || pos[e] - key < a.window || key < a.sinks);
              },
              [&](const float (&s)[2][4]) {
                if (a.weights == nullptr) return;
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                  for (int e = 0; e < 2; ++e) {
                    const int r = row0 + (lane >> 2) + 8 * e;
                    if (r < a.rows)
                      *reinterpret_cast<float2*>(a.scores + (score_row + r) * cap + key0 + 8 * n + 2 * (lane & 3)) =
                          make_float2(s[n][2 * e], s[n][2 * e + 1]);
                  }
              });
          if (i + kStages < last) fence_proxy_async_smem();      // TMA writes the stage again
          __syncwarp();
        }
        leave_result<T, kD>(w, reinterpret_cast<float*>(ring + ((i + kStages - 1) % kStages) * kStageBytes<T, kD>), s_stat[warp]);
      } else {
        // fp32 on the FMA units.  Scores: lane = (key, half of the features); outputs: lane = kD / 32 features of every row.
        Rows32<kD> w;
        const int n_rows = min(kRowTile, a.rows - row0);
        float* const qs = reinterpret_cast<float*>(smem + kAttendSmem<T, kD, kWarps>);         // [16][kD], the CTA's query rows
        float* const ps = qs + kRowTile * kD + warp * kRowTile * kStep;                // [16][16], the warp's weights
        for (int e = tid; e < kRowTile * kD; e += kWarps * 32) {
          const int r = row0 + e / kD, c = e % kD;
          qs[e] = r < a.rows && c < pg.D ? *(reinterpret_cast<const float*>(a.q) + b * a.qs[0] + (int64_t)(h * a.G + r / a.T) * a.qs[1] +
                                             (int64_t)(r % a.T) * a.qs[2] + c) : 0.f;
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < kRowTile; ++r) {
          w.m[r] = -INFINITY;
          w.l[r] = 0.f;
#pragma unroll
          for (int c = 0; c < kD / 32; ++c) w.o[r][c] = 0.f;
        }
        for (int k = first; k < count; k += kWarps, ++i) {
          const bool no_page = bad >> (i % kStages) & 1u;
          issue(i + kStages - 1, next);
          next = ask_page(i + kStages);
          const int key0 = sp.key(step0 + k);
          arrive(key0);
          const uint8_t* stage = ring + (i % kStages) * kStageBytes<T, kD>;
          const int j = lane & 15, half = lane >> 4;
          float s[kRowTile];
#pragma unroll
          for (int r = 0; r < kRowTile; ++r) s[r] = 0.f;
          for (int c = 0; c < kD / 8; ++c) {                   // the half's 16-byte chunks
            const int chunk = half * (kD / 8) + c;
            const float4 x = *reinterpret_cast<const float4*>(stage + chunk_at(j, chunk));
#pragma unroll
            for (int r = 0; r < kRowTile; ++r) {
              if (r >= n_rows) break;
              const float4 y = *reinterpret_cast<const float4*>(qs + r * kD + chunk * 4);
              s[r] = fmaf(x.x, y.x, fmaf(x.y, y.y, fmaf(x.z, y.z, fmaf(x.w, y.w, s[r]))));
            }
          }
#pragma unroll
          for (int r = 0; r < kRowTile; ++r) {
            if (r >= n_rows) break;
            float x = (s[r] + __shfl_xor_sync(0xffffffffu, s[r], 16)) * a.scale_log2;
            const int pos = p0 + a.token(row0 + r), key = key0 + j;
            if (no_page || key > pos || !(a.window == 0 || pos - key < a.window || key < a.sinks)) x = -INFINITY;
            if (a.weights != nullptr && half == 0) a.scores[(score_row + row0 + r) * cap + key] = x;
            float mx = x;
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) {
              const float y = __shfl_xor_sync(0xffffffffu, mx, o);
              mx = max3_nan(mx, y, y);
            }
            mx = max3_nan(mx, w.m[r], w.m[r]);
            const float shift = mx == -INFINITY ? 0.f : mx;
            const float f = ex2(w.m[r] - shift);
            w.m[r] = mx;
            const float p = exp2f(x - shift);
            w.l[r] = w.l[r] * f + (half == 0 ? p : 0.f);
#pragma unroll
            for (int c = 0; c < kD / 32; ++c) w.o[r][c] *= f;
            if (half == 0) ps[r * kStep + j] = p;
          }
          __syncwarp();
          const uint8_t* vs = stage + kSubTiles<T, kD> * kSubTile;
          for (int key = 0; key < kStep; ++key) {
            float v[kD / 32];
#pragma unroll
            for (int c = 0; c < kD / 32; ++c) {
              const int f = lane * (kD / 32) + c;
              v[c] = *reinterpret_cast<const float*>(vs + chunk_at(key, f / 4) + (f % 4) * 4);
            }
#pragma unroll
            for (int r = 0; r < kRowTile; ++r) {
              if (r >= n_rows) break;
              const float p = ps[r * kStep + key];
#pragma unroll
              for (int c = 0; c < kD / 32; ++c) w.o[r][c] = fmaf(p, v[c], w.o[r][c]);
            }
          }
          if (i + kStages < last) fence_proxy_async_smem();
          __syncwarp();
        }
        float* const result = reinterpret_cast<float*>(ring + ((i + kStages - 1) % kStages) * kStageBytes<T, kD>);
#pragma unroll
        for (int r = 0; r < kRowTile; ++r) {
          const float l = warp_sum(w.l[r]);
          if (lane == 0) s_stat[warp][r] = make_float2(w.m[r], l);
#pragma unroll
          for (int c = 0; c < kD / 32; ++c) result[r * kD + lane * (kD / 32) + c] = w.o[r][c];
        }
      }

      // the warps' results, joined, while the next item's rows are on their way
      const int free_stage = (i + kStages - 1) % kStages;
      if (lane == 0) s_free[warp] = free_stage;
      __syncthreads();
      {
        constexpr int kPer = kWarps * 2;               // threads a row
        const int r = tid / kPer, part = tid % kPer;
        const float* res[kWarps];
        float mx = -INFINITY, l = 0.f, f[kWarps];
#pragma unroll
        for (int k = 0; k < kWarps; ++k) {
          res[k] = reinterpret_cast<const float*>(smem + (k * kStages + s_free[k]) * kStageBytes<T, kD>);
          mx = max3_nan(mx, s_stat[k][r].x, s_stat[k][r].x);
        }
        const float shift = mx == -INFINITY ? 0.f : mx;
#pragma unroll
        for (int k = 0; k < kWarps; ++k) {
          f[k] = ex2(s_stat[k][r].x - shift);
          l += f[k] * s_stat[k][r].y;
        }
        const bool exists = row0 + r < a.rows, all = count == sp.steps;
        const int64_t slot = 2 * (int64_t)blockIdx.x + (step0 > 0 ? 0 : 1);
        const float inv = l == 0.f ? 0.f : 1.f / l;
        T* const orow = reinterpret_cast<T*>(a.o) + (((int64_t)b * a.H + h * a.G + a.head(row0 + r)) * a.T + a.token(row0 + r)) * pg.D;
        float* const arow = a.acc + (slot * kRowTile + r) * kD;
#pragma unroll
        for (int c = 0; c < kD / (4 * kPer); ++c) {
          const int col = (c * kPer + part) * 4;
          float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int k = 0; k < kWarps; ++k) {
            const float4 x = *reinterpret_cast<const float4*>(res[k] + r * kD + col);
            sum.x = fmaf(f[k], x.x, sum.x);
            sum.y = fmaf(f[k], x.y, sum.y);
            sum.z = fmaf(f[k], x.z, sum.z);
            sum.w = fmaf(f[k], x.w, sum.w);
          }
          if (!exists || col >= pg.D) continue;
          if (!all) {
            *reinterpret_cast<float4*>(arow + col) = sum;
          } else if constexpr (kF32) {
            *reinterpret_cast<float4*>(orow + col) = make_float4(sum.x * inv, sum.y * inv, sum.z * inv, sum.w * inv);
          } else {
            *reinterpret_cast<uint2*>(orow + col) = make_uint2(pack16<T>(sum.x * inv, sum.y * inv), pack16<T>(sum.z * inv, sum.w * inv));
          }
        }
        if (exists && part == 0) {
          if (!all) a.stat[slot * kRowTile + r] = make_float2(mx, l);
          else if (a.weights != nullptr) a.whole[(((int64_t)b * pg.Hkv + h) * a.tiles + row0 / kRowTile) * kRowTile + r] = make_float2(mx, l);
        }
      }
      fence_proxy_async_smem();                      // the outputs' stages belong to TMA again
      __syncthreads();
      at += count;
      now.step += count;
      settle(now);
    }
  };

  for (int x = blockIdx.x;; x += gridDim.x) {
    int b, item, step = 0, begin = 0, end;
    Span sp;
    if (a.one_piece) {
      if (x >= pg.B * per_seq) break;
      b = x / per_seq;
      item = x - b * per_seq;
      sp = span_of(length(b), a.T, a.window, a.sinks);
      end = sp.steps;
    } else {
      const int total = warp_total(pg.B, steps_of), piece = piece_of(a, total);
      if (blockIdx.x > (unsigned)(total / piece)) break;
      begin = blockIdx.x * piece;
      end = min(begin + piece, total);
      if (begin >= end) break;
      const Found f = warp_find(pg.B, begin, steps_of);
      b = f.b;
      sp = span_of(length(b), a.T, a.window, a.sinks);
      item = (begin - f.before) / sp.steps;
      step = begin - f.before - item * sp.steps;
    }
    if (begin < end) take(begin, end, {b, item, step, sp});
    if (!a.one_piece) break;
  }
}

// Behind the pieces: blocks 0 .. joins - 1 join the rows that several CTAs worked on, one (item, slice of 32 features) each; the others add
// every key's share of its group's rows to its weight, 1024 keys of a (sequence, key head) each.  Lengths are read ahead of the wait:
// they were complete before the attention kernel was behind its own.
constexpr int kJoinThreads = 256, kRunKeys = 4 * kJoinThreads;
template <typename T, int kD>
__global__ void __launch_bounds__(kJoinThreads) paged_finish_kernel(const __grid_constant__ AttendArgs a, int joins) {
  extern __shared__ float2 s_rows[];                 // (maximum, 1 / sum) of the group's rows
  const Pages& pg = a.pg;
  const int tid = threadIdx.x;
  const int per_seq = pg.Hkv * a.tiles;
  auto steps_of = [&](int i) { return per_seq * span_of(pg.length(i), a.T, a.window, a.sinks).steps; };
  const bool join = (int)blockIdx.x < joins;
  const int x = join ? blockIdx.x / (kD / 32) : blockIdx.x - joins, slice = blockIdx.x % (kD / 32);
  const int64_t cap = (int64_t)pg.max_pages << pg.shift;
  const int runs = (int)((cap + kRunKeys - 1) / kRunKeys);
  const int b = join ? x / per_seq : x / runs / pg.Hkv;
  const int piece = piece_of(a, warp_total(pg.B, steps_of)), before = warp_total(b, steps_of);
  const int len = pg.length(b);
  const Span sp = span_of(len, a.T, a.window, a.sinks);
  grid_dep_wait();
  grid_dep_launch();
  if (sp.steps == 0) return;
  auto first_cta = [&](int item) { return (before + item * sp.steps) / piece; };
  auto last_cta = [&](int item) { return (before + item * sp.steps + sp.steps - 1) / piece; };

  if (join) {
    const int item = x - b * per_seq, c0 = first_cta(item), c1 = last_cta(item);
    if (c0 == c1) return;
    const int h = item / a.tiles, row0 = (item - h * a.tiles) * kRowTile;
    const int n_rows = min(kRowTile, a.rows - row0);
    auto slot_of = [&](int c) { return 2 * (int64_t)c + (c == c0 ? 1 : 0); };
    const int r = tid >> 4, part = tid & 15;         // 16 threads a row
    float mx = -INFINITY, l = 0.f;
    if (r < n_rows)
      for (int c = c0 + part; c <= c1; c += 16) {
        const float m = a.stat[slot_of(c) * kRowTile + r].x;
        mx = max3_nan(mx, m, m);
      }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) {
      const float m = __shfl_xor_sync(0xffffffffu, mx, o);
      mx = max3_nan(mx, m, m);
    }
    const float shift = mx == -INFINITY ? 0.f : mx;
    const int col = slice * 32 + part * 2;
    if (r >= n_rows || col >= pg.D) return;
    float2 sum = make_float2(0.f, 0.f);
#pragma unroll 4
    for (int c = c0; c <= c1; ++c) {
      const float2 st = a.stat[slot_of(c) * kRowTile + r];
      const float2 v = *reinterpret_cast<const float2*>(a.acc + (slot_of(c) * kRowTile + r) * kD + col);
      const float f = ex2(st.x - shift);
      l = fmaf(f, st.y, l);
      sum.x = fmaf(f, v.x, sum.x);
      sum.y = fmaf(f, v.y, sum.y);
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    T* const to = reinterpret_cast<T*>(a.o) + (((int64_t)b * a.H + h * a.G + a.head(row0 + r)) * a.T + a.token(row0 + r)) * pg.D + col;
    to[0] = from_f32<T>(sum.x * inv);
    to[1] = from_f32<T>(sum.y * inv);
    return;
  }

  // weights[b, h, j] = decay weights[b, h, j] + sum over the rows of the group of e^{s_j - m} / l, for all j < length
  const int h = x / runs - b * pg.Hkv, j0 = (x % runs) * kRunKeys;
  if (j0 >= len) return;
  for (int r = tid; r < a.rows; r += kJoinThreads) {
    const int tile = r / kRowTile, rr = r - tile * kRowTile, item = h * a.tiles + tile, c0 = first_cta(item), c1 = last_cta(item);
    float2 y;
    if (a.one_piece || c0 == c1) {
      y = a.whole[((int64_t)b * per_seq + item) * kRowTile + rr];
    } else {
      y = make_float2(-INFINITY, 0.f);
      for (int c = c0; c <= c1; ++c) {
        const float2 z = a.stat[(2 * (int64_t)c + (c == c0 ? 1 : 0)) * kRowTile + rr];
        const float m = max3_nan(y.x, z.x, z.x), shift = m == -INFINITY ? 0.f : m;
        y.y = y.y * ex2(y.x - shift) + z.y * ex2(z.x - shift);
        y.x = m;
      }
    }
    s_rows[r] = make_float2(y.x == -INFINITY ? 0.f : y.x, y.y == 0.f ? 0.f : 1.f / y.y);
  }
  __syncthreads();
  const int j = j0 + tid * 4;                          // four keys a thread; whole steps are seen or not
  if (j >= len) return;
  float* const to = a.weights + ((int64_t)b * pg.Hkv + h) * cap + j;
  float4 w = make_float4(0.f, 0.f, 0.f, 0.f);          // decay 0: whatever stood there is not read
  if (a.decay != 0.f) {
    w = *reinterpret_cast<const float4*>(to);
    w = make_float4(a.decay * w.x, a.decay * w.y, a.decay * w.z, a.decay * w.w);
  }
  if (j < sp.first * kStep || j >= sp.lo) {
    const float* s = a.scores + ((int64_t)b * pg.Hkv + h) * a.rows * cap + j;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int r = 0; r < a.rows; ++r, s += cap) {
      const float4 v = *reinterpret_cast<const float4*>(s);
      const float2 st = s_rows[r];
      sum.x = fmaf(ex2(v.x - st.x), st.y, sum.x);
      sum.y = fmaf(ex2(v.y - st.x), st.y, sum.y);
      sum.z = fmaf(ex2(v.z - st.x), st.y, sum.z);
      sum.w = fmaf(ex2(v.w - st.x), st.y, sum.w);
    }
    w = make_float4(w.x + sum.x, w.y + sum.y, w.z + sum.z, w.w + sum.w);
  }
  if (j + 3 < len) {
    *reinterpret_cast<float4*>(to) = w;
  } else {
    to[0] = w.x;
    if (j + 1 < len) to[1] = w.y;
    if (j + 2 < len) to[2] = w.z;
  }
}

// ---------------------------------------------------------------------------------------------- append
// Rows 0 .. n_b - 1 of k_new, v_new go behind the sequence's tokens; the new keys' weights start at 0.
struct AppendArgs {
  Pages pg;
  const void *k_new, *v_new;
  int64_t kns[3], vns[3];
  void *k, *v;
  int* lengths;
  const int* counts;                   // [B] or null: all T rows
  float* weights;
  int T, chunks;                       // a CTA copies a chunk of rows of all heads
};
__device__ __forceinline__ int append_count(const AppendArgs& a, int b, int len) {
  const int want = a.counts != nullptr ? min(max(ld_behind_wait(a.counts + b), 0), a.T) : a.T;
  const int room = (a.pg.max_pages << a.pg.shift) - len;
  if (want > room && threadIdx.x == 0) note_condition(a.pg.status, kFull);
  return min(want, room);
}
template <typename V>                  // 16-byte vectors
__global__ void __launch_bounds__(256) paged_append_kernel(const __grid_constant__ AppendArgs a, int vecs, int size) {
  grid_dep_wait();
  grid_dep_launch();
  const Pages& pg = a.pg;
  const int b = blockIdx.y, len = pg.length(b);
  const int n = append_count(a, b, len);
  const int64_t cap = (int64_t)pg.max_pages << pg.shift;
  const int per_row = pg.Hkv * vecs;
  const int rows = (a.T + a.chunks - 1) / a.chunks, r0 = blockIdx.x * rows, r1 = min(n, r0 + rows);
  for (int64_t e = threadIdx.x; e < (int64_t)(r1 - r0) * per_row; e += blockDim.x) {
    const int r = r0 + (int)(e / per_row), x = (int)(e % per_row), h = x / vecs, c = x - h * vecs;
    const int at = len + r, id = pg.id(b, at >> pg.shift);
    if (a.weights != nullptr && c == 0) a.weights[((int64_t)b * pg.Hkv + h) * cap + at] = 0.f;      // (a key without a page counts too)
    if (id < 0 || id >= pg.n_pages) {
      note_condition(pg.status, kBadPage);
      continue;
    }
    const int64_t row = at & (pg.page - 1);
    auto bytes = [&](int64_t elements) { return elements * size; };
    const V xk = *reinterpret_cast<const V*>((const char*)a.k_new + bytes(b * a.kns[0] + h * a.kns[1] + r * a.kns[2]) + c * 16ll);
    const V xv = *reinterpret_cast<const V*>((const char*)a.v_new + bytes(b * a.vns[0] + h * a.vns[1] + r * a.vns[2]) + c * 16ll);
    *reinterpret_cast<V*>((char*)a.k + bytes((int64_t)id * pg.ks[0] + h * pg.ks[1] + row * pg.ks[2]) + c * 16ll) = xk;
    *reinterpret_cast<V*>((char*)a.v + bytes((int64_t)id * pg.vs[0] + h * pg.vs[1] + row * pg.vs[2]) + c * 16ll) = xv;
  }
  if (a.chunks == 1) {
    __syncthreads();                   // all threads have read the length
    if (threadIdx.x == 0) a.lengths[b] = len + n;
  }
}
// several CTAs a sequence: the lengths move on when all of them have read them
__global__ void __launch_bounds__(256) paged_advance_kernel(const __grid_constant__ AppendArgs a) {
  grid_dep_wait();
  grid_dep_launch();
  const int b = blockIdx.x * blockDim.x + threadIdx.x;
  if (b >= a.pg.B) return;
  const int len = a.pg.length(b);
  const int want = a.counts != nullptr ? min(max(ld_behind_wait(a.counts + b), 0), a.T) : a.T;
  a.lengths[b] = len + min(want, (a.pg.max_pages << a.pg.shift) - len);
}

// ---------------------------------------------------------------------------------------------- eviction
// Of a sequence with more than `budget` tokens the first `sinks`, the last `recent` and the most attended of the rest stay, in order.
//   1. select: a CTA per (sequence, key head).  The smallest weight that stays is found digit by digit (8 bits, most significant
//      first) from histograms of the weights' order-preserving bit patterns; of the keys with exactly that weight the first ones
//      stay.  Then one ordered pass with a running count writes the survivors' positions and weights.
//   2. move: their K and V rows are copied to the fresh pages, 16 bytes a thread and access; nothing is moved inside a page, so reads and
//      writes cannot meet, and pages that other sequences read stay as they are.
// Bytes: the survivors' rows once in and once out; the selection reads 4 bytes a key.
struct EvictArgs {
  Pages pg;
  void *k, *v;
  const float* weights;
  const int* fresh;
  int n_fresh, budget, recent, sinks;
  int *table_out, *lengths_out, *kept;
  float* weights_out;
};
constexpr int kSelectThreads = 1024, kSelectWarps = kSelectThreads / 32;
constexpr int kHists = 8;                                      // copies of the histogram, a warp in eight has one to itself
constexpr int kCachedKeys = 48 * 1024;                         // longer rows of weights are read from memory in every pass
// ascending as unsigned; the two zeros are equal, NaN counts as the largest.  On the bits alone: arithmetic may drop a NaN's sign.
__device__ __forceinline__ uint32_t order_bits(uint32_t u) {
  if ((u & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
  if ((u & 0x7fffffffu) == 0) return 0x80000000u;
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
template <bool kCached>
__global__ void __launch_bounds__(kSelectThreads) paged_select_kernel(const __grid_constant__ EvictArgs a) {
  extern __shared__ uint32_t s_w[];                            // kCached: the row's weights
  __shared__ int hist[kHists][256];
  __shared__ int s_stay[kSelectWarps], s_tie[kSelectWarps];
  __shared__ uint32_t s_prefix;
  __shared__ int s_left;
  grid_dep_wait();
  grid_dep_launch();
  const Pages& pg = a.pg;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int b = blockIdx.x / pg.Hkv, h = blockIdx.x - b * pg.Hkv;
  const int64_t cap = (int64_t)pg.max_pages << pg.shift, at = ((int64_t)b * pg.Hkv + h) * cap;
  const uint32_t* const w = reinterpret_cast<const uint32_t*>(a.weights) + at;
  uint32_t* const wo = reinterpret_cast<uint32_t*>(a.weights_out) + at;
  int* const kept = a.kept + ((int64_t)b * pg.Hkv + h) * a.budget;
  const int len = pg.length(b);
  const bool over = len > a.budget;
  if (h == 0) {
    for (int i = tid; i < pg.max_pages; i += kSelectThreads)
      a.table_out[(int64_t)b * pg.max_pages + i] =
          !over ? pg.id(b, i) : (i < a.n_fresh && ((int64_t)i << pg.shift) < a.budget ? ld_behind_wait(a.fresh + (int64_t)b * a.n_fresh + i) : -1);
    if (tid == 0) a.lengths_out[b] = over ? a.budget : len;
  }
  if (!over) {
    for (int64_t j = tid; j < cap; j += kSelectThreads) wo[j] = j < len ? w[j] : 0u;
    for (int j = tid; j < a.budget; j += kSelectThreads) kept[j] = j < len ? j : -1;
    return;
  }
  if constexpr (kCached) {
    const uint4* const from = reinterpret_cast<const uint4*>(w);            // rows are whole pages, so whole vectors
    for (int j = tid; j < (len + 3) / 4; j += kSelectThreads) reinterpret_cast<uint4*>(s_w)[j] = from[j];
  }
  auto bits = [&](int j) { return kCached ? s_w[j] : w[j]; };
  const int from = a.sinks, to = len - a.recent;               // the candidates
  const int want = a.budget - a.sinks - a.recent;              // < to - from
  uint32_t prefix = 0;
  int left = want;                                             // to be found among the keys that share the prefix
  if (want > 0) {
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (int i = tid; i < kHists * 256; i += kSelectThreads) hist[i >> 8][i & 255] = 0;
      __syncthreads();
      int* const mine = hist[warp % kHists];
      for (int j = from + tid; j < to; j += kSelectThreads) {
        const uint32_t u = order_bits(bits(j));
        if (shift == 24 || (u >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&mine[(u >> shift) & 255u], 1);
      }
      __syncthreads();
      if (warp == 0) {
        // bin of the key that is `left` places from the top: lane l sums the bins 255 - 8 l .. 248 - 8 l
        int c[8], sum = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          c[e] = 0;
#pragma unroll
          for (int k = 0; k < kHists; ++k) c[e] += hist[k][255 - 8 * lane - e];
          sum += c[e];
        }
        int inc = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int x = __shfl_up_sync(0xffffffffu, inc, o);
          if (lane >= o) inc += x;
        }
        int above = inc - sum;
        if (above < left && left <= inc) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            if (above < left && left <= above + c[e]) {
              s_prefix = prefix | (uint32_t)(255 - 8 * lane - e) << shift;
              s_left = left - above;
            }
            above += c[e];
          }
        }
      }
      __syncthreads();
      prefix = s_prefix;
      left = s_left;
    }
  } else if (kCached) {
    __syncthreads();
  }
  // Ordered: a key stays if it is a sink or recent, above the border, or among the first `left` on it.  A warp owns a run of keys: it
  // counts them, learns how many stay in front of its run, and writes them.
  const int rows = (len + kSelectThreads - 1) / kSelectThreads, j0 = warp * rows * 32;
  auto look = [&](int j, bool* stay, bool* tie) {
    const uint32_t x = j < len ? bits(j) : 0u, u = order_bits(x);
    const bool ends = j < from || j >= to;
    *stay = j < len && (ends || (want > 0 && u > prefix));
    *tie = j < len && !ends && want > 0 && u == prefix;
    return x;
  };
  int n_stay = 0, n_tie = 0;
  for (int r = 0; r < rows; ++r) {
    bool stay, tie;
    look(j0 + r * 32 + lane, &stay, &tie);
    n_stay += __popc(__ballot_sync(0xffffffffu, stay));
    n_tie += __popc(__ballot_sync(0xffffffffu, tie));
  }
  if (lane == 0) {
    s_stay[warp] = n_stay;
    s_tie[warp] = n_tie;
  }
  __syncthreads();
  int ties = __reduce_add_sync(0xffffffffu, lane < warp ? s_tie[lane] : 0);
  int out = __reduce_add_sync(0xffffffffu, lane < warp ? s_stay[lane] : 0) + min(ties, left);
  const unsigned below = (1u << lane) - 1u;
  for (int r = 0; r < rows; ++r) {
    const int j = j0 + r * 32 + lane;
    bool stay, tie;
    const uint32_t x = look(j, &stay, &tie);
    const unsigned tb = __ballot_sync(0xffffffffu, tie);
    stay |= tie && ties + __popc(tb & below) < left;
    const unsigned kb = __ballot_sync(0xffffffffu, stay);
    if (stay) {
      kept[out + __popc(kb & below)] = j;
      wo[out + __popc(kb & below)] = x;
    }
    ties += __popc(tb);
    out += __popc(kb);
  }
  for (int64_t j = a.budget + tid; j < cap; j += kSelectThreads) wo[j] = 0u;
}

constexpr int kMoveThreads = 256, kMoveRounds = 4;
__global__ void __launch_bounds__(kMoveThreads) paged_move_kernel(const __grid_constant__ EvictArgs a, int vecs, int size) {
  const Pages& pg = a.pg;
  const int b = blockIdx.y / pg.Hkv, h = blockIdx.y - b * pg.Hkv;
  const int per = kMoveThreads / vecs;                         // rows a round
  const int c = threadIdx.x % vecs, lr = threadIdx.x / vecs;
  const int base = blockIdx.x * per * kMoveRounds + lr;
  grid_dep_wait();
  grid_dep_launch();
  if (lr >= per || pg.length(b) <= a.budget) return;
  const int* const kept = a.kept + ((int64_t)b * pg.Hkv + h) * a.budget;
  auto at = [&](const int64_t (&s)[3], int64_t id, int64_t row) { return (id * s[0] + h * s[1] + row * s[2]) * size + c * 16ll; };
  int j[kMoveRounds], src[kMoveRounds], dst[kMoveRounds];
  // the rounds' loads one kind after the other: survivors, page numbers, rows
#pragma unroll
  for (int e = 0; e < kMoveRounds; ++e) {
    const int r = base + e * per, page_no = r >> pg.shift;
    j[e] = r < a.budget ? ld_behind_wait(kept + r) : -1;
    dst[e] = r < a.budget && page_no < a.n_fresh ? ld_behind_wait(a.fresh + (int64_t)b * a.n_fresh + page_no) : -1;
  }
#pragma unroll
  for (int e = 0; e < kMoveRounds; ++e) src[e] = j[e] >= 0 ? pg.id(b, j[e] >> pg.shift) : -1;
  uint4 xk[kMoveRounds], xv[kMoveRounds];
#pragma unroll
  for (int e = 0; e < kMoveRounds; ++e) {
    const bool from_ok = src[e] >= 0 && src[e] < pg.n_pages, to_ok = dst[e] >= 0 && dst[e] < pg.n_pages;
    if (j[e] >= 0 && !(from_ok && to_ok)) note_condition(pg.status, kBadPage);
    if (!to_ok) j[e] = -1;
    xk[e] = xv[e] = make_uint4(0u, 0u, 0u, 0u);      // a survivor that has no page: zeros, not what the fresh page held
    if (j[e] < 0 || !from_ok) continue;
    const int64_t from = j[e] & (pg.page - 1);
    xk[e] = *reinterpret_cast<const uint4*>((const char*)a.k + at(pg.ks, src[e], from));
    xv[e] = *reinterpret_cast<const uint4*>((const char*)a.v + at(pg.vs, src[e], from));
  }
#pragma unroll
  for (int e = 0; e < kMoveRounds; ++e) {
    if (j[e] < 0) continue;
    const int64_t to = (base + e * per) & (pg.page - 1);
    *reinterpret_cast<uint4*>((char*)a.k + at(pg.ks, dst[e], to)) = xk[e];
    *reinterpret_cast<uint4*>((char*)a.v + at(pg.vs, dst[e], to)) = xv[e];
  }
}

// ---------------------------------------------------------------------------------------------- host
int log2_of(int x) {
  int s = 0;
  while ((1 << s) < x) ++s;
  return s;
}
int check_pages(Pages& pg, const void* k, const void* v, const int64_t* ks, const int64_t* vs, const int* table, const int* lengths, int B,
                int Hkv, int D, int page, int n_pages, int max_pages, int dtype) {
  LMK_CHECK_ARG(k && v && table && lengths, "paged cache: k, v, table or lengths is null");
  LMK_CHECK_ARG(ks && vs, "paged cache: stride arrays are required");
  LMK_CHECK_ARG(dtype == LMK_F32 || dtype == LMK_F16 || dtype == LMK_BF16, "paged cache: bad dtype %d", dtype);
  LMK_CHECK_ARG(B >= 1 && Hkv >= 1 && n_pages >= 1 && max_pages >= 1, "paged cache: empty problem (B=%d Hkv=%d pages=%d per sequence=%d)", B, Hkv,
                n_pages, max_pages);
  LMK_CHECK_ARG((int64_t)B * Hkv <= 65535, "paged cache: B * Hkv = %lld exceeds 65535", (long long)B * Hkv);
  LMK_CHECK_ARG(D >= 8 && D <= 128 && D % 8 == 0, "paged cache: head dim %d must be a multiple of 8 up to 128", D);
  LMK_CHECK_ARG(page >= 16 && page <= 1024 && (page & (page - 1)) == 0, "paged cache: page size %d must be a power of two from 16 to 1024", page);
  LMK_CHECK_ARG((int64_t)max_pages * page <= (1 << 30), "paged cache: %lld tokens a sequence exceed 2^30", (long long)max_pages * page);
  const int vec = 16 / dtype_size(dtype);
  LMK_CHECK_ARG((((uintptr_t)k | (uintptr_t)v) & 15) == 0, "paged cache: pages must start on a 16-byte boundary");
  for (int i = 0; i < 3; ++i)
    LMK_CHECK_ARG(ks[i] >= 0 && vs[i] >= 0 && ks[i] % vec == 0 && vs[i] % vec == 0,
                  "paged cache: page, head and row strides must be multiples of 16 bytes");
  pg.k = k; pg.v = v;
  for (int i = 0; i < 3; ++i) { pg.ks[i] = ks[i]; pg.vs[i] = vs[i]; }
  pg.table = table; pg.lengths = lengths;
  pg.B = B; pg.Hkv = Hkv; pg.D = D; pg.page = page; pg.shift = log2_of(page); pg.n_pages = n_pages; pg.max_pages = max_pages;
  return LMK_OK;
}
int status_of(Pages& pg) {             // behind all checks of arguments
  pg.status = device_status_word();
  return pg.status == nullptr ? fail(LMK_ERR_CUDA, "no device status word") : LMK_OK;
}

template <typename T, int kD, int kWarps> constexpr int attend_smem() {
  return 1024 + kAttendSmem<T, kD, kWarps> + (std::is_same<T, float>::value ? (kRowTile * kD + kWarps * kRowTile * kStep) * 4 : 0);
}
// CTAs of the attention kernel an SM holds (by shared memory: 192 KB in 16 bits at D = 128 are two CTAs)
int attend_per_sm(int dtype, int D) { return dtype == LMK_F32 ? (D <= 64 ? 2 : 1) : (D <= 64 ? 4 : 2); }
constexpr int kLeastSteps = 8;         // of a CTA: two a warp
// Tables of up to this many steps a sequence: every row is one CTA's, and nothing is to be joined (us, whole / in pieces: 32 rows of 300 keys
// 8.8 / 14.3, of 1000 15.2 / 14.5; 512 rows of 300 23.5 / 34.1).  The host knows the table's width and not the lengths: a short history in a
// wide table takes the pieces (300 keys: 8.0 us in a table of 512, 12.8 in wider ones).
constexpr int kWholeSteps = 32;

struct AttendPlan {
  int grid, rows, tiles, kD;
  bool one_piece;
  size_t acc, stat, whole, scores, bytes;
};
int attend_plan(AttendPlan* p, int B, int H, int Hkv, int T, int D, int page, int max_pages, bool weights, int dtype) {
  int n_sm = 0, rc;
  if ((rc = sm_count(&n_sm)) != LMK_OK) return rc;
  p->grid = n_sm * attend_per_sm(dtype, D);
  p->rows = H / Hkv * T;
  p->tiles = (p->rows + kRowTile - 1) / kRowTile;
  p->kD = D <= 64 ? 64 : 128;
  auto up = [](size_t x) { return (x + 255) / 256 * 256; };
  p->one_piece = (int64_t)max_pages * page <= kWholeSteps * kStep;
  const size_t pieces = p->one_piece ? 0 : (size_t)2 * p->grid * kRowTile;
  p->acc = 0;
  p->stat = up(p->acc + sizeof(float) * pieces * p->kD);
  p->whole = up(p->stat + sizeof(float2) * pieces);
  p->scores = up(p->whole + (weights ? sizeof(float2) * B * Hkv * (size_t)p->tiles * kRowTile : 0));
  p->bytes = up(p->scores + (weights ? sizeof(float) * (size_t)B * Hkv * p->rows * max_pages * page : 0));
  return LMK_OK;
}
bool attend_sizes_ok(int B, int H, int Hkv, int T) {
  return B >= 1 && Hkv >= 1 && H >= Hkv && H % Hkv == 0 && T >= 1 && T <= 1024 && (int64_t)H / Hkv * T <= 4096 && (int64_t)B * H * T < (1 << 30);
}

// a step's rows of one head: 128 bytes of features x 16 rows
int page_map(CUtensorMap* m, const Pages& pg, const void* ptr, const int64_t st[3], int dtype) {
  return tensor_map_pages(m, ptr, dtype, pg.n_pages, pg.Hkv, pg.page, pg.D, st, kStep);
}
template <typename T, int kD, int kWarps>
int launch_attend(const AttendArgs& a, int dtype, cudaStream_t st) {
  constexpr int kSmem = attend_smem<T, kD, kWarps>();
  static_assert(kSmem <= 230000, "shared memory of one SM");
  static std::atomic<bool> ready[64];
  int dev = 0;
  LMK_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64) return fail(LMK_ERR_UNSUPPORTED, "device index %d out of range", dev);
  if (!ready[dev].load(std::memory_order_acquire)) {
    LMK_CUDA(cudaFuncSetAttribute(paged_attend_kernel<T, kD, kWarps>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem));
    ready[dev].store(true, std::memory_order_release);
  }
  CUtensorMap tk, tv;
  int rc = page_map(&tk, a.pg, a.pg.k, a.pg.ks, dtype);
  if (rc == LMK_OK) rc = page_map(&tv, a.pg, a.pg.v, a.pg.vs, dtype);
  if (rc != LMK_OK) return rc;
  const int64_t items = (int64_t)a.pg.B * a.pg.Hkv * a.tiles;
  const unsigned grid = a.one_piece && items < a.grid ? (unsigned)items : (unsigned)a.grid;
  LMK_CUDA(launch_overlapped(paged_attend_kernel<T, kD, kWarps>, dim3(grid), dim3(kWarps * 32), kSmem, st, tk, tv, a));
  const int64_t cap = (int64_t)a.pg.max_pages << a.pg.shift;
  const int64_t joins = !a.one_piece ? items * (kD / 32) : 0;
  const int64_t runs = a.weights != nullptr ? (cap + kRunKeys - 1) / kRunKeys * a.pg.B * a.pg.Hkv : 0;
  if (joins + runs > INT32_MAX) return fail(LMK_ERR_UNSUPPORTED, "paged attention: too many rows and keys for one call");
  if (joins + runs > 0)
    LMK_CUDA(launch_overlapped(paged_finish_kernel<T, kD>, dim3((unsigned)(joins + runs)), dim3(kJoinThreads), sizeof(float2) * a.rows, st, a, (int)joins));
  return LMK_OK;
}
// (8 warps of fp32 rows of 128 features would not fit an SM's shared memory)
template <typename T>
int dispatch_attend(const AttendArgs& a, int kD, int dtype, cudaStream_t st) {
  constexpr int kMore = std::is_same<T, float>::value ? 4 : 8;
  int n_sm = 0;
  const int rc = sm_count(&n_sm);
  if (rc != LMK_OK) return rc;
  const bool few = a.one_piece && (int64_t)a.pg.B * a.pg.Hkv * a.tiles <= n_sm;
  if (kD == 64) return few ? launch_attend<T, 64, 8>(a, dtype, st) : launch_attend<T, 64, 4>(a, dtype, st);
  return few ? launch_attend<T, 128, kMore>(a, dtype, st) : launch_attend<T, 128, 4>(a, dtype, st);
}

}  // namespace
}  // namespace lmk

using namespace lmk;

extern "C" size_t lmk_paged_attend_workspace(int B, int H, int Hkv, int T, int D, int page, int max_pages, int weights, int dtype) {
  AttendPlan p;
  if (!attend_sizes_ok(B, H, Hkv, T) || attend_plan(&p, B, H, Hkv, T, D, page, max_pages, weights != 0, dtype) != LMK_OK) return 0;
  return p.bytes;
}

extern "C" int lmk_paged_attend(const void* q, const int64_t q_strides[3], const void* k_pages, const void* v_pages,
                                const int64_t k_strides[3], const int64_t v_strides[3], const int* table, const int* lengths, void* o,
                                float* weights, float decay, void* workspace, size_t workspace_bytes, int B, int H, int Hkv, int T, int D,
                                int page, int n_pages, int max_pages, int window, int sinks, float sm_scale, int dtype, void* stream) {
  AttendArgs a = {};
  int rc = check_pages(a.pg, k_pages, v_pages, k_strides, v_strides, table, lengths, B, Hkv, D, page, n_pages, max_pages, dtype);
  if (rc != LMK_OK) return rc;
  LMK_CHECK_ARG(q && o && q_strides, "paged attention: q or o is null");
  LMK_CHECK_ARG(H >= Hkv && H % Hkv == 0, "paged attention: %d query heads are not a multiple of %d key heads", H, Hkv);
  LMK_CHECK_ARG(attend_sizes_ok(B, H, Hkv, T), "paged attention: T=%d tokens of %d heads a key head are too many (up to 1024 tokens, 4096 rows)", T, H / Hkv);
  LMK_CHECK_ARG(window >= 0 && sinks >= 0, "paged attention: window=%d and sinks=%d must not be negative", window, sinks);
  // the last piece may end behind the line, by less than one step a CTA
  LMK_CHECK_ARG((int64_t)B * Hkv * ((H / Hkv * T + kRowTile - 1) / kRowTile) * ((int64_t)max_pages * page / kStep) <= INT32_MAX - 65536,
                "paged attention: %d sequences of up to %lld tokens and %d key heads are too many for one call", B, (long long)max_pages * page, Hkv);
  LMK_CHECK_ARG((n_pages == 1 || (k_strides[0] > 0 && v_strides[0] > 0)) && (Hkv == 1 || (k_strides[1] > 0 && v_strides[1] > 0)) &&
                    k_strides[2] >= D && v_strides[2] >= D, "paged attention: pages must not be broadcast, nor their rows overlap");
  LMK_CHECK_ARG(isfinite(sm_scale) && isfinite(decay), "paged attention: scale and decay must be finite");
  LMK_CHECK_ARG(((uintptr_t)weights & 15) == 0, "paged attention: weights must start on a 16-byte boundary");
  const int pair = 4 / dtype_size(dtype);
  LMK_CHECK_ARG(((uintptr_t)q & 3) == 0 && q_strides[0] % pair == 0 && q_strides[1] % pair == 0 && q_strides[2] % pair == 0,
                "paged attention: q must lie on 4-byte boundaries");
  LMK_CHECK_ARG(((uintptr_t)o & 15) == 0, "paged attention: o must start on a 16-byte boundary");
  AttendPlan p;
  if ((rc = attend_plan(&p, B, H, Hkv, T, D, page, max_pages, weights != nullptr, dtype)) != LMK_OK) return rc;
  if (p.bytes > 0 && (workspace == nullptr || workspace_bytes < p.bytes || ((uintptr_t)workspace & 255) != 0))
    return fail(LMK_ERR_WORKSPACE, "paged attention: workspace of %zu bytes on a 256-byte boundary needed", p.bytes);
  if ((rc = status_of(a.pg)) != LMK_OK) return rc;
  a.q = q; a.o = o;
  for (int i = 0; i < 3; ++i) a.qs[i] = q_strides[i];
  a.weights = weights; a.decay = decay;
  char* ws = static_cast<char*>(workspace);
  a.acc = reinterpret_cast<float*>(ws + p.acc);
  a.stat = reinterpret_cast<float2*>(ws + p.stat);
  a.whole = reinterpret_cast<float2*>(ws + p.whole);
  a.scores = reinterpret_cast<float*>(ws + p.scores);
  a.H = H; a.T = T; a.G = H / Hkv; a.rows = p.rows; a.tiles = p.tiles; a.window = window; a.sinks = window > 0 ? sinks : 0; a.grid = p.grid;
  a.least = kLeastSteps;
  a.one_piece = p.one_piece;
  a.scale_log2 = sm_scale * kLog2e;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == LMK_BF16) return dispatch_attend<__nv_bfloat16>(a, p.kD, dtype, st);
  if (dtype == LMK_F16) return dispatch_attend<__half>(a, p.kD, dtype, st);
  return dispatch_attend<float>(a, p.kD, dtype, st);
}

extern "C" int lmk_paged_append(const void* k_new, const void* v_new, const int64_t k_new_strides[3], const int64_t v_new_strides[3],
                                void* k_pages, void* v_pages, const int64_t k_strides[3], const int64_t v_strides[3], const int* table,
                                int* lengths, const int* counts, float* weights, int B, int Hkv, int T, int D, int page, int n_pages,
                                int max_pages, int dtype, void* stream) {
  AppendArgs a = {};
  int rc = check_pages(a.pg, k_pages, v_pages, k_strides, v_strides, table, lengths, B, Hkv, D, page, n_pages, max_pages, dtype);
  if (rc != LMK_OK) return rc;
  LMK_CHECK_ARG(k_new && v_new && k_new_strides && v_new_strides, "paged append: k or v is null");
  LMK_CHECK_ARG(T >= 1 && T <= (1 << 30), "paged append: no rows (T=%d)", T);
  const int size = dtype_size(dtype), vec = 16 / size;
  LMK_CHECK_ARG((((uintptr_t)k_new | (uintptr_t)v_new) & 15) == 0, "paged append: rows must start on a 16-byte boundary");
  for (int i = 0; i < 3; ++i)
    LMK_CHECK_ARG(k_new_strides[i] % vec == 0 && v_new_strides[i] % vec == 0, "paged append: strides must be multiples of 16 bytes");
  if ((rc = status_of(a.pg)) != LMK_OK) return rc;
  a.k_new = k_new; a.v_new = v_new;
  for (int i = 0; i < 3; ++i) { a.kns[i] = k_new_strides[i]; a.vns[i] = v_new_strides[i]; }
  a.k = k_pages; a.v = v_pages; a.lengths = lengths; a.counts = counts; a.weights = weights; a.T = T;
  // one CTA a sequence moves its length on by itself; above about 2000 vectors it would be the slower way
  const int64_t vecs_all = (int64_t)T * Hkv * (D / vec);
  a.chunks = vecs_all <= 2048 ? 1 : (int)((vecs_all + 2047) / 2048 < 4096 ? (vecs_all + 2047) / 2048 : 4096);
  if (a.chunks > T) a.chunks = T;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  LMK_CUDA(launch_overlapped(paged_append_kernel<uint4>, dim3(a.chunks, B), dim3(256), 0, st, a, D / vec, size));
  if (a.chunks > 1) LMK_CUDA(launch_overlapped(paged_advance_kernel, dim3((B + 255) / 256), dim3(256), 0, st, a));
  return LMK_OK;
}

extern "C" int lmk_paged_evict(void* k_pages, void* v_pages, const int64_t k_strides[3], const int64_t v_strides[3], const int* table,
                               const int* lengths, const float* weights, const int* fresh, int n_fresh, int* table_out, int* lengths_out,
                               float* weights_out, int* kept, int B, int Hkv, int D, int page, int n_pages, int max_pages, int budget,
                               int recent, int sinks, int dtype, void* stream) {
  EvictArgs a = {};
  int rc = check_pages(a.pg, k_pages, v_pages, k_strides, v_strides, table, lengths, B, Hkv, D, page, n_pages, max_pages, dtype);
  if (rc != LMK_OK) return rc;
  LMK_CHECK_ARG((((uintptr_t)weights | (uintptr_t)weights_out) & 15) == 0, "paged evict: weights must start on a 16-byte boundary");
  LMK_CHECK_ARG(weights && fresh && table_out && lengths_out && weights_out && kept, "paged evict: an array is null");
  LMK_CHECK_ARG(table_out != table && lengths_out != lengths && weights_out != weights, "paged evict: outputs must not be the inputs");
  LMK_CHECK_ARG(budget >= 1 && recent >= 0 && sinks >= 0 && (int64_t)recent + sinks <= budget,
                "paged evict: budget %d must hold %d recent tokens and %d sinks", budget, recent, sinks);
  LMK_CHECK_ARG((int64_t)n_fresh * page >= budget && n_fresh <= max_pages, "paged evict: %d fresh pages of %d for %d tokens (at most %d pages a sequence)",
                n_fresh, page, budget, max_pages);
  if ((rc = status_of(a.pg)) != LMK_OK) return rc;
  a.k = k_pages; a.v = v_pages; a.weights = weights; a.fresh = fresh; a.n_fresh = n_fresh; a.budget = budget; a.recent = recent; a.sinks = sinks;
  a.table_out = table_out; a.lengths_out = lengths_out; a.weights_out = weights_out; a.kept = kept;
  const int size = dtype_size(dtype), vecs = D * size / 16;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if ((int64_t)max_pages * page <= kCachedKeys) {
    static std::atomic<bool> ready[64];
    int dev = 0;
    LMK_CUDA(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64) return fail(LMK_ERR_UNSUPPORTED, "device index %d out of range", dev);
    if (!ready[dev].load(std::memory_order_acquire)) {
      LMK_CUDA(cudaFuncSetAttribute(paged_select_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, kCachedKeys * 4));
      ready[dev].store(true, std::memory_order_release);
    }
    LMK_CUDA(launch_overlapped(paged_select_kernel<true>, dim3(B * Hkv), dim3(kSelectThreads), (size_t)max_pages * page * 4, st, a));
  } else {
    LMK_CUDA(launch_overlapped(paged_select_kernel<false>, dim3(B * Hkv), dim3(kSelectThreads), 0, st, a));
  }
  const int rows = (kMoveThreads / vecs) * kMoveRounds;
  LMK_CUDA(launch_overlapped(paged_move_kernel, dim3((budget + rows - 1) / rows, B * Hkv), dim3(kMoveThreads), 0, st, a, vecs, size));
  return LMK_OK;
}
