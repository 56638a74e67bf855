// Paged key-value cache: append, attention of a sequence's newest tokens over its pages, eviction by accumulated attention weight.
//
// Pages are [n_pages, Hkv, page, D] (any page, head and row strides); table [B, max_pages] names a sequence's pages in order, lengths [B]
// say how many of their rows are tokens.  Nothing here trusts either: lengths are held between 0 and the table's capacity, a table
// entry outside of the pool is never followed (its keys count as hidden, and the device status word says 601).
//
// Attention.  Query t of T stands at position p = length - T + t and sees key j if j <= p and (no window, p - j < window or j < sinks).
//   o = sum_j e^{s_j - m} v_j / sum_j e^{s_j - m}, m = max_j s_j, s_j = scale q . k_j  over the visible j; 0 where nothing is visible.
// Every visible row of K and V is read once, 512 bytes a key and head at D = 128 in 16 bits against 4 D multiply-adds a query row: bound
// by HBM.  What decides is how evenly the rows are dealt out and how many loads are in flight.
//   - The work of all sequences is one line of steps of 16 keys (sequence, key head, tile of 16 query rows, step).  Every CTA takes the same
//     length of it, so neither short sequences nor a large capacity leave SMs idle, whatever the lengths are; they are read on the
//     device, so a captured graph serves them as they grow.  A piece that holds all of its keys is written out at once; pieces of a
//     longer row leave their maximum, sum and unnormalised output, which a second kernel joins.
//   - A warp streams its own steps (every fourth of the CTA's) through its own ring in shared memory with cp.async: no barrier of the CTA in
//     the loop.  Rows that nobody sees are filled with zeros instead of loaded, so what they hold does not matter.
//   - The G T query rows of a key head are the 16 rows of an mma.sync tile (fp32: FMAs), so K and V are read once for all of them.
// Weights (for eviction): the scores are kept, 4 bytes a key and query row, and the second kernel, which knows every row's maximum and
// sum, adds e^{s - m} / l of a group's rows to the key's weight.  One thread adds up one key: no atomics, bit-reproducible.
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
constexpr int kWarps = 4;
constexpr int kStages = 3;
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kBadPage = 601, kFull = 602;

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

__device__ __forceinline__ void note(int* status, int what) { atomicCAS(status, 0, what); }

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
  float scale_log2;
};

// Where a piece of work lies: all sequences' steps in one line.
struct Line {
  int64_t total;                       // steps of all items
  int64_t piece;                       // steps a CTA takes
};
// Sum of f(b) over all sequences, and over those before `b` or up to the one that holds step `at`.  Whole warp.
struct Found { int b; int64_t before; };

template <typename F>
__device__ __forceinline__ int64_t warp_total(int B, F f) {
  int64_t sum = 0;
  for (int b = threadIdx.x & 31; b < B; b += 32) sum += f(b);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  return sum;
}
template <typename F>
__device__ __forceinline__ Found warp_find(int B, int64_t at, F f) {      // the last b whose steps begin at or before `at`
  const int lane = threadIdx.x & 31;
  int64_t before = 0;
  Found r{B, 0};
  for (int b0 = 0; b0 < B; b0 += 32) {
    const int64_t n = b0 + lane < B ? f(b0 + lane) : 0;
    int64_t inc = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t v = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += v;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, n > 0 && before + inc > at);
    if (hit) {
      const int src = __ffs((int)hit) - 1;
      r.b = b0 + src;
      r.before = __shfl_sync(0xffffffffu, before + inc - n, src);
      return r;
    }
    before += __shfl_sync(0xffffffffu, inc, 31);
  }
  r.before = before;
  return r;
}
template <typename F>
__device__ __forceinline__ int64_t warp_before(int B, int b, F f) {
  return warp_total(b < B ? b : B, f);
}

__device__ __forceinline__ Line line_of(const AttendArgs& a, int64_t total) {
  Line l;
  l.total = total;
  l.piece = max((total + a.grid - 1) / a.grid, (int64_t)a.least);
  return l;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool take) {
  const int bytes = take ? 16 : 0;     // 0: filled with zeros, src is not read
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

template <typename T, int kD> constexpr int kRowBytes = kD * (int)sizeof(T);
template <typename T, int kD> constexpr int kStageBytes = 2 * kStep * kRowBytes<T, kD>;      // K, then V
template <typename T, int kD> constexpr int kAttendSmem = kWarps * kStages * kStageBytes<T, kD>;

// byte offset of 16-byte chunk c of row r: chunks change places within a row so that eight rows' equal chunks lie in different banks
template <typename T, int kD>
__device__ __forceinline__ uint32_t chunk_at(int r, int c) { return (uint32_t)(r * kRowBytes<T, kD> + ((c ^ (r & 7)) << 4)); }

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
    base[e] = r < a.rows ? reinterpret_cast<const T*>(a.q) + b * a.qs[0] + (int64_t)(h * a.G + r / a.T) * a.qs[1] + (int64_t)(r % a.T) * a.qs[2]
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
  float s[2][4] = {};
  const int kr = (lane >> 4) * 8 + (lane & 7), kc = (lane >> 3) & 1;
#pragma unroll
  for (int kk = 0; kk < kD / 16; ++kk) {
    uint32_t f[4];
    ldmatrix_x4(f, stage + chunk_at<T, kD>(kr, kk * 2 + kc));
    mma16<T>(s[0], w.q[kk][0], w.q[kk][1], w.q[kk][2], w.q[kk][3], f[0], f[1]);
    mma16<T>(s[1], w.q[kk][0], w.q[kk][1], w.q[kk][2], w.q[kk][3], f[2], f[3]);
  }
  // element (n, e): row g + 8 (e / 2), key 8 n + 2 t + e % 2
  float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
  for (int n = 0; n < 2; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float x = s[n][e] * scale_log2;
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
  const uint8_t* vs = stage + kStep * kRowBytes<T, kD>;
  const int vr = ((lane >> 3) & 1) * 8 + (lane & 7), vc = lane >> 4;
#pragma unroll
  for (int n = 0; n < kD / 16; ++n) {
    uint32_t f[4];
    ldmatrix_x4_trans(f, vs + chunk_at<T, kD>(vr, n * 2 + vc));
    mma16<T>(w.o[2 * n], p0, p1, p2, p3, f[0], f[1]);
    mma16<T>(w.o[2 * n + 1], p0, p1, p2, p3, f[2], f[3]);
  }
}

// A warp's result of a piece in its own part of shared memory: [16][kD] floats, then 16 maxima and 16 sums
template <int kD> constexpr int kResultFloats = kRowTile * kD + 2 * kRowTile;
template <typename T, int kD>
__device__ __forceinline__ void leave_result(Rows16<T, kD>& w, float* to) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    w.l[e] += __shfl_xor_sync(0xffffffffu, w.l[e], 1);
    w.l[e] += __shfl_xor_sync(0xffffffffu, w.l[e], 2);
    if (t4 == 0) {
      to[kRowTile * kD + g + 8 * e] = w.m[e];
      to[kRowTile * kD + kRowTile + g + 8 * e] = w.l[e];
    }
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

template <typename T, int kD>
__global__ void __launch_bounds__(kWarps * 32) paged_attend_kernel(const __grid_constant__ AttendArgs a) {
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ int64_t s_total;
  __shared__ Found s_found;
  constexpr bool kF32 = std::is_same<T, float>::value;
  grid_dep_wait();
  grid_dep_launch();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const Pages& pg = a.pg;
  const int per_seq = pg.Hkv * a.tiles;
  auto steps_of = [&](int b) { return (int64_t)per_seq * span_of(pg.length(b), a.T, a.window, a.sinks).steps; };
  if (warp == 0) {
    const int64_t total = warp_total(pg.B, steps_of);
    const Line line = line_of(a, total);
    const Found f = warp_find(pg.B, blockIdx.x * line.piece, steps_of);
    if (lane == 0) {
      s_total = total;
      s_found = f;
    }
  }
  // sequences without keys: their outputs are zeros (a share of the sequences for every CTA)
  for (int b = blockIdx.x; b < pg.B; b += a.grid)
    if (pg.length(b) == 0)
      for (int64_t i = tid; i < (int64_t)a.H * a.T * pg.D; i += kWarps * 32) reinterpret_cast<T*>(a.o)[b * (int64_t)a.H * a.T * pg.D + i] = from_f32<T>(0.f);
  __syncthreads();
  const Line line = line_of(a, s_total);
  const int64_t begin = blockIdx.x * line.piece, end = min(begin + line.piece, line.total);
  if (begin >= end) return;
  int b = s_found.b;
  int64_t before = s_found.before;
  Span sp = span_of(pg.length(b), a.T, a.window, a.sinks);
  uint8_t* ring = smem + warp * kStages * kStageBytes<T, kD>;
  const uint32_t ring_at = smem_u32(ring);
  float* const result = reinterpret_cast<float*>(ring);
  static_assert(kResultFloats<kD> * 4 <= kStages * kStageBytes<T, kD>, "a warp's result fits its ring");

  for (int64_t at = begin; at < end;) {
    while (at >= before + (int64_t)per_seq * sp.steps) {      // the next sequence that has keys
      before += (int64_t)per_seq * sp.steps;
      ++b;
      sp = span_of(pg.length(b), a.T, a.window, a.sinks);
    }
    const int item = (int)((at - before) / sp.steps), step0 = (int)((at - before) - (int64_t)item * sp.steps);
    const int h = item / a.tiles, row0 = (item - h * a.tiles) * kRowTile;
    const int count = (int)min((int64_t)(sp.steps - step0), end - at);
    const int mine = (count - warp + kWarps - 1) / kWarps;     // steps step0 + warp, + kWarps, ...
    const int p0 = sp.len - a.T;                               // position of the first token's queries
    const int lo_seen = a.window > 0 && p0 >= a.window ? p0 - a.window + 1 : 0;

    auto page_id = [&](int i) { return i < mine ? pg.id(b, sp.key(step0 + warp + i * kWarps) >> pg.shift) : 0; };
    auto issue = [&](int i, int id) {
      if (i < mine) {
        const int key0 = sp.key(step0 + warp + i * kWarps);
        const bool ok = id >= 0 && id < pg.n_pages;
        if (!ok && lane == 0) note(pg.status, kBadPage);
        const int row = key0 & (pg.page - 1);
        const T* kp = reinterpret_cast<const T*>(pg.k) + (ok ? (int64_t)id * pg.ks[0] + h * pg.ks[1] + (int64_t)row * pg.ks[2] : 0);
        const T* vp = reinterpret_cast<const T*>(pg.v) + (ok ? (int64_t)id * pg.vs[0] + h * pg.vs[1] + (int64_t)row * pg.vs[2] : 0);
        const uint32_t to = ring_at + (uint32_t)(i % kStages) * kStageBytes<T, kD>;
        constexpr int kChunks = kRowBytes<T, kD> / 16, kVec = 16 / (int)sizeof(T);
#pragma unroll
        for (int e = 0; e < kStep * kChunks / 32; ++e) {
          const int r = (e * 32 + lane) / kChunks, c = (e * 32 + lane) % kChunks;
          const int key = key0 + r;
          const bool take = ok && key < sp.len && (key >= lo_seen || key < a.sinks) && c * kVec < pg.D;
          const int64_t off_k = take ? (int64_t)r * pg.ks[2] + c * kVec : 0, off_v = take ? (int64_t)r * pg.vs[2] + c * kVec : 0;
          cp_async16(to + chunk_at<T, kD>(r, c), kp + off_k, take);
          cp_async16(to + kStep * kRowBytes<T, kD> + chunk_at<T, kD>(r, c), vp + off_v, take);
        }
      }
      cp_async_commit();
    };

    // ids run ahead of the loads that need them
    int ids[kStages];
#pragma unroll
    for (int i = 0; i < kStages; ++i) ids[i] = page_id(i);
    unsigned bad = 0;                                          // bit i % kStages: the step in that stage has no page
    auto mark = [&](int i, int id) {
      const unsigned bit = 1u << (i % kStages);
      bad = (id >= 0 && id < pg.n_pages) ? bad & ~bit : bad | bit;
    };
    __syncwarp();
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) {
      issue(i, ids[i]);
      mark(i, ids[i]);
    }
    int next = ids[kStages - 1];
    const int64_t score_row = ((int64_t)b * pg.Hkv + h) * a.rows;
    const int64_t cap = (int64_t)pg.max_pages << pg.shift;

    if constexpr (!kF32) {
      Rows16<T, kD> w;
      load_queries<T, kD>(w, a, b, h, row0);
      int pos[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = row0 + (lane >> 2) + 8 * e;
        pos[e] = r < a.rows ? p0 + r % a.T : -1;
      }
      for (int i = 0; i < mine; ++i) {
        cp_async_wait<kStages - 2>();
        __syncwarp();
        issue(i + kStages - 1, next);
        const int id = next;
        next = page_id(i + kStages);
        const int key0 = sp.key(step0 + warp + i * kWarps);
        const bool no_page = bad >> (i % kStages) & 1u;
        mark(i + kStages - 1, id);
        // every row that exists sees all 16 keys (the last row of the window is the one that has gone furthest)
        const bool all = !no_page && p0 >= 0 && key0 + kStep - 1 <= p0 && (a.window == 0 || p0 + a.T - 1 - key0 < a.window);
        take_step<T, kD>(w, ring + (i % kStages) * kStageBytes<T, kD>, a.scale_log2, all,
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
      }
      cp_async_wait<0>();
      __syncwarp();
      leave_result<T, kD>(w, result);
    } else {
      // fp32 on the FMA units.  Scores: lane = (key, half of the features); outputs: lane = kD / 32 features of every row.
      Rows32<kD> w;
      const int n_rows = min(kRowTile, a.rows - row0);
      float* const qs = reinterpret_cast<float*>(smem + kAttendSmem<T, kD>);         // [16][kD], the CTA's query rows
      float* const ps = qs + kRowTile * kD + warp * kRowTile * kStep;                // [16][16], the warp's weights
      __syncthreads();                                                               // the piece before is done with the queries
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
      for (int i = 0; i < mine; ++i) {
        cp_async_wait<kStages - 2>();
        __syncwarp();
        issue(i + kStages - 1, next);
        const int id = next;
        next = page_id(i + kStages);
        const int key0 = sp.key(step0 + warp + i * kWarps);
        const bool no_page = bad >> (i % kStages) & 1u;
        mark(i + kStages - 1, id);
        const uint8_t* stage = ring + (i % kStages) * kStageBytes<T, kD>;
        const int j = lane & 15, half = lane >> 4;
        float s[kRowTile];
#pragma unroll
        for (int r = 0; r < kRowTile; ++r) s[r] = 0.f;
        for (int c = 0; c < kD / 8; ++c) {                   // the half's 16-byte chunks
          const int chunk = half * (kD / 8) + c;
          const float4 x = *reinterpret_cast<const float4*>(stage + chunk_at<T, kD>(j, chunk));
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
          const int pos = p0 + (row0 + r) % a.T, key = key0 + j;
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
        const uint8_t* vs = stage + kStep * kRowBytes<T, kD>;
        for (int k = 0; k < kStep; ++k) {
          float v[kD / 32];
#pragma unroll
          for (int c = 0; c < kD / 32; ++c) {
            const int f = lane * (kD / 32) + c;
            v[c] = *reinterpret_cast<const float*>(vs + chunk_at<T, kD>(k, f / 4) + (f % 4) * 4);
          }
#pragma unroll
          for (int r = 0; r < kRowTile; ++r) {
            if (r >= n_rows) break;
            const float p = ps[r * kStep + k];
#pragma unroll
            for (int c = 0; c < kD / 32; ++c) w.o[r][c] = fmaf(p, v[c], w.o[r][c]);
          }
        }
        __syncwarp();
      }
      cp_async_wait<0>();
      __syncwarp();
#pragma unroll
      for (int r = 0; r < kRowTile; ++r) {
        const float l = warp_sum(w.l[r]);
        if (lane == 0) {
          result[kRowTile * kD + r] = w.m[r];
          result[kRowTile * kD + kRowTile + r] = l;
        }
#pragma unroll
        for (int c = 0; c < kD / 32; ++c) result[r * kD + lane * (kD / 32) + c] = w.o[r][c];
      }
    }

    // the four warps' results, joined: 8 threads a row
    __syncthreads();
    {
      const int r = tid >> 3, part = tid & 7;
      const float* res[kWarps];
      float mx = -INFINITY, l = 0.f, f[kWarps];
#pragma unroll
      for (int k = 0; k < kWarps; ++k) {
        res[k] = reinterpret_cast<const float*>(smem + k * kStages * kStageBytes<T, kD>);
        const float mk = res[k][kRowTile * kD + r];
        mx = max3_nan(mx, mk, mk);
      }
      const float shift = mx == -INFINITY ? 0.f : mx;
#pragma unroll
      for (int k = 0; k < kWarps; ++k) {
        f[k] = ex2(res[k][kRowTile * kD + r] - shift);
        l += f[k] * res[k][kRowTile * kD + kRowTile + r];
      }
      const bool exists = row0 + r < a.rows, all = count == sp.steps;
      const int64_t slot = 2 * (int64_t)blockIdx.x + (step0 > 0 ? 0 : 1);
      const float inv = l == 0.f ? 0.f : 1.f / l;
      T* const orow = reinterpret_cast<T*>(a.o) + (((int64_t)b * a.H + h * a.G + (row0 + r) / a.T) * a.T + (row0 + r) % a.T) * pg.D;
      float* const arow = a.acc + (slot * kRowTile + r) * kD;
#pragma unroll
      for (int c = 0; c < kD / 32; ++c) {
        const int col = c * 32 + part * 4;
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
          uint2 x = make_uint2(pack16<T>(sum.x * inv, sum.y * inv), pack16<T>(sum.z * inv, sum.w * inv));
          *reinterpret_cast<uint2*>(orow + col) = x;
        }
      }
      if (exists && part == 0) {
        if (!all) a.stat[slot * kRowTile + r] = make_float2(mx, l);
        else if (a.weights != nullptr) a.whole[(((int64_t)b * pg.Hkv + h) * a.tiles + row0 / kRowTile) * kRowTile + r] = make_float2(mx, l);
      }
    }
    __syncthreads();
    at += count;
  }
}

// Joins the pieces of rows that several CTAs worked on; with weights: adds every key's share of its group's rows.
// Grid (items, slices): slice s joins the features [32 s, 32 s + 32) and takes every gridDim.y-th run of 1024 keys.
constexpr int kJoinThreads = 256;
template <typename T, int kD>
__global__ void __launch_bounds__(kJoinThreads) paged_join_kernel(const __grid_constant__ AttendArgs a) {
  __shared__ int64_t s_total, s_before;
  __shared__ float2 s_stat[kRowTile];
  grid_dep_wait();
  grid_dep_launch();
  const Pages& pg = a.pg;
  const int tid = threadIdx.x;
  const int per_seq = pg.Hkv * a.tiles;
  const int b = blockIdx.x / per_seq, item = blockIdx.x - b * per_seq;
  auto steps_of = [&](int i) { return (int64_t)per_seq * span_of(pg.length(i), a.T, a.window, a.sinks).steps; };
  if (tid < 32) {
    const int64_t total = warp_total(pg.B, steps_of), before = warp_before(pg.B, b, steps_of);
    if (tid == 0) {
      s_total = total;
      s_before = before;
    }
  }
  __syncthreads();
  const Span sp = span_of(pg.length(b), a.T, a.window, a.sinks);
  if (sp.steps == 0) return;
  const Line line = line_of(a, s_total);
  const int64_t start = s_before + (int64_t)item * sp.steps;
  const int c0 = (int)(start / line.piece), c1 = (int)((start + sp.steps - 1) / line.piece);
  const int h = item / a.tiles, row0 = (item - h * a.tiles) * kRowTile;
  const int n_rows = min(kRowTile, a.rows - row0);
  auto slot_of = [&](int c) { return 2 * (int64_t)c + (c == c0 ? 1 : 0); };
  if (c1 > c0) {
    const int r = tid >> 4, part = tid & 15;         // 16 threads a row
    float mx = -INFINITY, l = 0.f;
    if (r < n_rows) {
      for (int c = c0 + part; c <= c1; c += 16) {
        const float m = a.stat[slot_of(c) * kRowTile + r].x;
        mx = max3_nan(mx, m, m);
      }
    }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) {
      const float m = __shfl_xor_sync(0xffffffffu, mx, o);
      mx = max3_nan(mx, m, m);
    }
    const float shift = mx == -INFINITY ? 0.f : mx;
    if (r < n_rows)
      for (int c = c0 + part; c <= c1; c += 16) {
        const float2 x = a.stat[slot_of(c) * kRowTile + r];
        l += ex2(x.x - shift) * x.y;
      }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    if (part == 0) s_stat[r] = make_float2(mx, l);
    const int col = blockIdx.y * 32 + part * 2;
    if (r < n_rows && blockIdx.y < kD / 32 && col < pg.D) {
      const float inv = l == 0.f ? 0.f : 1.f / l;
      float2 sum = make_float2(0.f, 0.f);
      for (int c = c0; c <= c1; ++c) {
        const float f = ex2(a.stat[slot_of(c) * kRowTile + r].x - shift);
        const float2 x = *reinterpret_cast<const float2*>(a.acc + (slot_of(c) * kRowTile + r) * kD + col);
        sum.x = fmaf(f, x.x, sum.x);
        sum.y = fmaf(f, x.y, sum.y);
      }
      T* const to = reinterpret_cast<T*>(a.o) + (((int64_t)b * a.H + h * a.G + (row0 + r) / a.T) * a.T + (row0 + r) % a.T) * pg.D + col;
      to[0] = from_f32<T>(sum.x * inv);
      to[1] = from_f32<T>(sum.y * inv);
    }
  }
}

// weights[b, h, j] = decay weights[b, h, j] + sum over the rows of the group of e^{s_j - m} / l, for all j < length
template <typename T>
__global__ void __launch_bounds__(kJoinThreads) paged_weights_kernel(const __grid_constant__ AttendArgs a) {
  extern __shared__ float2 s_rows[];                 // (maximum, 1 / sum) of the group's rows
  __shared__ int64_t s_total, s_before;
  grid_dep_wait();
  grid_dep_launch();
  const Pages& pg = a.pg;
  const int tid = threadIdx.x;
  const int b = blockIdx.y / pg.Hkv, h = blockIdx.y - b * pg.Hkv;
  const int per_seq = pg.Hkv * a.tiles;
  auto steps_of = [&](int i) { return (int64_t)per_seq * span_of(pg.length(i), a.T, a.window, a.sinks).steps; };
  const int len = pg.length(b);
  if ((int64_t)blockIdx.x * kJoinThreads * 4 >= len) return;
  if (tid < 32) {
    const int64_t total = warp_total(pg.B, steps_of), before = warp_before(pg.B, b, steps_of);
    if (tid == 0) {
      s_total = total;
      s_before = before;
    }
  }
  __syncthreads();
  const Span sp = span_of(len, a.T, a.window, a.sinks);
  const Line line = line_of(a, s_total);
  for (int r = tid; r < a.rows; r += kJoinThreads) {
    const int tile = r / kRowTile, rr = r - tile * kRowTile;
    const int64_t start = s_before + (int64_t)(h * a.tiles + tile) * sp.steps;
    const int c0 = (int)(start / line.piece), c1 = (int)((start + sp.steps - 1) / line.piece);
    float2 x;
    if (c0 == c1) {
      x = a.whole[(((int64_t)b * pg.Hkv + h) * a.tiles + tile) * kRowTile + rr];
    } else {
      x = make_float2(-INFINITY, 0.f);
      for (int c = c0; c <= c1; ++c) {
        const float2 y = a.stat[(2 * (int64_t)c + (c == c0 ? 1 : 0)) * kRowTile + rr];
        const float m = max3_nan(x.x, y.x, y.x), shift = m == -INFINITY ? 0.f : m;
        x.y = x.y * ex2(x.x - shift) + y.y * ex2(y.x - shift);
        x.x = m;
      }
    }
    s_rows[r] = make_float2(x.x == -INFINITY ? 0.f : x.x, x.y == 0.f ? 0.f : 1.f / x.y);
  }
  __syncthreads();
  const int64_t cap = (int64_t)pg.max_pages << pg.shift;
  const float* const scores = a.scores + ((int64_t)b * pg.Hkv + h) * a.rows * cap;
  float* const weights = a.weights + ((int64_t)b * pg.Hkv + h) * cap;
  for (int e = 0; e < 4; ++e) {
    const int j = (blockIdx.x * 4 + e) * kJoinThreads + tid;
    if (j >= len) break;
    float w = a.decay == 0.f ? 0.f : a.decay * weights[j];         // decay 0: whatever stood there is not read
    if (j < sp.first * kStep || j >= sp.lo) {
      float sum = 0.f;
      for (int r = 0; r < a.rows; ++r) sum += ex2(scores[r * cap + j] - s_rows[r].x) * s_rows[r].y;
      w += sum;
    }
    weights[j] = w;
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
  if (want > room && threadIdx.x == 0) note(a.pg.status, kFull);
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
    if (id < 0 || id >= pg.n_pages) {
      note(pg.status, kBadPage);
      continue;
    }
    const int64_t row = at & (pg.page - 1);
    auto bytes = [&](int64_t elements) { return elements * size; };
    const V xk = *reinterpret_cast<const V*>((const char*)a.k_new + bytes(b * a.kns[0] + h * a.kns[1] + r * a.kns[2]) + c * 16ll);
    const V xv = *reinterpret_cast<const V*>((const char*)a.v_new + bytes(b * a.vns[0] + h * a.vns[1] + r * a.vns[2]) + c * 16ll);
    *reinterpret_cast<V*>((char*)a.k + bytes((int64_t)id * pg.ks[0] + h * pg.ks[1] + row * pg.ks[2]) + c * 16ll) = xk;
    *reinterpret_cast<V*>((char*)a.v + bytes((int64_t)id * pg.vs[0] + h * pg.vs[1] + row * pg.vs[2]) + c * 16ll) = xv;
    if (a.weights != nullptr && c == 0) a.weights[((int64_t)b * pg.Hkv + h) * cap + at] = 0.f;
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
constexpr int kSelectThreads = 1024;
// ascending as unsigned; the two zeros are equal, NaN counts as the largest.  On the bits alone: arithmetic may drop a NaN's sign.
__device__ __forceinline__ uint32_t order_bits(float w) {
  const uint32_t u = __float_as_uint(w);
  if ((u & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
  if ((u & 0x7fffffffu) == 0) return 0x80000000u;
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__global__ void __launch_bounds__(kSelectThreads) paged_select_kernel(const __grid_constant__ EvictArgs a) {
  __shared__ int hist[256];
  __shared__ int warp_sums[33];
  __shared__ uint32_t s_prefix;
  __shared__ int s_left;
  grid_dep_wait();
  grid_dep_launch();
  const Pages& pg = a.pg;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int b = blockIdx.x / pg.Hkv, h = blockIdx.x - b * pg.Hkv;
  const int64_t cap = (int64_t)pg.max_pages << pg.shift, at = ((int64_t)b * pg.Hkv + h) * cap;
  const float* const w = a.weights + at;
  float* const wo = a.weights_out + at;
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
    for (int64_t j = tid; j < cap; j += kSelectThreads) wo[j] = j < len ? ld_behind_wait(w + j) : 0.f;
    for (int j = tid; j < a.budget; j += kSelectThreads) kept[j] = j < len ? j : -1;
    return;
  }
  const int from = a.sinks, to = len - a.recent;               // the candidates
  const int want = a.budget - a.sinks - a.recent;              // < to - from
  uint32_t prefix = 0;
  int left = want;                                             // to be found among the keys that share the prefix
  if (want > 0) {
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (int i = tid; i < 256; i += kSelectThreads) hist[i] = 0;
      __syncthreads();
      for (int j = from + tid; j < to; j += kSelectThreads) {
        const uint32_t u = order_bits(ld_behind_wait(w + j));
        if (shift == 24 || (u >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&hist[(u >> shift) & 255u], 1);
      }
      __syncthreads();
      if (warp == 0) {
        // bin of the key that is `left` places from the top: lane l sums the bins 255 - 8 l .. 248 - 8 l
        int c[8], sum = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          c[e] = hist[255 - 8 * lane - e];
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
  }
  // ordered: a key stays if it is a sink or recent, above the border, or among the first `left` on it
  int out = 0, ties = 0;                                       // survivors and border keys in front of this round
  for (int j0 = 0; j0 < len; j0 += kSelectThreads) {
    const int j = j0 + tid;
    float x = 0.f;
    bool stay = false, tie = false;
    if (j < len) {
      x = ld_behind_wait(w + j);
      const uint32_t u = order_bits(x);
      const bool ends = j < from || j >= to;
      stay = ends || (want > 0 && u > prefix);
      tie = !ends && want > 0 && u == prefix;
    }
    const unsigned tb = __ballot_sync(0xffffffffu, tie), sb = __ballot_sync(0xffffffffu, stay);
    // border keys in front of this one, to know whether it stays
    if (lane == 0) warp_sums[warp] = __popc(tb) | __popc(sb) << 16;
    __syncthreads();
    int my_ties = ties, round_ties = 0;
    for (int k = 0; k < kSelectThreads / 32; ++k) {
      const int x2 = warp_sums[k] & 0xffff;
      if (k < warp) my_ties += x2;
      round_ties += x2;
    }
    __syncthreads();
    my_ties += __popc(tb & ((1u << lane) - 1u));
    stay |= tie && my_ties < left;
    const unsigned kb = __ballot_sync(0xffffffffu, stay);
    if (lane == 0) warp_sums[warp] = __popc(kb);
    __syncthreads();
    int my_out = out, round_out = 0;
    for (int k = 0; k < kSelectThreads / 32; ++k) {
      const int x2 = warp_sums[k];
      if (k < warp) my_out += x2;
      round_out += x2;
    }
    __syncthreads();
    my_out += __popc(kb & ((1u << lane) - 1u));
    if (stay) {
      kept[my_out] = j;
      wo[my_out] = x;
    }
    out += round_out;
    ties += round_ties;
  }
  for (int64_t j = a.budget + tid; j < cap; j += kSelectThreads) wo[j] = 0.f;
}

__global__ void __launch_bounds__(256) paged_move_kernel(const __grid_constant__ EvictArgs a, int vecs, int size) {
  grid_dep_wait();
  grid_dep_launch();
  const Pages& pg = a.pg;
  const int b = blockIdx.y / pg.Hkv, h = blockIdx.y - b * pg.Hkv;
  if (pg.length(b) <= a.budget) return;
  const int* const kept = a.kept + ((int64_t)b * pg.Hkv + h) * a.budget;
  const int per = 256 / vecs > 0 ? 256 / vecs : 1;             // rows a round
  const int c = threadIdx.x % vecs, lr = threadIdx.x / vecs;
  if (lr >= per) return;
  constexpr int kRounds = 8;
  const int base = blockIdx.x * per * kRounds;
#pragma unroll
  for (int e = 0; e < kRounds; ++e) {
    const int r = base + e * per + lr;
    if (r >= a.budget) break;
    const int j = ld_behind_wait(kept + r);
    const int src = pg.id(b, j >> pg.shift);
    const int page_no = r >> pg.shift;
    const int dst = page_no < a.n_fresh ? ld_behind_wait(a.fresh + (int64_t)b * a.n_fresh + page_no) : -1;
    if (src < 0 || src >= pg.n_pages || dst < 0 || dst >= pg.n_pages) {
      note(pg.status, kBadPage);
      continue;
    }
    const int64_t from = j & (pg.page - 1), to = r & (pg.page - 1);
    auto at = [&](const int64_t (&s)[3], int64_t id, int64_t row) { return (id * s[0] + h * s[1] + row * s[2]) * size + c * 16ll; };
    const uint4 xk = *reinterpret_cast<const uint4*>((const char*)a.k + at(pg.ks, src, from));
    const uint4 xv = *reinterpret_cast<const uint4*>((const char*)a.v + at(pg.vs, src, from));
    *reinterpret_cast<uint4*>((char*)a.k + at(pg.ks, dst, to)) = xk;
    *reinterpret_cast<uint4*>((char*)a.v + at(pg.vs, dst, to)) = xv;
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

template <typename T, int kD> constexpr int attend_smem() {
  return kAttendSmem<T, kD> + (std::is_same<T, float>::value ? (kRowTile * kD + kWarps * kRowTile * kStep) * 4 : 0);
}
// CTAs of the attention kernel an SM holds (by shared memory: 192 KB in 16 bits at D = 128 are two CTAs)
int attend_per_sm(int dtype, int D) { return dtype == LMK_F32 ? (D <= 64 ? 2 : 1) : (D <= 64 ? 4 : 2); }
constexpr int kLeastSteps = 8;         // of a CTA: two a warp

struct AttendPlan {
  int grid, rows, tiles, kD;
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
  p->acc = 0;
  p->stat = up(p->acc + sizeof(float) * 2 * p->grid * kRowTile * p->kD);
  p->whole = up(p->stat + sizeof(float2) * 2 * p->grid * kRowTile);
  p->scores = up(p->whole + (weights ? sizeof(float2) * B * Hkv * (size_t)p->tiles * kRowTile : 0));
  p->bytes = up(p->scores + (weights ? sizeof(float) * (size_t)B * Hkv * p->rows * max_pages * page : 0));
  return LMK_OK;
}
bool attend_sizes_ok(int B, int H, int Hkv, int T) {
  return B >= 1 && Hkv >= 1 && H >= Hkv && H % Hkv == 0 && T >= 1 && T <= 1024 && (int64_t)H / Hkv * T <= 4096 && (int64_t)B * H * T < (1 << 30);
}

template <typename T, int kD>
int launch_attend(const AttendArgs& a, cudaStream_t st) {
  static std::atomic<bool> ready[64];
  int dev = 0;
  LMK_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64) return fail(LMK_ERR_UNSUPPORTED, "device index %d out of range", dev);
  if (!ready[dev].load(std::memory_order_acquire)) {
    LMK_CUDA(cudaFuncSetAttribute(paged_attend_kernel<T, kD>, cudaFuncAttributeMaxDynamicSharedMemorySize, attend_smem<T, kD>()));
    ready[dev].store(true, std::memory_order_release);
  }
  LMK_CUDA(launch_overlapped(paged_attend_kernel<T, kD>, dim3(a.grid), dim3(kWarps * 32), attend_smem<T, kD>(), st, a));
  const int64_t cap = (int64_t)a.pg.max_pages << a.pg.shift;
  // a row is in several pieces only where its steps can exceed the least piece
  if (cap / kStep > 1) LMK_CUDA(launch_overlapped(paged_join_kernel<T, kD>, dim3(a.pg.B * a.pg.Hkv * a.tiles, kD / 32), dim3(kJoinThreads), 0, st, a));
  if (a.weights != nullptr) {
    const int runs = (int)((cap + kJoinThreads * 4 - 1) / (kJoinThreads * 4));
    LMK_CUDA(launch_overlapped(paged_weights_kernel<T>, dim3(runs, a.pg.B * a.pg.Hkv), dim3(kJoinThreads), sizeof(float2) * a.rows, st, a));
  }
  return LMK_OK;
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
  LMK_CHECK_ARG(isfinite(sm_scale) && isfinite(decay), "paged attention: scale and decay must be finite");
  const int pair = 4 / dtype_size(dtype);
  LMK_CHECK_ARG(((uintptr_t)q & 3) == 0 && q_strides[0] % pair == 0 && q_strides[1] % pair == 0 && q_strides[2] % pair == 0,
                "paged attention: q must lie on 4-byte boundaries");
  LMK_CHECK_ARG(((uintptr_t)o & 15) == 0, "paged attention: o must start on a 16-byte boundary");
  AttendPlan p;
  if ((rc = attend_plan(&p, B, H, Hkv, T, D, page, max_pages, weights != nullptr, dtype)) != LMK_OK) return rc;
  if (workspace == nullptr || workspace_bytes < p.bytes || ((uintptr_t)workspace & 255) != 0)
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
  a.scale_log2 = sm_scale * kLog2e;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
#define LMK_ATTEND(T) return p.kD == 64 ? launch_attend<T, 64>(a, st) : launch_attend<T, 128>(a, st)
  if (dtype == LMK_BF16) LMK_ATTEND(__nv_bfloat16);
  if (dtype == LMK_F16) LMK_ATTEND(__half);
  LMK_ATTEND(float);
#undef LMK_ATTEND
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
  LMK_CUDA(launch_overlapped(paged_select_kernel, dim3(B * Hkv), dim3(kSelectThreads), 0, st, a));
  const int rows = (256 / vecs) * 8;
  LMK_CUDA(launch_overlapped(paged_move_kernel, dim3((budget + rows - 1) / rows, B * Hkv), dim3(256), 0, st, a, vecs, size));
  return LMK_OK;
}
