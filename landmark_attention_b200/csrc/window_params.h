// Sliding-window attention with sinks: arguments, and which tiles of queries and keys meet.
#pragma once
#include <stdint.h>
#include <cuda_runtime.h>

namespace lmk {

// dK and dV of the key tiles that hold sinks get contributions from every later query.  Their query tiles are dealt out to several units:
// the ones that see the tile through the window (as for every key tile), and runs of `run` tiles of the others, at most `runs` of
// them.  Each unit leaves an fp32 sum for the sinks, and a last kernel adds these up in order; the tile's other keys are the first unit's alone.
struct SinkSplit {
  int tiles = 0;       // key tiles that hold sinks; 0: no tile is split
  int run = 0, runs = 0;
  float* part = nullptr;      // [B * Hkv][tiles][1 + runs][dK, dV][keys of a tile][D]
};

struct WindowParams {
  const void *q, *k, *v, *dO;
  void* o;                     // forward output / backward input
  void* rest;                  // what the rounding of o left, a byte a number (16-bit types; null: not wanted)
  float* lse;                  // [B*H, Lq]: log2 of the row's normaliser, +inf for a row that sees nothing (null: not wanted)
  const int* lengths;          // [B] or null
  void *dq, *dk, *dv;
  float* delta;                // [B*H, Lq] scratch (backward)
  int* next;                   // scratch (backward of 16-bit types): the next unit of the dK/dV kernel
  int B, H, Hkv, Lq, Lk, D, window, sinks;      // 1 <= window <= Lk, 0 <= sinks <= Lk
  int64_t qs[3], ks[3], vs[3], dos[3];          // element strides {batch, head, row}
  float scale;
  SinkSplit split;
};

// Tiles, all inclusive ranges of tile numbers; empty where first > last.
struct KeyTiles { int sink_tiles, first, last; };      // tiles 0 .. sink_tiles - 1 in front of first .. last
struct QueryTiles { int first, last, end; };           // first .. last through the window, last + 1 .. end through the sinks alone

// key tiles of kk keys that a tile of qt query rows sees; len: keys of the sequence
__host__ __device__ inline KeyTiles keys_of_queries(int tile, int qt, int kk, int Lq, int off, int len, int window, int sinks) {
  KeyTiles r;
  const int p0 = off + tile * qt;
  int p1 = p0 + qt - 1;
  if (p1 > off + Lq - 1) p1 = off + Lq - 1;
  if (p1 > len - 1) p1 = len - 1;
  if (p1 < p0) {
    r.sink_tiles = 0;
    r.first = 0;
    r.last = -1;
    return r;
  }
  const int lo = p0 - window + 1 > 0 ? p0 - window + 1 : 0;
  r.first = lo / kk;
  r.last = p1 / kk;
  const int st = (sinks + kk - 1) / kk;
  r.sink_tiles = st < r.first ? st : r.first;
  return r;
}
// tiles of qt query rows that see a tile of kk keys
__host__ __device__ inline QueryTiles queries_of_keys(int tile, int qt, int kk, int Lq, int off, int len, int window, int sinks) {
  QueryTiles r;
  const int k0 = tile * kk;
  const int top = len - 1 - off < Lq - 1 ? len - 1 - off : Lq - 1;      // the last row that is one
  if (k0 >= len || top < 0) {
    r.first = 0;
    r.last = r.end = -1;
    return r;
  }
  const int k1 = k0 + kk - 1 < len - 1 ? k0 + kk - 1 : len - 1;
  const int end = top / qt;
  r.first = k0 > off ? (k0 - off) / qt : 0;
  const int w = k1 + window - 1 - off;                                  // the last row that sees k1 through the window
  r.last = w < 0 ? r.first - 1 : (w / qt < end ? w / qt : end);
  if (r.last < r.first - 1) r.last = r.first - 1;
  r.end = k0 < sinks ? end : r.last;
  if (r.end < r.last) r.end = r.last;
  return r;
}
__host__ __device__ inline bool window_sees(int pos, int key, int window, int sinks) {
  return key <= pos && (pos - key < window || key < sinks);
}

// fp32, tiles of 64 query rows and 64 keys
int window_f32_fwd(const WindowParams& p, cudaStream_t st);
int window_f32_bwd(const WindowParams& p, cudaStream_t st);
// 16-bit types, tiles of 128 query rows; dK and dV in tiles of 128 keys
int window_sm100_fwd(const WindowParams& p, int dtype, cudaStream_t st);
int window_sm100_bwd(const WindowParams& p, int dtype, cudaStream_t st);
bool window_sm100_operand_ok(const void* p, const int64_t st[3], int D);
// adds up the parts of the sinks, in tiles of kk keys, into dk and dv
int window_join_parts(const WindowParams& p, int qt, int kk, int dtype, cudaStream_t st);

}  // namespace lmk
