// Rows of 16-bit tiles on their way between registers, shared memory and the outputs (sm_100a attention kernels).
#pragma once
#include "common.cuh"
#include "sm100_ptx.cuh"

namespace lmk {
namespace {

using namespace ptx;

template <bool kBf16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if (kBf16) {
    __nv_bfloat162 t = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&t);
  } else {
    __half2 t = __floats2half2_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&t);
  }
}

// write one row (64 16-bit values, given as 32 packed words) of a [128 x 64] K-major 128B-swizzled tile
__device__ __forceinline__ void store_row_sw128(uint32_t tile_base, int row, const uint32_t (&w)[32]) {
  const uint32_t row_addr = tile_base + row * 128;
#pragma unroll
  for (int c = 0; c < 8; ++c) {
    uint32_t addr = row_addr + ((c ^ (row & 7)) << 4);
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(w[4 * c]), "r"(w[4 * c + 1]),
                 "r"(w[4 * c + 2]), "r"(w[4 * c + 3])
                 : "memory");
  }
}

template <bool kBf16>
__device__ __forceinline__ uint32_t pack2p(uint64_t v) {
  float lo, hi;
  upk2(v, lo, hi);
  return pack2<kBf16>(lo, hi);
}

// Stores 32 accumulator columns of one TMEM lane per thread as 16-bit values.  Four neighbouring lanes exchange 16-byte
// chunks first, so that a warp's store covers 64 contiguous bytes of eight rows and not 16 bytes of thirty-two.
// row_off[j]: element offset of row j of the lane's four rows, or -1 for a row that is not stored.  An output of the C interface
// may start at any word: one off a 16-byte boundary is stored word by word.
template <bool kBf16>
__device__ __forceinline__ void store_acc_cols(void* out, const int64_t (&row_off)[4], const uint32_t (&r)[32], int col0, int D,
                                               int lane) {
  uint4 v[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    v[e].x = pack2<kBf16>(__uint_as_float(r[8 * e + 0]), __uint_as_float(r[8 * e + 1]));
    v[e].y = pack2<kBf16>(__uint_as_float(r[8 * e + 2]), __uint_as_float(r[8 * e + 3]));
    v[e].z = pack2<kBf16>(__uint_as_float(r[8 * e + 4]), __uint_as_float(r[8 * e + 5]));
    v[e].w = pack2<kBf16>(__uint_as_float(r[8 * e + 6]), __uint_as_float(r[8 * e + 7]));
  }
  // transpose of the 4 x 4 matrix (lane of the four, chunk): swap the off-diagonal chunks of 2 x 2 blocks, then the blocks
  auto swap = [&](uint4& a, uint4& b, int step) {      // lower lane: b <-> partner's a
    const bool up = (lane & step) != 0;
    uint4 x = up ? a : b;
    x.x = __shfl_xor_sync(0xffffffffu, x.x, step);
    x.y = __shfl_xor_sync(0xffffffffu, x.y, step);
    x.z = __shfl_xor_sync(0xffffffffu, x.z, step);
    x.w = __shfl_xor_sync(0xffffffffu, x.w, step);
    a = up ? x : a;
    b = up ? b : x;
  };
  swap(v[0], v[1], 1);
  swap(v[2], v[3], 1);
  swap(v[0], v[2], 2);
  swap(v[1], v[3], 2);
  const int col = col0 + 8 * (lane & 3);
  if (col >= D) return;
  const bool wide = ((uintptr_t)out & 15) == 0;       // rows and columns are multiples of 16 bytes
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (row_off[j] < 0) continue;
    uint32_t* to = reinterpret_cast<uint32_t*>(reinterpret_cast<uint16_t*>(out) + row_off[j] + col);
    if (wide) {
      *reinterpret_cast<uint4*>(to) = v[j];
    } else {
      to[0] = v[j].x;
      to[1] = v[j].y;
      to[2] = v[j].z;
      to[3] = v[j].w;
    }
  }
}

}  // namespace
}  // namespace lmk
