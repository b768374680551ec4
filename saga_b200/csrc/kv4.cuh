// Device helpers of the 4-bit paged cache.
//
// A tile is 32 positions of one head: 32 rows of D/2 bytes of codes, then 32 *
// D/64 words of scales. Byte b of a row holds value 2b in its low and 2b + 1 in
// its high four bits. The 16-byte chunks of a row are permuted by the row's
// number (kv4_swizzle): the eight rows that one ldmatrix phase reads, 64 (32)
// bytes apart, then lie in different banks, and a tile copied as it stands by
// one bulk copy can be read without conflicts. A word of scales holds a
// group's s in its low and z in its high half (bfloat16).
#pragma once

#include "common.cuh"
#include "kv4.h"

namespace saga {

// Waits until the kernels before this one in the stream have finished and their
// writes can be seen, then lets the next one start its own wait.
__device__ __forceinline__ void pdl_wait() {
  asm volatile("griddepcontrol.wait;\n" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
}

template <int D>
__device__ __forceinline__ int kv4_swizzle(int row) {
  return D == 128 ? (row >> 1) & 3 : (row >> 2) & 1;
}
// Byte offset in a tile of 16-byte chunk `ch` of row `row`.
template <int D>
__device__ __forceinline__ int kv4_chunk_off(int row, int ch) {
  return row * (D / 2) + ((ch ^ kv4_swizzle<D>(row)) << 4);
}
// Byte offset in a tile of the scale word of group `g` of row `row`.
template <int D>
__device__ __forceinline__ int kv4_meta_off(int row, int g) {
  return kKv4Tile * (D / 2) + (row * (D / 64) + g) * 4;
}
__device__ __forceinline__ float kv4_scale(uint32_t m) { return __uint_as_float(m << 16); }
__device__ __forceinline__ float kv4_zero(uint32_t m) { return __uint_as_float(m & 0xffff0000u); }

// First byte of the tile that holds offset `off` of page `page`, head `h` of H.
template <int D>
__device__ __forceinline__ int64_t kv4_tile_at(int64_t page, int h, int H, int off, int page_len) {
  return ((page * H + h) * (int64_t)(page_len / kKv4Tile) + off / kKv4Tile) * kv4_tile_bytes(D);
}

// Two binary32 values in one register pair: the packed forms issue one instruction for both.
using f32x2 = unsigned long long;
__device__ __forceinline__ f32x2 pack2(float lo, float hi) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void unpack2(f32x2 v, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// The greatest bfloat16 at or below x, the least at or above it.
__device__ __forceinline__ __nv_bfloat16 bf16_down(float x) { return __float2bfloat16_rd(x); }
__device__ __forceinline__ __nv_bfloat16 bf16_up(float x) { return __float2bfloat16_ru(x); }

}  // namespace saga
