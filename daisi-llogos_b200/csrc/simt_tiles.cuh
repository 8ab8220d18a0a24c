// Tiles of cached rows in shared memory as float32, for the CUDA-core kernels of drafted trees and key weights.
#pragma once
#include "common.cuh"

namespace {

// Copies `rows` rows of `width` elements that lie one behind the other at `src` into shared memory rows of `stride` floats, zeros behind
// `width` up to `padded` (a multiple of 4) and for the rows from `valid` on.  float32 rows of whole 16 bytes go asynchronously (cp.async; the
// caller commits and waits), everything else through registers.  A thread walks along the tile by a fixed step in (row, 16-byte chunk), which is
// worked out once: a division and a page look-up per chunk cost more than the products of a small tile.
template <int THREADS>
struct TileCopy {
  int padded4, row0, chunk0, row_step, chunk_step;
  __device__ __forceinline__ explicit TileCopy(int padded) {
    padded4 = padded / 4;
    row0 = threadIdx.x / padded4;
    chunk0 = threadIdx.x - row0 * padded4;
    row_step = THREADS / padded4;
    chunk_step = THREADS - row_step * padded4;
  }
  template <typename T>
  __device__ __forceinline__ void operator()(float* dst, int stride, const T* src, int rows, int valid, int width) const {
    int r = row0, c = chunk0;
    const bool wide = (width & 3) == 0;
    while (r < rows) {
      float* to = dst + r * stride + 4 * c;
      const T* from = src + (long long)r * width + 4 * c;
      const bool there = r < valid && 4 * c < width;
      if (wide && sizeof(T) == 4) {
        const int n = there ? 16 : 0;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(there ? from : src), "r"(n) : "memory");
      } else {
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        if (there) {
          v.x = to_f32(from[0]);
          if (4 * c + 1 < width) v.y = to_f32(from[1]);
          if (4 * c + 2 < width) v.z = to_f32(from[2]);
          if (4 * c + 3 < width) v.w = to_f32(from[3]);
        }
        *reinterpret_cast<float4*>(to) = v;
      }
      r += row_step;
      c += chunk_step;
      if (c >= padded4) {
        c -= padded4;
        ++r;
      }
    }
  }
};

__device__ __forceinline__ void tile_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void tile_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// A thread's share of `rows` query rows (`row(r)`: where row r's elements lie, null for a row of zeros): rows of whole 16 bytes go asynchronously, as above.
template <int THREADS, typename T, typename Row>
__device__ __forceinline__ void copy_rows(float* dst, int stride, int rows, int width, int padded, Row row) {
  const int padded4 = padded / 4;
  const bool wide = (width & 3) == 0;
  for (int x = threadIdx.x; x < rows * padded4; x += THREADS) {
    const int r = x / padded4, d = (x - r * padded4) * 4;
    const T* src = row(r);
    float* to = dst + r * stride + d;
    if (wide && sizeof(T) == 4 && src) {
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(src + d) : "memory");
    } else {
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      if (src) {
        v.x = d < width ? to_f32(src[d]) : 0.f;
        v.y = d + 1 < width ? to_f32(src[d + 1]) : 0.f;
        v.z = d + 2 < width ? to_f32(src[d + 2]) : 0.f;
        v.w = d + 3 < width ? to_f32(src[d + 3]) : 0.f;
      }
      *reinterpret_cast<float4*>(to) = v;
    }
  }
}

}  // namespace
