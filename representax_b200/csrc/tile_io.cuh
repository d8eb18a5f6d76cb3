// Moving 32-column pieces of bf16 tiles between global memory, registers and
// shared memory (64-byte swizzle of the store tensor maps).
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace rx {
namespace gemm {

__device__ __forceinline__ void load_bf16x32(const __nv_bfloat16* src, float (&v)[32]) {
  const uint4* s = reinterpret_cast<const uint4*>(src);
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    uint4 w = s[q];
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&w);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float2 f = __bfloat1622float2(h[j]);
      v[q * 8 + 2 * j] = f.x;
      v[q * 8 + 2 * j + 1] = f.y;
    }
  }
}

__device__ __forceinline__ void store_bf16x32(__nv_bfloat16* dst, const float (&v)[32]) {
  uint4* d = reinterpret_cast<uint4*>(dst);
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    uint4 w;
    __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&w);
#pragma unroll
    for (int j = 0; j < 4; ++j) h[j] = __floats2bfloat162_rn(v[q * 8 + 2 * j], v[q * 8 + 2 * j + 1]);
    d[q] = w;
  }
}

// Write one lane's 32 bf16 values as row `lane` of a 32 x 32 tile staged in
// shared memory with the 64-byte swizzle of the store tensor map.
__device__ __forceinline__ void stage_row32_sw64(uint8_t* buf, int lane, const float (&v)[32]) {
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    uint4 w;
    __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&w);
#pragma unroll
    for (int j = 0; j < 4; ++j) h[j] = __floats2bfloat162_rn(v[q * 8 + 2 * j], v[q * 8 + 2 * j + 1]);
    *reinterpret_cast<uint4*>(buf + lane * 64 + ((q ^ ((lane >> 1) & 3)) * 16)) = w;
  }
}

// A 32 x 32 bf16 tile (rows row0.., columns n_base..) from global to shared memory, 16-byte pieces, four lanes to a
// 64-byte row segment; rows >= rows_valid and columns >= cols_valid read as zero. In two steps, so the loads of the next
// tile can be in flight while the current one is computed: fetch into registers (lane holds pieces lane, lane + 32,
// lane + 64, lane + 96) ...
__device__ __forceinline__ void warp_fetch_tile32(const __nv_bfloat16* src, int64_t ld, int row0, int n_base,
                                                  int rows_valid, int cols_valid, int lane, uint4 (&w)[4]) {
#pragma unroll
  for (int it = 0; it < 4; ++it) {
    const int c = lane + 32 * it;
    const int row = c >> 2, piece = c & 3;
    const int m = row0 + row, n = n_base + piece * 8;
    w[it] = make_uint4(0u, 0u, 0u, 0u);
    if (m < rows_valid) {
      const __nv_bfloat16* g = src + static_cast<int64_t>(m) * ld + n;
      if (n + 8 <= cols_valid) {
        w[it] = *reinterpret_cast<const uint4*>(g);
      } else {
        __nv_bfloat16* e = reinterpret_cast<__nv_bfloat16*>(&w[it]);
        for (int k = 0; k < 8; ++k) e[k] = n + k < cols_valid ? g[k] : __float2bfloat16_rn(0.f);
      }
    }
  }
}

// ... then place it in `buf` with the 64-byte swizzle.
__device__ __forceinline__ void warp_put_tile32_sw64(uint8_t* buf, int lane, const uint4 (&w)[4]) {
#pragma unroll
  for (int it = 0; it < 4; ++it) {
    const int c = lane + 32 * it;
    const int row = c >> 2, piece = c & 3;
    *reinterpret_cast<uint4*>(buf + row * 64 + ((piece ^ ((row >> 1) & 3)) * 16)) = w[it];
  }
}

// Row `lane` of a 64-byte-swizzled 32 x 32 bf16 tile as 32 floats.
__device__ __forceinline__ void read_row32_sw64(const uint8_t* buf, int lane, float (&v)[32]) {
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const uint4 w = *reinterpret_cast<const uint4*>(buf + lane * 64 + ((q ^ ((lane >> 1) & 3)) * 16));
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&w);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = __bfloat1622float2(h[j]);
      v[q * 8 + 2 * j] = f.x;
      v[q * 8 + 2 * j + 1] = f.y;
    }
  }
}

}  // namespace gemm
}  // namespace rx
