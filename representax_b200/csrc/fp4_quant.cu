// Quantiser to microscaled 4-bit floating point and its inverse.
//
//   MXFP4  block of 32: e = max(-126, ceil(log2(amax / 6))), code = E2M1(x 2^-e)
//   NVFP4  row: f = 2^ceil(log2(rowmax / 2688)) (2688 = 6 * 448, at least 2^-126), block of 16:
//          s = E4M3(amax / 6 / f), code = E2M1(x / (s f))
//
// All roundings are to nearest, ties to even; zeros give code 0. The factor f
// is a power of two, so that s f and the comparisons with rounding boundaries
// are exact; it belongs to the row, not to the matrix, so that one pass over
// the rows finds it and tokens do not depend on one another. Blocks (MXFP4) or
// rows (NVFP4) that hold an infinity or a NaN get a NaN scale: their values
// and products are NaN.
//
// Bound by HBM: x is read once (2 or 4 bytes a value), half a byte a value and
// the scales are written. A lane takes 8 consecutive values (one or two 16-byte
// loads, one 4-byte store), so a warp covers 256 consecutive ones and a
// block's maximum needs one or two shuffles. A row belongs to 1, 2, 4 or 8 warps
// by its length; NVFP4 keeps up to 8 x kKeep values a lane in registers between the
// row's maximum and the codes and reads longer rows a second time.
#include "fp4.h"

#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "fp4.cuh"

namespace rx {
namespace fp4 {

constexpr int kQuantThreads = 256;
constexpr int kKeep = 4;

template <typename T>
__device__ __forceinline__ float to_float(T v) { return static_cast<float>(v); }
template <>
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }

template <typename T>
__device__ __forceinline__ T from_float(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_float(float v) { return __float2half_rn(v); }

// Eight consecutive values of a row from column c, zeros past K.
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* row, int c, int K, float (&v)[8]) {
  if (VEC && c + 8 <= K) {
    constexpr int kLoads = sizeof(T) / 2;
    uint4 w[kLoads];
#pragma unroll
    for (int i = 0; i < kLoads; ++i) w[i] = ldg_v4_issue(reinterpret_cast<const uint4*>(row + c) + i);
    const T* e = reinterpret_cast<const T*>(w);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = to_float(e[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c + i < K ? to_float(row[c + i]) : 0.f;
  }
}

__device__ __forceinline__ uint32_t top8(const float (&v)[8]) {
  uint32_t t = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) t = max(t, __float_as_uint(v[i]) & 0x7fffffffu);
  return t;
}

// 2^ceil(log2(top / 2688)) from the float bits of the row's largest magnitude.
__device__ __forceinline__ float row_factor(uint32_t top) {
  if (top >= 0x7f800000u) return __uint_as_float(0x7fc00000u);
  const uint32_t b = __float_as_uint(__fdiv_rn(__uint_as_float(top), 2688.f));
  if (b == 0u) return 1.f;
  return __uint_as_float(max((b >> 23) + ((b & 0x7fffffu) != 0u ? 1u : 0u), 1u) << 23);
}

__device__ __forceinline__ float e4m3_value(uint32_t byte) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(static_cast<__nv_fp8_storage_t>(byte), __NV_E4M3)));
}

// Rows of a CTA: kQuantThreads / (32 * warps_per_row). Every warp of a row walks
// the padded extent groups * (values of a group) in steps of 256 values, so all
// scale bytes of the row tiles, padding included, are written.
template <typename T, int FMT, bool VEC>
__global__ void __launch_bounds__(kQuantThreads)
    quantize_kernel(const QuantParams p, int warps_per_row) {
  __shared__ uint32_t tops[kQuantThreads / 32];
  const int warp = warp_id(), lane = lane_id();
  const int rows_per_cta = (kQuantThreads / 32) / warps_per_row;
  const int part_of_row = warp % warps_per_row;
  const int64_t padded = (p.rows + 127) / 128 * 128;
  const int64_t slot = static_cast<int64_t>(blockIdx.x) * rows_per_cta + warp / warps_per_row;  // row of the padded tiles
  const int64_t part = slot / padded, r = slot % padded;
  const bool in_grid = part < p.parts, live = in_grid && r < p.rows;
  const int64_t row = part * p.rows + r;
  const T* x = static_cast<const T*>(p.x) + row * p.ldx;
  const int extent = static_cast<int>(p.groups) * 4 * block_of(FMT);
  const int c0 = part_of_row * 256 + lane * 8, step = warps_per_row * 256;
  const int64_t sf_row = part * padded + r;

  float factor = 1.f;
  float keep[FMT == kNv ? kKeep : 1][8];
  if constexpr (FMT == kNv) {
    uint32_t top = 0;
    if (live) {
#pragma unroll
      for (int i = 0; i < kKeep; ++i) {
        if (c0 + i * step < p.K) {
          load8<T, VEC>(x, c0 + i * step, p.K, keep[i]);
          top = max(top, top8(keep[i]));
        }
      }
      for (int c = c0 + kKeep * step; c < p.K; c += step) {
        float v[8];
        load8<T, VEC>(x, c, p.K, v);
        top = max(top, top8(v));
      }
    }
    top = __reduce_max_sync(0xffffffffu, top);
    if (warps_per_row > 1) {  // the same for every thread of the CTA
      if (lane == 0) tops[warp] = top;
      __syncthreads();
      for (int i = 0; i < warps_per_row; ++i) top = max(top, tops[warp - part_of_row + i]);
    }
    factor = row_factor(top);
    if (live && part_of_row == 0 && lane == 0) p.row_scale[row] = factor;
  }
  if (!in_grid) return;

  auto emit = [&](const float (&v)[8], int c) {
    uint32_t top = top8(v);
    uint32_t byte, codes;
    float w[8];
    if constexpr (FMT == kMx) {
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      byte = mx_scale_byte(top);
      const float inv = mx_inverse(byte);
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = v[i] * inv;
    } else {
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      const float want = __fdiv_rn(__fdiv_rn(__uint_as_float(top), 6.f), factor);
      byte = __nv_cvt_float_to_fp8(want, __NV_SATFINITE, __NV_E4M3);
      const float scale = e4m3_value(byte) * factor;
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = scale > 0.f ? __fdiv_rn(v[i], scale) : 0.f;
    }
    codes = pack8(w);
    // four blocks' bytes -> one 4-byte word of the group, written by its first lane
    constexpr int kLanes = block_of(FMT) / 8;  // lanes of a block
    uint32_t word = byte << (8 * ((lane / kLanes) & 3));
#pragma unroll
    for (int o = kLanes; o < 4 * kLanes; o *= 2) word |= __shfl_xor_sync(0xffffffffu, word, o);
    if (c < extent) {
      if (lane % (4 * kLanes) == 0)
        *reinterpret_cast<uint32_t*>(p.sf + scale_offset(sf_row, c / block_of(FMT), p.groups)) = live ? word : 0u;
      if (live && (c >> 1) < p.ldq) *reinterpret_cast<uint32_t*>(p.q + row * p.ldq + (c >> 1)) = codes;
    }
  };

  int i = 0;
  for (int c = c0; c - lane * 8 < extent; c += step, ++i) {  // warp-uniform
    float v[8];
    if constexpr (FMT == kNv) {
      if (i < kKeep) {
#pragma unroll
        for (int j = 0; j < kKeep; ++j)
          if (j == i)
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = live && c < p.K ? keep[j][e] : 0.f;
        emit(v, c);
        continue;
      }
    }
    if (live && c < p.K) {
      load8<T, VEC>(x, c, p.K, v);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = 0.f;
    }
    emit(v, c);
  }
}

template <typename T, int FMT>
cudaError_t quantize_typed(const QuantParams& p, cudaStream_t stream) {
  const bool vec = reinterpret_cast<uintptr_t>(p.x) % 16 == 0 && p.ldx % (16 / sizeof(T)) == 0;
  const int64_t chunks = (p.K + 255) / 256;
  const int wpr = chunks <= 1 ? 1 : (chunks <= 2 ? 2 : (chunks <= 4 ? 4 : 8));
  const int64_t slots = p.parts * ((p.rows + 127) / 128 * 128);
  const int64_t grid = (slots * wpr + kQuantThreads / 32 - 1) / (kQuantThreads / 32);
  if (vec)
    quantize_kernel<T, FMT, true><<<static_cast<unsigned>(grid), kQuantThreads, 0, stream>>>(p, wpr);
  else
    quantize_kernel<T, FMT, false><<<static_cast<unsigned>(grid), kQuantThreads, 0, stream>>>(p, wpr);
  return cudaGetLastError();
}

cudaError_t quantize(const QuantParams& p, int fmt, int type, cudaStream_t stream) {
  const bool mx = fmt == kMx;
  switch (type) {
    case kBf16In: return mx ? quantize_typed<__nv_bfloat16, kMx>(p, stream) : quantize_typed<__nv_bfloat16, kNv>(p, stream);
    case kF16In: return mx ? quantize_typed<__half, kMx>(p, stream) : quantize_typed<__half, kNv>(p, stream);
    default: return mx ? quantize_typed<float, kMx>(p, stream) : quantize_typed<float, kNv>(p, stream);
  }
}

// One thread: 8 values of a row.
template <typename T, int FMT>
__global__ void __launch_bounds__(256) dequantize_kernel(const DequantParams p, bool vec) {
  const int64_t padded = (p.rows + 127) / 128 * 128;
  const int per_row = (p.K + 7) / 8;
  const int64_t total = p.parts * p.rows * per_row;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int64_t row = i / per_row;
    const int c = static_cast<int>(i - row * per_row) * 8;
    const int64_t part = row / p.rows;
    const uint32_t codes = *reinterpret_cast<const uint32_t*>(p.q + row * p.ldq + (c >> 1));
    const uint32_t byte = p.sf[scale_offset(part * padded + row - part * p.rows, c / block_of(FMT), p.groups)];
    float scale;
    if constexpr (FMT == kMx)
      scale = byte == 0xffu ? __uint_as_float(0x7fc00000u) : __uint_as_float(byte << 23);
    else
      scale = e4m3_value(byte) * p.row_scale[row];
    T v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t n = (codes >> (4 * j)) & 0xfu;
      // magnitude codes 0..7: 0, 0.5, then (1 + m / 2) 2^(e - 1)
      const uint32_t mag = n & 7u;
      const float m = mag < 2u ? 0.5f * mag : __uint_as_float(((mag >> 1) + 126u) << 23 | (mag & 1u) << 22);
      v[j] = from_float<T>((n & 8u ? -m : m) * scale);
    }
    T* dst = static_cast<T*>(p.out) + row * p.ldo + c;
    if (vec && c + 8 <= p.K) {
      constexpr int kStores = sizeof(T) / 2;
      const uint4* w = reinterpret_cast<const uint4*>(v);
#pragma unroll
      for (int j = 0; j < kStores; ++j) reinterpret_cast<uint4*>(dst)[j] = w[j];
    } else {
      for (int j = 0; j < 8 && c + j < p.K; ++j) dst[j] = v[j];
    }
  }
}

template <typename T>
cudaError_t dequantize_typed(const DequantParams& p, int fmt, cudaStream_t stream) {
  const bool vec = reinterpret_cast<uintptr_t>(p.out) % 16 == 0 && p.ldo % (16 / sizeof(T)) == 0;
  const int64_t total = p.parts * p.rows * ((p.K + 7) / 8);
  const int64_t want = (total + 255) / 256;
  const unsigned grid = static_cast<unsigned>(want < 148 * 32 ? want : 148 * 32);
  if (fmt == kMx)
    dequantize_kernel<T, kMx><<<grid, 256, 0, stream>>>(p, vec);
  else
    dequantize_kernel<T, kNv><<<grid, 256, 0, stream>>>(p, vec);
  return cudaGetLastError();
}

cudaError_t dequantize(const DequantParams& p, int fmt, int type, cudaStream_t stream) {
  switch (type) {
    case kBf16In: return dequantize_typed<__nv_bfloat16>(p, fmt, stream);
    case kF16In: return dequantize_typed<__half>(p, fmt, stream);
    default: return dequantize_typed<float>(p, fmt, stream);
  }
}

}  // namespace fp4
}  // namespace rx
