// Microscaled 4-bit floating point shared by the quantiser and the tensor-core
// kernels: E2M1 codes (0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign), two to a byte
// with the even column in the low nibble, and block scales in the order that
// the tensor core reads them.
//
//   MXFP4  one UE8M0 scale 2^(byte - 127) per 32 values
//   NVFP4  one UE4M3 scale per 16 values and one fp32 factor per row
//
// Scale layout: [row tiles of 128][K groups][512 bytes]; a group covers 4
// blocks (128 values in MXFP4, 64 in NVFP4) and its 512 bytes hold, for row
// r = 32 q + l of the tile and block j of the group, byte 16 l + 4 q + j. That
// is one tcgen05.cp 32x128b.warpx4: TMEM lane l gets the scales of rows l,
// l + 32, l + 64, l + 96 in four 32-bit columns, one byte per block. The number
// of groups is padded to 256 values of K, the extent of one pipeline stage, so
// a stage's groups are one contiguous bulk copy.
#pragma once
#include <cuda_fp16.h>
#include <cuda_fp4.h>
#include <stdint.h>

#include "elect.cuh"
#include "sm100.cuh"

namespace rx {
namespace fp4 {

enum Format : int { kMx = 1, kNv = 2 };

constexpr int kStageK = 256;       // values of K per pipeline stage (128 bytes of codes)
__host__ __device__ constexpr int block_of(int fmt) { return fmt == kMx ? 32 : 16; }
__host__ __device__ constexpr int groups_per_stage(int fmt) { return fmt == kMx ? 2 : 4; }
__host__ __device__ inline int64_t k_groups(int64_t k, int fmt) {
  return (k + kStageK - 1) / kStageK * groups_per_stage(fmt);
}

// Offset of the scale of (row, block) in a scale array with `groups` K groups.
__device__ __forceinline__ int64_t scale_offset(int64_t row, int block, int64_t groups) {
  const int r = static_cast<int>(row & 127);
  return ((row >> 7) * groups + (block >> 2)) * 512 + 16 * (r & 31) + 4 * (r >> 5) + (block & 3);
}

// Eight values -> eight E2M1 codes (round to nearest, ties to even, saturating
// at 6), value i in nibble i.
__device__ __forceinline__ uint32_t pack8(const float (&v)[8]) {
  uint32_t out;
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
      "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
      : "=r"(out)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return out;
}

// The inverse: eight codes -> their values (exact).
__device__ __forceinline__ void unpack8(uint32_t codes, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2_raw h = __nv_cvt_fp4x2_to_halfraw2(static_cast<__nv_fp4x2_storage_t>(codes >> (8 * i)), __NV_E2M1);
    const float2 f = __half22float2(__half2(h));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}

// MXFP4 scale byte of a block whose largest magnitude has the float bits `top`:
// e = ceil(log2(top / 6)), at least -126, so that no code saturates (the rule of
// the MXFP8 quantiser). With top = m 2^k, 1 <= m < 2, and 6 = 1.5 * 2^2 that is
// k - 2 for m <= 1.5 and k - 1 above: no division. Byte 127 (a factor of one) for
// a block of zeros; the NaN byte 0xff for a block that holds an infinity or a
// NaN, so that products with it are NaN.
__device__ __forceinline__ uint32_t mx_scale_byte(uint32_t top) {
  if (top >= 0x7f800000u) return 0xffu;
  if (top == 0u) return 127u;
  return static_cast<uint32_t>(max(static_cast<int>(top >> 23) - 2 + ((top & 0x7fffffu) > 0x400000u ? 1 : 0), 1));
}
// 2^-e of a scale byte (1 to 253; 0 for the NaN byte, whose codes do not matter).
__device__ __forceinline__ float mx_inverse(uint32_t byte) {
  return byte == 0xffu ? 0.f : __uint_as_float((254u - byte) << 23);
}

// Instruction descriptor of the 4-bit block-scaled kinds: E2M1 operands
// (K-major), fp32 accumulation, K = 64; the scale type is UE8M0 (MXFP4) or UE4M3
// (NVFP4). sf picks the first scale byte of a TMEM word for both operands.
__host__ __device__ constexpr uint32_t idesc(int m, int n, int fmt, int sf) {
  return (static_cast<uint32_t>(sf) << 4)            // B scale-factor id
         | (1u << 7)                                 // A: E2M1
         | (1u << 10)                                // B: E2M1
         | (static_cast<uint32_t>(n >> 3) << 17)     // N / 8
         | ((fmt == kMx ? 1u : 0u) << 23)            // scale type: 1 = UE8M0, 0 = UE4M3
         | (static_cast<uint32_t>(m >> 4) << 24)     // M / 16
         | (static_cast<uint32_t>(sf) << 29);        // A scale-factor id
}

// D[tmem] (+)= (A * sfa) . (B * sfb)^T over 64 values of K.
template <int FMT>
__device__ __forceinline__ void umma(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t id, uint32_t sfa,
                                     uint32_t sfb, uint32_t accumulate) {
  if constexpr (FMT == kMx) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%5], [%6], p;\n\t}" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(id), "r"(accumulate), "r"(sfa), "r"(sfb)
        : "memory");
  } else {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%5], [%6], p;\n\t}" ::"r"(
            d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(id), "r"(accumulate), "r"(sfa), "r"(sfb)
        : "memory");
  }
}

// The same over a CTA pair, issued by the even CTA (M = 256: A rows and scales of
// each CTA's own half, half of B's rows and all of B's scales in each CTA).
template <int FMT>
__device__ __forceinline__ void umma_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t id, uint32_t sfa,
                                          uint32_t sfb, uint32_t accumulate) {
  if constexpr (FMT == kMx) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%5], [%6], p;\n\t}" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(id), "r"(accumulate), "r"(sfa), "r"(sfb)
        : "memory");
  } else {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%5], [%6], p;\n\t}" ::"r"(
            d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(id), "r"(accumulate), "r"(sfa), "r"(sfb)
        : "memory");
  }
}

// Scale copy to TMEM in both CTAs of a pair, each from its own shared memory.
__device__ __forceinline__ void tmem_cp_scales_pair(uint32_t taddr, uint64_t src_desc) {
  asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(src_desc) : "memory");
}

}  // namespace fp4
}  // namespace rx
