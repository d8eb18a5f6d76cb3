// Host interface of the kernels for few token rows (few_rows.cu).
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace rx {
namespace few {

enum Kind : int { kBf16 = 0, kMxfp4 = 1, kNvfp4 = 2 };

// Which products run here rather than on the GEMMs' CTA pairs, whose 256 x 256 tiles (74 pairs make a wave) leave most
// of the GPU idle when there are few of them, while their time grows with K. Measured on both sides, us here / there,
// the operands of four calls in turn (4-bit with the quantiser):
//   up to 16 rows   bf16 x 2304, K 768 5.2 / 7.6, x 12288, K 2048 17.8 / 18.1; MXFP4 x 2304, K 768 6.8 / 8.0, x 12288
//                   8.0 / 9.9, one row x 24576 10.4 / 16.9, NVFP4 12.1 / 17.9
//   bf16, 17 to 64  [64, 768] x 2304 6.7 / 9.4, [64, 2048] x 12288 (48 tiles) 16.0 / 19.5, [64, 1024] x 16384 (64) 13.3 /
//                   13.2, [64, 2048] x 24576 (96) 26.6 / 23.4
//   bf16, more      a long K for few tiles: [128, 2304] x 768 (3 tiles, 36 stages) 8.0 / 17.9, [256, 6144] x 2048 (8, 96) 17.4 / 33.1,
//                   [300, 3416] x 1280 (10, 54) 14.6 / 25.9, [384, 6144] x 2048 (16, 96) 27.2 / 33.1, [512, 1152] x 768 (6, 18) 10.7 /
//                   10.8, [768, 2816] x 1024 (12, 44) 19.5 / 18.3, [700, 1152] x 768 (9, 18) 14.8 / 10.6, [384, 1024] x 2048 (16, 16)
//                   15.8 / 10.2, [700, 6144] x 2048 (24, 96) 34.2 / 33.3, [256, 320] x 256 (1, 5) 9.0 / 6.7
//   4-bit, 17 to 64 MXFP4 [64, 1024] x 6144 (24 tiles, 4 stages) 7.7 / 8.5, [64, 768] x 2304 (9, 3) 9.5 / 8.0, NVFP4 11.1 / 8.5;
//                   [32, 768] x 2304 7.8 / 8.0 and 8.8 / 8.5; [32, 2048] x 12288 (48, 8) 9.0 / 10.0 and 10.7 / 11.0, 64 rows 10.6 / 10.2
//   4-bit, more     MXFP4 [128, 6144] x 2048 (8, 24) 11.4 / 15.0, [256, 2048] x 2048 (8, 8) 9.0 / 9.9, [512, 4096] x 1024 (8, 16) 13.5 /
//                   12.6, [128, 1152] x 768 (3, 5) 10.5 / 8.7, [384, 6144] x 2048 (16, 24) 18.4 / 15.3; NVFP4 alike
//   bf16 gated      [32, 2048] x 2 x 6144 16.3 / 17.4, [33, 2048] 21.5 / 17.4, [64, 2048] x 2 x 2560 12.7 / 15.6, [64, 1024] x 2 x 2304
//                   10.9 / 10.6, [64, 768] x 2 x 1152 7.3 / 9.4, [64, 1024] x 2 x 2816 11.2 / 10.7
//   4-bit gated     (whole block) MXFP4 [16, 2048] x 2 x 6144 13.2 / 17.8, [32, 2048] 15.2 / 18.0, [64, 2048] 20.2 / 21.0,
//                   [32, 768] x 2 x 1152 13.7 / 13.2, [64, 768] 18.5 / 14.3; NVFP4 alike
// `stages`: pipeline stages along K (64 bf16 or 256 4-bit values).
inline bool takes(int kind, int64_t rows, int64_t cols, int64_t stages, bool gated) {
  if (gated) return rows <= 32 || (kind == kBf16 && rows <= 64 && cols <= 2560);
  if (rows <= 16) return true;
  const int64_t tiles = (rows + 255) / 256 * ((cols + 255) / 256);
  if (kind == kBf16) return rows <= 64 ? tiles <= 48 : tiles <= 16 && stages >= 8 && stages >= 3 * tiles;
  if (rows <= 32) return tiles <= 48;
  return rows <= 64 ? tiles <= 24 && stages >= 4 : tiles <= 8 && stages >= 8;
}

struct Params {
  int T, N, K;        // token rows, output columns (per part), contraction
  int k_blocks;       // pipeline stages along K (64 bf16 or 256 4-bit values each)
  int gated;          // 1: weight parts [gate; up], output act(g) * u; 0: one part, plain output
  int act;
  const __nv_bfloat16* bias;      // [parts * N] or null
  const __nv_bfloat16* residual;  // [T, N] or null (plain only)
  int64_t ld_res;
  __nv_bfloat16* out;             // [T, N], or null with q_out
  int64_t ld_out;
  int vec;                        // rows of out are 8-byte aligned
  // 4-bit operands
  const uint8_t* sf_x;
  const uint8_t* sf_w;
  int64_t groups;                 // K groups of both scale arrays
  const float* row_x;             // NVFP4 row factors [T] and [parts * N]
  const float* row_w;
  // gated MXFP4 output: codes [T, ld_q] and scales of the next layer's operand
  uint8_t* q_out;
  int64_t ld_q;
  uint8_t* q_sf;
  int64_t q_groups;
  // The kernel before this one in the stream writes x (and nothing else that this one reads) and
  // lets dependents start early: stream W before it has finished.
  int after_producer;
  int* status;
  uint64_t timeout_ns;
};

// Rows of a token tile for T token rows.
inline int tile_rows(int64_t t) { return t <= 16 ? 16 : (t <= 32 ? 32 : (t <= 64 ? 64 : 128)); }

// `map_x`: boxes of tile_rows(T) rows x 128 bytes; `map_w`: boxes of 128 rows x 128 bytes.
cudaError_t launch(int kind, const CUtensorMap& map_x, const CUtensorMap& map_w, const Params& p, int sms, int device,
                   cudaStream_t stream);

}  // namespace few
}  // namespace rx
