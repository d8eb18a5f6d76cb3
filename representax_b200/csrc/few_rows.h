// Host interface of the kernels for few token rows (few_rows.cu).
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace rx {
namespace few {

// Which products run here rather than on the GEMMs' CTA pairs, whose 256 x 256 tiles leave most of the GPU idle
// when there are few of them (74 pairs make a wave) while K is long. Measured on both sides, us here / there:
//   bf16 plain  [128, 6144] x 2048 outputs 16 / 35, [512, 2816] x 1024 14 / 21, [384, 6144] x 2048 29 / 36
//   MXFP4       [128, 6144] x 2048 10.5 / 15, [128, 1152] x 768 10.2 / 9.2, [128, 768] x 2304 12 / 6.7
//   NVFP4       [128, 6144] x 2048 11 / 19, [256, 768] x 2304 12.9 / 9.6; one row x 12288, K 2048: 8.9 / 13
//   bf16 gated  [32, 2048] x 2 x 6144 16 / 17, [64, 2048] 24 / 17, [64, 768] x 2 x 1152 7.0 / 9.2
// `stages`: pipeline stages along K (64 bf16 or 256 4-bit values).
inline bool takes(int64_t rows, int64_t cols, int64_t stages, bool gated) {
  if (gated) return rows <= 32;
  const int64_t tiles = (rows + 255) / 256 * ((cols + 255) / 256);
  return rows <= 16 || (rows <= 64 && tiles <= 24) || (tiles <= 12 && stages >= 8);
}

enum Kind : int { kBf16 = 0, kMxfp4 = 1, kNvfp4 = 2 };

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
