// Host interface of the microscaled 4-bit kernels (fp4_quant.cu, fp4_gemm.cu).
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace rx {
namespace fp4 {

enum Type : int { kBf16In = 0, kF16In = 1, kF32In = 2 };

struct QuantParams {
  const void* x;       // [rows, K], row stride ldx elements
  int64_t ldx;
  int64_t rows;        // rows of one part
  int64_t parts;       // the matrix has parts * rows rows
  int K;
  uint8_t* q;          // [parts * rows, ldq] bytes
  int64_t ldq;
  uint8_t* sf;         // [parts * ceil(rows / 128)][groups][512]
  int64_t groups;
  float* row_scale;    // NVFP4: [parts * rows]
};

// fmt: 1 MXFP4, 2 NVFP4; type: Type of x.
cudaError_t quantize(const QuantParams& p, int fmt, int type, cudaStream_t stream);

struct DequantParams {
  const uint8_t* q;
  int64_t ldq, rows, parts;
  int K;
  const uint8_t* sf;
  int64_t groups;
  const float* row_scale;
  void* out;           // [parts * rows, K], row stride ldo elements
  int64_t ldo;
};

cudaError_t dequantize(const DequantParams& p, int fmt, int type, cudaStream_t stream);

struct GemmParams {
  int M, N, K;         // N: output columns (per part)
  int m_tiles, n_tiles, k_stages;  // tiles of 256 rows x 256 columns (gated: 128)
  int gated, act;      // gated: B parts [gate; up], output act(g) * u
  int64_t groups;      // K groups of both scale arrays
  int a_tiles, b_tiles;  // scale row tiles of A and of one part of B
  const float* row_a;  // NVFP4 row factors [M], [parts * N]
  const float* row_b;
  const __nv_bfloat16* bias;      // [parts * N] or null
  const __nv_bfloat16* residual;  // [M, N] or null (plain only)
  int64_t ld_res;
  __nv_bfloat16* out;  // [M, N], or null with q_out
  int64_t ld_out;
  int vec;             // rows of out and residual are 16-byte aligned: `map_out` is valid
  uint8_t* q_out;      // gated MXFP4 output: codes [M, ld_q] and scales
  int64_t ld_q;
  uint8_t* q_sf;
  int64_t q_groups;
  int after_producer;  // the kernel before this one in the stream lets it start early; it waits for that one's end
  int* status;
  uint64_t timeout_ns;
};

// a, b: codes, boxes of 128 rows x 128 bytes. sf_a, sf_b: scales as 512-byte rows of 32-bit words, boxes of
// one stage's groups. out: 32 x 32 store map.
struct GemmMaps {
  CUtensorMap a, b, sf_a, sf_b, out;
};

cudaError_t gemm(const GemmMaps& maps, const GemmParams& p, int fmt, int sms, int device, cudaStream_t stream);

}  // namespace fp4
}  // namespace rx
