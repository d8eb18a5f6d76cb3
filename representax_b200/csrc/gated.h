// Host interface of the gated feed-forward kernels (gated.cu).
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace rx {
namespace gated {

// Forward; forward that keeps what the backward reads; backward (dz).
enum Mode : int { kForward = 0, kForwardSave = 1, kBackward = 2 };

struct Params {
  int M, N, K;  // N: columns of h (forward) or of dh (backward)
  int m_tiles, n_tiles, num_units;
  int act;
  const __nv_bfloat16* bias;  // forward: [2 N] (gate, up) or null
  __nv_bfloat16* out[2];      // h (forward) or the two halves of dz, [M, N]
  int64_t ld_out;
  uint4* saved;               // [ceil(M / 32)][ceil(N / 32)] tiles of 32 x 32 fp16: b, then a (4 KB)
  uint16_t* exps;             // [the same tiles][32]: low byte the block exponent of b, high byte that of a
  float* partial;             // backward: [ceil(M / 32)][2 N] column sums of 32 rows of dz, or null
  int* status;
  uint64_t timeout_ns;
};

// a: boxes of 128 rows x 64; b: 128 x 64 (forward, K-major) or 64 x 64 (backward, MN-major).
struct Maps {
  CUtensorMap a, b;
};

// Column sums of `rows` rows of partial sums [rows][cols], in a fixed order: added to acc (fp32), or written
// to out (bf16).
cudaError_t sum_partials(const float* partial, int64_t rows, int64_t cols, float* acc, __nv_bfloat16* out,
                         cudaStream_t stream);

cudaError_t launch(int mode, const Maps& maps, const Params& p, int sms, int device, cudaStream_t stream);

}  // namespace gated
}  // namespace rx
