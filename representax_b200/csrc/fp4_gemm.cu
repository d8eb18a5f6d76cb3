// Products of microscaled 4-bit operands on tcgen05 (kind::mxf4 and
// kind::mxf4nvf4, block scales applied by the tensor core):
//
//   y = A B^T (row factors) (+ bias) (+ residual)            one part
//   y = act(A Bg^T + bg) * (A Bu^T + bu)                     two parts [gate; up]
//
// with A [M, K], B [parts * N, K] as codes and scales (fp4.cuh), fp32
// accumulation, bf16 output; the gated product may leave as the MXFP4
// operand of the next layer: the 32 columns that a thread holds of its row are
// one scale block, so the fp32 product is quantised without a trip through
// memory or through bf16.
//
// Persistent, one CTA per SM: producer warp (TMA of a 128 x 256 A tile and two
// 128 x 256 B tiles per stage, 48 KB, and the stage's scales by bulk copies), one
// issuing thread (scales to TMEM, then four K = 64 MMAs of 128 x 256), eight
// epilogue warps. The two B tiles are adjacent columns, or the gate and up
// rows of the same 128 columns. The accumulator takes 256 of the 512 TMEM
// columns and the scales of all stages share the rest; instead of a second
// accumulator, an epilogue thread takes its 128 values into registers and
// frees the accumulator before it computes or stores, so the tensor core waits for a
// TMEM read only.
#include "fp4.h"

#include <algorithm>

#include "fp4.cuh"
#include "gated_act.cuh"

namespace rx {
namespace fp4 {

constexpr int kTile = 128 * 128;   // 128 rows x 256 codes
constexpr int kTiles = 3 * kTile;
constexpr int kGemmStages = 4;
constexpr int kEpiWarps = 8;
constexpr int kGemmThreads = 32 * (2 + kEpiWarps);

template <int FMT>
struct GemmShape {
  static constexpr int kGroups = groups_per_stage(FMT);
  static constexpr int kSf = 3 * kGroups * 512;
  static constexpr size_t kSmem = 1024 + kGemmStages * (kTiles + kSf) + 256;
  static constexpr int kSfCols = 3 * kGroups * 4;  // TMEM columns of a stage's scales
  static_assert(256 + kGemmStages * kSfCols <= 512 && kSmem <= 232448, "does not fit");
};

// 32 consecutive outputs of row m from column n.
__device__ __forceinline__ void store32(const GemmParams& p, int64_t m, int n, const float (&v)[32]) {
  __nv_bfloat16* dst = p.out + m * p.ld_out + n;
  if (p.vec && n + 32 <= p.N) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      uint4 w;
      __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&w);
#pragma unroll
      for (int j = 0; j < 4; ++j) h[j] = __floats2bfloat162_rn(v[8 * q + 2 * j], v[8 * q + 2 * j + 1]);
      reinterpret_cast<uint4*>(dst)[q] = w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (n + i < p.N) dst[i] = __float2bfloat16_rn(v[i]);
  }
}

// v += src[0..32), as far as column n + i < N.
__device__ __forceinline__ void add32(const __nv_bfloat16* src, bool vec, int n, int N, float (&v)[32]) {
  if (vec && n + 32 <= N) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const uint4 w = reinterpret_cast<const uint4*>(src)[q];
      const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&w);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 f = __bfloat1622float2(h[j]);
        v[8 * q + 2 * j] += f.x;
        v[8 * q + 2 * j + 1] += f.y;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (n + i < N) v[i] += __bfloat162float(src[i]);
  }
}

// Row factors and bias of 32 accumulators (columns n.. of B's part at row `part0`).
template <int FMT>
__device__ __forceinline__ void finish32(const GemmParams& p, float row_a, int64_t part0, int n, const uint32_t (&r)[32],
                                         float (&v)[32]) {
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
  if constexpr (FMT == kNv) {
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (n + i < p.N) v[i] *= row_a * p.row_b[part0 + n + i];
  }
  if (p.bias != nullptr) add32(p.bias + part0 + n, p.vec, n, p.N, v);
}

template <int FMT, bool GATED>
__global__ void __launch_bounds__(kGemmThreads, 1)
    fp4_gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const GemmParams p) {
  using S = GemmShape<FMT>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sf_base = base + kGemmStages * kTiles;
  uint64_t* full = reinterpret_cast<uint64_t*>(sf_base + kGemmStages * S::kSf);
  uint64_t* empty = full + kGemmStages;
  uint64_t* tfull = empty + kGemmStages;
  uint64_t* tempty = tfull + 1;
  uint64_t* drain = tempty + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = warp_id(), lane = lane_id();
  constexpr int kTileN = GATED ? 128 : 256;  // output columns of a tile

  if (threadIdx.x == 0) {
    for (int s = 0; s < kGemmStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(tfull, 1);
    mbar_init(tempty, kEpiWarps);
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_mbarrier_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const int num_units = p.m_tiles * p.n_tiles;
  const int b_tiles = (p.N + 127) >> 7;  // scale row tiles of one part of B

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    if (lane == 0) {
      tma_prefetch_map(&tmA);
      tma_prefetch_map(&tmB);
      int stage = 0;
      uint32_t phase = 0, issued = 0, parity = 0;
      bool ok = true;
      for (int u = blockIdx.x; ok && u < num_units; u += gridDim.x) {
        const int mt = u % p.m_tiles, nt = u / p.m_tiles;
        // rows and scale tiles of the two B tiles (a second tile past the end reads the last one's scales)
        const int row0 = nt * kTileN, row1 = GATED ? row0 + p.N : row0 + 128;
        const int64_t t0 = row0 >> 7, t1 = GATED ? t0 + b_tiles : min(static_cast<int>(t0) + 1, b_tiles - 1);
        for (int ks = 0; ks < p.k_stages; ++ks) {
          if (*abort_flag || !mbar_wait(&empty[stage], phase ^ 1, p.timeout_ns)) {
            report_status(p.status, kStatusTimeoutProducer);
            *abort_flag = 1;
            ok = false;
            break;
          }
          mbar_arrive_expect_tx(&full[stage], kTiles + S::kSf);
          uint8_t* tiles = base + stage * kTiles;
          uint8_t* sf = sf_base + stage * S::kSf;
          constexpr int kBytes = S::kGroups * 512;
          const int64_t g = static_cast<int64_t>(ks) * S::kGroups;
          tma_load_2d(tiles, &tmA, &full[stage], ks * 128, mt * 128);
          tma_load_2d(tiles + kTile, &tmB, &full[stage], ks * 128, row0);
          tma_load_2d(tiles + 2 * kTile, &tmB, &full[stage], ks * 128, row1);
          bulk_load(sf, p.sf_a + (mt * p.groups + g) * 512, kBytes, &full[stage]);
          bulk_load(sf + kBytes, p.sf_b + (t0 * p.groups + g) * 512, kBytes, &full[stage]);
          bulk_load(sf + 2 * kBytes, p.sf_b + (t1 * p.groups + g) * 512, kBytes, &full[stage]);
          issued |= 1u << stage;
          parity = (parity & ~(1u << stage)) | (phase << stage);
          if (++stage == kGemmStages) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
      // leave no copy in flight into shared memory that is about to be released
      for (int s = 0; s < kGemmStages; ++s)
        if (((issued >> s) & 1u) && !mbar_wait(&full[s], (parity >> s) & 1u, p.timeout_ns))
          report_status(p.status, kStatusTimeoutDrain);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    if (lane == 0) {
      int stage = 0, local = 0;
      uint32_t phase = 0;
      bool ok = true, issued_any = false;
      for (int u = blockIdx.x; ok && u < num_units; u += gridDim.x, ++local) {
        if (*abort_flag || !mbar_wait(tempty, (local & 1) ^ 1, p.timeout_ns)) {
          report_status(p.status, kStatusTimeoutMma);
          *abort_flag = 1;
          break;
        }
        tc_fence_after();
        for (int ks = 0; ks < p.k_stages; ++ks) {
          if (*abort_flag || !mbar_wait(&full[stage], phase, p.timeout_ns)) {
            report_status(p.status, kStatusTimeoutMma);
            *abort_flag = 1;
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t a = smem_u32(base + stage * kTiles), b = a + kTile;
          const uint32_t sf = smem_u32(sf_base + stage * S::kSf);
          const uint32_t sfa = tmem_base + 256 + stage * S::kSfCols, sfb = sfa + 4 * S::kGroups;
#pragma unroll
          for (int j = 0; j < S::kGroups; ++j) {
            tmem_cp_32x128b_warpx4(sfa + 4 * j, smem_desc_plain(sf + j * 512, 512, 128));
            tmem_cp_32x128b_warpx4(sfb + 8 * j, smem_desc_plain(sf + (S::kGroups + j) * 512, 512, 128));
            tmem_cp_32x128b_warpx4(sfb + 8 * j + 4, smem_desc_plain(sf + (2 * S::kGroups + j) * 512, 512, 128));
          }
          // 64-value steps past K would multiply zeros by scales that nothing defines
          const int steps = min(4, (p.K - ks * kStageK + 63) / 64);
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) {
            if (kk < steps) {
              const int atom = FMT == kMx ? kk >> 1 : kk;
              const uint32_t id = FMT == kMx ? 2u * (kk & 1) : 0u;
              umma<FMT>(tmem_base, smem_desc_sw128(a + kk * 32, 16, 1024), smem_desc_sw128(b + kk * 32, 16, 1024),
                        idesc(128, 256, FMT, id), (sfa + 4 * atom) | (id << 30), (sfb + 8 * atom) | (id << 30),
                        (ks > 0 || kk > 0) ? 1u : 0u);
            }
          }
          issued_any = true;
          umma_commit(&empty[stage]);
          if (++stage == kGemmStages) {
            stage = 0;
            phase ^= 1;
          }
        }
        if (!ok) break;
        umma_commit(tfull);
      }
      if (issued_any) {
        umma_commit(drain);
        if (!mbar_wait(drain, 0, p.timeout_ns)) report_status(p.status, kStatusTimeoutDrain);
      }
    }
  } else {
    // ------------------------------------------------------------ epilogue
    const int quad = warp & 3, half = (warp - 2) >> 2;
    int local = 0;
    for (int u = blockIdx.x; u < num_units; u += gridDim.x, ++local) {
      const int mt = u % p.m_tiles, nt = u / p.m_tiles;
      bool ok = (*abort_flag == 0) && mbar_wait(tfull, local & 1, p.timeout_ns);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) {
        if (lane == 0) report_status(p.status, kStatusTimeoutEpilogue);
        *abort_flag = 1;
        break;
      }
      tc_fence_after();
      // plain: 128 columns of this half; gated: 64 gate columns, then the 64 up columns of the same outputs
      const uint32_t t_row = tmem_base + (static_cast<uint32_t>(quad * 32) << 16);
      uint32_t r[4][32];
#pragma unroll
      for (int c = 0; c < 4; ++c)
        tmem_ld_32x32b_x32(t_row + (GATED ? half * 64 + (c & 1) * 32 + (c >> 1) * 128 : half * 128 + c * 32), r[c]);
      tmem_ld_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(tempty);
      const int64_t m = static_cast<int64_t>(mt) * 128 + quad * 32 + lane;
      if (m >= p.M) continue;
      const float row_a = FMT == kNv ? p.row_a[m] : 1.f;
      if constexpr (GATED) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int n = nt * kTileN + half * 64 + c * 32;
          // (a quantised output also defines the blocks past N of the tile)
          if (n >= p.N && p.q_out == nullptr) continue;
          float g[32], v[32];
          finish32<FMT>(p, row_a, 0, n, r[c], g);
          finish32<FMT>(p, row_a, p.N, n, r[2 + c], v);
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = n + i < p.N ? v[i] * gated::act_value(g[i], p.act) : 0.f;
          if (FMT == kMx && p.q_out != nullptr) {
            uint32_t top = 0;
#pragma unroll
            for (int i = 0; i < 32; ++i) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
            const uint32_t byte = mx_scale_byte(top);
            const float inv = mx_inverse(byte);
            uint32_t codes[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              float w[8];
#pragma unroll
              for (int i = 0; i < 8; ++i) w[i] = v[8 * q + i] * inv;
              codes[q] = pack8(w);
            }
            if ((n >> 1) < p.ld_q)
              *reinterpret_cast<uint4*>(p.q_out + m * p.ld_q + (n >> 1)) = make_uint4(codes[0], codes[1], codes[2], codes[3]);
            p.q_sf[scale_offset(m, n >> 5, p.q_groups)] = static_cast<uint8_t>(byte);
          } else {
            store32(p, m, n, v);
          }
        }
      } else {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int n = nt * kTileN + half * 128 + c * 32;
          if (n >= p.N) continue;
          float v[32];
          finish32<FMT>(p, row_a, 0, n, r[c], v);
          if (p.residual != nullptr) add32(p.residual + m * p.ld_res + n, p.vec, n, p.N, v);
          store32(p, m, n, v);
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem_base, 512);
}

template <int FMT, bool GATED>
cudaError_t launch(const CUtensorMap& ta, const CUtensorMap& tb, const GemmParams& p, int sms, int device,
                   cudaStream_t stream) {
  auto kern = fp4_gemm_kernel<FMT, GATED>;
  constexpr size_t smem = GemmShape<FMT>::kSmem;
  static bool configured[64] = {false};
  if (device < 0 || device >= 64 || !configured[device]) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    if (e != cudaSuccess) return e;
    if (device >= 0 && device < 64) configured[device] = true;
  }
  kern<<<std::min(p.m_tiles * p.n_tiles, sms), kGemmThreads, smem, stream>>>(ta, tb, p);
  return cudaGetLastError();
}

cudaError_t gemm(const CUtensorMap& map_a, const CUtensorMap& map_b, const GemmParams& p, int fmt, int sms, int device,
                 cudaStream_t stream) {
  if (fmt == kMx)
    return p.gated ? launch<kMx, true>(map_a, map_b, p, sms, device, stream)
                   : launch<kMx, false>(map_a, map_b, p, sms, device, stream);
  return p.gated ? launch<kNv, true>(map_a, map_b, p, sms, device, stream)
                 : launch<kNv, false>(map_a, map_b, p, sms, device, stream);
}

}  // namespace fp4
}  // namespace rx
