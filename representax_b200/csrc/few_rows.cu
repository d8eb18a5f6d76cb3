// y = x W^T for few token rows (1 to 64): a single query's tokens through a
// layer, in bf16 or with both operands in microscaled 4 bits, plain
// (+ bias + residual) or as the gated projection act(x Wg^T) * (x Wu^T).
//
// The work is reading W once, so everything serves memory parallelism. The
// roles of the operands are swapped: 128 weight rows are the M side of the
// tensor core's tile and the T tokens (padded to 16, 32 or 64) its N side, so no
// product is spent on 128-row padding of T and the output columns give many
// tiles. K is split over the CTAs of a cluster until the grid fills the GPU
// twice over; each CTA streams its share of W through a TMA ring (about 100 KB,
// two CTAs per SM) into fp32 TMEM accumulators. The partial sums meet in
// shared memory: after a cluster barrier every warp of the cluster takes
// groups of 32 outputs, reads the partials of all CTAs through distributed
// shared memory in rank order (so results do not depend on timing) and runs the
// epilogue.
//
// A gated tile has two accumulators, 128 gate rows and the 128 up rows of the
// same output columns, so one lane holds both operands of the product. With
// `q_out` the products leave as MXFP4: the 32 outputs of a warp's group are one
// scale block.
//
// Bound by HBM: floor = bytes of W / copy bandwidth. Every wait is bounded.
#include "few_rows.h"

#include <algorithm>

#include "fp4.cuh"
#include "gated_act.cuh"

namespace rx {
namespace few {

constexpr int kThreads = 192;  // producer, MMA issuer, four TMEM readers
constexpr int kWarps = kThreads / 32;
constexpr int kTileW = 128 * 128;  // 128 weight rows x 128 bytes
constexpr int kRingBytes = 100 * 1024;
constexpr int kPartLd = 132;       // floats per token row of the partial sums

template <int KIND, int PARTS, int NT>
struct Shape {
  static constexpr int kGroups = KIND == kBf16 ? 0 : fp4::groups_per_stage(KIND);
  static constexpr int kSfW = PARTS * kGroups * 512, kSfX = kGroups * 512;
  static constexpr int kTiles = PARTS * kTileW + NT * 128;
  static constexpr int kStage = kTiles + (kSfW + kSfX + 1023) / 1024 * 1024;
  static constexpr int kStages = kRingBytes / kStage;
  static constexpr int kPart = PARTS * NT * kPartLd * 4;
  static constexpr int kData = kStages * kStage > kPart ? kStages * kStage : kPart;
  static constexpr int kSmem = 1024 + kData + 256;
  // accumulators (read back 32 columns at a time, so the last one takes at least 32), then scales
  static constexpr int kAccCols = (PARTS - 1) * NT + (NT < 32 ? 32 : NT);
  static constexpr int kCols = kAccCols + (PARTS + 1) * kGroups * 4;
  static constexpr int kTmemCols = kCols <= 32 ? 32 : (kCols <= 64 ? 64 : (kCols <= 128 ? 128 : 256));
  static_assert(kStages >= 2 && kCols <= 256, "two CTAs per SM must fit");
};

__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

template <int KIND, int PARTS, int NT>
__global__ void __launch_bounds__(kThreads, 2)
    few_rows_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmW, const Params p) {
  using S = Shape<KIND, PARTS, NT>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(base + S::kData);
  uint64_t* empty = full + S::kStages;
  uint64_t* done = empty + S::kStages;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = warp_id(), lane = lane_id();
  const int rank = static_cast<int>(cluster_ctarank());
  const int splits = static_cast<int>(gridDim.y);  // the cluster spans the whole y dimension
  const int tile = blockIdx.x;
  const int kb0 = static_cast<int>(static_cast<int64_t>(p.k_blocks) * rank / splits);
  const int kb1 = static_cast<int>(static_cast<int64_t>(p.k_blocks) * (rank + 1) / splits);

  if (threadIdx.x == 0) {
    for (int s = 0; s < S::kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(done, 1);
    *abort_flag = 0;
    fence_mbarrier_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, S::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    if (lane == 0) {
      uint32_t issued = 0, parity = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        const int i = kb - kb0, s = i % S::kStages;
        const uint32_t phase = (i / S::kStages) & 1;
        if (*abort_flag || !mbar_wait(&empty[s], phase ^ 1, p.timeout_ns)) {
          report_status(p.status, kStatusTimeoutProducer);
          *abort_flag = 1;
          break;
        }
        mbar_arrive_expect_tx(&full[s], S::kTiles + S::kSfW + S::kSfX);
        uint8_t* dst = base + s * S::kStage;
        const int x = kb * (KIND == kBf16 ? 64 : 128);  // tensor-map column of the stage (elements of the map)
#pragma unroll
        for (int b = 0; b < PARTS; ++b) tma_load_2d(dst + b * kTileW, &tmW, &full[s], x, tile * 128 + b * p.N);
        tma_load_2d(dst + PARTS * kTileW, &tmX, &full[s], x, 0);
        if constexpr (KIND != kBf16) {
          uint8_t* sf = dst + S::kTiles;
          const int64_t row_tiles = (p.N + 127) >> 7;
          const int64_t g = static_cast<int64_t>(kb) * S::kGroups;
#pragma unroll
          for (int b = 0; b < PARTS; ++b)
            bulk_load(sf + b * S::kGroups * 512, p.sf_w + ((tile + b * row_tiles) * p.groups + g) * 512, S::kGroups * 512,
                      &full[s]);
          bulk_load(sf + S::kSfW, p.sf_x + g * 512, S::kSfX, &full[s]);
        }
        issued |= 1u << s;
        parity = (parity & ~(1u << s)) | (phase << s);
      }
      // leave no copy in flight into memory that is about to be reused
      for (int s = 0; s < S::kStages; ++s)
        if (((issued >> s) & 1u) && !mbar_wait(&full[s], (parity >> s) & 1u, p.timeout_ns))
          report_status(p.status, kStatusTimeoutDrain);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    if (lane == 0) {
      const uint32_t sf_cols = tmem_base + S::kAccCols;
      bool issued_any = false;
      for (int kb = kb0; kb < kb1; ++kb) {
        const int i = kb - kb0, s = i % S::kStages;
        if (*abort_flag || !mbar_wait(&full[s], (i / S::kStages) & 1, p.timeout_ns)) {
          report_status(p.status, kStatusTimeoutMma);
          *abort_flag = 1;
          break;
        }
        tc_fence_after();
        const uint32_t w = smem_u32(base + s * S::kStage), x = w + PARTS * kTileW;
        if constexpr (KIND == kBf16) {
          constexpr uint32_t IDESC = idesc_bf16_f32(128, NT, false, false);
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
#pragma unroll
            for (int b = 0; b < PARTS; ++b)
              umma_f16_ss(tmem_base + b * NT, smem_desc_sw128(w + b * kTileW + kk * 32, 16, 1024),
                          smem_desc_sw128(x + kk * 32, 16, 1024), IDESC, (i > 0 || kk > 0) ? 1u : 0u);
        } else {
          const uint32_t sf = w + S::kTiles;
#pragma unroll
          for (int a = 0; a < (PARTS + 1) * S::kGroups; ++a)
            tmem_cp_32x128b_warpx4(sf_cols + 4 * a, smem_desc_plain(sf + a * 512, 512, 128));
          // 64-value steps past K would multiply zeros by scales that nothing defines
          const int steps = min(4, (p.K - kb * fp4::kStageK + 63) / 64);
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) {
            if (kk < steps) {
              const int atom = KIND == kMxfp4 ? kk >> 1 : kk;
              const uint32_t id = KIND == kMxfp4 ? 2u * (kk & 1) : 0u;
#pragma unroll
              for (int b = 0; b < PARTS; ++b)
                fp4::umma<KIND>(tmem_base + b * NT, smem_desc_sw128(w + b * kTileW + kk * 32, 16, 1024),
                                smem_desc_sw128(x + kk * 32, 16, 1024), fp4::idesc(128, NT, KIND, id),
                                (sf_cols + 4 * (b * S::kGroups + atom)) | (id << 30),
                                (sf_cols + 4 * (PARTS * S::kGroups + atom)) | (id << 30), (i > 0 || kk > 0) ? 1u : 0u);
            }
          }
        }
        issued_any = true;
        umma_commit(&empty[s]);
      }
      // one arrival even without work (fewer K blocks than CTAs cannot happen, an abort can)
      umma_commit(done);
      if (issued_any && !mbar_wait(done, 0, p.timeout_ns)) report_status(p.status, kStatusTimeoutDrain);
    }
  }
  __syncthreads();  // every MMA has completed and no copy is in flight: the ring may be reused
  float* part = reinterpret_cast<float*>(base);
  if (warp >= 2) {
    // partial sums of weight row `quad * 32 + lane` for every token
    const int quad = warp & 3;
    tc_fence_after();
#pragma unroll
    for (int b = 0; b < PARTS; ++b) {
#pragma unroll
      for (int c = 0; c < (NT + 31) / 32; ++c) {
        uint32_t r[32];
        tmem_ld_32x32b_x32(tmem_base + (static_cast<uint32_t>(quad * 32) << 16) + b * NT + c * 32, r);
        tmem_ld_wait();
#pragma unroll
        for (int t = 0; t < (NT < 32 ? NT : 32); ++t)
          if (c * 32 + t < p.T)
            part[(b * NT + c * 32 + t) * kPartLd + quad * 32 + lane] = __uint_as_float(r[t]);
      }
    }
  }
  cluster_sync_all();

  // ------------------------------------------------------------ reduction and epilogue
  // Group g: token t = g / 4, the 32 output columns (g % 4) of the tile.
  const uint32_t part_addr = smem_u32(part);
  const bool aborted = *abort_flag != 0;
  if (!aborted) {
    for (int g = rank * kWarps + warp; g < p.T * 4; g += splits * kWarps) {
      const int t = g >> 2, col = (g & 3) * 32 + lane;
      const int n = tile * 128 + col;
      float v[PARTS];
#pragma unroll
      for (int b = 0; b < PARTS; ++b) v[b] = 0.f;
      for (int r = 0; r < splits; ++r) {
        const uint32_t peer = mapa_shared(part_addr, static_cast<uint32_t>(r));
#pragma unroll
        for (int b = 0; b < PARTS; ++b) v[b] += ld_cluster_f32(peer + ((b * NT + t) * kPartLd + col) * 4);
      }
      const bool live = n < p.N;
      if (live) {
#pragma unroll
        for (int b = 0; b < PARTS; ++b) {
          if constexpr (KIND == kNvfp4) v[b] *= p.row_x[t] * p.row_w[static_cast<int64_t>(b) * p.N + n];
          if (p.bias != nullptr) v[b] += __bfloat162float(p.bias[static_cast<int64_t>(b) * p.N + n]);
        }
      }
      float y = v[0];
      if constexpr (PARTS == 2) y = gated::act_value(v[0], p.act) * v[1];
      if constexpr (PARTS == 1)
        if (live && p.residual != nullptr) y += __bfloat162float(p.residual[static_cast<int64_t>(t) * p.ld_res + n]);
      if constexpr (PARTS == 2 && KIND == kMxfp4) {
        if (p.q_out != nullptr) {
          if (!live) y = 0.f;
          uint32_t top = __float_as_uint(y) & 0x7fffffffu;
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
          const uint32_t byte = fp4::mx_scale_byte(top);
          y *= fp4::mx_inverse(byte);
          float w8[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) w8[j] = __shfl_sync(0xffffffffu, y, (lane & 24) + j);
          const uint32_t codes = fp4::pack8(w8);
          const int64_t at = static_cast<int64_t>(t) * p.ld_q + (n >> 1);
          if ((lane & 7) == 0 && (n >> 1) + 4 <= p.ld_q) *reinterpret_cast<uint32_t*>(p.q_out + at) = codes;
          if (lane == 0) p.q_sf[fp4::scale_offset(t, n >> 5, p.q_groups)] = static_cast<uint8_t>(byte);
          continue;
        }
      }
      if (live) p.out[static_cast<int64_t>(t) * p.ld_out + n] = __float2bfloat16_rn(y);
    }
  }
  tc_fence_before();
  cluster_sync_all();  // no CTA leaves while another still reads its partial sums
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem_base, S::kTmemCols);
}

template <int KIND, int PARTS, int NT>
cudaError_t launch_shape(const CUtensorMap& map_x, const CUtensorMap& map_w, const Params& p, int sms, int device,
                         cudaStream_t stream) {
  using S = Shape<KIND, PARTS, NT>;
  auto kern = few_rows_kernel<KIND, PARTS, NT>;
  static bool configured[64] = {false};
  if (device < 0 || device >= 64 || !configured[device]) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem);
    if (e != cudaSuccess) return e;
    if (device >= 0 && device < 64) configured[device] = true;
  }
  // as many K splits as two CTAs per SM can hold at once, each with at least two stages of work
  const int tiles = (p.N + 127) / 128;
  const int splits = std::max(1, std::min({8, 2 * sms / tiles, p.k_blocks / 2}));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(tiles, splits);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = S::kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 1;
  attr[0].val.clusterDim.y = splits;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, map_x, map_w, p);
}

template <int KIND, int PARTS>
cudaError_t launch_parts(const CUtensorMap& mx, const CUtensorMap& mw, const Params& p, int sms, int device,
                         cudaStream_t stream) {
  switch (tile_rows(p.T)) {
    case 16: return launch_shape<KIND, PARTS, 16>(mx, mw, p, sms, device, stream);
    case 32: return launch_shape<KIND, PARTS, 32>(mx, mw, p, sms, device, stream);
    default: return launch_shape<KIND, PARTS, 64>(mx, mw, p, sms, device, stream);
  }
}

template <int KIND>
cudaError_t launch_kind(const CUtensorMap& mx, const CUtensorMap& mw, const Params& p, int sms, int device,
                        cudaStream_t stream) {
  return p.gated ? launch_parts<KIND, 2>(mx, mw, p, sms, device, stream)
                 : launch_parts<KIND, 1>(mx, mw, p, sms, device, stream);
}

cudaError_t launch(int kind, const CUtensorMap& map_x, const CUtensorMap& map_w, const Params& p, int sms, int device,
                   cudaStream_t stream) {
  switch (kind) {
    case kBf16: return launch_kind<kBf16>(map_x, map_w, p, sms, device, stream);
    case kMxfp4: return launch_kind<kMxfp4>(map_x, map_w, p, sms, device, stream);
    default: return launch_kind<kNvfp4>(map_x, map_w, p, sms, device, stream);
  }
}

}  // namespace few
}  // namespace rx
