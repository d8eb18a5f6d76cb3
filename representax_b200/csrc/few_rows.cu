// y = x W^T for few token rows: a single query's tokens through a layer, in bf16 or with both operands in microscaled 4 bits, plain
// (+ bias + residual) or as the gated projection act(x Wg^T) * (x Wu^T).
//
// The work is reading W once, so everything serves memory parallelism. The
// roles of the operands are swapped: 128 weight rows are the M side of the
// tensor core's tile and the T tokens (in tiles of 16, 32, 64 or 128) its N side,
// so little is spent on padding of T and the output columns give many tiles. K is split over the CTAs of a cluster until the grid fills the GPU
// twice over; each CTA streams its share of W through a TMA ring
// (two or three CTAs per SM) into fp32 TMEM accumulators. The partial sums meet in
// shared memory: after a cluster barrier every warp of the cluster takes
// a token's 128 outputs, adds the partials of all CTAs, read through
// distributed shared memory, in rank order (so results do not depend on timing)
// and runs the epilogue.
//
// A gated tile has two accumulators, 128 gate rows and the 128 up rows of the
// same output columns, so one lane holds both operands of the product. With
// `q_out` the products leave as MXFP4, eight lanes to a scale block.
//
// W does not depend on the kernel that produces x. Where the host says that
// kernel is the one just before (`after_producer`), this one is launched
// early: it fills its ring with W and waits for x only then.
//
// Bound by HBM: floor = bytes of W / copy bandwidth, and by the 4 us that a launch, the
// first bytes, the cluster barriers and the reduction take whatever the size. One
// token, weights of several layers in turn: K 2048, [6144 gate; 6144 up] bf16 (50 MB,
// floor 7.8 us) 11.9 us; down projection of it (25 MB, floor 3.9 us) 9.0 us; the two in a
// row 19.4 us (14.6 when one layer's weights stay in L2); NVFP4 12288 outputs (14 MB) with
// the quantiser 8.8 us. 128 tokens through the down projection 15.4 us against 36.5 us of
// the 256-row GEMM, which has only 8 tiles there. Every wait is bounded.
#include "few_rows.h"

#include <algorithm>

#include "elect.cuh"
#include "fp4.cuh"
#include "gated_act.cuh"

namespace rx {
namespace few {

constexpr int kThreads = 192;  // producer, MMA issuer, four TMEM readers
constexpr int kWarps = kThreads / 32;
constexpr int kTileW = 128 * 128;  // 128 weight rows x 128 bytes
constexpr int kPartLd = 132;       // floats per token row of the partial sums

template <int KIND, int PARTS, int NT>
struct Shape {
  static constexpr int kGroups = KIND == kBf16 ? 0 : fp4::groups_per_stage(KIND);
  static constexpr int kSfW = PARTS * kGroups * 512, kSfX = kGroups * 512;
  static constexpr int kTiles = PARTS * kTileW + NT * 128;
  static constexpr int kStage = kTiles + (kSfW + kSfX + 1023) / 1024 * 1024;
  // Ring: enough bytes in flight to cover the latency, little enough that three CTAs fit an SM. At one token
  // (K 2048, 12288 outputs, NVFP4) 104 KB took 9.0 us and 72 KB 6.6 us; the plain bf16 stream, which starts
  // under the gated kernel's tail, gained from 90 KB (block of one token 20.3 -> 19.5 us), 128-token tiles from a
  // third stage (128 tokens, K 6144: 18.6 -> 16.8 us).
  static constexpr int kRingBytes = (NT == 128 ? 104 : (KIND == kBf16 && PARTS == 1 ? 90 : 72)) * 1024;
  static constexpr int kStages = kRingBytes / kStage < 2 ? 2 : kRingBytes / kStage;
  static constexpr int kPart = PARTS * NT * kPartLd * 4;
  static constexpr int kData = kStages * kStage > kPart ? kStages * kStage : kPart;
  static constexpr int kSmem = 1024 + kData + 256;
  // accumulators (read back 32 columns at a time, so the last one takes at least 32), then scales
  static constexpr int kAccCols = (PARTS - 1) * NT + (NT < 32 ? 32 : NT);
  static constexpr int kCols = kAccCols + (PARTS + 1) * kGroups * 4;
  static constexpr int kTmemCols = kCols <= 32 ? 32 : (kCols <= 64 ? 64 : (kCols <= 128 ? 128 : 256));
  static_assert(kCols <= 256 && 2 * kSmem <= 220 * 1024, "two CTAs per SM must fit");
};

// Four consecutive floats of another CTA's shared memory.
__device__ __forceinline__ float4 ld_cluster_f4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr));
  return v;
}

template <int KIND, int PARTS, int NT>
__global__ void __launch_bounds__(kThreads, NT == 128 ? 2 : 3)
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
  const int tile = blockIdx.x, t0 = blockIdx.z * NT;  // weight rows (output columns), first token
  const int tokens = min(NT, p.T - t0);
  const int kb0 = static_cast<int>(static_cast<int64_t>(p.k_blocks) * rank / splits);
  const int kb1 = static_cast<int>(static_cast<int64_t>(p.k_blocks) * (rank + 1) / splits);

  // The weight tiles (and scales) of K block kb into stage s; the token tile follows in load_x.
  auto load_w = [&](int kb, int s) {
    mbar_arrive_expect_tx(&full[s], S::kTiles + S::kSfW + S::kSfX);
    uint8_t* dst = base + s * S::kStage;
    const int x = kb * (KIND == kBf16 ? 64 : 128);  // tensor-map column of the stage (elements of the map)
#pragma unroll
    for (int b = 0; b < PARTS; ++b) tma_load_2d(dst + b * kTileW, &tmW, &full[s], x, tile * 128 + b * p.N);
    if constexpr (KIND != kBf16) {
      const int64_t row_tiles = (p.N + 127) >> 7, g = static_cast<int64_t>(kb) * S::kGroups;
#pragma unroll
      for (int b = 0; b < PARTS; ++b)
        bulk_load(dst + S::kTiles + b * S::kGroups * 512, p.sf_w + ((tile + b * row_tiles) * p.groups + g) * 512,
                  S::kGroups * 512, &full[s]);
    }
  };
  auto load_x = [&](int kb, int s) {
    uint8_t* dst = base + s * S::kStage;
    tma_load_2d(dst + PARTS * kTileW, &tmX, &full[s], kb * (KIND == kBf16 ? 64 : 128), t0);
    if constexpr (KIND != kBf16)
      bulk_load(dst + S::kTiles + S::kSfW, p.sf_x + ((t0 >> 7) * p.groups + static_cast<int64_t>(kb) * S::kGroups) * 512,
                S::kSfX, &full[s]);
  };

  const int first = min(S::kStages, kb1 - kb0);  // K blocks that fill the empty ring
  if (threadIdx.x == 0) {
    tma_prefetch_map(&tmW);
    tma_prefetch_map(&tmX);
    for (int s = 0; s < S::kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(done, 1);
    *abort_flag = 0;
    fence_mbarrier_init();
    for (int i = 0; i < first; ++i) load_w(kb0 + i, i);  // W does not depend on the kernel before
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, S::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  grid_launch_dependents();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    if (lane == 0) {
      grid_dependency_wait();
      uint32_t issued = 0, parity = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        const int i = kb - kb0, s = i % S::kStages;
        const uint32_t phase = (i / S::kStages) & 1;
        if (i >= first) {
          if (*abort_flag || !mbar_wait(&empty[s], phase ^ 1, p.timeout_ns)) {
            report_status(p.status, kStatusTimeoutProducer);
            *abort_flag = 1;
            break;
          }
          load_w(kb, s);
        }
        load_x(kb, s);
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
    // (the whole warp runs the loop, one lane issues: operands stay in uniform registers)
    const uint32_t sf_cols = tmem_base + S::kAccCols;
    const uint64_t w0 = smem_desc_sw128(smem_u32(base), 16, 1024);
    const uint64_t f0 = smem_desc_plain(smem_u32(base + S::kTiles), 512, 128);
    bool ok = true, issued_any = false;
    int s = 0;
    uint32_t phase = 0;
    for (int kb = kb0; kb < kb1; ++kb) {
      ok = mbar_try_wait(&full[s], phase) || (*abort_flag == 0 && mbar_wait(&full[s], phase, p.timeout_ns));
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_fence_after();
      const uint64_t w = w0 + static_cast<uint32_t>(s * (S::kStage >> 4)), x = w + (PARTS * kTileW >> 4);
      const uint32_t more = kb > kb0 ? 1u : 0u;
      if (elect_one()) {
        if constexpr (KIND == kBf16) {
          constexpr uint32_t IDESC = idesc_bf16_f32(128, NT, false, false);
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
#pragma unroll
            for (int b = 0; b < PARTS; ++b)
              umma_f16_ss(tmem_base + b * NT, w + ((b * kTileW) >> 4) + kk * 2, x + kk * 2, IDESC, kk > 0 ? 1u : more);
        } else {
          const uint64_t f = f0 + static_cast<uint32_t>(s * (S::kStage >> 4));
#pragma unroll
          for (int a = 0; a < (PARTS + 1) * S::kGroups; ++a) tmem_cp_32x128b_warpx4(sf_cols + 4 * a, f + 32 * a);
          // 64-value steps past K would multiply zeros by scales that nothing defines
          const int steps = min(4, (p.K - kb * fp4::kStageK + 63) / 64);
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) {
            if (kk < steps) {
              const int atom = KIND == kMxfp4 ? kk >> 1 : kk;
              const uint32_t id = KIND == kMxfp4 ? 2u * (kk & 1) : 0u;
#pragma unroll
              for (int b = 0; b < PARTS; ++b)
                fp4::umma<KIND>(tmem_base + b * NT, w + ((b * kTileW) >> 4) + kk * 2, x + kk * 2,
                                fp4::idesc(128, NT, KIND, id), (sf_cols + 4 * (b * S::kGroups + atom)) | (id << 30),
                                (sf_cols + 4 * (PARTS * S::kGroups + atom)) | (id << 30), kk > 0 ? 1u : more);
            }
          }
        }
        umma_commit(&empty[s]);
      }
      __syncwarp();
      issued_any = true;
      if (++s == S::kStages) {
        s = 0;
        phase ^= 1;
      }
    }
    if (!ok) {
      if (lane == 0) report_status(p.status, kStatusTimeoutMma);
      *abort_flag = 1;
    }
    if (elect_one()) umma_commit(done);
    if (lane == 0 && issued_any && !mbar_wait(done, 0, p.timeout_ns)) report_status(p.status, kStatusTimeoutDrain);
    __syncwarp();
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
          if (c * 32 + t < tokens)
            part[(b * NT + c * 32 + t) * kPartLd + quad * 32 + lane] = __uint_as_float(r[t]);
      }
    }
  }
  cluster_sync_all();

  // ------------------------------------------------------------ reduction and epilogue
  // A warp takes a token's 128 columns of the tile, a lane four of them.
  grid_dependency_wait();
  const uint32_t part_addr = smem_u32(part) + lane * 16;
  const int n = tile * 128 + lane * 4;
  constexpr int kTok = PARTS == 1 ? 2 : 1;  // tokens of a warp at a time: their loads overlap
  // what belongs to the columns alone
  float col_factor[PARTS][4], bias[PARTS][4];
#pragma unroll
  for (int b = 0; b < PARTS; ++b) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t c = static_cast<int64_t>(b) * p.N + n + j;
      col_factor[b][j] = KIND == kNvfp4 && n + j < p.N ? p.row_w[c] : 1.f;
      bias[b][j] = n + j < p.N && p.bias != nullptr ? __bfloat162float(p.bias[c]) : 0.f;
    }
  }
  if (*abort_flag == 0) {
    const int step = splits * kWarps;
    for (int first_token = rank * kWarps + warp; first_token < tokens; first_token += kTok * step) {
      // what the epilogue reads from memory, then the partial sums of all CTAs, for every token of this round
      float row_factor[kTok], add[kTok][4];
      float4 in[kTok][PARTS][8];
#pragma unroll
      for (int k = 0; k < kTok; ++k) {
        const int tl = first_token + k * step;
        const bool live = tl < tokens;  // warp-uniform
        row_factor[k] = KIND == kNvfp4 && live ? p.row_x[t0 + tl] : 1.f;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          add[k][j] = PARTS == 1 && live && n + j < p.N && p.residual != nullptr
                          ? __bfloat162float(p.residual[static_cast<int64_t>(t0 + tl) * p.ld_res + n + j])
                          : 0.f;
        if (live) {
#pragma unroll
          for (int r = 0; r < 8; ++r) {
            if (r < splits) {
              const uint32_t peer = mapa_shared(part_addr, static_cast<uint32_t>(r));
#pragma unroll
              for (int b = 0; b < PARTS; ++b) in[k][b][r] = ld_cluster_f4(peer + (b * NT + tl) * kPartLd * 4);
            }
          }
        }
      }
#pragma unroll
      for (int k = 0; k < kTok; ++k) {
        const int tl = first_token + k * step;
        if (tl >= tokens) break;
        const int64_t t = t0 + tl;
        float v[PARTS][4];
#pragma unroll
        for (int b = 0; b < PARTS; ++b) {
          v[b][0] = v[b][1] = v[b][2] = v[b][3] = 0.f;
#pragma unroll
          for (int r = 0; r < 8; ++r) {
            if (r < splits) {
              v[b][0] += in[k][b][r].x;
              v[b][1] += in[k][b][r].y;
              v[b][2] += in[k][b][r].z;
              v[b][3] += in[k][b][r].w;
            }
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) v[b][j] = v[b][j] * (row_factor[k] * col_factor[b][j]) + bias[b][j];
        }
        float y[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] = PARTS == 2 ? v[1 % PARTS][j] : v[0][j] + add[k][j];
        if constexpr (PARTS == 2) gated::gate(p.act, v[0], y);
        if constexpr (PARTS == 2 && KIND == kMxfp4) {
          if (p.q_out != nullptr) {  // eight lanes hold a block of 32
            uint32_t top = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              if (n + j >= p.N) y[j] = 0.f;
              top = max(top, __float_as_uint(y[j]) & 0x7fffffffu);
            }
#pragma unroll
            for (int o = 1; o < 8; o *= 2) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
            const uint32_t byte = fp4::mx_scale_byte(top);
            const float inv = fp4::mx_inverse(byte);
            const float w8[8] = {y[0] * inv, y[1] * inv, y[2] * inv, y[3] * inv, 0.f, 0.f, 0.f, 0.f};
            if ((n >> 1) < p.ld_q)
              *reinterpret_cast<uint16_t*>(p.q_out + t * p.ld_q + (n >> 1)) = static_cast<uint16_t>(fp4::pack8(w8));
            if ((lane & 7) == 0) p.q_sf[fp4::scale_offset(t, n >> 5, p.q_groups)] = static_cast<uint8_t>(byte);
            continue;
          }
        }
        __nv_bfloat16* out = p.out + t * p.ld_out + n;
        if (p.vec && n + 4 <= p.N) {
          uint2 w;
          __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&w);
          h[0] = __floats2bfloat162_rn(y[0], y[1]);
          h[1] = __floats2bfloat162_rn(y[2], y[3]);
          *reinterpret_cast<uint2*>(out) = w;
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (n + j < p.N) out[j] = __float2bfloat16_rn(y[j]);
        }
      }
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
  const int tiles = (p.N + 127) / 128, token_tiles = (p.T + NT - 1) / NT;
  const int splits = std::max(1, std::min({8, 2 * sms / (tiles * token_tiles), p.k_blocks / 2}));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(tiles, splits, token_tiles);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = S::kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 1;
  attr[0].val.clusterDim.y = splits;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.after_producer ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kern, map_x, map_w, p);
}

template <int KIND, int PARTS>
cudaError_t launch_parts(const CUtensorMap& mx, const CUtensorMap& mw, const Params& p, int sms, int device,
                         cudaStream_t stream) {
  switch (tile_rows(p.T)) {
    case 16: return launch_shape<KIND, PARTS, 16>(mx, mw, p, sms, device, stream);
    case 32: return launch_shape<KIND, PARTS, 32>(mx, mw, p, sms, device, stream);
    case 64:
      if constexpr (PARTS == 1 || KIND == kBf16) return launch_shape<KIND, PARTS, 64>(mx, mw, p, sms, device, stream);
      break;
    default:
      if constexpr (PARTS == 1) return launch_shape<KIND, PARTS, 128>(mx, mw, p, sms, device, stream);
      break;
  }
  return cudaErrorInvalidValue;  // the hosts send gated products of more rows to the GEMM (`takes`)
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
