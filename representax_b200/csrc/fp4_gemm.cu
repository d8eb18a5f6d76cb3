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
// Persistent CTA pairs on tiles of 256 x 256 accumulators. CTA r of a pair loads
// A rows [128 r, 128 r + 128) and half of the B rows (plain: adjacent columns;
// gated: CTA 0 the gate rows, CTA 1 the up rows of the same 128 columns), 32 KB of
// codes per 256 values of K, with the scales of its A rows and of all B rows. One
// thread copies the scales to TMEM (one stage ahead of the products, so that the
// copies do not stand between them) and issues four K = 64 MMAs of 256 x 256 per
// stage; eight epilogue warps per CTA. The accumulator takes 256 of the 512 TMEM
// columns, the scales of all stages share the rest; instead of a second
// accumulator, an epilogue thread takes its 128 values into registers and
// frees the accumulator before it computes or stores, so the tensor core waits
// for a TMEM read only. bf16 results leave through shared memory and TMA tile stores.
//
// What measuring led here (12288 x 8192 outputs, K 2048): with `lane == 0` around the issuing
// loop every operand of an instruction was moved to uniform registers again, 60 to
// 90 cycles an instruction, 16 of them a stage: 128 us MXFP4 and 179 us NVFP4
// against 110 and 121 us with the warp-uniform loop. What bounds it now is the
// L2: without an epilogue the loads run at 12 TB/s over all SMs, 5.4 PFLOP/s;
// the epilogue's stores come on top. K 6144, 8192 x 2048 outputs + residual:
// 53 us MXFP4 (3.9 PFLOP/s), 54 us NVFP4; gated, K 2048, 8192 x 6144 outputs as
// MXFP4 codes: 95 us (4.3 PFLOP/s), NVFP4 with bf16 outputs 102 us.
#include "fp4.h"

#include <algorithm>

#include "fp4.cuh"
#include "gated_act.cuh"
#include "tile_io.cuh"

namespace rx {
namespace fp4 {

constexpr int kTile = 128 * 128;   // 128 rows x 256 codes
constexpr int kGemmStages = 5;
constexpr int kEpiWarps = 8;
constexpr int kFirstEpi = 4;  // warps 0 (producer) and 1 (MMA issuer) share a warpgroup with two idle ones
constexpr int kGemmThreads = 32 * (kFirstEpi + kEpiWarps);
// Registers of the two roles: an epilogue thread holds 128 accumulators. 128 * 64 + 256 * 216 is below the
// 384 * 168 that the block is launched with.
constexpr int kIssueRegs = 64, kEpiRegs = 216;
constexpr int kStaging = kEpiWarps * 2 * 2048;
constexpr int kRowLd = 34;  // row of a staged tile whose output rows have any address (17 words: no bank conflicts)

template <int FMT>
struct GemmShape {
  static constexpr int kGroups = groups_per_stage(FMT);
  static constexpr int kSf = 3 * kGroups * 512;    // one A tile's scales, two B tiles'
  static constexpr int kStage = 2 * kTile + kSf;
  static constexpr size_t kSmem = 1024 + kGemmStages * kStage + kStaging + 256;
  static constexpr int kSfCols = 3 * kGroups * 4;  // TMEM columns of a stage's scales
  static_assert(256 + kGemmStages * kSfCols <= 512 && kSmem <= 232448, "does not fit");
};

// Row factors and bias of 32 accumulators. Lane i holds what belongs to column i (`row_b`, `bias`), fetched
// before the accumulator was ready, and passes it to the others here: uniform loads by every lane, with their
// branches on N, stood between the values and took 104 -> 124 us (NVFP4, 12288 x 8192 outputs, K 2048), 101 -> 144 us (gated).
template <int FMT>
__device__ __forceinline__ void finish32(float row_a, float row_b, bool has_bias, float bias, const uint32_t (&r)[32],
                                         float (&v)[32]) {
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    v[i] = __uint_as_float(r[i]);
    if constexpr (FMT == kNv) v[i] *= row_a * __shfl_sync(0xffffffffu, row_b, i);
  }
  if (has_bias) {
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] += __shfl_sync(0xffffffffu, bias, i);
  }
}

template <int FMT, bool GATED, bool VEC>  // VEC: p.vec
__global__ void __launch_bounds__(kGemmThreads, 1)
    fp4_gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                    const __grid_constant__ CUtensorMap tmSfA, const __grid_constant__ CUtensorMap tmSfB,
                    const __grid_constant__ CUtensorMap tmOut, const GemmParams p) {
  using S = GemmShape<FMT>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sC = base + kGemmStages * 2 * kTile;  // code tiles, then staging, then scales
  uint8_t* sf_base = sC + kStaging;
  uint64_t* full = reinterpret_cast<uint64_t*>(sf_base + kGemmStages * S::kSf);
  uint64_t* empty = full + kGemmStages;
  uint64_t* tfull = empty + kGemmStages;
  uint64_t* tempty = tfull + 1;
  uint64_t* drain = tempty + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = warp_id(), lane = lane_id();
  const int rank = static_cast<int>(cluster_ctarank());
  const bool leader = rank == 0;
  const int cluster = blockIdx.x >> 1, clusters = gridDim.x >> 1;
  constexpr int kTileN = GATED ? 128 : 256;  // output columns of a tile

  if (threadIdx.x == 0) {
    for (int s = 0; s < kGemmStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(tfull, 1);
    mbar_init(tempty, 2 * kEpiWarps);
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_mbarrier_init();
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, 512);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  cluster_sync_all();  // both CTAs' barriers are initialised before any remote use
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const int num_units = p.m_tiles * p.n_tiles;
  // launched early (after_producer), this grid has come this far while the one before still ran
  grid_launch_dependents();
  grid_dependency_wait();

  if (warp >= kFirstEpi) {
    // ------------------------------------------------------------ epilogue (both CTAs)
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kEpiRegs));
    const int quad = warp & 3, half = (warp - kFirstEpi) >> 2;
    const uint32_t tempty_leader = mapa_shared(smem_u32(tempty), 0);
    uint8_t* const staging = sC + (warp - kFirstEpi) * 4096;
    int local = 0;
    uint32_t seq = 0;
    for (int u = cluster; u < num_units; u += clusters, ++local) {
      const int mt = u % p.m_tiles, nt = u / p.m_tiles;
      const int row0 = mt * 256 + rank * 128 + quad * 32;  // this warp's 32 rows
      uint4 next[4];  // the next chunk's residual tile, in flight
      const bool side = VEC && !GATED && p.residual != nullptr && row0 < p.M;
      if (side && nt * kTileN + half * 128 < p.N)
        gemm::warp_fetch_tile32(p.residual, p.ld_res, row0, nt * kTileN + half * 128, p.M, p.N, lane, next);
      // the same where rows have any address: lane = column, one load a row
      const bool any_side = !VEC && !GATED && p.residual != nullptr && row0 < p.M;
      const int n_end = min(p.N, nt * kTileN + half * 128 + 128);
      const bool rows_full = row0 + 32 <= p.M;
      __nv_bfloat16 next_any[32];
      auto fetch_any = [&](int n) {
        const __nv_bfloat16* src = p.residual + static_cast<int64_t>(row0) * p.ld_res + n + lane;
        if (rows_full && n + 32 <= p.N) {
#pragma unroll
          for (int i = 0; i < 32; ++i, src += p.ld_res) next_any[i] = *src;
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i, src += p.ld_res)
            next_any[i] = row0 + i < p.M && n + lane < p.N ? *src : __float2bfloat16_rn(0.f);
        }
      };
      if (any_side) fetch_any(nt * kTileN + half * 128);
      // row factors and biases of the four chunks of 32 columns, lane = column (gated: two of gate, two of up)
      const int64_t m = row0 + lane;
      const bool live = m < p.M;
      const float row_a = FMT == kNv && live ? p.row_a[m] : 1.f;
      float row_b[4] = {}, bias[4] = {};
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int n = nt * kTileN + (GATED ? half * 64 + (c & 1) * 32 : half * 128 + c * 32) + lane;
        if (n < p.N) {
          const int64_t at = (GATED && c >= 2 ? p.N : 0) + n;
          if constexpr (FMT == kNv) row_b[c] = p.row_b[at];
          if (p.bias != nullptr) bias[c] = __bfloat162float(p.bias[at]);
        }
      }
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
      if (lane == 0) mbar_arrive_cluster(tempty_leader);
      if (row0 >= p.M) continue;  // warp-uniform
      const bool has_bias = p.bias != nullptr;
      // 32 outputs of every row of the warp, from column n
      auto put = [&](int n, float (&v)[32], const uint4* res) {
        if constexpr (!VEC) {  // rows at any address: through shared memory, a warp writes 32 columns of one row at a time
          __nv_bfloat16* tile = reinterpret_cast<__nv_bfloat16*>(staging);
          uint32_t* row = reinterpret_cast<uint32_t*>(tile + lane * kRowLd);
          if (any_side) {
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 32; ++i) tile[i * kRowLd + lane] = next_any[i];
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const uint32_t w = row[i];
              v[2 * i] += __uint_as_float(w << 16);
              v[2 * i + 1] += __uint_as_float(w & 0xffff0000u);
            }
            if (n + 32 < n_end) fetch_any(n + 32);
          }
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
            row[i] = *reinterpret_cast<const uint32_t*>(&h);
          }
          __syncwarp();
          __nv_bfloat16* dst = p.out + static_cast<int64_t>(row0) * p.ld_out + n + lane;
          if (rows_full && n + 32 <= p.N) {
#pragma unroll
            for (int i = 0; i < 32; ++i, dst += p.ld_out) *dst = tile[i * kRowLd + lane];
          } else if (n + lane < p.N) {
#pragma unroll
            for (int i = 0; i < 32; ++i, dst += p.ld_out)
              if (row0 + i < p.M) *dst = tile[i * kRowLd + lane];
          }
          return;
        }
        uint8_t* buf = staging + (seq++ & 1) * 2048;
        if (lane == 0) tma_store_wait_read<1>();  // the store that last read `buf` is done reading
        __syncwarp();
        if (res != nullptr) {  // the tile's rows to their threads
          float add[32];
          gemm::warp_put_tile32_sw64(buf, lane, *reinterpret_cast<const uint4(*)[4]>(res));
          __syncwarp();
          gemm::read_row32_sw64(buf, lane, add);
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] += add[i];
        }
        gemm::stage_row32_sw64(buf, lane, v);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          tma_store_2d(&tmOut, buf, n, row0);
          tma_store_commit();
        }
      };
      if constexpr (GATED) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int n = nt * kTileN + half * 64 + c * 32;
          // (a quantised output also defines the blocks past N of the tile)
          if (n >= p.N && p.q_out == nullptr) continue;
          float g[32], v[32];
          finish32<FMT>(row_a, row_b[c], has_bias, bias[c], r[c], g);
          finish32<FMT>(row_a, row_b[2 + c], has_bias, bias[2 + c], r[2 + c], v);
          gated::gate(p.act, g, v);
          if (FMT == kMx && p.q_out != nullptr) {
            if (n + 32 > p.N) {  // columns past the end: zeros in the next layer's contraction
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (n + i >= p.N) v[i] = 0.f;
            }
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
            if (live && (n >> 1) < p.ld_q)
              *reinterpret_cast<uint4*>(p.q_out + m * p.ld_q + (n >> 1)) = make_uint4(codes[0], codes[1], codes[2], codes[3]);
            if (live) p.q_sf[scale_offset(m, n >> 5, p.q_groups)] = static_cast<uint8_t>(byte);
          } else {
            put(n, v, nullptr);
          }
        }
      } else {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int n = nt * kTileN + half * 128 + c * 32;
          if (n >= p.N) continue;
          float v[32];
          finish32<FMT>(row_a, row_b[c], has_bias, bias[c], r[c], v);
          if (side) {
            uint4 cur[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) cur[q] = next[q];
            if (c < 3 && n + 32 < p.N)
              gemm::warp_fetch_tile32(p.residual, p.ld_res, row0, n + 32, p.M, p.N, lane, next);
            put(n, v, cur);
          } else {
            put(n, v, nullptr);
          }
        }
      }
    }
    if (lane == 0) tma_store_wait<0>();  // every tile store has landed before the CTA exits
    __syncwarp();
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kIssueRegs));
    if (warp == 0) {
      // ------------------------------------------------------------ producer
      if (lane == 0) {
        tma_prefetch_map(&tmA);
        tma_prefetch_map(&tmB);
        tma_prefetch_map(&tmSfA);
        tma_prefetch_map(&tmSfB);
        const uint32_t full_leader0 = mapa_shared(smem_u32(&full[0]), 0);
        const int groups = static_cast<int>(p.groups);
        int stage = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (int u = cluster; ok && u < num_units; u += clusters) {
          const int mt = u % p.m_tiles, nt = u / p.m_tiles;
          const int m_row = mt * 256 + rank * 128;
          const int b_row = GATED ? nt * 128 + rank * p.N : nt * 256 + rank * 128;
          // scale row tiles (a tile past the end reads the last one's: its products are dropped)
          const int ta = min(2 * mt + rank, p.a_tiles - 1);
          const int tb0 = GATED ? nt : 2 * nt, tb1 = GATED ? nt + p.b_tiles : min(2 * nt + 1, p.b_tiles - 1);
          for (int ks = 0; ks < p.k_stages; ++ks) {
            if (*abort_flag || !mbar_wait(&empty[stage], phase ^ 1, p.timeout_ns)) {
              report_status(p.status, kStatusTimeoutProducer);
              *abort_flag = 1;
              ok = false;
              break;
            }
            if (leader) mbar_arrive_expect_tx(&full[stage], 2 * S::kStage);  // both CTAs' loads
            const uint32_t bar = full_leader0 + stage * 8;
            uint8_t* tiles = base + stage * 2 * kTile;
            uint8_t* sf = sf_base + stage * S::kSf;
            constexpr int kBytes = S::kGroups * 512;
            const int g = ks * S::kGroups;
            tma_load_2d_pair(tiles, &tmA, bar, ks * 128, m_row);
            tma_load_2d_pair(tiles + kTile, &tmB, bar, ks * 128, b_row);
            tma_load_2d_pair(sf, &tmSfA, bar, 0, ta * groups + g);
            tma_load_2d_pair(sf + kBytes, &tmSfB, bar, 0, tb0 * groups + g);
            tma_load_2d_pair(sf + 2 * kBytes, &tmSfB, bar, 0, tb1 * groups + g);
            if (++stage == kGemmStages) {
              stage = 0;
              phase ^= 1;
            }
          }
        }
        // every load was consumed once the MMAs of its stage have committed
        for (int s = 0; s < kGemmStages; ++s) {
          if (!mbar_wait(&empty[stage], phase ^ 1, p.timeout_ns)) {
            report_status(p.status, kStatusTimeoutDrain);
            break;
          }
          if (++stage == kGemmStages) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
    } else if (warp == 1) {
      // ------------------------------------------------------------ MMA issuer (even CTA)
      if (leader) {
        // The whole warp runs this loop and one lane issues. What the issuing costs bounds the stage, so its
        // instructions are kept few: descriptors are a base plus an offset in their address field, and the abort
        // flag is read only where a wait is not over at once.
        const uint64_t a0 = smem_desc_sw128(smem_u32(base), 16, 1024);
        const uint64_t f0 = smem_desc_plain(smem_u32(sf_base), 512, 128);
        const uint32_t tmem_sf = tmem_base + 256;
        auto ready = [&](uint64_t* bar, uint32_t parity) -> bool {
          const bool now = mbar_try_wait(bar, parity) || (*abort_flag == 0 && mbar_wait(bar, parity, p.timeout_ns));
          return __all_sync(0xffffffffu, now);
        };
        // Wait for a stage's data and copy its scales into the stage's TMEM columns.
        auto fetch = [&](int s, uint32_t phase) -> bool {
          if (!ready(&full[s], phase)) return false;
          tc_fence_after();
          const uint64_t f = f0 + static_cast<uint32_t>(s * (S::kSf >> 4));
          const uint32_t sfa = tmem_sf + s * S::kSfCols, sfb = sfa + 4 * S::kGroups;
          if (elect_one()) {
#pragma unroll
            for (int j = 0; j < S::kGroups; ++j) {
              tmem_cp_scales_pair(sfa + 4 * j, f + 32 * j);
              tmem_cp_scales_pair(sfb + 8 * j, f + 32 * (S::kGroups + j));
              tmem_cp_scales_pair(sfb + 8 * j + 4, f + 32 * (2 * S::kGroups + j));
            }
          }
          return true;
        };
        auto products = [&](int s, int kk, uint32_t accumulate) {
          const uint64_t a = a0 + static_cast<uint32_t>(s * (2 * kTile >> 4) + kk * 2);
          const uint32_t sfa = tmem_sf + s * S::kSfCols, sfb = sfa + 4 * S::kGroups;
          const int atom = FMT == kMx ? kk >> 1 : kk;
          const uint32_t id = FMT == kMx ? 2u * (kk & 1) : 0u;
          umma_pair<FMT>(tmem_base, a, a + (kTile >> 4), idesc(256, 256, FMT, id), (sfa + 4 * atom) | (id << 30),
                         (sfb + 8 * atom) | (id << 30), accumulate);
        };
        const int tail = (p.K - (p.k_stages - 1) * kStageK + 63) / 64;  // 64-value steps of the last stage
        int s = 0, local = 0;
        uint32_t phase = 0;
        bool ok = cluster >= num_units || fetch(0, 0);
        for (int u = cluster; ok && u < num_units; u += clusters, ++local) {
          ok = ready(tempty, static_cast<uint32_t>(local & 1) ^ 1u);
          tc_fence_after();
          for (int ks = 0; ok && ks < p.k_stages; ++ks) {
            int s1 = s + 1;
            if (s1 == kGemmStages) {
              s1 = 0;
              phase ^= 1;
            }
            const bool last = ks + 1 == p.k_stages;
            if (!last || u + clusters < num_units) ok = fetch(s1, phase);  // one stage ahead
            if (!ok) break;
            if (elect_one()) {
              if (!last || tail == 4) {
#pragma unroll
                for (int kk = 0; kk < 4; ++kk) products(s, kk, (ks > 0 || kk > 0) ? 1u : 0u);
              } else {  // steps past K would multiply zeros by scales that nothing defines
                for (int kk = 0; kk < tail; ++kk) products(s, kk, (ks > 0 || kk > 0) ? 1u : 0u);
              }
              umma_commit_pair(&empty[s], 0x3);
              if (last) umma_commit_pair(tfull, 0x3);
            }
            __syncwarp();
            s = s1;
          }
        }
        if (!ok) {
          if (lane == 0) report_status(p.status, kStatusTimeoutMma);
          *abort_flag = 1;
        }
        if (elect_one()) umma_commit_pair(drain, 0x3);
      }
      if (lane == 0 && !mbar_wait(drain, 0, p.timeout_ns)) report_status(p.status, kStatusTimeoutDrain);
      __syncwarp();
    }
  }

  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // no CTA leaves while its peer may still signal it
  tc_fence_after();
  if (warp == 1) tmem_dealloc_pair(tmem_base, 512);
}

template <int FMT, bool GATED, bool VEC>
cudaError_t launch_vec(const GemmMaps& maps, const GemmParams& p, int sms, int device, cudaStream_t stream) {
  auto kern = fp4_gemm_kernel<FMT, GATED, VEC>;
  constexpr size_t smem = GemmShape<FMT>::kSmem;
  static bool configured[64] = {false};
  if (device < 0 || device >= 64 || !configured[device]) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    if (e != cudaSuccess) return e;
    if (device >= 0 && device < 64) configured[device] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * std::min(p.m_tiles * p.n_tiles, sms / 2));
  cfg.blockDim = dim3(kGemmThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.after_producer ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kern, maps.a, maps.b, maps.sf_a, maps.sf_b, maps.out, p);
}

template <int FMT, bool GATED>
cudaError_t launch(const GemmMaps& maps, const GemmParams& p, int sms, int device, cudaStream_t stream) {
  return p.vec ? launch_vec<FMT, GATED, true>(maps, p, sms, device, stream)
               : launch_vec<FMT, GATED, false>(maps, p, sms, device, stream);
}

cudaError_t gemm(const GemmMaps& maps, const GemmParams& p, int fmt, int sms, int device, cudaStream_t stream) {
  if (fmt == kMx)
    return p.gated ? launch<kMx, true>(maps, p, sms, device, stream) : launch<kMx, false>(maps, p, sms, device, stream);
  return p.gated ? launch<kNv, true>(maps, p, sms, device, stream) : launch<kNv, false>(maps, p, sms, device, stream);
}

}  // namespace fp4
}  // namespace rx
