// Gated feed-forward block on tcgen05 CTA pairs (bf16 operands, fp32 accumulation).
//
//   forward    g = x Wg^T + bg,  u = x Wu^T + bu,  h = act(g) * u
//   backward   dh = dy Wd,  dz = [dh u act'(g) | dh act(g)]
//
// with the framework's fused weight [Wg; Wu] ([2 I, H]) and Wd ([H, I]). The
// other products of the block (y = h Wd^T, dx = dz [Wg; Wu], the weight
// gradients) are plain GEMMs of gemm*.cu.
//
// Forward: a cluster of two CTAs owns 256 rows x 128 columns of h. The pair's
// B tile is 256 rows of the fused weight: CTA 0 loads 128 gate rows, CTA 1 the
// 128 up rows of the same columns, so one M = 256, N = 256 tcgen05.mma leaves g
// in accumulator columns 0-127 and u in 128-255 of the same TMEM lane, and the
// thread that holds a row has both operands of the product: z is never
// written. Without the fusion z costs 4 T I bytes written and read again.
//
// For the backward pass the forward saves a = act(g) and b = u act'(g), so the
// epilogue that produces dz only multiplies: dz = [dh b | dh a]. Both are kept
// as fp16 with one power of two per row and 32 columns (an exponent byte that
// puts the block's largest value into [2^14, 2^15)): 11 significant bits down to
// 2^-29 of that value in the bytes of bf16's 8 bits, so the rounding of dz to bf16
// (which the tensor core needs) stays the only one that counts. They are laid
// out as 32 x 32 tiles of 2 KB, b and a side by side, in the order in which the
// lanes of a warp write and read them: whole cache lines, and no detour through
// shared memory. (Row-major, the 64-byte pieces of 32 rows were slower in both passes.)
//
// Backward: the input-gradient GEMM dy Wd with 256 x 256 pair tiles whose
// epilogue reads the saved tiles (prefetched one 32-column chunk ahead) and
// stores the two halves of dz; dh is never written. With biases it also leaves
// the column sums of each 32 rows, which a second launch adds up in a fixed
// order (the sums of a separate pass over dz took longer than dz itself).
//
// Bound by the tensor pipe and by power at training sizes. [8192, 2048] x
// [12288, 2048]: forward 252 us (1.64 PFLOP/s; 239 us without any epilogue; 279 us
// before the issuing warp ran uniformly), with the saved tiles 287 us; dz from [8192, 2048] x
// [2048, 6144] 167 us (1.23 PFLOP/s; 122 us without an epilogue, which moves 400 MB).
// The main loops follow the pair kernel of gemm_kernel.cuh: six 32 KB stages, TMA
// with the 128-byte swizzle, one issuing warp, two accumulator buffers so that an
// epilogue overlaps the next tile's products. Column tiles go fastest: groups of
// 4, 8 or 16 row tiles, which halve the operands' footprint in L2, were 2 to 5 % slower.
#include "gated.h"

#include <cuda_fp16.h>

#include <algorithm>

#include "elect.cuh"
#include "gated_act.cuh"
#include "sm100.cuh"
#include "tile_io.cuh"

namespace rx {
namespace gated {

constexpr int BM = 128, BK = 64;
constexpr int kEpilogueWarps = 8;  // two per TMEM lane quadrant, each owning half the columns
constexpr int kThreads = 64 + 32 * kEpilogueWarps;

constexpr int kStages = 6;
constexpr int kTile = BM * BK * 2;  // 16 KB: 128 rows x 64 bf16
constexpr int kStaging = kEpilogueWarps * 2048;  // a 32 x 32 tile of 16-bit values for each epilogue warp
constexpr size_t kSmem = 1024 + kStages * 2 * kTile + kStaging + 256;
static_assert(kSmem <= 232448, "shared memory beyond the opt-in limit");

// Exponent byte e of a block with largest magnitude `top`: values are stored
// times 2^(141 - e) and read back times 2^(e - 141). Clamped so that both
// factors are normal floats; an infinite or NaN value keeps being one.
__device__ __forceinline__ uint32_t block_byte(float top) {
  return min(max((__float_as_uint(top) >> 23) & 0xffu, 15u), 254u);
}
__device__ __forceinline__ float store_factor(uint32_t e) { return __uint_as_float((268u - e) << 23); }
__device__ __forceinline__ float load_factor(uint32_t e) { return __uint_as_float((e - 14u) << 23); }

// A lane's row of a saved 32 x 32 tile: four 16-byte pieces, piece q of all lanes together.
__device__ __forceinline__ void save_row32(uint4* tile, int lane, const float (&v)[32], float f) {
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    uint4 w;
    __half2* h = reinterpret_cast<__half2*>(&w);
#pragma unroll
    for (int j = 0; j < 4; ++j) h[j] = __floats2half2_rn(v[q * 8 + 2 * j] * f, v[q * 8 + 2 * j + 1] * f);
    tile[q * 32 + lane] = w;
  }
}
__device__ __forceinline__ void fetch_row32(const uint4* tile, int lane, uint4 (&w)[4]) {
#pragma unroll
  for (int q = 0; q < 4; ++q) w[q] = ldg_v4_issue(tile + q * 32 + lane);
}
// v[i] = saved value i * f * r[i]
__device__ __forceinline__ void times_row32(const uint4 (&w)[4], float f, const uint32_t (&r)[32], float (&v)[32]) {
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const __half2* h = reinterpret_cast<const __half2*>(&w[q]);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 t = __half22float2(h[j]);
      v[q * 8 + 2 * j] = t.x * f * __uint_as_float(r[q * 8 + 2 * j]);
      v[q * 8 + 2 * j + 1] = t.y * f * __uint_as_float(r[q * 8 + 2 * j + 1]);
    }
  }
}

// A warp's 32 x 32 tile of 16-bit values from its staging buffer to rows row0.. and columns n.. of a
// matrix: 16-byte pieces, four lanes to a 64-byte row segment.
__device__ __forceinline__ void store_tile32(const uint8_t* buf, __nv_bfloat16* dst, int64_t ld, int row0, int n, int rows, int cols,
                                             int lane) {
  __syncwarp();
#pragma unroll
  for (int it = 0; it < 4; ++it) {
    const int c = lane + 32 * it, row = c >> 2, piece = c & 3;
    const uint4 w = *reinterpret_cast<const uint4*>(buf + row * 64 + ((piece ^ ((row >> 1) & 3)) * 16));
    if (row0 + row < rows && n + piece * 8 < cols)
      *reinterpret_cast<uint4*>(dst + static_cast<int64_t>(row0 + row) * ld + n + piece * 8) = w;
  }
  __syncwarp();
}

// v[i] += lane i's `bias`: a warp fetches the biases of its columns before their accumulator is ready.
__device__ __forceinline__ void add_bias32(float bias, float (&v)[32]) {
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] += __shfl_sync(0xffffffffu, bias, i);
}

// Sum over the warp's lanes (rows) of each of 32 columns; lane c returns column c's.
__device__ __forceinline__ float column_sum32(float (&v)[32], int lane) {
#pragma unroll
  for (int o = 16; o > 0; o /= 2) {
#pragma unroll
    for (int i = 0; i < o; ++i) {
      const bool high = (lane & o) != 0;
      const float send = high ? v[i] : v[i + o], keep = high ? v[i + o] : v[i];
      v[i] = keep + __shfl_xor_sync(0xffffffffu, send, o);
    }
  }
  return v[0];
}

// Index of the saved tile that holds rows row0.. (of 32) and columns n.. (of 32).
__device__ __forceinline__ int64_t tile_of(const Params& p, int row0, int n) {
  return static_cast<int64_t>(row0 >> 5) * ((p.N + 31) >> 5) + (n >> 5);
}

template <int MODE>
__global__ void __launch_bounds__(kThreads, 1)
    gated_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const Params p) {
  constexpr bool kDz = MODE == kBackward;
  constexpr bool kSave = MODE == kForwardSave;
  constexpr int kTileCols = kDz ? 256 : 128;  // output columns of a tile
  constexpr uint32_t kTmemCols = 512;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = base;
  uint8_t* sB = base + kStages * kTile;
  uint8_t* sC = sB + kStages * kTile;
  uint64_t* full = reinterpret_cast<uint64_t*>(sC + kStaging);
  uint64_t* empty = full + kStages;
  uint64_t* tfull = empty + kStages;
  uint64_t* tempty = tfull + 2;
  uint64_t* drain = tempty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = warp_id(), lane = lane_id();
  const int rank = static_cast<int>(cluster_ctarank());
  const bool leader = rank == 0;
  const int cluster = blockIdx.x >> 1, clusters = gridDim.x >> 1;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tfull[a], 1);
      mbar_init(&tempty[a], 2 * kEpilogueWarps);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_mbarrier_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_map(&tmA);
    tma_prefetch_map(&tmB);
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, kTmemCols);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  cluster_sync_all();  // both CTAs' barriers are initialised before any remote use
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  grid_launch_dependents();  // the down projection may stream its weight meanwhile
  const int k_blocks = (p.K + BK - 1) / BK;

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    if (lane == 0) {
      const uint32_t full_leader0 = mapa_shared(smem_u32(&full[0]), 0);
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int u = cluster; ok && u < p.num_units; u += clusters) {
        const int m = (u / p.n_tiles) * (2 * BM) + rank * BM;
        const int n0 = (u % p.n_tiles) * kTileCols;
        for (int kb = 0; kb < k_blocks; ++kb) {
          if (*abort_flag || !mbar_wait(&empty[stage], phase ^ 1, p.timeout_ns)) {
            report_status(p.status, kStatusTimeoutProducer);
            *abort_flag = 1;
            ok = false;
            break;
          }
          if (leader) mbar_arrive_expect_tx(&full[stage], 4 * kTile);  // both CTAs' A and B halves
          const uint32_t bar = full_leader0 + stage * 8;
          uint8_t* a_dst = sA + stage * kTile;
          uint8_t* b_dst = sB + stage * kTile;
          tma_load_2d_pair(a_dst, &tmA, bar, kb * BK, m);
          if constexpr (kDz) {  // Wd [K, N] is MN-major: two 64 x 64 boxes
            tma_load_2d_pair(b_dst, &tmB, bar, n0 + rank * 128, kb * BK);
            tma_load_2d_pair(b_dst + 8192, &tmB, bar, n0 + rank * 128 + 64, kb * BK);
          } else {  // CTA 0: gate rows, CTA 1: up rows of the same columns
            tma_load_2d_pair(b_dst, &tmB, bar, kb * BK, n0 + rank * p.N);
          }
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
      // every load was consumed once the MMAs of its stage have committed
      for (int s = 0; s < kStages; ++s) {
        if (!mbar_wait(&empty[stage], phase ^ 1, p.timeout_ns)) {
          report_status(p.status, kStatusTimeoutDrain);
          break;
        }
        if (++stage == kStages) {
          stage = 0;
          phase ^= 1;
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer (even CTA)
    if (leader) {  // the whole warp runs the loop, one lane issues: operands stay in uniform registers
      constexpr uint32_t IDESC = idesc_bf16_f32(2 * BM, 256, false, kDz);
      const uint64_t a0 = smem_desc_sw128(smem_u32(sA), 16, 1024);
      const uint64_t b0 = kDz ? smem_desc_sw128(smem_u32(sB), 8192, 1024) : smem_desc_sw128(smem_u32(sB), 16, 1024);
      auto ready = [&](uint64_t* bar, uint32_t parity) -> bool {
        const bool now = mbar_try_wait(bar, parity) || (*abort_flag == 0 && mbar_wait(bar, parity, p.timeout_ns));
        return __all_sync(0xffffffffu, now);
      };
      int stage = 0, local = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int u = cluster; ok && u < p.num_units; u += clusters, ++local) {
        const int acc = local & 1;
        ok = ready(&tempty[acc], ((local >> 1) & 1) ^ 1);
        if (!ok) break;
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + static_cast<uint32_t>(acc * 256);
        for (int kb = 0; kb < k_blocks; ++kb) {
          ok = ready(&full[stage], phase);
          if (!ok) break;
          tc_fence_after();
          const uint64_t a = a0 + static_cast<uint32_t>(stage * (kTile >> 4));
          const uint64_t b = b0 + static_cast<uint32_t>(stage * (kTile >> 4));
          if (elect_one()) {
#pragma unroll
            for (int kk = 0; kk < BK / 16; ++kk)
              umma_f16_ss_pair(d_tmem, a + kk * 2, b + kk * (kDz ? 128 : 2), IDESC, (kb > 0 || kk > 0) ? 1u : 0u);
            umma_commit_pair(&empty[stage], 0x3);
            if (kb + 1 == k_blocks) umma_commit_pair(&tfull[acc], 0x3);
          }
          __syncwarp();
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1;
          }
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
  } else {
    // ------------------------------------------------------------ epilogue (both CTAs)
    const int quad = warp & 3;
    constexpr int kChunks = kTileCols / 32 / (kEpilogueWarps / 4);
    const int chunk0 = ((warp - 2) / 4) * kChunks;
    const uint32_t tempty_leader = mapa_shared(smem_u32(&tempty[0]), 0);
    uint8_t* const buf = sC + (warp - 2) * 2048;
    int local = 0;
    for (int u = cluster; u < p.num_units; u += clusters, ++local) {
      const int acc = local & 1;
      const int row0 = (u / p.n_tiles) * (2 * BM) + rank * BM + quad * 32;  // this warp's 32 rows
      const int n0 = (u % p.n_tiles) * kTileCols;
      uint4 next_b[4], next_a[4];
      uint32_t next_e = 0;
      if constexpr (kDz) {
        const int n = n0 + chunk0 * 32;
        if (n < p.N && row0 < p.M) {
          const int64_t t = tile_of(p, row0, n);
          fetch_row32(p.saved + t * 256, lane, next_b);
          fetch_row32(p.saved + t * 256 + 128, lane, next_a);
          next_e = p.exps[t * 32 + lane];
        }
      }
      float bias_g[2] = {}, bias_u[2] = {};
      if constexpr (!kDz) {
        static_assert(kChunks == 2, "two chunks of 32 columns a warp");
        if (p.bias != nullptr) {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const int n = n0 + (chunk0 + c) * 32 + lane;
            if (n < p.N) {
              bias_g[c] = __bfloat162float(p.bias[n]);
              bias_u[c] = __bfloat162float(p.bias[p.N + n]);
            }
          }
        }
      }
      bool ok = (*abort_flag == 0) && mbar_wait(&tfull[acc], (local >> 1) & 1, p.timeout_ns);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) {
        if (lane == 0) report_status(p.status, kStatusTimeoutEpilogue);
        *abort_flag = 1;
        break;
      }
      tc_fence_after();
      const uint32_t t_row = tmem_base + (static_cast<uint32_t>(quad * 32) << 16) + static_cast<uint32_t>(acc * 256);
#pragma unroll 1
      for (int c = chunk0; c < chunk0 + kChunks; ++c) {
        const int n = n0 + c * 32;
        const bool live = n < p.N && row0 < p.M;  // warp-uniform
        if constexpr (kDz) {
          uint32_t r[32];
          tmem_ld_32x32b_x32(t_row + c * 32, r);
          uint4 cur_b[4], cur_a[4];
          const uint32_t e = next_e;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            cur_b[q] = next_b[q];
            cur_a[q] = next_a[q];
          }
          if (c + 1 < chunk0 + kChunks && n + 32 < p.N && row0 < p.M) {
            const int64_t t = tile_of(p, row0, n + 32);
            fetch_row32(p.saved + t * 256, lane, next_b);
            fetch_row32(p.saved + t * 256 + 128, lane, next_a);
            next_e = p.exps[t * 32 + lane];
          }
          tmem_ld_wait();
          if (!live) continue;
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            float v[32];
            if (half == 0)
              times_row32(cur_b, load_factor(e & 0xffu), r, v);
            else
              times_row32(cur_a, load_factor(e >> 8), r, v);
            gemm::stage_row32_sw64(buf, lane, v);
            store_tile32(buf, p.out[half], p.ld_out, row0, n, p.M, p.N, lane);
            if (p.partial != nullptr) {  // the bias gradient, from the values before their rounding
              if (row0 + lane >= p.M) {
#pragma unroll
                for (int i = 0; i < 32; ++i) v[i] = 0.f;
              }
              const float sum = column_sum32(v, lane);
              if (n + lane < p.N)
                p.partial[(static_cast<int64_t>(row0 >> 5) * 2 + half) * p.N + n + lane] = sum;
            }
          }
        } else {
          uint32_t rg[32], ru[32];
          tmem_ld_32x32b_x32(t_row + c * 32, rg);
          tmem_ld_32x32b_x32(t_row + 128 + c * 32, ru);
          tmem_ld_wait();
          if (!live) continue;
          float g[32], v[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            g[i] = __uint_as_float(rg[i]);
            v[i] = __uint_as_float(ru[i]);
          }
          if (p.bias != nullptr) {
            add_bias32(c == chunk0 ? bias_g[0] : bias_g[1], g);
            add_bias32(c == chunk0 ? bias_u[0] : bias_u[1], v);
          }
          if (n + 32 > p.N) {  // columns past the end (the gate side holds up rows there) count as zero
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (n + i >= p.N) g[i] = v[i] = 0.f;
          }
          if constexpr (kSave) {
            float b[32];
            float top_a = 0.f, top_b = 0.f;
            gate_and_keep(p.act, g, v, b);
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              top_a = fmaxf(top_a, fabsf(g[i]));
              top_b = fmaxf(top_b, fabsf(b[i]));
            }
            const uint32_t ea = block_byte(top_a), eb = block_byte(top_b);
            const int64_t t = tile_of(p, row0, n);
            p.exps[t * 32 + lane] = static_cast<uint16_t>(eb | (ea << 8));
            save_row32(p.saved + t * 256, lane, b, store_factor(eb));
            save_row32(p.saved + t * 256 + 128, lane, g, store_factor(ea));
            gemm::stage_row32_sw64(buf, lane, v);
            store_tile32(buf, p.out[0], p.ld_out, row0, n, p.M, p.N, lane);
          } else {
            gate(p.act, g, v);
            gemm::stage_row32_sw64(buf, lane, v);
            store_tile32(buf, p.out[0], p.ld_out, row0, n, p.M, p.N, lane);
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(tempty_leader + acc * 8);
    }
  }

  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // no CTA leaves while its peer may still signal it
  tc_fence_after();
  if (warp == 1) tmem_dealloc_pair(tmem_base, kTmemCols);
}

// 32 columns x 8 row lanes; a column's rows are added in the same order every time.
__global__ void __launch_bounds__(256) sum_partials_kernel(const float* partial, int rows, int64_t cols, float* acc,
                                                           __nv_bfloat16* out) {
  __shared__ float part[8][32];
  const int lane = lane_id(), w = warp_id();
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + lane;
  float sum = 0.f;
  if (c < cols)
    for (int r = w; r < rows; r += 8) sum += partial[r * cols + c];
  part[w][lane] = sum;
  __syncthreads();
  if (w != 0 || c >= cols) return;
#pragma unroll
  for (int i = 1; i < 8; ++i) sum += part[i][lane];
  if (acc != nullptr)
    acc[c] += sum;
  else
    out[c] = __float2bfloat16_rn(sum);
}

cudaError_t sum_partials(const float* partial, int64_t rows, int64_t cols, float* acc, __nv_bfloat16* out,
                         cudaStream_t stream) {
  sum_partials_kernel<<<static_cast<unsigned>((cols + 31) / 32), 256, 0, stream>>>(partial, static_cast<int>(rows), cols, acc,
                                                                                   out);
  return cudaGetLastError();
}

template <int MODE>
cudaError_t launch_mode(const Maps& maps, const Params& p, int sms, int device, cudaStream_t stream) {
  auto kern = gated_kernel<MODE>;
  static bool configured[64] = {false};
  if (device < 0 || device >= 64 || !configured[device]) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kSmem));
    if (e != cudaSuccess) return e;
    if (device >= 0 && device < 64) configured[device] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * std::min(p.num_units, sms / 2));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, maps.a, maps.b, p);
}

cudaError_t launch(int mode, const Maps& maps, const Params& p, int sms, int device, cudaStream_t stream) {
  switch (mode) {
    case kForward: return launch_mode<kForward>(maps, p, sms, device, stream);
    case kForwardSave: return launch_mode<kForwardSave>(maps, p, sms, device, stream);
    default: return launch_mode<kBackward>(maps, p, sms, device, stream);
  }
}

}  // namespace gated
}  // namespace rx
