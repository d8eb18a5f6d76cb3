// Quantiser to microscaled 4-bit floating point and its inverse.
//
//   MXFP4  block of 32: e = max(-126, ceil(log2(amax / 6))), code = E2M1(x 2^-e)
//   NVFP4  row: f = 2^ceil(log2(rowmax / 2688)) (2688 = 6 * 448, at least 2^-126), block of 16:
//          s = E4M3(amax / 6 / f), code = E2M1(x / (s f))
//
// All roundings are to nearest, ties to even; zeros give code 0. The factor f
// is a power of two, so that s f and the comparisons with rounding boundaries
// are exact; it belongs to the row, not to the matrix, so that one pass over
// the rows finds it and tokens do not depend on one another. Blocks (MXFP4) or
// rows (NVFP4) that hold an infinity or a NaN get a NaN scale: their values
// and products are NaN.
//
// Bound by HBM: x is read once (2 or 4 bytes a value), half a byte a value and
// the scales are written; the instructions per value are the next limit, so
//  * a lane takes 16 consecutive values (32-byte loads, an 8-byte store): an NVFP4
//    block or half an MXFP4 block, so few lanes work out the same scale; maxima
//    are taken on the raw 16-bit pairs;
//  * a warp has up to four pieces of 512 values in flight; in NVFP4, whose codes need
//    the row's maximum first, up to eight warps hold a row of up to 16384 bf16 values in
//    their registers meanwhile (longer ones are read a second time);
//  * products and corrections are done two at a time (f32x2), rows and warps come
//    from the block's shape rather than from divisions;
//  * a quotient by an E4M3 scale is a product with its reciprocal and one
//    correction step (Markstein, "Computation of elementary functions on the
//    IBM RISC System/6000 processor", 1990): the correctly rounded quotient
//    in three operations, so ties fall as the definition says.
// [8192, 6144] bf16: MXFP4 26 us (127 MB, 4.9 TB/s), NVFP4 32 us (4.1 TB/s, 41 us when one warp a row read it twice);
// [12283, 2048] fp32: 23 us (5.0 TB/s) and 26 us (33 us); decoding that to fp32 23 us (114 MB, 4.9 TB/s).
#include "fp4.h"

#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <algorithm>
#include <type_traits>

#include "fp4.cuh"

namespace rx {
namespace fp4 {

constexpr int kQuantThreads = 256;
constexpr int kQuantWarps = kQuantThreads / 32;
constexpr int kLane = 16, kPiece = 32 * kLane;  // values of a lane and of a warp
// 32-byte read-only load, issued as written.
__device__ __forceinline__ void load32(const void* ptr, uint32_t* w) {
  asm volatile("ld.global.nc.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
               : "l"(ptr));
}

template <typename T>
__device__ __forceinline__ float to_float(T v) { return static_cast<float>(v); }
template <>
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }

template <typename T>
__device__ __forceinline__ T from_float(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_float(float v) { return __float2half_rn(v); }

// A lane's values as loaded: words of 16-bit pairs, or of fp32.
template <typename T>
struct Raw {
  static constexpr int kWords = kLane * sizeof(T) / 4;
  uint32_t w[kWords];

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = 0u;
  }
  // Columns c.. of an aligned row: loads of VEC bytes where all exist (always, with FULL), one by one with zeros past
  // K elsewhere.
  template <int VEC, bool FULL>
  __device__ __forceinline__ void load(const T* row, int c, int K) {
    if (VEC == 32 && (FULL || c + kLane <= K)) {
#pragma unroll
      for (int i = 0; i < kWords; i += 8) load32(reinterpret_cast<const uint32_t*>(row + c) + i, w + i);
    } else if (VEC == 16 && (FULL || c + kLane <= K)) {
#pragma unroll
      for (int i = 0; i < kWords; i += 4) {
        const uint4 v = ldg_v4_issue(reinterpret_cast<const uint32_t*>(row + c) + i);
        w[i] = v.x;
        w[i + 1] = v.y;
        w[i + 2] = v.z;
        w[i + 3] = v.w;
      }
    } else {
      clear();
      T* e = reinterpret_cast<T*>(w);
#pragma unroll
      for (int i = 0; i < kLane; ++i)
        if (c + i < K) e[i] = row[c + i];
    }
  }
  // The same for a row at any address: the warp reads its piece (columns c0.., c0 < K) in 16-byte pieces from the
  // boundary before it, those that cross the row's ends a value at a time, and hands the values out through
  // `scratch` (kScratch words of this warp; a word of padding after eight, so that lanes do not meet in a bank).
  static constexpr int kScratch = (kPiece * static_cast<int>(sizeof(T)) / 4 + 4) / 8 * 9 + 8;
  __device__ __forceinline__ void load_any(const T* row, int c0, int K, uint32_t* scratch, int lane) {
    constexpr int kSize = sizeof(T), kVecs = kPiece * kSize / 16;
    const int off = static_cast<int>(reinterpret_cast<uintptr_t>(row + c0) & 15);  // bytes of the first vector before the piece
    const char* base = reinterpret_cast<const char*>(row + c0) - off;
    const int64_t end = off + static_cast<int64_t>(K - c0) * kSize;  // of the row
    auto fetch = [&](int b) {                               // bytes b.. of the vectors
      uint4 v = make_uint4(0u, 0u, 0u, 0u);
      if ((b >= off || c0 > 0) && b + 16 <= end) {
        v = ldg_v4_issue(base + b);
      } else {
        T* e = reinterpret_cast<T*>(&v);
#pragma unroll
        for (int i = 0; i < 16 / kSize; ++i) {
          const int at = b + i * kSize;
          if (at >= off && at < end) e[i] = *reinterpret_cast<const T*>(base + at);
        }
      }
      return v;
    };
    auto put = [&](int word, const uint4& v) {  // word: a multiple of four
      uint32_t* dst = scratch + word + (word >> 3);
      dst[0] = v.x;
      dst[1] = v.y;
      dst[2] = v.z;
      dst[3] = v.w;
    };
    uint4 v[kVecs / 32];
#pragma unroll
    for (int i = 0; i < kVecs / 32; ++i) v[i] = fetch(16 * (lane + 32 * i));
    __syncwarp();
#pragma unroll
    for (int i = 0; i < kVecs / 32; ++i) put(4 * (lane + 32 * i), v[i]);
    if (lane == 0 && off > 0) put(4 * kVecs, fetch(16 * kVecs));
    __syncwarp();
    const int first = (off >> 2) + lane * kWords;
    auto word = [&](int i) { return scratch[first + i + ((first + i) >> 3)]; };
    if constexpr (kSize == 4) {
#pragma unroll
      for (int i = 0; i < kWords; ++i) w[i] = word(i);
    } else {
      const int shift = (off & 2) * 8;
      uint32_t low = word(0);
#pragma unroll
      for (int i = 0; i < kWords; ++i) {
        const uint32_t high = word(i + 1);
        w[i] = __funnelshift_r(low, high, shift);
        low = high;
      }
    }
  }
  // Largest magnitude, in each half of the word for 16-bit types; a NaN stays one.
  __device__ __forceinline__ uint32_t top() const {
    if constexpr (sizeof(T) == 4) {
      float t = fabsf(__uint_as_float(w[0]));
#pragma unroll
      for (int i = 1; i < kWords; ++i)
        asm("max.NaN.f32 %0, %1, %2;" : "=f"(t) : "f"(t), "f"(fabsf(__uint_as_float(w[i]))));
      return __float_as_uint(t);
    } else {
      uint32_t t = w[0] & kMagnitude;
#pragma unroll
      for (int i = 1; i < kWords; ++i) t = max_of(t, magnitude(w[i]));
      return t;
    }
  }
  static __device__ __forceinline__ uint32_t magnitude(uint32_t a) {
    if constexpr (std::is_same<T, __half>::value) {
      const __half2 m = __habs2(*reinterpret_cast<__half2*>(&a));
      return *reinterpret_cast<const uint32_t*>(&m);
    } else {
      const __nv_bfloat162 m = __habs2(*reinterpret_cast<__nv_bfloat162*>(&a));
      return *reinterpret_cast<const uint32_t*>(&m);
    }
  }
  static constexpr uint32_t kMagnitude = sizeof(T) == 2 ? 0x7fff7fffu : 0x7fffffffu;
  static __device__ __forceinline__ uint32_t max_of(uint32_t a, uint32_t b) {
    if constexpr (sizeof(T) == 4) return max(a, b);  // as integers: NaN above infinity above finite values
    if constexpr (std::is_same<T, __half>::value) {
      const __half2 m = __hmax2_nan(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
      return *reinterpret_cast<const uint32_t*>(&m);
    } else {
      const __nv_bfloat162 m = __hmax2_nan(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
      return *reinterpret_cast<const uint32_t*>(&m);
    }
  }
  // Float bits of a magnitude from top().
  static __device__ __forceinline__ uint32_t top_bits(uint32_t t) {
    if constexpr (sizeof(T) == 4) {
      return t;
    } else {
      const unsigned short h = static_cast<unsigned short>(max(t & 0xffffu, t >> 16));  // magnitudes order as integers
      return __float_as_uint(to_float(*reinterpret_cast<const T*>(&h))) & 0x7fffffffu;
    }
  }
  __device__ __forceinline__ void values(float (&v)[kLane]) const {
    const T* e = reinterpret_cast<const T*>(w);
#pragma unroll
    for (int i = 0; i < kLane; ++i) v[i] = to_float(e[i]);
  }
};

// 2^ceil(log2(top / 2688)) from the float bits of the row's largest magnitude.
__device__ __forceinline__ float row_factor(uint32_t top) {
  if (top >= 0x7f800000u) return __uint_as_float(0x7fc00000u);
  const uint32_t b = __float_as_uint(__fdiv_rn(__uint_as_float(top), 2688.f));
  if (b == 0u) return 1.f;
  return __uint_as_float(max((b >> 23) + ((b & 0x7fffffu) != 0u ? 1u : 0u), 1u) << 23);
}

__device__ __forceinline__ float e4m3_value(uint32_t byte) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(static_cast<__nv_fp8_storage_t>(byte), __NV_E4M3)));
}

// Two fp32 operations an instruction.
__device__ __forceinline__ uint64_t pair(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul_pair(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t fma_pair(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ void unpair(uint64_t p, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p)); }

// v[i] *= f
__device__ __forceinline__ void scale_values(float (&v)[kLane], float f) {
  const uint64_t ff = pair(f, f);
#pragma unroll
  for (int i = 0; i < kLane; i += 2) unpair(mul_pair(pair(v[i], v[i + 1]), ff), v[i], v[i + 1]);
}

// v[i] = quotient(v[i], s, inv)
__device__ __forceinline__ void divide_values(float (&v)[kLane], float s, float inv) {
  const uint64_t minus = pair(-s, -s), ii = pair(inv, inv);
#pragma unroll
  for (int i = 0; i < kLane; i += 2) {
    const uint64_t a = pair(v[i], v[i + 1]), guess = mul_pair(a, ii);
    unpair(fma_pair(fma_pair(guess, minus, a), ii, guess), v[i], v[i + 1]);
  }
}

// a / s correctly rounded, with inv = 1 / s correctly rounded (0 for s = 0): Markstein's correction of a * inv.
__device__ __forceinline__ float quotient(float a, float s, float inv) {
  const float guess = a * inv;
  return fmaf(fmaf(-guess, s, a), inv, guess);
}

// The warps of a row (blockDim.x / 32, up to 8) take spans of AHEAD pieces in turn; in MXFP4, where spans do not
// depend on one another, blockIdx.y goes over them. All scale bytes of the row tiles are written, those of the
// padding included. Occupancy: the registers of four 16-bit pieces let three CTAs fit; with four CTAs they spill
// ([12283, 2048] fp32 NVFP4 27.3 instead of 26.4 us). Rows at any address pass through shared memory and
// take at most two pieces and four CTAs ([8191, 5001] fp16 NVFP4: 46 us, four pieces 53, four and three CTAs 55).
template <typename T, int FMT, int VEC, int AHEAD>
__global__ void __launch_bounds__(kQuantThreads, VEC != 0 && AHEAD * sizeof(T) == 8 ? 3 : 4) quantize_kernel(const QuantParams p) {
  __shared__ uint32_t tops[kQuantWarps];
  grid_launch_dependents();  // a product of these codes may fetch its other operand meanwhile
  // threadIdx.y: the row, threadIdx.x: its warps' lanes
  const int place = threadIdx.x >> 5, lane = threadIdx.x & 31, warps_per_row = blockDim.x >> 5;
  const int warp = threadIdx.y * warps_per_row + place;
  const int64_t padded = (p.rows + 127) / 128 * 128;
  const int64_t slot = static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y;  // row of the padded tiles
  const int64_t part = p.parts == 1 ? 0 : slot / padded;
  const int64_t r = slot - part * padded;
  const bool in_grid = slot < p.parts * padded, live = in_grid && r < p.rows;
  const int64_t row = part * p.rows + r;
  const T* x = static_cast<const T*>(p.x) + row * p.ldx;
  const int extent = static_cast<int>(p.groups) * 4 * block_of(FMT);
  constexpr int kSpan = AHEAD * kPiece;                              // consecutive columns that a warp takes at a time
  const int p0 = (place + blockIdx.y * warps_per_row) * kSpan;          // its first (grid.y is 1 in NVFP4)
  const int stride = gridDim.y * warps_per_row * kSpan;
  const int K = live ? p.K : 0;  // rows of the padding hold nothing
  const bool kept = FMT == kNv && stride >= extent;  // the maximum's pass leaves the whole row in registers

  Raw<T> raw[AHEAD];
  __shared__ uint32_t scratch[VEC == 0 ? kQuantWarps * Raw<T>::kScratch : 1];
  // The pieces from column c on; those past K are zeros. At most one piece of a row ends inside.
  auto load_pieces = [&](int c) {
    const int full = min(max(K - c, 0) / kPiece, AHEAD);
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      if (VEC != 0 && i < full)
        raw[i].template load<VEC, true>(x, c + i * kPiece + lane * kLane, K);
      else if (VEC == 0 && c + i * kPiece < K)
        raw[i].load_any(x, c + i * kPiece, K, scratch + (VEC == 0 ? warp * Raw<T>::kScratch : 0), lane);
      else
        raw[i].clear();
    }
    if (VEC != 0 && full < AHEAD && c + full * kPiece < K) {
      Raw<T> last;
      last.template load<VEC, false>(x, c + full * kPiece + lane * kLane, K);
#pragma unroll
      for (int i = 0; i < AHEAD; ++i)
        if (i == full) raw[i] = last;
    }
  };
  float factor = 1.f, inv_factor = 1.f;
  bool fold = true;  // s f and 1 / (s f) are normal numbers for every E4M3 s
  if constexpr (FMT == kNv) {
    uint32_t t = 0;
    for (int c = p0; c < (kept ? extent : K); c += stride) {
      load_pieces(c);
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) t = Raw<T>::max_of(t, raw[i].top());
    }
    uint32_t top = __reduce_max_sync(0xffffffffu, Raw<T>::top_bits(t));
    if (warps_per_row > 1) {  // the same for every thread of the CTA
      if (lane == 0) tops[warp] = top;
      __syncthreads();
      for (int i = 0; i < warps_per_row; ++i) top = max(top, tops[warp - place + i]);
    }
    factor = row_factor(top);
    inv_factor = __uint_as_float(0x7f000000u - __float_as_uint(factor));  // 2^-e (any value for a NaN factor)
    fold = factor >= 0x1p-80f;
    if (live && place == 0 && lane == 0) p.row_scale[row] = factor;
  }
  if (!in_grid) return;

  const int64_t sf_row = part * padded + r;
  uint8_t* sf = p.sf + scale_offset(sf_row, 0, p.groups);
  uint8_t* q = p.q + row * p.ldq;
  auto emit = [&](const Raw<T>& in, int c, bool full) {
    uint32_t t = in.top(), byte;
    float v[kLane];
    in.values(v);
    if constexpr (FMT == kMx) {
      t = Raw<T>::max_of(t, __shfl_xor_sync(0xffffffffu, t, 1));
      byte = mx_scale_byte(Raw<T>::top_bits(t));
      const float inv = mx_inverse(byte);
      scale_values(v, inv);
    } else {
      const float want = quotient(__uint_as_float(Raw<T>::top_bits(t)) * inv_factor, 6.f, 1.f / 6.f);
      byte = __nv_cvt_float_to_fp8(want, __NV_SATFINITE, __NV_E4M3);
      // a row with a NaN factor is NaN by that factor whatever its codes; a zero scale has zero codes
      float s = e4m3_value(byte), inv = s > 0.f ? __frcp_rn(s) : 0.f;
      if (fold) {  // s f and its reciprocal, rounded like that of s: f is a power of two
        s *= factor;
        inv *= inv_factor;
      } else {
        scale_values(v, inv_factor);
      }
      divide_values(v, s, inv);
    }
    uint2 codes;
    codes.x = pack8(reinterpret_cast<const float(&)[8]>(v[0]));
    codes.y = pack8(reinterpret_cast<const float(&)[8]>(v[8]));
    // four blocks' bytes -> one 4-byte word of the group, written by its first lane
    constexpr int kLanes = block_of(FMT) / kLane;  // lanes of a block
    uint32_t word = byte << (8 * ((lane / kLanes) & 3));
#pragma unroll
    for (int o = kLanes; o < 4 * kLanes; o *= 2) word |= __shfl_xor_sync(0xffffffffu, word, o);
    if (full) {
      if (lane % (4 * kLanes) == 0) *reinterpret_cast<uint32_t*>(sf + static_cast<int64_t>(c / (4 * block_of(FMT))) * 512) = word;
      *reinterpret_cast<uint2*>(q + (c >> 1)) = codes;
    } else if (c < extent) {
      if (lane % (4 * kLanes) == 0) *reinterpret_cast<uint32_t*>(sf + static_cast<int64_t>(c / (4 * block_of(FMT))) * 512) = live ? word : 0u;
      if (live && (c >> 1) < p.ldq) *reinterpret_cast<uint2*>(q + (c >> 1)) = codes;
    }
  };
  // (in NVFP4 the row was read just before: its lines are still near)
  for (int c = p0; c < extent; c += stride) {
    if (!kept) load_pieces(c);
    const int full = min(max(K - c, 0) / kPiece, AHEAD);  // warp-uniform: no bounds inside
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
      if (i < full) emit(raw[i], c + i * kPiece + lane * kLane, true);
#pragma unroll 1
    for (int i = full; i < AHEAD && c + i * kPiece < extent; ++i) {  // the row's end, or a row of the padding
      Raw<T> in = raw[0];
#pragma unroll
      for (int j = 1; j < AHEAD; ++j)
        if (j == i) in = raw[j];
      emit(in, c + i * kPiece + lane * kLane, false);
    }
  }
}

template <typename T, int FMT, int VEC, int AHEAD>
cudaError_t launch_quantize(const QuantParams& p, cudaStream_t stream) {
  const int64_t slots = p.parts * ((p.rows + 127) / 128 * 128);
  const int64_t extent = p.groups * 4 * block_of(FMT), span = AHEAD * kPiece, spans = (extent + span - 1) / span;
  // NVFP4: all spans of a row at once, or as few equal rounds of them as eight warps need ([4096, 20000] bf16: 60 us, eight
  // warps with a last round of two 71, one warp a row 80)
  const int64_t rounds = (spans + kQuantWarps - 1) / kQuantWarps;
  const int wpr = FMT == kMx ? 1 : static_cast<int>((spans + rounds - 1) / rounds);
  const int rows_per_cta = kQuantWarps / wpr;
  const dim3 grid(static_cast<unsigned>((slots + rows_per_cta - 1) / rows_per_cta),
                  FMT == kMx ? static_cast<unsigned>(spans) : 1u);
  quantize_kernel<T, FMT, VEC, AHEAD><<<grid, dim3(32 * wpr, rows_per_cta), 0, stream>>>(p);
  return cudaGetLastError();
}

// (fp32: at most two pieces, which are as many registers as four of a 16-bit type)
template <typename T, int FMT, int VEC>
cudaError_t launch_ahead(int ahead, const QuantParams& p, cudaStream_t stream) {
  if (ahead == 1) return launch_quantize<T, FMT, VEC, 1>(p, stream);
  if constexpr (sizeof(T) == 2 && VEC != 0)
    if (ahead > 2) return launch_quantize<T, FMT, VEC, 4>(p, stream);
  return launch_quantize<T, FMT, VEC, 2>(p, stream);
}

template <typename T, int FMT>
cudaError_t quantize_typed(const QuantParams& p, cudaStream_t stream) {
  auto aligned = [&](unsigned bytes) {
    return reinterpret_cast<uintptr_t>(p.x) % bytes == 0 && p.ldx * static_cast<int64_t>(sizeof(T)) % bytes == 0;
  };
  // Pieces of a warp: many amortise its address arithmetic and keep more of a long row in registers (NVFP4
  // [8192, 6144] bf16: four 31.9 us, two 35.9; [12283, 2048] fp32: two 26.4, one 29.8), few spread a small matrix over more
  // warps ([1024, 2048] bf16 MXFP4: one 3.6 us, four 4.1; [4096, 1000] NVFP4: one 7.2, two 6.4) and leave none idle in short
  // rows ([8192, 768] NVFP4: two 8.5, four 10.3).
  const int64_t pieces = (p.K + kPiece - 1) / kPiece;
  const bool few = p.parts * p.rows * p.K < 3 << 20;
  const int ahead = pieces == 1 || (few && pieces <= kQuantWarps) ? 1 : pieces == 2 || (few && pieces <= 2 * kQuantWarps) ? 2 : 4;
  if (aligned(32)) return launch_ahead<T, FMT, 32>(ahead, p, stream);
  if (aligned(16)) return launch_ahead<T, FMT, 16>(ahead, p, stream);
  return launch_ahead<T, FMT, 0>(std::min(ahead, 2), p, stream);
}

cudaError_t quantize(const QuantParams& p, int fmt, int type, cudaStream_t stream) {
  const bool mx = fmt == kMx;
  switch (type) {
    case kBf16In: return mx ? quantize_typed<__nv_bfloat16, kMx>(p, stream) : quantize_typed<__nv_bfloat16, kNv>(p, stream);
    case kF16In: return mx ? quantize_typed<__half, kMx>(p, stream) : quantize_typed<__half, kNv>(p, stream);
    default: return mx ? quantize_typed<float, kMx>(p, stream) : quantize_typed<float, kNv>(p, stream);
  }
}

// Eight outputs, as one 16- or 32-byte store.
template <typename T>
__device__ __forceinline__ void store8(T* dst, const T (&v)[8]) {
  const uint32_t* w = reinterpret_cast<const uint32_t*>(v);
  if constexpr (sizeof(T) == 2)
    *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
  else
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst), "r"(w[0]), "r"(w[1]), "r"(w[2]),
                 "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
}

// A lane decodes eight consecutive values at a time, a warp 256. Rows as in the quantiser.
template <typename T, int FMT>
__global__ void __launch_bounds__(kQuantThreads) dequantize_kernel(const DequantParams p, bool vec) {
  const int place = threadIdx.x >> 5, lane = threadIdx.x & 31, warps_per_row = blockDim.x >> 5;
  const int warp = threadIdx.y * warps_per_row + place;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y;
  if (row >= p.parts * p.rows) return;
  const int64_t part = p.parts == 1 ? 0 : row / p.rows;
  const uint8_t* sf = p.sf + scale_offset(part * ((p.rows + 127) / 128 * 128) + row - part * p.rows, 0, p.groups);
  const uint8_t* q = p.q + row * p.ldq;
  const float factor = FMT == kNv ? p.row_scale[row] : 1.f;
  T* out = static_cast<T*>(p.out) + row * p.ldo;
  __shared__ T scratch[kQuantWarps][256];
#pragma unroll 4
  for (int c = place * 256 + lane * 8; c - lane * 8 < p.K; c += warps_per_row * 256) {  // warp-uniform
    if (vec && c >= p.K) continue;
    // (codes past K stay within the row of codes or count as zero)
    const uint32_t codes = (c >> 1) < p.ldq ? *reinterpret_cast<const uint32_t*>(q + (c >> 1)) : 0u;
    const int block = c / block_of(FMT);
    const uint32_t byte = sf[static_cast<int64_t>(block >> 2) * 512 + (block & 3)];
    float scale;
    if constexpr (FMT == kMx)
      scale = byte == 0xffu ? __uint_as_float(0x7fc00000u) : __uint_as_float(byte << 23);
    else
      scale = e4m3_value(byte) * factor;
    float f[8];
    unpack8(codes, f);
    T v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = from_float<T>(f[j] * scale);
    if (vec && c + 8 <= p.K) {
      store8(out + c, v);
    } else if (vec) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (c + j < p.K) out[c + j] = v[j];
    } else {  // rows at any address: the warp writes its 256 values a value a lane
      __syncwarp();
#pragma unroll
      for (int j = 0; j < 8; ++j) scratch[warp][lane * 8 + j] = v[j];
      __syncwarp();
      const int c0 = c - lane * 8;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (c0 + j * 32 + lane < p.K) out[c0 + j * 32 + lane] = scratch[warp][j * 32 + lane];
    }
  }
}

template <typename T>
cudaError_t dequantize_typed(const DequantParams& p, int fmt, cudaStream_t stream) {
  constexpr int kAlign = 8 * sizeof(T);
  const bool vec = reinterpret_cast<uintptr_t>(p.out) % kAlign == 0 && p.ldo % 8 == 0;
  const int64_t rows = p.parts * p.rows;
  // four pieces of 256 values a warp, fewer while that leaves SMs with less than 32 warps ([2048, 6144] bf16 MXFP4: a whole row a
  // warp 13.0 us, four pieces 10.3; [12288, 2048] 18.6 and 16.4, one piece 20.2)
  const int pieces = (p.K + 255) / 256;
  int wpr = std::min(kQuantWarps, (pieces + 3) / 4);
  if (rows * wpr < 148 * 32) wpr = std::min(kQuantWarps, pieces);
  const dim3 threads(32 * wpr, kQuantWarps / wpr);
  const unsigned grid = static_cast<unsigned>((rows + threads.y - 1) / threads.y);
  if (fmt == kMx)
    dequantize_kernel<T, kMx><<<grid, threads, 0, stream>>>(p, vec);
  else
    dequantize_kernel<T, kNv><<<grid, threads, 0, stream>>>(p, vec);
  return cudaGetLastError();
}

cudaError_t dequantize(const DequantParams& p, int fmt, int type, cudaStream_t stream) {
  switch (type) {
    case kBf16In: return dequantize_typed<__nv_bfloat16>(p, fmt, stream);
    case kF16In: return dequantize_typed<__half>(p, fmt, stream);
    default: return dequantize_typed<float>(p, fmt, stream);
  }
}

}  // namespace fp4
}  // namespace rx
