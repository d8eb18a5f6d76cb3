// Host entries of the microscaled 4-bit kernels and of the kernels for few
// token rows: argument checks, tensor maps, dispatch.
#include "fp4.h"

#include "common.h"
#include "few_rows.h"

namespace rx {

namespace {

constexpr int kMx = 1, kNv = 2;

int64_t scale_groups(int64_t k, int64_t fmt) { return (k + 255) / 256 * (fmt == kMx ? 2 : 4); }
int64_t row_tiles(int64_t rows) { return (rows + 127) / 128; }

void check_device(const at::Tensor& t, const char* name, int device) {
  RX_CHECK(t.is_cuda() && t.get_device() == device, name, " must be on device ", device);
}

void check_format(int64_t fmt) { RX_CHECK(fmt == kMx || fmt == kNv, "format must be 1 (MXFP4) or 2 (NVFP4), got ", fmt); }

// Codes, scales and row factors of `parts * rows` rows of K values.
void check_operand(const at::Tensor& q, const at::Tensor& sf, const c10::optional<at::Tensor>& row_scale, int64_t rows,
                   int64_t parts, int64_t K, int64_t fmt, int device, const char* name) {
  check_device(q, name, device);
  check_device(sf, name, device);
  RX_CHECK(q.scalar_type() == at::kByte && sf.scalar_type() == at::kByte, name, ": codes and scales must be uint8");
  RX_CHECK(q.dim() == 2 && q.size(0) == rows * parts && q.stride(1) == 1 && q.size(1) == (K + 31) / 32 * 16, name,
           ": codes must be [", rows * parts, ", ", (K + 31) / 32 * 16, "]");
  RX_CHECK(q.stride(0) % 16 == 0 && q.stride(0) >= q.size(1) && reinterpret_cast<uintptr_t>(q.data_ptr()) % 16 == 0, name,
           ": rows of codes must be 16-byte aligned");
  RX_CHECK(sf.is_contiguous() && sf.numel() == parts * row_tiles(rows) * scale_groups(K, fmt) * 512 &&
               reinterpret_cast<uintptr_t>(sf.data_ptr()) % 16 == 0,
           name, ": scales must be a contiguous, 16-byte aligned array of ",
           parts * row_tiles(rows) * scale_groups(K, fmt) * 512, " bytes");
  RX_CHECK(row_scale.has_value() == (fmt == kNv), name, ": row factors belong to NVFP4 and only to it");
  if (row_scale.has_value()) {
    check_device(*row_scale, name, device);
    RX_CHECK(row_scale->scalar_type() == at::kFloat && row_scale->is_contiguous() && row_scale->numel() == rows * parts, name,
             ": row factors must be a contiguous float32 vector of ", rows * parts);
  }
}

void check_sizes(int64_t rows, int64_t parts, int64_t K) {
  RX_CHECK(parts >= 1 && rows >= 0 && K > 0, "bad sizes");
  RX_CHECK(K < (1ll << 30) && (rows + 127) / 128 * 128 * parts < (1ll << 30), "matrix too large");
}

int input_type(const at::Tensor& t, const char* name) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return fp4::kBf16In;
    case at::kHalf: return fp4::kF16In;
    case at::kFloat: return fp4::kF32In;
    default: RX_CHECK(false, name, " must be bfloat16, float16 or float32");
  }
  return 0;
}

bool aligned_rows(const at::Tensor& t) {
  return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 && (t.dim() == 1 || (t.stride(0) * t.element_size()) % 16 == 0);
}

const __nv_bfloat16* bias_ptr(const c10::optional<at::Tensor>& bias, int64_t n, int device) {
  if (!bias.has_value()) return nullptr;
  check_device(*bias, "bias", device);
  check_bf16(*bias, "bias");
  RX_CHECK(bias->dim() == 1 && bias->numel() == n && bias->is_contiguous(), "bias must be a contiguous vector of ", n);
  return reinterpret_cast<const __nv_bfloat16*>(bias->data_ptr());
}

void check_matrix(const at::Tensor& t, const char* name, int64_t rows, int64_t cols, int device) {
  check_device(t, name, device);
  check_bf16(t, name);
  RX_CHECK(t.dim() == 2 && t.size(0) == rows && t.size(1) == cols && t.stride(1) == 1, name, " must be a row-major [", rows,
           ", ", cols, "]");
}

void check_launch(cudaError_t e, const char* what) {
  RX_CHECK(e == cudaSuccess, what, ": ", cudaGetErrorString(e));
}

}  // namespace

// x [parts * rows, K] (bf16, fp16 or fp32) -> codes q, scales sf (both padded, see fp4.cuh) and, for
// NVFP4, the row factors.
void fp4_quantize(const at::Tensor& x, int64_t parts, int64_t fmt, at::Tensor& q, at::Tensor& sf,
                  const c10::optional<at::Tensor>& row_scale) {
  check_cuda(x, "x");
  check_format(fmt);
  RX_CHECK(x.dim() == 2 && (x.stride(1) == 1 || x.size(1) == 1), "x must be a matrix with unit inner stride");
  RX_CHECK(parts >= 1 && x.size(0) % parts == 0, "the rows of x must split into ", parts, " equal parts");
  const int64_t rows = x.size(0) / parts, K = x.size(1);
  const int dev = x.get_device();
  check_sizes(rows, parts, K);
  check_operand(q, sf, row_scale, rows, parts, K, fmt, dev, "quantize");
  const int type = input_type(x, "x");
  if (rows == 0) return;
  fp4::QuantParams p{};
  p.x = x.data_ptr();
  p.ldx = x.stride(0);
  p.rows = rows;
  p.parts = parts;
  p.K = static_cast<int>(K);
  p.q = q.data_ptr<uint8_t>();
  p.ldq = q.stride(0);
  p.sf = sf.data_ptr<uint8_t>();
  p.groups = scale_groups(K, fmt);
  p.row_scale = row_scale.has_value() ? row_scale->data_ptr<float>() : nullptr;
  c10::cuda::CUDAGuard guard(dev);
  check_launch(fp4::quantize(p, static_cast<int>(fmt), type, at::cuda::getCurrentCUDAStream(dev).stream()), "fp4_quantize");
}

// The values that codes and scales stand for, into out [parts * rows, K].
void fp4_dequantize(const at::Tensor& q, const at::Tensor& sf, const c10::optional<at::Tensor>& row_scale, int64_t parts,
                    int64_t fmt, at::Tensor& out) {
  check_cuda(out, "out");
  check_format(fmt);
  RX_CHECK(out.dim() == 2 && (out.stride(1) == 1 || out.size(1) == 1), "out must be a matrix with unit inner stride");
  RX_CHECK(parts >= 1 && out.size(0) % parts == 0, "the rows of out must split into ", parts, " equal parts");
  const int64_t rows = out.size(0) / parts, K = out.size(1);
  const int dev = out.get_device();
  check_sizes(rows, parts, K);
  check_operand(q, sf, row_scale, rows, parts, K, fmt, dev, "dequantize");
  const int type = input_type(out, "out");
  if (rows == 0) return;
  fp4::DequantParams p{};
  p.q = q.data_ptr<uint8_t>();
  p.ldq = q.stride(0);
  p.rows = rows;
  p.parts = parts;
  p.K = static_cast<int>(K);
  p.sf = sf.data_ptr<uint8_t>();
  p.groups = scale_groups(K, fmt);
  p.row_scale = row_scale.has_value() ? row_scale->data_ptr<float>() : nullptr;
  p.out = out.data_ptr();
  p.ldo = out.stride(0);
  c10::cuda::CUDAGuard guard(dev);
  check_launch(fp4::dequantize(p, static_cast<int>(fmt), type, at::cuda::getCurrentCUDAStream(dev).stream()),
               "fp4_dequantize");
}

// Products of 4-bit operands a [M, K] and b [parts * N, K]. parts 1: out = a b^T (+ bias) (+ residual);
// parts 2 (gate, up): act(a bg^T + bg) * (a bu^T + bu), into `out` or, as an MXFP4 operand, into q_out / q_sf.
void fp4_gemm(const at::Tensor& a, const at::Tensor& a_sf, const c10::optional<at::Tensor>& a_row, const at::Tensor& b,
              const at::Tensor& b_sf, const c10::optional<at::Tensor>& b_row, int64_t K, int64_t fmt, int64_t parts,
              int64_t act, const c10::optional<at::Tensor>& bias, const c10::optional<at::Tensor>& residual,
              const c10::optional<at::Tensor>& out, const c10::optional<at::Tensor>& q_out,
              const c10::optional<at::Tensor>& q_sf, const at::Tensor& status) {
  check_cuda(a, "a");
  check_format(fmt);
  RX_CHECK(parts == 1 || parts == 2, "b has one part, or two (gate and up)");
  RX_CHECK(a.dim() == 2 && b.dim() == 2 && b.size(0) % parts == 0, "operands must be matrices of whole parts");
  const int64_t M = a.size(0), N = b.size(0) / parts;
  const int dev = a.get_device();
  check_sizes(M, 1, K);
  check_sizes(N, parts, K);
  check_operand(a, a_sf, a_row, M, 1, K, fmt, dev, "a");
  check_operand(b, b_sf, b_row, N, parts, K, fmt, dev, "b");
  RX_CHECK(act >= 0 && act <= 3, "unknown activation code ", act);
  RX_CHECK(out.has_value() != q_out.has_value() && q_out.has_value() == q_sf.has_value(),
           "give out, or q_out with q_sf");
  RX_CHECK(!q_out.has_value() || (parts == 2 && fmt == kMx), "a quantised output belongs to the gated MXFP4 product");
  RX_CHECK(!residual.has_value() || parts == 1, "the gated product takes no residual");
  const auto* bias_p = bias_ptr(bias, parts * N, dev);
  if (out.has_value()) check_matrix(*out, "out", M, N, dev);
  if (residual.has_value()) check_matrix(*residual, "residual", M, N, dev);
  if (q_out.has_value()) check_operand(*q_out, *q_sf, c10::nullopt, M, 1, N, kMx, dev, "q_out");
  if (M == 0 || N == 0) return;
  c10::cuda::CUDAGuard guard(dev);
  auto stream = at::cuda::getCurrentCUDAStream(dev).stream();
  const bool few = M <= few::kMaxRows;
  const CUtensorMap ta = make_tmap_2d_u8(a.data_ptr(), M, a.size(1), a.stride(0), few ? few::tile_rows(M) : 128);
  const CUtensorMap tb = make_tmap_2d_u8(b.data_ptr(), parts * N, b.size(1), b.stride(0), 128);
  auto* out_p = out.has_value() ? reinterpret_cast<__nv_bfloat16*>(out->data_ptr()) : nullptr;
  const auto* res_p = residual.has_value() ? reinterpret_cast<const __nv_bfloat16*>(residual->data_ptr()) : nullptr;
  const auto* row_a = a_row.has_value() ? a_row->data_ptr<float>() : nullptr;
  const auto* row_b = b_row.has_value() ? b_row->data_ptr<float>() : nullptr;
  if (few) {
    few::Params p{};
    p.T = static_cast<int>(M);
    p.N = static_cast<int>(N);
    p.K = static_cast<int>(K);
    p.k_blocks = static_cast<int>((K + 255) / 256);
    p.gated = parts == 2;
    p.act = static_cast<int>(act);
    p.bias = bias_p;
    p.residual = res_p;
    p.ld_res = residual.has_value() ? residual->stride(0) : 0;
    p.out = out_p;
    p.ld_out = out.has_value() ? out->stride(0) : 0;
    p.sf_x = a_sf.data_ptr<uint8_t>();
    p.sf_w = b_sf.data_ptr<uint8_t>();
    p.groups = scale_groups(K, fmt);
    p.row_x = row_a;
    p.row_w = row_b;
    if (q_out.has_value()) {
      p.q_out = q_out->data_ptr<uint8_t>();
      p.ld_q = q_out->stride(0);
      p.q_sf = q_sf->data_ptr<uint8_t>();
      p.q_groups = scale_groups(N, kMx);
    }
    p.status = status_ptr(status);
    p.timeout_ns = kWaitBudgetNs;
    check_launch(few::launch(static_cast<int>(fmt), ta, tb, p, num_sms(dev), dev, stream), "fp4_gemm");
    return;
  }
  fp4::GemmParams p{};
  p.M = static_cast<int>(M);
  p.N = static_cast<int>(N);
  p.K = static_cast<int>(K);
  p.m_tiles = static_cast<int>(row_tiles(M));
  p.n_tiles = static_cast<int>(parts == 2 ? (N + 127) / 128 : (N + 255) / 256);
  RX_CHECK(static_cast<int64_t>(p.m_tiles) * p.n_tiles < (1ll << 31), "too many tiles");
  p.k_stages = static_cast<int>((K + 255) / 256);
  p.gated = parts == 2;
  p.act = static_cast<int>(act);
  p.sf_a = a_sf.data_ptr<uint8_t>();
  p.sf_b = b_sf.data_ptr<uint8_t>();
  p.groups = scale_groups(K, fmt);
  p.row_a = row_a;
  p.row_b = row_b;
  p.bias = bias_p;
  p.residual = res_p;
  p.ld_res = residual.has_value() ? residual->stride(0) : 0;
  p.out = out_p;
  p.ld_out = out.has_value() ? out->stride(0) : 0;
  p.vec = (!out.has_value() || aligned_rows(*out)) && (!residual.has_value() || aligned_rows(*residual)) &&
          (!bias.has_value() || (aligned_rows(*bias) && (parts == 1 || N % 8 == 0)));
  if (q_out.has_value()) {
    p.q_out = q_out->data_ptr<uint8_t>();
    p.ld_q = q_out->stride(0);
    p.q_sf = q_sf->data_ptr<uint8_t>();
    p.q_groups = scale_groups(N, kMx);
  }
  p.status = status_ptr(status);
  p.timeout_ns = kWaitBudgetNs;
  check_launch(fp4::gemm(ta, tb, p, static_cast<int>(fmt), num_sms(dev), dev, stream), "fp4_gemm");
}

// bf16 products of 1 to 64 token rows x [T, K] with w [parts * N, K]: parts 1: x w^T (+ bias) (+ residual);
// parts 2 (gate, up): act(x wg^T + bg) * (x wu^T + bu).
void few_rows_linear(const at::Tensor& x, const at::Tensor& w, int64_t parts, int64_t act,
                     const c10::optional<at::Tensor>& bias, const c10::optional<at::Tensor>& residual, at::Tensor& out,
                     const at::Tensor& status) {
  check_cuda(x, "x");
  RX_CHECK(parts == 1 || parts == 2, "w has one part, or two (gate and up)");
  RX_CHECK(x.dim() == 2 && w.dim() == 2 && w.size(0) % parts == 0, "x and w must be matrices, w of whole parts");
  const int64_t T = x.size(0), K = x.size(1), N = w.size(0) / parts;
  const int dev = x.get_device();
  RX_CHECK(T >= 1 && T <= few::kMaxRows, "few_rows_linear takes 1 to ", few::kMaxRows, " rows, got ", T);
  RX_CHECK(K >= 1 && N >= 1 && K < (1ll << 30) && N < (1ll << 29), "bad sizes");
  check_matrix(x, "x", T, K, dev);
  check_matrix(w, "w", parts * N, K, dev);
  check_matrix(out, "out", T, N, dev);
  RX_CHECK(act >= 0 && act <= 3, "unknown activation code ", act);
  RX_CHECK(!residual.has_value() || parts == 1, "the gated product takes no residual");
  if (residual.has_value()) check_matrix(*residual, "residual", T, N, dev);
  few::Params p{};
  p.bias = bias_ptr(bias, parts * N, dev);
  p.T = static_cast<int>(T);
  p.N = static_cast<int>(N);
  p.K = static_cast<int>(K);
  p.k_blocks = static_cast<int>((K + 63) / 64);
  p.gated = parts == 2;
  p.act = static_cast<int>(act);
  p.residual = residual.has_value() ? reinterpret_cast<const __nv_bfloat16*>(residual->data_ptr()) : nullptr;
  p.ld_res = residual.has_value() ? residual->stride(0) : 0;
  p.out = reinterpret_cast<__nv_bfloat16*>(out.data_ptr());
  p.ld_out = out.stride(0);
  p.status = status_ptr(status);
  p.timeout_ns = kWaitBudgetNs;
  c10::cuda::CUDAGuard guard(dev);
  const CUtensorMap tx = make_tmap_2d_bf16(x.data_ptr(), T, K, x.stride(0), 64, few::tile_rows(T));
  const CUtensorMap tw = make_tmap_2d_bf16(w.data_ptr(), parts * N, K, w.stride(0), 64, 128);
  check_launch(few::launch(few::kBf16, tx, tw, p, num_sms(dev), dev, at::cuda::getCurrentCUDAStream(dev).stream()),
               "few_rows_linear");
}

}  // namespace rx
