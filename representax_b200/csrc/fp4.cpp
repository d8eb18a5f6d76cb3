// Host entries of the microscaled 4-bit kernels and of the kernels for few
// token rows: argument checks, tensor maps, dispatch.
#include "fp4.h"

#include "common.h"
#include "device_empty.h"
#include "few_rows.h"

namespace rx {

void gemm_tcgen05(const at::Tensor& A, const at::Tensor& B, at::Tensor& C, bool a_mn, bool b_mn, int64_t epi,
                  int64_t out_mode, double alpha, const c10::optional<at::Tensor>& bias,
                  const c10::optional<at::Tensor>& aux_in, const c10::optional<at::Tensor>& aux_out,
                  const c10::optional<at::Tensor>& residual, const at::Tensor& status, int64_t split_k, int64_t variant,
                  int64_t drop_seed, int64_t drop_stream, double drop_p, const c10::optional<at::Tensor>& colsum);

namespace {

using OptTensor = c10::optional<at::Tensor>;

constexpr int kMx = 1, kNv = 2;

int64_t scale_groups(int64_t k, int64_t fmt) { return (k + 255) / 256 * (fmt == kMx ? 2 : 4); }
int64_t row_tiles(int64_t rows) { return (rows + 127) / 128; }

void check_device(const at::Tensor& t, const char* name, int device) {
  RX_CHECK(t.is_cuda() && t.get_device() == device, name, " must be on device ", device);
}

// A matrix of parts * rows rows of K values in 4 bits (fp4.cuh).
struct Operand {
  uint8_t* q;
  int64_t ldq;
  uint8_t* sf;
  float* row;  // NVFP4
  int64_t rows, parts, K;
  int fmt;
  int64_t all_rows() const { return rows * parts; }
  int64_t code_bytes() const { return (K + 31) / 32 * 16; }  // of a row
  int64_t groups() const { return scale_groups(K, fmt); }
  int64_t scale_bytes() const { return parts * row_tiles(rows) * groups() * 512; }
  Operand part(int64_t i) const {
    Operand o = *this;
    o.parts = 1;
    o.q += i * rows * ldq;
    o.sf += i * row_tiles(rows) * groups() * 512;
    if (o.row != nullptr) o.row += i * rows;
    return o;
  }
};

void check_sizes(int64_t rows, int64_t parts, int64_t K) {
  RX_CHECK(parts >= 1 && rows >= 0 && K > 0, "bad sizes");
  RX_CHECK(K < (1ll << 24) && (rows + 127) / 128 * 128 * parts < (1ll << 30), "matrix too large");
}

// The operand that codes, scales and row factors hold, checked.
Operand operand(const at::Tensor& q, const at::Tensor& sf, const OptTensor& row_scale, int64_t parts, int64_t K, int64_t fmt,
                int device, const char* name) {
  RX_CHECK(fmt == kMx || fmt == kNv, "format must be 1 (MXFP4) or 2 (NVFP4), got ", fmt);
  check_device(q, name, device);
  check_device(sf, name, device);
  RX_CHECK(q.scalar_type() == at::kByte && sf.scalar_type() == at::kByte, name, ": codes and scales must be uint8");
  RX_CHECK(q.dim() == 2 && parts >= 1 && q.size(0) % parts == 0, name, ": codes must be a matrix of ", parts,
           " equal parts of rows");
  Operand o{};
  o.rows = q.size(0) / parts;
  o.parts = parts;
  o.K = K;
  o.fmt = static_cast<int>(fmt);
  check_sizes(o.rows, parts, K);
  RX_CHECK(q.size(1) == o.code_bytes() && (q.stride(1) == 1 || q.numel() == 0), name, ": rows of codes must be ",
           o.code_bytes(), " bytes");
  RX_CHECK(q.numel() == 0 || (q.stride(0) % 16 == 0 && q.stride(0) >= q.size(1) &&
                              reinterpret_cast<uintptr_t>(q.data_ptr()) % 16 == 0),
           name, ": rows of codes must be 16-byte aligned");
  RX_CHECK(sf.is_contiguous() && sf.numel() == o.scale_bytes() && reinterpret_cast<uintptr_t>(sf.data_ptr()) % 16 == 0, name,
           ": scales must be a contiguous, 16-byte aligned array of ", o.scale_bytes(), " bytes");
  RX_CHECK(row_scale.has_value() == (fmt == kNv), name, ": row factors belong to NVFP4 and only to it");
  if (row_scale.has_value()) {
    check_device(*row_scale, name, device);
    RX_CHECK(row_scale->scalar_type() == at::kFloat && row_scale->is_contiguous() && row_scale->numel() == q.size(0), name,
             ": row factors must be a contiguous float32 vector of ", q.size(0));
    o.row = row_scale->data_ptr<float>();
  }
  o.q = q.data_ptr<uint8_t>();
  o.ldq = q.stride(0);
  o.sf = sf.data_ptr<uint8_t>();
  return o;
}

// A temporary operand in one block of workspace (codes, scales, row factors).
struct Workspace {
  at::Tensor memory;
  Operand op;
  Workspace(int64_t rows, int64_t K, int fmt, int device) {
    op = Operand{nullptr, (K + 31) / 32 * 16, nullptr, nullptr, rows, 1, K, fmt};
    const int64_t codes = rows * op.ldq, scales = op.scale_bytes();
    memory = device_empty({codes + scales + (fmt == kNv ? 4 * rows : 0)}, at::kByte, device);
    op.q = memory.data_ptr<uint8_t>();
    op.sf = op.q + codes;
    if (fmt == kNv) op.row = reinterpret_cast<float*>(op.sf + scales);
  }
};

int input_type(const at::Tensor& t, const char* name) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return fp4::kBf16In;
    case at::kHalf: return fp4::kF16In;
    case at::kFloat: return fp4::kF32In;
    default: RX_CHECK(false, name, " must be bfloat16, float16 or float32");
  }
  return 0;
}

bool aligned_rows(const at::Tensor& t, uintptr_t bytes = 16) {
  return reinterpret_cast<uintptr_t>(t.data_ptr()) % bytes == 0 &&
         (t.dim() == 1 || (t.stride(0) * t.element_size()) % bytes == 0);
}

const __nv_bfloat16* bias_ptr(const OptTensor& bias, int64_t n, int device) {
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
  count_launches();
}

void check_input(const at::Tensor& x, int64_t parts) {
  check_cuda(x, "x");
  RX_CHECK(x.dim() == 2 && (x.stride(1) == 1 || x.size(1) <= 1), "x must be a matrix with unit inner stride");
  RX_CHECK(parts >= 1 && x.size(0) % parts == 0, "the rows of x must split into ", parts, " equal parts");
  check_sizes(x.size(0) / parts, parts, x.size(1));
}

void run_quantize(const at::Tensor& x, const Operand& o, cudaStream_t stream) {
  const int type = input_type(x, "x");
  if (o.rows == 0) return;
  fp4::QuantParams p{};
  p.x = x.data_ptr();
  p.ldx = x.stride(0);
  p.rows = o.rows;
  p.parts = o.parts;
  p.K = static_cast<int>(o.K);
  p.q = o.q;
  p.ldq = o.ldq;
  p.sf = o.sf;
  p.groups = o.groups();
  p.row_scale = o.row;
  check_launch(fp4::quantize(p, o.fmt, type, stream), "fp4_quantize");
}

void run_dequantize(const Operand& o, at::Tensor& out, cudaStream_t stream) {
  const int type = input_type(out, "out");
  if (o.rows == 0) return;
  fp4::DequantParams p{};
  p.q = o.q;
  p.ldq = o.ldq;
  p.rows = o.rows;
  p.parts = o.parts;
  p.K = static_cast<int>(o.K);
  p.sf = o.sf;
  p.groups = o.groups();
  p.row_scale = o.row;
  p.out = out.data_ptr();
  p.ldo = out.stride(0);
  check_launch(fp4::dequantize(p, o.fmt, type, stream), "fp4_dequantize");
}

// Tensor map of an operand's scales: rows of 512 bytes (128 32-bit words), boxes of one stage's groups.
CUtensorMap scale_map(const Operand& o) {
  CUtensorMap map;
  const int64_t rows = o.scale_bytes() / 512;
  RX_CHECK(rows < (1ll << 31), "too many scale groups");
  cuuint64_t dims[2] = {128u, static_cast<cuuint64_t>(rows)};
  cuuint64_t strides[1] = {512u};
  cuuint32_t box[2] = {128u, o.fmt == kMx ? 2u : 4u};
  cuuint32_t elem_strides[2] = {1, 1};
  const CUresult r = encode_tiled_fn()(&map, CU_TENSOR_MAP_DATA_TYPE_UINT32, 2, o.sf, dims, strides, box, elem_strides,
                                       CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE,
                                       CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  RX_CHECK(r == CUDA_SUCCESS, "cuTensorMapEncodeTiled (scales) failed with code ", static_cast<int>(r));
  return map;
}

// out = a b^T (+ bias) (+ residual) for one part of b; act(a bg^T + bg) * (a bu^T + bu) for two, into
// `out` or, in MXFP4, into the operand `q_out`. `after_producer`: a was written by the launch just before, which
// lets this one start early.
void run_product(const Operand& a, const Operand& b, int64_t act, const OptTensor& bias, const OptTensor& residual,
                 const at::Tensor* out, const Operand* q_out, bool after_producer, const at::Tensor& status, int dev,
                 cudaStream_t stream) {
  const int64_t M = a.rows, N = b.rows, K = a.K;
  RX_CHECK(a.parts == 1 && a.K == b.K && a.fmt == b.fmt, "operands differ in format or contraction");
  RX_CHECK(b.parts == 1 || b.parts == 2, "b has one part, or two (gate and up)");
  RX_CHECK(act >= 0 && act <= 3, "unknown activation code ", act);
  const auto* bias_p = bias_ptr(bias, b.all_rows(), dev);
  if (out != nullptr) check_matrix(*out, "out", M, N, dev);
  if (residual.has_value()) check_matrix(*residual, "residual", M, N, dev);
  if (M == 0 || N == 0) return;
  auto* out_p = out != nullptr ? reinterpret_cast<__nv_bfloat16*>(out->data_ptr()) : nullptr;
  const auto* res_p = residual.has_value() ? reinterpret_cast<const __nv_bfloat16*>(residual->data_ptr()) : nullptr;
  auto fill = [&](auto& p) {
    p.N = static_cast<int>(N);
    p.K = static_cast<int>(K);
    p.gated = b.parts == 2;
    p.act = static_cast<int>(act);
    p.bias = bias_p;
    p.residual = res_p;
    p.ld_res = residual.has_value() ? residual->stride(0) : 0;
    p.out = out_p;
    p.ld_out = out != nullptr ? out->stride(0) : 0;
    p.groups = a.groups();
    if (q_out != nullptr) {
      p.q_out = q_out->q;
      p.ld_q = q_out->ldq;
      p.q_sf = q_out->sf;
      p.q_groups = q_out->groups();
    }
    p.after_producer = after_producer;
    p.status = status_ptr(status);
    p.timeout_ns = kWaitBudgetNs;
  };
  const CUtensorMap tb = make_tmap_2d_u8(b.q, b.all_rows(), b.code_bytes(), b.ldq, 128);
  if (few::takes(a.fmt, M, N, (K + 255) / 256, b.parts == 2)) {
    const CUtensorMap ta = make_tmap_2d_u8(a.q, M, a.code_bytes(), a.ldq, few::tile_rows(M));
    few::Params p{};
    fill(p);
    p.T = static_cast<int>(M);
    p.k_blocks = static_cast<int>((K + 255) / 256);
    p.sf_x = a.sf;
    p.sf_w = b.sf;
    p.row_x = a.row;
    p.row_w = b.row;
    p.vec = out != nullptr && aligned_rows(*out, 8);
    check_launch(few::launch(a.fmt, ta, tb, p, num_sms(dev), dev, stream), "fp4 product");
    return;
  }
  fp4::GemmParams p{};
  fill(p);
  p.M = static_cast<int>(M);
  p.m_tiles = static_cast<int>((M + 255) / 256);
  p.n_tiles = static_cast<int>(b.parts == 2 ? (N + 127) / 128 : (N + 255) / 256);
  RX_CHECK(static_cast<int64_t>(p.m_tiles) * p.n_tiles < (1ll << 31), "too many tiles");
  p.k_stages = static_cast<int>((K + 255) / 256);
  p.a_tiles = static_cast<int>(row_tiles(M));
  p.b_tiles = static_cast<int>(row_tiles(N));
  p.row_a = a.row;
  p.row_b = b.row;
  p.vec = (out == nullptr || aligned_rows(*out)) && (!residual.has_value() || aligned_rows(*residual));
  fp4::GemmMaps maps;
  maps.a = make_tmap_2d_u8(a.q, M, a.code_bytes(), a.ldq, 128);
  maps.b = tb;
  maps.sf_a = scale_map(a);
  maps.sf_b = scale_map(b);
  maps.out = maps.a;
  if (p.vec && out != nullptr) maps.out = make_tmap_2d_bf16_store(out_p, M, N, p.ld_out);
  check_launch(fp4::gemm(maps, p, a.fmt, num_sms(dev), dev, stream), "fp4 product");
}

// out [M, parts * N] = a b^T (+ bias) (+ residual), part by part.
void run_linear(const Operand& a, const Operand& b, const OptTensor& bias, const OptTensor& residual, const at::Tensor& out,
                bool after_producer, const at::Tensor& status, int dev, cudaStream_t stream) {
  for (int64_t i = 0; i < b.parts; ++i) {
    if (b.parts == 1) {
      run_product(a, b, 0, bias, residual, &out, nullptr, after_producer, status, dev, stream);
      return;
    }
    const at::Tensor cut = out.narrow(1, i * b.rows, b.rows);
    run_product(a, b.part(i), 0, bias.has_value() ? OptTensor(bias->narrow(0, i * b.rows, b.rows)) : bias,
                residual.has_value() ? OptTensor(residual->narrow(1, i * b.rows, b.rows)) : residual, &cut, nullptr,
                after_producer && i == 0, status, dev, stream);
  }
}

// (a clone: a single column counts as contiguous whatever its inner stride says)
OptTensor unit_rows(const OptTensor& t) {
  if (!t.has_value() || t->dim() != 2 || t->stride(1) == 1) return t;
  return OptTensor(t->clone(at::MemoryFormat::Contiguous));
}

}  // namespace

// x [parts * rows, K] (bf16, fp16 or fp32) -> {codes, scales, row factors (NVFP4)}, the layout of fp4.cuh.
std::vector<at::Tensor> fp4_quantize(const at::Tensor& x, int64_t parts, int64_t fmt) {
  check_input(x, parts);
  RX_CHECK(fmt == kMx || fmt == kNv, "format must be 1 (MXFP4) or 2 (NVFP4), got ", fmt);
  const int64_t rows = x.size(0) / parts, K = x.size(1);
  const int dev = x.get_device();
  c10::cuda::CUDAGuard guard(dev);
  at::Tensor q = device_empty({x.size(0), (K + 31) / 32 * 16}, at::kByte, dev);
  at::Tensor sf = device_empty({parts * row_tiles(rows), scale_groups(K, fmt), 512}, at::kByte, dev);
  at::Tensor row;
  if (fmt == kNv) row = device_empty({x.size(0)}, at::kFloat, dev);
  const Operand o = operand(q, sf, fmt == kNv ? OptTensor(row) : c10::nullopt, parts, K, fmt, dev, "quantize");
  run_quantize(x, o, at::cuda::getCurrentCUDAStream(dev).stream());
  return {q, sf, row};
}

// The values that codes and scales stand for, into out [parts * rows, K].
void fp4_dequantize(const at::Tensor& q, const at::Tensor& sf, const OptTensor& row_scale, int64_t parts, int64_t fmt,
                    at::Tensor& out) {
  check_input(out, parts);
  const int dev = out.get_device();
  const Operand o = operand(q, sf, row_scale, parts, out.size(1), fmt, dev, "dequantize");
  RX_CHECK(o.all_rows() == out.size(0), "out must have the operand's rows");
  c10::cuda::CUDAGuard guard(dev);
  run_dequantize(o, out, at::cuda::getCurrentCUDAStream(dev).stream());
}

// bf16 [M, b rows] = a b^T (+ bias) (+ residual) for two operands of one format.
at::Tensor fp4_gemm(const at::Tensor& a, const at::Tensor& a_sf, const OptTensor& a_row, const at::Tensor& b,
                    const at::Tensor& b_sf, const OptTensor& b_row, int64_t parts, int64_t K, int64_t fmt,
                    const OptTensor& bias, const OptTensor& residual, const at::Tensor& status) {
  check_cuda(a, "a");
  const int dev = a.get_device();
  const Operand oa = operand(a, a_sf, a_row, 1, K, fmt, dev, "a"), ob = operand(b, b_sf, b_row, parts, K, fmt, dev, "b");
  c10::cuda::CUDAGuard guard(dev);
  at::Tensor out = device_empty({oa.rows, ob.all_rows()}, at::kBFloat16, dev);
  run_linear(oa, ob, bias, unit_rows(residual), out, false, status, dev, at::cuda::getCurrentCUDAStream(dev).stream());
  return out;
}

// bf16 [M, w rows] = Q(x) w^T (+ bias) (+ residual): the activations are quantised into workspace.
at::Tensor fp4_linear(const at::Tensor& x, const at::Tensor& w, const at::Tensor& w_sf, const OptTensor& w_row, int64_t parts,
                      int64_t fmt, const OptTensor& bias, const OptTensor& residual, const at::Tensor& status) {
  check_bf16(x, "x");
  check_input(x, 1);
  const int dev = x.get_device();
  const Operand ow = operand(w, w_sf, w_row, parts, x.size(1), fmt, dev, "weight");
  c10::cuda::CUDAGuard guard(dev);
  auto stream = at::cuda::getCurrentCUDAStream(dev).stream();
  at::Tensor out = device_empty({x.size(0), ow.all_rows()}, at::kBFloat16, dev);
  const Workspace xq(x.size(0), x.size(1), ow.fmt, dev);
  run_quantize(x, xq.op, stream);
  run_linear(xq.op, ow, bias, unit_rows(residual), out, true, status, dev, stream);
  return out;
}

// dx [M, K] = dy w for a 4-bit weight: its bf16 values (exact) in workspace, then the bf16 product.
at::Tensor fp4_linear_dgrad(const at::Tensor& dy_in, const at::Tensor& w, const at::Tensor& w_sf, const OptTensor& w_row,
                            int64_t parts, int64_t K, int64_t fmt, const at::Tensor& status) {
  check_bf16(dy_in, "dy");
  const int dev = dy_in.get_device();
  const Operand ow = operand(w, w_sf, w_row, parts, K, fmt, dev, "weight");
  const int64_t M = dy_in.size(0), N = ow.all_rows();
  RX_CHECK(dy_in.dim() == 2 && dy_in.size(1) == N, "dy must be [M, ", N, "]");
  c10::cuda::CUDAGuard guard(dev);
  if (M == 0 || N == 0) return at::zeros({M, K}, dy_in.options());
  at::Tensor dy = dy_in;
  if (!(dy.stride(1) == 1 && dy.stride(0) >= N && aligned_rows(dy))) {  // rows that the tensor map can read
    dy = device_empty({M, (N + 7) / 8 * 8}, at::kBFloat16, dev).narrow(1, 0, N);
    dy.copy_(dy_in);
  }
  const int64_t ld = (K + 7) / 8 * 8;
  at::Tensor wide = device_empty({N, ld}, at::kBFloat16, dev).narrow(1, 0, K);
  run_dequantize(ow, wide, at::cuda::getCurrentCUDAStream(dev).stream());
  at::Tensor dx = device_empty({M, ld}, at::kBFloat16, dev).narrow(1, 0, K);
  gemm_tcgen05(dy, wide, dx, false, true, 0, 0, 1.0, c10::nullopt, c10::nullopt, c10::nullopt, c10::nullopt, status, 0, 0, 0,
               0, 0.0, c10::nullopt);
  count_launches();
  return dx;
}

// The gated block over 4-bit operands: Q(h) down^T (+ bias) (+ residual), h = act(g) * u,
// [g u] = Q(x) gate_up^T (+ bias). In MXFP4 h leaves the first product as codes; in NVFP4 it passes
// through bf16, since its row factor needs the whole row.
at::Tensor fp4_ffn(const at::Tensor& x, const at::Tensor& gu, const at::Tensor& gu_sf, const OptTensor& gu_row,
                   int64_t gu_fmt, const at::Tensor& dn, const at::Tensor& dn_sf, const OptTensor& dn_row, int64_t dn_fmt,
                   int64_t act, const OptTensor& gu_bias, const OptTensor& dn_bias, const OptTensor& residual,
                   const at::Tensor& status) {
  check_bf16(x, "x");
  check_input(x, 1);
  const int dev = x.get_device();
  const Operand og = operand(gu, gu_sf, gu_row, 2, x.size(1), gu_fmt, dev, "gate_up");
  const Operand od = operand(dn, dn_sf, dn_row, 1, og.rows, dn_fmt, dev, "down");
  c10::cuda::CUDAGuard guard(dev);
  auto stream = at::cuda::getCurrentCUDAStream(dev).stream();
  const int64_t M = x.size(0);
  at::Tensor y = device_empty({M, od.rows}, at::kBFloat16, dev);
  const Workspace xq(M, x.size(1), og.fmt, dev), hq(M, og.rows, od.fmt, dev);
  run_quantize(x, xq.op, stream);
  if (og.fmt == kMx && od.fmt == kMx) {
    run_product(xq.op, og, act, gu_bias, c10::nullopt, nullptr, &hq.op, true, status, dev, stream);
  } else {
    const at::Tensor h = device_empty({M, og.rows}, at::kBFloat16, dev);
    run_product(xq.op, og, act, gu_bias, c10::nullopt, &h, nullptr, true, status, dev, stream);
    run_quantize(h, hq.op, stream);
  }
  run_product(hq.op, od, 0, dn_bias, unit_rows(residual), &y, nullptr, true, status, dev, stream);
  return y;
}

}  // namespace rx
