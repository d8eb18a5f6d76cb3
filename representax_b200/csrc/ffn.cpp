// Host entries of the gated feed-forward block: argument checks, tensor maps,
// and the block's forward and backward as one call each (its launches in a row,
// intermediates from the caching allocator on the current stream), so that a
// small call is not bound by the host.
#include "common.h"
#include "device_empty.h"
#include "few_rows.h"
#include "gated.h"

namespace rx {

void gemm_tcgen05(const at::Tensor& A, const at::Tensor& B, at::Tensor& C, bool a_mn, bool b_mn, int64_t epi,
                  int64_t out_mode, double alpha, const c10::optional<at::Tensor>& bias,
                  const c10::optional<at::Tensor>& aux_in, const c10::optional<at::Tensor>& aux_out,
                  const c10::optional<at::Tensor>& residual, const at::Tensor& status, int64_t split_k, int64_t variant,
                  int64_t drop_seed, int64_t drop_stream, double drop_p, const c10::optional<at::Tensor>& colsum);
void colsum_accumulate(const at::Tensor& x, at::Tensor& out);

namespace {

using OptTensor = c10::optional<at::Tensor>;

// The epilogue and output codes of gemm_kernel.cuh.
constexpr int64_t kBias = 1, kResidual = 8;
constexpr int64_t kOutBf16 = 0, kOutF32Atomic = 3;

void check_rows(const at::Tensor& t, const char* name, int64_t rows, int64_t cols, int device) {
  RX_CHECK(t.is_cuda() && t.get_device() == device, name, " must be on device ", device);
  RX_CHECK(t.dim() == 2 && t.size(0) == rows && t.size(1) == cols && t.stride(1) == 1, name, " must be a row-major [",
           rows, ", ", cols, "]");
  RX_CHECK((t.stride(0) * t.element_size()) % 16 == 0 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0, name,
           " rows must be 16-byte aligned");
}

void check_plain(const at::Tensor& t, const char* name, int64_t rows, int64_t cols, int device) {
  check_bf16(t, name);
  RX_CHECK(t.get_device() == device, name, " must be on device ", device);
  RX_CHECK(t.dim() == 2 && t.size(0) == rows && t.size(1) == cols && t.stride(1) == 1, name, " must be a row-major [", rows,
           ", ", cols, "]");
}

void check_sizes(int64_t T, int64_t H, int64_t I) {
  RX_CHECK(T > 0 && H > 0 && I > 0, "empty gated feed-forward");
  RX_CHECK(H % 8 == 0 && I % 8 == 0, "hidden and intermediate sizes must be multiples of 8");
  RX_CHECK(T < (1ll << 31) - 256 && H < (1ll << 30) && I < (1ll << 30), "gated feed-forward too large");
}

int64_t saved_tiles(int64_t T, int64_t I) { return (T + 31) / 32 * ((I + 31) / 32); }

// What the forward keeps (gated.h): fp16 [tiles, 2, 32, 32] and int16 [tiles, 32].
void check_saved(const at::Tensor& saved, const at::Tensor& exps, int64_t T, int64_t I, int device) {
  const int64_t tiles = saved_tiles(T, I);
  RX_CHECK(saved.is_cuda() && saved.get_device() == device && saved.scalar_type() == at::kHalf && saved.is_contiguous() &&
               saved.numel() == tiles * 2048 && reinterpret_cast<uintptr_t>(saved.data_ptr()) % 16 == 0,
           "saved must be a contiguous float16 array of ", tiles * 2048);
  RX_CHECK(exps.is_cuda() && exps.get_device() == device && exps.scalar_type() == at::kShort && exps.is_contiguous() &&
               exps.numel() == tiles * 32,
           "exps must be a contiguous int16 array of ", tiles * 32);
}

gated::Params make_params(int64_t T, int64_t I, int64_t H, int64_t tile_cols, const at::Tensor& status) {
  gated::Params p{};
  p.M = static_cast<int>(T);
  p.N = static_cast<int>(I);
  p.K = static_cast<int>(H);
  p.m_tiles = static_cast<int>((T + 255) / 256);
  p.n_tiles = static_cast<int>((I + tile_cols - 1) / tile_cols);
  RX_CHECK(static_cast<int64_t>(p.m_tiles) * p.n_tiles < (1ll << 31), "too many tiles");
  p.num_units = p.m_tiles * p.n_tiles;
  p.status = status_ptr(status);
  p.timeout_ns = kWaitBudgetNs;
  return p;
}

void run(int mode, const gated::Maps& maps, const gated::Params& p, int dev) {
  const cudaError_t e = gated::launch(mode, maps, p, num_sms(dev), dev, at::cuda::getCurrentCUDAStream(dev).stream());
  RX_CHECK(e == cudaSuccess, "gated feed-forward: ", cudaGetErrorString(e));
  count_launches();
}

// `t` if the tensor maps can read it (16-byte aligned rows), else a copy.
at::Tensor rows16(const at::Tensor& t) {
  const bool ok = t.stride(1) == 1 && (t.stride(0) * t.element_size()) % 16 == 0 && t.stride(0) >= t.size(1) &&
                  reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
  return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}

OptTensor vector16(const OptTensor& t) {
  if (!t.has_value()) return t;
  const bool ok = t->is_contiguous() && reinterpret_cast<uintptr_t>(t->data_ptr()) % 16 == 0;
  return ok ? t : OptTensor(t->clone(at::MemoryFormat::Contiguous));
}

// dy^T x: added into `acc` (fp32) where there is one, else a new tensor of type `dtype`.
at::Tensor weight_gradient(const at::Tensor& dy, const at::Tensor& x, const OptTensor& acc, at::ScalarType dtype,
                           const at::Tensor& status) {
  auto product = [&](at::Tensor& out, int64_t mode) {
    gemm_tcgen05(dy, x, out, true, true, 0, mode, 1.0, c10::nullopt, c10::nullopt, c10::nullopt, c10::nullopt, status, 0, 0,
                 0, 0, 0.0, c10::nullopt);
    count_launches();
  };
  if (acc.has_value()) {
    at::Tensor out = *acc;
    product(out, kOutF32Atomic);
    return at::Tensor();
  }
  const int64_t m = dy.size(1), n = x.size(1), k_blocks = (dy.size(0) + 63) / 64;
  const int64_t tiles = (m + 255) / 256 * ((n + 255) / 256);
  // Rounded once in the product's epilogue when its tiles (or a short contraction) leave nothing for a split of K to
  // gain over clearing, adding into and casting an fp32 buffer. Measured, epilogue / split: [768, 1152] over 2047 rows
  // 14.5 / 15.9 us, over 4096 23.5 / 29.7, over 8192 41.5 / 33.9; [768, 2304] over 8192 46.7 / 43.0; [2048, 6144]
  // over 8192 149 / 177.
  if (dtype == at::kBFloat16 && (2 * tiles >= num_sms(dy.get_device()) / 2 || k_blocks <= 64)) {
    at::Tensor out = device_empty({m, n}, at::kBFloat16, dy.get_device());
    product(out, kOutBf16);
    return out;
  }
  at::Tensor out = at::zeros({m, n}, dy.options().dtype(at::kFloat));
  product(out, kOutF32Atomic);
  return dtype == at::kFloat ? out : out.to(dtype);
}

at::Tensor bias_gradient(const at::Tensor& dy, const OptTensor& acc, at::ScalarType dtype) {
  at::Tensor out = acc.has_value() ? *acc : at::zeros({dy.size(1)}, dy.options().dtype(at::kFloat));
  colsum_accumulate(dy, out);
  count_launches((dy.size(1) + 8191) / 8192);  // blocks of columns
  if (acc.has_value()) return at::Tensor();
  return dtype == at::kFloat ? out : out.to(dtype);
}

// bf16 products of few token rows x [T, K] with w [parts * N, K]: parts 1: x w^T (+ bias) (+ residual);
// parts 2 (gate, up): act(x wg^T + bg) * (x wu^T + bu). `after_producer`: the launch just before, a gated projection,
// wrote x and nothing else that this one reads.
void few_rows_linear(const at::Tensor& x, const at::Tensor& w, int64_t parts, int64_t act,
                     const OptTensor& bias, const OptTensor& residual, at::Tensor& out,
                     bool after_producer, const at::Tensor& status) {
  check_cuda(x, "x");
  RX_CHECK(parts == 1 || parts == 2, "w has one part, or two (gate and up)");
  RX_CHECK(x.dim() == 2 && w.dim() == 2 && w.size(0) % parts == 0, "x and w must be matrices, w of whole parts");
  const int64_t T = x.size(0), K = x.size(1), N = w.size(0) / parts;
  const int dev = x.get_device();
  RX_CHECK(T >= 1 && T < (1ll << 20) && (parts == 1 || T <= 64), "few_rows_linear: too many rows, ", T);
  RX_CHECK(K >= 1 && N >= 1 && K < (1ll << 30) && N < (1ll << 29), "bad sizes");
  check_plain(x, "x", T, K, dev);
  check_plain(w, "w", parts * N, K, dev);
  check_plain(out, "out", T, N, dev);
  RX_CHECK(act >= 0 && act <= 3, "unknown activation code ", act);
  RX_CHECK(!residual.has_value() || parts == 1, "the gated product takes no residual");
  if (residual.has_value()) check_plain(*residual, "residual", T, N, dev);
  few::Params p{};
  if (bias.has_value()) {
    check_bf16(*bias, "bias");
    RX_CHECK(bias->get_device() == dev && bias->dim() == 1 && bias->numel() == parts * N && bias->is_contiguous(),
             "bias must be a contiguous vector of ", parts * N);
    p.bias = reinterpret_cast<const __nv_bfloat16*>(bias->data_ptr());
  }
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
  p.vec = reinterpret_cast<uintptr_t>(out.data_ptr()) % 8 == 0 && out.stride(0) % 4 == 0;
  p.after_producer = after_producer;
  p.status = status_ptr(status);
  p.timeout_ns = kWaitBudgetNs;
  c10::cuda::CUDAGuard guard(dev);
  const CUtensorMap tx = make_tmap_2d_bf16(x.data_ptr(), T, K, x.stride(0), 64, few::tile_rows(T));
  const CUtensorMap tw = make_tmap_2d_bf16(w.data_ptr(), parts * N, K, w.stride(0), 64, 128);
  const cudaError_t e =
      few::launch(few::kBf16, tx, tw, p, num_sms(dev), dev, at::cuda::getCurrentCUDAStream(dev).stream());
  RX_CHECK(e == cudaSuccess, "few_rows_linear: ", cudaGetErrorString(e));
  count_launches();
}

// h [T, I] = act(x Wg^T + bg) * (x Wu^T + bu) for x [T, H] and gate_up = [Wg; Wu] [2 I, H].
// With `saved` and `exps` (see check_saved) it also keeps what gated_backward reads.
void gated_forward(const at::Tensor& x, const at::Tensor& gate_up, const OptTensor& bias, at::Tensor& h,
                   const OptTensor& saved, const OptTensor& exps, int64_t act, const at::Tensor& status) {
  check_bf16(x, "x");
  check_bf16(gate_up, "gate_up");
  check_bf16(h, "h");
  RX_CHECK(x.dim() == 2 && gate_up.dim() == 2 && gate_up.size(0) % 2 == 0, "x and gate_up [2 I, H] must be matrices");
  const int64_t T = x.size(0), H = x.size(1), I = gate_up.size(0) / 2;
  const int dev = x.get_device();
  check_sizes(T, H, I);
  check_rows(x, "x", T, H, dev);
  check_rows(gate_up, "gate_up", 2 * I, H, dev);
  check_rows(h, "h", T, I, dev);
  RX_CHECK(act >= 0 && act <= 3, "unknown activation code ", act);
  RX_CHECK(saved.has_value() == exps.has_value(), "give saved and exps together");
  gated::Params p = make_params(T, I, H, 128, status);
  p.act = static_cast<int>(act);
  if (bias.has_value()) {
    check_bf16(*bias, "bias");
    RX_CHECK(bias->get_device() == dev && bias->dim() == 1 && bias->numel() == 2 * I && bias->is_contiguous() &&
                 reinterpret_cast<uintptr_t>(bias->data_ptr()) % 16 == 0,
             "bias must be a contiguous 16-byte aligned [2 I] vector");
    p.bias = reinterpret_cast<const __nv_bfloat16*>(bias->data_ptr());
  }
  c10::cuda::CUDAGuard guard(dev);
  gated::Maps maps;
  maps.a = make_tmap_2d_bf16(x.data_ptr(), T, H, x.stride(0), 64, 128);
  maps.b = make_tmap_2d_bf16(gate_up.data_ptr(), 2 * I, H, gate_up.stride(0), 64, 128);
  p.out[0] = reinterpret_cast<__nv_bfloat16*>(h.data_ptr());
  p.ld_out = h.stride(0);
  if (!saved.has_value()) {
    run(gated::kForward, maps, p, dev);
    return;
  }
  check_saved(*saved, *exps, T, I, dev);
  p.exps = reinterpret_cast<uint16_t*>(exps->data_ptr());
  p.saved = reinterpret_cast<uint4*>(saved->data_ptr());
  run(gated::kForwardSave, maps, p, dev);
}

// dz [T, 2 I] = [dh b | dh a] with dh = dy Wd (dy [T, H], down [H, I]) and what gated_forward saved.
// `partial` (fp32 [ceil(T / 32), 2 I]): also the column sums of dz over each 32 rows.
void gated_backward(const at::Tensor& dy, const at::Tensor& down, const at::Tensor& saved, const at::Tensor& exps,
                    at::Tensor& dz, const OptTensor& partial, const at::Tensor& status) {
  check_bf16(dy, "dy");
  check_bf16(down, "down");
  check_bf16(dz, "dz");
  RX_CHECK(dy.dim() == 2 && down.dim() == 2, "dy and down must be matrices");
  const int64_t T = dy.size(0), H = dy.size(1), I = down.size(1);
  const int dev = dy.get_device();
  check_sizes(T, H, I);
  check_rows(dy, "dy", T, H, dev);
  check_rows(down, "down", H, I, dev);
  check_rows(dz, "dz", T, 2 * I, dev);
  check_saved(saved, exps, T, I, dev);
  gated::Params p = make_params(T, I, H, 256, status);
  if (partial.has_value()) {
    check_f32(*partial, "partial");
    RX_CHECK(partial->get_device() == dev && partial->is_contiguous() && partial->numel() == (T + 31) / 32 * 2 * I,
             "partial must be a contiguous [ceil(T / 32), 2 I]");
    p.partial = partial->data_ptr<float>();
  }
  p.saved = reinterpret_cast<uint4*>(saved.data_ptr());
  p.exps = reinterpret_cast<uint16_t*>(exps.data_ptr());
  c10::cuda::CUDAGuard guard(dev);
  auto* zp = reinterpret_cast<__nv_bfloat16*>(dz.data_ptr());
  gated::Maps maps;
  maps.a = make_tmap_2d_bf16(dy.data_ptr(), T, H, dy.stride(0), 64, 128);
  maps.b = make_tmap_2d_bf16(down.data_ptr(), H, I, down.stride(0), 64, 64);
  p.out[0] = zp;
  p.out[1] = zp + I;
  p.ld_out = dz.stride(0);
  run(gated::kBackward, maps, p, dev);
}

}  // namespace

int64_t kernel_launches() { return launch_count().load(); }

// The block's forward: {y, h, saved, exps}; h, saved and exps are what the backward needs (saved and
// exps undefined without `save`).
std::vector<at::Tensor> gated_ffn_forward(const at::Tensor& x_in, const at::Tensor& gate_up_in, const at::Tensor& down_in,
                                          const OptTensor& gate_up_bias, const OptTensor& down_bias,
                                          const OptTensor& residual_in, int64_t act, bool save, const at::Tensor& status) {
  check_bf16(x_in, "x");
  const int dev = x_in.get_device();
  for (const OptTensor& t : {OptTensor(gate_up_in), OptTensor(down_in), gate_up_bias, down_bias, residual_in})
    RX_CHECK(!t.has_value() || (t->is_cuda() && t->get_device() == dev), "every operand must be on device ", dev, " of x");
  check_bf16(gate_up_in, "gate_up");
  check_bf16(down_in, "down");
  RX_CHECK(x_in.dim() == 2 && gate_up_in.dim() == 2 && down_in.dim() == 2, "x, gate_up and down must be matrices");
  c10::cuda::CUDAGuard guard(dev);
  const at::Tensor x = rows16(x_in), gate_up = rows16(gate_up_in), down = rows16(down_in);
  const OptTensor b1 = vector16(gate_up_bias), b2 = vector16(down_bias);
  const OptTensor residual = residual_in.has_value() ? OptTensor(rows16(*residual_in)) : residual_in;
  const int64_t T = x.size(0), I = down.size(1), H = down.size(0);
  at::Tensor h = device_empty({T, I}, at::kBFloat16, dev), y = device_empty({T, H}, at::kBFloat16, dev), saved, exps;
  const bool few_gated = !save && few::takes(few::kBf16, T, I, (H + 63) / 64, true);
  const bool few_down = few::takes(few::kBf16, T, H, (I + 63) / 64, false);
  if (save) {
    saved = device_empty({saved_tiles(T, I), 2, 32, 32}, at::kHalf, dev);
    exps = device_empty({saved_tiles(T, I), 32}, at::kShort, dev);
    gated_forward(x, gate_up, b1, h, saved, exps, act, status);
  } else if (few_gated) {
    few_rows_linear(x, gate_up, 2, act, b1, c10::nullopt, h, false, status);
  } else {
    gated_forward(x, gate_up, b1, h, c10::nullopt, c10::nullopt, act, status);
  }
  if (few_down) {
    few_rows_linear(h, down, 1, 0, b2, residual, y, true, status);
  } else {
    gemm_tcgen05(h, down, y, false, false, (b2.has_value() ? kBias : 0) | (residual.has_value() ? kResidual : 0), kOutBf16,
                 1.0, b2, c10::nullopt, c10::nullopt, residual, status, 0, 0, 0, 0, 0.0, c10::nullopt);
    count_launches();
  }
  return {y, h, saved, exps};
}

// The block's gradients {dx, dgate_up, ddown, dgate_up_bias, ddown_bias}, those that `need` asks for
// (in that order). A gradient with an fp32 accumulator `acc` is added into it, otherwise returned in
// the type of `like`.
std::vector<at::Tensor> gated_ffn_backward(const at::Tensor& dy_in, const OptTensor& x, const OptTensor& h,
                                           const at::Tensor& gate_up_in, const at::Tensor& down_in, const OptTensor& saved,
                                           const OptTensor& exps, const std::vector<bool>& need,
                                           const std::vector<OptTensor>& acc, const std::vector<at::ScalarType>& like,
                                           const at::Tensor& status) {
  check_bf16(dy_in, "dy");
  RX_CHECK(dy_in.dim() == 2 && need.size() == 5 && acc.size() == 5 && like.size() == 5, "bad gradient lists");
  c10::cuda::CUDAGuard guard(dy_in.get_device());
  const at::Tensor dy = rows16(dy_in);
  std::vector<at::Tensor> out(5);
  if (need[2]) {
    RX_CHECK(h.has_value(), "the gradient of down needs h");
    out[2] = weight_gradient(dy, rows16(*h), acc[2], like[2], status);
  }
  if (need[4]) out[4] = bias_gradient(dy, acc[4], like[4]);
  if (need[0] || need[1] || need[3]) {
    RX_CHECK(saved.has_value() && exps.has_value(), "the forward did not save for this gradient");
    const at::Tensor down = rows16(down_in);
    at::Tensor dz = device_empty({dy.size(0), 2 * down.size(1)}, at::kBFloat16, dy.get_device());
    at::Tensor partial;
    if (need[3]) partial = device_empty({(dy.size(0) + 31) / 32, 2 * down.size(1)}, at::kFloat, dy.get_device());
    gated_backward(dy, down, *saved, *exps, dz, need[3] ? OptTensor(partial) : c10::nullopt, status);
    if (need[1]) {
      RX_CHECK(x.has_value(), "the gradient of gate_up needs x");
      out[1] = weight_gradient(dz, rows16(*x), acc[1], like[1], status);
    }
    if (need[3]) {
      const int64_t cols = partial.size(1);
      const bool direct = !acc[3].has_value() && like[3] == at::kBFloat16;
      if (acc[3].has_value()) {
        check_f32(*acc[3], "accumulator");
        RX_CHECK(acc[3]->is_contiguous() && acc[3]->numel() == cols, "accumulator must be a contiguous vector of ", cols);
      }
      at::Tensor db = direct ? device_empty({cols}, at::kBFloat16, dy.get_device())
                             : (acc[3].has_value() ? *acc[3] : at::zeros({cols}, dy.options().dtype(at::kFloat)));
      const cudaError_t e = gated::sum_partials(
          partial.data_ptr<float>(), partial.size(0), cols, direct ? nullptr : db.data_ptr<float>(),
          direct ? reinterpret_cast<__nv_bfloat16*>(db.data_ptr()) : nullptr,
          at::cuda::getCurrentCUDAStream(dy.get_device()).stream());
      RX_CHECK(e == cudaSuccess, "gated feed-forward: ", cudaGetErrorString(e));
      count_launches();
      if (!acc[3].has_value()) out[3] = direct || like[3] == at::kFloat ? db : db.to(like[3]);
    }
    if (need[0]) {
      const at::Tensor gate_up = rows16(gate_up_in);
      out[0] = device_empty({dy.size(0), gate_up.size(1)}, at::kBFloat16, dy.get_device());
      gemm_tcgen05(dz, gate_up, out[0], false, true, 0, kOutBf16, 1.0, c10::nullopt, c10::nullopt, c10::nullopt,
                   c10::nullopt, status, 0, 0, 0, 0, 0.0, c10::nullopt);
      count_launches();
    }
  }
  return out;
}

}  // namespace rx
