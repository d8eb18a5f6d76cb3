// Autograd nodes of the gated feed-forward block and of the 4-bit linear layer
// for plain bf16 parameters. They run the same host entries as the Python
// functions of ops/ffn.py and ops/fp4.py (which serve parameters with fp32
// accumulators, compute copies or sharding); a small training step spends most
// of its time on the host, and a node without Python halves that.
#include "common.h"

namespace rx {

using OptTensor = c10::optional<at::Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

std::vector<at::Tensor> gated_ffn_forward(const at::Tensor& x, const at::Tensor& gate_up, const at::Tensor& down,
                                          const OptTensor& gate_up_bias, const OptTensor& down_bias,
                                          const OptTensor& residual, int64_t act, bool save, const at::Tensor& status);
std::vector<at::Tensor> gated_ffn_backward(const at::Tensor& dy, const OptTensor& x, const OptTensor& h,
                                           const at::Tensor& gate_up, const at::Tensor& down, const OptTensor& saved,
                                           const OptTensor& exps, const std::vector<bool>& need,
                                           const std::vector<OptTensor>& acc, const std::vector<at::ScalarType>& like,
                                           const at::Tensor& status);
at::Tensor fp4_linear(const at::Tensor& x, const at::Tensor& w, const at::Tensor& w_sf, const OptTensor& w_row,
                      int64_t parts, int64_t fmt, const OptTensor& bias, const OptTensor& residual,
                      const at::Tensor& status);
at::Tensor fp4_linear_dgrad(const at::Tensor& dy, const at::Tensor& w, const at::Tensor& w_sf, const OptTensor& w_row,
                            int64_t parts, int64_t K, int64_t fmt, const at::Tensor& status);
void colsum_accumulate(const at::Tensor& x, at::Tensor& out);

namespace {

at::Tensor value(const OptTensor& t) { return t.has_value() ? *t : at::Tensor(); }
OptTensor maybe(const at::Tensor& t) { return t.defined() ? OptTensor(t) : c10::nullopt; }
bool wants(const OptTensor& t) { return t.has_value() && t->requires_grad(); }

struct GatedFfnNode : public torch::autograd::Function<GatedFfnNode> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& gate_up, const at::Tensor& down,
                            const OptTensor& gate_up_bias, const OptTensor& down_bias, const OptTensor& residual,
                            int64_t act, const at::Tensor& status) {
    const std::vector<bool> need = {x.requires_grad(), gate_up.requires_grad(), down.requires_grad(), wants(gate_up_bias),
                                    wants(down_bias)};
    auto out = gated_ffn_forward(x, gate_up, down, gate_up_bias, down_bias, residual, act, need[0] || need[1] || need[3],
                                 status);
    // kept only as far as the gradients asked for need it
    ctx->save_for_backward({need[1] ? x : at::Tensor(), gate_up, down, need[2] ? out[1] : at::Tensor(), out[2], out[3]});
    ctx->saved_data["need"] = std::vector<int64_t>(need.begin(), need.end());
    ctx->saved_data["residual"] = wants(residual);
    ctx->saved_data["status"] = status;
    return out[0];
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    std::vector<bool> need;
    for (const int64_t n : ctx->saved_data["need"].toIntVector()) need.push_back(n != 0);
    const at::Tensor& dy = grads[0];
    const auto g = gated_ffn_backward(dy, maybe(saved[0]), maybe(saved[3]), saved[1], saved[2], maybe(saved[4]),
                                      maybe(saved[5]), need, std::vector<OptTensor>(5),
                                      std::vector<at::ScalarType>(5, at::kBFloat16), ctx->saved_data["status"].toTensor());
    return {g[0], g[1], g[2], g[3], g[4], ctx->saved_data["residual"].toBool() ? dy : at::Tensor(), at::Tensor(),
            at::Tensor()};
  }
};

struct Fp4LinearNode : public torch::autograd::Function<Fp4LinearNode> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& w, const at::Tensor& w_sf,
                            const OptTensor& w_row, int64_t parts, int64_t fmt, const OptTensor& bias,
                            const OptTensor& residual, const at::Tensor& status) {
    at::Tensor y = fp4_linear(x, w, w_sf, w_row, parts, fmt, bias, residual, status);
    ctx->save_for_backward({w, w_sf, value(w_row)});
    ctx->saved_data["sizes"] = std::vector<int64_t>{parts, x.size(1), fmt};
    ctx->saved_data["need"] = std::vector<int64_t>{x.requires_grad(), wants(bias), wants(residual)};
    ctx->saved_data["status"] = status;
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const auto sizes = ctx->saved_data["sizes"].toIntVector(), need = ctx->saved_data["need"].toIntVector();
    const at::Tensor& dy = grads[0];
    variable_list out(9);
    if (need[0])
      out[0] = fp4_linear_dgrad(dy, saved[0], saved[1], maybe(saved[2]), sizes[0], sizes[1], sizes[2],
                                ctx->saved_data["status"].toTensor());
    if (need[1]) {
      const bool direct = dy.is_contiguous() && dy.size(0) > 0 && dy.size(1) % 8 == 0 &&
                          reinterpret_cast<uintptr_t>(dy.data_ptr()) % 16 == 0;
      at::Tensor db;
      if (direct) {
        db = at::zeros({dy.size(1)}, dy.options().dtype(at::kFloat));
        colsum_accumulate(dy, db);
        count_launches((dy.size(1) + 8191) / 8192);  // blocks of columns
      } else {
        db = at::sum(dy, at::IntArrayRef{0}, false, at::kFloat);
      }
      out[6] = db.to(at::kBFloat16);
    }
    if (need[2]) out[7] = dy;
    return out;
  }
};

}  // namespace

at::Tensor gated_ffn_apply(const at::Tensor& x, const at::Tensor& gate_up, const at::Tensor& down,
                           const OptTensor& gate_up_bias, const OptTensor& down_bias, const OptTensor& residual, int64_t act,
                           const at::Tensor& status) {
  return GatedFfnNode::apply(x, gate_up, down, gate_up_bias, down_bias, residual, act, status);
}

at::Tensor fp4_linear_apply(const at::Tensor& x, const at::Tensor& w, const at::Tensor& w_sf, const OptTensor& w_row,
                            int64_t parts, int64_t fmt, const OptTensor& bias, const OptTensor& residual,
                            const at::Tensor& status) {
  return Fp4LinearNode::apply(x, w, w_sf, w_row, parts, fmt, bias, residual, status);
}

}  // namespace rx
