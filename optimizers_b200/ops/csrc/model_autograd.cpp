// Autograd nodes of the decoder's operators.  They live here, not in Python, because a training step calls them hundreds of times: a Python
// node costs 30 to 60 us of host time per call (forward and backward), as much as the kernels of a small model take.
//
// Gradients are first order and taken one at a time: differentiating a gradient again, or a batch of incoming gradients, raises an error.
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <atomic>

namespace ob200 {

using torch::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

std::tuple<Tensor, Tensor, Tensor, Tensor> add_norm_fwd(const Tensor& x, const std::optional<Tensor>& r, const Tensor& w, double eps, int64_t out, bool want_rstd);
std::tuple<Tensor, Tensor, Tensor> add_norm_bwd(const Tensor& dy, const std::optional<Tensor>& dh, const Tensor& h, const Tensor& w, const Tensor& rstd, bool dx_bf16,
                                                bool want_dr);
Tensor embed_fwd(const Tensor& ids, const Tensor& table, double scale, bool out_bf16);
Tensor embed_bwd(const Tensor& ids, const Tensor& dy, int64_t V, double scale, bool out_bf16);
int64_t embed_bwd_launches(int64_t tokens);
std::tuple<Tensor, Tensor> fp8_rows(const Tensor& x);
std::tuple<Tensor, Tensor, Tensor, Tensor> fp8_both(const Tensor& x);
std::tuple<Tensor, Tensor, Tensor> fp8_squares(const Tensor& w, bool transpose);
Tensor fp8_matmul(const Tensor& a, const Tensor& sa, const Tensor& b, const Tensor& sb, bool column_scales, bool out_bf16, const std::optional<Tensor>& addend, Tensor status,
                  std::optional<std::vector<int64_t>> shape);

namespace {

std::atomic<int64_t> launches{0};

bool is_bf16(const Tensor& t) { return t.scalar_type() == torch::kBFloat16; }

// fp32 or bf16, contiguous: what the kernels read.  (A batch of incoming gradients at once has no memory of its own to read.)
Tensor readable(const Tensor& t) {
  TORCH_CHECK(t.has_storage(), "this operator takes one gradient at a time, no batch of them (is_grads_batched, vmap)");
  return (t.scalar_type() == torch::kFloat32 || is_bf16(t) ? t : t.to(torch::kFloat32)).contiguous();
}

// Gradients that raise an error where somebody differentiates them again: they depend on a leaf through what comes in or, `depends`, through what
// the node itself keeps.
variable_list once(const variable_list& incoming, variable_list out, bool recorded, bool depends) {
  if (!recorded) return out;
  bool any = depends;
  for (const auto& g : incoming) any = any || (g.defined() && g.requires_grad());
  if (!any) return out;
  torch::AutoGradMode on(true);
  for (auto& t : out)
    if (t.defined()) t = t.detach().requires_grad_(true);
  auto error = std::make_shared<torch::autograd::DelayedError>("this operator's gradient cannot be differentiated again", out.size());
  return (*error)(std::move(out));
}

struct AddNorm : torch::autograd::Function<AddNorm> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& r, const Tensor& w, double eps, bool out_bf16) {
    // An fp32 x is added to a residual in fp32.
    const Tensor rr = !is_bf16(x) && is_bf16(r) ? r.to(torch::kFloat32).contiguous() : r.contiguous();
    const Tensor ww = w.contiguous();
    auto [y, scale, h, rstd] = add_norm_fwd(x.contiguous(), rr, ww, eps, out_bf16 ? 1 : 0, true);
    ++launches;
    ctx->save_for_backward({h, ww, rstd});
    ctx->saved_data["x_bf16"] = is_bf16(x);
    ctx->saved_data["r_bf16"] = is_bf16(r);
    ctx->set_materialize_grads(false);
    return {y, h};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const bool recorded = torch::GradMode::is_enabled();
    torch::NoGradGuard no_grad;
    const auto saved = ctx->get_saved_variables();
    const Tensor &h = saved[0], &w = saved[1], &rstd = saved[2];
    const bool x_bf16 = ctx->saved_data["x_bf16"].toBool();
    const auto r_type = ctx->saved_data["r_bf16"].toBool() ? torch::kBFloat16 : torch::kFloat32;
    const auto x_type = x_bf16 ? torch::kBFloat16 : torch::kFloat32;
    const Tensor &dy = grads[0], &dh = grads[1];
    if (!dy.defined()) {  // only the sum was used
      if (!dh.defined()) return variable_list(5);
      return once(grads, {dh.to(x_type, false, true), dh.to(r_type, false, true), torch::zeros_like(w), Tensor(), Tensor()}, recorded, false);
    }
    auto [dx, dr, dw] = add_norm_bwd(readable(dy), dh.defined() ? std::optional<Tensor>(dh.to(h.scalar_type()).contiguous()) : std::nullopt, h, w, rstd, x_bf16, true);
    launches += 2;
    return once(grads, {dx, dr.scalar_type() == r_type ? dr : dr.to(r_type), dw, Tensor(), Tensor()}, recorded, true);
  }
};

struct Embedding : torch::autograd::Function<Embedding> {
  static Tensor forward(AutogradContext* ctx, const Tensor& ids, const Tensor& table, double scale, bool out_bf16) {
    const Tensor i = ids.contiguous();
    ctx->save_for_backward({i});
    ctx->saved_data["rows"] = table.size(0);
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["bf16"] = is_bf16(table);
    launches += i.numel() > 0;
    return embed_fwd(i, table.contiguous(), scale, out_bf16);
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const bool recorded = torch::GradMode::is_enabled();
    torch::NoGradGuard no_grad;
    const Tensor ids = ctx->get_saved_variables()[0];
    launches += embed_bwd_launches(ids.numel());
    Tensor dw = embed_bwd(ids, readable(grads[0]), ctx->saved_data["rows"].toInt(), ctx->saved_data["scale"].toDouble(), ctx->saved_data["bf16"].toBool());
    return once(grads, {Tensor(), dw, Tensor(), Tensor()}, recorded, false);
  }
};

Tensor bytes(const Tensor& padded, int64_t cols) { return padded.slice(1, 0, cols); }

constexpr int64_t kMostWeights = 32;

// Products of x [..., K] with weights [N_i, K] in 8 bits.  `learns`: bit 0 for x, bit 1 + i for weight i.
struct Fp8Linear : torch::autograd::Function<Fp8Linear> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, at::TensorList weights, bool out_bf16, const Tensor& status, int64_t learns) {
    const int64_t K = x.size(-1);
    const Tensor x2 = x.reshape({-1, K}).contiguous();
    const int64_t T = x2.size(0);
    const bool need_dx = learns & 1, need_dw = learns >> 1;
    Tensor q, s, qt, st;
    if (need_dw) std::tie(q, s, qt, st) = fp8_both(x2);
    else std::tie(q, s) = fp8_rows(x2);
    variable_list saved, out;
    // Operands are kept whole, with their padding: hooks on saved tensors may copy them, and a copy of a slice would lose its pitch.
    if (need_dw) saved = {qt, st.t()};
    std::vector<int64_t> sizes = x.sizes().vec(), shapes, types;
    for (const Tensor& w : weights) {
      auto [qw, qwt, sw] = fp8_squares(w.contiguous(), need_dx);
      sizes.back() = w.size(0);
      out.push_back(fp8_matmul(bytes(q, K), s.t(), bytes(qw, K), sw, false, out_bf16, std::nullopt, status, sizes));
      if (need_dx) {
        saved.push_back(qwt);
        saved.push_back(sw.t());
      }
      types.push_back(is_bf16(w));
      launches += 2;
    }
    ++launches;
    ctx->saved_data["status"] = status;  // a word of its own, no operand: whatever mode it was made in
    ctx->save_for_backward(std::move(saved));
    ctx->saved_data["learns"] = learns;
    ctx->saved_data["types"] = types;
    ctx->saved_data["shape"] = x.sizes().vec();
    ctx->saved_data["x_bf16"] = is_bf16(x);
    ctx->set_materialize_grads(false);
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const bool recorded = torch::GradMode::is_enabled();
    torch::NoGradGuard no_grad;
    const auto saved = ctx->get_saved_variables();
    const int64_t learns = ctx->saved_data["learns"].toInt();
    const bool need_dx = learns & 1, need_dw = learns >> 1;
    const auto types = ctx->saved_data["types"].toIntVector();
    const auto shape = ctx->saved_data["shape"].toIntVector();
    const Tensor status = ctx->saved_data["status"].toTensor();
    const size_t first = need_dw ? 2 : 0, n = types.size();
    size_t last = 0;
    for (size_t i = 0; i < n; ++i)
      if (grads[i].defined()) last = i;
    variable_list out(n + 4);
    Tensor dx;
    for (size_t i = 0; i < n; ++i) {
      if (!grads[i].defined()) continue;
      const bool want_dw = learns >> (1 + i) & 1;
      if (!need_dx && !want_dw) continue;
      const int64_t N = grads[i].size(-1);
      const Tensor dy = readable(grads[i].reshape({-1, N}));
      const int64_t T = dy.size(0);
      Tensor q, s, qt, st;
      if (want_dw) std::tie(q, s, qt, st) = fp8_both(dy);
      else std::tie(q, s) = fp8_rows(dy);
      ++launches;
      if (need_dx) {  // sums over several layers stay in 32 bits until the last
        const bool bf16 = i == last && ctx->saved_data["x_bf16"].toBool();
        dx = fp8_matmul(bytes(q, N), s.t(), bytes(saved[first + 2 * i], N), saved[first + 2 * i + 1], false, bf16, dx.defined() ? std::optional<Tensor>(dx) : std::nullopt, status, shape);
        ++launches;
      }
      if (want_dw) {
        out[1 + i] = fp8_matmul(bytes(qt, T), st.t(), bytes(saved[0], T), saved[1], true, types[i], std::nullopt, status, std::nullopt);
        ++launches;
      }
    }
    out[0] = dx;
    return once(grads, std::move(out), recorded, need_dx && need_dw);
  }
};

}  // namespace

std::tuple<Tensor, Tensor> add_rms_norm(const Tensor& x, const Tensor& r, const Tensor& w, double eps, bool out_bf16) {
  auto out = AddNorm::apply(x, r, w, eps, out_bf16);
  return {out[0], out[1]};
}

Tensor embedding(const Tensor& ids, const Tensor& table, double scale, bool out_bf16) { return Embedding::apply(ids, table, scale, out_bf16); }

std::vector<Tensor> fp8_linear(const Tensor& x, const std::vector<Tensor>& weights, bool out_bf16, const Tensor& status) {
  TORCH_CHECK_VALUE(static_cast<int64_t>(weights.size()) <= kMostWeights, "linear takes at most ", kMostWeights, " weights at once");
  int64_t learns = 0;
  if (torch::GradMode::is_enabled()) {
    learns = x.requires_grad();
    for (size_t i = 0; i < weights.size(); ++i) learns |= static_cast<int64_t>(weights[i].requires_grad()) << (1 + i);
  }
  return Fp8Linear::apply(x, at::TensorList(weights), out_bf16, status, learns);
}

// x [..., K] with weights that are held in 8 bits (e4m3 bytes [N_i, K], rows at multiples of 16 bytes, scales per square); no gradient.
std::vector<Tensor> fp8_linear_held(const Tensor& x, const std::vector<Tensor>& data, const std::vector<Tensor>& scales, bool out_bf16, const Tensor& status) {
  TORCH_CHECK(data.size() == scales.size(), "fp8: a scale for every weight");
  torch::NoGradGuard no_grad;
  const int64_t K = x.size(-1);
  auto [q, s] = fp8_rows(x.reshape({-1, K}).contiguous());
  ++launches;
  std::vector<int64_t> sizes = x.sizes().vec();
  std::vector<Tensor> out;
  for (size_t i = 0; i < data.size(); ++i) {
    sizes.back() = data[i].size(0);
    out.push_back(fp8_matmul(bytes(q, K), s.t(), data[i].view(torch::kUInt8), scales[i], false, out_bf16, std::nullopt, status, sizes));
    ++launches;
  }
  return out;
}

void register_model_autograd(pybind11::module_& m) {
  namespace py = pybind11;
  const auto unlocked = py::call_guard<py::gil_scoped_release>();
  m.def("add_rms_norm", &add_rms_norm, unlocked);
  m.def("embedding", &embedding, unlocked);
  m.def("fp8_linear", &fp8_linear, unlocked);
  m.def("fp8_linear_held", &fp8_linear_held, unlocked);
  m.def("model_op_launches", [] { return launches.load(); });
}

}  // namespace ob200
