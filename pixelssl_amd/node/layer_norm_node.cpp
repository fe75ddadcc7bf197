// The autograd node of functional.layer_norm / layer_norm_channels: layouts, workspaces and the calls of libpixelhip's
// pxl_layer_norm_* entry points.  The kernels of a small call take 10 - 20 us; as a Python autograd.Function the host took 104 us for
// forward + backward of 1003 x 777 (the backward runs on a thread of the engine, where Python is two to three times as slow), as this
// node 65 us.  Host code only; the C entry points come in through bind().
#include <ATen/hip/HIPContext.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include <optional>
#include <string>
#include <vector>

#include "../../include/pixelhip.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using MaybeTensor = std::optional<Tensor>;

struct Entry {
  decltype(&pxl_layer_norm_fwd) rows_fwd = nullptr;
  decltype(&pxl_layer_norm_bwd) rows_bwd = nullptr;
  decltype(&pxl_layer_norm_bwd_workspace) rows_ws = nullptr;
  decltype(&pxl_layer_norm_nchw_fwd) chan_fwd = nullptr;
  decltype(&pxl_layer_norm_nchw_bwd) chan_bwd = nullptr;
  decltype(&pxl_layer_norm_nchw_bwd_workspace) chan_ws = nullptr;
  decltype(&pxl_last_error) last_error = nullptr;
} lib;

void bind(const std::vector<size_t>& at) {
  TORCH_CHECK(at.size() == 7, "seven entry points");
  lib.rows_fwd = reinterpret_cast<decltype(lib.rows_fwd)>(at[0]);
  lib.rows_bwd = reinterpret_cast<decltype(lib.rows_bwd)>(at[1]);
  lib.rows_ws = reinterpret_cast<decltype(lib.rows_ws)>(at[2]);
  lib.chan_fwd = reinterpret_cast<decltype(lib.chan_fwd)>(at[3]);
  lib.chan_bwd = reinterpret_cast<decltype(lib.chan_bwd)>(at[4]);
  lib.chan_ws = reinterpret_cast<decltype(lib.chan_ws)>(at[5]);
  lib.last_error = reinterpret_cast<decltype(lib.last_error)>(at[6]);
}

void check(int rc) { TORCH_CHECK(rc == PXL_OK, "libpixelhip error ", rc, ": ", lib.last_error()); }

// elements between the rows of a tensor whose last axis is contiguous and whose leading axes form one evenly spaced run without
// overlap; -1 where they do not
int64_t row_stride(const Tensor& x) {
  const int64_t C = x.size(-1);
  if (x.stride(-1) != 1 && C > 1) return -1;
  int64_t step = -1, span = 1;
  for (int64_t k = x.dim() - 2; k >= 0; --k) {
    const int64_t n = x.size(k);
    if (n == 1) continue;
    if (step < 0) step = x.stride(k);
    else if (x.stride(k) != step * span) return -1;
    span *= n;
  }
  if (step < 0) return C;
  return step >= C ? step : -1;
}

inline int code(at::ScalarType t) { return t == at::kFloat ? PXL_F32 : PXL_BF16; }
inline const void* at_(const MaybeTensor& t) { return t.has_value() && t->defined() ? t->const_data_ptr() : nullptr; }
inline void* stream_of(const Tensor& x) { return at::hip::getCurrentHIPStream(x.get_device()).stream(); }

struct Shape { int64_t C, S, rows, stride; };      // S: positions of a map (channels form only)
Shape shape_of(const Tensor& x, bool channels) {
  Shape s;
  if (channels) {
    s.C = x.size(1);
    s.S = x.numel() ? x.numel() / (x.size(0) * s.C) : 0;
    s.rows = x.size(0) * s.S;
    s.stride = 0;
  } else {
    s.C = x.size(-1);
    s.S = 0;
    s.rows = x.numel() / s.C;
    s.stride = x.is_contiguous() ? s.C : row_stride(x);
  }
  return s;
}

// x as the kernels take it -> y, and the statistics [2][rows] when wanted
Tensor launch_forward(const Tensor& x, const MaybeTensor& w, const MaybeTensor& b, double eps, bool channels, int pcode, Tensor* stats) {
  const c10::DeviceGuard guard(x.device());
  const Shape s = shape_of(x, channels);
  Tensor y = x.is_contiguous() ? at::empty_like(x) : at::empty(x.sizes(), x.options());
  float *mean = nullptr, *rstd = nullptr;
  if (stats != nullptr) {
    *stats = at::empty({2 * s.rows}, x.options().dtype(at::kFloat));
    mean = stats->mutable_data_ptr<float>();
    rstd = mean + s.rows;
  }
  if (channels)
    check(lib.chan_fwd(code(x.scalar_type()), pcode, x.size(0), (int)s.C, s.S, x.const_data_ptr(), at_(w), at_(b), (float)eps, y.mutable_data_ptr(), mean,
                       rstd, stream_of(x)));
  else
    check(lib.rows_fwd(code(x.scalar_type()), pcode, s.rows, (int)s.C, s.stride, x.const_data_ptr(), at_(w), at_(b), (float)eps, y.mutable_data_ptr(), mean,
                       rstd, stream_of(x)));
  return y;
}

enum { CHANNELS = 1, HAS_W = 2, HAS_B = 4, P16 = 8 };

struct LayerNormNode : public torch::autograd::Function<LayerNormNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const MaybeTensor& w, const MaybeTensor& b, double eps, int64_t flags) {
    Tensor stats;
    Tensor y = launch_forward(x, w, b, eps, flags & CHANNELS, flags & P16 ? PXL_BF16 : PXL_F32, &stats);
    ctx->save_for_backward({x, flags & HAS_W ? *w : Tensor(), stats});
    ctx->saved_data["flags"] = flags;
    return y;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(5);
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &w = saved[1], &stats = saved[2];
    const int64_t flags = ctx->saved_data["flags"].toInt();
    const bool channels = flags & CHANNELS;
    const c10::DeviceGuard guard(x.device());
    const Tensor dy = grads[0].contiguous();
    const Shape s = shape_of(x, channels);
    // edges are numbered over the tensors that are there
    const bool need_x = ctx->needs_input_grad(0), need_w = flags & HAS_W && ctx->needs_input_grad(1),
               need_b = flags & HAS_B && ctx->needs_input_grad(flags & HAS_W ? 2 : 1);
    const int pcode = flags & P16 ? PXL_BF16 : PXL_F32;
    const auto params = x.options().dtype(pcode == PXL_F32 ? at::kFloat : at::kBFloat16);
    Tensor ws;
    size_t bytes = 0;
    if (need_x) out[0] = at::empty(x.sizes(), x.options());
    if (need_w) out[1] = at::empty({s.C}, params);
    if (need_b) out[2] = at::empty({s.C}, params);
    if (need_w || need_b) {
      bytes = channels ? lib.chan_ws(x.size(0), (int)s.C, s.S) : lib.rows_ws(s.rows, (int)s.C);
      ws = at::empty({(int64_t)bytes}, x.options().dtype(at::kByte));
    }
    auto ptr = [](const Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; };
    const float* mean = stats.const_data_ptr<float>();
    const void* wp = w.defined() ? w.const_data_ptr() : nullptr;
    if (channels)
      check(lib.chan_bwd(code(x.scalar_type()), pcode, x.size(0), (int)s.C, s.S, x.const_data_ptr(), dy.const_data_ptr(), wp, mean, mean + s.rows,
                         ptr(out[0]), ptr(out[1]), ptr(out[2]), ptr(ws), bytes, stream_of(x)));
    else
      check(lib.rows_bwd(code(x.scalar_type()), pcode, s.rows, (int)s.C, s.stride, x.const_data_ptr(), dy.const_data_ptr(), wp, mean, mean + s.rows,
                         ptr(out[0]), ptr(out[1]), ptr(out[2]), ptr(ws), bytes, stream_of(x)));
    if (at::GradMode::is_enabled()) {             // create_graph: the gradients can be had, gradients of them cannot
      variable_list have;
      for (int k = 0; k < 3; ++k)
        if (out[k].defined()) have.push_back(out[k]);
      auto node = std::make_shared<torch::autograd::DelayedError>("layer_norm is differentiable once", (int64_t)have.size());
      for (auto& t : have) t.requires_grad_(true);
      have = (*node)(std::move(have));
      size_t at = 0;
      for (int k = 0; k < 3; ++k)
        if (out[k].defined()) out[k] = have[at++];
    }
    return out;
  }
};

// Recorders see the allocations of a call but not its kernels (a traced module would return what its memory held before), a tangent would stop
// at the outputs, and torch.func's wrappers have no memory
bool beyond_reach(const Tensor& x, const MaybeTensor& w, const MaybeTensor& b) {
  if (torch::jit::tracer::isTracing() || c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::FuncTorchDynamicLayerFrontMode) ||
      c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY).has_value())
    return true;
  auto tangent = [](const Tensor& t) { return t._fw_grad(/*level=*/0).defined(); };
  return tangent(x) || (w.has_value() && w->defined() && tangent(*w)) || (b.has_value() && b->defined() && tangent(*b));
}

// y, or nothing where an argument is not as the kernels take it: functional._layer_norm then says what (the checks in Python take 2 - 3 us)
MaybeTensor layer_norm(const Tensor& x0, const MaybeTensor& w0, const MaybeTensor& b0, double eps, bool channels) {
  const bool has_w = w0.has_value() && w0->defined(), has_b = b0.has_value() && b0->defined();
  const at::ScalarType t = x0.scalar_type();
  if (!x0.is_cuda() || x0.layout() != at::kStrided || (t != at::kFloat && t != at::kBFloat16) || x0.dim() < (channels ? 2 : 1) || !(eps >= 0) || beyond_reach(x0, w0, b0))
    return {};
  const int64_t C = x0.size(channels ? 1 : -1);
  if (C < 1 || C > (1 << 24)) return {};
  for (const MaybeTensor* q : {&w0, &b0}) {
    if (!(q == &w0 ? has_w : has_b)) continue;
    const Tensor& v = **q;
    if (v.dim() != 1 || v.size(0) != C || v.device() != x0.device() || (v.scalar_type() != at::kFloat && v.scalar_type() != t) ||
        (has_w && v.scalar_type() != w0->scalar_type()))
      return {};
  }
  if (channels && x0.dim() == 4 && !x0.is_contiguous() && x0.is_contiguous(at::MemoryFormat::ChannelsLast))      // read as it lies
    return layer_norm(x0.permute({0, 2, 3, 1}), w0, b0, eps, false)->permute({0, 3, 1, 2});
  Tensor x = x0;
  if (!x.is_contiguous() && (channels || row_stride(x) < 0)) x = x.contiguous();
  const MaybeTensor w = has_w ? MaybeTensor(w0->contiguous()) : MaybeTensor(), b = has_b ? MaybeTensor(b0->contiguous()) : MaybeTensor();
  const at::ScalarType p = has_w ? w->scalar_type() : (has_b ? b->scalar_type() : at::kFloat);
  const int64_t flags = (channels ? CHANNELS : 0) | (has_w ? HAS_W : 0) | (has_b ? HAS_B : 0) | (p == at::kBFloat16 ? P16 : 0);
  if (at::GradMode::is_enabled() && (x.requires_grad() || (has_w && w->requires_grad()) || (has_b && b->requires_grad())))
    return LayerNormNode::apply(x, w, b, eps, flags);
  return launch_forward(x, w, b, eps, channels, flags & P16 ? PXL_BF16 : PXL_F32, nullptr);
}

}  // namespace

PYBIND11_MODULE(_pxlnode, m) {
  m.def("bind", &bind);
  m.def("row_stride", &row_stride);
  m.def("layer_norm", &layer_norm);
}
