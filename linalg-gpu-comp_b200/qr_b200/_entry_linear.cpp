// Compiled call path of the linear layer (include/qrb200_nn.h): argument checks with Python's
// error types, ATen outputs and workspace, torch's current stream of x's device.
#include "_entry.h"
#include "_overlap.h"

#include "qrb200_nn.h"

namespace qrb_entry {
namespace {

int activation_of(const std::string& name) {
  if (name == "none") return QRB_ACT_NONE;
  if (name == "relu") return QRB_ACT_RELU;
  if (name == "silu") return QRB_ACT_SILU;
  if (name == "gelu") return QRB_ACT_GELU;
  TORCH_CHECK_VALUE(false, "activation must be 'none', 'relu', 'silu' or 'gelu' (got '", name, "')");
}

int dtype_of(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return QRB_F32;
    case at::kBFloat16: return QRB_BF16;
    case at::kHalf: return QRB_F16;
    default: TORCH_CHECK_TYPE(false, "x must be float32, bfloat16 or float16 (got ", t.scalar_type(), ")");
  }
}

void check_like(const at::Tensor& t, const char* name, const at::Tensor& x, at::IntArrayRef shape) {
  TORCH_CHECK_TYPE(t.scalar_type() == x.scalar_type(), name, " must be ", x.scalar_type(), " like x (got ",
                   t.scalar_type(), ")");
  TORCH_CHECK_VALUE(t.sizes() == shape, name, " must have shape ", shape, " (got ", t.sizes(), ")");
  TORCH_CHECK_VALUE(t.device() == x.device(), name, " must be on ", x.device(), " (got ", t.device(), ")");
}

// Rows of a tensor as a matrix with dense rows that do not overlap, copied where its strides do not
// allow that.
struct Rows {
  at::Tensor t;
  int64_t ld;
  explicit Rows(const at::Tensor& x) {
    const int64_t cols = x.size(-1);
    t = x.dim() == 2 ? x : x.reshape({x.numel() / (cols > 0 ? cols : 1), cols});
    if (!((cols <= 1 || t.stride(1) == 1) && (t.size(0) <= 1 || t.stride(0) >= cols))) t = t.contiguous();
    // a single row has no stride: one that keeps rows 16-byte aligned
    ld = t.size(0) <= 1 ? (cols + 7) / 8 * 8 : t.stride(0);
  }
  const void* p() const { return t.data_ptr(); }
};

std::vector<int64_t> out_shape(const at::Tensor& x, int64_t n) {
  std::vector<int64_t> s = x.sizes().vec();
  s.back() = n;
  return s;
}

void check_x_w(const at::Tensor& x, const at::Tensor& w) {
  TORCH_CHECK_VALUE(x.dim() >= 1, "x must have at least one dimension");
  TORCH_CHECK_VALUE(w.dim() == 2, "w must have shape (n, k) (got ", w.sizes(), ")");
  TORCH_CHECK_VALUE(x.size(-1) >= 1 && w.size(0) >= 1, "k and n must be at least 1 (got ", x.size(-1), ", ", w.size(0),
                    ")");
  check_like(w, "w", x, {w.size(0), x.size(-1)});
}

void check_cuda(const at::Tensor& x) {
  TORCH_CHECK_VALUE(x.is_cuda(), "x must be a CUDA tensor (got ", x.device(), "); libqrb200 has no CPU path");
}

void* stream_of(const at::Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

std::tuple<at::Tensor, std::optional<at::Tensor>> forward(const at::Tensor& x, const at::Tensor& w,
                                                          const std::optional<at::Tensor>& bias,
                                                          const std::string& activation,
                                                          const std::optional<at::Tensor>& residual, bool want_pre,
                                                          const std::optional<at::Tensor>& out) {
  check_no_tangent("linear", x, w, bias, residual, out);
  qrb_linear_args a{};
  a.dtype = dtype_of(x);
  a.activation = activation_of(activation);
  check_x_w(x, w);
  const int64_t k = x.size(-1), n = w.size(0);
  const std::vector<int64_t> shape = out_shape(x, n);
  if (bias.has_value()) check_like(*bias, "bias", x, {n});
  if (residual.has_value()) check_like(*residual, "residual", x, shape);
  if (out.has_value()) {
    check_like(*out, "out", x, shape);
    TORCH_CHECK_VALUE(out->is_contiguous() || (out->dim() == 2 && out->stride(1) == 1 && out->stride(0) >= n),
                      "out must be contiguous, or a matrix of dense rows");
    // blocks write rows of the result while others still read these
    const Range to(*out);
    TORCH_CHECK_VALUE(!overlap(to, x) && !overlap(to, w) && !overlap(to, bias),
                      "out must not overlap x, w or bias");
    TORCH_CHECK_VALUE(!residual.has_value() || same_place(*out, *residual) || !overlap(to, *residual),
                      "out may be residual itself, but not overlap it otherwise");
  }
  check_cuda(x);
  c10::cuda::CUDAGuard guard(x.device());
  at::Tensor y = out.has_value() ? *out : at::empty(shape, x.options()), bc;
  std::optional<at::Tensor> pre;
  if (want_pre) pre = at::empty(shape, x.options());
  Rows xr(x), wr(w), yr(y);
  a.m = xr.t.size(0);
  a.k = k;
  a.n = n;
  a.x = xr.p();
  a.ldx = xr.ld;
  a.w = wr.p();
  a.ldw = wr.ld;
  if (bias.has_value()) {
    bc = bias->contiguous();
    a.bias = bc.data_ptr();
  }
  std::optional<Rows> rr;
  if (residual.has_value()) {
    rr.emplace(*residual);
    a.residual = rr->p();
    a.ldr = rr->ld;
  }
  a.y = y.data_ptr();
  a.ldy = yr.ld;
  if (want_pre) {
    a.pre = pre->data_ptr();
    a.ldpre = n;
  }
  const size_t nb = qrb_linear_workspace_size(&a);
  at::Tensor ws = at::empty({static_cast<int64_t>(nb)}, x.options().dtype(at::kByte));
  check_status(qrb_linear_forward(&a, ws.data_ptr(), nb, stream_of(x)));
  if (out.has_value()) written(y);
  return {y, pre};
}

std::tuple<std::optional<at::Tensor>, std::optional<at::Tensor>, std::optional<at::Tensor>> backward(
    const at::Tensor& dy, const at::Tensor& x, const at::Tensor& w, const std::string& activation,
    const std::optional<at::Tensor>& pre, bool with_dx, bool with_dw, bool with_bias) {
  check_no_tangent("linear_backward", dy, x, w, pre);
  qrb_linear_backward_args a{};
  a.dtype = dtype_of(x);
  a.activation = activation_of(activation);
  check_x_w(x, w);
  const int64_t k = x.size(-1), n = w.size(0);
  const std::vector<int64_t> shape = out_shape(x, n);
  check_like(dy, "dy", x, shape);
  const bool needs_pre = a.activation != QRB_ACT_NONE;
  TORCH_CHECK_VALUE(!needs_pre || pre.has_value(), "activation '", activation, "' needs pre, the forward pass's x w^T + bias");
  if (needs_pre) check_like(*pre, "pre", x, shape);
  check_cuda(x);
  c10::cuda::CUDAGuard guard(x.device());
  Rows dyr(dy), xr(x), wr(w);
  std::optional<Rows> pr;
  a.m = xr.t.size(0);
  a.k = k;
  a.n = n;
  a.dy = dyr.p();
  a.lddy = dyr.ld;
  a.x = xr.p();
  a.ldx = xr.ld;
  a.w = wr.p();
  a.ldw = wr.ld;
  if (needs_pre) {
    pr.emplace(*pre);
    a.pre = pr->p();
    a.ldpre = pr->ld;
  }
  std::optional<at::Tensor> dx, dw, db;
  if (with_dx) {
    dx = at::empty(x.sizes(), x.options());
    a.dx = dx->data_ptr();
  }
  if (with_dw) {
    dw = at::empty(w.sizes(), w.options());
    a.dw = dw->data_ptr();
  }
  if (with_bias) {
    db = at::empty({n}, w.options());
    a.dbias = db->data_ptr();
  }
  const size_t nb = qrb_linear_backward_workspace_size(&a);
  at::Tensor ws = at::empty({static_cast<int64_t>(nb)}, x.options().dtype(at::kByte));
  check_status(qrb_linear_backward(&a, ws.data_ptr(), nb, stream_of(x)));
  return {dx, dw, db};
}

}  // namespace

void bind_linear(pybind11::module_& m) {
  m.def("linear_forward", &forward);
  m.def("linear_backward", &backward);
}

}  // namespace qrb_entry
