// Compiled call path of the gated delta rule (include/qrb200_nn.h): argument checks with
// Python's error types, ATen outputs and workspace, torch's current stream of q's device.
#include "_entry.h"
#include "_overlap.h"

#include "qrb200_nn.h"

namespace qrb_entry {
namespace {

int dtype_of(const at::Tensor& t, const char* name) {
  switch (t.scalar_type()) {
    case at::kFloat: return QRB_F32;
    case at::kBFloat16: return QRB_BF16;
    case at::kHalf: return QRB_F16;
    default: TORCH_CHECK_TYPE(false, name, " must be float32, bfloat16 or float16 (got ", t.scalar_type(), ")");
  }
}

// (batch, time, heads, d) or, without a time dimension, (batch, heads, d): the last dimension is
// made dense, the others keep their strides.
at::Tensor dense_last(const at::Tensor& t) {
  return t.size(-1) <= 1 || t.stride(-1) == 1 ? t : t.contiguous();
}

void check_like(const at::Tensor& t, const char* name, const at::Tensor& q, at::ScalarType type,
                at::IntArrayRef shape) {
  TORCH_CHECK_TYPE(t.scalar_type() == type, name, " must be ", type, " (got ", t.scalar_type(), ")");
  TORCH_CHECK_VALUE(t.sizes() == shape, name, " must have shape ", shape, " (got ", t.sizes(), ")");
  TORCH_CHECK_VALUE(t.device() == q.device(), name, " must be on ", q.device(), " (got ", t.device(), ")");
}

qrb_strides strides4(const at::Tensor& t) { return {t.stride(0), t.stride(1), t.stride(2)}; }
qrb_strides strides3(const at::Tensor& t) { return {t.stride(0), 0, t.stride(1)}; }

float scale_of(std::optional<double> scale, int64_t dk) {
  return static_cast<float>(scale.has_value() ? *scale : 1.0 / std::sqrt(static_cast<double>(dk)));
}

void check_sizes(int64_t hk, int64_t hv, int64_t dk, int64_t dv) {
  TORCH_CHECK_VALUE(hk >= 1 && hv >= 1 && hv % hk == 0, "v must have a multiple of q's heads (got ", hv, " and ", hk, ")");
  TORCH_CHECK_VALUE(dk >= 1 && dk <= QRB_DELTA_MAX_DK, "q and k must have 1 to ", QRB_DELTA_MAX_DK,
                    " columns a head (got ", dk, ")");
  TORCH_CHECK_VALUE(dv >= 1 && dv <= QRB_DELTA_MAX_DV, "v must have 1 to ", QRB_DELTA_MAX_DV,
                    " columns a head (got ", dv, ")");
}

void check_cuda(const at::Tensor& q) {
  TORCH_CHECK_VALUE(q.is_cuda(), "q must be a CUDA tensor (got ", q.device(), "); libqrb200 has no CPU path");
}

struct Inputs {
  at::Tensor q, k, v, g, beta, init, offsets;
  qrb_delta_args a{};

  Inputs(const at::Tensor& q_, const at::Tensor& k_, const at::Tensor& v_, const at::Tensor& g_,
         const at::Tensor& beta_, std::optional<double> scale, const std::optional<at::Tensor>& initial_state,
         const std::optional<at::Tensor>& seq_offsets) {
    a.dtype = dtype_of(q_, "q");
    TORCH_CHECK_VALUE(q_.dim() == 4, "q must have shape (batch, time, heads, dk) (got ", q_.sizes(), ")");
    TORCH_CHECK_VALUE(v_.dim() == 4, "v must have shape (batch, time, heads, dv) (got ", v_.sizes(), ")");
    const int64_t b = q_.size(0), t = q_.size(1), hk = q_.size(2), dk = q_.size(3), hv = v_.size(2), dv = v_.size(3);
    check_like(k_, "k", q_, q_.scalar_type(), {b, t, hk, dk});
    check_like(v_, "v", q_, q_.scalar_type(), {b, t, hv, dv});
    check_like(g_, "g", q_, at::kFloat, {b, t, hv});
    check_like(beta_, "beta", q_, at::kFloat, {b, t, hv});
    check_sizes(hk, hv, dk, dv);
    int64_t nseq = b;
    if (seq_offsets.has_value()) {
      const at::Tensor& so = *seq_offsets;
      TORCH_CHECK_TYPE(so.scalar_type() == at::kInt || so.scalar_type() == at::kLong,
                       "seq_offsets must be int32 or int64 (got ", so.scalar_type(), ")");
      TORCH_CHECK_VALUE(so.dim() == 1 && so.size(0) >= 2, "seq_offsets must have shape (sequences + 1,) (got ",
                        so.sizes(), ")");
      TORCH_CHECK_VALUE(b == 1, "packed sequences need batch 1 (got ", b, ")");
      TORCH_CHECK_VALUE(so.device() == q_.device(), "seq_offsets must be on ", q_.device(), " (got ", so.device(), ")");
      nseq = so.size(0) - 1;
    }
    if (initial_state.has_value()) check_like(*initial_state, "initial_state", q_, at::kFloat, {nseq, hv, dk, dv});
    if (seq_offsets.has_value()) offsets = seq_offsets->to(at::kInt).contiguous();
    if (initial_state.has_value()) init = initial_state->contiguous();
    q = dense_last(q_);
    k = dense_last(k_);
    v = dense_last(v_);
    g = g_;
    beta = beta_;
    a.hk = static_cast<int>(hk);
    a.hv = static_cast<int>(hv);
    a.dk = static_cast<int>(dk);
    a.dv = static_cast<int>(dv);
    a.batch = b;
    a.time = t;
    a.nseq = nseq;
    a.scale = scale_of(scale, dk);
    a.q = q.data_ptr();
    a.k = k.data_ptr();
    a.v = v.data_ptr();
    a.g = g.data_ptr<float>();
    a.beta = beta.data_ptr<float>();
    a.q_strides = strides4(q);
    a.k_strides = strides4(k);
    a.v_strides = strides4(v);
    a.g_strides = strides4(g.unsqueeze(-1));
    a.beta_strides = strides4(beta.unsqueeze(-1));
    if (offsets.defined()) a.seq_offsets = offsets.data_ptr<int32_t>();
    if (init.defined()) a.initial_state = init.data_ptr<float>();
  }

  at::Tensor workspace(bool backward) const {
    const size_t n = qrb_delta_workspace_size(&a, backward);
    return at::empty({static_cast<int64_t>(n)}, q.options().dtype(at::kByte));
  }
  at::Tensor states() const { return at::empty({a.nseq, a.hv, a.dk, a.dv}, q.options().dtype(at::kFloat)); }
};

void* stream_of(const at::Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

std::tuple<at::Tensor, at::Tensor> forward(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                                           const at::Tensor& g, const at::Tensor& beta, std::optional<double> scale,
                                           const std::optional<at::Tensor>& initial_state,
                                           const std::optional<at::Tensor>& seq_offsets,
                                           const std::optional<at::Tensor>& out_o,
                                           const std::optional<at::Tensor>& out_state) {
  check_no_tangent("gated_delta_rule", q, k, v, g, beta, initial_state, out_o, out_state);
  Inputs in(q, k, v, g, beta, scale, initial_state, seq_offsets);
  if (out_o.has_value()) {
    check_like(*out_o, "out[0]", q, q.scalar_type(), v.sizes());
    TORCH_CHECK_VALUE(out_o->size(-1) <= 1 || out_o->stride(-1) == 1, "out[0] must be dense in its last dimension");
  }
  if (out_state.has_value()) {
    check_like(*out_state, "out[1]", q, at::kFloat, {in.a.nseq, in.a.hv, in.a.dk, in.a.dv});
    TORCH_CHECK_VALUE(out_state->is_contiguous(), "out[1] must be contiguous");
  }
  // What the recurrence writes while other blocks read: q, k, v, g and beta are not among it, the kernel before
  // lays them out.
  if (out_o.has_value()) {
    TORCH_CHECK_VALUE(out_o->is_contiguous() || !Runs(*out_o).meets_itself(), "out[0]'s elements must not share memory");
    const Range to(*out_o);
    TORCH_CHECK_VALUE(!overlap(to, initial_state) && !overlap(to, seq_offsets) && !overlap(to, out_state),
                      "out[0] must not overlap initial_state, seq_offsets or out[1]");
  }
  if (out_state.has_value()) {
    TORCH_CHECK_VALUE(!initial_state.has_value() || same_place(*out_state, *initial_state) ||
                          !overlap(*out_state, *initial_state),
                      "out[1] may be initial_state itself, but not overlap it otherwise");
    TORCH_CHECK_VALUE(!overlap(*out_state, seq_offsets), "out[1] must not overlap seq_offsets");
  }
  check_cuda(q);
  c10::cuda::CUDAGuard guard(q.device());
  at::Tensor o, s;
  if (out_o.has_value()) {
    o = *out_o;
  } else {
    o = at::empty(v.sizes(), v.options());
    in.a.zero_tail = 1;
  }
  if (out_state.has_value()) {
    s = *out_state;
  } else {
    s = in.states();
  }
  in.a.o = o.data_ptr();
  in.a.o_strides = strides4(o);
  in.a.final_state = s.data_ptr<float>();
  at::Tensor ws = in.workspace(false);
  check_status(qrb_delta_forward(&in.a, ws.data_ptr(), ws.numel(), stream_of(q)));
  if (out_o.has_value()) written(o);
  if (out_state.has_value()) written(s);
  return {o, s};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor, std::optional<at::Tensor>> backward(
    const at::Tensor& d_o, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& g,
    const at::Tensor& beta, std::optional<double> scale, const std::optional<at::Tensor>& initial_state,
    const std::optional<at::Tensor>& seq_offsets, const std::optional<at::Tensor>& dfinal_state) {
  check_no_tangent("gated_delta_rule_backward", d_o, q, k, v, g, beta, initial_state, dfinal_state);
  Inputs in(q, k, v, g, beta, scale, initial_state, seq_offsets);
  check_like(d_o, "do", q, q.scalar_type(), v.sizes());
  if (dfinal_state.has_value())
    check_like(*dfinal_state, "dfinal_state", q, at::kFloat, {in.a.nseq, in.a.hv, in.a.dk, in.a.dv});
  check_cuda(q);
  c10::cuda::CUDAGuard guard(q.device());
  at::Tensor d = dense_last(d_o), df, di;
  in.a.d_o = d.data_ptr();
  in.a.do_strides = strides4(d);
  if (dfinal_state.has_value()) {
    df = dfinal_state->contiguous();
    in.a.dfinal_state = df.data_ptr<float>();
  }
  at::Tensor dq = at::empty(q.sizes(), q.options()), dk = at::empty(k.sizes(), k.options()),
             dv = at::empty(v.sizes(), v.options()), dg = at::empty(g.sizes(), g.options()),
             db = at::empty(beta.sizes(), beta.options());
  std::optional<at::Tensor> dinit;
  if (initial_state.has_value()) {
    di = in.states();
    in.a.dinitial_state = di.data_ptr<float>();
    dinit = di;
  }
  in.a.dq = dq.data_ptr();
  in.a.dk_ = dk.data_ptr();
  in.a.dv_ = dv.data_ptr();
  in.a.dg = dg.data_ptr<float>();
  in.a.dbeta = db.data_ptr<float>();
  in.a.zero_tail = 1;
  at::Tensor ws = in.workspace(true);
  check_status(qrb_delta_backward(&in.a, ws.data_ptr(), ws.numel(), stream_of(q)));
  return {dq, dk, dv, dg, db, dinit};
}

at::Tensor step(const at::Tensor& q_, const at::Tensor& k_, const at::Tensor& v_, const at::Tensor& g,
                const at::Tensor& beta, const at::Tensor& state, std::optional<double> scale,
                const std::optional<at::Tensor>& slots, const std::optional<at::Tensor>& state_out,
                const std::optional<at::Tensor>& out) {
  TORCH_CHECK(!wants_grad(q_, k_, v_, g, beta, state, state_out, out),
              "gated_delta_step has no gradient: call it under torch.no_grad(), or train with gated_delta_rule");
  check_no_tangent("gated_delta_step", q_, k_, v_, g, beta, state, state_out, out);
  qrb_delta_step_args a{};
  a.dtype = dtype_of(q_, "q");
  TORCH_CHECK_VALUE(q_.dim() == 3, "q must have shape (batch, heads, dk) (got ", q_.sizes(), ")");
  TORCH_CHECK_VALUE(v_.dim() == 3, "v must have shape (batch, heads, dv) (got ", v_.sizes(), ")");
  const int64_t b = q_.size(0), hk = q_.size(1), dk = q_.size(2), hv = v_.size(1), dv = v_.size(2);
  check_like(k_, "k", q_, q_.scalar_type(), {b, hk, dk});
  check_like(v_, "v", q_, q_.scalar_type(), {b, hv, dv});
  check_like(g, "g", q_, at::kFloat, {b, hv});
  check_like(beta, "beta", q_, at::kFloat, {b, hv});
  check_sizes(hk, hv, dk, dv);
  TORCH_CHECK_VALUE(state.dim() == 4, "state must have shape (slots, heads, dk, dv) (got ", state.sizes(), ")");
  const at::Tensor& so = state_out.has_value() ? *state_out : state;
  for (const at::Tensor* s : {&state, &so}) {
    const char* name = s == &state ? "state" : "state_out";
    check_like(*s, name, q_, at::kFloat, {state.size(0), hv, dk, dv});
    TORCH_CHECK_VALUE(s->numel() == 0 || s->select(0, 0).is_contiguous(), name,
                      " must be dense in its last three dimensions");
    TORCH_CHECK_VALUE(s->size(0) <= 1 || s->stride(0) >= hv * dk * dv, name, "'s slots must not overlap");
  }
  if (slots.has_value()) check_like(*slots, "slots", q_, at::kInt, {b});
  else
    TORCH_CHECK_VALUE(state.size(0) >= b, "state must have a slot for each of the ", b, " rows (got ", state.size(0), ")");
  if (out.has_value()) {
    check_like(*out, "out", q_, q_.scalar_type(), v_.sizes());
    TORCH_CHECK_VALUE(out->is_contiguous(), "out must be contiguous");
  }
  // What some blocks write while others read: a block reads all of q and k, but of v only what it then writes.
  const Range to_state(so), read[] = {q_, k_, g, beta, slots}, rv(v_);
  auto meets = [&](const Range& t) {
    for (const Range& r : read)
      if (overlap(t, r)) return true;
    return false;
  };
  TORCH_CHECK_VALUE(&so == &state || same_place(so, state) || !overlap(to_state, state),
                    "state_out may be state itself, but not overlap it otherwise");
  TORCH_CHECK_VALUE(!meets(to_state) && !overlap(to_state, rv), "state_out must not overlap q, k, v, g, beta or slots");
  if (out.has_value()) {
    const Range to(*out);
    TORCH_CHECK_VALUE(!meets(to) && !overlap(to, state) && !overlap(to, to_state) &&
                          (same_place(*out, v_) || !overlap(to, rv)),
                      "out must not overlap q, k, g, beta, slots, state or state_out, nor v unless it is v itself");
  }
  check_cuda(q_);
  c10::cuda::CUDAGuard guard(q_.device());
  at::Tensor q = dense_last(q_), k = dense_last(k_), v = dense_last(v_), o, sl;
  if (out.has_value()) {
    o = *out;
  } else {
    o = at::empty(v_.sizes(), v_.options());
  }
  if (slots.has_value()) sl = slots->contiguous();
  a.hk = static_cast<int>(hk);
  a.hv = static_cast<int>(hv);
  a.dk = static_cast<int>(dk);
  a.dv = static_cast<int>(dv);
  a.batch = b;
  a.num_slots = state.size(0);
  a.scale = scale_of(scale, dk);
  a.q = q.data_ptr();
  a.k = k.data_ptr();
  a.v = v.data_ptr();
  a.q_strides = strides3(q);
  a.k_strides = strides3(k);
  a.v_strides = strides3(v);
  a.g = g.data_ptr<float>();
  a.beta = beta.data_ptr<float>();
  a.g_strides = {g.stride(0), 0, g.stride(1)};
  a.beta_strides = {beta.stride(0), 0, beta.stride(1)};
  a.slots = sl.defined() ? sl.data_ptr<int32_t>() : nullptr;
  a.state = state.data_ptr<float>();
  a.state_out = so.data_ptr<float>();
  a.slot_stride = state.stride(0);
  a.slot_stride_out = so.stride(0);
  a.o = o.data_ptr();
  check_status(qrb_delta_step(&a, stream_of(q)));
  written(so);
  if (out.has_value()) written(o);
  return o;
}

}  // namespace

void bind_delta(pybind11::module_& m) {
  m.def("delta_forward", &forward);
  m.def("delta_backward", &backward);
  m.def("delta_step", &step);
}

}  // namespace qrb_entry
