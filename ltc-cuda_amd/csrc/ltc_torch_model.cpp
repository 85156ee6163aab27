// Torch glue of the token model's operators: argument checks, allocations and autograd
// nodes around their C-ABI entry points (include/ltc_capi.h).
#include "ltc_torch_util.h"

namespace {

using namespace ltc_torch;

// B sequences of T steps, or packed ones of T tokens in all.
struct Sequences {
  int B, T;
  bool packed;
};

Sequences check_sequences(const Tensor& x, const Tensor& cu, const char* channels) {
  Sequences s;
  s.packed = cu.defined();
  type_of(x, "x");
  if (s.packed) {
    TORCH_CHECK_VALUE(x.dim() == 2, "packed x must be (tokens, ", channels, "), got ", x.sizes());
    TORCH_CHECK_TYPE(cu.scalar_type() == at::kInt, "cu_seqlens must be int32, got ", cu.scalar_type());
    TORCH_CHECK_VALUE(cu.dim() == 1 && cu.size(0) >= 1, "cu_seqlens must be (sequences + 1,), got ",
                      cu.sizes());
    check_device(cu, x, "cu_seqlens");
    s.B = as_int(cu.size(0) - 1, "sequences");
    s.T = as_int(x.size(0), "tokens");
  } else {
    TORCH_CHECK_VALUE(x.dim() == 3, "x must be (B, T, ", channels, "), got ", x.sizes());
    s.B = as_int(x.size(0), "B");
    s.T = as_int(x.size(1), "T");
  }
  TORCH_CHECK_VALUE(x.size(-1) >= 1, "x has no channels");
  check_device(x, x, "x");
  return s;
}

long long stride_b(const Tensor& t, bool packed) { return packed || !t.defined() ? 0 : t.stride(0); }
long long stride_t(const Tensor& t, bool packed) { return t.defined() ? t.stride(packed ? 0 : 1) : 0; }

Tensor rows_or_none(const Tensor& t) { return t.defined() ? rows(t) : Tensor(); }
Tensor dense(const Tensor& t) { return t.defined() ? t.contiguous() : Tensor(); }

// A gradient's tensor, where the pass wants it.
Tensor grad_of(const Tensor& t, bool wanted) {
  return t.defined() && wanted ? at::empty(t.sizes(), t.options()) : Tensor();
}

void check_like(const Tensor& t, const Tensor& x, const char* name) {
  TORCH_CHECK_TYPE(t.scalar_type() == x.scalar_type(), name, " must have x's type ", x.scalar_type(), ", got ",
                   t.scalar_type());
  TORCH_CHECK_VALUE(t.sizes() == x.sizes(), name, " must have x's shape ", x.sizes(), ", got ", t.sizes());
  check_device(t, x, name);
}

void check_float(const Tensor& t, const Tensor& x, at::IntArrayRef shape, const char* name) {
  TORCH_CHECK_VALUE(t.sizes() == shape, name, " must be ", shape, ", got ", t.sizes());
  TORCH_CHECK_TYPE(t.scalar_type() == at::kFloat, name, " must be float32, got ", t.scalar_type());
  check_device(t, x, name);
}

// Whether two tensors' memory, from the first byte to the last, has a byte in common.
bool extents_meet(const Tensor& a, const Tensor& b) {
  if (a.numel() == 0 || b.numel() == 0) return false;
  const auto span = [](const Tensor& t) {
    int64_t n = 1;
    for (int64_t d = 0; d < t.dim(); ++d) n += (t.size(d) - 1) * t.stride(d);
    const auto lo = reinterpret_cast<uintptr_t>(t.data_ptr());
    return std::make_pair(lo, lo + (uintptr_t)(n * t.element_size()));
  };
  const auto p = span(a), q = span(b);
  return p.first < q.second && q.first < p.second;
}

Tensor check_slots(const OptTensor& slots_opt, const Tensor& x, const Tensor& state, int B) {
  if (!slots_opt.has_value()) {
    TORCH_CHECK_VALUE(state.size(0) == B, "state must have ", B, " rows without slots, got ", state.sizes());
    return Tensor();
  }
  const Tensor& slots = *slots_opt;
  TORCH_CHECK_TYPE(slots.scalar_type() == at::kInt, "slots must be int32, got ", slots.scalar_type());
  TORCH_CHECK_VALUE(slots.dim() == 1 && slots.size(0) == B, "slots must be (", B, ",), got ", slots.sizes());
  check_device(slots, x, "slots");
  return slots.contiguous();
}

// ---------------------------------------------------------------------------
// Causal convolution
// ---------------------------------------------------------------------------
struct ConvSizes : Sequences {
  int C, K;
};

void check_taps(const Tensor& x, const Tensor& w, const Tensor& bias, int* C, int* K) {
  *C = as_int(x.size(-1), "C");
  TORCH_CHECK_VALUE(w.dim() == 2 && w.size(0) == *C && w.size(1) >= 1 && w.size(1) <= LTC_CONV_TAPS_MAX,
                    "weight must be (", *C, ", K) with K from 1 to ", LTC_CONV_TAPS_MAX, ", got ", w.sizes());
  *K = (int)w.size(1);
  TORCH_CHECK_TYPE(w.scalar_type() == x.scalar_type() || w.scalar_type() == at::kFloat,
                   "weight must have x's type or float32, got ", w.scalar_type());
  check_device(w, x, "weight");
  if (bias.defined()) {
    TORCH_CHECK_VALUE(bias.dim() == 1 && bias.size(0) == *C, "bias must be (", *C, ",), got ", bias.sizes());
    TORCH_CHECK_TYPE(bias.scalar_type() == w.scalar_type(), "bias must have weight's type ", w.scalar_type(),
                     ", got ", bias.scalar_type());
    check_device(bias, x, "bias");
  }
}

ConvSizes check_conv(const Tensor& x, const Tensor& w, const Tensor& bias, const Tensor& state,
                     const Tensor& cu) {
  ConvSizes s;
  static_cast<Sequences&>(s) = check_sequences(x, cu, "C");
  check_taps(x, w, bias, &s.C, &s.K);
  if (state.defined()) {
    TORCH_CHECK_VALUE(state.dim() == 3 && state.size(0) == s.B && state.size(1) == s.K - 1 &&
                          state.size(2) == s.C,
                      "state must be (", s.B, ", ", s.K - 1, ", ", s.C, "), got ", state.sizes());
    TORCH_CHECK_TYPE(state.scalar_type() == x.scalar_type(), "state must have x's type ", x.scalar_type(),
                     ", got ", state.scalar_type());
    check_device(state, x, "state");
  }
  return s;
}

struct CausalConvBackward : public Node {
  SavedVariable x_, w_, bias_, state_, cu_;
  int act = 0;
  std::string name() const override { return "CausalConvBackward"; }
  void release_variables() override {
    for (SavedVariable* v : {&x_, &w_, &bias_, &state_, &cu_}) v->reset_data();
  }
  variable_list apply(variable_list&& grads) override {
    variable_list g;
    {
      at::AutoDispatchBelowADInplaceOrView guard;
      g = run(grads);
    }
    return first_order(std::move(g), "ltc_causal_conv");
  }
  variable_list run(const variable_list& grads) {
    const Tensor x = x_.unpack(), w = w_.unpack(), bias = bias_.unpack(), state = state_.unpack(),
                 cu = cu_.unpack();
    c10::DeviceGuard on(x.device());
    check_capture(*this, x);
    const ConvSizes s = check_conv(x, w, bias, state, cu);
    Tensor go = grads[0], gh = grads[1];
    if (go.defined()) go = rows(go.to(x.scalar_type()));
    if (gh.defined()) gh = gh.to(x.scalar_type()).contiguous();
    const Tensor xr = rows(x), wc = w.contiguous(), bc = dense(bias), st = dense(state), cc = dense(cu);
    const Tensor gx = grad_of(x, task_should_compute_output(0)), gw = grad_of(w, task_should_compute_output(1)),
                 gb = grad_of(bias, task_should_compute_output(2)),
                 gs = grad_of(state, task_should_compute_output(3));
    const int type = type_of(x, "x");
    const long long bytes = ltc_causal_conv_bwd_workspace_bytes(type, s.B, s.T, s.C, s.K, s.packed);
    const Workspace ws(bytes, x);
    check_rc(ltc_causal_conv_backward(ptr(xr), stride_b(xr, s.packed), stride_t(xr, s.packed), ptr(wc), ptr(bc),
                                      ptr(st), static_cast<const int*>(ptr(cc)), type, type_of(w, "weight"), act,
                                      s.B, s.T, s.C, s.K, ptr(go), stride_b(go, s.packed),
                                      stride_t(go, s.packed), ptr(gh), ptr(gx), ptr(gw), ptr(gb), ptr(gs), ws.p,
                                      bytes, stream_of(x)),
             "ltc_causal_conv_backward");
    return {gx, gw, gb, gs};
  }
};

std::vector<Tensor> causal_conv(const Tensor& x, const Tensor& w, const OptTensor& bias_opt,
                                const OptTensor& state_opt, const OptTensor& cu_opt, int64_t act) {
  const Tensor bias = bias_opt.value_or(Tensor()), state = state_opt.value_or(Tensor()),
               cu = cu_opt.value_or(Tensor());
  check_modes("ltc_causal_conv", x, w, bias, state);
  const ConvSizes s = check_conv(x, w, bias, state, cu);
  const bool needs_grad =
      torch::GradMode::is_enabled() && torch::autograd::compute_requires_grad(x, w, bias, state);
  c10::DeviceGuard on(x.device());
  Tensor out, hf;
  {
    at::AutoDispatchBelowADInplaceOrView guard;
    const Tensor xr = rows(x), wc = w.contiguous(), bc = dense(bias), st = dense(state), cc = dense(cu);
    out = at::empty(x.sizes(), x.options());
    hf = at::empty({s.B, s.K - 1, s.C}, x.options());
    check_rc(ltc_causal_conv_forward(ptr(xr), stride_b(xr, s.packed), stride_t(xr, s.packed), ptr(wc), ptr(bc),
                                     ptr(st), static_cast<const int*>(ptr(cc)), type_of(x, "x"),
                                     type_of(w, "weight"), (int)act, s.B, s.T, s.C, s.K, ptr(out), ptr(hf),
                                     stream_of(x)),
             "ltc_causal_conv_forward");
  }
  if (needs_grad) {
    auto node = make_node<CausalConvBackward>();
    node->set_next_edges(torch::autograd::collect_next_edges(x, w, bias, state));
    node->x_ = SavedVariable(x, false);
    node->w_ = SavedVariable(w, false);
    node->bias_ = SavedVariable(bias, false);
    node->state_ = SavedVariable(state, false);
    node->cu_ = SavedVariable(cu, false);
    node->act = (int)act;
    torch::autograd::set_history(out, node);
    torch::autograd::set_history(hf, node);
  }
  return {out, hf};
}

Tensor causal_conv_step(const Tensor& x, const Tensor& w, const Tensor& state, const OptTensor& bias_opt,
                        const OptTensor& slots_opt, int64_t act) {
  const Tensor bias = bias_opt.value_or(Tensor());
  check_modes("ltc_causal_conv_step", x, w, state, bias);
  TORCH_CHECK_VALUE(x.dim() == 2 && x.size(1) >= 1, "x must be (B, C), got ", x.sizes());
  const int type = type_of(x, "x");
  check_device(x, x, "x");
  int C, K;
  check_taps(x, w, bias, &C, &K);
  const int B = as_int(x.size(0), "B");
  TORCH_CHECK_TYPE(state.scalar_type() == x.scalar_type(), "state must have x's type ", x.scalar_type(),
                   ", got ", state.scalar_type());
  TORCH_CHECK_VALUE(state.dim() == 3 && state.size(1) == K - 1 && state.size(2) == C, "state must be (rows, ",
                    K - 1, ", ", C, "), got ", state.sizes());
  check_device(state, x, "state");
  // written in place: a copy would not do
  const int64_t P = state.size(0);
  TORCH_CHECK_VALUE(state.stride(2) == 1 || C == 1, "state must have unit stride along its channels");
  TORCH_CHECK_VALUE((K <= 2 || state.stride(1) >= C) &&
                        (P <= 1 || K == 1 || state.stride(0) >= (K > 2 ? (K - 2) * state.stride(1) : 0) + C),
                    "the rows of state overlap");
  const Tensor slots = check_slots(slots_opt, x, state, B);
  TORCH_CHECK_VALUE(!extents_meet(x, state) && !extents_meet(w, state) &&
                        !(bias.defined() && extents_meet(bias, state)),
                    "the inputs must not share memory with state, which is written in place");
  TORCH_CHECK(!torch::GradMode::is_enabled() ||
                  !torch::autograd::compute_requires_grad(x, w, state, bias),
              "ltc_causal_conv_step has no backward: call it under torch.no_grad(), or ltc_causal_conv");
  c10::DeviceGuard on(x.device());
  Tensor out;
  {
    at::AutoDispatchBelowADInplaceOrView guard;
    const Tensor xr = rows(x), wc = w.contiguous(), bc = dense(bias);
    out = at::empty(x.sizes(), x.options());
    check_rc(ltc_causal_conv_step(ptr(xr), xr.stride(0), ptr(wc), ptr(bc), ptr(state), state.stride(0),
                                  state.stride(1), static_cast<const int*>(ptr(slots)), type,
                                  type_of(w, "weight"), (int)act, B, C, K, as_int(P, "rows"), ptr(out),
                                  stream_of(x)),
             "ltc_causal_conv_step");
  }
  // saved copies of the state are stale now
  if (!state.is_inference()) torch::autograd::impl::bump_version(state);
  return out;
}

// ---------------------------------------------------------------------------
// Selective scan
// ---------------------------------------------------------------------------
struct ScanInputs {
  Tensor x, delta, A, B, C, D, z, bias, state, cu;
};

struct ScanSizes : Sequences {
  int H, N, G;
  bool grouped;  // B and C have a dimension of groups
};

// A (H,N), and B and C with `lead` dimensions before theirs: (..., N) or (..., G, N).
void check_states(const Tensor& x, const Tensor& A, const Tensor& B, const Tensor& C, ScanSizes* s) {
  s->H = as_int(x.size(-1), "H");
  TORCH_CHECK_VALUE(A.dim() == 2 && A.size(0) == s->H && A.size(1) >= 1 && A.size(1) <= LTC_STATES_MAX,
                    "A must be (", s->H, ", N) with N from 1 to ", LTC_STATES_MAX, ", got ", A.sizes());
  s->N = (int)A.size(1);
  check_float(A, x, A.sizes(), "A");
  const int64_t lead = x.dim() - 1;
  s->grouped = B.dim() == lead + 2;
  TORCH_CHECK_VALUE((s->grouped || B.dim() == lead + 1) && B.size(-1) == s->N &&
                        B.sizes().slice(0, lead) == x.sizes().slice(0, lead),
                    "B must be x's tokens by N or by (groups, N), with N = ", s->N, ", got ", B.sizes());
  s->G = s->grouped ? as_int(B.size(-2), "groups") : 1;
  TORCH_CHECK_VALUE(s->G >= 1 && s->H % s->G == 0, "the channels, ", s->H, ", must be a multiple of the groups, ",
                    s->G);
  TORCH_CHECK_VALUE(C.sizes() == B.sizes(), "C must have B's shape ", B.sizes(), ", got ", C.sizes());
  for (const auto& [t, name] : {std::make_pair(&B, "B"), std::make_pair(&C, "C")}) {
    TORCH_CHECK_TYPE(t->scalar_type() == x.scalar_type(), name, " must have x's type ", x.scalar_type(), ", got ",
                     t->scalar_type());
    check_device(*t, x, name);
  }
}

ScanSizes check_scan(const ScanInputs& in) {
  ScanSizes s;
  static_cast<Sequences&>(s) = check_sequences(in.x, in.cu, "H");
  check_like(in.delta, in.x, "delta");
  check_states(in.x, in.A, in.B, in.C, &s);
  if (in.z.defined()) check_like(in.z, in.x, "z");
  if (in.D.defined()) check_float(in.D, in.x, {s.H}, "D");
  if (in.bias.defined()) check_float(in.bias, in.x, {s.H}, "delta_bias");
  if (in.state.defined()) check_float(in.state, in.x, {s.B, s.H, s.N}, "state");
  return s;
}

// The inputs as the library reads them.
ScanInputs readable(const ScanInputs& in) {
  return {rows(in.x),  rows(in.delta), in.A.contiguous(), rows(in.B),      rows(in.C),
          dense(in.D), rows_or_none(in.z), dense(in.bias), dense(in.state), dense(in.cu)};
}

long long stride_g(const Tensor& t, const ScanSizes& s) { return s.grouped ? t.stride(-2) : 0; }

struct SelectiveScanBackward : public Node {
  SavedVariable x_, delta_, A_, B_, C_, D_, z_, bias_, state_, cu_, saved_;
  bool softplus = false;
  std::string name() const override { return "SelectiveScanBackward"; }
  void release_variables() override {
    for (SavedVariable* v :
         {&x_, &delta_, &A_, &B_, &C_, &D_, &z_, &bias_, &state_, &cu_, &saved_})
      v->reset_data();
  }
  variable_list apply(variable_list&& grads) override {
    variable_list g;
    {
      at::AutoDispatchBelowADInplaceOrView guard;
      g = run(grads);
    }
    return first_order(std::move(g), "ltc_selective_scan");
  }
  variable_list run(const variable_list& grads) {
    const ScanInputs in{x_.unpack(), delta_.unpack(), A_.unpack(),    B_.unpack(),     C_.unpack(),
                        D_.unpack(), z_.unpack(),     bias_.unpack(), state_.unpack(), cu_.unpack()};
    const Tensor saved = saved_.unpack();
    c10::DeviceGuard on(in.x.device());
    check_capture(*this, in.x);
    const ScanSizes s = check_scan(in);
    const ScanInputs r = readable(in);
    const bool p = s.packed;
    Tensor go = grads[0], gh = grads[1];
    if (go.defined()) go = rows(go.to(in.x.scalar_type()));
    if (gh.defined()) gh = gh.to(at::kFloat).contiguous();
    const Tensor* of[] = {&in.x, &in.delta, &in.A, &in.B, &in.C, &in.D, &in.z, &in.bias, &in.state};
    variable_list g;
    for (int i = 0; i < 9; ++i) g.push_back(grad_of(*of[i], task_should_compute_output(i)));
    const long long bytes = ltc_selective_scan_bwd_workspace_bytes(s.B, s.T, s.H, s.N, s.G, p);
    const Workspace ws(bytes, in.x);
    check_rc(ltc_selective_scan_backward(
                 ptr(r.x), stride_b(r.x, p), stride_t(r.x, p), ptr(r.delta), stride_b(r.delta, p),
                 stride_t(r.delta, p), fp(r.A), ptr(r.B), stride_b(r.B, p), stride_t(r.B, p), stride_g(r.B, s),
                 ptr(r.C), stride_b(r.C, p), stride_t(r.C, p), stride_g(r.C, s), fp(r.D), ptr(r.z),
                 stride_b(r.z, p), stride_t(r.z, p), fp(r.bias), fp(r.state), static_cast<const int*>(ptr(r.cu)),
                 type_of(in.x, "x"), softplus, s.B, s.T, s.H, s.N, s.G, fp(saved), ptr(go), stride_b(go, p),
                 stride_t(go, p), fp(gh), ptr(g[0]), ptr(g[1]), fp(g[2]), ptr(g[3]), ptr(g[4]), fp(g[5]),
                 ptr(g[6]), fp(g[7]), fp(g[8]), ws.p, bytes, stream_of(in.x)),
             "ltc_selective_scan_backward");
    return g;
  }
};

std::vector<Tensor> selective_scan(const Tensor& x, const Tensor& delta, const Tensor& A, const Tensor& B,
                                   const Tensor& C, const OptTensor& D, const OptTensor& z,
                                   const OptTensor& bias, const OptTensor& state, const OptTensor& cu,
                                   bool softplus) {
  const ScanInputs in{x,
                      delta,
                      A,
                      B,
                      C,
                      D.value_or(Tensor()),
                      z.value_or(Tensor()),
                      bias.value_or(Tensor()),
                      state.value_or(Tensor()),
                      cu.value_or(Tensor())};
  check_modes("ltc_selective_scan", x, delta, A, B, C, in.D, in.z, in.bias, in.state);
  const ScanSizes s = check_scan(in);
  const bool p = s.packed;
  const bool needs_grad =
      torch::GradMode::is_enabled() &&
      torch::autograd::compute_requires_grad(x, delta, A, B, C, in.D, in.z, in.bias, in.state);
  c10::DeviceGuard on(x.device());
  Tensor out, hf, saved;
  {
    at::AutoDispatchBelowADInplaceOrView guard;
    const ScanInputs r = readable(in);
    out = at::empty(x.sizes(), x.options());
    hf = at::empty({s.B, s.H, s.N}, x.options().dtype(at::kFloat));
    if (needs_grad) {
      const long long n = ltc_selective_scan_saved_floats(s.B, s.T, s.H, s.N, s.G, p);
      TORCH_CHECK(n >= 0, ltc_last_error());
      saved = at::empty({n}, x.options().dtype(at::kFloat));
    }
    const long long bytes = ltc_selective_scan_fwd_workspace_bytes(s.B, s.T, s.H, s.N, s.G, p);
    const Workspace ws(bytes, x);
    check_rc(ltc_selective_scan_forward(
                 ptr(r.x), stride_b(r.x, p), stride_t(r.x, p), ptr(r.delta), stride_b(r.delta, p),
                 stride_t(r.delta, p), fp(r.A), ptr(r.B), stride_b(r.B, p), stride_t(r.B, p), stride_g(r.B, s),
                 ptr(r.C), stride_b(r.C, p), stride_t(r.C, p), stride_g(r.C, s), fp(r.D), ptr(r.z),
                 stride_b(r.z, p), stride_t(r.z, p), fp(r.bias), fp(r.state), static_cast<const int*>(ptr(r.cu)),
                 type_of(x, "x"), softplus, s.B, s.T, s.H, s.N, s.G, needs_grad, ptr(out), fp(hf), fp(saved),
                 ws.p, bytes, stream_of(x)),
             "ltc_selective_scan_forward");
  }
  if (needs_grad) {
    auto node = make_node<SelectiveScanBackward>();
    node->set_next_edges(
        torch::autograd::collect_next_edges(x, delta, A, B, C, in.D, in.z, in.bias, in.state));
    node->x_ = SavedVariable(x, false);
    node->delta_ = SavedVariable(delta, false);
    node->A_ = SavedVariable(A, false);
    node->B_ = SavedVariable(B, false);
    node->C_ = SavedVariable(C, false);
    node->D_ = SavedVariable(in.D, false);
    node->z_ = SavedVariable(in.z, false);
    node->bias_ = SavedVariable(in.bias, false);
    node->state_ = SavedVariable(in.state, false);
    node->cu_ = SavedVariable(in.cu, false);
    node->saved_ = SavedVariable(saved, false);
    node->softplus = softplus;
    torch::autograd::set_history(out, node);
    torch::autograd::set_history(hf, node);
  }
  return {out, hf};
}

Tensor selective_scan_step(const Tensor& x, const Tensor& delta, const Tensor& A, const Tensor& B,
                           const Tensor& C, const Tensor& state, const OptTensor& D_opt, const OptTensor& z_opt,
                           const OptTensor& bias_opt, const OptTensor& slots_opt, bool softplus) {
  const Tensor D = D_opt.value_or(Tensor()), z = z_opt.value_or(Tensor()), bias = bias_opt.value_or(Tensor());
  check_modes("ltc_selective_scan_step", x, delta, A, B, C, state, D, z, bias);
  TORCH_CHECK_VALUE(x.dim() == 2 && x.size(1) >= 1, "x must be (B, H), got ", x.sizes());
  const int type = type_of(x, "x");
  check_device(x, x, "x");
  check_like(delta, x, "delta");
  ScanSizes s;
  check_states(x, A, B, C, &s);
  if (z.defined()) check_like(z, x, "z");
  if (D.defined()) check_float(D, x, {s.H}, "D");
  if (bias.defined()) check_float(bias, x, {s.H}, "delta_bias");
  const int rows_ = as_int(x.size(0), "B");
  TORCH_CHECK_VALUE(state.dim() == 3, "state must be (rows, ", s.H, ", ", s.N, "), got ", state.sizes());
  check_float(state, x, {state.size(0), s.H, s.N}, "state");
  // written in place: a copy would not do
  TORCH_CHECK_VALUE((s.N == 1 || state.stride(2) == 1) && (s.H == 1 || state.stride(1) == s.N),
                    "each row of state must be contiguous");
  TORCH_CHECK_VALUE(state.size(0) <= 1 || state.stride(0) >= (int64_t)s.H * s.N, "the rows of state overlap");
  const Tensor slots = check_slots(slots_opt, x, state, rows_);
  for (const Tensor& t : {x, delta, A, B, C, D, z, bias})
    TORCH_CHECK_VALUE(!t.defined() || !extents_meet(t, state),
                      "the inputs must not share memory with state, which is written in place");
  TORCH_CHECK(!torch::GradMode::is_enabled() ||
                  !torch::autograd::compute_requires_grad(x, delta, A, B, C, state, D, z, bias),
              "ltc_selective_scan_step has no backward: call it under torch.no_grad(), or ltc_selective_scan");
  c10::DeviceGuard on(x.device());
  Tensor out;
  {
    at::AutoDispatchBelowADInplaceOrView guard;
    const Tensor xr = rows(x), dr = rows(delta), Ac = A.contiguous(), Br = rows(B), Cr = rows(C), Dc = dense(D),
                 zr = rows_or_none(z), bc = dense(bias);
    out = at::empty(x.sizes(), x.options());
    check_rc(ltc_selective_scan_step(ptr(xr), xr.stride(0), ptr(dr), dr.stride(0), fp(Ac), ptr(Br),
                                     Br.stride(0), stride_g(Br, s), ptr(Cr), Cr.stride(0), stride_g(Cr, s),
                                     fp(Dc), ptr(zr), zr.defined() ? zr.stride(0) : 0, fp(bc), fp(state),
                                     state.stride(0), static_cast<const int*>(ptr(slots)), type, softplus, rows_,
                                     s.H, s.N, s.G, as_int(state.size(0), "rows"), ptr(out), stream_of(x)),
             "ltc_selective_scan_step");
  }
  // saved copies of the state are stale now
  if (!state.is_inference()) torch::autograd::impl::bump_version(state);
  return out;
}

// ---------------------------------------------------------------------------
// Embedding
// ---------------------------------------------------------------------------
struct EmbedBackward : public Node {
  SavedVariable ids_;
  int V = 0, H = 0;
  double scale = 1;
  at::TensorOptions options;
  std::string name() const override { return "EmbedBackward"; }
  void release_variables() override { ids_.reset_data(); }
  variable_list apply(variable_list&& grads) override {
    if (!grads[0].defined()) return {Tensor()};
    Tensor g;
    {
      at::AutoDispatchBelowADInplaceOrView guard;
      const Tensor ids = ids_.unpack();
      c10::DeviceGuard on(ids.device());
      check_capture(*this, ids);
      const int64_t n = ids.numel();
      const Tensor id = ids.contiguous();
      g = at::empty({V, H}, options);
      const Tensor go = flat(grads[0].to(g.scalar_type()), n, H);
      const long long bytes = ltc_embed_bwd_workspace_bytes(n, V, H);
      const Workspace ws(bytes, g);
      check_rc(ltc_embed_backward(ptr(id), ids.scalar_type() == at::kLong, type_of(g, "table"), n, V, H,
                                  (float)scale, ptr(go), go.stride(0), ptr(g), ws.p, bytes, stream_of(g)),
               "ltc_embed_backward");
    }
    return first_order({g}, "ltc_embed");
  }
};

Tensor embed(const Tensor& table, const Tensor& ids, double scale) {
  check_modes("ltc_embed", table);
  type_of(table, "table");
  TORCH_CHECK_VALUE(table.dim() == 2 && table.size(0) >= 1 && table.size(1) >= 1, "table must be (V, H), got ",
                    table.sizes());
  check_device(table, table, "table");
  const int id64 = check_ids(ids, table, "ids");
  TORCH_CHECK_VALUE(std::isfinite((float)scale), "scale must be finite, got ", scale);
  const int V = as_int(table.size(0), "V"), H = as_int(table.size(1), "H");
  const bool needs_grad = torch::GradMode::is_enabled() && table.requires_grad();
  c10::DeviceGuard on(table.device());
  Tensor out;
  {
    at::AutoDispatchBelowADInplaceOrView guard;
    const Tensor t = rows(table), id = ids.contiguous();
    auto shape = ids.sizes().vec();
    shape.push_back(H);
    out = at::empty(shape, table.options());
    check_rc(ltc_embed_forward(ptr(t), t.stride(0), ptr(id), id64, type_of(table, "table"), id.numel(), V, H,
                               (float)scale, ptr(out), stream_of(table)),
             "ltc_embed_forward");
  }
  if (needs_grad) {
    auto node = make_node<EmbedBackward>();
    node->set_next_edges(torch::autograd::collect_next_edges(table));
    node->ids_ = SavedVariable(ids, false);
    node->V = V;
    node->H = H;
    node->scale = scale;
    node->options = at::TensorOptions().dtype(table.scalar_type()).device(table.device());
    torch::autograd::set_history(out, node);
  }
  return out;
}

// ---------------------------------------------------------------------------
// Adjustments of logits
// ---------------------------------------------------------------------------
// (..., n) of the logits' rows, or (n,) for all of them, as rows with a stride.
struct Shared {
  Tensor t;
  long long stride = 0;
};
Shared shared_rows(const Tensor& t, at::IntArrayRef lead, int64_t N, const char* name) {
  if (!t.defined()) return {};
  if (t.dim() == 1 && lead.size() > 0) return {rows(t), 0};
  TORCH_CHECK_VALUE(t.dim() == (int64_t)lead.size() + 1 && t.sizes().slice(0, lead.size()) == lead, name,
                    " must be the logits' rows ", lead, " by its length, or one row, got ", t.sizes());
  const Tensor f = flat(t, N, t.size(-1));
  return {f, f.stride(0)};
}

// A penalty of every row: a number, or float32 of the rows' shape.
Tensor row_penalty(const OptTensor& t, const Tensor& logits, at::IntArrayRef lead, const char* name) {
  if (!t.has_value()) return Tensor();
  check_float(*t, logits, lead, name);
  return t->contiguous();
}

Tensor adjust_logits(const Tensor& logits, const OptTensor& context_opt, const OptTensor& prompt_opt,
                     const OptTensor& rep_opt, const OptTensor& freq_opt, const OptTensor& pres_opt, double rep0,
                     double freq0, double pres0, const OptTensor& bias_ids_opt, const OptTensor& bias_opt,
                     const OptTensor& mask_opt) {
  const Tensor bias = bias_opt.value_or(Tensor());
  check_modes("ltc_adjust_logits", logits, bias, rep_opt.value_or(Tensor()), freq_opt.value_or(Tensor()),
              pres_opt.value_or(Tensor()));
  const Rows r = check_logits(logits);
  const auto lead = logits.sizes().slice(0, logits.dim() - 1);
  TORCH_CHECK(!torch::GradMode::is_enabled() ||
                  !torch::autograd::compute_requires_grad(logits, bias, rep_opt.value_or(Tensor()),
                                                          freq_opt.value_or(Tensor()),
                                                          pres_opt.value_or(Tensor())),
              "ltc_adjust_logits has no backward: call it under torch.no_grad()");
  TORCH_CHECK_VALUE(rep_opt.has_value() || (rep0 > 0 && std::isfinite((float)rep0) && (float)rep0 > 0),
                    "repetition must be positive and finite, got ", rep0);
  TORCH_CHECK_VALUE((freq_opt.has_value() || std::isfinite((float)freq0)) &&
                        (pres_opt.has_value() || std::isfinite((float)pres0)),
                    "frequency and presence must be finite");
  c10::DeviceGuard on(logits.device());
  Tensor out;
  at::AutoDispatchBelowADInplaceOrView guard;
  Shared context, ids, values, mask;
  int context64 = 0, ids64 = 0, ctx = 0, K = 0;
  Tensor prompt;
  if (context_opt.has_value()) {
    context64 = check_ids(*context_opt, logits, "context");
    context = shared_rows(*context_opt, lead, r.N, "context");
    ctx = as_int(context.t.size(-1), "context");
  }
  if (prompt_opt.has_value()) {
    prompt = *prompt_opt;
    TORCH_CHECK_VALUE(context_opt.has_value(), "prompt_lens without a context");
    TORCH_CHECK_TYPE(prompt.scalar_type() == at::kInt, "prompt_lens must be int32, got ", prompt.scalar_type());
    TORCH_CHECK_VALUE(prompt.sizes() == lead, "prompt_lens must be ", lead, ", got ", prompt.sizes());
    check_device(prompt, logits, "prompt_lens");
    prompt = prompt.contiguous();
  }
  TORCH_CHECK_VALUE(bias_ids_opt.has_value() == bias.defined(), "bias_ids and bias go together");
  if (bias.defined()) {
    ids64 = check_ids(*bias_ids_opt, logits, "bias_ids");
    TORCH_CHECK_TYPE(bias.scalar_type() == at::kFloat, "bias must be float32, got ", bias.scalar_type());
    check_device(bias, logits, "bias");
    ids = shared_rows(*bias_ids_opt, lead, r.N, "bias_ids");
    values = shared_rows(bias, lead, r.N, "bias");
    TORCH_CHECK_VALUE(ids.t.size(-1) == values.t.size(-1) && ids.t.size(-1) <= LTC_BIAS_MAX,
                      "bias_ids and bias must have the same length, at most ", LTC_BIAS_MAX, ", got ",
                      ids.t.size(-1), " and ", values.t.size(-1));
    K = (int)ids.t.size(-1);
  }
  if (mask_opt.has_value()) {
    TORCH_CHECK_TYPE(mask_opt->scalar_type() == at::kInt, "mask must be int32, got ", mask_opt->scalar_type());
    check_device(*mask_opt, logits, "mask");
    mask = shared_rows(*mask_opt, lead, r.N, "mask");
    TORCH_CHECK_VALUE(mask.t.size(-1) == (r.V + 31) / 32, "mask must have a bit for each of ", r.V,
                      " tokens in words of 32, got ", mask.t.sizes());
  }
  const Tensor rep = row_penalty(rep_opt, logits, lead, "repetition"),
               freq = row_penalty(freq_opt, logits, lead, "frequency"),
               pres = row_penalty(pres_opt, logits, lead, "presence");
  const Tensor x = flat(logits, r.N, r.V);
  out = at::empty(logits.sizes(), logits.options());
  check_rc(ltc_adjust_logits(ptr(x), x.stride(0), ptr(context.t), context.stride, context64, ctx,
                             static_cast<const int*>(ptr(prompt)), fp(rep), fp(freq), fp(pres), (float)rep0,
                             (float)freq0, (float)pres0, ptr(ids.t), ids.stride, ids64, fp(values.t),
                             values.stride, K, static_cast<const int*>(ptr(mask.t)), mask.stride,
                             type_of(logits, "logits"), r.N, r.V, ptr(out), stream_of(logits)),
           "ltc_adjust_logits");
  return out;
}

}  // namespace

void bind_model_operators(pybind11::module_& m) {
  m.def("causal_conv", &causal_conv, "Short causal convolution (autograd-aware)");
  m.def("causal_conv_step", &causal_conv_step, "One token of each stream, states in place");
  m.def("selective_scan", &selective_scan, "Selective state space scan (autograd-aware)");
  m.def("selective_scan_step", &selective_scan_step, "One token of each stream, states in place");
  m.def("embed", &embed, "Embedding with scaling (autograd-aware)");
  m.def("adjust_logits", &adjust_logits, "Penalties, biases and masks on logits");
}
