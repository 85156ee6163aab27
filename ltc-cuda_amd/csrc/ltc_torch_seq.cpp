// Torch glue of the sequence and token operators: argument checks, allocations
// and autograd nodes around their C-ABI entry points (include/ltc_capi.h).
#include <torch/extension.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/graph_task.h>
#include <torch/csrc/autograd/saved_variable.h>

#include <ATen/MemoryOverlap.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/VirtualGuardImpl.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>

#include <algorithm>
#include <cstdint>
#include <limits>
#include <unordered_set>
#include <vector>

#include "../../include/ltc_capi.h"
#include "ltc_torch_checks.h"

namespace {

using ltc_torch::check_modes;
using torch::Tensor;
using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;
using OptTensor = c10::optional<Tensor>;

void check_rc(int rc, const char* what) {
  TORCH_CHECK(rc == LTC_OK, what, " failed (code ", rc, "): ", ltc_last_error());
}

void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
float* fp(const Tensor& t) { return t.defined() ? t.data_ptr<float>() : nullptr; }

// Device workspace of so many bytes, 256-byte aligned; none for 0.
struct Workspace {
  Tensor buf;
  void* p = nullptr;
  Workspace(long long bytes, const Tensor& like) {
    TORCH_CHECK(bytes >= 0, ltc_last_error());
    if (bytes == 0) return;
    buf = at::empty({bytes + 256}, like.options().dtype(at::kByte));
    p = reinterpret_cast<void*>((reinterpret_cast<uintptr_t>(buf.data_ptr()) + 255) & ~uintptr_t(255));
  }
};

hipStream_t stream_of(const Tensor& t) {
  return c10::hip::getCurrentHIPStream(t.device().index()).stream();
}

int type_of(const Tensor& t, const char* name) {
  switch (t.scalar_type()) {
    case at::kFloat: return LTC_F32;
    case at::kBFloat16: return LTC_BF16;
    case at::kHalf: return LTC_F16;
    default: TORCH_CHECK_TYPE(false, name, " must be float32, bfloat16 or float16, got ", t.scalar_type());
  }
}

void check_device(const Tensor& t, const Tensor& like, const char* name) {
  TORCH_CHECK_VALUE(like.is_cuda(), "the tensors must be on a CUDA (HIP) device");
  TORCH_CHECK_VALUE(t.device() == like.device(), name, " is on ", t.device(), ", expected ", like.device());
}

int as_int(int64_t v, const char* name) {
  TORCH_CHECK_VALUE(v <= std::numeric_limits<int>::max(), name, " = ", v, " is too large");
  return (int)v;
}

// t, with unit stride along its last dimension.
Tensor rows(const Tensor& t) {
  return t.dim() > 0 && (t.stride(-1) == 1 || t.size(-1) <= 1) ? t : t.contiguous();
}

// Gradients that are themselves differentiated (create_graph=True) would be
// wrong without an error otherwise.
variable_list first_order(variable_list&& g, const char* name) {
  if (!torch::GradMode::is_enabled()) return std::move(g);
  for (Tensor& t : g)
    if (t.defined()) t.set_requires_grad(true);
  auto err = std::make_shared<torch::autograd::DelayedError>(
      std::string(name) + " has no second derivatives", (int)g.size());
  return (*err)(std::move(g));
}

// A leaf's gradient accumulator belongs to the stream it was made on, and lives as
// long as any autograd graph of the leaf. If that is an eager graph of the default
// stream, autograd makes that stream wait for the one under capture as soon as a node
// returns the gradient to the accumulator, and the end of the capture then takes the
// process down. So that case is an error here, for all that the pass will reach from
// this node on (a module's parameters lie behind others). Other streams can join a
// capture, and do.
void check_capture(const Node& node, const Tensor& like) {
  if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
  const c10::Stream eager =
      c10::impl::VirtualGuardImpl(like.device().type()).getDefaultStream(like.device());
  // what the pass runs; empty: everything
  const auto* runs = torch::autograd::get_current_graph_task_exec_info();
  std::unordered_set<const Node*> seen;
  std::vector<const Node*> todo{&node};
  while (!todo.empty()) {
    const Node* n = todo.back();
    todo.pop_back();
    for (const auto& e : n->next_edges()) {
      if (!e.is_valid() || !seen.insert(e.function.get()).second) continue;
      if (runs != nullptr && !runs->empty()) {
        const auto it = runs->find(e.function.get());
        if (it == runs->end() || !it->second.should_execute()) continue;
      }
      const auto s = e.function->stream();
      TORCH_CHECK(!s.has_value() || s->id() != eager.id(), "a backward pass of ", node.name(),
                  " cannot be captured into a graph while an autograd graph of the same tensors made on "
                  "the default stream is alive: drop its outputs first");
      todo.push_back(e.function.get());
    }
  }
}

template <class N>
std::shared_ptr<N> make_node() {
  return std::shared_ptr<N>(new N(), torch::autograd::deleteNode);
}

// ---------------------------------------------------------------------------
// Gated linear recurrence
// ---------------------------------------------------------------------------
struct ScanShape {
  int B, T, H;
  bool packed;
};

ScanShape check_scan(const Tensor& x, const Tensor& gate, const Tensor& state, const Tensor& cu) {
  ScanShape s;
  s.packed = cu.defined();
  type_of(x, "x");
  TORCH_CHECK_TYPE(gate.scalar_type() == x.scalar_type() || gate.scalar_type() == at::kFloat,
                   "gate must have x's type or float32, got ", gate.scalar_type());
  if (s.packed) {
    TORCH_CHECK_VALUE(x.dim() == 2, "packed x must be (tokens, H), got ", x.sizes());
    TORCH_CHECK_TYPE(cu.scalar_type() == at::kInt, "cu_seqlens must be int32, got ", cu.scalar_type());
    TORCH_CHECK_VALUE(cu.dim() == 1 && cu.size(0) >= 1, "cu_seqlens must be (sequences + 1,), got ",
                      cu.sizes());
    check_device(cu, x, "cu_seqlens");
    s.B = as_int(cu.size(0) - 1, "sequences");
    s.T = as_int(x.size(0), "tokens");
  } else {
    TORCH_CHECK_VALUE(x.dim() == 3, "x must be (B, T, H), got ", x.sizes());
    s.B = as_int(x.size(0), "B");
    s.T = as_int(x.size(1), "T");
  }
  s.H = as_int(x.size(-1), "H");
  TORCH_CHECK_VALUE(s.H >= 1, "x has no channels");
  TORCH_CHECK_VALUE(gate.sizes() == x.sizes(), "gate must have x's shape ", x.sizes(), ", got ",
                    gate.sizes());
  check_device(gate, x, "gate");
  if (state.defined()) {
    TORCH_CHECK_VALUE(state.dim() == 2 && state.size(0) == s.B && state.size(1) == s.H, "state must be (",
                      s.B, ", ", s.H, "), got ", state.sizes());
    TORCH_CHECK_TYPE(state.scalar_type() == at::kFloat, "state must be float32, got ",
                     state.scalar_type());
    check_device(state, x, "state");
  }
  return s;
}

long long stride_b(const Tensor& t, bool packed) { return packed ? 0 : t.stride(0); }
long long stride_t(const Tensor& t, bool packed) { return t.stride(packed ? 0 : 1); }

struct GatedScanBackward : public Node {
  SavedVariable x_, gate_, state_, cu_, saved_;
  int form = 0;
  std::string name() const override { return "GatedScanBackward"; }
  void release_variables() override {
    for (SavedVariable* v : {&x_, &gate_, &state_, &cu_, &saved_}) v->reset_data();
  }
  variable_list apply(variable_list&& grads) override {
    variable_list g;
    {
      at::AutoDispatchBelowADInplaceOrView guard;
      g = run(grads);
    }
    return first_order(std::move(g), "ltc_gated_scan");
  }
  variable_list run(const variable_list& grads) {
    const Tensor x = x_.unpack(), gate = gate_.unpack(), state = state_.unpack(), cu = cu_.unpack(),
                 saved = saved_.unpack();
    c10::DeviceGuard on(x.device());
    check_capture(*this, x);
    const ScanShape s = check_scan(x, gate, state, cu);
    Tensor go = grads[0], gh = grads[1];
    if (go.defined()) go = rows(go.to(x.scalar_type()));
    if (gh.defined()) gh = gh.to(at::kFloat).contiguous();
    const Tensor xr = rows(x), gr = rows(gate);
    const Tensor st = state.defined() ? state.contiguous() : Tensor();
    const Tensor cc = cu.defined() ? cu.contiguous() : Tensor();
    Tensor gx, gg, gs;
    if (task_should_compute_output(0)) gx = at::empty(x.sizes(), x.options());
    if (task_should_compute_output(1)) gg = at::empty(gate.sizes(), gate.options());
    if (state.defined() && task_should_compute_output(2)) gs = at::empty(state.sizes(), state.options());
    const long long bytes = ltc_gated_scan_bwd_workspace_bytes(s.B, s.T, s.H, s.packed);
    const Workspace ws(bytes, x);
    check_rc(ltc_gated_scan_backward(
                 ptr(xr), stride_b(xr, s.packed), stride_t(xr, s.packed), ptr(gr),
                 stride_b(gr, s.packed), stride_t(gr, s.packed), fp(st),
                 static_cast<const int*>(ptr(cc)), type_of(x, "x"), type_of(gate, "gate"), form, s.B, s.T,
                 s.H, fp(saved), ptr(go), go.defined() ? stride_b(go, s.packed) : 0,
                 go.defined() ? stride_t(go, s.packed) : 0, fp(gh), ptr(gx), ptr(gg), fp(gs), ws.p, bytes,
                 stream_of(x)),
             "ltc_gated_scan_backward");
    return {gx, gg, gs};
  }
};

std::vector<Tensor> gated_scan(const Tensor& x, const Tensor& gate, const OptTensor& state_opt,
                               const OptTensor& cu_opt, int64_t form) {
  const Tensor state = state_opt.value_or(Tensor()), cu = cu_opt.value_or(Tensor());
  check_modes("ltc_gated_scan", x, gate, state);
  const ScanShape s = check_scan(x, gate, state, cu);
  check_device(x, x, "x");
  const bool needs_grad =
      torch::GradMode::is_enabled() && torch::autograd::compute_requires_grad(x, gate, state);
  c10::DeviceGuard on(x.device());
  Tensor out, hf, saved;
  {
    at::AutoDispatchBelowADInplaceOrView guard;
    const Tensor xr = rows(x), gr = rows(gate);
    const Tensor st = state.defined() ? state.contiguous() : Tensor();
    const Tensor cc = cu.defined() ? cu.contiguous() : Tensor();
    out = at::empty(x.sizes(), x.options());
    hf = at::empty({s.B, s.H}, x.options().dtype(at::kFloat));
    if (needs_grad) {
      const long long n = ltc_gated_scan_saved_floats(s.B, s.T, s.H, s.packed);
      TORCH_CHECK(n >= 0, ltc_last_error());
      saved = at::empty({n}, x.options().dtype(at::kFloat));
    }
    const long long bytes = ltc_gated_scan_fwd_workspace_bytes(s.B, s.T, s.H, s.packed);
    const Workspace ws(bytes, x);
    check_rc(ltc_gated_scan_forward(ptr(xr), stride_b(xr, s.packed), stride_t(xr, s.packed), ptr(gr),
                                    stride_b(gr, s.packed), stride_t(gr, s.packed), fp(st),
                                    static_cast<const int*>(ptr(cc)), type_of(x, "x"),
                                    type_of(gate, "gate"), (int)form, s.B, s.T, s.H, needs_grad, ptr(out),
                                    fp(hf), fp(saved), ws.p, bytes, stream_of(x)),
             "ltc_gated_scan_forward");
  }
  if (needs_grad) {
    auto node = make_node<GatedScanBackward>();
    node->set_next_edges(torch::autograd::collect_next_edges(x, gate, state));
    node->x_ = SavedVariable(x, false);
    node->gate_ = SavedVariable(gate, false);
    node->state_ = SavedVariable(state, false);
    node->cu_ = SavedVariable(cu, false);
    node->saved_ = SavedVariable(saved, false);
    node->form = (int)form;
    torch::autograd::set_history(out, node);
    torch::autograd::set_history(hf, node);
  }
  return {out, hf};
}

// Whether the rows of two matrices of unit stride share a byte. The rows of `table` lie
// apart from one another, those of t anyhow: of the table's rows that begin before the
// end of a row of t, the last one reaches furthest.
bool rows_meet(const Tensor& t, const Tensor& table) {
  if (t.numel() == 0 || table.numel() == 0) return false;
  const auto row_bytes = [](const Tensor& q) { return q.size(1) * q.element_size(); };
  const auto pitch = [](const Tensor& q) { return q.size(0) > 1 ? q.stride(0) * q.element_size() : 0; };
  const int64_t n = t.size(0), rows = table.size(0), width = row_bytes(table), step = pitch(table);
  // t's rows as distances from the table's beginning
  const int64_t begin = (int64_t)(reinterpret_cast<uintptr_t>(t.data_ptr()) -
                                  reinterpret_cast<uintptr_t>(table.data_ptr()));
  const auto meets = [&](int64_t lo) {
    const int64_t hi = lo + row_bytes(t);
    if (hi <= 0 || lo >= (rows - 1) * step + width) return false;
    const int64_t r = step > 0 ? std::min((hi - 1) / step, rows - 1) : 0;
    return r * step + width > lo;
  };
  if (begin + (n - 1) * pitch(t) + row_bytes(t) <= 0 || begin >= (rows - 1) * step + width) return false;
  for (int64_t i = 0; i < n; ++i)
    if (meets(begin + i * pitch(t))) return true;
  return false;
}

Tensor gated_scan_step(const Tensor& x, const Tensor& gate, const Tensor& state, const OptTensor& slots_opt,
                       int64_t form) {
  check_modes("ltc_gated_scan_step", x, gate, state);
  TORCH_CHECK_VALUE(x.dim() == 2, "x must be (B, H), got ", x.sizes());
  type_of(x, "x");
  TORCH_CHECK_TYPE(gate.scalar_type() == x.scalar_type() || gate.scalar_type() == at::kFloat,
                   "gate must have x's type or float32, got ", gate.scalar_type());
  TORCH_CHECK_VALUE(gate.sizes() == x.sizes(), "gate must have x's shape ", x.sizes(), ", got ",
                    gate.sizes());
  TORCH_CHECK_TYPE(state.scalar_type() == at::kFloat, "state must be float32, got ", state.scalar_type());
  const int B = as_int(x.size(0), "B"), H = as_int(x.size(1), "H");
  TORCH_CHECK_VALUE(H >= 1, "x has no channels");
  TORCH_CHECK_VALUE(state.dim() == 2 && state.size(1) == H, "state must be (rows, ", H, "), got ",
                    state.sizes());
  // written in place: a copy would not do
  TORCH_CHECK_VALUE(state.stride(1) == 1 || H == 1, "state must have unit stride along its channels");
  TORCH_CHECK_VALUE(state.size(0) <= 1 || state.stride(0) >= H, "the rows of state overlap");
  Tensor slots;
  if (slots_opt.has_value()) {
    slots = *slots_opt;
    TORCH_CHECK_TYPE(slots.scalar_type() == at::kInt, "slots must be int32, got ", slots.scalar_type());
    TORCH_CHECK_VALUE(slots.dim() == 1 && slots.size(0) == B, "slots must be (", B, ",), got ",
                      slots.sizes());
    check_device(slots, x, "slots");
  } else {
    TORCH_CHECK_VALUE(state.size(0) == B, "state must be (", B, ", ", H, ") without slots, got ",
                      state.sizes());
  }
  check_device(gate, x, "gate");
  check_device(state, x, "state");
  // workgroups read x and gate while others write the state
  at::assert_no_overlap(state, x);
  at::assert_no_overlap(state, gate);
  TORCH_CHECK(!torch::GradMode::is_enabled() ||
                  !torch::autograd::compute_requires_grad(x, gate, state),
              "ltc_gated_scan_step has no backward: call it under torch.no_grad(), or ltc_gated_scan");
  c10::DeviceGuard on(x.device());
  Tensor out;
  {
    at::AutoDispatchBelowADInplaceOrView guard;
    const Tensor xr = rows(x), gr = rows(gate);
    // what the checks above cannot tell: rows with gaps between them
    TORCH_CHECK(!rows_meet(xr, state) && !rows_meet(gr, state),
                "x and gate must not share memory with state, which is written in place");
    const Tensor sl = slots.defined() ? slots.contiguous() : Tensor();
    out = at::empty(x.sizes(), x.options());
    check_rc(ltc_gated_scan_step(ptr(xr), xr.stride(0), ptr(gr), gr.stride(0), fp(state),
                                 state.stride(0), static_cast<const int*>(ptr(sl)), type_of(x, "x"),
                                 type_of(gate, "gate"), (int)form, B, H, as_int(state.size(0), "rows"),
                                 ptr(out), stream_of(x)),
             "ltc_gated_scan_step");
  }
  // saved copies of the state are stale now
  if (!state.is_inference()) torch::autograd::impl::bump_version(state);
  return out;
}

// ---------------------------------------------------------------------------
// Log probabilities and distillation
// ---------------------------------------------------------------------------
// logits (..., V) as N rows.
struct Rows {
  int64_t N;
  int V;
};

Rows check_logits(const Tensor& logits) {
  TORCH_CHECK_VALUE(logits.dim() >= 1 && logits.size(-1) >= 1, "logits must be (..., V), got ",
                    logits.sizes());
  type_of(logits, "logits");
  check_device(logits, logits, "logits");
  const int V = as_int(logits.size(-1), "V");
  return {logits.numel() / V, V};
}

Tensor flat(const Tensor& t, int64_t N, int64_t n) { return rows(t.reshape({N, n})); }

int check_ids(const Tensor& ids, const Tensor& like, const char* name) {
  TORCH_CHECK_TYPE(ids.scalar_type() == at::kInt || ids.scalar_type() == at::kLong, name,
                   " must be int32 or int64, got ", ids.scalar_type());
  check_device(ids, like, name);
  return ids.scalar_type() == at::kLong;
}

// A row gradient as N floats with a stride.
Tensor row_grad(const Tensor& g, int64_t N) {
  return g.defined() ? g.to(at::kFloat).reshape({N}) : Tensor();
}

struct TokenLogprobsBackward : public Node {
  SavedVariable logits_, ids_, stats_;
  double temperature = 1;
  std::string name() const override { return "TokenLogprobsBackward"; }
  void release_variables() override {
    for (SavedVariable* v : {&logits_, &ids_, &stats_}) v->reset_data();
  }
  variable_list apply(variable_list&& grads) override {
    Tensor g;
    {
      at::AutoDispatchBelowADInplaceOrView guard;
      const Tensor logits = logits_.unpack(), ids = ids_.unpack(), stats = stats_.unpack();
      c10::DeviceGuard on(logits.device());
      check_capture(*this, logits);
      const Rows r = check_logits(logits);
      const Tensor x = flat(logits, r.N, r.V), id = ids.contiguous();
      const Tensor gp = row_grad(grads[0], r.N), ge = row_grad(grads[1], r.N);
      g = at::empty(logits.sizes(), logits.options());
      check_rc(ltc_token_logprobs_backward(
                   ptr(x), x.stride(0), ptr(id), ids.scalar_type() == at::kLong,
                   type_of(logits, "logits"), r.N, r.V, (float)temperature, fp(stats), fp(gp),
                   gp.defined() ? gp.stride(0) : 0, fp(ge), ge.defined() ? ge.stride(0) : 0, ptr(g),
                   stream_of(logits)),
               "ltc_token_logprobs_backward");
    }
    return first_order({g}, "ltc_token_logprobs");
  }
};

std::vector<Tensor> token_logprobs(const Tensor& logits, const Tensor& ids, int64_t top,
                                   double temperature) {
  check_modes("ltc_token_logprobs", logits);
  const Rows r = check_logits(logits);
  const int id64 = check_ids(ids, logits, "ids");
  const auto shape = logits.sizes().slice(0, logits.dim() - 1);
  TORCH_CHECK_VALUE(ids.sizes() == shape, "ids must be ", shape, ", got ", ids.sizes());
  TORCH_CHECK_VALUE(top >= 0 && top <= LTC_TOP_MAX && top <= r.V, "top must be between 0 and ",
                    LTC_TOP_MAX, " and at most V, got ", top);
  TORCH_CHECK_VALUE(temperature > 0, "temperature must be positive, got ", temperature);
  const bool needs_grad = torch::GradMode::is_enabled() && logits.requires_grad();
  c10::DeviceGuard on(logits.device());
  std::vector<Tensor> res;
  Tensor stats;
  {
    at::AutoDispatchBelowADInplaceOrView guard;
    const Tensor x = flat(logits, r.N, r.V), id = ids.contiguous();
    const auto f32 = logits.options().dtype(at::kFloat);
    res = {at::empty(shape, f32), at::empty(shape, f32)};
    if (top > 0) {
      auto ts = shape.vec();
      ts.push_back(top);
      res.push_back(at::empty(ts, f32));
      res.push_back(at::empty(ts, logits.options().dtype(at::kLong)));
    }
    if (needs_grad) stats = at::empty({r.N, 3}, f32);
    const long long bytes =
        ltc_token_logprobs_workspace_bytes(r.N, r.V, (int)top, type_of(logits, "logits"));
    const Workspace ws(bytes, logits);
    check_rc(ltc_token_logprobs_forward(
                 ptr(x), x.stride(0), ptr(id), id64, type_of(logits, "logits"), r.N, r.V, (int)top,
                 (float)temperature, fp(res[0]), fp(res[1]), top > 0 ? fp(res[2]) : nullptr,
                 top > 0 ? reinterpret_cast<long long*>(res[3].data_ptr<int64_t>()) : nullptr, fp(stats),
                 ws.p, bytes, stream_of(logits)),
             "ltc_token_logprobs_forward");
  }
  if (needs_grad) {
    auto node = make_node<TokenLogprobsBackward>();
    node->set_next_edges(torch::autograd::collect_next_edges(logits));
    node->logits_ = SavedVariable(logits, false);
    node->ids_ = SavedVariable(ids, false);
    node->stats_ = SavedVariable(stats, false);
    node->temperature = temperature;
    torch::autograd::set_history(res[0], node);
    torch::autograd::set_history(res[1], node);
  }
  return res;
}

struct TopDistillBackward : public Node {
  SavedVariable logits_, t_, ids_, stats_;
  double temperature = 1;
  std::string name() const override { return "TopDistillBackward"; }
  void release_variables() override {
    for (SavedVariable* v : {&logits_, &t_, &ids_, &stats_}) v->reset_data();
  }
  variable_list apply(variable_list&& grads) override {
    if (!grads[0].defined()) return {Tensor()};
    Tensor g;
    {
      at::AutoDispatchBelowADInplaceOrView guard;
      const Tensor logits = logits_.unpack(), teacher = t_.unpack(), ids = ids_.unpack(),
                   stats = stats_.unpack();
      c10::DeviceGuard on(logits.device());
      check_capture(*this, logits);
      const Rows r = check_logits(logits);
      const int64_t K = teacher.size(-1);
      const Tensor x = flat(logits, r.N, r.V), t = flat(teacher, r.N, K), id = flat(ids, r.N, K);
      const Tensor gl = row_grad(grads[0], r.N);
      g = at::empty(logits.sizes(), logits.options());
      check_rc(ltc_top_distill_backward(ptr(x), x.stride(0), ptr(t), t.stride(0), ptr(id), id.stride(0),
                                        ids.scalar_type() == at::kLong, type_of(logits, "logits"),
                                        type_of(teacher, "teacher_logits"), r.N, r.V, (int)K,
                                        (float)temperature, fp(stats), fp(gl), gl.stride(0), ptr(g),
                                        stream_of(logits)),
               "ltc_top_distill_backward");
    }
    return first_order({g}, "ltc_top_distill");
  }
};

Tensor top_distill(const Tensor& logits, const Tensor& teacher, const Tensor& ids, double temperature) {
  check_modes("ltc_top_distill", logits, teacher);
  const Rows r = check_logits(logits);
  const int id64 = check_ids(ids, logits, "teacher_ids");
  type_of(teacher, "teacher_logits");
  check_device(teacher, logits, "teacher_logits");
  const auto shape = logits.sizes().slice(0, logits.dim() - 1);
  TORCH_CHECK_VALUE(ids.dim() == logits.dim() && ids.sizes().slice(0, ids.dim() - 1) == shape,
                    "teacher_ids must be logits' rows ", shape, " by K, got ", ids.sizes());
  TORCH_CHECK_VALUE(teacher.sizes() == ids.sizes(), "teacher_logits must have teacher_ids' shape ",
                    ids.sizes(), ", got ", teacher.sizes());
  const int64_t K = ids.size(-1);
  TORCH_CHECK_VALUE(K >= 1 && K <= LTC_TEACHER_MAX, "K must be between 1 and ", LTC_TEACHER_MAX, ", got ",
                    K);
  TORCH_CHECK_VALUE(temperature > 0, "temperature must be positive, got ", temperature);
  TORCH_CHECK_VALUE(!torch::GradMode::is_enabled() || !teacher.requires_grad(),
                    "the teacher gets no gradient: detach teacher_logits");
  const bool needs_grad = torch::GradMode::is_enabled() && logits.requires_grad();
  c10::DeviceGuard on(logits.device());
  Tensor loss, stats;
  {
    at::AutoDispatchBelowADInplaceOrView guard;
    const Tensor x = flat(logits, r.N, r.V), t = flat(teacher, r.N, K), id = flat(ids, r.N, K);
    const auto f32 = logits.options().dtype(at::kFloat);
    loss = at::empty(shape, f32);
    if (needs_grad) stats = at::empty({r.N, 4}, f32);
    const long long bytes = ltc_top_distill_workspace_bytes(r.N, r.V, type_of(logits, "logits"));
    const Workspace ws(bytes, logits);
    check_rc(ltc_top_distill_forward(ptr(x), x.stride(0), ptr(t), t.stride(0), ptr(id), id.stride(0), id64,
                                     type_of(logits, "logits"), type_of(teacher, "teacher_logits"), r.N,
                                     r.V, (int)K, (float)temperature, fp(loss), fp(stats), ws.p, bytes,
                                     stream_of(logits)),
             "ltc_top_distill_forward");
  }
  if (needs_grad) {
    auto node = make_node<TopDistillBackward>();
    node->set_next_edges(torch::autograd::collect_next_edges(logits));
    node->logits_ = SavedVariable(logits, false);
    node->t_ = SavedVariable(teacher, false);
    node->ids_ = SavedVariable(ids, false);
    node->stats_ = SavedVariable(stats, false);
    node->temperature = temperature;
    torch::autograd::set_history(loss, node);
  }
  return loss;
}

}  // namespace

void bind_sequence_operators(pybind11::module_& m) {
  m.def("gated_scan", &gated_scan, "Gated linear recurrence (autograd-aware)");
  m.def("gated_scan_step", &gated_scan_step, "One token of each stream, states in place");
  m.def("token_logprobs", &token_logprobs, "Log probabilities, entropy, alternatives (autograd-aware)");
  m.def("top_distill", &top_distill, "Distillation from a teacher's top logits (autograd-aware)");
}
