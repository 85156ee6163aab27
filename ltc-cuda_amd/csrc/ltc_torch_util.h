// What the torch glue's operators share: argument checks, workspaces, and the rules of
// their autograd nodes.
#pragma once

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

namespace ltc_torch {

using torch::Tensor;
using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;
using OptTensor = c10::optional<Tensor>;

inline void check_rc(int rc, const char* what) {
  TORCH_CHECK(rc == LTC_OK, what, " failed (code ", rc, "): ", ltc_last_error());
}

inline void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
inline float* fp(const Tensor& t) { return t.defined() ? t.data_ptr<float>() : nullptr; }

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

inline hipStream_t stream_of(const Tensor& t) {
  return c10::hip::getCurrentHIPStream(t.device().index()).stream();
}

inline int type_of(const Tensor& t, const char* name) {
  switch (t.scalar_type()) {
    case at::kFloat: return LTC_F32;
    case at::kBFloat16: return LTC_BF16;
    case at::kHalf: return LTC_F16;
    default: TORCH_CHECK_TYPE(false, name, " must be float32, bfloat16 or float16, got ", t.scalar_type());
  }
}

inline void check_device(const Tensor& t, const Tensor& like, const char* name) {
  TORCH_CHECK_VALUE(like.is_cuda(), "the tensors must be on a CUDA (HIP) device");
  TORCH_CHECK_VALUE(t.device() == like.device(), name, " is on ", t.device(), ", expected ", like.device());
}

inline int as_int(int64_t v, const char* name) {
  TORCH_CHECK_VALUE(v <= std::numeric_limits<int>::max(), name, " = ", v, " is too large");
  return (int)v;
}

// t, with unit stride along its last dimension.
inline Tensor rows(const Tensor& t) {
  return t.dim() > 0 && (t.stride(-1) == 1 || t.size(-1) <= 1) ? t : t.contiguous();
}

// Gradients that are themselves differentiated (create_graph=True) would be
// wrong without an error otherwise.
inline variable_list first_order(variable_list&& g, const char* name) {
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
inline void check_capture(const Node& node, const Tensor& like) {
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

// Whether the rows of two matrices of unit stride share a byte. The rows of `table` lie
// apart from one another, those of t anyhow: of the table's rows that begin before the
// end of a row of t, the last one reaches furthest.
inline bool rows_meet(const Tensor& t, const Tensor& table) {
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

// logits (..., V) as N rows.
struct Rows {
  int64_t N;
  int V;
};

inline Rows check_logits(const Tensor& logits) {
  TORCH_CHECK_VALUE(logits.dim() >= 1 && logits.size(-1) >= 1, "logits must be (..., V), got ",
                    logits.sizes());
  type_of(logits, "logits");
  check_device(logits, logits, "logits");
  const int V = as_int(logits.size(-1), "V");
  return {logits.numel() / V, V};
}

inline Tensor flat(const Tensor& t, int64_t N, int64_t n) { return rows(t.reshape({N, n})); }

inline int check_ids(const Tensor& ids, const Tensor& like, const char* name) {
  TORCH_CHECK_TYPE(ids.scalar_type() == at::kInt || ids.scalar_type() == at::kLong, name,
                   " must be int32 or int64, got ", ids.scalar_type());
  check_device(ids, like, name);
  return ids.scalar_type() == at::kLong;
}

}  // namespace ltc_torch
