// C-ABI entry points of the sequence and token operators (include/ltc_capi.h):
// argument checks, workspace layout and launches. Allocates no device memory.
#include <hip/hip_runtime.h>

#include <climits>
#include <string>

#include "../../include/ltc_capi.h"
#include "ltc_seq_internal.h"

using ltc::host_clear_error;
using ltc::host_fail;
using ltc::host_hip_fail;
using ltc::host_timed;

namespace {

// Workgroups of one launch: the runtime counts threads, up to 512 each, in 32 bits.
constexpr long long kMaxGroups = (1LL << 32) / 512 - 1;

// Pieces of a workspace or of the saved buffer, each on 256 bytes; base null:
// sizes only.
struct Pieces {
  char* base;
  long long off = 0;
  template <class T>
  T* take(long long n) {
    T* p = base ? reinterpret_cast<T*>(base + off) : nullptr;
    off += (n * (long long)sizeof(T) + 255) / 256 * 256;
    return p;
  }
};

int check_workspace(long long need, const void* ws, long long have) {
  if (need > 0 && (ws == nullptr || have < need))
    return host_fail(LTC_EINVAL, "workspace too small: need " + std::to_string(need) + " bytes, got " +
                                     std::to_string(ws ? have : 0));
  if (reinterpret_cast<uintptr_t>(ws) % 256 != 0)
    return host_fail(LTC_EINVAL, "workspace must be 256-byte aligned");
  return LTC_OK;
}

bool known_type(int t) { return t == LTC_F32 || t == LTC_BF16 || t == LTC_F16; }
int type_bytes(int t) { return t == LTC_F32 ? 4 : 2; }

// ---------------------------------------------------------------------------
// Gated linear recurrence
// ---------------------------------------------------------------------------
long long tokens_in_all(int B, int T, int packed) { return packed ? T : (long long)B * T; }

int check_scan(int B, int T, int H, int packed) {
  if (B < 0 || T < 0 || H < 1)
    return host_fail(LTC_EINVAL, "dimensions must satisfy B >= 0, T >= 0, H >= 1");
  // sequence numbers share a word with two flags
  if (B > INT_MAX / 4 - 1) return host_fail(LTC_EUNSUPPORTED, "too many sequences");
  const long long N = tokens_in_all(B, T, packed);
  ltc::ScanArgs t{};
  ltc::scan_tiles(LTC_F32, N, H, &t);  // the type with the most blocks of channels
  // token numbers are 32-bit, up to a tile behind the last
  if (N > INT_MAX - 2 * ltc::kScanTile || t.ntiles > kMaxGroups / (t.per * t.ranges) || (long long)B > kMaxGroups * 256 / H)
    return host_fail(LTC_EUNSUPPORTED, "problem too large");
  return LTC_OK;
}

long long tiles_of(long long N) { return (N + ltc::kScanTile - 1) / ltc::kScanTile; }

struct ScanSaved {
  float* states;
  int* marks;
};
ScanSaved carve_saved(Pieces& c, long long N, int H, int packed) {
  ScanSaved s{};
  s.states = c.take<float>(tiles_of(N) * H);
  s.marks = packed ? c.take<int>(N) : nullptr;
  return s;
}

struct ScanWs {
  unsigned long long* words;
  long long nwords;
  unsigned* tickets;
  int* marks;
};
ScanWs carve_ws(Pieces& c, long long N, int T, int H, int packed, bool bwd) {
  ScanWs w{};
  if (packed && !bwd) w.marks = c.take<int>(N);
  if (N > 0 && ltc::scan_looks(N, T, packed != 0)) {
    w.nwords = (tiles_of(N) + tiles_of(N) / ltc::kScanGroup) * H;
    w.words = c.take<unsigned long long>(w.nwords);
    w.tickets = c.take<unsigned>(ltc::kScanRanges * ltc::kTicketStride);
  }
  return w;
}

int check_scan_call(const void* x, const void* gate, const int* cu, int x_type, int gate_type, int form,
                    int B, int T, int H) {
  int rc = check_scan(B, T, H, cu != nullptr);
  if (rc != LTC_OK) return rc;
  if (!known_type(x_type)) return host_fail(LTC_EINVAL, "x_type must be LTC_F32, LTC_BF16 or LTC_F16");
  if (gate_type != x_type && gate_type != LTC_F32)
    return host_fail(LTC_EINVAL, "gate_type must be x_type or LTC_F32");
  if (form != LTC_GATE_BLEND && form != LTC_GATE_DECAY)
    return host_fail(LTC_EINVAL, "form must be LTC_GATE_BLEND or LTC_GATE_DECAY");
  if (tokens_in_all(B, T, cu != nullptr) > 0 && (!x || !gate))
    return host_fail(LTC_EINVAL, "x/gate pointer is NULL");
  return LTC_OK;
}

// ---------------------------------------------------------------------------
// Log probabilities and distillation
// ---------------------------------------------------------------------------
int check_rows(long long N, int V, int type) {
  if (N < 0 || V < 1) return host_fail(LTC_EINVAL, "sizes must satisfy N >= 0, V >= 1");
  if (!known_type(type))
    return host_fail(LTC_EINVAL, "logits_type must be LTC_F32, LTC_BF16 or LTC_F16");
  if (N > kMaxGroups) return host_fail(LTC_EUNSUPPORTED, "too many rows");
  // indexes of a row are 32-bit, and pass V by less than one workgroup's stride
  if (V > INT_MAX - (1 << 16)) return host_fail(LTC_EUNSUPPORTED, "vocabulary too large");
  return LTC_OK;
}

int check_top(int V, int top) {
  if (top < 0 || top > LTC_TOP_MAX || top > V)
    return host_fail(LTC_EINVAL, "top must be between 0 and " + std::to_string(LTC_TOP_MAX) +
                                     " and at most V");
  return LTC_OK;
}

// log2(e) / t, by which the kernels scale: they would take 0 times an infinity.
float logit_scale(float t) { return (float)(1.4426950408889634 / (double)t); }

int check_temperature(float t) {
  if (!(t > 0.f) || !(t < __builtin_inff()) || !(logit_scale(t) < __builtin_inff()))
    return host_fail(LTC_EINVAL, "temperature must be positive and finite, and so must log2(e) over it");
  return LTC_OK;
}

ltc::TokArgs tok_args(const void* x, long long sx, const void* ids, int id64, int type, long long N, int V,
                      int top, float temperature) {
  ltc::TokArgs a{};
  a.x = x;
  a.sx = sx;
  a.ids = ids;
  a.sid = 1;
  a.id64 = id64;
  a.N = N;
  a.V = V;
  a.tau = temperature;
  a.inv_tau = 1.f / temperature;
  a.c = logit_scale(temperature);
  a.top = top;
  ltc::tok_split(N, V, type_bytes(type), top, &a.nsplit, &a.seg);
  return a;
}

void carve_parts(Pieces& c, ltc::TokArgs& a) {
  if (a.nsplit <= 1) return;
  a.part = c.take<float>(a.N * a.nsplit * 3);
  if (a.top > 0) a.part_top = c.take<unsigned long long>(a.N * a.nsplit * a.top);
}

long long parts_bytes(long long N, int V, int top, int type) {
  ltc::TokArgs a{};
  a.N = N;
  a.top = top;
  ltc::tok_split(N, V, type_bytes(type), top, &a.nsplit, &a.seg);
  Pieces c{nullptr};
  carve_parts(c, a);
  return c.off;
}

int check_distill(const void* logits, const void* t, const void* ids, int type, int t_type, long long N,
                  int V, int K, float temperature) {
  int rc = check_rows(N, V, type);
  if (rc != LTC_OK) return rc;
  if (!known_type(t_type))
    return host_fail(LTC_EINVAL, "teacher_type must be LTC_F32, LTC_BF16 or LTC_F16");
  if (K < 1 || K > LTC_TEACHER_MAX)
    return host_fail(LTC_EINVAL, "K must be between 1 and " + std::to_string(LTC_TEACHER_MAX));
  if ((rc = check_temperature(temperature)) != LTC_OK) return rc;
  if (N > 0 && (!logits || !t || !ids))
    return host_fail(LTC_EINVAL, "logits/teacher_logits/teacher_ids pointer is NULL");
  return LTC_OK;
}

}  // namespace

extern "C" {

long long ltc_gated_scan_saved_floats(int B, int T, int H, int packed) {
  if (check_scan(B, T, H, packed) != LTC_OK) return -1;
  Pieces c{nullptr};
  carve_saved(c, tokens_in_all(B, T, packed), H, packed);
  return c.off / 4;
}

long long ltc_gated_scan_fwd_workspace_bytes(int B, int T, int H, int packed) {
  if (check_scan(B, T, H, packed) != LTC_OK) return -1;
  Pieces c{nullptr};
  carve_ws(c, tokens_in_all(B, T, packed), T, H, packed, false);
  return c.off;
}

long long ltc_gated_scan_bwd_workspace_bytes(int B, int T, int H, int packed) {
  if (check_scan(B, T, H, packed) != LTC_OK) return -1;
  Pieces c{nullptr};
  carve_ws(c, tokens_in_all(B, T, packed), T, H, packed, true);
  return c.off;
}

int ltc_gated_scan_forward(const void* x, long long sxb, long long sxt, const void* gate, long long sgb,
                           long long sgt, const float* state, const int* cu_seqlens, int x_type,
                           int gate_type, int form, int B, int T, int H, int save, void* out,
                           float* state_final, float* saved, void* workspace, long long workspace_bytes,
                           void* stream) {
  host_clear_error();
  int rc = check_scan_call(x, gate, cu_seqlens, x_type, gate_type, form, B, T, H);
  if (rc != LTC_OK) return rc;
  const int packed = cu_seqlens != nullptr;
  const long long N = tokens_in_all(B, T, packed);
  if (N > 0 && !out) return host_fail(LTC_EINVAL, "out pointer is NULL");
  if (B > 0 && !state_final) return host_fail(LTC_EINVAL, "state_final pointer is NULL");
  if (save && N > 0 && !saved) return host_fail(LTC_EINVAL, "save set without a saved buffer");
  Pieces need{nullptr};
  carve_ws(need, N, T, H, packed, false);
  rc = check_workspace(need.off, workspace, workspace_bytes);
  if (rc != LTC_OK) return rc;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  Pieces cw{static_cast<char*>(workspace)}, cs{reinterpret_cast<char*>(saved)};
  const ScanWs w = carve_ws(cw, N, T, H, packed, false);
  ScanSaved sv{};
  if (save) sv = carve_saved(cs, N, H, packed);
  ltc::ScanArgs a{};
  a.x = x;
  a.g = gate;
  a.sxb = sxb;
  a.sxt = sxt;
  a.sgb = sgb;
  a.sgt = sgt;
  a.h0 = state;
  a.B = B;
  a.T = T;
  a.H = H;
  a.N = N;
  a.out = out;
  a.hf = state_final;
  a.states = sv.states;
  a.words = w.words;
  a.tickets = w.tickets;
  a.spin = ltc::host_spin_ticks();
  ltc::scan_tiles(x_type, N, H, &a);
  int* marks = save ? sv.marks : w.marks;
  a.cu = cu_seqlens;
  a.marks = marks;
  const bool ends = B > 0 && (packed || N == 0);
  const ltc::ScanPrep pr{w.words, w.nwords, w.tickets, cu_seqlens, marks, B, H, N, state,
                         ends ? state_final : nullptr};
  const hipError_t e = host_timed(ltc::K_SCAN_FWD, [&] {
    hipError_t e = hipSuccess;
    if (w.nwords > 0 || ends || (packed && N > 0)) e = ltc::launch_scan_prep(pr, s);
    if (e == hipSuccess && N > 0) e = ltc::launch_scan({x_type, gate_type, form}, a, false, s);
    return e;
  });
  return e == hipSuccess ? LTC_OK : host_hip_fail("gated scan launch", e);
}

int ltc_gated_scan_backward(const void* x, long long sxb, long long sxt, const void* gate, long long sgb,
                            long long sgt, const float* state, const int* cu_seqlens, int x_type,
                            int gate_type, int form, int B, int T, int H, const float* saved,
                            const void* grad_out, long long sob, long long sot,
                            const float* grad_state_final, void* grad_x, void* grad_gate,
                            float* grad_state, void* workspace, long long workspace_bytes, void* stream) {
  host_clear_error();
  int rc = check_scan_call(x, gate, cu_seqlens, x_type, gate_type, form, B, T, H);
  if (rc != LTC_OK) return rc;
  const int packed = cu_seqlens != nullptr;
  const long long N = tokens_in_all(B, T, packed);
  if (N > 0 && !saved) return host_fail(LTC_EINVAL, "saved pointer is NULL");
  Pieces need{nullptr};
  carve_ws(need, N, T, H, packed, true);
  rc = check_workspace(need.off, workspace, workspace_bytes);
  if (rc != LTC_OK) return rc;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  Pieces cw{static_cast<char*>(workspace)};
  Pieces cs{reinterpret_cast<char*>(const_cast<float*>(saved))};
  const ScanWs w = carve_ws(cw, N, T, H, packed, true);
  const ScanSaved sv = carve_saved(cs, N, H, packed);
  ltc::ScanArgs a{};
  a.x = x;
  a.g = gate;
  a.go = grad_out;
  a.sxb = sxb;
  a.sxt = sxt;
  a.sgb = sgb;
  a.sgt = sgt;
  a.sob = sob;
  a.sot = sot;
  a.h0 = state;
  a.gh = grad_state_final;
  a.cu = cu_seqlens;
  a.marks = sv.marks;
  a.B = B;
  a.T = T;
  a.H = H;
  a.N = N;
  a.states = sv.states;
  a.words = w.words;
  a.tickets = w.tickets;
  a.spin = ltc::host_spin_ticks();
  ltc::scan_tiles(x_type, N, H, &a);
  a.gx = grad_x;
  a.gg = grad_gate;
  a.gs = grad_state;
  const bool ends = B > 0 && grad_state && (packed || N == 0);
  const ltc::ScanPrep pr{w.words, w.nwords, w.tickets, cu_seqlens, nullptr, B, H, N, grad_state_final,
                         ends ? grad_state : nullptr};
  const hipError_t e = host_timed(ltc::K_SCAN_BWD, [&] {
    hipError_t e = hipSuccess;
    if (w.nwords > 0 || ends) e = ltc::launch_scan_prep(pr, s);
    if (e == hipSuccess && N > 0) e = ltc::launch_scan({x_type, gate_type, form}, a, true, s);
    return e;
  });
  return e == hipSuccess ? LTC_OK : host_hip_fail("gated scan backward launch", e);
}

int ltc_scan_status(int clear) {
  host_clear_error();
  int v = 0;
  const hipError_t e = ltc::scan_fault(&v, clear != 0);
  if (e != hipSuccess) return host_hip_fail("scan status read", e);
  if (v != 0)
    return host_fail(LTC_EHIP,
                     "a gated scan on this device gave up waiting for a state that another of its "
                     "workgroups hands on (the budget ran out, or two calls at once shared a "
                     "workspace); what comes from that state is NaN");
  return LTC_OK;
}

int ltc_gated_scan_step(const void* x, long long sxb, const void* gate, long long sgb, float* state,
                        long long ssp, const int* slots, int x_type, int gate_type, int form, int B, int H,
                        int P, void* out, void* stream) {
  host_clear_error();
  int rc = check_scan_call(x, gate, nullptr, x_type, gate_type, form, B, 1, H);
  if (rc != LTC_OK) return rc;
  // slots of no rows have no address
  if (P < 0 || (!slots && B > 0 && P != B))
    return host_fail(LTC_EINVAL, "P must be the states' number, B without slots");
  // rows are the grid's second dimension
  if (B > 65535) return host_fail(LTC_EUNSUPPORTED, "more than 65535 rows in a step");
  if (ssp < H && P > 1) return host_fail(LTC_EINVAL, "states overlap: row stride below H");
  if (B > 0 && ((!state && P > 0) || !out)) return host_fail(LTC_EINVAL, "state/out pointer is NULL");
  if (B == 0) return LTC_OK;
  const ltc::StepArgs a{x, gate, sxb, sgb, ssp, state, slots, B, H, P, out};
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const hipError_t e = host_timed(
      ltc::K_SCAN_STEP, [&] { return ltc::launch_scan_step(x_type, gate_type, form, a, s); });
  return e == hipSuccess ? LTC_OK : host_hip_fail("gated scan step launch", e);
}

long long ltc_token_logprobs_workspace_bytes(long long N, int V, int top, int logits_type) {
  if (check_rows(N, V, logits_type) != LTC_OK || check_top(V, top) != LTC_OK) return -1;
  return parts_bytes(N, V, top, logits_type);
}

int ltc_token_logprobs_forward(const void* logits, long long sl, const void* ids, int ids64,
                               int logits_type, long long N, int V, int top, float temperature,
                               float* logp, float* entropy, float* top_logp, long long* top_ids,
                               float* stats, void* workspace, long long workspace_bytes, void* stream) {
  host_clear_error();
  int rc = check_rows(N, V, logits_type);
  if (rc == LTC_OK) rc = check_top(V, top);
  if (rc == LTC_OK) rc = check_temperature(temperature);
  if (rc != LTC_OK) return rc;
  if (N > 0 && (!logits || !ids || !logp)) return host_fail(LTC_EINVAL, "logits/ids/logp pointer is NULL");
  if (N > 0 && top > 0 && (!top_logp || !top_ids))
    return host_fail(LTC_EINVAL, "top set without top_logp/top_ids");
  rc = check_workspace(parts_bytes(N, V, top, logits_type), workspace, workspace_bytes);
  if (rc != LTC_OK) return rc;
  if (N == 0) return LTC_OK;
  ltc::TokArgs a = tok_args(logits, sl, ids, ids64 != 0, logits_type, N, V, top, temperature);
  a.logp = logp;
  a.ent = entropy;
  a.top_logp = top_logp;
  a.top_ids = top_ids;
  a.stats = stats;
  Pieces c{static_cast<char*>(workspace)};
  carve_parts(c, a);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const hipError_t e =
      host_timed(ltc::K_LOGPROBS_FWD, [&] { return ltc::launch_logprobs_fwd(logits_type, a, s); });
  return e == hipSuccess ? LTC_OK : host_hip_fail("log probabilities launch", e);
}

int ltc_token_logprobs_backward(const void* logits, long long sl, const void* ids, int ids64,
                                int logits_type, long long N, int V, float temperature, const float* stats,
                                const float* grad_logp, long long slp, const float* grad_entropy,
                                long long sen, void* grad_logits, void* stream) {
  host_clear_error();
  int rc = check_rows(N, V, logits_type);
  if (rc == LTC_OK) rc = check_temperature(temperature);
  if (rc != LTC_OK) return rc;
  if (N == 0) return LTC_OK;
  if (!logits || !ids || !stats || !grad_logits)
    return host_fail(LTC_EINVAL, "logits/ids/stats/grad_logits pointer is NULL");
  ltc::TokArgs a = tok_args(logits, sl, ids, ids64 != 0, logits_type, N, V, 0, temperature);
  a.stats = const_cast<float*>(stats);
  a.gp = grad_logp;
  a.sgp = slp;
  a.ge = grad_entropy;
  a.sge = sen;
  a.gx = grad_logits;
  ltc::tok_split_bwd(N, V, type_bytes(logits_type), kMaxGroups, &a.nsplit, &a.seg);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const hipError_t e =
      host_timed(ltc::K_LOGPROBS_BWD, [&] { return ltc::launch_logprobs_bwd(logits_type, a, s); });
  return e == hipSuccess ? LTC_OK : host_hip_fail("log probabilities backward launch", e);
}

long long ltc_top_distill_workspace_bytes(long long N, int V, int logits_type) {
  if (check_rows(N, V, logits_type) != LTC_OK) return -1;
  return parts_bytes(N, V, 0, logits_type);
}

int ltc_top_distill_forward(const void* logits, long long sl, const void* teacher_logits, long long st,
                            const void* teacher_ids, long long si, int ids64, int logits_type,
                            int teacher_type, long long N, int V, int K, float temperature, float* loss,
                            float* stats, void* workspace, long long workspace_bytes, void* stream) {
  host_clear_error();
  int rc = check_distill(logits, teacher_logits, teacher_ids, logits_type, teacher_type, N, V, K,
                         temperature);
  if (rc != LTC_OK) return rc;
  if (N > 0 && !loss) return host_fail(LTC_EINVAL, "loss pointer is NULL");
  rc = check_workspace(parts_bytes(N, V, 0, logits_type), workspace, workspace_bytes);
  if (rc != LTC_OK) return rc;
  if (N == 0) return LTC_OK;
  ltc::TokArgs a = tok_args(logits, sl, teacher_ids, ids64 != 0, logits_type, N, V, 0, temperature);
  a.sid = si;
  a.t = teacher_logits;
  a.st = st;
  a.t_type = teacher_type;
  a.K = K;
  a.logp = loss;
  a.stats = stats;
  Pieces c{static_cast<char*>(workspace)};
  carve_parts(c, a);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const hipError_t e =
      host_timed(ltc::K_DISTILL_FWD, [&] { return ltc::launch_distill_fwd(logits_type, a, s); });
  return e == hipSuccess ? LTC_OK : host_hip_fail("distillation launch", e);
}

int ltc_top_distill_backward(const void* logits, long long sl, const void* teacher_logits, long long st,
                             const void* teacher_ids, long long si, int ids64, int logits_type,
                             int teacher_type, long long N, int V, int K, float temperature,
                             const float* stats, const float* grad_loss, long long sgl, void* grad_logits,
                             void* stream) {
  host_clear_error();
  int rc = check_distill(logits, teacher_logits, teacher_ids, logits_type, teacher_type, N, V, K,
                         temperature);
  if (rc != LTC_OK) return rc;
  if (N == 0) return LTC_OK;
  if (!stats || !grad_loss || !grad_logits)
    return host_fail(LTC_EINVAL, "stats/grad_loss/grad_logits pointer is NULL");
  ltc::TokArgs a = tok_args(logits, sl, teacher_ids, ids64 != 0, logits_type, N, V, 0, temperature);
  a.sid = si;
  a.t = teacher_logits;
  a.st = st;
  a.t_type = teacher_type;
  a.K = K;
  a.stats = const_cast<float*>(stats);
  a.gp = grad_loss;
  a.sgp = sgl;
  a.gx = grad_logits;
  ltc::tok_split_bwd(N, V, type_bytes(logits_type), kMaxGroups, &a.nsplit, &a.seg);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const hipError_t e =
      host_timed(ltc::K_DISTILL_BWD, [&] { return ltc::launch_distill_bwd(logits_type, a, s); });
  return e == hipSuccess ? LTC_OK : host_hip_fail("distillation backward launch", e);
}

}  // extern "C"
