// Internal interface of the sequence and token operators: entry points in
// ltc_seq_capi.hip, kernels in ltc_scan_device.hip (gated linear recurrence) and
// ltc_token_device.hip (log probabilities and distillation).
#pragma once

#include <hip/hip_runtime.h>

#include <string>

#include "ltc_internal.h"

namespace ltc {

// ---------------------------------------------------------------------------
// Gated linear recurrence
// ---------------------------------------------------------------------------

// Workgroups of the scan kernels: 256 threads = kScanSlots time slots of
// kScanLanes lanes; a lane holds 16 bytes of x (V channels) of each of its
// slot's tokens, so a slot reads rows of 128 bytes.
constexpr int kScanThreads = 256;
constexpr int kScanLanes = 8;
constexpr int kScanSlots = kScanThreads / kScanLanes;
// Consecutive tokens of a slot, forward and backward (which holds dL/dout and
// the recomputed states too).
constexpr int kScanTokensFwd = 8;
constexpr int kScanTokensBwd = 4;
constexpr int kScanTileFwd = kScanSlots * kScanTokensFwd;
constexpr int kScanTileBwd = kScanSlots * kScanTokensBwd;

struct ScanArgs {
  const void* x;
  const void* g;
  const void* go;  // backward: dL/dout, or null for zero
  long long sxb, sxt, sgb, sgt, sob, sot;  // element strides of x, gate, dL/dout
  const float* h0;   // (B,H) or null for zero
  const float* gh;   // backward: dL/d state_final (B,H) or null for zero
  const int* marks;  // packed: one word per token, see scan_marks_kernel; else null
  int B, T, H;       // sequences, tokens of each (packed: of all), channels
  long long N;       // tokens in all
  void* out;         // forward (N,H)
  float* hf;         // forward (B,H)
  float* states;     // state before every kScanTileBwd-th token, [.][H]; forward: may be null
  float* agg_a;      // workspace: per tile and channel the product of its decays,
  float* agg_b;      // what it adds,
  float* carry;      // and what enters it
  void* gx;          // backward (N,H), or null where not wanted
  void* gg;          // backward (N,H), or null
  float* gs;         // backward (B,H), or null
};

struct ScanPlan {
  int x_type, g_type, form;
  bool packed;
  int tile;          // tokens per workgroup
  long long ntiles;
  int cblocks;       // blocks of channels
};

ScanPlan scan_plan(int x_type, int g_type, int form, bool packed, long long N, int H, bool bwd);
hipError_t launch_scan_marks(const int* cu, int S, long long N, int* marks, hipStream_t s);
// Empty sequences: dst[s] = src[s] (0 for null src) where sequence s has no
// tokens; cu null: every sequence.
hipError_t launch_scan_empty(const int* cu, int S, int H, long long N, const float* src, float* dst,
                             hipStream_t s);
hipError_t launch_scan_fwd(const ScanPlan& p, const ScanArgs& a, hipStream_t s);
hipError_t launch_scan_bwd(const ScanPlan& p, const ScanArgs& a, hipStream_t s);

struct StepArgs {
  const void* x;
  const void* g;
  long long sxb, sgb, ssp;  // row strides of x, gate, state
  float* state;
  const int* slots;  // null: row b's state is row b
  int B, H, P;
  void* out;
};
hipError_t launch_scan_step(int x_type, int g_type, int form, const StepArgs& a, hipStream_t s);

// ---------------------------------------------------------------------------
// Log probabilities and distillation
// ---------------------------------------------------------------------------
constexpr int kTopMax = 32;        // alternatives returned
constexpr int kTeacherMax = 1024;  // teacher entries of a row
constexpr int kTokThreads = 256;

struct TokArgs {
  const void* x;      // logits (N,V), row stride sx
  long long sx;
  const void* ids;    // (N) tokens, or (N,K) teacher entries, row stride sid
  long long sid;
  int id64;           // ids are 64-bit
  const void* t;      // teacher logits (N,K), row stride st
  long long st;
  int t_type;
  long long N;
  int V, K, top;
  float tau, inv_tau, c;  // temperature, 1 / temperature, log2(e) / temperature
  float* logp;        // (N); the distillation's loss
  float* ent;         // (N) or null
  float* stats;       // (N,3): row maximum, log of the sum of exp((x - max)/tau), entropy; or null
  float* top_logp;    // (N,top)
  long long* top_ids; // (N,top)
  // workspace of rows split over workgroups
  int nsplit;
  int seg;            // logits per workgroup
  float* part;        // [N][nsplit][3]
  unsigned long long* part_top;  // [N][nsplit][top]
  // backward
  const float* gp;    // (N) dL/dlogp (or dL/dloss), null for zero; stride
  long long sgp;
  const float* ge;    // (N) dL/dentropy, null for zero; stride
  long long sge;
  void* gx;           // (N,V)
};

// Logits per workgroup and workgroups per row.
void tok_split(long long N, int V, int elem_bytes, int* nsplit, int* seg);
hipError_t launch_logprobs_fwd(int x_type, const TokArgs& a, hipStream_t s);
hipError_t launch_logprobs_bwd(int x_type, const TokArgs& a, hipStream_t s);
hipError_t launch_distill_fwd(int x_type, const TokArgs& a, hipStream_t s);
hipError_t launch_distill_bwd(int x_type, const TokArgs& a, hipStream_t s);

// ---------------------------------------------------------------------------
// Host services of ltc_capi.hip: the thread's error message and event timing
// ---------------------------------------------------------------------------
int host_fail(int code, const std::string& msg);
int host_hip_fail(const char* what, hipError_t e);
void host_clear_error();
// Runs launch(ctx); while timing is on, its kernels count under `id`.
hipError_t host_timed(int id, hipError_t (*launch)(void*), void* ctx);

template <class F>
hipError_t host_timed(int id, F f) {
  return host_timed(id, [](void* c) { return (*static_cast<F*>(c))(); }, &f);
}

}  // namespace ltc
