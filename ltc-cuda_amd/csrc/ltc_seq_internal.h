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

// Time slots of a workgroup.
constexpr int kScanSlots = 32;
// Consecutive tokens of a slot, and tokens of a workgroup.
constexpr int kScanTokens = 4;
constexpr int kScanTile = kScanSlots * kScanTokens;
// Tiles whose maps are composed into one.
constexpr int kScanGroup = 16;
// Reads of a word before a wait for it may be given up: some milliseconds.
constexpr int kScanPolls = 4096;
// Ranges of channel blocks, and the words between their counters.
constexpr int kScanRanges = 7;
constexpr int kTicketStride = 64;

struct ScanArgs {
  const void* x;
  const void* g;
  const void* go;  // backward: dL/dout, or null for zero
  long long sxb, sxt, sgb, sgt, sob, sot;  // element strides of x, gate, dL/dout
  const float* h0;   // (B,H) or null for zero
  const float* gh;   // backward: dL/d state_final (B,H) or null for zero
  const int* cu;     // packed: boundaries (B+1); else null
  const int* marks;  // packed: one word per token (scan_prep_kernel); else null
  int B, T, H;       // sequences, tokens of each (packed: of all), channels
  long long N;       // tokens in all
  long long ntiles;
  int cblocks;       // blocks of channels
  int per, ranges;   // blocks of a range, ranges (take_tile)
  void* out;         // forward (N,H)
  float* hf;         // forward (B,H)
  float* states;     // what enters each tile (ntiles,H); forward: may be null
  unsigned long long* words;  // maps of tiles (ntiles,H), then of groups of tiles
  unsigned* tickets;  // one for each range of channel blocks, every kTicketStride words
  long long spin;     // wait budget, wall-clock ticks
  void* gx;          // backward (N,H), or null where not wanted
  void* gg;          // backward (N,H), or null
  float* gs;         // backward (B,H), or null
};

struct ScanTypes {
  int x, g, form;
};

struct ScanPrep {
  unsigned long long* words;
  long long nwords;
  unsigned* tickets;
  const int* cu;
  int* marks;
  int S, H;
  long long N;
  const float* src;
  float* dst;
};

// The tiles of a call: fills in ntiles, cblocks, per and ranges.
void scan_tiles(int x_type, long long N, int H, ScanArgs* a);
bool scan_looks(long long N, int T, bool packed);
hipError_t launch_scan_prep(const ScanPrep& p, hipStream_t s);
hipError_t launch_scan(const ScanTypes& ty, const ScanArgs& a, bool bwd, hipStream_t s);

struct StepArgs {
  const void* x;
  const void* g;
  long long sxb, sgb, ssp;  // row strides of x, gate, state
  float* state;
  const int* slots;  // null: row b's state is row b
  int B, H, P;
  void* out;
};
// The current device's flag of scans that gave up a wait, as device_fault().
hipError_t scan_fault(int* value, bool clear);
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
  // (N,3): row maximum, log of the sum of exp((x - max)/tau), entropy. Distillation
  // (N,4): the same two, the teacher's maximum and its log of the sum. Or null.
  float* stats;
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
void tok_split(long long N, int V, int elem_bytes, int top, int* nsplit, int* seg);
// The same of the backward, which needs no join; `most` workgroups in all.
void tok_split_bwd(long long N, int V, int elem_bytes, long long most, int* nsplit, int* seg);
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
long long host_spin_ticks();  // ltc_set_cluster_spin_ticks
// Runs launch(ctx); while timing is on, its kernels count under `id`.
hipError_t host_timed(int id, hipError_t (*launch)(void*), void* ctx);

template <class F>
hipError_t host_timed(int id, F f) {
  return host_timed(id, [](void* c) { return (*static_cast<F*>(c))(); }, &f);
}

}  // namespace ltc
