/*
 * C-ABI of the MI355X (gfx950) LTC fused ODE-solver library, libltc_hip.so.
 *
 * This is the drop-in boundary that replaces the reference's pybind11
 * extension `ltc_cuda_kernels_v2` (built at ltc_cuda.py:211-217 and called
 * only from LTCCudaForward, ltc_cuda.py:270 and :331). Plain pointers and
 * sizes, no torch types: any host (ctypes, cgo, JNI, N-API) can bind it.
 *
 * Conventions
 *  - All tensors are fp32 device pointers on the current HIP device.
 *  - Parameters are contiguous in the reference's own layouts:
 *      recurrent (H,H) row-major [i][j], i presynaptic (ltc.py:22-26),
 *      sensory   (D,H) row-major [d][h] (ltc.py:27-30),
 *      per neuron (H).
 *  - x (B,T,D) and grad_out (B,T,H) take explicit element strides, so
 *    strided views (e.g. x[:,:,0::2]) and expanded gradients (stride 0) are
 *    read in place.
 *  - Every other output is written contiguous.
 *  - The library allocates nothing. The caller passes a device workspace of
 *    at least ltc_*_workspace_bytes() bytes, 256-byte aligned.
 *  - Work is enqueued on `stream` (a hipStream_t; NULL = the null stream).
 *    Calls return as soon as the work is queued.
 *  - Return value: 0 on success; LTC_EINVAL for bad arguments (nothing is
 *    launched), LTC_EUNSUPPORTED for shapes outside the supported range,
 *    LTC_EHIP when a HIP call or launch fails. ltc_last_error() then holds a
 *    message (thread-local).
 *  - Results are deterministic: every reduction of floating-point numbers has a fixed
 *    order (atomics count whole numbers only).
 */
#ifndef LTC_CAPI_H
#define LTC_CAPI_H

#ifdef __cplusplus
extern "C" {
#endif

#define LTC_ABI_VERSION 1

#define LTC_OK 0
#define LTC_EINVAL 1
#define LTC_EUNSUPPORTED 2
#define LTC_EHIP 3

/* Largest hidden size. Up to H = 1024 a single workgroup can hold a batch
 * row's neurons; above it the ODE kernels always run as clusters of Hp/64
 * workgroups (at most one per CU, in as many launches as the batch needs),
 * which needs Hp/64 <= the device's CU count. The reference has no limit;
 * 4096 keeps every operand image under 1 GiB and every byte offset inside
 * the 32-bit buffer range. */
#define LTC_MAX_HIDDEN 4096

/* ABI version of the loaded library (LTC_ABI_VERSION at build time). */
int ltc_abi_version(void);

/* Message of the last failed call on this thread ("" if none). */
const char* ltc_last_error(void);

/* Number of visible HIP devices; 0 on a host without a GPU or driver. The
 * Python loader uses it to decide whether the extension can serve calls
 * (the reference probes torch.cuda.is_available(), ltc_cuda.py:142). */
int ltc_device_count(void);

/* Floats in the `saved` buffer that ltc_full_forward fills for backward:
 * the pre-state of every unfold plus the final state, and the reciprocal of
 * every unfold's denominator. It replaces the reference's v_buffers_stacked (T,U,B,H) and
 * w_num/w_den_sens_stacked (T,B,H) (csrc/ltc_kernels.cu:1207-1211). */
long long ltc_saved_floats(int B, int T, int H, int ode_unfolds);

/* Workspace sizes in bytes for one forward / backward call. */
long long ltc_fwd_workspace_bytes(int B, int T, int D, int H, int ode_unfolds);
long long ltc_bwd_workspace_bytes(int B, int T, int D, int H, int ode_unfolds);

/*
 * Whole forward time loop. Replaces ltc_full_forward
 * (csrc/ltc_kernels.cu:1165-1182, bound at ltc_cuda.py:270-276).
 *   x            (B,T,D) with element strides sxb, sxt, sxd
 *   state        (B,H) initial state, contiguous; never written
 *   w_pos .. vleak  the 11 boundary parameters, in the reference's argument
 *                order (ltc_cuda.py:249-263)
 *   out          (B,T,H) outputs
 *   h_final      (B,H) final state
 *   saved        ltc_saved_floats() floats, written when save_intermediates
 *                is nonzero (training); may be NULL otherwise
 * Unlike the reference (which swaps the roles of its transposed copies), the
 * parameters are read in place: no transposed copies are returned.
 */
int ltc_full_forward(const float* x, long long sxb, long long sxt, long long sxd,
                     const float* state,
                     const float* w_pos, const float* w_erev, const float* mu,
                     const float* sigma,
                     const float* sensory_mu, const float* sensory_sigma,
                     const float* sensory_erev, const float* sensory_w_pos,
                     const float* cm_t, const float* gleak_pos, const float* vleak,
                     int B, int T, int D, int H, int ode_unfolds, float epsilon,
                     int save_intermediates,
                     float* out, float* h_final, float* saved,
                     void* workspace, long long workspace_bytes, void* stream);

/*
 * Whole backward time loop. Replaces ltc_full_backward
 * (csrc/ltc_kernels.cu:962-984, bound at ltc_cuda.py:331-339).
 *   x, parameters  as given to the forward
 *   saved          the buffer the forward filled
 *   grad_out       (B,T,H) dL/d out with element strides sgb, sgt, sgh
 *   grad_h_final   (B,H) dL/d h_final, contiguous, or NULL for zero
 *                  (the reference substitutes zeros, ltc_cuda.py:326-328)
 * Outputs, all contiguous, in Function-input order (ltc_cuda.py:342-355):
 *   grad_x (B,T,D), grad_state (B,H), grad_w_pos, grad_w_erev, grad_mu,
 *   grad_sigma (H,H), grad_sensory_mu, grad_sensory_sigma,
 *   grad_sensory_erev, grad_sensory_w_pos (D,H), grad_cm_t, grad_gleak_pos,
 *   grad_vleak (H).
 */
int ltc_full_backward(const float* x, long long sxb, long long sxt, long long sxd,
                      const float* w_pos, const float* w_erev, const float* mu,
                      const float* sigma,
                      const float* sensory_mu, const float* sensory_sigma,
                      const float* sensory_erev, const float* sensory_w_pos,
                      const float* cm_t, const float* gleak_pos, const float* vleak,
                      const float* saved,
                      const float* grad_out, long long sgb, long long sgt, long long sgh,
                      const float* grad_h_final,
                      int B, int T, int D, int H, int ode_unfolds, float epsilon,
                      float* grad_x, float* grad_state,
                      float* grad_w_pos, float* grad_w_erev, float* grad_mu,
                      float* grad_sigma,
                      float* grad_sensory_mu, float* grad_sensory_sigma,
                      float* grad_sensory_erev, float* grad_sensory_w_pos,
                      float* grad_cm_t, float* grad_gleak_pos, float* grad_vleak,
                      void* workspace, long long workspace_bytes, void* stream);

/*
 * ltc_full_forward without a workspace argument. No counterpart in the
 * reference: it is for callers that cannot allocate device memory (code under
 * HIP graph capture, tight serving loops, harnesses that forbid hipMalloc).
 * The kernels' scratch (parameter images, sensory sums, cluster exchange
 * words) lives in a static device array of LTC_NOALLOC_SCRATCH_BYTES bytes,
 * which the library holds on every GPU it runs on until the process ends.
 * Sizes whose ltc_fwd_workspace_bytes() exceeds it return LTC_EUNSUPPORTED
 * before anything is launched. The call allocates nothing and arguments
 * mean what they mean for ltc_full_forward. Every call on one GPU shares
 * that GPU's array, and each call rewrites what it reads, so a call does not
 * depend on an earlier one; calls that overlap on one GPU (two streams, two
 * host threads) race on the array and must be serialised by the caller.
 */
#define LTC_NOALLOC_SCRATCH_BYTES (64LL * 1024 * 1024)
int ltc_full_forward_noalloc(const float* x, long long sxb, long long sxt, long long sxd,
                             const float* state,
                             const float* w_pos, const float* w_erev, const float* mu,
                             const float* sigma,
                             const float* sensory_mu, const float* sensory_sigma,
                             const float* sensory_erev, const float* sensory_w_pos,
                             const float* cm_t, const float* gleak_pos, const float* vleak,
                             int B, int T, int D, int H, int ode_unfolds, float epsilon,
                             int save_intermediates,
                             float* out, float* h_final, float* saved, void* stream);

/*
 * Module-level path: the whole TrueLiquidTimeConstant.forward
 * (reference ltc.py:249-326) and its backward in one call each. The caller
 * passes the module's leaves instead of the boundary tensors, and the
 * library computes the pre-transforms of ltc.py:259-283 itself:
 *   xa = LayerNorm(x; ln_weight, ln_bias, ln_eps) * input_w + input_b
 *   w_pos = softplus(w) * mask, w_erev = w_pos * erev,
 *   cm_t = softplus(cm) / (dt / ode_unfolds), gleak_pos = softplus(gleak),
 *   sensory_w_pos = softplus(sensory_w) * sensory_mask
 * (softplus with torch's threshold 20). The backward returns gradients
 * with respect to the leaves. No counterpart in the reference, whose
 * module runs these steps as separate PyTorch ops around the fused call
 * (ltc.py:259-307). D <= 1024; larger inputs use ltc_full_forward.
 * `saved` holds ltc_module_saved_floats() floats: the boundary's saved
 * buffer followed by the normalised input, its row statistics and the
 * parameter images built from the leaves at forward time (the backward reads
 * them instead of rebuilding them, so the leaves must not change in between).
 * `state` may be NULL for a zero initial state (the module's default when no
 * h0 is given), and `grad_state` may then be NULL too (nothing is written).
 */
long long ltc_module_saved_floats(int B, int T, int D, int H, int ode_unfolds);
long long ltc_module_fwd_workspace_bytes(int B, int T, int D, int H, int ode_unfolds);
long long ltc_module_bwd_workspace_bytes(int B, int T, int D, int H, int ode_unfolds);

int ltc_module_forward(const float* x, long long sxb, long long sxt, long long sxd,
                       const float* state,
                       const float* w, const float* erev, const float* mask,
                       const float* mu, const float* sigma,
                       const float* sensory_w, const float* sensory_erev,
                       const float* sensory_mask, const float* sensory_mu,
                       const float* sensory_sigma,
                       const float* gleak, const float* vleak, const float* cm,
                       const float* input_w, const float* input_b,
                       const float* ln_weight, const float* ln_bias,
                       int B, int T, int D, int H, int ode_unfolds, float dt, float epsilon,
                       float ln_eps, int save_intermediates,
                       float* out, float* h_final, float* saved,
                       void* workspace, long long workspace_bytes, void* stream);

int ltc_module_backward(const float* x, long long sxb, long long sxt, long long sxd,
                        const float* w, const float* erev, const float* mask,
                        const float* mu, const float* sigma,
                        const float* sensory_w, const float* sensory_erev,
                        const float* sensory_mask, const float* sensory_mu,
                        const float* sensory_sigma,
                        const float* gleak, const float* vleak, const float* cm,
                        const float* input_w, const float* input_b,
                        const float* ln_weight, const float* ln_bias,
                        const float* saved,
                        const float* grad_out, long long sgb, long long sgt, long long sgh,
                        const float* grad_h_final,
                        int B, int T, int D, int H, int ode_unfolds, float dt, float epsilon,
                        float ln_eps,
                        float* grad_x, float* grad_state,
                        float* grad_w, float* grad_erev, float* grad_mu, float* grad_sigma,
                        float* grad_sensory_w, float* grad_sensory_erev,
                        float* grad_sensory_mu, float* grad_sensory_sigma,
                        float* grad_gleak, float* grad_vleak, float* grad_cm,
                        float* grad_input_w, float* grad_input_b,
                        float* grad_ln_weight, float* grad_ln_bias,
                        void* workspace, long long workspace_bytes, void* stream);

/*
 * Per-step entry points. The reference exports them beside the T-loop
 * drivers (csrc/ltc_kernels.cu:1308-1311) for a Python-level time loop; its
 * own Python no longer calls them. Each one runs the same kernels as the
 * drivers with T = 1. Tensors are contiguous unless strides are given, and
 * outputs must not alias inputs.
 */

/* One step's sensory sums. Replaces ltc_sensory_fwd
 * (csrc/ltc_kernels.cu:675-713), including its argument order (sigma, mu,
 * w_pos, erev).
 *   inputs       (B,D) with element strides sib, sid
 *   w_num_sensory, w_den_sensory   (B,H) outputs: sum_d Ws*sig*Es, sum_d Ws*sig */
long long ltc_sensory_fwd_workspace_bytes(int B, int D, int H);
int ltc_sensory_fwd(const float* inputs, long long sib, long long sid,
                    const float* sensory_sigma, const float* sensory_mu,
                    const float* sensory_w_pos, const float* sensory_erev,
                    int B, int D, int H,
                    float* w_num_sensory, float* w_den_sensory,
                    void* workspace, long long workspace_bytes, void* stream);

/* One step's U implicit-Euler unfolds. Replaces ltc_ode_unfold_fwd
 * (csrc/ltc_kernels.cu:716-777).
 *   state        (B,H) state before the step; never written
 *   w_num_sensory, w_den_sensory   (B,H) the step's sensory sums
 *   state_out    (B,H) state after the U unfolds
 *   v_buffer     (U,B,H) the pre-state of every unfold, written when
 *                save_intermediates is nonzero (may be NULL otherwise) */
long long ltc_ode_unfold_fwd_workspace_bytes(int B, int H, int ode_unfolds);
int ltc_ode_unfold_fwd(const float* state, const float* w_pos, const float* w_erev,
                       const float* mu, const float* sigma,
                       const float* w_num_sensory, const float* w_den_sensory,
                       const float* cm_t, const float* gleak_pos, const float* vleak,
                       int B, int H, int ode_unfolds, float epsilon, int save_intermediates,
                       float* state_out, float* v_buffer,
                       void* workspace, long long workspace_bytes, void* stream);

/* Backward of ltc_sensory_fwd. Replaces ltc_sensory_bwd
 * (csrc/ltc_kernels.cu:780-837), same output order.
 *   grad_w_num, grad_w_den   (B,H) dL/d w_num_sensory, dL/d w_den_sensory
 *   grad_inputs  (B,D) contiguous; the four (D,H) parameter gradients */
long long ltc_sensory_bwd_workspace_bytes(int B, int D, int H);
int ltc_sensory_bwd(const float* grad_w_num, const float* grad_w_den,
                    const float* inputs, long long sib, long long sid,
                    const float* sensory_sigma, const float* sensory_mu,
                    const float* sensory_w_pos, const float* sensory_erev,
                    int B, int D, int H,
                    float* grad_inputs, float* grad_sensory_sigma, float* grad_sensory_mu,
                    float* grad_sensory_w_pos, float* grad_sensory_erev,
                    void* workspace, long long workspace_bytes, void* stream);

/* Backward of ltc_ode_unfold_fwd. Replaces ltc_ode_unfold_bwd
 * (csrc/ltc_kernels.cu:845-950), same output order.
 *   v_buffer     (U,B,H) from ltc_ode_unfold_fwd. The unfolds are recomputed
 *                from v_buffer[0], as the reference's backward kernels
 *                recompute each unfold (csrc/ltc_kernels.cu:549-668); the
 *                other slices are not read.
 *   grad_output  (B,H) dL/d state_out
 * Outputs: grad_v (B,H) = dL/d state, grad_w_num_sensory and
 * grad_w_den_sensory (B,H), grad_w_pos, grad_w_erev, grad_mu, grad_sigma
 * (H,H), grad_cm_t, grad_gleak_pos, grad_vleak (H). */
long long ltc_ode_unfold_bwd_workspace_bytes(int B, int H, int ode_unfolds);
int ltc_ode_unfold_bwd(const float* v_buffer, const float* w_pos, const float* w_erev,
                       const float* mu, const float* sigma,
                       const float* w_num_sensory, const float* w_den_sensory,
                       const float* cm_t, const float* gleak_pos, const float* vleak,
                       const float* grad_output, int B, int H, int ode_unfolds, float epsilon,
                       float* grad_v, float* grad_w_num_sensory, float* grad_w_den_sensory,
                       float* grad_w_pos, float* grad_w_erev, float* grad_mu,
                       float* grad_sigma, float* grad_cm_t, float* grad_gleak_pos,
                       float* grad_vleak,
                       void* workspace, long long workspace_bytes, void* stream);

/*
 * Sequence and token operators. No counterpart in the reference: a recurrence
 * whose time axis is parallel, and what turns a layer's outputs into token
 * scores and training losses. Tensors are fp32, bf16 or fp16 (LTC_F32, LTC_BF16,
 * LTC_F16), unit stride along their last dimension, any alignment their type
 * has; states, sums and statistics are fp32. Results are deterministic. A
 * workspace (256-byte aligned) serves one call at a time: calls on one stream may
 * share it, calls that may run at once may not. Nothing in it has to be cleared or
 * kept between calls. Outputs overlap neither inputs nor one another.
 */
#define LTC_F32 0
#define LTC_BF16 1
#define LTC_F16 2

/* Gate forms: a = sigmoid(gate), h = a h + (1 - a) x; a = exp(gate), h = a h + x.
 * exp(gate) over 1 is taken as it is: the product of the decays of any run of a
 * sequence's tokens has to stay in fp32's range then, and its outputs may be infinite
 * or NaN where it does not. */
#define LTC_GATE_BLEND 0
#define LTC_GATE_DECAY 1

/*
 * Gated linear recurrence over B sequences of T steps, or, with cu_seqlens
 * (B + 1 ascending int32 boundaries on the device), over B packed sequences of T
 * tokens in all: sequence s is tokens cu_seqlens[s] up to cu_seqlens[s + 1], and
 * may be empty. Tokens outside every sequence give zeros, in out and in the
 * gradients. Boundaries outside 0 ... T or out of order give unspecified results
 * without an access out of range. Workgroups hand states on through the workspace;
 * one whose wait for another outlasts ltc_set_cluster_spin_ticks()'s budget goes on
 * with NaN, and a sticky flag of the device is raised (ltc_scan_status).
 *   x            (B,T,H) with element strides sxb, sxt; packed (T,H), stride sxt
 *   gate         likewise; its type is x's or LTC_F32
 *   state        (B,H) fp32 contiguous, or NULL for zero
 *   out          (B,T,H) or (T,H), x's type, contiguous
 *   state_final  (B,H) fp32: the last state; an empty sequence's initial one
 *   saved        ltc_gated_scan_saved_floats() floats, written when save is
 *                nonzero, for the backward of the same x, gate, state, cu_seqlens
 */
long long ltc_gated_scan_saved_floats(int B, int T, int H, int packed);
long long ltc_gated_scan_fwd_workspace_bytes(int B, int T, int H, int packed);
long long ltc_gated_scan_bwd_workspace_bytes(int B, int T, int H, int packed);
int ltc_gated_scan_forward(const void* x, long long sxb, long long sxt, const void* gate,
                           long long sgb, long long sgt, const float* state,
                           const int* cu_seqlens, int x_type, int gate_type, int form, int B,
                           int T, int H, int save, void* out, float* state_final, float* saved,
                           void* workspace, long long workspace_bytes, void* stream);

/*
 * Its backward. grad_out (NULL for zero) has x's shape and type and strides sob,
 * sot; grad_state_final (B,H) fp32 contiguous or NULL for zero. grad_x (x's type),
 * grad_gate (the gate's) and grad_state (B,H) fp32 are contiguous; each may be
 * NULL where it is not wanted.
 */
int ltc_gated_scan_backward(const void* x, long long sxb, long long sxt, const void* gate,
                            long long sgb, long long sgt, const float* state,
                            const int* cu_seqlens, int x_type, int gate_type, int form, int B,
                            int T, int H, const float* saved, const void* grad_out,
                            long long sob, long long sot, const float* grad_state_final,
                            void* grad_x, void* grad_gate, float* grad_state, void* workspace,
                            long long workspace_bytes, void* stream);

/*
 * Whether a scan on the current device has given up a wait, forward or backward: waits
 * for the device and returns LTC_EHIP with a message if so, clearing the flag when
 * `clear` is nonzero. ltc_device_status() reports the other kernels' waits, not these.
 * As that, not to be called under graph capture.
 */
int ltc_scan_status(int clear);

/*
 * One token of B streams: out[b] and the stream's new state, written over the old.
 *   x, gate      (B,H), row strides sxb, sgb
 *   state        (P,H) fp32, row stride ssp (at least H)
 *   slots        int32 (B): the row of state of each row, or NULL for row b (P = B).
 *                A negative slot is padding: its row of out is zero and no state is
 *                touched. A slot of P or more gives a row of NaN. Rows that name the
 *                same slot are taken in their order, as tokens of one stream.
 *   out          (B,H), x's type, contiguous
 */
int ltc_gated_scan_step(const void* x, long long sxb, const void* gate, long long sgb,
                        float* state, long long ssp, const int* slots, int x_type,
                        int gate_type, int form, int B, int H, int P, void* out, void* stream);

/*
 * Log probabilities of given tokens under softmax(logits / temperature), the
 * distribution's entropy, and its `top` most probable tokens.
 *   logits       (N,V), row stride sl
 *   ids          (N) int32 or (ids64 nonzero) int64. A negative id is a row without
 *                a token: log probability and entropy 0, gradient 0. An id of V or
 *                more gives NaN.
 *   logp, entropy   (N) fp32; entropy may be NULL
 *   top_logp, top_ids   (N,top) fp32 and int64, most probable first, equal logits by
 *                the lower id; every row, with a token or not. top <= LTC_TOP_MAX
 *                and <= V; 0 for none
 *   temperature  positive and finite, as log2(e) over it is (4.3e-39 and up)
 *   stats        (N,3) fp32 for the backward, or NULL
 * A logit of -inf has probability 0; a row of nothing else, or with a NaN or +inf,
 * gives NaN (in such a row top_ids are in range, but otherwise unspecified).
 */
#define LTC_TOP_MAX 32
long long ltc_token_logprobs_workspace_bytes(long long N, int V, int top, int logits_type);
int ltc_token_logprobs_forward(const void* logits, long long sl, const void* ids, int ids64,
                               int logits_type, long long N, int V, int top, float temperature,
                               float* logp, float* entropy, float* top_logp, long long* top_ids,
                               float* stats, void* workspace, long long workspace_bytes,
                               void* stream);
/* grad_logp, grad_entropy: (N) fp32 with strides slp, sen, or NULL for zero;
 * grad_logits (N,V) contiguous, the logits' type. */
int ltc_token_logprobs_backward(const void* logits, long long sl, const void* ids, int ids64,
                                int logits_type, long long N, int V, float temperature,
                                const float* stats, const float* grad_logp, long long slp,
                                const float* grad_entropy, long long sen, void* grad_logits,
                                void* stream);

/*
 * Distillation from a teacher's top logits:
 *   loss = temperature^2 sum_k p_k (log p_k - log q[teacher_ids[k]]),
 * p the softmax of the row's teacher_logits / temperature over the entries that are
 * there, q = softmax(logits / temperature) over the vocabulary.
 *   teacher_logits  (N,K), row stride st; any of the types
 *   teacher_ids     (N,K) int32 or int64, row stride si; a negative id is an entry
 *                that is not there, one of V or more gives NaN. An id may come twice.
 *                1 <= K <= LTC_TEACHER_MAX
 *   loss         (N) fp32; 0 for a row without entries, or whose entries' logits are
 *                all -inf
 * The backward gives dL/dlogits from grad_loss (N), stride sgl, and the forward's
 * stats, (N,4) fp32 or NULL there; the teacher gets none.
 */
#define LTC_TEACHER_MAX 1024
long long ltc_top_distill_workspace_bytes(long long N, int V, int logits_type);
int ltc_top_distill_forward(const void* logits, long long sl, const void* teacher_logits,
                            long long st, const void* teacher_ids, long long si, int ids64,
                            int logits_type, int teacher_type, long long N, int V, int K,
                            float temperature, float* loss, float* stats, void* workspace,
                            long long workspace_bytes, void* stream);
int ltc_top_distill_backward(const void* logits, long long sl, const void* teacher_logits,
                             long long st, const void* teacher_ids, long long si, int ids64,
                             int logits_type, int teacher_type, long long N, int V, int K,
                             float temperature, const float* stats, const float* grad_loss,
                             long long sgl, void* grad_logits, void* stream);

/*
 * Operators of a token model around the layer: what brings tokens in, mixes them and
 * adjusts the scores of the next. No counterpart in the reference. Types, workspaces and
 * determinism as above.
 */

/* Activations: none; v / (1 + exp(-v)). */
#define LTC_ACT_NONE 0
#define LTC_ACT_SILU 1

/*
 * Short causal convolution of each channel, over B sequences of T steps or packed ones
 * (cu_seqlens as in ltc_gated_scan_forward):
 *   out_t = act(bias + sum_k weight[:,k] in_{t-K+1+k}),
 * where in is the sequence with its state, its last K-1 inputs, before it.
 *   x            (B,T,C) with element strides sxb, sxt; packed (T,C), stride sxt
 *   weight       (C,K) contiguous; its type is x's or LTC_F32. K <= LTC_CONV_TAPS_MAX
 *   bias         (C), weight's type, or NULL for none
 *   state        (B,K-1,C) contiguous, x's type, or NULL for zero
 *   out          (B,T,C) or (T,C), contiguous, x's type
 *   state_final  (B,K-1,C) contiguous: the last K-1 inputs, the state's own among them
 *                where a sequence is shorter
 * The backward takes grad_out (NULL for zero; strides sob, sot) and grad_state_final
 * (contiguous, or NULL for zero). Its outputs are contiguous, of their input's type, and
 * each may be NULL where it is not wanted.
 */
#define LTC_CONV_TAPS_MAX 8
long long ltc_causal_conv_bwd_workspace_bytes(int x_type, int B, int T, int C, int K, int packed);
int ltc_causal_conv_forward(const void* x, long long sxb, long long sxt, const void* weight,
                            const void* bias, const void* state, const int* cu_seqlens,
                            int x_type, int weight_type, int activation, int B, int T, int C,
                            int K, void* out, void* state_final, void* stream);
int ltc_causal_conv_backward(const void* x, long long sxb, long long sxt, const void* weight,
                             const void* bias, const void* state, const int* cu_seqlens,
                             int x_type, int weight_type, int activation, int B, int T, int C,
                             int K, const void* grad_out, long long sob, long long sot,
                             const void* grad_state_final, void* grad_x, void* grad_weight,
                             void* grad_bias, void* grad_state, void* workspace,
                             long long workspace_bytes, void* stream);

/*
 * One token of B streams: out[b], and x[b] joins the stream's last inputs, the oldest
 * leaving. state (P,K-1,C) with strides ssp, sst and 1, its rows apart; slots as in
 * ltc_gated_scan_step.
 */
int ltc_causal_conv_step(const void* x, long long sxb, const void* weight, const void* bias,
                         void* state, long long ssp, long long sst, const int* slots,
                         int x_type, int weight_type, int activation, int B, int C, int K,
                         int P, void* out, void* stream);

/*
 * Selective state space scan, over B sequences of T steps or packed ones. Of channel h in
 * group g = h / (H / G), and state n:
 *   s_t = delta_t + delta_bias, or softplus of it
 *   v_t = exp(s_t A[h,n]) v_{t-1} + s_t B_t[g,n] x_t
 *   out_t = (sum_n C_t[g,n] v_t + D x_t) silu(z_t)      (without z: no factor)
 *   x, delta, z  (B,T,H) with element strides s.b, s.t; packed (T,H), stride s.t; z NULL
 *                for none
 *   A            (H,N) fp32 contiguous; taken as it is: above 0 states may grow without
 *                bound. N <= LTC_STATES_MAX
 *   B, C         (B,T,G,N) with element strides s.b, s.t, s.g; packed (T,G,N)
 *   D, delta_bias   (H) fp32, or NULL for none
 *   state        (B,H,N) fp32 contiguous, or NULL for zero
 *   out          (B,T,H) or (T,H), contiguous
 *   state_final  (B,H,N) fp32 contiguous: the last state; an empty sequence's initial one
 *   saved        ltc_selective_scan_saved_floats() floats, written when save is nonzero,
 *                for the backward of the same inputs
 * x, delta, z, B, C, out and their gradients have one type. Tokens outside every sequence
 * give zeros, in out and in the gradients, whatever lies there. For the backward every
 * sequence of a batch takes H N floats at least of saved, and as many of workspace, however
 * short it is; packed sequences do not.
 */
#define LTC_STATES_MAX 64
long long ltc_selective_scan_saved_floats(int B, int T, int H, int N, int G, int packed);
long long ltc_selective_scan_fwd_workspace_bytes(int B, int T, int H, int N, int G, int packed);
long long ltc_selective_scan_bwd_workspace_bytes(int B, int T, int H, int N, int G, int packed);
int ltc_selective_scan_forward(const void* x, long long sxb, long long sxt, const void* delta,
                               long long sdb, long long sdt, const float* A, const void* Bm,
                               long long sbb, long long sbt, long long sbg, const void* Cm,
                               long long scb, long long sct, long long scg, const float* D,
                               const void* z, long long szb, long long szt,
                               const float* delta_bias, const float* state,
                               const int* cu_seqlens, int type, int delta_softplus, int B,
                               int T, int H, int N, int G, int save, void* out,
                               float* state_final, float* saved, void* workspace,
                               long long workspace_bytes, void* stream);
/* grad_out (NULL for zero) has strides sob, sot; grad_state_final is contiguous or NULL for
 * zero. The gradients are contiguous, of their input's shape and type; each may be NULL
 * where it is not wanted. */
int ltc_selective_scan_backward(const void* x, long long sxb, long long sxt, const void* delta,
                                long long sdb, long long sdt, const float* A, const void* Bm,
                                long long sbb, long long sbt, long long sbg, const void* Cm,
                                long long scb, long long sct, long long scg, const float* D,
                                const void* z, long long szb, long long szt,
                                const float* delta_bias, const float* state,
                                const int* cu_seqlens, int type, int delta_softplus, int B,
                                int T, int H, int N, int G, const float* saved,
                                const void* grad_out, long long sob, long long sot,
                                const float* grad_state_final, void* grad_x, void* grad_delta,
                                float* grad_A, void* grad_B, void* grad_C, float* grad_D,
                                void* grad_z, float* grad_delta_bias, float* grad_state,
                                void* workspace, long long workspace_bytes, void* stream);

/*
 * One token of B streams: x, delta, z (B,H) with row strides, B and C (B,G,N); state
 * (P,H,N) fp32, row stride ssp (at least H N), written over; slots as in
 * ltc_gated_scan_step.
 */
int ltc_selective_scan_step(const void* x, long long sx, const void* delta, long long sd,
                            const float* A, const void* Bm, long long sbb, long long sbg,
                            const void* Cm, long long scb, long long scg, const float* D,
                            const void* z, long long sz, const float* delta_bias, float* state,
                            long long ssp, const int* slots, int type, int delta_softplus,
                            int B, int H, int N, int G, int P, void* out, void* stream);

/*
 * Embedding: out[i] = scale table[ids[i]].
 *   table        (V,H), row stride st
 *   ids          (n) int32 or (ids64 nonzero) int64. A negative id is a token that is not
 *                there: a row of zeros and no gradient; one of V or more gives NaN and
 *                no gradient
 *   out          (n,H) contiguous, the table's type
 * The backward writes grad_table (V,H) contiguous, every row: scale times the sum of
 * grad_out (n,H; row stride so) over the row's tokens, in their order.
 */
int ltc_embed_forward(const void* table, long long st, const void* ids, int ids64, int type,
                      long long n, int V, int H, float scale, void* out, void* stream);
long long ltc_embed_bwd_workspace_bytes(long long n, int V, int H);
int ltc_embed_backward(const void* ids, int ids64, int type, long long n, int V, int H,
                       float scale, const void* grad_out, long long so, void* grad_table,
                       void* workspace, long long workspace_bytes, void* stream);

/*
 * Logits adjusted for the choice of the next token. In fp32, of token v in row r, x its
 * logit, and in this order:
 *   v occurs in the context:               x / repetition where x > 0, else x repetition
 *   v occurs c > 0 times after the prompt: x - frequency c - presence
 *   v is in the list of biases:            plus the sum of its biases, in their order
 *   v is not allowed by the mask:          -inf, whatever x is
 *   logits       (R,V), row stride sl
 *   context      (R,ctx) int32 or (context64 nonzero) int64, row stride sc. Entries
 *                outside 0 ... V-1 are not there. ctx 0 for none
 *   prompt_lens  (R) int32: the entries of the context that are the prompt, its first; NULL
 *                for 0
 *   repetition, frequency, presence   (R) fp32, or NULL for the values of the same name
 *                with a 0, which are finite, repetition0 positive
 *   bias_ids     (R,K) int32 or int64, row stride sbi, entries outside 0 ... V-1 not there;
 *                bias (R,K) fp32, row stride sb. K <= LTC_BIAS_MAX, 0 for none
 *   mask         (R, (V + 31) / 32) int32 words, row stride sm: token v is allowed where
 *                bit v % 32 of word v / 32 is set; NULL for all
 *   out          (R,V) contiguous, the logits' type
 * Row strides of 0 share a row among all.
 */
#define LTC_BIAS_MAX 1024
int ltc_adjust_logits(const void* logits, long long sl, const void* context, long long sc,
                      int context64, int ctx, const int* prompt_lens, const float* repetition,
                      const float* frequency, const float* presence, float repetition0,
                      float frequency0, float presence0, const void* bias_ids, long long sbi,
                      int bias_ids64, const float* bias, long long sb, int K, const int* mask,
                      long long sm, int logits_type, long long R, int V, void* out,
                      void* stream);

/*
 * Launch plan of one call, for diagnostics and host-side bounds tests. No
 * counterpart in the reference. Writes up to n of: Hp, Dp, NB (batch rows
 * per ODE workgroup), KS (reduction split), RC (= Hp/KS), threads per ODE
 * workgroup, forward LDS bytes, backward LDS bytes (the chain launch's
 * request: with the module path's sensory companions, the larger of the
 * chain's and a companion's), NCH (recurrent gradient
 * chunks, or one per workgroup when fused), NRC (sensory backward row
 * chunks), ODE workgroups, 1 when the recurrent parameter gradients are
 * accumulated inside the chain kernel, then the chain kernel's own KS, RC
 * and threads (the fields before them describe the forward kernel), then CP
 * and NCL: with CP > 0 the ODE kernels run as NCL clusters of CP workgroups
 * that each own 64 columns of NB rows (threads and LDS fields then describe
 * one cluster member), then the chain kernel's cluster size, rows per
 * cluster and workgroups (its clusters may differ from the forward's when
 * its parameter gradients are fused), then 1 when the forward and 1 when the
 * chain kernel read compacted images (they then skip the recurrent synapses
 * that cannot contribute: zero weights in the forward, zero mask entries in
 * the module path's chain), then two module-path fields: 1 when the
 * forward's parameter-image launch also forms the sensory sums (few rows,
 * D <= 128, H a multiple of 4, and 16-byte aligned sensory leaves at the
 * call: no separate sensory launch), 1 when the backward runs the sensory
 * and LayerNorm backward inside the chain launch (Hp = 64), and 1 when it
 * forms the recurrent parameter-gradient sums inside the chain launch
 * (Hp = 128: no separate recurrent-gradient launch), then the launches of
 * the forward and of the chain ODE kernel per call: 1, or at Hp > 1024 with
 * more rows than one launch of at most one workgroup per CU holds, one
 * launch per NCL * NB rows, then 1 when the module forward's sensory launch
 * walks one list per neuron over all of D (64 < D <= 256 with many rows)
 * instead of per 64-input chunk, then five fields of the register-resident
 * forward clusters (128 < H <= 512 where the geometry above would stream its
 * operands): workgroups per cluster (0: not used, and the forward runs in the
 * geometry above), columns per workgroup, rows per cluster, launches per call
 * and LDS bytes per workgroup. They keep the state's NaN treatment of the
 * geometry they replace (cmp_fwd above); then five of the register-resident
 * chain (members of 32 columns, parameter gradients fused): workgroups per
 * cluster (0: not used), rows per cluster, launches per call, LDS bytes per
 * workgroup, and unfolds between the moves of its gradient sums out of the
 * registers (0: none); then 1 when the register-resident forward, and 1 when the
 * chain, takes its synapses from the dense image (few unfolds; a backward over
 * the boundary tensors always does). Returns the number of values written, or -1
 * for invalid sizes. The plan depends on the current device's CU count.
 */
#define LTC_PLAN_FIELDS 40
int ltc_launch_plan(int B, int T, int D, int H, int ode_unfolds, long long* out, int n);

/*
 * Cluster give-up. For H > 128 the ODE kernels run as clusters of workgroups
 * that exchange values every unfold and must all be resident at once (the
 * plan asks for at most one workgroup per CU). Each wait is bounded; when a
 * member runs out of its budget (another kernel held the CUs its partners
 * needed), the whole cluster leaves early, and the call then overwrites
 * every output it writes (out, h_final and saved for a forward; every
 * gradient for a backward) with NaN and raises a sticky per-device fault flag.
 * For 128 < H <= 192, and for larger batches at 192 < H <= 512 (plan field CP
 * = 0: the plan itself has no clusters), nothing is lost instead: kernels that
 * wait on nobody are queued behind the clusters and make the results, and no
 * flag is raised.
 * The module-path backward with one batch row per workgroup and B <= 64 also
 * runs companion workgroups that wait for the chain workgroups the same
 * bounded way, with the same outcome (every gradient, dL/dx and dL/dh0 NaN,
 * the flag raised) when one runs out:
 *   - at H <= 64 and D <= 128, one companion per row runs the sensory and
 *     LayerNorm backward from each step's dL/dsn, dL/dsd;
 *   - at 64 < H <= 128, two companions per row form the recurrent
 *     parameter-gradient sums from each unfold's alpha and beta, and with
 *     D <= 128 two more per row run the sensory and LayerNorm backward, the
 *     second of them also waiting for the first's dL/dxa sums.
 * The call itself has already returned LTC_OK by then (it only queues work);
 * ltc_device_status() waits for the current device, returns LTC_EHIP with a
 * message when the flag is raised, and clears it when `clear` is nonzero.
 * It synchronises the device, so it must not be called under graph capture.
 * The gated scan's waits have a flag of their own (ltc_scan_status()).
 * No counterpart in the reference, whose kernels have no inter-block waits.
 */
int ltc_device_status(int clear);

/* Wait budget of every cluster exchange (and companion wait, and of the gated
 * scan's waits), in ticks of the GPU's 100 MHz wall
 * clock (default 20000000 = 0.2 s), for calls made after it returns; returns
 * the previous budget, or -1 for a negative argument. A budget of 0 makes
 * every member give up at its first wait: a host-forced failure for tests of
 * the give-up path (every kernel still exits normally). No counterpart in the
 * reference. */
long long ltc_set_cluster_spin_ticks(long long ticks);

/*
 * Per-kernel event timing. No counterpart in the reference, whose bench
 * times with torch.cuda.Event around whole calls (bench_ltc.py:39-96).
 * While enabled, every kernel this library launches is bracketed by HIP
 * events recorded on the launch stream; ltc_timing_read() waits for them and
 * returns the summed duration and launch count of one kernel id.
 * ltc_timing_enable() clears the accumulators.
 */
int ltc_timing_enable(int on);
int ltc_timing_read(int kernel_id, double* total_ms, long long* launches);
int ltc_kernel_count(void);
const char* ltc_kernel_name(int kernel_id);

#ifdef __cplusplus
}
#endif

#endif /* LTC_CAPI_H */
