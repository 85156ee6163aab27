// C-ABI entry points of the token model's operators (include/ltc_capi.h): argument
// checks, workspace layout and launches. Allocates no device memory.
#include <hip/hip_runtime.h>

#include <climits>
#include <string>

#include "ltc_capi_util.h"
#include "ltc_model_internal.h"

using ltc::check_workspace;
using ltc::host_clear_error;
using ltc::host_fail;
using ltc::host_hip_fail;
using ltc::host_timed;
using ltc::kMaxGroups;
using ltc::known_type;
using ltc::Pieces;

namespace {

static_assert(LTC_CONV_TAPS_MAX == ltc::kConvTapsMax && LTC_STATES_MAX == ltc::kSsmStatesMax &&
                  LTC_BIAS_MAX == ltc::kBiasMax,
              "limits");

// Tokens are numbered in 32 bits, up to a workgroup's behind the last.
constexpr long long kMaxTokens = INT_MAX - (1 << 16);

int finish(hipError_t e, const char* what) { return e == hipSuccess ? LTC_OK : host_hip_fail(what, e); }

int check_step_rows(int B, int P, const void* slots) {
  if (P < 0 || (B > 0 && !slots && P != B))
    return host_fail(LTC_EINVAL, "P must be at least 0, and B without slots where there are rows");
  if (B > 65535) return host_fail(LTC_EUNSUPPORTED, "at most 65535 rows a step");
  return LTC_OK;
}

// ---------------------------------------------------------------------------
// Causal convolution
// ---------------------------------------------------------------------------
int check_conv(int B, int T, int C, int K, int packed) {
  if (B < 0 || T < 0 || C < 1 || K < 1 || K > LTC_CONV_TAPS_MAX)
    return host_fail(LTC_EINVAL, "dimensions must satisfy B >= 0, T >= 0, C >= 1, 1 <= K <= " +
                                     std::to_string(LTC_CONV_TAPS_MAX));
  if ((packed ? (long long)T : (long long)B * T) > kMaxTokens || C > INT_MAX / 16 || B > INT_MAX - 1)
    return host_fail(LTC_EUNSUPPORTED, "problem too large");
  return LTC_OK;
}

int conv_args(ltc::ConvArgs* a, int x_type, bool bwd, int B, int T, int C, int K, int packed) {
  int rc = check_conv(B, T, C, K, packed);
  if (rc != LTC_OK) return rc;
  if (!known_type(x_type)) return host_fail(LTC_EINVAL, "x_type must be LTC_F32, LTC_BF16 or LTC_F16");
  a->B = B;
  a->T = T;
  a->C = C;
  a->N = packed ? T : (long long)B * T;
  ltc::conv_tiles(x_type, bwd, a);
  if ((a->tiles + B) > kMaxGroups / a->cblocks) return host_fail(LTC_EUNSUPPORTED, "problem too large");
  return LTC_OK;
}

int check_conv_types(int x_type, int weight_type, int activation) {
  if (weight_type != x_type && weight_type != LTC_F32)
    return host_fail(LTC_EINVAL, "weight_type must be x_type or LTC_F32");
  if (activation != LTC_ACT_NONE && activation != LTC_ACT_SILU)
    return host_fail(LTC_EINVAL, "activation must be LTC_ACT_NONE or LTC_ACT_SILU");
  return LTC_OK;
}

// ---------------------------------------------------------------------------
// Selective scan
// ---------------------------------------------------------------------------
int ssm_args(ltc::SsmArgs* a, int B, int T, int H, int N, int G, int packed, bool bwd) {
  if (B < 0 || T < 0 || H < 1 || N < 1 || G < 1)
    return host_fail(LTC_EINVAL, "dimensions must satisfy B >= 0, T >= 0, H >= 1, N >= 1, G >= 1");
  if (H % G != 0) return host_fail(LTC_EINVAL, "H must be a multiple of G");
  if (N > LTC_STATES_MAX)
    return host_fail(LTC_EUNSUPPORTED, "at most " + std::to_string(LTC_STATES_MAX) + " states a channel");
  const long long ntok = packed ? T : (long long)B * T;
  if (ntok > kMaxTokens || H > INT_MAX / 1024 || B > INT_MAX - 1)
    return host_fail(LTC_EUNSUPPORTED, "problem too large");
  a->B = B;
  a->T = T;
  a->H = H;
  a->N = N;
  a->G = G;
  a->ntok = ntok;
  ltc::ssm_plan(a, packed != 0, bwd);
  const long long items = a->lines * a->chunks, hn = (long long)H * N;
  if (items > kMaxGroups / ((long long)G * a->hblocks) || ntok > kMaxGroups * 32 / ((long long)G * N) ||
      (a->lines + 1) > kMaxGroups * 256 / hn)
    return host_fail(LTC_EUNSUPPORTED, "problem too large");
  return LTC_OK;
}

long long saved_floats(const ltc::SsmArgs& a) {
  return a.lines * a.tiles * a.H * a.N;
}

void carve_ssm(Pieces& c, ltc::SsmArgs& a, bool bwd) {
  const long long items = a.lines * a.chunks, hn = (long long)a.H * a.N;
  if (a.chunks > 1) {
    a.ends = c.take<float>(items * hn);
    a.sumd = c.take<float>(items * a.H);
    a.drops = c.take<int>(items);
  }
  if (bwd) {
    constexpr int E = ltc::kSsmBwdStates;
    a.part_bc = c.take<float>(a.hblocks * a.ntok * a.G * ((a.N + E - 1) / E) * 2 * E);
    a.part_a = c.take<float>(items * hn);
    a.part_h = c.take<float>(items * 2 * a.H);
  }
}

int check_ssm_inputs(const ltc::SsmArgs& a, int type) {
  if (!known_type(type)) return host_fail(LTC_EINVAL, "type must be LTC_F32, LTC_BF16 or LTC_F16");
  if (!a.A) return host_fail(LTC_EINVAL, "A pointer is NULL");
  if (a.ntok > 0 && (!a.x || !a.d || !a.Bm || !a.Cm))
    return host_fail(LTC_EINVAL, "x/delta/B/C pointer is NULL");
  return LTC_OK;
}

// ---------------------------------------------------------------------------
// Embedding
// ---------------------------------------------------------------------------
int check_embed(int type, long long n, int V, int H) {
  if (n < 0 || V < 1 || H < 1) return host_fail(LTC_EINVAL, "sizes must satisfy n >= 0, V >= 1, H >= 1");
  if (!known_type(type)) return host_fail(LTC_EINVAL, "type must be LTC_F32, LTC_BF16 or LTC_F16");
  if (n > kMaxTokens || n > 2 * kMaxGroups || V > 2 * kMaxGroups || H > INT_MAX / 16)
    return host_fail(LTC_EUNSUPPORTED, "problem too large");
  return LTC_OK;
}

void carve_embed(Pieces& c, ltc::EmbedArgs& a) {
  ltc::embed_digits(&a);
  a.tiles = (int)((a.n + ltc::kSortTile - 1) / ltc::kSortTile);
  if (a.n == 0) return;
  for (int i = 0; i < 2; ++i) {
    a.key[i] = c.take<int>(a.n);
    a.pos[i] = c.take<int>(a.n);
  }
  a.counts = c.take<unsigned>((a.tiles + 1LL) << a.bits);
  a.begin = c.take<int>(a.V);
  a.end = c.take<int>(a.V);
  a.sums = c.take<float>((a.n + ltc::kEmbedPiece - 1) / ltc::kEmbedPiece * a.H);
}

}  // namespace

extern "C" {

long long ltc_causal_conv_bwd_workspace_bytes(int x_type, int B, int T, int C, int K, int packed) {
  ltc::ConvArgs a{};
  if (conv_args(&a, x_type, true, B, T, C, K, packed) != LTC_OK) return -1;
  Pieces c{nullptr};
  c.take<float>(a.tiles * (K + 1) * C);
  return c.off;
}

int ltc_causal_conv_forward(const void* x, long long sxb, long long sxt, const void* weight, const void* bias,
                            const void* state, const int* cu_seqlens, int x_type, int weight_type, int activation,
                            int B, int T, int C, int K, void* out, void* state_final, void* stream) {
  host_clear_error();
  ltc::ConvArgs a{};
  const int packed = cu_seqlens != nullptr;
  int rc = conv_args(&a, x_type, false, B, T, C, K, packed);
  if (rc != LTC_OK || (rc = check_conv_types(x_type, weight_type, activation)) != LTC_OK) return rc;
  if (!weight) return host_fail(LTC_EINVAL, "weight pointer is NULL");
  if (a.N > 0 && (!x || !out)) return host_fail(LTC_EINVAL, "x/out pointer is NULL");
  if (B > 0 && K > 1 && !state_final) return host_fail(LTC_EINVAL, "state_final pointer is NULL");
  a.x = x;
  a.sxb = sxb;
  a.sxt = sxt;
  a.w = weight;
  a.bias = bias;
  a.state = state;
  a.cu = cu_seqlens;
  a.w_f32 = weight_type == LTC_F32;
  a.silu = activation == LTC_ACT_SILU;
  a.out = out;
  a.hf = state_final;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  return finish(host_timed(ltc::K_CONV_FWD, [&] { return ltc::launch_conv_fwd(x_type, K, a, s); }),
                "causal convolution launch");
}

int ltc_causal_conv_backward(const void* x, long long sxb, long long sxt, const void* weight, const void* bias,
                             const void* state, const int* cu_seqlens, int x_type, int weight_type,
                             int activation, int B, int T, int C, int K, const void* grad_out, long long sob,
                             long long sot, const void* grad_state_final, void* grad_x, void* grad_weight,
                             void* grad_bias, void* grad_state, void* workspace, long long workspace_bytes,
                             void* stream) {
  host_clear_error();
  ltc::ConvArgs a{};
  const int packed = cu_seqlens != nullptr;
  int rc = conv_args(&a, x_type, true, B, T, C, K, packed);
  if (rc != LTC_OK || (rc = check_conv_types(x_type, weight_type, activation)) != LTC_OK) return rc;
  if (!weight) return host_fail(LTC_EINVAL, "weight pointer is NULL");
  if (a.N > 0 && !x) return host_fail(LTC_EINVAL, "x pointer is NULL");
  Pieces need{nullptr};
  need.take<float>(a.tiles * (K + 1) * C);
  rc = check_workspace(need.off, workspace, workspace_bytes);
  if (rc != LTC_OK) return rc;
  a.x = x;
  a.sxb = sxb;
  a.sxt = sxt;
  a.w = weight;
  a.bias = bias;
  a.state = state;
  a.cu = cu_seqlens;
  a.w_f32 = weight_type == LTC_F32;
  a.silu = activation == LTC_ACT_SILU;
  a.go = grad_out;
  a.sob = sob;
  a.sot = sot;
  a.gh = grad_state_final;
  a.gx = grad_x;
  a.gw = grad_weight;
  a.gb = grad_bias;
  a.gs = grad_state;
  if (grad_weight || grad_bias) a.part = static_cast<float*>(workspace);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  return finish(host_timed(ltc::K_CONV_BWD, [&] { return ltc::launch_conv_bwd(x_type, K, a, s); }),
                "causal convolution backward launch");
}

int ltc_causal_conv_step(const void* x, long long sxb, const void* weight, const void* bias, void* state,
                         long long ssp, long long sst, const int* slots, int x_type, int weight_type,
                         int activation, int B, int C, int K, int P, void* out, void* stream) {
  host_clear_error();
  int rc = check_conv(B, 1, C, K, 0);
  if (rc != LTC_OK) return rc;
  if (!known_type(x_type)) return host_fail(LTC_EINVAL, "x_type must be LTC_F32, LTC_BF16 or LTC_F16");
  if ((rc = check_conv_types(x_type, weight_type, activation)) != LTC_OK) return rc;
  if ((rc = check_step_rows(B, P, slots)) != LTC_OK) return rc;
  if (!weight) return host_fail(LTC_EINVAL, "weight pointer is NULL");
  if (K > 2 && P > 0 && sst < C) return host_fail(LTC_EINVAL, "the rows of state overlap");
  if (K > 1 && P > 1 && ssp < (K - 2) * sst + C) return host_fail(LTC_EINVAL, "the rows of state overlap");
  if (B > 0 && (!x || !out)) return host_fail(LTC_EINVAL, "x/out pointer is NULL");
  if (B > 0 && P > 0 && K > 1 && !state) return host_fail(LTC_EINVAL, "state pointer is NULL");
  const ltc::ConvStepArgs a{x,     sxb,   weight, bias, weight_type == LTC_F32, activation == LTC_ACT_SILU,
                            state, ssp,   sst,    slots, B, C, P, out};
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  return finish(host_timed(ltc::K_CONV_STEP, [&] { return ltc::launch_conv_step(x_type, K, a, s); }),
                "causal convolution step launch");
}

long long ltc_selective_scan_saved_floats(int B, int T, int H, int N, int G, int packed) {
  ltc::SsmArgs a{};
  return ssm_args(&a, B, T, H, N, G, packed, true) == LTC_OK ? saved_floats(a) : -1;
}

static long long ssm_bytes(int B, int T, int H, int N, int G, int packed, bool bwd) {
  ltc::SsmArgs a{};
  if (ssm_args(&a, B, T, H, N, G, packed, bwd) != LTC_OK) return -1;
  Pieces c{nullptr};
  carve_ssm(c, a, bwd);
  return c.off;
}
long long ltc_selective_scan_fwd_workspace_bytes(int B, int T, int H, int N, int G, int packed) {
  return ssm_bytes(B, T, H, N, G, packed, false);
}
long long ltc_selective_scan_bwd_workspace_bytes(int B, int T, int H, int N, int G, int packed) {
  return ssm_bytes(B, T, H, N, G, packed, true);
}

int ltc_selective_scan_forward(const void* x, long long sxb, long long sxt, const void* delta, long long sdb,
                               long long sdt, const float* A, const void* Bm, long long sbb, long long sbt,
                               long long sbg, const void* Cm, long long scb, long long sct, long long scg,
                               const float* D, const void* z, long long szb, long long szt,
                               const float* delta_bias, const float* state, const int* cu_seqlens, int type,
                               int delta_softplus, int B, int T, int H, int N, int G, int save, void* out,
                               float* state_final, float* saved, void* workspace, long long workspace_bytes,
                               void* stream) {
  host_clear_error();
  ltc::SsmArgs a{};
  int rc = ssm_args(&a, B, T, H, N, G, cu_seqlens != nullptr, false);
  if (rc != LTC_OK) return rc;
  a.x = x, a.sxb = sxb, a.sxt = sxt;
  a.d = delta, a.sdb = sdb, a.sdt = sdt;
  a.z = z, a.szb = szb, a.szt = szt;
  a.Bm = Bm, a.sbb = sbb, a.sbt = sbt, a.sbg = sbg;
  a.Cm = Cm, a.scb = scb, a.sct = sct, a.scg = scg;
  a.A = A;
  a.D = D;
  a.dbias = delta_bias;
  a.h0 = state;
  a.cu = cu_seqlens;
  a.softplus = delta_softplus != 0;
  if ((rc = check_ssm_inputs(a, type)) != LTC_OK) return rc;
  if (a.ntok > 0 && !out) return host_fail(LTC_EINVAL, "out pointer is NULL");
  if (B > 0 && !state_final) return host_fail(LTC_EINVAL, "state_final pointer is NULL");
  if (save && a.ntok > 0 && !saved) return host_fail(LTC_EINVAL, "save set without a saved buffer");
  Pieces need{nullptr};
  carve_ssm(need, a, false);
  if ((rc = check_workspace(need.off, workspace, workspace_bytes)) != LTC_OK) return rc;
  Pieces c{static_cast<char*>(workspace)};
  carve_ssm(c, a, false);
  a.saved = save ? saved : nullptr;
  a.out = out;
  a.hf = state_final;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  return finish(host_timed(ltc::K_SSM_FWD, [&] { return ltc::launch_ssm_fwd(type, a, s); }),
                "selective scan launch");
}

int ltc_selective_scan_backward(const void* x, long long sxb, long long sxt, const void* delta, long long sdb,
                                long long sdt, const float* A, const void* Bm, long long sbb, long long sbt,
                                long long sbg, const void* Cm, long long scb, long long sct, long long scg,
                                const float* D, const void* z, long long szb, long long szt,
                                const float* delta_bias, const float* state, const int* cu_seqlens, int type,
                                int delta_softplus, int B, int T, int H, int N, int G, const float* saved,
                                const void* grad_out, long long sob, long long sot,
                                const float* grad_state_final, void* grad_x, void* grad_delta, float* grad_A,
                                void* grad_B, void* grad_C, float* grad_D, void* grad_z,
                                float* grad_delta_bias, float* grad_state, void* workspace,
                                long long workspace_bytes, void* stream) {
  host_clear_error();
  ltc::SsmArgs a{};
  int rc = ssm_args(&a, B, T, H, N, G, cu_seqlens != nullptr, true);
  if (rc != LTC_OK) return rc;
  a.x = x, a.sxb = sxb, a.sxt = sxt;
  a.d = delta, a.sdb = sdb, a.sdt = sdt;
  a.z = z, a.szb = szb, a.szt = szt;
  a.Bm = Bm, a.sbb = sbb, a.sbt = sbt, a.sbg = sbg;
  a.Cm = Cm, a.scb = scb, a.sct = sct, a.scg = scg;
  a.A = A;
  a.D = D;
  a.dbias = delta_bias;
  a.h0 = state;
  a.cu = cu_seqlens;
  a.softplus = delta_softplus != 0;
  if ((rc = check_ssm_inputs(a, type)) != LTC_OK) return rc;
  if (a.ntok > 0 && !saved) return host_fail(LTC_EINVAL, "saved pointer is NULL");
  if (grad_z && !z) return host_fail(LTC_EINVAL, "grad_z without z");
  Pieces need{nullptr};
  carve_ssm(need, a, true);
  if ((rc = check_workspace(need.off, workspace, workspace_bytes)) != LTC_OK) return rc;
  Pieces c{static_cast<char*>(workspace)};
  carve_ssm(c, a, true);
  if (!grad_B && !grad_C) a.part_bc = nullptr;
  if (!grad_A && !grad_D && !grad_delta_bias) a.part_a = a.part_h = nullptr;
  a.saved = const_cast<float*>(saved);
  a.go = grad_out, a.sob = sob, a.sot = sot;
  a.gh = grad_state_final;
  a.gx = grad_x;
  a.gd = grad_delta;
  a.gz = grad_z;
  a.gA = grad_A;
  a.gB = grad_B;
  a.gC = grad_C;
  a.gD = grad_D;
  a.gbias = grad_delta_bias;
  a.gs = grad_state;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  return finish(host_timed(ltc::K_SSM_BWD, [&] { return ltc::launch_ssm_bwd(type, a, s); }),
                "selective scan backward launch");
}

int ltc_selective_scan_step(const void* x, long long sx, const void* delta, long long sd, const float* A,
                            const void* Bm, long long sbb, long long sbg, const void* Cm, long long scb,
                            long long scg, const float* D, const void* z, long long sz, const float* delta_bias,
                            float* state, long long ssp, const int* slots, int type, int delta_softplus, int B,
                            int H, int N, int G, int P, void* out, void* stream) {
  host_clear_error();
  ltc::SsmArgs sizes{};
  int rc = ssm_args(&sizes, B, 1, H, N, G, 0, false);
  if (rc != LTC_OK) return rc;
  if (!known_type(type)) return host_fail(LTC_EINVAL, "type must be LTC_F32, LTC_BF16 or LTC_F16");
  if ((rc = check_step_rows(B, P, slots)) != LTC_OK) return rc;
  if (!A) return host_fail(LTC_EINVAL, "A pointer is NULL");
  if (P > 1 && ssp < (long long)H * N) return host_fail(LTC_EINVAL, "the rows of state overlap");
  if (B > 0 && (!x || !delta || !Bm || !Cm || !out))
    return host_fail(LTC_EINVAL, "x/delta/B/C/out pointer is NULL");
  if (B > 0 && P > 0 && !state) return host_fail(LTC_EINVAL, "state pointer is NULL");
  ltc::SsmStepArgs a{};
  a.x = x, a.sx = sx;
  a.d = delta, a.sd = sd;
  a.z = z, a.sz = sz;
  a.Bm = Bm, a.sbb = sbb, a.sbg = sbg;
  a.Cm = Cm, a.scb = scb, a.scg = scg;
  a.A = A;
  a.D = D;
  a.dbias = delta_bias;
  a.softplus = delta_softplus != 0;
  a.state = state;
  a.ssp = ssp;
  a.slots = slots;
  a.B = B, a.H = H, a.N = N, a.G = G, a.P = P;
  a.out = out;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  return finish(host_timed(ltc::K_SSM_STEP, [&] { return ltc::launch_ssm_step(type, a, s); }),
                "selective scan step launch");
}

int ltc_embed_forward(const void* table, long long st, const void* ids, int ids64, int type, long long n, int V,
                      int H, float scale, void* out, void* stream) {
  host_clear_error();
  int rc = check_embed(type, n, V, H);
  if (rc != LTC_OK) return rc;
  if (n > 0 && (!table || !ids || !out)) return host_fail(LTC_EINVAL, "table/ids/out pointer is NULL");
  ltc::EmbedArgs a{};
  a.table = table;
  a.st = st;
  a.ids = ids;
  a.id64 = ids64 != 0;
  a.n = n;
  a.V = V;
  a.H = H;
  a.scale = scale;
  a.out = out;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  return finish(host_timed(ltc::K_EMBED_FWD, [&] { return ltc::launch_embed_fwd(type, a, s); }),
                "embedding launch");
}

long long ltc_embed_bwd_workspace_bytes(long long n, int V, int H) {
  if (check_embed(LTC_F32, n, V, H) != LTC_OK) return -1;
  ltc::EmbedArgs a{};
  a.n = n;
  a.V = V;
  a.H = H;
  Pieces c{nullptr};
  carve_embed(c, a);
  return c.off;
}

int ltc_embed_backward(const void* ids, int ids64, int type, long long n, int V, int H, float scale,
                       const void* grad_out, long long so, void* grad_table, void* workspace,
                       long long workspace_bytes, void* stream) {
  host_clear_error();
  int rc = check_embed(type, n, V, H);
  if (rc != LTC_OK) return rc;
  if (n > 0 && (!ids || !grad_out)) return host_fail(LTC_EINVAL, "ids/grad_out pointer is NULL");
  if (!grad_table) return host_fail(LTC_EINVAL, "grad_table pointer is NULL");
  ltc::EmbedArgs a{};
  a.ids = ids;
  a.id64 = ids64 != 0;
  a.n = n;
  a.V = V;
  a.H = H;
  a.scale = scale;
  a.go = grad_out;
  a.sgo = so;
  a.gt = grad_table;
  Pieces need{nullptr};
  carve_embed(need, a);
  if ((rc = check_workspace(need.off, workspace, workspace_bytes)) != LTC_OK) return rc;
  Pieces c{static_cast<char*>(workspace)};
  carve_embed(c, a);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  return finish(host_timed(ltc::K_EMBED_BWD, [&] { return ltc::launch_embed_bwd(type, a, s); }),
                "embedding backward launch");
}

int ltc_adjust_logits(const void* logits, long long sl, const void* context, long long sc, int context64, int ctx,
                      const int* prompt_lens, const float* repetition, const float* frequency,
                      const float* presence, float repetition0, float frequency0, float presence0,
                      const void* bias_ids, long long sbi, int bias_ids64, const float* bias, long long sb, int K,
                      const int* mask, long long sm, int logits_type, long long R, int V, void* out,
                      void* stream) {
  host_clear_error();
  if (R < 0 || V < 1 || ctx < 0) return host_fail(LTC_EINVAL, "sizes must satisfy R >= 0, V >= 1, ctx >= 0");
  if (K < 0 || K > LTC_BIAS_MAX)
    return host_fail(LTC_EINVAL, "K must be between 0 and " + std::to_string(LTC_BIAS_MAX));
  if (!known_type(logits_type))
    return host_fail(LTC_EINVAL, "logits_type must be LTC_F32, LTC_BF16 or LTC_F16");
  if (!repetition && !(repetition0 > 0.f && repetition0 < __builtin_inff()))
    return host_fail(LTC_EINVAL, "repetition must be positive and finite");
  if ((!frequency && !__builtin_isfinite(frequency0)) || (!presence && !__builtin_isfinite(presence0)))
    return host_fail(LTC_EINVAL, "frequency and presence must be finite");
  if (V > INT_MAX - (1 << 16) || R > kMaxGroups / ((V + 8191LL) / 8192))
    return host_fail(LTC_EUNSUPPORTED, "problem too large");
  if (R > 0 && (!logits || !out)) return host_fail(LTC_EINVAL, "logits/out pointer is NULL");
  if (R > 0 && ctx > 0 && !context) return host_fail(LTC_EINVAL, "context pointer is NULL");
  if (R > 0 && K > 0 && (!bias_ids || !bias)) return host_fail(LTC_EINVAL, "bias_ids/bias pointer is NULL");
  ltc::AdjustArgs a{};
  a.logits = logits, a.sl = sl;
  a.R = R, a.V = V;
  a.context = context, a.sc = sc, a.ctx = ctx, a.ctx64 = context64 != 0;
  a.prompt = prompt_lens;
  a.rep = repetition, a.freq = frequency, a.pres = presence;
  a.rep0 = repetition0, a.freq0 = frequency0, a.pres0 = presence0;
  a.bias_ids = bias_ids, a.sbi = sbi, a.bias64 = bias_ids64 != 0;
  a.bias = bias, a.sb = sb, a.K = K;
  a.mask = mask, a.sm = sm;
  a.out = out;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  return finish(host_timed(ltc::K_ADJUST, [&] { return ltc::launch_adjust(logits_type, a, s); }),
                "logit adjustment launch");
}

}  // extern "C"
