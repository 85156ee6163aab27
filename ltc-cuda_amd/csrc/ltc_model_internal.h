// Internal interface of the token model's operators: entry points in
// ltc_model_capi.hip, kernels in ltc_conv_device.hip (causal convolution),
// ltc_ssm_device.hip (selective scan) and ltc_vocab_device.hip (embedding and
// adjustments of logits).
#pragma once

#include <hip/hip_runtime.h>

#include "ltc_seq_internal.h"

namespace ltc {

// ---------------------------------------------------------------------------
// Causal convolution
// ---------------------------------------------------------------------------
constexpr int kConvTapsMax = 8;
constexpr int kConvThreads = 256;

struct ConvArgs {
  const void* x;
  long long sxb, sxt;   // element strides of sequences and steps
  const void* w;        // (C,K)
  const void* bias;     // (C) or null
  const void* state;    // (B,K-1,C) or null for zero
  const int* cu;        // packed: boundaries (B+1); else null
  int w_f32;            // weights are fp32, whatever x is
  int silu;
  int B, T, C;          // sequences, tokens of each (packed: of all), channels
  long long N;          // tokens in all
  int lanes, run;       // lanes of a row, tokens of a thread
  int cblocks;          // blocks of channels
  long long tiles;      // tiles of tokens
  void* out;            // (N,C)
  void* hf;             // (B,K-1,C)
  // backward
  const void* go;       // or null for zero
  long long sob, sot;
  const void* gh;       // (B,K-1,C) or null for zero
  void* gx;             // (N,C) or null where not wanted
  void* gw;             // (C,K) or null
  void* gb;             // (C) or null
  void* gs;             // (B,K-1,C) or null
  float* part;          // [tiles][K+1][C]: sums of the weights' and the bias's gradients
};

// The tiles of a call: fills in lanes, run, cblocks and tiles.
void conv_tiles(int x_type, bool bwd, ConvArgs* a);
hipError_t launch_conv_fwd(int x_type, int K, const ConvArgs& a, hipStream_t s);
hipError_t launch_conv_bwd(int x_type, int K, const ConvArgs& a, hipStream_t s);

struct ConvStepArgs {
  const void* x;
  long long sxb;
  const void* w;
  const void* bias;
  int w_f32, silu;
  void* state;          // (P,K-1,C), strides ssp, sst, 1
  long long ssp, sst;
  const int* slots;     // null: row b's state is row b
  int B, C, P;
  void* out;            // (B,C)
};
hipError_t launch_conv_step(int x_type, int K, const ConvStepArgs& a, hipStream_t s);

// ---------------------------------------------------------------------------
// Selective scan
// ---------------------------------------------------------------------------
constexpr int kSsmStatesMax = 64;
constexpr int kSsmTokens = 16;  // of a batch; a state is saved before every batch
constexpr int kSsmBwdStates = 2;  // of a wave
constexpr int kSsmWavesMax = 8;

struct SsmArgs {
  const void *x, *d, *z;  // z may be null
  long long sxb, sxt, sdb, sdt, szb, szt;  // element strides of sequences and steps
  const void *Bm, *Cm;    // (B,T,G,N)
  long long sbb, sbt, sbg, scb, sct, scg;
  const float* A;         // (H,N)
  const float *D, *dbias; // (H) or null
  const float* h0;        // (B,H,N) or null for zero
  const int* cu;          // packed: boundaries (B+1); else null
  int softplus;
  int B, T, H, N, G;      // sequences, tokens of each (packed: of all), channels, states, groups
  long long ntok;         // tokens in all
  // plan
  int hblocks;            // blocks of 64 channels in a group
  int len, chunks;        // tokens of a chunk; chunks of a sequence (packed: of all tokens)
  long long lines;        // sequences that are cut into chunks each (packed: 1)
  // workspace
  float* ends;            // [lines*chunks][H][N]: what leaves a chunk, then what enters it
  float* sumd;            // [lines*chunks][H]: sums of the step sizes
  int* drops;             // [lines*chunks]: whether what enters is lost in the chunk
  float* part_bc;         // [hblocks][G][pairs of states][ntok][4]: of B, then C
  float* part_a;          // [lines*chunks][H][N]
  float* part_h;          // [lines*chunks][2][H]: of D and of the bias
  long long tiles;        // batches of a line
  float* saved;           // [lines][tiles][H][N], or null
  void* out;              // (ntok,H)
  float* hf;              // (B,H,N)
  // backward
  const void* go;         // or null for zero
  long long sob, sot;
  const float* gh;        // (B,H,N) or null for zero
  void *gx, *gd, *gz;     // (ntok,H)
  float *gA, *gD, *gbias; // or null where not wanted
  void *gB, *gC;          // (ntok,G,N) or null
  float* gs;              // (B,H,N) or null
};

// The plan of a call from its sizes: fills in hblocks to lines, and tiles.
void ssm_plan(SsmArgs* a, bool packed, bool bwd);
hipError_t launch_ssm_fwd(int type, const SsmArgs& a, hipStream_t s);
hipError_t launch_ssm_bwd(int type, const SsmArgs& a, hipStream_t s);

struct SsmStepArgs {
  const void *x, *d, *z;
  long long sx, sd, sz;   // row strides
  const void *Bm, *Cm;
  long long sbb, sbg, scb, scg;
  const float* A;
  const float *D, *dbias;
  int softplus;
  float* state;           // (P,H,N), strides ssp, N, 1
  long long ssp;
  const int* slots;       // null: row b's state is row b
  int B, H, N, G, P;
  void* out;              // (B,H)
};
hipError_t launch_ssm_step(int type, const SsmStepArgs& a, hipStream_t s);

// ---------------------------------------------------------------------------
// Embedding
// ---------------------------------------------------------------------------
constexpr int kSortThreads = 1024;
constexpr int kSortTile = kSortThreads;      // ids of a workgroup
constexpr int kSortBitsMax = 10;             // of one pass
// Tiles up to which a workgroup adds up the other tiles' counts itself.
constexpr int kSortTilesDirect = 64;
constexpr int kEmbedPiece = 32;              // sorted ids that are summed together

struct EmbedArgs {
  const void* table;  // (V,H), row stride st
  long long st;
  const void* ids;    // (n)
  int id64;
  long long n;
  int V, H;
  float scale;
  void* out;          // (n,H)
  // backward
  const void* go;     // (n,H), row stride sgo
  long long sgo;
  void* gt;           // (V,H)
  // workspace: ids and places as sorted so far, two of each; counts of each tile's
  // digits; where each id's run begins and ends; sums of pieces
  int* key[2];
  int* pos[2];
  unsigned* counts;   // [tiles + 1][1 << bits]: of each tile, and of all
  int* begin;         // (V), -1 for an id that does not occur
  int* end;           // (V)
  float* sums;        // [pieces][H]
  int bits, passes;   // of a digit; digits
  int tiles;
};
// The digits of V ids and one more: fills in bits and passes.
void embed_digits(EmbedArgs* a);
hipError_t launch_embed_fwd(int type, const EmbedArgs& a, hipStream_t s);
hipError_t launch_embed_bwd(int type, const EmbedArgs& a, hipStream_t s);

// ---------------------------------------------------------------------------
// Adjustments of logits
// ---------------------------------------------------------------------------
constexpr int kBiasMax = 1024;

struct AdjustArgs {
  const void* logits;  // (R,V), row stride sl
  long long sl;
  long long R;
  int V;
  const void* context;  // (R,ctx), row stride sc; or null
  long long sc;
  int ctx, ctx64;
  const int* prompt;    // (R) or null
  const float *rep, *freq, *pres;  // (R), or null for the values below
  float rep0, freq0, pres0;
  const void* bias_ids;  // (R,K), row stride sbi
  long long sbi;
  const float* bias;     // (R,K), row stride sb
  long long sb;
  int K, bias64;
  const int* mask;       // (R,words), row stride sm; or null
  long long sm;
  void* out;             // (R,V)
  int seg;               // logits of a workgroup
  int segs;              // workgroups of a row
};
hipError_t launch_adjust(int type, AdjustArgs a, hipStream_t s);

}  // namespace ltc
