// Parameter blocks and launchers of the operators around the KDA prefill (C entry points: kda_capi.cu).
#pragma once
#include "kda_seq.cuh"

namespace kda {

enum { TYPE_BF16 = 0, TYPE_FP16 = 1, TYPE_FP32 = 2 };

struct ConvParams {
  const void* x;
  const void* weight;      // [C][W]
  const void* bias;        // [C] or nullptr
  void* out;
  const void* src;         // history rows [slot][W - 1][C]; nullptr: zeros
  void* dst;               // may be src
  SeqTable seq;
  long long ldx, ldo, src_stride, dst_stride;
  int C, W, silu, weight_type, zero_pad;
  int tile;                // rows of a block, set by the launcher
};
cudaError_t launch_conv(ConvParams p, int type, cudaStream_t stream);
cudaError_t launch_conv_step(ConvParams p, int type, cudaStream_t stream);

struct ScanParams {
  const void *u, *dt, *B, *C, *z;
  void* out;
  const float *A, *D, *dt_bias;
  const float* src;        // states [slot][Dm][Ns]; nullptr: zeros
  float* dst;
  SeqTable seq;
  long long ldu, lddt, ldb, ldc, ldz, ldo, src_stride, dst_stride;
  int Dm, Ns, groups, softplus, zero_pad;
  int piece;               // tokens of a piece, 0: sequences are not cut
  float *ws_state, *ws_sum;    // [pieces][Dm][Ns], [pieces][Dm]
  int async;               // set by the launcher: rows on 16 bytes
};
long long sscan_piece(long long T, int N, int Dm, int Ns);
cudaError_t launch_sscan(const ScanParams& p, int type, cudaStream_t stream);
cudaError_t launch_sscan_step(const ScanParams& p, int type, cudaStream_t stream);

struct StepParams {
  const __nv_bfloat16 *q, *k, *v;
  const void *g, *beta;    // bf16 (raw) or fp32 (plain)
  __nv_bfloat16* out;
  const float *A_log, *dt_bias;
  float* pool;             // [slot][H][128][128]
  SeqTable seq;
  long long ldq, ldk, ldv, ldg, ldbeta, ldo, slot_stride;
  float scale, lower_bound;
  int H, raw, zero_pad;      // raw: state value first, plain: key first
};
cudaError_t launch_kda_step(const StepParams& p, cudaStream_t stream);

constexpr int GATED_SCAN_TILE = 48;      // a training pass keeps the states in front of every so many tokens
struct GatedScanParams {
  const void *x, *r, *i;   // [T][C]; i may be nullptr
  void* out;
  const float *rate, *r_bias, *i_bias;   // [C]; each may be nullptr, rate: the form without it
  const float* src;        // states [slot][C]; nullptr: zeros
  float* dst;              // may be src; nullptr: not stored
  float* tiles;            // [tiles of T][C]: the states in front of them; nullptr: not kept
  SeqTable seq;
  long long ldx, ldr, ldi, ldo, src_stride, dst_stride;
  float rate_scale;
  int C, zero_pad;
  int tile;                // step: rows of a block, set by the launcher
  int more_maps;           // diagnostic: 1 = blocks wait for a map that nobody sends
  unsigned long long wait_ns;            // bound of a wait for maps
};
cudaError_t launch_gated_scan(const GatedScanParams& p, int type, cudaStream_t stream);
cudaError_t launch_gated_scan_step(const GatedScanParams& p, int type, cudaStream_t stream);

struct GatedScanGradParams {
  const void *x, *r, *i, *dy;            // i and dy may be nullptr
  void *dx, *dr, *di;      // [T][C]; di with i
  const float *rate, *r_bias, *i_bias;
  const float* tiles;      // of the forward pass
  const float* src;        // its initial states [N][C]; nullptr: zeros
  const float* dfinal;     // [N][C]; nullptr: zeros
  float* dsrc;             // [N][C]; nullptr: not wanted
  float *drate, *dr_bias, *di_bias;      // [C]; each nullptr: not wanted
  SeqTable seq;            // without slots
  long long ldx, ldr, ldi, lddy, lddx, lddr, lddi;
  float rate_scale;
  int C;
  int more_maps;           // as above
  unsigned long long wait_ns;
};
cudaError_t launch_gated_scan_grad(const GatedScanGradParams& p, int type, cudaStream_t stream);

// Norm of each group of D channels of a token, with an activation: of the gate z, or of the normalised value.
struct GroupNormParams {
  const void *x, *z, *dy;  // [T][G D]; z may be nullptr; dy: gradients only
  void* out;               // y, or dx
  void* dz;                // gradients with z
  const float *weight, *bias;            // [G D], or [D] with `shared`; may be nullptr
  float *dweight, *dbias;  // their gradients' sums; nullptr: not wanted
  float* partial;          // gradients: the workspace
  long long T, ldx, ldz, lddy, ldo, lddz;
  float eps;
  int G, D, act, center, shared;         // act: ACT_*
  int lanes, parts;        // set by the launcher: threads of a group, blocks along the rows
};
enum { ACT_NONE = 0, ACT_SILU = 1, ACT_SIGMOID = 2 };
constexpr int GROUP_NORM_MAX_WIDTH = 16384;
cudaError_t launch_group_norm(const GroupNormParams& p, int type, cudaStream_t stream);
cudaError_t launch_group_norm_grad(const GroupNormParams& p, int type, cudaStream_t stream);
long long group_norm_partial_floats(long long T, int G, int D, int type, bool shared);

constexpr int POOLS_MAX = 8, TABLES_MAX = 8;
struct PoolRows {          // the pools that share one table of slots
  unsigned char* base[POOLS_MAX];
  long long stride[POOLS_MAX], bytes[POOLS_MAX];
  int n;
};
// Copies named by a table: plan -> `moves` (source, destination; source -1: zeros), then the bytes.
struct PoolPlan {
  unsigned char* used;     // [slots] truth values
  const void* src;         // copy: sources; fork: parents; free: slots
  const void* dst;         // copy: destinations
  int src_is64, dst_is64;
  long long n;             // entries
  int* slots_out;          // fork: the new slots
  int* remap;              // compact: [slots]
  void* tables[TABLES_MAX];
  long long table_n[TABLES_MAX];
  int table_is64[TABLES_MAX];
  int n_tables;
  int* moves;              // the workspace: [0] count, pairs from [4], a plan's own tables behind them
  int* status;
  long long P;
};
cudaError_t launch_pool_copy(const PoolPlan& p, const PoolRows& rows, cudaStream_t stream);
cudaError_t launch_pool_fork(const PoolPlan& p, const PoolRows& rows, cudaStream_t stream);
cudaError_t launch_pool_free(const PoolPlan& p, cudaStream_t stream);
cudaError_t launch_pool_compact(const PoolPlan& p, const PoolRows& rows, cudaStream_t stream);

}  // namespace kda
