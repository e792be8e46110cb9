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
