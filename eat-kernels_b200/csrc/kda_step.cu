// One token of the KDA recurrence for each row of a decode batch, per head (K = V = 128, state fp32):
//   S' = S e^a (a: log-decay per key channel);  S = S' + k (beta (v - S'^T k));  o = scale S^T q
// With d1 = S'^T k, d2 = S'^T q and r = beta (v - d1) the output is scale (d2 + (q.k) r): both products run over the state as
// it is read, so every element is loaded and stored once.
#include "kda_common.cuh"
#include "kda_serving.cuh"

namespace kda {

namespace {

constexpr int STEP_THREADS = 128;
constexpr int STEP_ROWS = 32;            // value channels of a block: a quarter of a head's state, 16 KB

__device__ __forceinline__ float sigmoid_exact(float x) { return 1.0f / (1.0f + expf(-x)); }

// Value rows do not depend on one another, so a head is split over four blocks by value channels.  Value first (raw front-end): a warp
// holds 8 rows of 128 keys, 4 keys a lane, and sums over its lanes.  Key first (plain): 8 lanes hold 32 value columns, the
// 16 groups of lanes 8 keys each, and sum over shuffles and shared memory.  Bound by memory: 128 bytes a thread are in flight before the
// token's operands are needed and before the slots are looked through for repeats (48 rows of 64 heads: 70 us, 5.8 TB/s; with the
// look in front of the loads 80 us).
template <bool RAW>
__global__ void __launch_bounds__(STEP_THREADS) kda_step_kernel(const StepParams p) {
  constexpr bool KEY_FIRST = !RAW;
  __shared__ __align__(16) float s_k[D], s_q[D], s_a[D];
  __shared__ float s_v[STEP_ROWS], s_part[3][STEP_THREADS / 32], s_sum[2][STEP_THREADS / 32][STEP_ROWS];
  const int part = blockIdx.x % (D / STEP_ROWS), head = blockIdx.y;
  const int row = blockIdx.x / (D / STEP_ROWS);
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  int slot[1];
  row_slots(p.seq, row, 1, slot);
  __nv_bfloat16* out = p.out + row * p.ldo + head * D + part * STEP_ROWS;
  if (slot[0] == -2) {
    if (p.zero_pad && tid < STEP_ROWS) out[tid] = __float2bfloat16_rn(0.0f);
    return;
  }
  // the state's 16 KB: element i of a thread
  float* state = p.pool + (slot[0] < 0 ? 0 : slot[0]) * p.slot_stride + (long long)head * STATE_ELEMS;
  state += KEY_FIRST ? (warp * 4 + lane / 8) * D + part * STEP_ROWS + (lane % 8) * 4 : (part * STEP_ROWS + warp * 8) * D + lane * 4;
  constexpr int NEXT = KEY_FIRST ? 16 * D : D;
  float4 s[8];
  if (slot[0] >= 0) {
#pragma unroll
    for (int i = 0; i < 8; i++) s[i] = *reinterpret_cast<const float4*>(state + i * NEXT);
  }

  // the token's operands, one key channel a thread
  const long long hd = (long long)head * D + tid;
  float k = __bfloat162float(p.k[row * p.ldk + hd]), q = __bfloat162float(p.q[row * p.ldq + hd]), a, beta;
  if (RAW) {
    const float x = expf(p.A_log[head]) * (__bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p.g)[row * p.ldg + hd]) + p.dt_bias[hd]);
    a = expf(p.lower_bound * sigmoid_exact(x));
    beta = sigmoid_exact(__bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p.beta)[row * p.ldbeta + head]));
  } else {
    a = expf(reinterpret_cast<const float*>(p.g)[row * p.ldg + hd]);
    beta = reinterpret_cast<const float*>(p.beta)[row * p.ldbeta + head];
  }
  if (tid < STEP_ROWS) s_v[tid] = __bfloat162float(p.v[row * p.ldv + head * D + part * STEP_ROWS + tid]);
  float kk = k * k, qq = q * q, qk = q * k;
#pragma unroll
  for (int m = 16; m > 0; m /= 2) {
    kk += __shfl_xor_sync(0xffffffffu, kk, m);
    qq += __shfl_xor_sync(0xffffffffu, qq, m);
    qk += __shfl_xor_sync(0xffffffffu, qk, m);
  }
  if (lane == 0) { s_part[0][warp] = kk; s_part[1][warp] = qq; s_part[2][warp] = qk; }
  drop_repeats(p.seq, row, slot);
  if (slot[0] < 0) {
#pragma unroll
    for (int i = 0; i < 8; i++) s[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  }
  __syncthreads();
  qk = s_part[2][0] + s_part[2][1] + s_part[2][2] + s_part[2][3];
  if (RAW) {
    const float kn = 1.0f / fmaxf(sqrtf(s_part[0][0] + s_part[0][1] + s_part[0][2] + s_part[0][3]), 1e-6f);
    const float qn = 1.0f / fmaxf(sqrtf(s_part[1][0] + s_part[1][1] + s_part[1][2] + s_part[1][3]), 1e-6f);
    k *= kn; q *= qn; qk *= kn * qn;
  }
  s_k[tid] = k; s_q[tid] = q; s_a[tid] = a;
  __syncthreads();

  if constexpr (!KEY_FIRST) {
    const float4 fk = reinterpret_cast<const float4*>(s_k)[lane], fq = reinterpret_cast<const float4*>(s_q)[lane];
    const float4 fa = reinterpret_cast<const float4*>(s_a)[lane];
    float sums[16];                      // d1 of the 8 rows, d2 of the 8 rows
#pragma unroll
    for (int i = 0; i < 8; i++) {
      s[i].x *= fa.x; s[i].y *= fa.y; s[i].z *= fa.z; s[i].w *= fa.w;
      sums[i] = fmaf(s[i].x, fk.x, fmaf(s[i].y, fk.y, fmaf(s[i].z, fk.z, s[i].w * fk.w)));
      sums[8 + i] = fmaf(s[i].x, fq.x, fmaf(s[i].y, fq.y, fmaf(s[i].z, fq.z, s[i].w * fq.w)));
    }
    // sums over the lanes, halving the values that a lane holds: lane l ends with value l / 2
#pragma unroll
    for (int m = 16, n = 8; m >= 2; m /= 2, n /= 2) {
#pragma unroll
      for (int i = 0; i < n; i++) {
        const bool up = lane & m;
        const float give = up ? sums[i] : sums[n + i], keep = up ? sums[n + i] : sums[i];
        sums[i] = keep + __shfl_xor_sync(0xffffffffu, give, m);
      }
    }
    const float sum = sums[0] + __shfl_xor_sync(0xffffffffu, sums[0], 1);
    // lanes 0-15: d1 of row lane / 2, lanes 16-31: d2
    const int mine = (lane & 15) / 2;
    const float r = beta * (s_v[warp * 8 + mine] - __shfl_sync(0xffffffffu, sum, lane & 15));
    if (lane >= 16 && !(lane & 1)) out[warp * 8 + mine] = __float2bfloat16_rn(p.scale * fmaf(qk, r, sum));
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const float ri = __shfl_sync(0xffffffffu, r, 2 * i);
      s[i].x = fmaf(fk.x, ri, s[i].x); s[i].y = fmaf(fk.y, ri, s[i].y);
      s[i].z = fmaf(fk.z, ri, s[i].z); s[i].w = fmaf(fk.w, ri, s[i].w);
    }
  } else {
    const int key0 = warp * 4 + lane / 8, col = (lane % 8) * 4;
    float d1[4] = {}, d2[4] = {};
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const float fa = s_a[key0 + 16 * i], fk = s_k[key0 + 16 * i], fq = s_q[key0 + 16 * i];
      s[i].x *= fa; s[i].y *= fa; s[i].z *= fa; s[i].w *= fa;
      d1[0] = fmaf(s[i].x, fk, d1[0]); d1[1] = fmaf(s[i].y, fk, d1[1]); d1[2] = fmaf(s[i].z, fk, d1[2]); d1[3] = fmaf(s[i].w, fk, d1[3]);
      d2[0] = fmaf(s[i].x, fq, d2[0]); d2[1] = fmaf(s[i].y, fq, d2[1]); d2[2] = fmaf(s[i].z, fq, d2[2]); d2[3] = fmaf(s[i].w, fq, d2[3]);
    }
#pragma unroll
    for (int j = 0; j < 4; j++) {
#pragma unroll
      for (int m = 8; m <= 16; m *= 2) {
        d1[j] += __shfl_xor_sync(0xffffffffu, d1[j], m);
        d2[j] += __shfl_xor_sync(0xffffffffu, d2[j], m);
      }
      if (lane < 8) { s_sum[0][warp][col + j] = d1[j]; s_sum[1][warp][col + j] = d2[j]; }
    }
    __syncthreads();
    float r[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
      float a1 = 0.0f, a2 = 0.0f;
#pragma unroll
      for (int w = 0; w < STEP_THREADS / 32; w++) { a1 += s_sum[0][w][col + j]; a2 += s_sum[1][w][col + j]; }
      r[j] = beta * (s_v[col + j] - a1);
      if (tid < 8) out[col + j] = __float2bfloat16_rn(p.scale * fmaf(qk, r[j], a2));
    }
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const float fk = s_k[key0 + 16 * i];
      s[i].x = fmaf(fk, r[0], s[i].x); s[i].y = fmaf(fk, r[1], s[i].y); s[i].z = fmaf(fk, r[2], s[i].z); s[i].w = fmaf(fk, r[3], s[i].w);
    }
  }
  if (slot[0] < 0) return;
#pragma unroll
  for (int i = 0; i < 8; i++) *reinterpret_cast<float4*>(state + i * NEXT) = s[i];
}

}  // namespace

cudaError_t launch_kda_step(const StepParams& p, cudaStream_t stream) {
  const long long blocks = p.seq.T * (D / STEP_ROWS);
  if (blocks > 0x7fffffffLL || p.H > 65535) return cudaErrorInvalidValue;
  if (blocks == 0) return cudaSuccess;
  const dim3 grid((unsigned)blocks, (unsigned)p.H);
  if (p.raw) kda_step_kernel<true><<<grid, STEP_THREADS, 0, stream>>>(p);
  else kda_step_kernel<false><<<grid, STEP_THREADS, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace kda
