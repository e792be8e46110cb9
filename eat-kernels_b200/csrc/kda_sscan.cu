// Selective state space scan over packed sequences, per channel d with Ns state values n (states in fp32):
//   s = softplus(dt + dt_bias);  h[n] = exp(s A[d,n]) h[n] + s u B[n];  y = sum_n C[n] h[n] + D[d] u;  y *= silu(z)
#include "kda_serving.cuh"

namespace kda {

namespace {

constexpr int SCAN_THREADS = 128;

__device__ __forceinline__ float softplus(float x) { return fmaxf(x, 0.0f) + log1pf(expf(-fabsf(x))); }

// L lanes hold a channel's state, S values each (values behind Ns stay zero); a block walks one sequence's tokens for
// SCAN_THREADS / L channels, a row of a step is a sequence of one token.
template <typename T, int L, int S, bool STEP>
__global__ void __launch_bounds__(SCAN_THREADS) kda_selective_scan_kernel(const ScanParams p) {
  constexpr int CB = SCAN_THREADS / L;
  const int cblocks = (p.Dm + CB - 1) / CB;
  const int seq = blockIdx.x / cblocks, lane = threadIdx.x % L;
  const int d = (int)(blockIdx.x % cblocks) * CB + threadIdx.x / L;
  const bool mine = d < p.Dm;
  const int dc = mine ? d : p.Dm - 1;
  const int group = dc / (p.Dm / p.groups);
  const bool rejected = !STEP && cu_rejected(p.seq);
  const long long slot = STEP ? claim_row(p.seq, seq) : claim_slot(p.seq, seq);
  long long begin = seq, end = seq + 1;
  if (!STEP) { begin = rejected ? 0 : cu_at(p.seq, seq); end = rejected ? 0 : cu_at(p.seq, seq + 1); }
  const T* u = reinterpret_cast<const T*>(p.u) + dc;
  const T* dt = reinterpret_cast<const T*>(p.dt) + dc;
  const T* z = reinterpret_cast<const T*>(p.z) + dc;
  const T* B = reinterpret_cast<const T*>(p.B) + (long long)group * p.Ns;
  const T* C = reinterpret_cast<const T*>(p.C) + (long long)group * p.Ns;
  T* out = reinterpret_cast<T*>(p.out) + dc;

  if (slot != -2) {
    float a[S], h[S];
    const long long at = (long long)dc * p.Ns + lane * S;
#pragma unroll
    for (int i = 0; i < S; i++) {
      const bool on = lane * S + i < p.Ns;
      a[i] = on ? p.A[at + i] * 1.4426950408889634f : 0.0f;
      h[i] = on && p.src != nullptr && slot >= 0 ? p.src[slot * p.src_stride + at + i] : 0.0f;
    }
    const float skip = p.D != nullptr ? p.D[dc] : 0.0f, bias = p.dt_bias != nullptr ? p.dt_bias[dc] : 0.0f;
    for (long long t = begin; t < end; t++) {
      const float ut = to_float(u[t * p.ldu]);
      float st = to_float(dt[t * p.lddt]) + bias;
      if (p.softplus) st = softplus(st);
      const float su = st * ut;
      float y = 0.0f;
#pragma unroll
      for (int i = 0; i < S; i++) {
        if (lane * S + i < p.Ns) {
          h[i] = fmaf(exp2f(st * a[i]), h[i], su * to_float(B[t * p.ldb + lane * S + i]));
          y = fmaf(to_float(C[t * p.ldc + lane * S + i]), h[i], y);
        }
      }
#pragma unroll
      for (int m = 1; m < L; m *= 2) y += __shfl_xor_sync(0xffffffffu, y, m);
      if (lane == 0 && mine) {
        y = fmaf(skip, ut, y);
        if (p.z != nullptr) y *= silu<T>(to_float(z[t * p.ldz]));
        out[t * p.ldo] = from_float<T>(y);
      }
    }
    if (p.dst != nullptr && slot >= 0 && mine)
#pragma unroll
      for (int i = 0; i < S; i++)
        if (lane * S + i < p.Ns) p.dst[slot * p.dst_stride + at + i] = h[i];
  }
  // rows that no sequence owns
  if (lane != 0 || !mine) return;
  if (STEP) {
    if (slot == -2 && p.zero_pad) out[begin * p.ldo] = from_float<T>(0.0f);
  } else if (seq == p.seq.N - 1 && (rejected || p.zero_pad)) {
    for (long long t = end; t < p.seq.T; t++) out[t * p.ldo] = from_float<T>(0.0f);
  }
}

template <typename T, int L, int S>
cudaError_t launch_lanes(const ScanParams& p, bool step, cudaStream_t stream) {
  const long long blocks = (long long)((p.Dm + SCAN_THREADS / L - 1) / (SCAN_THREADS / L)) * p.seq.N;
  if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
  if (blocks == 0) return cudaSuccess;
  if (step) kda_selective_scan_kernel<T, L, S, true><<<(unsigned)blocks, SCAN_THREADS, 0, stream>>>(p);
  else kda_selective_scan_kernel<T, L, S, false><<<(unsigned)blocks, SCAN_THREADS, 0, stream>>>(p);
  return cudaGetLastError();
}

template <typename T>
cudaError_t launch_type(const ScanParams& p, bool step, cudaStream_t stream) {
  if (p.Ns <= 16) return launch_lanes<T, 4, 4>(p, step, stream);
  if (p.Ns <= 32) return launch_lanes<T, 8, 4>(p, step, stream);
  if (p.Ns <= 64) return launch_lanes<T, 16, 4>(p, step, stream);
  return launch_lanes<T, 32, 4>(p, step, stream);
}

cudaError_t launch_any(const ScanParams& p, int type, bool step, cudaStream_t stream) {
  if (type == TYPE_BF16) return launch_type<__nv_bfloat16>(p, step, stream);
  if (type == TYPE_FP16) return launch_type<__half>(p, step, stream);
  return launch_type<float>(p, step, stream);
}

}  // namespace

cudaError_t launch_sscan(const ScanParams& p, int type, cudaStream_t stream) { return launch_any(p, type, false, stream); }
cudaError_t launch_sscan_step(const ScanParams& p, int type, cudaStream_t stream) { return launch_any(p, type, true, stream); }

}  // namespace kda
