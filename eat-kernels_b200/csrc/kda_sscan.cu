// Selective state space scan over packed sequences, per channel d with Ns state values n (states in fp32):
//   s = softplus(dt + dt_bias);  h[n] = exp(s A[d,n]) h[n] + s u B[n];  y = sum_n C[n] h[n] + D[d] u;  y *= silu(z)
//
// What bounds it: one exponential a token, channel and state value, 16 a clock and SM in the special-function unit, which is
// two to three times the time of the tokens' bytes.  So everything else is kept away from that unit and from the instruction
// stream of the warps that feed it:
//   * a block has four scan warps, one a scheduler, and four helper warps.  The helpers load the tokens, work out the step
//     sizes, s u, D u and the gate, and write the outputs; the scan warps only see shared memory.  Two stages of tokens
//     between them, handed over by named barriers.
//   * a channel's state lies over L lanes, S values each; the products run two values an instruction.  Sums over the lanes are
//     taken for L tokens at once, each step of the exchange halving the tokens a lane holds (L - 1 exchanges for L tokens).
#include "kda_serving.cuh"

namespace kda {

namespace {

constexpr int SCAN_LANES = 128;          // scan threads of a block, and as many helpers
constexpr int SCAN_THREADS = 2 * SCAN_LANES;
constexpr int TILE = 32;                 // tokens a stage
constexpr float LOG2E_F = 1.4426950408889634f;

// Polynomials by minimax (Remez exchange) of the relative error, coefficients rounded to fp32: 1.8e-7 off with the roundings.
__device__ __forceinline__ float log1p_unit(float e) {     // log(1 + e), e in [0, 1]
  float p = 0.0052326940931379795f;
  p = fmaf(p, e, -0.02950523979961872f);
  p = fmaf(p, e, 0.07822595536708832f);
  p = fmaf(p, e, -0.13663245737552643f);
  p = fmaf(p, e, 0.19106006622314453f);
  p = fmaf(p, e, -0.2484298199415207f);
  p = fmaf(p, e, 0.3331909775733948f);
  p = fmaf(p, e, -0.4999949336051941f);
  p = fmaf(p, e, 0.9999999403953552f);
  return p * e;
}
__device__ __forceinline__ float exp2_fast(float x) {      // 2 ulp; below 2^-126 zero
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// max(x, 0) + log(1 + exp(-|x|)); NaN stays
__device__ __forceinline__ float softplus(float x) {
  const float e = exp2_fast(-fabsf(x) * LOG2E_F);
  return x != x ? x : fmaxf(x, 0.0f) + log1p_unit(e);
}

// two fp32 values an instruction
using F2 = unsigned long long;
__device__ __forceinline__ F2 f2(float a, float b) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void split(F2 v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

__device__ __forceinline__ void bar_sync(int id) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(SCAN_THREADS) : "memory"); }
__device__ __forceinline__ void bar_arrive(int id) { asm volatile("bar.arrive %0, %1;" ::"r"(id), "r"(SCAN_THREADS) : "memory"); }
enum { BAR_FULL = 1, BAR_DONE = 3 };     // + stage

template <int S>
struct Values {
  float v[S];
};
// S consecutive values of shared memory, in one access
template <int S>
__device__ __forceinline__ Values<S> load_values(const float* p) {
  Values<S> r;
  if constexpr (S == 4) {
    const float4 f = *reinterpret_cast<const float4*>(p);
    r.v[0] = f.x; r.v[1] = f.y; r.v[2] = f.z; r.v[3] = f.w;
  } else if constexpr (S == 2) {
    const float2 f = *reinterpret_cast<const float2*>(p);
    r.v[0] = f.x; r.v[1] = f.y;
  } else {
    r.v[0] = *p;
  }
  return r;
}

template <int L, int S>
struct ScanShared {
  static constexpr int CB = SCAN_LANES / L;          // channels of a block
  static constexpr int NP = L * S;                   // state values, padded
  static constexpr int YS = CB + CB / 4;             // row of outputs: L rows of a warp's channels fall into different banks
  float2 step[2][TILE][CB];                          // s, s u
  float b[2][TILE][NP], c[2][TILE][NP];
  float y[2][TILE][YS];                              // D u, then the outputs without the gate
  float gate[2][TILE][CB];
};

struct Work {                                        // a block's share
  int group, d0, channels;                           // group of channels, first channel, how many
  long long begin, end;                              // tokens
};

// The helpers' half: tokens in, outputs out.
template <typename T, int L, int S>
__device__ __forceinline__ void help(const ScanParams& p, const Work& w, ScanShared<L, S>& sh, int tid) {
  using Sh = ScanShared<L, S>;
  constexpr int CB = Sh::CB, NP = Sh::NP, E = TILE * CB / SCAN_LANES, EB = TILE * NP / SCAN_LANES;
  constexpr int ROWS = SCAN_LANES / CB;              // tokens that the helpers cover at a time
  const int c = tid % CB, row = tid / CB;
  const bool mine = c < w.channels;
  const int d = w.d0 + (mine ? c : 0);
  const float skip = p.D != nullptr ? p.D[d] : 0.0f, bias = p.dt_bias != nullptr ? p.dt_bias[d] : 0.0f;
  const T* u = reinterpret_cast<const T*>(p.u) + d;
  const T* dt = reinterpret_cast<const T*>(p.dt) + d;
  const T* z = reinterpret_cast<const T*>(p.z) + d;
  const T* B = reinterpret_cast<const T*>(p.B) + (long long)w.group * p.Ns;
  const T* C = reinterpret_cast<const T*>(p.C) + (long long)w.group * p.Ns;
  T* out = reinterpret_cast<T*>(p.out) + d;
  const int n = tid % NP, brow = tid / NP;           // NP divides the helpers' number
  constexpr int BROWS = SCAN_LANES / NP;
  const bool has_z = p.z != nullptr, state_in = n < p.Ns;

  T ru[E], rdt[E], rz[E], rb[EB], rc[EB];
  const T none = from_float<T>(0.0f);
  auto load = [&](long long t0) {
#pragma unroll
    for (int e = 0; e < E; e++) {
      const long long t = t0 + row + e * ROWS;
      const bool on = mine && t < w.end;
      ru[e] = on ? u[t * p.ldu] : none;
      rdt[e] = on ? dt[t * p.lddt] : none;
      rz[e] = on && has_z ? z[t * p.ldz] : none;
    }
#pragma unroll
    for (int e = 0; e < EB; e++) {
      const long long t = t0 + brow + e * BROWS;
      const bool on = state_in && t < w.end;
      rb[e] = on ? B[t * p.ldb + n] : none;
      rc[e] = on ? C[t * p.ldc + n] : none;
    }
  };
  auto store = [&](long long t0, int stage) {
#pragma unroll
    for (int e = 0; e < E; e++) {
      const int j = row + e * ROWS;
      if (mine && t0 + j < w.end) out[(t0 + j) * p.ldo] = from_float<T>(sh.y[stage][j][c] * sh.gate[stage][j][c]);
    }
  };

  const long long tiles = (w.end - w.begin + TILE - 1) / TILE;
  load(w.begin);
  for (long long i = 0; i < tiles; i++) {
    const int stage = (int)(i & 1);
    const long long t0 = w.begin + i * TILE;
    if (i >= 2) {
      bar_sync(BAR_DONE + stage);
      store(t0 - 2 * TILE, stage);
    }
#pragma unroll
    for (int e = 0; e < E; e++) {
      const int j = row + e * ROWS;
      const float uf = to_float(ru[e]);
      float s = to_float(rdt[e]) + bias;
      if (p.softplus) s = softplus(s);
      if (t0 + j >= w.end) s = 0.0f;                 // leaves the state as it is
      sh.step[stage][j][c] = make_float2(s, s * uf);
      sh.y[stage][j][c] = skip * uf;
      sh.gate[stage][j][c] = has_z ? silu<T>(to_float(rz[e])) : 1.0f;
    }
#pragma unroll
    for (int e = 0; e < EB; e++) {
      sh.b[stage][brow + e * BROWS][n] = to_float(rb[e]);
      sh.c[stage][brow + e * BROWS][n] = to_float(rc[e]);
    }
    bar_arrive(BAR_FULL + stage);
    load(t0 + TILE);
  }
  for (long long i = tiles > 2 ? tiles - 2 : 0; i < tiles; i++) {
    bar_sync(BAR_DONE + (int)(i & 1));
    store(w.begin + i * TILE, (int)(i & 1));
  }
}

// The scan warps' half.
template <int L, int S>
__device__ __forceinline__ void scan(const Work& w, ScanShared<L, S>& sh, int tid, const float (&a)[S], float (&h)[S]) {
  const int lane = tid % L, c = tid / L;
  const long long tiles = (w.end - w.begin + TILE - 1) / TILE;
  for (long long i = 0; i < tiles; i++) {
    const int stage = (int)(i & 1);
    const int left = (int)min((long long)TILE, w.end - w.begin - i * TILE);
    bar_sync(BAR_FULL + stage);
    for (int j0 = 0; j0 < left; j0 += L) {
      float part[L];
#pragma unroll
      for (int j = 0; j < L; j++) {
        const float2 st = sh.step[stage][j0 + j][c];
        const Values<S> b = load_values<S>(&sh.b[stage][j0 + j][lane * S]), cc = load_values<S>(&sh.c[stage][j0 + j][lane * S]);
        if constexpr (S > 1) {
          F2 sum;
#pragma unroll
          for (int k = 0; k < S; k += 2) {
            float x0, x1;
            split(mul2(f2(st.x, st.x), f2(a[k], a[k + 1])), x0, x1);
            const F2 hn = fma2(f2(exp2_fast(x0), exp2_fast(x1)), f2(h[k], h[k + 1]), mul2(f2(st.y, st.y), f2(b.v[k], b.v[k + 1])));
            split(hn, h[k], h[k + 1]);
            sum = k == 0 ? mul2(f2(cc.v[0], cc.v[1]), hn) : fma2(f2(cc.v[k], cc.v[k + 1]), hn, sum);
          }
          float s0, s1;
          split(sum, s0, s1);
          part[j] = s0 + s1;
        } else {
          h[0] = fmaf(exp2_fast(st.x * a[0]), h[0], st.y * b.v[0]);
          part[j] = cc.v[0] * h[0];
        }
      }
      // lane l ends with the sum of token j0 + l
#pragma unroll
      for (int m = L / 2; m >= 1; m /= 2) {
#pragma unroll
        for (int k = 0; k < m; k++) {
          const bool up = lane & m;
          const float give = up ? part[k] : part[m + k], keep = up ? part[m + k] : part[k];
          part[k] = keep + __shfl_xor_sync(0xffffffffu, give, m);
        }
      }
      sh.y[stage][j0 + lane][c] += part[0];
    }
    bar_arrive(BAR_DONE + stage);
  }
}

// One sequence and up to CB channels of one group a block.
template <typename T, int L, int S>
__global__ void __launch_bounds__(SCAN_THREADS) kda_selective_scan_kernel(const ScanParams p) {
  using Sh = ScanShared<L, S>;
  constexpr int CB = Sh::CB;
  extern __shared__ __align__(16) unsigned char smem[];
  Sh& sh = *reinterpret_cast<Sh*>(smem);
  const int per = p.Dm / p.groups, gblocks = (per + CB - 1) / CB;
  const int seq = blockIdx.x / (gblocks * p.groups), block = blockIdx.x % (gblocks * p.groups);
  const int tid = threadIdx.x % SCAN_LANES;
  const bool helper = threadIdx.x >= SCAN_LANES;
  Work w;
  w.group = block / gblocks;
  w.d0 = w.group * per + block % gblocks * CB;
  w.channels = min(CB, (w.group + 1) * per - w.d0);
  const bool rejected = cu_rejected(p.seq);
  const long long slot = claim_slot(p.seq, seq);
  w.begin = rejected ? 0 : cu_at(p.seq, seq);
  w.end = rejected ? 0 : cu_at(p.seq, seq + 1);
  if (helper) {
    help<T, L, S>(p, w, sh, tid);
    // rows behind the last sequence
    if (seq == p.seq.N - 1 && (rejected || p.zero_pad) && tid % CB < w.channels)
      for (long long t = w.end + tid / CB; t < p.seq.T; t += L) reinterpret_cast<T*>(p.out)[t * p.ldo + w.d0 + tid % CB] = from_float<T>(0.0f);
    return;
  }
  const int lane = tid % L, c = tid / L;
  const bool mine = c < w.channels;
  const long long at = (long long)(w.d0 + (mine ? c : 0)) * p.Ns + lane * S;
  float a[S], h[S];
#pragma unroll
  for (int k = 0; k < S; k++) {
    const bool on = mine && lane * S + k < p.Ns;
    a[k] = on ? p.A[at + k] * LOG2E_F : 0.0f;
    if (a[k] < -3.0e38f) a[k] = -3.0e38f;            // -inf times a step of zero (behind the last token) would be NaN
    h[k] = on && p.src != nullptr && slot >= 0 ? p.src[slot * p.src_stride + at + k] : 0.0f;
  }
  scan<L, S>(w, sh, tid, a, h);
  if (p.dst == nullptr || slot < 0 || !mine) return;
#pragma unroll
  for (int k = 0; k < S; k++)
    if (lane * S + k < p.Ns) p.dst[slot * p.dst_stride + at + k] = h[k];
}

// One token a row: L lanes hold a channel's state, S values each.  Bound by memory: the state goes through once.
template <typename T, int L, int S>
__global__ void __launch_bounds__(SCAN_LANES) kda_selective_scan_step_kernel(const ScanParams p) {
  constexpr int CB = SCAN_LANES / L;
  const int cblocks = (p.Dm + CB - 1) / CB;
  const long long row = blockIdx.x / cblocks;
  const int lane = threadIdx.x % L, d = (int)(blockIdx.x % cblocks) * CB + threadIdx.x / L;
  const bool mine = d < p.Dm;
  const int dc = mine ? d : p.Dm - 1;
  const int group = dc / (p.Dm / p.groups);
  const long long slot = claim_row(p.seq, (int)row);
  T* out = reinterpret_cast<T*>(p.out) + row * p.ldo + dc;
  if (slot == -2) {
    if (p.zero_pad && lane == 0 && mine) *out = from_float<T>(0.0f);
    return;
  }
  const long long at = (long long)dc * p.Ns + lane * S;
  float h[S];
#pragma unroll
  for (int k = 0; k < S; k++) h[k] = lane * S + k < p.Ns && slot >= 0 ? p.src[slot * p.src_stride + at + k] : 0.0f;
  const T* B = reinterpret_cast<const T*>(p.B) + row * p.ldb + (long long)group * p.Ns + lane * S;
  const T* C = reinterpret_cast<const T*>(p.C) + row * p.ldc + (long long)group * p.Ns + lane * S;
  const float u = to_float(reinterpret_cast<const T*>(p.u)[row * p.ldu + dc]);
  float s = to_float(reinterpret_cast<const T*>(p.dt)[row * p.lddt + dc]) + (p.dt_bias != nullptr ? p.dt_bias[dc] : 0.0f);
  if (p.softplus) s = softplus(s);
  float y = 0.0f;
#pragma unroll
  for (int k = 0; k < S; k++)
    if (lane * S + k < p.Ns) {
      h[k] = fmaf(exp2_fast(s * p.A[at + k] * LOG2E_F), h[k], s * u * to_float(B[k]));
      y = fmaf(to_float(C[k]), h[k], y);
      if (slot >= 0 && mine) p.dst[slot * p.dst_stride + at + k] = h[k];
    }
#pragma unroll
  for (int m = 1; m < L; m *= 2) y += __shfl_xor_sync(0xffffffffu, y, m);
  if (lane == 0 && mine) {
    if (p.D != nullptr) y = fmaf(p.D[dc], u, y);
    if (p.z != nullptr) y *= silu<T>(to_float(reinterpret_cast<const T*>(p.z)[row * p.ldz + dc]));
    *out = from_float<T>(y);
  }
}

template <typename T, int L, int S>
cudaError_t launch_lanes(const ScanParams& p, bool step, cudaStream_t stream) {
  constexpr int CB = SCAN_LANES / L;
  const int per = p.Dm / p.groups;
  const long long blocks = step ? (long long)((p.Dm + CB - 1) / CB) * p.seq.N : (long long)((per + CB - 1) / CB) * p.groups * p.seq.N;
  if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
  if (blocks == 0) return cudaSuccess;
  if (step) {
    kda_selective_scan_step_kernel<T, L, S><<<(unsigned)blocks, SCAN_LANES, 0, stream>>>(p);
  } else {
    constexpr int bytes = sizeof(ScanShared<L, S>);
    if (bytes > 48 * 1024) {
      const cudaError_t e = cudaFuncSetAttribute(kda_selective_scan_kernel<T, L, S>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
      if (e != cudaSuccess) return e;
    }
    kda_selective_scan_kernel<T, L, S><<<(unsigned)blocks, SCAN_THREADS, bytes, stream>>>(p);
  }
  return cudaGetLastError();
}

template <typename T>
cudaError_t launch_type(const ScanParams& p, bool step, cudaStream_t stream) {
  if (p.Ns <= 4) return launch_lanes<T, 4, 1>(p, step, stream);
  if (p.Ns <= 8) return launch_lanes<T, 4, 2>(p, step, stream);
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
