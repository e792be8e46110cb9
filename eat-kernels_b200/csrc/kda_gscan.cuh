// What the passes of the gated linear recurrence share.  Per channel, with s = sigmoid(r + r_bias), g = sigmoid(i + i_bias) (1 without i):
//   rate given:  l = -c softplus(rate) s, f = exp(l), gain = sqrt(1 - f^2);      without:  f = s, gain = 1 - s
//   h[t] = f[t] h[t-1] + gain[t] g[t] x[t],  y = h
//
// Time is cut without regard to the sequences of the batch: a warp has a slice of S consecutive tokens for 32 lanes of channels, a block
// the slices of its warps (a tile), the blocks of a cluster one tile each behind one another (a round), and the cluster goes over the
// batch round by round.  A slice is summed up by a map h -> F h + U (F: product of its decays); a sequence that starts inside it makes
// that map the constant U, which a flag says (0 times an infinite state in front would be NaN).  The maps of a block meet in
// shared memory, those of a cluster in the shared memory of all its blocks, one barrier a round each, always in the same order: results do
// not depend on timing, nothing is kept in memory between blocks, and ragged batches cost what their tokens cost.
#pragma once
#include "kda_serving.cuh"

namespace kda {

namespace gscan {

constexpr int WARPS = 8, THREADS = WARPS * 32;
constexpr int S = 8;                     // tokens of a slice
constexpr int TILE = WARPS * S;
constexpr int MAX_CLUSTER = 8;
constexpr long long NEVER = 0x7fffffffffffffffLL;
static_assert(TILE == GATED_SCAN_TILE, "the states that a training pass keeps are those in front of the tiles");

// A product of decays that underflows to zero is taken as the smallest positive number, so that an infinite state stays infinite, as it
// does token by token (a finite one is not changed by that).  Where a decay is NaN, so is the map's constant.
constexpr float LEAST = 1.4e-45f;
constexpr float LOG2E_F = 1.4426950408889634f, LN2_F = 0.6931471805599453f;

__device__ __forceinline__ float rsqrt_fast(float x) {
  float y;
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// a bias as sigmoid_pair takes it
template <typename T>
__device__ __forceinline__ float bias_of(const float* p, int c) {
  const float b = p != nullptr ? p[c] : 0.0f;
  return sizeof(T) == 4 ? b : -LOG2E_F * b;
}

// -(e^y - 1) for y = 2 ln2 l <= 0, e = 2^l given: near zero by a polynomial for (e^y - 1) / y on [-1/2, 0] (relative minimax, found by
// linear programming: 1.0e-7 off in fp32), which 1 - e e would lose its digits for
__device__ __forceinline__ float one_minus_square(float l, float e) {
  const float y = l * (2.0f * LN2_F);
  float q = fmaf(y, 0.006771687883883715f, 0.0410030297935009f);
  q = fmaf(y, q, 0.1665491908788681f);
  q = fmaf(y, q, 0.4999926686286926f);
  q = fmaf(y, q, 0.9999999403953552f);
  return y > -0.5f ? -y * q : fmaf(-e, e, 1.0f);
}

// softplus in full precision, once a channel
__device__ __forceinline__ float softplus_exact(float x) { return fmaxf(x, 0.0f) + log1pf(expf(-fabsf(x))); }

// The decay's factor in front of s: -c softplus(rate), for 16-bit tokens in powers of two; finite, since an infinite one times s = 0 would
// be NaN.
template <typename T>
__device__ __forceinline__ float decay_factor(const float* rate, int c, float scale) {
  const float k = -scale * softplus_exact(rate[c]) * (sizeof(T) == 4 ? 1.0f : LOG2E_F);
  return k < -3.0e38f ? -3.0e38f : k;
}

// A token's values of one channel.  `l` (POWER) is log f, natural for 32-bit tokens, else base 2; s, n: of the decay's gate; inv: 1 / gain.
struct Gates {
  float f, gain, s, n, l, inv;
};
template <typename T, bool POWER>
__device__ __forceinline__ Gates decay(float r, float bias, float k) {
  Gates a;
  sigmoid_pair<T>(r, bias, a.s, a.n);
  if constexpr (!POWER) {
    a.f = a.s; a.gain = a.n; a.l = a.inv = 0.0f;
  } else {
    a.l = k * a.s;
    if constexpr (sizeof(T) == 4) {
      a.f = expf(a.l);
      a.gain = sqrtf(-expm1f(2.0f * a.l));
      a.inv = 1.0f / fmaxf(a.gain, 1.0e-19f);
    } else {
      a.f = ex2_fast(a.l);
      const float q = one_minus_square(a.l, a.f);
      a.inv = rsqrt_fast(fmaxf(q, 1.0e-38f));          // l times it is 0 where l is
      a.gain = q * a.inv;
    }
  }
  return a;
}

// ---- sequences
// Called by a warp: the first entry from j on that is >= t (N + 1: none)
__device__ __forceinline__ int seek(const SeqTable& s, int j, long long t) {
  const int lane = threadIdx.x % 32;
  for (; j <= s.N; j += 32) {
    const unsigned at = __ballot_sync(0xffffffffu, j + lane > s.N || cu_at(s, j + lane) >= t);
    if (at != 0) return min(j + __ffs(at) - 1, s.N + 1);
  }
  return s.N + 1;
}

// Called by a warp: the slot of sequence i, or -1 where its entry is out of range or repeats an earlier one
__device__ __forceinline__ long long claim(const SeqTable& s, int i) {
  if (s.slots == nullptr) return i;
  const long long d = table_at(s.slots, s.slots_is64, i);
  int bad = d < 0 || d >= s.n_slots;
  for (int j = threadIdx.x % 32; j < i && !bad; j += 32)
    if (table_at(s.slots, s.slots_is64, j) == d) bad = 1;
  if (!__any_sync(0xffffffffu, bad)) return d;
  if (threadIdx.x % 32 == 0) report(s.status, SEQ_BAD_SLOT);
  return -1;
}

// ---- clusters
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ void put_remote(void* own, uint32_t rank, float v) {        // at the address of `own` in another block
  const uint32_t a = static_cast<uint32_t>(__cvta_generic_to_shared(own));
  asm volatile("{\n .reg .b32 t;\n mapa.shared::cluster.u32 t, %0, %1;\n st.shared::cluster.f32 [t], %2;\n}" ::"r"(a), "r"(rank), "f"(v) : "memory");
}
__device__ __forceinline__ void put_remote(uint32_t* own, uint32_t rank, uint32_t v) {
  const uint32_t a = static_cast<uint32_t>(__cvta_generic_to_shared(own));
  asm volatile("{\n .reg .b32 t;\n mapa.shared::cluster.u32 t, %0, %1;\n st.shared::cluster.u32 [t], %2;\n}" ::"r"(a), "r"(rank), "r"(v) : "memory");
}

// ---- tokens
// Channels of a lane: two 16-bit ones in an access of 4 bytes, or one
template <typename T, bool WIDE>
constexpr int CHANNELS = WIDE ? 4 / (int)sizeof(T) : 1;

// The rows of a slice, as they lie in memory, for one tensor: asked for a round ahead
template <typename T, int V>
struct Rows {
  Pack<T, V> v[S];
  __device__ __forceinline__ void ask(const void* base, long long ld, long long t0, int n, int c, bool mine) {
    const T* p = reinterpret_cast<const T*>(base) + c + t0 * ld;
#pragma unroll
    for (int s = 0; s < S; s++) {
      if (mine && s < n) v[s] = *reinterpret_cast<const Pack<T, V>*>(p + s * ld);
      else
#pragma unroll
        for (int k = 0; k < V; k++) v[s].v[k] = from_float<T>(0.0f);
    }
  }
};

__device__ __forceinline__ int count(long long t0, long long end) {        // tokens of the slice at t0
  const long long n = end - t0;
  return n < 0 ? 0 : (n > S ? S : (int)n);
}

// Rows [end, T) of an output are zeros, spread over the blocks of a cluster
template <typename T, int V>
__device__ __forceinline__ void zero_rest(void* out, long long ld, long long end, long long T_, int c, bool mine, uint32_t rank, uint32_t size) {
  Pack<T, V> zero;
#pragma unroll
  for (int k = 0; k < V; k++) zero.v[k] = from_float<T>(0.0f);
  if (mine)
    for (long long t = end + rank * WARPS + threadIdx.x / 32; t < T_; t += size * WARPS)
      *reinterpret_cast<Pack<T, V>*>(reinterpret_cast<T*>(out) + c + t * ld) = zero;
}

// Blocks along time: as many as give the card two blocks an SM, no more than the batch has tiles
inline int cluster_of(long long slabs, long long T) {
  int size = 1;
  while (size < MAX_CLUSTER && slabs * size < 2 * 148 && (long long)size * TILE < T) size *= 2;
  return size;
}

template <typename K, typename P>
cudaError_t launch_clusters(K kernel, const P& p, long long slabs, int size, cudaStream_t stream) {
  if (slabs * size > 0x7fffffffLL) return cudaErrorInvalidValue;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(slabs * size));
  cfg.blockDim = dim3(THREADS);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)size;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p);
  return e != cudaSuccess ? e : cudaGetLastError();
}

// Whether every row of a tensor starts on a multiple of `bytes`
inline bool rows_on(const void* p, long long ld, int size, int bytes) {
  return ((reinterpret_cast<uintptr_t>(p) | (uintptr_t)(ld * size)) & (uintptr_t)(bytes - 1)) == 0;
}

}  // namespace gscan

}  // namespace kda
