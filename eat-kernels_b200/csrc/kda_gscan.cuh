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
constexpr int MAX_CLUSTER = 8;
constexpr long long NEVER = 0x7fffffffffffffffLL;

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

// softplus in full precision, once a channel
__device__ __forceinline__ float softplus_exact(float x) { return fmaxf(x, 0.0f) + log1pf(expf(-fabsf(x))); }

// The decay's factor in front of s: -c softplus(rate), for 16-bit tokens in powers of two; finite, since an infinite one times s = 0 would
// be NaN.
template <typename T>
__device__ __forceinline__ float decay_factor(const float* rate, int c, float scale) {
  const float k = -scale * softplus_exact(rate[c]) * (sizeof(T) == 4 ? 1.0f : LOG2E_F);
  return k < -3.0e38f ? -3.0e38f : k;
}

// ---- sequences
// Called by a warp: the first of the entries [lo, hi) that is >= t, hi where none is.  32 entries are looked at at a time.
__device__ __forceinline__ int lower(const SeqTable& s, int lo, int hi, long long t) {
  const int lane = threadIdx.x % 32;
  while (lo < hi) {
    const int part = (hi - lo + 31) / 32;
    const long long at = (long long)lo + (long long)(lane + 1) * part - 1;
    const unsigned found = __ballot_sync(0xffffffffu, cu_at(s, at < hi ? at : hi - 1) >= t);
    if (found == 0) return hi;
    const int first = __ffs(found) - 1;
    hi = min(hi - 1, lo + (first + 1) * part - 1);
    lo = lo + first * part;
  }
  return lo;
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
// at the address of `own` in another block
__device__ __forceinline__ void put_remote(const void* own, uint32_t rank, float4 v) {
  const uint32_t a = static_cast<uint32_t>(__cvta_generic_to_shared(own));
  asm volatile("{\n .reg .b32 t;\n mapa.shared::cluster.u32 t, %0, %1;\n st.shared::cluster.v4.f32 [t], {%2, %3, %4, %5};\n}" ::"r"(a), "r"(rank), "f"(v.x),
               "f"(v.y), "f"(v.z), "f"(v.w) : "memory");
}
__device__ __forceinline__ void put_remote(const void* own, uint32_t rank, float v) {
  const uint32_t a = static_cast<uint32_t>(__cvta_generic_to_shared(own));
  asm volatile("{\n .reg .b32 t;\n mapa.shared::cluster.u32 t, %0, %1;\n st.shared::cluster.f32 [t], %2;\n}" ::"r"(a), "r"(rank), "f"(v) : "memory");
}
__device__ __forceinline__ void put_remote(const void* own, uint32_t rank, uint32_t v) {
  const uint32_t a = static_cast<uint32_t>(__cvta_generic_to_shared(own));
  asm volatile("{\n .reg .b32 t;\n mapa.shared::cluster.u32 t, %0, %1;\n st.shared::cluster.u32 [t], %2;\n}" ::"r"(a), "r"(rank), "r"(v) : "memory");
}

// ---- one or two channels at once (two: one instruction)
template <int V>
struct Vec {
  float v[V];
};
template <int V>
__device__ __forceinline__ Vec<V> vec(float a) {
  Vec<V> r;
#pragma unroll
  for (int k = 0; k < V; k++) r.v[k] = a;
  return r;
}
__device__ __forceinline__ Vec<1> fma(Vec<1> a, Vec<1> b, Vec<1> c) { return {fmaf(a.v[0], b.v[0], c.v[0])}; }
__device__ __forceinline__ Vec<1> mul(Vec<1> a, Vec<1> b) { return {a.v[0] * b.v[0]}; }
__device__ __forceinline__ Vec<1> add(Vec<1> a, Vec<1> b) { return {a.v[0] + b.v[0]}; }
__device__ __forceinline__ Vec<2> fma(Vec<2> a, Vec<2> b, Vec<2> c) {
  Vec<2> d;
  asm("{\n .reg .b64 ra, rb, rc, rd;\n mov.b64 ra, {%2,%3};\n mov.b64 rb, {%4,%5};\n mov.b64 rc, {%6,%7};\n fma.rn.f32x2 rd, ra, rb, rc;\n mov.b64 {%0,%1}, rd;\n}"
      : "=f"(d.v[0]), "=f"(d.v[1]) : "f"(a.v[0]), "f"(a.v[1]), "f"(b.v[0]), "f"(b.v[1]), "f"(c.v[0]), "f"(c.v[1]));
  return d;
}
__device__ __forceinline__ Vec<2> mul(Vec<2> a, Vec<2> b) {
  Vec<2> d;
  asm("{\n .reg .b64 ra, rb, rd;\n mov.b64 ra, {%2,%3};\n mov.b64 rb, {%4,%5};\n mul.rn.f32x2 rd, ra, rb;\n mov.b64 {%0,%1}, rd;\n}"
      : "=f"(d.v[0]), "=f"(d.v[1]) : "f"(a.v[0]), "f"(a.v[1]), "f"(b.v[0]), "f"(b.v[1]));
  return d;
}
__device__ __forceinline__ Vec<2> add(Vec<2> a, Vec<2> b) {
  Vec<2> d;
  asm("{\n .reg .b64 ra, rb, rd;\n mov.b64 ra, {%2,%3};\n mov.b64 rb, {%4,%5};\n add.rn.f32x2 rd, ra, rb;\n mov.b64 {%0,%1}, rd;\n}"
      : "=f"(d.v[0]), "=f"(d.v[1]) : "f"(a.v[0]), "f"(a.v[1]), "f"(b.v[0]), "f"(b.v[1]));
  return d;
}
template <int V>
__device__ __forceinline__ Vec<V> least(Vec<V> a) {        // at least LEAST
#pragma unroll
  for (int k = 0; k < V; k++) a.v[k] = fmaxf(a.v[k], LEAST);
  return a;
}
template <int V>
__device__ __forceinline__ Vec<V> pick(bool first, Vec<V> a, Vec<V> b) {
#pragma unroll
  for (int k = 0; k < V; k++) a.v[k] = first ? a.v[k] : b.v[k];
  return a;
}

// ---- tokens
// Channels of a lane: two 16-bit ones where rows start on 16 bytes, else one
template <typename T, bool ASYNC>
constexpr int CHANNELS = ASYNC ? 4 / (int)sizeof(T) : 1;

template <int S>
__device__ __forceinline__ int count(long long t0, long long end) {        // tokens of the slice at t0
  const long long n = end - t0;
  return n < 0 ? 0 : (n > S ? S : (int)n);
}

// A warp's slice of one tensor.  ASYNC: S rows of 128 bytes in shared memory, by copies of 16 bytes that are asked for rounds ahead;
// places behind the last token or channel are zeros.  Otherwise S registers, asked for a round ahead.
template <typename T, int S>
struct Slice {
  Pack<T, 4 / sizeof(T)> row[S][32];

  __device__ __forceinline__ void ask(const void* base, long long ld, long long t0, int n, int c0, int C) {
    const int lane = threadIdx.x % 32, chunk = lane % 8;
    const int c = c0 + chunk * (16 / (int)sizeof(T));
    const uint32_t to = static_cast<uint32_t>(__cvta_generic_to_shared(this)) + (uint32_t)(lane / 8 * 128 + chunk * 16);
    const T* from = reinterpret_cast<const T*>(base) + (t0 + lane / 8) * ld + c;
#pragma unroll
    for (int q = 0; q < S / 4; q++) {
      const bool on = c < C && lane / 8 + 4 * q < n;
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + 512u * q), "l"(on ? (const void*)from : base), "r"(on ? 16 : 0) : "memory");
      from += 4 * ld;
    }
  }
  // the first n rows to memory; the warp has written them
  __device__ __forceinline__ void store(void* base, long long ld, long long t0, int n, int c0, int C) const {
    const int lane = threadIdx.x % 32, chunk = lane % 8;
    const int c = c0 + chunk * (16 / (int)sizeof(T));
    T* to = reinterpret_cast<T*>(base) + (t0 + lane / 8) * ld + c;
#pragma unroll
    for (int q = 0; q < S / 4; q++) {
      if (c < C && lane / 8 + 4 * q < n) *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(this) + lane / 8 * 128 + chunk * 16 + 512 * q);
      to += 4 * ld;
    }
  }
};
template <typename T, int S>
struct Registers {
  T row[S];
  __device__ __forceinline__ void ask(const void* base, long long ld, long long t0, int n, int c, int C) {
    const T* from = reinterpret_cast<const T*>(base) + t0 * ld + c;
    if (c < C && n == S) {
#pragma unroll
      for (int s = 0; s < S; s++) {
        row[s] = *from;
        from += ld;
      }
    } else {
#pragma unroll
      for (int s = 0; s < S; s++) {
        row[s] = from_float<T>(0.0f);
        if (c < C && s < n) row[s] = *from;
        from += ld;
      }
    }
  }
};
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

template <typename T, int V>
__device__ __forceinline__ Vec<V> values(const Pack<T, V>& p) {
  Vec<V> r;
#pragma unroll
  for (int k = 0; k < V; k++) r.v[k] = to_float(p.v[k]);
  return r;
}

// Of V channels: sigmoid and 1 minus it
template <typename T, int V>
__device__ __forceinline__ void sigmoids(Vec<V> x, Vec<V> bias, Vec<V>& s, Vec<V>& n) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int k = 0; k < V; k++) sigmoid_pair<T>(x.v[k], bias.v[k], s.v[k], n.v[k]);
  } else {
    Vec<V> e = fma(x, vec<V>(-LOG2E_F), bias);
#pragma unroll
    for (int k = 0; k < V; k++) e.v[k] = ex2_fast(min_or_nan(e.v[k], 126.0f));
    s = add(e, vec<V>(1.0f));
#pragma unroll
    for (int k = 0; k < V; k++) s.v[k] = rcp_fast(s.v[k]);
    n = mul(e, s);
  }
}

// A token's values.  `l` (POWER) is log f, natural for 32-bit tokens, else base 2; s, n: of the decay's gate; inv: 1 / gain.
template <int V>
struct Gates {
  Vec<V> f, gain, s, n, l, inv;
};
template <typename T, bool POWER, int V>
__device__ __forceinline__ Gates<V> decay(Vec<V> r, Vec<V> bias, Vec<V> k_) {
  Gates<V> a;
  sigmoids<T, V>(r, bias, a.s, a.n);
  if constexpr (!POWER) {
    a.f = a.s; a.gain = a.n; a.l = a.inv = vec<V>(0.0f);
  } else {
    a.l = mul(k_, a.s);
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int k = 0; k < V; k++) {
        a.f.v[k] = expf(a.l.v[k]);
        a.gain.v[k] = sqrtf(-expm1f(2.0f * a.l.v[k]));
        a.inv.v[k] = 1.0f / fmaxf(a.gain.v[k], 1.0e-19f);
      }
    } else {
#pragma unroll
      for (int k = 0; k < V; k++) a.f.v[k] = ex2_fast(a.l.v[k]);
      // 1 - f^2 = -(e^y - 1), y = 2 ln2 l <= 0: near zero by a polynomial for (e^y - 1) / y on [-1/2, 0] (relative minimax, found by linear
      // programming, 1.0e-7 off in fp32), as the difference would lose its digits there
      const Vec<V> y = mul(a.l, vec<V>(2.0f * LN2_F));
      Vec<V> q = fma(y, vec<V>(0.006771687883883715f), vec<V>(0.0410030297935009f));
      q = fma(y, q, vec<V>(0.1665491908788681f));
      q = fma(y, q, vec<V>(0.4999926686286926f));
      q = fma(y, q, vec<V>(0.9999999403953552f));
      q = mul(q, y);
      const Vec<V> d = fma(a.f, a.f, vec<V>(-1.0f));
#pragma unroll
      for (int k = 0; k < V; k++) {
        const float m = y.v[k] > -0.5f ? -q.v[k] : -d.v[k];
        a.inv.v[k] = rsqrt_fast(fmaxf(m, 1.0e-38f));     // l times it is 0 where l is
        a.gain.v[k] = m * a.inv.v[k];
      }
    }
  }
  return a;
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
inline int cluster_of(long long slabs, long long T, int tile) {
  int size = 1;
  while (size < MAX_CLUSTER && slabs * size * 2 <= 2 * 148 && (long long)size * tile < T) size *= 2;
  return size;
}

template <typename K, typename P>
cudaError_t launch_clusters(K kernel, const P& p, long long slabs, int size, int bytes, cudaStream_t stream) {
  if (slabs * size > 0x7fffffffLL) return cudaErrorInvalidValue;
  if (bytes > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) return e;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(slabs * size));
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = (size_t)bytes;
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
