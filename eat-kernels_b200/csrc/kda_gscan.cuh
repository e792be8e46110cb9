// What the passes of the gated linear recurrence share.  Per channel, with s = sigmoid(r + r_bias), g = sigmoid(i + i_bias) (1 without i):
//   rate given:  l = -c softplus(rate) s, f = exp(l), gain = sqrt(1 - f^2);      without:  f = s, gain = 1 - s
//   h[t] = f[t] h[t-1] + gain[t] g[t] x[t],  y = h
//
// Time is cut without regard to the sequences of the batch: a warp has a slice of S consecutive tokens for 32 lanes of channels, a block
// the slices of its warps (a tile), the blocks of a cluster one tile each behind one another (a round), and the cluster goes over the
// batch round by round.  A slice is summed up by a map h -> F h + U (F: product of its decays); a sequence that starts inside it makes
// that map the constant U, which a flag says (0 times an infinite state in front would be NaN).  The maps of a block meet in
// shared memory, those of a cluster are sent to all its blocks, one barrier a round each, always in the same order: results do
// not depend on timing, nothing is kept in memory between blocks, tokens are read once, and ragged batches cost what their tokens cost.
//
// What bounds it: the floor is memory (8 bytes an element of 16 bits forward, 14 backward), but an element takes some 40 instructions
// and five operations of the special-function unit (backward 90 and eleven), so that unit's and the issue slots' times each come near the
// memory's, and a round's chain of barrier, exchange and barrier lies in front of its outputs.  Measured steps that mattered: plain
// slices without checks (120 -> 45 instructions an element), tokens by 16-byte asynchronous copies, no fence in the exchange, two blocks
// an SM without spills (slices of 12 tokens; 16 spill and are 20 % slower, 6 and 8 pay the round's chain more often), code that fits the
// instruction cache, slow paths included.
#pragma once
#include "kda_serving.cuh"
#include <atomic>

namespace kda {

namespace gscan {

constexpr int MAX_CLUSTER = 16, MAX_DEVICES = 64;
constexpr uint32_t NEVER = 0xffffffffu;

// A product of decays that underflows to zero is taken as the smallest positive number, so that an infinite state stays infinite, as it
// does token by token (a finite one is not changed by that).  Where a decay is NaN, so is the map's constant.
constexpr float LEAST = 1.4e-45f;
constexpr float LOG2E_F = 1.4426950408889634f, LOG2E_REST = 1.925963033500e-8f, LN2_F = 0.6931471805599453f;

__device__ __forceinline__ float sqrt_fast(float x) {
  float y;
  asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
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

// The decay's factor in front of s, to base 2: -c softplus(rate) log2(e); finite, since an infinite one times s = 0 would
// be NaN.
__device__ __forceinline__ float decay_factor(const float* rate, int c, float scale) {
  const float k = -scale * softplus_exact(rate[c]) * LOG2E_F;
  return k < -3.0e38f ? -3.0e38f : k;
}

// ---- sequences
// A block's view of the tables: where they are short, copies in shared memory, so that a slice in which sequences meet does not wait for one
// load after the other.  (The rounds of a cluster wait for its slowest block.)
constexpr int TABLE = 256;
template <bool SLOTS>
struct Tables {
  int cu[SLOTS ? TABLE : TABLE / 2], slot[SLOTS ? TABLE : 1];          // slot: -1 out of range
};
template <bool SLOTS>
struct Layout {
  const SeqTable& s;
  const Tables<SLOTS>* copy;             // nullptr: read where they lie
  __device__ __forceinline__ uint32_t at(int i) const { return copy != nullptr ? (uint32_t)copy->cu[i] : (uint32_t)cu_at(s, i); }
  __device__ __forceinline__ int slot_of(int i) const {
    if (SLOTS && copy != nullptr) return copy->slot[i];
    const long long d = s.slots != nullptr ? table_at(s.slots, s.slots_is64, i) : i;
    return d < 0 || d >= s.n_slots ? -1 : (int)d;
  }
};
// Called by the whole block, which meets a barrier before it uses the copy.  Not for a layout that is rejected.
template <bool SLOTS>
__device__ __forceinline__ Layout<SLOTS> layout_of(const SeqTable& s, Tables<SLOTS>& copy) {
  const Layout<SLOTS> direct = {s, nullptr};
  if (s.N >= (int)(sizeof(copy.cu) / sizeof(int))) return direct;
  for (int i = threadIdx.x; i <= s.N; i += blockDim.x) {
    copy.cu[i] = (int)cu_at(s, i);
    if (SLOTS) copy.slot[i] = i < s.N ? direct.slot_of(i) : -1;
  }
  return {s, &copy};
}

// Called by a warp: the first of the entries [lo, hi) of cu_seqlens that is >= t, hi where none is.  32 entries are looked at at a time.
template <bool SLOTS>
__device__ __forceinline__ int lower(const Layout<SLOTS>& l, int lo, int hi, uint32_t t) {
  const int lane = threadIdx.x % 32;
  while (lo < hi) {
    const int part = (hi - lo + 31) / 32;
    const long long at = (long long)lo + (long long)(lane + 1) * part - 1;
    const unsigned found = __ballot_sync(0xffffffffu, l.at(at < hi ? (int)at : hi - 1) >= t);
    if (found == 0) return hi;
    const int first = __ffs(found) - 1;
    hi = min(hi - 1, lo + (first + 1) * part - 1);
    lo = lo + first * part;
  }
  return lo;
}

// Called by a warp: the slot of sequence i, or -1 where its entry is out of range or repeats an earlier one
template <bool SLOTS>
__device__ __forceinline__ long long claim(const Layout<SLOTS>& l, int i) {
  if (l.s.slots == nullptr) return i;
  const int d = l.slot_of(i);
  int bad = d < 0;
  for (int j = threadIdx.x % 32; j < i && !bad; j += 32)
    if (l.slot_of(j) == d) bad = 1;
  if (!__any_sync(0xffffffffu, bad)) return d;
  if (threadIdx.x % 32 == 0) report(l.s.status, SEQ_BAD_SLOT);
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
// Values for another block, at the address of `own` there; they count towards the bytes that its barrier (at the address of `bar`) waits
// for.  No fence: a barrier of the cluster with release would wait for the block's outputs to be in memory, 1.4 of 5 cycles a warp
// spent per instruction.
__device__ __forceinline__ void send(const void* own, const void* bar, uint32_t rank, float4 v) {
  const uint32_t a = static_cast<uint32_t>(__cvta_generic_to_shared(own)), b = static_cast<uint32_t>(__cvta_generic_to_shared(bar));
  asm volatile("{\n .reg .b32 t, u;\n mapa.shared::cluster.u32 t, %0, %2;\n mapa.shared::cluster.u32 u, %1, %2;\n"
               " st.async.shared::cluster.mbarrier::complete_tx::bytes.v4.f32 [t], {%3, %4, %5, %6}, [u];\n}" ::"r"(a), "r"(b), "r"(rank), "f"(v.x), "f"(v.y),
               "f"(v.z), "f"(v.w) : "memory");
}
__device__ __forceinline__ void put_remote(const void* own, uint32_t rank, float v) {
  const uint32_t a = static_cast<uint32_t>(__cvta_generic_to_shared(own));
  asm volatile("{\n .reg .b32 t;\n mapa.shared::cluster.u32 t, %0, %1;\n st.shared::cluster.f32 [t], %2;\n}" ::"r"(a), "r"(rank), "f"(v) : "memory");
}
__device__ __forceinline__ void bar_init(const void* bar) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(bar))) : "memory");
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
}
__device__ __forceinline__ void bar_expect(const void* bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(bar))), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool bar_done(uint32_t b, uint32_t parity) {
  uint32_t done;
  asm volatile("{\n .reg .pred q;\n mbarrier.try_wait.parity.shared::cta.b64 q, [%1], %2;\n selp.u32 %0, 1, 0, q;\n}" : "=r"(done) : "r"(b), "r"(parity)
               : "memory");
  return done != 0;
}
// Called by a warp: whether the wait for a phase ran out, after `limit` ns.  A block that has lost its cluster goes on to its end
// without barriers, and sends nothing, so that the others lose it too; its results are wrong, and it says so.
__device__ __forceinline__ bool bar_lost(const void* bar, uint32_t parity, unsigned long long limit) {
  const uint32_t b = static_cast<uint32_t>(__cvta_generic_to_shared(bar));
  unsigned long long begin = 0, now;
  bool done = false;
  do {
    for (int i = 0; i < 64 && !done; i++) done = bar_done(b, parity);
    if (done) break;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(now));
    if (begin == 0) begin = now;
  } while (now - begin < limit);
  return __any_sync(0xffffffffu, !done);
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
__device__ __forceinline__ int count(uint32_t t0, uint32_t end) {          // tokens of the slice at t0
  return t0 >= end ? 0 : (end - t0 > S ? S : (int)(end - t0));
}

// A warp's slice of one tensor in shared memory: S rows of 128 bytes, which come and go in 16 bytes a lane.  Places behind the last token or
// channel are zeros.
template <typename T, int S>
struct Slice {
  Pack<T, 4 / sizeof(T)> row[S][32];
};
// Strides in bytes that a launch works out for a tensor: of four rows, of a round
struct Strides {
  long long four, round;
};
inline Strides strides(long long ld, int size, long long round) { return {4 * ld * size, round * ld * size}; }

// Where a lane's 16 bytes of a slice lie in memory: a row's, four rows on, ...
template <typename T, int S>
struct Cursor {
  const char* at;
  __device__ __forceinline__ Cursor(const void* base, long long ld, long long t0, int c0) {
    at = reinterpret_cast<const char*>(reinterpret_cast<const T*>(base) + (t0 + (int)(threadIdx.x % 32 / 8)) * ld + c0 + (int)(threadIdx.x % 8) * (16 / (int)sizeof(T)));
  }
  // n rows (`on`: the lane's channels exist) into a slice
  __device__ __forceinline__ void ask(Slice<T, S>& to, long long four, int n, bool on, const void* valid) const {
    const int row = threadIdx.x % 32 / 8;
    const uint32_t a = static_cast<uint32_t>(__cvta_generic_to_shared(&to)) + (uint32_t)(threadIdx.x % 32 * 16);
    const char* from = at;
    if (n == S && on) {
#pragma unroll
      for (int q = 0; q < (S + 3) / 4; q++) {
        if (4 * q + 3 < S || row + 4 * q < S) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(a + 512u * q), "l"(from) : "memory");
        from += four;
      }
    } else {
#pragma unroll
      for (int q = 0; q < (S + 3) / 4; q++) {
        const bool here = on && row + 4 * q < n;
        if (4 * q + 3 < S || row + 4 * q < S) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(a + 512u * q), "l"(here ? (const void*)from : valid), "r"(here ? 16 : 0) : "memory");
        from += four;
      }
    }
  }
  // the first n rows of a slice, which the warp has written, to memory
  __device__ __forceinline__ void store(const Slice<T, S>& from, long long four, int n, bool on) const {
    const int row = threadIdx.x % 32 / 8;
    const uint4* a = reinterpret_cast<const uint4*>(&from) + threadIdx.x % 32;
    char* to = const_cast<char*>(at);
#pragma unroll
    for (int q = 0; q < (S + 3) / 4; q++) {
      if (on && row + 4 * q < n) *reinterpret_cast<uint4*>(to) = a[32 * q];
      to += four;
    }
  }
};
// One channel a lane, read one by one a round ahead
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
template <>
__device__ __forceinline__ Vec<2> values(const Pack<__nv_bfloat16, 2>& p) {      // one instruction each
  const uint32_t w = *reinterpret_cast<const uint32_t*>(&p);
  return {__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)};
}

// Of V channels: sigmoid and, with BOTH, 1 minus it, both to relative accuracy.  The approximate exponential and reciprocal are good to
// 2^-22; for 32-bit tokens the exponential's argument is taken in two parts, since its rounding would be off by as much again for each unit of x.
// Alone, the sigmoid of an infinitely low x is zero; with the other one it stays at 2^-126, so that the product that makes that one is 1, or, with
// SHUTS, both become zero (the reciprocal of 2^127 does), for uses where the other one only stands in products with the first.
template <typename T, int V, bool BOTH = true, bool SHUTS = false>
__device__ __forceinline__ void sigmoids(Vec<V> x, Vec<V> bias, Vec<V>& s, Vec<V>& n) {
#pragma unroll
  for (int k = 0; k < V; k++) {
    constexpr float MOST = SHUTS ? 127.0f : 126.0f;
    float e;
    if constexpr (sizeof(T) == 4) {
      const float v = -(x.v[k] + bias.v[k]), hi = BOTH ? min_or_nan(v * LOG2E_F, MOST) : v * LOG2E_F;
      const float lo = fmaf(v, LOG2E_F, -hi) + v * LOG2E_REST;
      e = ex2_fast(hi);
      e = fabsf(hi) < 126.0f ? fmaf(e, lo * LN2_F, e) : e;
    } else {
      const float t = fmaf(x.v[k], -LOG2E_F, bias.v[k]);
      e = ex2_fast(BOTH ? min_or_nan(t, MOST) : t);
    }
    s.v[k] = rcp_fast(e + 1.0f);
    n.v[k] = BOTH ? e * s.v[k] : 0.0f;
  }
}

// f = 2^l and q = 1 - f^2, l <= 0.  Near zero q comes from a polynomial for (1 - 2^(2 l)) / l on [-0.36, 0] (relative minimax, found by linear
// programming, with its roundings 1.9e-7 off in fp32), as the difference d = 1 - f^2 would lose its digits there; and the approximate f,
// which may be two steps off, is put right by what d misses of q (Newton's step on f^2 = 1 - q, 1 / f taken as 1).  A state that decays
// slowly sums up that error 1 / (1 - f) times.
template <int V>
__device__ __forceinline__ void decay_pair(Vec<V> l, Vec<V>& f, Vec<V>& q) {
#pragma unroll
  for (int k = 0; k < V; k++) {                      // single values: pairs of constants would take registers, or moves
    const float a = l.v[k], e = ex2_fast(a), d = fmaf(-e, e, 1.0f);
    float m = fmaf(a, -0.03467162698507309f, -0.15143901109695435f);
    m = fmaf(a, m, -0.44371989369392395f);
    m = fmaf(a, m, -0.9608919620513916f);
    m = fmaf(a, m, -1.3862942457199097f);
    q.v[k] = a > -0.36f ? m * a : d;
    f.v[k] = fmaf(0.5f, d - q.v[k], e);
  }
}

// A token's values.  `l` (POWER) is log f to base 2; s, n: of the decay's gate; inv: 1 / gain.  What only gradients need comes with GRAD.
template <int V>
struct Gates {
  Vec<V> f, gain, s, n, l, inv;
};
template <typename T, bool POWER, int V, bool GRAD = false>
__device__ __forceinline__ Gates<V> decay(Vec<V> r, Vec<V> bias, Vec<V> k_) {
  Gates<V> a;
  sigmoids<T, V, GRAD || !POWER>(r, bias, a.s, a.n);
  if constexpr (!POWER) {
    a.f = a.s; a.gain = a.n; a.l = a.inv = vec<V>(0.0f);
#pragma unroll
    for (int k = 0; k < V; k++)                      // near one s is 1 - n to half a step
      if (a.n.v[k] < 0.5f) a.f.v[k] = 1.0f - a.n.v[k];
  } else {
    a.l = mul(k_, a.s);
    Vec<V> q;
    decay_pair(a.l, a.f, q);
#pragma unroll
    for (int k = 0; k < V; k++) {
      if (GRAD) {
        a.inv.v[k] = rsqrt_fast(fmaxf(q.v[k], 2.0e-38f));      // l times it is 0 where l is
        a.gain.v[k] = q.v[k] * a.inv.v[k];
      } else {
        a.gain.v[k] = sqrt_fast(q.v[k]);
      }
    }
  }
  return a;
}

// A token's decay f and term u.  With both gates in 16 bits u = sqrt(q) / (1 + e^-i) x, q = 1 - f^2, takes one reciprocal root,
// sqrt(q) / a = q rsqrt(q a^2): five operations of the special-function unit instead of six.  (An input gate below 2^-64 counts as shut:
// the square is infinite, a itself is not, so that q = 0 stays 0.)
template <typename T, bool POWER, bool GATED, int V>
__device__ __forceinline__ void token_terms(Vec<V> x, Vec<V> r, Vec<V> i, Vec<V> rb, Vec<V> ib, Vec<V> k_, Vec<V>& f, Vec<V>& u) {
  if constexpr (POWER && GATED && sizeof(T) == 2) {
    Vec<V> s, n;
    sigmoids<T, V, false>(r, rb, s, n);
    Vec<V> q;
    decay_pair(mul(k_, s), f, q);
    Vec<V> w;
#pragma unroll
    for (int k = 0; k < V; k++) {
      const float a = ex2_fast(min_or_nan(fmaf(i.v[k], -LOG2E_F, ib.v[k]), 126.0f)) + 1.0f;
      w.v[k] = rsqrt_fast(fmaf(q.v[k] * a, a, 2.0e-38f));
    }
    u = mul(mul(q, w), x);
  } else {
    const Gates<V> a = decay<T, POWER, V>(r, rb, k_);
    f = a.f;
    u = mul(a.gain, x);
    if constexpr (GATED) {
      Vec<V> g, n;
      sigmoids<T, V, false>(i, ib, g, n);
      u = mul(u, g);
    }
  }
}

// Rows [end, T) of an output are zeros, spread over the blocks of a cluster
template <typename T, int V>
__device__ __forceinline__ void zero_rest(void* out, long long ld, long long end, long long T_, int c, bool mine, uint32_t rank, uint32_t size) {
  Pack<T, V> zero;
#pragma unroll
  for (int k = 0; k < V; k++) zero.v[k] = from_float<T>(0.0f);
  if (mine)
    for (long long t = end + rank * (blockDim.x / 32) + threadIdx.x / 32; t < T_; t += size * (blockDim.x / 32))
      *reinterpret_cast<Pack<T, V>*>(reinterpret_cast<T*>(out) + c + t * ld) = zero;
}

inline void configure(cudaLaunchConfig_t& cfg, cudaLaunchAttribute* attr, long long blocks, int size, int threads, int bytes, cudaStream_t stream) {
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = (size_t)bytes;
  cfg.stream = stream;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)size;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
}

// Blocks along time: as many as the card holds at once for all slabs, no more than the batch has tiles.  A cluster lies within one of
// the card's groups of SMs, so the sizes that fit are asked for (once for a kernel and device).
template <typename K, typename B>
int cluster_of(K kernel, long long slabs, long long T, int tile, int threads, B bytes) {
  static std::atomic<int> room[MAX_DEVICES][MAX_CLUSTER + 1];        // clusters of a size that run at once, plus one; 0: not asked yet
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev >= MAX_DEVICES) return 1;
  int best = 1;
  for (int size = 2; size <= MAX_CLUSTER && (long long)(size - 1) * tile < T; size++) {
    if (room[dev][size] == 0) {
      cudaLaunchConfig_t cfg = {};
      cudaLaunchAttribute attr[1];
      configure(cfg, attr, size, size, threads, bytes(size), nullptr);
      int n = 0;
      if (size > 8) cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes(MAX_CLUSTER));
      if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess) {
        n = 0;
        cudaGetLastError();
      }
      room[dev][size] = n + 1;
    }
    if (slabs <= room[dev][size] - 1) best = size;
  }
  return best;
}

template <typename K, typename... P>
cudaError_t launch_clusters(K kernel, long long slabs, int size, int threads, int bytes, int most, cudaStream_t stream, const P&... p) {
  if (slabs * size > 0x7fffffffLL) return cudaErrorInvalidValue;
  // the same for all sizes: another thread may be about to launch a larger one
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
  if (e != cudaSuccess) return e;
  if (size > 8) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return e;
  }
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  configure(cfg, attr, slabs * size, size, threads, bytes, stream);
  e = cudaLaunchKernelEx(&cfg, kernel, p...);
  return e != cudaSuccess ? e : cudaGetLastError();
}

// Whether every row of a tensor starts on a multiple of `bytes`
inline bool rows_on(const void* p, long long ld, int size, int bytes) {
  return ((reinterpret_cast<uintptr_t>(p) | (uintptr_t)(ld * size)) & (uintptr_t)(bytes - 1)) == 0;
}

}  // namespace gscan

}  // namespace kda
