// Gated linear recurrence over packed sequences, forward, and its step for single tokens (formulas and layout: kda_gscan.cuh).
// Measured in bf16, both gates: 20 ragged prompts, 29 814 tokens of 4096 channels, 333 us (2.9 TB/s); 8192 tokens of 4096 channels in one
// sequence 93 us, of 2560 68, with 4095 channels (read one by one) 133, in fp32 129; 65 537 tokens of 1024 channels in fp16, one gate, 157 us.
// A slab of channels has 16 blocks along time at most, so 65 536 tokens of 64 channels take 138 us, as long as 256 channels do.
#include "kda_gscan.cuh"

namespace kda {

namespace {

using namespace gscan;

constexpr int WARPS = 8, THREADS = WARPS * 32;
constexpr int DEPTH = 2;                 // rounds of tokens on their way or worked on
constexpr int S = 12, TILE = WARPS * S;  // tokens of a slice, of a block: 16 a slice do not fit 128 registers with all that a ragged batch takes
static_assert(GATED_SCAN_TILE % S == 0 && TILE % GATED_SCAN_TILE == 0, "the states that a training pass keeps are those in front of slices");

// One round's maps of the warps' slices, {F, U} of a lane's channels, double-buffered against warps (blocks) that are a round ahead.
template <int V>
struct Shared {
  Vec<2 * V> map[2][WARPS][32];
  unsigned long long sent[2];            // barriers: the tiles' maps have arrived
  uint32_t starts[2][WARPS];             // whether a sequence starts there: the map is constant
  Tables<true> tables;
};
using Tile = float4[32];                 // of the cluster's tiles, sent by their blocks: {F, F, U, U}; F < 0: the map is constant

struct Steps {             // bytes from a row to the fourth behind it
  long long x, r, i, y;
};

// Stores the final states of the sequences that end at t, where they change.  h: the state in front of t.
template <int V>
__device__ __forceinline__ void finish(const GatedScanParams& p, const Layout<true> l, uint32_t t, bool all_empty, int c, bool mine, float h0, float h1) {
  if (p.dst == nullptr) return;
  const float h[2] = {h0, h1};
  for (int j = all_empty ? 1 : lower(l, 0, p.seq.N + 1, t); j <= p.seq.N; j++) {
    if (!all_empty && l.at(j) != t) return;
    if (j == 0) continue;
    const bool empty = all_empty || l.at(j - 1) == t;
    const long long slot = claim(l, j - 1);          // of an empty one too: a bad entry is reported
    if (slot < 0 || !mine || (empty && p.src == p.dst)) continue;
#pragma unroll
    for (int k = 0; k < V; k++)
      p.dst[slot * p.dst_stride + c + k] = !empty ? h[k] : (p.src != nullptr ? p.src[slot * p.src_stride + c + k] : 0.0f);
  }
}

template <typename T, bool ASYNC, bool POWER, bool GATED>
__global__ void __launch_bounds__(THREADS, 2) kda_gated_scan_kernel(const __grid_constant__ GatedScanParams p, const __grid_constant__ Steps g) {
  constexpr int V = CHANNELS<T, ASYNC>, NT = GATED ? 3 : 2;
  __shared__ Shared<V> sm;
  using Tokens = Slice<T, S>;
  constexpr int RAW = ASYNC ? DEPTH * WARPS * NT * (int)sizeof(Tokens) : 0;
  extern __shared__ __align__(128) unsigned char raw[];              // ASYNC: [DEPTH][WARPS][NT] slices; then [2][blocks of the cluster] tiles
  const uint32_t rank = cluster_rank(), size = cluster_size();
  Tile* const tiles = reinterpret_cast<Tile*>(raw + RAW);
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int c0 = (int)(blockIdx.x / size) * 32 * V, c = c0 + lane * V;
  const bool mine = c < p.C, chunk = c0 + lane % 8 * (16 / (int)sizeof(T)) < p.C;
  if (threadIdx.x == 0)
    for (int b = 0; b < 2; b++) bar_init(&sm.sent[b]);
  if (size > 1) cluster_arrive();                    // blocks write into one another: all of them have to be there
  const bool rejected = cu_rejected(p.seq);
  const Layout<true> tables = rejected ? Layout<true>{p.seq, nullptr} : layout_of(p.seq, sm.tables);
  const uint32_t end = rejected ? 0 : (uint32_t)cu_at(p.seq, p.seq.N);       // tokens fit 31 bits, and a round more 32
  const uint32_t step = size * TILE;
  const int rounds = end > 0 ? (int)(((long long)end + step - 1) / step) : 1;

  uint32_t t0 = rank * TILE + warp * S;
  Registers<T, S> rx, rr, ri;
  auto slice = [&](int slot, int k) -> Tokens& { return reinterpret_cast<Tokens*>(raw)[(slot * WARPS + warp) * NT + k]; };
  auto ask = [&](int ahead, int slot) {              // the tokens of a later round
    const uint32_t t = t0 + ahead * step;
    const int m = count<S>(t, end);
    if constexpr (ASYNC) {
      if (m > 0) {
        Cursor<T, S>(p.x, p.ldx, t, c0).ask(slice(slot, 0), g.x, m, chunk, p.x);
        Cursor<T, S>(p.r, p.ldr, t, c0).ask(slice(slot, 1), g.r, m, chunk, p.r);
        if (GATED) Cursor<T, S>(p.i, p.ldi, t, c0).ask(slice(slot, 2), g.i, m, chunk, p.i);
      }
      copies_commit();
    } else if (m > 0) {
      rx.ask(p.x, p.ldx, t, m, c, p.C);
      rr.ask(p.r, p.ldr, t, m, c, p.C);
      if (GATED) ri.ask(p.i, p.ldi, t, m, c, p.C);
    }
  };
#pragma unroll
  for (int k = 0; k < (ASYNC ? 2 : 1); k++) ask(k, k);
  Vec<V> rb, ib, k_;
#pragma unroll
  for (int k = 0; k < V; k++) {
    rb.v[k] = mine ? bias_of<T>(p.r_bias, c + k) : 0.0f;
    ib.v[k] = GATED && mine ? bias_of<T>(p.i_bias, c + k) : 0.0f;
    k_.v[k] = POWER && mine ? decay_factor(p.rate, c + k, p.rate_scale) : 0.0f;
  }
  uint32_t next = 0;                                 // the first entry of cu_seqlens that is not in front of the round's slice
  int early = -1;                                    // the first sequence that starts in it, where its state has been asked for
  Vec<V> carry = vec<V>(0.0f);                       // the state in front of a round
  bool lost = false;

  Vec<V> f[S], u[S];                                 // decays and terms of a round
  auto gates = [&](int s, const Tokens& x, const Tokens& r, const Tokens& i) {
    Vec<V> xs, rs, is;
    if constexpr (ASYNC) {
      xs = values(x.row[s][lane]); rs = values(r.row[s][lane]); is = values(i.row[s][lane]);
    } else {
      xs = vec<V>(to_float(rx.row[s])); rs = vec<V>(to_float(rr.row[s])); is = vec<V>(to_float(ri.row[s]));
    }
    token_terms<T, POWER, GATED, V>(xs, rs, is, rb, ib, k_, f[s], u[s]);
  };
  auto look = [&](uint32_t t, int buf) {             // for sequences that start in the slice at t, which is next; their place is that of its map
    early = -1;
    if (next < t) {
      const int j = lower(tables, 0, p.seq.N + 1, t);
      next = j <= p.seq.N ? tables.at(j) : NEVER;
    }
    if (next >= t + S || next >= end || p.src == nullptr) return;
    early = lower(tables, 0, p.seq.N + 1, next + 1) - 1;
    const long long from = claim(tables, early);
#pragma unroll
    for (int k = 0; k < V; k++) {
      const bool here = from >= 0 && mine;
      asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(&sm.map[buf][warp][lane].v[k]))),
                   "l"(here ? p.src + from * p.src_stride + c + k : p.src), "r"(here ? 4 : 0) : "memory");
    }
  };
  __syncthreads();                                   // the copies of the tables
  if (!rejected) look(t0, 0);
  if (ASYNC) {
    copies_wait<1>();
    __syncwarp();
  }
#pragma unroll
  for (int s = 0; s < S; s++) gates(s, slice(0, 0), slice(0, 1), slice(0, NT - 1));
  if (ASYNC) __syncwarp();
  if (ASYNC) ask(2, 0);
  else ask(1, 0);
  if (size > 1) cluster_wait();

  for (int round = 0; round < rounds; round++, t0 += step) {
    const int buf = round & 1, n = count<S>(t0, end);
    if (size > 1 && threadIdx.x == 0 && !lost) bar_expect(&sm.sent[buf], (size + p.more_maps) * 512);
    const bool begins = !rejected && next < t0 + n, plain = !begins && n == S && t0 + S != end;       // begins: some sequence starts in the slice
    Vec<V> F, U;                                     // the slice's map
    uint32_t starts = 0;
    if (plain) {
      F = f[0];
      U = u[0];
#pragma unroll
      for (int s = 1; s < S; s++) {
        U = fma(f[s], U, u[s]);
        F = mul(F, f[s]);
      }
    } else {
#pragma unroll
      for (int s = 0; s < S; s++)
        if (s >= n) { f[s] = vec<V>(1.0f); u[s] = vec<V>(0.0f); }
      // sequences that start in the slice: the state they enter with joins the first token's term
      if (begins) asm volatile("cp.async.wait_all;" ::: "memory");          // of `look`, whether they have joined a group or not
      for (int q = begins ? lower(tables, 0, p.seq.N + 1, t0) : p.seq.N; q < p.seq.N; q++) {
        const uint32_t b = tables.at(q);
        if (b >= t0 + n) break;
        if (tables.at(q + 1) == b) continue;
        const int at = (int)(b - t0);
        starts |= 1u << at;
        Vec<V> h0 = vec<V>(0.0f);
        if (q == early) {
#pragma unroll
          for (int k = 0; k < V; k++) h0.v[k] = sm.map[buf][warp][lane].v[k];
        } else if (p.src != nullptr) {
          const long long from = claim(tables, q);
#pragma unroll
          for (int k = 0; k < V; k++)
            if (from >= 0 && mine) h0.v[k] = p.src[from * p.src_stride + c + k];
        }
#pragma unroll
        for (int s = 0; s < S; s++)
          if (s == at) u[s] = fma(f[s], h0, u[s]);
      }
      F = vec<V>(1.0f);
      U = vec<V>(0.0f);
#pragma unroll
      for (int s = 0; s < S; s++) {
        U = pick(starts >> s & 1, u[s], fma(f[s], U, u[s]));
        F = mul(F, f[s]);
      }
    }
    F = least(F);
    Vec<2 * V> map;
#pragma unroll
    for (int k = 0; k < V; k++) { map.v[k] = F.v[k]; map.v[V + k] = U.v[k]; }
    sm.map[buf][warp][lane] = map;
    if (lane == 0) sm.starts[buf][warp] = starts;
    const bool some = __syncthreads_or(starts != 0);
    // the slices in front of this one
    Vec<V> Fb = vec<V>(1.0f), Ub = vec<V>(0.0f);
    bool cut = false;
#pragma unroll
    for (int q = 0; q < WARPS - 1; q++) {
      if (q >= warp) break;
      const Vec<2 * V> m = sm.map[buf][q][lane];
      Vec<V> Fq, Uq;
#pragma unroll
      for (int k = 0; k < V; k++) { Fq.v[k] = m.v[k]; Uq.v[k] = m.v[V + k]; }
      Ub = fma(Fq, Ub, Uq);
      Fb = mul(Fb, Fq);
      if (some && sm.starts[buf][q] != 0) {
        cut = true;
        Ub = Uq;
      }
    }
    Fb = least(Fb);
    Vec<V> enter = carry;
    if (size == 1) {
#pragma unroll
      for (int q = 0; q < WARPS; q++) {
        const Vec<2 * V> m = sm.map[buf][q][lane];
        Vec<V> Fq, Uq;
#pragma unroll
        for (int k = 0; k < V; k++) { Fq.v[k] = m.v[k]; Uq.v[k] = m.v[V + k]; }
        carry = fma(Fq, carry, Uq);
        if (some && sm.starts[buf][q] != 0) carry = Uq;
      }
    } else {
      if (warp == WARPS - 1 && !lost) {              // it has the tile's map: to every block of the cluster
        const Vec<V> Ut = starts ? U : fma(F, Ub, U);
        Vec<V> Ft = least(mul(Fb, F));
        if (cut || starts) Ft = vec<V>(-1.0f);
        for (uint32_t b = 0; b < size; b++) send(&tiles[buf * size + rank][lane], &sm.sent[buf], b, make_float4(Ft.v[0], Ft.v[V - 1], Ut.v[0], Ut.v[V - 1]));
      }
      if (!lost) lost = bar_lost(&sm.sent[buf], round >> 1 & 1, p.wait_ns);
#pragma unroll
      for (int b = 0; b < MAX_CLUSTER; b++) {
        if (b >= size) break;
        const float4 m = tiles[buf * size + b][lane];
        Vec<V> Fq, Uq;
        Fq.v[0] = m.x; Fq.v[V - 1] = m.y; Uq.v[0] = m.z; Uq.v[V - 1] = m.w;
        if (b == rank) enter = carry;
        carry = pick(m.x < 0.0f, Uq, fma(Fq, carry, Uq));
      }
    }
    Vec<V> h = cut ? Ub : fma(Fb, enter, Ub);
    if (p.tiles != nullptr && warp % (GATED_SCAN_TILE / S) == 0 && mine && n > 0) {
#pragma unroll
      for (int k = 0; k < V; k++) p.tiles[(long long)(t0 / GATED_SCAN_TILE) * p.C + c + k] = h.v[k];
    }
    T* out = reinterpret_cast<T*>(p.out) + (long long)t0 * p.ldo + c;
    if (!plain && n > 0) {                           // token by token, with the ends of sequences; u becomes the states
      Vec<V> v = h;
#pragma unroll
      for (int s = 0; s < S; s++) {
        if (s < n) {
          v = pick(starts >> s & 1, u[s], fma(f[s], v, u[s]));
          u[s] = v;
          if (mine) *reinterpret_cast<Pack<T, V>*>(out + s * p.ldo) = pack<T, V>(v.v);
        }
      }
      // entries within the tokens start some sequence
      for (uint32_t bits = starts | (t0 + n == end ? 1u << n : 0); bits != 0; bits &= bits - 1) {
        const int at = __ffs(bits) - 1;
        Vec<V> before = h;
#pragma unroll
        for (int s = 0; s < S; s++) before = pick(s + 1 == at, u[s], before);
        finish<V>(p, tables, t0 + at, false, c, mine, before.v[0], before.v[V - 1]);
      }
    }
    if (!rejected) look(t0 + step, buf ^ 1);
    // The round's outputs and the next one's gates together: what the exponentials' unit takes longest for lies beside the rest.  Outputs
    // go through shared memory, in the places of the tokens that were read there.
    Tokens &x = slice(round + 1 & 1, 0), &r = slice(round + 1 & 1, 1), &i = slice(round + 1 & 1, NT - 1);
    if (ASYNC) {
      copies_wait<1>();
      __syncwarp();
    }
#pragma unroll
    for (int s = 0; s < S; s++) {
      h = fma(f[s], h, u[s]);
      gates(s, x, r, i);
      if constexpr (ASYNC) x.row[s][lane] = pack<T, V>(h.v);
      else if (plain && mine) out[s * p.ldo] = from_float<T>(h.v[0]);
    }
    if constexpr (ASYNC) {
      __syncwarp();
      if (plain) Cursor<T, S>(p.out, p.ldo, t0, c0).store(x, g.y, S, chunk);
      __syncwarp();
    }
    ask(ASYNC ? 3 : 2, round + 1 & 1);
  }
  if (!rejected && end == 0 && rank == 0 && warp == 0) finish<V>(p, tables, 0, false, c, mine, 0.0f, 0.0f);
  if (lost) {                                        // others may still send here: those that have not left
    report(p.seq.status, SEQ_LOST);
    cluster_arrive();
    cluster_wait();
  }
  if (rejected && rank == 0 && warp == 0) finish<V>(p, tables, 0, true, c, mine, 0.0f, 0.0f);
  if (rejected || p.zero_pad) zero_rest<T, V>(p.out, p.ldo, end, p.seq.T, c, mine, rank, size);
}

template <typename T, bool ASYNC, bool POWER, bool GATED>
cudaError_t launch_gates(const GatedScanParams& p, cudaStream_t stream) {
  constexpr int V = CHANNELS<T, ASYNC>, B = sizeof(T);
  const long long slabs = (p.C + 32 * V - 1) / (32 * V);
  const auto bytes = [](int size) { return (ASYNC ? DEPTH * WARPS * (GATED ? 3 : 2) * (int)sizeof(Slice<T, S>) : 0) + 2 * size * (int)sizeof(Tile); };
  const auto kernel = kda_gated_scan_kernel<T, ASYNC, POWER, GATED>;
  const int size = cluster_of(kernel, slabs, p.seq.T, TILE, THREADS, bytes);
  const Steps g = {4 * p.ldx * B, 4 * p.ldr * B, 4 * p.ldi * B, 4 * p.ldo * B};
  return launch_clusters(kernel, slabs, size, THREADS, bytes(size), bytes(MAX_CLUSTER), stream, p, g);
}

template <typename T, bool ASYNC>
cudaError_t launch_form(const GatedScanParams& p, cudaStream_t stream) {
  if (p.rate != nullptr) return p.i != nullptr ? launch_gates<T, ASYNC, true, true>(p, stream) : launch_gates<T, ASYNC, true, false>(p, stream);
  return p.i != nullptr ? launch_gates<T, ASYNC, false, true>(p, stream) : launch_gates<T, ASYNC, false, false>(p, stream);
}

template <typename T>
cudaError_t launch_type(const GatedScanParams& p, cudaStream_t stream) {
  const int size = sizeof(T);
  const bool async = p.C % (16 / size) == 0 && rows_on(p.x, p.ldx, size, 16) && rows_on(p.r, p.ldr, size, 16) && rows_on(p.i, p.ldi, size, 16) &&
                     rows_on(p.out, p.ldo, size, 16);
  return async ? launch_form<T, true>(p, stream) : launch_form<T, false>(p, stream);
}

// ---- one token a row
constexpr int STEP_THREADS = 128, STEP_ROWS = 4;

// VEC channels a thread, up to STEP_ROWS rows a block; the rows' states and tokens are asked for before repeats are looked for.  The input gate
// of 32-bit tokens takes the exact exponential here and the approximate one in prompts: the two differ in last digits.
template <typename T, int VEC, bool POWER>
__global__ void __launch_bounds__(STEP_THREADS) kda_gated_scan_step_kernel(const GatedScanParams p) {
  using P = Pack<T, VEC>;
  using F = Pack<float, VEC>;
  const int cblocks = (p.C / VEC + STEP_THREADS - 1) / STEP_THREADS;
  const int row0 = blockIdx.x / cblocks * p.tile, rows = min(p.tile, (int)p.seq.T - row0);
  const int c = ((int)(blockIdx.x % cblocks) * STEP_THREADS + (int)threadIdx.x) * VEC;
  int slot[STEP_ROWS];
  row_slots(p.seq, row0, rows, slot);
  const bool mine = c < p.C;
  P x[STEP_ROWS], r[STEP_ROWS], i[STEP_ROWS];
  F state[STEP_ROWS];
#pragma unroll
  for (int q = 0; q < STEP_ROWS; q++) {
    const long long row = row0 + q;
    if (mine && slot[q] != -2) {
      x[q] = *reinterpret_cast<const P*>(reinterpret_cast<const T*>(p.x) + row * p.ldx + c);
      r[q] = *reinterpret_cast<const P*>(reinterpret_cast<const T*>(p.r) + row * p.ldr + c);
      if (p.i != nullptr) i[q] = *reinterpret_cast<const P*>(reinterpret_cast<const T*>(p.i) + row * p.ldi + c);
    }
    if (mine && slot[q] >= 0) state[q] = *reinterpret_cast<const F*>(p.src + slot[q] * p.src_stride + c);
  }
  float rb[VEC], ib[VEC], k_[VEC];
#pragma unroll
  for (int k = 0; k < VEC; k++) {
    rb[k] = mine ? bias_of<T>(p.r_bias, c + k) : 0.0f;
    ib[k] = mine && p.i != nullptr ? bias_of<T>(p.i_bias, c + k) : 0.0f;
    k_[k] = POWER && mine ? decay_factor(p.rate, c + k, p.rate_scale) : 0.0f;
  }
  drop_repeats(p.seq, row0, slot);
  if (!mine) return;
#pragma unroll
  for (int q = 0; q < STEP_ROWS; q++) {
    if (q >= rows) break;
    P* out = reinterpret_cast<P*>(reinterpret_cast<T*>(p.out) + (long long)(row0 + q) * p.ldo + c);
    float h[VEC];
    if (slot[q] == -2) {
#pragma unroll
      for (int k = 0; k < VEC; k++) h[k] = 0.0f;
      if (p.zero_pad) *out = pack<T, VEC>(h);
      continue;
    }
    F to;
#pragma unroll
    for (int k = 0; k < VEC; k++) {
      const Gates<1> a = decay<T, POWER, 1>({to_float(r[q].v[k])}, {rb[k]}, {k_[k]});
      h[k] = a.gain.v[0] * to_float(x[q].v[k]);
      if (p.i != nullptr) {
        float g, ng;
        sigmoid_pair<T>(to_float(i[q].v[k]), ib[k], g, ng);
        h[k] *= g;
      }
      h[k] = fmaf(a.f.v[0], slot[q] >= 0 ? state[q].v[k] : 0.0f, h[k]);
      to.v[k] = h[k];
    }
    *out = pack<T, VEC>(h);
    if (slot[q] >= 0) *reinterpret_cast<F*>(p.dst + slot[q] * p.dst_stride + c) = to;
  }
}

template <typename T, int VEC>
cudaError_t launch_step(GatedScanParams p, cudaStream_t stream) {
  const long long cblocks = (p.C / VEC + STEP_THREADS - 1) / STEP_THREADS;
  p.tile = STEP_ROWS;
  while (p.tile > 1 && (p.seq.T + p.tile - 1) / p.tile * cblocks < 2 * 148) p.tile /= 2;
  const long long blocks = (p.seq.T + p.tile - 1) / p.tile * cblocks;
  if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
  if (blocks == 0) return cudaSuccess;
  if (p.rate != nullptr) kda_gated_scan_step_kernel<T, VEC, true><<<(unsigned)blocks, STEP_THREADS, 0, stream>>>(p);
  else kda_gated_scan_step_kernel<T, VEC, false><<<(unsigned)blocks, STEP_THREADS, 0, stream>>>(p);
  return cudaGetLastError();
}

template <typename T>
cudaError_t launch_step_type(const GatedScanParams& p, cudaStream_t stream) {
  constexpr int VEC = 4, B = VEC * sizeof(T);
  const bool wide = p.C % VEC == 0 && rows_on(p.x, p.ldx, sizeof(T), B) && rows_on(p.r, p.ldr, sizeof(T), B) && rows_on(p.i, p.ldi, sizeof(T), B) &&
                    rows_on(p.out, p.ldo, sizeof(T), B) && rows_on(p.dst, p.dst_stride, 4, 16);
  return wide ? launch_step<T, VEC>(p, stream) : launch_step<T, 1>(p, stream);
}

}  // namespace

cudaError_t launch_gated_scan(const GatedScanParams& p, int type, cudaStream_t stream) {
  if (type == TYPE_BF16) return launch_type<__nv_bfloat16>(p, stream);
  if (type == TYPE_FP16) return launch_type<__half>(p, stream);
  return launch_type<float>(p, stream);
}

cudaError_t launch_gated_scan_step(const GatedScanParams& p, int type, cudaStream_t stream) {
  if (type == TYPE_BF16) return launch_step_type<__nv_bfloat16>(p, stream);
  if (type == TYPE_FP16) return launch_step_type<__half>(p, stream);
  return launch_step_type<float>(p, stream);
}

}  // namespace kda
