// Gated linear recurrence over packed sequences, forward, and its step for single tokens (formulas and layout: kda_gscan.cuh).
#include "kda_gscan.cuh"

namespace kda {

namespace {

using namespace gscan;

// Stores the final states of the sequences that end at t: those of entries j and behind.  h: the state in front of t.
template <int V>
__device__ __noinline__ void finish(const GatedScanParams& p, int j, long long t, bool all_empty, int c, bool mine, float h0, float h1) {
  if (p.dst == nullptr) return;
  const float h[2] = {h0, h1};
  for (; j <= p.seq.N; j++) {
    if (!all_empty && cu_at(p.seq, j) != t) return;
    if (j == 0) continue;
    const bool empty = all_empty || cu_at(p.seq, j - 1) == t;
    if (empty && p.src == p.dst) continue;
    const long long slot = claim(p.seq, j - 1);
    if (slot < 0 || !mine) continue;
#pragma unroll
    for (int k = 0; k < V; k++)
      p.dst[slot * p.dst_stride + c + k] = !empty ? h[k] : (p.src != nullptr ? p.src[slot * p.src_stride + c + k] : 0.0f);
  }
}

constexpr int DEPTH = 2;                 // rounds of tokens on their way or worked on

template <typename T, bool ASYNC>
constexpr int TOKENS = ASYNC ? 16 : 8;   // of a slice

// One round's maps of the warps' slices, {F, U} of a lane's channels, double-buffered against warps (blocks) that are a round ahead.
template <int V>
struct Shared {
  Vec<2 * V> map[2][WARPS][32];
  float4 tile[2][MAX_CLUSTER][32];       // of the cluster's tiles, written by their blocks: {F, F, U, U}
  uint32_t starts[2][WARPS], tile_starts[2][MAX_CLUSTER];          // whether a sequence starts there: the map is constant
};

template <typename T, bool ASYNC, bool POWER, bool GATED>
__global__ void __launch_bounds__(THREADS, 2) kda_gated_scan_kernel(const __grid_constant__ GatedScanParams p) {
  constexpr int V = CHANNELS<T, ASYNC>, S = TOKENS<T, ASYNC>, TILE = WARPS * S, NT = GATED ? 3 : 2;
  __shared__ Shared<V> sm;
  extern __shared__ __align__(128) unsigned char raw[];              // ASYNC: [DEPTH][WARPS][NT] slices
  using Tokens = Slice<T, S>;
  const uint32_t rank = cluster_rank(), size = cluster_size();
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int c0 = (int)(blockIdx.x / size) * 32 * V, c = c0 + lane * V;
  const bool mine = c < p.C;
  if (size > 1) cluster_arrive();                    // blocks write into one another: all of them have to be there
  const bool rejected = cu_rejected(p.seq);
  const long long end = rejected ? 0 : cu_at(p.seq, p.seq.N);
  const long long step = (long long)size * TILE;
  const int rounds = end > 0 ? (int)((end + step - 1) / step) : 1;

  long long t0 = (long long)rank * TILE + warp * S;
  Registers<T, S> rx, rr, ri;
  auto slice = [&](int slot, int k) -> Tokens& { return reinterpret_cast<Tokens*>(raw)[(slot * WARPS + warp) * NT + k]; };
  auto ask = [&](int ahead, int slot) {              // the tokens of a later round
    const long long t = t0 + ahead * step;
    const int m = count<S>(t, end);
    if constexpr (ASYNC) {
      if (m > 0) {
        slice(slot, 0).ask(p.x, p.ldx, t, m, c0, p.C);
        slice(slot, 1).ask(p.r, p.ldr, t, m, c0, p.C);
        if (GATED) slice(slot, 2).ask(p.i, p.ldi, t, m, c0, p.C);
      }
      copies_commit();
    } else if (m > 0) {
      rx.ask(p.x, p.ldx, t, m, c, p.C);
      rr.ask(p.r, p.ldr, t, m, c, p.C);
      if (GATED) ri.ask(p.i, p.ldi, t, m, c, p.C);
    }
  };
#pragma unroll
  for (int k = 0; k < (ASYNC ? DEPTH - 1 : 1); k++) ask(k, k);
  Vec<V> rb, ib, k_;
#pragma unroll
  for (int k = 0; k < V; k++) {
    rb.v[k] = mine ? bias_of<T>(p.r_bias, c + k) : 0.0f;
    ib.v[k] = GATED && mine ? bias_of<T>(p.i_bias, c + k) : 0.0f;
    k_.v[k] = POWER && mine ? decay_factor<T>(p.rate, c + k, p.rate_scale) : 0.0f;
  }
  int j = 0;                                         // first entry of cu_seqlens that is >= t0, once looked for
  long long next = 0;                                // that entry
  Vec<V> carry = vec<V>(0.0f);
  if (size > 1) cluster_wait();

  int slot = 0;
  for (int round = 0; round < rounds; round++) {
    const int buf = round & 1, n = count<S>(t0, end);
    if (next < t0) {
      j = lower(p.seq, j, p.seq.N + 1, t0);
      next = j <= p.seq.N ? cu_at(p.seq, j) : NEVER;
    }
    const bool begins = !rejected && next < t0 + n;  // some sequence starts in the slice
    Vec<V> f[S], u[S];
    if constexpr (ASYNC) {
      copies_wait<DEPTH - 2>();
      __syncwarp();                                  // the warp's copies have landed; the slot of the round before is no longer read
      const Tokens &x = slice(slot, 0), &r = slice(slot, 1), &i = slice(slot, NT - 1);
#pragma unroll
      for (int s = 0; s < S; s++) {
        const Gates<V> a = decay<T, POWER, V>(values(r.row[s][lane]), rb, k_);
        f[s] = a.f;
        u[s] = mul(a.gain, values(x.row[s][lane]));
        if constexpr (GATED) {
          Vec<V> g, ng;
          sigmoids<T, V>(values(i.row[s][lane]), ib, g, ng);
          u[s] = mul(u[s], g);
        }
      }
    } else {
#pragma unroll
      for (int s = 0; s < S; s++) {
        const Gates<V> a = decay<T, POWER, V>(vec<V>(to_float(rr.row[s])), rb, k_);
        f[s] = a.f;
        u[s] = mul(a.gain, vec<V>(to_float(rx.row[s])));
        if constexpr (GATED) {
          Vec<V> g, ng;
          sigmoids<T, V>(vec<V>(to_float(ri.row[s])), ib, g, ng);
          u[s] = mul(u[s], g);
        }
      }
    }
    // the next tokens: ASYNC into the slot of the round before
    if (ASYNC) ask(DEPTH - 1, slot == 0 ? DEPTH - 1 : slot - 1);
    else ask(1, 0);
    if (n < S) {
#pragma unroll
      for (int s = 0; s < S; s++)
        if (s >= n) { f[s] = vec<V>(1.0f); u[s] = vec<V>(0.0f); }
    }
    // sequences that start in the slice: the state they enter with joins the first token's term
    uint32_t starts = 0;
    if (begins) {
      for (int q = j; q < p.seq.N; q++) {
        const long long t = cu_at(p.seq, q);
        if (t >= t0 + n) break;
        if (cu_at(p.seq, q + 1) == t) continue;
        const long long from = claim(p.seq, q);
        const int at = (int)(t - t0);
        starts |= 1u << at;
        Vec<V> h0 = vec<V>(0.0f);
#pragma unroll
        for (int k = 0; k < V; k++)
          if (p.src != nullptr && from >= 0 && mine) h0.v[k] = p.src[from * p.src_stride + c + k];
#pragma unroll
        for (int s = 0; s < S; s++)
          if (s == at) u[s] = fma(f[s], h0, u[s]);
      }
    }
    Vec<V> F = f[0], U = u[0];
    if (starts == 0) {
#pragma unroll
      for (int s = 1; s < S; s++) {
        U = fma(f[s], U, u[s]);
        F = mul(F, f[s]);
      }
    } else {
#pragma unroll
      for (int s = 1; s < S; s++) {
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
    auto slice_map = [&](int w, Vec<V>& Fw, Vec<V>& Uw) {
      const Vec<2 * V> m = sm.map[buf][w][lane];
#pragma unroll
      for (int k = 0; k < V; k++) { Fw.v[k] = m.v[k]; Uw.v[k] = m.v[V + k]; }
    };
    // the slices in front of this one
    Vec<V> Fb = vec<V>(1.0f), Ub = vec<V>(0.0f);
    bool cut = false;
#pragma unroll
    for (int w = 0; w < WARPS - 1; w++) {
      if (w >= warp) break;
      Vec<V> Fw, Uw;
      slice_map(w, Fw, Uw);
      const bool constant = some && sm.starts[buf][w] != 0;
      cut |= constant;
      Ub = constant ? Uw : fma(Fw, Ub, Uw);
      Fb = least(mul(Fb, Fw));
    }
    Vec<V> h;
    if (size == 1) {
      h = cut ? Ub : fma(Fb, carry, Ub);
      carry = h;                                     // the next round's
#pragma unroll
      for (int w = 0; w < WARPS; w++) {
        if (w < warp) continue;
        Vec<V> Fw, Uw;
        slice_map(w, Fw, Uw);
        carry = some && sm.starts[buf][w] != 0 ? Uw : fma(Fw, carry, Uw);
      }
    } else {
      if (warp == WARPS - 1) {                       // it has the tile's map: to every block of the cluster
        const Vec<V> Ut = starts ? U : fma(F, Ub, U), Ft = least(mul(Fb, F));
        for (uint32_t b = 0; b < size; b++) put_remote(&sm.tile[buf][rank][lane], b, make_float4(Ft.v[0], Ft.v[V - 1], Ut.v[0], Ut.v[V - 1]));
        if (lane < size) put_remote(&sm.tile_starts[buf][rank], lane, (uint32_t)(cut || starts != 0));
      }
      cluster_arrive();
      cluster_wait();
      Vec<V> enter = carry;
#pragma unroll
      for (int b = 0; b < MAX_CLUSTER; b++) {
        if (b >= size) break;
        const float4 m = sm.tile[buf][b][lane];
        Vec<V> Fw, Uw;
        Fw.v[0] = m.x; Fw.v[V - 1] = m.y; Uw.v[0] = m.z; Uw.v[V - 1] = m.w;
        if (b == rank) enter = carry;
        carry = sm.tile_starts[buf][b] != 0 ? Uw : fma(Fw, carry, Uw);
      }
      h = cut ? Ub : fma(Fb, enter, Ub);
    }
    if (p.tiles != nullptr && warp % (GATED_SCAN_TILE / S) == 0 && mine && n > 0) {
#pragma unroll
      for (int k = 0; k < V; k++) p.tiles[(t0 / GATED_SCAN_TILE) * p.C + c + k] = h.v[k];
    }
    Tokens& y = slice(slot, 0);
    T* out = reinterpret_cast<T*>(p.out) + t0 * p.ldo + c;
    auto token = [&](int s) {
      if constexpr (ASYNC) y.row[s][lane] = pack<T, V>(h.v);
      else if (mine) *out = from_float<T>(h.v[0]);
      out += p.ldo;
    };
    if (!begins && n == S) {
#pragma unroll
      for (int s = 0; s < S; s++) {
        h = fma(f[s], h, u[s]);
        token(s);
      }
    } else {
#pragma unroll
      for (int s = 0; s < S; s++) {
        if (s < n) {
          if (begins && next <= t0 + s) {            // one of the entries may be this token
            const int q = lower(p.seq, j, p.seq.N + 1, t0 + s);
            if (q <= p.seq.N && cu_at(p.seq, q) == t0 + s) finish<V>(p, q, t0 + s, false, c, mine, h.v[0], h.v[V - 1]);
          }
          h = pick(starts >> s & 1, u[s], fma(f[s], h, u[s]));
          token(s);
        }
      }
    }
    if constexpr (ASYNC) {
      __syncwarp();
      y.store(p.out, p.ldo, t0, n, c0, p.C);
    }
    if (!rejected && ((n > 0 && t0 + n == end) || (end == 0 && t0 == 0))) finish<V>(p, lower(p.seq, j, p.seq.N + 1, end), end, false, c, mine, h.v[0], h.v[V - 1]);
    t0 += step;
    slot = slot == DEPTH - 1 ? 0 : slot + 1;
  }
  if (rejected && rank == 0 && warp == 0) finish<V>(p, 1, 0, true, c, mine, 0.0f, 0.0f);
  if (rejected || p.zero_pad) zero_rest<T, V>(p.out, p.ldo, end, p.seq.T, c, mine, rank, size);
}

template <typename T, bool ASYNC, bool POWER, bool GATED>
cudaError_t launch_gates(const GatedScanParams& p, cudaStream_t stream) {
  constexpr int V = CHANNELS<T, ASYNC>, S = TOKENS<T, ASYNC>;
  const long long slabs = (p.C + 32 * V - 1) / (32 * V);
  return launch_clusters(kda_gated_scan_kernel<T, ASYNC, POWER, GATED>, p, slabs, cluster_of(slabs, p.seq.T, WARPS * S),
                         ASYNC ? DEPTH * WARPS * (GATED ? 3 : 2) * (int)sizeof(Slice<T, S>) : 0, stream);
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

// VEC channels a thread, up to STEP_ROWS rows a block; the rows' states and tokens are asked for before repeats are looked for.
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
    k_[k] = POWER && mine ? decay_factor<T>(p.rate, c + k, p.rate_scale) : 0.0f;
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
