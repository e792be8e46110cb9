// Gated linear recurrence over packed sequences, gradients (formulas and layout of the forward pass: kda_gscan.cuh).  With dh[t] the
// gradient of h[t] and e[t] = f[t] dh[t] what flows on to the token in front:
//   dh[t] = dy[t] + e[t+1]   (behind a sequence's last token: the gradient of its final state);   e[first] = gradient of the initial state
//   b = dh g x:   dx = dh gain g,   di = b gain (1 - g)
//   rate given:   dr = (dh h[t-1] f l - b f^2 l / gain) (1 - s),  drate = sum (the same without 1 - s) sigmoid(rate) / softplus(rate)
//   without:      dr = (dh h[t-1] - b) s (1 - s)
// e runs backwards over the rounds by the same maps as h does forwards (e in front of a slice = F e behind it + G).  The states h
// are computed again from those that the forward pass kept in front of each tile, inside the block, at the same barrier.  A cluster
// has all tokens of its channels, so the sums over tokens are complete in its first block, always in the same order.
#include "kda_gscan.cuh"

namespace kda {

namespace {

using namespace gscan;

constexpr int DEPTH = 2;                 // rounds of tokens on their way or worked on
constexpr int S = 8, TILE = WARPS * S;   // tokens of a slice, of a block
static_assert(TILE == GATED_SCAN_TILE, "the forward pass keeps the states in front of the tiles");

template <int V>
struct Shared {
  Vec<4> map[2][WARPS][V][32];           // {F, U, G, -} of a channel
  float4 tile[2][MAX_CLUSTER][32];       // of the cluster's tiles, written by their blocks: {F, F, G, G}
  uint32_t starts[2][WARPS], tile_starts[2][MAX_CLUSTER];
  float tile_sums[3][MAX_CLUSTER][V][32];
};

template <typename T, bool ASYNC, bool POWER, bool GATED>
__global__ void __launch_bounds__(THREADS, 2) kda_gated_scan_grad_kernel(const __grid_constant__ GatedScanGradParams p) {
  constexpr int V = CHANNELS<T, ASYNC>, NT = GATED ? 4 : 3;
  __shared__ Shared<V> sm;
  extern __shared__ __align__(128) unsigned char raw[];              // ASYNC: [DEPTH][WARPS][NT] slices
  using Tokens = Slice<T, S>;
  const uint32_t rank = cluster_rank(), size = cluster_size();
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int c0 = (int)(blockIdx.x / size) * 32 * V, c = c0 + lane * V;
  const bool mine = c < p.C;
  if (size > 1) cluster_arrive();
  const bool rejected = cu_rejected(p.seq);
  const long long end = rejected ? 0 : cu_at(p.seq, p.seq.N);
  const long long step = (long long)size * TILE;
  const int rounds = (int)((end + step - 1) / step);

  long long t0 = (rounds - 1) * step + (long long)rank * TILE + warp * S;
  Registers<T, S> nx, nr, ni, nd;
  Vec<V> next_enter = vec<V>(0.0f);
  auto slice = [&](int slot, int k) -> Tokens& { return reinterpret_cast<Tokens*>(raw)[(slot * WARPS + warp) * NT + k]; };
  auto ask = [&](int ahead, int slot) {              // the tokens of a later round, which lie in front of this one's
    const long long t = t0 - ahead * step;
    const int m = t >= 0 ? count<S>(t, end) : 0;
    if constexpr (ASYNC) {
      if (m > 0) {
        slice(slot, 0).ask(p.x, p.ldx, t, m, c0, p.C);
        slice(slot, 1).ask(p.r, p.ldr, t, m, c0, p.C);
        if (p.dy != nullptr) slice(slot, 2).ask(p.dy, p.lddy, t, m, c0, p.C);
        if (GATED) slice(slot, 3).ask(p.i, p.ldi, t, m, c0, p.C);
      }
      copies_commit();
    } else if (m > 0) {
      nx.ask(p.x, p.ldx, t, m, c, p.C);
      nr.ask(p.r, p.ldr, t, m, c, p.C);
      if (p.dy != nullptr) nd.ask(p.dy, p.lddy, t, m, c, p.C);
      if (GATED) ni.ask(p.i, p.ldi, t, m, c, p.C);
    }
  };
  auto ask_state = [&](int ahead) {                  // the state in front of the tile
    const long long t = t0 - ahead * step;
#pragma unroll
    for (int k = 0; k < V; k++)
      if (mine && t >= 0 && t < end) next_enter.v[k] = p.tiles[t / TILE * p.C + c + k];
  };
#pragma unroll
  for (int k = 0; k < (ASYNC ? DEPTH - 1 : 1); k++) ask(k, k);
  ask_state(0);
  Vec<V> rb, ib, k_;
#pragma unroll
  for (int k = 0; k < V; k++) {
    rb.v[k] = mine ? bias_of<T>(p.r_bias, c + k) : 0.0f;
    ib.v[k] = GATED && mine ? bias_of<T>(p.i_bias, c + k) : 0.0f;
    k_.v[k] = POWER && mine ? decay_factor<T>(p.rate, c + k, p.rate_scale) : 0.0f;
  }
  // the gradients of empty sequences' states pass through; a rejected layout has no others
  if (p.dsrc != nullptr && rank == 0) {
    for (int q = warp; q < p.seq.N; q += WARPS) {
      if (!rejected && cu_at(p.seq, q) != cu_at(p.seq, q + 1)) continue;
#pragma unroll
      for (int k = 0; k < V; k++)
        if (mine) p.dsrc[(long long)q * p.C + c + k] = p.dfinal != nullptr ? p.dfinal[(long long)q * p.C + c + k] : 0.0f;
    }
  }
  int j = p.seq.N + 1;                               // first entry of cu_seqlens that is >= t0, once looked for
  long long below = NEVER;                           // the entry in front of that one
  Vec<V> carry = vec<V>(0.0f), sum_rate = vec<V>(0.0f), sum_r = vec<V>(0.0f), sum_i = vec<V>(0.0f);
  if (size > 1) cluster_wait();

  int slot = 0;
  for (int round = rounds - 1; round >= 0; round--) {
    const int buf = round & 1, n = count<S>(t0, end);
    // entries in [t0, t0 + n]: sequences end in front of them or start there
    bool touched = false;
    if (below >= t0) {
      j = lower(p.seq, 0, j, t0);
      below = j > 0 ? cu_at(p.seq, j - 1) : -1;
      touched = n > 0 && j <= p.seq.N && cu_at(p.seq, j) <= t0 + n;
    }
    Registers<T, S> rx, rr, ri, rd;
    if constexpr (ASYNC) {
      copies_wait<DEPTH - 2>();
      __syncwarp();
      ask(DEPTH - 1, slot == 0 ? DEPTH - 1 : slot - 1);
    } else {
      rx = nx; rr = nr; ri = ni; rd = nd;
      ask(1, 0);
    }
    Vec<V> enter = next_enter;
    ask_state(1);
    auto token = [&](int k, int s) {                 // 0: x, 1: r, 2: dy, 3: i
      if constexpr (ASYNC) return values(slice(slot, k).row[s][lane]);
      else return vec<V>(to_float(k == 0 ? rx.row[s] : k == 1 ? rr.row[s] : k == 2 ? rd.row[s] : ri.row[s]));
    };
    Vec<V> f[S], u[S], d[S];                         // u: terms, then states in front of the tokens
#pragma unroll
    for (int s = 0; s < S; s++) {
      const Gates<V> a = decay<T, POWER, V>(token(1, s), rb, k_);
      f[s] = a.f;
      u[s] = mul(a.gain, token(0, s));
      if constexpr (GATED) {
        Vec<V> g, ng;
        sigmoids<T, V>(token(3, s), ib, g, ng);
        u[s] = mul(u[s], g);
      }
      d[s] = p.dy != nullptr ? token(2, s) : vec<V>(0.0f);
    }
    if (n < S) {
#pragma unroll
      for (int s = 0; s < S; s++)
        if (s >= n) { f[s] = vec<V>(1.0f); u[s] = d[s] = vec<V>(0.0f); }
    }
    // a sequence's final state is its last token's: so is the gradient
    uint32_t starts = 0;
    if (touched) {
      for (int q = j; q <= p.seq.N; q++) {
        const long long t = cu_at(p.seq, q);
        if (t > t0 + n) break;
        const int at = (int)(t - t0);
        if (q > 0 && at > 0 && p.dfinal != nullptr && cu_at(p.seq, q - 1) < t) {
          Vec<V> v = vec<V>(0.0f);
#pragma unroll
          for (int k = 0; k < V; k++)
            if (mine) v.v[k] = p.dfinal[(long long)(q - 1) * p.C + c + k];
#pragma unroll
          for (int s = 0; s < S; s++)
            if (s + 1 == at) d[s] = add(d[s], v);
        }
        if (at < n && q < p.seq.N && cu_at(p.seq, q + 1) > t) starts |= 1u << at;
      }
    }
    auto entering = [&](int at, Vec<V>& h) {         // the initial state of the sequence that starts at that token
      int q = lower(p.seq, j, p.seq.N + 1, t0 + at);
      while (cu_at(p.seq, q + 1) == t0 + at) q++;
#pragma unroll
      for (int k = 0; k < V; k++) h.v[k] = mine && p.src != nullptr ? p.src[(long long)q * p.C + c + k] : 0.0f;
      return q;
    };
    // the slice's maps, forwards and backwards
    Vec<V> F = vec<V>(1.0f), U = vec<V>(0.0f), G = vec<V>(0.0f);
#pragma unroll
    for (int s = 0; s < S; s++) {
      if (starts >> s & 1) entering(s, U);
      U = fma(f[s], U, u[s]);
      F = mul(F, f[s]);
    }
#pragma unroll
    for (int s = S - 1; s >= 0; s--) {
      G = mul(f[s], add(d[s], G));
      if (starts >> s & 1) G = vec<V>(0.0f);
    }
    F = least(F);
#pragma unroll
    for (int k = 0; k < V; k++) sm.map[buf][warp][k][lane] = {F.v[k], U.v[k], G.v[k], 0.0f};
    if (lane == 0) sm.starts[buf][warp] = starts;
    const bool some = __syncthreads_or(starts != 0);
    auto slice_map = [&](int w, Vec<V>& Fw, Vec<V>& Uw, Vec<V>& Gw) {
#pragma unroll
      for (int k = 0; k < V; k++) {
        const Vec<4> m = sm.map[buf][w][k][lane];
        Fw.v[k] = m.v[0]; Uw.v[k] = m.v[1]; Gw.v[k] = m.v[2];
      }
    };
    Vec<V> h = enter, Fb = vec<V>(1.0f), Gb = vec<V>(0.0f);
    bool cut = false;
#pragma unroll
    for (int w = 0; w < WARPS; w++) {
      if (w >= warp) break;
      Vec<V> Fw, Uw, Gw;
      slice_map(w, Fw, Uw, Gw);
      h = some && sm.starts[buf][w] != 0 ? Uw : fma(Fw, h, Uw);
    }
#pragma unroll
    for (int w = WARPS - 1; w > 0; w--) {
      if (w <= warp) break;
      Vec<V> Fw, Uw, Gw;
      slice_map(w, Fw, Uw, Gw);
      const bool constant = some && sm.starts[buf][w] != 0;
      cut |= constant;
      Gb = constant ? Gw : fma(Fw, Gb, Gw);
      Fb = least(mul(Fb, Fw));
    }
    Vec<V> e;                                        // what flows into the slice from behind
    if (size == 1) {
      e = cut ? Gb : fma(Fb, carry, Gb);
      carry = e;
#pragma unroll
      for (int w = WARPS - 1; w >= 0; w--) {
        if (w > warp) continue;
        Vec<V> Fw, Uw, Gw;
        slice_map(w, Fw, Uw, Gw);
        carry = some && sm.starts[buf][w] != 0 ? Gw : fma(Fw, carry, Gw);
      }
    } else {
      if (warp == 0) {                               // it has the tile's map: to every block of the cluster
        const Vec<V> Gt = starts ? G : fma(F, Gb, G), Ft = least(mul(Fb, F));
        for (uint32_t b = 0; b < size; b++) put_remote(&sm.tile[buf][rank][lane], b, make_float4(Ft.v[0], Ft.v[V - 1], Gt.v[0], Gt.v[V - 1]));
        if (lane < size) put_remote(&sm.tile_starts[buf][rank], lane, (uint32_t)(cut || starts != 0));
      }
      cluster_arrive();
      cluster_wait();
      Vec<V> behind = carry;
#pragma unroll
      for (int b = MAX_CLUSTER - 1; b >= 0; b--) {
        if (b >= size) continue;
        const float4 m = sm.tile[buf][b][lane];
        Vec<V> Fw, Gw;
        Fw.v[0] = m.x; Fw.v[V - 1] = m.y; Gw.v[0] = m.z; Gw.v[V - 1] = m.w;
        if (b == rank) behind = carry;
        carry = sm.tile_starts[buf][b] != 0 ? Gw : fma(Fw, carry, Gw);
      }
      e = cut ? Gb : fma(Fb, behind, Gb);
    }
    // the states in front of the tokens
#pragma unroll
    for (int s = 0; s < S; s++) {
      if (starts >> s & 1) entering(s, h);
      const Vec<V> before = h;
      h = fma(f[s], h, u[s]);
      u[s] = before;
    }
    T* dx = reinterpret_cast<T*>(p.dx) + (t0 + n - 1) * p.lddx + c;
    T* dr = reinterpret_cast<T*>(p.dr) + (t0 + n - 1) * p.lddr + c;
    T* di = reinterpret_cast<T*>(p.di) + (t0 + n - 1) * p.lddi + c;
#pragma unroll
    for (int s = S - 1; s >= 0; s--) {
      if (s >= n) continue;
      const Gates<V> a = decay<T, POWER, V>(token(1, s), rb, k_);
      const Vec<V> dh = add(d[s], e);
      Vec<V> b = mul(dh, token(0, s)), gx = mul(dh, a.gain), gr, gi = vec<V>(0.0f);
      if constexpr (GATED) {
        Vec<V> g, ng;
        sigmoids<T, V>(token(3, s), ib, g, ng);
        b = mul(b, g);
        gx = mul(gx, g);
        gi = mul(mul(b, a.gain), ng);
        sum_i = add(sum_i, gi);
      }
      if constexpr (POWER) {
        const Vec<V> l = sizeof(T) == 4 ? a.l : mul(a.l, vec<V>(LN2_F));
        // f (dh h l - b f (l / gain))
        const Vec<V> m = mul(a.f, fma(mul(dh, u[s]), l, mul(mul(mul(b, vec<V>(-1.0f)), a.f), mul(l, a.inv))));
        gr = mul(m, a.n);
        sum_rate = add(sum_rate, m);
      } else {
        gr = mul(fma(dh, u[s], mul(b, vec<V>(-1.0f))), mul(a.s, a.n));
      }
      sum_r = add(sum_r, gr);
      e = mul(a.f, dh);
      if constexpr (ASYNC) {                         // in the places of the inputs that they are the gradients of
        slice(slot, 0).row[s][lane] = pack<T, V>(gx.v);
        slice(slot, 1).row[s][lane] = pack<T, V>(gr.v);
        if (GATED) slice(slot, 3).row[s][lane] = pack<T, V>(gi.v);
      } else {
        if (mine) {
          *dx = from_float<T>(gx.v[0]);
          *dr = from_float<T>(gr.v[0]);
          if (GATED) *di = from_float<T>(gi.v[0]);
        }
        dx -= p.lddx;
        dr -= p.lddr;
        if (GATED) di -= p.lddi;
      }
      if (starts >> s & 1) {
        Vec<V> unused;
        const int q = entering(s, unused);
#pragma unroll
        for (int k = 0; k < V; k++)
          if (p.dsrc != nullptr && mine) p.dsrc[(long long)q * p.C + c + k] = e.v[k];
        e = vec<V>(0.0f);
      }
    }
    if constexpr (ASYNC) {
      __syncwarp();
      slice(slot, 0).store(p.dx, p.lddx, t0, n, c0, p.C);
      slice(slot, 1).store(p.dr, p.lddr, t0, n, c0, p.C);
      if (GATED) slice(slot, 3).store(p.di, p.lddi, t0, n, c0, p.C);
    }
    t0 -= step;
    slot = slot == DEPTH - 1 ? 0 : slot + 1;
  }
  zero_rest<T, V>(p.dx, p.lddx, end, p.seq.T, c, mine, rank, size);
  zero_rest<T, V>(p.dr, p.lddr, end, p.seq.T, c, mine, rank, size);
  if (GATED) zero_rest<T, V>(p.di, p.lddi, end, p.seq.T, c, mine, rank, size);

  // sums over the tokens: of the warps (in the places of the maps), then of the cluster's blocks
  __syncthreads();
#pragma unroll
  for (int k = 0; k < V; k++) sm.map[0][warp][k][lane] = {sum_rate.v[k], sum_r.v[k], sum_i.v[k], 0.0f};
  __syncthreads();
  float total[V];
  if (warp < 3) {
#pragma unroll
    for (int k = 0; k < V; k++) {
      total[k] = 0.0f;
      for (int w = 0; w < WARPS; w++) total[k] += sm.map[0][w][k][lane].v[warp];
      if (size > 1) put_remote(&sm.tile_sums[warp][rank][k][lane], 0, total[k]);
    }
  }
  if (size > 1) {
    cluster_arrive();
    cluster_wait();
  }
  if (rank == 0 && warp < 3 && mine) {
    float* to = warp == 0 ? p.drate : (warp == 1 ? p.dr_bias : p.di_bias);
    if (to == nullptr) return;
#pragma unroll
    for (int k = 0; k < V; k++) {
      if (size > 1) {
        total[k] = 0.0f;
        for (uint32_t b = 0; b < size; b++) total[k] += sm.tile_sums[warp][b][k][lane];
      }
      if (warp == 0) {
        const float v = p.rate[c + k], soft = softplus_exact(v);
        total[k] *= soft > 0.0f ? 1.0f / (1.0f + expf(-v)) / soft : 1.0f;      // 1 in the limit of low rates
      }
      to[c + k] = total[k];
    }
  }
}

template <typename T, bool ASYNC, bool POWER, bool GATED>
cudaError_t launch_gates(const GatedScanGradParams& p, cudaStream_t stream) {
  constexpr int V = CHANNELS<T, ASYNC>;
  const long long slabs = (p.C + 32 * V - 1) / (32 * V);
  return launch_clusters(kda_gated_scan_grad_kernel<T, ASYNC, POWER, GATED>, p, slabs, cluster_of(slabs, p.seq.T, TILE),
                         ASYNC ? DEPTH * WARPS * (GATED ? 4 : 3) * (int)sizeof(Slice<T, S>) : 0, stream);
}

template <typename T, bool ASYNC>
cudaError_t launch_form(const GatedScanGradParams& p, cudaStream_t stream) {
  if (p.rate != nullptr) return p.i != nullptr ? launch_gates<T, ASYNC, true, true>(p, stream) : launch_gates<T, ASYNC, true, false>(p, stream);
  return p.i != nullptr ? launch_gates<T, ASYNC, false, true>(p, stream) : launch_gates<T, ASYNC, false, false>(p, stream);
}

template <typename T>
cudaError_t launch_type(const GatedScanGradParams& p, cudaStream_t stream) {
  const int size = sizeof(T);
  const bool async = p.C % (16 / size) == 0 && rows_on(p.x, p.ldx, size, 16) && rows_on(p.r, p.ldr, size, 16) && rows_on(p.i, p.ldi, size, 16) &&
                     rows_on(p.dy, p.lddy, size, 16) && rows_on(p.dx, p.lddx, size, 16) && rows_on(p.dr, p.lddr, size, 16) && rows_on(p.di, p.lddi, size, 16);
  return async ? launch_form<T, true>(p, stream) : launch_form<T, false>(p, stream);
}

}  // namespace

cudaError_t launch_gated_scan_grad(const GatedScanGradParams& p, int type, cudaStream_t stream) {
  if (type == TYPE_BF16) return launch_type<__nv_bfloat16>(p, stream);
  if (type == TYPE_FP16) return launch_type<__half>(p, stream);
  return launch_type<float>(p, stream);
}

}  // namespace kda
