// Gated linear recurrence over packed sequences, gradients (formulas and layout of the forward pass: kda_gscan.cuh).  With dh[t] the
// gradient of h[t] and e[t] = f[t] dh[t] what flows on to the token in front:
//   dh[t] = dy[t] + e[t+1]   (behind a sequence's last token: the gradient of its final state);   e[first] = gradient of the initial state
//   b = dh g x:   dx = dh gain g,   di = b gain (1 - g)
//   rate given:   dr = (dh h[t-1] f l - b f^2 l / gain) (1 - s),  drate = sum (the same without 1 - s) sigmoid(rate) / softplus(rate)
//   without:      dr = (dh h[t-1] - b) s (1 - s)
// e runs backwards over the rounds by the same maps as h does forwards (e in front of a slice = F e behind it + G).  The states h
// are computed again from those that the forward pass kept in front of each tile, inside the block, at the same barrier.  A cluster
// has all tokens of its channels, so the sums over tokens are complete in its first block, always in the same order.
// The gates are computed twice, once for the maps and once for the gradients: kept in registers, they would take 48 more.  (In shared memory
// they would fit; that is not done.)  The kernel for fp32 tokens read one by one, with rate and input gate, spills 4 bytes, the others none.
// Measured in bf16, both gates: 8 ragged sequences, 10 245 tokens of 4096 channels, 271 us (2.2 TB/s); 8192 tokens in one sequence 199 us, with
// 4095 channels 300, in fp32 292; 16 384 tokens of 512 channels in fp32, the form without rate, 94 us.  Slices of 12 tokens (twice the code): 325 us
// for the first.
#include "kda_gscan.cuh"

namespace kda {

namespace {

using namespace gscan;

constexpr int WARPS = 8, THREADS = WARPS * 32;
constexpr int DEPTH = 2;                 // rounds of tokens on their way or worked on
constexpr int S = 6, TILE = WARPS * S;   // tokens of a slice, of a block
static_assert(TILE == GATED_SCAN_TILE, "the forward pass keeps the states in front of the tiles");

// With 48 KB of tokens (16 bits, both gates) and 16 KB of tiles (16 blocks a cluster) some 77 KB a block: two an SM leave 36 KB each.
template <int V>
struct Shared {
  Vec<V> F[2][WARPS][32], U[2][WARPS][32], G[2][WARPS][32];          // the maps of the block's slices
  unsigned long long sent[2];            // barriers: the tiles' maps have arrived
  uint32_t cuts[2][WARPS];               // tokens that start a sequence, from bit 16 on those that end one: the maps are constant
  Tables<false> tables;
};
using Tile = float4[32];                 // of the cluster's tiles, sent by their blocks: {F, F, G, G}; F < 0: the map is constant

struct Steps {             // bytes from a row to the fourth behind it
  long long x, r, i, d, dx, dr, di;
};

// The row [N][C] of a table that belongs to the sequence of token t; zeros without a table.  Not inlined: its two dozen places in the
// kernel would not fit the instruction cache.
__device__ __noinline__ float2 state_of(const float* table, const Layout<false> l, uint32_t t, int C, int c, bool mine, int channels) {
  float2 h = make_float2(0.0f, 0.0f);
  if (table == nullptr) return h;
  const int q = lower(l, 0, l.s.N + 1, t + 1) - 1;
  const float* row = table + (long long)q * C + c;
  if (mine) {
    h.x = row[0];
    if (channels > 1) h.y = row[1];
  }
  return h;
}

template <typename T, bool ASYNC, bool POWER, bool GATED>
__global__ void __launch_bounds__(THREADS, 2) kda_gated_scan_grad_kernel(const __grid_constant__ GatedScanGradParams p, const __grid_constant__ Steps g) {
  constexpr int V = CHANNELS<T, ASYNC>, NT = GATED ? 4 : 3;
  using Tokens = Slice<T, S>;
  constexpr int RAW = ASYNC ? DEPTH * WARPS * NT * (int)sizeof(Tokens) : 0;
  __shared__ Shared<V> sm;
  extern __shared__ __align__(128) unsigned char raw[];              // ASYNC: [DEPTH][WARPS][NT] slices; then [2][blocks of the cluster] tiles
  const uint32_t rank = cluster_rank(), size = cluster_size();
  Tile* const tiles = reinterpret_cast<Tile*>(raw + RAW);
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int c0 = (int)(blockIdx.x / size) * 32 * V, c = c0 + lane * V;
  const bool mine = c < p.C, chunk = c0 + lane % 8 * (16 / (int)sizeof(T)) < p.C;
  if (threadIdx.x == 0)
    for (int b = 0; b < 2; b++) bar_init(&sm.sent[b]);
  if (size > 1) cluster_arrive();
  const bool rejected = cu_rejected(p.seq);
  const Layout<false> tables = rejected ? Layout<false>{p.seq, nullptr} : layout_of(p.seq, sm.tables);
  const uint32_t end = rejected ? 0 : (uint32_t)cu_at(p.seq, p.seq.N);
  const uint32_t step = size * TILE;
  const int rounds = (int)(((long long)end + step - 1) / step);
  __syncthreads();                                   // the copies of the tables

  uint32_t t0 = (uint32_t)(rounds - 1) * step + rank * TILE + warp * S;        // not used without rounds
  Registers<T, S> rx, rr, ri, rd;
  Vec<V> next_enter = vec<V>(0.0f);
  auto slice = [&](int slot, int k) -> Tokens& { return reinterpret_cast<Tokens*>(raw)[(slot * WARPS + warp) * NT + k]; };
  auto ask = [&](int round, int slot) {              // the tokens of a round
    const uint32_t t = (uint32_t)round * step + rank * TILE + warp * S;
    const int m = round >= 0 ? count<S>(t, end) : 0;
    if constexpr (ASYNC) {
      if (m > 0) {
        Cursor<T, S>(p.x, p.ldx, t, c0).ask(slice(slot, 0), g.x, m, chunk, p.x);
        Cursor<T, S>(p.r, p.ldr, t, c0).ask(slice(slot, 1), g.r, m, chunk, p.r);
        if (p.dy != nullptr) Cursor<T, S>(p.dy, p.lddy, t, c0).ask(slice(slot, 2), g.d, m, chunk, p.dy);
        if (GATED) Cursor<T, S>(p.i, p.ldi, t, c0).ask(slice(slot, 3), g.i, m, chunk, p.i);
      }
      copies_commit();
    } else if (m > 0) {
      rx.ask(p.x, p.ldx, t, m, c, p.C);
      rr.ask(p.r, p.ldr, t, m, c, p.C);
      if (p.dy != nullptr) rd.ask(p.dy, p.lddy, t, m, c, p.C);
      if (GATED) ri.ask(p.i, p.ldi, t, m, c, p.C);
    }
#pragma unroll
    for (int k = 0; k < V; k++)                      // the state in front of the tile
      if (mine && m > 0) next_enter.v[k] = p.tiles[(long long)(t / TILE) * p.C + c + k];
  };
  ask(rounds - 1, 0);
  Vec<V> rb, ib, k_;
#pragma unroll
  for (int k = 0; k < V; k++) {
    rb.v[k] = mine ? bias_of<T>(p.r_bias, c + k) : 0.0f;
    ib.v[k] = GATED && mine ? bias_of<T>(p.i_bias, c + k) : 0.0f;
    k_.v[k] = POWER && mine ? decay_factor(p.rate, c + k, p.rate_scale) : 0.0f;
  }
  // the gradients of empty sequences' states pass through; a rejected layout has no others
  if (p.dsrc != nullptr && rank == 0) {
    for (int q = warp; q < p.seq.N; q += WARPS) {
      if (!rejected && tables.at(q) != tables.at(q + 1)) continue;
#pragma unroll
      for (int k = 0; k < V; k++)
        if (mine) p.dsrc[(long long)q * p.C + c + k] = p.dfinal != nullptr ? p.dfinal[(long long)q * p.C + c + k] : 0.0f;
    }
  }
  auto state = [&](const float* table, uint32_t t) {
    Vec<V> h;
    const float2 v = state_of(table, tables, t, p.C, c, mine, V);
    h.v[0] = v.x;
    h.v[V - 1] = V > 1 ? v.y : v.x;
    return h;
  };
  uint32_t below = NEVER;                            // the last entry of cu_seqlens in front of the slices that are done
  Vec<V> carry = vec<V>(0.0f), sum_rate = vec<V>(0.0f), sum_r = vec<V>(0.0f), sum_i = vec<V>(0.0f);
  bool lost = false;
  if (size > 1) cluster_wait();

  for (int round = rounds - 1; round >= 0; round--, t0 -= step) {
    const int use = rounds - 1 - round, buf = use & 1, n = count<S>(t0, end);
    if (size > 1 && threadIdx.x == 0 && !lost) bar_expect(&sm.sent[buf], (size + p.more_maps) * 512);
    Vec<V> h = next_enter;
    if constexpr (ASYNC) {
      copies_wait<0>();
      __syncwarp();
      ask(round - 1, buf ^ 1);
    }
    // entries in [t0, t0 + n]: sequences start there, or end in front of them
    uint32_t starts = 0, ends = 0;
    if (below >= t0) {
      const int j = lower(tables, 0, p.seq.N + 1, t0);
      below = j > 0 ? tables.at(j - 1) : 0;
      if (j == 0) below = 0;
      for (int q = j; q <= p.seq.N; q++) {
        const uint32_t t = tables.at(q);
        if (t > t0 + n) break;
        if (t < t0 + n) starts |= 1u << (t - t0);
        if (t > t0) ends |= 1u << (t - t0 - 1);
      }
    }
    auto token = [&](int k, int s) {                 // 0: x, 1: r, 2: dy, 3: i
      if constexpr (ASYNC) return values(slice(buf, k).row[s][lane]);
      else return vec<V>(to_float(k == 0 ? rx.row[s] : k == 1 ? rr.row[s] : k == 2 ? rd.row[s] : ri.row[s]));
    };
    auto gradient = [&](int s) { return p.dy != nullptr ? token(2, s) : vec<V>(0.0f); };
    Vec<V> f[S], u[S];                               // decays; terms, then states in front of the tokens
#pragma unroll
    for (int s = 0; s < S; s++) token_terms<T, POWER, GATED, V>(token(0, s), token(1, s), token(3, s), rb, ib, k_, f[s], u[s]);
    // the slice's maps, forwards and backwards
    const bool plain = n == S && (starts | ends) == 0;
    Vec<V> F = f[0], U = u[0], G;
    if (plain) {
#pragma unroll
      for (int s = 1; s < S; s++) {
        U = fma(f[s], U, u[s]);
        F = mul(F, f[s]);
      }
      G = mul(f[S - 1], gradient(S - 1));
#pragma unroll
      for (int s = S - 2; s >= 0; s--) G = mul(f[s], add(gradient(s), G));
    } else {
      F = vec<V>(1.0f);
      U = G = vec<V>(0.0f);
#pragma unroll
      for (int s = 0; s < S; s++) {
        if (s >= n) { f[s] = vec<V>(1.0f); u[s] = vec<V>(0.0f); }
        if (starts >> s & 1) U = state(p.src, t0 + s);
        U = fma(f[s], U, u[s]);
        F = mul(F, f[s]);
      }
#pragma unroll
      for (int s = S - 1; s >= 0; s--) {
        if (ends >> s & 1) G = state(p.dfinal, t0 + s);
        if (s < n) G = mul(f[s], add(gradient(s), G));
      }
    }
    F = least(F);
    sm.F[buf][warp][lane] = F;
    sm.U[buf][warp][lane] = U;
    sm.G[buf][warp][lane] = G;
    if (lane == 0) sm.cuts[buf][warp] = starts | ends << 16;
    const bool some = __syncthreads_or((starts | ends) != 0);
    Vec<V> Fb = vec<V>(1.0f), Gb = vec<V>(0.0f);
    bool cut = false;
#pragma unroll
    for (int w = WARPS - 1; w > 0; w--) {
      if (w <= warp) break;
      const Vec<V> Fw = sm.F[buf][w][lane], Gw = sm.G[buf][w][lane];
      Gb = fma(Fw, Gb, Gw);
      Fb = mul(Fb, Fw);
      if (some && sm.cuts[buf][w] >> 16 != 0) {
        cut = true;
        Gb = Gw;
      }
    }
    Fb = least(Fb);
    Vec<V> e = carry;                                // what flows into the slice from behind
    if (size == 1) {
#pragma unroll
      for (int w = WARPS - 1; w >= 0; w--) {
        const Vec<V> Fw = sm.F[buf][w][lane], Gw = sm.G[buf][w][lane];
        carry = fma(Fw, carry, Gw);
        if (some && sm.cuts[buf][w] >> 16 != 0) carry = Gw;
      }
    } else if (warp == 0 && !lost) {                 // it has the tile's map: to every block of the cluster
      const Vec<V> Gt = ends ? G : fma(F, Gb, G);
      Vec<V> Ft = least(mul(Fb, F));
      if (cut || ends) Ft = vec<V>(-1.0f);
      const float4 v = make_float4(Ft.v[0], Ft.v[V - 1], Gt.v[0], Gt.v[V - 1]);
      for (uint32_t b = 0; b < size; b++) send(&tiles[buf * size + rank][lane], &sm.sent[buf], b, v);
    }
    // meanwhile the states in front of the tokens
#pragma unroll
    for (int w = 0; w < WARPS; w++) {
      if (w >= warp) break;
      const Vec<V> Uw = sm.U[buf][w][lane];
      h = fma(sm.F[buf][w][lane], h, Uw);
      if (some && (sm.cuts[buf][w] & 0xffffu) != 0) h = Uw;
    }
    if (starts == 0) {
#pragma unroll
      for (int s = 0; s < S; s++) {
        const Vec<V> before = h;
        h = fma(f[s], h, u[s]);
        u[s] = before;
      }
    } else {
#pragma unroll
      for (int s = 0; s < S; s++) {
        if (starts >> s & 1) h = state(p.src, t0 + s);
        const Vec<V> before = h;
        h = fma(f[s], h, u[s]);
        u[s] = before;
      }
    }
    if (size > 1) {
      if (!lost) lost = bar_lost(&sm.sent[buf], use >> 1 & 1, p.wait_ns);
#pragma unroll
      for (int b = MAX_CLUSTER - 1; b >= 0; b--) {
        if (b >= size) continue;
        const float4 m = tiles[buf * size + b][lane];
        Vec<V> Fw, Gw;
        Fw.v[0] = m.x; Fw.v[V - 1] = m.y; Gw.v[0] = m.z; Gw.v[V - 1] = m.w;
        if (b == rank) e = carry;
        carry = pick(m.x < 0.0f, Gw, fma(Fw, carry, Gw));
      }
    }
    e = cut ? Gb : fma(Fb, e, Gb);
    T* dx = reinterpret_cast<T*>(p.dx) + (long long)t0 * p.lddx + c;
    T* dr = reinterpret_cast<T*>(p.dr) + (long long)t0 * p.lddr + c;
    T* di = reinterpret_cast<T*>(p.di) + (long long)t0 * p.lddi + c;
    auto gradients = [&](int s) {
      const Vec<V> dh = add(gradient(s), e), x = token(0, s);
      const Gates<V> a = decay<T, POWER, V, true>(token(1, s), rb, k_);
      e = mul(f[s], dh);
      Vec<V> b = mul(dh, x), gx = mul(dh, a.gain), gr, gi = vec<V>(0.0f);
      if constexpr (GATED) {
        Vec<V> gate, ng;
        sigmoids<T, V, true, true>(token(3, s), ib, gate, ng);
        b = mul(b, gate);
        gx = mul(gx, gate);
        gi = mul(mul(gx, x), ng);
        sum_i = add(sum_i, gi);
      }
      if constexpr (POWER) {
        // l to base 2, whose ln 2 joins the sum at its end: f (dh h l - b f (l / gain))
        Vec<V> m;
#pragma unroll
        for (int k = 0; k < V; k++) {
          const float w = a.l.v[k] * a.inv.v[k];
          m.v[k] = f[s].v[k] * fmaf(dh.v[k] * u[s].v[k], a.l.v[k], -(b.v[k] * f[s].v[k] * w));
          gr.v[k] = m.v[k] * (a.n.v[k] * LN2_F);
        }
        sum_rate = add(sum_rate, m);
      } else {
#pragma unroll
        for (int k = 0; k < V; k++) gr.v[k] = fmaf(dh.v[k], u[s].v[k], -b.v[k]) * (a.s.v[k] * a.n.v[k]);
      }
      sum_r = add(sum_r, gr);
      if constexpr (ASYNC) {                         // in the places of the inputs that they are the gradients of
        slice(buf, 0).row[s][lane] = pack<T, V>(gx.v);
        slice(buf, 1).row[s][lane] = pack<T, V>(gr.v);
        if (GATED) slice(buf, 3).row[s][lane] = pack<T, V>(gi.v);
      } else if (mine) {
        dx[s * p.lddx] = from_float<T>(gx.v[0]);
        dr[s * p.lddr] = from_float<T>(gr.v[0]);
        if (GATED) di[s * p.lddi] = from_float<T>(gi.v[0]);
      }
    };
    if (plain) {
#pragma unroll
      for (int s = S - 1; s >= 0; s--) gradients(s);
    } else {
#pragma unroll
      for (int s = S - 1; s >= 0; s--) {
        if (s >= n) continue;
        if (ends >> s & 1) e = state(p.dfinal, t0 + s);
        gradients(s);
        if ((starts >> s & 1) && p.dsrc != nullptr) {
          const int q = lower(tables, 0, p.seq.N + 1, t0 + s + 1) - 1;
#pragma unroll
          for (int k = 0; k < V; k++)
            if (mine) p.dsrc[(long long)q * p.C + c + k] = e.v[k];
        }
      }
    }
    if constexpr (ASYNC) {
      __syncwarp();
      Cursor<T, S>(p.dx, p.lddx, t0, c0).store(slice(buf, 0), g.dx, n, chunk);
      Cursor<T, S>(p.dr, p.lddr, t0, c0).store(slice(buf, 1), g.dr, n, chunk);
      if (GATED) Cursor<T, S>(p.di, p.lddi, t0, c0).store(slice(buf, 3), g.di, n, chunk);
    } else {
      ask(round - 1, 0);                             // with a second set of registers, a round ahead, it spilled 100 to 800 bytes
    }
  }
  if (lost) report(p.seq.status, SEQ_LOST);
  zero_rest<T, V>(p.dx, p.lddx, end, p.seq.T, c, mine, rank, size);
  zero_rest<T, V>(p.dr, p.lddr, end, p.seq.T, c, mine, rank, size);
  if (GATED) zero_rest<T, V>(p.di, p.lddi, end, p.seq.T, c, mine, rank, size);

  // sums over the tokens: of the warps (in the places of the maps), then of the cluster's blocks (in that of the tiles)
  __syncthreads();
  sm.F[0][warp][lane] = sum_rate;
  sm.U[0][warp][lane] = sum_r;
  sm.G[0][warp][lane] = sum_i;
  __syncthreads();
  if (size > 1) {                                    // no block reads tiles any more
    cluster_arrive();
    cluster_wait();
  }
  Vec<V> total = vec<V>(0.0f);
  if (warp < 3) {
    for (int w = 0; w < WARPS; w++) total = add(total, warp == 0 ? sm.F[0][w][lane] : (warp == 1 ? sm.U[0][w][lane] : sm.G[0][w][lane]));
    if (size > 1) {                                  // three rows of a block: rows 3 rank ... of the 2 size there are, of 4 values a lane
#pragma unroll
      for (int k = 0; k < V; k++) put_remote(reinterpret_cast<float*>(tiles) + ((3 * rank + warp) * V + k) * 32 + lane, 0, total.v[k]);
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
        total.v[k] = 0.0f;
        for (uint32_t b = 0; b < size; b++) total.v[k] += reinterpret_cast<const float*>(tiles)[((3 * b + warp) * V + k) * 32 + lane];
      }
      if (warp == 0) {
        const float v = p.rate[c + k], soft = softplus_exact(v);
        total.v[k] *= LN2_F * (soft > 0.0f ? 1.0f / (1.0f + expf(-v)) / soft : 1.0f);      // 1 in the limit of low rates
      }
      to[c + k] = total.v[k];
    }
  }
}

template <typename T, bool ASYNC, bool POWER, bool GATED>
cudaError_t launch_gates(const GatedScanGradParams& p, cudaStream_t stream) {
  constexpr int V = CHANNELS<T, ASYNC>, B = sizeof(T);
  const long long slabs = (p.C + 32 * V - 1) / (32 * V);
  const auto bytes = [](int size) { return (ASYNC ? DEPTH * WARPS * (GATED ? 4 : 3) * (int)sizeof(Slice<T, S>) : 0) + 2 * size * (int)sizeof(Tile); };
  const auto kernel = kda_gated_scan_grad_kernel<T, ASYNC, POWER, GATED>;
  const int size = cluster_of(kernel, slabs, p.seq.T, TILE, THREADS, bytes);
  const Steps g = {4 * p.ldx * B, 4 * p.ldr * B, 4 * p.ldi * B, 4 * p.lddy * B, 4 * p.lddx * B, 4 * p.lddr * B, 4 * p.lddi * B};
  return launch_clusters(kernel, slabs, size, THREADS, bytes(size), bytes(MAX_CLUSTER), stream, p, g);
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
