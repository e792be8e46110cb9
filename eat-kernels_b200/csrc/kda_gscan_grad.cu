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

template <int V>
struct Shared {
  float F[2][WARPS][V][32], U[2][WARPS][V][32], G[2][WARPS][V][32];
  float cF[2][MAX_CLUSTER][V][32], cG[2][MAX_CLUSTER][V][32];
  uint32_t starts[2][WARPS], c_starts[2][MAX_CLUSTER];
  float sums[3][WARPS][V][32], c_sums[3][MAX_CLUSTER][V][32];
};

template <typename T, bool WIDE, bool POWER, bool GATED>
__global__ void __launch_bounds__(THREADS, 1) kda_gated_scan_grad_kernel(const GatedScanGradParams p) {
  constexpr int V = CHANNELS<T, WIDE>;
  __shared__ Shared<V> sm;
  const uint32_t rank = cluster_rank(), size = cluster_size();
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int c = ((int)(blockIdx.x / size) * 32 + lane) * V;
  const bool mine = c < p.C;
  if (size > 1) cluster_arrive();
  const bool rejected = cu_rejected(p.seq);
  const long long end = rejected ? 0 : cu_at(p.seq, p.seq.N);
  const long long step = (long long)size * TILE;
  const long long rounds = (end + step - 1) / step;

  float rb[V], ib[V], k_[V];
#pragma unroll
  for (int k = 0; k < V; k++) {
    rb[k] = mine ? bias_of<T>(p.r_bias, c + k) : 0.0f;
    ib[k] = GATED && mine ? bias_of<T>(p.i_bias, c + k) : 0.0f;
    k_[k] = POWER && mine ? decay_factor<T>(p.rate, c + k, p.rate_scale) : 0.0f;
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
  Rows<T, V> x, r, i, dy;
  float enter[V];                                    // the state in front of the tile
  long long t0 = (rounds - 1) * step + (long long)rank * TILE + warp * S;
  int n = rounds > 0 ? count(t0, end) : 0;
  auto ask = [&](long long t, int m) {
    x.ask(p.x, p.ldx, t, m, c, mine);
    r.ask(p.r, p.ldr, t, m, c, mine);
    if (GATED) i.ask(p.i, p.ldi, t, m, c, mine);
    dy.ask(p.dy, p.lddy, t, p.dy != nullptr ? m : 0, c, mine);
#pragma unroll
    for (int k = 0; k < V; k++) enter[k] = mine && m > 0 ? p.tiles[t / TILE * p.C + c + k] : 0.0f;
  };
  ask(t0, n);
  float carry[V] = {}, sum_rate[V] = {}, sum_r[V] = {}, sum_i[V] = {};
  if (size > 1) cluster_wait();

  for (long long round = rounds - 1; round >= 0; round--) {
    const int buf = (int)(round & 1);
    float f[S][V], u[S][V], d[S][V];                 // u: terms, then states in front of the tokens
#pragma unroll
    for (int s = 0; s < S; s++) {
#pragma unroll
      for (int k = 0; k < V; k++) {
        const Gates a = decay<T, POWER>(to_float(r.v[s].v[k]), rb[k], k_[k]);
        float g = 1.0f, ng;
        if (GATED) sigmoid_pair<T>(to_float(i.v[s].v[k]), ib[k], g, ng);
        f[s][k] = a.f;
        u[s][k] = a.gain * g * to_float(x.v[s].v[k]);
        d[s][k] = to_float(dy.v[s].v[k]);
        if (s >= n) { f[s][k] = 1.0f; u[s][k] = 0.0f; d[s][k] = 0.0f; }
      }
    }
    // entries of cu_seqlens in [t0, t0 + n]: a sequence ends in front of each (the final state's gradient joins its last token's), one
    // with tokens starts there (its initial state joins the first token's term)
    uint32_t starts = 0;
    int first = 0;
    if (n > 0) {
      first = seek(p.seq, 0, t0);
      for (int q = first; q <= p.seq.N; q++) {
        const long long t = cu_at(p.seq, q);
        if (t > t0 + n) break;
        const int at = (int)(t - t0);
        if (q > 0 && at > 0 && p.dfinal != nullptr && cu_at(p.seq, q - 1) < t) {
#pragma unroll
          for (int k = 0; k < V; k++) {
            const float v = mine ? p.dfinal[(long long)(q - 1) * p.C + c + k] : 0.0f;
#pragma unroll
            for (int s = 0; s < S; s++)
              if (s + 1 == at) d[s][k] += v;
          }
        }
        if (at < n && q < p.seq.N && cu_at(p.seq, q + 1) > t) starts |= 1u << at;
      }
    }
    auto entering = [&](int at, float (&h)[V]) {     // the initial state of the sequence that starts at that token
      int q = seek(p.seq, first, t0 + at);
      while (cu_at(p.seq, q + 1) == t0 + at) q++;
#pragma unroll
      for (int k = 0; k < V; k++) h[k] = mine && p.src != nullptr ? p.src[(long long)q * p.C + c + k] : 0.0f;
      return q;
    };
    // the slice's maps, forwards and backwards
    float F[V], U[V], G[V];
#pragma unroll
    for (int k = 0; k < V; k++) F[k] = 1.0f, U[k] = G[k] = 0.0f;
#pragma unroll
    for (int s = 0; s < S; s++) {
      if (starts >> s & 1) entering(s, U);
#pragma unroll
      for (int k = 0; k < V; k++) {
        U[k] = fmaf(f[s][k], U[k], u[s][k]);
        F[k] *= f[s][k];
      }
    }
#pragma unroll
    for (int s = S - 1; s >= 0; s--) {
#pragma unroll
      for (int k = 0; k < V; k++) G[k] = starts >> s & 1 ? 0.0f : f[s][k] * (d[s][k] + G[k]);
    }
#pragma unroll
    for (int k = 0; k < V; k++) {
      F[k] = fmaxf(F[k], LEAST);
      sm.F[buf][warp][k][lane] = F[k];
      sm.U[buf][warp][k][lane] = U[k];
      sm.G[buf][warp][k][lane] = G[k];
    }
    if (lane == 0) sm.starts[buf][warp] = starts;
    __syncthreads();
    float h[V], Fb[V], Gb[V];
    uint32_t cut = 0;
#pragma unroll
    for (int k = 0; k < V; k++) { h[k] = enter[k]; Fb[k] = 1.0f; Gb[k] = 0.0f; }
    for (int w = 0; w < warp; w++) {
      const bool constant = sm.starts[buf][w] != 0;
#pragma unroll
      for (int k = 0; k < V; k++) h[k] = constant ? sm.U[buf][w][k][lane] : fmaf(sm.F[buf][w][k][lane], h[k], sm.U[buf][w][k][lane]);
    }
    for (int w = WARPS - 1; w > warp; w--) {
      const bool constant = sm.starts[buf][w] != 0;
      cut |= constant;
#pragma unroll
      for (int k = 0; k < V; k++) {
        const float Fw = sm.F[buf][w][k][lane], Gw = sm.G[buf][w][k][lane];
        Gb[k] = constant ? Gw : fmaf(Fw, Gb[k], Gw);
        Fb[k] = fmaxf(Fb[k] * Fw, LEAST);
      }
    }
    float e[V];                                      // what flows into the slice from behind
    if (size == 1) {
#pragma unroll
      for (int k = 0; k < V; k++) {
        e[k] = cut ? Gb[k] : fmaf(Fb[k], carry[k], Gb[k]);
        carry[k] = e[k];
      }
      for (int w = warp; w >= 0; w--) {
        const bool constant = sm.starts[buf][w] != 0;
#pragma unroll
        for (int k = 0; k < V; k++) carry[k] = constant ? sm.G[buf][w][k][lane] : fmaf(sm.F[buf][w][k][lane], carry[k], sm.G[buf][w][k][lane]);
      }
    } else {
      if (warp == 0) {
#pragma unroll
        for (int k = 0; k < V; k++) {
          const float Gt = starts ? G[k] : fmaf(F[k], Gb[k], G[k]), Ft = fmaxf(Fb[k] * F[k], LEAST);
          for (uint32_t b = 0; b < size; b++) {
            put_remote(&sm.cF[buf][rank][k][lane], b, Ft);
            put_remote(&sm.cG[buf][rank][k][lane], b, Gt);
          }
        }
        if (lane < size) put_remote(&sm.c_starts[buf][rank], lane, cut | starts);
      }
      cluster_arrive();
      cluster_wait();
      float behind[V];
      for (int b = (int)size - 1; b >= 0; b--) {
        const bool constant = sm.c_starts[buf][b] != 0;
#pragma unroll
        for (int k = 0; k < V; k++) {
          if (b == (int)rank) behind[k] = carry[k];
          carry[k] = constant ? sm.cG[buf][b][k][lane] : fmaf(sm.cF[buf][b][k][lane], carry[k], sm.cG[buf][b][k][lane]);
        }
      }
#pragma unroll
      for (int k = 0; k < V; k++) e[k] = cut ? Gb[k] : fmaf(Fb[k], behind[k], Gb[k]);
    }
    // the states in front of the tokens
#pragma unroll
    for (int s = 0; s < S; s++) {
      if (starts >> s & 1) entering(s, h);
#pragma unroll
      for (int k = 0; k < V; k++) {
        const float before = h[k];
        h[k] = fmaf(f[s][k], h[k], u[s][k]);
        u[s][k] = before;
      }
    }
    T* dx = reinterpret_cast<T*>(p.dx) + t0 * p.lddx + c;
    T* dr = reinterpret_cast<T*>(p.dr) + t0 * p.lddr + c;
    T* di = reinterpret_cast<T*>(p.di) + t0 * p.lddi + c;
#pragma unroll
    for (int s = S - 1; s >= 0; s--) {
      if (s >= n) continue;
      float gx[V], gr[V], gi[V];
#pragma unroll
      for (int k = 0; k < V; k++) {
        const Gates a = decay<T, POWER>(to_float(r.v[s].v[k]), rb[k], k_[k]);
        float g = 1.0f, ng = 0.0f;
        if (GATED) sigmoid_pair<T>(to_float(i.v[s].v[k]), ib[k], g, ng);
        const float dh = d[s][k] + e[k], b = dh * g * to_float(x.v[s].v[k]);
        gx[k] = dh * a.gain * g;
        gi[k] = b * a.gain * ng;
        if (POWER) {
          const float l = sizeof(T) == 4 ? a.l : a.l * LN2_F;
          const float m = a.f * (dh * u[s][k] * l - b * a.f * (l * a.inv));
          gr[k] = m * a.n;
          sum_rate[k] += m;
        } else {
          gr[k] = (dh * u[s][k] - b) * a.s * a.n;
        }
        sum_r[k] += gr[k];
        sum_i[k] += gi[k];
        e[k] = a.f * dh;
      }
      if (mine) {
        *reinterpret_cast<Pack<T, V>*>(dx + s * p.lddx) = pack<T, V>(gx);
        *reinterpret_cast<Pack<T, V>*>(dr + s * p.lddr) = pack<T, V>(gr);
        if (GATED) *reinterpret_cast<Pack<T, V>*>(di + s * p.lddi) = pack<T, V>(gi);
      }
      if (starts >> s & 1) {
        float unused[V];
        const int q = entering(s, unused);
#pragma unroll
        for (int k = 0; k < V; k++) {
          if (p.dsrc != nullptr && mine) p.dsrc[(long long)q * p.C + c + k] = e[k];
          e[k] = 0.0f;
        }
      }
    }
    t0 -= step;
    n = round > 0 ? count(t0, end) : 0;
    ask(t0, n);
  }
  zero_rest<T, V>(p.dx, p.lddx, end, p.seq.T, c, mine, rank, size);
  zero_rest<T, V>(p.dr, p.lddr, end, p.seq.T, c, mine, rank, size);
  if (GATED) zero_rest<T, V>(p.di, p.lddi, end, p.seq.T, c, mine, rank, size);

  // sums over the tokens: of the warps, then of the cluster's blocks
#pragma unroll
  for (int k = 0; k < V; k++) {
    sm.sums[0][warp][k][lane] = sum_rate[k];
    sm.sums[1][warp][k][lane] = sum_r[k];
    sm.sums[2][warp][k][lane] = sum_i[k];
  }
  __syncthreads();
  float total[V];
  if (warp < 3) {
#pragma unroll
    for (int k = 0; k < V; k++) {
      total[k] = 0.0f;
      for (int w = 0; w < WARPS; w++) total[k] += sm.sums[warp][w][k][lane];
      if (size > 1) put_remote(&sm.c_sums[warp][rank][k][lane], 0, total[k]);
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
        for (uint32_t b = 0; b < size; b++) total[k] += sm.c_sums[warp][b][k][lane];
      }
      if (warp == 0) {
        const float v = p.rate[c + k], soft = softplus_exact(v);
        total[k] *= soft > 0.0f ? 1.0f / (1.0f + expf(-v)) / soft : 1.0f;      // 1 in the limit of low rates
      }
      to[c + k] = total[k];
    }
  }
}

template <typename T, bool WIDE, bool POWER>
cudaError_t launch_form(const GatedScanGradParams& p, cudaStream_t stream) {
  const long long slabs = (p.C + 32 * CHANNELS<T, WIDE> - 1) / (32 * CHANNELS<T, WIDE>);
  const int size = cluster_of(slabs, p.seq.T);
  return p.i != nullptr ? launch_clusters(kda_gated_scan_grad_kernel<T, WIDE, POWER, true>, p, slabs, size, stream)
                        : launch_clusters(kda_gated_scan_grad_kernel<T, WIDE, POWER, false>, p, slabs, size, stream);
}

template <typename T>
cudaError_t launch_type(const GatedScanGradParams& p, cudaStream_t stream) {
  if constexpr (sizeof(T) == 2) {
    const bool wide = p.C % 2 == 0 && rows_on(p.x, p.ldx, 2, 4) && rows_on(p.r, p.ldr, 2, 4) && rows_on(p.i, p.ldi, 2, 4) && rows_on(p.dy, p.lddy, 2, 4) &&
                      rows_on(p.dx, p.lddx, 2, 4) && rows_on(p.dr, p.lddr, 2, 4) && rows_on(p.di, p.lddi, 2, 4);
    if (wide) return p.rate != nullptr ? launch_form<T, true, true>(p, stream) : launch_form<T, true, false>(p, stream);
  }
  return p.rate != nullptr ? launch_form<T, false, true>(p, stream) : launch_form<T, false, false>(p, stream);
}

}  // namespace

cudaError_t launch_gated_scan_grad(const GatedScanGradParams& p, int type, cudaStream_t stream) {
  if (type == TYPE_BF16) return launch_type<__nv_bfloat16>(p, stream);
  if (type == TYPE_FP16) return launch_type<__half>(p, stream);
  return launch_type<float>(p, stream);
}

}  // namespace kda
