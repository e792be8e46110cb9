// Gated linear recurrence over packed sequences, forward, and its step for single tokens (formulas and layout: kda_gscan.cuh).
#include "kda_gscan.cuh"

namespace kda {

namespace {

using namespace gscan;

// One round: the maps of the warps' slices, double-buffered against warps (blocks) that are a round ahead.
template <int V>
struct Shared {
  float F[2][WARPS][V][32], U[2][WARPS][V][32];            // of the block's slices
  float cF[2][MAX_CLUSTER][V][32], cU[2][MAX_CLUSTER][V][32];       // of the cluster's tiles, written by their blocks
  uint32_t starts[2][WARPS], c_starts[2][MAX_CLUSTER];     // whether a sequence starts there: the map is constant
};

// Stores the final states of the sequences that end at t: those of entries j and behind.  h: the state in front of t.
template <int V>
__device__ __noinline__ void finish(const GatedScanParams& p, int j, long long t, bool all_empty, int c, bool mine, const float (&h)[V]) {
  if (p.dst == nullptr) return;
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

template <typename T, bool WIDE, bool POWER, bool GATED>
__global__ void __launch_bounds__(THREADS, 2) kda_gated_scan_kernel(const GatedScanParams p) {
  constexpr int V = CHANNELS<T, WIDE>;
  __shared__ Shared<V> sm;
  const uint32_t rank = cluster_rank(), size = cluster_size();
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int c = ((int)(blockIdx.x / size) * 32 + lane) * V;
  const bool mine = c < p.C;
  if (size > 1) cluster_arrive();                    // blocks write into one another: all of them have to be there
  const bool rejected = cu_rejected(p.seq);
  const long long end = rejected ? 0 : cu_at(p.seq, p.seq.N);
  const long long step = (long long)size * TILE;
  const long long rounds = end > 0 ? (end + step - 1) / step : 1;

  float rb[V], ib[V], k_[V];
#pragma unroll
  for (int k = 0; k < V; k++) {
    rb[k] = mine ? bias_of<T>(p.r_bias, c + k) : 0.0f;
    ib[k] = GATED && mine ? bias_of<T>(p.i_bias, c + k) : 0.0f;
    k_[k] = POWER && mine ? decay_factor<T>(p.rate, c + k, p.rate_scale) : 0.0f;
  }
  Rows<T, V> x, r, i;
  long long t0 = (long long)rank * TILE + warp * S;
  int n = count(t0, end);
  x.ask(p.x, p.ldx, t0, n, c, mine);
  r.ask(p.r, p.ldr, t0, n, c, mine);
  if (GATED) i.ask(p.i, p.ldi, t0, n, c, mine);
  int j = 0;                                         // first entry of cu_seqlens that is >= t0, once looked for
  long long next = 0;                                // that entry
  float carry[V] = {};
  if (size > 1) cluster_wait();

  for (long long round = 0; round < rounds; round++) {
    const int buf = (int)(round & 1);
    if (next < t0) {
      j = seek(p.seq, j, t0);
      next = j <= p.seq.N ? cu_at(p.seq, j) : NEVER;
    }
    float f[S][V], u[S][V];
#pragma unroll
    for (int s = 0; s < S; s++) {
#pragma unroll
      for (int k = 0; k < V; k++) {
        const Gates a = decay<T, POWER>(to_float(r.v[s].v[k]), rb[k], k_[k]);
        float g = 1.0f, ng;
        if (GATED) sigmoid_pair<T>(to_float(i.v[s].v[k]), ib[k], g, ng);
        f[s][k] = a.f;
        u[s][k] = a.gain * g * to_float(x.v[s].v[k]);
        if (s >= n) { f[s][k] = 1.0f; u[s][k] = 0.0f; }
      }
    }
    const long long t_next = t0 + step;
    const int n_next = round + 1 < rounds ? count(t_next, end) : 0;
    x.ask(p.x, p.ldx, t_next, n_next, c, mine);
    r.ask(p.r, p.ldr, t_next, n_next, c, mine);
    if (GATED) i.ask(p.i, p.ldi, t_next, n_next, c, mine);

    // sequences that start in the slice: the state they enter with joins the first token's term
    uint32_t starts = 0;
    if (!rejected && next < t0 + n) {
      for (int q = j; q < p.seq.N; q++) {
        const long long t = cu_at(p.seq, q);
        if (t >= t0 + n) break;
        if (cu_at(p.seq, q + 1) == t) continue;
        const long long slot = claim(p.seq, q);
        const int at = (int)(t - t0);
        starts |= 1u << at;
#pragma unroll
        for (int k = 0; k < V; k++) {
          const float h0 = p.src != nullptr && slot >= 0 && mine ? p.src[slot * p.src_stride + c + k] : 0.0f;
#pragma unroll
          for (int s = 0; s < S; s++)
            if (s == at) u[s][k] = fmaf(f[s][k], h0, u[s][k]);
        }
      }
    }
    float F[V], U[V];
#pragma unroll
    for (int k = 0; k < V; k++) {
      F[k] = 1.0f; U[k] = 0.0f;
#pragma unroll
      for (int s = 0; s < S; s++) {
        U[k] = starts >> s & 1 ? u[s][k] : fmaf(f[s][k], U[k], u[s][k]);
        F[k] *= f[s][k];
      }
      F[k] = fmaxf(F[k], LEAST);
      sm.F[buf][warp][k][lane] = F[k];
      sm.U[buf][warp][k][lane] = U[k];
    }
    if (lane == 0) sm.starts[buf][warp] = starts;
    __syncthreads();
    // the slices in front of this one
    float Fb[V], Ub[V];
    uint32_t cut = 0;
#pragma unroll
    for (int k = 0; k < V; k++) { Fb[k] = 1.0f; Ub[k] = 0.0f; }
    for (int w = 0; w < warp; w++) {
      const bool constant = sm.starts[buf][w] != 0;
      cut |= constant;
#pragma unroll
      for (int k = 0; k < V; k++) {
        const float Fw = sm.F[buf][w][k][lane], Uw = sm.U[buf][w][k][lane];
        Ub[k] = constant ? Uw : fmaf(Fw, Ub[k], Uw);
        Fb[k] = fmaxf(Fb[k] * Fw, LEAST);
      }
    }
    float h[V];
    if (size == 1) {
#pragma unroll
      for (int k = 0; k < V; k++) h[k] = cut ? Ub[k] : fmaf(Fb[k], carry[k], Ub[k]);
      // the next round's
#pragma unroll
      for (int k = 0; k < V; k++) carry[k] = h[k];
      for (int w = warp; w < WARPS; w++) {
        const bool constant = sm.starts[buf][w] != 0;
#pragma unroll
        for (int k = 0; k < V; k++) carry[k] = constant ? sm.U[buf][w][k][lane] : fmaf(sm.F[buf][w][k][lane], carry[k], sm.U[buf][w][k][lane]);
      }
    } else {
      if (warp == WARPS - 1) {                       // it has the tile's map: to every block of the cluster
#pragma unroll
        for (int k = 0; k < V; k++) {
          const float Ut = starts ? U[k] : fmaf(F[k], Ub[k], U[k]), Ft = fmaxf(Fb[k] * F[k], LEAST);
          for (uint32_t b = 0; b < size; b++) {
            put_remote(&sm.cF[buf][rank][k][lane], b, Ft);
            put_remote(&sm.cU[buf][rank][k][lane], b, Ut);
          }
        }
        if (lane < size) put_remote(&sm.c_starts[buf][rank], lane, cut | starts);
      }
      cluster_arrive();
      cluster_wait();
      float enter[V];
      for (uint32_t b = 0; b < size; b++) {
        const bool constant = sm.c_starts[buf][b] != 0;
#pragma unroll
        for (int k = 0; k < V; k++) {
          if (b == rank) enter[k] = carry[k];
          carry[k] = constant ? sm.cU[buf][b][k][lane] : fmaf(sm.cF[buf][b][k][lane], carry[k], sm.cU[buf][b][k][lane]);
        }
      }
#pragma unroll
      for (int k = 0; k < V; k++) h[k] = cut ? Ub[k] : fmaf(Fb[k], enter[k], Ub[k]);
    }
    if (p.tiles != nullptr && warp == 0 && mine && n > 0) {
#pragma unroll
      for (int k = 0; k < V; k++) p.tiles[(t0 / TILE) * p.C + c + k] = h[k];
    }
    T* out = reinterpret_cast<T*>(p.out) + t0 * p.ldo + c;
#pragma unroll
    for (int s = 0; s < S; s++) {
      if (s < n) {
        if (!rejected && next < t0 + n && next <= t0 + s) {        // one of the entries may be this token
          const int q = seek(p.seq, j, t0 + s);
          if (q <= p.seq.N && cu_at(p.seq, q) == t0 + s) finish(p, q, t0 + s, false, c, mine, h);
        }
#pragma unroll
        for (int k = 0; k < V; k++) h[k] = starts >> s & 1 ? u[s][k] : fmaf(f[s][k], h[k], u[s][k]);
        if (mine) *reinterpret_cast<Pack<T, V>*>(out + s * p.ldo) = pack<T, V>(h);
      }
    }
    if (!rejected && ((n > 0 && t0 + n == end) || (end == 0 && t0 == 0))) finish(p, seek(p.seq, j, end), end, false, c, mine, h);
    t0 = t_next;
    n = n_next;
  }
  if (rejected && rank == 0 && warp == 0) finish(p, 1, 0, true, c, mine, carry);
  if (rejected || p.zero_pad) zero_rest<T, V>(p.out, p.ldo, end, p.seq.T, c, mine, rank, size);
}

template <typename T, bool WIDE, bool POWER>
cudaError_t launch_form(const GatedScanParams& p, cudaStream_t stream) {
  const long long slabs = (p.C + 32 * CHANNELS<T, WIDE> - 1) / (32 * CHANNELS<T, WIDE>);
  const int size = cluster_of(slabs, p.seq.T);
  return p.i != nullptr ? launch_clusters(kda_gated_scan_kernel<T, WIDE, POWER, true>, p, slabs, size, stream)
                        : launch_clusters(kda_gated_scan_kernel<T, WIDE, POWER, false>, p, slabs, size, stream);
}

template <typename T>
cudaError_t launch_type(const GatedScanParams& p, cudaStream_t stream) {
  if constexpr (sizeof(T) == 2) {
    const bool wide = p.C % 2 == 0 && rows_on(p.x, p.ldx, 2, 4) && rows_on(p.r, p.ldr, 2, 4) && rows_on(p.i, p.ldi, 2, 4) && rows_on(p.out, p.ldo, 2, 4);
    if (wide) return p.rate != nullptr ? launch_form<T, true, true>(p, stream) : launch_form<T, true, false>(p, stream);
  }
  return p.rate != nullptr ? launch_form<T, false, true>(p, stream) : launch_form<T, false, false>(p, stream);
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
      const Gates a = decay<T, POWER>(to_float(r[q].v[k]), rb[k], k_[k]);
      float g = 1.0f, ng;
      if (p.i != nullptr) sigmoid_pair<T>(to_float(i[q].v[k]), ib[k], g, ng);
      h[k] = a.gain * g * to_float(x[q].v[k]);
      h[k] = fmaf(a.f, slot[q] >= 0 ? state[q].v[k] : 0.0f, h[k]);
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
