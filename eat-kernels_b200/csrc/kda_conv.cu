// Short causal convolution over packed sequences, depthwise:
//   y[t, c] = act(b[c] + sum_j w[c, j] x[t - (W - 1) + j, c])
// Rows in front of a sequence are the W - 1 history rows of its slot; its last W - 1 rows become the new history.
#include "kda_serving.cuh"

namespace kda {

namespace {

constexpr int CONV_THREADS = 128;
constexpr int GROUP = 4;                 // tokens whose rows are asked for together
// Blocks an SM that the prompt kernel's registers leave room for: two groups of rows in 16 bits fit 72 registers, in 32 bits 96 (W = 4, 3, 2
// on the batch below: 480, 454 and 438 us; with 72 registers, spilling 296 bytes, 565, 460 and 546; 80: 467, 524, 432; 128: 502, 494, 438).
template <typename T>
constexpr int BLOCKS_AN_SM = sizeof(T) == 4 ? 5 : 7;

// N consecutive values, in 8-byte accesses where they start on 8 bytes
template <typename T, int N>
__device__ __forceinline__ void load_run(const T* p, float (&f)[N]) {
  constexpr int PER = 8 / sizeof(T);
  if (N % PER == 0 && (reinterpret_cast<uintptr_t>(p) & 7) == 0) {
#pragma unroll
    for (int i = 0; i < N / PER; i++) {
      const Pack<T, PER> v = reinterpret_cast<const Pack<T, PER>*>(p)[i];
#pragma unroll
      for (int j = 0; j < PER; j++) f[i * PER + j] = to_float(v.v[j]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; i++) f[i] = to_float(p[i]);
  }
}

template <int N>
__device__ __forceinline__ void load_run(const void* p, int type, long long at, float (&f)[N]) {
  if (type == TYPE_BF16) load_run(reinterpret_cast<const __nv_bfloat16*>(p) + at, f);
  else if (type == TYPE_FP16) load_run(reinterpret_cast<const __half*>(p) + at, f);
  else load_run(reinterpret_cast<const float*>(p) + at, f);
}

template <int VEC, int W>
__device__ __forceinline__ void load_weights(const ConvParams& p, int c, float (&w)[W][VEC], float (&b)[VEC]) {
  float run[VEC * W];
  load_run(p.weight, p.weight_type, (long long)c * W, run);
#pragma unroll
  for (int i = 0; i < VEC; i++) {
#pragma unroll
    for (int j = 0; j < W; j++) w[j][i] = run[i * W + j];
    b[i] = 0.0f;
  }
  if (p.bias != nullptr) load_run(p.bias, p.weight_type, c, b);
}

// VEC channels a thread, a tile of tokens a block.  A sequence's first W - 1 tokens belong to the tile that holds its start,
// even where they reach into the next tile: only that tile reads the slot's history, and it writes the new one after that,
// so the pool is updated in place by one launch.  Bound by memory: the window slides in registers, a tile re-reads W - 1
// rows of the tile before it (out of L2); 55 846 tokens of 6144 channels, W = 4: 258-261 us in bf16, 5.3 TB/s, 480 us in fp32, 5.7 TB/s.
template <typename T, int VEC, int W>
__global__ void __launch_bounds__(CONV_THREADS, BLOCKS_AN_SM<T>) kda_short_conv_kernel(const ConvParams p) {
  constexpr int HW = W - 1;
  using P = Pack<T, VEC>;
  const int cblocks = (p.C / VEC + CONV_THREADS - 1) / CONV_THREADS;
  const long long t0 = (long long)(blockIdx.x / cblocks) * p.tile;
  const long long t1 = min(t0 + p.tile, p.seq.T);
  const bool last = t1 == p.seq.T;
  const int c = ((int)(blockIdx.x % cblocks) * CONV_THREADS + (int)threadIdx.x) * VEC;
  const bool mine = c < p.C;
  const T* x = reinterpret_cast<const T*>(p.x) + c;
  T* out = reinterpret_cast<T*>(p.out) + c;
  const T* src = reinterpret_cast<const T*>(p.src) + c;
  T* dst = reinterpret_cast<T*>(p.dst) + c;
  const int N = p.seq.N;
  P zero;
#pragma unroll
  for (int i = 0; i < VEC; i++) zero.v[i] = from_float<T>(0.0f);

  int lo;                                            // the first sequence that starts in this tile
  const bool rejected = cu_rejected(p.seq, t0, lo);
  float w[W][VEC], b[VEC];
  if (mine) load_weights<VEC, W>(p, c, w, b);

  auto token = [&](long long t, const P& row, float (&win)[HW][VEC]) {
    float cur[VEC], y[VEC];
    unpack(row, cur);
#pragma unroll
    for (int i = 0; i < VEC; i++) {
      float acc = b[i];
#pragma unroll
      for (int j = 0; j < HW; j++) acc = fmaf(w[j][i], win[j][i], acc);
      acc = fmaf(w[HW][i], cur[i], acc);
      y[i] = p.silu ? silu<T>(acc) : acc;
#pragma unroll
      for (int j = 0; j + 1 < HW; j++) win[j][i] = win[j + 1][i];
      win[HW - 1][i] = cur[i];
    }
    *reinterpret_cast<P*>(out + t * p.ldo) = pack<T, VEC>(y);
  };
  // tokens in groups: a group's rows are on their way while the group in front is worked on (two groups of four: 258 us on the
  // batch above in bf16, 252 in fp16, one of eight at a time 270 and 252, two of eight 271, two of two 300)
  auto run = [&](long long from, long long to, float (&win)[HW][VEC]) {
    if (from + GROUP <= to) {
      P rows[GROUP], next[GROUP];
#pragma unroll
      for (int g = 0; g < GROUP; g++) rows[g] = *reinterpret_cast<const P*>(x + (from + g) * p.ldx);
      for (; from + GROUP <= to; from += GROUP) {
        const bool more = from + 2 * GROUP <= to;
        if (more) {
#pragma unroll
          for (int g = 0; g < GROUP; g++) next[g] = *reinterpret_cast<const P*>(x + (from + GROUP + g) * p.ldx);
        }
#pragma unroll
        for (int g = 0; g < GROUP; g++) token(from + g, rows[g], win);
#pragma unroll
        for (int g = 0; g < GROUP; g++) rows[g] = next[g];
      }
    }
    for (; from < to; from++) token(from, *reinterpret_cast<const P*>(x + from * p.ldx), win);
  };

  // the sequence that reaches into this tile
  if (!rejected && mine && lo > 0 && lo <= N) {
    const long long begin = cu_at(p.seq, lo - 1), end = cu_at(p.seq, lo);
    const long long from = max(t0, begin + HW), to = min(end, t1);
    if (from < to) {
      float win[HW][VEC];
#pragma unroll
      for (int j = 0; j < HW; j++) unpack(*reinterpret_cast<const P*>(x + (from - HW + j) * p.ldx), win[j]);
      run(from, to, win);
    }
  }
  // sequences that start here, empty ones among them (behind a rejected layout all are empty and the first tile has them)
  for (int s = rejected ? (t0 == 0 ? 0 : N) : lo; s < N; s++) {
    const long long begin = rejected ? 0 : cu_at(p.seq, s), end = rejected ? 0 : cu_at(p.seq, s + 1);
    if (!rejected && begin >= t1 && !(last && begin == t1)) break;
    const long long slot = claim_slot(p.seq, s);
    if (!mine) continue;
    P hist[HW];
#pragma unroll
    for (int j = 0; j < HW; j++)
      hist[j] = p.src != nullptr && slot >= 0 ? *reinterpret_cast<const P*>(src + slot * p.src_stride + (long long)j * p.C) : zero;
    if (p.dst != nullptr && slot >= 0) {
      const long long len = end - begin;
#pragma unroll
      for (int j = 0; j < HW; j++) {
        P row = zero;
        if (len >= HW - j) row = *reinterpret_cast<const P*>(x + (end - HW + j) * p.ldx);
#pragma unroll
        for (int h = 0; h < HW; h++)
          if (h == len + j) row = hist[h];
        *reinterpret_cast<P*>(dst + slot * p.dst_stride + (long long)j * p.C) = row;
      }
    }
    float win[HW][VEC];
#pragma unroll
    for (int j = 0; j < HW; j++) unpack(hist[j], win[j]);
    run(begin, min(end, max(t1, begin + HW)), win);
  }
  if ((rejected || p.zero_pad) && mine)
    for (long long t = rejected ? t0 : max(t0, cu_at(p.seq, N)); t < t1; t++) *reinterpret_cast<P*>(out + t * p.ldo) = zero;
}

// One token a row, VEC channels a thread: the window is the slot's history and the token.  A block takes ROWS rows for one load of
// the weights, all their histories in flight at once.
constexpr int STEP_ROWS = 4;
template <typename T, int VEC, int W>
__global__ void __launch_bounds__(CONV_THREADS) kda_short_conv_step_kernel(const ConvParams p) {
  constexpr int HW = W - 1;
  using P = Pack<T, VEC>;
  const int cblocks = (p.C / VEC + CONV_THREADS - 1) / CONV_THREADS;
  const int row0 = blockIdx.x / cblocks * p.tile, rows = min(p.tile, (int)p.seq.T - row0);
  const int c = ((int)(blockIdx.x % cblocks) * CONV_THREADS + (int)threadIdx.x) * VEC;
  int slot[STEP_ROWS];
  row_slots(p.seq, row0, rows, slot);
  const bool mine = c < p.C;
  T* pool = reinterpret_cast<T*>(p.dst) + c;
  P hist[STEP_ROWS][HW], cur[STEP_ROWS];
#pragma unroll
  for (int r = 0; r < STEP_ROWS; r++) {
    if (mine && slot[r] != -2) cur[r] = *reinterpret_cast<const P*>(reinterpret_cast<const T*>(p.x) + (long long)(row0 + r) * p.ldx + c);
#pragma unroll
    for (int j = 0; j < HW; j++)
      if (mine && slot[r] >= 0) hist[r][j] = *reinterpret_cast<const P*>(pool + slot[r] * p.dst_stride + (long long)j * p.C);
  }
  drop_repeats(p.seq, row0, slot);
  if (!mine) return;
  float w[W][VEC], b[VEC];
  load_weights<VEC, W>(p, c, w, b);
#pragma unroll
  for (int r = 0; r < STEP_ROWS; r++) {
    if (r >= rows) break;
    P* out = reinterpret_cast<P*>(reinterpret_cast<T*>(p.out) + (long long)(row0 + r) * p.ldo + c);
    float y[VEC], f[VEC];
    if (slot[r] == -2) {
#pragma unroll
      for (int i = 0; i < VEC; i++) y[i] = 0.0f;
      if (p.zero_pad) *out = pack<T, VEC>(y);
      continue;
    }
#pragma unroll
    for (int i = 0; i < VEC; i++) y[i] = b[i];
    if (slot[r] >= 0) {
      T* to = pool + slot[r] * p.dst_stride;
#pragma unroll
      for (int j = 0; j + 1 < HW; j++) *reinterpret_cast<P*>(to + (long long)j * p.C) = hist[r][j + 1];
      *reinterpret_cast<P*>(to + (long long)(HW - 1) * p.C) = cur[r];
#pragma unroll
      for (int j = 0; j < HW; j++) {
        unpack(hist[r][j], f);
#pragma unroll
        for (int i = 0; i < VEC; i++) y[i] = fmaf(w[j][i], f[i], y[i]);
      }
    }
    unpack(cur[r], f);
#pragma unroll
    for (int i = 0; i < VEC; i++) {
      y[i] = fmaf(w[HW][i], f[i], y[i]);
      if (p.silu) y[i] = silu<T>(y[i]);
    }
    *out = pack<T, VEC>(y);
  }
}

// Four channels an access where every row starts on as many, single values elsewhere.  Eight 16-bit channels take 187 registers, which
// leaves two blocks an SM: 471 us for 56 k tokens of 6144 channels against 273 us with four (before the groups of four).
constexpr int WIDE = 4;
template <typename T>
bool wide(const ConvParams& p) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(p.x) | reinterpret_cast<uintptr_t>(p.out) | reinterpret_cast<uintptr_t>(p.src) |
                       reinterpret_cast<uintptr_t>(p.dst);
  return (at & (WIDE * sizeof(T) - 1)) == 0 && ((p.C | p.ldx | p.ldo | p.src_stride | p.dst_stride) & (WIDE - 1)) == 0;
}

template <typename T, int VEC>
cudaError_t launch_width(const ConvParams& p, bool step, cudaStream_t stream) {
  const long long cblocks = (p.C / VEC + CONV_THREADS - 1) / CONV_THREADS;
  const long long rows = step || p.seq.T > 0 ? (p.seq.T + p.tile - 1) / p.tile : 1;
  const long long blocks = cblocks * rows;
  if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
  if (blocks == 0) return cudaSuccess;
  const dim3 grid((unsigned)blocks);
  if (p.W == 2) step ? kda_short_conv_step_kernel<T, VEC, 2><<<grid, CONV_THREADS, 0, stream>>>(p) : kda_short_conv_kernel<T, VEC, 2><<<grid, CONV_THREADS, 0, stream>>>(p);
  if (p.W == 3) step ? kda_short_conv_step_kernel<T, VEC, 3><<<grid, CONV_THREADS, 0, stream>>>(p) : kda_short_conv_kernel<T, VEC, 3><<<grid, CONV_THREADS, 0, stream>>>(p);
  if (p.W == 4) step ? kda_short_conv_step_kernel<T, VEC, 4><<<grid, CONV_THREADS, 0, stream>>>(p) : kda_short_conv_kernel<T, VEC, 4><<<grid, CONV_THREADS, 0, stream>>>(p);
  return cudaGetLastError();
}

// Rows of a block: as many as leave two blocks an SM, so that small calls spread over the card and large ones share weights and
// the rows in front of a tile.
int tile_of(long long rows, long long cblocks, int least, int most) {
  int tile = most;
  while (tile > least && (rows + tile - 1) / tile * cblocks < 2 * 148) tile /= 2;
  return tile;
}

template <typename T>
cudaError_t launch_type(ConvParams p, bool step, cudaStream_t stream) {
  const bool w = wide<T>(p);
  const long long cblocks = (p.C / (w ? WIDE : 1) + CONV_THREADS - 1) / CONV_THREADS;
  p.tile = step ? tile_of(p.seq.T, cblocks, 1, STEP_ROWS) : tile_of(p.seq.T, cblocks, 8, 64);
  return w ? launch_width<T, WIDE>(p, step, stream) : launch_width<T, 1>(p, step, stream);
}

cudaError_t launch_any(const ConvParams& p, int type, bool step, cudaStream_t stream) {
  if (type == TYPE_BF16) return launch_type<__nv_bfloat16>(p, step, stream);
  if (type == TYPE_FP16) return launch_type<__half>(p, step, stream);
  return launch_type<float>(p, step, stream);
}

}  // namespace

cudaError_t launch_conv(ConvParams p, int type, cudaStream_t stream) { return launch_any(p, type, false, stream); }
cudaError_t launch_conv_step(ConvParams p, int type, cudaStream_t stream) { return launch_any(p, type, true, stream); }

}  // namespace kda
