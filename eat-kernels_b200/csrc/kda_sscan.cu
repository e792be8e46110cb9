// Selective state space scan over packed sequences, per channel d with Ns state values n (states in fp32):
//   s = softplus(dt + dt_bias);  h[n] = exp(s A[d,n]) h[n] + s u B[n];  y = sum_n C[n] h[n] + D[d] u;  y *= silu(z)
//
// What bounds it: one exponential a token, channel and state value, 16 a clock and SM in the special-function unit, which is
// about three times the time of the tokens' bytes; behind it the shared-memory pipe (a 16-byte access of a warp takes four
// cycles, also where lanes read the same) and the instructions issued.  So:
//   * a block has four scan warps and four helper warps.  The helpers bring the tokens by asynchronous copies, work out the step
//     sizes and s u, and write the outputs with D u and the gate; the scan warps only see shared memory.  Two stages of tokens
//     between them, handed over by named barriers.
//   * shared memory holds time rows: a lane takes four tokens in one access, and all products but the chain itself run two
//     tokens an instruction, without a value copied to make a pair.
//   * a lane has two channels, so that B and C are read once for both, and S state values of each; L lanes share a channel.
//     Sums over the lanes are taken for four tokens at once, each step of an exchange halving the tokens that a lane holds.
// Measured (16 state values): 8 ragged prompts, 10 245 tokens of 4096 channels, in bf16 270 us, the exponentials' unit busy 65 % of
// it (one channel a lane: 308 us, the shared-memory pipe at 84 %), in fp32 299 us; one prompt of 32 768 tokens on 512 channels 207 us
// in pieces (uncut 1725 us).  Rows that do not all start on 16 bytes are read value by value: the ragged prompts with 4095 channels
// 330 us, with 4 and 13 state values (B and C rows of 8 and 26 bytes, all tensors on that path) 332 and 336 us.
#include "kda_serving.cuh"

namespace kda {

namespace {

constexpr int SCAN_LANES = 128;          // scan threads of a block
constexpr int CH = 2;                    // channels of a lane
constexpr int HELPERS = 128;
constexpr int SCAN_THREADS = SCAN_LANES + HELPERS;
constexpr int STEP_LANES = 128;          // threads of a single token's block
constexpr int TILE = 16;                 // tokens a stage
constexpr int QUADS = TILE / 4;
constexpr float LOG2E_F = 1.4426950408889634f;

// log(1 + e) / e for e in [0, 1]: minimax polynomial (Remez exchange) of the relative error, coefficients rounded to fp32;
// 1.8e-7 off with its roundings.
__host__ __device__ constexpr float log1p_coef(int k) {
  constexpr float c[9] = {0.9999999403953552f,  -0.4999949336051941f,  0.3331909775733948f,  -0.2484298199415207f, 0.19106006622314453f,
                          -0.13663245737552643f, 0.07822595536708832f, -0.02950523979961872f, 0.0052326940931379795f};
  return c[k];
}
__device__ __forceinline__ float exp2_fast(float x) {      // 2 ulp; below 2^-126 zero
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// max(x, 0) + log(1 + exp(-|x|)); NaN stays, by the second term
__device__ __forceinline__ float softplus(float x) {
  const float e = exp2_fast(-fabsf(x) * LOG2E_F);
  float q = log1p_coef(8);
#pragma unroll
  for (int k = 7; k >= 0; k--) q = fmaf(q, e, log1p_coef(k));
  return fmaxf(x, 0.0f) + q * e;
}

// A in powers of two; finite, since an infinite rate times a step of zero (that of the places behind the last token, too) would be NaN:
// it keeps the state at such a step and forgets it at every other
__device__ __forceinline__ float decay_rate(float a) {
  a *= LOG2E_F;
  return a < -3.0e38f ? -3.0e38f : (a > 3.0e38f ? 3.0e38f : a);
}

// two fp32 values an instruction
using F2 = unsigned long long;
__device__ __forceinline__ F2 f2(float a, float b) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void split(F2 v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

// of two values, the polynomial for both at once
__device__ __forceinline__ F2 softplus2(float x, float y) {
  const F2 e = f2(exp2_fast(-fabsf(x) * LOG2E_F), exp2_fast(-fabsf(y) * LOG2E_F));
  F2 q = f2(log1p_coef(8), log1p_coef(8));
#pragma unroll
  for (int k = 7; k >= 0; k--) q = fma2(q, e, f2(log1p_coef(k), log1p_coef(k)));
  float p0, p1;
  split(mul2(q, e), p0, p1);
  return f2(fmaxf(x, 0.0f) + p0, fmaxf(y, 0.0f) + p1);
}

__device__ __forceinline__ void bar_sync(int id) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(SCAN_THREADS) : "memory"); }
__device__ __forceinline__ void bar_arrive(int id) { asm volatile("bar.arrive %0, %1;" ::"r"(id), "r"(SCAN_THREADS) : "memory"); }
enum { BAR_FULL = 1, BAR_DONE = 3, BAR_HELPERS = 5 };     // FULL, DONE: + stage

// Tokens as they lie in memory, on their way to the helpers: rows of time, for DEPTH tiles.
template <typename T, int L, int S>
struct RawShared {
  static constexpr int DEPTH = sizeof(T) == 4 ? 3 : 4;                   // what lets two blocks share an SM

  // rows of whole 16 bytes; 16-bit rows four apart fall into different halves of the banks
  static constexpr int XS = CH * SCAN_LANES / L + 8, NS = L * S < 8 ? 16 : L * S + 8;
  struct Slot {
    T x[3][TILE][XS];                                // u, dt, z
    T bc[2][TILE][NS];
  } slot[DEPTH];
};

template <int S>
struct Values {
  float v[S] = {};
};
// S consecutive values in one access
template <int S>
__device__ __forceinline__ Values<S> load_values(const float* p) {
  Values<S> r;
  const Pack<float, S> v = *reinterpret_cast<const Pack<float, S>*>(p);
#pragma unroll
  for (int k = 0; k < S; k++) r.v[k] = v.v[k];
  return r;
}
template <int S>
__device__ __forceinline__ void store_values(float* p, const Values<S>& v) {
  Pack<float, S> f;
#pragma unroll
  for (int k = 0; k < S; k++) f.v[k] = v.v[k];
  *reinterpret_cast<Pack<float, S>*>(p) = f;
}

template <int L, int S>
struct ScanShared {
  static constexpr int CB = CH * SCAN_LANES / L;     // channels of a block; a lane has c and c + CB / CH
  static_assert(CB >= 8 && L * S <= 128, "layouts");
  static constexpr int NP = L * S;                   // state values, padded
  // a row of time, both stages: eight rows' 16 bytes at one time fall into different banks
  static constexpr int R = 2 * TILE + 4;
  float step[CB][R], input[CB][R];                   // s, s u
  float y[CB][R];                                    // sums of C h
  float b[NP][R], c[NP][R];
};

struct Work {                                        // a block's share
  int group, d0, channels;                           // group of channels, first channel, how many
  int seq, piece, pieces, at;                        // sequence, which of its pieces, how many it has, piece of the launch
  int tokens;
  long long begin;                                   // first token
};

constexpr int RANKED = 128;                          // up to so many sequences the longest goes first, where not all blocks have room at once
constexpr int ROOM = 2 * 148;

// Pieces that a sequence is cut into (empty sequences have one, for their state).
__device__ __forceinline__ int pieces_of(const ScanParams& p, bool rejected, int seq) {
  const long long n = rejected ? 0 : cu_at(p.seq, seq + 1) - cu_at(p.seq, seq);
  return n > p.piece ? (int)((n + p.piece - 1) / p.piece) : 1;
}

// Which sequence holds piece `at` of the launch, and which of its pieces that is; false: none.  Each warp looks for itself: a lane
// counts the pieces of N / 32 sequences.
__device__ __forceinline__ bool find_piece(const ScanParams& p, bool rejected, int at, Work& w) {
  const int lane = threadIdx.x % 32, each = (p.seq.N + 31) / 32;
  const int first = min(p.seq.N, lane * each), last = min(p.seq.N, first + each);
  int sum = 0;
  for (int i = first; i < last; i++) sum += pieces_of(p, rejected, i);
  int before = sum;
#pragma unroll
  for (int m = 1; m < 32; m *= 2) {
    const int up = __shfl_up_sync(0xffffffffu, before, m);
    if (lane >= m) before += up;
  }
  before -= sum;
  const unsigned has = __ballot_sync(0xffffffffu, at >= before && at < before + sum);
  if (has == 0) return false;
  int seq = first, n = 0;
  if (at >= before && at < before + sum)
    for (;; seq++) {
      n = pieces_of(p, rejected, seq);
      if (at < before + n) break;
      before += n;
    }
  const int from = __ffs(has) - 1;
  w.seq = __shfl_sync(0xffffffffu, seq, from);
  w.pieces = __shfl_sync(0xffffffffu, n, from);
  w.piece = at - __shfl_sync(0xffffffffu, before, from);
  return true;
}

// The sequence of rank `r` by length, the longest first.
__device__ __forceinline__ int by_length(const ScanParams& p, int r) {
  const int lane = threadIdx.x % 32, N = p.seq.N;
  int found = 0;
  for (int i0 = 0; i0 < N; i0 += 32) {
    const int i = i0 + lane;
    const long long mine = i < N ? cu_at(p.seq, i + 1) - cu_at(p.seq, i) : -1;
    int rank = 0;
    for (int j0 = 0; j0 < N; j0 += 32) {
      const long long other = j0 + lane < N ? cu_at(p.seq, j0 + lane + 1) - cu_at(p.seq, j0 + lane) : -1;
      for (int j = 0; j < min(32, N - j0); j++) {
        const int theirs = __shfl_sync(0xffffffffu, (int)other, j);
        rank += theirs > (int)mine || (theirs == (int)mine && j0 + j < i);
      }
    }
    const unsigned has = __ballot_sync(0xffffffffu, i < N && rank == r);
    if (has != 0) found = i0 + __ffs(has) - 1;
  }
  return found;
}

// Helper `i` of a tile whose rows are `n` accesses wide: which access of the row and which quad of tokens.  Eight neighbours
// write 16 bytes each, of four accesses' rows and two quads, to different banks (accesses of two values).
__device__ __forceinline__ void place(int i, int n, int& access, int& quad) {
  if (n >= 4) {
    const int rest = i / 8;
    access = i % 4 + rest % (n / 4) * 4;
    quad = i / 4 % 2 + rest / (n / 4) * 2;
  } else {
    access = i % n;
    quad = i / n;
  }
}

__device__ __forceinline__ void copy16(unsigned to, const void* from, int bytes) {     // 16 bytes, or (0) zeros and nothing read
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}

// A tile's rows of WIDTH values, on their way into shared memory with zeros around them, for K tensors of one shape.  ASYNC: whole
// 16 bytes at a time, which needs rows that start on them; else value by value.
template <typename T, int WIDTH, int STRIDE, int K, bool ASYNC>
struct Bring {
  static constexpr int PER = ASYNC ? 16 / sizeof(T) : 1, CHUNKS = (WIDTH + PER - 1) / PER, STEP = HELPERS / CHUNKS > 0 ? HELPERS / CHUNKS : 1;
  static constexpr int N = (TILE + STEP - 1) / STEP;                     // accesses of a thread: rows t, t + STEP, ...
  static_assert(HELPERS % CHUNKS == 0, "every thread in one column");
  const T* from[K];        // the first access of this thread, one tile after the other
  long long ld[K];
  int t, c, left;          // row, column, rows from t on that there are
  __device__ __forceinline__ Bring(const void* const (&base)[K], const long long (&ld_)[K], long long row, long long col, int valid, int tokens, int tid) {
    t = tid / CHUNKS;
    c = tid % CHUNKS * PER;
    left = c < valid ? tokens - t : 0;
#pragma unroll
    for (int k = 0; k < K; k++) {
      ld[k] = ld_[k];
      from[k] = reinterpret_cast<const T*>(base[k]) + (row + t) * ld[k] + col + c;
    }
  }
  __device__ __forceinline__ void operator()(T (*to)[TILE][STRIDE], int used) {       // the first `used` of the tensors
    const unsigned at = (unsigned)__cvta_generic_to_shared(&to[0][t][c]);
    T v[K][N];
#pragma unroll
    for (int k = 0; k < K; k++) {
      if (k >= used) break;
      const T* q = from[k];
#pragma unroll
      for (int i = 0; i < N; i++) {
        if (TILE % STEP != 0 && t + i * STEP >= TILE) break;             // more threads than rows
        const bool on = i * STEP < left;
        if constexpr (ASYNC) {
          copy16(at + (unsigned)sizeof(T) * (k * TILE * STRIDE + i * STEP * STRIDE), q, on ? 16 : 0);
        } else {
          v[k][i] = from_float<T>(0.0f);
          if (on) v[k][i] = *q;
        }
        q += STEP * ld[k];
      }
      from[k] += TILE * ld[k];
    }
    if constexpr (!ASYNC) {
#pragma unroll
      for (int k = 0; k < K; k++) {
        if (k >= used) break;
#pragma unroll
        for (int i = 0; i < N; i++)
          if (t + i * STEP < TILE) to[k][t + i * STEP][c] = v[k][i];
      }
    }
    left -= TILE;
  }
};

// The helpers' half: tokens in, outputs out.  Asynchronous copies run DEPTH - 1 tiles ahead; read value by value, a tile's values come
// through registers, DEPTH - 1 tiles before they are used too, but each tile waits for them.  A thread then has two channels of four
// consecutive tokens at a time.
template <typename T, int L, int S, bool LOCAL, bool ASYNC>
__device__ __forceinline__ void help(const ScanParams& p, const Work& w, ScanShared<L, S>& sh, RawShared<T, L, S>& raw, int tid) {
  using Sh = ScanShared<L, S>;
  using Rw = RawShared<T, L, S>;
  using P = Pack<T, 2>;
  constexpr int DEPTH = Rw::DEPTH, R = Sh::R;
  constexpr int CA = Sh::CB / 2;
  static_assert(CA * QUADS <= HELPERS, "one block of two channels and four tokens a helper");
  constexpr int NA = Sh::NP / 2, BBLOCKS = (LOCAL ? 1 : 2) * NA * QUADS, EB = (BBLOCKS + HELPERS - 1) / HELPERS;     // blocks of B, then of C
  const bool has_z = !LOCAL && p.z != nullptr, has_skip = p.D != nullptr;
  const int tiles = (int)(((long long)w.tokens + TILE - 1) / TILE);
  Bring<T, Sh::CB, Rw::XS, 3, ASYNC> bx({p.u, p.dt, p.z}, {p.ldu, p.lddt, p.ldz}, w.begin, w.d0, w.channels, w.tokens, tid);
  Bring<T, Sh::NP, Rw::NS, 2, ASYNC> bbc({p.B, p.C}, {p.ldb, p.ldc}, w.begin, (long long)w.group * p.Ns, p.Ns, w.tokens, tid);
  auto bring_tile = [&](int i) {
    if (i < tiles) {
      typename Rw::Slot& to = raw.slot[i % DEPTH];
      bx(to.x, has_z ? 3 : 2);
      bbc(to.bc, LOCAL ? 1 : 2);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  int c, quad;
  place(tid, CA, c, quad);
  c *= 2;
  const int j = 4 * quad;                            // first token of this thread in a tile
  const bool mine = CA * QUADS == HELPERS || quad < QUADS;
  const int channels = mine ? w.channels - c : 0;    // of this thread, two at most
  T* out = reinterpret_cast<T*>(p.out) + (w.begin + j) * p.ldo + w.d0 + c;
  float skip[2], bias[2];
#pragma unroll
  for (int v = 0; v < 2; v++) {
    const int d = w.d0 + (v < channels ? c + v : 0);
    skip[v] = has_skip ? p.D[d] : 0.0f;
    bias[v] = p.dt_bias != nullptr ? p.dt_bias[d] : 0.0f;
  }
  float* const row = mine ? &sh.step[c][j] : &sh.step[0][0];               // step, input, y lie CB rows apart
  constexpr int ARRAY = Sh::CB * R;
  P u[2][4], z[2][4];                                // kept for the outputs, two tiles later
  int left = w.tokens - j;                           // tokens from this thread's on, of the tile that is filled
  // outputs of the tile two in front
  auto store = [&](const P (&uo)[4], const P (&zo)[4], int stage) {
    const int have = left + 2 * TILE;
    if (channels > 0 && have > 0) {
      const float4 f0 = *reinterpret_cast<const float4*>(row + stage * TILE + 2 * ARRAY);
      const float4 f1 = *reinterpret_cast<const float4*>(row + stage * TILE + 2 * ARRAY + R);
      float y[4][2] = {{f0.x, f1.x}, {f0.y, f1.y}, {f0.z, f1.z}, {f0.w, f1.w}};
      if (has_skip) {                                // 0 times an infinite u would be NaN
#pragma unroll
        for (int k = 0; k < 4; k++) {
          float uf[2];
          unpack(uo[k], uf);
          y[k][0] = fmaf(skip[0], uf[0], y[k][0]);
          y[k][1] = fmaf(skip[1], uf[1], y[k][1]);
        }
      }
#pragma unroll
      for (int k = 0; k < 4; k++) {
        float zf[2];
        if (has_z) {
          unpack(zo[k], zf);
          y[k][0] *= silu<T>(zf[0]);
          y[k][1] *= silu<T>(zf[1]);
        }
      }
      T* to = out;
      if (ASYNC && have >= 4) {
#pragma unroll
        for (int k = 0; k < 4; k++, to += p.ldo) *reinterpret_cast<P*>(to) = pack<T, 2>(y[k]);
      } else {
#pragma unroll
        for (int k = 0; k < 4; k++, to += p.ldo)
          if (k < have) {
            to[0] = from_float<T>(y[k][0]);
            if (channels > 1) to[1] = from_float<T>(y[k][1]);
          }
      }
    }
    out += TILE * p.ldo;
  };
  auto tile = [&](int i, P (&ui)[4], P (&zi)[4], int stage) {
    const typename Rw::Slot& slot = raw.slot[i % DEPTH];
    asm volatile("cp.async.wait_group %0;" ::"n"(DEPTH - 2) : "memory");
    asm volatile("bar.sync %0, %1;" ::"n"((int)BAR_HELPERS), "n"(HELPERS) : "memory");         // tile i is here, tile i - 1 has been read
    bring_tile(i + DEPTH - 1);
    if (i >= 2) {
      bar_sync(BAR_DONE + stage);
      if constexpr (!LOCAL) store(ui, zi, stage);
    }
    if (mine) {
      const T* x = &slot.x[0][j][c];
      constexpr int X = TILE * Rw::XS;
      float uf[4][2], df[4][2];
#pragma unroll
      for (int k = 0; k < 4; k++) {
        ui[k] = *reinterpret_cast<const P*>(x + k * Rw::XS);
        unpack(ui[k], uf[k]);
        unpack(*reinterpret_cast<const P*>(x + k * Rw::XS + X), df[k]);
        if (has_z) zi[k] = *reinterpret_cast<const P*>(x + k * Rw::XS + 2 * X);
      }
#pragma unroll
      for (int v = 0; v < 2; v++) {
        F2 s01 = f2(df[0][v] + bias[v], df[1][v] + bias[v]), s23 = f2(df[2][v] + bias[v], df[3][v] + bias[v]);
        float s[4];
        split(s01, s[0], s[1]);
        split(s23, s[2], s[3]);
        if (p.softplus) {
          split(softplus2(s[0], s[1]), s[0], s[1]);
          split(softplus2(s[2], s[3]), s[2], s[3]);
        }
        if (left < 4)
#pragma unroll
          for (int k = 0; k < 4; k++)
            if (k >= left) s[k] = 0.0f;              // leaves the state as it is
        s01 = f2(s[0], s[1]);
        s23 = f2(s[2], s[3]);
        float* to = row + stage * TILE + v * R;
        *reinterpret_cast<ulonglong2*>(to) = make_ulonglong2(s01, s23);
        *reinterpret_cast<ulonglong2*>(to + ARRAY) = make_ulonglong2(mul2(s01, f2(uf[0][v], uf[1][v])), mul2(s23, f2(uf[2][v], uf[3][v])));
      }
    }
    left -= TILE;
#pragma unroll
    for (int e = 0; e < EB; e++) {
      int n, q;
      const int id = tid + e * HELPERS, second = id >= NA * QUADS;
      place(id % (NA * QUADS), NA, n, q);
      if (BBLOCKS % HELPERS != 0 && id >= BBLOCKS) continue;
      float f[4][2];
#pragma unroll
      for (int k = 0; k < 4; k++) unpack(*reinterpret_cast<const P*>(&slot.bc[second][4 * q + k][2 * n]), f[k]);
      float* to = (second ? &sh.c[0][0] : &sh.b[0][0]) + 2 * n * R + stage * TILE + 4 * q;
      *reinterpret_cast<float4*>(to) = make_float4(f[0][0], f[1][0], f[2][0], f[3][0]);
      *reinterpret_cast<float4*>(to + R) = make_float4(f[0][1], f[1][1], f[2][1], f[3][1]);
    }
    bar_arrive(BAR_FULL + stage);
  };
  for (int i = 0; i < DEPTH - 1; i++) bring_tile(i);
  for (int i = 0; i < tiles; i += 2) {
    tile(i, u[0], z[0], 0);
    if (i + 1 < tiles) tile(i + 1, u[1], z[1], 1);
  }
  // the last two tiles' outputs, in order; `left` counts as if the tiles behind them were filled
  if (tiles > 1) {
    const int stage = tiles & 1;
    bar_sync(BAR_DONE + stage);
    if constexpr (!LOCAL) stage ? store(u[1], z[1], 1) : store(u[0], z[0], 0);
    left -= TILE;
  } else {
    left -= TILE;
  }
  if (tiles > 0) {
    const int stage = (tiles - 1) & 1;
    bar_sync(BAR_DONE + stage);
    if constexpr (!LOCAL) stage ? store(u[1], z[1], 1) : store(u[0], z[0], 0);
  }
}

// The scan warps' half: lane l of a channel holds the state values l + k L.  A tile is one run of instructions, four tokens after
// four; tokens behind the last one leave the state as it is.
// LOCAL: the state alone, and the sum of the steps.
// PADDED: there are only `states` of the L S state values.  The places behind them hold B = C = 0, which an infinite step or s u turns
// into NaN (0 times inf): the sums take them as zeros, and nothing else reads them.  The lower half of a lane's places always has values.
// The ragged prompts with 13 values, and with 24 on 2048 channels: 336 and 286 us, without the care 335 and 279.
template <int L, int S, bool LOCAL, bool PADDED>
__device__ __forceinline__ void scan(const Work& w, ScanShared<L, S>& sh, int tid, int states, const float (&a)[CH][S], float (&h)[CH][S],
                                     float (&sum)[CH]) {
  constexpr int R = ScanShared<L, S>::R, NEXT = ScanShared<L, S>::CB / CH * R;
  constexpr int SUMS = 4;                            // tokens that are summed over the lanes at a time
  const int lane = tid % L, c = tid / L;
  const int tiles = (int)(((long long)w.tokens + TILE - 1) / TILE);
  for (int i = 0; i < tiles; i++) {
    const int stage = i & 1;
    bar_sync(BAR_FULL + stage);
    const float *step = &sh.step[c][stage * TILE], *input = &sh.input[c][stage * TILE];
    const float *b = &sh.b[lane][stage * TILE], *cc = &sh.c[lane][stage * TILE];
    float* out = &sh.y[c][stage * TILE + lane * SUMS / L];
#pragma unroll
    for (int j = 0; j < TILE; j += 4) {
      ulonglong2 st[CH], in[CH];
      F2 y01[CH], y23[CH];
#pragma unroll
      for (int m = 0; m < CH; m++) {
        st[m] = *reinterpret_cast<const ulonglong2*>(step + m * NEXT + j);
        in[m] = *reinterpret_cast<const ulonglong2*>(input + m * NEXT + j);
      }
#pragma unroll
      for (int k = 0; k < S; k++) {
        const ulonglong2 bk = *reinterpret_cast<const ulonglong2*>(b + k * L * R + j);
        ulonglong2 ck = {0, 0};
        if constexpr (!LOCAL) ck = *reinterpret_cast<const ulonglong2*>(cc + k * L * R + j);
#pragma unroll
        for (int m = 0; m < CH; m++) {
          const F2 ak = f2(a[m][k], a[m][k]);
          float x0, x1, x2, x3, i0, i1, i2, i3;
          split(mul2(st[m].x, ak), x0, x1);
          split(mul2(st[m].y, ak), x2, x3);
          split(mul2(in[m].x, bk.x), i0, i1);
          split(mul2(in[m].y, bk.y), i2, i3);
          const float h0 = fmaf(exp2_fast(x0), h[m][k], i0), h1 = fmaf(exp2_fast(x1), h0, i1), h2 = fmaf(exp2_fast(x2), h1, i2);
          h[m][k] = fmaf(exp2_fast(x3), h2, i3);
          if constexpr (!LOCAL) {
            F2 h01 = f2(h0, h1), h23 = f2(h2, h[m][k]);
            if (PADDED && k >= S / 2 && lane + k * L >= states) h01 = h23 = 0;
            y01[m] = k == 0 ? mul2(ck.x, h01) : fma2(ck.x, h01, y01[m]);
            y23[m] = k == 0 ? mul2(ck.y, h23) : fma2(ck.y, h23, y23[m]);
          }
        }
      }
#pragma unroll
      for (int m = 0; m < CH; m++) {
        if constexpr (LOCAL) {
          float s0, s1, s2, s3;
          split(st[m].x, s0, s1);
          split(st[m].y, s2, s3);
          sum[m] += (s0 + s1) + (s2 + s3);
        } else {
          float part[SUMS];
          split(y01[m], part[0], part[1]);
          split(y23[m], part[2], part[3]);
          // a step of the exchange leaves half of the tokens with each lane: lane l ends with the sum of token l SUMS / L (L > SUMS:
          // neighbours with the same one)
#pragma unroll
          for (int q = L / 2, n = SUMS / 2; q >= 1; q /= 2, n /= 2) {
            if (n >= 1) {
#pragma unroll
              for (int k = 0; k < n; k++) {
                const bool up = lane & q;
                const float give = up ? part[k] : part[n + k], keep = up ? part[n + k] : part[k];
                part[k] = keep + __shfl_xor_sync(0xffffffffu, give, q);
              }
            } else {
              part[0] += __shfl_xor_sync(0xffffffffu, part[0], q);
            }
          }
          out[m * NEXT + j] = part[0];
        }
      }
    }
    bar_arrive(BAR_DONE + stage);
  }
}

// A sequence, or a piece of one, and up to CB channels of one group a block.
template <typename T, int L, int S, bool LOCAL, bool ASYNC>
__global__ void __launch_bounds__(SCAN_THREADS, LOCAL ? 3 : 2) kda_selective_scan_kernel(const ScanParams p) {
  using Sh = ScanShared<L, S>;
  constexpr int CB = Sh::CB;
  extern __shared__ __align__(16) unsigned char smem[];
  Sh& sh = *reinterpret_cast<Sh*>(smem);
  RawShared<T, L, S>& raw = *reinterpret_cast<RawShared<T, L, S>*>(smem + sizeof(Sh));
  const int per = p.Dm / p.groups, gblocks = (per + CB - 1) / CB, block = blockIdx.x % (gblocks * p.groups);
  const int tid = threadIdx.x % SCAN_LANES;          // scan threads first
  const bool helper = threadIdx.x >= SCAN_LANES;
  Work w;
  w.group = block / gblocks;
  w.d0 = w.group * per + block % gblocks * CB;
  w.channels = min(CB, (w.group + 1) * per - w.d0);
  const bool rejected = cu_rejected(p.seq);
  w.at = blockIdx.x / (gblocks * p.groups);
  if (p.piece > 0) {
    if (!find_piece(p, rejected, w.at, w) || (LOCAL && w.piece + 1 == w.pieces)) return;
  } else {
    w.seq = p.seq.N > 1 && p.seq.N <= RANKED && gridDim.x > ROOM && !rejected ? by_length(p, w.at) : w.at;
    w.piece = 0;
    w.pieces = 1;
  }
  const long long slot = claim_slot(p.seq, w.seq);
  long long end = rejected ? 0 : cu_at(p.seq, w.seq + 1);
  w.begin = (rejected ? 0 : cu_at(p.seq, w.seq)) + (long long)w.piece * p.piece;
  if (w.piece + 1 < w.pieces) end = w.begin + p.piece;
  w.tokens = __reduce_max_sync(0xffffffffu, (int)(end - w.begin));       // the same in all lanes, and known to be: no divergence in the loops
  if (helper) {
    help<T, L, S, LOCAL, ASYNC>(p, w, sh, raw, tid);
    // rows behind the last sequence
    if (!LOCAL && w.seq == p.seq.N - 1 && w.piece + 1 == w.pieces && (rejected || p.zero_pad) && tid % CB < w.channels)
      for (long long t = end + tid / CB; t < p.seq.T; t += HELPERS / CB) reinterpret_cast<T*>(p.out)[t * p.ldo + w.d0 + tid % CB] = from_float<T>(0.0f);
    return;
  }
  const int lane = tid % L, c = tid / L;
  const long long rows = (long long)p.Dm * p.Ns;
  float* const own = p.ws_state + w.at * rows;       // a piece's state: first what it adds to the state, then the state it starts from
  const float* from = w.pieces > 1 ? own : (p.src != nullptr && slot >= 0 ? p.src + slot * p.src_stride : nullptr);
  float a[CH][S], h[CH][S], sum[CH];
#pragma unroll
  for (int m = 0; m < CH; m++) {
    const int cm = c + m * CB / CH;
    const long long at = (long long)(w.d0 + cm) * p.Ns + lane;
    sum[m] = 0.0f;
#pragma unroll
    for (int k = 0; k < S; k++) {
      const bool on = cm < w.channels && lane + k * L < p.Ns;
      a[m][k] = on ? decay_rate(p.A[at + k * L]) : 0.0f;
      h[m][k] = !LOCAL && on && from != nullptr ? from[at + k * L] : 0.0f;
    }
  }
  if (LOCAL || p.Ns == L * S) scan<L, S, LOCAL, false>(w, sh, tid, p.Ns, a, h, sum);
  else scan<L, S, LOCAL, !LOCAL>(w, sh, tid, p.Ns, a, h, sum);
  float* to = LOCAL ? own : (w.piece + 1 == w.pieces && p.dst != nullptr && slot >= 0 ? p.dst + slot * p.dst_stride : nullptr);
  if (to == nullptr) return;
#pragma unroll
  for (int m = 0; m < CH; m++) {
    const int cm = c + m * CB / CH;
    const long long at = (long long)(w.d0 + cm) * p.Ns + lane;
    if (cm >= w.channels) break;
#pragma unroll
    for (int k = 0; k < S; k++)
      if (lane + k * L < p.Ns) to[at + k * L] = h[m][k];
    if (LOCAL && lane == 0) p.ws_sum[(long long)w.at * p.Dm + w.d0 + cm] = sum[m];
  }
}

// Between the passes over pieces: from what each piece adds to the state (and exp(A sum of its steps), what it leaves of the
// state in front) to the state that each starts from.  A thread follows one state value through its sequence.
constexpr int JOIN_THREADS = 256;

// 2^x h + add where the product does not tell: step by step a state of zero stays zero however far the exponential is beyond fp32's
// range, an infinite one stays infinite however small it is, and a small state grows into the range.
__device__ __forceinline__ float join_rare(float x, float h, float add) {
  if (h != 0.0f && !isinf(h))
    for (int i = 0; i < 3; i++) {                    // 2^300 lifts the least state out of the range
      const float part = x > 100.0f ? 100.0f : x;
      h *= exp2_fast(part);
      x -= part;
    }
  return h + add;
}
__global__ void __launch_bounds__(JOIN_THREADS) kda_selective_scan_join_kernel(const ScanParams p) {
  const long long rows = (long long)p.Dm * p.Ns;
  const int blocks = (int)((rows + JOIN_THREADS - 1) / JOIN_THREADS), seq = blockIdx.x / blocks;
  const bool rejected = cu_rejected(p.seq);
  const int n = pieces_of(p, rejected, seq);
  if (n < 2) return;
  const long long slot = claim_slot(p.seq, seq);
  int first = 0;
  for (int i = threadIdx.x % 32; i < seq; i += 32) first += pieces_of(p, rejected, i);
  first = __reduce_add_sync(0xffffffffu, first);
  const long long at = (long long)(blockIdx.x % blocks) * JOIN_THREADS + threadIdx.x;
  if (at >= rows) return;
  const long long d = at / p.Ns;
  const float a = decay_rate(p.A[at]);
  float h = p.src != nullptr && slot >= 0 ? p.src[slot * p.src_stride + at] : 0.0f;
  float *state = p.ws_state + first * rows + at, *sums = p.ws_sum + (long long)first * p.Dm + d;
  constexpr int AHEAD = 8;
  for (int i0 = 0; i0 < n; i0 += AHEAD) {
    float add[AHEAD], keep[AHEAD], x[AHEAD];
    const float h0 = h;
    float most = 0.0f;
#pragma unroll
    for (int i = 0; i < AHEAD; i++) {
      const bool on = i0 + i + 1 < n;                // the last piece adds nothing here
      add[i] = on ? state[(i0 + i) * rows] : 0.0f;
      x[i] = on ? a * sums[(long long)(i0 + i) * p.Dm] : 0.0f;
      keep[i] = exp2_fast(x[i]);
      most = fmaxf(most, x[i]);
    }
#pragma unroll
    for (int i = 0; i < AHEAD; i++)
      if (i0 + i < n) {
        state[(i0 + i) * rows] = h;
        h = fmaf(keep[i], h, add[i]);
      }
    // finite exponentials and a finite state behind them: none of these steps was 0 times inf (inf and NaN stay, once in the state)
    if (fabsf(h) < INFINITY && most <= 127.0f) continue;
    h = h0;                                          // once more with care
#pragma unroll
    for (int i = 0; i < AHEAD; i++)
      if (i0 + i < n) {
        state[(i0 + i) * rows] = h;
        h = h == 0.0f || isinf(h) || x[i] > 127.0f ? join_rare(x[i], h, add[i]) : fmaf(keep[i], h, add[i]);
      }
  }
}

// One token a row, ROWS rows a block for one load of A (256 rows of 4096 channels, 16 values: 37 us, 3.8 TB/s; a row a block with
// every lane working out its step 57 us).  L lanes hold a channel's state, S consecutive values each; lane r works out
// the step, the gate and the output of row r and hands the step round.  Bound by memory: the states of all rows are asked for before
// anything else, and go through once.
constexpr int ROWS = 4;
template <typename T, int L, int S, bool WIDE>
__global__ void __launch_bounds__(STEP_LANES) kda_selective_scan_step_kernel(const ScanParams p) {
  static_assert(L >= ROWS, "a lane for each row");
  constexpr int CB = STEP_LANES / L;
  const int lane = threadIdx.x % L;
  const int row0 = blockIdx.y * ROWS, rows = min(ROWS, (int)p.seq.T - row0);
  const int d = (int)blockIdx.x * CB + threadIdx.x / L;
  const bool mine = d < p.Dm;
  const int dc = mine ? d : p.Dm - 1, group = p.groups > 1 ? dc / (p.Dm / p.groups) : 0, n = lane * S;
  int slot[ROWS];
  row_slots(p.seq, row0, rows, slot);
  const long long at = (long long)dc * p.Ns + n;
  // S consecutive values of a row of states: one access where WIDE
  auto values = [&](const float* q) {
    Values<S> v;
    if constexpr (WIDE) {
      v = load_values<S>(q);
    } else {
#pragma unroll
      for (int k = 0; k < S; k++) v.v[k] = n + k < p.Ns ? q[k] : 0.0f;
    }
    return v;
  };
  auto tokens = [&](const T* q) {
    Pack<T, S> v;
    if constexpr (WIDE) {
      v = *reinterpret_cast<const Pack<T, S>*>(q);
    } else {
#pragma unroll
      for (int k = 0; k < S; k++) v.v[k] = n + k < p.Ns ? q[k] : from_float<T>(0.0f);
    }
    return v;
  };
  Values<S> h[ROWS];
#pragma unroll
  for (int r = 0; r < ROWS; r++)
    if (slot[r] >= 0) h[r] = values(p.src + slot[r] * p.src_stride + at);
  // what a row of padding brings is worked on like the rest, and dropped: tokens that wait for the slots cost 43 us for the 256 rows
  // above instead of 37
  Pack<T, S> rb[ROWS], rc[ROWS];
  const T* B = reinterpret_cast<const T*>(p.B) + row0 * p.ldb + (long long)group * p.Ns + n;
  const T* C = reinterpret_cast<const T*>(p.C) + row0 * p.ldc + (long long)group * p.Ns + n;
#pragma unroll
  for (int r = 0; r < ROWS; r++) {
    rb[r] = tokens(B);
    rc[r] = tokens(C);
    if (r + 1 < rows) {
      B += p.ldb;
      C += p.ldc;
    }
  }
  // lane r: row r
  const long long mine_row = row0 + min(lane, rows - 1);
  const float u = to_float(reinterpret_cast<const T*>(p.u)[mine_row * p.ldu + dc]);
  float s = to_float(reinterpret_cast<const T*>(p.dt)[mine_row * p.lddt + dc]) + (p.dt_bias != nullptr ? p.dt_bias[dc] : 0.0f);
  const float z = p.z != nullptr ? to_float(reinterpret_cast<const T*>(p.z)[mine_row * p.ldz + dc]) : 0.0f;
  const float skip = p.D != nullptr ? p.D[dc] : 0.0f;
  Values<S> a = values(p.A + at);
#pragma unroll
  for (int k = 0; k < S; k++) a.v[k] = decay_rate(a.v[k]);
  if (p.softplus) s = softplus(s);
  const float su = s * u;
  if (drop_repeats(p.seq, row0, slot)) {
#pragma unroll
    for (int r = 0; r < ROWS; r++)
      if (slot[r] < 0) h[r] = Values<S>();
  }
  float part[ROWS];
#pragma unroll
  for (int r = 0; r < ROWS; r++) {
    const float sr = __shfl_sync(0xffffffffu, s, r, L), sur = __shfl_sync(0xffffffffu, su, r, L);
    float b[S], c[S];
    unpack(rb[r], b);
    unpack(rc[r], c);
#pragma unroll
    for (int k = 0; k < S; k++) {
      h[r].v[k] = fmaf(exp2_fast(sr * a.v[k]), h[r].v[k], sur * b[k]);
      part[r] = k == 0 ? c[k] * h[r].v[k] : fmaf(c[k], h[r].v[k], part[r]);
    }
    // places behind the state values hold B = C = 0, which an infinite s u turns into NaN (0 times inf): a sum without them
    if (!WIDE && !(fabsf(sur) < INFINITY)) {
      part[r] = 0.0f;
#pragma unroll
      for (int k = 0; k < S; k++)
        if (n + k < p.Ns) part[r] = fmaf(c[k], h[r].v[k], part[r]);
    }
    if (slot[r] >= 0 && mine) {
      float* to = p.dst + slot[r] * p.dst_stride + at;
      if constexpr (WIDE) {
        store_values<S>(to, h[r]);
      } else {
#pragma unroll
        for (int k = 0; k < S; k++)
          if (n + k < p.Ns) to[k] = h[r].v[k];
      }
    }
  }
  // sums over the lanes: lane r ends with row r (L > ROWS: the first of L / ROWS lanes, which hands it on)
#pragma unroll
  for (int m = L / 2, k = ROWS / 2; m >= 1; m /= 2, k /= 2) {
    if (k >= 1) {
#pragma unroll
      for (int r = 0; r < k; r++) {
        const bool up = lane & m;
        const float give = up ? part[r] : part[k + r], keep = up ? part[k + r] : part[r];
        part[r] = keep + __shfl_xor_sync(0xffffffffu, give, m);
      }
    } else {
      part[0] += __shfl_xor_sync(0xffffffffu, part[0], m);
    }
  }
  float y = __shfl_sync(0xffffffffu, part[0], min(lane, ROWS - 1) * (L / ROWS), L);
  int own = -2;
#pragma unroll
  for (int r = 0; r < ROWS; r++)
    if (lane == r) own = slot[r];
  if (lane >= rows || !mine) return;
  T* out = reinterpret_cast<T*>(p.out) + mine_row * p.ldo + dc;
  if (own == -2) {
    if (p.zero_pad) *out = from_float<T>(0.0f);
    return;
  }
  y = fmaf(skip, fabsf(u) < INFINITY || p.D != nullptr ? u : 0.0f, y);       // 0 times an infinite u would be NaN
  if (p.z != nullptr) y *= silu<T>(z);
  *out = from_float<T>(y);
}

template <typename T, int L, int S, bool LOCAL, bool ASYNC>
cudaError_t launch_copies(const ScanParams& p, long long pieces, cudaStream_t stream) {
  constexpr int bytes = sizeof(ScanShared<L, S>) + sizeof(RawShared<T, L, S>), CB = ScanShared<L, S>::CB;
  const long long blocks = (long long)((p.Dm / p.groups + CB - 1) / CB) * p.groups * pieces;
  if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
  const cudaError_t e = cudaFuncSetAttribute(kda_selective_scan_kernel<T, L, S, LOCAL, ASYNC>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) return e;
  kda_selective_scan_kernel<T, L, S, LOCAL, ASYNC><<<(unsigned)blocks, SCAN_THREADS, bytes, stream>>>(p);
  return cudaGetLastError();
}

template <typename T, int L, int S, bool LOCAL>
cudaError_t launch_pass(const ScanParams& p, long long pieces, cudaStream_t stream) {
  return p.async ? launch_copies<T, L, S, LOCAL, true>(p, pieces, stream) : launch_copies<T, L, S, LOCAL, false>(p, pieces, stream);
}

template <typename T, int L, int S>
cudaError_t launch_lanes(const ScanParams& p, cudaStream_t stream) {
  if (p.piece == 0) return launch_pass<T, L, S, false>(p, p.seq.N, stream);
  const long long pieces = p.seq.T / p.piece + p.seq.N;
  cudaError_t e = launch_pass<T, L, S, true>(p, pieces, stream);
  if (e != cudaSuccess) return e;
  const long long rows = (long long)p.Dm * p.Ns, blocks = (rows + JOIN_THREADS - 1) / JOIN_THREADS * p.seq.N;
  if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
  kda_selective_scan_join_kernel<<<(unsigned)blocks, JOIN_THREADS, 0, stream>>>(p);
  e = cudaGetLastError();
  return e != cudaSuccess ? e : launch_pass<T, L, S, false>(p, pieces, stream);
}

// Whether the rows that `p` and `ld` name start on 16 bytes, and are whole 16 bytes wide.
template <typename T>
bool rows16(const void* p, long long ld, long long width) {
  return ((reinterpret_cast<uintptr_t>(p) | (uintptr_t)(ld * (long long)sizeof(T)) | (uintptr_t)(width * (long long)sizeof(T))) & 15) == 0;
}

template <typename T>
cudaError_t launch_type(ScanParams p, cudaStream_t stream) {
  const long long per = p.Dm / p.groups;
  p.async = rows16<T>(p.u, p.ldu, per) && rows16<T>(p.dt, p.lddt, per) && rows16<T>(p.z, p.ldz, per) && rows16<T>(p.out, p.ldo, per) &&
            rows16<T>(p.B, p.ldb, p.Ns) && rows16<T>(p.C, p.ldc, p.Ns);
  if (p.Ns <= 4) return launch_lanes<T, 4, 1>(p, stream);
  if (p.Ns <= 8) return launch_lanes<T, 4, 2>(p, stream);
  if (p.Ns <= 16) return launch_lanes<T, 4, 4>(p, stream);
  if (p.Ns <= 32) return launch_lanes<T, 8, 4>(p, stream);
  if (p.Ns <= 64) return launch_lanes<T, 16, 4>(p, stream);
  return launch_lanes<T, 32, 4>(p, stream);
}

template <typename T, int L, int S>
cudaError_t launch_step(const ScanParams& p, cudaStream_t stream) {
  const long long rows = (p.seq.T + ROWS - 1) / ROWS;
  if (rows == 0) return cudaSuccess;
  if (rows > 65535) return cudaErrorInvalidValue;
  const dim3 grid((unsigned)((p.Dm + STEP_LANES / L - 1) / (STEP_LANES / L)), (unsigned)rows);
  // one access for S values where all start on as many and no lane has fewer
  const uintptr_t f = reinterpret_cast<uintptr_t>(p.src) | reinterpret_cast<uintptr_t>(p.A) | (uintptr_t)(p.src_stride * 4);
  const uintptr_t t = reinterpret_cast<uintptr_t>(p.B) | reinterpret_cast<uintptr_t>(p.C) | (uintptr_t)((p.ldb | p.ldc) * (long long)sizeof(T));
  if ((f & (S * 4 - 1)) == 0 && (t & (S * sizeof(T) - 1)) == 0 && p.Ns == L * S) kda_selective_scan_step_kernel<T, L, S, true><<<grid, STEP_LANES, 0, stream>>>(p);
  else kda_selective_scan_step_kernel<T, L, S, false><<<grid, STEP_LANES, 0, stream>>>(p);
  return cudaGetLastError();
}

template <typename T>
cudaError_t launch_step_type(const ScanParams& p, cudaStream_t stream) {
  if (p.Ns <= 4) return launch_step<T, 4, 1>(p, stream);
  if (p.Ns <= 8) return launch_step<T, 4, 2>(p, stream);
  if (p.Ns <= 16) return launch_step<T, 4, 4>(p, stream);
  if (p.Ns <= 32) return launch_step<T, 8, 4>(p, stream);
  if (p.Ns <= 64) return launch_step<T, 16, 4>(p, stream);
  return launch_step<T, 32, 4>(p, stream);
}

}  // namespace

// Where whole sequences would leave SMs without work, they are cut: a first pass over the pieces finds what each adds to the
// state, the states are joined, a second pass computes the outputs.  That is about 1.6 times the work, for two rounds of blocks
// that fill the card (two an SM): 0 = no cut, else the tokens of a piece.  The lengths lie on the device, so the rule goes by the
// number of sequences, and by all channels together: groups that end inside a block launch more blocks than it counts, so that
// small groups get shorter pieces than two rounds.  32 768 tokens on 512 channels: uncut 1725 us, two rounds of pieces 207 us, four 218 us,
// eight 241 us; 8192 tokens on 4096 channels (64 blocks uncut, 160 cycles a token: some 690 us) 379 us.
long long sscan_piece(long long T, int N, int Dm, int Ns) {
  const int lanes = Ns <= 16 ? 4 : (Ns <= 32 ? 8 : (Ns <= 64 ? 16 : 32));
  const long long blocks = (Dm + CH * SCAN_LANES / lanes - 1) / (CH * SCAN_LANES / lanes);
  if (blocks * N >= ROOM || N > ROOM || T < 512) return 0;
  const long long piece = (T * blocks / (2 * ROOM) + TILE - 1) / TILE * TILE;
  return piece < 128 ? 128 : piece;
}

cudaError_t launch_sscan(const ScanParams& p, int type, cudaStream_t stream) {
  if (type == TYPE_BF16) return launch_type<__nv_bfloat16>(p, stream);
  if (type == TYPE_FP16) return launch_type<__half>(p, stream);
  return launch_type<float>(p, stream);
}

cudaError_t launch_sscan_step(const ScanParams& p, int type, cudaStream_t stream) {
  if (type == TYPE_BF16) return launch_step_type<__nv_bfloat16>(p, stream);
  if (type == TYPE_FP16) return launch_step_type<__half>(p, stream);
  return launch_step_type<float>(p, stream);
}

}  // namespace kda
