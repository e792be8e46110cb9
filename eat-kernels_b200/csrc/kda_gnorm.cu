// Norm of groups of channels of a token, with an activation, and its gradients.  Of a group's D values x:
//   xh = (x - mean) rsqrt(mean((x - mean)^2) + eps)  (mean 0 without `center`),  n = xh w + b,  y = n act(z), or act(n) without z
//   dn = dy act(z) | dy act'(n);  dz = dy n act'(z);  dw = sum xh dn;  db = sum dn;  k = dn w
//   dx = (k - mean(k) - xh mean(k xh)) rstd            (without mean(k) without `center`)
// Bound by memory: x, z (and dy) are read once and stay in registers, mean and squares are taken of the values there.  A group lies
// in `lanes` neighbouring lanes; a thread keeps its channels for all the rows that it goes over, so that weights are read and their
// gradients summed in registers.  Measured in bf16: 20 000 rows of 32 groups of 128, gated, one weight for all, 99 us (5.0 TB/s); 8192 rows of
// 16 groups of 256 with all gradients 176 us for both passes (3.0 TB/s), in fp32 76 us forward and 112 for the gradients (5.3 and 6.0 TB/s).  Groups wider
// than a warp holds are a block's work, which reads them again out of the caches: 16 384 rows of 4096 channels as one group 169 us forward (2.4 TB/s),
// 1069 for the gradients.  Lanes of a group are a power of two: widths of 80, 160 and 320 leave three eighths of them idle (176, 179 and 255 us where
// 128 takes 116).  Gradients with 32 single values a lane take 255 registers and spill 64 (fp32) or 112 bytes.
#include "kda_serving.cuh"

namespace kda {

namespace {

constexpr int THREADS = 256, WARPS = THREADS / 32;
constexpr int BLOCKS = 2 * 148;          // of a gradient launch, about: each leaves a row of partial sums (three and four an SM: no gain)

struct Act {
  float a, slope;
};
template <typename T>
__device__ __forceinline__ Act activation(float v, int act) {
  Act r;
  if (act == ACT_NONE) {
    r.a = v; r.slope = 1.0f;
    return r;
  }
  float s, n;
  sigmoid_pair<T>(v, 0.0f, s, n);
  if (act == ACT_SIGMOID) {
    r.a = s; r.slope = s * n;
  } else {
    r.a = v * s; r.slope = s * fmaf(v, n, 1.0f);
  }
  return r;
}

template <int N>
__device__ __forceinline__ void add_lanes(float (&v)[N], int lanes) {
#pragma unroll
  for (int m = 16; m > 0; m /= 2) {
    if (m >= lanes) continue;
#pragma unroll
    for (int i = 0; i < N; i++) v[i] += __shfl_xor_sync(0xffffffffu, v[i], m);
  }
}

// Which group and rows a thread has: blocks of THREADS / lanes groups side by side; where a token has fewer, a block takes several rows
// at once.
struct Place {
  int g, row, rows;        // group (or -1: none), row among the block's first ones, how many those are
};
__device__ __forceinline__ Place place(int G, int lanes) {
  const int per = THREADS / lanes, q = threadIdx.x / lanes;
  Place a;
  if (G >= per) {
    a.rows = 1; a.row = 0;
    a.g = (int)blockIdx.x * per + q < G ? (int)blockIdx.x * per + q : -1;
  } else {
    a.rows = per / G; a.row = q / G;
    a.g = a.row < a.rows ? q % G : -1;
  }
  return a;
}

template <typename T, int VEC, int CH>
struct Values {
  Pack<T, VEC> v[CH];
};

// CH accesses of VEC values a thread, `lanes` threads a group
template <typename T, int VEC, int CH, bool GRAD>
__global__ void __launch_bounds__(THREADS, VEC * CH <= 8 ? (GRAD ? 2 : 4) : (VEC * CH <= 16 && !GRAD ? 2 : 1)) kda_group_norm_kernel(const GroupNormParams p) {
  using P = Pack<T, VEC>;
  const Place at = place(p.G, p.lanes);
  const int lane = threadIdx.x % p.lanes, D = p.D;
  const bool gated = p.z != nullptr;
  const float inv_d = 1.0f / (float)D;
  const long long base = (long long)(at.g < 0 ? 0 : at.g) * D;
  float w[CH][VEC], b[CH][VEC], dw[CH][VEC], db[CH][VEC];
  bool on[CH];
#pragma unroll
  for (int j = 0; j < CH; j++) {
    const int d = (j * p.lanes + lane) * VEC;
    on[j] = at.g >= 0 && d < D;
#pragma unroll
    for (int k = 0; k < VEC; k++) {
      const long long e = (p.shared ? 0 : base) + d + k;
      w[j][k] = on[j] && p.weight != nullptr ? p.weight[e] : 1.0f;
      b[j][k] = on[j] && p.bias != nullptr ? p.bias[e] : 0.0f;
      dw[j][k] = db[j][k] = 0.0f;
    }
  }
  const long long step = (long long)at.rows * p.parts;
  Values<T, VEC, CH> x, z, dy;
  auto ask = [&](long long row) {                    // places of no row or channel: zeros
    const bool live = row < p.T;
#pragma unroll
    for (int j = 0; j < CH; j++) {
      const long long d = base + (j * p.lanes + lane) * VEC;
      const bool here = on[j] && live;
#pragma unroll
      for (int k = 0; k < VEC; k++) x.v[j].v[k] = z.v[j].v[k] = dy.v[j].v[k] = from_float<T>(0.0f);
      if (here) x.v[j] = *reinterpret_cast<const P*>(reinterpret_cast<const T*>(p.x) + row * p.ldx + d);
      if (here && gated) z.v[j] = *reinterpret_cast<const P*>(reinterpret_cast<const T*>(p.z) + row * p.ldz + d);
      if (GRAD && here) dy.v[j] = *reinterpret_cast<const P*>(reinterpret_cast<const T*>(p.dy) + row * p.lddy + d);
    }
  };
  // gradients: a row is on its way while the one in front is worked on, where registers allow (the forward pass has warps enough and
  // loses by it: 20 000 rows of 32 groups of 128 99 us without, 113 with)
  constexpr bool AHEAD = GRAD && VEC * CH <= 16;
  if (AHEAD) ask((long long)blockIdx.y * at.rows + at.row);
  for (long long row0 = (long long)blockIdx.y * at.rows; row0 < p.T; row0 += step) {
    const long long row = row0 + at.row;
    const bool live = row < p.T;
    if (!AHEAD) ask(row);
    const Values<T, VEC, CH> zc = z, dyc = dy;
    float xh[CH][VEC], sum[1] = {0.0f};
#pragma unroll
    for (int j = 0; j < CH; j++) {
      unpack(x.v[j], xh[j]);
#pragma unroll
      for (int k = 0; k < VEC; k++) sum[0] += xh[j][k];
    }
    if (AHEAD) ask(row + step);
    if (p.center) {
      add_lanes(sum, p.lanes);
      const float mean = sum[0] * inv_d;
#pragma unroll
      for (int j = 0; j < CH; j++)
#pragma unroll
        for (int k = 0; k < VEC; k++) xh[j][k] = on[j] ? xh[j][k] - mean : 0.0f;
    }
    sum[0] = 0.0f;
#pragma unroll
    for (int j = 0; j < CH; j++)
#pragma unroll
      for (int k = 0; k < VEC; k++) sum[0] = fmaf(xh[j][k], xh[j][k], sum[0]);
    add_lanes(sum, p.lanes);
    const float rstd = rsqrtf(fmaf(sum[0], inv_d, p.eps));
    if constexpr (!GRAD) {
#pragma unroll
      for (int j = 0; j < CH; j++) {
        float y[VEC], zf[VEC];
        unpack(zc.v[j], zf);
#pragma unroll
        for (int k = 0; k < VEC; k++) {
          const float n = fmaf(xh[j][k] * rstd, w[j][k], b[j][k]);
          y[k] = gated ? n * activation<T>(zf[k], p.act).a : activation<T>(n, p.act).a;
        }
        if (on[j] && live) *reinterpret_cast<P*>(reinterpret_cast<T*>(p.out) + row * p.ldo + base + (j * p.lanes + lane) * VEC) = pack<T, VEC>(y);
      }
    } else {
      float kk[CH][VEC], sums[2] = {0.0f, 0.0f};
#pragma unroll
      for (int j = 0; j < CH; j++) {
        float zf[VEC], g[VEC], dz[VEC];
        unpack(zc.v[j], zf);
        unpack(dyc.v[j], g);
#pragma unroll
        for (int k = 0; k < VEC; k++) {
          xh[j][k] *= rstd;
          const float n = fmaf(xh[j][k], w[j][k], b[j][k]);
          const Act a = activation<T>(gated ? zf[k] : n, p.act);
          dz[k] = g[k] * n * a.slope;
          const float dn = g[k] * (gated ? a.a : a.slope);
          if (on[j] && live) {                       // places of no row may be NaN: an infinite value's sum is
            dw[j][k] = fmaf(xh[j][k], dn, dw[j][k]);
            db[j][k] += dn;
          }
          kk[j][k] = on[j] ? dn * w[j][k] : 0.0f;
          sums[0] += kk[j][k];
          sums[1] = fmaf(kk[j][k], xh[j][k], sums[1]);
        }
        if (gated && on[j] && live) *reinterpret_cast<P*>(reinterpret_cast<T*>(p.dz) + row * p.lddz + base + (j * p.lanes + lane) * VEC) = pack<T, VEC>(dz);
      }
      add_lanes(sums, p.lanes);
      const float m0 = p.center ? sums[0] * inv_d : 0.0f, m1 = sums[1] * inv_d;
#pragma unroll
      for (int j = 0; j < CH; j++) {
        float dx[VEC];
#pragma unroll
        for (int k = 0; k < VEC; k++) dx[k] = (kk[j][k] - m0 - xh[j][k] * m1) * rstd;
        if (on[j] && live) *reinterpret_cast<P*>(reinterpret_cast<T*>(p.out) + row * p.ldo + base + (j * p.lanes + lane) * VEC) = pack<T, VEC>(dx);
      }
    }
  }
  if constexpr (GRAD) {
    if (p.partial == nullptr) return;
    // the block's sums: [2][columns] of a row of `partial`; threads that share a channel add one after the other
    extern __shared__ float s_sum[];
    const bool alone = at.rows == 1 && !p.shared;
    const int cols = p.shared ? D : p.G * D;
    float* to = p.partial + ((long long)blockIdx.y * (p.shared ? gridDim.x : 1) + (p.shared ? blockIdx.x : 0)) * 2 * cols;
    if (alone) {
#pragma unroll
      for (int j = 0; j < CH; j++)
#pragma unroll
        for (int k = 0; k < VEC; k++)
          if (on[j]) {
            to[base + (j * p.lanes + lane) * VEC + k] = dw[j][k];
            to[cols + base + (j * p.lanes + lane) * VEC + k] = db[j][k];
          }
      return;
    }
    for (int i = threadIdx.x; i < 2 * cols; i += THREADS) s_sum[i] = 0.0f;
    // turns: of the rows (each group has its own channels), with `shared` of every group's lanes
    const int per = THREADS / p.lanes, turns = p.shared ? per : at.rows, mine = p.shared ? (int)threadIdx.x / p.lanes : at.row;
    for (int turn = 0; turn < turns; turn++) {
      __syncthreads();
      if (mine != turn || at.g < 0) continue;
#pragma unroll
      for (int j = 0; j < CH; j++)
#pragma unroll
        for (int k = 0; k < VEC; k++)
          if (on[j]) {
            const int e = (p.shared ? 0 : (int)base) + (j * p.lanes + lane) * VEC + k;
            s_sum[e] += dw[j][k];
            s_sum[cols + e] += db[j][k];
          }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * cols; i += THREADS) to[i] = s_sum[i];
  }
}

template <int N>
__device__ __forceinline__ void add_block(float (&v)[N], float (*s)[WARPS]) {
  add_lanes(v, 32);
  __syncthreads();                                   // the values of the sum before this one have been read
  if (threadIdx.x % 32 == 0)
#pragma unroll
    for (int i = 0; i < N; i++) s[i][threadIdx.x / 32] = v[i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; i++) {
    v[i] = 0.0f;
    for (int w = 0; w < WARPS; w++) v[i] += s[i][w];
  }
}

// Wide groups: a block for a group of a row, blockIdx.x the group
template <typename T, bool GRAD>
__global__ void __launch_bounds__(THREADS) kda_group_norm_wide_kernel(const GroupNormParams p) {
  extern __shared__ float s_sum[];                   // gradients: [2][D]
  __shared__ float s_add[2][WARPS];
  const int D = p.D, tid = threadIdx.x;
  const bool gated = p.z != nullptr, sums = GRAD && p.partial != nullptr;
  const float inv_d = 1.0f / (float)D;
  const long long base = (long long)blockIdx.x * D, wbase = p.shared ? 0 : base;
  if (sums)
    for (int d = tid; d < 2 * D; d += THREADS) s_sum[d] = 0.0f;          // a thread's own channels
  if (sums) __syncthreads();
  for (long long row = blockIdx.y; row < p.T; row += p.parts) {
    const T* x = reinterpret_cast<const T*>(p.x) + row * p.ldx + base;
    const T* z = reinterpret_cast<const T*>(p.z) + row * p.ldz + base;
    const T* dy = reinterpret_cast<const T*>(p.dy) + row * p.lddy + base;
    T* out = reinterpret_cast<T*>(p.out) + row * p.ldo + base;
    T* dz = reinterpret_cast<T*>(p.dz) + row * p.lddz + base;
    float mean = 0.0f, v[1] = {0.0f};
    if (p.center) {
      for (int d = tid; d < D; d += THREADS) v[0] += to_float(x[d]);
      add_block(v, s_add);
      mean = v[0] * inv_d;
    }
    v[0] = 0.0f;
    for (int d = tid; d < D; d += THREADS) {
      const float e = to_float(x[d]) - mean;
      v[0] = fmaf(e, e, v[0]);
    }
    add_block(v, s_add);
    const float rstd = rsqrtf(fmaf(v[0], inv_d, p.eps));
    auto value = [&](int d, float& xh, float& n, float& w) {
      xh = (to_float(x[d]) - mean) * rstd;
      w = p.weight != nullptr ? p.weight[wbase + d] : 1.0f;
      n = fmaf(xh, w, p.bias != nullptr ? p.bias[wbase + d] : 0.0f);
    };
    float xh, n, w;
    if constexpr (!GRAD) {
      for (int d = tid; d < D; d += THREADS) {
        value(d, xh, n, w);
        out[d] = from_float<T>(gated ? n * activation<T>(to_float(z[d]), p.act).a : activation<T>(n, p.act).a);
      }
    } else {
      float m[2] = {0.0f, 0.0f};
      for (int d = tid; d < D; d += THREADS) {
        value(d, xh, n, w);
        const float g = to_float(dy[d]);
        const Act a = activation<T>(gated ? to_float(z[d]) : n, p.act);
        const float dn = g * (gated ? a.a : a.slope);
        if (gated) dz[d] = from_float<T>(g * n * a.slope);
        if (sums) {
          s_sum[d] = fmaf(xh, dn, s_sum[d]);
          s_sum[D + d] += dn;
        }
        m[0] += dn * w;
        m[1] = fmaf(dn * w, xh, m[1]);
      }
      add_block(m, s_add);
      m[0] = p.center ? m[0] * inv_d : 0.0f;
      m[1] *= inv_d;
      for (int d = tid; d < D; d += THREADS) {
        value(d, xh, n, w);
        const float dn = to_float(dy[d]) * (gated ? activation<T>(to_float(z[d]), p.act).a : activation<T>(n, p.act).slope);
        out[d] = from_float<T>((dn * w - m[0] - xh * m[1]) * rstd);
      }
    }
  }
  if (sums) {
    const int cols = p.shared ? D : p.G * D;
    float* to = p.partial + (p.shared ? (long long)blockIdx.y * gridDim.x + blockIdx.x : (long long)blockIdx.y) * 2 * cols + wbase;
    for (int d = tid; d < D; d += THREADS) {
      to[d] = s_sum[d];
      to[cols + d] = s_sum[D + d];
    }
  }
}

// Sums of the rows of `partial`, 32 columns a block, in one order whatever the timing
__global__ void __launch_bounds__(THREADS) kda_group_norm_sum_kernel(const float* partial, int rows, int cols, float* dweight, float* dbias) {
  __shared__ float s[WARPS][32];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const long long c = (long long)blockIdx.x * 32 + lane;
  constexpr int AT_ONCE = 8;                         // rows asked for together: 148 of them and 8192 columns 6.7 us, one by one 11.4
  float v = 0.0f;
  if (c < 2LL * cols)
    for (int r0 = warp; r0 < rows; r0 += AT_ONCE * WARPS) {
      float f[AT_ONCE];
#pragma unroll
      for (int k = 0; k < AT_ONCE; k++) f[k] = r0 + k * WARPS < rows ? partial[(long long)(r0 + k * WARPS) * 2 * cols + c] : 0.0f;
#pragma unroll
      for (int k = 0; k < AT_ONCE; k++) v += f[k];
    }
  s[warp][lane] = v;
  __syncthreads();
  if (warp != 0 || c >= 2LL * cols) return;
  v = 0.0f;
#pragma unroll
  for (int w = 0; w < WARPS; w++) v += s[w][lane];
  float* to = c < cols ? dweight : dbias;
  if (to != nullptr) to[c < cols ? c : c - cols] = v;
}

bool on16(const void* p, long long ld, int size) { return ((reinterpret_cast<uintptr_t>(p) | (uintptr_t)(ld * size)) & 15) == 0; }

struct Shape {
  int ch, lanes;           // ch 0: a block for a group
  long long blocks;        // side by side
  long long parts(long long T, int G, bool grad) const {
    const int per = ch > 0 ? THREADS / lanes : 1, rows = ch > 0 && G < per ? per / G : 1;
    const long long need = (T + rows - 1) / rows, room = (grad ? BLOCKS : 8 * BLOCKS) / blocks;
    const long long n = need < room ? need : room;
    return n < 1 ? 1 : (n > 65535 ? 65535 : n);
  }
};
// `vec` values an access.  Forward a lane has 16 values at most, in gradients four accesses, of single values 32.  Forward, eight gated groups a row:
// 15 625 rows of 320 in fp32 166 us with 16 values a lane, 595 as a block's work, 9765 of 512 119 and 398; in bf16 13 020 rows of 768 385 with
// 32 a lane, 360 as a block's work, 9765 of 1024 367 and 291.  Gradients of 4096 rows of four groups of 1024 in bf16 97 and 258 us.  (Single values:
// groups of 127 take 240 us where 128 take 99.)
Shape shape_of(int G, int D, int vec, bool grad) {
  Shape s = {1, 4, 0};
  const int need = (D + vec - 1) / vec, most = vec > 1 ? (grad ? 4 : 16 / vec) : 32;
  while (s.lanes < 32 && s.lanes < need) s.lanes *= 2;
  while (s.ch <= most && s.ch * s.lanes < need) s.ch *= 2;
  if (s.ch > most) s.ch = 0;
  const int per = THREADS / s.lanes;
  s.blocks = s.ch == 0 ? G : (G >= per ? (G + per - 1) / per : 1);
  return s;
}

template <typename T, int VEC, int CH, bool GRAD>
cudaError_t launch_one(const GroupNormParams& p, const dim3& grid, cudaStream_t stream) {
  const int bytes = GRAD && p.partial != nullptr && (p.shared || p.G < THREADS / p.lanes) ? 2 * 4 * (p.shared ? p.D : p.G * p.D) : 0;
  constexpr int most = 2 * 4 * THREADS * VEC * CH;   // whatever this call needs: another thread may be about to launch one that needs more
  if (GRAD && most > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(kda_group_norm_kernel<T, VEC, CH, GRAD>, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
    if (e != cudaSuccess) return e;
  }
  kda_group_norm_kernel<T, VEC, CH, GRAD><<<grid, THREADS, bytes, stream>>>(p);
  return cudaGetLastError();
}

template <typename T, bool GRAD>
cudaError_t launch_wide(const GroupNormParams& p, const dim3& grid, cudaStream_t stream) {
  const int bytes = GRAD && p.partial != nullptr ? 8 * p.D : 0;
  if (GRAD) {
    const cudaError_t e = cudaFuncSetAttribute(kda_group_norm_wide_kernel<T, GRAD>, cudaFuncAttributeMaxDynamicSharedMemorySize, 8 * GROUP_NORM_MAX_WIDTH);
    if (e != cudaSuccess) return e;
  }
  kda_group_norm_wide_kernel<T, GRAD><<<grid, THREADS, bytes, stream>>>(p);
  return cudaGetLastError();
}

template <typename T, bool GRAD>
cudaError_t launch_type(GroupNormParams p, cudaStream_t stream) {
  constexpr int VEC = 16 / sizeof(T);
  const int size = sizeof(T);
  const bool wide = p.D % VEC == 0 && on16(p.x, p.ldx, size) && on16(p.z, p.ldz, size) && on16(p.dy, p.lddy, size) && on16(p.out, p.ldo, size) &&
                    on16(p.dz, p.lddz, size);
  const Shape s = shape_of(p.G, p.D, wide ? VEC : 1, GRAD);
  p.lanes = s.lanes;
  p.parts = (int)s.parts(p.T, p.G, GRAD);
  const dim3 grid((unsigned)s.blocks, (unsigned)p.parts);
  cudaError_t e;
  if (p.T == 0) e = cudaSuccess;
  else if (s.ch == 0) e = launch_wide<T, GRAD>(p, grid, stream);
  else if (wide && s.ch <= 2) e = s.ch == 1 ? launch_one<T, VEC, 1, GRAD>(p, grid, stream) : launch_one<T, VEC, 2, GRAD>(p, grid, stream);
  else if (wide) e = launch_one<T, VEC, 4, GRAD || VEC == 8>(p, grid, stream);       // 16 bits: gradients only
  else if (s.ch <= 4) e = launch_one<T, 1, 4, GRAD>(p, grid, stream);
  else if (s.ch <= 8) e = launch_one<T, 1, 8, GRAD>(p, grid, stream);
  else if (s.ch <= 16) e = launch_one<T, 1, 16, GRAD>(p, grid, stream);
  else e = launch_one<T, 1, 32, GRAD>(p, grid, stream);
  if (!GRAD || e != cudaSuccess || p.partial == nullptr) return e;
  const int cols = p.shared ? p.D : p.G * p.D, rows = p.T == 0 ? 0 : p.parts * (p.shared ? (int)s.blocks : 1);
  kda_group_norm_sum_kernel<<<(unsigned)((2LL * cols + 31) / 32), THREADS, 0, stream>>>(p.partial, rows, cols, p.dweight, p.dbias);
  return cudaGetLastError();
}

template <bool GRAD>
cudaError_t launch_any(const GroupNormParams& p, int type, cudaStream_t stream) {
  if (type == TYPE_BF16) return launch_type<__nv_bfloat16, GRAD>(p, stream);
  if (type == TYPE_FP16) return launch_type<__half, GRAD>(p, stream);
  return launch_type<float, GRAD>(p, stream);
}

}  // namespace

// The larger of what aligned and other rows take
long long group_norm_partial_floats(long long T, int G, int D, int type, bool shared) {
  long long most = 0;
  for (int vec : {1, type == TYPE_FP32 ? 4 : 8}) {
    const Shape s = shape_of(G, D, vec, true);
    const long long n = s.parts(T, G, true) * (shared ? s.blocks : 1) * 2 * (shared ? D : (long long)G * D);
    if (n > most) most = n;
  }
  return most;
}

cudaError_t launch_group_norm(const GroupNormParams& p, int type, cudaStream_t stream) {
  if (p.T == 0) return cudaSuccess;
  return launch_any<false>(p, type, stream);
}
cudaError_t launch_group_norm_grad(const GroupNormParams& p, int type, cudaStream_t stream) { return launch_any<true>(p, type, stream); }

}  // namespace kda
