// Upkeep of the slots that several pools share: copies, forks, frees, compaction.  A one-block kernel works out on the device
// what is to be copied (nothing is read on the host, so a captured call follows its tables), a second one copies.
#include "kda_serving.cuh"

namespace kda {

namespace {

constexpr int PLAN_THREADS = 1024;
constexpr int COPY_THREADS = 256;
constexpr int COPY_CHUNK = 16384;        // bytes of one row that a block moves at a time

// Sum of x over the threads in front of this one; `total`: over all.
__device__ __forceinline__ int scan_block(int x, int& total) {
  __shared__ int s_warp[PLAN_THREADS / 32];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  int incl = x;
#pragma unroll
  for (int m = 1; m < 32; m *= 2) {
    const int up = __shfl_up_sync(0xffffffffu, incl, m);
    if (lane >= m) incl += up;
  }
  __syncthreads();
  if (lane == 31) s_warp[warp] = incl;
  __syncthreads();
  int w = s_warp[lane];
#pragma unroll
  for (int m = 1; m < 32; m *= 2) {
    const int up = __shfl_up_sync(0xffffffffu, w, m);
    if (lane >= m) w += up;
  }
  total = __shfl_sync(0xffffffffu, w, 31);
  const int before = __shfl_sync(0xffffffffu, w, (warp + 31) % 32);
  return incl - x + (warp > 0 ? before : 0);
}

// The run of slots that thread i looks after: [first, last).
__device__ __forceinline__ void share_of(long long n, long long& first, long long& last) {
  const long long each = (n + PLAN_THREADS - 1) / PLAN_THREADS;
  first = min(n, each * threadIdx.x);
  last = min(n, first + each);
}

// dst[i] <- src[i].  A destination that an earlier entry names, or that some entry reads, would make the result depend on the
// order: such entries are left out, as are those out of range.  A negative destination is padding, a negative source zeros.
// Each slot that is named has the first entry that writes it, and whether one reads it, in two tables behind the moves.
__global__ void __launch_bounds__(PLAN_THREADS, 1) kda_pool_copy_plan_kernel(const PoolPlan p) {
  __shared__ int s_count;
  int *first = p.moves + 4 + 2 * p.n, *read = first + p.P;
  if (threadIdx.x == 0) s_count = 0;
  // an entry of a table: -1 negative, P out of range
  auto entry = [&](const void* table, int is64, long long i) {
    const long long d = table_at(table, is64, i);
    return d < 0 ? -1 : (int)min(d, p.P);
  };
  for (long long i = threadIdx.x; i < p.n; i += PLAN_THREADS) {
    const int d = entry(p.dst, p.dst_is64, i);
    if (d >= 0 && d < p.P) {
      first[d] = 0x7fffffff;
      read[d] = 0;
    }
  }
  __syncthreads();
  for (long long i = threadIdx.x; i < p.n; i += PLAN_THREADS) {
    const int d = entry(p.dst, p.dst_is64, i), s = entry(p.src, p.src_is64, i);
    if (d < 0) continue;
    if (d < p.P) atomicMin(&first[d], (int)i);
    if (s >= 0 && s < p.P) read[s] = 1;
  }
  __syncthreads();
  for (long long i = threadIdx.x; i < p.n; i += PLAN_THREADS) {
    const int d = entry(p.dst, p.dst_is64, i), s = entry(p.src, p.src_is64, i);
    if (d < 0 || (d == s && d < p.P)) continue;      // padding; a row onto itself
    if (d >= p.P || s >= p.P || first[d] != (int)i || read[d] != 0) {
      report(p.status, SEQ_BAD_SLOT);
      continue;
    }
    const int at = atomicAdd(&s_count, 1);
    p.moves[4 + 2 * at] = s;
    p.moves[5 + 2 * at] = d;
  }
  __syncthreads();
  if (threadIdx.x == 0) p.moves[0] = s_count;
}

// Entry i with a parent in use (or none) takes the lowest slot that is free and that no earlier entry took.
__global__ void __launch_bounds__(PLAN_THREADS, 1) kda_pool_fork_plan_kernel(const PoolPlan p) {
  int* free_slots = p.moves + 4 + 2 * p.n;           // room for n behind the pairs
  long long first, last;
  share_of(p.P, first, last);
  int mine = 0, n_free;
  for (long long i = first; i < last; i++) mine += p.used[i] == 0;
  int rank = scan_block(mine, n_free);
  for (long long i = first; i < last && rank < p.n; i++)
    if (p.used[i] == 0) free_slots[rank++] = (int)i;
  __syncthreads();
  int base = 0;                                      // entries with a good parent so far
  for (long long i0 = 0; i0 < p.n; i0 += PLAN_THREADS) {
    const long long i = i0 + threadIdx.x;
    long long parent = -1;
    bool good = false;
    if (i < p.n) {
      parent = table_at(p.src, p.src_is64, i);
      // a slot that this call hands out is among the free ones, whose marks change only below, behind the last look
      good = parent < 0 || (parent < p.P && p.used[parent] != 0);
      if (!good) report(p.status, SEQ_BAD_SLOT);
    }
    int total;
    const int at = base + scan_block(good, total);
    int slot = -1;
    if (good && at < n_free) {
      slot = free_slots[at];
      p.moves[4 + 2 * at] = parent < 0 ? -1 : (int)parent;
      p.moves[5 + 2 * at] = slot;
    } else if (good) {
      report(p.status, SEQ_POOL_FULL);
    }
    if (i < p.n) p.slots_out[i] = slot;
    base += total;
  }
  const int taken = min(base, n_free);
  __syncthreads();
  for (int i = threadIdx.x; i < taken; i += PLAN_THREADS) p.used[free_slots[i]] = 1;
  if (threadIdx.x == 0) p.moves[0] = taken;
}

__global__ void __launch_bounds__(PLAN_THREADS, 1) kda_pool_free_kernel(const PoolPlan p) {
  for (long long i0 = 0; i0 < p.n; i0 += PLAN_THREADS) {
    const long long i = i0 + threadIdx.x;
    long long slot = i < p.n ? table_at(p.src, p.src_is64, i) : -1;
    if (slot >= 0) {
      bool ok = slot < p.P && p.used[slot] != 0;     // entries of earlier passes have cleared theirs
      for (long long j = i0; j < i && ok; j++) ok = table_at(p.src, p.src_is64, j) != slot;
      if (!ok) { report(p.status, SEQ_BAD_SLOT); slot = -1; }
    }
    __syncthreads();
    if (slot >= 0) p.used[slot] = 0;
    __syncthreads();
  }
}

// With n slots in use, the k-th one behind the first n moves into the k-th hole among them.
__global__ void __launch_bounds__(PLAN_THREADS, 1) kda_pool_compact_plan_kernel(const PoolPlan p) {
  long long first, last;
  share_of(p.P, first, last);
  int mine = 0, live, holes, movers;
  for (long long i = first; i < last; i++) mine += p.used[i] != 0;
  scan_block(mine, live);
  int h = 0, m = 0;
  for (long long i = first; i < last; i++) {
    h += i < live && p.used[i] == 0;
    m += i >= live && p.used[i] != 0;
  }
  h = scan_block(h, holes);
  m = scan_block(m, movers);
  for (long long i = first; i < last; i++)
    if (i < live && p.used[i] == 0) p.moves[5 + 2 * h++] = (int)i;
  __syncthreads();
  for (long long i = first; i < last; i++) {
    const bool on = p.used[i] != 0;
    int to = on ? (int)i : -1;
    if (on && i >= live) {
      to = p.moves[5 + 2 * m];
      p.moves[4 + 2 * m++] = (int)i;
    }
    p.remap[i] = to;
    p.used[i] = i < live;
  }
  if (threadIdx.x == 0) p.moves[0] = movers;
  __syncthreads();
  for (int t = 0; t < p.n_tables; t++)
    for (long long i = threadIdx.x; i < p.table_n[t]; i += PLAN_THREADS) {
      const long long old = table_at(p.tables[t], p.table_is64[t], i);
      if (old < 0) continue;
      const int to = old < p.P ? p.remap[old] : -1;
      if (to < 0) report(p.status, SEQ_BAD_SLOT);
      if (p.table_is64[t]) reinterpret_cast<long long*>(p.tables[t])[i] = to;
      else reinterpret_cast<int*>(p.tables[t])[i] = to;
    }
}

template <typename U>
__device__ __forceinline__ void copy_chunk(unsigned char* dst, const unsigned char* src, int bytes) {
  constexpr int EACH = 4;
  const int n = bytes / (int)sizeof(U);
  for (int i0 = threadIdx.x; i0 < n; i0 += EACH * COPY_THREADS) {
    U v[EACH];
#pragma unroll
    for (int e = 0; e < EACH; e++) {
      const int i = i0 + e * COPY_THREADS;
      v[e] = U();
      if (src != nullptr && i < n) v[e] = reinterpret_cast<const U*>(src)[i];
    }
#pragma unroll
    for (int e = 0; e < EACH; e++) {
      const int i = i0 + e * COPY_THREADS;
      if (i < n) reinterpret_cast<U*>(dst)[i] = v[e];
    }
  }
}

// Bound by memory.  The number of moves is known on the device only: the grid covers the card and takes chunk after chunk.  64 rows
// of 1.04 MB: 18 us behind 5 us of plan.
__global__ void __launch_bounds__(COPY_THREADS) kda_pool_copy_kernel(const PoolRows r, const int* __restrict__ moves) {
  int chunks = 0;
  for (int k = 0; k < r.n; k++) chunks += (int)((r.bytes[k] + COPY_CHUNK - 1) / COPY_CHUNK);
  const long long items = (long long)moves[0] * chunks;
  for (long long item = blockIdx.x; item < items; item += gridDim.x) {
    const int move = (int)(item / chunks);
    int chunk = (int)(item % chunks), k = 0;
    for (;; k++) {
      const int n = (int)((r.bytes[k] + COPY_CHUNK - 1) / COPY_CHUNK);
      if (chunk < n) break;
      chunk -= n;
    }
    const int from = moves[4 + 2 * move], to = moves[5 + 2 * move];
    const long long at = (long long)chunk * COPY_CHUNK;
    const int bytes = (int)min((long long)COPY_CHUNK, r.bytes[k] - at);
    unsigned char* dst = r.base[k] + to * r.stride[k] + at;
    const unsigned char* src = from < 0 ? nullptr : r.base[k] + from * r.stride[k] + at;
    // the widest access that base, stride and length allow (chunks start at multiples of 16 KB)
    const uintptr_t unit = reinterpret_cast<uintptr_t>(r.base[k]) | (uintptr_t)r.stride[k] | (uintptr_t)r.bytes[k];
    if ((unit & 15) == 0) copy_chunk<uint4>(dst, src, bytes);
    else if ((unit & 3) == 0) copy_chunk<unsigned int>(dst, src, bytes);
    else if ((unit & 1) == 0) copy_chunk<unsigned short>(dst, src, bytes);
    else copy_chunk<unsigned char>(dst, src, bytes);
  }
}

cudaError_t launch_copy(const PoolPlan& p, const PoolRows& rows, long long most, cudaStream_t stream) {
  long long chunks = 0;
  for (int k = 0; k < rows.n; k++) chunks += (rows.bytes[k] + COPY_CHUNK - 1) / COPY_CHUNK;
  const long long blocks = most * chunks < 148 * 8 ? most * chunks : 148 * 8;
  if (blocks == 0) return cudaSuccess;
  kda_pool_copy_kernel<<<(unsigned)blocks, COPY_THREADS, 0, stream>>>(rows, p.moves);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_pool_copy(const PoolPlan& p, const PoolRows& rows, cudaStream_t stream) {
  kda_pool_copy_plan_kernel<<<1, PLAN_THREADS, 0, stream>>>(p);
  const cudaError_t e = cudaGetLastError();
  return e != cudaSuccess ? e : launch_copy(p, rows, p.n, stream);
}

cudaError_t launch_pool_fork(const PoolPlan& p, const PoolRows& rows, cudaStream_t stream) {
  kda_pool_fork_plan_kernel<<<1, PLAN_THREADS, 0, stream>>>(p);
  const cudaError_t e = cudaGetLastError();
  return e != cudaSuccess ? e : launch_copy(p, rows, p.n < p.P ? p.n : p.P, stream);
}

cudaError_t launch_pool_free(const PoolPlan& p, cudaStream_t stream) {
  kda_pool_free_kernel<<<1, PLAN_THREADS, 0, stream>>>(p);
  return cudaGetLastError();
}

cudaError_t launch_pool_compact(const PoolPlan& p, const PoolRows& rows, cudaStream_t stream) {
  kda_pool_compact_plan_kernel<<<1, PLAN_THREADS, 0, stream>>>(p);
  const cudaError_t e = cudaGetLastError();
  return e != cudaSuccess ? e : launch_copy(p, rows, p.P / 2, stream);
}

}  // namespace kda
