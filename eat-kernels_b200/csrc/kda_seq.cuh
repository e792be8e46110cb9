// What the operators around the KDA prefill share on the device: the caller's sequence and slot tables, read where they lie
// and checked by whoever uses them, and the token types.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace kda {

constexpr int SEQ_BAD_CU = 1, SEQ_BAD_SLOT = 2, SEQ_POOL_FULL = 32;      // KDA_STATUS_* of these operators

// Sequences of a packed batch and the slots of their states.  Without `cu` there is one sequence [0, T) (a step: T sequences
// of one token); without `slots` sequence i uses slot i.
struct SeqTable {
  const void* cu;
  const void* slots;
  int* status;
  long long T, n_slots;
  int cu_is64, slots_is64, N;
};

__device__ __forceinline__ long long table_at(const void* p, int is64, long long i) {
  return is64 ? reinterpret_cast<const long long*>(p)[i] : (long long)reinterpret_cast<const int*>(p)[i];
}

__device__ __forceinline__ long long cu_at(const SeqTable& s, long long i) {
  return s.cu != nullptr ? table_at(s.cu, s.cu_is64, i) : (i == 0 ? 0 : s.T);
}

__device__ __forceinline__ void report(int* status, int bits) {
  if (status != nullptr) atomicOr(status, bits);
}

// Called by the whole block: is cu_seqlens not 0-based, decreasing or beyond T?  Every block looks for itself (N + 1 entries
// out of L2, one pass of a block up to its number of threads) instead of waiting for a planner launch in front.
__device__ __forceinline__ bool cu_rejected(const SeqTable& s) {
  if (s.cu == nullptr) return false;
  int bad = 0;
  for (int i = threadIdx.x; i <= s.N; i += blockDim.x) {
    const long long c0 = cu_at(s, i), c1 = i < s.N ? cu_at(s, i + 1) : c0;
    if (c0 < 0 || c0 > s.T || c1 < c0 || (i == 0 && c0 != 0)) bad = 1;
  }
  const bool rejected = __syncthreads_or(bad) != 0;
  if (rejected && threadIdx.x == 0) report(s.status, SEQ_BAD_CU);
  return rejected;
}

// The same, and how many entries lie below t (of a layout that is not rejected: the first sequence that starts at t or behind).
__device__ __forceinline__ bool cu_rejected(const SeqTable& s, long long t, int& below) {
  int bad = 0;
  below = 0;
  for (int i0 = 0; i0 <= s.N; i0 += blockDim.x) {
    const int i = i0 + threadIdx.x;
    long long c0 = t;
    if (i <= s.N) {
      c0 = cu_at(s, i);
      const long long c1 = i < s.N ? cu_at(s, i + 1) : c0;
      if (c0 < 0 || c0 > s.T || c1 < c0 || (i == 0 && c0 != 0)) bad = 1;
    }
    below += __syncthreads_count(c0 < t);
  }
  const bool rejected = __syncthreads_or(bad) != 0;
  if (rejected && threadIdx.x == 0) report(s.status, SEQ_BAD_CU);
  return rejected;
}

// Called by the whole block: the slot of sequence i, or -1 where its entry is out of range or repeats an earlier one (the
// first claim keeps the slot, as in the prefill's planner).
__device__ __forceinline__ long long claim_slot(const SeqTable& s, int i) {
  if (s.slots == nullptr) return i;
  const long long d = table_at(s.slots, s.slots_is64, i);
  int bad = d < 0 || d >= s.n_slots;
  for (int j = threadIdx.x; j < i && !bad; j += blockDim.x)
    if (table_at(s.slots, s.slots_is64, j) == d) bad = 1;
  if (__syncthreads_or(bad) == 0) return d;
  if (threadIdx.x == 0) report(s.status, SEQ_BAD_SLOT);
  return -1;
}

// An entry of a slot table of a step: itself, -1 out of range, -2 padding.  Slots fit 31 bits.
__device__ __forceinline__ int slot_entry(const SeqTable& s, int i) {
  if (s.slots_is64) {
    const long long d = reinterpret_cast<const long long*>(s.slots)[i];
    return d < 0 ? -2 : (d < s.n_slots ? (int)d : -1);
  }
  const int d = reinterpret_cast<const int*>(s.slots)[i];
  return d < 0 ? -2 : (d < (int)s.n_slots ? d : -1);
}

// The slots of R rows of a step from row0 on, `rows` of them there are (others: -2), in two parts, so that a block can ask for the
// states before it has looked for repeats.  First the entries.
template <int R>
__device__ __forceinline__ void row_slots(const SeqTable& s, int row0, int rows, int (&slot)[R]) {
#pragma unroll
  for (int r = 0; r < R; r++) {
    slot[r] = -2;
    if (r < rows) slot[r] = s.slots != nullptr ? slot_entry(s, row0 + r) : row0 + r;
  }
}

// Then, called by the whole block: -1 for a slot that an earlier row has claimed too.  Says whether any row is at -1 now.
template <int R>
__device__ __forceinline__ bool drop_repeats(const SeqTable& s, int row0, int (&slot)[R]) {
  if (s.slots == nullptr) return false;
  int bad = 0;
  for (int j = threadIdx.x; j < row0; j += blockDim.x) {
    const int d = slot_entry(s, j);
#pragma unroll
    for (int r = 0; r < R; r++)
      if (d >= 0 && d == slot[r]) bad |= 1 << r;
  }
#pragma unroll
  for (int r = 0; r < R; r++) {
    if (slot[r] == -1) bad |= 1 << r;
#pragma unroll
    for (int q = 0; q < r; q++)
      if (slot[r] >= 0 && slot[r] == slot[q]) bad |= 1 << r;
  }
  if (__syncthreads_or(bad) == 0) return false;
#pragma unroll
  for (int r = 0; r < R; r++)
    if (__syncthreads_or(bad >> r & 1)) slot[r] = -1;
  if (threadIdx.x == 0) report(s.status, SEQ_BAD_SLOT);
  return true;
}

// ---- token types
__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
template <typename T> __device__ __forceinline__ T from_float(float x);
template <> __device__ __forceinline__ float from_float<float>(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }

// VEC consecutive values of a row: one access of VEC * sizeof(T) bytes, aligned to that.
template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Pack {
  T v[VEC];
};
template <typename T, int VEC>
__device__ __forceinline__ void unpack(const Pack<T, VEC>& p, float (&f)[VEC]) {
#pragma unroll
  for (int i = 0; i < VEC; i++) f[i] = to_float(p.v[i]);
}
template <typename T, int VEC>
__device__ __forceinline__ Pack<T, VEC> pack(const float (&f)[VEC]) {
  Pack<T, VEC> p;
#pragma unroll
  for (int i = 0; i < VEC; i++) p.v[i] = from_float<T>(f[i]);
  return p;
}

// x / (1 + e^-x): the approximate exponential and reciprocal are off by some 2^-21, which 16-bit outputs do not show; 32-bit
// ones take the exact functions.
template <typename T>
__device__ __forceinline__ float silu(float x) {
  if constexpr (sizeof(T) == 4) return x / (1.0f + expf(-x));
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(x * -1.4426950408889634f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
  return x * r;
}

}  // namespace kda
