// 16-byte chunks of rows, for the memory-bound kernels. RAGGED rows have any length (at least a chunk) and
// alignment (of the element) and go through the unaligned 128-bit accesses that the hardware takes. The last
// chunk of a ragged row ends at the row's end: it shares columns with the chunk before it, and both
// chunks' threads compute and store the same values there. Ragged rows share cache lines between
// waves and rows, so they are loaded and stored normally where aligned ones stream.
#pragma once

#include "krsi_device.h"

namespace krsi {

typedef u32x4 u32x4_any __attribute__((aligned(2)));
typedef f32x4 f32x4_any __attribute__((aligned(4)));

// Read once: non-temporal where aligned.
template <bool RAGGED, typename T>
__device__ __forceinline__ u32x4 stream_chunk(const T* p) {
  if constexpr (RAGGED) return *reinterpret_cast<const u32x4_any*>(p);
  return __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p));
}
template <bool RAGGED, typename T>
__device__ __forceinline__ u32x4 load_chunk(const T* p) {
  if constexpr (RAGGED) return *reinterpret_cast<const u32x4_any*>(p);
  return *reinterpret_cast<const u32x4*>(p);
}
template <bool RAGGED, typename T>
__device__ __forceinline__ void store_chunk(T* p, const u32x4& v) {
  if constexpr (RAGGED)
    *reinterpret_cast<u32x4_any*>(p) = v;
  else
    __builtin_nontemporal_store(v, reinterpret_cast<u32x4*>(p));
}

// First column of chunk c (of E elements) of a row of n, and how many of its leading columns the chunk before it has.
template <bool RAGGED, int E>
__device__ __forceinline__ int chunk_col(int c, int n) {
  return RAGGED ? min(c * E, n - E) : c * E;
}
template <bool RAGGED, int E>
__device__ __forceinline__ int chunk_shared(int c, int n) {
  return RAGGED ? max(c * E - (n - E), 0) : 0;
}
// The chunk's address. Aligned rows index whole chunks: added to the row's offset as a count of elements, each
// chunk held one more address register (RMSNorm backward, fp32 rows of 8192: one wave per SIMD instead of two).
template <bool RAGGED, int E, typename T>
__device__ __forceinline__ const T* chunk_at(const T* row, int c, int n) {
  if constexpr (RAGGED) return row + chunk_col<true, E>(c, n);
  return reinterpret_cast<const T*>(reinterpret_cast<const u32x4*>(row) + c);
}
template <bool RAGGED, int E, typename T>
__device__ __forceinline__ T* chunk_at(T* row, int c, int n) {
  if constexpr (RAGGED) return row + chunk_col<true, E>(c, n);
  return reinterpret_cast<T*>(reinterpret_cast<u32x4*>(row) + c);
}

// C consecutive elements of any alignment, in registers.
template <int DT, int C>
struct Piece {
  using T = typename Elem<DT>::T;
  T e[C];
  __device__ __forceinline__ void load(const T* p) { __builtin_memcpy(e, p, sizeof(e)); }
  __device__ __forceinline__ void store(T* p) const { __builtin_memcpy(p, e, sizeof(e)); }
  // Written once, not read back: non-temporal where it is a whole 16-byte chunk.
  __device__ __forceinline__ void store_stream(T* p) const {
    if constexpr (sizeof(e) == 16)
      __builtin_nontemporal_store(__builtin_bit_cast(u32x4, *this), reinterpret_cast<u32x4_any*>(p));
    else
      store(p);
  }
  __device__ __forceinline__ void get(float* f) const {
#pragma unroll
    for (int j = 0; j < C; ++j) f[j] = Elem<DT>::load(e[j]);
  }
  __device__ __forceinline__ void set(const float* f) {
#pragma unroll
    for (int j = 0; j < C; ++j) e[j] = Elem<DT>::store(f[j]);
  }
};

// Entry i of an index tensor of int32 or int64 (bytes 4 or 8).
__device__ __forceinline__ int64_t load_index(const void* p, int bytes, int64_t i) {
  return bytes == 8 ? static_cast<const int64_t*>(p)[i] : static_cast<const int32_t*>(p)[i];
}

}  // namespace krsi
