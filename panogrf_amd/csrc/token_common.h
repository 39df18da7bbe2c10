// Shared by the token operators (block_norm.hip, rotary.hip, diff_attn*.hip): element types, vector loads, wave reductions.
#pragma once
#include <hip/hip_runtime.h>

#include "pgrf_internal.h"

namespace pgrf {
namespace tok {

using bf16 = __bf16;
using f16 = _Float16;

// V elements of T moved by one instruction (V * sizeof(T) in {2, 4, 8, 16} bytes)
template <typename T, int V>
struct alignas(V * sizeof(T)) Vec {
  T e[V];
};

template <typename T, int V>
__device__ __forceinline__ Vec<T, V> load_vec(const T* p) {
  return *reinterpret_cast<const Vec<T, V>*>(p);
}
template <typename T, int V>
__device__ __forceinline__ void store_vec(T* p, const Vec<T, V>& v) {
  *reinterpret_cast<Vec<T, V>*>(p) = v;
}

inline size_t dtype_bytes(int dtype) { return dtype == PGRF_DTYPE_F32 ? 4 : 2; }
inline bool dtype_ok(int dtype) { return dtype >= PGRF_DTYPE_F32 && dtype <= PGRF_DTYPE_F16; }
inline bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

template <int W>
__device__ __forceinline__ float group_sum(float v) {   // sum over aligned groups of W lanes, every lane gets it
#pragma unroll
  for (int o = 1; o < W; o <<= 1) v += __shfl_xor(v, o, 64);
  return v;
}

#define PGRF_TOK_LAUNCHED(name)                                                                               \
  do {                                                                                                        \
    hipError_t e_ = hipGetLastError();                                                                        \
    if (e_ != hipSuccess) return set_error(PGRF_ERR_LAUNCH, "%s: %s", name, hipGetErrorString(e_));           \
  } while (0)

}  // namespace tok
}  // namespace pgrf
