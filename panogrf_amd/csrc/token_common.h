// Shared by the token operators (block_norm.hip, rotary.hip, diff_attn*.hip): element types, vector loads, wave reductions.
#pragma once
#include <hip/hip_runtime.h>

#include <type_traits>

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

// Sum over aligned groups of W lanes, every lane gets it: neighbours, quads, mirrored eights and sixteens by lane permutes of the add itself, then rows of 16 and
// halves by swaps (no LDS; the order is the same in every lane)
template <int W>
__device__ __forceinline__ float group_sum(float v) {
  auto moved = [](float x, auto ctrl) { return __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), decltype(ctrl)::value, 0xf, 0xf, true)); };
  if constexpr (W >= 2) v += moved(v, std::integral_constant<int, 0xB1>{});
  if constexpr (W >= 4) v += moved(v, std::integral_constant<int, 0x4E>{});
  if constexpr (W >= 8) v += moved(v, std::integral_constant<int, 0x141>{});
  if constexpr (W >= 16) v += moved(v, std::integral_constant<int, 0x140>{});
  if constexpr (W >= 32) {
    const auto x = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(x[0]) + __uint_as_float(x[1]);
  }
  if constexpr (W >= 64) {
    const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(x[0]) + __uint_as_float(x[1]);
  }
  return v;
}

#define PGRF_TOK_LAUNCHED(name)                                                                               \
  do {                                                                                                        \
    hipError_t e_ = hipGetLastError();                                                                        \
    if (e_ != hipSuccess) return set_error(PGRF_ERR_LAUNCH, "%s: %s", name, hipGetErrorString(e_));           \
  } while (0)

}  // namespace tok
}  // namespace pgrf
