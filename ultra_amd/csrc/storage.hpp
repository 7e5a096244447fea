// Storage types of the stand-alone operators (norm.hip, tensors.hip): fp32, bf16 and fp16 in memory, fp32 in registers.
#pragma once
#include "common.hpp"

namespace ultr {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

// One rounding per stored value, to nearest even, NaN kept: the compiler's conversions do both.
template <typename T>
__device__ __forceinline__ float to_f32(T v) { return (float)v; }
template <typename T>
__device__ __forceinline__ T from_f32(float v) { return (T)v; }

// A 16-byte (or shorter) piece of a row.  Its address is only as aligned as an element: gfx950 loads and stores
// dwords at any byte address, so rows of odd width or stride take the same wide accesses as aligned ones.
template <typename T, int V>
struct Piece {
  typedef T type __attribute__((ext_vector_type(V), aligned(sizeof(T))));
};
// NT: past the caches, for data that nothing reads again before it would be gone from them anyway.
template <int V, bool NT = false, typename T>
__device__ __forceinline__ void load_piece(const T* p, float (&v)[V]) {
  typedef const typename Piece<T, V>::type P;
  const auto q = NT ? __builtin_nontemporal_load(reinterpret_cast<P*>(p)) : *reinterpret_cast<P*>(p);
#pragma unroll
  for (int j = 0; j < V; ++j) v[j] = to_f32(q[j]);
}
template <int V, bool NT = false, typename T>
__device__ __forceinline__ void store_piece(T* p, const float (&v)[V]) {
  typedef typename Piece<T, V>::type P;
  P q;
#pragma unroll
  for (int j = 0; j < V; ++j) q[j] = from_f32<T>(v[j]);
  if (NT) __builtin_nontemporal_store(q, reinterpret_cast<P*>(p));
  else *reinterpret_cast<P*>(p) = q;
}

static inline bool known_dtype(int d) { return d == ULTR_DTYPE_F32 || d == ULTR_DTYPE_BF16 || d == ULTR_DTYPE_F16; }
static inline int dtype_bytes(int d) { return d == ULTR_DTYPE_F32 ? 4 : 2; }

}  // namespace ultr
