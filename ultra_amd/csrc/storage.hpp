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

static inline bool known_dtype(int d) { return d == ULTR_DTYPE_F32 || d == ULTR_DTYPE_BF16 || d == ULTR_DTYPE_F16; }
static inline int dtype_bytes(int d) { return d == ULTR_DTYPE_F32 ? 4 : 2; }

}  // namespace ultr
