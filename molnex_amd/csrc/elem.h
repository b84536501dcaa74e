// Element types of the training kernels: float32, bfloat16 and float16 in memory, float32 in registers.
#pragma once

#include "common.h"

namespace mnx {

enum : int { kF32 = MNX_F32, kBF16 = MNX_BF16, kF16 = MNX_F16 };

inline bool elem_valid(int dtype) { return dtype == kF32 || dtype == kBF16 || dtype == kF16; }
inline int elem_bytes(int dtype) { return dtype == kF32 ? 4 : 2; }

template <int DT>
struct Elem;
template <>
struct Elem<kF32> {
    using T = float;
};
template <>
struct Elem<kBF16> {
    using T = __bf16;
};
template <>
struct Elem<kF16> {
    using T = _Float16;
};

// One value of a vector whose type is known at run time (weights: read once per wavefront, not per row).
__device__ __forceinline__ float load_elem(const void* p, int64_t i, int dtype) {
    if (dtype == kF32) return static_cast<const float*>(p)[i];
    if (dtype == kBF16) return static_cast<float>(static_cast<const __bf16*>(p)[i]);
    return static_cast<float>(static_cast<const _Float16*>(p)[i]);
}
// Rounded to nearest, ties to even.
__device__ __forceinline__ void store_elem(void* p, int64_t i, int dtype, float v) {
    if (dtype == kF32) static_cast<float*>(p)[i] = v;
    else if (dtype == kBF16) static_cast<__bf16*>(p)[i] = static_cast<__bf16>(v);
    else static_cast<_Float16*>(p)[i] = static_cast<_Float16>(v);
}

}  // namespace mnx
