// What the training-side kernels (embed.hip, block_norm.hip, grad_clip.hip) share.
#pragma once
#include "common.hpp"

// 16 bytes of T: the unit of every wide load and store
template <typename T> struct alignas(16) word16 {
    static constexpr int N = (int)(16 / sizeof(T));
    T v[16 / sizeof(T)];
};

// The one rounding of a result to its storage type.  f16: the binary32 value is kept out of the compiler's sight, which otherwise folds
// the last multiplication and the conversion of SINGLE elements into v_fma_mixlo_f16 (rounding once from the exact product) but not
// those of pairs: a result's bits would depend on whether its tensor is aligned.
template <typename T> __device__ __forceinline__ T to_storage(float x) {
    if constexpr (sizeof(T) == 2) asm("" : "+v"(x));
    return (T)x;
}
