// What the training-side kernels (embed.hip, block_norm.hip, grad_clip.hip) share.
#pragma once
#include "common.hpp"

// 16 bytes of T: the unit of every wide load and store
template <typename T> struct alignas(16) word16 {
    static constexpr int N = (int)(16 / sizeof(T));
    T v[16 / sizeof(T)];
};

// The same at any address of a 16-bit element: global memory takes unaligned vector accesses, so that rows of odd length and views into a
// buffer are loaded and stored as wide as others.
typedef u32x4 u32x4_any __attribute__((aligned(2), may_alias));

// A row of C elements as words of W = 16 / sizeof(T) where C is no multiple of W (but at least W), and at any address.  The word at
// element c is loaded as it stands; the last one, of which the row has less, where it is whole, and shifted when it is needed: zeros
// behind the row's end.
template <typename T> __device__ __forceinline__ int row_word_start(int c, int C) { return c + word16<T>::N <= C ? c : C - word16<T>::N; }
template <typename T> __device__ __forceinline__ u32x4 row_word_load(const T* p, int c, int C) { return *(const u32x4_any*)(p + row_word_start<T>(c, C)); }
template <typename T> __device__ __forceinline__ u32x4 row_word_shift(u32x4 w, int c, int C) {
    return __builtin_bit_cast(u32x4, __builtin_bit_cast(unsigned __int128, w) >> ((c - row_word_start<T>(c, C)) * 8 * (int)sizeof(T)));
}

// A launch has fewer than 2^32 threads along an axis: more are cut off without an error (67 million rows of 8 channels, a wave each, are as
// many).  Launches whose number of workgroups grows with the call lie in two axes from 2^20 on; workgroups behind the last one end at once.
static inline dim3 grid_of(long long workgroups) {
    return dim3((unsigned)(workgroups < (1 << 20) ? workgroups : 1 << 20), (unsigned)((workgroups + (1 << 20) - 1) >> 20));
}
__device__ __forceinline__ long long workgroup() { return ((long long)blockIdx.y << 20) + blockIdx.x; }

// The one rounding of a result to its storage type.  f16: the binary32 value is kept out of the compiler's sight, which otherwise folds
// the last multiplication and the conversion of SINGLE elements into v_fma_mixlo_f16 (rounding once from the exact product) but not
// those of pairs: a result's bits would depend on whether its tensor is aligned.
template <typename T> __device__ __forceinline__ T to_storage(float x) {
    if constexpr (sizeof(T) == 2) asm("" : "+v"(x));
    return (T)x;
}

// Whether a call's stores go past the memory-side cache: when what the call reads and writes does not fit in its 256 MB, its outputs cannot
// stay there for whoever reads them next, and storing them as usual pushes out what the call (or the next one) still reads.  Smaller
// calls store as usual.  Measured: 1024 prompts' embedding (202 MB behind a table of 126 MB) 72 -> 47 us, clipping 1.4 GB 789 -> 735 us;
// against it 152 MB of zero rows (inside the cache) 22 -> 28 us.
static inline bool streams_past_cache(double bytes) { return bytes > 256.0 * 1024 * 1024; }

template <typename T, typename WORD = u32x4> __device__ __forceinline__ void store16(T* p, const word16<T>& w, bool stream) {
    const u32x4 bits = __builtin_bit_cast(u32x4, w);
    if (stream) {                   // (the empty statements keep the compiler from merging the two stores into one ordinary one)
        asm volatile("" ::: "memory");
        __builtin_nontemporal_store(bits, (WORD*)p);
        asm volatile("" ::: "memory");
    } else {
        *(WORD*)p = bits;
    }
}
// the word at p[c] of a row of C elements: what lies behind the row's end is not written
template <typename T> __device__ __forceinline__ void store_row_word(T* p, int c, int C, const word16<T>& w, bool stream) {
    if (c + word16<T>::N <= C) {
        store16<T, u32x4_any>(p + c, w, stream);
    } else {
#pragma unroll
        for (int j = 0; j < word16<T>::N; ++j)
            if (c + j < C) p[c + j] = w.v[j];
    }
}

// Sum over the wave's 64 lanes on the VALU's cross-lane paths (DPP), the same in every lane: four steps inside rows of 16 lanes, two
// broadcasts across them.  (A shuffle goes through LDS: six of them are ten times the latency, and a row's norm is a chain of sums.)
template <int CTRL, int ROWS> __device__ __forceinline__ float dpp_of(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, ROWS, 0xf, false));
}
__device__ __forceinline__ float wave_total(float v) {
    v += dpp_of<0xB1, 0xf>(v);      // quad_perm [1, 0, 3, 2]
    v += dpp_of<0x4E, 0xf>(v);      // quad_perm [2, 3, 0, 1]
    v += dpp_of<0x141, 0xf>(v);     // row_half_mirror
    v += dpp_of<0x140, 0xf>(v);     // row_mirror
    v += dpp_of<0x142, 0xa>(v);     // row_bcast15 into rows 1 and 3 (others add 0)
    v += dpp_of<0x143, 0xc>(v);     // row_bcast31 into rows 2 and 3
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}

// p[first * pitch] + p[(first + step) * pitch] + ... up to (not with) index `end`, in that order, eight loads at a time.  The indices of the
// last round that lie behind the end read the first one again: a loop for the rest would wait for each of its loads.
__device__ __forceinline__ float sum_strided(const float* __restrict__ p, long long pitch, int first, int end, int step) {
    float s = 0.f;
    for (int k = first; k < end; k += 8 * step) {
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = p[(long long)(k + j * step < end ? k + j * step : first) * pitch];
#pragma unroll
        for (int j = 0; j < 8; ++j) s += k + j * step < end ? v[j] : 0.f;
    }
    return s;
}
