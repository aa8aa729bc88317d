// Global gradient norm over many tensors, and clipping to it.
//
//   norm = sqrt(sum over all tensors of g^2)   or   max |g|;      g <- g * min(1, max_norm / (norm + 1e-6))
//
// Bound by HBM: the norm reads every element once, clipping reads it again and writes it (the factor is known only after the last
// element).  The tensors' addresses travel in the kernel arguments (GC_TENSORS of them a launch), not through a table in device memory:
// gradients move between steps, and a captured launch then carries them itself.
//
// Every workgroup leaves ONE partial result in the workspace; the clipping launch's workgroups each add up the (at most GC_GRID)
// partials in the same fixed order, so there is no third launch and no float atomic: the same inputs give the same bits.
// Squares are summed in binary64: a binary32 square of a gradient below 1e-23 is zero and of one above 2e19 infinite, both inside the range
// of bf16 and f32 gradients, and the conversions stay below the time of the loads.
//
// Measured (MI355X; a large copy moves 4.9 TB/s): 340 M gradients in 290 tensors 364 us, 695 M bf16 in 388 tensors 738 us: two reads and a
// write at 5.6 TB/s.  The clipping goes backwards, so that it starts with what the norm has read last (the memory-side cache holds 256 MB).
#include "train_common.hpp"
#include <stdlib.h>

#define GC_TENSORS 128          /* per launch: 128 * 25 + 129 * 4 bytes of kernel arguments, below the 4 KB that every launch may carry */
#define GC_CHUNK 8192           /* elements of one tensor that a workgroup takes at a time */
#define GC_GRID 2048            /* 8 workgroups of 256 threads per CU: what is resident at once */

struct gc_table {
    const void* src[GC_TENSORS];
    void* dst[GC_TENSORS];
    long long n[GC_TENSORS];
    int start[GC_TENSORS + 1];  // first chunk of each tensor
    unsigned char dtype[GC_TENSORS];
    int count;
};

__device__ __forceinline__ double gc_wave_sum(double v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}
// a NaN operand has to come out (fmax drops it): a NaN gradient makes the norm NaN
__device__ __forceinline__ double gc_max(double a, double b) { return (a > b || a != a) ? a : b; }
__device__ __forceinline__ double gc_wave_max(double v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = gc_max(v, __shfl_xor(v, o, 64));
    return v;
}

template <bool INF> __device__ __forceinline__ double gc_combine(double a, double b) { return INF ? gc_max(a, b) : a + b; }
template <bool INF> __device__ __forceinline__ double gc_add(double acc, float x) {
    return INF ? gc_max(acc, (double)fabsf(x)) : __builtin_fma((double)x, (double)x, acc);
}

// the workgroup's result in every thread
template <bool INF>
__device__ double gc_block(double v, double* lds) {
    v = INF ? gc_wave_max(v) : gc_wave_sum(v);
    const int waves = blockDim.x >> 6;
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    v = lds[0];
    for (int w = 1; w < waves; ++w) v = gc_combine<INF>(v, lds[w]);
    __syncthreads();
    return v;
}

__device__ __forceinline__ int gc_find(const gc_table& t, int chunk) {
    int lo = 0, hi = t.count;                               // start[lo] <= chunk < start[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (t.start[mid] <= chunk) lo = mid; else hi = mid;
    }
    return lo;
}

// elements in front of the first 16-byte boundary of p (0 .. 7)
template <typename T> __device__ __forceinline__ int gc_head(const void* p) { return (int)((16 - ((uintptr_t)p & 15)) & 15) / (int)sizeof(T); }

// f(element index, 16 bytes) over whole 16-byte words of chunk `chunk` (CHUNK elements), g(element index) over the rest; `head` = elements in
// front of the first boundary of the tensor.  Chunk 0 of a tensor also takes the head.  BATCH words a thread are loaded at a time (behind
// the last: the thread's first one again, not handed on).
template <typename T, int CHUNK, int BATCH, typename F, typename G>
__device__ __forceinline__ void gc_range(const T* p, long long n, int chunk, int head, bool last_use, F&& f, G&& g) {
    constexpr int V = word16<T>::N;
    if (head > n) head = (int)n;
    const long long lo = head + (long long)chunk * CHUNK;
    const long long hi = lo + CHUNK < n ? lo + CHUNK : n;
    if (chunk == 0 && (int)threadIdx.x < head) g((long long)threadIdx.x);
    const int words = hi > lo ? (int)((hi - lo) / V) : 0;
    const u32x4* const w = (const u32x4*)(p + lo);
    for (int i = threadIdx.x; i < words; i += BATCH * blockDim.x) {
        u32x4 x[BATCH];
#pragma unroll
        for (int j = 0; j < BATCH; ++j) {
            const u32x4* at = w + (i + j * (int)blockDim.x < words ? i + j * (int)blockDim.x : i);
            x[j] = last_use ? __builtin_nontemporal_load(at) : *at;
        }
#pragma unroll
        for (int j = 0; j < BATCH; ++j)
            if (i + j * (int)blockDim.x < words) f(lo + (long long)(i + j * (int)blockDim.x) * V, __builtin_bit_cast(word16<T>, x[j]));
    }
    const long long tail = lo + (long long)words * V + threadIdx.x;
    if (tail < hi) g(tail);
}

template <typename T, int CHUNK, bool INF>
__device__ __forceinline__ double gc_norm_chunk(const void* src, long long n, int chunk, double acc) {
    const T* p = (const T*)src;
    gc_range<T, CHUNK, (int)sizeof(T) * 2>(p, n, chunk, gc_head<T>(src), false,
        [&](long long, word16<T> x) {
#pragma unroll
            for (int j = 0; j < word16<T>::N; ++j) acc = gc_add<INF>(acc, (float)x.v[j]);
        },
        [&](long long i) { acc = gc_add<INF>(acc, (float)p[i]); });
    return acc;
}

template <typename T, int CHUNK>
__device__ __forceinline__ void gc_scale_chunk(const void* src, void* dst, long long n, int chunk, float f, bool stream) {
    const T* p = (const T*)src;
    T* q = (T*)dst;
    gc_range<T, CHUNK, (int)sizeof(T) * 2>(p, n, chunk, gc_head<T>(src), true,
        [&](long long i, word16<T> x) {
#pragma unroll
            for (int j = 0; j < word16<T>::N; ++j) x.v[j] = to_storage<T>((float)x.v[j] * f);
            store16<T, u32x4_any>(q + i, x, stream);        // (the words are the source's; where the destination's
                                                            // boundaries lie elsewhere, 128 MB to 128 MB take 76 us, else 70)
        },
        [&](long long i) { q[i] = to_storage<T>((float)p[i] * f); });
}

template <int CHUNK, bool INF>
__device__ __forceinline__ double gc_norm_table(const gc_table& t, double acc) {
    for (int c = blockIdx.x; c < t.start[t.count]; c += gridDim.x) {
        const int k = gc_find(t, c), local = c - t.start[k];
        if (t.dtype[k] == GD_F32) acc = gc_norm_chunk<float, CHUNK, INF>(t.src[k], t.n[k], local, acc);
        else if (t.dtype[k] == GD_F16) acc = gc_norm_chunk<f16_t, CHUNK, INF>(t.src[k], t.n[k], local, acc);
        else acc = gc_norm_chunk<bf16_t, CHUNK, INF>(t.src[k], t.n[k], local, acc);
    }
    return acc;
}

template <int CHUNK>
__device__ __forceinline__ void gc_scale_table(const gc_table& t, float f, bool stream) {
    for (int c = t.start[t.count] - 1 - (int)blockIdx.x; c >= 0; c -= gridDim.x) {
        const int k = gc_find(t, c), local = c - t.start[k];
        if (f == 1.0f && t.dst[k] == t.src[k]) continue;    // g * 1 is g: nothing to write in place
        if (t.dtype[k] == GD_F32) gc_scale_chunk<float, CHUNK>(t.src[k], t.dst[k], t.n[k], local, f, stream);
        else if (t.dtype[k] == GD_F16) gc_scale_chunk<f16_t, CHUNK>(t.src[k], t.dst[k], t.n[k], local, f, stream);
        else gc_scale_chunk<bf16_t, CHUNK>(t.src[k], t.dst[k], t.n[k], local, f, stream);
    }
}

// min(1, max_norm / (norm + 1e-6)), from the binary64 norm: one beyond the range of f32 still gives its factor.  A NaN norm gives a NaN
// factor (every gradient then becomes NaN: nothing is hidden).
__device__ __forceinline__ float gc_factor(double norm, float max_norm) {
    const float f = (float)((double)max_norm / (norm + 1e-6));
    return f < 1.0f || f != f ? f : 1.0f;
}

template <bool INF>
__global__ void __launch_bounds__(256) k_grad_norm(const gc_table t, int first, double* __restrict__ part) {
    __shared__ double lds[4];
    const double v = gc_block<INF>(gc_norm_table<GC_CHUNK, INF>(t, 0.0), lds);
    if (threadIdx.x == 0) part[blockIdx.x] = first ? v : gc_combine<INF>(part[blockIdx.x], v);
}

template <bool INF>
__device__ __forceinline__ double gc_total(const double* __restrict__ part, int parts, double* lds) {
    double v = 0.0;
    for (int i = threadIdx.x; i < parts; i += blockDim.x) v = gc_combine<INF>(v, part[i]);
    v = gc_block<INF>(v, lds);
    return INF ? v : sqrt(v);
}

template <bool INF>
__global__ void __launch_bounds__(256) k_grad_norm_total(const double* __restrict__ part, int parts, float* __restrict__ norm) {
    __shared__ double lds[4];
    const double v = gc_total<INF>(part, parts, lds);
    if (threadIdx.x == 0) norm[0] = (float)v;
}

template <bool INF>
__global__ void __launch_bounds__(256) k_grad_clip(const gc_table t, const double* __restrict__ part, int parts, float max_norm, bool stream, float* __restrict__ norm) {
    __shared__ double lds[4];
    const double v = gc_total<INF>(part, parts, lds);
    if (blockIdx.x == 0 && threadIdx.x == 0) norm[0] = (float)v;
    gc_scale_table<GC_CHUNK>(t, gc_factor(v, max_norm), stream);
}

// A few tensors of few elements: one workgroup does both steps, the chunks being whole tensors.  At 315 KB (an embedding of 77 x 1024 f32) it
// takes 12.8 us for 4.7 + 5.2 us of two launches, but a call every 13.3 us for 15.9: the second launch costs the host 3.3 us.  The two
// meet at about 400 KB; and one tensor after another costs it 2 us each.
#define GC_SMALL_BYTES (384 * 1024)
#define GC_SMALL_TENSORS 4
#define GC_SMALL (1 << 18)      /* elements: no tensor of a small call is cut */
template <bool INF>
__global__ void __launch_bounds__(1024) k_grad_clip_small(const gc_table t, float max_norm, int scale, float* __restrict__ norm) {
    __shared__ double lds[16];
    double v = gc_block<INF>(gc_norm_table<GC_SMALL, INF>(t, 0.0), lds);
    if (!INF) v = sqrt(v);
    if (threadIdx.x == 0) norm[0] = (float)v;
    if (scale) gc_scale_table<GC_SMALL>(t, gc_factor(v, max_norm), false);
}

// tensors [at, ..) into one launch's table; -> how many were taken.  Tensors of no elements take a place but no chunk.
static int gc_fill(gc_table& t, const void* const* src, void* const* dst, const int64_t* n, const int32_t* dtype, int at, int count, int chunk) {
    const int k = count - at < GC_TENSORS ? count - at : GC_TENSORS;
    long long chunks = 0;
    t.count = k;
    for (int i = 0; i < k; ++i) {
        t.src[i] = src[at + i];
        t.dst[i] = dst ? dst[at + i] : nullptr;
        t.n[i] = n[at + i];
        t.dtype[i] = (unsigned char)dtype[at + i];
        t.start[i] = (int)chunks;
        chunks += (n[at + i] + chunk - 1) / chunk;
    }
    t.start[k] = (int)chunks;
    return k;
}

extern "C" size_t gd_grad_norm_workspace_bytes(void) { return GC_GRID * sizeof(double); }

template <bool INF>
static int gc_launch(const void* const* src, void* const* dst, const int64_t* n, const int32_t* dtype, int count, float max_norm, double* part, float* norm,
                     hipStream_t st) {
    gc_table t;
    int parts = 0;
    double bytes = 0, read = 0;
    for (int i = 0; i < count; ++i) {
        const double size = (double)n[i] * (dtype[i] == GD_F32 ? 4 : 2);
        read += size;
        bytes += dst && dst[i] != src[i] ? 2 * size : size;
    }
    if (count <= GC_SMALL_TENSORS && read <= GC_SMALL_BYTES) {
        gc_fill(t, src, dst, n, dtype, 0, count, GC_SMALL);
        k_grad_clip_small<INF><<<1, 1024, 0, st>>>(t, max_norm, dst != nullptr, norm);
        GD_CHECK_LAUNCH("gd_grad_norm");
        return GD_OK;
    }
    for (int at = 0; at < count || at == 0; at += GC_TENSORS) {
        gc_fill(t, src, dst, n, dtype, at, count, GC_CHUNK);
        // one table: as many workgroups as it has chunks; several: all of them, since every launch adds to the first one's partials
        const int grid = count <= GC_TENSORS && t.start[t.count] < GC_GRID ? (t.start[t.count] > 0 ? t.start[t.count] : 1) : GC_GRID;
        k_grad_norm<INF><<<grid, 256, 0, st>>>(t, at == 0, part);
        parts = grid;
    }
    if (!dst) {
        k_grad_norm_total<INF><<<1, 256, 0, st>>>(part, parts, norm);
    } else {
        // backwards: what the norm read last is still in the memory-side cache
        for (int at = (count > 0 ? (count - 1) / GC_TENSORS : 0) * GC_TENSORS; at >= 0; at -= GC_TENSORS) {
            if (count > GC_TENSORS) gc_fill(t, src, dst, n, dtype, at, count, GC_CHUNK);
            const int chunks = t.start[t.count];
            k_grad_clip<INF><<<chunks < 1 ? 1 : chunks < GC_GRID ? chunks : GC_GRID, 256, 0, st>>>(t, part, parts, max_norm, streams_past_cache(bytes), norm);
        }
    }
    GD_CHECK_LAUNCH("gd_grad_norm");
    return GD_OK;
}

// Whether a destination shares memory with another destination or with another tensor's source: its elements would be scaled twice or read
// after they were written, in an order that the launch does not fix.  -1: no memory for the check.
struct gc_span { uintptr_t lo, hi; bool dst; };
static int gc_overlap(const void* const* src, void* const* dst, const int64_t* n, const int32_t* dtype, int count) {
    gc_span* s = (gc_span*)malloc(sizeof(gc_span) * 2 * (size_t)(count ? count : 1));
    if (!s) return -1;
    int k = 0;
    for (int i = 0; i < count; ++i) {
        if (n[i] == 0) continue;
        const uintptr_t bytes = (uintptr_t)n[i] * (dtype[i] == GD_F32 ? 4 : 2);
        s[k++] = {(uintptr_t)dst[i], (uintptr_t)dst[i] + bytes, true};
        if (src[i] != dst[i]) s[k++] = {(uintptr_t)src[i], (uintptr_t)src[i] + bytes, false};
    }
    qsort(s, (size_t)k, sizeof(gc_span), [](const void* a, const void* b) {
        const uintptr_t x = ((const gc_span*)a)->lo, y = ((const gc_span*)b)->lo;
        return x < y ? -1 : x > y ? 1 : 0;
    });
    uintptr_t any = 0, written = 0;
    int bad = 0;
    for (int i = 0; i < k && !bad; ++i) {
        bad = s[i].lo < (s[i].dst ? any : written);
        if (s[i].hi > any) any = s[i].hi;
        if (s[i].dst && s[i].hi > written) written = s[i].hi;
    }
    free(s);
    return bad;
}

extern "C" int gd_grad_norm(const void* const* src, void* const* dst, const int64_t* n, const int32_t* dtype, int count, int inf_norm, float max_norm,
                            void* workspace, size_t workspace_bytes, float* norm, void* stream) {
    GD_REQUIRE(count >= 0 && (count == 0 || (src && n && dtype)) && workspace && norm, GD_EINVAL, "gd_grad_norm: null pointer");
    GD_REQUIRE(workspace_bytes >= gd_grad_norm_workspace_bytes(), GD_EWORKSPACE, "gd_grad_norm: workspace of %zu bytes needed", gd_grad_norm_workspace_bytes());
    GD_REQUIRE(!dst || max_norm >= 0.f, GD_EINVAL, "gd_grad_norm: max_norm must not be negative or NaN");
    for (int i = 0; i < count; ++i) {
        GD_REQUIRE(n[i] >= 0 && n[i] < (1ll << 36), GD_EINVAL, "gd_grad_norm: tensor %d has %lld elements", i, (long long)n[i]);
        GD_REQUIRE(dtype[i] == GD_F16 || dtype[i] == GD_BF16 || dtype[i] == GD_F32, GD_EINVAL, "gd_grad_norm: tensor %d: dtype must be f16/bf16/f32", i);
        const uintptr_t mask = dtype[i] == GD_F32 ? 3 : 1;
        GD_REQUIRE(n[i] == 0 || (src[i] && ((uintptr_t)src[i] & mask) == 0 && (!dst || (dst[i] && ((uintptr_t)dst[i] & mask) == 0))), GD_EINVAL,
                   "gd_grad_norm: tensor %d: null or misaligned pointer", i);
    }
    if (dst) {
        const int bad = gc_overlap(src, dst, n, dtype, count);
        GD_REQUIRE(bad >= 0, GD_ELAUNCH, "gd_grad_norm: out of host memory");
        GD_REQUIRE(!bad, GD_EINVAL, "gd_grad_norm: a destination overlaps another tensor of the call");
    }
    hipStream_t st = as_stream(stream);
    return inf_norm ? gc_launch<true>(src, dst, n, dtype, count, max_norm, (double*)workspace, norm, st)
                    : gc_launch<false>(src, dst, n, dtype, count, max_norm, (double*)workspace, norm, st);
}
