// Token embedding with scaling, and its gradients.
//
//   y[i] = scale * W[id[i]] + P[i mod L]                      (rows of C channels; P optional)
//   dW[v] = scale * sum over {i: id[i] = v} of dy[i]          dP[l] = sum over the sequences of dy[b, l]
//
// Every row of dW is written: the rows of no token with zeros.  A row's terms are added in binary32 in the order of their positions (dealt
// out to a fixed number of partial sums), without float atomics: the same inputs give the same bits.
// Bound by HBM (dy once, the table's gradient once); for a few prompts by the launch.  Measured (MI355X; a large copy moves 4.9 TB/s):
//   lookup, 1024 x 77 rows of 1280 f16 from a table of 126 MB       41 us: the 202 MB that it writes at 4.9 TB/s, the table out of the cache
//   gradient, 4 x 77 rows into 49408 x 768 f32                       25 us: 152 MB of zeros at 6.1 TB/s, one launch
//   gradient, 2048 x 77 rows of 1024 bf16 into 49408 rows            96 us for the sums (438 MB, 4.5 TB/s), 27 for the sort, 14 for the joins
//   position gradient of the same                                    49 + 5 us (323 MB, a part of it still in the cache)
#include "train_common.hpp"

// A lane's N channels of a slice of 64 * N: one word of 16 bytes at any address (VEC), or, of rows shorter than a word, N single elements,
// neighbouring lanes on neighbouring elements.  Where C is no multiple of the word, a row's last word lies over the one before it: both
// lanes compute and store the same bits for the channels that they share.  (Gradient of 1024 x 77 rows of 1279 f16 channels: element by
// element 197 us, so 84; 1280 channels 80.  Lookup of the same: 127, 65 and 59.)
template <typename T, bool VEC>
struct em_cols {
    static constexpr int N = VEC ? (int)(16 / sizeof(T)) : 8, SLICE = 64 * N;
    // the lane's first channel (C and above: none) and the distance to its next ones
    static constexpr int STEP = VEC ? 1 : 64;
    static __device__ __forceinline__ int col(int slice, int lane, int C) {
        const int c = slice * SLICE + lane * (VEC ? N : 1);
        return VEC && c < C ? row_word_start<T>(c, C) : c;
    }
    static __device__ __forceinline__ void load(const T* __restrict__ p, int slice, int lane, int C, float* v) {
        if constexpr (VEC) {
            const int c = col(slice, lane, C);
            word16<T> a = {};
            if (c < C) a = __builtin_bit_cast(word16<T>, *(const u32x4_any*)(p + c));
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = (float)a.v[i];
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int c = col(slice, lane, C) + i * STEP;
                v[i] = c < C ? (float)p[c] : 0.f;
            }
        }
    }
    static __device__ __forceinline__ void store(T* p, int slice, int lane, int C, const float* v, bool stream) {
        if constexpr (VEC) {
            const int c = col(slice, lane, C);
            word16<T> a;
#pragma unroll
            for (int i = 0; i < N; ++i) a.v[i] = to_storage<T>(v[i]);
            if (c < C) store16<T, u32x4_any>(p + c, a, stream);
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int c = col(slice, lane, C) + i * STEP;
                if (c < C) p[c] = to_storage<T>(v[i]);
            }
        }
    }
    static __device__ __forceinline__ void store_sums(float* p, int slice, int lane, int C, const float* v) {
        const int c = col(slice, lane, C);
        if (c < C) {
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (VEC || c + i * STEP < C) p[c + i * STEP] = v[i];
        }
    }
};

struct em_ids {
    const void* p;
    int wide;                   // 64-bit ids
    __device__ __forceinline__ long long operator[](long long i) const { return wide ? ((const long long*)p)[i] : (long long)((const int*)p)[i]; }
};

// one word (VEC) or element of a row
template <typename T, bool VEC> struct em_piece { T v[VEC ? word16<T>::N : 1]; };
template <typename T, bool VEC> __device__ __forceinline__ em_piece<T, VEC> em_load(const T* p) {
    if constexpr (VEC) return __builtin_bit_cast(em_piece<T, VEC>, *(const u32x4_any*)p);
    else return em_piece<T, VEC>{{*p}};
}
template <typename T, bool VEC> __device__ __forceinline__ void em_store(T* p, const em_piece<T, VEC>& v, bool stream) {
    if constexpr (VEC) store16<T, u32x4_any>(p, __builtin_bit_cast(word16<T>, v), stream);
    else *p = v.v[0];
}
// words or elements of a row of C, and where unit u of it begins
template <typename T, bool VEC> __device__ __forceinline__ int em_units(int C) { return VEC ? (C + word16<T>::N - 1) / word16<T>::N : C; }
template <typename T, bool VEC> __device__ __forceinline__ int em_start(int u, int C) { return VEC ? row_word_start<T>(u * word16<T>::N, C) : u; }

// How a wave covers rows of `units` words (VEC) or elements: 2^shift lanes a row, 64 >> shift rows at a time
static int em_lane_shift(int units) {
    int s = 0;
    while (s < 6 && (1 << s) < units) ++s;
    return s;
}

// An id outside the table gives a row of NaN (there is no such row, and no way to raise from here).
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) k_embed(const em_ids ids, long long n, const T* __restrict__ table, const T* __restrict__ pos, int L, int V, int C,
                                               float scale, bool stream, int shift, T* y) {
    constexpr int W = VEC ? word16<T>::N : 1, BATCH = VEC && sizeof(T) == 2 ? 2 : 4;       // (f16, 1280 channels: 2 words 43.5 us, 4 47.6; f32: 43 and 41)
    const int lane = threadIdx.x & 63, units = em_units<T, VEC>(C), lanes = 1 << shift;
    const long long row = ((workgroup() * 4 + (threadIdx.x >> 6)) << (6 - shift)) + (lane >> shift);
    if (row >= n) return;
    const long long id = ids[row];
    const bool in = id >= 0 && id < V;
    const T* src = table + (in ? id : 0) * C;
    const T* ps = pos ? pos + (long long)((unsigned)row % (unsigned)L) * C : nullptr;
    T* out = y + row * C;
    for (int u0 = 0; u0 < units; u0 += BATCH * lanes) {
        em_piece<T, VEC> w[BATCH], q[BATCH];
        const int u = u0 + (lane & (lanes - 1));
#pragma unroll
        for (int j = 0; j < BATCH; ++j)
            if (u0 + j * lanes < units) {                    // (the same for the whole wave)
                const int at = u + j * lanes < units ? em_start<T, VEC>(u + j * lanes, C) : 0;
                w[j] = em_load<T, VEC>(src + at);
                if (ps) q[j] = em_load<T, VEC>(ps + at);
            }
#pragma unroll
        for (int j = 0; j < BATCH; ++j)
            if (u + j * lanes < units) {
                em_piece<T, VEC> o;
#pragma unroll
                for (int i = 0; i < W; ++i) o.v[i] = to_storage<T>(in ? __builtin_fmaf(scale, (float)w[j].v[i], ps ? (float)q[j].v[i] : 0.f) : __builtin_nanf(""));
                em_store<T, VEC>(out + em_start<T, VEC>(u + j * lanes, C), o, stream);
            }
    }
}

// Zeros in those of the rows [v0, v0 + rows) of the table that `there` (of the row's offset) does not name.
template <typename T, bool VEC, typename THERE>
__device__ __forceinline__ void em_zero_rows(T* dtable, long long v0, int rows, int C, int shift, bool stream, THERE&& there) {
    const int lane = threadIdx.x & 63, units = em_units<T, VEC>(C), lanes = 1 << shift;
    for (int r = ((threadIdx.x >> 6) << (6 - shift)) + (lane >> shift); r < rows; r += (blockDim.x >> 6) << (6 - shift)) {
        if (there(r)) continue;
        T* p = dtable + (v0 + r) * C;
        for (int u = lane & (lanes - 1); u < units; u += lanes) em_store<T, VEC>(p + em_start<T, VEC>(u, C), em_piece<T, VEC>{}, stream);
    }
}

// rows of the table that a workgroup looks after for zeros: about 48 KB of them
#define EM_ZERO_MAX 256
static int em_zero_rows_of(int C, int elem) {
    const int r = 48 * 1024 / (C * elem) / 16 * 16;
    return r < 16 ? 16 : r > EM_ZERO_MAX ? EM_ZERO_MAX : r;
}
// positions that every workgroup may look through by itself, one a thread; with more, they are sorted first
#define EM_SCAN_MAX 1024

// The first workgroups: (position, slice).  The one at a token's first position adds up all of that token's rows, its 16 waves side by side; the
// others end at once.  The workgroups behind them: zero_rows rows of the table each, zeros where no position has the row's token.
template <typename T, bool VEC>
__global__ void __launch_bounds__(EM_SCAN_MAX) k_embed_bwd_scan(const em_ids ids, int n, const T* __restrict__ dy, int V, int C, long long padding, float scale,
                                                                bool stream, int zero_rows, int shift, T* dtable) {
    using COLS = em_cols<T, VEC>;
    constexpr int N = COLS::N, AHEAD = 4, WAVES = EM_SCAN_MAX / 64;
    __shared__ float lds[WAVES][64 * N];
    __shared__ int list[EM_SCAN_MAX], count[WAVES];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int slices = (C + COLS::SLICE - 1) / COLS::SLICE;
    const long long owners = (long long)n * slices, wg = workgroup();
    const long long mine = tid < n ? ids[tid] : -1;
    if (wg < owners) {                                       // (at most 1024 positions of 2^14 slices)
        const int first = (int)((unsigned)wg / slices), sl = (int)((unsigned)wg % slices);
        const long long id = ids[first];
        if (id < 0 || id >= V || id == padding) return;
        const bool same = tid < n && mine == id;
        if (__syncthreads_or(same && tid < first)) return;
        const unsigned long long mask = __ballot(same);
        if (lane == 0) count[wave] = __popcll(mask);
        __syncthreads();
        int at = 0, total = 0;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            if (w < wave) at += count[w];
            total += count[w];
        }
        if (same) list[at + __popcll(mask & ((1ull << lane) - 1))] = tid;
        __syncthreads();
        float acc[N] = {};
        for (int m = wave; m < total; m += AHEAD * WAVES) {  // (behind the last: the first again, adding nothing)
            float v[AHEAD][N];
#pragma unroll
            for (int j = 0; j < AHEAD; ++j) COLS::load(dy + (long long)list[m + WAVES * j < total ? m + WAVES * j : m] * C, sl, lane, C, v[j]);
#pragma unroll
            for (int j = 0; j < AHEAD; ++j)
#pragma unroll
                for (int i = 0; i < N; ++i) acc[i] += m + WAVES * j < total ? v[j][i] : 0.f;
        }
        // the waves that had a row, in their order
        const int waves = total < WAVES ? total : WAVES;
        if (waves > 1) {
#pragma unroll
            for (int i = 0; i < N; ++i) lds[wave][i * 64 + lane] = acc[i];
            __syncthreads();
            if (wave == 0)
                for (int w = 1; w < waves; ++w)
#pragma unroll
                    for (int i = 0; i < N; ++i) acc[i] += lds[w][i * 64 + lane];
        }
        if (wave == 0) {
#pragma unroll
            for (int i = 0; i < N; ++i) acc[i] *= scale;
            COLS::store(dtable + id * C, sl, lane, C, acc, stream);
        }
        return;
    }
    const long long v0 = (wg - owners) * zero_rows;
    if (v0 >= V) return;
    const int rows = v0 + zero_rows < V ? zero_rows : (int)(V - v0);
    if (tid < rows) list[tid] = 0;
    __syncthreads();
    if (mine >= v0 && mine < v0 + rows && mine != padding) list[mine - v0] = 1;
    __syncthreads();
    em_zero_rows<T, VEC>(dtable, v0, rows, C, shift, stream, [&](int r) { return list[r] != 0; });
}

// ---- many positions: the positions sorted by token ---------------------------------------------------------------------------------------
// A stable least-significant-digit radix sort of (token, position), 8 bits a pass, two launches each.  Ids that add nothing get the key
// `vocab` and end up last.  A workgroup counts / moves EM_SORT_KEYS consecutive entries or more, each of its sixteen waves a run of them; the
// rank among equal digits of a round of 64 is a match of the digit's bits over the wave, so that the order of equal tokens is that of their
// positions.  The scatter's workgroups each add up the whole table of counts themselves (at most EM_SORT_BLOCKS rows of 256): a launch
// less than a scan would need.
#define EM_SORT_KEYS 2048
#define EM_SORT_BLOCKS 512

struct em_sort {
    long long n;
    int per_block;              // a multiple of 1024
    int blocks;
};

static em_sort em_sort_of(long long n) {
    long long blocks = (n + EM_SORT_KEYS - 1) / EM_SORT_KEYS;
    if (blocks > EM_SORT_BLOCKS) blocks = EM_SORT_BLOCKS;
    const long long per = ((n + blocks - 1) / blocks + 1023) / 1024 * 1024;
    return em_sort{n, (int)per, (int)((n + per - 1) / per)};
}

struct em_keys {                // a pass's input: the ids themselves, or the last pass's output
    em_ids ids;
    const uint32_t *key, *pos;
    unsigned vocab;
    long long padding;
    __device__ __forceinline__ uint32_t operator()(long long i) const {
        if (key) return key[i];
        const long long id = ids[i];
        return id >= 0 && id < (long long)vocab && id != padding ? (uint32_t)id : vocab;
    }
};

// lanes of the wave whose digit is this lane's (0 for lanes without a key)
__device__ __forceinline__ unsigned long long em_match(int digit, bool live) {
    const unsigned long long all = __ballot(live);
    uint32_t lo = (uint32_t)all, hi = (uint32_t)(all >> 32);
#pragma unroll
    for (int b = 0; b < 8; ++b) {
        const int bit = (int)((unsigned)digit << (31 - b)) >> 31;    // 0 or ~0
        const unsigned long long s = __ballot(bit);
        lo &= ~((uint32_t)s ^ (uint32_t)bit);
        hi &= ~((uint32_t)(s >> 32) ^ (uint32_t)bit);
    }
    return live ? (unsigned long long)hi << 32 | lo : 0;
}

// What this wave's lanes wrote to LDS is what its lanes read from here on (a wave's LDS instructions stay in order; volatile accesses would
// go through the flat path, waiting for each: 24 us instead of 21 for 20000 positions in one launch).
__device__ __forceinline__ void em_wave_order() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
    __builtin_amdgcn_wave_barrier();
}

// counts[digit] += occurrences in the wave's entries [lo, hi)
__device__ __forceinline__ void em_count(const em_keys& k, long long lo, long long hi, int shift, int* counts) {
    const int lane = threadIdx.x & 63;
    for (long long base = lo; base < hi; base += 64) {
        const long long i = base + lane;
        const bool live = i < hi;
        const int d = live ? (int)(k(i) >> shift) & 255 : 0;
        const unsigned long long m = em_match(d, live);
        if (live && (m & ((1ull << lane) - 1)) == 0) counts[d] += __popcll(m);
        em_wave_order();
    }
}

// Exclusive sums over the digits: thread d < 256 gives its digit's count and gets the sum of those below.  All threads call it (it has
// a barrier, behind which what they wrote to LDS before is seen).
__device__ __forceinline__ int em_below(int c, int* sums) {
    const int tid = threadIdx.x, lane = tid & 63;
    int v = c;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int u = __shfl_up(v, o, 64);
        if (lane >= o) v += u;
    }
    if (tid < 256 && lane == 63) sums[tid >> 6] = v;
    __syncthreads();
    const int w = tid >> 6;
    return v - c + (w > 0 ? sums[0] : 0) + (w > 1 ? sums[1] : 0) + (w > 2 ? sums[2] : 0);
}

__global__ void __launch_bounds__(1024) k_embed_sort_count(const em_keys k, const em_sort s, int shift, int* __restrict__ table, uint32_t* __restrict__ there, int there_words) {
    __shared__ int counts[16][256];
    const int tid = threadIdx.x, wave = tid >> 6;
    for (int i = tid; i < 16 * 256; i += 1024) counts[0][i] = 0;
    // the first pass also clears the marks of the tokens that occur, for the last one
    for (int i = blockIdx.x * 1024 + tid; i < there_words; i += gridDim.x * 1024) there[i] = 0;
    __syncthreads();
    const long long run = s.per_block / 16, lo = (long long)blockIdx.x * s.per_block + wave * run, hi = lo + run < s.n ? lo + run : s.n;
    em_count(k, lo, hi, shift, counts[wave]);
    __syncthreads();
    if (tid < 256) {
        int c = 0;
#pragma unroll
        for (int w = 0; w < 16; ++w) c += counts[w][tid];
        table[blockIdx.x * 256 + tid] = c;
    }
}

__global__ void __launch_bounds__(1024) k_embed_sort_move(const em_keys k, const em_sort s, int shift, const int* __restrict__ table, uint32_t* __restrict__ key_out,
                                                          uint32_t* __restrict__ pos_out, unsigned char* __restrict__ there) {
    __shared__ int counts[16][256], part[4][2][256], sums[4];
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, d0 = tid & 255, q = tid >> 8;
    const long long run = s.per_block / 16, lo = (long long)blockIdx.x * s.per_block + wave * run, hi = lo + run < s.n ? lo + run : s.n;
    // up to two rounds of entries (EM_SORT_KEYS a workgroup) stay in registers, loaded before anything else
    const bool few = s.per_block <= EM_SORT_KEYS;
    uint32_t key_of[2] = {}, pos_of[2] = {};
    if (few) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const long long i = lo + 64 * r + lane;
            if (i < hi) {
                key_of[r] = k(i);
                pos_of[r] = k.key ? k.pos[i] : (uint32_t)i;
            }
        }
    }
    for (int i = tid; i < 16 * 256; i += 1024) counts[0][i] = 0;
    // how many entries of digit d0 lie in earlier workgroups, and in all: four threads share a digit
    int before = 0, all = 0;
    for (int b0 = q; b0 < s.blocks; b0 += 32) {
        int c[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) c[j] = table[(b0 + 4 * j < s.blocks ? b0 + 4 * j : b0) * 256 + d0];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int b = b0 + 4 * j;
            before += b < (int)blockIdx.x ? c[j] : 0;
            all += b < s.blocks ? c[j] : 0;
        }
    }
    part[q][0][d0] = before;
    part[q][1][d0] = all;
    __syncthreads();
    int* place = counts[wave];
    int round = 0;
    for (long long base = lo; base < hi; base += 64, ++round) {
        const bool live = base + lane < hi;
        const int d = live ? (int)((few ? key_of[round & 1] : k(base + lane)) >> shift) & 255 : 0;
        const unsigned long long m = em_match(d, live);
        if (live && (m & ((1ull << lane) - 1)) == 0) place[d] += __popcll(m);
        em_wave_order();
    }
    before = part[0][0][d0] + part[1][0][d0] + part[2][0][d0] + part[3][0][d0];
    all = part[0][1][d0] + part[1][1][d0] + part[2][1][d0] + part[3][1][d0];
    int at = em_below(all, sums) + before;                   // first place of this digit's entries of this workgroup
    if (q == 0) {
#pragma unroll
        for (int w = 0; w < 16; ++w) {
            const int c = counts[w][d0];
            counts[w][d0] = at;
            at += c;
        }
    }
    __syncthreads();
    round = 0;
    for (long long base = lo; base < hi; base += 64, ++round) {
        const long long i = base + lane;
        const bool live = i < hi;
        const uint32_t key = few ? key_of[round & 1] : live ? k(i) : 0;
        const int d = (int)(key >> shift) & 255;
        const unsigned long long m = em_match(d, live);
        const int rank = __popcll(m & ((1ull << lane) - 1));
        const int first = live ? place[d] : 0;
        em_wave_order();
        if (live && rank == 0) place[d] = first + __popcll(m);
        em_wave_order();
        if (live) {
            key_out[first + rank] = key;
            pos_out[first + rank] = few ? pos_of[round & 1] : k.key ? k.pos[i] : (uint32_t)i;
            if (there && key < k.vocab) there[key] = 1;
        }
    }
}

// Fewer positions, in one launch: every workgroup looks through all ids and puts those of its own 256 tokens in their places, behind the
// number of smaller ones, which it has counted on the way.  A thread keeps its ids in registers from the one look on, and one digit is left
// to rank by.  (Bound by the workgroup with the padding and the most frequent words, which ranks most of the positions, where the others
// find that they have none among 64, and in large tables by the looks.  The gradient (bf16, by this sort and by the passes above): 5400
// positions and 12000 rows of 64 channels 25 and 36 us, 8192 26 and 37, 16384 35 and 39, 24000 44 and 40; 8192 positions and 300000 rows 30
// and 46, 1000000 rows 52 and 50.)
#define EM_RANGE_MAX 16384
static bool em_by_ranges(long long n, long long vocab) { return n <= EM_RANGE_MAX && vocab < (1 << 20) && n * vocab <= 1ll << 32; }

template <int CHUNKS>
__global__ void __launch_bounds__(1024) k_embed_sort_ranges(const em_ids ids, int n, unsigned vocab, long long padding, uint32_t* __restrict__ key_out,
                                                            uint32_t* __restrict__ pos_out, unsigned char* __restrict__ there) {
    __shared__ int counts[16][256], sums[4], smaller[16];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int chunks = (n + 1023) / 1024, lo = wave * chunks * 64 + lane;
    const uint32_t from = blockIdx.x * 256;
    uint32_t e[CHUNKS];                                      // the key (vocab: no row of the table; ~0: no position), then rank << 9 | 256 | digit, or 0
    const auto look = [&](auto* p) {
        decltype(*p + 0) id[CHUNKS];
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c)
            if (c < chunks) id[c] = p[lo + c * 64 < n ? lo + c * 64 : n - 1];
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c)
            if (c < chunks) e[c] = lo + c * 64 >= n ? ~0u : id[c] >= 0 && (long long)id[c] < (long long)vocab && (long long)id[c] != padding ? (uint32_t)id[c] : vocab;
    };
    if (ids.wide) look((const long long*)ids.p);
    else look((const int*)ids.p);
    for (int i = tid; i < 16 * 256; i += 1024) counts[0][i] = 0;
    __syncthreads();
    int* count = counts[wave];
    int less = 0;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c)
        if (c < chunks) {
            const uint32_t d = e[c] - from;
            const bool live = d < 256 && e[c] != ~0u;
            less += __popcll(__ballot(e[c] < from));
            e[c] = 0;
            if (__ballot(live)) {
                const unsigned long long m = em_match((int)d & 255, live);
                const int rank = __popcll(m & ((1ull << lane) - 1)), first = live ? count[d] : 0;
                em_wave_order();
                if (live && rank == 0) count[d] = first + __popcll(m);
                em_wave_order();
                if (live) e[c] = (uint32_t)(first + rank) << 9 | 256 | d;
            }
        }
    if (lane == 0) smaller[wave] = less;
    __syncthreads();
    int all = 0;
    if (tid < 256) {
#pragma unroll
        for (int w = 0; w < 16; ++w) all += counts[w][tid];
        if (from + tid < vocab) there[from + tid] = all != 0;
    }
    int at = em_below(all, sums);
#pragma unroll
    for (int w = 0; w < 16; ++w) at += smaller[w];
    if (tid < 256) {
#pragma unroll
        for (int w = 0; w < 16; ++w) {
            const int c = counts[w][tid];
            counts[w][tid] = at;
            at += c;
        }
    }
    __syncthreads();
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c)
        if (c < chunks && e[c]) {
            const int d = e[c] & 255, to = counts[wave][d] + (int)(e[c] >> 9);
            key_out[to] = from + d;
            pos_out[to] = (uint32_t)(lo + c * 64);
        }
}

// Sums over the sorted entries: a wave takes a tile of them (at most 64) and one slice of channels, and writes the tokens that begin in its
// tile.  A token that goes on into the next tile but not beyond it is finished by the wave of the tile where it begins (the next one
// leaves it out); one that goes on further leaves a partial sum in each of its tiles: `tail` in the first, `head` in the others.  The
// workgroups behind those write the zero rows.
struct em_sum {
    const uint32_t *key, *pos;
    const unsigned char* there;
    float *head, *tail;         // [tiles, C]
    long long n;
    int tile, tiles, slices, C;
    unsigned vocab;
    float scale;
    bool stream;
    int zero_rows, shift;
};

template <typename T, bool VEC>
__global__ void __launch_bounds__(256) k_embed_bwd_sum(const em_sum a, const T* __restrict__ dy, T* dtable) {
    using COLS = em_cols<T, VEC>;
    constexpr int N = COLS::N, AHEAD = 4;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), C = a.C;
    const long long items = (long long)a.tiles * a.slices;
    const long long item_blocks = (items + 3) / 4;
    if (blockIdx.x < item_blocks) {
        const long long item = (long long)blockIdx.x * 4 + wave;
        if (item >= items) return;
        const int t = (int)(item / a.slices), sl = (int)(item % a.slices);
        const long long e0 = (long long)t * a.tile, e1 = e0 + a.tile;
        // lane = entry: its key, its position; the next tile's beside them
        const bool mine = lane < a.tile && e0 + lane < a.n, theirs = lane < a.tile && e1 + lane < a.n;
        const uint32_t key = mine ? a.key[e0 + lane] : a.vocab, pos = mine ? a.pos[e0 + lane] : 0;
        const uint32_t key2 = theirs ? a.key[e1 + lane] : a.vocab, pos2 = theirs ? a.pos[e1 + lane] : 0;
        const uint32_t next = mine && e0 + lane + 1 < a.n ? a.key[e0 + lane + 1] : 0xffffffffu;
        // (the entries are sorted: two equal ones have only equal ones between them)
        const uint32_t prev = e0 > 0 ? a.key[e0 - 1] : 0xffffffffu, before = e0 > a.tile ? a.key[e0 - a.tile - 1] : 0xffffffffu;
        const uint32_t behind = e1 + a.tile < a.n ? a.key[e1 + a.tile] : 0xffffffffu;
        const uint32_t first = __builtin_amdgcn_readfirstlane(key);
        const bool from_before = prev == first, long_before = before == first;
        unsigned long long ends = __ballot(key != next);     // entries that are their token's last
        const int live = __popcll(__ballot(key < a.vocab));  // sorted: the entries without a row of the table are the last ones
        if (live == 0) return;
        const uint32_t last = __builtin_amdgcn_readlane(key, live - 1);
        int e = 0, stop = live;
        bool partial = false;                                // the token at the front is one of the long ones
        if (from_before) {
            if (!long_before && (ends & (~0ull >> (64 - live)))) e = __builtin_ctzll(ends) + 1;      // finished by the tile before: it began there and ends here
            else partial = true;
        }
        const bool goes = !((ends >> (live - 1)) & 1);
        const bool own_last = !from_before || (ends & ((1ull << (live - 1)) - 1)) != 0;      // the last token begins in this tile
        if (goes && own_last && behind != last) {
            // short: the next tile's entries of it are ours
            const unsigned long long more = __ballot(theirs && key2 == last);
            stop = live + (~more ? __builtin_ctzll(~more) : 64);
        }
        const auto at = [&](int k) { return (uint32_t)(k < a.tile ? __builtin_amdgcn_readlane(pos, k) : __builtin_amdgcn_readlane(pos2, k - a.tile)); };
        float acc[N] = {};
        for (; e < stop; e += AHEAD) {
            float v[AHEAD][N];
#pragma unroll
            for (int j = 0; j < AHEAD; ++j)                  // (the last entry again instead of a branch between the loads)
                COLS::load(dy + (long long)at(e + j < stop ? e + j : stop - 1) * C, sl, lane, C, v[j]);
#pragma unroll
            for (int j = 0; j < AHEAD; ++j) {
                const int k = e + j;
                if (k >= stop) break;
#pragma unroll
                for (int i = 0; i < N; ++i) acc[i] += v[j][i];
                if (stop > live ? k == stop - 1 || (k < live && ((ends >> k) & 1)) : (ends >> k) & 1) {
                    if (partial) {
                        COLS::store_sums(a.head + (long long)t * C, sl, lane, C, acc);
                    } else {
#pragma unroll
                        for (int i = 0; i < N; ++i) acc[i] *= a.scale;
                        const uint32_t row = __builtin_amdgcn_readlane(key, k < live ? k : live - 1);
                        COLS::store(dtable + (long long)row * C, sl, lane, C, acc, a.stream);
                    }
#pragma unroll
                    for (int i = 0; i < N; ++i) acc[i] = 0.f;
                    partial = false;
                }
            }
        }
        if (goes && stop == live) {
            COLS::store_sums((partial ? a.head : a.tail) + (long long)t * C, sl, lane, C, acc);
        }
        return;
    }
    const long long v0 = ((long long)blockIdx.x - item_blocks) * a.zero_rows;
    const int rows = v0 + a.zero_rows < a.vocab ? a.zero_rows : (int)(a.vocab - v0);
    em_zero_rows<T, VEC>(dtable, v0, rows, C, a.shift, a.stream, [&](int r) { return a.there[v0 + r] != 0; });
}

// The tokens that go on for two tiles and more: the tail of the tile where they begin + the heads of the others (padding has half of all
// tiles).  Tiles form groups of EM_GROUP.  The first launch finishes the tokens whose tiles lie in one group; of the others it adds up, group
// by group, the heads from the group's first tile on (into that tile's head), and the tail and heads of the group where they begin (into the
// tail).  The second launch adds those, one for each group.  All rows are read whole: a CU has a bounded number of cache lines on their way.
#define EM_GROUP 64

template <int W> struct alignas(4 * W) em_sums { float v[W]; };

// sum of rows lo, lo + step, .. below hi of `rows`, channels c .. c + W - 1, added to s: 16 rows at a time (8: a join of 64 takes 0.8 us
// more; behind the last: the first again, adding nothing)
template <int W>
__device__ __forceinline__ void em_rows(em_sums<W>& s, const float* __restrict__ rows, long long lo, long long hi, long long step, int C, int c) {
    for (long long k = lo; k < hi; k += 16 * step) {
        em_sums<W> v[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) v[j] = *(const em_sums<W>*)(rows + (k + j * step < hi ? k + j * step : lo) * C + c);
#pragma unroll
        for (int j = 0; j < 16; ++j)
#pragma unroll
            for (int i = 0; i < W; ++i) s.v[i] += k + j * step < hi ? v[j].v[i] : 0.f;
    }
}

template <typename T, int W>
__device__ __forceinline__ void em_write_row(T* __restrict__ p, const em_sums<W>& s, float scale) {
#pragma unroll
    for (int i = 0; i < W; ++i) p[i] = to_storage<T>(s.v[i] * scale);
}

// whether the run of `key` has begun before tile u and goes on into it (the entries are sorted; u in range)
__device__ __forceinline__ bool em_into(const em_sum& a, long long u, uint32_t key) { return u > 0 && a.key[u * a.tile - 1] == key && a.key[u * a.tile] == key; }

// W: channels a thread (4 where C is a multiple of 4, else 1)
template <typename T, int W>
__global__ void __launch_bounds__(256) k_embed_bwd_join(const em_sum a, T* __restrict__ dtable) {
    const int lane = threadIdx.x & 63, C = a.C;
    const int wide = (C + 256 * W - 1) / (256 * W), groups = a.tiles > EM_GROUP ? (a.tiles + EM_GROUP - 1) / EM_GROUP : 0;
    if ((int)blockIdx.x >= groups * wide) {
        const int t = blockIdx.x - groups * wide;            // (a run of three tiles begins in front of the last two)
        const long long e1 = (long long)(t + 1) * a.tile, q = (t / EM_GROUP + 1) * EM_GROUP;
        const uint32_t key = a.key[e1], in_tile = a.key[e1 - 1], behind = a.key[e1 + a.tile], before = t > 0 ? a.key[(long long)t * a.tile - 1] : 0xffffffffu;
        const bool crosses = q < a.tiles && a.key[q * a.tile] == key;
        if (key >= a.vocab || in_tile != key || behind != key || before == key || crosses) return;
        const long long u = (long long)t + 1 + lane;
        const int more = __builtin_ctzll(~__ballot(u < a.tiles && u < q && a.key[u * a.tile] == key));
        for (int c = threadIdx.x * W; c < C; c += 256 * W) {
            em_sums<W> s = *(const em_sums<W>*)(a.tail + (long long)t * C + c);
            em_rows<W>(s, a.head, t + 1, t + 1 + more, 1, C, c);
            em_write_row<T, W>(dtable + (long long)key * C + c, s, a.scale);
        }
        return;
    }
    const int c = (blockIdx.x / groups * 256 + threadIdx.x) * W;
    const long long q = (long long)(blockIdx.x % groups) * EM_GROUP, q2 = q + EM_GROUP, u = q + lane;
    const uint32_t key = a.key[q * a.tile];
    if (q > 0 && key < a.vocab && a.key[q * a.tile - 1] == key) {
        const unsigned long long on = __ballot(u < a.tiles && a.key[u * a.tile] == key);
        const int m = ~on ? __builtin_ctzll(~on) : 64;
        if (m > 1 && c < C) {
            em_sums<W> s = {};
            em_rows<W>(s, a.head, q, q + m, 1, C, c);
            *(em_sums<W>*)(a.head + q * C + c) = s;
        }
    }
    if (q2 >= a.tiles) return;
    const uint32_t key2 = a.key[q2 * a.tile];
    if (key2 >= a.vocab || a.key[q2 * a.tile - 1] != key2 || (q > 0 && a.key[q * a.tile - 1] == key2)) return;
    const int m = __popcll(__ballot(em_into(a, u, key2)));  // the group's last m tiles (not its first: the run begins behind that one's start)
    if (m > 0 && c < C) {
        float* const tail = a.tail + (q2 - 1 - m) * C + c;
        em_sums<W> s = *(const em_sums<W>*)tail;
        em_rows<W>(s, a.head, q2 - m, q2, 1, C, c);
        *(em_sums<W>*)tail = s;
    }
}

template <typename T, int W>
__global__ void __launch_bounds__(256) k_embed_bwd_join_groups(const em_sum a, T* __restrict__ dtable) {
    const int lane = threadIdx.x & 63, C = a.C, c = (blockIdx.y * 256 + threadIdx.x) * W;
    const long long q = (long long)(blockIdx.x + 1) * EM_GROUP, g = q - EM_GROUP;
    const uint32_t key = a.key[q * a.tile], behind = q + 1 < a.tiles ? a.key[(q + 1) * a.tile] : 0xffffffffu;
    if (key >= a.vocab || a.key[q * a.tile - 1] != key || (g > 0 && a.key[g * a.tile - 1] == key)) return;
    const int m = __popcll(__ballot(em_into(a, g + lane, key)));
    if (m == 0 && behind != key) return;                     // two tiles: finished by the wave of the first one
    long long groups = 0;
    for (;; groups += 64) {
        const long long u = q + (groups + lane) * EM_GROUP;
        const unsigned long long on = __ballot(u < a.tiles && a.key[u * a.tile] == key);
        if (~on) {
            groups += __builtin_ctzll(~on);
            break;
        }
    }
    if (c < C) {
        em_sums<W> s = *(const em_sums<W>*)(a.tail + (q - 1 - m) * C + c);
        em_rows<W>(s, a.head, q, q + groups * EM_GROUP, EM_GROUP, C, c);
        em_write_row<T, W>(dtable + (long long)key * C + c, s, a.scale);
    }
}

template <typename T, int W>
static void em_join(const em_sum& a, T* dtable, hipStream_t st) {
    const unsigned wide = (unsigned)((a.C + 256 * W - 1) / (256 * W)), groups = (unsigned)((a.tiles + EM_GROUP - 1) / EM_GROUP);
    if (a.tiles > 2) k_embed_bwd_join<T, W><<<(a.tiles - 2) + (groups > 1 ? groups * wide : 0), 256, 0, st>>>(a, dtable);
    if (groups > 1) k_embed_bwd_join_groups<T, W><<<dim3(groups - 1, wide), 256, 0, st>>>(a, dtable);
}

// dP is the column sum of dy as a [B, L * C] matrix.  A thread has one word (16 bytes; VEC) or element of a row and adds EM_POS_ROWS sequences
// or more of it; the workgroups of one column lie blockIdx.y apart and leave their sums in `part` [gridDim.y, L * C], where there is
// more than one.
#define EM_POS_ROWS 64

template <typename T, bool VEC, bool NT>
__device__ __forceinline__ void em_column(const T* p, long long width, long long b0, long long b1, float* acc) {
    for (long long b = b0; b < b1; b += 8) {
        em_piece<T, VEC> w[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const T* at = p + (b + j < b1 ? b + j : b0) * width;
            if constexpr (NT) w[j] = __builtin_bit_cast(em_piece<T, VEC>, __builtin_nontemporal_load((const u32x4_any*)at));
            else w[j] = em_load<T, VEC>(at);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int i = 0; i < (VEC ? word16<T>::N : 1); ++i) acc[i] += b + j < b1 ? (float)w[j].v[i] : 0.f;
    }
}

// where a thread of k_embed_pos_bwd has its word: those of the sums, then those of the zeros behind them, the last of each moved back to
// end where they end (the zeros are rows of C, which is a word at least)
template <typename T, bool VEC> __device__ __forceinline__ long long em_pos_start(long long u, long long width, long long out_width) {
    constexpr int N = VEC ? word16<T>::N : 1;
    const long long sums = (width + N - 1) / N;
    if (u < sums) return u * N + N <= width ? u * N : width - N;
    const long long at = width + (u - sums) * N;
    return at + N <= out_width || at >= out_width ? at : out_width - N;
}

// stream: dy is larger than the memory-side cache: it is read past it, so that the part which the table's gradient has left there is
// still there when its turn comes
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) k_embed_pos_bwd(const T* __restrict__ dy, long long B, long long width, long long out_width, long long per, bool stream,
                                                       float* __restrict__ part, T* __restrict__ dpos) {
    constexpr int N = VEC ? word16<T>::N : 1;
    const long long at = em_pos_start<T, VEC>((((long long)blockIdx.z << 20) + blockIdx.x) * 256 + threadIdx.x, width, out_width);
    if (at >= out_width) return;
    float acc[N] = {};
    if (at < width) {
        const long long b0 = (long long)blockIdx.y * per, b1 = b0 + per < B ? b0 + per : B;
        if (VEC && stream) em_column<T, VEC, VEC>(dy + at, width, b0, b1, acc);
        else em_column<T, VEC, false>(dy + at, width, b0, b1, acc);
    }
    if (part) {
        if (at < width) {
#pragma unroll
            for (int i = 0; i < N; ++i) part[(long long)blockIdx.y * width + at + i] = acc[i];
        }
    } else {
        em_piece<T, VEC> w;
#pragma unroll
        for (int i = 0; i < N; ++i) w.v[i] = to_storage<T>(acc[i]);
        em_store<T, VEC>(dpos + at, w, false);
    }
}

template <typename T>
__global__ void __launch_bounds__(256) k_embed_pos_join(const float* __restrict__ part, int parts, long long width, long long out_width, T* __restrict__ dpos) {
    const long long at = workgroup() * 256 + threadIdx.x;
    if (at >= out_width) return;
    dpos[at] = to_storage<T>(at < width ? sum_strided(part + at, width, 0, parts, 1) : 0.f);
}

// a row has a word at least
static bool em_vec(int C, int elem) { return C * elem >= 16; }

// picks T and VEC for a launch expression
#define EM_LAUNCH(dtype, vec, CALL)                                                                           \
    do {                                                                                                      \
        if ((dtype) == GD_F32) { using T = float; if (vec) { constexpr bool VEC = true; CALL; } else { constexpr bool VEC = false; CALL; } }   \
        else if ((dtype) == GD_F16) { using T = f16_t; if (vec) { constexpr bool VEC = true; CALL; } else { constexpr bool VEC = false; CALL; } } \
        else { using T = bf16_t; if (vec) { constexpr bool VEC = true; CALL; } else { constexpr bool VEC = false; CALL; } }                     \
    } while (0)

#define EM_ELEM(dtype) ((dtype) == GD_F32 ? 4 : 2)

static int em_check(int64_t n, int64_t vocab, int C, int dtype, const char* who) {
    GD_REQUIRE(n >= 0 && n < (1ll << 30), GD_EUNSUPPORTED, "%s: %lld positions (less than 2^30)", who, (long long)n);
    GD_REQUIRE(vocab > 0 && vocab < (1ll << 31) - 1, GD_EUNSUPPORTED, "%s: a table of %lld rows", who, (long long)vocab);
    GD_REQUIRE(C > 0 && C <= (1 << 20), GD_EUNSUPPORTED, "%s: C=%d", who, C);
    GD_REQUIRE(dtype == GD_F16 || dtype == GD_BF16 || dtype == GD_F32, GD_EINVAL, "%s: dtype must be f16/bf16/f32", who);
    return GD_OK;
}

extern "C" int gd_embed(const void* ids, int ids64, int64_t n, const void* table, int64_t vocab, const void* pos, int L, int C, float scale, void* y, int dtype,
                        void* stream) {
    const int rc = em_check(n, vocab, C, dtype, "gd_embed");
    if (rc != GD_OK) return rc;
    GD_REQUIRE(n > 0 && ids && table && y, GD_EINVAL, "gd_embed: null pointer or no positions");
    GD_REQUIRE(!pos || L > 0, GD_EINVAL, "gd_embed: position rows need the sequence length");
    const bool vec = em_vec(C, EM_ELEM(dtype));
    hipStream_t st = as_stream(stream);
    const int shift = em_lane_shift(vec ? (C * EM_ELEM(dtype) + 15) / 16 : C);
    const long long waves = (n + (64 >> shift) - 1) >> (6 - shift);
    const bool past = streams_past_cache((double)EM_ELEM(dtype) * C * ((double)n + (n < vocab ? n : vocab)));
    EM_LAUNCH(dtype, vec, (k_embed<T, VEC><<<grid_of((waves + 3) / 4), 256, 0, st>>>(em_ids{ids, ids64}, n, (const T*)table, (const T*)pos, L, (int)vocab, C, scale, past, shift, (T*)y)));
    GD_CHECK_LAUNCH("gd_embed");
    return GD_OK;
}

struct em_plan {
    em_sort sort;
    bool ranges;
    int passes, tile, tiles;
    size_t key[2], pos[2], table, there, head, tail, bytes;
};

static em_plan em_plan_of(long long n, long long vocab, int C) {
    em_plan p = {};
    if (n <= EM_SCAN_MAX) return p;
    p.sort = em_sort_of(n);
    p.ranges = em_by_ranges(n, vocab);
    p.passes = 1;
    while (p.passes < 4 && ((unsigned long long)vocab >> (8 * p.passes))) ++p.passes;
    // 64 entries a tile where they give each CU 32 waves (times the slices of 512 channels): a partial sum costs two entries' traffic.  With
    // fewer waves shorter tiles, down to 8, until there are 16 a CU.  (157696 positions of 1024 channels: 64 a tile 153 us, 32 141 us;
    // 600000: 353 and 379 us; 40000 of 768 channels: 32 a tile 67, 16 58, 8 65 us.)
    const long long slices = (C + 511) / 512;
    p.tile = n / 64 * slices >= 8192 ? 64 : 32;
    while (p.tile > 8 && n / p.tile * slices < 4096) p.tile /= 2;
    p.tiles = (int)((n + p.tile - 1) / p.tile);
    size_t at = 0;
    const auto take = [&](size_t bytes) { const size_t here = at; at += (bytes + 255) / 256 * 256; return here; };
    for (int k = 0; k < 2; ++k) { p.key[k] = take(4 * (size_t)n); p.pos[k] = take(4 * (size_t)n); }
    p.table = take(4 * 256 * (size_t)p.sort.blocks);
    p.there = take((size_t)vocab);
    p.head = take(4 * (size_t)p.tiles * C);
    p.tail = take(4 * (size_t)p.tiles * C);
    p.bytes = at;
    return p;
}

extern "C" size_t gd_embed_bwd_workspace_bytes(int64_t n, int64_t vocab, int C) {
    return n < 0 || vocab <= 0 || C <= 0 ? 0 : em_plan_of(n, vocab, C).bytes;
}

extern "C" int gd_embed_bwd(const void* ids, int ids64, int64_t n, const void* dy, int64_t vocab, int C, int64_t padding, float scale, void* dtable,
                            void* workspace, size_t workspace_bytes, int dtype, void* stream) {
    const int rc = em_check(n, vocab, C, dtype, "gd_embed_bwd");
    if (rc != GD_OK) return rc;
    GD_REQUIRE(dtable && (n == 0 || (ids && dy)), GD_EINVAL, "gd_embed_bwd: null pointer");
    const bool vec = em_vec(C, EM_ELEM(dtype));
    const int slice = vec ? 64 * (16 / EM_ELEM(dtype)) : 512, slices = (C + slice - 1) / slice;
    const int zero_rows = em_zero_rows_of(C, EM_ELEM(dtype)), shift = em_lane_shift(vec ? (C * EM_ELEM(dtype) + 15) / 16 : C);
    const long long zeros = (vocab + zero_rows - 1) / zero_rows;
    const bool past = streams_past_cache((double)EM_ELEM(dtype) * C * ((double)n + vocab));
    const em_plan p = em_plan_of(n, vocab, C);
    GD_REQUIRE(!p.bytes || (workspace && workspace_bytes >= p.bytes && ((uintptr_t)workspace & 15) == 0), GD_EWORKSPACE, "gd_embed_bwd: workspace of %zu bytes needed", p.bytes);
    hipStream_t st = as_stream(stream);
    const em_ids in = {ids, ids64};
    if (!p.bytes) {
        const long long grid = n * slices + zeros;
        GD_REQUIRE(grid < (1ll << 31), GD_EUNSUPPORTED, "gd_embed_bwd: table too large");
        EM_LAUNCH(dtype, vec, (k_embed_bwd_scan<T, VEC><<<grid_of(grid), EM_SCAN_MAX, 0, st>>>(in, (int)n, (const T*)dy, (int)vocab, C, padding, scale, past, zero_rows, shift, (T*)dtable)));
    } else {
        const long long grid = ((long long)p.tiles * slices + 3) / 4 + zeros;
        // (the launches of 256 threads below: each less than 2^32)
        GD_REQUIRE(grid < (1ll << 24) && p.tiles + (p.tiles + EM_GROUP - 1ll) / EM_GROUP * ((C + 255) / 256) < (1ll << 24), GD_EUNSUPPORTED,
                   "gd_embed_bwd: too many positions for this width");
        char* const ws = (char*)workspace;
        em_keys k = {in, nullptr, nullptr, (unsigned)vocab, padding};
        const int there_words = (int)((vocab + 3) / 4);
        if (p.ranges) {
            uint32_t *const key = (uint32_t*)(ws + p.key[0]), *const pos = (uint32_t*)(ws + p.pos[0]);
            const unsigned ranges = (unsigned)(vocab / 256 + 1);    // (with the key `vocab`)
            if (n <= 8192) k_embed_sort_ranges<8><<<ranges, 1024, 0, st>>>(in, (int)n, (unsigned)vocab, padding, key, pos, (unsigned char*)(ws + p.there));
            else k_embed_sort_ranges<EM_RANGE_MAX / 1024><<<ranges, 1024, 0, st>>>(in, (int)n, (unsigned)vocab, padding, key, pos, (unsigned char*)(ws + p.there));
            k.key = key;
            k.pos = pos;
        } else {
            for (int i = 0; i < p.passes; ++i) {
                const bool last = i + 1 == p.passes;
                uint32_t *const key = (uint32_t*)(ws + p.key[i & 1]), *const pos = (uint32_t*)(ws + p.pos[i & 1]);
                k_embed_sort_count<<<p.sort.blocks, 1024, 0, st>>>(k, p.sort, 8 * i, (int*)(ws + p.table), (uint32_t*)(ws + p.there), i == 0 ? there_words : 0);
                k_embed_sort_move<<<p.sort.blocks, 1024, 0, st>>>(k, p.sort, 8 * i, (const int*)(ws + p.table), key, pos, last ? (unsigned char*)(ws + p.there) : nullptr);
                k.key = key;
                k.pos = pos;
            }
        }
        const em_sum a = {k.key, k.pos, (const unsigned char*)(ws + p.there), (float*)(ws + p.head), (float*)(ws + p.tail), n, p.tile, p.tiles, slices, C, (unsigned)vocab, scale, past, zero_rows, shift};
        EM_LAUNCH(dtype, vec, (k_embed_bwd_sum<T, VEC><<<(unsigned)grid, 256, 0, st>>>(a, (const T*)dy, (T*)dtable)));
        EM_LAUNCH(dtype, C % 4 == 0, (em_join<T, VEC ? 4 : 1>(a, (T*)dtable, st)));
    }
    GD_CHECK_LAUNCH("gd_embed_bwd");
    return GD_OK;
}

// sequences a workgroup adds, and how many workgroups share a column: as many as give each EM_POS_ROWS, or fewer rows, down to 8, where
// that leaves most CUs without a wave; from 64 sequences on (below, one workgroup and no second launch) and at most 32 (every further one
// is another row of sums to write and read).  (f16, 77 positions, 8 to 32 rows against 64: 256 x 64 channels 6.3 and 9.3 us, 100 x 768 8.5
// and 10.4; 256 x 768, beyond the bound, 11.7 and 10.7; 32 sequences of 768 channels in 4 workgroups 5.5, in one 4.8.)
static int em_pos_parts(long long B, long long width, long long* per) {
    long long rows = EM_POS_ROWS;
    if (B >= 64)
        while (rows > 8 && B / rows * width < 400 * 64 * 8) rows /= 2;
    long long parts = B / rows;
    parts = parts < 1 ? 1 : parts > 32 ? 32 : parts;
    *per = (B + parts - 1) / parts;
    return *per > 0 ? (int)((B + *per - 1) / *per) : 1;
}

extern "C" size_t gd_embed_pos_bwd_workspace_bytes(int64_t B, int L, int C) {
    long long per;
    if (B < 0 || L <= 0 || C <= 0) return 0;
    const int parts = em_pos_parts(B, (long long)L * C, &per);
    return parts > 1 ? sizeof(float) * (size_t)parts * L * C : 0;
}

extern "C" int gd_embed_pos_bwd(const void* dy, int64_t B, int L, int C, int pos_rows, void* dpos, void* workspace, size_t workspace_bytes, int dtype, void* stream) {
    GD_REQUIRE(dpos && B >= 0 && L >= 0 && pos_rows >= L && pos_rows > 0 && (B == 0 || L == 0 || dy), GD_EINVAL, "gd_embed_pos_bwd: bad argument");
    const int rc = em_check(0, 1, C, dtype, "gd_embed_pos_bwd");
    if (rc != GD_OK) return rc;
    const size_t need = gd_embed_pos_bwd_workspace_bytes(B, L, C);
    GD_REQUIRE(!need || (workspace && workspace_bytes >= need), GD_EWORKSPACE, "gd_embed_pos_bwd: workspace of %zu bytes needed", need);
    long long per;
    const int parts = em_pos_parts(B, (long long)L * C, &per);
    const long long width = (long long)L * C, out_width = (long long)pos_rows * C;
    const bool vec = em_vec(C, EM_ELEM(dtype));
    const int word = vec ? 16 / EM_ELEM(dtype) : 1;
    const long long words = (width + word - 1) / word + (out_width - width + word - 1) / word, grid = (words + 255) / 256;
    GD_REQUIRE((out_width + 255) / 256 < (1ll << 31), GD_EUNSUPPORTED, "gd_embed_pos_bwd: too many positions for this width");
    const dim3 g1 = grid_of(grid);
    float* const part = parts > 1 ? (float*)workspace : nullptr;
    hipStream_t st = as_stream(stream);
    EM_LAUNCH(dtype, vec, (k_embed_pos_bwd<T, VEC><<<dim3(g1.x, parts, g1.y), 256, 0, st>>>((const T*)dy, B, width, out_width, per,
                      streams_past_cache((double)B * width * EM_ELEM(dtype)), part, (T*)dpos)));
    if (parts > 1) {
        const dim3 g = grid_of((out_width + 255) / 256);
        if (dtype == GD_F32) k_embed_pos_join<float><<<g, 256, 0, st>>>(part, parts, width, out_width, (float*)dpos);
        else if (dtype == GD_F16) k_embed_pos_join<f16_t><<<g, 256, 0, st>>>(part, parts, width, out_width, (f16_t*)dpos);
        else k_embed_pos_join<bf16_t><<<g, 256, 0, st>>>(part, parts, width, out_width, (bf16_t*)dpos);
    }
    GD_CHECK_LAUNCH("gd_embed_pos_bwd");
    return GD_OK;
}
