// The norms before and after a transformer block, fused with the block's gate and the scaled residual:
//
//   h = post(x)                      norm on the block's output (or x itself)
//   s = alpha * res + gate * h       the residual stream behind the block; gate [C], [groups, C] (one row per sample) or 1
//   y = pre(s)                       norm in front of the next block
//
// with   layer: xh = (v - mean v) / sqrt(var v + eps)     rms: xh = v / sqrt(mean v^2 + eps)     norm(v) = xh * gamma + beta.
//
// Backward, for gy = dL/dy and gs = dL/ds (what reaches the stream behind y):
//   ds   = N'(gy * gamma_pre, xh_s) + gs,     N'(g, xh) = r (g - mean g [layer only] - xh mean(g xh)),  r = 1 / deviation of the row
//   dres = alpha ds;   dgate = sum ds h;   dh = gate ds;   dx = N'(dh * gamma_post, xh_x) or dh
//   dgamma = sum g_out xh, dbeta = sum g_out over all rows, for each of the two norms.
//
// Bound by HBM: the forward reads x, res and writes s, y once, the backward reads x, res, gy, gs and writes dx, dres once (above 4096
// channels it reads them a second time for the sums of a gate or a norm on x: a launch of their own).  A row stays in registers from its
// load to its last use (64 / 256 / 512 / 1024 threads a row, 8 or 16 channels a thread), so that the two-pass variance and both norms cost
// no second read.  Everything between the loads and the one rounding of each result is binary32; y comes from the sum s
// BEFORE its rounding, and the backward recomputes that sum from x and res instead of reading the rounded s: the gradients are those of
// the function that the forward computed, at the same traffic.
//
// Measured (MI355X; a large copy moves 4.9 TB/s): 32768 x 1280 f32, rms norms on both sides, a gate for each sample: forward 125 us
// (671 MB, 5.4 TB/s), backward 194 us (1.0 GB, 5.2 TB/s) + 7 us for the column sums.  4096 x 640 bf16, one layer norm, one gate: 7.8, 14.6 and
// 3.9 us (the data lie in the caches: the chain of loads and sums of a few rows a wave).  77 x 1024 bf16, forward: 3.9 us.
#include "train_common.hpp"

template <typename T> __device__ __forceinline__ uint32_t bits16(float x) {
    if constexpr (sizeof(T) == 2) return __builtin_bit_cast(unsigned short, (T)x);
    else return 0;
}

// How a thread's N channels lie in a row: words of 16 bytes (8 or 4 channels), neighbouring threads on neighbouring words (BN_WORDS: C and
// every address are multiples of a word; BN_ODD: rows of any length and address); rows shorter than a word element by element (BN_ELEMENTS).
// An object holds them as they are stored (words: packed, half the registers for 16-bit types), so that a load is under way until
// settle() or a value asks for it.  (4096 x 4001 bf16 with a gate, forward and backward: element by element 47 and 113 us, odd words 36 and
// 67; the aligned words of 4096 x 4096 27 and 59.)
enum { BN_ELEMENTS, BN_WORDS, BN_ODD };
template <typename T, int TPR, int N, int MODE> struct bn_part {
    static constexpr bool VEC = MODE != BN_ELEMENTS;
    static constexpr int W = VEC ? word16<T>::N : 1;
    static __device__ __forceinline__ int col(int t, int i) { return ((i / W) * TPR + t) * W + i % W; }
    u32x4 word[VEC ? N / word16<T>::N : 1];
    T one[VEC ? 1 : N];
    __device__ __forceinline__ void load(const T* __restrict__ p, int t, int C) {
        if constexpr (VEC) {
#pragma unroll
            for (int i = 0; i < N; i += W) {
                const int c = col(t, i);
                word[i / W] = u32x4{0, 0, 0, 0};
                if (c < C) {
                    if constexpr (MODE == BN_ODD) word[i / W] = row_word_load<T>(p, c, C);
                    else word[i / W] = *(const u32x4*)(p + c);
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int c = col(t, i);
                one[i] = (T)0.f;
                if (c < C) one[i] = p[c];
            }
        }
    }
    // before the first value after a load
    __device__ __forceinline__ void settle(int t, int C) {
        if constexpr (MODE == BN_ODD) {
#pragma unroll
            for (int i = 0; i < N; i += W)
                if (col(t, i) < C) word[i / W] = row_word_shift<T>(word[i / W], col(t, i), C);
        }
    }
    __device__ __forceinline__ void fill(float x) {
        if constexpr (VEC) {
            const uint32_t bits = sizeof(T) == 4 ? __builtin_bit_cast(uint32_t, x) : 0x10001u * bits16<T>(x);
#pragma unroll
            for (int i = 0; i < N / W; ++i) word[i] = u32x4{bits, bits, bits, bits};
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) one[i] = (T)x;
        }
    }
    __device__ __forceinline__ float operator[](int i) const {
        if constexpr (!VEC) return (float)one[i];
        else if constexpr (sizeof(T) == 4) {
            const uint32_t u = word[i / 4][i % 4];
            return __builtin_bit_cast(float, u);
        }
        else {
            const uint32_t two = word[i / 8][i % 8 / 2];
            return (float)__builtin_bit_cast(T, (unsigned short)(i & 1 ? two >> 16 : two & 0xffffu));
        }
    }
    static __device__ __forceinline__ void store(T* p, int t, int C, const float* v, bool stream) {
#pragma unroll
        for (int i = 0; i < N; i += W) {
            const int c = col(t, i);
            if (c < C) {
                if constexpr (VEC) {
                    word16<T> a;
#pragma unroll
                    for (int j = 0; j < W; ++j) a.v[j] = to_storage<T>(v[i + j]);
                    if constexpr (MODE == BN_ODD) store_row_word(p, c, C, a, stream);
                    else store16(p + c, a, stream);
                } else {
                    p[c] = to_storage<T>(v[i]);
                }
            }
        }
    }
};

// sums of K values over the row's threads, in every one of them.  TPR > 64: through one half of `lds` (2 * K * 16 floats); the halves take
// turns, so that one barrier a sum is enough (whoever writes a half again has passed the barrier of the sum between, behind its reads).
// The caller's row loop is uniform over the workgroup.
template <int TPR, int K>
__device__ __forceinline__ void bn_row_sum(float* v, float* lds, int& turn) {
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = wave_total(v[k]);
    if constexpr (TPR > 64) {
        constexpr int WAVES = TPR / 64;
        float* half = lds + turn * 32;
        turn ^= 1;
        if ((threadIdx.x & 63) == 0) {
#pragma unroll
            for (int k = 0; k < K; ++k) half[k * WAVES + (threadIdx.x >> 6)] = v[k];
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < K; ++k) {
            float s = 0.f;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) s += half[k * WAVES + w];
            v[k] = s;
        }
    }
}

// v -> (mean, 1 / deviation); mean is 0 for the rms norm.  Two passes over the registers: no cancellation for rows far from zero.
template <typename PART, int TPR, int N>
__device__ __forceinline__ void bn_stats(const float* v, int t, int C, int kind, float eps, float* lds, int& turn, float& mean, float& r) {
    mean = 0.f;
    if (kind == GD_NORM_LAYER) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) s += v[i];
        bn_row_sum<TPR, 1>(&s, lds, turn);
        mean = s / (float)C;
    }
    float q = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float d = PART::col(t, i) < C ? v[i] - mean : 0.f;
        q = __builtin_fmaf(d, d, q);
    }
    bn_row_sum<TPR, 1>(&q, lds, turn);
    r = rsqrtf(q / (float)C + eps);
}

template <typename T, int TPR, int N, int MODE>
__global__ void __launch_bounds__(TPR < 256 ? 256 : TPR) k_block_norm(const gd_block_norm_t a, bool stream) {
    using PART = bn_part<T, TPR, N, MODE>;
    constexpr int RPB = TPR < 256 ? 256 / TPR : 1;           // rows a workgroup
    __shared__ float lds[64];
    int turn = 0;
    const int t = threadIdx.x % TPR, C = a.C;
    const long long row = workgroup() * RPB + (TPR < 256 ? __builtin_amdgcn_readfirstlane(threadIdx.x / TPR) : 0);
    if (row >= a.rows) return;                               // TPR >= 256: the whole workgroup has one row
    // everything that the row needs is on its way before the first sum waits for x
    PART x, res, gate, og, ob, eg, eb;
    x.load((const T*)a.x + row * C, t, C);
    if (a.res) res.load((const T*)a.res + row * C, t, C);
    if (a.post_gamma) og.load((const T*)a.post_gamma, t, C);
    if (a.post_beta) ob.load((const T*)a.post_beta, t, C);
    if (a.gate) gate.load((const T*)a.gate + (a.rows_per_gate == a.rows ? 0 : row / a.rows_per_gate) * a.gate_ld, t, C);
    if (a.pre_gamma) eg.load((const T*)a.pre_gamma, t, C);
    if (a.pre_beta) eb.load((const T*)a.pre_beta, t, C);
    float h[N], mean = 0.f, r = 1.f;
    x.settle(t, C);
#pragma unroll
    for (int i = 0; i < N; ++i) h[i] = x[i];
    if (a.post_kind) bn_stats<PART, TPR, N>(h, t, C, a.post_kind, a.post_eps, lds, turn, mean, r);
    if (a.stats && t == 0) { a.stats[row * 4] = mean; a.stats[row * 4 + 1] = r; }
    if (a.post_kind) {
#pragma unroll
        for (int i = 0; i < N; ++i) h[i] = PART::col(t, i) < C ? (h[i] - mean) * r : 0.f;
        if (a.post_gamma) {
            og.settle(t, C);
#pragma unroll
            for (int i = 0; i < N; ++i) h[i] *= og[i];
        }
        if (a.post_beta) {
            ob.settle(t, C);
#pragma unroll
            for (int i = 0; i < N; ++i) h[i] += ob[i];
        }
    }
    if (a.gate) {
        gate.settle(t, C);
#pragma unroll
        for (int i = 0; i < N; ++i) h[i] *= gate[i];
    }
    if (a.res) {
        res.settle(t, C);
#pragma unroll
        for (int i = 0; i < N; ++i) h[i] = __builtin_fmaf(a.res_scale, res[i], h[i]);
    }
    if (a.s) PART::store((T*)a.s + row * C, t, C, h, stream);
    mean = 0.f;
    r = 1.f;
    if (a.pre_kind) bn_stats<PART, TPR, N>(h, t, C, a.pre_kind, a.pre_eps, lds, turn, mean, r);
    if (a.stats && t == 0) { a.stats[row * 4 + 2] = mean; a.stats[row * 4 + 3] = r; }
    if (!a.pre_kind) return;
#pragma unroll
    for (int i = 0; i < N; ++i) h[i] = (h[i] - mean) * r;
    if (a.pre_gamma) {
        eg.settle(t, C);
#pragma unroll
        for (int i = 0; i < N; ++i) h[i] *= eg[i];
    }
    if (a.pre_beta) {
        eb.settle(t, C);
#pragma unroll
        for (int i = 0; i < N; ++i) h[i] += eb[i];
    }
    PART::store((T*)a.y + row * C, t, C, h, stream);
}

// ---- backward -------------------------------------------------------------------------------------------------------------------------
// Bound by HBM like the forward; a row's four loads are issued while the row before is worked on (without that, and with the parameters
// loaded inside the loop, the f32 case above took 417 us: one row's latency after the other).
// Workgroup w takes the rows [w * R, (w + 1) * R) in order; its threads keep the column sums of their channels in registers and leave
// them in the workspace, one row of C floats for each sum: four sums over all rows (slot w) and the gate's, which ends wherever the rows
// of one gate end.  Going through (w, gate row) in order, each step raises w or the gate row by one, so that slot w + gate row is
// a workgroup's own.  k_block_norm_cols then adds the slots of each column in their order: no float atomics, the same bits every time.
enum { BN_PRE_G, BN_PRE_B, BN_POST_G, BN_POST_B, BN_SUMS };

struct bn_bwd_args {
    gd_block_norm_bwd_t a;
    float* sums[BN_SUMS];       // [workgroups, C] or null
    float* gate_sums;           // [workgroups + gate rows - 1, C] or null
    long long rows_per_wg;
    bool stream;
};

// column sums of the workgroup's rows-in-parallel, then to the workspace (threads of the first row)
template <typename PART, int TPR, int N>
__device__ __forceinline__ void bn_flush(float* acc, float* __restrict__ out, int C, float* lds) {
    const int t = threadIdx.x % TPR;
    if constexpr (TPR < 256) {                               // one wave a row: the four waves' sums meet in LDS
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) lds[(threadIdx.x >> 6) * (64 * N) + i * 64 + t] = acc[i];
        __syncthreads();
        // each wave adds and writes a quarter of the channels
#pragma unroll
        for (int k = 0; k < N / 4; ++k) {
            const int i = (threadIdx.x >> 6) * (N / 4) + k, c = PART::col(t, i);
            if (c < C) out[c] = (lds[i * 64 + t] + lds[64 * N + i * 64 + t]) + (lds[2 * 64 * N + i * 64 + t] + lds[3 * 64 * N + i * 64 + t]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int c = PART::col(t, i);
            if (c < C) out[c] = acc[i];
        }
    }
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] = 0.f;
}

// one row's data as the loop carries it from one turn to the next: its loads are under way while the row before it is worked on
template <typename PART> struct bn_row {
    PART x, res, gy, gs;
    float stats[4];
};

// WRAP: there is a gate or a norm on x (their registers otherwise serve occupancy).  SUMS: BN_ALL, or the two halves of a launch whose
// column sums together do not fit the registers (WRAP above 4096 channels): BN_OUT writes dx, dres and sums for the norm in front of the
// next block, BN_WRAP sums for the gate and the norm on x.  (2048 x 8192 bf16 with both: one launch 213 us, spilling, two 110.)
enum { BN_ALL, BN_OUT, BN_WRAP };
template <typename T, int TPR, int N, int MODE, bool WRAP, int SUMS>
__global__ void __launch_bounds__(TPR < 256 ? 256 : TPR) k_block_norm_bwd(const bn_bwd_args b) {
    using PART = bn_part<T, TPR, N, MODE>;
    constexpr int RPB = TPR < 256 ? 256 / TPR : 1;
    // the next row's data beside this one's and the parameters over all rows, where the registers hold them: 1024 threads a row leave none
    constexpr bool AHEAD = TPR * N < 8192;
    __shared__ float lds[TPR < 256 ? 4 * 64 * N : 64];
    int turn = 0;
    const gd_block_norm_bwd_t& a = b.a;
    const int t = threadIdx.x % TPR, C = a.f.C, wave = TPR < 256 ? __builtin_amdgcn_readfirstlane(threadIdx.x / TPR) : 0;
    const long long r0 = (long long)blockIdx.x * b.rows_per_wg, r1 = r0 + b.rows_per_wg < a.f.rows ? r0 + b.rows_per_wg : a.f.rows;
    float pre_g[N] = {}, pre_b[N] = {}, post_g[N] = {}, post_b[N] = {}, dgate[N] = {};
    PART og, ob, eg, gate;
    const auto params = [&](long long gate_row) {
        if (a.f.pre_gamma) eg.load((const T*)a.f.pre_gamma, t, C), eg.settle(t, C); else eg.fill(1.f);
        if constexpr (WRAP) {
            if (a.f.post_gamma) og.load((const T*)a.f.post_gamma, t, C), og.settle(t, C); else og.fill(1.f);
            if (a.f.post_beta) ob.load((const T*)a.f.post_beta, t, C), ob.settle(t, C); else ob.fill(0.f);
            if (a.f.gate) gate.load((const T*)a.f.gate + gate_row * a.f.gate_ld, t, C), gate.settle(t, C); else gate.fill(1.f);
        }
    };
    if (AHEAD) params(0);
    bn_row<PART> cur, next;
    long long held = -1;                                     // the row in `next`
    const auto fetch = [&](long long row) {
        held = row;
        next.x.load((const T*)a.f.x + row * C, t, C);
        if (a.f.res) next.res.load((const T*)a.f.res + row * C, t, C); else next.res.fill(0.f);
        if (a.gy) next.gy.load((const T*)a.gy + row * C, t, C); else next.gy.fill(0.f);
        if (a.gs) next.gs.load((const T*)a.gs + row * C, t, C); else next.gs.fill(0.f);
        if (a.f.stats) {
#pragma unroll
            for (int k = 0; k < 4; ++k) next.stats[k] = a.f.stats[row * 4 + k];
        }
    };
    const long long per = WRAP && a.f.gate ? a.f.rows_per_gate : a.f.rows;
    if (AHEAD && r0 + wave < r1) fetch(r0 + wave);
    for (long long g0 = r0; g0 < r1;) {
        const long long gate_row = per == a.f.rows ? 0 : g0 / per;
        const long long g1 = (gate_row + 1) * per < r1 ? (gate_row + 1) * per : r1;
        if constexpr (WRAP && AHEAD) {
            if (a.f.gate) gate.load((const T*)a.f.gate + gate_row * a.f.gate_ld, t, C), gate.settle(t, C);
        }
        for (long long row = g0 + wave; row < g1; row += RPB) {        // (TPR >= 256: the same rows for the whole workgroup)
            if constexpr (!AHEAD) {
                asm volatile("" ::: "memory");               // (else the parameters are held in registers over all rows, as floats)
                params(gate_row);
            }
            if (!AHEAD || held != row) fetch(row);           // (held: not so for a wave that had no row of the gate before)
            cur = next;
            if constexpr (AHEAD) {
                // the row behind this one: of this gate, or the first of the next gate's rows
                const long long then = row + RPB < g1 ? row + RPB : g1 + wave;
                if (then < r1) fetch(then);
            }
            cur.x.settle(t, C);
            if (a.f.res) cur.res.settle(t, C);
            if (a.gy) cur.gy.settle(t, C);
            if (a.gs) cur.gs.settle(t, C);
            float d[N], sv[N], xh[N];
            // forward again: xh = normalised x, h = post(x), sv = the sum
            const float post_mean = WRAP && a.f.post_kind ? cur.stats[0] : 0.f, post_r = WRAP && a.f.post_kind ? cur.stats[1] : 1.f;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                xh[i] = PART::col(t, i) < C ? (cur.x[i] - post_mean) * post_r : 0.f;
                float h = xh[i];
                if constexpr (WRAP) h = gate[i] * __builtin_fmaf(h, og[i], ob[i]);
                sv[i] = __builtin_fmaf(a.f.res_scale, cur.res[i], h);
            }
            // ds
            if (a.gy) {
                const float mean = cur.stats[2], r = cur.stats[3];
                float m[2] = {0.f, 0.f};
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    sv[i] = PART::col(t, i) < C ? (sv[i] - mean) * r : 0.f;
                    const float g = cur.gy[i];
                    if constexpr (SUMS != BN_WRAP) {
                        pre_g[i] = __builtin_fmaf(g, sv[i], pre_g[i]);
                        pre_b[i] += g;
                    }
                    d[i] = g * eg[i];
                    m[0] += d[i];
                    m[1] = __builtin_fmaf(d[i], sv[i], m[1]);
                }
                bn_row_sum<TPR, 2>(m, lds, turn);
                const float m0 = a.f.pre_kind == GD_NORM_LAYER ? m[0] / (float)C : 0.f, m1 = m[1] / (float)C;
#pragma unroll
                for (int i = 0; i < N; ++i) d[i] = PART::col(t, i) < C ? __builtin_fmaf(r, d[i] - m0 - sv[i] * m1, cur.gs[i]) : 0.f;
            } else {
#pragma unroll
                for (int i = 0; i < N; ++i) d[i] = cur.gs[i];
            }
            if (SUMS != BN_WRAP && a.dres) {
                float w[N];
#pragma unroll
                for (int i = 0; i < N; ++i) w[i] = a.f.res_scale * d[i];
                PART::store((T*)a.dres + row * C, t, C, w, b.stream);
            }
            if constexpr (WRAP) {
                float m[2] = {0.f, 0.f};
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    if constexpr (SUMS != BN_OUT) dgate[i] = __builtin_fmaf(d[i], __builtin_fmaf(xh[i], og[i], ob[i]), dgate[i]);
                    d[i] *= gate[i];
                    if constexpr (SUMS != BN_OUT) {
                        post_g[i] = __builtin_fmaf(d[i], xh[i], post_g[i]);
                        post_b[i] += d[i];
                    }
                    if (a.f.post_kind) {
                        d[i] *= og[i];
                        m[0] += d[i];
                        m[1] = __builtin_fmaf(d[i], xh[i], m[1]);
                    }
                }
                if (SUMS != BN_WRAP && a.f.post_kind) {
                    bn_row_sum<TPR, 2>(m, lds, turn);
                    const float m0 = a.f.post_kind == GD_NORM_LAYER ? m[0] / (float)C : 0.f, m1 = m[1] / (float)C;
#pragma unroll
                    for (int i = 0; i < N; ++i) d[i] = post_r * (d[i] - m0 - xh[i] * m1);
                }
            }
            if (SUMS != BN_WRAP && a.dx) PART::store((T*)a.dx + row * C, t, C, d, b.stream);
        }
        if constexpr (WRAP && SUMS != BN_OUT) {
            if (b.gate_sums) bn_flush<PART, TPR, N>(dgate, b.gate_sums + ((long long)blockIdx.x + gate_row) * C, C, lds);
        }
        g0 = g1;
    }
    if constexpr (SUMS != BN_WRAP) {
        if (b.sums[BN_PRE_G]) bn_flush<PART, TPR, N>(pre_g, b.sums[BN_PRE_G] + (long long)blockIdx.x * C, C, lds);
        if (b.sums[BN_PRE_B]) bn_flush<PART, TPR, N>(pre_b, b.sums[BN_PRE_B] + (long long)blockIdx.x * C, C, lds);
    }
    if constexpr (WRAP && SUMS != BN_OUT) {
        if (b.sums[BN_POST_G]) bn_flush<PART, TPR, N>(post_g, b.sums[BN_POST_G] + (long long)blockIdx.x * C, C, lds);
        if (b.sums[BN_POST_B]) bn_flush<PART, TPR, N>(post_b, b.sums[BN_POST_B] + (long long)blockIdx.x * C, C, lds);
    }
}

// out[c] = sum over the slots of one sum.  blockIdx.y < BN_SUMS: a sum over all workgroups; above: the gate row blockIdx.y - BN_SUMS, which
// workgroups floor(g per / R) .. floor((g per + per - 1) / R) have.  16 channels a workgroup, 64 slots side by side.
template <typename T>
__global__ void __launch_bounds__(1024) k_block_norm_cols(const bn_bwd_args b, int workgroups) {
    __shared__ float lds[64][17];
    const gd_block_norm_bwd_t& a = b.a;
    const int C = a.f.C, c = blockIdx.x * 16 + (threadIdx.x & 15), lane = threadIdx.x >> 4;
    const float* src;
    T* out;
    long long lo = 0, hi = workgroups;
    if (blockIdx.y < BN_SUMS) {
        void* const dst[BN_SUMS] = {a.dpre_gamma, a.dpre_beta, a.dpost_gamma, a.dpost_beta};
        src = b.sums[blockIdx.y];
        out = (T*)dst[blockIdx.y];
        if (!src) return;
    } else {
        const long long g = blockIdx.y - BN_SUMS, per = a.f.rows_per_gate;
        lo = g * per / b.rows_per_wg;
        hi = ((g + 1) * per - 1) / b.rows_per_wg + 1;
        src = b.gate_sums + g * C;
        out = (T*)a.dgate + g * C;
    }
    float s = c < C ? sum_strided(src + c, C, (int)lo + lane, (int)hi, 64) : 0.f;
    lds[lane][threadIdx.x & 15] = s;
    __syncthreads();
    if (lane == 0 && c < C) {
        s = lds[0][threadIdx.x];
#pragma unroll 8
        for (int w = 1; w < 64; ++w) s += lds[w][threadIdx.x];
        out[c] = to_storage<T>(s);
    }
}

static bool bn_aligned(const void* p) { return ((uintptr_t)p & 15) == 0; }

static bool bn_words(const gd_block_norm_t& f, int elem) {
    return f.C * elem % 16 == 0 && bn_aligned(f.x) && bn_aligned(f.res) && bn_aligned(f.gate) && (!f.gate || f.gate_ld * elem % 16 == 0) &&
           bn_aligned(f.post_gamma) && bn_aligned(f.post_beta) && bn_aligned(f.pre_gamma) && bn_aligned(f.pre_beta) && bn_aligned(f.s) && bn_aligned(f.y);
}

#define BN_MAX_C 16384

// threads a row: a wave up to 1024 channels (no barrier), then more of them; 8 channels a thread where they suffice
#define BN_SHAPE(C, X)                                                                                        \
    do {                                                                                                      \
        if ((C) <= 512) X(64, 8);                                                                             \
        else if ((C) <= 1024) X(64, 16);                                                                      \
        else if ((C) <= 2048) X(256, 8);                                                                      \
        else if ((C) <= 4096) X(512, 8);                                                                      \
        else if ((C) <= 8192) X(1024, 8);                                                                     \
        else X(1024, 16);                                                                                     \
    } while (0)

static int bn_check(const gd_block_norm_t* f, int dtype, const char* who) {
    GD_REQUIRE(f && f->x, GD_EINVAL, "%s: null pointer", who);
    GD_REQUIRE(f->rows > 0 && f->C > 0, GD_EINVAL, "%s: rows and C must be positive", who);
    GD_REQUIRE(f->C <= BN_MAX_C, GD_EUNSUPPORTED, "%s: at most %d channels (C=%d)", who, BN_MAX_C, f->C);
    GD_REQUIRE(f->rows < (1ll << 31), GD_EUNSUPPORTED, "%s: too many rows", who);
    GD_REQUIRE(f->post_kind >= 0 && f->post_kind <= GD_NORM_RMS && f->pre_kind >= 0 && f->pre_kind <= GD_NORM_RMS, GD_EINVAL, "%s: bad norm kind", who);
    // (the forward would not apply them, the backward would)
    GD_REQUIRE((f->post_kind || (!f->post_gamma && !f->post_beta)) && (f->pre_kind || (!f->pre_gamma && !f->pre_beta)), GD_EINVAL, "%s: gamma or beta without its norm", who);
    GD_REQUIRE(!f->gate || (f->rows_per_gate > 0 && f->rows % f->rows_per_gate == 0 && f->gate_ld >= f->C), GD_EINVAL,
               "%s: gate rows must divide the rows and be at least C apart", who);
    // (the backward's column sums have a row of workgroups for each; the forward refuses what could not be differentiated)
    GD_REQUIRE(!f->gate || f->rows / f->rows_per_gate <= 65535 - BN_SUMS, GD_EUNSUPPORTED, "%s: at most %d gate rows", who, 65535 - BN_SUMS);
    GD_REQUIRE(dtype == GD_F16 || dtype == GD_BF16 || dtype == GD_F32, GD_EINVAL, "%s: dtype must be f16/bf16/f32", who);
    return GD_OK;
}

template <typename T>
static void bn_launch(const gd_block_norm_t& a, hipStream_t st) {
    const bool stream = streams_past_cache((double)a.rows * a.C * sizeof(T) * (1 + !!a.res + !!a.s + !!a.y));
    const bool words = bn_words(a, sizeof(T));
    if (a.C < word16<T>::N) {
        k_block_norm<T, 64, 8, BN_ELEMENTS><<<grid_of((a.rows + 3) / 4), 256, 0, st>>>(a, stream);
        return;
    }
#define BN_GO(TPR, N)                                                                                         \
    do {                                                                                                      \
        constexpr int rpb = TPR < 256 ? 256 / TPR : 1;                                                        \
        const dim3 grid = grid_of((a.rows + rpb - 1) / rpb);                                                  \
        if (words) k_block_norm<T, TPR, N, BN_WORDS><<<grid, rpb * TPR, 0, st>>>(a, stream);                  \
        else k_block_norm<T, TPR, N, BN_ODD><<<grid, rpb * TPR, 0, st>>>(a, stream);                          \
    } while (0)
    BN_SHAPE(a.C, BN_GO);
#undef BN_GO
}

extern "C" int gd_block_norm(const gd_block_norm_t* f, int dtype, void* stream) {
    const int rc = bn_check(f, dtype, "gd_block_norm");
    if (rc != GD_OK) return rc;
    GD_REQUIRE(f->s || f->y, GD_EINVAL, "gd_block_norm: no output");
    GD_REQUIRE(!f->pre_kind == !f->y, GD_EINVAL, "gd_block_norm: y goes with the norm in front of the next block");
    hipStream_t st = as_stream(stream);
    if (dtype == GD_F32) bn_launch<float>(*f, st);
    else if (dtype == GD_F16) bn_launch<f16_t>(*f, st);
    else bn_launch<bf16_t>(*f, st);
    GD_CHECK_LAUNCH("gd_block_norm");
    return GD_OK;
}

// As many workgroups as are resident at once: one a CU for the kernels with 16 channels or 512 threads a row and more (their registers leave
// one wave a SIMD), two for the others.  Every further one is another row of partial sums to write and add.  At least 4 rows
// each, but for the first ones: the 64 slots that k_block_norm_cols reads side by side cost no more than one (with four waves a row; where
// one wave has a row and a workgroup four, 16: the rows of a gate each are worked on one after the other).
// (16384 x 1024 bf16 with gate and both norms: 256 workgroups 46 us, 512 53, 1024 69; 4096 x 4096 bf16: 41, 47, 59; 16384 x 1280 f32: 119, 109, 116.
// 4 samples of one row of 1280 with a gate each: in one workgroup 19 us, in four 11.5; 64 rows: 16 and 64 workgroups 15.4 and 12.2, of 1000
// channels 11.8 and 12.7.)
static long long bn_workgroups(long long rows, int C) {
    const long long first = C > 1024 ? 64 : 16, n = rows < first ? rows : rows < 4 * first ? first : (rows + 3) / 4;
    const long long most = (C > 512 && C <= 1024) || C > 2048 ? 256 : 512;
    return n < most ? n : most;
}

extern "C" size_t gd_block_norm_bwd_workspace_bytes(int64_t rows, int C, int64_t gate_rows) {
    const long long wg = bn_workgroups(rows, C);
    return sizeof(float) * (size_t)C * (size_t)(BN_SUMS * wg + (gate_rows > 0 ? wg + gate_rows - 1 : 0));
}

template <typename T, int TPR, int N, int MODE>
static void bn_go_bwd(const bn_bwd_args& b, int wg, bool wrap, bool wrap_sums, hipStream_t st) {
    constexpr int threads = TPR < 256 ? 256 : TPR;
    if (!wrap) {
        k_block_norm_bwd<T, TPR, N, MODE, false, BN_ALL><<<wg, threads, 0, st>>>(b);
    } else if constexpr (TPR * N >= 8192) {
        k_block_norm_bwd<T, TPR, N, MODE, true, BN_OUT><<<wg, threads, 0, st>>>(b);
        if (wrap_sums) k_block_norm_bwd<T, TPR, N, MODE, true, BN_WRAP><<<wg, threads, 0, st>>>(b);
    } else {
        k_block_norm_bwd<T, TPR, N, MODE, true, BN_ALL><<<wg, threads, 0, st>>>(b);
    }
}

template <typename T>
static void bn_launch_bwd(const gd_block_norm_bwd_t& a, float* ws, hipStream_t st) {
    bn_bwd_args b;
    b.a = a;
    b.stream = streams_past_cache((double)a.f.rows * a.f.C * sizeof(T) * (1 + !!a.f.res + !!a.gy + !!a.gs + !!a.dx + !!a.dres));
    const long long wg0 = bn_workgroups(a.f.rows, a.f.C);
    b.rows_per_wg = (a.f.rows + wg0 - 1) / wg0;
    const int wg = (int)((a.f.rows + b.rows_per_wg - 1) / b.rows_per_wg);
    void* const dst[BN_SUMS] = {a.dpre_gamma, a.dpre_beta, a.dpost_gamma, a.dpost_beta};
    int any = 0;
    for (int k = 0; k < BN_SUMS; ++k) {
        b.sums[k] = dst[k] ? ws + (size_t)k * wg0 * a.f.C : nullptr;
        any |= dst[k] != nullptr;
    }
    b.gate_sums = a.dgate ? ws + (size_t)BN_SUMS * wg0 * a.f.C : nullptr;
    const bool wrap = a.f.gate || a.f.post_kind, wrap_sums = a.dgate || a.dpost_gamma || a.dpost_beta;
    const bool words = bn_words(a.f, sizeof(T)) && bn_aligned(a.gy) && bn_aligned(a.gs) && bn_aligned(a.dx) && bn_aligned(a.dres);
#define BN_GO(TPR, N)                                                                                         \
    do {                                                                                                      \
        if (words) bn_go_bwd<T, TPR, N, BN_WORDS>(b, wg, wrap, wrap_sums, st);                                \
        else bn_go_bwd<T, TPR, N, BN_ODD>(b, wg, wrap, wrap_sums, st);                                        \
    } while (0)
    if (a.f.C < word16<T>::N) k_block_norm_bwd<T, 64, 8, BN_ELEMENTS, true, BN_ALL><<<wg, 256, 0, st>>>(b);
    else BN_SHAPE(a.f.C, BN_GO);
#undef BN_GO
    const int gates = a.dgate ? (int)(a.f.rows / a.f.rows_per_gate) : 0;
    if (any || gates) k_block_norm_cols<T><<<dim3((a.f.C + 15) / 16, BN_SUMS + gates), 1024, 0, st>>>(b, wg);
}

extern "C" int gd_block_norm_bwd(const gd_block_norm_bwd_t* a, void* workspace, size_t workspace_bytes, int dtype, void* stream) {
    GD_REQUIRE(a, GD_EINVAL, "gd_block_norm_bwd: null pointer");
    const int rc = bn_check(&a->f, dtype, "gd_block_norm_bwd");
    if (rc != GD_OK) return rc;
    GD_REQUIRE(a->gy || a->gs, GD_EINVAL, "gd_block_norm_bwd: no incoming gradient");
    GD_REQUIRE(!a->gy || a->f.pre_kind, GD_EINVAL, "gd_block_norm_bwd: gy goes with the norm in front of the next block");
    GD_REQUIRE(a->f.stats || (!a->gy && !a->f.post_kind), GD_EINVAL, "gd_block_norm_bwd: the forward's stats are needed");
    GD_REQUIRE(a->gy || (!a->dpre_gamma && !a->dpre_beta), GD_EINVAL, "gd_block_norm_bwd: dpre_gamma / dpre_beta need gy");
    GD_REQUIRE(a->f.post_kind || (!a->dpost_gamma && !a->dpost_beta), GD_EINVAL, "gd_block_norm_bwd: dpost_gamma / dpost_beta need the norm on x");
    GD_REQUIRE(a->f.gate || !a->dgate, GD_EINVAL, "gd_block_norm_bwd: dgate needs the gate");
    GD_REQUIRE(a->f.res || !a->dres, GD_EINVAL, "gd_block_norm_bwd: dres needs the residual");
    const bool sums = a->dpre_gamma || a->dpre_beta || a->dpost_gamma || a->dpost_beta || a->dgate;
    const size_t need = sums ? gd_block_norm_bwd_workspace_bytes(a->f.rows, a->f.C, a->dgate ? a->f.rows / a->f.rows_per_gate : 0) : 0;
    GD_REQUIRE(!need || (workspace && workspace_bytes >= need), GD_EWORKSPACE, "gd_block_norm_bwd: workspace of %zu bytes needed", need);
    hipStream_t st = as_stream(stream);
    if (dtype == GD_F32) bn_launch_bwd<float>(*a, (float*)workspace, st);
    else if (dtype == GD_F16) bn_launch_bwd<f16_t>(*a, (float*)workspace, st);
    else bn_launch_bwd<bf16_t>(*a, (float*)workspace, st);
    GD_CHECK_LAUNCH("gd_block_norm_bwd");
    return GD_OK;
}
