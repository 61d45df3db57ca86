// Group norm over channels-last activations with an activation behind it, forward and backward.
//
// x [B, P, C] (P positions of a sample, C channels, G groups of cg = C / G neighbouring channels).  Per sample and group, over the
// P * cg values:  mean,  rstd = 1 / sqrt(var + eps);   xhat = (x - mean) rstd,  z = xhat gamma_c + beta_c,  y = act(z).
// Backward, g = gy act'(z):   gbeta_c = sum g,  ggamma_c = sum g xhat  (over samples and positions),
//                             gx = rstd (gamma_c g - mean(gamma g) - xhat mean(gamma g xhat)).
//
// A block takes a tile of channels (whole groups, or a slice of one wide group) over a piece of a sample's positions.  A thread owns
// E neighbouring channels - 16 bytes - of some positions, so that a wavefront's loads are consecutive bytes of channels-last rows.
// Everything is held in float; variances are sums of squares about a mean that is known (never E[x^2] - mean^2), and pieces
// are joined by the pairwise formula (Chan, Golub, LeVeque 1979), in a fixed order: results are the same bits from run to run.
//
// Where a sample's tile fits the registers of a block (gn_one_shape), one launch reads it once, and small samples share a block; the
// backward needs one more launch for sums over samples.  Else a direction takes three launches (statistics or sums, a join, the result)
// and reads its inputs twice; results go past the caches, so that the second read finds its lines there.
// Bound by memory, or by a block's chain of sums and barriers where samples are small.  us: 256 x 24 x 24 x 32 fp32, 8 groups, forward 13
// (three launches: 24), backward 18 + 4 (32); 16 x 95 x 97 x 320 bf16, 32 groups, statistics 29, result 34, backward's sums 40 and result
// 49 (5.8 TB/s), 14 in three small launches; 8192 x 16000 fp32 in 16 groups forward 490, backward 650 (2.1 and 2.4 TB/s: the chain).
#include "dl_types.h"

#define GN_THREADS 256
#define GN_ONE_THREADS 1024
#define GN_ONE_WIDTH 2048  // channels of a tile of the one-block forms

enum { GN_NONE = DL_ACT_NONE, GN_RELU = DL_ACT_RELU, GN_SILU = DL_ACT_SILU, GN_SIGMOID = DL_ACT_SIGMOID };

struct GnShape {
    int B, C, G, cg;
    long long P;
    int tile_groups;   // groups per tile of channels; 0: a tile is a slice of one group
    int tile_width;    // channels of a tile (the last one may hold fewer)
    int slices;        // slices per group (1 with whole groups)
    int tiles;         // tiles of channels per sample
    int pieces;        // pieces of a sample's positions
    int piece_rows;    // positions of a piece
    int samples;       // samples of a block (one-block forms; 1 otherwise)
};

// (exponential and reciprocal as the hardware has them: an ulp each, and |z| u from the product with log2 e)
__device__ __forceinline__ float gn_sigmoid(float z) { return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * -1.44269504f)); }
template <int ACT>
__device__ __forceinline__ float gn_act(float z) {
    if (ACT == GN_RELU) return z > 0.0f || z != z ? z : 0.0f;
    if (ACT == GN_SILU) return z * gn_sigmoid(z);
    if (ACT == GN_SIGMOID) return gn_sigmoid(z);
    return z;
}
template <int ACT>
__device__ __forceinline__ float gn_slope(float z) {
    if (ACT == GN_RELU) return z > 0.0f ? 1.0f : 0.0f;
    if (ACT == GN_NONE) return 1.0f;
    const float s = gn_sigmoid(z), r = fmaf(-s, s, s);  // s (1 - s)
    return ACT == GN_SILU ? fmaf(z, r, s) : r;
}
// gamma or beta of channel c (stored as `type`); `fallback` where the norm has none
__device__ __forceinline__ float gn_param(const void *p, int type, int c, float fallback) {
    if (!p) return fallback;
    if (type == DL_F32) return ((const float *)p)[c];
    return type == DL_BF16 ? (float)((const dl_bf16 *)p)[c] : (float)((const dl_f16 *)p)[c];
}
__device__ __forceinline__ void gn_param_store(void *p, int type, int c, float v) {
    if (!p) return;
    if (type == DL_F32) ((float *)p)[c] = v;
    else if (type == DL_BF16) ((dl_bf16 *)p)[c] = (dl_bf16)v;
    else ((dl_f16 *)p)[c] = (dl_f16)v;
}

// Sum over a wavefront in a fixed order; every lane gets it.
__device__ __forceinline__ float gn_wave_sum(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

// (count, mean, M2) of two disjoint sets of values
struct GnMoments {
    float n, mean, m2;
};
__device__ __forceinline__ GnMoments gn_join(GnMoments a, GnMoments b) {
    const float n = a.n + b.n;
    if (n == 0.0f) return {0.0f, 0.0f, 0.0f};
    const float d = b.mean - a.mean, f = b.n / n;
    return {n, a.mean + d * f, a.m2 + b.m2 + d * d * a.n * f};
}

// What a thread works on: E channels from `c` on (those below c_end are real), positions row0, row0 + rows, ... of the piece
struct GnPlace {
    int c, c_end, first_group, groups;  // the tile's groups
    int col, row0, rows;                // column of vectors, row of threads, rows of threads
    int sample, first, step;            // one-block forms: the thread's sample in the block, its first position, and how far the next one is
    bool active;
    long long p_begin, p_end;
};
template <int E>
__device__ __forceinline__ GnPlace gn_place(const GnShape &s, int tile, int piece, int threads) {
    GnPlace w;
    int c0;
    if (s.tile_groups) {
        w.first_group = tile * s.tile_groups;
        w.groups = min(s.tile_groups, s.G - w.first_group);
        c0 = w.first_group * s.cg;
        w.c_end = c0 + w.groups * s.cg;
    } else {
        w.first_group = tile / s.slices;
        w.groups = 1;
        c0 = w.first_group * s.cg + (tile % s.slices) * s.tile_width;
        w.c_end = min(c0 + s.tile_width, (w.first_group + 1) * s.cg);
    }
    const int vectors = (w.c_end - c0 + E - 1) / E;
    w.rows = max(1, threads / vectors);
    w.col = threadIdx.x % vectors;
    w.row0 = threadIdx.x / vectors;
    w.active = w.row0 < w.rows;
    w.sample = 0, w.first = w.row0, w.step = w.rows;
    if (s.samples > 1) {
        w.step = (int)s.P;
        w.sample = w.row0 / w.step, w.first = w.row0 % w.step;
        w.active = w.active && w.sample < s.samples;
    }
    w.c = c0 + w.col * E;
    w.p_begin = (long long)piece * s.piece_rows;
    w.p_end = min(w.p_begin + s.piece_rows, s.P);
    return w;
}
template <typename T, int E, bool VEC>
__device__ __forceinline__ void gn_read(const T *p, int real, float (&f)[E]) {
    if constexpr (VEC) {
        dl_unpack<T>(*reinterpret_cast<const dl_words *>(p), f);
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) f[e] = e < real ? (float)p[e] : 0.0f;
    }
}
// PAST: of a tensor that no launch of the call reads again, next to ones that the next launch does
template <typename T, int E, bool VEC, bool PAST>
__device__ __forceinline__ void gn_write(T *p, int real, const float (&f)[E]) {
    if constexpr (VEC) {
        if constexpr (PAST) dl_store_past(p, f);
        else dl_store(p, f);
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (e < real) p[e] = (T)f[e];
    }
}

// Sums of the tile's groups: every thread brings one value per channel, sums[sample * groups + g] (in LDS) are the groups' totals.
// slots: LDS of threads * E floats.
template <int E, int THREADS>
__device__ void gn_group_sums(const GnShape &s, const GnPlace &w, const float (&v)[E], float *slots, float *sums) {
    const int width = w.c_end - (w.c - w.col * E);  // channels of the tile
    const int vectors = (width + E - 1) / E;
    const bool by_vector = s.tile_groups == 0 || s.cg % E == 0;  // a vector's channels belong to one group
    if (by_vector) {
        float t = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) t += v[e];
        slots[threadIdx.x] = w.active ? t : 0.0f;
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) slots[threadIdx.x * E + e] = w.active ? v[e] : 0.0f;
    }
    __syncthreads();
    const int per_row = by_vector ? vectors : vectors * E, per_group = s.tile_groups == 0 ? per_row : (by_vector ? s.cg / E : s.cg);
    // as many lanes as a group has values
    const int rows = s.samples > 1 ? (int)s.P : w.rows, n = rows * per_group, all = s.samples * w.groups;
    int bits = 6;
    while (bits > 0 && n <= 1 << (bits - 1)) --bits;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, first = lane & ((1 << bits) - 1), at_once = 64 >> bits;
    for (int k0 = wave * at_once; k0 < all; k0 += THREADS / 64 * at_once) {
        const int k = k0 + (lane >> bits), sample = s.samples > 1 ? k / w.groups : 0, g = k - sample * w.groups;
        const float *from = slots + sample * rows * per_row + g * per_group;
        float t = 0.0f;
        if (k < all)
#pragma unroll 2
            for (int j = first; j < n; j += 1 << bits) {
                const int row = j / per_group;
                t += from[row * (per_row - per_group) + j];
            }
        for (int o = 1 << bits >> 1; o > 0; o >>= 1) t += __shfl_xor(t, o);
        if (k < all && first == 0) sums[k] = t;
    }
    __syncthreads();
}

// Per channel of the tile, the sum over the block's rows of threads: every thread brings E values, totals[c] (LDS, may be slots) gets
// them.  Two steps: every thread adds a share of one channel's rows, then a thread per channel adds the shares.
template <int E, int THREADS>
__device__ void gn_channel_sums(const GnPlace &w, int width, const float (&v)[E], float *slots, float *totals) {
    const int vectors = (width + E - 1) / E, padded = vectors * E;
    __syncthreads();
    if ((int)threadIdx.x < w.rows * vectors) {
        const float zero[E] = {};
        if (w.active) dl_store(slots + threadIdx.x * E, v);
        else dl_store(slots + threadIdx.x * E, zero);
    }
    __syncthreads();
    const int shares = max(1, THREADS / padded);
    float t = 0.0f;
    if (shares > 1 && (int)threadIdx.x < shares * padded) {
        const int c = threadIdx.x % padded, first = threadIdx.x / padded;
#pragma unroll 4
        for (int r = first; r < w.rows; r += shares) t += slots[r * padded + c];
    }
    __syncthreads();
    if (shares > 1) {
        if ((int)threadIdx.x < shares * padded) slots[threadIdx.x] = t;
        __syncthreads();
    }
    const int parts = shares > 1 ? shares : w.rows;
    float sum[E] = {};
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int c = threadIdx.x + e * THREADS;  // (padded <= THREADS * E)
        if (c < padded)
#pragma unroll 4
            for (int r = 0; r < parts; ++r) sum[e] += slots[r * padded + c];
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < E; ++e)
        if ((int)(threadIdx.x + e * THREADS) < padded) totals[threadIdx.x + e * THREADS] = sum[e];
    __syncthreads();
}

// ---------------------------------------------------------------------------------- forward
// E neighbouring elements as they lie in memory (16 bytes); those past `real` are 0
template <typename T, int E, bool VEC>
__device__ __forceinline__ dl_words gn_raw(const T *p, int real) {
    if constexpr (VEC) return *reinterpret_cast<const dl_words *>(p);
    DlVec<T, E> t;
#pragma unroll
    for (int e = 0; e < E; ++e) t.v[e] = e < real ? p[e] : (T)0.0f;
    return __builtin_bit_cast(dl_words, t);
}
// Their values, unpacked anew at every use: kept as floats, two uses' worth would not fit the registers
template <typename T, int E>
__device__ __forceinline__ void gn_values(dl_words &w, float (&f)[E]) {
    asm volatile("" : "+v"(w));
    dl_unpack<T>(w, f);
}

// A sample's tile - or several small samples - in one block: the values stay in registers from the one read to y.
template <typename T, bool VEC, int NV, int THREADS, int ACT>
__global__ __launch_bounds__(THREADS) void gn_forward_one(const T *__restrict__ x, const void *__restrict__ gamma,
                                                           const void *__restrict__ beta, int ptype, T *__restrict__ y,
                                                           float2 *__restrict__ stats, GnShape s, float eps) {
    constexpr int E = 16 / sizeof(T);
    __shared__ float slots[THREADS * E], sums[GN_ONE_WIDTH];
    const int tile = blockIdx.x % s.tiles, b0 = blockIdx.x / s.tiles * s.samples;
    GnPlace w = gn_place<E>(s, tile, 0, THREADS);
    const int real = w.c_end - w.c, c0 = w.c - w.col * E, b = b0 + w.sample;
    w.active = w.active && b < s.B;
    const long long base = (long long)b * s.P * s.C + w.c;
    const int P = (int)s.P;
    dl_words v[NV];
    int group[E];
    float t[E], m[E], ga[E], be[E];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int p = w.first + i * w.step;
        v[i] = w.active && p < P ? gn_raw<T, E, VEC>(x + base + (long long)p * s.C, real) : dl_words{0, 0, 0, 0};
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
        group[e] = w.active && e < real ? w.sample * w.groups + (w.c + e - c0) / s.cg : 0;
        ga[e] = w.active && e < real ? gn_param(gamma, ptype, w.c + e, 1.0f) : 0.0f;
        be[e] = w.active && e < real ? gn_param(beta, ptype, w.c + e, 0.0f) : 0.0f;
        t[e] = 0.0f;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        float f[E];
        gn_values<T>(v[i], f);
#pragma unroll
        for (int e = 0; e < E; ++e) t[e] += f[e];
    }
    gn_group_sums<E, THREADS>(s, w, t, slots, sums);
    const float per = 1.0f / ((float)P * (float)s.cg);
#pragma unroll
    for (int e = 0; e < E; ++e) {
        m[e] = sums[group[e]] * per;
        t[e] = 0.0f;
    }
    __syncthreads();
    float mean[E];  // of the groups that this thread reports
#pragma unroll
    for (int k = 0; k < E; ++k) mean[k] = (int)(threadIdx.x + k * THREADS) < s.samples * w.groups ? sums[threadIdx.x + k * THREADS] * per : 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        float f[E];
        gn_values<T>(v[i], f);
        if (!w.active || w.first + i * w.step >= P) continue;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float d = e < real ? f[e] - m[e] : 0.0f;
            t[e] = fmaf(d, d, t[e]);
        }
    }
    gn_group_sums<E, THREADS>(s, w, t, slots, sums);
#pragma unroll
    for (int k = 0; k < E; ++k) {
        const int g = threadIdx.x + k * THREADS, of = b0 + g / w.groups;
        if (g < s.samples * w.groups && of < s.B) stats[(long long)of * s.G + w.first_group + g % w.groups] = make_float2(mean[k], 1.0f / sqrtf(fmaf(sums[g], per, eps)));
    }
    if (!w.active) return;
#pragma unroll
    for (int e = 0; e < E; ++e) ga[e] *= 1.0f / sqrtf(fmaf(sums[group[e]], per, eps));
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int p = w.first + i * w.step;
        float o[E];
        gn_values<T>(v[i], o);
        if (p >= P) continue;
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = gn_act<ACT>(fmaf(o[e] - m[e], ga[e], be[e]));
        gn_write<T, E, VEC, false>(y + base + (long long)p * s.C, real, o);
    }
}

// Statistics of a piece of a sample: mean and sum of squares about it per group, [B][G][slices * pieces] (mean, M2).  One read:
// a thread's sums are about its own first value, whose square about the mean is one of the terms that it sums, so that no more than
// a factor of its number of rows is lost to cancellation, whatever the values.
template <typename T, bool VEC, int THREADS>
__global__ __launch_bounds__(THREADS) void gn_stats(const T *__restrict__ x, float2 *__restrict__ part, GnShape s) {
    constexpr int E = 16 / sizeof(T);
    __shared__ float slots[THREADS * E], sums[THREADS * E];
    const int tile = blockIdx.x % s.tiles, piece = blockIdx.x / s.tiles % s.pieces, b = blockIdx.x / s.tiles / s.pieces;
    const GnPlace w = gn_place<E>(s, tile, piece, THREADS);
    const int real = w.c_end - w.c, c0 = w.c - w.col * E;
    const T *from = x + ((long long)b * s.P + w.p_begin) * s.C + w.c;
    const int rows = (int)(w.p_end - w.p_begin);
    float first[E], sum[E] = {}, square[E] = {}, t[E];
    if (w.active && w.row0 < rows) {
        gn_read<T, E, VEC>(from + (long long)w.row0 * s.C, real, first);
#pragma unroll 4
        for (int p = w.row0 + w.rows; p < rows; p += w.rows) {
            float v[E];
            gn_read<T, E, VEC>(from + (long long)p * s.C, real, v);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float d = v[e] - first[e];
                sum[e] += d;
                square[e] = fmaf(d, d, square[e]);
            }
        }
    }
    const float n = w.active && w.row0 < rows ? (float)((rows - 1 - w.row0) / w.rows + 1) : 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) t[e] = n > 0.0f ? fmaf(n, first[e], sum[e]) : 0.0f;
    gn_group_sums<E, THREADS>(s, w, t, slots, sums);
    const float all = (float)rows * (float)(s.tile_groups ? s.cg : w.c_end - c0);
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int group = s.tile_groups && w.active && e < real ? (w.c + e - c0) / s.cg : 0;
        t[e] = 0.0f;
        if (n > 0.0f && e < real) {
            const float mine = sum[e] / n, d = first[e] + mine - sums[group] / all;
            t[e] = fmaxf(square[e] - sum[e] * mine, 0.0f) + n * d * d;
            if (square[e] != square[e]) t[e] = square[e];  // (fmaxf drops a NaN)
        }
    }
    const int slice = s.tile_groups ? 0 : tile % s.slices;
    float2 *to = part + ((long long)b * s.G + w.first_group) * (s.slices * s.pieces) + (long long)piece * s.slices + slice;
    for (int g = threadIdx.x; g < w.groups; g += THREADS) to[(long long)g * (s.slices * s.pieces)].x = sums[g] / all;
    __syncthreads();
    gn_group_sums<E, THREADS>(s, w, t, slots, sums);
    for (int g = threadIdx.x; g < w.groups; g += THREADS) to[(long long)g * (s.slices * s.pieces)].y = sums[g];
}

// mean and rstd of every (sample, group) from its parts: one wavefront each.
__global__ __launch_bounds__(256) void gn_join_stats(const float2 *__restrict__ part, float2 *__restrict__ stats, GnShape s, float eps) {
    const int lane = threadIdx.x & 63;
    const long long bg = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (bg >= (long long)s.B * s.G) return;
    const int parts = s.slices * s.pieces;
    GnMoments a = {0.0f, 0.0f, 0.0f};
    for (int j = lane; j < parts; j += 64) {
        const float2 q = part[bg * parts + j];
        const long long p0 = (long long)(j / s.slices) * s.piece_rows;
        const int width = s.tile_groups ? s.cg : min(s.tile_width, s.cg - (j % s.slices) * s.tile_width);
        a = gn_join(a, {(float)min((long long)s.piece_rows, s.P - p0) * (float)width, q.x, q.y});
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        GnMoments other = {__shfl_xor(a.n, o), __shfl_xor(a.mean, o), __shfl_xor(a.m2, o)};
        a = (lane & o) ? gn_join(other, a) : gn_join(a, other);  // the lower lane's first, on both sides
    }
    if (lane == 0) stats[bg] = make_float2(a.mean, 1.0f / sqrtf(a.m2 / a.n + eps));
}

// y = act((x - mean) rstd gamma + beta) where the statistics are known
template <typename T, bool VEC, int THREADS, int ACT>
__global__ __launch_bounds__(THREADS) void gn_apply(const T *__restrict__ x, const void *__restrict__ gamma, const void *__restrict__ beta,
                                                     int ptype, T *__restrict__ y, const float2 *__restrict__ stats, GnShape s) {
    constexpr int E = 16 / sizeof(T);
    const int tile = blockIdx.x % s.tiles, piece = blockIdx.x / s.tiles % s.pieces, b = blockIdx.x / s.tiles / s.pieces;
    const GnPlace w = gn_place<E>(s, tile, piece, THREADS);
    if (!w.active) return;
    const int real = w.c_end - w.c, rows = (int)(w.p_end - w.p_begin);
    const long long base = ((long long)b * s.P + w.p_begin) * s.C + w.c;
    float scale[E], shift[E], mean[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int c = min(w.c + e, s.C - 1);
        const float2 st = stats[(long long)b * s.G + c / s.cg];
        mean[e] = st.x;
        scale[e] = st.y * gn_param(gamma, ptype, c, 1.0f);
        shift[e] = gn_param(beta, ptype, c, 0.0f);
    }
#pragma unroll 4
    for (int p = w.row0; p < rows; p += w.rows) {
        float v[E];
        gn_read<T, E, VEC>(x + base + (long long)p * s.C, real, v);
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = gn_act<ACT>(fmaf(v[e] - mean[e], scale[e], shift[e]));
        gn_write<T, E, VEC, true>(y + base + (long long)p * s.C, real, v);
    }
}

// ---------------------------------------------------------------------------------- backward
// A thread's channels: what g and xhat are made of
template <int E>
struct GnChannels {
    float mean[E], rstd[E], ga[E], be[E];
    __device__ __forceinline__ GnChannels(const GnShape &s, const GnPlace &w, int b, const float2 *stats, const void *gamma, const void *beta, int ptype) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int c = min(w.c + e, s.C - 1);
            const float2 st = stats[(long long)b * s.G + c / s.cg];
            mean[e] = st.x, rstd[e] = st.y;
            ga[e] = gn_param(gamma, ptype, c, 1.0f), be[e] = gn_param(beta, ptype, c, 0.0f);
        }
    }
    template <int ACT>
    __device__ __forceinline__ void at(int e, float x, float gy, float &hat, float &g) const {
        hat = (x - mean[e]) * rstd[e];
        g = ACT == GN_NONE ? gy : gy * gn_slope<ACT>(fmaf(hat, ga[e], be[e]));
    }
};

// A sample's tile - or several small samples - in one block: x and gy stay in registers from the one read to gx.  A block takes every
// gridDim.x / tiles-th one: its channels are the same ones, whose sums stay in registers until the last; they go to
// [gridDim.x / tiles][2][C].
template <typename T, bool VEC, int NV, int THREADS, int ACT>
__global__ __launch_bounds__(THREADS, NV == 1 && sizeof(T) == 4 ? 4 : 1) void gn_backward_one(const T *__restrict__ x, const T *__restrict__ gy, const void *__restrict__ gamma,
                                                            const void *__restrict__ beta, int ptype, const float2 *__restrict__ stats,
                                                            float *__restrict__ channel, T *__restrict__ gx, void *__restrict__ ggamma,
                                                            void *__restrict__ gbeta, GnShape s) {
    constexpr int E = 16 / sizeof(T);
    __shared__ float slots[THREADS * E], mean_g[GN_ONE_WIDTH + E], mean_x[GN_ONE_WIDTH + E];
    const int tile = blockIdx.x % s.tiles, block0 = blockIdx.x / s.tiles, blocks = gridDim.x / s.tiles;
    const GnPlace w = gn_place<E>(s, tile, 0, THREADS);
    const int real = w.c_end - w.c, c0 = w.c - w.col * E, width = w.c_end - c0, P = (int)s.P;
    const float per = 1.0f / ((float)P * (float)s.cg);
    float all_g[E] = {}, all_x[E] = {};
    for (int block = block0; (long long)block * s.samples < s.B; block += blocks) {
        const int b = min(block * s.samples + w.sample, s.B - 1);
        GnPlace here = w;
        here.active = w.active && block * s.samples + w.sample < s.B;
        const long long base = (long long)b * s.P * s.C + w.c;
        dl_words v[NV] = {}, d[NV] = {};
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int p = w.first + i * w.step;
            if (here.active && p < P) {
                v[i] = gn_raw<T, E, VEC>(x + base + (long long)p * s.C, real);
                d[i] = gn_raw<T, E, VEC>(gy + base + (long long)p * s.C, real);
            }
        }
        const GnChannels<E> ch(s, w, b, stats, gamma, beta, ptype);
        float sg[E] = {}, sx[E] = {};
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float x_[E], d_[E];
            gn_values<T>(v[i], x_), gn_values<T>(d[i], d_);
            if (!here.active || w.first + i * w.step >= P) continue;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                float hat, g;
                ch.template at<ACT>(e, x_[e], d_[e], hat, g);
                sg[e] += g;
                sx[e] = fmaf(g, hat, sx[e]);
            }
        }
#pragma unroll
        for (int e = 0; e < E; ++e) {
            all_g[e] += sg[e], all_x[e] += sx[e];
            sg[e] *= ch.ga[e] * per, sx[e] *= ch.ga[e] * per;
        }
        if (!gx) {
            if constexpr (THREADS != GN_THREADS) break;
            continue;
        }
        // the groups' means of gamma g and of gamma g xhat
        gn_group_sums<E, THREADS>(s, here, sg, slots, mean_g);
        gn_group_sums<E, THREADS>(s, here, sx, slots, mean_x);
        if (here.active) {
            float ma[E], mq[E];
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const int g = w.sample * w.groups + (e < real ? (w.c + e - c0) / s.cg : 0);
                ma[e] = mean_g[g], mq[e] = mean_x[g];
            }
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int p = w.first + i * w.step;
                float x_[E], o[E];
                gn_values<T>(v[i], x_), gn_values<T>(d[i], o);
                if (p >= P) continue;
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    float hat, g;
                    ch.template at<ACT>(e, x_[e], o[e], hat, g);
                    o[e] = ch.rstd[e] * (fmaf(g, ch.ga[e], -ma[e]) - hat * mq[e]);
                }
                gn_write<T, E, VEC, false>(gx + base + (long long)p * s.C, real, o);
            }
        }
        if constexpr (THREADS != GN_THREADS) break;  // (one round: with a second one's values next to these the registers spill)
        __syncthreads();  // the means have been read
    }
    // (from a single block of the tile they are the parameters' gradients already)
    const auto put = [&](int which, void *gradient) {
        for (int c = threadIdx.x; c < width; c += THREADS) {
            if (blocks == 1) gn_param_store(gradient, ptype, c0 + c, slots[c]);
            else channel[((long long)block0 * 2 + which) * s.C + c0 + c] = slots[c];
        }
    };
    gn_channel_sums<E, THREADS>(w, width, all_g, slots, slots);
    put(0, gbeta);
    gn_channel_sums<E, THREADS>(w, width, all_x, slots, slots);
    put(1, ggamma);
}

// Per channel of a piece: sum g and sum g xhat, [B][pieces][2][C].
template <typename T, bool VEC, int THREADS, int ACT>
__global__ __launch_bounds__(THREADS) void gn_backward_sums(const T *__restrict__ x, const T *__restrict__ gy, const void *__restrict__ gamma,
                                                             const void *__restrict__ beta, int ptype, const float2 *__restrict__ stats,
                                                             float *__restrict__ part, GnShape s) {
    constexpr int E = 16 / sizeof(T);
    __shared__ float slots[THREADS * E];
    const int tile = blockIdx.x % s.tiles, piece = blockIdx.x / s.tiles % s.pieces, b = blockIdx.x / s.tiles / s.pieces;
    const GnPlace w = gn_place<E>(s, tile, piece, THREADS);
    const int real = w.c_end - w.c, c0 = w.c - w.col * E, width = w.c_end - c0, rows = (int)(w.p_end - w.p_begin);
    const long long base = ((long long)b * s.P + w.p_begin) * s.C + w.c;
    float sg[E] = {}, sx[E] = {};
    if (w.active) {
        const GnChannels<E> ch(s, w, b, stats, gamma, beta, ptype);
#pragma unroll 4
        for (int p = w.row0; p < rows; p += w.rows) {
            float v[E], d[E];
            gn_read<T, E, VEC>(x + base + (long long)p * s.C, real, v);
            gn_read<T, E, VEC>(gy + base + (long long)p * s.C, real, d);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                float hat, g;
                ch.template at<ACT>(e, v[e], d[e], hat, g);
                sg[e] += g;
                sx[e] = fmaf(g, hat, sx[e]);
            }
        }
    }
    float *out = part + ((long long)b * s.pieces + piece) * 2 * s.C + c0;
    gn_channel_sums<E, THREADS>(w, width, sg, slots, slots);
    for (int c = threadIdx.x; c < width; c += THREADS) out[c] = slots[c];
    gn_channel_sums<E, THREADS>(w, width, sx, slots, slots);
    for (int c = threadIdx.x; c < width; c += THREADS) out[s.C + c] = slots[c];
}

// Per sample: the channels' sums over its pieces ([B][2][C], or null: of a single piece they are there already) and, per group,
// mean(gamma g) and mean(gamma g xhat).
// One block per (sample, group): threads are (channel, share of the pieces).
__global__ __launch_bounds__(256) void gn_backward_join(const float *__restrict__ part, const void *__restrict__ gamma, int ptype,
                                                         float *__restrict__ channel, float2 *__restrict__ group, GnShape s) {
    __shared__ float share[2][256], red[2][4];
    const int g = blockIdx.x % s.G, b = blockIdx.x / s.G;
    const int across = min(s.cg, 256), shares = 256 / across, mine = threadIdx.x / across, col = threadIdx.x % across;
    float a = 0.0f, q = 0.0f;
    for (int c0 = 0; c0 < s.cg; c0 += across) {
        const int c = g * s.cg + c0 + col;
        float sg = 0.0f, sx = 0.0f;
        if (mine < shares && c0 + col < s.cg)
#pragma unroll 4
            for (int i = mine; i < s.pieces; i += shares) {
                const float *row = part + ((long long)b * s.pieces + i) * 2 * s.C + c;
                sg += row[0];
                sx += row[s.C];
            }
        __syncthreads();
        share[0][threadIdx.x] = sg, share[1][threadIdx.x] = sx;
        __syncthreads();
        if (mine == 0 && c0 + col < s.cg) {
            for (int i = 1; i < shares; ++i) sg += share[0][i * across + col], sx += share[1][i * across + col];
            if (channel) {
                channel[(long long)b * 2 * s.C + c] = sg;
                channel[(long long)b * 2 * s.C + s.C + c] = sx;
            }
            const float ga = gn_param(gamma, ptype, c, 1.0f);
            a = fmaf(ga, sg, a);
            q = fmaf(ga, sx, q);
        }
    }
    a = gn_wave_sum(a), q = gn_wave_sum(q);
    if ((threadIdx.x & 63) == 0) red[0][threadIdx.x >> 6] = a, red[1][threadIdx.x >> 6] = q;
    __syncthreads();
    if (threadIdx.x == 0) {
        const float n = (float)s.P * (float)s.cg;
        group[(long long)b * s.G + g] = make_float2((red[0][0] + red[0][1] + red[0][2] + red[0][3]) / n,
                                                    (red[1][0] + red[1][1] + red[1][2] + red[1][3]) / n);
    }
}

template <typename T, bool VEC, int THREADS, int ACT>
__global__ __launch_bounds__(THREADS) void gn_backward_apply(const T *__restrict__ x, const T *__restrict__ gy, const void *__restrict__ gamma,
                                                              const void *__restrict__ beta, int ptype, const float2 *__restrict__ stats,
                                                              const float2 *__restrict__ group, T *__restrict__ gx, GnShape s) {
    constexpr int E = 16 / sizeof(T);
    const int tile = blockIdx.x % s.tiles, piece = blockIdx.x / s.tiles % s.pieces, b = blockIdx.x / s.tiles / s.pieces;
    const GnPlace w = gn_place<E>(s, tile, piece, THREADS);
    if (!w.active) return;
    const int real = w.c_end - w.c, rows = (int)(w.p_end - w.p_begin);
    const long long base = ((long long)b * s.P + w.p_begin) * s.C + w.c;
    const GnChannels<E> ch(s, w, b, stats, gamma, beta, ptype);
    float ma[E], mq[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const float2 gr = group[(long long)b * s.G + min(w.c + e, s.C - 1) / s.cg];
        ma[e] = gr.x, mq[e] = gr.y;
    }
#pragma unroll 4
    for (int p = w.row0; p < rows; p += w.rows) {
        float v[E], d[E];
        gn_read<T, E, VEC>(x + base + (long long)p * s.C, real, v);
        gn_read<T, E, VEC>(gy + base + (long long)p * s.C, real, d);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            float hat, g;
            ch.template at<ACT>(e, v[e], d[e], hat, g);
            v[e] = ch.rstd[e] * (fmaf(g, ch.ga[e], -ma[e]) - hat * mq[e]);
        }
        gn_write<T, E, VEC, true>(gx + base + (long long)p * s.C, real, v);
    }
}

// ggamma_c = sum g xhat, gbeta_c = sum g over n rows of [2][C]: a block takes 32 channels of a share of the rows, 8 at a step, added in a
// fixed order.  With `part` the shares' sums go there, as rows of the same kind.
__global__ __launch_bounds__(256) void gn_param_grads(const float *__restrict__ channel, float *__restrict__ part, void *__restrict__ ggamma,
                                                       void *__restrict__ gbeta, int ptype, int n, int C, int share, int shares) {
    __shared__ float red[2][8][32];
    const int lane = threadIdx.x & 31, r = threadIdx.x >> 5, columns = (C + 31) / 32;
    const unsigned items = (unsigned)columns * shares;  // (below 2^26 times GN_SHARES)
    for (unsigned item = blockIdx.x;; item += gridDim.x) {
        const int c = (int)(item % columns) * 32 + lane, mine = item / columns;
        float sg = 0.0f, sx = 0.0f;
        const int end = min((mine + 1) * (long long)share, (long long)n);
        if (c < C)
#pragma unroll 8
            for (int i = mine * share + r; i < end; i += 8) {
                sg += channel[(long long)i * 2 * C + c];
                sx += channel[(long long)i * 2 * C + C + c];
            }
        red[0][r][lane] = sg, red[1][r][lane] = sx;
        __syncthreads();
        if (threadIdx.x < 64 && c < C) {
            const int which = threadIdx.x >> 5;
            float t = 0.0f;
            for (int i = 0; i < 8; ++i) t += red[which][i][lane];
            if (part) part[((long long)mine * 2 + which) * C + c] = t;
            else gn_param_store(which ? ggamma : gbeta, ptype, c, t);
        }
        if (items - item <= gridDim.x) return;
        __syncthreads();
    }
}

// ---------------------------------------------------------------------------------- host
// (channels are counted in 32 bits, some of them by a tile past the last)
static bool gn_shape_ok(int B, long long P, int C, int G) {
    return B > 0 && P > 0 && C > 0 && C < (1LL << 31) - 65536 && G > 0 && C % G == 0 && P < (1LL << 31) && (long long)B * G < (1LL << 31);
}
// The tiles of channels for blocks of `threads` threads that hold E channels each.
static GnShape gn_tiles(int B, long long P, int C, int G, int E, int threads) {
    GnShape s = {};
    s.B = B, s.P = P, s.C = C, s.G = G, s.cg = C / G;
    const int most = threads * E;
    if (s.cg > most) {
        s.tile_groups = 0;
        s.slices = dl_ceil_div(s.cg, most);
        s.tile_width = dl_ceil_div(dl_ceil_div(s.cg, s.slices), E) * E;
        s.slices = dl_ceil_div(s.cg, s.tile_width);
        s.tiles = G * s.slices;
    } else {
        s.tile_groups = most / s.cg < G ? most / s.cg : G;
        // whole vectors: a tile of several groups starts at a multiple of E where C is one
        while (s.tile_groups > 1 && s.tile_groups < G && (s.tile_groups * s.cg) % E) --s.tile_groups;
        s.slices = 1;
        s.tile_width = s.tile_groups * s.cg;
        s.tiles = dl_ceil_div(G, s.tile_groups);
    }
    s.pieces = s.samples = 1;
    s.piece_rows = (int)(P < (1 << 30) ? P : (1 << 30));
    return s;
}
// Vector loads: every tile's first channel and every row start at 16 bytes.
static bool gn_vectors(const GnShape &s, int E, const void *a, const void *b, const void *c) {
    if (!dl_aligned16(a) || !dl_aligned16(b) || !dl_aligned16(c) || s.C % E) return false;
    if (s.tile_groups == 0) return s.cg % E == 0;
    return s.tiles == 1 || s.tile_width % E == 0;
}
// Pieces of `rows` positions at least, about `blocks` blocks in all
static void gn_pieces(GnShape &s, int rows, int blocks) {
    long long most = (s.P + rows - 1) / rows, want = (blocks + (long long)s.B * s.tiles - 1) / ((long long)s.B * s.tiles);
    long long pieces = want < most ? want : most;
    if (pieces < 1) pieces = 1;
    s.piece_rows = (int)((s.P + pieces - 1) / pieces);
    s.pieces = (int)((s.P + s.piece_rows - 1) / s.piece_rows);
}
static int gn_rows_per_step(const GnShape &s, int E, int threads) {
    const int vectors = (s.tile_width + E - 1) / E;
    return threads / vectors > 0 ? threads / vectors : 1;
}
// 16-byte units that a thread of the one-block forms holds, of x, or of x and of gy: about 48 registers (64 spill)
#define GN_ONE_FORWARD(E) ((E) == 8 ? 10 : 12)
#define GN_ONE_BACKWARD(E) ((E) == 8 ? 4 : 6)
#define GN_SHARES 64  // of many samples, in the sums of the parameters' gradients
#define GN_PARAM_BLOCKS (1 << 20)  // of their launch

static GnShape gn_pieces_shape(int B, long long P, int C, int G, int E) {
    GnShape s = gn_tiles(B, P, C, G, E, GN_THREADS);
    gn_pieces(s, gn_rows_per_step(s, E, GN_THREADS) * 4, 1024);
    return s;
}
static int gn_blocks(const GnShape &s) { return dl_ceil_div(s.B, s.samples) * s.tiles; }  // of the one-block forms
static bool gn_grid_ok(const GnShape &s, int threads) {
    return dl_grid_ok(((long long)s.B + s.samples - 1) / s.samples * s.tiles * s.pieces, threads);
}
static bool gn_pieces_grid_ok(const GnShape &s) { return gn_grid_ok(s, GN_THREADS) && dl_grid_ok((long long)s.B * s.G, 256); }

// The one-block form: tiles of whole groups over all of a sample's positions that a block's registers hold; false where there are
// none, or only tiles of less than 64 bytes per position of a large tensor, whose lines every block would fetch anew.
static bool gn_one_shape(GnShape &s, int B, long long P, int C, int G, int E, int units, int threads) {
    const int cg = C / G;
    const long long vectors = (long long)threads * units / P < threads ? (long long)threads * units / P : threads;
    long long groups = vectors * E / cg < G ? vectors * E / cg : G;  // as many as could fit; fewer are tried below
    // enough blocks for the card's 256 CUs, as long as a position's piece is 64 bytes
    while (groups > 1 && (long long)B * dl_ceil_div(G, groups) < 256 && (groups / 2) * cg >= 4 * E) groups /= 2;
    for (; groups >= 1; --groups) {
        if (groups < G && groups > 1 && groups * cg % E) continue;  // tiles that begin at whole vectors
        s = gn_tiles(B, P, C, G, E, threads);
        s.tile_groups = (int)groups;
        s.slices = 1;
        s.tile_width = (int)groups * cg;
        s.tiles = dl_ceil_div(G, groups);
        s.pieces = 1;
        s.piece_rows = (int)P;
        const int rows = gn_rows_per_step(s, E, threads);
        if ((s.tile_width + E - 1) / E <= threads && s.tile_width <= GN_ONE_WIDTH && (long long)rows * units >= P) {
            // small samples share a block: all of them where that takes a few (the backward then needs no sums over blocks), else as long as
            // there are 512 blocks (65536 rows of 64 channels: 16 a block)
            if (groups == G && threads == GN_THREADS) {
                s.samples = P <= rows ? (int)(rows / P) : 1;
                if (dl_ceil_div(B, s.samples) > 4)
                    while (s.samples > 1 && dl_ceil_div(B, s.samples) < 512) s.samples /= 2;
            }
            return groups == G || s.tile_width >= 4 * E || (long long)B * P * C <= (1 << 18);
        }
    }
    return false;
}

// Which form a direction takes: the threads of a block of the one-block form, 0 for pieces.  `units`: of the larger one-block form.
// (the workspace sizes and the calls both go by this)
static int gn_form(GnShape &s, int B, long long P, int C, int G, int E, int units) {
    for (const int threads : {GN_THREADS, GN_ONE_THREADS})
        if (gn_one_shape(s, B, P, C, G, E, threads == GN_THREADS ? 4 : units, threads)) return threads;
    s = gn_pieces_shape(B, P, C, G, E);
    return 0;
}

// What the backward keeps between its launches, as offsets into the workspace
struct GnBackwardPlan {
    GnShape s;
    int threads;        // gn_form
    int rows;           // of channels' sums, from which the parameters' gradients come; one of the one-block form: they are written at once
    int share, shares;  // rows of a share, and how many shares many rows are added in first (0: all in one launch)
    size_t channel, group, part, share_sums, bytes;
};
static GnBackwardPlan gn_backward_plan(int B, long long P, int C, int G, int E) {
    GnBackwardPlan q = {};
    q.threads = gn_form(q.s, B, P, C, G, E, GN_ONE_BACKWARD(E));
    q.rows = B;
    if (q.threads) {
        q.rows = dl_ceil_div(B, q.s.samples);
        if (q.threads == GN_THREADS) {
            // as many blocks as the card holds at a time, rounds of them after that; a few rounds instead of a launch for the sums over samples
            const int most = 2048 / q.s.tiles > 0 ? 2048 / q.s.tiles : 1;
            q.rows = q.rows <= 4 ? 1 : q.rows < most ? q.rows : most;
        }
    }
    if (q.rows > 512) q.share = dl_ceil_div(q.rows, GN_SHARES), q.shares = dl_ceil_div(q.rows, q.share);
    const auto take = [&](size_t floats) {
        const size_t at = q.bytes;
        q.bytes += dl_align256(floats * sizeof(float));
        return at;
    };
    const bool pieces = !q.threads;
    q.channel = take(pieces ? (q.s.pieces > 1 ? (size_t)B * 2 * C : 0) : q.rows > 1 ? (size_t)q.rows * 2 * C : 0);
    q.group = take(pieces ? (size_t)B * G * 2 : 0);
    q.part = take(pieces ? (size_t)B * q.s.pieces * 2 * C : 0);
    q.share_sums = take((size_t)q.shares * 2 * C);
    if (!q.bytes) q.bytes = 256;  // (a call always has one)
    return q;
}

#define GN_BY_ACT(act, ACT, ...)                   \
    do {                                           \
        if ((act) == GN_NONE) {                    \
            constexpr int ACT = GN_NONE;           \
            __VA_ARGS__;                           \
        } else if ((act) == GN_RELU) {             \
            constexpr int ACT = GN_RELU;           \
            __VA_ARGS__;                           \
        } else if ((act) == GN_SILU) {             \
            constexpr int ACT = GN_SILU;           \
            __VA_ARGS__;                           \
        } else {                                   \
            constexpr int ACT = GN_SIGMOID;        \
            __VA_ARGS__;                           \
        }                                          \
    } while (0)

extern "C" size_t dl_group_norm_fwd_workspace_bytes(int type, int B, long long P, int C, int G) {
    if (!dl_type_known(type) || !gn_shape_ok(B, P, C, G)) return 0;
    const int E = 16 / dl_type_bytes(type);
    GnShape s;
    if (gn_form(s, B, P, C, G, E, GN_ONE_FORWARD(E))) return 256;  // (nothing is kept, but a call always has one)
    return dl_align256((size_t)B * G * s.slices * s.pieces * sizeof(float2));
}

extern "C" int dl_group_norm_fwd(const void *x, const void *gamma, const void *beta, void *y, float *stats, int type, int ptype, int B,
                                 long long P, int C, int G, float eps, int act, void *ws, size_t ws_bytes, void *stream) {
    if (!x || !y || !stats || !ws) return DL_ERR_NULL;
    if (!dl_type_known(type) || !dl_type_known(ptype) || act < DL_ACT_NONE || act > DL_ACT_SIGMOID) return DL_ERR_UNSUPPORTED;
    if (!gn_shape_ok(B, P, C, G) || !(eps >= 0.0f)) return DL_ERR_SHAPE;
    if (ws_bytes < dl_group_norm_fwd_workspace_bytes(type, B, P, C, G)) return DL_ERR_WORKSPACE;
    hipStream_t st = (hipStream_t)stream;
    const int E = 16 / dl_type_bytes(type);
    GnShape s;
    const int threads = gn_form(s, B, P, C, G, E, GN_ONE_FORWARD(E));
    if (threads) {
        if (!gn_grid_ok(s, threads)) return DL_ERR_UNSUPPORTED;
        const bool vec = gn_vectors(s, E, x, y, nullptr);
        const bool few = s.samples > 1 || P <= gn_rows_per_step(s, E, threads);  // a position per thread
        dl_prof_begin("gn_forward_one", st);
#define ONE(VEC, NV, THREADS) \
    gn_forward_one<T, VEC, NV, THREADS, ACT><<<gn_blocks(s), THREADS, 0, st>>>((const T *)x, gamma, beta, ptype, (T *)y, (float2 *)stats, s, eps)
        DL_BY_TYPE(type, T, GN_BY_ACT(act, ACT, if (threads == GN_THREADS) {
                if (few) { if (vec) ONE(true, 1, GN_THREADS); else ONE(false, 1, GN_THREADS); }
                else { if (vec) ONE(true, 4, GN_THREADS); else ONE(false, 4, GN_THREADS); }
            }
                                      else { if (vec) ONE(true, GN_ONE_FORWARD(16 / sizeof(T)), GN_ONE_THREADS); else ONE(false, GN_ONE_FORWARD(16 / sizeof(T)), GN_ONE_THREADS); }));
#undef ONE
        dl_prof_end(st);
        return dl_launch_status();
    }
    if (!gn_pieces_grid_ok(s)) return DL_ERR_UNSUPPORTED;
    const bool vec = gn_vectors(s, E, x, y, nullptr);
    const int blocks = B * s.tiles * s.pieces;
#define FORWARD(VEC)                                                                                                                  \
    DL_TIMED("gn_stats", st, (gn_stats<T, VEC, GN_THREADS><<<blocks, GN_THREADS, 0, st>>>((const T *)x, (float2 *)ws, s)));           \
    DL_TIMED("gn_join_stats", st, (gn_join_stats<<<dl_ceil_div((long long)B * G, 4), 256, 0, st>>>((const float2 *)ws, (float2 *)stats, s, eps))); \
    GN_BY_ACT(act, ACT, DL_TIMED("gn_apply", st, (gn_apply<T, VEC, GN_THREADS, ACT><<<blocks, GN_THREADS, 0, st>>>(                   \
        (const T *)x, gamma, beta, ptype, (T *)y, (const float2 *)stats, s))))
    DL_BY_TYPE(type, T, if (vec) { FORWARD(true); } else { FORWARD(false); });
#undef FORWARD
    return dl_launch_status();
}

extern "C" size_t dl_group_norm_bwd_workspace_bytes(int type, int B, long long P, int C, int G) {
    if (!dl_type_known(type) || !gn_shape_ok(B, P, C, G)) return 0;
    return gn_backward_plan(B, P, C, G, 16 / dl_type_bytes(type)).bytes;
}

extern "C" int dl_group_norm_bwd(const void *x, const void *gy, const void *gamma, const void *beta, const float *stats, void *gx,
                                 void *ggamma, void *gbeta, int type, int ptype, int B, long long P, int C, int G, int act, void *ws,
                                 size_t ws_bytes, void *stream) {
    if (!x || !gy || !stats || !ws || !(gx || ggamma || gbeta)) return DL_ERR_NULL;
    if (!dl_type_known(type) || !dl_type_known(ptype) || act < DL_ACT_NONE || act > DL_ACT_SIGMOID) return DL_ERR_UNSUPPORTED;
    if (!gn_shape_ok(B, P, C, G)) return DL_ERR_SHAPE;
    const int E = 16 / dl_type_bytes(type);
    const GnBackwardPlan plan = gn_backward_plan(B, P, C, G, E);
    if (ws_bytes < plan.bytes) return DL_ERR_WORKSPACE;
    hipStream_t st = (hipStream_t)stream;
    const GnShape &s = plan.s;
    const int threads = plan.threads;
    float *channel = (float *)((char *)ws + plan.channel), *part = (float *)((char *)ws + plan.part);
    float2 *group = (float2 *)((char *)ws + plan.group);
    if (threads) {
        if (!gn_grid_ok(s, threads)) return DL_ERR_UNSUPPORTED;
        const bool vec = gn_vectors(s, E, x, gy, gx);
        const bool few = s.samples > 1 || P <= gn_rows_per_step(s, E, threads);
        dl_prof_begin("gn_backward_one", st);
#define ONE(VEC, NV, THREADS) \
    gn_backward_one<T, VEC, NV, THREADS, ACT><<<plan.rows * s.tiles, THREADS, 0, st>>>((const T *)x, (const T *)gy, gamma, beta, ptype, \
                                                                                 (const float2 *)stats, channel, (T *)gx, ggamma, gbeta, s)
        DL_BY_TYPE(type, T, GN_BY_ACT(act, ACT, if (threads == GN_THREADS) {
                if (few) { if (vec) ONE(true, 1, GN_THREADS); else ONE(false, 1, GN_THREADS); }
                else { if (vec) ONE(true, 4, GN_THREADS); else ONE(false, 4, GN_THREADS); }
            }
                                      else { if (vec) ONE(true, GN_ONE_BACKWARD(16 / sizeof(T)), GN_ONE_THREADS); else ONE(false, GN_ONE_BACKWARD(16 / sizeof(T)), GN_ONE_THREADS); }));
#undef ONE
        dl_prof_end(st);
    } else {
        if (!gn_pieces_grid_ok(s)) return DL_ERR_UNSUPPORTED;
        const bool vec = gn_vectors(s, E, x, gy, gx);
        const int blocks = B * s.tiles * s.pieces;
#define BACKWARD(VEC)                                                                                                            \
    GN_BY_ACT(act, ACT, DL_TIMED("gn_backward_sums", st, (gn_backward_sums<T, VEC, GN_THREADS, ACT><<<blocks, GN_THREADS, 0, st>>>( \
        (const T *)x, (const T *)gy, gamma, beta, ptype, (const float2 *)stats, part, s))));                                      \
    DL_TIMED("gn_backward_join", st, (gn_backward_join<<<B * G, 256, 0, st>>>(part, gamma, ptype, s.pieces > 1 ? channel : nullptr, group, s))); \
    if (gx)                                                                                                                       \
        GN_BY_ACT(act, ACT, DL_TIMED("gn_backward_apply", st, (gn_backward_apply<T, VEC, GN_THREADS, ACT><<<blocks, GN_THREADS, 0, st>>>( \
            (const T *)x, (const T *)gy, gamma, beta, ptype, (const float2 *)stats, (const float2 *)group, (T *)gx, s))))
        DL_BY_TYPE(type, T, if (vec) { BACKWARD(true); } else { BACKWARD(false); });
#undef BACKWARD
    }
    if ((ggamma || gbeta) && !(threads && plan.rows == 1)) {
        int n = plan.rows;
        const float *rows = threads || s.pieces > 1 ? channel : part;
        const auto blocks = [&](int shares) {  // of all channels, each of every shares' rows; the blocks go on where there are more than a launch takes
            const long long all = (long long)dl_ceil_div(C, 32) * shares;
            return (int)(all < GN_PARAM_BLOCKS ? all : GN_PARAM_BLOCKS);
        };
        if (plan.shares) {
            float *sums = (float *)((char *)ws + plan.share_sums);
            DL_TIMED("gn_param_grads", st, (gn_param_grads<<<blocks(plan.shares), 256, 0, st>>>(rows, sums, nullptr, nullptr, ptype, n, C, plan.share, plan.shares)));
            n = plan.shares, rows = sums;
        }
        DL_TIMED("gn_param_grads", st, (gn_param_grads<<<blocks(1), 256, 0, st>>>(rows, nullptr, ggamma, gbeta, ptype, n, C, n, 1)));
    }
    return dl_launch_status();
}
