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
#include "dl_types.h"

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
};

__device__ __forceinline__ float gn_sigmoid(float z) { return 1.0f / (1.0f + __expf(-z)); }
__device__ __forceinline__ float gn_act(int act, float z) {
    if (act == GN_RELU) return z > 0.0f || z != z ? z : 0.0f;
    if (act == GN_SILU) return z * gn_sigmoid(z);
    if (act == GN_SIGMOID) return gn_sigmoid(z);
    return z;
}
__device__ __forceinline__ float gn_slope(int act, float z) {
    if (act == GN_RELU) return z > 0.0f ? 1.0f : 0.0f;
    if (act == GN_NONE) return 1.0f;
    const float s = gn_sigmoid(z);
    return act == GN_SILU ? s * (1.0f + z * (1.0f - s)) : s * (1.0f - s);
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
    int col, row0, rows;                // column of vectors, first position, positions per step
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
    w.c = c0 + w.col * E;
    w.p_begin = (long long)piece * s.piece_rows;
    w.p_end = min(w.p_begin + s.piece_rows, s.P);
    return w;
}
template <typename T, int E, bool VEC>
__device__ __forceinline__ void gn_read(const T *p, int real, float (&f)[E]) {
    if constexpr (VEC) {
        dl_load(p, f);
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) f[e] = e < real ? (float)p[e] : 0.0f;
    }
}
template <typename T, int E, bool VEC>
__device__ __forceinline__ void gn_write(T *p, int real, const float (&f)[E]) {
    if constexpr (VEC) {
        dl_store(p, f);
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (e < real) p[e] = (T)f[e];
    }
}

// Sums of the tile's groups: every thread brings one value per channel, sums[g] (in LDS) are the groups' totals.  slots: LDS of
// threads * E floats.
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
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    for (int g = wave; g < w.groups; g += THREADS / 64) {
        float t = 0.0f;
        for (int j = lane; j < w.rows * per_group; j += 64) t += slots[(j / per_group) * per_row + g * per_group + j % per_group];
        t = gn_wave_sum(t);
        if (lane == 0) sums[g] = t;
    }
    __syncthreads();
}

// ---------------------------------------------------------------------------------- forward
// Statistics of a piece: mean and sum of squares about it per group, [B][G][slices * pieces] (mean, M2).  The piece stays in
// registers between the two sums.  ONE: the piece is the whole sample, so the block goes on to write y.
template <typename T, int E, bool VEC, int NV, int THREADS, bool ONE>
__global__ __launch_bounds__(THREADS) void gn_forward(const T *__restrict__ x, const void *__restrict__ gamma,
                                                       const void *__restrict__ beta, int ptype, T *__restrict__ y,
                                                       float2 *__restrict__ stats, float2 *__restrict__ part, GnShape s, float eps, int act) {
    __shared__ float slots[THREADS * E];
    __shared__ float sums[THREADS * E], mean[THREADS * E];
    const int tile = blockIdx.x % s.tiles, piece = blockIdx.x / s.tiles % s.pieces, b = blockIdx.x / s.tiles / s.pieces;
    const GnPlace w = gn_place<E>(s, tile, piece, THREADS);
    const int real = w.c_end - w.c;
    float v[NV][E];
    float t[E] = {};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const long long p = w.p_begin + w.row0 + (long long)i * w.rows;
        if (w.active && p < w.p_end) gn_read<T, E, VEC>(x + ((long long)b * s.P + p) * s.C + w.c, real, v[i]);
        else
#pragma unroll
            for (int e = 0; e < E; ++e) v[i][e] = 0.0f;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < E; ++e) t[e] += v[i][e];
    gn_group_sums<E, THREADS>(s, w, t, slots, sums);
    const int c0 = w.c - w.col * E;
    const float n = (float)(w.p_end - w.p_begin) * (float)(s.tile_groups ? s.cg : w.c_end - c0);
    for (int g = threadIdx.x; g < w.groups; g += THREADS) mean[g] = sums[g] / n;
    __syncthreads();
    int group[E];
    float m[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        group[e] = s.tile_groups && w.active && e < real ? (w.c + e - c0) / s.cg : 0;
        m[e] = mean[group[e]];
        t[e] = 0.0f;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const long long p = w.p_begin + w.row0 + (long long)i * w.rows;
        if (!w.active || p >= w.p_end) continue;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float d = e < real ? v[i][e] - m[e] : 0.0f;
            t[e] += d * d;
        }
    }
    gn_group_sums<E, THREADS>(s, w, t, slots, sums);
    if (!ONE) {
        const int slice = s.tile_groups ? 0 : tile % s.slices;
        for (int g = threadIdx.x; g < w.groups; g += THREADS)
            part[((long long)b * s.G + w.first_group + g) * (s.slices * s.pieces) + (long long)piece * s.slices + slice] = make_float2(mean[g], sums[g]);
        return;
    }
    for (int g = threadIdx.x; g < w.groups; g += THREADS) {
        const float rstd = 1.0f / sqrtf(sums[g] / n + eps);
        sums[g] = rstd;
        if (stats) stats[(long long)b * s.G + w.first_group + g] = make_float2(mean[g], rstd);
    }
    __syncthreads();
    if (!w.active) return;
    float ga[E], be[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        ga[e] = e < real ? gn_param(gamma, ptype, w.c + e, 1.0f) : 0.0f;
        be[e] = e < real ? gn_param(beta, ptype, w.c + e, 0.0f) : 0.0f;
        t[e] = sums[group[e]];
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const long long p = w.p_begin + w.row0 + (long long)i * w.rows;
        if (p >= w.p_end) continue;
        float o[E];
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = gn_act(act, (v[i][e] - m[e]) * t[e] * ga[e] + be[e]);
        gn_write<T, E, VEC>(y + ((long long)b * s.P + p) * s.C + w.c, real, o);
    }
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
template <typename T, int E, bool VEC, int THREADS>
__global__ __launch_bounds__(THREADS) void gn_apply(const T *__restrict__ x, const void *__restrict__ gamma, const void *__restrict__ beta,
                                                     int ptype, T *__restrict__ y, const float2 *__restrict__ stats, GnShape s, int act) {
    const int tile = blockIdx.x % s.tiles, piece = blockIdx.x / s.tiles % s.pieces, b = blockIdx.x / s.tiles / s.pieces;
    const GnPlace w = gn_place<E>(s, tile, piece, THREADS);
    if (!w.active) return;
    const int real = w.c_end - w.c;
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
    for (long long p = w.p_begin + w.row0; p < w.p_end; p += w.rows) {
        const long long at = ((long long)b * s.P + p) * s.C + w.c;
        float v[E];
        gn_read<T, E, VEC>(x + at, real, v);
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = gn_act(act, (v[e] - mean[e]) * scale[e] + shift[e]);
        gn_write<T, E, VEC>(y + at, real, v);
    }
}

// ---------------------------------------------------------------------------------- backward
// Per channel of a piece: sum g and sum g xhat, [B][pieces][2][C].
template <typename T, int E, bool VEC, int THREADS>
__global__ __launch_bounds__(THREADS) void gn_backward_sums(const T *__restrict__ x, const T *__restrict__ gy, const void *__restrict__ gamma,
                                                             const void *__restrict__ beta, int ptype, const float2 *__restrict__ stats,
                                                             float *__restrict__ part, GnShape s, int act) {
    __shared__ float slots[2][THREADS * E];
    const int tile = blockIdx.x % s.tiles, piece = blockIdx.x / s.tiles % s.pieces, b = blockIdx.x / s.tiles / s.pieces;
    const GnPlace w = gn_place<E>(s, tile, piece, THREADS);
    const int real = w.c_end - w.c;
    float sg[E] = {}, sx[E] = {};
    if (w.active) {
        float mean[E], rstd[E], ga[E], be[E];
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int c = min(w.c + e, s.C - 1);
            const float2 st = stats[(long long)b * s.G + c / s.cg];
            mean[e] = st.x, rstd[e] = st.y;
            ga[e] = gn_param(gamma, ptype, c, 1.0f), be[e] = gn_param(beta, ptype, c, 0.0f);
        }
#pragma unroll 2
        for (long long p = w.p_begin + w.row0; p < w.p_end; p += w.rows) {
            const long long at = ((long long)b * s.P + p) * s.C + w.c;
            float v[E], g[E];
            gn_read<T, E, VEC>(x + at, real, v);
            gn_read<T, E, VEC>(gy + at, real, g);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float hat = (v[e] - mean[e]) * rstd[e], d = g[e] * gn_slope(act, hat * ga[e] + be[e]);
                sg[e] += d;
                sx[e] += d * hat;
            }
        }
    }
    const int vectors = (w.c_end - (w.c - w.col * E) + E - 1) / E;
#pragma unroll
    for (int e = 0; e < E; ++e) slots[0][threadIdx.x * E + e] = w.active ? sg[e] : 0.0f, slots[1][threadIdx.x * E + e] = w.active ? sx[e] : 0.0f;
    __syncthreads();
    // column sums over the rows of threads, in order
    const int c0 = w.c - w.col * E, width = w.c_end - c0;
    float *out = part + ((long long)b * s.pieces + piece) * 2 * s.C + c0;
    for (int j = threadIdx.x; j < 2 * width; j += THREADS) {
        const int which = j >= width, c = j - which * width;
        float t = 0.0f;
        for (int r = 0; r < w.rows; ++r) t += slots[which][r * vectors * E + c];
        out[(long long)which * s.C + c] = t;
    }
}

// Per sample: the channels' sums over its pieces ([B][2][C]) and, per group, mean(gamma g) and mean(gamma g xhat).
// One block per (sample, group).
__global__ __launch_bounds__(256) void gn_backward_join(const float *__restrict__ part, const void *__restrict__ gamma, int ptype,
                                                         float *__restrict__ channel, float2 *__restrict__ group, GnShape s) {
    __shared__ float red[2][4];
    const int g = blockIdx.x % s.G, b = blockIdx.x / s.G;
    float a = 0.0f, q = 0.0f;
    for (int c = g * s.cg + threadIdx.x; c < (g + 1) * s.cg; c += 256) {
        float sg = 0.0f, sx = 0.0f;
        for (int i = 0; i < s.pieces; ++i) {
            const float *row = part + ((long long)b * s.pieces + i) * 2 * s.C + c;
            sg += row[0];
            sx += row[s.C];
        }
        channel[(long long)b * 2 * s.C + c] = sg;
        channel[(long long)b * 2 * s.C + s.C + c] = sx;
        const float ga = gn_param(gamma, ptype, c, 1.0f);
        a += ga * sg;
        q += ga * sx;
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

template <typename T, int E, bool VEC, int THREADS>
__global__ __launch_bounds__(THREADS) void gn_backward_apply(const T *__restrict__ x, const T *__restrict__ gy, const void *__restrict__ gamma,
                                                              const void *__restrict__ beta, int ptype, const float2 *__restrict__ stats,
                                                              const float2 *__restrict__ group, T *__restrict__ gx, GnShape s, int act) {
    const int tile = blockIdx.x % s.tiles, piece = blockIdx.x / s.tiles % s.pieces, b = blockIdx.x / s.tiles / s.pieces;
    const GnPlace w = gn_place<E>(s, tile, piece, THREADS);
    if (!w.active) return;
    const int real = w.c_end - w.c;
    float mean[E], rstd[E], ga[E], be[E], ma[E], mq[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int c = min(w.c + e, s.C - 1);
        const float2 st = stats[(long long)b * s.G + c / s.cg], gr = group[(long long)b * s.G + c / s.cg];
        mean[e] = st.x, rstd[e] = st.y, ma[e] = gr.x, mq[e] = gr.y;
        ga[e] = gn_param(gamma, ptype, c, 1.0f), be[e] = gn_param(beta, ptype, c, 0.0f);
    }
#pragma unroll 2
    for (long long p = w.p_begin + w.row0; p < w.p_end; p += w.rows) {
        const long long at = ((long long)b * s.P + p) * s.C + w.c;
        float v[E], g[E];
        gn_read<T, E, VEC>(x + at, real, v);
        gn_read<T, E, VEC>(gy + at, real, g);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float hat = (v[e] - mean[e]) * rstd[e], d = g[e] * gn_slope(act, hat * ga[e] + be[e]);
            v[e] = rstd[e] * (d * ga[e] - ma[e] - hat * mq[e]);
        }
        gn_write<T, E, VEC>(gx + at, real, v);
    }
}

// ggamma_c = sum_b sum g xhat, gbeta_c = sum_b sum g: 32 channels x 8 samples a step per block, added in a fixed order.
__global__ __launch_bounds__(256) void gn_param_grads(const float *__restrict__ channel, void *__restrict__ ggamma, void *__restrict__ gbeta,
                                                       int ptype, int B, int C) {
    __shared__ float red[2][8][32];
    const int c = blockIdx.x * 32 + (threadIdx.x & 31), r = threadIdx.x >> 5;
    float sg = 0.0f, sx = 0.0f;
    if (c < C)
#pragma unroll 8
        for (int b = r; b < B; b += 8) {
            sg += channel[(long long)b * 2 * C + c];
            sx += channel[(long long)b * 2 * C + C + c];
        }
    red[0][r][threadIdx.x & 31] = sg, red[1][r][threadIdx.x & 31] = sx;
    __syncthreads();
    if (threadIdx.x >= 64) return;
    const int which = threadIdx.x >> 5, cc = blockIdx.x * 32 + (threadIdx.x & 31);
    if (cc >= C) return;
    float t = 0.0f;
    for (int i = 0; i < 8; ++i) t += red[which][i][threadIdx.x & 31];
    gn_param_store(which ? ggamma : gbeta, ptype, cc, t);
}

// ---------------------------------------------------------------------------------- host
static bool gn_shape_ok(int B, long long P, int C, int G) {
    return B > 0 && P > 0 && C > 0 && G > 0 && C % G == 0 && P < (1LL << 31) && (long long)B * G < (1LL << 31);
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
    s.pieces = 1;
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
#define GN_THREADS 256
#define GN_NV 8  // positions that a thread of the statistics kernel holds

static GnShape gn_stats_shape(int B, long long P, int C, int G, int E) {
    GnShape s = gn_tiles(B, P, C, G, E, GN_THREADS);
    s.piece_rows = gn_rows_per_step(s, E, GN_THREADS) * GN_NV;
    s.pieces = (int)((P + s.piece_rows - 1) / s.piece_rows);
    return s;
}
static GnShape gn_sums_shape(int B, long long P, int C, int G, int E) {
    GnShape s = gn_tiles(B, P, C, G, E, GN_THREADS);
    gn_pieces(s, gn_rows_per_step(s, E, GN_THREADS) * 4, 2048);
    return s;
}
static bool gn_grid_ok(const GnShape &s) { return (long long)s.B * s.tiles * s.pieces < (1LL << 31); }

extern "C" size_t dl_group_norm_fwd_workspace_bytes(int type, int B, long long P, int C, int G) {
    if (!dl_type_known(type) || !gn_shape_ok(B, P, C, G)) return 0;
    const GnShape s = gn_stats_shape(B, P, C, G, 16 / dl_type_bytes(type));
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
    const GnShape a = gn_stats_shape(B, P, C, G, E), b = gn_sums_shape(B, P, C, G, E);
    if (!gn_grid_ok(a) || !gn_grid_ok(b)) return DL_ERR_UNSUPPORTED;
    const bool vec = gn_vectors(a, E, x, y, nullptr);
    const int blocks_a = B * a.tiles * a.pieces, blocks_b = B * b.tiles * b.pieces;
#define FORWARD(VEC)                                                                                                                  \
    DL_TIMED("gn_forward", st, (gn_forward<T, 16 / sizeof(T), VEC, GN_NV, GN_THREADS, false><<<blocks_a, GN_THREADS, 0, st>>>(        \
        (const T *)x, gamma, beta, ptype, (T *)y, (float2 *)stats, (float2 *)ws, a, eps, act)));                                      \
    DL_TIMED("gn_join_stats", st, (gn_join_stats<<<dl_ceil_div((long long)B * G, 4), 256, 0, st>>>((const float2 *)ws, (float2 *)stats, a, eps))); \
    DL_TIMED("gn_apply", st, (gn_apply<T, 16 / sizeof(T), VEC, GN_THREADS><<<blocks_b, GN_THREADS, 0, st>>>(                          \
        (const T *)x, gamma, beta, ptype, (T *)y, (const float2 *)stats, b, act)))
    DL_BY_TYPE(type, T, if (vec) { FORWARD(true); } else { FORWARD(false); });
#undef FORWARD
    return dl_launch_status();
}

extern "C" size_t dl_group_norm_bwd_workspace_bytes(int type, int B, long long P, int C, int G) {
    if (!dl_type_known(type) || !gn_shape_ok(B, P, C, G)) return 0;
    const GnShape s = gn_sums_shape(B, P, C, G, 16 / dl_type_bytes(type));
    return dl_align256((size_t)B * s.pieces * 2 * C * sizeof(float)) + dl_align256((size_t)B * 2 * C * sizeof(float)) +
           dl_align256((size_t)B * G * sizeof(float2));
}

extern "C" int dl_group_norm_bwd(const void *x, const void *gy, const void *gamma, const void *beta, const float *stats, void *gx,
                                 void *ggamma, void *gbeta, int type, int ptype, int B, long long P, int C, int G, int act, void *ws,
                                 size_t ws_bytes, void *stream) {
    if (!x || !gy || !stats || !ws || !(gx || ggamma || gbeta)) return DL_ERR_NULL;
    if (!dl_type_known(type) || !dl_type_known(ptype) || act < DL_ACT_NONE || act > DL_ACT_SIGMOID) return DL_ERR_UNSUPPORTED;
    if (!gn_shape_ok(B, P, C, G)) return DL_ERR_SHAPE;
    if (ws_bytes < dl_group_norm_bwd_workspace_bytes(type, B, P, C, G)) return DL_ERR_WORKSPACE;
    hipStream_t st = (hipStream_t)stream;
    const int E = 16 / dl_type_bytes(type);
    const GnShape s = gn_sums_shape(B, P, C, G, E);
    if (!gn_grid_ok(s)) return DL_ERR_UNSUPPORTED;
    const bool vec = gn_vectors(s, E, x, gy, gx);
    float *part = (float *)ws;
    float *channel = (float *)((char *)part + dl_align256((size_t)B * s.pieces * 2 * C * sizeof(float)));
    float2 *group = (float2 *)((char *)channel + dl_align256((size_t)B * 2 * C * sizeof(float)));
    const int blocks = B * s.tiles * s.pieces;
#define BACKWARD(VEC)                                                                                                            \
    DL_TIMED("gn_backward_sums", st, (gn_backward_sums<T, 16 / sizeof(T), VEC, GN_THREADS><<<blocks, GN_THREADS, 0, st>>>(        \
        (const T *)x, (const T *)gy, gamma, beta, ptype, (const float2 *)stats, part, s, act)));                                  \
    DL_TIMED("gn_backward_join", st, (gn_backward_join<<<B * G, 256, 0, st>>>(part, gamma, ptype, channel, group, s)));           \
    if (gx)                                                                                                                       \
        DL_TIMED("gn_backward_apply", st, (gn_backward_apply<T, 16 / sizeof(T), VEC, GN_THREADS><<<blocks, GN_THREADS, 0, st>>>(  \
            (const T *)x, (const T *)gy, gamma, beta, ptype, (const float2 *)stats, group, (T *)gx, s, act)))
    DL_BY_TYPE(type, T, if (vec) { BACKWARD(true); } else { BACKWARD(false); });
#undef BACKWARD
    if (ggamma || gbeta)
        DL_TIMED("gn_param_grads", st, (gn_param_grads<<<dl_ceil_div(C, 32), 256, 0, st>>>(channel, ggamma, gbeta, ptype, B, C)));
    return dl_launch_status();
}
