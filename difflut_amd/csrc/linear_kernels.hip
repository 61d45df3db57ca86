// Entry points of the matrix products, their plans, and the gradient in front of the backward's products (linear.h has the mathematics and
// the product kernel).
#include <math.h>

#include "linear.h"

// ------------------------------------------------------------------ operands whose rows are not whole units, or lie far apart
// src [rows][n], ld apart -> dst [rows][padded], zeros from n on; padded is a multiple of 16 bytes
template <typename T>
__global__ __launch_bounds__(256) void lin_pad(const T *__restrict__ src, long long ld, T *__restrict__ dst, long long rows, long long n,
                                               long long padded) {
    constexpr int E = 16 / sizeof(T);
    const long long units = rows * (padded / E);
    for (long long u = (long long)blockIdx.x * 256 + threadIdx.x; u < units; u += (long long)gridDim.x * 256) {
        const long long r = u / (padded / E), c = u % (padded / E) * E;
        DlVec<T, E> out;
#pragma unroll
        for (int i = 0; i < E; ++i) out.v[i] = c + i < n ? src[r * ld + c + i] : (T)0;
        *reinterpret_cast<DlVec<T, E> *>(dst + r * padded + c) = out;
    }
}

// ------------------------------------------------------------------ the gradient in front of the products, and its column sums
// gz [M, ldg] (null: not written) from gy and z as it was kept (null: no activation, gz is gy), and a share of sum_m gz per block of rows (null: not
// asked for).  A thread takes E columns of every fourth row of its block's; gated: of the gate and of the other half.  Rows of gz are whole units of
// 16 bytes, zeros behind the N-th column, as the products read them; those of gy may begin anywhere and end inside a unit (ODD).  Memory bounds it:
// 12544 x 8192 of a gate in bf16, 616 MB, 134 us, 4.6 TB/s.
#define LIN_SLOPE_ROWS 64
struct LinKept {
    const void *high;
    const uint8_t *low;
    long long ld;
    int half;
};
template <typename T, int E>
__device__ __forceinline__ void lin_kept(const LinKept &k, long long at, float (&f)[E]) {
    if constexpr (sizeof(T) == 4) dl_load<float, E>((const float *)k.high + at, f);
    else {
        const DlVec<uint16_t, E> high = *reinterpret_cast<const DlVec<uint16_t, E> *>((const uint16_t *)k.high + at);
        const DlVec<uint8_t, E> low = *reinterpret_cast<const DlVec<uint8_t, E> *>(k.low + at);
#pragma unroll
        for (int i = 0; i < E; ++i) f[i] = __uint_as_float((uint32_t)high.v[i] << 16 | (uint32_t)low.v[i] << 8);
    }
}
template <typename T, bool GATED, bool ODD>
__global__ __launch_bounds__(256) void lin_gradient(const T *__restrict__ gy, LinKept kept, T *__restrict__ gz, float *__restrict__ shares, long long M, int N,
                                                    long long ldg, int act, int col_tiles, int rows) {
    constexpr int H = GATED ? 2 : 1, E = 16 / sizeof(T);
    __shared__ float part[H * 4][64 * E];
    const int lane = threadIdx.x & 63, team = threadIdx.x >> 6, width = GATED ? N / 2 : N;
    const int c = ((int)(blockIdx.x % col_tiles) * 64 + lane) * E, n = width - c;
    const long long piece = blockIdx.x / col_tiles, m0 = piece * rows, m1 = m0 + rows < M ? m0 + rows : M;
    float sum[H][E];
#pragma unroll
    for (int h = 0; h < H; ++h)
#pragma unroll
        for (int i = 0; i < E; ++i) sum[h][i] = 0.0f;
    if (n > 0)
        for (long long m = m0 + team; m < m1; m += 4) {
            float g[H][E];
            if (ODD) dl_load_some<T, E>(gy + m * width + c, n, g[0]);
            else dl_load<T, E>(gy + m * width + c, g[0]);
            if (kept.high) {
                float a[H][E];
                lin_kept<T, E>(kept, m * kept.ld + c, a[0]);
                if (GATED) lin_kept<T, E>(kept, m * kept.ld + kept.half + c, a[H - 1]);
#pragma unroll
                for (int i = 0; i < E; ++i) {
                    float value;
                    const float slope = lin_slope(a[0][i], act, value), gi = g[0][i];
                    g[0][i] = GATED ? gi * a[H - 1][i] * slope : gi * slope;
                    if (GATED) g[H - 1][i] = gi * value;
                }
            }
#pragma unroll
            for (int h = 0; h < H; ++h) {
                if (gz && ODD) dl_store_some<T, E>(gz + m * ldg + h * width + c, n, g[h]);
                if (gz && !ODD) dl_store<T, E>(gz + m * ldg + h * width + c, g[h]);
#pragma unroll
                for (int i = 0; i < E; ++i) sum[h][i] += g[h][i];
            }
            if (ODD && gz && c == 0)
                for (int i = N; i < ldg; ++i) gz[m * ldg + i] = (T)0.0f;
        }
    if (!shares) return;
#pragma unroll
    for (int h = 0; h < H; ++h)
#pragma unroll
        for (int i = 0; i < E; ++i) part[h * 4 + team][i * 64 + lane] = sum[h][i];
    __syncthreads();
    if (team != 0) return;
#pragma unroll
    for (int h = 0; h < H; ++h)
#pragma unroll
        for (int i = 0; i < E; ++i) {
            if (i >= n) continue;
            float t = 0.0f;
            for (int q = 0; q < 4; ++q) t += part[h * 4 + q][i * 64 + lane];
            shares[piece * N + h * width + c + i] = t;
        }
}
// the shares of 16 columns per block, each column by 64 threads one after the other, then theirs  (784 shares of 1024 columns: 9.2 us by 16 threads, so
// 4.9)
template <typename T>
__global__ __launch_bounds__(1024) void lin_columns(const float *__restrict__ shares, T *__restrict__ out, int count, int N) {
    const int column = (int)blockIdx.x * 16 + (threadIdx.x & 15);
    const float t = dl_column_sum(shares, count, N, column);
    if (threadIdx.x < 16 && column < N) out[column] = (T)t;
}

// ------------------------------------------------------------------ plans
#define LIN_MOST ((1LL << 31) - 65536)
#define LIN_MOST_ROW ((long long)DL_LINEAR_ROW)  // bytes of an operand's row: what a tile and a stage read lies within 2^32 of its beginning

static int lin_size(int type) { return type == DL_E4M3 ? 1 : type == DL_F32 ? 4 : 2; }

// An operand of a product: R rows of C along K, or (turned) K rows along R.  `rows` of `length` values lie in memory.
struct LinOperand {
    const void *p;
    long long ld, rows, length;
    bool turned;
    bool padded = false;  // rows go on to a whole unit, with zeros
    long long count() const { return turned ? length : rows; }
};
static bool lin_direct(const LinOperand &o, int type) {
    const int size = lin_size(type);
    return dl_aligned16(o.p) && o.ld * size % 16 == 0 && o.ld * size <= LIN_MOST_ROW && (o.padded || o.length * size % 16 == 0);
}
static long long lin_padded(const LinOperand &o, int type) { const int unit = 16 / lin_size(type); return (o.length + unit - 1) / unit * unit; }
static size_t lin_operand_bytes(const LinOperand &o, int type) {
    return lin_direct(o, type) ? 0 : dl_align256((size_t)o.rows * (size_t)lin_padded(o, type) * lin_size(type));
}
// Tile and split: the least of an estimate over both tiles and the splits that leave a part four stages.  A stage takes a block of 256 x 256
// 1.55 us, the two blocks of 128 x 128 that share a CU 0.95, one that has it alone 0.6 (float32: three times that); a tile's beginning and end
// take 5 and 3 us; sums are written and read at 4 bytes/ps, with 4 us for the launch that joins them.  (bf16, 8192^3: 256 787 us, 128 970; 1024 x 4096 over
// 12544, us with the join: 256 in 4 parts 98, 128 in 2 parts 104, 256 whole 360.  The join's share is set too high: that of two parts is 9.7 us and
// counted as 20.8, so that here the estimate, 118 and 117, takes the second.)
static LinPlan lin_plan(const LinOperand &a, const LinOperand &b, int type, long long K, bool gated) {
    LinPlan p;
    const long long R = a.count(), C = b.count(), stages = (K * lin_size(type) + LIN_STAGE_BYTES - 1) / LIN_STAGE_BYTES;
    p.a_bytes = lin_operand_bytes(a, type), p.b_bytes = lin_operand_bytes(b, type), p.part_bytes = 0;
    p.few = !a.turned && !b.turned && lin_few_rows(R, C, K, lin_size(type), gated);
    if (p.few) {
        p.a_bytes = p.b_bytes = 0, p.tile = 0, p.splits = p.chunk = 1;
        return p;
    }
    double best = 1e30;
    for (int tile = 128; tile <= 256; tile += 128) {
        const double tiles = (double)((R + tile - 1) / tile) * (double)((C + tile - 1) / tile), slots = tile == 256 ? LIN_CUS : 2 * LIN_CUS;
        for (int splits = 1; splits <= 64; splits += splits < 4 ? 1 : splits / 2) {
            if (splits > 1 && (stages / splits < 4 || tiles * (splits - 1) >= slots)) break;
            const long long chunk = (stages + splits - 1) / splits;
            const double stage = (type == DL_F32 ? 3.0 : 1.0) * (tile == 256 ? 1.55 : tiles * splits <= LIN_CUS ? 0.6 : 0.95), rounds = ceil(tiles * splits / slots);
            const double us = rounds * ((double)chunk * stage + (tile == 256 ? 5.0 : 3.0)) + (splits > 1 ? 4.0 + 8.0 * splits * (double)R * (double)C / 4e6 : 0.0);
            if (us < best) best = us, p.tile = tile, p.splits = (int)((stages + chunk - 1) / chunk), p.chunk = (int)chunk;  // (no part is without a stage)
        }
    }
    p.part_bytes = p.splits > 1 ? dl_align256((size_t)p.splits * (size_t)R * (size_t)C * 4) : 0;
    return p;
}

template <typename T>
static void lin_pad_as(const LinOperand &o, void *dst, long long padded, hipStream_t s) {
    const long long blocks = (o.rows * (padded * (long long)sizeof(T) / 16) + 255) / 256;
    DL_TIMED("lin_pad", s, hipLaunchKernelGGL((lin_pad<T>), dim3((unsigned)(blocks < 16384 ? blocks : 16384)), dim3(256), 0, s, (const T *)o.p, o.ld, (T *)dst, o.rows, o.length, padded));
}
// the operand as the product reads it, and its row stride in bytes
static const char *lin_lay_out(const LinOperand &o, int type, void *room, long long &ld, hipStream_t s) {
    if (lin_direct(o, type)) {
        ld = o.ld * lin_size(type);
        return (const char *)o.p;
    }
    const long long padded = lin_padded(o, type);
    ld = padded * lin_size(type);
    if (type == DL_F32) lin_pad_as<float>(o, room, padded, s);
    else if (type == DL_E4M3) lin_pad_as<uint8_t>(o, room, padded, s);
    else lin_pad_as<uint16_t>(o, room, padded, s);
    return (const char *)room;
}

// One product: operands laid out, tiles, what follows
static int lin_run(const LinOperand &a, const LinOperand &b, int type, int out_type, long long K, bool gated, LinEnd end, char *ws, hipStream_t s) {
    LinPlan p = lin_plan(a, b, type, K, gated);
    LinArgs g{};
    if (p.few) g.A = (const char *)a.p, g.lda = a.ld * lin_size(type), g.B = (const char *)b.p, g.ldb = b.ld * lin_size(type);
    else g.A = lin_lay_out(a, type, ws, g.lda, s), g.B = lin_lay_out(b, type, ws + p.a_bytes, g.ldb, s);
    g.part = (float *)(ws + p.a_bytes + p.b_bytes);
    end.R = (int)a.count(), end.C = (int)b.count(), end.F = end.C / 2;
    const int width = gated ? end.F : end.C, size = dl_type_bytes(out_type);
    end.vec = width % 8 == 0 && dl_aligned16(end.y) && dl_aligned16(end.bias) && dl_aligned16(end.res) && dl_aligned16(end.col_scale) && end.ldr * size % 16 == 0;
    g.K = K, g.stages = dl_ceil_div(K * lin_size(type), LIN_STAGE_BYTES), g.chunk = p.chunk, g.splits = p.splits;
    if (!p.few) g.row_tiles = dl_ceil_div(end.R, p.tile), g.col_tiles = gated && p.splits == 1 ? dl_ceil_div(end.F, p.tile / 2) : dl_ceil_div(end.C, p.tile);
    g.end = end;
    int code = DL_ERR_UNSUPPORTED;
    if (type == DL_E4M3) code = lin_launch_e4m3(g, p, out_type, gated, s);
    else if (type == DL_F32) code = lin_launch_f32(g, p, a.turned, b.turned, gated, s);
    else if (type == DL_BF16) code = lin_launch_bf16(g, p, a.turned, b.turned, gated, s);
    else code = lin_launch_f16(g, p, a.turned, b.turned, gated, s);
    return code != DL_OK ? code : dl_launch_status();
}

static int lin_check(int type, int out_type, long long M, long long N, long long K, int act, int gated) {
    if (M <= 0 || N <= 0 || K <= 0 || M >= LIN_MOST || N >= LIN_MOST || K >= LIN_MOST) return DL_ERR_SHAPE;
    if (gated && N % 2 != 0) return DL_ERR_SHAPE;
    if (!(dl_type_known(type) ? out_type == type : type == DL_E4M3 && dl_type_known(out_type))) return DL_ERR_UNSUPPORTED;
    if (act < DL_ACT_NONE || act > DL_ACT_SIGMOID) return DL_ERR_UNSUPPORTED;
    if (K * lin_size(type) > LIN_MOST_ROW) return DL_ERR_UNSUPPORTED;
    return DL_OK;
}

extern "C" size_t dl_linear_fwd_workspace_bytes(const void *x, long long ldx, const void *w, long long ldw, int type, long long M, long long N, long long K,
                                                int gated) {
    if (lin_check(type, type == DL_E4M3 ? DL_F32 : type, M, N, K, 0, gated) != DL_OK) return 0;
    return lin_plan({x, ldx, M, K, false}, {w, ldw, N, K, false}, type, K, gated != 0).bytes();
}

// what is kept for the backward: rows of whole sixteens (gated: of both halves), of 16-bit types in two planes
static void lin_keep_in(LinEnd &end, void *kept, int type, long long M, long long N, bool gated) {
    end.half = (int)((N / 2 + 15) / 16 * 16), end.ldk = gated ? 2LL * end.half : (N + 15) / 16 * 16, end.kept = kept;
    end.kept_low = kept && type != DL_F32 ? (uint8_t *)kept + dl_align256((size_t)M * end.ldk * 2) : nullptr;
}
extern "C" size_t dl_linear_kept_bytes(int type, long long M, long long N, int gated) {
    if (lin_check(type, type, M, N, 1, 0, gated) != DL_OK || !dl_type_known(type)) return 0;
    LinEnd end{};
    lin_keep_in(end, nullptr, type, M, N, gated != 0);
    return type == DL_F32 ? (size_t)M * end.ldk * 4 : dl_align256((size_t)M * end.ldk * 2) + (size_t)M * end.ldk;
}

extern "C" int dl_linear_fwd(const void *x, long long ldx, const float *x_scale, const void *w, long long ldw, const float *w_scale, const void *bias,
                             const void *residual, long long ldr, void *y, void *kept, int type, int out_type, long long M, long long N, long long K, int act,
                             int gated, void *ws, size_t ws_bytes, void *stream) {
    if (!x || !w || !y || ((x_scale || w_scale) != (type == DL_E4M3)) || (type == DL_E4M3 && (!x_scale || !w_scale))) return DL_ERR_NULL;
    const int bad = lin_check(type, out_type, M, N, K, act, gated);
    if (bad) return bad;
    if (ldx < K || ldw < K || (residual && ldr < (gated ? N / 2 : N))) return DL_ERR_SHAPE;
    if (kept && (type == DL_E4M3 || N * lin_size(type) > LIN_MOST_ROW)) return DL_ERR_UNSUPPORTED;  // (such rows have no backward)
    if (!dl_aligned16(kept)) return DL_ERR_WORKSPACE;
    const size_t need = dl_linear_fwd_workspace_bytes(x, ldx, w, ldw, type, M, N, K, gated);
    if (need && !ws) return DL_ERR_NULL;
    if (ws_bytes < need || (need && !dl_aligned16(ws))) return DL_ERR_WORKSPACE;
    LinEnd end{};
    end.y = y, end.bias = bias, end.res = residual, end.ldr = residual ? ldr : 0, end.row_scale = x_scale, end.col_scale = w_scale, end.act = act;
    if (kept) lin_keep_in(end, kept, type, M, N, gated != 0);
    return lin_run({x, ldx, M, K, false}, {w, ldw, N, K, false}, type, out_type, K, gated != 0, end, (char *)ws, (hipStream_t)stream);
}

// ------------------------------------------------------------------ backward
struct LinBack {
    size_t gz, shares, products;
    int pieces, rows;
    size_t bytes() const { return gz + shares + products; }
};
static LinBack lin_back(const LinOperand &gz, const LinOperand &x, const LinOperand &w, int type, bool kept, int wants, long long N, long long K) {
    LinBack b{};
    const long long M = gz.rows;
    b.gz = kept ? dl_align256((size_t)M * (size_t)gz.ld * lin_size(type)) : 0;
    // rows of a block: from one a team up, as few as leave 1024 blocks or fewer over the columns (vectors of 16 bytes)
    const long long across = (N + 64 * (16 / lin_size(type)) - 1) / (64 * (16 / lin_size(type)));
    b.rows = 4;
    while ((M + b.rows - 1) / b.rows * across > 1024 && (b.rows < LIN_SLOPE_ROWS || (M + b.rows - 1) / b.rows > 1024)) b.rows *= 2;
    b.pieces = dl_ceil_div(M, b.rows);
    b.shares = wants & 4 ? dl_align256((size_t)b.pieces * (size_t)N * 4) : 0;
    const LinOperand gt = {gz.p, gz.ld, M, N, true, gz.padded}, wt = {w.p, w.ld, N, K, true}, xt = {x.p, x.ld, M, K, true};
    if (wants & 1) b.products = lin_plan(gz, wt, type, N, false).bytes();
    if (wants & 2) {
        const size_t n = lin_plan(gt, xt, type, M, false).bytes();
        if (n > b.products) b.products = n;
    }
    return b;
}
// gz: gy itself, or in the workspace's beginning (on 16 bytes: any pointer of that alignment stands for it) in rows of whole units
static LinOperand lin_gz(const void *ws, const void *gy, bool kept, int type, long long M, long long N) {
    if (!kept) return {gy, N, M, N, false};
    const long long unit = 16 / lin_size(type);
    return {ws ? ws : (const void *)256, (N + unit - 1) / unit * unit, M, N, false, true};
}

extern "C" size_t dl_linear_bwd_workspace_bytes(const void *x, long long ldx, const void *w, long long ldw, const void *kept, const void *gy, int wants, int type,
                                                long long M, long long N, long long K) {
    if (lin_check(type, type, M, N, K, 0, 0) != DL_OK) return 0;
    return lin_back(lin_gz(nullptr, gy, kept != nullptr, type, M, N), {x, ldx, M, K, false}, {w, ldw, N, K, false}, type, kept != nullptr, wants, N, K).bytes();
}

extern "C" int dl_linear_bwd(const void *x, long long ldx, const void *w, long long ldw, const void *keeping, const void *gy, void *gx, void *gw, void *gb, int type,
                             long long M, long long N, long long K, int act, int gated, void *ws, size_t ws_bytes, void *stream) {
    if (!gy || (gx && !w) || (gw && !x) || ((gated || act != DL_ACT_NONE) && !keeping)) return DL_ERR_NULL;
    const int bad = lin_check(type, type, M, N, K, act, gated);
    if (bad) return bad;
    if (N * lin_size(type) > LIN_MOST_ROW) return DL_ERR_UNSUPPORTED;
    if ((gx && ldw < K) || (gw && ldx < K)) return DL_ERR_SHAPE;
    const int wants = (gx ? 1 : 0) | (gw ? 2 : 0) | (gb ? 4 : 0);
    if (!wants) return DL_OK;
    if (!dl_aligned16(keeping)) return DL_ERR_WORKSPACE;
    const bool kept = keeping != nullptr;
    const LinOperand gz = lin_gz(ws, gy, kept, type, M, N), xo = {x, ldx, M, K, false}, wo = {w, ldw, N, K, false};
    const LinBack p = lin_back(gz, xo, wo, type, kept, wants, N, K);
    if (p.bytes() && !ws) return DL_ERR_NULL;
    if (ws_bytes < p.bytes() || !dl_aligned16(ws)) return DL_ERR_WORKSPACE;
    const hipStream_t s = (hipStream_t)stream;
    float *shares = gb ? (float *)((char *)ws + p.gz) : nullptr;
    if (kept || gb) {
        void *out = kept ? ws : nullptr;
        const int width = (int)(gated ? N / 2 : N);
        LinKept factors{};
        if (kept) {
            LinEnd layout{};
            lin_keep_in(layout, const_cast<void *>(keeping), type, M, N, gated != 0);
            factors = {keeping, layout.kept_low, layout.ldk, layout.half};
        }
#define LIN_GRADIENT(GATED, ODD) hipLaunchKernelGGL((lin_gradient<T, GATED, ODD>), dim3((unsigned)blocks), dim3(256), 0, s, (const T *)gy, factors, (T *)out, shares, M, (int)N, gz.ld, act, col_tiles, p.rows)
        DL_BY_TYPE(type, T, {
            const int col_tiles = dl_ceil_div(width, 64 * (16 / (int)sizeof(T)));
            const long long blocks = (long long)col_tiles * p.pieces;
            if (!dl_grid_ok(blocks, 256)) return DL_ERR_UNSUPPORTED;
            const bool odd = width % (16 / (int)sizeof(T)) != 0 || !dl_aligned16(gy);
            DL_TIMED("lin_gradient", s, if (gated) { if (odd) LIN_GRADIENT(true, true); else LIN_GRADIENT(true, false); }
                     else if (odd) LIN_GRADIENT(false, true); else LIN_GRADIENT(false, false));
            if (gb) DL_TIMED("lin_columns", s, hipLaunchKernelGGL((lin_columns<T>), dim3(dl_ceil_div(N, 16)), dim3(1024), 0, s, shares, (T *)gb, p.pieces, (int)N));
        });
#undef LIN_GRADIENT
    }
    char *room = (char *)ws + p.gz + p.shares;
    LinEnd end{};
    if (gx) {
        end.y = gx;
        const int code = lin_run(gz, {w, ldw, N, K, true}, type, type, N, false, end, room, s);
        if (code != DL_OK) return code;
    }
    if (gw) {
        end.y = gw;
        const int code = lin_run({gz.p, gz.ld, M, N, true, gz.padded}, {x, ldx, M, K, true}, type, type, M, false, end, room, s);
        if (code != DL_OK) return code;
    }
    return dl_launch_status();
}
