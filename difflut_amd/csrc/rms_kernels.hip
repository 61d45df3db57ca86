// Root-mean-square norm over the last dimension with the residual's addition in front of it, forward and backward, and rows in 8 bits.
//
//   h = x + residual (rounded to their type: the stream that is handed on),  rstd = 1 / sqrt(mean(h^2) + eps),  y_c = h_c rstd gamma_c
//   codes: scale = max |y| / 448 per row, code_c = e4m3(y_c / scale)  (448: the type's largest value)
//   backward, g = gy gamma, hat = h rstd:   gh = rstd (g - hat mean(g hat)) + (gradient that reached h itself),   ggamma_c = sum gy hat
//
// A team of 8 to 1024 threads takes a row and holds it in registers, V vectors of 16 bytes a thread, so that every tensor is read once
// and written once; rows that 1024 threads cannot hold so (16384 values of float32, 32768 of 16 bits) are read again instead, from the L2.  The backward's teams go
// through rows in steps and keep their columns' sums of ggamma in registers: a share per block, added up in order by one more launch.
// Sums are floats in a fixed order: the same bits from run to run.  Memory bounds all of it: 65521 x 1024 bf16 with a residual, forward 86 us and
// backward 112 (537 MB each, 6.2 and 4.8 TB/s), in 8 bits 87 (470 MB, 5.4 TB/s).
#include "dl_types.h"

#define RMS_THREADS 256
#define RMS_SHARES 1024           // shares of ggamma at most
#define RMS_CODE_MAX 448.0f       // largest e4m3 value
#define RMS_CODE_SMALL 0x1p-100f  // scales below it are brought up before they are divided by

typedef uint8_t rms_code;

template <int TEAM>
struct RmsTeam {
    static constexpr int THREADS = TEAM > RMS_THREADS ? TEAM : RMS_THREADS;
    static constexpr int TEAMS = THREADS / TEAM;
};

// Sum or maximum over a team, in a fixed order; every thread gets it.  `part`: a word per wavefront, of a call of its own.
template <int TEAM, bool MAX>
__device__ __forceinline__ float rms_reduce(float v, float *part) {
#pragma unroll
    for (int o = (TEAM < 64 ? TEAM : 64) / 2; o > 0; o >>= 1) {
        const float w = __shfl_xor(v, o);
        v = MAX ? (w > v || w != w ? w : v) : v + w;  // (a NaN stays)
    }
    if (TEAM > 64) {
        const int wave = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0) part[wave] = v;
        __syncthreads();
        const int first = (wave / (TEAM / 64)) * (TEAM / 64);
        v = part[first];
#pragma unroll
        for (int i = 1; i < TEAM / 64; ++i) {
            const float w = part[first + i];
            v = MAX ? (w > v || w != w ? w : v) : v + w;
        }
    }
    return v;
}

// E values of a row, `left` of them there and at any alignment (ODD), or all and aligned
template <bool ODD, typename T, int E>
__device__ __forceinline__ void rms_load(const T *p, int left, float (&f)[E]) {
    if constexpr (ODD) dl_load_some<T, E>(p, left, f);
    else dl_load<T, E>(p, f);
}
template <bool ODD, typename T, int E>
__device__ __forceinline__ void rms_store(T *p, int left, const float (&f)[E]) {
    if constexpr (ODD) dl_store_some<T, E>(p, left, f);
    else dl_store<T, E>(p, f);
}
template <bool ODD, int E>
__device__ __forceinline__ void rms_gammas(const void *p, int type, int c, int left, float (&f)[E]) {
#pragma unroll
    for (int i = 0; i < E; ++i) f[i] = 1.0f;
    if (!p) return;
    DL_BY_TYPE(type, T, (rms_load<ODD, T, E>((const T *)p + c, left, f)));
}

// values as e4m3, rounded to nearest even
template <bool ODD, int E>
__device__ __forceinline__ void rms_store_codes(rms_code *p, int left, const float (&f)[E]) {
    DlVec<uint32_t, E / 4> w;
#pragma unroll
    for (int i = 0; i < E / 4; ++i) {
        const int t = __builtin_amdgcn_cvt_pk_fp8_f32(f[4 * i], f[4 * i + 1], 0, false);
        w.v[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(f[4 * i + 2], f[4 * i + 3], t, true);
    }
    if (!ODD) *reinterpret_cast<DlVec<uint32_t, E / 4> *>(p) = w;
    else if (left >= E) __builtin_memcpy(p, &w, E);
    else
#pragma unroll
        for (int i = 0; i < E; ++i)
            if (i < left) p[i] = (rms_code)(w.v[i / 4] >> (i % 4 * 8));
}
__device__ __forceinline__ float rms_clamped(float v) { return v > RMS_CODE_MAX ? RMS_CODE_MAX : v < -RMS_CODE_MAX ? -RMS_CODE_MAX : v; }

struct RmsArgs {
    const void *x, *res, *gamma, *gy, *gh;
    void *h, *y, *gx;
    float *rstd, *scale, *shares;
    long long rows, ldx, ldr;
    int D, ptype, plain;  // plain: no norm, x itself (rows to 8 bits)
    float eps;
};

// CODES: y is bytes, and the rows' scales are written.  HELD: the row stays in registers (V vectors of E a thread).  ODD: rows begin anywhere and may
// end inside a vector.
template <typename T, int E, int V, int TEAM, bool CODES, bool HELD, bool ODD>
__global__ __launch_bounds__(RmsTeam<TEAM>::THREADS) void rms_fwd(RmsArgs g) {
    constexpr int TEAMS = RmsTeam<TEAM>::TEAMS, THREADS = RmsTeam<TEAM>::THREADS, UNROLL = HELD ? V : 1;
    __shared__ float part[2][THREADS / 64];
    const int lane = threadIdx.x % TEAM;
    const long long row_ = (long long)blockIdx.x * TEAMS + threadIdx.x / TEAM;
    const bool real = row_ < g.rows;
    const long long row = real ? row_ : g.rows - 1;  // teams without a row go along (there are barriers)
    const T *x = (const T *)g.x + row * g.ldx, *res = g.res ? (const T *)g.res + row * g.ldr : nullptr;
    T *h = g.h ? (T *)g.h + row * g.D : nullptr;
    const int turns = HELD ? V : (g.D + TEAM * E - 1) / (TEAM * E);
    float v[HELD ? V : 1][E], sum = 0.0f, big = 0.0f;

    auto fetch = [&](int j, float (&f)[E]) __attribute__((always_inline)) {
        const int c = (j * TEAM + lane) * E;
#pragma unroll
        for (int i = 0; i < E; ++i) f[i] = 0.0f;
        if (c >= g.D) return;
        rms_load<ODD, T, E>(x + c, g.D - c, f);
        if (res) {
            float r[E];
            rms_load<ODD, T, E>(res + c, g.D - c, r);
#pragma unroll
            for (int i = 0; i < E; ++i) f[i] = (float)(T)(f[i] + r[i]);
        }
    };
#pragma unroll UNROLL
    for (int j = 0; j < turns; ++j) {
        float(&f)[E] = v[HELD ? j : 0];
        fetch(j, f);
        const int c = (j * TEAM + lane) * E;
        if (h && real && c < g.D) rms_store<ODD, T, E>(h + c, g.D - c, f);
#pragma unroll
        for (int i = 0; i < E; ++i) sum = fmaf(f[i], f[i], sum);
    }
    float rstd = 1.0f;
    if (!g.plain) {
        sum = rms_reduce<TEAM, false>(sum, part[0]);
        rstd = 1.0f / sqrtf(sum / (float)g.D + g.eps);
        if (g.rstd && lane == 0 && real) g.rstd[row] = rstd;
    }
#pragma unroll UNROLL
    for (int j = 0; j < turns; ++j) {
        const int c = (j * TEAM + lane) * E;
        float(&f)[E] = v[HELD ? j : 0];
        if (!HELD) fetch(j, f);
        if (c >= g.D) continue;
        float w[E];
        rms_gammas<ODD, E>(g.gamma, g.ptype, c, g.D - c, w);
#pragma unroll
        for (int i = 0; i < E; ++i) {
            f[i] = f[i] * rstd * w[i];
            const float a = fabsf(f[i]);
            if (CODES) big = a > big || a != a ? a : big;
        }
        if (!CODES && real) rms_store<ODD, T, E>((T *)g.y + row * g.D + c, g.D - c, f);
    }
    if (!CODES) return;
    big = rms_reduce<TEAM, true>(big, part[1]);
    const float scale = big / RMS_CODE_MAX, up = scale < RMS_CODE_SMALL ? 0x1p64f : 1.0f;  // (exact; a scale below 2^-128 has no reciprocal)
    const float factor = scale > 0.0f || scale != scale ? 1.0f / (scale * up) : 0.0f;      // a row of zeros: codes and scale 0
    if (!real) return;
    if (lane == 0) g.scale[row] = scale;
#pragma unroll UNROLL
    for (int j = 0; j < turns; ++j) {
        const int c = (j * TEAM + lane) * E;
        float(&f)[E] = v[HELD ? j : 0];
        if (c >= g.D) continue;
        if (!HELD) {
            float w[E];
            fetch(j, f);
            rms_gammas<ODD, E>(g.gamma, g.ptype, c, g.D - c, w);
#pragma unroll
            for (int i = 0; i < E; ++i) f[i] = f[i] * rstd * w[i];
        }
#pragma unroll
        for (int i = 0; i < E; ++i) f[i] = rms_clamped(f[i] * up * factor);
        rms_store_codes<ODD, E>((rms_code *)g.y + row * g.D + c, g.D - c, f);
    }
}

// shares [gridDim.x][D] of ggamma (null: not asked for), in the order of rows, then teams
template <typename T, int E, int V, int TEAM, bool HELD, bool ODD>
__global__ __launch_bounds__(RmsTeam<TEAM>::THREADS) void rms_bwd(RmsArgs g) {
    constexpr int TEAMS = RmsTeam<TEAM>::TEAMS, THREADS = RmsTeam<TEAM>::THREADS, UNROLL = HELD ? V : 1;
    __shared__ float part[2][THREADS / 64];
    __shared__ float sums[HELD && TEAMS > 1 ? TEAMS * TEAM * E : 1];
    const int lane = threadIdx.x % TEAM, team = threadIdx.x / TEAM;
    float gg[HELD ? V : 1][E];
#pragma unroll
    for (int j = 0; j < (HELD ? V : 1); ++j)
#pragma unroll
        for (int i = 0; i < E; ++i) gg[j][i] = 0.0f;
    const int turns = HELD ? V : (g.D + TEAM * E - 1) / (TEAM * E);
    float *share = g.shares ? g.shares + (long long)blockIdx.x * g.D : nullptr;
    if (!HELD && share) {
        for (int c = lane; c < g.D; c += TEAM) share[c] = 0.0f;
        __syncthreads();
    }
    const long long step = (long long)gridDim.x * TEAMS;
    int turn = 0;
    for (long long first = (long long)blockIdx.x * TEAMS; first < g.rows; first += step, turn ^= 1) {
        const bool real = first + team < g.rows;
        const long long row = real ? first + team : g.rows - 1;
        const T *h = (const T *)g.x + row * g.ldx, *gy = g.gy ? (const T *)g.gy + row * g.D : nullptr;
        const float rstd = g.rstd[row];
        float a[HELD ? V : 1][E], b[HELD ? V : 1][E], dot = 0.0f;  // hat and g
        auto fetch = [&](int j, float (&hat)[E], float (&gw)[E], bool sum) __attribute__((always_inline)) {
            const int c = (j * TEAM + lane) * E;
#pragma unroll
            for (int i = 0; i < E; ++i) hat[i] = gw[i] = 0.0f;
            if (c >= g.D) return;
            float w[E];
            rms_load<ODD, T, E>(h + c, g.D - c, hat);
            if (gy) rms_load<ODD, T, E>(gy + c, g.D - c, gw);
            rms_gammas<ODD, E>(g.gamma, g.ptype, c, g.D - c, w);
#pragma unroll
            for (int i = 0; i < E; ++i) {
                hat[i] *= rstd;
                if (sum && real) {
                    if (HELD) gg[HELD ? j : 0][i] = fmaf(gw[i], hat[i], gg[HELD ? j : 0][i]);
                    else if (share && c + i < g.D) share[c + i] = fmaf(gw[i], hat[i], share[c + i]);
                }
                gw[i] *= w[i];
                if (sum) dot = fmaf(gw[i], hat[i], dot);
            }
        };
#pragma unroll UNROLL
        for (int j = 0; j < turns; ++j) fetch(j, a[HELD ? j : 0], b[HELD ? j : 0], true);
        if (!g.gx) continue;
        const float mean = rms_reduce<TEAM, false>(dot, part[turn]) / (float)g.D;
#pragma unroll UNROLL
        for (int j = 0; j < turns; ++j) {
            const int c = (j * TEAM + lane) * E;
            float(&hat)[E] = a[HELD ? j : 0], (&gw)[E] = b[HELD ? j : 0];
            if (!HELD) fetch(j, hat, gw, false);
            if (c >= g.D || !real) continue;
            float r[E];
#pragma unroll
            for (int i = 0; i < E; ++i) r[i] = 0.0f;
            if (g.gh) rms_load<ODD, T, E>((const T *)g.gh + row * g.D + c, g.D - c, r);
#pragma unroll
            for (int i = 0; i < E; ++i) r[i] = fmaf(rstd, gw[i] - hat[i] * mean, r[i]);
            rms_store<ODD, T, E>((T *)g.gx + row * g.D + c, g.D - c, r);
        }
    }
    if (!HELD || !share) return;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int c = (j * TEAM + lane) * E;
        if (TEAMS == 1) {
            if (c < g.D) rms_store<ODD, float, E>(share + c, g.D - c, gg[HELD ? j : 0]);
            continue;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < E; ++i) sums[TEAMS > 1 ? (team * E + i) * TEAM + lane : 0] = gg[HELD ? j : 0][i];
        __syncthreads();
        for (int e = threadIdx.x; e < TEAM * E; e += THREADS) {
            const int column = (j * TEAM + e % TEAM) * E + e / TEAM;
            float t = 0.0f;
            for (int k = 0; k < TEAMS; ++k) t += sums[TEAMS > 1 ? k * E * TEAM + e : 0];
            if (column < g.D) share[column] = t;
        }
    }
}

// ggamma: the shares of 16 columns per block, each column by 64 threads one after the other, then theirs  (1024 shares of 1024 columns: 21 us by 16
// threads, so 5.1)
__global__ __launch_bounds__(1024) void rms_join(const float *__restrict__ shares, void *__restrict__ out, int ptype, int count, int D) {
    const int column = (int)blockIdx.x * 16 + (threadIdx.x & 15);
    const float t = dl_column_sum(shares, count, D, column);
    if (threadIdx.x >= 16 || column >= D) return;
    if (ptype == DL_F32) ((float *)out)[column] = t;
    else if (ptype == DL_BF16) ((dl_bf16 *)out)[column] = (dl_bf16)t;
    else ((dl_f16 *)out)[column] = (dl_f16)t;
}

// ------------------------------------------------------------------ which form
// The smallest team that holds a row in up to 4 vectors a thread (8 threads, a wavefront, 256 threads, 1024 threads); -1: none does.
static int rms_team(int D, int e) { return D <= 8 * 4 * e ? 8 : D <= 64 * 4 * e ? 64 : D <= 256 * 4 * e ? 256 : D <= 1024 * 4 * e ? 1024 : -1; }
static int rms_team_rows(int team) { return team < 0 || team > RMS_THREADS ? 1 : RMS_THREADS / team; }

// whether rows begin off a vector of 16 bytes, or end inside one
static bool rms_odd(const RmsArgs &g, int type, int out_bytes) {
    const int size = dl_type_bytes(type), e = 16 / size;
    const int psize = g.gamma ? dl_type_bytes(g.ptype) : 2;
    const auto fits = [&](const void *p, int width) { return ((uintptr_t)p & (uintptr_t)(width * e < 16 ? width * e - 1 : 15)) == 0; };
    const bool fine = g.D % e == 0 && g.ldx % e == 0 && g.ldr % e == 0 && fits(g.x, size) && fits(g.res, size) && fits(g.h, size) &&
                      fits(g.gy, size) && fits(g.gh, size) && fits(g.gx, size) && fits(g.y, out_bytes) && fits(g.gamma, psize);
    // (gamma of float next to 16-bit rows: two loads of 16 bytes)
    return !fine;
}

template <typename T, bool CODES, bool ODD>
static void rms_launch_fwd(const RmsArgs &g, hipStream_t s) {
    constexpr int E = 16 / sizeof(T);
    const int team = rms_team(g.D, E);
    const long long blocks = (g.rows + rms_team_rows(team) - 1) / rms_team_rows(team);
    const int vectors = team > 0 ? (g.D + team * E - 1) / (team * E) : 0;
#define RMS_FWD(TEAM, V, HELD) hipLaunchKernelGGL((rms_fwd<T, E, V, TEAM, CODES, HELD, ODD>), dim3((unsigned)blocks), dim3(RmsTeam<TEAM>::THREADS), 0, s, g)
#define RMS_FWD_V(TEAM) \
    do { if (vectors <= 1) RMS_FWD(TEAM, 1, true); else if (vectors <= 2) RMS_FWD(TEAM, 2, true); else RMS_FWD(TEAM, 4, true); } while (0)
    DL_TIMED("rms_fwd", s, if (team == 8) RMS_FWD_V(8); else if (team == 64) RMS_FWD_V(64); else if (team == 256) RMS_FWD_V(256);
             else if (team == 1024) RMS_FWD_V(1024); else RMS_FWD(1024, 1, false));
#undef RMS_FWD_V
#undef RMS_FWD
}
template <typename T, bool ODD>
static void rms_launch_bwd(const RmsArgs &g, int blocks, hipStream_t s) {
    constexpr int E = 16 / sizeof(T);
    const int team = rms_team(g.D, E), vectors = team > 0 ? (g.D + team * E - 1) / (team * E) : 0;
#define RMS_BWD(TEAM, V, HELD) hipLaunchKernelGGL((rms_bwd<T, E, V, TEAM, HELD, ODD>), dim3((unsigned)blocks), dim3(RmsTeam<TEAM>::THREADS), 0, s, g)
#define RMS_BWD_V(TEAM) \
    do { if (vectors <= 1) RMS_BWD(TEAM, 1, true); else if (vectors <= 2) RMS_BWD(TEAM, 2, true); else RMS_BWD(TEAM, 4, true); } while (0)
    DL_TIMED("rms_bwd", s, if (team == 8) RMS_BWD_V(8); else if (team == 64) RMS_BWD_V(64); else if (team == 256) RMS_BWD_V(256);
             else if (team == 1024) RMS_BWD_V(1024); else RMS_BWD(1024, 1, false));
#undef RMS_BWD_V
#undef RMS_BWD
}

// blocks of the backward: as many as have rows, up to RMS_SHARES 
static long long rms_bwd_blocks(long long rows, int team) {
    const long long need = (rows + rms_team_rows(team) - 1) / rms_team_rows(team);
    return need < RMS_SHARES ? need : RMS_SHARES;
}

static int rms_check(int type, int ptype, const void *gamma, long long rows, int D) {
    if (rows <= 0 || D <= 0 || rows >= (1LL << 31) - 65536 || D >= (1LL << 31) - 65536) return DL_ERR_SHAPE;
    if (!dl_type_known(type) || (gamma && !dl_type_known(ptype))) return DL_ERR_UNSUPPORTED;
    return DL_OK;
}
// a launch has a block per row or fewer
static bool rms_grid_fits(long long rows, int D, int e) {
    const int team = rms_team(D, e), per = rms_team_rows(team);
    return dl_grid_ok((rows + per - 1) / per, team < 0 || team > RMS_THREADS ? 1024 : RMS_THREADS);
}

extern "C" int dl_rms_norm_fwd(const void *x, long long ldx, const void *residual, long long ldr, const void *gamma, void *h, void *y, float *rstd,
                               float *scale, int type, int ptype, long long rows, int D, float eps, void *stream) {
    if (!x || !y) return DL_ERR_NULL;
    if (residual && !h) return DL_ERR_NULL;
    const int bad = rms_check(type, ptype, gamma, rows, D);
    if (bad) return bad;
    if (ldx < D || (residual && ldr < D) || !(eps >= 0.0f)) return DL_ERR_SHAPE;
    RmsArgs g{};
    g.x = x, g.ldx = ldx, g.res = residual, g.ldr = residual ? ldr : 0, g.gamma = gamma, g.h = residual ? h : nullptr, g.y = y, g.rstd = rstd, g.scale = scale;
    g.rows = rows, g.D = D, g.ptype = ptype, g.eps = eps;
    const bool odd = rms_odd(g, type, scale ? 1 : dl_type_bytes(type));
    if (!rms_grid_fits(rows, D, 16 / dl_type_bytes(type))) return DL_ERR_UNSUPPORTED;
    const hipStream_t s = (hipStream_t)stream;
    DL_BY_TYPE(type, T, {
        if (scale) { if (odd) rms_launch_fwd<T, true, true>(g, s); else rms_launch_fwd<T, true, false>(g, s); }
        else if (odd) rms_launch_fwd<T, false, true>(g, s);
        else rms_launch_fwd<T, false, false>(g, s);
    });
    return dl_launch_status();
}

extern "C" int dl_quantize_rows(const void *x, long long ldx, void *codes, float *scale, int type, long long rows, int D, void *stream) {
    if (!x || !codes || !scale) return DL_ERR_NULL;
    const int bad = rms_check(type, 0, nullptr, rows, D);
    if (bad) return bad;
    if (ldx < D) return DL_ERR_SHAPE;
    RmsArgs g{};
    g.x = x, g.ldx = ldx, g.y = codes, g.scale = scale, g.rows = rows, g.D = D, g.plain = 1;
    const bool odd = rms_odd(g, type, 1);
    if (!rms_grid_fits(rows, D, 16 / dl_type_bytes(type))) return DL_ERR_UNSUPPORTED;
    const hipStream_t s = (hipStream_t)stream;
    DL_BY_TYPE(type, T, {
        if (odd) rms_launch_fwd<T, true, true>(g, s); else rms_launch_fwd<T, true, false>(g, s);
    });
    return dl_launch_status();
}

extern "C" size_t dl_rms_norm_bwd_workspace_bytes(long long rows, int D) {
    if (rows <= 0 || D <= 0) return 0;
    return dl_align256((size_t)(rows < RMS_SHARES ? rows : RMS_SHARES) * (size_t)D * 4);
}

extern "C" int dl_rms_norm_bwd(const void *h, long long ldh, const void *gamma, const float *rstd, const void *gy, const void *gh, void *gx, void *ggamma,
                               int type, int ptype, long long rows, int D, void *ws, size_t ws_bytes, void *stream) {
    if (!h || !rstd || (!gy && !gh)) return DL_ERR_NULL;
    if (ggamma && (!gamma || !ws)) return DL_ERR_NULL;
    const int bad = rms_check(type, ptype, gamma, rows, D);
    if (bad) return bad;
    if (ldh < D) return DL_ERR_SHAPE;
    if (ggamma && ws_bytes < dl_rms_norm_bwd_workspace_bytes(rows, D)) return DL_ERR_WORKSPACE;
    if (!gx && !ggamma) return DL_OK;
    RmsArgs g{};
    g.x = h, g.ldx = ldh, g.gamma = gamma, g.rstd = const_cast<float *>(rstd), g.gy = gy, g.gh = gh, g.gx = gx, g.shares = ggamma ? (float *)ws : nullptr;
    g.rows = rows, g.D = D, g.ptype = ptype;
    const bool odd = rms_odd(g, type, dl_type_bytes(type));
    const int blocks = (int)rms_bwd_blocks(rows, rms_team(D, 16 / dl_type_bytes(type)));
    const hipStream_t s = (hipStream_t)stream;
    DL_BY_TYPE(type, T, {
        if (odd) rms_launch_bwd<T, true>(g, blocks, s); else rms_launch_bwd<T, false>(g, blocks, s);
    });
    if (ggamma) DL_TIMED("rms_join", s, hipLaunchKernelGGL(rms_join, dim3(dl_ceil_div(D, 16)), dim3(1024), 0, s, (const float *)ws, ggamma, ptype, blocks, D));
    return dl_launch_status();
}
