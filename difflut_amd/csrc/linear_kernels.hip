// Matrix products with bias, activation, a gate and a residual in the same launch, and their backward pass, on the 16-bit and
// 8-bit matrix cores with fp32 accumulation.
//
//   linear    z[m,n] = sum_k x[m,k] w[n,k] + b[n],   y = act(z) + residual
//   gated     z over 2 F rows of w, gate first:      y[m,f] = act(z[m,f]) z[m,F+f]
//   backward  gz = gy act'(z)   (gated: gz[f] = gy z[F+f] act'(z[f]),  gz[F+f] = gy act(z[f])),  gb = sum_m gz,  gx = gz w,  gw = gz^T x
//
// One product kernel serves all of them: C[r,c] = sum_k A[r,k] B[c,k], both operands with the reduction along their rows of memory.
// Operands that are not laid out so (w for gx, gz and x for gw), whose rows do not start on 16 bytes or end inside 16, are laid out by
// a pass in front of it, reductions padded with zeros.
//
// float32 operands are cut into three bf16 planes (8 + 8 + 8 significant bits, each the rounding of what the ones above left) by that
// pass; a product is the six plane products hi*hi, hi*mid, mid*hi, mid*mid, hi*lo, lo*hi, small ones first, as six reductions in a
// row into the same sums.  What is left out is below 2^-26 of |a b|, less than the 2^-24 of one fp32 multiply-add.  Six bf16 products
// at 2.5 PFLOP/s are 417 TFLOP/s of fp32 work against 157 on the fp32 matrix cores.  (Planes carry no infinities: such a product
// is NaN where a value of finite sign would be infinite.)
#include "dl_types.h"

typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 halfx8 __attribute__((ext_vector_type(8)));
typedef int intx4 __attribute__((ext_vector_type(4)));
typedef int intx8 __attribute__((ext_vector_type(8)));

#define LIN_STAGE_BYTES 128  // of a row in a stage: 64 16-bit or 128 8-bit values
#define LIN_PLANES 3
#define LIN_COMBOS 6
#define LIN_CUS 256

struct LinBf16 { static constexpr int SIZE = 2; };
struct LinF16 { static constexpr int SIZE = 2; };
struct LinE4m3 { static constexpr int SIZE = 1; };

// (exponential and reciprocal as the hardware has them: an ulp each, and |z| u from the product with log2 e)
__device__ __forceinline__ float lin_sigmoid(float z) { return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * -1.44269504f)); }
__device__ __forceinline__ float lin_act(float z, int act) {
    if (act == DL_ACT_RELU) return z > 0.0f || z != z ? z : 0.0f;
    if (act == DL_ACT_SILU) return z * lin_sigmoid(z);
    if (act == DL_ACT_SIGMOID) return lin_sigmoid(z);
    return z;
}
// the activation's value and slope
__device__ __forceinline__ float lin_slope(float z, int act, float &value) {
    if (act == DL_ACT_RELU) {
        value = z > 0.0f || z != z ? z : 0.0f;
        return z > 0.0f ? 1.0f : 0.0f;
    }
    if (act == DL_ACT_NONE) {
        value = z;
        return 1.0f;
    }
    const float s = lin_sigmoid(z), r = fmaf(-s, s, s);
    value = act == DL_ACT_SILU ? z * s : s;
    return act == DL_ACT_SILU ? fmaf(z, r, s) : r;
}

// ------------------------------------------------------------------ operands laid out for the product
__device__ __forceinline__ uint16_t lin_bf16_bits(float v) { return __builtin_bit_cast(uint16_t, (dl_bf16)v); }
__device__ __forceinline__ float lin_of_bits(uint16_t v) { return __uint_as_float((uint32_t)v << 16); }
// the planes of a value; infinities and NaN are in the first alone
__device__ __forceinline__ void lin_planes(float v, uint16_t (&p)[LIN_PLANES]) {
    p[0] = lin_bf16_bits(v);
    const float rest = v - lin_of_bits(p[0]);
    const bool fine = fabsf(rest) < __builtin_inff();
    p[1] = fine ? lin_bf16_bits(rest) : 0;
    p[2] = fine ? lin_bf16_bits(rest - lin_of_bits(p[1])) : 0;
}

template <typename T>
struct LinCell { typedef T type; };
template <>
struct LinCell<float> { typedef uint16_t type; };

// src [R][K], rows ld apart -> dst [R][Kp] (planes of R * Kp for float), zeros from K on
template <typename T>
__global__ __launch_bounds__(256) void lin_pad(const T *__restrict__ src, long long ld, typename LinCell<T>::type *__restrict__ dst, long long R,
                                               long long K, long long Kp) {
    typedef typename LinCell<T>::type Cell;
    const long long units = R * (Kp / 8);
    for (long long u = (long long)blockIdx.x * 256 + threadIdx.x; u < units; u += (long long)gridDim.x * 256) {
        const long long r = u / (Kp / 8), k = u % (Kp / 8) * 8;
        T v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = k + i < K ? src[r * ld + k + i] : (T)0;
        if constexpr (__is_same(T, float)) {
            DlVec<Cell, 8> out[LIN_PLANES];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                uint16_t p[LIN_PLANES];
                lin_planes(v[i], p);
#pragma unroll
                for (int q = 0; q < LIN_PLANES; ++q) out[q].v[i] = p[q];
            }
#pragma unroll
            for (int q = 0; q < LIN_PLANES; ++q) *reinterpret_cast<DlVec<Cell, 8> *>(dst + q * R * Kp + r * Kp + k) = out[q];
        } else {
            DlVec<Cell, 8> out;
#pragma unroll
            for (int i = 0; i < 8; ++i) out.v[i] = v[i];
            *reinterpret_cast<DlVec<Cell, 8> *>(dst + r * Kp + k) = out;
        }
    }
}

// src [K][R], rows ld apart -> dst [R][Kp], zeros from K on: tiles of 64 x 64 turned in the LDS
template <typename T>
__global__ __launch_bounds__(256) void lin_turn(const T *__restrict__ src, long long ld, typename LinCell<T>::type *__restrict__ dst, long long R,
                                                long long K, long long Kp, int row_tiles) {
    typedef typename LinCell<T>::type Cell;
    __shared__ T tile[64][65];
    const long long r0 = (long long)(blockIdx.x % row_tiles) * 64, k0 = (long long)(blockIdx.x / row_tiles) * 64;
    const int c = threadIdx.x & 63;
#pragma unroll
    for (int q = 0; q < 16; ++q) {
        const int k = (threadIdx.x >> 6) + q * 4;
        tile[k][c] = k0 + k < K && r0 + c < R ? src[(k0 + k) * ld + r0 + c] : (T)0;
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        const int r = (threadIdx.x >> 3) + q * 32, k = (threadIdx.x & 7) * 8;
        if (r0 + r >= R) continue;
        const long long at = (r0 + r) * Kp + k0 + k;
        if constexpr (__is_same(T, float)) {
            DlVec<Cell, 8> out[LIN_PLANES];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                uint16_t p[LIN_PLANES];
                lin_planes(tile[k + i][r], p);
#pragma unroll
                for (int s = 0; s < LIN_PLANES; ++s) out[s].v[i] = p[s];
            }
#pragma unroll
            for (int s = 0; s < LIN_PLANES; ++s) *reinterpret_cast<DlVec<Cell, 8> *>(dst + s * R * Kp + at) = out[s];
        } else {
            DlVec<Cell, 8> out;
#pragma unroll
            for (int i = 0; i < 8; ++i) out.v[i] = tile[k + i][r];
            *reinterpret_cast<DlVec<Cell, 8> *>(dst + at) = out;
        }
    }
}

// ------------------------------------------------------------------ what follows a product
struct LinEnd {
    void *y, *z;                // z (null: not kept): what the activation is applied to, in y's type
    const void *bias, *res;
    const float *row_scale, *col_scale;  // of 8-bit operands
    long long ldr;
    int R, C, F, act;           // C: rows of w; F: columns of y where gated
    bool vec;                   // whole vectors of eight everywhere
};

// Eight columns from c on of row r, from their sums; those past the end are left out.  Gated: the columns are f's, u their other halves.
template <typename Out, bool GATED>
__device__ __forceinline__ void lin_finish(const LinEnd &g, int r, int c, float (&v)[8], float (&u)[8]) {
    const int width = GATED ? g.F : g.C;
    if (r >= g.R || c >= width) return;
    const long long ldz = g.C;
    const bool whole = g.vec;  // (width is a multiple of eight then)
    const float rs = g.row_scale ? g.row_scale[r] : 1.0f;
#pragma unroll
    for (int half = 0; half < (GATED ? 2 : 1); ++half) {
        float(&a)[8] = half ? u : v;
        const int at = half ? g.F + c : c;
        if (g.col_scale) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (whole || c + i < width) a[i] *= rs * g.col_scale[at + i];
        }
        if (g.bias) {
            if (whole) {
                float b[8];
                dl_load<Out, 8>((const Out *)g.bias + at, b);
#pragma unroll
                for (int i = 0; i < 8; ++i) a[i] += b[i];
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (c + i < width) a[i] += (float)((const Out *)g.bias)[at + i];
            }
        }
        if (g.z) {
            Out *z = (Out *)g.z + r * ldz + at;
            if (whole) dl_store<Out, 8>(z, a);
            else
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (c + i < width) z[i] = (Out)a[i];
        }
    }
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = lin_act(v[i], g.act) * (GATED ? u[i] : 1.0f);
    if (g.res) {
        const Out *res = (const Out *)g.res + r * g.ldr + c;
        if (whole) {
            float t[8];
            dl_load<Out, 8>(res, t);
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] += t[i];
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (c + i < width) y[i] += (float)res[i];
        }
    }
    Out *out = (Out *)g.y + (long long)r * width + c;
    if (whole) dl_store<Out, 8>(out, y);
    else
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (c + i < width) out[i] = (Out)y[i];
}

// ------------------------------------------------------------------ the product
struct LinArgs {
    const char *A, *B;
    long long lda, ldb, plane_a, plane_b;  // bytes
    int k_bytes;                           // of the reduction, a multiple of 16
    int stages, combos, chunk;             // stages of one reduction, reductions, stages of a block (all of them without PARTIAL)
    int row_tiles, col_tiles;
    float *part;                           // PARTIAL: sums [splits][R][C]
    LinEnd end;
};
__device__ const uint4 lin_zeros = {0, 0, 0, 0};  // what lies behind a reduction's end

// Loads that bypass the registers: lane l's 16 bytes land at LDS address lds + 16 l.  The compiler does not count them: a stage waits.
__device__ __forceinline__ void lin_to_lds(unsigned lds, const char *base, unsigned voff) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(voff), "s"(base) : "memory", "m0");
}
__device__ __forceinline__ void lin_to_lds_far(unsigned lds, const char *at) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds), "v"(at) : "memory", "m0");
}
// this wavefront's loads have landed, its LDS reads are done, and every wavefront has got here
__device__ __forceinline__ void lin_stage_barrier() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

template <typename In>
__device__ __forceinline__ floatx16 lin_mfma(const intx4 (&a)[2], const intx4 (&b)[2], floatx16 c) {
    if constexpr (__is_same(In, LinE4m3)) {
        const intx8 x = __builtin_shufflevector(a[0], a[1], 0, 1, 2, 3, 4, 5, 6, 7), y = __builtin_shufflevector(b[0], b[1], 0, 1, 2, 3, 4, 5, 6, 7);
        return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(x, y, c, 0, 0, 0, 0x7f7f7f7f, 0, 0x7f7f7f7f);  // block scales of 2^0
    } else if constexpr (__is_same(In, LinBf16)) {
        c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a[0]), __builtin_bit_cast(bf16x8, b[0]), c, 0, 0, 0);
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a[1]), __builtin_bit_cast(bf16x8, b[1]), c, 0, 0, 0);
    } else {
        c = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(halfx8, a[0]), __builtin_bit_cast(halfx8, b[0]), c, 0, 0, 0);
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(halfx8, a[1]), __builtin_bit_cast(halfx8, b[1]), c, 0, 0, 0);
    }
}

// A block makes a tile of TR x TC in stages of 128 bytes of every row, two in the LDS: while one is worked on the next one comes.
// A row's eight units of 16 bytes are kept in turned order (unit u in slot u ^ (row & 7)), so that the eight lanes of an LDS read
// that take the same unit of eight rows find them on different banks; the loads fetch in that order.
// A wavefront makes TR / WR rows by 64 columns; gated, these are 32 columns of the gate and the 32 that belong to them.
template <typename In, typename Out, int TR, int TC, int WR, int WC, bool GATED, bool PARTIAL>
__global__ __launch_bounds__(64 * WR * WC, 2) void lin_product(LinArgs g) {
    extern __shared__ __align__(16) char lds[];
    constexpr int WAVES = WR * WC, FA = TR / WR / 32, FB = 2, STAGE = (TR + TC) * LIN_STAGE_BYTES;
    constexpr int NA = TR / 8 / WAVES, NB = TC / 8 / WAVES;
    static_assert(TC == WC * 64 && TR == WR * FA * 32 && TR % (8 * WAVES) == 0 && TC % (8 * WAVES) == 0, "whole tiles");
    typedef __attribute__((address_space(3))) char lds_char;
    const unsigned lds_base = (unsigned)(uintptr_t)(lds_char *)lds;
    const int lane = threadIdx.x & 63, wave = dl_uniform(threadIdx.x >> 6);

    // tiles: every XCD takes a run of them, eight rows of tiles at a time, so that its L2 holds what neighbours share
    const int tiles = g.row_tiles * g.col_tiles, per = (tiles + DL_XCDS - 1) / DL_XCDS;
    const int split = blockIdx.x / (per * DL_XCDS), id = blockIdx.x % (per * DL_XCDS);
    const int tile = (id % DL_XCDS) * per + id / DL_XCDS;
    if (tile >= tiles) return;
    const int band = tile / (8 * g.col_tiles), in_band = tile % (8 * g.col_tiles), band_rows = min(8, g.row_tiles - band * 8);
    const int r0 = (band * 8 + in_band % band_rows) * TR, c_tile = in_band / band_rows;
    const int c0 = c_tile * (GATED ? TC / 2 : TC);

    const int first = split * g.chunk, count = min(g.combos * g.stages - first, g.chunk);

    // ---- what this lane fetches: row 8 p + lane / 8 of a load p, the unit that belongs into slot lane % 8
    const unsigned unit = ((lane & 7) ^ (lane >> 3)) * 16;
    unsigned a_off[NA], b_off[NB];
    const char *b_base[NB];
    const char *a_base = g.A + (long long)r0 * g.lda;
#pragma unroll
    for (int j = 0; j < NA; ++j) a_off[j] = (unsigned)(min(r0 + (wave + j * WAVES) * 8 + (lane >> 3), g.end.R - 1) - r0) * (unsigned)g.lda + unit;
#pragma unroll
    for (int j = 0; j < NB; ++j) {
        const int row = (wave + j * WAVES) * 8;  // of the tile, the lane's own row not counted
        if (GATED) {
            const int f = (row / 64) * 32 + row % 32;
            b_base[j] = g.B + ((long long)c0 + (row % 64 >= 32 ? g.end.F : 0)) * g.ldb;
            b_off[j] = (unsigned)(min(c0 + f + (lane >> 3), g.end.F - 1) - c0) * (unsigned)g.ldb + unit;
        } else {
            b_base[j] = g.B + (long long)c0 * g.ldb;
            b_off[j] = (unsigned)(min(c0 + row + (lane >> 3), g.end.C - 1) - c0) * (unsigned)g.ldb + unit;
        }
    }
    const bool ragged = g.k_bytes % LIN_STAGE_BYTES != 0;
    auto issue = [&](int st, int buf) __attribute__((always_inline)) {
        const int combo = g.combos > 1 ? st / g.stages : 0, k = (st - combo * g.stages) * LIN_STAGE_BYTES;
        // planes of the six products, a digit each from the lowest on: small ones first
        const int pa = g.combos > 1 ? (0x010120 >> 4 * combo) & 15 : 0, pb = g.combos > 1 ? (0x001102 >> 4 * combo) & 15 : 0;
        const long long at_a = pa * g.plane_a + k, at_b = pb * g.plane_b + k;
        const unsigned base = lds_base + buf * STAGE;
        if (ragged && k + LIN_STAGE_BYTES > g.k_bytes) {
            const bool real = k + (int)unit < g.k_bytes;
#pragma unroll
            for (int j = 0; j < NA; ++j)
                lin_to_lds_far(base + (wave + j * WAVES) * 1024, real ? a_base + at_a + a_off[j] : (const char *)&lin_zeros);
#pragma unroll
            for (int j = 0; j < NB; ++j)
                lin_to_lds_far(base + TR * LIN_STAGE_BYTES + (wave + j * WAVES) * 1024, real ? b_base[j] + at_b + b_off[j] : (const char *)&lin_zeros);
            return;
        }
#pragma unroll
        for (int j = 0; j < NA; ++j) lin_to_lds(base + (wave + j * WAVES) * 1024, a_base + at_a, a_off[j]);
#pragma unroll
        for (int j = 0; j < NB; ++j) lin_to_lds(base + TR * LIN_STAGE_BYTES + (wave + j * WAVES) * 1024, b_base[j] + at_b, b_off[j]);
    };

    floatx16 acc[FA][FB];
#pragma unroll
    for (int i = 0; i < FA; ++i)
#pragma unroll
        for (int j = 0; j < FB; ++j)
#pragma unroll
            for (int v = 0; v < 16; ++v) acc[i][j][v] = 0.0f;

    const int kh = lane >> 5, l32 = lane & 31, wr = wave / WC * (TR / WR), wc = wave % WC * 64;
    const unsigned a_rd = (wr + l32) * LIN_STAGE_BYTES, b_rd = (TR + wc + l32) * LIN_STAGE_BYTES;
    unsigned slot[2][2];  // of the two units that go into step kk
#pragma unroll
    for (int kk = 0; kk < 2; ++kk)
#pragma unroll
        for (int q = 0; q < 2; ++q) slot[kk][q] = ((4 * kk + 2 * q + kh) ^ (lane & 7)) * 16;
    auto compute = [&](int buf) __attribute__((always_inline)) {
        const char *at = lds + buf * STAGE;
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            intx4 a[FA][2], b[FB][2];
#pragma unroll
            for (int q = 0; q < 2; ++q) {
#pragma unroll
                for (int j = 0; j < FB; ++j) b[j][q] = *reinterpret_cast<const intx4 *>(at + b_rd + slot[kk][q] + j * 32 * LIN_STAGE_BYTES);
#pragma unroll
                for (int i = 0; i < FA; ++i) a[i][q] = *reinterpret_cast<const intx4 *>(at + a_rd + slot[kk][q] + i * 32 * LIN_STAGE_BYTES);
            }
#pragma unroll
            for (int i = 0; i < FA; ++i)
#pragma unroll
                for (int j = 0; j < FB; ++j) acc[i][j] = lin_mfma<In>(a[i], b[j], acc[i][j]);
        }
    };

    issue(first, 0);
    for (int s = 0; s < count; ++s) {
        lin_stage_barrier();  // stage s is there, and nobody reads the other buffer any more
        if (s + 1 < count) issue(first + s + 1, (s + 1) & 1);
        compute(s & 1);
    }

    // C: row (v % 4) + 8 (v / 4) + 4 (lane / 32) of a tile of 32 x 32, column lane % 32
    if (PARTIAL) {
        float *part = g.part + (long long)split * g.end.R * g.end.C;
#pragma unroll
        for (int i = 0; i < FA; ++i)
#pragma unroll
            for (int j = 0; j < FB; ++j)
#pragma unroll
                for (int v = 0; v < 16; ++v) {
                    const int r = r0 + wr + i * 32 + (v & 3) + 8 * (v >> 2) + 4 * kh, c = c0 + wc + j * 32 + l32;
                    if (r < g.end.R && c < g.end.C) part[(long long)r * g.end.C + c] = acc[i][j][v];
                }
        return;
    }
    // through the LDS, 32 rows at a time, every wavefront in a place of its own: a lane then has eight columns of a row
    constexpr int LD = 64 + 4;
    static_assert(WAVES * 32 * LD * 4 <= 2 * STAGE, "fits the stages");
    lin_stage_barrier();
    float *mine = reinterpret_cast<float *>(lds) + wave * 32 * LD;
#pragma unroll
    for (int i = 0; i < FA; ++i) {
#pragma unroll
        for (int j = 0; j < FB; ++j)
#pragma unroll
            for (int v = 0; v < 16; ++v) mine[((v & 3) + 8 * (v >> 2) + 4 * kh) * LD + j * 32 + l32] = acc[i][j][v];
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        constexpr int LANES = GATED ? 4 : 8, ROWS = 64 / LANES;  // lanes of a row, rows at a time
#pragma unroll
        for (int t = 0; t < 32 / ROWS; ++t) {
            const int row = t * ROWS + lane / LANES, col = lane % LANES * 8;
            float v[8], u[8];
            *reinterpret_cast<float4 *>(v) = *reinterpret_cast<const float4 *>(mine + row * LD + col);
            *reinterpret_cast<float4 *>(v + 4) = *reinterpret_cast<const float4 *>(mine + row * LD + col + 4);
            if (GATED) {
                *reinterpret_cast<float4 *>(u) = *reinterpret_cast<const float4 *>(mine + row * LD + 32 + col);
                *reinterpret_cast<float4 *>(u + 4) = *reinterpret_cast<const float4 *>(mine + row * LD + 32 + col + 4);
            }
            lin_finish<Out, GATED>(g.end, r0 + wr + i * 32 + row, c0 + (GATED ? wc / 2 : wc) + col, v, u);
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
}

// The sums of a reduction that was split, in order, and what follows
template <typename Out, bool GATED>
__global__ __launch_bounds__(256) void lin_join(LinArgs g, int splits) {
    const int width = GATED ? g.end.F : g.end.C, units = (width + 7) / 8;
    const long long total = (long long)g.end.R * units, plane = (long long)g.end.R * g.end.C;
    for (long long e = (long long)blockIdx.x * 256 + threadIdx.x; e < total; e += (long long)gridDim.x * 256) {
        const int r = (int)(e / units), c = (int)(e % units) * 8;
        float v[8], u[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = u[i] = 0.0f;
        const float *at = g.part + (long long)r * g.end.C + c;
        for (int s = 0; s < splits; ++s, at += plane) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (c + i >= width) continue;
                v[i] += at[i];
                if (GATED) u[i] += at[g.end.F + i];
            }
        }
        lin_finish<Out, GATED>(g.end, r, c, v, u);
    }
}

// ------------------------------------------------------------------ the gradient in front of the products, and its column sums
// gz [M, N] (null: not written) from gy and z (null: no activation, gz is gy), and a share of sum_m gz per block of rows (null: not asked for).
// A thread takes E columns of every fourth row of its block's; gated: of the gate and of the other half.
#define LIN_SLOPE_ROWS 64
template <typename T, int E, bool GATED>
__global__ __launch_bounds__(256) void lin_gradient(const T *__restrict__ gy, const T *__restrict__ z, T *__restrict__ gz, float *__restrict__ shares,
                                                    long long M, int N, int act, int col_tiles, int rows) {
    constexpr int H = GATED ? 2 : 1;
    __shared__ float part[H * 4][64 * E];
    const int lane = threadIdx.x & 63, team = threadIdx.x >> 6, width = GATED ? N / 2 : N;
    const int c = ((int)(blockIdx.x % col_tiles) * 64 + lane) * E;
    const long long piece = blockIdx.x / col_tiles, m0 = piece * rows, m1 = m0 + rows < M ? m0 + rows : M;
    float sum[H][E];
#pragma unroll
    for (int h = 0; h < H; ++h)
#pragma unroll
        for (int i = 0; i < E; ++i) sum[h][i] = 0.0f;
    if (c < width)
        for (long long m = m0 + team; m < m1; m += 4) {
            float g[H][E];
            dl_load<T, E>(gy + m * width + c, g[0]);
            if (z) {
                float a[H][E];
                dl_load<T, E>(z + m * N + c, a[0]);
                if (GATED) dl_load<T, E>(z + m * N + width + c, a[H - 1]);
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
                if (gz) dl_store<T, E>(gz + m * N + h * width + c, g[h]);
#pragma unroll
                for (int i = 0; i < E; ++i) sum[h][i] += g[h][i];
            }
        }
    if (!shares) return;
#pragma unroll
    for (int h = 0; h < H; ++h)
#pragma unroll
        for (int i = 0; i < E; ++i) part[h * 4 + team][i * 64 + lane] = sum[h][i];
    __syncthreads();
    if (team != 0 || c >= width) return;
#pragma unroll
    for (int h = 0; h < H; ++h)
#pragma unroll
        for (int i = 0; i < E; ++i) {
            float t = 0.0f;
            for (int q = 0; q < 4; ++q) t += part[h * 4 + q][i * 64 + lane];
            shares[piece * N + h * width + c + i] = t;
        }
}
// the shares of 16 columns per block, each column by 16 threads one after the other, then theirs
template <typename T>
__global__ __launch_bounds__(256) void lin_columns(const float *__restrict__ shares, T *__restrict__ out, int count, int N) {
    __shared__ float part[16][17];
    const int c = threadIdx.x & 15, k = threadIdx.x >> 4, column = (int)blockIdx.x * 16 + c;
    float t = 0.0f;
    if (column < N)
        for (int s = k; s < count; s += 16) t += shares[(long long)s * N + column];
    part[k][c] = t;
    __syncthreads();
    if (k != 0 || column >= N) return;
    for (int i = 1; i < 16; ++i) t += part[i][c];
    out[column] = (T)t;
}

// ------------------------------------------------------------------ plans
#define LIN_MOST ((1LL << 31) - 65536)
#define LIN_MOST_ROW (1LL << 23)  // bytes of an operand's row: a tile's 256 rows lie within 2^32 of each other

static int lin_size(int type) { return type == DL_E4M3 ? 1 : type == DL_F32 ? 4 : 2; }
static long long lin_padded(int type, long long K) { const int step = type == DL_E4M3 ? 128 : 64; return (K + step - 1) / step * step; }

// An operand of a product: R rows along K, or (turned) K rows along R
struct LinOperand {
    const void *p;
    long long ld, R;
    bool turned;
};
static bool lin_direct(const LinOperand &o, int type, long long K) {
    const int size = lin_size(type);
    return type != DL_F32 && !o.turned && dl_aligned16(o.p) && o.ld * size % 16 == 0 && K * size % 16 == 0;
}
static size_t lin_operand_bytes(const LinOperand &o, int type, long long K) {
    if (lin_direct(o, type, K)) return 0;
    return dl_align256((size_t)o.R * (size_t)lin_padded(type, K) * (type == DL_E4M3 ? 1 : 2) * (type == DL_F32 ? LIN_PLANES : 1));
}
struct LinPlan {
    int tile, splits, chunk;  // 256 or 128; parts of the reduction, and their stages
    size_t a_bytes, b_bytes, part_bytes;
    size_t bytes() const { return a_bytes + b_bytes + part_bytes; }
};
// Tile and split.
static LinPlan lin_plan(const LinOperand &a, const LinOperand &b, int type, long long K) {
    LinPlan p;
    p.a_bytes = lin_operand_bytes(a, type, K), p.b_bytes = lin_operand_bytes(b, type, K);
    const auto tiles = [&](int t) { return (double)((a.R + t - 1) / t) * (double)((b.R + t - 1) / t); };
    p.tile = tiles(256) >= LIN_CUS ? 256 : 128;
    const long long stages = (lin_padded(type, K) * (type == DL_E4M3 ? 1 : 2) / LIN_STAGE_BYTES) * (type == DL_F32 ? LIN_COMBOS : 1);
    p.splits = 1;
    if (p.tile == 128)
        while (p.splits < 64 && tiles(128) * p.splits * 2 <= 2 * LIN_CUS && stages / (p.splits * 2) >= 4) p.splits *= 2;
    p.chunk = (int)((stages + p.splits - 1) / p.splits);
    p.splits = (int)((stages + p.chunk - 1) / p.chunk);  // (none without a stage)
    p.part_bytes = p.splits > 1 ? dl_align256((size_t)p.splits * (size_t)a.R * (size_t)b.R * 4) : 0;
    return p;
}

template <typename T>
static void lin_lay_out_as(const LinOperand &o, void *dst, long long K, long long Kp, hipStream_t s) {
    typedef typename LinCell<T>::type Cell;
    if (o.turned) {
        const int row_tiles = dl_ceil_div(o.R, 64);
        DL_TIMED("lin_turn", s, hipLaunchKernelGGL((lin_turn<T>), dim3((unsigned)(row_tiles * (Kp / 64))), dim3(256), 0, s, (const T *)o.p, o.ld, (Cell *)dst, o.R, K, Kp, row_tiles));
    } else {
        const long long blocks = (o.R * (Kp / 8) + 255) / 256;
        DL_TIMED("lin_pad", s, hipLaunchKernelGGL((lin_pad<T>), dim3((unsigned)(blocks < 16384 ? blocks : 16384)), dim3(256), 0, s, (const T *)o.p, o.ld, (Cell *)dst, o.R, K, Kp));
    }
}
// the operand as the product reads it, and its row and plane strides in bytes
static const char *lin_lay_out(const LinOperand &o, int type, long long K, void *room, long long &ld, long long &plane, hipStream_t s) {
    const int size = type == DL_E4M3 ? 1 : 2;
    plane = 0;
    if (lin_direct(o, type, K)) {
        ld = o.ld * size;
        return (const char *)o.p;
    }
    const long long Kp = lin_padded(type, K);
    ld = Kp * size, plane = o.R * ld;
    if (type == DL_F32) lin_lay_out_as<float>(o, room, K, Kp, s);
    else if (type == DL_E4M3) lin_lay_out_as<uint8_t>(o, room, K, Kp, s);
    else lin_lay_out_as<uint16_t>(o, room, K, Kp, s);
    return (const char *)room;
}

template <typename In, typename Out, int T, int WR, int WC>
static int lin_launch_tile(const LinArgs &g, int splits, bool gated, hipStream_t s) {
    constexpr int BYTES = 4 * T * LIN_STAGE_BYTES;
    const long long blocks = (long long)splits * DL_XCDS * dl_ceil_div((long long)g.row_tiles * g.col_tiles, DL_XCDS);
    if (!dl_grid_ok(blocks, 64 * WR * WC)) return DL_ERR_UNSUPPORTED;
#define LIN_GO(GATED, PARTIAL)                                                                                                           \
    do {                                                                                                                                 \
        if (BYTES > 65536) {                                                                                                             \
            const hipError_t room = hipFuncSetAttribute(reinterpret_cast<const void *>(&lin_product<In, Out, T, T, WR, WC, GATED, PARTIAL>),  \
                                                        hipFuncAttributeMaxDynamicSharedMemorySize, BYTES);                              \
            if (room != hipSuccess) return (int)room;                                                                                    \
        }                                                                                                                                \
        DL_TIMED("lin_product", s, hipLaunchKernelGGL((lin_product<In, Out, T, T, WR, WC, GATED, PARTIAL>), dim3((unsigned)blocks), dim3(64 * WR * WC), BYTES, s, g)); \
    } while (0)
    if (splits > 1) LIN_GO(false, true);
    else if (gated) LIN_GO(true, false);
    else LIN_GO(false, false);
#undef LIN_GO
    return DL_OK;
}
template <typename In, typename Out>
static int lin_launch(LinArgs &g, const LinPlan &p, bool gated, hipStream_t s) {
    const int code = p.tile == 256 ? lin_launch_tile<In, Out, 256, 2, 4>(g, p.splits, gated, s) : lin_launch_tile<In, Out, 128, 2, 2>(g, p.splits, gated, s);
    if (code != DL_OK || p.splits == 1) return code;
    const long long blocks = ((long long)g.end.R * (((gated ? g.end.F : g.end.C) + 7) / 8) + 255) / 256;
    const dim3 grid((unsigned)(blocks < 16384 ? blocks : 16384));
    if (gated) DL_TIMED("lin_join", s, hipLaunchKernelGGL((lin_join<Out, true>), grid, dim3(256), 0, s, g, p.splits));
    else DL_TIMED("lin_join", s, hipLaunchKernelGGL((lin_join<Out, false>), grid, dim3(256), 0, s, g, p.splits));
    return DL_OK;
}

// One product: operands laid out, tiles, what follows
static int lin_run(const LinOperand &a, const LinOperand &b, int type, int out_type, long long K, bool gated, LinEnd end, char *ws, hipStream_t s) {
    const LinPlan p = lin_plan(a, b, type, K);
    LinArgs g{};
    g.A = lin_lay_out(a, type, K, ws, g.lda, g.plane_a, s);
    g.B = lin_lay_out(b, type, K, ws + p.a_bytes, g.ldb, g.plane_b, s);
    if (g.lda > LIN_MOST_ROW || g.ldb > LIN_MOST_ROW) return DL_ERR_UNSUPPORTED;
    g.part = (float *)(ws + p.a_bytes + p.b_bytes);
    g.k_bytes = (int)((K * (type == DL_E4M3 ? 1 : 2) + 15) / 16 * 16);
    g.stages = dl_ceil_div(g.k_bytes, LIN_STAGE_BYTES), g.combos = type == DL_F32 ? LIN_COMBOS : 1;
    g.chunk = p.chunk;
    const bool halves = gated && p.splits == 1;
    g.row_tiles = dl_ceil_div(a.R, p.tile), g.col_tiles = halves ? dl_ceil_div(b.R / 2, p.tile / 2) : dl_ceil_div(b.R, p.tile);
    end.R = (int)a.R, end.C = (int)b.R, end.F = (int)(b.R / 2);
    const int width = gated ? end.F : end.C, size = dl_type_bytes(out_type);
    end.vec = width % 8 == 0 && dl_aligned16(end.y) && dl_aligned16(end.z) && dl_aligned16(end.bias) && dl_aligned16(end.res) && end.ldr * size % 16 == 0;
    g.end = end;
    int code = DL_ERR_UNSUPPORTED;
    if (type == DL_E4M3) DL_BY_TYPE(out_type, Out, code = lin_launch<LinE4m3, Out>(g, p, gated, s));
    else if (type == DL_F32) code = lin_launch<LinBf16, float>(g, p, gated, s);
    else if (type == DL_BF16) code = lin_launch<LinBf16, dl_bf16>(g, p, gated, s);
    else code = lin_launch<LinF16, dl_f16>(g, p, gated, s);
    return code != DL_OK ? code : dl_launch_status();
}

static int lin_check(int type, int out_type, long long M, long long N, long long K, int act, int gated) {
    if (M <= 0 || N <= 0 || K <= 0 || M >= LIN_MOST || N >= LIN_MOST || K >= LIN_MOST) return DL_ERR_SHAPE;
    if (gated && N % 2 != 0) return DL_ERR_SHAPE;
    if (!(dl_type_known(type) ? out_type == type : type == DL_E4M3 && dl_type_known(out_type))) return DL_ERR_UNSUPPORTED;
    if (act < DL_ACT_NONE || act > DL_ACT_SIGMOID) return DL_ERR_UNSUPPORTED;
    if (K * 2 > LIN_MOST_ROW) return DL_ERR_UNSUPPORTED;
    return DL_OK;
}

extern "C" size_t dl_linear_fwd_workspace_bytes(const void *x, long long ldx, const void *w, long long ldw, int type, long long M, long long N, long long K,
                                                int gated) {
    if (lin_check(type, type == DL_E4M3 ? DL_F32 : type, M, N, K, 0, gated) != DL_OK) return 0;
    return lin_plan({x, ldx, M, false}, {w, ldw, N, false}, type, K).bytes();
}

extern "C" int dl_linear_fwd(const void *x, long long ldx, const float *x_scale, const void *w, long long ldw, const float *w_scale, const void *bias,
                             const void *residual, long long ldr, void *y, void *z, int type, int out_type, long long M, long long N, long long K, int act,
                             int gated, void *ws, size_t ws_bytes, void *stream) {
    if (!x || !w || !y || ((x_scale || w_scale) != (type == DL_E4M3)) || (type == DL_E4M3 && (!x_scale || !w_scale))) return DL_ERR_NULL;
    const int bad = lin_check(type, out_type, M, N, K, act, gated);
    if (bad) return bad;
    if (ldx < K || ldw < K || (residual && ldr < (gated ? N / 2 : N))) return DL_ERR_SHAPE;
    const size_t need = dl_linear_fwd_workspace_bytes(x, ldx, w, ldw, type, M, N, K, gated);
    if (need && !ws) return DL_ERR_NULL;
    if (ws_bytes < need || (need && !dl_aligned16(ws))) return DL_ERR_WORKSPACE;
    LinEnd end{};
    end.y = y, end.z = z, end.bias = bias, end.res = residual, end.ldr = residual ? ldr : 0, end.row_scale = x_scale, end.col_scale = w_scale, end.act = act;
    return lin_run({x, ldx, M, false}, {w, ldw, N, false}, type, out_type, K, gated != 0, end, (char *)ws, (hipStream_t)stream);
}

// ------------------------------------------------------------------ backward
struct LinBack {
    size_t gz, shares, products;
    int pieces, rows;
    size_t bytes() const { return gz + shares + products; }
};
static LinBack lin_back(const LinOperand &gz, const LinOperand &x, const LinOperand &w, int type, bool kept, int wants, long long N, long long K) {
    LinBack b{};
    const long long M = gz.R;
    b.gz = kept ? dl_align256((size_t)M * (size_t)N * lin_size(type)) : 0;
    b.rows = LIN_SLOPE_ROWS;
    while ((M + b.rows - 1) / b.rows > 1024) b.rows *= 2;
    b.pieces = dl_ceil_div(M, b.rows);
    b.shares = wants & 4 ? dl_align256((size_t)b.pieces * (size_t)N * 4) : 0;
    const LinOperand gt = {gz.p, gz.ld, N, true}, wt = {w.p, w.ld, K, true}, xt = {x.p, x.ld, K, true};
    if (wants & 1) b.products = lin_plan(gz, wt, type, N).bytes();
    if (wants & 2) {
        const size_t n = lin_plan(gt, xt, type, M).bytes();
        if (n > b.products) b.products = n;
    }
    return b;
}
// (the workspace begins on 16 bytes, as gz in it does, so a pointer of that alignment stands for it)
static const void *lin_gz_place(const void *ws, const void *gy, bool kept) { return kept ? (ws ? ws : (const void *)256) : gy; }

extern "C" size_t dl_linear_bwd_workspace_bytes(const void *x, long long ldx, const void *w, long long ldw, const void *z, const void *gy, int wants, int type,
                                                long long M, long long N, long long K) {
    if (lin_check(type, type, M, N, K, 0, 0) != DL_OK) return 0;
    return lin_back({lin_gz_place(nullptr, gy, z != nullptr), N, M, false}, {x, ldx, M, false}, {w, ldw, N, false}, type, z != nullptr, wants, N, K).bytes();
}

extern "C" int dl_linear_bwd(const void *x, long long ldx, const void *w, long long ldw, const void *z, const void *gy, void *gx, void *gw, void *gb, int type,
                             long long M, long long N, long long K, int act, int gated, void *ws, size_t ws_bytes, void *stream) {
    if (!gy || (gx && !w) || (gw && !x) || ((gated || act != DL_ACT_NONE) && !z)) return DL_ERR_NULL;
    const int bad = lin_check(type, type, M, N, K, act, gated);
    if (bad) return bad;
    if (N * 2 > LIN_MOST_ROW || (gw && M * 2 > LIN_MOST_ROW)) return DL_ERR_UNSUPPORTED;
    if ((gx && ldw < K) || (gw && ldx < K)) return DL_ERR_SHAPE;
    const int wants = (gx ? 1 : 0) | (gw ? 2 : 0) | (gb ? 4 : 0);
    if (!wants) return DL_OK;
    const bool kept = z != nullptr;
    LinOperand gz = {lin_gz_place(ws, gy, kept), N, M, false};
    const LinOperand xo = {x, ldx, M, false}, wo = {w, ldw, N, false};
    const LinBack p = lin_back(gz, xo, wo, type, kept, wants, N, K);
    if (p.bytes() && !ws) return DL_ERR_NULL;
    if (ws_bytes < p.bytes() || !dl_aligned16(ws)) return DL_ERR_WORKSPACE;
    const hipStream_t s = (hipStream_t)stream;
    float *shares = gb ? (float *)((char *)ws + p.gz) : nullptr;
    if (kept || gb) {
        void *out = kept ? ws : nullptr;
#define LIN_GRADIENT(E, GATED) hipLaunchKernelGGL((lin_gradient<T, E, GATED>), dim3((unsigned)blocks), dim3(256), 0, s, (const T *)gy, (const T *)z, (T *)out, shares, M, (int)N, act, col_tiles, p.rows)
        const int width = (int)(gated ? N / 2 : N);
        DL_BY_TYPE(type, T, {
            constexpr int E = 16 / sizeof(T);
            const bool vec = width % E == 0 && dl_aligned16(gy) && dl_aligned16(z);
            const int col_tiles = dl_ceil_div(width, 64 * (vec ? E : 1));
            const long long blocks = (long long)col_tiles * p.pieces;
            if (!dl_grid_ok(blocks, 256)) return DL_ERR_UNSUPPORTED;
            DL_TIMED("lin_gradient", s, if (gated) { if (vec) LIN_GRADIENT(E, true); else LIN_GRADIENT(1, true); }
                     else if (vec) LIN_GRADIENT(E, false); else LIN_GRADIENT(1, false));
            if (gb) DL_TIMED("lin_columns", s, hipLaunchKernelGGL((lin_columns<T>), dim3(dl_ceil_div(N, 16)), dim3(256), 0, s, shares, (T *)gb, p.pieces, (int)N));
        });
#undef LIN_GRADIENT
    }
    char *room = (char *)ws + p.gz + p.shares;
    LinEnd end{};
    if (gx) {
        end.y = gx;
        const int code = lin_run(gz, {w, ldw, K, true}, type, type, N, false, end, room, s);
        if (code != DL_OK) return code;
    }
    if (gw) {
        end.y = gw;
        const int code = lin_run({gz.p, N, N, true}, {x, ldx, K, true}, type, type, M, false, end, room, s);
        if (code != DL_OK) return code;
    }
    return dl_launch_status();
}
