// Matrix products with bias, activation, a gate and a residual in the same launch, and their backward pass, on the 16-bit and
// 8-bit matrix cores with fp32 accumulation.
//
//   linear    z[m,n] = sum_k x[m,k] w[n,k] + b[n],   y = act(z) + residual
//   gated     z over 2 F rows of w, gate first:      y[m,f] = act(z[m,f]) z[m,F+f]
//   backward  gz = gy act'(z)   (gated: gz[f] = gy z[F+f] act'(z[f]),  gz[F+f] = gy act(z[f])),  gb = sum_m gz,  gx = gz w,  gw = gz^T x
//
// One product kernel serves all of them: C[r,c] = sum_k A(r,k) B(c,k).  An operand lies with the reduction along its rows of memory, or
// (w for gx, gz and x for gw) with the reduction across them, and is turned on the way out of the LDS.  Operands whose rows do not
// start on 16 bytes or end inside 16 are copied to rows that do, by a pass in front of it.
//
// float32 values are cut into three bf16 planes on the way out of the LDS (8 + 8 + 8 significant bits, each the rounding of what the ones
// above left); a product is the six plane products hi*lo, lo*hi, mid*mid, hi*mid, mid*hi, hi*hi, small ones first.  What is left out is
// below 2^-26 of |a b|, less than the 2^-24 of one fp32 multiply-add.  Six bf16 products at 2.5 PFLOP/s are 417 TFLOP/s of fp32 work
// against 157 on the fp32 matrix cores.  (Planes carry no infinities: such a product is NaN.)
#pragma once
#include <utility>

#include "dl_types.h"

typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 halfx8 __attribute__((ext_vector_type(8)));
typedef int intx4 __attribute__((ext_vector_type(4)));
typedef int intx8 __attribute__((ext_vector_type(8)));

#define LIN_STAGE_BYTES 128  // of a row in a stage: 32 float32, 64 16-bit or 128 8-bit values
#define LIN_PLANES 3
#define LIN_CUS 256

struct LinF32 { static constexpr int SIZE = 4; };
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

// ------------------------------------------------------------------ what follows a product
struct LinEnd {
    void *y, *z;                // z (null: not kept): what the activation is applied to, in y's type
    const void *bias, *res;
    const float *row_scale, *col_scale;  // of 8-bit operands
    long long ldr;
    int R, C, F, act;           // C: rows of w; F: columns of y where gated
    bool vec;                   // whole vectors of eight everywhere
};

// What belongs to eight columns from c on, whatever the row; gated: of the gate and of the other half.  Past the last column: nothing.
template <typename Out, bool GATED>
struct LinColumns {
    static constexpr int H = GATED ? 2 : 1;
    float scale[H][8], bias[H][8];
    __device__ __forceinline__ LinColumns(const LinEnd &g, int c) {
#pragma unroll
        for (int h = 0; h < H; ++h) {
#pragma unroll
            for (int i = 0; i < 8; ++i) scale[h][i] = 1.0f, bias[h][i] = 0.0f;
            if (c >= (GATED ? g.F : g.C)) continue;
            if (g.col_scale) dl_load<float, 8>(g.col_scale + h * g.F + c, scale[h]);
            if (g.bias) dl_load<Out, 8>((const Out *)g.bias + h * g.F + c, bias[h]);
        }
    }
};
// of eight columns of a row, as it lies
template <typename Out>
__device__ __forceinline__ DlVec<Out, 8> lin_residual(const LinEnd &g, int width, int r, int c) {
    DlVec<Out, 8> f;
#pragma unroll
    for (int i = 0; i < 8; ++i) f.v[i] = (Out)0.0f;
    if (g.res && r < g.R && c < width) f = *reinterpret_cast<const DlVec<Out, 8> *>((const Out *)g.res + r * g.ldr + c);
    return f;
}
// Eight columns from c on of row r, from their sums v (gated: the gate's, u the other half's), the row's scale and the residual
template <typename Out, bool GATED>
__device__ __forceinline__ void lin_finish(const LinEnd &g, const LinColumns<Out, GATED> &k, int r, int c, float (&v)[8], float (&u)[8], float row_scale, const DlVec<Out, 8> &res) {
    const int width = GATED ? g.F : g.C;
    if (r >= g.R || c >= width) return;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        v[i] = fmaf(v[i], row_scale * k.scale[0][i], k.bias[0][i]);
        if (GATED) u[i] = fmaf(u[i], row_scale * k.scale[LinColumns<Out, GATED>::H - 1][i], k.bias[LinColumns<Out, GATED>::H - 1][i]);
    }
    if (g.z) {
        Out *z = (Out *)g.z + (long long)r * g.C + c;
        dl_store<Out, 8>(z, v);
        if (GATED) dl_store<Out, 8>(z + g.F, u);
    }
    if (g.act == DL_ACT_RELU) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = lin_act(v[i], DL_ACT_RELU);
    } else if (g.act != DL_ACT_NONE) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float s = lin_sigmoid(v[i]);
            v[i] = g.act == DL_ACT_SILU ? v[i] * s : s;
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (GATED ? v[i] * u[i] : v[i]) + (float)res.v[i];
    dl_store<Out, 8>((Out *)g.y + (long long)r * width + c, v);
}
// One column, where not everything is whole vectors of eight
template <typename Out, bool GATED>
__device__ __forceinline__ void lin_finish_one(const LinEnd &g, int r, int c, float v, float u) {
    const int width = GATED ? g.F : g.C;
    if (r >= g.R || c >= width) return;
    const float row_scale = g.row_scale ? g.row_scale[r] : 1.0f;
    v = fmaf(v, row_scale * (g.col_scale ? g.col_scale[c] : 1.0f), g.bias ? (float)((const Out *)g.bias)[c] : 0.0f);
    if (GATED) u = fmaf(u, row_scale * (g.col_scale ? g.col_scale[g.F + c] : 1.0f), g.bias ? (float)((const Out *)g.bias)[g.F + c] : 0.0f);
    if (g.z) {
        Out *z = (Out *)g.z + (long long)r * g.C + c;
        z[0] = (Out)v;
        if (GATED) z[g.F] = (Out)u;
    }
    const float y = lin_act(v, g.act);
    ((Out *)g.y)[(long long)r * width + c] = (Out)((GATED ? y * u : y) + (g.res ? (float)((const Out *)g.res)[r * g.ldr + c] : 0.0f));
}

// ------------------------------------------------------------------ the product
struct LinArgs {
    const char *A, *B;
    long long lda, ldb;          // bytes
    long long K;                 // of the reduction, values
    int stages, chunk;           // of the reduction; of a block (all of them without PARTIAL)
    int row_tiles, col_tiles;
    float *part;                 // PARTIAL: sums [splits][R][C]
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
// this wavefront's loads but the last N have landed, its LDS reads are done, and every wavefront has got here
template <int N>
__device__ __forceinline__ void lin_stage_barrier() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// What a lane gives to a step of the matrix cores: 8 values of 16 bits or 32 of 8 bits; of float32 8 values as planes
template <typename In>
struct LinFragment {
    static constexpr int WORDS = __is_same(In, LinE4m3) ? 8 : 4, PLANES = __is_same(In, LinF32) ? LIN_PLANES : 1;
    int w[PLANES][WORDS];
};
__device__ __forceinline__ unsigned lin_pk_bf16(float a, float b) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    typedef float floatx2 __attribute__((ext_vector_type(2)));
    const floatx2 v = {a, b};
    return __builtin_bit_cast(unsigned, __builtin_convertvector(v, bf16x2));
}
// values 2 i and 2 i + 1
__device__ __forceinline__ void lin_cut(const float (&f)[8], int i, LinFragment<LinF32> &out) {
    float a = f[2 * i], b = f[2 * i + 1];
#pragma unroll
    for (int p = 0; p < LIN_PLANES; ++p) {
        const unsigned w = lin_pk_bf16(a, b);
        out.w[p][i] = (int)w;
        a -= __uint_as_float(w << 16);
        b -= __uint_as_float(w & 0xffff0000u);
    }
}
template <typename In>
__device__ __forceinline__ floatx16 lin_mfma(const LinFragment<In> &a, const LinFragment<In> &b, floatx16 c, int t) {
    if constexpr (__is_same(In, LinE4m3)) {  // block scales of 2^0
        return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(__builtin_bit_cast(intx8, a), __builtin_bit_cast(intx8, b), c, 0, 0, 0, 0x7f7f7f7f, 0, 0x7f7f7f7f);
    } else if constexpr (__is_same(In, LinBf16)) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    } else if constexpr (__is_same(In, LinF16)) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(halfx8, a), __builtin_bit_cast(halfx8, b), c, 0, 0, 0);
    } else {
        constexpr int PA[6] = {0, 2, 1, 0, 1, 0}, PB[6] = {2, 0, 1, 1, 0, 0};
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a.w[PA[t]]), __builtin_bit_cast(bf16x8, b.w[PB[t]]), c, 0, 0, 0);
    }
}

// An operand's tile in the LDS: T rows (or columns) of C by a stage of the reduction, loaded by 1 KB per wavefront and load.
// Reduction along the memory's rows: T rows of 128 bytes, whose eight units of 16 bytes are kept in turned order (unit u in slot
//   u ^ (row & 7)), so that the eight lanes of an LDS read that take one unit of eight rows find them on different banks.
// Reduction across them (TURNED): LIN_STAGE_BYTES / SIZE rows of T values.  16-bit values are turned by ds_read_b64_tr_b16, sixteen lanes
//   of which read four rows of 16 values: units of row k are kept in slots u ^ 4 (k & 3).  float32 values are read one by one, lanes along
//   the row, half the wavefront eight rows further on: slots u ^ 8 (k / 8 & 1).
// The loads fetch in that order, so the LDS is written in the order of its addresses.
template <typename In, int T, bool TURNED>
struct LinTile {
    static constexpr int SIZE = In::SIZE, KS = LIN_STAGE_BYTES / SIZE, ROW = TURNED ? T * SIZE : LIN_STAGE_BYTES, UNITS = ROW / 16, PER = 64 / UNITS, BYTES = T * LIN_STAGE_BYTES,
                         LOADS = T / 8;
    static_assert(!TURNED || SIZE >= 2, "8-bit operands have the reduction along their rows");
    static __device__ __forceinline__ int row_of(int load, int lane) { return load * PER + lane / UNITS; }
    static __device__ __forceinline__ int unit_of(int row, int lane) {
        const int slot = lane % UNITS;
        return !TURNED ? slot ^ (row & 7) : SIZE == 2 ? slot ^ (4 * (row & 3)) : slot ^ (8 * (row >> 3 & 1));
    }
};

// The F fragments of 32 rows each, from row `first` of the tile on.  Lane l has row l % 32 of a fragment, and of a step's values along the
// reduction the eight (of 8 bits 2 x 16) at l / 32.  A fragment comes in PER reads; float32 fragments come raw, and are cut a pair of
// values at a time.
template <typename In, int T, bool TURNED, int F>
struct LinReader {
    typedef LinTile<In, T, TURNED> Tile;
    static constexpr int PER = Tile::SIZE == 1 || (Tile::SIZE == 2 && TURNED) ? 2 : 1;
    unsigned at[F];
    unsigned turn;  // the lane's unit of the first step
    __device__ __forceinline__ LinReader(int first, int lane) {
        const int kh = lane >> 5, l32 = lane & 31;
        turn = (unsigned)(((Tile::SIZE == 4 ? 2 * kh : kh) ^ (lane & 7)) * 16);
#pragma unroll
        for (int i = 0; i < F; ++i) {
            if (!TURNED) at[i] = (first + i * 32 + l32) * Tile::ROW;
            else if (Tile::SIZE == 2) {  // lane: row kh * 8 + q / 4, columns 16 oh + 4 (q % 4)
                const int q = lane & 15, oh = lane >> 4 & 1, granule = (first / 16 + 2 * i + oh) ^ (2 * (q >> 2));
                at[i] = (kh * 8 + (q >> 2)) * Tile::ROW + granule * 32 + (q & 3) * 8;
            } else at[i] = kh * 8 * Tile::ROW + (((first + i * 32 + l32) * 4) ^ (kh * 128));
        }
    }
    // units 4 (of 16-bit values 2) and part further on: exclusive or keeps their turned order
    __device__ __forceinline__ void read(const char *tile, int step, int i, int part, LinFragment<In> &out) const {
        const char *p = tile + at[i];
        if constexpr (__is_same(In, LinE4m3)) {
            *reinterpret_cast<intx4 *>(&out.w[0][4 * part]) = *reinterpret_cast<const intx4 *>(p + (turn ^ (64 * step + 32 * part)));
        } else if constexpr (!TURNED) {
            *reinterpret_cast<intx4 *>(&out.w[0][0]) = *reinterpret_cast<const intx4 *>(p + (turn ^ (32 * step)));
        } else {
            typedef short shortx4 __attribute__((ext_vector_type(4)));
            typedef int intx2 __attribute__((ext_vector_type(2)));
            typedef __attribute__((address_space(3))) shortx4 lds_shortx4;
            *reinterpret_cast<intx2 *>(&out.w[0][2 * part]) = __builtin_bit_cast(intx2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_shortx4 *)(p + (step * 16 + part * 4) * Tile::ROW)));
        }
    }
    __device__ __forceinline__ void read_raw(const char *tile, int step, int i, float (&f)[8]) const {
        const char *p = tile + at[i];
        if constexpr (!TURNED) {
#pragma unroll
            for (int q = 0; q < 2; ++q) *reinterpret_cast<float4 *>(f + 4 * q) = *reinterpret_cast<const float4 *>(p + (turn ^ (64 * step + 16 * q)));
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = *reinterpret_cast<const float *>(p + (step * 16 + e) * Tile::ROW);
        }
    }
};
// f(0), ..., f(N - 1) with the number as a constant
template <int N>
struct LinIs {
    static constexpr int value = N;
};
template <int BASE, typename F, int... I>
__device__ __forceinline__ void lin_each_of(std::integer_sequence<int, I...>, F f) { (f(LinIs<BASE + I>()), ...); }
template <int FROM, int TO, typename F>
__device__ __forceinline__ void lin_each(F f) {
    if constexpr (TO > FROM) lin_each_of<FROM>(std::make_integer_sequence<int, TO - FROM>(), f);
}

// A block of four wavefronts makes a tile of TR x TC, a wavefront a quarter of it, in stages of 128 bytes along the reduction: three of A and two of
// B are in the LDS.  A stage has 2 or 4 steps of the matrix cores; a step's fragments are read while the one before is worked on, across
// stages too: by the last step of a stage all of it has been read and the next one has landed.  B's stage after the next is sent for
// then, into the same place, A's one step later, so that loads are spread over the matrix instructions and have a stage's time to land.  One wavefront
// a SIMD issues everything, so reads, loads and (of float32) cuts stand between the matrix instructions in the order written here; left
// to itself the compiler puts the reads in front of their use.  Where the reduction ends inside a stage, that stage comes first.
// Gated, a wavefront's columns are those of the gate, then the ones that belong to them.
template <typename In, typename Out, int TR, int TC, bool TURN_A, bool TURN_B, bool GATED, bool PARTIAL>
__global__ __launch_bounds__(256, TR * TC > 128 * 128 ? 1 : 2) void lin_product(LinArgs g) {
    extern __shared__ __align__(16) char lds[];
    typedef LinTile<In, TR, TURN_A> TileA;
    typedef LinTile<In, TC, TURN_B> TileB;
    constexpr int WAVES = 4, FA = TR / 64, FB = TC / 64, B_PLACE = 3 * TileA::BYTES, KS = TileA::KS;
    constexpr int NA = TileA::LOADS / WAVES, NB = TileB::LOADS / WAVES, STEPS = In::SIZE == 2 ? 4 : 2, HALF = FB * 16;
    static_assert(STEPS % 2 == 0, "a stage begins in the first of two sets of fragments");
    typedef __attribute__((address_space(3))) char lds_char;
    const unsigned lds_base = (unsigned)(uintptr_t)(lds_char *)lds;
    const int lane = threadIdx.x & 63, wave = dl_uniform(threadIdx.x >> 6);

    // tiles: every XCD takes a run of them, eight rows of tiles at a time, so that its L2 holds what neighbours share
    const int tiles = g.row_tiles * g.col_tiles, per = (tiles + DL_XCDS - 1) / DL_XCDS;
    const int split = blockIdx.x / (per * DL_XCDS), id = blockIdx.x % (per * DL_XCDS);
    const int tile = (id % DL_XCDS) * per + id / DL_XCDS;
    if (tile >= tiles) return;
    const int band = tile / (8 * g.col_tiles), in_band = tile % (8 * g.col_tiles), band_rows = min(8, g.row_tiles - band * 8);
    const int r0 = (band * 8 + in_band % band_rows) * TR, c0 = in_band / band_rows * (GATED ? TC / 2 : TC);
    const int first = split * g.chunk, count = min(g.stages - first, g.chunk);

    // ---- what this lane fetches: offsets from the tile's first row and the stage's first value
    unsigned a_off[NA], b_off[NB];
    const char *a_base = TURN_A ? g.A : g.A + (long long)r0 * g.lda;
    const char *b_base = TURN_B ? g.B : g.B + (long long)c0 * g.ldb, *b_other = GATED ? b_base + g.end.F * g.ldb : b_base;
#pragma unroll
    for (int j = 0; j < NA; ++j) {
        const int row = TileA::row_of(wave + j * WAVES, lane), unit = TileA::unit_of(row, lane);
        a_off[j] = TURN_A ? (unsigned)row * (unsigned)g.lda + (unsigned)min(r0 * In::SIZE + unit * 16, (g.end.R * In::SIZE + 15) / 16 * 16 - 16)
                          : (unsigned)(min(r0 + row, g.end.R - 1) - r0) * (unsigned)g.lda + unit * 16;
    }
#pragma unroll
    for (int j = 0; j < NB; ++j) {
        const int row = TileB::row_of(wave + j * WAVES, lane), unit = TileB::unit_of(row, lane);
        // (gated: rows of the tile are HALF of the gate, HALF of the other, and so on)
        const int f = GATED ? row / (2 * HALF) * HALF + row % HALF : row, most = GATED ? g.end.F : g.end.C;
        b_off[j] = TURN_B ? (unsigned)row * (unsigned)g.ldb + (unsigned)min(c0 * In::SIZE + unit * 16, (g.end.C * In::SIZE + 15) / 16 * 16 - 16)
                          : (unsigned)(min(c0 + f, most - 1) - c0) * (unsigned)g.ldb + unit * 16;
    }
    static_assert(!GATED || (WAVES * TileB::PER <= HALF && HALF % (WAVES * TileB::PER) == 0), "the four wavefronts' loads are of one half");
    constexpr auto other = [](int j) { return GATED && j * WAVES * TileB::PER % (2 * HALF) >= HALF; };
    // where the reduction ends inside a stage: that stage is the block's first
    const int whole = (int)(g.K / KS), left = (int)(g.K - (long long)whole * KS), tail = first + count - min(first + count, whole);
    const auto stage_of = [&](int s) { return s == 0 ? first + (count - 1) * tail : first + s - tail; };
    const auto begin_a = [&](int s) { return a_base + (long long)stage_of(s) * KS * (TURN_A ? g.lda : In::SIZE); };
    const auto begin_b = [&](int s, const char *base) { return base + (long long)stage_of(s) * KS * (TURN_B ? g.ldb : In::SIZE); };
    const auto load_a = [&](const char *from, unsigned to, int j) __attribute__((always_inline)) { lin_to_lds(to + (wave + j * WAVES) * 1024, from, a_off[j]); };
    const auto load_b = [&](const char *from, const char *from_other, unsigned to, int j) __attribute__((always_inline)) {
        lin_to_lds(to + (wave + j * WAVES) * 1024, other(j) ? from_other : from, b_off[j]);
    };

    floatx16 acc[FA][FB];
#pragma unroll
    for (int i = 0; i < FA; ++i)
#pragma unroll
        for (int j = 0; j < FB; ++j)
#pragma unroll
            for (int v = 0; v < 16; ++v) acc[i][j][v] = 0.0f;

    const int kh = lane >> 5, l32 = lane & 31, wr = wave / 2 * (TR / 2), wc = wave % 2 * (TC / 2);
    const LinReader<In, TR, TURN_A, FA> read_a(wr, lane);
    const LinReader<In, TC, TURN_B, FB> read_b(wc, lane);
    LinFragment<In> a[2][FA], b[2][FB];

    // the first two stages
    if (tail) {
#pragma unroll
        for (int j = 0; j < NA; ++j) {
            const int row = TileA::row_of(wave + j * WAVES, lane), value = TURN_A ? row : TileA::unit_of(row, lane) * (16 / In::SIZE);
            lin_to_lds_far(lds_base + (wave + j * WAVES) * 1024, value < left ? begin_a(0) + a_off[j] : (const char *)&lin_zeros);
        }
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            const int row = TileB::row_of(wave + j * WAVES, lane), value = TURN_B ? row : TileB::unit_of(row, lane) * (16 / In::SIZE);
            lin_to_lds_far(lds_base + B_PLACE + (wave + j * WAVES) * 1024, value < left ? begin_b(0, other(j) ? b_other : b_base) + b_off[j] : (const char *)&lin_zeros);
        }
    } else {
#pragma unroll
        for (int j = 0; j < NA; ++j) load_a(begin_a(0), lds_base, j);
#pragma unroll
        for (int j = 0; j < NB; ++j) load_b(begin_b(0, b_base), begin_b(0, b_other), lds_base + B_PLACE, j);
    }
    if (count > 1) {
#pragma unroll
        for (int j = 0; j < NA; ++j) load_a(begin_a(1), lds_base + TileA::BYTES, j);
#pragma unroll
        for (int j = 0; j < NB; ++j) load_b(begin_b(1, b_base), begin_b(1, b_other), lds_base + B_PLACE + TileB::BYTES, j);
        lin_stage_barrier<NA + NB>();
    } else lin_stage_barrier<0>();

    // Side work of a step, one piece after the other: fragments in the order in which the next step takes them (A's first, all of B, the rest of A)
    constexpr bool CUT = __is_same(In, LinF32);
    constexpr int FRAGMENTS = FA + FB, PA = LinReader<In, TR, TURN_A, FA>::PER, PB = LinReader<In, TC, TURN_B, FB>::PER;
    constexpr int PIECES = CUT ? 5 * (FRAGMENTS + 1) : FA * PA + FB * PB, PRODUCTS = CUT ? 6 : 1, SLOTS = FA * FB * PRODUCTS;
    constexpr int READ_SLOTS = CUT ? SLOTS : SLOTS * 3 / 4;  // (the last reads are answered by the next step)
    float raw[2][8];
    const auto piece = [&](auto number, unsigned from_a, unsigned from_b, int step, int set) __attribute__((always_inline)) {
        constexpr int o = decltype(number)::value;
        if constexpr (CUT) {  // read a fragment, then cut the one before
            constexpr int f = o / 5, r = o % 5, q = f - 1;
            if constexpr (r == 0 && f < FRAGMENTS) {
                if constexpr (f == 0 || f > FB) read_a.read_raw(lds + from_a, step, f == 0 ? 0 : f - FB, raw[f & 1]);
                else read_b.read_raw(lds + B_PLACE + from_b, step, f - 1, raw[f & 1]);
            }
            if constexpr (r > 0 && f > 0) {
                if constexpr (q == 0 || q > FB) lin_cut(raw[q & 1], r - 1, a[set][q == 0 ? 0 : q - FB]);
                else lin_cut(raw[q & 1], r - 1, b[set][q - 1]);
            }
        } else if constexpr (o < PA) read_a.read(lds + from_a, step, 0, o, a[set][0]);
        else if constexpr (o < PA + FB * PB) read_b.read(lds + B_PLACE + from_b, step, (o - PA) / PB, (o - PA) % PB, b[set][(o - PA) / PB]);
        else read_a.read(lds + from_a, step, (o - FB * PB) / PA, (o - FB * PB) % PA, a[set][(o - FB * PB) / PA]);
    };
    lin_each<0, PIECES>([&](auto o) __attribute__((always_inline)) { piece(o, 0, 0, 0, 0); });

    unsigned a_now = 0, a_next = TileA::BYTES, a_free = 2 * TileA::BYTES, b_now = 0;
    const char *from_a = begin_a(2);  // (not followed where there are no three stages)
    const char *from_b = begin_b(2, b_base), *from_other = begin_b(2, b_other);
    // MORE: stages behind this one, 2 standing for two or more
    const auto stage = [&](auto more) __attribute__((always_inline)) {
        constexpr int MORE = decltype(more)::value;
        lin_each<0, STEPS>([&](auto step) __attribute__((always_inline)) {
            constexpr int st = decltype(step)::value;
            constexpr bool last = st + 1 == STEPS;
            if constexpr (last && MORE > 0) lin_stage_barrier<MORE == 2 ? NA : 0>();  // the next stage is there, and nobody reads this one any more
            __builtin_amdgcn_sched_barrier(0);
            lin_each<0, SLOTS>([&](auto slot) __attribute__((always_inline)) {
                constexpr int m = decltype(slot)::value, o0 = m * PIECES / READ_SLOTS, o1 = (m + 1) * PIECES / READ_SLOTS;
                if constexpr (!last || MORE > 0)
                    lin_each<(o0 < PIECES ? o0 : PIECES), (o1 < PIECES ? o1 : PIECES)>([&](auto o) __attribute__((always_inline)) {
                        piece(o, last ? a_next : a_now, last ? TileB::BYTES - b_now : b_now, last ? 0 : st + 1, (st + 1) & 1);
                    });
                if constexpr (MORE == 2 && last)
                    lin_each<m * NB / SLOTS, (m + 1) * NB / SLOTS>([&](auto j) __attribute__((always_inline)) { load_b(from_b, from_other, lds_base + B_PLACE + b_now, decltype(j)::value); });
                if constexpr (MORE == 2 && st == 0)
                    lin_each<m * NA / SLOTS, (m + 1) * NA / SLOTS>([&](auto j) __attribute__((always_inline)) { load_a(from_a, lds_base + a_free, decltype(j)::value); });
                constexpr int i = m / (FB * PRODUCTS), t = m / FB % PRODUCTS, j = m % FB;
                acc[i][j] = lin_mfma<In>(a[st & 1][i], b[st & 1][j], acc[i][j], t);
                __builtin_amdgcn_sched_barrier(0);
            });
        });
        const unsigned was = a_now;
        a_now = a_next, a_next = a_free, a_free = was;
        b_now = TileB::BYTES - b_now;
        from_a += KS * (TURN_A ? g.lda : In::SIZE), from_b += KS * (TURN_B ? g.ldb : In::SIZE), from_other += KS * (TURN_B ? g.ldb : In::SIZE);
    };
    for (int s = 0; s + 2 < count; ++s) stage(LinIs<2>());
    if (count > 1) stage(LinIs<1>());
    stage(LinIs<0>());

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
    // through the LDS, 64 rows at a time, every wavefront in a place of its own: a lane then has eight columns of a row
    constexpr int W = FB * 32, LD = W + 4, COLUMNS = GATED ? HALF : W, LANES = COLUMNS / 8, ROWS = 64 / LANES, TURNS = 4;  // lanes of a row, rows at a time
    static_assert(FA % 2 == 0 && 64 % (ROWS * TURNS) == 0 && WAVES * 64 * LD * 4 <= 3 * TileA::BYTES + 2 * TileB::BYTES, "fits the stages");
    lin_stage_barrier<0>();
    float *mine = reinterpret_cast<float *>(lds) + wave * 64 * LD;
    const int width = GATED ? g.end.F : g.end.C, begin = c0 + (GATED ? wc / 2 : wc), col = lane % LANES * 8, c = begin + col;
    const LinColumns<Out, GATED> columns(g.end, g.end.vec ? c : width);
    lin_each<0, FA / 2>([&](auto phase) __attribute__((always_inline)) {
        constexpr int i0 = 2 * decltype(phase)::value;
        const int first_row = r0 + wr + i0 * 32;
        DlVec<Out, 8> next[TURNS];  // residuals, asked for a round ahead
        float next_scale[TURNS];
        const auto ask = [&](int row) __attribute__((always_inline)) {
#pragma unroll
            for (int t = 0; t < TURNS; ++t) {
                const int r = first_row + row + t * ROWS;
                next[t] = lin_residual<Out>(g.end, row < 64 ? width : 0, r, c);
                next_scale[t] = g.end.row_scale && r < g.end.R ? g.end.row_scale[r] : 1.0f;
            }
        };
        if (g.end.vec) ask(lane / LANES);
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < FB; ++j)
#pragma unroll
                for (int v = 0; v < 16; ++v) mine[(i * 32 + (v & 3) + 8 * (v >> 2) + 4 * kh) * LD + j * 32 + l32] = acc[i0 + i][j][v];
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        if (g.end.vec) {
#pragma unroll 1
            for (int row = lane / LANES; row < 64; row += ROWS * TURNS) {
                DlVec<Out, 8> res[TURNS];
                float scale[TURNS];
#pragma unroll
                for (int t = 0; t < TURNS; ++t) res[t] = next[t], scale[t] = next_scale[t];
                ask(row + ROWS * TURNS);
#pragma unroll
                for (int t = 0; t < TURNS; ++t) {
                    const float *at = mine + (row + t * ROWS) * LD + col;
                    float v[8], u[8];
                    *reinterpret_cast<float4 *>(v) = *reinterpret_cast<const float4 *>(at);
                    *reinterpret_cast<float4 *>(v + 4) = *reinterpret_cast<const float4 *>(at + 4);
                    if (GATED) {
                        *reinterpret_cast<float4 *>(u) = *reinterpret_cast<const float4 *>(at + HALF);
                        *reinterpret_cast<float4 *>(u + 4) = *reinterpret_cast<const float4 *>(at + HALF + 4);
                    }
                    lin_finish<Out, GATED>(g.end, columns, first_row + row + t * ROWS, c, v, u, scale[t], res[t]);
                }
            }
        } else {
#pragma unroll 1
            for (int e = lane; e < 64 * COLUMNS; e += 64) {
                const float *at = mine + e / COLUMNS * LD + e % COLUMNS;
                lin_finish_one<Out, GATED>(g.end, first_row + e / COLUMNS, begin + e % COLUMNS, at[0], GATED ? at[HALF] : 0.0f);
            }
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    });
}

// The sums of a reduction that was split, in order, and what follows
template <typename Out, bool GATED>
__global__ __launch_bounds__(256) void lin_join(LinArgs g, int splits) {
    const int width = GATED ? g.end.F : g.end.C, per = g.end.vec ? 8 : 1, units = width / per;
    const long long total = (long long)g.end.R * units, plane = (long long)g.end.R * g.end.C;
    for (long long e = (long long)blockIdx.x * 256 + threadIdx.x; e < total; e += (long long)gridDim.x * 256) {
        const int r = (int)(e / units), c = (int)(e % units) * per;
        const float *at = g.part + (long long)r * g.end.C + c;
        if (!g.end.vec) {
            float v = 0.0f, u = 0.0f;
#pragma unroll 4
            for (int s = 0; s < splits; ++s) {
                v += at[s * plane];
                if (GATED) u += at[s * plane + g.end.F];
            }
            lin_finish_one<Out, GATED>(g.end, r, c, v, u);
            continue;
        }
        float v[8], u[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = u[i] = 0.0f;
        const DlVec<Out, 8> res = lin_residual<Out>(g.end, width, r, c);
#pragma unroll 4
        for (int s = 0; s < splits; ++s) {
            float p[8], q[8];
            dl_load<float, 8>(at + s * plane, p);
            if (GATED) dl_load<float, 8>(at + s * plane + g.end.F, q);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                v[i] += p[i];
                if (GATED) u[i] += q[i];
            }
        }
        lin_finish<Out, GATED>(g.end, LinColumns<Out, GATED>(g.end, c), r, c, v, u, g.end.row_scale ? g.end.row_scale[r] : 1.0f, res);
    }
}

// ------------------------------------------------------------------ launches
struct LinPlan {
    int tile_rows, tile_cols;
    int splits, chunk;  // parts of the reduction, and their stages
    size_t a_bytes, b_bytes, part_bytes;
    size_t bytes() const { return a_bytes + b_bytes + part_bytes; }
};
template <typename In, typename Out, int TR, int TC, bool TURN_A, bool TURN_B, bool GATED, bool PARTIAL>
static int lin_go(const LinArgs &g, int splits, hipStream_t s) {
    constexpr int BYTES = (3 * TR + 2 * TC) * LIN_STAGE_BYTES;
    const long long blocks = (long long)splits * DL_XCDS * dl_ceil_div((long long)g.row_tiles * g.col_tiles, DL_XCDS);
    if (!dl_grid_ok(blocks, 256)) return DL_ERR_UNSUPPORTED;
    const auto kernel = lin_product<In, Out, TR, TC, TURN_A, TURN_B, GATED, PARTIAL>;
    if (BYTES > 65536) {
        const hipError_t room = hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, BYTES);
        if (room != hipSuccess) return (int)room;
    }
    DL_TIMED("lin_product", s, hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(256), BYTES, s, g));
    return DL_OK;
}
template <typename In, typename Out, int T, bool TURN_A, bool TURN_B>
static int lin_launch_tile(const LinArgs &g, int splits, bool gated, hipStream_t s) {
    if (splits > 1) return lin_go<In, Out, T, T, TURN_A, TURN_B, false, true>(g, splits, s);
    if constexpr (!TURN_A && !TURN_B)
        if (gated) return lin_go<In, Out, T, T, false, false, true, false>(g, splits, s);
    return lin_go<In, Out, T, T, TURN_A, TURN_B, false, false>(g, splits, s);
}
template <typename In, typename Out, bool TURN_A, bool TURN_B>
static int lin_launch(LinArgs &g, const LinPlan &p, bool gated, hipStream_t s) {
    const int code = p.tile_rows == 256 ? lin_launch_tile<In, Out, 256, TURN_A, TURN_B>(g, p.splits, gated, s) : lin_launch_tile<In, Out, 128, TURN_A, TURN_B>(g, p.splits, gated, s);
    if (code != DL_OK || p.splits == 1) return code;
    const long long blocks = ((long long)g.end.R * ((gated ? g.end.F : g.end.C) / (g.end.vec ? 8 : 1)) + 255) / 256;
    const dim3 grid((unsigned)(blocks < 16384 ? blocks : 16384));
    if (gated) DL_TIMED("lin_join", s, hipLaunchKernelGGL((lin_join<Out, true>), grid, dim3(256), 0, s, g, p.splits));
    else DL_TIMED("lin_join", s, hipLaunchKernelGGL((lin_join<Out, false>), grid, dim3(256), 0, s, g, p.splits));
    return DL_OK;
}
// (forward: neither is turned; gx: the second; gw: both)
template <typename In, typename Out>
static int lin_launch_turned(LinArgs &g, const LinPlan &p, bool turn_a, bool turn_b, bool gated, hipStream_t s) {
    if (turn_a) return lin_launch<In, Out, true, true>(g, p, gated, s);
    return turn_b ? lin_launch<In, Out, false, true>(g, p, gated, s) : lin_launch<In, Out, false, false>(g, p, gated, s);
}

// One translation unit for every type of operands
int lin_launch_f32(LinArgs &g, const LinPlan &p, bool turn_a, bool turn_b, bool gated, hipStream_t s);
int lin_launch_bf16(LinArgs &g, const LinPlan &p, bool turn_a, bool turn_b, bool gated, hipStream_t s);
int lin_launch_f16(LinArgs &g, const LinPlan &p, bool turn_a, bool turn_b, bool gated, hipStream_t s);
int lin_launch_e4m3(LinArgs &g, const LinPlan &p, int out_type, bool gated, hipStream_t s);
