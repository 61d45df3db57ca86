// Matrix products with bias, activation, a gate and a residual in the same launch, and their backward pass, on the 16-bit and
// 8-bit matrix cores with fp32 accumulation.
//
//   linear    z[m,n] = sum_k x[m,k] w[n,k] + b[n],   y = act(z) + residual
//   gated     z over 2 F rows of w, gate first:      y[m,f] = act(z[m,f]) z[m,F+f]
//   backward  gz = gy act'(z)   (gated: gz[f] = gy z[F+f] act'(z[f]),  gz[F+f] = gy act(z[f])),  gb = sum_m gz,  gx = gz w,  gw = gz^T x
//   kept for the backward: z.  In 16 bits that and gz would be two roundings, together with the gradient's own three of one size; so of 16-bit types
//   24 bits of a float are kept, as a plane of 16 and one of 8.
//
// One product kernel serves all of them: C[r,c] = sum_k A(r,k) B(c,k).  An operand lies with the reduction along its rows of memory, or
// (w for gx, gz and x for gw) with the reduction across them, and is turned on the way out of the LDS.  Operands whose rows do not
// start on 16 bytes, end inside 16 or lie more than 2^23 bytes apart are copied to rows that do not, by a pass in front of it.
//
// float32 values are cut into three bf16 planes on the way out of the LDS (8 + 8 + 8 significant bits, each the rounding of what the ones
// above left); a product is the six plane products hi*lo, lo*hi, mid*mid, hi*mid, mid*hi, hi*hi, small ones first.  What is left out is
// below 2^-24 of |a b|, what one fp32 multiply-add rounds off (root mean square: below 2^-27).  Six bf16 products at 2.5 PFLOP/s are 417 TFLOP/s of fp32 work
// against 157 on the fp32 matrix cores; 4096^3 takes 600 us (229 TFLOP/s), 2 M N K on the fp32 cores by the library 900.  What bounds it is the cuts'
// instructions, which do not run beside a matrix instruction: 6144 cycles of these a stage of 256 x 256 and 3264 of those are the 4.7 us that one takes.
// (Planes carry no infinities: such a product is NaN.  Nor anything below 2^-133: values under 2^-110 lose their last bits to that.)
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
#define LIN_BF16_MAX 0x1.fep127f  // the largest
#define LIN_CUS 256
enum { LIN_SUMS, LIN_PLAIN, LIN_PLAIN_ODD, LIN_ENDS, LIN_ENDS_ODD, LIN_KEEPS, LIN_KEEPS_ODD };

struct LinF32 { static constexpr int SIZE = 4; };
struct LinBf16 { static constexpr int SIZE = 2; };
struct LinF16 { static constexpr int SIZE = 2; };
struct LinE4m3 { static constexpr int SIZE = 1; };

// (exponential and reciprocal as the hardware has them: an ulp each, and |z| u from the product with log2 e)
__device__ __forceinline__ float lin_sigmoid(float z) { return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * -1.44269504f)); }
__device__ __forceinline__ float lin_relu(float z) { return z > 0.0f || z != z ? z : 0.0f; }
__device__ __forceinline__ float lin_act(float z, int act) {
    if (act == DL_ACT_RELU) return lin_relu(z);
    if (act == DL_ACT_NONE) return z;
    const float s = lin_sigmoid(z);
    return act == DL_ACT_SILU ? z * s : s;
}
// the activation's value and slope
__device__ __forceinline__ float lin_slope(float z, int act, float &value) {
    if (act == DL_ACT_RELU) {
        value = lin_relu(z);
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
    void *y, *kept;             // kept (null: not) for the backward: ldk values a row, gated the other half from `half` on; of 16-bit types their upper halves,
    uint8_t *kept_low;          // and the eight bits below them
    long long ldk;
    int half;
    const void *bias, *res;
    const float *row_scale, *col_scale;  // of 8-bit operands
    long long ldr;
    int R, C, F, act;           // C: rows of w; F: columns of y where gated
    bool vec;                   // whole vectors of eight of everything, aligned
};

// rounded to 24 bits (what comes of 16-bit values carries no NaN that this would turn over)
__device__ __forceinline__ uint32_t lin_kept_bits(float f) { return __float_as_uint(f) + 0x80u; }
template <typename Out, int E>
__device__ __forceinline__ void lin_keep(const LinEnd &g, int r, int c, const float (&f)[E]) {
    const long long at = r * g.ldk + c;
    if constexpr (sizeof(Out) == 4) dl_store<float, E>((float *)g.kept + at, f);
    else {
        DlVec<uint16_t, E> high;
        DlVec<uint8_t, E> low;
#pragma unroll
        for (int i = 0; i < E; ++i) high.v[i] = (uint16_t)(lin_kept_bits(f[i]) >> 16), low.v[i] = (uint8_t)(lin_kept_bits(f[i]) >> 8);
        *reinterpret_cast<DlVec<uint16_t, E> *>((uint16_t *)g.kept + at) = high;
        *reinterpret_cast<DlVec<uint8_t, E> *>(g.kept_low + at) = low;
    }
}

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
        constexpr int H = GATED ? 1 : 0;
        v[i] = fmaf(v[i], row_scale * k.scale[0][i], k.bias[0][i]);
        if (GATED) u[i] = fmaf(u[i], row_scale * k.scale[H][i], k.bias[H][i]);
    }
    if (g.kept) {
        lin_keep<Out, 8>(g, r, c, v);
        if (GATED) lin_keep<Out, 8>(g, r, g.half + c, u);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = lin_act(v[i], g.act);
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
    if (g.kept) {
        const float first[1] = {v}, second[1] = {u};
        lin_keep<Out, 1>(g, r, c, first);
        if (GATED) lin_keep<Out, 1>(g, r, g.half + c, second);
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
    int row_tiles, col_tiles, splits;
    float *part;                 // PARTIAL: sums [splits][R][C]
    LinEnd end;
};
__device__ const uint4 lin_zeros = {0, 0, 0, 0};  // what lies behind a reduction's end

// Loads that bypass the registers: lane l's 16 bytes land at LDS address lds + 16 l.  The compiler does not count them: a stage waits.
// A buffer of no bytes is not read.
__device__ __forceinline__ void lin_to_lds(unsigned lds, intx4 buffer, unsigned voff) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds), "v"(voff), "s"(buffer) : "memory", "m0");
}
__device__ __forceinline__ intx4 lin_buffer(uint64_t at, int size) {  // size: -1, or 0 for none
    return intx4{(int)(uint32_t)at, (int)(uint32_t)(at >> 32), size, DL_BUFFER_WORD3};
}
// what is the same in every lane, in scalar registers also where the compiler works it out in the lanes' (loads above take nothing else)
__device__ __forceinline__ uint64_t lin_scalar(uint64_t v) {
    int low = (int)(uint32_t)v, high = (int)(uint32_t)(v >> 32);
    asm("" : "+v"(low), "+v"(high));
    return (uint64_t)(uint32_t)dl_uniform(high) << 32 | (uint32_t)dl_uniform(low);
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
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ unsigned lin_pk_bf16(float a, float b) {
    typedef float floatx2 __attribute__((ext_vector_type(2)));
    const floatx2 v = {a, b};
    return __builtin_bit_cast(unsigned, __builtin_convertvector(v, bf16x2));
}
// Eight values into planes in five parts: the first plane, what it leaves, the second, what it leaves, the third.  What is left of a value is
// its product with -1 of the plane's pair, and 0 of its neighbour, added to it: exact, and at once from the packed pair.  (Cycles of one wavefront: rounding
// a pair 8.6, such a product 6.4, to unpack or subtract 5.6 each, so a pair takes 51 instead of 71.  The parts keep results away from their use, which
// would cost waits.)  From 2^128 - 2^119 on the first plane's rounding is infinite, and the value's products are NaN; WIDE: these too are cut, by the largest bf16,
// for two instructions a pair more.
template <bool WIDE>
__device__ __forceinline__ void lin_cut(float (&f)[8], int part, LinFragment<LinF32> &out) {
    unsigned low = 0x0000BF80u, high = 0xBF800000u;  // (-1, 0) and (0, -1)
    asm("" : "+s"(low), "+s"(high));  // in registers: as the instruction's own constant -1 the first would stand in the other half
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        int &w = out.w[part / 2][i];
        if (WIDE && part == 0) w = (int)lin_pk_bf16(__builtin_amdgcn_fmed3f(f[2 * i], -LIN_BF16_MAX, LIN_BF16_MAX), __builtin_amdgcn_fmed3f(f[2 * i + 1], -LIN_BF16_MAX, LIN_BF16_MAX));
        else if (part % 2 == 0) w = (int)lin_pk_bf16(f[2 * i], f[2 * i + 1]);
        else {
            f[2 * i] = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, w), __builtin_bit_cast(bf16x2, low), f[2 * i], false);
            f[2 * i + 1] = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, w), __builtin_bit_cast(bf16x2, high), f[2 * i + 1], false);
        }
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
//   u ^ (row / 2 & 7)), so that the sixteen lanes that an LDS read serves at once, one unit of eight even and eight odd rows, find them on
//   different banks.
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
        return !TURNED ? slot ^ (row >> 1 & 7) : SIZE == 2 ? slot ^ (4 * (row & 3)) : slot ^ (8 * (row >> 3 & 1));
    }
};

// The F fragments of 32 rows each, from row `first` of the tile on.  Lane l has row l % 32 of a fragment, and of a step's values along the
// reduction the eight (of 8 bits 2 x 16) at l / 32.  A fragment comes in PER reads; float32 fragments come raw, and are cut a part
// at a time.
template <typename In, int T, bool TURNED, int F>
struct LinReader {
    typedef LinTile<In, T, TURNED> Tile;
    static constexpr int PER = Tile::SIZE == 1 || (Tile::SIZE == 2 && TURNED) ? 2 : 1;
    unsigned at[F];
    unsigned turn;  // the lane's unit of the first step
    __device__ __forceinline__ LinReader(int first, int lane) {
        const int kh = lane >> 5, l32 = lane & 31;
        turn = (unsigned)(((Tile::SIZE == 4 ? 2 * kh : kh) ^ (lane >> 1 & 7)) * 16);
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

__device__ __forceinline__ void lin_lds_done() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }
template <bool FIRST, typename A, typename B>
struct LinChoose { typedef A type; };
template <typename A, typename B>
struct LinChoose<false, A, B> { typedef B type; };

// A wavefront's place in the LDS for 32 rows of WIDTH values on their way to or from memory: units of 16 bytes of a row in turned order, so that
// sixteen rows' units of one column, and sixteen units of one row, lie on different banks.
template <typename T, int WIDTH>
struct LinPlace {
    static constexpr int E = 16 / sizeof(T), UNITS = WIDTH / E, TURNS = 32 * UNITS / 64, BYTES = 32 * WIDTH * (int)sizeof(T), SHARED = UNITS >= 16 ? 0 : UNITS == 8 ? 1 : 2;
    static_assert(UNITS >= 4 && 64 % UNITS == 0, "a lane has the same unit in every turn");
    static __device__ __forceinline__ int spot(int row, int unit) { return (row * UNITS + (unit ^ ((row >> SHARED) & (UNITS >= 16 ? 15 : UNITS - 1)))) * 16; }
    static __device__ __forceinline__ int four(int row, int column) { return spot(row, column / E) + column % E * (int)sizeof(T); }
    // four values from a column that is a multiple of four
    static __device__ __forceinline__ void put(char *place, int row, int column, const float (&f)[4]) { dl_store<T, 4>((T *)(place + four(row, column)), f); }
    static __device__ __forceinline__ void get(const char *place, int row, int column, float (&f)[4]) { dl_load<T, 4>((const T *)(place + four(row, column)), f); }
    // to memory of any alignment: `to` is the place's first value's, `rows` and `columns` are there.  HALVES: the second half of a row goes `apart`
    // further on.  ODD: a row may end inside a unit, which goes value by value, all lanes taking some.
    template <bool ODD, bool HALVES = false>
    static __device__ __forceinline__ void send(const char *place, int lane, T *to, long long ld, int rows, int columns, int apart = 0) {
        constexpr int PART = HALVES ? WIDTH / 2 : WIDTH;
        const int unit = lane % UNITS, column = unit * E % PART, ends = ODD && columns > 0 && columns < PART ? columns % E : 0;
        T *at = to + column + (HALVES && unit * E >= PART ? apart : 0) + lane / UNITS * ld;
        dl_words v[TURNS];
#pragma unroll
        for (int t = 0; t < TURNS; ++t) v[t] = *reinterpret_cast<const dl_words *>(place + spot(t * (64 / UNITS) + lane / UNITS, unit));
        lin_lds_done();  // (all of them are read before the first is written)
        if (rows >= 32 && columns >= PART) {
#pragma unroll
            for (int t = 0; t < TURNS; ++t, at += 64 / UNITS * ld) __builtin_memcpy(at, &v[t], 16);
        } else if (column + E <= columns) {
#pragma unroll
            for (int t = 0; t < TURNS; ++t, at += 64 / UNITS * ld)
                if (t * (64 / UNITS) + lane / UNITS < rows) __builtin_memcpy(at, &v[t], 16);
        }
        if (ends == 0) return;
#pragma unroll 1
        for (int e = lane; e < 32 * ends * (HALVES ? 2 : 1); e += 64) {
            const int half = e / (32 * ends), row = e / ends % 32, i = e % ends, c = columns - ends + i;
            if (row < rows) to[row * ld + half * apart + c] = *reinterpret_cast<const T *>(place + spot(row, (half * PART + c) / E) + c % E * (int)sizeof(T));
        }
    }
    template <bool ODD>
    static __device__ __forceinline__ void keep(char *place, int lane, const dl_words (&v)[TURNS], const T *from, long long ld, int rows, int columns) {
#pragma unroll
        for (int t = 0; t < TURNS; ++t) *reinterpret_cast<dl_words *>(place + spot(t * (64 / UNITS) + lane / UNITS, lane % UNITS)) = v[t];
        const int ends = ODD && columns > 0 && columns < WIDTH ? columns % E : 0;
        if (ends == 0) return;
        lin_lds_done();
#pragma unroll 1
        for (int e = lane; e < 32 * ends; e += 64) {
            const int row = e / ends, c = columns - ends + e % ends;
            if (row < rows) *reinterpret_cast<T *>(place + spot(row, c / E) + c % E * (int)sizeof(T)) = from[row * ld + c];
        }
    }
    // from memory of any alignment: whole units by way of registers, asked for early; then these and the unit that a row ends in into the place
    static __device__ __forceinline__ void fetch(dl_words (&v)[TURNS], int lane, const T *from, long long ld, int rows, int columns) {
        const int column = lane % UNITS * E;
#pragma unroll
        for (int t = 0; t < TURNS; ++t) {
            const int row = t * (64 / UNITS) + lane / UNITS;
            v[t] = dl_words{0, 0, 0, 0};
            if (row < rows && column + E <= columns) __builtin_memcpy(&v[t], from + row * ld + column, 16);
        }
    }
};
// Four values that belong to columns, bias or scales, as they lie
template <typename T>
struct LinFour {
    uint32_t w[sizeof(T)];
    __device__ __forceinline__ float value(int i) const {
        if constexpr (sizeof(T) == 4) return __uint_as_float(w[i]);
        else if constexpr (__is_same(T, dl_bf16)) return __uint_as_float(i % 2 ? w[i / 2] & 0xFFFF0000u : w[i / 2] << 16);
        else return (float)__builtin_bit_cast(dl_f16, (uint16_t)(w[i / 2] >> (i % 2 * 16)));
    }
    __device__ __forceinline__ void again() {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T); ++i) asm volatile("" : "+v"(w[i]));
    }
    // columns from `column` on of the `width` that begin at p + from (p null: `otherwise`); ones that are not there are as the last
    __device__ __forceinline__ void load(const T *p, long long from, int column, int width, bool vec, T otherwise) {
        DlVec<T, 4> v;
#pragma unroll
        for (int i = 0; i < 4; ++i) v.v[i] = otherwise;
        if (p) {
            if (vec) v = *reinterpret_cast<const DlVec<T, 4> *>(p + from + min(column, width - 4));
            else
#pragma unroll
                for (int i = 0; i < 4; ++i) v.v[i] = p[from + min(column + i, width - 1)];
        }
        __builtin_memcpy(w, &v, sizeof(w));
    }
};

// What follows from it is worked out where it is needed, not held through a loop around
__device__ __forceinline__ int lin_anew(int v) {
    asm volatile("" : "+v"(v));
    return v;
}

// A block of four wavefronts makes tiles of TR x TC, a wavefront a quarter of one, in stages of 128 bytes along the reduction: three of A and two of
// B are in the LDS.  A stage has 2 or 4 steps of the matrix cores; a step's fragments are read while the one before is worked on, across
// stages too: by the last step of a stage all of it has been read and the next one has landed.  B's stage after the next is sent for
// then, into the same place, A's one step later, so that loads are spread over the matrix instructions and have a stage's time to land.  One wavefront
// a SIMD issues everything, so reads, loads and (of float32) cuts stand between the matrix instructions in the order written here; left
// to itself the compiler puts the reads in front of their use.  Where the reduction ends inside a stage, that stage comes first.
// WHAT becomes of the sums: LIN_SUMS partial sums, LIN_PLAIN nothing but the result, LIN_ENDS what follows, LIN_KEEPS that and
// what is kept for the backward; ODD: not all is in aligned whole vectors.
// There are as many blocks as the chip holds; one sends for its next tile's first stages before it writes a tile out.
// bf16, 8192^3: 787 us, 1.40 PFLOP/s, a large library product's rate; what bounds it is power: the matrix cores are busy half of the time at 1.8 to 2.2 GHz
// (2.4 without load), in every form tried.  8 bits, 8192 x 4096 x 16384 with silu: 480 us, 2.29 PFLOP/s.  A tile's end takes 5 us where nothing follows
// the product (a stage takes 1.6), 9 with a gate and what is kept: 12544 x 1024 x 8192 gated and kept 267 us, the plain product 187.
// Gated, a wavefront's columns are those of the gate, then the ones that belong to them.
template <typename In, typename Out, int TR, int TC, bool TURN_A, bool TURN_B, bool GATED, int WHAT>
__global__ __launch_bounds__(256, TR * TC > 128 * 128 ? 1 : 2) void lin_product(LinArgs g) {
    extern __shared__ __align__(16) char lds[];
    typedef LinTile<In, TR, TURN_A> TileA;
    typedef LinTile<In, TC, TURN_B> TileB;
    constexpr int WAVES = 4, FA = TR / 64, FB = TC / 64, KS = TileA::KS;
    constexpr int A0 = 0, A1 = TileA::BYTES, B0 = 2 * TileA::BYTES, B1 = B0 + TileB::BYTES, A2 = B1 + TileB::BYTES;  // places; tiles are written out through the last two
    constexpr int NA = TileA::LOADS / WAVES, NB = TileB::LOADS / WAVES, STEPS = In::SIZE == 2 ? 4 : 2, HALF = FB * 16;
    static_assert(STEPS % 2 == 0, "a stage begins in the first of two sets of fragments");
    typedef __attribute__((address_space(3))) char lds_char;
    const unsigned lds_base = (unsigned)(uintptr_t)(lds_char *)lds;
    const int lane = threadIdx.x & 63, wave = dl_uniform(threadIdx.x >> 6);

    // tiles: every XCD takes a run of them, eight rows of tiles at a time, so that its L2 holds what neighbours share; its blocks take turns
    const int tiles = g.row_tiles * g.col_tiles, per = (tiles + DL_XCDS - 1) / DL_XCDS, xcd = blockIdx.x % DL_XCDS, items = per * g.splits, most = GATED ? g.end.F : g.end.C;
    const unsigned band_tiles = 8 * g.col_tiles, band_reciprocal = dl_uniform(0xFFFFFFFFu / band_tiles);  // (its product is short by one at most)
    int item = blockIdx.x / DL_XCDS, r0, c0;
    const auto settle = [&]() __attribute__((always_inline)) {
        for (; item < items; item += gridDim.x / DL_XCDS) {
            const unsigned tile = xcd * per + (g.splits == 1 ? item : item % per);
            if (tile >= (unsigned)tiles) continue;
            unsigned band = __umulhi(tile, band_reciprocal), in_band = tile - band * band_tiles;
            if (in_band >= band_tiles) ++band, in_band -= band_tiles;
            const unsigned band_rows = min(8, g.row_tiles - (int)band * 8), column = band_rows == 8 ? in_band / 8 : in_band / band_rows;
            r0 = (int)(band * 8 + in_band - column * band_rows) * TR, c0 = (int)column * (GATED ? TC / 2 : TC);
            return true;
        }
        return false;
    };
    if (!settle()) return;

    // ---- what this lane fetches of a tile: offsets from its first row and the stage's first value
    int split, first, count, tail;
    unsigned a_off[NA], b_off[NB];
    uint64_t a_first, a_second, b_first, b_second;  // where its first two stages begin; the others follow
    const int whole = (int)(g.K / KS), left = (int)(g.K - (long long)whole * KS);
    const uint64_t a_step = TURN_A ? g.lda * KS : LIN_STAGE_BYTES, b_step = TURN_B ? g.ldb * KS : LIN_STAGE_BYTES, b_half = GATED ? lin_scalar(g.end.F * g.ldb) : 0;
    bool inside = false;  // the offsets are those of a tile that ends at no edge
    const auto place = [&]() __attribute__((always_inline)) {
        split = g.splits == 1 ? 0 : item / per, first = split * g.chunk, count = min(g.stages - first, g.chunk);
        tail = first + count - min(first + count, whole);  // 1: the reduction ends inside the last stage, which comes first
        const char *const a = g.A + (long long)r0 * (TURN_A ? In::SIZE : g.lda), *const b = g.B + (long long)c0 * (TURN_B ? In::SIZE : g.ldb);
        const uint64_t first_stage = first + (count - 1) * tail, second_stage = first + 1 - tail;
        a_first = lin_scalar((uint64_t)a + first_stage * a_step), a_second = lin_scalar((uint64_t)a + second_stage * a_step);
        b_first = lin_scalar((uint64_t)b + first_stage * b_step), b_second = lin_scalar((uint64_t)b + second_stage * b_step);
        const bool ends = r0 + TR > g.end.R || c0 + (GATED ? TC / 2 : TC) > most;
        if (inside && !ends) return;
        inside = !ends;
        const int lane = lin_anew(threadIdx.x & 63);
#pragma unroll
        for (int j = 0; j < NA; ++j) {
            const int row = TileA::row_of(wave + j * WAVES, lane), unit = TileA::unit_of(row, lane);
            a_off[j] = TURN_A ? (unsigned)row * (unsigned)g.lda + (unsigned)min(unit * 16, (g.end.R * In::SIZE + 15) / 16 * 16 - 16 - r0 * In::SIZE)
                              : (unsigned)min(row, g.end.R - 1 - r0) * (unsigned)g.lda + unit * 16;
        }
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            const int row = TileB::row_of(wave + j * WAVES, lane), unit = TileB::unit_of(row, lane);
            // (gated: rows of the tile are HALF of the gate, HALF of the other, and so on)
            const int f = GATED ? row / (2 * HALF) * HALF + row % HALF : row;
            b_off[j] = TURN_B ? (unsigned)row * (unsigned)g.ldb + (unsigned)min(unit * 16, (g.end.C * In::SIZE + 15) / 16 * 16 - 16 - c0 * In::SIZE)
                              : (unsigned)min(f, most - 1 - c0) * (unsigned)g.ldb + unit * 16;
        }
    };
    static_assert(!GATED || (WAVES * TileB::PER <= HALF && HALF % (WAVES * TileB::PER) == 0), "the four wavefronts' loads are of one half");
    constexpr auto other = [](int j) { return GATED && j * WAVES * TileB::PER % (2 * HALF) >= HALF; };
    const auto load_a = [&](intx4 from, unsigned to, int j) __attribute__((always_inline)) { lin_to_lds(to + (wave + j * WAVES) * 1024, from, a_off[j]); };
    const auto load_b = [&](intx4 from, intx4 from_other, unsigned to, int j) __attribute__((always_inline)) {
        lin_to_lds(to + (wave + j * WAVES) * 1024, other(j) ? from_other : from, b_off[j]);
    };

    const auto there = [&](int s) {
        int behind = s - count;
        asm("" : "+s"(behind));  // (as a comparison it would be taken through the lanes' registers)
        return behind >> 31;
    };
    // a tile's first stages: the first of both, the second of A
    const auto begin = [&]() __attribute__((always_inline)) {
        if (tail) {
            const int lane = lin_anew(threadIdx.x & 63);
#pragma unroll
            for (int j = 0; j < NA; ++j) {
                const int row = TileA::row_of(wave + j * WAVES, lane), value = TURN_A ? row : TileA::unit_of(row, lane) * (16 / In::SIZE);
                lin_to_lds_far(lds_base + A0 + (wave + j * WAVES) * 1024, value < left ? (const char *)a_first + a_off[j] : (const char *)&lin_zeros);
            }
#pragma unroll
            for (int j = 0; j < NB; ++j) {
                const int row = TileB::row_of(wave + j * WAVES, lane), value = TURN_B ? row : TileB::unit_of(row, lane) * (16 / In::SIZE);
                lin_to_lds_far(lds_base + B0 + (wave + j * WAVES) * 1024, value < left ? (const char *)b_first + (other(j) ? b_half : 0) + b_off[j] : (const char *)&lin_zeros);
            }
        } else {
#pragma unroll
            for (int j = 0; j < NA; ++j) load_a(lin_buffer(a_first, -1), lds_base + A0, j);
#pragma unroll
            for (int j = 0; j < NB; ++j) load_b(lin_buffer(b_first, -1), lin_buffer(b_first + b_half, -1), lds_base + B0, j);
        }
#pragma unroll
        for (int j = 0; j < NA; ++j) load_a(lin_buffer(a_second, there(1)), lds_base + A1, j);
    };

    const int wr = wave / 2 * (TR / 2), wc = wave % 2 * (TC / 2);
    const LinReader<In, TR, TURN_A, FA> read_a(wr, lane);
    const LinReader<In, TC, TURN_B, FB> read_b(wc, lane);
    floatx16 acc[FA][FB];
    LinFragment<In> a[2][FA], b[2][FB];

    // Side work of a step, one piece after the other: fragments in the order in which the next step takes them (A's first, all of B, the rest of A)
    constexpr bool CUT = __is_same(In, LinF32);
    constexpr int FRAGMENTS = FA + FB, PA = LinReader<In, TR, TURN_A, FA>::PER, PB = LinReader<In, TC, TURN_B, FB>::PER;
    constexpr int PIECES = CUT ? 6 * (FRAGMENTS + 1) : FA * PA + FB * PB, PRODUCTS = CUT ? 6 : 1, SLOTS = FA * FB * PRODUCTS;
    constexpr int READ_SLOTS = CUT ? SLOTS : SLOTS * 3 / 4;  // (the last reads are answered by the next step)
    float raw[2][8];
    const auto piece = [&](auto number, auto wide, unsigned from_a, unsigned from_b, int step, int set) __attribute__((always_inline)) {
        constexpr int o = decltype(number)::value;
        if constexpr (CUT) {  // read a fragment, then cut the one before
            constexpr int f = o / 6, r = o % 6, q = f - 1;
            if constexpr (r == 0 && f < FRAGMENTS) {
                if constexpr (f == 0 || f > FB) read_a.read_raw(lds + from_a, step, f == 0 ? 0 : f - FB, raw[f & 1]);
                else read_b.read_raw(lds + from_b, step, f - 1, raw[f & 1]);
            }
            if constexpr (r > 0 && f > 0) {
                if constexpr (q == 0 || q > FB) lin_cut<decltype(wide)::value>(raw[q & 1], r - 1, a[set][q == 0 ? 0 : q - FB]);
                else lin_cut<decltype(wide)::value>(raw[q & 1], r - 1, b[set][q - 1]);
            }
        } else if constexpr (o < PA) read_a.read(lds + from_a, step, 0, o, a[set][0]);
        else if constexpr (o < PA + FB * PB) read_b.read(lds + from_b, step, (o - PA) / PB, (o - PA) % PB, b[set][(o - PA) / PB]);
        else read_a.read(lds + from_a, step, (o - FB * PB) / PA, (o - FB * PB) % PA, a[set][(o - FB * PB) / PA]);
    };

    unsigned a_now, a_next, a_free, b_now;
    intx4 from_a, from_b, from_other;
    // A stage, FIRST of a tile or another.  What it sends for and reads behind the last one is not there, and not used.
    const auto stage = [&](auto is_first, auto wide) __attribute__((always_inline)) {
        constexpr bool FIRST = decltype(is_first)::value;
        lin_each<0, STEPS>([&](auto step) __attribute__((always_inline)) {
            constexpr int st = decltype(step)::value;
            constexpr bool last = st + 1 == STEPS;
            if constexpr (last) lin_stage_barrier<NA>();  // the next stage is there, and nobody reads this one any more
            __builtin_amdgcn_sched_barrier(0);
            lin_each<0, SLOTS>([&](auto slot) __attribute__((always_inline)) {
                constexpr int m = decltype(slot)::value, o0 = m * PIECES / READ_SLOTS, o1 = (m + 1) * PIECES / READ_SLOTS;
                lin_each<(o0 < PIECES ? o0 : PIECES), (o1 < PIECES ? o1 : PIECES)>([&](auto o) __attribute__((always_inline)) {
                    piece(o, wide, last ? a_next : a_now, last ? B0 + B1 - b_now : b_now, last ? 0 : st + 1, (st + 1) & 1);
                });
                if constexpr (last)
                    lin_each<m * NB / SLOTS, (m + 1) * NB / SLOTS>([&](auto j) __attribute__((always_inline)) { load_b(from_b, from_other, lds_base + b_now, decltype(j)::value); });
                if constexpr (st == 0)
                    lin_each<m * NA / SLOTS, (m + 1) * NA / SLOTS>([&](auto j) __attribute__((always_inline)) { load_a(from_a, lds_base + a_free, decltype(j)::value); });
                constexpr int i = m / (FB * PRODUCTS), t = m / FB % PRODUCTS, j = m % FB;
                if constexpr (FIRST && st == 0 && t == 0) {
                    floatx16 none;
#pragma unroll
                    for (int v = 0; v < 16; ++v) none[v] = 0.0f;
                    acc[i][j] = lin_mfma<In>(b[0][j], a[0][i], none, 0);
                } else acc[i][j] = lin_mfma<In>(b[st & 1][j], a[st & 1][i], acc[i][j], t);
                __builtin_amdgcn_sched_barrier(0);
            });
        });
        const unsigned was = a_now;
        a_now = a_next, a_next = a_free, a_free = was;
        b_now = B0 + B1 - b_now;
    };

    // C: a lane has row lane % 32 of a tile of 32 x 32, and columns (v % 4) + 8 (v / 4) + 4 (lane / 32) of it
    constexpr int W = FB * 32, H = GATED ? FB / 2 : FB;
    constexpr bool PARTIAL = WHAT == LIN_SUMS, PLAIN = WHAT == LIN_PLAIN || WHAT == LIN_PLAIN_ODD, ODD = WHAT != LIN_PLAIN && WHAT != LIN_ENDS && WHAT != LIN_KEEPS, KEEPS = WHAT == LIN_KEEPS || WHAT == LIN_KEEPS_ODD;
    typedef typename LinChoose<PARTIAL, float, Out>::type Stored;
    typedef LinPlace<Stored, W> Products;               // partial sums, results of the backward
    typedef LinPlace<uint16_t, W> KeptHigh;
    typedef LinPlace<uint8_t, W> KeptLow;
    typedef LinPlace<Stored, GATED ? HALF : W> Results;
    constexpr int PLACE = (TileA::BYTES + TileB::BYTES) / WAVES;  // of a wavefront, in the last two places
    static_assert(Products::BYTES <= PLACE && KeptHigh::BYTES + KeptLow::BYTES <= PLACE, "fits the last two places");
    constexpr bool SCALED = In::SIZE == 1;
    static_assert(!PLAIN || (!SCALED && !GATED), "something follows");
    const auto write_plain = [&](int row0, int column0, int plane) __attribute__((always_inline)) {
        const int lane = lin_anew(threadIdx.x & 63), c = column0 + wc;
        Stored *const out = PARTIAL ? (Stored *)(void *)g.part + (long long)plane * g.end.R * g.end.C : (Stored *)g.end.y;
        char *mine = lds + B1 + wave * PLACE;
        lin_each<0, FA>([&](auto phase) __attribute__((always_inline)) {
            constexpr int i = decltype(phase)::value;
            const int r = row0 + wr + i * 32;
            if constexpr (TR * TC > 128 * 128) {
#pragma unroll
                for (int j = 0; j < FB; ++j) asm volatile("" : "+a"(acc[i][j]));  // (no earlier than here out of the accumulators' registers)
            }
#pragma unroll
            for (int j = 0; j < FB; ++j)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const float f[4] = {acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
                    Products::put(mine, lane & 31, j * 32 + 8 * q + 4 * (lane >> 5), f);
                }
            lin_lds_done();
            Products::template send<ODD>(mine, lane, out + (long long)r * g.end.C + c, g.end.C, g.end.R - r, g.end.C - c);
            lin_lds_done();
        });
    };
    const auto write = [&](int row0, int column0) __attribute__((always_inline)) {
        const int lane0 = threadIdx.x & 63;
        const LinEnd &e = g.end;
        char *mine = lds + B1 + wave * PLACE;
        const int width = GATED ? e.F : e.C, c = column0 + (GATED ? wc / 2 : wc), columns = width - c;
        LinFour<Stored> bias[FB][4];
        LinFour<float> scale[SCALED ? FB : 1][4];
        const auto of_columns = [&]() __attribute__((always_inline)) {
            const int first = lin_anew(c + 4 * (lane0 >> 5));
#pragma unroll
            for (int j = 0; j < FB; ++j)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const long long from = (j / H) * (long long)e.F;  // (gated: of the gate's or the other's columns)
                    const int column = first + j % H * 32 + 8 * q;
                    bias[j][q].load((const Stored *)e.bias, from, column, width, !ODD, (Stored)0.0f);
                    if (SCALED) scale[SCALED ? j : 0][q].load(e.col_scale, from, column, width, !ODD, 1.0f);
                }
        };
        constexpr bool HELD = sizeof(Stored) == 2;  // through the tile; more would not fit the registers
        if (HELD) of_columns();
        lin_each<0, FA>([&](auto phase) __attribute__((always_inline)) {
            constexpr int i = decltype(phase)::value;
            const int lane = lin_anew(lane0), kh = lane >> 5, l32 = lane & 31;
            const int r = row0 + wr + i * 32, rows = e.R - r;
            if constexpr (TR * TC > 128 * 128) {
#pragma unroll
                for (int j = 0; j < FB; ++j) asm volatile("" : "+a"(acc[i][j]));  // (no earlier than here out of the accumulators' registers)
            }
            const Stored *const res = (const Stored *)e.res + r * e.ldr + c;
            dl_words residual[Results::TURNS];
            if (e.res && !SCALED) Results::fetch(residual, lane, res, e.ldr, rows, columns);  // (scales take the registers that it would wait in)
            const float row_scale = SCALED ? e.row_scale[min(r + l32, e.R - 1)] : 1.0f;
            if (!HELD) of_columns();
            else {
#pragma unroll
                for (int j = 0; j < FB; ++j)
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        bias[j][q].again();  // (held as words, not as what they become)
                        if (SCALED) scale[SCALED ? j : 0][q].again();
                    }
            }
            float f[FB][16];
#pragma unroll
            for (int j = 0; j < FB; ++j)
#pragma unroll
                for (int v = 0; v < 16; ++v) {
                    const float b = bias[j][v / 4].value(v % 4);
                    f[j][v] = SCALED ? fmaf(acc[i][j][v], row_scale * scale[SCALED ? j : 0][v / 4].value(v % 4), b) : acc[i][j][v] + b;
                }
            const auto keep = [&](int column, const float (&v)[16]) __attribute__((always_inline)) {
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int at = column + 8 * q + 4 * kh;
                    if constexpr (sizeof(Stored) == 4) Products::put(mine, l32, at, {v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]});
                    else {
                        uint32_t w[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) w[i] = lin_kept_bits(v[4 * q + i]);
                        // (selectors: bytes 3 and 2 of both; byte 1 of both)
                        *reinterpret_cast<uint2 *>(mine + KeptHigh::four(l32, at)) = uint2{__builtin_amdgcn_perm(w[1], w[0], 0x07060302), __builtin_amdgcn_perm(w[3], w[2], 0x07060302)};
                        *reinterpret_cast<uint32_t *>(mine + KeptHigh::BYTES + KeptLow::four(l32, at)) =
                            __builtin_amdgcn_perm(__builtin_amdgcn_perm(w[3], w[2], 0x0c0c0501), __builtin_amdgcn_perm(w[1], w[0], 0x0c0c0501), 0x05040100);
                    }
                }
            };
            if constexpr (KEEPS) {
#pragma unroll
                for (int j = 0; j < FB; ++j) keep(j * 32, f[j]);
                const long long at = r * e.ldk + c;
                const int padded = (columns + 15) / 16 * 16;  // (its rows are)
                lin_lds_done();
                if constexpr (sizeof(Stored) == 4) Products::template send<false, GATED>(mine, lane, (Stored *)e.kept + at, e.ldk, rows, padded, e.half);
                else {
                    KeptHigh::template send<false, GATED>(mine, lane, (uint16_t *)e.kept + at, e.ldk, rows, padded, e.half);
                    KeptLow::template send<false, GATED>(mine + KeptHigh::BYTES, lane, e.kept_low + at, e.ldk, rows, padded, e.half);
                }
                lin_lds_done();
            }
            if (e.res) {
                if (SCALED) Results::fetch(residual, lane, res, e.ldr, rows, columns);
                Results::template keep<ODD>(mine, lane, residual, res, e.ldr, rows, columns);
                lin_lds_done();
            }
#pragma unroll
            for (int j = 0; j < H; ++j) {
                const auto follow = [&](int act) __attribute__((always_inline)) {
#pragma unroll
                    for (int v = 0; v < 16; ++v) {
                        f[j][v] = lin_act(f[j][v], act);
                        if (GATED) f[j][v] *= f[j + FB - H][v];
                    }
                };
                if (e.act == DL_ACT_NONE) follow(DL_ACT_NONE);
                else if (e.act == DL_ACT_RELU) follow(DL_ACT_RELU);
                else if (e.act == DL_ACT_SILU) follow(DL_ACT_SILU);
                else follow(DL_ACT_SIGMOID);
                if (e.res) {
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        float r4[4];
                        Results::get(mine, l32, j * 32 + 8 * q + 4 * kh, r4);
#pragma unroll
                        for (int v = 0; v < 4; ++v) f[j][4 * q + v] += r4[v];
                    }
                }
#pragma unroll
                for (int q = 0; q < 4; ++q) Results::put(mine, l32, j * 32 + 8 * q + 4 * kh, {f[j][4 * q], f[j][4 * q + 1], f[j][4 * q + 2], f[j][4 * q + 3]});
            }
            lin_lds_done();
            Results::template send<ODD>(mine, lane, (Stored *)e.y + (long long)r * width + c, width, rows, columns);
            lin_lds_done();
        });
    };

    place();
    begin();
    for (;;) {
        const auto multiply = [&](auto wide) __attribute__((always_inline)) {
            lin_stage_barrier<0>();  // the first stages are there, and the tile before is written out of the LDS
#pragma unroll
            for (int j = 0; j < NB; ++j) load_b(lin_buffer(b_second, there(1)), lin_buffer(b_second + b_half, there(1)), lds_base + B1, j);
            a_now = A0, a_next = A1, a_free = A2, b_now = B0;
            uint64_t at_a = a_second, at_b = b_second;
            const auto send_for = [&](int s) __attribute__((always_inline)) {
                at_a += a_step, at_b += b_step;
                from_a = lin_buffer(at_a, there(s)), from_b = lin_buffer(at_b, there(s)), from_other = lin_buffer(at_b + b_half, there(s));
            };
            lin_each<0, PIECES>([&](auto o) __attribute__((always_inline)) { piece(o, wide, A0, B0, 0, 0); });
            send_for(2);
            stage(LinIs<1>(), wide);
            for (int s = 1; s < count; ++s) {
                send_for(s + 2);
                stage(LinIs<0>(), wide);
            }
        };
        multiply(LinIs<0>());
        if constexpr (CUT) {
            // A value that the planes do not hold makes every sum of its row or column NaN, so one column's and one row's sums show it; then the tile is
            // multiplied again by cuts that hold it.  (In every cut these would take 3 to 7 % of a product's time.)
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < FA; ++i) sum += acc[i][0][0];
#pragma unroll
            for (int j = 0; j < FB; ++j)
#pragma unroll
                for (int v = 0; v < 16; ++v) sum += acc[0][j][v];
            lin_stage_barrier<0>();  // everybody has read the last stage
            int *const marks = (int *)(lds + B1);
            if (lane == 0) marks[wave] = 0;
            if (sum != sum) marks[wave] = 1;
            lin_stage_barrier<0>();
            const int any = dl_uniform(marks[0] | marks[1] | marks[2] | marks[3]);
            lin_stage_barrier<0>();
            if (any) {
                begin();
                multiply(LinIs<1>());
            }
        }

        const int row = r0, column = c0, plane = split;
        item += gridDim.x / DL_XCDS;
        const bool more = settle();
        lin_stage_barrier<0>();  // everybody has read the last stage
        if (more) {
            place();
            begin();
        }
        if constexpr (PARTIAL || PLAIN) write_plain(row, column, plane);
        else write(row, column);
        if (!more) return;
    }
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

// ------------------------------------------------------------------ few rows
// Up to 64 rows of x, a token or some: what counts is that w is read once, at the memory's rate, by as many wavefronts as there are.  A wavefront takes
// 16 rows of w (G times, gated: 16 of the gate and theirs of the other), straight into the registers as the matrix cores take them (four lanes read 64
// bytes of a row); x comes out of the caches.  Of a block's eight wavefronts SHARING have the same rows, every one a step of 64 or 128 bytes in turn; their
// sums are added in order in the LDS, and what follows is done there: one launch, no workspace, rows of any alignment.  A token of 1024 to 131072 in bf16,
// 269 MB: 40 us, 6.7 TB/s (the memory and the last cache).
// Which of those: up to 16 always; up to 32 float32, but for few long rows of w, and of the others what w has up to 2^23 values of; up to 64 that and gated (x
// serves gate and other), not float32.  (us, so and by tiles: bf16 8 x 1024 over 8192 6.8, 11.2, over 131072 52, 51; 32 x 1024 over 8192 8.1, 12.0,
// over 10240 10.5, 10.8, over 12288 10.3, 8.2, over 32768 18, 13; gated 64 x 1024 over 2 x 4096 8.9, 11.7, over 2 x 5120 13.9, 9.8, over 2 x 16384
// 25, 14, 48 x 1024 over 2 x 8192 12.7, 11.6; 64 x 1024 not gated 14, 11; float32 32 x 1024 over 32768 37, 54, 32 x 4096 over 1024 24, 18.)
static inline bool lin_few_rows(long long M, long long N, long long K, int size, bool gated) {
    const bool small = N * K <= 1LL << 23 && K <= 2048;
    return M <= 16 || (M <= 32 && (size == 4 ? K <= 2048 || N >= 4096 : small)) || (M <= 64 && gated && size < 4 && small);
}
typedef float floatx4 __attribute__((ext_vector_type(4)));
template <typename In>
__device__ __forceinline__ floatx4 lin_mfma16(const LinFragment<In> &a, const LinFragment<In> &b, floatx4 c) {
    if constexpr (__is_same(In, LinE4m3)) {
        return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(__builtin_bit_cast(intx8, a), __builtin_bit_cast(intx8, b), c, 0, 0, 0, 0x7f7f7f7f, 0, 0x7f7f7f7f);
    } else if constexpr (__is_same(In, LinBf16)) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    } else if constexpr (__is_same(In, LinF16)) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(halfx8, a), __builtin_bit_cast(halfx8, b), c, 0, 0, 0);
    } else {
        constexpr int PA[6] = {0, 2, 1, 0, 1, 0}, PB[6] = {2, 0, 1, 1, 0, 0};
#pragma unroll
        for (int t = 0; t < 6; ++t)
            c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a.w[PA[t]]), __builtin_bit_cast(bf16x8, b.w[PB[t]]), c, 0, 0, 0);
        return c;
    }
}
template <typename In, typename Out, int MT, int G, bool GATED, int SHARING>
__global__ __launch_bounds__(512) void lin_few(LinArgs g) {
    constexpr int WAVES = 8, Q = In::SIZE == 2 ? 1 : 2, STEP = 64 * Q, ROOM = (MT == 1 ? 12 : 8) / (Q * (G + MT)), U = ROOM > 4 ? 4 : ROOM > 1 ? ROOM : 1;  // steps asked for at once: two such sets fit the registers
    __shared__ float sums[WAVES][G][MT][256];
    struct Raw { uint32_t w[4 * Q]; };
    const int lane = threadIdx.x & 63, wave = dl_uniform(threadIdx.x >> 6), row = lane & 15, unit = (lane >> 4) * 16;
    constexpr int H = GATED ? 1 : G;
    constexpr int GROUPS = WAVES / SHARING;
    const int part = wave % SHARING, group = wave / SHARING, width = GATED ? g.end.F : g.end.C;
    const long long n_first = (long long)blockIdx.x * GROUPS * 16 * H;
    const int n0 = (int)(n_first + group * 16 * H < width ? n_first + group * 16 * H : width - 1);  // (wavefronts without rows go along: there is a barrier)
    const char *w[G], *x[MT];
#pragma unroll
    for (int i = 0; i < G; ++i) w[i] = g.B + (long long)(GATED ? i * g.end.F + min(n0 + row, width - 1) : min(n0 + 16 * i + row, width - 1)) * g.ldb;
#pragma unroll
    for (int t = 0; t < MT; ++t) x[t] = g.A + (long long)min(16 * t + row, g.end.R - 1) * g.lda;
    const long long bytes = g.K * In::SIZE;
    const int whole = (int)(bytes / STEP);
    const auto fetch = [&](const char *from, int step, Raw &to) __attribute__((always_inline)) {
#pragma unroll
        for (int q = 0; q < Q; ++q) __builtin_memcpy(to.w + 4 * q, from + (long long)step * STEP + q * 64 + unit, 16);  // (of any alignment)
    };
    const auto fragment = [&](const Raw &from) __attribute__((always_inline)) {
        LinFragment<In> f;
        if constexpr (__is_same(In, LinF32)) {
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(from.w[i]);
#pragma unroll
            for (int part = 0; part < 5; ++part) lin_cut<true>(v, part, f);  // (it costs nothing here)
        } else {
#pragma unroll
            for (int i = 0; i < 4 * Q; ++i) f.w[0][i] = (int)from.w[i];
        }
        return f;
    };
    floatx4 acc[G][MT];
#pragma unroll
    for (int i = 0; i < G; ++i)
#pragma unroll
        for (int t = 0; t < MT; ++t) acc[i][t] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
    const auto multiply = [&](const Raw (&rw)[G], const Raw (&rx)[MT]) __attribute__((always_inline)) {
        LinFragment<In> fw[G];
#pragma unroll
        for (int i = 0; i < G; ++i) fw[i] = fragment(rw[i]);
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            const LinFragment<In> fx = fragment(rx[t]);
#pragma unroll
            for (int i = 0; i < G; ++i) acc[i][t] = lin_mfma16<In>(fw[i], fx, acc[i][t]);
        }
    };
    Raw rw[2][U][G], rx[2][U][MT];
    const auto batch = [&](int step, int set) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int at = step + u * SHARING;
            if (at < whole) {
#pragma unroll
                for (int i = 0; i < G; ++i) fetch(w[i], at, rw[set][u][i]);
#pragma unroll
                for (int t = 0; t < MT; ++t) fetch(x[t], at, rx[set][u][t]);
            } else {
#pragma unroll
                for (int i = 0; i < G; ++i) rw[set][u][i] = Raw{};
#pragma unroll
                for (int t = 0; t < MT; ++t) rx[set][u][t] = Raw{};
            }
        }
    };
    batch(part, 0);
    for (int step = part; step < whole; step += 2 * U * SHARING) {
        batch(step + U * SHARING, 1);
#pragma unroll
        for (int u = 0; u < U; ++u) multiply(rw[0][u], rx[0][u]);
        batch(step + 2 * U * SHARING, 0);
#pragma unroll
        for (int u = 0; u < U; ++u) multiply(rw[1][u], rx[1][u]);
    }
    if (whole * (long long)STEP < bytes && whole % SHARING == part) {  // the reduction ends inside a step: value by value
        Raw tw[G], tx[MT];
        const auto some = [&](const char *from, Raw &to) __attribute__((always_inline)) {
            to = Raw{};
#pragma unroll
            for (int e = 0; e < 16 * Q / In::SIZE; ++e) {
                const long long at = (long long)whole * STEP + e * In::SIZE / 16 * 64 + unit + e * In::SIZE % 16;
                if (at >= bytes) continue;
                uint32_t v = 0;
                __builtin_memcpy(&v, from + at, In::SIZE);
                to.w[e * In::SIZE / 4] |= v << (e * In::SIZE % 4 * 8);
            }
        };
#pragma unroll
        for (int i = 0; i < G; ++i) some(w[i], tw[i]);
#pragma unroll
        for (int t = 0; t < MT; ++t) some(x[t], tx[t]);
        multiply(tw, tx);
    }
    // a lane has x's row lane % 16, and of w's four from 4 (lane / 16) on
#pragma unroll
    for (int i = 0; i < G; ++i)
#pragma unroll
        for (int t = 0; t < MT; ++t) *reinterpret_cast<floatx4 *>(&sums[wave][i][t][lane * 4]) = acc[i][t];
    __syncthreads();
    for (int e = threadIdx.x; e < 256 * MT * H * GROUPS; e += 512) {
        const int n = e % (16 * H * GROUPS), m = e / (16 * H * GROUPS), i = n / 16 % H, from = n / (16 * H) * SHARING, at = (n % 16 / 4 * 16 + m % 16) * 4 + n % 4;
        float v = 0.0f, u = 0.0f;
        for (int q = 0; q < SHARING; ++q) {
            v += sums[from + q][i][m / 16][at];
            if (GATED) u += sums[from + q][G - 1][m / 16][at];
        }
        if (n_first + n < width) lin_finish_one<Out, GATED>(g.end, m, (int)n_first + n, v, u);
    }
}
template <typename In, typename Out>
static int lin_launch_few(LinArgs &g, bool gated, hipStream_t s) {
    const int width = gated ? g.end.F : g.end.C, rows = g.end.R;
    // 32 rows of w a wavefront where x has more than 16 (its loads serve both) or 1024 have some; two to share them instead of eight where eight would
    // have less than four steps each and 512 blocks are left
    const bool pairs = !gated && (rows > 16 || width >= 1024 * 32);
    const int rows_each = pairs ? 32 : 16;
    const bool two = g.K * In::SIZE < 32 * (In::SIZE == 2 ? 64 : 128) && width >= 512 * 4 * rows_each;
    const long long blocks = dl_ceil_div(width, rows_each * (two ? 4 : 1));
    if (!dl_grid_ok(blocks, 512)) return DL_ERR_UNSUPPORTED;
#define LIN_FEW_GO(MT, G, GATED, SHARING) hipLaunchKernelGGL((lin_few<In, Out, MT, G, GATED, SHARING>), dim3((unsigned)blocks), dim3(512), 0, s, g)
#define LIN_FEW_ROWS(SHARING) \
    do { \
        if (gated) { if (rows <= 16) LIN_FEW_GO(1, 2, true, SHARING); else if (rows <= 32) LIN_FEW_GO(2, 2, true, SHARING); else if constexpr (In::SIZE < 4) LIN_FEW_GO(4, 2, true, SHARING); } \
        else if (rows > 16) LIN_FEW_GO(2, 2, false, SHARING); \
        else if (pairs) LIN_FEW_GO(1, 2, false, SHARING); \
        else LIN_FEW_GO(1, 1, false, SHARING); \
    } while (0)
    DL_TIMED("lin_few", s, if (two) LIN_FEW_ROWS(2); else LIN_FEW_ROWS(8));
#undef LIN_FEW_ROWS
#undef LIN_FEW_GO
    return DL_OK;
}

// ------------------------------------------------------------------ launches
struct LinPlan {
    bool few;    // by lin_few
    int tile;
    int splits, chunk;  // parts of the reduction, and their stages
    size_t a_bytes, b_bytes, part_bytes;
    size_t bytes() const { return a_bytes + b_bytes + part_bytes; }
};
template <typename In, typename Out, int T, bool TURN_A, bool TURN_B, bool GATED, int WHAT>
static int lin_go(const LinArgs &g, hipStream_t s) {
    constexpr int BYTES = 5 * T * LIN_STAGE_BYTES;
    const long long items = (long long)g.splits * DL_XCDS * (((long long)g.row_tiles * g.col_tiles + DL_XCDS - 1) / DL_XCDS), most = LIN_CUS * (T > 128 ? 1 : 2);
    if (items >= 1LL << 30) return DL_ERR_UNSUPPORTED;
    const auto kernel = lin_product<In, Out, T, T, TURN_A, TURN_B, GATED, WHAT>;
    const hipError_t room = hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, BYTES);
    if (room != hipSuccess) return (int)room;
    DL_TIMED("lin_product", s, hipLaunchKernelGGL(kernel, dim3((unsigned)(items < most ? items : most)), dim3(256), BYTES, s, g));
    return DL_OK;
}
// (the backward's products: nothing follows)
template <typename In, typename Out, int T, bool TURN_A, bool TURN_B>
int lin_launch_tile(const LinArgs &g, bool gated, hipStream_t s) {
    const LinEnd &e = g.end;
    if (g.splits > 1) return lin_go<In, Out, T, TURN_A, TURN_B, false, LIN_SUMS>(g, s);
    const bool plain = TURN_B || (!gated && !e.row_scale && !e.bias && !e.res && !e.kept && e.act == DL_ACT_NONE);
    if constexpr (In::SIZE > 1)
        if (plain) return e.vec ? lin_go<In, Out, T, TURN_A, TURN_B, false, LIN_PLAIN>(g, s) : lin_go<In, Out, T, TURN_A, TURN_B, false, LIN_PLAIN_ODD>(g, s);
    if constexpr (!TURN_B) {
        if constexpr (In::SIZE > 1)
            if (e.kept) {
                if (gated) return e.vec ? lin_go<In, Out, T, false, false, true, LIN_KEEPS>(g, s) : lin_go<In, Out, T, false, false, true, LIN_KEEPS_ODD>(g, s);
                return e.vec ? lin_go<In, Out, T, false, false, false, LIN_KEEPS>(g, s) : lin_go<In, Out, T, false, false, false, LIN_KEEPS_ODD>(g, s);
            }
        if (gated) return e.vec ? lin_go<In, Out, T, false, false, true, LIN_ENDS>(g, s) : lin_go<In, Out, T, false, false, true, LIN_ENDS_ODD>(g, s);
        return e.vec ? lin_go<In, Out, T, false, false, false, LIN_ENDS>(g, s) : lin_go<In, Out, T, false, false, false, LIN_ENDS_ODD>(g, s);
    }
    return DL_ERR_UNSUPPORTED;
}
template <typename In, typename Out, bool TURN_A, bool TURN_B>
static int lin_launch(LinArgs &g, const LinPlan &p, bool gated, hipStream_t s) {
    const int code = p.tile == 256 ? lin_launch_tile<In, Out, 256, TURN_A, TURN_B>(g, gated, s) : lin_launch_tile<In, Out, 128, TURN_A, TURN_B>(g, gated, s);
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
    if (p.few) return lin_launch_few<In, Out>(g, gated, s);
    if (turn_a) return lin_launch<In, Out, true, true>(g, p, gated, s);
    return turn_b ? lin_launch<In, Out, false, true>(g, p, gated, s) : lin_launch<In, Out, false, false>(g, p, gated, s);
}

// Translation units: one for every type of operands, where its kernels are few; else these are instantiated in units of their own.
#define LIN_TILE(In, Out, T, TURN_A, TURN_B) template int lin_launch_tile<In, Out, T, TURN_A, TURN_B>(const LinArgs &g, bool gated, hipStream_t s)
int lin_launch_f32(LinArgs &g, const LinPlan &p, bool turn_a, bool turn_b, bool gated, hipStream_t s);
int lin_launch_bf16(LinArgs &g, const LinPlan &p, bool turn_a, bool turn_b, bool gated, hipStream_t s);
int lin_launch_f16(LinArgs &g, const LinPlan &p, bool turn_a, bool turn_b, bool gated, hipStream_t s);
int lin_launch_e4m3(LinArgs &g, const LinPlan &p, int out_type, bool gated, hipStream_t s);
