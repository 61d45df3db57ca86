// Element types of the operators that take float32, bfloat16 and float16 tensors: loads widen to float, stores round once
// (to nearest, ties to even).
#pragma once
#include "dl_common.h"

typedef __bf16 dl_bf16;
typedef _Float16 dl_f16;

template <typename T, int N>
struct alignas(sizeof(T) * N) DlVec {
    T v[N];
};
template <typename T, int N>
__device__ __forceinline__ void dl_load(const T *p, float (&f)[N]) {
    const DlVec<T, N> t = *reinterpret_cast<const DlVec<T, N> *>(p);
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = (float)t.v[i];
}
template <typename T, int N>
__device__ __forceinline__ void dl_store(T *p, const float (&f)[N]) {
    DlVec<T, N> t;
#pragma unroll
    for (int i = 0; i < N; ++i) t.v[i] = (T)f[i];
    *reinterpret_cast<DlVec<T, N> *>(p) = t;
}

// 16 bytes as they lie in memory (arrays of 16-bit elements would take a register each), and their values
typedef uint32_t dl_words __attribute__((ext_vector_type(4)));
template <typename T, int N>
__device__ __forceinline__ void dl_unpack(dl_words w, float (&f)[N]) {
    static_assert(sizeof(T) * N == 16, "16 bytes");
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < N; ++i) f[i] = __uint_as_float(w[i]);
    } else {
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
            if constexpr (__is_same(T, dl_bf16)) {
                f[2 * i] = __uint_as_float(w[i] << 16);
                f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
            } else {
                f[2 * i] = (float)__builtin_bit_cast(dl_f16, (uint16_t)w[i]);
                f[2 * i + 1] = (float)__builtin_bit_cast(dl_f16, (uint16_t)(w[i] >> 16));
            }
        }
    }
}

// A store past the caches' retention: for results that a launch does not read again and that would push out what it does
template <typename T, int N>
__device__ __forceinline__ void dl_store_past(T *p, const float (&f)[N]) {
    if constexpr (sizeof(T) * N == 16) {
        DlVec<T, N> t;
#pragma unroll
        for (int i = 0; i < N; ++i) t.v[i] = (T)f[i];
        __builtin_nontemporal_store(__builtin_bit_cast(dl_words, t), reinterpret_cast<dl_words *>(p));
    } else {
        dl_store(p, f);
    }
}

static inline bool dl_type_known(int type) { return type == DL_F32 || type == DL_BF16 || type == DL_F16; }
static inline int dl_type_bytes(int type) { return type == DL_F32 ? 4 : 2; }
static inline bool dl_grid_ok(long long blocks, int threads) { return blocks * threads < (1LL << 32); }  // work items of a launch
static inline bool dl_aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

// DL_BY_TYPE(type, T, statement): the statement with T as the element type
#define DL_BY_TYPE(type, T, ...)                    \
    do {                                            \
        if ((type) == DL_F32) {                     \
            typedef float T;                        \
            __VA_ARGS__;                            \
        } else if ((type) == DL_BF16) {             \
            typedef dl_bf16 T;                      \
            __VA_ARGS__;                            \
        } else {                                    \
            typedef dl_f16 T;                       \
            __VA_ARGS__;                            \
        }                                           \
    } while (0)
