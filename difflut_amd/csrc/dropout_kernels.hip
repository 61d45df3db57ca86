// Dropout and bit flips from a counter-based generator; the mask is never stored.
//
// Element e is hit where word e % 4 of Philox 4x32-10 (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as
// 1, 2, 3", 2011) at counter (e / 4, offset) under the key `seed` is below round(p 2^32): whoever knows seed and offset knows
// the mask, so the backward draws it again instead of reading it.
//   zero:  y = hit ? 0 : x / (1 - p)     (a selection: a NaN or infinity in a hit place is gone)
//   flip:  y = hit ? 1 - x : x           (the bit-flip augmentation; noise, so its backward is the identity)
//
// Bound by memory: ten rounds are twenty 32 by 32 bit products per four elements (a quarter of the rate each), about 30 instructions an
// element, hidden behind the loads and stores.  4096 x 16384 bf16: 44 us a direction, 6.1 TB/s (52 with stores that the
// caches keep); 256 x 3136 fp32: 4 us.
#include "dl_types.h"

#define DROP_THREADS 256
#define DROP_UNITS 4  // 16-byte units per thread

struct DropKey {
    uint64_t seed, offset;
};

// Words of one counter.  The key schedule is the same for every thread (scalar registers).
__device__ __forceinline__ void drop_words(uint64_t counter, DropKey k, uint32_t (&w)[4]) {
    uint32_t c0 = (uint32_t)counter, c1 = (uint32_t)(counter >> 32), c2 = (uint32_t)k.offset, c3 = (uint32_t)(k.offset >> 32);
    uint32_t k0 = (uint32_t)k.seed, k1 = (uint32_t)(k.seed >> 32);
#pragma unroll
    for (int round = 0; round < 10; ++round) {
        const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
        c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
        c1 = (uint32_t)b;
        c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
        c3 = (uint32_t)a;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    w[0] = c0, w[1] = c1, w[2] = c2, w[3] = c3;
}

template <bool FLIP>
__device__ __forceinline__ float drop_one(float x, uint32_t word, uint64_t below, float scale) {
    const bool hit = (uint64_t)word < below;
    return FLIP ? (hit ? 1.0f - x : x) : (hit ? 0.0f : x * scale);
}

template <typename T, bool FLIP, bool VEC>
__global__ __launch_bounds__(DROP_THREADS) void dropout_kernel(const T *__restrict__ x, T *__restrict__ y, long long n, uint64_t below,
                                                                float scale, DropKey key, const long long *__restrict__ state,
                                                                long long *__restrict__ used) {
    constexpr int E = 16 / sizeof(T);  // elements per unit: one counter for float32, two for the 16-bit types
    if (state) {
        key.seed = (uint64_t)state[0], key.offset = (uint64_t)state[1];
        if (used && blockIdx.x == 0 && threadIdx.x == 0) used[0] = state[0], used[1] = state[1];
    }
    const long long first = (long long)blockIdx.x * (DROP_THREADS * DROP_UNITS) + threadIdx.x;
#pragma unroll
    for (int u = 0; u < DROP_UNITS; ++u) {
        const long long e = (first + u * DROP_THREADS) * E;
        if (e >= n) return;
        uint32_t w[E];
#pragma unroll
        for (int q = 0; q < E / 4; ++q) {
            uint32_t four[4];
            drop_words((uint64_t)e / 4 + q, key, four);
#pragma unroll
            for (int j = 0; j < 4; ++j) w[4 * q + j] = four[j];
        }
        if (VEC && e + E <= n) {
            float f[E];
            dl_load(x + e, f);
#pragma unroll
            for (int j = 0; j < E; ++j) f[j] = drop_one<FLIP>(f[j], w[j], below, scale);
            dl_store_past(y + e, f);
        } else {
#pragma unroll
            for (int j = 0; j < E; ++j)
                if (e + j < n) y[e + j] = (T)drop_one<FLIP>((float)x[e + j], w[j], below, scale);
        }
    }
}

extern "C" int dl_dropout(const void *x, void *y, int type, long long numel, double p, int mode, unsigned long long seed,
                          unsigned long long offset, const long long *state, long long *used, void *stream) {
    if (!dl_type_known(type) || (mode != DL_DROP_ZERO && mode != DL_DROP_FLIP)) return DL_ERR_UNSUPPORTED;
    if (numel < 0 || !(p >= 0.0 && p <= 1.0)) return DL_ERR_SHAPE;
    if (numel > 0 && (!x || !y)) return DL_ERR_NULL;
    if (numel == 0 && !(state && used)) return DL_OK;
    hipStream_t s = (hipStream_t)stream;
    const uint64_t below = (uint64_t)floor(p * 4294967296.0 + 0.5);
    const float scale = p < 1.0 ? (float)(1.0 / (1.0 - p)) : 0.0f;
    const long long per_block = (long long)DROP_THREADS * DROP_UNITS * (16 / dl_type_bytes(type));
    const long long blocks = numel > 0 ? (numel + per_block - 1) / per_block : 1;
    if (!dl_grid_ok(blocks, DROP_THREADS)) return DL_ERR_UNSUPPORTED;
    const DropKey key = {seed, offset};
    const bool vec = dl_aligned16(x) && dl_aligned16(y);
    dl_prof_begin("dropout", s);
#define LAUNCH(FLIP, VEC) dropout_kernel<T, FLIP, VEC><<<(int)blocks, DROP_THREADS, 0, s>>>((const T *)x, (T *)y, numel, below, scale, key, state, used)
    DL_BY_TYPE(type, T, if (mode == DL_DROP_FLIP) { if (vec) LAUNCH(true, true); else LAUNCH(true, false); }
                        else { if (vec) LAUNCH(false, true); else LAUNCH(false, false); });
#undef LAUNCH
    dl_prof_end(s);
    return dl_launch_status();
}
