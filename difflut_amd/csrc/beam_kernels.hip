// A step of beam search: the best continuations of every sequence's beams over the vocabulary, and the beams' states in their order.
//
//   candidate (k, v) of a sequence:  c = scores[k] + logits[k, v] - log sum_u exp(logits[k, u]);  a beam that has ended: (k, end) alone, c = scores[k]
//   the `count` largest, equal ones by k, then v
//
// The best of all are among the best `count` logits of each beam.  One pass over the logits: a block takes a row or a piece of one in
// rounds of BEAM_ROUND, keeps the running maximum and sum of the softmax (float within a round, double over rounds) and a list of what
// may be among the best in the LDS.  The first round bounds them from below - of the threads' largest logits the count-th is passed by
// `count` values at least - later ones append what passes the bound, a few values a round; a list that grows is cut to the best
// and the bound raised to the last of these.  A second launch joins the pieces and picks among the rows' lists.
// Values are compared as doubles, c from double logarithms, so that neighbours of different beams stand in the right order.
#include "dl_types.h"

#define BEAM_THREADS 256
#define BEAM_PER_THREAD 16
#define BEAM_ROUND (BEAM_THREADS * BEAM_PER_THREAD)
#define BEAM_CUT 512       // list length from which it is cut
#define BEAM_RANK 1024     // list length up to which ranks are counted
#define BEAM_MOST 64       // beams, and answers
#define BEAM_PICKS 4096    // candidates that the second launch takes
#define BEAM_LOG2E 1.44269504f

typedef unsigned long long beam_key;  // the logit's order above, the index's order (lowest first) below; 0: none

__device__ __forceinline__ beam_key beam_make(float v, uint32_t i) {
    const uint32_t b = __float_as_uint(v + 0.0f);  // (one zero)
    return (beam_key)(b & 0x80000000u ? ~b : b | 0x80000000u) << 32 | (0xFFFFFFFFu - i);
}
__device__ __forceinline__ float beam_value(beam_key k) {
    const uint32_t b = (uint32_t)(k >> 32);
    return __uint_as_float(b & 0x80000000u ? b & 0x7FFFFFFFu : ~b);
}
__device__ __forceinline__ uint32_t beam_index(beam_key k) { return 0xFFFFFFFFu - (uint32_t)k; }

// what a piece of a row is for the join
struct BeamPart {
    double sum;  // of exp(logit - largest)
    float largest;
    int pad;
};

struct BeamArgs {
    const void *logits;
    long long ldl;
    const float *scores;
    const uint8_t *ended;
    long long end;
    float *out_scores;
    long long *parents, *tokens;
    BeamPart *parts;  // [B K][pieces]
    beam_key *keys;   // [B K][pieces][count], best first
    int B, K, V, count, pieces, piece;
};

// The best `count` of the list's n keys, in order, to out (LDS or device memory; past n: 0).  Every thread of the block; the list is left as it was.
__device__ void beam_select(const beam_key *list, int n, int count, beam_key *out, beam_key *best) {
    const int tid = threadIdx.x;
    if (n <= BEAM_RANK) {  // every key counts the better ones
        for (int e = tid; e < n; e += BEAM_THREADS) {
            const beam_key mine = list[e];
            int rank = 0;
            for (int j = 0; j < n; ++j) rank += list[j] > mine ? 1 : 0;
            if (rank < count) out[rank] = mine;
        }
        for (int e = n + tid; e < count; e += BEAM_THREADS) out[e] = 0;
        return;
    }
    beam_key below = ~0ull;  // the largest below the last one found, `count` times
    for (int k = 0; k < count; ++k) {
        beam_key mine = 0;
        for (int e = tid; e < n; e += BEAM_THREADS) {
            const beam_key v = list[e];
            if (v < below && v > mine) mine = v;
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            const beam_key v = __shfl_xor(mine, o);
            mine = v > mine ? v : mine;
        }
        if ((tid & 63) == 0) best[tid >> 6] = mine;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < BEAM_THREADS / 64; ++w) mine = best[w] > mine ? best[w] : mine;
        __syncthreads();
        if (tid == 0) out[k] = mine;
        below = mine;
    }
}

template <typename T, int E>
__global__ __launch_bounds__(BEAM_THREADS) void beam_rows(BeamArgs g) {
    constexpr int Q = BEAM_PER_THREAD / E;
    __shared__ beam_key list[BEAM_CUT + BEAM_ROUND], chosen[BEAM_MOST], best[BEAM_THREADS / 64];
    __shared__ float tops[BEAM_THREADS], bound_of;
    __shared__ double sums[BEAM_THREADS / 64];
    __shared__ int length;
    const int tid = threadIdx.x;
    const long long row = blockIdx.x / g.pieces;
    const int piece = blockIdx.x % g.pieces;
    if (g.ended && g.ended[row]) return;
    const T *logits = (const T *)g.logits + row * g.ldl;
    const int v0 = piece * g.piece, v1 = min(v0 + g.piece, g.V);
    const float inf = __builtin_inff();

    float next[Q][E];
    auto fetch = [&](int at) __attribute__((always_inline)) {
#pragma unroll
        for (int q = 0; q < Q; ++q) {
            const int c = at + (q * BEAM_THREADS + tid) * E;
            if (c < v1) dl_load<T, E>(logits + c, next[q]);
            else
#pragma unroll
                for (int i = 0; i < E; ++i) next[q][i] = -inf;
        }
    };
    if (tid == 0) length = 0;
    float largest = -inf, bound = -inf;
    beam_key past = 0;  // keys up to it are out
    double sum = 0.0;
    fetch(v0);
    for (int at = v0; at < v1; at += BEAM_ROUND) {
        float v[Q][E], top = -inf;
#pragma unroll
        for (int q = 0; q < Q; ++q)
#pragma unroll
            for (int i = 0; i < E; ++i) {
                const float x = next[q][i];
                v[q][i] = x != x ? -inf : fminf(x, 3.4028234663852886e38f);  // NaN: no candidate; infinity: the largest number
                top = fmaxf(top, v[q][i]);
            }
        if (at + BEAM_ROUND < v1) fetch(at + BEAM_ROUND);
        if (top > largest) {
            sum *= (double)__builtin_amdgcn_exp2f((largest - top) * BEAM_LOG2E);
            largest = top;
        }
        if (largest > -inf) {
            float part = 0.0f;
#pragma unroll
            for (int q = 0; q < Q; ++q)
#pragma unroll
                for (int i = 0; i < E; ++i) part += __builtin_amdgcn_exp2f((v[q][i] - largest) * BEAM_LOG2E);
            sum += (double)part;
        }
        if (at == v0) {
            tops[tid] = top;
            if (tid == 0) bound_of = -inf;
            __syncthreads();
            int rank = 0;
            for (int j = 0; j < BEAM_THREADS; ++j) rank += tops[j] > top || (tops[j] == top && j < tid) ? 1 : 0;
            if (rank == g.count - 1) bound_of = top;
            __syncthreads();
            bound = bound_of;
        }
        if (top >= bound && top > -inf) {
#pragma unroll
            for (int q = 0; q < Q; ++q)
#pragma unroll
                for (int i = 0; i < E; ++i) {
                    if (!(v[q][i] >= bound && v[q][i] > -inf)) continue;
                    const beam_key key = beam_make(v[q][i], (uint32_t)(at + (q * BEAM_THREADS + tid) * E + i));
                    if (key > past) list[atomicAdd(&length, 1)] = key;
                }
        }
        __syncthreads();
        const int n = length;
        __syncthreads();
        if (n > BEAM_CUT) {  // (then there are more than `count`)
            beam_select(list, n, g.count, chosen, best);
            __syncthreads();
            if (tid < g.count) list[tid] = chosen[tid];
            past = chosen[g.count - 1], bound = beam_value(past);
            if (tid == 0) length = g.count;
            __syncthreads();
        }
    }
    const int n = length;
    beam_select(list, n, g.count, g.keys + (row * g.pieces + piece) * g.count, best);

    // the threads' sums, on one maximum, in a fixed order
    float most = largest;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor(most, o));
    __syncthreads();
    if ((tid & 63) == 0) tops[tid >> 6] = most;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < BEAM_THREADS / 64; ++w) most = fmaxf(most, tops[w]);
    sum = largest > -inf ? sum * exp((double)largest - (double)most) : 0.0;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
    if ((tid & 63) == 0) sums[tid >> 6] = sum;
    __syncthreads();
    if (tid == 0) {
        sum = 0.0;
        for (int w = 0; w < BEAM_THREADS / 64; ++w) sum += sums[w];
        g.parts[row * g.pieces + piece] = {sum, most, 0};
    }
}

// A block of THREADS takes a sequence's K * pieces * count candidates.
template <int THREADS>
__global__ __launch_bounds__(THREADS) void beam_pick(BeamArgs g) {
    __shared__ double value[BEAM_PICKS], norm[BEAM_MOST], wave_value[THREADS / 64];
    __shared__ int wave_at[THREADS / 64];
    const int tid = threadIdx.x, b = blockIdx.x, per = g.pieces * g.count, n = g.K * per;
    const double inf = __builtin_inf();
    if (tid < g.K) {
        const long long row = (long long)b * g.K + tid;
        double result = inf;  // nothing to go on with
        if (!(g.ended && g.ended[row])) {
            const BeamPart *p = g.parts + row * g.pieces;
            float most = -__builtin_inff();
            for (int i = 0; i < g.pieces; ++i) most = fmaxf(most, p[i].largest);
            if (most > -__builtin_inff()) {
                double sum = 0.0;
                for (int i = 0; i < g.pieces; ++i)
                    if (p[i].sum > 0.0) sum += p[i].sum * exp((double)p[i].largest - (double)most);
                result = (double)most + log(sum);
            }
        }
        norm[tid] = result;
    }
    __syncthreads();
    const beam_key *keys = g.keys + (long long)b * n;
    double mine = -inf;
    int mine_at = n;
    for (int e = tid; e < n; e += THREADS) {
        const int k = e / per;
        const long long row = (long long)b * g.K + k;
        double c = -inf;
        if (g.ended && g.ended[row]) {
            if (e == k * per) c = (double)g.scores[row];
        } else {
            const beam_key key = keys[e];
            if (key) c = (double)g.scores[row] + ((double)beam_value(key) - norm[k]);
        }
        if (c != c) c = -inf;
        value[e] = c;
        if (c > mine) mine = c, mine_at = e;
    }
    for (int j = 0; j < g.count; ++j) {
        // the largest, the first of equal ones
        double best = mine;
        int at = mine_at;
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            const double v = __shfl_xor(best, o);
            const int w = __shfl_xor(at, o);
            if (v > best || (v == best && w < at)) best = v, at = w;
        }
        if (THREADS > 64) {
            if ((tid & 63) == 0) wave_value[tid >> 6] = best, wave_at[tid >> 6] = at;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < THREADS / 64; ++w)
                if (wave_value[w] > best || (wave_value[w] == best && wave_at[w] < at)) best = wave_value[w], at = wave_at[w];
            __syncthreads();
        }
        const bool none = at >= n || best == -inf;
        if (tid == 0) {
            const long long out = (long long)b * g.count + j;
            const int k = none ? 0 : at / per;
            const long long row = (long long)b * g.K + k;
            g.out_scores[out] = (float)best;
            g.parents[out] = k;
            g.tokens[out] = none ? -1 : g.ended && g.ended[row] ? g.end : (long long)beam_index(keys[at]);
        }
        if (!none && at % THREADS == tid) {  // its next one
            value[at] = -inf;
            mine = -inf, mine_at = n;
            for (int e = tid; e < n; e += THREADS)
                if (value[e] > mine) mine = value[e], mine_at = e;
        }
    }
}

// ------------------------------------------------------------------ states
struct BeamStates {
    const char *src[DL_BEAM_STATES];
    char *dst[DL_BEAM_STATES];
    long long row_bytes[DL_BEAM_STATES], first[DL_BEAM_STATES + 1];  // first block of each tensor
    int unit[DL_BEAM_STATES], pieces[DL_BEAM_STATES];
    const long long *parents;
    int B, K, count, n;
};
#define BEAM_COPY (BEAM_THREADS * 16 * 4)  // bytes of a block
template <typename U>
__device__ __forceinline__ void beam_copy(const char *src, char *dst, long long from, long long to) {
    for (long long at = from + (long long)threadIdx.x * sizeof(U); at < to; at += BEAM_THREADS * sizeof(U)) {
        U v{};
        if (src) v = *reinterpret_cast<const U *>(src + at);
        *reinterpret_cast<U *>(dst + at) = v;
    }
}
__global__ __launch_bounds__(BEAM_THREADS) void beam_states(BeamStates g) {
    int t = 0;
    while (t + 1 < g.n && (long long)blockIdx.x >= g.first[t + 1]) ++t;
    const long long block = (long long)blockIdx.x - g.first[t], out = block / g.pieces[t], b = out / g.count, bytes = g.row_bytes[t];
    const long long parent = g.parents[out];
    const bool known = parent >= 0 && parent < g.K;  // others: zeros
    const char *src = known ? g.src[t] + (b * g.K + parent) * bytes : nullptr;
    char *dst = g.dst[t] + out * bytes;
    const long long from = block % g.pieces[t] * BEAM_COPY, to = from + BEAM_COPY < bytes ? from + BEAM_COPY : bytes;
    if (g.unit[t] == 16) beam_copy<uint4>(src, dst, from, to);
    else if (g.unit[t] == 4) beam_copy<uint32_t>(src, dst, from, to);
    else beam_copy<uint8_t>(src, dst, from, to);
}

// ------------------------------------------------------------------ entry points
// Pieces of a row: enough blocks for the chip, whole rounds, no more candidates than the second launch takes
static void beam_split(BeamArgs &g) {
    const long long rows = (long long)g.B * g.K;
    const long long rounds = ((long long)g.V + BEAM_ROUND - 1) / BEAM_ROUND;
    long long pieces = (1024 + rows - 1) / rows;
    if (pieces > rounds) pieces = rounds;
    if (pieces > BEAM_PICKS / (g.K * g.count)) pieces = BEAM_PICKS / (g.K * g.count);
    if (pieces < 1) pieces = 1;
    const long long per = (rounds + pieces - 1) / pieces;
    g.piece = (int)(per * BEAM_ROUND), g.pieces = (int)((rounds + per - 1) / per);
}
static int beam_check(int type, int B, int K, int V, int count) {
    if (B <= 0 || K <= 0 || V <= 0 || count <= 0) return DL_ERR_SHAPE;
    if (!dl_type_known(type) || K > BEAM_MOST || count > BEAM_MOST || V > 1 << 30) return DL_ERR_UNSUPPORTED;
    return dl_grid_ok((long long)B * K * 1024, 1) ? DL_OK : DL_ERR_UNSUPPORTED;
}
static size_t beam_parts_bytes(const BeamArgs &g) { return dl_align256((size_t)g.B * g.K * g.pieces * sizeof(BeamPart)); }

extern "C" size_t dl_beam_step_workspace_bytes(int B, int K, int V, int count) {
    if (beam_check(DL_F32, B, K, V, count) != DL_OK) return 0;
    BeamArgs g{};
    g.B = B, g.K = K, g.V = V, g.count = count;
    beam_split(g);
    return beam_parts_bytes(g) + dl_align256((size_t)B * K * g.pieces * count * sizeof(beam_key));
}

extern "C" int dl_beam_step(const void *logits, long long ldl, int type, const float *scores, const uint8_t *ended, long long end, float *out_scores,
                            long long *parents, long long *tokens, void *ws, size_t ws_bytes, int B, int K, int V, int count, void *stream) {
    if (!logits || !scores || !out_scores || !parents || !tokens || !ws) return DL_ERR_NULL;
    const int bad = beam_check(type, B, K, V, count);
    if (bad) return bad;
    if (ldl < V) return DL_ERR_SHAPE;
    if (ws_bytes < dl_beam_step_workspace_bytes(B, K, V, count) || !dl_aligned16(ws)) return DL_ERR_WORKSPACE;
    BeamArgs g{};
    g.logits = logits, g.ldl = ldl, g.scores = scores, g.ended = ended, g.end = end, g.out_scores = out_scores, g.parents = parents, g.tokens = tokens;
    g.B = B, g.K = K, g.V = V, g.count = count;
    beam_split(g);
    g.parts = (BeamPart *)ws, g.keys = (beam_key *)((char *)ws + beam_parts_bytes(g));
    const long long blocks = (long long)B * K * g.pieces;
    if (!dl_grid_ok(blocks, BEAM_THREADS)) return DL_ERR_UNSUPPORTED;
    const hipStream_t s = (hipStream_t)stream;
    DL_BY_TYPE(type, T, {
        constexpr int E = 16 / sizeof(T);
        if (V % E == 0 && ldl % E == 0 && dl_aligned16(logits))
            DL_TIMED("beam_rows", s, hipLaunchKernelGGL((beam_rows<T, E>), dim3((unsigned)blocks), dim3(BEAM_THREADS), 0, s, g));
        else
            DL_TIMED("beam_rows", s, hipLaunchKernelGGL((beam_rows<T, 1>), dim3((unsigned)blocks), dim3(BEAM_THREADS), 0, s, g));
    });
    if (K * g.pieces * count <= 1024) DL_TIMED("beam_pick", s, hipLaunchKernelGGL((beam_pick<64>), dim3(B), dim3(64), 0, s, g));
    else DL_TIMED("beam_pick", s, hipLaunchKernelGGL((beam_pick<256>), dim3(B), dim3(256), 0, s, g));
    return dl_launch_status();
}

extern "C" int dl_beam_reorder(const void *const *src, void *const *dst, const long long *row_bytes, int n, const long long *parents, int B, int K, int count,
                               void *stream) {
    if (!src || !dst || !row_bytes || !parents) return DL_ERR_NULL;
    if (n <= 0 || B <= 0 || K <= 0 || count <= 0) return DL_ERR_SHAPE;
    if (n > DL_BEAM_STATES) return DL_ERR_UNSUPPORTED;
    BeamStates g{};
    long long blocks = 0;
    for (int t = 0; t < n; ++t) {
        if (!src[t] || !dst[t]) return DL_ERR_NULL;
        if (row_bytes[t] <= 0) return DL_ERR_SHAPE;
        const uintptr_t bits = (uintptr_t)src[t] | (uintptr_t)dst[t] | (uintptr_t)row_bytes[t];
        g.src[t] = (const char *)src[t], g.dst[t] = (char *)dst[t], g.row_bytes[t] = row_bytes[t], g.unit[t] = bits % 16 == 0 ? 16 : bits % 4 == 0 ? 4 : 1;
        const long long pieces = (row_bytes[t] + BEAM_COPY - 1) / BEAM_COPY;
        if (pieces >= 1LL << 31) return DL_ERR_UNSUPPORTED;
        g.pieces[t] = (int)pieces, g.first[t] = blocks;
        blocks += pieces * B * count;
        if (!dl_grid_ok(blocks, BEAM_THREADS)) return DL_ERR_UNSUPPORTED;
    }
    g.first[n] = blocks, g.parents = parents, g.B = B, g.K = K, g.count = count, g.n = n;
    const hipStream_t s = (hipStream_t)stream;
    DL_TIMED("beam_states", s, hipLaunchKernelGGL(beam_states, dim3((unsigned)blocks), dim3(BEAM_THREADS), 0, s, g));
    return dl_launch_status();
}
