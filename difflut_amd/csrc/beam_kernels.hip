// A step of beam search: the best continuations of every sequence's beams over the vocabulary, and the beams' states in their order.
//
//   candidate (k, v) of a sequence:  c = scores[k] + logits[k, v] - log sum_u exp(logits[k, u]);  a beam that has ended: (k, end) alone, c = scores[k]
//   the `count` largest, equal ones by k, then logit (they may differ where the scores are so far from zero that c does not), then v
//
// The best of all are among the best `count` logits of each beam.  One pass over the logits: a block takes a row or a piece of one, each of its
// wavefronts in rounds of BEAM_ROUND / 4 values, without waiting for the others.  A thread keeps the sum of the softmax (float within a round,
// double over rounds) on a maximum that it changes only where a logit lies far above; a wavefront keeps a list of what may be among
// the best in the LDS.  The first round bounds them from below - the count-th of the lanes' largest logits is passed by `count` values at
// least - later ones append what passes the bound, a few values a round; a list that grows is cut and the bound raised.  The thresholds are
// searched bit by bit, with a ballot for a count.  A second launch joins the pieces and picks among the rows' lists.
// Values are compared as doubles, c from double logarithms of sums that are right to about 2^-22 (float exponentials; measured: off by up to 2^-22.8, at 1000 logits and
// more 2^-23.2): a beam's continuations stand in the right order always, those of different beams where they are not closer than that.
// 64 x 8 rows of 131072 float32, 268 MB: the pass 45 us (memory), the second launch 9 and the states' order 6 (latency); before, with the block's wavefronts in
// step and a list in common, the pass took 63.
#include "dl_types.h"

#define BEAM_THREADS 256
#define BEAM_WAVES 4
#define BEAM_PER_THREAD 16
#define BEAM_ROUND (BEAM_THREADS * BEAM_PER_THREAD)
#define BEAM_CUT 128       // length from which a wavefront's list is cut, at most
#define BEAM_LIST (BEAM_CUT + 64 * 8)  // and what eight values a lane may append
#define BEAM_MOST 64       // beams, and answers
#define BEAM_PICKS 4096    // candidates that the second launch takes
#define BEAM_LOG2E 1.44269504f
#define BEAM_LOWEST 0x00800000u  // the order of the lowest number; below it is -infinity's

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

__device__ __forceinline__ uint32_t beam_order(beam_key k) { return (uint32_t)(k >> 32); }
// the largest T of which BITS from the top may be set with `count` lanes or more whose values (V a lane) reach it; 0 where there are fewer
template <int BITS, int V>
__device__ __forceinline__ uint32_t beam_threshold(const uint32_t (&order)[V], int count) {
    uint32_t t = 0;
#pragma unroll 4
    for (int bit = 31; bit > 31 - BITS; --bit) {
        const uint32_t higher = t | 1u << bit;
        int n = 0;
#pragma unroll
        for (int i = 0; i < V; ++i) n += __popcll(__ballot(order[i] >= higher));
        if (n >= count) t = higher;
    }
    return t;
}
// a wavefront's own LDS reads and writes, in the order written
__device__ __forceinline__ void beam_in_order() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); }

// A wavefront's list of n keys, cut: to those that reach the count-th value, or where these are too many (equal ones, a long list) to exactly
// `count`.  Returns how many; `past`: keys up to it are out.
__device__ int beam_shorten(beam_key *list, int n, int count, int most, beam_key &past) {
    const int lane = threadIdx.x & 63;
    if (n <= 256) {
        beam_key mine[4];
        uint32_t order[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int e = i * 64 + lane;
            mine[i] = e < n ? list[e] : 0;
            order[i] = beam_order(mine[i]);
        }
        const uint32_t t = beam_threshold<32>(order, count);
        int kept = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) kept += __popcll(__ballot(mine[i] != 0 && order[i] >= t));
        if (kept <= most) {
            beam_in_order();
            int at = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const bool keep = mine[i] != 0 && order[i] >= t;
                const unsigned long long those = __ballot(keep);
                if (keep) list[at + __popcll(those & ((1ull << lane) - 1))] = mine[i];
                at += __popcll(those);
            }
            beam_in_order();
            if (((beam_key)t << 32) > past + 1) past = ((beam_key)t << 32) - 1;  // (lower values are out)
            return kept;
        }
    }
    // the largest below the last one found, `count` times; they take the places that it has passed
    beam_key below = ~0ull, first = 0;
    for (int k = 0; k < count; ++k) {
        beam_key mine = 0;
        for (int e = lane; e < n; e += 64) {
            const beam_key v = list[e];
            if (v < below && v > mine) mine = v;
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            const beam_key v = __shfl_xor(mine, o);
            mine = v > mine ? v : mine;
        }
        below = mine;
        if (lane == k) first = mine;  // (count is 64 at most)
    }
    beam_in_order();
    if (lane < count) list[lane] = first;
    beam_in_order();
    past = below;
    return count;
}

// ODD: rows begin anywhere, and may end inside a vector of 16 bytes.
template <typename T, bool ODD>
__global__ __launch_bounds__(BEAM_THREADS) void beam_rows(BeamArgs g) {
    constexpr int E = 16 / sizeof(T), Q = BEAM_PER_THREAD / E;
    __shared__ beam_key lists[BEAM_WAVES][BEAM_LIST];
    __shared__ __align__(16) beam_key merged[BEAM_WAVES * BEAM_CUT];
    __shared__ float tops[BEAM_WAVES];
    __shared__ double sums[BEAM_WAVES];
    __shared__ int lengths[BEAM_WAVES];
    const int tid = threadIdx.x, lane = tid & 63, wave = dl_uniform(tid >> 6);
    const long long row = blockIdx.x / g.pieces;
    const int piece = blockIdx.x % g.pieces;
    if (g.ended && g.ended[row]) return;
    const T *logits = (const T *)g.logits + row * g.ldl;
    const int v0 = piece * g.piece, v1 = min(v0 + g.piece, g.V), most = g.count <= 32 ? 64 : BEAM_CUT;
    const float inf = __builtin_inff();
    beam_key *list = lists[wave];

    float next[Q][E];
    auto fetch = [&](int at) __attribute__((always_inline)) {
#pragma unroll
        for (int q = 0; q < Q; ++q) {
            const int c = at + (q * BEAM_THREADS + tid) * E;
            if (!ODD && c < v1) dl_load<T, E>(logits + c, next[q]);
            else if (ODD && c + E <= v1) dl_load_some<T, E>(logits + c, E, next[q]);
            else if (ODD && c < v1)
#pragma unroll
                for (int i = 0; i < E; ++i) next[q][i] = c + i < v1 ? (float)logits[c + i] : -inf;
            else
#pragma unroll
                for (int i = 0; i < E; ++i) next[q][i] = -inf;
        }
    };
    float ref = -inf, bound = -inf;  // of the thread's sum; of the wavefront's list
    beam_key past = 0;
    double sum = 0.0;
    int length = 0;
    fetch(v0);
    for (int at = v0; at < v1; at += BEAM_ROUND) {
        float v[Q][E], top = -inf;
#pragma unroll
        for (int q = 0; q < Q; ++q)
#pragma unroll
            for (int i = 0; i < E; ++i) {
                v[q][i] = fminf(fmaxf(next[q][i], -inf), 3.4028234663852886e38f);  // NaN: no candidate; infinity: the largest number
                top = fmaxf(top, v[q][i]);
            }
        if (at + BEAM_ROUND < v1) fetch(at + BEAM_ROUND);
        if (top > ref + 8.0f || (ref == -inf && top > -inf)) {  // (no higher, as the exponent's rounding grows with it)
            sum *= ref == -inf ? 0.0 : exp((double)ref - (double)top);
            ref = top;
        }
        if (ref > -inf) {
            float part = 0.0f;
#pragma unroll
            for (int q = 0; q < Q; ++q)
#pragma unroll
                for (int i = 0; i < E; ++i) part += __builtin_amdgcn_exp2f((v[q][i] - ref) * BEAM_LOG2E);
            sum += (double)part;
        }
        if (at == v0) {
            const uint32_t order[1] = {beam_order(beam_make(top, 0))}, t = beam_threshold<20>(order, g.count);
            if (t >= BEAM_LOWEST) bound = beam_value((beam_key)t << 32);
        }
        if (!__ballot(top >= bound && top > -inf)) continue;
#pragma unroll
        for (int e = 0; e < BEAM_PER_THREAD; ++e) {
            const int q = e / E, i = e % E;
            if (__ballot(v[q][i] >= bound)) {
                const beam_key key = beam_make(v[q][i], (uint32_t)(at + (q * BEAM_THREADS + tid) * E + i));
                const bool in = v[q][i] >= bound && v[q][i] > -inf && key > past;
                const unsigned long long those = __ballot(in);
                if (in) list[length + __popcll(those & ((1ull << lane) - 1))] = key;
                length += __popcll(those);
            }
            if (e % 8 == 7 && length > most) {  // (then there are more than `count`)
                beam_in_order();
                length = beam_shorten(list, length, g.count, most, past);
                const float last = beam_value(past + 1);
                bound = last > bound ? last : bound;
            }
        }
    }

    // the wavefronts' lists are one; every key counts the better ones
    if (lane == 0) lengths[wave] = length;
    __syncthreads();
    int before = 0, n = 0;
#pragma unroll
    for (int w = 0; w < BEAM_WAVES; ++w) {
        before += w < wave ? lengths[w] : 0;
        n += lengths[w];
    }
    for (int e = lane; e < length; e += 64) merged[before + e] = list[e];
    if (tid == 0 && (n & 1)) merged[n] = 0;  // (n is odd: below the end)
    __syncthreads();
    beam_key *out = g.keys + (row * g.pieces + piece) * g.count;
    for (int e = tid; e < n; e += BEAM_THREADS) {
        const beam_key mine = merged[e];
        int rank = 0;
#pragma unroll 8
        for (int j = 0; j < n; j += 2) {
            const ulonglong2 two = *reinterpret_cast<const ulonglong2 *>(merged + j);
            rank += (two.x > mine ? 1 : 0) + (two.y > mine ? 1 : 0);
        }
        if (rank < g.count) out[rank] = mine;
    }
    for (int e = n + tid; e < g.count; e += BEAM_THREADS) out[e] = 0;

    // the threads' sums, on one maximum, in a fixed order
    float largest = ref;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) largest = fmaxf(largest, __shfl_xor(largest, o));
    if (lane == 0) tops[wave] = largest;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < BEAM_WAVES; ++w) largest = fmaxf(largest, tops[w]);
    sum = ref > -inf ? sum * exp((double)ref - (double)largest) : 0.0;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
    if (lane == 0) sums[wave] = sum;
    __syncthreads();
    if (tid == 0) {
        sum = 0.0;
        for (int w = 0; w < BEAM_WAVES; ++w) sum += sums[w];
        g.parts[row * g.pieces + piece] = {sum, largest, 0};
    }
}

// A block takes a sequence's K * pieces lists of `count` candidates, best first.  The count-th of the lists' best bounds them from below, where
// there are as many lists; every candidate that passes it counts the better ones, or where there are many the best of all is taken `count` times.
// Ranking m takes about 0.3 ns m^2, taking the best count times 1.4 us each.
#define BEAM_RANKS 512
__device__ __forceinline__ bool beam_ranked(int m, int count) { return m <= BEAM_RANKS && m * m <= 4096 * count; }
__device__ __forceinline__ bool beam_before(double a, beam_key ka, double b, beam_key kb) { return a > b || (a == b && ka > kb); }
__global__ __launch_bounds__(BEAM_THREADS) void beam_pick(BeamArgs g) {
    __shared__ double value[BEAM_PICKS], norm[BEAM_MOST], base[BEAM_MOST], wave_value[BEAM_WAVES], bound;
    __shared__ double kept_value[BEAM_RANKS];
    // Of equal candidates the one with the larger key comes first: the earlier beam's, of one beam the larger logit's, then the one that lies first in
    // the lists, at the place that the last bits say.  (Before that the lists' largest.)
    __shared__ beam_key key[BEAM_PICKS], kept_key[BEAM_RANKS], wave_key[BEAM_WAVES];
    __shared__ int kept, ended[BEAM_MOST];
    const int tid = threadIdx.x, b = blockIdx.x, per = g.pieces * g.count, n = g.K * per, lists = g.K * g.pieces;
    const double inf = __builtin_inf();
    const beam_key *keys = g.keys + (long long)b * n;

    // everything that is read, asked for at once
    const BeamPart *parts = g.parts + (long long)b * lists;
    constexpr int EARLY = 4;
    beam_key early[EARLY];
#pragma unroll
    for (int i = 0; i < EARLY; ++i) early[i] = i * BEAM_THREADS + tid < n ? keys[i * BEAM_THREADS + tid] : 0;
    if (tid < g.K) {
        const long long row = (long long)b * g.K + tid;
        ended[tid] = g.ended && g.ended[row] ? 1 : 0;
        base[tid] = (double)g.scores[row];
    }
    for (int e = tid; e < lists; e += BEAM_THREADS) {
        const BeamPart p = parts[e];
        value[e] = p.sum, key[e] = __float_as_uint(p.largest);
    }
    if (tid == 0) kept = 0, bound = -inf;
    __syncthreads();
    // the rows' logarithms: every list's share of its row's sum, then a thread a row  (what was never written of rows that have ended is not used)
    for (int e = tid; e < lists; e += BEAM_THREADS) {
        const int first = e / g.pieces * g.pieces;
        if (ended[e / g.pieces]) continue;
        float most = -__builtin_inff();
        for (int i = 0; i < g.pieces; ++i) most = fmaxf(most, __uint_as_float((uint32_t)key[first + i]));
        value[e] = value[e] > 0.0 ? value[e] * exp((double)__uint_as_float((uint32_t)key[e]) - (double)most) : 0.0;
        if (e == first) norm[e / g.pieces] = (double)most;
    }
    __syncthreads();
    if (tid < g.K && !ended[tid]) {
        double sum = 0.0;
        for (int i = 0; i < g.pieces; ++i) sum += value[tid * g.pieces + i];
        norm[tid] = norm[tid] > -inf ? norm[tid] + log(sum) : inf;  // (infinity: nothing to go on with)
    }
    __syncthreads();
    const auto candidate = [&](int e, beam_key of_row) __attribute__((always_inline)) {
        const int k = e / per;
        double c = -inf;
        if (ended[k]) {
            if (e == k * per) c = base[k];
        } else if (of_row) c = base[k] + ((double)beam_value(of_row) - norm[k]);
        value[e] = c == c ? c : -inf;
        key[e] = (beam_key)(BEAM_MOST - k) << 44 | (beam_key)beam_order(of_row) << 12 | (beam_key)(BEAM_PICKS - 1 - e);
    };
#pragma unroll
    for (int i = 0; i < EARLY; ++i)
        if (i * BEAM_THREADS + tid < n) candidate(i * BEAM_THREADS + tid, early[i]);
    for (int e = EARLY * BEAM_THREADS + tid; e < n; e += BEAM_THREADS) candidate(e, keys[e]);
    __syncthreads();
    if (lists >= g.count && lists <= 2 * BEAM_THREADS)
        for (int e = tid; e < lists; e += BEAM_THREADS) {
            const double mine = value[e * g.count];
            int rank = 0;
#pragma unroll 4
            for (int j = 0; j < lists; ++j) rank += value[j * g.count] > mine || (value[j * g.count] == mine && j < e) ? 1 : 0;
            if (rank == g.count - 1) bound = mine;
        }
    __syncthreads();
    const double least = bound;
    const auto place = [](beam_key k) { return BEAM_PICKS - 1 - (int)(k & (BEAM_PICKS - 1)); };
    for (int e = tid; e < n; e += BEAM_THREADS) {
        const double c = value[e];
        if (!(c >= least && c > -inf)) continue;
        const int at = atomicAdd(&kept, 1);  // (their order plays no part)
        if (at < BEAM_RANKS) kept_value[at] = c, kept_key[at] = key[e];
    }
    __syncthreads();
    const auto answer = [&](int j, double c, int at) __attribute__((always_inline)) {
        const long long out = (long long)b * g.count + j;
        const int k = at < 0 ? 0 : at / per;
        g.out_scores[out] = (float)c;
        g.parents[out] = k;
        g.tokens[out] = at < 0 ? -1 : ended[k] ? g.end : (long long)beam_index(keys[at]);
    };
    const int m = kept;
    for (int j = m + tid; j < g.count; j += BEAM_THREADS) answer(j, -inf, -1);
    if (beam_ranked(m, g.count)) {
        for (int e = tid; e < m; e += BEAM_THREADS) {
            const double mine = kept_value[e];
            const beam_key mine_key = kept_key[e];
            int rank = 0;
#pragma unroll 4
            for (int j = 0; j < m; ++j) rank += beam_before(kept_value[j], kept_key[j], mine, mine_key) ? 1 : 0;
            if (rank < g.count) answer(rank, mine, place(mine_key));
        }
        return;
    }
    double mine = -inf;
    beam_key mine_key = 0;
    const auto own_best = [&]() __attribute__((always_inline)) {
        mine = -inf, mine_key = 0;
        if (g.pieces > 1) {
            for (int e = tid; e < n; e += BEAM_THREADS)
                if (beam_before(value[e], key[e], mine, mine_key)) mine = value[e], mine_key = key[e];
            return;
        }
        int at = -1;  // of one list a beam the first of equal ones has the largest key  (1 x 64 x 50000: 227 us with the loop above, 200)
        for (int e = tid; e < n; e += BEAM_THREADS)
            if (value[e] > mine) mine = value[e], at = e;
        if (at >= 0) mine_key = key[at];
    };
    own_best();
    for (int j = 0; j < g.count; ++j) {  // (there are more than `count` above -infinity)
        double best = mine;
        beam_key best_key = mine_key;
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            const double v = __shfl_xor(best, o);
            const beam_key w = __shfl_xor(best_key, o);
            if (beam_before(v, w, best, best_key)) best = v, best_key = w;
        }
        if ((tid & 63) == 0) wave_value[tid >> 6] = best, wave_key[tid >> 6] = best_key;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < BEAM_WAVES; ++w)
            if (beam_before(wave_value[w], wave_key[w], best, best_key)) best = wave_value[w], best_key = wave_key[w];
        __syncthreads();
        const int at = place(best_key);
        if (tid == 0) answer(j, best, at);
        if (at % BEAM_THREADS == tid) {  // its next one
            value[at] = -inf;
            own_best();
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
            DL_TIMED("beam_rows", s, hipLaunchKernelGGL((beam_rows<T, false>), dim3((unsigned)blocks), dim3(BEAM_THREADS), 0, s, g));
        else
            DL_TIMED("beam_rows", s, hipLaunchKernelGGL((beam_rows<T, true>), dim3((unsigned)blocks), dim3(BEAM_THREADS), 0, s, g));
    });
    DL_TIMED("beam_pick", s, hipLaunchKernelGGL(beam_pick, dim3(B), dim3(BEAM_THREADS), 0, s, g));
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
