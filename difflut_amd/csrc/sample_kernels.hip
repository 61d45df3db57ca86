// Sampling one index per row of logits, with temperature, top-k, top-p and min-p, from given random numbers.
//
// A row's indices are ordered by logit, descending, equal ones by index.  With w_i = exp((l_i - max l) / T):
//   top-k   keeps the first k;   top-p  of these the shortest prefix whose weights reach p times the sum over these (one at least);
//   min-p   of these the ones with w_i >= m (the first stays).   Whatever is kept is therefore a prefix of the order, and its end
//   - the cut - is one (logit, index) pair.
//   The draw: in index order, the first kept one whose running sum of weights exceeds u times the kept sum.
// T <= 0, p <= 0, k = 1 and m > 1 leave the first alone.  NaN counts as -infinity; a row without a larger logit gives -1.
//
// Neighbouring running sums lie close together, so weights are 64-bit integers, round(2^shift w) with shift = 62 - ceil(log2 V), from
// exponentials in double: sums fit, are exact in any order - blocks and atomics can split them as they like, every run gives the
// same index - and a weight is off by 2^-(shift + 1), 2^-46 at V = 131072.
//
// Up to 64 columns: a few lanes per row compare every pair.  Up to SMP_SORTED: a block sorts the row in LDS.  More: the row is
// split over blocks, four launches:
//   sample_max      the chunks' largest logits
//   sample_hist     number and weight of the logits in SMP_BINS classes of (max - l) / T (a monotone function of l)
//   sample_collect  the classes that the cuts can fall into are known now: weights of the classes before them, by chunk, and a
//                   list of the indices in them
//   sample_draw     sorts the list, finds the cut, then the chunk and in it the index.  A list that is too long (many equal
//                   logits) is searched over the whole row instead.
#include "dl_types.h"

#define SMP_SORTED 4096
#define SMP_BINS 2048
#define SMP_BINS_PER_Z 32.0  // classes per unit of (max - l) / T: the last one holds what weighs less than e^-63.9
#define SMP_LIST 4096
#define SMP_THREADS 256
#define SMP_DRAW_THREADS 1024
#define SMP_MAX_CHUNKS 256

typedef unsigned long long u64;

struct SampleArgs {
    const void *logits;
    long long ldl;
    const float *uniform, *temperature, *top_p, *min_p;  // [B]; the last three may be null: the numbers below hold for every row
    const int *top_k;
    float T, p, m;
    int k, B, V, shift;
    long long *out;
    // rows split over blocks
    int chunk, chunks;
    uint32_t *chunk_key;  // [B][chunks]
    u64 *chunk_sum;       // [B][chunks]
    u64 *bin_weight;      // [B][SMP_BINS]
    uint32_t *bin_count;  // [B][SMP_BINS]
    uint32_t *listed;     // [B]
    u64 *list;            // [B][SMP_LIST]
};

// A row's settings in the form the kernels use
struct SampleRow {
    double rT, p, m, u;
    int k;
    bool first_only, cut_k, cut_p;
};
__device__ __forceinline__ SampleRow smp_row(const SampleArgs &a, int b) {
    SampleRow r;
    const float T = a.temperature ? a.temperature[b] : a.T, p = a.top_p ? a.top_p[b] : a.p, m = a.min_p ? a.min_p[b] : a.m;
    const int k = a.top_k ? a.top_k[b] : a.k;
    const float u = a.uniform[b];
    r.first_only = !(T > 0.0f) || !(p > 0.0f) || !(m <= 1.0f) || k == 1;
    r.rT = 1.0 / (double)T;
    r.p = p, r.m = m;
    r.u = u > 0.0f ? fmin((double)u, 1.0) : 0.0;
    r.cut_k = k > 0 && k < a.V;
    r.k = r.cut_k ? k : a.V;
    r.cut_p = !(p >= 1.0f);
    return r;
}

// Logits as integers of the same order; -infinity and NaN share the least one, -0 is 0.
#define SMP_DEAD 0x007FFFFFu
__device__ __forceinline__ uint32_t smp_key(float l) {
    const uint32_t bits = __float_as_uint(l + 0.0f);
    return l != l ? SMP_DEAD : (bits & 0x80000000u) ? ~bits : bits | 0x80000000u;
}
__device__ __forceinline__ float smp_logit(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key & 0x7FFFFFFFu : ~key); }
// (key, index) pairs in the row's order: larger ones first
__device__ __forceinline__ u64 smp_pair(uint32_t key, uint32_t index) { return (u64)key << 32 | (0xFFFFFFFFu - index); }

__device__ __forceinline__ double smp_exp(uint32_t key, uint32_t top, const SampleRow &r) {
    if (key == top) return 1.0;
    const double M = smp_logit(top);
    if (key <= SMP_DEAD || M > 3.5e38) return 0.0;
    return exp(((double)smp_logit(key) - M) * r.rT);
}
__device__ __forceinline__ u64 smp_fixed(double e, int shift) { return (u64)(ldexp(e, shift) + 0.5); }
// weight of an index that no cut but min-p takes away
__device__ __forceinline__ u64 smp_weight(uint32_t key, uint32_t top, const SampleRow &r, int shift) {
    const double e = smp_exp(key, top, r);
    return e >= r.m || key == top ? smp_fixed(e, shift) : 0;
}
__device__ __forceinline__ u64 smp_target(const SampleRow &r, u64 total) {  // the running sum that has to be exceeded
    const u64 t = (u64)(r.u * (double)total);
    return t < total ? t : total - 1;
}

__device__ __forceinline__ uint32_t smp_wave_max(uint32_t v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, o));
    return v;
}
__device__ __forceinline__ u64 smp_wave_sum(u64 v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
}
// Exclusive prefix sum over the block's threads; `total` of all.  red: THREADS / 64 values of LDS.
template <int THREADS>
__device__ __forceinline__ u64 smp_scan(u64 v, u64 &total, u64 *red) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    u64 run = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const u64 up = __shfl_up(run, o);
        if (lane >= o) run += up;
    }
    __syncthreads();  // red may still be read from the last call
    if (lane == 63) red[wave] = run;
    __syncthreads();
    u64 before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) {
        if (w < wave) before += red[w];
        all += red[w];
    }
    total = all;
    return before + run - v;
}
template <int THREADS>
__device__ __forceinline__ uint32_t smp_max(uint32_t v, u64 *red) {
    v = smp_wave_max(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) v = max(v, (uint32_t)red[w]);
    return v;
}
// Descending, n a power of two
template <int THREADS>
__device__ void smp_sort(u64 *pairs, int n) {
    for (int size = 2; size <= n; size <<= 1)
        for (int step = size >> 1; step > 0; step >>= 1) {
            __syncthreads();
            for (int i = threadIdx.x; i < n / 2; i += THREADS) {
                const int lo = 2 * i - (i & (step - 1)), hi = lo + step;
                const u64 x = pairs[lo], y = pairs[hi];
                if ((x < y) == ((lo & size) == 0)) pairs[lo] = y, pairs[hi] = x;
            }
        }
    __syncthreads();
}

// ---------------------------------------------------------------------------------- up to 64 columns
template <typename T, int SEG>
__global__ __launch_bounds__(SMP_THREADS) void sample_pairs(SampleArgs a) {
    const int i = threadIdx.x & (SEG - 1);
    const long long b0 = ((long long)blockIdx.x * SMP_THREADS + threadIdx.x) / SEG;
    const int b = (int)(b0 < a.B ? b0 : a.B - 1);
    const SampleRow r = smp_row(a, b);
    const uint32_t key = i < a.V ? smp_key((float)((const T *)a.logits)[b * a.ldl + i]) : 0;
    uint32_t top = key;
#pragma unroll
    for (int o = SEG / 2; o > 0; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o, SEG));
    const double e = r.first_only ? (key == top ? 1.0 : 0.0) : smp_exp(key, top, r);
    const u64 w = smp_fixed(e, a.shift);
    int rank = 0;
    u64 before = 0;
#pragma unroll 8
    for (int j = 0; j < SEG; ++j) {
        const uint32_t kj = (uint32_t)__shfl((int)key, j, SEG);
        const u64 wj = __shfl(w, j, SEG);
        if (kj > key || (kj == key && j < i)) ++rank, before += wj;
    }
    const bool alive = key > SMP_DEAD;
    u64 sum = alive && rank < r.k ? w : 0;
#pragma unroll
    for (int o = SEG / 2; o > 0; o >>= 1) sum += __shfl_xor(sum, o, SEG);
    const bool in_p = !r.cut_p || (double)before < r.p * (double)sum;
    const bool keep = alive && (rank == 0 || (!r.first_only && rank < r.k && in_p && e >= r.m));
    u64 run = keep ? w : 0;
#pragma unroll
    for (int o = 1; o < SEG; o <<= 1) {
        const u64 up = __shfl_up(run, o, SEG);
        if (i >= o) run += up;
    }
    const u64 total = __shfl(run, SEG - 1, SEG);
    const u64 past = __ballot(total > 0 && run > smp_target(r, total));
    const u64 mine = SEG == 64 ? past : (past >> (threadIdx.x & 63 & ~(SEG - 1))) & ((1ull << (SEG & 63)) - 1);
    if (i == 0 && b0 < a.B) a.out[b] = mine ? __builtin_ctzll(mine) : -1;
}

// ---------------------------------------------------------------------------------- a row in LDS
// In index order, over [i0, i1): the first index whose running sum of kept weights exceeds `target`; a thread per run of indices.
template <typename T, int THREADS>
__device__ void smp_draw(const SampleArgs &a, const SampleRow &r, int b, int i0, int i1, u64 cut, uint32_t top, bool draw_rest, u64 target,
                         u64 *red) {
    const T *row = (const T *)a.logits + b * a.ldl;
    const int per = (i1 - i0 + THREADS - 1) / THREADS, begin = min(i0 + (int)threadIdx.x * per, i1), end = min(begin + per, i1);
    u64 mine = 0, total;
    for (int i = begin; i < end; ++i) {
        const uint32_t key = smp_key((float)row[i]);
        if (smp_pair(key, i) >= cut) mine += smp_weight(key, top, r, a.shift);
    }
    u64 run = smp_scan<THREADS>(mine, total, red);
    if (!draw_rest) target = total ? smp_target(r, total) : 0;
    if (total == 0) {
        if (threadIdx.x == 0) a.out[b] = -1;
        return;
    }
    if (run <= target && target < run + mine)
        for (int i = begin; i < end; ++i) {
            const uint32_t key = smp_key((float)row[i]);
            if (smp_pair(key, i) >= cut) run += smp_weight(key, top, r, a.shift);
            if (run > target) {
                a.out[b] = i;
                break;
            }
        }
}

template <typename T, int THREADS>
__global__ __launch_bounds__(THREADS) void sample_sorted(SampleArgs a, int n) {
    extern __shared__ u64 pairs[];  // [n], n a power of two >= V
    __shared__ u64 red[THREADS / 64];
    const int b = blockIdx.x;
    const T *row = (const T *)a.logits + b * a.ldl;
    const SampleRow r = smp_row(a, b);
    u64 best = 0;
    for (int i = threadIdx.x; i < n; i += THREADS) {
        const u64 pair = i < a.V ? smp_pair(smp_key((float)row[i]), i) : 0;
        pairs[i] = pair;
        best = max(best, pair);
    }
    const uint32_t top = smp_max<THREADS>((uint32_t)(best >> 32), red);
    if (top <= SMP_DEAD || r.first_only) {
        const uint32_t low = smp_max<THREADS>((uint32_t)(best >> 32) == top ? (uint32_t)best : 0, red);
        if (threadIdx.x == 0) a.out[b] = top <= SMP_DEAD ? -1 : (long long)(0xFFFFFFFFu - low);
        return;
    }
    u64 cut = (u64)(SMP_DEAD + 1) << 32;  // everything that is not dead
    if (r.cut_k || r.cut_p) {
        smp_sort<THREADS>(pairs, n);
        const int per = max(1, n / THREADS), begin = min((int)threadIdx.x * per, n), end = min(begin + per, n);
        u64 mine = 0, total, kept = 0;
        for (int j = begin; j < end; ++j)
            if (j < r.k) mine += smp_fixed(smp_exp((uint32_t)(pairs[j] >> 32), top, r), a.shift);
        u64 before = smp_scan<THREADS>(mine, total, red);
        const double limit = r.p * (double)total;
        for (int j = begin; j < end; ++j) {
            const uint32_t key = (uint32_t)(pairs[j] >> 32);
            if (j >= r.k || key <= SMP_DEAD || (j > 0 && r.cut_p && !((double)before < limit))) break;
            before += smp_fixed(smp_exp(key, top, r), a.shift);
            ++kept;
        }
        smp_scan<THREADS>(kept, total, red);
        cut = pairs[total - 1];
    }
    smp_draw<T, THREADS>(a, r, b, 0, a.V, cut, top, false, 0, red);
}

// ---------------------------------------------------------------------------------- rows split over blocks
__device__ __forceinline__ int smp_bin(uint32_t key, double M, const SampleRow &r) {
    return (int)fmin((M - (double)smp_logit(key)) * r.rT * SMP_BINS_PER_Z, (double)(SMP_BINS - 1));
}
template <int THREADS>
__device__ __forceinline__ uint32_t smp_top(const SampleArgs &a, int b, u64 *red) {
    uint32_t v = 0;
    for (int c = threadIdx.x; c < a.chunks; c += THREADS) v = max(v, a.chunk_key[(long long)b * a.chunks + c]);
    return smp_max<THREADS>(v, red);
}

template <typename T>
__global__ __launch_bounds__(SMP_THREADS) void sample_max(SampleArgs a) {
    __shared__ u64 red[SMP_THREADS / 64];
    const int c = blockIdx.x % a.chunks, b = blockIdx.x / a.chunks;
    const T *row = (const T *)a.logits + b * a.ldl;
    const int i1 = min((c + 1) * (long long)a.chunk, (long long)a.V);
    uint32_t v = 0;
#pragma unroll 4
    for (int i = c * a.chunk + threadIdx.x; i < i1; i += SMP_THREADS) v = max(v, smp_key((float)row[i]));
    v = smp_max<SMP_THREADS>(v, red);
    if (threadIdx.x == 0) a.chunk_key[(long long)b * a.chunks + c] = v;
    // the row's classes and list begin empty
    for (int i = c * SMP_THREADS + threadIdx.x; i < SMP_BINS; i += a.chunks * SMP_THREADS)
        a.bin_weight[(long long)b * SMP_BINS + i] = 0, a.bin_count[(long long)b * SMP_BINS + i] = 0;
    if (c == 0 && threadIdx.x == 0) a.listed[b] = 0;
}

template <typename T>
__global__ __launch_bounds__(SMP_THREADS) void sample_hist(SampleArgs a) {
    __shared__ u64 weight[SMP_BINS];
    __shared__ uint32_t count[SMP_BINS];
    __shared__ u64 red[SMP_THREADS / 64];
    const int c = blockIdx.x % a.chunks, b = blockIdx.x / a.chunks;
    const SampleRow r = smp_row(a, b);
    if (r.first_only || !(r.cut_k || r.cut_p)) return;
    const uint32_t top = smp_top<SMP_THREADS>(a, b, red);
    if (top <= SMP_DEAD) return;
    for (int i = threadIdx.x; i < SMP_BINS; i += SMP_THREADS) weight[i] = 0, count[i] = 0;
    __syncthreads();
    const T *row = (const T *)a.logits + b * a.ldl;
    const int i1 = min((c + 1) * (long long)a.chunk, (long long)a.V);
    const double M = smp_logit(top);
    for (int i = c * a.chunk + threadIdx.x; i < i1; i += SMP_THREADS) {
        const uint32_t key = smp_key((float)row[i]);
        if (key <= SMP_DEAD) continue;
        const int bin = key == top ? 0 : smp_bin(key, M, r);
        atomicAdd(&count[bin], 1u);
        if (bin < SMP_BINS - 1) atomicAdd(&weight[bin], smp_fixed(smp_exp(key, top, r), a.shift));
    }
    __syncthreads();
    for (int i = threadIdx.x; i < SMP_BINS; i += SMP_THREADS)
        if (count[i]) {
            atomicAdd(&a.bin_count[(long long)b * SMP_BINS + i], count[i]);
            if (weight[i]) atomicAdd(&a.bin_weight[(long long)b * SMP_BINS + i], weight[i]);
        }
}

// Where the cuts can be: the class of the k-th index, the classes of top-p's last one
struct SampleCut {
    int k_bin, p_first, p_last;  // SMP_BINS: none
    int sure;                    // classes below are kept for certain (but for min-p)
    uint32_t k_before;           // indices in the classes before k_bin
    u64 k_weight, p_weight;      // weight of the classes before k_bin, before p_first
};
__device__ __forceinline__ bool smp_open(const SampleCut &c, int bin) { return bin == c.k_bin || (bin >= c.p_first && bin <= c.p_last); }

template <int THREADS>
__device__ SampleCut smp_resolve(const SampleArgs &a, const SampleRow &r, int b, u64 *red, SampleCut *shared) {
    constexpr int PER = SMP_BINS / THREADS;
    uint32_t n[PER];
    u64 w[PER], mine_n = 0, mine_w = 0, all_n, all_w;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        n[j] = a.bin_count[(long long)b * SMP_BINS + threadIdx.x * PER + j];
        w[j] = a.bin_weight[(long long)b * SMP_BINS + threadIdx.x * PER + j];
        mine_n += n[j], mine_w += w[j];
    }
    const u64 n0 = smp_scan<THREADS>(mine_n, all_n, red), w0 = smp_scan<THREADS>(mine_w, all_w, red);
    if (threadIdx.x == 0) *shared = {SMP_BINS, SMP_BINS, SMP_BINS, SMP_BINS, 0, all_w, 0};
    __syncthreads();
    u64 cn = n0, cw = w0;
    if (r.cut_k)
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            // (a cut in the last class takes nothing away that weighs anything)
            if (cn < (u64)r.k && cn + n[j] >= (u64)r.k && threadIdx.x * PER + j < SMP_BINS - 1)
                shared->k_bin = threadIdx.x * PER + j, shared->k_before = (uint32_t)cn, shared->k_weight = cw;
            cn += n[j], cw += w[j];
        }
    __syncthreads();
    const int k_bin = shared->k_bin;
    const u64 low = shared->k_weight;
    u64 high = low;
    if (k_bin < SMP_BINS) high += a.bin_weight[(long long)b * SMP_BINS + k_bin];
    if (r.cut_p) {
        cw = w0;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const bool begin = cw == 0 && w[j] > 0;  // the first class with weight (class 0)
            const double p_low = r.p * (double)low, p_high = r.p * (double)high;
            if ((begin || (double)cw < p_low) && (double)(cw + w[j]) >= p_low && w[j] > 0) shared->p_first = threadIdx.x * PER + j, shared->p_weight = cw;
            if ((begin || (double)cw < p_high) && (double)(cw + w[j]) >= p_high && w[j] > 0) shared->p_last = threadIdx.x * PER + j;
            cw += w[j];
        }
    }
    __syncthreads();
    SampleCut c = *shared;
    c.sure = min(c.k_bin, c.p_first);
    return c;
}

template <typename T>
__global__ __launch_bounds__(SMP_THREADS) void sample_collect(SampleArgs a) {
    __shared__ u64 red[SMP_THREADS / 64];
    __shared__ SampleCut shared;
    const int c = blockIdx.x % a.chunks, b = blockIdx.x / a.chunks;
    const SampleRow r = smp_row(a, b);
    if (r.first_only) return;
    const uint32_t top = smp_top<SMP_THREADS>(a, b, red);
    if (top <= SMP_DEAD) return;
    const bool cuts = r.cut_k || r.cut_p;
    SampleCut cut = {SMP_BINS, SMP_BINS, SMP_BINS, SMP_BINS, 0, 0, 0};
    if (cuts) cut = smp_resolve<SMP_THREADS>(a, r, b, red, &shared);
    const T *row = (const T *)a.logits + b * a.ldl;
    const int i1 = min((c + 1) * (long long)a.chunk, (long long)a.V);
    const double M = smp_logit(top);
    const int lane = threadIdx.x & 63;
    u64 sum = 0;
    for (int i0 = c * a.chunk; i0 < i1; i0 += SMP_THREADS) {
        const int i = i0 + threadIdx.x;
        const uint32_t key = i < i1 ? smp_key((float)row[i]) : 0;
        const int bin = key <= SMP_DEAD ? SMP_BINS : key == top ? 0 : smp_bin(key, M, r);
        if (bin < cut.sure) sum += smp_weight(key, top, r, a.shift);
        const bool open = bin < SMP_BINS && smp_open(cut, bin);
        const u64 takes = __ballot(open);
        if (takes) {
            uint32_t at = 0;
            if (lane == 0) at = atomicAdd(&a.listed[b], (uint32_t)__popcll(takes));
            at = (uint32_t)__shfl((int)at, 0) + __popcll(takes & ((1ull << lane) - 1));
            if (open && at < SMP_LIST) a.list[(long long)b * SMP_LIST + at] = smp_pair(key, i);
        }
    }
    u64 total;
    smp_scan<SMP_THREADS>(sum, total, red);
    if (threadIdx.x == 0) a.chunk_sum[(long long)b * a.chunks + c] = total;
}

// Sums over the whole row by one block: number and weight of the keys >= `least` (of those in open classes: their extremes)
template <typename T, int THREADS>
__device__ void smp_row_sums(const SampleArgs &a, const SampleRow &r, int b, uint32_t top, uint32_t least, u64 &count, u64 &weight, u64 *red) {
    const T *row = (const T *)a.logits + b * a.ldl;
    u64 n = 0, w = 0;
    for (int i = threadIdx.x; i < a.V; i += THREADS) {
        const uint32_t key = smp_key((float)row[i]);
        if (key < least || key <= SMP_DEAD) continue;
        ++n;
        w += smp_fixed(smp_exp(key, top, r), a.shift);
    }
    smp_scan<THREADS>(n, count, red);
    smp_scan<THREADS>(w, weight, red);
}
// The least and the largest key in classes [first, last]
template <typename T, int THREADS>
__device__ void smp_key_range(const SampleArgs &a, const SampleRow &r, int b, uint32_t top, int first, int last, uint32_t &low, uint32_t &high, u64 *red) {
    const T *row = (const T *)a.logits + b * a.ldl;
    const double M = smp_logit(top);
    uint32_t lo = 0, hi = 0;  // (lo: of the complements)
    for (int i = threadIdx.x; i < a.V; i += THREADS) {
        const uint32_t key = smp_key((float)row[i]);
        if (key <= SMP_DEAD) continue;
        const int bin = key == top ? 0 : smp_bin(key, M, r);
        if (bin < first || bin > last) continue;
        hi = max(hi, key), lo = max(lo, ~key);
    }
    high = smp_max<THREADS>(hi, red);
    low = ~smp_max<THREADS>(lo, red);
}

// The cut of a row whose open classes hold more than the list: by bisection over the keys, then over equal ones by index.
template <typename T, int THREADS>
__device__ u64 smp_search(const SampleArgs &a, const SampleRow &r, const SampleCut &c, int b, uint32_t top, u64 *red) {
    uint32_t lo, hi, cut_key = SMP_DEAD + 1;
    u64 n, w, ties = ~0ull, sum = c.k_weight;  // the indices kept among those with cut_key; the weight under top-k
    if (c.k_bin < SMP_BINS) {
        smp_key_range<T, THREADS>(a, r, b, top, c.k_bin, c.k_bin, lo, hi, red);
        while (lo < hi) {  // the largest key that at least k reach
            const uint32_t mid = lo + (hi - lo + 1) / 2;
            smp_row_sums<T, THREADS>(a, r, b, top, mid, n, w, red);
            if (n >= (u64)r.k) lo = mid;
            else hi = mid - 1;
        }
        cut_key = lo;
        smp_row_sums<T, THREADS>(a, r, b, top, lo + 1, n, w, red);
        ties = (u64)r.k - n;
        sum = w + ties * smp_fixed(smp_exp(lo, top, r), a.shift);
    }
    if (r.cut_p && c.p_first < SMP_BINS) {
        const double limit = r.p * (double)sum;
        smp_key_range<T, THREADS>(a, r, b, top, c.p_first, min(c.p_last, SMP_BINS - 1), lo, hi, red);
        lo = max(lo, cut_key);
        while (lo < hi) {  // the largest key whose weight and that of all larger ones reach the limit
            const uint32_t mid = lo + (hi - lo + 1) / 2;
            smp_row_sums<T, THREADS>(a, r, b, top, mid, n, w, red);
            if ((double)w >= limit) lo = mid;
            else hi = mid - 1;
        }
        smp_row_sums<T, THREADS>(a, r, b, top, lo + 1, n, w, red);
        const u64 each = smp_fixed(smp_exp(lo, top, r), a.shift);
        u64 take = each ? (u64)fmax((limit - (double)w) / (double)each, 0.0) : 0;
        while (each && (double)(w + take * each) < limit) ++take;
        while (take > 1 && !((double)(w + (take - 1) * each) < limit)) --take;
        take = max(take, (u64)(n == 0 ? 1 : 0));  // the first stays
        if (lo > cut_key || take < ties) ties = take;
        cut_key = max(cut_key, lo);
    }
    if (ties == ~0ull) return (u64)cut_key << 32;
    if (ties == 0) return (u64)(cut_key + 1) << 32;
    // the index of the last one kept among equals: a thread per run of indices
    const T *row = (const T *)a.logits + b * a.ldl;
    const int per = (a.V + THREADS - 1) / THREADS, begin = (int)min((long long)threadIdx.x * per, (long long)a.V), end = (int)min((long long)begin + per, (long long)a.V);
    u64 mine = 0, all;
    for (int i = begin; i < end; ++i) mine += smp_key((float)row[i]) == cut_key;
    u64 run = smp_scan<THREADS>(mine, all, red);
    __syncthreads();
    if (ties > all) ties = all;
    if (run < ties && ties <= run + mine)
        for (int i = begin; i < end; ++i)
            if (smp_key((float)row[i]) == cut_key && ++run == ties) red[0] = smp_pair(cut_key, i);
    __syncthreads();
    const u64 cut = red[0];
    __syncthreads();
    return cut;
}

template <typename T>
__global__ __launch_bounds__(SMP_DRAW_THREADS) void sample_draw(SampleArgs a) {
    constexpr int THREADS = SMP_DRAW_THREADS;
    __shared__ u64 pairs[SMP_LIST], red[THREADS / 64], chunk_sum[SMP_MAX_CHUNKS];
    __shared__ SampleCut shared;
    __shared__ int chosen;
    const int b = blockIdx.x;
    const T *row = (const T *)a.logits + b * a.ldl;
    const SampleRow r = smp_row(a, b);
    const uint32_t top = smp_top<THREADS>(a, b, red);
    if (top <= SMP_DEAD) {
        if (threadIdx.x == 0) a.out[b] = -1;
        return;
    }
    if (r.first_only) {  // the first index of the first chunk that holds the largest logit
        uint32_t first = 0;
        for (int c = threadIdx.x; c < a.chunks; c += THREADS)
            if (a.chunk_key[(long long)b * a.chunks + c] == top) first = max(first, ~(uint32_t)c);
        const int c = (int)~smp_max<THREADS>(first, red);
        const int i1 = min((c + 1) * (long long)a.chunk, (long long)a.V);
        uint32_t low = 0;
        for (int i = c * a.chunk + threadIdx.x; i < i1; i += THREADS)
            if (smp_key((float)row[i]) == top) low = max(low, ~(uint32_t)i);
        low = smp_max<THREADS>(low, red);
        if (threadIdx.x == 0) a.out[b] = (long long)(uint32_t)~low;
        return;
    }
    for (int c = threadIdx.x; c < a.chunks; c += THREADS) chunk_sum[c] = a.chunk_sum[(long long)b * a.chunks + c];
    u64 cut = (u64)(SMP_DEAD + 1) << 32, total;
    if (r.cut_k || r.cut_p) {
        const SampleCut c = smp_resolve<THREADS>(a, r, b, red, &shared);
        const uint32_t n = a.listed[b];
        if (n > SMP_LIST) {
            cut = smp_search<T, THREADS>(a, r, c, b, top, red);
            // the chunks' sums anew: a wavefront per chunk
            for (int q = threadIdx.x >> 6; q < a.chunks; q += THREADS / 64) {
                const int i1 = min((q + 1) * (long long)a.chunk, (long long)a.V);
                u64 sum = 0;
                for (int i = q * a.chunk + (threadIdx.x & 63); i < i1; i += 64) {
                    const uint32_t key = smp_key((float)row[i]);
                    if (smp_pair(key, i) >= cut) sum += smp_weight(key, top, r, a.shift);
                }
                sum = smp_wave_sum(sum);
                if ((threadIdx.x & 63) == 0) chunk_sum[q] = sum;
            }
        } else if (n > 0) {
            int size = 1;
            while (size < (int)n) size <<= 1;
            for (int i = threadIdx.x; i < size; i += THREADS) pairs[i] = i < (int)n ? a.list[(long long)b * SMP_LIST + i] : 0;
            smp_sort<THREADS>(pairs, size);
            const double M = smp_logit(top);
            // the list in order: classes [p_first, p_last], then k_bin where that is another one
            const int per = max(1, size / THREADS), begin = min((int)threadIdx.x * per, (int)n), end = min(begin + per, (int)n);
            u64 in_k = 0, k_from = 0, kept = 0, mine = 0;
            for (int j = begin; j < end; ++j) {  // entries before the k-th's class
                const uint32_t key = (uint32_t)(pairs[j] >> 32);
                k_from += (key == top ? 0 : smp_bin(key, M, r)) != c.k_bin;
            }
            smp_scan<THREADS>(k_from, k_from, red);
            const u64 k_end = c.k_bin < SMP_BINS ? k_from + ((u64)r.k - c.k_before) : n;  // list entries that top-k keeps
            for (int j = begin; j < end; ++j) {
                const u64 w = smp_fixed(smp_exp((uint32_t)(pairs[j] >> 32), top, r), a.shift);
                if ((u64)j >= k_from && (u64)j < k_end) in_k += w;
                mine += w;
            }
            smp_scan<THREADS>(in_k, total, red);
            const double limit = r.p * (double)(c.k_weight + total);
            u64 before = smp_scan<THREADS>(mine, total, red) + c.p_weight;
            for (int j = begin; j < end; ++j) {
                const uint32_t key = (uint32_t)(pairs[j] >> 32);
                const int bin = key == top ? 0 : smp_bin(key, M, r);
                const bool in_p = !r.cut_p || (bin <= c.p_last && ((double)before < limit || (j == 0 && c.p_weight == 0)));
                if ((u64)j >= k_end || !in_p) break;
                before += smp_fixed(smp_exp(key, top, r), a.shift);
                ++kept;
            }
            smp_scan<THREADS>(kept, total, red);
            cut = total ? pairs[total - 1] : pairs[0] + 1;
            for (int j = threadIdx.x; j < (int)total; j += THREADS) {
                const u64 w = smp_weight((uint32_t)(pairs[j] >> 32), top, r, a.shift);
                if (w) atomicAdd(&chunk_sum[(0xFFFFFFFFu - (uint32_t)pairs[j]) / a.chunk], w);
            }
        }
    }
    __syncthreads();
    u64 mine = (int)threadIdx.x < a.chunks ? chunk_sum[threadIdx.x] : 0;  // chunks <= SMP_MAX_CHUNKS <= THREADS
    const u64 before = smp_scan<THREADS>(mine, total, red);
    const u64 target = smp_target(r, total);
    if (before <= target && target < before + mine) chosen = threadIdx.x, shared.k_weight = target - before;
    __syncthreads();
    const int c = chosen;
    smp_draw<T, THREADS>(a, r, b, c * a.chunk, (int)min((c + 1) * (long long)a.chunk, (long long)a.V), cut, top, true, shared.k_weight, red);
}

// ---------------------------------------------------------------------------------- host
static int smp_chunk(int B, int V) {
    // about 2048 blocks in all, of 4096 columns at least; a row has SMP_MAX_CHUNKS chunks at most
    long long want = 2048 / B < 1 ? 1 : 2048 / B;
    if (want > SMP_MAX_CHUNKS) want = SMP_MAX_CHUNKS;
    long long chunk = (V + want - 1) / want;
    if (chunk < 4096) chunk = 4096;
    return (int)((chunk + 1023) / 1024 * 1024 < V ? (chunk + 1023) / 1024 * 1024 : V);
}
static size_t smp_layout(SampleArgs &a, char *ws) {
    size_t at = 0;
    const auto take = [&](size_t bytes) {
        char *p = ws + at;
        at += dl_align256(bytes);
        return p;
    };
    a.chunk = smp_chunk(a.B, a.V);
    a.chunks = dl_ceil_div(a.V, a.chunk);
    a.chunk_key = (uint32_t *)take((size_t)a.B * a.chunks * sizeof(uint32_t));
    a.chunk_sum = (u64 *)take((size_t)a.B * a.chunks * sizeof(u64));
    a.bin_weight = (u64 *)take((size_t)a.B * SMP_BINS * sizeof(u64));
    a.bin_count = (uint32_t *)take((size_t)a.B * SMP_BINS * sizeof(uint32_t));
    a.listed = (uint32_t *)take((size_t)a.B * sizeof(uint32_t));
    a.list = (u64 *)take((size_t)a.B * SMP_LIST * sizeof(u64));
    return at;
}

extern "C" size_t dl_sample_workspace_bytes(int B, int V) {
    if (B <= 0 || V <= SMP_SORTED) return 0;
    SampleArgs a = {};
    a.B = B, a.V = V;
    return smp_layout(a, nullptr);
}

extern "C" int dl_sample(const void *logits, long long ldl, int type, const float *uniform, const float *temperature, const int *top_k,
                         const float *top_p, const float *min_p, float temperature_all, int top_k_all, float top_p_all, float min_p_all,
                         long long *out, void *ws, size_t ws_bytes, int B, int V, void *stream) {
    if (!dl_type_known(type)) return DL_ERR_UNSUPPORTED;
    if (B < 0 || V <= 0 || ldl < V) return DL_ERR_SHAPE;
    if (B == 0) return DL_OK;
    if (!logits || !uniform || !out) return DL_ERR_NULL;
    if (V > (1 << 30)) return DL_ERR_UNSUPPORTED;
    const size_t need = dl_sample_workspace_bytes(B, V);
    if (need && !ws) return DL_ERR_NULL;
    if (ws_bytes < need) return DL_ERR_WORKSPACE;
    hipStream_t s = (hipStream_t)stream;
    SampleArgs a = {};
    a.logits = logits, a.ldl = ldl, a.uniform = uniform, a.temperature = temperature, a.top_k = top_k, a.top_p = top_p, a.min_p = min_p;
    a.T = temperature_all, a.k = top_k_all, a.p = top_p_all, a.m = min_p_all, a.out = out, a.B = B, a.V = V;
    int bits = 0;
    while ((1LL << bits) < V) ++bits;
    a.shift = 62 - bits;
    if (V <= 64) {
        const int seg = V <= 8 ? 8 : V <= 16 ? 16 : V <= 32 ? 32 : 64;
        const long long blocks = ((long long)B * seg + SMP_THREADS - 1) / SMP_THREADS;
        if (blocks > 0x7fffffffLL) return DL_ERR_UNSUPPORTED;
        dl_prof_begin("sample_pairs", s);
        DL_BY_TYPE(type, T, if (seg == 8) sample_pairs<T, 8><<<(int)blocks, SMP_THREADS, 0, s>>>(a);
                   else if (seg == 16) sample_pairs<T, 16><<<(int)blocks, SMP_THREADS, 0, s>>>(a);
                   else if (seg == 32) sample_pairs<T, 32><<<(int)blocks, SMP_THREADS, 0, s>>>(a);
                   else sample_pairs<T, 64><<<(int)blocks, SMP_THREADS, 0, s>>>(a));
        dl_prof_end(s);
        return dl_launch_status();
    }
    if (V <= SMP_SORTED) {
        const int n = 1 << bits;
        dl_prof_begin("sample_sorted", s);
        DL_BY_TYPE(type, T, if (n <= 1024) sample_sorted<T, 256><<<B, 256, n * sizeof(u64), s>>>(a, n);
                   else sample_sorted<T, 1024><<<B, 1024, n * sizeof(u64), s>>>(a, n));
        dl_prof_end(s);
        return dl_launch_status();
    }
    smp_layout(a, (char *)ws);
    if ((long long)B * a.chunks > 0x7fffffffLL) return DL_ERR_UNSUPPORTED;
    const int blocks = B * a.chunks;
    // (settings on the device: the kernels look for themselves whether a row has cuts)
    const bool may_cut = top_k || top_p || (top_k_all > 0 && top_k_all < V) || !(top_p_all >= 1.0f);
    DL_BY_TYPE(type, T, DL_TIMED("sample_max", s, (sample_max<T><<<blocks, SMP_THREADS, 0, s>>>(a)));
               if (may_cut) DL_TIMED("sample_hist", s, (sample_hist<T><<<blocks, SMP_THREADS, 0, s>>>(a)));
               DL_TIMED("sample_collect", s, (sample_collect<T><<<blocks, SMP_THREADS, 0, s>>>(a)));
               DL_TIMED("sample_draw", s, (sample_draw<T><<<B, SMP_DRAW_THREADS, 0, s>>>(a))));
    return dl_launch_status();
}
