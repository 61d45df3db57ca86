// Sampling one index per row of logits, with temperature, top-k, top-p and min-p, from given random numbers.
//
// A row's indices are ordered by logit, descending, equal ones by index.  With w_i = exp((l_i - max l) / T):
//   top-k   keeps the first k;   top-p  of these the shortest prefix whose weights reach p times the sum over these (one at least);
//   min-p   of these the ones with w_i >= m (the first stays).   Whatever is kept is therefore a prefix of the order, and its end
//   - the cut - is one (logit, index) pair.
//   The draw: in index order, the first kept one whose running sum of weights exceeds u times the kept sum.
// T <= 0, p <= 0, k = 1 and m > 1 leave the first alone.  NaN counts as -infinity; a row without a larger logit gives -1.
//
// Neighbouring running sums lie close together, so weights are 64-bit integers, round(2^shift w) with shift = min(51, 62 - ceil(log2 V)),
// from exponentials in double: sums fit, are exact in any order - blocks and atomics can split them as they like, every run gives the
// same index - and a weight is off by 2^-(shift + 1), 2^-46 at V = 131072.  Only top-p's limit, and the weight before the classes that its
// cut can be in, come from other sums in rows of more than SMP_WAVE columns: of classes (smp_class_term), whole numbers as well, off from the
// weights' by as much as a weight and a few roundings of a double.
//
// Up to 64 columns: a few lanes per row compare every pair.  Up to SMP_WAVE: a wavefront per row, in its registers.  More: a block per row
// (sample_row), which reads it anew for every pass, mostly from the L2; or, for few long rows, four launches over pieces of rows
// (sample_max, sample_hist, sample_collect, sample_draw).  Both go the same way:
//   - the largest logit;
//   - number or weight of the logits in SMP_BINS classes of (max - l) / T, a monotone function of l: they say which classes the cuts
//     fall into;
//   - the weights of what lies before those classes, piece by piece of the row, and a list of the indices in them (with a small
//     enough top-k: a list of all that is kept, and no sums over the row);
//   - the list, sorted, gives the cut; then the piece that the target falls into, then the index.  A list that is too long
//     (many equal logits) is searched over the whole row instead.
//
// What bounds it: short rows, the chain of barriers and wavefront sums; long ones, instructions per logit - 26 for its class's sum, an
// exponential's 30 for the few that are kept.  us: 256 rows of 131072 fp32, top-p of 0.9: 100 (largest 20, classes 25, pieces and list
// 26, the rest 22; 260 in four launches with library exponentials); one row of 49999 bf16, all filters: 15; 64 rows of 32768
// fp16, top-k up to 80: 17, 32 with a row that has no top-k; 8192 x 1000 fp32, top-k and top-p: 45 (178 sorted in LDS); 8192 x 10: 5.
#include "dl_types.h"

#define SMP_WAVE 1024
#define SMP_BINS 2048
#define SMP_BINS_PER_Z 32.0  // classes per unit of (max - l) / T: the last one holds what weighs less than e^-63.9, so nothing
#define SMP_LIST 4096
#define SMP_THREADS 256
#define SMP_MOST_ROWS (1 << 21)  // of a launch (2^32 work items)
#define SMP_DRAW_THREADS 1024
#define SMP_MAX_CHUNKS 256
#define SMP_GATHER 128  // logits that a wavefront gathers: fewer than 64 left and one of every lane
#define SMP_FEW_LISTED 128
#define SMP_FEW 768  // top-k up to this goes by the threads' largest logits

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
    double scale, p, u;  // log2(e) / T
    double classes;      // SMP_BINS_PER_Z / T: classes per logit
    u64 least;           // min-p's weight
    int k;
    bool first_only, cut_k, cut_p;
};
__device__ __forceinline__ SampleRow smp_row(const SampleArgs &a, int b) {
    SampleRow r;
    const float T = a.temperature ? a.temperature[b] : a.T, p = a.top_p ? a.top_p[b] : a.p, m = a.min_p ? a.min_p[b] : a.m;
    const int k = a.top_k ? a.top_k[b] : a.k;
    const float u = a.uniform[b];
    r.first_only = !(T > 0.0f) || !(p > 0.0f) || !(m <= 1.0f) || k == 1;
    r.scale = 1.44269504088896341 / (double)T;
    r.classes = SMP_BINS_PER_Z / (double)T;
    r.p = p;
    r.least = m > 0.0f && m <= 1.0f ? (u64)ceil(ldexp((double)m, a.shift)) : 0;
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

// round(2^shift exp((l - max) / T)).  2^y = 2^n 2^f, |f| <= 1/2: 2^f by its polynomial through the Chebyshev nodes of degree 10 (off by
// 2^-51.5), both roundings to whole numbers by adding a power of two: double instructions, which run at float's rate here.
// 2^shift at the maximum itself, 0 at -infinity.
__device__ __forceinline__ u64 smp_fixed(uint32_t key, uint32_t top, const SampleRow &r, int shift) {
    const float M = smp_logit(top);
    if (M > 3.4e38f && __builtin_isinf(M)) return key == top ? 1ull << shift : 0;
    const double y = fmax(((double)smp_logit(key) - (double)M) * r.scale, -1000.0);  // (0 times -infinity, T infinite: -1000)
    const double n = y + 6755399441055744.0, f = y - (n - 6755399441055744.0);
    double e = 7.072585949269223e-09;
    e = fma(e, f, 1.0208690299958306e-07);
    e = fma(e, f, 1.321544258792169e-06);
    e = fma(e, f, 1.5252657260200837e-05);
    e = fma(e, f, 0.0001540353044173605);
    e = fma(e, f, 0.0013333558230164974);
    e = fma(e, f, 0.009618129107606888);
    e = fma(e, f, 0.05550410866444772);
    e = fma(e, f, 0.24022650695910097);
    e = fma(e, f, 0.69314718055995);
    e = fma(e, f, 1.0);
    const double x = ldexp(e, (int)(uint32_t)__double_as_longlong(n) + shift) + 4503599627370496.0;
    return (u64)__double_as_longlong(x) & ((1ull << 52) - 1);
}
// weight of an index that no cut but min-p takes away
__device__ __forceinline__ u64 smp_weight(uint32_t key, uint32_t top, const SampleRow &r, int shift) {
    const u64 w = smp_fixed(key, top, r, shift);
    return w >= r.least || key == top ? w : 0;
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
__device__ __forceinline__ void smp_sort(u64 *pairs, int n) {
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

// The same for n pairs of any number (all different; `size` slots, n <= size): few by counting who is larger, without a barrier per
// step (64 of them: 1 us for 4).
template <int THREADS>
__device__ __forceinline__ void smp_order(u64 *pairs, int n) {
    if (n <= 512) {
        const u64 mine = (int)threadIdx.x < n ? pairs[threadIdx.x] : 0;
        int rank = 0;
        __syncthreads();
        if ((int)threadIdx.x < n) {
#pragma unroll 8
            for (int j = 0; j < n; ++j) rank += pairs[j] > mine;
        }
        __syncthreads();
        if ((int)threadIdx.x < n) pairs[rank] = mine;
        __syncthreads();
        return;
    }
    int size = 1024;
    while (size < n) size <<= 1;
    for (int i = n + threadIdx.x; i < size; i += THREADS) pairs[i] = 0;
    smp_sort<THREADS>(pairs, size);
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
    const u64 w = r.first_only ? (key == top ? 1ull << a.shift : 0) : smp_fixed(key, top, r, a.shift);
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
    const bool keep = alive && (rank == 0 || (!r.first_only && rank < r.k && in_p && w >= r.least));
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

// In index order, over [i0, i1): the first index whose running sum of kept weights exceeds `target`; a thread per run of indices.
template <typename T, int THREADS>
__device__ __forceinline__ void smp_draw(const SampleArgs &a, const SampleRow &r, int b, int i0, int i1, u64 cut, uint32_t top, u64 target, u64 *red) {
    const T *row = (const T *)a.logits + b * a.ldl;
    const int per = (i1 - i0 + THREADS - 1) / THREADS, begin = min(i0 + (int)threadIdx.x * per, i1), end = min(begin + per, i1);
    u64 mine = 0, total;
    // 16 at a time: which of them are kept, then their weights, the lanes' first ones together
    for (int i0 = begin; i0 < end; i0 += 16) {
        uint32_t kept = 0;
#pragma unroll
        for (int u = 0; u < 16; ++u) kept |= (uint32_t)(i0 + u < end && smp_pair(smp_key((float)row[i0 + u < end ? i0 + u : begin]), i0 + u) >= cut) << u;
        for (; kept; kept &= kept - 1) mine += smp_weight(smp_key((float)row[i0 + __builtin_ctz(kept)]), top, r, a.shift);
    }
    u64 run = smp_scan<THREADS>(mine, total, red);
    // in the run of the thread that it falls into: a wavefront, an index a lane
    __shared__ int chosen;
    __shared__ u64 chosen_run;
    if (run <= target && target < run + mine) chosen = begin, chosen_run = run;
    __syncthreads();
    if (threadIdx.x >= 64) return;
    run = chosen_run;
    for (int i = chosen + (int)threadIdx.x;; i += 64) {
        const uint32_t key = i < i1 ? smp_key((float)row[i]) : 0;
        u64 up, sum = i < i1 && smp_pair(key, i) >= cut ? smp_weight(key, top, r, a.shift) : 0;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            up = __shfl_up(sum, o);
            if ((int)threadIdx.x >= o) sum += up;
        }
        const u64 past = __ballot(run + sum > target);
        if (past) {
            if ((int)threadIdx.x == __builtin_ctzll(past)) a.out[b] = i;
            return;
        }
        run += __shfl(sum, 63);
        if (i - (int)threadIdx.x + 64 >= i1) return;
    }
}

// All that top-k keeps is in a list of n <= SMP_FEW_LISTED: the cuts and the draw by one wavefront, two pairs a lane, every pair against
// every other one (no barrier and no sorting).  The list's room behind the pairs takes their weights.
__device__ __forceinline__ void smp_few_draw(const SampleArgs &a, const SampleRow &r, int b, uint32_t top, u64 *pairs, int n) {
    const int lane = threadIdx.x & 63;
    u64 *const weights = pairs + SMP_FEW_LISTED;
    u64 p[2], w[2], before[2] = {}, run[2] = {}, in_k = 0, all = 0;
    int rank[2] = {};
#pragma unroll
    for (int m = 0; m < 2; ++m) {
        const int i = m * 64 + lane;
        p[m] = i < n ? pairs[i] : 0;
        w[m] = i < n ? smp_fixed((uint32_t)(p[m] >> 32), top, r, a.shift) : 0;
        weights[i] = w[m];
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll 8
    for (int j = 0; j < n; ++j) {
        const u64 pj = pairs[j], wj = weights[j];
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            const bool ahead = pj > p[m];
            rank[m] += ahead;
            before[m] += ahead ? wj : 0;
        }
    }
#pragma unroll
    for (int m = 0; m < 2; ++m) in_k += rank[m] < r.k ? w[m] : 0;
    const double limit = r.p * (double)smp_wave_sum(in_k);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
    for (int m = 0; m < 2; ++m) {
        const bool stays = (!r.cut_p || (double)before[m] < limit) && (w[m] >= r.least || (uint32_t)(p[m] >> 32) == top);
        if (!(p[m] != 0 && rank[m] < r.k && (rank[m] == 0 || stays))) w[m] = 0;  // (of weight 0: never drawn)
        weights[m * 64 + lane] = w[m];
        all += w[m];
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll 8
    for (int j = 0; j < n; ++j) {
        const u64 wj = weights[j];
        const uint32_t at = (uint32_t)pairs[j];
#pragma unroll
        for (int m = 0; m < 2; ++m) run[m] += at >= (uint32_t)p[m] ? wj : 0;  // (indices are complements: those up to its own)
    }
    const u64 target = smp_target(r, smp_wave_sum(all));
#pragma unroll
    for (int m = 0; m < 2; ++m)
        if (w[m] > 0 && run[m] > target && run[m] - w[m] <= target) a.out[b] = (long long)(0xFFFFFFFFu - (uint32_t)p[m]);
}

// ---------------------------------------------------------------------------------- a wavefront per row
// Up to SMP_WAVE columns, N a lane: index e * 64 + lane.  Cuts by bisection over the keys - the largest one that k logits, or that
// p of the weight, reach - and equal keys at the cut by index; a small top-k leaves a list for smp_few_draw.
template <typename T, int N>
__global__ __launch_bounds__(SMP_THREADS) void sample_wave(SampleArgs a) {
    __shared__ u64 lists[SMP_THREADS / 64][2 * SMP_FEW_LISTED];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const long long b0 = (long long)blockIdx.x * (SMP_THREADS / 64) + wave;
    if (b0 >= a.B) return;  // (no barrier below)
    const int b = (int)b0;
    const T *row = (const T *)a.logits + b * a.ldl;
    const SampleRow r = smp_row(a, b);
    uint32_t key[N], top = 0;
#pragma unroll
    for (int e = 0; e < N; ++e) {
        key[e] = e * 64 + lane < a.V ? smp_key((float)row[e * 64 + lane]) : 0;
        top = max(top, key[e]);
    }
    top = smp_wave_max(top);
    if (top <= SMP_DEAD || r.first_only) {
        int first = -1;
#pragma unroll
        for (int e = N - 1; e >= 0; --e) {
            const u64 equal = __ballot(key[e] == top);
            if (equal) first = e * 64 + __builtin_ctzll(equal);
        }
        if (lane == 0) a.out[b] = top <= SMP_DEAD ? -1 : first;
        return;
    }
    const auto reach = [&](uint32_t least) {  // logits of this key or a larger one
        int n = 0;
#pragma unroll
        for (int e = 0; e < N; ++e) n += __popcll(__ballot(key[e] >= least));
        return n;
    };
    // keeps the first `most` of the logits with key `least`, and all larger ones
    uint32_t kept = 0;
    const auto keep = [&](uint32_t least, int most) {
        int before = 0;
        uint32_t now = 0;
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const u64 equal = __ballot(key[e] == least);
            const bool stays = key[e] > least || (key[e] == least && before + __popcll(equal & ((1ull << lane) - 1)) < most);
            now |= (uint32_t)stays << e;
            before += __popcll(equal);
        }
        kept = now;
    };
    uint32_t lo = SMP_DEAD + 1;
    int most = a.V;
    if (r.cut_k && reach(lo) > r.k) {
        uint32_t hi = top;
        int n = 0;
        while (lo < hi) {
            const uint32_t mid = lo + (hi - lo) / 2 + 1;
            n = reach(mid);
            if (n >= r.k) lo = mid;
            else hi = mid - 1;
            if (n == r.k) break;
        }
        n = reach(lo);
        if (n <= SMP_FEW_LISTED) {
            int at = 0;
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const u64 takes = __ballot(key[e] >= lo);
                if (key[e] >= lo) lists[wave][at + __popcll(takes & ((1ull << lane) - 1))] = smp_pair(key[e], e * 64 + lane);
                at += __popcll(takes);
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            smp_few_draw(a, r, b, top, lists[wave], n);
            return;
        }
        most = r.k - reach(lo + 1);
    }
    keep(lo, most);
    u64 w[N], sum = 0;
#pragma unroll
    for (int e = 0; e < N; ++e) {
        w[e] = kept >> e & 1 ? smp_fixed(key[e], top, r, a.shift) : 0;
        sum += w[e];
    }
    if (r.cut_p) {
        const double limit = r.p * (double)smp_wave_sum(sum);
        const auto weigh = [&](uint32_t least) {
            u64 t = 0;
#pragma unroll
            for (int e = 0; e < N; ++e) t += key[e] >= least ? w[e] : 0;
            return smp_wave_sum(t);
        };
        uint32_t hi = top;
        int from_lo = reach(lo), past_hi = 0;
        while (lo < hi && from_lo - past_hi > 1) {
            const uint32_t mid = lo + (hi - lo) / 2 + 1;
            const int n = reach(mid);
            if ((double)weigh(mid) >= limit) lo = mid, from_lo = n;
            else hi = mid - 1, past_hi = n;
        }
        if (lo < hi) {  // one logit is left between them
            lo = 0;
#pragma unroll
            for (int e = 0; e < N; ++e) lo = key[e] <= hi ? max(lo, key[e]) : lo;
            lo = smp_wave_max(lo);
        }
        // of the equal ones those that what lies before them does not reach the limit (the first of the row always)
        const u64 larger = weigh(lo + 1), each = smp_fixed(lo, top, r, a.shift);
        int before = 0;
        sum = 0;
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const u64 equal = __ballot(key[e] == lo);
            const int mine = before + __popcll(equal & ((1ull << lane) - 1));
            if (key[e] < lo || (key[e] == lo && !((double)(larger + mine * each) < limit) && !(lo == top && mine == 0))) w[e] = 0;
            before += __popcll(equal);
        }
    }
    sum = 0;
#pragma unroll
    for (int e = 0; e < N; ++e) {
        if (w[e] < r.least && key[e] != top) w[e] = 0;
        sum += w[e];
    }
    const u64 target = smp_target(r, smp_wave_sum(sum));
    u64 run = 0;
#pragma unroll
    for (int e = 0; e < N; ++e) {
        u64 upto = w[e];
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const u64 up = __shfl_up(upto, o);
            if (lane >= o) upto += up;
        }
        const u64 past = __ballot(run + upto > target);
        if (past) {
            if (lane == 0) a.out[b] = e * 64 + __builtin_ctzll(past);
            return;
        }
        run += __shfl(upto, 63);
    }
}

// ---------------------------------------------------------------------------------- rows split over blocks
// The class of a logit: (max - l) / T in 32nds, to the nearest one, and what is left of it (-1/2 .. 1/2; within the last class: anything)
// (of a finite maximum; -infinity and NaN are of the last class)
__device__ __forceinline__ int smp_class(float l, double M, const SampleRow &r, double &rest) {
    const double y = fmin((M - (double)l) * r.classes, (double)(SMP_BINS - 1));  // (infinity times 0, T infinite: the last class)
    const double n = y + 6755399441055744.0;
    rest = y - (n - 6755399441055744.0);
    return (int)(uint32_t)__double_as_longlong(n);
}
__device__ __forceinline__ int smp_bin(uint32_t key, uint32_t top, const SampleRow &r, double &rest) {
    const float M = smp_logit(top);
    if (__builtin_isinf(M)) {  // only its equals weigh anything
        rest = 0.0;
        return key == top ? 0 : SMP_BINS - 1;
    }
    return smp_class(smp_logit(key), (double)M, r, rest);
}
__device__ __forceinline__ int smp_bin(uint32_t key, uint32_t top, const SampleRow &r) {
    double rest;
    return smp_bin(key, top, r, rest);
}
// A class's weight is e^(-class / 32) times the sum of e^(-rest / 32) over its logits; that sum, whose terms lie within 1.6 % of 1, is kept
// as 2^(62 - ceil(log2 V)) of it: a polynomial of degree 5 and no power of two per logit.  The polynomial is Taylor's with d^6 / 720 taken
// into the even terms (least largest error on |d| <= 1/64 with 1 kept at 0): off by 2^-50.1; of degree 4, Taylor's is off by 2^-36.9, which
// moves a nucleus' end by a logit where its limit comes that near to one.
__device__ __forceinline__ u64 smp_class_term(double rest, double unit) {
    const double d = rest * (-1.0 / SMP_BINS_PER_Z);
    double e = fma(d, 1.0 / 120.0, 0.04166713877524326);
    e = fma(e, d, 1.0 / 6.0);
    e = fma(e, d, 0.49999999996433814);
    e = fma(e, d, 1.0);
    e = fma(e, d, 1.0);
    return (u64)__double_as_longlong(fma(e, unit, 4503599627370496.0)) & ((1ull << 52) - 1);
}
__device__ __forceinline__ u64 smp_class_weight(int bin, u64 sum, int shift, int term_shift) {
    return sum ? (u64)((double)sum * exp(bin * (-1.0 / SMP_BINS_PER_Z)) * ldexp(1.0, shift - term_shift) + 0.5) : 0;
}
// terms of 2^term_shift: under 2^52, and their sum under 2^63
__device__ __forceinline__ int smp_term_shift(const SampleArgs &a) { return a.shift < 51 ? a.shift : 50; }
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
    const double unit = ldexp(1.0, smp_term_shift(a));
    for (int i = c * a.chunk + threadIdx.x; i < i1; i += SMP_THREADS) {
        const uint32_t key = smp_key((float)row[i]);
        if (key <= SMP_DEAD) continue;
        double rest;
        const int bin = smp_bin(key, top, r, rest);
        if (r.cut_k) atomicAdd(&count[bin], 1u);
        if (r.cut_p) atomicAdd(&weight[bin], smp_class_term(rest, unit));
    }
    __syncthreads();
    for (int i = threadIdx.x; i < SMP_BINS; i += SMP_THREADS) {
        if (count[i]) atomicAdd(&a.bin_count[(long long)b * SMP_BINS + i], count[i]);
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

// (count and sum: the row's classes, in LDS or in memory; those that no cut asks for are zero)
template <int THREADS>
__device__ __forceinline__ SampleCut smp_resolve(const SampleArgs &a, const uint32_t *count, const u64 *sum, const SampleRow &r, u64 *red, SampleCut *shared) {
    constexpr int PER = SMP_BINS / THREADS;
    uint32_t n[PER];
    u64 w[PER], mine_n = 0, mine_w = 0, all_n, all_w;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        n[j] = count[threadIdx.x * PER + j];
        w[j] = smp_class_weight(threadIdx.x * PER + j, sum[threadIdx.x * PER + j], a.shift, smp_term_shift(a));
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
    if (k_bin < SMP_BINS) high += smp_class_weight(k_bin, sum[k_bin], a.shift, smp_term_shift(a));
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
    if (cuts) cut = smp_resolve<SMP_THREADS>(a, a.bin_count + (long long)b * SMP_BINS, a.bin_weight + (long long)b * SMP_BINS, r, red, &shared);
    const T *row = (const T *)a.logits + b * a.ldl;
    const int i1 = min((c + 1) * (long long)a.chunk, (long long)a.V);
    const int lane = threadIdx.x & 63;
    u64 sum = 0;
    for (int i0 = c * a.chunk; i0 < i1; i0 += SMP_THREADS) {
        const int i = i0 + threadIdx.x;
        const uint32_t key = i < i1 ? smp_key((float)row[i]) : 0;
        const int bin = key <= SMP_DEAD ? SMP_BINS : smp_bin(key, top, r);
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
__device__ __forceinline__ void smp_row_sums(const SampleArgs &a, const SampleRow &r, int b, uint32_t top, uint32_t least, u64 &count, u64 &weight, u64 *red) {
    const T *row = (const T *)a.logits + b * a.ldl;
    u64 n = 0, w = 0;
    for (int i = threadIdx.x; i < a.V; i += THREADS) {
        const uint32_t key = smp_key((float)row[i]);
        if (key < least || key <= SMP_DEAD) continue;
        ++n;
        w += smp_fixed(key, top, r, a.shift);
    }
    smp_scan<THREADS>(n, count, red);
    smp_scan<THREADS>(w, weight, red);
}
// The least and the largest key in classes [first, last]
template <typename T, int THREADS>
__device__ __forceinline__ void smp_key_range(const SampleArgs &a, const SampleRow &r, int b, uint32_t top, int first, int last, uint32_t &low, uint32_t &high, u64 *red) {
    const T *row = (const T *)a.logits + b * a.ldl;
    uint32_t lo = 0, hi = 0;  // (lo: of the complements)
    for (int i = threadIdx.x; i < a.V; i += THREADS) {
        const uint32_t key = smp_key((float)row[i]);
        if (key <= SMP_DEAD) continue;
        const int bin = smp_bin(key, top, r);
        if (bin < first || bin > last) continue;
        hi = max(hi, key), lo = max(lo, ~key);
    }
    high = smp_max<THREADS>(hi, red);
    low = ~smp_max<THREADS>(lo, red);
}

// The cut of a row whose open classes hold more than the list: by bisection over the keys, then over equal ones by index.
template <typename T, int THREADS>
__device__ __forceinline__ u64 smp_search(const SampleArgs &a, const SampleRow &r, const SampleCut &c, int b, uint32_t top, u64 *red) {
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
        sum = w + ties * smp_fixed(lo, top, r, a.shift);
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
        const u64 each = smp_fixed(lo, top, r, a.shift);
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

// The cut from the list of the n indices in open classes (from `list`, or in pairs already where that is null): sorted into pairs, the
// first `kept` of them stay.
template <int THREADS>
__device__ __forceinline__ u64 smp_list_cut(const SampleArgs &a, const SampleRow &r, const SampleCut &c, uint32_t top, u64 *pairs, int n, const u64 *list,
                            u64 *red, u64 &cut) {
    if (list)
        for (int i = threadIdx.x; i < n; i += THREADS) pairs[i] = list[i];
    __syncthreads();
    smp_order<THREADS>(pairs, n);
    // in order: classes [p_first, p_last], then k_bin where that is another one
    const int per = (n + THREADS - 1) / THREADS, begin = min((int)threadIdx.x * per, n), end = min(begin + per, n);
    u64 in_k = 0, k_from = 0, kept = 0, mine = 0, total;
    for (int j = begin; j < end; ++j) k_from += smp_bin((uint32_t)(pairs[j] >> 32), top, r) != c.k_bin;  // entries before the k-th's class
    smp_scan<THREADS>(k_from, total, red);
    k_from = total;
    const u64 k_end = c.k_bin < SMP_BINS ? k_from + ((u64)r.k - c.k_before) : (u64)n;  // list entries that top-k keeps
    for (int j = begin; j < end; ++j) {
        const u64 w = smp_fixed((uint32_t)(pairs[j] >> 32), top, r, a.shift);
        if ((u64)j >= k_from && (u64)j < k_end) in_k += w;
        mine += w;
    }
    smp_scan<THREADS>(in_k, total, red);
    const double limit = r.p * (double)(c.k_weight + total);
    u64 before = smp_scan<THREADS>(mine, total, red) + c.p_weight;
    for (int j = begin; j < end; ++j) {
        const uint32_t key = (uint32_t)(pairs[j] >> 32);
        const bool in_p = !r.cut_p || (smp_bin(key, top, r) <= c.p_last && ((double)before < limit || (j == 0 && c.p_weight == 0)));
        if ((u64)j >= k_end || !in_p) break;
        before += smp_fixed(key, top, r, a.shift);
        ++kept;
    }
    smp_scan<THREADS>(kept, total, red);
    cut = total ? pairs[total - 1] : pairs[0] + 1;
    return total;
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
        const SampleCut c = smp_resolve<THREADS>(a, a.bin_count + (long long)b * SMP_BINS, a.bin_weight + (long long)b * SMP_BINS, r, red, &shared);
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
            const u64 kept = smp_list_cut<THREADS>(a, r, c, top, pairs, (int)n, a.list + (long long)b * SMP_LIST, red, cut);
            for (int j = threadIdx.x; j < (int)kept; j += THREADS) {
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
    smp_draw<T, THREADS>(a, r, b, c * a.chunk, (int)min((c + 1) * (long long)a.chunk, (long long)a.V), cut, top, shared.k_weight, red);
}

// ---------------------------------------------------------------------------------- a block per row
// A list in LDS that wavefronts append to; `size` counts what did not fit as well
__device__ __forceinline__ void smp_append(u64 *list, uint32_t *size, bool take, u64 pair) {
    const u64 takes = __ballot(take);
    if (!take) return;
    const int lane = threadIdx.x & 63, leader = __builtin_ctzll(takes);
    uint32_t at = 0;
    if (lane == leader) at = atomicAdd(size, (uint32_t)__popcll(takes));
    at = (uint32_t)__builtin_amdgcn_readlane((int)at, leader) + __popcll(takes & ((1ull << lane) - 1));
    if (at < SMP_LIST) list[at] = pair;
}

// A row's elements, 16 bytes at a time: a wavefront takes a run of units.  The up to E - 1 elements before the first whole unit and behind
// the last one are single ones.  (Rows are read again for every pass, mostly from the L2: held in registers they left too few of those.)
template <typename T>
struct SampleReader {
    static constexpr int E = 16 / sizeof(T), THREADS = SMP_DRAW_THREADS;
    const T *row;
    int V, head, units, run;  // units of a wavefront (whole groups of 64)

    __device__ __forceinline__ SampleReader(const T *row, int V) : row(row), V(V) {
        head = min((int)((16 - ((uintptr_t)row & 15)) & 15) / (int)sizeof(T), V);
        units = (V - head) / E;
        run = (units + THREADS - 1) / THREADS * 64;
    }
    __device__ __forceinline__ dl_words unit(int j) const { return *reinterpret_cast<const dl_words *>(row + head + j * E); }
    __device__ __forceinline__ int first() const { return (threadIdx.x >> 6) * run + (threadIdx.x & 63); }
    // f(unit number, values, whether the thread has one), by all threads of a wavefront
    template <typename F>
    __device__ __forceinline__ void units_of(F f) const {
        constexpr int AHEAD = E == 4 ? 4 : 2;  // units in flight while as many are worked on
        dl_words v[AHEAD], next[AHEAD];
        const auto fetch = [&](dl_words (&to)[AHEAD], int i0) {
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {
                const int i = i0 + u * 64;
                if (i < run && first() + i < units) to[u] = unit(first() + i);
            }
        };
        fetch(v, 0);
#pragma unroll 1
        for (int i0 = 0; i0 < run; i0 += AHEAD * 64) {
            fetch(next, i0 + AHEAD * 64);
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {
                const int i = i0 + u * 64, j = first() + i;
                if (i < run) {
                    float values[E];
                    dl_unpack<T>(v[u], values);
                    f(j, values, j < units);
                }
            }
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) v[u] = next[u];
        }
    }
    // the single element of a thread: its index, or -1
    __device__ __forceinline__ int single() const {
        const int t = threadIdx.x, tail = head + units * E;
        return t < head ? t : tail + (t - head) < V ? tail + (t - head) : -1;
    }
    // the thread's largest element, as a key
    __device__ __forceinline__ uint32_t largest() const {
        const int i = single();
        float m = i >= 0 ? fmaxf((float)row[i], -INFINITY) : -INFINITY;  // (the larger of a NaN and a number is the number)
        units_of([&](int, const float (&v)[E], bool has) {
#pragma unroll
            for (int e = 0; e < E; ++e) m = has ? fmaxf(m, v[e]) : m;
        });
        return smp_key(m);
    }
    // f(key, index) for every element
    template <typename F>
    __device__ __forceinline__ void each(F f) const {
        const int i = single();
        if (i >= 0) f(smp_key((float)row[i]), i);
        units_of([&](int j, const float (&v)[E], bool has) {
            if (!has) return;
#pragma unroll
            for (int e = 0; e < E; ++e) f(smp_key(v[e]), head + j * E + e);
        });
    }
    // Appends the elements that take(value) says (not a NaN) to a list in LDS; `size` counts what does not fit as well
    template <typename F>
    __device__ __forceinline__ void list(u64 *pairs, uint32_t *size, F take) const {
        const int i = single();
        const float l = i >= 0 ? (float)row[i] : 0.0f;
        smp_append(pairs, size, i >= 0 && take(l), smp_pair(smp_key(l), i));
        units_of([&](int j, const float (&v)[E], bool has) {
            uint32_t mask = 0;
#pragma unroll
            for (int e = 0; e < E; ++e) mask |= (uint32_t)(has && take(v[e])) << e;
            if (__ballot(mask != 0) == 0) return;
#pragma unroll
            for (int e = 0; e < E; ++e) smp_append(pairs, size, mask >> e & 1, smp_pair(smp_key(v[e]), head + j * E + e));
        });
    }
};

// The least key (above -infinity) of a class or a lower one: classes go down as keys go up.  32 steps, by every thread alike.
__device__ __forceinline__ uint32_t smp_first_key(int bin, uint32_t top, const SampleRow &r) {
    uint32_t lo = SMP_DEAD + 1, hi = top;
    while (lo < hi) {
        const uint32_t mid = lo + (hi - lo) / 2;
        if (smp_bin(mid, top, r) <= bin) hi = mid;
        else lo = mid + 1;
    }
    return lo;
}

// The same for a longer list.
template <int THREADS>
__device__ __forceinline__ void smp_list_draw(const SampleArgs &a, const SampleRow &r, int b, uint32_t top, u64 *pairs, int n, u64 *red) {
    smp_order<THREADS>(pairs, n);
    n = min(n, r.k);
    const int per = (n + THREADS - 1) / THREADS, begin = min((int)threadIdx.x * per, n), end = min(begin + per, n);
    u64 mine = 0, total, kept = 0;
    for (int j = begin; j < end; ++j) mine += smp_fixed((uint32_t)(pairs[j] >> 32), top, r, a.shift);
    u64 before = smp_scan<THREADS>(mine, total, red);
    const double limit = r.p * (double)total;
    for (int j = begin; j < end; ++j) {
        const u64 w = smp_fixed((uint32_t)(pairs[j] >> 32), top, r, a.shift);
        if (j > 0 && ((r.cut_p && !((double)before < limit)) || (w < r.least && (uint32_t)(pairs[j] >> 32) != top))) break;
        before += w;
        ++kept;
    }
    smp_scan<THREADS>(kept, total, red);
    n = (int)total;
    // what is left in index order: the halves of the pairs change places
    for (int j = threadIdx.x; j < n; j += THREADS) pairs[j] = pairs[j] << 32 | pairs[j] >> 32;
    __syncthreads();
    smp_order<THREADS>(pairs, n);
    const int per_n = (n + THREADS - 1) / THREADS, first = min((int)threadIdx.x * per_n, n), last = min(first + per_n, n);
    mine = 0;
    for (int j = first; j < last; ++j) mine += smp_fixed((uint32_t)pairs[j], top, r, a.shift);
    u64 run = smp_scan<THREADS>(mine, total, red);
    const u64 target = smp_target(r, total);
    if (run <= target && target < run + mine)
        for (int j = first; j < last; ++j) {
            run += smp_fixed((uint32_t)pairs[j], top, r, a.shift);
            if (run > target) {
                a.out[b] = (long long)(0xFFFFFFFFu - (uint32_t)(pairs[j] >> 32));
                break;
            }
        }
}

template <typename T>
__global__ __launch_bounds__(SMP_DRAW_THREADS) void sample_row(SampleArgs a) {
    constexpr int THREADS = SMP_DRAW_THREADS, E = 16 / sizeof(T), WAVES = THREADS / 64;
    __shared__ union {
        struct {
            u64 weight[SMP_BINS];
            uint32_t count[SMP_BINS];
        } bins;
        struct {
            float value[WAVES * SMP_GATHER];
            uint32_t index[WAVES * SMP_GATHER];
        } gathered;
    } of;
    __shared__ u64 pairs[SMP_LIST], red[WAVES], slot[WAVES + 2], left;
    __shared__ uint32_t limit[4], listed, least;
    u64 *const weight = of.bins.weight;
    uint32_t *const count = of.bins.count;
    __shared__ SampleCut shared;
    __shared__ int chosen;
    const int b = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const SampleReader<T> row((const T *)a.logits + b * a.ldl, a.V);
    const SampleRow r = smp_row(a, b);
    if (threadIdx.x == 0) listed = 0;
    const uint32_t own = row.largest();
    const uint32_t top = smp_max<THREADS>(own, red);
    if (top <= SMP_DEAD) {
        if (threadIdx.x == 0) a.out[b] = -1;
        return;
    }
    if (r.first_only) {
        uint32_t low = 0;
        row.each([&](uint32_t key, int i) { low = key == top ? max(low, ~(uint32_t)i) : low; });
        low = smp_max<THREADS>(low, red);
        if (threadIdx.x == 0) a.out[b] = (long long)(uint32_t)~low;
        return;
    }
    if (r.cut_k && r.k <= SMP_FEW) {
        // k of the threads' largest logits reach some number, so at least k logits do, and hardly more: every thread has the largest of
        // its own.  A wavefront looks for that number, by bisection.
        count[threadIdx.x] = own;
        __syncthreads();
        if (wave == 0) {
            uint32_t v[WAVES], most = 0;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) v[w] = count[w * 64 + lane], most = max(most, v[w]);
            uint32_t lo = r.k <= 64 ? ~smp_wave_max(~most) : 0, hi = top;  // 64 reach the least of the lanes' largest
            while (lo < hi) {
                const uint32_t mid = lo + (hi - lo) / 2 + 1;
                int n = 0;
#pragma unroll
                for (int w = 0; w < WAVES; ++w) n += __popcll(__ballot(v[w] >= mid));
                if (n >= r.k) lo = mid;
                else hi = mid - 1;
                if (n >= r.k && n <= r.k + r.k / 8) break;
            }
            if (lane == 0) least = max(lo, SMP_DEAD + 1);
        }
        __syncthreads();
        const float from = smp_logit(least);
        row.list(pairs, &listed, [&](float l) { return l >= from; });
        __syncthreads();
        const uint32_t n = listed;
        if (n <= SMP_FEW_LISTED) {
            if (wave == 0) smp_few_draw(a, r, b, top, pairs, (int)n);
            return;
        }
        if (n <= SMP_LIST) {
            smp_list_draw<THREADS>(a, r, b, top, pairs, (int)n, red);
            return;
        }
        __syncthreads();  // (many equal ones)
        if (threadIdx.x == 0) listed = 0;
    }
    for (int i = threadIdx.x; i < SMP_BINS; i += THREADS) weight[i] = 0, count[i] = 0;
    __syncthreads();
    SampleCut c = {SMP_BINS, SMP_BINS, SMP_BINS, SMP_BINS, 0, 0, 0};
    if (r.cut_k) {
        row.each([&](uint32_t key, int) {
            if (key > SMP_DEAD) atomicAdd(&count[smp_bin(key, top, r)], 1u);
        });
        __syncthreads();
        SampleRow only_k = r;
        only_k.cut_p = false;
        c = smp_resolve<THREADS>(a, count, weight, only_k, red, &shared);
        if (c.k_bin < SMP_BINS && c.k_before + count[c.k_bin] <= SMP_LIST) {  // all that top-k keeps fits the list
            const float from = smp_logit(smp_first_key(c.k_bin, top, r));
            row.list(pairs, &listed, [&](float l) { return l >= from; });
            __syncthreads();
            smp_list_draw<THREADS>(a, r, b, top, pairs, (int)listed, red);
            return;
        }
    }
    if (r.cut_p) {
        const double unit = ldexp(1.0, smp_term_shift(a)), M = smp_logit(top);
        if (M <= 3.4028234663852886e38) {
            const auto add = [&](float l) {
                double rest;
                const int bin = smp_class(l, M, r, rest);
                atomicAdd(&weight[bin], smp_class_term(rest, unit));  // (what is dead as well: the last class weighs nothing)
            };
            const int i = row.single();
            if (i >= 0) add((float)row.row[i]);
            row.units_of([&](int, const float (&v)[E], bool has) {
                if (!has) return;
#pragma unroll
                for (int e = 0; e < E; ++e) add(v[e]);
            });
        } else {
            row.each([&](uint32_t key, int) {
                if (key == top) atomicAdd(&weight[0], smp_class_term(0.0, unit));
            });
        }
        __syncthreads();
        c = smp_resolve<THREADS>(a, count, weight, r, red, &shared);
    }
    // Pieces of the row in index order: the elements before the first unit, the wavefronts' runs of units, those behind.
    const auto slot_of = [&](int i) { return i < row.head ? 0 : i >= row.head + row.units * E ? WAVES + 1 : (i - row.head) / (row.run * E) + 1; };
    if (threadIdx.x < WAVES + 2) slot[threadIdx.x] = 0;
    // the classes' limits as logits: kept for certain from `sure` on, open are those of [p_from, sure) down to top-p's last class and [k_from, k_to)
    if (wave < 4) {
        const int bin = wave == 0 ? c.sure - 1 : wave == 1 ? c.p_last : wave == 2 ? c.k_bin - 1 : c.k_bin;
        const uint32_t key = bin < 0 ? top + 1 : bin >= SMP_BINS - 1 ? SMP_DEAD + 1 : smp_first_key(bin, top, r);
        if (lane == 0) limit[wave] = key;
    }
    __syncthreads();
    // (top + 1 of an infinite maximum is a NaN, which nothing reaches)
    const float sure = smp_logit(limit[0]), p_from = c.p_first < SMP_BINS ? smp_logit(limit[1]) : INFINITY,
                k_to = smp_logit(limit[2]), k_from = c.k_bin < SMP_BINS ? smp_logit(limit[3]) : INFINITY;
    const auto is_sure = [&](float l) { return l >= sure; };
    const auto is_open = [&](float l) { return !(l >= sure) && ((c.p_first < SMP_BINS && l >= p_from) || (c.k_bin < SMP_BINS && l >= k_from && !(l >= k_to))); };
    {
        const int i = row.single();
        const float l = i >= 0 ? (float)row.row[i] : -INFINITY;
        if (is_sure(l)) atomicAdd(&slot[slot_of(i)], smp_weight(smp_key(l), top, r, a.shift));
        smp_append(pairs, &listed, is_open(l), smp_pair(smp_key(l), i));
    }
    // Few of a nucleus' logits are kept, most wavefronts have some: they are gathered with their indices (where the classes' sums and counts
    // were), so that all lanes work on every exponential, and what is open is looked for among them only.
    const float from = c.k_bin < SMP_BINS ? k_from : c.p_first < SMP_BINS ? p_from : sure;
    float *const values = of.gathered.value + wave * SMP_GATHER;
    uint32_t *const indices = of.gathered.index + wave * SMP_GATHER;
    int waiting = 0;
    u64 sum = 0;
    const auto work_on = [&](int at, bool has) {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        const float l = has ? values[at] : -INFINITY;
        const uint32_t index = has ? indices[at] : 0;
        if (is_sure(l)) sum += smp_weight(smp_key(l), top, r, a.shift);
        smp_append(pairs, &listed, is_open(l), smp_pair(smp_key(l), index));
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    };
    if (!r.cut_k && !r.cut_p) {  // all of them
        row.units_of([&](int, const float (&v)[E], bool has) {
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const u64 w = smp_weight(smp_key(v[e]), top, r, a.shift);
                sum += has ? w : 0;
            }
        });
    } else {
        row.units_of([&](int j, const float (&v)[E], bool has) {
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const bool take = has && v[e] >= from;
                const u64 takes = __ballot(take);
                if (take) {
                    const int at = waiting + __popcll(takes & ((1ull << lane) - 1));
                    values[at] = v[e];
                    indices[at] = (uint32_t)(row.head + j * E + e);
                }
                waiting += __popcll(takes);
                if (waiting >= 64) waiting -= 64, work_on(waiting + lane, true);
            }
        });
        work_on(lane, lane < waiting);
    }
    sum = smp_wave_sum(sum);
    if (lane == 0) slot[wave + 1] = sum;
    __syncthreads();
    u64 cut = (u64)(SMP_DEAD + 1) << 32, total;
    const uint32_t n = listed;
    if (n > SMP_LIST) {
        cut = smp_search<T, THREADS>(a, r, c, b, top, red);
        if (threadIdx.x < WAVES + 2) slot[threadIdx.x] = 0;
        __syncthreads();
        sum = 0;
        row.units_of([&](int j, const float (&v)[E], bool has) {
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (has && smp_pair(smp_key(v[e]), row.head + j * E + e) >= cut) sum += smp_weight(smp_key(v[e]), top, r, a.shift);
        });
        sum = smp_wave_sum(sum);
        if (lane == 0) slot[wave + 1] = sum;
        const int i = row.single();
        if (i >= 0 && smp_pair(smp_key((float)row.row[i]), i) >= cut) atomicAdd(&slot[slot_of(i)], smp_weight(smp_key((float)row.row[i]), top, r, a.shift));
    } else if (n > 0) {
        const u64 kept = smp_list_cut<THREADS>(a, r, c, top, pairs, (int)n, nullptr, red, cut);
        for (int j = threadIdx.x; j < (int)kept; j += THREADS) {
            const u64 w = smp_weight((uint32_t)(pairs[j] >> 32), top, r, a.shift);
            if (w) atomicAdd(&slot[slot_of((int)(0xFFFFFFFFu - (uint32_t)pairs[j]))], w);
        }
    }
    __syncthreads();
    const u64 mine = threadIdx.x < WAVES + 2 ? slot[threadIdx.x] : 0, before = smp_scan<THREADS>(mine, total, red);
    const u64 target = smp_target(r, total);
    if (before <= target && target < before + mine) chosen = threadIdx.x, left = target - before;
    __syncthreads();
    const int piece = chosen, last = row.head + row.units * E;
    const int i0 = piece == 0 ? 0 : piece == WAVES + 1 ? last : row.head + (piece - 1) * row.run * E;
    smp_draw<T, THREADS>(a, r, b, i0, piece == 0 ? row.head : piece == WAVES + 1 ? a.V : min(i0 + row.run * E, last), cut, top, left, red);
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

// Whether a block takes a row of its own (its time goes by the row's length, whatever the number of rows up to the card's 256 CUs) or
// rows are split over blocks.  us for fp32 rows, block per row / split:
//   a small top-k (top_k_all in 1 .. SMP_FEW): 131072 columns, 1 row 25 / 40, 16 rows 25 / 51; 262144, 1 row 39 / 41, 16 rows 39 / 64
//   no cut at all: 32768, 1 row 23 / 22; 131072, 16 rows 70 / 24, 64 rows 70 / 41
//   else (top-p of 0.9): 65536, 1 row 43 / 42; 131072, 1 row 70 / 44, 16 rows 71 / 67, 64 rows 72 / 129
static bool smp_by_row(int B, int V, int top_k_all, bool may_cut) {
    if (top_k_all > 0 && top_k_all <= SMP_FEW) return V <= 262144 || B >= 16;
    if (!may_cut) return V <= 32768 || B >= 128;
    return V <= 65536 || B >= 16;
}
// (negative numbers stand for settings on the device: the kernels look for themselves whether a row has cuts)
static bool smp_may_cut(int V, int top_k_all, float top_p_all) { return top_k_all < 0 || (top_k_all > 0 && top_k_all < V) || !(top_p_all >= 1.0f); }

extern "C" size_t dl_sample_workspace_bytes(int B, int V, int top_k_all, float top_p_all) {
    if (B <= 0 || V <= SMP_WAVE || smp_by_row(B, V, top_k_all, smp_may_cut(V, top_k_all, top_p_all))) return 0;
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
    if (B > SMP_MOST_ROWS) {  // halves: each still has a block or a wavefront per row, and no workspace
        const int m = B / 2;
        const int rc = dl_sample(logits, ldl, type, uniform, temperature, top_k, top_p, min_p, temperature_all, top_k_all, top_p_all, min_p_all, out,
                                 ws, ws_bytes, m, V, stream);
        return rc != DL_OK ? rc : dl_sample((const char *)logits + m * ldl * dl_type_bytes(type), ldl, type, uniform + m,
                                            temperature ? temperature + m : nullptr, top_k ? top_k + m : nullptr, top_p ? top_p + m : nullptr,
                                            min_p ? min_p + m : nullptr, temperature_all, top_k_all, top_p_all, min_p_all, out + m, ws, ws_bytes,
                                            B - m, V, stream);
    }
    const int k_rule = top_k ? -1 : top_k_all;  // (as the size function was asked: by the number itself)
    const float p_rule = top_p ? -1.0f : top_p_all;
    const size_t need = dl_sample_workspace_bytes(B, V, k_rule, p_rule);
    if (need && !ws) return DL_ERR_NULL;
    if (ws_bytes < need) return DL_ERR_WORKSPACE;
    hipStream_t s = (hipStream_t)stream;
    SampleArgs a = {};
    a.logits = logits, a.ldl = ldl, a.uniform = uniform, a.temperature = temperature, a.top_k = top_k, a.top_p = top_p, a.min_p = min_p;
    a.T = temperature_all, a.k = top_k_all > 0 ? top_k_all : 0, a.p = top_p_all, a.m = min_p_all, a.out = out, a.B = B, a.V = V;
    int bits = 0;
    while ((1LL << bits) < V) ++bits;
    a.shift = 62 - bits < 51 ? 62 - bits : 51;
    if (V <= 64) {
        const int seg = V <= 8 ? 8 : V <= 16 ? 16 : V <= 32 ? 32 : 64;
        const long long blocks = ((long long)B * seg + SMP_THREADS - 1) / SMP_THREADS;
        dl_prof_begin("sample_pairs", s);
        DL_BY_TYPE(type, T, if (seg == 8) sample_pairs<T, 8><<<(int)blocks, SMP_THREADS, 0, s>>>(a);
                   else if (seg == 16) sample_pairs<T, 16><<<(int)blocks, SMP_THREADS, 0, s>>>(a);
                   else if (seg == 32) sample_pairs<T, 32><<<(int)blocks, SMP_THREADS, 0, s>>>(a);
                   else sample_pairs<T, 64><<<(int)blocks, SMP_THREADS, 0, s>>>(a));
        dl_prof_end(s);
        return dl_launch_status();
    }
    if (V <= SMP_WAVE) {
        const int blocks = dl_ceil_div(B, SMP_THREADS / 64);
        dl_prof_begin("sample_wave", s);
        DL_BY_TYPE(type, T, if (V <= 128) sample_wave<T, 2><<<blocks, SMP_THREADS, 0, s>>>(a);
                   else if (V <= 256) sample_wave<T, 4><<<blocks, SMP_THREADS, 0, s>>>(a);
                   else if (V <= 512) sample_wave<T, 8><<<blocks, SMP_THREADS, 0, s>>>(a);
                   else sample_wave<T, 16><<<blocks, SMP_THREADS, 0, s>>>(a));
        dl_prof_end(s);
        return dl_launch_status();
    }
    if (!need) {
        dl_prof_begin("sample_row", s);
        DL_BY_TYPE(type, T, sample_row<T><<<B, SMP_DRAW_THREADS, 0, s>>>(a));
        dl_prof_end(s);
        return dl_launch_status();
    }
    smp_layout(a, (char *)ws);
    const int blocks = B * a.chunks;  // (about 2048)
    DL_BY_TYPE(type, T, DL_TIMED("sample_max", s, (sample_max<T><<<blocks, SMP_THREADS, 0, s>>>(a)));
               if (smp_may_cut(V, k_rule, p_rule)) DL_TIMED("sample_hist", s, (sample_hist<T><<<blocks, SMP_THREADS, 0, s>>>(a)));
               DL_TIMED("sample_collect", s, (sample_collect<T><<<blocks, SMP_THREADS, 0, s>>>(a)));
               DL_TIMED("sample_draw", s, (sample_draw<T><<<B, SMP_DRAW_THREADS, 0, s>>>(a))));
    return dl_launch_status();
}
