// Embedding lookup with scaling, and the weight gradient by sorted tokens.
//
//   y[t] = scale W[token_t],      gW[v] = scale * sum over t with token_t = v of gy[t]
//
// A token outside [0, V) gives a row of zeros and adds nothing to the gradient; one that equals `padding` adds nothing either.
//
// The gradient of many tokens takes three launches (six where a long list is parted first) and no atomics on floats, so its bits do not
// depend on the schedule:
//   embed_sort   positions sorted by token, ascending within one.  Block b owns the tokens v with v mod blocks = b and reads
//                the whole token list (it stays in the L2): how many tokens belong to lower blocks is where its own begin.  Owning
//                every blocks-th token spreads the frequent ones, which lie together at the low ids of a vocabulary.
//   embed_sum    teams of threads walk pieces of 16 or 32 sorted positions - equal work however uneven the frequencies - and write
//                a token's sum where all of its positions lie in the piece, else a partial; the rest of the grid writes the rows of
//                tokens that do not occur.
//   embed_join   adds the partials of tokens that reach over pieces, in order.
// Up to EMB_FEW tokens take one launch (embed_few).
//
// Bound by memory but for the sort.  us at 65521 tokens, 131072 x 1024 bf16: lookup 32 (results stored past the caches; 52 before), sums and
// empty rows 78 (435 MB, 5.6 TB/s; 120 with 16 rows of 8 values in flight, which left two wavefronts a SIMD), sort 24 (every block
// reads 64 tokens per wavefront and step, 16 instructions each; 60 with a second read of the list), join 6 (84 by one team per
// token).  At 12544 tokens, 16384 x 784 fp32: 12, 17, 11, 5.
#include "dl_types.h"

#define EMB_THREADS 256
#define EMB_SORT_THREADS 1024
#define EMB_SORT_WAVES (EMB_SORT_THREADS / 64)
#define EMB_MAX_OWNED 512  // tokens that a block of the sort owns at most (a thread each; 32 KB of counts)
#define EMB_AHEAD 8         // groups of 64 tokens that a wavefront of the sort has in flight
#define EMB_FOUND 480       // tokens of its own that a wavefront remembers, as 23 bits of position and 9 bits of place (EMB_MAX_OWNED)
#define EMB_ROWS(E) ((E) == 8 ? 8 : 16)  // rows that a team of the sums has in flight (more registers leave too few wavefronts)
#define EMB_FEW 512         // tokens up to which the gradient takes one launch
#define EMB_LONG 81920      // tokens from which on they are parted by owner before they are sorted
#define EMB_CHUNKS 1024     // pieces of the list there, at most
#define EMB_JOIN_THREADS 512
#define EMB_JOIN_WAVES (EMB_JOIN_THREADS / 64)
#define EMB_JOIN_SPLIT 16  // partials from which on the block's wavefronts share them

// ---------------------------------------------------------------------------------- lookup
// A team of `lanes` threads per row (a power of two), R rows of a team in flight at once.
template <typename T, typename TOKEN, bool VEC, int R>
__global__ __launch_bounds__(EMB_THREADS) void embed_lookup(const TOKEN *__restrict__ tokens, const T *__restrict__ weight, long long ldw,
                                                             T *__restrict__ y, long long n, long long V, int D, float scale, int lane_bits) {
    constexpr int E = VEC ? 16 / sizeof(T) : 1;
    const int lane = threadIdx.x & ((1 << lane_bits) - 1);
    const long long teams = (long long)gridDim.x * (EMB_THREADS >> lane_bits);
    const long long team = (long long)blockIdx.x * (EMB_THREADS >> lane_bits) + (threadIdx.x >> lane_bits);
    const T *src[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const long long t = team + r * teams;
        const long long v = t < n ? (long long)tokens[t] : -1;
        src[r] = v >= 0 && v < V ? weight + v * ldw : nullptr;
    }
    for (int c = lane * E; c < D; c += E << lane_bits) {
        float f[R][E];
#pragma unroll
        for (int r = 0; r < R; ++r) {
#pragma unroll
            for (int e = 0; e < E; ++e) f[r][e] = 0.0f;
            if (src[r]) dl_load(src[r] + c, f[r]);
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const long long t = team + r * teams;
            if (t >= n) continue;
#pragma unroll
            for (int e = 0; e < E; ++e) f[r][e] *= scale;
            dl_store_past(y + t * D + c, f[r]);
        }
    }
}

// ---------------------------------------------------------------------------------- sort
// A token as 32 bits; ~0: not summed (V < 2^31).
template <typename TOKEN>
__device__ __forceinline__ unsigned emb_token(TOKEN t, unsigned V, unsigned padding) {
    const bool known = sizeof(TOKEN) == 4 ? (unsigned)t < V : (unsigned long long)t < (unsigned long long)V;
    return known && (unsigned)t != padding ? (unsigned)t : ~0u;
}
// EMB_AHEAD groups of 64 tokens from group g on, those before g1 and n; -1 past them
template <typename TOKEN>
__device__ __forceinline__ void emb_fetch(const TOKEN *__restrict__ tokens, int g, int g1, int n, TOKEN (&t)[EMB_AHEAD]) {
    const TOKEN *from = tokens + (long long)g * 64 + (threadIdx.x & 63);
    if (g + EMB_AHEAD <= g1 && (long long)(g + EMB_AHEAD) * 64 <= n) {
#pragma unroll
        for (int u = 0; u < EMB_AHEAD; ++u) t[u] = from[u * 64];
    } else {
#pragma unroll
        for (int u = 0; u < EMB_AHEAD; ++u) t[u] = g + u < g1 && (g + u) * 64 + (int)(threadIdx.x & 63) < n ? from[u * 64] : (TOKEN)-1;
    }
}

// Lanes of one slot (of `bits` bits) are ranked among themselves and go to next[slot] on; `next`, a wavefront's own in LDS, moves on.  Which
// lanes share a slot comes from a ballot per bit, so the cost does not go by the number of different slots.  (volatile: a
// wavefront's lanes see each other's stores, which are in order)
template <typename F>
__device__ __forceinline__ void emb_put(bool here, unsigned slot, int bits, volatile int *next, F store) {
    unsigned long long same = __ballot(here);
    if (same == 0) return;
    for (int k = 0; k < bits; ++k) {
        const bool bit = slot >> k & 1;
        const unsigned long long set = __ballot(bit);
        same &= bit ? set : ~set;
    }
    if (!here) return;
    const int lane = threadIdx.x & 63, first = next[slot];
    store(first + __popcll(same & ((1ull << lane) - 1)));
    if (lane == __builtin_ctzll(same)) next[slot] = first + __popcll(same);
}

template <typename TOKEN>
__global__ __launch_bounds__(EMB_SORT_THREADS) void embed_sort(const TOKEN *__restrict__ tokens, int n, unsigned V, unsigned padding,
                                                                int block_bits, int *__restrict__ order, int *__restrict__ token_of,
                                                                int *__restrict__ begin_of, int *__restrict__ count, int *__restrict__ total) {
    extern __shared__ int place[];  // [waves][owned]: counts, then where the wave's next position of a token goes
    __shared__ unsigned found[EMB_SORT_WAVES][EMB_FOUND];  // a wave's own tokens, in order
    __shared__ int below_of[EMB_SORT_WAVES], scan[EMB_SORT_WAVES];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const unsigned b = blockIdx.x, mask = (1u << block_bits) - 1;
    const int owned = (int)((V - b + mask) >> block_bits);  // tokens b, b + blocks, ...  (b <= mask: no wrap below -mask)
    for (int i = threadIdx.x; i < EMB_SORT_WAVES * owned; i += EMB_SORT_THREADS) place[i] = 0;
    __syncthreads();
    // a wave takes a run of whole groups of 64 positions, EMB_AHEAD of them in flight
    const int groups = (n + 63) >> 6, per_wave = (groups + EMB_SORT_WAVES - 1) / EMB_SORT_WAVES;
    const int g0 = min(wave * per_wave, groups), g1 = min(g0 + per_wave, groups);
    int below = 0, mine = 0;
    TOKEN t[EMB_AHEAD], ahead[EMB_AHEAD];
    emb_fetch(tokens, g0, g1, n, t);
    for (int g = g0; g < g1; g += EMB_AHEAD) {
        emb_fetch(tokens, g + EMB_AHEAD, g1, n, ahead);
#pragma unroll
        for (int u = 0; u < EMB_AHEAD; ++u) {
            const unsigned v = emb_token(t[u], V, padding), owner = v == ~0u ? v : v & mask;
            const bool here = owner == b;
            below += __popcll(__ballot(owner < b));
            const unsigned long long takes = __ballot(here);
            if (takes == 0) continue;
            if (here) {
                atomicAdd(&place[wave * owned + (v >> block_bits)], 1);
                const int at = mine + __popcll(takes & ((1ull << lane) - 1));
                if (at < EMB_FOUND) found[wave][at] = (unsigned)((g + u - g0) * 64 + lane) << 9 | v >> block_bits;
            }
            mine += __popcll(takes);
        }
#pragma unroll
        for (int u = 0; u < EMB_AHEAD; ++u) t[u] = ahead[u];
    }
    if (lane == 0) below_of[wave] = below;
    __syncthreads();
    // per token, where each wave's positions begin (a thread per token: owned <= EMB_MAX_OWNED)
    int tokens_here = 0;
    if ((int)threadIdx.x < owned)
        for (int w = 0; w < EMB_SORT_WAVES; ++w) {
            const int c = place[w * owned + threadIdx.x];
            place[w * owned + threadIdx.x] = tokens_here;
            tokens_here += c;
        }
    int before = tokens_here;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int up = __shfl_up(before, o);
        if (lane >= o) before += up;
    }
    if (lane == 63) scan[wave] = before;
    __syncthreads();
    int base = 0, all = 0;
    for (int w = 0; w < EMB_SORT_WAVES; ++w) {
        base += below_of[w];
        if (w < wave) before += scan[w];
        all += scan[w];
    }
    before += base - tokens_here;
    if ((int)threadIdx.x < owned) {
        for (int w = 0; w < EMB_SORT_WAVES; ++w) place[w * owned + threadIdx.x] += before;
        const unsigned v = b + (threadIdx.x << block_bits);
        count[v] = tokens_here;
        begin_of[v] = before;
    }
    if (b == mask && threadIdx.x == 0) *total = base + all;
    __syncthreads();
    // the positions themselves, in order
    const int bits = 32 - __clz(max(owned - 1, 0));
    const auto put = [&](bool here, int t, unsigned v) {
        emb_put(here, v >> block_bits, bits, place + wave * owned, [&](int at) { order[at] = t, token_of[at] = (int)v; });
    };
    if (mine <= EMB_FOUND && per_wave <= 1 << 17) {
        for (int i = 0; i < mine; i += 64) {
            const unsigned f = i + lane < mine ? found[wave][i + lane] : 0;
            put(i + lane < mine, g0 * 64 + (int)(f >> 9), (f & 511) << block_bits | b);
        }
    } else {  // a frequent token: the list was too short, the tokens are read again
        for (int g = g0; g < g1; g += EMB_AHEAD) {
            emb_fetch(tokens, g, g1, n, t);
#pragma unroll
            for (int u = 0; u < EMB_AHEAD; ++u) {
                const unsigned v = emb_token(t[u], V, padding);
                put(v != ~0u && (v & mask) == b, (g + u) * 64 + lane, v);
            }
        }
    }
}

// ---------------------------------------------------------------------------------- long lists
// From EMB_LONG tokens on every block reading all of them is what the time goes into; they are parted by owner first, in order:
//   embed_part_count   how many tokens of a chunk belong to each owner, [owner][chunk]
//   embed_part_scan    where each of those begins
//   embed_part         positions and tokens, an owner's together
//   embed_sort_part    an owner's, by token
// The gradient in us, every block reading all / parted, rows of 64 floats: 65536 tokens of 50000 41 / 48, 131072 146 / 56 (blocks of frequent
// tokens read the list twice), 262144 271 / 80; of 500000 80 / 70, 112 / 81, 304 / 109.
// (1 048 576 tokens of 50000, rows of 256 floats: the gradient 1.07 -> 0.51 ms, 0.31 of it the sums; the block of the most frequent token, 6 % of
// the list, is what embed_sort_part's 0.11 wait for.)

template <typename TOKEN>
__global__ __launch_bounds__(EMB_SORT_THREADS) void embed_part_count(const TOKEN *__restrict__ tokens, int n, unsigned V, unsigned padding,
                                                                      int block_bits, int chunk, int chunks, int *__restrict__ counts) {
    extern __shared__ int place[];  // [owners]
    const int owners = 1 << block_bits;
    for (int i = threadIdx.x; i < owners; i += EMB_SORT_THREADS) place[i] = 0;
    __syncthreads();
    const int begin = blockIdx.x * chunk, end = (int)min((long long)begin + chunk, (long long)n);
    for (int t = begin + threadIdx.x; t < end; t += EMB_SORT_THREADS) {
        const unsigned v = emb_token(tokens[t], V, padding);
        if (v != ~0u) atomicAdd(&place[v & (owners - 1)], 1);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < owners; i += EMB_SORT_THREADS) counts[(long long)i * chunks + blockIdx.x] = place[i];
}

// begins[owner][chunk]: where its tokens go, of all in that order; the total stands behind them.  A block per owner (chunks <= its threads)
// adds up the lower owners' counts for itself.
__global__ __launch_bounds__(EMB_SORT_THREADS) void embed_part_scan(const int *__restrict__ counts, int chunks, int *__restrict__ begins,
                                                                     int *__restrict__ total) {
    __shared__ int scan[EMB_SORT_WAVES], lower[EMB_SORT_WAVES];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, own = blockIdx.x * chunks;
    int below = 0;
#pragma unroll 8
    for (int i = threadIdx.x; i < own; i += EMB_SORT_THREADS) below += counts[i];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) below += __shfl_xor(below, o);
    const int mine = (int)threadIdx.x < chunks ? counts[own + threadIdx.x] : 0;
    int before = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int up = __shfl_up(before, o);
        if (lane >= o) before += up;
    }
    if (lane == 63) scan[wave] = before, lower[wave] = below;
    __syncthreads();
    for (int w = 0; w < EMB_SORT_WAVES; ++w) {
        before += lower[w];
        if (w < wave) before += scan[w];
    }
    if ((int)threadIdx.x < chunks) begins[own + threadIdx.x] = before - mine;
    if (blockIdx.x == gridDim.x - 1 && threadIdx.x == EMB_SORT_THREADS - 1) begins[own + chunks] = *total = before;
}

template <typename TOKEN>
__global__ __launch_bounds__(EMB_SORT_THREADS) void embed_part(const TOKEN *__restrict__ tokens, int n, unsigned V, unsigned padding,
                                                                int block_bits, int chunk, int chunks, const int *__restrict__ begins,
                                                                int *__restrict__ positions, unsigned *__restrict__ parted) {
    extern __shared__ int place[];  // [waves][owners]
    const int owners = 1 << block_bits, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    for (int i = threadIdx.x; i < EMB_SORT_WAVES * owners; i += EMB_SORT_THREADS) place[i] = 0;
    __syncthreads();
    const int begin = blockIdx.x * chunk, end = (int)min((long long)begin + chunk, (long long)n);
    const int per_wave = (chunk / 64 + EMB_SORT_WAVES - 1) / EMB_SORT_WAVES * 64;  // (chunk: whole groups of 64)
    const int t0 = min(begin + wave * per_wave, end), t1 = min(t0 + per_wave, end);
    for (int t = t0 + lane; t < t1; t += 64) {
        const unsigned v = emb_token(tokens[t], V, padding);
        if (v != ~0u) atomicAdd(&place[wave * owners + (v & (owners - 1))], 1);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < owners; i += EMB_SORT_THREADS) {
        int at = begins[(long long)i * chunks + blockIdx.x];
        for (int w = 0; w < EMB_SORT_WAVES; ++w) {
            const int c = place[w * owners + i];
            place[w * owners + i] = at;
            at += c;
        }
    }
    __syncthreads();
    for (int t = t0; t < t1; t += 64) {
        const unsigned v = t + lane < t1 ? emb_token(tokens[t + lane], V, padding) : ~0u;
        emb_put(v != ~0u, v & (owners - 1), block_bits, place + wave * owners, [&](int at) { positions[at] = t + lane, parted[at] = v; });
    }
}

__global__ __launch_bounds__(EMB_SORT_THREADS) void embed_sort_part(const int *__restrict__ positions, const unsigned *__restrict__ parted, unsigned V,
                                                                     int block_bits, int chunks, const int *__restrict__ begins,
                                                                     int *__restrict__ order, int *__restrict__ token_of,
                                                                     int *__restrict__ begin_of, int *__restrict__ count) {
    extern __shared__ int place[];  // [waves][owned]
    __shared__ int scan[EMB_SORT_WAVES];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const unsigned b = blockIdx.x, mask = (1u << block_bits) - 1;
    const int owned = (int)((V - b + mask) >> block_bits);
    for (int i = threadIdx.x; i < EMB_SORT_WAVES * owned; i += EMB_SORT_THREADS) place[i] = 0;
    __syncthreads();
    const int begin = begins[(long long)b * chunks], end = begins[(long long)(b + 1) * chunks];  // (the total stands behind the last)
    const int per_wave = ((end - begin + 63) / 64 + EMB_SORT_WAVES - 1) / EMB_SORT_WAVES * 64;
    const int i0 = min(begin + wave * per_wave, end), i1 = min(i0 + per_wave, end);
#pragma unroll 4
    for (int i = i0 + lane; i < i1; i += 64) atomicAdd(&place[wave * owned + (int)(parted[i] >> block_bits)], 1);
    __syncthreads();
    int here = 0;
    if ((int)threadIdx.x < owned)
        for (int w = 0; w < EMB_SORT_WAVES; ++w) here += place[w * owned + threadIdx.x];
    int before = here;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int up = __shfl_up(before, o);
        if (lane >= o) before += up;
    }
    if (lane == 63) scan[wave] = before;
    __syncthreads();
    for (int w = 0; w < wave; ++w) before += scan[w];
    before += begin - here;
    if ((int)threadIdx.x < owned) {
        const unsigned v = b + (threadIdx.x << block_bits);
        count[v] = here, begin_of[v] = before;
        for (int w = 0; w < EMB_SORT_WAVES; ++w) {
            const int c = place[w * owned + threadIdx.x];
            place[w * owned + threadIdx.x] = before;
            before += c;
        }
    }
    __syncthreads();
    const int bits = 32 - __clz(max(owned - 1, 0));
    for (int i = i0; i < i1; i += 4 * 64) {
        unsigned v[4];
        int t[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int at = i + u * 64 + lane;
            v[u] = at < i1 ? parted[at] : 0, t[u] = at < i1 ? positions[at] : 0;
        }
#pragma unroll
        for (int u = 0; u < 4; ++u)
            emb_put(i + u * 64 + lane < i1, v[u] >> block_bits, bits, place + wave * owned, [&](int at) { order[at] = t[u], token_of[at] = (int)v[u]; });
    }
}

// ---------------------------------------------------------------------------------- sums
struct EmbArgs {
    const int *order, *token_of, *begin_of, *count, *total;
    float *part;  // [pieces][2][D]: of the token that began in an earlier piece, of the one that goes on into the next
    long long V;
    int D, lane_bits, pieces, piece;  // sorted positions are walked in `pieces` pieces of `piece`
    unsigned sum_blocks;
    float scale;
};

template <typename T, bool VEC>
__global__ __launch_bounds__(EMB_THREADS) void embed_sum(const T *__restrict__ gy, T *__restrict__ gw, EmbArgs a) {
    constexpr int E = VEC ? 16 / sizeof(T) : 1;
    const int lanes = 1 << a.lane_bits, lane = threadIdx.x & (lanes - 1), teams_here = EMB_THREADS >> a.lane_bits;
    const int team_here = threadIdx.x >> a.lane_bits;
    if (blockIdx.x >= a.sum_blocks) {  // rows of tokens that do not occur
        const float zero[E] = {};
        const long long teams = (long long)(gridDim.x - a.sum_blocks) * teams_here;
        for (long long v0 = (long long)(blockIdx.x - a.sum_blocks) * teams_here + team_here; v0 < a.V; v0 += 4 * teams) {
            int n[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) n[u] = v0 + u * teams < a.V ? a.count[v0 + u * teams] : 1;
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (n[u] == 0)
                    for (int c = lane * E; c < a.D; c += E << a.lane_bits) dl_store_past(gw + (v0 + u * teams) * a.D + c, zero);
        }
        return;
    }
    constexpr int ROWS = EMB_ROWS(E);
    const int total = *a.total, piece = blockIdx.x * teams_here + team_here;
    const int i0 = piece * a.piece, i1 = min(i0 + a.piece, total);
    if (piece >= a.pieces || i0 >= total) return;
    const int before = i0 > 0 ? a.token_of[i0 - 1] : -1, after = i1 < total ? a.token_of[i1] : -1;
    for (int c = lane * E; c < a.D; c += E << a.lane_bits) {
        float acc[E] = {};
        bool first = true;  // of the piece's tokens
        for (int j0 = i0; j0 < i1; j0 += ROWS) {
            float f[ROWS][E];
#pragma unroll
            for (int j = 0; j < ROWS; ++j)
                if (j0 + j < i1) dl_load(gy + (long long)a.order[j0 + j] * a.D + c, f[j]);
#pragma unroll
            for (int j = 0; j < ROWS; ++j) {
                if (j0 + j >= i1) break;
                const bool last = j0 + j + 1 == i1;
                const int v = a.token_of[j0 + j], next = last ? after : a.token_of[j0 + j + 1];
#pragma unroll
                for (int e = 0; e < E; ++e) acc[e] += f[j][e];
                if (next == v && !last) continue;
                if (first && before == v) dl_store(a.part + ((long long)piece * 2) * a.D + c, acc);
                else if (last && next == v) dl_store(a.part + ((long long)piece * 2 + 1) * a.D + c, acc);
                else {
#pragma unroll
                    for (int e = 0; e < E; ++e) acc[e] *= a.scale;
                    dl_store_past(gw + (long long)v * a.D + c, acc);
                }
                first = false;
#pragma unroll
                for (int e = 0; e < E; ++e) acc[e] = 0.0f;
            }
        }
    }
}

// Tokens that reach over pieces.  A wavefront takes a piece, whose last token may go on, and 64 vectors of columns; the partials of a frequent
// token (thousands) are split over the block's wavefronts, whose sums are added in order.
template <typename T, bool VEC>
__global__ __launch_bounds__(EMB_JOIN_THREADS) void embed_join(T *__restrict__ gw, EmbArgs a, int columns) {
    constexpr int E = VEC ? 4 : 1;
    __shared__ DlVec<float, E> sums[EMB_JOIN_WAVES][64];
    __shared__ int parts_of[EMB_JOIN_WAVES];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, total = *a.total;
    const int c = (blockIdx.x % columns * 64 + lane) * E;
    const long long piece0 = (long long)(blockIdx.x / columns) * EMB_JOIN_WAVES;
    // the pieces behind `piece` that begin with sums of its last token (0: it ends here, began earlier, or there is none)
    const auto joins = [&](long long piece, int &v) {
        const long long i0 = piece * a.piece, i1 = i0 + a.piece;
        if (i1 >= total) return 0;
        v = a.token_of[i1 - 1];
        const int begin = a.begin_of[v], end = begin + a.count[v];
        return end <= i1 || begin < i0 ? 0 : (end - 1) / a.piece - (int)piece;
    };
    // sum of partials [p0, p1) behind `piece`, on top of acc
    const auto add = [&](long long piece, int p0, int p1, float (&acc)[E]) {
        const float *rest = a.part + (piece + 1) * 2 * a.D + c;
#pragma unroll 8
        for (int p = p0; p < p1; ++p) {
            float f[E];
            dl_load(rest + (long long)p * 2 * a.D, f);
#pragma unroll
            for (int e = 0; e < E; ++e) acc[e] += f[e];
        }
    };
    const auto write = [&](int v, float (&acc)[E]) {
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] *= a.scale;
        dl_store(gw + (long long)v * a.D + c, acc);
    };
    int v = 0;
    const long long own = piece0 + wave;
    const int parts = own < a.pieces ? joins(own, v) : 0;
    if (lane == 0) parts_of[wave] = parts;
    if (parts > 0 && parts < EMB_JOIN_SPLIT && c < a.D) {
        float acc[E];
        dl_load(a.part + (own * 2 + 1) * a.D + c, acc);
        add(own, 0, parts, acc);
        write(v, acc);
    }
    __syncthreads();
    for (int w = 0; w < EMB_JOIN_WAVES; ++w) {
        const int n = parts_of[w];
        if (n < EMB_JOIN_SPLIT) continue;
        const int per = (n + EMB_JOIN_WAVES - 1) / EMB_JOIN_WAVES, p0 = min(wave * per, n);
        float acc[E] = {};
        if (c < a.D) {
            if (wave == 0) dl_load(a.part + ((piece0 + w) * 2 + 1) * a.D + c, acc);
            add(piece0 + w, p0, min(p0 + per, n), acc);
        }
        dl_store(&sums[wave][lane].v[0], acc);
        __syncthreads();
        if (wave == w && c < a.D) {  // (v is this wavefront's)
#pragma unroll
            for (int e = 0; e < E; ++e) acc[e] = sums[0][lane].v[e];
#pragma unroll
            for (int k = 1; k < EMB_JOIN_WAVES; ++k)
#pragma unroll
                for (int e = 0; e < E; ++e) acc[e] += sums[k][lane].v[e];
            write(v, acc);
        }
        __syncthreads();
    }
}

// ---------------------------------------------------------------------------------- few tokens
// Up to EMB_FEW tokens the whole gradient takes one launch: a block owns every gridDim.x-th token of the vocabulary, picks their
// positions out of the list - in order, a wavefront's turn after the other - and writes their rows, most of them zeros.
template <typename T, typename TOKEN, bool VEC>
__global__ __launch_bounds__(EMB_THREADS) void embed_few(const TOKEN *__restrict__ tokens, const T *__restrict__ gy, T *__restrict__ gw, int n,
                                                          unsigned V, unsigned padding, int D, int lane_bits, float scale) {
    constexpr int E = VEC ? 16 / sizeof(T) : 1, WAVES = EMB_THREADS / 64, TURNS = EMB_FEW / EMB_THREADS;
    __shared__ unsigned token_of[EMB_FEW];
    __shared__ int position[EMB_FEW], found_in[TURNS][WAVES];
    const int wave = threadIdx.x >> 6, lane64 = threadIdx.x & 63;
    unsigned mine[TURNS];
    unsigned long long takes[TURNS];
#pragma unroll
    for (int u = 0; u < TURNS; ++u) {
        const int t = u * EMB_THREADS + threadIdx.x;
        mine[u] = t < n ? emb_token(tokens[t], V, padding) : ~0u;
        takes[u] = __ballot(mine[u] != ~0u && mine[u] % gridDim.x == blockIdx.x);
        if (lane64 == 0) found_in[u][wave] = __popcll(takes[u]);
    }
    __syncthreads();
    int m = 0;
#pragma unroll
    for (int u = 0; u < TURNS; ++u)
        for (int w = 0; w < WAVES; ++w) {
            if (w == wave && (takes[u] >> lane64 & 1)) {
                const int at = m + __popcll(takes[u] & ((1ull << lane64) - 1));
                token_of[at] = mine[u], position[at] = u * EMB_THREADS + threadIdx.x;
            }
            m += found_in[u][w];
        }
    __syncthreads();
    const int lane = threadIdx.x & ((1 << lane_bits) - 1), teams = EMB_THREADS >> lane_bits;
    for (unsigned long long v = blockIdx.x + (unsigned long long)(threadIdx.x >> lane_bits) * gridDim.x; v < V; v += (unsigned long long)teams * gridDim.x)
        for (int c = lane * E; c < D; c += E << lane_bits) {
            float acc[E] = {};
#pragma unroll 4
            for (int j = 0; j < m; ++j)
                if (token_of[j] == (unsigned)v) {
                    float f[E];
                    dl_load(gy + (long long)position[j] * D + c, f);
#pragma unroll
                    for (int e = 0; e < E; ++e) acc[e] += f[e];
                }
#pragma unroll
            for (int e = 0; e < E; ++e) acc[e] *= scale;
            dl_store_past(gw + (long long)v * D + c, acc);
        }
}

// ---------------------------------------------------------------------------------- host
// (positions and columns are counted in 32 bits, some of them by a block's step past the last)
static bool emb_sizes_ok(long long n, long long V, int D) {
    return n >= 0 && n < (1LL << 31) - 65536 && V > 0 && V < (1LL << 31) && D > 0 && D < (1LL << 31) - 65536;
}
static int emb_lane_bits(int D, int E) {  // a team of up to a block's threads, as many as a row has vectors
    int bits = 0;
    while (bits < 8 && ((long long)E << bits) < D) ++bits;
    return bits;
}
static int emb_block_bits(long long V) {  // blocks of the sort: one per CU, more where a block would own too many tokens
    int bits = 0;
    while (bits < 8 && (1LL << bits) < V) ++bits;
    while (((V + (1LL << bits) - 1) >> bits) > EMB_MAX_OWNED) ++bits;
    return bits;
}

extern "C" int dl_embedding_fwd(const void *tokens, int token_bits, const void *weight, long long ldw, void *y, int type, long long n,
                                long long V, int D, float scale, void *stream) {
    if (!dl_type_known(type) || (token_bits != 32 && token_bits != 64)) return DL_ERR_UNSUPPORTED;
    if (!emb_sizes_ok(n, V, D) || ldw < D) return DL_ERR_SHAPE;
    if (n == 0) return DL_OK;
    if (!tokens || !weight || !y) return DL_ERR_NULL;
    hipStream_t s = (hipStream_t)stream;
    const int E = 16 / dl_type_bytes(type);
    const bool vec = dl_aligned16(weight) && dl_aligned16(y) && D % E == 0 && ldw % E == 0;
    const int bits = emb_lane_bits(D, vec ? E : 1);
    const long long per_block = EMB_THREADS >> bits;
    const bool many = n >= 4 * 2048 * per_block;  // enough rows for every team to take four
    const long long blocks = (n + per_block * (many ? 4 : 1) - 1) / (per_block * (many ? 4 : 1));
    if (!dl_grid_ok(blocks, EMB_THREADS)) {  // (tens of millions of odd rows)
        const long long half = n / 2;
        const int rc = dl_embedding_fwd(tokens, token_bits, weight, ldw, y, type, half, V, D, scale, stream);
        return rc != DL_OK ? rc : dl_embedding_fwd((const char *)tokens + half * (token_bits / 8), token_bits, weight, ldw,
                                                   (char *)y + half * D * dl_type_bytes(type), type, n - half, V, D, scale, stream);
    }
#define LOOKUP(TOKEN, VEC, R) \
    embed_lookup<T, TOKEN, VEC, R><<<(int)blocks, EMB_THREADS, 0, s>>>((const TOKEN *)tokens, (const T *)weight, ldw, (T *)y, n, V, D, scale, bits)
#define LOOKUP_R(TOKEN, VEC) if (many) LOOKUP(TOKEN, VEC, 4); else LOOKUP(TOKEN, VEC, 1)
    dl_prof_begin("embed_lookup", s);
    DL_BY_TYPE(type, T,
               if (token_bits == 32) { if (vec) { LOOKUP_R(int, true); } else { LOOKUP_R(int, false); } }
               else { if (vec) { LOOKUP_R(long long, true); } else { LOOKUP_R(long long, false); } });
    dl_prof_end(s);
#undef LOOKUP_R
#undef LOOKUP
    return dl_launch_status();
}

// Sorted positions per piece: a piece ends inside a token's run twice, for two partials to write and to read again, so longer ones move
// less; but there have to be enough teams.  The gradient in us with 16 / 32 positions, by tokens x features in millions: 4.2 (16384 x 256)
// 24.4 / 29.0, 8.4 (65521 x 128) 47.7 / 53.6, 9.8 (12544 x 784) 32.0 / 37.1, 16.8 (32768 x 512) 42.7 / 45.8, 19.3 (24576 x 784) 49.0 / 48.7,
// 25.2 (65521 x 384) 63.9 / 63.0, 25.7 (32768 x 784) 57.8 / 56.6, 33.6 (131072 x 256) 77.3 / 74.5, 67 (65521 x 1024 bf16) 109.0 / 105.6.
static int emb_piece(long long n, int D) { return n * D >= (1LL << 24) + (1LL << 23) ? 32 : 16; }
static long long emb_pieces(long long n, int D) { return (n + emb_piece(n, D) - 1) / emb_piece(n, D); }

// Parting a long list: chunks of whole groups of 64 tokens, and the owners that their counts' LDS has room for: up to 1024 of 512 rows.  A
// larger vocabulary's blocks all read the whole list, so time goes by tokens times rows (rows of 16 floats, us, 524288 rows / 524289 /
// 4194304: 131072 tokens 66 / 154 / 552, 1048576 tokens 226 / 1132 / 3837).
static int emb_chunk(long long n) {
    const long long chunk = (n + EMB_CHUNKS - 1) / EMB_CHUNKS;
    return (int)((chunk > 4096 ? chunk + 63 : 4096) / 64 * 64);
}
static bool emb_long(long long n, long long V) { return n >= EMB_LONG && emb_block_bits(V) <= 10; }  // (64 KB of LDS)

extern "C" size_t dl_embedding_bwd_workspace_bytes(long long n, long long V, int D) {
    if (!emb_sizes_ok(n, V, D) || n <= EMB_FEW) return 0;
    return 256 + 2 * dl_align256((size_t)n * sizeof(int)) + 2 * dl_align256((size_t)V * sizeof(int)) +
           dl_align256((size_t)emb_pieces(n, D) * 2 * D * sizeof(float)) +
           (emb_long(n, V) ? 2 * dl_align256((size_t)n * sizeof(int)) +
                                 2 * dl_align256((((size_t)dl_ceil_div(n, emb_chunk(n)) << emb_block_bits(V)) + 1) * sizeof(int)) : 0);
}

extern "C" int dl_embedding_bwd(const void *tokens, int token_bits, const void *gy, void *gw, int type, long long n, long long V, int D,
                                float scale, long long padding, void *ws, size_t ws_bytes, void *stream) {
    if (!dl_type_known(type) || (token_bits != 32 && token_bits != 64)) return DL_ERR_UNSUPPORTED;
    if (!emb_sizes_ok(n, V, D)) return DL_ERR_SHAPE;
    const size_t need = dl_embedding_bwd_workspace_bytes(n, V, D);
    if (!gw || (need && !ws) || (n > 0 && (!tokens || !gy))) return DL_ERR_NULL;
    if (ws_bytes < need) return DL_ERR_WORKSPACE;
    hipStream_t s = (hipStream_t)stream;
    const int E = 16 / dl_type_bytes(type);
    const bool vec = dl_aligned16(gy) && dl_aligned16(gw) && D % E == 0;
    const unsigned skip = padding >= 0 && padding < V ? (unsigned)padding : ~0u;
    if (!need) {
        const int bits = emb_lane_bits(D, vec ? E : 1);
        const long long rows = (V + (EMB_THREADS >> bits) - 1) / (EMB_THREADS >> bits);
        const int blocks = (int)(rows < 2048 ? rows : 2048);
#define FEW(TOKEN, VEC) embed_few<T, TOKEN, VEC><<<blocks, EMB_THREADS, 0, s>>>((const TOKEN *)tokens, (const T *)gy, (T *)gw, (int)n, (unsigned)V, skip, D, bits, scale)
        dl_prof_begin("embed_few", s);
        DL_BY_TYPE(type, T, if (token_bits == 32) { if (vec) FEW(int, true); else FEW(int, false); }
                   else { if (vec) FEW(long long, true); else FEW(long long, false); });
        dl_prof_end(s);
#undef FEW
        return dl_launch_status();
    }
    int *total = (int *)ws, *order = (int *)((char *)ws + 256);
    int *token_of = (int *)((char *)order + dl_align256((size_t)n * sizeof(int)));
    int *count = (int *)((char *)token_of + dl_align256((size_t)n * sizeof(int)));
    int *begin_of = (int *)((char *)count + dl_align256((size_t)V * sizeof(int)));
    EmbArgs a = {};
    a.order = order, a.token_of = token_of, a.begin_of = begin_of, a.count = count, a.total = total;
    a.part = (float *)((char *)begin_of + dl_align256((size_t)V * sizeof(int)));
    a.V = V, a.D = D, a.scale = scale;
    a.lane_bits = emb_lane_bits(D, vec ? E : 1);
    a.piece = emb_piece(n, D), a.pieces = (int)emb_pieces(n, D);
    const int teams = EMB_THREADS >> a.lane_bits;
    a.sum_blocks = (unsigned)((a.pieces + teams - 1) / teams);
    const int bits = emb_block_bits(V);
    const size_t lds = (size_t)EMB_SORT_WAVES * (size_t)((V + (1LL << bits) - 1) >> bits) * sizeof(int);
    // every launch of the call, before the first one: those behind a launch that fails would take what it left unwritten for indices
    if (!dl_grid_ok(1LL << bits, EMB_SORT_THREADS) ||
        !dl_grid_ok((long long)dl_ceil_div(a.pieces, EMB_JOIN_WAVES) * dl_ceil_div(D, vec ? 256 : 64), EMB_JOIN_THREADS) ||
        !dl_grid_ok((long long)a.sum_blocks + 2048, EMB_THREADS))
        return DL_ERR_UNSUPPORTED;
#define SORT(TOKEN) \
    embed_sort<TOKEN><<<1 << bits, EMB_SORT_THREADS, lds, s>>>((const TOKEN *)tokens, (int)n, (unsigned)V, skip, bits, order, token_of, begin_of, count, total)
    if (emb_long(n, V)) {
        const int chunk = emb_chunk(n), chunks = dl_ceil_div(n, chunk), owners = 1 << bits;
        int *positions = (int *)((char *)a.part + dl_align256((size_t)a.pieces * 2 * D * sizeof(float)));
        unsigned *parted = (unsigned *)((char *)positions + dl_align256((size_t)n * sizeof(int)));
        int *begins = (int *)((char *)parted + dl_align256((size_t)n * sizeof(int)));
        int *counts = (int *)((char *)begins + dl_align256(((size_t)owners * chunks + 1) * sizeof(int)));
#define PART(TOKEN)                                                                                                                    \
    DL_TIMED("embed_part_count", s, (embed_part_count<TOKEN><<<chunks, EMB_SORT_THREADS, owners * sizeof(int), s>>>(                   \
        (const TOKEN *)tokens, (int)n, (unsigned)V, skip, bits, chunk, chunks, counts)));                                              \
    DL_TIMED("embed_part_scan", s, (embed_part_scan<<<owners, EMB_SORT_THREADS, 0, s>>>(counts, chunks, begins, total)));              \
    DL_TIMED("embed_part", s, (embed_part<TOKEN><<<chunks, EMB_SORT_THREADS, EMB_SORT_WAVES * owners * sizeof(int), s>>>(              \
        (const TOKEN *)tokens, (int)n, (unsigned)V, skip, bits, chunk, chunks, begins, positions, parted)))
        if (token_bits == 32) { PART(int); }
        else { PART(long long); }
#undef PART
        DL_TIMED("embed_sort_part", s, (embed_sort_part<<<owners, EMB_SORT_THREADS, lds, s>>>(positions, parted, (unsigned)V, bits, chunks, begins,
                                                                                             order, token_of, begin_of, count)));
    } else {
        dl_prof_begin("embed_sort", s);
        if (token_bits == 32) SORT(int);
        else SORT(long long);
        dl_prof_end(s);
    }
#undef SORT
    const long long zero_teams = (V + teams - 1) / teams;
    const unsigned zero_blocks = (unsigned)(zero_teams < 2048 ? zero_teams : 2048);
#define SUMS(VEC)                                                                                                                    \
    DL_TIMED("embed_sum", s, (embed_sum<T, VEC><<<a.sum_blocks + zero_blocks, EMB_THREADS, 0, s>>>((const T *)gy, (T *)gw, a)));     \
    if (a.pieces > 1) {                                                                                                              \
        const int columns = dl_ceil_div(D, VEC ? 256 : 64);                                                                          \
        const int joins = dl_ceil_div(a.pieces, EMB_JOIN_WAVES) * columns;                                                           \
        DL_TIMED("embed_join", s, (embed_join<T, VEC><<<joins, EMB_JOIN_THREADS, 0, s>>>((T *)gw, a, columns)));                \
    }
    DL_BY_TYPE(type, T, if (vec) { SUMS(true); } else { SUMS(false); });
#undef SUMS
    return dl_launch_status();
}
