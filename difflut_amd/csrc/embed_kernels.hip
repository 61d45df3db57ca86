// Embedding lookup with scaling, and the weight gradient by sorted tokens.
//
//   y[t] = scale W[token_t],      gW[v] = scale * sum over t with token_t = v of gy[t]
//
// A token outside [0, V) gives a row of zeros and adds nothing to the gradient; one that equals `padding` adds nothing either.
//
// The gradient takes three launches and no atomics on floats, so its bits do not depend on the schedule:
//   embed_sort   positions sorted by token, ascending within one.  Block b owns the tokens v with v mod blocks = b and reads
//                the whole token list (it stays in the L2): how many tokens belong to lower blocks is where its own begin.  Owning
//                every blocks-th token spreads the frequent ones, which lie together at the low ids of a vocabulary.
//   embed_sum    teams of threads walk pieces of EMB_PIECE sorted positions - equal work however uneven the frequencies - and write
//                a token's sum where all of its positions lie in the piece, else a partial; the rest of the grid writes the rows of
//                tokens that do not occur.
//   embed_join   adds the partials of tokens that reach over pieces, in order.
#include "dl_types.h"

#define EMB_THREADS 256
#define EMB_SORT_THREADS 1024
#define EMB_SORT_WAVES (EMB_SORT_THREADS / 64)
#define EMB_MAX_OWNED 512  // tokens that a block of the sort owns at most (a thread each; 32 KB of counts)
#define EMB_PIECE 16

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
            dl_store(y + t * D + c, f[r]);
        }
    }
}

// ---------------------------------------------------------------------------------- sort
// The block and the place in it of a token; -1: not summed.
template <typename TOKEN>
__device__ __forceinline__ int emb_token(const TOKEN *__restrict__ tokens, int t, int n, long long V, long long padding) {
    if (t >= n) return -1;
    const long long v = (long long)tokens[t];
    return v >= 0 && v < V && v != padding ? (int)v : -1;
}

template <typename TOKEN>
__global__ __launch_bounds__(EMB_SORT_THREADS) void embed_sort(const TOKEN *__restrict__ tokens, int n, long long V, long long padding,
                                                                int block_bits, int *__restrict__ order, int *__restrict__ token_of,
                                                                int *__restrict__ count, int *__restrict__ total) {
    extern __shared__ int place[];  // [waves][owned]: counts, then where the wave's next position of a token goes
    __shared__ int below_of[EMB_SORT_WAVES], scan[EMB_SORT_WAVES];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, b = blockIdx.x, mask = (1 << block_bits) - 1;
    const int owned = (int)((V - b + mask) >> block_bits);  // tokens b, b + blocks, ...
    for (int i = threadIdx.x; i < EMB_SORT_WAVES * owned; i += EMB_SORT_THREADS) place[i] = 0;
    __syncthreads();
    // a wave takes a run of whole groups of 64 positions
    const int groups = (n + 63) >> 6, per_wave = (groups + EMB_SORT_WAVES - 1) / EMB_SORT_WAVES;
    const int g0 = min(wave * per_wave, groups), g1 = min(g0 + per_wave, groups);
    int below = 0, mine = 0;
#pragma unroll 4
    for (int g = g0; g < g1; ++g) {
        const int v = emb_token(tokens, g * 64 + lane, n, V, padding);
        if (v < 0) continue;
        const int owner = v & mask;
        below += owner < b;
        if (owner == b) {
            atomicAdd(&place[wave * owned + (v >> block_bits)], 1);
            ++mine;
        }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        below += __shfl_xor(below, o);
        mine += __shfl_xor(mine, o);
    }
    if (lane == 0) below_of[wave] = below;
    __syncthreads();
    // per token, where each wave's positions begin (a thread per token: owned <= EMB_MAX_OWNED)
    int tokens_here = 0;
    if ((int)threadIdx.x < owned) {
        for (int w = 0; w < EMB_SORT_WAVES; ++w) {
            const int c = place[w * owned + threadIdx.x];
            place[w * owned + threadIdx.x] = tokens_here;
            tokens_here += c;
        }
        count[b + ((long long)threadIdx.x << block_bits)] = tokens_here;
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
    if ((int)threadIdx.x < owned)
        for (int w = 0; w < EMB_SORT_WAVES; ++w) place[w * owned + threadIdx.x] += before;
    if (b == mask && threadIdx.x == 0) *total = base + all;
    __syncthreads();
    if (mine == 0) return;
    // the positions themselves, in order: lanes of one token are ranked among themselves (volatile: a wavefront's lanes see each other's
    // stores, which are in order)
    volatile int *next = place;
    for (int g = g0; g < g1; ++g) {
        const int t = g * 64 + lane, v = emb_token(tokens, t, n, V, padding);
        const bool here = v >= 0 && (v & mask) == b;
        const int slot = here ? wave * owned + (v >> block_bits) : -1;
        unsigned long long left = __ballot(here);
        while (left) {
            const int leader = __builtin_ctzll(left), its = __builtin_amdgcn_readlane(slot, leader);
            const unsigned long long same = __ballot(slot == its);
            const int first = next[its];
            if (slot == its) {
                const int at = first + __popcll(same & ((1ull << lane) - 1));
                order[at] = t;
                token_of[at] = v;
            }
            if (lane == leader) next[its] = first + __popcll(same);
            left &= ~same;
        }
    }
}

// ---------------------------------------------------------------------------------- sums
struct EmbArgs {
    const int *order, *token_of, *count, *total;
    float *part;  // [pieces][2][D]: of the token that began in an earlier piece, of the one that goes on into the next
    long long V, ldg;
    int D, lane_bits, pieces;
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
        for (long long v = (long long)(blockIdx.x - a.sum_blocks) * teams_here + team_here; v < a.V; v += teams)
            if (a.count[v] == 0)
                for (int c = lane * E; c < a.D; c += E << a.lane_bits) dl_store(gw + v * a.D + c, zero);
        return;
    }
    const int total = *a.total, piece = blockIdx.x * teams_here + team_here;
    const int i0 = piece * EMB_PIECE, i1 = min(i0 + EMB_PIECE, total);
    if (piece >= a.pieces || i0 >= total) return;
    const int before = i0 > 0 ? a.token_of[i0 - 1] : -1, after = i1 < total ? a.token_of[i1] : -1;
    for (int c = lane * E; c < a.D; c += E << a.lane_bits) {
        float f[EMB_PIECE][E], acc[E] = {};
#pragma unroll
        for (int j = 0; j < EMB_PIECE; ++j)
            if (i0 + j < i1) dl_load(gy + (long long)a.order[i0 + j] * a.D + c, f[j]);
        bool first = true;  // of the piece's tokens
#pragma unroll
        for (int j = 0; j < EMB_PIECE; ++j) {
            if (i0 + j >= i1) break;
            const int v = a.token_of[i0 + j], next = i0 + j + 1 < i1 ? a.token_of[i0 + j + 1] : after;
#pragma unroll
            for (int e = 0; e < E; ++e) acc[e] += f[j][e];
            const bool last = i0 + j + 1 == i1;
            if (next == v && !last) continue;
            if (first && before == v) dl_store(a.part + ((long long)piece * 2) * a.D + c, acc);
            else if (last && next == v) dl_store(a.part + ((long long)piece * 2 + 1) * a.D + c, acc);
            else {
#pragma unroll
                for (int e = 0; e < E; ++e) acc[e] *= a.scale;
                dl_store(gw + (long long)v * a.D + c, acc);
            }
            first = false;
#pragma unroll
            for (int e = 0; e < E; ++e) acc[e] = 0.0f;
        }
    }
}

template <typename T, bool VEC>
__global__ __launch_bounds__(EMB_THREADS) void embed_join(T *__restrict__ gw, EmbArgs a) {
    constexpr int E = VEC ? 16 / sizeof(T) : 1;
    const int lanes = 1 << a.lane_bits, lane = threadIdx.x & (lanes - 1), teams_here = EMB_THREADS >> a.lane_bits;
    const int total = *a.total, piece = blockIdx.x * teams_here + (threadIdx.x >> a.lane_bits);
    const long long i0 = (long long)piece * EMB_PIECE, i1 = i0 + EMB_PIECE;
    if (i1 >= total) return;  // nothing goes on behind the last piece
    const int v = a.token_of[i1 - 1];
    if (a.token_of[i1] != v || (a.token_of[i0] == v && i0 > 0 && a.token_of[i0 - 1] == v)) return;  // ends here, or began earlier
    // the last piece that holds v
    int last = piece + 1;
    while ((long long)(last + 1) * EMB_PIECE < total && a.token_of[(long long)(last + 1) * EMB_PIECE] == v) ++last;
    for (int c = lane * E; c < a.D; c += E << a.lane_bits) {
        float acc[E];
        dl_load(a.part + ((long long)piece * 2 + 1) * a.D + c, acc);
#pragma unroll 8
        for (int p = piece + 1; p <= last; ++p) {
            float f[E];
            dl_load(a.part + (long long)p * 2 * a.D + c, f);
#pragma unroll
            for (int e = 0; e < E; ++e) acc[e] += f[e];
        }
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] *= a.scale;
        dl_store(gw + (long long)v * a.D + c, acc);
    }
}

// ---------------------------------------------------------------------------------- host
static bool emb_sizes_ok(long long n, long long V, int D) { return n >= 0 && n < (1LL << 31) - 64 && V > 0 && V < (1LL << 31) && D > 0; }
static int emb_lane_bits(int D, int E) {  // a team of up to a block's threads, as many as a row has vectors
    int bits = 0;
    while (bits < 8 && ((long long)E << bits) < D) ++bits;
    return bits;
}
static int emb_block_bits(long long V) {  // blocks of the sort: 512 of them, more where a block would own too many tokens
    int bits = 0;
    while (bits < 9 && (1LL << bits) < V) ++bits;
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

static long long emb_pieces(long long n) { return (n + EMB_PIECE - 1) / EMB_PIECE; }

extern "C" size_t dl_embedding_bwd_workspace_bytes(long long n, long long V, int D) {
    if (!emb_sizes_ok(n, V, D)) return 0;
    return 256 + 2 * dl_align256((size_t)n * sizeof(int)) + dl_align256((size_t)V * sizeof(int)) +
           dl_align256((size_t)emb_pieces(n) * 2 * D * sizeof(float));
}

extern "C" int dl_embedding_bwd(const void *tokens, int token_bits, const void *gy, void *gw, int type, long long n, long long V, int D,
                                float scale, long long padding, void *ws, size_t ws_bytes, void *stream) {
    if (!dl_type_known(type) || (token_bits != 32 && token_bits != 64)) return DL_ERR_UNSUPPORTED;
    if (!emb_sizes_ok(n, V, D)) return DL_ERR_SHAPE;
    if (!gw || !ws || (n > 0 && (!tokens || !gy))) return DL_ERR_NULL;
    if (ws_bytes < dl_embedding_bwd_workspace_bytes(n, V, D)) return DL_ERR_WORKSPACE;
    hipStream_t s = (hipStream_t)stream;
    const int E = 16 / dl_type_bytes(type);
    const bool vec = dl_aligned16(gy) && dl_aligned16(gw) && D % E == 0;
    int *total = (int *)ws, *order = (int *)((char *)ws + 256);
    int *token_of = (int *)((char *)order + dl_align256((size_t)n * sizeof(int)));
    int *count = (int *)((char *)token_of + dl_align256((size_t)n * sizeof(int)));
    EmbArgs a = {};
    a.order = order, a.token_of = token_of, a.count = count, a.total = total;
    a.part = (float *)((char *)count + dl_align256((size_t)V * sizeof(int)));
    a.V = V, a.D = D, a.scale = scale;
    a.lane_bits = emb_lane_bits(D, vec ? E : 1);
    a.pieces = (int)emb_pieces(n);
    const int teams = EMB_THREADS >> a.lane_bits;
    a.sum_blocks = (unsigned)((a.pieces + teams - 1) / teams);
    const int bits = emb_block_bits(V);
    const size_t lds = (size_t)EMB_SORT_WAVES * (size_t)((V + (1LL << bits) - 1) >> bits) * sizeof(int);
    dl_prof_begin("embed_sort", s);
    if (token_bits == 32) embed_sort<int><<<1 << bits, EMB_SORT_THREADS, lds, s>>>((const int *)tokens, (int)n, V, padding, bits, order, token_of, count, total);
    else embed_sort<long long><<<1 << bits, EMB_SORT_THREADS, lds, s>>>((const long long *)tokens, (int)n, V, padding, bits, order, token_of, count, total);
    dl_prof_end(s);
    const long long zero_teams = (V + teams - 1) / teams;
    const unsigned zero_blocks = (unsigned)(zero_teams < 4096 ? zero_teams : 4096);
#define SUMS(VEC)                                                                                                                    \
    DL_TIMED("embed_sum", s, (embed_sum<T, VEC><<<a.sum_blocks + zero_blocks, EMB_THREADS, 0, s>>>((const T *)gy, (T *)gw, a)));     \
    if (a.pieces > 1) DL_TIMED("embed_join", s, (embed_join<T, VEC><<<a.sum_blocks, EMB_THREADS, 0, s>>>((T *)gw, a)))
    DL_BY_TYPE(type, T, if (vec) { SUMS(true); } else { SUMS(false); });
#undef SUMS
    return dl_launch_status();
}
