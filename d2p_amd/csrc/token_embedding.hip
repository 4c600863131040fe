// token_embedding.hip -- rows of a table by token, and the table's gradient
// (include/d2p_amd_training.h).
//
// Forward: bound by reading rows and writing the result; a team of lanes copies rows, eight
// numbers a lane, four rows in flight (two: 42 us for 38 at [262144, 256] of 30000, eight 44), in up
// to eight workgroups a compute unit (as many as there are rows: 67).  (Of 30000 some of which are
// frequent; of as many that all occur alike 44 us.)  bf16 [131072, 1024] of 65536 tokens in 80 us:
// 3.4 TB/s written, about 5 with what is read.
//
// Backward: the gradient's rows of one token have to come together.  Positions are sorted by
// token (a stable radix sort of up to ten bits a pass, so that sums have one order), cut into chunks
// of equal length, and a team of lanes adds up its chunk's rows, run by run.  A run inside a
// chunk goes to the table; one that crosses a border leaves its part in the workspace, and a
// last kernel joins those.  Tokens that do not occur are marked by the sort's last pass, and
// their rows zeroed beside the sums, so that every row is written once.
//
// bf16 [131072, 1024] of 65536 tokens in 108 us: two passes of the sort 2 (4.8 + 11.4), sums 71 (the
// gradient read and the table written at 5.6 TB/s), joins 5.5.  Sums by atomics into the table
// would need it in float32, cleared, and rounded at the end, and their order would change from run to
// run.
#include <algorithm>
#include <type_traits>

#include "training.hip.h"

namespace d2p_amd {
namespace enc {

constexpr int SLAB = 64 * RUN;      // features that one wave takes

struct EmbedArgs {
    d2p_token_embedding_params p;
    const void* weight;
    void* out;
    int lanes;
    Divisor by_length;
};
constexpr int DEEP = 4;             // rows that a team has in flight
// As much as the card's last cache holds is written past it: bf16 [131072, 1024] of 65536 tokens
// 80 us, 103 without; with the norm that reads it next 201 either way.  Less is left for that norm:
// [65536, 512] 42.4 us, 44.2 past the caches.
constexpr long long CACHES = 256 << 20;

// The token at position n of [B, L]: its row; ABSENT for padding and past its sequence's
// length; WRONG for one that the table does not have or whose sequence's length is out of range.
constexpr int ABSENT = -1, WRONG = -2;
__device__ __forceinline__ int token_at(const d2p_token_embedding_params& p,
                                        const Divisor& by_length, int n) {
    if (p.lengths) {
        const int b = by_length(n), l = n - b * p.L, length = p.lengths[b];
        if (length < 0 || length > p.L) return WRONG;
        if (l >= length) return ABSENT;
    }
    const long long t = p.token_bytes == 8 ? ((const long long*)p.tokens)[n]
                                           : ((const int*)p.tokens)[n];
    if (t == p.padding && t >= 0) return ABSENT;
    return t >= 0 && t < p.V ? (int)t : WRONG;
}

// PAST: more is written than any cache keeps
template <class TW, class TO, bool PAST>
__global__ void __launch_bounds__(256) token_embedding_kernel(EmbedArgs a) {
    const d2p_token_embedding_params& p = a.p;
    const int n0 = threadIdx.x & (a.lanes - 1), teams = 256 / a.lanes;
    const long long rows = (long long)p.B * p.L, step = (long long)gridDim.x * teams;
    for (long long row = (long long)blockIdx.x * teams + threadIdx.x / a.lanes; row < rows;
         row += DEEP * step) {
        int t[DEEP];
#pragma unroll
        for (int u = 0; u < DEEP; ++u)
            t[u] = row + u * step < rows ? token_at(p, a.by_length, (int)(row + u * step)) : ABSENT;
        for (int at = n0 * RUN; at < p.D; at += a.lanes * RUN) {
            Eight<TW> r[DEEP];
#pragma unroll
            for (int u = 0; u < DEEP; ++u)
                r[u] = load_run((const TW*)a.weight + (long long)max(t[u], 0) * p.D, at, p.D);
#pragma unroll
            for (int u = 0; u < DEEP; ++u) {
                float x[RUN];
                unpack(r[u], at, p.D, t[u] >= 0, x);
#pragma unroll
                for (int e = 0; e < RUN; ++e) x[e] = t[u] == WRONG ? __builtin_nanf("") : x[e] * p.scale;
                if (row + u * step < rows)
                    store_run<PAST>((TO*)a.out + (row + u * step) * p.D + at, p.D - at, x);
            }
        }
    }
}

// ---------------------------------------------------------------------------
// sort
// ---------------------------------------------------------------------------
constexpr int SORT_THREADS = 1024, SORT_WAVES = SORT_THREADS / 64;
constexpr int MOST_BITS = 10, MOST_TILES = 128;

struct SortArgs {
    d2p_token_embedding_params p;
    Divisor by_length;
    int N;                          // positions
    int tiles, tile_bits;           // of 1 << tile_bits positions each
    int shift, bits;                // the digit of this pass
    int first, last;                // first, last pass
    const unsigned *keys, *at;      // of the pass before: tokens (V for none) and positions
    unsigned *keys_to, *at_to;
    unsigned* counts;               // [tiles][1 << bits]
    unsigned char* present;         // [V rounded up to 16]
};

__device__ __forceinline__ unsigned key_at(const SortArgs& a, int n) {
    if (!a.first) return a.keys[n];
    const int t = token_at(a.p, a.by_length, n);
    return t < 0 ? (unsigned)a.p.V : (unsigned)t;
}

__device__ __forceinline__ void clear_present(const SortArgs& a, long long from, long long step) {
    const long long n = (a.p.V + 15LL) / 16;
    for (long long i = from; i < n; i += step) ((u4v*)a.present)[i] = u4v{};
}

// How often each digit occurs in each tile; the first pass clears the marks too.
__global__ void __launch_bounds__(SORT_THREADS) count_digits_kernel(SortArgs a) {
    __shared__ unsigned count[1 << MOST_BITS];
    const long long me = (long long)blockIdx.x * SORT_THREADS + threadIdx.x;
    const long long all = (long long)gridDim.x * SORT_THREADS;
    const int digits = 1 << a.bits;
    if (a.first) clear_present(a, me, all);
    if ((int)blockIdx.x >= a.tiles) return;
    if ((int)threadIdx.x < digits) count[threadIdx.x] = 0;
    __syncthreads();
    const long long n0 = (long long)blockIdx.x << a.tile_bits;
    const long long n1 = min(n0 + (1LL << a.tile_bits), (long long)a.N);
    for (long long n = n0 + threadIdx.x; n < n1; n += SORT_THREADS)
        atomicAdd(&count[key_at(a, (int)n) >> a.shift & (digits - 1)], 1u);
    __syncthreads();
    if ((int)threadIdx.x < digits)
        a.counts[(long long)blockIdx.x * digits + threadIdx.x] = count[threadIdx.x];
}

// What a sort keeps in LDS for digits of `bits` bits.
struct SortLds {
    unsigned* wave;     // [SORT_WAVES][digits]: of each wave's share: counts, then next places
    unsigned* base;     // [digits]: the next key's place
    unsigned* part;     // [2][SORT_THREADS]
    unsigned* scan;     // [SORT_WAVES]
    int digits;
    __device__ __forceinline__ SortLds(unsigned* lds, int bits) : digits(1 << bits) {
        part = lds;
        scan = part + 2 * SORT_THREADS;
        base = scan + SORT_WAVES;
        wave = base + digits;
    }
    static size_t bytes(int bits) {
        return (2 * SORT_THREADS + SORT_WAVES + (size_t)(SORT_WAVES + 1) * (1 << bits)) * 4;
    }
    // base[d] = the `all` of smaller digits + before, by the thread of digit d (others: zeros)
    __device__ __forceinline__ void set_bases(unsigned all, unsigned before) {
        const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
        unsigned sum = all;
#pragma unroll
        for (int o = 1; o < 64; o *= 2) {
            const unsigned x = __shfl_up(sum, o, 64);
            if (lane >= o) sum += x;
        }
        if (lane == 63) scan[w] = sum;
        __syncthreads();
        if ((int)threadIdx.x >= digits) return;
        unsigned below = 0;
        for (int i = 0; i < w; ++i) below += scan[i];
        base[threadIdx.x] = below + sum - all + before;
    }
};

// The bases of a tile's digits: keys of smaller digits anywhere, keys of the digit in the tiles
// before.  The threads that no digit has take a share of the tiles.
__device__ __forceinline__ void digit_bases(SortLds& s, const unsigned* counts, int tiles, int tile) {
    const int d = threadIdx.x & (s.digits - 1), g = threadIdx.x / s.digits;
    const int groups = SORT_THREADS / s.digits;
    unsigned all = 0, before = 0;
#pragma unroll 16
    for (int t = g; t < tiles; t += groups) {
        const unsigned c = counts[(long long)t * s.digits + d];
        all += c;
        before += t < tile ? c : 0;
    }
    s.part[threadIdx.x] = all;
    s.part[SORT_THREADS + threadIdx.x] = before;
    __syncthreads();
    all = before = 0;
    if (g == 0)
        for (int i = 0; i < groups; ++i) {
            all += s.part[i * s.digits + d];
            before += s.part[SORT_THREADS + i * s.digits + d];
        }
    s.set_bases(all, before);
}

// Lanes of the wave whose digit is this lane's, among the lanes that are `on`.
__device__ __forceinline__ unsigned long long same_digit(unsigned digit, int bits, bool on) {
    unsigned long long m = __ballot(on);
    for (int b = 0; b < bits; ++b) {
        const unsigned long long ones = __ballot(digit >> b & 1);
        m &= digit >> b & 1 ? ones : ~ones;
    }
    return m;
}

// One part of a tile of ITEMS keys a thread: wave w has the keys 64 ITEMS w .. of it, in order.
// place[i]: where key i goes; s.base moves on by the part's counts.
template <int ITEMS>
__device__ __forceinline__ void place_keys(SortLds& s, int bits, const unsigned (&digit)[ITEMS],
                                           int here, unsigned (&place)[ITEMS]) {
    const int lane = threadIdx.x & 63;
    unsigned* mine = s.wave + (threadIdx.x >> 6) * s.digits;
    for (int i = lane; i < s.digits; i += 64) mine[i] = 0;
    // places among the wave's keys.  (A wave's LDS accesses run in their order: all lanes have
    // read before the first one of a digit writes)
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        const bool on = 64 * i + lane < here;
        const unsigned long long peers = same_digit(digit[i], bits, on);
        const int rank = __popcll(peers & ((1ULL << lane) - 1));
        __builtin_amdgcn_wave_barrier();
        const unsigned before = on ? mine[digit[i]] : 0;
        __builtin_amdgcn_wave_barrier();
        if (on && rank == 0) mine[digit[i]] = before + __popcll(peers);
        place[i] = before + rank;
    }
    __syncthreads();
    if ((int)threadIdx.x < s.digits) {
        unsigned next = s.base[threadIdx.x], c[SORT_WAVES];
#pragma unroll
        for (int w = 0; w < SORT_WAVES; ++w) c[w] = s.wave[w * s.digits + threadIdx.x];
#pragma unroll
        for (int w = 0; w < SORT_WAVES; ++w) {
            s.wave[w * s.digits + threadIdx.x] = next;
            next += c[w];
        }
        s.base[threadIdx.x] = next;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < ITEMS; ++i)
        if (64 * i + lane < here) place[i] += mine[digit[i]];
}

// Moves each key and its position to their places by the digit.  (Counting the next pass's digits
// here, where the keys arrive, took 40 us in global atomics for the 5 of its own kernel.)
template <int ITEMS>
__global__ void __launch_bounds__(SORT_THREADS) move_keys_kernel(SortArgs a) {
    extern __shared__ unsigned sort_lds[];
    SortLds s(sort_lds, a.bits);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long long n0 = (long long)blockIdx.x << a.tile_bits;
    const long long n1 = min(n0 + (1LL << a.tile_bits), (long long)a.N);
    for (long long part = n0; part < n1; part += SORT_THREADS * ITEMS) {
        const long long w0 = part + wave * 64 * ITEMS;
        const int here = (int)min(max(n1 - w0, 0LL), 64LL * ITEMS);
        unsigned key[ITEMS], at[ITEMS], digit[ITEMS], place[ITEMS];
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const int k = 64 * i + lane, n = (int)(w0 + k);
            key[i] = k < here ? key_at(a, n) : 0;
            at[i] = k < here && !a.first ? a.at[n] : (unsigned)n;
            digit[i] = key[i] >> a.shift & (s.digits - 1);
        }
        __syncthreads();        // (the part before has its places)
        if (part == n0) digit_bases(s, a.counts, a.tiles, blockIdx.x);
        place_keys(s, a.bits, digit, here, place);
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            if (64 * i + lane >= here) continue;
            a.keys_to[place[i]] = key[i];
            a.at_to[place[i]] = at[i];
            if (a.last && key[i] < (unsigned)a.p.V) a.present[key[i]] = 1;
        }
    }
}

// All of a short sort in one workgroup: the passes exchange through LDS.
template <int ITEMS>
__global__ void __launch_bounds__(SORT_THREADS) sort_short_kernel(SortArgs a, int passes) {
    constexpr int MOST = SORT_THREADS * ITEMS;
    extern __shared__ unsigned sort_lds[];
    SortLds s(sort_lds + 2 * MOST, a.bits);
    unsigned *keys = sort_lds, *ats = sort_lds + MOST;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int w0 = wave * 64 * ITEMS;
    const int here = min(max(a.N - w0, 0), 64 * ITEMS);
    clear_present(a, threadIdx.x, SORT_THREADS);
    unsigned key[ITEMS], at[ITEMS];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        const int n = w0 + 64 * i + lane;
        key[i] = n < a.N ? key_at(a, n) : 0;
        at[i] = n;
    }
    for (int pass = 0; pass < passes; ++pass) {
        unsigned digit[ITEMS], place[ITEMS];
        s.part[threadIdx.x] = 0;        // (one tile, whose counts lie here)
        __syncthreads();
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            digit[i] = key[i] >> (pass * a.bits) & (s.digits - 1);
            if (64 * i + lane < here) atomicAdd(&s.part[digit[i]], 1u);
        }
        __syncthreads();
        s.set_bases((int)threadIdx.x < s.digits ? s.part[threadIdx.x] : 0, 0);
        __syncthreads();
        place_keys(s, a.bits, digit, here, place);
#pragma unroll
        for (int i = 0; i < ITEMS; ++i)
            if (64 * i + lane < here) {
                keys[place[i]] = key[i];
                ats[place[i]] = at[i];
            }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const int n = w0 + 64 * i + lane;
            key[i] = n < a.N ? keys[n] : 0;
            at[i] = n < a.N ? ats[n] : 0;
        }
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        const int n = w0 + 64 * i + lane;
        if (n >= a.N) continue;
        a.keys_to[n] = key[i];
        a.at_to[n] = at[i];
        if (key[i] < (unsigned)a.p.V) a.present[key[i]] = 1;
    }
}

// ---------------------------------------------------------------------------
// sums
// ---------------------------------------------------------------------------
struct TableArgs {
    d2p_token_embedding_params p;
    const void* grad;
    void* dweight;
    const unsigned *keys, *at;      // sorted, and room for eight behind them
    const unsigned char* present;
    float *head, *tail;             // [chunks][D]: parts of runs that come from the chunk before
                                    // (or go through it), that begin in a chunk and go on
    Divisor by_length;
    int N, chunk, chunks;           // positions of a chunk: a multiple of eight
    int lanes, slabs;               // of a team; of SLAB features
    int sum_blocks, zero_blocks;
};

template <class TW, class TO>
__global__ void __launch_bounds__(256) table_grad_kernel(TableArgs a) {
    const d2p_token_embedding_params& p = a.p;
    const int D = p.D, teams = 256 / a.lanes;
    const unsigned V = p.V;
    const int team = threadIdx.x / a.lanes, n0 = (threadIdx.x & (a.lanes - 1)) * RUN;
    float acc[RUN] = {};
    if ((int)blockIdx.x >= a.sum_blocks) {
        // rows of tokens that do not occur
        for (long long v = (long long)(blockIdx.x - a.sum_blocks) * teams + team; v < V;
             v += (long long)a.zero_blocks * teams) {
            if (a.present[v]) continue;
            for (int f = n0; f < D; f += a.lanes * RUN)
                store_run((TW*)a.dweight + v * D + f, D - f, acc);
        }
        return;
    }
    const int c = (blockIdx.x / a.slabs) * teams + team, f = blockIdx.x % a.slabs * SLAB + n0;
    if (c >= a.chunks || f >= D) return;
    const int left = D - f;
    const unsigned N = a.N, i0 = c * a.chunk, i1 = min(i0 + a.chunk, N);   // (N + 8 may pass 2^31)
    unsigned run = i0 ? a.keys[i0 - 1] : V;     // the token before the chunk
    bool inside = false;                        // the run began in the chunk
    auto flush = [&](bool ended) {
        if (run >= V || (!inside && i0 == 0)) return;
        if (inside && ended) {
#pragma unroll
            for (int e = 0; e < RUN; ++e) acc[e] *= p.scale;
            store_run((TW*)a.dweight + (long long)run * D + f, left, acc);
        } else {
            store_run((inside ? a.tail : a.head) + (long long)c * D + f, left, acc);
        }
    };
    bool any = false;                           // acc holds a part of `run`
    // the next eight rows' places are under way with these eight rows
    u4v next[4];
    auto places = [&](unsigned i) {
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            next[q] = *(const u4v*)(a.keys + i + 4 * q);
            next[2 + q] = *(const u4v*)(a.at + i + 4 * q);
        }
    };
    places(i0);
    for (unsigned i = i0; i < i1; i += 8) {
        const u4v k[2] = {next[0], next[1]}, n[2] = {next[2], next[3]};
        if (k[0][0] >= V) break;                // only unused positions are left
        Eight<TO> r[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const bool on = i + u < i1 && k[u >> 2][u & 3] < V;
            const unsigned at = on ? n[u >> 2][u & 3] : 0;
            const unsigned b = a.by_length(at), l = at - b * p.L;
            r[u] = load_run<true>((const TO*)a.grad + (long long)b * p.grad.batch +
                                  (long long)l * p.grad.row, f, D);
        }
        places(min(i + 8, i1 - 1 & ~7u));
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            if (i + u >= i1) break;
            const unsigned key = k[u >> 2][u & 3];
            if (key != run) {
                if (any) flush(true);
#pragma unroll
                for (int e = 0; e < RUN; ++e) acc[e] = 0.0f;
                run = key;
                inside = true;
            }
            any = true;
            float x[RUN];
            unpack(r[u], f, D, key < V, x);
#pragma unroll
            for (int e = 0; e < RUN; ++e) acc[e] += x[e];
        }
    }
    if (any) flush(i1 >= N || a.keys[i1] != run);
}

// Joins the parts of each run that begins in chunk c and ends in a later one: the teams of a
// workgroup take them in turn, four at a time, and their sums meet in order.
template <class TW>
__global__ void __launch_bounds__(256) join_runs_kernel(TableArgs a) {
    __shared__ __align__(16) float part[256 * RUN];
    const int D = a.p.D, c = blockIdx.x / a.slabs, f0 = blockIdx.x % a.slabs * SLAB;
    const int lane = threadIdx.x & 63, team = threadIdx.x / a.lanes, teams = 256 / a.lanes;
    const unsigned i0 = c * a.chunk, i1 = i0 + a.chunk;
    if (i1 >= (unsigned)a.N) return;
    const unsigned run = a.keys[i1 - 1];
    if (run >= (unsigned)a.p.V || a.keys[i1] != run) return;            // none goes on
    if (a.keys[i0] == run && i0 && a.keys[i0 - 1] == run) return;      // it began earlier
    // the chunk that the run ends in: the first whose last key, or the one after, is another
    int last = c + 1;
    for (;;) {
        const long long n = ((long long)last + lane + 1) * a.chunk;
        const unsigned long long on = __ballot(n < a.N && a.keys[min(n, (long long)a.N - 1)] == run);
        if (~on) {
            last += __builtin_ctzll(~on);
            break;
        }
        last += 64;
    }
    const int f = f0 + (threadIdx.x & (a.lanes - 1)) * RUN;
    float acc[RUN] = {};
    if (team == 0) unpack(load_run(a.tail + (long long)c * D, f, D), f, D, true, acc);
    for (int k = c + 1 + team; k <= last; k += 4 * teams) {
        Eight<float> r[4];
#pragma unroll
        for (int u = 0; u < 4; ++u)
            r[u] = load_run(a.head + (long long)min(k + teams * u, last) * D, f, D);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            float x[RUN];
            unpack(r[u], f, D, k + teams * u <= last, x);
#pragma unroll
            for (int e = 0; e < RUN; ++e) acc[e] += x[e];
        }
    }
    f4v* mine = (f4v*)(part + threadIdx.x * RUN);
    mine[0] = f4v{acc[0], acc[1], acc[2], acc[3]};
    mine[1] = f4v{acc[4], acc[5], acc[6], acc[7]};
    __syncthreads();
    const int numbers = a.lanes * RUN;
    for (int d = threadIdx.x; d < min(numbers, D - f0); d += 256) {
        float s = 0.0f;
        for (int t = 0; t < teams; ++t) s += part[t * numbers + d];
        ((TW*)a.dweight)[(long long)run * D + f0 + d] = (TW)(s * a.p.scale);
    }
}

// ---------------------------------------------------------------------------
// small tables
// ---------------------------------------------------------------------------
// A table of few tokens needs no sort: a workgroup keeps a sum for each token and each of 512
// features in LDS, where a thread adds to the numbers of its own two features only, in the order
// of its rows.  The workgroups' tables are added up by rows.hip.
struct SmallArgs {
    d2p_token_embedding_params p;
    Divisor by_length;
    const void* grad;
    float* partial;                 // [splits][V][D]
    int lanes, slabs, rows;         // lanes: threads of a team, two features each; rows of a split
};
constexpr int SMALL_ROWS = 512;     // whose tokens are looked up at a time

template <class TO> __global__ void __launch_bounds__(256) table_grad_small_kernel(SmallArgs a) {
    constexpr int ROWS = 16;        // in flight
    struct Two { TO v[2]; };
    extern __shared__ float sums[]; // [V][2][256], and the tokens
    const d2p_token_embedding_params& p = a.p;
    int* tokens = (int*)(sums + p.V * SLAB);
    const int me = threadIdx.x, teams = 256 / a.lanes, team = me / a.lanes;
    const int split = blockIdx.x / a.slabs;
    const int f = blockIdx.x % a.slabs * SLAB + (me & (a.lanes - 1)) * 2;
    const long long N = (long long)p.B * p.L;
    const unsigned r0 = min((long long)split * a.rows, N), r1 = min((long long)r0 + a.rows, N);
    // behind the features' end the last two are read; of a lone last one, it and the one before
    const int f0 = min(f, p.D - 2);
    const bool lone = f == p.D - 1;
    for (int i = 0; i < p.V * 2; ++i) sums[i * 256 + me] = 0.0f;
    for (unsigned part = r0; part < r1; part += SMALL_ROWS) {
        const int rows = min(SMALL_ROWS, (int)(r1 - part));
        __syncthreads();
        for (int i = me; i < rows; i += 256) tokens[i] = token_at(p, a.by_length, part + i);
        __syncthreads();
        for (int r = team; r < rows; r += ROWS * teams) {
            Two x[ROWS];
            int t[ROWS];
#pragma unroll
            for (int u = 0; u < ROWS; ++u) {
                const int i = min(r + u * teams, rows - 1);
                const unsigned n = part + i, b = a.by_length(n);
                x[u] = *(const Two*)((const TO*)a.grad + (long long)b * p.grad.batch +
                                     (long long)(n - b * p.L) * p.grad.row + f0);
                t[u] = r + u * teams < rows ? tokens[i] : ABSENT;
            }
#pragma unroll
            for (int u = 0; u < ROWS; ++u) {
                if (t[u] < 0) continue;
                float* to = sums + t[u] * SLAB + me;
                // (LDS additions as such, ds_add_f32, take 300 cycles a wave)
                const float s0 = to[0], s1 = to[256];
                to[0] = s0 + (float)(lone ? x[u].v[1] : x[u].v[0]);
                to[256] = s1 + (float)x[u].v[1];
            }
        }
    }
    __syncthreads();
    // the teams' tables, in order
    float* to = a.partial + (long long)split * p.V * p.D;
    for (int v = team; v < p.V; v += teams) {
        const float* from = sums + v * SLAB + (me & (a.lanes - 1));
        float s0 = 0.0f, s1 = 0.0f;
        for (int k = 0; k < 256; k += a.lanes) {
            s0 += from[k];
            s1 += from[k + 256];
        }
        if (f < p.D) to[(long long)v * p.D + f] = s0;
        if (f + 1 < p.D) to[(long long)v * p.D + f + 1] = s1;
    }
}

namespace {

int check(const d2p_token_embedding_params* p) {
    D2P_REQUIRE(p != nullptr, "null parameters");
    D2P_REQUIRE(known_pair(p->weight_dtype, p->dtype),
                "unknown element types, or a pair other than equal ones and 16 bits beside float32");
    D2P_REQUIRE(p->B >= 0 && p->L >= 0, "negative size");
    D2P_REQUIRE((long long)p->B * p->L < 1LL << 31, "too many tokens");
    D2P_REQUIRE(p->V >= 1 && p->V < 0x7fffffff, "the table must have between 1 and 2^31 - 2 rows");
    D2P_REQUIRE(p->D >= RUN && p->D <= 1 << 20, "features must be between 8 and 2^20");
    D2P_REQUIRE(p->token_bytes == 4 || p->token_bytes == 8, "tokens must have 4 or 8 bytes");
    D2P_REQUIRE(p->padding >= -1 && p->padding < p->V, "padding must be a token, or -1");
    D2P_REQUIRE(p->scale > -__builtin_inff() && p->scale < __builtin_inff(), "scale must be finite");
    return D2P_OK;
}

size_t round16(size_t n) { return (n + 15) & ~(size_t)15; }

// Up to here one workgroup sorts all keys.  bf16 [N, 256], V 4097, the whole gradient: N 64 11.4 us
// (by tiles 18.6), 1024 15.0 (22.6), 4096 21.9 (27.7); 8192 keys 31.8 (29.9).
constexpr int SHORT = 4 * SORT_THREADS;
// A table of up to SMALL tokens and SMALL_TABLE numbers needs no sort.  bf16, 16384 rows: V 21, D 256
// 13.5 us (21.5 sorted), V 21, D 512 19.0 (22.2), V 64, D 64 11.7 (18.3); above, V 32, D 512 20.8
// (21.3) and with 131072 rows 51.7 (47.4), V 64, D 256 22.2 (19.0).
constexpr int SMALL = 64, SMALL_TABLE = 12288;

// How the backward pass splits its work, and its workspace.
struct Plan {
    int N, bits, passes, tile_bits, tiles;
    bool short_sort;
    int splits;             // of a small table's rows; 0 for another table
    int lanes, slabs, chunk, chunks;
    size_t keys, counts, present, parts, total;

    explicit Plan(const d2p_token_embedding_params& p) {
        N = p.B * p.L;
        bits = 1;
        while (bits < 31 && (p.V >> bits) != 0) ++bits;     // of V, which stands for no token
        passes = cdiv(bits, MOST_BITS);
        bits = cdiv(bits, passes);
        short_sort = N <= SHORT && p.V <= 1 << 20;
        // tiles of one key a thread, and where those would be too many for each to add up all
        // counts, of two and more (bf16, V 65536: [32768, 64] 31.7 us, 37.9 with two a thread;
        // [1048576, 64] 133.8, 138.8 with one)
        tile_bits = N <= MOST_TILES * SORT_THREADS ? 10 : 11;
        while (cdiv(N, 1 << tile_bits) > MOST_TILES) ++tile_bits;
        tiles = std::max(1, cdiv(N, 1 << tile_bits));
        lanes = std::min(team_of(p.D), 64);
        slabs = cdiv(p.D, SLAB);
        splits = 0;
        if (p.V <= SMALL && (long long)p.V * p.D <= SMALL_TABLE) {
            // workgroups that the card's LDS holds at a time, but no more than rows.hip adds up as fast,
            // each with more rows than its table has (bf16, V 4, 16384 rows, D 64 8.8 us, D 512 13.1;
            // with eight rows and 2048 workgroups 18.1 and 22.4)
            const int groups = 256 * std::min(4, 156 / (2 * p.V));
            splits = std::max(1, std::min(groups / slabs, N / std::max(32, 2 * p.V)));
            if (splits > 256) splits -= splits % 256;       // as many for each compute unit
            if (N) splits = cdiv(N, cdiv(N, splits));
            total = (size_t)splits * p.V * p.D * 4;
            return;
        }
        // As many waves as the card has SIMDs, of chunks from 8 to 128 positions; longer ones where
        // that leaves very many.  bf16, us with 16, 32, 64, 128, 256 positions (* taken):
        //   N 16384,   V 4097,  D 512:    33*  35   42   56   85   (8: 36)
        //   N 131072,  V 65536, D 64:     48*  49   56   74  112   (8: 54)
        //   N 131072,  V 200,   D 1024:  124   95   77   67*  73
        //   N 131072,  V 65536, D 1024:  120  112  107  107* 121
        //   N 4194304, V 65536, D 64:    592  482  419  390* 379
        const long long waves = (long long)N * slabs * lanes / 64;
        chunk = 8;
        while (chunk < (waves / chunk >= 1 << 16 ? 256 : 128) && waves / chunk > 1024) chunk *= 2;
        chunks = cdiv(N, chunk);
        keys = round16(((size_t)N + 8) * 4);
        counts = round16(((size_t)tiles << bits) * 4);
        present = round16(p.V);
        parts = round16((size_t)chunks * p.D * 4);
        total = 4 * keys + counts + present + 2 * parts;
    }
};

int launch_small(const d2p_token_embedding_params& p, const Plan& plan, const void* grad,
                 float* partial, void* dweight, hipStream_t st) {
    int lanes = 1;
    while (lanes < 256 && 2 * lanes < p.D) lanes *= 2;
    const SmallArgs a{p, Divisor(p.L), grad, partial, lanes, plan.slabs,
                      plan.N ? cdiv(plan.N, plan.splits) : 0};
    SumJobs jobs;
    jobs.init(p.V * p.D);
    jobs.scale = p.scale;
    jobs.add(partial, dweight, p.weight_dtype, plan.N ? plan.splits : 0, 1);
    if (plan.N)
        D2P_TRY(with_pair(p.dtype, p.dtype, [&](auto to, auto) {
            using TO = typename decltype(to)::type;
            static LdsAllowed known;
            D2P_TRY(allow_lds((const void*)table_grad_small_kernel<TO>, known));
            D2P_LAUNCH("token_embedding_backward", table_grad_small_kernel<TO>,
                       dim3(plan.splits * plan.slabs), dim3(256),
                       (p.V * SLAB + SMALL_ROWS) * sizeof(float), st,
                       a);
            D2P_HIP(hipGetLastError());
            return D2P_OK;
        }));
    return launch_sum_rows("token_embedding_sum", jobs, st);
}

int launch_sort(const d2p_token_embedding_params& p, const Plan& plan, char* ws, TableArgs& t,
                hipStream_t st) {
    unsigned* key[2] = {(unsigned*)ws, (unsigned*)(ws + plan.keys)};
    unsigned* at[2] = {(unsigned*)(ws + 2 * plan.keys), (unsigned*)(ws + 3 * plan.keys)};
    SortArgs a{};
    a.p = p;
    a.by_length = Divisor(p.L);
    a.N = plan.N;
    a.tiles = plan.tiles;
    a.tile_bits = plan.tile_bits;
    a.bits = plan.bits;
    a.first = 1;
    a.keys_to = key[0];
    a.at_to = at[0];
    a.counts = (unsigned*)(ws + 4 * plan.keys);
    a.present = (unsigned char*)(ws + 4 * plan.keys + plan.counts);
    t.present = a.present;
    if (plan.short_sort) {
        const auto sort = [&](auto items) {
            static LdsAllowed known;
            D2P_TRY(allow_lds((const void*)sort_short_kernel<items()>, known));
            D2P_LAUNCH("token_sort", sort_short_kernel<items()>, dim3(1), dim3(SORT_THREADS),
                       2 * SORT_THREADS * items() * sizeof(unsigned) + SortLds::bytes(plan.bits), st,
                       a, plan.passes);
            D2P_HIP(hipGetLastError());
            return D2P_OK;
        };
        D2P_TRY(plan.N <= SORT_THREADS       ? sort(std::integral_constant<int, 1>{})
                : plan.N <= 2 * SORT_THREADS ? sort(std::integral_constant<int, 2>{})
                                             : sort(std::integral_constant<int, 4>{}));
    }
    for (int n = 0; n < plan.passes && !plan.short_sort; ++n) {
        a.first = n == 0;
        a.last = n == plan.passes - 1;
        a.shift = plan.bits * n;
        a.keys = key[(n + 1) & 1];
        a.at = at[(n + 1) & 1];
        a.keys_to = key[n & 1];
        a.at_to = at[n & 1];
        const int clearing = a.first ? (int)std::min<long long>(256, p.V / (64 << 10) + 1) : 1;
        D2P_LAUNCH("token_sort_count", count_digits_kernel, dim3(std::max(plan.tiles, clearing)),
                   dim3(SORT_THREADS), 0, st, a);
        D2P_HIP(hipGetLastError());
        const auto move = [&](auto items) {
            static LdsAllowed known;
            D2P_TRY(allow_lds((const void*)move_keys_kernel<items()>, known));
            D2P_LAUNCH("token_sort_move", move_keys_kernel<items()>, dim3(plan.tiles),
                       dim3(SORT_THREADS), SortLds::bytes(plan.bits), st, a);
            D2P_HIP(hipGetLastError());
            return D2P_OK;
        };
        D2P_TRY(plan.tile_bits == 10 ? move(std::integral_constant<int, 1>{})
                                     : move(std::integral_constant<int, 2>{}));
    }
    t.keys = a.keys_to;
    t.at = a.at_to;
    return D2P_OK;
}

}  // namespace
}  // namespace enc
}  // namespace d2p_amd

using namespace d2p_amd;
using namespace d2p_amd::enc;

extern "C" int d2p_token_embedding(const d2p_token_embedding_params* p, const void* weight,
                                   void* out, void* stream) {
    D2P_TRY(check(p));
    if ((long long)p->B * p->L == 0) return D2P_OK;
    D2P_REQUIRE(p->tokens && out && weight, "null pointer argument");
    EmbedArgs a{*p, weight, out, std::min(team_of(p->D), 64), Divisor(p->L)};
    const int most = 8 * std::max(device_cus(), 1);
    // a workgroup for each compute unit first, then as many rows as a team has in flight (float32 to
    // bf16 [16384, 512]: 8.1 us, 9.3 with more workgroups of fewer rows)
    const int rows = p->B * p->L, teams = 256 / a.lanes;
    const int grid = std::min({cdiv(rows, teams), std::max(most / 8, cdiv(rows, DEEP * teams)), most});
    return with_pair(p->weight_dtype, p->dtype, [&](auto tw, auto to) {
        using TW = typename decltype(tw)::type;
        using TO = typename decltype(to)::type;
        const bool past = (long long)p->B * p->L * p->D * (int)sizeof(TO) >= CACHES;
        const auto kernel = past ? token_embedding_kernel<TW, TO, true>
                                 : token_embedding_kernel<TW, TO, false>;
        D2P_LAUNCH("token_embedding", kernel, dim3(grid), dim3(256), 0, (hipStream_t)stream, a);
        D2P_HIP(hipGetLastError());
        return D2P_OK;
    });
}

extern "C" size_t d2p_token_embedding_backward_workspace_bytes(const d2p_token_embedding_params* p) {
    if (!p || p->B < 0 || p->L < 0 || p->V < 1 || p->D < RUN || p->D > 1 << 20 ||
        p->V >= 0x7fffffff || (long long)p->B * p->L >= 1LL << 31)
        return 0;
    return Plan(*p).total;
}

extern "C" int d2p_token_embedding_backward(const d2p_token_embedding_params* p, const void* grad,
                                            void* dweight, void* workspace, size_t workspace_bytes,
                                            void* stream) {
    D2P_TRY(check(p));
    const bool rows = (long long)p->B * p->L > 0;
    D2P_REQUIRE(dweight && (!rows || (p->tokens && grad)), "null pointer argument");
    const Plan plan(*p);
    D2P_REQUIRE(workspace && workspace_bytes >= plan.total, "workspace too small");
    D2P_REQUIRE(((uintptr_t)workspace & 15) == 0, "the workspace must be aligned to 16 bytes");
    hipStream_t st = (hipStream_t)stream;
    if (plan.splits)
        return launch_small(*p, plan, grad, (float*)workspace, dweight, st);
    TableArgs a{};
    a.p = *p;
    a.grad = grad;
    a.dweight = dweight;
    a.by_length = Divisor(p->L);
    a.N = plan.N;
    a.lanes = plan.lanes;
    a.slabs = plan.slabs;
    a.chunk = plan.chunk;
    a.chunks = plan.chunks;
    char* ws = (char*)workspace;
    a.head = (float*)(ws + plan.total - 2 * plan.parts);
    a.tail = (float*)(ws + plan.total - plan.parts);
    const int teams = 256 / plan.lanes;
    D2P_REQUIRE((long long)plan.chunks * plan.slabs < 1LL << 24, "too many tokens and features");
    a.sum_blocks = cdiv(plan.chunks, teams) * plan.slabs;
    a.zero_blocks = std::min(cdiv(p->V, teams), 4 * std::max(device_cus(), 1));
    D2P_TRY(launch_sort(*p, plan, ws, a, st));
    return with_pair(p->weight_dtype, p->dtype, [&](auto tw, auto to) {
        using TW = typename decltype(tw)::type;
        using TO = typename decltype(to)::type;
        D2P_LAUNCH("token_embedding_backward", (table_grad_kernel<TW, TO>),
                   dim3(a.sum_blocks + a.zero_blocks), dim3(256), 0, st, a);
        D2P_HIP(hipGetLastError());
        if (a.chunks > 1) {
            D2P_LAUNCH("token_embedding_join", join_runs_kernel<TW>, dim3(a.chunks * a.slabs),
                       dim3(256), 0, st, a);
            D2P_HIP(hipGetLastError());
        }
        return D2P_OK;
    });
}
