// token_embedding.hip -- rows of a table by token, and the table's gradient
// (include/d2p_amd_training.h).
//
// Forward: bound by writing the result; a team of lanes copies rows, eight numbers a lane.
//
// Backward: the gradient's rows of one token have to come together.  Positions are sorted by
// token (a stable radix sort of 8 bits a pass, so that sums have one order), cut into chunks
// of equal length, and a team of lanes adds up its chunk's rows, run by run.  A run inside a
// chunk goes to the table; one that crosses a border leaves its part in the workspace, and a
// last kernel joins those.  Tokens that do not occur are marked by the sort's last pass, and
// their rows zeroed beside the sums, so that every row is written once.
#include <algorithm>

#include "training.hip.h"

namespace d2p_amd {
namespace enc {

constexpr int SLAB = 64 * RUN;      // features that one wave takes

struct EmbedArgs {
    d2p_token_embedding_params p;
    const void* weight;
    void* out;
    int lanes;
};

// The token at position n of [B, L]: its row; ABSENT for padding and past its sequence's
// length; WRONG for one that the table does not have or whose sequence's length is out of range.
constexpr int ABSENT = -1, WRONG = -2;
__device__ __forceinline__ int token_at(const d2p_token_embedding_params& p, int n) {
    if (p.lengths) {
        const int l = n % p.L, length = p.lengths[n / p.L];
        if (length < 0 || length > p.L) return WRONG;
        if (l >= length) return ABSENT;
    }
    const long long t = p.token_bytes == 8 ? ((const long long*)p.tokens)[n]
                                           : ((const int*)p.tokens)[n];
    if (t == p.padding && t >= 0) return ABSENT;
    return t >= 0 && t < p.V ? (int)t : WRONG;
}

template <class TW, class TO>
__global__ void __launch_bounds__(256) token_embedding_kernel(EmbedArgs a) {
    const d2p_token_embedding_params& p = a.p;
    const int n0 = threadIdx.x & (a.lanes - 1), teams = 256 / a.lanes;
    const int rows = p.B * p.L;
    for (long long row = (long long)blockIdx.x * teams + threadIdx.x / a.lanes; row < rows;
         row += (long long)gridDim.x * teams) {
        const int t = token_at(p, (int)row);
        for (int at = n0 * RUN; at < p.D; at += a.lanes * RUN) {
            float x[RUN];
            load_run((const TW*)a.weight + (long long)max(t, 0) * p.D + at, t < 0 ? 0 : p.D - at, x);
#pragma unroll
            for (int e = 0; e < RUN; ++e) x[e] = t == WRONG ? __builtin_nanf("") : x[e] * p.scale;
            store_run((TO*)a.out + row * p.D + at, p.D - at, x);
        }
    }
}

// ---------------------------------------------------------------------------
// sort
// ---------------------------------------------------------------------------
constexpr int DIGITS = 256, SORT_THREADS = 1024, SORT_WAVES = SORT_THREADS / 64;
constexpr int MOST_TILES = 256;

struct SortArgs {
    d2p_token_embedding_params p;
    int N;                          // positions
    int tiles, tile;                // of `tile` positions each
    int shift, first, last;         // first, last pass
    const unsigned *keys, *at;      // of the pass before: tokens (V for none) and positions
    unsigned *keys_to, *at_to;
    unsigned* counts;               // [tiles][DIGITS]
    unsigned char* present;         // [V rounded up to 16]
};

__device__ __forceinline__ unsigned key_at(const SortArgs& a, int n) {
    if (!a.first) return a.keys[n];
    const int t = token_at(a.p, n);
    return t < 0 ? (unsigned)a.p.V : (unsigned)t;
}

__device__ __forceinline__ void clear_present(const SortArgs& a, long long from, long long step) {
    const long long n = (a.p.V + 15LL) / 16;
    for (long long i = from; i < n; i += step) ((u4v*)a.present)[i] = u4v{};
}

// How often each digit occurs in each tile; the first pass clears the marks too.
__global__ void __launch_bounds__(SORT_THREADS) count_digits_kernel(SortArgs a) {
    __shared__ unsigned count[DIGITS];
    if (a.first)
        clear_present(a, (long long)blockIdx.x * SORT_THREADS + threadIdx.x,
                      (long long)gridDim.x * SORT_THREADS);
    if ((int)blockIdx.x >= a.tiles) return;
    if (threadIdx.x < DIGITS) count[threadIdx.x] = 0;
    __syncthreads();
    const long long n0 = (long long)blockIdx.x * a.tile;
    const long long n1 = min(n0 + a.tile, (long long)a.N);
    for (long long n = n0 + threadIdx.x; n < n1; n += SORT_THREADS)
        atomicAdd(&count[key_at(a, (int)n) >> a.shift & (DIGITS - 1)], 1u);
    __syncthreads();
    if (threadIdx.x < DIGITS)
        a.counts[(long long)blockIdx.x * DIGITS + threadIdx.x] = count[threadIdx.x];
}

struct SortLds {
    unsigned wave[SORT_WAVES][DIGITS];   // of each wave's share: counts, then next places
    unsigned base[DIGITS];
    unsigned part[2][4][DIGITS];
    unsigned scan[4];
};

// s.base[d] = keys of smaller digits anywhere + keys of digit d in the tiles before this one
__device__ __forceinline__ void digit_bases(SortLds& s, const unsigned* counts, int tiles, int tile) {
    const int d = threadIdx.x & (DIGITS - 1), g = threadIdx.x / DIGITS;
    unsigned all = 0, before = 0;
#pragma unroll 8
    for (int t = g; t < tiles; t += 4) {
        const unsigned c = counts[(long long)t * DIGITS + d];
        all += c;
        before += t < tile ? c : 0;
    }
    s.part[0][g][d] = all;
    s.part[1][g][d] = before;
    __syncthreads();
    if (g == 0) {
        all = before = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            all += s.part[0][i][d];
            before += s.part[1][i][d];
        }
        unsigned sum = all;
        const int lane = d & 63;
#pragma unroll
        for (int o = 1; o < 64; o *= 2) {
            const unsigned x = __shfl_up(sum, o, 64);
            if (lane >= o) sum += x;
        }
        if (lane == 63) s.scan[d >> 6] = sum;
        s.base[d] = sum - all + before;
    }
    __syncthreads();
    if (g == 0) {
        unsigned below = 0;
        for (int w = 0; w < d >> 6; ++w) below += s.scan[w];
        s.base[d] += below;
    }
}

// Lanes of the wave whose digit is this lane's, among the lanes that are `on`.
__device__ __forceinline__ unsigned long long same_digit(unsigned digit, bool on) {
    unsigned long long m = __ballot(on);
#pragma unroll
    for (int b = 0; b < 8; ++b) {
        const unsigned long long ones = __ballot(digit >> b & 1);
        m &= digit >> b & 1 ? ones : ~ones;
    }
    return m;
}

// One part of a tile of ITEMS keys a thread: wave w has the keys 64 ITEMS w .. of it, in order.
// place[i]: where key i goes; s.base moves on by the part's counts.
template <int ITEMS>
__device__ __forceinline__ void place_keys(SortLds& s, const unsigned (&digit)[ITEMS], int here,
                                           unsigned (&place)[ITEMS]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int i = threadIdx.x; i < SORT_WAVES * DIGITS; i += SORT_THREADS) (&s.wave[0][0])[i] = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < ITEMS; ++i)
        if (64 * i + lane < here) atomicAdd(&s.wave[wave][digit[i]], 1u);
    __syncthreads();
    if (threadIdx.x < DIGITS) {
        unsigned next = s.base[threadIdx.x];
#pragma unroll
        for (int w = 0; w < SORT_WAVES; ++w) {
            const unsigned c = s.wave[w][threadIdx.x];
            s.wave[w][threadIdx.x] = next;
            next += c;
        }
        s.base[threadIdx.x] = next;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        const bool on = 64 * i + lane < here;
        const unsigned long long peers = same_digit(digit[i], on);
        const int rank = __popcll(peers & ((1ULL << lane) - 1));
        place[i] = on ? s.wave[wave][digit[i]] + rank : 0;
        // (a wave's LDS accesses run in their order: all have read before the first one adds)
        __builtin_amdgcn_wave_barrier();
        if (on && rank == 0) atomicAdd(&s.wave[wave][digit[i]], (unsigned)__popcll(peers));
        __builtin_amdgcn_wave_barrier();
    }
}

// Moves each key and its position to their places by the digit.
template <int ITEMS>
__global__ void __launch_bounds__(SORT_THREADS) move_keys_kernel(SortArgs a) {
    __shared__ SortLds s;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    digit_bases(s, a.counts, a.tiles, blockIdx.x);
    const long long n0 = (long long)blockIdx.x * a.tile;
    const long long n1 = min(n0 + a.tile, (long long)a.N);
    for (long long part = n0; part < n1; part += SORT_THREADS * ITEMS) {
        const long long w0 = part + wave * 64 * ITEMS;
        const int here = (int)min(max(n1 - w0, 0LL), 64LL * ITEMS);
        unsigned key[ITEMS], at[ITEMS], digit[ITEMS], place[ITEMS];
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const int k = 64 * i + lane, n = (int)(w0 + k);
            key[i] = k < here ? key_at(a, n) : 0;
            at[i] = k < here && !a.first ? a.at[n] : (unsigned)n;
            digit[i] = key[i] >> a.shift & (DIGITS - 1);
        }
        __syncthreads();
        place_keys(s, digit, here, place);
#pragma unroll
        for (int i = 0; i < ITEMS; ++i)
            if (64 * i + lane < here) {
                a.keys_to[place[i]] = key[i];
                a.at_to[place[i]] = at[i];
                if (a.last && key[i] < (unsigned)a.p.V) a.present[key[i]] = 1;
            }
    }
}

// All of a short sort in one workgroup: the passes exchange through LDS.
constexpr int SHORT_ITEMS = 8, SHORT = SORT_THREADS * SHORT_ITEMS;
__global__ void __launch_bounds__(SORT_THREADS) sort_short_kernel(SortArgs a, int bits) {
    __shared__ SortLds s;
    __shared__ unsigned keys[SHORT], ats[SHORT];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int w0 = wave * 64 * SHORT_ITEMS;
    const int here = min(max(a.N - w0, 0), 64 * SHORT_ITEMS);
    clear_present(a, threadIdx.x, SORT_THREADS);
    unsigned key[SHORT_ITEMS], at[SHORT_ITEMS];
#pragma unroll
    for (int i = 0; i < SHORT_ITEMS; ++i) {
        const int n = w0 + 64 * i + lane;
        key[i] = n < a.N ? key_at(a, n) : 0;
        at[i] = n;
    }
    for (int shift = 0; shift < bits; shift += 8) {
        unsigned digit[SHORT_ITEMS], place[SHORT_ITEMS];
        if (threadIdx.x < DIGITS) s.part[0][0][threadIdx.x] = 0;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < SHORT_ITEMS; ++i) {
            digit[i] = key[i] >> shift & (DIGITS - 1);
            if (64 * i + lane < here) atomicAdd(&s.part[0][0][digit[i]], 1u);
        }
        __syncthreads();
        // (one tile, whose counts lie in LDS)
        const unsigned all = threadIdx.x < DIGITS ? s.part[0][0][threadIdx.x] : 0;
        unsigned sum = all;
#pragma unroll
        for (int o = 1; o < 64; o *= 2) {
            const unsigned x = __shfl_up(sum, o, 64);
            if (lane >= o) sum += x;
        }
        if (threadIdx.x < DIGITS && lane == 63) s.scan[wave] = sum;
        __syncthreads();
        if (threadIdx.x < DIGITS) {
            unsigned below = 0;
            for (int w = 0; w < wave; ++w) below += s.scan[w];
            s.base[threadIdx.x] = below + sum - all;
        }
        __syncthreads();
        place_keys(s, digit, here, place);
#pragma unroll
        for (int i = 0; i < SHORT_ITEMS; ++i)
            if (64 * i + lane < here) {
                keys[place[i]] = key[i];
                ats[place[i]] = at[i];
            }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < SHORT_ITEMS; ++i) {
            const int n = w0 + 64 * i + lane;
            key[i] = n < a.N ? keys[n] : 0;
            at[i] = n < a.N ? ats[n] : 0;
        }
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < SHORT_ITEMS; ++i) {
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
    const int left = D - f, i0 = c * a.chunk, i1 = min(i0 + a.chunk, a.N);
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
    for (int i = i0; i < i1; i += 8) {
        u4v k[2], n[2];
        k[0] = *(const u4v*)(a.keys + i);
        k[1] = *(const u4v*)(a.keys + i + 4);
        n[0] = *(const u4v*)(a.at + i);
        n[1] = *(const u4v*)(a.at + i + 4);
        if (k[0][0] >= V) break;                // only unused positions are left
        float x[8][RUN];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const bool on = i + u < i1 && k[u >> 2][u & 3] < V;
            const unsigned at = on ? n[u >> 2][u & 3] : 0;
            const TO* g = (const TO*)a.grad + (long long)(at / (unsigned)p.L) * p.grad.batch +
                          (long long)(at % (unsigned)p.L) * p.grad.row + f;
            load_run(g, on ? left : 0, x[u]);
        }
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
#pragma unroll
            for (int e = 0; e < RUN; ++e) acc[e] += x[u][e];
        }
    }
    if (any) flush(i1 >= a.N || a.keys[i1] != run);
}

// Joins the parts of each run that begins in chunk c and ends in a later one: the waves of a
// workgroup take them in turn, four at a time, and their sums meet in order.
template <class TW>
__global__ void __launch_bounds__(256) join_runs_kernel(TableArgs a) {
    __shared__ float part[4][SLAB];
    const int D = a.p.D, c = blockIdx.x / a.slabs, f0 = blockIdx.x % a.slabs * SLAB;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int i0 = c * a.chunk, i1 = i0 + a.chunk;
    if (i1 >= a.N) return;
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
    const int f = f0 + lane * RUN, left = D - f;
    float acc[RUN] = {};
    if (wave == 0) load_run(a.tail + (long long)c * D + f, left, acc);
    int k = c + 1 + wave;
    for (; k + 12 <= last; k += 16) {
        float x[4][RUN];
#pragma unroll
        for (int u = 0; u < 4; ++u) load_run(a.head + (long long)(k + 4 * u) * D + f, left, x[u]);
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int e = 0; e < RUN; ++e) acc[e] += x[u][e];
    }
    for (; k <= last; k += 4) {
        float x[RUN];
        load_run(a.head + (long long)k * D + f, left, x);
#pragma unroll
        for (int e = 0; e < RUN; ++e) acc[e] += x[e];
    }
#pragma unroll
    for (int e = 0; e < RUN; ++e) part[wave][64 * e + lane] = acc[e];
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int e = 0; e < RUN; ++e) {
        float s = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w) s += part[w][64 * e + lane];
        acc[e] = s * a.p.scale;
    }
    store_run((TW*)a.dweight + (long long)run * D + f, left, acc);
}

namespace {

int check(const d2p_token_embedding_params* p) {
    D2P_REQUIRE(p != nullptr, "null parameters");
    D2P_REQUIRE(known_pair(p->weight_dtype, p->dtype),
                "unknown element types, or a pair other than equal ones and 16 bits beside float32");
    D2P_REQUIRE(p->B >= 0 && p->L >= 0 && p->V >= 0, "negative size");
    D2P_REQUIRE((long long)p->B * p->L < 1LL << 31, "too many tokens");
    D2P_REQUIRE(p->V < 0x7fffffff, "too many rows");
    D2P_REQUIRE(p->D >= 1 && p->D <= 1 << 20, "features must be between 1 and 2^20");
    D2P_REQUIRE(p->token_bytes == 4 || p->token_bytes == 8, "tokens must have 4 or 8 bytes");
    D2P_REQUIRE(p->padding >= -1 && p->padding < std::max(p->V, 1), "padding must be a token, or -1");
    D2P_REQUIRE(p->scale > -__builtin_inff() && p->scale < __builtin_inff(), "scale must be finite");
    return D2P_OK;
}

size_t round16(size_t n) { return (n + 15) & ~(size_t)15; }

// How the backward pass splits its work, and its workspace.
struct Plan {
    int N, bits, passes, tile, tiles;
    bool short_sort;
    int lanes, slabs, chunk, chunks;
    size_t keys, counts, present, parts, total;

    explicit Plan(const d2p_token_embedding_params& p) {
        N = p.B * p.L;
        bits = 1;
        while (bits < 31 && (p.V >> bits) != 0) ++bits;     // of V, which stands for no token
        passes = (bits + 7) / 8;
        short_sort = N <= SHORT && p.V <= 1 << 20;
        const int part = 2 * SORT_THREADS;
        tiles = std::max(1, std::min(MOST_TILES, cdiv(N, part)));
        tile = std::max(1, cdiv(cdiv(N, tiles), part)) * part;
        tiles = std::max(1, cdiv(N, tile));
        lanes = std::min(team_of(p.D), 64);
        slabs = cdiv(p.D, SLAB);
        // chunks of 64 positions where they give the card's waves work, shorter ones where
        // positions are few, longer ones where the joins of long runs would be
        const long long waves = (long long)N * slabs * lanes / 64;
        chunk = 8;
        while (chunk < 256 && waves / chunk > 4096) chunk *= 2;
        chunks = cdiv(N, chunk);
        keys = round16(((size_t)N + 8) * 4);
        counts = (size_t)tiles * DIGITS * 4;
        present = round16(p.V);
        parts = round16((size_t)chunks * p.D * 4);
        total = 4 * keys + counts + present + 2 * parts;
    }
};

int launch_sort(const d2p_token_embedding_params& p, const Plan& plan, char* ws, TableArgs& t,
                hipStream_t st) {
    unsigned* key[2] = {(unsigned*)ws, (unsigned*)(ws + plan.keys)};
    unsigned* at[2] = {(unsigned*)(ws + 2 * plan.keys), (unsigned*)(ws + 3 * plan.keys)};
    SortArgs a{};
    a.p = p;
    a.N = plan.N;
    a.tiles = plan.tiles;
    a.tile = plan.tile;
    a.first = a.last = 1;
    a.keys_to = key[0];
    a.at_to = at[0];
    a.counts = (unsigned*)(ws + 4 * plan.keys);
    a.present = (unsigned char*)(ws + 4 * plan.keys + plan.counts);
    t.present = a.present;
    t.keys = key[0];
    t.at = at[0];
    if (plan.short_sort) {
        D2P_LAUNCH("token_sort", sort_short_kernel, dim3(1), dim3(SORT_THREADS), 0, st, a, plan.bits);
        D2P_HIP(hipGetLastError());
        return D2P_OK;
    }
    const int clearing = (int)std::min<long long>(256, p.V / (64 << 10) + 1);
    for (int n = 0; n < plan.passes; ++n) {
        a.first = n == 0;
        a.last = n == plan.passes - 1;
        a.shift = 8 * n;
        a.keys = key[(n + 1) & 1];
        a.at = at[(n + 1) & 1];
        a.keys_to = key[n & 1];
        a.at_to = at[n & 1];
        D2P_LAUNCH("token_sort_count", count_digits_kernel,
                   dim3(std::max(plan.tiles, a.first ? clearing : 1)), dim3(SORT_THREADS), 0, st, a);
        D2P_HIP(hipGetLastError());
        D2P_LAUNCH("token_sort_move", move_keys_kernel<2>, dim3(plan.tiles), dim3(SORT_THREADS), 0,
                   st, a);
        D2P_HIP(hipGetLastError());
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
    D2P_REQUIRE(p->tokens && out && (weight || p->V == 0), "null pointer argument");
    EmbedArgs a{*p, weight, out, std::min(team_of(p->D), 64)};
    const int most = 8 * std::max(device_cus(), 1);
    const int grid = std::min(cdiv(p->B * p->L, 256 / a.lanes), most);
    return with_pair(p->weight_dtype, p->dtype, [&](auto tw, auto to) {
        using TW = typename decltype(tw)::type;
        using TO = typename decltype(to)::type;
        D2P_LAUNCH("token_embedding", (token_embedding_kernel<TW, TO>), dim3(grid), dim3(256), 0,
                   (hipStream_t)stream, a);
        D2P_HIP(hipGetLastError());
        return D2P_OK;
    });
}

extern "C" size_t d2p_token_embedding_backward_workspace_bytes(const d2p_token_embedding_params* p) {
    if (!p || p->B < 0 || p->L < 0 || p->V < 0 || p->D < 1 || p->D > 1 << 20 ||
        p->V >= 0x7fffffff || (long long)p->B * p->L >= 1LL << 31)
        return 0;
    return Plan(*p).total;
}

extern "C" int d2p_token_embedding_backward(const d2p_token_embedding_params* p, const void* grad,
                                            void* dweight, void* workspace, size_t workspace_bytes,
                                            void* stream) {
    D2P_TRY(check(p));
    if (p->V == 0) return D2P_OK;
    const bool rows = (long long)p->B * p->L > 0;
    D2P_REQUIRE(dweight && (!rows || (p->tokens && grad)), "null pointer argument");
    const Plan plan(*p);
    D2P_REQUIRE(workspace && workspace_bytes >= plan.total, "workspace too small");
    D2P_REQUIRE(((uintptr_t)workspace & 15) == 0, "the workspace must be aligned to 16 bytes");
    hipStream_t st = (hipStream_t)stream;
    TableArgs a{};
    a.p = *p;
    a.grad = grad;
    a.dweight = dweight;
    a.N = plan.N;
    a.lanes = plan.lanes;
    a.slabs = plan.slabs;
    a.chunk = plan.chunk;
    a.chunks = plan.chunks;
    char* ws = (char*)workspace;
    a.head = (float*)(ws + plan.total - 2 * plan.parts);
    a.tail = (float*)(ws + plan.total - plan.parts);
    const int teams = 256 / plan.lanes;
    D2P_REQUIRE((long long)plan.chunks * plan.slabs < 1LL << 30, "too many tokens and features");
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
