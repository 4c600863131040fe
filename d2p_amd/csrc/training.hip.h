// training.hip.h -- what the kernels around the attention layer share (token embedding, the
// residual stream's norms, gradient clipping): runs of eight numbers of any alignment, pairs
// of element types, sums over the team of lanes that holds a row.
#pragma once
#include "encoder.hip.h"
#include "../../include/d2p_amd_training.h"

namespace d2p_amd {
namespace enc {

constexpr int RUN = 8;   // numbers that a lane holds of a row

// Eight numbers wherever an element may lie: gfx950 takes 16-byte accesses at any address, so
// rows of odd sizes need no second kernel.
template <class T> struct Eight {
    T v[RUN];
};

// Eight numbers moved `by` (0 to 7) places to the front, zeros behind them: shifts by four, two
// and one.
template <class T> __device__ __forceinline__ Eight<T> to_front(const Eight<T>& a, int by) {
    constexpr int W = sizeof(Eight<T>) / 4, PER = RUN / W;      // words, numbers of one
    struct Words { unsigned v[W]; };
    Words w = bits<Words>(a);
#pragma unroll
    for (int step = 4; step >= PER; step /= 2) {
        const bool on = by & step;
#pragma unroll
        for (int i = 0; i < W; ++i) {
            const unsigned next = i + step / PER < W ? w.v[i + step / PER] : 0;
            w.v[i] = on ? next : w.v[i];
        }
    }
    if constexpr (PER == 2) {
        const int half = by & 1 ? 16 : 0;
#pragma unroll
        for (int i = 0; i < W; ++i)
            w.v[i] = __builtin_amdgcn_alignbit(i + 1 < W ? w.v[i + 1] : 0, w.v[i], half);
    }
    return bits<Eight<T>>(w);
}

// The eight numbers of a row of D (eight at least) from `at` on, in two steps, so that all loads
// of a turn are under way before the first is waited for: load_run reads eight numbers of the
// row whatever `at` is, at the row's end the last eight, which unpack then moves into place.
// (A branch around each load, and its conversion behind it, made the loads wait for each other.)
//
// PAST: past the caches, for what is read once (a table's gradient from bf16 [16, 8192, 1024]: its
// kernel 102 -> 82 us).  Of 16-bit numbers only: float32 takes two loads a lane, each of half of
// what the wave reads of a line, which then comes twice (a norm's backward pass over 1.6 GB: 421 us,
// 441 past the caches).
typedef u4v u4v_any __attribute__((aligned(2)));
template <bool PAST = false, class T>
__device__ __forceinline__ Eight<T> load_run(const T* row, int at, int D) {
    const T* p = row + min(at, D - RUN);
    if constexpr (PAST && sizeof(T) == 2)
        return bits<Eight<T>>(__builtin_nontemporal_load((const u4v_any*)p));
    return *(const Eight<T>*)p;
}
// x = the numbers; zeros behind the row's end, and where the row is not wanted.  EVEN: D is known to
// be a multiple of eight.
template <bool EVEN = false, class T>
__device__ __forceinline__ void unpack(const Eight<T>& a, int at, int D, bool wanted, float* x) {
    Eight<T> b = a;
    if (!EVEN && D % RUN) b = to_front(a, min(max(at - (D - RUN), 0), RUN - 1));
    const bool on = wanted && at < D;
#pragma unroll
    for (int e = 0; e < RUN; ++e) x[e] = on ? (float)b.v[e] : 0.0f;
}

template <class T, int N> struct Few {
    T v[N];
};
template <bool PAST = false, class T>
__device__ __forceinline__ void store_run(T* p, int left, const float* x) {
    Eight<T> a;
#pragma unroll
    for (int e = 0; e < RUN; ++e) a.v[e] = (T)x[e];
    if (left >= RUN) {
        if constexpr (PAST && sizeof(T) == 2)
            __builtin_nontemporal_store(bits<u4v>(a), (u4v_any*)p);
        else
            *(Eight<T>*)p = a;
    } else if (left > 0) {      // four, two and one
        const bool four = left & 4, two = left & 2;
        if (four) *(Few<T, 4>*)p = {a.v[0], a.v[1], a.v[2], a.v[3]};
        if (two)
            *(Few<T, 2>*)(p + (left & 4)) = {four ? a.v[4] : a.v[0], four ? a.v[5] : a.v[1]};
        if (left & 1)
            p[left & 6] = four ? (two ? a.v[6] : a.v[4]) : (two ? a.v[2] : a.v[0]);
    }
}
// one number whose type is known only at run time
__device__ __forceinline__ float load_as(const void* p, int dtype, long long at) {
    return dtype == D2P_FLOAT32 ? ((const float*)p)[at]
           : dtype == D2P_FLOAT16 ? (float)((const _Float16*)p)[at] : (float)((const __bf16*)p)[at];
}
__device__ __forceinline__ void store_as(void* p, int dtype, long long at, float x) {
    if (dtype == D2P_FLOAT32) ((float*)p)[at] = x;
    else if (dtype == D2P_FLOAT16) ((_Float16*)p)[at] = (_Float16)x;
    else ((__bf16*)p)[at] = (__bf16)x;
}

inline bool known_type(int dtype) {
    return dtype == D2P_FLOAT32 || dtype == D2P_FLOAT16 || dtype == D2P_BFLOAT16;
}
// A wide type and a narrow one: the same, or 16 bits beside float32.
inline bool known_pair(int wide, int narrow) {
    return known_type(wide) && known_type(narrow) && (wide == narrow || wide == D2P_FLOAT32);
}
template <class T> struct Type {
    using type = T;
};
// f(Type<wide>, Type<narrow>) for a known pair
template <class F> int with_pair(int wide, int narrow, F f) {
    if (wide == D2P_FLOAT16) return f(Type<_Float16>{}, Type<_Float16>{});
    if (wide == D2P_BFLOAT16) return f(Type<__bf16>{}, Type<__bf16>{});
    if (narrow == D2P_FLOAT16) return f(Type<float>{}, Type<_Float16>{});
    if (narrow == D2P_BFLOAT16) return f(Type<float>{}, Type<__bf16>{});
    return f(Type<float>{}, Type<float>{});
}

// Lanes that share a row of D numbers, eight each: a power of two.
inline int team_of(int D) {
    int n = 1;
    while (n * RUN < D) n *= 2;
    return n;
}

// s / n, n a whole number below 2^24: the product with 1 / n and what it leaves, which gives
// exact quotients exactly (a mean of equal numbers is that number).  An infinite s leaves nothing
// (infinity less infinity): it is infinite, so that a row whose squares overflow is normed to zeros.
__device__ __forceinline__ float divided(float s, float n) {
    const float per = __builtin_amdgcn_rcpf(n), q = s * per, left = fmaf(-q, n, s);
    return __builtin_isinf(s) ? q : fmaf(left, per, q);
}
// 1 / sqrt(x) within two roundings, where x is below the normal numbers too
__device__ __forceinline__ float inverse_root(float x) {
    const bool tiny = x < 0x1p-96f;
    return __builtin_amdgcn_rsqf(tiny ? x * 0x1p96f : x) * (tiny ? 0x1p48f : 1.0f);
}

// n / d for n below 2^31, by a product (T. Granlund and P. Montgomery, "Division by invariant
// integers using multiplication", PLDI 1994).
struct Divisor {
    unsigned d, magic, shift;
    Divisor() = default;
    explicit Divisor(int d_) : d(d_ > 0 ? d_ : 1), magic(0), shift(0) {
        while ((1ULL << shift) < d) ++shift;
        magic = (unsigned)((((1ULL << shift) - d) << 32) / d + 1);
    }
    __device__ __forceinline__ unsigned operator()(unsigned n) const {
        return (__umulhi(n, magic) + n) >> shift;
    }
};

// The threads that hold one row.  Up to 64 lanes of one wave, or (WIDE) whole waves, which
// exchange their sums through LDS: two sets of them in turn, so that one barrier a sum does.
template <bool WIDE> struct Team {
    int lanes, n;               // threads of a team, and this one's place among them
    float2* slots;              // WIDE: [2][16]
    int turn = 0;

    __device__ __forceinline__ Team(int lanes_, float2* slots_)
        : lanes(lanes_), n(threadIdx.x & (lanes_ - 1)), slots(slots_) {}

    // sums of a and b over the team
    __device__ __forceinline__ float2 sum(float a, float b) {
        if (!WIDE) return {group_sum(a, lanes), group_sum(b, lanes)};
        return exchange(group_sum(a, 64), group_sum(b, 64));
    }
    __device__ __forceinline__ float sum(float a) {
        return WIDE ? exchange(group_sum(a, 64), 0.0f).x : group_sum(a, lanes);
    }
    // Mean and the sum of squares around it of D numbers, `there` being 1 for the lane's numbers
    // and 0 (x too) behind the row's end: in two passes over the registers, each wave around a
    // mean of its own.
    __device__ __forceinline__ float2 spread(const float* x, const float* there, int D) {
        float s = 0.0f, m2 = 0.0f;
#pragma unroll
        for (int e = 0; e < RUN; ++e) s += x[e];
        const int members = WIDE ? 64 : lanes;
        const int count = WIDE ? min(max(D - (n & ~63) * RUN, 0), 64 * RUN) : D;
        s = group_sum(s, members);
        const float mean = divided(s, (float)max(count, 1));
#pragma unroll
        for (int e = 0; e < RUN; ++e) {
            const float c = fmaf(-mean, there[e], x[e]);
            m2 += c * c;
        }
        m2 = group_sum(m2, members);
        if (!WIDE) return {mean, m2};
        // the waves' own: around the common mean a wave adds count (mean - common)^2
        float2* at = put(s, m2);
        const int waves = lanes >> 6;
        float total = 0.0f, squares = 0.0f;
        for (int w = 0; w < waves; ++w) total += at[w].x;
        const float common = divided(total, (float)D);
        for (int w = 0; w < waves; ++w) {
            const int c = min(max(D - w * 64 * RUN, 0), 64 * RUN);
            const float d = c ? divided(at[w].x, (float)c) - common : 0.0f;
            squares += at[w].y + c * d * d;
        }
        return {common, squares};
    }

   private:
    // the team's waves' numbers, in order
    __device__ __forceinline__ float2* put(float a, float b) {
        const int wave = threadIdx.x >> 6;
        float2* set = slots + 16 * turn;
        turn ^= 1;
        if ((threadIdx.x & 63) == 0) set[wave] = {a, b};
        __syncthreads();
        return set + (wave & ~((lanes >> 6) - 1));
    }
    __device__ __forceinline__ float2 exchange(float a, float b) {
        const float2* at = put(a, b);
        const int waves = lanes >> 6;
        float2 s = at[0];
        for (int w = 1; w < waves; ++w) {
            s.x += at[w].x;
            s.y += at[w].y;
        }
        return s;
    }
};

// Sums of `count` rows of D numbers in float32, as one entry point's last step: `groups` results of
// D numbers, group g's rows from src + g count D on.
struct SumJob {
    const float* src;
    void* dst;
    int dtype, count, groups, first;   // first: the job's first workgroup
};
struct SumJobs {
    SumJob job[6];
    int jobs, D, tiles;                // tiles of 64 numbers
    int blocks;
    float scale;                       // of all results

    void init(int D_) {
        D = D_;
        scale = 1.0f;
        tiles = cdiv(D_, 64);
        jobs = blocks = 0;
    }
    void add(const float* src, void* dst, int dtype, int count, int groups) {
        if (!dst) return;
        job[jobs++] = {src, dst, dtype, count, groups, blocks};
        blocks += groups * tiles;
    }
};

// rows.hip
int launch_sum_rows(const char* name, const SumJobs& a, hipStream_t st);

}  // namespace enc
}  // namespace d2p_amd
