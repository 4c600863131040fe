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

// x = the first `left` of eight numbers from p on (left may be zero or less, or past eight),
// zeros behind them
template <class T> __device__ __forceinline__ void load_run(const T* p, int left, float* x) {
    if (left >= RUN) {
        const Eight<T> a = *(const Eight<T>*)p;
#pragma unroll
        for (int e = 0; e < RUN; ++e) x[e] = (float)a.v[e];
    } else {
#pragma unroll
        for (int e = 0; e < RUN; ++e) x[e] = e < left ? (float)p[e] : 0.0f;
    }
}
template <class T> __device__ __forceinline__ void store_run(T* p, int left, const float* x) {
    if (left >= RUN) {
        Eight<T> a;
#pragma unroll
        for (int e = 0; e < RUN; ++e) a.v[e] = (T)x[e];
        *(Eight<T>*)p = a;
    } else {
#pragma unroll
        for (int e = 0; e < RUN; ++e)
            if (e < left) p[e] = (T)x[e];
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
    // Mean and the sum of squares around it of D numbers, x[e] being there for e < left: in two
    // passes over the registers, each wave around a mean of its own.
    __device__ __forceinline__ float2 spread(const float* x, int left, int D) {
        float s = 0.0f, m2 = 0.0f;
#pragma unroll
        for (int e = 0; e < RUN; ++e) s += x[e];
        const int members = WIDE ? 64 : lanes;
        const int count = WIDE ? min(max(D - (n & ~63) * RUN, 0), 64 * RUN) : D;
        s = group_sum(s, members);
        const float mean = s / max(count, 1);
#pragma unroll
        for (int e = 0; e < RUN; ++e) {
            const float c = e < left ? x[e] - mean : 0.0f;
            m2 += c * c;
        }
        m2 = group_sum(m2, members);
        if (!WIDE) return {mean, m2};
        // the waves' own: around the common mean a wave adds count (mean - common)^2
        float2* at = put(s, m2);
        const int waves = lanes >> 6;
        float total = 0.0f, squares = 0.0f;
        for (int w = 0; w < waves; ++w) total += at[w].x;
        const float common = total / D;
        for (int w = 0; w < waves; ++w) {
            const int c = min(max(D - w * 64 * RUN, 0), 64 * RUN);
            const float d = c ? at[w].x / c - common : 0.0f;
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

    void init(int D_) {
        D = D_;
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
