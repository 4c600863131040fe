// attention_forward.hip.h -- softmax attention, one pass over the keys.
//
// Scores are formed transposed, S^T = K Q^T, so that a lane holds one query and 16 keys of
// each 32: its softmax is lane-local but for one exchange of the two half waves, and P^T
// is the second operand of O^T = V^T P^T as it stands (encoder.hip.h).
#pragma once
#include "encoder.hip.h"

namespace d2p_amd {
namespace enc {

struct ForwardArgs {
    d2p_attention_params p;
    const void *q, *k, *v;
    void* out;
    float* stats;
};

// The scores of one 32 x 32 tile, lane = query, accumulators = keys j0 + 8 g + 4 h + r: in
// units of log2, with the bias, -inf where the key is at or past `limit`.  at: the query's
// place among the keys; far: 0, or the bias of the whole tile is that of one clipped
// distance (-1, 1: see bias_reach).
template <bool BIAS, bool FULL>
__device__ __forceinline__ void score_tile(f16v s, float c, const float* bias, int R, int far,
                                           int j0, int at, int limit, int lane, float* x) {
    const int j = j0 + 4 * (lane >> 5);
    float b = 0.0f;
    if (BIAS && far) b = bias[far < 0 ? 0 : 2 * R];
#pragma unroll
    for (int v = 0; v < 16; ++v) {
        const int n = 8 * (v >> 2) + (v & 3);
        float y = s[v] * c;
        if (BIAS) {
            if (far == 0) b = bias[min(max(j + n - at, -R), R) + R];
            y += b;
        }
        x[v] = FULL || j + n < limit ? y : -__builtin_inff();
    }
}

// Whether every pair of queries placed at0 .. at0 + 31 and keys j0 .. j1 lies at or past
// the clipping distance behind (-1) or ahead (1); 0: neither.
__device__ __forceinline__ int bias_reach(int j0, int j1, int at0, int R) {
    return j1 - at0 <= -R ? -1 : j0 - (at0 + 31) >= R ? 1 : 0;
}

// A workgroup takes 128 queries of one head, 32 a wave, and passes over the keys 64 at a
// time: K and V tiles through registers to LDS, one tile ahead.
template <class T, int DP, bool BIAS, bool DROP>
__global__ void __launch_bounds__(256) attention_forward_kernel(ForwardArgs a) {
    using TL = Tile<T, DP>;
    constexpr int BK = 64, DT = DP / 32;
    extern __shared__ __align__(16) u4v sm[];
    u4v* Ks = sm;
    u4v* Vs = Ks + TL::bytes(BK) / 16;
    float* bias = (float*)(Vs + TL::bytes(BK) / 16);
    const d2p_attention_params& p = a.p;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, h = lane >> 5;
    const int nb = (p.Lq + 127) / 128;
    const unsigned w = near_xcd(blockIdx.x, gridDim.x);
    const int bh = w / nb, b = bh / p.Hq, hq = bh % p.Hq;
    // causal: the blocks with the most keys first
    const int q0 = (p.causal ? nb - 1 - (int)(w % nb) : (int)(w % nb)) * 128;
    const Span e(p, b);
    const int D = p.D, wq = q0 + 32 * wave, i = wq + (lane & 31), at = i + e.off;
    const Rows qr = head_rows<T>(a.q, p.q, b, hq, e.nq, D);
    const Rows kr = head_rows<T>(a.k, p.k, b, hq / (p.Hq / p.Hkv), e.nk, D);
    const Rows vr = head_rows<T>(a.v, p.v, b, hq / (p.Hq / p.Hkv), e.nk, D);
    if (BIAS) load_bias<T>(bias, p, hq, tid, 256);

    u4v qf[TL::STEPS];
    {
        const __amdgpu_buffer_rsrc_t r = qr.from(q0);
#pragma unroll
        for (int s = 0; s < TL::STEPS; ++s)
            qf[s] = __builtin_amdgcn_raw_buffer_load_b128(r, qr.at(i - q0, 2 * s + h), 0, 0);
    }
    const float c = p.scale * LOG2E;
    const Drop drop(p, bh);
    f16v o[DT] = {};
    float m = -__builtin_inff(), l = 0.0f;
    // keys that the block's, the wave's first and the lane's query see
    const int end = q0 < e.nq ? e.limit(p, min(q0 + 127, e.nq - 1)) : 0;
    const int wave_full = e.limit(p, wq);
    const int limit = e.limit(p, i);

    Stage<T, DP, BK, 256> ks, vs;
    if (end > 0) {
        ks.load(kr, 0, tid);
        vs.load(vr, 0, tid);
    }
    for (int j0 = 0; j0 < end; j0 += BK) {
        __syncthreads();
        ks.store(Ks, tid);
        vs.store(Vs, tid);
        __syncthreads();
        if (j0 + BK < end) {
            ks.load(kr, j0 + BK, tid);
            vs.load(vr, j0 + BK, tid);
        }
        float x[32];
        const int far = BIAS ? bias_reach(j0, j0 + BK - 1, wq + e.off, p.max_distance) : 0;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            f16v s = {};
#pragma unroll
            for (int n = 0; n < TL::STEPS; ++n)
                s = Elem<T>::mma(TL::frag(Ks, 32 * t, n, lane), qf[n], s);
            if (j0 + BK <= wave_full)
                score_tile<BIAS, true>(s, c, bias, p.max_distance, far, j0 + 32 * t, at, limit,
                                       lane, x + 16 * t);
            else
                score_tile<BIAS, false>(s, c, bias, p.max_distance, far, j0 + 32 * t, at, limit,
                                        lane, x + 16 * t);
        }
        float top = x[0];
#pragma unroll
        for (int v = 1; v < 32; ++v) top = fmaxf(top, x[v]);
        top = fmaxf(m, both_max(top));
        const float ref = (top == -__builtin_inff() ? 0.0f : top) - FORWARD_SHIFT<T>;
        const float old = exp2_(m - (FORWARD_SHIFT<T> + ref));   // nothing seen yet: 0
        m = top;
        l *= old;
#pragma unroll
        for (int d = 0; d < DT; ++d) o[d] *= old;
#pragma unroll
        for (int v = 0; v < 32; ++v) {
            x[v] = exp2_(x[v] - ref);
            l += x[v];
        }
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            if (DROP) {
                const u4v kw = drop.by_query(wq, j0 + 32 * t, lane);
#pragma unroll
                for (int v = 0; v < 16; ++v)
                    x[16 * t + v] = drop.keeps(kw, v) ? x[16 * t + v] : 0.0f;
            }
#pragma unroll
            for (int f = 0; f < TL::FRAGS; ++f) {
                // P in the type of V: its rounding is that of one factor of each product
                const u4v pf = Elem<T>::pack(x + 16 * t + TL::PER * f);
#pragma unroll
                for (int d = 0; d < DT; ++d)
                    o[d] = Elem<T>::mma(TL::frag_t(Vs, 32 * t, 32 * d, f, lane), pf, o[d]);
            }
        }
    }

    l = both_sum(l);
    if (i >= p.Lq) return;
    const float nan = __builtin_nanf("");
    float f = l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : nan);
    if (DROP) f *= drop.scale;
    if (i >= e.nq) f = 0.0f;
    if (e.bad) f = nan;
    const bool none = i >= e.nq || !(l != 0.0f);   // no key: zeros, whatever the accumulators hold
    char* row = (char*)a.out + (((long long)b * p.Lq + i) * p.Hq + hq) * D * (long long)sizeof(T);
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int d0 = 32 * d + 8 * g + 4 * h;
            float y[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) y[r] = none ? (e.bad ? nan : 0.0f) : o[d][4 * g + r] * f;
            if (d0 < D) Elem<T>::store4(row + d0 * (int)sizeof(T), y);
        }
    if (h == 0) {
        const long long n = (long long)p.B * p.Hq * p.Lq, at_row = (long long)bh * p.Lq + i;
        a.stats[at_row] = e.bad ? nan : none ? -__builtin_inff() : m;
        a.stats[n + at_row] = none ? 0.0f : log2_(l) - FORWARD_SHIFT<T>;
    }
}

template <class T, int DP, bool BIAS, bool DROP>
int launch_forward_as(const ForwardArgs& a, hipStream_t st) {
    auto kernel = attention_forward_kernel<T, DP, BIAS, DROP>;
    const int lds = 2 * Tile<T, DP>::bytes(64) + (BIAS ? (2 * a.p.max_distance + 1) * 4 : 0);
    D2P_HIP(hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize,
                                lds));
    const long long n = (long long)a.p.B * a.p.Hq * cdiv(a.p.Lq, 128);
    D2P_REQUIRE(n <= 0x7fffffffLL, "too many query blocks");
    if (n == 0) return D2P_OK;
    D2P_LAUNCH("attention_forward", kernel, dim3((unsigned)n), dim3(256), lds, st, a);
    D2P_HIP(hipGetLastError());
    return D2P_OK;
}

template <class T, int DP> int launch_forward_dp(const ForwardArgs& a, hipStream_t st) {
    if (a.p.bias)
        return a.p.drop ? launch_forward_as<T, DP, true, true>(a, st)
                        : launch_forward_as<T, DP, true, false>(a, st);
    return a.p.drop ? launch_forward_as<T, DP, false, true>(a, st)
                    : launch_forward_as<T, DP, false, false>(a, st);
}

template <class T> int launch_forward(const ForwardArgs& a, hipStream_t st) {
    switch (padded(a.p.D)) {
        case 32: return launch_forward_dp<T, 32>(a, st);
        case 64: return launch_forward_dp<T, 64>(a, st);
        default: return launch_forward_dp<T, 128>(a, st);
    }
}

int launch_forward_f32(const ForwardArgs& a, hipStream_t st);
int launch_forward_f16(const ForwardArgs& a, hipStream_t st);
int launch_forward_bf16(const ForwardArgs& a, hipStream_t st);

}  // namespace enc
}  // namespace d2p_amd
