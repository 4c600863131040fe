// attention_forward.hip.h -- softmax attention, one pass over the keys.
//
// Scores are formed transposed, S^T = K Q^T, so that a lane holds one query and 16 keys of
// each 32: its softmax is lane-local but for one exchange of the two half waves, and P^T
// is the second operand of O^T = V^T P^T as it stands (encoder.hip.h).
//
// Bound, for 64 keys and 32 queries of 128 features of 16 bits: 32 MFMAs of 32 cycles against
// 32 exponentials (16 cycles a wave) and about 150 other vector operations (4 cycles) a lane,
// 1000 to 1100 cycles each on a SIMD, and 32 KiB of LDS reads for the wave, which four SIMDs'
// matrix cores would take in those 1000 cycles too.  Two waves a SIMD, one's exponentials
// beside the other's products; accumulators in architectural registers (256 a wave), where
// the vector units read them without a copy.
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

// Whether every pair of queries placed at0 .. at0 + 31 and keys j0 .. j1 lies at or past
// the clipping distance behind (-1) or ahead (1); 0: neither.
__device__ __forceinline__ int bias_reach(int j0, int j1, int at0, int R) {
    return j1 - at0 <= -R ? -1 : j0 - (at0 + 31) >= R ? 1 : 0;
}

// s c + bias, in units of log2, of 16 accumulators: distance d + SIGN (8 g + r) for v = 4 g + r
template <int SIGN>
__device__ __forceinline__ void add_bias_at(f16v& s, float c, const float* bias, int R, int d) {
#pragma unroll
    for (int v = 0; v < 16; ++v) {
        const int n = d + SIGN * (8 * (v >> 2) + (v & 3));
        s[v] = fmaf(s[v], c, bias[min(max(n, -R), R) + R]);
    }
}
// a tile whose distances are all within the table: no clipping
template <int SIGN>
__device__ __forceinline__ void add_bias_inside(f16v& s, float c, const float* bias, int R, int d) {
    const float* b = bias + R + d;
#pragma unroll
    for (int v = 0; v < 16; ++v) s[v] = fmaf(s[v], c, b[SIGN * (8 * (v >> 2) + (v & 3))]);
}
template <int SIGN>
__device__ __forceinline__ void add_bias_to(f16v& s, float c, const float* bias, int R, int j0,
                                            int at0, int d) {
    const int far = bias_reach(j0, j0 + 31, at0, R);
    if (far) {
        const float b = bias[far < 0 ? 0 : 2 * R];
#pragma unroll
        for (int v = 0; v < 16; ++v) s[v] = fmaf(s[v], c, b);
    } else if (j0 - (at0 + 31) >= -R && j0 + 31 - at0 <= R) {
        add_bias_inside<SIGN>(s, c, bias, R, d);
    } else {
        add_bias_at<SIGN>(s, c, bias, R, d);
    }
}
// lane = query placed at, accumulators = keys from j0; at0: the tile's first query
__device__ __forceinline__ void add_bias(f16v& s, float c, const float* bias, int R, int j0,
                                         int at0, int at, int lane) {
    add_bias_to<1>(s, c, bias, R, j0, at0, j0 + 4 * (lane >> 5) - at);
}
// lane = key j0 + l % 32, accumulators = queries placed from at0 on
__device__ __forceinline__ void add_bias_by_key(f16v& s, float c, const float* bias, int R,
                                                int j0, int at0, int lane) {
    add_bias_to<-1>(s, c, bias, R, j0, at0, j0 + (lane & 31) - at0 - 4 * (lane >> 5));
}

// Shared by the waves of a workgroup: K and V tiles of 64 keys, two of each, which go to
// LDS without passing through registers while the tiles before them are worked on.
//
// A wave takes 32 queries.  In one turn of its loop the matrix cores form the
// next tile's scores while its vector units take the exponentials of this one, and P V of
// each half of the keys while they take those of the other half and the next maximum.  The
// accumulators are scaled to a new maximum only when it has grown by more than 2^8 (a
// branch that is soon rare); until then the old one is a reference as good.
template <class T, int DP, int NW, bool BIAS, bool DROP> struct Forward {
    using TL = Tile<T, DP>;
    using E = Elem<T>;
    static constexpr int BK = 64, DT = DP / 32, TILE = TL::bytes(BK) / 16;
    static constexpr int LDS = 4 * TL::bytes(BK);   // and the bias's table

    const ForwardArgs& a;
    const d2p_attention_params& p;
    const u4v* Ks;
    const u4v* Vs;
    const float* bias;
    const Drop drop;
    int lane, h, wq, at0;
    int at, limit;
    u4v qf[TL::STEPS];
    f16v o[DT] = {};
    float m = -__builtin_inff(), ref = 0.0f, l = 0.0f;
    float c;

    __device__ __forceinline__ Forward(const ForwardArgs& a_, const Span& e, const Rows& qr,
                                       const u4v* sm, const float* bias_, int bh, int wq_,
                                       int lane_)
        : a(a_), p(a_.p), Ks(sm), Vs(sm + 2 * TILE), bias(bias_), drop(a_.p, bh), lane(lane_),
          h(lane_ >> 5), wq(wq_), at0(wq_ + e.off) {
        c = p.scale * LOG2E;
        const __amdgpu_buffer_rsrc_t r = qr.from(wq);
        const int i = wq + (lane & 31);
        at = i + e.off;
        limit = e.limit(p, i);
#pragma unroll
        for (int s = 0; s < TL::STEPS; ++s)
            qf[s] = __builtin_amdgcn_raw_buffer_load_b128(r, qr.at(lane & 31, 2 * s + h), 0, 0);
    }

    __device__ __forceinline__ void scores(f16v (&s)[2], int buf, int ra) const {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            s[k] = f16v{};
#pragma unroll
            for (int n = 0; n < TL::STEPS; ++n)
                s[k] = E::mma(TL::frag(Ks + buf * TILE, 32 * k, n, ra), qf[n], s[k]);
        }
    }

    // Bias and mask of the tile from key j0 on, and its place against the reference.
    __device__ __forceinline__ void settle(f16v (&s)[2], int j0, bool full) {
        const int R = p.max_distance;
        const float inf = __builtin_inff();
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            if (BIAS) add_bias(s[k], c, bias, R, j0 + 32 * k, at0, at, lane);
            if (!full) {
                const int left = limit - (j0 + 32 * k + 4 * h);
#pragma unroll
                for (int v = 0; v < 16; ++v)
                    s[k][v] = 8 * (v >> 2) + (v & 3) < left ? s[k][v] : -inf;
            }
        }
        float top = s[0][0];
#pragma unroll
        for (int v = 1; v < 32; ++v) top = fmaxf(top, s[v >> 4][v & 15]);
        top = both_max(top) * (BIAS ? 1.0f : c);
        if (__any(top > m + 8.0f)) {
            const float to = fmaxf(m, top);
            const float f = to > m ? exp2_(m - to) : 1.0f;   // 0 from -inf
            m = to;
            // (without a bias the shift is part of it, rounded like the scores themselves)
            ref = to == -inf ? 0.0f : BIAS ? to : to - FORWARD_SHIFT<T>;
            l *= f;
#pragma unroll
            for (int d = 0; d < DT; ++d) o[d] *= f;
        }
    }

    // exponentials of half k of a tile: P, ready for the matrix cores
    __device__ __forceinline__ void weights(const f16v (&s)[2], int k, int j0,
                                            u4v (&pf)[TL::FRAGS]) {
        float x[16];
#pragma unroll
        for (int v = 0; v < 16; ++v) {
            x[v] = exp2_(BIAS ? shifted<T>(s[k][v] - ref) : fmaf(s[k][v], c, -ref));
            l += x[v];
        }
        u4v kw;
        if (DROP) kw = drop.by_query(wq, j0 + 32 * k, lane);
        if (DROP && sizeof(T) == 4) {
#pragma unroll
            for (int v = 0; v < 16; ++v) x[v] = drop.keeps(kw, v) ? x[v] : 0.0f;
        }
        // P in the type of V: its rounding is that of one factor of each product
#pragma unroll
        for (int f = 0; f < TL::FRAGS; ++f) {
            pf[f] = E::pack(x + TL::PER * f);
            if (DROP && sizeof(T) == 2) pf[f] = drop.keep16(pf[f], kw, f);
        }
    }

    __device__ __forceinline__ void values(const u4v (&pf)[TL::FRAGS], int k, int buf, int ca) {
#pragma unroll
        for (int f = 0; f < TL::FRAGS; ++f)
#pragma unroll
            for (int d = 0; d < DT; ++d)
                o[d] = E::mma(TL::frag_t(Vs + buf * TILE, 32 * k, 32 * d, f, ca), pf[f], o[d]);
    }

    __device__ __forceinline__ void store(const Span& e, int b, int hq, int bh) {
        const int D = p.D;
        const float nan = __builtin_nanf("");
        const int i = wq + (lane & 31);
        const float sum = both_sum(l);
        if (i >= p.Lq) return;
        // no key: zeros, whatever the accumulators hold
        const bool none = i >= e.nq || !(sum != 0.0f);
        const float f = (DROP ? drop.scale : 1.0f) / sum;
        char* row = (char*)a.out + (((long long)b * p.Lq + i) * p.Hq + hq) * D * (long long)sizeof(T);
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int d0 = 32 * d + 8 * g + 4 * h;
                float y[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) y[r] = e.bad ? nan : none ? 0.0f : o[d][4 * g + r] * f;
                if (d0 < D) E::store4(row + d0 * (int)sizeof(T), y);
            }
        if (h == 0) {
            const long long n = (long long)p.B * p.Hq * p.Lq, x = (long long)bh * p.Lq + i;
            a.stats[x] = e.bad ? nan : none ? -__builtin_inff() : m;
            a.stats[n + x] = none ? 0.0f : log2_(sum) - FORWARD_SHIFT<T>;
        }
    }
};

// Waves a SIMD that the registers are dealt for: the vector work of bias and dropout together
// gains by a third one at 64 features of 16 bits ([8, 2048, 8, 64] bfloat16 causal: 85 -> 75 us, two
// registers in scratch); dropout alone loses by it (nine in scratch, 65 -> 71 us).
template <class T, int DP, bool BIAS, bool DROP> constexpr int forward_waves() {
    return sizeof(T) * DP >= 512 ? 1 : sizeof(T) * DP == 128 && BIAS && DROP ? 3 : 2;
}

template <class T, int DP, int NW, bool BIAS, bool DROP>
__global__ void __launch_bounds__(64 * NW, (forward_waves<T, DP, BIAS, DROP>()))
attention_forward_kernel(ForwardArgs a) {
    using F = Forward<T, DP, NW, BIAS, DROP>;
    using TL = Tile<T, DP>;
    constexpr int BK = F::BK, ROWS = 32 * NW;
    extern __shared__ __align__(16) u4v sm[];
    u4v* Ks = sm;
    u4v* Vs = sm + 2 * F::TILE;
    float* bias = (float*)(sm + 4 * F::TILE);
    const d2p_attention_params& p = a.p;
    const int tid = threadIdx.x, lane = tid & 63, wave = wave_of(tid);
    const int nb = (p.Lq + ROWS - 1) / ROWS;
    int bh, block;
    place(blockIdx.x, p.B * p.Hq, nb, p.causal, &bh, &block);
    const int b = bh / p.Hq, hq = bh % p.Hq, hk = hq / (p.Hq / p.Hkv);
    const int q0 = (p.causal ? nb - 1 - block : block) * ROWS;   // the most keys first
    const Span e(p, b);
    const Rows qr = head_rows<T>(a.q, p.q, b, hq, e.nq, p.D);
    const Rows kr = head_rows<T>(a.k, p.k, b, hk, e.nk, p.D);
    const Rows vr = head_rows<T>(a.v, p.v, b, hk, e.nk, p.D);
    // keys that the block's last query sees, in tiles
    const int end = q0 < e.nq ? e.limit(p, min(q0 + ROWS, e.nq) - 1) : 0;
    const int tiles = (end + BK - 1) / BK;

    const int ra = TL::row_at(lane), ca = TL::col_at(lane);
    TileDma<T, DP, BK, NW> dk, dv;
    dk.init(kr, wave, lane);
    dv.init(vr, wave, lane);
    if (tiles > 0) dk.issue(kr, 0, Ks, wave);
    if (BIAS) load_bias<T>(bias, p, hq, tid, 64 * NW);
    F f(a, e, qr, sm, bias, bh, q0 + 32 * wave, lane);
    // keys that all, that any of the wave's queries see
    const int wave_full = e.limit(p, f.wq);
    const int wave_end = f.wq < e.nq ? e.limit(p, min(f.wq + 32, e.nq) - 1) : 0;
    if (tiles > 0) {
        f16v s0[2], s1[2];
        wait_dma();
        __syncthreads();
        dv.issue(vr, 0, Vs, wave);
        if (tiles > 1) dk.issue(kr, BK, Ks + F::TILE, wave);
        f.scores(s0, 0, ra);
        f.settle(s0, 0, BK <= wave_full);
        auto turn = [&](f16v (&now)[2], f16v (&next)[2], int n, int buf) {
            wait_dma();
            meet();
            if (n + 1 < tiles) dv.issue(vr, (n + 1) * BK, Vs + (buf ^ 1) * F::TILE, wave);
            if (n + 2 < tiles) dk.issue(kr, (n + 2) * BK, Ks + buf * F::TILE, wave);
            u4v p0[TL::FRAGS], p1[TL::FRAGS];
            if (n * BK >= wave_end) return;
            // (float32 by 128: [4, 1024, 8, 128] 207 -> 169 us; 16 bits by 128 have the registers,
            // and lose by it: [2, 8192, 16, 128] 1045 -> 1240 us)
            constexpr bool WIDE = TL::ROW == 512;
            const int rn = WIDE ? fresh(ra, n) : ra, cn = WIDE ? fresh(ca, n) : ca;
            f.scores(next, buf ^ 1, rn);   // past the wave's last tile: of no use, and harmless
            f.weights(now, 0, n * BK, p0);
            f.values(p0, 0, buf, cn);
            f.weights(now, 1, n * BK, p1);
            f.values(p1, 1, buf, cn);
            if ((n + 1) * BK < wave_end)
                f.settle(next, (n + 1) * BK, (n + 2) * BK <= wave_full);
        };
        for (int n = 0; n < tiles; n += 2) {
            turn(s0, s1, n, 0);
            if (n + 1 < tiles) turn(s1, s0, n + 1, 1);
        }
    }
    f.store(e, b, hq, bh);
}

template <class T, int DP, int NW, bool BIAS, bool DROP>
int launch_forward_as(const ForwardArgs& a, hipStream_t st) {
    auto kernel = attention_forward_kernel<T, DP, NW, BIAS, DROP>;
    const int lds = Forward<T, DP, NW, BIAS, DROP>::LDS +
                    (BIAS ? (2 * a.p.max_distance + 1) * 4 : 0);
    static LdsAllowed known;
    D2P_TRY(allow_lds((const void*)kernel, known));
    const long long n = (long long)a.p.B * a.p.Hq * cdiv(a.p.Lq, 32 * NW);
    D2P_REQUIRE(n <= 0x7fffffffLL, "too many query blocks");
    if (n == 0) return D2P_OK;
    D2P_LAUNCH("attention_forward", kernel, dim3((unsigned)n), dim3(64 * NW), lds, st, a);
    D2P_HIP(hipGetLastError());
    return D2P_OK;
}

// Waves of 32 queries in a workgroup: eight share K and V tiles where features are many and
// the card is filled twice even so ([2, 8192, 16, 128] bfloat16: 989 us, 1112 TFLOP/s, against
// 1117 with four; [2, 4096, 16, 128] causal: 147 against 154); four otherwise, whose blocks
// fill it sooner ([4, 4096, 16, 64]: 330 us against 357; [4, 1023, 12, 80] causal: 40 against 46).
template <class T, int DP, bool BIAS, bool DROP>
int launch_forward_shape(const ForwardArgs& a, hipStream_t st) {
    if constexpr (DP == 128 && sizeof(T) == 2)
        if ((long long)a.p.B * a.p.Hq * cdiv(a.p.Lq, 256) >= 2LL * device_cus())
            return launch_forward_as<T, DP, 8, BIAS, DROP>(a, st);
    return launch_forward_as<T, DP, 4, BIAS, DROP>(a, st);
}

template <class T, int DP> int launch_forward_dp(const ForwardArgs& a, hipStream_t st) {
    if (a.p.bias)
        return a.p.drop ? launch_forward_shape<T, DP, true, true>(a, st)
                        : launch_forward_shape<T, DP, true, false>(a, st);
    return a.p.drop ? launch_forward_shape<T, DP, false, true>(a, st)
                    : launch_forward_shape<T, DP, false, false>(a, st);
}

template <class T> int launch_forward(const ForwardArgs& a, hipStream_t st) {
    switch (padded(a.p.D, a.p.dtype)) {
        case 32: return launch_forward_dp<T, 32>(a, st);
        case 64: return launch_forward_dp<T, 64>(a, st);
        case 96:
            if constexpr (sizeof(T) == 2) return launch_forward_dp<T, 96>(a, st);
        default: return launch_forward_dp<T, 128>(a, st);
    }
}

int launch_forward_f32(const ForwardArgs& a, hipStream_t st);
int launch_forward_f16(const ForwardArgs& a, hipStream_t st);
int launch_forward_bf16(const ForwardArgs& a, hipStream_t st);

}  // namespace enc
}  // namespace d2p_amd
