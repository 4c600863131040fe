// attention_backward.hip.h -- gradients of softmax attention.
//
// The probabilities are computed again from the scores and each row's two statistics.  Two
// kernels, each with its sums in registers from beginning to end: one over queries (delta,
// dQ, the bias's gradient), one over keys (dK, dV).  They form S and dP twice, 7 products
// where 5 would do, and in return nothing is added across workgroups: no atomics, no order
// that changes results, no partial gradients in memory.
#pragma once
#include <algorithm>

#include "attention_forward.hip.h"

namespace d2p_amd {
namespace enc {

struct BackwardArgs {
    d2p_attention_params p;
    const void *grad, *q, *k, *v, *out;
    const float* stats;
    void *dq, *dk, *dv, *dbias;
    float* delta;     // [B, Hq, Lq]: sum_j p_ij dp_ij = <out_i, grad_i>
    float* partial;   // [Hq][B blocks of queries][2 R + 1]: sums of ds by clipped distance
    float* heads;     // [2][B, Lk, Hq, D]: dK, dV of each query head where a group is split
    float* largest;   // [B Hq blocks of queries, 4 waves]: largest |grad| (half precision)
};

__host__ __device__ inline int query_blocks(const d2p_attention_params& p) {
    return cdiv(p.Lq, 128);
}

// Sums of ds by clipped distance, for the bias's gradient.  A tile at or past the clipping
// distance adds to one register.  Another goes to LDS skewed, so that a diagonal is a column:
// lane d sums column d.  What lies between the diagonals is zero from the start and never
// written.  Lanes and waves have their own places, joined at the end in a fixed order.
struct BiasSums {
    static constexpr int PITCH = 64, TILE = 32 * PITCH;   // 63 diagonals
    float behind = 0.0f, ahead = 0.0f, near = 0.0f;   // sums of ds
    float p_behind = 0.0f, p_ahead = 0.0f;            // of p
    // ds, p: lane = query, accumulators = keys from j0; at0: place of the wave's first query;
    // tile: of this wave, hist: its 2 R + 1 sums; down: what ds is scaled by, undone
    template <bool SCALED>
    __device__ __forceinline__ void add(const float* ds, const float* p, int j0, int at0, int R,
                                        float down, float* tile, float* hist, int lane) {
        const int far = bias_reach(j0, j0 + 31, at0, R);
        float s = 0.0f;
#pragma unroll
        for (int v = 0; v < 16; ++v) s += ds[v];
        if (far) {
            float w = 0.0f;
#pragma unroll
            for (int v = 0; v < 16; ++v) w += p[v];
            if (far < 0) { behind += s; p_behind += w; }
            else { ahead += s; p_ahead += w; }
            return;
        }
        near += s;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        const int q = lane & 31;
        float* row = tile + q * PITCH + 4 * (lane >> 5) + 31 - q;
#pragma unroll
        for (int v = 0; v < 16; ++v) row[8 * (v >> 2) + (v & 3)] = SCALED ? ds[v] * down : ds[v];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        float t[4] = {};
#pragma unroll
        for (int r = 0; r < 32; ++r) t[r & 3] += tile[r * PITCH + lane];
        const float sum = (t[0] + t[1]) + (t[2] + t[3]);
        const int d = j0 - at0 + lane - 31;   // (lane 63: no diagonal, zeros)
        // the ends of the table belong to the registers' sums; these pairs' p are not in
        // p_behind, p_ahead, so they stay out of the correction
        if (d > -R && d < R) hist[d + R] += sum;
        else if (d <= -R) edge_lo += sum;
        else edge_hi += sum;
    }
    float edge_lo = 0.0f, edge_hi = 0.0f;   // of tiles that reach past an end in part
};

// Queries of a workgroup's waves, 32 each; keys BK at a time, straight to LDS, two tiles of K
// and V each.
//
// Bound, for 64 keys and 32 queries of 128 features of 16 bits: 48 MFMAs of 32 cycles (S, dP,
// dQ) against near 1000 cycles of vector work; the fragments of K, V and K^T are 48 KiB of LDS
// reads, as many cycles as the MFMAs for four SIMDs.  Two waves a SIMD.
template <class T, int DP, bool BIAS, bool DROP, bool DBIAS> struct Dq {
    static constexpr int NW = 4, ROWS = 32 * NW;
    // two workgroups of a compute unit fit its LDS with the skewed tiles (one, with 32 bits)
    static constexpr int BK = DBIAS && (sizeof(T) == 2 ? Tile<T, DP>::ROW == 256
                                                       : Tile<T, DP>::ROW == 512) ? 32 : 64;
    static constexpr int TILE = Tile<T, DP>::bytes(BK) / 16;
    static int lds(const d2p_attention_params& p) {
        const int span = 2 * p.max_distance + 1;
        return 4 * TILE * 16 + (BIAS ? span * 4 : 0) +
               (DBIAS ? NW * (BiasSums::TILE + span) * 4 : 0);
    }
};

template <class T, int DP, bool BIAS, bool DROP, bool DBIAS>
__global__ void __launch_bounds__(256, sizeof(T) * DP >= 512 ? 1 : 2)
attention_dq_kernel(BackwardArgs a) {
    using TL = Tile<T, DP>;
    using K = Dq<T, DP, BIAS, DROP, DBIAS>;
    constexpr int BK = K::BK, DT = DP / 32, NW = K::NW;
    extern __shared__ __align__(16) u4v sm[];
    u4v* Ks = sm;
    u4v* Vs = sm + 2 * K::TILE;
    float* bias = (float*)(sm + 4 * K::TILE);
    const d2p_attention_params& p = a.p;
    const int R = p.max_distance, span = 2 * R + 1;
    const int tid = threadIdx.x, lane = tid & 63, wave = wave_of(tid), h = lane >> 5;
    float* tile = bias + span + wave * BiasSums::TILE;
    float* hists = bias + span + NW * BiasSums::TILE;
    const int nb = query_blocks(p);
    int bh, block;
    place(blockIdx.x, p.B * p.Hq, nb, p.causal, &bh, &block);
    const int b = bh / p.Hq, hq = bh % p.Hq, hk = hq / (p.Hq / p.Hkv);
    const int qb = p.causal ? nb - 1 - block : block, q0 = qb * K::ROWS;
    const Span e(p, b);
    const int D = p.D, wq = q0 + 32 * wave, i = wq + (lane & 31), at = i + e.off;
    const Rows kr = head_rows<T>(a.k, p.k, b, hk, e.nk, D);
    const Rows vr = head_rows<T>(a.v, p.v, b, hk, e.nk, D);
    const int end = q0 < e.nq ? e.limit(p, min(q0 + K::ROWS, e.nq) - 1) : 0;
    const int tiles = (end + BK - 1) / BK;
    TileDma<T, DP, BK, NW> dmk, dmv;
    dmk.init(kr, wave, lane);
    dmv.init(vr, wave, lane);
    if (tiles > 0) {
        dmk.issue(kr, 0, Ks, wave);
        dmv.issue(vr, 0, Vs, wave);
    }
    if (BIAS) load_bias<T>(bias, p, hq, tid, 64 * NW);
    if (DBIAS) {
        // each wave its own, which no other reads before the barrier of the join: a block without
        // tiles meets no barrier ahead of that
        for (int t = lane; t < span; t += 64) hists[wave * span + t] = 0.0f;
        for (int t = lane; t < BiasSums::TILE; t += 64) tile[t] = 0.0f;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }

    u4v qf[TL::STEPS], gf[TL::STEPS];
    float delta = 0.0f, big = 0.0f;
    {
        const d2p_strides own = {(long long)p.Lq * p.Hq * D, (long long)p.Hq * D, D};
        const Rows qr = head_rows<T>(a.q, p.q, b, hq, e.nq, D);
        const Rows gr = head_rows<T>(a.grad, p.grad, b, hq, e.nq, D);
        const Rows orow = head_rows<T>(a.out, own, b, hq, e.nq, D);
        const __amdgpu_buffer_rsrc_t rq = qr.from(q0), rg = gr.from(q0), ro = orow.from(q0);
#pragma unroll
        for (int s = 0; s < TL::STEPS; ++s) {
            qf[s] = __builtin_amdgcn_raw_buffer_load_b128(rq, qr.at(i - q0, 2 * s + h), 0, 0);
            gf[s] = __builtin_amdgcn_raw_buffer_load_b128(rg, gr.at(i - q0, 2 * s + h), 0, 0);
        }
#pragma unroll
        for (int s = 0; s < TL::STEPS; ++s) {
            const u4v of = __builtin_amdgcn_raw_buffer_load_b128(ro, orow.at(i - q0, 2 * s + h),
                                                                 0, 0);
            float x[TL::PER], y[TL::PER];
            Elem<T>::unpack(of, x);
            Elem<T>::unpack(gf[s], y);
#pragma unroll
            for (int n = 0; n < TL::PER; ++n) {
                delta += x[n] * y[n];
                if (NARROW<T>) big = fmaxf(big, fabsf(y[n]));
            }
        }
        delta = both_sum(delta);
    }
    const long long rows = (long long)p.B * p.Hq * p.Lq, at_row = (long long)bh * p.Lq + i;
    float m = __builtin_inff(), ll = 0.0f;   // a row without keys: every p is 0
    if (i < e.nq) {
        m = a.stats[at_row];
        ll = a.stats[rows + at_row];
        if (m == -__builtin_inff()) m = __builtin_inff();
    }
    const float lse = m + ll;
    const float c = p.scale * LOG2E;
    const Drop drop(p, bh);
    const float kept = DROP ? drop.scale : 1.0f;
    float up = 1.0f, down = 1.0f;   // scale of ds and back
    if (NARROW<T>) {
        big = both_max(big);
        up = pow2(DS_SHIFT<T> - exponent(big));
        down = pow2(exponent(big) - DS_SHIFT<T>);
#pragma unroll
        for (int s = 16; s > 0; s >>= 1) big = fmaxf(big, __shfl_xor(big, s, 64));
        if (lane == 0) a.largest[((long long)bh * nb + qb) * NW + wave] = big;
    }
    const float ups = kept * up;
    f16v dq[DT] = {};
    BiasSums sums;
    // keys that all, that any of the wave's queries see
    const int wave_full = e.limit(p, wq);
    const int wave_end = wq < e.nq ? e.limit(p, min(wq + 32, e.nq) - 1) : 0;
    // (rows past the last see none: a bias of distances that only they have may be NaN)
    const int limit = !BIAS || i < e.nq ? e.limit(p, i) : 0;
    const int unmasked = !BIAS || wq + 32 <= e.nq ? wave_full : 0;

    const int ra = TL::row_at(lane), ca = TL::col_at(lane);
    // probabilities x and kept gradients dp (not yet scaled) of 32 keys of a tile
    auto tile_of = [&](const u4v* kt, const u4v* vt, int t, int jt, float* x, f16v& dp) {
        f16v s = {};
        dp = f16v{};
#pragma unroll
        for (int n = 0; n < TL::STEPS; ++n) s = Elem<T>::mma(TL::frag(kt, 32 * t, n, ra), qf[n], s);
#pragma unroll
        for (int n = 0; n < TL::STEPS; ++n)
            dp = Elem<T>::mma(TL::frag(vt, 32 * t, n, ra), gf[n], dp);
        if (BIAS) add_bias(s, c, bias, R, jt, wq + e.off, at, lane);
        if (jt + 32 > unmasked) {
            const int left = limit - (jt + 4 * h);
#pragma unroll
            for (int v = 0; v < 16; ++v)
                s[v] = 8 * (v >> 2) + (v & 3) < left ? s[v] : -__builtin_inff();
        }
        // (a bias may be as low as its type goes: m and ll apart, or ll would be lost)
#pragma unroll
        for (int v = 0; v < 16; ++v)
            x[v] = exp2_(BIAS ? s[v] - m - ll : fmaf(s[v], c, -lse));
        if (DROP) {
            const u4v kw = drop.by_query(wq, jt, lane);
#pragma unroll
            for (int v = 0; v < 16; ++v) dp[v] = drop.keeps(kw, v) ? dp[v] : 0.0f;
        }
    };
    float less = delta * up;
    auto turn = [&](int n, int buf) {
        wait_dma();
        meet();
        if (n + 1 < tiles) {
            dmk.issue(kr, (n + 1) * BK, Ks + (buf ^ 1) * K::TILE, wave);
            dmv.issue(vr, (n + 1) * BK, Vs + (buf ^ 1) * K::TILE, wave);
        }
        if (n * BK >= wave_end) return;
        const u4v *kt = Ks + buf * K::TILE, *vt = Vs + buf * K::TILE;
        if (n == 0 && wave_full <= BK) {
            // Rows whose keys are all here: delta from p and dp themselves.  <out, grad>
            // carries the rounding of P and of out, which a long row averages away.
            float own_delta = 0.0f;
#pragma unroll 1
            for (int t = 0; t < BK / 32; ++t) {
                float x[16];
                f16v dp;
                tile_of(kt, vt, t, 32 * t, x, dp);
#pragma unroll
                for (int v = 0; v < 16; ++v) own_delta += x[v] * dp[v];
            }
            own_delta = both_sum(own_delta) * kept;
            if (limit <= BK) delta = own_delta;
            less = delta * up;
        }
#pragma unroll
        for (int t = 0; t < BK / 32; ++t) {
            const int jt = n * BK + 32 * t;
            float x[16], y[16];
            f16v dp;
            tile_of(kt, vt, t, jt, x, dp);
#pragma unroll
            for (int v = 0; v < 16; ++v) y[v] = x[v] * fmaf(dp[v], ups, -less);
            if (DBIAS)
                sums.template add<NARROW<T>>(y, x, jt, wq + e.off, R, down, tile,
                                             hists + wave * span, lane);
#pragma unroll
            for (int f = 0; f < TL::FRAGS; ++f) {
                // dS in the type of K, as P in the forward
                const u4v df = Elem<T>::pack(y + TL::PER * f);
#pragma unroll
                for (int d = 0; d < DT; ++d)
                    dq[d] = Elem<T>::mma(TL::frag_t(kt, 32 * t, 32 * d, f, ca), df, dq[d]);
            }
        }
    };
    for (int n = 0; n < tiles; n += 2) {
        turn(n, 0);
        if (n + 1 < tiles) turn(n + 1, 1);
    }

    if (DBIAS) {
        // A row's ds sum to nothing but what delta was off by; that much p's share of it
        // goes from the far distances' sums, and all of it from what dK uses.
        const float off = both_sum(sums.behind + sums.ahead + sums.near);
        delta += off * down;
        float lo = (sums.behind - off * sums.p_behind) * down + sums.edge_lo;
        float hi = (sums.ahead - off * sums.p_ahead) * down + sums.edge_hi;
#pragma unroll
        for (int s = 32; s > 0; s >>= 1) {
            lo += __shfl_xor(lo, s, 64);
            hi += __shfl_xor(hi, s, 64);
        }
        float* hist = hists + wave * span;
        if (lane == 0) {
            hist[0] += lo;
            hist[2 * R] += hi;
        }
        __syncthreads();
        float* to = a.partial + (((long long)hq * p.B + b) * nb + qb) * span;
        for (int t = tid; t < span; t += 64 * NW) {
            const float s = hists[t] + hists[span + t] + hists[2 * span + t] + hists[3 * span + t];
            to[t] = e.bad ? __builtin_nanf("") : s;
        }
    }
    if (i >= p.Lq) return;
    if (h == 0) a.delta[at_row] = delta;
    char* row = (char*)a.dq + (((long long)b * p.Lq + i) * p.Hq + hq) * D * (long long)sizeof(T);
    const float nan = __builtin_nanf("");
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int d0 = 32 * d + 8 * g + 4 * h;
            float y[4];
#pragma unroll
            for (int r = 0; r < 4; ++r)
                y[r] = e.bad ? nan : i >= e.nq ? 0.0f : dq[d][4 * g + r] * (p.scale * down);
            if (d0 < D) Elem<T>::store4(row + d0 * (int)sizeof(T), y);
        }
}

// Keys of one key head a workgroup, 32 a wave; the group's query heads one after the other
// (or one of them, its sums joined by a further kernel), queries BQ at a time, straight to
// LDS, two tiles of Q and dO each.  S and dP stand untransposed (lane = key), so that P and dS
// are the second operands of dV^T = dO^T P and dK^T = Q^T dS as they stand.
//
// Bound as the kernel over queries, with a fourth product.  dK and dV of 128 features of 16
// bits take half of the 256 registers that two waves a SIMD leave each, K's fragments an
// eighth: V's come from LDS there ([2, 4096, 16, 128] bfloat16 causal: 313 us, 878 TFLOP/s; when
// this was chosen 338, against 471 with them in the registers of one wave a SIMD, and 366 where
// eight waves share the tiles of queries).
template <class T, int DP> struct Dkv {
    static constexpr int NW = 4, KEYS = 32 * NW;
    static constexpr bool WIDE = Tile<T, DP>::ROW >= 256;   // V in LDS
    static constexpr int BQ = WIDE ? 32 : 64;
    static constexpr int TILE = Tile<T, DP>::bytes(BQ) / 16;
    static constexpr int V = WIDE ? Tile<T, DP>::bytes(KEYS) / 16 : 0;
    static int lds(const d2p_attention_params& p) {
        return (4 * TILE + V) * 16 + 2 * 3 * BQ * 4 + (p.bias ? (2 * p.max_distance + 1) * 4 : 0);
    }
};

template <class T, int DP, bool BIAS, bool DROP>
__global__ void __launch_bounds__(256, sizeof(T) * DP >= 512 ? 1 : 2)
attention_dkv_kernel(BackwardArgs a) {
    using TL = Tile<T, DP>;
    using K = Dkv<T, DP>;
    constexpr int BQ = K::BQ, DT = DP / 32, NW = K::NW;
    extern __shared__ __align__(16) u4v sm[];
    u4v* Qs = sm;
    u4v* Gs = sm + 2 * K::TILE;
    u4v* Vs = sm + 4 * K::TILE;
    float* stats = (float*)(Vs + K::V);   // [2][m, log2 of the sum, delta][BQ]
    float* bias = stats + 2 * 3 * BQ;
    const d2p_attention_params& p = a.p;
    const int R = p.max_distance;
    // (a wave's place as lanes' numbers: known to be the same in all of them, it makes branches
    // of the masks, which the products of two tiles no longer cross: 649 -> 680 us for
    // [4, 4096, 16, 64] bfloat16)
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, h = lane >> 5;
    const int mine = wave_of(tid);
    const int nb = cdiv(p.Lk, K::KEYS), group = p.Hq / p.Hkv;
    const bool split = a.heads != nullptr;   // a workgroup for each query head
    int bh, block;
    place(blockIdx.x, p.B * (split ? p.Hq : p.Hkv), nb, p.causal, &bh, &block);
    const int b = bh / (split ? p.Hq : p.Hkv), hx = bh % (split ? p.Hq : p.Hkv);
    const int hk = split ? hx / group : hx;
    const int g0 = split ? hx % group : 0, g1 = split ? g0 + 1 : group;
    const int k0 = block * K::KEYS;   // causal: the first have the most queries
    const Span e(p, b);
    const int D = p.D, wk = k0 + 32 * wave, j = wk + (lane & 31);

    u4v kf[TL::STEPS], vreg[K::WIDE ? 1 : TL::STEPS];
    {
        const Rows kr = head_rows<T>(a.k, p.k, b, hk, e.nk, D);
        const Rows vr = head_rows<T>(a.v, p.v, b, hk, e.nk, D);
        const __amdgpu_buffer_rsrc_t rk = kr.from(k0), rv = vr.from(k0);
#pragma unroll
        for (int s = 0; s < TL::STEPS; ++s) {
            kf[s] = __builtin_amdgcn_raw_buffer_load_b128(rk, kr.at(j - k0, 2 * s + h), 0, 0);
            if (!K::WIDE)
                vreg[s] = __builtin_amdgcn_raw_buffer_load_b128(rv, vr.at(j - k0, 2 * s + h), 0, 0);
        }
        if (K::WIDE) {
            TileDma<T, DP, K::KEYS, NW> dmv;
            dmv.init(vr, mine, lane);
            dmv.issue(vr, k0, Vs, mine);
        }
    }
    const int ra = TL::row_at(lane), ca = TL::col_at(lane);
    auto vf = [&](int s, int rn) {
        return K::WIDE ? TL::frag(Vs, 32 * mine, s, rn) : vreg[s];
    };
    const float c = p.scale * LOG2E;
    f16v dk[DT] = {}, dv[DT] = {};
    const long long rows = (long long)p.B * p.Hq * p.Lq;
    // causal: the first query that sees key k0, in whole tiles of 32
    const int first = p.causal ? max(k0 - e.off, 0) & ~31 : 0;
    const bool work = k0 < e.nk && first < e.nq;
    const int tiles = work ? (e.nq - first + BQ - 1) / BQ : 0;
    int e_ds = 0;   // dS is scaled by 2^(DS_SHIFT - e_ds)

    for (int g = g0; g < g1 && work; ++g) {
        const int hq = hk * group + g;
        const Rows qr = head_rows<T>(a.q, p.q, b, hq, e.nq, D);
        const Rows gr = head_rows<T>(a.grad, p.grad, b, hq, e.nq, D);
        const long long row0 = ((long long)b * p.Hq + hq) * p.Lq;
        const Drop drop(p, b * p.Hq + hq);
        const float kept = DROP ? drop.scale : 1.0f;
        float up = 1.0f;
        if (NARROW<T>) {
            // the head's largest gradient; what is summed so far goes to its scale
            const int n = 4 * query_blocks(p);
            const float* from = a.largest + ((long long)b * p.Hq + hq) * n;
            float big = 0.0f;
            for (int t = lane; t < n; t += 64) big = fmaxf(big, from[t]);
#pragma unroll
            for (int s = 32; s > 0; s >>= 1) big = fmaxf(big, __shfl_xor(big, s, 64));
            const int e_new = max(exponent(big), g > g0 ? e_ds : -100);
            if (g > g0 && e_new != e_ds) {
                const float f = pow2(max(e_ds - e_new, -126));
#pragma unroll
                for (int d = 0; d < DT; ++d) dk[d] *= f;
            }
            e_ds = e_new;
            up = pow2(DS_SHIFT<T> - e_ds - BACKWARD_SHIFT<T>);
        }
        const float ups = kept * up;
        TileDma<T, DP, BQ, NW> dmq, dmg;
        dmq.init(qr, mine, lane);
        dmg.init(gr, mine, lane);
        // a row's statistics, one thread a row, on their way to LDS
        float sm_ = 0.0f, sl_ = 0.0f, sd_ = 0.0f;
        auto load_stats = [&](int i0) {
            if (tid < BQ) {
                const bool in = i0 + tid < e.nq;
                const long long at = row0 + (in ? i0 + tid : 0);
                sm_ = a.stats[at];
                sl_ = a.stats[rows + at];
                sd_ = a.delta[at];
                // a row without keys, or past the last: every p is 0
                if (!in || sm_ == -__builtin_inff()) sm_ = __builtin_inff();
                sl_ = in ? sl_ - BACKWARD_SHIFT<T> : 0.0f;
                sd_ = in ? sd_ * up : 0.0f;
                if (!BIAS) sm_ += sl_;
            }
        };
        auto store_stats = [&](int buf) {
            if (tid < BQ) {
                float* to = stats + buf * 3 * BQ + tid;
                to[0] = sm_;
                if (BIAS) to[BQ] = sl_;
                to[2 * BQ] = sd_;
            }
        };
        __syncthreads();   // the head before is done with LDS
        load_stats(first);
        store_stats(0);
        dmq.issue(qr, first, Qs, mine);
        dmg.issue(gr, first, Gs, mine);
        if (BIAS) load_bias<T>(bias, p, hq, tid, 64 * NW);

        auto turn = [&](int n, int buf) {
            const int i0 = first + n * BQ;
            wait_dma();
            meet();
            if (n + 1 < tiles) {
                load_stats(i0 + BQ);
                dmq.issue(qr, i0 + BQ, Qs + (buf ^ 1) * K::TILE, mine);
                dmg.issue(gr, i0 + BQ, Gs + (buf ^ 1) * K::TILE, mine);
            }
            const int rn = K::WIDE ? fresh(ra, n) : ra, cn = K::WIDE ? fresh(ca, n) : ca;
            const u4v *qt = Qs + buf * K::TILE, *gt = Gs + buf * K::TILE;
            const float* st = stats + buf * 3 * BQ;
#pragma unroll
            for (int t = 0; t < BQ / 32; ++t) {
                const int it = i0 + 32 * t;
                f16v s = {}, dp = {};
#pragma unroll
                for (int n = 0; n < TL::STEPS; ++n)
                    s = Elem<T>::mma(TL::frag(qt, 32 * t, n, rn), kf[n], s);
#pragma unroll
                for (int n = 0; n < TL::STEPS; ++n)
                    dp = Elem<T>::mma(TL::frag(gt, 32 * t, n, rn), vf(n, rn), dp);
                float pr[16], ds[16];
                if (BIAS) add_bias_by_key(s, c, bias, R, wk, it + e.off, lane);
                // (a key past the last spoils only its own row, which is not written)
                if (p.causal && wk + 31 > it + e.off) {
                    const int from = j - (it + 4 * h + e.off);
#pragma unroll
                    for (int v = 0; v < 16; ++v)
                        s[v] = 8 * (v >> 2) + (v & 3) >= from ? s[v] : -__builtin_inff();
                }
                if (BIAS && it + 32 > e.nq) {
                    // as in the kernel over queries
                    const int left = e.nq - (it + 4 * h);
#pragma unroll
                    for (int v = 0; v < 16; ++v)
                        s[v] = 8 * (v >> 2) + (v & 3) < left ? s[v] : -__builtin_inff();
                }
                const u4v kw = DROP ? drop.by_key(it, wk, lane) : u4v{};
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const f4v m4 = *(const f4v*)(st + 32 * t + 8 * q + 4 * h);
                    const f4v d4 = *(const f4v*)(st + 2 * BQ + 32 * t + 8 * q + 4 * h);
                    f4v l4 = {};
                    if (BIAS) l4 = *(const f4v*)(st + BQ + 32 * t + 8 * q + 4 * h);
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int v = 4 * q + r;
                        const float x = exp2_(BIAS ? s[v] - m4[r] - l4[r] : fmaf(s[v], c, -m4[r]));
                        const bool keep = !DROP || drop.keeps(kw, v);
                        pr[v] = keep ? x : 0.0f;
                        ds[v] = x * fmaf(keep ? dp[v] : 0.0f, ups, -d4[r]);
                    }
                }
#pragma unroll
                for (int f = 0; f < TL::FRAGS; ++f) {
                    u4v pf = Elem<T>::pack(pr + TL::PER * f);
#pragma unroll
                    for (int d = 0; d < DT; ++d)
                        dv[d] = Elem<T>::mma(TL::frag_t(gt, 32 * t, 32 * d, f, cn), pf, dv[d]);
                }
#pragma unroll
                for (int f = 0; f < TL::FRAGS; ++f) {
                    const u4v df = Elem<T>::pack(ds + TL::PER * f);
#pragma unroll
                    for (int d = 0; d < DT; ++d)
                        dk[d] = Elem<T>::mma(TL::frag_t(qt, 32 * t, 32 * d, f, cn), df, dk[d]);
                }
            }
            if (n + 1 < tiles) store_stats(buf ^ 1);
        };
        if (K::WIDE) {
            for (int n = 0; n < tiles; ++n) turn(n, n & 1);
        } else {
            for (int n = 0; n < tiles; n += 2) {
                turn(n, 0);
                if (n + 1 < tiles) turn(n + 1, 1);
            }
        }
    }
    if (j >= p.Lk) return;
    // the scales of P and dS, undone
    const float kept = DROP ? 256.0f / (256 - p.drop) : 1.0f;
    const float fv = kept * pow2(-BACKWARD_SHIFT<T>);
    const float fk = p.scale * (NARROW<T> ? pow2(e_ds - DS_SHIFT<T>) : 1.0f);
    const long long row = split ? (((long long)b * p.Lk + j) * p.Hq + hx) * D
                                : (((long long)b * p.Lk + j) * p.Hkv + hk) * D;
    const long long all = (long long)p.B * p.Lk * p.Hq * D;
    const float nan = __builtin_nanf("");
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int d0 = 32 * d + 8 * g + 4 * h;
            float y[4], z[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                y[r] = e.bad ? nan : j >= e.nk ? 0.0f : dk[d][4 * g + r] * fk;
                z[r] = e.bad ? nan : j >= e.nk ? 0.0f : dv[d][4 * g + r] * fv;
            }
            if (d0 >= D) continue;
            if (split) {
                Elem<float>::store4(a.heads + row + d0, y);
                Elem<float>::store4(a.heads + all + row + d0, z);
            } else {
                Elem<T>::store4((T*)a.dk + row + d0, y);
                Elem<T>::store4((T*)a.dv + row + d0, z);
            }
        }
}

// dK and dV of a key head: the sums of its query heads', in order, rounded once.  A thread
// takes four features; the rows of dK, then those of dV.
template <class T> __global__ void __launch_bounds__(256) join_heads_kernel(BackwardArgs a) {
    const d2p_attention_params& p = a.p;
    const int quads = p.D / 4, group = p.Hq / p.Hkv;
    const long long half = (long long)p.B * p.Lk * p.Hkv * quads;
    const long long all = (long long)p.B * p.Lk * p.Hq * p.D;
    for (long long n = (long long)blockIdx.x * 256 + threadIdx.x; n < 2 * half;
         n += (long long)gridDim.x * 256) {
        const long long m = n < half ? n : n - half;
        const long long row = m / quads, q = m % quads;   // (b, j, key head)
        const float* from = a.heads + (n < half ? 0 : all) + row * group * p.D + 4 * q;
        f4v s = *(const f4v*)from;
        for (int g = 1; g < group; ++g) s += *(const f4v*)(from + (long long)g * p.D);
        float y[4] = {s[0], s[1], s[2], s[3]};
        Elem<T>::store4((T*)(n < half ? a.dk : a.dv) + row * p.D + 4 * q, y);
    }
}

// dbias[n, h] = sum of the partial sums of head h whose distance lies in bucket n, in one
// order: a workgroup a head; its 16 waves take 64 distances each and, where those are few,
// slices of the blocks of queries; then 16 lanes a bucket.
template <class T>
__global__ void __launch_bounds__(1024) bias_grad_kernel(BackwardArgs a, int blocks) {
    extern __shared__ __align__(16) u4v sm[];
    const d2p_attention_params& p = a.p;
    const int span = 2 * p.max_distance + 1, h = blockIdx.x;
    float* part = (float*)sm;            // [16][64]
    float* sums = part + 16 * 64;        // [span]
    int* map = (int*)(sums + span);      // [span]
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int chunks = cdiv(span, 64), width = min(chunks, 16), slices = 16 / width;
    const int rows = p.B * blocks;
    for (int t = tid; t < span; t += 1024) map[t] = p.buckets[t];
    for (int c0 = 0; c0 < chunks; c0 += width) {
        const int t = (c0 + wave % width) * 64 + lane, slice = wave / width;
        float s[16] = {};
        if (t < span && slice < slices) {
            const float* from = a.partial + (long long)h * rows * span + t;
            auto at = [&](int n) { return from[(long long)n * span]; };
            int n = slice;
            for (; n + 15 * slices < rows; n += 16 * slices) {
#pragma unroll
                for (int u = 0; u < 16; ++u) s[u] += at(n + u * slices);
            }
            for (; n < rows; n += slices) s[0] += at(n);
        }
#pragma unroll
        for (int u = 8; u > 0; u >>= 1)
#pragma unroll
            for (int r = 0; r < u; ++r) s[r] += s[r + u];
        part[wave * 64 + lane] = s[0];
        __syncthreads();
        if (wave < width && t < span) {
            float y = 0.0f;
            for (int n = 0; n < slices; ++n) y += part[(n * width + wave) * 64 + lane];
            sums[t] = y;
        }
        __syncthreads();
    }
    for (int n = tid / 16; n < p.num_buckets; n += 64) {
        float s = 0.0f;
        for (int t = tid & 15; t < span; t += 16) s += map[t] == n ? sums[t] : 0.0f;
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
        if ((tid & 15) == 0) {
            const long long i = (long long)n * p.Hq + h;
            if (p.bias_dtype == D2P_FLOAT32) ((float*)a.dbias)[i] = s;
            else Elem<T>::store(a.dbias, i, s);
        }
    }
}

template <class T, int DP, bool BIAS, bool DROP, bool DBIAS>
int launch_dq_as(const BackwardArgs& a, hipStream_t st) {
    using K = Dq<T, DP, BIAS, DROP, DBIAS>;
    auto kernel = attention_dq_kernel<T, DP, BIAS, DROP, DBIAS>;
    const int lds = K::lds(a.p);
    static LdsAllowed known;
    D2P_TRY(allow_lds((const void*)kernel, known));
    const long long n = (long long)a.p.B * a.p.Hq * query_blocks(a.p);
    D2P_REQUIRE(n <= 0x7fffffffLL, "too many query blocks");
    if (n == 0) return D2P_OK;
    D2P_LAUNCH("attention_dq", kernel, dim3((unsigned)n), dim3(64 * K::NW), lds, st, a);
    D2P_HIP(hipGetLastError());
    return D2P_OK;
}

// Whether the query heads of a group go to workgroups of their own: where whole groups
// would leave compute units without work.
inline bool split_groups(const d2p_attention_params& p) {
    return p.Hq > p.Hkv &&
           (long long)p.B * p.Hkv * cdiv(p.Lk, 128) < 2LL * std::max(device_cus(), 1);
}

template <class T, int DP, bool BIAS, bool DROP>
int launch_dkv_as(const BackwardArgs& a, hipStream_t st) {
    using K = Dkv<T, DP>;
    auto kernel = attention_dkv_kernel<T, DP, BIAS, DROP>;
    const int lds = K::lds(a.p);
    static LdsAllowed known;
    D2P_TRY(allow_lds((const void*)kernel, known));
    const long long n = (long long)a.p.B * (a.heads ? a.p.Hq : a.p.Hkv) * cdiv(a.p.Lk, K::KEYS);
    D2P_REQUIRE(n <= 0x7fffffffLL, "too many key blocks");
    if (n == 0) return D2P_OK;
    D2P_LAUNCH("attention_dkv", kernel, dim3((unsigned)n), dim3(64 * K::NW), lds, st, a);
    D2P_HIP(hipGetLastError());
    if (!a.heads) return D2P_OK;
    const long long quads = 2LL * a.p.B * a.p.Lk * a.p.Hkv * (a.p.D / 4);
    D2P_LAUNCH("attention_join_heads", join_heads_kernel<T>,
               dim3((unsigned)std::min<long long>((quads + 255) / 256, 1 << 16)), dim3(256), 0, st,
               a);
    D2P_HIP(hipGetLastError());
    return D2P_OK;
}

template <class T, int DP> int launch_backward_dp(const BackwardArgs& a, hipStream_t st) {
    const bool drop = a.p.drop != 0;
    if (a.p.Lq > 0) {
        if (a.dbias)
            D2P_TRY(drop ? launch_dq_as<T, DP, true, true, true>(a, st)
                         : launch_dq_as<T, DP, true, false, true>(a, st));
        else if (a.p.bias)
            D2P_TRY(drop ? launch_dq_as<T, DP, true, true, false>(a, st)
                         : launch_dq_as<T, DP, true, false, false>(a, st));
        else
            D2P_TRY(drop ? launch_dq_as<T, DP, false, true, false>(a, st)
                         : launch_dq_as<T, DP, false, false, false>(a, st));
    }
    if (a.p.Lk > 0) {
        if (a.p.bias)
            D2P_TRY(drop ? launch_dkv_as<T, DP, true, true>(a, st)
                         : launch_dkv_as<T, DP, true, false>(a, st));
        else
            D2P_TRY(drop ? launch_dkv_as<T, DP, false, true>(a, st)
                         : launch_dkv_as<T, DP, false, false>(a, st));
    }
    return D2P_OK;
}

template <class T> int launch_backward(const BackwardArgs& a, hipStream_t st) {
    switch (padded(a.p.D, a.p.dtype)) {
        case 32: D2P_TRY(launch_backward_dp<T, 32>(a, st)); break;
        case 64: D2P_TRY(launch_backward_dp<T, 64>(a, st)); break;
        case 96:
            if constexpr (sizeof(T) == 2) { D2P_TRY(launch_backward_dp<T, 96>(a, st)); break; }
        default: D2P_TRY(launch_backward_dp<T, 128>(a, st));
    }
    if (!a.dbias) return D2P_OK;
    const int lds = (16 * 64 + 2 * (2 * a.p.max_distance + 1)) * 4;
    D2P_LAUNCH("attention_bias_grad", bias_grad_kernel<T>, dim3(a.p.Hq), dim3(1024), lds, st, a,
               query_blocks(a.p));
    D2P_HIP(hipGetLastError());
    return D2P_OK;
}

int launch_backward_f32(const BackwardArgs& a, hipStream_t st);
int launch_backward_f16(const BackwardArgs& a, hipStream_t st);
int launch_backward_bf16(const BackwardArgs& a, hipStream_t st);

}  // namespace enc
}  // namespace d2p_amd
