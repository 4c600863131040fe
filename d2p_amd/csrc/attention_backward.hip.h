// attention_backward.hip.h -- gradients of softmax attention.
//
// The probabilities are computed again from the scores and each row's two statistics.  Two
// kernels, each with its sums in registers from beginning to end: one over queries (delta,
// dQ, the bias's gradient), one over keys (dK, dV).  They form S and dP twice, 7 products
// where 5 would do, and in return nothing is added across workgroups: no atomics, no order
// that changes results, no partial gradients in memory.
#pragma once
#include "attention_forward.hip.h"

namespace d2p_amd {
namespace enc {

struct BackwardArgs {
    d2p_attention_params p;
    const void *grad, *q, *k, *v, *out;
    const float* stats;
    void *dq, *dk, *dv, *dbias;
    float* delta;     // [B, Hq, Lq]: sum_j p_ij dp_ij = <out_i, grad_i>
    float* partial;   // [B Hq blocks of queries, 2 R + 1]: sums of ds by clipped distance
    float* largest;   // [B Hq blocks of queries, 4 waves]: largest |grad| (half precision)
};

__host__ __device__ inline int query_blocks(const d2p_attention_params& p) {
    return cdiv(p.Lq, 128);
}

// Sums of ds by clipped distance.  A tile at or past the clipping distance adds to one
// register; another goes through LDS, where each lane sums one of its 63 diagonals.  Lanes
// and waves have their own places, joined at the end in a fixed order.
struct BiasSums {
    float behind = 0.0f, ahead = 0.0f;
    // x: ds, lane = query, accumulators = keys from j0; at0: place of the wave's first
    // query; tile: 32 x 33 floats of this wave, hist: its 2 R + 1 sums
    __device__ __forceinline__ void add(const float* x, int j0, int at0, int R, float* tile,
                                        float* hist, int lane) {
        const int far = bias_reach(j0, j0 + 31, at0, R);
        if (far) {
            float s = 0.0f;
#pragma unroll
            for (int v = 0; v < 16; ++v) s += x[v];
            if (far < 0) behind += s; else ahead += s;
            return;
        }
#pragma unroll
        for (int v = 0; v < 16; ++v)
            tile[(lane & 31) * 33 + 8 * (v >> 2) + 4 * (lane >> 5) + (v & 3)] = x[v];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        float s = 0.0f;
#pragma unroll
        for (int r = 0; r < 32; ++r) {
            const int n = lane - 31 + r;   // key of row r on diagonal lane - 31
            const float y = tile[n >= 0 && n < 32 ? r * 33 + n : 0];
            s += n >= 0 && n < 32 ? y : 0.0f;
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        const int d = j0 - at0 + lane - 31;
        if (lane == 63) return;             // 63 diagonals
        if (d <= -R) behind += s;
        else if (d >= R) ahead += s;
        else hist[d + R] += s;
    }
};

// 128 queries of one head a workgroup, 32 a wave, keys 64 at a time.
template <class T, int DP, bool BIAS, bool DROP, bool DBIAS>
__global__ void __launch_bounds__(256) attention_dq_kernel(BackwardArgs a) {
    using TL = Tile<T, DP>;
    constexpr int BK = 64, DT = DP / 32;
    extern __shared__ __align__(16) u4v sm[];
    u4v* Ks = sm;
    u4v* Vs = Ks + TL::bytes(BK) / 16;
    float* bias = (float*)(Vs + TL::bytes(BK) / 16);
    const d2p_attention_params& p = a.p;
    const int R = p.max_distance, span = 2 * R + 1;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, h = lane >> 5;
    float* tile = bias + span + wave * (32 * 33);
    float* hists = bias + span + 4 * 32 * 33;
    const int nb = (p.Lq + 127) / 128;
    const unsigned w = near_xcd(blockIdx.x, gridDim.x);
    const int bh = w / nb, b = bh / p.Hq, hq = bh % p.Hq;
    const int qb = p.causal ? nb - 1 - (int)(w % nb) : (int)(w % nb), q0 = qb * 128;
    const Span e(p, b);
    const int D = p.D, wq = q0 + 32 * wave, i = wq + (lane & 31), at = i + e.off;
    const Rows kr = head_rows<T>(a.k, p.k, b, hq / (p.Hq / p.Hkv), e.nk, D);
    const Rows vr = head_rows<T>(a.v, p.v, b, hq / (p.Hq / p.Hkv), e.nk, D);
    const d2p_strides own = {(long long)p.Lq * p.Hq * D, (long long)p.Hq * D, D};
    if (BIAS) load_bias<T>(bias, p, hq, tid, 256);
    if (DBIAS)
        for (int t = tid; t < 4 * span; t += 256) hists[t] = 0.0f;

    u4v qf[TL::STEPS], gf[TL::STEPS];
    float delta = 0.0f, big = 0.0f;
    {
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
        if (lane == 0) a.largest[((long long)bh * nb + qb) * 4 + wave] = big;
    }
    const float ups = kept * up;
    f16v dq[DT] = {};
    BiasSums sums;
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
        const bool full = j0 + BK <= wave_full;
        // probabilities x and kept gradients y (not yet scaled up) of 32 of the tile's keys
        auto tile_of = [&](int t, float* x, float* y) {
            f16v s = {}, dp = {};
#pragma unroll
            for (int n = 0; n < TL::STEPS; ++n) {
                s = Elem<T>::mma(TL::frag(Ks, 32 * t, n, lane), qf[n], s);
                dp = Elem<T>::mma(TL::frag(Vs, 32 * t, n, lane), gf[n], dp);
            }
            const int jt = j0 + 32 * t;
            const int far = BIAS ? bias_reach(jt, jt + 31, wq + e.off, R) : 0;
            if (full)
                score_tile<BIAS, true>(s, c, bias, R, far, jt, at, limit, lane, x);
            else
                score_tile<BIAS, false>(s, c, bias, R, far, jt, at, limit, lane, x);
            const u4v kw = DROP ? drop.by_query(wq, jt, lane) : u4v{};
#pragma unroll
            for (int v = 0; v < 16; ++v) {
                x[v] = exp2_(x[v] - m - ll);
                y[v] = !DROP || drop.keeps(kw, v) ? dp[v] : 0.0f;
            }
        };
        if (j0 == 0 && e.limit(p, wq) <= BK) {
            // Rows whose keys are all here: delta from p and dp themselves.  <out, grad>
            // carries the rounding of P and of out, which a long row averages away.
            float own_delta = 0.0f;
#pragma unroll 1
            for (int t = 0; t < 2; ++t) {
                float x[16], y[16];
                tile_of(t, x, y);
#pragma unroll
                for (int v = 0; v < 16; ++v) own_delta += x[v] * y[v];
            }
            own_delta = both_sum(own_delta) * kept;
            if (limit <= BK) delta = own_delta;
        }
        const float less = delta * up;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            float x[16], y[16];
            tile_of(t, x, y);
            const int jt = j0 + 32 * t;
#pragma unroll
            for (int v = 0; v < 16; ++v) x[v] *= fmaf(y[v], ups, -less);
            if (DBIAS && NARROW<T>) {
#pragma unroll
                for (int v = 0; v < 16; ++v) y[v] = x[v] * down;
                sums.add(y, jt, wq + e.off, R, tile, hists + wave * span, lane);
            }
            if (DBIAS && !NARROW<T>)
                sums.add(x, jt, wq + e.off, R, tile, hists + wave * span, lane);
#pragma unroll
            for (int f = 0; f < TL::FRAGS; ++f) {
                // dS in the type of K, as P in the forward
                const u4v df = Elem<T>::pack(x + TL::PER * f);
#pragma unroll
                for (int d = 0; d < DT; ++d)
                    dq[d] = Elem<T>::mma(TL::frag_t(Ks, 32 * t, 32 * d, f, lane), df, dq[d]);
            }
        }
    }

    if (DBIAS) {
        float lo = sums.behind, hi = sums.ahead;
#pragma unroll
        for (int s = 32; s > 0; s >>= 1) {
            lo += __shfl_xor(lo, s, 64);
            hi += __shfl_xor(hi, s, 64);
        }
        if (lane == 0) {
            hists[wave * span] += lo;
            hists[wave * span + 2 * R] += hi;
        }
        __syncthreads();
        float* to = a.partial + ((long long)bh * nb + qb) * span;
        for (int t = tid; t < span; t += 256) {
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

// 128 keys of one key head a workgroup, 32 a wave; the group's query heads one after the
// other, queries 64 at a time.  S and dP stand untransposed (lane = key), so that P and dS
// are the second operands of dV^T = dO^T P and dK^T = Q^T dS as they stand.
template <class T, int DP, bool BIAS, bool DROP>
__global__ void __launch_bounds__(256) attention_dkv_kernel(BackwardArgs a) {
    using TL = Tile<T, DP>;
    constexpr int BQ = 64, DT = DP / 32;
    extern __shared__ __align__(16) u4v sm[];
    u4v* Qs = sm;
    u4v* Gs = Qs + TL::bytes(BQ) / 16;
    float* row_m = (float*)(Gs + TL::bytes(BQ) / 16);   // statistics of the tile's rows
    float* row_l = row_m + BQ;
    float* row_d = row_l + BQ;
    float* bias = row_d + BQ;
    const d2p_attention_params& p = a.p;
    const int R = p.max_distance;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, h = lane >> 5;
    const int nb = (p.Lk + 127) / 128, group = p.Hq / p.Hkv;
    const unsigned w = near_xcd(blockIdx.x, gridDim.x);
    const int bh = w / nb, b = bh / p.Hkv, hk = bh % p.Hkv;
    const int k0 = (int)(w % nb) * 128;   // causal: the first have the most queries
    const Span e(p, b);
    const int D = p.D, wk = k0 + 32 * wave, j = wk + (lane & 31);

    u4v kf[TL::STEPS], vf[TL::STEPS];
    {
        const Rows kr = head_rows<T>(a.k, p.k, b, hk, e.nk, D);
        const Rows vr = head_rows<T>(a.v, p.v, b, hk, e.nk, D);
        const __amdgpu_buffer_rsrc_t rk = kr.from(k0), rv = vr.from(k0);
#pragma unroll
        for (int s = 0; s < TL::STEPS; ++s) {
            kf[s] = __builtin_amdgcn_raw_buffer_load_b128(rk, kr.at(j - k0, 2 * s + h), 0, 0);
            vf[s] = __builtin_amdgcn_raw_buffer_load_b128(rv, vr.at(j - k0, 2 * s + h), 0, 0);
        }
    }
    const float c = p.scale * LOG2E;
    f16v dk[DT] = {}, dv[DT] = {};
    const long long rows = (long long)p.B * p.Hq * p.Lq;
    // causal: the first query that sees key k0, in whole tiles of 32
    const int first = p.causal ? max(k0 - e.off, 0) & ~31 : 0;
    const bool work = k0 < e.nk && first < e.nq;
    int e_ds = 0;   // dS is scaled by 2^(DS_SHIFT - e_ds)

    for (int g = 0; g < group && work; ++g) {
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
            const int e_new = max(exponent(big), g ? e_ds : -100);
            if (g && e_new != e_ds) {
                const float f = pow2(max(e_ds - e_new, -126));
#pragma unroll
                for (int d = 0; d < DT; ++d) dk[d] *= f;
            }
            e_ds = e_new;
            up = pow2(DS_SHIFT<T> - e_ds - BACKWARD_SHIFT<T>);
        }
        const float ups = kept * up;
        Stage<T, DP, BQ, 256> qs, gs;
        float sm_ = 0.0f, sl_ = 0.0f, sd_ = 0.0f;
        auto load = [&](int i0) {
            qs.load(qr, i0, tid);
            gs.load(gr, i0, tid);
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
            }
        };
        load(first);
        for (int i0 = first; i0 < e.nq; i0 += BQ) {
            __syncthreads();
            qs.store(Qs, tid);
            gs.store(Gs, tid);
            if (tid < BQ) {
                row_m[tid] = sm_;
                row_l[tid] = sl_;
                row_d[tid] = sd_;
            }
            if (BIAS && i0 == first) load_bias<T>(bias, p, hq, tid, 256);
            __syncthreads();
            if (i0 + BQ < e.nq) load(i0 + BQ);
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const int it = i0 + 32 * t;
                f16v s = {}, dp = {};
#pragma unroll
                for (int n = 0; n < TL::STEPS; ++n) {
                    s = Elem<T>::mma(TL::frag(Qs, 32 * t, n, lane), kf[n], s);
                    dp = Elem<T>::mma(TL::frag(Gs, 32 * t, n, lane), vf[n], dp);
                }
                float pr[16], ds[16];
                const int far = BIAS ? bias_reach(wk, wk + 31, it + e.off, R) : 0;
                float bb = 0.0f;
                if (BIAS && far) bb = bias[far < 0 ? 0 : 2 * R];
                // every key of the wave seen by every query of the tile?
                const bool full = wk + 32 <= e.nk && (!p.causal || wk + 31 <= it + e.off);
                const u4v kw = DROP ? drop.by_key(it, wk, lane) : u4v{};
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const f4v m4 = *(const f4v*)(row_m + 32 * t + 8 * q + 4 * h);
                    const f4v l4 = *(const f4v*)(row_l + 32 * t + 8 * q + 4 * h);
                    const f4v d4 = *(const f4v*)(row_d + 32 * t + 8 * q + 4 * h);
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int v = 4 * q + r, at = it + 8 * q + 4 * h + r + e.off;
                        float y = s[v] * c;
                        if (BIAS) {
                            if (far == 0) bb = bias[min(max(j - at, -R), R) + R];
                            y += bb;
                        }
                        float x = exp2_(y - m4[r] - l4[r]);
                        if (!full) x = j < e.nk && (!p.causal || j <= at) ? x : 0.0f;
                        const bool keep = !DROP || drop.keeps(kw, v);
                        pr[v] = keep ? x : 0.0f;
                        ds[v] = x * fmaf(keep ? dp[v] : 0.0f, ups, -d4[r]);
                    }
                }
#pragma unroll
                for (int f = 0; f < TL::FRAGS; ++f) {
                    const u4v pf = Elem<T>::pack(pr + TL::PER * f);
                    const u4v df = Elem<T>::pack(ds + TL::PER * f);
#pragma unroll
                    for (int d = 0; d < DT; ++d) {
                        dv[d] = Elem<T>::mma(TL::frag_t(Gs, 32 * t, 32 * d, f, lane), pf, dv[d]);
                        dk[d] = Elem<T>::mma(TL::frag_t(Qs, 32 * t, 32 * d, f, lane), df, dk[d]);
                    }
                }
            }
        }
    }
    if (j >= p.Lk) return;
    // the scales of P and dS, undone
    const float kept = DROP ? 256.0f / (256 - p.drop) : 1.0f;
    const float fv = kept * pow2(-BACKWARD_SHIFT<T>);
    const float fk = p.scale * (NARROW<T> ? pow2(e_ds - DS_SHIFT<T>) : 1.0f);
    const long long row = (((long long)b * p.Lk + j) * p.Hkv + hk) * D * (long long)sizeof(T);
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
            if (d0 < D) {
                Elem<T>::store4((char*)a.dk + row + d0 * (int)sizeof(T), y);
                Elem<T>::store4((char*)a.dv + row + d0 * (int)sizeof(T), z);
            }
        }
}

// dbias[n, h] = sum of the partial sums of head h whose distance lies in bucket n, in one
// order: workgroup h, 16 waves over the blocks of queries, then one thread a bucket.
template <class T>
__global__ void __launch_bounds__(1024) bias_grad_kernel(BackwardArgs a, int blocks) {
    extern __shared__ __align__(16) u4v sm[];
    float* part = (float*)sm;            // [16][64]
    float* sums = part + 16 * 64;        // [2 R + 1]
    const d2p_attention_params& p = a.p;
    const int span = 2 * p.max_distance + 1, h = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    for (int t0 = 0; t0 < span; t0 += 64) {
        const int t = t0 + lane;
        float s = 0.0f;
        if (t < span)
            for (int n = wave; n < p.B * blocks; n += 16)
                s += a.partial[(((long long)(n / blocks) * p.Hq + h) * blocks + n % blocks) * span + t];
        part[wave * 64 + lane] = s;
        __syncthreads();
        if (wave == 0 && t < span) {
            s = 0.0f;
#pragma unroll
            for (int n = 0; n < 16; ++n) s += part[n * 64 + lane];
            sums[t] = s;
        }
        __syncthreads();
    }
    for (int n = tid; n < p.num_buckets; n += 1024) {
        float s = 0.0f;
        for (int t = 0; t < span; ++t)
            if (p.buckets[t] == n) s += sums[t];
        const long long i = (long long)n * p.Hq + h;
        if (p.bias_dtype == D2P_FLOAT32) ((float*)a.dbias)[i] = s;
        else Elem<T>::store(a.dbias, i, s);
    }
}

template <class T, int DP, bool BIAS, bool DROP, bool DBIAS>
int launch_dq_as(const BackwardArgs& a, hipStream_t st) {
    auto kernel = attention_dq_kernel<T, DP, BIAS, DROP, DBIAS>;
    const int span = 2 * a.p.max_distance + 1;
    const int lds = 2 * Tile<T, DP>::bytes(64) + (BIAS ? span * 4 : 0) +
                    (DBIAS ? (4 * 32 * 33 + 4 * span) * 4 : 0);
    D2P_HIP(hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize,
                                lds));
    const long long n = (long long)a.p.B * a.p.Hq * query_blocks(a.p);
    D2P_REQUIRE(n <= 0x7fffffffLL, "too many query blocks");
    if (n == 0) return D2P_OK;
    D2P_LAUNCH("attention_dq", kernel, dim3((unsigned)n), dim3(256), lds, st, a);
    D2P_HIP(hipGetLastError());
    return D2P_OK;
}

template <class T, int DP, bool BIAS, bool DROP>
int launch_dkv_as(const BackwardArgs& a, hipStream_t st) {
    auto kernel = attention_dkv_kernel<T, DP, BIAS, DROP>;
    const int lds = 2 * Tile<T, DP>::bytes(64) + 3 * 64 * 4 +
                    (BIAS ? (2 * a.p.max_distance + 1) * 4 : 0);
    D2P_HIP(hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize,
                                lds));
    const long long n = (long long)a.p.B * a.p.Hkv * cdiv(a.p.Lk, 128);
    D2P_REQUIRE(n <= 0x7fffffffLL, "too many key blocks");
    if (n == 0) return D2P_OK;
    D2P_LAUNCH("attention_dkv", kernel, dim3((unsigned)n), dim3(256), lds, st, a);
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
    switch (padded(a.p.D)) {
        case 32: D2P_TRY(launch_backward_dp<T, 32>(a, st)); break;
        case 64: D2P_TRY(launch_backward_dp<T, 64>(a, st)); break;
        default: D2P_TRY(launch_backward_dp<T, 128>(a, st));
    }
    if (!a.dbias) return D2P_OK;
    const int lds = (16 * 64 + 2 * a.p.max_distance + 1) * 4;
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
