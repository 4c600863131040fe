// attention_few.hip.h -- attention of few queries (single tokens of a cache) over many keys.
//
// Bound by reading K and V once.  The rows of one key head, its group's query heads times
// the queries, fill tiles of 32 together; the keys are split over workgroups and, in one,
// over its four waves, each with its own running maximum and sum, joined at the end in a
// fixed order.  A wave keeps one tile of 32 keys in flight while it works on another: K in
// the registers that the matrix cores read, V through registers to its own part of LDS.
#pragma once
#include <cmath>

#include "attention_forward.hip.h"

namespace d2p_amd {
namespace enc {

// How a call is cut: rows of a key head in tiles of 32, keys in parts of part_tiles tiles.
struct FewPlan {
    int rows, row_tiles, parts, part_tiles;
};

struct FewArgs {
    ForwardArgs f;
    FewPlan plan;
    float* acc;       // [B Hkv rows][parts][D]: sums of the parts, not yet divided
    float* part_m;    // [B Hkv rows][parts]
    float* part_l;
};

template <class T, int DP, bool BIAS>
__global__ void __launch_bounds__(256) attention_few_kernel(FewArgs fa) {
    using TL = Tile<T, DP>;
    constexpr int DT = DP / 32, VC = 32 * TL::NCH / 64;   // chunks of a V tile a lane loads
    extern __shared__ __align__(16) u4v sm[];
    const ForwardArgs& a = fa.f;
    const d2p_attention_params& p = a.p;
    const FewPlan& pl = fa.plan;
    const int tid = threadIdx.x, lane = tid & 63, wave = wave_of(tid), h = lane >> 5;
    const int R = p.max_distance, group = p.Hq / p.Hkv, D = p.D;
    u4v* Vs = sm + wave * (TL::bytes(32) / 16);
    float* all_o = (float*)sm;                                   // [4][32][DP + 4], after the loop
    constexpr int OP = DP + 4;
    constexpr int tail = (4 * TL::bytes(32) > 4 * 32 * OP * 4 ? 4 * TL::bytes(32) : 4 * 32 * OP * 4);
    float* all_m = (float*)((char*)sm + tail);                   // [4][32]
    float* all_l = all_m + 128;
    int* map = (int*)(all_l + 128);                              // the bucket of each distance
    unsigned w = near_xcd(blockIdx.x, gridDim.x);
    const int part = w % pl.parts;
    w /= pl.parts;
    const int rt = w % pl.row_tiles, bk = w / pl.row_tiles, b = bk / p.Hkv, hk = bk % p.Hkv;
    const Span e(p, b);
    const int row = rt * 32 + (lane & 31);
    const bool in = row < pl.rows && row % p.Lq < e.nq;
    const int i = in ? row % p.Lq : 0, hq = hk * group + (in ? row / p.Lq : 0), at = i + e.off;
    const Rows kr = head_rows<T>(a.k, p.k, b, hk, e.nk, D);
    const Rows vr = head_rows<T>(a.v, p.v, b, hk, e.nk, D);
    const int begin = part * pl.part_tiles * 32;
    const int end = min(e.nk, begin + pl.part_tiles * 32);
    // places of the tile's rows: the last and the first query of the element at most
    const int at_lo = e.off, at_hi = max(e.nq - 1, 0) + e.off;

    float behind = 0.0f, ahead = 0.0f;
    auto bias_of = [&](int n) {
        float v = __builtin_nanf("");
        if (n >= 0 && n < p.num_buckets) {
            const long long x = (long long)n * p.Hq + hq;
            v = p.bias_dtype == D2P_FLOAT32 ? ((const float*)p.bias)[x] : Elem<T>::load(p.bias, x);
            v = in_log2(v);
        }
        return v;
    };
    if (BIAS) {
        for (int t = tid; t <= 2 * R; t += 256) map[t] = p.buckets[t];
        behind = bias_of(p.buckets[0]);
        ahead = bias_of(p.buckets[2 * R]);
        __syncthreads();
    }

    u4v qf[TL::STEPS] = {};
    if (in) {
        const char* q = (const char*)a.q +
                        (b * p.q.batch + (long long)i * p.q.row + hq * p.q.head) * (long long)sizeof(T);
#pragma unroll
        for (int s = 0; s < TL::STEPS; ++s)
            if (2 * s + h < D / TL::PER) qf[s] = *(const u4v*)(q + (2 * s + h) * 16);
    }
    const float c = p.scale * LOG2E;
    const int limit = in ? e.limit(p, i) : 0;
    const int all_see = p.causal ? min(e.nk, at_lo + 1) : e.nk;   // keys that every row sees
    f16v o[DT] = {};
    float m = -__builtin_inff(), l = 0.0f;

    const int ca = TL::col_at(lane);
    u4v kf[TL::STEPS], vf[VC];
    auto load = [&](int j0) {
        const __amdgpu_buffer_rsrc_t rk = kr.from(j0), rv = vr.from(j0);
#pragma unroll
        for (int s = 0; s < TL::STEPS; ++s)
            kf[s] = __builtin_amdgcn_raw_buffer_load_b128(rk, kr.at(lane & 31, 2 * s + h), 0, 0);
#pragma unroll
        for (int n = 0; n < VC; ++n)
            vf[n] = __builtin_amdgcn_raw_buffer_load_b128(
                rv, vr.at(n * (64 / TL::NCH) + lane / TL::NCH, lane % TL::NCH), 0, 0);
    };
    int j0 = begin + 32 * wave;
    if (j0 < end) load(j0);
    for (; j0 < end; j0 += 128) {
        f16v s = {};
#pragma unroll
        for (int n = 0; n < TL::STEPS; ++n) s = Elem<T>::mma(kf[n], qf[n], s);
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int n = 0; n < VC; ++n)
            Vs[TL::slot(n * (64 / TL::NCH) + lane / TL::NCH, lane % TL::NCH)] = vf[n];
        if (j0 + 128 < end) load(j0 + 128);
        float x[16];
        const bool full = j0 + 32 <= all_see;
        float bb = 0.0f;
        int far = 0;
        if (BIAS) {
            far = j0 + 31 - at_lo <= -R ? -1 : j0 - at_hi >= R ? 1 : 0;
            bb = far < 0 ? behind : ahead;
        }
        float top = -__builtin_inff();
#pragma unroll
        for (int v = 0; v < 16; ++v) {
            const int j = j0 + 4 * h + 8 * (v >> 2) + (v & 3);
            float y = s[v] * c;
            if (BIAS) {
                if (far == 0) bb = bias_of(map[min(max(j - at, -R), R) + R]);
                y += bb;
            }
            x[v] = full || j < limit ? y : -__builtin_inff();
            top = fmaxf(top, x[v]);
        }
        top = fmaxf(m, both_max(top));
        const float ref = top == -__builtin_inff() ? 0.0f : top;
        const float old = exp2_(m - ref);
        m = top;
        l *= old;
#pragma unroll
        for (int d = 0; d < DT; ++d) o[d] *= old;
#pragma unroll
        for (int v = 0; v < 16; ++v) {
            x[v] = exp2_(shifted<T>(x[v] - ref));
            l += x[v];
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int f = 0; f < TL::FRAGS; ++f) {
            const u4v pf = Elem<T>::pack(x + TL::PER * f);
#pragma unroll
            for (int d = 0; d < DT; ++d)
                o[d] = Elem<T>::mma(TL::frag_t(Vs, 0, 32 * d, f, ca), pf, o[d]);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }

    // the four waves, in order
    l = both_sum(l);
    __syncthreads();
    float* mine = all_o + (wave * 32 + (lane & 31)) * OP;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g)
            *(f4v*)(mine + 32 * d + 8 * g + 4 * h) =
                f4v{o[d][4 * g], o[d][4 * g + 1], o[d][4 * g + 2], o[d][4 * g + 3]};
    if (h == 0) {
        all_m[wave * 32 + (lane & 31)] = m;
        all_l[wave * 32 + (lane & 31)] = l;
    }
    __syncthreads();
    const float nan = __builtin_nanf("");
    // eight threads a row
    const int r = tid >> 3, rr = rt * 32 + r;
    if (rr >= pl.rows) return;
    float ms[4], f[4], top = -__builtin_inff(), sum = 0.0f;
#pragma unroll
    for (int n = 0; n < 4; ++n) {
        ms[n] = all_m[n * 32 + r];
        top = fmaxf(top, ms[n]);
    }
#pragma unroll
    for (int n = 0; n < 4; ++n) {
        f[n] = exp2_(ms[n] - (top == -__builtin_inff() ? 0.0f : top));
        sum += f[n] * all_l[n * 32 + r];
    }
    const bool whole = pl.parts == 1;
    const int ri = rr % p.Lq, rh = hk * group + rr / p.Lq;
    const bool none = ri >= e.nq || !(sum != 0.0f);
    const float inv = !whole ? 1.0f : none ? 0.0f : 1.0f / sum;
    const long long prow = ((long long)bk * pl.rows + rr) * pl.parts + part;
    char* out = (char*)a.out + (((long long)b * p.Lq + ri) * p.Hq + rh) * D * (long long)sizeof(T);
    for (int d = (tid & 7) * 4; d < D; d += 32) {
        f4v y = {};
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            const f4v z = *(const f4v*)(all_o + (n * 32 + r) * OP + d);
            y += z * f[n];
        }
        if (whole) {
            float yy[4];
#pragma unroll
            for (int n = 0; n < 4; ++n) yy[n] = e.bad ? nan : none ? 0.0f : y[n] * inv;
            Elem<T>::store4(out + d * (int)sizeof(T), yy);
        } else {
            *(f4v*)(fa.acc + prow * D + d) = y;
        }
    }
    if ((tid & 7) == 0) {
        if (whole) {
            const long long n = (long long)p.B * p.Hq * p.Lq;
            const long long x = ((long long)b * p.Hq + rh) * p.Lq + ri;
            a.stats[x] = e.bad ? nan : none ? -__builtin_inff() : top;
            a.stats[n + x] = none ? 0.0f : log2_(sum) - FORWARD_SHIFT<T>;
        } else {
            fa.part_m[prow] = top;
            fa.part_l[prow] = sum;
        }
    }
}

// Joins the parts of a row: one workgroup a row, D / 4 threads across the features and the
// rest of its 256 across the parts, in one order, with eight parts' loads in flight (64 rows of
// 256 parts by 64 features: 10.2 -> 9.1 us).
template <class T>
__global__ void __launch_bounds__(256) attention_join_kernel(FewArgs fa) {
    __shared__ float fac[256], red_m[4], red_l[4];
    __shared__ f4v red[256];
    const ForwardArgs& a = fa.f;
    const d2p_attention_params& p = a.p;
    const FewPlan& pl = fa.plan;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const long long prow = (long long)blockIdx.x * pl.parts;
    const int rr = blockIdx.x % pl.rows, bk = blockIdx.x / pl.rows, b = bk / p.Hkv;
    const int ri = rr % p.Lq, rh = bk % p.Hkv * (p.Hq / p.Hkv) + rr / p.Lq;
    const Span e(p, b);
    const int D = p.D;
    // parts are at most 256: one a thread
    const float pm = tid < pl.parts ? fa.part_m[prow + tid] : -__builtin_inff();
    const float pll = tid < pl.parts ? fa.part_l[prow + tid] : 0.0f;
    float top = pm;
#pragma unroll
    for (int s = 32; s > 0; s >>= 1) top = fmaxf(top, __shfl_xor(top, s, 64));
    if (lane == 0) red_m[wave] = top;
    __syncthreads();
    top = fmaxf(fmaxf(red_m[0], red_m[1]), fmaxf(red_m[2], red_m[3]));
    const float f = exp2_(pm - (top == -__builtin_inff() ? 0.0f : top));
    fac[tid] = f;
    float sum = tid < pl.parts ? f * pll : 0.0f;
#pragma unroll
    for (int s = 32; s > 0; s >>= 1) sum += __shfl_xor(sum, s, 64);
    if (lane == 0) red_l[wave] = sum;
    __syncthreads();
    sum = (red_l[0] + red_l[1]) + (red_l[2] + red_l[3]);
    const bool none = ri >= e.nq || !(sum != 0.0f);
    const int quads = D / 4, slices = 256 / quads, q = tid % quads, s0 = tid / quads;
    f4v y = {};
    if (s0 < slices) {
        // (a part that saw no key holds zeros, or what a NaN bias left there)
        const float* from = fa.acc + prow * D + 4 * q;
        int n = s0;
        for (; n + 7 * slices < pl.parts; n += 8 * slices) {
            f4v z[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) z[u] = *(const f4v*)(from + (long long)(n + u * slices) * D);
#pragma unroll
            for (int u = 0; u < 8; ++u) y += z[u] * fac[n + u * slices];
        }
        for (; n < pl.parts; n += slices) y += *(const f4v*)(from + (long long)n * D) * fac[n];
    }
    red[tid] = y;
    __syncthreads();
    if (tid < quads) {
        y = red[tid];
        for (int n = 1; n < slices; ++n) y += red[n * quads + tid];
        float yy[4];
        const float nan = __builtin_nanf("");
#pragma unroll
        for (int n = 0; n < 4; ++n) yy[n] = e.bad ? nan : none ? 0.0f : y[n] / sum;
        Elem<T>::store4((char*)a.out + ((((long long)b * p.Lq + ri) * p.Hq + rh) * D + 4 * q) *
                                           (long long)sizeof(T), yy);
        if (tid == 0) {
            const long long n = (long long)p.B * p.Hq * p.Lq;
            const long long x = ((long long)b * p.Hq + rh) * p.Lq + ri;
            a.stats[x] = e.bad ? nan : none ? -__builtin_inff() : top;
            a.stats[n + x] = none ? 0.0f : log2_(sum) - FORWARD_SHIFT<T>;
        }
    }
}

inline int few_features(const d2p_attention_params& p) {
    return p.D <= 32 ? 32 : p.D <= 64 ? 64 : 128;
}

// Whether a call goes this way, and how it is cut.
//
// Both ways' times in us, from what they measured on 256 compute units.  attention_forward
// passes over all keys with each of its blocks of 128 queries: 0.8 to 1 us for each 64 keys
// and each block that a compute unit gets.  This way costs 55 keys (of 128 features) a us and
// compute unit for each tile of 32 rows, and the join 1 us for each 1000 rows.  Measured, one
// way / the other (16 batch elements, 8 key heads of 128, 2048 keys, 4 query heads each): 1 query
// 67 / 37 us, 16 queries 66 / 59, 32 queries 64 / 78; 2 heads over 16384 keys: 1 query 263 / 15,
// 256 queries 267 / 38; 32 heads of 8 over 1024 keys, 128 queries: 23 / 28.
inline bool plan_few(const d2p_attention_params& p, FewPlan* pl) {
    if (p.drop || p.B == 0 || p.Lq == 0) return false;
    const int cus = device_cus() > 0 ? device_cus() : 256, dp = few_features(p);
    const bool wide = p.dtype == D2P_FLOAT32;
    const long long rows = (long long)p.Hq / p.Hkv * p.Lq;
    if (rows > 1 << 20) return false;
    const double all = (double)p.B * p.Hq * p.Lq;
    const double blocks = (double)p.B * p.Hq * cdiv(p.Lq, 128);
    const double forward = std::ceil(blocks / cus) * cdiv(p.Lk, 64) *
                           (wide ? dp / 12.8 : 0.6 + dp / 320.0);
    const double few = 3 + all / 1000 + (double)p.B * p.Hkv * cdiv((int)rows, 32) * p.Lk /
                       (cus * (wide ? 3264.0 : 7040.0) / dp);
    if (few > forward) return false;
    pl->rows = (int)rows;
    pl->row_tiles = cdiv(pl->rows, 32);
    const long long base = (long long)p.B * p.Hkv * pl->row_tiles;
    const int tiles = std::max(1, cdiv(p.Lk, 32));
    // two workgroups a compute unit, at least two tiles a wave
    long long parts = std::max<long long>(1, 2LL * cus / base);
    parts = std::min<long long>(parts, std::min(256, std::max(1, tiles / 8)));
    pl->part_tiles = (int)((tiles + parts - 1) / parts);
    pl->parts = cdiv(tiles, pl->part_tiles);
    return base * pl->parts <= 0x7fffffff && (long long)p.B * p.Hkv * rows <= 0x7fffffff;
}

// Floats of workspace: nothing where a row is one part.
inline size_t few_floats(const d2p_attention_params& p, const FewPlan& pl) {
    if (pl.parts == 1) return 0;
    return (size_t)p.B * p.Hkv * pl.rows * pl.parts * (p.D + 2);
}

template <class T, int DP, bool BIAS> int launch_few_as(const FewArgs& a, hipStream_t st) {
    auto kernel = attention_few_kernel<T, DP, BIAS>;
    const d2p_attention_params& p = a.f.p;
    const int lds = std::max(4 * Tile<T, DP>::bytes(32), 4 * 32 * (DP + 4) * 4) + 256 * 4 +
                    (BIAS ? (2 * p.max_distance + 1) * 4 : 0);
    static LdsAllowed known;
    D2P_TRY(allow_lds((const void*)kernel, known));
    const long long n = (long long)p.B * p.Hkv * a.plan.row_tiles * a.plan.parts;
    D2P_LAUNCH("attention_few", kernel, dim3((unsigned)n), dim3(256), lds, st, a);
    D2P_HIP(hipGetLastError());
    if (a.plan.parts == 1) return D2P_OK;
    D2P_LAUNCH("attention_join", attention_join_kernel<T>,
               dim3((unsigned)((long long)p.B * p.Hkv * a.plan.rows)), dim3(256), 0, st, a);
    D2P_HIP(hipGetLastError());
    return D2P_OK;
}

template <class T> int launch_few(const FewArgs& a, hipStream_t st) {
    const bool bias = a.f.p.bias != nullptr;
    switch (few_features(a.f.p)) {
        case 32: return bias ? launch_few_as<T, 32, true>(a, st) : launch_few_as<T, 32, false>(a, st);
        case 64: return bias ? launch_few_as<T, 64, true>(a, st) : launch_few_as<T, 64, false>(a, st);
        default: return bias ? launch_few_as<T, 128, true>(a, st) : launch_few_as<T, 128, false>(a, st);
    }
}

int launch_few_f32(const FewArgs& a, hipStream_t st);
int launch_few_f16(const FewArgs& a, hipStream_t st);
int launch_few_bf16(const FewArgs& a, hipStream_t st);

}  // namespace enc
}  // namespace d2p_amd
