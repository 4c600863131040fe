// qk_norm_rope.hip -- root-mean-square norm of each head of queries and keys with the
// rotation by position in the same pass, and its gradients (include/d2p_amd_encoder.h).
//
// Bound by memory: each element is read once and written once.  A group of lanes holds one
// row (one token's one head): lane n of it the pairs VEC n .. VEC n + VEC - 1, as two runs
// of VEC neighbours, the pairs' first and second features, which one vector load each
// brings in.  A group walks over heads of one token, whose angles it keeps in registers.
// Workgroups take queries or keys, never both, so that a lane keeps one weight and one sum
// for each of its features.  [32, 512, 8 + 8, 64] bfloat16: 16 us
// forward (4.2 TB/s), 25.5 us backward (3.9 TB/s); a copy of 4 GiB here reaches 4.8 TB/s.
#include <algorithm>

#include "encoder.hip.h"

namespace d2p_amd {
namespace enc {

// Queries or keys.
struct NormSide {
    const void *x, *g;      // rows, and their results' gradients
    void* out;              // results (forward) or gradients (backward)
    d2p_strides sx, sg;
    const float* weight;
    int heads, part;        // heads of a token, and of a unit
    int units_a_token;
    int blocks;             // workgroups
};

struct NormArgs {
    d2p_qk_norm_rope_params p;
    NormSide side[2];
    float* partial;         // [workgroups][D]: sums for the weights' gradients
    int lanes;              // of a group, a power of two
};

template <class T, int N> struct alignas(sizeof(T) * N) Run { T v[N]; };

template <class T, int VEC> struct Row {
    float x[2 * VEC];
    __device__ __forceinline__ void load(const T* p, int p0, int p1) {
        const Run<T, VEC> a = *(const Run<T, VEC>*)(p + p0), b = *(const Run<T, VEC>*)(p + p1);
#pragma unroll
        for (int e = 0; e < VEC; ++e) { x[e] = (float)a.v[e]; x[VEC + e] = (float)b.v[e]; }
    }
    __device__ __forceinline__ void store(T* p, int p0, int p1) const {
        Run<T, VEC> a, b;
#pragma unroll
        for (int e = 0; e < VEC; ++e) { a.v[e] = (T)x[e]; b.v[e] = (T)x[VEC + e]; }
        *(Run<T, VEC>*)(p + p0) = a;
        *(Run<T, VEC>*)(p + p1) = b;
    }
};

// What a lane keeps: where its features are, their angles and weights.
template <class T, int VEC> struct Lane {
    int p0, p1;           // first features of its two runs
    bool on;              // it has a pair
    bool pairs_adjacent;  // pair e is features 2 e, 2 e + 1 of the two runs together
    float co[VEC], si[VEC];
    float w[2 * VEC];

    __device__ __forceinline__ Lane(const d2p_qk_norm_rope_params& p, const float* weight, int n) {
        const int first = n * VEC, turned = p.R / 2;
        on = first < p.D / 2;
        pairs_adjacent = p.interleaved && first < turned;
        if (first >= turned) {            // not turned: any two runs
            p0 = p.R + 2 * (first - turned);
            p1 = p0 + VEC;
        } else if (p.interleaved) {
            p0 = 2 * first;
            p1 = p0 + VEC;
        } else {
            p0 = first;
            p1 = first + turned;
        }
        if (!on) p0 = p1 = 0;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            w[e] = on && weight ? weight[p0 + e] : 1.0f;
            w[VEC + e] = on && weight ? weight[p1 + e] : 1.0f;
        }
    }
    // the angles of token l of sequence b
    __device__ __forceinline__ void angles(const d2p_qk_norm_rope_params& p, long long token,
                                           int n) {
        const long long pos = p.positions ? p.positions[token] : token % p.L;
        const bool known = p.R == 0 || (pos >= 0 && pos < p.table_rows);
        const int first = n * VEC;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            co[e] = 1.0f;
            si[e] = 0.0f;
        }
        if (!known) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) co[e] = si[e] = __builtin_nanf("");
        } else if (on && first < p.R / 2) {
            const float* c = p.cos + pos * (p.R / 2) + first;
            const float* s = p.sin + pos * (p.R / 2) + first;
            if constexpr (VEC >= 4) {
#pragma unroll
                for (int e = 0; e < VEC; e += 4) {
                    const f4v cv = *(const f4v*)(c + e), sv = *(const f4v*)(s + e);
#pragma unroll
                    for (int r = 0; r < 4; ++r) { co[e + r] = cv[r]; si[e + r] = sv[r]; }
                }
            } else {
#pragma unroll
                for (int e = 0; e < VEC; ++e) { co[e] = c[e]; si[e] = s[e]; }
            }
        }
    }
    // x turned by the angles (sign 1) or back (sign -1)
    __device__ __forceinline__ void turn(float* x, float sign) const {
        if (VEC > 1 && pairs_adjacent) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float a = x[2 * e], c = x[2 * e + 1], s = sign * si[e];
                x[2 * e] = a * co[e] - c * s;
                x[2 * e + 1] = c * co[e] + a * s;
            }
        } else {
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float a = x[e], c = x[VEC + e], s = sign * si[e];
                x[e] = a * co[e] - c * s;
                x[VEC + e] = c * co[e] + a * s;
            }
        }
    }
};

template <int CTRL> __device__ __forceinline__ float plus_dpp(float s) {
    return s + bits<float>(__builtin_amdgcn_mov_dpp(bits<int>(s), CTRL, 0xf, 0xf, true));
}
// The sum over a group of lanes.  Neighbours by data-parallel moves: after the pairs and
// the fours, mirroring eight lanes or sixteen brings the other half's sum.
__device__ __forceinline__ float group_sum(float s, int lanes) {
    if (lanes > 1) s = plus_dpp<0xB1>(s);
    if (lanes > 2) s = plus_dpp<0x4E>(s);
    if (lanes > 4) s = plus_dpp<0x141>(s);
    if (lanes > 8) s = plus_dpp<0x140>(s);
    if (lanes > 16) s += __shfl_xor(s, 16, 64);
    if (lanes > 32) s = both_sum(s);
    return s;
}

template <class T>
__device__ __forceinline__ const T* row_of(const void* base, const d2p_strides& s, int b, int l,
                                           int h) {
    return (const T*)base + b * s.batch + l * s.row + h * s.head;
}

// Threads of a workgroup: the backward's are more, so that its partial sums are few.
template <bool BACK> constexpr int THREADS = BACK ? 512 : 256;

template <class T, int VEC, bool BACK>
__global__ void __launch_bounds__(THREADS<BACK>) qk_norm_rope_kernel(NormArgs a) {
    const d2p_qk_norm_rope_params& p = a.p;
    const bool keys = (int)blockIdx.x >= a.side[0].blocks;
    const NormSide& side = a.side[keys];
    const int block = keys ? blockIdx.x - a.side[0].blocks : blockIdx.x;
    const int n = threadIdx.x & (a.lanes - 1), D = p.D;
    const int groups = THREADS<BACK> / a.lanes;
    const long long units = (long long)p.B * p.L * side.units_a_token;
    Lane<T, VEC> ln(p, side.weight, n);
    float sums[2 * VEC] = {};   // the weight's gradient
    for (long long u = (long long)block * groups + threadIdx.x / a.lanes; u < units;
         u += (long long)side.blocks * groups) {
        const long long token = u / side.units_a_token;
        const int b = (int)(token / p.L), l = (int)(token % p.L);
        const int h0 = (int)(u % side.units_a_token) * side.part;
        const int h1 = min(h0 + side.part, side.heads);
        ln.angles(p, token, n);
        for (int h = h0; h < h1; ++h) {
            Row<T, VEC> x, g;
            float ss = 0.0f;
            if (ln.on) {
                x.load(row_of<T>(side.x, side.sx, b, l, h), ln.p0, ln.p1);
                if (BACK) g.load(row_of<T>(side.g, side.sg, b, l, h), ln.p0, ln.p1);
#pragma unroll
                for (int e = 0; e < 2 * VEC; ++e) ss += x.x[e] * x.x[e];
            }
            const float r = 1.0f / sqrtf(group_sum(ss, a.lanes) / D + p.eps);
            T* dst = (T*)side.out + (token * side.heads + h) * D;
            if (!BACK) {
#pragma unroll
                for (int e = 0; e < 2 * VEC; ++e) x.x[e] *= r * ln.w[e];
                ln.turn(x.x, 1.0f);
                if (ln.on) x.store(dst, ln.p0, ln.p1);
            } else {
                float dot = 0.0f;
                if (ln.on) {
                    ln.turn(g.x, -1.0f);
#pragma unroll
                    for (int e = 0; e < 2 * VEC; ++e) {
                        x.x[e] *= r;
                        sums[e] += g.x[e] * x.x[e];
                        g.x[e] *= ln.w[e];
                        dot += g.x[e] * x.x[e];
                    }
                }
                dot = group_sum(dot, a.lanes) / D;
                if (ln.on) {
#pragma unroll
                    for (int e = 0; e < 2 * VEC; ++e) x.x[e] = r * (g.x[e] - x.x[e] * dot);
                    x.store(dst, ln.p0, ln.p1);
                }
            }
        }
    }
    if (BACK && a.partial) {
        // the wave's groups, then the waves, in one order
        constexpr int WAVES = THREADS<BACK> / 64;
        __shared__ float part[WAVES][128];
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
        for (int e = 0; e < 2 * VEC; ++e)
            for (int o = 32; o >= a.lanes; o >>= 1) sums[e] += __shfl_xor(sums[e], o, 64);
        if (lane < a.lanes && ln.on) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                part[wave][ln.p0 + e] = sums[e];
                part[wave][ln.p1 + e] = sums[VEC + e];
            }
        }
        __syncthreads();
        const int d = threadIdx.x;
        if (d < D) {
            float s = 0.0f;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) s += part[w][d];
            a.partial[(long long)blockIdx.x * D + d] = s;
        }
    }
}

// dw[d] = sum over the workgroups of queries (or keys): 64 features a workgroup, 16 waves over
// the rows
__global__ void __launch_bounds__(1024)
weight_grad_kernel(const float* partial, int q_rows, int k_rows, int D, float* dwq, float* dwk) {
    __shared__ float part[16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int tiles = (D + 63) / 64;
    const bool keys = (int)blockIdx.x >= tiles;
    const int d = ((int)blockIdx.x - (keys ? tiles : 0)) * 64 + lane;
    const int rows = keys ? k_rows : q_rows;
    const float* from = partial + (keys ? (long long)q_rows * D : 0) + d;
    float s = 0.0f;
    if (d < D) {
        float t[8] = {};
        int r = wave;
        for (; r + 7 * 16 < rows; r += 8 * 16) {
#pragma unroll
            for (int u = 0; u < 8; ++u) t[u] += from[(long long)(r + 16 * u) * D];
        }
        for (; r < rows; r += 16) t[0] += from[(long long)r * D];
#pragma unroll
        for (int u = 0; u < 8; ++u) s += t[u];
    }
    part[wave][lane] = s;
    __syncthreads();
    float* to = keys ? dwk : dwq;
    if (wave || d >= D || !to) return;
    s = 0.0f;
#pragma unroll
    for (int w = 0; w < 16; ++w) s += part[w][lane];
    to[d] = s;
}

namespace {

constexpr int BACK_GROUPS = 512;   // workgroups of the backward pass at most

bool multiple(const d2p_strides& s, int n) {
    return s.batch % n == 0 && s.row % n == 0 && s.head % n == 0;
}

// The widest runs that the sizes, strides and addresses allow: 16 bytes at best.
int run_width(const NormArgs& a, bool back) {
    const d2p_qk_norm_rope_params& p = a.p;
    const int size = type_bytes(p.dtype);
    int v = 16 / size;
    if (((uintptr_t)p.cos | (uintptr_t)p.sin) & 15) v = std::min(v, 2);
    for (; v > 1; v >>= 1) {
        uintptr_t at = 0;
        for (const NormSide& side : a.side)
            at |= (uintptr_t)side.x | (uintptr_t)side.out | (back ? (uintptr_t)side.g : 0);
        const bool strides = multiple(p.q, v) && multiple(p.k, v) &&
                             (!back || (multiple(p.gq, v) && multiple(p.gk, v)));
        if ((p.R / 2) % v == 0 && ((p.D - p.R) / 2) % v == 0 && strides && at % (v * size) == 0)
            break;
    }
    return v;
}

int check(const d2p_qk_norm_rope_params* p) {
    D2P_REQUIRE(p != nullptr, "null parameters");
    D2P_REQUIRE(p->dtype == D2P_FLOAT32 || p->dtype == D2P_FLOAT16 || p->dtype == D2P_BFLOAT16,
                "unknown element type");
    D2P_REQUIRE(p->B >= 0 && p->L >= 0 && p->Hq >= 0 && p->Hkv >= 0, "negative size");
    D2P_REQUIRE((long long)p->Hq + p->Hkv <= 0x7fffffff, "too many heads");
    D2P_REQUIRE(p->D >= 8 && p->D <= 128 && p->D % 8 == 0,
                "head size must be a multiple of 8 from 8 to 128");
    D2P_REQUIRE(p->R >= 0 && p->R <= p->D && p->R % 2 == 0,
                "the rotated features must be even in number and at most the head size");
    D2P_REQUIRE(p->R == 0 || (p->cos && p->sin), "null pointer argument");
    D2P_REQUIRE(p->positions || p->R == 0 || p->table_rows >= p->L,
                "the tables must have a row for each position");
    D2P_REQUIRE(p->eps >= 0.0f, "eps must not be negative");
    return D2P_OK;
}

template <class T, int VEC, bool BACK> int launch_as(const NormArgs& a, int grid, hipStream_t st) {
    D2P_LAUNCH(BACK ? "qk_norm_rope_backward" : "qk_norm_rope", (qk_norm_rope_kernel<T, VEC, BACK>),
               dim3(grid), dim3(THREADS<BACK>), 0, st, a);
    D2P_HIP(hipGetLastError());
    return D2P_OK;
}

template <class T, bool BACK> int launch_type(const NormArgs& a, int v, int grid, hipStream_t st) {
    switch (v) {
        case 8:
            if constexpr (sizeof(T) == 2) return launch_as<T, 8, BACK>(a, grid, st);
        case 4: return launch_as<T, 4, BACK>(a, grid, st);
        case 2: return launch_as<T, 2, BACK>(a, grid, st);
        default: return launch_as<T, 1, BACK>(a, grid, st);
    }
}

// Lanes of a group, heads of a unit and the numbers of workgroups.
template <bool BACK> int plan(NormArgs& a, int v) {
    const d2p_qk_norm_rope_params& p = a.p;
    a.lanes = 1;
    while (a.lanes * v < p.D / 2) a.lanes *= 2;
    const int groups = THREADS<BACK> / a.lanes;
    const long long tokens = (long long)p.B * p.L;
    // all heads of a token where there are tokens enough to fill the card, one where not
    const long long fill = 512LL / a.lanes * std::max(device_cus(), 1);
    for (NormSide& s : a.side) {
        s.blocks = 0;
        if (s.heads == 0) continue;
        s.part = (int)std::min<long long>(s.heads, std::max<long long>(1, tokens * (p.Hq + p.Hkv) / fill));
        s.units_a_token = cdiv(s.heads, s.part);
        const long long want = (tokens * s.units_a_token + groups - 1) / groups;
        const long long most = BACK ? std::max<long long>(1, (long long)BACK_GROUPS * s.heads /
                                                                 (p.Hq + p.Hkv)) : 1 << 22;
        s.blocks = (int)std::min(want, most);
    }
    return a.side[0].blocks + a.side[1].blocks;
}

template <bool BACK> int launch(NormArgs& a, hipStream_t st) {
    const int v = run_width(a, BACK);
    const int grid = plan<BACK>(a, v);
    switch (a.p.dtype) {
        case D2P_FLOAT32: return launch_type<float, BACK>(a, v, grid, st);
        case D2P_FLOAT16: return launch_type<_Float16, BACK>(a, v, grid, st);
        default: return launch_type<__bf16, BACK>(a, v, grid, st);
    }
}

}  // namespace
}  // namespace enc
}  // namespace d2p_amd

using namespace d2p_amd;
using namespace d2p_amd::enc;

extern "C" int d2p_qk_norm_rope(const d2p_qk_norm_rope_params* p, const void* q, const void* k,
                                void* q_out, void* k_out, void* stream) {
    D2P_TRY(check(p));
    if ((long long)p->B * p->L * (p->Hq + p->Hkv) == 0) return D2P_OK;
    D2P_REQUIRE((p->Hq == 0 || (q && q_out)) && (p->Hkv == 0 || (k && k_out)),
                "null pointer argument");
    NormArgs a{};
    a.p = *p;
    a.side[0] = {q, nullptr, q_out, p->q, p->q, p->q_weight, p->Hq};
    a.side[1] = {k, nullptr, k_out, p->k, p->k, p->k_weight, p->Hkv};
    return launch<false>(a, (hipStream_t)stream);
}

extern "C" size_t d2p_qk_norm_rope_backward_workspace_bytes(const d2p_qk_norm_rope_params* p) {
    return p && p->B > 0 && p->L > 0 ? (size_t)(BACK_GROUPS + 2) * p->D * 4 : 0;
}

extern "C" int d2p_qk_norm_rope_backward(const d2p_qk_norm_rope_params* p, const void* gq,
                                         const void* gk, const void* q, const void* k, void* dq,
                                         void* dk, float* dq_weight, float* dk_weight,
                                         void* workspace, size_t workspace_bytes, void* stream) {
    D2P_TRY(check(p));
    hipStream_t st = (hipStream_t)stream;
    const bool weights = dq_weight || dk_weight;
    NormArgs a{};
    a.p = *p;
    if ((long long)p->B * p->L * (p->Hq + p->Hkv) != 0) {
        D2P_REQUIRE((p->Hq == 0 || (q && gq && dq)) && (p->Hkv == 0 || (k && gk && dk)),
                    "null pointer argument");
        D2P_REQUIRE(!weights || (workspace && workspace_bytes >=
                                 d2p_qk_norm_rope_backward_workspace_bytes(p)),
                    "workspace too small");
        a.side[0] = {q, gq, dq, p->q, p->gq, p->q_weight, p->Hq};
        a.side[1] = {k, gk, dk, p->k, p->gk, p->k_weight, p->Hkv};
        a.partial = weights ? (float*)workspace : nullptr;
        D2P_TRY(launch<true>(a, st));
    }
    if (!weights) return D2P_OK;
    // no rows: zeros
    D2P_LAUNCH("qk_norm_rope_weight_grad", weight_grad_kernel, dim3(2 * cdiv(p->D, 64)),
               dim3(1024), 0, st, (const float*)workspace, a.side[0].blocks, a.side[1].blocks,
               p->D, dq_weight, dk_weight);
    D2P_HIP(hipGetLastError());
    return D2P_OK;
}
