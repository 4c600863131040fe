// qk_norm_rope.hip -- root-mean-square norm of each head of queries and keys with the
// rotation by position in the same pass, and its gradients (include/d2p_amd_encoder.h).
//
// Bound by memory: each element is read once and written once.  A group of lanes holds one
// row (one token's one head): lane n of it the pairs VEC n .. VEC n + VEC - 1, as two runs
// of VEC neighbours, the pairs' first and second features, which one vector load each
// brings in.  A group walks over heads of one token, whose angles it keeps in registers.
#include <algorithm>

#include "encoder.hip.h"

namespace d2p_amd {
namespace enc {

struct NormArgs {
    d2p_qk_norm_rope_params p;
    const void *q, *k, *gq, *gk;
    void *oq, *ok;        // results (forward) or gradients of q, k (backward)
    float* partial;       // [workgroups][2][D]: sums for the weights' gradients
    int lanes;            // of a group, a power of two
    int chunks, heads;    // parts of a token's heads, heads of a part
    long long units;      // tokens * chunks
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
    float wq[2 * VEC], wk[2 * VEC];

    __device__ __forceinline__ Lane(const d2p_qk_norm_rope_params& p, int n) {
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
            wq[e] = on && p.q_weight ? p.q_weight[p0 + e] : 1.0f;
            wq[VEC + e] = on && p.q_weight ? p.q_weight[p1 + e] : 1.0f;
            wk[e] = on && p.k_weight ? p.k_weight[p0 + e] : 1.0f;
            wk[VEC + e] = on && p.k_weight ? p.k_weight[p1 + e] : 1.0f;
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

__device__ __forceinline__ float group_sum(float s, int lanes) {
    for (int o = lanes >> 1; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    return s;
}

template <class T>
__device__ __forceinline__ const T* row_of(const void* base, const d2p_strides& s, int b, int l,
                                           int h) {
    return (const T*)base + b * s.batch + l * s.row + h * s.head;
}

template <class T, int VEC, bool BACK>
__global__ void __launch_bounds__(256) qk_norm_rope_kernel(NormArgs a) {
    const d2p_qk_norm_rope_params& p = a.p;
    const int n = threadIdx.x & (a.lanes - 1);
    const int groups = 256 / a.lanes;
    const int D = p.D, H = p.Hq + p.Hkv;
    Lane<T, VEC> ln(p, n);
    float sq[2 * VEC] = {}, sk[2 * VEC] = {};   // the weights' gradients
    for (long long u = (long long)blockIdx.x * groups + threadIdx.x / a.lanes; u < a.units;
         u += (long long)gridDim.x * groups) {
        const long long token = u / a.chunks;
        const int b = (int)(token / p.L), l = (int)(token % p.L);
        const int h0 = (int)(u % a.chunks) * a.heads, h1 = min(h0 + a.heads, H);
        ln.angles(p, token, n);
        for (int h = h0; h < h1; ++h) {
            const bool isq = h < p.Hq;
            const int hh = isq ? h : h - p.Hq;
            const T* src = isq ? row_of<T>(a.q, p.q, b, l, hh) : row_of<T>(a.k, p.k, b, l, hh);
            T* dst = isq ? (T*)a.oq + (token * p.Hq + hh) * D : (T*)a.ok + (token * p.Hkv + hh) * D;
            Row<T, VEC> x, g;
            float ss = 0.0f;
            if (ln.on) {
                x.load(src, ln.p0, ln.p1);
                if (BACK)
                    g.load(isq ? row_of<T>(a.gq, p.gq, b, l, hh) : row_of<T>(a.gk, p.gk, b, l, hh),
                           ln.p0, ln.p1);
#pragma unroll
                for (int e = 0; e < 2 * VEC; ++e) ss += x.x[e] * x.x[e];
            }
            const float r = 1.0f / sqrtf(group_sum(ss, a.lanes) / D + p.eps);
            const float* w = isq ? ln.wq : ln.wk;
            if (!BACK) {
#pragma unroll
                for (int e = 0; e < 2 * VEC; ++e) x.x[e] *= r * w[e];
                ln.turn(x.x, 1.0f);
                if (ln.on) x.store(dst, ln.p0, ln.p1);
            } else {
                float dot = 0.0f;
                if (ln.on) {
                    ln.turn(g.x, -1.0f);
#pragma unroll
                    for (int e = 0; e < 2 * VEC; ++e) {
                        x.x[e] *= r;
                        const float t = g.x[e] * x.x[e];
                        if (isq) sq[e] += t; else sk[e] += t;
                        g.x[e] *= w[e];
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
        // the wave's groups, then the four waves, in one order
        __shared__ float sums[4][2][128];
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
        for (int e = 0; e < 2 * VEC; ++e)
            for (int o = 32; o >= a.lanes; o >>= 1) {
                sq[e] += __shfl_xor(sq[e], o, 64);
                sk[e] += __shfl_xor(sk[e], o, 64);
            }
        if (lane < a.lanes && ln.on) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                sums[wave][0][ln.p0 + e] = sq[e];
                sums[wave][0][ln.p1 + e] = sq[VEC + e];
                sums[wave][1][ln.p0 + e] = sk[e];
                sums[wave][1][ln.p1 + e] = sk[VEC + e];
            }
        }
        __syncthreads();
        const int which = threadIdx.x >> 7, d = threadIdx.x & 127;
        if (d < D)
            a.partial[((long long)blockIdx.x * 2 + which) * D + d] =
                sums[0][which][d] + sums[1][which][d] + sums[2][which][d] + sums[3][which][d];
    }
}

// dw[which][d] = sum over the workgroups: 64 columns a workgroup, 16 waves over the rows
__global__ void __launch_bounds__(1024)
weight_grad_kernel(const float* partial, int rows, int D, float* dwq, float* dwk) {
    __shared__ float part[16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int col = blockIdx.x * 64 + lane;
    float s = 0.0f;
    if (col < 2 * D)
        for (int r = wave; r < rows; r += 16) s += partial[(long long)r * 2 * D + col];
    part[wave][lane] = s;
    __syncthreads();
    if (wave || col >= 2 * D) return;
    s = 0.0f;
#pragma unroll
    for (int w = 0; w < 16; ++w) s += part[w][lane];
    if (col < D) { if (dwq) dwq[col] = s; }
    else if (dwk) dwk[col - D] = s;
}

namespace {

constexpr int BACK_GROUPS = 1024;   // workgroups of the backward pass at most

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
        uintptr_t at = (uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.oq | (uintptr_t)a.ok;
        if (back) at |= (uintptr_t)a.gq | (uintptr_t)a.gk;
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
               dim3(grid), dim3(256), 0, st, a);
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

// Lanes of a group, parts of a token's heads and the number of workgroups.
template <bool BACK> int plan(NormArgs& a, int v) {
    const d2p_qk_norm_rope_params& p = a.p;
    a.lanes = 1;
    while (a.lanes * v < p.D / 2) a.lanes *= 2;
    const int H = p.Hq + p.Hkv, groups = 256 / a.lanes;
    const long long tokens = (long long)p.B * p.L;
    // whole tokens where there are enough of them to fill the card, single heads where not
    const long long fill = 8LL * std::max(device_cus(), 1) * groups / 4;
    a.heads = (int)std::min<long long>(H, std::max<long long>(1, tokens * H / fill));
    a.chunks = cdiv(H, a.heads);
    a.units = tokens * a.chunks;
    const long long want = (a.units + groups - 1) / groups;
    return (int)std::min<long long>(want, BACK ? BACK_GROUPS : 0x7fffffffLL / 256);
}

template <bool BACK> int launch(NormArgs& a, int* grid, hipStream_t st) {
    const int v = run_width(a, BACK);
    *grid = plan<BACK>(a, v);
    switch (a.p.dtype) {
        case D2P_FLOAT32: return launch_type<float, BACK>(a, v, *grid, st);
        case D2P_FLOAT16: return launch_type<_Float16, BACK>(a, v, *grid, st);
        default: return launch_type<__bf16, BACK>(a, v, *grid, st);
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
    a.q = q; a.k = k; a.oq = q_out; a.ok = k_out;
    int grid;
    return launch<false>(a, &grid, (hipStream_t)stream);
}

extern "C" size_t d2p_qk_norm_rope_backward_workspace_bytes(const d2p_qk_norm_rope_params* p) {
    return p && p->B > 0 && p->L > 0 ? (size_t)BACK_GROUPS * 2 * p->D * 4 : 0;
}

extern "C" int d2p_qk_norm_rope_backward(const d2p_qk_norm_rope_params* p, const void* gq,
                                         const void* gk, const void* q, const void* k, void* dq,
                                         void* dk, float* dq_weight, float* dk_weight,
                                         void* workspace, size_t workspace_bytes, void* stream) {
    D2P_TRY(check(p));
    hipStream_t st = (hipStream_t)stream;
    const bool weights = dq_weight || dk_weight;
    int grid = 0;
    NormArgs a{};
    a.p = *p;
    if ((long long)p->B * p->L * (p->Hq + p->Hkv) != 0) {
        D2P_REQUIRE((p->Hq == 0 || (q && gq && dq)) && (p->Hkv == 0 || (k && gk && dk)),
                    "null pointer argument");
        D2P_REQUIRE(!weights || (workspace && workspace_bytes >=
                                 d2p_qk_norm_rope_backward_workspace_bytes(p)),
                    "workspace too small");
        a.q = q; a.k = k; a.gq = gq; a.gk = gk; a.oq = dq; a.ok = dk;
        a.partial = weights ? (float*)workspace : nullptr;
        D2P_TRY(launch<true>(a, &grid, st));
    }
    if (!weights) return D2P_OK;
    // no rows: zeros
    D2P_LAUNCH("qk_norm_rope_weight_grad", weight_grad_kernel, dim3(cdiv(2 * p->D, 64)),
               dim3(1024), 0, st, (const float*)workspace, grid, p->D, dq_weight, dk_weight);
    D2P_HIP(hipGetLastError());
    return D2P_OK;
}
