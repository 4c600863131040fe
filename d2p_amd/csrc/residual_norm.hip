// residual_norm.hip -- the norms before and after a block of a residual network with its gate
// and the stream around it, and their gradients (include/d2p_amd_training.h).
//
// Bound by memory: every tensor is read once and written once, rows stay in registers in
// between.  A team of lanes holds a row, eight numbers a lane; rows of more than 512 numbers
// take several waves, whose sums meet in LDS.  Teams walk over rows with the learned vectors
// in registers; in the backward pass each lane also keeps its features' sums for the vectors'
// gradients there, which a second kernel adds up over the workgroups.
#include <algorithm>
#include <type_traits>

#include "training.hip.h"

namespace d2p_amd {
namespace enc {

struct ResidualArgs {
    d2p_residual_norm_params p;
    const void *x, *y;
    void *h, *n;
    float* stats;
    int lanes;
};

// The learned vectors of a call in LDS, in 32 bits: `lanes` runs each, zeros behind D.  (In
// registers they would take the backward pass's waves from four a SIMD to two.)
struct Vectors {
    float* lds;
    int padded;                 // numbers of one vector

    __device__ __forceinline__ Vectors(float* lds_, int lanes) : lds(lds_), padded(lanes * RUN) {}
    __device__ __forceinline__ void load(int k, const d2p_vector& v, float other, int D) {
        for (int d = threadIdx.x; d < padded; d += blockDim.x)
            lds[k * padded + d] = d >= D ? 0.0f : v.data ? load_as(v.data, v.dtype, d) : other;
    }
    // (by the threads that loaded it)
    __device__ __forceinline__ void scale(int k, const d2p_vector& v, float by, int D) {
        for (int d = threadIdx.x; d < D; d += blockDim.x)
            lds[k * padded + d] *= by * (v.data ? load_as(v.data, v.dtype, d) : 1.0f);
    }
    // vector k of the lane whose run begins at `at`
    __device__ __forceinline__ void get(int k, int at, float* x) const {
        const f4v* p = (const f4v*)(lds + k * padded + at);
        const f4v lo = p[0], hi = p[1];
#pragma unroll
        for (int e = 0; e < 4; ++e) { x[e] = lo[e]; x[4 + e] = hi[e]; }
    }
};
// the forward pass keeps W, PW, PC and C, the backward pass FEATURE_GATE in C's place
enum Vector { W, PW, PC, C, FEATURE_GATE = C, VECTORS };
constexpr int SLOTS = 64;       // numbers of a Team's slots, at the start of the LDS

// v's mean (none for D2P_NORM_RMS) and 1 / sqrt(its spread + eps)
template <bool WIDE>
__device__ __forceinline__ float2 norm_stats(Team<WIDE>& team, int kind, const float* v, int left,
                                             int D, float eps) {
    float2 s = {0.0f, 0.0f};
    if (kind == D2P_NORM_LAYER) {
        s = team.spread(v, left, D);
    } else {
        float q = 0.0f;
#pragma unroll
        for (int e = 0; e < RUN; ++e) q += v[e] * v[e];
        s.y = team.sum(q);
    }
    return {s.x, 1.0f / sqrtf(s.y / D + eps)};
}

template <class T>
__device__ __forceinline__ const T* row_at(const void* base, const d2p_row_strides& s, int b,
                                           int l) {
    return (const T*)base + b * s.batch + l * s.row;
}

// a gate by sequence or token, in float32 or the block's type
template <class TY>
__device__ __forceinline__ void load_gate(const d2p_residual_norm_params& p, int b, int l, int at,
                                          int have, float* gate) {
    if (p.gate_dtype == p.block_dtype)
        load_run(row_at<TY>(p.gate, p.gate_strides, b, l) + at, have, gate);
    else
        load_run(row_at<float>(p.gate, p.gate_strides, b, l) + at, have, gate);
}

// TX: the stream's type; TY: the block's
// MOST: threads of a workgroup at most
template <class TX, class TY, bool BLOCK, int MOST>
__global__ void __launch_bounds__(MOST) residual_norm_kernel(ResidualArgs a) {
    constexpr bool WIDE = MOST > 256;
    extern __shared__ __align__(16) float lds[];
    const d2p_residual_norm_params& p = a.p;
    Team<WIDE> team(a.lanes, (float2*)lds);
    const int D = p.D, at = team.n * RUN, left = D - at;
    const int teams = blockDim.x / a.lanes;
    const unsigned rows = (unsigned)p.B * p.L;
    Vectors vec(lds + SLOTS, a.lanes);
    const bool by_row = p.gate_kind > D2P_GATE_FEATURE;
    if (p.norm != D2P_NORM_NONE) {
        vec.load(W, p.weight, 1.0f, D);
        vec.load(C, p.bias, 0.0f, D);
    }
    if (BLOCK) {
        // what is left of a row's own gate goes into the second norm's vectors
        const d2p_vector gate = {by_row ? nullptr : p.gate, p.gate_dtype};
        vec.load(PW, p.post_weight, 1.0f, D);
        vec.load(PC, p.post_bias, 0.0f, D);
        vec.scale(PW, gate, p.scale, D);
        vec.scale(PC, gate, p.scale, D);
    }
    __syncthreads();
    // (all teams of a workgroup take as many turns: they meet in their sums)
    for (unsigned base = blockIdx.x * teams; base < rows; base += gridDim.x * teams) {
        const unsigned row = base + threadIdx.x / a.lanes;
        const int have = row < rows ? left : 0;
        const int b = row / (unsigned)p.L, l = row % (unsigned)p.L;
        float v[RUN], x[RUN], w[RUN], c[RUN];
        float2 s = {0.0f, 0.0f}, ps = {0.0f, 0.0f};
        load_run(row_at<TX>(a.x, p.x, b, l) + at, have, x);
        if (BLOCK) {
            load_run(row_at<TY>(a.y, p.y, b, l) + at, have, v);
            if (by_row) load_gate<TY>(p, b, l, at, have, c);
            if (p.post_norm != D2P_NORM_NONE) {
                ps = norm_stats(team, p.post_norm, v, left, D, p.eps);
#pragma unroll
                for (int e = 0; e < RUN; ++e) v[e] = (v[e] - ps.x) * ps.y;
            }
            float pw[RUN], pc[RUN];
            vec.get(PW, at, pw);
            vec.get(PC, at, pc);
#pragma unroll
            for (int e = 0; e < RUN; ++e) {
                v[e] = v[e] * pw[e] + pc[e];
                if (by_row) v[e] *= c[e];
                x[e] = e < left ? p.residual_scale * x[e] + v[e] : 0.0f;
            }
            store_run((TX*)a.h + (long long)row * D + at, have, x);
        }
        if (p.norm != D2P_NORM_NONE) {
            s = norm_stats(team, p.norm, x, left, D, p.eps);
            vec.get(W, at, w);
            vec.get(C, at, c);
#pragma unroll
            for (int e = 0; e < RUN; ++e) v[e] = (x[e] - s.x) * s.y * w[e] + c[e];
            store_run((TY*)a.n + (long long)row * D + at, have, v);
        }
        if (a.stats && team.n == 0 && row < rows)
            *(f4v*)(a.stats + 4 * (long long)row) = f4v{s.x, s.y, ps.x, ps.y};
    }
}

// ---------------------------------------------------------------------------
// backward
// ---------------------------------------------------------------------------
enum Sum { WEIGHT, BIAS, POST_WEIGHT, POST_BIAS, GATE, SUMS };

struct ResidualBackArgs {
    d2p_residual_norm_params p;
    const void *dh, *dn, *h, *y;
    const float* stats;
    void *dx, *dy, *dgate;
    float* partial[SUMS];   // [workgroups][D]; the gate's: [segments][D]; null: not wanted
    int lanes;
    int batches, length;    // rows as segments are cut from them: [B, L], or [1, B L]
    int splits;             // segments of `length` rows
};

// The team's numbers of one feature summed over the workgroup's teams, into dst [D].
__device__ __forceinline__ void flush(float* lds, const float* sums, float* dst, int lanes, int D) {
    const int at = (threadIdx.x & (lanes - 1)) * RUN;
    if ((int)blockDim.x == lanes) {
        store_run(dst + at, D - at, sums);
        return;
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < RUN; ++e) lds[threadIdx.x * RUN + e] = sums[e];
    __syncthreads();
    for (int d = threadIdx.x; d < D; d += blockDim.x) {
        float s = 0.0f;
        for (int t = 0; t < (int)blockDim.x; t += lanes) s += lds[t * RUN + d];
        dst[d] = s;
    }
}

template <class TX, class TY, bool BLOCK, int MOST>
__global__ void __launch_bounds__(MOST) residual_norm_backward_kernel(ResidualBackArgs a) {
    constexpr bool WIDE = MOST > 256;
    // the teams' slots; the vectors; then, for the teams' sums, eight numbers a thread
    extern __shared__ __align__(16) float lds[];
    const d2p_residual_norm_params& p = a.p;
    Team<WIDE> team(a.lanes, (float2*)lds);
    const int D = p.D, at = team.n * RUN, left = D - at;
    const int teams = blockDim.x / a.lanes;
    Vectors vec(lds + SLOTS, a.lanes);
    const bool by_row = p.gate_kind > D2P_GATE_FEATURE, post = p.post_norm != D2P_NORM_NONE;
    if (a.dn) vec.load(W, p.weight, 1.0f, D);
    if (BLOCK) {
        vec.load(PW, p.post_weight, 1.0f, D);
        vec.load(PC, p.post_bias, 0.0f, D);
        if (!by_row) vec.load(FEATURE_GATE, {p.gate, p.gate_dtype}, 1.0f, D);
    }
    __syncthreads();
    float sums[SUMS][RUN] = {};
    const int segments = a.batches * a.splits;
    for (int seg = blockIdx.x; seg < segments; seg += gridDim.x) {
        const int part = seg % a.splits;
        const unsigned start = (unsigned)(seg / a.splits) * (unsigned)a.length;
        const unsigned r0 = start + (unsigned)((long long)a.length * part / a.splits);
        const unsigned r1 = start + (unsigned)((long long)a.length * (part + 1) / a.splits);
        for (unsigned base = r0; base < r1; base += teams) {
            const unsigned row = base + threadIdx.x / a.lanes;
            const int have = row < r1 ? left : 0;
            const int b = row / (unsigned)p.L, l = row % (unsigned)p.L;
            const long long flat = (long long)row * D + at;
            float H[RUN], dn[RUN], hh[RUN], y[RUN], gate[RUN], w[RUN];
            f4v st = {};
            if (a.stats && row < r1) st = *(const f4v*)(a.stats + 4 * (long long)row);
            load_run(row_at<TX>(a.dh, p.dh, b, l) + at, a.dh ? have : 0, H);
            if (a.dn) {
                load_run(row_at<TY>(a.dn, p.dn, b, l) + at, have, dn);
                load_run(row_at<TX>(a.h, p.x, b, l) + at, have, hh);
            }
            if (BLOCK) {
                load_run(row_at<TY>(a.y, p.y, b, l) + at, a.y ? have : 0, y);
                if (by_row) load_gate<TY>(p, b, l, at, have, gate);
            }
            if (a.dn) {
                float2 m = {0.0f, 0.0f};
                vec.get(W, at, w);
#pragma unroll
                for (int e = 0; e < RUN; ++e) {
                    hh[e] = (hh[e] - st[0]) * st[1];
                    sums[WEIGHT][e] += dn[e] * hh[e];
                    sums[BIAS][e] += dn[e];
                    dn[e] *= w[e];
                    m.x += dn[e];
                    m.y += dn[e] * hh[e];
                }
                if (p.norm == D2P_NORM_LAYER) m = team.sum(m.x, m.y);
                else m = {0.0f, team.sum(m.y)};
                m.x /= D;
                m.y /= D;
#pragma unroll
                for (int e = 0; e < RUN; ++e)
                    H[e] = e < have ? H[e] + st[1] * (dn[e] - m.x - hh[e] * m.y) : 0.0f;
            }
            float dx[RUN];
#pragma unroll
            for (int e = 0; e < RUN; ++e) dx[e] = p.residual_scale * H[e];
            store_run((TX*)a.dx + flat, have, dx);
            if (!BLOCK) continue;       // no y, or its gradient is x's
            float2 m = {0.0f, 0.0f};
            float dgate[RUN], pc[RUN];
            if (!by_row) vec.get(FEATURE_GATE, at, gate);
            if (post) {
                vec.get(PW, at, w);
                vec.get(PC, at, pc);
            }
#pragma unroll
            for (int e = 0; e < RUN; ++e) {
                if (post) y[e] = e < have ? (y[e] - st[2]) * st[3] : 0.0f;
                H[e] *= p.scale;
                dgate[e] = H[e] * (post ? y[e] * w[e] + pc[e] : y[e]);
                sums[GATE][e] += dgate[e];
                H[e] *= gate[e];
                if (post) {
                    sums[POST_WEIGHT][e] += H[e] * y[e];
                    sums[POST_BIAS][e] += H[e];
                    H[e] *= w[e];
                    m.x += H[e];
                    m.y += H[e] * y[e];
                }
            }
            if (a.dgate && p.gate_kind == D2P_GATE_TOKEN) {
                if (p.gate_dtype == p.block_dtype) store_run((TY*)a.dgate + flat, have, dgate);
                else store_run((float*)a.dgate + flat, have, dgate);
            }
            if (post) {
                if (p.post_norm == D2P_NORM_LAYER) m = team.sum(m.x, m.y);
                else m = {0.0f, team.sum(m.y)};
                m.x /= D;
                m.y /= D;
#pragma unroll
                for (int e = 0; e < RUN; ++e) H[e] = st[3] * (H[e] - m.x - y[e] * m.y);
            }
            store_run((TY*)a.dy + flat, have, H);
        }
        if (BLOCK && a.partial[GATE]) {
            flush(lds + SLOTS + VECTORS * vec.padded, sums[GATE], a.partial[GATE] + (long long)seg * D, a.lanes, D);
#pragma unroll
            for (int e = 0; e < RUN; ++e) sums[GATE][e] = 0.0f;
        }
    }
#pragma unroll
    for (int k = 0; k < GATE; ++k)
        if ((BLOCK || k < POST_WEIGHT) && a.partial[k])
            flush(lds + SLOTS + VECTORS * vec.padded, sums[k], a.partial[k] + (long long)blockIdx.x * D, a.lanes, D);
}

namespace {

constexpr int MOST_GROUPS = 1024;   // workgroups of the backward pass at most

int check_vector(const d2p_vector& v) {
    D2P_REQUIRE(!v.data || known_type(v.dtype), "unknown element type of a learned vector");
    return D2P_OK;
}

int check(const d2p_residual_norm_params* p) {
    D2P_REQUIRE(p != nullptr, "null parameters");
    D2P_REQUIRE(known_pair(p->dtype, p->block_dtype),
                "unknown element types, or a pair other than equal ones and 16 bits beside float32");
    D2P_REQUIRE(p->B >= 0 && p->L >= 0, "negative size");
    D2P_REQUIRE((long long)p->B * p->L < 1LL << 31, "too many rows");
    D2P_REQUIRE(p->D >= 1 && p->D <= 8192, "features must be between 1 and 8192");
    for (int kind : {p->norm, p->post_norm})
        D2P_REQUIRE(kind >= D2P_NORM_NONE && kind <= D2P_NORM_LAYER, "unknown norm");
    for (const d2p_vector* v : {&p->weight, &p->bias, &p->post_weight, &p->post_bias})
        D2P_TRY(check_vector(*v));
    D2P_REQUIRE(p->gate_kind >= D2P_GATE_NONE && p->gate_kind <= D2P_GATE_TOKEN, "unknown gate");
    D2P_REQUIRE(p->gate_kind == D2P_GATE_NONE || p->gate_dtype == D2P_FLOAT32 ||
                    p->gate_dtype == p->block_dtype,
                "the gate must be float32 or of the block's type");
    D2P_REQUIRE(p->gate_kind == D2P_GATE_NONE || (long long)p->B * p->L == 0 || p->gate,
                "null pointer argument");
    D2P_REQUIRE(p->eps >= 0.0f, "eps must not be negative");
    return D2P_OK;
}

// Strides of a gate that has one number for several rows say nothing.
d2p_row_strides gate_steps(const d2p_residual_norm_params& p) {
    return {p.gate_kind >= D2P_GATE_SEQUENCE ? p.gate_strides.batch : 0,
            p.gate_kind == D2P_GATE_TOKEN ? p.gate_strides.row : 0};
}

int threads_of(int lanes) { return std::max(lanes, 256); }
// LDS of the teams' slots, the vectors and, in a backward pass of more teams than one, of their sums
size_t lds_bytes(int lanes, bool back) {
    return (SLOTS + (VECTORS * lanes + (back && lanes < 256 ? 256 : 0)) * RUN) * sizeof(float);
}

template <class Args>
int launch(const char* name, void (*kernel)(Args), LdsAllowed& known, const Args& a, int grid,
           bool back, hipStream_t st) {
    D2P_TRY(allow_lds((const void*)kernel, known));
    D2P_LAUNCH(name, kernel, dim3(grid), dim3(threads_of(a.lanes)), lds_bytes(a.lanes, back), st, a);
    D2P_HIP(hipGetLastError());
    return D2P_OK;
}
template <class TX, class TY, bool BLOCK, int MOST>
int launch_forward(const ResidualArgs& a, int grid, hipStream_t st) {
    static LdsAllowed known;
    return launch("residual_norm", residual_norm_kernel<TX, TY, BLOCK, MOST>, known, a, grid, false,
                  st);
}
template <class TX, class TY, bool BLOCK, int MOST>
int launch_backward(const ResidualBackArgs& a, int grid, hipStream_t st) {
    static LdsAllowed known;
    return launch("residual_norm_backward", residual_norm_backward_kernel<TX, TY, BLOCK, MOST>,
                  known, a, grid, true, st);
}

// f(threads of a workgroup at most): rows within a wave, or of waves that leave a thread 256
// registers, or of more
template <class F> int by_lanes(int lanes, F f) {
    return lanes <= 64    ? f(std::integral_constant<int, 256>{})
           : lanes <= 512 ? f(std::integral_constant<int, 512>{})
                          : f(std::integral_constant<int, 1024>{});
}

// How the backward pass cuts rows into segments: at most MOST_GROUPS of them, four turns of a
// workgroup at least, and each of one sequence where the gate's gradient is by sequence.
struct Cut {
    int batches, length, splits, grid;
    Cut(const d2p_residual_norm_params& p, int lanes) {
        const int teams = threads_of(lanes) / lanes;
        const bool by_sequence = p.gate_kind == D2P_GATE_SEQUENCE;
        batches = by_sequence ? p.B : 1;
        length = by_sequence ? p.L : p.B * p.L;
        const int most = std::max(1, MOST_GROUPS / std::max(batches, 1));
        splits = std::min(most, std::max(1, length / (4 * teams)));
        grid = (int)std::min<long long>((long long)batches * splits, MOST_GROUPS);
    }
};

}  // namespace
}  // namespace enc
}  // namespace d2p_amd

using namespace d2p_amd;
using namespace d2p_amd::enc;

extern "C" int d2p_residual_norm(const d2p_residual_norm_params* p, const void* x, const void* y,
                                 void* h, void* n, float* stats, void* stream) {
    D2P_TRY(check(p));
    if ((long long)p->B * p->L == 0) return D2P_OK;
    D2P_REQUIRE(x && (p->norm == D2P_NORM_NONE || n), "null pointer argument");
    D2P_REQUIRE(!y == !h && !y == !p->with_y, "with_y, y and h go together");
    D2P_REQUIRE(y || (p->post_norm == D2P_NORM_NONE && p->gate_kind == D2P_GATE_NONE),
                "a gate or a second norm needs y");
    ResidualArgs a{*p, x, y, h, n, stats, team_of(p->D)};
    a.p.gate_strides = gate_steps(*p);
    const int teams = threads_of(a.lanes) / a.lanes;
    const int most = 8 * 256 * std::max(device_cus(), 1) / threads_of(a.lanes);
    const int grid = std::min(cdiv(p->B * p->L, teams), most);
    return with_pair(p->dtype, p->block_dtype, [&](auto tx, auto ty) {
        using TX = typename decltype(tx)::type;
        using TY = typename decltype(ty)::type;
        const auto st = (hipStream_t)stream;
        return y ? by_lanes(a.lanes, [&](auto most) {
                       return launch_forward<TX, TY, true, most()>(a, grid, st);
                   })
                 : by_lanes(a.lanes, [&](auto most) {
                       return launch_forward<TX, TY, false, most()>(a, grid, st);
                   });
    });
}

extern "C" size_t d2p_residual_norm_backward_workspace_bytes(const d2p_residual_norm_params* p) {
    if (!p || p->B < 0 || p->L < 0 || p->D < 1 || p->D > 8192 || (long long)p->B * p->L >= 1LL << 31)
        return 0;
    const Cut cut(*p, team_of(p->D));
    const size_t gate = p->gate_kind == D2P_GATE_FEATURE || p->gate_kind == D2P_GATE_SEQUENCE
                            ? (size_t)cut.batches * cut.splits : 0;
    return ((size_t)GATE * cut.grid + gate) * p->D * 4;
}

extern "C" int d2p_residual_norm_backward(const d2p_residual_norm_params* p, const void* dh,
                                          const void* dn, const void* h, const void* y,
                                          const float* stats, void* dx, void* dy, void* dgate,
                                          void* dweight, void* dbias, void* dpost_weight,
                                          void* dpost_bias, void* workspace,
                                          size_t workspace_bytes, void* stream) {
    D2P_TRY(check(p));
    const bool rows = (long long)p->B * p->L > 0;
    const bool norm = dn && p->norm != D2P_NORM_NONE;
    if (rows) {
        D2P_REQUIRE(dx && (!norm || (h && stats)), "null pointer argument");
        D2P_REQUIRE(p->post_norm == D2P_NORM_NONE || (y && stats), "null pointer argument");
        D2P_REQUIRE(!dgate || y, "the gate's gradient needs y");
        D2P_REQUIRE(dy || (p->post_norm == D2P_NORM_NONE && p->gate_kind == D2P_GATE_NONE &&
                           (!p->with_y || (p->scale == p->residual_scale &&
                                           p->dtype == p->block_dtype))),
                    "dy is not dx with a gate, a second norm, or scales or types that differ");
        D2P_REQUIRE(p->with_y || !dy, "dy needs y");
        D2P_REQUIRE(((uintptr_t)stats & 15) == 0, "stats must be aligned to 16 bytes");
    }
    D2P_REQUIRE(workspace_bytes >= d2p_residual_norm_backward_workspace_bytes(p) && workspace,
                "workspace too small");
    ResidualBackArgs a{};
    a.p = *p;
    a.p.gate_strides = gate_steps(*p);
    // h lies as the forward pass wrote it; without y it is x
    if (p->with_y) a.p.x = {(long long)p->L * p->D, p->D};
    else a.p.residual_scale = 1.0f;
    a.dh = dh;
    a.dn = norm ? dn : nullptr;
    a.h = h;
    a.y = y;
    a.stats = stats;
    a.dx = dx;
    a.dy = dy;
    a.dgate = dgate;
    a.lanes = team_of(p->D);
    const Cut cut(*p, a.lanes);
    a.batches = cut.batches;
    a.length = cut.length;
    a.splits = cut.splits;
    float* ws = (float*)workspace;
    void* const out[] = {dweight, dbias, dpost_weight, dpost_bias, dgate};
    const int type[] = {p->weight.dtype, p->bias.dtype, p->post_weight.dtype, p->post_bias.dtype,
                        p->gate_dtype};
    SumJobs jobs;
    jobs.init(p->D);
    for (int k = 0; k < SUMS; ++k) {
        if (!out[k] || (k == GATE && p->gate_kind == D2P_GATE_TOKEN)) continue;
        const bool gate = k == GATE;
        D2P_REQUIRE(known_type(type[k]), "unknown element type of a learned vector");
        a.partial[k] = ws;
        const int count = gate ? cut.splits : cut.grid, groups = gate ? cut.batches : 1;
        D2P_REQUIRE((long long)groups * jobs.tiles + jobs.blocks < 1LL << 31, "too many sequences");
        jobs.add(ws, out[k], type[k], rows ? count : 0, groups);
        ws += (size_t)count * groups * p->D;
    }
    if (rows)
        D2P_TRY(with_pair(p->dtype, p->block_dtype, [&](auto tx, auto ty) {
            using TX = typename decltype(tx)::type;
            using TY = typename decltype(ty)::type;
            const auto st = (hipStream_t)stream;
            return dy ? by_lanes(a.lanes, [&](auto most) {
                            return launch_backward<TX, TY, true, most()>(a, cut.grid, st);
                        })
                      : by_lanes(a.lanes, [&](auto most) {
                            return launch_backward<TX, TY, false, most()>(a, cut.grid, st);
                        });
        }));
    return launch_sum_rows("residual_norm_vector_grads", jobs, (hipStream_t)stream);
}
