// residual_norm.hip -- the norms before and after a block of a residual network with its gate
// and the stream around it, and their gradients (include/d2p_amd_training.h).
//
// Bound by memory: every tensor is read once and written once, rows stay in registers in
// between.  A team of lanes holds a row, eight numbers a lane; rows of more than 512 numbers
// take several waves, whose sums meet in LDS.  Teams walk over rows with the learned vectors
// in LDS; in the backward pass each lane keeps its features' sums for the vectors' gradients in
// registers, which a second kernel adds up over the workgroups.
//
// With r = 1 / sqrt(spread + eps) and v' = (v - mean) r the gradient of v' w + b through to v is
//   r (a - mean(a) - v' mean(a v')),  a = dn w          (for an RMS norm without mean(a))
// so that a row's backward pass needs its statistics (kept by the forward pass) and two sums.
//
// bf16, no gate or second norm: [131072, 512] forward 105 us, 5.1 TB/s, backward 130 us, 5.2 (a copy
// of as much: 5.2); [32768, 2048] 103 and 133 us; 333 features, of which rows begin at odd
// addresses and the team's 64 lanes have 42 at work, 4.2 and 3.8 TB/s.  float32 beside bf16, RMS on
// both sides and a gate by feature, [65536, 512]: 84 us, 4.8 TB/s, and 122 us, 5.0.
//   LDS, not registers, for the vectors: four waves a SIMD in the backward pass instead of two.
//   All loads of a row before the first is used, in no branch: [131072, 512] 114 -> 105 us and 155
//   -> 130.
//   The next row's loads ahead of this row's stores: within 2 % for 16 bits, and for float32
//   beside bf16 122 -> 134 us, since the registers do not suffice.
//   Forward loads past the caches: 105 -> 91 us for the kernel by itself, but 283 -> 295 for [4,
//   8192, 2048] with its backward pass, which reads x and y again.
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
    Divisor by_length;
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
// the forward pass keeps W, PW, PC and C; the backward pass, in C's place, what of scale * gate all
// rows have alike
enum Vector { W, PW, PC, C, GATED = C, VECTORS };
constexpr int SLOTS = 64;       // numbers of a Team's slots, at the start of the LDS

// v's mean (none for D2P_NORM_RMS) and 1 / sqrt(its spread + eps)
template <bool WIDE>
__device__ __forceinline__ float2 norm_stats(Team<WIDE>& team, int kind, const float* v,
                                             const float* there, int D, float eps) {
    float2 s = {0.0f, 0.0f};
    if (kind == D2P_NORM_LAYER) {
        s = team.spread(v, there, D);
    } else {
        float q = 0.0f;
#pragma unroll
        for (int e = 0; e < RUN; ++e) q += v[e] * v[e];
        s.y = team.sum(q);
    }
    return {s.x, inverse_root(divided(s.y, (float)D) + eps)};
}

// Where a row begins, and a lane's run in it.
struct Place {
    const d2p_residual_norm_params& p;
    unsigned b, l;
    int at;
    long long flat;     // the row in a contiguous tensor

    __device__ __forceinline__ Place(const d2p_residual_norm_params& p_, const Divisor& by_length,
                                     unsigned row, int at_)
        : p(p_), at(at_), flat((long long)row * p_.D) {
        b = by_length(row);
        l = row - b * p.L;
    }
    // (the strides of a contiguous tensor are told apart once for all lanes)
    template <class T>
    __device__ __forceinline__ const T* in(const void* base, const d2p_row_strides& s) const {
        const bool dense = s.row == p.D && s.batch == (long long)p.L * p.D;
        return (const T*)base + (dense ? flat : (long long)b * s.batch + (long long)l * s.row);
    }
};

// a gate by sequence or token, in float32 or the block's type
template <class TY, bool EVEN> struct GateRun {
    Eight<float> wide;
    Eight<TY> narrow;

    __device__ __forceinline__ void load(const Place& place) {
        const d2p_residual_norm_params& p = place.p;
        if (sizeof(TY) == 4 || p.gate_dtype == D2P_FLOAT32)
            wide = load_run(place.in<float>(p.gate, p.gate_strides), place.at, p.D);
        else
            narrow = load_run(place.in<TY>(p.gate, p.gate_strides), place.at, p.D);
    }
    __device__ __forceinline__ void get(const Place& place, bool wanted, float* x) const {
        const d2p_residual_norm_params& p = place.p;
        if (sizeof(TY) == 4 || p.gate_dtype == D2P_FLOAT32)
            unpack<EVEN>(wide, place.at, p.D, wanted, x);
        else
            unpack<EVEN>(narrow, place.at, p.D, wanted, x);
    }
};

// EVEN: rows of whole runs; MOST: threads of a workgroup at most
template <class TX, class TY, bool BLOCK, bool EVEN, int MOST>
__global__ void __launch_bounds__(MOST) residual_norm_kernel(ResidualArgs a) {
    constexpr bool WIDE = MOST > 256;
    extern __shared__ __align__(16) float lds[];
    const d2p_residual_norm_params& p = a.p;
    Team<WIDE> team(a.lanes, (float2*)lds);
    const int D = p.D, at = team.n * RUN, left = D - at;
    const int teams = blockDim.x / a.lanes;
    const unsigned rows = (unsigned)p.B * p.L;
    Vectors vec(lds + SLOTS, a.lanes);
    // A gate by feature goes into the weight that z is made with.  Beside a bias it is taken as a
    // row's own gate is, from one row of no stride: an infinite one times w and times b may be
    // infinities of opposite sign, where times w v + b it is one.
    const bool by_row = p.gate_kind > D2P_GATE_FEATURE ||
                        (p.gate_kind == D2P_GATE_FEATURE && p.post_bias.data);
    if (p.norm != D2P_NORM_NONE) {
        vec.load(W, p.weight, 1.0f, D);
        vec.load(C, p.bias, 0.0f, D);
    }
    if (BLOCK) {
        vec.load(PW, p.post_weight, 1.0f, D);
        vec.load(PC, p.post_bias, 0.0f, D);
        vec.scale(PW, {by_row ? nullptr : p.gate, p.gate_dtype}, p.scale, D);
        vec.scale(PC, {}, p.scale, D);
    }
    __syncthreads();
    float there[RUN];
#pragma unroll
    for (int e = 0; e < RUN; ++e) there[e] = e < left ? 1.0f : 0.0f;
    // (all teams of a workgroup take as many turns: they meet in their sums.  Behind a row's end
    // all is zero: what is loaded, and the vectors that it is multiplied with)
    for (unsigned base = blockIdx.x * teams; base < rows; base += gridDim.x * teams) {
        const unsigned row = base + threadIdx.x / a.lanes;
        const int have = row < rows ? left : 0;
        // (a team that is left over reads the last row again)
        const Place place(p, a.by_length, min(row, rows - 1), at);
        const int vat = fresh(at, base);    // the vectors are read anew, not kept in registers
        float v[RUN], x[RUN], w[RUN], c[RUN];
        float2 s = {0.0f, 0.0f}, ps = {0.0f, 0.0f};
        const Eight<TX> rx = load_run(place.in<TX>(a.x, p.x), at, D);
        Eight<TY> ry;
        GateRun<TY, EVEN> rg;
        if (BLOCK) {
            ry = load_run(place.in<TY>(a.y, p.y), at, D);
            if (by_row) rg.load(place);
        }
        unpack<EVEN>(rx, at, D, true, x);
        if (BLOCK) {
            unpack<EVEN>(ry, at, D, true, v);
            if (by_row) rg.get(place, true, c);
            if (p.post_norm != D2P_NORM_NONE) {
                ps = norm_stats(team, p.post_norm, v, there, D, p.eps);
#pragma unroll
                for (int e = 0; e < RUN; ++e) v[e] = (v[e] - ps.x) * ps.y;
            }
            float pw[RUN], pc[RUN];
            vec.get(PW, vat, pw);
            vec.get(PC, vat, pc);
#pragma unroll
            for (int e = 0; e < RUN; ++e) {
                v[e] = v[e] * pw[e] + pc[e];
                if (by_row) v[e] *= c[e];
                x[e] = p.residual_scale * x[e] + v[e];
            }
            store_run((TX*)a.h + place.flat + at, have, x);
        }
        if (p.norm != D2P_NORM_NONE) {
            s = norm_stats(team, p.norm, x, there, D, p.eps);
            vec.get(W, vat, w);
            vec.get(C, vat, c);
#pragma unroll
            for (int e = 0; e < RUN; ++e) v[e] = (x[e] - s.x) * s.y * w[e] + c[e];
            store_run((TY*)a.n + place.flat + at, have, v);
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
    const void *dh, *dn, *stream, *y;   // stream: h for float32, x for 16 bits or without y
    const float* stats;
    bool has_dh, has_dn, has_y;         // elsewise the pointer is to something else, of no stride
    long long stats_step;               // 4, or 0 without stats
    void *dx, *dy, *dgate;
    float* partial[SUMS];   // [workgroups][D]; the gate's: [segments][D]; null: not wanted
    int lanes;
    Divisor by_length;
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

// Waves a SIMD that the backward pass's registers are held to: four, but three where h is formed
// again and the biases' sums are kept too.  That is for rows within a wave; the kernels of longer
// rows are built for workgroups of up to 1024 threads, four waves a SIMD, and there keep a few
// registers in scratch.  As many workgroups as that leaves room for: fp16 [5, 1023, 333], layer norms
// and a gate by token, kernel 30 -> 20 us; bf16 [131072, 512], layer and RMS norm, 200 -> 165.
constexpr int ONE_WAVE = 256, MORE_WAVES = 1024;    // threads of a workgroup at most (MOST)
constexpr int BACK_WAVES = 4;
__host__ __device__ constexpr int back_waves(bool again, bool biases, int most) {
    return again && biases && most == ONE_WAVE ? 3 : BACK_WAVES;
}

// BLOCK: y has a gradient of its own (or, in 16 bits, h is formed from it again); BIASES: some
// bias wants its gradient
template <class TX, class TY, bool BLOCK, bool BIASES, bool EVEN, int MOST>
__global__ void __launch_bounds__(MOST, back_waves(BLOCK && sizeof(TX) == 2, BIASES, MOST))
residual_norm_backward_kernel(ResidualBackArgs a) {
    constexpr bool WIDE = MOST > 256, AGAIN = BLOCK && sizeof(TX) == 2;
    // the teams' slots; the vectors; then, for the teams' sums, eight numbers a thread
    extern __shared__ __align__(16) float lds[];
    const d2p_residual_norm_params& p = a.p;
    Team<WIDE> team(a.lanes, (float2*)lds);
    const int D = p.D, at = team.n * RUN, left = D - at;
    const int teams = blockDim.x / a.lanes;
    Vectors vec(lds + SLOTS, a.lanes);
    const bool by_row = p.gate_kind > D2P_GATE_FEATURE, post = p.post_norm != D2P_NORM_NONE;
    if (a.has_dn) vec.load(W, p.weight, 1.0f, D);
    if (BLOCK) {
        vec.load(PW, p.post_weight, 1.0f, D);
        vec.load(PC, p.post_bias, 0.0f, D);
        vec.load(GATED, {by_row ? nullptr : p.gate, p.gate_dtype}, 1.0f, D);
        vec.scale(GATED, {}, p.scale, D);
    }
    __syncthreads();
    // Behind a row's end H is no zero after n's norm, but then meets vectors that are.
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
            // (a team that is left over reads the last row again, and adds zeros)
            // (what a lane's place in the row gives is computed in each turn: kept, it would
            // take more registers than there are)
            const int vat = fresh(at, base);
            const Place place(p, a.by_length, min(row, r1 - 1), vat);
            const long long flat = place.flat + vat;
            float H[RUN], dn[RUN], hh[RUN], y[RUN], gate[RUN], w[RUN], c[RUN];
            // (what is not there is read all the same, from one row of something else that is, and
            // taken for zeros: no load waits for a branch.  Past the caches, since nothing is read
            // after this: bf16 [4, 8192, 2048], both passes, 293 -> 282 us)
            Eight<TY> ry;
            GateRun<TY, EVEN> rg;
            f4v st = *(const f4v*)(a.stats + a.stats_step * min(row, r1 - 1));
            const Eight<TX> rdh = load_run<true>(place.in<TX>(a.dh, p.dh), vat, D);
            const Eight<TY> rdn = load_run<true>(place.in<TY>(a.dn, p.dn), vat, D);
            const Eight<TX> rs = load_run<true>(place.in<TX>(a.stream, p.x), vat, D);
            if (BLOCK) {
                ry = load_run<true>(place.in<TY>(a.y, p.y), vat, D);
                if (by_row) rg.load(place);
            }
            const bool there = row < r1;
            if (BLOCK) {
                // without a norm of its own z is y: mean 0, one over the spread 1, weight 1, bias 0
                st[2] = post ? st[2] : 0.0f;
                st[3] = post ? st[3] : 1.0f;
                unpack<EVEN>(ry, vat, D, there && a.has_y, y);
#pragma unroll
                for (int e = 0; e < RUN; ++e) y[e] = (y[e] - st[2]) * st[3];
            }
            if (a.has_dn) {
                unpack<EVEN>(rs, vat, D, there, hh);
                if (AGAIN) {
                    vec.get(PW, vat, w);
                    vec.get(PC, vat, c);
#pragma unroll
                    for (int e = 0; e < RUN; ++e) w[e] = y[e] * w[e] + c[e];
                    vec.get(GATED, vat, c);
                    if (by_row) {
                        rg.get(place, there, gate);
#pragma unroll
                        for (int e = 0; e < RUN; ++e) c[e] *= gate[e];
                    }
#pragma unroll
                    for (int e = 0; e < RUN; ++e) hh[e] = p.residual_scale * hh[e] + c[e] * w[e];
                }
                float2 m = {0.0f, 0.0f};
                vec.get(W, vat, w);
                unpack<EVEN>(rdn, vat, D, there, dn);
#pragma unroll
                for (int e = 0; e < RUN; ++e) {
                    hh[e] = (hh[e] - st[0]) * st[1];
                    sums[WEIGHT][e] += dn[e] * hh[e];
                    if (BIASES) sums[BIAS][e] += dn[e];
                    dn[e] *= w[e];
                    m.x += dn[e];
                    m.y += dn[e] * hh[e];
                }
                if (p.norm == D2P_NORM_LAYER) m = team.sum(m.x, m.y);
                else m = {0.0f, team.sum(m.y)};
                m.x = divided(m.x, (float)D);
                m.y = divided(m.y, (float)D);
                unpack<EVEN>(rdh, vat, D, there && a.has_dh, H);
#pragma unroll
                for (int e = 0; e < RUN; ++e) H[e] += st[1] * (dn[e] - m.x - hh[e] * m.y);
            } else {
                unpack<EVEN>(rdh, vat, D, there && a.has_dh, H);
            }
#pragma unroll
            for (int e = 0; e < RUN; ++e) c[e] = p.residual_scale * H[e];
            store_run((TX*)a.dx + flat, have, c);
            if (!BLOCK || !a.dy) continue;      // no y, or its gradient is x's
            if (a.dgate) {
                vec.get(PW, vat, w);
                vec.get(PC, vat, c);
#pragma unroll
                for (int e = 0; e < RUN; ++e) {
                    c[e] = p.scale * H[e] * (y[e] * w[e] + c[e]);
                    sums[GATE][e] += c[e];
                }
                if (p.gate_kind == D2P_GATE_TOKEN) {
                    if (p.gate_dtype == D2P_FLOAT32) store_run((float*)a.dgate + flat, have, c);
                    else store_run((TY*)a.dgate + flat, have, c);
                }
            }
            vec.get(GATED, vat, c);
            if (by_row) {
                rg.get(place, there, gate);
#pragma unroll
                for (int e = 0; e < RUN; ++e) c[e] *= gate[e];
            }
#pragma unroll
            for (int e = 0; e < RUN; ++e) H[e] *= c[e];
            if (post) {
                float2 m = {0.0f, 0.0f};
                vec.get(PW, vat, w);
#pragma unroll
                for (int e = 0; e < RUN; ++e) {
                    sums[POST_WEIGHT][e] += H[e] * y[e];
                    if (BIASES) sums[POST_BIAS][e] += H[e];
                    H[e] *= w[e];
                    m.x += H[e];
                    m.y += H[e] * y[e];
                }
                if (p.post_norm == D2P_NORM_LAYER) m = team.sum(m.x, m.y);
                else m = {0.0f, team.sum(m.y)};
                m.x = divided(m.x, (float)D);
                m.y = divided(m.y, (float)D);
#pragma unroll
                for (int e = 0; e < RUN; ++e) H[e] = st[3] * (H[e] - m.x - y[e] * m.y);
            }
            store_run((TY*)a.dy + flat, have, H);
        }
        if (BLOCK && a.partial[GATE]) {
            flush(lds + SLOTS + VECTORS * vec.padded, sums[GATE],
                  a.partial[GATE] + (long long)seg * D, a.lanes, D);
#pragma unroll
            for (int e = 0; e < RUN; ++e) sums[GATE][e] = 0.0f;
        }
    }
#pragma unroll
    for (int k = 0; k < GATE; ++k)
        if ((BLOCK || k < POST_WEIGHT) && (BIASES || (k != BIAS && k != POST_BIAS)) && a.partial[k])
            flush(lds + SLOTS + VECTORS * vec.padded, sums[k],
                  a.partial[k] + (long long)blockIdx.x * D, a.lanes, D);
}

namespace {

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
    D2P_REQUIRE(p->D >= RUN && p->D <= 8192, "features must be between 8 and 8192");
    for (int kind : {p->norm, p->post_norm})
        D2P_REQUIRE(kind >= D2P_NORM_NONE && kind <= D2P_NORM_LAYER, "unknown norm");
    for (const d2p_vector* v : {&p->weight, &p->bias, &p->post_weight, &p->post_bias})
        D2P_TRY(check_vector(*v));
    D2P_REQUIRE((p->norm != D2P_NORM_NONE || !(p->weight.data || p->bias.data)) &&
                    (p->post_norm != D2P_NORM_NONE || !(p->post_weight.data || p->post_bias.data)),
                "a norm's weight and bias need the norm");
    D2P_REQUIRE(p->gate_kind >= D2P_GATE_NONE && p->gate_kind <= D2P_GATE_TOKEN, "unknown gate");
    D2P_REQUIRE(p->gate_kind == D2P_GATE_NONE || p->gate_dtype == D2P_FLOAT32 ||
                    p->gate_dtype == p->block_dtype,
                "the gate must be float32 or of the block's type");
    D2P_REQUIRE(p->gate_kind == D2P_GATE_NONE || (long long)p->B * p->L == 0 || p->gate,
                "null pointer argument");
    D2P_REQUIRE(p->eps >= 0.0f, "eps must not be negative");
    return D2P_OK;
}

// Strides over one of something say nothing: those of a contiguous tensor stand in their place.
d2p_row_strides plain(const d2p_row_strides& s, const d2p_residual_norm_params& p) {
    const long long row = p.L > 1 ? s.row : p.D;
    return {p.B > 1 ? s.batch : p.L * row, row};
}
d2p_row_strides gate_steps(const d2p_residual_norm_params& p) {
    if (p.gate_kind == D2P_GATE_TOKEN) return plain(p.gate_strides, p);
    return {p.gate_kind == D2P_GATE_SEQUENCE ? p.gate_strides.batch : 0, 0};
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
template <class TX, class TY, bool BLOCK, bool EVEN, int MOST>
int launch_forward(const ResidualArgs& a, int grid, hipStream_t st) {
    static LdsAllowed known;
    return launch("residual_norm", residual_norm_kernel<TX, TY, BLOCK, EVEN, MOST>, known, a, grid,
                  false, st);
}
template <class TX, class TY, bool BLOCK, bool EVEN, int MOST>
int launch_backward(const ResidualBackArgs& a, int grid, hipStream_t st) {
    static LdsAllowed known[2];
    if (a.partial[BIAS] || a.partial[POST_BIAS])
        return launch("residual_norm_backward",
                      residual_norm_backward_kernel<TX, TY, BLOCK, true, EVEN, MOST>, known[1], a,
                      grid, true, st);
    return launch("residual_norm_backward",
                  residual_norm_backward_kernel<TX, TY, BLOCK, false, EVEN, MOST>, known[0], a, grid,
                  true, st);
}

int most_threads(int D) { return D <= 64 * RUN ? ONE_WAVE : MORE_WAVES; }
// f(rows of whole runs, threads of a workgroup at most): rows within a wave, or of several
template <class F> int by_rows(int D, F f) {
    const auto more = [&](auto most) {
        return D % RUN ? f(std::false_type{}, most) : f(std::true_type{}, most);
    };
    return most_threads(D) == ONE_WAVE ? more(std::integral_constant<int, ONE_WAVE>{})
                                       : more(std::integral_constant<int, MORE_WAVES>{});
}

// How the backward pass cuts rows into segments: at most as many as the card's 256 compute units
// hold at `waves` waves a SIMD, no fewer while there are rows for it, and each of one sequence
// where the gate's gradient is by sequence.
struct Cut {
    int batches, length, splits, grid;
    Cut(const d2p_residual_norm_params& p, int lanes, int waves) {
        const int teams = threads_of(lanes) / lanes;
        const bool by_sequence = p.gate_kind == D2P_GATE_SEQUENCE;
        batches = by_sequence ? p.B : 1;
        length = by_sequence ? p.L : p.B * p.L;
        const int groups = 256 * 256 * waves / threads_of(lanes);
        const int most = std::max(1, groups / std::max(batches, 1));
        // (whole turns of a workgroup's teams: float32 beside bf16 [5, 1023, 333], layer norms, 640
        // workgroups of 8 rows 24 us, 1024 of 5 rows 29)
        splits = std::max(1, cdiv(length, std::max(1, cdiv(cdiv(length, most), teams) * teams)));
        grid = (int)std::min<long long>((long long)batches * splits, groups);
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
    D2P_REQUIRE(((uintptr_t)stats & 15) == 0, "stats must be aligned to 16 bytes");
    ResidualArgs a{*p, x, y, h, n, stats, team_of(p->D), Divisor(p->L)};
    for (d2p_row_strides* s : {&a.p.x, &a.p.y}) *s = plain(*s, *p);
    a.p.gate_strides = gate_steps(*p);
    const int teams = threads_of(a.lanes) / a.lanes;
    const int most = 8 * 256 * std::max(device_cus(), 1) / threads_of(a.lanes);
    const int grid = std::min(cdiv(p->B * p->L, teams), most);
    return with_pair(p->dtype, p->block_dtype, [&](auto tx, auto ty) {
        using TX = typename decltype(tx)::type;
        using TY = typename decltype(ty)::type;
        const auto st = (hipStream_t)stream;
        return by_rows(p->D, [&](auto even, auto most) {
            return y ? launch_forward<TX, TY, true, even(), most()>(a, grid, st)
                     : launch_forward<TX, TY, false, even(), most()>(a, grid, st);
        });
    });
}

extern "C" size_t d2p_residual_norm_backward_workspace_bytes(const d2p_residual_norm_params* p) {
    if (!p || p->B < 0 || p->L < 0 || p->D < RUN || p->D > 8192 || (long long)p->B * p->L >= 1LL << 31)
        return 0;
    const Cut cut(*p, team_of(p->D), BACK_WAVES);
    const size_t gate = p->gate_kind == D2P_GATE_FEATURE || p->gate_kind == D2P_GATE_SEQUENCE
                            ? (size_t)cut.batches * cut.splits : 0;
    return ((size_t)GATE * cut.grid + gate) * p->D * 4;
}

extern "C" int d2p_residual_norm_backward(const d2p_residual_norm_params* p, const void* dh,
                                          const void* dn, const void* stream_in, const void* y,
                                          const float* stats, void* dx, void* dy, void* dgate,
                                          void* dweight, void* dbias, void* dpost_weight,
                                          void* dpost_bias, void* workspace,
                                          size_t workspace_bytes, void* stream) {
    D2P_TRY(check(p));
    const bool rows = (long long)p->B * p->L > 0, wide = p->dtype == D2P_FLOAT32;
    const bool norm = dn && p->norm != D2P_NORM_NONE;
    const bool again = norm && p->with_y && !wide;      // h is formed anew
    if (rows) {
        D2P_REQUIRE(dh || norm, "dh or dn is needed");
        D2P_REQUIRE(dx && (!norm || (stream_in && stats)), "null pointer argument");
        D2P_REQUIRE(p->post_norm == D2P_NORM_NONE || (y && stats), "null pointer argument");
        D2P_REQUIRE(y || !(dgate || again), "y is needed");
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
    if (p->with_y && wide) a.p.x = {(long long)p->L * p->D, p->D};
    if (!p->with_y) a.p.residual_scale = 1.0f;
    for (d2p_row_strides* s : {&a.p.x, &a.p.y, &a.p.dh, &a.p.dn}) *s = plain(*s, *p);
    // dh and what n was formed from are of the wide type: a row of them has room for any
    const void* const other = dh ? dh : stream_in;
    auto or_else = [&](const void* x, d2p_row_strides& s) {
        if (!x) s = {0, 0};
        return x ? x : other;
    };
    a.has_dh = dh;
    a.has_dn = norm;
    a.has_y = y;
    a.dh = or_else(dh, a.p.dh);
    a.dn = or_else(norm ? dn : nullptr, a.p.dn);
    a.stream = or_else(norm ? stream_in : nullptr, a.p.x);
    a.y = or_else(y, a.p.y);
    a.stats = stats ? stats : (const float*)other;
    a.stats_step = stats ? 4 : 0;
    a.dx = dx;
    a.dy = dy;
    a.dgate = dgate;
    a.lanes = team_of(p->D);
    a.by_length = Divisor(p->L);
    const Cut cut(*p, a.lanes,
                  back_waves((dy || again) && !wide, dbias || dpost_bias, most_threads(p->D)));
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
            return by_rows(p->D, [&](auto even, auto most) {
                return dy || again ? launch_backward<TX, TY, true, even(), most()>(a, cut.grid, st)
                                   : launch_backward<TX, TY, false, even(), most()>(a, cut.grid, st);
            });
        }));
    return launch_sum_rows("residual_norm_vector_grads", jobs, (hipStream_t)stream);
}
