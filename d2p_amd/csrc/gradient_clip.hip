// gradient_clip.hip -- the norm over all numbers of a list of tensors, and the list scaled to
// a largest norm (include/d2p_amd_training.h).
//
// Bound by memory: one pass for the norm, one for the scaling.  The list goes along as the first
// kernel's argument, so that a call needs no copy to the device and a captured one keeps its
// pointers; longer lists take several launches.  They leave the list in the workspace for the
// second pass, which is one launch.  Tensors are cut into pieces of PIECE numbers; a workgroup
// takes neighbouring ones, so that it looks its tensor up once, and takes them in falling order
// in the second pass, which so begins with what the first one has left in the caches (320 M bf16:
// 383 us in rising order, 367 in falling).  Squares are summed in float64: no gradient's
// overflows it, and the vector units have the time.
//
// 320 M bf16 in 40 tensors: the norm in 113 us, 5.7 TB/s (a read alone reaches 6.1), clipping in 371
// for both passes, 5.2 TB/s.  24 M numbers of three types in 301 tensors: 11 us for each of two lists,
// 27 for the scaling.  280 k in 18 tensors: 6.5 and 5.5 us, most of it launches and the lookup.
#include <algorithm>

#include "training.hip.h"

namespace d2p_amd {
namespace enc {

constexpr int LIST = 180;                       // tensors of one launch
constexpr int THREADS = 256, DEEP = 4;          // runs that a thread has in flight
constexpr int PIECE = THREADS * RUN * DEEP;
constexpr int BLOCKS = 1024;                    // workgroups of a pass, and partial sums

// A tensor: where it is, its type in the source's two highest bits, its first piece (counted
// over the whole list) and the numbers of its last one less one.
struct ClipList {
    unsigned long long src[LIST], dst[LIST];
    int first[LIST + 1];
    unsigned short last[LIST];
};
// The same for all tensors, in the workspace.
struct ClipTable {
    unsigned long long *src, *dst;
    int* first;
    unsigned short* last;
};
struct ClipArgs {
    double* partial;            // [BLOCKS]
    float* norm;
    double max_norm;
    ClipTable table;
    int count, from;            // tensors of this launch, and those before
    int keep;                   // the list goes into the table
};
static_assert(sizeof(ClipList) + sizeof(ClipArgs) <= 4096, "kernel arguments");
constexpr int TYPE_SHIFT = 62;

// Pieces p0 .. p1 - 1 of one tensor.
struct Pieces {
    unsigned long long src;
    int dtype, whole, part;     // whole pieces; numbers of the one behind them, or 0
    long long at;               // the first number's place in the tensor
    __device__ __forceinline__ Pieces(unsigned long long src_, int p0, int p1, int first, int end,
                                      int last)
        : src(src_ & ~(3ULL << TYPE_SHIFT)), dtype((int)(src_ >> TYPE_SHIFT)), whole(p1 - p0),
          part(0), at((long long)(p0 - first) * PIECE) {
        if (p1 == end && last + 1 < PIECE) {
            --whole;
            part = last + 1;
        }
    }
};

__device__ __forceinline__ double block_sum(double x) {
    __shared__ double part[THREADS / 64];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = x;
    __syncthreads();
    x = 0.0;
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) x += part[w];
    return x;
}

__device__ __forceinline__ int block_count(int x) {
    __shared__ int part[THREADS / 64];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o, 64);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = x;
    __syncthreads();
    x = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) x += part[w];
    return x;
}

// f(place, numbers) for each run of the thread in the pieces; BACK: the last piece first.  A
// piece's loads are under way while the piece before it is worked on.
template <class T, bool BACK, class F> __device__ __forceinline__ void each_run(const Pieces& a, F f) {
    // (a pointer made of a number has to be told to be the device's)
    const T* src = (const T*)(const __attribute__((address_space(1))) T*)a.src + a.at;
    const int me = threadIdx.x * RUN;
    float x[RUN];
    if (a.part >= RUN) {
        const T* row = src + (long long)a.whole * PIECE;
        Eight<T> r[DEEP];
#pragma unroll
        for (int u = 0; u < DEEP; ++u) r[u] = load_run(row, u * THREADS * RUN + me, a.part);
#pragma unroll
        for (int u = 0; u < DEEP; ++u) {
            const int at = u * THREADS * RUN + me;
            unpack(r[u], at, a.part, true, x);
            f((long long)a.whole * PIECE + at, a.part - at, x);
        }
    } else if (threadIdx.x == 0 && a.part > 0) {
        const T* row = src + (long long)a.whole * PIECE;
#pragma unroll
        for (int e = 0; e < RUN; ++e) x[e] = e < a.part ? (float)row[e] : 0.0f;
        f((long long)a.whole * PIECE, a.part, x);
    }
    if (a.whole == 0) return;
    Eight<T> now[DEEP], next[DEEP];
    auto load = [&](int q, Eight<T> (&r)[DEEP]) {
        const T* row = src + (long long)(BACK ? a.whole - 1 - q : q) * PIECE + me;
#pragma unroll
        for (int u = 0; u < DEEP; ++u) r[u] = *(const Eight<T>*)(row + u * THREADS * RUN);
    };
    load(0, now);
    for (int q = 0; q < a.whole; ++q) {
        load(min(q + 1, a.whole - 1), next);
#pragma unroll
        for (int u = 0; u < DEEP; ++u) {
#pragma unroll
            for (int e = 0; e < RUN; ++e) x[e] = (float)now[u].v[e];
            f((long long)(BACK ? a.whole - 1 - q : q) * PIECE + u * THREADS * RUN + me, RUN, x);
            now[u] = next[u];
        }
    }
}
template <class T> __device__ __forceinline__ double squares_of(const Pieces& a) {
    double s = 0.0;
    each_run<T, false>(a, [&](long long, int, const float* x) {
#pragma unroll
        for (int e = 0; e < RUN; ++e) s += (double)x[e] * x[e];
    });
    return s;
}
template <class T>
__device__ __forceinline__ void scale_pieces(const Pieces& a, unsigned long long to, float c) {
    T* dst = (T*)(__attribute__((address_space(1))) T*)to + a.at;
    each_run<T, true>(a, [&](long long at, int left, float* x) {
#pragma unroll
        for (int e = 0; e < RUN; ++e) x[e] *= c;
        store_run(dst + at, left, x);
    });
}

// A workgroup's share of pieces first .. end
__device__ __forceinline__ void share(int first, int end, int* p0, int* p1) {
    const long long n = end - first;
    *p0 = first + (int)(n * blockIdx.x / gridDim.x);
    *p1 = first + (int)(n * (blockIdx.x + 1) / gridDim.x);
}

__global__ void __launch_bounds__(THREADS) squares_kernel(ClipList list, ClipArgs a) {
    if (a.keep && blockIdx.x == 0) {
        for (int i = threadIdx.x; i <= a.count; i += THREADS) {
            a.table.first[a.from + i] = list.first[i];
            if (i == a.count) break;
            a.table.src[a.from + i] = list.src[i];
            a.table.dst[a.from + i] = list.dst[i];
            a.table.last[a.from + i] = list.last[i];
        }
    }
    // the tensor of the share's first piece: the last that begins there or before (one look at
    // all of them, where a search would wait for one after the other)
    int p0, p1, before = 0;
    share(list.first[0], list.first[a.count], &p0, &p1);
    static_assert(LIST <= THREADS, "a thread looks at one tensor");
    if ((int)threadIdx.x < a.count) before = list.first[threadIdx.x] <= p0;
    int lo = __builtin_amdgcn_readfirstlane(block_count(before)) - 1;
    double s = 0.0;
    for (int p = p0; p < p1; ++lo) {
        const int end = list.first[lo + 1], to = min(p1, end);
        if (to > p) {
            const Pieces at(list.src[lo], p, to, list.first[lo], end, list.last[lo]);
            s += at.dtype == D2P_FLOAT32 ? squares_of<float>(at)
                 : at.dtype == D2P_FLOAT16 ? squares_of<_Float16>(at) : squares_of<__bf16>(at);
            p = to;
        }
    }
    s = block_sum(s);
    if (threadIdx.x == 0) a.partial[blockIdx.x] = a.from ? a.partial[blockIdx.x] + s : s;
}

// sqrt of the sum of all partial sums, the same in every workgroup
__device__ __forceinline__ double whole_norm(const double* partial) {
    double s = 0.0;
#pragma unroll
    for (int i = 0; i < BLOCKS / THREADS; ++i) s += partial[i * THREADS + threadIdx.x];
    return sqrt(block_sum(s));
}

__global__ void __launch_bounds__(THREADS) norm_kernel(ClipArgs a) {
    const double norm = whole_norm(a.partial);
    if (threadIdx.x == 0) *a.norm = (float)norm;
}

__global__ void __launch_bounds__(THREADS) clip_kernel(ClipArgs a) {
    const ClipTable& list = a.table;
    int p0, p1, before = 0;
    share(0, list.first[a.count], &p0, &p1);
    // the tensor of the share's last piece
    for (int i = threadIdx.x; i < a.count; i += THREADS) before += list.first[i] < p1;
    int t = __builtin_amdgcn_readfirstlane(block_count(before)) - 1;
    const double norm = whole_norm(a.partial);
    if (blockIdx.x == 0 && threadIdx.x == 0) *a.norm = (float)norm;
    const bool fits = norm <= a.max_norm;
    const float c = fits ? 1.0f : (float)(a.max_norm / norm);
    for (int p = p1; p > p0; --t) {
        const int first = list.first[t], from = max(p0, first);
        const Pieces at(list.src[t], from, p, first, list.first[t + 1], list.last[t]);
        const unsigned long long dst = list.dst[t];
        p = from;
        if (fits && dst == at.src) continue;
        if (at.dtype == D2P_FLOAT32) scale_pieces<float>(at, dst, c);
        else if (at.dtype == D2P_FLOAT16) scale_pieces<_Float16>(at, dst, c);
        else scale_pieces<__bf16>(at, dst, c);
    }
}

namespace {

int check(const d2p_tensor* tensors, int count, const float* norm, const void* workspace,
          size_t bytes, bool clip) {
    D2P_REQUIRE(count >= 0 && (tensors || count == 0) && norm, "null pointer argument");
    for (int i = 0; i < count; ++i) {
        const d2p_tensor& t = tensors[i];
        D2P_REQUIRE(known_type(t.dtype), "unknown element type");
        D2P_REQUIRE(t.n >= 0, "negative size");
        D2P_REQUIRE(t.n == 0 || (t.src && (!clip || t.dst)), "null pointer argument");
        D2P_REQUIRE(t.n <= (1LL << 41), "a tensor is too long");
        D2P_REQUIRE(((uintptr_t)t.src | (clip ? (uintptr_t)t.dst : 0)) % type_bytes(t.dtype) == 0,
                    "a tensor is not aligned to its element");
    }
    D2P_REQUIRE(workspace && bytes >= d2p_global_norm_workspace_bytes(count), "workspace too small");
    D2P_REQUIRE(((uintptr_t)workspace & 7) == 0, "the workspace must be aligned to 8 bytes");
    return D2P_OK;
}

// The partial sums' pass.  `all`: pieces and tensors (those with no number are left out).
int launch_squares(const d2p_tensor* tensors, int count, ClipArgs a, int* all, int* filled,
                   hipStream_t st) {
    int from = 0;
    long long pieces = 0;
    do {
        ClipList list;
        int k = 0;
        list.first[0] = (int)pieces;
        for (; from < count && k < LIST; ++from) {
            const d2p_tensor& t = tensors[from];
            if (t.n == 0) continue;
            const long long more = (t.n + PIECE - 1) / PIECE;
            pieces += more;
            D2P_REQUIRE(pieces < 0x7fffffff, "too many numbers");
            list.src[k] = (unsigned long long)t.src | (unsigned long long)t.dtype << TYPE_SHIFT;
            list.dst[k] = (unsigned long long)t.dst;
            list.last[k] = (unsigned short)(t.n - (more - 1) * PIECE - 1);
            list.first[++k] = (int)pieces;
        }
        a.count = k;
        D2P_LAUNCH("gradient_squares", squares_kernel, dim3(BLOCKS), dim3(THREADS), 0, st, list, a);
        D2P_HIP(hipGetLastError());
        a.from += k;
    } while (from < count);
    *all = (int)pieces;
    *filled = a.from;
    return D2P_OK;
}

}  // namespace
}  // namespace enc
}  // namespace d2p_amd

using namespace d2p_amd;
using namespace d2p_amd::enc;

extern "C" size_t d2p_global_norm_workspace_bytes(int count) {
    return BLOCKS * sizeof(double) + (size_t)std::max(count, 0) * (8 + 8 + 4 + 2) + 8;
}

extern "C" int d2p_global_norm(const d2p_tensor* tensors, int count, float* norm, void* workspace,
                               size_t workspace_bytes, void* stream) {
    D2P_TRY(check(tensors, count, norm, workspace, workspace_bytes, false));
    hipStream_t st = (hipStream_t)stream;
    ClipArgs a{};
    a.partial = (double*)workspace;
    a.norm = norm;
    int pieces, filled;
    D2P_TRY(launch_squares(tensors, count, a, &pieces, &filled, st));
    D2P_LAUNCH("gradient_norm", norm_kernel, dim3(1), dim3(THREADS), 0, st, a);
    D2P_HIP(hipGetLastError());
    return D2P_OK;
}

extern "C" int d2p_clip_by_norm(const d2p_tensor* tensors, int count, double max_norm, float* norm,
                                void* workspace, size_t workspace_bytes, void* stream) {
    D2P_TRY(check(tensors, count, norm, workspace, workspace_bytes, true));
    D2P_REQUIRE(max_norm >= 0.0, "max_norm must not be negative");
    hipStream_t st = (hipStream_t)stream;
    ClipArgs a{};
    a.partial = (double*)workspace;
    a.norm = norm;
    a.max_norm = max_norm;
    a.table.src = (unsigned long long*)(a.partial + BLOCKS);
    a.table.dst = a.table.src + count;
    a.table.first = (int*)(a.table.dst + count);
    a.table.last = (unsigned short*)(a.table.first + count + 1);
    a.keep = 1;
    int pieces;
    D2P_TRY(launch_squares(tensors, count, a, &pieces, &a.count, st));
    D2P_LAUNCH("gradient_clip", clip_kernel, dim3(std::max(1, std::min(BLOCKS, pieces))),
               dim3(THREADS), 0, st, a);
    D2P_HIP(hipGetLastError());
    return D2P_OK;
}
