// gradient_clip.hip -- the norm over all numbers of a list of tensors, and the list scaled to
// a largest norm (include/d2p_amd_training.h).
//
// Bound by memory: one pass for the norm, one for the scaling.  The list goes along as the
// kernels' argument, so that a call needs no copy to the device and a captured one keeps its
// pointers; longer lists take several launches.  Tensors are cut into pieces of PIECE numbers,
// which workgroups take in turn.  Squares are summed in float64: no gradient's overflows it,
// and the vector units have the time.  The second pass takes the pieces in falling order, so
// that it begins with what the first one has left in the caches.
#include <algorithm>

#include "training.hip.h"

namespace d2p_amd {
namespace enc {

constexpr int LIST = 128;                       // tensors of one launch
constexpr int THREADS = 256, DEEP = 4;          // runs that a thread has in flight
constexpr int PIECE = THREADS * RUN * DEEP;
constexpr int BLOCKS = 1024;                    // workgroups of a pass, and partial sums

struct ClipList {
    const void* src[LIST];
    void* dst[LIST];
    long long n[LIST];
    int first[LIST + 1];        // a tensor's first piece
    unsigned char dtype[LIST];
    int count;
};
struct ClipArgs {
    double* partial;            // [BLOCKS]
    float* norm;
    double max_norm;
    int add;                    // to the sums of the launches before
};
static_assert(sizeof(ClipList) + sizeof(ClipArgs) <= 4096, "kernel arguments");

// The tensor that a piece is of.
__device__ __forceinline__ int tensor_of(const ClipList& a, int piece) {
    int lo = 0, hi = a.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (a.first[mid] <= piece) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

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

template <class T> __device__ __forceinline__ double piece_squares(const T* src, long long left) {
    float x[DEEP][RUN];
#pragma unroll
    for (int u = 0; u < DEEP; ++u) {
        const int at = (u * THREADS + threadIdx.x) * RUN;
        load_run(src + at, (int)min(max(left - at, 0LL), (long long)RUN), x[u]);
    }
    double s = 0.0;
#pragma unroll
    for (int u = 0; u < DEEP; ++u)
#pragma unroll
        for (int e = 0; e < RUN; ++e) s += (double)x[u][e] * x[u][e];
    return s;
}

template <class T>
__device__ __forceinline__ void scale_piece(const T* src, T* dst, long long left, float c) {
    float x[DEEP][RUN];
    int have[DEEP];
#pragma unroll
    for (int u = 0; u < DEEP; ++u) {
        const int at = (u * THREADS + threadIdx.x) * RUN;
        have[u] = (int)min(max(left - at, 0LL), (long long)RUN);
        load_run(src + at, have[u], x[u]);
    }
#pragma unroll
    for (int u = 0; u < DEEP; ++u) {
#pragma unroll
        for (int e = 0; e < RUN; ++e) x[u][e] *= c;
        store_run(dst + (u * THREADS + threadIdx.x) * RUN, have[u], x[u]);
    }
}

__global__ void __launch_bounds__(THREADS) squares_kernel(ClipList list, ClipArgs a) {
    const int pieces = list.first[list.count];
    double s = 0.0;
    for (int piece = blockIdx.x; piece < pieces; piece += gridDim.x) {
        const int t = tensor_of(list, piece);
        const long long at = (long long)(piece - list.first[t]) * PIECE, left = list.n[t] - at;
        const int dtype = list.dtype[t];
        s += dtype == D2P_FLOAT32 ? piece_squares((const float*)list.src[t] + at, left)
             : dtype == D2P_FLOAT16 ? piece_squares((const _Float16*)list.src[t] + at, left)
                                    : piece_squares((const __bf16*)list.src[t] + at, left);
    }
    s = block_sum(s);
    if (threadIdx.x == 0) a.partial[blockIdx.x] = a.add ? a.partial[blockIdx.x] + s : s;
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

__global__ void __launch_bounds__(THREADS) clip_kernel(ClipList list, ClipArgs a) {
    const int pieces = list.first[list.count];
    const double norm = whole_norm(a.partial);
    if (a.norm && blockIdx.x == 0 && threadIdx.x == 0) *a.norm = (float)norm;
    const bool fits = norm <= a.max_norm;
    const float c = fits ? 1.0f : (float)(a.max_norm / norm);
    for (int i = blockIdx.x; i < pieces; i += gridDim.x) {
        const int piece = pieces - 1 - i, t = tensor_of(list, piece);
        if (fits && list.src[t] == list.dst[t]) continue;
        const long long at = (long long)(piece - list.first[t]) * PIECE, left = list.n[t] - at;
        const int dtype = list.dtype[t];
        if (dtype == D2P_FLOAT32)
            scale_piece((const float*)list.src[t] + at, (float*)list.dst[t] + at, left, c);
        else if (dtype == D2P_FLOAT16)
            scale_piece((const _Float16*)list.src[t] + at, (_Float16*)list.dst[t] + at, left, c);
        else
            scale_piece((const __bf16*)list.src[t] + at, (__bf16*)list.dst[t] + at, left, c);
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
    D2P_REQUIRE(workspace && bytes >= BLOCKS * sizeof(double), "workspace too small");
    D2P_REQUIRE(((uintptr_t)workspace & 7) == 0, "the workspace must be aligned to 8 bytes");
    return D2P_OK;
}

// The next launch's part of the list, from tensor `from` on; where the one after begins.
int next_list(const d2p_tensor* tensors, int count, int from, ClipList& list) {
    long long pieces = 0;
    list.count = 0;
    list.first[0] = 0;
    for (; from < count && list.count < LIST; ++from) {
        const d2p_tensor& t = tensors[from];
        if (t.n == 0) continue;
        const long long more = (t.n + PIECE - 1) / PIECE;
        if (list.count && pieces + more > 0x3fffffff) break;
        const int k = list.count++;
        list.src[k] = t.src;
        list.dst[k] = t.dst;
        list.n[k] = t.n;
        list.dtype[k] = (unsigned char)t.dtype;
        pieces += more;
        list.first[k + 1] = (int)pieces;
    }
    return from;
}

int launch_squares(const d2p_tensor* tensors, int count, ClipArgs a, hipStream_t st) {
    int from = 0;
    do {
        ClipList list;
        from = next_list(tensors, count, from, list);
        D2P_LAUNCH("gradient_squares", squares_kernel, dim3(BLOCKS), dim3(THREADS), 0, st, list, a);
        D2P_HIP(hipGetLastError());
        a.add = 1;
    } while (from < count);
    return D2P_OK;
}

}  // namespace
}  // namespace enc
}  // namespace d2p_amd

using namespace d2p_amd;
using namespace d2p_amd::enc;

extern "C" size_t d2p_global_norm_workspace_bytes(void) { return BLOCKS * sizeof(double); }

extern "C" int d2p_global_norm(const d2p_tensor* tensors, int count, float* norm, void* workspace,
                               size_t workspace_bytes, void* stream) {
    D2P_TRY(check(tensors, count, norm, workspace, workspace_bytes, false));
    hipStream_t st = (hipStream_t)stream;
    const ClipArgs a{(double*)workspace, norm, 0.0, 0};
    D2P_TRY(launch_squares(tensors, count, a, st));
    D2P_LAUNCH("gradient_norm", norm_kernel, dim3(1), dim3(THREADS), 0, st, a);
    D2P_HIP(hipGetLastError());
    return D2P_OK;
}

extern "C" int d2p_clip_by_norm(const d2p_tensor* tensors, int count, double max_norm, float* norm,
                                void* workspace, size_t workspace_bytes, void* stream) {
    D2P_TRY(check(tensors, count, norm, workspace, workspace_bytes, true));
    D2P_REQUIRE(max_norm >= 0.0, "max_norm must not be negative");
    hipStream_t st = (hipStream_t)stream;
    ClipArgs a{(double*)workspace, norm, max_norm, 0};
    D2P_TRY(launch_squares(tensors, count, a, st));
    int from = 0;
    do {
        ClipList list;
        from = next_list(tensors, count, from, list);
        D2P_LAUNCH("gradient_clip", clip_kernel, dim3(std::max(1, std::min(BLOCKS, list.first[list.count]))),
                   dim3(THREADS), 0, st, list, a);
        D2P_HIP(hipGetLastError());
        a.norm = nullptr;
    } while (from < count);
    return D2P_OK;
}
