// rows.hip -- sums of rows of float32 numbers in a fixed order: the last step of gradients
// that workgroups have summed in parts.  From caches, and so bound by the loads' latency: 1024 rows
// of 512 numbers, twice, in 5.2 us.
#include <algorithm>

#include "training.hip.h"

namespace d2p_amd {
namespace enc {

// 64 numbers a workgroup, 16 waves over the rows, eight loads in flight each; the waves' sums
// then in order.
__global__ void __launch_bounds__(1024) sum_rows_kernel(SumJobs a) {
    __shared__ float part[16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int j = 0;
    for (unsigned block = blockIdx.x; block < (unsigned)a.blocks; block += gridDim.x) {
        while (j + 1 < a.jobs && block >= (unsigned)a.job[j + 1].first) ++j;
        const SumJob job = a.job[j];
        const int at = block - job.first, group = at / a.tiles;
        const int d = (at % a.tiles) * 64 + lane;
        float s = 0.0f;
        if (d < a.D) {
            const float* from = job.src + (long long)group * job.count * a.D + d;
            float t[8] = {};
            int r = wave;
            for (; r + 7 * 16 < job.count; r += 8 * 16) {
#pragma unroll
                for (int u = 0; u < 8; ++u) t[u] += from[(long long)(r + 16 * u) * a.D];
            }
            for (; r < job.count; r += 16) t[0] += from[(long long)r * a.D];
#pragma unroll
            for (int u = 0; u < 8; ++u) s += t[u];
        }
        __syncthreads();
        part[wave][lane] = s;
        __syncthreads();
        if (wave || d >= a.D) continue;
        s = 0.0f;
#pragma unroll
        for (int w = 0; w < 16; ++w) s += part[w][lane];
        store_as(job.dst, job.dtype, (long long)group * a.D + d, s * a.scale);
    }
}

int launch_sum_rows(const char* name, const SumJobs& a, hipStream_t st) {
    if (a.blocks == 0) return D2P_OK;
    // (a launch has fewer than 2^32 threads)
    D2P_LAUNCH(name, sum_rows_kernel, dim3(std::min(a.blocks, 1 << 20)), dim3(1024), 0, st, a);
    D2P_HIP(hipGetLastError());
    return D2P_OK;
}

}  // namespace enc
}  // namespace d2p_amd
