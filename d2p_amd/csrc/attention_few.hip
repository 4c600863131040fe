// attention_few.hip -- the kernels for few queries, all element types.
#include <algorithm>

#include "attention_few.hip.h"

int d2p_amd::enc::launch_few_f32(const FewArgs& a, hipStream_t st) { return launch_few<float>(a, st); }
int d2p_amd::enc::launch_few_f16(const FewArgs& a, hipStream_t st) {
    return launch_few<_Float16>(a, st);
}
int d2p_amd::enc::launch_few_bf16(const FewArgs& a, hipStream_t st) {
    return launch_few<__bf16>(a, st);
}
