// attention_backward_bf16.hip -- the attention backward kernels for __bf16.
#include "attention_backward.hip.h"

int d2p_amd::enc::launch_backward_bf16(const BackwardArgs& a, hipStream_t st) {
    return launch_backward<__bf16>(a, st);
}
