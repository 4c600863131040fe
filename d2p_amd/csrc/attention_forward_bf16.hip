// attention_forward_bf16.hip -- the attention forward kernels for __bf16.
#include "attention_forward.hip.h"

int d2p_amd::enc::launch_forward_bf16(const ForwardArgs& a, hipStream_t st) {
    return launch_forward<__bf16>(a, st);
}
