// attention_forward_f32.hip -- the attention forward kernels for float.
#include "attention_forward.hip.h"

int d2p_amd::enc::launch_forward_f32(const ForwardArgs& a, hipStream_t st) {
    return launch_forward<float>(a, st);
}
