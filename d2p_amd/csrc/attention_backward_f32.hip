// attention_backward_f32.hip -- the attention backward kernels for float.
#include "attention_backward.hip.h"

int d2p_amd::enc::launch_backward_f32(const BackwardArgs& a, hipStream_t st) {
    return launch_backward<float>(a, st);
}
