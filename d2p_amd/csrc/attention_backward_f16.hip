// attention_backward_f16.hip -- the attention backward kernels for _Float16.
#include "attention_backward.hip.h"

int d2p_amd::enc::launch_backward_f16(const BackwardArgs& a, hipStream_t st) {
    return launch_backward<_Float16>(a, st);
}
