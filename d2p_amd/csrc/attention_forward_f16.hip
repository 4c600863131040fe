// attention_forward_f16.hip -- the attention forward kernels for _Float16.
#include "attention_forward.hip.h"

int d2p_amd::enc::launch_forward_f16(const ForwardArgs& a, hipStream_t st) {
    return launch_forward<_Float16>(a, st);
}
