// Cross attention of fp32 values at fp32 accuracy (three bf16 terms of each factor).
#include "cross_attention_kernel.h"

namespace tsplat {

int launch_cross_f32(const CrossParams& p, hipStream_t stream) { return cross::launch_terms<float, 3>(p, stream); }

}  // namespace tsplat
