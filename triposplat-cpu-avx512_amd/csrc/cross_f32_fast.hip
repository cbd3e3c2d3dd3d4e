// Cross attention of fp32 values in two bf16 terms or one of each factor.
#include "cross_attention_kernel.h"

namespace tsplat {

int launch_cross_f32_fast(const CrossParams& p, hipStream_t stream) {
  return p.terms == 2 ? cross::launch_terms<float, 2>(p, stream) : cross::launch_terms<float, 1>(p, stream);
}

}  // namespace tsplat
