// The causal attention kernels for f32 elements (see causal_attention.h); a unit of its own so that the types build in
// parallel.
#include "causal_attention.h"

namespace rdv {

void launch_causal_f32(CausalKernel which, const CausalArgs& a, unsigned blocks, hipStream_t stream) {
  launch_causal_typed<float>(which, a, blocks, stream);
}

}  // namespace rdv
