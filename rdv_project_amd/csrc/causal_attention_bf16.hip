// The causal attention kernels for bf16 elements (see causal_attention.h); a unit of its own so that the types build in
// parallel.
#include "causal_attention.h"

namespace rdv {

void launch_causal_bf16(CausalKernel which, const CausalArgs& a, unsigned blocks, hipStream_t stream) {
  launch_causal_typed<bf16_t>(which, a, blocks, stream);
}

}  // namespace rdv
