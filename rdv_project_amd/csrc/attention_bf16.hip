// The attention kernels for bf16 elements (see attention.h); a unit of its own so that the types build in parallel.
#include "attention.h"

namespace rdv {

void launch_attn_bf16(AttnKernel which, const AttnArgs& a, unsigned blocks, hipStream_t stream) {
  launch_attn_typed<bf16_t>(which, a, blocks, stream);
}

}  // namespace rdv
