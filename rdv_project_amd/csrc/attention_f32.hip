// The attention kernels for f32 elements (see attention.h); a unit of its own so that the types build in parallel.
#include "attention.h"

namespace rdv {

void launch_attn_f32(AttnKernel which, const AttnArgs& a, unsigned blocks, hipStream_t stream) {
  launch_attn_typed<float>(which, a, blocks, stream);
}

}  // namespace rdv
