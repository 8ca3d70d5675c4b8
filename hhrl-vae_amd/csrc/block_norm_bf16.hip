// The bf16 kernels of the norms around a block.
#include "block_norm.h"

namespace hhrl {

void norm_launch_bf16(const NormArgs& a, bool vec, int tpr, int blocks, bool bwd, hipStream_t st) { norm_launch<__bf16, 8>(a, vec, tpr, blocks, bwd, st); }

}  // namespace hhrl
