// The bfloat16 instances of the block-scaled attention kernel.
#include "kvhip_block_attend.hpp"

namespace kvhip {

hipError_t launch_block_attend_bf16(const BlockAttend &x, hipStream_t stream) { return block_attend_dtype<1>(x, stream); }

}  // namespace kvhip
