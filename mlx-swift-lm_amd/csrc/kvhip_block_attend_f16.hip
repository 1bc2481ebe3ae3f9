// The float16 instances of the block-scaled attention kernel.
#include "kvhip_block_attend.hpp"

namespace kvhip {

hipError_t launch_block_attend_f16(const BlockAttend &x, hipStream_t stream) { return block_attend_dtype<0>(x, stream); }

}  // namespace kvhip
