// Host build of the chunks that a balanced launch over the 4-bit cache takes
// (colormlm_amd/csrc/s14_attn_plan.h)
#include <stdint.h>

#include "s14_attn_plan.h"

extern "C" uint32_t attn_balanced(uint64_t total, uint32_t fill, uint32_t least) { return s14::balanced_steps(total, fill, least); }
