// Host build of the chunks that a balanced launch over the 4-bit cache takes
// (colormlm_amd/csrc/s14_attn_plan.h)
#include <stdint.h>

#include "s14_attn_plan.h"

extern "C" uint32_t attn_balanced(uint64_t total, uint32_t fill, uint32_t least) { return s14::balanced_steps(total, fill, least); }

// Whether a kernel of so many row tiles is compiled with chunks that balance
extern "C" uint32_t attn_may_balance(uint32_t dim, uint32_t row_tiles) { return s14::paged_balances(dim, row_tiles); }

// The kernels that take a plan are launched by its head size and row tiles: 512 by 1 or 2, 256 by 1 or 4, others by 1, 2, 4 or 8
static_assert(!s14::paged_balances(512, 1) && s14::paged_balances(512, 2), "");
static_assert(!s14::paged_balances(256, 1) && !s14::paged_balances(256, 4), "");
static_assert(!s14::paged_balances(128, 4) && s14::paged_balances(128, 8) && !s14::paged_balances(64, 8), "");
