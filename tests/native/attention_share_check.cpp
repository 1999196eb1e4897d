// Host build of the attention operands' overlap test (colormlm_amd/csrc/
// s14_attn_share.h).
#include <stdint.h>

#include "s14_attn_share.h"

// a, b: at, token, head, row (bytes), heads
extern "C" int attn_share(const uint64_t a[5], const uint64_t b[5], uint32_t tokens, int own) {
  const s14::RowBytes x{a[0], a[1], a[2], a[3], uint32_t(a[4])}, y{b[0], b[1], b[2], b[3], uint32_t(b[4])};
  return s14::rows_share(x, y, tokens, own != 0);
}
