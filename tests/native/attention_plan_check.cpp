// Host build of paged_attention's work split (colormlm_amd/csrc/
// s14_attn_plan.h) for the CPU test of its limits.
#include <stdint.h>

#include "s14_attn_plan.h"

// shape: seqs, heads, key heads, dim, max_new, max_len, window, reach;
// plan: row tiles, rows of a record, chunk, chunks, fused, workgroups
extern "C" void attn_plan(const uint32_t shape[8], uint64_t plan[6]) {
  const s14::PagedPlan p = s14::paged_plan({shape[0], shape[1], shape[2], shape[3], shape[4], shape[5], shape[6], shape[7]});
  plan[0] = p.row_tiles, plan[1] = p.rec_rows, plan[2] = p.chunk, plan[3] = p.chunks, plan[4] = p.fused, plan[5] = p.blocks;
}

extern "C" void attn_cut(uint32_t span, uint32_t chunk, uint32_t chunks, uint32_t cut[2]) {
  const s14::PagedCut c = s14::paged_cut(span, chunk, chunks);
  cut[0] = c.chunk, cut[1] = c.chunks;
}

extern "C" int32_t attn_end(int32_t begin, int32_t hi, uint32_t chunk) { return s14::paged_end(begin, hi, chunk); }

extern "C" void attn_limits(uint64_t *part_floats, uint32_t *counters) {
  *part_floats = s14::kPagedPartFloats;
  *counters = s14::kPagedCounters;
}
