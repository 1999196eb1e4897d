// Work split of paged_attention: the rows of a workgroup, and the chunks that a
// long sequence is cut into.  Plain C++ (no HIP types): the library and a
// host-only test include it.
#pragma once

#include <cstdint>

namespace s14 {

// What a launch is planned by.  reach: the positions that the page table can
// hold, 2^31 - 2^16 at most; a promise (max_len) past it is one of that.
struct PagedShape {
  uint32_t seqs, heads, kv_heads, dim, max_new, max_len, window, reach;
};

// Work split of a paged launch.
struct PagedPlan {
  uint32_t row_tiles;  // 16-row tiles of a workgroup
  uint32_t staged;     // a row tile's K and V go through LDS (k_paged_rows)
  uint32_t rec_rows;   // rows of a chunk's partial result
  uint32_t chunk;      // tokens of one workgroup, a multiple of 64
  uint32_t chunks;     // of the longest sequence; above 1 the partial results go to the workspace
  uint32_t fused;      // the last workgroup of a row tile joins its chunks; else a second launch
  uint64_t blocks;     // workgroups
};
constexpr uint64_t kPagedPartFloats = 16ull << 20;  // the workspace: 64 MiB
constexpr uint32_t kPagedCounters = 16384;          // arrivals at a row tile, 0 between launches

// The chunks of a row tile that reads `span` tokens: the plan's, and larger
// ones where the sequence is longer than the launch was planned for.
struct PagedCut {
  uint32_t chunk, chunks;
};
constexpr PagedCut paged_cut(uint32_t span, uint32_t chunk, uint32_t chunks) {
  const uint32_t least = ((span + chunks - 1) / chunks + 63u) & ~63u;
  const uint32_t c = chunk > least ? chunk : least;
  return {c, (span + c - 1) / c};
}

// The end of the chunk that starts at begin <= hi, in 31 bits whatever the two
// and the chunk are.
constexpr int32_t paged_end(int32_t begin, int32_t hi, uint32_t chunk) {
  return uint32_t(hi - begin) > chunk ? begin + int32_t(chunk) : hi;
}

// Rows of a workgroup: all of the longest new block's up to 64 (of 32 of
// heads of 512), or K and V are read and turned into bf16 again for each row
// tile; 128 where there are more, at heads of 128, and more than 256 at heads
// of 64 (8 sequences of 64 new tokens of 3,000: 59 us, with tiles of 64 rows
// 64; 6 of 24 of up to 5,000, heads of 64: 27, with tiles of 128 38).  Up to
// 16 rows a wavefront reads K and V for itself; more go through LDS, but for
// one sequence of 32 rows, where a compute unit so has more bytes in flight
// (us, direct / staged: one of 40,000 tokens 24 / 28, 32 of 4,000 73 / 66, 3 of
// up to 51,525 40 / 30, 38 of up to 422, window 161, 18 / 12).
//
// Chunks.  Where the launch alone would leave compute units idle: as many
// workgroups as the card holds at once (a second round for a few of them costs
// as much as the first), of several sequences twice as many, since their
// lengths differ and short ones leave chunks empty (us, once / twice: 16
// sequences of up to 8,192 tokens 36 / 29 ragged, 55 / 55 equal; 4 of up to
// 9,000, 64 heads of 512, 49 / 37 and 56 / 72; 3 of 200 new of up to 6,000 96 /
// 80; 8 of 64 new of 3,000 51 / 59).  Where it fills the card: chunks of 2,048
// tokens, so that one long sequence does not outlast the rest.
//
// A row tile of 4 rows whose partial results stay within 64 KB is joined by its
// last workgroup, a row a wavefront (1 token of 4,097: 12.4 us with a second
// launch, 10.4 without; 32 rows of 2 chunks take it 9 us longer than a launch).
// Where a second launch would join them, a sequence of few steps is left whole
// (20 sequences of 300 tokens, 32 rows: 10 us, in two chunks 21; one of 500
// tokens and 8 of them 11, 20), and small chunks start at shorter ones (4 of 48
// rows of 300 tokens, heads of 256: 12 us in chunks of 64, 19 of 256).
inline PagedPlan paged_plan(const PagedShape &a) {
  PagedPlan p{};
  const uint64_t rows = uint64_t(a.max_new) * (a.heads / a.kv_heads);
  const uint32_t dim = a.dim;
  p.row_tiles = rows <= 16                          ? 1
                : dim == 512                        ? 2
                : rows <= 32 && dim <= 128          ? 2
                : rows > 64 && dim == 128           ? 8
                : rows > 256 && dim == 64           ? 8
                                                    : 4;
  p.staged = dim < 512 && (p.row_tiles >= 4 || (p.row_tiles == 2 && a.seqs > 1));
  const uint64_t tiles = (rows + 16 * p.row_tiles - 1) / (16 * p.row_tiles);
  const uint64_t base = tiles * a.kv_heads * a.seqs;  // workgroups of an uncut launch
  uint64_t span = a.max_len < a.reach ? a.max_len : a.reach;
  if (!span) span = 1;  // a chunk is never of no tokens: the kernels divide by it
  if (a.window && uint64_t(a.window) + a.max_new + 63 < span) span = uint64_t(a.window) + a.max_new + 63;
  // workgroups that the card holds at once, by a wavefront's registers and by LDS
  const uint32_t words = (dim == 512 ? 128 : dim) * p.row_tiles;
  const uint64_t per_cu = p.staged ? (dim == 256 ? 2 : (dim == 64 ? 4 : 3) - p.row_tiles / 8)
                                   : (words <= 64 ? 3 : words <= 128 || dim == 512 ? 2 : 1);
  const uint64_t slots = 256 * per_cu;
  const uint64_t least = dim == 512 ? 64 : !p.staged ? 256 : span <= 512 ? 64 : span <= 1024 ? 128 : 256;
  constexpr uint64_t kMost = 2048, kFuse = 64 * 1024;
  p.rec_rows = uint32_t(rows < 16 * p.row_tiles ? rows : 16 * p.row_tiles);
  const uint64_t rec = uint64_t(p.rec_rows) * (dim + 4);
  uint64_t chunks = base < slots ? slots * (a.seqs > 1 ? 2 : 1) / base : (span + kMost - 1) / kMost;
  const uint64_t fit = kPagedPartFloats / (rec * base);
  if (chunks > fit) chunks = fit;
  if (chunks > (span + least - 1) / least) chunks = (span + least - 1) / least;
  if (chunks < 1) chunks = 1;
  p.fused = chunks <= 64 && base <= kPagedCounters && p.rec_rows <= 4 && rec * 4 * chunks <= kFuse;
  if (!p.fused && span <= (dim == 512 ? 128 : dim == 256 ? 256 : 512)) chunks = 1;
  p.chunk = uint32_t(((span + chunks - 1) / chunks + least - 1) / least * least);
  p.chunks = uint32_t((span + p.chunk - 1) / p.chunk);
  p.blocks = base * p.chunks;
  return p;
}

}  // namespace s14
