// What the paged attention kernels of both caches share: which rows and cached
// tokens a workgroup works on, how it finds their pages, and how the partial
// results of a long sequence's chunks are joined.  Unnamed namespace: each
// kernel file gets its own copy.
#pragma once

#include "s14_attn.hpp"
#include "s14_attn_util.hpp"
#include "s14_device_util.hpp"

namespace s14 {
namespace {

// What a row tile of a sequence reads: tokens lo .. hi - 1 in chunks of
// `chunk` (a multiple of 64, as lo is).  Its rows see none before `seen`.
struct Span {
  uint32_t first, rows;  // first packed token; (token, head) rows of the sequence
  int32_t len, pos0, seen, lo, hi;
  uint32_t chunk, chunks;
  uint32_t wrong;  // status: its length is outside the table, or it has rows that no workgroup takes
};

// The sum of v over a wavefront.
__device__ __forceinline__ uint32_t wave_sum_u32(uint32_t v) {
  v += uint32_t(dpp_i<0xb1>(0, int(v)));   // quad_perm [1,0,3,2]
  v += uint32_t(dpp_i<0x4e>(0, int(v)));   // quad_perm [2,3,0,1]
  v += uint32_t(dpp_i<0x141>(0, int(v)));  // row_half_mirror
  v += uint32_t(dpp_i<0x140>(0, int(v)));  // row_mirror
  return __builtin_amdgcn_readlane(v, 0) + __builtin_amdgcn_readlane(v, 16) + __builtin_amdgcn_readlane(v, 32) +
         __builtin_amdgcn_readlane(v, 48);
}

// The chunk of a plan that balances (PagedPlan::fill): the cached tokens that the
// launch reads in all, over the workgroups that shall have them.  The same in every
// wavefront.
__device__ __forceinline__ uint32_t balanced_chunk(const PagedArgs &a, const PagedPlan &p) {
  uint32_t steps = 0;  // of 64 tokens: up to 2^25 of a sequence, of kMostBalanced / 64 sequences a lane
  const int64_t room = int64_t(a.table_width) * a.cache.page;
  for (uint32_t s = threadIdx.x & 63u; s < a.seqs; s += 64) {
    const int64_t n = clamp_row(a.cu[s + 1], a.tokens) - clamp_row(a.cu[s], a.tokens), len = a.len[s];
    const int64_t hi = n <= 0 || len < 0 ? 0 : len < room ? len : room;
    const int64_t lo = a.window && hi - n - a.window + 1 > 0 ? hi - n - a.window + 1 : 0;
    if (hi > lo) steps += uint32_t((hi - (lo & ~63ll) + 63) >> 6);
  }
  const uint64_t total = (uint64_t(wave_sum_u32(steps >> 16)) << 16) + wave_sum_u32(steps & 0xffffu);
  return 64 * balanced_steps(total, p.fill, p.least / 64);
}

__device__ __forceinline__ Span paged_span(const PagedArgs &a, const PagedPlan &p, uint32_t seq, uint32_t row0, uint32_t planned) {
  Span s;
  const uint32_t group = a.heads / a.cache.heads;
  s.first = uint32_t(clamp_row(a.cu[seq], a.tokens));
  const int32_t n = int32_t(clamp_row(a.cu[seq + 1], a.tokens)) - int32_t(s.first);
  // no more rows than the launch was planned for: below 2^31 in all
  s.rows = n <= 0 ? 0u : (uint32_t(n) < a.max_new ? uint32_t(n) : a.max_new) * group;
  const int64_t room = int64_t(a.table_width) * a.cache.page;
  const int64_t len = a.len[seq];
  s.len = int32_t(len < 0 ? 0 : len < room ? len : room);
  s.wrong = n > 0 && (len != s.len || uint32_t(n) > a.max_new) ? kStatusBadCounts : 0u;
  s.pos0 = s.len - n;
  const uint32_t last = (row0 + 16 * p.row_tiles < s.rows ? row0 + 16 * p.row_tiles : s.rows) - 1;
  const int32_t first_pos = s.pos0 + int32_t(row0 / group), last_pos = s.pos0 + int32_t(last / group);
  s.hi = last_pos + 1 < 0 ? 0 : last_pos + 1;
  const int64_t lo = a.window ? int64_t(first_pos) - a.window + 1 : 0;
  s.seen = int32_t(lo < 0 ? 0 : lo);
  s.lo = s.seen & ~63;
  const uint32_t span = s.hi > s.lo ? s.hi - s.lo : 0;
  const PagedCut cut = paged_cut(span, planned, p.chunks);
  s.chunk = cut.chunk, s.chunks = cut.chunks;
  return s;
}

__device__ __forceinline__ Span paged_span(const PagedArgs &a, const PagedPlan &p, uint32_t seq, uint32_t row0) {
  return paged_span(a, p, seq, row0, p.chunk);
}

// The same of a kernel whose plans may balance (paged_balances).  The joining launch
// takes the chunk from the end of the workspace.
__device__ __forceinline__ uint32_t *chunk_word(float *part) { return reinterpret_cast<uint32_t *>(part + kPagedPartFloats - 4); }
template <bool kBalanced>
__device__ __forceinline__ Span balanced_span(const PagedArgs &a, const PagedPlan &p, uint32_t seq, uint32_t row0, float *part) {
  uint32_t planned = p.chunk;
  if (kBalanced && p.fill) {
    planned = balanced_chunk(a, p);
    if (blockIdx.x == 0 && threadIdx.x == 0) *chunk_word(part) = planned;
  }
  return paged_span(a, p, seq, row0, planned);
}
template <bool kBalanced>
__device__ __forceinline__ Span joined_span(const PagedArgs &a, const PagedPlan &p, uint32_t seq, uint32_t row0, const float *part) {
  return paged_span(a, p, seq, row0, kBalanced && p.fill ? *chunk_word(const_cast<float *>(part)) : p.chunk);
}

__device__ __forceinline__ void store_out(const AttnOut &o, uint64_t at, float a, float b, float c, float d) {
  if (o.bf16)
    *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(o.p) + at) = make_uint2(bf16_pair(a, b), bf16_pair(c, d));
  else
    *reinterpret_cast<float4 *>(static_cast<float *>(o.p) + at) = make_float4(a, b, c, d);
}

// What a workgroup works on.  Row tiles, which read the same pages, are 8
// workgroups apart, on one XCD at about the same time (64 sequences of 4,000
// tokens, 64 heads of 512 in two row tiles: 118 us a whole launch apart, 105 so;
// 4 of 100 new of up to 4,000: 63 and 48).  Chunks are the slowest index of the
// others, so that the late chunks, which short sequences lack, are together:
// among the sequences the empty workgroups fell to the same compute units (128
// ragged sequences of 8,192 tokens at most, 4 chunks: 228 us; 160 now).
// Workgroup i runs on XCD i % 8: where (sequence, key head) pairs are few, a
// chunk's pairs are rotated each time their start comes back to the first XCD,
// or one long sequence would have but some of the XCDs.
struct Item {
  uint32_t tile, chunk, seq, head;
};
__device__ __forceinline__ Item item_of(const PagedArgs &a, const PagedPlan &p, uint32_t kvh) {
  const uint32_t pairs = kvh * a.seqs, items = pairs * p.chunks;
  const uint32_t tiles = gridDim.x / items, whole = items & ~7u, i = blockIdx.x;
  uint32_t tile, item;
  if (i < whole * tiles) {
    tile = i / 8 % tiles, item = i / (8 * tiles) * 8 + i % 8;
  } else {
    tile = (i - whole * tiles) / (items - whole), item = whole + (i - whole * tiles) % (items - whole);
  }
  const uint32_t chunk = item / pairs;
  const uint32_t zeros = __builtin_ctz(pairs | 8u);
  const uint32_t pair = (item % pairs + (chunk >> (3 - zeros))) % pairs;
  return {tile, chunk, pair / kvh, pair % kvh};
}

__device__ __forceinline__ uint64_t record_of(const PagedArgs &a, const PagedPlan &p, const Item &i, uint32_t kvh) {
  return ((uint64_t(i.tile) * p.chunks + i.chunk) * a.seqs + i.seq) * kvh + i.head;
}

// What a wavefront needs to find a step's pages.  A lane's tokens, 4 T
// neighbours, lie in one page; tokens behind the sequence take its last page,
// tokens of the first 64 before the window its first one (both are masked: what
// a table holds for pages that nobody sees is not looked at).  An id is looked
// at when it is used, a step after its load: looking at once would wait for
// every load in flight.
struct Pages {
  const int32_t *table;
  int32_t seen, last;
  uint32_t pages, shift;
  __device__ __forceinline__ int32_t id(int32_t tok) const { return table[uint32_t(min(max(tok, seen), last)) >> shift]; }
  __device__ __forceinline__ uint32_t checked(int32_t id, bool &bad) const {
    const bool out = uint32_t(id) >= pages;
    bad |= out;
    return out ? 0u : uint32_t(id);
  }
};

// A row of a chunk's partial result: D sums, the maximum and the weights' sum.
template <int D>
constexpr uint32_t kRecord = D + 4;

// Where the chunks of a row are joined.  A second launch costs about 4 us, its
// workgroups share the rows; the workgroup that arrives last at a (row tile,
// sequence, key head) does it at once, but reads all its partial results
// alone: the plan fuses where those are few (PagedPlan::fused: 4 rows at the most).
//
// The last one sees the others' results, across the XCDs, because they are
// written through to the device's coherence point (agent scope, sc1), each
// wavefront waits for its stores before the barrier that precedes the count,
// and they are read from there.  A release fence would write back the L2.
constexpr int kAgent = 0x10;  // buffer cache policy: sc1

// kFuse: the kernel has plans that fuse (those of one row tile).
template <bool kFuse>
struct PartStore {
  __amdgpu_buffer_rsrc_t r;
  uint32_t fused;
  float *p;
  __device__ __forceinline__ PartStore(float *rec, uint32_t floats, uint32_t fused) : fused(fused), p(rec) {
    r = __builtin_amdgcn_make_buffer_rsrc(rec, 0, int(floats * 4), 0x00020000);
  }
  __device__ __forceinline__ void operator()(uint32_t at, f32x4 v) const {
    if (kFuse && fused)
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), r, at * 4, 0, kAgent);
    else
      *reinterpret_cast<f32x4 *>(p + at) = v;
  }
};

// Counts this workgroup's arrival; true in every thread of the last one.
__device__ __forceinline__ bool arrived_last(uint32_t *count, uint32_t chunks) {
  __shared__ uint32_t s_last;
  __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): this wavefront's stores are done
  __syncthreads();
  if (threadIdx.x == 0) {
    const bool last = __hip_atomic_fetch_add(count, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1 == chunks;
    if (last) __hip_atomic_store(count, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);  // for the next launch
    s_last = last;
  }
  __syncthreads();
  return s_last != 0;
}

// Row row0 + k of a tile from its partial results, by one wavefront: lane c
// holds chunk c's maximum and sum (64 chunks at most), then the chunks' rows in
// order, the first of them loaded with the maxima.
template <int D, int kPolicy>
__device__ __forceinline__ void join_row(const PagedArgs &a, const PagedPlan &p, const Span &sp, const Item &it,
                                         uint32_t row0, uint32_t k, const float *part) {
  constexpr uint32_t kLanes = D / 4 < 64 ? D / 4 : 64, kSpan = D / (4 * kLanes), kSets = 64 / kLanes;
  const uint32_t kvh = a.cache.heads, group = a.heads / kvh, l = threadIdx.x & 63u;
  const uint32_t lane = l % kLanes, set = l / kLanes;
  const uint64_t rec = uint64_t(p.rec_rows) * kRecord<D>;
  const uint32_t next = uint32_t(uint64_t(kvh) * a.seqs * rec * 4);  // bytes to the next chunk's record
  const float *first = part + record_of(a, p, Item{it.tile, 0, it.seq, it.head}, kvh) * rec;
  const auto r = __builtin_amdgcn_make_buffer_rsrc(const_cast<float *>(first), 0,
                                                   int((sp.chunks - 1) * next + uint32_t(rec) * 4), 0x00020000);
  const uint32_t at = k * kRecord<D> * 4;
  constexpr uint32_t kAt = D == 512 ? 4 : 8;  // loads of each lane at once
  u32x4 x[kAt][kSpan];
  const auto load = [&](uint32_t c0) {
#pragma unroll
    for (uint32_t j = 0; j < kAt; ++j)
#pragma unroll
      for (uint32_t i = 0; i < kSpan; ++i)  // past the last chunk: zeros (descriptor range), weight 0
        x[j][i] = __builtin_amdgcn_raw_buffer_load_b128(
            r, (c0 + j * kSets + set) * next + at + 16 * (lane + kLanes * i), 0, kPolicy);
  };
  // lanes without a chunk: past the range too
  const auto ml = __builtin_amdgcn_raw_buffer_load_b64(r, l * next + at + D * 4, 0, kPolicy);
  load(0);
  const float m = l < sp.chunks ? __uint_as_float(ml[0]) : -INFINITY, sum = l < sp.chunks ? __uint_as_float(ml[1]) : 0.0f;
  float top = m;
#pragma unroll
  for (int d = 32; d; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
  const float w = __builtin_amdgcn_exp2f(m - (top == -INFINITY ? 0.0f : top));  // 0 in lanes without a chunk
  float total = sum * w;
#pragma unroll
  for (int d = 32; d; d >>= 1) total += __shfl_xor(total, d);
  f32x4 o[kSpan] = {};
  for (uint32_t c0 = 0;;) {
#pragma unroll
    for (uint32_t j = 0; j < kAt; ++j) {
      const float f = __shfl(w, int((c0 + j * kSets + set) & 63u));
      const bool in = c0 + j * kSets + set < sp.chunks;
#pragma unroll
      for (uint32_t i = 0; i < kSpan; ++i) o[i] += __builtin_bit_cast(f32x4, x[j][i]) * (in ? f : 0.0f);
    }
    c0 += kAt * kSets;
    if (c0 >= sp.chunks) break;
    load(c0);
  }
#pragma unroll
  for (uint32_t d = kLanes; d < 64; d <<= 1)
#pragma unroll
    for (uint32_t i = 0; i < kSpan; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[i][e] += __shfl_xor(o[i][e], int(d));
  const uint32_t row = row0 + k;
  const uint64_t t = uint64_t(sp.first + row / group);
  const uint32_t h = it.head * group + row % group;
  if constexpr (D < 512) total = checked_sum(total, top);  // (k_paged_wide scales its scores before it compares them)
  const float inv = total == 0.0f ? 0.0f : 1.0f / total;
  if (set == 0) {
#pragma unroll
    for (uint32_t i = 0; i < kSpan; ++i) {
      const f32x4 y = o[i] * inv;
      store_out(a.out, t * a.out.token + uint64_t(h) * a.out.head + 4 * (lane + kLanes * i), y[0], y[1], y[2], y[3]);
    }
  }
  if (a.lse && l == 0) a.lse[t * a.heads + h] = total == 0.0f ? -INFINITY : top * kLn2 + __logf(total);
}

// All rows of a tile, by its last workgroup.
template <int D>
__device__ __forceinline__ void join_tile(const PagedArgs &a, const PagedPlan &p, const Span &sp, const Item &it,
                                          uint32_t row0, const float *part) {
  for (uint32_t k = threadIdx.x / 64; k < p.rec_rows && row0 + k < sp.rows; k += 4)
    join_row<D, kAgent>(a, p, sp, it, row0, k, part);
}

// Joins the chunks of one row a workgroup, in an order that its size alone
// sets: the chunks' maxima in the lanes, then their rows in groups of
// threads at once.
template <int D, bool kBalanced>
__global__ __launch_bounds__(256) void k_paged_join(PagedArgs a, PagedPlan p, const float *part) {
  constexpr uint32_t kLanes = D / 4 < 64 ? D / 4 : 64, kSpan = D / (4 * kLanes);  // float4s of a row a thread
  constexpr uint32_t kGroups = 256 / kLanes;
  const uint32_t kvh = a.cache.heads, group = a.heads / kvh, tid = threadIdx.x;
  const uint32_t seq = blockIdx.y, head = blockIdx.z, r = blockIdx.x;
  const uint32_t per = 16 * p.row_tiles, tile = r / per;
  const Span sp = joined_span<kBalanced>(a, p, seq, tile * per, part);
  if (r >= sp.rows || sp.chunks <= 1) return;
  const uint64_t rec = uint64_t(p.rec_rows) * kRecord<D>;
  const float *row = part + record_of(a, p, Item{tile, 0, seq, head}, kvh) * rec + r % per * kRecord<D>;
  const uint64_t next = uint64_t(kvh) * a.seqs * rec;  // the next chunk's record
  float top = -INFINITY;
  for (uint32_t c = tid & 63u; c < sp.chunks; c += 64) top = fmaxf(top, row[c * next + D]);
#pragma unroll
  for (int m = 32; m; m >>= 1) top = fmaxf(top, __shfl_xor(top, m));
  const float at = top == -INFINITY ? 0.0f : top;
  const uint32_t lane = tid % kLanes, first = tid / kLanes;
  float total = 0.0f;
  f32x4 o[kSpan] = {};
#pragma unroll 4
  for (uint32_t c = first; c < sp.chunks; c += kGroups) {
    const float *x = row + c * next;
    const float fade = __builtin_amdgcn_exp2f(x[D] - at);
    total += x[D + 1] * fade;
#pragma unroll
    for (uint32_t i = 0; i < kSpan; ++i) o[i] += *reinterpret_cast<const f32x4 *>(x + 4 * (lane + kLanes * i)) * fade;
  }
  __shared__ f32x4 s_o[kGroups][kSpan][kLanes];
  __shared__ float s_l[kGroups];
#pragma unroll
  for (uint32_t i = 0; i < kSpan; ++i) s_o[first][i][lane] = o[i];
  if (lane == 0) s_l[first] = total;
  __syncthreads();
  if (first) return;
#pragma unroll
  for (uint32_t w = 1; w < kGroups; ++w) {
    total += s_l[w];
#pragma unroll
    for (uint32_t i = 0; i < kSpan; ++i) o[i] += s_o[w][i][lane];
  }
  const uint64_t t = uint64_t(sp.first + r / group);
  const uint32_t h = head * group + r % group;
  if constexpr (D < 512) total = checked_sum(total, top);  // (wide heads: as in k_paged_wide)
  const float inv = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
  for (uint32_t i = 0; i < kSpan; ++i) {
    const f32x4 y = o[i] * inv;
    store_out(a.out, t * a.out.token + uint64_t(h) * a.out.head + 4 * (lane + kLanes * i), y[0], y[1], y[2], y[3]);
  }
  if (a.lse && lane == 0) a.lse[t * a.heads + h] = total == 0.0f ? -INFINITY : top * kLn2 + __logf(total);
}

// Up to 16 chunks of a row: a row a wavefront, which reads them at once (128
// rows of 8 sequences, 8 key heads, 8 chunks, 69 MB: 78 us with the attention,
// a row a workgroup 98).
template <int D, bool kBalanced>
__global__ __launch_bounds__(256) void k_paged_join_rows(PagedArgs a, PagedPlan p, const float *part) {
  const uint32_t r = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + threadIdx.x / 64), per = 16 * p.row_tiles;
  const Item it{r / per, 0, blockIdx.y, blockIdx.z};
  const Span sp = joined_span<kBalanced>(a, p, it.seq, it.tile * per, part);
  if (r >= sp.rows || sp.chunks <= 1) return;
  join_row<D, 0>(a, p, sp, it, it.tile * per, r % per, part);
}

template <int D, bool kBalanced = false, class Kernel>
hipError_t launch(hipStream_t s, const PagedArgs &a, const PagedPlan &p, float *part, Kernel kernel) {
  kernel<<<uint32_t(p.blocks), 256, 0, s>>>(a, p, part);
  if (p.chunks > 1 && !p.fused) {
    const uint32_t rows = uint32_t(a.max_new) * (a.heads / a.cache.heads);
    if (p.chunks <= 16)
      k_paged_join_rows<D, kBalanced><<<dim3((rows + 3) / 4, a.seqs, a.cache.heads), 256, 0, s>>>(a, p, part);
    else
      k_paged_join<D, kBalanced><<<dim3(rows, a.seqs, a.cache.heads), 256, 0, s>>>(a, p, part);
  }
  return hipGetLastError();
}

}  // namespace
}  // namespace s14
