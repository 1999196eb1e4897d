// Attention of new tokens over the paged 8-bit cache.
//
// Both products run on v_mfma_f32_16x16x32_bf16 with the tokens as the rows:
// S^T = K Q^T, then O^T = V^T P^T.  The result layout of the first (lane = 16
// g + n holds query row n, four tokens of each 16-token tile) is the operand
// layout of the second, if each 16-token tile t of a step takes the tokens
// 4 T g + 4 t + i (T tiles a step, i < 4) as its rows: P stays in its lane's
// registers.  A lane's V operand is then 4 T neighbouring tokens of one
// dimension, which is why V pages lie [dim][slot].  E4M3 codes become bf16
// exactly, so the products are of the stored values; page scales multiply the
// scores (K) and the codes as they become bf16 (V; on the weights the scale of
// an infinity's page would pass bf16's range), and are one per lane, since the
// 4 T tokens of a lane group lie in one page.
//
// A row is a (token, query head of the key head) pair: the group's heads share
// the K and V that are read.  Up to 16 rows (k_paged_attention), the four
// wavefronts of a workgroup take steps of 16 T tokens in turn and join through
// LDS; with more rows they share the tokens' codes through LDS (k_paged_rows),
// or, with heads of 512, the dimensions (k_paged_wide).  A long sequence is cut
// into chunks of workgroups, whose partial results are joined by the last of
// them or by a second launch.  Few rows are bound by the cache's bytes: 128
// sequences of up to 8,192 tokens, 8 key heads of 128, 160 us, 4.8 TB/s.
#include "s14_attn.hpp"
#include "s14_attn_util.hpp"
#include "s14_device.hpp"

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

__device__ __forceinline__ Span paged_span(const PagedArgs &a, const PagedPlan &p, uint32_t seq, uint32_t row0) {
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
  const PagedCut cut = paged_cut(span, p.chunk, p.chunks);
  s.chunk = cut.chunk, s.chunks = cut.chunks;
  return s;
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

// The least code that is no finite bf16 value at a page's scale: the NaN code,
// and at scales from 2^120 on, which an infinity's page has, large ones.
__device__ __forceinline__ uint32_t odd_code(uint32_t scale) { return scale < 247u ? 0x7fu : 0x78u - 8u * (scale - 247u); }

// The top bit of each byte whose code is `from` (0x7f at the most) or larger in magnitude.
__device__ __forceinline__ uint32_t odd_codes(uint32_t c, uint32_t from) {
  return ((c & 0x7f7f7f7fu) + (0x80u - from) * 0x01010101u) & 0x80808080u;
}

// Those bytes as zeros.
__device__ __forceinline__ uint32_t no_odd(uint32_t c, uint32_t from) { return c & ~((odd_codes(c, from) >> 7) * 0xffu); }

// What such a code stands for: NaN or an infinity; of another 0.
__device__ __forceinline__ float odd_value(uint32_t c, uint32_t from) {
  return (c & 0x7fu) < from ? 0.0f : __uint_as_float((c & 0x7fu) == 0x7fu ? 0x7fc00000u : 0x7f800000u | ((c & 0x80u) << 24));
}

template <int D, int NT>
__global__ __launch_bounds__(256, D * NT <= 64 ? 4 : D * NT <= 128 ? 2 : 1) void k_paged_attention(PagedArgs a, PagedPlan p, float *part) {
  constexpr int T = 4;        // 16-token tiles a step
  constexpr int C = D / 64;   // 16-byte pieces of a K row a lane holds
  constexpr int DT = D / 16;  // 16-dimension tiles of O
  constexpr int W = T;        // 32-bit words of V codes a lane holds of one dimension
  const uint32_t kvh = a.cache.heads, group = a.heads / kvh;
  const Item it = item_of(a, p, kvh);
  const uint32_t tile = it.tile, head = it.head, seq = it.seq, chunk = it.chunk;
  const uint32_t row0 = tile * 16 * NT;
  const Span sp = paged_span(a, p, seq, row0);
  if (row0 >= sp.rows || (chunk && chunk >= sp.chunks)) return;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), l = threadIdx.x & 63u, n = l & 15u, g = l >> 4;
  const uint32_t P = a.cache.page;
  const uint32_t shift = __builtin_ctz(P);
  const Pages pages{a.page_table + uint64_t(seq) * a.table_width, sp.seen, sp.len - 1, a.cache.pages, shift};
  const int32_t begin = sp.lo + int32_t(chunk * sp.chunk);
  const int32_t end = paged_end(begin, sp.hi, sp.chunk);

  // each lane's row of every tile: its position, and Q in the operand layout
  Visible see[NT];
  bf16x8 q[NT][2 * C];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const uint32_t r = row0 + 16 * nt + n;
    const uint32_t rr = r < sp.rows ? r : sp.rows - 1;
    see[nt] = Visible(sp.pos0 + int32_t(rr / group), a.window);
    const uint16_t *row = a.q + uint64_t(sp.first + rr / group) * a.q_token +
                          uint64_t(head * group + rr % group) * a.q_head;
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int h = 0; h < 2; ++h) q[nt][2 * c + h] = *reinterpret_cast<const bf16x8 *>(row + 64 * c + 16 * g + 8 * h);
  }
  const int32_t pos_lo = sp.pos0 + int32_t(row0 / group);
  const int32_t pos_hi = sp.hi - 1;

  f32x4 o[NT][DT] = {};
  float m[NT], sum[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) m[nt] = -INFINITY, sum[nt] = 0.0f;
  bool bad = false, odd = false;
  const float scale = a.scale * kLog2e;
  const uint64_t page_bytes = uint64_t(P) * D;

  // A step's operands: codes in registers, loaded one step ahead (K as soon as
  // the first product has read the step before, V after the second), their
  // pages' ids another step ahead.
  uint4 kk[T][C];
  uint32_t vv[DT][W];
  uint8_t ksc = 0, vsc = 0;  // (as loaded: widened where they are used, not while in flight)
  int32_t idk = 0, idv = 0;  // of the next step
  uint32_t pagev = 0;
  auto load_ids = [&](int32_t b, int32_t &k, int32_t &v) {
    k = pages.id(b + 4 * T * int32_t(n / 4));
    v = pages.id(b + 4 * T * int32_t(g));
  };
  auto load_k = [&](int32_t b) {
    const uint32_t at = (uint32_t(b + 4 * T * int32_t(n / 4)) & (P - 1)) + (n & 3u);
    pagev = pages.checked(idv, bad);
    const uint64_t sat = uint64_t(pagev) * kvh + head;
    ksc = a.cache.ks[sat], vsc = a.cache.vs[sat];  // first: they are waited for before K
    const uint8_t *kp = a.cache.k + (uint64_t(pages.checked(idk, bad)) * kvh + head) * page_bytes + at * uint32_t(D) + 16 * g;
#pragma unroll
    for (int t = 0; t < T; ++t)
#pragma unroll
      for (int c = 0; c < C; ++c) kk[t][c] = *reinterpret_cast<const uint4 *>(kp + 4 * t * D + 64 * c);
  };
  auto load_v = [&](int32_t b) {
    const uint8_t *vp = a.cache.v + (uint64_t(pagev) * kvh + head) * page_bytes + n * P +
                        (uint32_t(b + 4 * T * int32_t(g)) & (P - 1));
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      const uint4 x = *reinterpret_cast<const uint4 *>(vp + 16 * dt * P);
      vv[dt][0] = x.x, vv[dt][1] = x.y, vv[dt][2] = x.z, vv[dt][3] = x.w;
    }
  };
  constexpr int32_t kStride = 4 * 16 * T;  // the wavefronts' steps interleave
  int32_t b = begin + 16 * T * int32_t(wave);
  const int32_t last = b + (end - 1 - b) / kStride * kStride;
  if (b < end) {
    int32_t idk1, idv1;
    load_ids(b, idk, idv);
    load_ids(min(b + kStride, last), idk1, idv1);
    load_k(b);
    load_v(b);
    // waited for here and not, with K and V, in every step
    asm volatile("" : "+v"(idk1), "+v"(idv1));
    idk = idk1, idv = idv1;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2 * C; ++c) asm volatile("; a step's operands" : "+v"(q[nt][c]));
  } else {  // on this way to the loop too; in other words, or both would be done where the ways meet
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2 * C; ++c) asm volatile("; no step" : "+v"(q[nt][c]));
  }

  for (; b < end; b += kStride) {
    const int32_t tv = b + 4 * T * int32_t(g);
    // past the last step that step's again: a load behind a branch makes every
    // later wait one for all loads
    const int32_t next = min(b + kStride, last);
    int32_t idk2, idv2;  // ahead of the K and V loads below
    load_ids(min(b + 2 * kStride, last), idk2, idv2);
    const float ks = fmaxf(scale * power_of_two(int(ksc) - 127), 0x1p-126f);  // above 0: a masked score stays -inf
    const float vs = power_of_two(int(vsc) - 127);
    f32x4 s[NT][T];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int t = 0; t < T; ++t) s[nt][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int t = 0; t < T; ++t)
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const bf16x8 k0 = e4m3_bf16(kk[t][c].x, kk[t][c].y), k1 = e4m3_bf16(kk[t][c].z, kk[t][c].w);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          s[nt][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k0, q[nt][2 * c], s[nt][t], 0, 0, 0);
          s[nt][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k1, q[nt][2 * c + 1], s[nt][t], 0, 0, 0);
        }
      }
    load_k(next);
    const bool partial = b + 16 * T - 1 > pos_lo || (a.window && int64_t(b) <= int64_t(pos_hi) - a.window);
    bf16x8 pb[NT][T / 2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float x[4 * T];
#pragma unroll
      for (int i = 0; i < 4 * T; ++i) x[i] = s[nt][i / 4][i % 4];
      if (partial) {
        keep_branch();
#pragma unroll
        for (int i = 0; i < 4 * T; ++i) x[i] = see[nt](tv + i) ? x[i] : -INFINITY;
      }
      float top = x[0];
#pragma unroll
      for (int i = 1; i < 4 * T; ++i) top = fmaxf(top, x[i]);
      top = fmaxf(m[nt], max_lane16(top * ks));
      // the maximum that the weights are taken from moves only where they
      // would pass 2^kRise: O is seldom multiplied
      if (__any(top > m[nt] + kRise)) {
        const float fade = __builtin_amdgcn_exp2f(m[nt] - (top == -INFINITY ? 0.0f : top));
        m[nt] = top;
        sum[nt] *= fade;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[nt][dt] *= fade;
      }
      const float at = m[nt] == -INFINITY ? 0.0f : m[nt];  // no key seen yet: every weight 0
      u32x4 w[T / 2];
#pragma unroll
      for (int t = 0; t < T; ++t) {
        float e[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[4 * t + i], ks, -at));
          sum[nt] += e[i];
        }
        // rounded to bf16, half a step of each weight: the matrix operand's type
        w[t / 2][2 * (t & 1)] = bf16_pair(e[0], e[1]);
        w[t / 2][2 * (t & 1) + 1] = bf16_pair(e[2], e[3]);
      }
#pragma unroll
      for (int u = 0; u < T / 2; ++u) pb[nt][u] = __builtin_bit_cast(bf16x8, w[u]);
    }
    if (partial) {
      // what lies behind the sequence is not read; a NaN or infinity that some
      // row must not see leaves the product (0 times it is NaN), and the rows
      // that see it get it back below
      uint32_t found = 0;
      const uint32_t from = odd_code(__float_as_uint(vs) >> 23);  // (vsc is the next step's)
#pragma unroll
      for (int k = 0; k < W; ++k) {
        const int32_t left = sp.len - (tv + 4 * k);
        const uint32_t keep = left >= 4 ? ~0u : left <= 0 ? 0u : (1u << (8 * left)) - 1u;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) vv[dt][k] &= keep, found |= odd_codes(vv[dt][k], from);
      }
      if (__any(found != 0)) {
        odd = true;
#pragma unroll
        for (int k = 0; k < W; ++k)
#pragma unroll
          for (int dt = 0; dt < DT; ++dt) vv[dt][k] = no_odd(vv[dt][k], from);
      }
    }
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int u = 0; u < T / 2; ++u) {
        const bf16x8 v = e4m3_bf16(vv[dt][2 * u], vv[dt][2 * u + 1], vs);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
          o[nt][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, pb[nt][u], o[nt][dt], 0, 0, 0);
      }
    load_v(next);
    idk = idk2, idv = idv2;
  }

  if (odd) {  // uniform, and rare: one token after the other
    for (int32_t b0 = begin + 16 * T * int32_t(wave); b0 < end; b0 += kStride) {
      if (b0 + 16 * T - 1 <= pos_lo && !(a.window && int64_t(b0) <= int64_t(pos_hi) - a.window)) continue;
      for (int32_t j = b0; j < min(b0 + 16 * T, sp.len); ++j) {
        const uint64_t at = uint64_t(pages.checked(pages.id(j), bad)) * kvh + head;
        const uint32_t from = odd_code(a.cache.vs[at]);
        const uint8_t *vp = a.cache.v + at * page_bytes + (uint32_t(j) & (P - 1));
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          f32x4 odds;
#pragma unroll
          for (int i = 0; i < 4; ++i) odds[i] = odd_value(vp[(16 * dt + 4 * g + i) * P], from);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const bool in = see[nt](j);
            f32x4 back;
#pragma unroll
            for (int i = 0; i < 4; ++i) back[i] = in ? odds[i] : 0.0f;
            o[nt][dt] += back;
          }
        }
      }
    }
  }

  // join the four wavefronts: 2 and 3 into 0 and 1, then 1 into 0
  __shared__ float s_m[4][NT][16], s_l[4][NT][16];
  __shared__ f32x4 s_o[2][NT * DT][64];
  const bool bad_page = __any(bad);
  if (const uint32_t status = sp.wrong | (bad_page ? kStatusBadCachePage : 0u); status && l == 0) atomicOr(a.status, status);
  if (bad_page) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) sum[nt] = __uint_as_float(0x7fc00000u);
  }
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    sum[nt] = sum_lane16(sum[nt]);
    if (g == 0) s_m[wave][nt][n] = m[nt], s_l[wave][nt][n] = sum[nt];
  }
  __syncthreads();
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    float top = s_m[0][nt][n];
#pragma unroll
    for (int w = 1; w < 4; ++w) top = fmaxf(top, s_m[w][nt][n]);
    const float at = top == -INFINITY ? 0.0f : top;
    float total = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; ++w) total += s_l[w][nt][n] * __builtin_amdgcn_exp2f(s_m[w][nt][n] - at);
    const float fade = __builtin_amdgcn_exp2f(m[nt] - at);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[nt][dt] *= fade;
    m[nt] = top, sum[nt] = total;
  }
#pragma unroll
  for (int half = 2; half; half >>= 1) {
    if (wave >= uint32_t(half) && wave < 2 * uint32_t(half)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) s_o[wave - half][nt * DT + dt][l] = o[nt][dt];
    }
    __syncthreads();
    if (wave < uint32_t(half)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[nt][dt] += s_o[wave][nt * DT + dt][l];
    }
    __syncthreads();
  }
  if (sp.chunks <= 1) {
    if (wave) return;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const uint32_t r = row0 + 16 * nt + n;
      if (r >= sp.rows) continue;
      const uint64_t t = uint64_t(sp.first + r / group);
      const uint32_t h = head * group + r % group;
      const float total = checked_sum(sum[nt], m[nt]), inv = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
        store_out(a.out, t * a.out.token + uint64_t(h) * a.out.head + 16 * dt + 4 * g, o[nt][dt][0] * inv,
                  o[nt][dt][1] * inv, o[nt][dt][2] * inv, o[nt][dt][3] * inv);
      if (a.lse && g == 0) a.lse[t * a.heads + h] = total == 0.0f ? -INFINITY : m[nt] * kLn2 + __logf(total);
    }
    return;
  }
  if (wave == 0) {
    const uint32_t floats = p.rec_rows * kRecord<D>;
    const PartStore<NT == 1> store(part + record_of(a, p, it, kvh) * floats, floats, p.fused);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      if (16 * nt + n >= p.rec_rows) continue;
      const uint32_t row = (16 * nt + n) * kRecord<D>;
      if (g == 0) store(row + D, f32x4{m[nt], sum[nt], 0.0f, 0.0f});
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) store(row + 16 * dt + 4 * g, o[nt][dt]);
    }
  }
  if constexpr (NT == 1) {
    if (!p.fused) return;
    if (arrived_last(a.count + (tile * a.seqs + seq) * kvh + head, sp.chunks)) join_tile<D>(a, p, sp, it, row0, part);
  }
}

// Heads of 512 (one wide key head for many query heads): 16 NT rows of Q and O
// do not fit a wavefront, and rows in pieces of 16 would read every page again
// for each.  Here no byte of the cache goes to two wavefronts.  Of a step's 64
// tokens a wavefront takes 16 for the first product, all dimensions of them,
// against Q from LDS; the wavefronts' maxima meet there, each weights its own
// scores, and P goes through LDS for the second product, of which a wavefront
// takes 128 dimensions, all tokens.  Two workgroups a compute unit: with 64
// rows, one of them, 64 sequences of 4,000 tokens of 64 heads took 109 us, 97
// here (2.8 TB/s, 346 TFLOP/s).  Instruction issue bounds it, two wavefronts a
// SIMD, about 900 instructions a step beside 1,024 clocks of the matrix unit.
template <int NT>
__global__ __launch_bounds__(256, 2) void k_paged_wide(PagedArgs a, PagedPlan p, float *part) {
  constexpr int D = 512, C = 8, DT = 8;
  const uint32_t kvh = a.cache.heads, group = a.heads / kvh;
  const Item it = item_of(a, p, kvh);
  const uint32_t tile = it.tile, head = it.head, seq = it.seq, chunk = it.chunk;
  const uint32_t row0 = tile * 16 * NT;
  const Span sp = paged_span(a, p, seq, row0);
  if (row0 >= sp.rows || (chunk && chunk >= sp.chunks)) return;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), l = threadIdx.x & 63u, n = l & 15u, g = l >> 4;
  const uint32_t P = a.cache.page, d0 = 128 * wave;
  const uint32_t shift = __builtin_ctz(P);
  const Pages pages{a.page_table + uint64_t(seq) * a.table_width, sp.seen, sp.len - 1, a.cache.pages, shift};
  const int32_t begin = sp.lo + int32_t(chunk * sp.chunk);
  const int32_t end = paged_end(begin, sp.hi, sp.chunk);
  const auto row_of = [&](int nt) {
    const uint32_t r = row0 + 16 * nt + n;
    return r < sp.rows ? r : sp.rows - 1;
  };
  Visible see[NT];

  __shared__ bf16x8 s_q[NT][2 * C][64];  // the first product's operands
  __shared__ bf16x8 s_p[NT][2][64];      // the second's
  __shared__ float s_m[4][NT][16], s_l[4][NT][16];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const uint32_t rr = row_of(nt);
    see[nt] = Visible(sp.pos0 + int32_t(rr / group), a.window);
    const uint16_t *row = a.q + uint64_t(sp.first + rr / group) * a.q_token +
                          uint64_t(head * group + rr % group) * a.q_head;
#pragma unroll
    for (int c = 0; c < C / 4; ++c)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        s_q[nt][2 * (2 * wave + c) + h][l] = *reinterpret_cast<const bf16x8 *>(row + 64 * (2 * wave + c) + 16 * g + 8 * h);
  }
  const int32_t pos_lo = sp.pos0 + int32_t(row0 / group), pos_hi = sp.hi - 1;

  f32x4 o[NT][DT] = {};
  float m[NT], sum[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) m[nt] = -INFINITY, sum[nt] = 0.0f;
  bool bad = false, odd = false;
  const float scale = a.scale * kLog2e;
  const uint64_t page_bytes = uint64_t(P) * D;

  // K: 16 dimensions of token 16 wave + n eight times; V: 16 tokens from 16 g of
  // dimensions d0 + 16 dt + n.  (The K tokens' page is one for the wavefront,
  // but not said so: a scalar id or scale would be waited for where it is
  // loaded, with all loads before it.)
  constexpr int32_t kStep = 64;
  const uint32_t k_tok = threadIdx.x / 64 * 16;
  uint4 kk[C], vv[DT];
  uint8_t ksc = 0, vsc = 0;  // (as loaded: widened where they are used, not while in flight)
  int32_t idk = 0, idv = 0;  // of the next step
  auto load_ids = [&](int32_t b, int32_t &k, int32_t &v) {
    k = pages.id(b + int32_t(k_tok));
    v = pages.id(b + 16 * int32_t(g));
  };
  uint32_t pagev = 0;
  auto load_k = [&](int32_t b) {
    const uint64_t at = uint64_t(pages.checked(idk, bad)) * kvh + head;
    pagev = pages.checked(idv, bad);
    ksc = a.cache.ks[at], vsc = a.cache.vs[uint64_t(pagev) * kvh + head];  // first: they are waited for before K
    const uint8_t *kp = a.cache.k + at * page_bytes + ((uint32_t(b + int32_t(k_tok)) & (P - 1)) + n) * uint32_t(D) + 16 * g;
#pragma unroll
    for (int c = 0; c < C; ++c) kk[c] = *reinterpret_cast<const uint4 *>(kp + 64 * c);
  };
  auto load_v = [&](int32_t b) {
    const uint8_t *vp = a.cache.v + (uint64_t(pagev) * kvh + head) * page_bytes + (d0 + n) * P +
                        (uint32_t(b + 16 * int32_t(g)) & (P - 1));
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) vv[dt] = *reinterpret_cast<const uint4 *>(vp + 16 * dt * P);
  };
  const int32_t last = begin + (end - 1 - begin) / kStep * kStep;
  if (begin < end) {
    int32_t idk1, idv1;
    load_ids(begin, idk, idv);
    load_ids(min(begin + kStep, last), idk1, idv1);
    load_k(begin);
    load_v(begin);
    asm volatile("" : "+v"(idk1), "+v"(idv1));  // waited for here and not, with K and V, in every step
    idk = idk1, idv = idv1;
  }
  __syncthreads();

  for (int32_t b = begin; b < end; b += kStep) {
    const int32_t tv = b + 16 * int32_t(g), tk = b + int32_t(k_tok) + 4 * int32_t(g);
    // past the last step that step's again: a load behind a branch makes every
    // later wait one for all loads
    const int32_t next = min(b + kStep, last);
    int32_t idk2, idv2;  // ahead of the K and V loads below
    load_ids(min(b + 2 * kStep, last), idk2, idv2);
    const float ks = scale * power_of_two(int(ksc) - 127);
    const float vs = power_of_two(int(vsc) - 127);
    const bool partial = b + kStep - 1 > pos_lo || (a.window && int64_t(b) <= int64_t(pos_hi) - a.window);
    f32x4 s[NT][2] = {};
    // Q a piece ahead of its use (left to itself the compiler reads it right before:
    // 4 x 4 of up to 9,000 tokens 34.5 us so, 35.1)
    bf16x8 qa[2][NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) qa[0][nt][0] = s_q[nt][0][l], qa[0][nt][1] = s_q[nt][1][l];
#pragma unroll
    for (int c = 0; c < C; ++c) {
      if (c + 1 < C) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) qa[(c + 1) & 1][nt][0] = s_q[nt][2 * c + 2][l], qa[(c + 1) & 1][nt][1] = s_q[nt][2 * c + 3][l];
      }
      const bf16x8 k0 = e4m3_bf16(kk[c].x, kk[c].y), k1 = e4m3_bf16(kk[c].z, kk[c].w);
      __builtin_amdgcn_sched_barrier(0x1 | 0x2 | 0x4 | 0x8);  // LDS reads stay ahead
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        s[nt][0] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k0, qa[c & 1][nt][0], s[nt][0], 0, 0, 0);
        s[nt][1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k1, qa[c & 1][nt][1], s[nt][1], 0, 0, 0);
      }
    }
    load_k(next);
    float x[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int i = 0; i < 4; ++i) x[nt][i] = (s[nt][0][i] + s[nt][1][i]) * ks;
      if (partial) {
        keep_branch();
#pragma unroll
        for (int i = 0; i < 4; ++i) x[nt][i] = see[nt](tk + i) ? x[nt][i] : -INFINITY;
      }
      const float top = max_lane16(fmaxf(fmaxf(x[nt][0], x[nt][1]), fmaxf(x[nt][2], x[nt][3])));
      if (g == 0) s_m[wave][nt][n] = top;
    }
    __syncthreads();
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const float top = fmaxf(fmaxf(fmaxf(s_m[0][nt][n], s_m[1][nt][n]), fmaxf(s_m[2][nt][n], s_m[3][nt][n])), m[nt]);
      if (__any(top > m[nt] + kRise)) {  // the same in every wavefront
        const float fade = __builtin_amdgcn_exp2f(m[nt] - (top == -INFINITY ? 0.0f : top));
        m[nt] = top;
        sum[nt] *= fade;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[nt][dt] *= fade;
      }
      const float at = m[nt] == -INFINITY ? 0.0f : m[nt];
      float e[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        e[i] = __builtin_amdgcn_exp2f(x[nt][i] - at);
        sum[nt] += e[i];
      }
      // half a step of each weight: the matrix operand's type
      reinterpret_cast<uint2 *>(&s_p[nt][g / 2][16 * wave + n])[g & 1] =
          make_uint2(bf16_pair(e[0], e[1]), bf16_pair(e[2], e[3]));
    }
    __syncthreads();
    if (partial) {  // as in k_paged_attention
      uint32_t found = 0;
      const uint32_t from = odd_code(__float_as_uint(vs) >> 23);  // (vsc is the next step's)
      uint32_t keep[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int32_t left = sp.len - (tv + 4 * k);
        keep[k] = left >= 4 ? ~0u : left <= 0 ? 0u : (1u << (8 * left)) - 1u;
      }
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        vv[dt].x &= keep[0], vv[dt].y &= keep[1], vv[dt].z &= keep[2], vv[dt].w &= keep[3];
        found |= odd_codes(vv[dt].x, from) | odd_codes(vv[dt].y, from) | odd_codes(vv[dt].z, from) | odd_codes(vv[dt].w, from);
      }
      if (__any(found != 0)) {
        odd = true;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          vv[dt].x = no_odd(vv[dt].x, from), vv[dt].y = no_odd(vv[dt].y, from);
          vv[dt].z = no_odd(vv[dt].z, from), vv[dt].w = no_odd(vv[dt].w, from);
        }
      }
    }
    bf16x8 pb[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) pb[nt][0] = s_p[nt][0][l], pb[nt][1] = s_p[nt][1][l];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      const bf16x8 v0 = e4m3_bf16(vv[dt].x, vv[dt].y, vs), v1 = e4m3_bf16(vv[dt].z, vv[dt].w, vs);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        o[nt][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v0, pb[nt][0], o[nt][dt], 0, 0, 0);
        o[nt][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v1, pb[nt][1], o[nt][dt], 0, 0, 0);
      }
    }
    load_v(next);
    idk = idk2, idv = idv2;
  }

  if (odd) {  // uniform, and rare: one token after the other
    for (int32_t b0 = begin; b0 < end; b0 += kStep) {
      if (b0 + kStep - 1 <= pos_lo && !(a.window && int64_t(b0) <= int64_t(pos_hi) - a.window)) continue;
      for (int32_t j = b0; j < min(b0 + kStep, sp.len); ++j) {
        const uint64_t at = uint64_t(pages.checked(pages.id(j), bad)) * kvh + head;
        const uint32_t from = odd_code(a.cache.vs[at]);
        const uint8_t *vp = a.cache.v + at * page_bytes + d0 * P + (uint32_t(j) & (P - 1));
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          f32x4 odds;
#pragma unroll
          for (int i = 0; i < 4; ++i) odds[i] = odd_value(vp[(16 * dt + 4 * g + i) * P], from);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const bool in = see[nt](j);
            f32x4 back;
#pragma unroll
            for (int i = 0; i < 4; ++i) back[i] = in ? odds[i] : 0.0f;
            o[nt][dt] += back;
          }
        }
      }
    }
  }
  const bool bad_page = __any(bad);  // every wavefront has read the same V ids
  if (const uint32_t status = sp.wrong | (bad_page ? kStatusBadCachePage : 0u); status && l == 0) atomicOr(a.status, status);
  if (bad_page) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) sum[nt] = __uint_as_float(0x7fc00000u);
  }
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    sum[nt] = sum_lane16(sum[nt]);
    if (g == 0) s_l[wave][nt][n] = sum[nt];
  }
  __syncthreads();
  const uint32_t floats = p.rec_rows * kRecord<D>;
  const PartStore<NT == 1> store(part + record_of(a, p, it, kvh) * floats, floats, p.fused);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const uint32_t r = row0 + 16 * nt + n;
    if (r >= sp.rows) continue;
    const float top = m[nt], total = s_l[0][nt][n] + s_l[1][nt][n] + s_l[2][nt][n] + s_l[3][nt][n];
    if (sp.chunks > 1) {
      const uint32_t row = (16 * nt + n) * kRecord<D>;
      if (wave == 0 && g == 0) store(row + D, f32x4{top, total, 0.0f, 0.0f});
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) store(row + d0 + 16 * dt + 4 * g, o[nt][dt]);
      continue;
    }
    const uint64_t t = uint64_t(sp.first + r / group);
    const uint32_t h = head * group + r % group;
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
      store_out(a.out, t * a.out.token + uint64_t(h) * a.out.head + d0 + 16 * dt + 4 * g, o[nt][dt][0] * inv,
                o[nt][dt][1] * inv, o[nt][dt][2] * inv, o[nt][dt][3] * inv);
    if (a.lse && wave == 0 && g == 0) a.lse[t * a.heads + h] = total == 0.0f ? -INFINITY : top * kLn2 + __logf(total);
  }
  if constexpr (NT == 1) {
    if (sp.chunks <= 1 || !p.fused) return;
    if (arrived_last(a.count + (tile * a.seqs + seq) * kvh + head, sp.chunks)) join_tile<D>(a, p, sp, it, row0, part);
  }
}

// Where a row's 16-byte piece of K or V lies in LDS: piece ^ turn(row), so that
// the 16 lanes of a read, one piece of each of 16 rows, meet no bank twice (64
// banks of 4 bytes).  K: a row is a token of D values, and a lane's token is
// 8 (n / 4) + n % 4 of its 32.  V: a row is a dimension of TK values.
template <int D>
__device__ __forceinline__ uint32_t turn_k(uint32_t tok) {
  return D == 64 ? ((tok >> 1) & 1u) | ((tok >> 2) & 6u) : (tok & 3u) | ((tok >> 1) & 12u);
}
template <int TK>
__device__ __forceinline__ uint32_t turn_v(uint32_t dim) {
  return TK == 64 ? (dim >> 1) & 7u : (dim >> 2) & 3u;
}

// More rows: each wavefront has 16 NT of its own (of two row tiles, two
// wavefronts share one, half the tokens each), and all read the same TK tokens
// from LDS, where the workgroup has put them as bf16 with their page's scale,
// once for all its rows.  In registers 64 rows of 128 leave one wavefront a
// SIMD, with spills, and their four partial sums to join: 8 sequences of 64 new
// tokens of 3,000 104 us so, 59 here (420 TFLOP/s); 32 of 8 of 4,000 73 and 66
// (4.1 TB/s); 74 of 17 of 67 75 and 21.  Short ones are bound by the chain of
// loads before their first product, long ones by LDS reads (2 bytes a multiply,
// half the matrix rate at NT = 1) and the softmax beside them.
template <int D, int NT, int RW>
__global__ __launch_bounds__(256, D * NT > 128 ? 2 : D * NT < 128 ? 5 : RW == 2 ? 4 : 3) void k_paged_rows(PagedArgs a, PagedPlan p, float *part) {
  constexpr int TK = D <= 128 ? 64 : 32;  // tokens a step
  constexpr int TW = 4 / RW;              // wavefronts that share a row tile's tokens
  constexpr int U = TK / 32 / TW, T = 2 * U, DT = D / 16, C = D / 32;
  constexpr int R = D * TK / 4096;                // 16-code pieces of K, and of V, a thread
  constexpr int kTokens = 4096 / D;               // of K in 256 pieces
  constexpr int I = kTokens >= 16 ? R : TK / 16;  // pages of a thread's K pieces
  const uint32_t kvh = a.cache.heads, group = a.heads / kvh;
  const Item it = item_of(a, p, kvh);
  const uint32_t tile = it.tile, head = it.head, seq = it.seq, chunk = it.chunk;
  const uint32_t row0 = tile * 16 * NT * RW;
  const Span sp = paged_span(a, p, seq, row0);
  if (row0 >= sp.rows || (chunk && chunk >= sp.chunks)) return;
  const uint32_t tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / 64), l = tid & 63u, n = l & 15u, g = l >> 4;
  const uint32_t P = a.cache.page;
  const Pages pages{a.page_table + uint64_t(seq) * a.table_width, sp.seen, sp.len - 1, a.cache.pages, uint32_t(__builtin_ctz(P))};
  const int32_t begin = sp.lo + int32_t(chunk * sp.chunk);
  const int32_t end = paged_end(begin, sp.hi, sp.chunk);
  const uint32_t mine = row0 + 16 * NT * (wave % RW), u0 = U * (wave / RW);  // the wavefront's rows and 32-token parts
  const bool active = mine < sp.rows;

  Visible see[NT];
  bf16x8 q[NT][C];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const uint32_t r = mine + 16 * nt + n;
    const uint32_t rr = r < sp.rows ? r : sp.rows - 1;
    see[nt] = Visible(sp.pos0 + int32_t(rr / group), a.window);
    const uint16_t *row = a.q + uint64_t(sp.first + rr / group) * a.q_token +
                          uint64_t(head * group + rr % group) * a.q_head;
#pragma unroll
    for (int c = 0; c < C; ++c) q[nt][c] = *reinterpret_cast<const bf16x8 *>(row + 32 * c + 8 * g);
  }
  const int32_t pos_lo = sp.pos0 + int32_t(row0 / group), pos_hi = sp.hi - 1;
  const auto partial_at = [&](int32_t b) {
    return b + TK - 1 > pos_lo || (a.window && int64_t(b) <= int64_t(pos_hi) - a.window);
  };

  constexpr uint32_t kPieces = TK * D / 8;
  __shared__ u32x4 s_rows[2 * kPieces];  // K, V
  __shared__ uint32_t s_flags;
  if (tid == 0) s_flags = 0;

  f32x4 o[NT][DT] = {};
  float m[NT], sum[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) m[nt] = -INFINITY, sum[nt] = 0.0f;
  bool bad = false, odd = false;
  const float scale = a.scale * kLog2e;
  const uint64_t page_bytes = uint64_t(P) * D;

  // A step's pieces: K piece i of a thread is 16 dimensions of token 4096 / D *
  // i + tid / (D / 16), V piece i 16 tokens of dimension 4096 / TK * i + tid /
  // (TK / 16).  Loaded two steps ahead of their use, turned into bf16 one
  // ahead (a step more in flight measured no better); their pages' ids are
  // loaded another step ahead.
  const uint32_t k_tok = tid / (D / 16), k_dim = tid % (D / 16) * 16;
  const uint32_t v_dim = tid / (TK / 16), v_tok = tid % (TK / 16) * 16;
  uint4 kk[R], vv[R];
  uint32_t ksc[I], vsc;
  int32_t idk[I], idv = 0;
  auto load_ids = [&](int32_t b) {
#pragma unroll
    for (int i = 0; i < I; ++i) idk[i] = pages.id(b + int32_t(k_tok) + (kTokens >= 16 ? kTokens : 16) * i);
    idv = pages.id(b + int32_t(v_tok));
  };
  auto load = [&](int32_t b) {
#pragma unroll
    for (int i = 0; i < I; ++i) {
      const uint64_t at = uint64_t(pages.checked(idk[i], bad)) * kvh + head;
      ksc[i] = a.cache.ks[at];
#pragma unroll
      for (int j = 0; j < R / I; ++j) {
        const uint32_t slot = uint32_t(b + int32_t(k_tok) + kTokens * (R / I * i + j)) & (P - 1);
        kk[R / I * i + j] = *reinterpret_cast<const uint4 *>(a.cache.k + at * page_bytes + slot * uint32_t(D) + k_dim);
      }
    }
    const uint64_t at = uint64_t(pages.checked(idv, bad)) * kvh + head;
    vsc = a.cache.vs[at];
    const uint8_t *vp = a.cache.v + at * page_bytes + v_dim * P + (uint32_t(b + int32_t(v_tok)) & (P - 1));
#pragma unroll
    for (int i = 0; i < R; ++i) vv[i] = *reinterpret_cast<const uint4 *>(vp + 4096 / TK * i * P);
  };
  auto put = [&](u32x4 *to, uint32_t row, uint32_t pieces, uint32_t piece, uint32_t turn, uint4 x, float f) {
    to[row * pieces + (piece ^ turn)] = __builtin_bit_cast(u32x4, e4m3_bf16(x.x, x.y, f));
    to[row * pieces + ((piece + 1) ^ turn)] = __builtin_bit_cast(u32x4, e4m3_bf16(x.z, x.w, f));
  };
  auto stage = [&](int32_t b, u32x4 *to) {
    if (partial_at(b)) {
      // as in k_paged_attention: nothing from behind the sequence, and no NaN or
      // infinity that some row must not see
      uint32_t found = 0;
      const uint32_t from = odd_code(vsc);
      uint32_t keep[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int32_t left = sp.len - (b + int32_t(v_tok) + 4 * k);
        keep[k] = left >= 4 ? ~0u : left <= 0 ? 0u : (1u << (8 * left)) - 1u;
      }
#pragma unroll
      for (int i = 0; i < R; ++i) {
        vv[i].x &= keep[0], vv[i].y &= keep[1], vv[i].z &= keep[2], vv[i].w &= keep[3];
        found |= odd_codes(vv[i].x, from) | odd_codes(vv[i].y, from) | odd_codes(vv[i].z, from) | odd_codes(vv[i].w, from);
      }
      if (__any(found != 0)) {
        odd = true;
#pragma unroll
        for (int i = 0; i < R; ++i)
          vv[i].x = no_odd(vv[i].x, from), vv[i].y = no_odd(vv[i].y, from), vv[i].z = no_odd(vv[i].z, from),
          vv[i].w = no_odd(vv[i].w, from);
      }
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const uint32_t tok = k_tok + kTokens * i;
      put(to, tok, D / 8, k_dim / 8, turn_k<D>(tok), kk[i], power_of_two(int(ksc[i / (R / I)]) - 127));
    }
    const float vs = power_of_two(int(vsc) - 127);
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const uint32_t dim = v_dim + 4096 / TK * i;
      put(to + kPieces, dim, TK / 8, v_tok / 8, turn_v<TK>(dim), vv[i], vs);
    }
  };
  const uint32_t k_row = 8 * (n / 4) + n % 4, k_turn = turn_k<D>(k_row), v_turn = turn_v<TK>(n);

  if (begin < end) load_ids(begin);
  // Q is waited for here, with the ids, or it would be in every step
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int c = 0; c < C; ++c) asm volatile("" : "+v"(q[nt][c]));
  if (begin < end) {
    load(begin);
    if (begin + TK < end) load_ids(begin + TK);
    stage(begin, s_rows);
    if (begin + TK < end) load(begin + TK);
    if (begin + 2 * TK < end) load_ids(begin + 2 * TK);
  }
  __syncthreads();

  for (int32_t b = begin; b < end; b += TK) {
    const u32x4 *sk = s_rows, *sv = sk + kPieces;
    bf16x8 pb[NT][U];
    if (active) {
      f32x4 s[NT][T] = {};
#pragma unroll
      for (int t = 0; t < T; ++t)
#pragma unroll
        for (int c = 0; c < C; ++c) {
          const uint32_t row = 32 * (u0 + t / 2) + 4 * (t & 1) + k_row;
          const bf16x8 k = __builtin_bit_cast(bf16x8, sk[row * (D / 8) + ((4 * c + g) ^ k_turn)]);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) s[nt][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k, q[nt][c], s[nt][t], 0, 0, 0);
        }
      const bool partial = partial_at(b);
      const int32_t tv = b + 32 * int32_t(u0) + 8 * int32_t(g);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float x[4 * T];
#pragma unroll
        for (int i = 0; i < 4 * T; ++i) x[i] = s[nt][i / 4][i % 4];
        if (partial) {
          keep_branch();
#pragma unroll
          for (int i = 0; i < 4 * T; ++i) x[i] = see[nt](tv + 32 * (i / 8) + i % 8) ? x[i] : -INFINITY;
        }
        float top = x[0];
#pragma unroll
        for (int i = 1; i < 4 * T; ++i) top = fmaxf(top, x[i]);
        top = fmaxf(m[nt], max_lane16(top) * scale);
        if (__any(top > m[nt] + kRise)) {
          const float fade = __builtin_amdgcn_exp2f(m[nt] - (top == -INFINITY ? 0.0f : top));
          m[nt] = top;
          sum[nt] *= fade;
#pragma unroll
          for (int dt = 0; dt < DT; ++dt) o[nt][dt] *= fade;
        }
        const float at = m[nt] == -INFINITY ? 0.0f : m[nt];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          u32x4 w;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float e0 = __builtin_amdgcn_exp2f(__builtin_fmaf(x[8 * u + 2 * j], scale, -at));
            const float e1 = __builtin_amdgcn_exp2f(__builtin_fmaf(x[8 * u + 2 * j + 1], scale, -at));
            sum[nt] += e0;
            sum[nt] += e1;
            w[j] = bf16_pair(e0, e1);  // half a step of each weight: the matrix operand's type
          }
          pb[nt][u] = __builtin_bit_cast(bf16x8, w);
        }
      }
    }
    if (active) {
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const bf16x8 v = __builtin_bit_cast(bf16x8, sv[(16 * dt + n) * (TK / 8) + ((4 * (u0 + u) + g) ^ v_turn)]);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) o[nt][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, pb[nt][u], o[nt][dt], 0, 0, 0);
        }
    }
    __syncthreads();
    if (b + TK < end) {
      stage(b + TK, s_rows);
      if (b + 2 * TK < end) load(b + 2 * TK);
      if (b + 3 * TK < end) load_ids(b + 3 * TK);
      __syncthreads();
    }
  }

  // the lane's place again from the thread's number: kept over the loop it was
  // spilled (32 of 8 new and 300 tokens 9.8 us, 9.6 so)
  uint32_t lane = tid & 63u;
  asm volatile("" : "+v"(lane));
  const uint32_t group4 = lane >> 4;
  if (bad || odd) atomicOr(&s_flags, (bad ? 1u : 0u) | (odd ? 2u : 0u));
  __syncthreads();
  const uint32_t flags = s_flags;
  if constexpr (TW == 2) {  // the token parts' sums: part 1 into 0, both taken from the larger maximum
    float *x = reinterpret_cast<float *>(s_rows) + (wave % RW) * (64 * NT * (4 * DT + 2));
    if (u0) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float *y = x + nt * 64 * (4 * DT + 2);
        y[lane] = m[nt], y[64 + lane] = sum[nt];
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) reinterpret_cast<f32x4 *>(y + 128)[64 * dt + lane] = o[nt][dt];
      }
    }
    __syncthreads();
    if (!u0) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float *y = x + nt * 64 * (4 * DT + 2);
        const float other = y[lane], top = fmaxf(m[nt], other), at = top == -INFINITY ? 0.0f : top;
        const float f0 = __builtin_amdgcn_exp2f(m[nt] - at), f1 = __builtin_amdgcn_exp2f(other - at);
        m[nt] = top, sum[nt] = sum[nt] * f0 + y[64 + lane] * f1;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[nt][dt] = o[nt][dt] * f0 + reinterpret_cast<const f32x4 *>(y + 128)[64 * dt + lane] * f1;
      }
    }
  }
  if ((flags & 2u) && !u0) {  // rare: one token after the other
    for (int32_t b0 = begin; b0 < end; b0 += TK) {
      if (!partial_at(b0)) continue;
      for (int32_t j = b0; j < min(b0 + TK, sp.len); ++j) {
        const uint64_t at = uint64_t(pages.checked(pages.id(j), bad)) * kvh + head;
        const uint32_t from = odd_code(a.cache.vs[at]);
        const uint8_t *vp = a.cache.v + at * page_bytes + (uint32_t(j) & (P - 1));
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          f32x4 odds;
#pragma unroll
          for (int i = 0; i < 4; ++i) odds[i] = odd_value(vp[(16 * dt + 4 * group4 + i) * P], from);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const bool in = see[nt](j);
            f32x4 back;
#pragma unroll
            for (int i = 0; i < 4; ++i) back[i] = in ? odds[i] : 0.0f;
            o[nt][dt] += back;
          }
        }
      }
    }
  }
  if (const uint32_t status = sp.wrong | (flags & 1u ? kStatusBadCachePage : 0u); status && tid == 0) atomicOr(a.status, status);
  const uint32_t floats = p.rec_rows * kRecord<D>;
  const PartStore<false> store(part + record_of(a, p, it, kvh) * floats, floats, 0);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const float total = flags & 1u ? __uint_as_float(0x7fc00000u) : sum_lane16(sum[nt]);
    const uint32_t r = mine + 16 * nt + lane % 16;
    if (r >= sp.rows || u0) continue;
    if (sp.chunks > 1) {
      const uint32_t row = (r - row0) * kRecord<D>;
      if (group4 == 0) store(row + D, f32x4{m[nt], total, 0.0f, 0.0f});
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) store(row + 16 * dt + 4 * group4, o[nt][dt]);
      continue;
    }
    const uint64_t t = uint64_t(sp.first + r / group);
    const uint32_t h = head * group + r % group;
    const float row_sum = checked_sum(total, m[nt]), inv = row_sum == 0.0f ? 0.0f : 1.0f / row_sum;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
      store_out(a.out, t * a.out.token + uint64_t(h) * a.out.head + 16 * dt + 4 * group4, o[nt][dt][0] * inv,
                o[nt][dt][1] * inv, o[nt][dt][2] * inv, o[nt][dt][3] * inv);
    if (a.lse && group4 == 0) a.lse[t * a.heads + h] = row_sum == 0.0f ? -INFINITY : m[nt] * kLn2 + __logf(row_sum);
  }
}

// Joins the chunks of one row a workgroup, in an order that its size alone
// sets: the chunks' maxima in the lanes, then their rows in groups of
// threads at once.
template <int D>
__global__ __launch_bounds__(256) void k_paged_join(PagedArgs a, PagedPlan p, const float *part) {
  constexpr uint32_t kLanes = D / 4 < 64 ? D / 4 : 64, kSpan = D / (4 * kLanes);  // float4s of a row a thread
  constexpr uint32_t kGroups = 256 / kLanes;
  const uint32_t kvh = a.cache.heads, group = a.heads / kvh, tid = threadIdx.x;
  const uint32_t seq = blockIdx.y, head = blockIdx.z, r = blockIdx.x;
  const uint32_t per = 16 * p.row_tiles, tile = r / per;
  const Span sp = paged_span(a, p, seq, tile * per);
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
template <int D>
__global__ __launch_bounds__(256) void k_paged_join_rows(PagedArgs a, PagedPlan p, const float *part) {
  const uint32_t r = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + threadIdx.x / 64), per = 16 * p.row_tiles;
  const Item it{r / per, 0, blockIdx.y, blockIdx.z};
  const Span sp = paged_span(a, p, it.seq, it.tile * per);
  if (r >= sp.rows || sp.chunks <= 1) return;
  join_row<D, 0>(a, p, sp, it, it.tile * per, r % per, part);
}

template <int D, class Kernel>
hipError_t launch(hipStream_t s, const PagedArgs &a, const PagedPlan &p, float *part, Kernel kernel) {
  kernel<<<uint32_t(p.blocks), 256, 0, s>>>(a, p, part);
  if (p.chunks > 1 && !p.fused) {
    const uint32_t rows = uint32_t(a.max_new) * (a.heads / a.cache.heads);
    if (p.chunks <= 16)
      k_paged_join_rows<D><<<dim3((rows + 3) / 4, a.seqs, a.cache.heads), 256, 0, s>>>(a, p, part);
    else
      k_paged_join<D><<<dim3(rows, a.seqs, a.cache.heads), 256, 0, s>>>(a, p, part);
  }
  return hipGetLastError();
}

template <int D>
hipError_t launch_dim(hipStream_t s, const PagedArgs &a, const PagedPlan &p, float *part) {
  if constexpr (D == 512) {
    if (p.row_tiles == 2) return launch<D>(s, a, p, part, k_paged_wide<2>);
    return launch<D>(s, a, p, part, k_paged_wide<1>);
  } else {
    if constexpr (D <= 128) {
      if (p.row_tiles == 8) return launch<D>(s, a, p, part, k_paged_rows<D, 2, 4>);
      if (p.row_tiles == 2 && p.staged) return launch<D>(s, a, p, part, k_paged_rows<D, 1, 2>);
      if (p.row_tiles == 2) return launch<D>(s, a, p, part, k_paged_attention<D, 2>);
    }
    if (p.row_tiles == 4) return launch<D>(s, a, p, part, k_paged_rows<D, 1, 4>);
    return launch<D>(s, a, p, part, k_paged_attention<D, 1>);
  }
}

}  // namespace

hipError_t launch_paged_attention(hipStream_t s, const PagedArgs &a, const PagedPlan &p, float *part) {
  switch (a.cache.dim) {
    case 64: return launch_dim<64>(s, a, p, part);
    case 128: return launch_dim<128>(s, a, p, part);
    case 256: return launch_dim<256>(s, a, p, part);
    case 512: return launch_dim<512>(s, a, p, part);
  }
  return hipErrorInvalidValue;
}

}  // namespace s14
