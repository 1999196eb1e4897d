// Append of keys and values to the paged 4-bit cache (E2M1 codes, E8M0 scales of
// 32 dimensions of a key and of 128 of a value, 64 at heads of 64).
//
// A block's scale is 2^e, e the least with 6 2^e >= the largest magnitude (6 is
// E2M1's largest), held in -100 .. 100; codes are rounded to nearest, ties to even,
// and end at 6.  A token's scales are its own: nothing that was stored before is
// touched, so the unit of work is a block of kSlots neighbouring slots of a page
// (16, the slots of a unit of V codes, or 4 where few tokens are new), head and
// side, of D / 8 lanes a slot.  21 prompts of up to 4,000 tokens, 8 heads of 128: 78 MB
// in 22.4 us, 3.5 TB/s, a third over what the bytes take: a workgroup of some 32 B a
// thread starts with a chain of its own, the search for its sequence (64 counts and six
// LDS permutes), the page's id, then the rows, and the card takes several rounds of
// them.  With the keys' norm and rotation 30.4 (f32 rows 39.1).  For a few tokens that
// chain is all (96 single ones: 4.3 us).
#include "s14_attn_rows.hpp"

namespace s14 {
namespace {

template <int kCtrl>
__device__ __forceinline__ uint32_t dpp_u(uint32_t v) {
  return uint32_t(dpp_i<kCtrl>(0, int(v)));
}

// Unsigned maximum over kLanes neighbouring lanes, in each of them.
template <int kLanes>
__device__ __forceinline__ uint32_t lane_max(uint32_t v) {
  static_assert(kLanes == 4 || kLanes == 8 || kLanes == 16, "");
  v = max(v, dpp_u<0xb1>(v));  // quad_perm [1,0,3,2]
  v = max(v, dpp_u<0x4e>(v));  // quad_perm [2,3,0,1]
  if constexpr (kLanes >= 8) v = max(v, dpp_u<0x141>(v));   // row_half_mirror
  if constexpr (kLanes >= 16) v = max(v, dpp_u<0x140>(v));  // row_mirror
  return v;
}

// A block's E8M0 code by the bits of its largest magnitude: 6 = 1.5 * 2^2, so the
// exponent less 2, and one more where the mantissa passes 1.5.  The scales end at
// 2^-100 and 2^100: products of a score and weights stay normal numbers.  A NaN
// (bits above infinity's) makes the block NaN: 255.
__device__ __forceinline__ uint32_t block_code(uint32_t amax) {
  const int e = int(amax >> 23) - 2 + ((amax & 0x7fffffu) > 0x400000u ? 1 : 0);
  return amax > 0x7f800000u ? 255u : uint32_t(min(max(e, 27), 227));
}


// A lane's eight values of a row, and what turns them.
struct Row {
  Quad p, q;
  Weight w;
  Angles n;
  Unit x;
};

// The bits of its largest magnitude: magnitudes order as their bits.
__device__ __forceinline__ uint32_t row_amax(const Row &r) {
  uint32_t amax = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    amax = max(amax, max(__float_as_uint(r.p.v[i]) & 0x7fffffffu, __float_as_uint(r.q.v[i]) & 0x7fffffffu));
  return amax;
}

// Its eight codes.
__device__ __forceinline__ uint32_t block_word(const Row &r, uint32_t code) {
  if (code == 255u) return 0u;
  const float inv = __uint_as_float((254u - code) << 23);
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, r.p.v[0] * inv, r.p.v[1] * inv, 1.0f, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, r.p.v[2] * inv, r.p.v[3] * inv, 1.0f, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, r.q.v[0] * inv, r.q.v[1] * inv, 1.0f, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, r.q.v[2] * inv, r.q.v[3] * inv, 1.0f, 3);
}

// Where a block of kSlots tokens lies, and which of its slots are new: kept ..
// full - 1.  (t.page counts blocks.)
struct Block {
  int64_t start, id;
  uint32_t kept, full, head, slot0;  // slot0: of the page
  uint64_t place;
};
template <int kSlots>
__device__ __forceinline__ Block block_of(const AppendArgs &a, const Touched &t, uint32_t head) {
  const uint32_t P = a.cache.page;
  Block b;
  b.start = t.page * kSlots;
  const int64_t end = t.past + (t.last - t.first), page = b.start / P;
  b.id = page < int64_t(a.table_width) ? a.page_table[uint64_t(t.seq) * a.table_width + page] : -1;
  b.kept = t.past > b.start ? uint32_t(t.past - b.start) : 0u;
  b.full = end - b.start < int64_t(kSlots) ? uint32_t(end - b.start) : kSlots;
  b.head = head, b.slot0 = uint32_t(b.start) & (P - 1);
  b.place = uint64_t(b.id) * a.cache.heads + head;
  return b;
}

template <int kDim, bool kTurn, bool kIn16>
__device__ __forceinline__ Row load_row(const AppendArgs &a, const Touched &t, const Block &b, uint32_t side) {
  const uint32_t lane = threadIdx.x % (kDim / 8), row = threadIdx.x / (kDim / 8);
  const uint32_t r = row < b.kept ? b.kept : row < b.full ? row : b.full - 1;  // whole wavefronts sum
  const AttnRows in = a.in[side];
  RopeArgs rope = a.rope;
  if (!kTurn || side) rope.table = nullptr;
  Row v{};
  v.x = unit_of(lane, rope);
  const uint64_t at = uint64_t(t.first + (b.start + r - t.past)) * in.token + uint64_t(b.head) * in.head;
  v.p = load_quad<kIn16>(in.p, at + v.x.a), v.q = load_quad<kIn16>(in.p, at + v.x.b);
  if (kTurn && !side && a.k_weight) v.w = load_weight(a.k_weight, v.x);
  if (rope.table) v.n = load_angles(rope, v.x, int32_t(min(b.start + r, int64_t(INT_MAX))));
  return v;
}

template <int kDim, int kSlots, bool kTurn>
__device__ __forceinline__ void store_keys(const AppendArgs &a, const Block &b, Row &r) {
  constexpr uint32_t kLanes = kDim / 8;
  const uint32_t P = a.cache.page, lane = threadIdx.x % kLanes, row = threadIdx.x / kLanes, slot = b.slot0 + row;
  const bool live = row >= b.kept && row < b.full;
  if constexpr (kTurn) {
    if (a.k_weight) row_norm<kLanes>(r.p, r.q, r.w, a.eps);
    if (a.rope.table) {
      row_rotate(r.p, r.q, a.rope, r.x, r.n);
      if (!r.n.good && live && lane == 0) atomicOr(a.status, kStatusBadPosition);
    }
    // eight neighbouring dimensions a lane, where the rotation had them otherwise
    if (a.rope.table && !a.rope.interleaved) {
      __shared__ float s_row[kSlots][kDim];
      if (row < kSlots) {
        *reinterpret_cast<float4 *>(&s_row[row][r.x.a]) = make_float4(r.p.v[0], r.p.v[1], r.p.v[2], r.p.v[3]);
        *reinterpret_cast<float4 *>(&s_row[row][r.x.b]) = make_float4(r.q.v[0], r.q.v[1], r.q.v[2], r.q.v[3]);
      }
      __syncthreads();
      if (row < kSlots) {
        const float4 y = *reinterpret_cast<const float4 *>(&s_row[row][8 * lane]);
        const float4 z = *reinterpret_cast<const float4 *>(&s_row[row][8 * lane + 4]);
        r.p.v[0] = y.x, r.p.v[1] = y.y, r.p.v[2] = y.z, r.p.v[3] = y.w;
        r.q.v[0] = z.x, r.q.v[1] = z.y, r.q.v[2] = z.z, r.q.v[3] = z.w;
      }
    }
  }
  const uint32_t code = block_code(lane_max<4>(row_amax(r)));
  if (!live) return;
  *reinterpret_cast<uint32_t *>(a.cache.k + (b.place * P + slot) * (kDim / 2) + 4 * lane) = block_word(r, code);
  if (lane % 4 == 0)
    a.cache.ks[b.place * (kDim / 32 * P) + lane / 4 * P + (slot & ~15u) + 4 * (slot & 3u) + ((slot >> 2) & 3u)] = uint8_t(code);
}

template <int kDim, int kSlots>
__device__ __forceinline__ void store_values(const AppendArgs &a, const Block &b, const Row &r) {
  constexpr uint32_t kLanes = kDim / 8, kParts = kDim < 128 ? 1 : kDim / 128;
  const uint32_t P = a.cache.page, lane = threadIdx.x % kLanes, row = threadIdx.x / kLanes;
  const bool live = row >= b.kept && row < b.full;
  const uint32_t code = block_code(lane_max<kDim < 128 ? 8 : 16>(row_amax(r)));
  if (live && lane % (kDim < 128 ? 8 : 16) == 0) a.cache.vs[(b.place * kParts + lane / 16) * P + b.slot0 + row] = uint8_t(code);
  // two slots a byte: the slots of a dimension come together through LDS
  __shared__ uint32_t s_code[kSlots][kLanes];
  if (row < kSlots) s_code[row][lane] = block_word(r, code);
  __syncthreads();
  // nibbles kept .. full - 1 are new, the others stay
  constexpr uint32_t kWords = kSlots / 8 ? kSlots / 8 : 1;
  uint32_t mask[kWords];
#pragma unroll
  for (uint32_t k = 0; k < kWords; ++k) {
    const uint32_t from = b.kept > 8 * k ? min(b.kept - 8 * k, 8u) : 0u, to = b.full > 8 * k ? min(b.full - 8 * k, 8u) : 0u;
    mask[k] = uint32_t((1ull << (4 * to)) - 1u) & ~uint32_t((1ull << (4 * from)) - 1u);
  }
  const auto gather = [&](uint32_t dim, uint32_t k) {  // eight slots (or four) of a dimension
    uint32_t c = 0;
#pragma unroll
    for (uint32_t j = 0; j < (kSlots < 8 ? kSlots : 8); ++j) c |= ((s_code[8 * k + j][dim / 8] >> (4 * (dim % 8))) & 15u) << (4 * j);
    return c;
  };
  uint8_t *to = a.cache.v + b.place * P * (kDim / 2);
  if constexpr (kSlots == 16) {
    // a unit of 16 bytes: dimensions d and d + 16, 16 slots
    for (uint32_t u = threadIdx.x; u < kDim / 2; u += blockDim.x) {
      const uint32_t d = u / 16 * 32 + u % 16;
      uint4 *unit = reinterpret_cast<uint4 *>(to + (u / 16 * P + b.slot0 + u % 16) * 16);
      uint4 y = make_uint4(gather(d, 0), gather(d, 1), gather(d + 16, 0), gather(d + 16, 1));
      if ((mask[0] & mask[1]) != ~0u) {  // uniform
        const uint4 old = *unit;
        y.x = (old.x & ~mask[0]) | (y.x & mask[0]), y.y = (old.y & ~mask[1]) | (y.y & mask[1]);
        y.z = (old.z & ~mask[0]) | (y.z & mask[0]), y.w = (old.w & ~mask[1]) | (y.w & mask[1]);
      }
      *unit = y;
    }
  } else {
    static_assert(kSlots == 4, "two bytes of a dimension");
    for (uint32_t d = threadIdx.x; d < kDim; d += blockDim.x) {
      uint16_t *pair = reinterpret_cast<uint16_t *>(to + (d / 32 * P + (b.slot0 & ~15u) + d % 16) * 16 + d / 16 % 2 * 8 +
                                                    (b.slot0 & 15u) / 2);
      uint32_t y = gather(d, 0);
      if (mask[0] != 0xffffu) y = (*pair & ~mask[0]) | (y & mask[0]);
      *pair = uint16_t(y);
    }
  }
}

template <int kDim, int kSlots, bool kBoth, bool kTurn, bool kK16, bool kV16>
__device__ __forceinline__ void append_block(const AppendArgs &a, const Touched &t, uint32_t head, uint32_t side) {
  const Block b = block_of<kSlots>(a, t, head);
  // (the id is a scalar load that the compiler waits for here, and it has sunk the rows'
  // loads behind: a trip to memory each)
  const auto good = [&] {
    if (b.id >= 0 && b.id < int64_t(a.cache.pages)) return true;
    if (threadIdx.x == 0) atomicOr(a.status, kStatusBadCachePage);
    return false;
  };
  if constexpr (kBoth) {
    Row k = load_row<kDim, kTurn, kK16>(a, t, b, 0);
    const Row v = load_row<kDim, false, kV16>(a, t, b, 1);
    if (!good()) return;
    store_keys<kDim, kSlots, kTurn>(a, b, k);
    store_values<kDim, kSlots>(a, b, v);
  } else if (side == 0) {
    Row k = load_row<kDim, kTurn, kK16>(a, t, b, 0);
    if (good()) store_keys<kDim, kSlots, kTurn>(a, b, k);
  } else {
    const Row v = load_row<kDim, false, kV16>(a, t, b, 1);
    if (good()) store_values<kDim, kSlots>(a, b, v);
  }
}

// kBoth: keys and values by one workgroup, which looks for its sequence and page once.
// kTurn: K takes a norm or a rotation on the way.
template <int kDim, int kSlots, bool kBoth, bool kTurn>
__global__ __launch_bounds__(kSlots * kDim / 8 < 64 ? 64 : kSlots * kDim / 8) void k_kv_append4(AppendArgs a, uint32_t direct) {
  const uint32_t head = kBoth ? blockIdx.y : blockIdx.y >> 1, side = blockIdx.y & 1u;
  AppendArgs b = a;
  b.cache.page = kSlots;  // blocks are looked for as pages of these
  Touched t{};
  bool any;
  if (direct) {
    const uint32_t seq = blockIdx.x / direct;
    any = sequence_page(b, seq, clamp_row(a.cu[seq], a.tokens), clamp_row(a.cu[seq + 1], a.tokens), a.past[seq],
                        blockIdx.x % direct, t);
  } else {
    any = find_page(b, blockIdx.x, threadIdx.x & 63u, t);
  }
  if (any) {
    if (a.in[0].bf16)
      a.in[1].bf16 ? append_block<kDim, kSlots, kBoth, kTurn, true, true>(a, t, head, side)
                   : append_block<kDim, kSlots, kBoth, kTurn, true, false>(a, t, head, side);
    else
      a.in[1].bf16 ? append_block<kDim, kSlots, kBoth, kTurn, false, true>(a, t, head, side)
                   : append_block<kDim, kSlots, kBoth, kTurn, false, false>(a, t, head, side);
  }
  if (t.wrong && threadIdx.x == 0) atomicOr(a.status, t.wrong);
}

template <int kDim, int kSlots>
hipError_t append(hipStream_t s, const AppendArgs &a) {
  // the blocks that new tokens can touch: of the longest count, and in all
  const uint32_t each = (a.max_new + kSlots - 2) / kSlots + 1;
  const uint64_t most = uint64_t(a.seqs) * each;
  const uint64_t all = (uint64_t(a.tokens) + kSlots - 1) / kSlots + 2ull * a.seqs;
  // a few blocks each: a workgroup knows its sequence; else it looks for it
  const uint32_t direct = each <= 2 || most <= all ? each : 0;
  const uint32_t blocks = uint32_t(direct ? most : all);
  constexpr uint32_t kThreads = kSlots * kDim / 8 < 64 ? 64 : kSlots * kDim / 8;
  const auto launch = [&](auto kernel, uint32_t sides) {
    kernel<<<dim3(blocks, sides * a.cache.heads), kThreads, 0, s>>>(a, direct);
    return hipGetLastError();
  };
  const bool turn = a.k_weight || a.rope.table;
  // more workgroups than the card holds at once: keys and values by one (21 prompts
  // of up to 4,000 tokens, 8 heads of 128: 22.4 us, apart 30.3); else apart (8 tokens
  // of one head of 512 in blocks of 16: 4.6 us, by one 5.5)
  if constexpr (kSlots == 16)
    if (uint64_t(blocks) * a.cache.heads * kThreads > 256 * 2048)
      return turn ? launch(k_kv_append4<kDim, kSlots, true, true>, 1) : launch(k_kv_append4<kDim, kSlots, true, false>, 1);
  return turn ? launch(k_kv_append4<kDim, kSlots, false, true>, 2) : launch(k_kv_append4<kDim, kSlots, false, false>, 2);
}

// Blocks of 4 slots for up to 16 tokens of a sequence, more and smaller workgroups (us
// of 4 and 16 slots: 96 single tokens, 8 heads of 128, 4.4 / 6.0; 8 tokens of a head of
// 512 4.3 / 5.1; 32 sequences of 8 4.5 / 5.3; 8 of 16 4.4 / 4.4).
template <int kDim>
hipError_t append_dim(hipStream_t s, const AppendArgs &a) {
  return a.max_new <= 16 ? append<kDim, 4>(s, a) : append<kDim, 16>(s, a);
}

}  // namespace

hipError_t launch_kv4_append(hipStream_t s, const AppendArgs &a) {
  switch (a.cache.dim) {
    case 64: return append_dim<64>(s, a);
    case 128: return append_dim<128>(s, a);
    case 256: return append_dim<256>(s, a);
    case 512: return append_dim<512>(s, a);
  }
  return hipErrorInvalidValue;
}

}  // namespace s14
