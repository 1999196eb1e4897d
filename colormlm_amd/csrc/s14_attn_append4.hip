// Append of keys and values to the paged 4-bit cache (E2M1 codes, E8M0 scales of
// 32 dimensions of a key and of 128 of a value, 64 at heads of 64).
//
// A block's scale is 2^e, e the least with 6 2^e >= the largest magnitude (6 is
// E2M1's largest), held in -100 .. 100; codes are rounded to nearest, ties to even,
// and end at 6.  A token's scales are its own: nothing that was stored before is
// touched, so the unit of work is a block of kSlots neighbouring slots of a page
// (16, the slots of a unit of V codes, or 4 where few tokens are new), head and
// side, of D / 8 lanes a slot.  Bound by the bytes moved, for a few tokens by the
// launch.
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

// Eight codes of a block.
__device__ __forceinline__ uint32_t block_word(const float (&x)[8], uint32_t code) {
  if (code == 255u) return 0u;
  const float inv = __uint_as_float((254u - code) << 23);
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0] * inv, x[1] * inv, 1.0f, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2] * inv, x[3] * inv, 1.0f, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4] * inv, x[5] * inv, 1.0f, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6] * inv, x[7] * inv, 1.0f, 3);
}

// t.page counts blocks of kSlots tokens.
template <int kDim, int kSlots, bool kTurn, bool kIn16>
__device__ __forceinline__ void append_block(const AppendArgs &a, const Touched &t, uint32_t head, uint32_t side) {
  constexpr uint32_t kLanes = kDim / 8, kParts = kDim < 128 ? 1 : kDim / 128;
  const uint32_t P = a.cache.page;
  const int64_t start = t.page * kSlots, end = t.past + (t.last - t.first);
  const int64_t page = start / P;
  const int64_t id = page < int64_t(a.table_width) ? a.page_table[uint64_t(t.seq) * a.table_width + page] : -1;
  // new tokens take slots kept .. full - 1 of the block
  const uint32_t kept = t.past > start ? uint32_t(t.past - start) : 0u;
  const uint32_t full = end - start < int64_t(kSlots) ? uint32_t(end - start) : kSlots;
  const uint32_t lane = threadIdx.x % kLanes, row = threadIdx.x / kLanes;
  const bool live = row >= kept && row < full;
  const uint32_t r = row < kept ? kept : row < full ? row : full - 1;  // whole wavefronts sum
  const AttnRows in = a.in[side];
  RopeArgs rope = a.rope;
  if (!kTurn || side) rope.table = nullptr;
  const float *weight = !kTurn || side ? nullptr : a.k_weight;
  const Unit x = unit_of(lane, rope);
  const uint64_t at = uint64_t(t.first + (start + r - t.past)) * in.token + uint64_t(head) * in.head;
  Quad p = load_quad<kIn16>(in.p, at + x.a), q = load_quad<kIn16>(in.p, at + x.b);
  Weight w{};
  if (weight) w = load_weight(weight, x);
  Angles n{};
  if (rope.table) n = load_angles(rope, x, int32_t(min(start + r, int64_t(INT_MAX))));
  // (the id's load is in flight with the rows')
  if (id < 0 || id >= int64_t(a.cache.pages)) {
    if (threadIdx.x == 0) atomicOr(a.status, kStatusBadCachePage);
    return;
  }
  if (weight) row_norm<kLanes>(p, q, w, a.eps);
  if (rope.table) {
    row_rotate(p, q, rope, x, n);
    if (!n.good && live && lane == 0) atomicOr(a.status, kStatusBadPosition);
  }

  const uint32_t slot0 = uint32_t(start) & (P - 1), slot = slot0 + row;  // of the page
  const uint64_t place = uint64_t(id) * a.cache.heads + head;
  if (side == 0) {
    // eight neighbouring dimensions a lane, where the rotation had them otherwise
    __shared__ float s_row[kSlots][kDim];
    if (rope.table && !rope.interleaved) {
      if (row < kSlots) {
        *reinterpret_cast<float4 *>(&s_row[row][x.a]) = make_float4(p.v[0], p.v[1], p.v[2], p.v[3]);
        *reinterpret_cast<float4 *>(&s_row[row][x.b]) = make_float4(q.v[0], q.v[1], q.v[2], q.v[3]);
      }
      __syncthreads();
      if (row < kSlots) {
        const float4 y = *reinterpret_cast<const float4 *>(&s_row[row][8 * lane]);
        const float4 z = *reinterpret_cast<const float4 *>(&s_row[row][8 * lane + 4]);
        p.v[0] = y.x, p.v[1] = y.y, p.v[2] = y.z, p.v[3] = y.w;
        q.v[0] = z.x, q.v[1] = z.y, q.v[2] = z.z, q.v[3] = z.w;
      }
    }
  }
  float v[8];
  uint32_t amax = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    v[i] = i < 4 ? p.v[i & 3] : q.v[i & 3];
    amax = max(amax, __float_as_uint(v[i]) & 0x7fffffffu);  // magnitudes order as their bits
  }
  if (side == 0) {
    const uint32_t code = block_code(lane_max<4>(amax));
    if (!live) return;
    *reinterpret_cast<uint32_t *>(a.cache.k + (place * P + slot) * (kDim / 2) + 4 * lane) = block_word(v, code);
    if (lane % 4 == 0)
      a.cache.ks[place * (kDim / 32 * P) + lane / 4 * P + (slot & ~15u) + 4 * (slot & 3u) + ((slot >> 2) & 3u)] = uint8_t(code);
    return;
  }
  const uint32_t code = block_code(lane_max<kDim < 128 ? 8 : 16>(amax));
  if (live && lane % (kDim < 128 ? 8 : 16) == 0) a.cache.vs[(place * kParts + lane / 16) * P + slot] = uint8_t(code);
  // two slots a byte: the slots of a dimension come together through LDS
  __shared__ uint32_t s_code[kSlots][kLanes];
  if (row < kSlots) s_code[row][lane] = block_word(v, code);
  __syncthreads();
  // nibbles kept .. full - 1 are new, the others stay
  constexpr uint32_t kWords = kSlots / 8 ? kSlots / 8 : 1;
  uint32_t mask[kWords];
#pragma unroll
  for (uint32_t k = 0; k < kWords; ++k) {
    const uint32_t from = kept > 8 * k ? min(kept - 8 * k, 8u) : 0u, to = full > 8 * k ? min(full - 8 * k, 8u) : 0u;
    mask[k] = uint32_t((1ull << (4 * to)) - 1u) & ~uint32_t((1ull << (4 * from)) - 1u);
  }
  const auto gather = [&](uint32_t dim, uint32_t k) {  // eight slots (or four) of a dimension
    uint32_t c = 0;
#pragma unroll
    for (uint32_t j = 0; j < (kSlots < 8 ? kSlots : 8); ++j) c |= ((s_code[8 * k + j][dim / 8] >> (4 * (dim % 8))) & 15u) << (4 * j);
    return c;
  };
  uint8_t *to = a.cache.v + place * P * (kDim / 2);
  if constexpr (kSlots == 16) {
    // a unit of 16 bytes: dimensions d and d + 16, 16 slots
    for (uint32_t u = threadIdx.x; u < kDim / 2; u += blockDim.x) {
      const uint32_t d = u / 16 * 32 + u % 16;
      uint4 *unit = reinterpret_cast<uint4 *>(to + (u / 16 * P + slot0 + u % 16) * 16);
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
      uint16_t *pair = reinterpret_cast<uint16_t *>(to + (d / 32 * P + (slot0 & ~15u) + d % 16) * 16 + d / 16 % 2 * 8 +
                                                    (slot0 & 15u) / 2);
      uint32_t y = gather(d, 0);
      if (mask[0] != 0xffffu) y = (*pair & ~mask[0]) | (y & mask[0]);
      *pair = uint16_t(y);
    }
  }
}

// kTurn: K takes a norm or a rotation on the way.
template <int kDim, int kSlots, bool kTurn>
__global__ __launch_bounds__(kSlots * kDim / 8 < 64 ? 64 : kSlots * kDim / 8) void k_kv_append4(AppendArgs a, uint32_t direct) {
  const uint32_t head = blockIdx.y >> 1, side = blockIdx.y & 1u;
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
    if (a.in[side].bf16)
      append_block<kDim, kSlots, kTurn, true>(a, t, head, side);
    else
      append_block<kDim, kSlots, kTurn, false>(a, t, head, side);
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
  const dim3 grid(uint32_t(direct ? most : all), 2 * a.cache.heads);
  constexpr uint32_t kThreads = kSlots * kDim / 8 < 64 ? 64 : kSlots * kDim / 8;
  if (a.k_weight || a.rope.table)
    k_kv_append4<kDim, kSlots, true><<<grid, kThreads, 0, s>>>(a, direct);
  else
    k_kv_append4<kDim, kSlots, false><<<grid, kThreads, 0, s>>>(a, direct);
  return hipGetLastError();
}

template <int kDim>
hipError_t append_dim(hipStream_t s, const AppendArgs &a) {
  return a.max_new <= 4 ? append<kDim, 4>(s, a) : append<kDim, 16>(s, a);
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
