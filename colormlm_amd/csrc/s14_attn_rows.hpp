// A row's values in lanes, its norm and rotation, and the pages that an append
// touches: shared by the kernels of norms and appends (s14_attn_rows.hip,
// s14_attn_append4.hip).  Unnamed namespace: each kernel file gets its own copy.
#pragma once

#include "s14_attn.hpp"
#include "s14_attn_util.hpp"
#include "s14_device_util.hpp"

namespace s14 {
namespace {

// One lane's four neighbouring values of a row.
struct Quad {
  float v[4];
};

template <bool k16>
__device__ __forceinline__ Quad load_quad(const void *p, uint64_t at) {
  Quad q;
  if constexpr (k16) {
    const uint2 w = *reinterpret_cast<const uint2 *>(static_cast<const uint16_t *>(p) + at);
    q.v[0] = __uint_as_float(w.x << 16);
    q.v[1] = __uint_as_float(w.x & 0xffff0000u);
    q.v[2] = __uint_as_float(w.y << 16);
    q.v[3] = __uint_as_float(w.y & 0xffff0000u);
  } else {
    const float4 w = *reinterpret_cast<const float4 *>(static_cast<const float *>(p) + at);
    q.v[0] = w.x, q.v[1] = w.y, q.v[2] = w.z, q.v[3] = w.w;
  }
  return q;
}

template <bool k16>
__device__ __forceinline__ void store_quad(void *p, uint64_t at, const Quad &q) {
  if constexpr (k16) {
    *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(p) + at) =
        make_uint2(bf16_pair(q.v[0], q.v[1]), bf16_pair(q.v[2], q.v[3]));
  } else {
    *reinterpret_cast<float4 *>(static_cast<float *>(p) + at) = make_float4(q.v[0], q.v[1], q.v[2], q.v[3]);
  }
}

// What a lane holds of a row: two quads, at dimensions a and b.  A row of D
// values lies in D / 8 neighbouring lanes, so that both members of each
// rotated pair are in one lane and nothing but the norm's sum crosses lanes:
// in the half layout the first rot / 8 lanes hold the pairs (start + 4 u ..,
// rot / 2 further on) and the others the rest of the head in order, eight
// values each; otherwise lane u holds dimensions 8 u .. 8 u + 7.
struct Unit {
  uint32_t a, b;
  uint32_t angle;  // its first of four angles, where turned
  bool turned;
};
__device__ __forceinline__ Unit unit_of(uint32_t u, const RopeArgs &r) {
  Unit x{8 * u, 8 * u + 4, 0, false};
  if (!r.table) return x;
  if (r.interleaved) {
    x.turned = 8 * u - r.start < r.rot;  // wraps below start; start and rot are whole units
    x.angle = x.turned ? (8 * u - r.start) / 2 : 0;
  } else if (u < r.rot / 8) {
    x = Unit{r.start + 4 * u, r.start + 4 * u + r.rot / 2, 4 * u, true};
  } else {
    x.a = 8 * u - r.rot;
    if (x.a >= r.start) x.a += r.rot;
    x.b = x.a + 4;
  }
  return x;
}

// The sum of v over kLanes neighbouring lanes, in each of them: rows of 16 by
// DPP, then gfx950's permlane swaps.  No LDS permute.
template <int kLanes>
__device__ __forceinline__ float lane_sum(float v) {
  v += dpp_f<0xb1>(0.0f, v);   // quad_perm [1,0,3,2]
  v += dpp_f<0x4e>(0.0f, v);   // quad_perm [2,3,0,1]
  v += dpp_f<0x141>(0.0f, v);  // row_half_mirror
  if constexpr (kLanes >= 16) v += dpp_f<0x140>(0.0f, v);  // row_mirror
  if constexpr (kLanes >= 32) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  if constexpr (kLanes >= 64) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  return v;
}

struct Weight {
  float4 a, b;
};
__device__ __forceinline__ Weight load_weight(const float *w, const Unit &x) {
  return {*reinterpret_cast<const float4 *>(w + x.a), *reinterpret_cast<const float4 *>(w + x.b)};
}

// x * rsqrt(mean(x^2) + eps) * w.
template <int kLanes>
__device__ __forceinline__ void row_norm(Quad &a, Quad &b, const Weight &w, float eps) {
  float s = 0.0f;
#pragma unroll
  for (int j = 0; j < 4; ++j) s += a.v[j] * a.v[j] + b.v[j] * b.v[j];
  s = lane_sum<kLanes>(s);
  const float r = rsqrtf(s * (1.0f / float(8 * kLanes)) + eps);
  a.v[0] = a.v[0] * r * w.a.x, a.v[1] = a.v[1] * r * w.a.y, a.v[2] = a.v[2] * r * w.a.z, a.v[3] = a.v[3] * r * w.a.w;
  b.v[0] = b.v[0] * r * w.b.x, b.v[1] = b.v[1] * r * w.b.y, b.v[2] = b.v[2] * r * w.b.z, b.v[3] = b.v[3] * r * w.b.w;
}

// (p, q) -> (p c - q s, q c + p s) over a lane's four pairs at position pos.
// A position outside the table gives a row of NaN.
struct Angles {
  float4 c, s;
  bool good;
};
__device__ __forceinline__ Angles load_angles(const RopeArgs &r, const Unit &x, int32_t pos) {
  Angles n;
  n.good = uint32_t(pos) < r.positions;
  const float *row = r.table + uint64_t(n.good ? pos : 0) * r.rot + x.angle;
  n.c = *reinterpret_cast<const float4 *>(row);
  n.s = *reinterpret_cast<const float4 *>(row + r.rot / 2);
  return n;
}
__device__ __forceinline__ void row_rotate(Quad &a, Quad &b, const RopeArgs &r, const Unit &x, const Angles &n) {
  const float c[4] = {n.c.x, n.c.y, n.c.z, n.c.w}, s[4] = {n.s.x, n.s.y, n.s.z, n.s.w};
  const Quad p = a, q = b;
  if (x.turned) {
    if (r.interleaved) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        a.v[2 * j] = p.v[2 * j] * c[j] - p.v[2 * j + 1] * s[j];
        a.v[2 * j + 1] = p.v[2 * j + 1] * c[j] + p.v[2 * j] * s[j];
        b.v[2 * j] = q.v[2 * j] * c[j + 2] - q.v[2 * j + 1] * s[j + 2];
        b.v[2 * j + 1] = q.v[2 * j + 1] * c[j + 2] + q.v[2 * j] * s[j + 2];
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        a.v[j] = p.v[j] * c[j] - q.v[j] * s[j];
        b.v[j] = q.v[j] * c[j] + p.v[j] * s[j];
      }
    }
  }
  if (!n.good) {
#pragma unroll
    for (int j = 0; j < 4; ++j) a.v[j] = b.v[j] = __uint_as_float(0x7fc00000u);
  }
}

// The page that workgroup `index` of a (head, side) writes: pages of the first
// sequence first.  A sequence has the pages that its new tokens touch, the
// first max_new of them: the grid and the workgroups are made for these.
struct Touched {
  uint32_t seq;
  int64_t first, last, past, page;  // packed rows, and the page of the sequence
  uint32_t wrong;                   // status of the sequence's counts
};
// Page `k` of those that the sequence of rows first .. last - 1 touches.
__device__ __forceinline__ bool sequence_page(const AppendArgs &a, uint32_t seq, int64_t first, int64_t last,
                                              int64_t past, uint32_t k, Touched &t) {
  const int64_t end = min(last, first + int64_t(a.max_new));
  t = Touched{seq, first, end, past, past / a.cache.page + k, 0};
  if (last > first) t.wrong = past < 0 ? kStatusBadPast : last > end ? kStatusBadCounts : 0u;
  return past >= 0 && end > first && t.page * a.cache.page < past + (end - first);
}
__device__ __forceinline__ bool find_page(const AppendArgs &a, uint32_t index, uint32_t lane, Touched &t) {
  const uint32_t P = a.cache.page;
  uint32_t before = 0;
  for (uint32_t s0 = 0; s0 < a.seqs; s0 += 64) {
    const uint32_t s = s0 + lane;
    int32_t first = 0, last = 0, past = 0;  // packed rows fit 31 bits
    if (s < a.seqs) {
      first = int32_t(clamp_row(a.cu[s], a.tokens)), last = int32_t(clamp_row(a.cu[s + 1], a.tokens));
      past = a.past[s];
    }
    const uint32_t count = last > first ? min(uint32_t(last - first), a.max_new) : 0;
    const uint32_t pages = count ? (uint32_t(past) % P + count + P - 1) / P : 0;
    uint32_t sum = pages;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const uint32_t o = __shfl_up(sum, d);
      if (lane >= uint32_t(d)) sum += o;
    }
    const uint64_t here = __ballot(index - before < sum);
    if (here) {
      const int l = __builtin_amdgcn_readfirstlane(__builtin_ctzll(here));
      const auto of = [&](int32_t v) { return __builtin_amdgcn_readlane(v, l); };
      return sequence_page(a, s0 + l, of(first), of(last), of(past), index - before - uint32_t(of(sum) - of(pages)), t);
    }
    before += __builtin_amdgcn_readlane(sum, 63);
  }
  return false;
}

}  // namespace
}  // namespace s14
