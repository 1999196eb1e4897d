// Per-head norms with the position rotation, the rotation's table, and the
// append of keys and values to the paged 8-bit cache.  All three are bound by
// the bytes they move, and for a few tokens by the launch.
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

// Four codes by the hardware's conversion (to nearest even).  The scale keeps
// every value within 448 but an infinity, which is brought there; a NaN
// keeps its place as the NaN code.
__device__ __forceinline__ uint32_t e4m3_word(const Quad &x, float inv) {
  float y[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    y[j] = x.v[j] * inv;
    y[j] = y[j] > 448.0f ? 448.0f : y[j] < -448.0f ? -448.0f : y[j];
  }
  const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
  return uint32_t(__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], lo, true));
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

// ---------------------------------------------------------------------------
// norms of queries and keys with the rotation
// ---------------------------------------------------------------------------

// One row per D / 8 lanes.  A workgroup's rows are all of one side and numbered
// (token, head), so that what it takes from the arguments is scalar: rows of
// both sides in a workgroup fetched their strides and pointers by lane (16,384
// tokens of 40 heads: 124 us; so 94, 5.4 TB/s).  Two and four rows a lane
// group were 92 and 97 us.
template <int kDim, bool kIn16, bool kOut16>
__device__ __forceinline__ void norm_rope_rows(const NormRopeArgs &a, uint32_t side, uint32_t block) {
  constexpr int kLanes = kDim / 8;
  const uint32_t lane = threadIdx.x % kLanes;
  const AttnRows in = a.in[side];
  const AttnOut out = a.out[side];
  const float *weight = a.weight[side];
  const uint32_t rows = a.tokens * in.heads;
  const Unit x = unit_of(lane, a.rope);
  uint32_t row = block * (256 / kLanes) + threadIdx.x / kLanes;
  const bool live = row < rows;
  if (!live) row = rows - 1;  // whole wavefronts sum
  const uint32_t t = row / in.heads, h = row % in.heads;
  const uint64_t at = t * in.token + uint64_t(h) * in.head;
  Quad p = load_quad<kIn16>(in.p, at + x.a), q = load_quad<kIn16>(in.p, at + x.b);
  Angles n;
  if (a.rope.table) n = load_angles(a.rope, x, a.positions[t]);
  if (weight) row_norm<kLanes>(p, q, load_weight(weight, x), a.eps);
  if (a.rope.table) {
    row_rotate(p, q, a.rope, x, n);
    if (!n.good && live && lane == 0) atomicOr(a.status, kStatusBadPosition);
  }
  if (!live) return;
  const uint64_t to = t * out.token + uint64_t(h) * out.head;
  store_quad<kOut16>(out.p, to + x.a, p);
  store_quad<kOut16>(out.p, to + x.b, q);
}

template <int kDim>
__global__ __launch_bounds__(256) void k_norm_rope(NormRopeArgs a, uint32_t q_blocks) {
  const uint32_t side = blockIdx.x < q_blocks ? 0u : 1u, block = blockIdx.x - (side ? q_blocks : 0u);
  if (a.in[side].bf16) {
    if (a.out[side].bf16)
      norm_rope_rows<kDim, true, true>(a, side, block);
    else
      norm_rope_rows<kDim, true, false>(a, side, block);
  } else {
    if (a.out[side].bf16)
      norm_rope_rows<kDim, false, true>(a, side, block);
    else
      norm_rope_rows<kDim, false, false>(a, side, block);
  }
}

// cos and sin of position p times each frequency, from an angle in 64 bits
// (a far position's angle in 32 bits is off by whole turns' worth of its last
// digits).  Frequencies theta^(-2 i / rot), divided by `factor` where the
// context is stretched: all of them (original 0), or, where the trained
// length is given, those that turn less than `slow` times in it fully, those
// that turn more than `fast` times not at all, and those between in part.
__global__ __launch_bounds__(256) void k_rope_table(RopeTableArgs a) {
  const uint32_t half = a.rot / 2;
  const uint64_t i = uint64_t(blockIdx.x) * 256 + threadIdx.x;
  if (i >= uint64_t(a.positions) * half) return;
  const uint32_t p = uint32_t(i / half), f = uint32_t(i % half);
  double inv = pow(a.theta, -2.0 * double(f) / double(a.rot));
  if (a.factor != 1.0) {
    double part = 1.0;  // how far this frequency is divided
    if (a.original > 0.0) {
      const double per = 2.0 * log(a.theta) / double(a.rot);  // ln of the ratio of neighbouring frequencies
      const double two_pi = 6.283185307179586476925286766559;
      const double lo = fmax(floor(log(a.original / (a.fast * two_pi)) / per), 0.0);
      double hi = fmin(ceil(log(a.original / (a.slow * two_pi)) / per), double(a.rot) - 1.0);
      if (hi <= lo) hi = lo + 0.001;
      part = fmin(fmax((double(f) - lo) / (hi - lo), 0.0), 1.0);
    }
    inv = inv / a.factor * part + inv * (1.0 - part);
  }
  double s, c;
  sincos(double(p) * inv, &s, &c);
  a.out[uint64_t(p) * a.rot + f] = float(c * a.amplitude);
  a.out[uint64_t(p) * a.rot + half + f] = float(s * a.amplitude);
}

// ---------------------------------------------------------------------------
// append to the paged cache
// ---------------------------------------------------------------------------

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

// One workgroup per (page that the new tokens touch, key head, side).
// It finds the largest magnitude of its new rows, raises the page's E8M0
// scale where they need it (an earlier token's codes are then divided by a
// power of two: exact but for those that fall below 2^-6), and writes the new
// rows' codes.  K codes lie [slot][dim]; V codes [dim][slot], so that the
// attention's second product reads them as its operand without a transpose.
//
// A lane holds eight dimensions (Unit) of four neighbouring slots, kIt times
// over: four V codes of a dimension are one word.
template <int kDim, int kIt, bool kTurn, bool kIn16>
__device__ __forceinline__ void append_page(const AppendArgs &a, const Touched &t, uint32_t head, uint32_t side) {
  constexpr uint32_t kLanes = kDim / 8;
  const uint32_t P = a.cache.page;
  const int64_t start = t.page * P, end = t.past + (t.last - t.first);
  const int64_t id = t.page < int64_t(a.table_width) ? a.page_table[uint64_t(t.seq) * a.table_width + t.page] : -1;
  // new tokens take slots kept .. full - 1
  const uint32_t kept = t.past > start ? uint32_t(t.past - start) : 0u;
  const uint32_t full = end - start < int64_t(P) ? uint32_t(end - start) : P;
  const uint32_t lane = threadIdx.x % kLanes, groups = blockDim.x / kLanes;
  const uint32_t slot0 = kept / 4 * 4 + 4 * (threadIdx.x / kLanes);
  const AttnRows in = a.in[side];
  RopeArgs rope = a.rope;
  if (!kTurn || side) rope.table = nullptr;
  const float *weight = !kTurn || side ? nullptr : a.k_weight;
  const Unit x = unit_of(lane, rope);

  Quad p[kIt][4], q[kIt][4];
#pragma unroll
  for (int it = 0; it < kIt; ++it)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t slot = slot0 + 4 * groups * it + j;
      const uint32_t s = slot < kept ? kept : slot < full ? slot : full - 1;  // whole wavefronts sum
      const uint64_t at = uint64_t(t.first + (start + s - t.past)) * in.token + uint64_t(head) * in.head;
      p[it][j] = load_quad<kIn16>(in.p, at + x.a), q[it][j] = load_quad<kIn16>(in.p, at + x.b);
    }
  Weight w{};
  if (weight) w = load_weight(weight, x);
  // (the id's load is in flight with the rows')
  if (id < 0 || id >= int64_t(a.cache.pages)) {
    if (threadIdx.x == 0) atomicOr(a.status, kStatusBadCachePage);
    return;
  }
  float amax = 0.0f;
#pragma unroll
  for (int it = 0; it < kIt; ++it) {
    if (kept / 4 * 4 + 4 * groups * it >= full) continue;  // uniform: past the last slot
    Angles n[4];
    const auto angles = [&](int j) {
      const uint32_t slot = slot0 + 4 * groups * it + j;
      const uint32_t s = slot < kept ? kept : slot < full ? slot : full - 1;
      n[j] = load_angles(rope, x, int32_t(min(start + s, int64_t(INT_MAX))));
    };
    if (kIt == 1 && rope.table) {  // (kIt 2 has no registers for all at once)
#pragma unroll
      for (int j = 0; j < 4; ++j) angles(j);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (weight) row_norm<kLanes>(p[it][j], q[it][j], w, a.eps);
      if (rope.table) {
        if (kIt > 1) angles(j);
        row_rotate(p[it][j], q[it][j], rope, x, n[j]);
        if (!n[j].good && lane == 0) atomicOr(a.status, kStatusBadPosition);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {  // a NaN is never greater
        amax = fabsf(p[it][j].v[i]) > amax ? fabsf(p[it][j].v[i]) : amax;
        amax = fabsf(q[it][j].v[i]) > amax ? fabsf(q[it][j].v[i]) : amax;
      }
    }
  }
  __shared__ uint32_t s_amax[16];
  amax = __uint_as_float(wave_max_u32(__float_as_uint(amax)));  // magnitudes order as their bits
  if ((threadIdx.x & 63u) == 0) s_amax[threadIdx.x / 64] = __float_as_uint(amax);
  uint8_t *scale = (side ? a.cache.vs : a.cache.ks) + uint64_t(id) * a.cache.heads + head;
  uint8_t *codes = (side ? a.cache.v : a.cache.k) + (uint64_t(id) * a.cache.heads + head) * P * kDim;
  const uint32_t before = kept ? *scale : 0u;
  __syncthreads();  // and every thread has read the old scale
  for (uint32_t w = 0; w < blockDim.x / 64; ++w) amax = fmaxf(amax, __uint_as_float(s_amax[w]));

  // the largest finite scale holds an infinity, whose code is the largest value's
  const uint32_t code = max(before, min(requant_code(amax), 254u));
  if (threadIdx.x == 0) *scale = uint8_t(code);
  const float inv = power_of_two(127 - int(code));
  if (kept && before != code) {
    const float shift = power_of_two(int(before) - int(code));
    for (uint32_t e = threadIdx.x; e < kept * uint32_t(kDim); e += blockDim.x) {
      const uint32_t at = side ? e / kept * P + e % kept : e;
      const uint32_t c = codes[at];
      if ((c & 0x7fu) != 0x7fu) codes[at] = uint8_t(s14x::e4m3_rne_sat(e4m3_f32(c) * shift));
    }
  }
#pragma unroll
  for (int it = 0; it < kIt; ++it) {
    const uint32_t slot = slot0 + 4 * groups * it;
    if (slot >= full) continue;
    uint32_t w[2][4];  // word j: slot slot + j, four dimensions
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      w[0][j] = e4m3_word(p[it][j], inv);
      w[1][j] = e4m3_word(q[it][j], inv);
    }
    if (side == 0) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (slot + j < kept || slot + j >= full) continue;
        *reinterpret_cast<uint32_t *>(codes + (slot + j) * kDim + x.a) = w[0][j];
        *reinterpret_cast<uint32_t *>(codes + (slot + j) * kDim + x.b) = w[1][j];
      }
    } else {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const uint32_t lo0 = __builtin_amdgcn_perm(w[k][1], w[k][0], 0x05010400u);  // dimensions 0, 1 of slots 0, 1
        const uint32_t hi0 = __builtin_amdgcn_perm(w[k][1], w[k][0], 0x07030602u);  // dimensions 2, 3
        const uint32_t lo1 = __builtin_amdgcn_perm(w[k][3], w[k][2], 0x05010400u);
        const uint32_t hi1 = __builtin_amdgcn_perm(w[k][3], w[k][2], 0x07030602u);
        const uint32_t c[4] = {(lo0 & 0xffffu) | (lo1 << 16), (lo0 >> 16) | (lo1 & 0xffff0000u),
                               (hi0 & 0xffffu) | (hi1 << 16), (hi0 >> 16) | (hi1 & 0xffff0000u)};
        uint8_t *to = codes + (k ? x.b : x.a) * P + slot;
        const bool whole = slot >= kept && slot + 4 <= full;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (whole) {
            *reinterpret_cast<uint32_t *>(to + i * P) = c[i];
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (slot + j >= kept && slot + j < full) to[i * P + j] = uint8_t(c[i] >> (8 * j));
          }
        }
      }
    }
  }
}

// kTurn: K takes a norm or a rotation on the way.
template <int kDim, int kIt, bool kTurn>
__global__ __launch_bounds__(1024) void k_kv_append(AppendArgs a, uint32_t direct) {
  const uint32_t head = blockIdx.y >> 1, side = blockIdx.y & 1u;
  Touched t{};
  bool any;
  if (direct) {
    const uint32_t seq = blockIdx.x / direct;
    any = sequence_page(a, seq, clamp_row(a.cu[seq], a.tokens), clamp_row(a.cu[seq + 1], a.tokens), a.past[seq],
                        blockIdx.x % direct, t);
  } else {
    any = find_page(a, blockIdx.x, threadIdx.x & 63u, t);
  }
  if (any) {
    if (a.in[side].bf16)
      append_page<kDim, kIt, kTurn, true>(a, t, head, side);
    else
      append_page<kDim, kIt, kTurn, false>(a, t, head, side);
  }
  if (t.wrong && threadIdx.x == 0) atomicOr(a.status, t.wrong);
}

}  // namespace

hipError_t launch_rope_table(hipStream_t s, const RopeTableArgs &a) {
  const uint64_t n = uint64_t(a.positions) * (a.rot / 2);
  k_rope_table<<<uint32_t((n + 255) / 256), 256, 0, s>>>(a);
  return hipGetLastError();
}

template <int kDim>
static hipError_t norm_rope(hipStream_t s, const NormRopeArgs &a) {
  constexpr uint64_t kRows = 256 / (kDim / 8);
  const uint64_t q = (uint64_t(a.tokens) * a.in[0].heads + kRows - 1) / kRows;
  const uint64_t k = (uint64_t(a.tokens) * a.in[1].heads + kRows - 1) / kRows;
  k_norm_rope<kDim><<<uint32_t(q + k), 256, 0, s>>>(a, uint32_t(q));
  return hipGetLastError();
}

hipError_t launch_norm_rope(hipStream_t s, const NormRopeArgs &a) {
  switch (a.dim) {
    case 64: return norm_rope<64>(s, a);
    case 128: return norm_rope<128>(s, a);
    case 256: return norm_rope<256>(s, a);
    case 512: return norm_rope<512>(s, a);
  }
  return hipErrorInvalidValue;
}

template <int kDim>
static hipError_t kv_append(hipStream_t s, const AppendArgs &a) {
  constexpr uint32_t kLanes = kDim / 8;
  const uint32_t P = a.cache.page;
  // the pages that new tokens can touch: of the longest count, and in all
  const uint32_t each = (a.max_new + P - 2) / P + 1;
  const uint64_t most = uint64_t(a.seqs) * each;
  const uint64_t all = (uint64_t(a.tokens) + P - 1) / P + 2ull * a.seqs;
  // a few pages each: a workgroup knows its sequence; else it looks for it
  const uint32_t direct = each <= 2 || most <= all ? each : 0;
  const dim3 grid(uint32_t(direct ? most : all), 2 * a.cache.heads);
  // threads for the slot groups (of four) that a sequence can fill
  uint32_t groups = (a.max_new + 2) / 4 + 1;
  if (groups > P / 4) groups = P / 4;
  const uint32_t threads = (groups * kLanes + 63) / 64 * 64;
  const bool turn = a.k_weight || a.rope.table;
  const auto launch = [&](auto kernel) {
    kernel<<<grid, threads < 1024 ? threads : 1024, 0, s>>>(a, direct);
    return hipGetLastError();
  };
  if constexpr (kDim == 512)
    if (threads > 1024) return turn ? launch(k_kv_append<kDim, 2, true>) : launch(k_kv_append<kDim, 2, false>);
  return turn ? launch(k_kv_append<kDim, 1, true>) : launch(k_kv_append<kDim, 1, false>);
}

hipError_t launch_kv_append(hipStream_t s, const AppendArgs &a) {
  switch (a.cache.dim) {
    case 64: return kv_append<64>(s, a);
    case 128: return kv_append<128>(s, a);
    case 256: return kv_append<256>(s, a);
    case 512: return kv_append<512>(s, a);
  }
  return hipErrorInvalidValue;
}

}  // namespace s14
