// Per-head norms with the position rotation, the rotation's table, and the
// append of keys and values to the paged 8-bit cache.  All three are bound by
// the bytes they move, and for a few tokens by the launch.
#include "s14_attn_rows.hpp"

namespace s14 {
namespace {

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
