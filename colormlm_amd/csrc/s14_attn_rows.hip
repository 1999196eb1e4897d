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

__device__ __forceinline__ Quad load_quad(const AttnRows &r, uint64_t at) {
  Quad q;
  if (r.bf16) {
    const uint2 w = *reinterpret_cast<const uint2 *>(static_cast<const uint16_t *>(r.p) + at);
    q.v[0] = __uint_as_float(w.x << 16);
    q.v[1] = __uint_as_float(w.x & 0xffff0000u);
    q.v[2] = __uint_as_float(w.y << 16);
    q.v[3] = __uint_as_float(w.y & 0xffff0000u);
  } else {
    const float4 w = *reinterpret_cast<const float4 *>(static_cast<const float *>(r.p) + at);
    q.v[0] = w.x, q.v[1] = w.y, q.v[2] = w.z, q.v[3] = w.w;
  }
  return q;
}

__device__ __forceinline__ void store_quad(const AttnOut &o, uint64_t at, const Quad &q) {
  if (o.bf16) {
    *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(o.p) + at) =
        make_uint2(bf16_pair(q.v[0], q.v[1]), bf16_pair(q.v[2], q.v[3]));
  } else {
    *reinterpret_cast<float4 *>(static_cast<float *>(o.p) + at) = make_float4(q.v[0], q.v[1], q.v[2], q.v[3]);
  }
}

// x * rsqrt(mean(x^2) + eps) * w over a row that `lanes` neighbouring lanes
// hold, kQ quads a lane (quad i of lane l: dimensions 4 * (l + lanes * i)).
template <int kLanes, int kQ>
__device__ __forceinline__ void row_norm(Quad (&q)[kQ], const float *weight, uint32_t lane, float eps) {
  float s = 0.0f;
#pragma unroll
  for (int i = 0; i < kQ; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) s += q[i].v[j] * q[i].v[j];
#pragma unroll
  for (int m = kLanes / 2; m; m >>= 1) s += __shfl_xor(s, m);
  const float r = 1.0f / __fsqrt_rn(s * (1.0f / float(4 * kLanes * kQ)) + eps);
#pragma unroll
  for (int i = 0; i < kQ; ++i) {
    const float4 w = *reinterpret_cast<const float4 *>(weight + 4 * (lane + kLanes * i));
    q[i].v[0] = q[i].v[0] * r * w.x;
    q[i].v[1] = q[i].v[1] * r * w.y;
    q[i].v[2] = q[i].v[2] * r * w.z;
    q[i].v[3] = q[i].v[3] * r * w.w;
  }
}

// The rotation of a row's dimensions start .. start + rot: (a, b) -> (a c -
// b s, b c + a s), a pair being neighbours (interleaved) or rot / 2 apart.
// rot / 2 and start are multiples of 4, so in the half layout a quad's
// partners are a quad of another lane, fetched by a lane permute: the whole
// wavefront takes part.  A position outside the table gives NaN.
template <int kLanes, int kQ>
__device__ __forceinline__ void row_rotate(Quad (&q)[kQ], const RopeArgs &r, uint32_t lane, int32_t pos,
                                           uint32_t *status, bool live) {
  const bool good = uint32_t(pos) < r.positions;
  if (!good && live && lane == 0) atomicOr(status, kStatusBadPosition);
  const float *row = r.table + uint64_t(good ? pos : 0) * r.rot;
  const uint32_t half = r.rot / 2;
  Quad old[kQ];
#pragma unroll
  for (int i = 0; i < kQ; ++i) old[i] = q[i];
#pragma unroll
  for (int i = 0; i < kQ; ++i) {
    const uint32_t d = 4 * (lane + kLanes * i) - r.start;  // wraps below start: >= rot
    const bool in = d < r.rot;
    if (r.interleaved) {
      if (!in) continue;
      const float2 c = *reinterpret_cast<const float2 *>(row + d / 2);
      const float2 s = *reinterpret_cast<const float2 *>(row + half + d / 2);
      const Quad x = old[i];
      q[i].v[0] = x.v[0] * c.x - x.v[1] * s.x;
      q[i].v[1] = x.v[1] * c.x + x.v[0] * s.x;
      q[i].v[2] = x.v[2] * c.y - x.v[3] * s.y;
      q[i].v[3] = x.v[3] * c.y + x.v[2] * s.y;
    } else {
      const bool first = d < half;
      const uint32_t pd = in ? (first ? d + half : d - half) + r.start : 4 * lane;  // partner dimension
      const uint32_t src = ((threadIdx.x & 63u) & ~uint32_t(kLanes - 1)) + (pd / 4) % kLanes;
      const uint32_t pi = pd / 4 / kLanes;
      Quad y{};
#pragma unroll
      for (int k = 0; k < kQ; ++k) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float f = __shfl(old[k].v[j], int(src));
          if (pi == uint32_t(k)) y.v[j] = f;
        }
      }
      if (!in) continue;
      const uint32_t e = first ? d : d - half;
      const float4 c = *reinterpret_cast<const float4 *>(row + e);
      const float4 s = *reinterpret_cast<const float4 *>(row + half + e);
      const float cs[4] = {c.x, c.y, c.z, c.w}, sn[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
      for (int j = 0; j < 4; ++j)
        q[i].v[j] = first ? old[i].v[j] * cs[j] - y.v[j] * sn[j] : old[i].v[j] * cs[j] + y.v[j] * sn[j];
    }
  }
  if (!good) {
#pragma unroll
    for (int i = 0; i < kQ; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) q[i].v[j] = __uint_as_float(0x7fc00000u);
  }
}

// ---------------------------------------------------------------------------
// norms of queries and keys with the rotation
// ---------------------------------------------------------------------------

// One row of kDim values per kLanes lanes, 16 bytes of f32 (8 of bf16) a lane
// and load.  Rows are numbered (token, query heads then key heads).
template <int kDim>
__global__ __launch_bounds__(256) void k_norm_rope(NormRopeArgs a) {
  constexpr int kLanes = kDim / 4 < 64 ? kDim / 4 : 64;
  constexpr int kQ = kDim / (4 * kLanes);
  constexpr uint32_t kRows = 256 / kLanes;
  const uint32_t lane = threadIdx.x % kLanes;
  const uint32_t heads = a.in[0].heads + a.in[1].heads;
  const uint64_t rows = uint64_t(a.tokens) * heads;
  uint64_t row = uint64_t(blockIdx.x) * kRows + threadIdx.x / kLanes;
  const bool live = row < rows;
  if (!live) row = rows - 1;  // whole wavefronts permute
  const uint32_t t = uint32_t(row / heads), h = uint32_t(row % heads);
  const uint32_t side = h < a.in[0].heads ? 0 : 1;
  const AttnRows in = a.in[side];
  const AttnOut out = a.out[side];
  const float *weight = a.weight[side];
  const uint32_t hh = side ? h - a.in[0].heads : h;
  Quad q[kQ];
  const uint64_t at = uint64_t(t) * in.token + uint64_t(hh) * in.head;
#pragma unroll
  for (int i = 0; i < kQ; ++i) q[i] = load_quad(in, at + 4 * (lane + kLanes * i));
  Quad n[kQ];
#pragma unroll
  for (int i = 0; i < kQ; ++i) n[i] = q[i];
  if (a.weight[0] || a.weight[1]) {  // uniform: the sum crosses lanes of both sides
    const float *w = weight ? weight : (a.weight[0] ? a.weight[0] : a.weight[1]);
    row_norm<kLanes, kQ>(n, w, lane, a.eps);
    if (!weight) {
#pragma unroll
      for (int i = 0; i < kQ; ++i) n[i] = q[i];
    }
  }
  if (a.rope.table) row_rotate<kLanes, kQ>(n, a.rope, lane, a.positions[t], a.status, live);
  if (!live) return;
  const uint64_t to = uint64_t(t) * out.token + uint64_t(hh) * out.head;
#pragma unroll
  for (int i = 0; i < kQ; ++i) store_quad(out, to + 4 * (lane + kLanes * i), n[i]);
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

// One workgroup per (page that the new tokens touch, key head, side, sequence).
// It finds the largest magnitude of its new rows, raises the page's E8M0
// scale where they need it (an earlier token's codes are then divided by a
// power of two: exact but for those that fall below 2^-6), and writes the new
// rows' codes.  K codes lie [slot][dim]; V codes [dim][slot], so that the
// attention's second product reads them as its operand without a transpose.
//
// Each thread keeps up to kIt quads of rows between the two passes.
template <int kDim, int kIt>
__global__ __launch_bounds__(1024) void k_kv_append(AppendArgs a) {
  constexpr int kLanes = kDim / 4 < 64 ? kDim / 4 : 64;
  constexpr int kQ = kDim / (4 * kLanes);
  const uint32_t seq = blockIdx.z, head = blockIdx.y >> 1, side = blockIdx.y & 1u;
  const uint32_t P = a.cache.page;
  const int64_t first = clamp_row(a.cu[seq], a.tokens), last = clamp_row(a.cu[seq + 1], a.tokens);
  const int64_t past = a.past[seq];
  if (last <= first || past < 0) return;
  const int64_t page = past / P + blockIdx.x;  // page of the sequence
  const int64_t lo = max(past, page * int64_t(P)), hi = min(past + (last - first), (page + 1) * int64_t(P));
  if (lo >= hi) return;
  const int64_t id = page < int64_t(a.table_width) ? a.page_table[uint64_t(seq) * a.table_width + page] : -1;
  if (id < 0 || id >= int64_t(a.cache.pages)) {
    if (threadIdx.x == 0) atomicOr(a.status, kStatusBadCachePage);
    return;
  }
  const uint32_t kept = uint32_t(lo - page * P), n = uint32_t(hi - lo);  // earlier and new tokens of the page
  const uint32_t lane = threadIdx.x % kLanes, row0 = threadIdx.x / kLanes, rows = blockDim.x / kLanes;
  const AttnRows in = a.in[side];
  const uint64_t base = uint64_t(first + lo - past) * in.token + uint64_t(head) * in.head;

  Quad q[kIt][kQ];
  float amax = 0.0f;
#pragma unroll
  for (int it = 0; it < kIt; ++it) {
    const uint32_t r = row0 + rows * it;
    if (rows * it >= n) continue;  // uniform
    const uint32_t rr = r < n ? r : n - 1;
#pragma unroll
    for (int i = 0; i < kQ; ++i) q[it][i] = load_quad(in, base + rr * in.token + 4 * (lane + kLanes * i));
    if (side == 0) {
      if (a.k_weight) row_norm<kLanes, kQ>(q[it], a.k_weight, lane, a.eps);
      if (a.rope.table)
        row_rotate<kLanes, kQ>(q[it], a.rope, lane, int32_t(min(lo + rr, int64_t(INT_MAX))), a.status, true);
    }
#pragma unroll
    for (int i = 0; i < kQ; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) amax = fabsf(q[it][i].v[j]) > amax ? fabsf(q[it][i].v[j]) : amax;  // NaN: no part
  }
  __shared__ float s_amax[16];
#pragma unroll
  for (int m = 32; m; m >>= 1) {
    const float o = __shfl_xor(amax, m);
    amax = o > amax ? o : amax;
  }
  if ((threadIdx.x & 63u) == 0) s_amax[threadIdx.x / 64] = amax;
  __syncthreads();
  for (uint32_t w = 0; w < blockDim.x / 64; ++w) amax = s_amax[w] > amax ? s_amax[w] : amax;

  uint8_t *scale = (side ? a.cache.vs : a.cache.ks) + uint64_t(id) * a.cache.heads + head;
  uint8_t *codes = (side ? a.cache.v : a.cache.k) + (uint64_t(id) * a.cache.heads + head) * P * kDim;
  const uint32_t before = kept ? *scale : 0u;
  // the largest finite scale holds an infinity, whose code is the largest value's
  const uint32_t code = max(before, min(requant_code(amax), 254u));
  __syncthreads();  // every thread has read the old scale
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
    const uint32_t r = row0 + rows * it;
    if (r >= n) continue;
#pragma unroll
    for (int i = 0; i < kQ; ++i) {
      const uint32_t d = 4 * (lane + kLanes * i);
      uint32_t w = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) w |= s14x::e4m3_rne_sat(q[it][i].v[j] * inv) << (8 * j);
      if (side == 0) {
        *reinterpret_cast<uint32_t *>(codes + (kept + r) * uint32_t(kDim) + d) = w;
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) codes[(d + j) * P + kept + r] = uint8_t(w >> (8 * j));
      }
    }
  }
}

}  // namespace

hipError_t launch_rope_table(hipStream_t s, const RopeTableArgs &a) {
  const uint64_t n = uint64_t(a.positions) * (a.rot / 2);
  k_rope_table<<<uint32_t((n + 255) / 256), 256, 0, s>>>(a);
  return hipGetLastError();
}

template <int kDim>
static hipError_t norm_rope(hipStream_t s, const NormRopeArgs &a) {
  constexpr uint32_t kLanes = kDim / 4 < 64 ? kDim / 4 : 64;
  const uint64_t rows = uint64_t(a.tokens) * (a.in[0].heads + a.in[1].heads);
  const uint64_t per = 256 / kLanes;
  k_norm_rope<kDim><<<uint32_t((rows + per - 1) / per), 256, 0, s>>>(a);
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
  // a page's values at 32 a thread, 64 where that passes 1,024 threads
  const uint32_t values = a.cache.page * kDim;
  const uint32_t threads = values / 32 > 1024 ? 1024 : values / 32 < 64 ? 64 : values / 32;
  const dim3 grid((a.max_new + a.cache.page - 2) / a.cache.page + 1, 2 * a.cache.heads, a.seqs);
  constexpr int kQ = kDim > 256 ? 2 : 1;
  if (values > 32 * 1024)
    k_kv_append<kDim, 16 / kQ><<<grid, threads, 0, s>>>(a);
  else
    k_kv_append<kDim, 8 / kQ><<<grid, threads, 0, s>>>(a);
  return hipGetLastError();
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
