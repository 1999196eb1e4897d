// Residual addition, root-mean-square norm of the rows, and their E4M3 codes with
// E8M0 scales, in one pass: a row stays in its threads' registers between the sum
// of its squares and what is written, but for rows of more than 32,768 values, of which
// 43 to 70 registers a thread go to scratch memory and back.  Bound by the bytes
// moved (16,384 rows of 4,096, f32 with a bf16 residual: 604 MB in 105 us, 5.8 TB/s);
// for a few rows by the launch and two trips to memory, the row with its weight and
// the stores (one row: 3.5 us).
#include "s14_attn_rows.hpp"

namespace s14 {
namespace {

struct Octet {
  float v[8];
};
template <bool k16>
__device__ __forceinline__ Octet load_octet(const void *p, uint64_t at) {
  Octet o;
  if constexpr (k16) {
    const uint4 w = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(p) + at);
    const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) o.v[2 * i] = __uint_as_float(x[i] << 16), o.v[2 * i + 1] = __uint_as_float(x[i] & 0xffff0000u);
  } else {
    const Quad a = load_quad<false>(p, at), b = load_quad<false>(p, at + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) o.v[i] = a.v[i], o.v[4 + i] = b.v[i];
  }
  return o;
}
__device__ __forceinline__ void store_octet(const AttnOut &out, uint64_t at, const Octet &o) {
  if (out.bf16) {
    *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(out.p) + at) =
        make_uint4(bf16_pair(o.v[0], o.v[1]), bf16_pair(o.v[2], o.v[3]), bf16_pair(o.v[4], o.v[5]), bf16_pair(o.v[6], o.v[7]));
  } else {
    float4 *to = reinterpret_cast<float4 *>(static_cast<float *>(out.p) + at);
    to[0] = make_float4(o.v[0], o.v[1], o.v[2], o.v[3]);
    to[1] = make_float4(o.v[4], o.v[5], o.v[6], o.v[7]);
  }
}

// kV times eight values a thread, blockDim.x threads a row (whole wavefronts),
// blockDim.y rows a workgroup (of one wavefront each where there are several).
template <bool kX16, bool kR16, int kV>
__global__ __launch_bounds__(1024) void k_add_norm(AddNormArgs a) {
  const uint32_t T = blockDim.x, octets = a.k / 8, row = blockIdx.x * blockDim.y + threadIdx.y;
  if (row >= a.rows) return;  // a wavefront's row; of several wavefronts a row, all of them
  Octet h[kV];
#pragma unroll
  for (int j = 0; j < kV; ++j) {
    const uint32_t i = threadIdx.x + j * T;
    if (i < octets)
      h[j] = load_octet<kX16>(a.x.p, row * a.x.token + 8 * i);
    else
      h[j] = Octet{};
  }
  if (a.residual.p) {
    Octet r[kV];
#pragma unroll
    for (int j = 0; j < kV; ++j) {
      const uint32_t i = threadIdx.x + j * T;
      r[j] = i < octets ? load_octet<kR16>(a.residual.p, row * a.residual.token + 8 * i) : Octet{};
    }
#pragma unroll
    for (int j = 0; j < kV; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) h[j].v[e] += r[j].v[e];
  }
  Octet w[kV];
#pragma unroll
  for (int j = 0; j < kV; ++j) {
    const uint32_t i = threadIdx.x + j * T;
    w[j] = i < octets ? load_octet<false>(a.weight, 8 * i) : Octet{};
  }
  float sum = 0.0f;
#pragma unroll
  for (int j = 0; j < kV; ++j)
#pragma unroll
    for (int e = 0; e < 8; ++e) sum += h[j].v[e] * h[j].v[e];
  sum = lane_sum<64>(sum);
  __shared__ float s_sum[16];
  if (T > 64) {
    if ((threadIdx.x & 63u) == 0) s_sum[threadIdx.x / 64] = sum;
    __syncthreads();  // and the row is read: its place may be written
    sum = 0.0f;
    for (uint32_t k = 0; k < T / 64; ++k) sum += s_sum[k];
  }
  const float f = rsqrtf(sum / float(a.k) + a.eps);
#pragma unroll
  for (int j = 0; j < kV; ++j) {
    const uint32_t i = threadIdx.x + j * T;
    if (i >= octets) continue;  // a scale's lanes together: k is whole groups
    if (a.residual_out.p) store_octet(a.residual_out, row * a.residual_out.token + 8 * i, h[j]);
    Octet y;
#pragma unroll
    for (int e = 0; e < 8; ++e) y.v[e] = h[j].v[e] * f * w[j].v[e];
    if (a.y.p) store_octet(a.y, row * a.y.token + 8 * i, y);
    if (a.group) {
      float amax = 0.0f;  // a NaN is never greater
#pragma unroll
      for (int e = 0; e < 8; ++e) amax = fabsf(y.v[e]) > amax ? fabsf(y.v[e]) : amax;
      amax = fmaxf(amax, dpp_f<0xb1>(0.0f, amax));  // quad_perm [1,0,3,2]
      amax = fmaxf(amax, dpp_f<0x4e>(0.0f, amax));  // quad_perm [2,3,0,1]
      if (a.group >= 64) amax = fmaxf(amax, dpp_f<0x141>(0.0f, amax));   // row_half_mirror
      if (a.group >= 128) amax = fmaxf(amax, dpp_f<0x140>(0.0f, amax));  // row_mirror
      const GroupQuant gq(amax);
      *reinterpret_cast<uint2 *>(a.q + uint64_t(row) * a.k + 8 * i) =
          make_uint2(gq.word(y.v[0], y.v[1], y.v[2], y.v[3]), gq.word(y.v[4], y.v[5], y.v[6], y.v[7]));
      const uint32_t lanes = a.group / 8;
      if (i % lanes == 0) a.scales[uint64_t(row) * (a.k / a.group) + i / lanes] = uint8_t(gq.code);
    }
  }
}

template <int kV>
hipError_t add_norm(hipStream_t s, const AddNormArgs &a, uint32_t threads) {
  const uint32_t per = threads == 64 ? 4 : 1;
  const dim3 grid((a.rows + per - 1) / per), block(threads, per);
  if (a.x.bf16)
    if (a.residual.bf16)
      k_add_norm<true, true, kV><<<grid, block, 0, s>>>(a);
    else
      k_add_norm<true, false, kV><<<grid, block, 0, s>>>(a);
  else if (a.residual.bf16)
    k_add_norm<false, true, kV><<<grid, block, 0, s>>>(a);
  else
    k_add_norm<false, false, kV><<<grid, block, 0, s>>>(a);
  return hipGetLastError();
}

}  // namespace

// As few values a thread as a workgroup's threads allow (us of 1 and of 16,384 rows of
// 4,096 values: eight 3.6 and 152, sixteen 4.4 and 159, a wavefront a row 10.8 and 230;
// 1 and 8,192 of 8,192: eight 4.2 and 167, sixteen 4.5 and 162).  2,048 rows, f32 with a
// bf16 residual: of 16,384 values 61 us (5.0 TB/s), of 32,768 139 (4.4), with the spills
// of 40,960 311 (2.4) and of 65,536 426 (2.8); one row of 65,536 27 us.
hipError_t launch_add_norm(hipStream_t s, const AddNormArgs &a) {
  const uint32_t octets = a.k / 8;
  const auto threads = [&](uint32_t v) { return ((octets + v - 1) / v + 63) / 64 * 64; };
  if (threads(1) <= 1024) return add_norm<1>(s, a, threads(1));
  if (threads(2) <= 1024) return add_norm<2>(s, a, threads(2));
  if (threads(4) <= 1024) return add_norm<4>(s, a, threads(4));
  if (threads(8) <= 1024) return add_norm<8>(s, a, threads(8));
  return hipErrorInvalidValue;
}

}  // namespace s14
