// Attention of new tokens over the paged 4-bit cache (E2M1 codes, E8M0 scales).
//
// Both products run on v_mfma_f32_16x16x32_bf16 with the tokens as the rows:
// S^T = K Q^T, then O^T = V^T P^T, P staying in its lane's registers where a
// wavefront does both (the result layout of the first is the operand layout of
// the second if each 16-token tile t of a step takes the tokens 16 g + 4 t + i,
// i < 4, as its rows 4 g + i).  E2M1 codes become bf16 exactly.  A key's scales
// are of 32 dimensions, which one lane holds: they go into the conversion.  A
// value's scale is of 128 dimensions of one token: in the second product the
// tokens are what is summed over, so the scale goes onto the token's weight, one
// multiplication for 128 dimensions, exact and before the weight's rounding.
//
// The formats follow from that.  K codes lie [slot][dim], two dimensions a byte:
// a lane's 16 bytes are the 32 dimensions of a scale.  V codes lie in units of 16
// bytes, 16 slots of dimension d and of d + 16, two slots a byte: a unit is what a
// lane multiplies of two 16-dimension tiles, and 64 lanes' units lie in a row.
//
// A row is a (token, query head of the key head) pair: the group's heads share
// the K and V that are read.  Which kernel takes how many rows, how long
// sequences are cut and joined: s14_attn_plan.h, s14_attn_split.hpp.
#include "s14_attn_split.hpp"

namespace s14 {
namespace {

// Eight E2M1 codes (a word, the low half of each byte first) times a scale as
// bf16.  Of the scale the conversion takes the exponent's bits alone (looked at
// for several signs and mantissas): a byte shifted there needs no mask.  The
// exponent 255 gives NaN for every code.
__device__ __forceinline__ bf16x8 e2m1_bf16(uint32_t w, float scale = 1.0f) {
  const u32x4 v = {__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0)),
                   __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1)),
                   __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2)),
                   __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3))};
  return __builtin_bit_cast(bf16x8, v);
}

// Byte i of a word of E8M0 codes where a float has its exponent, other bits around it.
__device__ __forceinline__ float rough_scale(uint32_t w, int i) {
  return __uint_as_float(i < 3 ? w << (23 - 8 * i) : w >> 1);
}
// And alone: 2^(code - 127), NaN for 255, by the conversion of an 8-bit one.
__device__ __forceinline__ float clean_scale(uint32_t w, int i) {
  return __builtin_amdgcn_cvt_scalef32_f32_fp8(0x38, rough_scale(w, i), 0);
}

// A slot's place among a block's key scales: of each 16 slots the 4 x 4 transposed,
// so that the four tiles' scales of a lane are one word.
__device__ __forceinline__ uint32_t scale_slot(uint32_t slot) { return (slot & ~15u) + 4 * (slot & 3u) + ((slot >> 2) & 3u); }

// A value scale that is NaN.  A token that a row sees makes it NaN, however small its
// weight is: else the order of the tokens and the cuts would decide whether the weight
// was 0 when the scale came.  A masked token's scale may be anything.  Either its scale
// is selected to 0 where a step has masked tokens (k_paged4 with one row tile, wide
// heads), and the product is an ordinary one.  Or, where that takes registers that the
// step has not (us, start / selects / this: 8 tokens of 40,000 21.0 / 22.5 / 21.2; 32
// sequences of 8 of 4,000 54.2 / 61.8 / 54.8; but 16 of one token of up to 8,192, one
// row tile, 24.7 / 24.8 / 25.9), the product is 0 where the weight is 0 (the
// instruction's own rule), steps with a NaN among their scales are remembered, and
// after the loop the rows look through those.
extern "C" __device__ float s14_mul_zero(float a, float b) __asm("llvm.amdgcn.fmul.legacy");
template <bool kSelect>
__device__ __forceinline__ float weighted(float weight, float scale) {
  return kSelect ? weight * scale : s14_mul_zero(weight, scale);
}

// Bit c: of the tokens first .. last + 63 (steps of 64) one that the row sees has a NaN
// scale of its 128 dimensions c.  By a whole wavefront, a token a lane.
template <int B>
__device__ uint32_t nan_parts(const PagedArgs &a, const Pages &pages, uint32_t head, int32_t first, int32_t last,
                              const Visible &see) {
  const uint32_t P = a.cache.page;
  uint32_t hit = 0;
  for (int32_t b = first; b <= last; b += 64) {
    const int32_t tok = b + int32_t(threadIdx.x & 63u);
    bool bad = false;  // (who loaded the step has said so)
    const uint64_t at = uint64_t(pages.checked(pages.id(tok), bad)) * a.cache.heads + head;
    for (int c = 0; c < B; ++c)
      for (uint64_t m = __ballot(a.cache.vs[(at * B + c) * P + (uint32_t(tok) & (P - 1))] == 255); m; m &= m - 1)
        if (see(b + __builtin_ctzll(m))) hit |= 1u << c;
  }
  return hit;
}

// The dimensions of `parts` of a row become NaN.
template <int DT>
__device__ __forceinline__ void spoil(f32x4 (&o)[DT], uint32_t parts) {
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int i = 0; i < 4; ++i) o[dt][i] = parts >> (dt / 8) & 1u ? __uint_as_float(0x7fc00000u) : o[dt][i];
}

// Scales above 0: a masked score times it stays -inf.
__device__ __forceinline__ float score_scale(float scale) { return fmaxf(scale * kLog2e, 0x1p-126f); }

// Up to 16 NT rows: the four wavefronts take steps of 64 tokens in turn and join
// through LDS.  Bound by the cache's bytes: 96 sequences of 2,048 tokens, 8 key heads
// of 128, 40.5 us, 5.2 TB/s (a large read alone takes 5.7); 128 of up to 8,192 85 to
// 90 us, 4.5 TB/s, by how their lengths fall on the compute units.  A fourth
// wavefront a SIMD spills (128 us); with two row tiles eight wavefronts are no faster
// (8 tokens of 40,000: 18.6 us, 19.8).
template <int D, int NT>
__global__ __launch_bounds__(256, D * NT <= 64 ? 4 : D * NT <= 128 ? 3 : 2) void k_paged4(PagedArgs a, PagedPlan p, float *part) {
  constexpr int T = 4;                       // 16-token tiles a step
  constexpr int H = D / 32;                  // words of K codes a lane holds of a token, products of a tile
  constexpr int B = D < 128 ? 1 : D / 128;   // key scales of those, and value scales of a token
  constexpr int U = D / 32, DT = D / 16;     // units of V a lane holds, 16-dimension tiles of O
  constexpr bool kSelect = NT == 1;
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
  bf16x8 q[NT][H];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const uint32_t r = row0 + 16 * nt + n;
    const uint32_t rr = r < sp.rows ? r : sp.rows - 1;
    see[nt] = Visible(sp.pos0 + int32_t(rr / group), a.window);
    const uint16_t *row = a.q + uint64_t(sp.first + rr / group) * a.q_token +
                          uint64_t(head * group + rr % group) * a.q_head;
#pragma unroll
    for (int h = 0; h < H; ++h)
      q[nt][h] = *reinterpret_cast<const bf16x8 *>(row + (D == 64 ? 16 * g + 8 * h : 128 * (h / 4) + 32 * g + 8 * (h % 4)));
  }
  const int32_t pos_lo = sp.pos0 + int32_t(row0 / group);
  const int32_t pos_hi = sp.hi - 1;

  f32x4 o[NT][DT] = {};
  float m[NT], sum[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) m[nt] = -INFINITY, sum[nt] = 0.0f;
  bool bad = false;
  const float scale = score_scale(a.scale);
  const uint64_t page_bytes = uint64_t(P) * (D / 2);

  // A step's operands, loaded one step ahead (K as soon as the first product has
  // read the step before, V after the second), their pages' ids another step
  // ahead.
  uint32_t kk[T][H], ksc[B];
  uint4 vv[U], vsc[B];
  int32_t idk = 0, idv = 0;  // of the next step
  auto load_ids = [&](int32_t b, int32_t &k, int32_t &v) {
    k = pages.id(b + 16 * int32_t(n / 4));
    v = pages.id(b + 16 * int32_t(g));
  };
  auto load_k = [&](int32_t b) {
    const uint32_t slot = uint32_t(b + 16 * int32_t(n / 4)) & (P - 1);
    const uint64_t at = uint64_t(pages.checked(idk, bad)) * kvh + head;
    const uint8_t *sc = a.cache.ks + at * (H * P) + (D == 64 ? g / 2 : g) * P + slot + 4 * (n & 3u);
#pragma unroll
    for (int c = 0; c < B; ++c) ksc[c] = *reinterpret_cast<const uint32_t *>(sc + 4 * c * P);
    const uint8_t *kp = a.cache.k + at * page_bytes + (slot + (n & 3u)) * uint32_t(D / 2) + (D == 64 ? 8 : 16) * g;
#pragma unroll
    for (int t = 0; t < T; ++t) {
      if constexpr (D == 64) {
        const uint2 x = *reinterpret_cast<const uint2 *>(kp + 4 * t * (D / 2));
        kk[t][0] = x.x, kk[t][1] = x.y;
      } else {
#pragma unroll
        for (int c = 0; c < B; ++c) {
          const uint4 x = *reinterpret_cast<const uint4 *>(kp + 4 * t * (D / 2) + 64 * c);
          kk[t][4 * c] = x.x, kk[t][4 * c + 1] = x.y, kk[t][4 * c + 2] = x.z, kk[t][4 * c + 3] = x.w;
        }
      }
    }
  };
  auto load_v = [&](int32_t b) {
    const uint32_t slot = uint32_t(b + 16 * int32_t(g)) & (P - 1);
    const uint64_t at = uint64_t(pages.checked(idv, bad)) * kvh + head;
    const uint8_t *sc = a.cache.vs + at * (B * P) + slot;
#pragma unroll
    for (int c = 0; c < B; ++c) vsc[c] = *reinterpret_cast<const uint4 *>(sc + c * P);
    const uint8_t *vp = a.cache.v + at * page_bytes + (slot + n) * 16;
#pragma unroll
    for (int u = 0; u < U; ++u) vv[u] = *reinterpret_cast<const uint4 *>(vp + u * P * 16);
  };
  int32_t nan_first = INT_MAX, nan_last = -1;  // of the steps with a NaN value scale
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
      for (int h = 0; h < H; ++h) asm volatile("; a step's operands" : "+v"(q[nt][h]));
  } else {  // on this way to the loop too; in other words, or both would be done where the ways meet
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int h = 0; h < H; ++h) asm volatile("; no step" : "+v"(q[nt][h]));
  }

  for (; b < end; b += kStride) {
    const int32_t tv = b + 4 * T * int32_t(g);
    // past the last step that step's again: a load behind a branch makes every
    // later wait one for all loads
    const int32_t next = min(b + kStride, last);
    int32_t idk2, idv2;  // ahead of the K and V loads below
    load_ids(min(b + 2 * kStride, last), idk2, idv2);
    f32x4 s[NT][T];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int t = 0; t < T; ++t) s[nt][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int t = 0; t < T; ++t)
#pragma unroll
      for (int h = 0; h < H; ++h) {
        const bf16x8 k = e2m1_bf16(kk[t][h], rough_scale(ksc[h / 4], t));
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) s[nt][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k, q[nt][h], s[nt][t], 0, 0, 0);
      }
    load_k(next);
    const bool partial = b + 16 * T - 1 > pos_lo || (a.window && int64_t(b) <= int64_t(pos_hi) - a.window);
    bf16x8 pb[B][NT][T / 2];
    uint32_t most = 0;  // the value scales' bits
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float x[4 * T], f[B][4 * T];
#pragma unroll
      for (int i = 0; i < 4 * T; ++i) {
        x[i] = s[nt][i / 4][i % 4];
#pragma unroll
        for (int c = 0; c < B; ++c)
          f[c][i] = clean_scale(i < 4 ? vsc[c].x : i < 8 ? vsc[c].y : i < 12 ? vsc[c].z : vsc[c].w, i % 4);
      }
      if (partial) {
        keep_branch();
#pragma unroll
        for (int i = 0; i < 4 * T; ++i) {
          const bool in = see[nt](tv + i);
          x[i] = in ? x[i] : -INFINITY;
          if constexpr (kSelect) {
#pragma unroll
            for (int c = 0; c < B; ++c) f[c][i] = in ? f[c][i] : 0.0f;
          }
        }
      }
      float top = x[0];
#pragma unroll
      for (int i = 1; i < 4 * T; ++i) top = fmaxf(top, x[i]);
      top = fmaxf(m[nt], max_lane16(top) * scale);
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
      u32x4 w[B][T / 2];
#pragma unroll
      for (int t = 0; t < T; ++t) {
        float e[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[4 * t + i], scale, -at));
          sum[nt] += e[i];
        }
        // rounded to bf16, half a step of each weight: the matrix operand's type
#pragma unroll
        for (int c = 0; c < B; ++c) {
          const float *v = &f[c][4 * t];
          if (!kSelect && nt == 0) {
            most = max(most, max(__float_as_uint(v[0]), __float_as_uint(v[1])));
            most = max(most, max(__float_as_uint(v[2]), __float_as_uint(v[3])));
          }
          w[c][t / 2][2 * (t & 1)] = bf16_pair(weighted<kSelect>(e[0], v[0]), weighted<kSelect>(e[1], v[1]));
          w[c][t / 2][2 * (t & 1) + 1] = bf16_pair(weighted<kSelect>(e[2], v[2]), weighted<kSelect>(e[3], v[3]));
        }
      }
#pragma unroll
      for (int c = 0; c < B; ++c)
#pragma unroll
        for (int u = 0; u < T / 2; ++u) pb[c][nt][u] = __builtin_bit_cast(bf16x8, w[c][u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t word[2][2] = {{vv[u].x, vv[u].y}, {vv[u].z, vv[u].w}};
#pragma unroll
      for (int d = 0; d < 2; ++d)
#pragma unroll
        for (int h = 0; h < T / 2; ++h) {
          const bf16x8 v = e2m1_bf16(word[d][h]);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            o[nt][2 * u + d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, pb[u / 4][nt][h], o[nt][2 * u + d], 0, 0, 0);
        }
    }
    if (!kSelect && __any(most > 0x7f800000u)) nan_first = min(nan_first, b), nan_last = b;
    load_v(next);
    idk = idk2, idv = idv2;
  }
  if (!kSelect && nan_last >= 0) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) spoil(o[nt], nan_parts<B>(a, pages, head, nan_first, nan_last, see[nt]));
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

// Heads of 512 (one wide key head for many query heads).  Here no byte of the
// cache goes to two wavefronts: of a step's 64 tokens a wavefront takes 16 for the
// first product, all dimensions of them, against Q from LDS; the wavefronts'
// maxima meet there, each weights its own scores, once for each of the four value
// scales of a token, and P goes through LDS for the second product, of which a
// wavefront takes the 128 dimensions of one scale, all tokens.  64 sequences of 4,000
// tokens, 64 heads, 68 us, 495 TFLOP/s; issue bounds it, 480 instructions of the
// vector unit a step beside 1,024 clocks of the matrix unit, and for few sequences
// the partial results (33 MB of one of 4,000 tokens).  Codes two steps ahead are no
// faster (256 sequences of 1,024: 59.6 us, 62.8).
template <int NT>
__global__ __launch_bounds__(256, 2) void k_paged4_wide(PagedArgs a, PagedPlan p, float *part) {
  constexpr int D = 512, C = 4, DT = 8;
  const uint32_t kvh = a.cache.heads, group = a.heads / kvh;
  const Item it = item_of(a, p, kvh);
  const uint32_t tile = it.tile, head = it.head, seq = it.seq, chunk = it.chunk;
  const uint32_t row0 = tile * 16 * NT;
  const Span sp = balanced_span<paged_balances(D, NT)>(a, p, seq, row0, part);
  if (row0 >= sp.rows || (chunk && chunk >= sp.chunks)) return;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), l = threadIdx.x & 63u, n = l & 15u, g = l >> 4;
  const uint32_t P = a.cache.page, d0 = 128 * wave;
  const uint32_t shift = __builtin_ctz(P);
  const Pages pages{a.page_table + uint64_t(seq) * a.table_width, sp.seen, sp.len - 1, a.cache.pages, shift};
  const int32_t begin = sp.lo + int32_t(chunk * sp.chunk);
  const int32_t end = paged_end(begin, sp.hi, sp.chunk);
  Visible see[NT];

  __shared__ bf16x8 s_q[NT][4 * C][64];    // the first product's operands
  __shared__ bf16x8 s_p[4][NT][2][64];     // the second's, with each value scale
  __shared__ float s_m[4][NT][16], s_l[4][NT][16];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const uint32_t r = row0 + 16 * nt + n;
    const uint32_t rr = r < sp.rows ? r : sp.rows - 1;
    see[nt] = Visible(sp.pos0 + int32_t(rr / group), a.window);
    const uint16_t *row = a.q + uint64_t(sp.first + rr / group) * a.q_token +
                          uint64_t(head * group + rr % group) * a.q_head;
#pragma unroll
    for (int h = 0; h < 4; ++h)
      s_q[nt][4 * wave + h][l] = *reinterpret_cast<const bf16x8 *>(row + d0 + 32 * g + 8 * h);
  }
  const int32_t pos_lo = sp.pos0 + int32_t(row0 / group), pos_hi = sp.hi - 1;

  f32x4 o[NT][DT] = {};
  float m[NT], sum[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) m[nt] = -INFINITY, sum[nt] = 0.0f;
  bool bad = false;
  const float scale = a.scale * kLog2e;
  const uint64_t page_bytes = uint64_t(P) * (D / 2);

  // K: 32 dimensions of token 16 wave + n four times, and the value scales of the
  // tokens 16 wave + 4 g ..; V: 16 tokens from 16 g of dimensions d0 + 32 u + n and
  // 16 further.  (The K tokens' page is one for the wavefront, but not said so: a
  // scalar id would be waited for where it is loaded, with all loads before it.)
  constexpr int32_t kStep = 64;
  const uint32_t k_tok = threadIdx.x / 64 * 16;
  uint4 kk[C], vv[C];
  uint8_t ksc[C];  // (as loaded: widened where they are used, not while in flight)
  uint32_t vsc[C];
  int32_t idk = 0, idv = 0;  // of the next step
  auto load_ids = [&](int32_t b, int32_t &k, int32_t &v) {
    k = pages.id(b + int32_t(k_tok));
    v = pages.id(b + 16 * int32_t(g));
  };
  auto load_k = [&](int32_t b) {
    const uint64_t at = uint64_t(pages.checked(idk, bad)) * kvh + head;
    const uint32_t slot = uint32_t(b + int32_t(k_tok)) & (P - 1);
    const uint8_t *ks = a.cache.ks + at * (16 * P) + g * P + scale_slot(slot + n);
    const uint8_t *vs = a.cache.vs + at * (4 * P) + slot + 4 * g;
#pragma unroll
    for (int c = 0; c < C; ++c) ksc[c] = ks[4 * c * P];
#pragma unroll
    for (int c = 0; c < C; ++c) vsc[c] = *reinterpret_cast<const uint32_t *>(vs + c * P);
    const uint8_t *kp = a.cache.k + at * page_bytes + (slot + n) * uint32_t(D / 2) + 16 * g;
#pragma unroll
    for (int c = 0; c < C; ++c) kk[c] = *reinterpret_cast<const uint4 *>(kp + 64 * c);
  };
  auto load_v = [&](int32_t b) {
    const uint32_t slot = uint32_t(b + 16 * int32_t(g)) & (P - 1);
    const uint8_t *vp = a.cache.v + (uint64_t(pages.checked(idv, bad)) * kvh + head) * page_bytes +
                        (4 * wave * P + slot + n) * 16;
#pragma unroll
    for (int u = 0; u < C; ++u) vv[u] = *reinterpret_cast<const uint4 *>(vp + u * P * 16);
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
    const int32_t tk = b + int32_t(k_tok) + 4 * int32_t(g);
    // past the last step that step's again: a load behind a branch makes every
    // later wait one for all loads
    const int32_t next = min(b + kStep, last);
    int32_t idk2, idv2;  // ahead of the K and V loads below
    load_ids(min(b + 2 * kStep, last), idk2, idv2);
    const bool partial = b + kStep - 1 > pos_lo || (a.window && int64_t(b) <= int64_t(pos_hi) - a.window);
    f32x4 s[NT][2] = {};
    // Q two words ahead of its use (read right before it, as the compiler leaves it: 68 -> 70 us)
    bf16x8 qa[4][NT];
    const auto read_q = [&](int w) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) qa[w & 3][nt] = s_q[nt][w][l];
    };
    read_q(0), read_q(1);
#pragma unroll
    for (int w = 0; w < 4 * C; ++w) {
      if (w + 2 < 4 * C) read_q(w + 2);
      const uint32_t word = w % 4 == 0 ? kk[w / 4].x : w % 4 == 1 ? kk[w / 4].y : w % 4 == 2 ? kk[w / 4].z : kk[w / 4].w;
      const bf16x8 k = e2m1_bf16(word, __uint_as_float(uint32_t(ksc[w / 4]) << 23));
      __builtin_amdgcn_sched_barrier(0x1 | 0x2 | 0x4 | 0x8);  // LDS reads stay ahead
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) s[nt][w & 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k, qa[w & 3][nt], s[nt][w & 1], 0, 0, 0);
    }
    float f[C][4];
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) f[c][i] = clean_scale(vsc[c], i);
    load_k(next);
    float x[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int i = 0; i < 4; ++i) x[nt][i] = (s[nt][0][i] + s[nt][1][i]) * scale;
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
#pragma unroll
      for (int c = 0; c < C; ++c) {
        float w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = weighted<true>(e[i], f[c][i]);
        if (partial) {
          keep_branch();
#pragma unroll
          for (int i = 0; i < 4; ++i) w[i] = see[nt](tk + i) ? w[i] : 0.0f;
        }
        // half a step of each weight: the matrix operand's type
        reinterpret_cast<uint2 *>(&s_p[c][nt][g / 2][16 * wave + n])[g & 1] =
            make_uint2(bf16_pair(w[0], w[1]), bf16_pair(w[2], w[3]));
      }
    }
    __syncthreads();
    bf16x8 pb[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) pb[nt][0] = s_p[wave][nt][0][l], pb[nt][1] = s_p[wave][nt][1][l];
#pragma unroll
    for (int u = 0; u < C; ++u) {
      const uint32_t word[2][2] = {{vv[u].x, vv[u].y}, {vv[u].z, vv[u].w}};
#pragma unroll
      for (int d = 0; d < 2; ++d)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const bf16x8 v = e2m1_bf16(word[d][h]);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            o[nt][2 * u + d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, pb[nt][h], o[nt][2 * u + d], 0, 0, 0);
        }
    }
    load_v(next);
    idk = idk2, idv = idv2;
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
// from LDS, where the workgroup has put them as bf16, the keys with their scales,
// once for all its rows; the values' scales lie beside them.  A step of 128 rows takes
// 1.2 us a compute unit (880 TFLOP/s of a running one); what 8 sequences of 64 new of
// 3,000 tokens take beyond that, 52 us in all, is the start, and 35 MB of partial
// results written and read.  Tried without gain there: a step's products between the
// next one's weights with two buffers (58 us), eight wavefronts that halve the partial
// results (59), 64 rows a workgroup (54).
template <int D, int NT, int RW>
__global__ __launch_bounds__(256, D * NT > 128 ? 2 : D * NT < 128 ? 4 : RW == 2 ? 4 : 3) void k_paged4_rows(PagedArgs a, PagedPlan p, float *part) {
  constexpr int TK = D <= 128 ? 64 : 32;  // tokens a step
  constexpr int TW = 4 / RW;              // wavefronts that share a row tile's tokens
  constexpr int U = TK / 32 / TW, T = 2 * U, DT = D / 16, C = D / 32;
  constexpr int B = D < 128 ? 1 : D / 128;  // value scales of a token
  constexpr int W = D * TK / 2048;          // words of K, and of V, a thread loads: 8 codes each
  static_assert(W == 2 || W == 4, "a thread's codes are one load");
  const uint32_t kvh = a.cache.heads, group = a.heads / kvh;
  const Item it = item_of(a, p, kvh);
  const uint32_t tile = it.tile, head = it.head, seq = it.seq, chunk = it.chunk;
  const uint32_t row0 = tile * 16 * NT * RW;
  const Span sp = balanced_span<paged_balances(D, NT * RW)>(a, p, seq, row0, part);
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
  __shared__ f32x4 s_vs[B * TK / 4];
  __shared__ uint32_t s_flags;
  __shared__ int32_t s_first, s_last;  // of the steps with a NaN value scale
  if (tid == 0) s_flags = 0, s_first = INT_MAX, s_last = -1;

  f32x4 o[NT][DT] = {};
  float m[NT], sum[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) m[nt] = -INFINITY, sum[nt] = 0.0f;
  bool bad = false;
  const float scale = score_scale(a.scale);
  const uint64_t page_bytes = uint64_t(P) * (D / 2);

  // A step's codes: a thread's K are 8 W dimensions of one token, its V 16 tokens
  // of W / 2 dimensions 16 apart; threads below B TK have a value scale each.
  // Loaded two steps ahead of their use, turned into bf16 one ahead; their pages'
  // ids are loaded another step ahead.
  constexpr uint32_t kTokPieces = D / (8 * W), kHalves = 4 / W;
  const uint32_t k_tok = tid / kTokPieces, k_dim = tid % kTokPieces * (8 * W);
  const uint32_t v_unit = tid / kHalves, v_half = tid % kHalves;
  const uint32_t v_tok = v_unit / 16 % (TK / 16) * 16, v_dim = v_unit / (16 * (TK / 16)) * 32 + v_unit % 16 + 16 * v_half;
  const uint32_t s_tok = tid % TK, s_part = tid / TK;
  uint32_t kk[W], vv[W];
  uint8_t ksc = 0, vsc = 0;
  int32_t idk = 0, idv = 0, ids = 0;
  auto load_ids = [&](int32_t b) {
    idk = pages.id(b + int32_t(k_tok));
    idv = pages.id(b + int32_t(v_tok));
    ids = pages.id(b + int32_t(s_tok));
  };
  const auto load_words = [&](uint32_t *to, const uint8_t *from) {
    if constexpr (W == 2) {
      const uint2 x = *reinterpret_cast<const uint2 *>(from);
      to[0] = x.x, to[1] = x.y;
    } else {
      const uint4 x = *reinterpret_cast<const uint4 *>(from);
      to[0] = x.x, to[1] = x.y, to[2] = x.z, to[3] = x.w;
    }
  };
  auto load = [&](int32_t b) {
    const uint32_t slot = uint32_t(b + int32_t(k_tok)) & (P - 1), v_slot = uint32_t(b + int32_t(v_tok)) & (P - 1);
    const uint64_t at = uint64_t(pages.checked(idk, bad)) * kvh + head;
    ksc = a.cache.ks[at * (D / 32 * P) + k_dim / 32 * P + scale_slot(slot)];
    load_words(kk, a.cache.k + at * page_bytes + slot * uint32_t(D / 2) + k_dim / 2);
    const uint64_t vat = uint64_t(pages.checked(idv, bad)) * kvh + head;
    load_words(vv, a.cache.v + vat * page_bytes + (v_dim / 32 * P + v_slot + v_dim % 16) * 16 + 8 * v_half);
    const uint64_t sat = uint64_t(pages.checked(ids, bad)) * kvh + head;
    vsc = a.cache.vs[(sat * B + (s_part < B ? s_part : 0u)) * P + (uint32_t(b + int32_t(s_tok)) & (P - 1))];
  };
  auto stage = [&](int32_t b, u32x4 *to) {
    const float ks = __uint_as_float(uint32_t(ksc) << 23);
#pragma unroll
    for (int w = 0; w < W; ++w)
      to[k_tok * (D / 8) + ((k_dim / 8 + w) ^ turn_k<D>(k_tok))] = __builtin_bit_cast(u32x4, e2m1_bf16(kk[w], ks));
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const uint32_t dim = v_dim + 16 * (w / 2);
      to[kPieces + dim * (TK / 8) + ((v_tok / 8 + w % 2) ^ turn_v<TK>(dim))] = __builtin_bit_cast(u32x4, e2m1_bf16(vv[w]));
    }
    if (tid < B * TK) reinterpret_cast<float *>(s_vs)[tid] = clean_scale(vsc, 0);
    if (vsc == 255) atomicMin(&s_first, b), atomicMax(&s_last, b);
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
    __syncthreads();
    stage(begin, s_rows);
    if (begin + TK < end) load(begin + TK);
    if (begin + 2 * TK < end) load_ids(begin + 2 * TK);
  }
  __syncthreads();

  for (int32_t b = begin; b < end; b += TK) {
    const u32x4 *sk = s_rows, *sv = sk + kPieces;
    bf16x8 pb[B][NT][U];
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
          float e[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            e[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[8 * u + j], scale, -at));
            sum[nt] += e[j];
          }
#pragma unroll
          for (int c = 0; c < B; ++c) {
            const f32x4 f0 = s_vs[c * (TK / 4) + 8 * (u0 + u) + 2 * g], f1 = s_vs[c * (TK / 4) + 8 * (u0 + u) + 2 * g + 1];
            float y[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] = weighted<false>(e[j], j < 4 ? f0[j] : f1[j - 4]);
            u32x4 w;
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = bf16_pair(y[2 * j], y[2 * j + 1]);  // half a step of each weight: the matrix operand's type
            pb[c][nt][u] = __builtin_bit_cast(bf16x8, w);
          }
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
          for (int nt = 0; nt < NT; ++nt) o[nt][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, pb[dt / 8][nt][u], o[nt][dt], 0, 0, 0);
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

  // the lane's place again from the thread's number, not kept over the loop
  uint32_t lane = tid & 63u;
  asm volatile("" : "+v"(lane));
  const uint32_t group4 = lane >> 4;
  if (bad) atomicOr(&s_flags, 1u);
  __syncthreads();
  const uint32_t flags = s_flags;
  if (active && s_last >= 0) {
    const int32_t first = __builtin_amdgcn_readfirstlane(s_first) & ~63, last = __builtin_amdgcn_readfirstlane(s_last);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const uint32_t r = mine + 16 * nt + lane % 16, rr = r < sp.rows ? r : sp.rows - 1;
      spoil(o[nt], nan_parts<B>(a, pages, head, first, last, Visible(sp.pos0 + int32_t(rr / group), a.window)));
    }
  }
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
  if (const uint32_t status = sp.wrong | (flags ? kStatusBadCachePage : 0u); status && tid == 0) atomicOr(a.status, status);
  const uint32_t floats = p.rec_rows * kRecord<D>;
  const PartStore<false> store(part + record_of(a, p, it, kvh) * floats, floats, 0);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const float total = flags ? __uint_as_float(0x7fc00000u) : sum_lane16(sum[nt]);
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

template <int D>
hipError_t launch_dim(hipStream_t s, const PagedArgs &a, const PagedPlan &p, float *part) {
  if constexpr (D == 512) {
    if (p.row_tiles == 2) return launch<D, paged_balances(D, 2)>(s, a, p, part, k_paged4_wide<2>);
    return launch<D>(s, a, p, part, k_paged4_wide<1>);
  } else {
    if constexpr (D <= 128) {
      if (p.row_tiles == 8) return launch<D, paged_balances(D, 8)>(s, a, p, part, k_paged4_rows<D, 2, 4>);
      if (p.row_tiles == 2 && p.staged) return launch<D>(s, a, p, part, k_paged4_rows<D, 1, 2>);
      if (p.row_tiles == 2) return launch<D>(s, a, p, part, k_paged4<D, 2>);
    }
    if (p.row_tiles == 4) return launch<D>(s, a, p, part, k_paged4_rows<D, 1, 4>);
    return launch<D>(s, a, p, part, k_paged4<D, 1>);
  }
}

}  // namespace

hipError_t launch_paged4_attention(hipStream_t s, const PagedArgs &a, const PagedPlan &p, float *part) {
  switch (a.cache.dim) {
    case 64: return launch_dim<64>(s, a, p, part);
    case 128: return launch_dim<128>(s, a, p, part);
    case 256: return launch_dim<256>(s, a, p, part);
    case 512: return launch_dim<512>(s, a, p, part);
  }
  return hipErrorInvalidValue;
}

}  // namespace s14
