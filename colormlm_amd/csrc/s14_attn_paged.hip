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
#include "s14_attn_split.hpp"

namespace s14 {
namespace {

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
