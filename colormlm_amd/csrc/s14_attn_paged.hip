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
// scores (K) and the weights (V), and are one per lane, since the 4 T tokens
// of a lane group lie in one page.
//
// A row is a (token, query head of the key head) pair: the group's heads
// share the K and V that a wavefront loads.  The four wavefronts of a
// workgroup take steps of 16 T tokens in turn and join through LDS; a long
// sequence is cut into chunks of workgroups whose partial results a second
// launch joins.
#include "s14_attn.hpp"
#include "s14_attn_util.hpp"
#include "s14_device.hpp"

namespace s14 {
namespace {

// What a row tile of a sequence reads: tokens lo .. hi - 1 in chunks of
// `chunk` (a multiple of 64, as lo is).
struct Span {
  int64_t first, rows;  // first packed token; (token, head) rows of the sequence
  int32_t len, pos0, lo, hi;
  uint32_t chunk, chunks;
};

__device__ __forceinline__ Span paged_span(const PagedArgs &a, const PagedPlan &p, uint32_t seq, uint32_t row0) {
  Span s;
  const uint32_t group = a.heads / a.cache.heads;
  s.first = clamp_row(a.cu[seq], a.tokens);
  const int64_t n = clamp_row(a.cu[seq + 1], a.tokens) - s.first;
  s.rows = n > 0 ? n * group : 0;
  const int64_t room = int64_t(a.table_width) * a.cache.page;
  const int64_t len = a.len[seq] < 0 ? 0 : a.len[seq];
  s.len = int32_t(len < room ? len : room);
  s.pos0 = int32_t(s.len - n);
  const int64_t last = (row0 + 16 * p.row_tiles < s.rows ? row0 + 16 * p.row_tiles : s.rows) - 1;
  const int32_t first_pos = s.pos0 + int32_t(row0 / group), last_pos = s.pos0 + int32_t(last / group);
  s.hi = last_pos + 1 < 0 ? 0 : last_pos + 1;
  int64_t lo = a.window ? int64_t(first_pos) - a.window + 1 : 0;
  s.lo = int32_t(lo < 0 ? 0 : lo) & ~63;
  const uint32_t span = s.hi > s.lo ? s.hi - s.lo : 0;
  // a sequence longer than the launch was planned for: larger chunks
  const uint32_t least = ((span + p.chunks - 1) / p.chunks + 63u) & ~63u;
  s.chunk = p.chunk > least ? p.chunk : least;
  s.chunks = (span + s.chunk - 1) / s.chunk;
  return s;
}

__device__ __forceinline__ void store_out(const AttnOut &o, uint64_t at, float a, float b, float c, float d) {
  if (o.bf16)
    *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(o.p) + at) = make_uint2(bf16_pair(a, b), bf16_pair(c, d));
  else
    *reinterpret_cast<float4 *>(static_cast<float *>(o.p) + at) = make_float4(a, b, c, d);
}

// The page of token group `tok` (held inside the sequence): its id, or -1.
__device__ __forceinline__ int32_t page_of(const PagedArgs &a, const int32_t *table, int32_t tok, int32_t len,
                                           bool &bad) {
  const uint32_t t = uint32_t(tok < len ? tok : len - 1);
  int32_t id = table[t / a.cache.page];
  if (uint32_t(id) >= a.cache.pages) bad = true, id = 0;
  return id;
}

template <int D, int NT, int T>
__global__ __launch_bounds__(256) void k_paged_attention(PagedArgs a, PagedPlan p, float *part) {
  constexpr int C = D / 64;   // 16-byte pieces of a K row a lane holds
  constexpr int DT = D / 16;  // 16-dimension tiles of O
  constexpr int W = T;        // 32-bit words of V codes a lane holds of one dimension
  const uint32_t kvh = a.cache.heads, group = a.heads / kvh;
  // row tiles are the slowest index: those that read the same pages are a
  // multiple of `items` apart
  const uint32_t items = kvh * p.chunks * a.seqs, tile = blockIdx.x / items, item = blockIdx.x % items;
  const uint32_t head = item % kvh, chunk = item / kvh % p.chunks, seq = item / kvh / p.chunks;
  const uint32_t row0 = tile * 16 * NT;
  const Span sp = paged_span(a, p, seq, row0);
  if (int64_t(row0) >= sp.rows || (chunk && chunk >= sp.chunks)) return;
  const uint32_t wave = threadIdx.x / 64, l = threadIdx.x & 63u, n = l & 15u, g = l >> 4;
  const uint32_t P = a.cache.page;
  const int32_t *table = a.page_table + uint64_t(seq) * a.table_width;
  const int32_t begin = sp.lo + int32_t(chunk * sp.chunk);
  const int32_t end = min(sp.hi, begin + int32_t(sp.chunk));

  // each lane's row of every tile: its position, and Q in the operand layout
  Visible see[NT];
  bf16x8 q[NT][2 * C];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int64_t r = int64_t(row0) + 16 * nt + n;
    const int64_t rr = r < sp.rows ? r : sp.rows - 1;
    see[nt] = Visible(sp.pos0 + int32_t(rr / group), a.window);
    const uint16_t *row = a.q + uint64_t(sp.first + rr / group) * a.q_token +
                          uint64_t(head * group + uint32_t(rr % group)) * a.q_head;
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
  bool bad = false;
  const float scale = a.scale * kLog2e;
  const uint64_t page_bytes = uint64_t(P) * D;

  for (int32_t b = begin + 16 * T * int32_t(wave); b < end; b += 4 * 16 * T) {
    const int32_t tk = b + 4 * T * int32_t(n / 4), tv = b + 4 * T * int32_t(g);
    const int32_t idk = page_of(a, table, tk, sp.len, bad), idv = page_of(a, table, tv, sp.len, bad);
    const uint8_t *kp = a.cache.k + (uint64_t(idk) * kvh + head) * page_bytes +
                        (uint32_t(tk) % P + (n & 3u)) * uint32_t(D) + 16 * g;
    const uint8_t *vp = a.cache.v + (uint64_t(idv) * kvh + head) * page_bytes + n * P + uint32_t(tv) % P;
    uint4 kk[T][C];
#pragma unroll
    for (int t = 0; t < T; ++t)
#pragma unroll
      for (int c = 0; c < C; ++c) kk[t][c] = *reinterpret_cast<const uint4 *>(kp + 4 * t * D + 64 * c);
    uint32_t vv[DT][W];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      if constexpr (T == 4) {
        const uint4 x = *reinterpret_cast<const uint4 *>(vp + 16 * dt * P);
        vv[dt][0] = x.x, vv[dt][1] = x.y, vv[dt][2] = x.z, vv[dt][3] = x.w;
      } else {
        const uint2 x = *reinterpret_cast<const uint2 *>(vp + 16 * dt * P);
        vv[dt][0] = x.x, vv[dt][1] = x.y;
      }
    }
    const uint64_t sat = uint64_t(idv) * kvh + head;
    const float ks = scale * power_of_two(int(a.cache.ks[sat]) - 127);
    const float vs = power_of_two(int(a.cache.vs[sat]) - 127);

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
    const bool partial = b + 16 * T - 1 > pos_lo || (a.window && int64_t(b) <= int64_t(pos_hi) - a.window);
    bf16x8 pb[NT][T / 2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float x[4 * T];
      float top = -INFINITY;
#pragma unroll
      for (int i = 0; i < 4 * T; ++i) {
        x[i] = s[nt][i / 4][i % 4] * ks;
        if (partial) x[i] = see[nt](tv + i) ? x[i] : -INFINITY;
        top = fmaxf(top, x[i]);
      }
      top = fmaxf(m[nt], max_lane16(top));
      const float at = top == -INFINITY ? 0.0f : top;  // no key seen yet: every weight 0
      const float fade = __builtin_amdgcn_exp2f(m[nt] - at);
      m[nt] = top;
      sum[nt] *= fade;
      if (__any(fade != 1.0f)) {
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[nt][dt] *= fade;
      }
      u32x4 w[T / 2];
#pragma unroll
      for (int t = 0; t < T; ++t) {
        float e[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          e[i] = __builtin_amdgcn_exp2f(x[4 * t + i] - at);
          sum[nt] += e[i];
        }
        // rounded to bf16, half a step of each weight: the matrix operand's type
        w[t / 2][2 * (t & 1)] = bf16_pair(e[0] * vs, e[1] * vs);
        w[t / 2][2 * (t & 1) + 1] = bf16_pair(e[2] * vs, e[3] * vs);
      }
#pragma unroll
      for (int u = 0; u < T / 2; ++u) pb[nt][u] = __builtin_bit_cast(bf16x8, w[u]);
    }
    if (partial) {
      // what lies behind the sequence is not read; a NaN code that some row
      // must not see leaves the product (0 * NaN is NaN) and reaches the rows
      // that see it afterwards, as the count of such codes they see
      bool nan = false;
      uint32_t hit[DT][W];
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int k = 0; k < W; ++k) {
          const int32_t left = sp.len - (tv + 4 * k);
          const uint32_t keep = left >= 4 ? ~0u : left <= 0 ? 0u : (1u << (8 * left)) - 1u;
          uint32_t c = vv[dt][k] & keep;
          const uint32_t is = ((c & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;  // byte's top bit: a NaN code
          hit[dt][k] = is;
          nan |= is != 0;
          vv[dt][k] = c & ~((is >> 7) * 0xffu);
        }
      if (__any(nan)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int dt = 0; dt < DT; ++dt) {
            f32x4 count = {};
#pragma unroll
            for (int u = 0; u < T / 2; ++u) {
              u32x4 seen;
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const int32_t j = tv + 8 * u + 2 * k;
                seen[k] = (see[nt](j) ? 0x3f80u : 0u) | (see[nt](j + 1) ? 0x3f800000u : 0u);
              }
              const uint32_t h0 = (hit[dt][2 * u] >> 7) * 0x38u, h1 = (hit[dt][2 * u + 1] >> 7) * 0x38u;  // 1 in E4M3
              count = __builtin_amdgcn_mfma_f32_16x16x32_bf16(e4m3_bf16(h0, h1), __builtin_bit_cast(bf16x8, seen),
                                                              count, 0, 0, 0);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) o[nt][dt][i] += count[i] > 0.0f ? __uint_as_float(0x7fc00000u) : 0.0f;
          }
      }
    }
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int u = 0; u < T / 2; ++u) {
        const bf16x8 v = e4m3_bf16(vv[dt][2 * u], vv[dt][2 * u + 1]);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
          o[nt][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, pb[nt][u], o[nt][dt], 0, 0, 0);
      }
  }

  // join the four wavefronts: 2 and 3 into 0 and 1, then 1 into 0
  __shared__ float s_m[4][NT][16], s_l[4][NT][16];
  __shared__ f32x4 s_o[2][NT * DT][64];
  if (__any(bad)) {
    if (l == 0) atomicOr(a.status, kStatusBadCachePage);
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
  if (wave) return;

  if (sp.chunks <= 1) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int64_t r = int64_t(row0) + 16 * nt + n;
      if (r >= sp.rows) continue;
      const uint64_t t = uint64_t(sp.first + r / group);
      const uint32_t h = head * group + uint32_t(r % group);
      const float inv = sum[nt] == 0.0f ? 0.0f : 1.0f / sum[nt];
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
        store_out(a.out, t * a.out.token + uint64_t(h) * a.out.head + 16 * dt + 4 * g, o[nt][dt][0] * inv,
                  o[nt][dt][1] * inv, o[nt][dt][2] * inv, o[nt][dt][3] * inv);
      if (a.lse && g == 0) a.lse[t * a.heads + h] = sum[nt] == 0.0f ? -INFINITY : m[nt] * kLn2 + __logf(sum[nt]);
    }
    return;
  }
  float *rec = part + uint64_t(blockIdx.x) * (16 * NT * (D + 2));
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    float *row = rec + (16 * nt + n) * (D + 2);
    if (g == 0) row[D] = m[nt], row[D + 1] = sum[nt];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      float2 *to = reinterpret_cast<float2 *>(row + 16 * dt + 4 * g);  // rows of D + 2 floats: 8-byte aligned
      to[0] = make_float2(o[nt][dt][0], o[nt][dt][1]);
      to[1] = make_float2(o[nt][dt][2], o[nt][dt][3]);
    }
  }
}

// Joins the chunks of one row a wavefront, in their order.
template <int D>
__global__ __launch_bounds__(256) void k_paged_join(PagedArgs a, PagedPlan p, const float *part) {
  constexpr int V = D / 64;
  const uint32_t kvh = a.cache.heads, group = a.heads / kvh, l = threadIdx.x & 63u;
  const uint32_t seq = blockIdx.y, head = blockIdx.z;
  const int64_t r = int64_t(blockIdx.x) * 4 + threadIdx.x / 64;
  const uint32_t per = 16 * p.row_tiles, tile = uint32_t(r / per);
  const Span sp = paged_span(a, p, seq, tile * per);
  if (r >= sp.rows || sp.chunks <= 1) return;
  const uint64_t rec = uint64_t(per) * (D + 2);
  const float *row = part + (uint64_t(tile) * kvh * p.chunks * a.seqs + uint64_t(seq) * p.chunks * kvh + head) * rec +
                     uint32_t(r % per) * (D + 2);
  const uint64_t next = kvh * rec;  // the next chunk's record
  float top = -INFINITY;
  for (uint32_t c = 0; c < sp.chunks; ++c) top = fmaxf(top, row[c * next + D]);
  const float at = top == -INFINITY ? 0.0f : top;
  float total = 0.0f, o[V] = {};
  for (uint32_t c = 0; c < sp.chunks; ++c) {
    const float *x = row + c * next;
    const float fade = __builtin_amdgcn_exp2f(x[D] - at);
    total += x[D + 1] * fade;
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] += x[V * l + i] * fade;
  }
  const uint64_t t = uint64_t(sp.first + r / group);
  const uint32_t h = head * group + uint32_t(r % group);
  const float inv = total == 0.0f ? 0.0f : 1.0f / total;
  const uint64_t to = t * a.out.token + uint64_t(h) * a.out.head + V * l;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    if (a.out.bf16)
      static_cast<uint16_t *>(a.out.p)[to + i] = uint16_t(bf16_pair(o[i] * inv, 0.0f));
    else
      static_cast<float *>(a.out.p)[to + i] = o[i] * inv;
  }
  if (a.lse && l == 0) a.lse[t * a.heads + h] = total == 0.0f ? -INFINITY : top * kLn2 + __logf(total);
}

template <int D, int NT, int T>
hipError_t launch(hipStream_t s, const PagedArgs &a, const PagedPlan &p, float *part) {
  k_paged_attention<D, NT, T><<<uint32_t(p.blocks), 256, 0, s>>>(a, p, part);
  if (p.chunks > 1) {
    const uint32_t rows = uint32_t(a.max_new) * (a.heads / a.cache.heads);
    k_paged_join<D><<<dim3((rows + 3) / 4, a.seqs, a.cache.heads), 256, 0, s>>>(a, p, part);
  }
  return hipGetLastError();
}

template <int D>
hipError_t launch_dim(hipStream_t s, const PagedArgs &a, const PagedPlan &p, float *part) {
  if constexpr (D <= 128)
    if (p.row_tiles == 4) return launch<D, 4, 4>(s, a, p, part);
  if constexpr (D <= 256)
    if (p.row_tiles == 2) return launch<D, 2, D == 256 ? 2 : 4>(s, a, p, part);
  return launch<D, 1, D == 512 ? 2 : 4>(s, a, p, part);
}

}  // namespace

// Rows a wavefront holds: as many 16-row tiles as the longest new block fills
// and the registers of the head size leave room for (64 rows of 128, 32 of
// 256, 16 of 512).  Chunks: enough workgroups to fill the card where there
// are few rows, none below one step a wavefront.
PagedPlan paged_plan(const PagedArgs &a) {
  PagedPlan p{};
  const uint64_t rows = uint64_t(a.max_new) * (a.heads / a.cache.heads);
  const uint32_t dim = a.cache.dim, most = dim <= 128 ? 4 : dim == 256 ? 2 : 1;
  p.row_tiles = rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
  if (p.row_tiles > most) p.row_tiles = most;
  const uint64_t tiles = (rows + 16 * p.row_tiles - 1) / (16 * p.row_tiles);
  const uint64_t base = tiles * a.cache.heads * a.seqs;  // workgroups of an uncut launch
  uint64_t span = a.max_len;
  if (a.window && uint64_t(a.window) + a.max_new + 63 < span) span = uint64_t(a.window) + a.max_new + 63;
  constexpr uint64_t kWant = 2048, kLeast = 256;
  const uint64_t rec = 16ull * p.row_tiles * (dim + 2);
  uint64_t chunks = (kWant + base - 1) / base;
  const uint64_t fit = kPagedPartFloats / (rec * base);
  if (chunks > fit) chunks = fit;
  if (chunks > (span + kLeast - 1) / kLeast) chunks = (span + kLeast - 1) / kLeast;
  if (chunks < 1) chunks = 1;
  p.chunk = uint32_t(((span + chunks - 1) / chunks + kLeast - 1) / kLeast * kLeast);
  p.chunks = span ? uint32_t((span + p.chunk - 1) / p.chunk) : 1;
  p.blocks = base * p.chunks;
  return p;
}

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
