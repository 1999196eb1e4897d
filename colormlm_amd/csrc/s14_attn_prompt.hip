// Causal attention over whole packed prompts, bf16, grouped heads.
//
// A workgroup takes 128 rows of one sequence and key head, a row being a
// (token, query head of the group) pair: the group's heads share the K and V
// tiles, and a short prompt's rows still fill the tile.  Each wavefront keeps
// 32 rows of Q and O in registers and walks the key tiles that the workgroup
// stages in LDS: S^T = K Q^T and O^T = V^T P^T on v_mfma_f32_32x32x16_bf16.
// With the tokens as rows the first product's result (lane = 32 h + n: query
// row n, tokens 8 a + 4 h + i of a 32-token tile) is the second's operand as
// it stands if the lane's V operand takes the same tokens, which the
// transposing LDS read gives: P stays in registers.
//
// LDS rows are D values in 16-byte pieces, piece c of row r at place c ^
// swizzle(r), so that neither read of eight rows meets a bank twice.
#include "s14_attn.hpp"
#include "s14_attn_util.hpp"

namespace s14 {
namespace {

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
typedef __attribute__((address_space(3))) void lds_void;

constexpr uint32_t kPromptRows = 128;

// Row block `index` of the packed sequences: its sequence's first token and
// length, and the block within it.  Every sequence has its rows in whole
// blocks, the last ones first (the longest work leads).
struct Block {
  int64_t first;
  int32_t len;
  uint32_t row0;
};
__device__ __forceinline__ bool find_block(const PromptArgs &a, uint32_t index, uint32_t group, Block &out) {
  const uint32_t l = threadIdx.x & 63u;
  uint32_t before = 0;
  for (uint32_t s0 = 0; s0 < a.seqs; s0 += 64) {
    const uint32_t s = s0 + l;
    int64_t first = 0, len = 0;
    if (s < a.seqs) {
      first = clamp_row(a.cu[s], a.tokens);
      len = clamp_row(a.cu[s + 1], a.tokens) - first;
    }
    const uint32_t blocks = len > 0 ? uint32_t((uint64_t(len) * group + kPromptRows - 1) / kPromptRows) : 0;
    uint32_t sum = blocks;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const uint32_t o = __shfl_up(sum, d);
      if (l >= uint32_t(d)) sum += o;
    }
    const uint64_t here = __ballot(index - before < sum);
    if (here) {
      const int lane = __builtin_ctzll(here);
      const uint32_t end = __shfl(sum, lane);
      out.first = __shfl(first, lane);
      out.len = int32_t(__shfl(len, lane));
      out.row0 = (end - 1 - (index - before)) * kPromptRows;
      return true;
    }
    before += __shfl(sum, 63);
  }
  return false;
}

template <int D>
__device__ __forceinline__ uint32_t swizzle(uint32_t row) {
  return D == 64 ? ((row >> 1) & 3u) * 2u : (row & 7u) * 2u;
}

// KT rows of D values from `base` (rows `stride` >= 2 D bytes apart, `valid`
// >= 1 of them there: the rest become zeros) into LDS.
template <int D, int KT>
__device__ __forceinline__ void stage(const uint16_t *base, uint32_t stride, int32_t valid, uint16_t *lds) {
  constexpr uint32_t kPieces = D / 8, kPasses = KT * kPieces / 256;
  const uint32_t rows = valid < KT ? uint32_t(valid) : uint32_t(KT);
  const auto r = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t *>(base), 0, int((rows - 1) * stride + 2 * D), 0x00020000);
#pragma unroll
  for (uint32_t i = 0; i < kPasses; ++i) {
    const uint32_t at = i * 256 + threadIdx.x, row = at / kPieces, piece = (at % kPieces) ^ swizzle<D>(row);
    const uint32_t wave_at = i * 256 + (threadIdx.x & ~63u);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void *)(lds + wave_at * 8), 16, row * stride + piece * 16, 0, 0, 0);
  }
}

__device__ __forceinline__ uint32_t odd_halves(uint32_t w) {  // 0x8000 in each half that is no finite bf16
  const uint32_t e = w & 0x7f807f80u;
  return ((e + 0x00800080u) & 0x80008000u);
}

template <int D, int KT>
__global__ __launch_bounds__(256) void k_prompt_attention(PromptArgs a) {
  constexpr int KS = D / 16, DT = D / 32, ST = KT / 32, U = KT / 16;
  __shared__ __align__(16) uint16_t lds_k[2][KT * D], lds_v[2][KT * D];
  const uint32_t group = a.heads / a.kv_heads, head = blockIdx.x % a.kv_heads;
  Block blk;
  if (!find_block(a, blockIdx.x / a.kv_heads, group, blk)) return;
  const uint32_t wave = threadIdx.x / 64, l = threadIdx.x & 63u, n = l & 31u, h = l >> 5;
  const uint64_t rows = uint64_t(blk.len) * group;
  const uint32_t wrow = blk.row0 + 32 * wave;

  const uint64_t r = wrow + n < rows ? wrow + n : rows - 1;
  const int32_t pos = int32_t(r / group);
  const Visible see(pos, a.window);
  bf16x8 q[KS];
  {
    const uint16_t *row = a.q + uint64_t(blk.first + pos) * a.q_token +
                          uint64_t(head * group + uint32_t(r % group)) * a.q_head;
#pragma unroll
    for (int k = 0; k < KS; ++k) q[k] = *reinterpret_cast<const bf16x8 *>(row + 16 * k + 8 * h);
  }
  // tokens that the workgroup, and this wavefront, walk
  const uint64_t blk_last = (blk.row0 + kPromptRows < rows ? blk.row0 + kPromptRows : rows) - 1;
  const int32_t hi = int32_t(blk_last / group) + 1;
  const int32_t blk_first = int32_t(blk.row0 / group);
  const int32_t lo = a.window && blk_first + 1 > int64_t(a.window) ? (blk_first + 1 - int32_t(a.window)) & ~(KT - 1) : 0;
  const bool live = wrow < rows;
  const int32_t wpos_lo = int32_t(wrow / group);
  const int32_t wpos_hi = live ? int32_t((wrow + 31 < rows ? wrow + 31 : rows - 1) / group) : -1;

  f32x16 o[DT] = {};
  float m = -INFINITY, sum = 0.0f;
  const float scale = a.scale * kLog2e;
  const uint16_t *kb = a.k + uint64_t(blk.first) * a.k_token + uint64_t(head) * a.k_head;
  const uint16_t *vb = a.v + uint64_t(blk.first) * a.v_token + uint64_t(head) * a.v_head;
  const uint32_t ks = uint32_t(a.k_token * 2), vs = uint32_t(a.v_token * 2);

  // this lane's places in LDS: its K row (per 32-token tile), and its piece of
  // a V row for the transposing read
  const uint32_t v_row = 4 * h + (l & 15u) / 4, v_piece = ((l >> 4) & 1u) * 2 + ((l & 3u) >> 1), v_byte = (l & 1u) * 8;

  stage<D, KT>(kb + uint64_t(lo) * a.k_token, ks, blk.len - lo, lds_k[0]);
  stage<D, KT>(vb + uint64_t(lo) * a.v_token, vs, blk.len - lo, lds_v[0]);
  uint32_t buf = 0;
  for (int32_t b = lo; b < hi; b += KT, buf ^= 1) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (b + KT < hi) {
      stage<D, KT>(kb + uint64_t(b + KT) * a.k_token, ks, blk.len - b - KT, lds_k[buf ^ 1]);
      stage<D, KT>(vb + uint64_t(b + KT) * a.v_token, vs, blk.len - b - KT, lds_v[buf ^ 1]);
    }
    if (b > wpos_hi || (a.window && int64_t(b) + KT - 1 <= int64_t(wpos_lo) - a.window)) continue;
    const uint8_t *lk = reinterpret_cast<const uint8_t *>(lds_k[buf]);
    const uint16_t *lv = lds_v[buf];

    f32x16 s[ST];
#pragma unroll
    for (int t = 0; t < ST; ++t) {
      s[t] = f32x16{};
      const uint32_t row = 32 * t + n;
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        const bf16x8 kf = *reinterpret_cast<const bf16x8 *>(lk + row * (2 * D) + ((2 * k + h) ^ swizzle<D>(row)) * 16);
        s[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf, q[k], s[t], 0, 0, 0);
      }
    }
    const bool partial = b + KT - 1 > wpos_lo || (a.window && int64_t(b) <= int64_t(wpos_hi) - a.window);
    float x[16 * ST];
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < 16 * ST; ++i) {
      x[i] = s[i / 16][i % 16];
      if (partial) x[i] = see(b + 8 * (i / 4) + 4 * int32_t(h) + i % 4) ? x[i] : -INFINITY;
      top = fmaxf(top, x[i]);
    }
    {
      const auto y = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
      top = fmaxf(__uint_as_float(y[0]), __uint_as_float(y[1]));
    }
    top = fmaxf(m, top * scale);
    const float at = top == -INFINITY ? 0.0f : top;
    const float fade = __builtin_amdgcn_exp2f(m - at);
    m = top;
    sum *= fade;
    if (__any(fade != 1.0f)) {
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) o[dt] *= fade;
    }
    bf16x8 pb[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      u32x4 w;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float e0 = __builtin_amdgcn_exp2f(__builtin_fmaf(x[8 * u + 2 * j], scale, -at));
        const float e1 = __builtin_amdgcn_exp2f(__builtin_fmaf(x[8 * u + 2 * j + 1], scale, -at));
        sum += e0;
        sum += e1;
        w[j] = bf16_pair(e0, e1);  // half a step of each weight: the matrix operand's type
      }
      pb[u] = __builtin_bit_cast(bf16x8, w);
    }
    auto v_frag = [&](int dt, int u) {
      union {
        s16x4 x[2];
        bf16x8 v;
      } f;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const uint32_t row = 16 * u + 8 * half + v_row;
        const uint32_t piece = (4 * dt + v_piece) ^ swizzle<D>(row);
        f.x[half] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (lds_s16x4 *)(reinterpret_cast<const uint8_t *>(lv) + row * (2 * D) + piece * 16 + v_byte));
      }
      return f.v;
    };
    // An infinity or NaN in a V row that some rows must not see would reach
    // them through 0 * inf: such values leave the product, and the rows that
    // see them get them back from a count.
    bool odd = false;
    if (partial) {
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const u32x4 w = __builtin_bit_cast(u32x4, v_frag(dt, u));
          odd |= (odd_halves(w[0]) | odd_halves(w[1]) | odd_halves(w[2]) | odd_halves(w[3])) != 0;
        }
    }
    if (__any(odd)) {
      u32x4 seen[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int32_t tok = b + 16 * u + 8 * (j / 2) + 4 * int32_t(h) + 2 * (j % 2);
          seen[u][j] = (see(tok) ? 0x3f80u : 0u) | (see(tok + 1) ? 0x3f800000u : 0u);
        }
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        f32x16 up = {}, down = {};
#pragma unroll
        for (int u = 0; u < U; ++u) {
          u32x4 w = __builtin_bit_cast(u32x4, v_frag(dt, u)), pos_w, neg_w;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint32_t clean = 0, pw = 0, nw = 0;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const uint32_t x = (w[j] >> (16 * e)) & 0xffffu;
              const bool fin = (x & 0x7f80u) != 0x7f80u, nan = !fin && (x & 0x7fu);
              if (fin) clean |= x << (16 * e);
              if (nan || x == 0x7f80u) pw |= 0x3f80u << (16 * e);
              if (nan || x == 0xff80u) nw |= 0x3f80u << (16 * e);
            }
            w[j] = clean, pos_w[j] = pw, neg_w[j] = nw;
          }
          const bf16x8 sv = __builtin_bit_cast(bf16x8, seen[u]);
          o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, w), pb[u], o[dt], 0, 0, 0);
          up = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, pos_w), sv, up, 0, 0, 0);
          down = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, neg_w), sv, down, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < 16; ++i)
          o[dt][i] += (up[i] > 0.0f ? INFINITY : 0.0f) + (down[i] > 0.0f ? -INFINITY : 0.0f);
      }
    } else {
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int u = 0; u < U; ++u)
          o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v_frag(dt, u), pb[u], o[dt], 0, 0, 0);
    }
  }

  {
    const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(sum), __float_as_uint(sum), false, false);
    sum = __uint_as_float(x[0]) + __uint_as_float(x[1]);
  }
  if (wrow + n >= rows) return;
  const uint64_t t = uint64_t(blk.first + pos);
  const uint32_t qh = head * group + uint32_t(r % group);
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  const uint64_t to = t * a.out.token + uint64_t(qh) * a.out.head + 4 * h;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      const uint64_t at = to + 32 * dt + 2 * i;
      if (a.out.bf16)
        *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(a.out.p) + at) =
            make_uint2(bf16_pair(o[dt][i] * inv, o[dt][i + 1] * inv), bf16_pair(o[dt][i + 2] * inv, o[dt][i + 3] * inv));
      else
        *reinterpret_cast<float4 *>(static_cast<float *>(a.out.p) + at) =
            make_float4(o[dt][i] * inv, o[dt][i + 1] * inv, o[dt][i + 2] * inv, o[dt][i + 3] * inv);
    }
  if (a.lse && h == 0) a.lse[t * a.heads + qh] = sum == 0.0f ? -INFINITY : m * kLn2 + __logf(sum);
}

}  // namespace

hipError_t launch_prompt_attention(hipStream_t s, const PromptArgs &a) {
  const uint32_t group = a.heads / a.kv_heads;
  const uint64_t blocks = (uint64_t(a.tokens) * group + kPromptRows - 1) / kPromptRows + a.seqs;
  const uint32_t grid = uint32_t(blocks * a.kv_heads);
  switch (a.dim) {
    case 64: k_prompt_attention<64, 64><<<grid, 256, 0, s>>>(a); break;
    case 128: k_prompt_attention<128, 64><<<grid, 256, 0, s>>>(a); break;
    case 256: k_prompt_attention<256, 32><<<grid, 256, 0, s>>>(a); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

}  // namespace s14
