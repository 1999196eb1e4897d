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
// swizzle(r), so that neither read meets a bank twice.
#include <type_traits>

#include "s14_attn.hpp"
#include "s14_attn_util.hpp"
#include "s14_device_util.hpp"

namespace s14 {
namespace {

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
typedef __attribute__((address_space(3))) void lds_void;

constexpr uint32_t kPromptRows = 128;

// Row block `index` of the packed sequences: its sequence's first token and
// length, and the block within it.  Every sequence has its rows in whole
// blocks, its last ones, with the most keys to walk, first.  kMixed (up to 64
// sequences, of 8 blocks in the mean): of each sequence the blocks 8 q .. 8 q +
// 7, which share its tiles in L2, from the highest q down, so that no long
// block is left for the end (us, one sequence after the other / mixed: 12 of
// up to 2,749 tokens 130 / 120, 7 of up to 2,977 142 / 135, 64 of up to 1,000 89
// / 90: finding the block takes a little longer).  A window's blocks are alike.
struct Block {
  int64_t first;
  int32_t len;
  uint32_t row0;
};
constexpr uint32_t kTogether = 8;

// The sum of v over the wavefront, in each lane.
__device__ __forceinline__ uint32_t wave_sum(uint32_t v) {
  v += uint32_t(__builtin_amdgcn_update_dpp(0, int(v), 0xb1, 0xf, 0xf, false));   // quad_perm [1,0,3,2]
  v += uint32_t(__builtin_amdgcn_update_dpp(0, int(v), 0x4e, 0xf, 0xf, false));   // quad_perm [2,3,0,1]
  v += uint32_t(__builtin_amdgcn_update_dpp(0, int(v), 0x141, 0xf, 0xf, false));  // row_half_mirror
  v += uint32_t(__builtin_amdgcn_update_dpp(0, int(v), 0x140, 0xf, 0xf, false));  // row_mirror
  auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = r[0] + r[1];
  r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return r[0] + r[1];
}

// The sums of v over the lanes up to each.
__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {
  const uint32_t l = threadIdx.x & 63u;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t o = __shfl_up(v, d);
    if (l >= uint32_t(d)) v += o;
  }
  return v;
}

template <bool kMixed>
__device__ __forceinline__ bool find_block(const PromptArgs &a, uint32_t index, uint32_t group, Block &out) {
  const uint32_t l = threadIdx.x & 63u;
  uint32_t before = 0;
  for (uint32_t s0 = 0; s0 < a.seqs; s0 += 64) {
    const uint32_t s = s0 + l;
    int32_t first = 0, len = 0;  // packed rows fit 31 bits
    if (s < a.seqs) {
      first = int32_t(clamp_row(a.cu[s], a.tokens));
      len = int32_t(clamp_row(a.cu[s + 1], a.tokens)) - first;
    }
    const uint32_t blocks = len > 0 ? uint32_t((uint64_t(len) * group + kPromptRows - 1) / kPromptRows) : 0;
    // of every sequence, the blocks from number `low` on, `most` at the most
    uint32_t low = 0, most = ~0u;
    if constexpr (kMixed) {
      const auto above = [&](uint32_t q) {  // blocks from number 8 q on
        const uint32_t from = kTogether * q;
        return uint32_t(__builtin_amdgcn_readfirstlane(wave_sum(blocks > from ? blocks - from : 0)));
      };
      uint32_t q = 0, end = (wave_max_u32(blocks) + kTogether - 1) / kTogether;
      while (end - q > 1) {
        const uint32_t mid = (q + end) / 2, n = above(mid);
        if (index < n)
          q = mid;
        else
          end = mid, before = n;
      }
      low = kTogether * q, most = kTogether;
    }
    const uint32_t here_blocks = blocks > low ? (blocks - low < most ? blocks - low : most) : 0;
    const uint32_t sum = wave_scan(here_blocks);
    const uint64_t here = __ballot(index - before < sum);
    if (here) {
      // one lane's values: the block is uniform, its descriptors and bounds scalar
      const int lane = __builtin_amdgcn_readfirstlane(__builtin_ctzll(here));
      out.first = __builtin_amdgcn_readlane(first, lane);
      out.len = __builtin_amdgcn_readlane(len, lane);
      out.row0 = (low + __builtin_amdgcn_readlane(sum, lane) - 1 - (index - before)) * kPromptRows;
      return true;
    }
    before += __builtin_amdgcn_readlane(sum, 63);
  }
  return false;
}

// K: sixteen neighbouring rows' pieces of one number, the first product's
// read, are in different banks.  V: so are the pieces of four rows and 32
// dimensions, which half a wavefront reads for the second.
template <int D, bool kV>
__device__ __forceinline__ uint32_t swizzle(uint32_t row) {
  if (kV) return D == 64 ? (row & 2u) * 2u : (row & 3u) * 4u;
  return D == 64 ? (row >> 1) & 7u : row & 15u;
}

__device__ __forceinline__ uint32_t lds_at(const void *p) { return uint32_t(reinterpret_cast<uintptr_t>((lds_void *)p)); }

// KT rows of D values from `base` (rows `stride` >= 2 D bytes apart, `valid`
// >= 1 of them there: the rest become zeros) into LDS.
template <int D, int KT, bool kV>
__device__ __forceinline__ void stage(const uint16_t *base, uint32_t stride, int32_t valid, uint16_t *lds) {
  constexpr uint32_t kPieces = D / 8, kPasses = KT * kPieces / 256, kRows = 256 / kPieces;  // rows a pass
  const uint32_t rows = valid < KT ? uint32_t(valid) : uint32_t(KT);
  const uint32_t to = lds_at(lds) + (threadIdx.x & ~63u) * 16;
  // In asm: the compiler would let every LDS read wait for these loads, whose
  // halves of the double buffer it cannot tell apart.  No register waits for
  // them; the wait at the head of the next tile does.
  // m0 cannot be named as changed (the compiler reserves it, and warns); nothing
  // else in these kernels reads it: gfx950's other LDS instructions do not.
#pragma unroll
  for (uint32_t i = 0; i < kPasses; ++i) {
    const uint32_t in = threadIdx.x / kPieces, piece = (threadIdx.x % kPieces) ^ swizzle<D, kV>(i * kRows + in);
    const uint64_t at = reinterpret_cast<uint64_t>(base) + uint64_t(i * kRows) * stride;
    const u32x4 r = {uint32_t(at), uint32_t(at >> 32), rows > i * kRows ? (rows - i * kRows - 1) * stride + 2 * D : 0u,
                     0x00020000u};
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(
                     __builtin_amdgcn_readfirstlane(to) + i * 4096),
                 "v"(in * stride + piece * 16), "s"(r)
                 : "memory");
  }
}

__device__ __forceinline__ uint32_t odd_halves(uint32_t w) {  // 0x8000 in each half that is no finite bf16
  const uint32_t e = w & 0x7f807f80u;
  return ((e + 0x00800080u) & 0x80008000u);
}

template <int D, int KT, bool kWindow, bool kMixed>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void k_prompt_attention(PromptArgs a) {
  constexpr int KS = D / 16, DT = D / 32, ST = KT / 32, U = KT / 16;
  __shared__ __align__(1024) uint16_t lds_k[2][KT * D], lds_v[2][KT * D];
  const uint32_t group = a.heads / a.kv_heads, head = blockIdx.x % a.kv_heads;
  Block blk;
  if (!find_block<kMixed>(a, blockIdx.x / a.kv_heads, group, blk)) return;
  const uint32_t wave = threadIdx.x / 64, l = threadIdx.x & 63u, n = l & 31u, h = l >> 5;
  const uint32_t rows = uint32_t(blk.len) * group;  // below 2^31 in all: so the launch is checked
  const uint32_t wrow = blk.row0 + 32 * wave;

  const uint32_t r = wrow + n < rows ? wrow + n : rows - 1;
  const int32_t pos = int32_t(r / group);
  const uint32_t window = kWindow ? a.window : 0u;
  const Visible see(pos, window);
  // tokens that the workgroup, and this wavefront, walk
  const uint32_t blk_last = (blk.row0 + kPromptRows < rows ? blk.row0 + kPromptRows : rows) - 1;
  const int32_t hi = int32_t(blk_last / group) + 1;
  const int32_t blk_first = int32_t(blk.row0 / group);
  const int32_t lo = kWindow && blk_first + 1 > int64_t(window) ? (blk_first + 1 - int32_t(window)) & ~(KT - 1) : 0;
  // (a wavefront without rows takes the last one's part, and stores nothing)
  const int32_t wpos_lo = int32_t((wrow < rows ? wrow : rows - 1) / group);
  const int32_t wpos_hi = int32_t((wrow + 31 < rows ? wrow + 31 : rows - 1) / group);

  bf16x8 q[KS];
  const auto load_q = [&]() {
    const uint16_t *row = a.q + uint64_t(blk.first + pos) * a.q_token +
                          uint64_t(head * group + r % group) * a.q_head;
#pragma unroll
    for (int k = 0; k < KS; ++k) q[k] = *reinterpret_cast<const bf16x8 *>(row + 16 * k + 8 * h);
    // Q is here before the walk: its first use, in the loop, would otherwise
    // wait for every load in flight, each time round
#pragma unroll
    for (int k = 0; k < KS; ++k) asm volatile("" : "+v"(q[k]));
  };
  const auto is_partial = [&](int32_t b) {
    return b + KT - 1 > wpos_lo || (kWindow && int64_t(b) <= int64_t(wpos_hi) - window);
  };

  f32x16 o[DT] = {};
  bool odd = false;
  const float scale = a.scale * kLog2e;
  const uint16_t *kb = a.k + uint64_t(blk.first) * a.k_token + uint64_t(head) * a.k_head;
  const uint16_t *vb = a.v + uint64_t(blk.first) * a.v_token + uint64_t(head) * a.v_head;
  const uint32_t ks = uint32_t(a.k_token * 2), vs = uint32_t(a.v_token * 2);

  // This lane's places in an LDS tile: piece h of its K row, from which the
  // others are an exclusive or away (rows 32 apart: a constant), and its part
  // of a V row for the transposing read (dimensions 32 apart: an exclusive or,
  // rows 8 apart: a constant).
  const uint32_t k_at = n * (2 * D) + (h ^ swizzle<D, false>(n)) * 16;
  const uint32_t v_row = 4 * h + (l & 15u) / 4;
  const uint32_t v_at = v_row * (2 * D) + ((((l >> 4) & 1u) * 2 + ((l & 3u) >> 1)) ^ swizzle<D, true>(v_row)) * 16 + (l & 1u) * 8;

  // The scores of the tile to come are computed while this one's weights are:
  // the first product's matrix instructions stand between the exponentials,
  // in this order (left to itself the compiler puts one after the other).
  float x[16 * ST];  // scores of the next tile to be weighted
  bf16x8 pb[U];      // weights
  float m = -INFINITY, sum = 0.0f;
  constexpr int kAhead = 4;  // LDS reads this many matrix instructions ahead of their use
  const auto step = [&](uint32_t buf, auto weigh, auto tail) {
    constexpr int N = ST * KS, E = 16 * ST / N;  // matrix instructions, weights at each
    const uint32_t lk = lds_at(lds_k[buf]) + k_at;
    const auto k_frag = [&](int i) {
      const int t = i % ST, k = i / ST;
      return *(const __attribute__((address_space(3))) bf16x8 *)(uintptr_t)((lk ^ (32u * k)) + 64 * D * t);
    };
    f32x16 s[ST] = {};
    bf16x8 kf[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) kf[i] = k_frag(i);
    const float at = m == -INFINITY ? 0.0f : m;
    uint32_t w[4 * U];
    float even = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      s[i % ST] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[i % kAhead], q[i / ST], s[i % ST], 0, 0, 0);
      if (i + kAhead < N)
        kf[i % kAhead] = k_frag(i + kAhead);
      else
        tail(i + kAhead - N);
      if constexpr (decltype(weigh)::value) {
#pragma unroll
        for (int e = i * E; e < (i + 1) * E; ++e) {
          const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(x[e], scale, -at));
          sum += p;
          if (e % 2) {
            w[e / 2] = bf16_pair(even, p);  // half a step of each weight: the matrix operand's type
            asm volatile("" : "+v"(w[e / 2]));
          } else {
            even = p;
          }
        }
        asm volatile("" : "+v"(sum));  // here, not when it is needed: the weights' registers are
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    if constexpr (decltype(weigh)::value) {
#pragma unroll
      for (int u = 0; u < U; ++u) pb[u] = __builtin_bit_cast(bf16x8, u32x4{w[4 * u], w[4 * u + 1], w[4 * u + 2], w[4 * u + 3]});
    }
#pragma unroll
    for (int i = 0; i < 16 * ST; ++i) x[i] = s[i / 16][i % 16];
  };
  // Hides what tile b's rows must not see.
  const auto hide = [&](int32_t b) {
    if (is_partial(b)) {
      keep_branch();
#pragma unroll
      for (int i = 0; i < 16 * ST; ++i) x[i] = see(b + 8 * (i / 4) + 4 * int32_t(h) + i % 4) ? x[i] : -INFINITY;
    }
  };
  // Moves the maximum, where the weights would pass 2^kRise: O is seldom multiplied.
  const auto raise = [&](float top) {
    const auto y = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
    top = fmaxf(m, fmaxf(__uint_as_float(y[0]), __uint_as_float(y[1])) * scale);
    if (__any(top > m + kRise)) {
      const float fade = __builtin_amdgcn_exp2f(m - (top == -INFINITY ? 0.0f : top));
      m = top;
      sum *= fade;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) o[dt] *= fade;
    }
  };
  const auto largest = [&]() {
    float top = x[0];
#pragma unroll
    for (int i = 1; i < 16 * ST; ++i) top = fmaxf(top, x[i]);
    return top;
  };

  // At the head of tile b the LDS holds K of b + KT and V of b; K of b, whose
  // scores are in registers, and V of b - KT give their places to the loads.
  stage<D, KT, false>(kb + uint64_t(lo) * a.k_token, ks, blk.len - lo, lds_k[0]);
  stage<D, KT, true>(vb + uint64_t(lo) * a.v_token, vs, blk.len - lo, lds_v[0]);
  if (lo + KT < hi) stage<D, KT, false>(kb + uint64_t(lo + KT) * a.k_token, ks, blk.len - lo - KT, lds_k[1]);
  load_q();
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  step(0, std::false_type{}, [](int) {});
  hide(lo);
  raise(largest());
  uint32_t buf = 0;
  int32_t b = lo;
  const auto next_tile = [&]() {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (b + 2 * KT < hi) stage<D, KT, false>(kb + uint64_t(b + 2 * KT) * a.k_token, ks, blk.len - b - 2 * KT, lds_k[buf]);
    if (b + KT < hi) stage<D, KT, true>(vb + uint64_t(b + KT) * a.v_token, vs, blk.len - b - KT, lds_v[buf ^ 1]);
  };
  constexpr int N = DT * U;
  bf16x8 vf[kAhead];
  const auto v_frag = [&](int i) {
    const int dt = i % DT, u = i / DT;
    const uint32_t lv = lds_at(lds_v[buf]) + v_at;
    union {
      s16x4 x[2];
      bf16x8 v;
    } f;
#pragma unroll
    for (int half = 0; half < 2; ++half)
      f.x[half] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (lds_s16x4 *)(uintptr_t)((lv ^ (64u * dt)) + (16 * u + 8 * half) * (2 * D)));
    return f.v;
  };
  // (after the wavefront's last tile: scores of no tile, unused)
  const auto weigh = [&]() { step(buf ^ 1, std::true_type{}, [&](int i) { vf[i] = v_frag(i); }); };
  const auto add = [&]() {  // the second product; the largest of the next scores
    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int i = 0; i < N; ++i) {
      o[i % DT] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[i % kAhead], pb[i / DT], o[i % DT], 0, 0, 0);
      if (i + kAhead < N) vf[i % kAhead] = v_frag(i + kAhead);
#pragma unroll
      for (int e = i * 16 * ST / N; e < (i + 1) * 16 * ST / N; e += 2) top[i % 2] = fmaxf(top[i % 2], fmaxf(x[e], x[e + 1]));
      asm volatile("" : "+v"(top[i % 2]));
      __builtin_amdgcn_sched_barrier(0);
    }
    return fmaxf(top[0], top[1]);
  };
  // Tiles that every row of the workgroup sees whole: the walk's bulk, without
  // a branch, which would move O and x from registers to registers where its
  // sides meet.  (A window's walk is short and has a branch.)
  if constexpr (!kWindow) {
    const int32_t whole = (blk_first + 1) & ~(KT - 1);  // tiles before this lie before every row
    for (; b + 2 * KT <= whole; b += KT, buf ^= 1) {
      next_tile();
      weigh();
      raise(add());
    }
    if (b + KT <= whole) {  // the last of them
      next_tile();
      weigh();
      hide(b + KT);
      raise(add());
      b += KT, buf ^= 1;
    }
  }
  const int32_t careful = b;
  for (; b < hi; b += KT, buf ^= 1) {
    next_tile();
    weigh();
    hide(b + KT);
    float top;
    if (kWindow && !is_partial(b)) {
      top = add();
    } else {
      // An infinity or NaN in a V row that some rows must not see would reach
      // them through 0 * inf: such values leave the product, and the rows that
      // see them get them back below.
#pragma unroll
      for (int i = 0; i < N; ++i) {
        u32x4 w = __builtin_bit_cast(u32x4, vf[i % kAhead]);
        if (i + kAhead < N) vf[i % kAhead] = v_frag(i + kAhead);
        u32x4 t;
#pragma unroll
        for (int j = 0; j < 4; ++j) t[j] = odd_halves(w[j]);
        if (__any((t[0] | t[1] | t[2] | t[3]) != 0)) {
          odd = true;
          w &= ~(t | (t - (t >> 15)));  // 0x8000 in a half becomes 0xffff
        }
        o[i % DT] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, w), pb[i / DT], o[i % DT], 0, 0, 0);
      }
      top = largest();
    }
    if (b + KT < hi) raise(top);
  }

  if (odd) {  // uniform, and rare: one token after the other
    for (b = careful; b < hi; b += KT) {
      if (kWindow && !is_partial(b)) continue;
      for (int32_t j = b; j < min(b + KT, hi); ++j) {
        const uint16_t *row = vb + uint64_t(j) * a.v_token + 4 * h;
        const bool in = see(j);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          f32x16 back;
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float v = __uint_as_float(uint32_t(row[32 * dt + 8 * (i / 4) + i % 4]) << 16);
            back[i] = (in & !(fabsf(v) < INFINITY)) ? v : 0.0f;
          }
          o[dt] += back;
        }
      }
    }
  }

  {
    const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(sum), __float_as_uint(sum), false, false);
    sum = checked_sum(__uint_as_float(x[0]) + __uint_as_float(x[1]), m);
  }
  const bool mine = wrow + n < rows;
  const uint64_t t = uint64_t(blk.first + pos);
  const uint32_t qh = head * group + r % group;
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  const uint64_t to = t * a.out.token + uint64_t(qh) * a.out.head;
  if (a.out.bf16) {
    // lanes l and l + 32 have the halves of a row's eight values; after the
    // swap one has the first eight, the other the next
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int i = 0; i < 16; i += 8) {
        const auto y = __builtin_amdgcn_permlane32_swap(bf16_pair(o[dt][i] * inv, o[dt][i + 1] * inv),
                                                        bf16_pair(o[dt][i + 4] * inv, o[dt][i + 5] * inv), false, false);
        const auto z = __builtin_amdgcn_permlane32_swap(bf16_pair(o[dt][i + 2] * inv, o[dt][i + 3] * inv),
                                                        bf16_pair(o[dt][i + 6] * inv, o[dt][i + 7] * inv), false, false);
        if (mine) {
          const u32x4 w = {y[0], z[0], y[1], z[1]};
          *reinterpret_cast<u32x4 *>(static_cast<uint16_t *>(a.out.p) + to + 32 * dt + 2 * i + 8 * h) = w;
        }
      }
  } else if (mine) {
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int i = 0; i < 16; i += 4)
        *reinterpret_cast<float4 *>(static_cast<float *>(a.out.p) + to + 32 * dt + 2 * i + 4 * h) =
            make_float4(o[dt][i] * inv, o[dt][i + 1] * inv, o[dt][i + 2] * inv, o[dt][i + 3] * inv);
  }
  if (!mine) return;
  if (a.lse && h == 0) a.lse[t * a.heads + qh] = sum == 0.0f ? -INFINITY : m * kLn2 + __logf(sum);
}

}  // namespace

hipError_t launch_prompt_attention(hipStream_t s, const PromptArgs &a) {
  const uint32_t group = a.heads / a.kv_heads;
  const uint64_t blocks = (uint64_t(a.tokens) * group + kPromptRows - 1) / kPromptRows + a.seqs;
  const uint32_t grid = uint32_t(blocks * a.kv_heads);
  const bool mixed = !a.window && a.seqs > 1 && a.seqs <= 64 && uint64_t(a.tokens) * group / kPromptRows >= 8ull * a.seqs;
  const auto launch = [&](auto dim, auto keys) {
    constexpr int D = decltype(dim)::value, KT = decltype(keys)::value;
    const auto go = [&](auto kernel) { kernel<<<grid, 256, 0, s>>>(a); };
    if (a.window)
      go(k_prompt_attention<D, KT, true, false>);
    else if (mixed)
      go(k_prompt_attention<D, KT, false, true>);
    else
      go(k_prompt_attention<D, KT, false, false>);
  };
  using std::integral_constant;
  switch (a.dim) {
    case 64: launch(integral_constant<int, 64>{}, integral_constant<int, 64>{}); break;
    case 128: launch(integral_constant<int, 128>{}, integral_constant<int, 64>{}); break;
    case 256: launch(integral_constant<int, 256>{}, integral_constant<int, 32>{}); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

}  // namespace s14
