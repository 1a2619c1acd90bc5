// Attention of few query rows (decode, verify) over the group-affine cache, on the matrix cores.
//
// A workgroup takes up to RPT query rows of one kv head and a slab of its tokens; each of its waves walks a part
// of the slab alone, 16 NT tokens a step, without LDS or barriers until the end.  Codes are exact in 16-bit floats, so
// they go into the products as they are and the scales meet the f32 sums:
//   scores  C[token][row] = sum over a group's coordinates of code * q (v_mfma_f32_16x16x32_f16, one accumulator a
//           group), S = sum_g s_g C_g + b_g sum(q)_g.  A code's bits are or'ed into an f16's mantissa, two at once: 64
//           + c (4 bits) or 1024 + c (8 bits, one byte permutation); b_g - 64 s_g or b_g - 1024 s_g takes b_g's place.
//           q is taken to f16 by a power of two of its row, largest magnitude in [2^13, 2^14): every coordinate over
//           2^-28 of it keeps all its bits, smaller ones are off by 2^-27 of it at most.
//   values  O[row][coordinate] = sum_t (p_t s_t) code (v_mfma_f32_16x16x32_bf16): rows of A carry p s_g, codes are
//           128 + c (4 bits; a product with 128s is taken off at the end) or c in bf16.  A lane unpacks the same word of the
//           tokens its k indices stand for, in pairs, straight into B operands: columns are words, and word
//           coordinate j is the j-th product.  As a word's group is its column's, the 16 rows of A hold one block of
//           RPT rows per group, and a result counts where row and column agree on the group.  Where RPT times the
//           groups is under 16, the rows also hold TI blocks of tokens, so that a lane weighs 4 NT / TI tokens and
//           none twice.  p s goes in as two bf16 pieces (16 bits), sum_t p b and the 128s are added in f32.
// C's lanes hold row = lane % 16 and tokens 4 (lane / 16) + j, which is what A's lanes want when value tokens are
// taken in that order: weights never move between lanes.
//
// Softmax: one reference maximum a row, moved only when a score passes it by 8 (base 2), so a step without a new
// maximum rescales nothing; weights stay under 2^8.
// What bounds it: memory at long caches (32 ragged sequences of d = 256, 546 MB: 127 us, 4.3 TB/s; 4 x 4 rows over
// 4 x 131,076 tokens of d = 128, 604 MB: 129 us, 4.7 TB/s, where a large copy reaches 4.8), the loads' latency, the
// queries' preparation and the join of the waves at short ones (8 heads of 512 tokens 10 us, of 32,768 15 us).  A
// step's codes load as soon as the last step's are used up, and in the same number on every way through the loop, so
// that a wait for one step's never becomes one for the next's.
#pragma once

#include <type_traits>

#include "tq_affine.h"
#include "tq_pieces.h"

namespace tq {

// Rows of pairs are dword-aligned only.
typedef uint32_t u32x2_a4 __attribute__((ext_vector_type(2), aligned(4)));
typedef uint32_t u32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));

// The layout of one instantiation.  KB, VB: bits; DP: head dims up to it; GS: group; RPT: query rows a workgroup.
template <int KB, int VB, int DP, int GS, int RPT>
struct RowsShape {
  static constexpr int NP = 2;                            // pieces of p s
  static constexpr int NG = DP / GS;                      // groups a row
  static constexpr int CH = GS / 32;                      // k steps a group
  static constexpr int KW = GS * KB / 128;                // words a lane holds of a token's group
  // coordinates that 16 columns of words cover: half words where a set of whole ones would need two A operands
  static constexpr int SETD = VB == 8 || DP == 64 || GS * 16 < 128 * RPT ? 64 : 128;
  static constexpr int NS = DP / SETD;                    // such sets
  static constexpr int UD = SETD / 16;                    // coordinates a column: products a set
  static constexpr int NGB = SETD > GS ? SETD / GS : 1;   // groups a set
  static constexpr int NA = NGB * RPT > 16 ? NGB * RPT / 16 : 1;  // A operands a set
  static constexpr int GA = NGB / NA;                     // groups an A operand
  static constexpr int TI = 16 / (GA * RPT);              // blocks of tokens an A operand
  // 16-token tiles a step: four where a block of tokens is one or the sums are few (d = 64, 16 rows of 64 x 32,768 tokens
  // 66 us, by two 72); two elsewhere, for the registers (d = 256, 4 rows of 32 x 16,384 tokens 40 us, by four 108; d =
  // 128, 4 rows of 8 x 32,768 tokens 20.1, by four 20.7)
  static constexpr int NT = TI == 4 || DP == 64 ? 4 : 2;
  static constexpr int NU = NT / TI;                      // tiles a lane weighs
  static constexpr int STEP = 16 * NT;
  // registers that live through a step: sums, queries, codes, weights; with the temporaries, two waves a SIMD have 256
  // each, and what needs more runs one (32 heads of 16,384 tokens, d = 256: 16 rows 59 us, by eight waves 76; 4 rows
  // in groups of 32 57 us, by eight 243; d = 192, 4 rows 55 / 76; d = 128, 16 rows by eight 44 us, by four 57)
  static constexpr int LIVE = NS * NA * (UD + 1) * 4 + DP / 8 + NG + NT * NG * KW + NS * NT * 4 + 2 * NG +
                              NU * 4 + NS * NA * NP * NU * 2;
  static constexpr int WAVES = LIVE > 182 ? 4 : 8;
  static constexpr int PLANES = 4 * NG * STEP;            // floats of a wave's pairs in LDS
  static constexpr int JOIN = RPT * (DP + NG + 2);        // floats of a wave's results there, after the loop
  static constexpr int LDS = WAVES * (PLANES > JOIN ? PLANES : JOIN) * 4;
  static constexpr float OFF = KB == 4 ? 64.f : 1024.f;   // what a key code enters with
  static_assert(GA * TI * RPT == 16 && NT % TI == 0 && NT % 2 == 0, "rows of A");
};

// bf16 bits of two small integers held in f32 (exact to 8 bits): the upper halves.
__device__ __forceinline__ uint32_t top_halves(float lo, float hi) {
  return __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u);
}

typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));

__device__ __forceinline__ f32x4_t mfma_f16(u32x4_t a, u32x4_t b, f32x4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0,
                                                0);
}

// Eight key codes as f16.  4 bits: one word, 64 + c (the code in mantissa bits 4..7), register r holds coordinates
// (r, r + 4); 8 bits: two words, 1024 + c, register r holds (2 r, 2 r + 1).
template <int KB>
__device__ __forceinline__ u32x4_t key_operand(const uint32_t* w, uint32_t mask, uint32_t with) {
  u32x4_t o;
  if constexpr (KB == 4) {  // mask 0x00f000f0, with 0x54005400
    o[0] = ((w[0] << 4) & mask) | with;
    o[1] = (w[0] & mask) | with;
    o[2] = ((w[0] >> 4) & mask) | with;
    o[3] = ((w[0] >> 8) & mask) | with;
  } else {
#pragma unroll
    for (int r = 0; r < 4; ++r)  // bytes: code, 0x64, code, 0x64
      o[r] = __builtin_amdgcn_perm(0x64646464u, w[r >> 1], r & 1 ? 0x04030402u : 0x04010400u);
  }
  return o;
}

template <int DT, int KB, int VB, int DP, int GS, int RPT, bool FULL, bool MASK>
__global__ __launch_bounds__((64 * RowsShape<KB, VB, DP, GS, RPT>::WAVES)) void affine_rows_kernel(const AffineAttnParams p) {
  using S = RowsShape<KB, VB, DP, GS, RPT>;
  __shared__ __attribute__((aligned(16))) float lds[S::LDS / 4];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 15, q4 = lane >> 4;
  const int split = blockIdx.x % p.splits;
  const int blk = blockIdx.x / p.splits;
  const int row_blocks = (p.rows + RPT - 1) / RPT;
  const int bh = blk / row_blocks, row0 = (blk % row_blocks) * RPT;
  const int b = bh / p.Hkv, h = bh % p.Hkv;

  // this lane's row of the weights: group in its A operand, block of tokens, query row
  const int r_l = c % RPT, i_l = (c / RPT) % S::TI, g_l = c / (RPT * S::TI);
  const int row = min(row0 + r_l, p.rows - 1);
  const int q_l = row / p.R, q_r = row % p.R;

  const int kg = FULL ? S::NG : p.k_dim / GS, vg = FULL ? S::NG : p.v_dim / GS;
  const int kw = kg * (GS * KB / 32), vw = vg * (GS * VB / 32);

  // queries: lane (row, q4) holds coordinates GS g + q4 GS / 4 .. of every group
  u32x4_t qop[S::NG][S::CH];
  float qsum[S::NG], row_scale;
  {
    const uint16_t* q = static_cast<const uint16_t*>(p.q) + b * p.q_sb + (static_cast<int64_t>(h) * p.R + q_r) * p.q_sh +
                        static_cast<int64_t>(q_l) * p.q_sl;
    uint4 raw[S::NG][S::CH];
    float big = 0.f;
#pragma unroll
    for (int g = 0; g < S::NG; ++g)
#pragma unroll
      for (int ch = 0; ch < S::CH; ++ch) {
        raw[g][ch] = make_uint4(0, 0, 0, 0);
        if (FULL || g < kg) raw[g][ch] = *reinterpret_cast<const uint4*>(q + g * GS + q4 * (GS / 4) + ch * 8);
        const uint32_t w[4] = {raw[g][ch].x, raw[g][ch].y, raw[g][ch].z, raw[g][ch].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 t = pair16<DT>(w[j]);
          big = fmaxf(big, fmaxf(fabsf(t.x), fabsf(t.y)));
        }
      }
    big = fmaxf(big, __shfl_xor(big, 16));
    big = fmaxf(big, __shfl_xor(big, 32));
    // 2^up takes the row's largest magnitude to [2^13, 2^14); exponents clamped so that both factors stay normal
    const int up = min(max(13 - (static_cast<int>(__float_as_uint(big) >> 23) - 127), -113), 113);
    // (a negative scale turns the queries' signs, so that the largest product has the largest score)
    const float scale_up = __uint_as_float((p.scale < 0.f ? 0x80000000u : 0u) | (static_cast<uint32_t>(127 + up) << 23));
    row_scale = fabsf(p.scale) * __uint_as_float(static_cast<uint32_t>(127 - up) << 23);
#pragma unroll
    for (int g = 0; g < S::NG; ++g) {
      float sum = 0.f;
#pragma unroll
      for (int ch = 0; ch < S::CH; ++ch) {
        const uint32_t w[4] = {raw[g][ch].x, raw[g][ch].y, raw[g][ch].z, raw[g][ch].w};
        _Float16 f[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 t = pair16<DT>(w[j]);
          f[2 * j] = static_cast<_Float16>(t.x * scale_up), f[2 * j + 1] = static_cast<_Float16>(t.y * scale_up);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) sum += static_cast<float>(f[j]);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const f16x2_t two = {f[KB == 4 ? r : 2 * r], f[KB == 4 ? r + 4 : 2 * r + 1]};
          qop[g][ch][r] = __builtin_bit_cast(uint32_t, two);
        }
      }
      sum += __shfl_xor(sum, 16);
      sum += __shfl_xor(sum, 32);
      qsum[g] = sum;
    }
  }

  const uint32_t key_mask = held_scalar(0x00f000f0u), key_with = held_vector(0x54005400u);
  const uint32_t value_mask = held_scalar(0x000f000fu), value_with = held_vector(0x43004300u);
  int64_t start64, end64;
  affine_range(p, b, start64, end64);
  const int end = static_cast<int>(end64);
  int s0 = static_cast<int>(min(start64 + split * p.split_tokens, end64));
  int s1 = static_cast<int>(min(end64, s0 + p.split_tokens));
  if (MASK && p.keep.range) {  // a split of the tokens that any of these rows sees
    const int64_t at = ((static_cast<int64_t>(p.keep.nb > 1 ? b : 0) * p.keep.ng + (p.keep.ng > 1 ? h : 0)) * p.keep.nr +
                        (p.keep.nr > 1 ? q_r : 0)) * p.keep.nl + (p.keep.nl > 1 ? q_l : 0);
    int2 t = p.keep.range[at];
#pragma unroll
    for (int m = 1; m < 16; m *= 2) t = make_int2(min(t.x, __shfl_xor(t.x, m)), max(t.y, __shfl_xor(t.y, m)));
    const int first = __builtin_amdgcn_readfirstlane(t.x), stop = __builtin_amdgcn_readfirstlane(t.y);
    const int part = (stop - first + p.splits - 1) / p.splits;
    s0 = first + static_cast<int>(min(static_cast<int64_t>(split) * part, static_cast<int64_t>(stop - first)));
    s1 = min(stop, s0 + part);
  }
  const int lim = p.causal ? end - p.L + q_l : INT32_MAX;
  const int lim_min = p.causal ? end - p.L + row0 / p.R : INT32_MAX;
  // this wave's part of the slab, whole steps
  const int per = ((s1 - s0 + S::WAVES * S::STEP - 1) / (S::WAVES * S::STEP)) * S::STEP;
  const int t0 = s0 + min(wave * per, s1 - s0);
  const int t1 = min(s1, t0 + per);
  const int64_t base = static_cast<int64_t>(bh) * p.capacity;
  const int64_t mask_at = MASK ? b * p.mask_s[0] + h * p.mask_s[1] + q_r * p.mask_s[2] + q_l * p.mask_s[3] : 0;

  float m = -INFINITY, ref = 0.f, l = 0.f;
  f32x4_t acc[S::NS][S::NA][S::UD];
  f32x4_t extra[S::NS][S::NA];  // 128 times the weights' sum, which 4-bit codes bring in
  float corr[S::NS][S::NA];
#pragma unroll
  for (int s = 0; s < S::NS; ++s)
#pragma unroll
    for (int a = 0; a < S::NA; ++a) {
      corr[s][a] = 0.f;
      extra[s][a] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int r = 0; r < S::UD; ++r) acc[s][a][r] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    }

  // One step's codes and pairs.  Each part of the next step loads as soon as this step's is used up.  Addresses: a
  // uniform base of the tile's first token and a 32-bit offset of the lane's, which a whole step leaves alone; the last
  // step holds its offsets to tokens that exist.
  // Pairs load a token a lane, a few instructions a step (sixteen lanes want every one of them), and reach the lanes
  // as f32 through LDS, a wave's own: planes [key scales, key biases, value scales, value biases][group][token].
  uint32_t kreg[S::NT][S::NG][S::KW], vreg[S::NS][S::NT][4];
  constexpr int kSides = S::STEP == 64 ? 2 : 1;  // of 32 tokens, half the wave loads keys' pairs and half values'
  uint32_t pairs[kSides][S::NG];
  const uint32_t tok_a = c, tok_b = q4 * 4, tok_p = lane & (S::STEP - 1);
  const bool lane_values = S::STEP == 32 && lane >= 32;
  float* planes = lds + wave * S::PLANES;

  auto load_keys = [&](int t, auto is_whole) {
    constexpr bool whole = decltype(is_whole)::value;
    const uint32_t last = static_cast<uint32_t>(min(t1 - t, S::STEP)) - 1;
#pragma unroll
    for (int n = 0; n < S::NT; ++n) {
      const uint32_t* from = p.k_codes + (base + t + (whole ? n * 16 : 0)) * kw;
      const uint32_t tok = whole ? tok_a : min(n * 16 + tok_a, last);
#pragma unroll
      for (int g = 0; g < S::NG; ++g) {
        const uint32_t* group = from + (FULL ? g : min(g, kg - 1)) * (GS * KB / 32);
        const uint32_t at = tok * (kw * 4) + q4 * (S::KW * 4);
        if constexpr (S::KW == 1) {
          kreg[n][g][0] = load_at<uint32_t>(group, at);
        } else if constexpr (S::KW == 2) {
          const uint2 u = load_at<uint2>(group, at);
          kreg[n][g][0] = u.x, kreg[n][g][1] = u.y;
        } else {
#pragma unroll
          for (int i = 0; i < S::KW; i += 4) {
            const uint4 u = load_at<uint4>(group + i, at);
            kreg[n][g][i] = u.x, kreg[n][g][i + 1] = u.y, kreg[n][g][i + 2] = u.z, kreg[n][g][i + 3] = u.w;
          }
        }
      }
    }
  };
  auto load_pairs = [&](int t, auto is_whole) {
    constexpr bool whole = decltype(is_whole)::value;
    const uint32_t last = static_cast<uint32_t>(min(t1 - t, S::STEP)) - 1;
    const uint32_t tok = whole ? tok_p : min(tok_p, last);
#pragma unroll
    for (int side = 0; side < kSides; ++side) {
      const bool values = kSides == 2 ? side == 1 : lane_values;
      const int groups = values ? vg : kg;
      const uint32_t* from = static_cast<const uint32_t*>(values ? p.v_params : p.k_params) + (base + t) * groups;
      if constexpr (FULL && S::NG % 4 == 0) {
#pragma unroll
        for (int g = 0; g < S::NG; g += 4) {
          const u32x4_a4 w = load_at<u32x4_a4>(from + g, tok * (groups * 4));
#pragma unroll
          for (int i = 0; i < 4; ++i) pairs[side][g + i] = w[i];
        }
      } else if constexpr (FULL && S::NG == 2) {
        const u32x2_a4 w = load_at<u32x2_a4>(from, tok * (groups * 4));
        pairs[side][0] = w[0], pairs[side][1] = w[1];
      } else {
#pragma unroll
        for (int g = 0; g < S::NG; ++g)
          pairs[side][g] = load_at<uint32_t>(from + (FULL ? g : min(g, groups - 1)), tok * (groups * 4));
      }
    }
  };
  // the loaded pairs into LDS; whether a value's pair is not finite
  auto place_pairs = [&]() -> bool {
    bool odd = false;
#pragma unroll
    for (int side = 0; side < kSides; ++side) {
      float* to = planes + (kSides == 2 ? side : lane_values ? 1 : 0) * 2 * S::NG * S::STEP + tok_p;
#pragma unroll
      for (int g = 0; g < S::NG; ++g) {
        const float2 sb = pair16<DT>(pairs[side][g]);
        to[g * S::STEP] = sb.x;
        // keys: less what their codes enter with
        const bool key = kSides == 2 ? side == 0 : !lane_values;
        to[(S::NG + g) * S::STEP] = key ? __builtin_fmaf(-S::OFF, sb.x, sb.y) : sb.y;
        if (kSides == 1 || side == 1) odd |= !(fabsf(sb.x) < INFINITY) || !(fabsf(sb.y) < INFINITY);
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    return __any(odd);
  };
  auto plane4 = [&](int plane, int g, int tile) {  // of tokens 4 q4 .. 4 q4 + 3 of a tile
    return *reinterpret_cast<const float4*>(planes + (plane * S::NG + g) * S::STEP + tile * 16 + q4 * 4);
  };
  auto load_values = [&](int t, auto is_whole) {
    constexpr bool whole = decltype(is_whole)::value;
    const uint32_t last = static_cast<uint32_t>(min(t1 - t, S::STEP)) - 1;
#pragma unroll
    for (int n = 0; n < S::NT; ++n)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t* from = p.v_codes + (base + t + (whole ? n * 16 + j : 0)) * vw;
        const uint32_t tok = whole ? tok_b : min(n * 16 + j + tok_b, last);
#pragma unroll
        for (int s = 0; s < S::NS; ++s) {
          constexpr int kBytes = S::UD * VB / 8;  // of a lane's part of a row
          const uint32_t part = FULL ? c * kBytes : min((s * 16 + c) * kBytes, vw * 4 - kBytes);
          const char* set = reinterpret_cast<const char*>(from) + (FULL ? s * 16 * kBytes : 0);
          if constexpr (kBytes == 2)
            vreg[s][n][j] = load_at<uint16_t>(set, tok * (vw * 4) + part);
          else
            vreg[s][n][j] = load_at<uint32_t>(set, tok * (vw * 4) + part);
        }
      }
  };

  // load(t) of a whole step or of the last.  Past the end it loads the last token again: both ways issue the same loads,
  // so that what waits for this step's loads may leave the next one's on their way.
  auto step_of = [&](int t, auto&& load) {
    if (t + S::STEP <= t1)
      load(t, std::true_type{});
    else
      load(min(t, t1 - 1), std::false_type{});
  };

  if (t0 < t1) {
    step_of(t0, load_pairs);
    step_of(t0, load_keys);
    step_of(t0, load_values);
  }

  for (int t = t0; t < t1; t += S::STEP) {
    const int next = t + S::STEP;
    __builtin_amdgcn_wave_barrier();  // the pairs of the step before have been read
    const bool odd = place_pairs();
    step_of(next, load_pairs);
    // scores; each lane keeps those of its own block of tokens
    float x[S::NU][4];
#pragma unroll
    for (int u = 0; u < S::NU; ++u) {
      f32x4_t dot[S::NG];
#pragma unroll
      for (int i = 0; i < S::TI; ++i)
#pragma unroll
        for (int g = 0; g < S::NG; ++g) {
          f32x4_t C = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int ch = 0; ch < S::CH; ++ch)
            C = mfma_f16(key_operand<KB>(&kreg[u * S::TI + i][g][ch * (KB / 4)], key_mask, key_with), qop[g][ch], C);
          if (i == 0) {
            dot[g] = C;
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) dot[g][j] = i_l == i ? C[j] : dot[g][j];
          }
        }
#pragma unroll
      for (int j = 0; j < 4; ++j) x[u][j] = 0.f;
#pragma unroll
      for (int g = 0; g < S::NG; ++g) {
        const float4 sc = plane4(0, g, u * S::TI + i_l), bi = plane4(1, g, u * S::TI + i_l);
        const float s4[4] = {sc.x, sc.y, sc.z, sc.w}, b4[4] = {bi.x, bi.y, bi.z, bi.w};
#pragma unroll
        for (int j = 0; j < 4; ++j)
          x[u][j] = __builtin_fmaf(s4[j], dot[g][j], __builtin_fmaf(b4[j], qsum[g], x[u][j]));
      }
    }
    step_of(next, load_keys);
    // scores are x times `unit`
    float unit = row_scale;
    if (MASK || t + S::STEP - 1 > lim_min || t + S::STEP > t1) {
      unit = 1.f;
#pragma unroll
      for (int u = 0; u < S::NU; ++u)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int tok = t + (u * S::TI + i_l) * 16 + q4 * 4 + j;
          float y = x[u][j] * row_scale;
          if constexpr (MASK) y = affine_mask(p, mask_at + min(tok, t1 - 1) * p.mask_s[4], y);
          if (tok > lim && y != -INFINITY) y = -FLT_MAX;
          if (tok >= t1) y = -INFINITY;
          x[u][j] = y;
        }
    }
    float top = -INFINITY;
#pragma unroll
    for (int u = 0; u < S::NU; ++u)
#pragma unroll
      for (int j = 0; j < 4; ++j) top = fmaxf(top, x[u][j]);
    top *= unit;
    if (__any(top > m + 8.f)) {
      top = fmaxf(top, __shfl_xor(top, 16));
      top = fmaxf(top, __shfl_xor(top, 32));
#pragma unroll
      for (int o = RPT; o < RPT * S::TI; o *= 2) top = fmaxf(top, __shfl_xor(top, o));
      const float to = fmaxf(m, top);
      const float ref_to = to == -INFINITY ? 0.f : to;
      const float a = __builtin_amdgcn_exp2f(m - ref_to);
      m = to, ref = ref_to;
      l *= a;
      float ar[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) ar[j] = __shfl(a, (q4 * 4 + j) % RPT);
#pragma unroll
      for (int s = 0; s < S::NS; ++s)
#pragma unroll
        for (int k = 0; k < S::NA; ++k) {
          corr[s][k] *= a;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            extra[s][k][j] *= ar[j];
#pragma unroll
            for (int r = 0; r < S::UD; ++r) acc[s][k][r][j] *= ar[j];
          }
        }
    }
    uint32_t ps[S::NS][S::NA][S::NP][S::NU][2];
#pragma unroll
    for (int u = 0; u < S::NU; ++u) {
      float w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        w[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[u][j], unit, -ref));
        l += w[j];
      }
#pragma unroll
      for (int s = 0; s < S::NS; ++s)
#pragma unroll
        for (int a = 0; a < S::NA; ++a) {
          const int g = s * S::SETD / GS + a * S::GA + g_l;
          const float4 sc = plane4(2, g, u * S::TI + i_l), bi = plane4(3, g, u * S::TI + i_l);
          float s4[4] = {sc.x, sc.y, sc.z, sc.w}, b4[4] = {bi.x, bi.y, bi.z, bi.w};
          if (odd) {  // what a row masks may be NaN
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              s4[j] = w[j] == 0.f ? 0.f : s4[j];
              b4[j] = w[j] == 0.f ? 0.f : b4[j];
            }
          }
          float v[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            v[j] = w[j] * s4[j];
            corr[s][a] = __builtin_fmaf(w[j], b4[j], corr[s][a]);
          }
#pragma unroll
          for (int j = 0; j < 4; j += 2) {
            float lo = v[j], hi = v[j + 1];
#pragma unroll
            for (int n = 0; n < S::NP; ++n) {
              const bf16x2_t two = {static_cast<__bf16>(lo), static_cast<__bf16>(hi)};
              const uint32_t bits = __builtin_bit_cast(uint32_t, two);
              ps[s][a][n][u][j / 2] = bits;
              lo -= __uint_as_float(bits << 16), hi -= __uint_as_float(bits & 0xffff0000u);
            }
          }
        }
    }
    // values, two tiles (32 tokens) a product
#pragma unroll
    for (int s = 0; s < S::NS; ++s) {
#pragma unroll
      for (int pair = 0; pair < S::NT / 2; ++pair) {
        u32x4_t A[S::NA][S::NP];
#pragma unroll
        for (int a = 0; a < S::NA; ++a)
#pragma unroll
          for (int n = 0; n < S::NP; ++n)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              const int tile = 2 * pair + half;
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                const uint32_t bits = ps[s][a][n][tile / S::TI][j];
                A[a][n][2 * half + j] = S::TI == 1 || i_l == tile % S::TI ? bits : 0u;
              }
            }
        if constexpr (VB == 4) {
          const u32x4_t b128 = {0x43004300u, 0x43004300u, 0x43004300u, 0x43004300u};
#pragma unroll
          for (int a = 0; a < S::NA; ++a)
#pragma unroll
            for (int n = 0; n < S::NP; ++n) extra[s][a] = mfma_bf16(A[a][n], b128, extra[s][a]);
        }
        uint32_t w[4][2];  // register j of B: tokens (w[j][0], w[j][1])
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          w[j][0] = vreg[s][2 * pair + j / 2][2 * (j & 1)];
          w[j][1] = vreg[s][2 * pair + j / 2][2 * (j & 1) + 1];
        }
#pragma unroll
        for (int r = 0; r < S::UD; ++r) {
          u32x4_t B;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if constexpr (VB == 4) {
              const uint32_t both = S::UD == 4 ? w[j][0] | (w[j][1] << 16)
                                               : __builtin_amdgcn_perm(w[j][1], w[j][0], r < 4 ? 0x05040100u : 0x07060302u);
              B[j] = ((both >> (4 * (r & 3))) & value_mask) | value_with;
            } else {
              B[j] = top_halves(static_cast<float>((w[j][0] >> (8 * r)) & 0xffu),
                                static_cast<float>((w[j][1] >> (8 * r)) & 0xffu));
            }
          }
#pragma unroll
          for (int a = 0; a < S::NA; ++a)
#pragma unroll
            for (int n = 0; n < S::NP; ++n) acc[s][a][r] = mfma_bf16(A[a][n], B, acc[s][a][r]);
        }
      }
    }
    step_of(next, load_values);
  }

  __syncthreads();  // the planes' LDS is free
  // The wave's sums: l and corr over its lanes of a row, O over the blocks of tokens; then the waves' in LDS.
  l += __shfl_xor(l, 16);
  l += __shfl_xor(l, 32);
#pragma unroll
  for (int o = RPT; o < RPT * S::TI; o *= 2) l += __shfl_xor(l, o);
  float* wave_o = lds + wave * RPT * DP;                                      // [RPT][DP]
  float* wave_c = lds + S::WAVES * RPT * DP + wave * RPT * S::NG;           // [RPT][NG]
  float* ml = lds + S::WAVES * RPT * (DP + S::NG);                          // [waves][RPT][2]
  if (q4 == 0 && c < RPT) {
    ml[(wave * RPT + c) * 2] = m;
    ml[(wave * RPT + c) * 2 + 1] = l;
  }
  const int row_i = (q4 * 4 / RPT) % S::TI;           // C rows 4 q4 + j: block of tokens,
  const int row_g = q4 * 4 / (RPT * S::TI);           // group in the A operand
  const int col_g = c * S::UD / GS;                   // group in the set of this lane's column
#pragma unroll
  for (int s = 0; s < S::NS; ++s)
#pragma unroll
    for (int a = 0; a < S::NA; ++a) {
      float cs = corr[s][a];
      cs += __shfl_xor(cs, 16);
      cs += __shfl_xor(cs, 32);
#pragma unroll
      for (int o = RPT; o < RPT * S::TI; o *= 2) cs += __shfl_xor(cs, o);
      // SETD < GS: several sets share a group, and each holds the whole sum
      if (q4 == 0 && i_l == 0 && (s * S::SETD) % GS < S::SETD)
        wave_c[r_l * S::NG + s * S::SETD / GS + a * S::GA + g_l] = cs;
#pragma unroll
      for (int r = 0; r < S::UD; ++r)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float o = acc[s][a][r][j] - (VB == 4 ? extra[s][a][j] : 0.f);
          if constexpr (S::TI > 1) {
            // blocks of tokens lie RPT rows apart
            o += __shfl_xor(o, RPT == 4 ? 16 : 32);
            if constexpr (S::TI > 2) o += __shfl_xor(o, 32);
          }
          const int rr = (q4 * 4 + j) % RPT;
          if (row_i == 0 && col_g == a * S::GA + row_g) wave_o[rr * DP + s * S::SETD + c * S::UD + r] = o;
        }
    }
  __syncthreads();
  for (int e = tid; e < RPT * DP; e += 64 * S::WAVES) {
    const int rr = e / DP, d = e % DP;
    if (row0 + rr >= p.rows || (!FULL && d >= p.v_dim)) continue;
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < S::WAVES; ++w) M = fmaxf(M, ml[(w * RPT + rr) * 2]);
    const float to = M == -INFINITY ? 0.f : M;
    float sum = 0.f, o = 0.f;
#pragma unroll
    for (int w = 0; w < S::WAVES; ++w) {
      const float a = __builtin_amdgcn_exp2f(ml[(w * RPT + rr) * 2] - to);
      sum = __builtin_fmaf(a, ml[(w * RPT + rr) * 2 + 1], sum);
      const float x = lds[(w * RPT + rr) * DP + d] + lds[S::WAVES * RPT * DP + (w * RPT + rr) * S::NG + d / GS];
      o = a == 0.f ? o : __builtin_fmaf(a, x, o);
    }
    const int row_e = row0 + rr;
    if (p.splits == 1) {
      const int64_t head = static_cast<int64_t>(bh) * p.R + row_e % p.R;
      store_elem<DT>(p.out, (head * p.L + row_e / p.R) * p.v_dim + d, sum == 0.f ? 0.f : o / sum);
    } else {
      const int64_t at = (static_cast<int64_t>(bh) * p.rows + row_e) * p.splits + split;
      p.part_o[at * p.v_dim + d] = o;
      if (d == 0) p.part_ml[2 * at] = M, p.part_ml[2 * at + 1] = sum;
    }
  }
}

// Query rows a workgroup of the larger variant takes: 16, or 8 where 16 would need more than two A operands a set
// (their sums would not fit in the registers).
constexpr int rows_large(int DP, int GS) { return DP == 256 && GS == 32 ? 8 : 16; }

template <int DT, int KB, int VB, int DP, int GS, int RPT, bool FULL, bool MASK>
int launch_rows_of(const AffineAttnParams& p, hipStream_t st) {
  const int64_t blocks = static_cast<int64_t>(p.B) * p.Hkv * ((p.rows + RPT - 1) / RPT) * p.splits;
  if (blocks > INT32_MAX / 512) return fail(TQ_ERR_UNSUPPORTED, "tq_attention_affine: %lld workgroups", static_cast<long long>(blocks));
  affine_rows_kernel<DT, KB, VB, DP, GS, RPT, FULL, MASK>
      <<<static_cast<unsigned>(blocks), 64 * RowsShape<KB, VB, DP, GS, RPT>::WAVES, 0, st>>>(p);
  return check_launch("affine_rows_kernel");
}

template <int DT, int KB, int VB, int DP, int GS, bool FULL>
int launch_rows_at(const AffineAttnParams& p, int rpt, hipStream_t st) {
  constexpr int kLarge = rows_large(DP, GS);
  if constexpr (!FULL) {
    if constexpr (GS <= 64) {
      if (p.mask_kind != TQ_MASK_NONE && rpt == 4) return launch_rows_of<DT, KB, VB, DP, GS, 4, false, true>(p, st);
    }
    if (p.mask_kind != TQ_MASK_NONE) return launch_rows_of<DT, KB, VB, DP, GS, kLarge, false, true>(p, st);
  }
  if constexpr (GS <= 64) {
    if (rpt == 4) return launch_rows_of<DT, KB, VB, DP, GS, 4, FULL, false>(p, st);
  }
  return launch_rows_of<DT, KB, VB, DP, GS, kLarge, FULL, false>(p, st);
}

template <int DT, int KB, int VB>
int launch_rows_bits(const AffineAttnParams& p, const RowsChoice& r, hipStream_t st) {
  if (r.full && r.dim == 64 && p.group == 32) return launch_rows_at<DT, KB, VB, 64, 32, true>(p, r.rows, st);
  if (r.full && r.dim == 64) return launch_rows_at<DT, KB, VB, 64, 64, true>(p, r.rows, st);
  if (r.full && r.dim == 128 && p.group == 32) return launch_rows_at<DT, KB, VB, 128, 32, true>(p, r.rows, st);
  if (r.full && r.dim == 128) return launch_rows_at<DT, KB, VB, 128, 64, true>(p, r.rows, st);
  if (r.full && p.group == 32) return launch_rows_at<DT, KB, VB, 256, 32, true>(p, r.rows, st);
  if (r.full) return launch_rows_at<DT, KB, VB, 256, 64, true>(p, r.rows, st);
  if (r.dim == 128 && p.group == 32) return launch_rows_at<DT, KB, VB, 128, 32, false>(p, r.rows, st);
  if (r.dim == 128 && p.group == 64) return launch_rows_at<DT, KB, VB, 128, 64, false>(p, r.rows, st);
  if (r.dim == 128) return launch_rows_at<DT, KB, VB, 128, 128, false>(p, r.rows, st);
  if (p.group == 32) return launch_rows_at<DT, KB, VB, 256, 32, false>(p, r.rows, st);
  if (p.group == 64) return launch_rows_at<DT, KB, VB, 256, 64, false>(p, r.rows, st);
  return launch_rows_at<DT, KB, VB, 256, 128, false>(p, r.rows, st);
}

}  // namespace tq
