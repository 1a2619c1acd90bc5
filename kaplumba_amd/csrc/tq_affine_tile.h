// Attention of many query rows (prefill chunks) over the group-affine cache, on the matrix cores.
//
// A workgroup takes 8 waves x RT x 16 query rows of one kv head.  Every 64 tokens it decodes keys and values into LDS
// once for all of them, as f16 (scale * code + bias in f32, rounded once), half the waves the keys and half the values,
// while the tile before is worked on:
//   scores  C[token][row] = K Q^T (v_mfma_f32_16x16x32_f16), keys row by row in LDS, queries in registers, each row
//           times a power of two.
//   values  O[row][coordinate] = P V: C's lanes hold row = lane % 16 and tokens 4 (lane / 16) + j of every 16-token
//           tile, which is A's layout when 32 tokens are taken in the order (lane / 16, tile, j); values lie in LDS
//           transposed and in that order, so weights go from C to A in registers, and the sum of a row's rounded
//           weights is one more product with ones.
// Softmax: one reference a row, moved only when a score passes it by 8 (base 2).  Weights go in as one f16 (off by 2^-11
// of themselves, by 2^-25 below 2^-14; of f16 vectors up to 2^15, of bf16 ones up to 2^8, so that large values times
// weights stay finite); they are divided by the sum of the same rounded numbers.
// f16 and not the vectors' own type where that is bf16: eight times smaller errors of keys, weights and values.
// Outputs of 512 bf16 queries over 8192 tokens are then as far from 64 bits as their own rounding (0.0017, against
// 0.0036 with bf16 operands, 4 us faster); f16 outputs are 0.0005 off where rounding alone is 0.0002.  Exact codes in
// the products with the pairs in f32 behind them, as few rows have it, take more registers than there are (275 us
// instead of 109).
//
// What f16 does not hold (NaN, infinite, past 65504; bf16 groups below 2^-15, where f16's spacing near zero is coarser
// than bf16's own) is zeros in LDS and a flag for the token: its scores, or its values for the rows that weigh it, are
// worked out in f32 from the codes, one token at a time.  What a row masks may so be NaN.
//
// What bounds it, d = 128, a step of 64 tokens and 256 rows a CU: matrix products 2048 cycles, LDS reads 2048, vector
// instructions about 2400 a SIMD (softmax 7 a score, decoding 3 an element).
#pragma once

#include "tq_affine.h"
#include "tq_pieces.h"

namespace tq {

constexpr int kTileWaves = 8;
constexpr int kTileStep = 64;  // tokens in LDS at a time

template <int KS, int CT>
struct TileShape {
  static constexpr int DK = 32 * KS, DV = 16 * CT;
  static constexpr int RT = KS <= 4 && CT <= 8 ? 2 : 1;  // 16-row tiles a wave
  static constexpr int ROWS = kTileWaves * 16 * RT;
  // 16-byte pieces in LDS.  Sixteen lanes read one piece of sixteen rows, four pieces at once; a read is served in groups
  // of lanes that mix rows and pieces, so a piece's place is its number xor the row's (or half the row's, where two
  // rows span the banks): any such group then meets every bank once.  Rows of 12 or 24 pieces are padded instead.
  static constexpr bool SWIZZLE = KS == 2 || KS == 4 || KS == 8;
  static constexpr int KROW = DK + (SWIZZLE ? 0 : 8);  // 16-bit elements of a token's row of keys
  static constexpr int VROW = kTileStep;               // of a coordinate's row of values
  static constexpr int KBUF = kTileStep * KROW, VBUF = DV * VROW;
  __device__ static __forceinline__ int k_at(int tok, int piece) {
    const int place = !SWIZZLE ? piece : KS == 2 ? piece ^ ((tok >> 1) & 7) : piece ^ (tok & 15);
    return tok * KROW + place * 8;
  }
  __device__ static __forceinline__ int v_at(int d, int piece) { return d * VROW + (piece ^ ((d >> 1) & 7)) * 8; }
  static constexpr int KU = KS;                // 8-coordinate pieces of keys a decoding thread has (256 threads)
  static constexpr int VU = (CT + 7) / 8;      // (4 tokens x 8 coordinates) units of values
};

typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));

__device__ __forceinline__ f32x4_t mfma_of(u32x4_t a, u32x4_t b, f32x4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0,
                                                0);
}

// Two f32 as f16, to nearest even.
__device__ __forceinline__ uint32_t pack_of(float lo, float hi) {
  const f16x2_t t = {static_cast<_Float16>(lo), static_cast<_Float16>(hi)};
  return __builtin_bit_cast(uint32_t, t);
}

// Eight codes as f32: one word of 4-bit codes or two of 8-bit ones.
template <int BITS>
__device__ __forceinline__ void codes_f32(const uint32_t* w, float (&f)[8]) {
  if constexpr (BITS == 4) {
    const uint32_t even = w[0] & 0x0f0f0f0fu, odd = (w[0] >> 4) & 0x0f0f0f0fu;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      f[2 * j] = static_cast<float>((even >> (8 * j)) & 0xffu);
      f[2 * j + 1] = static_cast<float>((odd >> (8 * j)) & 0xffu);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = static_cast<float>((w[j >> 2] >> (8 * (j & 3))) & 0xffu);
  }
}

// Whether a group's values scale * code + bias go in as f16: finite numbers of it, and its spacing near zero (2^-24)
// no more than bf16's own at the group's largest.
template <int DT, int BITS>
__device__ __forceinline__ bool fits_f16(float2 sb) {
  const float most = fabsf(sb.y) + static_cast<float>((1 << BITS) - 1) * fabsf(sb.x);
  if (DT == TQ_DTYPE_BF16 && most < 0x1p-15f) return most == 0.f;
  return most <= 65504.f;  // false for NaN
}

template <int DT, int KB, int VB, int KS, int CT, bool MASK>
__global__ __launch_bounds__(64 * kTileWaves) void affine_tile_kernel(const AffineAttnParams p) {
  using S = TileShape<KS, CT>;
  constexpr int RT = S::RT;
  __shared__ __attribute__((aligned(16))) uint16_t k_lds[2][S::KBUF];
  __shared__ __attribute__((aligned(16))) uint16_t v_lds[2][S::VBUF];
  __shared__ __attribute__((aligned(16))) uint32_t odd_lds[3][4];  // three steps' tokens whose keys, and values, f16 lacks
  __shared__ int range_lds[2];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 15, q4 = lane >> 4;
  const int row_blocks = (p.rows + S::ROWS - 1) / S::ROWS;
  const int split = blockIdx.x % p.splits;
  const int blk = blockIdx.x / p.splits;
  const int bh = blk / row_blocks, block_row0 = (blk % row_blocks) * S::ROWS;
  const int b = bh / p.Hkv, h = bh % p.Hkv;
  const int row0 = block_row0 + wave * 16 * RT;

  int64_t start, end;
  affine_range(p, b, start, end);

  // tokens that any row of this workgroup sees
  int first = static_cast<int>(start), stop = static_cast<int>(end);
  if constexpr (MASK) {
    if (tid == 0) range_lds[0] = stop, range_lds[1] = first;
    __syncthreads();
    int lo = stop, hi = first;
    for (int i = tid; i < S::ROWS; i += 64 * kTileWaves) {
      const int row = min(block_row0 + i, p.rows - 1);
      const int l = row / p.R, r = row % p.R;
      const int64_t at = ((static_cast<int64_t>(p.keep.nb > 1 ? b : 0) * p.keep.ng + (p.keep.ng > 1 ? h : 0)) * p.keep.nr +
                          (p.keep.nr > 1 ? r : 0)) * p.keep.nl + (p.keep.nl > 1 ? l : 0);
      const int2 t = p.keep.range[at];
      lo = min(lo, t.x), hi = max(hi, t.y);
    }
    atomicMin(&range_lds[0], lo);
    atomicMax(&range_lds[1], hi);
    __syncthreads();
    first = range_lds[0], stop = range_lds[1];
  } else if (p.causal) {
    const int l_lo = block_row0 / p.R, l_hi = (min(block_row0 + S::ROWS, p.rows) - 1) / p.R;
    if (end - p.L + l_lo >= start) stop = static_cast<int>(end - p.L + l_hi + 1);
  }
  const int per = ((stop - first + p.splits - 1) / p.splits + kTileStep - 1) / kTileStep * kTileStep;
  const int t0 = first + min(static_cast<int64_t>(split) * per, static_cast<int64_t>(stop - first));
  const int t1 = min(stop, t0 + per);

  // this lane's query rows, as columns of C
  u32x4_t qop[RT][KS];
  float unit[RT];  // scores are this times the products
  int lim[RT];
  int64_t mask_at[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int row = min(row0 + rt * 16 + c, p.rows - 1);
    const int l = row / p.R, r = row % p.R;
    const uint16_t* q = static_cast<const uint16_t*>(p.q) + b * p.q_sb + (static_cast<int64_t>(h) * p.R + r) * p.q_sh +
                        static_cast<int64_t>(l) * p.q_sl;
    // times the power of two that takes the row's largest magnitude to [1, 2): coordinates over 2^-14 of it keep all
    // their bits, smaller ones are off by 2^-25 of it at most.  A negative scale turns the signs, so that the largest
    // product has the largest score.  Exponents are clamped so that both factors stay normal.
    float big = 0.f;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const uint4 u = *reinterpret_cast<const uint4*>(q + s * 32 + q4 * 8);
      qop[rt][s] = u32x4_t{u.x, u.y, u.z, u.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 two = pair16<DT>(qop[rt][s][j]);
        big = fmaxf(big, fmaxf(fabsf(two.x), fabsf(two.y)));
      }
    }
    big = fmaxf(big, __shfl_xor(big, 16));
    big = fmaxf(big, __shfl_xor(big, 32));
    const int up = min(max(127 - static_cast<int>(__float_as_uint(big) >> 23), -113), 113);
    const float lift =
        __uint_as_float((p.scale < 0.f ? 0x80000000u : 0u) | (static_cast<uint32_t>(127 + up) << 23));
    unit[rt] = fabsf(p.scale) * __uint_as_float(static_cast<uint32_t>(127 - up) << 23);
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 two = pair16<DT>(qop[rt][s][j]);
        qop[rt][s][j] = pack_of(two.x * lift, two.y * lift);
      }
    lim[rt] = p.causal ? static_cast<int>(end) - p.L + l : INT32_MAX;
    mask_at[rt] = MASK ? b * p.mask_s[0] + h * p.mask_s[1] + r * p.mask_s[2] + l * p.mask_s[3] : 0;
  }
  const bool quads = MASK && p.mask_kind == TQ_MASK_BOOL && p.mask_s[4] == 1;
  // the causal rule leaves a step of tokens alone when its last one is within the first row's limit
  const int lim_min = p.causal ? static_cast<int>(end) - p.L + row0 / p.R : INT32_MAX;

  float m[RT], ref[RT];
  f32x4_t acc[RT][CT], sum[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    m[rt] = -INFINITY, ref[rt] = 0.f;
    sum[rt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int n = 0; n < CT; ++n) acc[rt][n] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }

  // ---- decoding: waves 0..3 keys, 4..7 values
  const bool keys = wave < kTileWaves / 2;
  const int dtid = tid & 255;
  const int64_t base = static_cast<int64_t>(bh) * p.capacity;
  const int shift = p.group == 32 ? 2 : p.group == 64 ? 3 : 4;  // 8-coordinate pieces a group
  constexpr int KWORDS = KB / 4, VWORDS = VB / 4;
  constexpr int KREGS = S::KU * (KWORDS + 1), VREGS = S::VU * 4 * (VWORDS + 1);
  uint32_t raw[KREGS > VREGS ? KREGS : VREGS];

  // The thread's number within its half, by a way that the compiler does not look through: it would keep every address
  // made from it for the whole loop, past what the registers hold, and fetching one back from scratch memory waits for
  // all codes on their way.
  auto half_id = [&]() {
    uint32_t id = dtid;
    asm volatile("" : "+v"(id));
    return id;
  };

  auto load = [&](int t) {
    const int last = min(t1 - t, kTileStep) - 1;
    const uint32_t id = half_id();
    if (keys) {
      const uint32_t* codes = p.k_codes + (base + t) * (S::DK * KB / 32);
      const uint32_t* pairs = static_cast<const uint32_t*>(p.k_params) + (base + t) * (S::DK >> (shift + 3));
#pragma unroll
      for (int i = 0; i < S::KU; ++i) {
        const uint32_t unit = i * 256 + id;
        const uint32_t tok = min(static_cast<int>(unit / (KS * 4)), last), piece = unit % (KS * 4);
        const uint32_t at = (tok * (S::DK * KB / 32) + piece * KWORDS) * 4;
        if constexpr (KWORDS == 1) {
          raw[i * 2] = load_at<uint32_t>(codes, at);
        } else {
          const uint2 u = load_at<uint2>(codes, at);
          raw[i * 3] = u.x, raw[i * 3 + 1] = u.y;
        }
        raw[i * (KWORDS + 1) + KWORDS] = load_at<uint32_t>(pairs, (tok * (S::DK >> (shift + 3)) + (piece >> shift)) * 4);
      }
    } else {
      const uint32_t* codes = p.v_codes + (base + t) * (S::DV * VB / 32);
      const uint32_t* pairs = static_cast<const uint32_t*>(p.v_params) + (base + t) * (S::DV >> (shift + 3));
#pragma unroll
      for (int i = 0; i < S::VU; ++i) {
        const uint32_t unit = i * 256 + id;
        const uint32_t quad = unit % 16, piece = min(unit / 16, static_cast<uint32_t>(CT * 2 - 1));
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t tok = min(static_cast<int>(quad * 4 + j), last);
          const uint32_t at = (tok * (S::DV * VB / 32) + piece * VWORDS) * 4;
          uint32_t* to = raw + (i * 4 + j) * (VWORDS + 1);
          if constexpr (VWORDS == 1) {
            to[0] = load_at<uint32_t>(codes, at);
          } else {
            const uint2 u = load_at<uint2>(codes, at);
            to[0] = u.x, to[1] = u.y;
          }
          to[VWORDS] = load_at<uint32_t>(pairs, (tok * (S::DV >> (shift + 3)) + (piece >> shift)) * 4);
        }
      }
    }
  };

  auto decode_keys = [&](int buf, int flags) {
    const uint32_t id = half_id();
    {
#pragma unroll
      for (int i = 0; i < S::KU; ++i) {
        const uint32_t unit = i * 256 + id;
        const uint32_t tok = unit / (KS * 4), piece = unit % (KS * 4);
        const uint32_t* w = raw + i * (KWORDS + 1);
        float2 sb = pair16<DT>(w[KWORDS]);
        if (!fits_f16<DT, KB>(sb)) {
          atomicOr(&odd_lds[flags][tok >> 5], 1u << (tok & 31));
          sb = make_float2(0.f, 0.f);
        }
        float f[8];
        codes_f32<KB>(w, f);
        u32x4_t o;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          o[j] = pack_of(__builtin_fmaf(sb.x, f[2 * j], sb.y), __builtin_fmaf(sb.x, f[2 * j + 1], sb.y));
        *reinterpret_cast<u32x4_t*>(&k_lds[buf][S::k_at(tok, piece)]) = o;
      }
    }
  };
  auto decode_values = [&](int buf, int flags) {
    const uint32_t id = half_id();
    {
#pragma unroll
      for (int i = 0; i < S::VU; ++i) {
        const uint32_t unit = i * 256 + id;
        const uint32_t quad = unit % 16, piece = unit / 16;
        if (piece >= CT * 2) break;
        float v[4][8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t* w = raw + (i * 4 + j) * (VWORDS + 1);
          float2 sb = pair16<DT>(w[VWORDS]);
          if (!fits_f16<DT, VB>(sb)) {
            atomicOr(&odd_lds[flags][2 + (quad >> 3)], 1u << ((quad * 4 + j) & 31));
            sb = make_float2(0.f, 0.f);
          }
          codes_f32<VB>(w, v[j]);
#pragma unroll
          for (int e = 0; e < 8; ++e) v[j][e] = __builtin_fmaf(sb.x, v[j][e], sb.y);
        }
        // tokens 4 quad + j: 32 (quad / 8) + 8 (quad % 4) + 4 (quad / 4 % 2) + j in the order of A's k indices
        const uint32_t pos = (quad >> 3) * 32 + (quad & 3) * 8 + ((quad >> 2) & 1) * 4;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint2 two = make_uint2(pack_of(v[0][e], v[1][e]), pack_of(v[2][e], v[3][e]));
          *reinterpret_cast<uint2*>(&v_lds[buf][S::v_at(piece * 8 + e, pos >> 3) + (pos & 4)]) = two;
        }
      }
    }
  };

  if (tid < 12) odd_lds[tid >> 2][tid & 3] = 0;
  __syncthreads();
  if (t0 < t1) {
    load(t0);
    if (keys)
      decode_keys(0, 0);
    else
      decode_values(0, 0);
    if (t0 + kTileStep < t1) load(t0 + kTileStep);
  }
  __syncthreads();

  int buf = 0, flags = 0;  // flags: a step's, the next's (written now) and the one after (cleared now)
  for (int t = t0; t < t1; t += kTileStep, buf ^= 1, flags = flags == 2 ? 0 : flags + 1) {
    const bool more = t + kTileStep < t1;
    // four tokens' bytes of a contiguous boolean mask, on their way while the scores are computed
    uint32_t quad[RT][4] = {};
    const bool by_quads = quads && t + kTileStep <= t1;
    if (MASK && by_quads) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int ti = 0; ti < 4; ++ti)
          __builtin_memcpy(&quad[rt][ti], static_cast<const uint8_t*>(p.mask) + mask_at[rt] + t + ti * 16 + q4 * 4, 4);
    }
    // The next tile goes into the other half of LDS, and its successor's codes on their way: the waves of the values do
    // it here, the waves of the keys at the end, so that of a SIMD's two waves one is at vector work while the other is
    // at matrix work all through the step.
    if (tid < 4) odd_lds[flags == 0 ? 2 : flags - 1][tid] = 0;
    if (!keys && more) decode_values(buf ^ 1, flags == 2 ? 0 : flags + 1);
    if (!MASK && !keys && t + 2 * kTileStep < t1) load(t + 2 * kTileStep);
    const u32x4_t odd_of = *reinterpret_cast<const u32x4_t*>(odd_lds[flags]);
    auto odd_tokens = [&](int at) {  // the same for all lanes
      const uint32_t lo = __builtin_amdgcn_readfirstlane(odd_of[at]), hi = __builtin_amdgcn_readfirstlane(odd_of[at + 1]);
      return static_cast<uint64_t>(hi) << 32 | lo;
    };
    // ---- scores
    // operands a tile ahead of the products: a read of LDS takes longer than the products of the one before
    f32x4_t C[RT][4];
    u32x4_t kop[2][KS];
    auto read_keys = [&](int ti) {
#pragma unroll
      for (int s = 0; s < KS; ++s)
        kop[ti & 1][s] = *reinterpret_cast<const u32x4_t*>(&k_lds[buf][S::k_at(ti * 16 + c, s * 4 + q4)]);
    };
    read_keys(0);
#pragma unroll
    for (int ti = 0; ti < 4; ++ti) {
      if (ti < 3) read_keys(ti + 1);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) C[rt][ti] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) C[rt][ti] = mfma_of(kop[ti & 1][s], qop[rt][s], C[rt][ti]);
      __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (MASK) {  // the mask has arrived here on every way: nothing later waits for it and the codes behind it
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int ti = 0; ti < 4; ++ti) asm volatile("" : "+v"(quad[rt][ti]));
    }
    // ---- tokens whose keys f16 does not hold: their products in f32
#pragma unroll 1
    for (uint64_t odd = odd_tokens(0); __builtin_expect(odd != 0, 0); odd &= odd - 1) {
      const int tok = __builtin_ctzll(odd);
      if (t + tok >= t1) break;
      const int64_t at = base + t + tok;
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        const int row = min(row0 + rt * 16 + c, p.rows - 1);
        const uint16_t* q = static_cast<const uint16_t*>(p.q) + b * p.q_sb +
                            (static_cast<int64_t>(h) * p.R + row % p.R) * p.q_sh + static_cast<int64_t>(row / p.R) * p.q_sl;
        const float lift = unit[rt] == 0.f ? 0.f : p.scale / unit[rt];  // a power of two
        float dot = 0.f;
#pragma unroll 1
        for (int d = q4 * (S::DK / 4); d < (q4 + 1) * (S::DK / 4); ++d) {
          const float2 sb = pair16<DT>(static_cast<const uint32_t*>(p.k_params)[at * (S::DK >> (shift + 3)) + (d >> (shift + 3))]);
          const uint32_t word = p.k_codes[at * (S::DK * KB / 32) + d * KB / 32];
          const float k = __builtin_fmaf(sb.x, static_cast<float>((word >> (d * KB % 32)) & ((1u << KB) - 1u)), sb.y);
          dot = __builtin_fmaf(pair16<DT>(q[d]).x * lift, k, dot);
        }
        dot += __shfl_xor(dot, 16);
        dot += __shfl_xor(dot, 32);
        if (q4 == tok % 16 / 4) {
#pragma unroll
          for (int ti = 0; ti < 4; ++ti)
#pragma unroll
            for (int j = 0; j < 4; ++j) C[rt][ti][j] = tok / 16 == ti && tok % 4 == j ? dot : C[rt][ti][j];
        }
      }
    }
    if (MASK && !keys && t + 2 * kTileStep < t1) load(t + 2 * kTileStep);

    // ---- softmax
    bool plain = !MASK && t + kTileStep - 1 <= lim_min && t + kTileStep <= t1;
    if (MASK && by_quads && t + kTileStep - 1 <= lim_min) {  // every byte of the tile set: nothing to mask
      bool hidden = false;
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int ti = 0; ti < 4; ++ti) {
          const uint32_t w = quad[rt][ti];
          hidden |= ((w - 0x01010101u) & ~w & 0x80808080u) != 0;  // a byte of w is 0
        }
      plain = !__any(hidden);
    }
    u32x4_t A[RT][2];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      float top;
      if (__builtin_expect(plain, 1)) {
        top = C[rt][0][0];
#pragma unroll
        for (int ti = 0; ti < 4; ++ti)
#pragma unroll
          for (int j = 0; j < 4; ++j) top = fmaxf(top, C[rt][ti][j]);
        top *= unit[rt];
      } else {
        top = -INFINITY;
#pragma unroll
        for (int ti = 0; ti < 4; ++ti)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            float y = C[rt][ti][j] * unit[rt];
            const int tok = t + ti * 16 + q4 * 4 + j;
            if (MASK && by_quads)
              y = (quad[rt][ti] >> (8 * j)) & 0xffu ? y : -FLT_MAX;
            else if constexpr (MASK)
              y = affine_mask(p, mask_at[rt] + min(tok, t1 - 1) * p.mask_s[4], y);
            if (tok > lim[rt] && y != -INFINITY) y = -FLT_MAX;
            if (tok >= t1) y = -INFINITY;
            C[rt][ti][j] = y;
            top = fmaxf(top, y);
          }
      }
      if (__builtin_expect(__any(top > m[rt] + 8.f), 0)) {
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        const float to = fmaxf(m[rt], top);
        // f16 weights reach 2^(8 + 7)
        const float ref_to = to == -INFINITY ? 0.f : DT == TQ_DTYPE_F16 ? to - 7.f : to;
        const float a = m[rt] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ref[rt] - ref_to);
        m[rt] = to, ref[rt] = ref_to;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float aj = __shfl(a, q4 * 4 + j);
          sum[rt][j] *= aj;
#pragma unroll
          for (int n = 0; n < CT; ++n) acc[rt][n][j] *= aj;
        }
      }
      if (__builtin_expect(plain, 1)) {
#pragma unroll
        for (int ti = 0; ti < 4; ++ti)
#pragma unroll
          for (int j = 0; j < 4; ++j) C[rt][ti][j] = __builtin_amdgcn_exp2f(__builtin_fmaf(C[rt][ti][j], unit[rt], -ref[rt]));
      } else {
#pragma unroll
        for (int ti = 0; ti < 4; ++ti)
#pragma unroll
          for (int j = 0; j < 4; ++j) C[rt][ti][j] = __builtin_amdgcn_exp2f(C[rt][ti][j] - ref[rt]);
      }
#pragma unroll
      for (int pr = 0; pr < 2; ++pr)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float lo = C[rt][2 * pr + j / 2][2 * (j & 1)], hi = C[rt][2 * pr + j / 2][2 * (j & 1) + 1];
          A[rt][pr][j] = pack_of(lo, hi);
        }
    }

    // ---- values: groups of VG operands, one ahead of the products
    constexpr uint32_t kOnes = 0x3c003c00u;
    constexpr int VG = KS == 8 ? 2 : CT % 4 == 0 ? 4 : 3, NGR = CT / VG;
    const u32x4_t ones = {kOnes, kOnes, kOnes, kOnes};
    u32x4_t vop[2][VG];
    auto read_values = [&](int at) {  // group at % NGR of the half step at / NGR
#pragma unroll
      for (int i = 0; i < VG; ++i)
        vop[at & 1][i] = *reinterpret_cast<const u32x4_t*>(
            &v_lds[buf][S::v_at(((at % NGR) * VG + i) * 16 + c, (at / NGR) * 4 + q4)]);
    };
    read_values(0);
#pragma unroll
    for (int at = 0; at < 2 * NGR; ++at) {
      const int pr = at / NGR;
      if (at + 1 < 2 * NGR) read_values(at + 1);
      __builtin_amdgcn_sched_barrier(0);
      if (at % NGR == 0) {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) sum[rt] = mfma_of(A[rt][pr], ones, sum[rt]);
      }
#pragma unroll
      for (int i = 0; i < VG; ++i)
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
          acc[rt][(at % NGR) * VG + i] = mfma_of(A[rt][pr], vop[at & 1][i], acc[rt][(at % NGR) * VG + i]);
      __builtin_amdgcn_sched_barrier(0);
    }

    // ---- tokens with values that f16 does not hold, for the rows that weigh them
#pragma unroll 1
    for (uint64_t odd = odd_tokens(2); __builtin_expect(odd != 0, 0); odd &= odd - 1) {
      const int tok = __builtin_ctzll(odd);
      if (t + tok >= t1) break;
      const int64_t at = base + t + tok;
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        // the rounded weight: tile tok / 16, two tokens a register
        uint32_t two = 0;
#pragma unroll
        for (int pr = 0; pr < 2; ++pr)
#pragma unroll
          for (int j = 0; j < 4; ++j) two = tok / 32 == pr && tok / 16 % 2 * 2 + tok % 4 / 2 == j ? A[rt][pr][j] : two;
        const float2 both = pair16<TQ_DTYPE_F16>(two);
        const float w = tok % 2 ? both.y : both.x;
        float wr[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) wr[j] = __shfl(w, (tok % 16) / 4 * 16 + q4 * 4 + j);
#pragma unroll
        for (int n = 0; n < CT; ++n) {
          const int d = n * 16 + c;
          const float2 sb = pair16<DT>(static_cast<const uint32_t*>(p.v_params)[at * (S::DV >> (shift + 3)) + (d >> (shift + 3))]);
          if (fits_f16<DT, VB>(sb)) continue;  // in LDS already
          const uint32_t word = p.v_codes[at * (S::DV * VB / 32) + d * VB / 32];
          const float v = __builtin_fmaf(sb.x, static_cast<float>((word >> (d * VB % 32)) & ((1u << VB) - 1u)), sb.y);
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[rt][n][j] = wr[j] == 0.f ? acc[rt][n][j] : __builtin_fmaf(wr[j], v, acc[rt][n][j]);
        }
      }
    }
    if (keys && more) decode_keys(buf ^ 1, flags == 2 ? 0 : flags + 1);
    if (keys && t + 2 * kTileStep < t1) load(t + 2 * kTileStep);
    __syncthreads();
  }

  // ---- results: rows 4 q4 + j, coordinates 16 n + c
#pragma unroll
  for (int rt = 0; rt < RT; ++rt)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int row = row0 + rt * 16 + q4 * 4 + j;
      const float row_ref = __shfl(m[rt] == -INFINITY ? -INFINITY : ref[rt], q4 * 4 + j);
      if (row >= p.rows) continue;
      const float l = sum[rt][j];
      if (p.splits == 1) {
        const int64_t head = static_cast<int64_t>(bh) * p.R + row % p.R;
        const int64_t to = (head * p.L + row / p.R) * S::DV + c;
        const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
        for (int n = 0; n < CT; ++n) store_elem<DT>(p.out, to + n * 16, l == 0.f ? 0.f : acc[rt][n][j] * inv);
      } else {
        const int64_t at = (static_cast<int64_t>(bh) * p.rows + row) * p.splits + split;
#pragma unroll
        for (int n = 0; n < CT; ++n) p.part_o[at * S::DV + n * 16 + c] = acc[rt][n][j];
        if (c == 0) p.part_ml[2 * at] = row_ref, p.part_ml[2 * at + 1] = l;
      }
    }
}

template <int DT, int KB, int VB, int KS, int CT>
int launch_tile_at(const AffineAttnParams& p, hipStream_t st) {
  constexpr int kRows = TileShape<KS, CT>::ROWS;
  static_assert(kRows == tile_rows(32 * KS, 16 * CT), "rows a workgroup");
  const int64_t blocks = static_cast<int64_t>(p.B) * p.Hkv * ((p.rows + kRows - 1) / kRows) * p.splits;
  if (blocks > INT32_MAX / 512) return fail(TQ_ERR_UNSUPPORTED, "tq_attention_affine: %lld workgroups", static_cast<long long>(blocks));
  if (p.mask_kind != TQ_MASK_NONE)
    affine_tile_kernel<DT, KB, VB, KS, CT, true><<<static_cast<unsigned>(blocks), 64 * kTileWaves, 0, st>>>(p);
  else
    affine_tile_kernel<DT, KB, VB, KS, CT, false><<<static_cast<unsigned>(blocks), 64 * kTileWaves, 0, st>>>(p);
  return check_launch("affine_tile_kernel");
}

template <int DT, int KB, int VB>
int launch_tile_bits(const AffineAttnParams& p, hipStream_t st) {
  switch (p.k_dim) {
    case 64: return launch_tile_at<DT, KB, VB, 2, 4>(p, st);
    case 96: return launch_tile_at<DT, KB, VB, 3, 6>(p, st);
    case 128: return launch_tile_at<DT, KB, VB, 4, 8>(p, st);
    case 192: return launch_tile_at<DT, KB, VB, 6, 8>(p, st);
    case 256: return launch_tile_at<DT, KB, VB, 8, 16>(p, st);
    default: return fail(TQ_ERR_UNSUPPORTED, "tq_attention_affine: no tile kernel for head dims %d / %d", p.k_dim, p.v_dim);
  }
}

}  // namespace tq
