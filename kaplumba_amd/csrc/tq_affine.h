// Group-affine cache: what its kernels share.
//
// A row of dim coordinates is stored as dim * bits / 32 words (bits 4 or 8, coordinate i at bits i * bits, least
// significant first) and one (scale, bias) pair per group of 32, 64 or 128 coordinates, in the type T of the
// vectors: coordinate i stands for scale * code_i + bias.
#pragma once

#include "tq_common.h"

namespace tq {

// The tokens that rows of the array mask see: the first and one past the last kept one of a row's tokens (those of its
// sequence, and within its limit under the causal rule), or all of them where it keeps none (such a row weighs them
// alike).  Rows are told apart by the axes the mask has, and by b and l where windows or the causal rule differ.
struct MaskRows {
  int2* range;            // [nb, ng, nr, nl]
  int nb, ng, nr, nl;
};

struct AffineAttnParams {
  const void* q;
  int64_t q_sb, q_sh, q_sl;
  const uint32_t* k_codes;
  const void* k_params;
  const uint32_t* v_codes;
  const void* v_params;
  const int32_t* starts;
  const int32_t* lens;
  const void* mask;
  int64_t mask_s[5];
  int mask_kind;
  MaskRows keep;          // no ranges: every token of a sequence is looked at
  int causal;
  int64_t capacity, max_tokens;
  int B, Hkv, R, L;       // R query heads a kv head
  int rows;               // R * L; row = l * R + r
  int k_dim, v_dim;
  int group;
  float scale;            // of the scores, times log2(e)
  int splits;
  int64_t split_tokens;   // tokens a split takes of every sequence
  void* out;
  float* part_o;          // [B * Hkv * rows, splits, v_dim]
  float* part_ml;         // [B * Hkv * rows, splits, 2]: running maximum (base 2), sum
};

// Which instantiation of the few-rows kernel (tq_affine_rows.h) takes a call: head dims up to `dim`, exactly it and no
// array mask where `full`, and `rows` query rows a workgroup.  (The mask's loads, between the codes' and their use, would
// make every call wait for the next step's codes.)
struct RowsChoice {
  int dim, rows;
  bool full;
};

int launch_rows_k4v4(const AffineAttnParams& p, const RowsChoice& r, int dtype, hipStream_t st);
int launch_rows_k8v4(const AffineAttnParams& p, const RowsChoice& r, int dtype, hipStream_t st);
int launch_rows_k8v8(const AffineAttnParams& p, const RowsChoice& r, int dtype, hipStream_t st);

// The many-rows kernel (tq_affine_tile.h): 32 ks key and 16 ct value coordinates; rows a workgroup takes, 0 where no
// instantiation has these dims.
constexpr int tile_rows(int k_dim, int v_dim) {
  return k_dim == v_dim && (k_dim == 64 || k_dim == 96 || k_dim == 128) ? 256
         : (k_dim == 192 && v_dim == 128) || (k_dim == 256 && v_dim == 256) ? 128 : 0;
}

int launch_tile_k4v4(const AffineAttnParams& p, int dtype, hipStream_t st);
int launch_tile_k8v4(const AffineAttnParams& p, int dtype, hipStream_t st);
int launch_tile_k8v8(const AffineAttnParams& p, int dtype, hipStream_t st);

// Tokens [start, end) of sequence b, as the device arrays say, within the cache.
__device__ __forceinline__ void affine_range(const AffineAttnParams& p, int b, int64_t& start, int64_t& end) {
  // uniform: b is the workgroup's
  end = p.lens ? min(static_cast<int64_t>(__builtin_amdgcn_readfirstlane(p.lens[b])), p.max_tokens) : p.max_tokens;
  start = p.starts ? max(static_cast<int64_t>(__builtin_amdgcn_readfirstlane(p.starts[b])), static_cast<int64_t>(0)) : 0;
  if (end < start) end = start;
}

// The score x (base 2 units) of query row (b, g, r, l) for cache row t under the array mask.  An added
// -FLT_MAX keeps its place above -inf, as in the other attention kernels.
__device__ __forceinline__ float affine_mask(const AffineAttnParams& p, int64_t off, float x) {
  if (p.mask_kind == TQ_MASK_BOOL) return static_cast<const uint8_t*>(p.mask)[off] ? x : -FLT_MAX;
  const float m = p.mask_kind == TQ_MASK_ADD_F32   ? static_cast<const float*>(p.mask)[off]
                  : p.mask_kind == TQ_MASK_ADD_F16 ? f16_bits_to_f32(static_cast<const uint16_t*>(p.mask)[off])
                                                   : bf16_bits_to_f32(static_cast<const uint16_t*>(p.mask)[off]);
  if (m == -INFINITY) return m;  // also where the score is not finite
  const float t = __builtin_fmaf(m, 1.44269504088896341f, x);
  return t == -INFINITY ? -FLT_MAX : t;
}

// A load at a uniform base and a lane's offset in bytes, in 32 bits: the form that global loads have for it (an index
// of words would first be widened and added on the vector units).
template <typename T>
__device__ __forceinline__ T load_at(const void* base, uint32_t bytes) {
  return *reinterpret_cast<const T*>(static_cast<const char*>(base) + bytes);
}

// A constant that the compiler holds in a register.  Neither operand of (x & mask) | with fits v_and_or_b32 as a
// literal, so it takes two instructions for constants it knows.  Only vector instructions may read the result of the
// asm: the wait states between a vector write and a matrix instruction's read are the compiler's to insert, and it
// does not look into asm.
__device__ __forceinline__ uint32_t held_vector(uint32_t x) {
  uint32_t o;
  asm("v_mov_b32 %0, %1" : "=v"(o) : "s"(x));
  return o;
}
__device__ __forceinline__ uint32_t held_scalar(uint32_t x) {
  uint32_t o;
  asm("s_mov_b32 %0, %1" : "=s"(o) : "i"(x));
  return o;
}

// (scale, bias) of a packed pair of 16-bit values.
template <int DT>
__device__ __forceinline__ float2 pair16(uint32_t u) {
  if constexpr (DT == TQ_DTYPE_F16) return make_float2(f16_bits_to_f32(u & 0xffffu), f16_bits_to_f32(u >> 16));
  return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}

// (scale, bias) of one group.
template <int DT>
__device__ __forceinline__ float2 affine_pair(const void* params, int64_t i) {
  if constexpr (DT == TQ_DTYPE_F32) {
    return static_cast<const float2*>(params)[i];
  } else {
    return pair16<DT>(static_cast<const uint32_t*>(params)[i]);
  }
}

}  // namespace tq
