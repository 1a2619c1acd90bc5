// Attention over the group-affine cache: entry points, the vector kernel and the merge.
#include <algorithm>

#include "tq_affine_rows.h"

namespace tq {
namespace {

constexpr int kVecRows = 4;     // query rows a workgroup of the vector kernel takes
constexpr int kVecTokens = 64;  // tokens a step
constexpr int kMaxDim = 512;

template <int DT, int BITS>
__device__ __forceinline__ float code_of(const uint32_t* row, int d) {
  constexpr int kPer = 32 / BITS;
  return static_cast<float>((row[d / kPer] >> (d % kPer * BITS)) & ((1u << BITS) - 1u));
}

// S = scale * sum_g (s_g (q . c)_g + b_g sum(q)_g), an online softmax per row, O = sum p (s c + b): all in f32.
// Wave = a quarter of the 32-coordinate blocks and lane = token for the scores, wave = row for the softmax,
// thread = coordinate for the values.  Bound by its vector instructions, about rows * (Dk + Dv) multiply-adds a
// token, and by their latency at few waves; it serves f32 and the dims that the matrix-core kernels do not take (16
// heads of 32,724 tokens, d = 128, 8 bits: 132 us, 1.3 TB/s).
template <int DT, int KB, int VB>
__global__ __launch_bounds__(256) void affine_vector_kernel(const AffineAttnParams p) {
  __shared__ float qs[kVecRows][kMaxDim];
  __shared__ float qsum[kVecRows][kMaxDim / 32];
  __shared__ float part[4][kVecRows][kVecTokens];
  __shared__ float pr[kVecRows][kVecTokens];
  __shared__ float alpha[kVecRows];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int split = blockIdx.x % p.splits;
  const int blk = blockIdx.x / p.splits;
  const int row_blocks = (p.rows + kVecRows - 1) / kVecRows;
  const int bh = blk / row_blocks, row0 = (blk % row_blocks) * kVecRows;
  const int b = bh / p.Hkv, h = bh % p.Hkv;

  for (int i = tid; i < kVecRows * p.k_dim; i += 256) {
    const int s = i / p.k_dim, d = i % p.k_dim;
    const int row = min(row0 + s, p.rows - 1);
    qs[s][d] = load_elem<DT>(p.q, b * p.q_sb + (static_cast<int64_t>(h) * p.R + row % p.R) * p.q_sh +
                                      static_cast<int64_t>(row / p.R) * p.q_sl + d);
  }
  __syncthreads();
  const int blocks32 = p.k_dim / 32;
  for (int i = tid; i < kVecRows * blocks32; i += 256) {
    const int s = i / blocks32, c = i % blocks32;
    float t = 0.f;
    for (int d = 0; d < 32; ++d) t += qs[s][c * 32 + d];
    qsum[s][c] = t;
  }
  __syncthreads();

  int64_t start, end;
  affine_range(p, b, start, end);
  const int64_t t0 = start + split * p.split_tokens;
  const int64_t t1 = min(end, t0 + p.split_tokens);
  const int kw = p.k_dim * KB / 32, vw = p.v_dim * VB / 32;
  const int kg = p.k_dim / p.group, vg = p.v_dim / p.group;
  const int64_t base = static_cast<int64_t>(bh) * p.capacity;
  const int my_row = min(row0 + wave, p.rows - 1);
  const int my_l = my_row / p.R, my_r = my_row % p.R;
  const int64_t lim = p.causal ? end - p.L + my_l : INT64_MAX;
  float m = -INFINITY, l = 0.f;
  float acc[kVecRows][2] = {};

  for (int64_t t = t0; t < t1; t += kVecTokens) {
    const int64_t tok = min(t + lane, t1 - 1);
    float dot[kVecRows] = {};
    for (int c = wave; c < blocks32; c += 4) {
      const uint32_t* row = p.k_codes + (base + tok) * kw + c * KB;
      const float2 sb = affine_pair<DT>(p.k_params, (base + tok) * kg + c * 32 / p.group);
      float part32[kVecRows] = {};
      for (int w = 0; w < KB; ++w) {
        const uint32_t word = row[w];
#pragma unroll
        for (int j = 0; j < 32 / KB; ++j) {
          const float code = static_cast<float>((word >> (j * KB)) & ((1u << KB) - 1u));
#pragma unroll
          for (int s = 0; s < kVecRows; ++s)
            part32[s] = __builtin_fmaf(qs[s][c * 32 + w * (32 / KB) + j], code, part32[s]);
        }
      }
#pragma unroll
      for (int s = 0; s < kVecRows; ++s)
        dot[s] = __builtin_fmaf(sb.x, part32[s], __builtin_fmaf(sb.y, qsum[s][c], dot[s]));
    }
#pragma unroll
    for (int s = 0; s < kVecRows; ++s) part[wave][s][lane] = dot[s];
    __syncthreads();
    {
      float x = (part[0][wave][lane] + part[1][wave][lane]) + (part[2][wave][lane] + part[3][wave][lane]);
      x *= p.scale;
      if (p.mask_kind != TQ_MASK_NONE)
        x = affine_mask(p, b * p.mask_s[0] + h * p.mask_s[1] + my_r * p.mask_s[2] + my_l * p.mask_s[3] + tok * p.mask_s[4], x);
      if (tok > lim && x != -INFINITY) x = -FLT_MAX;
      if (t + lane >= t1) x = -INFINITY;
      float mx = x;
      for (int o = 32; o; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o));
      const float m_new = fmaxf(m, mx);
      const float ref = m_new == -INFINITY ? 0.f : m_new;
      const float w = exp2f(x - ref);
      const float a = exp2f(m - ref);
      float sum = w;
      for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o);
      l = l * a + sum;
      m = m_new;
      pr[wave][lane] = w;
      if (lane == 0) alpha[wave] = a;
    }
    __syncthreads();
    const int n = static_cast<int>(min(static_cast<int64_t>(kVecTokens), t1 - t));
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int d = tid + e * 256;
      if (d >= p.v_dim) break;
#pragma unroll
      for (int s = 0; s < kVecRows; ++s) acc[s][e] *= alpha[s];
      for (int i = 0; i < n; ++i) {
        const float2 sb = affine_pair<DT>(p.v_params, (base + t + i) * vg + d / p.group);
        const float v = __builtin_fmaf(sb.x, code_of<DT, VB>(p.v_codes + (base + t + i) * vw, d), sb.y);
#pragma unroll
        for (int s = 0; s < kVecRows; ++s) {
          const float w = pr[s][i];
          acc[s][e] = w == 0.f ? acc[s][e] : __builtin_fmaf(w, v, acc[s][e]);  // what a row masks may be NaN
        }
      }
    }
    __syncthreads();
  }

#pragma unroll
  for (int s = 0; s < kVecRows; ++s) {
    const int row = row0 + s;
    if (row >= p.rows) break;
    const int64_t at = (static_cast<int64_t>(bh) * p.rows + row) * p.splits + split;
#pragma unroll
    for (int e = 0; e < 2; ++e)
      if (tid + e * 256 < p.v_dim) p.part_o[at * p.v_dim + tid + e * 256] = acc[s][e];
  }
  if (lane == 0 && row0 + wave < p.rows) {
    const int64_t at = (static_cast<int64_t>(bh) * p.rows + row0 + wave) * p.splits + split;
    p.part_ml[2 * at] = m;
    p.part_ml[2 * at + 1] = l;
  }
}

// out = sum_s 2^(m_s - M) o_s / sum_s 2^(m_s - M) l_s over a row's splits; a row without a token, or whose every
// score is -inf, gives zeros.  One workgroup a row: its waves take splits and its lanes four coordinates each, then
// the waves' sums meet in LDS.
template <int DT>
__global__ __launch_bounds__(256) void affine_merge_kernel(const AffineAttnParams p) {
  __shared__ float part[4][kMaxDim + 1];
  const int64_t at = blockIdx.x;  // (b, h, row)
  const int row = static_cast<int>(at % p.rows);
  const int64_t bh = at / p.rows;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const float2* ml = reinterpret_cast<const float2*>(p.part_ml) + at * p.splits;
  float M = -INFINITY;
  for (int s = lane; s < p.splits; s += 64) M = fmaxf(M, ml[s].x);
  for (int o = 32; o; o >>= 1) M = fmaxf(M, __shfl_xor(M, o));
  const float ref = M == -INFINITY ? 0.f : M;
  float4 o[2] = {};
  float sum = 0.f;
  for (int s = wave; s < p.splits; s += 4) {
    const float2 t = ml[s];
    const float w = __builtin_amdgcn_exp2f(t.x - ref);
    sum = __builtin_fmaf(w, t.y, sum);
    const float4* from = reinterpret_cast<const float4*>(p.part_o + (at * p.splits + s) * p.v_dim);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      if ((lane + 64 * e) * 4 >= p.v_dim) break;
      const float4 x = from[lane + 64 * e];
      if (w != 0.f) {
        o[e].x = __builtin_fmaf(w, x.x, o[e].x), o[e].y = __builtin_fmaf(w, x.y, o[e].y);
        o[e].z = __builtin_fmaf(w, x.z, o[e].z), o[e].w = __builtin_fmaf(w, x.w, o[e].w);
      }
    }
  }
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int d = (lane + 64 * e) * 4;
    if (d >= p.v_dim) break;
    part[wave][d] = o[e].x, part[wave][d + 1] = o[e].y, part[wave][d + 2] = o[e].z, part[wave][d + 3] = o[e].w;
  }
  if (lane == 0) part[wave][kMaxDim] = sum;
  __syncthreads();
  const float all = (part[0][kMaxDim] + part[1][kMaxDim]) + (part[2][kMaxDim] + part[3][kMaxDim]);
  const int64_t head = bh * p.R + row % p.R;  // b * Hq + query head
  const int64_t to = (head * p.L + row / p.R) * p.v_dim;
  for (int d = threadIdx.x; d < p.v_dim; d += 256) {
    const float x = (part[0][d] + part[1][d]) + (part[2][d] + part[3][d]);
    store_elem<DT>(p.out, to + d, all == 0.f ? 0.f : x / all);
  }
}

// The same for few splits: a thread takes four coordinates of a row over all of them, so that prefill's many rows
// are one stream of the partial results.
template <int DT>
__global__ __launch_bounds__(256) void affine_merge_flat_kernel(const AffineAttnParams p, uint32_t quads, uint32_t all) {
  const uint32_t i = blockIdx.x * 256 + threadIdx.x;
  if (i >= all) return;
  const uint32_t at = i / quads;  // (b, h, row)
  const uint32_t d = (i - at * quads) * 4;
  const float2* ml = reinterpret_cast<const float2*>(p.part_ml) + static_cast<int64_t>(at) * p.splits;
  const float* from = p.part_o + static_cast<int64_t>(at) * p.splits * p.v_dim + d;
  float M = -INFINITY;
  for (int s = 0; s < p.splits; ++s) M = fmaxf(M, ml[s].x);
  const float ref = M == -INFINITY ? 0.f : M;
  float4 o = {};
  float sum = 0.f;
#pragma unroll 4
  for (int s = 0; s < p.splits; ++s) {
    const float2 t = ml[s];
    const float4 x = *reinterpret_cast<const float4*>(from + static_cast<int64_t>(s) * p.v_dim);
    const float w = __builtin_amdgcn_exp2f(t.x - ref);
    sum = __builtin_fmaf(w, t.y, sum);
    o.x = w == 0.f ? o.x : __builtin_fmaf(w, x.x, o.x), o.y = w == 0.f ? o.y : __builtin_fmaf(w, x.y, o.y);
    o.z = w == 0.f ? o.z : __builtin_fmaf(w, x.z, o.z), o.w = w == 0.f ? o.w : __builtin_fmaf(w, x.w, o.w);
  }
  const uint32_t row = at % p.rows;
  const int64_t bh = at / p.rows;
  const int64_t to = ((bh * p.R + row % p.R) * p.L + row / p.R) * p.v_dim + d;
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  store_elem<DT>(p.out, to, sum == 0.f ? 0.f : o.x * inv);
  store_elem<DT>(p.out, to + 1, sum == 0.f ? 0.f : o.y * inv);
  store_elem<DT>(p.out, to + 2, sum == 0.f ? 0.f : o.z * inv);
  store_elem<DT>(p.out, to + 3, sum == 0.f ? 0.f : o.w * inv);
}

template <int DT>
void launch_merge(const AffineAttnParams& p, int64_t rows, hipStream_t st) {
  const int64_t quads = rows * (p.v_dim / 4);
  // Few splits of many rows stream through one thread for four coordinates (16,384 rows of 4 splits 9 us, 500 x 64 rows
  // of d = 64 6 us; a workgroup a row 19 and 31); a workgroup a row hides the splits' latency where there are many of
  // them and few rows (32 rows of 32 splits 6 us; 16).
  if (p.splits <= 16 && quads >= 65536 && quads <= INT32_MAX)
    affine_merge_flat_kernel<DT><<<static_cast<unsigned>((quads + 255) / 256), 256, 0, st>>>(
        p, static_cast<uint32_t>(p.v_dim / 4), static_cast<uint32_t>(quads));
  else
    affine_merge_kernel<DT><<<static_cast<unsigned>(rows), 256, 0, st>>>(p);
}

// One workgroup a row of MaskRows: from the front to the first kept token and from the back to the last, in pieces of
// 16 bytes a thread where the row is contiguous bytes, four single elements otherwise.  Bound by the loads' latency, a
// round of them a step: 8 KiB of bytes in one of 512 threads, which few rows have (8 us before 131,072 tokens; 256
// threads 18, 1024 at 16,384 tokens 3 more).  Many rows have 256.
__global__ __launch_bounds__(512) void affine_mask_range_kernel(const AffineAttnParams p) {
  __shared__ int lo_s, hi_s;
  const int tid = threadIdx.x, threads = blockDim.x;
  int at = blockIdx.x;
  const int l = at % p.keep.nl;
  at /= p.keep.nl;
  const int r = at % p.keep.nr;
  at /= p.keep.nr;
  const int g = at % p.keep.ng, b = at / p.keep.ng;
  int64_t start64, end64;
  affine_range(p, b, start64, end64);
  const int start = static_cast<int>(start64), end = static_cast<int>(end64);
  const int seen = p.causal ? static_cast<int>(max(start64, min(end64, end64 - p.L + l + 1))) : end;
  if (tid == 0) lo_s = INT32_MAX, hi_s = 0;
  __syncthreads();
  const int64_t from = b * p.mask_s[0] + g * p.mask_s[1] + r * p.mask_s[2] + l * p.mask_s[3];
  // a NaN counts as kept
  auto kept = [&](int t) {
    return !(affine_mask(p, from + t * p.mask_s[4], 0.f) <= (p.mask_kind == TQ_MASK_BOOL ? -FLT_MAX : -INFINITY));
  };
  const bool bytes = p.mask_kind == TQ_MASK_BOOL && p.mask_s[4] == 1 && seen - start >= 16;
  const int chunk = threads * (bytes ? 16 : 4);
  // the first and one past the last kept token of this thread's part of [t, t + chunk)
  auto look = [&](int64_t t, int& lo, int& hi) {
    if (bytes) {
      // pieces over an end move inwards, over tokens that another thread looks at too
      int64_t mine = t + tid * 16;
      if (mine < seen && mine + 16 > start) {
        mine = min(max(mine, start64), static_cast<int64_t>(seen) - 16);
        uint64_t w[2];
        __builtin_memcpy(w, static_cast<const uint8_t*>(p.mask) + from + mine, 16);
#pragma unroll
        for (int i = 0; i < 2; ++i)
          if (w[i]) {
            const int at0 = static_cast<int>(mine) + 8 * i;
            lo = min(lo, at0 + (__ffsll(static_cast<unsigned long long>(w[i])) - 1) / 8);
            hi = max(hi, at0 + (63 - __clzll(static_cast<long long>(w[i]))) / 8 + 1);
          }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int64_t e = t + i * threads + tid;
        if (e >= start && e < seen && kept(static_cast<int>(e)))
          lo = min(lo, static_cast<int>(e)), hi = max(hi, static_cast<int>(e) + 1);
      }
    }
  };
  // from both ends at once, until each has met a kept token; the front's way alone covers every token
  int lo = INT32_MAX, hi = 0, unused_lo = INT32_MAX, unused_hi = 0;
  bool front = true, back = true;
  for (int64_t t = start, e = static_cast<int64_t>(seen) - chunk; front && t < seen; t += chunk, e -= chunk) {
    look(t, lo, unused_hi);
    if (back) look(e, unused_lo, hi);
    front = !__syncthreads_or(lo != INT32_MAX);
    back = back && !__syncthreads_or(hi != 0);
    if (!front)
      for (; back; back = !__syncthreads_or(hi != 0)) look(e -= chunk, unused_lo, hi);
  }
  atomicMin(&lo_s, lo);
  atomicMax(&hi_s, hi);
  __syncthreads();
  if (tid == 0) p.keep.range[blockIdx.x] = hi_s > 0 ? make_int2(lo_s, hi_s) : make_int2(start, end);
}

int64_t align256(int64_t n) { return (n + 255) & ~static_cast<int64_t>(255); }

struct Plan {
  int splits;
  int64_t split_tokens;
};

// Workgroups to aim at.  Vector kernel: two a CU, four where each still has 128 tokens (16 heads of 32,724 tokens in f32
// 231 -> 132 us; 8 heads of 8192, 128 splits of 64 tokens instead of 64: 36 us against 31).
constexpr int64_t kVecTarget = 512, kVecMore = 1024;
// Few-rows kernel: its eight waves, two a SIMD, on every CU (8 heads of 32,768 tokens 21 us; 128: 23; 512: 31; 4 x 4
// query rows over 4 x 131,076 tokens 149; 222; 157).
constexpr int64_t kRowsTarget = 256;
// Where sequences end at different tokens: finer, so that CUs share the long ones (32 sequences to 8192 tokens of
// d = 256: 127 us; 256 workgroups 129, 1024 144, 2048 174).
constexpr int64_t kRaggedTarget = 768;
constexpr int kRowsTokens = 512;  // tokens of one step of a workgroup's eight waves

// A split for every `unit` tokens at most, and about `target` workgroups in all.
Plan plan_splits(int64_t blocks, int64_t max_tokens, int64_t target, int unit) {
  const int64_t most = (max_tokens + unit - 1) / unit;
  const int64_t s = std::max<int64_t>(1, std::min(target / blocks, most));
  const int64_t per = std::max<int64_t>(1, ((max_tokens + s - 1) / s + unit - 1) / unit) * unit;
  return {static_cast<int>(std::max<int64_t>(1, (max_tokens + per - 1) / per)), per};
}

Plan vector_plan(int64_t blocks, int64_t max_tokens) {
  const Plan two = plan_splits(blocks, max_tokens, kVecTarget, kVecTokens);
  const Plan four = plan_splits(blocks, max_tokens, kVecMore, 2 * kVecTokens);
  return four.splits > two.splits ? four : two;
}

int64_t rows_of(int B, int Hq, int L) { return static_cast<int64_t>(B) * Hq * L; }

// The few-rows kernel takes 16-bit types and head dims to 256 and counts tokens in 32 bits (f32, larger dims, 4-bit keys
// with 8-bit values: the vector kernel).
bool rows_kernel(int dtype, int k_dim, int v_dim, int k_bits, int v_bits, int64_t max_tokens) {
  return max_tokens <= (1 << 30) && dtype != TQ_DTYPE_F32 && k_dim <= 256 && v_dim <= 256 && !(k_bits == 4 && v_bits == 8);
}

// Four query rows have a layout of their own at groups to 64 (8 heads of 4 x 16,384 tokens, one query each: d = 96 27 us,
// in the layout of 16 rows 45; 192/128 38 / 55; d = 128 under a mask 33 / 40, 256 56 / 93); at groups of 128 that of 16
// is the faster (d = 128 22 us, of four 23).
RowsChoice rows_choice(int64_t rows, int k_dim, int v_dim, int group, int mask_kind) {
  RowsChoice r;
  r.full = k_dim == v_dim && (k_dim == 64 || k_dim == 128 || k_dim == 256) && group <= 64 && mask_kind == TQ_MASK_NONE;
  r.dim = r.full ? k_dim : std::max(k_dim, v_dim) <= 128 ? 128 : 256;
  r.rows = group <= 64 && rows <= 4 ? 4 : rows_large(r.dim, group);
  return r;
}

// The many-rows kernel takes what the few-rows kernel does at its head dims, where it is the faster of the two: a block
// of its rows costs what `worth` blocks of 16 cost there, whether it is full or not, and about 128 Ki tokens of those
// pass while its first step and its join are on their way.  Microseconds, few rows / many rows: head dim 128, 64 heads
// of 4096 tokens, 32 rows 26 / 58, 64 rows 38 / 57, 128 rows 72 / 62; 8 heads, 128 rows 21 / 27; 64: 64 rows 22 / 47,
// 128 rows 41 / 50 and with a mask 125 / 95; 256: 32 rows 58 / 78, 48 rows 90 / 79; 96: 32 rows 47 / 54, 48 rows 70 / 54.
bool tile_kernel(int64_t rows, int k_dim, int v_dim, int64_t heads, int64_t max_tokens, int mask_kind) {
  const int block = tile_rows(k_dim, v_dim);
  if (block == 0) return false;
  const int worth = k_dim == 64 ? (mask_kind == TQ_MASK_NONE ? 9 : 5) : k_dim == 128 ? 5 : 2;
  const int64_t more = (rows + 15) / 16 - (rows + block - 1) / block * worth;
  return heads * max_tokens * more > 128 << 10;
}

// Tokens times blocks of rows from which the few-rows kernel has the masks' ranges found first.  That costs 8 us, which
// a mask that keeps tokens everywhere pays for nothing (2 x 8 heads of 32,768 tokens, d = 128, one query 34 -> 42 us,
// eight 70 -> 78); a window of 512 takes 34 -> 24 and 69 -> 25 there, 805 -> 36 at 8 queries over 8 x 131,072 of 192/128.
constexpr int64_t kRangeTokens = 512 << 10;

constexpr int64_t kTileTarget = 256;  // workgroups at once: its eight waves fill a CU

// Splits with the least estimated time: rounds of one workgroup a CU, each of its tokens and about 256 tokens' worth of
// prologue and results; and the partial results' way through memory, 64 tokens' worth a round of 256 x 256 rows.
Plan tile_plan(int64_t blocks, int64_t max_tokens) {
  int64_t best = 1;
  double best_time = 0;
  const int64_t most = std::min<int64_t>(std::max<int64_t>(1, 2 * kTileTarget / blocks), (max_tokens + 255) / 256);
  for (int64_t s = 1; s <= std::max<int64_t>(1, most); ++s) {
    const double rounds = static_cast<double>((blocks * s + kTileTarget - 1) / kTileTarget);
    const double time = rounds * (static_cast<double>(max_tokens) / s + 256) +
                        (s > 1 ? 128 + 128.0 * blocks * s / kTileTarget : 0);
    if (s == 1 || time < best_time) best = s, best_time = time;
  }
  return {static_cast<int>(best), 0};  // the kernel divides the tokens that its rows see
}

// Rows times splits of any plan with at most these sequences, queries and tokens: n workgroups of k rows have at most
// target / n splits, and at least one.
int64_t most_partials(int B, int Hq, int Hkv, int L, int64_t max_tokens) {
  const int64_t rows = rows_of(B, Hq, L), most = std::max<int64_t>(1, (max_tokens + kVecTokens - 1) / kVecTokens);
  const int64_t few = std::max(kVecMore * kVecRows, kRaggedTarget * 16);
  const int64_t many = static_cast<int64_t>(Hq / Hkv) * L > 16 ? std::max(few, 2 * kTileTarget * 256) : few;
  return std::min(rows * most, many + rows);
}

int64_t workspace_bytes(int B, int Hq, int Hkv, int L, int v_dim, int64_t max_tokens) {
  const int64_t n = most_partials(B, Hq, Hkv, L, max_tokens);
  return align256(n * 8) + align256(n * v_dim * 4) + align256(rows_of(B, Hq, L) * 8);
}

template <int DT>
void launch_vector(const AffineAttnParams& p, int k_bits, int v_bits, unsigned blocks, hipStream_t stream) {
  if (k_bits == 4 && v_bits == 4)
    affine_vector_kernel<DT, 4, 4><<<blocks, 256, 0, stream>>>(p);
  else if (k_bits == 8 && v_bits == 4)
    affine_vector_kernel<DT, 8, 4><<<blocks, 256, 0, stream>>>(p);
  else if (k_bits == 8)
    affine_vector_kernel<DT, 8, 8><<<blocks, 256, 0, stream>>>(p);
  else
    affine_vector_kernel<DT, 4, 8><<<blocks, 256, 0, stream>>>(p);
}

bool dims_ok(int k_dim, int v_dim, int group) {
  return (group == 32 || group == 64 || group == 128) && k_dim >= group && v_dim >= group && k_dim <= kMaxDim &&
         v_dim <= kMaxDim && k_dim % group == 0 && v_dim % group == 0;
}

}  // namespace
}  // namespace tq

using namespace tq;

extern "C" {

int64_t tq_attention_affine_workspace_size(int B, int Hq, int Hkv, int L, int k_dim, int v_dim, int64_t max_tokens) {
  if (B <= 0 || Hq <= 0 || Hkv <= 0 || L <= 0 || Hq % Hkv || max_tokens < 0 || k_dim <= 0 || v_dim <= 0 ||
      k_dim > kMaxDim || v_dim > kMaxDim)
    return 0;
  return workspace_bytes(B, Hq, Hkv, L, v_dim, max_tokens);
}

int tq_attention_affine(const void* q, int q_dtype, int B, int Hq, int Hkv, int L, int k_dim, int v_dim,
                        int64_t q_stride_b, int64_t q_stride_h, int64_t q_stride_l, float scale,
                        const uint32_t* k_codes, const void* k_params, int k_bits, const uint32_t* v_codes,
                        const void* v_params, int v_bits, int group, int64_t capacity, int64_t max_tokens,
                        const int32_t* seq_starts, const int32_t* seq_lens, int causal, const void* mask,
                        int mask_kind, const int64_t* mask_strides, void* out, void* workspace,
                        int64_t workspace_bytes_given, void* stream) {
  if (q_dtype < TQ_DTYPE_F32 || q_dtype > TQ_DTYPE_BF16)
    return fail(TQ_ERR_INVALID_ARGUMENT, "tq_attention_affine: q_dtype %d", q_dtype);
  if (B < 0 || Hq < 0 || L < 0 || Hkv < 1 || Hq % Hkv)
    return fail(TQ_ERR_INVALID_ARGUMENT, "tq_attention_affine: bad sizes B=%d, heads %d over %d kv heads, L=%d", B, Hq, Hkv, L);
  if ((k_bits != 4 && k_bits != 8) || (v_bits != 4 && v_bits != 8))
    return fail(TQ_ERR_INVALID_ARGUMENT, "tq_attention_affine: bits %d / %d are not 4 or 8", k_bits, v_bits);
  if (!dims_ok(k_dim, v_dim, group))
    return fail(TQ_ERR_UNSUPPORTED, "tq_attention_affine: head dims %d / %d in groups of %d (multiples of a group of 32, 64 or 128, to %d)",
                k_dim, v_dim, group, kMaxDim);
  if (capacity < 0 || capacity > INT32_MAX || max_tokens < 0 || max_tokens > capacity)
    return fail(TQ_ERR_INVALID_ARGUMENT, "tq_attention_affine: %lld tokens of a capacity of %lld", static_cast<long long>(max_tokens),
                static_cast<long long>(capacity));
  if (mask_kind < TQ_MASK_NONE || mask_kind > TQ_MASK_ADD_BF16)
    return fail(TQ_ERR_INVALID_ARGUMENT, "tq_attention_affine: mask_kind %d", mask_kind);
  if (mask_kind != TQ_MASK_NONE && max_tokens > 0 && (!mask || !mask_strides))
    return fail(TQ_ERR_INVALID_ARGUMENT, "tq_attention_affine: a mask without its pointer or strides");
  const int64_t rows64 = static_cast<int64_t>(Hq / Hkv) * L;
  if (rows64 > INT32_MAX / 4 || rows_of(B, Hq, L) > INT32_MAX / 4)
    return fail(TQ_ERR_UNSUPPORTED, "tq_attention_affine: %lld query rows", static_cast<long long>(rows_of(B, Hq, L)));
  if (B == 0 || Hq == 0 || L == 0) return TQ_OK;
  if (!q || !out || (max_tokens > 0 && (!k_codes || !k_params || !v_codes || !v_params)))
    return fail(TQ_ERR_INVALID_ARGUMENT, "tq_attention_affine: null pointer");
  const int64_t need = workspace_bytes(B, Hq, Hkv, L, v_dim, max_tokens);
  if (!workspace || workspace_bytes_given < need)
    return fail(TQ_ERR_WORKSPACE, "tq_attention_affine: workspace of %lld bytes, %lld needed",
                static_cast<long long>(workspace_bytes_given), static_cast<long long>(need));

  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k_codes) | reinterpret_cast<uintptr_t>(v_codes) |
       static_cast<uintptr_t>((q_stride_b | q_stride_h | q_stride_l) * (q_dtype == TQ_DTYPE_F32 ? 4 : 2))) & 15)
    return fail(TQ_ERR_INVALID_ARGUMENT, "tq_attention_affine: queries, their strides and the codes must be 16-byte aligned");

  const bool by_rows = rows_kernel(q_dtype, k_dim, v_dim, k_bits, v_bits, max_tokens);
  const RowsChoice rc = rows_choice(rows64, k_dim, v_dim, group, mask_kind);
  const bool by_tile = by_rows && tile_kernel(rows64, k_dim, v_dim, static_cast<int64_t>(B) * Hkv, max_tokens, mask_kind);
  const int block_rows = by_tile ? tile_rows(k_dim, v_dim) : by_rows ? rc.rows : kVecRows;
  const int64_t blocks1 = static_cast<int64_t>(B) * Hkv * ((rows64 + block_rows - 1) / block_rows);
  const bool ragged = seq_lens || seq_starts;
  const Plan pl = by_tile ? tile_plan(blocks1, max_tokens)
                  : by_rows ? plan_splits(blocks1, max_tokens, ragged ? kRaggedTarget : kRowsTarget, kRowsTokens)
                            : vector_plan(blocks1, max_tokens);
  AffineAttnParams p{};
  p.q = q;
  p.q_sb = q_stride_b, p.q_sh = q_stride_h, p.q_sl = q_stride_l;
  p.k_codes = k_codes, p.k_params = k_params, p.v_codes = v_codes, p.v_params = v_params;
  p.starts = seq_starts, p.lens = seq_lens;
  p.mask = mask, p.mask_kind = mask_kind;
  if (mask_kind != TQ_MASK_NONE && mask_strides)
    for (int i = 0; i < 5; ++i) p.mask_s[i] = mask_strides[i];
  p.causal = causal;
  p.capacity = capacity, p.max_tokens = max_tokens;
  p.B = B, p.Hkv = Hkv, p.R = Hq / Hkv, p.L = L;
  p.rows = static_cast<int>(rows64);
  p.k_dim = k_dim, p.v_dim = v_dim, p.group = group;
  p.scale = scale * 1.44269504088896341f;
  p.splits = pl.splits, p.split_tokens = pl.split_tokens;
  p.out = out;
  const int64_t n = rows_of(B, Hq, L) * pl.splits;
  p.part_ml = static_cast<float*>(workspace);
  p.part_o = reinterpret_cast<float*>(static_cast<char*>(workspace) + align256(n * 8));

  const int64_t blocks = blocks1 * pl.splits;
  if (blocks > INT32_MAX / 512) return fail(TQ_ERR_UNSUPPORTED, "tq_attention_affine: %lld workgroups", static_cast<long long>(blocks));
  hipStream_t st = static_cast<hipStream_t>(stream);
  const unsigned n_blocks = static_cast<unsigned>(blocks);
  if (mask_kind != TQ_MASK_NONE && (by_tile || (by_rows && blocks1 * max_tokens >= kRangeTokens))) {
    p.keep.range = reinterpret_cast<int2*>(static_cast<char*>(workspace) + align256(n * 8) + align256(n * v_dim * 4));
    p.keep.nb = p.mask_s[0] || ragged ? B : 1;
    p.keep.ng = p.mask_s[1] ? Hkv : 1;
    p.keep.nr = p.mask_s[2] ? p.R : 1;
    p.keep.nl = p.mask_s[3] || causal ? L : 1;
    const unsigned mask_rows = static_cast<unsigned>(p.keep.nb * p.keep.ng * p.keep.nr * p.keep.nl);
    affine_mask_range_kernel<<<mask_rows, mask_rows <= 256 ? 512 : 256, 0, st>>>(p);
  }
  if (by_tile) {
    const int rc_launch = k_bits == 4   ? launch_tile_k4v4(p, q_dtype, st)
                          : v_bits == 4 ? launch_tile_k8v4(p, q_dtype, st)
                                        : launch_tile_k8v8(p, q_dtype, st);
    if (rc_launch != TQ_OK || pl.splits == 1) return rc_launch;
  } else if (by_rows) {
    const int rc_launch = k_bits == 4   ? launch_rows_k4v4(p, rc, q_dtype, st)
                          : v_bits == 4 ? launch_rows_k8v4(p, rc, q_dtype, st)
                                        : launch_rows_k8v8(p, rc, q_dtype, st);
    if (rc_launch != TQ_OK || pl.splits == 1) return rc_launch;
  } else if (q_dtype == TQ_DTYPE_F32) {
    launch_vector<TQ_DTYPE_F32>(p, k_bits, v_bits, n_blocks, st);
  } else if (q_dtype == TQ_DTYPE_F16) {
    launch_vector<TQ_DTYPE_F16>(p, k_bits, v_bits, n_blocks, st);
  } else {
    launch_vector<TQ_DTYPE_BF16>(p, k_bits, v_bits, n_blocks, st);
  }
  const int64_t out_rows = rows_of(B, Hq, L);
  if (q_dtype == TQ_DTYPE_F32)
    launch_merge<TQ_DTYPE_F32>(p, out_rows, st);
  else if (q_dtype == TQ_DTYPE_F16)
    launch_merge<TQ_DTYPE_F16>(p, out_rows, st);
  else
    launch_merge<TQ_DTYPE_BF16>(p, out_rows, st);
  return check_launch("tq_attention_affine");
}

}  // extern "C"
