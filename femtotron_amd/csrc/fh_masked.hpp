// What the kernels of attention under a mask share: the table of what a token sees,
// the scores' cap and bias, and products that keep infinities and NaN where they are
// seen.
#pragma once

#include "femtohip_packed.h"
#include "fh_attn.hpp"

namespace fh {

// fh_attn_mask's table: a row's ranges, their bounds over 32 rows, and for more than
// kOrderedRows rows the blocks of 128 queries, 128 keys and 64 keys by falling work.  A row sees keys [x, y) and is seen by queries [z, w); of 32
// rows `keys` and `queries` hold (smallest first, largest end, largest first, smallest
// end) over the rows that see (are seen by) something: a range that misses [x, y) has
// nothing for them, one inside [z, w) is seen by all of them.
struct MaskTable {
  const int4* rows;
  const int4* keys;
  const int4* queries;
  const int* order_q;  // null: as they come
  const int* order_k128;
  const int* order_k64;
};

constexpr int kMaskRows = 32;
// Up to here a head's blocks run at once whatever their order.
constexpr int64_t kOrderedRows = 1024;

inline int64_t mask_tiles(int64_t tokens) { return (tokens + kMaskRows - 1) / kMaskRows; }
inline int64_t mask_blocks(int64_t tokens, int64_t rows) { return (tokens + rows - 1) / rows; }

inline size_t mask_bytes(int64_t tokens) {
  const int64_t order = tokens > kOrderedRows ? 2 * mask_blocks(tokens, 128) + mask_blocks(tokens, 64) : 0;
  return static_cast<size_t>(tokens + 2 * mask_tiles(tokens)) * sizeof(int4) + static_cast<size_t>(order) * sizeof(int);
}

inline MaskTable mask_table(const void* table, int64_t tokens) {
  const int4* rows = static_cast<const int4*>(table);
  const int4* keys = rows + tokens;
  const int4* queries = keys + mask_tiles(tokens);
  if (tokens <= kOrderedRows) return {rows, keys, queries, nullptr, nullptr, nullptr};
  const int* order = reinterpret_cast<const int*>(queries + mask_tiles(tokens));
  const int64_t n = mask_blocks(tokens, 128);
  return {rows, keys, queries, order, order + n, order + 2 * n};
}

namespace {

// Ranges' bounds over tiles [t, t + N), those before `tiles` (nothing: x > y); t is uniform,
// and so is the result, in scalar registers: what it decides are branches, not selects.
template <int N>
__device__ __forceinline__ int4 mask_bounds(const int4* b, int t, int tiles) {
  int4 r = make_int4(0x7fffffff, 0, 0, 0x7fffffff);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int4 v = b[min(t + i, tiles - 1)];  // a tile twice changes nothing
    if (t < tiles) r = make_int4(min(r.x, v.x), max(r.y, v.y), max(r.z, v.z), min(r.w, v.w));
  }
  return make_int4(__builtin_amdgcn_readfirstlane(r.x), __builtin_amdgcn_readfirstlane(r.y),
                   __builtin_amdgcn_readfirstlane(r.z), __builtin_amdgcn_readfirstlane(r.w));
}

// The order's buckets: blocks whose lengths are the same in these units come in any order.
__device__ __forceinline__ int order_unit(int T) { return max(32, (T + 1022) / 1023); }

// Which block and head (y) a workgroup takes.  Ranks run by falling work, the heaviest first
// on every XCD (workgroup L runs on XCD L % 8): with a multiple of eight heads each XCD has
// heads of its own, whose tensors stay in its L2; else ranks and heads are dealt out in turn.
// 16384 tokens in rows of 2048, 32/4 heads of 64, backward: XCDs by position in the row (block
// x on XCD x % 8) 956 us, dealt out by falling work 635.
__device__ __forceinline__ XcdOrder masked_order() {
  if (gridDim.y % 8 == 0) return xcd_order();
  const int L = blockIdx.x + gridDim.x * blockIdx.y, ny = gridDim.y;
  return {L / ny, L % ny};
}
// The same of the grid's first `ny` heads' worth of workgroups; y = ny: none is left.
__device__ __forceinline__ XcdOrder masked_order(int ny) {
  const int L = blockIdx.x + gridDim.x * blockIdx.y;
  if (L >= static_cast<int>(gridDim.x) * ny) return {0, ny};
  if (ny % 8 != 0) return {L / ny, L % ny};
  const int j = L >> 3, nyx = ny >> 3;
  return {j / nyx, (L & 7) * nyx + j % nyx};
}

// --------------------------------------------------------------------- scores
// Scores in log2 units, from the raw products x = q . k:
//   z2 = x scale_log2                                      MODE 0
//   z2 = cap_log2 tanh(x scale / cap)                      kCap
//   z2 -= slope_log2 |i - j|                               kBias
// tanh(u) = 1 - 2 r with r = 1 / (1 + e^2u), its derivative 4 r (1 - r): one v_exp and one
// v_rcp, off by about 2^-23 of tanh's 1 (of the cap in the scores).  What counts is the
// number of vector instructions, and the two cost no more than others, so z2 = cap_log2 - 2
// cap_log2 r is folded into the sums with the maximum or -lse that follow, and the 4 into
// the scale of the gradients.  (Polynomials of (x scale / cap)^2 for tiles whose scores are
// small, without either: 8192 tokens, 32/8 heads of 128, forward 663 -> 678 us, backward 2547
// -> 2947.)
constexpr int kCap = 1, kBias = 2;

struct ScoreArgs {
  float scale;       // of the gradients of q and k
  float scale_log2;  // scale * log2(e)
  float in;          // scale / cap
  float in2;         // 2 log2(e) scale / cap
  float cap_log2;    // cap * log2(e)
  const float* slopes;
};

template <int MODE>
struct Score {
  float a;    // on the raw product: scale_log2, or in2 before the cap
  float c;    // -2 cap_log2, on r
  float b;    // cap_log2, without a cap 0
  float slope;
  __device__ __forceinline__ Score(const ScoreArgs& s, int h) {
    a = (MODE & kCap) ? s.in2 : s.scale_log2;
    c = (MODE & kCap) ? -2.f * s.cap_log2 : 1.f;
    b = (MODE & kCap) ? s.cap_log2 : 0.f;
    slope = (MODE & kBias) ? s.slopes[h] * kLog2e : 0.f;
  }
  // r of the comment above.
  __device__ __forceinline__ float half_sigmoid(float x) const {
    return __builtin_amdgcn_rcpf(1.f + fast_exp2(x * a));
  }
  // The score, `away` tokens apart.
  __device__ __forceinline__ float operator()(float x, float away) const {
    const float low = (MODE & kBias) ? fmaf(-slope, fabsf(away), b) : b;
    if constexpr (MODE & kCap) return fmaf(c, half_sigmoid(x), low);
    return fmaf(x, a, low);
  }
  // e^(z - lse) with nl = b - lse * log2(e), and under a cap a quarter of the score's derivative,
  // 0 for a score that is NaN (the weight is NaN then, and 0 where the score is not seen: 0 times
  // this stays 0).  The bounds are a modifier of the fma.
  __device__ __forceinline__ float weight(float x, float away, float nl, float& quarter) const {
    const float low = (MODE & kBias) ? fmaf(-slope, fabsf(away), nl) : nl;
    if constexpr (MODE & kCap) {
      const float r = half_sigmoid(x);
      quarter = __builtin_amdgcn_fmed3f(fmaf(-r, r, r), 0.f, 1.f);
      return fast_exp2(fmaf(c, r, low));
    } else {
      quarter = 1.f;
      return fast_exp2(fmaf(x, a, low));
    }
  }
};

// What the sums of dS k and dS q are times: the scale, and the 4 of the cap's derivative.
template <int MODE>
__device__ __forceinline__ float grad_scale(const ScoreArgs& s) {
  return (MODE & kCap) ? 4.f * s.scale : s.scale;
}

// ------------------------------------------------------------ o beyond bf16
// The four fp32 values x as bf16 (pk_bf16) and the next eight bits of each, signed: what
// its bits are over those of the bf16 value, in steps of 2^8 (a bf16 step is 2^16).
__device__ __forceinline__ uint32_t low_bits(const float (&x)[4], uint2 rounded) {
  const uint32_t r[4] = {rounded.x << 16, rounded.x & 0xffff0000u, rounded.y << 16, rounded.y & 0xffff0000u};
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int d = static_cast<int>(__float_as_uint(x[i]) - r[i]);  // within +-2^15
    w |= (static_cast<uint32_t>(min((d + 128) >> 8, 127)) & 0xffu) << (8 * i);
  }
  return w;
}

// A bf16 value's bits (in the high half) with its low_bits byte i of w.
__device__ __forceinline__ float with_low(uint32_t high, uint32_t w, int i) {
  return __uint_as_float(high + static_cast<uint32_t>(static_cast<int>(static_cast<int8_t>(w >> (8 * i))) << 8));
}

// ------------------------------------------------------- what is not seen
// A weight of 0 does not keep an infinity or a NaN out of a sum on the matrix cores
// (0 * inf).  A tile that some column sees a part of may bring one from a row that the
// column does not see; the sums then hold a NaN, for a sum that has met one never loses
// it.  The kernels therefore look at their finished sums once, and where a column that
// sees something holds no finite value, the workgroup computes all of it again with
// wsum_careful in those tiles, at a sixteenth of the speed: what is left are the
// infinities and NaN that the column does see.

// Whether the sums hold an infinity or a NaN.
template <int ND>
__device__ __forceinline__ bool not_finite(const f32x16 (&acc)[ND]) {
  float s = 0.f;
#pragma unroll
  for (int dt = 0; dt < ND; ++dt)
#pragma unroll
    for (int j = 0; j < 16; ++j) s = fmaf(acc[dt][j], 0.f, s);
  return s != s;
}

// acc += X^T f over rows row0 .. row0+15 of the tile X, of which this lane's column sees
// rows lo <= row < hi: one row at a time, the others zero, and the columns that do not see
// it keep their sums.
template <int HD>
__device__ __forceinline__ void wsum_careful(f32x16 (&acc)[HD / 32], bf16x8 f, const char* tile, int b0, int b8,
                                             int row0, int lo, int hi, int hl) {
#pragma unroll 1
  for (int n = 0; n < 16; ++n) {
    // Row n is element e of the lanes of one half (the permuted order of lds_frag_tr).
    const int e = (n & 3) + ((n >> 3) << 2);
    const bool mine = hl == ((n >> 2) & 1);
    const uint32_t m = (e & 1) ? 0xffff0000u : 0x0000ffffu;
    const uint32_t m0 = mine && (e >> 1) == 0 ? m : 0, m1 = mine && (e >> 1) == 1 ? m : 0;
    const uint32_t m2 = mine && (e >> 1) == 2 ? m : 0, m3 = mine && (e >> 1) == 3 ? m : 0;
    const bool seen = row0 + n >= lo && row0 + n < hi;
#pragma unroll
    for (int dt = 0; dt < HD / 32; ++dt) {
      const uint4 u = __builtin_bit_cast(uint4, lds_frag_tr<HD>(tile, b0, b8, row0, dt));
      const f32x16 t = mfma(as_bf16x8(make_uint4(u.x & m0, u.y & m1, u.z & m2, u.w & m3)), f, acc[dt]);
#pragma unroll
      for (int j = 0; j < 16; ++j) acc[dt][j] = seen ? t[j] : acc[dt][j];
      __builtin_amdgcn_sched_barrier(0);  // one block's 16 registers at a time
    }
  }
}

// x = `none` outside lo <= c < hi, c = the accumulator entry's row (less 4 hl) plus `first`.
// Steps seen in part are few, so each side is a branch of its own, kept one by the empty
// asm (as selects that every step pays for: 32 comparisons and selects of a forward step's
// 270 vector instructions).
__device__ __forceinline__ void mask_range(f32x16& x, bool ends, bool starts, int lo, int hi, int first, float none) {
  if (ends) {
    asm volatile("");
#pragma unroll
    for (int j = 0; j < 16; ++j) x[j] = first + acc_row(j, 0) < hi ? x[j] : none;
  }
  if (starts) {
    asm volatile("");
#pragma unroll
    for (int j = 0; j < 16; ++j) x[j] = first + acc_row(j, 0) >= lo ? x[j] : none;
  }
}

// What pack_frag's rounding leaves of entries j0 .. j0+7, rounded again.
__device__ __forceinline__ bf16x8 rest_frag(const f32x16& acc, int j0) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float a = acc[j0 + 2 * i], b = acc[j0 + 2 * i + 1];
    const uint32_t r = pk_bf16(a, b);
    w[i] = pk_bf16(a - __uint_as_float(r << 16), b - __uint_as_float(r & 0xffff0000u));
  }
  return as_bf16x8(make_uint4(w[0], w[1], w[2], w[3]));
}

// acc += X^T f over rows row0 .. row0+15 of the tile X.
template <int HD>
__device__ __forceinline__ void wsum(f32x16 (&acc)[HD / 32], bf16x8 f, const char* tile, int b0, int b8, int row0) {
#pragma unroll
  for (int dt = 0; dt < HD / 32; ++dt) acc[dt] = mfma(lds_frag_tr<HD>(tile, b0, b8, row0, dt), f, acc[dt]);
}

}  // namespace

// ------------------------------------------------------------------------ host
// The checks and constants of a call, for every dtype.
struct MaskedArgs {
  int64_t tokens, n_heads, n_kv_heads, head_dim;
  ScoreArgs score;
  int mode;
};

int masked_args(const char* name, fh_dtype dt, int64_t tokens, int64_t n_heads, int64_t n_kv_heads, int64_t head_dim,
                float scale, float cap, const float* slopes, MaskedArgs& a);

// A row stride of heads of head_dim.
int masked_stride(const char* name, const char* what, int64_t ld, int64_t heads, int64_t head_dim);

struct MaskedFwd {
  const void *q, *k, *v;
  int64_t ldq, ldk, ldv;
  void* o;
  int64_t ldo;
  float* lse;
  int8_t* o_low;
  MaskTable table;
};

struct MaskedBwd {
  const void *q, *k, *v, *o, *dout;
  int64_t ldq, ldk, ldv, ldo, lddo;
  const float* lse;
  const int8_t* o_low;
  void *dq, *dk, *dv;
  int64_t lddq, lddk, lddv;
  MaskTable table;
  float* workspace;
};

void masked_fwd_bf16(const MaskedFwd& c, const MaskedArgs& a, hipStream_t stream);
void masked_bwd_bf16(const MaskedBwd& c, const MaskedArgs& a, hipStream_t stream);
void masked_fwd_f32(const MaskedFwd& c, const MaskedArgs& a, hipStream_t stream);
void masked_bwd_f32(const MaskedBwd& c, const MaskedArgs& a, hipStream_t stream);

// Workspace of the backward, in floats: delta and -lse * log2(e) [n_heads, tokens], then
// from `parts` on the sums of a kv head's query heads where they are split.
struct MaskedWorkspace {
  int64_t parts, total;
  int split, long_split;  // where what sees the keys is long (long_split >= split)
};
MaskedWorkspace masked_workspace(fh_dtype dt, int64_t tokens, int64_t n_heads, int64_t n_kv_heads, int64_t head_dim);

template <typename F>
void dispatch_masked(int64_t head_dim, int mode, F&& f) {
  auto with_mode = [&](auto hd) {
    if (mode == 0) f(hd, std::integral_constant<int, 0>{});
    else if (mode == kCap) f(hd, std::integral_constant<int, kCap>{});
    else if (mode == kBias) f(hd, std::integral_constant<int, kBias>{});
    else f(hd, std::integral_constant<int, kCap | kBias>{});
  };
  if (head_dim == 32) with_mode(std::integral_constant<int, 32>{});
  else if (head_dim == 64) with_mode(std::integral_constant<int, 64>{});
  else with_mode(std::integral_constant<int, 128>{});
}

}  // namespace fh
