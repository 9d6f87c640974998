// What the attention kernels share (gfx950, wave64): exchanges between a wave's halves,
// the order of workgroups, the loops over key blocks, and the fp32 operand forms.
// Layouts are those of fh_mfma.hpp; tensors are token-major.
#pragma once

#include <math.h>

#include "fh_common.hpp"
#include "fh_mfma.hpp"

namespace fh {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// The forward keeps a stale running maximum until a block's maximum exceeds it
// by more than this (log2 units): the softmax weights then stay <= 2^8, and
// the output rescale runs only when the maximum really grows.
constexpr float kRescaleSlack = 8.f;

// 2^x on the transcendental unit (v_exp_f32).  Denormal results flush to
// zero, which is harmless for softmax weights.
__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// max over lanes i and i^32 (v_permlane32_swap exchanges the two row halves).
__device__ __forceinline__ float xor32_max(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

__device__ __forceinline__ float xor32_sum(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

__device__ __forceinline__ bool wave_any(bool p) { return __builtin_amdgcn_ballot_w64(p) != 0; }

// 8 consecutive bf16 from global memory.
__device__ __forceinline__ bf16x8 ld_frag(const uint16_t* p) {
  return as_bf16x8(*reinterpret_cast<const uint4*>(p));
}

// Accumulator entries j0..j0+7 rounded to bf16 as an MFMA operand.
__device__ __forceinline__ bf16x8 pack_frag(const f32x16& acc, int j0) {
  return as_bf16x8(make_uint4(pk_bf16(acc[j0 + 0], acc[j0 + 1]), pk_bf16(acc[j0 + 2], acc[j0 + 3]),
                              pk_bf16(acc[j0 + 4], acc[j0 + 5]), pk_bf16(acc[j0 + 6], acc[j0 + 7])));
}

// XCD-aware block order.  Workgroup L = blockIdx.x + gridDim.x*blockIdx.y is
// dispatched to XCD L % 8 (8 XCDs, each with its own L2).  Grids here are
// (work items along x, heads along y) with causal work varying along x, so the
// identity mapping gives XCD k only the x == k (mod 8) items of every head: an
// up to 2.4x imbalance between XCDs at 16 items per head.  This maps XCD k's
// j-th workgroup to head y = k*(gridDim.y/8) + j % (gridDim.y/8) and rank
// x = j / (gridDim.y/8): every XCD covers all x of its own contiguous set of
// heads (balanced work; one head's K/V/Q/dO stay in one L2), ranks in order
// (rank 0 = dispatched first).  Needs gridDim.y % 8 == 0, else identity.
struct XcdOrder {
  int rank, y;
};
__device__ __forceinline__ XcdOrder xcd_order() {
  const int nx = gridDim.x, ny = gridDim.y;
  if (ny % 8 != 0) return {static_cast<int>(blockIdx.x), static_cast<int>(blockIdx.y)};
  const int L = blockIdx.x + nx * blockIdx.y;
  const int xcd = L & 7, j = L >> 3, nyx = ny >> 3;
  return {j / nyx, xcd * nyx + j % nyx};
}

// Stores a transposed accumulator tile (rows = head dims d, column = this
// lane's token) scaled by `mul` into one token-major output row.
template <int HD>
__device__ __forceinline__ void store_rows_T(uint16_t* out_row, const f32x16 (&acc)[HD / 32],
                                             float mul, int hl) {
#pragma unroll
  for (int dt = 0; dt < HD / 32; ++dt)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      uint2 w;
      w.x = pk_bf16(acc[dt][4 * g] * mul, acc[dt][4 * g + 1] * mul);
      w.y = pk_bf16(acc[dt][4 * g + 2] * mul, acc[dt][4 * g + 3] * mul);
      *reinterpret_cast<uint2*>(out_row + dt * 32 + 8 * g + 4 * hl) = w;
    }
}

// Rotary tables of the RoPE backward fused into the dQ and dK stores:
// cos / sin rows of head_dim elements in the gradients' dtype, one row per
// position (per_token == 0) or per token; cos == null means plain stores.
template <typename T>
struct RopeRows {
  const T* cos;
  const T* sin;
  int per_token;
  // Row of position `pos` of the sequence whose first token is row tok0.
  __device__ __forceinline__ int64_t row(int64_t tok0, int pos) const { return per_token ? tok0 + pos : pos; }
};

__device__ __forceinline__ void unpack4_bf16(uint2 w, float (&v)[4]) {
  v[0] = __uint_as_float(w.x << 16);
  v[1] = __uint_as_float(w.x & 0xffff0000u);
  v[2] = __uint_as_float(w.y << 16);
  v[3] = __uint_as_float(w.y & 0xffff0000u);
}

// The key-block loop of the forward and dQ kernels (4 waves): block kb + 1's
// K and V go straight into the other LDS stage (dma_tile) while
// body(kb, K, V) multiplies block kb; each wave waits for its own loads
// before the barrier that ends the block.  The two stages are separate
// arrays and the loop is unrolled by two, so every access names its stage
// and the compiler can tell that the loads into one stage do not alias the
// reads of the other (it would otherwise wait for them before every read).
// FAST: per-lane load addresses computed once (TileDma: no vector address
// arithmetic per load, 4-8 more registers); the dQ kernel, at the edge of an
// occupancy step, computes them per load instead (dma_tile).
// pre() runs once after block 0's loads are issued, before they are waited
// for (the kernel's own loads then overlap them).
template <int BN, int HD, bool FAST, int NW, class Body, class Pre>
__device__ __forceinline__ void kv_block_loop(const uint16_t* kb_ptr, int64_t ldk, const uint16_t* vb_ptr,
                                              int64_t ldv, int nkb, int S, char* sk0, char* sk1, char* sv0,
                                              char* sv1, int wave, int lane, Body&& body, Pre&& pre) {
  TileDma<BN, HD, NW> dk, dv;
  dk.init(ldk, wave, lane);
  dv.init(ldv, wave, lane);
  auto load = [&](int r0, char* KN, char* VN) __attribute__((always_inline)) {
    if constexpr (FAST) {
      dk.load(kb_ptr, ldk, r0, S - 1, KN, wave, lane);
      dv.load(vb_ptr, ldv, r0, S - 1, VN, wave, lane);
    } else {
      dk.load_asm(kb_ptr, ldk, r0, S - 1, KN, wave, lane);
      dv.load_asm(vb_ptr, ldv, r0, S - 1, VN, wave, lane);
    }
  };
  load(0, sk0, sv0);
  pre();
  wait_loads();
  __syncthreads();
  auto step = [&](int kb, const char* K, const char* V, char* KN, char* VN) __attribute__((always_inline)) {
    if (kb + 1 < nkb) load((kb + 1) * BN, KN, VN);
    if (kb < nkb) body(kb, K, V);
    wait_loads();
    __syncthreads();
  };
  for (int kb = 0; kb < nkb; kb += 2) {
    step(kb, sk0, sv0, sk1, sv1);
    step(kb + 1, sk1, sv1, sk0, sv0);
  }
}

// kv_block_loop with three LDS stages (the forward): block kb + 2's K and V are
// loaded while block kb is multiplied, so each block's loads have two blocks'
// time to land.  The barrier that ends a block waits for block kb + 1's loads
// only (vmcnt: the vector memory counter retires a wave's loads in issue
// order, and block kb + 2's loads are the wave's last ones), not for the ones
// still in flight into the third stage.
template <int BN, int HD, int NW, class Body, class Pre>
__device__ __forceinline__ void kv_block_loop3(const uint16_t* kb_ptr, int64_t ldk, const uint16_t* vb_ptr,
                                               int64_t ldv, int nkb, int S, char* sk0, char* sk1, char* sk2,
                                               char* sv0, char* sv1, char* sv2, int wave, int lane, Body&& body,
                                               Pre&& pre) {
  using Dma = TileDma<BN, HD, NW>;
  Dma dk, dv;
  dk.init(ldk, wave, lane);
  dv.init(ldv, wave, lane);
  // Loads this wave issues per block (K and V alike, in either of TileDma's paths).
  int per_wave = 0;
#pragma unroll
  for (int i = 0; i < Dma::PER; ++i) per_wave += (i * NW + wave < Dma::RUNS) ? 1 : 0;
  // The loads as inline asm (load_asm): the compiler, which cannot see the
  // waits below retire a stage's loads, would otherwise wait for every load
  // in flight before reading a stage.
  auto load = [&](int r0, char* KN, char* VN) __attribute__((always_inline)) {
    dk.load_asm(kb_ptr, ldk, r0, S - 1, KN, wave, lane);
    dv.load_asm(vb_ptr, ldv, r0, S - 1, VN, wave, lane);
  };
  load(0, sk0, sv0);
  if (nkb > 1) load(BN, sk1, sv1);
  pre();
  // vmcnt(0) as the builtin, which the compiler's own wait placement sees: it
  // then knows pre()'s loads have landed and puts no waits for them in the loop.
  __builtin_amdgcn_s_waitcnt(0x0f70);
  __syncthreads();
  auto step = [&](int kb, const char* K, const char* V, char* KN, char* VN) __attribute__((always_inline)) {
    const bool ahead = kb + 2 < nkb;
    if (ahead) load((kb + 2) * BN, KN, VN);
    if (kb < nkb) body(kb, K, V);
    if (ahead && per_wave == 1) asm volatile("s_waitcnt vmcnt(2)" ::: "memory");
    else if (ahead && per_wave == 2) asm volatile("s_waitcnt vmcnt(4)" ::: "memory");
    else wait_loads();
    lds_barrier();
  };
  for (int kb = 0; kb < nkb; kb += 3) {
    step(kb, sk0, sv0, sk2, sv2);
    step(kb + 1, sk1, sv1, sk0, sv0);
    step(kb + 2, sk2, sv2, sk1, sv1);
  }
}

// ------------------------------------------ backward: dK, dV (bf16), few workgroups
// The dK/dV kernels give a workgroup a key block of one kv head and loop over
// all of the group's query heads, so one short sequence with few kv heads is few
// workgroups (1 x 256 tokens, 32 / 4 heads of 64: 4 of them on 256 CUs).  There
// the group's heads are split over `n` workgroups (HeadSplit), each of which
// writes its fp32 sums to `part`; k_attn_dkdv_sum adds them in head order and
// stores dK and dV as the kernels do.  63 -> 12 + 6 us at that size, 81 -> 21 + 7 us at
// 3 x 333.
struct HeadSplit {
  float* part;  // [n][2][B*S][nkv][HD] (dK, dV), n > 1
  int n;
  __device__ __forceinline__ float* row(int split, int which, int64_t tokens, int64_t tok, int nkv, int kvh,
                                        int hd) const {
    return part + (((static_cast<int64_t>(split) * 2 + which) * tokens + tok) * nkv + kvh) * hd;
  }
};

// store_rows_T's elements as fp32.
template <int HD>
__device__ __forceinline__ void store_rows_T_f32(float* out_row, const f32x16 (&acc)[HD / 32], int hl) {
#pragma unroll
  for (int dt = 0; dt < HD / 32; ++dt)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      *reinterpret_cast<float4*>(out_row + dt * 32 + 8 * g + 4 * hl) =
          make_float4(acc[dt][4 * g], acc[dt][4 * g + 1], acc[dt][4 * g + 2], acc[dt][4 * g + 3]);
}

// One thread: dims d .. d+3 and d + HD/2 .. of one (token, kv head) of dK and dV.
template <int HD>
__device__ __forceinline__ void attn_dkdv_sum(HeadSplit hs, uint16_t* __restrict__ dk, int64_t lddk,
                                              uint16_t* __restrict__ dv, int64_t lddv, int S, int64_t tokens, int nkv,
                                              float scale, RopeRows<uint16_t> rope) {
  constexpr int C = HD / 8;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= tokens * nkv * C) return;
  const int d = static_cast<int>(i % C) * 4;
  const int64_t th = i / C, t = th / nkv;
  const int kvh = static_cast<int>(th - t * nkv);
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    float a[8];
    for (int sp = 0; sp < hs.n; ++sp) {
      const float* p = hs.row(sp, which, tokens, t, nkv, kvh, HD) + d;
      const float4 lo = *reinterpret_cast<const float4*>(p), hi = *reinterpret_cast<const float4*>(p + HD / 2);
      const float v[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
      for (int e = 0; e < 8; ++e) a[e] = sp == 0 ? v[e] : a[e] + v[e];
    }
    if (which == 0) {
#pragma unroll
      for (int e = 0; e < 8; ++e) a[e] *= scale;
      if (rope.cos) {
        const int64_t b = t / S, at = rope.row(b * S, static_cast<int>(t - b * S)) * HD + d;
        float c0[4], c1[4], s0[4], s1[4];
        unpack4_bf16(*reinterpret_cast<const uint2*>(rope.cos + at), c0);
        unpack4_bf16(*reinterpret_cast<const uint2*>(rope.cos + at + HD / 2), c1);
        unpack4_bf16(*reinterpret_cast<const uint2*>(rope.sin + at), s0);
        unpack4_bf16(*reinterpret_cast<const uint2*>(rope.sin + at + HD / 2), s1);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float o0, o1;
          rope_pair<uint16_t, true>(round_bf(a[e]), round_bf(a[e + 4]), c0[e], c1[e], s0[e], s1[e], o0, o1);
          a[e] = o0;
          a[e + 4] = o1;
        }
      }
    }
    uint16_t* out = which == 0 ? dk + t * lddk : dv + t * lddv;
    out += static_cast<int64_t>(kvh) * HD + d;
    *reinterpret_cast<uint2*>(out) = make_uint2(pk_bf16(a[0], a[1]), pk_bf16(a[2], a[3]));
    *reinterpret_cast<uint2*>(out + HD / 2) = make_uint2(pk_bf16(a[4], a[5]), pk_bf16(a[6], a[7]));
  }
}

template <int HD>
__global__ __launch_bounds__(256) void k_attn_dkdv_sum(HeadSplit hs, uint16_t* __restrict__ dk, int64_t lddk,
                                                       uint16_t* __restrict__ dv, int64_t lddv, int S,
                                                       int64_t tokens, int nkv, float scale,
                                                       RopeRows<uint16_t> rope) {
  attn_dkdv_sum<HD>(hs, dk, lddk, dv, lddv, S, tokens, nkv, scale, rope);
}

// ------------------------------------------------------------- fp32 operands
// v_mfma_f32_16x16x4_f32, whose products and sums are fp32.  Lane i of an operand
// holds row / column r = i%16 and k index c = i/16 of four; lane i of the accumulator
// holds column r and rows 4c .. 4c+3.
__device__ __forceinline__ f32x4 mfma_f32(float a, float b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ f32x4 zero4() { return f32x4{0.f, 0.f, 0.f, 0.f}; }

// max / sum over the four lanes that share a column (same r, c = 0..3).
__device__ __forceinline__ float col_max(float v) {
  v = fmaxf(v, __shfl_xor(v, 16, kWave));
  return fmaxf(v, __shfl_xor(v, 32, kWave));
}
__device__ __forceinline__ float col_sum(float v) {
  v += __shfl_xor(v, 16, kWave);
  return v + __shfl_xor(v, 32, kWave);
}

template <int HD>
using FragF32 = f32x4[HD / 16];

template <int HD>
__device__ __forceinline__ void load_frag_f32(FragF32<HD>& f, const float* row, int c) {
#pragma unroll
  for (int u = 0; u < HD / 16; ++u) f[u] = *reinterpret_cast<const f32x4*>(row + 16 * u + 4 * c);
}

// a b^T over the head dims: accumulator rows = a's rows, columns = b's rows.
template <int HD>
__device__ __forceinline__ f32x4 dot_f32(const FragF32<HD>& a, const FragF32<HD>& b) {
  f32x4 acc = zero4();
#pragma unroll
  for (int u = 0; u < HD / 16; ++u)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc = mfma_f32(a[u][e], b[u][e], acc);
  return acc;
}

// acc[dt] (rows m: dim ND*m + dt, columns as w's) += sum over the block's 32 rows
// of row[.][dim] * w[row][column]; row n of the block is rows + min(n, last) * ld.
// Rows with n outside [lo, hi) of this lane's column are masked (their w is 0).
// `partial`: some row is masked for some column.  There a row that holds an
// infinity or a NaN must not reach the columns that do not see it (0 * inf), so
// 16 rows with one are summed row by row on the vector unit.
template <int HD>
__device__ __forceinline__ void wsum_f32(f32x4 (&acc)[HD / 16], const f32x4 (&w)[2], const float* rows, int64_t ld,
                                         int last, bool partial, int lo, int hi, int r, int c) {
  constexpr int ND = HD / 16;
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    float v[4][ND];
    bool bad = false;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float* src = rows + min(16 * t + 4 * c + e, last) * ld + ND * r;
#pragma unroll
      for (int d = 0; d < ND; d += 2) {
        const float2 p = *reinterpret_cast<const float2*>(src + d);
        v[e][d] = p.x;
        v[e][d + 1] = p.y;
        bad |= !(fabsf(p.x) < INFINITY) || !(fabsf(p.y) < INFINITY);
      }
    }
    if (partial && wave_any(bad)) {
      for (int n = 0; n < 16; ++n) {
        const int e = n & 3;
        const float mine = e == 0 ? w[t][0] : e == 1 ? w[t][1] : e == 2 ? w[t][2] : w[t][3];
        const float p = __shfl(mine, r + 16 * (n >> 2), kWave);
        if (16 * t + n < lo || 16 * t + n >= hi) continue;
        const float* src = rows + min(16 * t + n, last) * ld + 4 * ND * c;
#pragma unroll
        for (int g = 0; g < 4; ++g)
#pragma unroll
          for (int dt = 0; dt < ND; ++dt) acc[dt][g] = fmaf(p, src[ND * g + dt], acc[dt][g]);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int dt = 0; dt < ND; ++dt) acc[dt] = mfma_f32(v[e][dt], w[t][e], acc[dt]);
    }
  }
}

// A wave's accumulators into an LDS tile [16 columns][HD + 4] (one row per
// accumulator column).
template <int HD>
__device__ __forceinline__ void put_tile_f32(float* tile, const f32x4 (&acc)[HD / 16], int r, int c) {
  constexpr int ND = HD / 16;
#pragma unroll
  for (int e = 0; e < 4; ++e)
#pragma unroll
    for (int dt = 0; dt < ND; ++dt) tile[r * (HD + 4) + ND * (4 * c + e) + dt] = acc[dt][e];
}

template <int HD>
__device__ __forceinline__ void add_tile_f32(f32x4 (&acc)[HD / 16], const float* tile, int r, int c) {
  constexpr int ND = HD / 16;
#pragma unroll
  for (int e = 0; e < 4; ++e)
#pragma unroll
    for (int dt = 0; dt < ND; ++dt) acc[dt][e] += tile[r * (HD + 4) + ND * (4 * c + e) + dt];
}

// Sums the NW waves' accumulators into wave 0's, pairs of waves in a fixed order.
template <int HD, int NW>
__device__ __forceinline__ void sum_waves_f32(f32x4 (&acc)[HD / 16], float* tiles, int wave, int r, int c) {
  constexpr int TILE = 16 * (HD + 4);
#pragma unroll
  for (int half = NW / 2; half > 0; half >>= 1) {
    if (wave >= half && wave < 2 * half) put_tile_f32<HD>(tiles + (wave - half) * TILE, acc, r, c);
    __syncthreads();
    if (wave < half) add_tile_f32<HD>(acc, tiles + wave * TILE, r, c);
    __syncthreads();
  }
}

// Rows pos0 .. pos0 + 15 (those before S) of an output from an LDS tile, times
// mul, followed by the RoPE backward of each row when rope.cos is set.
template <int HD, int NT>
__device__ __forceinline__ void store_tile_f32(float* out, int64_t ld, const float* tile, int pos0, int S, float mul,
                                               const RopeRows<float>& rope, int64_t tok0) {
  for (int i = threadIdx.x; i < 16 * (HD / 2); i += NT) {
    const int row = i / (HD / 2), d = i % (HD / 2), pos = pos0 + row;
    if (pos >= S) break;  // rows ascend with i
    float o0 = tile[row * (HD + 4) + d] * mul, o1 = tile[row * (HD + 4) + d + HD / 2] * mul;
    if (rope.cos) {
      const int64_t t = rope.row(tok0, pos) * HD + d;
      rope_pair<float, true>(o0, o1, rope.cos[t], rope.cos[t + HD / 2], rope.sin[t], rope.sin[t + HD / 2], o0, o1);
    }
    float* dst = out + (tok0 + pos) * ld + d;
    dst[0] = o0;
    dst[HD / 2] = o1;
  }
}

}  // namespace
}  // namespace fh
