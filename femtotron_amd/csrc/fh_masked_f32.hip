// Attention under a mask in fp32 (fp32 models: debugging and parity runs), forward and
// backward, on v_mfma_f32_16x16x4_f32 in the operand forms of fh_attn.hpp: 16 queries of
// a head (16 keys of a kv head) a workgroup, the blocks of 32 keys that they see (the
// blocks of 32 queries that see them, of each query head) shared out over its waves.
// tanh is the math library's: v_exp and v_rcp leave 2^-23 of the cap in the scores, ten
// times what the products leave.  One causal document, 32/4 heads of 64, forward and backward:
// 1024 tokens 96 and 425 us (45 and 25 TFLOP/s), 4096 909 and 3860 (76 and 45); 32/8 heads of
// 128, 4096 tokens, 1762 and 7365 (78 and 47), the causal kernels' times; a large fp32
// product runs at 153.
#include <type_traits>

#include "fh_masked.hpp"

namespace fh {
namespace {

template <int MODE>
struct ScoreF32 {
  float a, b, slope;
  __device__ __forceinline__ ScoreF32(const ScoreArgs& s, int h) {
    a = (MODE & kCap) ? s.in : s.scale_log2;
    b = s.cap_log2;
    slope = (MODE & kBias) ? s.slopes[h] * kLog2e : 0.f;
  }
  // The score of x in log2 units, `away` tokens apart, and its derivative by s.
  __device__ __forceinline__ float operator()(float x, int away, float& slope_of) const {
    float z;
    slope_of = 1.f;
    if constexpr (MODE & kCap) {
      const float t = tanhf(x * a);
      slope_of = fmaf(-t, t, 1.f);
      z = t * b;
    } else {
      z = x * a;
    }
    return (MODE & kBias) ? fmaf(-slope, static_cast<float>(abs(away)), z) : z;
  }
};

// Rows pos0 .. pos0 + 15 (those before T) of an output from an LDS tile, times mul.
template <int HD, int NT>
__device__ __forceinline__ void store_rows_f32(float* out, int64_t ld, const float* tile, int pos0, int T, float mul) {
  store_tile_f32<HD, NT>(out, ld, tile, pos0, T, mul, RopeRows<float>{nullptr, nullptr, 0}, 0);
}

template <int ND>
__device__ __forceinline__ void zero_unless(f32x4 (&acc)[ND], bool some) {
#pragma unroll
  for (int dt = 0; dt < ND; ++dt)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[dt][e] = some ? acc[dt][e] : 0.f;
}

template <int HD, int MODE>
__global__ __launch_bounds__(256) void k_masked_fwd_f32(const float* __restrict__ q, int64_t ldq,
                                                        const float* __restrict__ k, int64_t ldk,
                                                        const float* __restrict__ v, int64_t ldv,
                                                        float* __restrict__ o, int64_t ldo, float* __restrict__ lse,
                                                        int T, int group, ScoreArgs args, MaskTable mask) {
  constexpr int NU = HD / 16, TILE = 16 * (HD + 4);
  __shared__ __align__(16) float tiles[2 * TILE];
  __shared__ float sm[4][16], sl[4][16];
  const int lane = threadIdx.x & 63, r = lane & 15, c = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int h = blockIdx.y, kvh = h / group;
  const int q0 = static_cast<int>(gridDim.x - 1 - blockIdx.x) * 16, qi = q0 + r, qc = min(qi, T - 1);
  const int4 mine = mask.keys[q0 / kMaskRows];
  const int2 sees = qi < T ? *reinterpret_cast<const int2*>(mask.rows + qi) : make_int2(0, 0);
  const bool some = sees.x < sees.y;
  const ScoreF32<MODE> score(args, h);
  FragF32<HD> qf;
  load_frag_f32<HD>(qf, q + static_cast<int64_t>(qc) * ldq + static_cast<int64_t>(h) * HD, c);
  f32x4 oacc[NU];
#pragma unroll
  for (int dt = 0; dt < NU; ++dt) oacc[dt] = zero4();
  float m = -INFINITY, l = 0.f;
  const float* kp = k + static_cast<int64_t>(kvh) * HD;
  const float* vp = v + static_cast<int64_t>(kvh) * HD;
  const int n_steps = mine.y > mine.x ? (mine.y - mine.x + 31) / 32 : 0;
  for (int kb = wave; kb < n_steps; kb += 4) {
    const int k0 = mine.x + kb * 32;
    const int lo = sees.x - k0, hi = sees.y - k0;  // keys n of the block with lo <= n < hi are seen
    f32x4 x[2];  // rows = keys, column = query
    float mloc = -INFINITY;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      FragF32<HD> kf;
      load_frag_f32<HD>(kf, kp + static_cast<int64_t>(min(k0 + 16 * t + r, T - 1)) * ldk, c);
      x[t] = dot_f32<HD>(kf, qf);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int n = 16 * t + 4 * c + e;
        float d;
        const float z = score(x[t][e], qi - k0 - n, d);
        x[t][e] = n >= lo && n < hi ? z : -INFINITY;
        mloc = fmaxf(mloc, x[t][e]);
      }
    }
    const float mn = fmaxf(m, col_max(mloc));
    const float ms = mn == -INFINITY ? 0.f : mn;  // no key so far: weights 0, not exp2(-inf + inf)
    const float alpha = fast_exp2(m - ms);
    m = mn;
    l *= alpha;
#pragma unroll
    for (int dt = 0; dt < NU; ++dt) oacc[dt] *= alpha;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[t][e] = fast_exp2(x[t][e] - ms);
        l += x[t][e];
      }
    wsum_f32<HD>(oacc, x, vp + static_cast<int64_t>(k0) * ldv, ldv, T - 1 - k0, !(mine.z <= k0 && mine.w >= k0 + 32),
                 lo, hi, r, c);
  }
  // The waves' results meet: weights 2^(m_w - m), zero for a wave without keys.
  l = col_sum(l);
  if (c == 0) {
    sm[wave][r] = m;
    sl[wave][r] = l;
  }
  __syncthreads();
  const float mt = fmaxf(fmaxf(sm[0][r], sm[1][r]), fmaxf(sm[2][r], sm[3][r]));
  float lt = 0.f;
#pragma unroll
  for (int w = 0; w < 4; ++w) lt += sl[w][r] * fast_exp2(sm[w][r] - mt);
  const float mul = fast_exp2(m - mt) / lt;
#pragma unroll
  for (int dt = 0; dt < NU; ++dt) oacc[dt] *= mul;
  zero_unless<NU>(oacc, some);
  sum_waves_f32<HD, 4>(oacc, tiles, wave, r, c);
  if (wave == 0) {
    put_tile_f32<HD>(tiles, oacc, r, c);
    if (lse != nullptr && c == 0 && qi < T) lse[static_cast<int64_t>(h) * T + qi] = some ? (mt + log2f(lt)) * kLn2 : 0.f;
  }
  __syncthreads();
  store_rows_f32<HD, 256>(o + static_cast<int64_t>(h) * HD, ldo, tiles, q0, T, 1.f);
}

// Also writes delta = rowsum(dO O) and -lse * log2(e), which the dK/dV kernel reads.
template <int HD, int MODE>
__global__ __launch_bounds__(256) void k_masked_dq_f32(
    const float* __restrict__ q, int64_t ldq, const float* __restrict__ k, int64_t ldk, const float* __restrict__ v,
    int64_t ldv, const float* __restrict__ o, int64_t ldo, const float* __restrict__ dO, int64_t lddo,
    const float* __restrict__ lse, float* __restrict__ delta, float* __restrict__ nl2, float* __restrict__ dq,
    int64_t lddq, int T, int group, ScoreArgs args, MaskTable mask) {
  constexpr int NU = HD / 16, TILE = 16 * (HD + 4);
  __shared__ __align__(16) float tiles[2 * TILE];
  const int lane = threadIdx.x & 63, r = lane & 15, c = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int h = blockIdx.y, kvh = h / group;
  const int q0 = static_cast<int>(gridDim.x - 1 - blockIdx.x) * 16, qi = q0 + r, qc = min(qi, T - 1);
  const int4 mine = mask.keys[q0 / kMaskRows];
  const int2 sees = qi < T ? *reinterpret_cast<const int2*>(mask.rows + qi) : make_int2(0, 0);
  const bool some = sees.x < sees.y;
  const ScoreF32<MODE> score(args, h);
  const int64_t col = static_cast<int64_t>(h) * HD;
  FragF32<HD> qf, gf;
  float dl = 0.f;
  {
    FragF32<HD> of;
    load_frag_f32<HD>(qf, q + qc * ldq + col, c);
    load_frag_f32<HD>(gf, dO + qc * lddo + col, c);
    load_frag_f32<HD>(of, o + qc * ldo + col, c);
#pragma unroll
    for (int u = 0; u < NU; ++u)
#pragma unroll
      for (int e = 0; e < 4; ++e) dl = fmaf(gf[u][e], of[u][e], dl);
  }
  dl = col_sum(dl);
  const int64_t at = static_cast<int64_t>(h) * T + qc;
  const float nlse2 = -lse[at] * kLog2e;
  if (wave == 0 && c == 0 && qi < T) {
    delta[at] = dl;
    nl2[at] = nlse2;
  }
  f32x4 acc[NU];
#pragma unroll
  for (int dt = 0; dt < NU; ++dt) acc[dt] = zero4();
  const float* kp = k + static_cast<int64_t>(kvh) * HD;
  const float* vp = v + static_cast<int64_t>(kvh) * HD;
  const int n_steps = mine.y > mine.x ? (mine.y - mine.x + 31) / 32 : 0;
  for (int kb = wave; kb < n_steps; kb += 4) {
    const int k0 = mine.x + kb * 32;
    const int lo = sees.x - k0, hi = sees.y - k0;
    f32x4 x[2];  // dS^T: rows = keys, column = query
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int64_t row = min(k0 + 16 * t + r, T - 1);
      FragF32<HD> f;
      load_frag_f32<HD>(f, kp + row * ldk, c);
      x[t] = dot_f32<HD>(f, qf);
      load_frag_f32<HD>(f, vp + row * ldv, c);
      const f32x4 y = dot_f32<HD>(f, gf);  // dP^T
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int n = 16 * t + 4 * c + e;
        float ds;
        const float z = score(x[t][e], qi - k0 - n, ds);
        x[t][e] = n >= lo && n < hi ? fast_exp2(z + nlse2) * (y[e] - dl) * ds : 0.f;
      }
    }
    wsum_f32<HD>(acc, x, kp + static_cast<int64_t>(k0) * ldk, ldk, T - 1 - k0, !(mine.z <= k0 && mine.w >= k0 + 32), lo,
                 hi, r, c);
  }
  zero_unless<NU>(acc, some);
  sum_waves_f32<HD, 4>(acc, tiles, wave, r, c);
  if (wave == 0) put_tile_f32<HD>(tiles, acc, r, c);
  __syncthreads();
  store_rows_f32<HD, 256>(dq + col, lddq, tiles, q0, T, args.scale);
}

// Waves of a dK/dV workgroup: 16 where the registers allow four per SIMD.
template <int HD>
constexpr int kMaskedWavesF32 = HD == 32 ? 16 : 8;

template <int HD, int MODE>
__global__ __launch_bounds__(64 * kMaskedWavesF32<HD>) void k_masked_dkdv_f32(
    const float* __restrict__ q, int64_t ldq, const float* __restrict__ k, int64_t ldk, const float* __restrict__ v,
    int64_t ldv, const float* __restrict__ dO, int64_t lddo, const float* __restrict__ nl2,
    const float* __restrict__ delta, float* __restrict__ dk, int64_t lddk, float* __restrict__ dv, int64_t lddv, int T,
    int group, ScoreArgs args, MaskTable mask) {
  constexpr int NU = HD / 16, TILE = 16 * (HD + 4), NW = kMaskedWavesF32<HD>;
  __shared__ __align__(16) float tiles[NW / 2 * TILE];
  const int lane = threadIdx.x & 63, r = lane & 15, c = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kvh = blockIdx.y;
  const int k0 = static_cast<int>(blockIdx.x) * 16, ki = k0 + r, kc = min(ki, T - 1);
  const int4 mine = mask.queries[k0 / kMaskRows];
  const int2 seen_by = ki < T ? *(reinterpret_cast<const int2*>(mask.rows + ki) + 1) : make_int2(0, 0);
  const bool some = seen_by.x < seen_by.y;
  FragF32<HD> kf, vf;
  load_frag_f32<HD>(kf, k + static_cast<int64_t>(kc) * ldk + static_cast<int64_t>(kvh) * HD, c);
  load_frag_f32<HD>(vf, v + static_cast<int64_t>(kc) * ldv + static_cast<int64_t>(kvh) * HD, c);
  f32x4 ak[NU], av[NU];
#pragma unroll
  for (int dt = 0; dt < NU; ++dt) ak[dt] = av[dt] = zero4();
  const int n_blocks = mine.y > mine.x ? (mine.y - mine.x + 31) / 32 : 0;  // of queries
  for (int it = wave; it < group * n_blocks; it += NW) {
    const int hh = it / n_blocks, q0 = mine.x + (it - hh * n_blocks) * 32;
    const int h = kvh * group + hh;
    const float* qp = q + static_cast<int64_t>(q0) * ldq + static_cast<int64_t>(h) * HD;
    const float* gp = dO + static_cast<int64_t>(q0) * lddo + static_cast<int64_t>(h) * HD;
    const int64_t srow = static_cast<int64_t>(h) * T + q0;
    const int last = T - 1 - q0;
    const int lo = seen_by.x - q0, hi = seen_by.y - q0;  // queries n of the block with lo <= n < hi see the key
    const ScoreF32<MODE> score(args, h);
    f32x4 x[2], y[2];  // P, dS: rows = queries, column = key
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int row = min(16 * t + r, last);
      FragF32<HD> f;
      load_frag_f32<HD>(f, qp + row * ldq, c);
      x[t] = dot_f32<HD>(f, kf);
      load_frag_f32<HD>(f, gp + row * lddo, c);
      y[t] = dot_f32<HD>(f, vf);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int n = 16 * t + 4 * c + e;
        const int64_t at = srow + min(n, last);
        const bool live = n >= lo && n < hi;
        float ds;
        const float p = fast_exp2(score(x[t][e], q0 + n - ki, ds) + nl2[at]);
        x[t][e] = live ? p : 0.f;
        y[t][e] = live ? p * (y[t][e] - delta[at]) * ds : 0.f;
      }
    }
    const bool partial = !(mine.z <= q0 && mine.w >= q0 + 32);
    wsum_f32<HD>(av, x, gp, lddo, last, partial, lo, hi, r, c);
    wsum_f32<HD>(ak, y, qp, ldq, last, partial, lo, hi, r, c);
  }
  zero_unless<NU>(av, some);
  zero_unless<NU>(ak, some);
  sum_waves_f32<HD, NW>(av, tiles, wave, r, c);
  if (wave == 0) put_tile_f32<HD>(tiles, av, r, c);
  __syncthreads();
  store_rows_f32<HD, 64 * NW>(dv + static_cast<int64_t>(kvh) * HD, lddv, tiles, k0, T, 1.f);
  __syncthreads();
  sum_waves_f32<HD, NW>(ak, tiles, wave, r, c);
  if (wave == 0) put_tile_f32<HD>(tiles, ak, r, c);
  __syncthreads();
  store_rows_f32<HD, 64 * NW>(dk + static_cast<int64_t>(kvh) * HD, lddk, tiles, k0, T, args.scale);
}

}  // namespace

void masked_fwd_f32(const MaskedFwd& c, const MaskedArgs& a, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>((a.tokens + 15) / 16), static_cast<unsigned>(a.n_heads));
  dispatch_masked(a.head_dim, a.mode, [&](auto hd, auto mode) {
    hipLaunchKernelGGL((k_masked_fwd_f32<hd(), mode()>), grid, dim3(256), 0, stream, static_cast<const float*>(c.q), c.ldq,
                       static_cast<const float*>(c.k), c.ldk, static_cast<const float*>(c.v), c.ldv,
                       static_cast<float*>(c.o), c.ldo, c.lse, static_cast<int>(a.tokens),
                       static_cast<int>(a.n_heads / a.n_kv_heads), a.score, c.table);
  });
}

void masked_bwd_f32(const MaskedBwd& c, const MaskedArgs& a, hipStream_t stream) {
  float* delta = c.workspace;
  float* nl2 = delta + a.tokens * a.n_heads;
  const int T = static_cast<int>(a.tokens), group = static_cast<int>(a.n_heads / a.n_kv_heads);
  const auto q = static_cast<const float*>(c.q), k = static_cast<const float*>(c.k);
  const auto v = static_cast<const float*>(c.v), g = static_cast<const float*>(c.dout);
  const unsigned tiles = static_cast<unsigned>((a.tokens + 15) / 16);
  dispatch_masked(a.head_dim, a.mode, [&](auto hd, auto mode) {
    constexpr int HD = decltype(hd)::value, MODE = decltype(mode)::value;
    hipLaunchKernelGGL((k_masked_dq_f32<HD, MODE>), dim3(tiles, static_cast<unsigned>(a.n_heads)), dim3(256), 0, stream, q,
                       c.ldq, k, c.ldk, v, c.ldv, static_cast<const float*>(c.o), c.ldo, g, c.lddo, c.lse, delta, nl2,
                       static_cast<float*>(c.dq), c.lddq, T, group, a.score, c.table);
    hipLaunchKernelGGL((k_masked_dkdv_f32<HD, MODE>), dim3(tiles, static_cast<unsigned>(a.n_kv_heads)),
                       dim3(64 * kMaskedWavesF32<HD>), 0, stream, q, c.ldq, k, c.ldk, v, c.ldv, g, c.lddo, nl2, delta,
                       static_cast<float*>(c.dk), c.lddk, static_cast<float*>(c.dv), c.lddv, T, group, a.score, c.table);
  });
}

}  // namespace fh
