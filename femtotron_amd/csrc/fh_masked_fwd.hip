// Attention under a mask, bf16 forward.
//
// The layout and the products are those of the causal kernel (fh_attention.hip): four
// waves of 32 queries of one head, 64 keys a step, S^T = K Q^T with one query a lane,
// an online softmax in fp32, O^T += V^T P^T.  Here the steps run over what the
// workgroup's 128 queries see, from the first of those keys on: keys that none of them
// sees are not read, a wave skips steps that its own 32 do not see, and only steps of
// which some query sees a part are masked.
#include <type_traits>

#include "fh_masked.hpp"

namespace fh {
namespace {

// Finite, so that a query without a key yet has weights 0 and not exp2(-inf + inf).
constexpr float kNoMax = -3.0e38f;

// One step of a wave: raw scores of 64 keys from K, the update of (m, l, oacc), and
// oacc += V^T P^T.  base = the query's row - k0 - 4 hl; it sees keys lo <= c < hi of the
// step (less 4 hl).  ends, starts: some query sees no key from within the step on, before
// a key within it.
template <int HD, int MODE, bool CAREFUL>
__device__ __forceinline__ void masked_step(const char* K, const char* V, const bf16x8 (&qf)[HD / 16],
                                            f32x16 (&oacc)[HD / 32], float& m, float& l, int a_off, int b0, int b8,
                                            const Score<MODE>& score, float base, bool ends, bool starts, int lo,
                                            int hi, int hl) {
  constexpr int BN = 64, NS = HD / 16, ND = HD / 32;
  f32x16 x[BN / 32];
  __builtin_amdgcn_iglp_opt(0);  // LDS reads interleaved with MFMAs
#pragma unroll
  for (int t = 0; t < BN / 32; ++t) {
    x[t] = zero16();
#pragma unroll
    for (int s = 0; s < NS; ++s) x[t] = mfma(lds_frag<HD>(K, a_off, 32 * t, s), qf[s], x[t]);
  }
  // What x holds now: raw products, under a cap alone r (which falls as the score rises), and
  // with a bias the scores.
  if constexpr (MODE != 0) {
#pragma unroll
    for (int t = 0; t < BN / 32; ++t)
#pragma unroll
      for (int j = 0; j < 16; ++j)
        x[t][j] = MODE == kCap ? score.half_sigmoid(x[t][j]) : score(x[t][j], base - (32 * t + acc_row(j, 0)));
  }
  constexpr float kNone = MODE == kCap ? INFINITY : -INFINITY;
  mask_range(x[0], ends, starts, lo, hi, 0, kNone);
  mask_range(x[1], ends, starts, lo, hi, 32, kNone);
  float mloc = kNone;
#pragma unroll
  for (int t = 0; t < BN / 32; ++t)
#pragma unroll
    for (int j = 0; j < 16; ++j) mloc = MODE == kCap ? fminf(mloc, x[t][j]) : fmaxf(mloc, x[t][j]);
  if constexpr (MODE == kCap) mloc = fmaf(score.c, mloc, score.b);
  mloc = xor32_max(mloc);
  if constexpr (MODE == 0) mloc *= score.a;
  if (wave_any(mloc > m + kRescaleSlack)) {
    const float mnew = fmaxf(m, mloc);
    const float alpha = fast_exp2(m - mnew);
    m = mnew;
    l *= alpha;
#pragma unroll
    for (int dt = 0; dt < ND; ++dt)
#pragma unroll
      for (int j = 0; j < 16; ++j) oacc[dt][j] *= alpha;
  }
  const float nm = MODE == kCap ? score.b - m : -m;
#pragma unroll
  for (int t = 0; t < BN / 32; ++t)
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      if constexpr (MODE == 0) x[t][j] = fast_exp2(fmaf(x[t][j], score.a, nm));
      else if constexpr (MODE == kCap) x[t][j] = fast_exp2(fmaf(score.c, x[t][j], nm));
      else x[t][j] = fast_exp2(x[t][j] + nm);
    }
  // The row sums add the bf16 weights that P V multiplies, so that the normalisation
  // matches the weights used.
  float lsum = 0.f;
#pragma unroll
  for (int s = 0; s < BN / 16; ++s) {
    const bf16x8 pf = pack_frag(x[s >> 1], 8 * (s & 1));
    lsum = sum_bf16x8(pf, lsum);
    if constexpr (CAREFUL) {
      if (ends || starts) {
        wsum_careful<HD>(oacc, pf, V, b0, b8, 16 * s, lo + 4 * hl, hi + 4 * hl, hl);
        continue;
      }
    }
    wsum<HD>(oacc, pf, V, b0, b8, 16 * s);
  }
  l += lsum;
}

// Four waves a SIMD up to head_dim 64: what the registers (128) then lack, at 64 with a pair of
// heads 68 bytes a lane (204 under a cap), is spilled in the careful pass and in the addresses
// of tiles that end past the last row.  16384 tokens, 32/4 heads of 64, documents of about 600: 105 us with
// three waves a SIMD (one workgroup a CU), 83 with four (390 TFLOP/s; the matrix units are
// busy 17% of it and the vector units 45%).  8192 tokens, 32/8 heads of 128, capped: 657 us,
// 840 TFLOP/s; without the cap 542.
// HPB = 2: 8 waves take the same rows of two query heads of one kv head, which read the
// same K and V tiles.
template <int HD, int HPB, int MODE>
__global__ __launch_bounds__(256 * HPB) __attribute__((amdgpu_waves_per_eu(HD == 128 ? 2 : HPB == 2 ? 4 : 3))) void k_masked_fwd(
    const uint16_t* __restrict__ q, int64_t ldq, const uint16_t* __restrict__ k, int64_t ldk,
    const uint16_t* __restrict__ v, int64_t ldv, uint16_t* __restrict__ o, int64_t ldo, float* __restrict__ lse,
    int8_t* __restrict__ o_low, int T, int group, ScoreArgs args, MaskTable mask) {
  constexpr int BM = 128, BN = 64, NS = HD / 16, ND = HD / 32, TILE = BN * 2 * HD;
  // Three K/V stages up to head_dim 64 (48 KB); at 128 they would leave room for one
  // workgroup a CU.
  constexpr int STAGES = HD <= 64 ? 3 : 2, TILE3 = STAGES == 3 ? TILE : 16;
  __shared__ __align__(16) char sk0[TILE], sk1[TILE], sk2[TILE3], sv0[TILE], sv1[TILE], sv2[TILE3];
  const int tid = threadIdx.x, lane = tid & 63, hl = lane >> 5, l32 = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const XcdOrder ord = masked_order();
  const int h = ord.y * HPB + (wave >> 2), kvh = h / group;
  // The blocks that see most first, or else the latest.
  const int q0 = (mask.order_q != nullptr ? mask.order_q[ord.rank] : static_cast<int>(gridDim.x) - 1 - ord.rank) * BM;
  const int qw = q0 + (wave & 3) * 32, qi = qw + l32;
  const int tiles = (T + kMaskRows - 1) / kMaskRows;
  const int4 all = mask_bounds<BM / kMaskRows>(mask.keys, q0 / kMaskRows, tiles);
  const int4 mine = mask_bounds<1>(mask.keys, qw / kMaskRows, tiles);
  const int2 sees = qi < T ? *reinterpret_cast<const int2*>(mask.rows + qi) : make_int2(0, 0);
  const int kbeg = all.x, n_steps = all.y > all.x ? (all.y - all.x + BN - 1) / BN : 0;
  const Score<MODE> score(args, h);
  int a_off = lane_off_a<HD>(lane);
  int b0 = lane_off_b<HD>(lane, 0), b8 = lane_off_b<HD>(lane, 8);

  bf16x8 qf[NS];
  auto load_q = [&]() __attribute__((always_inline)) {
    const uint16_t* qrow = q + static_cast<int64_t>(qi) * ldq + static_cast<int64_t>(h) * HD + 8 * hl;
#pragma unroll
    for (int s = 0; s < NS; ++s) qf[s] = qi < T ? ld_frag(qrow + 16 * s) : as_bf16x8(make_uint4(0, 0, 0, 0));
  };
  f32x16 oacc[ND];
  float m, l;
  const bool some = sees.x < sees.y;
  if (n_steps > 0) {  // uniform
    const uint16_t* kp = k + static_cast<int64_t>(kbeg) * ldk + static_cast<int64_t>(kvh) * HD;
    const uint16_t* vp = v + static_cast<int64_t>(kbeg) * ldv + static_cast<int64_t>(kvh) * HD;
    auto run = [&](auto careful) __attribute__((always_inline)) {
      m = kNoMax;
      l = 0.f;
#pragma unroll
      for (int dt = 0; dt < ND; ++dt) oacc[dt] = zero16();
      auto body = [&](int kb, const char* K, const char* V) __attribute__((always_inline)) {
        refresh_offsets(a_off, b0, b8);
        const int k0 = kbeg + kb * BN;
        if (mine.x >= k0 + BN || mine.y <= k0) return;  // nothing for this wave's queries
        masked_step<HD, MODE, decltype(careful)::value>(K, V, qf, oacc, m, l, a_off, b0, b8, score,
                                                        static_cast<float>(qi - k0 - 4 * hl),
                                                        mine.w < k0 + BN, mine.z > k0, sees.x - k0 - 4 * hl,
                                                        sees.y - k0 - 4 * hl, hl);
      };
      if constexpr (STAGES == 3)
        kv_block_loop3<BN, HD, 4 * HPB>(kp, ldk, vp, ldv, n_steps, T - kbeg, sk0, sk1, sk2, sv0, sv1, sv2, wave, lane,
                                        body, load_q);
      else
        kv_block_loop<BN, HD, true, 4 * HPB>(kp, ldk, vp, ldv, n_steps, T - kbeg, sk0, sk1, sv0, sv1, wave, lane, body,
                                             load_q);
    };
    run(std::false_type{});
    if (__builtin_expect(__syncthreads_or(some && not_finite<ND>(oacc)), 0)) run(std::true_type{});
  }
  if (qi < T) {
    const float lt = n_steps > 0 ? xor32_sum(l) : 0.f;
    if (!some) {
#pragma unroll
      for (int dt = 0; dt < ND; ++dt) oacc[dt] = zero16();
    }
    const float mul = some ? 1.f / lt : 0.f;
    uint16_t* row = o + static_cast<int64_t>(qi) * ldo + static_cast<int64_t>(h) * HD + 8 * hl;
    int8_t* low = o_low + static_cast<int64_t>(qi) * (gridDim.y * HPB * HD) + static_cast<int64_t>(h) * HD + 8 * hl;
    // Lane half hl holds dims 8 g + 4 hl .. +3; the halves exchange so that each stores the 8
    // dims of the groups g with g % 2 == hl.
#pragma unroll
    for (int dt = 0; dt < ND; ++dt)
#pragma unroll
      for (int g = 0; g < 4; g += 2) {
        uint2 w[2];
        uint32_t b[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int j = 4 * (g + i);
          const float x[4] = {oacc[dt][j] * mul, oacc[dt][j + 1] * mul, oacc[dt][j + 2] * mul, oacc[dt][j + 3] * mul};
          w[i] = make_uint2(pk_bf16(x[0], x[1]), pk_bf16(x[2], x[3]));
          b[i] = low_bits(x, w[i]);
        }
        const auto x = __builtin_amdgcn_permlane32_swap(w[0].x, w[1].x, false, false);
        const auto y = __builtin_amdgcn_permlane32_swap(w[0].y, w[1].y, false, false);
        *reinterpret_cast<uint4*>(row + dt * 32 + 8 * g) = make_uint4(x[0], y[0], x[1], y[1]);
        if (o_low != nullptr) {
          const auto z = __builtin_amdgcn_permlane32_swap(b[0], b[1], false, false);
          *reinterpret_cast<uint2*>(low + dt * 32 + 8 * g) = make_uint2(z[0], z[1]);
        }
      }
    if (lse != nullptr && hl == 0) lse[static_cast<int64_t>(h) * T + qi] = some ? (m + log2f(lt)) * kLn2 : 0.f;
  }
}

}  // namespace

void masked_fwd_bf16(const MaskedFwd& c, const MaskedArgs& a, hipStream_t stream) {
  const int group = static_cast<int>(a.n_heads / a.n_kv_heads);
  const int64_t blocks = (a.tokens + 127) / 128;
  // Pairs of heads where they leave a workgroup for every CU: 8192 tokens, 32/8 heads of 128, 565
  // -> 542 us, 16384 tokens of 32/4 heads of 64 183 -> 171; but 999 tokens of those 16 -> 18 (capped 22).
  const bool pair = group % 2 == 0 && (a.n_heads / 2) % 8 == 0 && blocks * (a.n_heads / 2) >= 256;
  const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(a.n_heads / (pair ? 2 : 1)));
  dispatch_masked(a.head_dim, a.mode, [&](auto hd, auto mode) {
    auto launch = [&](auto hpb) {
      hipLaunchKernelGGL((k_masked_fwd<hd(), hpb(), mode()>), grid, dim3(256 * hpb()), 0, stream,
                         static_cast<const uint16_t*>(c.q), c.ldq, static_cast<const uint16_t*>(c.k), c.ldk,
                         static_cast<const uint16_t*>(c.v), c.ldv, static_cast<uint16_t*>(c.o), c.ldo, c.lse, c.o_low,
                         static_cast<int>(a.tokens), group, a.score, c.table);
    };
    if (pair) launch(std::integral_constant<int, 2>{});
    else launch(std::integral_constant<int, 1>{});
  });
}

}  // namespace fh
