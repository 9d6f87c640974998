// Attention under a mask, bf16 backward:
//   P = exp(Z - lse), dP = dO V^T, dZ = P (dP - delta), dS = dZ dz/ds,
//   dQ = scale dS K, dK = scale dS^T Q, dV = P^T dO,   delta = rowsum(dO O).
// The layout and the products are those of the causal kernels (fh_attention.hip): dQ
// over the keys that a workgroup's 128 queries see, dK and dV over the queries that see
// its keys (128 up to head_dim 64, 64 at 128) and the query heads of their kv head, so
// that each sum is complete inside one workgroup, without atomics.  Steps of which a
// wave's rows see nothing are skipped, and only steps seen in part are masked.
#include <type_traits>

#include "fh_masked.hpp"

namespace fh {
namespace {

// ------------------------------------------------------------------------- dQ
// One step of 64 keys of a wave (see masked_step).  dS enters its product in two bf16 parts,
// the value and what rounding it left, on the same fragments of K; `sum` adds up dZ, which is
// 0 over a row whose delta is exact.  delta comes from o, whose weights the forward rounded:
// in rows that look at few tokens that error is as large as the roundings of dS and of dQ
// together, 1.5 to 1.9 times what rounding dQ alone leaves; with the second part 1.05 to
// 1.15 (8192 tokens, 32/8 heads of 128, capped: 2451 -> 2655 us for the backward; 16384
// tokens, 32/4 heads of 64, documents of about 600, 305 -> 311).
template <int HD, int MODE, bool CAREFUL>
__device__ __forceinline__ void masked_dq_step(const char* K, const char* V, const bf16x8 (&qf)[HD / 16],
                                               const bf16x8 (&gf)[HD / 16], f32x16 (&dqacc)[HD / 32], float& sum,
                                               float nlse2, float dl, int a_off, int b0, int b8, const Score<MODE>& score,
                                               float base, bool ends, bool starts, int lo, int hi, int hl) {
  constexpr int BN = 64, NS = HD / 16;
#pragma unroll
  for (int t = 0; t < BN / 32; ++t) {
    f32x16 x = zero16(), y = zero16();  // S^T, dP^T
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      x = mfma(lds_frag<HD>(K, a_off, 32 * t, s), qf[s], x);
      y = mfma(lds_frag<HD>(V, a_off, 32 * t, s), gf[s], y);
    }
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      float ds;
      const float p = score.weight(x[j], base - (32 * t + acc_row(j, 0)), nlse2, ds);
      x[j] = p * (y[j] - dl);
      y[j] = ds;
    }
    mask_range(x, ends, starts, lo, hi, 32 * t, 0.f);
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      sum += x[j];
      if constexpr (MODE & kCap) x[j] *= y[j];
    }
#pragma unroll
    for (int s2 = 0; s2 < 2; ++s2) {
      const bf16x8 df = pack_frag(x, 8 * s2);
      const int row0 = 32 * t + 16 * s2;
      if constexpr (CAREFUL) {
        if (ends || starts) {
          wsum_careful<HD>(dqacc, df, K, b0, b8, row0, lo + 4 * hl, hi + 4 * hl, hl);
          continue;
        }
      }
      const bf16x8 dr = rest_frag(x, 8 * s2);
#pragma unroll
      for (int dt = 0; dt < HD / 32; ++dt) {
        const bf16x8 k = lds_frag_tr<HD>(K, b0, b8, row0, dt);
        dqacc[dt] = mfma(k, df, dqacc[dt]);
        dqacc[dt] = mfma(k, dr, dqacc[dt]);
      }
    }
  }
}

// Also writes -lse * log2(e) (plus cap_log2: see Score) and delta, put right by the sum of dZ,
// which the dK/dV kernels read.  142-147 us at 16384 tokens, 32/4 heads of 64, documents of
// about 600; 1100-1140 at 8192 tokens, 32/8 heads of 128, capped: bound by the vector work of
// scores and dS and, at 128, by two waves a SIMD that cover each other's waits in part.  (The
// scratch of the compiled kernels, 964 to 1540 bytes a lane at 128 and 276 or 616 at 64 under
// a cap, belongs to the careful pass, at 64 also to the addresses of tiles that end past the
// last row.)
template <int HD, int MODE>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(HD <= 64 ? 3 : 2))) void k_masked_dq(
    const uint16_t* __restrict__ q, int64_t ldq, const uint16_t* __restrict__ k, int64_t ldk,
    const uint16_t* __restrict__ v, int64_t ldv, const uint16_t* __restrict__ o, int64_t ldo,
    const uint16_t* __restrict__ dO, int64_t lddo, const float* __restrict__ lse,
    const int8_t* __restrict__ o_low, float* __restrict__ delta, float* __restrict__ nl2, uint16_t* __restrict__ dq, int64_t lddq, int T, int group, ScoreArgs args,
    MaskTable mask) {
  constexpr int BM = 128, BN = 64, NS = HD / 16, ND = HD / 32, TILE = BN * 2 * HD;
  __shared__ __align__(16) char sk0[TILE], sk1[TILE], sv0[TILE], sv1[TILE];
  const int tid = threadIdx.x, lane = tid & 63, hl = lane >> 5, l32 = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const XcdOrder ord = masked_order();
  const int h = ord.y, kvh = h / group;
  const int q0 = (mask.order_q != nullptr ? mask.order_q[ord.rank] : static_cast<int>(gridDim.x) - 1 - ord.rank) * BM;
  const int qw = q0 + wave * 32, qi = qw + l32;
  const int tiles = (T + kMaskRows - 1) / kMaskRows;
  const int4 all = mask_bounds<BM / kMaskRows>(mask.keys, q0 / kMaskRows, tiles);
  const int4 mine = mask_bounds<1>(mask.keys, qw / kMaskRows, tiles);
  const int2 sees = qi < T ? *reinterpret_cast<const int2*>(mask.rows + qi) : make_int2(0, 0);
  const int kbeg = all.x, n_steps = all.y > all.x ? (all.y - all.x + BN - 1) / BN : 0;
  const Score<MODE> score(args, h);
  int a_off = lane_off_a<HD>(lane);
  int b0 = lane_off_b<HD>(lane, 0), b8 = lane_off_b<HD>(lane, 8);

  bf16x8 qf[NS], gf[NS];
  float nlse2 = 0.f, dl = 0.f;
  {
    const int64_t col = static_cast<int64_t>(h) * HD + 8 * hl;
    const uint16_t* qrow = q + static_cast<int64_t>(qi) * ldq + col;
    const uint16_t* grow = dO + static_cast<int64_t>(qi) * lddo + col;
    const uint16_t* orow = o + static_cast<int64_t>(qi) * ldo + col;
    const int8_t* lrow = o_low + static_cast<int64_t>(qi) * (gridDim.y * HD) + col;
    float part = 0.f;
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      uint4 gz = make_uint4(0, 0, 0, 0), oz = make_uint4(0, 0, 0, 0);
      uint2 lz = make_uint2(0, 0);
      qf[s] = as_bf16x8(gz);
      if (qi < T) {
        qf[s] = ld_frag(qrow + 16 * s);
        gz = *reinterpret_cast<const uint4*>(grow + 16 * s);
        oz = *reinterpret_cast<const uint4*>(orow + 16 * s);
        lz = *reinterpret_cast<const uint2*>(lrow + 16 * s);
      }
      gf[s] = as_bf16x8(gz);
      float gv[8];
      Elem<uint16_t>::unpack(gz, gv);
      const uint32_t ow[4] = {oz.x, oz.y, oz.z, oz.w};
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t high = (e & 1) ? ow[e >> 1] & 0xffff0000u : ow[e >> 1] << 16;
        part = fmaf(gv[e], with_low(high, e < 4 ? lz.x : lz.y, e & 3), part);
      }
    }
    dl = xor32_sum(part);
    if (qi < T) {
      const int64_t at = static_cast<int64_t>(h) * T + qi;
      nlse2 = fmaf(-kLog2e, lse[at], score.b);
      if (hl == 0) nl2[at] = nlse2;
    }
  }
  f32x16 dqacc[ND];
  float sum = 0.f;  // of dZ over the lane's keys
  const bool some = sees.x < sees.y;
  if (n_steps > 0) {  // uniform
    const uint16_t* kp = k + static_cast<int64_t>(kbeg) * ldk + static_cast<int64_t>(kvh) * HD;
    const uint16_t* vp = v + static_cast<int64_t>(kbeg) * ldv + static_cast<int64_t>(kvh) * HD;
    auto run = [&](auto careful) __attribute__((always_inline)) {
#pragma unroll
      for (int dt = 0; dt < ND; ++dt) dqacc[dt] = zero16();
      sum = 0.f;
      kv_block_loop<BN, HD, false, 4>(
          kp, ldk, vp, ldv, n_steps, T - kbeg, sk0, sk1, sv0, sv1, wave, lane,
          [&](int kb, const char* K, const char* V) __attribute__((always_inline)) {
            refresh_offsets(a_off, b0, b8);
            const int k0 = kbeg + kb * BN;
            if (mine.x >= k0 + BN || mine.y <= k0) return;
            masked_dq_step<HD, MODE, decltype(careful)::value>(
                K, V, qf, gf, dqacc, sum, nlse2, dl, a_off, b0, b8, score, static_cast<float>(qi - k0 - 4 * hl),
                mine.w < k0 + BN, mine.z > k0, sees.x - k0 - 4 * hl, sees.y - k0 - 4 * hl, hl);
          },
          [] {});
    };
    run(std::false_type{});
    if (__builtin_expect(__syncthreads_or(some && not_finite<ND>(dqacc)), 0)) run(std::true_type{});
  }
  if (qi < T) {
    const float off = xor32_sum(sum);
    if (hl == 0) delta[static_cast<int64_t>(h) * T + qi] = dl + (some ? off : 0.f);
    if (!some) {
#pragma unroll
      for (int dt = 0; dt < ND; ++dt) dqacc[dt] = zero16();
    }
    store_rows_T<HD>(dq + static_cast<int64_t>(qi) * lddq + static_cast<int64_t>(h) * HD, dqacc, grad_scale<MODE>(args), hl);
  }
}

// ---------------------------------------------------------------------- dK, dV
// The (query tile, query head) items of a workgroup's loop, from the last tile that sees
// its keys to the first, over the group's query heads within a tile, and the loads of
// their Q, dO, -lse * log2(e) and delta straight into an LDS stage (the last wave loads
// 64 rows of the two).  q, dO, nl2 and delta point at row qbeg of the group's first query
// head; rows past T - 1 read that row again, masked.
template <int HD, int BQ, int NT>
struct MaskedItems {
  int qt, hh = 0;  // the item to load next
  TileDma<BQ, HD, NT / 64> tq, tg;
  __device__ __forceinline__ void start(int n_tiles, int64_t ldq, int64_t lddo, int wave, int lane) {
    qt = n_tiles - 1;
    hh = 0;
    tq.init(ldq, wave, lane);
    tg.init(lddo, wave, lane);
  }
  __device__ __forceinline__ void load(const uint16_t* q, int64_t ldq, const uint16_t* dO, int64_t lddo,
                                       const float* nl2, const float* delta, int T, int last, int heads, char* sq,
                                       char* sg, float* sl, float* sd, int wave, int lane) {
    typedef __attribute__((address_space(1))) const void* gptr;
    typedef __attribute__((address_space(3))) void* lptr;
    static_assert(BQ <= 64, "one load covers the tile's rows");
    const int qs = max(qt, 0) * BQ;
    const int64_t col = static_cast<int64_t>(hh) * HD;
    tq.load(q + col, ldq, qs, last, sq, wave, lane);
    tg.load(dO + col, lddo, qs, last, sg, wave, lane);
    if (wave == NT / 64 - 1) {
      const int64_t row = static_cast<int64_t>(hh) * T + min(qs + lane, last);
      __builtin_amdgcn_global_load_lds((gptr)(nl2 + row), (lptr)sl, 4, 0, 0);
      __builtin_amdgcn_global_load_lds((gptr)(delta + row), (lptr)sd, 4, 0, 0);
    }
    if (++hh == heads) {
      hh = 0;
      --qt;
    }
  }
};

// A wave's share of an item up to head_dim 64: the 32 queries at row hrow of the tiles Q
// and dO against the wave's 32 keys.  base = the item's first query + 4 hl - the lane's
// key; the lane's key is seen by the queries lo <= c < hi of the 32 (less 4 hl); ends and
// starts as in masked_step, of keys.
template <int HD, int MODE, bool CAREFUL>
__device__ __forceinline__ void masked_dkdv_item(const char* Q, const char* G, const float* sl, const float* sd,
                                                 const bf16x8 (&kf)[HD / 16], const bf16x8 (&vf)[HD / 16],
                                                 f32x16 (&dkacc)[HD / 32], f32x16 (&dvacc)[HD / 32], int a_off, int b0,
                                                 int b8, int hrow, const Score<MODE>& score, float base, bool ends,
                                                 bool starts, int lo, int hi, int hl) {
  constexpr int NS = HD / 16;
  f32x16 x = zero16(), y = zero16();  // S, dP (rows = queries, column = key)
  __builtin_amdgcn_iglp_opt(0);
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    x = mfma(lds_frag<HD>(Q, a_off, 0, s), kf[s], x);
    y = mfma(lds_frag<HD>(G, a_off, 0, s), vf[s], y);
  }
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const float4 L4 = *reinterpret_cast<const float4*>(&sl[hrow + 8 * g + 4 * hl]);
    const float4 D4 = *reinterpret_cast<const float4*>(&sd[hrow + 8 * g + 4 * hl]);
    const float Lv[4] = {L4.x, L4.y, L4.z, L4.w};
    const float Dv[4] = {D4.x, D4.y, D4.z, D4.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int j = 4 * g + e;
      float ds;
      const float p = score.weight(x[j], base + acc_row(j, 0), Lv[e], ds);
      const float dz = p * (y[j] - Dv[e]);
      x[j] = p;
      y[j] = (MODE & kCap) ? dz * ds : dz;
    }
  }
  mask_range(x, ends, starts, lo, hi, 0, 0.f);
  mask_range(y, ends, starts, lo, hi, 0, 0.f);
#pragma unroll
  for (int s2 = 0; s2 < 2; ++s2) {
    const bf16x8 pf = pack_frag(x, 8 * s2);
    const bf16x8 df = pack_frag(y, 8 * s2);
    if constexpr (CAREFUL) {
      if (ends || starts) {
        wsum_careful<HD>(dvacc, pf, G, b0, b8, 16 * s2, lo + 4 * hl, hi + 4 * hl, hl);
        wsum_careful<HD>(dkacc, df, Q, b0, b8, 16 * s2, lo + 4 * hl, hi + 4 * hl, hl);
        continue;
      }
    }
#pragma unroll
    for (int dt = 0; dt < HD / 32; ++dt) {
      dvacc[dt] = mfma(lds_frag_tr<HD>(G, b0, b8, 16 * s2, dt), pf, dvacc[dt]);
      dkacc[dt] = mfma(lds_frag_tr<HD>(Q, b0, b8, 16 * s2, dt), df, dkacc[dt]);
    }
  }
}

// Workgroups that a kv head's query heads are split over: `split`, or hs.n where the block
// that is seen by most is seen by about kLongRows rows or more (in the order's buckets, so that it
// does not hang on which of a bucket comes first).  The workgroups of long rows are few and of
// unlike length, and the last of them leave a CU to themselves; the sums of the parts cost the same
// in short ones, where nothing is gained.  The backward with twice the parts, 8192 tokens, 32/8
// heads of 128: one document 2303 -> 2155 us, documents of 600 283 -> 316; with up to four times
// the parts, 32/4 heads of 64: one document 1835 -> 1226 (4096 tokens 490 -> 365).
constexpr int kLongRows = 4096;
constexpr int kFusedKeys = 128, kSplitKeys = 64;  // of a workgroup, up to head_dim 64 and at 128
template <int HD>
__device__ __forceinline__ int dkdv_split(const MaskTable& mask, int T, const HeadSplit& hs, int split) {
  const int* order = HD <= 64 ? mask.order_k128 : mask.order_k64;
  if (split == hs.n || order == nullptr) return split;
  constexpr int TILES = (HD <= 64 ? kFusedKeys : kSplitKeys) / kMaskRows;
  const int4 most = mask_bounds<TILES>(mask.queries, order[0] * TILES, (T + kMaskRows - 1) / kMaskRows);
  const int unit = order_unit(T);
  return most.y > most.x && (most.y - most.x + unit - 1) / unit * unit >= kLongRows ? hs.n : split;
}

template <int HD>
__global__ __launch_bounds__(256) void k_masked_dkdv_sum(HeadSplit hs, int split, MaskTable mask, uint16_t* __restrict__ dk,
                                                         int64_t lddk, uint16_t* __restrict__ dv, int64_t lddv, int T,
                                                         int nkv, float scale) {
  hs.n = dkdv_split<HD>(mask, T, hs, split);
  if (hs.n > 1) attn_dkdv_sum<HD>(hs, dk, lddk, dv, lddv, T, T, nkv, scale, RopeRows<uint16_t>{nullptr, nullptr, 0});
}

// Up to head_dim 64: 8 waves, 128 keys; wave w holds K and V of keys 32 (w % 4) .. +31 in
// registers and takes queries 32 (w / 4) .. +31 of each 64-query item; the halves' sums
// meet in LDS at the end, in a fixed order.  Two items a stage, two stages.  190-199 us at
// 16384 tokens, 32/4 heads of 64, documents of about 600: 133 KB of LDS let one workgroup onto
// a CU, 1.6 waves a SIMD on average, and the matrix units are busy 16% of it, the vector units
// 25%: it waits.
template <int HD, int MODE>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2))) void k_masked_dkdv_fused(
    const uint16_t* __restrict__ q, int64_t ldq, const uint16_t* __restrict__ k, int64_t ldk,
    const uint16_t* __restrict__ v, int64_t ldv, const uint16_t* __restrict__ dO, int64_t lddo,
    const float* __restrict__ nl2, const float* __restrict__ delta, uint16_t* __restrict__ dk, int64_t lddk,
    uint16_t* __restrict__ dv, int64_t lddv, int T, int nkv, int group, ScoreArgs args, MaskTable mask, HeadSplit hs,
    int n_split) {
  constexpr int NWH = 4, NT = 512, BQ = 64, NS = HD / 16, ND = HD / 32, TILE = BQ * 2 * HD;
  // The tiles first, below 64 KB: their bases are the reads' immediate offsets.
  struct Lds {
    char sq0a[TILE], sq0b[TILE], sq1a[TILE], sq1b[TILE];
    char sg0a[TILE], sg0b[TILE], sg1a[TILE], sg1b[TILE];
    float sl0a[BQ], sl0b[BQ], sl1a[BQ], sl1b[BQ];  // -lse*log2(e)
    float sd0a[BQ], sd0b[BQ], sd1a[BQ], sd1b[BQ];  // delta
    float xchg[2][NWH][ND * 16][64];               // [0]: dV of half 0, [1]: dK of half 1
  };
  __shared__ __align__(16) Lds lds;
  const int tid = threadIdx.x, lane = tid & 63, hl = lane >> 5, l32 = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int half = wave / NWH, wq = wave % NWH;
  const int parts = dkdv_split<HD>(mask, T, hs, n_split);
  const XcdOrder ord = masked_order(nkv * parts);
  if (ord.y == nkv * parts) return;  // (as below)
  const int kvh = ord.y / parts, split = ord.y - kvh * parts;
  const int gs = group / parts;  // query heads of this workgroup
  const int h0 = kvh * group + split * gs;
  const int k0 = (mask.order_k128 != nullptr ? mask.order_k128[ord.rank] : ord.rank) * kFusedKeys, kw = k0 + wq * 32, ki = kw + l32;
  const int tiles = (T + kMaskRows - 1) / kMaskRows;
  const int4 all = mask_bounds<kFusedKeys / kMaskRows>(mask.queries, k0 / kMaskRows, tiles);
  const int4 mine = mask_bounds<1>(mask.queries, kw / kMaskRows, tiles);
  const int2 seen_by = ki < T ? *(reinterpret_cast<const int2*>(mask.rows + ki) + 1) : make_int2(0, 0);
  const int qbeg = all.x, n_tiles = all.y > all.x ? (all.y - all.x + BQ - 1) / BQ : 0;
  const int hrow = 32 * half;  // this wave's first query row within an item
  int a_off = lane_off_a<HD>(lane) + hrow * 2 * HD;
  int b0 = lane_off_b<HD>(lane, 0) + hrow * 2 * HD, b8 = lane_off_b<HD>(lane, 8) + hrow * 2 * HD;
  f32x16 dkacc[ND], dvacc[ND];
#pragma unroll
  for (int dt = 0; dt < ND; ++dt) {
    dkacc[dt] = zero16();
    dvacc[dt] = zero16();
  }
  const bool some = seen_by.x < seen_by.y;
  if (n_tiles > 0) {  // uniform
    bf16x8 kf[NS], vf[NS];
    {
      const bool ok = ki < T;
      const uint16_t* krow = k + static_cast<int64_t>(ki) * ldk + static_cast<int64_t>(kvh) * HD + 8 * hl;
      const uint16_t* vrow = v + static_cast<int64_t>(ki) * ldv + static_cast<int64_t>(kvh) * HD + 8 * hl;
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        kf[s] = ok ? ld_frag(krow + 16 * s) : as_bf16x8(make_uint4(0, 0, 0, 0));
        vf[s] = ok ? ld_frag(vrow + 16 * s) : as_bf16x8(make_uint4(0, 0, 0, 0));
      }
    }
    const uint16_t* qg = q + static_cast<int64_t>(qbeg) * ldq + static_cast<int64_t>(h0) * HD;
    const uint16_t* gg = dO + static_cast<int64_t>(qbeg) * lddo + static_cast<int64_t>(h0) * HD;
    const float* lg = nl2 + static_cast<int64_t>(h0) * T + qbeg;
    const float* dg = delta + static_cast<int64_t>(h0) * T + qbeg;
    const int n_it = gs * n_tiles, last = T - 1 - qbeg;
    auto run = [&](auto careful) __attribute__((always_inline)) {
      constexpr bool CAREFUL = decltype(careful)::value;
      MaskedItems<HD, BQ, NT> items;
      items.start(n_tiles, ldq, lddo, wave, lane);
      auto load = [&](char* sq, char* sg, float* sl, float* sd) __attribute__((always_inline)) {
        items.load(qg, ldq, gg, lddo, lg, dg, T, last, gs, sq, sg, sl, sd, wave, lane);
      };
      load(lds.sq0a, lds.sg0a, lds.sl0a, lds.sd0a);
      if (n_it > 1) load(lds.sq0b, lds.sg0b, lds.sl0b, lds.sd0b);
      wait_loads();
      __syncthreads();
      int qt = n_tiles - 1, hh = 0;  // the current item
      // Item `it` from the stage (Q, G, L, D), item it + 2 into (QN, GN, LN, DN).
      auto item = [&](int it, const char* Q, const char* G, const float* L, const float* D, char* QN, char* GN,
                      float* LN, float* DN) __attribute__((always_inline)) {
        refresh_offsets(a_off, b0, b8);
        if (it + 2 < n_it) load(QN, GN, LN, DN);
        const int qh = qbeg + qt * BQ + hrow;
        if (it < n_it && mine.x < qh + 32 && mine.y > qh) {
          const Score<MODE> score(args, h0 + hh);
          masked_dkdv_item<HD, MODE, CAREFUL>(Q, G, L, D, kf, vf, dkacc, dvacc, a_off, b0, b8, hrow, score,
                                              static_cast<float>(qh + 4 * hl - ki), mine.w < qh + 32, mine.z > qh,
                                              seen_by.x - qh - 4 * hl, seen_by.y - qh - 4 * hl, hl);
        }
        if (++hh == gs) {
          hh = 0;
          --qt;
        }
      };
      for (int it = 0; it < n_it; it += 4) {
        item(it, lds.sq0a, lds.sg0a, lds.sl0a, lds.sd0a, lds.sq1a, lds.sg1a, lds.sl1a, lds.sd1a);
        item(it + 1, lds.sq0b, lds.sg0b, lds.sl0b, lds.sd0b, lds.sq1b, lds.sg1b, lds.sl1b, lds.sd1b);
        wait_loads();
        __syncthreads();
        item(it + 2, lds.sq1a, lds.sg1a, lds.sl1a, lds.sd1a, lds.sq0a, lds.sg0a, lds.sl0a, lds.sd0a);
        item(it + 3, lds.sq1b, lds.sg1b, lds.sl1b, lds.sd1b, lds.sq0b, lds.sg0b, lds.sl0b, lds.sd0b);
        wait_loads();
        __syncthreads();
      }
    };
    run(std::false_type{});
    if (__builtin_expect(__syncthreads_or(some && (not_finite<ND>(dkacc) || not_finite<ND>(dvacc))), 0)) {
#pragma unroll
      for (int dt = 0; dt < ND; ++dt) {
        dkacc[dt] = zero16();
        dvacc[dt] = zero16();
      }
      run(std::true_type{});
    }
  }
  // The halves meet: half 0 hands over its dV, half 1 its dK.
  float(*out)[64] = lds.xchg[half][wq];
#pragma unroll
  for (int dt = 0; dt < ND; ++dt)
#pragma unroll
    for (int j = 0; j < 16; ++j) out[dt * 16 + j][lane] = half == 0 ? dvacc[dt][j] : dkacc[dt][j];
  __syncthreads();
  const float(*other)[64] = lds.xchg[half ^ 1][wq];
  f32x16 sum[ND];
#pragma unroll
  for (int dt = 0; dt < ND; ++dt)
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const float b = other[dt * 16 + j][lane];
      sum[dt][j] = !some ? 0.f : half == 0 ? dkacc[dt][j] + b : b + dvacc[dt][j];
    }
  if (ki < T) {
    if (parts > 1) {
      store_rows_T_f32<HD>(hs.row(split, half, T, ki, nkv, kvh, HD), sum, hl);
    } else {
      uint16_t* row = half == 0 ? dk + static_cast<int64_t>(ki) * lddk : dv + static_cast<int64_t>(ki) * lddv;
      store_rows_T<HD>(row + static_cast<int64_t>(kvh) * HD, sum, half == 0 ? grad_scale<MODE>(args) : 1.f, hl);
    }
  }
}

// head_dim 128: 4 waves, 64 keys; each 32 keys are shared by a wave that holds K and sums
// dV (role A: S, P, handed over through LDS) and one that holds V and sums dK (role B).
// 1400-1520 us at 8192 tokens, 32/8 heads of 128, capped: the matrix units are busy 35% of it
// and the vector units 46%, the rest are the roles' waits for one another.  (344 bytes of
// scratch a lane, of the careful pass.  The
// roles of a workgroup's waves swapped in every other one, so that each SIMD has both: 2631
// -> 2644 us for the backward.)
template <int HD, int MODE>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(3))) void k_masked_dkdv(
    const uint16_t* __restrict__ q, int64_t ldq, const uint16_t* __restrict__ k, int64_t ldk,
    const uint16_t* __restrict__ v, int64_t ldv, const uint16_t* __restrict__ dO, int64_t lddo,
    const float* __restrict__ nl2, const float* __restrict__ delta, uint16_t* __restrict__ dk, int64_t lddk,
    uint16_t* __restrict__ dv, int64_t lddv, int T, int nkv, int group, ScoreArgs args, MaskTable mask, HeadSplit hs,
    int n_split) {
  constexpr int NKS = 2, NT = 256, BQ = 32, NS = HD / 16, ND = HD / 32, TILE = BQ * 2 * HD;
  // Two stages, each the Q tile and then the dO tile: a role picks by offset within the
  // stage's array, so the compiler knows which array a read touches.
  __shared__ __align__(16) char st0[2 * TILE], st1[2 * TILE];
  __shared__ __align__(16) float sl0[64], sl1[64], sd0[64], sd1[64];
  // P, under a cap times dz/ds, of each 32 keys, [j/4][lane][4].
  __shared__ __align__(16) float sp[NKS][16 * 64];
  const int tid = threadIdx.x, lane = tid & 63, hl = lane >> 5, l32 = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const bool role_a = wave < NKS;
  const int sub = role_a ? wave : wave - NKS;
  const int parts = dkdv_split<HD>(mask, T, hs, n_split);
  const XcdOrder ord = masked_order(nkv * parts);
  if (ord.y == nkv * parts) return;  // (the last of the grid: among the others they would take every other CU)
  const int kvh = ord.y / parts, split = ord.y - kvh * parts;
  const int gs = group / parts, h0 = kvh * group + split * gs;
  const int k0 = (mask.order_k64 != nullptr ? mask.order_k64[ord.rank] : ord.rank) * kSplitKeys, kw = k0 + sub * 32, ki = kw + l32;
  const int tiles = (T + kMaskRows - 1) / kMaskRows;
  const int4 all = mask_bounds<kSplitKeys / kMaskRows>(mask.queries, k0 / kMaskRows, tiles);
  const int4 mine = mask_bounds<1>(mask.queries, kw / kMaskRows, tiles);
  const int2 seen_by = ki < T ? *(reinterpret_cast<const int2*>(mask.rows + ki) + 1) : make_int2(0, 0);
  const int qbeg = all.x, n_tiles = all.y > all.x ? (all.y - all.x + BQ - 1) / BQ : 0;
  int a_off = lane_off_a<HD>(lane);
  int b0 = lane_off_b<HD>(lane, 0), b8 = lane_off_b<HD>(lane, 8);
  f32x16 acc[ND];  // dV^T (role A) or dK^T (role B)
#pragma unroll
  for (int dt = 0; dt < ND; ++dt) acc[dt] = zero16();
  const bool some = seen_by.x < seen_by.y;
  if (n_tiles > 0) {  // uniform
    bf16x8 kv[NS];  // K (role A) or V (role B) of this lane's key
    {
      const uint16_t* src = role_a ? k + static_cast<int64_t>(ki) * ldk : v + static_cast<int64_t>(ki) * ldv;
      src += static_cast<int64_t>(kvh) * HD + 8 * hl;
#pragma unroll
      for (int s = 0; s < NS; ++s) kv[s] = ki < T ? ld_frag(src + 16 * s) : as_bf16x8(make_uint4(0, 0, 0, 0));
    }
    const uint16_t* qg = q + static_cast<int64_t>(qbeg) * ldq + static_cast<int64_t>(h0) * HD;
    const uint16_t* gg = dO + static_cast<int64_t>(qbeg) * lddo + static_cast<int64_t>(h0) * HD;
    const float* lg = nl2 + static_cast<int64_t>(h0) * T + qbeg;
    const float* dg = delta + static_cast<int64_t>(h0) * T + qbeg;
    const int n_it = gs * n_tiles, last = T - 1 - qbeg;
    const int xoff = role_a ? 0 : TILE;  // phase 1 reads Q (A) or dO (B), phase 2 the other
    auto run = [&](auto careful) __attribute__((always_inline)) {
      constexpr bool CAREFUL = decltype(careful)::value;
      MaskedItems<HD, BQ, NT> items;
      items.start(n_tiles, ldq, lddo, wave, lane);
      items.load(qg, ldq, gg, lddo, lg, dg, T, last, gs, st0, st0 + TILE, sl0, sd0, wave, lane);
      wait_loads();
      __syncthreads();
      int qt = n_tiles - 1, hh = 0;
      auto step = [&](int it, const char* X0, const float* L, const float* D, char* XN, float* LN, float* DN)
                      __attribute__((always_inline)) {
        refresh_offsets(a_off, b0, b8);
        if (it + 1 < n_it) items.load(qg, ldq, gg, lddo, lg, dg, T, last, gs, XN, XN + TILE, LN, DN, wave, lane);
        const int qs = qbeg + qt * BQ;
        const bool active = it < n_it && mine.x < qs + BQ && mine.y > qs;  // the same for both roles
        const bool ends = mine.w < qs + BQ, starts = mine.z > qs;
        const int lo = seen_by.x - qs - 4 * hl, hi = seen_by.y - qs - 4 * hl;
        f32x16 x;  // S then P (role A) / dP then dS (role B), rows = queries, column = key
        if (active) {
          const char* X = X0 + xoff;
          x = zero16();
#pragma unroll
          for (int s = 0; s < NS; ++s) x = mfma(lds_frag<HD>(X, a_off, 0, s), kv[s], x);
          if (role_a) {
            const Score<MODE> score(args, h0 + hh);
            const float base = static_cast<float>(qs + 4 * hl - ki);
            f32x16 ds;
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              const float4 L4 = *reinterpret_cast<const float4*>(&L[8 * g + 4 * hl]);
              const float Lv[4] = {L4.x, L4.y, L4.z, L4.w};
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                float d;
                x[4 * g + e] = score.weight(x[4 * g + e], base + acc_row(4 * g + e, 0), Lv[e], d);
                if constexpr (MODE & kCap) ds[4 * g + e] = d;
              }
            }
            mask_range(x, ends, starts, lo, hi, 0, 0.f);
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              if constexpr (MODE & kCap) {
#pragma unroll
                for (int e = 0; e < 4; ++e) ds[4 * g + e] *= x[4 * g + e];
              } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) ds[4 * g + e] = x[4 * g + e];
              }
              *reinterpret_cast<float4*>(&sp[sub][(g * 64 + lane) * 4]) =
                  make_float4(ds[4 * g], ds[4 * g + 1], ds[4 * g + 2], ds[4 * g + 3]);
            }
          }
        }
        lds_barrier();  // P is in LDS; the loads into the other stage may still be in flight
        if (active) {
          if (!role_a) {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              const float4 D4 = *reinterpret_cast<const float4*>(&D[8 * g + 4 * hl]);
              const float4 P4 = *reinterpret_cast<const float4*>(&sp[sub][(g * 64 + lane) * 4]);
              const float Dv[4] = {D4.x, D4.y, D4.z, D4.w};
              const float Pv[4] = {P4.x, P4.y, P4.z, P4.w};
#pragma unroll
              for (int e = 0; e < 4; ++e) x[4 * g + e] = Pv[e] * (x[4 * g + e] - Dv[e]);
            }
            // P is 0 there, but what it is multiplied by need not be finite
            mask_range(x, ends, starts, lo, hi, 0, 0.f);
          }
          const char* Y = X0 + (TILE - xoff);
#pragma unroll
          for (int s2 = 0; s2 < 2; ++s2) {
            const bf16x8 f = pack_frag(x, 8 * s2);
            if constexpr (CAREFUL) {
              if (ends || starts) {
                wsum_careful<HD>(acc, f, Y, b0, b8, 16 * s2, lo + 4 * hl, hi + 4 * hl, hl);
                continue;
              }
            }
            wsum<HD>(acc, f, Y, b0, b8, 16 * s2);
          }
        }
        if (++hh == gs) {
          hh = 0;
          --qt;
        }
        wait_loads();
        __syncthreads();
      };
      for (int it = 0; it < n_it; it += 2) {
        step(it, st0, sl0, sd0, st1, sl1, sd1);
        step(it + 1, st1, sl1, sd1, st0, sl0, sd0);
      }
    };
    run(std::false_type{});
    if (__builtin_expect(__syncthreads_or(some && not_finite<ND>(acc)), 0)) {
#pragma unroll
      for (int dt = 0; dt < ND; ++dt) acc[dt] = zero16();
      run(std::true_type{});
    }
  }
  if (!some) {
#pragma unroll
    for (int dt = 0; dt < ND; ++dt) acc[dt] = zero16();
  }
  if (ki < T) {
    if (parts > 1) {
      store_rows_T_f32<HD>(hs.row(split, role_a ? 1 : 0, T, ki, nkv, kvh, HD), acc, hl);
    } else {
      uint16_t* row = role_a ? dv + static_cast<int64_t>(ki) * lddv : dk + static_cast<int64_t>(ki) * lddk;
      store_rows_T<HD>(row + static_cast<int64_t>(kvh) * HD, acc, role_a ? 1.f : grad_scale<MODE>(args), hl);
    }
  }
}

}  // namespace

// Workgroups that a kv head's query heads are split over: the smallest divisor of the
// group that gives every CU one workgroup (at head_dim 128 four, of which three run at once), and
// in long rows four (eight): dkdv_split.  A second kernel then adds their fp32 sums, whose
// bytes alone limit it: 256 MB.  head_dim 128, four a CU instead of two: 4096 tokens, 32/8
// heads, 844 -> 631 us for the backward, 8192 of 32/4 3343 -> 2313, in documents of 600 191 -> 166
// and 369 -> 296.  Up to 64 more than one loses in short rows: 16384 tokens, 32/4 heads of 64,
// documents of 600 308 -> 332.
MaskedWorkspace masked_workspace(fh_dtype dt, int64_t tokens, int64_t n_heads, int64_t n_kv_heads, int64_t head_dim) {
  MaskedWorkspace w{};
  w.split = w.long_split = 1;
  w.parts = (2 * tokens * n_heads + 3) / 4 * 4;
  w.total = w.parts;
  if (dt != FH_BF16) return w;
  const int64_t keys = head_dim <= 64 ? kFusedKeys : kSplitKeys, group = n_heads / n_kv_heads;
  const int64_t blocks = (tokens + keys - 1) / keys * n_kv_heads, want = head_dim <= 64 ? 256 : 1024;
  const int64_t most = int64_t(64) << 20;
  const int64_t part = 2 * tokens * n_kv_heads * head_dim;
  auto split = [&](int64_t wanted) {
    int s = 1;
    for (int64_t d = 2; d <= group && blocks * s < wanted; ++d)
      if (group % d == 0 && d * part <= most) s = static_cast<int>(d);
    return s;
  };
  w.split = split(want);
  w.long_split = tokens < kLongRows ? w.split : split(head_dim <= 64 ? 4 * want : 2 * want);
  if (w.long_split > 1) w.total += w.long_split * part;
  return w;
}

void masked_bwd_bf16(const MaskedBwd& c, const MaskedArgs& a, hipStream_t stream) {
  const MaskedWorkspace w = masked_workspace(FH_BF16, a.tokens, a.n_heads, a.n_kv_heads, a.head_dim);
  float* delta = c.workspace;
  float* nl2 = delta + a.tokens * a.n_heads;
  const int T = static_cast<int>(a.tokens), nkv = static_cast<int>(a.n_kv_heads);
  const int group = static_cast<int>(a.n_heads / a.n_kv_heads);
  const HeadSplit hs{c.workspace + w.parts, w.long_split};
  const auto q = static_cast<const uint16_t*>(c.q), k = static_cast<const uint16_t*>(c.k);
  const auto v = static_cast<const uint16_t*>(c.v), g = static_cast<const uint16_t*>(c.dout);
  const auto dk = static_cast<uint16_t*>(c.dk), dv = static_cast<uint16_t*>(c.dv);
  dispatch_masked(a.head_dim, a.mode, [&](auto hd, auto mode) {
    constexpr int HD = decltype(hd)::value, MODE = decltype(mode)::value;
    hipLaunchKernelGGL((k_masked_dq<HD, MODE>), dim3(static_cast<unsigned>((a.tokens + 127) / 128), static_cast<unsigned>(a.n_heads)),
                       dim3(256), 0, stream, q, c.ldq, k, c.ldk, v, c.ldv, static_cast<const uint16_t*>(c.o), c.ldo, g,
                       c.lddo, c.lse, c.o_low, delta, nl2, static_cast<uint16_t*>(c.dq), c.lddq, T, group, a.score, c.table);
    constexpr int64_t keys = HD <= 64 ? kFusedKeys : kSplitKeys;
    const dim3 grid(static_cast<unsigned>((a.tokens + keys - 1) / keys), static_cast<unsigned>(nkv * hs.n));
    if constexpr (HD <= 64)
      hipLaunchKernelGGL((k_masked_dkdv_fused<HD, MODE>), grid, dim3(512), 0, stream, q, c.ldq, k, c.ldk, v, c.ldv, g,
                         c.lddo, nl2, delta, dk, c.lddk, dv, c.lddv, T, nkv, group, a.score, c.table, hs, w.split);
    else
      hipLaunchKernelGGL((k_masked_dkdv<HD, MODE>), grid, dim3(256), 0, stream, q, c.ldq, k, c.ldk, v, c.ldv, g, c.lddo,
                         nl2, delta, dk, c.lddk, dv, c.lddv, T, nkv, group, a.score, c.table, hs, w.split);
    if (hs.n > 1) {
      const int64_t threads = a.tokens * nkv * (HD / 8);
      hipLaunchKernelGGL((k_masked_dkdv_sum<HD>), dim3(static_cast<unsigned>((threads + 255) / 256)), dim3(256), 0, stream,
                         hs, w.split, c.table, dk, c.lddk, dv, c.lddv, T, nkv, (MODE & kCap ? 4.f : 1.f) * a.score.scale);
    }
  });
}

}  // namespace fh
