// The norms after and before a block with the block's gate and residual scale:
//   n = RMSNorm(a; w_post)     (or a, without w_post)
//   h = to_dtype(x + s g n)    (g: one value a channel, or one a token and channel, or none)
//   y = RMSNorm(h; w_pre)      (nothing, without w_pre)
// and the backward of both outputs.  a is a block's output, x the residual
// stream, y the next block's input.
//
// Arithmetic is fp32 with one rounding where a tensor is stored: the
// normalised values are not rounded on the way (fh_add_rmsnorm_fwd rounds them
// where Hugging Face's module does; no module of the reference has this form).
// y is the norm of h as stored, which is what any later reader of h sees.
//
// Both are HBM-bound: forward 4 and backward 6 passes over [rows, cols] (one and
// two more with a per-token gate), each tensor read or written once, the rows in
// registers between the two reductions.  WPR waves share a row (at most 1024
// columns each, NVW <= 2 chunks of 8 a lane), which keeps the backward's four
// rows, three vectors and two sums under 128 registers: four waves a SIMD.
// 16384 x 2048 bf16 with a channel gate: forward 45.9 us call after call (268 MB,
// 5.8 TB/s) and 52 with a backward between (5.1), backward 75.5 us (403 MB, 5.3)
// and its sums 4; a copy runs at 5.4.  Non-temporal stores of h and y cost 4.1 us
// (55.5 -> 59.6 with a backward between), of dx and da 2.7 (81.4 -> 84.1).  With a gate
// per token, 8192 x 4096: forward 59 us (336 MB, 5.7 TB/s), backward 100 (537 MB, 5.4).
// fp32: 16384 x 2048 with a channel gate 110 and 160 (537 and 805 MB, 4.9 and 5.0),
// 8192 x 4096 with a gate per token 126 and 216 (671 and 1074 MB, 5.3 and 5.0).
#include "femtohip_blocks.h"
#include "fh_common.hpp"
#include "fh_parts.hpp"

namespace fh {
namespace {

constexpr int kNoGate = 0, kChannelGate = 1, kTokenGate = 2;
constexpr int kWaves = 8;  // waves of a block

// Sum of v over the WPR waves of a row, given to all of them (the row's waves
// are neighbours in the block; red: one float a wave, not reused before the
// next barrier but one).
template <int WPR>
__device__ __forceinline__ float row_sum(float v, float* red, int wave, int lane) {
  v = wave_sum(v);
  if constexpr (WPR == 1) return v;
  if (lane == 0) red[wave] = v;
  __syncthreads();
  const int first = wave / WPR * WPR;
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < WPR; ++i) s += red[first + i];
  return s;
}

// A block takes kWaves / WPR rows a step; its barriers are reached by every wave
// (the step loop is uniform, rows behind the last one are computed on zeros).
// Non-temporal loads, 16384 x 2048, us: backward 86.6 -> 81.4, forward with a per-token
// gate (8192 x 4096) 62.1 -> 56.7; the forward's two rows without one 45.9 against
// 47.1, so not there.
template <typename T, int NVW, int WPR, int GATE, bool POST, bool PRE>
__global__ __launch_bounds__(64 * kWaves) void k_block_norms_fwd(
    const T* __restrict__ x, const T* __restrict__ a, const T* __restrict__ w_post, const T* __restrict__ w_pre,
    const T* __restrict__ gate, float scale, T* __restrict__ h, T* __restrict__ y, float* __restrict__ rstd_a,
    float* __restrict__ rstd_h, int64_t rows, int cols, float eps) {
  using E = Elem<T>;
  using Raw = typename E::Raw;
  constexpr int RPB = kWaves / WPR;
  __shared__ float red[2][2][kWaves];  // [step parity][a | h][wave]
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x >> 6;
  const int rsub = wave / WPR, slice = wave % WPR;
  auto col = [&](int i) { return ((slice * NVW + i) * kWave + lane) * 8; };

  [[maybe_unused]] Raw wpo[NVW], wpr[NVW], gc[NVW];
#pragma unroll
  for (int i = 0; i < NVW; ++i) {
    if (col(i) >= cols) continue;
    if constexpr (POST) wpo[i] = E::ldraw(w_post + col(i));
    if constexpr (PRE) wpr[i] = E::ldraw(w_pre + col(i));
    if constexpr (GATE == kChannelGate) gc[i] = E::ldraw(gate + col(i));
  }
  const float inv_cols = 1.f / static_cast<float>(cols);
  int par = 0;
  for (int64_t step0 = static_cast<int64_t>(blockIdx.x) * RPB; step0 < rows;
       step0 += static_cast<int64_t>(gridDim.x) * RPB, par ^= 1) {
    const int64_t row = step0 + rsub, base = row * cols;
    const bool valid = row < rows;
    auto in = [&](int i) { return valid && col(i) < cols; };
    Raw xr[NVW], ar[NVW];
    [[maybe_unused]] Raw gr[NVW];
#pragma unroll
    for (int i = 0; i < NVW; ++i) {
      if (!in(i)) continue;
      ar[i] = load_if<T, GATE == kTokenGate>(a + base + col(i));
      xr[i] = load_if<T, GATE == kTokenGate>(x + base + col(i));
      if constexpr (GATE == kTokenGate) gr[i] = load_if<T, GATE == kTokenGate>(gate + base + col(i));
    }
    float ra = 1.f;
    if constexpr (POST) {
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < NVW; ++i) {
        if (!in(i)) continue;
        float v[8];
        E::unpack(ar[i], v);
#pragma unroll
        for (int j = 0; j < 8; ++j) ss = fmaf(v[j], v[j], ss);
      }
      ra = rsqrtf(row_sum<WPR>(ss, red[par][0], wave, lane) * inv_cols + eps);
      if (rstd_a != nullptr && valid && slice == 0 && lane == 0) rstd_a[row] = ra;
    }
    // (a r) w_post and s g first, then their product, and (h r) w_pre below: where a
    // row's squares overflow r is 0, and so is a r w_post, while a w_post may be infinite.
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < NVW; ++i) {
      if (!in(i)) continue;
      float v[8], n[8], t[8];
      E::unpack(xr[i], v);
      E::unpack(ar[i], n);
      if constexpr (POST) {
        E::unpack(wpo[i], t);
#pragma unroll
        for (int j = 0; j < 8; ++j) n[j] = n[j] * ra * t[j];
      }
      if constexpr (GATE != kNoGate) E::unpack(GATE == kChannelGate ? gc[i] : gr[i], t);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        v[j] = E::rnd(fmaf(n[j], GATE != kNoGate ? scale * t[j] : scale, v[j]));
        ss = fmaf(v[j], v[j], ss);
      }
      xr[i] = E::pack(v);
      E::straw(h + base + col(i), xr[i]);
    }
    if constexpr (PRE) {
      const float rh = rsqrtf(row_sum<WPR>(ss, red[par][1], wave, lane) * inv_cols + eps);
      if (rstd_h != nullptr && valid && slice == 0 && lane == 0) rstd_h[row] = rh;
#pragma unroll
      for (int i = 0; i < NVW; ++i) {
        if (!in(i)) continue;
        float v[8], t[8];
        E::unpack(xr[i], v);
        E::unpack(wpr[i], t);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = v[j] * rh * t[j];
        E::store8(y + base + col(i), v);
      }
    }
  }
}

// Backward of (dh, dy), the gradients of h and y:
//   D  = dh + r_h (dy w_pre - n_h mean(dy w_pre n_h)),   n_h = h r_h
//   dx = D,  dw_pre = sum dy n_h
//   P  = s g D,  n_a = a r_a (or a)
//   da = r_a (P w_post - n_a mean(P w_post n_a))         (or P)
//   dw_post = sum P n_a
//   dg = s D n_a w_post, summed over the rows for a channel gate
// D stays in fp32 registers between the two norms.  Of a channel gate both
// dw_post and dg come from S = sum s D n_a: dw_post = g S, dg = w_post S.  part:
// per block one row of sum dy n_h (PRE) and one of S, or of sum P n_a for a token
// gate (SUM), in fp32; k_block_norms_sums adds them in a fixed order.
template <typename T, int NVW, int WPR, int GATE, bool POST, bool PRE>
__global__ __launch_bounds__(64 * kWaves) void k_block_norms_bwd(
    const T* __restrict__ dh, const T* __restrict__ dy, const T* __restrict__ h, const T* __restrict__ a,
    const T* __restrict__ w_post, const T* __restrict__ w_pre, const T* __restrict__ gate, float scale,
    const float* __restrict__ rstd_a, const float* __restrict__ rstd_h, T* __restrict__ dx, T* __restrict__ da,
    T* __restrict__ dgate, float* __restrict__ part, int64_t rows, int cols) {
  using E = Elem<T>;
  using Raw = typename E::Raw;
  constexpr int RPB = kWaves / WPR;
  constexpr bool SUM = POST || GATE == kChannelGate;  // a sum over rows besides dw_pre
  constexpr bool A = POST || GATE != kNoGate;         // a's values are needed
  extern __shared__ float acc_lds[];                  // cols floats
  __shared__ float red[2][2][kWaves];                 // [step parity][h | a][wave]
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x >> 6;
  const int rsub = wave / WPR, slice = wave % WPR;
  auto col = [&](int i) { return ((slice * NVW + i) * kWave + lane) * 8; };

  [[maybe_unused]] Raw wpo[NVW], wpr[NVW], gc[NVW];
  [[maybe_unused]] float acc_pre[NVW][8], acc_sum[NVW][8];
#pragma unroll
  for (int i = 0; i < NVW; ++i) {
#pragma unroll
    for (int j = 0; j < 8; ++j) acc_pre[i][j] = acc_sum[i][j] = 0.f;
    if (col(i) >= cols) continue;
    if constexpr (POST) wpo[i] = E::ldraw(w_post + col(i));
    if constexpr (PRE) wpr[i] = E::ldraw(w_pre + col(i));
    if constexpr (GATE == kChannelGate) gc[i] = E::ldraw(gate + col(i));
  }
  const float inv_cols = 1.f / static_cast<float>(cols);
  int par = 0;
  for (int64_t step0 = static_cast<int64_t>(blockIdx.x) * RPB; step0 < rows;
       step0 += static_cast<int64_t>(gridDim.x) * RPB, par ^= 1) {
    const int64_t row = step0 + rsub, base = row * cols;
    const bool valid = row < rows;
    auto in = [&](int i) { return valid && col(i) < cols; };
    Raw dhr[NVW];
    [[maybe_unused]] Raw dyr[NVW], hr[NVW], ar[NVW], gr[NVW];
#pragma unroll
    for (int i = 0; i < NVW; ++i) {
      if (!in(i)) continue;
      if constexpr (PRE) {
        dyr[i] = load_if<T, true>(dy + base + col(i));
        hr[i] = load_if<T, true>(h + base + col(i));
      }
      dhr[i] = load_if<T, true>(dh + base + col(i));
      if constexpr (A) ar[i] = load_if<T, true>(a + base + col(i));
      if constexpr (GATE == kTokenGate) gr[i] = load_if<T, true>(gate + base + col(i));
    }
    float D[NVW][8];
    float dot = 0.f, rh = 0.f;
    if constexpr (PRE) {
      rh = valid ? rstd_h[row] : 0.f;
#pragma unroll
      for (int i = 0; i < NVW; ++i) {
        if (!in(i)) continue;
        float g[8], v[8], w[8];
        E::unpack(dyr[i], g);
        E::unpack(hr[i], v);
        E::unpack(wpr[i], w);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float n = v[j] * rh;
          dot = fmaf(g[j] * w[j], n, dot);
          acc_pre[i][j] = fmaf(g[j], n, acc_pre[i][j]);
        }
      }
      dot = row_sum<WPR>(dot, red[par][0], wave, lane) * inv_cols;
    }
    float ra = 1.f, dot2 = 0.f;
    if constexpr (POST) ra = valid ? rstd_a[row] : 0.f;
#pragma unroll
    for (int i = 0; i < NVW; ++i) {
      if (!in(i)) continue;
      E::unpack(dhr[i], D[i]);
      if constexpr (PRE) {
        float g[8], v[8], w[8];
        E::unpack(dyr[i], g);
        E::unpack(hr[i], v);
        E::unpack(wpr[i], w);
#pragma unroll
        for (int j = 0; j < 8; ++j) D[i][j] += rh * (g[j] * w[j] - v[j] * rh * dot);
      }
      E::store8(dx + base + col(i), D[i]);
      if constexpr (A) {
        float n[8], w[8], g[8];
        E::unpack(ar[i], n);
        if constexpr (POST) E::unpack(wpo[i], w);
        if constexpr (GATE == kChannelGate) E::unpack(gc[i], g);
        if constexpr (GATE == kTokenGate) E::unpack(gr[i], g);
        float o[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if constexpr (POST) n[j] *= ra;
          const float sD = scale * D[i][j];
          if constexpr (GATE == kTokenGate) {
            o[j] = sD * n[j];
            if constexpr (POST) o[j] *= w[j];
          }
          float P = sD;
          if constexpr (GATE != kNoGate) P *= g[j];
          if constexpr (SUM) acc_sum[i][j] = fmaf(GATE == kChannelGate ? sD : P, n[j], acc_sum[i][j]);
          if constexpr (POST) {
            P *= w[j];
            dot2 = fmaf(P, n[j], dot2);
          }
          D[i][j] = P;
        }
        if constexpr (GATE == kTokenGate) E::store8(dgate + base + col(i), o);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) D[i][j] *= scale;
      }
    }
    if constexpr (POST) dot2 = row_sum<WPR>(dot2, red[par][1], wave, lane) * inv_cols;
#pragma unroll
    for (int i = 0; i < NVW; ++i) {
      if (!in(i)) continue;
      if constexpr (POST) {
        float n[8];
        E::unpack(ar[i], n);
#pragma unroll
        for (int j = 0; j < 8; ++j) D[i][j] = ra * (D[i][j] - n[j] * ra * dot2);
      }
      E::store8(da + base + col(i), D[i]);
    }
  }

  // The waves' sums, row groups in order, to this block's partial rows.
  float* dst = part + static_cast<int64_t>(blockIdx.x) * ((PRE ? 1 : 0) + (SUM ? 1 : 0)) * cols;
  auto put = [&](const float (&acc)[NVW][8]) {
    __syncthreads();
    for (int s = 0; s < RPB; ++s) {
      if (rsub == s) {
#pragma unroll
        for (int i = 0; i < NVW; ++i) {
          const int c = col(i);
          if (c >= cols) continue;
#pragma unroll
          for (int j = 0; j < 8; ++j) acc_lds[c + j] = s == 0 ? acc[i][j] : acc_lds[c + j] + acc[i][j];
        }
      }
      __syncthreads();
    }
    for (int c = threadIdx.x; c < cols; c += blockDim.x) dst[c] = acc_lds[c];
    dst += cols;
  };
  if constexpr (PRE) put(acc_pre);
  if constexpr (SUM) put(acc_sum);
}

// The sums over the partial rows (fh_parts.hpp; blockIdx.y: which of a row's) and, from
// them, the vectors' gradients.
template <typename T>
__global__ __launch_bounds__(256) void k_block_norms_sums(const float* __restrict__ part, int nparts, int nsums,
                                                          int cols, bool pre, const T* __restrict__ w_post,
                                                          const T* __restrict__ gate, bool channel,
                                                          T* __restrict__ dw_pre, T* __restrict__ dw_post,
                                                          T* __restrict__ dgate) {
  const float t = sum_parts(part + static_cast<int64_t>(blockIdx.y) * cols, static_cast<int64_t>(nsums) * cols, nparts, cols);
  const int c = blockIdx.x * 16 + static_cast<int>(threadIdx.x);
  if (threadIdx.x >= 16 || c >= cols) return;
  if (pre && blockIdx.y == 0) {
    Elem<T>::st1(dw_pre + c, t);
  } else {
    if (dw_post != nullptr) Elem<T>::st1(dw_post + c, channel ? t * Elem<T>::ld1(gate + c) : t);
    if (channel) Elem<T>::st1(dgate + c, w_post != nullptr ? t * Elem<T>::ld1(w_post + c) : t);
  }
}

// Largest grids: the forward two blocks a CU; the backward one, since each leaves
// partial rows (512 blocks 92.6 us and 384 98, 256 86.6 at 16384 x 2048).  Loading
// the next step's rows ahead gained nothing (82.7 against 81.4).
constexpr int kMaxBlocks[2] = {512, 256};

// Waves a row: at most two chunks of 8 a lane (one: 91.6 us; four spill).
constexpr int waves_per_row(int64_t cols) { return cols <= 1024 ? 1 : cols <= 2048 ? 2 : cols <= 4096 ? 4 : 8; }

// f(chunks of 8 a lane, waves a row).
template <typename F>
void dispatch_cols(int cols, F&& f) {
  using std::integral_constant;
  auto go = [&](auto c) {
    constexpr int wpr = waves_per_row(c());
    f(integral_constant<int, c() / 512 / wpr>{}, integral_constant<int, wpr>{});
  };
  if (cols <= 512) go(integral_constant<int, 512>{});
  else if (cols <= 1024) go(integral_constant<int, 1024>{});
  else if (cols <= 2048) go(integral_constant<int, 2048>{});
  else if (cols <= 4096) go(integral_constant<int, 4096>{});
  else go(integral_constant<int, 8192>{});
}

int grid_of(int64_t rows, int64_t cols, bool bwd) {
  const int64_t rpb = kWaves / waves_per_row(cols), need = (rows + rpb - 1) / rpb;
  return static_cast<int>(need < kMaxBlocks[bwd] ? need : kMaxBlocks[bwd]);
}

// f(element tag, gate mode, has w_post, has w_pre); one of the norms is there.
template <typename F>
void dispatch_mode(fh_dtype dt, bool gate, bool token, bool post, bool pre, F&& f) {
  auto norms = [&](auto tag, auto g) {
    if (post && pre) f(tag, g, std::true_type{}, std::true_type{});
    else if (post) f(tag, g, std::true_type{}, std::false_type{});
    else f(tag, g, std::false_type{}, std::true_type{});
  };
  auto gates = [&](auto tag) {
    if (!gate) norms(tag, std::integral_constant<int, kNoGate>{});
    else if (token) norms(tag, std::integral_constant<int, kTokenGate>{});
    else norms(tag, std::integral_constant<int, kChannelGate>{});
  };
  if (dt == FH_BF16) gates(uint16_t{});
  else gates(float{});
}

int check(fh_dtype dt, int64_t rows, int64_t cols, const void* w_post, const void* w_pre) {
  FH_REQUIRE(dt == FH_BF16 || dt == FH_F32, "block_norms: dtype must be FH_BF16 or FH_F32");
  FH_REQUIRE(rows >= 0, "block_norms: rows must be >= 0");
  FH_REQUIRE(cols > 0 && cols % 8 == 0 && cols <= 8192,
             "block_norms: cols must be a positive multiple of 8 and <= 8192");
  FH_REQUIRE(w_post || w_pre, "block_norms: at least one of w_post and w_pre is needed");
  return FH_OK;
}

template <typename... P>
bool all_aligned(const P*... p) {
  return (aligned16(p) && ...);  // a null pointer is aligned
}

}  // namespace
}  // namespace fh

using namespace fh;

extern "C" int fh_block_norms_fwd(fh_dtype dt, const void* x, const void* a, const void* w_post, const void* w_pre,
                                  const void* gate, int gate_per_token, float scale, void* h, void* y, float* rstd_post,
                                  float* rstd_pre, int64_t rows, int64_t cols, float eps, hipStream_t stream) {
  if (int e = check(dt, rows, cols, w_post, w_pre)) return e;
  if (rows == 0) return FH_OK;
  FH_REQUIRE(x && a && h && (y || !w_pre), "block_norms_fwd: null pointer");
  FH_REQUIRE(all_aligned(x, a, w_post, w_pre, gate, h, y), "block_norms_fwd: pointers must be 16-byte aligned");
  FH_REQUIRE(h != x && h != a && h != gate, "block_norms_fwd: h must not alias x, a or the gate");
  const int c = static_cast<int>(cols), blocks = grid_of(rows, cols, false);
  dispatch_mode(dt, gate != nullptr, gate_per_token != 0, w_post != nullptr, w_pre != nullptr,
                [&](auto tag, auto gm, auto post, auto pre) {
    using T = decltype(tag);
    dispatch_cols(c, [&](auto nvw, auto wpr) {
      hipLaunchKernelGGL((k_block_norms_fwd<T, nvw(), wpr(), gm(), post(), pre()>), dim3(blocks), dim3(64 * kWaves), 0,
                         stream, static_cast<const T*>(x), static_cast<const T*>(a), static_cast<const T*>(w_post),
                         static_cast<const T*>(w_pre), static_cast<const T*>(gate), scale, static_cast<T*>(h),
                         static_cast<T*>(y), rstd_post, rstd_pre, rows, c, eps);
    });
  });
  return check_launch("fh_block_norms_fwd");
}

extern "C" size_t fh_block_norms_bwd_workspace_size(int64_t rows, int64_t cols) {
  if (rows <= 0 || cols <= 0) return 0;
  return static_cast<size_t>(grid_of(rows, cols, true)) * 2 * static_cast<size_t>(cols) * sizeof(float);
}

extern "C" int fh_block_norms_bwd(fh_dtype dt, const void* dh, const void* dy, const void* h, const void* a,
                                  const void* w_post, const void* w_pre, const void* gate, int gate_per_token,
                                  float scale, const float* rstd_post, const float* rstd_pre, void* dx, void* da,
                                  void* dw_post, void* dw_pre, void* dgate, void* workspace, int64_t rows, int64_t cols,
                                  hipStream_t stream) {
  if (int e = check(dt, rows, cols, w_post, w_pre)) return e;
  const bool token = gate && gate_per_token, channel = gate && !gate_per_token;
  FH_REQUIRE((dw_post || !w_post) && (dw_pre || !w_pre) && (dgate || !channel), "block_norms_bwd: null pointer");
  const int c = static_cast<int>(cols);
  const int nsums = (w_pre ? 1 : 0) + (w_post || channel ? 1 : 0);
  int blocks = 0;
  if (rows > 0) {
    FH_REQUIRE(dh && dx && da && workspace, "block_norms_bwd: null pointer");
    FH_REQUIRE(!w_pre || (dy && h && rstd_pre), "block_norms_bwd: null pointer (dy, h and rstd_pre with w_pre)");
    FH_REQUIRE(!w_post || rstd_post, "block_norms_bwd: null pointer (rstd_post with w_post)");
    FH_REQUIRE(a || !(w_post || gate), "block_norms_bwd: null pointer (a with w_post or a gate)");
    FH_REQUIRE(!token || dgate, "block_norms_bwd: null pointer (dgate with a gate)");
    FH_REQUIRE(all_aligned(dh, dy, h, a, w_post, w_pre, gate, dx, da, dgate, workspace),
               "block_norms_bwd: pointers (workspace included) must be 16-byte aligned");
    blocks = grid_of(rows, cols, true);
    dispatch_mode(dt, gate != nullptr, token, w_post != nullptr, w_pre != nullptr,
                  [&](auto tag, auto gm, auto post, auto pre) {
      using T = decltype(tag);
      dispatch_cols(c, [&](auto nvw, auto wpr) {
        hipLaunchKernelGGL((k_block_norms_bwd<T, nvw(), wpr(), gm(), post(), pre()>), dim3(blocks), dim3(64 * kWaves),
                           static_cast<size_t>(cols) * sizeof(float), stream, static_cast<const T*>(dh),
                           static_cast<const T*>(dy), static_cast<const T*>(h), static_cast<const T*>(a),
                           static_cast<const T*>(w_post), static_cast<const T*>(w_pre), static_cast<const T*>(gate),
                           scale, rstd_post, rstd_pre, static_cast<T*>(dx), static_cast<T*>(da),
                           static_cast<T*>(dgate), static_cast<float*>(workspace), rows, c);
      });
    });
  }
  // With no rows the sums are over no partial rows: zeros.
  auto sums = [&](auto tag) {
    using T = decltype(tag);
    hipLaunchKernelGGL((k_block_norms_sums<T>), dim3((c + 15) / 16, nsums), dim3(256), 0, stream,
                       static_cast<const float*>(workspace), blocks, nsums, c, w_pre != nullptr,
                       static_cast<const T*>(w_post), static_cast<const T*>(gate), channel, static_cast<T*>(dw_pre),
                       static_cast<T*>(dw_post), static_cast<T*>(dgate));
  };
  if (dt == FH_BF16) sums(uint16_t{});
  else sums(float{});
  return check_launch("fh_block_norms_bwd");
}
