// RMSNorm forward / residual-add + RMSNorm forward / RMSNorm backward: the
// kernels of fh_norm.hip (x in the model's dtype) and fh_norm8.hip (x kept in 8
// bits, or packed on the way).
//
// Reference arithmetic: LlamaRMSNorm.forward, transformers 5.15.0
// models/llama/modeling_llama.py:62-67, and the residual adds at :317/:323.
//
// Layout: lane l of a wave owns the 8-element chunks starting at columns
// (i*64 + l)*8 of its share of a row, so each load instruction of a wave
// covers one contiguous 1 KiB (bf16) span; rows stay in registers, packed as
// loaded, between the reduction and the normalisation, so every input is read
// from HBM exactly once.  The weight row is loaded once per wave, together
// with the first data, so its latency is never on a row's critical path.
//
// XS (RowsT or Rows8) is how x is read; an x kept in 8 bits unpacks to values
// that T holds exactly, so every result equals, bit for bit, that of the
// unpacked tensor.  RND: the normalised value and dy * w are rounded to T, as
// LlamaRMSNorm's tensors are; without it only what is stored is rounded.
#pragma once

#include "fh_common.hpp"
#include "fh_pack8.hpp"
#include "fh_parts.hpp"

namespace fh {
namespace {

// x as rows of T.
template <typename T>
struct RowsT {
  static constexpr bool kPacked = false;
  using Item = T;
  using Raw = typename Elem<T>::Raw;
  // Elements c..c+7 of the row that starts at base (and, kept in 8 bits, its
  // exponents at ebase): both computed once a row, outside the column tests.
  __device__ __forceinline__ static Raw load(const T* x, const uint8_t*, int64_t base, int64_t, int c) {
    return Elem<T>::ldraw(x + base + c);
  }
  __device__ __forceinline__ static void unpack(const Raw& q, float v[8]) { Elem<T>::unpack(q, v); }
};

// x as codes and exponent bytes (fh_pack8.hpp).
template <int FMT>
struct Rows8 {
  static constexpr bool kPacked = true;
  using Item = uint8_t;
  using Raw = Raw8;
  __device__ __forceinline__ static Raw load(const uint8_t* x, const uint8_t* xe, int64_t base, int64_t ebase, int c) {
    return load8_codes(x + base, xe + ebase, c);
  }
  __device__ __forceinline__ static void unpack(const Raw& q, float v[8]) { unpack8<FMT>(q, v); }
};

template <typename T, bool RND>
__device__ __forceinline__ float rnd_if(float f) {
  if constexpr (RND) return Elem<T>::rnd(f);
  else return f;
}

constexpr int kWavesPerBlock = 4;  // 256 threads

// Forward: each wave takes rows row, row + stride, ... (stride = 4 x grid).
// With PIPE the next row's loads are issued before this row is reduced and
// stored, so a wave keeps two rows in flight; without it the grid covers every
// row once (one row per wave).  The pipelined form is used for add+RMSNorm
// (two input rows): 45.2 -> 43.1 us at T = 16384, H = 2048 and 50.5 -> 48.8 us
// at T = 8192, H = 4096; the one-input form measured no gain from it.
// PACK: x also goes out in 8 bits (a format of fh_pack8.hpp; kNoPack: it does not).
// The arguments of packed calls alone stand last: the others fill one 64-byte line,
// and in the second one rows and cols cost every wave a wait (add + norm of 8192 x
// 4096 47.2 us, 48.2 with them there).
// WPR waves share a row, each NV chunks a lane; with more than one a block's waves
// go through its steps together (rows behind the last one are computed on zeros).
template <typename T, typename XS, int NV, int WPR, bool ADD, bool PIPE, int PACK, bool RND>
__global__ __launch_bounds__(256) void k_rmsnorm_fwd(
    const typename XS::Item* __restrict__ x, const T* __restrict__ a, const T* __restrict__ w, T* __restrict__ h,
    T* __restrict__ y, float* __restrict__ rstd, int64_t rows, int cols, float eps, const uint8_t* __restrict__ xe,
    uint8_t* __restrict__ codes, uint8_t* __restrict__ exps) {
  using Raw = typename Elem<T>::Raw;
  using XRaw = typename XS::Raw;
  constexpr int RPB = kWavesPerBlock / WPR;  // rows of a block's step
  [[maybe_unused]] __shared__ float red[2][kWavesPerBlock];  // [step parity][wave]
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x >> 6;
  const int rsub = wave / WPR, slice = wave % WPR;
  int64_t row = static_cast<int64_t>(blockIdx.x) * RPB + rsub;
  const int64_t stride = static_cast<int64_t>(gridDim.x) * RPB;
  if (WPR == 1 && row >= rows) return;  // uniform per wave
  auto col = [&](int i) { return ((slice * NV + i) * kWave + lane) * 8; };
  auto in = [&](int c, int64_t rr) { return c < cols && (WPR == 1 || rr < rows); };

  XRaw xn[NV];
  Raw wr[NV];
  [[maybe_unused]] Raw an[NV];
  auto load_row = [&](int64_t rr) {
    const int64_t base = rr * cols;
    [[maybe_unused]] const int64_t ebase = XS::kPacked ? rr * blocks8(cols) : 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = col(i);
      if (in(c, rr)) {
        xn[i] = XS::load(x, xe, base, ebase, c);
        if constexpr (ADD) an[i] = Elem<T>::ldraw(a + base + c);
      }
    }
  };
  load_row(row);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = col(i);
    if (c < cols) wr[i] = Elem<T>::ldraw(w + c);
  }
  [[maybe_unused]] int par = 0;
  // Normalises row rr from its loaded chunks (xr, and ar with ADD).
  auto norm_row = [&](int64_t rr, XRaw* xr, [[maybe_unused]] Raw* ar) {
    const int64_t base = rr * cols;
    [[maybe_unused]] const int64_t ebase = PACK != kNoPack ? rr * blocks8(cols) : 0;
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = col(i);
      if (in(c, rr)) {
        float v[8];
        XS::unpack(xr[i], v);
        if constexpr (ADD) {  // h = to_dtype(x + a), kept packed (in x's place, or a's) for the normalisation
          float b[8];
          Elem<T>::unpack(ar[i], b);
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] = Elem<T>::rnd(v[j] + b[j]);
          auto& hr = [&]() -> Raw& {
            if constexpr (XS::kPacked) return ar[i];
            else return xr[i];
          }();
          hr = Elem<T>::pack(v);
          Elem<T>::straw(h + base + c, hr);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) ss = fmaf(v[j], v[j], ss);
      }
      if constexpr (PACK != kNoPack) {
        float v[8] = {};
        if (in(c, rr)) XS::unpack(xr[i], v);
        pack8_store<PACK>(v, codes + base, exps + ebase, in(c, rr), c);
      }
    }
    ss = wave_sum(ss);
    if constexpr (WPR > 1) {
      if (lane == 0) red[par][wave] = ss;
      __syncthreads();
      ss = 0.f;
#pragma unroll
      for (int s = 0; s < WPR; ++s) ss += red[par][rsub * WPR + s];
      par ^= 1;
    }
    const float r = rsqrtf(ss / static_cast<float>(cols) + eps);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = col(i);
      if (in(c, rr)) {
        float v[8], wv[8], o[8];
        if constexpr (ADD && XS::kPacked) Elem<T>::unpack(ar[i], v);
        else XS::unpack(xr[i], v);
        Elem<T>::unpack(wr[i], wv);
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] = Elem<T>::rnd(wv[j] * rnd_if<T, RND>(v[j] * r));
        Elem<T>::store8(y + base + c, o);
      }
    }
    if (rstd != nullptr && lane == 0 && slice == 0 && (WPR == 1 || rr < rows)) rstd[rr] = r;
  };
  if constexpr (!PIPE) {
    norm_row(row, xn, an);
  } else {
    for (; row - rsub * (WPR > 1) < rows; row += stride) {  // uniform per wave, and per block where waves share rows
      XRaw xr[NV];
      [[maybe_unused]] Raw ar[NV];
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        xr[i] = xn[i];
        if constexpr (ADD) ar[i] = an[i];
      }
      if (row + stride < rows) load_row(row + stride);
      norm_row(row, xr, ar);
    }
  }
}

// Backward.  WPR waves share a row (WPR = 2 above 2048 columns), each holding
// NVW chunks of 8 per lane, so every width keeps the register footprint of a
// 2048-column row.  A block's 4 waves take 4/WPR rows per step; the step loop
// is uniform across the block (its barriers combine the WPR per-wave partial
// sums of a row in a fixed order, through a parity-double-buffered LDS slot).
// Per row:
//   r   = rstd (given) or rsqrt(mean(x^2) + eps)
//   dn  = to_dtype(dy * w)          (the gradient at the bf16 normalised value)
//   dot = mean(dn * x * r)
//   dx  = r * (dn - x * r * dot) [+ dres]
//   dw += dy * to_dtype(x * r)      (per-wave registers)
// The weight-gradient partials of the block's waves are summed in a fixed
// order through LDS into one fp32 row per block (deterministic), which
// k_reduce_parts folds into dw.
// Next-row prefetch (PF): measured 50.6 -> 43.5 us without the residual
// gradient at T=16384, H=2048; with it (3 input rows) at that width the extra
// registers cost a wave of occupancy and it gained nothing (60.8 vs 62.3 us);
// BwdSplit chooses it per width.
template <typename T, typename XS, int NVW, int WPR, int NWB, bool RES, bool HAVE_RSTD, bool PF, bool RND,
          bool STREAM>
__global__ __launch_bounds__(64 * NWB) void k_rmsnorm_bwd(
    const T* __restrict__ dy, const typename XS::Item* __restrict__ x, const T* __restrict__ w,
    const float* __restrict__ rstd, const T* __restrict__ dres, T* __restrict__ dx, float* __restrict__ part,
    int64_t rows, int cols, float eps, const uint8_t* __restrict__ xe) {
  using Raw = typename Elem<T>::Raw;
  using XRaw = typename XS::Raw;
  constexpr int RPB = NWB / WPR;  // rows per block step (NWB waves per block)
  extern __shared__ float lds_acc[];          // cols floats
  __shared__ float red[2][2][NWB];  // [step parity][ss | dot][wave]
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = threadIdx.x >> 6;
  const int rsub = wave / WPR, slice = wave % WPR;
  auto col = [&](int i) { return ((slice * NVW + i) * kWave + lane) * 8; };

  Raw wr[NVW];
#pragma unroll
  for (int i = 0; i < NVW; ++i)
    if (col(i) < cols) wr[i] = Elem<T>::ldraw(w + col(i));
  float acc[NVW][8];
#pragma unroll
  for (int i = 0; i < NVW; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[i][j] = 0.f;

  const float inv_cols = 1.f / static_cast<float>(cols);
  const int64_t stride = static_cast<int64_t>(gridDim.x) * RPB;
  // Loads of one row; with PF the next step's row is loaded while this one is
  // processed (two rows of this wave in flight).
  XRaw xn[NVW];
  Raw gn[NVW];
  [[maybe_unused]] Raw rn[NVW];
  auto load_row = [&](int64_t row) {
    if (row >= rows) return;
    const int64_t base = row * cols;
    [[maybe_unused]] const int64_t ebase = XS::kPacked ? row * blocks8(cols) : 0;
#pragma unroll
    for (int i = 0; i < NVW; ++i) {
      const int c = col(i);
      if (c < cols) {
        xn[i] = XS::load(x, xe, base, ebase, c);
        gn[i] = load_if<T, STREAM>(dy + base + c);
        if constexpr (RES) rn[i] = load_if<T, STREAM>(dres + base + c);
      }
    }
  };
  int par = 0;
  if constexpr (PF) load_row(static_cast<int64_t>(blockIdx.x) * RPB + rsub);
  for (int64_t step0 = static_cast<int64_t>(blockIdx.x) * RPB; step0 < rows;
       step0 += stride, par ^= 1) {
    const int64_t row = step0 + rsub;
    const bool valid = row < rows;  // uniform per wave
    const int64_t base = row * cols;
    if constexpr (!PF) load_row(row);
    XRaw xr[NVW];
    Raw gr[NVW];
    [[maybe_unused]] Raw rr[NVW];
#pragma unroll
    for (int i = 0; i < NVW; ++i) {
      xr[i] = xn[i];
      gr[i] = gn[i];
      if constexpr (RES) rr[i] = rn[i];
    }
    if constexpr (PF) load_row(row + stride);
    float r;
    if constexpr (HAVE_RSTD) {
      r = valid ? rstd[row] : 0.f;
    } else {
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < NVW; ++i) {
        if (valid && col(i) < cols) {
          float xv[8];
          XS::unpack(xr[i], xv);
#pragma unroll
          for (int j = 0; j < 8; ++j) ss = fmaf(xv[j], xv[j], ss);
        }
      }
      ss = wave_sum(ss);
      if constexpr (WPR > 1) {
        if (lane == 0) red[par][0][wave] = ss;
        __syncthreads();
        ss = 0.f;
#pragma unroll
        for (int s = 0; s < WPR; ++s) ss += red[par][0][rsub * WPR + s];
      }
      r = rsqrtf(ss * inv_cols + eps);
    }
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < NVW; ++i) {
      if (valid && col(i) < cols) {
        float wv[8], xv[8], gv[8];
        Elem<T>::unpack(wr[i], wv);
        XS::unpack(xr[i], xv);
        Elem<T>::unpack(gr[i], gv);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float n = xv[j] * r;
          dot = fmaf(rnd_if<T, RND>(gv[j] * wv[j]), n, dot);
          acc[i][j] = fmaf(gv[j], rnd_if<T, RND>(n), acc[i][j]);
        }
      }
    }
    dot = wave_sum(dot);
    if constexpr (WPR > 1) {
      if (lane == 0) red[par][1][wave] = dot;
      __syncthreads();
      dot = 0.f;
#pragma unroll
      for (int s = 0; s < WPR; ++s) dot += red[par][1][rsub * WPR + s];
    }
    dot *= inv_cols;
#pragma unroll
    for (int i = 0; i < NVW; ++i) {
      const int c = col(i);
      if (valid && c < cols) {
        float wv[8], xv[8], gv[8], o[8];
        Elem<T>::unpack(wr[i], wv);
        XS::unpack(xr[i], xv);
        Elem<T>::unpack(gr[i], gv);
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] = r * (rnd_if<T, RND>(gv[j] * wv[j]) - xv[j] * r * dot);
        if constexpr (RES) {
          float rv[8];
          Elem<T>::unpack(rr[i], rv);
#pragma unroll
          for (int j = 0; j < 8; ++j) o[j] += rv[j];
        }
        Elem<T>::store8(dx + base + c, o);
      }
    }
  }

  // Fixed-order combination of the per-wave partials (waves with the same
  // slice cover the same columns; row groups rsub = 0, 1, ... in order).
  for (int s = 0; s < RPB; ++s) {
    if (rsub == s) {
#pragma unroll
      for (int i = 0; i < NVW; ++i) {
        const int c = col(i);
        if (c < cols) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            if (s == 0) lds_acc[c + j] = acc[i][j];
            else lds_acc[c + j] += acc[i][j];
          }
        }
      }
    }
    __syncthreads();
  }
  float* dst = part + static_cast<int64_t>(blockIdx.x) * cols;
  for (int c = threadIdx.x; c < cols; c += blockDim.x) dst[c] = lds_acc[c];
}

// dw[c] = sum_p part[p, c] (fh_parts.hpp).
template <typename T>
__global__ __launch_bounds__(256) void k_reduce_parts(const float* __restrict__ part, int nparts,
                                                      int cols, T* __restrict__ out) {
  const float t = sum_parts(part, cols, nparts, cols);
  const int c = blockIdx.x * 16 + static_cast<int>(threadIdx.x);
  if (threadIdx.x < 16 && c < cols) Elem<T>::st1(out + c, t);
}

template <typename T>
__global__ __launch_bounds__(256) void k_fill_zero(T* __restrict__ out, int n) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i < n) Elem<T>::st1(out + i, 0.f);
}

// Backward grid cap: fewer blocks mean fewer fp32 dw partial rows to reduce;
// 512 measured best at T=16384, H=2048 (256 and 1024 both slower).
#ifndef FH_NORM_BWD_BLOCKS
#define FH_NORM_BWD_BLOCKS 512
#endif
constexpr int kMaxBwdBlocks = FH_NORM_BWD_BLOCKS;

// Grid cap of the pipelined add+RMSNorm forward (768 measured best of 512,
// 768, 1024 and 2048 at T = 16384, H = 2048).
constexpr int64_t kFwdPipeBlocks = 768;
// Grid cap of the pipelined one-input forward (2049-4096 bf16 columns).
constexpr int64_t kFwdPipeBlocks1 = 512;
// Grid cap of the pipelined forward of a packed x (1025-2048 bf16 columns).
constexpr int64_t kFwdPipeBlocks8 = 1024;

// codes, exps: the kept x that is read (XS = Rows8; x is then null) or written (PACK).
template <typename T, typename XS, int PACK, int NV, bool RND = true>
void launch_fwd(const void* x, const void* a, const void* w, void* h, void* y, float* rstd, const void* codes,
                const uint8_t* exps, int64_t rows, int cols, float eps, hipStream_t s) {
  using Item = typename XS::Item;
  constexpr int kRaw = sizeof(typename Elem<T>::Raw);
  constexpr bool kBf16 = kRaw == 16;
  // A call that does not promise fh_rmsnorm_fwd's bits (its order of a row's sum)
  // gives a wave at most 4096 bf16 or 2048 fp32 columns.  One and more waves a row,
  // us: 8192 x 8192 bf16, packed x 65.1 and 35.5, its add + norm 117 and 92, packing
  // 71.7 and 66.8; 4096 x 8192 25.2 and 18.9, 48.9 and 41.3, 37.7 and 34.0; fp32 8192
  // x 4096 34.1 and 28.5, 105 and 89, 56.8 and 51.6.
  constexpr int WPR = !RND && NV * kRaw > 128 ? NV * kRaw / 128 : 1, NVW = NV / WPR;
  constexpr int kRows = kWavesPerBlock / WPR;
  const int64_t need = (rows + kRows - 1) / kRows;
  const Item* const xp = static_cast<const Item*>(XS::kPacked ? codes : x);
  auto* const co = const_cast<uint8_t*>(static_cast<const uint8_t*>(codes));
  auto* const eo = const_cast<uint8_t*>(exps);
  auto go = [&](auto add, auto pipe, int64_t blocks) {
    if constexpr (PACK == kNoPack || !add())
      hipLaunchKernelGGL((k_rmsnorm_fwd<T, XS, NVW, WPR, add(), pipe(), PACK, RND>), dim3(static_cast<unsigned>(blocks)),
                         dim3(256), 0, s, xp, static_cast<const T*>(a), static_cast<const T*>(w), static_cast<T*>(h),
                         static_cast<T*>(y), rstd, rows, cols, eps, exps, co, eo);
  };
  constexpr std::true_type yes{};
  constexpr std::false_type no{};
  if (a != nullptr) {
    // add+RMSNorm: pipelined over a capped grid where the two rows of x and a
    // in flight fit the registers (bf16 up to 4096 columns, fp32 up to 2048)
    constexpr bool kPipe = NVW * kRaw <= 128;
    go(yes, std::bool_constant<kPipe>{}, kPipe && need > kFwdPipeBlocks ? kFwdPipeBlocks : need);
    return;
  }
  // One input, pipelined over a capped grid: 2049-4096 bf16 columns (kernel time
  // 15.3 -> 14.1 us at T = 4096, 26.1 -> 23.7 us at 8192, H = 4096) and rows that waves
  // share; of a packed x also 1025-2048 bf16 columns (19.2 -> 17.1 us at T = 16384,
  // H = 2048: half the loads of a bf16 row in flight a wave; at 1024 columns no gain).
  constexpr int64_t kCap = XS::kPacked && NV == 4 && kBf16          ? kFwdPipeBlocks8
                           : (NVW == 8 && kBf16) || WPR > 1         ? kFwdPipeBlocks1
                                                                    : 0;
  if constexpr (kCap > 0) {
    if (need > kCap) {
      go(no, yes, kCap);
      return;
    }
  }
  go(no, no, need);
}

// Backward row split: WPR waves per row, NVW chunks of 8 per lane, NWB waves
// per block (RPB = NWB / WPR rows per block step), PF: next-row prefetch.
// Rows of 1025-2048 columns with the residual gradient (the layer's two
// norms) take two waves each in blocks of 8: twice the waves in flight at the
// same partial-row count, 60 -> 56 us at T = 16384, H = 2048 (one wave per
// row in blocks of 8 or 16 needs more than the 128 registers of four waves
// per SIMD).  Rows of 2049-4096 columns with the residual gradient take four
// waves each, with the next row prefetched: kernel time 37.7 -> 33.7 us at
// T = 4096, 60.1 -> 53.8 us at 8192, 206.9 -> 191.6 us at 32768 (H = 4096).
template <int NV, bool RES>
struct BwdSplit {
  static constexpr bool kWide = NV == 8 && RES;
  static constexpr int WPR = kWide ? 4 : NV > 4 || (NV == 4 && RES) ? 2 : 1;
  static constexpr int NVW = NV / WPR;
  static constexpr int NWB = kWide || (NV == 4 && RES) ? 8 : 4;
  static constexpr int RPB = NWB / WPR;
  static constexpr bool PF = !RES || kWide, STREAM = false;
  static constexpr int kBlocks = kMaxBwdBlocks;
};

// The split of a backward of a packed x that does not have to give
// fh_rmsnorm_bwd's bits (RND false): two chunks a lane whatever the width, the next
// row prefetched, one block of 8 waves a CU (256 partial rows), non-temporal loads.
// Kernel and reduction against BwdSplit's, without and with the residual gradient:
// 16384 x 2048 34.6 and 42.5 us against 36.0 and 44.9, 8192 x 4096 33.7 and 42.4
// against 36.5 and 45.4, 4096 x 8192 35.3 and 43.6 against 57.8 and 94.8.  Without
// the prefetch 43.7 and 51.2 (16384 x 2048), 512 blocks 34.3 and 45.6, four chunks a
// lane 36.5 and 45.5.
template <int NV, bool RES>
struct Bwd8Split {
  static constexpr int NVW = NV < 2 ? NV : 2;
  static constexpr int WPR = NV / NVW;
  static constexpr int NWB = 8;
  static constexpr int RPB = NWB / WPR;
  static constexpr bool PF = true, STREAM = true;
  static constexpr int kBlocks = 256;
};

// Blocks of the backward: one per RPB rows, at most `most` (each writes one fp32
// partial row of dw).
inline int bwd_blocks(int64_t rows, int rpb, int most) {
  const int64_t need = (rows + rpb - 1) / rpb;
  return static_cast<int>(need < most ? need : most);
}

template <typename T, typename XS, typename SP, bool RES, bool HR, bool RND>
void launch_bwd_k(const void* dy, const void* x, const uint8_t* xe, const void* w, const float* rstd,
                  const void* dres, void* dx, float* part, int64_t rows, int cols, float eps,
                  int blocks, hipStream_t s) {
  hipLaunchKernelGGL((k_rmsnorm_bwd<T, XS, SP::NVW, SP::WPR, SP::NWB, RES, HR, SP::PF, RND, SP::STREAM>), dim3(blocks),
                     dim3(64 * SP::NWB), static_cast<size_t>(cols) * sizeof(float), s, static_cast<const T*>(dy),
                     static_cast<const typename XS::Item*>(x), static_cast<const T*>(w), rstd,
                     static_cast<const T*>(dres), static_cast<T*>(dx), part, rows, cols, eps, xe);
}

template <typename T, typename XS, int NV, bool RND = true>
void launch_bwd(const void* dy, const void* x, const uint8_t* xe, const void* w, const float* rstd,
                const void* dres, void* dx, void* dw, float* part, int64_t rows, int cols,
                float eps, hipStream_t s) {
  auto go = [&](auto res) {
    // The rows' sums are added in the split's order: where a call promises
    // fh_rmsnorm_bwd's bits it takes fh_rmsnorm_bwd's split.  So do fp32 rows of up to
    // 2048 columns (with the residual gradient 42.6 us against 44.5 at 8192 x 2048;
    // 89.2 against 78.1 at 8192 x 4096).
    constexpr bool kStock = RND || (NV <= 4 && sizeof(typename Elem<T>::Raw) > 16);
    using SP = std::conditional_t<kStock, BwdSplit<NV, res()>, Bwd8Split<NV, res()>>;
    const int blocks = bwd_blocks(rows, SP::RPB, SP::kBlocks);
    if (rstd != nullptr) launch_bwd_k<T, XS, SP, res(), true, RND>(dy, x, xe, w, rstd, dres, dx, part, rows, cols, eps, blocks, s);
    else launch_bwd_k<T, XS, SP, res(), false, RND>(dy, x, xe, w, rstd, dres, dx, part, rows, cols, eps, blocks, s);
    hipLaunchKernelGGL((k_reduce_parts<T>), dim3((cols + 15) / 16), dim3(256), 0, s, part, blocks, cols,
                       static_cast<T*>(dw));
  };
  if (dres != nullptr) go(std::true_type{});
  else go(std::false_type{});
}

// Chunks of 8 per lane: cols <= 512*NV.
template <typename F>
int dispatch_nv(int cols, F&& f) {
  if (cols <= 512) return f(std::integral_constant<int, 1>{});
  if (cols <= 1024) return f(std::integral_constant<int, 2>{});
  if (cols <= 2048) return f(std::integral_constant<int, 4>{});
  if (cols <= 4096) return f(std::integral_constant<int, 8>{});
  return f(std::integral_constant<int, 16>{});
}

int validate_rows(fh_dtype dt, int64_t rows, int64_t cols) {
  FH_REQUIRE(dt == FH_BF16 || dt == FH_F32, "rmsnorm: dtype must be FH_BF16 or FH_F32");
  FH_REQUIRE(rows >= 0, "rmsnorm: rows must be >= 0");
  FH_REQUIRE(cols > 0 && cols % 8 == 0 && cols <= 8192,
             "rmsnorm: cols must be a positive multiple of 8 and <= 8192");
  return FH_OK;
}

}  // namespace
}  // namespace fh
