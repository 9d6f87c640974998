// Activations in 8 bits: the storage, its packing and unpacking in registers.
//
// 32 consecutive elements of a row (the last block of a row may be shorter)
// share an exponent E, kept as the byte E + 127; an element is code * 2^E, 8.25
// bits an element.  (The e4m3 bytes are those of the OCP microscaling format
// MXFP8-E4M3.  MXINT8 has the same codes, but counts them in 2^-6: its scale byte
// is this one plus 6.)  With m the block's largest magnitude and e = floor(log2 m):
//   int8:  E = e - 6, code = rint(x 2^-E) with ties to even, at most 127 in
//          magnitude (only a magnitude above 127.5 * 2^E is cut);
//   e4m3:  E = e - 8, one more where m 2^-E would pass 448, the largest e4m3
//          value; code = x 2^-E rounded to e4m3, at E = 120 at most 240 in magnitude
//          (only from 248 * 2^120 on is one cut: 256 * 2^120 is infinite).
// A power of two, and not m / 127: the scaling is then exact in fp32, the codes
// do not depend on how a quotient rounds, and code * 2^E is a value that bf16
// holds, so a kernel that reads codes gives the bits that it gives for the
// unpacked tensor.  What it costs is up to one bit of int8's seven (steps of
// m/127 to m/64); e4m3 has its step in each element's own exponent, and so loses
// none of its bits to it, down to the format's smallest step 2^(E-9): an element
// is off by at most 2^-4 of itself or 2^(E-10), which is under 2^-17 m.  E is at
// least -118: no step is under 2^-118 in int8, 2^-127 in e4m3.  A block with an infinity or a NaN has the byte 255 and
// codes 0 and reads as NaN throughout, so that a bad activation reaches the
// gradients instead of being cut to a finite one.
#pragma once

#include "fh_common.hpp"

namespace fh {

constexpr int kNoPack = -1;
constexpr int kFmtInt8 = 0, kFmtE4M3 = 1;  // FH_INT8, FH_E4M3
constexpr int kBlock8 = 32;
constexpr uint32_t kMinExpByte = 9;    // E = -118
constexpr uint32_t kNanExpByte = 255;
constexpr uint32_t kTopExpByteE4M3 = 247;  // E = 120, e4m3's largest: 256 * 2^E is infinite

__host__ __device__ __forceinline__ int64_t blocks8(int64_t cols) { return (cols + kBlock8 - 1) / kBlock8; }

// 8 codes of a row, and their block's exponent byte.
struct Raw8 {
  uint2 c;
  uint32_t e;
};

// Codes c..c+7 of the row at codes and exps (c % 8 == 0, so within one block); a
// row is a multiple of 8 codes, which keeps them 8-byte aligned.
__device__ __forceinline__ Raw8 load8_codes(const uint8_t* codes, const uint8_t* exps, int c) {
  Raw8 r;
  r.c = *reinterpret_cast<const uint2*>(codes + c);
  r.e = exps[c / kBlock8];
  return r;
}

template <int FMT>
__device__ __forceinline__ void unpack8(const Raw8& q, float v[8]) {
  const float s = __uint_as_float(q.e << 23);  // 2^E; the byte 255 gives infinity, and 0 * infinity NaN
  const uint32_t w[2] = {q.c.x, q.c.y};
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if constexpr (FMT == kFmtInt8) {
#pragma unroll
      for (int j = 0; j < 4; ++j) v[4 * i + j] = static_cast<float>(static_cast<int8_t>(w[i] >> (8 * j))) * s;
    } else {
      const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(w[i], false);
      const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8(w[i], true);
      v[4 * i + 0] = lo[0] * s;
      v[4 * i + 1] = lo[1] * s;
      v[4 * i + 2] = hi[0] * s;
      v[4 * i + 3] = hi[1] * s;
    }
  }
}

template <int CTRL>
__device__ __forceinline__ uint32_t dpp_u32(uint32_t v) {
  return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, 0xf, 0xf, false));
}

// The exponent byte of a block whose lane quad holds 8 elements a lane (all four
// lanes active; one behind the row's end holds zeros).  As bit patterns
// magnitudes order like integers, an infinity above every finite value and a
// NaN above that.
template <int FMT>
__device__ __forceinline__ uint32_t exp_byte(const float v[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(v[j]) & 0x7fffffffu);
  m = max(m, dpp_u32<0xB1>(m));  // quad_perm [1,0,3,2]
  m = max(m, dpp_u32<0x4E>(m));  // quad_perm [2,3,0,1]
  if (m >= 0x7f800000u) return kNanExpByte;
  int b = static_cast<int>(m >> 23);
  if constexpr (FMT == kFmtInt8) b -= 6;
  else b += ((m & 0x7fffffu) > 0x600000u ? 1 : 0) - 8;  // 1.75 * 2^8 = 448
  return static_cast<uint32_t>(max(b, static_cast<int>(kMinExpByte)));
}

// The codes of 8 elements of a block with exponent byte e.
template <int FMT>
__device__ __forceinline__ uint2 codes8(const float v[8], uint32_t e) {
  const float inv = __uint_as_float((254u - e) << 23);  // 2^-E (e is 9 to 248)
  uint32_t w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if constexpr (FMT == kFmtInt8) {
      // Adding 1.5 * 2^23 rounds to a whole number, ties to even, and leaves it
      // in two's complement in the low bits.
      uint32_t u[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        u[j] = __float_as_uint(__builtin_amdgcn_fmed3f(v[4 * i + j] * inv, -127.f, 127.f) + 12582912.f);
      w[i] = __builtin_amdgcn_perm(u[1], u[0], 0x0c0c0400u) | __builtin_amdgcn_perm(u[3], u[2], 0x04000c0cu);
    } else {
      const float most = e == kTopExpByteE4M3 ? 240.f : 448.f;
      float u[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) u[j] = __builtin_amdgcn_fmed3f(v[4 * i + j] * inv, -most, most);
      int t = __builtin_amdgcn_cvt_pk_fp8_f32(u[0], u[1], 0, false);
      t = __builtin_amdgcn_cvt_pk_fp8_f32(u[2], u[3], t, true);
      w[i] = static_cast<uint32_t>(t);
    }
  }
  const bool bad = e == kNanExpByte;
  return make_uint2(bad ? 0u : w[0], bad ? 0u : w[1]);
}

// Packs elements c..c+7 of the row at codes and exps; the four lanes of a quad hold
// one block (lane l of a wave at c = 8 l modulo 512) and all call this, those behind
// the row's end (!in) with zeros, of which nothing is stored.
template <int FMT>
__device__ __forceinline__ void pack8_store(const float v[8], uint8_t* codes, uint8_t* exps, bool in, int c) {
  const uint32_t e = exp_byte<FMT>(v);
  if (!in) return;
  *reinterpret_cast<uint2*>(codes + c) = codes8<FMT>(v, e);
  if ((c & (kBlock8 - 1)) == 0) exps[c / kBlock8] = static_cast<uint8_t>(e);
}

}  // namespace fh
