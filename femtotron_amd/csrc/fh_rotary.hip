// Rotary positions from positions and frequencies: q and k heads turned by the
// angle position * inv_freq[i], pair i of the rotated part of each head being
//   half layout         dims (off + i, off + n + i)
//   interleaved layout  dims (off + 2i, off + 2i + 1)        (i < n = rot_dim / 2)
//   o0 = x0 c - x1 s,  o1 = x1 c + x0 s,  c = factor cos, s = factor sin;
// dims outside the rotated part pass.  The backward turns back: s -> -s.
//
// Angles are fp64 up to the turn's remainder: at position 2^20 an fp32 angle is
// off by 2^-5 of a radian, and bf16 tables (fh_rope_fwd's) hold cos to 2^-9.  The
// remainder goes to [-pi/4, pi/4] in fp64 and to fp32 there, where Taylor's
// polynomials of sin (to x^9) and cos (to x^10) are off by less than 2^-27.
//
// HBM-bound: q and k are read and written once and the angles, n a token, are
// computed by each block once into LDS for all its heads (1/80 to 1/20 of the
// elements), so no table is read.
#include "femtohip_blocks.h"
#include "fh_common.hpp"

namespace fh {
namespace {

// V consecutive elements between memory and fp32 registers in one access
// (fp32 of 8: two).
template <typename T, int V>
struct Vec {
  __device__ __forceinline__ static void load(const T* p, float v[V]) {
    if constexpr (V == 8) {
      Elem<T>::load8(p, v);
    } else if constexpr (V == 4 && sizeof(T) == 2) {
      const uint2 q = *reinterpret_cast<const uint2*>(p);
      v[0] = __uint_as_float(q.x << 16);
      v[1] = __uint_as_float(q.x & 0xffff0000u);
      v[2] = __uint_as_float(q.y << 16);
      v[3] = __uint_as_float(q.y & 0xffff0000u);
    } else if constexpr (V == 4) {
      const float4 q = *reinterpret_cast<const float4*>(p);
      v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
    } else {
      v[0] = Elem<T>::ld1(p);
    }
  }
  __device__ __forceinline__ static void store(T* p, const float v[V]) {
    if constexpr (V == 8) {
      Elem<T>::store8(p, v);
    } else if constexpr (V == 4 && sizeof(T) == 2) {
      *reinterpret_cast<uint2*>(p) = make_uint2(pk_bf16(v[0], v[1]), pk_bf16(v[2], v[3]));
    } else if constexpr (V == 4) {
      *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
      Elem<T>::st1(p, v[0]);
    }
  }
};

// sin and cos of p * f, p a position.
__device__ __forceinline__ void sincos_of(int64_t p, double f, float& s, float& c) {
  const double t = static_cast<double>(p) * f * 0.15915494309189533577;  // turns (1 / 2 pi)
  const double r = t - rint(t);                                           // in [-1/2, 1/2]
  const double k = rint(4.0 * r);
  const float x = static_cast<float>((r - 0.25 * k) * 6.28318530717958647693);  // in [-pi/4, pi/4]
  const float x2 = x * x;
  const float sx = x + x * x2 * fmaf(x2, fmaf(x2, fmaf(x2, 1.f / 362880, -1.f / 5040), 1.f / 120), -1.f / 6);
  const float cx = fmaf(x2, fmaf(x2, fmaf(x2, fmaf(x2, fmaf(x2, -1.f / 3628800, 1.f / 40320), -1.f / 720), 1.f / 24), -0.5f), 1.f);
  const int q = static_cast<int>(k) & 3;  // quarter turns
  const float a = q & 1 ? cx : sx, b = q & 1 ? sx : cx;
  s = q & 2 ? -a : a;
  c = (q == 1 || q == 2) ? -b : b;
}

struct RotaryArgs {
  const void* q;
  const void* k;
  void* qo;
  void* ko;
  int64_t ldq, ldk, ldqo, ldko;  // row strides in elements
  const int64_t* pos;
  const double* inv_freq;
  int64_t tokens, npos;
  float factor;
  int nq, heads, head_dim, n, off;  // heads: q's and k's; n = rot_dim / 2
  int rot_items, items, tpb;        // items a head (the first rot_items turn), tokens a block
  int inplace;
  FastDiv per_head, per_token;
};

constexpr int kItemsPerBlock = 1024;
constexpr int kMaxPairs = 2048;  // angles of a block, 16 KB

// An item is V pairs of one head of one token, or 2V of its passing elements.
// blockIdx.x: tokens tpb at a time; blockIdx.y: kItemsPerBlock of their items.
template <typename T, int V, bool INTER, bool BWD>
__global__ __launch_bounds__(256) void k_rotary(RotaryArgs p) {
  __shared__ __align__(16) float cs[kMaxPairs], sn[kMaxPairs];
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * p.tpb;
  const int nt = static_cast<int>(min(static_cast<int64_t>(p.tpb), p.tokens - t0));
  for (int i = threadIdx.x; i < nt * p.n; i += 256) {
    const int tt = i / p.n;
    const int64_t t = t0 + tt;
    float s, c;
    sincos_of(p.pos[t < p.npos ? t : t % p.npos], p.inv_freq[i - tt * p.n], s, c);
    cs[i] = c * p.factor;
    sn[i] = BWD ? -s * p.factor : s * p.factor;
  }
  __syncthreads();
  const int all = nt * p.heads * p.items;
  const int end = min(all, static_cast<int>(blockIdx.y + 1) * kItemsPerBlock);
  for (int i = blockIdx.y * kItemsPerBlock + threadIdx.x; i < end; i += 256) {
    const int tt = static_cast<int>(p.per_token.div(i));
    const int in_token = i - tt * p.heads * p.items;
    const int head = static_cast<int>(p.per_head.div(in_token));
    const int item = in_token - head * p.items;
    const bool is_q = head < p.nq;
    const int64_t t = t0 + tt;
    const int hd = (is_q ? head : head - p.nq) * p.head_dim;
    const T* src = static_cast<const T*>(is_q ? p.q : p.k) + t * (is_q ? p.ldq : p.ldk) + hd;
    T* dst = static_cast<T*>(is_q ? p.qo : p.ko) + t * (is_q ? p.ldqo : p.ldko) + hd;
    if (item < p.rot_items) {
      const int d0 = p.off + (INTER ? 2 : 1) * item * V, d1 = INTER ? d0 + V : d0 + p.n;
      float u[2 * V], o[2 * V];
      Vec<T, V>::load(src + d0, u);
      Vec<T, V>::load(src + d1, u + V);
      const float* cb = cs + tt * p.n + item * V;
      const float* sb = sn + tt * p.n + item * V;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int a = INTER ? 2 * j : j, b = INTER ? 2 * j + 1 : j + V;
        o[a] = u[a] * cb[j] - u[b] * sb[j];
        o[b] = u[b] * cb[j] + u[a] * sb[j];
      }
      Vec<T, V>::store(dst + d0, o);
      Vec<T, V>::store(dst + d1, o + V);
    } else {
      const int pass = p.head_dim - 2 * p.n;
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        int d = (2 * (item - p.rot_items) + m) * V;
        if (d >= pass) break;
        if (d >= p.off) d += 2 * p.n;
        float u[V];
        Vec<T, V>::load(src + d, u);
        Vec<T, V>::store(dst + d, u);
      }
    }
  }
}

template <bool BWD>
int rotary_impl(fh_dtype dt, const void* q, int64_t ldq, int64_t n_q, const void* k, int64_t ldk, int64_t n_k, void* qo,
                int64_t ldqo, void* ko, int64_t ldko, int64_t tokens, int64_t head_dim, int64_t rot_dim,
                int64_t offset, fh_rotary_layout layout, const int64_t* positions, int64_t n_positions,
                const double* inv_freq, float factor, hipStream_t s) {
  FH_REQUIRE(dt == FH_BF16 || dt == FH_F32, "rotary: dtype must be FH_BF16 or FH_F32");
  FH_REQUIRE(layout == FH_ROTARY_HALF || layout == FH_ROTARY_INTERLEAVED,
             "rotary: layout must be FH_ROTARY_HALF or FH_ROTARY_INTERLEAVED");
  FH_REQUIRE(tokens >= 0 && tokens < (int64_t(1) << 24) * 256, "rotary: tokens must be >= 0 and < 2^32");
  FH_REQUIRE(n_q >= 0 && n_k >= 0, "rotary: negative number of heads");
  FH_REQUIRE(head_dim > 0 && head_dim <= 1024, "rotary: head_dim must be 1 to 1024");
  FH_REQUIRE(rot_dim > 0 && rot_dim % 2 == 0 && offset >= 0 && offset + rot_dim <= head_dim,
             "rotary: rot_dim must be even and positive, and offset + rot_dim within the head");
  FH_REQUIRE((n_q + n_k) * head_dim <= (int64_t(1) << 20), "rotary: (n_q + n_k) * head_dim must be <= 2^20");
  FH_REQUIRE(ldq >= n_q * head_dim && ldqo >= n_q * head_dim && ldk >= n_k * head_dim && ldko >= n_k * head_dim,
             "rotary: a row stride is smaller than its heads");
  if (tokens == 0 || n_q + n_k == 0) return FH_OK;
  FH_REQUIRE((n_q == 0 || (q && qo)) && (n_k == 0 || (k && ko)) && positions && inv_freq, "rotary: null pointer");
  FH_REQUIRE(n_positions > 0 && tokens % n_positions == 0, "rotary: tokens must be a multiple of n_positions");
  const size_t size = dt == FH_BF16 ? 2 : 4;
  FH_REQUIRE((!n_q || q != qo || ldq == ldqo) && (!n_k || k != ko || ldk == ldko),
             "rotary: in place, input and output share their row stride");
  RotaryArgs p{};
  p.inplace = (n_q == 0 || q == qo) && (n_k == 0 || k == ko);
  // Accesses of 8 elements where every part of a head is whole in them and every
  // row aligned, else of 4, else single ones.
  const int64_t n = rot_dim / 2;
  auto fits = [&](int64_t v) {
    auto ok = [&](const void* ptr, int64_t ld) {
      return reinterpret_cast<uintptr_t>(ptr) % (v * size < 16 ? v * size : 16) == 0 && ld % v == 0;
    };
    return n % v == 0 && offset % v == 0 && head_dim % v == 0 && (!n_q || (ok(q, ldq) && ok(qo, ldqo))) &&
           (!n_k || (ok(k, ldk) && ok(ko, ldko)));
  };
  const int v = fits(8) ? 8 : fits(4) ? 4 : 1;
  FH_REQUIRE(reinterpret_cast<uintptr_t>(q) % size == 0 && reinterpret_cast<uintptr_t>(k) % size == 0 &&
                 reinterpret_cast<uintptr_t>(qo) % size == 0 && reinterpret_cast<uintptr_t>(ko) % size == 0,
             "rotary: pointers must be aligned to their elements");
  p.q = q; p.k = k; p.qo = qo; p.ko = ko;
  p.ldq = ldq; p.ldk = ldk; p.ldqo = ldqo; p.ldko = ldko;
  p.pos = positions;
  p.inv_freq = inv_freq;
  p.tokens = tokens;
  p.npos = n_positions;
  p.factor = factor;
  p.nq = static_cast<int>(n_q);
  p.heads = static_cast<int>(n_q + n_k);
  p.head_dim = static_cast<int>(head_dim);
  p.n = static_cast<int>(n);
  p.off = static_cast<int>(offset);
  p.rot_items = static_cast<int>(n) / v;
  const int64_t pass = p.inplace ? 0 : head_dim - rot_dim;
  p.items = p.rot_items + static_cast<int>((pass + 2 * v - 1) / (2 * v));
  const int per_token = p.heads * p.items;
  p.per_head = FastDiv(static_cast<uint32_t>(p.items));
  p.per_token = FastDiv(static_cast<uint32_t>(per_token));
  int64_t tpb = kItemsPerBlock / per_token;
  if (tpb * n > kMaxPairs) tpb = kMaxPairs / n;
  p.tpb = static_cast<int>(tpb < 1 ? 1 : tpb > tokens ? tokens : tpb);
  const int64_t gx = (tokens + p.tpb - 1) / p.tpb;
  const int64_t gy = (static_cast<int64_t>(p.tpb) * per_token + kItemsPerBlock - 1) / kItemsPerBlock;
  FH_REQUIRE(gx < (int64_t(1) << 24), "rotary: too many tokens for one call");  // fewer than 2^32 threads
  const dim3 grid(static_cast<unsigned>(gx), static_cast<unsigned>(gy));
  auto go = [&](auto tag, auto vec) {
    using T = decltype(tag);
    if (layout == FH_ROTARY_HALF) hipLaunchKernelGGL((k_rotary<T, vec(), false, BWD>), grid, dim3(256), 0, s, p);
    else hipLaunchKernelGGL((k_rotary<T, vec(), true, BWD>), grid, dim3(256), 0, s, p);
  };
  auto by_vec = [&](auto tag) {
    if (v == 8) go(tag, std::integral_constant<int, 8>{});
    else if (v == 4) go(tag, std::integral_constant<int, 4>{});
    else go(tag, std::integral_constant<int, 1>{});
  };
  if (dt == FH_BF16) by_vec(uint16_t{});
  else by_vec(float{});
  return check_launch(BWD ? "fh_rotary_bwd" : "fh_rotary_fwd");
}

}  // namespace
}  // namespace fh

using namespace fh;

extern "C" int fh_rotary_fwd(fh_dtype dt, const void* q, int64_t ldq, int64_t n_q, const void* k, int64_t ldk,
                             int64_t n_k, void* q_out, int64_t ldqo, void* k_out, int64_t ldko, int64_t tokens,
                             int64_t head_dim, int64_t rot_dim, int64_t offset, fh_rotary_layout layout,
                             const int64_t* positions, int64_t n_positions, const double* inv_freq, float factor,
                             hipStream_t stream) {
  return rotary_impl<false>(dt, q, ldq, n_q, k, ldk, n_k, q_out, ldqo, k_out, ldko, tokens, head_dim, rot_dim, offset,
                            layout, positions, n_positions, inv_freq, factor, stream);
}

extern "C" int fh_rotary_bwd(fh_dtype dt, const void* dq, int64_t lddq, int64_t n_q, const void* dk, int64_t lddk,
                             int64_t n_k, void* dq_out, int64_t lddqo, void* dk_out, int64_t lddko, int64_t tokens,
                             int64_t head_dim, int64_t rot_dim, int64_t offset, fh_rotary_layout layout,
                             const int64_t* positions, int64_t n_positions, const double* inv_freq, float factor,
                             hipStream_t stream) {
  return rotary_impl<true>(dt, dq, lddq, n_q, dk, lddk, n_k, dq_out, lddqo, dk_out, lddko, tokens, head_dim, rot_dim,
                           offset, layout, positions, n_positions, inv_freq, factor, stream);
}
