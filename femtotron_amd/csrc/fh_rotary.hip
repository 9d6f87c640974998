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
// HBM-bound: q and k are read and written once.  The angles, n a token, are
// computed by each block into LDS for the heads it has of a token, so no table is
// read.  bf16, us a launch: 16384 tokens of 36 heads of 64 28 (151 MB, 5.4 TB/s),
// 32768 tokens of 64 heads of 128, half of each turned, 182-185 (1074 MB, 5.8-5.9).
// fp32: 16384 tokens of 36 heads of 64 67 (302 MB, 4.5), of what was just written 51
// (5.9); 8192 tokens of 40 heads of 128 69 and 57 (336 MB, 4.9 and 5.9).
#include "femtohip_blocks.h"
#include "fh_common.hpp"

namespace fh {
namespace {

// V consecutive elements, moved in one access (fp32 of 8: two) and kept as loaded.
template <typename T, int V>
struct Vec;

template <typename T>
struct Vec<T, 8> {
  using Raw = typename Elem<T>::Raw;
  __device__ __forceinline__ static Raw load(const T* p) { return Elem<T>::ldraw(p); }
  __device__ __forceinline__ static void store(T* p, const Raw& q) { Elem<T>::straw(p, q); }
  __device__ __forceinline__ static void unpack(const Raw& q, float* v) { Elem<T>::unpack(q, v); }
  __device__ __forceinline__ static Raw pack(const float* v) { return Elem<T>::pack(v); }
};

template <>
struct Vec<uint16_t, 4> {
  using Raw = uint2;
  __device__ __forceinline__ static Raw load(const uint16_t* p) { return *reinterpret_cast<const uint2*>(p); }
  __device__ __forceinline__ static void store(uint16_t* p, const Raw& q) { *reinterpret_cast<uint2*>(p) = q; }
  __device__ __forceinline__ static void unpack(const Raw& q, float* v) {
    v[0] = __uint_as_float(q.x << 16);
    v[1] = __uint_as_float(q.x & 0xffff0000u);
    v[2] = __uint_as_float(q.y << 16);
    v[3] = __uint_as_float(q.y & 0xffff0000u);
  }
  __device__ __forceinline__ static Raw pack(const float* v) {
    return make_uint2(pk_bf16(v[0], v[1]), pk_bf16(v[2], v[3]));
  }
};

template <>
struct Vec<float, 4> {
  using Raw = float4;
  __device__ __forceinline__ static Raw load(const float* p) { return *reinterpret_cast<const float4*>(p); }
  __device__ __forceinline__ static void store(float* p, const Raw& q) { *reinterpret_cast<float4*>(p) = q; }
  __device__ __forceinline__ static void unpack(const Raw& q, float* v) {
    v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
  }
  __device__ __forceinline__ static Raw pack(const float* v) { return make_float4(v[0], v[1], v[2], v[3]); }
};

template <typename T>
struct Vec<T, 1> {
  using Raw = T;
  __device__ __forceinline__ static Raw load(const T* p) { return *p; }
  __device__ __forceinline__ static void store(T* p, const Raw& q) { *p = q; }
  __device__ __forceinline__ static void unpack(const Raw& q, float* v) { v[0] = Elem<T>::ld1(&q); }
  __device__ __forceinline__ static Raw pack(const float* v) {
    Raw q;
    Elem<T>::st1(&q, v[0]);
    return q;
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
  float factor;
  uint32_t total;                         // items of the call
  int nq, head_dim, n, off;               // n = rot_dim / 2
  int rot_items, items;                   // items a head (the first rot_items turn)
  FastDiv per_head, per_token;            // items of a head and of a token
  FastDiv pairs, positions;               // n, and the number of positions
};

// Angles of a block: 256 items touch whole tokens and two cut ones at most, so at
// most 254 V + rot_dim pairs.  Six blocks fit a CU; eight, with as much as a call
// needs, measured slower (32768 tokens of 64 heads of 128 373 us against 366).
constexpr int kMaxPairs = 254 * 8 + 1024;

// An item is V pairs of one head of one token, or 2V of its passing elements: two
// accesses of V elements each way.  A thread has one, of the call's items token by
// token, and has its loads under way before the block computes the angles of the
// tokens it touches.  Measured otherwise, forward and backward, 16384 tokens of 36
// heads of 64 and 32768 of 64 heads of 128, half of each turned: this 56 and 366 us;
// blocks of whole tokens 55 and 388; those with two, four and eight items a thread
// 60, 63 and 69, and (with eight) 413; with four, the loads behind the angles, 86
// and 537.
template <typename T, int V, bool INTER, bool BWD>
__global__ __launch_bounds__(256) void k_rotary(RotaryArgs p) {
  __shared__ __align__(16) float cs[kMaxPairs], sn[kMaxPairs];
  const uint32_t base = blockIdx.x * 256u, last = min(base + 255u, p.total - 1);
  const uint32_t t0 = p.per_token.div(base), nt = p.per_token.div(last) - t0 + 1;
  const uint32_t i = base + threadIdx.x;
  const bool mine = i <= last;
  typename Vec<T, V>::Raw u, v;
  T *du = nullptr, *dv = nullptr;
  int angle = -1;  // where the item's angles start; -1: it passes
  if (mine) {
    const uint32_t t = p.per_token.div(i);
    const int in_token = static_cast<int>(i - t * p.per_token.d);
    const int head = static_cast<int>(p.per_head.div(in_token));
    const int item = in_token - head * p.items;
    const bool is_q = head < p.nq;
    const int hd = (is_q ? head : head - p.nq) * p.head_dim;
    int d0, d1;
    if (item < p.rot_items) {
      d0 = p.off + (INTER ? 2 : 1) * item * V;
      d1 = INTER ? d0 + V : d0 + p.n;
      angle = static_cast<int>(t - t0) * p.n + item * V;
    } else {
      const int pass = p.head_dim - 2 * p.n;
      d0 = 2 * (item - p.rot_items) * V;
      d1 = d0 + V < pass ? d0 + V : d0;  // an odd last one twice
      if (d0 >= p.off) d0 += 2 * p.n;
      if (d1 >= p.off) d1 += 2 * p.n;
    }
    const int64_t row = t;
    const T* src = static_cast<const T*>(is_q ? p.q : p.k) + row * (is_q ? p.ldq : p.ldk) + hd;
    T* dst = static_cast<T*>(is_q ? p.qo : p.ko) + row * (is_q ? p.ldqo : p.ldko) + hd;
    u = Vec<T, V>::load(src + d0);
    v = Vec<T, V>::load(src + d1);
    du = dst + d0;
    dv = dst + d1;
  }
  for (uint32_t a = threadIdx.x; a < nt * p.n; a += 256) {
    const uint32_t tt = p.pairs.div(a), t = t0 + tt;
    float s, c;
    sincos_of(p.pos[t - p.positions.div(t) * p.positions.d], p.inv_freq[a - tt * p.n], s, c);
    cs[a] = c * p.factor;
    sn[a] = BWD ? -s * p.factor : s * p.factor;
  }
  __syncthreads();
  if (!mine) return;
  if (angle >= 0) {
    float x[2 * V], o[2 * V], c[V], s[V];
    Vec<T, V>::unpack(u, x);
    Vec<T, V>::unpack(v, x + V);
    Vec<float, V>::unpack(Vec<float, V>::load(cs + angle), c);
    Vec<float, V>::unpack(Vec<float, V>::load(sn + angle), s);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int a = INTER ? 2 * j : j, b = INTER ? 2 * j + 1 : j + V;
      o[a] = x[a] * c[j] - x[b] * s[j];
      o[b] = x[b] * c[j] + x[a] * s[j];
    }
    u = Vec<T, V>::pack(o);
    v = Vec<T, V>::pack(o + V);
  }
  Vec<T, V>::store(du, u);
  Vec<T, V>::store(dv, v);
}

template <bool BWD>
int rotary_impl(fh_dtype dt, const void* q, int64_t ldq, int64_t n_q, const void* k, int64_t ldk, int64_t n_k, void* qo,
                int64_t ldqo, void* ko, int64_t ldko, int64_t tokens, int64_t head_dim, int64_t rot_dim,
                int64_t offset, fh_rotary_layout layout, const int64_t* positions, int64_t n_positions,
                const double* inv_freq, float factor, hipStream_t s) {
  FH_REQUIRE(dt == FH_BF16 || dt == FH_F32, "rotary: dtype must be FH_BF16 or FH_F32");
  FH_REQUIRE(layout == FH_ROTARY_HALF || layout == FH_ROTARY_INTERLEAVED,
             "rotary: layout must be FH_ROTARY_HALF or FH_ROTARY_INTERLEAVED");
  FH_REQUIRE(tokens >= 0, "rotary: tokens must be >= 0");
  FH_REQUIRE(n_q >= 0 && n_k >= 0 && n_q <= (1 << 20) && n_k <= (1 << 20),
             "rotary: a number of heads is negative or over 2^20");
  FH_REQUIRE(head_dim > 0 && head_dim <= 1024, "rotary: head_dim must be 1 to 1024");
  FH_REQUIRE(rot_dim > 0 && rot_dim % 2 == 0 && rot_dim <= head_dim && offset >= 0 && offset <= head_dim - rot_dim,
             "rotary: rot_dim must be even and positive, and offset + rot_dim within the head");
  FH_REQUIRE((n_q + n_k) * head_dim <= (int64_t(1) << 20), "rotary: (n_q + n_k) * head_dim must be <= 2^20");
  FH_REQUIRE(ldq >= n_q * head_dim && ldqo >= n_q * head_dim && ldk >= n_k * head_dim && ldko >= n_k * head_dim,
             "rotary: a row stride is smaller than its heads");
  FH_REQUIRE(ldq <= (1 << 28) && ldqo <= (1 << 28) && ldk <= (1 << 28) && ldko <= (1 << 28),
             "rotary: a row stride is over 2^28");
  if (tokens == 0 || n_q + n_k == 0) return FH_OK;
  FH_REQUIRE((n_q == 0 || (q && qo)) && (n_k == 0 || (k && ko)) && positions && inv_freq, "rotary: null pointer");
  FH_REQUIRE(n_positions > 0 && tokens % n_positions == 0, "rotary: tokens must be a multiple of n_positions");
  const size_t size = dt == FH_BF16 ? 2 : 4;
  FH_REQUIRE((!n_q || q != qo || ldq == ldqo) && (!n_k || k != ko || ldk == ldko),
             "rotary: in place, input and output share their row stride");
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
  auto at = [](const void* ptr, size_t bytes) { return reinterpret_cast<uintptr_t>(ptr) % bytes == 0; };
  FH_REQUIRE(at(q, size) && at(k, size) && at(qo, size) && at(ko, size) && at(positions, 8) && at(inv_freq, 8),
             "rotary: pointers must be aligned to their elements");
  const bool inplace = (n_q == 0 || q == qo) && (n_k == 0 || k == ko);  // passing dims stay where they are
  const int64_t pass = inplace ? 0 : head_dim - rot_dim;
  const int64_t items = n / v + (pass + 2 * v - 1) / (2 * v), per_token = (n_q + n_k) * items;
  FH_REQUIRE(tokens <= ((int64_t(1) << 32) - 256) / per_token,
             "rotary: too many elements for one call (2^32 items of 16 elements, or fewer where rows are not aligned)");
  // An output is its input or apart from every operand: by rows of one stride their
  // columns, of different strides their whole extents.
  auto apart = [&](const void* a, int64_t lda, int64_t wa, const void* b, int64_t ldb, int64_t wb) {
    if (wa == 0 || wb == 0) return true;
    const auto pa = reinterpret_cast<intptr_t>(a), pb = reinterpret_cast<intptr_t>(b);
    const auto bytes = [&](int64_t ld, int64_t w) { return static_cast<intptr_t>(((tokens - 1) * ld + w) * static_cast<int64_t>(size)); };
    if (pa + bytes(lda, wa) <= pb || pb + bytes(ldb, wb) <= pa) return true;
    if (lda != ldb || tokens == 1) return false;
    const intptr_t row = static_cast<intptr_t>(lda * static_cast<int64_t>(size));
    const intptr_t d = ((pb - pa) % row + row) % row;  // where b's rows start within a's
    return d >= wa * static_cast<int64_t>(size) && d + wb * static_cast<int64_t>(size) <= row;
  };
  const int64_t wq = n_q * head_dim, wk = n_k * head_dim;
  FH_REQUIRE((qo == q || apart(qo, ldqo, wq, q, ldq, wq)) && (ko == k || apart(ko, ldko, wk, k, ldk, wk)) &&
                 apart(qo, ldqo, wq, k, ldk, wk) && apart(ko, ldko, wk, q, ldq, wq) && apart(qo, ldqo, wq, ko, ldko, wk),
             "rotary: an output overlaps an operand that is not its own input");
  RotaryArgs p{};
  p.q = q; p.k = k; p.qo = qo; p.ko = ko;
  p.ldq = ldq; p.ldk = ldk; p.ldqo = ldqo; p.ldko = ldko;
  p.pos = positions;
  p.inv_freq = inv_freq;
  p.factor = factor;
  p.total = static_cast<uint32_t>(tokens * per_token);
  p.nq = static_cast<int>(n_q);
  p.head_dim = static_cast<int>(head_dim);
  p.n = static_cast<int>(n);
  p.off = static_cast<int>(offset);
  p.rot_items = static_cast<int>(n / v);
  p.items = static_cast<int>(items);
  p.per_head = FastDiv(static_cast<uint32_t>(items));
  p.per_token = FastDiv(static_cast<uint32_t>(per_token));
  p.pairs = FastDiv(static_cast<uint32_t>(n));
  p.positions = FastDiv(static_cast<uint32_t>(n_positions));
  const dim3 grid(static_cast<unsigned>((p.total + 255ll) / 256));
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
