// The norm of all gradients of a model and their clipping:
//   norm = sqrt(sum g^2),  c = min(1, max_norm / (norm + 1e-6)),  out = c g.
//
// HBM-bound: one pass reads every gradient for the sum, a second reads them again and
// writes.  The tensors' pointers travel in the kernels' arguments (kTensors a launch), so
// there is no table to upload, and a captured call keeps its own copy.  A workgroup takes a
// contiguous run of chunks of kChunkElems elements, across tensors; its sum of squares (in
// fp64: exact products of fp32 values, no overflow below 1e154) is one partial, and every
// workgroup of the second pass folds the at most kPartials partials by itself, in
// one order, which is cheaper than a launch in between.  Within a launch the second pass takes
// the runs from the last to the first: of up to kTensors tensors, what the first pass read last
// is still in the cache.  (More tensors are several launches, the same way round in both
// passes: there the cache holds the end of the last.)  TinyLlama's 1.1e9 gradients, two
// launches, bf16 to fp32: 376 us for the sums (5.9 TB/s) and 1286 for the outputs
// (5.1, a third of it read); 5 + 6 us for a few small layers.
#include <algorithm>
#include <new>
#include <vector>

#include "femtohip_packed.h"
#include "fh_common.hpp"

namespace fh {
namespace {

constexpr int kThreads = 256;
constexpr int kVecs = 4;                                  // of 8 elements, a thread and chunk
constexpr int64_t kChunkElems = kThreads * 8 * kVecs;     // 8192
constexpr int kTensors = 128;                             // a launch: 3.7 KB of arguments
// Workgroups of a launch: four a CU, which all run at once.  (With eight, of which the
// registers let six run, the last two rounds cost as much as three: 164 us a launch of 96
// TinyLlama tensors, 1.0 GB; with a share of them by the launch's elements, a launch of
// nine tensors left half of the chip idle.)
constexpr int64_t kBlocks = 1024;
constexpr int64_t kPartials = 16384;                      // in all; fewer workgroups a launch above 16 of them

// Tensor i's chunks are first[i] .. first[i + 1] of the launch.
struct Table {
  const void* grad[kTensors];
  void* out[kTensors];
  int64_t numel[kTensors];
  uint32_t first[kTensors + 1];
  uint8_t kind[kTensors];  // 1: gradient bf16, 2: out bf16, 4: 16-byte aligned
  int n;
};
static_assert(sizeof(Table) <= 3840, "kernel arguments hold 4 KB");

__device__ __forceinline__ int tensor_of(const Table& t, uint32_t chunk) {
  int lo = 0, hi = t.n;  // the last tensor whose first chunk is at or before `chunk`
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (t.first[mid] <= chunk) lo = mid;
    else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ double block_sum(double v) {
  __shared__ double part[kThreads / kWave];
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, kWave);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  return (part[0] + part[1]) + (part[2] + part[3]);
}

// Eight elements at p, of the row of n left (fewer: element by element), `vec`: in one access.
template <typename T>
__device__ __forceinline__ void load_some(const T* p, int64_t n, bool vec, float (&v)[8]) {
  if (vec && n >= 8) {
    Elem<T>::load8(p, v);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = e < n ? Elem<T>::ld1(p + e) : 0.f;
  }
}

template <typename T>
__device__ __forceinline__ double chunk_squares(const T* g, int64_t left, bool vec) {
  double s = 0.0;
  if (vec && left >= kChunkElems) {
    typename Elem<T>::Raw raw[kVecs];
#pragma unroll
    for (int i = 0; i < kVecs; ++i) raw[i] = Elem<T>::ldraw(g + (i * kThreads + threadIdx.x) * 8);
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      float v[8];
      Elem<T>::unpack(raw[i], v);
#pragma unroll
      for (int e = 0; e < 8; ++e) s = fma(static_cast<double>(v[e]), static_cast<double>(v[e]), s);
    }
  } else {
    for (int i = 0; i < kVecs; ++i) {
      const int64_t at = (i * kThreads + threadIdx.x) * 8;
      if (at >= left) break;
      float v[8];
      load_some(g + at, left - at, vec, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) s = fma(static_cast<double>(v[e]), static_cast<double>(v[e]), s);
    }
  }
  return s;
}

// Run b of `runs` over the launch's chunks: [lo, hi).
__device__ __forceinline__ void run_of(uint32_t chunks, int64_t runs, int64_t b, uint32_t& lo, uint32_t& hi) {
  lo = static_cast<uint32_t>(chunks * b / runs);
  hi = static_cast<uint32_t>(chunks * (b + 1) / runs);
}

__global__ __launch_bounds__(kThreads) void k_grad_squares(Table t, double* __restrict__ partials) {
  uint32_t lo, hi;
  run_of(t.first[t.n], gridDim.x, blockIdx.x, lo, hi);
  double s = 0.0;
  int i = tensor_of(t, lo);
  for (uint32_t c = lo; c < hi; ++c) {
    while (c >= t.first[i + 1]) ++i;
    const int64_t at = static_cast<int64_t>(c - t.first[i]) * kChunkElems, left = t.numel[i] - at;
    const bool vec = t.kind[i] & 4;
    if (t.kind[i] & 1) s += chunk_squares(static_cast<const uint16_t*>(t.grad[i]) + at, left, vec);
    else s += chunk_squares(static_cast<const float*>(t.grad[i]) + at, left, vec);
  }
  s = block_sum(s);
  if (threadIdx.x == 0) partials[blockIdx.x] = s;
}

// N consecutive elements in one access, each of them read and written for the last time here
// (non-temporal).
template <typename T, int N>
struct Pack {
  typedef uint32_t W __attribute__((ext_vector_type(sizeof(T) * N / 4)));
  __device__ __forceinline__ static W load(const T* p) { return __builtin_nontemporal_load(reinterpret_cast<const W*>(p)); }
  __device__ __forceinline__ static void store(T* p, const float (&v)[N]) {
    W w;
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int e = 0; e < N / 2; ++e) w[e] = pk_bf16(v[2 * e], v[2 * e + 1]);
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) w[e] = __float_as_uint(v[e]);
    }
    __builtin_nontemporal_store(w, reinterpret_cast<W*>(p));
  }
  __device__ __forceinline__ static void unpack(const W& w, float (&v)[N]) {
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int e = 0; e < N / 2; ++e) {
        v[2 * e] = __uint_as_float(w[e] << 16);
        v[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
      }
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) v[e] = __uint_as_float(w[e]);
    }
  }
};

template <typename T, typename U>
__device__ __forceinline__ void chunk_scale(const T* g, U* out, int64_t left, bool vec, float f) {
  if (vec && left >= kChunkElems) {
    // A wave's accesses are runs of whole lines on both sides: 16 bytes a lane on the wider.
    constexpr int N = sizeof(T) == 4 || sizeof(U) == 4 ? 4 : 8, I = kChunkElems / (kThreads * N);
    typename Pack<T, N>::W raw[I];
#pragma unroll
    for (int i = 0; i < I; ++i) raw[i] = Pack<T, N>::load(g + (i * kThreads + threadIdx.x) * N);
#pragma unroll
    for (int i = 0; i < I; ++i) {
      float v[N];
      Pack<T, N>::unpack(raw[i], v);
#pragma unroll
      for (int e = 0; e < N; ++e) v[e] *= f;
      Pack<U, N>::store(out + (i * kThreads + threadIdx.x) * N, v);
    }
  } else {
    for (int i = 0; i < kVecs; ++i) {
      const int64_t at = (i * kThreads + threadIdx.x) * 8;
      if (at >= left) break;
      float v[8];
      load_some(g + at, left - at, vec, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] *= f;
      if (vec && left - at >= 8) {
        Elem<U>::store8(out + at, v);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (at + e < left) Elem<U>::st1(out + at + e, v[e]);
      }
    }
  }
}

// The norm from the partials, the same in every workgroup.
__device__ __forceinline__ double fold_norm(const double* __restrict__ partials, int n) {
  double s = 0.0;
  for (int i = threadIdx.x; i < n; i += kThreads) s += partials[i];
  return sqrt(block_sum(s));
}

__global__ __launch_bounds__(kThreads) void k_grad_scale(Table t, const double* __restrict__ partials, int n,
                                                         float max_norm, float* __restrict__ norm, bool tell) {
  const double all = fold_norm(partials, n);
  if (tell && blockIdx.x == 0 && threadIdx.x == 0) *norm = static_cast<float>(all);
  const double c = static_cast<double>(max_norm) / (all + 1e-6);
  const float f = c > 1.0 ? 1.f : static_cast<float>(c);  // NaN stays
  uint32_t lo, hi;
  run_of(t.first[t.n], gridDim.x, gridDim.x - 1 - blockIdx.x, lo, hi);
  int i = tensor_of(t, lo);
  for (uint32_t k = lo; k < hi; ++k) {
    while (k >= t.first[i + 1]) ++i;
    const int64_t at = static_cast<int64_t>(k - t.first[i]) * kChunkElems, left = t.numel[i] - at;
    const int kind = t.kind[i];
    const bool vec = kind & 4;
    if (f == 1.f && t.out[i] == t.grad[i]) continue;  // as it is
    const auto gb = static_cast<const uint16_t*>(t.grad[i]);
    const auto gf = static_cast<const float*>(t.grad[i]);
    const auto ob = static_cast<uint16_t*>(t.out[i]);
    const auto of = static_cast<float*>(t.out[i]);
    if ((kind & 3) == 3) chunk_scale(gb + at, ob + at, left, vec, f);
    else if ((kind & 3) == 1) chunk_scale(gb + at, of + at, left, vec, f);
    else if ((kind & 3) == 2) chunk_scale(gf + at, ob + at, left, vec, f);
    else chunk_scale(gf + at, of + at, left, vec, f);
  }
}

__global__ __launch_bounds__(kThreads) void k_grad_norm(const double* __restrict__ partials, int n,
                                                        float* __restrict__ norm) {
  const double all = fold_norm(partials, n);
  if (threadIdx.x == 0) *norm = static_cast<float>(all);
}

size_t bytes_of(int32_t dt) { return dt == FH_BF16 ? 2 : 4; }

// Whether an output overlaps anything but its own gradient.
bool overlaps(int64_t count, const fh_grad* g) {
  struct Range {
    uintptr_t lo, hi;
    bool out;
  };
  std::vector<Range> r;
  r.reserve(static_cast<size_t>(2 * count));
  for (int64_t i = 0; i < count; ++i) {
    if (g[i].numel == 0) continue;
    const uintptr_t a = reinterpret_cast<uintptr_t>(g[i].grad), b = reinterpret_cast<uintptr_t>(g[i].out);
    const uintptr_t an = a + static_cast<uintptr_t>(g[i].numel) * bytes_of(g[i].grad_dtype);
    const uintptr_t bn = b + static_cast<uintptr_t>(g[i].numel) * bytes_of(g[i].out_dtype);
    if (a != b) r.push_back({a, an, false});
    else if (an != bn) return true;  // in place in another type
    r.push_back({b, bn, true});
  }
  std::sort(r.begin(), r.end(), [](const Range& x, const Range& y) { return x.lo < y.lo; });
  uintptr_t outs = 0, all = 0;  // the furthest ends so far
  for (const Range& x : r) {
    if (x.lo < outs || (x.out && x.lo < all)) return true;
    all = std::max(all, x.hi);
    if (x.out) outs = std::max(outs, x.hi);
  }
  return false;
}

int clip_grads(int64_t count, const fh_grad* grads, float max_norm, float* norm, double* partials, hipStream_t stream) {
  FH_REQUIRE(count >= 0 && count <= (int64_t(1) << 20), "clip_grads: bad count");
  FH_REQUIRE(norm != nullptr && partials != nullptr && (count == 0 || grads != nullptr), "clip_grads: null pointer");
  FH_REQUIRE(aligned16(partials), "clip_grads: workspace must be 16-byte aligned");
  FH_REQUIRE(max_norm >= 0.f, "clip_grads: max_norm must not be negative");
  bool write = false;
  int64_t chunks = 0;
  for (int64_t i = 0; i < count; ++i) {
    const fh_grad& g = grads[i];
    FH_REQUIRE(g.numel >= 0 && g.numel < (int64_t(1) << 44), "clip_grads: bad numel");
    FH_REQUIRE((g.grad_dtype == FH_BF16 || g.grad_dtype == FH_F32) && (g.out_dtype == FH_BF16 || g.out_dtype == FH_F32),
               "clip_grads: dtypes must be FH_BF16 or FH_F32");
    FH_REQUIRE(g.numel == 0 || g.grad != nullptr, "clip_grads: null gradient");
    FH_REQUIRE(reinterpret_cast<uintptr_t>(g.grad) % bytes_of(g.grad_dtype) == 0 &&
                   reinterpret_cast<uintptr_t>(g.out) % bytes_of(g.out_dtype) == 0,
               "clip_grads: pointers must be aligned to their elements");
    write |= g.out != nullptr;
    chunks += (g.numel + kChunkElems - 1) / kChunkElems;
  }
  for (int64_t i = 0; i < count; ++i)
    FH_REQUIRE(!write || grads[i].out != nullptr || grads[i].numel == 0, "clip_grads: some outputs are null");
  FH_REQUIRE(!write || !overlaps(count, grads), "clip_grads: an output overlaps another operand");
  FH_REQUIRE(chunks < (int64_t(1) << 31), "clip_grads: too many elements");

  // The launches: runs of kTensors tensors.
  int n_partials = 0;
  int64_t tensors = 0;
  for (int64_t i = 0; i < count; ++i) tensors += grads[i].numel > 0;
  const int64_t launches = std::max<int64_t>(1, (tensors + kTensors - 1) / kTensors);
  const int64_t most = std::max<int64_t>(1, std::min(kBlocks, kPartials / launches));
  auto each = [&](auto&& launch) {
    int64_t i = 0;
    while (i < count) {
      Table t;
      t.n = 0;
      uint32_t at = 0;
      for (; i < count && t.n < kTensors; ++i) {
        const fh_grad& g = grads[i];
        if (g.numel == 0) continue;
        t.grad[t.n] = g.grad;
        t.out[t.n] = g.out;
        t.numel[t.n] = g.numel;
        t.first[t.n] = at;
        t.kind[t.n] = static_cast<uint8_t>((g.grad_dtype == FH_BF16 ? 1 : 0) | (g.out_dtype == FH_BF16 ? 2 : 0) |
                                           (aligned16(g.grad) && aligned16(g.out) ? 4 : 0));
        at += static_cast<uint32_t>((g.numel + kChunkElems - 1) / kChunkElems);
        ++t.n;
      }
      if (t.n == 0) continue;
      t.first[t.n] = at;
      launch(t, static_cast<unsigned>(std::min<int64_t>(most, at)));
    }
  };
  each([&](const Table& t, unsigned blocks) {
    hipLaunchKernelGGL(k_grad_squares, dim3(blocks), dim3(kThreads), 0, stream, t, partials + n_partials);
    n_partials += static_cast<int>(blocks);
  });
  if (!write || n_partials == 0) {
    hipLaunchKernelGGL(k_grad_norm, dim3(1), dim3(kThreads), 0, stream, partials, n_partials, norm);
  } else {
    bool tell = true;
    each([&](const Table& t, unsigned blocks) {
      hipLaunchKernelGGL(k_grad_scale, dim3(blocks), dim3(kThreads), 0, stream, t, partials, n_partials, max_norm, norm, tell);
      tell = false;
    });
  }
  return check_launch("fh_clip_grads");
}

}  // namespace
}  // namespace fh

using namespace fh;

extern "C" size_t fh_clip_grads_workspace_size(int64_t count) {
  if (count < 0) return 0;
  return static_cast<size_t>(std::max<int64_t>(kPartials, (count + kTensors - 1) / kTensors + 2)) * sizeof(double);
}

extern "C" int fh_clip_grads(int64_t count, const fh_grad* grads, float max_norm, float* norm, void* workspace,
                             hipStream_t stream) {
  try {
    return clip_grads(count, grads, max_norm, norm, static_cast<double*>(workspace), stream);
  } catch (const std::bad_alloc&) {
    return fail(FH_ERR_INVALID, "clip_grads: out of host memory");
  }
}
