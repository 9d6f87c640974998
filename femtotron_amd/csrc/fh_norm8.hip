// Activations kept in 8 bits (fh_pack8.hpp): pack and unpack, and the RMSNorm
// kernels of fh_norm.hpp that pack what they read or read what was packed.
//
// All are HBM-bound streams.  Keeping x costs the forward's norm 1.03 bytes an
// element more to write and no pass of its own; the backward's norms read 1.03
// bytes where they read 2 (bf16), and the 16-bit tensor is never laid out.  bf16 in
// int8, us a launch: pack 70 and unpack 67 at 32768 x 4096 (407 MB, 5.8 and 6.1
// TB/s); at 16384 x 2048 the norm that packs 28 (169 MB, 5.9), the norm from codes
// 17 (102 MB, 6.0), its add + norm 38 (236 MB, 6.1), the backward with the residual
// gradient 39 (236 MB, 6.1) and its reduction 4.  A copy runs at 5.4.  Those norms are
// rounded once; with llama_rounding, which eight_bit_checkpoint asks for, the norm
// from codes takes 21, in one run of all (the codes read by others before) the
// backward 51 against 49, the others within 2 us.
#include "femtohip_blocks.h"
#include "fh_norm.hpp"

namespace fh {
namespace {

// One thread = 8 elements.  Rows are counted in blocks of 32 (four threads), so
// that a quad of lanes holds one block also where a row ends inside it: thread
// -> (row, chunk of 8) over ceil(cols / 32) * 4 chunks a row.  16 elements a thread
// pack 16384 x 2048 in 17.9 us against 19.5, but unpack them in 18.9 against 16.5 and
// gain nothing at 32768 x 4096; two or four pieces a thread are slower at most sizes.
__device__ __forceinline__ void row_chunk(uint32_t idx, int cpr, const FastDiv& fd, int64_t& row, int& c) {
  const uint32_t q = fd.div(idx);
  row = q;
  c = static_cast<int>(idx - q * static_cast<uint32_t>(cpr)) * 8;
}

// STREAM: x with non-temporal loads.  An x that was read or written just before is
// still in the 256 MB cache below 128 MiB, and plain loads are then faster; one that
// is not there is faster streamed, at every size.  From 128 MiB on it hardly stays,
// and streaming wins both ways.  The kernel, us, plain and streamed, packed call after
// call (two x in turn) | with 1 GiB copied before:
//   bf16 4096 x 2048     6.6   7.6 |  8.4   7.1
//   bf16 16384 x 2048   18.2  20.8 | 21.9  19.9
//   bf16 32768 x 2048   43.7  36.5 | 40.4  37.5
//   bf16 32768 x 4096   80.0  71.9 | 74.0  69.3
//   fp32 8192 x 2048    13.5  18.4 | 19.9  16.1
//   fp32 16384 x 4096   78.2  61.5 | 70.9  61.6
// What unpacks the codes takes the same either way: 66.0 and 66.1 us at 32768 x 4096
// with 1 GiB copied between, as between a forward and its backward.
template <typename T, int FMT, bool STREAM>
__global__ __launch_bounds__(256) void k_pack8(const T* __restrict__ x, uint8_t* __restrict__ codes,
                                               uint8_t* __restrict__ exps, int64_t rows, int cols, int cpr,
                                               FastDiv fd) {
  const uint32_t idx = blockIdx.x * 256u + threadIdx.x;
  int64_t row;
  int c;
  row_chunk(idx, cpr, fd, row, c);
  const bool in = row < rows && c < cols;
  float v[8] = {};
  if (in) Elem<T>::unpack(load_if<T, STREAM>(x + row * cols + c), v);
  pack8_store<FMT>(v, codes + row * cols, exps + row * blocks8(cols), in, c);
}

template <typename T, int FMT>
__global__ __launch_bounds__(256) void k_unpack8(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ exps,
                                                 T* __restrict__ x, int64_t rows, int cols, int cpr, FastDiv fd) {
  const uint32_t idx = blockIdx.x * 256u + threadIdx.x;
  int64_t row;
  int c;
  row_chunk(idx, cpr, fd, row, c);
  if (row >= rows || c >= cols) return;
  float v[8];
  unpack8<FMT>(load8_codes(codes + row * cols, exps + row * blocks8(cols), c), v);
  Elem<T>::store8(x + row * cols + c, v);
}

int check_fmt(fh_dtype dt, fh_fmt8 fmt, const char* what) {
  if (dt != FH_BF16 && dt != FH_F32) return fail(FH_ERR_INVALID, std::string(what) + ": dtype must be FH_BF16 or FH_F32");
  if (fmt != FH_INT8 && fmt != FH_E4M3) return fail(FH_ERR_INVALID, std::string(what) + ": format must be FH_INT8 or FH_E4M3");
  return FH_OK;
}

bool aligned8(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 7u) == 0; }

// A launch has fewer than 2^32 threads, and the forward takes a wave a row.
int check_rows(fh_dtype dt, int64_t rows, int64_t cols) {
  if (int e = validate_rows(dt, rows, cols)) return e;
  FH_REQUIRE(rows < (int64_t(1) << 26), "rmsnorm: rows of a packed call must be < 2^26");
  return FH_OK;
}

// f(element type tag, format, std::bool_constant<flag>) for a checked dtype and format;
// the flag is a norm's rounding, or pack's streaming.
template <typename F>
void with_types(fh_dtype dt, fh_fmt8 fmt, bool flag, F&& f) {
  auto go = [&](auto tag, auto flg) {
    if (fmt == FH_INT8) f(tag, std::integral_constant<int, kFmtInt8>{}, flg);
    else f(tag, std::integral_constant<int, kFmtE4M3>{}, flg);
  };
  auto type = [&](auto tag) {
    if (flag) go(tag, std::true_type{});
    else go(tag, std::false_type{});
  };
  if (dt == FH_BF16) type(uint16_t{});
  else type(float{});
}

// Grid of a pack or unpack: FH_ERR_INVALID where it would pass the largest.
int stream_grid(int64_t rows, int64_t cols, const char* what, int64_t& threads) {
  if (rows < 0 || cols <= 0 || cols % 8 || cols > (int64_t(1) << 30))
    return fail(FH_ERR_INVALID, std::string(what) + ": rows must be >= 0 and cols a positive multiple of 8 (<= 2^30)");
  const int64_t cpr = blocks8(cols) * 4;
  // a launch has fewer than 2^32 threads
  if (rows > ((int64_t(1) << 32) - 256) / cpr)
    return fail(FH_ERR_INVALID, std::string(what) + ": too many elements for one call (2^35 or more)");
  threads = rows * cpr;
  return FH_OK;
}

}  // namespace
}  // namespace fh

using namespace fh;

extern "C" int fh_blocks_abi_version(void) { return FH_BLOCKS_ABI_VERSION; }

extern "C" int fh_pack8(fh_dtype dt, fh_fmt8 fmt, const void* x, void* codes, uint8_t* exps, int64_t rows, int64_t cols,
                        hipStream_t stream) {
  if (int e = check_fmt(dt, fmt, "pack8")) return e;
  int64_t threads = 0;
  if (int e = stream_grid(rows, cols, "pack8", threads)) return e;
  if (rows == 0) return FH_OK;
  FH_REQUIRE(x && codes && exps, "pack8: null pointer");
  FH_REQUIRE(aligned16(x) && aligned8(codes), "pack8: x must be 16-byte and codes 8-byte aligned");
  const int cpr = static_cast<int>(blocks8(cols) * 4);
  const FastDiv fd(static_cast<uint32_t>(cpr));
  const bool stream_x = rows * cols * (dt == FH_BF16 ? 2 : 4) >= (int64_t(128) << 20);
  with_types(dt, fmt, stream_x, [&](auto tag, auto f, auto st) {
    using T = decltype(tag);
    hipLaunchKernelGGL((k_pack8<T, f(), st()>), dim3(static_cast<unsigned>((threads + 255) / 256)), dim3(256), 0,
                       stream, static_cast<const T*>(x), static_cast<uint8_t*>(codes), exps, rows,
                       static_cast<int>(cols), cpr, fd);
  });
  return check_launch("fh_pack8");
}

extern "C" int fh_unpack8(fh_dtype dt, fh_fmt8 fmt, const void* codes, const uint8_t* exps, void* x, int64_t rows,
                          int64_t cols, hipStream_t stream) {
  if (int e = check_fmt(dt, fmt, "unpack8")) return e;
  int64_t threads = 0;
  if (int e = stream_grid(rows, cols, "unpack8", threads)) return e;
  if (rows == 0) return FH_OK;
  FH_REQUIRE(x && codes && exps, "unpack8: null pointer");
  FH_REQUIRE(aligned16(x) && aligned8(codes), "unpack8: x must be 16-byte and codes 8-byte aligned");
  const int cpr = static_cast<int>(blocks8(cols) * 4);
  const FastDiv fd(static_cast<uint32_t>(cpr));
  with_types(dt, fmt, true, [&](auto tag, auto f, auto) {
    using T = decltype(tag);
    hipLaunchKernelGGL((k_unpack8<T, f()>), dim3(static_cast<unsigned>((threads + 255) / 256)), dim3(256), 0,
                       stream, static_cast<const uint8_t*>(codes), exps, static_cast<T*>(x), rows,
                       static_cast<int>(cols), cpr, fd);
  });
  return check_launch("fh_unpack8");
}

extern "C" int fh_rmsnorm_fwd_pack8(fh_dtype dt, fh_fmt8 fmt, const void* x, const void* w, void* y, void* codes,
                                    uint8_t* exps, float* rstd, int64_t rows, int64_t cols, float eps,
                                    int llama_rounding, hipStream_t stream) {
  if (int e = check_fmt(dt, fmt, "rmsnorm_fwd_pack8")) return e;
  if (int e = check_rows(dt, rows, cols)) return e;
  if (rows == 0) return FH_OK;
  FH_REQUIRE(x && w && y && codes && exps, "rmsnorm_fwd_pack8: null pointer");
  FH_REQUIRE(aligned16(x) && aligned16(w) && aligned16(y) && aligned8(codes),
             "rmsnorm_fwd_pack8: pointers must be 16-byte aligned (codes 8-byte)");
  const int c = static_cast<int>(cols);
  with_types(dt, fmt, llama_rounding != 0, [&](auto tag, auto f, auto rnd) {
    using T = decltype(tag);
    dispatch_nv(c, [&](auto nv) {
      launch_fwd<T, RowsT<T>, f(), nv(), rnd()>(x, nullptr, w, nullptr, y, rstd, codes, exps, rows, c, eps, stream);
      return 0;
    });
  });
  return check_launch("fh_rmsnorm_fwd_pack8");
}

extern "C" int fh_rmsnorm_fwd8(fh_dtype dt, fh_fmt8 fmt, const void* codes, const uint8_t* exps, const void* w, void* y,
                               float* rstd, int64_t rows, int64_t cols, float eps,
                               int llama_rounding, hipStream_t stream) {
  if (int e = check_fmt(dt, fmt, "rmsnorm_fwd8")) return e;
  if (int e = check_rows(dt, rows, cols)) return e;
  if (rows == 0) return FH_OK;
  FH_REQUIRE(codes && exps && w && y, "rmsnorm_fwd8: null pointer");
  FH_REQUIRE(aligned8(codes) && aligned16(w) && aligned16(y),
             "rmsnorm_fwd8: pointers must be 16-byte aligned (codes 8-byte)");
  const int c = static_cast<int>(cols);
  with_types(dt, fmt, llama_rounding != 0, [&](auto tag, auto f, auto rnd) {
    using T = decltype(tag);
    dispatch_nv(c, [&](auto nv) {
      launch_fwd<T, Rows8<f()>, kNoPack, nv(), rnd()>(nullptr, nullptr, w, nullptr, y, rstd, codes, exps, rows, c, eps, stream);
      return 0;
    });
  });
  return check_launch("fh_rmsnorm_fwd8");
}

extern "C" int fh_add_rmsnorm_fwd8(fh_dtype dt, fh_fmt8 fmt, const void* codes, const uint8_t* exps, const void* a,
                                   const void* w, void* h, void* y, float* rstd, int64_t rows, int64_t cols, float eps,
                                   int llama_rounding, hipStream_t stream) {
  if (int e = check_fmt(dt, fmt, "add_rmsnorm_fwd8")) return e;
  if (int e = check_rows(dt, rows, cols)) return e;
  if (rows == 0) return FH_OK;
  FH_REQUIRE(codes && exps && a && w && h && y, "add_rmsnorm_fwd8: null pointer");
  FH_REQUIRE(aligned8(codes) && aligned16(a) && aligned16(w) && aligned16(h) && aligned16(y),
             "add_rmsnorm_fwd8: pointers must be 16-byte aligned (codes 8-byte)");
  FH_REQUIRE(h != a, "add_rmsnorm_fwd8: h must not alias a");
  const int c = static_cast<int>(cols);
  with_types(dt, fmt, llama_rounding != 0, [&](auto tag, auto f, auto rnd) {
    using T = decltype(tag);
    dispatch_nv(c, [&](auto nv) {
      launch_fwd<T, Rows8<f()>, kNoPack, nv(), rnd()>(nullptr, a, w, h, y, rstd, codes, exps, rows, c, eps, stream);
      return 0;
    });
  });
  return check_launch("fh_add_rmsnorm_fwd8");
}

extern "C" size_t fh_rmsnorm_bwd8_workspace_size(int64_t rows, int64_t cols) {
  if (rows <= 0 || cols <= 0 || cols > 8192) return 0;
  // the partial rows of the split that a call takes: fh_rmsnorm_bwd's, or its own
  size_t blocks = 0;
  dispatch_nv(static_cast<int>(cols), [&](auto nv) {
    using SP = Bwd8Split<nv(), false>;
    blocks = static_cast<size_t>(bwd_blocks(rows, SP::RPB, SP::kBlocks));
    return 0;
  });
  const size_t own = blocks * static_cast<size_t>(cols) * sizeof(float), other = fh_rmsnorm_bwd_workspace_size(rows, cols);
  return own > other ? own : other;
}

extern "C" int fh_rmsnorm_bwd8(fh_dtype dt, fh_fmt8 fmt, const void* dy, const void* codes, const uint8_t* exps,
                               const void* w, const float* rstd, const void* dres, void* dx, void* dw, void* workspace,
                               int64_t rows, int64_t cols, float eps,
                               int llama_rounding, hipStream_t stream) {
  if (int e = check_fmt(dt, fmt, "rmsnorm_bwd8")) return e;
  if (int e = check_rows(dt, rows, cols)) return e;
  FH_REQUIRE(w && dw, "rmsnorm_bwd8: null pointer");
  if (rows == 0)  // the weight gradient alone, zeros
    return fh_rmsnorm_bwd(dt, nullptr, nullptr, w, nullptr, nullptr, nullptr, dw, nullptr, 0, cols, eps, stream);
  FH_REQUIRE(dy && codes && exps && dx && workspace, "rmsnorm_bwd8: null pointer");
  FH_REQUIRE(aligned16(dy) && aligned8(codes) && aligned16(w) && aligned16(dx) &&
                 (dres == nullptr || aligned16(dres)) && aligned16(workspace),
             "rmsnorm_bwd8: pointers (workspace included) must be 16-byte aligned (codes 8-byte)");
  const int c = static_cast<int>(cols);
  float* part = static_cast<float*>(workspace);
  with_types(dt, fmt, llama_rounding != 0, [&](auto tag, auto f, auto rnd) {
    using T = decltype(tag);
    dispatch_nv(c, [&](auto nv) {
      launch_bwd<T, Rows8<f()>, nv(), rnd()>(dy, codes, exps, w, rstd, dres, dx, dw, part, rows, c, eps, stream);
      return 0;
    });
  });
  return check_launch("fh_rmsnorm_bwd8");
}
