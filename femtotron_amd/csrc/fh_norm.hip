// RMSNorm forward / residual-add + RMSNorm forward / RMSNorm backward: entry
// points (kernels and launches in fh_norm.hpp).
#include <mutex>

#include "fh_norm.hpp"

using namespace fh;

extern "C" int fh_rmsnorm_fwd(fh_dtype dt, const void* x, const void* w, void* y, float* rstd,
                              int64_t rows, int64_t cols, float eps, hipStream_t stream) {
  if (int e = validate_rows(dt, rows, cols)) return e;
  if (rows == 0) return FH_OK;
  FH_REQUIRE(x && w && y, "rmsnorm_fwd: null pointer");
  FH_REQUIRE(aligned16(x) && aligned16(w) && aligned16(y), "rmsnorm_fwd: pointers must be 16-byte aligned");
  const int c = static_cast<int>(cols);
  dispatch_nv(c, [&](auto nv) {
    if (dt == FH_BF16) launch_fwd<uint16_t, RowsT<uint16_t>, kNoPack, nv()>(x, nullptr, w, nullptr, y, rstd, nullptr, nullptr, rows, c, eps, stream);
    else launch_fwd<float, RowsT<float>, kNoPack, nv()>(x, nullptr, w, nullptr, y, rstd, nullptr, nullptr, rows, c, eps, stream);
    return 0;
  });
  return check_launch("fh_rmsnorm_fwd");
}

extern "C" int fh_add_rmsnorm_fwd(fh_dtype dt, const void* x, const void* a, const void* w,
                                  void* h, void* y, float* rstd, int64_t rows, int64_t cols,
                                  float eps, hipStream_t stream) {
  if (int e = validate_rows(dt, rows, cols)) return e;
  if (rows == 0) return FH_OK;
  FH_REQUIRE(x && a && w && h && y, "add_rmsnorm_fwd: null pointer");
  FH_REQUIRE(aligned16(x) && aligned16(a) && aligned16(w) && aligned16(h) && aligned16(y),
             "add_rmsnorm_fwd: pointers must be 16-byte aligned");
  FH_REQUIRE(h != x && h != a, "add_rmsnorm_fwd: h must not alias x or a");
  const int c = static_cast<int>(cols);
  dispatch_nv(c, [&](auto nv) {
    if (dt == FH_BF16) launch_fwd<uint16_t, RowsT<uint16_t>, kNoPack, nv()>(x, a, w, h, y, rstd, nullptr, nullptr, rows, c, eps, stream);
    else launch_fwd<float, RowsT<float>, kNoPack, nv()>(x, a, w, h, y, rstd, nullptr, nullptr, rows, c, eps, stream);
    return 0;
  });
  return check_launch("fh_add_rmsnorm_fwd");
}

extern "C" size_t fh_rmsnorm_bwd_workspace_size(int64_t rows, int64_t cols) {
  if (rows <= 0 || cols <= 0) return 0;
  // one fp32 partial row per backward block (4 rows per block, 2 above 2048
  // columns)
  const int64_t nrows = bwd_blocks(rows, cols > 2048 ? 2 : 4, kMaxBwdBlocks);
  return static_cast<size_t>(nrows) * static_cast<size_t>(cols) * sizeof(float);
}

namespace fh {
namespace {

// Scratch of the allocation-free backward: the fp32 partial rows of the
// largest valid call (kMaxBwdBlocks partial rows of at most 8192 columns),
// 16.8 MB per device, held until the process ends.
constexpr size_t kNoAllocScratchFloats = static_cast<size_t>(kMaxBwdBlocks) * 8192;
__device__ __align__(256) float scratch[kNoAllocScratchFloats];

// Device address of `scratch` on the current device, looked up once per
// device (each device holds its own copy of the array at its own address;
// the host-side symbol is only a stand-in and must never reach a kernel).
float* scratch_on_current_device(int* status) {
  constexpr int kMaxDevices = 64;
  static std::once_flag once[kMaxDevices];
  static float* addr[kMaxDevices] = {};
  static hipError_t err[kMaxDevices] = {};
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= kMaxDevices) {
    *status = fail(FH_ERR_LAUNCH, "rmsnorm_bwd_noalloc: no current HIP device");
    return nullptr;
  }
  std::call_once(once[dev], [dev]() {
    void* p = nullptr;
    err[dev] = hipGetSymbolAddress(&p, HIP_SYMBOL(scratch));
    addr[dev] = static_cast<float*>(p);
  });
  if (err[dev] != hipSuccess || addr[dev] == nullptr) {
    *status = fail(FH_ERR_LAUNCH, std::string("rmsnorm_bwd_noalloc: hipGetSymbolAddress failed: ") +
                                      hipGetErrorString(err[dev]));
    return nullptr;
  }
  *status = FH_OK;
  return addr[dev];
}

}  // namespace
}  // namespace fh

extern "C" int fh_rmsnorm_bwd(fh_dtype dt, const void* dy, const void* x, const void* w,
                              const float* rstd, const void* dres, void* dx, void* dw,
                              void* workspace, int64_t rows, int64_t cols, float eps,
                              hipStream_t stream) {
  if (int e = validate_rows(dt, rows, cols)) return e;
  FH_REQUIRE(w && dw, "rmsnorm_bwd: null pointer");
  const int c = static_cast<int>(cols);
  if (rows == 0) {
    // Empty batch: the weight gradient is an all-zero row (a reduction over
    // zero partials; a kernel rather than hipMemsetAsync so the call stays
    // safe inside a captured graph).
    if (dt == FH_BF16)
      hipLaunchKernelGGL((k_fill_zero<uint16_t>), dim3((c + 255) / 256), dim3(256), 0, stream,
                         static_cast<uint16_t*>(dw), c);
    else
      hipLaunchKernelGGL((k_fill_zero<float>), dim3((c + 255) / 256), dim3(256), 0, stream,
                         static_cast<float*>(dw), c);
    return check_launch("fh_rmsnorm_bwd");
  }
  FH_REQUIRE(dy && x && dx && workspace, "rmsnorm_bwd: null pointer");
  FH_REQUIRE(aligned16(dy) && aligned16(x) && aligned16(w) && aligned16(dx) &&
                 (dres == nullptr || aligned16(dres)) && aligned16(workspace),
             "rmsnorm_bwd: pointers (workspace included) must be 16-byte aligned");
  float* part = static_cast<float*>(workspace);
  dispatch_nv(c, [&](auto nv) {
    if (dt == FH_BF16) launch_bwd<uint16_t, RowsT<uint16_t>, nv()>(dy, x, nullptr, w, rstd, dres, dx, dw, part, rows, c, eps, stream);
    else launch_bwd<float, RowsT<float>, nv()>(dy, x, nullptr, w, rstd, dres, dx, dw, part, rows, c, eps, stream);
    return 0;
  });
  return check_launch("fh_rmsnorm_bwd");
}

extern "C" size_t fh_rmsnorm_bwd_noalloc_max_workspace(void) {
  return kNoAllocScratchFloats * sizeof(float);
}

extern "C" int fh_rmsnorm_bwd_noalloc(fh_dtype dt, const void* dy, const void* x, const void* w,
                                      const float* rstd, const void* dres, void* dx, void* dw,
                                      int64_t rows, int64_t cols, float eps, hipStream_t stream) {
  if (int e = validate_rows(dt, rows, cols)) return e;
  FH_REQUIRE(fh_rmsnorm_bwd_workspace_size(rows, cols) <= kNoAllocScratchFloats * sizeof(float),
             "rmsnorm_bwd_noalloc: the call needs more scratch than the library holds");
  if (rows == 0)  // no scratch needed: dw = 0
    return fh_rmsnorm_bwd(dt, dy, x, w, rstd, dres, dx, dw, nullptr, rows, cols, eps, stream);
  int status = FH_OK;
  float* ws = scratch_on_current_device(&status);
  if (ws == nullptr) return status;
  return fh_rmsnorm_bwd(dt, dy, x, w, rstd, dres, dx, dw, ws, rows, cols, eps, stream);
}
