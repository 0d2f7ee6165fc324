// Argument checks that the entry points without a context workspace share (api8.hip, api_packed.hip).
#pragma once
#include "common.hpp"

namespace fvsr {

int ctx_device(const fvsr_ctx* ctx);   // api.hip

#define FVSR_REQUIRE(cond, status, msg) \
  do {                                  \
    if (!(cond)) return set_error((status), (msg)); \
  } while (0)

// the context's device current for the call, the caller's again afterwards
class DeviceScope {
 public:
  explicit DeviceScope(int device) {
    ok_ = hipGetDevice(&prev_) == hipSuccess && (prev_ == device || hipSetDevice(device) == hipSuccess);
    moved_ = ok_ && prev_ != device;
  }
  ~DeviceScope() {
    if (moved_) (void)hipSetDevice(prev_);
  }
  bool ok() const { return ok_; }

 private:
  int prev_ = 0;
  bool ok_ = false, moved_ = false;
};

#define FVSR_ON_DEVICE(ctx)                 \
  DeviceScope scope(ctx_device(ctx));       \
  FVSR_REQUIRE(scope.ok(), FVSR_ERR_HIP, "the context's device cannot be made current")

inline bool dtype_ok(int d) { return d == FVSR_DTYPE_F32 || d == FVSR_DTYPE_BF16; }
inline bool aligned(const void* p, int to) { return ((uintptr_t)p & (to - 1)) == 0; }

inline int check_rows(const fvsr_ctx* ctx, int64_t rows, int channels, int most) {
  FVSR_REQUIRE(ctx != nullptr, FVSR_ERR_INVALID_ARG, "ctx is NULL");
  FVSR_REQUIRE(rows >= 0 && channels > 0, FVSR_ERR_INVALID_ARG, "rows must be >= 0 and channels > 0");
  FVSR_REQUIRE(rows <= (int64_t)1 << 40, FVSR_ERR_UNSUPPORTED, "too many rows");
  FVSR_REQUIRE(channels <= most, FVSR_ERR_UNSUPPORTED, "at most " + std::to_string(most) + " channels");
  return FVSR_OK;
}

inline int check_8(const void* codes, const void* scales, const char* what) {
  FVSR_REQUIRE(codes && scales, FVSR_ERR_INVALID_ARG, std::string(what) + ": codes and scales must be non-NULL");
  FVSR_REQUIRE(aligned(codes, 16) && aligned(scales, 4), FVSR_ERR_INVALID_ARG,
               std::string(what) + ": codes must be 16-byte and scales 4-byte aligned");
  return FVSR_OK;
}

inline int check_params(int dtype, int param_dtype, const void* w, const void* b) {
  FVSR_REQUIRE(dtype_ok(dtype), FVSR_ERR_INVALID_ARG, "dtype must be FVSR_DTYPE_F32 or FVSR_DTYPE_BF16");
  FVSR_REQUIRE((!w && !b) || param_dtype == FVSR_DTYPE_F32 || param_dtype == dtype, FVSR_ERR_INVALID_ARG,
               "weight and bias must be fp32 or of the tokens' type");
  return FVSR_OK;
}

}  // namespace fvsr
