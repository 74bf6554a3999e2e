// What the kernels of csrc/nn share: element types, streams, small device helpers.
#pragma once

#include <hip/hip_runtime.h>

#include <cmath>

#include "twg_ew_packs.h"
#include "twg_internal.h"

namespace twg {
namespace {

typedef _Float16 F16;
typedef __bf16 BF16;  // converts with v_cvt_pk_bf16_f32: round to nearest even, NaN stays NaN

inline bool nn_dtype(int32_t dt) { return dt == TWG_DT_F16 || dt == TWG_DT_BF16 || dt == TWG_DT_F32; }
inline int nn_size(int32_t dt) { return dt == TWG_DT_F32 ? 4 : 2; }

// A launch goes to the calling thread's current device, and so does the null stream, but
// pointers and streams are device 0's, which the library is bound to: device 0 is made current while a call
// works, its initialisation included, and the caller's own device afterwards.
class OnBoundDevice {
 public:
  OnBoundDevice() {
    if (hipGetDevice(&was_) != hipSuccess) was_ = 0;  // (no device: the initialisation says so)
    if (was_ != 0) status_ = (int)hipSetDevice(0);
    if (status_ == 0) status_ = ensure_init();
  }
  ~OnBoundDevice() {
    if (was_ != 0) (void)hipSetDevice(was_);
  }
  OnBoundDevice(const OnBoundDevice &) = delete;
  OnBoundDevice &operator=(const OnBoundDevice &) = delete;
  int status() const { return status_; }

 private:
  int was_ = 0, status_ = 0;
};

// NULL is the library's own stream, TWG_STREAM_NULL the null stream of device 0.
inline hipStream_t nn_stream(twg_stream_t s) {
  return s == TWG_STREAM_NULL ? hipStream_t(nullptr) : resolve_stream(s);
}

// fn(T()) for the element type of a dtype that nn_dtype accepts
template <typename Fn>
int nn_dispatch(int32_t dt, Fn fn) {
  switch (dt) {
    case TWG_DT_F16: return fn(F16());
    case TWG_DT_BF16: return fn(BF16());
    default: return fn(float());
  }
}

// a + b for extents and offsets that a caller may have made up: false on overflow
inline bool add_product(int64_t &sum, int64_t a, int64_t b) {
  int64_t p;
  return !__builtin_mul_overflow(a, b, &p) && !__builtin_add_overflow(sum, p, &sum);
}

}  // namespace
}  // namespace twg
