// Dropout whose mask is a function of the element's index and is never stored.
//
// The random bits of element e come from Philox4x32-10, the counter-based generator of
// Salmon, Moraes, Dror and Shaw ("Parallel random numbers: as easy as 1, 2, 3", SC 2011):
// ten rounds of two 32x32 -> 64 bit products over a 128-bit counter.  The counter is
// (e / 8, offset), the key is the seed, so the backward pass runs the same kernel on the
// incoming gradient and finds the same elements.
#include "twg_geom.h"
#include "twg_nn.h"

namespace twg {
namespace {

constexpr int kPer = 8;  // elements per Philox call, 16 bits each

struct Words {
  uint32_t w[4];
};

__device__ __forceinline__ Words philox(uint64_t block, uint64_t offset, uint64_t seed) {
  uint32_t c0 = (uint32_t)block, c1 = (uint32_t)(block >> 32);
  uint32_t c2 = (uint32_t)offset, c3 = (uint32_t)(offset >> 32);
  uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t p0 = (uint64_t)c0 * 0xD2511F53u, p1 = (uint64_t)c2 * 0xCD9E8D57u;
    c0 = (uint32_t)(p1 >> 32) ^ c1 ^ k0;
    c2 = (uint32_t)(p0 >> 32) ^ c3 ^ k1;
    c1 = (uint32_t)p1;
    c3 = (uint32_t)p0;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return Words{{c0, c1, c2, c3}};
}

struct DropArgs {
  uint64_t seed, offset;
  const uint64_t *d_offset;
  uint32_t threshold;  // dropped where the 16 bits are below it: 0..65536
  float scale;
};

// residual + keep * x * scale in binary32, rounded once by the caller
__device__ __forceinline__ float dropped(float x, float res, uint32_t bits, const DropArgs &a) {
  return res + (bits < a.threshold ? 0.0f : x * a.scale);
}

__device__ __forceinline__ uint64_t total_offset(const DropArgs &a) {
  return a.offset + (a.d_offset ? *a.d_offset : 0);
}

// Any strides: a lane takes one group of 8 elements in logical order.
template <typename T, bool RES>
__global__ void __launch_bounds__(kThreads) dropout_any(T *out, const T *x, const T *res, Geom g, DropArgs a) {
  const int64_t group = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  int64_t e = group * kPer;
  if (e >= g.numel) return;
  const Words w = philox((uint64_t)group, total_offset(a), a.seed);
#pragma unroll
  for (int j = 0; j < kPer; ++j, ++e) {
    if (e >= g.numel) break;
    int64_t rest = e, oo = 0, ox = 0, orr = 0;
    for (int d = 0; d < g.ndim; ++d) {
      const int64_t q = rest / g.shape[d], i = rest - q * g.shape[d];
      rest = q;
      oo += i * g.stride[TWG_OUT][d];
      ox += i * g.stride[TWG_A][d];
      if (RES) orr += i * g.stride[TWG_B][d];
    }
    const uint32_t bits = (w.w[j / 2] >> (16 * (j & 1))) & 0xFFFFu;
    out[oo] = (T)dropped((float)x[ox], RES ? (float)res[orr] : 0.0f, bits, a);
  }
}

template <typename T>
int launch_dropout(T *out, const T *x, const T *res, const Geom &g, const DropArgs &a, hipStream_t s) {
  const int64_t groups = (g.numel + kPer - 1) / kPer, blocks = (groups + kThreads - 1) / kThreads;
  if (blocks > INT32_MAX) return TWG_E_TOO_LARGE;
  if (res)
    dropout_any<T, true><<<(unsigned)blocks, kThreads, 0, s>>>(out, x, res, g, a);
  else
    dropout_any<T, false><<<(unsigned)blocks, kThreads, 0, s>>>(out, x, res, g, a);
  return (int)hipGetLastError();
}

}  // namespace
}  // namespace twg

using namespace twg;

extern "C" int twg_dropout(void *out, const void *x, const void *residual, int32_t dtype, double p,
                           uint64_t seed, uint64_t offset, const uint64_t *d_offset,
                           const twg_iter_t *it, twg_stream_t stream) {
  if (!nn_dtype(dtype) || !(p >= 0.0 && p <= 1.0)) return TWG_E_INVALID_ARG;
  Geom g;
  int rc = canonicalize(it, residual ? 3 : 2, &g, /*reorder=*/false);
  if (rc) return rc;
  if (g.numel == 0) return 0;
  if (!out || !x) return TWG_E_INVALID_ARG;
  const size_t size = (size_t)nn_size(dtype);
  if (!aligned_to(out, size) || !aligned_to(x, size) || !aligned_to(residual, size) ||
      !aligned_to(d_offset, 8))
    return TWG_E_INVALID_ARG;
  for (int d = 0; d < g.ndim; ++d)  // several elements in one place: no order among their stores
    if (g.stride[TWG_OUT][d] == 0) return TWG_E_INVALID_ARG;
  if ((rc = ensure_init())) return rc;
  DropArgs a;
  a.seed = seed;
  a.offset = offset;
  a.d_offset = d_offset;
  a.threshold = (uint32_t)std::floor(p * 65536.0 + 0.5);
  a.scale = a.threshold < 65536 ? (float)(65536.0 / (65536.0 - a.threshold)) : 0.0f;
  return nn_dispatch(dtype, [&](auto t) {
    using T = decltype(t);
    return launch_dropout<T>(static_cast<T *>(out), static_cast<const T *>(x),
                             static_cast<const T *>(residual), g, a, nn_stream(stream));
  });
}
