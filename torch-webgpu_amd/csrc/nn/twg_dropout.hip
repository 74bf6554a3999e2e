// Dropout whose mask is a function of the element's index and is never stored.
//
// The random bits of element e come from Philox4x32-10, the counter-based generator of
// Salmon, Moraes, Dror and Shaw ("Parallel random numbers: as easy as 1, 2, 3", SC 2011):
// ten rounds of two 32x32 -> 64 bit products over a 128-bit counter.  The counter is
// (e / 8, offset), the key is the seed, so the backward pass runs the same kernel on the
// incoming gradient and finds the same elements.
//
// Bound by memory where the operands are dense: 2^27 bfloat16 elements with a residual 121 us (6.7 TB/s), 2^28
// float32 elements 332 us (6.5 TB/s); the generator's 20 products a call keep the vector units busy
// for a quarter to a half of that time.  With 32 random bits an element instead of 16 it would be
// twice that, and the bound.
#include "twg_geom.h"
#include "twg_nn.h"

namespace twg {
namespace {

constexpr int kPer = 8;  // elements per Philox call, 16 bits each
constexpr int kDenseThreads = 64;

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

// Rows whose elements lie side by side, whole groups of 8 and aligned to 16 bytes in every
// operand: packs of 16 bytes.  DENSE: one long row, the last group of which may be short.
// Bound by memory (2 or 3 x 8 elements per lane against ten rounds of two products): one group
// per lane and no loop, as for the framework's other dense kernels.
template <typename T, bool RES, bool DENSE, bool STREAM>
__global__ void __launch_bounds__(kDenseThreads) dropout_packs(T *out, const T *x, const T *res, Geom g, DropArgs a) {
  constexpr int E = 16 / (int)sizeof(T), P = kPer / E;
  typedef Pack<T, E> Vec;
  const int64_t group = (int64_t)blockIdx.x * kDenseThreads + threadIdx.x;
  const int64_t e = group * kPer;
  if (e >= g.numel) return;
  int64_t oo = e, ox = e, orr = e;
  if constexpr (!DENSE) {
    int64_t rest = e / g.shape[0], i = e - rest * g.shape[0];
    oo = ox = orr = i;
    for (int d = 1; d < g.ndim; ++d) {
      const int64_t q = rest / g.shape[d];
      i = rest - q * g.shape[d];
      rest = q;
      oo += i * g.stride[TWG_OUT][d];
      ox += i * g.stride[TWG_A][d];
      if (RES) orr += i * g.stride[TWG_B][d];
    }
  }
  const int count = DENSE && g.numel - e < kPer ? (int)(g.numel - e) : kPer;
  Pack<T, kPer> vx, vr, vo;
  if (count == kPer) {
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const Vec l = load_pack<STREAM>(reinterpret_cast<const Vec *>(x + ox) + p);
      __builtin_memcpy(&vx.v[p * E], &l, 16);
      if (RES) {
        const Vec m = load_pack<STREAM>(reinterpret_cast<const Vec *>(res + orr) + p);
        __builtin_memcpy(&vr.v[p * E], &m, 16);
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      if (j >= count) continue;
      vx.v[j] = x[ox + j];
      if (RES) vr.v[j] = res[orr + j];
    }
  }
  const Words w = philox((uint64_t)group, total_offset(a), a.seed);
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const uint32_t bits = (w.w[j / 2] >> (16 * (j & 1))) & 0xFFFFu;
    vo.v[j] = (T)dropped((float)vx.v[j], RES ? (float)vr.v[j] : 0.0f, bits, a);
  }
  if (count == kPer) {
#pragma unroll
    for (int p = 0; p < P; ++p) {
      Vec l;
      __builtin_memcpy(&l, &vo.v[p * E], 16);
      store_pack<STREAM>(reinterpret_cast<Vec *>(out + oo) + p, l);
    }
  } else {
#pragma unroll
    for (int j = 0; j < kPer; ++j)
      if (j < count) out[oo + j] = vo.v[j];
  }
}

// The same for dense float32, where a group is two packs: lane by lane, a wavefront's loads and
// stores would each touch every other 16 bytes.  The lanes take packs side by side
// instead, 64 and the next 64, and find the words of a pack's group in LDS, where lane g has put those of
// group g.
template <bool RES, bool STREAM>
__global__ void __launch_bounds__(64) dropout_pairs(float *out, const float *x, const float *res, int64_t numel, DropArgs a) {
  typedef Pack<float, 4> Vec;
  __shared__ Pack<uint32_t, 4> words[64];
  const int lane = threadIdx.x;
  const int64_t e0 = (int64_t)blockIdx.x * 64 * kPer;
  Vec vx[2], vr[2];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int64_t e = e0 + (u * 64 + lane) * 4;
    if (e + 4 <= numel) {
      vx[u] = load_pack<STREAM>(reinterpret_cast<const Vec *>(x + e));
      if (RES) vr[u] = load_pack<STREAM>(reinterpret_cast<const Vec *>(res + e));
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (e + j >= numel) continue;
        vx[u].v[j] = x[e + j];
        if (RES) vr[u].v[j] = res[e + j];
      }
    }
  }
  const Words w = philox((uint64_t)(e0 / kPer + lane), total_offset(a), a.seed);
  words[lane] = Pack<uint32_t, 4>{{w.w[0], w.w[1], w.w[2], w.w[3]}};
  __syncthreads();
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int64_t e = e0 + (u * 64 + lane) * 4;
    const uint32_t *half = &words[u * 32 + lane / 2].v[2 * (lane & 1)];
    const uint32_t h0 = half[0], h1 = half[1];
    Vec o;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t bits = ((j < 2 ? h0 : h1) >> (16 * (j & 1))) & 0xFFFFu;
      o.v[j] = dropped(vx[u].v[j], RES ? vr[u].v[j] : 0.0f, bits, a);
    }
    if (e + 4 <= numel) {
      store_pack<STREAM>(reinterpret_cast<Vec *>(out + e), o);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (e + j < numel) out[e + j] = o.v[j];
    }
  }
}

// Whether every operand's groups of 8 elements are two or one aligned packs.
bool packs_fit(const Geom &g, const void *out, const void *x, const void *res, int size) {
  if (!aligned_to(out, 16) || !aligned_to(x, 16) || !aligned_to(res, 16)) return false;
  const int ops = res ? 3 : 2;
  for (int o = 0; o < ops; ++o) {
    if (g.ndim && g.stride[o][0] != 1) return false;
    for (int d = 1; d < g.ndim; ++d)
      if (g.stride[o][d] * size % 16) return false;
  }
  return g.ndim <= 1 || g.shape[0] % kPer == 0;
}

template <typename T>
int launch_dropout(T *out, const T *x, const T *res, const Geom &g, const DropArgs &a, hipStream_t s) {
  const int64_t groups = (g.numel + kPer - 1) / kPer, blocks = (groups + kThreads - 1) / kThreads;
  if (blocks * kThreads > UINT32_MAX) return TWG_E_TOO_LARGE;  // a launch's threads are counted in 32 bits
  if (packs_fit(g, out, x, res, (int)sizeof(T))) {
    const int64_t small = (groups + kDenseThreads - 1) / kDenseThreads;
    const bool stream = g.numel * (int64_t)sizeof(T) * (res ? 3 : 2) > kStreamBytes, dense = g.ndim <= 1;
    if constexpr (sizeof(T) == 4) {
      if (dense) {
        if (res && stream) dropout_pairs<true, true><<<(unsigned)small, 64, 0, s>>>(out, x, res, g.numel, a);
        else if (res) dropout_pairs<true, false><<<(unsigned)small, 64, 0, s>>>(out, x, res, g.numel, a);
        else if (stream) dropout_pairs<false, true><<<(unsigned)small, 64, 0, s>>>(out, x, res, g.numel, a);
        else dropout_pairs<false, false><<<(unsigned)small, 64, 0, s>>>(out, x, res, g.numel, a);
        return (int)hipGetLastError();
      }
    }
#define TWG_DROP(RES, DENSE, STREAM) \
  dropout_packs<T, RES, DENSE, STREAM><<<(unsigned)small, kDenseThreads, 0, s>>>(out, x, res, g, a)
    if (sizeof(T) == 2 && dense) {
      if (res && stream) TWG_DROP(true, sizeof(T) == 2, true);
      else if (res) TWG_DROP(true, sizeof(T) == 2, false);
      else if (stream) TWG_DROP(false, sizeof(T) == 2, true);
      else TWG_DROP(false, sizeof(T) == 2, false);
    } else {
      if (res && stream) TWG_DROP(true, false, true);
      else if (res) TWG_DROP(true, false, false);
      else if (stream) TWG_DROP(false, false, true);
      else TWG_DROP(false, false, false);
    }
#undef TWG_DROP
    return (int)hipGetLastError();
  }
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
  const OnBoundDevice device;
  if ((rc = device.status())) return rc;
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
