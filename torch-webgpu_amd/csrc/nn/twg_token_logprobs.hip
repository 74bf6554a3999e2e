// Log probabilities of given tokens, the rows' entropies and top alternatives, and the
// gradient with respect to the logits.
//
//   m = max x, s = sum e^(c (x - m)), logprob = c (x_t - m) - log s,
//   entropy = log s - (1/s) sum e^(c (x - m)) c (x - m)
//   grad_j = c (g_lp ([j = t] - p_j) - g_H p_j (log p_j + entropy)),  p_j = e^(c (x_j - m)) / s
#include "twg_nn.h"

namespace twg {
namespace {

constexpr float kLog2e = 0x1.715476p+0f;
constexpr float kLn2f = 0x1.62e430p-1f;

struct LogprobArgs {
  const void *logits, *targets;
  int64_t rows, row_stride, ignore_index;
  int32_t vocab, top_k;
  int32_t wide_targets;  // int64 instead of int32
  float scale;
  float *logprob, *entropy, *row_max, *row_sum, *top_logprobs;
  int64_t *top_ids;
  const float *g_logprob, *g_entropy;
  const float *in_max, *in_sum, *in_entropy;
  void *grad;
  int64_t grad_stride;
};

__device__ __forceinline__ int64_t target_of(const LogprobArgs &a, int64_t row) {
  return a.wide_targets ? ((const int64_t *)a.targets)[row] : (int64_t)((const int32_t *)a.targets)[row];
}

// Order of the alternatives as one number: the value (-0 as +0, NaN on top), then the lower id.
__device__ __forceinline__ uint64_t key_of(float x, uint32_t id) {
  const uint32_t b = __float_as_uint(x + 0.0f);
  const uint32_t v = x != x ? 0xFFFFFFFFu : b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
  return (uint64_t)v << 32 | (uint32_t)~id;
}
__device__ __forceinline__ float value_of(uint64_t key) {
  const uint32_t v = (uint32_t)(key >> 32);
  if (v == 0xFFFFFFFFu) return __uint_as_float(0x7FC00000u);
  return __uint_as_float(v & 0x80000000u ? v ^ 0x80000000u : ~v);
}
__device__ __forceinline__ uint32_t id_of(uint64_t key) { return ~(uint32_t)key; }

// A running softmax sum: m the largest entry so far, s = sum e^(c (x - m)) and
// t = sum e^(c (x - m)) c (x - m), the last in base 2.  -inf entries add nothing; before the
// first other entry m is -inf and s is 0.
struct Run {
  float m, s, t;
};

__device__ __forceinline__ float exponent(float x, float m, float c2) { return (x - m) * c2; }

__device__ __forceinline__ void add_to(Run &r, float x, float c2) {
  if (x > r.m) {
    if (r.s > 0.0f) {
      const float d = fmaxf(exponent(r.m, x, c2), -300.0f), f = exp2f(d);
      r.t = f * __fmaf_rn(d, r.s, r.t);
      r.s *= f;
    }
    r.m = x;
  }
  if (x == -INFINITY) return;
  const float d = exponent(x, r.m, c2), e = exp2f(d);
  r.s += e;
  r.t = __fmaf_rn(e, fmaxf(d, -300.0f), r.t);
}

__device__ __forceinline__ Run join(const Run &a, const Run &b, float c2) {
  const bool swap = b.m > a.m;
  const Run &hi = swap ? b : a, &lo = swap ? a : b;
  Run r = hi;
  // (a sum that is 0 has no entries; one that is NaN is passed on)
  if (lo.s != 0.0f) {
    const float d = hi.m == lo.m ? 0.0f : fmaxf(exponent(lo.m, hi.m, c2), -300.0f), f = exp2f(d);
    r.s += lo.s * f;
    r.t += f * __fmaf_rn(d, lo.s, lo.t);
  }
  return r;
}

__device__ __forceinline__ Run shuffled(const Run &r, int lanes) {
  return Run{__shfl_xor(r.m, lanes), __shfl_xor(r.s, lanes), __shfl_xor(r.t, lanes)};
}

// (in base e: an entry of the type's lowest value times log2 e would leave binary32's range)
__device__ __forceinline__ float log_prob(float x, const Run &r, float scale) {
  return r.s == 0.0f ? -INFINITY : (x - r.m) * scale - kLn2f * log2f(r.s);
}

// one row by one workgroup
template <typename T>
__global__ void __launch_bounds__(kThreads) logprobs_rows(LogprobArgs a) {
  __shared__ Run runs[kThreads / 64];
  __shared__ uint64_t best[kThreads / 64];
  const int64_t row = blockIdx.x;
  const T *x = (const T *)a.logits + row * a.row_stride;
  const float c2 = a.scale * kLog2e;
  Run r{-INFINITY, 0.0f, 0.0f};
  for (int i = threadIdx.x; i < a.vocab; i += kThreads) add_to(r, (float)x[i], c2);
  for (int i = 1; i < 64; i <<= 1) r = join(r, shuffled(r, i), c2);
  if ((threadIdx.x & 63) == 0) runs[threadIdx.x >> 6] = r;
  __syncthreads();
  r = runs[0];
  for (int i = 1; i < kThreads / 64; ++i) r = join(r, runs[i], c2);
  const bool empty = r.s == 0.0f;
  const float log2_s = log2f(r.s);
  if (threadIdx.x == 0) {
    const int64_t t = target_of(a, row);
    float lp = 0.0f;
    if (t != a.ignore_index) {
      lp = __uint_as_float(0x7FC00000u);
      if (t >= 0 && t < a.vocab) lp = log_prob((float)x[t], r, a.scale);
    }
    if (a.logprob) a.logprob[row] = lp;
    if (a.entropy) a.entropy[row] = empty ? 0.0f : kLn2f * (log2_s - r.t / r.s);
    if (a.row_max) a.row_max[row] = r.m;
    if (a.row_sum) a.row_sum[row] = r.s;
  }
  uint64_t below = ~0ull;  // keys are unique: the next alternative is the largest key below the last
  for (int k = 0; k < a.top_k; ++k) {
    uint64_t mine = 0;
    for (int i = threadIdx.x; i < a.vocab; i += kThreads) {
      const uint64_t key = key_of((float)x[i], (uint32_t)i);
      if (key < below && key > mine) mine = key;
    }
    for (int i = 1; i < 64; i <<= 1) {
      const uint64_t other = __shfl_xor((unsigned long long)mine, i);
      mine = other > mine ? other : mine;
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 0) best[threadIdx.x >> 6] = mine;
    __syncthreads();
    below = best[0];
    for (int i = 1; i < kThreads / 64; ++i) below = best[i] > below ? best[i] : below;
    if (threadIdx.x == 0) {
      if (a.top_ids) a.top_ids[row * a.top_k + k] = id_of(below);
      if (a.top_logprobs)
        a.top_logprobs[row * a.top_k + k] = log_prob(value_of(below), r, a.scale);
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) logprobs_grad(LogprobArgs a) {
  const int64_t row = blockIdx.x;
  const T *x = (const T *)a.logits + row * a.row_stride;
  T *grad = (T *)a.grad + row * a.grad_stride;
  const int64_t t = target_of(a, row);
  const bool ignored = t == a.ignore_index;
  float g_lp = a.g_logprob && !ignored ? a.g_logprob[row] : 0.0f;
  const float g_h = a.g_entropy ? a.g_entropy[row] : 0.0f;
  const float s = a.in_sum[row], m = a.in_max[row];
  if (!ignored && g_lp != 0.0f && (t < 0 || t >= a.vocab)) g_lp = __uint_as_float(0x7FC00000u);
  const bool none = (g_lp == 0.0f && g_h == 0.0f) || s == 0.0f;
  const float c2 = a.scale * kLog2e, inv_s = 1.0f / s;
  const float shift = g_h != 0.0f ? a.in_entropy[row] - logf(s) : 0.0f;
  for (int j = blockIdx.y * kThreads + threadIdx.x; j < a.vocab; j += gridDim.y * kThreads) {
    float g = 0.0f;
    if (!none) {
      const float d = exponent((float)x[j], m, c2), p = exp2f(d) * inv_s;
      const float logs = __fmaf_rn(fmaxf(d, -300.0f), kLn2f, shift);
      g = a.scale * ((j == t ? g_lp : 0.0f) - p * __fmaf_rn(g_h, logs, g_lp));
    }
    grad[j] = (T)g;
  }
}

// ------------------------------------------------------------------ host side

// 0 = nothing to do, 1 = go on, negative = refused
int check(const twg_token_logprobs_t *d, bool backward) {
  if (!d || !nn_dtype(d->dtype)) return TWG_E_INVALID_ARG;
  if (d->target_dtype != TWG_DT_I32 && d->target_dtype != TWG_DT_I64) return TWG_E_INVALID_ARG;
  if (d->rows < 0 || d->vocab < 1 || d->vocab > INT32_MAX) return TWG_E_INVALID_ARG;
  if (!(d->scale > 0.0f) || std::isinf(d->scale)) return TWG_E_INVALID_ARG;
  if (!backward && (d->top_k < 0 || d->top_k > TWG_LOGPROBS_MAX_TOP_K || d->top_k > d->vocab))
    return TWG_E_INVALID_ARG;
  if (d->rows == 0) return 0;
  if (d->rows > INT32_MAX) return TWG_E_TOO_LARGE;
  if (!d->logits || !d->targets) return TWG_E_INVALID_ARG;
  const size_t size = (size_t)nn_size(d->dtype);
  if (!aligned_to(d->logits, size) || !aligned_to(d->targets, d->target_dtype == TWG_DT_I64 ? 8 : 4))
    return TWG_E_INVALID_ARG;
  const float *const vectors[] = {d->logprob, d->entropy, d->row_max, d->row_sum, d->top_logprobs, d->g_logprob, d->g_entropy};
  for (const float *v : vectors)
    if (!aligned_to(v, 4)) return TWG_E_INVALID_ARG;
  if (!backward) return aligned_to(d->top_ids, 8) ? 1 : TWG_E_INVALID_ARG;
  if (!d->grad || !d->row_max || !d->row_sum || (d->g_entropy && !d->entropy)) return TWG_E_INVALID_ARG;
  if (!aligned_to(d->grad, size)) return TWG_E_INVALID_ARG;
  // rows of the gradient that share memory: no order among their stores
  if (d->rows > 1 && d->grad_stride < d->vocab && -d->grad_stride < d->vocab) return TWG_E_INVALID_ARG;
  return 1;
}

LogprobArgs args_of(const twg_token_logprobs_t *d) {
  LogprobArgs a{};
  a.logits = d->logits;
  a.targets = d->targets;
  a.rows = d->rows;
  a.row_stride = d->row_stride;
  a.ignore_index = d->ignore_index;
  a.vocab = (int32_t)d->vocab;
  a.top_k = d->top_k;
  a.wide_targets = d->target_dtype == TWG_DT_I64;
  a.scale = d->scale;
  return a;
}

}  // namespace
}  // namespace twg

using namespace twg;

extern "C" {

size_t twg_token_logprobs_scratch_bytes(const twg_token_logprobs_t *) { return 0; }

int twg_token_logprobs(const twg_token_logprobs_t *d, void *, size_t, twg_stream_t stream) {
  int rc = check(d, false);
  if (rc <= 0) return rc;
  if ((rc = ensure_init())) return rc;
  LogprobArgs a = args_of(d);
  a.logprob = d->logprob;
  a.entropy = d->entropy;
  a.row_max = d->row_max;
  a.row_sum = d->row_sum;
  a.top_logprobs = d->top_logprobs;
  a.top_ids = d->top_ids;
  return nn_dispatch(d->dtype, [&](auto t) {
    logprobs_rows<decltype(t)><<<(unsigned)d->rows, kThreads, 0, nn_stream(stream)>>>(a);
    return (int)hipGetLastError();
  });
}

int twg_token_logprobs_backward(const twg_token_logprobs_t *d, twg_stream_t stream) {
  int rc = check(d, true);
  if (rc <= 0) return rc;
  if ((rc = ensure_init())) return rc;
  LogprobArgs a = args_of(d);
  a.in_max = d->row_max;
  a.in_sum = d->row_sum;
  a.in_entropy = d->entropy;
  a.g_logprob = d->g_logprob;
  a.g_entropy = d->g_entropy;
  a.grad = d->grad;
  a.grad_stride = d->grad_stride;
  return nn_dispatch(d->dtype, [&](auto t) {
    const unsigned chunks = (unsigned)((d->vocab + 16 * kThreads - 1) / (16 * kThreads));
    logprobs_grad<decltype(t)><<<dim3((unsigned)d->rows, chunks < 65535 ? chunks : 65535), kThreads, 0,
                                 nn_stream(stream)>>>(a);
    return (int)hipGetLastError();
  });
}

}  // extern "C"
