// The transformer-step entry points called while another device than the library's is current: every
// launch has to find device 0 current, and the caller has to find its own again.  This program brings
// HIP functions of its own, which stand before the runtime's, so it needs no GPU: nothing is launched.
#include <hip/hip_runtime_api.h>

#include <cstdint>
#include <cstdio>
#include <cstring>

#include "twg.h"

static int current = 0, launches = 0, elsewhere = 0;
static hipStream_t last_stream = nullptr;
static dim3 g_grid, g_block;
static size_t g_shared = 0;
static hipStream_t g_stream = nullptr;
static char own_stream, callers_stream, array[512];

extern "C" {
hipError_t hipGetDeviceCount(int *n) { *n = 2; return hipSuccess; }
hipError_t hipGetDevice(int *d) { *d = current; return hipSuccess; }
hipError_t hipSetDevice(int d) { current = d; return hipSuccess; }
hipError_t hipGetLastError(void) { return hipSuccess; }
hipError_t hipGetDevicePropertiesR0600(hipDeviceProp_tR0600 *p, int) {
  std::memset(p, 0, sizeof *p);
  p->multiProcessorCount = 256;
  return hipSuccess;
}
hipError_t hipStreamCreateWithFlags(hipStream_t *s, unsigned) {
  *s = reinterpret_cast<hipStream_t>(&own_stream);
  return hipSuccess;
}
hipError_t hipEventCreateWithFlags(hipEvent_t *e, unsigned) {
  *e = reinterpret_cast<hipEvent_t>(&own_stream);
  return hipSuccess;
}
hipError_t hipGetSymbolAddress(void **p, const void *) {
  *p = reinterpret_cast<void *>((reinterpret_cast<uintptr_t>(array) + 255) / 256 * 256);
  return hipSuccess;
}
hipError_t __hipPushCallConfiguration(dim3 grid, dim3 block, size_t shared, hipStream_t s) {
  g_grid = grid, g_block = block, g_shared = shared, g_stream = s;
  return hipSuccess;
}
hipError_t __hipPopCallConfiguration(dim3 *grid, dim3 *block, size_t *shared, hipStream_t *s) {
  *grid = g_grid, *block = g_block, *shared = g_shared, *s = g_stream;
  return hipSuccess;
}
hipError_t hipLaunchKernel(const void *, dim3, dim3, void **, size_t, hipStream_t s) {
  ++launches;
  elsewhere += current != 0;
  last_stream = s;
  return hipSuccess;
}
}

static int failures = 0;
static void expect(bool ok, const char *what, const char *where) {
  if (ok) return;
  ++failures;
  std::printf("%s: %s\n", where, what);
}

template <typename Call>
static void check(const char *name, Call call) {
  struct { twg_stream_t given; hipStream_t want; } const streams[] = {
      {nullptr, reinterpret_cast<hipStream_t>(&own_stream)},
      {TWG_STREAM_NULL, nullptr},
      {reinterpret_cast<twg_stream_t>(&callers_stream), reinterpret_cast<hipStream_t>(&callers_stream)}};
  for (int device = 1; device >= 0; --device)
    for (const auto &s : streams) {
      current = device;
      launches = elsewhere = 0;
      expect(call(s.given) == 0, "refused", name);
      expect(launches > 0, "nothing launched", name);
      expect(elsewhere == 0, "launched on another device", name);
      expect(last_stream == s.want, "on another stream", name);
      expect(current == device, "the caller's device is another afterwards", name);
    }
}

int main() {
  void *const p = reinterpret_cast<void *>(uintptr_t(1) << 20);  // no launch, so nothing touches it
  twg_norm_rope_t r{};
  r.dtype = r.weight_dtype = TWG_DT_F32;
  r.position_dtype = TWG_DT_I64;
  r.norm = r.n_axes = 1;
  r.head_dim = r.rot_dim = 64;
  r.eps = 1e-6f;
  r.batch = r.tokens = 1;
  r.positions = p;
  r.inv_freq = static_cast<const float *>(p);
  r.part[0].heads = 1;
  r.part[0].x = r.part[0].dy = p;
  r.part[0].out = r.part[0].dweight = p;
  for (int i = 0; i < 3; ++i) r.part[0].x_stride[i] = r.part[0].dy_stride[i] = r.part[0].out_stride[i] = 64;
  twg_token_logprobs_t l{};
  l.dtype = TWG_DT_F32;
  l.target_dtype = TWG_DT_I64;
  l.rows = 1;
  l.vocab = l.row_stride = l.grad_stride = 100000;
  l.logits = l.targets = p;
  l.scale = 1.0f;
  l.top_k = 2;
  l.row_max = l.row_sum = l.entropy = static_cast<float *>(p);
  l.g_logprob = l.g_entropy = static_cast<const float *>(p);
  l.grad = p;
  twg_iter_t it{};
  it.ndim = 1;
  it.numel = it.shape[0] = 100;
  for (int o = 0; o < 3; ++o) it.stride[o][0] = 1;

  const size_t room = size_t(1) << 30;
  check("norm_rope", [&](twg_stream_t s) { return twg_norm_rope(&r, s); });
  check("norm_rope_backward", [&](twg_stream_t s) { return twg_norm_rope_backward(&r, p, room, s); });
  check("token_logprobs", [&](twg_stream_t s) { return twg_token_logprobs(&l, p, room, s); });
  check("token_logprobs_backward", [&](twg_stream_t s) { return twg_token_logprobs_backward(&l, s); });
  check("dropout", [&](twg_stream_t s) { return twg_dropout(p, p, nullptr, TWG_DT_F32, 0.5, 1, 0, nullptr, &it, s); });
  if (failures == 0) std::printf("every launch on device 0\n");
  return failures != 0;
}
