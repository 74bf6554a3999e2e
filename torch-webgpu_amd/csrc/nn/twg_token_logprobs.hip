// Log probabilities of given tokens, the rows' entropies and top alternatives, and the
// gradient with respect to the logits.
//
//   m = max x, s = sum e^(c (x - m)), logprob = c (x_t - m) - log s,
//   entropy = log s - (1/s) sum e^(c (x - m)) c (x - m)
//   grad_j = c (g_lp ([j = t] - p_j) - g_H p_j (log p_j + entropy)),  p_j = e^(c (x_j - m)) / s
//
// The forward pass reads the logits once: every lane keeps a running maximum and the two sums
// relative to it, every wavefront a sorted list of its best alternatives, one per lane.  A row is
// one workgroup's, or one wavefront's if it is short; few long rows are split over
// several workgroups, whose results a second kernel joins.
//
// Long rows are bound by memory and by vector instructions at nearly the same time: an element costs 5.5
// (widen, maximum, multiply-add, exponential, sum, weighted sum), so that 2-byte elements at 6 TB/s keep
// the vector units busy for three quarters of the time.  4096 x 131072: bfloat16 with 5
// alternatives 176 us (6.1 TB/s), float32 314 us (6.8 TB/s).  Rows of a few thousand elements are
// bound by the chain of a row's own steps: first maxima, lists, join.  The backward pass takes 183 us for
// 2048 x 151643 bfloat16, a quarter of the rows without a gradient (5.9 TB/s).
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
  int32_t splits;        // workgroups per row
  float scale;
  float *logprob, *entropy, *row_max, *row_sum, *top_logprobs;
  int64_t *top_ids;
  uint64_t *scratch;  // with splits > 1: [rows][splits][top_k] keys, then [rows][splits] Run
  const float *g_logprob, *g_entropy;
  const float *in_max, *in_sum, *in_entropy;
  void *grad;
  int64_t grad_stride;
};

__device__ __forceinline__ int64_t target_of(const LogprobArgs &a, int64_t row) {
  return a.wide_targets ? ((const int64_t *)a.targets)[row] : (int64_t)((const int32_t *)a.targets)[row];
}

// Order of the alternatives as one number: the value (-0 as +0, NaN on top), then the lower
// id.  0 is below every key.
__device__ __forceinline__ uint32_t rank_of(float x) {
  const uint32_t b = __float_as_uint(x + 0.0f);
  return x != x ? 0xFFFFFFFFu : b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of_rank(uint32_t v) {
  if (v == 0xFFFFFFFFu) return __uint_as_float(0x7FC00000u);
  return __uint_as_float(v & 0x80000000u ? v ^ 0x80000000u : ~v);
}
__device__ __forceinline__ uint64_t key_of(float x, uint32_t id) { return (uint64_t)rank_of(x) << 32 | (uint32_t)~id; }
__device__ __forceinline__ float value_of(uint64_t key) { return value_of_rank((uint32_t)(key >> 32)); }
__device__ __forceinline__ uint32_t id_of(uint64_t key) { return ~(uint32_t)key; }

// A running softmax sum in base 2: with b = base(m), s = sum 2^(c2 x - b) and
// t = sum 2^(c2 x - b) (c2 x - b), c2 = scale log2 e.  c2 x - b is one fused multiply-add, rounded
// once.  base(m) is c2 m rounded to binary32; the rounding is the same in every term and
// cancels.  It is kept within +-1e37, so that 2^(c2 x - b) stays finite arithmetic where the largest
// entry so far is -inf or near the type's lowest value: such entries then add 0.
// A row of nothing else, and one with infinities or NaN, is recognised by its
// sum and done again by slow_row().
struct Run {
  float m, s, t;
};

__device__ __forceinline__ float base_of(float m, float c2) { return fminf(fmaxf(m * c2, -1e37f), 1e37f); }
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

__device__ __forceinline__ Run join(const Run &a, const Run &b, float c2) {
  const bool swap = b.m > a.m;
  const float m = swap ? b.m : a.m;
  const float hs = swap ? b.s : a.s, ht = swap ? b.t : a.t, ls = swap ? a.s : b.s, lt = swap ? a.t : b.t;
  const float d = fmaxf(base_of(swap ? a.m : b.m, c2) - base_of(m, c2), -300.0f), f = exp2_fast(d);
  return Run{m, __fmaf_rn(f, ls, hs), __fmaf_rn(f, __fmaf_rn(d, ls, lt), ht)};
}

// One value from the 64 lanes' in all of them, by moves within rows of 16 lanes and across them
// (DPP); `none` takes the place of lanes that a move does not reach.
template <typename Op>
__device__ __forceinline__ uint32_t over_lanes(uint32_t v, uint32_t none, Op op) {
#define TWG_STEP(ctrl, rows) v = op(v, (uint32_t)__builtin_amdgcn_update_dpp((int)none, (int)v, ctrl, rows, 0xF, false))
  TWG_STEP(0x111, 0xF);  // row_shr:1
  TWG_STEP(0x112, 0xF);  // row_shr:2
  TWG_STEP(0x114, 0xF);  // row_shr:4
  TWG_STEP(0x118, 0xF);  // row_shr:8: lane 15 of each row has the row's
  TWG_STEP(0x142, 0xA);  // row_bcast:15
  TWG_STEP(0x143, 0xC);  // row_bcast:31: lane 63 has all
#undef TWG_STEP
  return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}
__device__ __forceinline__ uint32_t max_of_lanes(uint32_t v) {
  return over_lanes(v, 0, [](uint32_t a, uint32_t b) { return max(a, b); });
}
__device__ __forceinline__ float fmax_of_lanes(float v) {
  return __uint_as_float(over_lanes(__float_as_uint(v), 0xFF800000u, [](uint32_t a, uint32_t b) {
    return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
  }));
}
__device__ __forceinline__ float sum_of_lanes(float v) {
  return __uint_as_float(over_lanes(__float_as_uint(v), 0, [](uint32_t a, uint32_t b) {
    return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
  }));
}

// The lanes' sums against the largest entry of all.
__device__ __forceinline__ Run join_lanes(const Run &r, float c2) {
  const float m = fmax_of_lanes(r.m);
  const float d = fmaxf(base_of(r.m, c2) - base_of(m, c2), -300.0f), f = exp2_fast(d);
  return Run{m, sum_of_lanes(f * r.s), sum_of_lanes(f * __fmaf_rn(d, r.s, r.t))};
}

// What a row's results are computed from: s against the true maximum, in base e.
struct RowStats {
  float m, s, log_s, entropy;
};
__device__ __forceinline__ RowStats stats_of(const Run &r, float c2) {
  if (r.s == 0.0f) return RowStats{r.m, 0.0f, 0.0f, 0.0f};
  const float shift = __fmaf_rn(r.m, c2, -base_of(r.m, c2)), l = log2f(r.s);
  return RowStats{r.m, r.s * exp2_fast(-shift), kLn2f * (l - shift), kLn2f * (l - r.t / r.s)};
}
// Whether the sums say what they should: 1 or more (less the rounding of base(m)) and finite, or 0
// in a row of -inf.
__device__ __forceinline__ bool plain_row(const Run &r) {
  return r.m == -INFINITY ? r.s == 0.0f : r.s >= 0.5f && r.s < INFINITY;
}
// (in base e: an entry of the type's lowest value times log2 e would leave binary32's range)
__device__ __forceinline__ float log_prob(float x, const RowStats &r, float scale) {
  return r.s == 0.0f ? -INFINITY : (x - r.m) * scale - r.log_s;
}

template <typename T>
__device__ __forceinline__ void put_row(const LogprobArgs &a, int64_t row, const RowStats &r) {
  const int64_t t = target_of(a, row);
  float lp = 0.0f;
  if (t != a.ignore_index) {
    lp = __uint_as_float(0x7FC00000u);
    if (t >= 0 && t < a.vocab) lp = log_prob((float)((const T *)a.logits)[row * a.row_stride + t], r, a.scale);
  }
  if (a.logprob) a.logprob[row] = lp;
  if (a.entropy) a.entropy[row] = r.s == 0.0f ? 0.0f : r.entropy;
  if (a.row_max) a.row_max[row] = r.m;
  if (a.row_sum) a.row_sum[row] = r.s;
}
__device__ __forceinline__ void put_top(const LogprobArgs &a, int64_t row, int k, uint64_t key, const RowStats &r) {
  if (a.top_ids) a.top_ids[row * a.top_k + k] = id_of(key);
  if (a.top_logprobs) a.top_logprobs[row * a.top_k + k] = log_prob(value_of(key), r, a.scale);
}

// (fmaxf would leave NaN out)
__device__ __forceinline__ float max_or_nan(float a, float b) { return a != a || a > b ? a : b; }

// Any row, by its definition: one pass for the maximum, one for the sums, one for each alternative.
// For rows that the single pass cannot do: nothing but entries near the type's limits,
// infinities, NaN.  `room`: LDS for one value per wavefront, two of them.
template <typename T, int WAVES>
__device__ void slow_row(const LogprobArgs &a, int64_t row, uint64_t (*room)[WAVES]) {
  const T *x = (const T *)a.logits + row * a.row_stride;
  const int wave = threadIdx.x >> 6;
  float *f0 = (float *)room[0], *f1 = (float *)room[1];
  float m = -INFINITY;
  for (int i = threadIdx.x; i < a.vocab; i += 64 * WAVES) m = max_or_nan(m, (float)x[i]);
  for (int i = 1; i < 64; i <<= 1) m = max_or_nan(m, __shfl_xor(m, i));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) f0[wave] = m;
  __syncthreads();
  for (int i = 0; i < WAVES; ++i) m = max_or_nan(m, f0[i]);
  float s = 0.0f, t = 0.0f;
  for (int i = threadIdx.x; i < a.vocab; i += 64 * WAVES) {
    const float v = (float)x[i];
    if (v == -INFINITY) continue;
    const float d = (v - m) * a.scale, e = expf(d);
    s += e;
    t = __fmaf_rn(e, fmaxf(d, -300.0f), t);
  }
  for (int i = 1; i < 64; i <<= 1) {
    s += __shfl_xor(s, i);
    t += __shfl_xor(t, i);
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 0) {
    f0[wave] = s;
    f1[wave] = t;
  }
  __syncthreads();
  s = f0[0];
  t = f1[0];
  for (int i = 1; i < WAVES; ++i) {
    s += f0[i];
    t += f1[i];
  }
  const float log_s = logf(s);
  const RowStats r{m, s, log_s, log_s - t / s};
  if (threadIdx.x == 0) put_row<T>(a, row, r);
  uint64_t below = ~0ull;  // keys are unique: the next alternative is the largest key below the last
  for (int k = 0; k < a.top_k; ++k) {
    uint64_t mine = 0;
    for (int i = threadIdx.x; i < a.vocab; i += 64 * WAVES) {
      const uint64_t key = key_of((float)x[i], (uint32_t)i);
      if (key < below && key > mine) mine = key;
    }
    for (int i = 1; i < 64; i <<= 1) {
      const uint64_t other = __shfl_xor((unsigned long long)mine, i);
      mine = other > mine ? other : mine;
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 0) room[0][wave] = mine;
    __syncthreads();
    below = room[0][0];
    for (int i = 1; i < WAVES; ++i) below = room[0][i] > below ? room[0][i] : below;
    if (threadIdx.x == 0) put_top(a, row, k, below, r);
  }
}

// ---- a wavefront's best alternatives: lane l holds the l-th best key, 0 where there is none yet

__device__ __forceinline__ uint64_t read_lane(uint64_t v, int lane) {
  const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)v, lane);
  const uint32_t hi = __builtin_amdgcn_readlane((uint32_t)(v >> 32), lane);
  return (uint64_t)hi << 32 | lo;
}
__device__ __forceinline__ int lanes_below(uint64_t mask) {
  return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
}

// LDS written by some lanes of a wavefront and read by others of the same one: in order by itself,
// the compiler has to keep it so.
__device__ __forceinline__ void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// Merge n waiting keys (in LDS) with a wavefront's list `mine`: every key's place is the number of
// larger ones.  About 10 instructions a key that do not depend on each other; putting the
// keys into place one after the other was 25 in one long chain.  `room`: LDS for 64 keys.
__device__ __forceinline__ uint64_t merged_list(uint64_t mine, const uint64_t *wait, int n, uint64_t *room, int lane) {
  wave_fence();
  const uint64_t key = lane < n ? wait[lane] : 0;
  int place = 0, mine_place = lane;
  for (int i = 0; i < n; ++i) {
    const uint64_t other = read_lane(key, i);
    const int larger = __popcll(__ballot(mine > other));
    place += (other > key ? 1 : 0) + (lane == i ? larger : 0);
    mine_place += other > mine ? 1 : 0;
  }
  const int all = __popcll(__ballot(mine != 0)) + n;
  if (mine && mine_place < 64) room[mine_place] = mine;
  if (key && place < 64) room[place] = key;
  wave_fence();
  return lane < all ? room[lane] : 0;
}

// A value that at least k lanes' values reach, and the upper half of the k-th largest of them: bit
// by bit, the largest that k lanes still reach.
__device__ __forceinline__ uint32_t kth_of_lanes(uint32_t v, int k) {
  uint32_t found = 0;
  for (uint32_t bit = 0x80000000u; bit >= 0x10000u; bit >>= 1)
    if (__popcll(__ballot(v >= (found | bit))) >= k) found |= bit;
  return found;
}

// the larger of three in one instruction (fmaxf first makes sure of each operand)
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}

constexpr int kUnroll = 4;  // packs of 16 bytes a lane loads before it looks at the first

// One row, or the part `split` of it, by one workgroup of WAVES wavefronts.
template <typename T, int WAVES, bool TOP>
__global__ void __launch_bounds__(64 * WAVES) logprobs_rows(LogprobArgs a) {
  constexpr int E = 16 / (int)sizeof(T), N = E * kUnroll, THREADS = 64 * WAVES;
  __shared__ Run runs[WAVES];
  __shared__ uint64_t room[2][WAVES];
  __shared__ uint32_t floors[WAVES];
  __shared__ int found;
  __shared__ uint64_t waiting[TOP ? WAVES : 1][64], merged[TOP ? WAVES : 1][64];
  __shared__ Pack<T, E> packed[TOP ? WAVES : 1][64];
  __shared__ int from[TOP ? WAVES : 1][64];
  __shared__ uint64_t lists[TOP ? WAVES * TWG_LOGPROBS_MAX_TOP_K : 1], joined[TOP ? TWG_LOGPROBS_MAX_TOP_K : 1];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, k = a.top_k;
  const int64_t row = a.splits == 1 ? blockIdx.x : blockIdx.x / a.splits;
  const int split = a.splits == 1 ? 0 : blockIdx.x - (int)row * a.splits;
  const T *x = (const T *)a.logits + row * a.row_stride;
  const float c2 = a.scale * kLog2e;

  // elements before the first 16-byte boundary, whole packs, elements behind them
  const int lead = (int)((-(uintptr_t)x & 15) / sizeof(T));
  const int head = lead < a.vocab ? lead : a.vocab;
  const int packs = (a.vocab - head) / E, tail = a.vocab - head - packs * E;
  const int per = (packs + a.splits - 1) / a.splits;
  const int first = min(split * per, packs), last = min(first + per, packs);
  const Pack<T, E> *body = (const Pack<T, E> *)(x + head);

  Run r{-INFINITY, 0.0f, 0.0f};
  float b = base_of(r.m, c2);
  uint64_t mine = 0, kth = 0;  // this lane's alternative, and the wavefront's last that counts
  int pending = 0;             // keys in `waiting`

  bool masked = false;  // the same in all lanes
  // n values of this lane, `top` the largest, into its running sums
  auto add = [&](const float *v, float top, auto n) {
    if (top > r.m) {
      const float nb = base_of(top, c2), d = fmaxf(b - nb, -300.0f), f = exp2_fast(d);
      r.t = f * __fmaf_rn(d, r.s, r.t);
      r.s *= f;
      r.m = top;
      b = nb;
    }
    // An entry of -inf makes the product 0 * -inf: from the first one on the wavefront keeps
    // its exponents finite, one instruction more for each element.  A lane without an element counts as one: at
    // a ragged end, and for the first wavefront of a row that does not begin on a pack's boundary.
    const Run before = r;
    if (!masked) {
#pragma unroll
      for (int j = 0; j < decltype(n)::value; ++j) {
        const float d = __fmaf_rn(v[j], c2, -b), e = exp2_fast(d);
        r.s += e;
        r.t = __fmaf_rn(e, d, r.t);
      }
      masked = __ballot(r.t != r.t) != 0;
      if (!masked) return;
      r = before;
    }
    float base = b;
    asm("" : "+v"(base));  // computed anew: the exponents above are not kept in registers for this
#pragma unroll
    for (int j = 0; j < decltype(n)::value; ++j) {
      const float d = __fmaf_rn(v[j], c2, -base), e = exp2_fast(d);
      r.s += e;
      r.t = __fmaf_rn(e, fmaxf(d, -300.0f), r.t);
    }
  };
  auto merge = [&]() {
    mine = merged_list(mine, waiting[TOP ? wave : 0], pending, merged[TOP ? wave : 0], lane);
    kth = read_lane(mine, k - 1);
    pending = 0;
  };
  // the few single elements at an end of the row: the first lanes of the first wavefront
  auto edge = [&](int start, int n) {
    if (wave != 0 || n == 0) return;
    const bool has = lane < n;
    const float v = has ? (float)x[start + lane] : -INFINITY;
    add(&v, v, std::integral_constant<int, 1>());
    if (TOP) {
      if (has) waiting[0][pending + lane] = key_of(v, (uint32_t)(start + lane));
      pending += n;
    }
  };
  // The bar for alternatives: candidates are above it; while `any`, -inf counts, too.
  const int share = TOP ? (k + WAVES - 1) / WAVES : 1;
  uint32_t floor = 0;  // a rank that at least k elements of the row reach, as far as known
  bool any = true;
  float bar = -INFINITY;
  auto lowest_floor = [&]() {
    uint32_t f = 0xFFFFFFFFu;
#pragma unroll
    for (int w = 0; w < WAVES; ++w)
      f = min(f, __hip_atomic_load(&floors[w], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP));
    return (uint32_t)__builtin_amdgcn_readfirstlane((int)f);
  };
  auto raise_floor = [&]() {
    const uint32_t at = (uint32_t)(read_lane(mine, share - 1) >> 32);
    if (WAVES > 1 && lane == 0 && at > floors[wave])
      __hip_atomic_store(&floors[wave], at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
  };
  auto set_bar = [&]() {
    const uint32_t least = max(floor, kth ? (uint32_t)(kth >> 32) + 1 : 0u);
    any = least <= rank_of(-INFINITY);
    // the value one rank below (0x7FFFFFFF, which would be -0, is not in use)
    bar = any ? -INFINITY : value_of_rank(least - (least == 0x80000000u ? 2 : 1));
  };
  // kUnroll packs of this lane, the first one pack `p` + threadIdx.x
  // The next step's packs are on their way while a lane looks at one step's (517 rows of 131072 float32
  // with 5 alternatives 67 -> 53 us, 4096 rows of 8192 bfloat16 without 18.6 -> 15.3).  With 16-bit
  // elements and alternatives together it takes 102 registers instead of 87, and 4 wavefronts per SIMD are left of
  // 5: 1100 rows of 50257 with 20 alternatives 39 -> 45 us, 4096 rows 109 -> 114; only 517 rows, whose
  // workgroups leave room anyway, gain (28.9 -> 27.9).
  constexpr bool AHEAD = sizeof(T) == 4 || !TOP;
  Pack<T, E> coming[kUnroll];
  auto fetch = [&](int p, auto whole) {
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int at = p + u * THREADS + (int)threadIdx.x;
      coming[u] = load_pack<true>(body + (decltype(whole)::value ? at : min(at, last - 1)));
    }
  };
  auto step = [&](int p, auto whole) {
    Pack<T, E> raw[kUnroll];
    bool in[kUnroll];
    if (!AHEAD) fetch(p, whole);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      raw[u] = coming[u];
      in[u] = decltype(whole)::value || p + u * THREADS + (int)threadIdx.x < last;
    }
    if (AHEAD && decltype(whole)::value && p + kUnroll * THREADS < last) fetch(p + kUnroll * THREADS, std::false_type());
    float v[N], most[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
#pragma unroll
      for (int j = 0; j < E; ++j) v[u * E + j] = in[u] ? (float)raw[u].v[j] : -INFINITY;
      most[u] = max3(v[u * E], v[u * E + 1], v[u * E + 2]);
#pragma unroll
      for (int j = 3; j < E; j += 2) most[u] = max3(most[u], v[u * E + j], v[u * E + (j + 1 < E ? j + 1 : j)]);
    }
    float top = most[0];
#pragma unroll
    for (int u = 1; u < kUnroll; ++u) top = fmaxf(top, most[u]);
    add(v, top, std::integral_constant<int, N>());
    if constexpr (TOP) {
      // Which elements may be among the best k.  One of a later step has a higher id than all in
      // the wavefront's list, so it has to be larger than a k-th there.  And at least k elements
      // of the row reach `floor`, the smallest of the wavefronts' `floors`: in its first step
      // each knows a value that ceil(k / WAVES) of its lanes' maxima reach, later the
      // ceil(k / WAVES)-th of its list.
      if (p == first) {
        const uint32_t known = kth_of_lanes(rank_of(top), share);
        if (WAVES > 1) {
          if (lane == 0) floors[wave] = known;
          __syncthreads();
        }
        floor = WAVES > 1 ? lowest_floor() : known;
        set_bar();
      }
      if (any || __ballot(top > bar)) {
        if (WAVES > 1 && p != first) {
          floor = max(floor, lowest_floor());
          set_bar();
        }
        // The packs that hold a candidate go through LDS, so that each lane has one element of them
        // to look at.
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
          const int at = p + u * THREADS + (int)threadIdx.x;
          const uint64_t holds = __ballot(in[u] && (any || most[u] > bar));
          if (!holds) continue;
          if (holds >> lane & 1) {
            const int place = lanes_below(holds);
            packed[wave][place] = raw[u];
            from[wave][place] = at;
          }
          wave_fence();
          const int n = __popcll(holds) * E;
          for (int i = lane; i - lane < n; i += 64) {
            const float e = i < n ? (float)((const T *)packed[wave])[i] : 0.0f;
            const uint64_t key = i < n ? key_of(e, (uint32_t)(head + from[wave][i / E] * E + i % E)) : 0;
            bool cand = key > kth && (any || e > bar);
            uint64_t mask = __ballot(cand);
            if (pending + __popcll(mask) > 64) {
              merge();
              cand = cand && key > kth;
              mask = __ballot(cand);
            }
            if (cand) waiting[wave][pending + lanes_below(mask)] = key;
            pending += __popcll(mask);
          }
          wave_fence();
        }
        merge();
        raise_floor();
        set_bar();
      }
    }
  };

  if (split == 0) edge(0, head);
  int p = first;
  if (AHEAD && p < last) fetch(p, std::false_type());
  for (; p + kUnroll * THREADS <= last; p += kUnroll * THREADS) {
    step(p, std::true_type());
  }
  if (p < last) step(p, std::false_type());
  if (split == a.splits - 1) edge(a.vocab - tail, tail);
  if (TOP && pending) merge();

  // join the lanes, then the wavefronts
  r = join_lanes(r, c2);
  if (WAVES > 1) {
    if (lane == 0) runs[wave] = r;
    if (TOP) {  // of the lists only what reaches the last floor is looked at
      if (first == last && lane == 0) floors[wave] = 0;
      raise_floor();
      if (threadIdx.x == 0) found = 0;
      if ((int)threadIdx.x < k) joined[threadIdx.x] = 0;
    }
    __syncthreads();
    r = runs[0];
#pragma unroll
    for (int i = 1; i < WAVES; ++i) r = join(r, runs[i], c2);
    if (TOP) {  // the place of each key among all of them
      if (lane < k && mine && (uint32_t)(mine >> 32) >= lowest_floor())
        lists[__hip_atomic_fetch_add(&found, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP)] = mine;
      __syncthreads();
      const int n = found;
      if ((int)threadIdx.x < n) {
        const uint64_t key = lists[threadIdx.x];
        int place = 0;
        for (int i = 0; i < n; ++i) place += lists[i] > key;
        if (place < k) joined[place] = key;
      }
      __syncthreads();
      mine = lane < k ? joined[lane] : 0;
    }
  }
  if (a.splits > 1) {
    const int64_t part = blockIdx.x;
    if (TOP && (int)threadIdx.x < k) a.scratch[part * k + threadIdx.x] = mine;
    if (threadIdx.x == 0) {
      Run *to = (Run *)(a.scratch + a.rows * a.splits * k) + part;
      *to = r;
    }
    return;
  }
  if (!plain_row(r)) {  // the same in all threads
    slow_row<T, WAVES>(a, row, room);
    return;
  }
  const RowStats st = stats_of(r, c2);
  if (threadIdx.x == 0) put_row<T>(a, row, st);
  if (TOP && (int)threadIdx.x < k) put_top(a, row, threadIdx.x, mine, st);
}

constexpr int kMaxSplits = 64;  // one lane each when they are joined

// The parts of a row, joined by one workgroup.
template <typename T>
__global__ void __launch_bounds__(kThreads) logprobs_join(LogprobArgs a) {
  constexpr int WAVES = kThreads / 64;
  __shared__ uint64_t lists[kMaxSplits * TWG_LOGPROBS_MAX_TOP_K];
  __shared__ uint64_t room[2][WAVES];
  __shared__ Run whole;
  const int64_t row = blockIdx.x;
  const int k = a.top_k, splits = a.splits;
  for (int i = threadIdx.x; i < splits * k; i += kThreads) lists[i] = a.scratch[row * splits * k + i];
  const float c2 = a.scale * kLog2e;
  if (threadIdx.x < 64) {
    const Run *parts = (const Run *)(a.scratch + a.rows * splits * k) + row * splits;
    Run r{-INFINITY, 0.0f, 0.0f};
    if ((int)threadIdx.x < splits) r = parts[threadIdx.x];
    r = join_lanes(r, c2);
    if (threadIdx.x == 0) whole = r;
  }
  __syncthreads();
  if (!plain_row(whole)) {
    slow_row<T, WAVES>(a, row, room);
    return;
  }
  if (threadIdx.x >= 64) return;
  const RowStats st = stats_of(whole, c2);
  const int lane = threadIdx.x;
  if (lane == 0) put_row<T>(a, row, st);
  // Lane l stands at the next entry of part l's list.  The parts follow each other in the row, so
  // of equal values the lowest lane's has the lowest id.
  int at = 0;
  uint64_t next = lane < splits && k ? lists[lane * k] : 0, mine = 0;
  for (int i = 0; i < k; ++i) {
    const uint32_t rank = (uint32_t)(next >> 32);
    const int from = __builtin_ctzll(__ballot(rank == max_of_lanes(rank)));
    const uint64_t key = read_lane(next, from);
    if (lane == i) mine = key;
    if (lane == from) next = ++at < k ? lists[lane * k + at] : 0;
  }
  if (lane < k) put_top(a, row, lane, mine, st);
}

constexpr int kGradPacks = 2;  // packs of 16 bytes per lane

// One workgroup: a stretch of one row.  What the elements share is the same for the whole
// workgroup; each element costs one exponential.
template <typename T, bool STREAM>
__global__ void __launch_bounds__(kThreads) logprobs_grad(LogprobArgs a) {
  constexpr int E = 16 / (int)sizeof(T), PER = kGradPacks * kThreads;
  typedef Pack<T, E> Vec;
  const uint32_t chunks = (uint32_t)a.splits;  // workgroups of a row, one behind the other in memory
  const int64_t row = blockIdx.x / chunks;
  const int first_chunk = (int)(blockIdx.x - (uint32_t)row * chunks);
  const T *x = (const T *)a.logits + row * a.row_stride;
  T *grad = (T *)a.grad + row * a.grad_stride;
  const int64_t t = target_of(a, row);
  const bool ignored = t == a.ignore_index;
  float g_lp = a.g_logprob && !ignored ? a.g_logprob[row] : 0.0f;
  const float g_h = a.g_entropy ? a.g_entropy[row] : 0.0f;
  const float s = a.in_sum[row], m = a.in_max[row];
  if (!ignored && g_lp != 0.0f && (t < 0 || t >= a.vocab)) g_lp = __uint_as_float(0x7FC00000u);
  const bool none = (g_lp == 0.0f && g_h == 0.0f) || s == 0.0f;
  // grad = c [j = t] g_lp - 2^d (d h + l) with d = log2 e c (x - m), h = c g_H ln 2 / s,
  // l = c (g_lp + g_H (entropy - log s)) / s
  const float c2 = a.scale * kLog2e, by_s = a.scale / s, hit = a.scale * g_lp;
  const float l = by_s * (g_h != 0.0f ? __fmaf_rn(g_h, a.in_entropy[row] - logf(s), g_lp) : g_lp);
  const float h = by_s * g_h * kLn2f;
  auto one = [&](float v, int j) {
    const float d = (v - m) * c2, p = exp2_fast(d);
    const float g = -p * __fmaf_rn(fmaxf(d, -300.0f), h, l);
    return j == t ? g + hit : g;
  };
  // elements before the gradient's first line of 128 bytes, whole packs, elements behind them: a line that
  // two workgroups share, on different XCDs, would be written in two pieces
  const int lead = (int)((-(uintptr_t)grad & 127) / sizeof(T));
  const int head = lead < a.vocab ? lead : a.vocab;
  const int packs = (a.vocab - head) / E, tail = a.vocab - head - packs * E;
  const bool alike = (((uintptr_t)x ^ (uintptr_t)grad) & 15) == 0;  // the logits' packs are aligned, too
  for (int chunk = first_chunk; chunk * PER < packs || chunk == 0; chunk += chunks) {
    if (chunk == 0 && (int)threadIdx.x < head + tail) {
      const int j = (int)threadIdx.x < head ? threadIdx.x : a.vocab - tail + (int)threadIdx.x - head;
      grad[j] = (T)(none ? 0.0f : one((float)x[j], j));
    }
    Vec v[kGradPacks];
#pragma unroll
    for (int u = 0; u < kGradPacks; ++u) {
      const int p = chunk * PER + u * kThreads + threadIdx.x;
      if (p >= packs || none) continue;
      const T *from = x + head + p * E;
      if (alike) {
        v[u] = load_pack<STREAM>((const Vec *)from);
      } else {
#pragma unroll
        for (int j = 0; j < E; ++j) v[u].v[j] = from[j];
      }
    }
#pragma unroll
    for (int u = 0; u < kGradPacks; ++u) {
      const int p = chunk * PER + u * kThreads + threadIdx.x;
      if (p >= packs) continue;
      Vec o;
#pragma unroll
      for (int j = 0; j < E; ++j) o.v[j] = (T)(none ? 0.0f : one((float)v[u].v[j], head + p * E + j));
      store_pack<STREAM>((Vec *)(grad + head) + p, o);
    }
  }
}

// ------------------------------------------------------------------ host side

// 0 = nothing to do, 1 = go on, negative = refused
int check(const twg_token_logprobs_t *d, bool backward) {
  if (!d || !nn_dtype(d->dtype)) return TWG_E_INVALID_ARG;
  if (d->target_dtype != TWG_DT_I32 && d->target_dtype != TWG_DT_I64) return TWG_E_INVALID_ARG;
  if (d->rows < 0 || d->vocab < 1 || d->vocab > TWG_LOGPROBS_MAX_VOCAB) return TWG_E_INVALID_ARG;
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

struct RowShape {
  int waves;   // wavefronts per workgroup: 1, 4 or 8
  int splits;  // workgroups per row
};

// A row that one wavefront reads in two steps is one wavefront's.  Of longer rows, up to 512 are
// workgroups of 8 wavefronts: with alternatives (87 registers) the chip holds 2 of those per compute unit, 512
// in all, and one row more would wait for a second generation.  More rows take workgroups of 4, of which
// 5 fit.  16-bit elements, 20 alternatives, 8 and 4 wavefronts: 512 rows of 50257 24 and 28 us, 517 rows
// 35 and 29, 1023 rows 44 and 35; of 131072 38 and 45, 56 and 48, 70 and 57.  float32: 512 rows of 50257 28 and
// 32, 517 rows 32 and 32.  Without alternatives, 256 rows of 131072 16 and 23, 512 rows 26 and 27, 512 rows of
// 50257 16 and 15, 517 rows 20 and 17.  Fewer than 256 rows are split into workgroups of 4 wavefronts that
// read one step of their own at least, about 1024 in all.
RowShape shape_of(const twg_token_logprobs_t *d) {
  const int64_t step = 16 * kUnroll / nn_size(d->dtype) * 64;  // elements a wavefront takes at a time
  if (d->vocab <= 2 * step) return RowShape{1, 1};
  if (d->rows > 512) return RowShape{4, 1};
  if (d->rows >= 256) return RowShape{8, 1};
  int64_t splits = (1024 + d->rows - 1) / d->rows;
  const int64_t steps = (d->vocab + 4 * step - 1) / (4 * step);
  splits = splits < steps ? splits : steps;
  return RowShape{4, (int)(splits < kMaxSplits ? splits : kMaxSplits)};
}

// Rows of one launch: its threads, 256 a row at most and more where a row has several workgroups, have
// to be counted in 32 bits.  More rows go in several launches.
constexpr int64_t kMaxRows = INT64_C(1) << 22;

template <typename Call>
int in_slabs(const twg_token_logprobs_t *d, Call call) {
  const auto past = [](auto *p, int64_t n) { return p ? p + n : p; };
  for (int64_t r = 0; r < d->rows; r += kMaxRows) {
    twg_token_logprobs_t part = *d;
    const int64_t size = nn_size(d->dtype);
    part.rows = d->rows - r < kMaxRows ? d->rows - r : kMaxRows;
    part.logits = static_cast<const char *>(d->logits) + r * d->row_stride * size;
    part.targets = static_cast<const char *>(d->targets) + r * (d->target_dtype == TWG_DT_I64 ? 8 : 4);
    part.logprob = past(d->logprob, r);
    part.entropy = past(d->entropy, r);
    part.row_max = past(d->row_max, r);
    part.row_sum = past(d->row_sum, r);
    part.top_logprobs = past(d->top_logprobs, r * d->top_k);
    part.top_ids = past(d->top_ids, r * d->top_k);
    part.g_logprob = past(d->g_logprob, r);
    part.g_entropy = past(d->g_entropy, r);
    part.grad = past(static_cast<char *>(d->grad), r * d->grad_stride * size);
    if (const int rc = call(&part)) return rc;
  }
  return 0;
}

size_t scratch_of(const twg_token_logprobs_t *d, int splits) {
  if (splits == 1) return 0;
  const size_t parts = (size_t)d->rows * (size_t)splits;
  return (parts * ((size_t)d->top_k * 8 + sizeof(Run)) + 7) / 8 * 8;
}

}  // namespace
}  // namespace twg

using namespace twg;

extern "C" {

size_t twg_token_logprobs_scratch_bytes(const twg_token_logprobs_t *d) {
  if (check(d, false) <= 0) return 0;
  twg_token_logprobs_t last = *d;  // of several launches only the last can have few rows
  if (d->rows > kMaxRows) last.rows = (d->rows - 1) % kMaxRows + 1;
  return scratch_of(&last, shape_of(&last).splits);
}

int twg_token_logprobs(const twg_token_logprobs_t *d, void *scratch, size_t scratch_bytes, twg_stream_t stream) {
  int rc = check(d, false);
  if (rc <= 0) return rc;
  if (d->rows > kMaxRows) {
    if (scratch_bytes < twg_token_logprobs_scratch_bytes(d)) return TWG_E_SCRATCH_SMALL;  // before the first launch
    return in_slabs(d, [&](const twg_token_logprobs_t *part) { return twg_token_logprobs(part, scratch, scratch_bytes, stream); });
  }
  const RowShape shape = shape_of(d);
  if (shape.splits > 1) {
    if (!scratch || scratch_bytes < scratch_of(d, shape.splits)) return TWG_E_SCRATCH_SMALL;
    if (!aligned_to(scratch, 8)) return TWG_E_INVALID_ARG;
  }
  const OnBoundDevice device;
  if ((rc = device.status())) return rc;
  LogprobArgs a = args_of(d);
  a.splits = shape.splits;
  a.scratch = static_cast<uint64_t *>(scratch);
  a.logprob = d->logprob;
  a.entropy = d->entropy;
  a.row_max = d->row_max;
  a.row_sum = d->row_sum;
  a.top_logprobs = d->top_logprobs;
  a.top_ids = d->top_ids;
  const hipStream_t s = nn_stream(stream);
  return nn_dispatch(d->dtype, [&](auto t) {
    using T = decltype(t);
    const unsigned grid = (unsigned)(d->rows * shape.splits);
    const auto go = [&](auto waves) {
      constexpr int W = decltype(waves)::value;
      if (a.top_k)
        logprobs_rows<T, W, true><<<grid, 64 * W, 0, s>>>(a);
      else
        logprobs_rows<T, W, false><<<grid, 64 * W, 0, s>>>(a);
    };
    if (shape.waves == 1) go(std::integral_constant<int, 1>());
    else if (shape.waves == 4) go(std::integral_constant<int, 4>());
    else go(std::integral_constant<int, 8>());
    if (shape.splits > 1) logprobs_join<T><<<(unsigned)d->rows, kThreads, 0, s>>>(a);
    return (int)hipGetLastError();
  });
}

int twg_token_logprobs_backward(const twg_token_logprobs_t *d, twg_stream_t stream) {
  int rc = check(d, true);
  if (rc <= 0) return rc;
  if (d->rows > kMaxRows)
    return in_slabs(d, [&](const twg_token_logprobs_t *part) { return twg_token_logprobs_backward(part, stream); });
  const OnBoundDevice device;
  if ((rc = device.status())) return rc;
  LogprobArgs a = args_of(d);
  a.in_max = d->row_max;
  a.in_sum = d->row_sum;
  a.in_entropy = d->entropy;
  a.g_logprob = d->g_logprob;
  a.g_entropy = d->g_entropy;
  a.grad = d->grad;
  a.grad_stride = d->grad_stride;
  return nn_dispatch(d->dtype, [&](auto t) {
    using T = decltype(t);
    const int64_t per = kGradPacks * kThreads * 16 / (int)sizeof(T), most = INT32_MAX / kThreads / d->rows;
    const int64_t chunks = (d->vocab + per - 1) / per;
    a.splits = (int32_t)(chunks < most ? chunks : most);
    const unsigned grid = (unsigned)(d->rows * a.splits);
    if (2.0 * (double)d->rows * (double)d->vocab * sizeof(T) > (double)kStreamBytes)
      logprobs_grad<T, true><<<grid, kThreads, 0, nn_stream(stream)>>>(a);
    else
      logprobs_grad<T, false><<<grid, kThreads, 0, nn_stream(stream)>>>(a);
    return (int)hipGetLastError();
  });
}

}  // extern "C"
