// RMS norm of each query and key head and the rotation of its pairs by position, in one pass
// over the heads; one or several position axes; forward and backward.
//
//   forward   r = (mean x^2 + eps)^(-1/2), u = x r, z = u w, y = R(a) z
//   backward  dz = R(-a) dy, dw = sum dz u, g = dz w, dx = r (g - u mean(g u))
//
// R(a) turns pair i of a head by a_i = position[axis(i)] * inv_freq[i].  The angles of a token
// are the same for all of its heads: a workgroup computes them once for its tokens and keeps
// cosines and sines in LDS.
//
// Bound by memory: 16384 tokens x 40 heads of 128 in bfloat16 (336 MB in and out) take 64 us forward and, with 503 MB,
// 101 us backward (and 6 us for the weights' sums): 5.3 and 5.0 TB/s of the 6.7 that a large copy
// reaches.  The vector units are busy for half of that time (rotation, widening and rounding of 16 elements a
// lane), which 4 wavefronts per SIMD do not hide entirely.  Calls below 20 us are bound by the chain
// position -> angle -> barrier -> head and by the launch.
#include "twg_nn.h"

namespace twg {
namespace {

constexpr int kMaxPairs = TWG_ROPE_MAX_HEAD_DIM / 2;
constexpr int kTrigRoom = 1024;  // cosines (and sines) a workgroup holds: 8 KiB of LDS
constexpr int kMaxTile = 16;     // tokens a workgroup takes at most
constexpr int kSteps = 4;        // heads a group takes in a piece of work where there are many

// Queries and keys are two parts, each with workgroups of its own: what differs between the parts
// is the same for a whole workgroup.
struct PartArgs {
  const void *x, *dy, *weight;
  void *out;
  float *partial;               // backward: [grid][head_dim] sums of dz u, or NULL
  int64_t xs[3], ys[3], os[3];  // batch, token, head
  int32_t heads;
  int32_t tile;   // tokens of one piece of work
  int32_t split;  // pieces that share a tile's heads
  int32_t work;   // pieces
  int32_t grid;   // workgroups: piece i, i + grid, ... are one workgroup's
};

struct RopeArgs {
  int32_t pairs, rot_pairs;  // head_dim / 2, rot_dim / 2
  int32_t log_g;             // log2 of the lanes per head
  int32_t position_dtype;
  int32_t norm, n_axes;
  float eps, inv_dim;
  uint32_t all_tokens, tokens;  // batch * tokens, tokens of one sequence
  int64_t pos_stride[3];
  const void *positions;
  const float *inv_freq;
  PartArgs part[2];
  uint8_t pair_axis[kMaxPairs];
};

__device__ __forceinline__ double position_at(const RopeArgs &a, int axis, int64_t b, int64_t t) {
  const int64_t o = axis * a.pos_stride[0] + b * a.pos_stride[1] + t * a.pos_stride[2];
  switch (a.position_dtype) {
    case TWG_DT_I32: return (double)((const int32_t *)a.positions)[o];
    case TWG_DT_I64: return (double)((const int64_t *)a.positions)[o];
    default: return (double)((const float *)a.positions)[o];
  }
}

// cos and sin of position * inv_freq.  The angle is formed in turns in binary64 and only its
// fraction, at most half a turn, goes on in binary32: the error is 2^-52 of the number of
// turns, 4e-11 turns at position 10^6, where a binary32 angle would be off by 0.06 radians.
__device__ __forceinline__ void turn(double pos, float inv_freq, float *c, float *s) {
  constexpr double kPerTurn = 0.15915494309189533577;  // 1 / (2 pi)
  const double turns = pos * ((double)inv_freq * kPerTurn);
  const float half_turns = (float)(2.0 * (turns - rint(turns)));
  sincospif(half_turns, s, c);
}

// What a lane holds of chunk c of a head: V pairs as two runs of V elements of memory, and where
// their cosines are.  With pairs in halves the runs hold the pairs' first and second members; beyond the
// rotated elements they are neighbours.  With adjacent pairs a run is V / 2 whole pairs, and the lanes'
// runs lie side by side, so that every load is of whole lines.
template <int V, bool ADJ>
struct Runs {
  static constexpr bool kWhole = ADJ && V > 1;  // runs of whole pairs
  int first, second;                            // element offsets in the head
  bool has0, has1;                              // inside the head
  bool rot0, rot1;                              // rotated
  int trig0, trig1;                             // pair numbers
  __device__ __forceinline__ Runs(int pairs, int rot_pairs, int log_g, int c, int lane) {
    if constexpr (kWhole) {
      first = (((2 * c) << log_g) + lane) * V;
      second = (((2 * c + 1) << log_g) + lane) * V;
      has0 = first < 2 * pairs;
      has1 = second < 2 * pairs;
      rot0 = first < 2 * rot_pairs;
      rot1 = second < 2 * rot_pairs;
      trig0 = first / 2;
      trig1 = second / 2;
    } else {
      const int p0 = ((c << log_g) + lane) * V;
      const bool halves = !ADJ && p0 < rot_pairs;
      first = halves ? p0 : 2 * p0;
      second = halves ? p0 + rot_pairs : 2 * p0 + V;
      has0 = has1 = p0 < pairs;
      rot0 = rot1 = p0 < rot_pairs;
      trig0 = trig1 = p0;
    }
  }
};

template <typename T, int V>
__device__ __forceinline__ void load_run(float *to, const T *from) {
  if constexpr (V * sizeof(T) > 16) {  // binary32 weights beside 16-bit heads
    load_run<T, V / 2>(to, from);
    load_run<T, V / 2>(to + V / 2, from + V / 2);
    return;
  }
  constexpr int N = V * sizeof(T) > 16 ? 16 / (int)sizeof(T) : V;
  const Pack<T, N> p = load_pack<false>(reinterpret_cast<const Pack<T, N> *>(from));
#pragma unroll
  for (int v = 0; v < N; ++v) to[v] = (float)p.v[v];
}
template <bool NT, typename T, int V>
__device__ __forceinline__ void store_run(T *to, const float *from) {
  Pack<T, V> p;
#pragma unroll
  for (int v = 0; v < V; ++v) p.v[v] = (T)from[v];
  store_pack<NT>(reinterpret_cast<Pack<T, V> *>(to), p);
}

__device__ __forceinline__ void turn_pair(float &lo, float &hi, float c, float s) {
  const float l = lo, h = hi;
  lo = __fmaf_rn(l, c, -(h * s));
  hi = __fmaf_rn(h, c, l * s);
}
// z: the two runs, one after the other; sign = 1 turns forward, -1 back
template <int V, bool ADJ>
__device__ __forceinline__ void rotate(float *z, const Runs<V, ADJ> &at, const float *cs, const float *sn, float sign) {
  if constexpr (Runs<V, ADJ>::kWhole) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      if (!(r ? at.rot1 : at.rot0)) continue;
      const int t = r ? at.trig1 : at.trig0;
#pragma unroll
      for (int v = 0; v < V / 2; ++v) turn_pair(z[r * V + 2 * v], z[r * V + 2 * v + 1], cs[t + v], sign * sn[t + v]);
    }
  } else if (at.rot0) {
#pragma unroll
    for (int v = 0; v < V; ++v) turn_pair(z[v], z[V + v], cs[at.trig0 + v], sign * sn[at.trig0 + v]);
  }
}

// Sum over the 2^log_g lanes of a group, the same bits in all of them.  Within 16 lanes by DPP:
// neighbours, pairs, then mirrored halves and rows, whose members all hold their part's sum.
__device__ __forceinline__ float group_sum(float v, int log_g) {
#define TWG_DPP(ctrl) __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), ctrl, 0xF, 0xF, false))
  if (log_g > 0) v += TWG_DPP(0xB1);   // quad_perm 1 0 3 2
  if (log_g > 1) v += TWG_DPP(0x4E);   // quad_perm 2 3 0 1
  if (log_g > 2) v += TWG_DPP(0x141);  // row_half_mirror
  if (log_g > 3) v += TWG_DPP(0x140);  // row_mirror
#undef TWG_DPP
  if (log_g > 4) v += __shfl_xor(v, 16);
  if (log_g > 5) v += __shfl_xor(v, 32);
  return v;
}

// What the heads of a token share: its angles' cosines and sines, and where it starts in the
// inputs and results.
struct TokenRoom {
  float cs[kTrigRoom], sn[kTrigRoom];
  int64_t x[kMaxTile], dy[kMaxTile], out[kMaxTile];
};

__device__ __forceinline__ void fill_offsets(const RopeArgs &a, const PartArgs &part, uint32_t t0, int n, TokenRoom &room) {
  if ((int)threadIdx.x < n) {
    const uint32_t b = (t0 + threadIdx.x) / a.tokens, t = t0 + threadIdx.x - b * a.tokens;
    room.x[threadIdx.x] = b * part.xs[0] + t * part.xs[1];
    room.dy[threadIdx.x] = b * part.ys[0] + t * part.ys[1];
    room.out[threadIdx.x] = b * part.os[0] + t * part.os[1];
  }
}
__device__ __forceinline__ void fill_trig(const RopeArgs &a, uint32_t t0, int n, TokenRoom &room) {
  for (int i = threadIdx.x; i < n * a.rot_pairs; i += kThreads) {
    const uint32_t lt = (uint32_t)i / (uint32_t)a.rot_pairs, p = i - lt * a.rot_pairs;
    const uint32_t b = (t0 + lt) / a.tokens, t = t0 + lt - b * a.tokens;
    float c, s;
    turn(position_at(a, a.n_axes == 1 ? 0 : a.pair_axis[p], b, t), a.inv_freq[p], &c, &s);
    room.cs[i] = c;
    room.sn[i] = s;
  }
}

// A piece of work: tokens t0 .. t0 + n - 1, of whose heads (token after token) a group takes
// every step-th, starting with head `h` of token `lt`.
struct Piece {
  uint32_t t0;
  int n, lt, h, by, heads;
  __device__ __forceinline__ Piece(const RopeArgs &a, const PartArgs &part, int index) {
    const int tile = index / part.split, share = index - tile * part.split, groups = kThreads >> a.log_g;
    t0 = (uint32_t)tile * (uint32_t)part.tile;
    n = (int)min((uint32_t)part.tile, a.all_tokens - t0);
    heads = part.heads;
    by = groups * part.split;
    lt = 0;
    h = 0;
    step(share * groups + (int)(threadIdx.x >> a.log_g));
  }
  __device__ __forceinline__ void step(int k) {
    h += k;
    while (h >= heads && lt < n) {
      h -= heads;
      ++lt;
    }
  }
  __device__ __forceinline__ void next() { step(by); }
  __device__ __forceinline__ bool more() const { return lt < n; }
};

// A lane's V pairs of a head as they lie in memory: two runs of V elements.
template <typename T, int V, int C>
struct Raw {
  Pack<T, V> v[C][2];
};

template <bool NT, typename T, int V, int C, bool ADJ>
__device__ __forceinline__ void fetch(const RopeArgs &a, const void *base, int64_t offset, int lane, Raw<T, V, C> &to) {
  const T *from = (const T *)base + offset;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const Runs<V, ADJ> at(a.pairs, a.rot_pairs, a.log_g, c, lane);
    if (at.has0) to.v[c][0] = load_pack<NT>((const Pack<T, V> *)(from + at.first));
    if (at.has1) to.v[c][1] = load_pack<NT>((const Pack<T, V> *)(from + at.second));
  }
}

// The runs as binary32; zeros outside the head.
template <typename T, int V>
__device__ __forceinline__ void widen_runs(const Pack<T, V> *raw, bool has0, bool has1, float *z) {
#pragma unroll
  for (int j = 0; j < 2 * V; ++j) z[j] = (j < V ? has0 : has1) ? (float)raw[j / V].v[j % V] : 0.0f;
}

// The lane's elements of a norm weight; ones without it.
template <typename TW, int V, int C, bool ADJ>
__device__ __forceinline__ void fetch_weight(const RopeArgs &a, const PartArgs &part, int lane, float (*w)[2 * V]) {
  const TW *from = (const TW *)part.weight;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const Runs<V, ADJ> at(a.pairs, a.rot_pairs, a.log_g, c, lane);
#pragma unroll
    for (int j = 0; j < 2 * V; ++j) w[c][j] = 1.0f;
    if (from && at.has0) load_run<TW, V>(w[c], from + at.first);
    if (from && at.has1) load_run<TW, V>(w[c] + V, from + at.second);
  }
}

// A group of 2^log_g lanes works on one head at a time, a lane on V pairs in each of C chunks of
// it.  The group's next head is on its way meanwhile, the first one while the angles are computed.
// (All of a piece's heads asked for at once: 104 registers instead of 76, 17.8 -> 21.6 us
// for 4096 tokens x 40 heads of 128.)
template <typename T, typename TW, int V, int C, bool ADJ, bool STREAM>
__global__ void __launch_bounds__(kThreads) rope_forward(RopeArgs a) {
  __shared__ TokenRoom room;
  const bool second_part = (int)blockIdx.x >= a.part[0].grid;
  const PartArgs &part = a.part[second_part];
  const int lane = threadIdx.x & ((1 << a.log_g) - 1);
  Piece at(a, part, (int)blockIdx.x - (second_part ? a.part[0].grid : 0));
  fill_offsets(a, part, at.t0, at.n, room);
  __syncthreads();
  Raw<T, V, C> coming;
  if (at.more()) fetch<STREAM, T, V, C, ADJ>(a, part.x, room.x[at.lt] + at.h * part.xs[2], lane, coming);
  float w[C][2 * V];
  if (a.norm) fetch_weight<TW, V, C, ADJ>(a, part, lane, w);
  fill_trig(a, at.t0, at.n, room);
  __syncthreads();
  while (at.more()) {
    const Raw<T, V, C> x = coming;
    const int lt = at.lt;
    T *out = (T *)part.out + room.out[lt] + at.h * part.os[2];
    at.next();
    if (at.more()) fetch<STREAM, T, V, C, ADJ>(a, part.x, room.x[at.lt] + at.h * part.xs[2], lane, coming);
    float z[C][2 * V];
    float sq = 0.0f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const Runs<V, ADJ> run(a.pairs, a.rot_pairs, a.log_g, c, lane);
      widen_runs<T, V>(x.v[c], run.has0, run.has1, z[c]);
#pragma unroll
      for (int j = 0; j < 2 * V; ++j) sq = __fmaf_rn(z[c][j], z[c][j], sq);
    }
    float r = 1.0f;
    if (a.norm) r = 1.0f / sqrtf(__fmaf_rn(group_sum(sq, a.log_g), a.inv_dim, a.eps));
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const Runs<V, ADJ> run(a.pairs, a.rot_pairs, a.log_g, c, lane);
      if (a.norm) {
#pragma unroll
        for (int j = 0; j < 2 * V; ++j) z[c][j] = z[c][j] * r * w[c][j];
      }
      rotate<V, ADJ>(z[c], run, room.cs + lt * a.rot_pairs, room.sn + lt * a.rot_pairs, 1.0f);
      if (run.has0) store_run<STREAM, T, V>(out + run.first, z[c]);
      if (run.has1) store_run<STREAM, T, V>(out + run.second, z[c] + V);
    }
  }
}

// The same walk, over as many pieces as there are for the workgroup, the group's next head on its way
// while it works on one: its sums of dz u for the weight's gradient stay in registers until the last
// piece is done.  Held to 128 registers, 4 wavefronts per SIMD: heads of 16-bit elements in runs of 8 would take 132
// (adjacent pairs 143), and 3.  They put 8 (12) bytes a lane into scratch for it.  16384 tokens x 40 heads of
// 128 115 -> 106 us, adjacent 124 -> 117, x 24 heads of 64 51 -> 44; 4096 tokens x 40 39 -> 40.
template <typename T, typename TW, int V, int C, bool ADJ, bool STREAM>
__global__ void __launch_bounds__(kThreads, 4) rope_backward(RopeArgs a) {
  __shared__ TokenRoom room;
  __shared__ float joined[2 * kMaxPairs];
  const bool second_part = (int)blockIdx.x >= a.part[0].grid;
  const PartArgs &part = a.part[second_part];
  const int block = (int)blockIdx.x - (second_part ? a.part[0].grid : 0);
  const int lane = threadIdx.x & ((1 << a.log_g) - 1);
  float dw[C][2 * V], w[C][2 * V];
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int j = 0; j < 2 * V; ++j) dw[c][j] = 0.0f;
  if (a.norm) fetch_weight<TW, V, C, ADJ>(a, part, lane, w);
  for (int64_t piece = block; piece < part.work; piece += part.grid) {
    Piece at(a, part, (int)piece);
    __syncthreads();
    fill_offsets(a, part, at.t0, at.n, room);
    __syncthreads();
    Raw<T, V, C> coming_x, coming_y;
    auto get = [&]() {
      fetch<STREAM, T, V, C, ADJ>(a, part.dy, room.dy[at.lt] + at.h * part.ys[2], lane, coming_y);
      if (a.norm) fetch<STREAM, T, V, C, ADJ>(a, part.x, room.x[at.lt] + at.h * part.xs[2], lane, coming_x);
    };
    if (at.more()) get();
    fill_trig(a, at.t0, at.n, room);
    __syncthreads();
    while (at.more()) {
      const Raw<T, V, C> x = coming_x, y = coming_y;
      const int lt = at.lt;
      T *out = (T *)part.out + room.out[lt] + at.h * part.os[2];
      at.next();
      if (at.more()) get();
      float z[C][2 * V], g[C][2 * V];
      float sq = 0.0f, dot = 0.0f;
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const Runs<V, ADJ> run(a.pairs, a.rot_pairs, a.log_g, c, lane);
        widen_runs<T, V>(y.v[c], run.has0, run.has1, g[c]);
        rotate<V, ADJ>(g[c], run, room.cs + lt * a.rot_pairs, room.sn + lt * a.rot_pairs, -1.0f);
        if (a.norm) {
          widen_runs<T, V>(x.v[c], run.has0, run.has1, z[c]);
#pragma unroll
          for (int j = 0; j < 2 * V; ++j) sq = __fmaf_rn(z[c][j], z[c][j], sq);
        }
      }
      float r = 1.0f;
      if (a.norm) {
        r = 1.0f / sqrtf(__fmaf_rn(group_sum(sq, a.log_g), a.inv_dim, a.eps));
#pragma unroll
        for (int c = 0; c < C; ++c) {
#pragma unroll
          for (int j = 0; j < 2 * V; ++j) {
            z[c][j] *= r;
            dw[c][j] = __fmaf_rn(g[c][j], z[c][j], dw[c][j]);
            g[c][j] *= w[c][j];
            dot = __fmaf_rn(g[c][j], z[c][j], dot);
          }
        }
        dot = group_sum(dot, a.log_g) * a.inv_dim;
      }
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const Runs<V, ADJ> run(a.pairs, a.rot_pairs, a.log_g, c, lane);
        if (a.norm) {
#pragma unroll
          for (int j = 0; j < 2 * V; ++j) g[c][j] = r * __fmaf_rn(-z[c][j], dot, g[c][j]);
        }
        if (run.has0) store_run<STREAM, T, V>(out + run.first, g[c]);
        if (run.has1) store_run<STREAM, T, V>(out + run.second, g[c] + V);
      }
    }
  }
  if (!part.partial) return;
  // join the groups of each wavefront, then the wavefronts in their order
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int j = 0; j < 2 * V; ++j)
      for (int i = a.log_g; i < 6; ++i) dw[c][j] += __shfl_xor(dw[c][j], 1 << i);
  for (int wave = 0; wave < kThreads / 64; ++wave) {
    if ((int)(threadIdx.x >> 6) == wave && (int)(threadIdx.x & 63) < (1 << a.log_g)) {
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const Runs<V, ADJ> run(a.pairs, a.rot_pairs, a.log_g, c, lane);
#pragma unroll
        for (int j = 0; j < 2 * V; ++j) {
          if (!(j < V ? run.has0 : run.has1)) continue;
          float &to = joined[j < V ? run.first + j : run.second + j - V];
          to = wave ? to + dw[c][j] : dw[c][j];
        }
      }
    }
    __syncthreads();
  }
  const int dim = 2 * a.pairs;
  for (int i = threadIdx.x; i < dim; i += kThreads) part.partial[(int64_t)block * dim + i] = joined[i];
}

// Sum of the workgroups' partial rows, one part per grid row: 32 columns per workgroup, 32 lanes
// down each column with eight rows on their way at a time.  Binary32 for a lane's rows (eight chains of at most 16),
// binary64 for the 32 lanes' sums.
struct SumArgs {
  const float *partial[2];
  int32_t rows[2];
  void *to[2];
  int32_t dim;
};
template <typename TW>
__global__ void __launch_bounds__(1024) rope_weight_sum(SumArgs a) {
  __shared__ float part[32][33];
  const int k = blockIdx.y, col = blockIdx.x * 32 + (threadIdx.x & 31), y = threadIdx.x >> 5;
  if (!a.to[k]) return;
  const float *from = a.partial[k] + col;
  float sum[8] = {};
  if (col < a.dim) {
    for (int r0 = y; r0 < a.rows[k]; r0 += 8 * 32) {
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int r = r0 + u * 32;
        sum[u] += r < a.rows[k] ? from[(int64_t)r * a.dim] : 0.0f;
      }
    }
  }
  part[y][threadIdx.x & 31] = ((sum[0] + sum[1]) + (sum[2] + sum[3])) + ((sum[4] + sum[5]) + (sum[6] + sum[7]));
  __syncthreads();
  if (y || col >= a.dim) return;
  double total = 0.0;
  for (int i = 0; i < 32; ++i) total += (double)part[i][threadIdx.x];
  ((TW *)a.to[k])[col] = (TW)(float)total;
}

// ------------------------------------------------------------------ host side

int64_t total_heads(const twg_norm_rope_t *d) { return d->part[0].heads + d->part[1].heads; }

// (a part without heads has a weight gradient, too: zeros)
bool wants_dweight(const twg_norm_rope_t *d, int k) { return d->norm && d->part[k].dweight; }
bool wants_dweight(const twg_norm_rope_t *d) { return wants_dweight(d, 0) || wants_dweight(d, 1); }

// 0 = nothing to do, 1 = go on, negative = refused
int check(const twg_norm_rope_t *d, bool backward) {
  if (!d || !nn_dtype(d->dtype)) return TWG_E_INVALID_ARG;
  if (d->position_dtype != TWG_DT_I32 && d->position_dtype != TWG_DT_I64 && d->position_dtype != TWG_DT_F32)
    return TWG_E_INVALID_ARG;
  if (d->head_dim < 2 || d->head_dim > TWG_ROPE_MAX_HEAD_DIM || d->head_dim % 2) return TWG_E_INVALID_ARG;
  if (d->rot_dim < 0 || d->rot_dim > d->head_dim || d->rot_dim % 2) return TWG_E_INVALID_ARG;
  if (d->n_axes < 1 || d->n_axes > TWG_ROPE_MAX_AXES) return TWG_E_INVALID_ARG;
  if (d->norm) {
    if (!nn_dtype(d->weight_dtype) || !(d->eps >= 0.0f) || std::isinf(d->eps)) return TWG_E_INVALID_ARG;
    if (d->weight_dtype != TWG_DT_F32 && d->weight_dtype != d->dtype) return TWG_E_UNSUPPORTED;
  }
  for (int i = 0; i < d->rot_dim / 2; ++i)
    if (d->pair_axis[i] >= d->n_axes) return TWG_E_INVALID_ARG;
  if (d->batch < 0 || d->tokens < 0) return TWG_E_INVALID_ARG;
  for (const twg_rope_part_t &p : d->part)
    if (p.heads < 0 || p.heads > INT32_MAX / 64) return TWG_E_INVALID_ARG;
  int64_t all = 0;
  if (!add_product(all, d->batch, d->tokens)) return TWG_E_INVALID_ARG;
  if (all > INT32_MAX) return TWG_E_TOO_LARGE;
  const bool none = all == 0 || total_heads(d) == 0;
  const size_t size = (size_t)nn_size(d->dtype), wsize = (size_t)nn_size(d->weight_dtype);
  for (const twg_rope_part_t &p : d->part) {
    if (d->norm && (p.heads || backward) && !aligned_to(p.dweight, wsize)) return TWG_E_INVALID_ARG;
    if (!p.heads) continue;
    if (d->norm && !aligned_to(p.weight, wsize)) return TWG_E_INVALID_ARG;
    if (all == 0) continue;
    const bool reads_x = !backward || d->norm;
    if (!p.out || (reads_x && !p.x) || (backward && !p.dy)) return TWG_E_INVALID_ARG;
    if (!aligned_to(p.out, size) || !aligned_to(p.x, size) || !aligned_to(p.dy, size)) return TWG_E_INVALID_ARG;
    // two heads in one place: no order among their stores
    if ((d->batch > 1 && p.out_stride[0] == 0) || (d->tokens > 1 && p.out_stride[1] == 0) ||
        (p.heads > 1 && p.out_stride[2] == 0))
      return TWG_E_INVALID_ARG;
  }
  if (none) return 0;
  if (d->rot_dim && (!d->positions || !d->inv_freq)) return TWG_E_INVALID_ARG;
  const size_t psize = d->position_dtype == TWG_DT_I64 ? 8 : 4;
  if (!aligned_to(d->positions, psize) || !aligned_to(d->inv_freq, 4)) return TWG_E_INVALID_ARG;
  return 1;
}

// Whether every run of v elements that a lane moves is aligned to its own size.
bool runs_aligned(const twg_norm_rope_t *d, bool backward, int v) {
  const int whole = d->adjacent && v > 1 ? 2 : 1;  // pairs in a run's elements
  if ((d->head_dim * whole / 2) % v || (d->rot_dim * whole / 2) % v) return false;
  const size_t bytes = (size_t)(v * nn_size(d->dtype));
  const size_t wbytes = (size_t)(v * nn_size(d->weight_dtype) > 16 ? 16 : v * nn_size(d->weight_dtype));
  for (const twg_rope_part_t &p : d->part) {
    if (!p.heads) continue;
    for (int k = 0; k < 3; ++k)
      if (p.x_stride[k] % v || p.out_stride[k] % v || (backward && p.dy_stride[k] % v)) return false;
    if (!aligned_to(p.x, bytes) || !aligned_to(p.out, bytes) || (backward && !aligned_to(p.dy, bytes))) return false;
    if (d->norm && !aligned_to(p.weight, wbytes)) return false;
  }
  return true;
}

// Elements of a run and lanes of a group: the widest runs that everything is aligned to, 16 bytes
// of T where possible.
struct Lanes {
  int v, log_g;
};
Lanes lanes_of(const twg_norm_rope_t *d, bool backward) {
  Lanes l{16 / nn_size(d->dtype), 0};
  while (l.v > 1 && !runs_aligned(d, backward, l.v)) l.v /= 2;
  while ((l.v << l.log_g) < d->head_dim / 2 && l.log_g < 6) ++l.log_g;
  return l;
}

// Workgroups that leave sums for the weights' gradients, for both parts together at most, each with the
// same number of pieces.  (1016, all that the chip holds at a time: 121 us instead of 117
// for the backward call of 16384 tokens x 40 heads of 128; 8192: 113 instead of 108 with the hint below.)
constexpr int kMaxSums = 4096;
// How a part is cut into pieces: as many tokens as give each group kSteps heads (fewer where that would
// leave less than about 1024 pieces, one generation of workgroups: 3075 tokens x 24 heads backward 20.7 us
// with two heads a group and a fifth of the workgroups in a second generation, 17.4 with three), or a
// share of one token's heads.
void cut(const twg_norm_rope_t *d, bool backward, int k, PartArgs &p) {
  const int64_t all = d->batch * d->tokens, heads = d->part[k].heads;
  p.heads = (int32_t)heads;
  p.tile = p.split = 1;
  p.work = p.grid = 0;
  if (!heads || !all) return;
  const int groups = kThreads >> lanes_of(d, backward).log_g;
  const int64_t passes = (all * total_heads(d) / groups + 1023) / 1024;
  const int64_t want = groups * (passes < 1 ? 1 : passes < kSteps ? passes : kSteps);
  const int rot = d->rot_dim > 2 ? d->rot_dim / 2 : 1;
  int64_t tile = want / heads > 0 ? want / heads : 1;
  if (tile > kMaxTile) tile = kMaxTile;
  if (tile > kTrigRoom / rot) tile = kTrigRoom / rot;
  if (tile > all) tile = all;
  const int64_t split = (tile * heads + want - 1) / want;
  const int64_t tiles = (all + tile - 1) / tile;
  p.tile = (int32_t)tile;
  p.split = (int32_t)(tiles * split > INT32_MAX / 2 ? 1 : split);
  p.work = (int32_t)(tiles * p.split);
  p.grid = p.work;
}
// Both parts.  Where the backward call sums for a weight, its workgroups stay for several pieces.
void cut_both(const twg_norm_rope_t *d, bool backward, PartArgs *p) {
  for (int k = 0; k < 2; ++k) cut(d, backward, k, p[k]);
  if (!backward || !wants_dweight(d)) return;
  const int64_t work = (int64_t)p[0].work + p[1].work, rounds = (work + kMaxSums - 1) / kMaxSums;
  for (int k = 0; k < 2; ++k)
    if (p[k].work) p[k].grid = (int32_t)((p[k].work + rounds - 1) / rounds);
}

template <typename T, typename TW, int V, int C, bool ADJ>
int launch(const RopeArgs &a, bool backward, bool stream, hipStream_t s) {
  const unsigned grid = (unsigned)(a.part[0].grid + a.part[1].grid);
  constexpr bool HINT = V * sizeof(T) == 16 && !ADJ;  // (the hint is for pairs in halves only, see run())
  if (backward && stream && HINT)
    rope_backward<T, TW, V, C, ADJ, HINT><<<grid, kThreads, 0, s>>>(a);
  else if (backward)
    rope_backward<T, TW, V, C, ADJ, false><<<grid, kThreads, 0, s>>>(a);
  else if (stream && HINT)
    rope_forward<T, TW, V, C, ADJ, HINT><<<grid, kThreads, 0, s>>>(a);
  else
    rope_forward<T, TW, V, C, ADJ, false><<<grid, kThreads, 0, s>>>(a);
  return (int)hipGetLastError();
}

template <typename T, typename TW>
int launch_typed(const RopeArgs &a, int v, bool adjacent, bool backward, bool stream, hipStream_t s) {
#define TWG_ROPE_V(V, C) \
  (adjacent ? launch<T, TW, V, C, true>(a, backward, stream, s) : launch<T, TW, V, C, false>(a, backward, stream, s))
  if constexpr (sizeof(T) == 2)
    if (v == 8) return TWG_ROPE_V(8, 1);
  if (v == 4) return TWG_ROPE_V(4, 1);
  if (v == 2) return TWG_ROPE_V(2, 2);
  return TWG_ROPE_V(1, 4);
#undef TWG_ROPE_V
}

int run(const twg_norm_rope_t *d, bool backward, void *scratch, size_t scratch_bytes, twg_stream_t stream) {
  int rc = check(d, backward);
  if (rc < 0) return rc;
  const bool dw = backward && wants_dweight(d);
  if (rc > 0 && dw) {
    const size_t need = twg_norm_rope_backward_scratch_bytes(d);
    if (need && (!scratch || scratch_bytes < need)) return TWG_E_SCRATCH_SMALL;  // (0: only for a part without heads)
    if (!aligned_to(scratch, 4)) return TWG_E_INVALID_ARG;
  }
  if (rc == 0 && !dw) return 0;
  const OnBoundDevice device;
  if (int e = device.status()) return e;
  const hipStream_t s = nn_stream(stream);
  SumArgs sums{};
  sums.dim = d->head_dim;
  for (int k = 0; k < 2; ++k) sums.to[k] = d->part[k].dweight;
  if (rc > 0) {
    RopeArgs a{};
    const Lanes lanes = lanes_of(d, backward);
    a.pairs = d->head_dim / 2;
    a.rot_pairs = d->rot_dim / 2;
    a.log_g = lanes.log_g;
    a.all_tokens = (uint32_t)(d->batch * d->tokens);
    a.tokens = (uint32_t)d->tokens;
    a.position_dtype = d->position_dtype;
    a.norm = d->norm != 0;
    a.n_axes = d->n_axes;
    a.eps = d->eps;
    a.inv_dim = 1.0f / (float)d->head_dim;
    a.positions = d->positions;
    a.inv_freq = d->inv_freq;
    for (int k = 0; k < 3; ++k) a.pos_stride[k] = d->pos_stride[k];
    float *room = static_cast<float *>(scratch);
    cut_both(d, backward, a.part);
    for (int k = 0; k < 2; ++k) {
      const twg_rope_part_t &p = d->part[k];
      PartArgs &to = a.part[k];
      to.x = p.x;
      to.dy = p.dy;
      to.weight = p.weight;
      to.out = p.out;
      if (backward && wants_dweight(d, k)) {
        to.partial = room;
        sums.partial[k] = room;
        sums.rows[k] = to.grid;
        room += (size_t)to.grid * (size_t)d->head_dim;
      }
      for (int i = 0; i < 3; ++i) {
        to.xs[i] = p.x_stride[i];
        to.ys[i] = p.dy_stride[i];
        to.os[i] = p.out_stride[i];
      }
    }
    // a launch's threads are counted in 32 bits
    if (((int64_t)a.part[0].grid + a.part[1].grid) * kThreads > UINT32_MAX) return TWG_E_TOO_LARGE;
    for (int i = 0; i < a.rot_pairs; ++i) a.pair_axis[i] = d->pair_axis[i];
    const double bytes = (double)a.all_tokens * (double)total_heads(d) * d->head_dim * nn_size(d->dtype) * (backward && d->norm ? 3 : 2);
    // Nontemporal loads and stores where every run of a head is whole 128-byte lines and more is moved
    // than the last-level cache holds: 32768 tokens x 40 heads of 128, bfloat16, forward 133 -> 121 us,
    // backward 217 -> 196; with 84 MB 18.0 -> 20.3, with runs of 64 bytes (heads of 64) 67 -> 70.
    const bool stream = bytes > 256.0 * (1 << 20) && !d->adjacent && d->rot_dim == d->head_dim &&
                        (d->head_dim / 2 * nn_size(d->dtype)) % 128 == 0;
    rc = nn_dispatch(d->dtype, [&](auto t) {
      using T = decltype(t);
      // weights come in the heads' type or in binary32
      if (d->norm && d->weight_dtype == TWG_DT_F32)
        return launch_typed<T, float>(a, lanes.v, d->adjacent != 0, backward, stream, s);
      return launch_typed<T, T>(a, lanes.v, d->adjacent != 0, backward, stream, s);
    });
    if (rc) return rc;
  }
  if (!dw) return 0;
  return nn_dispatch(d->weight_dtype, [&](auto t) {
    rope_weight_sum<decltype(t)><<<dim3((d->head_dim + 31) / 32, 2), 1024, 0, s>>>(sums);
    return (int)hipGetLastError();
  });
}

}  // namespace
}  // namespace twg

using namespace twg;

extern "C" {

int twg_norm_rope(const twg_norm_rope_t *d, twg_stream_t stream) { return run(d, false, nullptr, 0, stream); }

int twg_norm_rope_backward(const twg_norm_rope_t *d, void *scratch, size_t scratch_bytes, twg_stream_t stream) {
  return run(d, true, scratch, scratch_bytes, stream);
}

size_t twg_norm_rope_backward_scratch_bytes(const twg_norm_rope_t *d) {
  if (check(d, true) <= 0 || !wants_dweight(d)) return 0;
  size_t rows = 0;
  PartArgs p[2] = {};
  cut_both(d, true, p);
  for (int k = 0; k < 2; ++k)
    if (wants_dweight(d, k)) rows += (size_t)p[k].grid;
  return rows * (size_t)d->head_dim * sizeof(float);
}

}  // extern "C"
