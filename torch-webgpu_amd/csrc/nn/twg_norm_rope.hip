// RMS norm of each query and key head and the rotation of its pairs by position, in one pass
// over the heads; one or several position axes; forward and backward.
//
//   forward   r = (mean x^2 + eps)^(-1/2), u = x r, z = u w, y = R(a) z
//   backward  dz = R(-a) dy, dw = sum dz u, g = dz w, dx = r (g - u mean(g u))
//
// R(a) turns pair i of a head by a_i = position[axis(i)] * inv_freq[i].  The angles of a token
// are the same for all of its heads: a workgroup computes them once for its tokens and keeps
// cosines and sines in LDS.
#include "twg_nn.h"

namespace twg {
namespace {

constexpr int kMaxPairs = TWG_ROPE_MAX_HEAD_DIM / 2;
constexpr int kTrigRoom = 1024;  // cosines (and sines) a workgroup holds: 8 KiB of LDS
constexpr int kMaxTile = 16;     // tokens a workgroup takes at most

struct PartArgs {
  const void *x, *dy, *weight;
  void *out;
  int64_t xs[3], ys[3], os[3];  // batch, token, head
};

struct RopeArgs {
  int32_t pairs, rot_pairs;  // head_dim / 2, rot_dim / 2
  int32_t heads0, heads;     // of part 0, of both
  int32_t tile;              // tokens per workgroup
  int32_t log_g;             // log2 of the lanes per head
  int32_t position_dtype;
  int32_t norm;
  float eps, inv_dim;
  int64_t all_tokens, tokens;  // batch * tokens, tokens of one sequence
  int64_t pos_stride[3];
  const void *positions;
  const float *inv_freq;
  float *partial;  // backward: [workgroup][2][head_dim] sums of dz u, or NULL
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
// turns, 2e-10 turns at a million positions, where a binary32 angle would be off by 0.06.
__device__ __forceinline__ void turn(double pos, float inv_freq, float *c, float *s) {
  constexpr double kPerTurn = 0.15915494309189533577;  // 1 / (2 pi)
  const double turns = pos * ((double)inv_freq * kPerTurn);
  const float half_turns = (float)(2.0 * (turns - rint(turns)));
  sincospif(half_turns, s, c);
}

// What a lane holds of one head: V pairs as two runs of V elements of memory.  `first` is
// where the run of the first elements starts, `second` the other.  Pairs beyond the rotated
// ones are neighbours.
template <int V, bool ADJ>
__device__ __forceinline__ void runs_of(const RopeArgs &a, int p0, int *first, int *second) {
  const bool halves = !ADJ && p0 < a.rot_pairs;
  *first = halves ? p0 : 2 * p0;
  *second = halves ? p0 + a.rot_pairs : 2 * p0 + V;
}

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
template <typename T, int V>
__device__ __forceinline__ void store_run(T *to, const float *from) {
  Pack<T, V> p;
#pragma unroll
  for (int v = 0; v < V; ++v) p.v[v] = (T)from[v];
  store_pack<false>(reinterpret_cast<Pack<T, V> *>(to), p);
}

// Index in the lane's 2V elements (two runs, one after the other) of pair v's members.
template <int V, bool ADJ>
__device__ __forceinline__ constexpr int lo_of(int v) { return ADJ ? 2 * v : v; }
template <int V, bool ADJ>
__device__ __forceinline__ constexpr int hi_of(int v) { return ADJ ? 2 * v + 1 : V + v; }

// sign = 1 turns forward, -1 back
template <int V, bool ADJ>
__device__ __forceinline__ void rotate(float *z, const float *cs, const float *sn, float sign) {
#pragma unroll
  for (int v = 0; v < V; ++v) {
    float &lo = z[lo_of<V, ADJ>(v)], &hi = z[hi_of<V, ADJ>(v)];
    const float c = cs[v], s = sign * sn[v], l = lo, h = hi;
    lo = __fmaf_rn(l, c, -(h * s));
    hi = __fmaf_rn(h, c, l * s);
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
  int64_t x[kMaxTile][2], dy[kMaxTile][2], out[kMaxTile][2];
};

__device__ __forceinline__ void fill(const RopeArgs &a, uint32_t t0, int n, TokenRoom &room) {
  const uint32_t tokens = (uint32_t)a.tokens;
  for (int i = threadIdx.x; i < n * a.rot_pairs; i += kThreads) {
    const uint32_t lt = (uint32_t)i / (uint32_t)a.rot_pairs, p = i - lt * a.rot_pairs;
    const uint32_t b = (t0 + lt) / tokens, t = t0 + lt - b * tokens;
    float c, s;
    turn(position_at(a, a.pair_axis[p], b, t), a.inv_freq[p], &c, &s);
    room.cs[i] = c;
    room.sn[i] = s;
  }
  if ((int)threadIdx.x < 2 * n) {
    const int lt = threadIdx.x >> 1, k = threadIdx.x & 1;
    const uint32_t b = (t0 + lt) / tokens, t = t0 + lt - b * tokens;
    room.x[lt][k] = b * a.part[k].xs[0] + t * a.part[k].xs[1];
    room.dy[lt][k] = b * a.part[k].ys[0] + t * a.part[k].ys[1];
    room.out[lt][k] = b * a.part[k].os[0] + t * a.part[k].os[1];
  }
}

// The heads of a tile, token after token, dealt to the groups: head `h` of token `lt`, stepping on
// by the number of groups.
struct Place {
  int lt, h;
  __device__ __forceinline__ void step(int by, int heads) {
    h += by;
    while (h >= heads) {
      h -= heads;
      ++lt;
    }
  }
};

// A lane's V pairs of a head as they lie in memory: two runs of V elements.
template <typename T, int V, int C>
struct Raw {
  Pack<T, V> v[C][2];
};

template <typename T, int V, int C, bool ADJ>
__device__ __forceinline__ void fetch(const RopeArgs &a, const T *from, int lane, Raw<T, V, C> &to) {
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int p0 = ((c << a.log_g) + lane) * V;
    if (p0 < a.pairs) {
      int first, second;
      runs_of<V, ADJ>(a, p0, &first, &second);
      to.v[c][0] = load_pack<false>((const Pack<T, V> *)(from + first));
      to.v[c][1] = load_pack<false>((const Pack<T, V> *)(from + second));
    }
  }
}

// The lane's elements of a norm weight; ones without it.
template <typename TW, int V, int C, bool ADJ>
__device__ __forceinline__ void fetch_weight(const RopeArgs &a, int k, int lane, float (*w)[2 * V]) {
  const TW *from = (const TW *)a.part[k].weight;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int p0 = ((c << a.log_g) + lane) * V;
#pragma unroll
    for (int j = 0; j < 2 * V; ++j) w[c][j] = 1.0f;
    if (from && p0 < a.pairs) {
      int first, second;
      runs_of<V, ADJ>(a, p0, &first, &second);
      load_run<TW, V>(w[c], from + first);
      load_run<TW, V>(w[c] + V, from + second);
    }
  }
}

// One workgroup: `tile` tokens, their heads dealt to groups of 2^log_g lanes; a lane holds V
// pairs in each of C chunks of a head.  A group's next head is on its way while it works
// on one; the first is fetched before the angles are computed.
template <typename T, typename TW, int V, int C, bool ADJ>
__global__ void __launch_bounds__(kThreads) rope_forward(RopeArgs a) {
  __shared__ TokenRoom room;
  const uint32_t t0 = blockIdx.x * (uint32_t)a.tile;
  const int n = min(a.tile, (int)(a.all_tokens - t0));
  const int lane = threadIdx.x & ((1 << a.log_g) - 1), groups = (kThreads >> a.log_g) * gridDim.y;
  fill(a, t0, n, room);
  float w[2][C][2 * V];
  if (a.norm) {
    fetch_weight<TW, V, C, ADJ>(a, 0, lane, w[0]);
    fetch_weight<TW, V, C, ADJ>(a, 1, lane, w[1]);
  }
  __syncthreads();
  Place at{0, 0};
  at.step((int)(blockIdx.y * (kThreads >> a.log_g) + (threadIdx.x >> a.log_g)), a.heads);
  auto source = [&](const Place &q) {
    const int k = q.h >= a.heads0;
    return (const T *)a.part[k].x + room.x[q.lt][k] + (q.h - (k ? a.heads0 : 0)) * a.part[k].xs[2];
  };
  Raw<T, V, C> next;
  if (at.lt < n) fetch<T, V, C, ADJ>(a, source(at), lane, next);
  while (at.lt < n) {
    const Raw<T, V, C> x = next;
    const Place here = at;
    at.step(groups, a.heads);
    if (at.lt < n) fetch<T, V, C, ADJ>(a, source(at), lane, next);
    const int k = here.h >= a.heads0;
    T *out = (T *)a.part[k].out + room.out[here.lt][k] + (here.h - (k ? a.heads0 : 0)) * a.part[k].os[2];
    float z[C][2 * V];
    float sq = 0.0f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      if (((c << a.log_g) + lane) * V >= a.pairs) continue;
#pragma unroll
      for (int j = 0; j < 2 * V; ++j) {
        z[c][j] = (float)x.v[c][j / V].v[j % V];
        sq = __fmaf_rn(z[c][j], z[c][j], sq);
      }
    }
    float r = 1.0f;
    if (a.norm) r = 1.0f / sqrtf(__fmaf_rn(group_sum(sq, a.log_g), a.inv_dim, a.eps));
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int p0 = ((c << a.log_g) + lane) * V;
      if (p0 >= a.pairs) continue;
      int first, second;
      runs_of<V, ADJ>(a, p0, &first, &second);
      if (a.norm) {
#pragma unroll
        for (int j = 0; j < 2 * V; ++j) z[c][j] = z[c][j] * r * (k ? w[1][c][j] : w[0][c][j]);
      }
      if (p0 < a.rot_pairs)
        rotate<V, ADJ>(z[c], room.cs + here.lt * a.rot_pairs + p0, room.sn + here.lt * a.rot_pairs + p0, 1.0f);
      store_run<T, V>(out + first, z[c]);
      store_run<T, V>(out + second, z[c] + V);
    }
  }
}

// The same walk; a workgroup takes tiles blockIdx.x, blockIdx.x + gridDim.x, ... and keeps its
// sums of dz u for the weights' gradients in registers until its last tile is done.
template <typename T, typename TW, int V, int C, bool ADJ>
__global__ void __launch_bounds__(kThreads) rope_backward(RopeArgs a) {
  __shared__ TokenRoom room;
  __shared__ float joined[2][2 * kMaxPairs];
  const int lane = threadIdx.x & ((1 << a.log_g) - 1), groups = kThreads >> a.log_g;
  float dw[2][C][2 * V], w[2][C][2 * V];
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int j = 0; j < 2 * V; ++j) dw[k][c][j] = 0.0f;
  if (a.norm) {
    fetch_weight<TW, V, C, ADJ>(a, 0, lane, w[0]);
    fetch_weight<TW, V, C, ADJ>(a, 1, lane, w[1]);
  }
  for (int64_t start = (int64_t)blockIdx.x * a.tile; start < a.all_tokens; start += (int64_t)gridDim.x * a.tile) {
    const uint32_t t0 = (uint32_t)start;
    const int n = min(a.tile, (int)(a.all_tokens - start));
    __syncthreads();
    fill(a, t0, n, room);
    __syncthreads();
    Place at{0, 0};
    at.step((int)(threadIdx.x >> a.log_g), a.heads);
    Raw<T, V, C> next_x, next_y;
    auto get = [&](const Place &q) {
      const int k = q.h >= a.heads0;
      const int64_t h = q.h - (k ? a.heads0 : 0);
      fetch<T, V, C, ADJ>(a, (const T *)a.part[k].dy + room.dy[q.lt][k] + h * a.part[k].ys[2], lane, next_y);
      if (a.norm) fetch<T, V, C, ADJ>(a, (const T *)a.part[k].x + room.x[q.lt][k] + h * a.part[k].xs[2], lane, next_x);
    };
    if (at.lt < n) get(at);
    while (at.lt < n) {
      const Raw<T, V, C> x = next_x, y = next_y;
      const Place here = at;
      at.step(groups, a.heads);
      if (at.lt < n) get(at);
      const int k = here.h >= a.heads0;
      T *out = (T *)a.part[k].out + room.out[here.lt][k] + (here.h - (k ? a.heads0 : 0)) * a.part[k].os[2];
      float z[C][2 * V], g[C][2 * V];
      float sq = 0.0f, dot = 0.0f;
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const int p0 = ((c << a.log_g) + lane) * V;
        if (p0 >= a.pairs) continue;
#pragma unroll
        for (int j = 0; j < 2 * V; ++j) g[c][j] = (float)y.v[c][j / V].v[j % V];
        if (p0 < a.rot_pairs)
          rotate<V, ADJ>(g[c], room.cs + here.lt * a.rot_pairs + p0, room.sn + here.lt * a.rot_pairs + p0, -1.0f);
        if (a.norm) {
#pragma unroll
          for (int j = 0; j < 2 * V; ++j) {
            z[c][j] = (float)x.v[c][j / V].v[j % V];
            sq = __fmaf_rn(z[c][j], z[c][j], sq);
          }
        }
      }
      float r = 1.0f;
      if (a.norm) {
        r = 1.0f / sqrtf(__fmaf_rn(group_sum(sq, a.log_g), a.inv_dim, a.eps));
#pragma unroll
        for (int c = 0; c < C; ++c) {
          if (((c << a.log_g) + lane) * V >= a.pairs) continue;
#pragma unroll
          for (int j = 0; j < 2 * V; ++j) {
            z[c][j] *= r;
            if (k) dw[1][c][j] = __fmaf_rn(g[c][j], z[c][j], dw[1][c][j]);
            else dw[0][c][j] = __fmaf_rn(g[c][j], z[c][j], dw[0][c][j]);
            g[c][j] *= k ? w[1][c][j] : w[0][c][j];
            dot = __fmaf_rn(g[c][j], z[c][j], dot);
          }
        }
        dot = group_sum(dot, a.log_g) * a.inv_dim;
      }
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const int p0 = ((c << a.log_g) + lane) * V;
        if (p0 >= a.pairs) continue;
        int first, second;
        runs_of<V, ADJ>(a, p0, &first, &second);
        if (a.norm) {
#pragma unroll
          for (int j = 0; j < 2 * V; ++j) g[c][j] = r * __fmaf_rn(-z[c][j], dot, g[c][j]);
        }
        store_run<T, V>(out + first, g[c]);
        store_run<T, V>(out + second, g[c] + V);
      }
    }
  }
  if (!a.partial) return;
  // join the groups of each wavefront, then the wavefronts in their order
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int j = 0; j < 2 * V; ++j)
        for (int i = a.log_g; i < 6; ++i) dw[k][c][j] += __shfl_xor(dw[k][c][j], 1 << i);
  for (int wave = 0; wave < kThreads / 64; ++wave) {
    if ((int)(threadIdx.x >> 6) == wave && (int)(threadIdx.x & 63) < (1 << a.log_g)) {
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int c = 0; c < C; ++c) {
          const int p0 = ((c << a.log_g) + lane) * V;
          if (p0 < a.pairs) {
            int first, second;
            runs_of<V, ADJ>(a, p0, &first, &second);
#pragma unroll
            for (int j = 0; j < 2 * V; ++j) {
              float &to = joined[k][j < V ? first + j : second + j - V];
              to = wave ? to + dw[k][c][j] : dw[k][c][j];
            }
          }
        }
    }
    __syncthreads();
  }
  const int dim = 2 * a.pairs;
  float *mine = a.partial + (int64_t)blockIdx.x * 2 * dim;
  for (int i = threadIdx.x; i < 2 * dim; i += kThreads) mine[i] = joined[i >= dim][i >= dim ? i - dim : i];
}

// Sum of the workgroups' partial rows: 32 columns per workgroup, 32 lanes down each column with
// eight rows on their way at a time.
template <typename TW>
__global__ void __launch_bounds__(1024) rope_weight_sum(const float *partial, int rows, int dim, TW *dw0, TW *dw1) {
  __shared__ float part[32][33];
  const int col = blockIdx.x * 32 + (threadIdx.x & 31), y = threadIdx.x >> 5;
  float sum[8] = {};
  if (col < 2 * dim) {
    for (int r0 = y; r0 < rows; r0 += 8 * 32) {
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int r = r0 + u * 32;
        sum[u] += r < rows ? partial[(int64_t)r * 2 * dim + col] : 0.0f;
      }
    }
  }
  part[y][threadIdx.x & 31] = ((sum[0] + sum[1]) + (sum[2] + sum[3])) + ((sum[4] + sum[5]) + (sum[6] + sum[7]));
  __syncthreads();
  if (y || col >= 2 * dim) return;
  double total = 0.0;
  for (int i = 0; i < 32; ++i) total += (double)part[i][threadIdx.x];
  TW *to = col < dim ? dw0 : dw1;
  if (to) to[col < dim ? col : col - dim] = (TW)(float)total;
}

// ------------------------------------------------------------------ host side

constexpr int kMaxPartials = 1024;

int64_t total_heads(const twg_norm_rope_t *d) { return d->part[0].heads + d->part[1].heads; }

bool wants_dweight(const twg_norm_rope_t *d) {
  return d->norm && ((d->part[0].heads && d->part[0].dweight) || (d->part[1].heads && d->part[1].dweight));
}

// tokens per workgroup: enough heads for its groups, as far as the cosines fit
int tile_of(const twg_norm_rope_t *d, int64_t all_tokens) {
  const int rot = d->rot_dim / 2 > 0 ? d->rot_dim / 2 : 1;
  int tile = 1;
  while (tile < kMaxTile && 2 * tile * rot <= kTrigRoom && tile * total_heads(d) < 128 &&
         all_tokens / (2 * tile) >= 1024)
    tile *= 2;
  return tile;
}

int partial_rows(const twg_norm_rope_t *d) {
  const int64_t all = d->batch * d->tokens;
  const int64_t tiles = (all + tile_of(d, all) - 1) / tile_of(d, all);
  return (int)(tiles < kMaxPartials ? tiles : kMaxPartials);
}

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
    if (!p.heads) continue;
    if (d->norm && (!aligned_to(p.weight, wsize) || !aligned_to(p.dweight, wsize))) return TWG_E_INVALID_ARG;
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
  if ((d->head_dim / 2) % v || (d->rot_dim / 2) % v) return false;
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

template <typename T, typename TW, int V, int C, bool ADJ>
int launch(const RopeArgs &a, bool backward, dim3 grid, hipStream_t s) {
  if (backward)
    rope_backward<T, TW, V, C, ADJ><<<grid, kThreads, 0, s>>>(a);
  else
    rope_forward<T, TW, V, C, ADJ><<<grid, kThreads, 0, s>>>(a);
  return (int)hipGetLastError();
}

template <typename T, typename TW>
int launch_typed(const twg_norm_rope_t *d, RopeArgs a, bool backward, hipStream_t s) {
  // the widest runs that everything is aligned to: 16 bytes of T where possible
  constexpr int W = 16 / (int)sizeof(T);
  const int v = runs_aligned(d, backward, W) ? W : runs_aligned(d, backward, 4) ? 4
              : runs_aligned(d, backward, 2) ? 2 : 1;
  const int lanes = (a.pairs + v - 1) / v;
  a.log_g = 0;
  while ((1 << a.log_g) < lanes && a.log_g < 6) ++a.log_g;
  const int64_t tiles = (a.all_tokens + a.tile - 1) / a.tile;
  dim3 grid((unsigned)tiles, 1);
  if (backward) {
    if (a.partial) grid.x = (unsigned)partial_rows(d);
  } else {
    // few tokens: their heads are spread over several workgroups, one head per group
    const int64_t per_pass = kThreads >> a.log_g, units = (int64_t)a.tile * a.heads;
    const int64_t split = (units + per_pass - 1) / per_pass;
    while ((int64_t)grid.y * 2 <= split && tiles * grid.y < 1024) grid.y *= 2;
  }
  const bool adj = d->adjacent != 0;
#define TWG_ROPE_V(V, C)                                                   \
  (adj ? launch<T, TW, V, C, true>(a, backward, grid, s)                   \
       : launch<T, TW, V, C, false>(a, backward, grid, s))
  if constexpr (W == 8)
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
    if (!scratch || scratch_bytes < need) return TWG_E_SCRATCH_SMALL;
    if (!aligned_to(scratch, 4)) return TWG_E_INVALID_ARG;
  }
  if (rc == 0 && !dw) return 0;
  if (int e = ensure_init()) return e;
  const hipStream_t s = nn_stream(stream);
  int rows = 0;
  if (rc > 0) {
    RopeArgs a{};
    a.pairs = d->head_dim / 2;
    a.rot_pairs = d->rot_dim / 2;
    a.heads0 = (int32_t)d->part[0].heads;
    a.heads = (int32_t)total_heads(d);
    a.all_tokens = d->batch * d->tokens;
    a.tokens = d->tokens;
    a.tile = tile_of(d, a.all_tokens);
    a.position_dtype = d->position_dtype;
    a.norm = d->norm != 0;
    a.eps = d->eps;
    a.inv_dim = 1.0f / (float)d->head_dim;
    a.positions = d->positions;
    a.inv_freq = d->inv_freq;
    a.partial = dw ? static_cast<float *>(scratch) : nullptr;
    for (int k = 0; k < 3; ++k) a.pos_stride[k] = d->pos_stride[k];
    for (int k = 0; k < 2; ++k) {
      const twg_rope_part_t &p = d->part[k];
      a.part[k].x = p.x;
      a.part[k].dy = p.dy;
      a.part[k].weight = p.weight;
      a.part[k].out = p.out;
      for (int i = 0; i < 3; ++i) {
        a.part[k].xs[i] = p.x_stride[i];
        a.part[k].ys[i] = p.dy_stride[i];
        a.part[k].os[i] = p.out_stride[i];
      }
    }
    for (int i = 0; i < a.rot_pairs; ++i) a.pair_axis[i] = d->pair_axis[i];
    rc = nn_dispatch(d->dtype, [&](auto t) {
      using T = decltype(t);
      // weights come in the heads' type or in binary32
      if (d->norm && d->weight_dtype == TWG_DT_F32) return launch_typed<T, float>(d, a, backward, s);
      return launch_typed<T, T>(d, a, backward, s);
    });
    if (rc) return rc;
    rows = dw ? partial_rows(d) : 0;
  }
  if (!dw) return 0;
  return nn_dispatch(d->weight_dtype, [&](auto t) {
    using TW = decltype(t);
    const auto to = [&](int k) { return d->part[k].heads ? static_cast<TW *>(d->part[k].dweight) : nullptr; };
    rope_weight_sum<TW><<<(2 * d->head_dim + 31) / 32, 1024, 0, s>>>(static_cast<const float *>(scratch), rows,
                                                                     d->head_dim, to(0), to(1));
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
  return (size_t)partial_rows(d) * 2 * (size_t)d->head_dim * sizeof(float);
}

}  // extern "C"
