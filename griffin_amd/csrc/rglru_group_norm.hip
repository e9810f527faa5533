// Group norm with an activation over channels-last features x[N, L, C]:
//   xhat = (x - mean) rstd,  mean and variance over the L positions and C / G channels of a (row, group);  rstd = 1 / sqrt(var + eps)
//   y = act(xhat w + b),  act: none, silu or the tanh form of gelu
// and its reverse mode, with t = dy act'(xhat w + b):
//   dw_c = sum of t xhat,  db_c = sum of t,  dx = rstd (w t - m1 - xhat m2),  m1 = mean of w t,  m2 = mean of w t xhat over the group
//
// One position (the heads' norm behind a recurrence: every token on its own): a group is a run of C / G elements, which 4 to 64
// lanes hold in registers.  Everything is read once and written once.
// 16384 rows of 1024 in 8 groups (bf16): 14 us forward, 29 + 5 backward, where the bytes take 13 and 20 at the rate of a large copy.
// The backward pass keeps half as many waves: each leaves a set of partial parameter gradients (16 waves a compute unit instead of
// 8: 35 + 9 instead of 37 + 5 us at the time).
// Many positions: the positions are cut into chunks, two workgroups a compute unit, one kernel leaves each chunk's sums, the next joins
// them and writes (four a compute unit: more sums to join, 25.6 -> 26.4 and 21.3 -> 22.4 us for the two that write).  8 rows of 2048 x 1024: 10 + 17 us
// forward, 22 + 26 + 4 backward.  Bound by memory and by the chain in front of it; the first vectors are requested before
// the sums are joined (apply 21 -> 17 us).
// All sums are fp32.  Variances come from deviations from a mean (of the run, or of the batch of values a thread holds) and are joined
// with the difference of the means, never from a difference of squares.

#include <hip/hip_runtime.h>

#include <cstring>

#include "rglru_device.h"
#include "rglru_host.h"
#include "rglru_sums.h"

namespace rglru {

constexpr int kGroupThreads = 256;
constexpr int kGroupSlots = 4;                // most vectors a lane of the one-position kernel

struct GroupArgs {
  const void *x, *dy, *weight, *bias;
  void *y, *dx;
  float *stats;                               // [N, G, 2]: mean and rstd
  float *entries;                             // [N, G, E, 3 or 2]: a chunk's count, mean and squared deviations, or its two sums
  float *dweight, *dbias;                     // partial sums [sets][C]
  long long rows;                             // one position: N * G
  int N, L, C, G, activation, vec_dtype;
  int Cg, width;                              // channels of a group; in vectors
  int columns, lines, blocks, per_group;      // many positions: vector columns of a workgroup, positions at a time, column blocks, blocks a group
  int chunks, chunk;                          // chunks of positions, positions in one
  int row0, rows_apart;                       // many positions: first row of the launch; the kernel of the sums goes on rows_apart further
  int lanes, waves;                           // one position: lanes a run, waves of the launch
  float eps, inv_count;
};

template <typename IO, int V> struct Run {
  typedef IO Raw __attribute__((ext_vector_type(V)));
  static RGLRU_DEVICE void load(const void* p, long long at, float (&v)[V]) {
    const Raw r = *reinterpret_cast<const Raw*>((const IO*)p + at);
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = (float)r[e];
  }
  static RGLRU_DEVICE Raw request(const void* p, long long at) { return *reinterpret_cast<const Raw*>((const IO*)p + at); }
  static RGLRU_DEVICE void unpack(const Raw& r, float (&v)[V]) {
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = (float)r[e];
  }
  // Written through: whole 128-byte lines
  static RGLRU_DEVICE void store(rsrc_t r, unsigned at, const float (&v)[V]) {
    if constexpr (V > 1) {
      Raw raw;
#pragma unroll
      for (int e = 0; e < V; ++e) raw[e] = (IO)v[e];
      buf_store_b128<kWriteThrough>(__builtin_bit_cast(i32x4, raw), r, at * (unsigned)sizeof(IO));
    } else {
      BufIo<IO>::store((IO)v[0], r, at * (unsigned)sizeof(IO), 0);
    }
  }
  static RGLRU_DEVICE rsrc_t rows(void* p, long long at) { return make_rsrc((IO*)p + at, 0xfffffff0u); }
};

// V parameters from channel c on (a multiple of V); `absent` without a tensor.
template <int V> RGLRU_DEVICE void group_params(const void* p, int c, int dtype, float absent, float (&out)[V]) {
  if (V > 1 && p != nullptr && ((unsigned long long)p & 15) == 0) {  // by vectors where the tensor lies on their boundaries
    typedef __bf16 Half __attribute__((ext_vector_type(V)));
    typedef float Full __attribute__((ext_vector_type(V)));
    if (dtype == 1) {
      const Half h = *reinterpret_cast<const Half*>((const __bf16*)p + c);
#pragma unroll
      for (int e = 0; e < V; ++e) out[e] = (float)h[e];
    } else {
      const Full f = *reinterpret_cast<const Full*>((const float*)p + c);
#pragma unroll
      for (int e = 0; e < V; ++e) out[e] = f[e];
    }
    return;
  }
#pragma unroll
  for (int e = 0; e < V; ++e) out[e] = p == nullptr ? absent : dtype == 1 ? (float)((const __bf16*)p)[c + e] : ((const float*)p)[c + e];
}

RGLRU_DEVICE float group_act(float v, int activation) {
  return activation == RGLRU_ACT_SILU ? v * sigmoid_fast(v) : activation == RGLRU_ACT_GELU ? gelu_tanh_parts(v).gelu : v;
}
RGLRU_DEVICE float group_slope(float v, int activation) {
  if (activation == RGLRU_ACT_SILU) {
    const float s = sigmoid_fast(v);
    return s * fmaf(v, 1.f - s, 1.f);
  }
  return activation == RGLRU_ACT_GELU ? gelu_tanh_parts(v).dgelu : 1.f;
}

// Sum over runs of `lanes` lanes (a power of two).  Within sixteen lanes by data-parallel moves: once the lanes of a quad (of eight)
// hold one number, mirroring eight (sixteen) lanes brings the other half's.
template <int CONTROL> RGLRU_DEVICE float lane_move(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CONTROL, 0xf, 0xf, true));
}
RGLRU_DEVICE float lanes_sum(float v, int lanes) {
  if (lanes >= 2) v += lane_move<0xb1>(v);                  // quad: 1 0 3 2
  if (lanes >= 4) v += lane_move<0x4e>(v);                  // quad: 2 3 0 1
  if (lanes >= 8) v += lane_move<0x141>(v);                 // eight lanes mirrored
  if (lanes >= 16) v += lane_move<0x140>(v);                // sixteen lanes mirrored
  for (int m = 16; m < lanes; m <<= 1) v += __shfl_xor(v, m, 64);
  return v;
}

// ---- one position ---------------------------------------------------------------------------------------------------
// `lanes` lanes share a run of Cg elements, a wave takes 64 / lanes runs at a time.  The launch's runs a round are a multiple of
// G, so a lane keeps its channels, whose parameter gradients it adds up in registers.
template <typename IO, int V, int SLOTS, bool BACKWARD> __global__ __launch_bounds__(kGroupThreads) void group_norm_rows_kernel(GroupArgs p) {
  typedef Run<IO, V> R;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(blockIdx.x * (kGroupThreads / 64) + (threadIdx.x >> 6));
  if (wave >= p.waves) return;
  const int runs = 64 / p.lanes, l = lane % p.lanes, first = wave * runs + lane / p.lanes;
  const unsigned here = (unsigned)(lane / p.lanes * p.Cg);   // from the wave's first run on
  const long long round = (long long)p.waves * runs;
  const int c0 = first % p.G * p.Cg;
  bool has[SLOTS];
#pragma unroll
  for (int s = 0; s < SLOTS; ++s) has[s] = l + p.lanes * s < p.width;
  typename R::Raw next[SLOTS], next_up[SLOTS];
  float next_mean = 0.f, next_rstd = 0.f;
  auto request = [&](long long run) {
    if constexpr (BACKWARD)
      if (run < p.rows) next_mean = p.stats[2 * run], next_rstd = p.stats[2 * run + 1];
#pragma unroll
    for (int s = 0; s < SLOTS; ++s) {
      const bool ok = run < p.rows && has[s];
      const long long at = run * p.Cg + (l + p.lanes * s) * V;
      next[s] = typename R::Raw{};
      if (ok) next[s] = R::request(p.x, at);
      if constexpr (BACKWARD) {
        next_up[s] = typename R::Raw{};
        if (ok) next_up[s] = R::request(p.dy, at);
      }
    }
  };
  request(first);
  float w[SLOTS][V], b[SLOTS][V], dw[BACKWARD ? SLOTS : 1][V], db[BACKWARD ? SLOTS : 1][V];
#pragma unroll
  for (int s = 0; s < SLOTS; ++s) {
    const int c = has[s] ? c0 + (l + p.lanes * s) * V : 0;
    group_params<V>(p.weight, c, p.vec_dtype, 1.f, w[s]);
    group_params<V>(p.bias, c, p.vec_dtype, 0.f, b[s]);
    if constexpr (BACKWARD)
#pragma unroll
      for (int e = 0; e < V; ++e) dw[s][e] = db[s][e] = 0.f;
  }
  for (long long start = (long long)wave * runs; start < p.rows; start += round) {
    const long long run = start + lane / p.lanes;
    float x[SLOTS][V], up[BACKWARD ? SLOTS : 1][V];
#pragma unroll
    for (int s = 0; s < SLOTS; ++s) {
      R::unpack(next[s], x[s]);
      if constexpr (BACKWARD) R::unpack(next_up[s], up[s]);
    }
    const float mean_there = next_mean, rstd_there = next_rstd;
    request(run + round);
    const bool live = run < p.rows;
    if constexpr (!BACKWARD) {
      float sum = 0.f, squares = 0.f;
#pragma unroll
      for (int s = 0; s < SLOTS; ++s)
#pragma unroll
        for (int e = 0; e < V; ++e) sum += x[s][e];         // zeros past the run
      const float mean = lanes_sum(sum, p.lanes) * p.inv_count;
#pragma unroll
      for (int s = 0; s < SLOTS; ++s)
#pragma unroll
        for (int e = 0; e < V; ++e) {
          x[s][e] = has[s] ? x[s][e] - mean : 0.f;
          squares = fmaf(x[s][e], x[s][e], squares);
        }
      const float rstd = __builtin_amdgcn_rsqf(fmaf(lanes_sum(squares, p.lanes), p.inv_count, p.eps));
      if (p.stats && live && l == 0) p.stats[2 * run] = mean, p.stats[2 * run + 1] = rstd;
#pragma unroll
      for (int s = 0; s < SLOTS; ++s) {
#pragma unroll
        for (int e = 0; e < V; ++e) x[s][e] = group_act(fmaf(x[s][e] * rstd, w[s][e], b[s][e]), p.activation);
        if (live && has[s]) R::store(R::rows(p.y, start * p.Cg), here + (unsigned)((l + p.lanes * s) * V), x[s]);
      }
    } else {
      const float mean = mean_there, rstd = rstd_there;
      float m1 = 0.f, m2 = 0.f;
#pragma unroll
      for (int s = 0; s < SLOTS; ++s)
#pragma unroll
        for (int e = 0; e < V; ++e) {
          x[s][e] = has[s] ? (x[s][e] - mean) * rstd : 0.f;
          const float t = up[s][e] * group_slope(fmaf(x[s][e], w[s][e], b[s][e]), p.activation);
          if (live) db[s][e] += t, dw[s][e] = fmaf(t, x[s][e], dw[s][e]);
          up[s][e] = t * w[s][e];
          m1 += up[s][e];
          m2 = fmaf(up[s][e], x[s][e], m2);
        }
      m1 = lanes_sum(m1, p.lanes) * p.inv_count;
      m2 = lanes_sum(m2, p.lanes) * p.inv_count;
#pragma unroll
      for (int s = 0; s < SLOTS; ++s) {
#pragma unroll
        for (int e = 0; e < V; ++e) x[s][e] = rstd * (up[s][e] - fmaf(x[s][e], m2, m1));
        if (live && has[s]) R::store(R::rows(p.dx, start * p.Cg), here + (unsigned)((l + p.lanes * s) * V), x[s]);
      }
    }
  }
  if constexpr (BACKWARD) {
    if (p.dweight) {
      const long long at = (long long)(first / p.G) * p.C + c0;
#pragma unroll
      for (int s = 0; s < SLOTS; ++s)
        if (has[s])
#pragma unroll
          for (int e = 0; e < V; ++e) {
            p.dweight[at + (l + p.lanes * s) * V + e] = dw[s][e];
            p.dbias[at + (l + p.lanes * s) * V + e] = db[s][e];
          }
    }
  }
}

// ---- many positions -------------------------------------------------------------------------------------------------
// A workgroup takes a chunk of positions of a row and a block of vector columns: whole groups where 256 vectors hold one, else
// a part of one group.  Thread (column, line): one vector of every lines-th position.
constexpr int kGroupGrid = 1 << 22;           // most workgroups of a launch; further rows take another one
// Most workgroups a compute unit of the kernel of the sums: it goes on to further rows and adds their parameter gradients up, of which each workgroup
// leaves one set.  A million rows of 2 x 64: 33 MiB of scratch instead of 544 and 12.1 ms a training step instead of 19.6.
constexpr int kGroupSums = 8;
struct GroupPlace {
  int n, chunk, block, first_group, groups, part;            // groups of the block; part of the group where it is one
  int col, line, c;                                         // c: first channel
  int from, to;                                             // positions
  bool live;
};
template <int V> RGLRU_DEVICE GroupPlace group_place(const GroupArgs& p) {
  GroupPlace g;
  long long i = blockIdx.x;
  g.block = (int)(i % p.blocks), i /= p.blocks;
  g.chunk = (int)(i % p.chunks), g.n = p.row0 + (int)(i / p.chunks);
  g.part = p.per_group > 1 ? g.block % p.per_group : 0;
  const int each = p.per_group > 1 ? 1 : p.columns / p.width;
  g.first_group = p.per_group > 1 ? g.block / p.per_group : g.block * each;
  g.groups = p.G - g.first_group < each ? p.G - g.first_group : each;
  g.col = threadIdx.x % p.columns, g.line = threadIdx.x / p.columns;
  const int vectors = p.per_group > 1 ? (p.width - g.part * p.columns < p.columns ? p.width - g.part * p.columns : p.columns) : g.groups * p.width;
  g.live = g.line < p.lines && g.col < vectors;
  g.c = g.first_group * p.Cg + (g.part * p.columns + (g.live ? g.col : 0)) * V;
  g.from = g.chunk * p.chunk;
  g.to = g.from + p.chunk < p.L ? g.from + p.chunk : p.L;
  return g;
}

struct Moments { float n, mean, m2; };
RGLRU_DEVICE Moments join(const Moments& a, const Moments& b) {
  const float n = a.n + b.n, part = n > 0.f ? b.n * __builtin_amdgcn_rcpf(n) : 0.f, d = b.mean - a.mean;
  return {n, fmaf(d, part, a.mean), a.m2 + b.m2 + d * d * part * a.n};
}

// Values of the block's threads joined for each group: over the lines first, then over the group's columns.  Returns it to the
// thread of line 0 that holds a group's first column.  (`mine` of the moments takes 28 bytes of scratch a lane, written and read once.)
template <typename T, typename JOIN> RGLRU_DEVICE T group_join(T mine, const T& none, const GroupArgs& p, const GroupPlace& g, T* shared, JOIN both) {
  shared[threadIdx.x] = g.live ? mine : none;
  __syncthreads();
  if (g.line == 0)
    for (int i = 1; i < p.lines; ++i) mine = both(mine, shared[i * p.columns + g.col]);
  if (!g.live) mine = none;
  __syncthreads();
  const int width = p.per_group > 1 ? p.columns : p.width, at = g.col % width;
  for (int d = 1; d < width; d <<= 1) {
    if (g.line == 0) shared[g.col] = mine;
    __syncthreads();
    if (g.line == 0 && at % (2 * d) == 0 && at + d < width) mine = both(mine, shared[g.col + d]);
    __syncthreads();
  }
  return mine;
}

template <typename IO, int V> __global__ __launch_bounds__(kGroupThreads) void group_norm_moments_kernel(GroupArgs p) {
  typedef Run<IO, V> R;
  constexpr int U = 4;
  __shared__ Moments shared[kGroupThreads];
  const GroupPlace g = group_place<V>(p);
  Moments m = {0.f, 0.f, 0.f};
  const long long base = (long long)g.n * p.L * p.C + g.c;
  if (g.live) {
    int l = g.from + g.line;
    for (; l + (U - 1) * p.lines < g.to; l += U * p.lines) {
      float v[U][V], sum = 0.f, squares = 0.f;
#pragma unroll
      for (int u = 0; u < U; ++u) R::load(p.x, base + (long long)(l + u * p.lines) * p.C, v[u]);
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < V; ++e) sum += v[u][e];
      const float mean = sum * (1.f / (U * V));
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < V; ++e) squares = fmaf(v[u][e] - mean, v[u][e] - mean, squares);
      m = join(m, {(float)(U * V), mean, squares});
    }
    for (; l < g.to; l += p.lines) {
      float v[V], sum = 0.f, squares = 0.f;
      R::load(p.x, base + (long long)l * p.C, v);
#pragma unroll
      for (int e = 0; e < V; ++e) sum += v[e];
      const float mean = sum * (1.f / V);
#pragma unroll
      for (int e = 0; e < V; ++e) squares = fmaf(v[e] - mean, v[e] - mean, squares);
      m = join(m, {(float)V, mean, squares});
    }
  }
  m = group_join(m, Moments{0.f, 0.f, 0.f}, p, g, shared, [](const Moments& a, const Moments& b) { return join(a, b); });
  const int width = p.per_group > 1 ? p.columns : p.width;
  if (g.line == 0 && g.col % width == 0 && g.live) {
    const long long entries = (long long)p.chunks * p.per_group;
    float* out = p.entries + (((long long)g.n * p.G + g.first_group + g.col / width) * entries + (long long)g.chunk * p.per_group + g.part) * 3;
    out[0] = m.n, out[1] = m.mean, out[2] = m.m2;
  }
}

// mean and rstd of the block's groups from the chunks' entries: eight lanes a group.
RGLRU_DEVICE void group_statistics(const GroupArgs& p, const GroupPlace& g, float (&mean)[kGroupThreads], float (&rstd)[kGroupThreads]) {
  const int entries = p.chunks * p.per_group, sub = threadIdx.x & 7;
  for (int i = threadIdx.x >> 3; i < g.groups; i += kGroupThreads / 8) {
    const long long group = (long long)g.n * p.G + g.first_group + i;
    Moments m = {0.f, 0.f, 0.f};
#pragma unroll 4
    for (int e = sub; e < entries; e += 8) {
      const float* at = p.entries + (group * entries + e) * 3;
      m = join(m, {at[0], at[1], at[2]});
    }
#pragma unroll
    for (int d = 4; d >= 1; d >>= 1) m = join(m, {__shfl_down(m.n, d, 8), __shfl_down(m.mean, d, 8), __shfl_down(m.m2, d, 8)});
    if (sub == 0) {
      mean[i] = m.mean;
      rstd[i] = __builtin_amdgcn_rsqf(fmaf(m.m2, p.inv_count, p.eps));
      if (p.stats && g.chunk == 0 && g.part == 0) p.stats[2 * group] = m.mean, p.stats[2 * group + 1] = rstd[i];
    }
  }
}

// A thread's next U vectors of its column, on their way while the ones before are worked on (and, the first, while the statistics and the
// parameters are read).  Zeros behind the chunk.
template <typename IO, int V, int U> struct GroupAhead {
  typedef Run<IO, V> R;
  typename R::Raw next[U];
  RGLRU_DEVICE void request(const GroupArgs& p, const GroupPlace& g, const void* from, int l0) {
    const long long base = (long long)g.n * p.L * p.C + g.c;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int l = l0 + g.line + u * p.lines;
      next[u] = typename R::Raw{};
      if (g.live && l < g.to) next[u] = R::request(from, base + (long long)l * p.C);
    }
  }
  RGLRU_DEVICE void take(float (&v)[U][V]) const {
#pragma unroll
    for (int u = 0; u < U; ++u) R::unpack(next[u], v[u]);
  }
};

template <typename IO, int V> __global__ __launch_bounds__(kGroupThreads) void group_norm_apply_kernel(GroupArgs p) {
  typedef Run<IO, V> R;
  constexpr int U = 4;
  __shared__ float mean[kGroupThreads], rstd[kGroupThreads];
  const GroupPlace g = group_place<V>(p);
  GroupAhead<IO, V, U> x;
  x.request(p, g, p.x, g.from);
  float w[V], b[V];
  group_params<V>(p.weight, g.c, p.vec_dtype, 1.f, w);
  group_params<V>(p.bias, g.c, p.vec_dtype, 0.f, b);
  group_statistics(p, g, mean, rstd);
  __syncthreads();
  if (!g.live) return;
  const int mine = p.per_group > 1 ? 0 : g.col / p.width;
  const float mu = mean[mine], rs = rstd[mine];
  for (int l0 = g.from; l0 < g.to; l0 += U * p.lines) {
    const rsrc_t to = R::rows(p.y, ((long long)g.n * p.L + l0) * p.C);
    float v[U][V];
    x.take(v);
    x.request(p, g, p.x, l0 + U * p.lines);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (l0 + g.line + u * p.lines < g.to) {
#pragma unroll
        for (int e = 0; e < V; ++e) v[u][e] = group_act(fmaf((v[u][e] - mu) * rs, w[e], b[e]), p.activation);
        R::store(to, (unsigned)((g.line + u * p.lines) * p.C + g.c), v[u]);
      }
  }
}

struct TwoSums { float a, b; };

template <typename IO, int V> __global__ __launch_bounds__(kGroupThreads) void group_norm_sums_kernel(GroupArgs p) {
  constexpr int U = 4;
  __shared__ TwoSums shared[kGroupThreads];
  __shared__ float lines[2][kGroupThreads * V];
  GroupPlace g = group_place<V>(p);
  GroupAhead<IO, V, U> next_x, next_up;
  next_x.request(p, g, p.x, g.from);
  next_up.request(p, g, p.dy, g.from);
  float w[V], b[V], all_dw[V], all_db[V];                   // over the workgroup's rows
  group_params<V>(p.weight, g.c, p.vec_dtype, 1.f, w);
  group_params<V>(p.bias, g.c, p.vec_dtype, 0.f, b);
#pragma unroll
  for (int e = 0; e < V; ++e) all_dw[e] = all_db[e] = 0.f;
  const int row0 = g.n;
  while (true) {
    float dw[V], db[V];
#pragma unroll
    for (int e = 0; e < V; ++e) dw[e] = db[e] = 0.f;
    const long long group = (long long)g.n * p.G + g.c / p.Cg;
    const float mu = p.stats[2 * group], rs = p.stats[2 * group + 1];
    for (int l0 = g.from; g.live && l0 < g.to; l0 += U * p.lines) {
      float x[U][V], up[U][V];
      next_x.take(x);
      next_up.take(up);
      next_x.request(p, g, p.x, l0 + U * p.lines);
      next_up.request(p, g, p.dy, l0 + U * p.lines);
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (l0 + g.line + u * p.lines < g.to)
#pragma unroll
          for (int e = 0; e < V; ++e) {
            const float xhat = (x[u][e] - mu) * rs, t = up[u][e] * group_slope(fmaf(xhat, w[e], b[e]), p.activation);
            db[e] += t;
            dw[e] = fmaf(t, xhat, dw[e]);
          }
    }
    TwoSums s = {0.f, 0.f};
#pragma unroll
    for (int e = 0; e < V; ++e) {
      s.a = fmaf(w[e], db[e], s.a);
      s.b = fmaf(w[e], dw[e], s.b);
      all_dw[e] += dw[e], all_db[e] += db[e];
    }
    const int n = g.n;
    g.n += p.rows_apart;
    const bool more = g.n < p.N;
    if (more) next_x.request(p, g, p.x, g.from), next_up.request(p, g, p.dy, g.from);
    s = group_join(s, TwoSums{0.f, 0.f}, p, g, shared, [](const TwoSums& a, const TwoSums& b) { return TwoSums{a.a + b.a, a.b + b.b}; });
    const int width = p.per_group > 1 ? p.columns : p.width;
    if (g.line == 0 && g.col % width == 0 && g.live) {
      const long long entries = (long long)p.chunks * p.per_group;
      float* out = p.entries + (((long long)n * p.G + g.first_group + g.col / width) * entries + (long long)g.chunk * p.per_group + g.part) * 2;
      out[0] = s.a, out[1] = s.b;
    }
    if (!more) break;
  }
  if (!p.dweight) return;
#pragma unroll
  for (int e = 0; e < V; ++e) lines[0][threadIdx.x * V + e] = all_dw[e], lines[1][threadIdx.x * V + e] = all_db[e];
  __syncthreads();
  if (g.line == 0 && g.live) {
    const long long at = ((long long)row0 * p.chunks + g.chunk) * p.C + g.c;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      for (int i = 1; i < p.lines; ++i) {
        all_dw[e] += lines[0][(i * p.columns + g.col) * V + e];
        all_db[e] += lines[1][(i * p.columns + g.col) * V + e];
      }
      p.dweight[at + e] = all_dw[e], p.dbias[at + e] = all_db[e];
    }
  }
}

template <typename IO, int V> __global__ __launch_bounds__(kGroupThreads) void group_norm_dx_kernel(GroupArgs p) {
  typedef Run<IO, V> R;
  constexpr int U = 4;
  __shared__ float first[kGroupThreads], second[kGroupThreads];
  const GroupPlace g = group_place<V>(p);
  GroupAhead<IO, V, U> next_x, next_up;
  next_x.request(p, g, p.x, g.from);
  next_up.request(p, g, p.dy, g.from);
  const long long own = (long long)g.n * p.G + g.c / p.Cg;
  const float mu = p.stats[2 * own], rs = p.stats[2 * own + 1];
  float w[V], b[V];
  group_params<V>(p.weight, g.c, p.vec_dtype, 1.f, w);
  group_params<V>(p.bias, g.c, p.vec_dtype, 0.f, b);
  const int entries = p.chunks * p.per_group, sub = threadIdx.x & 7;
  for (int i = threadIdx.x >> 3; i < g.groups; i += kGroupThreads / 8) {
    const long long group = (long long)g.n * p.G + g.first_group + i;
    float a = 0.f, b = 0.f;
#pragma unroll 4
    for (int e = sub; e < entries; e += 8) a += p.entries[(group * entries + e) * 2], b += p.entries[(group * entries + e) * 2 + 1];
#pragma unroll
    for (int d = 4; d >= 1; d >>= 1) a += __shfl_down(a, d, 8), b += __shfl_down(b, d, 8);
    if (sub == 0) first[i] = a * p.inv_count, second[i] = b * p.inv_count;
  }
  __syncthreads();
  if (!g.live) return;
  const int mine = p.per_group > 1 ? 0 : g.col / p.width;
  const float m1 = first[mine], m2 = second[mine];
  for (int l0 = g.from; l0 < g.to; l0 += U * p.lines) {
    const rsrc_t to = R::rows(p.dx, ((long long)g.n * p.L + l0) * p.C);
    float x[U][V], up[U][V];
    next_x.take(x);
    next_up.take(up);
    next_x.request(p, g, p.x, l0 + U * p.lines);
    next_up.request(p, g, p.dy, l0 + U * p.lines);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (l0 + g.line + u * p.lines < g.to) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float xhat = (x[u][e] - mu) * rs, t = up[u][e] * group_slope(fmaf(xhat, w[e], b[e]), p.activation);
          x[u][e] = rs * (fmaf(t, w[e], -m1) - xhat * m2);
        }
        R::store(to, (unsigned)((g.line + u * p.lines) * p.C + g.c), x[u]);
      }
  }
}

__global__ __launch_bounds__(256) void group_norm_params_kernel(SumJob weight, SumJob bias) {
  __shared__ float red[8][32];
  if (blockIdx.y == 0) {
    if ((int)blockIdx.x < weight.blocks) run_sum_job(weight, blockIdx.x, red);
  } else if ((int)blockIdx.x < bias.blocks) {
    run_sum_job(bias, blockIdx.x, red);
  }
}

// ---- host -----------------------------------------------------------------------------------------------------------

// What the sizes say about the launches; the scratch sizes come from the same rules with the smallest vector, which needs no less.
struct GroupPlan {
  bool rows;                                                // one position, runs that fit the registers
  int V, slots;
  int64_t sets, entries;                                    // partial parameter gradients; entries of a group
  int64_t rows_side_by_side, sum_rows;                      // many positions: rows of a launch; of the kernel of the sums
};
static GroupPlan group_plan(GroupArgs& a, int64_t N, int64_t L, int64_t C, int64_t G, int V, bool backward) {
  GroupPlan plan;
  memset(&plan, 0, sizeof(plan));
  a.N = (int)N, a.L = (int)L, a.C = (int)C, a.G = (int)G, a.Cg = (int)(C / G), a.width = a.Cg / V;
  a.rows = N * G;
  a.inv_count = (float)(1.0 / ((double)L * (double)a.Cg));
  plan.V = V;
  if (L == 1 && a.width <= 64 * kGroupSlots) {
    plan.rows = true;
    a.lanes = 1;
    while (a.lanes < 64 && a.lanes < a.width) a.lanes *= 2;
    plan.slots = (a.width + a.lanes - 1) / a.lanes;
    const int64_t runs = 64 / a.lanes;
    int64_t step = G;                                       // waves whose runs are a multiple of G
    for (int64_t r = runs; r > 1 && step % 2 == 0; r /= 2) step /= 2;
    const int64_t all = (a.rows + runs - 1) / runs, most = (int64_t)num_compute_units() * (backward ? 8 : 16);
    int64_t waves = all < most ? all : most;
    waves = (waves + step - 1) / step * step;
    a.waves = (int)waves;
    plan.sets = waves * runs / G;
    return plan;
  }
  a.columns = a.width <= kGroupThreads ? a.width * (kGroupThreads / a.width) : kGroupThreads;
  if (a.columns > C / V) a.columns = (int)(C / V);
  a.per_group = (a.width + a.columns - 1) / a.columns;
  a.blocks = a.per_group > 1 ? (int)(G * a.per_group) : (int)((C / V + a.columns - 1) / a.columns);
  a.lines = kGroupThreads / a.columns;
  const int64_t wanted = (2 * (int64_t)num_compute_units() + N * a.blocks - 1) / (N * a.blocks), most = (L + 8 * a.lines - 1) / (8 * a.lines);
  int64_t chunks = wanted < most ? wanted : most;
  if (chunks < 1) chunks = 1;
  a.chunk = (int)((L + chunks - 1) / chunks);
  a.chunks = (int)((L + a.chunk - 1) / a.chunk);
  const int64_t each = (int64_t)a.chunks * a.blocks;
  auto rows = [&](int64_t workgroups) { return each >= workgroups ? 1 : N < workgroups / each ? N : workgroups / each; };
  plan.rows_side_by_side = rows(kGroupGrid);
  plan.sum_rows = rows((int64_t)num_compute_units() * kGroupSums);
  plan.sets = plan.sum_rows * a.chunks;
  plan.entries = (int64_t)a.chunks * a.per_group;
  return plan;
}

static size_t group_up(size_t n) { return (n + 255) & ~(size_t)255; }
static size_t group_entries_bytes(const GroupArgs& a, const GroupPlan& plan, bool backward) {
  return group_up((size_t)a.rows * plan.entries * (backward ? 2 : 3) * 4);
}

static int group_check(const char* who, int64_t N, int64_t L, int64_t C, int64_t G, int activation, int dtype, int vec_dtype) {
  if (N <= 0 || L <= 0 || C <= 0 || G <= 0 || C % G) return fail(RGLRU_E_ARG, "%s: bad sizes N=%lld L=%lld C=%lld groups=%lld", who, (long long)N, (long long)L, (long long)C, (long long)G);
  if (activation != RGLRU_ACT_NONE && activation != RGLRU_ACT_SILU && activation != RGLRU_ACT_GELU) return fail(RGLRU_E_ARG, "%s: unknown activation %d", who, activation);
  for (int d : {dtype, vec_dtype})
    if (d != RGLRU_F32 && d != RGLRU_BF16) return fail(RGLRU_E_ARG, "%s: unknown dtype %d", who, d);
  if (L >= (1ll << 30) || C >= (1ll << 24) || N >= (1ll << 30) / G || N >= (1ll << 38) / (L * C)) return fail(RGLRU_E_UNSUPPORTED, "%s: too large for one launch", who);
  return RGLRU_OK;
}

static int group_vector(int64_t Cg, int dtype, std::initializer_list<const void*> tensors) {
  const int v = dtype == RGLRU_BF16 ? 8 : 4;
  for (const void* t : tensors)
    if (reinterpret_cast<uintptr_t>(t) % 16 != 0) return 1;
  return Cg % v == 0 ? v : 1;
}

template <bool BACKWARD> static void group_rows(const GroupArgs& a, const GroupPlan& plan, int dtype, hipStream_t s) {
  const dim3 grid((unsigned)((a.waves + kGroupThreads / 64 - 1) / (kGroupThreads / 64)));
#define RGLRU_GROUP_ROWS(IO, V)                                                                                                    \
  do {                                                                                                                            \
    if (plan.slots <= 1) hipLaunchKernelGGL((group_norm_rows_kernel<IO, V, 1, BACKWARD>), grid, dim3(kGroupThreads), 0, s, a);      \
    else if (plan.slots <= 2) hipLaunchKernelGGL((group_norm_rows_kernel<IO, V, 2, BACKWARD>), grid, dim3(kGroupThreads), 0, s, a); \
    else hipLaunchKernelGGL((group_norm_rows_kernel<IO, V, kGroupSlots, BACKWARD>), grid, dim3(kGroupThreads), 0, s, a);            \
  } while (0)
  if (dtype == RGLRU_BF16) { if (plan.V > 1) RGLRU_GROUP_ROWS(__bf16, 8); else RGLRU_GROUP_ROWS(__bf16, 1); }
  else { if (plan.V > 1) RGLRU_GROUP_ROWS(float, 4); else RGLRU_GROUP_ROWS(float, 1); }
#undef RGLRU_GROUP_ROWS
}

// One launch, or several where there are more rows than one holds.
template <typename LAUNCH> static int group_rows_launches(GroupArgs a, const GroupPlan& plan, const char* what, LAUNCH launch) {
  for (int64_t row = 0; row < a.N; row += plan.rows_side_by_side) {
    const int64_t rows = a.N - row < plan.rows_side_by_side ? a.N - row : plan.rows_side_by_side;
    a.row0 = (int)row;
    launch(a, dim3((unsigned)(rows * a.chunks * a.blocks)));
    const int rc = check_launch(what);
    if (rc) return rc;
  }
  return RGLRU_OK;
}

#define RGLRU_GROUP_LAUNCH(KERNEL, dtype, V, grid, s, a)                                                                          \
  do {                                                                                                                            \
    if (dtype == RGLRU_BF16) { if (V > 1) hipLaunchKernelGGL((KERNEL<__bf16, 8>), grid, dim3(kGroupThreads), 0, s, a); else hipLaunchKernelGGL((KERNEL<__bf16, 1>), grid, dim3(kGroupThreads), 0, s, a); } \
    else { if (V > 1) hipLaunchKernelGGL((KERNEL<float, 4>), grid, dim3(kGroupThreads), 0, s, a); else hipLaunchKernelGGL((KERNEL<float, 1>), grid, dim3(kGroupThreads), 0, s, a); } \
  } while (0)

}  // namespace rglru

using namespace rglru;

extern "C" {

size_t rglru_hip_group_norm_scratch_bytes(int64_t N, int64_t L, int64_t C, int64_t G, int backward) {
  if (N <= 0 || L <= 0 || C <= 0 || G <= 0 || C % G) return 0;
  size_t most = 0;
  for (int v : {1, 4, 8}) {
    if ((C / G) % v) continue;
    GroupArgs a;
    memset(&a, 0, sizeof(a));
    const GroupPlan plan = group_plan(a, N, L, C, G, v, backward != 0);
    const size_t n = group_entries_bytes(a, plan, backward != 0) + (backward ? 2 * group_up((size_t)plan.sets * C * 4) : 0);
    if (n > most) most = n;
  }
  return most ? most : 256;
}

int rglru_hip_group_norm_fwd(const void* x, const void* weight, const void* bias, void* y, float* stats, void* scratch, int64_t N, int64_t L,
                             int64_t C, int64_t G, float eps, int activation, int dtype, int vec_dtype, void* stream) {
  int rc = group_check("group_norm_fwd", N, L, C, G, activation, dtype, vec_dtype);
  if (rc) return rc;
  if (!x || !y || !scratch) return fail(RGLRU_E_ARG, "group_norm_fwd: null pointer");
  GroupArgs a;
  memset(&a, 0, sizeof(a));
  const GroupPlan plan = group_plan(a, N, L, C, G, group_vector(C / G, dtype, {x, y}), false);
  a.x = x, a.weight = weight, a.bias = bias, a.y = y, a.stats = stats, a.entries = (float*)scratch;
  a.eps = eps, a.activation = activation, a.vec_dtype = vec_dtype;
  hipStream_t s = (hipStream_t)stream;
  if (plan.rows) {
    group_rows<false>(a, plan, dtype, s);
    return check_launch("group_norm_fwd");
  }
  rc = group_rows_launches(a, plan, "group_norm_fwd moments", [&](const GroupArgs& a, dim3 grid) { RGLRU_GROUP_LAUNCH(group_norm_moments_kernel, dtype, plan.V, grid, s, a); });
  if (rc) return rc;
  return group_rows_launches(a, plan, "group_norm_fwd", [&](const GroupArgs& a, dim3 grid) { RGLRU_GROUP_LAUNCH(group_norm_apply_kernel, dtype, plan.V, grid, s, a); });
}

int rglru_hip_group_norm_bwd(const void* x, const void* weight, const void* bias, const float* stats, const void* dy, void* scratch, void* dx,
                             void* dweight, void* dbias, int64_t N, int64_t L, int64_t C, int64_t G, int activation, int dtype, int vec_dtype,
                             int grad_dtype, void* stream) {
  int rc = group_check("group_norm_bwd", N, L, C, G, activation, dtype, vec_dtype);
  if (rc) return rc;
  if (grad_dtype != RGLRU_F32 && grad_dtype != RGLRU_BF16) return fail(RGLRU_E_ARG, "group_norm_bwd: unknown gradient dtype %d", grad_dtype);
  if (!x || !stats || !dy || !scratch || !dx) return fail(RGLRU_E_ARG, "group_norm_bwd: null pointer");
  GroupArgs a;
  memset(&a, 0, sizeof(a));
  const GroupPlan plan = group_plan(a, N, L, C, G, group_vector(C / G, dtype, {x, dy, dx}), true);
  a.x = x, a.weight = weight, a.bias = bias, a.dy = dy, a.dx = dx, a.stats = const_cast<float*>(stats), a.entries = (float*)scratch;
  a.activation = activation, a.vec_dtype = vec_dtype;
  const bool params = dweight || dbias;
  if (params) {
    a.dweight = (float*)((char*)scratch + group_entries_bytes(a, plan, true));
    a.dbias = (float*)((char*)a.dweight + group_up((size_t)plan.sets * C * 4));
  }
  hipStream_t s = (hipStream_t)stream;
  if (plan.rows) {
    group_rows<true>(a, plan, dtype, s);
    rc = check_launch("group_norm_bwd");
  } else {
    a.rows_apart = (int)plan.sum_rows;
    const dim3 grid((unsigned)(plan.sum_rows * a.chunks * a.blocks));
    RGLRU_GROUP_LAUNCH(group_norm_sums_kernel, dtype, plan.V, grid, s, a);
    rc = check_launch("group_norm_bwd sums");
    if (rc) return rc;
    rc = group_rows_launches(a, plan, "group_norm_bwd", [&](const GroupArgs& a, dim3 grid) { RGLRU_GROUP_LAUNCH(group_norm_dx_kernel, dtype, plan.V, grid, s, a); });
  }
  if (rc || !params) return rc;
  SumJob jobs[2];
  memset(jobs, 0, sizeof(jobs));
  unsigned blocks = 0;
  for (int i = 0; i < 2; ++i) {
    SumJob& j = jobs[i];
    j.dst = i ? dbias : dweight;
    if (!j.dst) continue;                                   // no workgroups
    j.src = i ? a.dbias : a.dweight, j.n = C, j.sets = (int)plan.sets, j.dst_bf16 = grad_dtype == RGLRU_BF16;
    plan_sum_job(j);
    blocks = (unsigned)j.blocks > blocks ? (unsigned)j.blocks : blocks;
  }
  hipLaunchKernelGGL(group_norm_params_kernel, dim3(blocks, 2), dim3(256), 0, s, jobs[0], jobs[1]);
  return check_launch("group_norm_bwd parameters");
}

}  // extern "C"
