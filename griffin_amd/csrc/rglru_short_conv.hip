// Short causal depthwise convolution with an activation in front of a selective scan, whole sequences (forward, reverse mode) and single tokens:
//   pre_t = bias + sum over lags j < K of tap[K - 1 - j] x_{t - j},  y_t = act(pre_t)
// where t - j counts the active tokens of t's document only: a document starts with an empty window, inactive tokens stay out of it and give zeros.
// Reverse mode, with dpre = dy act'(pre):  dx_t = sum over j of tap[K - 1 - j] dpre_{t + j},  dtap[K - 1 - j] = sum of dpre_t x_{t - j},  dbias = sum of dpre
//
// A thread takes a vector of channels through a run of tokens with the window in registers, so that x is read once (and K - 1 tokens around each run
// a second time); the activation's slope is made again from x.  Bound by memory.

#include <hip/hip_runtime.h>

#include <cstring>

#include "rglru_device.h"
#include "rglru_host.h"
#include "rglru_sums.h"

namespace rglru {

constexpr int kShortThreads = 256;
constexpr int kShortTaps = 4;
constexpr int kShortRun = 16;                 // tokens of a run
constexpr int kShortVecs = 32, kShortRuns = kShortThreads / kShortVecs;  // channel vectors and runs of a workgroup

struct ShortArgs {
  const void *x, *state, *taps, *bias, *dy;   // state, bias: or null
  const unsigned char* flags;                 // or null
  void *y, *new_state, *dx, *dstate;          // new_state, dstate: or null
  float* partial;                             // [B][run groups][K + 1][W]
  long long sxb, sxt;                         // elements between x's batch rows and tokens
  int B, T, W, nvec, runs, vec_dtype, activation;
};

template <typename IO, int V> struct ShortRow {
  typedef IO Raw __attribute__((ext_vector_type(V)));
  static RGLRU_DEVICE void load(const IO* p, float (&v)[V]) {
    if constexpr (V == 1) {
      v[0] = (float)*p;
    } else {
      const Raw r = *reinterpret_cast<const Raw*>(p);
#pragma unroll
      for (int e = 0; e < V; ++e) v[e] = (float)r[e];
    }
  }
  static RGLRU_DEVICE void store(IO* p, const float (&v)[V]) {
    if constexpr (V == 1) {
      *p = (IO)v[0];
    } else {
      Raw r;
#pragma unroll
      for (int e = 0; e < V; ++e) r[e] = (IO)v[e];
      *reinterpret_cast<Raw*>(p) = r;
    }
  }
};

RGLRU_DEVICE float short_param(const void* p, long long i, int dtype) { return dtype == RGLRU_BF16 ? (float)((const __bf16*)p)[i] : ((const float*)p)[i]; }

template <int V, int K> RGLRU_DEVICE void short_taps(const ShortArgs& p, int c0, float (&tap)[K][V], float (&bias)[V]) {
#pragma unroll
  for (int v = 0; v < V; ++v) {
    bias[v] = p.bias ? short_param(p.bias, c0 + v, p.vec_dtype) : 0.f;
#pragma unroll
    for (int j = 0; j < K; ++j) tap[j][v] = short_param(p.taps, (long long)(c0 + v) * K + K - 1 - j, p.vec_dtype);  // by lag
  }
}

// The window in front of token t0: win[j] is the input of lag j + 1, zero in front of the document.  Rows of the carried state stand in front of token 0
// and count as the document's.
template <typename IO, int V, int K, bool MASKED>
RGLRU_DEVICE void short_window(const ShortArgs& p, int b, int c0, int t0, float (&win)[K > 1 ? K - 1 : 1][V]) {
  const IO* x = (const IO*)p.x + b * p.sxb + c0;
#pragma unroll
  for (int j = 0; j < K - 1; ++j)
#pragma unroll
    for (int v = 0; v < V; ++v) win[j][v] = 0.f;
  int t = t0 - 1;
  bool open = true;
#pragma unroll
  for (int j = 0; j < K - 1; ++j) {
    unsigned f = 0;
    if constexpr (MASKED) {
      const unsigned char* flags = p.flags + (long long)b * p.T;
      // past inactive tokens, 32 at a time where there are so many
      while (open && t >= 31) {
        unsigned long long w[4];
        __builtin_memcpy(w, flags + t - 31, 32);
        if ((w[0] & w[1] & w[2] & w[3] & 0x0202020202020202ull) != 0x0202020202020202ull) break;
        t -= 32;
      }
      while (open && t >= 0 && (flags[t] & 2u)) --t;
      f = open && t >= 0 ? flags[t] : 0u;
    }
    if (open && t >= 0) {
      ShortRow<IO, V>::load(x + t * p.sxt, win[j]);
      if (f & 1u) open = false;
      --t;
    } else if (open) {                                       // state rows, the newest last
      const int row = K - 1 + t;
      if (p.state && row >= 0) ShortRow<IO, V>::load((const IO*)p.state + ((long long)b * (K - 1) + row) * p.W + c0, win[j]);
      --t;
    }
  }
}

RGLRU_DEVICE float short_act(float v, int activation) { return activation == RGLRU_ACT_SILU ? v * sigmoid_fast(v) : v; }
RGLRU_DEVICE float short_slope(float v, int activation) {
  if (activation != RGLRU_ACT_SILU) return 1.f;
  const float s = sigmoid_fast(v);
  return s * fmaf(v, 1.f - s, 1.f);
}

struct ShortItem { int b, group, run, c0, vec; bool ok; };
// A workgroup: kShortVecs channel vectors of kShortRuns runs of one row, vectors fastest.
template <int V> RGLRU_DEVICE ShortItem short_item(const ShortArgs& p) {
  ShortItem it;
  const unsigned vec_groups = (unsigned)(p.nvec + kShortVecs - 1) / kShortVecs, run_groups = (unsigned)(p.runs + kShortRuns - 1) / kShortRuns;
  unsigned i = blockIdx.x;
  const int vg = (int)(i % vec_groups); i /= vec_groups;
  it.group = (int)(i % run_groups);
  it.b = (int)(i / run_groups);
  it.vec = vg * kShortVecs + (int)(threadIdx.x % kShortVecs);
  it.run = it.group * kShortRuns + (int)(threadIdx.x / kShortVecs);
  it.ok = it.vec < p.nvec && it.run < p.runs;
  it.c0 = (it.vec < p.nvec ? it.vec : 0) * V;
  return it;
}

template <typename IO, int V, int K, bool MASKED> __global__ __launch_bounds__(kShortThreads) void short_conv_kernel(ShortArgs p) {
  const ShortItem it = short_item<V>(p);
  if (!it.ok) return;
  const int b = it.b, c0 = it.c0, t0 = it.run * kShortRun, n = p.T - t0 < kShortRun ? p.T - t0 : kShortRun;
  float tap[K][V], bias[V], win[K > 1 ? K - 1 : 1][V];
  short_taps<V, K>(p, c0, tap, bias);
  short_window<IO, V, K, MASKED>(p, b, c0, t0, win);
  const IO* x = (const IO*)p.x + b * p.sxb + t0 * p.sxt + c0;
  IO* y = (IO*)p.y + ((long long)b * p.T + t0) * p.W + c0;
#pragma unroll 8
  for (int i = 0; i < kShortRun; ++i) {
    if (i >= n) break;
    unsigned f = 0;
    if constexpr (MASKED) f = p.flags[(long long)b * p.T + t0 + i];
    const bool live = !(f & 2u), start = (f & 3u) == 1u;
    float cur[V], out[V];
    ShortRow<IO, V>::load(x + i * p.sxt, cur);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float a = fmaf(cur[v], tap[0][v], bias[v]);
      if constexpr (MASKED) {
#pragma unroll
        for (int j = 0; j < K - 1; ++j) win[j][v] = start ? 0.f : win[j][v];
      }
#pragma unroll
      for (int j = K - 2; j >= 0; --j) {
        a = fmaf(win[j][v], tap[j + 1][v], a);
        if (!MASKED || live) win[j][v] = j ? win[j ? j - 1 : 0][v] : cur[v];
      }
      out[v] = live ? short_act(a, p.activation) : 0.f;
    }
    ShortRow<IO, V>::store(y + (long long)i * p.W, out);
  }
  if (K > 1 && p.new_state && it.run == p.runs - 1) {
#pragma unroll
    for (int j = 0; j < K - 1; ++j) ShortRow<IO, V>::store((IO*)p.new_state + ((long long)b * (K - 1) + K - 2 - j) * p.W + c0, win[j]);
  }
}

// A run owns the gradients of its inputs (the first one those of the state as well).  It walks its outputs and those behind it that still read its
// inputs; a gradient is complete, and written, when K - 1 active tokens of the document are past or the document ends.
template <typename IO, int V, int K, bool MASKED> __global__ __launch_bounds__(kShortThreads) void short_conv_bwd_kernel(ShortArgs p) {
  __shared__ float red[kShortRuns][(K + 1) * V][kShortVecs + 1];
  const ShortItem it = short_item<V>(p);
  const int b = it.b, c0 = it.c0, t0 = it.run * kShortRun, t1 = t0 + kShortRun < p.T ? t0 + kShortRun : p.T;
  float dtap[K][V], dbias[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    dbias[v] = 0.f;
#pragma unroll
    for (int j = 0; j < K; ++j) dtap[j][v] = 0.f;
  }
  if (it.ok) {
    float tap[K][V], bias[V], win[K > 1 ? K - 1 : 1][V], grad[K][V];   // grad[j]: gradient so far of the input of lag j
    int place[K];                                                       // where it goes: a token, -1 - row of the state, or kNowhere
    constexpr int kNowhere = -(1 << 20);
    short_taps<V, K>(p, c0, tap, bias);
    short_window<IO, V, K, MASKED>(p, b, c0, t0, win);
#pragma unroll
    for (int j = 0; j < K; ++j) {
      place[j] = it.run == 0 && j >= 1 ? -1 - (K - 1 - j) : kNowhere;  // before the first token: lag j is the state's row K - 1 - j
#pragma unroll
      for (int v = 0; v < V; ++v) grad[j][v] = 0.f;
    }
    const IO* x = (const IO*)p.x + b * p.sxb + c0;
    const IO* dy = (const IO*)p.dy + (long long)b * p.T * p.W + c0;
    IO* dx = (IO*)p.dx + (long long)b * p.T * p.W + c0;
    auto put = [&](int where, const float (&g)[V]) {
      if (where >= 0) ShortRow<IO, V>::store(dx + (long long)where * p.W, g);
      else if (where != kNowhere && p.dstate) ShortRow<IO, V>::store((IO*)p.dstate + ((long long)b * (K - 1) - 1 - where) * p.W + c0, g);
    };
    // before a token comes in, lag j stands in grad[j - 1]'s place: entry j holds lag j + 1 seen from the next token
    if constexpr (K > 1) {
#pragma unroll
      for (int j = 0; j < K - 1; ++j) place[j] = place[j + 1];
    }
    place[K - 1] = kNowhere;
    int owned = it.run == 0 && K > 1 ? K - 1 : 0;            // entries that wait for outputs
    for (int t = t0; t < p.T && (t < t1 || owned > 0); ++t) {
      unsigned f = 0;
      if constexpr (MASKED) f = p.flags[(long long)b * p.T + t];
      if (MASKED && (f & 2u)) {
        if (t < t1) {
          float none[V];
#pragma unroll
          for (int v = 0; v < V; ++v) none[v] = 0.f;
          ShortRow<IO, V>::store(dx + (long long)t * p.W, none);
        }
        continue;
      }
      if (MASKED && (f & 1u)) {                              // the document ends: what waits is complete
#pragma unroll
        for (int j = 0; j < K - 1; ++j) {
          put(place[j], grad[j]);
          place[j] = kNowhere;
#pragma unroll
          for (int v = 0; v < V; ++v) win[j][v] = 0.f;
        }
        owned = 0;
        if (t >= t1) break;
      }
      float cur[V], up[V];
      ShortRow<IO, V>::load(x + t * p.sxt, cur);
      ShortRow<IO, V>::load(dy + (long long)t * p.W, up);
      // shift: entry j becomes lag j
#pragma unroll
      for (int j = K - 1; j > 0; --j) {
        place[j] = place[j - 1];
#pragma unroll
        for (int v = 0; v < V; ++v) grad[j][v] = grad[j - 1][v];
      }
      place[0] = t < t1 ? t : kNowhere;
      if (t < t1) ++owned;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float a = fmaf(cur[v], tap[0][v], bias[v]);
#pragma unroll
        for (int j = K - 1; j >= 1; --j) a = fmaf(win[j - 1][v], tap[j][v], a);
        const float d = up[v] * short_slope(a, p.activation);
        grad[0][v] = d * tap[0][v];
#pragma unroll
        for (int j = 1; j < K; ++j) grad[j][v] = fmaf(d, tap[j][v], grad[j][v]);
        if (t < t1) {
          dbias[v] += d;
          dtap[0][v] = fmaf(d, cur[v], dtap[0][v]);
#pragma unroll
          for (int j = 1; j < K; ++j) dtap[j][v] = fmaf(d, win[j - 1][v], dtap[j][v]);
        }
#pragma unroll
        for (int j = K - 2; j >= 0; --j) win[j][v] = j ? win[j ? j - 1 : 0][v] : cur[v];
      }
      if (place[K - 1] != kNowhere) {                        // read by its last output
        put(place[K - 1], grad[K - 1]);
        place[K - 1] = kNowhere;
        --owned;
      }
    }
#pragma unroll
    for (int j = 0; j < K - 1; ++j) put(place[j], grad[j]);  // the row ends
  }
#pragma unroll
  for (int v = 0; v < V; ++v) {
    red[threadIdx.x / kShortVecs][K * V + v][threadIdx.x % kShortVecs] = dbias[v];
#pragma unroll
    for (int j = 0; j < K; ++j) red[threadIdx.x / kShortVecs][(K - 1 - j) * V + v][threadIdx.x % kShortVecs] = dtap[j][v];
  }
  __syncthreads();
  const unsigned vec_groups = (unsigned)(p.nvec + kShortVecs - 1) / kShortVecs;
  float* part = p.partial + (long long)(blockIdx.x / vec_groups) * (K + 1) * p.W;
  const int first = (int)(blockIdx.x % vec_groups) * kShortVecs;
  for (int idx = threadIdx.x; idx < (K + 1) * V * kShortVecs; idx += kShortThreads) {
    const int row = idx / kShortVecs, lv = idx - row * kShortVecs, k = row / V, v = row - k * V, ch = (first + lv) * V + v;
    if (first + lv < p.nvec) {
      float sum = 0.f;
#pragma unroll
      for (int q = 0; q < kShortRuns; ++q) sum += red[q][row][lv];
      part[(long long)k * p.W + ch] = sum;
    }
  }
}

template <typename IO, int V, int K> __global__ __launch_bounds__(kShortThreads) void short_conv_step_kernel(ShortArgs p) {
  const long long item = (long long)blockIdx.x * kShortThreads + threadIdx.x;
  if (item >= (long long)p.B * p.nvec) return;
  const int b = (int)(item / p.nvec), c0 = (int)(item - (long long)b * p.nvec) * V;
  const unsigned f = p.flags ? p.flags[b] : 0u;
  IO* y = (IO*)p.y + (long long)b * p.W + c0;
  IO* state = (IO*)p.new_state + (long long)b * (K - 1) * p.W + c0;
  float out[V];
  if (f & 2u) {
#pragma unroll
    for (int v = 0; v < V; ++v) out[v] = 0.f;
    ShortRow<IO, V>::store(y, out);
    return;
  }
  float tap[K][V], bias[V], win[K][V];
  short_taps<V, K>(p, c0, tap, bias);
  ShortRow<IO, V>::load((const IO*)p.x + b * p.sxb + c0, win[0]);
#pragma unroll
  for (int j = 1; j < K; ++j) {
    if (f & 1u) {
#pragma unroll
      for (int v = 0; v < V; ++v) win[j][v] = 0.f;
    } else {
      ShortRow<IO, V>::load(state + (long long)(K - 1 - j) * p.W, win[j]);
    }
  }
#pragma unroll
  for (int v = 0; v < V; ++v) {
    float a = bias[v];
#pragma unroll
    for (int j = 0; j < K; ++j) a = fmaf(win[j][v], tap[j][v], a);
    out[v] = short_act(a, p.activation);
  }
  ShortRow<IO, V>::store(y, out);
#pragma unroll
  for (int j = 0; j < K - 1; ++j) ShortRow<IO, V>::store(state + (long long)(K - 2 - j) * p.W, win[j]);
}

static __global__ __launch_bounds__(256) void short_sums_kernel(SumJob j) {
  __shared__ float red[8][32];
  run_sum_job(j, (int)blockIdx.x, red);
}

static int short_check(const char* who, ShortArgs* a, int64_t B, int64_t T, int64_t W, int64_t K, int64_t sxb, int64_t sxt, int dtype, int vec_dtype,
                       int activation, std::initializer_list<const void*> rows) {
  if (dtype != RGLRU_F32 && dtype != RGLRU_BF16) return fail(RGLRU_E_ARG, "%s: dtype must be RGLRU_F32 or RGLRU_BF16, got %d", who, dtype);
  if (vec_dtype != RGLRU_F32 && vec_dtype != RGLRU_BF16) return fail(RGLRU_E_ARG, "%s: unknown parameter dtype %d", who, vec_dtype);
  if (activation != RGLRU_ACT_NONE && activation != RGLRU_ACT_SILU) return fail(RGLRU_E_ARG, "%s: unknown activation %d", who, activation);
  if (B <= 0 || T <= 0 || W <= 0) return fail(RGLRU_E_ARG, "%s: sizes B=%lld T=%lld W=%lld", who, (long long)B, (long long)T, (long long)W);
  if (K < 1 || K > kShortTaps) return fail(RGLRU_E_UNSUPPORTED, "%s: kernel size %lld outside 1..%d", who, (long long)K, kShortTaps);
  memset(a, 0, sizeof(*a));
  const int v = dtype == RGLRU_BF16 ? 8 : 4;
  bool whole = W % v == 0 && sxb % v == 0 && sxt % v == 0;
  for (const void* q : rows) whole = whole && (uintptr_t)q % 16 == 0;
  if (B >= (1ll << 31) || T >= (1ll << 31) - 64 || W >= (1ll << 31)) return fail(RGLRU_E_UNSUPPORTED, "%s: tensor too large", who);
  a->sxb = sxb; a->sxt = sxt; a->B = (int)B; a->T = (int)T; a->W = (int)W; a->vec_dtype = vec_dtype; a->activation = activation;
  a->nvec = (int)(whole ? W / v : W);
  a->runs = (int)((T + kShortRun - 1) / kShortRun);
  return RGLRU_OK;
}
static long long short_run_groups(long long T) { return ((T + kShortRun - 1) / kShortRun + kShortRuns - 1) / kShortRuns; }
static long long short_blocks(const ShortArgs& a) { return a.B * short_run_groups(a.T) * ((a.nvec + kShortVecs - 1) / kShortVecs); }

#define RGLRU_SHORT_K(KERNEL, IO, V, ...)                                                                                          \
  switch (K) {                                                                                                                     \
    case 1: hipLaunchKernelGGL((KERNEL<IO, V, 1 __VA_ARGS__>), grid, dim3(kShortThreads), 0, (hipStream_t)stream, a); break;       \
    case 2: hipLaunchKernelGGL((KERNEL<IO, V, 2 __VA_ARGS__>), grid, dim3(kShortThreads), 0, (hipStream_t)stream, a); break;       \
    case 3: hipLaunchKernelGGL((KERNEL<IO, V, 3 __VA_ARGS__>), grid, dim3(kShortThreads), 0, (hipStream_t)stream, a); break;       \
    default: hipLaunchKernelGGL((KERNEL<IO, V, 4 __VA_ARGS__>), grid, dim3(kShortThreads), 0, (hipStream_t)stream, a); break;      \
  }
#define RGLRU_SHORT_LAUNCH(KERNEL, ...)                                                                                            \
  do {                                                                                                                             \
    if (dtype == RGLRU_BF16) { if (a.nvec < a.W) { RGLRU_SHORT_K(KERNEL, __bf16, 8, __VA_ARGS__) } else { RGLRU_SHORT_K(KERNEL, __bf16, 1, __VA_ARGS__) } } \
    else { if (a.nvec < a.W) { RGLRU_SHORT_K(KERNEL, float, 4, __VA_ARGS__) } else { RGLRU_SHORT_K(KERNEL, float, 1, __VA_ARGS__) } } \
  } while (0)
#define RGLRU_COMMA ,

}  // namespace rglru

using namespace rglru;

extern "C" {

int rglru_hip_short_conv_fwd(const void* x, int64_t x_batch, int64_t x_token, const void* state, const void* taps, const void* bias, const uint8_t* flags,
                             void* y, void* new_state, int activation, int64_t B, int64_t T, int64_t W, int64_t K, int dtype, int vec_dtype, void* stream) {
  ShortArgs a;
  int rc = short_check("short_conv_fwd", &a, B, T, W, K, x_batch, x_token, dtype, vec_dtype, activation, {x, state, y, new_state});
  if (rc) return rc;
  if (!x || !taps || !y) return fail(RGLRU_E_ARG, "short_conv_fwd: null pointer");
  if (short_blocks(a) >= (1ll << 24)) return fail(RGLRU_E_UNSUPPORTED, "short_conv_fwd: tensor too large");
  a.x = x; a.state = state; a.taps = taps; a.bias = bias; a.flags = flags; a.y = y; a.new_state = new_state;
  const dim3 grid((unsigned)short_blocks(a));
  if (flags) RGLRU_SHORT_LAUNCH(short_conv_kernel, RGLRU_COMMA true); else RGLRU_SHORT_LAUNCH(short_conv_kernel, RGLRU_COMMA false);
  return check_launch("short_conv_fwd");
}

size_t rglru_hip_short_conv_scratch_bytes(int64_t B, int64_t T, int64_t W, int64_t K) {
  if (B <= 0 || T <= 0 || W <= 0 || K < 1 || K > kShortTaps) return 0;
  return (size_t)B * (size_t)short_run_groups(T) * (size_t)(K + 1) * (size_t)W * 4;
}

int rglru_hip_short_conv_bwd(const void* x, int64_t x_batch, int64_t x_token, const void* state, const void* taps, const void* bias, const uint8_t* flags,
                             const void* dy, void* scratch, void* dx, void* dstate, void* dtaps, void* dbias, int activation, int64_t B, int64_t T,
                             int64_t W, int64_t K, int dtype, int vec_dtype, int grad_dtype, void* stream) {
  ShortArgs a;
  int rc = short_check("short_conv_bwd", &a, B, T, W, K, x_batch, x_token, dtype, vec_dtype, activation, {x, state, dy, dx, dstate});
  if (rc) return rc;
  if (!x || !taps || !dy || !scratch || !dx) return fail(RGLRU_E_ARG, "short_conv_bwd: null pointer");
  if (grad_dtype != RGLRU_F32 && grad_dtype != RGLRU_BF16) return fail(RGLRU_E_ARG, "short_conv_bwd: unknown gradient dtype %d", grad_dtype);
  if (short_blocks(a) >= (1ll << 24)) return fail(RGLRU_E_UNSUPPORTED, "short_conv_bwd: tensor too large");
  a.x = x; a.state = state; a.taps = taps; a.bias = bias; a.flags = flags; a.dy = dy; a.dx = dx; a.dstate = dstate; a.partial = (float*)scratch;
  const dim3 grid((unsigned)short_blocks(a));
  if (flags) RGLRU_SHORT_LAUNCH(short_conv_bwd_kernel, RGLRU_COMMA true); else RGLRU_SHORT_LAUNCH(short_conv_bwd_kernel, RGLRU_COMMA false);
  rc = check_launch("short_conv_bwd");
  if (rc || (!dtaps && !dbias)) return rc;
  SumJob j = conv_sum_job(a.partial, dtaps, dbias, W, K, B * short_run_groups(T), grad_dtype);
  plan_sum_job(j);
  hipLaunchKernelGGL(short_sums_kernel, dim3((unsigned)j.blocks), dim3(256), 0, (hipStream_t)stream, j);
  return check_launch("short_conv_bwd sums");
}

int rglru_hip_short_conv_step(const void* x, int64_t x_batch, const void* taps, const void* bias, const uint8_t* flags, void* state, void* y, int activation,
                              int64_t B, int64_t W, int64_t K, int dtype, int vec_dtype, void* stream) {
  ShortArgs a;
  int rc = short_check("short_conv_step", &a, B, 1, W, K, x_batch, 0, dtype, vec_dtype, activation, {x, state, y});
  if (rc) return rc;
  if (!x || !taps || !y || (K > 1 && !state)) return fail(RGLRU_E_ARG, "short_conv_step: null pointer");
  a.x = x; a.taps = taps; a.bias = bias; a.flags = flags; a.y = y; a.new_state = state;
  const long long blocks = (B * (long long)a.nvec + kShortThreads - 1) / kShortThreads;
  if (blocks >= (1ll << 24)) return fail(RGLRU_E_UNSUPPORTED, "short_conv_step: tensor too large");
  const dim3 grid((unsigned)blocks);
  RGLRU_SHORT_LAUNCH(short_conv_step_kernel, );
  return check_launch("short_conv_step");
}

}  // extern "C"
