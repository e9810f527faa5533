// Gated delta rule, one token a row with the state updated in place, and the C entry points of all its kernels.

#include <hip/hip_runtime.h>

#include <cstring>

#include "rglru_delta.h"
#include "rglru_host.h"

namespace rglru {

int delta_launch_forward(const DeltaArgs& a, bool save, int dtype, hipStream_t s);
int delta_launch_pad(const void* src, void* dst, int B, int T, int H, int K, int width, long long b_s, long long t_s, long long h_s, int dtype, hipStream_t s);
int delta_launch_backward(const DeltaArgs& a, int dtype, hipStream_t s);

struct DeltaStepArgs {
  const void *q, *k, *v, *log_decay, *beta;
  const unsigned char* flags;
  float* state;
  void* out;
  int H, HV, K, V, groups, decay_dtype, beta_dtype;
  float scale;
};

// A workgroup takes the rows of LC * N columns of one head's state through its registers: read once, written once.  With r = S k and
// s = S q of the state before the token, the state after it is a S + k u, u = beta (v - a r), and the output scale (a s + (q . k) u), so
// both sums over the key run before anything is written.  Bound by that traffic: 256 rows of 8 heads of 128 x 128 (256 MiB) take 53 us,
// 5.0 TB/s, of what a large copy reaches 5.1.
//   Eight lanes of four columns and 32 row groups: a wave reads eight rows' whole 128-byte lines, and enough workgroups are there to fill the
//   device from 16 rows of 8 heads on.  Whole rows of 128 columns a wave take 7.1 us there instead of 6.0, and 38.7 instead of 29.6 for 256 x 16
//   heads of 64 x 64, whose rows they leave half empty.
//   PAST: states of 16 MiB or more go past the caches; by the next token the states of other layers have been there.  us a token past them and
//   through them, by MiB of state: twelve layers in turn 8.1 : 11.9 (16), 15.3 : 20.7 (32), 28.3 : 34.2 (64), 51 : 60 (128), 99 : 117 (256); one state over and
//   over 7.4 : 7.5 (16), 25.9 : 28.4 (64), 49.9 : 48.4 (128), 72.9 : 68.4 (192), 98 : 104 (256).  Below that 6.0 : 6.5 (8) and 4.9 : 5.2 (4) in
//   turn, but 7.0 : 5.9 over and over (37 rows of 12 heads of 72 x 40, 5 MiB).
template <typename IO, int LC, int N, bool PAST> __global__ __launch_bounds__(kDeltaThreads) void delta_step_kernel(DeltaStepArgs p) {
  typedef float vec __attribute__((ext_vector_type(N)));
  constexpr int RG = kDeltaThreads / LC, ROWS = kDeltaMaxKey / RG, WAVES = kDeltaThreads / 64;
  __shared__ float parts[2 * WAVES][LC * N];
  __shared__ float pairs[WAVES];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, lc = tid % LC, rg = tid / LC;
  const int group = blockIdx.x % (unsigned)p.groups, head = blockIdx.x / (unsigned)p.groups, hv = head % p.HV, b = head / p.HV;
  const int h = hv / (p.HV / p.H), col = (group * LC + lc) * N;
  const bool live = col < p.V;
  const unsigned flag = p.flags ? p.flags[b] : 0u;
  IO* out = (IO*)p.out + (long long)head * p.V + col;
  if (flag & 2u) {                                          // a masked token: the state stays as it is
    if (rg == 0 && live)
      for (int e = 0; e < N; ++e) out[e] = (IO)0.f;
    return;
  }
  const float g = delta_gate(p.log_decay, head, p.decay_dtype), beta = delta_gate(p.beta, head, p.beta_dtype);
  const bool fresh = (flag & 1u) || g < kDeltaCut;
  const float decay = fresh ? 0.f : expf(g);
  const IO *k = (const IO*)p.k + ((long long)b * p.H + h) * p.K, *q = (const IO*)p.q + ((long long)b * p.H + h) * p.K;
  float* state = p.state + (long long)head * p.K * p.V + col;
  vec s[ROWS], read = {}, asked = {};
  float key[ROWS], pair = 0.f;
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int row = rg + RG * i;
    s[i] = vec{};
    if (row < p.K && live && !fresh) {
      const vec* at = reinterpret_cast<const vec*>(state + (long long)row * p.V);
      s[i] = PAST ? __builtin_nontemporal_load(at) : *at;
    }
  }
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int row = rg + RG * i;
    key[i] = row < p.K ? (float)k[row] : 0.f;
    const float query = row < p.K ? (float)q[row] : 0.f;
    pair = fmaf(key[i], query, pair);
#pragma unroll
    for (int e = 0; e < N; ++e) {
      read[e] = fmaf(key[i], s[i][e], read[e]);
      asked[e] = fmaf(query, s[i][e], asked[e]);
    }
  }
#pragma unroll
  for (int m = LC; m < 64; m <<= 1) {
    pair += __shfl_xor(pair, m, 64);
#pragma unroll
    for (int e = 0; e < N; ++e) {
      read[e] += __shfl_xor(read[e], m, 64);
      asked[e] += __shfl_xor(asked[e], m, 64);
    }
  }
  if (lane < LC) {
#pragma unroll
    for (int e = 0; e < N; ++e) parts[wave][lane * N + e] = read[e], parts[WAVES + wave][lane * N + e] = asked[e];
    if (lane == 0) pairs[wave] = pair;
  }
  __syncthreads();
  if (!live) return;
  vec change, result;
  pair = 0.f;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) pair += pairs[w];
  const IO* v = (const IO*)p.v + (long long)head * p.V + col;
#pragma unroll
  for (int e = 0; e < N; ++e) {
    float r = 0.f, a = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) r += parts[w][lc * N + e], a += parts[WAVES + w][lc * N + e];
    change[e] = beta * fmaf(-decay, r, (float)v[e]);
    result[e] = p.scale * fmaf(decay, a, pair * change[e]);
  }
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int row = rg + RG * i;
    vec next;
#pragma unroll
    for (int e = 0; e < N; ++e) next[e] = fmaf(decay, s[i][e], key[i] * change[e]);
    if (row < p.K) {
      vec* at = reinterpret_cast<vec*>(state + (long long)row * p.V);
      if constexpr (PAST) __builtin_nontemporal_store(next, at);
      else *at = next;
    }
  }
  if (rg == 0) {
#pragma unroll
    for (int e = 0; e < N; ++e) out[e] = (IO)result[e];
  }
}

// One launch, or several where there are more rows than one holds.
template <typename IO> static int delta_step(DeltaStepArgs a, int64_t B, bool vec, hipStream_t s) {
  const bool past = B * a.HV * a.K * a.V >= (16ll << 20) / 4;
  a.groups = (a.V + 31) / 32;
  const int64_t fit = (kDeltaGrid - 1) / ((int64_t)a.HV * a.groups), each = fit < B ? fit : B;
  auto moved = [](const void* p, int64_t elements, int dtype) { return (const char*)p + elements * (dtype == RGLRU_BF16 ? 2 : 4); };
  const int dtype = sizeof(IO) == 2 ? RGLRU_BF16 : RGLRU_F32;
  for (int64_t row = 0; row < B; row += each) {
    const dim3 grid((unsigned)((B - row < each ? B - row : each) * a.HV * a.groups)), block(kDeltaThreads);
    if (!vec) hipLaunchKernelGGL((delta_step_kernel<IO, 32, 1, false>), grid, block, 0, s, a);
    else if (!past) hipLaunchKernelGGL((delta_step_kernel<IO, 8, 4, false>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((delta_step_kernel<IO, 8, 4, true>), grid, block, 0, s, a);
    const int rc = check_launch("gated_delta_step");
    if (rc) return rc;
    a.q = moved(a.q, each * a.H * a.K, dtype), a.k = moved(a.k, each * a.H * a.K, dtype), a.v = moved(a.v, each * a.HV * a.V, dtype);
    a.out = (void*)moved(a.out, each * a.HV * a.V, dtype), a.state += each * a.HV * a.K * a.V;
    a.log_decay = moved(a.log_decay, each * a.HV, a.decay_dtype), a.beta = moved(a.beta, each * a.HV, a.beta_dtype);
    if (a.flags) a.flags += each;
  }
  return RGLRU_OK;
}

// ---- host -----------------------------------------------------------------------------------------------------------

// Segments of `length` chunks that a sequence is walked in side by side.  One walk takes as long as its chunks, however many compute units
// stand idle; in segments, all of them are walked twice (what a segment adds to the state and what it makes of it, 128 further
// columns; then the outputs from the joined states).  The number is the one with the least time by what launches of both kinds measure, us a
// chunk of a round of workgroups (bf16, keys and values of 128; it is their ratios that decide, also for other sizes and fp32).  Against the best of
// twelve numbers tried, of seven shapes with and without gradients (B1 T2048 H4 of 64 x 64 to B1 T32768 H4 of 128 x 128): bf16 within 5 %, fp32 within
// 10 %, but for prefills of B3 T777 H8 of 96 x 80, which it leaves whole: 57 us instead of 52, 133 instead of 107.
static int64_t delta_best_segments(int64_t heads, int64_t columns, int64_t width, int64_t nC, bool two, bool keep) {
  const int64_t cus = num_compute_units(), groups = (columns + 63) / 64, units = (width + 63) / 64;
  auto rounds = [&](int64_t n, double alone, double shared) {  // one workgroup a compute unit, or two that share it
    if (n <= cus) return alone;
    return two ? (double)((n + 2 * cus - 1) / (2 * cus)) * shared : (double)((n + cus - 1) / cus) * alone;
  };
  int64_t best = 1;
  double least = 0.;
  for (int64_t s = 1; s <= nC && s <= 64; ++s) {
    const int64_t length = (nC + s - 1) / s;
    if (s > 1 && (nC + length - 1) / length != s) continue;
    double us = rounds(heads * groups * s, keep ? 6.5 : 4.8, keep ? 12. : 7.);
    if (s == 1 && two && heads * ((columns + 31) / 32) <= cus) us = keep ? 5. : 4.;
    if (keep) us *= 2.;                                      // the backward walk takes about as long
    if (s > 1) {
      us += rounds(heads * (groups * (s - 1) + units * (keep ? s : s - 1)), 3.2, 4.3);
      if (keep) us += rounds(heads * groups * (s - 1), 3.8, 5.5);
    }
    us = us * (double)length + (s > 1 ? 4. * (double)s * (keep ? 2. : 1.) + 5. : 0.);
    if (s == 1 || us < 0.9 * least || (best > 1 && us < least)) best = s, least = us;
  }
  return best;
}
static void delta_segments(int64_t heads, int64_t columns, int64_t nC, int64_t width, int dtype, bool keep, int64_t& segments, int64_t& length) {
  segments = delta_best_segments(heads, columns, width, nC, dtype == RGLRU_BF16, keep);
  length = (nC + segments - 1) / segments;
  segments = (nC + length - 1) / length;
}

struct DeltaSizes {
  int64_t chunks, columns, width, row, value_row;          // rows: elements of a key and of a value as the kernels read them
  size_t gates, solve, within, q, k, v, states, values, total;  // offsets in the workspace; q, k, v: room where rows have to be padded
  size_t padded_v, through, local, edges, cut, segment_states;
  int64_t segments, length;
  DeltaSizes(int64_t B, int64_t T, int64_t H, int64_t HV, int64_t K, int64_t V, int dtype, bool keep) {
    const int64_t e = dtype == RGLRU_BF16 ? 8 : 4;
    row = (K + e - 1) / e * e, value_row = (V + e - 1) / e * e;
    chunks = B * HV * ((T + kDeltaChunk - 1) / kDeltaChunk);
    columns = (V + 15) / 16 * 16;
    width = (K + 31) / 32 * 32;
    auto up = [](size_t n) { return (n + 255) & ~(size_t)255; };
    const size_t square = up((size_t)chunks * 4096 * 4);
    gates = 0;
    solve = up((size_t)chunks * kDeltaGates * 4);
    within = solve + square;
    const size_t padded = row != K ? up((size_t)(B * T * H * row) * (16 / e)) : 0;
    q = within + square;
    k = q + padded;
    v = k + padded;
    padded_v = value_row != V ? up((size_t)(B * T * HV * value_row) * (16 / e)) : 0;
    states = v + padded_v;
    values = states + (keep ? up((size_t)chunks * columns * width * 4) : 0);
    through = values + (keep ? up((size_t)chunks * columns * 64 * 4) : 0);
    delta_segments(B * HV, columns, (T + kDeltaChunk - 1) / kDeltaChunk, width, dtype, keep, segments, length);
    segment_states = segments > 1 ? up((size_t)(B * HV * segments * columns * width) * 4) : 0;
    local = through + (segments > 1 ? up((size_t)(B * HV * segments * width * width) * 4) : 0);
    edges = local + segment_states;
    cut = edges + segment_states;
    total = cut + (segments > 1 ? up((size_t)(B * HV * segments) * sizeof(int)) : 0);
  }
  size_t scratch_values() const { return ((size_t)chunks * columns * width * 4 + 255) & ~(size_t)255; }
  size_t scratch_up() const { return scratch_values() + (((size_t)chunks * columns * 64 * 4 + 255) & ~(size_t)255); }
  size_t scratch_local() const { return scratch_up() + padded_v; }
  size_t scratch() const { return scratch_local() + 2 * segment_states; }
};

static int delta_check(const char* who, int64_t B, int64_t T, int64_t H, int64_t HV, int64_t K, int64_t V, int dtype, int decay_dtype, int beta_dtype) {
  if (B <= 0 || T <= 0 || H <= 0 || HV <= 0 || K <= 0 || V <= 0) return fail(RGLRU_E_ARG, "%s: sizes must be positive", who);
  if (HV % H) return fail(RGLRU_E_ARG, "%s: %lld value heads do not share %lld key heads evenly", who, (long long)HV, (long long)H);
  for (int d : {dtype, decay_dtype, beta_dtype})
    if (d != RGLRU_F32 && d != RGLRU_BF16) return fail(RGLRU_E_ARG, "%s: unknown dtype %d", who, d);
  if (K > kDeltaMaxKey) return fail(RGLRU_E_UNSUPPORTED, "%s: keys of %lld elements, at most %d are covered", who, (long long)K, kDeltaMaxKey);
  const int64_t most = (int64_t)1 << 30;
  if (B * T * H >= (1ll << 38) / kDeltaMaxKey || B * T * HV >= (1ll << 38) / (V + 8)) return fail(RGLRU_E_UNSUPPORTED, "%s: too large for one launch", who);
  if (H * K >= most / 256 || HV * V >= most / 256) return fail(RGLRU_E_UNSUPPORTED, "%s: tokens wider than %lld elements", who, (long long)(most / 256));
  if (T >= (1ll << 30) || B * HV * ((V + 63) / 64) >= most || B * HV * ((T + kDeltaChunk - 1) / kDeltaChunk) >= most)
    return fail(RGLRU_E_UNSUPPORTED, "%s: too large for one launch", who);
  return RGLRU_OK;
}

// Sizes, strides and the parts of the workspace.
static int delta_operands(const char* who, DeltaArgs& a, const void* q, const void* k, const void* v, const int64_t* strides, void* ws, bool keep,
                          int64_t B, int64_t T, int64_t H, int64_t HV, int64_t K, int64_t V, int dtype) {
  const int64_t dense[9] = {T * H * K, H * K, K, T * H * K, H * K, K, T * HV * V, HV * V, V};
  const int64_t* st = strides ? strides : dense;
  for (int i = 0; i < 9; ++i)
    if (st[i] < 0) return fail(RGLRU_E_ARG, "%s: negative stride", who);
  for (int i = 1; i < 9; i += 3)
    if (st[i] >= (1ll << 30) / 256) return fail(RGLRU_E_UNSUPPORTED, "%s: tokens %lld elements apart", who, (long long)st[i]);
  a.q = q, a.k = k, a.v = v;
  a.q_b = st[0], a.q_t = st[1], a.q_h = st[2], a.k_b = st[3], a.k_t = st[4], a.k_h = st[5], a.v_b = st[6], a.v_t = st[7], a.v_h = st[8];
  a.B = (int)B, a.T = (int)T, a.H = (int)H, a.HV = (int)HV, a.K = (int)K, a.V = (int)V;
  a.nC = (int)((T + kDeltaChunk - 1) / kDeltaChunk);
  a.columns = (int)((V + 15) / 16 * 16);
  const DeltaSizes z(B, T, H, HV, K, V, dtype, keep);
  a.width = (int)z.row, a.value_width = (int)z.value_row;
  const int64_t e = dtype == RGLRU_BF16 ? 8 : 4;
  bool whole = reinterpret_cast<uintptr_t>(q) % 16 == 0 && reinterpret_cast<uintptr_t>(k) % 16 == 0;
  for (int i = 0; i < 6; ++i) whole = whole && st[i] % e == 0;
  if (z.row == K && !whole) return fail(RGLRU_E_UNSUPPORTED, "%s: rows of queries and keys must be 16-byte aligned", who);
  whole = reinterpret_cast<uintptr_t>(v) % 16 == 0;
  for (int i = 6; i < 9; ++i) whole = whole && st[i] % e == 0;
  if (v && z.value_row == V && !whole) return fail(RGLRU_E_UNSUPPORTED, "%s: rows of values must be 16-byte aligned", who);
  if (B * HV * ((V + 63) / 64) >= kDeltaGrid || z.chunks >= kDeltaGrid || (keep && z.chunks >= kDeltaGrid / 2))
    return fail(RGLRU_E_UNSUPPORTED, "%s: too large for one launch", who);
  a.segments = (int)z.segments, a.length = (int)z.length;
  const long long kept = z.chunks * z.columns * (z.width + 64) * 4;
  a.past = kept > kLastCache / 2 && kept <= kLastCache;
  char* base = (char*)ws;
  a.through = base + z.through, a.local = (float*)(base + z.local), a.edges = (float*)(base + z.edges), a.cut = (int*)(base + z.cut);
  a.gates = (float*)(base + z.gates);
  a.solve = base + z.solve, a.within = base + z.within;
  if (keep) a.states = base + z.states, a.values = base + z.values;
  return RGLRU_OK;
}
// Queries and keys that are no whole vectors are read from padded copies, which the forward call makes.
static void delta_padded(DeltaArgs& a, void* ws, const DeltaSizes& z) {
  a.q = (char*)ws + z.q, a.k = (char*)ws + z.k;
  a.q_h = a.k_h = a.width, a.q_t = a.k_t = (long long)a.H * a.width, a.q_b = a.k_b = a.T * a.q_t;
}

}  // namespace rglru

using namespace rglru;

extern "C" {

int rglru_hip_gated_delta_max_key_size(void) { return kDeltaMaxKey; }

size_t rglru_hip_gated_delta_workspace_bytes(int64_t B, int64_t T, int64_t H, int64_t HV, int64_t K, int64_t V, int dtype, int keep) {
  if (B <= 0 || T <= 0 || H <= 0 || HV <= 0 || K <= 0 || V <= 0 || K > kDeltaMaxKey || (dtype != RGLRU_F32 && dtype != RGLRU_BF16)) return 0;
  return DeltaSizes(B, T, H, HV, K, V, dtype, keep != 0).total;
}

size_t rglru_hip_gated_delta_scratch_bytes(int64_t B, int64_t T, int64_t HV, int64_t K, int64_t V, int dtype) {
  if (B <= 0 || T <= 0 || HV <= 0 || K <= 0 || V <= 0 || K > kDeltaMaxKey || (dtype != RGLRU_F32 && dtype != RGLRU_BF16)) return 0;
  return DeltaSizes(B, T, 1, HV, K, V, dtype, true).scratch();
}

int rglru_hip_gated_delta_fwd(const void* q, const void* k, const void* v, const int64_t* strides, const void* log_decay, const void* beta,
                              const float* h0, const uint8_t* flags, void* out, float* h_last, void* ws, int keep, float scale, int64_t B, int64_t T,
                              int64_t H, int64_t HV, int64_t K, int64_t V, int dtype, int decay_dtype, int beta_dtype, void* stream) {
  int rc = delta_check("gated_delta_fwd", B, T, H, HV, K, V, dtype, decay_dtype, beta_dtype);
  if (rc) return rc;
  if (!q || !k || !v || !log_decay || !beta || !out || !ws) return fail(RGLRU_E_ARG, "gated_delta_fwd: null pointer");
  if (flags == RGLRU_FLAGS_FIRST_RESET) return fail(RGLRU_E_ARG, "gated_delta_fwd: RGLRU_FLAGS_FIRST_RESET is not a flag array");
  DeltaArgs a;
  memset(&a, 0, sizeof(a));
  rc = delta_operands("gated_delta_fwd", a, q, k, v, strides, ws, keep != 0, B, T, H, HV, K, V, dtype);
  if (rc) return rc;
  a.log_decay = log_decay, a.beta = beta, a.flags = flags, a.h0 = h0, a.out = out, a.h_last = h_last;
  a.decay_dtype = decay_dtype, a.beta_dtype = beta_dtype, a.scale = scale;
  const DeltaSizes z(B, T, H, HV, K, V, dtype, keep != 0);
  char* base = (char*)ws;
  if (a.width != a.K) {
    rc = delta_launch_pad(q, base + z.q, a.B, a.T, a.H, a.K, a.width, a.q_b, a.q_t, a.q_h, dtype, (hipStream_t)stream);
    if (!rc) rc = delta_launch_pad(k, base + z.k, a.B, a.T, a.H, a.K, a.width, a.k_b, a.k_t, a.k_h, dtype, (hipStream_t)stream);
    if (rc) return rc;
    delta_padded(a, ws, z);
  }
  if (a.value_width != a.V) {
    rc = delta_launch_pad(v, base + z.v, a.B, a.T, a.HV, a.V, a.value_width, a.v_b, a.v_t, a.v_h, dtype, (hipStream_t)stream);
    if (rc) return rc;
    a.v = base + z.v;
    a.v_h = a.value_width, a.v_t = (long long)a.HV * a.value_width, a.v_b = a.T * a.v_t;
  }
  return delta_launch_forward(a, keep != 0, dtype, (hipStream_t)stream);
}

int rglru_hip_gated_delta_bwd(const void* q, const void* k, const int64_t* strides, const void* log_decay, const void* beta, const uint8_t* flags,
                              const void* dout, const float* dh_last, void* ws, void* scratch, void* dq, void* dk, void* dv, void* dlog_decay,
                              void* dbeta, float* dh0, float scale, int64_t B, int64_t T, int64_t H, int64_t HV, int64_t K, int64_t V, int dtype,
                              int decay_dtype, int beta_dtype, void* stream) {
  int rc = delta_check("gated_delta_bwd", B, T, H, HV, K, V, dtype, decay_dtype, beta_dtype);
  if (rc) return rc;
  if (!q || !k || !log_decay || !beta || !dout || !ws || !scratch || !dq || !dk || !dv || !dlog_decay || !dbeta)
    return fail(RGLRU_E_ARG, "gated_delta_bwd: null pointer");
  if (flags == RGLRU_FLAGS_FIRST_RESET) return fail(RGLRU_E_ARG, "gated_delta_bwd: RGLRU_FLAGS_FIRST_RESET is not a flag array");
  DeltaArgs a;
  memset(&a, 0, sizeof(a));
  rc = delta_operands("gated_delta_bwd", a, q, k, nullptr, strides, ws, true, B, T, H, HV, K, V, dtype);
  if (rc) return rc;
  const DeltaSizes z(B, T, H, HV, K, V, dtype, true);
  if (a.width != a.K) delta_padded(a, ws, z);
  a.log_decay = log_decay, a.beta = beta, a.flags = flags, a.dout = dout, a.dh_last = dh_last;
  a.dq = dq, a.dk = dk, a.dv = dv, a.dlog_decay = dlog_decay, a.dbeta = dbeta, a.dh0 = dh0;
  a.decay_dtype = decay_dtype, a.beta_dtype = beta_dtype, a.scale = scale;
  a.dstates = scratch, a.dvalues = (char*)scratch + z.scratch_values();
  a.local = (float*)((char*)scratch + z.scratch_local()), a.edges = (float*)((char*)scratch + z.scratch_local() + z.segment_states);
  if (a.value_width != a.V) {
    void* up = (char*)scratch + z.scratch_up();
    rc = delta_launch_pad(dout, up, a.B, a.T, a.HV, a.V, a.value_width, T * HV * V, HV * V, V, dtype, (hipStream_t)stream);
    if (rc) return rc;
    a.dout = up;
  } else if (reinterpret_cast<uintptr_t>(dout) % 16 != 0) {
    return fail(RGLRU_E_UNSUPPORTED, "gated_delta_bwd: dout must be 16-byte aligned");
  }
  a.up_h = a.value_width, a.up_t = (long long)a.HV * a.value_width, a.up_b = a.T * a.up_t;
  return delta_launch_backward(a, dtype, (hipStream_t)stream);
}

int rglru_hip_gated_delta_step(const void* q, const void* k, const void* v, const void* log_decay, const void* beta, float* state,
                               const uint8_t* flags, void* out, float scale, int64_t B, int64_t H, int64_t HV, int64_t K, int64_t V, int dtype,
                               int decay_dtype, int beta_dtype, void* stream) {
  int rc = delta_check("gated_delta_step", B, 1, H, HV, K, V, dtype, decay_dtype, beta_dtype);
  if (rc) return rc;
  if (!q || !k || !v || !log_decay || !beta || !state || !out) return fail(RGLRU_E_ARG, "gated_delta_step: null pointer");
  if (flags == RGLRU_FLAGS_FIRST_RESET) return fail(RGLRU_E_ARG, "gated_delta_step: RGLRU_FLAGS_FIRST_RESET is not a flag array");
  DeltaStepArgs a;
  memset(&a, 0, sizeof(a));
  a.q = q, a.k = k, a.v = v, a.log_decay = log_decay, a.beta = beta, a.state = state, a.flags = flags, a.out = out;
  a.H = (int)H, a.HV = (int)HV, a.K = (int)K, a.V = (int)V, a.decay_dtype = decay_dtype, a.beta_dtype = beta_dtype, a.scale = scale;
  const bool vec = V % 4 == 0 && reinterpret_cast<uintptr_t>(state) % 16 == 0;
  return dtype == RGLRU_BF16 ? delta_step<__bf16>(a, B, vec, (hipStream_t)stream) : delta_step<float>(a, B, vec, (hipStream_t)stream);
}

}  // extern "C"
