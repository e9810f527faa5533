// Gated delta rule over whole sequences, forward.  A value head carries a [dk, dv] state S:
//   S_t = a_t (I - beta_t k_t k_t^T) S_{t-1} + beta_t k_t v_t^T,   o_t = scale S_t^T q_t,   a_t = exp(log_decay_t)
// Per chunk of 64 tokens, with G the running log decay in the chunk and D_ij = e^(G_i - G_j) for j <= i in one document:
//   Z  = T (V - rho K S)            T = (I + stril(D . K K^T) diag(beta))^-1,  rho_i = e^(G_i), 0 behind a document start
//   O  = scale rho Q S + P Z        P = scale tril(D . Q K^T) diag(beta)
//   S' = rho_63 S + K^T (w Z)       w_j = beta_j e^(G_63 - G_j), 0 in front of a document start
// T and P do not depend on the state: a first kernel makes them for all chunks side by side.  The second walks along the chunks:
// a wave owns 16 columns of the state, whose products never need another wave's columns.

#include <hip/hip_runtime.h>

#include <cstring>

#include "rglru_delta.h"
#include "rglru_host.h"

namespace rglru {

constexpr int kLowStride = 68, kInvStride = 20;            // fp32 rows in LDS, whole vectors, banks apart

// Block column J of T = (I + A)^-1 from A (fp32, strictly lower, `low`) and the inverses of its four diagonal blocks (`inv`):
// T_IJ = -T_II sum over J <= M < I of A_IM T_MJ.  fp32 products: what T is off, every state behind it inherits.
template <int J> RGLRU_DEVICE void delta_solve_column(const float* low, const float* inv, int lane, f32x4 (&column)[4]) {
  const int c = lane & 15, g = lane >> 4;
#pragma unroll
  for (int i = 0; i < 4; ++i) column[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int e = 0; e < 4; ++e) column[J][e] = inv[(J * 16 + 4 * g + e) * kInvStride + c];
#pragma unroll
  for (int i = J + 1; i < 4; ++i) {
    f32x4 sum = {0.f, 0.f, 0.f, 0.f}, solved = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int m = J; m < i; ++m) {
      const f32x4 a = *reinterpret_cast<const f32x4*>(low + (16 * i + c) * kLowStride + 16 * m + 4 * g);
#pragma unroll
      for (int e = 0; e < 4; ++e) sum = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], column[m][e], sum, 0, 0, 0);
    }
    const f32x4 d = *reinterpret_cast<const f32x4*>(inv + (16 * i + c) * kInvStride + 4 * g);
#pragma unroll
    for (int e = 0; e < 4; ++e) solved = __builtin_amdgcn_mfma_f32_16x16x4f32(d[e], sum[e], solved, 0, 0, 0);
    column[i] = -solved;
  }
}

// T, P and the gate record of one chunk and value head.
template <typename IO, int KS> __global__ __launch_bounds__(kDeltaThreads) void delta_prepare_kernel(DeltaArgs p) {
  typedef Mx<IO> M;
  constexpr int DK = 32 * KS;
  typedef Tile<IO, DK> Keys;
  __shared__ __attribute__((aligned(16))) IO keys[kDeltaChunk * DK], queries[kDeltaChunk * DK];
  __shared__ __attribute__((aligned(16))) float low[64 * kLowStride], inv[64 * kInvStride];
  __shared__ double total[64];
  __shared__ float beta[64];
  __shared__ int segment[64];
  const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const long long chunk = blockIdx.x;
  const int n = (int)(chunk % p.nC), head = (int)(chunk / p.nC), hv = head % p.HV, b = head / p.HV, h = hv / (p.HV / p.H);
  const int t0 = n * kDeltaChunk;
  const ChunkGates gate = chunk_gates(p, b, hv, n, lane);
  const unsigned long long counts = __ballot(gate.counts);
  {
    KeyRows<IO, DK, kDeltaThreads> k, q;
    k.request((const IO*)p.k + b * p.k_b + t0 * p.k_t + h * p.k_h, p.k_t, p.width, counts, true, tid);
    q.request((const IO*)p.q + b * p.q_b + t0 * p.q_t + h * p.q_h, p.q_t, p.width, counts, true, tid);
    if (wave == 0) {
      total[lane] = gate.total;
      beta[lane] = gate.beta;
      segment[lane] = gate.segment;
      float* record = p.gates + chunk * kDeltaGates;
      record[lane] = gate.segment == 0 ? expf((float)gate.total) : 0.f;
      record[64 + lane] = gate.segment == gate.segments ? gate.beta * expf((float)(gate.end - gate.total)) : 0.f;
      if (lane < 2) record[128 + lane] = __uint_as_float((unsigned)(counts >> (32 * lane)));
    }
    k.put(keys, tid);
    q.put(queries, tid);
  }
  __syncthreads();
  const int i0 = 16 * wave + 4 * g;                        // first of the lane's four rows
  IO* within = (IO*)p.within + chunk * (4096 * M::kPlanes);
#pragma unroll
  for (int jt = 0; jt < 4; ++jt) {
    const int j = 16 * jt + c;
    f32x4 kk = {0.f, 0.f, 0.f, 0.f}, qk = {0.f, 0.f, 0.f, 0.f};
    if (jt <= wave) {
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const auto at_j = Keys::along_row(keys, j, 32 * ks, g);
        kk = M::ee(Keys::along_row(keys, 16 * wave + c, 32 * ks, g), at_j, kk);
        qk = M::ee(Keys::along_row(queries, 16 * wave + c, 32 * ks, g), at_j, qk);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = i0 + e;
        const bool joined = i >= j && segment[i] == segment[j];
        const float d = joined ? beta[j] * expf((float)(total[i] - total[j])) : 0.f;
        kk[e] = joined && i > j ? d * kk[e] : 0.f;
        qk[e] = joined ? p.scale * d * qk[e] : 0.f;
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) low[(i0 + e) * kLowStride + j] = kk[e];
    }
    M::put(within + j * 64 + i0, 4096, qk);
  }
  wave_lds_fence();
  // inverse of the wave's diagonal block by substitution, a column a lane (the four quarters do the same)
  {
    float x[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float s = i == c ? 1.f : 0.f;
#pragma unroll
      for (int j = 0; j < i; ++j) s = fmaf(-low[(16 * wave + i) * kLowStride + 16 * wave + j], x[j], s);
      x[i] = s;
    }
    if (lane < 16) {
#pragma unroll
      for (int i = 0; i < 16; ++i) inv[(16 * wave + i) * kInvStride + c] = x[i];
    }
  }
  __syncthreads();
  f32x4 column[4];
  if (wave == 0) delta_solve_column<0>(low, inv, lane, column);
  else if (wave == 1) delta_solve_column<1>(low, inv, lane, column);
  else if (wave == 2) delta_solve_column<2>(low, inv, lane, column);
  else delta_solve_column<3>(low, inv, lane, column);
  IO* solve = (IO*)p.solve + chunk * (4096 * M::kPlanes);
#pragma unroll
  for (int it = 0; it < 4; ++it) M::put(solve + (16 * wave + c) * 64 + 16 * it + 4 * g, 4096, column[it]);
}

// The walk along the chunks.  SAVE: what the backward pass needs is left behind; OUT: the outputs are wanted.
// A chunk's results are stored in front of the next one's requests: behind them, the wait for the requests would be one for the stores.
template <typename IO, int KS, int WAVES, bool SAVE, bool OUT>
__global__ __launch_bounds__(64 * WAVES, 1) void delta_forward_kernel(DeltaArgs p) {
  typedef Mx<IO> M;
  typedef typename M::Wide Wide;
  constexpr int DK = 32 * KS, PL = M::kPlanes, THREADS = 64 * WAVES, COLUMNS = 16 * WAVES;
  typedef Tile<IO, DK> Keys;
  typedef Tile<IO, 64> Square;
  typedef ChunkTiles<IO, KS, THREADS, OUT> Tiles;
  constexpr int STAGES = Tiles::kStages;
  __shared__ __attribute__((aligned(1024))) unsigned char lds[STAGES * Tiles::kBytes];
  const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int groups = (p.columns + COLUMNS - 1) / COLUMNS, total = groups * p.B * p.HV;
  const int work = xcd_order(blockIdx.x, total);
  if (work < 0) return;
  const int group = work % groups, head = work / groups, hv = head % p.HV, b = head / p.HV, h = hv / (p.HV / p.H);
  const int col = group * COLUMNS + wave * 16 + c;
  const bool mine = group * COLUMNS + wave * 16 < p.columns, live = mine && col < p.V;
  const long long first = (long long)head * p.nC;
  const unsigned lds0 = lds_address(lds);

  Tiles tiles;
  tiles.setup(p, tid);
  f32x4 state[2 * KS], o[4], z[4];
  int v[4][4];
  auto request = [&](int n, int stage) {
    tiles.request(p, first + n, n, b, h, lds0 + (unsigned)(stage * Tiles::kBytes), wave);
    const int t0 = n * kDeltaChunk;
    const ColumnIo<IO> values((const IO*)p.v + b * p.v_b + t0 * p.v_t + hv * p.v_h, p.v_t, p.T - t0, p.V, col, live, g);
#pragma unroll
    for (int mt = 0; mt < 4; ++mt)
#pragma unroll
      for (int e = 0; e < 4; ++e) v[mt][e] = values.raw(mt, e);
  };
  auto put = [&](int n) {                                  // results of chunk n
    if constexpr (SAVE) {
      if (mine) {
        IO* at = (IO*)p.values + ((first + n) * PL * p.columns + col) * 64;
#pragma unroll
        for (int mt = 0; mt < 4; ++mt) M::put(at + 16 * mt + 4 * g, (long long)p.columns * 64, z[mt]);
      }
    }
    if constexpr (OUT) {
      const int t0 = n * kDeltaChunk;
      const ColumnIo<IO> out((const IO*)p.out + (((long long)b * p.T + t0) * p.HV + hv) * p.V, (long long)p.HV * p.V, p.T - t0, p.V, col, live, g);
#pragma unroll
      for (int mt = 0; mt < 4; ++mt)
#pragma unroll
        for (int e = 0; e < 4; ++e) out.store(mt, e, o[mt][e]);
    }
  };
  request(0, 0);
#pragma unroll
  for (int t = 0; t < 2 * KS; ++t)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int row = 16 * t + 4 * g + e;
      state[t][e] = p.h0 && live && row < p.K ? p.h0[((long long)head * p.K + row) * p.V + col] : 0.f;
    }
  wait_for_all();
  for (int n = 0; n < p.nC; ++n) {
    const int stage = STAGES == 2 ? n & 1 : 0;
    unsigned char* tile = lds + stage * Tiles::kBytes;
    const IO *keys = (const IO*)(tile + Tiles::kKeys), *queries = (const IO*)(tile + Tiles::kQueries), *solve = (const IO*)(tile + Tiles::kSolve),
             *within = (const IO*)(tile + Tiles::kWithin);
    const float* record = (const float*)(tile + Tiles::kRecord);
    const unsigned long long counts = counts_of(record);
    f32x4 r[4];
#pragma unroll
    for (int mt = 0; mt < 4; ++mt)
#pragma unroll
      for (int e = 0; e < 4; ++e) r[mt][e] = ColumnIo<IO>::value(v[mt][e]);
    if (counts != ~0ull) {
      Tiles::clear_rows(tile, counts, tid);
#pragma unroll
      for (int mt = 0; mt < 4; ++mt)
#pragma unroll
        for (int e = 0; e < 4; ++e) r[mt][e] = (counts >> (16 * mt + 4 * g + e)) & 1 ? r[mt][e] : 0.f;
      lds_barrier();
    }
    Wide s[KS];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) s[ks] = M::wide(state[2 * ks], state[2 * ks + 1]);
    if (n) put(n - 1);
    if constexpr (SAVE) {
      if (mine) {
        IO* at = (IO*)p.states + ((first + n) * PL * p.columns + col) * DK;
#pragma unroll
        for (int t = 0; t < 2 * KS; ++t) M::put(at + 16 * t + 4 * g, (long long)p.columns * DK, state[t]);
      }
    }
    if (STAGES == 2 && n + 1 < p.nC) request(n + 1, stage ^ 1);
    if (mine) {
      f32x4 rho[4];
#pragma unroll
      for (int mt = 0; mt < 4; ++mt) rho[mt] = *reinterpret_cast<const f32x4*>(record + 16 * mt + 4 * g);
      const float carry = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(record[63])));
      // R = V - rho K S; where nothing is carried into a document, nothing of it is read either, whatever it is
      f32x4 acc[4] = {};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int mt = 0; mt < 4; ++mt) acc[mt] = M::ew(Keys::along_row(keys, 16 * mt + c, 32 * ks, g), s[ks], acc[mt]);
      if (carry == 0.f) {
#pragma unroll
        for (int mt = 0; mt < 4; ++mt)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[mt][e] = rho[mt][e] == 0.f ? 0.f : acc[mt][e];
      }
#pragma unroll
      for (int mt = 0; mt < 4; ++mt)
#pragma unroll
        for (int e = 0; e < 4; ++e) r[mt][e] = fmaf(-rho[mt][e], acc[mt][e], r[mt][e]);
      // Z = T R
      {
        const Wide rw[2] = {M::wide(r[0], r[1]), M::wide(r[2], r[3])};
#pragma unroll
        for (int mt = 0; mt < 4; ++mt) z[mt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
          for (int mt = 2 * ks; mt < 4; ++mt) z[mt] = M::ww(Square::wide_down_rows(solve, 4096, 32 * ks, 16 * mt, lane), rw[ks], z[mt]);
      }
      // S' = rho_63 S + K^T (w Z)
      {
        f32x4 wz[4];
#pragma unroll
        for (int mt = 0; mt < 4; ++mt) wz[mt] = z[mt] * *reinterpret_cast<const f32x4*>(record + 64 + 16 * mt + 4 * g);
        const Wide zw[2] = {M::wide(wz[0], wz[1]), M::wide(wz[2], wz[3])};
        if (carry == 0.f) {
#pragma unroll
          for (int t = 0; t < 2 * KS; ++t) state[t] = f32x4{0.f, 0.f, 0.f, 0.f};
        } else {
#pragma unroll
          for (int t = 0; t < 2 * KS; ++t) state[t] *= carry;
        }
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
          for (int t = 0; t < 2 * KS; ++t) state[t] = M::ew(Keys::down_rows(keys, 32 * ks, 16 * t, lane), zw[ks], state[t]);
      }
      if constexpr (OUT) {
        const Wide zw[2] = {M::wide(z[0], z[1]), M::wide(z[2], z[3])};
#pragma unroll
        for (int mt = 0; mt < 4; ++mt) o[mt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
          for (int mt = 0; mt < 4; ++mt) o[mt] = M::ew(Keys::along_row(queries, 16 * mt + c, 32 * ks, g), s[ks], o[mt]);
        if (carry == 0.f) {
#pragma unroll
          for (int mt = 0; mt < 4; ++mt)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[mt][e] = rho[mt][e] == 0.f ? 0.f : o[mt][e];
        }
#pragma unroll
        for (int mt = 0; mt < 4; ++mt) o[mt] *= rho[mt] * p.scale;
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
          for (int mt = 2 * ks; mt < 4; ++mt) o[mt] = M::ww(Square::wide_down_rows(within, 4096, 32 * ks, 16 * mt, lane), zw[ks], o[mt]);
      }
    }
    if (STAGES == 1 && n + 1 < p.nC) {
      lds_barrier();                                       // the tiles have been read
      request(n + 1, 0);
    }
    wait_for_all();
  }
  put(p.nC - 1);
  if (p.h_last && live) {
#pragma unroll
    for (int t = 0; t < 2 * KS; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int row = 16 * t + 4 * g + e;
        if (row < p.K) p.h_last[((long long)head * p.K + row) * p.V + col] = state[t][e];
      }
  }
}

template <typename IO, int KS, int WAVES> static void delta_walk_forward(const DeltaArgs& a, bool save, hipStream_t s) {
  const int total = (a.columns + 16 * WAVES - 1) / (16 * WAVES) * a.B * a.HV;
  const dim3 grid((unsigned)((total + 7) / 8 * 8)), block(64 * WAVES);
  if (save) hipLaunchKernelGGL((delta_forward_kernel<IO, KS, WAVES, true, true>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((delta_forward_kernel<IO, KS, WAVES, false, true>), grid, block, 0, s, a);
}

template <typename IO, int KS> static int delta_forward(const DeltaArgs& a, bool save, hipStream_t s) {
  hipLaunchKernelGGL((delta_prepare_kernel<IO, KS>), dim3((unsigned)((long long)a.B * a.HV * a.nC)), dim3(kDeltaThreads), 0, s, a);
  int rc = check_launch("gated_delta_fwd prepare");
  if (rc) return rc;
  if (delta_narrow(a)) delta_walk_forward<IO, KS, 2>(a, save, s);
  else delta_walk_forward<IO, KS, 4>(a, save, s);
  return check_launch("gated_delta_fwd");
}

// Keys that are no whole 16-byte vectors, as rows that are, zeros behind them.
template <typename IO> __global__ __launch_bounds__(256) void delta_pad_kernel(DeltaArgs p, IO* q, IO* k) {
  const long long rows = (long long)p.B * p.T * p.H, i = blockIdx.x * 256ll + threadIdx.x;
  if (i >= rows * p.width) return;
  const long long row = i / p.width;
  const int col = (int)(i % p.width), h = (int)(row % p.H);
  const long long token = row / p.H, b = token / p.T, t = token % p.T;
  q[i] = col < p.K ? ((const IO*)p.q)[b * p.q_b + t * p.q_t + h * p.q_h + col] : (IO)0.f;
  k[i] = col < p.K ? ((const IO*)p.k)[b * p.k_b + t * p.k_t + h * p.k_h + col] : (IO)0.f;
}
int delta_launch_pad(const DeltaArgs& a, void* q, void* k, int dtype, hipStream_t s) {
  const long long n = (long long)a.B * a.T * a.H * a.width;
  if (dtype == RGLRU_BF16) hipLaunchKernelGGL((delta_pad_kernel<__bf16>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, a, (__bf16*)q, (__bf16*)k);
  else hipLaunchKernelGGL((delta_pad_kernel<float>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, a, (float*)q, (float*)k);
  return check_launch("gated_delta_fwd keys");
}

int delta_launch_forward(const DeltaArgs& a, bool save, int dtype, hipStream_t s) {
  switch ((a.K + 31) / 32) {
#define RGLRU_DELTA(KS) case KS: return dtype == RGLRU_BF16 ? delta_forward<__bf16, KS>(a, save, s) : delta_forward<float, KS>(a, save, s)
    RGLRU_DELTA(1);
    RGLRU_DELTA(2);
    RGLRU_DELTA(3);
    RGLRU_DELTA(4);
#undef RGLRU_DELTA
  }
  return fail(RGLRU_E_UNSUPPORTED, "gated_delta_fwd: key size %d", a.K);
}

}  // namespace rglru
