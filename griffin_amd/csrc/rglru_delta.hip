// Gated delta rule over whole sequences, forward.  A value head carries a [dk, dv] state S:
//   S_t = a_t (I - beta_t k_t k_t^T) S_{t-1} + beta_t k_t v_t^T,   o_t = scale S_t^T q_t,   a_t = exp(log_decay_t)
// Per chunk of 64 tokens, with G the running log decay in the chunk and D_ij = e^(G_i - G_j) for j <= i in one document:
//   Z  = T (V - rho K S)            T = (I + stril(D . K K^T) diag(beta))^-1,  rho_i = e^(G_i), 0 behind a document start
//   O  = scale rho Q S + P Z        P = scale tril(D . Q K^T) diag(beta)
//   S' = rho_63 S + K^T (w Z)       w_j = beta_j e^(G_63 - G_j), 0 in front of a document start
// T and P do not depend on the state: a first kernel makes them for all chunks side by side.  The second walks along the chunks:
// a wave owns 16 columns of the state, whose products never need another wave's columns.  Where there are fewer such walks than the
// device has room for, a sequence is walked in segments (delta_best_segments): what each adds to the state and makes of it, the
// states joined along the segments, the outputs from these.
//
// Chunks of 64: the products within a chunk grow with its length (64 x 64 x 128 twice), those with the state do not, and
// the tiles of two chunks fit the LDS.  B8 T2048, 8 heads of 128 x 128 in bf16, saving for the backward pass: 43 + 155 us, against 97 for
// the 500 MB of both kernels at the rate of a large copy.  One sequence of 32768 tokens and 20 heads: 179 + 310 + 43 + 300 us, against 385 for 1.97 GB.

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

// T, P and the gate record of one chunk and value head.  A wave owns 16 rows of both; its operands come straight from memory (a row's
// 64 bytes a quarter of the wave) and T and P take turns in LDS, so that five workgroups share a compute unit: what one of them does
// is short, and one after the other.  (Keys of 128 in bf16 put one register aside in scratch for it.)
template <typename IO, int KS> __global__ __launch_bounds__(kDeltaThreads, sizeof(IO) == 2 ? 5 : 3) void delta_prepare_kernel(DeltaArgs p) {
  typedef Mx<IO> M;
  typedef typename M::Frag Frag;
  typedef Tile<IO, 64> Square;
  constexpr int PL = M::kPlanes;
  // A, T in its place once it has been read, P behind that
  __shared__ __attribute__((aligned(16))) unsigned char area[64 * kLowStride * 4];
  __shared__ __attribute__((aligned(16))) float inv[64 * kInvStride];
  float* const low = (float*)area;
  __shared__ double total[64];
  __shared__ float beta[64];
  __shared__ int segment[64];
  const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // the heads of a chunk side by side: what they read lies side by side
  const int work = xcd_order(blockIdx.x, p.nC * p.B * p.HV);
  if (work < 0) return;
  const int hv = work % p.HV, n = work / p.HV % p.nC, b = work / p.HV / p.nC, h = hv / (p.HV / p.H);
  const long long chunk = ((long long)b * p.HV + hv) * p.nC + n;
  const int t0 = n * kDeltaChunk, left = p.T - t0;
  const IO *keys = (const IO*)p.k + b * p.k_b + t0 * p.k_t + h * p.k_h, *queries = (const IO*)p.q + b * p.q_b + t0 * p.q_t + h * p.q_h;
  auto rows = [&](const IO* base, long long stride, int row, Frag (&f)[KS]) {
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      i32x4 v[sizeof(IO) / 2] = {};
      const int col = 32 * ks + 8 * g;
#pragma unroll
      for (int i = 0; i < (int)sizeof(IO) / 2; ++i)
        if (row < left && col + i * 4 < p.width) v[i] = *reinterpret_cast<const i32x4*>(base + row * stride + col + i * 4);
      __builtin_memcpy(&f[ks], v, sizeof(Frag));
    }
  };
  auto mask = [&](Frag (&f)[KS], bool counts) {              // whatever a masked token holds
    if (!counts) __builtin_memset(&f, 0, sizeof(f));
  };
  Frag ki[KS], qi[KS], kj[KS];
  rows(keys, p.k_t, 16 * wave + c, ki);
  rows(queries, p.q_t, 16 * wave + c, qi);
  const ChunkGates gate = chunk_gates(p, b, hv, n, lane);
  const unsigned long long counts = __ballot(gate.counts), starts = __ballot(gate.starts);
  if (wave == 0) {
    total[lane] = gate.total;
    beta[lane] = gate.beta;
    segment[lane] = gate.segment;
    float* record = p.gates + chunk * kDeltaGates;
    record[lane] = gate.counts && gate.segment == 0 ? expf((float)gate.total) : 0.f;
    record[64 + lane] = gate.segment == gate.segments ? gate.beta * expf((float)(gate.end - gate.total)) : 0.f;
    if (lane < 2) record[128 + lane] = __uint_as_float((unsigned)(counts >> (32 * lane)));
    if (lane == 2) record[130] = (starts & (0 - counts) & counts) != 0 ? 1.f : 0.f;
    if (lane == 3) record[131] = gate.segments == 0 ? expf((float)gate.end) : 0.f;
  }
  mask(ki, (counts >> (16 * wave + c)) & 1);
  mask(qi, (counts >> (16 * wave + c)) & 1);
  __syncthreads();
  const int i0 = 16 * wave + 4 * g;                        // first of the lane's four rows
  double total_i[4];
  int segment_i[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) total_i[e] = total[i0 + e], segment_i[e] = segment[i0 + e];
  f32x4 within[4] = {};
#pragma unroll
  for (int jt = 0; jt < 4; ++jt) {
    const int j = 16 * jt + c;
    if (jt <= wave) {
      f32x4 kk = {0.f, 0.f, 0.f, 0.f}, qk = {0.f, 0.f, 0.f, 0.f};
      rows(keys, p.k_t, j, kj);
      mask(kj, (counts >> j) & 1);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        kk = M::ee(ki[ks], kj[ks], kk);
        qk = M::ee(qi[ks], kj[ks], qk);
      }
      const double total_j = total[j];
      const float beta_j = beta[j];
      const int segment_j = segment[j];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = i0 + e;
        const bool joined = i >= j && segment_i[e] == segment_j;
        const float d = beta_j * __expf(joined ? (float)(total_i[e] - total_j) : 0.f);
        kk[e] = joined && i > j ? d * kk[e] : 0.f;
        within[jt][e] = joined ? p.scale * d * qk[e] : 0.f;
        low[i * kLowStride + j] = kk[e];
      }
    }
    phase();
  }
  wave_lds_fence();
  // inverse of the wave's diagonal block by substitution, a column a lane (the four quarters do the same)
  {
    float x[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float s = i == c ? 1.f : 0.f;
#pragma unroll
      for (int j0 = 0; j0 < i; j0 += 4) {
        const f32x4 a = *reinterpret_cast<const f32x4*>(low + (16 * wave + i) * kLowStride + 16 * wave + j0);
#pragma unroll
        for (int j = j0; j < j0 + 4; ++j)
          if (j < i) s = fmaf(-a[j - j0], x[j], s);
      }
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
  // whole rows at a time; the quarter above the diagonal is not read by anyone
  auto rows_out = [&](IO* to) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int at = tid + i * kDeltaThreads, row = at / Square::U, u = at % Square::U;
      if ((row & 32) && u < Square::U / 2) continue;
      *reinterpret_cast<i32x4*>(to + chunk * (4096 * PL) + row * 64 + u * Square::E) = *reinterpret_cast<const i32x4*>((const IO*)area + Square::unit(row, u));
    }
    __syncthreads();
  };
  __syncthreads();
#pragma unroll
  for (int it = 0; it < 4; ++it) M::put((IO*)area + Square::at(16 * wave + c, 16 * it + 4 * g), 4096, column[it]);
  rows_out((IO*)p.solve);
#pragma unroll
  for (int jt = 0; jt < 4; ++jt) M::put((IO*)area + Square::at(16 * jt + c, i0), 4096, within[jt]);
  rows_out((IO*)p.within);
}

// The walk along a segment's chunks.  SAVE: what the backward pass needs is left behind.  !OUT: what the segment does to the state, without
// outputs: column groups behind those of the values walk the columns of the unit matrix, with values of nothing.
// STAGES 2: the next chunk's tiles are requested in front of this one's products, and a chunk's results are stored in front of the
// next one's requests (behind them, the wait for the requests would be one for the stores).  STAGES 1: two workgroups share a
// compute unit, one computes while the other waits.
//   A chunk takes 4.9 us with two waves on a compute unit, 7.0 with eight (128 x 128, bf16).  Of the former a third is vector issue (740
// instructions of a wave, half of them conversions of operands), a fifth the matrix units, a fifth waiting for memory; without
// its requests and stores the walk of B8 T2048 takes 104 of 157 us.  What stands in the way is the chain of products from state to state.
template <typename IO, int KS, int WAVES, int STAGES, bool SAVE, bool OUT>
__global__ __launch_bounds__(64 * WAVES, WAVES == 4 && STAGES * KS * (int)sizeof(IO) <= 8 ? 2 : 1) void delta_forward_kernel(DeltaArgs p) {
  typedef Mx<IO> M;
  typedef typename M::Wide Wide;
  typedef typename M::Frag Frag;
  constexpr int DK = 32 * KS, PL = M::kPlanes, THREADS = 64 * WAVES, COLUMNS = 16 * WAVES;
  typedef Tile<IO, DK> Keys;
  typedef Tile<IO, 64> Square;
  typedef Tile<IO, COLUMNS> Values;
  typedef ChunkTiles<IO, KS, WAVES, OUT> Tiles;
  __shared__ __attribute__((aligned(1024))) unsigned char lds[STAGES * Tiles::kBytes];
  const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int value_groups = (p.columns + COLUMNS - 1) / COLUMNS, groups = value_groups + (OUT ? 0 : (DK + COLUMNS - 1) / COLUMNS);
  const int work = xcd_order(blockIdx.x, groups * p.segments * p.B * p.HV);
  if (work < 0) return;
  const int group = work % groups, segment = work / groups % p.segments, head = work / groups / p.segments;
  const int hv = head % p.HV, b = head / p.HV, h = hv / (p.HV / p.H);
  const bool unit = !OUT && group >= value_groups;
  // nothing starts behind the last segment; what it makes of its state is for the backward pass
  if (!OUT && segment == p.segments - 1 && !(unit && p.states)) return;
  const int col = (unit ? group - value_groups : group) * COLUMNS + wave * 16 + c, width = unit ? DK : p.columns;
  const bool mine = col - c < width, live = mine && (unit || col < p.V);
  const int begin = segment * p.length, end = begin + p.length < p.nC ? begin + p.length : p.nC;
  const long long first = (long long)head * p.nC;
  const unsigned lds0 = lds_address(lds);

  Tiles tiles;
  tiles.setup(p, tid, (const IO*)p.v + b * p.v_b + hv * p.v_h + group * COLUMNS, p.v_t, unit ? 0 : p.value_width - group * COLUMNS, first + begin,
              begin, b, h, 1);
  const bool vectors = p.value_width == p.V;
  bool cut = false;                                        // some chunk leaves nothing of the state
  f32x4 state[2 * KS], o[4], z[4];
  Wide zw[2];
  WaveRows<IO, COLUMNS> rows_out;
  auto request = [&](int stage) { tiles.request(p, lds0 + (unsigned)(stage * Tiles::kBytes), wave); };
  // a chunk's matrix of `rows` elements a column, by eight of a column a lane
  const unsigned plane_bytes = (unsigned)p.columns * (unsigned)sizeof(IO);
  const bool past = WAVES == 2 && p.past != 0;
  auto matrix = [&](void* base, int n, int rows) {
    return make_rsrc((IO*)base + (first + n) * PL * p.columns * rows, PL * plane_bytes * (unsigned)rows);
  };
  auto put = [&](int n) {                                  // results of chunk n
    if constexpr (SAVE) {
      if (mine) {
        const rsrc_t r = matrix(p.values, n, 64);
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) M::put(r, (unsigned)(col * 64 + 32 * ks + 8 * g) * (unsigned)sizeof(IO), plane_bytes * 64, zw[ks], past);
      }
    }
    if constexpr (OUT) {
      const int t0 = n * kDeltaChunk;
      const long long stride = (long long)p.HV * p.V;
      IO* at = (IO*)p.out + (((long long)b * p.T + t0) * p.HV + hv) * p.V;
      if (vectors) {
        if (mine) rows_out.store(at, stride, p.T - t0, p.V, col - c, lane);
      } else {
        ColumnIo<IO>(at, stride, p.T - t0, p.V, col, live, 8 * g).store(o);
      }
    }
  };
  request(0);
  if (!OUT) {
#pragma unroll
    for (int t = 0; t < 2 * KS; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) state[t][e] = unit && tile_index(t, 4 * g + e) == col ? 1.f : 0.f;
  } else if (p.segments > 1) {
    const float* at = p.edges + (((long long)head * p.segments + segment) * p.columns + (mine ? col : 0)) * DK;
#pragma unroll
    for (int t = 0; t < 2 * KS; ++t) state[t] = *reinterpret_cast<const f32x4*>(at + tile_index(t, 4 * g));
  } else {
#pragma unroll
    for (int t = 0; t < 2 * KS; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int row = tile_index(t, 4 * g + e);
        state[t][e] = p.h0 && live && row < p.K ? p.h0[((long long)head * p.K + row) * p.V + col] : 0.f;
      }
  }
  wait_for_all();
  for (int n = begin; n < end; ++n) {
    const int stage = STAGES == 2 ? (n - begin) & 1 : 0;
    unsigned char* tile = lds + stage * Tiles::kBytes;
    const IO *keys = (const IO*)(tile + Tiles::kKeys), *queries = (const IO*)(tile + Tiles::kQueries), *solve = (const IO*)(tile + Tiles::kSolve),
             *within = (const IO*)(tile + Tiles::kWithin);
    const float* record = (const float*)(tile + Tiles::kRecord);
    const ChunkFacts facts(record);
    const float carry = facts.carry;
    if (!OUT) cut = cut || carry == 0.f;
    if (!facts.plain) {
      if (facts.fresh) {
#pragma unroll
        for (int t = 0; t < 2 * KS; ++t) state[t] = f32x4{0.f, 0.f, 0.f, 0.f};
      }
      Tiles::clear_rows(tile, facts.counts, tid);
      lds_barrier();
    }
    if (STAGES == 2 && n > begin) put(n - 1);
    if (STAGES == 2 && n + 1 < end) request(stage ^ 1);
    if (mine) {
      // operands of the next phase are requested in front of a phase's products, or at its start where another workgroup's
      // products fill the wait and the registers are for two
      constexpr int D = STAGES == 2 ? 2 : 1;
      Frag ka[D][4], qa[D][4], kt[D][2 * KS];
      Wide ta[D][4];
      auto rows = [&](int ks) {
#pragma unroll
        for (int mt = 0; mt < 4; ++mt) {
          ka[ks % D][mt] = Keys::along_row(keys, tile_index(mt, c), 32 * ks, g);
          if constexpr (OUT) qa[ks % D][mt] = Keys::along_row(queries, tile_index(mt, c), 32 * ks, g);
        }
      };
      auto square = [&](const IO* x, int ks) {             // lower triangular: rows in front of the columns are zeros
#pragma unroll
        for (int mt = 2 * ks; mt < 4; ++mt) ta[ks % D][mt] = Square::wide_down_rows_tile(x, 4096, 32 * ks, mt, lane);
      };
      auto turned = [&](int ks) {
#pragma unroll
        for (int t = 0; t < 2 * KS; ++t) kt[ks % D][t] = Keys::down_rows_tile(keys, 32 * ks, t, lane);
      };
      phase();
      if (D == 2) rows(0);
      f32x4 rho[4], r[4];
#pragma unroll
      for (int mt = 0; mt < 4; ++mt) rho[mt] = tile_rows(record, mt, g);
      IO* const value_tile = (IO*)(tile + Tiles::kValues);
      // K S and Q S (o) side by side: a tile of the state becomes an operand once
      f32x4 acc[4] = {};
#pragma unroll
      for (int mt = 0; mt < 4; ++mt) o[mt] = f32x4{0.f, 0.f, 0.f, 0.f};
      const rsrc_t saved = matrix(p.states, n, SAVE ? DK : 0);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        if (D == 1) rows(ks);
        else if (ks + 1 < KS) rows(ks + 1);
        else square(solve, 0);
        phase();
        const Wide s = M::wide(state[2 * ks], state[2 * ks + 1]);
        M::ew(acc, ka[ks % D], s);
        if constexpr (OUT) M::ew(o, qa[ks % D], s);
        if constexpr (SAVE) M::put(saved, (unsigned)(col * DK + 32 * ks + 8 * g) * (unsigned)sizeof(IO), plane_bytes * DK, s, past);
        phase();
      }
      square(solve, D - 1);
      if (OUT || !unit) {
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) M::apart(Values::down_rows(value_tile, 32 * ks, 16 * wave, lane), r[2 * ks], r[2 * ks + 1]);
      } else {
#pragma unroll
        for (int mt = 0; mt < 4; ++mt) r[mt] = f32x4{0.f, 0.f, 0.f, 0.f};
      }
      phase();
      // what a masked token would read, whatever it is
      if (!facts.plain) {
#pragma unroll
        for (int mt = 0; mt < 4; ++mt)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[mt][e] = rho[mt][e] == 0.f ? 0.f : acc[mt][e], o[mt][e] = rho[mt][e] == 0.f ? 0.f : o[mt][e];
      }
      // Z = T R, R = V - rho K S
#pragma unroll
      for (int mt = 0; mt < 4; ++mt) {
#pragma unroll
        for (int e = 0; e < 4; ++e) r[mt][e] = fmaf(-rho[mt][e], acc[mt][e], r[mt][e]);
        if constexpr (OUT) o[mt] *= rho[mt] * p.scale;
        z[mt] = f32x4{0.f, 0.f, 0.f, 0.f};
      }
      M::template ww<0, 4>(z, ta[0], M::wide(r[0], r[1]));
      phase();
      if (D == 2) turned(0);
      else square(solve, 1);
      phase();
      M::template ww<2, 4>(z, ta[1 % D], M::wide(r[2], r[3]));
      phase();
      turned(D - 1);
      if (OUT && D == 2) square(within, 0);
      phase();
      // S' = rho_63 S + K^T (w Z)
#pragma unroll
      for (int t = 0; t < 2 * KS; ++t) state[t] *= carry;
      M::ew(state, kt[0], M::wide(z[0] * tile_rows(record + 64, 0, g), z[1] * tile_rows(record + 64, 1, g)));
      phase();
      if (D == 1) turned(1);
      else if (OUT) square(within, 1);
      phase();
      M::ew(state, kt[1 % D], M::wide(z[2] * tile_rows(record + 64, 2, g), z[3] * tile_rows(record + 64, 3, g)));
      if constexpr (OUT) {
        phase();
        if (D == 1) square(within, 0);
        zw[0] = M::wide(z[0], z[1]), zw[1] = M::wide(z[2], z[3]);
        M::template ww<0, 4>(o, ta[0], zw[0]);
        if (D == 1) phase(), square(within, 1);
        M::template ww<2, 4>(o, ta[1 % D], zw[1]);
        if (vectors) rows_out.turn(value_tile, o, wave, lane);
      }
      phase();
    }
    if constexpr (STAGES == 1) {
      lds_barrier();                                       // the tiles have been read
      if (n + 1 < end) request(0);
      put(n);
    }
    wait_for_all();
  }
  if (STAGES == 2) put(end - 1);
  if (!OUT) {
    if (mine && unit) {
      IO* at = (IO*)p.through + (((long long)head * p.segments + segment) * PL * DK + col) * DK;
#pragma unroll
      for (int t = 0; t < 2 * KS; ++t) M::put(at + tile_index(t, 4 * g), DK * DK, state[t]);
      if (group == value_groups && tid == 0) p.cut[(long long)head * p.segments + segment] = cut;
    } else if (mine) {
      float* at = p.local + (((long long)head * p.segments + segment) * p.columns + col) * DK;
#pragma unroll
      for (int t = 0; t < 2 * KS; ++t) *reinterpret_cast<f32x4*>(at + tile_index(t, 4 * g)) = state[t];
    }
  } else if (p.h_last && live && end == p.nC) {
#pragma unroll
    for (int t = 0; t < 2 * KS; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int row = tile_index(t, 4 * g + e);
        if (row < p.K) p.h_last[((long long)head * p.K + row) * p.V + col] = state[t][e];
      }
  }
}

// The states that segments start from: S' = L + M S with what a segment adds (`local`) and makes of its state (`through`, [in][out]).
// BACKWARD: the gradients behind the segments, dS = L + M^T dS'.  A wave owns 16 columns again; M goes to LDS a segment ahead.  Where a
// segment leaves nothing of its state (`cut`: a document starts in it), S' = L without the product, whatever S holds.
template <typename IO, int KS, bool BACKWARD> __global__ __launch_bounds__(kDeltaThreads) void delta_join_kernel(DeltaArgs p) {
  typedef Mx<IO> M;
  typedef typename M::Wide Wide;
  constexpr int DK = 32 * KS, PL = M::kPlanes;
  typedef Tile<IO, DK> Square;
  typedef TileLoad<IO, PL * DK, DK, kDeltaThreads> Load;
  __shared__ __attribute__((aligned(1024))) unsigned char lds[2 * Load::kBytes];
  const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int groups = (p.columns + 63) / 64, group = (int)(blockIdx.x % (unsigned)groups), head = (int)(blockIdx.x / (unsigned)groups);
  const int col = group * 64 + wave * 16 + c;
  const bool mine = col - c < p.columns, live = col < p.V;
  const unsigned lds0 = lds_address(lds);
  const int from = BACKWARD ? p.segments - 1 : 0, to = BACKWARD ? 0 : p.segments - 1, step = BACKWARD ? -1 : 1;
  const float* first = BACKWARD ? p.dh_last : p.h0;
  Load load;
  load.setup(tid, DK, DK);
  auto request = [&](int s, int stage) {
    load.request(delta_rsrc((const IO*)p.through + ((long long)head * p.segments + s) * (PL * DK * DK), Load::kBytes), lds0 + (unsigned)(stage * Load::kBytes), wave);
  };
  f32x4 state[2 * KS], next[2 * KS];
  int next_cut = 0;
  auto added = [&](int s) {
    next_cut = p.cut[(long long)head * p.segments + s];
    const float* at = p.local + (((long long)head * p.segments + s) * p.columns + (mine ? col : 0)) * DK;
#pragma unroll
    for (int t = 0; t < 2 * KS; ++t) next[t] = *reinterpret_cast<const f32x4*>(at + tile_index(t, 4 * g));
  };
  request(from, 0);
  added(from);
#pragma unroll
  for (int t = 0; t < 2 * KS; ++t)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int row = tile_index(t, 4 * g + e);
      state[t][e] = first && live && row < p.K ? first[((long long)head * p.K + row) * p.V + col] : 0.f;
    }
  for (int s = from;; s += step) {
    if (mine) {
      float* at = p.edges + (((long long)head * p.segments + s) * p.columns + col) * DK;
#pragma unroll
      for (int t = 0; t < 2 * KS; ++t) *reinterpret_cast<f32x4*>(at + tile_index(t, 4 * g)) = state[t];
    }
    if (s == to) break;
    const int stage = (s - from) & 1;
    f32x4 sum[2 * KS];
    wait_for_all();
#pragma unroll
    for (int t = 0; t < 2 * KS; ++t) sum[t] = next[t];
    const bool passes = __builtin_amdgcn_readfirstlane(next_cut) == 0;
    if (s + step != to) request(s + step, stage ^ 1), added(s + step);
    const IO* through = (const IO*)(lds + stage * Load::kBytes);
    if (passes) {
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const Wide x = M::wide(state[2 * ks], state[2 * ks + 1]);
        Wide a[2 * KS];
#pragma unroll
        for (int t = 0; t < 2 * KS; ++t)
          a[t] = BACKWARD ? Square::wide_along_row(through, DK * DK, tile_index(t, c), 32 * ks, g) : Square::wide_down_rows_tile(through, DK * DK, 32 * ks, t, lane);
        M::template ww<0, 2 * KS>(sum, a, x);
        phase();
      }
    }
#pragma unroll
    for (int t = 0; t < 2 * KS; ++t) state[t] = sum[t];
  }
}
template <typename IO, int KS> int delta_join(const DeltaArgs& a, bool backward, hipStream_t s) {
  const dim3 grid((unsigned)((a.columns + 63) / 64 * a.B * a.HV));
  if (backward) hipLaunchKernelGGL((delta_join_kernel<IO, KS, true>), grid, dim3(kDeltaThreads), 0, s, a);
  else hipLaunchKernelGGL((delta_join_kernel<IO, KS, false>), grid, dim3(kDeltaThreads), 0, s, a);
  return check_launch("gated_delta segments");
}

template <typename IO, int KS, int WAVES, int STAGES, bool SAVE, bool OUT> static int delta_walk(const DeltaArgs& a, hipStream_t s) {
  const int width = 16 * WAVES, groups = (a.columns + width - 1) / width + (OUT ? 0 : (32 * KS + width - 1) / width);
  const long long total = (long long)groups * a.segments * a.B * a.HV;
  hipLaunchKernelGGL((delta_forward_kernel<IO, KS, WAVES, STAGES, SAVE, OUT>), xcd_grid(total), dim3(64 * WAVES), 0, s, a);
  return check_launch("gated_delta_fwd");
}

template <typename IO, int KS> static int delta_forward(const DeltaArgs& a, bool save, hipStream_t s) {
  hipLaunchKernelGGL((delta_prepare_kernel<IO, KS>), xcd_grid((long long)a.B * a.HV * a.nC), dim3(kDeltaThreads), 0, s, a);
  int rc = check_launch("gated_delta_fwd prepare");
  if (rc) return rc;
  constexpr bool kTwo = sizeof(IO) == 2;                    // two chunks' tiles fit the LDS
  if (a.segments > 1) {
    rc = delta_walk<IO, KS, 4, 1, false, false>(a, s);
    if (!rc) rc = delta_join<IO, KS>(a, false, s);
    if (rc) return rc;
  }
  if constexpr (kTwo)
    if (delta_narrow(a)) return save ? delta_walk<IO, KS, 2, 2, true, true>(a, s) : delta_walk<IO, KS, 2, 2, false, true>(a, s);
  return save ? delta_walk<IO, KS, 4, 1, true, true>(a, s) : delta_walk<IO, KS, 4, 1, false, true>(a, s);
}

// Rows [B, T, H, K] that are no whole 16-byte vectors, as dense ones that are, zeros behind them.
template <typename IO> __global__ __launch_bounds__(256) void delta_pad_kernel(const IO* src, IO* dst, long long rows, int T, int H, int K, int width, long long b_s, long long t_s, long long h_s) {
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < rows * width; i += gridDim.x * 256ll) {
    const long long row = i / width, token = row / H;
    const int col = (int)(i % width);
    dst[i] = col < K ? src[token / T * b_s + token % T * t_s + row % H * h_s + col] : (IO)0.f;
  }
}
int delta_launch_pad(const void* src, void* dst, int B, int T, int H, int K, int width, long long b_s, long long t_s, long long h_s, int dtype, hipStream_t s) {
  const long long rows = (long long)B * T * H, blocks = (rows * width + 255) / 256;
  const dim3 grid((unsigned)(blocks < kDeltaGrid ? blocks : kDeltaGrid));
  if (dtype == RGLRU_BF16) hipLaunchKernelGGL((delta_pad_kernel<__bf16>), grid, dim3(256), 0, s, (const __bf16*)src, (__bf16*)dst, rows, T, H, K, width, b_s, t_s, h_s);
  else hipLaunchKernelGGL((delta_pad_kernel<float>), grid, dim3(256), 0, s, (const float*)src, (float*)dst, rows, T, H, K, width, b_s, t_s, h_s);
  return check_launch("gated_delta rows");
}

int delta_launch_join(const DeltaArgs& a, int dtype, hipStream_t s) {
  switch ((a.K + 31) / 32) {
#define RGLRU_DELTA(KS) case KS: return dtype == RGLRU_BF16 ? delta_join<__bf16, KS>(a, true, s) : delta_join<float, KS>(a, true, s)
    RGLRU_DELTA(1);
    RGLRU_DELTA(2);
    RGLRU_DELTA(3);
    RGLRU_DELTA(4);
#undef RGLRU_DELTA
  }
  return fail(RGLRU_E_UNSUPPORTED, "gated_delta_bwd: key size %d", a.K);
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
