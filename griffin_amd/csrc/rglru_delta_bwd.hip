// Gated delta rule, reverse mode.  With the notation of the forward pass, dO the upstream gradient and dS' the gradient of the
// state behind a chunk:
//   dZ = P^T dO + w K dS'            Y = T^T dZ            dV = Y
//   dS = rho_63 dS' + Q^T (scale rho dO) - K^T (rho Y)
//   N1 = scale tril(D . dO Z^T)      N2 = -stril(D . Y Z^T)
//   dQ = scale rho dO S^T + (N1 beta) K          dK = E + beta F,  dbeta = k . F
//   E  = -rho Y S^T + (N2 beta) K                F  = N1^T Q + N2^T K + e^(G_63 - G) Z dS'^T
//   dlog_decay_t = sum over i >= t of (scale rho q dO S^T - rho k Y S^T)_i + rho_63 <S, dS'> + sum over j < t of beta_j k_j . e^(G_63 - G_j) (Z dS'^T)_j
//                  + sum over i >= t > j of beta_j (N1_ij q_i + N2_ij k_i) . k_j
// (everything that decays by token t: what is read behind it of what was written in front of it.  Sums over all that a token reads less all that it
// writes would be the same, but their common terms do not cancel to the last bit: what little crosses a strong decay would drown in them, and a
// document's gradient in its neighbours'.  The price is the products of all keys with queries and keys once more: 8 us of the step below.)
// The first kernel walks back along the chunks with dS' as the forward pass walks with S; the second one has no order: a workgroup a chunk and
// key head, which adds up its value heads.
// B8 T2048, 8 heads of 128 x 128 in bf16: 151 + 164 us.  The walk is bound like the forward one.  The second kernel reads what both walks left,
// 490 MB, and takes 112 us with its loads alone, 58 with its products over the columns alone: it is bound by memory in front and by
// what each workgroup does behind its last column, where nothing is loaded.

#include <hip/hip_runtime.h>

#include <cstring>

#include "rglru_delta.h"
#include "rglru_host.h"

namespace rglru {

// LOCAL: what a segment adds to the gradient of the state, from nothing behind it; nothing else is written.
template <typename IO, int KS, int WAVES, int STAGES, bool LOCAL>
__global__ __launch_bounds__(64 * WAVES, WAVES == 4 && STAGES * KS * (int)sizeof(IO) <= 8 ? 2 : 1) void delta_backward_kernel(DeltaArgs p) {
  typedef Mx<IO> M;
  typedef typename M::Wide Wide;
  typedef typename M::Frag Frag;
  constexpr int DK = 32 * KS, PL = M::kPlanes, THREADS = 64 * WAVES, COLUMNS = 16 * WAVES;
  typedef Tile<IO, DK> Keys;
  typedef Tile<IO, 64> Square;
  typedef Tile<IO, COLUMNS> Values;
  typedef ChunkTiles<IO, KS, WAVES, true> Tiles;
  __shared__ __attribute__((aligned(1024))) unsigned char lds[STAGES * Tiles::kBytes];
  const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int groups = (p.columns + COLUMNS - 1) / COLUMNS, total = groups * p.B * p.HV;
  const int work = xcd_order(blockIdx.x, total * p.segments);
  if (work < 0) return;
  const int group = work % groups, segment = work / groups % p.segments, head = work / groups / p.segments;
  const int hv = head % p.HV, b = head / p.HV, h = hv / (p.HV / p.H);
  if (LOCAL && segment == 0) return;                        // nothing ends in front of the first segment
  const int col = group * COLUMNS + wave * 16 + c;
  const bool mine = group * COLUMNS + wave * 16 < p.columns, live = mine && col < p.V;
  const long long first = (long long)head * p.nC;
  const unsigned lds0 = lds_address(lds);

  const int begin = segment * p.length, last = (begin + p.length < p.nC ? begin + p.length : p.nC) - 1;
  Tiles tiles;
  tiles.setup(p, tid, (const IO*)p.dout + b * p.up_b + hv * p.up_h + group * COLUMNS, p.up_t, p.value_width - group * COLUMNS, first + last, last, b, h, -1);
  const bool vectors = p.value_width == p.V;
  f32x4 dstate[2 * KS], y[4];
  WaveRows<IO, COLUMNS> rows_out;
  auto request = [&](int stage) { tiles.request(p, lds0 + (unsigned)(stage * Tiles::kBytes), wave); };
  // a chunk's matrix of `rows` elements a column, by eight of a column a lane
  const unsigned plane_bytes = (unsigned)p.columns * (unsigned)sizeof(IO);
  const bool past = WAVES == 2 && p.past != 0;
  auto matrix = [&](void* base, int n, int rows) {
    return make_rsrc((IO*)base + (first + n) * PL * p.columns * rows, PL * plane_bytes * (unsigned)rows);
  };
  auto put = [&](int n) {                                  // results of chunk n
    if (mine) {
      const rsrc_t r = matrix(p.dvalues, n, 64);
#pragma unroll
      for (int ks = 0; ks < 2; ++ks)
        M::put(r, (unsigned)(col * 64 + 32 * ks + 8 * g) * (unsigned)sizeof(IO), plane_bytes * 64, M::wide(y[2 * ks], y[2 * ks + 1]), past);
    }
    const int t0 = n * kDeltaChunk;
    const long long stride = (long long)p.HV * p.V;
    IO* at = (IO*)p.dv + (((long long)b * p.T + t0) * p.HV + hv) * p.V;
    if (vectors) {
      if (mine) rows_out.store(at, stride, p.T - t0, p.V, col - c, lane);
    } else {
      ColumnIo<IO>(at, stride, p.T - t0, p.V, col, live, 8 * g).store(y);
    }
  };
  request(0);
  if (LOCAL) {
#pragma unroll
    for (int t = 0; t < 2 * KS; ++t) dstate[t] = f32x4{0.f, 0.f, 0.f, 0.f};
  } else if (p.segments > 1) {
    const float* at = p.edges + (((long long)head * p.segments + segment) * p.columns + (mine ? col : 0)) * DK;
#pragma unroll
    for (int t = 0; t < 2 * KS; ++t) dstate[t] = *reinterpret_cast<const f32x4*>(at + tile_index(t, 4 * g));
  } else {
#pragma unroll
    for (int t = 0; t < 2 * KS; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int row = tile_index(t, 4 * g + e);
        dstate[t][e] = p.dh_last && live && row < p.K ? p.dh_last[((long long)head * p.K + row) * p.V + col] : 0.f;
      }
  }
  wait_for_all();
  for (int n = last; n >= begin; --n) {
    const int stage = STAGES == 2 ? (last - n) & 1 : 0;
    unsigned char* tile = lds + stage * Tiles::kBytes;
    const IO *keys = (const IO*)(tile + Tiles::kKeys), *queries = (const IO*)(tile + Tiles::kQueries), *solve = (const IO*)(tile + Tiles::kSolve),
             *within = (const IO*)(tile + Tiles::kWithin);
    const float* record = (const float*)(tile + Tiles::kRecord);
    const ChunkFacts facts(record);
    const float carry = facts.carry;
    if (!facts.plain) {
      Tiles::clear_rows(tile, facts.counts, tid);
      lds_barrier();
    }
    if (STAGES == 2 && !LOCAL && n != last) put(n + 1);
    if (STAGES == 2 && n > begin) request(stage ^ 1);
    if (mine) {
      // operands of the next phase are requested in front of a phase's products, or at its start (as in the forward walk)
      constexpr int D = STAGES == 2 ? 2 : 1;
      Frag ka[D][4], kt[D][2 * KS], uf[2];
      Wide ta[D][4];
      auto rows = [&](int ks) {
#pragma unroll
        for (int mt = 0; mt < 4; ++mt) ka[ks % D][mt] = Keys::along_row(keys, tile_index(mt, c), 32 * ks, g);
      };
      auto square = [&](const IO* x, int ks) {             // upper triangular: rows behind the columns are zeros
#pragma unroll
        for (int mt = 0; mt < 2 * ks + 2; ++mt) ta[ks % D][mt] = Square::wide_along_row(x, 4096, tile_index(mt, c), 32 * ks, g);
      };
      auto turned = [&](const IO* x, int ks) {
#pragma unroll
        for (int t = 0; t < 2 * KS; ++t) kt[ks % D][t] = Keys::down_rows_tile(x, 32 * ks, t, lane);
      };
      phase();
      if (D == 2) rows(0);
      f32x4 rho[4], up[4];
      IO* const up_tile = (IO*)(tile + Tiles::kValues);
#pragma unroll
      for (int mt = 0; mt < 4; ++mt) rho[mt] = tile_rows(record, mt, g);
      // dZ = P^T dO + w K dS'
      f32x4 dz[4] = {};
      const rsrc_t saved = matrix(p.dstates, n, LOCAL ? 0 : DK);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        if (D == 1) rows(ks);
        else if (ks + 1 < KS) rows(ks + 1);
        else square(within, 0);
        phase();
        const Wide d = M::wide(dstate[2 * ks], dstate[2 * ks + 1]);
        M::ew(dz, ka[ks % D], d);
        if constexpr (!LOCAL) M::put(saved, (unsigned)(col * DK + 32 * ks + 8 * g) * (unsigned)sizeof(IO), plane_bytes * DK, d, past);
        phase();
      }
      square(within, D - 1);
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        uf[ks] = Values::down_rows(up_tile, 32 * ks, 16 * wave, lane);
        M::apart(uf[ks], up[2 * ks], up[2 * ks + 1]);
      }
      // what a masked token would receive, whatever it is
      if (!facts.plain) {
#pragma unroll
        for (int mt = 0; mt < 4; ++mt) {
          const f32x4 w = tile_rows(record + 64, mt, g);
#pragma unroll
          for (int e = 0; e < 4; ++e) dz[mt][e] = w[e] == 0.f ? 0.f : dz[mt][e];
        }
      }
#pragma unroll
      for (int mt = 0; mt < 4; ++mt) dz[mt] *= tile_rows(record + 64, mt, g), up[mt] *= rho[mt] * p.scale;
      phase();
      M::template we<0, 2>(dz, ta[0], uf[0]);
      phase();
      if (D == 2) square(solve, 0), turned(queries, 0);
      else square(within, 1);
      phase();
      M::template we<0, 4>(dz, ta[1 % D], uf[1]);
#pragma unroll
      for (int t = 0; t < 2 * KS; ++t) dstate[t] *= carry;
      phase();
      if (D == 2) square(solve, 1);
      else square(solve, 0), turned(queries, 0);
      phase();
      // dS = rho_63 dS' + Q^T (scale rho dO) - K^T (rho Y),  Y = T^T dZ
      M::ew(dstate, kt[0], M::wide(up[0], up[1]));
#pragma unroll
      for (int mt = 0; mt < 4; ++mt) y[mt] = f32x4{0.f, 0.f, 0.f, 0.f};
      M::template ww<0, 2>(y, ta[0], M::wide(dz[0], dz[1]));
      phase();
      if (D == 1) square(solve, 1);
      turned(queries, 1);
      phase();
      M::template ww<0, 4>(y, ta[1 % D], M::wide(dz[2], dz[3]));
      phase();
      if (D == 2) turned(keys, 0);
      phase();
      M::ew(dstate, kt[1 % D], M::wide(up[2], up[3]));
      phase();
      turned(keys, D - 1);
      phase();
      M::ew(dstate, kt[0], M::wide(-rho[0] * y[0], -rho[1] * y[1]));
      if (D == 1) phase(), turned(keys, 1);
      M::ew(dstate, kt[1 % D], M::wide(-rho[2] * y[2], -rho[3] * y[3]));
      if (vectors && !LOCAL) rows_out.turn(up_tile, y, wave, lane);
      phase();
      if (facts.fresh) {
#pragma unroll
        for (int t = 0; t < 2 * KS; ++t) dstate[t] = f32x4{0.f, 0.f, 0.f, 0.f};
      }
    }
    if (STAGES == 1) {
      lds_barrier();                                       // the tiles have been read
      if (n > begin) request(0);
      if (!LOCAL) put(n);
    }
    wait_for_all();
  }
  if (STAGES == 2 && !LOCAL) put(begin);
  if (LOCAL) {
    if (mine) {
      float* at = p.local + (((long long)head * p.segments + segment) * p.columns + col) * DK;
#pragma unroll
      for (int t = 0; t < 2 * KS; ++t) *reinterpret_cast<f32x4*>(at + tile_index(t, 4 * g)) = dstate[t];
    }
  } else if (p.dh0 && live && begin == 0) {
#pragma unroll
    for (int t = 0; t < 2 * KS; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int row = tile_index(t, 4 * g + e);
        if (row < p.K) p.dh0[((long long)head * p.K + row) * p.V + col] = dstate[t][e];
      }
  }
}

// Sum over the sixteen columns of an accumulator row: the lanes of a row of sixteen turn by 8, 4, 2 and 1.
RGLRU_DEVICE float sixteen_sum(float v) {
  v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x128, 0xf, 0xf, true));
  v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x124, 0xf, 0xf, true));
  v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x122, 0xf, 0xf, true));
  v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x121, 0xf, 0xf, true));
  return v;
}

// Sum over the lanes in front, of the same sixteen.
template <int N> RGLRU_DEVICE float sixteen_shift(float v) {  // N lanes up, zeros behind
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x110 | N, 0xf, 0xf, true));
}
RGLRU_DEVICE float sixteen_in_front(float v) {
  v = sixteen_shift<1>(v);
  v += sixteen_shift<1>(v);
  v += sixteen_shift<2>(v);
  v += sixteen_shift<4>(v);
  v += sixteen_shift<8>(v);
  return v;
}
// Sum over the four lanes of a column: rows of sixteen exchanged in pairs, then halves of the wave.
RGLRU_DEVICE float four_rows_sum(float v) {
  const auto rows = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(rows[0]) + __uint_as_float(rows[1]);
  const auto halves = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(halves[0]) + __uint_as_float(halves[1]);
}

// Gradients of queries, keys and gates of one chunk and key head.  Eight waves: four times 16 tokens, by two halves of the key's
// columns; the first half's waves make N1, the second half's N2.  The contractions over the value columns take 32 of them at a time
// through LDS, the next 32 on their way there where two fit; queries, keys, N1 and N2 come where the columns lay.
// Two workgroups share a compute unit in bf16 (kGradShared; one alone: 195 us instead of 176 at B8 T2048 H8 of 128 at the time); fp32 operands and
// the sums over value heads need the registers of one.  Keys of 128 in bf16 put 22 registers aside in scratch for it (96 elements: 6), and so
// does fp32 with value heads that share keys of 128 (13).
constexpr int kGradThreads = 512;
template <typename IO, bool GROUPED> constexpr bool kGradShared = (sizeof(IO) == 2) && !GROUPED;
template <typename IO, int KS, bool GROUPED>
__global__ __launch_bounds__(kGradThreads, (kGradShared<IO, GROUPED>) ? 4 : 2) void delta_grads_kernel(DeltaArgs p) {
  typedef Mx<IO> M;
  typedef typename M::Wide Wide;
  typedef typename M::Frag Frag;
  constexpr int DK = 32 * KS, PL = M::kPlanes, CB = 32, THREADS = kGradThreads;
  typedef Tile<IO, DK> Keys;
  typedef Tile<IO, 64> Square;
  typedef Tile<IO, CB> Ups;
  typedef TileLoad<IO, 64, DK, THREADS> KeyLoad;
  typedef TileLoad<IO, 64, CB, THREADS> UpLoad;
  typedef TileLoad<IO, CB, 64, THREADS> ValueLoad;          // one plane
  typedef TileLoad<IO, CB, DK, THREADS> StateLoad;
  constexpr int kUp = 0, kValues = kUp + UpLoad::kBytes, kDValues = kValues + PL * ValueLoad::kBytes, kStates = kDValues + PL * ValueLoad::kBytes,
                kDStates = kStates + PL * StateLoad::kBytes, kStage = kDStates + PL * StateLoad::kBytes, kRows = 2 * KeyLoad::kBytes + 2 * PL * 4096 * (int)sizeof(IO);
  constexpr int STAGES = 2 * kStage + 6144 <= (kGradShared<IO, GROUPED> ? 80 : 160) * 1024 ? 2 : 1;
  __shared__ __attribute__((aligned(1024))) unsigned char lds[STAGES * kStage > kRows ? STAGES * kStage : kRows];
  __shared__ double total[64];
  __shared__ float beta[64], to_end[64], reads[2][64], writes[2][64], leaves[2][64], sums[8], crossing[2][64], columns_of[8][48];
  __shared__ int segment[64];
  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), block = wave & 3, half = wave >> 2;
  // the heads of a chunk side by side: what they read and write lies side by side
  const int work = xcd_order(blockIdx.x, p.nC * p.B * p.H);
  if (work < 0) return;
  const int h = work % p.H, n = work / p.H % p.nC, b = work / p.H / p.nC;
  const int t0 = n * kDeltaChunk, left = p.T - t0, share = p.HV / p.H;
  if (p.flags) {                                            // no token counts: zeros, whatever state and gradient pass by
    const int t = t0 + (tid & 63);
    if (__ballot(t < p.T && !(p.flags[(long long)b * p.T + (t < p.T ? t : 0)] & 2u)) == 0) {
      const int rows = left < kDeltaChunk ? left : kDeltaChunk;
      for (int row = wave; row < rows; row += THREADS / 64) {
        const long long token = (long long)b * p.T + t0 + row;
        for (int i = tid & 63; i < p.K; i += 64) ((IO*)p.dq)[(token * p.H + h) * p.K + i] = ((IO*)p.dk)[(token * p.H + h) * p.K + i] = (IO)0.f;
        for (int s = tid & 63; s < share; s += 64) {
          delta_put_gate(p.dlog_decay, token * p.HV + h * share + s, p.decay_dtype, 0.f);
          delta_put_gate(p.dbeta, token * p.HV + h * share + s, p.beta_dtype, 0.f);
        }
      }
      return;
    }
  }
  IO *const keys = (IO*)lds, *const queries = (IO*)(lds + KeyLoad::kBytes), *const area = (IO*)(lds + 2 * KeyLoad::kBytes);
  const unsigned lds0 = lds_address(lds);
  f32x4 all_dq[KS] = {}, all_dk[KS] = {};                   // over the value heads that share the key head
  ValueLoad value_load;
  StateLoad state_load;
  value_load.setup(tid, 64, 64);
  state_load.setup(tid, DK, DK);

  for (int s = 0; s < (GROUPED ? share : 1); ++s) {
    // no address that hangs on the lane is kept from head to head: there are more of them than registers
    int lane = tid & 63;
    if (GROUPED) asm("" : "+v"(lane) : "s"(s));
    const int c = lane & 15, g = lane >> 4, row0 = 16 * block + 4 * g;
    const int hv = h * share + s, head = b * p.HV + hv;
    const long long chunk = (long long)head * p.nC + n;
    auto request = [&](int c0, int stage) {
      const int there = p.columns - c0;                     // columns of the values from here on
      const unsigned to = lds0 + (unsigned)(stage * kStage);
      // zeros past the value's last column: what lies there are other heads' and other tokens' gradients, whatever they hold
      const int width = p.value_width - c0 < CB ? p.value_width - c0 : CB;
      UpLoad up_load;
      up_load.setup(tid, p.up_t, width);
      up_load.request(delta_rsrc((const IO*)p.dout + b * p.up_b + t0 * p.up_t + hv * p.up_h + c0, UpLoad::extent(p.up_t, width, left)), to + kUp, wave);
#pragma unroll
      for (int plane = 0; plane < PL; ++plane) {
        const long long at = (chunk * PL + plane) * p.columns + c0;
        value_load.request(delta_rsrc((const IO*)p.values + at * 64, ValueLoad::extent(64, 64, there)), to + kValues + plane * ValueLoad::kBytes, wave);
        value_load.request(delta_rsrc((const IO*)p.dvalues + at * 64, ValueLoad::extent(64, 64, there)), to + kDValues + plane * ValueLoad::kBytes, wave);
        state_load.request(delta_rsrc((const IO*)p.states + at * DK, StateLoad::extent(DK, DK, there)), to + kStates + plane * StateLoad::kBytes, wave);
        state_load.request(delta_rsrc((const IO*)p.dstates + at * DK, StateLoad::extent(DK, DK, there)), to + kDStates + plane * StateLoad::kBytes, wave);
      }
    };
    if (s > 0) __syncthreads();                             // the head before is through with the shared arrays
    request(0, 0);
    const ChunkGates gate = chunk_gates(p, b, hv, n, lane);
    const unsigned long long counts = __ballot(gate.counts);
    const float carry = gate.segments == 0 ? expf((float)gate.end) : 0.f;
    if (wave == 0) {
      total[lane] = gate.total;
      beta[lane] = gate.beta;
      segment[lane] = gate.segment;
      to_end[lane] = gate.segment == gate.segments ? expf((float)(gate.end - gate.total)) : 0.f;
    }
    f32x4 dq[KS] = {}, dr[KS] = {}, dw[KS] = {}, pairs[4] = {};
    float carried = 0.f;                                   // <S, dS'>
    wait_for_all();
    for (int c0 = 0; c0 < p.columns; c0 += CB) {
      const int stage = STAGES == 2 ? (c0 / CB) & 1 : 0;
      unsigned char* tile = lds + stage * kStage;
      if (counts != ~0ull) {                               // zeros for the rows of tokens that do not count
        for (int at = tid; at < 64 * Ups::U; at += THREADS)
          if (!((counts >> (at / Ups::U)) & 1)) *reinterpret_cast<i32x4*>(tile + kUp + at * 16) = i32x4{0, 0, 0, 0};
        lds_barrier();
      }
      if (STAGES == 2 && c0 + CB < p.columns) request(c0 + CB, stage ^ 1);
      const IO *ups = (const IO*)(tile + kUp), *values = (const IO*)(tile + kValues), *dvalues = (const IO*)(tile + kDValues),
               *states = (const IO*)(tile + kStates), *dstates = (const IO*)(tile + kDStates);
      const Frag uf = Ups::along_row(ups, 16 * block + c, 0, g);
      const Wide zf = Square::wide_down_rows(values, CB * 64, 0, 16 * block, lane);
      const Wide yf = Square::wide_down_rows(dvalues, CB * 64, 0, 16 * block, lane);
#pragma unroll
      for (int jt = 0; jt < 4; ++jt)
        if (jt <= block) {
          const Wide zj = Square::wide_down_rows(values, CB * 64, 0, 16 * jt, lane);
          pairs[jt] = half == 0 ? M::ew(uf, zj, pairs[jt]) : M::ww(yf, zj, pairs[jt]);
          phase();
        }
#pragma unroll
      for (int t = 0; t < KS; ++t) {
        const Wide sf = Keys::wide_down_rows(states, CB * DK, 0, 16 * (half * KS + t), lane);
        const Wide df = Keys::wide_down_rows(dstates, CB * DK, 0, 16 * (half * KS + t), lane);
        dq[t] = M::ew(uf, sf, dq[t]);
        dr[t] = M::ww(yf, sf, dr[t]);
        dw[t] = M::ww(zf, df, dw[t]);
        phase();
      }
      for (int at = tid; at < CB * Keys::U; at += THREADS) {
        typedef IO Unit __attribute__((ext_vector_type(Keys::E)));
        const Unit a = *reinterpret_cast<const Unit*>(states + at * Keys::E), d = *reinterpret_cast<const Unit*>(dstates + at * Keys::E);
        if constexpr (PL == 2) {
          const Unit al = *reinterpret_cast<const Unit*>(states + CB * DK + at * Keys::E), dl = *reinterpret_cast<const Unit*>(dstates + CB * DK + at * Keys::E);
#pragma unroll
          for (int e = 0; e < Keys::E; ++e) {
            carried = fmaf((float)a[e] + (float)al[e], (float)d[e] + (float)dl[e], carried);
          }
        } else {
#pragma unroll
          for (int e = 0; e < Keys::E; ++e) carried = fmaf((float)a[e], (float)d[e], carried);
        }
      }
      if (STAGES == 1 && c0 + CB < p.columns) {
        lds_barrier();                                     // the columns have been read
        request(c0 + CB, 0);
      }
      if (c0 + CB < p.columns) wait_for_all();
    }
    lds_barrier();
    {
      KeyLoad k;
      k.setup(tid, p.k_t, p.width);
      k.request(delta_rsrc((const IO*)p.k + b * p.k_b + t0 * p.k_t + h * p.k_h, KeyLoad::extent(p.k_t, p.width, left)), lds0, wave);
      k.setup(tid, p.q_t, p.width);
      k.request(delta_rsrc((const IO*)p.q + b * p.q_b + t0 * p.q_t + h * p.q_h, KeyLoad::extent(p.q_t, p.width, left)), lds0 + KeyLoad::kBytes, wave);
    }
    // the factors of what reads the carried state and of what is left for the next chunk; the decays of the pairs
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = row0 + e;
      const float rho = segment[i] == 0 ? expf((float)total[i]) : 0.f, end = to_end[i];
#pragma unroll
      for (int t = 0; t < KS; ++t) dq[t][e] *= p.scale * rho, dr[t][e] *= -rho, dw[t][e] *= end;
      phase();
#pragma unroll
      for (int jt = 0; jt < 4; ++jt) {
        const int j = 16 * jt + c;
        const bool joined = i >= j + half && segment[i] == segment[j];   // N2: strictly in front
        const float d = __expf(joined ? (float)(total[i] - total[j]) : 0.f);
        pairs[jt][e] = joined ? (half == 0 ? p.scale * d : -d) * pairs[jt][e] : 0.f;
      }
    }
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) carried += __shfl_xor(carried, m, 64);
    if (lane == 0) sums[wave] = carried;
    auto put_pairs = [&](bool strengths) {                 // kept [j][i]; blocks above the diagonal that a product touches are zeros
#pragma unroll
      for (int jt = 0; jt < 4; ++jt)
        if (jt <= (block | 1)) M::put(area + half * PL * 4096 + Square::at(16 * jt + c, row0), 4096, pairs[jt] * (strengths ? beta[16 * jt + c] : 1.f));
    };
    put_pairs(false);
    wait_for_all();
    if (counts != ~0ull) {
      for (int at = tid; at < 64 * Keys::U; at += THREADS)
        if (!((counts >> (at / Keys::U)) & 1)) {
          *reinterpret_cast<i32x4*>((unsigned char*)keys + at * 16) = i32x4{0, 0, 0, 0};
          *reinterpret_cast<i32x4*>((unsigned char*)queries + at * 16) = i32x4{0, 0, 0, 0};
        }
      lds_barrier();
    }
    {
      int lane = tid & 63;                                 // addresses anew: there are no registers to keep them in
      asm("" : "+v"(lane) : "s"(n));
      const int c = lane & 15, g = lane >> 4, row0 = 16 * block + 4 * g;
      f32x4 read = {}, dot = {};                           // of the state in front of the chunk; of the one behind it
#pragma unroll
      for (int t = 0; t < KS; ++t) {
        const f32x4 k = Keys::accumulator_tile(keys, 16 * block, 16 * (half * KS + t), lane);
        read += Keys::accumulator_tile(queries, 16 * block, 16 * (half * KS + t), lane) * dq[t] + k * dr[t];
        dot += dw[t] * k;
        phase();
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float from = sixteen_sum(read[e]), sum = sixteen_sum(dot[e]);
        if (c == 0) reads[half][row0 + e] = from, leaves[half][row0 + e] = beta[row0 + e] * sum;
      }
      phase();
    }
    // F = N1^T Q + N2^T K + ...: pairs in which the wave's tokens are the written ones
    for (int ks = block >> 1; ks < 2; ++ks) {
      const Wide a = Square::wide_along_row(area, 4096, 16 * block + c, 32 * ks, g);
      const Wide a2 = Square::wide_along_row(area + PL * 4096, 4096, 16 * block + c, 32 * ks, g);
#pragma unroll
      for (int t = 0; t < KS; ++t) {
        dw[t] = M::we(a, Keys::down_rows(queries, 32 * ks, 16 * (half * KS + t), lane), dw[t]);
        dw[t] = M::we(a2, Keys::down_rows(keys, 32 * ks, 16 * (half * KS + t), lane), dw[t]);
        phase();
      }
    }
    __syncthreads();
    put_pairs(true);
    __syncthreads();
    for (int ks = 0; ks <= (block >> 1); ++ks) {
      const Wide a = Square::wide_down_rows(area, 4096, 32 * ks, 16 * block, lane);
      const Wide a2 = Square::wide_down_rows(area + PL * 4096, 4096, 32 * ks, 16 * block, lane);
#pragma unroll
      for (int t = 0; t < KS; ++t) {
        const Frag kf = Keys::down_rows(keys, 32 * ks, 16 * (half * KS + t), lane);
        dq[t] = M::we(a, kf, dq[t]);
        dr[t] = M::we(a2, kf, dr[t]);
        phase();
      }
    }
    f32x4 written = {}, strength;
#pragma unroll
    for (int e = 0; e < 4; ++e) strength[e] = beta[row0 + e];
#pragma unroll
    for (int t = 0; t < KS; ++t) {
      const f32x4 k = Keys::accumulator_tile(keys, 16 * block, 16 * (half * KS + t), lane);
      written += k * dw[t];
      dr[t] += strength * dw[t];
      all_dq[t] = GROUPED ? all_dq[t] + dq[t] : dq[t];
      all_dk[t] = GROUPED ? all_dk[t] + dr[t] : dr[t];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float back = sixteen_sum(written[e]);
      if (c == 0) writes[half][row0 + e] = back;
    }
    // pairs across each token: N1 with q_i . k_j, N2 with k_i . k_j; the wave reads what it has put there itself.  Of its sixteen rows, for its
    // own sixteen tokens t the sums over i >= t as a product with a triangle of ones, then over j < t; for tokens in front of them
    // all rows, column by column, and the sums over j < t.
    {
      int lane = tid & 63;
      asm("" : "+v"(lane) : "s"(n));
      const int c = lane & 15, g = lane >> 4, row0 = 16 * block + 4 * g;
      float earlier = 0.f;
      f32x4 before = {}, own = {};                         // columns in front of the wave's tokens, added up; its own
      const IO* const rows = half == 0 ? queries : keys;
#pragma unroll
      for (int jt = 0; jt < 4; ++jt)
        if (jt <= block) {
          f32x4 w = {};
#pragma unroll
          for (int ks = 0; ks < KS; ++ks) w = M::ee(Keys::along_row(rows, 16 * block + c, 32 * ks, g), Keys::along_row(keys, 16 * jt + c, 32 * ks, g), w);
          const f32x4 pair = M::get(area + half * PL * 4096 + Square::at(16 * jt + c, row0), 4096);
#pragma unroll
          for (int e = 0; e < 4; ++e) w[e] = pair[e] == 0.f ? 0.f : pair[e] * w[e];
          if (jt < block) {
            before += w;
            const float sum = four_rows_sum((w[0] + w[1]) + (w[2] + w[3]));
            const float in_front = sixteen_in_front(sum);
            if (g == 0) columns_of[wave][16 * jt + c] = earlier + in_front;
            earlier += sixteen_sum(sum);
          } else {
            own = w;
          }
          phase();
        }
      f32x4 in_front = {}, among = {};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float one = 4 * g + e >= c ? 1.f : 0.f;
        in_front = __builtin_amdgcn_mfma_f32_16x16x4f32(one, before[e], in_front, 0, 0, 0);
        among = __builtin_amdgcn_mfma_f32_16x16x4f32(one, own[e], among, 0, 0, 0);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float sum = sixteen_sum(in_front[e] + (c < 4 * g + e ? among[e] : 0.f));
        if (c == 0) crossing[half][row0 + e] = sum;
      }
      phase();
    }
    __syncthreads();
    if (wave == 0) {                                       // what crosses each token
      const float written = writes[0][lane] + writes[1][lane];
      // read from the token on; written in front of it: for the state behind the chunk, for tokens of the second, third and last sixteen
      float from = reads[0][lane] + reads[1][lane], to = leaves[0][lane] + leaves[1][lane];
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const float other = __shfl_down(from, d, 64);
        if (lane + d < 64) from += other;
        const float before = __shfl_up(to, d, 64);
        if (lane >= d) to += before;
      }
      to = __shfl_up(to, 1, 64);
      float across = 0.f, pairs_across = (crossing[0][lane] + crossing[1][lane]) + (lane > 0 ? to : 0.f);
#pragma unroll
      for (int w = 0; w < THREADS / 64; ++w) across += sums[w];
      across = carry == 0.f ? 0.f : carry * across;
#pragma unroll
      for (int i = 1; i < 4; ++i)
        if (lane < 16 * i) pairs_across += columns_of[i][lane] + columns_of[4 + i][lane];
      const float d = gate.counts && !gate.starts ? from + (across + pairs_across) : 0.f;
      const long long at = ((long long)b * p.T + t0 + lane) * p.HV + hv;
      if (lane < left) {
        delta_put_gate(p.dlog_decay, at, p.decay_dtype, d);
        delta_put_gate(p.dbeta, at, p.beta_dtype, written);
      }
    }
  }
  const int c = tid & 15, g = (tid & 63) >> 4, row0 = 16 * block + 4 * g;
  const long long stride = (long long)p.H * p.K, base = ((long long)b * p.T + t0) * stride + (long long)h * p.K;
  if (p.width == p.K) {                                     // through the tiles of queries and keys, which all waves are through with
#pragma unroll
    for (int t = 0; t < KS; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int at = Keys::at(row0 + e, 16 * (half * KS + t) + c);
        queries[at] = (IO)all_dq[t][e];
        keys[at] = (IO)all_dk[t][e];
      }
    __syncthreads();
    for (int at = tid; at < 64 * Keys::U; at += THREADS) {
      const int row = at / Keys::U, u = at % Keys::U;
      if (row >= left || u * Keys::E >= p.K) continue;
      const long long to = base + row * stride + u * Keys::E;
      *reinterpret_cast<i32x4*>((IO*)p.dq + to) = *reinterpret_cast<const i32x4*>(queries + Keys::unit(row, u));
      *reinterpret_cast<i32x4*>((IO*)p.dk + to) = *reinterpret_cast<const i32x4*>(keys + Keys::unit(row, u));
    }
  } else {
#pragma unroll
    for (int t = 0; t < KS; ++t) {
      const int col = 16 * (half * KS + t) + c;
      const ColumnIo<IO> q_out((const IO*)p.dq + base, stride, left, p.K, col, col < p.K, 4 * g), k_out((const IO*)p.dk + base, stride, left, p.K, col, col < p.K, 4 * g);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        q_out.store(16 * block + e, all_dq[t][e]);
        k_out.store(16 * block + e, all_dk[t][e]);
      }
    }
  }
}

int delta_launch_join(const DeltaArgs& a, int dtype, hipStream_t s);

template <typename IO, int KS, int WAVES, int STAGES, bool LOCAL> static int delta_walk_back(const DeltaArgs& a, hipStream_t s) {
  const long long total = (long long)((a.columns + 16 * WAVES - 1) / (16 * WAVES)) * a.segments * a.B * a.HV;
  hipLaunchKernelGGL((delta_backward_kernel<IO, KS, WAVES, STAGES, LOCAL>), xcd_grid(total), dim3(64 * WAVES), 0, s, a);
  return check_launch("gated_delta_bwd");
}

template <typename IO, int KS> static int delta_backward(const DeltaArgs& a, hipStream_t s) {
  constexpr bool kTwo = sizeof(IO) == 2;                    // two chunks' tiles fit the LDS
  int rc = RGLRU_OK;
  if (a.segments > 1) {
    rc = delta_walk_back<IO, KS, 4, 1, true>(a, s);
    if (!rc) rc = delta_launch_join(a, kTwo ? RGLRU_BF16 : RGLRU_F32, s);
    if (rc) return rc;
  }
  bool narrow = false;
  if constexpr (kTwo) {
    narrow = delta_narrow(a);
    if (narrow) rc = delta_walk_back<IO, KS, 2, 2, false>(a, s);
  }
  if (!narrow) rc = delta_walk_back<IO, KS, 4, 1, false>(a, s);
  if (rc) return rc;
  const dim3 grid = xcd_grid((long long)a.B * a.H * a.nC);
  if (a.HV > a.H) hipLaunchKernelGGL((delta_grads_kernel<IO, KS, true>), grid, dim3(kGradThreads), 0, s, a);
  else hipLaunchKernelGGL((delta_grads_kernel<IO, KS, false>), grid, dim3(kGradThreads), 0, s, a);
  return check_launch("gated_delta_bwd gradients");
}

int delta_launch_backward(const DeltaArgs& a, int dtype, hipStream_t s) {
  switch ((a.K + 31) / 32) {
#define RGLRU_DELTA(KS) case KS: return dtype == RGLRU_BF16 ? delta_backward<__bf16, KS>(a, s) : delta_backward<float, KS>(a, s)
    RGLRU_DELTA(1);
    RGLRU_DELTA(2);
    RGLRU_DELTA(3);
    RGLRU_DELTA(4);
#undef RGLRU_DELTA
  }
  return fail(RGLRU_E_UNSUPPORTED, "gated_delta_bwd: key size %d", a.K);
}

}  // namespace rglru
