// Selective state space scan, reverse mode (the forward's mathematics and the layout: rglru_selective.h).  With y_t the sum in front of the gate,
//   dy_t = dout_t silu(z_t),  dz_t = dout_t y_t silu'(z_t),  dh_t = C_t dy_t + a_{t+1} dh_{t+1},  a_t = exp(s_t A)
//   dC_t = sum over w of dy_t h_t,  dB_t = sum over w of s_t u_t dh_t,  along_t = sum over n of B_t dh_t,  q_t = dh_t a_t h_{t-1}
//   ds_t = sum over n of A q_t + u_t along_t,  ddt_t = ds_t softplus'(dt_t + bias),  du_t = s_t along_t + D dy_t
//   dA = sum over b, t of s_t q_t,  dD = sum of dy_t u_t,  dbias = sum of ddt_t
// The walk goes from the last tile to the first.  A tile's decays and states are made again from the state that the forward pass kept in front of it and
// stay in registers (128 of them) for the way back.  Sums over channels: a row of 16 lanes adds up four tokens' values at a time, each step handing
// half of what a lane holds to the lane that keeps it, the workgroup's waves add up in LDS, and its sets are added by a kernel of their own in
// a fixed order.

#include <hip/hip_runtime.h>

#include <cstring>

#include "rglru_selective.h"
#include "rglru_sums.h"

namespace rglru {

// What a segment hands back of a gradient of zeros at its last state.  (Its sums of step sizes and document starts are made again here: the forward
// pass keeps them only until its own join.)
template <typename IO, int SLABS, bool MASKED> __global__ __launch_bounds__(kSelThreads) void sel_reverse_kernel(SelArgs p) {
  __shared__ float2 rates[kSelWaves][kSelTile][kSelLanes];
  const SelPlace at = sel_place<SLABS>(p);
  if (at.seg == 0) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, j = lane >> 4;
  const int in_group = at.cg * kSelLanes + c, n0 = at.slab * kSelStates + 4 * j;
  const bool ok = in_group < p.Wg;
  const int w = at.g * p.Wg + (ok ? in_group : 0);
  const int first = at.seg * p.seg_tiles, last = first + p.seg_tiles < p.tiles ? first + p.seg_tiles : p.tiles;
  float a2[4], carry[4] = {0.f, 0.f, 0.f, 0.f};
  sel_load_states(p.A, w, n0, p.N, ok, a2);
#pragma unroll
  for (int i = 0; i < 4; ++i) a2[i] *= kLog2e;
  const float bias = ok && p.bias ? p.bias[w] : 0.f;
  const bool gated = p.z != nullptr;
  SelStream<IO> next_dt, next_z, next_d;
  SelVector<IO> next_C;
  auto request = [&](int tile) {
    const long long t0 = (long long)tile * kSelTile;
    const int left = (int)(p.T - t0 < kSelTile ? p.T - t0 : kSelTile);
    next_dt.load(p.dt, at.b * p.sdb + t0 * p.sdt, (unsigned)p.sdt, w, left, ok, j);
    next_d.load(p.dout, ((long long)at.b * p.T + t0) * p.W, (unsigned)p.W, w, left, ok, j);
    if (gated) next_z.load(p.z, at.b * p.szb + t0 * p.szt, (unsigned)p.szt, w, left, ok, j);
    next_C.load(p.Cm, at.b * p.sCb + t0 * p.sCt + at.g * p.sCg, (unsigned)p.sCt, n0, p.N, left, c, p.vector);
  };
  request(last - 1);
  float total = 0.f;
  bool cut = false;
  for (int tile = last - 1; tile >= first; --tile) {
    const long long t0 = (long long)tile * kSelTile;
    const int left = (int)(p.T - t0 < kSelTile ? p.T - t0 : kSelTile);
    const SelMasks m = sel_masks<MASKED>(p.flags, (long long)at.b * p.T + t0, left, lane);
    float C[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const bool live = (m.live >> (4 * q + j)) & 1u;
      const float s = live ? sel_rate(next_dt.v[q] + bias, p.softplus).s : 0.f;
      float dy = live ? next_d.v[q] : 0.f;
      if (gated && live) dy *= next_z.v[q] * sigmoid_fast(next_z.v[q]);
      rates[wave][4 * q + j][c] = make_float2(s, dy);
      total += s;
    }
    const bool mine = (m.live >> c) & 1u;
#pragma unroll
    for (int i = 0; i < 4; ++i) C[i] = mine ? next_C.v[i] : 0.f;
    wave_order();
    if (tile > first) request(tile - 1);
    if (MASKED) cut = cut || m.starts;
    sel_each<kSelTile>([&](auto token) {
      constexpr int t = kSelTile - 1 - decltype(token)::value;
      const float2 rate = rates[wave][t][c];
#pragma unroll
      for (int i = 0; i < 4; ++i) carry[i] = fmaf(row_bcast<t>(C[i]), rate.y, carry[i]) * __builtin_amdgcn_exp2f(a2[i] * rate.x);
      if constexpr (MASKED)
        if ((m.starts >> t) & 1u) carry[0] = carry[1] = carry[2] = carry[3] = 0.f;
    });
    wave_order();
  }
  const long long row = ((long long)at.b * p.S + at.seg) * p.W + w;
  sel_store_states(p.ends, row, n0, p.N, ok, carry);
  total = all_rows_sum(total);
  if (ok && j == 0 && at.slab == 0) { p.sums[2 * row] = total; p.sums[2 * row + 1] = cut ? 1.f : 0.f; }
}

template <typename IO, int SLABS, bool MASKED> __global__ __launch_bounds__(kSelThreads, 1) void sel_backward_kernel(SelArgs p) {
  __shared__ f32x4 rates[kSelWaves][kSelTile][kSelLanes];   // step size, that times u, dy
  __shared__ float vectors[2][2][kSelWaves][4][64];         // dB and dC of a tile, by waves; two tiles in turn
  __shared__ float parts[SLABS > 1 ? 2 : 1][SLABS > 1 ? kSelWaves : 1][3][4][64];
  const SelPlace at = sel_place<SLABS>(p);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, j = lane >> 4;
  const int in_group = at.cg * kSelLanes + c, n0 = at.slab * kSelStates + 4 * j;
  const bool ok = in_group < p.Wg;
  const int w = at.g * p.Wg + (ok ? in_group : 0);
  const int first = at.seg * p.seg_tiles, last = first + p.seg_tiles < p.tiles ? first + p.seg_tiles : p.tiles;
  float a2[4], carry[4] = {0.f, 0.f, 0.f, 0.f}, dA[4] = {0.f, 0.f, 0.f, 0.f}, dD = 0.f, dbias = 0.f;
  sel_load_states(p.A, w, n0, p.N, ok, a2);
#pragma unroll
  for (int i = 0; i < 4; ++i) a2[i] *= kLog2e;
  const float bias = ok && p.bias ? p.bias[w] : 0.f, skip = ok && p.D ? p.D[w] : 0.f;
  if (p.dh_last) sel_load_states(p.dh_last, (long long)at.b * p.W + w, n0, p.N, ok, carry);
  sel_join<true>(p, at, w, n0, ok, a2, carry);
  const bool gated = p.z != nullptr;
  SelStream<IO> next_u, next_dt, next_z, next_d;
  SelVector<IO> next_B, next_C;
  float next_h[4];
  auto request = [&](int tile) {
    const long long t0 = (long long)tile * kSelTile;
    const int left = (int)(p.T - t0 < kSelTile ? p.T - t0 : kSelTile);
    next_u.load(p.u, at.b * p.sub + t0 * p.sut, (unsigned)p.sut, w, left, ok, j);
    next_dt.load(p.dt, at.b * p.sdb + t0 * p.sdt, (unsigned)p.sdt, w, left, ok, j);
    next_d.load(p.dout, ((long long)at.b * p.T + t0) * p.W, (unsigned)p.W, w, left, ok, j);
    if (gated) next_z.load(p.z, at.b * p.szb + t0 * p.szt, (unsigned)p.szt, w, left, ok, j);
    next_B.load(p.Bm, at.b * p.sBb + t0 * p.sBt + at.g * p.sBg, (unsigned)p.sBt, n0, p.N, left, c, p.vector);
    next_C.load(p.Cm, at.b * p.sCb + t0 * p.sCt + at.g * p.sCg, (unsigned)p.sCt, n0, p.N, left, c, p.vector);
    sel_load_states(p.kept, ((long long)at.b * p.tiles + tile) * p.W + w, n0, p.N, ok, next_h);
  };
  request(last - 1);
  for (int tile = last - 1; tile >= first; --tile) {
    const long long t0 = (long long)tile * kSelTile;
    const int left = (int)(p.T - t0 < kSelTile ? p.T - t0 : kSelTile);
    const SelMasks m = sel_masks<MASKED>(p.flags, (long long)at.b * p.T + t0, left, lane);
    float u[4], s[4], slope[4], d[4], z[4], dy[4], B[4], C[4], before[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const bool live = (m.live >> (4 * q + j)) & 1u;
      const SelRate rate = sel_rate(next_dt.v[q] + bias, p.softplus);
      s[q] = live ? rate.s : 0.f;
      slope[q] = live ? rate.slope : 0.f;
      u[q] = live ? next_u.v[q] : 0.f;
      d[q] = live ? next_d.v[q] : 0.f;
      z[q] = live && gated ? next_z.v[q] : 0.f;
      dy[q] = gated ? d[q] * (z[q] * sigmoid_fast(z[q])) : d[q];
      rates[wave][4 * q + j][c] = (f32x4){s[q], s[q] * u[q], dy[q], 0.f};
    }
    const bool mine = (m.live >> c) & 1u;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      B[i] = mine ? next_B.v[i] : 0.f;
      C[i] = mine ? next_C.v[i] : 0.f;
      before[i] = next_h[i];
    }
    wave_order();
    if (tile > first) request(tile - 1);
    // decays and states of the tile, and y where the gate asks for it
    float a[kSelTile][4], h[kSelTile][4], y[4];
    sel_each<4>([&](auto group) {
      float sums[4];
      sel_each<4>([&](auto token) {
        constexpr int t = 4 * decltype(group)::value + decltype(token)::value;
        const float2 rate = *reinterpret_cast<const float2*>(&rates[wave][t][c]);
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float old = t ? h[t ? t - 1 : 0][i] : before[i];
          if constexpr (MASKED) old = (m.starts >> t) & 1u ? 0.f : old;
          a[t][i] = __builtin_amdgcn_exp2f(a2[i] * rate.x);
          h[t][i] = fmaf(a[t][i], old, row_bcast<t>(B[i]) * rate.y);
          sum = fmaf(row_bcast<t>(C[i]), h[t][i], sum);
        }
        sums[decltype(token)::value] = sum;
      });
      y[decltype(group)::value] = gated ? four_rows_sum(sums) : 0.f;
    });
    float along[4], through[4], tile_dA[4] = {0.f, 0.f, 0.f, 0.f}, tile_dD = 0.f, tile_dbias = 0.f;  // tile by tile: a long sum loses less
    sel_each<4>([&](auto back) {
      constexpr int g4 = 3 - decltype(back)::value;
      float dB[4][4], dC[4][4], sum_b[4], sum_a[4];
      sel_each<4>([&](auto token) {
        constexpr int k = 3 - decltype(token)::value, t = 4 * g4 + k;
        const f32x4 rate = rates[wave][t][c];
        float sb = 0.f, sa = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float dh = fmaf(row_bcast<t>(C[i]), rate[2], carry[i]);
          dC[k][i] = rate[2] * h[t][i];
          dB[k][i] = rate[1] * dh;
          sb = fmaf(row_bcast<t>(B[i]), dh, sb);
          float old = t ? h[t ? t - 1 : 0][i] : before[i];
          carry[i] = a[t][i] * dh;
          if constexpr (MASKED) {
            const bool cut = (m.starts >> t) & 1u;
            old = cut ? 0.f : old;
            carry[i] = cut ? 0.f : carry[i];
          }
          const float q = carry[i] * old;
          sa = fmaf(a2[i], q, sa);
          tile_dA[i] = fmaf(rate[0], q, tile_dA[i]);
        }
        sum_b[k] = sb;
        sum_a[k] = sa;
      });
      along[g4] = four_rows_sum(sum_b);
      through[g4] = four_rows_sum(sum_a);
      vectors[tile & 1][0][wave][g4][lane] = lanes_scatter_sum(dB, lane);
      vectors[tile & 1][1][wave][g4][lane] = lanes_scatter_sum(dC, lane);
    });
    if constexpr (SLABS > 1) {
      float (*mem)[3][4][64] = parts[tile & 1];
#pragma unroll
      for (int q = 0; q < 4; ++q) { mem[wave][0][q][lane] = along[q]; mem[wave][1][q][lane] = through[q]; mem[wave][2][q][lane] = y[q]; }
    }
    __syncthreads();                                        // the other buffer's readers are past the barrier before
    if constexpr (SLABS > 1) {
      float (*mem)[3][4][64] = parts[tile & 1];
      const int head = wave - at.slab;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        float x[3] = {0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < SLABS; ++k)
#pragma unroll
          for (int e = 0; e < 3; ++e) x[e] += mem[head + k][e][q][lane];
        along[q] = x[0]; through[q] = x[1]; y[q] = x[2];
      }
    }
    // dB and dC of the workgroup's channels: thread (slab, group of tokens, lane as lanes_scatter_sum leaves it)
    for (int idx = threadIdx.x; idx < 2 * SLABS * 256; idx += kSelThreads) {
      const int which = idx / (SLABS * 256), slab = idx / 256 % SLABS, q = idx / 64 % 4, l = idx & 63;
      const int t = 4 * q + 2 * ((l >> 3) & 1) + ((l >> 2) & 1), n = slab * kSelStates + 4 * (l >> 4) + (l & 3);
      float sum = 0.f;
#pragma unroll
      for (int k = slab; k < kSelWaves; k += SLABS) sum += vectors[tile & 1][which][k][q][l];
      if (t < left && n < p.N) {
        float* out = (which ? p.dC : p.dB) + ((((long long)at.set * p.B + at.b) * p.T + t0 + t) * p.G + at.g) * p.N + n;
        *out = (m.live >> t) & 1u ? sum : 0.f;
      }
    }
    float du[4], ddt[4], dz[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const float ds = fmaf(u[q], along[q], through[q] * kLn2);
      const bool live = (m.live >> (4 * q + j)) & 1u;
      ddt[q] = live ? ds * slope[q] : 0.f;
      du[q] = live ? fmaf(s[q], along[q], skip * dy[q]) : 0.f;
      tile_dD = fmaf(dy[q], u[q], tile_dD);
      tile_dbias += ddt[q];
      if (gated) {
        const float sig = sigmoid_fast(z[q]);
        dz[q] = live ? d[q] * fmaf(skip, u[q], y[q]) * sig * fmaf(z[q], 1.f - sig, 1.f) : 0.f;
      }
    }
    dD += tile_dD;
    dbias += tile_dbias;
#pragma unroll
    for (int i = 0; i < 4; ++i) dA[i] += tile_dA[i];
    if (SLABS == 1 || at.slab == 0) {
      const long long place = ((long long)at.b * p.T + t0) * p.W;
      sel_store<IO>(du, p.du, place, (unsigned)p.W, w, left, ok, j);
      sel_store<IO>(ddt, p.ddt, place, (unsigned)p.W, w, left, ok, j);
      if (gated) sel_store<IO>(dz, p.dz, place, (unsigned)p.W, w, left, ok, j);
    }
  }
  const long long row = ((long long)at.b * p.S + at.seg) * p.W + w;
  sel_store_states(p.dA, row, n0, p.N, ok, dA);
  dD = all_rows_sum(dD);
  dbias = all_rows_sum(dbias);
  if (ok && j == 0 && at.slab == 0) { p.dD[row] = dD; p.dbias[row] = dbias; }
  if (at.seg == 0 && p.dh0) sel_store_states(p.dh0, (long long)at.b * p.W + w, n0, p.N, ok, carry);
}

// The sums of all partial gradients in one launch.
struct SelSums {
  SumJob job[5];
  int first[6];
};
static __global__ __launch_bounds__(256) void sel_sums_kernel(SelSums jobs) {
  __shared__ float red[8][32];
  int i = 0;
  while (i < 4 && (int)blockIdx.x >= jobs.first[i + 1]) ++i;
  run_sum_job(jobs.job[i], (int)blockIdx.x - jobs.first[i], red);
}

template <typename IO, int SLABS, bool MASKED> static void sel_backward_masked(const SelArgs& a, hipStream_t s) {
  const dim3 grid((unsigned)(a.B * (long long)a.S * a.G * a.per_group)), block(kSelThreads);
  if (a.S > 1) hipLaunchKernelGGL((sel_reverse_kernel<IO, SLABS, MASKED>), grid, block, 0, s, a);
  hipLaunchKernelGGL((sel_backward_kernel<IO, SLABS, MASKED>), grid, block, 0, s, a);
}
template <typename IO> static void sel_backward_typed(const SelArgs& a, hipStream_t s) {
  const int slabs = (a.N + kSelStates - 1) / kSelStates;
  if (slabs == 1) { if (a.flags) sel_backward_masked<IO, 1, true>(a, s); else sel_backward_masked<IO, 1, false>(a, s); }
  else if (slabs == 2) { if (a.flags) sel_backward_masked<IO, 2, true>(a, s); else sel_backward_masked<IO, 2, false>(a, s); }
  else { if (a.flags) sel_backward_masked<IO, 4, true>(a, s); else sel_backward_masked<IO, 4, false>(a, s); }
}

int sel_launch_backward(const SelArgs& a, void* dB, void* dC, float* dA, float* dD, float* dbias, int dtype, hipStream_t s) {
  if (dtype == RGLRU_BF16) sel_backward_typed<__bf16>(a, s); else sel_backward_typed<float>(a, s);
  int rc = check_launch("selective_bwd");
  if (rc) return rc;
  SelSums jobs;
  memset(&jobs, 0, sizeof(jobs));
  const long long vectors = (long long)a.B * a.T * a.G * a.N;
  const struct { const float* src; void* dst; long long n; int sets, bf16; } list[5] = {
      {a.dB, dB, vectors, a.per_group, dtype == RGLRU_BF16}, {a.dC, dC, vectors, a.per_group, dtype == RGLRU_BF16},
      {a.dA, dA, (long long)a.W * a.N, a.B * a.S, 0}, {a.dD, dD, a.W, a.B * a.S, 0}, {a.dbias, dbias, a.W, a.B * a.S, 0}};
  int blocks = 0;
  for (int i = 0; i < 5; ++i) {
    SumJob& j = jobs.job[i];
    j.src = list[i].src; j.dst = list[i].dst; j.n = list[i].n; j.sets = list[i].sets; j.dst_bf16 = list[i].bf16;
    plan_sum_job(j);
    if (!j.dst) j.blocks = 0;
    jobs.first[i] = blocks;
    blocks += j.blocks;
  }
  jobs.first[5] = blocks;
  hipLaunchKernelGGL(sel_sums_kernel, dim3((unsigned)blocks), dim3(256), 0, s, jobs);
  return check_launch("selective_bwd sums");
}

}  // namespace rglru
