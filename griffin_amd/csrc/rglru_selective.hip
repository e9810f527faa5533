// Selective state space scan over whole sequences, forward (the mathematics and the layout: rglru_selective.h).

#include <hip/hip_runtime.h>

#include <cstring>

#include "rglru_selective.h"

namespace rglru {

// SUMMARY: what a segment leaves of a state of zeros and its sum of step sizes.  Otherwise outputs, the last state and, for a backward pass, the state
// in front of every tile.
template <typename IO, int SLABS, bool MASKED, bool SUMMARY> __global__ __launch_bounds__(kSelThreads) void sel_forward_kernel(SelArgs p) {
  __shared__ float2 rates[kSelWaves][kSelTile][kSelLanes];
  __shared__ float parts[SLABS > 1 && !SUMMARY ? 2 : 1][SLABS > 1 && !SUMMARY ? kSelWaves : 1][4][64];
  const SelPlace at = sel_place<SLABS>(p);
  if (SUMMARY && at.seg == p.S - 1) return;                 // nothing asks what the last one leaves
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, j = lane >> 4;
  const int in_group = at.cg * kSelLanes + c, n0 = at.slab * kSelStates + 4 * j;
  const bool ok = in_group < p.Wg;
  const int w = at.g * p.Wg + (ok ? in_group : 0);
  const int first = at.seg * p.seg_tiles, last = first + p.seg_tiles < p.tiles ? first + p.seg_tiles : p.tiles;
  float a2[4], h[4] = {0.f, 0.f, 0.f, 0.f};
  sel_load_states(p.A, w, n0, p.N, ok, a2);
#pragma unroll
  for (int i = 0; i < 4; ++i) a2[i] *= kLog2e;
  const float bias = ok && p.bias ? p.bias[w] : 0.f, skip = ok && p.D ? p.D[w] : 0.f;
  if constexpr (!SUMMARY) {
    if (p.h0) sel_load_states(p.h0, (long long)at.b * p.W + w, n0, p.N, ok, h);
    sel_join<false>(p, at, w, n0, ok, a2, h);
  }
  SelStream<IO> next_u, next_dt, next_z;
  SelVector<IO> next_B, next_C;
  const bool gated = !SUMMARY && p.z != nullptr;
  auto request = [&](int tile) {
    const long long t0 = (long long)tile * kSelTile;
    const int left = (int)(p.T - t0 < kSelTile ? p.T - t0 : kSelTile);
    next_u.load(p.u, at.b * p.sub + t0 * p.sut, (unsigned)p.sut, w, left, ok, j);
    next_dt.load(p.dt, at.b * p.sdb + t0 * p.sdt, (unsigned)p.sdt, w, left, ok, j);
    if (gated) next_z.load(p.z, at.b * p.szb + t0 * p.szt, (unsigned)p.szt, w, left, ok, j);
    next_B.load(p.Bm, at.b * p.sBb + t0 * p.sBt + at.g * p.sBg, (unsigned)p.sBt, n0, p.N, left, c, p.vector);
    if (!SUMMARY) next_C.load(p.Cm, at.b * p.sCb + t0 * p.sCt + at.g * p.sCg, (unsigned)p.sCt, n0, p.N, left, c, p.vector);
  };
  request(first);
  float total = 0.f;
  bool cut = false;
  for (int tile = first; tile < last; ++tile) {
    const long long t0 = (long long)tile * kSelTile;
    const int left = (int)(p.T - t0 < kSelTile ? p.T - t0 : kSelTile);
    const SelMasks m = sel_masks<MASKED>(p.flags, (long long)at.b * p.T + t0, left, lane);
    float u[4], z[4], B[4], C[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const bool live = (m.live >> (4 * q + j)) & 1u;
      const float s = live ? sel_rate(next_dt.v[q] + bias, p.softplus).s : 0.f;
      u[q] = live ? next_u.v[q] : 0.f;
      z[q] = live && gated ? next_z.v[q] : 0.f;
      rates[wave][4 * q + j][c] = make_float2(s, s * u[q]);
      if (SUMMARY) total += s;
    }
    const bool mine = (m.live >> c) & 1u;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      B[i] = mine ? next_B.v[i] : 0.f;
      C[i] = !SUMMARY && mine ? next_C.v[i] : 0.f;
    }
    wave_order();
    if (tile + 1 < last) request(tile + 1);
    if (!SUMMARY && p.kept) sel_store_states(p.kept, ((long long)at.b * p.tiles + tile) * p.W + w, n0, p.N, ok, h);
    if (MASKED) cut = cut || m.starts;
    float y[4];
    sel_each<4>([&](auto group) {
      float sums[4];
      sel_each<4>([&](auto token) {
        constexpr int t = 4 * decltype(group)::value + decltype(token)::value;
        const float2 rate = rates[wave][t][c];
        if constexpr (MASKED)
          if ((m.starts >> t) & 1u) h[0] = h[1] = h[2] = h[3] = 0.f;
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float a = __builtin_amdgcn_exp2f(a2[i] * rate.x);
          h[i] = fmaf(a, h[i], row_bcast<t>(B[i]) * rate.y);
          if (!SUMMARY) sum = fmaf(row_bcast<t>(C[i]), h[i], sum);
        }
        sums[decltype(token)::value] = sum;
      });
      if (!SUMMARY) y[decltype(group)::value] = four_rows_sum(sums);
    });
    wave_order();                                           // the next tile's rates come after these reads
    if constexpr (SUMMARY) continue;
    if constexpr (SLABS > 1) {                              // the other states of these channels: each wave takes its share of the tokens
      float (*mem)[4][64] = parts[tile & 1];
#pragma unroll
      for (int q = 0; q < 4; ++q) mem[wave][q][lane] = y[q];
      __syncthreads();
      const int head = wave - at.slab;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        float sum = 0.f;
#pragma unroll
        for (int k = 0; k < SLABS; ++k) sum += mem[head + k][q][lane];
        y[q] = sum;
      }
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      y[q] = fmaf(skip, u[q], y[q]);
      if (gated) y[q] *= z[q] * sigmoid_fast(z[q]);
      if (!((m.live >> (4 * q + j)) & 1u)) y[q] = 0.f;
    }
    if (SLABS == 1 || at.slab == 0)
      sel_store<IO>(y, p.y, ((long long)at.b * p.T + t0) * p.W, (unsigned)p.W, w, left, ok, j);
  }
  if constexpr (SUMMARY) {
    const long long row = ((long long)at.b * p.S + at.seg) * p.W + w;
    sel_store_states(p.ends, row, n0, p.N, ok, h);
    total = all_rows_sum(total);
    if (ok && j == 0 && at.slab == 0) { p.sums[2 * row] = total; p.sums[2 * row + 1] = cut ? 1.f : 0.f; }
  } else if (at.seg == p.S - 1) {
    sel_store_states(p.h_last, (long long)at.b * p.W + w, n0, p.N, ok, h);
  }
}

template <typename IO, int SLABS, bool MASKED> static void sel_forward_masked(const SelArgs& a, hipStream_t s) {
  const dim3 grid((unsigned)(a.B * (long long)a.S * a.G * a.per_group)), block(kSelThreads);
  if (a.S > 1) hipLaunchKernelGGL((sel_forward_kernel<IO, SLABS, MASKED, true>), grid, block, 0, s, a);
  hipLaunchKernelGGL((sel_forward_kernel<IO, SLABS, MASKED, false>), grid, block, 0, s, a);
}
template <typename IO> static void sel_forward_typed(const SelArgs& a, hipStream_t s) {
  const int slabs = (a.N + kSelStates - 1) / kSelStates;
  if (slabs == 1) { if (a.flags) sel_forward_masked<IO, 1, true>(a, s); else sel_forward_masked<IO, 1, false>(a, s); }
  else if (slabs == 2) { if (a.flags) sel_forward_masked<IO, 2, true>(a, s); else sel_forward_masked<IO, 2, false>(a, s); }
  else { if (a.flags) sel_forward_masked<IO, 4, true>(a, s); else sel_forward_masked<IO, 4, false>(a, s); }
}

int sel_launch_forward(const SelArgs& a, int dtype, hipStream_t s) {
  if (dtype == RGLRU_BF16) sel_forward_typed<__bf16>(a, s); else sel_forward_typed<float>(a, s);
  return check_launch("selective_fwd");
}

}  // namespace rglru
