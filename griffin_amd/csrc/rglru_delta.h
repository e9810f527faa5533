// Building blocks of the gated delta rule's kernels (gfx950, wave64): 16 x 16 matrix products whose operands come from LDS
// tiles or straight from the accumulators of the product before.
//
// An accumulator tile of v_mfma_f32_16x16 gives lane (c = lane % 16, g = lane / 16) the rows 4 g .. 4 g + 3 of column c.  The
// B operand of the next product wants lane (c, g) to hold the contraction indices 8 g .. 8 g + 7 of 32 for column c.  Which index a
// tile's row stands for is free: with row 4 g + e of the tiles 2 p and 2 p + 1 standing for 32 p + 8 g + e and 32 p + 8 g + 4 + e (tile_index),
// the two tiles ARE that operand.  So a wave that owns 16 columns of the state takes it from product to product in its
// registers; LDS holds only what comes from memory, sixteen bytes a lane and read.
//
// bf16 storage: keys, queries and upstream gradients are exact matrix operands; what is computed (state, solved values, the
// chunk's triangular matrices) enters as the sum of two bf16 numbers, 2^-17 relative, because one bf16 number would round the
// carried state to 2^-9 once a chunk.  fp32 storage: v_mfma_f32_16x16x4_f32 throughout.
#pragma once

#include "rglru_device.h"
#include "rglru_host.h"

namespace rglru {

constexpr int kDeltaChunk = 64;              // tokens of a chunk
constexpr int kDeltaThreads = 256;
constexpr int kDeltaMaxKey = 128;            // widest key that the kernels take
// Floats per chunk of the gate record: rho[64], w[64] (zeros for tokens that do not count), four words of facts (ChunkFacts), padding
constexpr int kDeltaGates = 136;
constexpr int kDeltaGrid = (1 << 24) - 8;    // most workgroups of 256 threads in a launch, whose threads have to stay below 2^32 (rounded up for the XCDs)
constexpr float kDeltaCut = -1e4f;           // a log decay below this discards the history (exp of it is 0 in any type)

// What a pass leaves for the next one goes past the caches (`past`: stores without a place in the last one, of 256 MiB) in walks of two waves, where
// it fills more than half of that cache and not more than all of it: training steps of 8 heads of 128 x 128, us with and without, by MiB a walk:
//   B5 T2048 (120) 382 : 384, B6 (144) 427 : 438, B7 (168) 459 : 473, B8 (192) 487 : 501, B8 T2560 (240) 610 : 616, B8 T2816 (264) 690 : 682, B8 T4096 (384)
//   1032 : 994; B4 T2048 (96) 324 : 320.
// Walks of four waves lose at every size: B16 T1024 (192) 438 : 411, B12 T2048 (288) 727 : 674, in segments B4 T4096 (192) 596 : 569.
constexpr int kPastCaches = 2;
constexpr long long kLastCache = 256ll << 20;

typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

template <typename IO> struct Mx;

template <> struct Mx<__bf16> {
  typedef bf16x8 Frag;                       // an exact operand
  struct Wide { Frag hi, lo; };              // an fp32 operand
  static constexpr int kPlanes = 2;          // arrays that hold an fp32 matrix as operands
  static RGLRU_DEVICE f32x4 mma(Frag a, Frag b, f32x4 acc) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, acc, 0, 0, 0); }
  static RGLRU_DEVICE f32x4 ew(const Frag& a, const Wide& b, f32x4 acc) { return mma(a, b.lo, mma(a, b.hi, acc)); }
  static RGLRU_DEVICE f32x4 we(const Wide& a, const Frag& b, f32x4 acc) { return mma(a.lo, b, mma(a.hi, b, acc)); }
  static RGLRU_DEVICE f32x4 ww(const Wide& a, const Wide& b, f32x4 acc) { return mma(a.lo, b.hi, mma(a.hi, b.lo, mma(a.hi, b.hi, acc))); }
  static RGLRU_DEVICE f32x4 ee(const Frag& a, const Frag& b, f32x4 acc) { return mma(a, b, acc); }
  // acc[i] += a[i] b with the parts of an fp32 operand one after the other: products that follow each other do not wait for each other
  template <int N> static RGLRU_DEVICE void ew(f32x4 (&acc)[N], const Frag (&a)[N], const Wide& b) {
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] = mma(a[i], b.hi, acc[i]);
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] = mma(a[i], b.lo, acc[i]);
  }
  template <int FROM, int TO, int N> static RGLRU_DEVICE void we(f32x4 (&acc)[N], const Wide (&a)[N], const Frag& b) {
#pragma unroll
    for (int i = FROM; i < TO; ++i) acc[i] = mma(a[i].hi, b, acc[i]);
#pragma unroll
    for (int i = FROM; i < TO; ++i) acc[i] = mma(a[i].lo, b, acc[i]);
  }
  template <int FROM, int TO, int N> static RGLRU_DEVICE void ww(f32x4 (&acc)[N], const Wide (&a)[N], const Wide& b) {
#pragma unroll
    for (int i = FROM; i < TO; ++i) acc[i] = mma(a[i].hi, b.hi, acc[i]);
#pragma unroll
    for (int i = FROM; i < TO; ++i) acc[i] = mma(a[i].hi, b.lo, acc[i]);
#pragma unroll
    for (int i = FROM; i < TO; ++i) acc[i] = mma(a[i].lo, b.hi, acc[i]);
  }
  // nearest bf16, and the nearest to what is left: off by at most 2^-9 2^-9 of the value.  The rest comes from the value and the
  // product of the pair with (-1, 0) or (0, -1), one instruction where taking the pair apart is two (a chunk converts 80 values a lane:
  // backward walk of B8 T2048 H8 of 128 223 -> 210 us).
  static RGLRU_DEVICE void halves(f32x4 v, bf16x4& hi, bf16x4& lo) {
    // from registers: as an inline constant of this instruction -1 means another pair
    unsigned lower = 0x0000bf80u, upper = 0xbf800000u;
    asm("" : "+s"(lower), "+s"(upper));
    const bf16x2 first = __builtin_bit_cast(bf16x2, lower), second = __builtin_bit_cast(bf16x2, upper);
#pragma unroll
    for (int e = 0; e < 4; e += 2) {
      const f32x2 pair = {v[e], v[e + 1]};
      const bf16x2 h = __builtin_convertvector(pair, bf16x2);
      const f32x2 rest = {__builtin_amdgcn_fdot2_f32_bf16(h, first, v[e], false), __builtin_amdgcn_fdot2_f32_bf16(h, second, v[e + 1], false)};
      const bf16x2 l = __builtin_convertvector(rest, bf16x2);
      hi[e] = h[0], hi[e + 1] = h[1];
      lo[e] = l[0], lo[e + 1] = l[1];
    }
  }
  static RGLRU_DEVICE Wide wide(f32x4 a, f32x4 b) {
    bf16x4 ah, al, bh, bl;
    halves(a, ah, al);
    halves(b, bh, bl);
    Wide w;
    w.hi = __builtin_shufflevector(ah, bh, 0, 1, 2, 3, 4, 5, 6, 7);
    w.lo = __builtin_shufflevector(al, bl, 0, 1, 2, 3, 4, 5, 6, 7);
    return w;
  }
  static RGLRU_DEVICE void apart(const Frag& f, f32x4& a, f32x4& b) {
#pragma unroll
    for (int e = 0; e < 4; ++e) a[e] = (float)f[e], b[e] = (float)f[4 + e];
  }
  // four consecutive elements of an fp32 matrix, kept in two planes `plane` elements apart
  static RGLRU_DEVICE void put(__bf16* at, long long plane, f32x4 v) {
    bf16x4 hi, lo;
    halves(v, hi, lo);
    *reinterpret_cast<bf16x4*>(at) = hi;
    *reinterpret_cast<bf16x4*>(at + plane) = lo;
  }
  static RGLRU_DEVICE f32x4 get(const __bf16* at, long long plane) {
    const bf16x4 hi = *reinterpret_cast<const bf16x4*>(at), lo = *reinterpret_cast<const bf16x4*>(at + plane);
    return f32x4{(float)hi[0] + (float)lo[0], (float)hi[1] + (float)lo[1], (float)hi[2] + (float)lo[2], (float)hi[3] + (float)lo[3]};
  }
  // the eight consecutive elements that an operand holds; `at` and `plane` in bytes
  static RGLRU_DEVICE void put(rsrc_t r, unsigned at, unsigned plane, const Wide& w, bool past) {
    const i32x4 hi = __builtin_bit_cast(i32x4, w.hi), lo = __builtin_bit_cast(i32x4, w.lo);
    if (past) {
      __builtin_amdgcn_raw_buffer_store_b128(hi, r, at, 0, kPastCaches);
      __builtin_amdgcn_raw_buffer_store_b128(lo, r, at, plane, kPastCaches);
    } else {
      __builtin_amdgcn_raw_buffer_store_b128(hi, r, at, 0, kWriteBack);
      __builtin_amdgcn_raw_buffer_store_b128(lo, r, at, plane, kWriteBack);
    }
  }
};

template <> struct Mx<float> {
  struct Frag { f32x4 lo, hi; };
  typedef Frag Wide;
  static constexpr int kPlanes = 1;
  static RGLRU_DEVICE f32x4 mma(const Frag& a, const Frag& b, f32x4 acc) {
#pragma unroll
    for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a.lo[e], b.lo[e], acc, 0, 0, 0);
#pragma unroll
    for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a.hi[e], b.hi[e], acc, 0, 0, 0);
    return acc;
  }
  static RGLRU_DEVICE f32x4 ew(const Frag& a, const Wide& b, f32x4 acc) { return mma(a, b, acc); }
  static RGLRU_DEVICE f32x4 we(const Wide& a, const Frag& b, f32x4 acc) { return mma(a, b, acc); }
  static RGLRU_DEVICE f32x4 ww(const Wide& a, const Wide& b, f32x4 acc) { return mma(a, b, acc); }
  static RGLRU_DEVICE f32x4 ee(const Frag& a, const Frag& b, f32x4 acc) { return mma(a, b, acc); }
  template <int FROM, int TO, int N> static RGLRU_DEVICE void ww(f32x4 (&acc)[N], const Frag (&a)[N], const Frag& b) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int i = FROM; i < TO; ++i) acc[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i].lo[e], b.lo[e], acc[i], 0, 0, 0);
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int i = FROM; i < TO; ++i) acc[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i].hi[e], b.hi[e], acc[i], 0, 0, 0);
  }
  template <int FROM, int TO, int N> static RGLRU_DEVICE void we(f32x4 (&acc)[N], const Frag (&a)[N], const Frag& b) { ww<FROM, TO>(acc, a, b); }
  template <int N> static RGLRU_DEVICE void ew(f32x4 (&acc)[N], const Frag (&a)[N], const Frag& b) { ww<0, N>(acc, a, b); }
  static RGLRU_DEVICE Wide wide(f32x4 a, f32x4 b) { return {a, b}; }
  static RGLRU_DEVICE void apart(const Frag& f, f32x4& a, f32x4& b) { a = f.lo, b = f.hi; }
  static RGLRU_DEVICE void put(float* at, long long, f32x4 v) { *reinterpret_cast<f32x4*>(at) = v; }
  static RGLRU_DEVICE f32x4 get(const float* at, long long) { return *reinterpret_cast<const f32x4*>(at); }
  static RGLRU_DEVICE void put(rsrc_t r, unsigned at, unsigned, const Wide& w, bool past) {
    const i32x4 first = __builtin_bit_cast(i32x4, w.lo), second = __builtin_bit_cast(i32x4, w.hi);
    if (past) {
      __builtin_amdgcn_raw_buffer_store_b128(first, r, at, 0, kPastCaches);
      __builtin_amdgcn_raw_buffer_store_b128(second, r, at + 16, 0, kPastCaches);
    } else {
      __builtin_amdgcn_raw_buffer_store_b128(first, r, at, 0, kWriteBack);
      __builtin_amdgcn_raw_buffer_store_b128(second, r, at + 16, 0, kWriteBack);
    }
  }
};

// The index that row m of accumulator tile t stands for (see above).
RGLRU_DEVICE int tile_index(int t, int m) { return 32 * (t >> 1) + 8 * (m >> 2) + 4 * (t & 1) + (m & 3); }

// A row-major [rows][COLS] tile in LDS.  Its 16-byte units are exchanged within a row by a pattern of the row.  LDS has 64 banks of
// 4 bytes; a read of 16 bytes a lane takes 4 cycles where the lanes that are served together lie in all of them.  Which lanes
// those are was found by timing all patterns that are linear in a row's lowest four bits: these are the simplest of those that every
// read below is at full rate with (4.6 .. 5.4 cycles a read with four waves reading, 8.1 .. 16 with the units as they come).
template <typename IO, int COLS> struct Tile {
  typedef Mx<IO> M;
  typedef typename M::Frag Frag;
  typedef typename M::Wide Wide;
  static constexpr int E = 16 / (int)sizeof(IO), U = COLS / E;
  static_assert(U % (COLS * (int)sizeof(IO) % 256 == 0 ? 16 : COLS * (int)sizeof(IO) % 128 == 0 ? 8 : 4) == 0, "units are exchanged in fours, eights or sixteens");
  static RGLRU_DEVICE int pattern(int row) {
    constexpr int bytes = COLS * (int)sizeof(IO), low = sizeof(IO) == 2 ? 1 : 0;
    const int r0 = row & 1, r1 = row >> 1 & 1, r3 = row >> 3 & 1;
    if constexpr (bytes % 256 == 0) return r0 << low | r3 << 2 | r1 << 3;
    else if constexpr (bytes % 128 == 0) return sizeof(IO) == 2 ? r1 << 1 | r3 << 2 : r3 | r1 << 2;
    else return r3 << low;
  }
  static RGLRU_DEVICE int unit(int row, int u) { return row * COLS + (u ^ pattern(row)) * E; }
  static RGLRU_DEVICE int at(int row, int col) { return unit(row, col / E) + col % E; }
  // operand whose contraction runs along a row: indices k0 .. k0 + 31 of row `row`
  static RGLRU_DEVICE Frag along_row(const IO* t, int row, int k0, int g) {
    if constexpr (sizeof(IO) == 2) return *reinterpret_cast<const bf16x8*>(t + at(row, k0 + 8 * g));
    else return {*reinterpret_cast<const f32x4*>(t + at(row, k0 + 8 * g)), *reinterpret_cast<const f32x4*>(t + at(row, k0 + 8 * g + 4))};
  }
  // ... runs down the rows: rows k0 .. k0 + 31 of column col0 + step (c / 4) + c % 4
  static RGLRU_DEVICE Frag down_rows(const IO* t, int k0, int col0, int step, int lane) {
    const int c = lane & 15, g = lane >> 4;
    if constexpr (sizeof(IO) == 2) {
      // ds_read_b64_tr_b16: lane i of sixteen names row i / 4, four columns of block i % 4 and receives column i, rows 0 .. 3
      typedef __attribute__((address_space(3))) bf16x4_lds* lds_ptr_t;
      const int row = k0 + 8 * g + (c >> 2), col = col0 + step * (c & 3);
      const bf16x4_lds lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_ptr_t)(t + at(row, col)));
      const bf16x4_lds hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_ptr_t)(t + at(row + 4, col)));
      return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    } else {
      const int col = col0 + step * (c >> 2) + (c & 3);
      Frag f;
#pragma unroll
      for (int e = 0; e < 4; ++e) f.lo[e] = t[at(k0 + 8 * g + e, col)], f.hi[e] = t[at(k0 + 8 * g + 4 + e, col)];
      return f;
    }
  }
  // the same for accumulator tile t of what comes out, and for sixteen columns in their order
  static RGLRU_DEVICE Frag down_rows_tile(const IO* x, int k0, int t, int lane) { return down_rows(x, k0, 32 * (t >> 1) + 4 * (t & 1), 8, lane); }
  static RGLRU_DEVICE Frag down_rows(const IO* x, int k0, int col0, int lane) { return down_rows(x, k0, col0, 4, lane); }
  // the elements that an accumulator tile's lanes hold: rows row0 + 4 g .. + 3 of column col0 + c
  static RGLRU_DEVICE f32x4 accumulator_tile(const IO* t, int row0, int col0, int lane) {
    const int c = lane & 15, g = lane >> 4;
    f32x4 v;
    if constexpr (sizeof(IO) == 2) {
      typedef __attribute__((address_space(3))) bf16x4_lds* lds_ptr_t;
      const bf16x4_lds x = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_ptr_t)(t + at(row0 + 4 * g + (c >> 2), col0 + 4 * (c & 3))));
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = (float)x[e];
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = t[at(row0 + 4 * g + e, col0 + c)];
    }
    return v;
  }
  // an fp32 matrix, whose second plane lies `plane` elements behind the first
  static RGLRU_DEVICE Wide wide_along_row(const IO* t, int plane, int row, int k0, int g) {
    if constexpr (sizeof(IO) == 2) return {along_row(t, row, k0, g), along_row(t + plane, row, k0, g)};
    else return along_row(t, row, k0, g);
  }
  static RGLRU_DEVICE Wide wide_down_rows_tile(const IO* x, int plane, int k0, int t, int lane) {
    if constexpr (sizeof(IO) == 2) return {down_rows_tile(x, k0, t, lane), down_rows_tile(x + plane, k0, t, lane)};
    else return down_rows_tile(x, k0, t, lane);
  }
  static RGLRU_DEVICE Wide wide_down_rows(const IO* x, int plane, int k0, int col0, int lane) {
    if constexpr (sizeof(IO) == 2) return {down_rows(x, k0, col0, lane), down_rows(x + plane, k0, col0, lane)};
    else return down_rows(x, k0, col0, lane);
  }
};

// Everything that the kernels of one pass read and write.  Strides in elements; the last axis of q, k, v is contiguous.
// Matrices that one kernel leaves for the next are kept as operands (Mx::put), per chunk and value head, transposed where they
// come from accumulators: lanes hold four consecutive rows of one column there.
struct DeltaArgs {
  const void *q, *k, *v, *log_decay, *beta, *dout;
  const unsigned char* flags;
  const float *h0, *dh_last;
  void *out, *dq, *dk, *dv, *dlog_decay, *dbeta;
  float *h_last, *dh0;
  void *solve, *within;              // [chunks][64 j][64 i]: T and P of a chunk, transposed
  float* gates;                      // [chunks][kDeltaGates]
  void *states, *values;             // [chunks][dv][dk], [chunks][dv][64]: state in front of a chunk, solved values (both transposed)
  void *dstates, *dvalues;           // the same of the backward pass: gradient behind a chunk, gradient of the values
  // A sequence in several segments of `length` chunks that are walked side by side: [heads][segments][columns][padded K] and, for
  // `through`, [heads][segments][padded K in][padded K out]
  float *local, *edges;              // what a segment adds to the state (or its gradient); the state a segment starts from
  void* through;                     // what a segment makes of the state it starts from, as an operand
  int* cut;                          // [heads][segments]: whether a segment leaves nothing of that state
  int segments, length, past;
  long long q_b, q_t, q_h, k_b, k_t, k_h, v_b, v_t, v_h;
  int B, T, H, HV, K, V, nC, columns;       // columns: V in whole tiles of 16
  int decay_dtype, beta_dtype;
  int width;                                // of the rows of q and k as the kernels read them: K in whole 16-byte vectors
  int value_width;                          // the same of v and dout
  long long up_b, up_t, up_h;               // strides of dout as the kernels read it
  float scale;
};

RGLRU_DEVICE float delta_gate(const void* p, long long i, int dtype) {
  return dtype == 1 ? (float)((const __bf16*)p)[i] : ((const float*)p)[i];
}
RGLRU_DEVICE void delta_put_gate(void* p, long long i, int dtype, float v) {
  if (dtype == 1) ((__bf16*)p)[i] = (__bf16)v;
  else ((float*)p)[i] = v;
}

// Running log decay of a chunk, one token a lane.  64 bits: the products need differences of sums that may be thousands apart.
// A reset (or a decay of nothing) starts a segment; nothing is carried from one segment into the next.
struct ChunkGates {
  double total;          // sum of the log decays up to this token, segment starts left out
  double end;            // ... up to the chunk's end
  int segment, segments; // segment of this token, of the last one
  bool counts, starts;   // token of the sequence that is not masked; its history is discarded
  float beta;
};
RGLRU_DEVICE ChunkGates chunk_gates(const DeltaArgs& p, int b, int hv, int n, int lane) {
  ChunkGates r;
  const int t = n * kDeltaChunk + lane;
  const unsigned flag = t < p.T && p.flags ? p.flags[(long long)b * p.T + t] : 0u;
  r.counts = t < p.T && !(flag & 2u);
  const long long at = ((long long)b * p.T + t) * p.HV + hv;
  float g = r.counts ? delta_gate(p.log_decay, at, p.decay_dtype) : 0.f;
  r.beta = r.counts ? delta_gate(p.beta, at, p.beta_dtype) : 0.f;
  r.starts = r.counts && ((flag & 1u) || g < kDeltaCut);
  if (r.starts) g = 0.f;
  const unsigned long long starts = __ballot(r.starts);
  r.segment = __popcll(starts & (~0ull >> (63 - lane)));
  r.segments = __popcll(starts);
  double sum = (double)g;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const double other = __shfl_up(sum, d, 64);
    if (lane >= d) sum += other;
  }
  r.total = sum;
  r.end = __shfl(sum, 63, 64);
  return r;
}

RGLRU_DEVICE i32x4 delta_rsrc(const void* base, unsigned bytes) {
  const unsigned long long at = (unsigned long long)base;
  i32x4 r;
  r[0] = __builtin_amdgcn_readfirstlane((int)(unsigned)at);
  r[1] = __builtin_amdgcn_readfirstlane((int)((unsigned)(at >> 32) & 0xffffu));
  r[2] = __builtin_amdgcn_readfirstlane((int)bytes);
  r[3] = 0x00020000;
  return r;
}
RGLRU_DEVICE unsigned lds_address(const void* p) {
  return __builtin_amdgcn_readfirstlane((unsigned)(size_t)(const __attribute__((address_space(3))) char*)p);
}
// Sixteen bytes a lane from memory to LDS, once or four times `STEP` bytes apart there; the wave's lanes lie one behind the other from
// `lds` on, offsets past the descriptor's extent give zeros.  The compiler does not count these loads: whoever reads the tile waits for all
// of the wave's (and for the other waves' at a barrier).  The wait states in front are for a descriptor that a vector instruction has
// just written (a uniform value, or one that was put aside).
RGLRU_DEVICE void memory_to_lds(i32x4 r, unsigned off, unsigned lds) {
  asm volatile("s_nop 4\n\ts_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds), "v"(off), "s"(r) : "memory", "m0");
}
template <int STEP> RGLRU_DEVICE void memory_to_lds(i32x4 r, unsigned off0, unsigned off1, unsigned off2, unsigned off3, unsigned lds) {
  asm volatile(
      "s_nop 4\n\ts_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %5, 0 offen lds\n\t"
      "s_add_u32 m0, m0, %6\n\ts_nop 0\n\tbuffer_load_dwordx4 %2, %5, 0 offen lds\n\t"
      "s_add_u32 m0, m0, %6\n\ts_nop 0\n\tbuffer_load_dwordx4 %3, %5, 0 offen lds\n\t"
      "s_add_u32 m0, m0, %6\n\ts_nop 0\n\tbuffer_load_dwordx4 %4, %5, 0 offen lds" ::"s"(lds),
      "v"(off0), "v"(off1), "v"(off2), "v"(off3), "s"(r), "n"(STEP)
      : "memory", "m0", "scc");
}
RGLRU_DEVICE void wait_for_all() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// A row-major matrix on its way into an LDS tile.
template <typename IO, int ROWS, int COLS, int THREADS> struct TileLoad {
  typedef Tile<IO, COLS> T;
  static constexpr int kBytes = ROWS * COLS * (int)sizeof(IO), kUnits = ROWS * T::U, kWhole = kUnits / THREADS, N = (kUnits + THREADS - 1) / THREADS;
  static_assert(kUnits % 64 == 0, "whole waves");
  unsigned off[N];
  RGLRU_DEVICE void setup(int tid, long long stride, int width) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int at = tid + i * THREADS, row = at / T::U, col = ((at % T::U) ^ T::pattern(row)) * T::E;
      off[i] = col < width ? (unsigned)row * (unsigned)(stride * (int)sizeof(IO)) + (unsigned)col * (unsigned)sizeof(IO) : kOutOfRange;
    }
  }
  // bytes from the first element to the end of the last of `rows` rows
  static RGLRU_DEVICE unsigned extent(long long stride, int width, int rows) {
    rows = rows < ROWS ? rows : ROWS;
    return rows > 0 ? (unsigned)((rows - 1) * stride + width) * (unsigned)sizeof(IO) : 0u;
  }
  RGLRU_DEVICE void request(i32x4 r, unsigned lds, int wave) const {
    constexpr int STEP = THREADS * 16;
    lds += (unsigned)wave * 1024u;
#pragma unroll
    for (int i = 0; i + 4 <= kWhole; i += 4) memory_to_lds<STEP>(r, off[i], off[i + 1], off[i + 2], off[i + 3], lds + (unsigned)(i * STEP));
#pragma unroll
    for (int i = kWhole / 4 * 4; i < N; ++i)
      if (i < kWhole || i * THREADS + wave * 64 < kUnits) memory_to_lds(r, off[i], lds + (unsigned)(i * STEP));
  }
};

// A chunk's rows of a [tokens, columns] tensor, a lane's column.  Only a lane's own offset is checked against the descriptor's extent,
// so rows go into the scalar offset where the chunk is whole, else into the lane's: those past the end are not written.
template <typename IO> struct ColumnIo {
  rsrc_t rsrc;
  unsigned row_bytes, first;
  bool whole;
  // lane_row: the first of the lane's rows
  RGLRU_DEVICE ColumnIo(const IO* base, long long stride, int rows, int width, int col, bool live, int lane_row)
      : rsrc(make_rsrc(base, (unsigned)(((rows < kDeltaChunk ? rows : kDeltaChunk) - 1) * stride + width) * (unsigned)sizeof(IO))),
        row_bytes((unsigned)(stride * (long long)sizeof(IO))),
        first(live ? (unsigned)lane_row * row_bytes + (unsigned)col * (unsigned)sizeof(IO) : kOutOfRange), whole(rows >= kDeltaChunk) {}
  RGLRU_DEVICE unsigned at(int row) const { return first == kOutOfRange ? kOutOfRange : first + (unsigned)row * row_bytes; }
  // four accumulator tiles of rows; the lane's first row is 8 g
  static RGLRU_DEVICE int tile_row(int i) { return 32 * (i >> 3) + 4 * ((i >> 2) & 1) + (i & 3); }
  RGLRU_DEVICE void store(int row, float v) const { BufIo<IO>::store((IO)v, rsrc, at(row), 0); }
  RGLRU_DEVICE void store(const f32x4 (&v)[4]) const {
    if (whole) {
#pragma unroll
      for (int i = 0; i < 16; ++i) BufIo<IO>::store((IO)v[i / 4][i % 4], rsrc, first, (unsigned)tile_row(i) * row_bytes);
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) BufIo<IO>::store((IO)v[i / 4][i % 4], rsrc, at(tile_row(i)), 0);
    }
  }
};

// What a walk along the chunks has in LDS of one chunk, and how it gets there: keys, queries, T, P, the gate record, and `COLUMNS` columns of
// the values or the upstream gradients.
template <typename IO, int KS, int WAVES, bool OUT> struct ChunkTiles {
  static constexpr int DK = 32 * KS, PL = Mx<IO>::kPlanes, THREADS = 64 * WAVES, COLUMNS = 16 * WAVES;
  typedef TileLoad<IO, 64, DK, THREADS> KeyLoad;
  typedef TileLoad<IO, PL * 64, 64, THREADS> SquareLoad;
  typedef TileLoad<IO, 64, COLUMNS, THREADS> ValueLoad;
  static constexpr int kKeys = 0, kSolve = KeyLoad::kBytes, kValues = kSolve + SquareLoad::kBytes, kQueries = kValues + ValueLoad::kBytes,
                       kWithin = kQueries + (OUT ? KeyLoad::kBytes : 0), kRecord = kWithin + (OUT ? SquareLoad::kBytes : 0),
                       kBytes = kRecord + 1024;             // the record: one vector a lane of one wave
  KeyLoad k, q;
  SquareLoad square;
  ValueLoad value;
  unsigned record;
  const IO *keys, *queries, *values, *solve, *within;      // of the chunk that is requested next
  const float* gates;
  long long value_stride;
  int value_width, left, step;
  // From chunk n of a sequence on (`chunk` of all), forwards or backwards; first_values: the sequence's first row at the group's first column
  RGLRU_DEVICE void setup(const DeltaArgs& p, int tid, const IO* first_values, long long stride, int width, long long chunk, int n, int b, int h, int step_) {
    k.setup(tid, p.k_t, p.width);
    if constexpr (OUT) q.setup(tid, p.q_t, p.width);
    square.setup(tid, 64, 64);
#pragma unroll
    for (int i = 0; i < SquareLoad::N; ++i)                 // the quarter above the diagonal is neither written nor used
      if ((square.off[i] / (64 * (unsigned)sizeof(IO)) & 32) && (square.off[i] & (32 * (unsigned)sizeof(IO)))== 0) square.off[i] = kOutOfRange;
    value_stride = stride, value_width = width < COLUMNS ? width : COLUMNS;
    value.setup(tid, stride, width);
    record = (tid & 63) * 16 < kDeltaGates * 4 ? (unsigned)(tid & 63) * 16u : kOutOfRange;
    const long long t0 = (long long)n * kDeltaChunk;
    keys = (const IO*)p.k + b * p.k_b + t0 * p.k_t + h * p.k_h;
    queries = (const IO*)p.q + b * p.q_b + t0 * p.q_t + h * p.q_h;
    values = first_values + t0 * stride;
    solve = (const IO*)p.solve + chunk * (4096 * PL);
    within = (const IO*)p.within + chunk * (4096 * PL);
    gates = p.gates + chunk * kDeltaGates;
    left = p.T - (int)t0, step = step_;
  }
  RGLRU_DEVICE void request(const DeltaArgs& p, unsigned lds, int wave) {
    k.request(delta_rsrc(keys, KeyLoad::extent(p.k_t, p.width, left)), lds + kKeys, wave);
    square.request(delta_rsrc(solve, SquareLoad::kBytes), lds + kSolve, wave);
    if (value_width > 0) value.request(delta_rsrc(values, ValueLoad::extent(value_stride, value_width, left)), lds + kValues, wave);
    if constexpr (OUT) {
      q.request(delta_rsrc(queries, KeyLoad::extent(p.q_t, p.width, left)), lds + kQueries, wave);
      square.request(delta_rsrc(within, SquareLoad::kBytes), lds + kWithin, wave);
    }
    if (wave == 0) memory_to_lds(delta_rsrc(gates, kDeltaGates * 4), record, lds + kRecord);
    keys += step * kDeltaChunk * p.k_t, queries += step * kDeltaChunk * p.q_t, values += step * kDeltaChunk * value_stride;
    solve += step * 4096 * PL, within += step * 4096 * PL, gates += step * kDeltaGates, left -= step * kDeltaChunk;
  }
  // zeros for the rows of tokens that do not count
  template <typename LOAD> static RGLRU_DEVICE void clear(unsigned char* tile, unsigned long long counts, int tid) {
    for (int at = tid; at < 64 * LOAD::T::U; at += THREADS)
      if (!((counts >> (at / LOAD::T::U)) & 1)) *reinterpret_cast<i32x4*>(tile + at * 16) = i32x4{0, 0, 0, 0};
  }
  static RGLRU_DEVICE void clear_rows(unsigned char* stage, unsigned long long counts, int tid) {
    clear<KeyLoad>(stage + kKeys, counts, tid);
    clear<ValueLoad>(stage + kValues, counts, tid);
    if constexpr (OUT) clear<KeyLoad>(stage + kQueries, counts, tid);
  }
};

// Sixteen columns of 64 tokens that a wave has in its accumulators on their way to memory, through the wave's columns of a value tile:
// whole vectors of a row a lane.
template <typename IO, int COLUMNS> struct WaveRows {
  typedef Tile<IO, COLUMNS> T;
  static constexpr int VECTORS = 16 / T::E, N = 64 * VECTORS / 64;       // vectors of a row; of a lane
  i32x4 v[N];
  RGLRU_DEVICE void turn(IO* tile, const f32x4 (&x)[4], int wave, int lane) {
    const int c = lane & 15, g = lane >> 4;
#pragma unroll
    for (int i = 0; i < 16; ++i) tile[T::at(tile_index(i / 4, 4 * g + i % 4), 16 * wave + c)] = (IO)x[i / 4][i % 4];
    wave_lds_fence();
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = *reinterpret_cast<const i32x4*>(tile + T::at((i * 64 + lane) / VECTORS, 16 * wave + lane % VECTORS * T::E));
  }
  // rows: that are there; width: of the tensor
  RGLRU_DEVICE void store(IO* base, long long stride, int rows, int width, int col, int lane) const {
    const rsrc_t r = make_rsrc(base, (unsigned)(((rows < kDeltaChunk ? rows : kDeltaChunk) - 1) * stride + width) * (unsigned)sizeof(IO));
    const int at = col + lane % VECTORS * T::E;
#pragma unroll
    for (int i = 0; i < N; ++i)
      buf_store_b128(v[i], r, at < width ? ((unsigned)((i * 64 + lane) / VECTORS) * (unsigned)stride + (unsigned)at) * (unsigned)sizeof(IO) : kOutOfRange);
  }
};

// A chunk's products come in phases; the operands of the next one are requested in front of each.  The scheduler keeps to that: by itself
// it requests those of all phases at once and runs out of registers.
RGLRU_DEVICE void phase() { __builtin_amdgcn_sched_barrier(0); }

// Four rows of each of the tiles 2 p and 2 p + 1 from an array of 64 numbers.
RGLRU_DEVICE f32x4 tile_rows(const float* a, int mt, int g) { return *reinterpret_cast<const f32x4*>(a + 32 * (mt >> 1) + 8 * g + 4 * (mt & 1)); }

// What a gate record says about its chunk.  Where the first token that counts starts a document (`fresh`), the chunk reads nothing of the state
// in front of it and hands no gradient back; where no token counts, both pass by.  Whatever they hold: a factor of zero would keep a NaN.
struct ChunkFacts {
  unsigned long long counts;         // tokens that count, a bit each
  bool fresh, plain;                 // plain: all of them count, and not fresh
  float carry;                       // what the chunk leaves of the state in front of it
  RGLRU_DEVICE explicit ChunkFacts(const float* record) {
    const f32x4 words = *reinterpret_cast<const f32x4*>(record + 128);
    const unsigned lo = __builtin_amdgcn_readfirstlane(__float_as_uint(words[0])), hi = __builtin_amdgcn_readfirstlane(__float_as_uint(words[1]));
    counts = (unsigned long long)lo | (unsigned long long)hi << 32;
    fresh = __builtin_amdgcn_readfirstlane(__float_as_uint(words[2])) != 0;
    carry = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(words[3])));
    plain = counts == ~0ull && !fresh;
  }
};

// Whether a walk's workgroups are of two waves with two chunks' tiles in LDS (they fit in bf16 only) instead of four waves with one: where there
// are so few that each has a compute unit to itself and the time a chunk takes is all that counts.
inline bool delta_narrow(const DeltaArgs& a) { return a.segments == 1 && (long long)((a.columns + 31) / 32) * a.B * a.HV <= num_compute_units(); }

// XCDs take workgroups round-robin; each gets a contiguous run of the work, so that neighbours share its L2.  -1: none left.
RGLRU_DEVICE int xcd_order(int block, int total) {
  const int per = (total + 7) >> 3, at = (block & 7) * per + (block >> 3);
  return (block >> 3) < per && at < total ? at : -1;
}

inline dim3 xcd_grid(long long total) { return dim3((unsigned)((total + 7) / 8 * 8)); }

}  // namespace rglru
