// Building blocks of the gated delta rule's kernels (gfx950, wave64): 16 x 16 matrix products whose operands come from LDS
// tiles or straight from the accumulators of the product before.
//
// An accumulator tile of v_mfma_f32_16x16 gives lane (c = lane % 16, g = lane / 16) the rows 4 g .. 4 g + 3 of column c.  The
// B operand of the next product wants lane (c, g) to hold eight contraction indices of column c, and a contraction may run over
// its indices in any order that both operands share: with the order 4 g .. 4 g + 3, 16 + 4 g .. 16 + 4 g + 3 of 32 indices, two
// accumulator tiles ARE that operand.  So a wave that owns 16 columns of the state takes it from product to product in its
// registers; LDS holds only what comes from memory, and every A operand is read in that order.
//
// bf16 storage: keys, queries and upstream gradients are exact matrix operands; what is computed (state, solved values, the
// chunk's triangular matrices) enters as the sum of two bf16 numbers, 2^-17 relative, because one bf16 number would round the
// carried state to 2^-9 once a chunk.  fp32 storage: v_mfma_f32_16x16x4_f32 throughout.
#pragma once

#include "rglru_device.h"

namespace rglru {

constexpr int kDeltaChunk = 64;              // tokens of a chunk
constexpr int kDeltaThreads = 256;
constexpr int kDeltaMaxKey = 128;            // widest key that the kernels take
constexpr int kDeltaGates = 136;             // floats per chunk of the gate record: rho[64], write[64], 64 bits of "token counts", padding
constexpr float kDeltaCut = -1e4f;           // a log decay below this discards the history (exp of it is 0 in any type)

typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

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
  // nearest bf16, and the nearest to what is left: off by at most 2^-9 2^-9 of the value
  static RGLRU_DEVICE void halves(f32x4 v, bf16x4& hi, bf16x4& lo) {
#pragma unroll
    for (int e = 0; e < 4; ++e) hi[e] = (__bf16)v[e];
#pragma unroll
    for (int e = 0; e < 4; ++e) lo[e] = (__bf16)(v[e] - (float)hi[e]);
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
  static RGLRU_DEVICE Frag exact(f32x4 a, f32x4 b) {
    Frag f;
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = (__bf16)a[e], f[4 + e] = (__bf16)b[e];
    return f;
  }
  // four consecutive elements of an fp32 matrix, kept in two planes `plane` elements apart
  static RGLRU_DEVICE void put(__bf16* at, long long plane, f32x4 v) {
    bf16x4 hi, lo;
    halves(v, hi, lo);
    *reinterpret_cast<bf16x4*>(at) = hi;
    *reinterpret_cast<bf16x4*>(at + plane) = lo;
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
  static RGLRU_DEVICE Wide wide(f32x4 a, f32x4 b) { return {a, b}; }
  static RGLRU_DEVICE Frag exact(f32x4 a, f32x4 b) { return {a, b}; }
  static RGLRU_DEVICE void put(float* at, long long, f32x4 v) { *reinterpret_cast<f32x4*>(at) = v; }
};

constexpr int delta_pow2_divisor(int n, int most) {
  int p = 1;
  while (p < most && n % (2 * p) == 0) p *= 2;
  return p;
}
constexpr int delta_bank_period(int row_bytes) {           // rows after which a column lies in the same bank again, as a shift
  int s = 0;
  while (s < 2 && (row_bytes << s) % 256 != 0) ++s;
  return s;
}

// A row-major [rows][COLS] tile in LDS.  Its 16-byte units are exchanged within a row by a pattern of the row, so that sixteen
// rows of one column (what one operand read touches) spread over all banks without padding.
template <typename IO, int COLS> struct Tile {
  typedef Mx<IO> M;
  typedef typename M::Frag Frag;
  typedef typename M::Wide Wide;
  static constexpr int E = 16 / (int)sizeof(IO), U = COLS / E;
  static constexpr int kShift = delta_bank_period(COLS * (int)sizeof(IO)), kMask = delta_pow2_divisor(U, 16) - 1;
  static RGLRU_DEVICE int unit(int row, int u) { return row * COLS + ((u ^ ((row >> kShift) & kMask)) * E); }
  static RGLRU_DEVICE int at(int row, int col) { return unit(row, col / E) + col % E; }
  // A (or B) operand whose contraction runs along a row: indices k0 .. k0 + 31 of row `row`
  static RGLRU_DEVICE Frag along_row(const IO* t, int row, int k0, int g) {
    const IO *a = t + at(row, k0 + 4 * g), *b = t + at(row, k0 + 16 + 4 * g);
    if constexpr (sizeof(IO) == 2) {
      const bf16x4 lo = *reinterpret_cast<const bf16x4*>(a), hi = *reinterpret_cast<const bf16x4*>(b);
      return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    } else {
      return {*reinterpret_cast<const f32x4*>(a), *reinterpret_cast<const f32x4*>(b)};
    }
  }
  // ... runs down the rows: rows k0 .. k0 + 31 of column col0 + c
  static RGLRU_DEVICE Frag down_rows(const IO* t, int k0, int col0, int lane) {
    const int c = lane & 15, g = lane >> 4;
    if constexpr (sizeof(IO) == 2) {
      // ds_read_b64_tr_b16: lane i of sixteen names row i / 4, columns 4 (i % 4) .. + 3 and receives column i, rows 0 .. 3
      typedef __attribute__((address_space(3))) bf16x4_lds* lds_ptr_t;
      const int row = k0 + 4 * g + (c >> 2), col = col0 + 4 * (c & 3);
      const bf16x4_lds lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_ptr_t)(t + at(row, col)));
      const bf16x4_lds hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_ptr_t)(t + at(row + 16, col)));
      return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    } else {
      Frag f;
#pragma unroll
      for (int e = 0; e < 4; ++e) f.lo[e] = t[at(k0 + 4 * g + e, col0 + c)], f.hi[e] = t[at(k0 + 16 + 4 * g + e, col0 + c)];
      return f;
    }
  }
  // the same for an fp32 matrix; its second plane lies `plane` elements behind the first
  static RGLRU_DEVICE Wide wide_along_row(const IO* t, int plane, int row, int k0, int g) {
    if constexpr (sizeof(IO) == 2) return {along_row(t, row, k0, g), along_row(t + plane, row, k0, g)};
    else return along_row(t, row, k0, g);
  }
  static RGLRU_DEVICE Wide wide_down_rows(const IO* t, int plane, int k0, int col0, int lane) {
    if constexpr (sizeof(IO) == 2) return {down_rows(t, k0, col0, lane), down_rows(t + plane, k0, col0, lane)};
    else return down_rows(t, k0, col0, lane);
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
  long long q_b, q_t, q_h, k_b, k_t, k_h, v_b, v_t, v_h;
  int B, T, H, HV, K, V, nC, columns;       // columns: V in whole tiles of 16
  int decay_dtype, beta_dtype;
  int vec_q, vec_k;                         // rows of q and k can be read as 16-byte vectors
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

// Rows of keys or queries of a chunk as an LDS tile, zeros where a token does not count or the tile is wider than the key.
// The vectors are requested into registers and put down later, so that a whole chunk's work lies between the two.
template <typename IO, int COLS, int THREADS> struct KeyRows {
  typedef Tile<IO, COLS> T;
  static constexpr int N = kDeltaChunk * T::U / THREADS;   // vectors a thread
  i32x4 v[N];
  RGLRU_DEVICE void request(const IO* rows, long long stride, int width, int left, unsigned long long counts, bool vec, int tid) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int at = tid + i * THREADS, row = at / T::U, col = at % T::U * T::E;
      v[i] = i32x4{0, 0, 0, 0};
      if (row < left && ((counts >> row) & 1) && col < width) {
        const IO* src = rows + (long long)row * stride + col;
        if (vec) {
          v[i] = *reinterpret_cast<const i32x4*>(src);
        } else {
          IO e[T::E];
#pragma unroll
          for (int j = 0; j < T::E; ++j) e[j] = col + j < width ? src[j] : (IO)0.0f;
          __builtin_memcpy(&v[i], e, 16);
        }
      }
    }
  }
  RGLRU_DEVICE void put(IO* tile, int tid) const {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int at = tid + i * THREADS;
      *reinterpret_cast<i32x4*>(tile + T::unit(at / T::U, at % T::U)) = v[i];
    }
  }
};

// Planes of an fp32 matrix [ROWS][COLS] in memory as LDS tiles, one behind the other.
template <typename IO, int ROWS, int COLS, int THREADS> struct MatrixRows {
  typedef Tile<IO, COLS> T;
  static constexpr int kUnits = Mx<IO>::kPlanes * ROWS * T::U, N = (kUnits + THREADS - 1) / THREADS;
  static_assert(kUnits % THREADS == 0, "whole vectors a thread");
  i32x4 v[N];
  // `src`: first plane's first row to take; `plane`: elements from plane to plane; `rows`: rows that are there
  RGLRU_DEVICE void request(const IO* src, long long plane, int rows, int tid) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int at = tid + i * THREADS, which = at / (ROWS * T::U), row = at / T::U % ROWS, u = at % T::U;
      v[i] = row < rows ? *reinterpret_cast<const i32x4*>(src + which * plane + (long long)row * COLS + u * T::E) : i32x4{0, 0, 0, 0};
    }
  }
  RGLRU_DEVICE void put(IO* tile, int tid) const {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int at = tid + i * THREADS, which = at / (ROWS * T::U), row = at / T::U % ROWS, u = at % T::U;
      *reinterpret_cast<i32x4*>(tile + which * ROWS * COLS + T::unit(row, u)) = v[i];
    }
  }
};

// One element of a [tokens, columns] tensor a lane: rows 16 mt + 4 g + e of the chunk, one column.
template <typename IO> struct ColumnIo {
  rsrc_t rows;
  unsigned row_bytes, col_bytes;
  RGLRU_DEVICE ColumnIo(const IO* base, long long stride, int col, bool live)
      : rows(make_rsrc(base, 0x40000000u)), row_bytes((unsigned)(stride * (long long)sizeof(IO))), col_bytes(live ? (unsigned)col * (unsigned)sizeof(IO) : kOutOfRange) {}
  RGLRU_DEVICE unsigned at(int row, bool ok) const { return ok && col_bytes != kOutOfRange ? (unsigned)row * row_bytes + col_bytes : kOutOfRange; }
  RGLRU_DEVICE float load(int row, bool ok) const { return BufIo<IO>::load(rows, at(row, ok), 0); }
  RGLRU_DEVICE void store(int row, bool ok, float v) const { BufIo<IO>::store((IO)v, rows, at(row, ok), 0); }
};

// XCDs take workgroups round-robin; each gets a contiguous run of the work, so that neighbours share its L2.  -1: none left.
RGLRU_DEVICE int xcd_order(int block, int total) {
  const int per = (total + 7) >> 3, at = (block & 7) * per + (block >> 3);
  return (block >> 3) < per && at < total ? at : -1;
}

}  // namespace rglru
