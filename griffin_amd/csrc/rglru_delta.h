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
#include "rglru_host.h"

namespace rglru {

constexpr int kDeltaChunk = 64;              // tokens of a chunk
constexpr int kDeltaThreads = 256;
constexpr int kDeltaMaxKey = 128;            // widest key that the kernels take
constexpr int kDeltaGates = 136;             // floats per chunk of the gate record: rho[64], w[64], 64 bits that say which tokens count, padding
constexpr float kDeltaCut = -1e4f;           // a log decay below this discards the history (exp of it is 0 in any type)

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
  // nearest bf16, and the nearest to what is left: off by at most 2^-9 2^-9 of the value
  static RGLRU_DEVICE void halves(f32x4 v, bf16x4& hi, bf16x4& lo) {
#pragma unroll
    for (int e = 0; e < 4; e += 2) {
      const f32x2 pair = {v[e], v[e + 1]};
      const bf16x2 h = __builtin_convertvector(pair, bf16x2);
      const unsigned bits = __builtin_bit_cast(unsigned, h);
      const f32x2 rest = {v[e] - __uint_as_float(bits << 16), v[e + 1] - __uint_as_float(bits & 0xffff0000u)};
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
  int width;                                // of the rows of q and k as the kernels read them: K in whole 16-byte vectors
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

// Rows of keys, queries or upstream gradients of a chunk as an LDS tile, zeros where a token does not count or the tile is wider than
// the row.  The vectors are requested into registers and put down later.
template <typename IO, int COLS, int THREADS> struct KeyRows {
  typedef Tile<IO, COLS> T;
  static constexpr int N = kDeltaChunk * T::U / THREADS;   // vectors a thread
  i32x4 v[N];
  RGLRU_DEVICE void request(const IO* rows, long long stride, int width, unsigned long long counts, bool vec, int tid) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int at = tid + i * THREADS, row = at / T::U, col = at % T::U * T::E;
      v[i] = i32x4{0, 0, 0, 0};
      if (((counts >> row) & 1) && col < width) {
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
  static constexpr int kBytes = ROWS * COLS * (int)sizeof(IO), N = ROWS * T::U / THREADS;
  static_assert(N * THREADS == ROWS * T::U, "whole vectors a thread");
  unsigned off[N];
  RGLRU_DEVICE void setup(int tid, long long stride, int width) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int at = tid + i * THREADS, row = at / T::U, col = ((at % T::U) ^ ((row >> T::kShift) & T::kMask)) * T::E;
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
    for (int i = 0; i + 4 <= N; i += 4) memory_to_lds<STEP>(r, off[i], off[i + 1], off[i + 2], off[i + 3], lds + (unsigned)(i * STEP));
#pragma unroll
    for (int i = N / 4 * 4; i < N; ++i) memory_to_lds(r, off[i], lds + (unsigned)(i * STEP));
  }
};

// One element of a [tokens, columns] tensor a lane: rows 16 mt + 4 g + e of a chunk, one column.  Rows past the `rows` there are read
// as zeros and not written.
template <typename IO> struct ColumnIo {
  rsrc_t rsrc;
  unsigned row_bytes, first;
  RGLRU_DEVICE ColumnIo(const IO* base, long long stride, int rows, int width, int col, bool live, int g)
      : rsrc(make_rsrc(base, (unsigned)(((rows < kDeltaChunk ? rows : kDeltaChunk) - 1) * stride + width) * (unsigned)sizeof(IO))),
        row_bytes((unsigned)(stride * (long long)sizeof(IO))),
        first(live ? (unsigned)(4 * g) * row_bytes + (unsigned)col * (unsigned)sizeof(IO) : kOutOfRange) {}
  // the offset of a lane without a column stays out of range: at most 64 rows of 2^22 elements are added to it, modulo 2^32
  RGLRU_DEVICE unsigned at(int mt, int e) const { return first == kOutOfRange ? kOutOfRange : first + (unsigned)(16 * mt + e) * row_bytes; }
  // as it lies in memory, so that nothing waits for it before it is used
  static RGLRU_DEVICE float value(int raw) { return sizeof(IO) == 2 ? __uint_as_float((unsigned)raw << 16) : __uint_as_float((unsigned)raw); }
  RGLRU_DEVICE int raw(int mt, int e) const {
    if constexpr (sizeof(IO) == 2) return (int)(unsigned short)__builtin_amdgcn_raw_buffer_load_b16(rsrc, at(mt, e), 0, 0);
    else return (int)__builtin_amdgcn_raw_buffer_load_b32(rsrc, at(mt, e), 0, 0);
  }
  RGLRU_DEVICE void store(int mt, int e, float v) const { BufIo<IO>::store((IO)v, rsrc, at(mt, e), 0); }
};

// What a walk along the chunks has in LDS of one chunk, and how it gets there.  Two of them where they fit: the next chunk's is
// filled while this one's is worked on.
template <typename IO, int KS, int THREADS, bool OUT> struct ChunkTiles {
  static constexpr int DK = 32 * KS, PL = Mx<IO>::kPlanes;
  typedef TileLoad<IO, 64, DK, THREADS> KeyLoad;
  typedef TileLoad<IO, PL * 64, 64, THREADS> SquareLoad;
  static constexpr int kKeys = 0, kSolve = KeyLoad::kBytes, kQueries = kSolve + SquareLoad::kBytes,
                       kWithin = kQueries + (OUT ? KeyLoad::kBytes : 0), kRecord = kWithin + (OUT ? SquareLoad::kBytes : 0),
                       kBytes = kRecord + 1024;             // the record: one vector a lane of one wave
  static constexpr int kStages = 2 * kBytes <= 160 * 1024 ? 2 : 1;
  KeyLoad k, q;
  SquareLoad square;
  unsigned record;
  RGLRU_DEVICE void setup(const DeltaArgs& p, int tid) {
    k.setup(tid, p.k_t, p.width);
    if constexpr (OUT) q.setup(tid, p.q_t, p.width);
    square.setup(tid, 64, 64);
    record = (tid & 63) * 16 < kDeltaGates * 4 ? (unsigned)(tid & 63) * 16u : kOutOfRange;
  }
  RGLRU_DEVICE void request(const DeltaArgs& p, long long chunk, int n, int b, int h, unsigned lds, int wave) const {
    const int t0 = n * kDeltaChunk, left = p.T - t0;
    const i32x4 rk = delta_rsrc((const IO*)p.k + b * p.k_b + t0 * p.k_t + h * p.k_h, KeyLoad::extent(p.k_t, p.width, left));
    const i32x4 rs = delta_rsrc((const IO*)p.solve + chunk * (4096 * PL), SquareLoad::kBytes);
    const i32x4 rq = delta_rsrc((const IO*)p.q + b * p.q_b + t0 * p.q_t + h * p.q_h, OUT ? KeyLoad::extent(p.q_t, p.width, left) : 0u);
    const i32x4 rw = delta_rsrc((const IO*)p.within + chunk * (4096 * PL), SquareLoad::kBytes);
    const i32x4 rr = delta_rsrc(p.gates + chunk * kDeltaGates, kDeltaGates * 4);
    k.request(rk, lds + kKeys, wave);
    square.request(rs, lds + kSolve, wave);
    if constexpr (OUT) {
      q.request(rq, lds + kQueries, wave);
      square.request(rw, lds + kWithin, wave);
    }
    if (wave == 0) memory_to_lds(rr, record, lds + kRecord);
  }
  // zeros for the rows of tokens that do not count
  static RGLRU_DEVICE void clear_rows(unsigned char* stage, unsigned long long counts, int tid) {
    for (int at = tid; at < 64 * KeyLoad::T::U; at += THREADS) {
      const int row = at / KeyLoad::T::U;
      if ((counts >> row) & 1) continue;
      *reinterpret_cast<i32x4*>(stage + kKeys + at * 16) = i32x4{0, 0, 0, 0};
      if constexpr (OUT) *reinterpret_cast<i32x4*>(stage + kQueries + at * 16) = i32x4{0, 0, 0, 0};
    }
  }
};
RGLRU_DEVICE unsigned long long counts_of(const float* record) {
  const unsigned lo = __builtin_amdgcn_readfirstlane(__float_as_uint(record[128])), hi = __builtin_amdgcn_readfirstlane(__float_as_uint(record[129]));
  return (unsigned long long)lo | (unsigned long long)hi << 32;
}

// Whether a walk's workgroups are of two waves instead of four: where those of four leave compute units without one.
inline bool delta_narrow(const DeltaArgs& a) { return (long long)(a.columns + 63) / 64 * a.B * a.HV < num_compute_units(); }

// XCDs take workgroups round-robin; each gets a contiguous run of the work, so that neighbours share its L2.  -1: none left.
RGLRU_DEVICE int xcd_order(int block, int total) {
  const int per = (total + 7) >> 3, at = (block & 7) * per + (block >> 3);
  return (block >> 3) < per && at < total ? at : -1;
}

}  // namespace rglru
