// The matrix-product tile of the gated unit (gated.hip): C = A * B with both
// operands read as they lie in memory, whichever way their contraction runs.
//
//   TR = false: operand [row][k], k contiguous  (x and dG in X W, dG W^T)
//   TR = true:  operand [k][row], row contiguous (W in X W, both in X^T dG)
//
// 256 threads, 4 waves as 2 x 2, one wave per SIMD; a wave holds FM x FN
// fragments of v_mfma_f32_16x16x32 (FM = FN = 8: a 256 x 256 tile, 256
// accumulator registers a lane). Wide wave tiles are what the LDS allows: per
// 32 k a wave reads 16 (FM + FN) rows of 64 bytes for FM FN products of 16
// cycles, 64 B/cycle of the CU's 128 at 8 x 8, but 96 for 8 waves of 8 x 4.
//
// Stages of 64 (or 32) k go straight from memory to LDS (16 bytes a lane), into
// two buffers in turn or four; the fragments of the next 32 k are read while
// the present ones multiply, so a stage costs one barrier. Buffer loads put
// zeros where rows, columns or the contraction end.
#pragma once

#include "common.h"

namespace dvgg {

typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
typedef __attribute__((address_space(3))) s16x8 lds_s16x8;
typedef __attribute__((address_space(3))) void lds_void;
typedef __attribute__((address_space(3))) char lds_char;

// c += a * b on a fragment pair. Written out so that the accumulator stays
// where it is: through the builtin, result and addend are two registers and
// the loop around them copies 128 and more of them a turn. In this order the
// source is the schedule: products and the reads between them stay put.
// The compiler knows nothing of the instruction's timing here: accumulators
// are set to 0 well before their first product, mfma_wait() ends every piece
// of straight code with products in it, since the compiler may move
// accumulators about where pieces join, and mfma_done() comes before any use.
// tests/test_accumulator_waits.py looks at what was built.
template <class T>
DEV void mfma32(f32x4& c, s16x8 a, s16x8 b);
template <>
DEV void mfma32<__bf16>(f32x4& c, s16x8 a, s16x8 b) {
  asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0"
               : "+a"(c) : "v"(a), "v"(b));
}
template <>
DEV void mfma32<_Float16>(f32x4& c, s16x8 a, s16x8 b) {
  asm volatile("v_mfma_f32_16x16x32_f16 %0, %1, %2, %0"
               : "+a"(c) : "v"(a), "v"(b));
}
// 11 wait states before another instruction may touch the result; behind its
// own builtin the compiler leaves 8
DEV void mfma_wait() {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_nop 10");
  __builtin_amdgcn_sched_barrier(0);
}
template <int FM, int FN>
DEV void mfma_done(f32x4 (&c)[FM][FN]) {
  mfma_wait();
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) asm volatile("" : "+a"(c[i][j]));
}

using u64 = unsigned long long;

constexpr u32 OUT_OF_RANGE = 0x80000000u;   // no buffer here reaches it

// A value that all lanes share, in a scalar register: the compiler does not
// see it of every one, and a buffer that it takes to differ between lanes
// costs a loop over them.
DEV u32 uniform(u32 v) { return __builtin_amdgcn_readfirstlane(v); }
DEV const u16* uniform(const u16* p) {
  u64 v = reinterpret_cast<u64>(p);
  return reinterpret_cast<const u16*>(
      u64(uniform(u32(v >> 32))) << 32 | uniform(u32(v)));
}

// One half of an operand's rows in one stage: ROWS rows x BK k (64 or 32).
template <bool TR, int ROWS, int BK>
struct Panel {
  static constexpr int BYTES = ROWS * BK * 2;
  static constexpr int LOADS = BYTES / 4096;    // 16-byte loads a thread
  static constexpr int PITCH = TR ? ROWS * 2 : BK * 2;

  // 16-byte segments (TR = false) trade places by row so that the 16 rows
  // that a fragment reads together fall into 16 different bank groups.
  // TR = true: 32-byte chunks trade places by k so that the 4 + 4 rows of k
  // that two 16-lane groups read together do.
  DEV static int swz(int r) {
    if (!TR) return BK == 64 ? (r >> 1) & 7 : (r >> 2) & 3;
    if (ROWS >= 128) return (r & 3) | ((r >> 3) & 1) << 2;
    return ((r >> 1) & 1) | ((r >> 3) & 1) << 1;
  }

  u32 voff[LOADS];     // byte offset of this lane's segment in the stage
  int kpos[LOADS];     // its first k (TR = false)
  DEV void init(int wave, int lane, u32 ld, int rows_left) {
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      int byte = (wave * LOADS + i) * 1024 + lane * 16;
      int r = byte / PITCH, seg = byte % PITCH / 16;
      int src = TR ? (((seg >> 1) ^ swz(r)) << 1 | (seg & 1)) : seg ^ swz(r);
      kpos[i] = src * 8;
      // the buffer's length ends the outer direction, this the inner one
      bool in = !TR || src * 8 < rows_left;
      voff[i] = in ? u32(r) * ld * 2 + src * 16 : OUT_OF_RANGE;
    }
  }

  // Load number i. base: the operand at (row 0 of the panel, k 0 of this
  // stage); k_left: how much of the contraction is left from there.
  DEV void load(lds_char* dst, const u16* base, u32 ld, int rows_left,
                int k_left, int wave, int i) const {
    // rows of memory are whole vectors: a last one that the operand fills
    // in part is followed by its padding
    const int kk = max(min(k_left, BK), 0);
    const int rr = max(min(rows_left, ROWS), 0);
    const int outer = TR ? kk : rr, inner = ((TR ? rr : kk) + 7) & ~7;
    const u32 bytes = min(outer, 1) * min(inner, 1) *
                      ((outer - 1) * ld + inner) * 2;
    auto rsrc = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<u16*>(uniform(base)), 0, uniform(bytes), 0x00020000);
    u32 off = TR || kpos[i] < k_left ? voff[i] : OUT_OF_RANGE;
    __builtin_amdgcn_raw_ptr_buffer_load_lds(
        rsrc, (lds_void*)(dst + (wave * LOADS + i) * 1024), 16, off, 0, 0, 0);
  }
};

// Reads a wave's fragments out of a panel: F fragments of 16 rows from row
// `first` (a multiple of 16 * F, or of 64).
template <bool TR, int ROWS, int BK, int F>
struct Frags {
  using P = Panel<TR, ROWS, BK>;
  u32 addr[TR ? F : 1];
  DEV void init(int lane, int first) {
    if (!TR) {
      int r = first + (lane & 15);
      addr[0] = r * BK * 2 + (((lane >> 4) ^ P::swz(r)) << 4);
    } else {
      int k = (lane >> 4) * 8 + ((lane & 15) >> 2);
#pragma unroll
      for (int j = 0; j < F; ++j) {
        int chunk = (first / 16 + j) ^ P::swz(k);
        addr[j] = k * ROWS * 2 + chunk * 32 + (lane & 3) * 8;
      }
    }
  }
  DEV s16x8 read(const lds_char* panel, int j, int half) const {
    if (!TR) {
      u32 a = addr[0] ^ (half << 6);
      return *(const lds_s16x8*)(panel + a + j * 32 * BK);
    }
    const lds_char* p = panel + addr[j] + half * 32 * ROWS * 2;
    s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p);
    s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (lds_s16x4*)(p + 4 * ROWS * 2));
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  }
};

// The stages' buffers: up to four objects, so that reads of one do not wait for
// loads into the others. (An array of them would become a constant in memory.)
struct Bufs {
  lds_char *b0, *b1, *b2, *b3;
  template <int N>
  DEV lds_char* at() const {
    return N == 0 ? b0 : N == 1 ? b1 : N == 2 ? b2 : b3;
  }
};

constexpr int max_(int a, int b) { return a > b ? a : b; }

// What one tile multiplies. The contraction may come in two parts with
// memory of their own (dG Wg^T + dU Wu^T): their stages take turns. So may
// the two halves of the tile's columns (X Wg | X Wu).
struct TileSrc {
  const u16* a[2];          // [part]: row 0 of the tile, k 0
  const u16* b[2][2];       // [part][half]: column 0 of the half, k 0
  u32 lda, ldb;
  int rows_a, rows_b[2];    // rows of A, columns of each half that exist
  int k_first, k_last;      // the contraction [k_first, k_last) of each part
};

// RING: buffers, 2 or 4. With four, three stages are under way while one is
// multiplied, and a tile needs no other on its CU to cover for it.
// BK: k of a stage. Stages of 64 take a barrier for every two steps of 32
// and keep rows of 128 bytes together; stages of 32 take half the LDS, and
// more tiles share a CU.
// PAIRED: a wave takes the same columns of both halves, else all columns of
// one. SHORT: the whole contraction is one stage, which then is all the LDS
// that the tile needs; more tiles share a CU.
template <class T, bool ATR, bool BTR, int PARTS, int FM, int FN, int BK,
          int RING, bool PAIRED, bool SHORT>
struct Tile {
  static constexpr int BM = 32 * FM, BN = 32 * FN, HALF = BN / 2;
  using PA = Panel<ATR, BM, BK>;
  using PB = Panel<BTR, HALF, BK>;
  static constexpr int STAGE = PA::BYTES + 2 * PB::BYTES;
  static constexpr int LOADS = PA::LOADS + 2 * PB::LOADS;
  static constexpr int FH = PAIRED ? FN / 2 : FN;  // fragments in a half

  PA pa;
  PB pb[2];
  Frags<ATR, BM, BK, FM> ra;
  Frags<BTR, HALF, BK, FH> rb;
  // B's fragments twice where registers allow, of this step and of the next
  static constexpr int SETS = FM * FN >= 64 ? 2 : 1;
  s16x8 fa[FM], fb[SETS][FN];
  int wave;

  // Loads number `i` of a stage. Behind the last k the buffers are empty:
  // zeros land in LDS and no memory moves.
  template <int PART>
  DEV void load(const TileSrc& s, lds_char* dst, int k, int i) {
    const int left = s.k_last - k;
    const i64 ka = ATR ? (i64)k * s.lda : k, kb = BTR ? (i64)k * s.ldb : k;
    if (i < PA::LOADS)
      pa.load(dst, s.a[PART] + ka, s.lda, s.rows_a, left, wave, i);
    else if (i < PA::LOADS + PB::LOADS)
      pb[0].load(dst + PA::BYTES, s.b[PART][0] + kb, s.ldb, s.rows_b[0],
                 left, wave, i - PA::LOADS);
    else
      pb[1].load(dst + PA::BYTES + PB::BYTES, s.b[PART][1] + kb, s.ldb,
                 s.rows_b[1], left, wave, i - PA::LOADS - PB::LOADS);
  }
  DEV void fetch_a(const lds_char* src, int half, int i) {
    fa[i] = ra.read(src, i, half);
  }
  DEV void fetch_b(const lds_char* src, int half, int set, int j) {
    const int h = PAIRED ? j / FH : wave & 1;
    fb[set][j] = rb.read(src + PA::BYTES + h * PB::BYTES, j % FH, half);
  }

  // 32 k: the products of the fragments at hand, row by row of A, from set
  // SET of B's. Between them, one or two at a time and spread evenly (a
  // product keeps the matrix core for 16 cycles and issues in 4; the LDS
  // needs 8 for a read of each of four waves: bunched up, the others hold the
  // products up):
  //   - the reads of the next fragments, from half `half` of `src` (LAST:
  //     there are none), A's behind the last use of each, B's into the other
  //     set or, where there is one, behind the last use. That of A's last row
  //     comes in the next step, so this one begins with its own, from half
  //     `own` of `cur`;
  //   - REFILL, the step that changes over to the next stage: after its first
  //     rows every wave is done reading `dst` and its own loads into `src`
  //     have landed, so it syncs there, with products still queued; then the
  //     loads that refill `dst`.
  enum Kind { PLAIN, REFILL, LAST };
  template <Kind KIND, int STEP, int PART>
  DEV void step(const TileSrc& s, const lds_char* cur, int own,
                const lds_char* src, int half, lds_char* dst, int k,
                f32x4 (&acc)[FM][FN]) {
    constexpr bool FILL = KIND == REFILL;
    constexpr int SET = STEP % SETS, NEXT = (STEP + 1) % SETS;
    constexpr int ROW0 = !FILL ? 0 : FM > 2 ? 2 : 1;    // first row of reads
    constexpr int SLOTS = (FM - ROW0) * FN;
    // where the loads go: not into a last row that is full of reads
    constexpr int ROOM = SETS == 2 ? SLOTS : max_(FM - 1 - ROW0, 1) * FN;
#pragma unroll
    for (int i = 0; i < FM; ++i) {
#pragma unroll
      for (int j = 0; j < FN; ++j) {
        mfma32<T>(acc[i][j], fb[SET][j], fa[i]);
        if (i == 0 && j == 0) fetch_a(cur, own, FM - 1);
        if (KIND != LAST && i >= ROW0) {
          const int t = (i - ROW0) * FN + j;
          if (j == 1 && i > 0) fetch_a(src, half, i - 1);
          if (j == 3 && i == 2 && ROW0 == 2) fetch_a(src, half, 0);
          if (SETS == 1 && i == FM - 1) fetch_b(src, half, 0, j);
          if (SETS == 2) {
#pragma unroll
            for (int b = 0; b < FN; ++b)
              if (b * SLOTS / FN + 2 == t) fetch_b(src, half, NEXT, b);
          }
          if (FILL) {
#pragma unroll
            for (int l = 0; l < LOADS; ++l)
              if (l * ROOM / LOADS == t) load<PART>(s, dst, k, l);
          }
        }
      }
      if (FILL && i == ROW0 - 1) sync<(RING - 2) * LOADS>();
    }
    __builtin_amdgcn_sched_barrier(0);
  }

  // this wave's loads have landed but for the last LEFT, and its reads are
  // done; then all waves'
  template <int LEFT>
  DEV static void sync() {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" :: "n"(LEFT) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  }

  // acc[i][j]: rows 16 i + lane % 16 of the wave's 16 FM; columns
  // 16 (j % FH) + 4 (lane / 16) + 0..3 of the wave's in half j / FH (PAIRED)
  // or in its own half.
  DEV void run(const Bufs& buf, const TileSrc& s, int wave_,
               int lane, f32x4 (&acc)[FM][FN]) {
    constexpr int LASTH = BK / 32 - 1;          // last half of a stage
    wave = wave_;
    pa.init(wave, lane, s.lda, s.rows_a);
    pb[0].init(wave, lane, s.ldb, s.rows_b[0]);
    pb[1].init(wave, lane, s.ldb, s.rows_b[1]);
    ra.init(lane, (wave >> 1) * 16 * FM);
    rb.init(lane, PAIRED ? (wave & 1) * 8 * FN : 0);
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j) {
        acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
        asm volatile("" : "+a"(acc[i][j]));   // here, not just before its use
      }
    first<0>(buf, s);
    sync<(SHORT ? 0 : RING - 1) * LOADS>();
#pragma unroll
    for (int j = 0; j < FN; ++j) fetch_b(buf.at<0>(), 0, 0, j);
#pragma unroll
    for (int i = 0; i < FM - 1; ++i) fetch_a(buf.at<0>(), 0, i);
    if constexpr (SHORT) {
      lds_char* one = buf.at<0>();
      if (BK == 64) step<PLAIN, 0, 0>(s, one, 0, one, 1, one, 0, acc);
      step<LAST, LASTH, 0>(s, one, LASTH, one, 0, one, 0, acc);
    } else {
      // turns of all buffers: missing last stages are zeros
      for (int k = s.k_first; k < s.k_last; k += TURN) {
        stages<0>(buf, s, k, acc);
        mfma_wait();        // behind the loop accumulators may be moved
      }
    }
    // zeros still on their way must not land in what comes after
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    mfma_done(acc);
  }

  // k of a turn of all buffers, and where in it buffer n is
  static constexpr int TURN = RING * BK / PARTS;
  static constexpr int k_of(int n) { return n / PARTS * BK; }
  template <int N>
  DEV void first(const Bufs& buf, const TileSrc& s) {
#pragma unroll
    for (int l = 0; l < LOADS; ++l)
      load<N % PARTS>(s, buf.at<N>(), s.k_first + k_of(N), l);
    if constexpr (!SHORT && N + 1 < RING) first<N + 1>(buf, s);
  }
  template <int N>
  DEV void stages(const Bufs& buf, const TileSrc& s, int k,
                  f32x4 (&acc)[FM][FN]) {
    constexpr int LASTH = BK / 32 - 1, NEXT = (N + 1) % RING;
    lds_char* now = buf.at<N>();
    if constexpr (BK == 64)
      step<PLAIN, 0, N % PARTS>(s, now, 0, now, 1, now, 0, acc);
    step<REFILL, BK == 64 ? 1 : N & 1, N % PARTS>(
        s, now, LASTH, buf.at<NEXT>(), 0, now, k + TURN + k_of(N), acc);
    if constexpr (N + 1 < RING) stages<N + 1>(buf, s, k, acc);
  }
};

}  // namespace dvgg
