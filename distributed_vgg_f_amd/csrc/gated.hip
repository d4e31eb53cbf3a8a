// The gated fully connected unit:
//
//   G = X Wg + bg, U = X Wu + bu, H = keep act(G) U / (1 - p)
//
// with X [M][K], W [K][N] and the mask of dropout (philox.h). The forward
// pass is one product whose tiles hold the same columns of G and U, so the
// activation, the product and the mask are its epilogue. Backward:
//
//   dU = keep dH act(G) / (1-p), dG = keep dH U act'(G) / (1-p)
//   dX = dG Wg^T + dU Wu^T, dWg = X^T dG, dWu = X^T dU, db = column sums
//
// one pass over dH, G and U, then two products on the same tiles.
//
// Roundings: sums, biases, the activation and the column sums stay in 32
// bits, and so do G and U kept for the backward pass: rounded to 16 they
// nearly double the error of the gradients (bf16, 256 x 9216 x 4096: 0.0031
// of their size instead of 0.0024, one rounding of the result being 0.0017),
// and they are 3 to 4 % of the time at the largest sizes, less elsewhere. dG and
// dU are rounded to the type of x, which the matrix instructions take; that is
// all of the difference between the 0.0024 and the 0.0017. Gradients are
// rounded to the type of x whatever the type of the buffer that they go to.

#include <torch/extension.h>
#include <ATen/hip/HIPContext.h>

#include "mfma_tile.h"
#include "philox.h"

namespace dvgg {

static inline hipStream_t cur_stream() {
  return at::hip::getCurrentHIPStreamMasqueradingAsCUDA().stream();
}

// ------------------------------------------------------------- activations
enum Act { SILU, GELU, GELU_TANH, RELU, SIGMOID };

DEV float sigmoid_f(float z) {
  return __builtin_amdgcn_rcpf(1.f + __expf(-z));
}

typedef __attribute__((ext_vector_type(8))) float f32x8;

// act(g) and act'(g) of 8 elements; the switch stands outside their loop.
// tanh(z) = 2 sigmoid(2z) - 1, so the tanh form of gelu is g sigmoid(2z):
// nothing cancels. NaN passes through all of them.
template <class F>
DEV f32x8 each(f32x8 g, F f) {
#pragma unroll
  for (int r = 0; r < 8; ++r) g[r] = f(g[r], r);
  return g;
}
DEV f32x8 act8(int act, f32x8 g, f32x8& d) {
  switch (act) {
    case RELU:
      d = each(g, [](float v, int) { return v <= 0.f ? 0.f : 1.f; });
      return each(g, [](float v, int) { return v <= 0.f ? 0.f : v; });
    case GELU:
      // g Phi(g). For x = |g| / sqrt(2), erfc(x) = exp(-x^2) t (a1 + t (a2 +
      // ... a8)), t = 1 / (1 + 7/16 x): coefficients of the least squares of
      // the relative error under weights that Lawson's method evens out, off
      // by at most 1.7e-7 of erfc for x to 14. Relative, since g Phi(g) is
      // nothing but erfc for g < 0: with 7.1.26 of Abramowitz and Stegun, off
      // by 1.5e-7 of 1, gelu(-5) was off by 0.2 % and gelu(-8) by 1 %. What is
      // left are the 3.5 g^2 2^-24 of the rounded exponent. The derivative
      // takes the same exponential.
      return each(g, [&](float v, int r) {
        float x = 0.70710678118654752f * __builtin_fabsf(v);
        float t = __builtin_amdgcn_rcpf(1.f + 0.4375f * x);
        float e = __expf(-x * x);
        float c = 0.5f * e * t * (0.24679698f + t * (0.2477052f + t *
                  (0.21449493f + t * (0.22275093f + t * (-0.03513595f + t *
                  (0.317385f + t * (-0.28582388f + t * 0.07182687f)))))));
        c = v > 0.f ? 1.f - c : c;
        d[r] = c + v * 0.39894228040143268f * e;
        return v * c;
      });
    case GELU_TANH:
      return each(g, [&](float v, int r) {
        float s = sigmoid_f(1.5957691216057308f * (v + 0.044715f * v * v * v));
        float w = s * (1.f - s);
        // w is 0 where v * v no longer fits 32 bits
        d[r] = w > 0.f ? s + v * w * 1.5957691216057308f *
                             (1.f + 0.134145f * v * v) : s;
        return v * s;
      });
    case SIGMOID:
      // s' = e / (1 + e)^2 with e = exp(-g): s (1 - s) would cancel where s
      // is near 1, by 0.5 % at 12. Past 1e38 s is 0, and e may be infinite.
      return each(g, [&](float v, int r) {
        float e = __expf(-v), s = __builtin_amdgcn_rcpf(1.f + e);
        d[r] = __builtin_fminf(e, 1e38f) * s * s;
        return s;
      });
    default:
      return each(g, [&](float v, int r) {
        float s = sigmoid_f(v);
        d[r] = s * (1.f + v * (1.f - s));
        return v * s;
      });
  }
}

// Bits 0..7: which of the 8 elements from flat index i stay. They lie in two
// blocks of the generator if i is a multiple of 4, else in three.
DEV u32 keep8(const DropArgs& d, u32 off, i64 i) {
  const u32 sh = u32(i & 3);
  i >>= 2;
  u32 k = keep4(d, off, i) | keep4(d, off, i + 1) << 4;
  if (sh) k = (k | keep4(d, off, i + 2) << 8) >> sh;
  return k & 255u;
}

// The same for 4 elements: one block, or two.
DEV u32 keep4_from(const DropArgs& d, u32 off, i64 i) {
  const u32 sh = u32(i & 3);
  i >>= 2;
  u32 k = keep4(d, off, i);
  if (sh) k = (k | keep4(d, off, i + 1) << 4) >> sh;
  return k & 15u;
}

// ---------------------------------------------------------------- epilogue
struct OutArgs {
  u16* h;             // [M][N]
  float* gu;          // [2][M][ldg] or null
  const u16* bias[2]; // [N] or null
  int M, N;
  i64 ldg;
  int act;
  int drop;           // 1: keep/scale by `d`
  DropArgs d;
};

DEV f32x8 load8f(const float* v) {
  f32x4 a = *reinterpret_cast<const f32x4*>(v);
  f32x4 b = *reinterpret_cast<const f32x4*>(v + 4);
  return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}
DEV void store8f(float* p, f32x8 v) {
  *reinterpret_cast<f32x4*>(p) = __builtin_shufflevector(v, v, 0, 1, 2, 3);
  *reinterpret_cast<f32x4*>(p + 4) = __builtin_shufflevector(v, v, 4, 5, 6, 7);
}

// 8 columns to row c of N. Rows of odd lengths start anywhere: those stores
// are as wide as the compiler makes them for 2-byte alignment.
DEV void store8(u16* c, int n, int N, s16x8 v) {
  if ((N & 7) == 0) {
    *reinterpret_cast<s16x8*>(c + n) = v;
  } else if (n + 8 <= N) {
    __builtin_memcpy(c + n, &v, 16);
  } else {
#pragma unroll
    for (int r = 0; r < 8; ++r)
      if (n + r < N) c[n + r] = u16(v[r]);
  }
}
// 8 columns of a row of N, zeros behind it
DEV s16x8 load8(const u16* c, int n, int N) {
  s16x8 v = {0, 0, 0, 0, 0, 0, 0, 0};
  if (n + 8 <= N) {
    __builtin_memcpy(&v, c + n, 16);
  } else {
#pragma unroll
    for (int r = 0; r < 8; ++r)
      if (n + r < N) v[r] = short(c[n + r]);
  }
  return v;
}

template <class T>
DEV s16x8 round8(f32x8 v) {
  s16x8 o;
#pragma unroll
  for (int r = 0; r < 8; ++r) o[r] = short(from_f(v[r], T()));
  return o;
}

template <class T>
DEV f32x8 widen8(s16x8 v) {
  f32x8 o;
#pragma unroll
  for (int r = 0; r < 8; ++r) o[r] = to_f(u16(v[r]), T());
  return o;
}

// 8 columns of a bias from column n, a multiple of 8
template <class T>
DEV f32x8 bias8(const u16* b, int n, int N) {
  f32x8 v{};
  if (b) {
#pragma unroll
    for (int r = 0; r < 8; ++r) v[r] = to_f(b[min(n + r, N - 1)], T());
  }
  return v;
}

// 8 columns of one row of G and U, n a multiple of 8.
template <class T>
DEV void finish8(const OutArgs& o, u32 off, int m, int n, f32x8 g, f32x8 u) {
  if (o.gu) {         // rows of ldg, a multiple of 8, hold all eight
    float* gp = o.gu + (i64)m * o.ldg + n;
    store8f(gp, g);
    store8f(gp + (i64)o.M * o.ldg, u);
  }
  f32x8 d;
  u *= act8(o.act, g, d);
  if (o.drop) {
    const u32 keep = keep8(o.d, off, (i64)m * o.N + n);
#pragma unroll
    for (int r = 0; r < 8; ++r) u[r] = (keep >> r & 1) ? u[r] * o.d.scale : 0.f;
  }
  store8(o.h + (i64)m * o.N, n, o.N, round8<T>(u));
}

// ---------------------------------------------------------------- products
// FWD    [M][2N] = X [Wg | Wu]             a tile: 16 FN columns of each
// DGRAD  [M][K]  = dG Wg^T + dU Wu^T       two parts of the contraction
// WGRAD  2 x [K][N] = X^T dG, X^T dU       a tile lies in one of the two; or
//                                          one of them alone
enum Mode { FWD, DGRAD, WGRAD };

struct ProductArgs {
  const u16* a[2];
  const u16* b[2];
  i64 lda, ldb;
  int rows, cols;       // of one output matrix
  int k_len;
  int splits;
  int tiles_m, tiles_n;
  int mats;             // output matrices: FWD 2, DGRAD 1, WGRAD either
  float* slab;          // [splits][mats][rows][slab_ld] if splits > 1
  i64 slab_ld;          // cols rounded up to 8
  u16* c[2];            // outputs of DGRAD ([0]) and WGRAD
  OutArgs out;          // of FWD
};

// Four columns each of two neighbouring fragments, rounded, and traded
// between the 16-lane rows so that each lane has 8 columns side by side: rows
// 0 and 2 the first and last 8 of fragment a, rows 1 and 3 those of b.
template <class T>
DEV s16x8 trade(f32x4 a, f32x4 b) {
  union { u32 w[4]; s16x4 h[2]; s16x8 v; } t;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    t.h[0][r] = short(from_f(a[r], T()));
    t.h[1][r] = short(from_f(b[r], T()));
  }
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    auto p = __builtin_amdgcn_permlane16_swap(t.w[k], t.w[k + 2], false, false);
    t.w[k] = p[0];
    t.w[k + 2] = p[1];
  }
  return t.v;
}

// The tiles by rule: make_plan() below. At 8192 x 4096 x 8192 in bf16, each
// product 1.1 TFLOP: forward 0.96 ms (1.15 PFLOP/s; 0.67 GB leave it, G and U
// among them), dX 0.87 (1.27), both weights 0.81 (1.36), all of 256 x 256
// tiles with the matrix cores busy for 60, 66 and 73 % of the cycles. What
// bounds it there is power: the clock falls to 1.9 GHz, of the 2.4 that short
// kernels run at, and 32x32x16 products took 917 and 970 us in place of 840
// and 876. At 256 x 9216 x 4096 the forward product takes 60 us, joined in 2,
// for 151 MB of weights and 17 of slabs (with weights that the last-level cache
// holds 43). That is 2.9 TB/s, where rows_kernel streams such weights at 5.1:
// no limit of the memory but of loads and products that wait for each other;
// wider reads of the weights (tiles of 64 x 256) took 73.
template <class T, int MODE, int FM, int FN, int BK, int RING,
          bool SHORT = false>
__global__ __launch_bounds__(256, SHORT || BK * RING == 64 ? 4
                                  : RING == 4 || FM * FN == 64 ? 1 : 2)
void product_kernel(ProductArgs p) {
  constexpr bool ATR = MODE == WGRAD, BTR = MODE != DGRAD;
  using TL = Tile<T, ATR, BTR, MODE == DGRAD ? 2 : 1, FM, FN, BK,
                  RING, MODE == FWD, SHORT>;
  // an object each, so that reads of one do not wait for loads into others
  constexpr int SECOND = SHORT ? 16 : TL::STAGE;
  constexpr int MORE = RING == 4 ? TL::STAGE : 16;
  __shared__ __attribute__((aligned(1024))) char lds0[TL::STAGE];
  __shared__ __attribute__((aligned(1024))) char lds1[SECOND];
  __shared__ __attribute__((aligned(1024))) char lds2[MORE];
  __shared__ __attribute__((aligned(1024))) char lds3[MORE];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

  // neighbours on one XCD share panels: tiles run down groups of 8 rows
  u32 id = xcd_swizzle(blockIdx.x, gridDim.x);
  const int tiles = p.tiles_m * p.tiles_n;
  const int split = __builtin_amdgcn_readfirstlane(id / tiles);
  int t = id - split * tiles;
  const int group = 8 * p.tiles_n;
  const int g0 = t / group * 8, gs = min(8, p.tiles_m - g0);
  t %= group;
  const int m0 = __builtin_amdgcn_readfirstlane((g0 + t % gs) * TL::BM);
  int tn = __builtin_amdgcn_readfirstlane(t / gs);
  // WGRAD of both: the second half of the tile columns belongs to dU
  const int which = MODE == WGRAD && p.mats == 2 && tn >= p.tiles_n / 2;
  if (which) tn -= p.tiles_n / 2;
  const int n0 = tn * (MODE == FWD ? TL::HALF : TL::BN);

  TileSrc s;
  s.lda = u32(p.lda);
  s.ldb = u32(p.ldb);
  s.rows_a = p.rows - m0;
  s.rows_b[0] = p.cols - n0;
  s.rows_b[1] = MODE == FWD ? p.cols - n0 : p.cols - n0 - TL::HALF;
  const i64 am = ATR ? m0 : (i64)m0 * p.lda;
  const i64 bn = BTR ? n0 : (i64)n0 * p.ldb;
  const i64 bh = BTR ? TL::HALF : (i64)TL::HALF * p.ldb;
  s.a[0] = p.a[0] + am;
  s.a[1] = p.a[MODE == DGRAD] + am;
  if (MODE == FWD) {
    s.b[0][0] = s.b[1][0] = p.b[0] + bn;
    s.b[0][1] = s.b[1][1] = p.b[1] + bn;
  } else {
    s.b[0][0] = (which ? p.b[1] : p.b[0]) + bn;
    s.b[0][1] = s.b[0][0] + bh;
    s.b[1][0] = p.b[1] + bn;
    s.b[1][1] = s.b[1][0] + bh;
  }
  // parts of whole turns of the loop
  constexpr int TURN = TL::TURN;
  const int turns = (p.k_len + TURN - 1) / TURN;
  const int each_ = turns / p.splits, more = turns % p.splits;
  s.k_first = (split * each_ + min(split, more)) * TURN;
  s.k_last = min(s.k_first + (each_ + (split < more)) * TURN, p.k_len);

  f32x4 acc[FM][FN];
  TL tile;
  Bufs buf;
  buf.b0 = (lds_char*)lds0;
  buf.b1 = (lds_char*)lds1;
  buf.b2 = (lds_char*)lds2;
  buf.b3 = (lds_char*)lds3;
  tile.run(buf, s, wave, lane, acc);

  // Straight from the accumulators: a trip through LDS for wider stores took
  // 5 us a 256 x 256 tile, of 14 in all besides its products. Lane (c, q):
  // rows 16 i + c, columns 16 j + 4 q + 0..3 of fragment j, or, traded, the
  // 8 from column 16 (j + q % 2) + 8 (q / 2) of the fragments j and j + 1.
  const int c = lane & 15, q = lane >> 4;
  const int mw = m0 + (wave >> 1) * 16 * FM + c;
  const int wide = 16 * (q & 1) + 8 * (q >> 1);
  if constexpr (MODE != FWD) {
    const int nw = n0 + (wave & 1) * TL::HALF;
#pragma unroll
    for (int i = 0; i < FM; ++i) {
      const int m = mw + 16 * i;
      if (m >= p.rows) continue;
      if (p.splits == 1) {
        u16* o = (which ? p.c[1] : p.c[0]) + (i64)m * p.cols;
#pragma unroll
        for (int j = 0; j < FN; j += 2) {
          s16x8 v = trade<T>(acc[i][j], acc[i][j + 1]);
          const int n = nw + 16 * j + wide;
          if (n < p.cols) store8(o, n, p.cols, v);
        }
      } else {
        float* o = p.slab +
            (((i64)split * p.mats + which) * p.rows + m) * p.slab_ld;
#pragma unroll
        for (int j = 0; j < FN; ++j) {
          const int n = nw + 16 * j + 4 * q;
          if (n < p.cols) *reinterpret_cast<f32x4*>(o + n) = acc[i][j];
        }
      }
    }
  } else {
    constexpr int H = FN / 2;               // fragments of G and of U
    const int nw = n0 + (wave & 1) * 8 * FN;
    if (p.splits > 1) {
#pragma unroll
      for (int i = 0; i < FM; ++i) {
        const int m = mw + 16 * i;
        if (m >= p.rows) continue;
        float* o = p.slab + ((i64)split * 2 * p.rows + m) * p.slab_ld;
#pragma unroll
        for (int j = 0; j < H; ++j) {
          const int n = nw + 16 * j + 4 * q;
          if (n >= p.cols) continue;
          *reinterpret_cast<f32x4*>(o + n) = acc[i][j];
          *reinterpret_cast<f32x4*>(o + (i64)p.rows * p.slab_ld + n) =
              acc[i][j + H];
        }
      }
      return;
    }
    const OutArgs& o = p.out;
    if constexpr (FM * FN == 64) {
      // Here the straight form spills and runs through ten thousand
      // instructions once a tile: besides its products a round of tiles took
      // 16.5 us, through LDS in pieces of 32 rows 14.2, and in this form, 64
      // rows of a wave at a time, which is all of the LDS, in a loop that has
      // the next read under way, 12.8. 16-byte chunks trade places by row.
      static_assert(TL::STAGE == 65536 && RING == 2, "32 KB a wave");
      __syncthreads();
      float* mine = reinterpret_cast<float*>((wave & 2 ? lds1 : lds0) +
                                             (wave & 1) * 32768);
      const u32 off = o.drop ? o.d.off() : 0;
      const int n = nw + (lane & 7) * 8;
      const f32x8 bg = bias8<T>(o.bias[0], n, o.N);
      const f32x8 bu = bias8<T>(o.bias[1], n, o.N);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < FN; ++j)
            *reinterpret_cast<f32x4*>(mine + (16 * i + c) * 128 +
                                      ((4 * j + q) ^ c) * 4) =
                acc[4 * half + i][j];
        auto chunk = [&](int row, int k) {
          return *reinterpret_cast<const f32x4*>(mine + row * 128 +
                                                 (k ^ (row & 15)) * 4);
        };
        f32x4 v[4];
        auto read = [&](int it) {
          const int row = (it & 7) * 8 + (lane >> 3), k = (lane & 7) * 2;
          v[0] = chunk(row, k);
          v[1] = chunk(row, k + 1);
          v[2] = chunk(row, k + 16);
          v[3] = chunk(row, k + 17);
        };
        read(0);
        const int m0w = m0 + (wave >> 1) * 128 + half * 64 + (lane >> 3);
#pragma unroll 1
        for (int it = 0; it < 8; ++it) {
          f32x8 g = __builtin_shufflevector(v[0], v[1], 0, 1, 2, 3, 4, 5, 6, 7);
          f32x8 u = __builtin_shufflevector(v[2], v[3], 0, 1, 2, 3, 4, 5, 6, 7);
          read(it + 1);
          const int m = m0w + it * 8;
          if (m < p.rows && n < p.cols)
            finish8<T>(o, off, m, n, g + bg, u + bu);
        }
      }
      return;
    }
    // the mask first, BITS bits a row, in one loop that is not unrolled: one
    // copy of the generator
    constexpr int BITS = 4 * H, WORDS = (FM * BITS + 31) / 32;
    u32 keep[WORDS];
#pragma unroll
    for (int w = 0; w < WORDS; ++w) keep[w] = 0;
    if (o.drop) {
      const u32 off = o.d.off();
#pragma unroll 1
      for (int i = 0; i < FM; ++i) {
        u32 k = 0;
#pragma unroll
        for (int j = 0; j < H; ++j)
          k |= keep4_from(o.d, off, (i64)(mw + 16 * i) * o.N + nw + 16 * j +
                                        4 * q) << (4 * j);
#pragma unroll
        for (int w = 0; w < WORDS - 1; ++w)
          keep[w] = keep[w] >> BITS | keep[w + 1] << (32 - BITS);
        keep[WORDS - 1] = keep[WORDS - 1] >> BITS | k << (32 - BITS);
      }
    }
    float bias[2][H][4];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int j = 0; j < H; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          bias[h][j][r] = o.bias[h] ? to_f(o.bias[h][min(
              nw + 16 * j + 4 * q + r, o.N - 1)], T()) : 0.f;
#pragma unroll
    for (int i = 0; i < FM; ++i) {
      const int m = mw + 16 * i;
      if (m >= p.rows) continue;
#pragma unroll
      for (int j = 0; j < H; j += 2) {
        f32x8 g, u, d;
#pragma unroll
        for (int r = 0; r < 8; ++r) {
          g[r] = acc[i][j + r / 4][r % 4] + bias[0][j + r / 4][r % 4];
          u[r] = acc[i][j + H + r / 4][r % 4] + bias[1][j + r / 4][r % 4];
        }
        if (o.gu) {       // rows of ldg, a multiple of 8, hold all four
          float* gp = o.gu + (i64)m * o.ldg + nw + 16 * j + 4 * q;
          float* up = gp + (i64)o.M * o.ldg;
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            if (nw + 16 * (j + k) + 4 * q >= p.cols) continue;
            *reinterpret_cast<f32x4*>(gp + 16 * k) =
                f32x4{g[4 * k], g[4 * k + 1], g[4 * k + 2], g[4 * k + 3]};
            *reinterpret_cast<f32x4*>(up + 16 * k) =
                f32x4{u[4 * k], u[4 * k + 1], u[4 * k + 2], u[4 * k + 3]};
          }
        }
        u *= act8(o.act, g, d);
        if (o.drop) {
          constexpr int SKIP = 32 * WORDS - FM * BITS;
          const int at = SKIP + i * BITS + 4 * j;
          const u32 k = keep[at / 32] >> (at % 32);
#pragma unroll
          for (int r = 0; r < 8; ++r)
            u[r] = (k >> r & 1) ? u[r] * o.d.scale : 0.f;
        }
        s16x8 v = trade<T>(f32x4{u[0], u[1], u[2], u[3]},
                           f32x4{u[4], u[5], u[6], u[7]});
        const int n = nw + 16 * j + wide;
        if (n < p.cols) store8(o.h + (i64)m * o.N, n, o.N, v);
        __builtin_amdgcn_sched_barrier(0);    // keeps the registers at hand
      }
    }
  }
}

// ------------------------------------------------- joining a split product
// Sums the slabs in a fixed order (the same result every time; atomics would
// not give that). 256 x 4096 of a contraction in 2 parts: 17 MB read and 10
// written in 8.5 us, out of the caches that they were just written to. 8 columns a
// thread; WIDE, for few columns and many slabs: 8 threads, each an eighth of
// the slabs (one row of 25088 x 64 in 49 slabs: 21.5 -> 9.3 us
// with its product).
template <class T, bool WIDE>
__global__ __launch_bounds__(256) void join_gated_kernel(
    const float* __restrict__ slab, int splits, i64 slab_ld, OutArgs o) {
  const u32 off = o.drop ? o.d.off() : 0;
  const int per = int(slab_ld / 8);
  const i64 one = (i64)o.M * slab_ld, chunks = (i64)o.M * per;
  constexpr int LANES = WIDE ? 8 : 1;   // threads of a chunk, 8 lanes apart
  const int lane = threadIdx.x & 63, mine = WIDE ? lane >> 3 : 0;
  const i64 first = (i64)blockIdx.x * (blockDim.x / LANES) +
                    (WIDE ? (threadIdx.x >> 6) * 8 + (lane & 7)
                          : threadIdx.x);
  // whole waves stay together: the threads of a chunk exchange their sums
  for (i64 c = first; c - (WIDE ? lane & 7 : 0) < chunks;
       c += (i64)gridDim.x * (blockDim.x / LANES)) {
    const bool in = c < chunks;
    const float* sp = slab + (in ? c : 0) * 8 + mine * 2 * one;
    f32x8 g{}, u{};
#pragma unroll 4
    for (int s = mine; s < splits; s += LANES) {
      g += load8f(sp);
      u += load8f(sp + one);
      sp += 2 * LANES * one;
    }
    if (WIDE) {
#pragma unroll
      for (int d = 8; d < 64; d *= 2)
#pragma unroll
        for (int r = 0; r < 8; ++r) {
          g[r] += __shfl_xor(g[r], d);
          u[r] += __shfl_xor(u[r], d);
        }
    }
    if (!in || mine) continue;
    const int m = int(c / per), n = int(c - (i64)m * per) * 8;
    finish8<T>(o, off, m, n, g + bias8<T>(o.bias[0], n, o.N),
               u + bias8<T>(o.bias[1], n, o.N));
  }
}

template <class T>
__global__ __launch_bounds__(256) void join_plain_kernel(
    const float* __restrict__ slab, int splits, i64 slab_ld, int rows,
    int cols, int mats, u16* c0, u16* c1) {
  const int per = int(slab_ld / 8);
  const i64 one = (i64)rows * slab_ld * mats;
  for (i64 c = (i64)blockIdx.x * 256 + threadIdx.x;
       c < (i64)rows * mats * per; c += (i64)gridDim.x * 256) {
    const float* sp = slab + c * 8;
    f32x8 v{};
#pragma unroll 4
    for (int s = 0; s < splits; ++s, sp += one) v += load8f(sp);
    i64 m = c / per;
    int n = int(c - m * per) * 8;
    u16* out = m < rows ? c0 + m * cols : c1 + (m - rows) * cols;
    store8(out, n, cols, round8<T>(v));
  }
}

// ------------------------------------------------- few rows: the weights
// Up to 16 rows of X: the forward pass is one reading of both weights, and a
// tile's way through LDS only delays it. Here a wave takes 128 columns of
// each weight and a part of the contraction and loads 32 k of them straight
// into registers: lane (c, q) = (lane % 16, lane / 16) rows 8 q .. 8 q + 7 of
// columns 8 c .. 8 c + 7. Eight rows of eight columns are turned over by
// v_perm into eight fragments, one for each column j of the eight, of which
// lane (c, q) holds column 8 c + j and its 8 k: what the matrix instruction
// takes. The next 32 k are on their way meanwhile (16 KB a wave). The four
// waves of a block, each with its part of the contraction, meet in LDS; parts
// of several blocks meet in join_gated_kernel. (With the fragments of 32 or 64
// rows the tiles are faster: 64 x 25088 x 4096 in 91 us, this way in 112.)
// Memory bounds it: 16 x 25088 x 4096 takes 80 us, the 411 MB of its weights
// at 5.1 TB/s, a large copy's rate; through the tiles it took 104. One row of
// 4096 x 4096 takes 16 us for 67 MB, two launches and a ramp among them.
struct RowsArgs {
  const u16* x;
  const u16* w[2];
  i64 ldx, ldw;
  int M, K, N;
  int splits;
  float* slab;          // [splits][2][M][slab_ld] if splits > 1
  i64 slab_ld;
  OutArgs out;
};

typedef __attribute__((ext_vector_type(4))) u32 u32x4v;

DEV s16x8 pick_column(const u32x4v (&w)[8], int j) {
  u32x4v f;
#pragma unroll
  for (int t = 0; t < 4; ++t)
    f[t] = __builtin_amdgcn_perm(w[2 * t + 1][j / 2], w[2 * t][j / 2],
                                 j & 1 ? 0x07060302u : 0x05040100u);
  return __builtin_bit_cast(s16x8, f);
}
DEV f32x4 mfma_of(s16x8 a, s16x8 b, f32x4 c, __bf16) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(
      __builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0,
      0);
}
DEV f32x4 mfma_of(s16x8 a, s16x8 b, f32x4 c, _Float16) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(
      __builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// ANY: rows that start anywhere and end inside a vector, loaded as they lie. A
// lane's 8 columns then end at the last one at the latest: what two lanes
// hold twice comes out the same twice. 1 x 4097 x 4095 takes 21 us and 8 x
// 5336 x 3267 24 (15 and 22 at whole vectors); copied to whole vectors first,
// as the tiles need them, 42 and 47.
template <class T, bool ANY>
__global__ __launch_bounds__(256, 2) void rows_kernel(RowsArgs p) {
  __shared__ __attribute__((aligned(16))) float red[4][2][16][128];
  const int lane = threadIdx.x & 63, c = lane & 15, q = lane >> 4;
  const int wave = uniform(threadIdx.x >> 6);
  const int n0 = blockIdx.x * 128, split = blockIdx.y;

  // steps of 32 k: [first, last) of this wave
  const int steps = (p.K + 31) / 32, parts = p.splits * 4;
  const int part = split * 4 + wave;
  const int each_ = steps / parts, more = steps % parts;
  const int first = part * each_ + min(part, more);
  const int last = first + each_ + (part < more);

  const u32 ldw2 = u32(p.ldw) * 2;
  const bool col_in = n0 + c * 8 < p.N, row_in = c < p.M;
  u32 woff[8];
#pragma unroll
  for (int r = 0; r < 8; ++r)
    woff[r] = col_in ? (8 * q + r) * ldw2 + c * 16 : OUT_OF_RANGE;
  const u32 xoff = u32(c) * u32(p.ldx) * 2 + q * 16;

  u32x4v w[2][2][8];    // [buffer][weight][row]
  u32x4v xf[2];
  const int n_last = ANY ? p.N - 8 - n0 : 120;   // of the block's columns
  if (ANY) {
#pragma unroll
    for (int r = 0; r < 8; ++r)
      woff[r] = (8 * q + r) * ldw2 + (n0 + min(c * 8, n_last)) * 2;
  }
  auto fetch_any = [&](int b, int step) {
    const int k = step * 32, left = step < last ? p.K - k : 0;
    if (left <= 0) {
#pragma unroll
      for (int r = 0; r < 8; ++r) w[b][0][r] = w[b][1][r] = u32x4v{0, 0, 0, 0};
      xf[b] = u32x4v{0, 0, 0, 0};
      return;
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      auto base = reinterpret_cast<const char*>(p.w[h] + (i64)k * p.ldw);
      if (left >= 32) {
#pragma unroll
        for (int r = 0; r < 8; ++r)
          __builtin_memcpy(&w[b][h][r], base + woff[r], 16);
      } else {      // rows behind the contraction: the last one's place, zeros
#pragma unroll
        for (int r = 0; r < 8; ++r) {
          const int back = max(8 * q + r - (left - 1), 0);
          __builtin_memcpy(&w[b][h][r], base + (woff[r] - back * ldw2), 16);
          if (back) w[b][h][r] = u32x4v{0, 0, 0, 0};
        }
      }
    }
    xf[b] = __builtin_bit_cast(
        u32x4v, load8(p.x + (i64)min(c, p.M - 1) * p.ldx, k + 8 * q, p.K));
  };
  auto fetch = [&](int b, int step) {
    if constexpr (ANY) {
      fetch_any(b, step);
      return;
    }
    const int k = step * 32;
    // an empty buffer behind this wave's part: zeros, no memory moves
    const int rows = step < last ? min(p.K - k, 32) : 0;
    const u32 bytes = rows * ldw2 - min(rows, 1) * n0 * 2;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      auto rsrc = __builtin_amdgcn_make_buffer_rsrc(
          const_cast<u16*>(uniform(p.w[h] + (i64)k * p.ldw + n0)), 0,
          uniform(bytes), 0x00020000);
#pragma unroll
      for (int r = 0; r < 8; ++r)
        w[b][h][r] = __builtin_amdgcn_raw_buffer_load_b128(rsrc, woff[r], 0,
                                                           0);
    }
    const u32 xbytes = rows > 0 ? u32(p.M - 1) * u32(p.ldx) * 2 +
                                      ((rows + 7) & ~7) * 2 : 0;
    auto rx = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<u16*>(uniform(p.x + k)), 0, uniform(xbytes), 0x00020000);
    xf[b] = __builtin_amdgcn_raw_buffer_load_b128(
        rx, row_in && q * 8 < rows ? xoff : OUT_OF_RANGE, 0, 0);
  };
  f32x4 acc[2][8];
#pragma unroll
  for (int j = 0; j < 8; ++j) acc[0][j] = acc[1][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto multiply = [&](int b) {
    const s16x8 x = __builtin_bit_cast(s16x8, xf[b]);
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int j = 0; j < 8; ++j)
        acc[h][j] = mfma_of(pick_column(w[b][h], j), x, acc[h][j], T());
  };
  fetch(0, first);
  for (int step = first; step < last; step += 2) {
    fetch(1, step + 1);
    multiply(0);
    fetch(0, step + 2);
    multiply(1);
  }

  // lane: row c of X, columns 8 (4 q + r) + j
  if (row_in) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        f32x8 v;
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = acc[h][j][r];
        if (ANY) {
          const int at = min((4 * q + r) * 8, n_last);
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (at + j >= 0) red[wave][h][c][at + j] = v[j];
        } else {
          store8f(&red[wave][h][c][(4 * q + r) * 8], v);
        }
      }
  }
  __syncthreads();
  const u32 off = p.out.drop ? p.out.d.off() : 0;
  const int m = threadIdx.x / 16, k = threadIdx.x % 16 * 8, n = n0 + k;
  if (m >= p.M || n >= p.N) return;
  f32x8 g = load8f(&red[0][0][m][k]), u = load8f(&red[0][1][m][k]);
#pragma unroll
  for (int v = 1; v < 4; ++v) {
    g += load8f(&red[v][0][m][k]);
    u += load8f(&red[v][1][m][k]);
  }
  if (p.splits == 1) {
    finish8<T>(p.out, off, m, n, g + bias8<T>(p.out.bias[0], n, p.N),
               u + bias8<T>(p.out.bias[1], n, p.N));
  } else {
    float* sp = p.slab + ((i64)split * 2 * p.M + m) * p.slab_ld + n;
    store8f(sp, g);
    store8f(sp + (i64)p.M * p.slab_ld, u);
  }
}

// ------------------------------------------- between dH and the products
// dG and dU (rows of ldg, zeros behind N) and, where biases want them, their
// column sums: of each block's rows as part [gridDim.y][2][ldg], or, if one
// block takes all rows, the gradients themselves. A thread takes 8 columns, a
// block CB, its groups of CB / 8 threads every (2048 / CB)th row. CB = 64 for
// up to 64 rows: the sums then need no second kernel (64 x 4096: 6.3 us in
// place of 9.5; 256 x 4096: 14.3 and 9.5). Memory bounds it: 8192 x 8192
// without biases, 0.94 GB, in 200 us (4.7 TB/s; a large copy 5.1).
struct MidArgs {
  const u16* dh;
  i64 ldh;
  const float* gu;
  u16* dgu;
  float* part;
  u16* db[2];
  int M, N;
  i64 ldg;
  int rows_per_block;
  int act, drop;
  DropArgs d;
};

template <class T, int CB>
__global__ __launch_bounds__(256) void mid_kernel(MidArgs a) {
  constexpr int GROUPS = 2048 / CB;
  __shared__ float red[GROUPS][2][CB];
  const int tx = threadIdx.x % (CB / 8), ty = threadIdx.x / (CB / 8);
  const int n = blockIdx.x * CB + tx * 8;
  const u32 off = a.drop ? a.d.off() : 0;
  f32x8 sg{}, su{};
  const int r0 = blockIdx.y * a.rows_per_block;
  const int r1 = min(a.M, r0 + a.rows_per_block);
  const bool wide = (a.N & 7) == 0 && (a.ldh & 7) == 0 &&
                    (reinterpret_cast<uintptr_t>(a.dh) & 15) == 0;
  if (n < a.ldg) {
    for (int m = r0 + ty; m < r1; m += GROUPS) {
      const float* gp = a.gu + (i64)m * a.ldg + n;
      f32x8 g = load8f(gp), u = load8f(gp + (i64)a.M * a.ldg);
      const u16* hp = a.dh + (i64)m * a.ldh;
      s16x8 h = wide ? *reinterpret_cast<const s16x8*>(hp + n)
                     : load8(hp, n, a.N);
      u32 keep = 255u;
      if (a.drop) {
        i64 i = (i64)m * a.N + n;
        keep = keep8(a.d, off, i);
      }
      f32x8 d, act = act8(a.act, g, d), v = widen8<T>(h), dg, du;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (a.drop) v[j] *= a.d.scale;
        // what was dropped, or lies behind N, passes nothing on
        const bool in = (keep >> j & 1) && n + j < a.N;
        dg[j] = in ? v[j] * u[j] * d[j] : 0.f;
        du[j] = in ? v[j] * act[j] : 0.f;
      }
      sg += dg;
      su += du;
      s16x8 og = round8<T>(dg), ou = round8<T>(du);
      u16* op = a.dgu + (i64)m * a.ldg + n;
      *reinterpret_cast<s16x8*>(op) = og;
      *reinterpret_cast<s16x8*>(op + (i64)a.M * a.ldg) = ou;
    }
  }
  if (!a.part && !a.db[0] && !a.db[1]) return;
  store8f(&red[ty][0][tx * 8], sg);
  store8f(&red[ty][1][tx * 8], su);
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * CB; i += 256) {
    const int h = i / CB, c = blockIdx.x * CB + i % CB;
    float v = 0.f;
#pragma unroll
    for (int r = 0; r < GROUPS; ++r) v += red[r][h][i % CB];
    if (a.part) {
      if (c < a.ldg) a.part[((i64)blockIdx.y * 2 + h) * a.ldg + c] = v;
    } else if (c < a.N && a.db[h]) {
      a.db[h][c] = from_f(v, T());
    }
  }
}

// 32 columns a block, 32 groups of threads a part of the blocks' sums each:
// what bounds it is the latency of a thread's loads one after another (8071
// rows of 96, 1009 blocks: 6.0 us, with 8 groups 14.1; 256 rows of 4096, 32
// blocks: 3 either way).
template <class T>
__global__ __launch_bounds__(1024) void bias_join_kernel(
    const float* __restrict__ part, int blocks, int N, i64 ldg, u16* dbg,
    u16* dbu) {
  constexpr int GROUPS = 32;
  __shared__ float red[GROUPS][32];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + tx;
  u16* out = blockIdx.y ? dbu : dbg;
  if (!out) return;
  float v = 0.f;
  if (c < N) {
    part += blockIdx.y * ldg + c;
#pragma unroll 8
    for (int b = ty; b < blocks; b += GROUPS) v += part[(i64)b * 2 * ldg];
  }
  red[ty][tx] = v;
  __syncthreads();
  if (ty || c >= N) return;
#pragma unroll
  for (int r = 1; r < GROUPS; ++r) v += red[r][tx];
  out[c] = from_f(v, T());
}

// -------------------------------------------------------------- rows apart
// Copies rows of any length and alignment to rows of whole vectors, zeros
// behind them: what the tiles cannot load goes through here once a call, all
// operands in one launch.
struct PadArgs {
  const u16* in[3];
  u16* out[3];
  i64 sr[3], sc[3], rows[3];
  int cols[3], ld[3];
};
__global__ __launch_bounds__(256) void pad_rows_kernel(PadArgs a) {
  const int t = blockIdx.y;
  const int per = a.ld[t] / 8, cols = a.cols[t];
  const i64 sc = a.sc[t];
  for (i64 c = (i64)blockIdx.x * 256 + threadIdx.x; c < a.rows[t] * per;
       c += (i64)gridDim.x * 256) {
    const i64 r = c / per;
    const int n = int(c - r * per) * 8;
    const u16* in = a.in[t] + r * a.sr[t];
    s16x8 v;
    if (sc == 1) {
      v = load8(in, n, cols);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        v[j] = n + j < cols ? short(in[(n + j) * sc]) : short(0);
    }
    *reinterpret_cast<s16x8*>(a.out[t] + c * 8) = v;
  }
}

// ==================================================================== host
static i64 up(i64 v, i64 to) { return (v + to - 1) / to * to; }

static const u16* cptr(const at::Tensor& t) {
  return reinterpret_cast<const u16*>(t.data_ptr());
}
static u16* mptr(const at::Tensor& t) {
  return reinterpret_cast<u16*>(t.data_ptr());
}

// A matrix that the tiles can load: unit column stride, rows that start on
// 16 bytes and whose last vector may be read whole, and that lie close enough
// for 256 of them to be reached by 31 bits.
constexpr i64 LD_MAX = 1 << 21;
static bool loadable(const at::Tensor& t) {
  return t.stride(1) == 1 && t.size(1) % 8 == 0 &&
         (t.size(0) == 1 ||
          (t.stride(0) % 8 == 0 && t.stride(0) >= t.size(1) &&
           t.stride(0) <= LD_MAX)) &&
         reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
}
// Makes all of them loadable, copies of those that are not.
static void make_loadable(at::Tensor (&t)[3]) {
  PadArgs a{};
  i64 most = 0;
  int n = 0;
  for (auto& m : t) {
    if (loadable(m)) continue;
    auto out = at::empty({m.size(0), up(m.size(1), 8)}, m.options());
    a.in[n] = cptr(m);
    a.out[n] = mptr(out);
    a.sr[n] = m.stride(0);
    a.sc[n] = m.stride(1);
    a.rows[n] = m.size(0);
    a.cols[n] = int(m.size(1));
    a.ld[n] = int(out.size(1));
    most = std::max<i64>(most, out.numel() / 8);
    ++n;
    m = out;
  }
  if (!most) return;
  dim3 grid(u32(std::min<i64>((most + 255) / 256, 8192)), n);
  hipLaunchKernelGGL(pad_rows_kernel, grid, dim3(256), 0, cur_stream(), a);
  HIP_CHECK(hipGetLastError());
}
// a single row may carry any stride
static i64 ld_of(const at::Tensor& t) {
  return t.size(0) == 1 ? t.size(1) : t.stride(0);
}

constexpr int ROWS_MAX = 16, ROWS_TARGET = 256;

struct Plan { int fm, fn, bk, ring, splits, tiles_m, tiles_n; bool brief; };

// Which tile, and into how many parts the contraction is split: the least
// time by a model of what the tiles measured over the 138 products of 46
// shapes of 17 to 8192 rows and 64 to 25088 columns. It ranks them: what it
// picks there is 1.5 % slower than the best of all tiles and splits in the
// mean, 10 % at worst. Its times are off by 13 % in the mean, and low where
// the clock falls (forward at 8192 x 4096 x 8192: 714 us for 959) and at
// ragged widths, for which it has no term (1003 x 1001 x 2747: 18 for 30).
// Microseconds. A stage costs `one` if a tile has its CU to itself and `all`
// if the CU is full; `edge` is a tile's first loads and its epilogue.
// Four buffers are for launches of about one tile a CU: two leave such a tile
// waiting for memory at every stage (0.69 and 0.61 us in place of 0.52 and
// 0.38; 2048 x 4096 x 1000: 51.4 -> 39.2, 512 x 4096 x 4096: 54.3 -> 46.3).
// Two tiles on a CU cover for each other, and then two buffers each are the
// faster (797 x 5368 x 3032: 91 us, with four buffers 107).
static Plan make_plan(int mode, i64 rows, i64 cols, i64 k_len, int mats) {
  struct Kind {
    int fm, fn, bk, ring, per_cu;
    double one, all, edge;
    bool brief;
  };
  static const Kind kinds[] = {{8, 8, 64, 2, 1, 1.24, 1.24, 9.8, false},
                               {4, 4, 64, 2, 2, 0.69, 0.96, 3.9, false},
                               {4, 4, 64, 4, 1, 0.52, 0.52, 3.7, false},
                               {2, 4, 64, 2, 3, 0.61, 0.93, 2.8, false},
                               {2, 4, 64, 4, 1, 0.38, 0.38, 2.8, false},
                               {4, 4, 32, 2, 4, 0.69, 1.85, 4.0, false},
                               {4, 4, 64, 2, 4, 0.69, 1.85, 3.9, true}};
  constexpr double CUS = 256, MEM = 4.5e6, JOIN_MEM = 7e6;
  const double join = mode == FWD ? 4.0 : 2.4;
  const double out = double(rows) * cols;
  // bytes that the product moves at least
  const double ab = mode == FWD ? rows + 2. * cols
                  : mode == DGRAD ? 2. * rows + 2. * cols
                                  : rows + double(mats) * cols;
  const double mem = 2 * (ab * k_len + (mode == FWD ? 3 : mats) * out) / MEM;
  Plan best{};
  double least = 0;
  for (const Kind& k : kinds) {
    // Stages of 32 k pay where both operands lie along their rows and
    // contractions are short (256 x 9216 x 4096: 73.5 -> 60.3 us), and for dX
    // of up to 96 columns of G, which leave half of a wider turn empty (8072 x
    // 12800 x 96: 84.5 -> 67.7; at 128 columns 18.4 and 18.7); else their rows
    // of 64 bytes cost more than four tiles a CU gain.
    if (k.bk == 32 && mode != WGRAD && (mode != DGRAD || k_len > 96)) continue;
    if (k.brief && (mode != WGRAD || k_len > 64)) continue;
    const int tm = ceil_div(rows, 32 * k.fm);
    const int tn = ceil_div(cols, (mode == FWD ? 16 : 32) * k.fn) *
                   (mode == WGRAD ? mats : 1);
    // turns of the loop: a stage in each buffer (of 64 k: stages of 32 k come
    // two at a time), of DGRAD's two parts in turns
    const int turns = ceil_div(k_len, 64 * k.ring / (mode == DGRAD ? 2 : 1));
    // 1 2 3 4 6 8 12 16 24 32
    for (int sp = 1; sp <= turns && sp <= 32;
         sp += sp < 4 ? 1 : sp & (sp - 1) ? sp / 3 : sp / 2) {
      const double wgs = double(tm) * tn * sp, slots = CUS * k.per_cu;
      // a launch holds less than 2^32 threads; tiles of 256 x 128 and wider,
      // unsplit, stay below this for whatever fits in memory
      if (wgs > (1 << 23) && !(k.fm == 8 && sp == 1)) continue;
      const double depth = k.brief ? 1 : k.ring * ceil_div(turns, sp);
      auto round = [&](double n) {
        const double share = k.per_cu > 1
            ? (std::ceil(n / CUS) - 1) / (k.per_cu - 1) : 1;
        return n > 0 ? k.edge + depth * (k.one + (k.all - k.one) * share) : 0;
      };
      const double full = std::floor(wgs / slots);
      double t = full * round(slots) + round(wgs - full * slots);
      t = std::sqrt(std::sqrt(t * t * t * t + mem * mem * mem * mem));
      if (sp > 1) t += join + double(sp) * mats * out * 8 / JOIN_MEM;
      if (least == 0 || t < least) {
        least = t;
        best = Plan{k.fm, k.fn, k.bk, k.ring, sp, tm, tn, k.brief};
      }
    }
  }
  return best;
}

// What make_plan chooses, for tests that want every tile: fm, fn, bk, ring,
// brief, splits. product: 0 forward, 1 dX, 2 both weight gradients, 3 one.
std::vector<int64_t> gated_plan(int64_t product, int64_t rows, int64_t cols,
                                int64_t k_len) {
  TORCH_CHECK(product >= FWD && product <= WGRAD + 1 && rows > 0 && cols > 0 &&
              k_len > 0, "gated_plan: no such product");
  const Plan p = make_plan(int(std::min<int64_t>(product, WGRAD)), rows, cols,
                           k_len, product % 2 ? 1 : 2);
  return {p.fm, p.fn, p.bk, p.ring, p.brief, p.splits};
}

template <class T, int MODE>
static void launch(const Plan& pl, const ProductArgs& a) {
  dim3 grid(u32(pl.tiles_m) * pl.tiles_n * pl.splits);
  auto st = cur_stream();
  if (pl.brief) {
    hipLaunchKernelGGL((product_kernel<T, WGRAD, 4, 4, 64, 2, true>), grid,
                       dim3(256), 0, st, a);
    HIP_CHECK(hipGetLastError());
    return;
  }
#define TILE_CASE(FM, FN, BK, RING)                                        \
  if (pl.fm == FM && pl.fn == FN && pl.bk == BK && pl.ring == RING) {      \
    hipLaunchKernelGGL((product_kernel<T, MODE, FM, FN, BK, RING>), grid,  \
                       dim3(256), 0, st, a);                               \
    HIP_CHECK(hipGetLastError());                                          \
    return;                                                                \
  }
  TILE_CASE(8, 8, 64, 2)
  TILE_CASE(4, 4, 64, 2)
  TILE_CASE(4, 4, 64, 4)
  TILE_CASE(2, 4, 64, 2)
  TILE_CASE(2, 4, 64, 4)
  if constexpr (MODE != FWD) { TILE_CASE(4, 4, 32, 2) }
#undef TILE_CASE
  TORCH_CHECK(false, "gated_linear: no tile of this size");
}

template <class T>
static void join_gated_of(const float* slab, int splits, i64 slab_ld,
                          const OutArgs& out) {
  i64 chunks = (i64)out.M * slab_ld / 8;
  const bool wide = splits >= 8 && chunks < 8192;
  // few chunks: a wave a block, so that they reach more CUs
  const int threads = chunks < 65536 ? 64 : 256;
  const int per = wide ? threads / 8 : threads;
  dim3 grid(u32(std::min<i64>((chunks + per - 1) / per, 8192)));
  auto kernel = wide ? join_gated_kernel<T, true> : join_gated_kernel<T, false>;
  hipLaunchKernelGGL(kernel, grid, dim3(threads), 0, cur_stream(), slab,
                     splits, slab_ld, out);
  HIP_CHECK(hipGetLastError());
}
static void join_gated(bool half, const float* slab, int splits, i64 slab_ld,
                       const OutArgs& out) {
  if (half) join_gated_of<_Float16>(slab, splits, slab_ld, out);
  else join_gated_of<__bf16>(slab, splits, slab_ld, out);
}

template <int MODE>
static void product(at::ScalarType type, ProductArgs& a,
                    const at::TensorOptions& opt) {
  const Plan pl = make_plan(MODE, a.rows, a.cols, a.k_len, a.mats);
  a.splits = pl.splits;
  a.tiles_m = pl.tiles_m;
  a.tiles_n = pl.tiles_n;
  a.slab_ld = up(a.cols, 8);
  at::Tensor slab;
  if (pl.splits > 1) {
    slab = at::empty({(i64)pl.splits * a.mats * a.rows * a.slab_ld},
                     opt.dtype(at::kFloat));
    a.slab = slab.data_ptr<float>();
  }
  const bool half = type == at::kHalf;
  if (half) launch<_Float16, MODE>(pl, a);
  else launch<__bf16, MODE>(pl, a);
  if (pl.splits == 1) return;
  if (MODE == FWD) {
    join_gated(half, a.slab, pl.splits, a.slab_ld, a.out);
    return;
  }
  i64 chunks = (i64)a.rows * a.mats * a.slab_ld / 8;
  dim3 grid(u32(std::min<i64>((chunks + 255) / 256, 8192)));
  auto st = cur_stream();
  if (half) {
    hipLaunchKernelGGL(join_plain_kernel<_Float16>, grid, dim3(256), 0, st,
                       a.slab, pl.splits, a.slab_ld, a.rows, a.cols, a.mats,
                       a.c[0], a.c[1]);
  } else {
    hipLaunchKernelGGL(join_plain_kernel<__bf16>, grid, dim3(256), 0, st,
                       a.slab, pl.splits, a.slab_ld, a.rows, a.cols, a.mats,
                       a.c[0], a.c[1]);
  }
  HIP_CHECK(hipGetLastError());
}

// Few rows: about one block a CU (12 x 9216 x 4096: 37.0 us; 128 blocks 43.0,
// 512 38.7, 1024 46.3), and at least 2 steps of 32 k a wave. Letting the last
// block of a column join the parts in place of a second kernel took 23.8 us
// instead of 19.1 for one row of 4096 x 4096: what it waits for, the caches
// of eight XCDs written back, costs more than a launch.
static void product_rows(at::ScalarType type, const ProductArgs& a, bool any,
                         const at::TensorOptions& opt) {
  RowsArgs p{a.a[0], {a.b[0], a.b[1]}, a.lda, a.ldb, a.rows, a.k_len, a.cols,
             1, nullptr, up(a.cols, 8), a.out};
  const int blocks = ceil_div(a.cols, 128);
  p.splits = int(std::max<i64>(
      1, std::min<i64>(ROWS_TARGET / blocks, a.k_len / (32 * 4 * 2))));
  at::Tensor slab;
  if (p.splits > 1) {
    slab = at::empty({(i64)p.splits * 2 * a.rows * p.slab_ld},
                     opt.dtype(at::kFloat));
    p.slab = slab.data_ptr<float>();
  }
  const bool half = type == at::kHalf;
  auto st = cur_stream();
  dim3 grid(blocks, p.splits);
  auto kernel = half ? (any ? rows_kernel<_Float16, true>
                            : rows_kernel<_Float16, false>)
                     : (any ? rows_kernel<__bf16, true>
                            : rows_kernel<__bf16, false>);
  hipLaunchKernelGGL(kernel, grid, dim3(256), 0, st, p);
  HIP_CHECK(hipGetLastError());
  if (p.splits > 1) join_gated(half, p.slab, p.splits, p.slab_ld, a.out);
}

static void check_operand(const at::Tensor& t, const char* name,
                          const at::Tensor& x, i64 rows, i64 cols) {
  TORCH_CHECK(t.device() == x.device(), "gated_linear: ", name, " is on ",
              t.device(), ", x on ", x.device());
  TORCH_CHECK(t.scalar_type() == x.scalar_type(), "gated_linear: ", name,
              " is ", t.scalar_type(), ", x is ", x.scalar_type());
  bool shape = rows < 0 ? t.dim() == 1 && t.size(0) == cols
                        : t.dim() == 2 && t.size(0) == rows &&
                              t.size(1) == cols;
  TORCH_CHECK(shape, "gated_linear: ", name, " has shape ", t.sizes(),
              " instead of ",
              rows < 0 ? std::to_string(cols)
                       : std::to_string(rows) + " x " + std::to_string(cols));
}

static DropArgs gated_drop(const at::Tensor& x, double p, int64_t seed,
                           int64_t offset,
                           const c10::optional<at::Tensor>& offset_t) {
  if (offset_t)
    TORCH_CHECK(offset_t->device() == x.device() &&
                offset_t->scalar_type() == at::kLong &&
                offset_t->numel() == 1,
                "gated_linear: offset must be one int64 on x's device");
  return drop_args(p, seed, offset,
                   offset_t ? reinterpret_cast<const i64*>(
                                  offset_t->data_ptr<int64_t>())
                            : nullptr);
}

__global__ void copy_offset_kernel(const i64* in, i64* out) { *out = *in; }

// Returns h [M][N], and with `train` also what backward wants: G and U as
// one [2][M][N up to a vector] in 32 bits, the three operands as the tiles
// load them, and the offset that the mask was drawn with if it came from the
// device.
std::vector<at::Tensor> gated_fwd(
    const at::Tensor& x, const at::Tensor& wg, const at::Tensor& wu,
    const c10::optional<at::Tensor>& bg, const c10::optional<at::Tensor>& bu,
    int64_t act, double p, int64_t seed, int64_t offset,
    const c10::optional<at::Tensor>& offset_t, bool train) {
  TORCH_CHECK(x.is_cuda() && x.dim() == 2, "gated_linear: x must be a GPU "
              "matrix");
  auto type = x.scalar_type();
  TORCH_CHECK(type == at::kBFloat16 || type == at::kHalf,
              "gated_linear: x must be bf16 or fp16 on the GPU, got ", type);
  const i64 M = x.size(0), K = x.size(1);
  TORCH_CHECK(wg.dim() == 2, "gated_linear: w_gate must be a matrix");
  const i64 N = wg.size(1);
  check_operand(wg, "w_gate", x, K, N);
  check_operand(wu, "w_up", x, K, N);
  if (bg) check_operand(*bg, "bias_gate", x, -1, N);
  if (bu) check_operand(*bu, "bias_up", x, -1, N);
  TORCH_CHECK(K > 0 && N > 0, "gated_linear: K and N must not be 0");
  TORCH_CHECK(act >= 0 && act <= SIGMOID, "gated_linear: unknown activation");
  TORCH_CHECK(p >= 0.0 && p < 1.0, "gated_linear: p must lie in [0, 1)");
  TORCH_CHECK(M < (1 << 30) && K <= LD_MAX && N <= LD_MAX,
              "gated_linear: x must have less than 2^30 rows, x and the "
              "weights at most 2^21 columns");
  c10::DeviceGuard guard(x.device());
  DropArgs d = gated_drop(x, p, seed, offset, offset_t);
  auto h = at::empty({M, N}, x.options());
  at::Tensor gu, used;
  const i64 ldg = up(N, 8);
  if (train) gu = at::empty({2, M, ldg}, x.options().dtype(at::kFloat));
  if (train && offset_t) {
    used = at::empty({1}, offset_t->options());
    hipLaunchKernelGGL(copy_offset_kernel, dim3(1), dim3(1), 0, cur_stream(),
                       d.offset_ptr,
                       reinterpret_cast<i64*>(used.data_ptr<int64_t>()));
    HIP_CHECK(hipGetLastError());
  }
  at::Tensor ops_[3] = {x, wg, wu};
  at::Tensor &xl = ops_[0], &gl = ops_[1], &ul = ops_[2];
  // an answer of few rows takes rows that start anywhere
  const bool any =
      !train && M <= ROWS_MAX && N >= 8 &&
      !(loadable(x) && loadable(wg) && loadable(wu)) &&
      x.stride(1) == 1 && wg.stride(1) == 1 && wu.stride(1) == 1 &&
      ld_of(wg) == ld_of(wu) && ld_of(wg) <= LD_MAX;
  if (!any) make_loadable(ops_);
  if (ld_of(ul) != ld_of(gl)) {           // one pitch for both
    gl = gl.contiguous();
    ul = ul.contiguous();
  }
  at::Tensor bgc, buc;
  if (bg) bgc = bg->contiguous();
  if (bu) buc = bu->contiguous();
  if (M > 0) {
    ProductArgs a{};
    a.a[0] = a.a[1] = cptr(xl);
    a.b[0] = cptr(gl);
    a.b[1] = cptr(ul);
    a.lda = ld_of(xl);
    a.ldb = ld_of(gl);
    a.rows = int(M);
    a.cols = int(N);
    a.k_len = int(K);
    a.mats = 2;
    a.out = OutArgs{mptr(h), train ? gu.data_ptr<float>() : nullptr,
                    {bg ? cptr(bgc) : nullptr, bu ? cptr(buc) : nullptr},
                    int(M), int(N), ldg, int(act), p > 0.0, d};
    if (M <= ROWS_MAX) product_rows(type, a, any, x.options());
    else product<FWD>(type, a, x.options());
  }
  if (!train) return {h};
  std::vector<at::Tensor> r{h, gu, xl, gl, ul};
  if (used.defined()) r.push_back(used);
  return r;
}

// x, wg, wu as gated_fwd returned them; K, N: their true column counts.
// need: bits dx, dWg, dWu, dbg, dbu. *_out: where the caller wants them.
std::vector<at::Tensor> gated_bwd(
    const at::Tensor& dh_, const at::Tensor& gu, const at::Tensor& x,
    const at::Tensor& wg, const at::Tensor& wu, int64_t K, int64_t N,
    int64_t act, double p, int64_t seed, int64_t offset,
    const c10::optional<at::Tensor>& offset_t, int64_t need,
    const std::vector<c10::optional<at::Tensor>>& outs) {
  const i64 M = x.size(0), ldg = gu.size(2);
  auto type = x.scalar_type();
  TORCH_CHECK(dh_.device() == x.device() && dh_.scalar_type() == type &&
              dh_.dim() == 2 && dh_.size(0) == M && dh_.size(1) == N,
              "gated_linear: bad gradient");
  c10::DeviceGuard guard(x.device());
  auto opt = x.options();
  auto dh = dh_.stride(1) == 1 ? dh_ : dh_.contiguous();
  DropArgs d = gated_drop(x, p, seed, offset, offset_t);
  const i64 shapes[5][2] = {{M, K}, {K, N}, {K, N}, {1, N}, {1, N}};
  std::vector<at::Tensor> grads(5), result(5);
  for (int i = 0; i < 5; ++i) {
    if (!(need >> i & 1)) continue;
    auto& out = outs[i];
    if (out)
      TORCH_CHECK(out->is_contiguous() && out->device() == x.device() &&
                  out->numel() == shapes[i][0] * shapes[i][1] &&
                  out->const_data_ptr(),
                  "gated_linear: bad gradient buffer");
    // a buffer of another type, or one that vectors do not fit, is filled by
    // a copy at the end
    bool direct = out && out->scalar_type() == type &&
                  reinterpret_cast<uintptr_t>(out->data_ptr()) % 16 == 0;
    grads[i] = direct ? *out
                      : at::empty({shapes[i][0], shapes[i][1]}, opt);
    result[i] = out ? *out : i < 3 ? grads[i] : grads[i].view({N});
  }
  for (int i = 1; i < 5; i += 2)
    TORCH_CHECK(!result[i].defined() || !result[i + 1].defined() ||
                !outs[i] || !outs[i + 1] ||
                outs[i]->data_ptr() != outs[i + 1]->data_ptr(),
                "gated_linear: gate and up share one gradient buffer");
  auto ptr = [&](int i) {
    return grads[i].defined() ? mptr(grads[i]) : nullptr;
  };
  if (M == 0) {
    for (auto& g : grads) if (g.defined()) g.zero_();
  } else {
    auto dgu = at::empty({2, M, ldg}, opt);
    const bool bias = (need & 24) != 0;
    MidArgs a{};
    a.dh = cptr(dh);
    a.ldh = M == 1 ? N : dh.stride(0);
    a.gu = gu.data_ptr<float>();
    a.dgu = mptr(dgu);
    a.M = int(M);
    a.N = int(N);
    a.ldg = ldg;
    a.act = int(act);
    a.drop = p > 0.0;
    a.d = d;
    const bool half = type == at::kHalf, one = M <= 64;
    const int bx = ceil_div(ldg, one ? 64 : 256);
    // about 2048 blocks; 8 rows a turn
    a.rows_per_block =
        one ? int(M) : int(std::max<i64>(8, up(ceil_div(M * bx, 2048), 8)));
    const int by = ceil_div(M, a.rows_per_block);
    TORCH_CHECK(by < 65536, "gated_linear: too many rows");
    at::Tensor part;
    if (bias && one) {
      a.db[0] = ptr(3);
      a.db[1] = ptr(4);
    } else if (bias) {
      part = at::empty({by, 2, ldg}, opt.dtype(at::kFloat));
      a.part = part.data_ptr<float>();
    }
    auto st = cur_stream();
    auto mid = one ? (half ? mid_kernel<_Float16, 64> : mid_kernel<__bf16, 64>)
                   : (half ? mid_kernel<_Float16, 256>
                           : mid_kernel<__bf16, 256>);
    hipLaunchKernelGGL(mid, dim3(bx, by), dim3(256), 0, st, a);
    if (a.part) {
      auto join = half ? bias_join_kernel<_Float16> : bias_join_kernel<__bf16>;
      hipLaunchKernelGGL(join, dim3(ceil_div(N, 32), 2), dim3(1024), 0, st,
                         a.part, by, int(N), ldg, ptr(3), ptr(4));
    }
    HIP_CHECK(hipGetLastError());
    const u16* dg = cptr(dgu);
    const u16* du = dg + M * ldg;
    if (need & 1) {
      ProductArgs q{};
      q.a[0] = dg;
      q.a[1] = du;
      q.b[0] = cptr(wg);
      q.b[1] = cptr(wu);
      q.lda = ldg;
      q.ldb = ld_of(wg);
      q.rows = int(M);
      q.cols = int(K);
      q.k_len = int(N);
      q.mats = 1;
      q.c[0] = ptr(0);
      product<DGRAD>(type, q, opt);
    }
    if (need & 6) {
      const bool gate = need & 2, both = (need & 6) == 6;
      ProductArgs q{};
      q.a[0] = q.a[1] = cptr(x);
      q.b[0] = gate ? dg : du;
      q.b[1] = both ? du : nullptr;
      q.lda = ld_of(x);
      q.ldb = ldg;
      q.rows = int(K);
      q.cols = int(N);
      q.k_len = int(M);
      q.mats = both ? 2 : 1;
      q.c[0] = ptr(gate ? 1 : 2);
      q.c[1] = both ? ptr(2) : nullptr;
      product<WGRAD>(type, q, opt);
    }
  }
  for (int i = 0; i < 5; ++i)
    if (result[i].defined() && result[i].data_ptr() != grads[i].data_ptr())
      result[i].view(-1).copy_(grads[i].view(-1));
  return result;
}

}  // namespace dvgg
