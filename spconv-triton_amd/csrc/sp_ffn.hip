// Gated feed-forward block on feature rows, forward and backward, on 32x32 MFMA
// tiles with fp32 accumulation:
//
//   g = x Wg', u = x Wu', h = act(g) * u, y = h Wd' (+ residual)
//   dh = dy Wd, dg = dh * u * act'(g), du = dh * act(g)
//   dx = dg Wg + du Wu, dWg = dg' x, dWu = du' x, dWd = dy' h
//
// Both projections share the tiles of x and end in one epilogue, so that g and u
// never leave the registers.  The backward pass forms g, u and dh again in one
// kernel whose epilogue writes h, dg and du; nothing of the hidden width is kept
// between the passes.  In 16-bit calls h, dg and du are rounded to the rows' type, for they
// are operands of the products that follow, as they are where each step is a call of its
// own; g, u, dh, the gate and every sum stay in fp32.
//
// This file has the kernels for rows of any type and width, a tile of the product a workgroup,
// and the choice between them and the one-kernel passes of narrow 16-bit rows
// (sp_ffn_fused.hip, sp_ffn_grad.hip).
#include "sp_tiles.h"

namespace sp {

// h = act(x Wg') * (x Wu'), rows of Fp values, of which those from F on stand for nothing: who reads h
// stops at F.  50k x 512 -> 1 376 bf16 194 us (725 TFLOP/s), 75k x 256 -> 688 111.
template <typename T, typename S, bool ASYNC>
__global__ __launch_bounds__(S::THREADS, 2) void ffn_up(Rows<T> x, Rows<T> wg, Rows<T> wu, int act,
                                                     T* __restrict__ h, int Fp) {
  __shared__ __attribute__((aligned(16))) char lds[2 * S::BYTES];
  constexpr int NH = S::WT / 2, HIDDEN = S::W / 2;  // a wave's tiles of each, the workgroup's units
  const int wave = int(threadIdx.x) >> 6, wm = wave / S::WW, wn = wave % S::WW;
  const int lane = int(threadIdx.x) & 31;
  const int cols = (Fp + HIDDEN - 1) / HIDDEN;
  const int64_t place = place_of((x.n + S::X - 1) / S::X * cols);
  if (place < 0) return;
  const int64_t x0 = place / cols * S::X;
  const int f0 = int(place % cols) * HIDDEN, xrow = wm * 32 * S::XT;
  floatx16 acc[S::XT][S::WT];
  clear(acc);
  int wrow[S::WT];
#pragma unroll
  for (int i = 0; i < NH; ++i) {
    wrow[i] = (wn * NH + i) * 32;
    wrow[NH + i] = HIDDEN + (wn * NH + i) * 32;
  }
  products<T, S, ASYNC, S::WT>(x, x0, wg, &wu, f0, wrow, xrow, lds, acc);
  with_act(act, [&](auto kind) {
#pragma unroll
    for (int j = 0; j < S::XT; ++j)
#pragma unroll
      for (int i = 0; i < NH; ++i) {
        const floatx16 z = acc[j][i];
        gate16<sizeof(T) == 2, kind.value>(
            z, [&](int k, float value, float) { acc[j][i][k] = value * acc[j][NH + i][k]; });
        write_piece_row<T>(h, Fp, x0 + xrow + 32 * j + lane, x.n, f0 + wrow[i], Fp, true,
                           [&](int k, int) { return acc[j][i][k]; });
      }
  });
}

// dg, du and h in rows of 3 Fp values, zeros from F to Fp.  wdt: Wd transposed.  The operands of dh take a
// second pass over the same stages, so that the three accumulators of a unit meet in one epilogue: 16-bit
// writes of three arrays (413 MB for 50k rows and 1 376 units: 84 us of 413 at a copy's rate), which
// only another workgroup on the CU hides.  Those 413 us are 510 TFLOP/s bf16; fp32, 30k rows
// of 96 -> 256, takes 68 (65 TFLOP/s, the matrix cores give 154).
template <typename T, typename S, bool ASYNC>
__global__ __launch_bounds__(S::THREADS, 2) void ffn_grad_hidden(Rows<T> x, Rows<T> wg, Rows<T> wu,
                                                              Rows<T> dy, Rows<T> wdt, int act,
                                                              T* __restrict__ out, int Fp) {
  __shared__ __attribute__((aligned(16))) char lds[2 * S::BYTES];
  constexpr int NH = S::WT / 2, HIDDEN = S::W / 2;
  const int wave = int(threadIdx.x) >> 6, wm = wave / S::WW, wn = wave % S::WW;
  const int lane = int(threadIdx.x) & 31;
  const int cols = (Fp + HIDDEN - 1) / HIDDEN;
  const int64_t place = place_of((x.n + S::X - 1) / S::X * cols);
  if (place < 0) return;
  const int64_t x0 = place / cols * S::X;
  const int f0 = int(place % cols) * HIDDEN, xrow = wm * 32 * S::XT;
  const int F = int(wg.n);
  floatx16 acc[S::XT][S::WT], dh[S::XT][NH];
  clear(acc);
  clear(dh);
  int wrow[S::WT], drow[NH];
#pragma unroll
  for (int i = 0; i < NH; ++i) {
    drow[i] = wrow[i] = (wn * NH + i) * 32;
    wrow[NH + i] = HIDDEN + wrow[i];
  }
  products<T, S, ASYNC, S::WT>(x, x0, wg, &wu, f0, wrow, xrow, lds, acc);
  if (wdt.n > f0 + HIDDEN) wdt.n = f0 + HIDDEN;  // (half of a stage's weight rows)
  products<T, S, ASYNC, NH>(dy, x0, wdt, nullptr, f0, drow, xrow, lds, dh);
  if (F < Fp && f0 + HIDDEN > F) {  // (else infinities of unit F - 1 would meet the zeros of Wg and Wu)
#pragma unroll
    for (int j = 0; j < S::XT; ++j)
#pragma unroll
      for (int n = 0; n < NH; ++n)
        each_column<T>(f0 + drow[n], [&](int i, int c) {
          if (c >= F) acc[j][n][i] = acc[j][NH + n][i] = dh[j][n][i] = 0.f;
        });
  }
  with_act(act, [&](auto kind) {
#pragma unroll
    for (int j = 0; j < S::XT; ++j)
#pragma unroll
      for (int n = 0; n < NH; ++n) {
        const floatx16 z = acc[j][n];
        gate16<sizeof(T) == 2, kind.value>(z, [&](int i, float value, float slope) {
          const float u = acc[j][NH + n][i], d = dh[j][n][i];
          acc[j][n][i] = d * u * slope;
          acc[j][NH + n][i] = d * value;
          dh[j][n][i] = value * u;
        });
      }
  });
#pragma unroll
  for (int j = 0; j < S::XT; ++j)
#pragma unroll
    for (int n = 0; n < NH; ++n) {
      const int64_t r = x0 + xrow + 32 * j + lane, ld = 3 * int64_t(Fp);
      const int f = f0 + drow[n];
      write_piece_row<T>(out, ld, r, x.n, f, Fp, true, [&](int k, int) { return acc[j][n][k]; });
      write_piece_row<T>(out + Fp, ld, r, x.n, f, Fp, true,
                         [&](int k, int) { return acc[j][NH + n][k]; });
      write_piece_row<T>(out + 2 * Fp, ld, r, x.n, f, Fp, true,
                         [&](int k, int) { return dh[j][n][k]; });
    }
}

// out = a w' (+ residual, added in fp32).  50k x 1 376 -> 512 bf16 109 us and x 2 752 -> 512 190 (645 and 740
// TFLOP/s; 392 tiles are 1.5 rounds of workgroups); fp32 30k x 256 -> 96 21 us and x 512 -> 96 35 (71 and
// 83, of 154: one tile a CU, whose waves take loads and products in turn).  The residual is read value by value
// in the epilogue: 40 us more at 75k x 688 -> 256, 60 at 50k x 1 376 -> 512, for 8 and 10 of its bytes' own.
// Rows of w whose width V does not divide go through registers value by value: 75k x 256 -> 682 291 us in all
// for 120 at 688, 50k x 512 -> 1 365 727 for 259 at 1 360.
template <typename T>
struct RowsOut {
  const T* residual;
  int64_t ldr;
  T* out;
  int n, vec;
};

template <typename T, typename S, bool ASYNC>
__device__ __forceinline__ void rows_tile(const Rows<T>& a, const Rows<T>& w, const RowsOut<T>& o,
                                          int64_t x0, int n0, char* lds) {
  const int wave = int(threadIdx.x) >> 6, wm = wave / S::WW, wn = wave % S::WW;
  const int lane = int(threadIdx.x) & 31, xrow = wm * 32 * S::XT;
  floatx16 acc[S::XT][S::WT];
  clear(acc);
  int wrow[S::WT];
#pragma unroll
  for (int i = 0; i < S::WT; ++i) wrow[i] = (wn * S::WT + i) * 32;
  products<T, S, ASYNC, S::WT>(a, x0, w, nullptr, n0, wrow, xrow, lds, acc);
#pragma unroll
  for (int j = 0; j < S::XT; ++j)
#pragma unroll
    for (int i = 0; i < S::WT; ++i) {
      const int64_t r = x0 + xrow + 32 * j + lane;
      write_piece_row<T>(o.out, o.n, r, a.n, n0 + wrow[i], o.n, o.vec, [&](int k, int c) {
        return o.residual && c < o.n ? acc[j][i][k] + to_f32(o.residual[r * o.ldr + c])
                                     : acc[j][i][k];
      });
    }
}

template <typename T, typename S, bool ASYNC>
__global__ __launch_bounds__(S::THREADS, 2) void ffn_rows(Rows<T> a, Rows<T> w, RowsOut<T> o) {
  __shared__ __attribute__((aligned(16))) char lds[2 * S::BYTES];
  const int cols = (o.n + S::W - 1) / S::W;
  const int64_t place = place_of((a.n + S::X - 1) / S::X * cols);
  if (place < 0) return;
  rows_tile<T, S, ASYNC>(a, w, o, place / cols * S::X, int(place % cols) * S::W, lds);
}

// The same with `whole` large tiles (a multiple of 256: full rounds of the CUs) and each of the others as
// four of a quarter its size.
template <typename T>
__global__ __launch_bounds__(LargeTile::THREADS, 2) void ffn_rows_split(Rows<T> a, Rows<T> w,
                                                                        RowsOut<T> o, int whole) {
  static_assert(QuickTile::THREADS == LargeTile::THREADS && 2 * QuickTile::X == LargeTile::X &&
                    2 * QuickTile::W == LargeTile::W, "quarters");
  __shared__ __attribute__((aligned(16))) char lds[2 * LargeTile::BYTES];
  const int cols = (o.n + LargeTile::W - 1) / LargeTile::W;
  const int64_t tiles = (a.n + LargeTile::X - 1) / LargeTile::X * cols;
  if (int(blockIdx.x) < whole) {
    const int64_t place = place_of(whole);
    rows_tile<T, LargeTile, true>(a, w, o, place / cols * LargeTile::X,
                                  int(place % cols) * LargeTile::W, lds);
    return;
  }
  const int64_t place = place_of(4 * (tiles - whole), int64_t(blockIdx.x) - whole);
  if (place < 0) return;
  const int64_t tile = whole + place / 4;
  const int64_t x0 = tile / cols * LargeTile::X + (place >> 1 & 1) * QuickTile::X;
  const int n0 = int(tile % cols) * LargeTile::W + int(place & 1) * QuickTile::W;
  if (x0 < a.n && n0 < o.n) rows_tile<T, QuickTile, true>(a, w, o, x0, n0, lds);
}

// dst [cols][ldd] = src [rows][cols] transposed, zeros from rows to rows_out.
template <typename T>
struct Transpose {
  const T* src;
  T* dst;
  int rows, cols, rows_out;
  int64_t ldd;
};

// Three matrices in one launch (a launch costs the host as much as the transposition takes).
template <typename T>
__global__ __launch_bounds__(kFfnThreads) void ffn_transpose(Transpose<T> m0, Transpose<T> m1,
                                                             Transpose<T> m2) {
  __shared__ T tile[32][33];
  const Transpose<T> m = blockIdx.z == 0 ? m0 : blockIdx.z == 1 ? m1 : m2;
  const int r0 = int(blockIdx.x) * 32, c0 = int(blockIdx.y) * 32;
  if (r0 >= m.rows_out || c0 >= m.cols) return;
  const int tx = int(threadIdx.x) & 31, ty = int(threadIdx.x) >> 5;
#pragma unroll
  for (int j = 0; j < 32; j += 8) {
    const int r = r0 + ty + j, c = c0 + tx;
    tile[ty + j][tx] = r < m.rows && c < m.cols ? m.src[int64_t(r) * m.cols + c] : T(0.f);
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < 32; j += 8) {
    const int c = c0 + ty + j, r = r0 + tx;
    if (c < m.cols && r < m.rows_out) m.dst[int64_t(c) * m.ldd + r] = tile[tx][ty + j];
  }
}

// ---- weight gradients ------------------------------------------------------------
// Partials of a' b over a share of the rows: a [rows, P] is of the hidden width, b [rows, Q] of x's
// or dy's, TP x TQ of the result a workgroup.  Rows are the MFMA's reduction: 64 of them
// (fp32: 32) a stage lie in LDS as in memory, 16-bit operands come out of it
// transposed (ds_read_b64_tr_b16: sixteen lanes take a 4 x 16 block and get a column of it each),
// fp32 ones value by value.
template <typename T>
struct Gram {
  const T *a, *b;
  int64_t lda, ldb;
  int P, Q;
  int tiles_q, tiles;  // tiles along Q, and all
  int vec_a, vec_b;
  float* part;  // [shares][P][Q]
};

// Waves of TP / 64 x 2, each with 64 x TQ / 2 of the tile, or where TQ is 96 of 32 x 96.  The partials of
// a share of the rows are fp32 and joined in a fixed order, so that two calls give the same gradients.
// 50k rows, 512 channels, 1 376 units bf16: 317 us, 667 TFLOP/s, bound as the products above, and by the
// transposed reads, two for each operand; 75k rows, 256, 688: 130.  fp32, 30k rows, 96, 256: 57 (78
// TFLOP/s; 66 us with 128 columns, a quarter of them empty).
template <typename T, int TP, int TQ>
__global__ __launch_bounds__(2 * TP, 2) void ffn_gram(Gram<T> g0, Gram<T> g1, int64_t rows,
                                                      int64_t share, int shares) {
  constexpr int THREADS = 2 * TP, ROWS = gram_rows<T>();
  constexpr int NP = TQ == 96 ? 1 : 2, NQ = TQ == 96 ? 3 : TQ / 64;
  constexpr int STAGE = kGramStage * (TP + TQ);
  using SA = GramStage<T, TP, THREADS>;
  using SB = GramStage<T, TQ, THREADS>;
  __shared__ __attribute__((aligned(16))) char lds[2 * STAGE];
  const int tiles = g0.tiles + g1.tiles;
  const int64_t place = place_of(int64_t(tiles) * shares);
  if (place < 0) return;
  const int64_t lo = place / tiles * share;
  int tile = int(place % tiles);
  const bool second = tile >= g0.tiles;
  if (second) tile -= g0.tiles;
  const Gram<T> g = second ? g1 : g0;
  const int p0 = tile / g.tiles_q * TP, q0 = tile % g.tiles_q * TQ;
  const int64_t hi = lo + share < rows ? lo + share : rows;
  const int wave = int(threadIdx.x) >> 6, wp = TQ == 96 ? wave * 32 : (wave >> 1) * 64;
  const int wq = TQ == 96 ? 0 : (wave & 1) * (TQ / 2);
  floatx16 acc[NP][NQ];
  clear(acc);
  SA sa;
  SB sb;
  auto fetch = [&](int64_t m) {
    sa.load(g.a, g.lda, g.vec_a, m, hi, p0, g.P);
    sb.load(g.b, g.ldb, g.vec_b, m, hi, q0, g.Q);
  };
  fetch(lo);
  int s = 0;
  for (int64_t m = lo; m < hi; m += ROWS, s ^= 1) {
    char* la = lds + s * STAGE;
    char* lb = la + kGramStage * TP;
    sa.store(la, hi - m);
    sb.store(lb, hi - m);
    __syncthreads();  // (the other buffer's readers are past their previous barrier)
    if (m + ROWS < hi) fetch(m + ROWS);
    auto read = [&](int k) {
      Operands<T, NP, NQ> f;
#pragma unroll
      for (int i = 0; i < NP; ++i) f.x[i] = SA::read(la, k * 2 * Mfma<T>::V, wp + 32 * i);
#pragma unroll
      for (int i = 0; i < NQ; ++i) f.w[i] = SB::read(lb, k * 2 * Mfma<T>::V, wq + 32 * i);
      return f;
    };
    Batched<Operands<T, NP, NQ>, ROWS / (2 * Mfma<T>::V), 1> steps;
    steps.start(read);
    steps.run(read, [&](int, const Operands<T, NP, NQ>& f) {
#pragma unroll
      for (int i = 0; i < NP; ++i)
#pragma unroll
        for (int j = 0; j < NQ; ++j) Mfma<T>::mma(f.x[i], f.w[j], acc[i][j]);
    });
  }
  float* part = g.part + lo / share * g.P * g.Q;
  const int lane = int(threadIdx.x) & 31, half = (int(threadIdx.x) >> 5) & 1;
#pragma unroll
  for (int i = 0; i < NP; ++i)
#pragma unroll
    for (int j = 0; j < NQ; ++j)
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        const int p = p0 + wp + 32 * i + (k & 3) + 8 * (k >> 2) + 4 * half;
        const int q = q0 + wq + 32 * j + lane;
        if (p < g.P && q < g.Q) part[int64_t(p) * g.Q + q] = acc[i][j][k];
      }
}

// The three weight gradients from their partials: dWg and dWu [F][C] from rows 0 and Fp on of the
// first product, dWd [Co][F] from the second, [F][Co].  64 V values a workgroup, four runs of the shares
// summed apart and then in order.  Bound by the partials' reads, which come from the cache behind the L2s: 59 MB
// each for 75k x 256 -> 688 (28 shares) 13.3 us, value by value 16.5, and for 50k x 512 -> 1 376 (7 shares) 15.5
// and 24.5; 240k x 64 -> 256 (125 shares, 25 MB) 7.2 and 6.5.
template <typename T, int V>
__global__ __launch_bounds__(kFfnThreads) void ffn_reduce(const float* __restrict__ part0,
                                                          const float* __restrict__ part1,
                                                          int shares, int C, int F, int Fp, int Co,
                                                          T* __restrict__ dwg, T* __restrict__ dwu,
                                                          T* __restrict__ dwd) {
  typedef float vec __attribute__((ext_vector_type(V)));
  __shared__ vec lds[4][64];
  const int lane = int(threadIdx.x) & 63, run = int(threadIdx.x) >> 6;
  const int64_t i = (int64_t(blockIdx.x) * 64 + lane) * V;
  const int64_t n0 = int64_t(F) * C, n1 = int64_t(F) * Co;
  const int which = int(blockIdx.y);
  T* dst = which == 0 ? dwg : which == 1 ? dwu : dwd;
  if (!dst) return;
  const bool in = i < (which == 2 ? n1 : n0);
  const float* p = which == 2 ? part1 + i : part0 + (which ? int64_t(Fp) * C : 0) + i;
  const int64_t stride = which == 2 ? n1 : 2 * int64_t(Fp) * C;
  vec v = vec(0.f);
  if (in) {
    const int per = (shares + 3) / 4, end = (run + 1) * per < shares ? (run + 1) * per : shares;
#pragma unroll 8
    for (int s = run * per; s < end; ++s) v += *reinterpret_cast<const vec*>(p + int64_t(s) * stride);
  }
  lds[run][lane] = v;
  __syncthreads();
  if (run != 0 || !in) return;
  v = ((lds[0][lane] + lds[1][lane]) + lds[2][lane]) + lds[3][lane];
  const int64_t f = i / Co;  // (a piece lies in one row of Wd')
#pragma unroll
  for (int k = 0; k < V; ++k)
    dst[which == 2 ? (i + k - f * Co) * F + f : i + k] = from_f32<T>(v[k]);
}

// ---- a few rows ------------------------------------------------------------------
// For up to four rows the weights are read once and nothing else counts: a group of lanes takes an
// output, each lane pieces of its weight row against the same pieces of every row, and h stays
// fp32.  One row of 512 -> 1376 bf16 8.7 us (tiles 22.3), of 64 -> 172 fp16 6.5 (one kernel 9.7); four rows
// 19 and 10, eight 34 and 16.


template <typename T, int R>
__global__ __launch_bounds__(kFfnThreads) void ffn_few_up(Rows<T> x, Rows<T> wg, Rows<T> wu,
                                                          int act, int log_lanes,
                                                          float* __restrict__ h) {
  constexpr int V = Mfma<T>::V;
  const int lanes = 1 << log_lanes, lane = int(threadIdx.x) & (lanes - 1);
  const int64_t f = int64_t(blockIdx.x) * (kFfnThreads >> log_lanes) + (int(threadIdx.x) >> log_lanes);
  float a[2 * R];
#pragma unroll
  for (int i = 0; i < 2 * R; ++i) a[i] = 0.f;
  if (f < wg.n)
    for (int k = lane * V; k < x.K; k += lanes * V) {
      const auto g = piece_of(wg, f, k), u = piece_of(wu, f, k);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const auto v = piece_of(x, r < x.n ? r : x.n - 1, k);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          a[r] = __builtin_fmaf(to_f32(v[i]), to_f32(g[i]), a[r]);
          a[R + r] = __builtin_fmaf(to_f32(v[i]), to_f32(u[i]), a[R + r]);
        }
      }
    }
  sum_lanes(a, lanes);
  if (f >= wg.n || lane != 0) return;
  with_act(act, [&](auto kind) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float value, slope;
      gate<false, kind.value>(a[r], value, slope);
      if (r < x.n) h[r * wg.n + f] = value * a[R + r];
    }
  });
}

template <typename T, int R>
__global__ __launch_bounds__(kFfnThreads) void ffn_few_down(const float* __restrict__ h, int rows,
                                                            Rows<T> wd,
                                                            const T* __restrict__ residual,
                                                            int64_t ldr, int log_lanes,
                                                            T* __restrict__ y) {
  constexpr int V = Mfma<T>::V;
  const int lanes = 1 << log_lanes, lane = int(threadIdx.x) & (lanes - 1);
  const int64_t c = int64_t(blockIdx.x) * (kFfnThreads >> log_lanes) + (int(threadIdx.x) >> log_lanes);
  float a[R];
#pragma unroll
  for (int i = 0; i < R; ++i) a[i] = 0.f;
  if (c < wd.n)
    for (int k = lane * V; k < wd.K; k += lanes * V) {
      const auto w = piece_of(wd, c, k);
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int i = 0; i < V; ++i)
          if (k + i < wd.K)
            a[r] = __builtin_fmaf(h[int64_t(r < rows ? r : rows - 1) * wd.K + k + i], to_f32(w[i]),
                                  a[r]);
    }
  sum_lanes(a, lanes);
  if (c >= wd.n || lane != 0) return;
#pragma unroll
  for (int r = 0; r < R; ++r)
    if (r < rows) {
      const float v = residual ? a[r] + to_f32(residual[r * ldr + c]) : a[r];
      y[r * wd.n + c] = from_f32<T>(v);
    }
}

// ---- host ------------------------------------------------------------------------
// Tiles of the weight gradients: 128 x 64, 96 or 128, the fewest columns that both widths fit in, and for wider
// rows 256 x 256, with which the L2 hands out half as much (50k rows of 512 channels, 1 376
// hidden units: 1.7 GB for 3.3).
struct GramShape {
  int p, q;
};
static GramShape gram_shape(int64_t C, int64_t Co) {
  const int64_t n = C > Co ? C : Co;
  if (n <= 64) return {128, 64};
  if (n <= 96) return {128, 96};
  if (n <= 128) return {128, 128};
  return {256, 256};
}

static int64_t gram_tiles(int64_t P, int64_t Q, GramShape t) { return cdiv(P, t.p) * cdiv(Q, t.q); }

// Shares of the rows in the weight gradients: two workgroups of 128 hidden units a CU or one of
// 256, none of which waits for a second round, each with at least 256 rows.
static int64_t gram_shares(int64_t rows, int64_t tiles, GramShape t) {
  const int64_t want = (t.p == 256 ? 256 : 512) / tiles, most = cdiv(rows, 256);
  return want < 1 ? 1 : want < most ? want : most;
}

// The backward pass's workspace, and which kernels it takes: for 16-bit rows of up to 128 channels two
// that form everything again (fused, fused_weights), up to 192 one that also writes the hidden
// rows, from which ffn_gram makes the weight gradients (fused); else ffn_grad_hidden,
// ffn_rows and ffn_gram.
struct FfnLayout {
  bool fused, fused_weights;
  size_t x, weights, hid, wdt, wt, part0, part1, total;
  int Fp, Cop;
  int64_t shares;
};

static FfnLayout backward_layout(int32_t dtype, int64_t rows, int64_t C, int64_t F, int64_t Co,
                                 bool codes) {
  FfnLayout l{};
  const int V = vec_of(dtype);
  const size_t z = size_of(dtype);
  l.fused = fused_backward_takes(dtype, rows, C, Co);
  l.fused_weights = l.fused && C <= kFusedGramWidth && Co <= kFusedGramWidth;
  l.Fp = int(cdiv(F, V) * V);
  l.Cop = int(cdiv(Co, V) * V);
  const GramShape t = gram_shape(C, Co);
  l.shares = l.fused_weights
                 ? fused_weights_shares(rows, C, F, Co)
                 : gram_shares(rows, gram_tiles(2 * int64_t(l.Fp), C, t) + gram_tiles(F, Co, t), t);
  size_t off = 0;
  auto take = [&](size_t bytes) {
    const size_t at = off;
    off = align_up(off + bytes, 256);
    return at;
  };
  if (codes && !l.fused_weights) l.x = take(size_t(rows) * C * z);
  if (l.fused) l.weights = take(fused_weights_bytes(C, F, Co));
  if (!l.fused_weights) l.hid = take(size_t(rows) * 3 * l.Fp * z);
  if (!l.fused) {
    l.wdt = take(size_t(F) * l.Cop * z);
    l.wt = take(size_t(C) * 2 * l.Fp * z);
  }
  l.part0 = take(size_t(l.shares) * 2 * l.Fp * C * sizeof(float));
  l.part1 = take(size_t(l.shares) * Co * F * sizeof(float));
  l.total = off;
  return l;
}

template <typename T, typename S, bool ASYNC>
static int launch_up(const Rows<T>& x, const Rows<T>& wg, const Rows<T>& wu, int act, T* h,
                     int Fp, hipStream_t s) {
  const int64_t groups = tile_groups<S>(x.n, cdiv(Fp, S::W / 2));
  SP_CHECK_ARG(groups <= kMaxGridX, "gated_ffn: too many rows");
  ffn_up<T, S, ASYNC><<<unsigned(groups), S::THREADS, 0, s>>>(x, wg, wu, act, h, Fp);
  SP_LAUNCHED();
  return SP_OK;
}

template <typename T, typename S, bool ASYNC>
static int launch_rows(const Rows<T>& a, const Rows<T>& w, const RowsOut<T>& o, hipStream_t s) {
  const int64_t groups = tile_groups<S>(a.n, cdiv(o.n, S::W));
  SP_CHECK_ARG(groups <= kMaxGridX, "gated_ffn: too many rows");
  ffn_rows<T, S, ASYNC><<<unsigned(groups), S::THREADS, 0, s>>>(a, w, o);
  SP_LAUNCHED();
  return SP_OK;
}

template <typename T>
static int run_rows(const Rows<T>& a, const Rows<T>& w, const void* residual, int64_t ldr,
                    void* out, int n, hipStream_t s) {
  const RowsOut<T> o{static_cast<const T*>(residual), ldr, static_cast<T*>(out), n,
                     aligned(out) && n % Mfma<T>::V == 0};
  if (!whole(a) || !whole(w)) return launch_rows<T, SmallTile, false>(a, w, o, s);
  const int64_t tiles = cdiv(a.n, LargeTile::X) * cdiv(n, LargeTile::W), last = tiles % 256;
  if (n > 128 && tiles >= 256) {
    // (a last round of up to 64 tiles is one of up to 256 quarters: forward and backward pass 119 and 396 us
    // for 107 and 377 at 70k x 256 -> 688, last 18; 203 and 684 for 187 and 663 at 40k x 512 -> 1 376, last 58;
    // 140 and 478 for 137 and 479 with 96 left, 242 and 818 for 259 and 843 with 136)
    if (last == 0 || last > 64) return launch_rows<T, LargeTile, true>(a, w, o, s);
    const int64_t groups = tiles - last + cdiv(4 * last, 8) * 8;
    SP_CHECK_ARG(groups <= kMaxGridX, "gated_ffn: too many rows");
    ffn_rows_split<T><<<unsigned(groups), LargeTile::THREADS, 0, s>>>(a, w, o, int(tiles - last));
    SP_LAUNCHED();
    return SP_OK;
  }
  // (the wider of the low tiles once the others would give a CU two: 30k rows fp32, 256 -> 96 24.6 us for 20.7,
  // 512 -> 96 43.6 for 35.4; 10k rows 15 for 20)
  if (n > 64 && n <= 96 && cdiv(a.n, ThinTile::X) > 256)
    return launch_rows<T, NarrowTile, true>(a, w, o, s);
  if (fills<LongTile>(a.n, cdiv(n, LongTile::W))) return launch_rows<T, LongTile, true>(a, w, o, s);
  return launch_rows<T, ThinTile, true>(a, w, o, s);
}

template <typename T>
static int forward(const FfnCall& a) {
  const int Fp = int(cdiv(a.F, Mfma<T>::V) * Mfma<T>::V);
  T* h = static_cast<T*>(a.ws);
  const Rows<T> x = operand<T>(a.x, a.ldx, a.rows, a.C);
  const Rows<T> wg = operand<T>(a.wg, a.C, a.F, a.C), wu = operand<T>(a.wu, a.C, a.F, a.C);
  int rc;
  if (!whole(x) || !whole(wg) || !whole(wu))
    rc = launch_up<T, SmallTile, false>(x, wg, wu, a.act, h, Fp, a.stream);
  // (four stages and less: one workgroup's epilogue beside another's products is worth more than fewer
  // reads; 75k x 256 -> 688 142 us with QuickTile, 151 with LargeTile, 50k x 512 -> 1 376 269 and 257)
  else if (a.C > 4 * kStagePieces * Mfma<T>::V && fills<LargeTile>(a.rows, cdiv(Fp, LargeTile::W / 2)))
    rc = launch_up<T, LargeTile, true>(x, wg, wu, a.act, h, Fp, a.stream);
  else if (fills<QuickTile>(a.rows, cdiv(Fp, QuickTile::W / 2)))
    rc = launch_up<T, QuickTile, true>(x, wg, wu, a.act, h, Fp, a.stream);
  else
    rc = launch_up<T, ThinTile, true>(x, wg, wu, a.act, h, Fp, a.stream);
  if (rc) return rc;
  return run_rows<T>(operand<T>(h, Fp, a.rows, a.F), operand<T>(a.wd, a.F, a.Co, a.F), a.residual,
                     a.ldr, a.y, a.Co, a.stream);
}

template <typename T, int R>
static int launch_few(const FfnCall& a) {
  constexpr int V = Mfma<T>::V;
  float* h = static_cast<float*>(a.ws);
  const int lu = few_lanes(a.C, V), ld = few_lanes(a.F, V);
  ffn_few_up<T, R><<<unsigned(cdiv(a.F, kFfnThreads >> lu)), kFfnThreads, 0, a.stream>>>(
      operand<T>(a.x, a.ldx, a.rows, a.C), operand<T>(a.wg, a.C, a.F, a.C),
      operand<T>(a.wu, a.C, a.F, a.C), a.act, lu, h);
  SP_LAUNCHED();
  ffn_few_down<T, R><<<unsigned(cdiv(a.Co, kFfnThreads >> ld)), kFfnThreads, 0, a.stream>>>(
      h, int(a.rows), operand<T>(a.wd, a.F, a.Co, a.F), static_cast<const T*>(a.residual), a.ldr,
      ld, static_cast<T*>(a.y));
  SP_LAUNCHED();
  return SP_OK;
}

template <typename T>
static int few_forward(const FfnCall& a) {
  if (a.rows == 1) return launch_few<T, 1>(a);
  if (a.rows == 2) return launch_few<T, 2>(a);
  return launch_few<T, 4>(a);
}

template <typename T, typename S, bool ASYNC>
static int launch_hidden(const Rows<T>& x, const Rows<T>& wg, const Rows<T>& wu, const Rows<T>& dy,
                         const Rows<T>& wdt, int act, T* hid, int Fp, hipStream_t s) {
  const int64_t groups = tile_groups<S>(x.n, cdiv(Fp, S::W / 2));
  SP_CHECK_ARG(groups <= kMaxGridX, "gated_ffn_bwd: too many rows");
  ffn_grad_hidden<T, S, ASYNC><<<unsigned(groups), S::THREADS, 0, s>>>(x, wg, wu, dy, wdt, act,
                                                                       hid, Fp);
  SP_LAUNCHED();
  return SP_OK;
}

// dg, du and h of all rows, and dx, by the kernels of their own.
template <typename T>
static int hidden_and_dx(const FfnCall& a, const FfnLayout& l, T* hid) {
  char* ws = static_cast<char*>(a.ws);
  T* wdt = reinterpret_cast<T*>(ws + l.wdt);
  T* wt = reinterpret_cast<T*>(ws + l.wt);
  const int64_t ld2 = 2 * int64_t(l.Fp);
  const Transpose<T> d0{static_cast<const T*>(a.wd), wdt, a.Co, a.F, l.Cop, l.Cop};
  const Transpose<T> d1{static_cast<const T*>(a.wg), wt, a.F, a.C, l.Fp, ld2};
  const Transpose<T> d2{static_cast<const T*>(a.wu), wt + l.Fp, a.F, a.C, l.Fp, ld2};
  const int most_rows = l.Cop > l.Fp ? l.Cop : l.Fp, most_cols = a.F > a.C ? a.F : a.C;
  ffn_transpose<T><<<dim3(unsigned(cdiv(most_rows, 32)), unsigned(cdiv(most_cols, 32)),
                          a.dx ? 3 : 1),
                     kFfnThreads, 0, a.stream>>>(d0, d1, d2);
  SP_LAUNCHED();
  const Rows<T> x = operand<T>(a.x, a.ldx, a.rows, a.C), dy = operand<T>(a.dy, a.lddy, a.rows, a.Co);
  const Rows<T> wg = operand<T>(a.wg, a.C, a.F, a.C), wu = operand<T>(a.wu, a.C, a.F, a.C);
  // (Wd' has zeros past Co)
  const Rows<T> d = operand<T>(wdt, l.Cop, a.F, a.Co);
  int rc;
  if (!whole(x) || !whole(wg) || !whole(wu) || !whole(dy))
    rc = launch_hidden<T, SmallTile, false>(x, wg, wu, dy, d, a.act, hid, l.Fp, a.stream);
  else
    // (one workgroup's epilogue, three arrays, beside another's products: 75k x 256 -> 688 backward 428
    // us, with 256-row tiles, of which a CU holds one, 458)
    rc = launch_hidden<T, QuickTile, true>(x, wg, wu, dy, d, a.act, hid, l.Fp, a.stream);
  if (rc) return rc;
  if (!a.dx) return SP_OK;
  return run_rows<T>(operand<T>(hid, 3 * int64_t(l.Fp), a.rows, ld2),
                     operand<T>(wt, ld2, a.C, ld2), nullptr, 0, a.dx, a.C, a.stream);
}

// The weight gradients' partials from the hidden rows.
template <typename T>
static int weight_products(const FfnCall& a, const FfnLayout& l, const T* hid, float* part0,
                           float* part1, int64_t* shares) {
  Gram<T> g0{}, g1{};
  const GramShape t = gram_shape(a.C, a.Co);
  auto gram = [&](const T* h, int P, const void* b, int64_t ldb, int Q, float* part) {
    return Gram<T>{h, static_cast<const T*>(b), 3 * int64_t(l.Fp), ldb, P, Q, int(cdiv(Q, t.q)),
                   int(gram_tiles(P, Q, t)), 1, aligned(b) && ldb % Mfma<T>::V == 0, part};
  };
  if (a.dwg || a.dwu) g0 = gram(hid, 2 * l.Fp, a.x, a.ldx, a.C, part0);
  if (a.dwd) g1 = gram(hid + 2 * int64_t(l.Fp), a.F, a.dy, a.lddy, a.Co, part1);
  constexpr int stage = gram_rows<T>();
  const int64_t share = cdiv(cdiv(a.rows, l.shares), stage) * stage;
  *shares = cdiv(a.rows, share);
  const unsigned groups = unsigned(cdiv(*shares * (g0.tiles + g1.tiles), 8) * 8);
  if (t.p == 256)
    ffn_gram<T, 256, 256><<<groups, 512, 0, a.stream>>>(g0, g1, a.rows, share, int(*shares));
  else if (t.q == 64)
    ffn_gram<T, 128, 64><<<groups, 256, 0, a.stream>>>(g0, g1, a.rows, share, int(*shares));
  else if (t.q == 96)
    ffn_gram<T, 128, 96><<<groups, 256, 0, a.stream>>>(g0, g1, a.rows, share, int(*shares));
  else
    ffn_gram<T, 128, 128><<<groups, 256, 0, a.stream>>>(g0, g1, a.rows, share, int(*shares));
  SP_LAUNCHED();
  return SP_OK;
}

template <typename T>
static int backward(int32_t dtype, FfnCall a, const FfnLayout& l) {
  char* ws = static_cast<char*>(a.ws);
  if (a.codes && !l.fused_weights) {
    if (int rc = sp_restore_rows(a.codes, a.scales, a.rows, a.C, dtype, ws + l.x, a.stream))
      return rc;
    a.x = ws + l.x;
    a.ldx = a.C;
    a.codes = nullptr;
  }
  const bool weights = a.dwg || a.dwu || a.dwd;
  float* part0 = reinterpret_cast<float*>(ws + l.part0);
  float* part1 = reinterpret_cast<float*>(ws + l.part1);
  T* hid = reinterpret_cast<T*>(ws + l.hid);
  int64_t shares = 0;
  if (l.fused) {
    FusedGrad o{};
    o.weights = ws + l.weights;
    o.Fp = l.Fp;
    o.shares = l.shares;
    if (!weights) {
    } else if (l.fused_weights) {
      o.part0 = part0, o.part1 = part1;
    } else {
      o.hid = hid;
    }
    if (int rc = fused_backward(dtype, a, o, &shares)) return rc;
  } else {
    if (int rc = hidden_and_dx<T>(a, l, hid)) return rc;
  }
  if (!weights) return SP_OK;
  if (!l.fused_weights)
    if (int rc = weight_products<T>(a, l, hid, part0, part1, &shares)) return rc;
  const int64_t most = int64_t(a.F) * (a.C > a.Co ? a.C : a.Co);
  // (four values a lane where that still gives every CU a workgroup for each gradient)
  const bool vec = a.C % 4 == 0 && a.Co % 4 == 0 && most >= 65536;
  auto reduce = [&](auto kernel, int V) {
    kernel<<<dim3(unsigned(cdiv(most, 64 * V)), 3), kFfnThreads, 0, a.stream>>>(
        part0, part1, int(shares), a.C, a.F, l.Fp, a.Co, static_cast<T*>(a.dwg),
        static_cast<T*>(a.dwu), static_cast<T*>(a.dwd));
  };
  if (vec)
    reduce(ffn_reduce<T, 4>, 4);
  else
    reduce(ffn_reduce<T, 1>, 1);
  SP_LAUNCHED();
  return SP_OK;
}

static int check_ffn(const char* what, int32_t dtype, int64_t rows, int64_t C, int64_t F,
                     int64_t Co, int32_t act) {
  SP_CHECK_ARG(dtype == SP_F16 || dtype == SP_BF16 || dtype == SP_F32,
               "%s: dtype %d not supported (f16/bf16/f32)", what, dtype);
  SP_CHECK_ARG(rows >= 0 && C >= 1 && F >= 1 && Co >= 1 && C < 65536 && F < 65536 && Co < 65536,
               "%s: bad sizes rows=%lld C=%lld F=%lld Co=%lld", what, (long long)rows,
               (long long)C, (long long)F, (long long)Co);
  SP_CHECK_ARG(rows < (int64_t(1) << 31), "%s: 2^31 rows or more", what);
  SP_CHECK_ARG(act >= kActSilu && act <= kActRelu, "%s: unknown activation %d", what, act);
  return SP_OK;
}

}  // namespace sp

using namespace sp;

extern "C" size_t sp_gated_ffn_workspace(int32_t dtype, int64_t rows, int64_t C, int64_t F,
                                         int64_t Co) {
  if (check_ffn("gated_ffn", dtype, rows, C, F, Co, 0) != SP_OK || rows == 0) return 0;
  if (rows <= kFewRows) return size_t(rows) * F * sizeof(float);
  if (fused_forward_takes(dtype, rows, C, Co)) return fused_weights_bytes(C, F, Co);
  return size_t(rows) * (cdiv(F, vec_of(dtype)) * vec_of(dtype)) * size_of(dtype);
}

extern "C" int sp_gated_ffn(const void* x, int64_t ldx, int32_t dtype, int64_t rows, int64_t C,
                            const void* w_gate, const void* w_up, int64_t F, const void* w_down,
                            int64_t Co, int32_t act, const void* residual, int64_t ldr, void* y,
                            void* ws, size_t ws_bytes, void* stream) {
  if (int rc = check_ffn("gated_ffn", dtype, rows, C, F, Co, act)) return rc;
  if (rows == 0) return SP_OK;
  SP_CHECK_ARG(x && w_gate && w_up && w_down && y && ws, "gated_ffn: null pointer");
  SP_CHECK_ARG(ldx >= C && (!residual || ldr >= Co), "gated_ffn: rows overlap");
  SP_CHECK_ARG(aligned(ws), "gated_ffn: the workspace must be 16-byte aligned");
  const size_t need = sp_gated_ffn_workspace(dtype, rows, C, F, Co);
  if (ws_bytes < need)
    return set_error(SP_ERR_WORKSPACE, "gated_ffn: workspace of %zu bytes, needs %zu", ws_bytes,
                     need);
  FfnCall a{};
  a.x = x, a.wg = w_gate, a.wu = w_up, a.wd = w_down, a.residual = residual;
  a.ldx = ldx, a.ldr = ldr, a.rows = rows;
  a.C = int(C), a.F = int(F), a.Co = int(Co), a.act = act;
  a.y = y, a.ws = ws, a.stream = as_stream(stream);
  if (rows <= kFewRows)
    return dtype == SP_F16 ? few_forward<_Float16>(a)
                           : dtype == SP_BF16 ? few_forward<__bf16>(a) : few_forward<float>(a);
  if (fused_forward_takes(dtype, rows, C, Co)) return fused_forward(dtype, a);
  return dtype == SP_F16 ? forward<_Float16>(a)
                         : dtype == SP_BF16 ? forward<__bf16>(a) : forward<float>(a);
}

extern "C" size_t sp_gated_ffn_bwd_workspace(int32_t dtype, int64_t rows, int64_t C, int64_t F,
                                             int64_t Co, int32_t int8) {
  if (check_ffn("gated_ffn_bwd", dtype, rows, C, F, Co, 0) != SP_OK || rows == 0) return 0;
  return backward_layout(dtype, rows, C, F, Co, int8 != 0).total;
}

extern "C" int sp_gated_ffn_bwd(const void* dy, int64_t lddy, const void* x, int64_t ldx,
                                const int8_t* codes, const float* scales, int32_t dtype,
                                int64_t rows, int64_t C, const void* w_gate, const void* w_up,
                                int64_t F, const void* w_down, int64_t Co, int32_t act, void* dx,
                                void* dw_gate, void* dw_up, void* dw_down, void* ws,
                                size_t ws_bytes, void* stream) {
  if (int rc = check_ffn("gated_ffn_bwd", dtype, rows, C, F, Co, act)) return rc;
  if (rows == 0) return SP_OK;
  SP_CHECK_ARG((x == nullptr) != (codes == nullptr) && (codes == nullptr) == (scales == nullptr),
               "gated_ffn_bwd: either x or its codes and scales");
  SP_CHECK_ARG(dy && w_gate && w_up && w_down && ws, "gated_ffn_bwd: null pointer");
  SP_CHECK_ARG((codes || ldx >= C) && lddy >= Co, "gated_ffn_bwd: rows overlap");
  SP_CHECK_ARG(aligned(ws), "gated_ffn_bwd: the workspace must be 16-byte aligned");
  const FfnLayout l = backward_layout(dtype, rows, C, F, Co, codes != nullptr);
  if (ws_bytes < l.total)
    return set_error(SP_ERR_WORKSPACE, "gated_ffn_bwd: workspace of %zu bytes, needs %zu",
                     ws_bytes, l.total);
  FfnCall a{};
  a.dy = dy, a.x = x, a.wg = w_gate, a.wu = w_up, a.wd = w_down;
  a.ldx = ldx, a.lddy = lddy, a.rows = rows;
  a.codes = codes, a.scales = scales;
  a.C = int(C), a.F = int(F), a.Co = int(Co), a.act = act;
  a.dx = dx, a.dwg = dw_gate, a.dwu = dw_up, a.dwd = dw_down;
  a.ws = ws, a.stream = as_stream(stream);
  return dtype == SP_F16 ? backward<_Float16>(dtype, a, l)
                         : dtype == SP_BF16 ? backward<__bf16>(dtype, a, l)
                                            : backward<float>(dtype, a, l);
}
