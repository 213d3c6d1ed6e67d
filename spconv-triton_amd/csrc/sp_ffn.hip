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
// between the passes.
#include "sp_ffn.h"

namespace sp {

// Pieces [128 rows][8] of an operand on their way from memory to LDS; thread t holds piece
// t % 8 of rows t / 8 + 32 j.
template <typename T>
struct Stage {
  using frag = typename Mfma<T>::frag;
  static constexpr int V = Mfma<T>::V;
  frag r[4];

  __device__ __forceinline__ static frag piece(const Rows<T>& a, int64_t row, int k) {
    frag f = {};
    if (row >= a.n || k >= a.K) return f;
    const T* q = a.p + row * a.ld + k;
    if (a.vec && k + V <= a.K) return *reinterpret_cast<const frag*>(q);
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (k + i < a.K) f[i] = q[i];
    return f;
  }

  // 128 rows from row0, or where `b` is given 64 of each
  __device__ __forceinline__ void load(const Rows<T>& a, int64_t row0, int k0) {
    const int c = int(threadIdx.x) & 7, t = int(threadIdx.x) >> 3;
#pragma unroll
    for (int j = 0; j < 4; ++j) r[j] = piece(a, row0 + t + 32 * j, k0 + c * V);
  }
  __device__ __forceinline__ void load(const Rows<T>& a, const Rows<T>& b, int64_t row0, int k0) {
    const int c = int(threadIdx.x) & 7, t = int(threadIdx.x) >> 3;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      r[j] = piece(a, row0 + t + 32 * j, k0 + c * V);
      r[j + 2] = piece(b, row0 + t + 32 * j, k0 + c * V);
    }
  }
  __device__ __forceinline__ void store(char* lds) const {
    const int c = int(threadIdx.x) & 7, t = int(threadIdx.x) >> 3;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int row = t + 32 * j;
      *reinterpret_cast<frag*>(lds + (row * 8 + swizzled<8>(row, c)) * 16) = r[j];
    }
  }
  __device__ __forceinline__ static frag read(const char* lds, int row, int c) {
    return *reinterpret_cast<const frag*>(lds + (row * 8 + swizzled<8>(row, c)) * 16);
  }
};

// acc[j][i] += the products of W rows wrow[i] .. + 31 and X rows xrow + 32 j .. + 31 over
// all of K.  The MFMA's rows are W's and its columns X's, so that lane l holds
// four neighbouring outputs of X row l & 31 in every four registers.
// w2: the second half of the W tile comes from there.
template <typename T, int NW>
__device__ __forceinline__ void products(const Rows<T>& x, int64_t x0, const Rows<T>& w,
                                         const Rows<T>* w2, int64_t w0, const int (&wrow)[NW],
                                         int xrow, char* lds, floatx16 (&acc)[2][NW]) {
  constexpr int STEP = kStagePieces * Mfma<T>::V;
  const int lane = int(threadIdx.x) & 31, half = (int(threadIdx.x) >> 5) & 1;
  Stage<T> sx, sw;
  auto fetch = [&](int k) {
    sx.load(x, x0, k);
    if (w2)
      sw.load(w, *w2, w0, k);
    else
      sw.load(w, w0, k);
  };
  const int steps = (x.K + STEP - 1) / STEP;
  fetch(0);
  for (int s = 0; s < steps; ++s) {
    char* bx = lds + (s & 1) * (2 * kStageBytes);
    char* bw = bx + kStageBytes;
    sx.store(bx);
    sw.store(bw);
    __syncthreads();  // (the other buffer's readers are past their previous barrier)
    if (s + 1 < steps) fetch((s + 1) * STEP);
#pragma unroll
    for (int c = 0; c < kStagePieces; c += 2) {
      typename Mfma<T>::frag fx[2], fw[NW];
#pragma unroll
      for (int j = 0; j < 2; ++j) fx[j] = Stage<T>::read(bx, xrow + 32 * j + lane, c + half);
#pragma unroll
      for (int i = 0; i < NW; ++i) fw[i] = Stage<T>::read(bw, wrow[i] + lane, c + half);
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int i = 0; i < NW; ++i) Mfma<T>::mma(fw[i], fx[j], acc[j][i]);
    }
  }
  __syncthreads();
}

// One 32 x 32 accumulator to LDS rows of `pitch` bytes, as values of type S.
template <typename S, typename F>
__device__ __forceinline__ void put_tile(char* lds, int pitch, int row, int col, F&& value) {
  const int lane = int(threadIdx.x) & 31, half = (int(threadIdx.x) >> 5) & 1;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    struct alignas(sizeof(S) * 4) Four {
      S v[4];
    } f;
#pragma unroll
    for (int i = 0; i < 4; ++i) f.v[i] = S(value(4 * q + i));
    *reinterpret_cast<Four*>(lds + (row + lane) * pitch + (col + 8 * q + 4 * half) * int(sizeof(S))) = f;
  }
}

// LDS rows of COLS values to memory, columns below n.  (out rows start at 16 bytes, n is a
// multiple of V.)
template <typename T, int COLS>
__device__ __forceinline__ void write_rows(const char* lds, int pitch, T* __restrict__ out,
                                           int64_t ld, int64_t row0, int64_t rows, int col0,
                                           int n) {
  using frag = typename Mfma<T>::frag;
  constexpr int V = Mfma<T>::V, PER = COLS / V;
  for (int i = int(threadIdx.x); i < kTileRows * PER; i += kFfnThreads) {
    const int r = i / PER, c = (i - r * PER) * V;
    if (row0 + r < rows && col0 + c < n)
      *reinterpret_cast<frag*>(out + (row0 + r) * ld + col0 + c) =
          *reinterpret_cast<const frag*>(lds + r * pitch + c * int(sizeof(T)));
  }
}

template <int N>
__device__ __forceinline__ void clear(floatx16 (&acc)[2][N]) {
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int k = 0; k < 16; ++k) acc[j][i][k] = 0.f;
}

// h = act(x Wg') * (x Wu'), 128 rows x 64 hidden units a workgroup; columns from F to the
// padded width are zeros.
template <typename T>
__global__ __launch_bounds__(kFfnThreads) void ffn_up(Rows<T> x, Rows<T> wg, Rows<T> wu, int act,
                                                      T* __restrict__ h, int Fp) {
  __shared__ __attribute__((aligned(16))) char lds[4 * kStageBytes];
  const int wave = int(threadIdx.x) >> 6, wm = wave >> 1, wn = wave & 1;
  const int64_t x0 = int64_t(blockIdx.y) * kTileRows;
  const int f0 = int(blockIdx.x) * kHiddenTile;
  floatx16 acc[2][2];
  clear(acc);
  const int wrow[2] = {wn * 32, kHiddenTile + wn * 32};
  products<T, 2>(x, x0, wg, &wu, f0, wrow, wm * 64, lds, acc);
  constexpr int pitch = kHiddenTile * int(sizeof(T)) + 16;
  with_gate<sizeof(T) == 2>(act, [&](auto gate) {
#pragma unroll
    for (int j = 0; j < 2; ++j)
      put_tile<T>(lds, pitch, wm * 64 + 32 * j, wn * 32, [&](int i) {
        float value, slope;
        gate(acc[j][0][i], value, slope);
        return value * acc[j][1][i];
      });
  });
  __syncthreads();
  write_rows<T, kHiddenTile>(lds, pitch, h, Fp, x0, x.n, f0, Fp);
}

// dg, du and h of 128 rows x 64 hidden units, in rows of 3 Fp values.  wdt: Wd transposed.
template <typename T>
__global__ __launch_bounds__(kFfnThreads) void ffn_grad_hidden(Rows<T> x, Rows<T> wg, Rows<T> wu,
                                                               Rows<T> dy, Rows<T> wdt, int act,
                                                               T* __restrict__ out, int Fp) {
  __shared__ __attribute__((aligned(16))) char lds[4 * kStageBytes];
  const int wave = int(threadIdx.x) >> 6, wm = wave >> 1, wn = wave & 1;
  const int64_t x0 = int64_t(blockIdx.y) * kTileRows;
  const int f0 = int(blockIdx.x) * kHiddenTile;
  floatx16 acc[2][2], dh[2][1];
  clear(acc);
  clear(dh);
  const int wrow[2] = {wn * 32, kHiddenTile + wn * 32}, drow[1] = {wn * 32};
  products<T, 2>(x, x0, wg, &wu, f0, wrow, wm * 64, lds, acc);
  products<T, 1>(dy, x0, wdt, nullptr, f0, drow, wm * 64, lds, dh);
  constexpr int pitch = kHiddenTile * int(sizeof(T)) + 16;
  with_gate<sizeof(T) == 2>(act, [&](auto gate) {
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float value, slope;
        gate(acc[j][0][i], value, slope);
        const float u = acc[j][1][i], d = dh[j][0][i];
        acc[j][0][i] = d * u * slope;
        acc[j][1][i] = d * value;
        dh[j][0][i] = value * u;
      }
  });
#pragma unroll
  for (int part = 0; part < 3; ++part) {
    if (part) __syncthreads();
#pragma unroll
    for (int j = 0; j < 2; ++j)
      put_tile<T>(lds, pitch, wm * 64 + 32 * j, wn * 32, [&](int i) {
        return part == 0 ? acc[j][0][i] : part == 1 ? acc[j][1][i] : dh[j][0][i];
      });
    __syncthreads();
    write_rows<T, kHiddenTile>(lds, pitch, out + int64_t(part) * Fp, 3 * int64_t(Fp), x0, x.n, f0,
                               Fp);
  }
}

// out = a w' (+ residual), 128 rows x 128 columns a workgroup; fp32 until the residual is in.
template <typename T>
__global__ __launch_bounds__(kFfnThreads) void ffn_rows(Rows<T> a, Rows<T> w,
                                                        const T* __restrict__ residual,
                                                        int64_t ldr, T* __restrict__ out, int n) {
  constexpr int pitch = kTileRows * 4 + 16;
  __shared__ __attribute__((aligned(16))) char
      lds[4 * kStageBytes > kTileRows * pitch ? 4 * kStageBytes : kTileRows * pitch];
  const int wave = int(threadIdx.x) >> 6, wm = wave >> 1, wn = wave & 1;
  const int64_t x0 = int64_t(blockIdx.y) * kTileRows;
  const int n0 = int(blockIdx.x) * kTileRows;
  floatx16 acc[2][2];
  clear(acc);
  const int wrow[2] = {wn * 64, wn * 64 + 32};
  products<T, 2>(a, x0, w, nullptr, n0, wrow, wm * 64, lds, acc);
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int i = 0; i < 2; ++i)
      put_tile<float>(lds, pitch, wm * 64 + 32 * j, wn * 64 + 32 * i,
                      [&](int k) { return acc[j][i][k]; });
  __syncthreads();
  for (int i = int(threadIdx.x); i < kTileRows * kTileRows; i += kFfnThreads) {
    const int r = i / kTileRows, c = i - r * kTileRows;
    if (x0 + r < a.n && n0 + c < n) {
      float v = *reinterpret_cast<const float*>(lds + r * pitch + c * 4);
      if (residual) v += to_f32(residual[(x0 + r) * ldr + n0 + c]);
      out[(x0 + r) * int64_t(n) + n0 + c] = from_f32<T>(v);
    }
  }
}

// dst [cols, ldd] = src [rows, cols] transposed, columns from rows to ldd's share as zeros:
// dst[c * ldd + r] for r < rows_out.
template <typename T>
__global__ __launch_bounds__(kFfnThreads) void ffn_transpose(const T* __restrict__ src, int rows,
                                                             int cols, int rows_out,
                                                             int cols_out, int64_t ldd,
                                                             T* __restrict__ dst) {
  __shared__ T tile[32][33];
  const int r0 = int(blockIdx.x) * 32, c0 = int(blockIdx.y) * 32;
  const int tx = int(threadIdx.x) & 31, ty = int(threadIdx.x) >> 5;
#pragma unroll
  for (int j = 0; j < 32; j += 8) {
    const int r = r0 + ty + j, c = c0 + tx;
    tile[ty + j][tx] = r < rows && c < cols ? src[int64_t(r) * cols + c] : T(0.f);
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < 32; j += 8) {
    const int c = c0 + ty + j, r = r0 + tx;
    if (c < cols_out && r < rows_out) dst[int64_t(c) * ldd + r] = tile[tx][ty + j];
  }
}

// ---- weight gradients ------------------------------------------------------------
// Partials of a' b over a share of the rows: a [rows, P] is of the hidden width, b [rows, Q] of x's
// or dy's, 128 x TQ of the result a workgroup.  Rows are the MFMA's reduction: 64 of them
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

constexpr int kGramP = 128;
constexpr int kGramStage = 16384;  // bytes of 128 columns in a stage

template <typename T>
constexpr int gram_rows() { return kGramStage / (kGramP * int(sizeof(T))); }

typedef short short4v __attribute__((ext_vector_type(4)));

// COLS columns of a stage in LDS.  16-bit rows hold their 16-byte pieces permuted: the four rows that
// sixteen lanes read at once, 32 bytes of each, fall on different banks, and so do the 64 bytes of
// each that 32 lanes read.
template <typename T, int COLS>
struct GramStage {
  using frag = typename Mfma<T>::frag;
  static constexpr int V = Mfma<T>::V, PER = COLS / V, ROWS = gram_rows<T>();
  static constexpr int N = ROWS * PER / kFfnThreads;
  frag r[N];

  __device__ __forceinline__ static int slot(int row, int piece) {
    if constexpr (sizeof(T) == 4) return piece;
    if constexpr (COLS == 128) return piece ^ ((row & 1) * 4 + ((row >> 1) & 1) * 10);
    return piece ^ ((row & 3) << 1);
  }
  __device__ __forceinline__ void load(const T* p, int64_t ld, int vec, int64_t m, int64_t hi,
                                       int c0, int n) {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int i = int(threadIdx.x) + j * kFfnThreads, row = i / PER;
      const int c = c0 + (i - row * PER) * V;
      r[j] = frag{};
      if (m + row >= hi || c >= n) continue;
      const T* q = p + (m + row) * ld + c;
      if (vec && c + V <= n) {
        r[j] = *reinterpret_cast<const frag*>(q);
      } else {
#pragma unroll
        for (int k = 0; k < V; ++k)
          if (c + k < n) r[j][k] = q[k];
      }
    }
  }
  __device__ __forceinline__ void store(char* lds) const {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int i = int(threadIdx.x) + j * kFfnThreads, row = i / PER;
      *reinterpret_cast<frag*>(lds + (row * PER + slot(row, i - row * PER)) * 16) = r[j];
    }
  }
  // columns c0 .. c0 + 31, rows k .. k + 2 V - 1, as the MFMA wants them (rows in one order for
  // both of its operands)
  __device__ __forceinline__ static frag read(const char* lds, int k, int c0) {
    const int lane = int(threadIdx.x) & 63, half = lane >> 5;
    if constexpr (sizeof(T) == 4) {
      frag f;
#pragma unroll
      for (int i = 0; i < V; ++i)
        f[i] = *reinterpret_cast<const T*>(lds + ((k + half * V + i) * COLS + c0 + (lane & 31)) * 4);
      return f;
    } else {
      const int t = lane & 15, c = c0 + (lane & 16) + (t & 3) * 4;
      union {
        short4v q[2];
        frag f;
      } u;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int row = k + 8 * half + 4 * j + (t >> 2);
        const char* at = lds + (row * PER + slot(row, c >> 3)) * 16 + (c & 7) * 2;
        u.q[j] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) short4v*)(at));
      }
      return u.f;
    }
  }
};

template <typename T, int TQ>
__global__ __launch_bounds__(kFfnThreads, 2) void ffn_gram(Gram<T> g0, Gram<T> g1, int64_t rows,
                                                           int64_t share) {
  using frag = typename Mfma<T>::frag;
  constexpr int ROWS = gram_rows<T>(), NQ = TQ / 64;
  constexpr int STAGE = kGramStage + kGramStage / kGramP * TQ;
  __shared__ __attribute__((aligned(16))) char lds[2 * STAGE];
  int tile = int(blockIdx.x);
  const bool second = tile >= g0.tiles;
  if (second) tile -= g0.tiles;
  const Gram<T> g = second ? g1 : g0;
  const int p0 = tile / g.tiles_q * kGramP, q0 = tile % g.tiles_q * TQ;
  const int64_t lo = int64_t(blockIdx.y) * share;
  const int64_t hi = lo + share < rows ? lo + share : rows;
  const int wave = int(threadIdx.x) >> 6, wp = (wave >> 1) * 64, wq = (wave & 1) * (TQ / 2);
  floatx16 acc[2][NQ];
  clear(acc);
  GramStage<T, kGramP> sa;
  GramStage<T, TQ> sb;
  auto fetch = [&](int64_t m) {
    sa.load(g.a, g.lda, g.vec_a, m, hi, p0, g.P);
    sb.load(g.b, g.ldb, g.vec_b, m, hi, q0, g.Q);
  };
  fetch(lo);
  int s = 0;
  for (int64_t m = lo; m < hi; m += ROWS, s ^= 1) {
    char* la = lds + s * STAGE;
    char* lb = la + kGramStage;
    sa.store(la);
    sb.store(lb);
    __syncthreads();
    if (m + ROWS < hi) fetch(m + ROWS);
#pragma unroll
    for (int k = 0; k < ROWS; k += 2 * Mfma<T>::V) {
      frag fa[2], fb[NQ];
#pragma unroll
      for (int i = 0; i < 2; ++i) fa[i] = GramStage<T, kGramP>::read(la, k, wp + 32 * i);
#pragma unroll
      for (int i = 0; i < NQ; ++i) fb[i] = GramStage<T, TQ>::read(lb, k, wq + 32 * i);
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < NQ; ++j) Mfma<T>::mma(fa[i], fb[j], acc[i][j]);
    }
  }
  float* part = g.part + int64_t(blockIdx.y) * g.P * g.Q;
  const int lane = int(threadIdx.x) & 31, half = (int(threadIdx.x) >> 5) & 1;
#pragma unroll
  for (int i = 0; i < 2; ++i)
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
// first product, dWd [Co][F] from the second, [F][Co].  64 values a workgroup, four runs of the shares
// summed apart and then in order.
template <typename T>
__global__ __launch_bounds__(kFfnThreads) void ffn_reduce(const float* __restrict__ part0,
                                                          const float* __restrict__ part1,
                                                          int shares, int C, int F, int Fp, int Co,
                                                          T* __restrict__ dwg, T* __restrict__ dwu,
                                                          T* __restrict__ dwd) {
  __shared__ float lds[4][64];
  const int lane = int(threadIdx.x) & 63, run = int(threadIdx.x) >> 6;
  const int64_t i = int64_t(blockIdx.x) * 64 + lane;
  const int64_t n0 = int64_t(F) * C, n1 = int64_t(F) * Co;
  const int which = int(blockIdx.y);
  T* dst = which == 0 ? dwg : which == 1 ? dwu : dwd;
  if (!dst) return;
  const bool in = i < (which == 2 ? n1 : n0);
  const float* p = which == 2 ? part1 + i : part0 + (which ? int64_t(Fp) * C : 0) + i;
  const int64_t stride = which == 2 ? n1 : 2 * int64_t(Fp) * C;
  float v = 0.f;
  if (in) {
    const int per = (shares + 3) / 4, end = (run + 1) * per < shares ? (run + 1) * per : shares;
#pragma unroll 8
    for (int s = run * per; s < end; ++s) v += p[int64_t(s) * stride];
  }
  lds[run][lane] = v;
  __syncthreads();
  if (run != 0 || !in) return;
  v = ((lds[0][lane] + lds[1][lane]) + lds[2][lane]) + lds[3][lane];
  const int64_t f = i / Co;
  dst[which == 2 ? (i - f * Co) * F + f : i] = from_f32<T>(v);
}

// ---- host ------------------------------------------------------------------------
// Columns of a weight gradient's tile: 128, or 64 where both widths fit (half of a 128-wide tile would be
// idle).
static int gram_tile_q(int64_t C, int64_t Co) { return C <= 64 && Co <= 64 ? 64 : 128; }

static int64_t gram_tiles(int64_t P, int64_t Q, int tq) { return cdiv(P, kGramP) * cdiv(Q, tq); }

// Shares of the rows in the weight gradients: two workgroups a CU, each with at least 256 rows.
static int64_t gram_shares(int64_t rows, int64_t tiles) {
  const int64_t want = cdiv(512, tiles), most = cdiv(rows, 256);
  return want < most ? want : most;
}

// The backward pass's workspace, and which kernels it takes: for 16-bit rows of up to 128 channels two
// that form everything again (fused, fused_weights), up to 256 one that also writes the hidden
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
  l.fused = fused_backward_takes(dtype, C, Co);
  l.fused_weights = fused_weights_take(dtype, C, Co);
  l.Fp = int(cdiv(F, V) * V);
  l.Cop = int(cdiv(Co, V) * V);
  const int tq = gram_tile_q(C, Co);
  l.shares = l.fused_weights
                 ? fused_weights_shares(rows, C, F, Co)
                 : gram_shares(rows, gram_tiles(2 * int64_t(l.Fp), C, tq) + gram_tiles(F, Co, tq));
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

template <typename T>
static int launch_rows(const Rows<T>& a, const Rows<T>& w, const void* residual, int64_t ldr,
                       void* out, int n, hipStream_t s) {
  const dim3 grid(unsigned(cdiv(n, kTileRows)), unsigned(cdiv(a.n, kTileRows)));
  ffn_rows<T><<<grid, kFfnThreads, 0, s>>>(a, w, static_cast<const T*>(residual), ldr,
                                           static_cast<T*>(out), n);
  SP_LAUNCHED();
  return SP_OK;
}

template <typename T>
static int forward(const FfnCall& a) {
  const int Fp = int(cdiv(a.F, Mfma<T>::V) * Mfma<T>::V);
  T* h = static_cast<T*>(a.ws);
  const dim3 grid(unsigned(cdiv(a.F, kHiddenTile)), unsigned(cdiv(a.rows, kTileRows)));
  ffn_up<T><<<grid, kFfnThreads, 0, a.stream>>>(
      operand<T>(a.x, a.ldx, a.rows, a.C), operand<T>(a.wg, a.C, a.F, a.C),
      operand<T>(a.wu, a.C, a.F, a.C), a.act, h, Fp);
  SP_LAUNCHED();
  return launch_rows<T>(operand<T>(h, Fp, a.rows, a.F), operand<T>(a.wd, a.F, a.Co, a.F),
                        a.residual, a.ldr, a.y, a.Co, a.stream);
}

template <typename T>
static int transpose(const void* src, int rows, int cols, int rows_out, int64_t ldd, T* dst,
                     hipStream_t s) {
  const dim3 grid(unsigned(cdiv(rows_out, 32)), unsigned(cdiv(cols, 32)));
  ffn_transpose<T><<<grid, kFfnThreads, 0, s>>>(static_cast<const T*>(src), rows, cols, rows_out,
                                                cols, ldd, dst);
  SP_LAUNCHED();
  return SP_OK;
}

// dg, du and h of all rows, and dx, by the kernels of their own.
template <typename T>
static int hidden_and_dx(const FfnCall& a, const FfnLayout& l, T* hid) {
  char* ws = static_cast<char*>(a.ws);
  T* wdt = reinterpret_cast<T*>(ws + l.wdt);
  T* wt = reinterpret_cast<T*>(ws + l.wt);
  if (int rc = transpose<T>(a.wd, a.Co, a.F, l.Cop, l.Cop, wdt, a.stream)) return rc;
  const dim3 grid(unsigned(cdiv(a.F, kHiddenTile)), unsigned(cdiv(a.rows, kTileRows)));
  ffn_grad_hidden<T><<<grid, kFfnThreads, 0, a.stream>>>(
      operand<T>(a.x, a.ldx, a.rows, a.C), operand<T>(a.wg, a.C, a.F, a.C),
      operand<T>(a.wu, a.C, a.F, a.C), operand<T>(a.dy, a.lddy, a.rows, a.Co),
      operand<T>(wdt, l.Cop, a.F, a.Co), a.act, hid, l.Fp);
  SP_LAUNCHED();
  if (!a.dx) return SP_OK;
  if (int rc = transpose<T>(a.wg, a.F, a.C, l.Fp, 2 * int64_t(l.Fp), wt, a.stream)) return rc;
  if (int rc = transpose<T>(a.wu, a.F, a.C, l.Fp, 2 * int64_t(l.Fp), wt + l.Fp, a.stream))
    return rc;
  return launch_rows<T>(operand<T>(hid, 3 * int64_t(l.Fp), a.rows, 2 * int64_t(l.Fp)),
                        operand<T>(wt, 2 * int64_t(l.Fp), a.C, 2 * int64_t(l.Fp)), nullptr, 0,
                        a.dx, a.C, a.stream);
}

// The weight gradients' partials from the hidden rows.
template <typename T>
static int weight_products(const FfnCall& a, const FfnLayout& l, const T* hid, float* part0,
                           float* part1, int64_t* shares) {
  Gram<T> g0{}, g1{};
  const int tq = gram_tile_q(a.C, a.Co);
  auto gram = [&](const T* h, int P, const void* b, int64_t ldb, int Q, float* part) {
    return Gram<T>{h, static_cast<const T*>(b), 3 * int64_t(l.Fp), ldb, P, Q, int(cdiv(Q, tq)),
                   int(gram_tiles(P, Q, tq)), 1, aligned(b) && ldb % Mfma<T>::V == 0, part};
  };
  if (a.dwg || a.dwu) g0 = gram(hid, 2 * l.Fp, a.x, a.ldx, a.C, part0);
  if (a.dwd) g1 = gram(hid + 2 * int64_t(l.Fp), a.F, a.dy, a.lddy, a.Co, part1);
  constexpr int stage = gram_rows<T>();
  const int64_t share = cdiv(cdiv(a.rows, l.shares), stage) * stage;
  *shares = cdiv(a.rows, share);
  const dim3 grid(unsigned(g0.tiles + g1.tiles), unsigned(*shares));
  if (tq == 64)
    ffn_gram<T, 64><<<grid, kFfnThreads, 0, a.stream>>>(g0, g1, a.rows, share);
  else
    ffn_gram<T, 128><<<grid, kFfnThreads, 0, a.stream>>>(g0, g1, a.rows, share);
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
  ffn_reduce<T><<<dim3(unsigned(cdiv(most, 64)), 3), kFfnThreads, 0, a.stream>>>(
      part0, part1, int(shares), a.C, a.F, l.Fp, a.Co, static_cast<T*>(a.dwg),
      static_cast<T*>(a.dwu), static_cast<T*>(a.dwd));
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
  // (workgroups along the rows are a grid's y)
  SP_CHECK_ARG(cdiv(rows, kTileRows) <= 65535, "%s: more than %lld rows", what,
               (long long)kTileRows * 65535);
  SP_CHECK_ARG(act >= kActSilu && act <= kActRelu, "%s: unknown activation %d", what, act);
  return SP_OK;
}

}  // namespace sp

using namespace sp;

extern "C" size_t sp_gated_ffn_workspace(int32_t dtype, int64_t rows, int64_t C, int64_t F,
                                         int64_t Co) {
  if (check_ffn("gated_ffn", dtype, rows, C, F, Co, 0) != SP_OK || rows == 0) return 0;
  if (fused_forward_takes(dtype, rows, C, F, Co)) return fused_weights_bytes(C, F, Co);
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
  if (fused_forward_takes(dtype, rows, C, F, Co)) return fused_forward(dtype, a);
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
