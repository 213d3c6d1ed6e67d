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
#include "sp_common.h"
#include "sp_mfma.h"

namespace sp {

constexpr int kFfnThreads = 256;
constexpr int kTileRows = 128;  // rows of an operand in a stage
constexpr int kStagePieces = 8;  // 16-byte pieces of a row in a stage: 64 16-bit values
constexpr int kStageBytes = kTileRows * kStagePieces * 16;
constexpr int kHiddenTile = 64;  // hidden units of a workgroup where it forms gate and up

enum { kActSilu = 0, kActGelu = 1, kActRelu = 2 };

// The gate's activation and its derivative.
__device__ __forceinline__ void gate(int act, float z, float& value, float& slope) {
  if (act == kActSilu) {
    const float sig = 1.f / (1.f + expf(-z));
    value = z * sig;
    slope = sig * (1.f + z * (1.f - sig));
  } else if (act == kActGelu) {
    const float cdf = 0.5f * (1.f + erff(z * 0.70710678118654752f));
    value = z * cdf;
    slope = cdf + z * expf(-0.5f * z * z) * 0.39894228040143268f;
  } else {
    value = z < 0.f ? 0.f : z;  // (a NaN stays)
    slope = z > 0.f ? 1.f : 0.f;
  }
}

// A row-major operand: rows of K values; vec: rows start at multiples of 16 bytes.
template <typename T>
struct Rows {
  const T* p;
  int64_t ld;
  int64_t n;  // rows; what lies past them reads as zero
  int K;
  int vec;
};

// Pieces [128 rows][8] of an operand on their way from memory to LDS; thread t holds piece
// t % 8 of rows t / 8 + 32 j.  In LDS piece c of row r lies at r * 8 + (c ^ (r & 7)),
// so that the eight lanes that write a row and the rows that an MFMA operand
// reads (one piece of 32 rows) spread over all banks.
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
      *reinterpret_cast<frag*>(lds + (row * 8 + (c ^ (row & 7))) * 16) = r[j];
    }
  }
  __device__ __forceinline__ static frag read(const char* lds, int row, int c) {
    return *reinterpret_cast<const frag*>(lds + (row * 8 + (c ^ (row & 7))) * 16);
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
#pragma unroll
  for (int j = 0; j < 2; ++j)
    put_tile<T>(lds, pitch, wm * 64 + 32 * j, wn * 32, [&](int i) {
      float value, slope;
      gate(act, acc[j][0][i], value, slope);
      return value * acc[j][1][i];
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
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float value, slope;
      gate(act, acc[j][0][i], value, slope);
      const float u = acc[j][1][i], d = dh[j][0][i];
      acc[j][0][i] = d * u * slope;
      acc[j][1][i] = d * value;
      dh[j][0][i] = value * u;
    }
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

// Partials of a' b over a share of the rows: a [rows, P], b [rows, Q], 64 x 64 of the result a
// workgroup.  Rows are the reduction: 32 of them a stage, read from LDS one value at a time.
template <typename T>
struct Gram {
  const T *a, *b;
  int64_t lda, ldb;
  int P, Q;
  int tiles_q, tiles;   // 64 x 64 tiles along Q, and all
  float* part;          // [shares][P][Q]
};

constexpr int kGramTile = 64;
constexpr int kGramRows = 32;

template <typename T>
__global__ __launch_bounds__(kFfnThreads) void ffn_gram(Gram<T> g0, Gram<T> g1, int64_t rows,
                                                        int64_t share) {
  using frag = typename Mfma<T>::frag;
  constexpr int V = Mfma<T>::V;
  __shared__ T sa[kGramRows][kGramTile + 2], sb[kGramRows][kGramTile + 2];
  int tile = int(blockIdx.x);
  const bool second = tile >= g0.tiles;
  const Gram<T>& g = second ? g1 : g0;
  if (second) tile -= g0.tiles;
  const int p0 = tile / g.tiles_q * kGramTile, q0 = tile % g.tiles_q * kGramTile;
  const int64_t lo = int64_t(blockIdx.y) * share;
  const int64_t hi = lo + share < rows ? lo + share : rows;
  const int wave = int(threadIdx.x) >> 6, wp = (wave >> 1) * 32, wq = (wave & 1) * 32;
  const int lane = int(threadIdx.x) & 31, half = (int(threadIdx.x) >> 5) & 1;
  floatx16 acc;
#pragma unroll
  for (int i = 0; i < 16; ++i) acc[i] = 0.f;
  for (int64_t m = lo; m < hi; m += kGramRows) {
    for (int i = int(threadIdx.x); i < kGramRows * kGramTile; i += kFfnThreads) {
      const int r = i / kGramTile, c = i % kGramTile;
      sa[r][c] = m + r < hi && p0 + c < g.P ? g.a[(m + r) * g.lda + p0 + c] : T(0.f);
      sb[r][c] = m + r < hi && q0 + c < g.Q ? g.b[(m + r) * g.ldb + q0 + c] : T(0.f);
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kGramRows; k += 2 * V) {
      frag fa, fb;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        fa[i] = sa[k + half * V + i][wp + lane];
        fb[i] = sb[k + half * V + i][wq + lane];
      }
      Mfma<T>::mma(fa, fb, acc);
    }
    __syncthreads();
  }
  float* part = g.part + int64_t(blockIdx.y) * g.P * g.Q;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int p = p0 + wp + (i & 3) + 8 * (i >> 2) + 4 * half, q = q0 + wq + lane;
    if (p < g.P && q < g.Q) part[int64_t(p) * g.Q + q] = acc[i];
  }
}

// dst = the partials of every value in ascending share.  Rows of the partial from `skip_at` on
// lie `skip` rows further (the second of two padded blocks).
template <typename T>
__global__ __launch_bounds__(kFfnThreads) void ffn_reduce(const float* __restrict__ part,
                                                          int64_t stride, int shares, int64_t n,
                                                          T* __restrict__ dst) {
  const int64_t i = int64_t(blockIdx.x) * kFfnThreads + threadIdx.x;
  if (i >= n) return;
  float v = 0.f;
#pragma unroll 8
  for (int s = 0; s < shares; ++s) v += part[int64_t(s) * stride + i];
  dst[i] = from_f32<T>(v);
}

// ---- host ------------------------------------------------------------------------
static bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <typename T>
static Rows<T> operand(const void* p, int64_t ld, int64_t n, int64_t K) {
  return Rows<T>{static_cast<const T*>(p), ld, n, int(K), aligned(p) && ld % Mfma<T>::V == 0};
}

static int vec_of(int32_t dtype) { return dtype == SP_F32 ? 4 : 8; }
static size_t size_of(int32_t dtype) { return dtype == SP_F32 ? 4 : 2; }

struct FfnCall {
  const void *x, *wg, *wu, *wd, *residual, *dy;
  int64_t ldx, ldr, lddy, rows;
  int C, F, Co, act;
  void *y, *dx, *dwg, *dwu, *dwd;
  void* ws;
  hipStream_t stream;
};

// Shares of the rows in the weight gradients: enough workgroups for the chip, each with 256 rows.
static int64_t gram_shares(int64_t rows, int64_t tiles) {
  const int64_t want = cdiv(2048, tiles), most = cdiv(rows, 256);
  return want < most ? want : most;
}

static int64_t gram_tiles(int64_t P, int64_t Q) {
  return cdiv(P, kGramTile) * cdiv(Q, kGramTile);
}

struct FfnLayout {
  size_t h, wdt, wt, part0, part1, total;
  int Fp, Cop;
  int64_t shares;
};

static FfnLayout backward_layout(int32_t dtype, int64_t rows, int64_t C, int64_t F, int64_t Co) {
  FfnLayout l{};
  const int V = vec_of(dtype);
  const size_t z = size_of(dtype);
  l.Fp = int(cdiv(F, V) * V);
  l.Cop = int(cdiv(Co, V) * V);
  l.shares = gram_shares(rows, gram_tiles(2 * int64_t(l.Fp), C) + gram_tiles(Co, F));
  size_t off = 0;
  auto take = [&](size_t bytes) {
    const size_t at = off;
    off = align_up(off + bytes, 256);
    return at;
  };
  l.h = take(size_t(rows) * 3 * l.Fp * z);
  l.wdt = take(size_t(F) * l.Cop * z);
  l.wt = take(size_t(C) * 2 * l.Fp * z);
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

template <typename T>
static int reduce(const float* part, int64_t stride, int64_t shares, int64_t n, void* dst,
                  hipStream_t s) {
  ffn_reduce<T><<<unsigned(cdiv(n, kFfnThreads)), kFfnThreads, 0, s>>>(
      part, stride, int(shares), n, static_cast<T*>(dst));
  SP_LAUNCHED();
  return SP_OK;
}

template <typename T>
static int backward(const FfnCall& a, const FfnLayout& l) {
  char* ws = static_cast<char*>(a.ws);
  T* hid = reinterpret_cast<T*>(ws + l.h);
  T* wdt = reinterpret_cast<T*>(ws + l.wdt);
  T* wt = reinterpret_cast<T*>(ws + l.wt);
  if (int rc = transpose<T>(a.wd, a.Co, a.F, l.Cop, l.Cop, wdt, a.stream)) return rc;
  if (int rc = transpose<T>(a.wg, a.F, a.C, l.Fp, 2 * int64_t(l.Fp), wt, a.stream)) return rc;
  if (int rc = transpose<T>(a.wu, a.F, a.C, l.Fp, 2 * int64_t(l.Fp), wt + l.Fp, a.stream))
    return rc;
  const dim3 grid(unsigned(cdiv(a.F, kHiddenTile)), unsigned(cdiv(a.rows, kTileRows)));
  ffn_grad_hidden<T><<<grid, kFfnThreads, 0, a.stream>>>(
      operand<T>(a.x, a.ldx, a.rows, a.C), operand<T>(a.wg, a.C, a.F, a.C),
      operand<T>(a.wu, a.C, a.F, a.C), operand<T>(a.dy, a.lddy, a.rows, a.Co),
      operand<T>(wdt, l.Cop, a.F, a.Co), a.act, hid, l.Fp);
  SP_LAUNCHED();
  if (a.dx) {
    if (int rc = launch_rows<T>(operand<T>(hid, 3 * int64_t(l.Fp), a.rows, 2 * int64_t(l.Fp)),
                                operand<T>(wt, 2 * int64_t(l.Fp), a.C, 2 * int64_t(l.Fp)),
                                nullptr, 0, a.dx, a.C, a.stream))
      return rc;
  }
  Gram<T> g0{}, g1{};
  const int64_t ld = 3 * int64_t(l.Fp);
  if (a.dwg || a.dwu) {
    g0 = Gram<T>{hid, static_cast<const T*>(a.x), ld, a.ldx, 2 * l.Fp, a.C,
                 int(cdiv(a.C, kGramTile)), int(gram_tiles(2 * int64_t(l.Fp), a.C)),
                 reinterpret_cast<float*>(ws + l.part0)};
  }
  if (a.dwd) {
    g1 = Gram<T>{static_cast<const T*>(a.dy), hid + 2 * int64_t(l.Fp), a.lddy, ld, a.Co, a.F,
                 int(cdiv(a.F, kGramTile)), int(gram_tiles(a.Co, a.F)),
                 reinterpret_cast<float*>(ws + l.part1)};
  }
  if (g0.tiles + g1.tiles == 0) return SP_OK;
  const int64_t share = cdiv(cdiv(a.rows, l.shares), kGramRows) * kGramRows;
  const int64_t shares = cdiv(a.rows, share);
  ffn_gram<T><<<dim3(unsigned(g0.tiles + g1.tiles), unsigned(shares)), kFfnThreads, 0,
                a.stream>>>(g0, g1, a.rows, share);
  SP_LAUNCHED();
  const int64_t s0 = 2 * int64_t(l.Fp) * a.C, n0 = int64_t(a.F) * a.C;
  if (a.dwg)
    if (int rc = reduce<T>(g0.part, s0, shares, n0, a.dwg, a.stream)) return rc;
  if (a.dwu)
    if (int rc = reduce<T>(g0.part + int64_t(l.Fp) * a.C, s0, shares, n0, a.dwu, a.stream))
      return rc;
  if (a.dwd)
    if (int rc = reduce<T>(g1.part, int64_t(a.Co) * a.F, shares, int64_t(a.Co) * a.F, a.dwd,
                           a.stream))
      return rc;
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
  return dtype == SP_F16 ? forward<_Float16>(a)
                         : dtype == SP_BF16 ? forward<__bf16>(a) : forward<float>(a);
}

extern "C" size_t sp_gated_ffn_bwd_workspace(int32_t dtype, int64_t rows, int64_t C, int64_t F,
                                             int64_t Co) {
  if (check_ffn("gated_ffn_bwd", dtype, rows, C, F, Co, 0) != SP_OK || rows == 0) return 0;
  return backward_layout(dtype, rows, C, F, Co).total;
}

extern "C" int sp_gated_ffn_bwd(const void* dy, int64_t lddy, const void* x, int64_t ldx,
                                int32_t dtype, int64_t rows, int64_t C, const void* w_gate,
                                const void* w_up, int64_t F, const void* w_down, int64_t Co,
                                int32_t act, void* dx, void* dw_gate, void* dw_up, void* dw_down,
                                void* ws, size_t ws_bytes, void* stream) {
  if (int rc = check_ffn("gated_ffn_bwd", dtype, rows, C, F, Co, act)) return rc;
  if (rows == 0) return SP_OK;
  SP_CHECK_ARG(dy && x && w_gate && w_up && w_down && ws, "gated_ffn_bwd: null pointer");
  SP_CHECK_ARG(ldx >= C && lddy >= Co, "gated_ffn_bwd: rows overlap");
  SP_CHECK_ARG(aligned(ws), "gated_ffn_bwd: the workspace must be 16-byte aligned");
  const FfnLayout l = backward_layout(dtype, rows, C, F, Co);
  if (ws_bytes < l.total)
    return set_error(SP_ERR_WORKSPACE, "gated_ffn_bwd: workspace of %zu bytes, needs %zu",
                     ws_bytes, l.total);
  FfnCall a{};
  a.dy = dy, a.x = x, a.wg = w_gate, a.wu = w_up, a.wd = w_down;
  a.ldx = ldx, a.lddy = lddy, a.rows = rows;
  a.C = int(C), a.F = int(F), a.Co = int(Co), a.act = act;
  a.dx = dx, a.dwg = dw_gate, a.dwu = dw_up, a.dwd = dw_down;
  a.ws = ws, a.stream = as_stream(stream);
  return dtype == SP_F16 ? backward<_Float16>(a, l)
                         : dtype == SP_BF16 ? backward<__bf16>(a, l) : backward<float>(a, l);
}
