// Products of rows with weight rows on tiles of 32x32 MFMAs, and of rows with rows: what the feed-forward
// block's kernels and the linear layer's share.
#pragma once

#include "sp_ffn.h"

namespace sp {

// ---- rows with weight rows -------------------------------------------------------
// A workgroup's tile: WX x WW waves, each with XT x WT tiles of 32 rows of x and of 32 weight rows.  The
// MFMA's rows are the weights' and its columns x's, so that a lane holds one row of x and
// neighbouring outputs of it, which it writes in 16 bytes.  Larger tiles read less: with 128 rows and
// 64 hidden units a workgroup the L2 hands out 2.2 GB for the gate and up products of 50k rows of 512
// channels and 1 376 hidden units, with 256 and 128 half of that, 307 and 200 us (700 TFLOP/s bf16,
// where the library's product of these sizes without the gate reaches 500).  What bounds the large
// tiles then: the eight waves of a CU meet at a barrier each stage and read its first operands with
// the matrix cores idle (these work for 44 % of the time that a CU is busy), and 50k rows leave the last
// round of workgroups half empty (1.5 rounds for w_down).  Four stages of half the length, with
// three in flight: 7 % slower.
template <int XT_, int WT_, int WX_, int WW_>
struct TileShape {
  static constexpr int XT = XT_, WT = WT_, WX = WX_, WW = WW_;
  static constexpr int X = 32 * XT * WX, W = 32 * WT * WW;  // rows of a stage
  static constexpr int THREADS = 64 * WX * WW;
  static constexpr int PIECES = (X + W) * kStagePieces, BYTES = PIECES * 16;
};
using ThinTile = TileShape<1, 2, 2, 2>;    // 64 x 128, four waves
using SmallTile = TileShape<2, 2, 2, 2>;   // 128 x 128, four waves, for operands that go through registers
using QuickTile = TileShape<1, 2, 4, 2>;   // 128 x 128, eight waves, two such workgroups a CU
using NarrowTile = TileShape<1, 3, 4, 1>;  // 128 x 96, four waves
using LongTile = TileShape<2, 2, 4, 2>;    // 256 x 128, eight waves
using LargeTile = TileShape<2, 4, 4, 2>;   // 256 x 256, eight waves

// Weight row of operand row m: 16-bit lanes then hold eight neighbouring outputs in eight
// registers, fp32 ones (as it is) four in four.
template <typename T>
__device__ __forceinline__ int weight_row(int m) {
  return sizeof(T) == 2 ? (m & ~31) + unit_of(m & 31) : m;
}

// A stage: 128 bytes of X rows of x and of W weight rows, from w, or the first half of them from w and
// the other from w2.  ASYNC: straight to LDS, for operands whose rows start at multiples of 16 bytes
// and have whole pieces; rows past an operand's end are its last one, whose products no output
// takes up (a hidden column past F meets zeros).  Else through registers, with zeros past the ends.
template <typename T, typename S, bool ASYNC>
struct Stage {
  using frag = typename Mfma<T>::frag;
  static constexpr int V = Mfma<T>::V, N = S::PIECES / S::THREADS;
  const T* from[N];  // of this thread's pieces, at k
  frag r[ASYNC ? 1 : N];
  unsigned in;  // whether a piece's row exists
  int k, K;

  // LDS slot i = j THREADS + thread holds piece i % 8 (permuted) of operand row i / 8
  __device__ __forceinline__ static int first_k() {
    const int row = int(threadIdx.x) >> 3;  // (j THREADS / 8 rows further the order is the same)
    return swizzled<8>(row, int(threadIdx.x) & 7) * V;
  }
  __device__ __forceinline__ Stage(const Rows<T>& x, int64_t x0, const Rows<T>& w,
                                   const Rows<T>* w2, int64_t w0)
      : in(0u), k(first_k()), K(x.K) {
    static_assert(S::THREADS % 256 == 0 && S::X * 8 % S::THREADS == 0 &&
                      S::W * 8 % S::THREADS == 0, "whole rounds of an operand");
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int row = (j * S::THREADS + int(threadIdx.x)) >> 3;
      const bool second = w2 && j * S::THREADS >= (S::X + S::W / 2) * 8;
      const bool weights = j * S::THREADS >= S::X * 8;
      const Rows<T>& a = second ? *w2 : weights ? w : x;
      int64_t at = !weights ? x0 + row
                            : w0 + weight_row<T>(row - S::X - (second ? S::W / 2 : 0));
      if (at < a.n)
        in |= 1u << j;
      else
        at = a.n - 1;
      from[j] = a.p + at * a.ld + k;
    }
  }
  // tail: the operands end within this stage
  __device__ __forceinline__ void start(const Rows<T>& x, const Rows<T>& w, char* lds, bool tail) {
    const int at = wave_of() * 64;
    if (ASYNC && !tail) {
#pragma unroll
      for (int j = 0; j < N; ++j) {
        copy_piece(from[j], lds + (j * S::THREADS + at) * 16);
        from[j] += kStagePieces * V;
      }
      k += kStagePieces * V;
      return;
    }
#pragma unroll
    for (int j = 0; j < N; ++j) {
      if constexpr (ASYNC) {
        copy_piece(k < K ? static_cast<const void*>(from[j]) : &g_zero_piece,
                   lds + (j * S::THREADS + at) * 16);
      } else {
        const bool vec = j * S::THREADS >= S::X * 8 ? w.vec : x.vec;
        r[j] = frag{};
        if (in >> j & 1) {
          if (vec && k + V <= K) {
            r[j] = *reinterpret_cast<const frag*>(from[j]);
          } else {
#pragma unroll
            for (int i = 0; i < V; ++i)
              if (k + i < K) r[j][i] = from[j][i];
          }
        }
      }
      from[j] += kStagePieces * V;
    }
    k += kStagePieces * V;
  }
  __device__ __forceinline__ void finish(char* lds) const {
    if constexpr (ASYNC) {
      loads_in_flight<0>();
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j)
        *reinterpret_cast<frag*>(lds + (j * S::THREADS + int(threadIdx.x)) * 16) = r[j];
    }
  }
  __device__ __forceinline__ static frag read(const char* lds, int row, int c) {
    return *reinterpret_cast<const frag*>(lds + (row * 8 + swizzled<8>(row, c)) * 16);
  }
};

template <typename T, int M, int N>
struct Operands {
  typename Mfma<T>::frag x[M], w[N];
};

struct Nothing {
  __device__ __forceinline__ void operator()() const {}
};

// acc[j][i] += the products of x rows xrow + 32 j .. + 31 and weight rows wrow[i] .. + 31 of the stage
// over all of K.  `meanwhile` runs while the first stage is on its way.
template <typename T, typename S, bool ASYNC, int NW, typename F = Nothing>
__device__ __forceinline__ void products(const Rows<T>& x, int64_t x0, const Rows<T>& w,
                                         const Rows<T>* w2, int64_t w0, const int (&wrow)[NW],
                                         int xrow, char* lds, floatx16 (&acc)[S::XT][NW],
                                         F&& meanwhile = F()) {
  using Stg = Stage<T, S, ASYNC>;
  constexpr int STEP = kStagePieces * Mfma<T>::V;
  const int lane = int(threadIdx.x) & 31, half = (int(threadIdx.x) >> 5) & 1;
  Stg stage(x, x0, w, w2, w0);
  const int steps = (x.K + STEP - 1) / STEP;
  stage.start(x, w, lds, x.K < STEP);
  meanwhile();
  for (int s = 0; s < steps; ++s) {
    char* buf = lds + (s & 1) * S::BYTES;
    stage.finish(buf);
    __syncthreads();  // (the other buffer's readers are past their previous barrier)
    if (s + 1 < steps)
      stage.start(x, w, lds + ((s + 1) & 1) * S::BYTES, (s + 2) * STEP > x.K);
    auto read = [&](int c) {
      Operands<T, S::XT, NW> f;
#pragma unroll
      for (int j = 0; j < S::XT; ++j) f.x[j] = Stg::read(buf, xrow + 32 * j + lane, 2 * c + half);
#pragma unroll
      for (int i = 0; i < NW; ++i) f.w[i] = Stg::read(buf, S::X + wrow[i] + lane, 2 * c + half);
      return f;
    };
    Batched<Operands<T, S::XT, NW>, kStagePieces / 2, 1> steps_of;
    steps_of.start(read);
    steps_of.run(read, [&](int, const Operands<T, S::XT, NW>& f) {
#pragma unroll
      for (int j = 0; j < S::XT; ++j)
#pragma unroll
        for (int i = 0; i < NW; ++i) Mfma<T>::mma(f.w[i], f.x[j], acc[j][i]);
    });
  }
  __syncthreads();
}

template <int M, int N>
__device__ __forceinline__ void clear(floatx16 (&acc)[M][N]) {
#pragma unroll
  for (int j = 0; j < M; ++j)
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int k = 0; k < 16; ++k) acc[j][i][k] = 0.f;
}

// f(register, column) for the lane's outputs of an accumulator of columns from c0 on (write_piece_row's order).
template <typename T, typename F>
__device__ __forceinline__ void each_column(int c0, F&& f) {
  constexpr int V = Mfma<T>::V;
  const int half = (int(threadIdx.x) >> 5) & 1;
#pragma unroll
  for (int i = 0; i < 16; ++i) f(i, c0 + i / V * 2 * V + V * half + i % V);
}

// The lane's outputs of an accumulator: pieces of V of row r, columns c0 .. c0 + 31, those below n.
// value(i): of register i, or with a residual what is added to it.
template <typename T, typename F>
__device__ __forceinline__ void write_piece_row(T* out, int64_t ld, int64_t r, int64_t rows,
                                                int c0, int n, bool vec, F&& value) {
  using frag = typename Mfma<T>::frag;
  constexpr int V = Mfma<T>::V;
  const int half = (int(threadIdx.x) >> 5) & 1;
  if (r >= rows) return;
#pragma unroll
  for (int p = 0; p < 16 / V; ++p) {
    const int c = c0 + 2 * V * p + V * half;
    if (c >= n) continue;
    frag f;
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = from_f32<T>(value(p * V + i, c + i));
    T* to = out + r * ld + c;
    if (vec && c + V <= n) {
      *reinterpret_cast<frag*>(to) = f;
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (c + i < n) to[i] = f[i];
    }
  }
}

// The place of this workgroup among `total`: consecutive workgroups go to the eight XCDs in turn; here each XCD
// gets an eighth of the places in a row, so that tiles which share rows meet in one L2.
__device__ __forceinline__ int64_t place_of(int64_t total, int64_t id = blockIdx.x) {
  const int64_t per = (total + 7) >> 3;
  const int64_t k = (id >> 3) < per ? (id & 7) * per + (id >> 3) : total;
  return k < total ? k : -1;
}

// ---- rows with rows (weight gradients) -------------------------------------------
constexpr int kGramStage = 128;  // bytes of a column in a stage

template <typename T>
constexpr int gram_rows() { return kGramStage / int(sizeof(T)); }

typedef short short4v __attribute__((ext_vector_type(4)));

// COLS columns of a stage in LDS.  16-bit rows hold their 16-byte pieces permuted: the four rows that 32 lanes
// read at once, 64 bytes of each, fall on different banks.
template <typename T, int COLS, int THREADS>
struct GramStage {
  using frag = typename Mfma<T>::frag;
  static constexpr int V = Mfma<T>::V, PER = COLS / V, ROWS = gram_rows<T>();
  static constexpr int N = ROWS * PER / THREADS;
  frag r[N];

  __device__ __forceinline__ static int slot(int row, int piece) {
    if constexpr (sizeof(T) == 4 || COLS == 96) return piece;  // (rows of 192 bytes fall apart by themselves)
    if constexpr (COLS % 128 == 0) return piece ^ ((row & 3) << 2);
    return piece ^ ((row & 3) << 1);
  }
  __device__ __forceinline__ void load(const T* p, int64_t ld, int vec, int64_t m, int64_t hi,
                                       int c0, int n) {
    if (vec && n % V == 0) {
      // Whole pieces: no branch of lanes, behind which each load would wait for the one before it (the gradient of
      // 1024 x 256 bf16 weights over 75k rows: 152 us with one, 77 without).  Rows past the end are zeroed on
      // their way to LDS; columns past it meet outputs that are not written.
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const int i = int(threadIdx.x) + j * THREADS, row = i / PER;
        const int c = c0 + (i - row * PER) * V;
        const int64_t at = m + row < hi ? m + row : hi - 1;
        r[j] = *reinterpret_cast<const frag*>(p + at * ld + (c < n ? c : n - V));
      }
      return;
    }
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int i = int(threadIdx.x) + j * THREADS, row = i / PER;
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
  // left: rows that there are from the stage's first on
  __device__ __forceinline__ void store(char* lds, int64_t left) {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int i = int(threadIdx.x) + j * THREADS, row = i / PER;
      if (row >= left) r[j] = frag{};
      *reinterpret_cast<frag*>(lds + (row * PER + slot(row, i - row * PER)) * 16) = r[j];
    }
  }
  // s += what was stored: a thread's pieces are of the same columns, thread % PER of them
  __device__ __forceinline__ void sum(float (&s)[V]) const {
    static_assert(THREADS % PER == 0, "a thread's columns");
#pragma unroll
    for (int j = 0; j < N; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) s[i] += to_f32(r[j][i]);
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

// ---- a few rows ------------------------------------------------------------------
constexpr int kFewRows = 4;  // a weight row's dot products rather than tiles

// The sums of a over `lanes` lanes, on each of them.
template <int N>
__device__ __forceinline__ void sum_lanes(float (&a)[N], int lanes) {
  for (int off = lanes >> 1; off >= 1; off >>= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) a[i] += __shfl_xor(a[i], off, 64);
}

template <typename T>
__device__ __forceinline__ typename Mfma<T>::frag piece_of(const Rows<T>& a, int64_t r, int k) {
  typename Mfma<T>::frag f = {};
  constexpr int V = Mfma<T>::V;
  const T* p = a.p + r * a.ld + k;
  if (a.vec && k + V <= a.K) return *reinterpret_cast<const typename Mfma<T>::frag*>(p);
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (k + i < a.K) f[i] = p[i];
  return f;
}

// ---- host ------------------------------------------------------------------------
// Lanes of an output: as many as its weight row has pieces, up to a wave.
inline int few_lanes(int64_t K, int V) {
  int l = 0;
  while (l < 6 && (int64_t(V) << l) < K) ++l;
  return l;
}

template <typename T>
bool whole(const Rows<T>& a) { return a.vec && a.K % Mfma<T>::V == 0; }

// Workgroups of tiles of S: whole eights (place_of).
template <typename S>
int64_t tile_groups(int64_t rows, int64_t cols) {
  return cdiv(cdiv(rows, S::X) * cols, 8) * 8;
}

// The larger tiles where they still give every CU a workgroup or more: below that the smaller ones
// spread the work further.
template <typename S>
bool fills(int64_t rows, int64_t cols) { return cdiv(rows, S::X) * cols >= 256; }

}  // namespace sp
