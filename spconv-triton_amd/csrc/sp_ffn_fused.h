// What the one-kernel passes of the gated feed-forward block share (16-bit rows): chunks of the
// weights in LDS and the operands' orders.
#pragma once

#include "sp_ffn.h"

namespace sp {

constexpr int kFusedRows = 32;  // of a wave's tile

// The weights as they lie in memory: rows of ldu (g, u) and ldd (d) elements.
template <typename T>
struct Weights {
  const T *g, *u, *d;
  int F, Co;        // hidden units, channels out
  int C, Fw, Cow;   // extents in memory, where it has zeros past F, Co and x's channels: multiples of 8
  int ldu, ldd;
};

// A chunk of the weights in LDS: 32 rows of Wg, 32 of Wu and CP of Wd (32 hidden units each), CP * 64
// bytes each.
template <int CP>
struct Chunk {
  static constexpr int UP = CP / 8;      // pieces of a Wg or Wu row
  static constexpr int MATRIX = CP * 4;  // pieces of a matrix
  static constexpr int BYTES = 3 * MATRIX * 16;

  __device__ __forceinline__ static const char* up(const char* chunk, int which, int m, int c) {
    return chunk + which * (MATRIX * 16) + (m * UP + swizzled<UP>(m, c)) * 16;
  }
  __device__ __forceinline__ static const char* down(const char* chunk, int m, int c) {
    return chunk + 2 * (MATRIX * 16) + (m * 4 + swizzled<4>(m, c)) * 16;
  }

  // Loads a chunk.  Whole chunks of whole matrices take addresses of one part that is the wave's
  // and one that is the lane's for good; the others go by piece, with zeros past the ends.
  template <typename T>
  __device__ __forceinline__ static void load(const Weights<T>& w, int f0, char* to) {
    constexpr int ROUNDS = (MATRIX + kFfnThreads - 1) / kFfnThreads;
    const int tid = int(threadIdx.x);
    const bool whole = f0 + 32 <= w.Fw && w.C == CP && w.Cow == CP;
#pragma unroll
    for (int j = 0; j < ROUNDS; ++j) {
      const int i = j * kFfnThreads + tid;
      if (MATRIX % kFfnThreads != 0 && j * kFfnThreads + wave_of() * 64 >= MATRIX) break;
      const int mu = i / UP, cu = swizzled<UP>(mu, i - mu * UP) * 8, fu = unit_of(mu);
      const int md = i >> 2, fd = swizzled<4>(md, i & 3) * 8, cd = (md & ~31) + unit_of(md & 31);
      const unsigned ou = unsigned(fu * w.ldu + cu), od = unsigned(cd * w.ldd + fd);
      const T* bg = w.g + int64_t(f0) * w.ldu;
      const T* bu = w.u + int64_t(f0) * w.ldu;
      const T* bd = w.d + f0;
      char* at = to + (j * kFfnThreads + wave_of() * 64) * 16;
      if (whole) {
        copy_piece(bg + ou, at);
        copy_piece(bu + ou, at + MATRIX * 16);
        copy_piece(bd + od, at + 2 * MATRIX * 16);
      } else {
        const bool in = f0 + fu < w.Fw && cu < w.C, ind = cd < w.Cow && f0 + fd < w.Fw;
        const void* zero = &g_zero_piece;
        copy_piece(in ? static_cast<const void*>(bg + ou) : zero, at);
        copy_piece(in ? static_cast<const void*>(bu + ou) : zero, at + MATRIX * 16);
        copy_piece(ind ? static_cast<const void*>(bd + od) : zero, at + 2 * MATRIX * 16);
      }
    }
  }
};

// The chunks of a call's weights, two of them in LDS: `next` waits until a chunk is there, for all waves' loads
// of it, and starts the following one into the buffer that all waves have left.
template <typename T, int CP>
struct Chunks {
  using C = Chunk<CP>;
  const Weights<T>& w;
  char* lds;
  int f = 0, at = 0;
  __device__ __forceinline__ Chunks(const Weights<T>& w_, char* lds_) : w(w_), lds(lds_) {
    C::load(w, 0, lds);
  }
  __device__ __forceinline__ const char* next() {
    loads_in_flight<0>();
    __syncthreads();
    f += 32;
    const char* chunk = lds + at * C::BYTES;
    at ^= 1;
    if (f < w.F) C::load(w, f, lds + at * C::BYTES);
    return chunk;
  }
};

// A lane's 8 values of a row; past n zeros.
template <typename T>
__device__ __forceinline__ typename Mfma<T>::frag row_piece(const T* row, int c, int n, bool vec) {
  typename Mfma<T>::frag f = {};
  if (vec && c + 8 <= n) return *reinterpret_cast<const typename Mfma<T>::frag*>(row + c);
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (c + i < n) f[i] = row[c + i];
  return f;
}

// 32 rows of x as operands: row r is the lane's.
template <typename T, int CP>
__device__ __forceinline__ void load_rows(const Rows<T>& x, int64_t r,
                                          typename Mfma<T>::frag (&f)[CP / 16]) {
  const int half = (int(threadIdx.x) >> 5) & 1;
#pragma unroll
  for (int k = 0; k < CP / 16; ++k) {
    f[k] = typename Mfma<T>::frag{};
    if (r < x.n) f[k] = row_piece<T>(x.p + r * x.ld, k * 16 + half * 8, x.K, x.vec);
  }
}

// Operands of 32 hidden units from f0 on, with zeros from F on: the weights there are zeros, but an
// infinity of x or dy makes their values NaN, which would meet other zeros in the next product.
template <typename Frag>
__device__ __forceinline__ void end_units(Frag (&h)[2], int f0, int F) {
  const int half = (int(threadIdx.x) >> 5) & 1;
#pragma unroll
  for (int i = 0; i < 16; ++i)
    if (f0 + 16 * (i >> 3) + 8 * half + (i & 7) >= F) h[i >> 3][i & 7] = 0;
}

template <typename T>
struct FragPair {
  typename Mfma<T>::frag a, b;
};

// 32 hidden units of a wave's 32 rows: their gate and up values, ...
template <typename T, int CP>
__device__ __forceinline__ void fused_up(const char* chunk,
                                         const typename Mfma<T>::frag (&x)[CP / 16], floatx16& g,
                                         floatx16& u) {
  using frag = typename Mfma<T>::frag;
  const int lane = int(threadIdx.x) & 31, half = (int(threadIdx.x) >> 5) & 1;
  auto read = [&](int k) {
    return FragPair<T>{
        *reinterpret_cast<const frag*>(Chunk<CP>::up(chunk, 0, lane, 2 * k + half)),
        *reinterpret_cast<const frag*>(Chunk<CP>::up(chunk, 1, lane, 2 * k + half))};
  };
  Batched<FragPair<T>, CP / 16, 4> w;
  w.start(read);
#pragma unroll
  for (int i = 0; i < 16; ++i) g[i] = u[i] = 0.f;
  w.run(read, [&](int k, const FragPair<T>& f) {
    Mfma<T>::mma(f.a, x[k], g);
    Mfma<T>::mma(f.b, x[k], u);
  });
}

template <int N>
__device__ __forceinline__ void clear_rows(floatx16 (&y)[N]) {
#pragma unroll
  for (int t = 0; t < N; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) y[t][i] = 0.f;
}

// (sp_ffn_fused.hip) The weights of a call; where their rows do not start at multiples of 16 bytes,
// copies made in ws (fused_weights_bytes).
template <typename T>
int fused_weights(const FfnCall& c, T* ws, Weights<T>& w);

}  // namespace sp
