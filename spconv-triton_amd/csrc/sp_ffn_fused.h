// What the one-kernel passes of the gated feed-forward block share (16-bit rows): chunks of the
// weights in LDS and the operands' orders.
#pragma once

#include "sp_ffn.h"

namespace sp {

constexpr int kFusedRows = 32;  // of a wave's tile

// Row of a 32-row weight block that lies at operand row m: then accumulator register i of lane half b is
// row 16 (i >> 3) + 8 b + (i & 7).
__device__ __forceinline__ int unit_of(int m) {
  return 16 * (m >> 4) + 8 * ((m >> 2) & 1) + 4 * ((m >> 3) & 1) + (m & 3);
}

// Where piece c (16 bytes) of row r lies in LDS rows of PIECES pieces.  Rows of whole 128 bytes are
// permuted by three bits of r, others by two, so that both kinds of reads meet different banks: one
// piece of eight rows (16 bytes a lane), and 32 or 64 bytes of four rows (transposed).
template <int PIECES>
__device__ __forceinline__ int swizzled(int r, int c) {
  if constexpr (PIECES % 8 == 0) return c ^ (((r & 3) << 1) | ((r >> 2) & 1));
  return c ^ ((r & 2) | ((r >> 2) & 1));
}

__device__ const uint4 g_zero_piece = {0, 0, 0, 0};

// 16 bytes from memory to LDS at `to` (the wave's first lane's) + 16 * lane.
__device__ __forceinline__ void copy_piece(const void* from, char* to) {
  __builtin_amdgcn_global_load_lds(
      (const __attribute__((address_space(1))) void*)from,
      (__attribute__((address_space(3))) void*)to, 16, 0, 0);
}

__device__ __forceinline__ void copies_done() {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
}

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
  static constexpr int UP = CP / 8;         // pieces of a Wg or Wu row
  static constexpr int MATRIX = CP * 4;     // pieces of a matrix
  static constexpr int BYTES = 3 * MATRIX * 16;

  __device__ __forceinline__ static const char* up(const char* chunk, int m, int c) {
    return chunk + (m * UP + swizzled<UP>(m & 31, c)) * 16;
  }
  __device__ __forceinline__ static const char* down(const char* chunk, int m, int c) {
    return chunk + (2 * MATRIX + m * 4 + swizzled<4>(m, c)) * 16;
  }

  // Loads a chunk.  Whole chunks of whole matrices take addresses of one part that is the
  // wave's and one that is the lane's for good; the others go by piece, zeros past the ends.
  template <typename T>
  __device__ __forceinline__ static void load(const Weights<T>& w, int f0, char* to) {
    constexpr int THREADS = kFfnThreads, LOADS = (MATRIX + THREADS - 1) / THREADS;
    const int tid = int(threadIdx.x);
    const bool whole = f0 + 32 <= w.Fw && w.C == CP && w.Cow == CP;
#pragma unroll
    for (int j = 0; j < LOADS; ++j) {
      const int i = j * THREADS + tid;
      if (LOADS * THREADS > MATRIX && i >= MATRIX) break;  // (whole waves)
      const int mu = i / UP, cu = swizzled<UP>(mu, i - mu * UP) * 8, fu = unit_of(mu);
      const int md = i >> 2, fd = swizzled<4>(md, i & 3) * 8, cd = (md & ~31) + unit_of(md & 31);
      const unsigned ou = unsigned(fu * w.ldu + cu), od = unsigned(cd * w.ldd + fd);
      const T* bu = w.g + int64_t(f0) * w.ldu;
      const T* bv = w.u + int64_t(f0) * w.ldu;
      const T* bd = w.d + f0;
      char* at = to + (i - (tid & 63)) * 16;
      if (whole) {
        copy_piece(bu + ou, at);
        copy_piece(bv + ou, at + MATRIX * 16);
        copy_piece(bd + od, at + 2 * MATRIX * 16);
      } else {
        const bool in = f0 + fu < w.Fw && cu < w.C;
        const void* zero = &g_zero_piece;
        copy_piece(in ? static_cast<const void*>(bu + ou) : zero, at);
        copy_piece(in ? static_cast<const void*>(bv + ou) : zero, at + MATRIX * 16);
        copy_piece(cd < w.Cow && f0 + fd < w.Fw ? static_cast<const void*>(bd + od) : zero,
                   at + 2 * MATRIX * 16);
      }
    }
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

// 32 hidden units of a wave's 32 rows: their gate and up values, ...
template <typename T, int CP>
__device__ __forceinline__ void fused_up(const char* chunk,
                                         const typename Mfma<T>::frag (&x)[CP / 16], floatx16& g,
                                         floatx16& u) {
  using frag = typename Mfma<T>::frag;
  const int lane = int(threadIdx.x) & 31, half = (int(threadIdx.x) >> 5) & 1;
#pragma unroll
  for (int i = 0; i < 16; ++i) g[i] = u[i] = 0.f;
#pragma unroll
  for (int k = 0; k < CP / 16; ++k) {
    const frag fg = *reinterpret_cast<const frag*>(Chunk<CP>::up(chunk, lane, 2 * k + half));
    const frag fu = *reinterpret_cast<const frag*>(Chunk<CP>::up(chunk, lane + 32, 2 * k + half));
    Mfma<T>::mma(fg, x[k], g);
    Mfma<T>::mma(fu, x[k], u);
  }
}

// ... and what they add to y.
template <typename T, int CP>
__device__ __forceinline__ void fused_down(const char* chunk,
                                           const typename Mfma<T>::frag (&h)[2],
                                           floatx16 (&y)[CP / 32]) {
  using frag = typename Mfma<T>::frag;
  const int lane = int(threadIdx.x) & 31, half = (int(threadIdx.x) >> 5) & 1;
#pragma unroll
  for (int t = 0; t < CP / 32; ++t)
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const frag fd = *reinterpret_cast<const frag*>(
          Chunk<CP>::down(chunk, t * 32 + lane, 2 * s + half));
      Mfma<T>::mma(fd, h[s], y[t]);
    }
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
