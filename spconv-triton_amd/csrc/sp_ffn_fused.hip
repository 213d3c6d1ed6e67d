// The gated feed-forward block's forward pass in one kernel, for 16-bit rows of at most 256
// channels: hidden values exist in registers only.
//
// Everything is computed transposed, with the rows of x as the MFMAs' columns:
//   G' = Wg x', U' = Wu x', H' = act(G') * U', Y' += Wd H'
// A wave keeps 32 rows of x as operands and their Y' as accumulators, and goes through the hidden
// units 32 at a time.  Lane l of an accumulator holds row l & 31 of x and 16 hidden units, and an
// MFMA operand is the same row with 8 of them: H' goes straight from the accumulators of the
// first products into the operand of the second.  For its units to be the ones that Wd's operand
// has, operand row m of a 32-row block holds weight row unit_of(m), in LDS and for Wd's rows too (so that a lane
// ends with 8 neighbouring channels of y).
//
// The weights pass through LDS in chunks of 32 hidden units, loaded by direct loads to LDS while the
// chunk before is in use, and are read by all four waves.
#include "sp_ffn.h"

namespace sp {

constexpr int kFusedRows = 32;  // of a wave's tile

// Row of a 32-row weight block that lies at operand row m: then accumulator register i of lane half b is
// row 16 (i >> 3) + 8 b + (i & 7).
__device__ __forceinline__ int unit_of(int m) {
  return 16 * (m >> 4) + 8 * ((m >> 2) & 1) + 4 * ((m >> 3) & 1) + (m & 3);
}

// Where piece c (16 bytes) of row r lies in LDS rows of PIECES pieces: rows whose pitch is a
// multiple of 128 bytes differ in the low three bits, others in two, so that eight
// rows' pieces of one column lie on different banks.
template <int PIECES>
__device__ __forceinline__ int swizzled(int r, int c) {
  return PIECES % 8 == 0 ? c ^ (r & 7) : c ^ ((r >> 1) & 3);
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

template <typename T>
struct FusedArgs {
  const T *x, *wg, *wu, *wd, *residual;
  T* y;
  int64_t ldx, ldr, rows;
  int C, F, Co;    // as the rows have them
  int ldu, ldd;    // elements from row to row of wg and wu, and of wd
  int Cw, Fw, Cow; // extents of the weights as they lie there: multiples of 8
  int vec_x, vec_y, vec_r;
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

// CP: channels, rounded up to 32, of x and y.  R: tiles of 32 rows of a wave.
template <typename T, int ACT, int CP, int R, int MINW>
__global__ __launch_bounds__(kFfnThreads, MINW) void ffn_fused(FusedArgs<T> a) {
  using frag = typename Mfma<T>::frag;
  constexpr int UP = CP / 8;              // pieces of a Wg or Wu row
  constexpr int PIECES = 64 * UP + CP * 4;  // of a chunk: Wg and Wu 32 rows each, Wd CP rows
  constexpr int LOADS = (PIECES + kFfnThreads - 1) / kFfnThreads;
  __shared__ __attribute__((aligned(16))) char lds[2][PIECES * 16];
  const int tid = int(threadIdx.x), wave = tid >> 6, lane = tid & 31, half = (tid >> 5) & 1;
  const int64_t r0 = (int64_t(blockIdx.x) * 4 + wave) * (kFusedRows * R) + lane;

  auto load_chunk = [&](int f0, char* to) {
#pragma unroll
    for (int j = 0; j < LOADS; ++j) {
      const int i = j * kFfnThreads + tid;
      if (LOADS * kFfnThreads > PIECES && i >= PIECES) break;  // (whole waves)
      const T* from;
      bool in;
      if (i < 64 * UP) {
        const int m = i / UP, c = swizzled<UP>(m, i - m * UP) * 8;
        const int f = f0 + unit_of(m & 31);
        in = f < a.Fw && c < a.Cw;
        from = (m < 32 ? a.wg : a.wu) + int64_t(f) * a.ldu + c;
      } else {
        const int k = i - 64 * UP, m = k >> 2, f = f0 + swizzled<4>(m, k & 3) * 8;
        const int co = (m & ~31) + unit_of(m & 31);
        in = co < a.Cow && f < a.Fw;
        from = a.wd + int64_t(co) * a.ldd + f;
      }
      copy_piece(in ? static_cast<const void*>(from) : &g_zero_piece, to + (i - (tid & 63)) * 16);
    }
  };

  load_chunk(0, lds[0]);
  frag x[R][CP / 16];
#pragma unroll
  for (int q = 0; q < R; ++q) {
    const int64_t r = r0 + q * kFusedRows;
#pragma unroll
    for (int k = 0; k < CP / 16; ++k)
      x[q][k] = r < a.rows ? row_piece<T>(a.x + r * a.ldx, k * 16 + half * 8, a.C, a.vec_x)
                           : frag{};
  }
  floatx16 y[R][CP / 32];
#pragma unroll
  for (int q = 0; q < R; ++q)
#pragma unroll
    for (int t = 0; t < CP / 32; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) y[q][t][i] = 0.f;
  copies_done();

  int buf = 0;
  for (int f0 = 0; f0 < a.F; f0 += 32, buf ^= 1) {
    if (f0 + 32 < a.F) load_chunk(f0 + 32, lds[buf ^ 1]);
    const char* up = lds[buf];
    const char* down = up + 64 * UP * 16;
    floatx16 g[R], u[R];
#pragma unroll
    for (int q = 0; q < R; ++q)
#pragma unroll
      for (int i = 0; i < 16; ++i) g[q][i] = u[q][i] = 0.f;
#pragma unroll
    for (int k = 0; k < CP / 16; ++k) {
      const int c = swizzled<UP>(lane, 2 * k + half);
      const frag fg = *reinterpret_cast<const frag*>(up + (lane * UP + c) * 16);
      const frag fu = *reinterpret_cast<const frag*>(up + ((lane + 32) * UP + c) * 16);
#pragma unroll
      for (int q = 0; q < R; ++q) {
        Mfma<T>::mma(fg, x[q][k], g[q]);
        Mfma<T>::mma(fu, x[q][k], u[q]);
      }
    }
    frag h[R][2];
#pragma unroll
    for (int q = 0; q < R; ++q)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float value, slope;
        gate<true, ACT>(g[q][i], value, slope);
        h[q][i >> 3][i & 7] = T(value * u[q][i]);
      }
#pragma unroll
    for (int t = 0; t < CP / 32; ++t)
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const int m = t * 32 + lane;
        const frag fd = *reinterpret_cast<const frag*>(
            down + (m * 4 + swizzled<4>(m, 2 * s + half)) * 16);
#pragma unroll
        for (int q = 0; q < R; ++q) Mfma<T>::mma(fd, h[q][s], y[q][t]);
      }
    copies_done();
  }

#pragma unroll
  for (int q = 0; q < R; ++q) {
    const int64_t r = r0 + q * kFusedRows;
    if (r >= a.rows) continue;
#pragma unroll
    for (int t = 0; t < CP / 32; ++t)
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const int c = t * 32 + 16 * s + 8 * half;
        if (c >= a.Co) continue;
        frag res = {};
        if (a.residual) res = row_piece<T>(a.residual + r * a.ldr, c, a.Co, a.vec_r);
        frag o;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float v = y[q][t][8 * s + i];
          o[i] = T(a.residual ? v + float(res[i]) : v);
        }
        T* to = a.y + r * a.Co + c;
        if (a.vec_y) {
          *reinterpret_cast<frag*>(to) = o;
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (c + i < a.Co) to[i] = o[i];
        }
      }
  }
}

// dst [rows_out][ldd] = src [rows][cols] with zeros around, both wg and wu or wd alone.
template <typename T>
__global__ __launch_bounds__(kFfnThreads) void ffn_pad(const T* __restrict__ s0,
                                                       const T* __restrict__ s1,
                                                       const T* __restrict__ s2, int C, int F,
                                                       int Co, int Cp, int Fp, int Cop,
                                                       T* __restrict__ dst) {
  const int n0 = Fp * Cp, n = 2 * n0 + Cop * Fp;
  for (int i = int(blockIdx.x) * kFfnThreads + int(threadIdx.x); i < n;
       i += int(gridDim.x) * kFfnThreads) {
    T v = T(0.f);
    if (i < 2 * n0) {
      const int k = i < n0 ? i : i - n0, f = k / Cp, c = k - f * Cp;
      if (f < F && c < C) v = (i < n0 ? s0 : s1)[int64_t(f) * C + c];
    } else {
      const int k = i - 2 * n0, c = k / Fp, f = k - c * Fp;
      if (f < F && c < Co) v = s2[int64_t(c) * F + f];
    }
    dst[i] = v;
  }
}

static int up8(int64_t v) { return int(cdiv(v, 8) * 8); }

bool fused_forward_takes(int32_t dtype, int64_t rows, int64_t C, int64_t F, int64_t Co) {
  return dtype != SP_F32 && C <= kFusedWidth && Co <= kFusedWidth && rows >= 1;
}

size_t fused_forward_workspace(int64_t C, int64_t F, int64_t Co) {
  return (2 * size_t(up8(F)) * up8(C) + size_t(up8(Co)) * up8(F)) * 2;
}

template <typename T, int CP, int R, int MINW>
static int launch_fused(const FusedArgs<T>& a, int act, hipStream_t s) {
  const int64_t blocks = cdiv(a.rows, 4 * kFusedRows * R);
  SP_CHECK_ARG(blocks <= kMaxGridX, "gated_ffn: too many rows");
  using Kern = void (*)(FusedArgs<T>);
  const Kern kern = act == kActSilu   ? Kern(ffn_fused<T, kActSilu, CP, R, MINW>)
                    : act == kActGelu ? Kern(ffn_fused<T, kActGelu, CP, R, MINW>)
                                      : Kern(ffn_fused<T, kActRelu, CP, R, MINW>);
  kern<<<unsigned(blocks), kFfnThreads, 0, s>>>(a);
  SP_LAUNCHED();
  return SP_OK;
}

template <typename T>
static int run_fused(const FfnCall& c) {
  FusedArgs<T> a{};
  a.x = static_cast<const T*>(c.x);
  a.residual = static_cast<const T*>(c.residual);
  a.y = static_cast<T*>(c.y);
  a.ldx = c.ldx, a.ldr = c.ldr, a.rows = c.rows;
  a.C = c.C, a.F = c.F, a.Co = c.Co;
  a.vec_x = aligned(c.x) && c.ldx % 8 == 0;
  a.vec_y = aligned(c.y) && c.Co % 8 == 0;
  a.vec_r = aligned(c.residual) && c.ldr % 8 == 0;
  a.wg = static_cast<const T*>(c.wg);
  a.wu = static_cast<const T*>(c.wu);
  a.wd = static_cast<const T*>(c.wd);
  a.ldu = a.Cw = c.C;
  a.ldd = a.Fw = c.F;
  a.Cow = c.Co;
  // weights whose rows do not start at multiples of 16 bytes are copied first
  if (c.C % 8 != 0 || c.F % 8 != 0 || !aligned(c.wg) || !aligned(c.wu) || !aligned(c.wd)) {
    const int Cp = up8(c.C), Fp = up8(c.F), Cop = up8(c.Co);
    T* w = static_cast<T*>(c.ws);
    ffn_pad<T><<<unsigned(cdiv(int64_t(Fp) * (2 * Cp + Cop), kFfnThreads * 4)), kFfnThreads, 0,
                 c.stream>>>(a.wg, a.wu, a.wd, c.C, c.F, c.Co, Cp, Fp, Cop, w);
    SP_LAUNCHED();
    a.wg = w;
    a.wu = w + int64_t(Fp) * Cp;
    a.wd = w + 2 * int64_t(Fp) * Cp;
    a.ldu = a.Cw = Cp;
    a.ldd = a.Fw = Fp;
    a.Cow = Cop;
  }
  const int widest = c.C > c.Co ? c.C : c.Co;
  if (widest <= 32) return launch_fused<T, 32, 1, 4>(a, c.act, c.stream);
  if (widest <= 64) return launch_fused<T, 64, 1, 4>(a, c.act, c.stream);
  if (widest <= 96) return launch_fused<T, 96, 1, 3>(a, c.act, c.stream);
  if (widest <= 128) return launch_fused<T, 128, 1, 2>(a, c.act, c.stream);
  if (widest <= 160) return launch_fused<T, 160, 1, 2>(a, c.act, c.stream);
  if (widest <= 192) return launch_fused<T, 192, 1, 2>(a, c.act, c.stream);
  return launch_fused<T, 256, 1, 1>(a, c.act, c.stream);
}

int fused_forward(int32_t dtype, const FfnCall& a) {
  return dtype == SP_F16 ? run_fused<_Float16>(a) : run_fused<__bf16>(a);
}

}  // namespace sp
