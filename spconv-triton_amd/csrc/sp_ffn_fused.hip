// The gated feed-forward block's forward pass in one kernel, for 16-bit rows of at most 192
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
//
// h is rounded to the rows' type on its way into the last products, as a stored h would be; the sums
// of y are fp32 and the residual is added to them before their one rounding.
#include "sp_ffn_fused.h"

namespace sp {

template <typename T>
struct FusedArgs {
  Rows<T> x, residual;
  Weights<T> w;
  T* y;
  int vec_y;
};

template <typename T, int CP>
__device__ __forceinline__ void fused_store(const FusedArgs<T>& a, int64_t r,
                                            const floatx16 (&y)[CP / 32]) {
  using frag = typename Mfma<T>::frag;
  const int half = (int(threadIdx.x) >> 5) & 1;
  if (r >= a.x.n) return;
#pragma unroll
  for (int t = 0; t < CP / 32; ++t)
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int c = t * 32 + 16 * s + 8 * half;
      if (c >= a.w.Co) continue;
      frag res = {};
      if (a.residual.p)
        res = row_piece<T>(a.residual.p + r * a.residual.ld, c, a.w.Co, a.residual.vec);
      frag o;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float v = y[t][8 * s + i];
        o[i] = T(a.residual.p ? v + float(res[i]) : v);
      }
      T* to = a.y + r * a.w.Co + c;
      if (a.vec_y) {
        *reinterpret_cast<frag*>(to) = o;
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (c + i < a.w.Co) to[i] = o[i];
      }
    }
}

// CP: channels of x and y, rounded up to 32.  200k x 64 -> 256 fp16 31-36 us (51 MB of rows would take 10,
// the products 14 at the rate of large ones; the two kernels that store h took 137 in their first form).
// A wave's gate, 16 exponentials and reciprocals for each 32 x 32 block, is as long as the block's
// MFMAs; other waves' MFMAs run beside it, four waves a SIMD, whose 128 registers are two to seven too
// few for silu and gelu (these go to scratch memory).  The 1 563 workgroups of those 200k rows are a round and
// a half of the 1 024 that are resident at a time: the second round is half empty.
template <typename T, int ACT, int CP, int MINW>
__global__ __launch_bounds__(kFfnThreads, MINW) void ffn_fused(FusedArgs<T> a) {
  using frag = typename Mfma<T>::frag;
  constexpr int TILES = CP / 32;
  __shared__ __attribute__((aligned(16))) char lds[2 * Chunk<CP>::BYTES];
  const int wave = int(threadIdx.x) >> 6, lane = int(threadIdx.x) & 31;
  const int half = (int(threadIdx.x) >> 5) & 1;
  const int64_t r = (int64_t(blockIdx.x) * 4 + wave) * kFusedRows + lane;
  Chunks<T, CP> chunks(a.w, lds);
  frag x[CP / 16];
  load_rows<T, CP>(a.x, r, x);
  floatx16 y[CP / 32];
  clear_rows(y);
  for (int f0 = 0; f0 < a.w.F; f0 += 32) {
    const char* chunk = chunks.next();
    floatx16 g, u;
    fused_up<T, CP>(chunk, x, g, u);
    // Wd's 32 channels i % TILES, its 16 hidden units i / TILES: an MFMA that adds to the result of the one
    // before it waits for it (84 clocks for 32)
    auto read = [&](int i) {
      return *reinterpret_cast<const frag*>(
          Chunk<CP>::down(chunk, i % TILES * 32 + lane, 2 * (i / TILES) + half));
    };
    Batched<frag, CP / 16, 4> down;
    down.start(read);
    frag h[2];
    gate16<true, ACT>(g, [&](int i, float value, float) { h[i >> 3][i & 7] = T(value * u[i]); });
    if (f0 + 32 > a.w.F) end_units(h, f0, a.w.F);
    down.run(read, [&](int i, const frag& f) { Mfma<T>::mma(f, h[i / TILES], y[i % TILES]); });
  }
  fused_store<T, CP>(a, r, y);
}

// dst = Wg and Wu as [Fp][Cp] and Wd as [Cop][Fp], with zeros past F, C and Co.
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

// A wave goes through all hidden units one chunk after the other, so a call lasts as long as that at
// least; the tiled kernels' chains are shorter, but write and read h.  Measured, one kernel against two
// (us; 128 -> 344 fp16): 1 000 rows 14.9 / 12.3, 8 000 15.5 / 14.7, 16 000 16.1 / 19.3, 32 000 17.6 / 28.8;
// 64 -> 256 8.7 / 10.6 at 1 000 rows; 192 -> 512 26.8 / 24.6 at 16 000 and 29.7 / 39.5 at 32 000;
// 256 -> 688 bf16 at 75 000 rows 149 / 138 (a wave a SIMD: its registers hold no more).  All of these have
// hidden widths of 2.7 to 4 times the channels; other ratios were not measured.
bool fused_forward_takes(int32_t dtype, int64_t rows, int64_t C, int64_t Co) {
  const int64_t n = C > Co ? C : Co;
  return dtype != SP_F32 && n <= kFusedWidth && (n <= 64 || rows >= 96 * n);
}

size_t fused_weights_bytes(int64_t C, int64_t F, int64_t Co) {
  return (2 * size_t(up8(F)) * up8(C) + size_t(up8(Co)) * up8(F)) * 2;
}

template <typename T, int CP, int MINW>
static int launch_fused(const FusedArgs<T>& a, int act, hipStream_t s) {
  const int64_t tiles = cdiv(a.x.n, kFusedRows);
  SP_CHECK_ARG(tiles <= kMaxGridX, "gated_ffn: too many rows");
  using Kern = void (*)(FusedArgs<T>);
  const Kern kern = act == kActSilu   ? Kern(ffn_fused<T, kActSilu, CP, MINW>)
                    : act == kActGelu ? Kern(ffn_fused<T, kActGelu, CP, MINW>)
                                      : Kern(ffn_fused<T, kActRelu, CP, MINW>);
  kern<<<unsigned(cdiv(tiles, 4)), kFfnThreads, 0, s>>>(a);
  SP_LAUNCHED();
  return SP_OK;
}

// The call's weights, where their rows do not start at multiples of 16 bytes as copies in ws.
template <typename T>
int fused_weights(const FfnCall& c, T* ws, Weights<T>& w) {
  w.g = static_cast<const T*>(c.wg);
  w.u = static_cast<const T*>(c.wu);
  w.d = static_cast<const T*>(c.wd);
  w.F = c.F, w.Co = c.Co;
  w.C = w.ldu = c.C;
  w.Fw = w.ldd = c.F;
  w.Cow = c.Co;
  if (c.C % 8 == 0 && c.F % 8 == 0 && aligned(c.wg) && aligned(c.wu) && aligned(c.wd))
    return SP_OK;
  const int Cp = up8(c.C), Fp = up8(c.F), Cop = up8(c.Co);
  ffn_pad<T><<<unsigned(cdiv(int64_t(Fp) * (2 * Cp + Cop), kFfnThreads * 4)), kFfnThreads, 0,
               c.stream>>>(w.g, w.u, w.d, c.C, c.F, c.Co, Cp, Fp, Cop, ws);
  SP_LAUNCHED();
  w.g = ws;
  w.u = ws + int64_t(Fp) * Cp;
  w.d = ws + 2 * int64_t(Fp) * Cp;
  w.C = w.ldu = Cp;
  w.Fw = w.ldd = Fp;
  w.Cow = Cop;
  return SP_OK;
}
template int fused_weights<_Float16>(const FfnCall&, _Float16*, Weights<_Float16>&);
template int fused_weights<__bf16>(const FfnCall&, __bf16*, Weights<__bf16>&);

template <typename T>
static int run_fused(const FfnCall& c) {
  FusedArgs<T> a{};
  a.x = operand<T>(c.x, c.ldx, c.rows, c.C);
  a.residual = operand<T>(c.residual, c.ldr, c.rows, c.Co);
  a.y = static_cast<T*>(c.y);
  a.vec_y = aligned(c.y) && c.Co % 8 == 0;
  if (int rc = fused_weights(c, static_cast<T*>(c.ws), a.w)) return rc;
  const int widest = c.C > c.Co ? c.C : c.Co;
  if (widest <= 32) return launch_fused<T, 32, 4>(a, c.act, c.stream);
  if (widest <= 64) return launch_fused<T, 64, 4>(a, c.act, c.stream);
  if (widest <= 96) return launch_fused<T, 96, 3>(a, c.act, c.stream);
  if (widest <= 128) return launch_fused<T, 128, 2>(a, c.act, c.stream);
  if (widest <= 160) return launch_fused<T, 160, 2>(a, c.act, c.stream);
  return launch_fused<T, 192, 2>(a, c.act, c.stream);
}

int fused_forward(int32_t dtype, const FfnCall& a) {
  return dtype == SP_F16 ? run_fused<_Float16>(a) : run_fused<__bf16>(a);
}

}  // namespace sp
