// What the kernels of the gated feed-forward block share.
#pragma once

#include <type_traits>

#include "sp_common.h"
#include "sp_mfma.h"

namespace sp {

constexpr int kFfnThreads = 256;
constexpr int kStagePieces = 8;  // 16-byte pieces of a row in a stage: 64 16-bit values

enum { kActSilu = 0, kActGelu = 1, kActRelu = 2 };

// 1 / (1 + exp(-z)) from the hardware's exponential and reciprocal, each of about one ulp: for
// values that are rounded to 16 bits (a fp32 row takes expf and a division).
__device__ __forceinline__ float sigmoid_fast(float z) {
  return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(z * -1.4426950408889634f));
}

// gelu(z) = z * cdf(z) by Abramowitz & Stegun, Handbook of Mathematical Functions, 7.1.26: erfc(x) =
// (a1 t + .. + a5 t^5) exp(-x^2), t = 1 / (1 + p x), x >= 0, to 1.5e-7; the exponential is the
// derivative's too.
__device__ __forceinline__ void gelu_start(float z, float& t, float& e) {
  const float x = __builtin_fabsf(z) * 0.70710678118654752f;
  t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.3275911f, x, 1.f));
  e = __builtin_amdgcn_exp2f(x * x * -1.4426950408889634f);
}
__device__ __forceinline__ void gelu_finish(float z, float t, float e, float& value,
                                            float& slope) {
  float p = __builtin_fmaf(1.061405429f, t, -1.453152027f);
  p = __builtin_fmaf(p, t, 1.421413741f);
  p = __builtin_fmaf(p, t, -0.284496736f);
  p = __builtin_fmaf(p, t, 0.254829592f) * t;
  const float tail = 0.5f * p * e, cdf = z < 0.f ? tail : 1.f - tail;
  value = z * cdf;
  slope = __builtin_fmaf(z * 0.39894228040143268f, e, cdf);
}

// The gate's activation and its derivative, FAST for 16-bit rows.
template <bool FAST, int ACT>
__device__ __forceinline__ void gate(float z, float& value, float& slope) {
  if constexpr (ACT == kActSilu) {
    const float sig = FAST ? sigmoid_fast(z) : 1.f / (1.f + expf(-z));
    value = z * sig;
    slope = __builtin_fmaf(value, 1.f - sig, sig);
  } else if constexpr (ACT == kActGelu && FAST) {
    float t, e;
    gelu_start(z, t, e);
    gelu_finish(z, t, e, value, slope);
  } else if constexpr (ACT == kActGelu) {
    const float cdf = 0.5f * (1.f + erff(z * 0.70710678118654752f));
    value = z * cdf;
    slope = cdf + z * expf(-0.5f * z * z) * 0.39894228040143268f;
  } else {
    value = z < 0.f ? 0.f : z;  // (a NaN stays)
    slope = z > 0.f ? 1.f : 0.f;
  }
}

// The gate of sixteen values of an accumulator, f(i, value, slope) for each, in stages, so that the
// exponentials and reciprocals of one value do not wait for each other.
template <bool FAST, int ACT, typename F>
__device__ __forceinline__ void gate16(const floatx16& z, F&& f) {
  if constexpr (ACT == kActSilu && FAST) {
    float t[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) t[i] = __builtin_amdgcn_exp2f(z[i] * -1.4426950408889634f);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < 16; ++i) t[i] = __builtin_amdgcn_rcpf(1.f + t[i]);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float value = z[i] * t[i];
      f(i, value, __builtin_fmaf(value, 1.f - t[i], t[i]));
    }
  } else if constexpr (ACT == kActGelu && FAST) {
#pragma unroll
    for (int b = 0; b < 16; b += 8) {
      float t[8], e[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) gelu_start(z[b + i], t[i], e[i]);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float value, slope;
        gelu_finish(z[b + i], t[i], e[i], value, slope);
        f(b + i, value, slope);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float value, slope;
      gate<FAST, ACT>(z[i], value, slope);
      f(i, value, slope);
    }
  }
}

// loop(kind) with the call's activation as a constant: one branch around the whole of it.
template <typename Loop>
__device__ __forceinline__ void with_act(int act, Loop&& loop) {
  if (act == kActSilu)
    loop(std::integral_constant<int, kActSilu>());
  else if (act == kActGelu)
    loop(std::integral_constant<int, kActGelu>());
  else
    loop(std::integral_constant<int, kActRelu>());
}

// Where piece c (16 bytes) of row r lies in LDS rows of PIECES pieces, so that no two lanes of a group
// meet on a bank.  The LDS has 64 banks, one row of which serves 16 lanes of a 16-byte read, lanes 0-3, 12-15
// and 20-27 or 4-11, 16-19 and 28-31 of either half (measured: pairs of lanes on one bank), and 32
// lanes of a transposed 8-byte one.  The first kind reads one piece of as many rows, whose r >> 2
// differ in their low two bits or whose r & 3 differ; the second four rows from a multiple
// of four on, four pieces of each.
template <int PIECES>
__device__ __forceinline__ int swizzled(int r, int c) {
  if constexpr (PIECES % 16 == 0) return c ^ (((r & 3) << 2) | ((r >> 2) & 3));
  if constexpr (PIECES % 8 == 0) return c ^ (((r & 2) << 1) | ((r >> 2) & 3));
  static_assert(PIECES % 4 == 0, "pieces are permuted within four, eight or sixteen");
  return c ^ ((r >> 2) & 3);
}

// Row of a 32-row weight block that lies at operand row m: then accumulator register i of lane half b is
// row 16 (i >> 3) + 8 b + (i & 7).
__device__ __forceinline__ int unit_of(int m) {
  return 16 * (m >> 4) + 8 * ((m >> 2) & 1) + 4 * ((m >> 3) & 1) + (m & 3);
}

__device__ const uint4 g_zero_piece = {0, 0, 0, 0};

// 16 bytes from memory to LDS at `to` (the wave's first lane's) + 16 * lane.
__device__ __forceinline__ void copy_piece(const void* from, char* to) {
  __builtin_amdgcn_global_load_lds(
      (const __attribute__((address_space(1))) void*)from,
      (__attribute__((address_space(3))) void*)to, 16, 0, 0);
}

// The wave's number in its workgroup, as one value for all of its lanes.
__device__ __forceinline__ int wave_of() {
  return __builtin_amdgcn_readfirstlane(int(threadIdx.x) >> 6);
}

// At most N of the wave's loads still on their way.
template <int N>
__device__ __forceinline__ void loads_in_flight() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// STEPS steps of products whose operands F come from LDS, B steps' reads at a time: a batch is read while
// the one before is in use.  Left to itself the compiler reads and waits step by step, for the
// LDS's latency each time (75k x 256 -> 688 bf16 in one kernel: 193 us, 168 so).  `start` may come
// early.
template <typename F, int STEPS, int B>
struct Batched {
  static constexpr int BATCHES = (STEPS + B - 1) / B;
  F f[2][B];
  template <typename Read>
  __device__ __forceinline__ void start(Read&& read) {
#pragma unroll
    for (int i = 0; i < B && i < STEPS; ++i) f[0][i] = read(i);
  }
  template <typename Read, typename Use>
  __device__ __forceinline__ void run(Read&& read, Use&& use) {
#pragma unroll
    for (int b = 0; b < BATCHES; ++b) {
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < B; ++i)
        if ((b + 1) * B + i < STEPS) f[(b + 1) & 1][i] = read((b + 1) * B + i);
#pragma unroll
      for (int i = 0; i < B; ++i)
        if (b * B + i < STEPS) use(b * B + i, f[b & 1][i]);
    }
    __builtin_amdgcn_sched_barrier(0);
  }
};

inline bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// A row-major operand: rows of K values; vec: rows start at multiples of 16 bytes.
template <typename T>
struct Rows {
  const T* p;
  int64_t ld;
  int64_t n;  // rows; what lies past them reads as zero
  int K;
  int vec;
};

template <typename T>
Rows<T> operand(const void* p, int64_t ld, int64_t n, int64_t K) {
  return Rows<T>{static_cast<const T*>(p), ld, n, int(K), aligned(p) && ld % Mfma<T>::V == 0};
}

inline int vec_of(int32_t dtype) { return dtype == SP_F32 ? 4 : 8; }
inline size_t size_of(int32_t dtype) { return dtype == SP_F32 ? 4 : 2; }

struct FfnCall {
  const void *x, *wg, *wu, *wd, *residual, *dy;
  int64_t ldx, ldr, lddy, rows;
  int C, F, Co, act;
  const int8_t* codes;  // of x, with scales, instead of x itself (backward)
  const float* scales;
  void *y, *dx, *dwg, *dwu, *dwd;
  void* ws;
  hipStream_t stream;
};

// The one-kernel passes, for 16-bit rows of at most kFusedWidth channels on either side
// (sp_ffn_fused.hip, sp_ffn_grad.hip).  `weights`: what copies of weights may take whose rows do not
// start at multiples of 16 bytes.
constexpr int kFusedWidth = 192;
constexpr int kFusedGramWidth = 128;  // the weight gradients' own kernel
size_t fused_weights_bytes(int64_t C, int64_t F, int64_t Co);
bool fused_forward_takes(int32_t dtype, int64_t rows, int64_t C, int64_t Co);
int fused_forward(int32_t dtype, const FfnCall& a);

// The backward pass: dx, and either the weight gradients' partials or the hidden rows for a
// kernel that makes them (wider than kFusedGramWidth).
struct FusedGrad {
  void *weights, *hid;
  float *part0, *part1;
  int64_t shares;
  int Fp;
};
bool fused_backward_takes(int32_t dtype, int64_t rows, int64_t C, int64_t Co);
int64_t fused_weights_shares(int64_t rows, int64_t C, int64_t F, int64_t Co);
// *shares: how many partials there are (at most o.shares)
int fused_backward(int32_t dtype, const FfnCall& a, const FusedGrad& o, int64_t* shares);

}  // namespace sp
