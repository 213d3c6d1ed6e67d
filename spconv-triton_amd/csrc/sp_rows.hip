// Operators on whole feature rows: the root-mean-square norm with the residual's
// addition, its gradients, and rows in 8 bits with a scale for each 128 channels.
//
//   s = x + residual, inv = 1 / sqrt(mean(s^2) + eps), y = s * inv * w
//   ds = dsum + inv * t - s * inv^3 * mean(t * s), t = dy * w
//   dw = sum over rows of dy * s * inv
//   step = max|y| / 127 over a row's group of 128 channels, code = rint(y * (127 / max|y|))
//
// All are bound by memory: rows are read once and written once.  2^k neighbouring
// lanes of a wave hold a row (V values, 16 bytes, each, and up to four such pieces), so
// that sums and maxima over a row are butterflies within the wave and 64-channel
// rows go eight to a wave.  Statistics and sums are fp32; the 8-bit copy is of y as rounded to the
// rows' type, so that it equals quantising the stored rows.
#include <type_traits>

#include "sp_common.h"
#include "sp_mfma.h"

namespace sp {

constexpr int kRowThreads = 256;
constexpr int kRowGroup = 128;   // channels that share a scale
constexpr int kRowPieces = 4;    // pieces of a lane at most: wider rows take the looping kernels
constexpr int kRowPartials = 1024;  // workgroups of the norm's backward pass at most
constexpr int kWideStrip = 64;   // channels of a workgroup in the wide weight gradient
// Workgroups of a launch at most: HIP takes grids of fewer than 2^32 threads.
constexpr int64_t kRowGrid = 0xffffffffLL / kRowThreads;

template <typename T, int V>
struct alignas(sizeof(T) * V) Piece {
  T v[V];
};

// ---- 8-bit steps -----------------------------------------------------------
// A group with an infinity or a NaN has no finite step: its step is NaN, and so are the
// values it stands for.  Below 2^-100 the factor 127 / max could overflow: such a group
// is zeros.
__device__ __forceinline__ uint32_t magnitude_bits(float v) {
  return __float_as_uint(v) & 0x7fffffffu;  // ordered as the magnitudes, NaN above infinity
}

__device__ __forceinline__ void group_step(uint32_t top, float& step, float& up) {
  const float a = __uint_as_float(top);
  if (top >= 0x7f800000u) {
    step = __uint_as_float(0x7fc00000u);
    up = 0.f;
  } else if (a < 0x1p-100f) {
    step = up = 0.f;
  } else {
    step = a / 127.f;
    up = 127.f / a;
  }
}

__device__ __forceinline__ int8_t code_of(float v, float up) {
  return up == 0.f ? int8_t(0) : int8_t(int(rintf(v * up)));
}

// ---- rows held by 2^k lanes --------------------------------------------------
__device__ __forceinline__ float row_sum(float v, int lanes) {
  for (int off = lanes >> 1; off >= 1; off >>= 1) v += __shfl_xor(v, off, 64);
  return v;
}

__device__ __forceinline__ uint32_t lanes_max(uint32_t v, int lanes) {
  for (int off = lanes >> 1; off >= 1; off >>= 1) {
    const uint32_t o = __shfl_xor(v, off, 64);
    v = o > v ? o : v;
  }
  return v;
}

// Codes and scales of a row whose values (as stored) the lanes hold.  A group is 128 / V
// neighbouring lanes, or with V = 1 two pieces of all 64.
template <typename T, int V, int PIECES>
__device__ __forceinline__ void emit_codes(const Piece<T, V> (&y)[PIECES], bool live, int64_t r,
                                           int lane, int lanes, int C, int groups,
                                           int8_t* __restrict__ codes,
                                           float* __restrict__ scales) {
  uint32_t top[PIECES];
#pragma unroll
  for (int p = 0; p < PIECES; ++p) {
    top[p] = 0u;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const uint32_t m = magnitude_bits(float(y[p].v[i]));
      top[p] = m > top[p] ? m : top[p];
    }
  }
  if constexpr (V == 1 && PIECES > 1) {
#pragma unroll
    for (int p = 0; p < PIECES; p += 2) {
      if (p + 1 < PIECES) top[p] = top[p + 1] = top[p] > top[p + 1] ? top[p] : top[p + 1];
    }
  }
  const int span = V == 1 ? lanes : (lanes < kRowGroup / V ? lanes : kRowGroup / V);
#pragma unroll
  for (int p = 0; p < PIECES; ++p) {
    float step, up;
    group_step(lanes_max(top[p], span), step, up);
    const int c = (p * lanes + lane) * V;
    if (!live || c >= C) continue;
    Piece<int8_t, V> q;
#pragma unroll
    for (int i = 0; i < V; ++i) q.v[i] = code_of(float(y[p].v[i]), up);
    *reinterpret_cast<Piece<int8_t, V>*>(codes + r * C + c) = q;
    if (c % kRowGroup == 0) scales[r * groups + c / kRowGroup] = step;
  }
}

template <typename P, int V, int PIECES>
__device__ __forceinline__ void load_scale(const void* w, int lane, int lanes, int C,
                                           float (&f)[PIECES][V]) {
#pragma unroll
  for (int p = 0; p < PIECES; ++p) {
    const int c = (p * lanes + lane) * V;
#pragma unroll
    for (int i = 0; i < V; ++i)
      f[p][i] = w && c < C ? float(static_cast<const P*>(w)[c + i]) : 1.f;
  }
}

// ---- norm, forward -----------------------------------------------------------
// NORM false: the 8-bit codes of x alone.  All loads of a workgroup's rows (two for each group of
// lanes) start before its first sum, which is what hides the memory's latency; nothing is
// read twice.  At a copy's rate (4.9 TB/s between arrays past the caches): residual, norm and codes of
// 200k x 64 fp16, 116 MB, 24 us; residual and norm of 240k x 128 bf16, 246 MB, 52 us; codes alone of
// 400k x 64 fp16, 78 MB, 17 us.  Rows of 99 fp32 channels, value by value: 79 MB, 18 us.
template <typename T, typename P, int V, int PIECES, int ROWS, bool NORM>
__global__ __launch_bounds__(kRowThreads) void rms_rows(
    const T* __restrict__ x, int64_t ldx, const T* __restrict__ res, int64_t ldr,
    const void* __restrict__ w, float eps, int64_t rows, int C, int log_lanes,
    T* __restrict__ y, T* __restrict__ sum, int8_t* __restrict__ codes,
    float* __restrict__ scales) {
  using vec = Piece<T, V>;
  const int lanes = 1 << log_lanes, lane = int(threadIdx.x) & (lanes - 1);
  const int per = kRowThreads >> log_lanes;
  const int64_t first = int64_t(blockIdx.x) * (per * ROWS) + (int(threadIdx.x) >> log_lanes);
  const int groups = (C + kRowGroup - 1) / kRowGroup;
  vec a[ROWS][PIECES], b[ROWS][PIECES];
#pragma unroll
  for (int j = 0; j < ROWS; ++j) {
    const int64_t r = first + int64_t(j) * per;
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
      const int c = (p * lanes + lane) * V;
      a[j][p] = vec{};
      b[j][p] = vec{};
      if (r < rows && c < C) {
        a[j][p] = *reinterpret_cast<const vec*>(x + r * ldx + c);
        if (NORM && res) b[j][p] = *reinterpret_cast<const vec*>(res + r * ldr + c);
      }
    }
  }
  float f[PIECES][V];
  if constexpr (NORM) load_scale<P, V, PIECES>(w, lane, lanes, C, f);
#pragma unroll
  for (int j = 0; j < ROWS; ++j) {
    const int64_t r = first + int64_t(j) * per;
    if constexpr (NORM) {
      float s[PIECES][V], sq = 0.f;
#pragma unroll
      for (int p = 0; p < PIECES; ++p)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          s[p][i] = float(a[j][p].v[i]) + (res ? float(b[j][p].v[i]) : 0.f);
          sq = __builtin_fmaf(s[p][i], s[p][i], sq);
        }
      const float inv = 1.f / sqrtf(row_sum(sq, lanes) / float(C) + eps);
#pragma unroll
      for (int p = 0; p < PIECES; ++p) {
        const int c = (p * lanes + lane) * V;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          b[j][p].v[i] = T(s[p][i]);
          a[j][p].v[i] = T(s[p][i] * inv * f[p][i]);
        }
        if (r < rows && c < C) {
          *reinterpret_cast<vec*>(y + r * C + c) = a[j][p];
          if (sum) *reinterpret_cast<vec*>(sum + r * C + c) = b[j][p];
        }
      }
    }
    if (codes)
      emit_codes<T, V, PIECES>(a[j], r < rows, r, lane, lanes, C, groups, codes, scales);
  }
}

// ---- any width: a workgroup a row ----------------------------------------------
// Rows wider than a wave holds (or, where they are not aligned, than 256 channels) are read twice,
// the second time from the caches.
__device__ __forceinline__ float block_sum(float v, float* lds) {
  v = row_sum(v, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0.f;
#pragma unroll
  for (int i = 0; i < kRowThreads / 64; ++i) v += lds[i];
  return v;
}

template <typename T, typename P, bool NORM>
__global__ __launch_bounds__(kRowThreads) void rms_wide(
    const T* __restrict__ x, int64_t ldx, const T* __restrict__ res, int64_t ldr,
    const void* __restrict__ w, float eps, int64_t rows, int C, T* __restrict__ y,
    T* __restrict__ sum, int8_t* __restrict__ codes, float* __restrict__ scales) {
  __shared__ float lds[kRowThreads / 64];
  const int wave = int(threadIdx.x) >> 6, lane = int(threadIdx.x) & 63;
  const int groups = (C + kRowGroup - 1) / kRowGroup;
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const T* xr = x + r * ldx;
    const T* rr = res ? res + r * ldr : nullptr;
    float inv = 0.f;
    if constexpr (NORM) {
      float sq = 0.f;
      for (int c = int(threadIdx.x); c < C; c += kRowThreads) {
        const float s = float(xr[c]) + (rr ? float(rr[c]) : 0.f);
        sq = __builtin_fmaf(s, s, sq);
      }
      inv = 1.f / sqrtf(block_sum(sq, lds) / float(C) + eps);
    }
    // a wave takes whole groups: two channels a lane
    for (int g = wave; g < groups; g += kRowThreads / 64) {
      T v[2];
      uint32_t top = 0u;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int c = g * kRowGroup + h * 64 + lane;
        v[h] = T(0.f);
        if (c < C) {
          v[h] = xr[c];
          if constexpr (NORM) {
            const float s = float(xr[c]) + (rr ? float(rr[c]) : 0.f);
            v[h] = T(s * inv * (w ? float(static_cast<const P*>(w)[c]) : 1.f));
            y[r * C + c] = v[h];
            if (sum) sum[r * C + c] = T(s);
          }
        }
        const uint32_t m = magnitude_bits(float(v[h]));
        top = m > top ? m : top;
      }
      if (!codes) continue;
      float step, up;
      group_step(lanes_max(top, 64), step, up);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int c = g * kRowGroup + h * 64 + lane;
        if (c < C) codes[r * C + c] = code_of(float(v[h]), up);
      }
      if (lane == 0) scales[r * groups + g] = step;
    }
  }
}

// ---- norm, backward ------------------------------------------------------------
// Each workgroup goes through rows of its own, every lane summing dw of its channels in fp32
// registers, and leaves one partial a channel, which rms_dw_reduce sums in a fixed order (no atomics:
// two calls give the same gradient).  The statistics are formed again from s as it is stored
// (rounded to the rows' type, which adds to dw as much error as dw's own rounding: 0.0024 for 0.0017 relative in
// bf16; an fp32 sum would be 2 C bytes more a row in each direction).
// 240k x 128 bf16 with a gradient of the sum, 246 MB, 45 us (5.5 TB/s); 50k x 99 fp32, value by value
// and two pieces a lane, 79 MB, 24 us.
template <typename T, typename P, int V, int PIECES, int ROWS>
__global__ __launch_bounds__(kRowThreads) void rms_rows_bwd(
    const T* __restrict__ dy, int64_t lddy, const T* __restrict__ dsum, int64_t ldds,
    const T* __restrict__ s, int64_t lds_, const void* __restrict__ w, float eps, int64_t rows,
    int C, int log_lanes, T* __restrict__ ds, float* __restrict__ part, P* __restrict__ dw) {
  using vec = Piece<T, V>;
  constexpr int NW = kRowThreads / 64;
  __shared__ float lds[NW][64 * V * PIECES];
  const int lanes = 1 << log_lanes, lane = int(threadIdx.x) & (lanes - 1);
  const int per = kRowThreads >> log_lanes;
  const int64_t stride = int64_t(gridDim.x) * (per * ROWS);
  float f[PIECES][V], acc[PIECES][V];
  load_scale<P, V, PIECES>(w, lane, lanes, C, f);
#pragma unroll
  for (int p = 0; p < PIECES; ++p)
#pragma unroll
    for (int i = 0; i < V; ++i) acc[p][i] = 0.f;
  // (the bound is the workgroup's, so that whole waves take the butterflies)
  for (int64_t base = int64_t(blockIdx.x) * (per * ROWS); base < rows; base += stride) {
    vec a[ROWS][PIECES], b[ROWS][PIECES], d[ROWS][PIECES];
#pragma unroll
    for (int j = 0; j < ROWS; ++j) {
      const int64_t r = base + int64_t(j) * per + (int(threadIdx.x) >> log_lanes);
#pragma unroll
      for (int p = 0; p < PIECES; ++p) {
        const int c = (p * lanes + lane) * V;
        a[j][p] = vec{};
        b[j][p] = vec{};
        d[j][p] = vec{};
        if (r < rows && c < C) {
          a[j][p] = *reinterpret_cast<const vec*>(s + r * lds_ + c);
          b[j][p] = *reinterpret_cast<const vec*>(dy + r * lddy + c);
          if (dsum) d[j][p] = *reinterpret_cast<const vec*>(dsum + r * ldds + c);
        }
      }
    }
#pragma unroll
    for (int j = 0; j < ROWS; ++j) {
      const int64_t r = base + int64_t(j) * per + (int(threadIdx.x) >> log_lanes);
      float sq = 0.f, dot = 0.f;
#pragma unroll
      for (int p = 0; p < PIECES; ++p)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float sv = float(a[j][p].v[i]);
          sq = __builtin_fmaf(sv, sv, sq);
          dot = __builtin_fmaf(float(b[j][p].v[i]) * f[p][i], sv, dot);
        }
      const float inv = 1.f / sqrtf(row_sum(sq, lanes) / float(C) + eps);
      const float back = row_sum(dot, lanes) / float(C) * inv * inv;
#pragma unroll
      for (int p = 0; p < PIECES; ++p) {
        const int c = (p * lanes + lane) * V;
        vec o;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float sv = float(a[j][p].v[i]), g = float(b[j][p].v[i]);
          // (past the end inv may be infinite, with eps = 0)
          acc[p][i] = __builtin_fmaf(g, r < rows ? sv * inv : 0.f, acc[p][i]);
          const float t = inv * __builtin_fmaf(-sv, back, g * f[p][i]);
          o.v[i] = T(dsum ? float(d[j][p].v[i]) + t : t);
        }
        if (r < rows && c < C) *reinterpret_cast<vec*>(ds + r * C + c) = o;
      }
    }
  }
  if (!part && !dw) return;
  const int wave = int(threadIdx.x) >> 6;
#pragma unroll
  for (int p = 0; p < PIECES; ++p)
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float v = acc[p][i];
      for (int off = lanes; off < 64; off <<= 1) v += __shfl_xor(v, off, 64);
      if ((int(threadIdx.x) & 63) < lanes) lds[wave][(p * lanes + lane) * V + i] = v;
    }
  __syncthreads();
  for (int c = int(threadIdx.x); c < C; c += kRowThreads) {
    float v = lds[0][c];
#pragma unroll
    for (int q = 1; q < NW; ++q) v += lds[q][c];
    if (dw)  // (the only workgroup)
      dw[c] = P(v);
    else
      part[int64_t(blockIdx.x) * C + c] = v;
  }
}

template <typename T, typename P>
__global__ __launch_bounds__(kRowThreads) void rms_wide_bwd(
    const T* __restrict__ dy, int64_t lddy, const T* __restrict__ dsum, int64_t ldds,
    const T* __restrict__ s, int64_t lds_, const void* __restrict__ w, float eps, int64_t rows,
    int C, T* __restrict__ ds, float* __restrict__ invs) {
  __shared__ float lds[kRowThreads / 64];
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    float sq = 0.f, dot = 0.f;
    for (int c = int(threadIdx.x); c < C; c += kRowThreads) {
      const float sv = float(s[r * lds_ + c]);
      const float f = w ? float(static_cast<const P*>(w)[c]) : 1.f;
      sq = __builtin_fmaf(sv, sv, sq);
      dot = __builtin_fmaf(float(dy[r * lddy + c]) * f, sv, dot);
    }
    const float inv = 1.f / sqrtf(block_sum(sq, lds) / float(C) + eps);
    const float back = block_sum(dot, lds) / float(C) * inv * inv;
    for (int c = int(threadIdx.x); c < C; c += kRowThreads) {
      const float sv = float(s[r * lds_ + c]);
      const float f = w ? float(static_cast<const P*>(w)[c]) : 1.f;
      const float t = inv * __builtin_fmaf(-sv, back, float(dy[r * lddy + c]) * f);
      ds[r * C + c] = T(dsum ? float(dsum[r * ldds + c]) + t : t);
    }
    if (invs && threadIdx.x == 0) invs[r] = inv;
  }
}

// The wide weight gradient's partials: 64 channels and a share of the rows a workgroup.
template <typename T>
__global__ __launch_bounds__(kRowThreads) void rms_wide_dw(
    const T* __restrict__ dy, int64_t lddy, const T* __restrict__ s, int64_t lds_,
    const float* __restrict__ invs, int64_t rows, int C, int64_t share,
    float* __restrict__ part) {
  constexpr int NW = kRowThreads / 64;
  __shared__ float lds[NW][kWideStrip];
  const int c = int(blockIdx.x) * kWideStrip + (int(threadIdx.x) & 63);
  const int wave = int(threadIdx.x) >> 6;
  const int64_t lo = int64_t(blockIdx.y) * share;
  const int64_t hi = lo + share < rows ? lo + share : rows;
  float v = 0.f;
  if (c < C)
    for (int64_t r = lo + wave; r < hi; r += NW)
      v = __builtin_fmaf(float(dy[r * lddy + c]), float(s[r * lds_ + c]) * invs[r], v);
  lds[wave][threadIdx.x & 63] = v;
  __syncthreads();
  if (wave == 0 && c < C) {
    v = lds[0][threadIdx.x];
#pragma unroll
    for (int q = 1; q < NW; ++q) v += lds[q][threadIdx.x];
    part[int64_t(blockIdx.y) * C + c] = v;
  }
}

// dw[c] = the partials of channel c, 16 runs of them summed apart and then in order.  4.5 us for 1 024
// partials of 128 channels: half a megabyte, a chain of loads.
template <typename P>
__global__ __launch_bounds__(kRowThreads) void rms_dw_reduce(const float* __restrict__ part,
                                                             int n, int C, P* __restrict__ dw) {
  __shared__ float lds[16][17];
  const int cl = int(threadIdx.x) & 15, run = int(threadIdx.x) >> 4;
  const int c = int(blockIdx.x) * 16 + cl;
  float v = 0.f;
  if (c < C) {
#pragma unroll 8
    for (int i = run; i < n; i += 16) v += part[int64_t(i) * C + c];
  }
  lds[run][cl] = v;
  __syncthreads();
  if (run == 0 && c < C) {
#pragma unroll
    for (int q = 1; q < 16; ++q) v += lds[q][cl];
    dw[c] = P(v);
  }
}

// ---- 8 bits back to rows ---------------------------------------------------------
// code * step in fp32, one rounding to the rows' type.  400k x 64 fp16, 78 MB, 14 us (5.6 TB/s).
template <typename T, int V>
__global__ __launch_bounds__(kRowThreads) void restore_rows(const int8_t* __restrict__ codes,
                                                            const float* __restrict__ scales,
                                                            int64_t pieces, int C,
                                                            T* __restrict__ out) {
  const int64_t step = int64_t(gridDim.x) * kRowThreads;
  const int row_pieces = C / V, groups = (C + kRowGroup - 1) / kRowGroup;
  for (int64_t i = int64_t(blockIdx.x) * kRowThreads + threadIdx.x; i < pieces; i += step) {
    const int64_t r = i / row_pieces;
    const int c = int(i - r * row_pieces) * V;
    const Piece<int8_t, V> q = *reinterpret_cast<const Piece<int8_t, V>*>(codes + i * V);
    const float scale = scales[r * groups + c / kRowGroup];
    Piece<T, V> o;
#pragma unroll
    for (int k = 0; k < V; ++k) o.v[k] = T(float(q.v[k]) * scale);
    *reinterpret_cast<Piece<T, V>*>(out + i * V) = o;
  }
}

// ---- host ------------------------------------------------------------------------
static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Lanes (as a power of two) and pieces of a row in units of V values.
static void row_shape(int C, int V, int& log_lanes, int& pieces) {
  const int units = (C + V - 1) / V;
  log_lanes = 0;
  while (log_lanes < 6 && (1 << log_lanes) < units) ++log_lanes;
  pieces = int(cdiv(units, 64));
}

struct NormCall {
  const void *x, *res, *w;
  int64_t ldx, ldr, rows;
  int C;
  float eps;
  void *y, *sum;
  int8_t* codes;
  float* scales;
  hipStream_t stream;
};

template <typename T, typename P, int V, int PIECES, bool NORM>
static int launch_rows(const NormCall& a, int log_lanes) {
  constexpr int ROWS = PIECES == 1 ? 2 : 1;
  const int64_t per = int64_t(kRowThreads >> log_lanes) * ROWS, most = kRowGrid * per;
  const int groups = int(cdiv(a.C, kRowGroup));
  auto from = [](auto* p, int64_t at) { return p ? p + at : nullptr; };
  for (int64_t r = 0; r < a.rows; r += most) {
    const int64_t rows = a.rows - r < most ? a.rows - r : most;
    rms_rows<T, P, V, PIECES, ROWS, NORM>
        <<<unsigned(cdiv(rows, per)), kRowThreads, 0, a.stream>>>(
            static_cast<const T*>(a.x) + r * a.ldx, a.ldx,
            from(static_cast<const T*>(a.res), r * a.ldr), a.ldr, a.w, a.eps, rows, a.C, log_lanes,
            from(static_cast<T*>(a.y), r * a.C), from(static_cast<T*>(a.sum), r * a.C),
            from(a.codes, r * a.C), from(a.scales, r * groups));
    SP_LAUNCHED();
  }
  return SP_OK;
}

template <typename T, typename P, int V, bool NORM>
static int dispatch_rows(const NormCall& a) {
  int log_lanes, pieces;
  row_shape(a.C, V, log_lanes, pieces);
  if (pieces == 1) return launch_rows<T, P, V, 1, NORM>(a, log_lanes);
  if (pieces == 2) return launch_rows<T, P, V, 2, NORM>(a, log_lanes);
  return launch_rows<T, P, V, 4, NORM>(a, log_lanes);
}

template <typename T, typename P, bool NORM>
static int run_rows(const NormCall& a) {
  constexpr int V = 16 / int(sizeof(T));
  const bool vec = a.C % V == 0 && a.ldx % V == 0 && aligned16(a.x) && aligned16(a.y) &&
                   aligned16(a.sum) && (!a.res || (a.ldr % V == 0 && aligned16(a.res))) &&
                   (reinterpret_cast<uintptr_t>(a.codes) & (V - 1)) == 0;
  if (vec && a.C <= 64 * V * kRowPieces) return dispatch_rows<T, P, V, NORM>(a);
  if (a.C <= 64 * kRowPieces) return dispatch_rows<T, P, 1, NORM>(a);
  const int64_t blocks = a.rows < 65536 ? a.rows : 65536;
  rms_wide<T, P, NORM><<<unsigned(blocks), kRowThreads, 0, a.stream>>>(
      static_cast<const T*>(a.x), a.ldx, static_cast<const T*>(a.res), a.ldr, a.w, a.eps, a.rows,
      a.C, static_cast<T*>(a.y), static_cast<T*>(a.sum), a.codes, a.scales);
  SP_LAUNCHED();
  return SP_OK;
}

struct NormGrad {
  const void *dy, *dsum, *s, *w;
  int64_t lddy, ldds, lds, rows;
  int C;
  float eps;
  void *ds, *dw;
  void* ws;
  hipStream_t stream;
};

// Workgroups of the wide weight gradient along the rows.
static int64_t wide_shares(int64_t rows) { return rows < 64 * 64 ? cdiv(rows, 64) : 64; }

template <typename P>
static int reduce_dw(const float* part, int64_t n, const NormGrad& a) {
  rms_dw_reduce<P><<<unsigned(cdiv(a.C, 16)), kRowThreads, 0, a.stream>>>(
      part, int(n), a.C, static_cast<P*>(a.dw));
  SP_LAUNCHED();
  return SP_OK;
}

// A few rows (64 of 64 channels, two turns of a workgroup) go to one workgroup, which needs no partials: the
// other launch and the workspace cost the host 4 us of the call's 13.
static bool one_workgroup(int64_t rows, int64_t C) { return C <= 256 && rows * C <= 4096; }

template <typename T, typename P, int V, int PIECES>
static int launch_bwd(const NormGrad& a, int log_lanes) {
  constexpr int ROWS = PIECES == 1 ? 2 : 1;
  int64_t blocks = cdiv(a.rows, int64_t(kRowThreads >> log_lanes) * ROWS);
  if (blocks > kRowPartials) blocks = kRowPartials;
  const bool alone = a.dw && one_workgroup(a.rows, a.C);
  if (alone) blocks = 1;
  float* part = a.dw && !alone ? static_cast<float*>(a.ws) : nullptr;
  rms_rows_bwd<T, P, V, PIECES, ROWS><<<unsigned(blocks), kRowThreads, 0, a.stream>>>(
      static_cast<const T*>(a.dy), a.lddy, static_cast<const T*>(a.dsum), a.ldds,
      static_cast<const T*>(a.s), a.lds, a.w, a.eps, a.rows, a.C, log_lanes,
      static_cast<T*>(a.ds), part, alone ? static_cast<P*>(a.dw) : nullptr);
  SP_LAUNCHED();
  return part ? reduce_dw<P>(part, blocks, a) : SP_OK;
}

template <typename T, typename P, int V>
static int dispatch_bwd(const NormGrad& a) {
  int log_lanes, pieces;
  row_shape(a.C, V, log_lanes, pieces);
  if (pieces == 1) return launch_bwd<T, P, V, 1>(a, log_lanes);
  if (pieces == 2) return launch_bwd<T, P, V, 2>(a, log_lanes);
  return launch_bwd<T, P, V, 4>(a, log_lanes);
}

template <typename T, typename P>
static int run_bwd(const NormGrad& a) {
  constexpr int V = 16 / int(sizeof(T));
  const bool vec = a.C % V == 0 && a.lddy % V == 0 && a.lds % V == 0 && aligned16(a.dy) &&
                   aligned16(a.s) && aligned16(a.ds) &&
                   (!a.dsum || (a.ldds % V == 0 && aligned16(a.dsum)));
  if (vec && a.C <= 64 * V * kRowPieces) return dispatch_bwd<T, P, V>(a);
  if (a.C <= 64 * kRowPieces) return dispatch_bwd<T, P, 1>(a);
  const int64_t blocks = a.rows < 65536 ? a.rows : 65536;
  const int64_t shares = wide_shares(a.rows);
  float* part = static_cast<float*>(a.ws);
  float* invs = a.dw ? part + shares * a.C : nullptr;
  rms_wide_bwd<T, P><<<unsigned(blocks), kRowThreads, 0, a.stream>>>(
      static_cast<const T*>(a.dy), a.lddy, static_cast<const T*>(a.dsum), a.ldds,
      static_cast<const T*>(a.s), a.lds, a.w, a.eps, a.rows, a.C, static_cast<T*>(a.ds), invs);
  SP_LAUNCHED();
  if (!a.dw) return SP_OK;
  rms_wide_dw<T><<<dim3(unsigned(cdiv(a.C, kWideStrip)), unsigned(shares)), kRowThreads, 0,
                   a.stream>>>(static_cast<const T*>(a.dy), a.lddy, static_cast<const T*>(a.s),
                               a.lds, invs, a.rows, a.C, cdiv(a.rows, shares), part);
  SP_LAUNCHED();
  return reduce_dw<P>(part, shares, a);
}

template <typename T>
static int run_restore(const int8_t* codes, const float* scales, int64_t rows, int C, void* out,
                       hipStream_t s) {
  constexpr int V = 16 / int(sizeof(T));
  const bool vec =
      C % V == 0 && aligned16(out) && (reinterpret_cast<uintptr_t>(codes) & (V - 1)) == 0;
  const int64_t pieces = rows * (vec ? C / V : C);
  const int64_t blocks = cdiv(pieces, kRowThreads);
  const unsigned grid = unsigned(blocks < kRowGrid ? blocks : kRowGrid);
  if (vec)
    restore_rows<T, V><<<grid, kRowThreads, 0, s>>>(codes, scales, pieces, C,
                                                    static_cast<T*>(out));
  else
    restore_rows<T, 1><<<grid, kRowThreads, 0, s>>>(codes, scales, pieces, C,
                                                    static_cast<T*>(out));
  SP_LAUNCHED();
  return SP_OK;
}

static bool row_type(int32_t dtype) {
  return dtype == SP_F16 || dtype == SP_BF16 || dtype == SP_F32;
}

// f(row type, parameter type) for the calls' types
template <typename F>
static int with_types(int32_t dtype, bool f32, F&& f) {
  switch (dtype) {
    case SP_F16:
      return f32 ? f(_Float16(), float()) : f(_Float16(), _Float16());
    case SP_BF16:
      return f32 ? f(__bf16(), float()) : f(__bf16(), __bf16());
    default:
      return f(float(), float());
  }
}

}  // namespace sp

using namespace sp;

extern "C" int sp_rms_norm(const void* x, int64_t ldx, const void* residual, int64_t ldr,
                           int32_t dtype, int64_t rows, int64_t C, const void* weight,
                           int32_t param_dtype, float eps, void* y, void* sum, int8_t* codes,
                           float* scales, void* stream) {
  SP_CHECK_ARG(rows >= 0 && C >= 1 && C < 65536, "rms_norm: bad sizes rows=%lld C=%lld",
               (long long)rows, (long long)C);
  SP_CHECK_ARG(row_type(dtype), "rms_norm: dtype %d not supported (f16/bf16/f32)", dtype);
  SP_CHECK_ARG(param_dtype == dtype || param_dtype == SP_F32,
               "rms_norm: the weight must be of the rows' type or fp32");
  SP_CHECK_ARG(eps >= 0.f, "rms_norm: eps is negative");
  if (rows == 0) return SP_OK;
  SP_CHECK_ARG(x && y, "rms_norm: null pointer");
  SP_CHECK_ARG(ldx >= C && (!residual || ldr >= C), "rms_norm: rows overlap");
  SP_CHECK_ARG((codes == nullptr) == (scales == nullptr), "rms_norm: codes without scales");
  const NormCall a{x,  residual, weight, ldx,   ldr,    rows, int(C),
                   eps, y,        sum,    codes, scales, as_stream(stream)};
  return with_types(dtype, param_dtype == SP_F32, [&](auto t, auto p) {
    return run_rows<decltype(t), decltype(p), true>(a);
  });
}

extern "C" size_t sp_rms_norm_bwd_workspace(int64_t rows, int64_t C) {
  if (rows <= 0 || C <= 0 || one_workgroup(rows, C)) return 0;
  const size_t fast = size_t(rows < kRowPartials ? rows : kRowPartials) * size_t(C);
  const size_t wide = size_t(wide_shares(rows)) * size_t(C) + size_t(rows);
  return (fast > wide ? fast : wide) * sizeof(float);
}

extern "C" int sp_rms_norm_bwd(const void* dy, int64_t lddy, const void* dsum, int64_t ldds,
                               const void* s, int64_t lds, int32_t dtype, int64_t rows, int64_t C,
                               const void* weight, int32_t param_dtype, float eps, void* ds,
                               void* dweight, void* ws, size_t ws_bytes, void* stream) {
  SP_CHECK_ARG(rows >= 0 && C >= 1 && C < 65536, "rms_norm_bwd: bad sizes rows=%lld C=%lld",
               (long long)rows, (long long)C);
  SP_CHECK_ARG(row_type(dtype), "rms_norm_bwd: dtype %d not supported (f16/bf16/f32)", dtype);
  SP_CHECK_ARG(param_dtype == dtype || param_dtype == SP_F32,
               "rms_norm_bwd: the weight must be of the rows' type or fp32");
  if (rows == 0) return SP_OK;
  SP_CHECK_ARG(dy && s && ds, "rms_norm_bwd: null pointer");
  SP_CHECK_ARG(lddy >= C && lds >= C && (!dsum || ldds >= C), "rms_norm_bwd: rows overlap");
  if (dweight && !one_workgroup(rows, C)) {
    SP_CHECK_ARG(ws && aligned16(ws), "rms_norm_bwd: the workspace must be 16-byte aligned");
    if (ws_bytes < sp_rms_norm_bwd_workspace(rows, C))
      return set_error(SP_ERR_WORKSPACE, "rms_norm_bwd: workspace of %zu bytes, needs %zu",
                       ws_bytes, sp_rms_norm_bwd_workspace(rows, C));
  }
  const NormGrad a{dy,  dsum, s,  weight,  lddy, ldds,
                   lds, rows, int(C), eps, ds,   dweight, ws, as_stream(stream)};
  return with_types(dtype, param_dtype == SP_F32, [&](auto t, auto p) {
    return run_bwd<decltype(t), decltype(p)>(a);
  });
}

extern "C" int sp_quantize_rows(const void* x, int64_t ldx, int32_t dtype, int64_t rows, int64_t C,
                                int8_t* codes, float* scales, void* stream) {
  SP_CHECK_ARG(rows >= 0 && C >= 1 && C < 65536, "quantize_rows: bad sizes rows=%lld C=%lld",
               (long long)rows, (long long)C);
  SP_CHECK_ARG(row_type(dtype), "quantize_rows: dtype %d not supported (f16/bf16/f32)", dtype);
  if (rows == 0) return SP_OK;
  SP_CHECK_ARG(x && codes && scales, "quantize_rows: null pointer");
  SP_CHECK_ARG(ldx >= C, "quantize_rows: rows overlap");
  NormCall a{};
  a.x = x;
  a.ldx = ldx;
  a.rows = rows;
  a.C = int(C);
  a.codes = codes;
  a.scales = scales;
  a.stream = as_stream(stream);
  return with_types(dtype, false, [&](auto t, auto) {
    return run_rows<decltype(t), decltype(t), false>(a);
  });
}

extern "C" int sp_restore_rows(const int8_t* codes, const float* scales, int64_t rows, int64_t C,
                               int32_t dtype, void* out, void* stream) {
  SP_CHECK_ARG(rows >= 0 && C >= 1 && C < 65536, "restore_rows: bad sizes rows=%lld C=%lld",
               (long long)rows, (long long)C);
  SP_CHECK_ARG(row_type(dtype), "restore_rows: dtype %d not supported (f16/bf16/f32)", dtype);
  if (rows == 0) return SP_OK;
  SP_CHECK_ARG(codes && scales && out, "restore_rows: null pointer");
  hipStream_t s = as_stream(stream);
  return with_types(dtype, false, [&](auto t, auto) {
    return run_restore<decltype(t)>(codes, scales, rows, int(C), out, s);
  });
}
