// Group norm of feature rows, sample by sample, with an activation after it:
//
//   mean, var of a sample's rows in a group of C / groups channels, inv = 1 / sqrt(var + eps)
//   u = (x - mean) inv, z = u w + b, y = act(z)
//   dz = dy act'(z), dw = sum dz u, db = sum dz
//   dx = inv (w dz - mean(w dz) - u mean(w dz u))      (means over the same rows and group)
//
// Bound by memory.  x passes twice (the statistics, then the values), in the backward pass x and dy do; the second
// time comes from the caches as far as they hold it.  A thread has V channels (16 bytes) of some rows of
// a chunk.  The statistics of a chunk are each channel's mean and sum of squares about it, formed
// from a few rows in registers and joined by Chan, Golub and LeVeque's formula, so that a mean far
// from zero costs no digits; everything is fp32 and joined in a fixed order.
//
// 240k x 128 bf16 (61 MB) in two samples: moments 19 us (3.2 TB/s), statistics 7, values 27 (4.6 TB/s), the gradients' sums 31
// (4.0), their joins 7, dx 35 (5.3).  What the two joins take is latency: a launch of few workgroups and a
// batch of loads (one load after the other: 9).
#include "sp_attention.h"  // sequences in packed rows

namespace sp {

constexpr int kNormThreads = 256;
constexpr int kNormRows = 4;       // rows of a thread at a time; chunks are whole steps of them
constexpr int kNormLoads = 8;      // partials that a thread of a join loads at a time
constexpr int kNormChunks = 1024;  // chunks that a call is cut into, about
// Calls of up to so many values, and samples of up to so many on average, take a workgroup a part, in one launch (the
// gradients of several parts in two), for three of several workgroups each.  fp16, 64 channels, us in a graph: one part of 256
// rows 12.3 forward and 9.1 back; of 1 024 rows 19.6 and 16.5, where several workgroups take 14.3 and 11.2; four
// parts of 256 rows 12.7 and 11.6, for 15.6 and 12.6 of several.
constexpr int64_t kNormSmall = 65536, kNormSmallPart = 16384;
constexpr int kSmallThreads = 512;
// The parameters' gradients are summed over the parts in slabs of so many rows, slabs over slabs until one is left: four
// runs of a slab apart and then in order, 64 channels a workgroup.  (A thread a channel going through all parts: a
// backward pass over 65 536 parts of 4 rows of 64 bf16 channels 17 650 us, 1 915 so; of 196 windows of 1 024 rows 80
// and 43; and a chain of 70 000 sums was off by 2^-13.)
constexpr int kNormSlab = 256;

enum { kActNone = 3 };  // beside the feed-forward block's activations

template <typename T, int V>
struct alignas(sizeof(T) * V) NormPiece {
  T v[V];
};

// n values' mean and their sum of squares about it.
struct Moments {
  float n, mean, m2;
  __device__ __forceinline__ void join(float on, float omean, float om2) {
    const float all = n + on;
    if (on == 0.f) return;
    const float d = omean - mean, w = on * __builtin_amdgcn_rcpf(all);  // (one ulp of a weight)
    mean = __builtin_fmaf(d, w, mean);
    m2 += __builtin_fmaf(d * d, n * w, om2);
    n = all;
  }
};

template <bool FAST, int ACT>
__device__ __forceinline__ void norm_act(float z, float& value, float& slope) {
  if constexpr (ACT == kActNone) {
    value = z;
    slope = 1.f;
  } else {
    gate<FAST, ACT>(z, value, slope);
  }
}

// How the threads of a workgroup lie over rows and channels: L threads of V channels a row, `per` rows
// at a time; blocks of L V channels where a row has more.
struct NormShape {
  int C, groups, cg, L, per, blocks;
  int64_t chunk;  // rows
};

template <typename T, typename P>
struct NormArgs {
  const T *x, *dy;
  int64_t ldx, lddy;
  Seqs seqs;
  NormShape s;
  const P *w, *b;
  float eps;
  T *y, *dx;
  P *dw, *db;
  float2* stats;  // [parts][groups]: mean, inv
  float2* part;   // [slots][C]: a chunk's moments; sums of dz and dz u
  float2* sums;   // [parts][C]: sums of dz and dz u
  const float2* rows;  // [n_rows][C]: these, or their sums over slabs of them
  int n_rows;
  float2* back;   // [parts][groups]: mean(w dz), mean(w dz u)
};

// This thread's channels and rows.
struct NormLane {
  int c, row;  // first channel; first row of the chunk, per rows apart
  bool on;
};
template <int V>
__device__ __forceinline__ NormLane norm_lane(const NormShape& s, int block) {
  const int row = int(threadIdx.x) / s.L, c = (block * s.L + int(threadIdx.x) - row * s.L) * V;
  return NormLane{c, row, row < s.per && c < s.C};
}

// Moments of V channels over rows first, first + per, ... below end.
template <int ROWS, typename T, int V>
__device__ __forceinline__ void row_moments(const T* x, int64_t ldx, int64_t first, int64_t end,
                                            int per, int c, Moments (&m)[V]) {
  using vec = NormPiece<T, V>;
#pragma unroll
  for (int i = 0; i < V; ++i) m[i] = Moments{0.f, 0.f, 0.f};
  // (the next rows are loaded before these are summed)
  vec a[2][ROWS];
  auto load = [&](vec (&to)[ROWS], int64_t r) {
#pragma unroll
    for (int j = 0; j < ROWS; ++j) {
      to[j] = vec{};
      if (r + int64_t(j) * per < end)
        to[j] = *reinterpret_cast<const vec*>(x + (r + int64_t(j) * per) * ldx + c);
    }
  };
  auto use = [&](const vec (&v)[ROWS], int64_t r) {
    int n = 0;
#pragma unroll
    for (int j = 0; j < ROWS; ++j) n += r + int64_t(j) * per < end;
    if (n == 0) return;
    const float one = __builtin_amdgcn_rcpf(float(n));
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float sum = 0.f, sq = 0.f;
#pragma unroll
      for (int j = 0; j < ROWS; ++j) sum += to_f32(v[j].v[i]);
      const float mean = sum * one;
#pragma unroll
      for (int j = 0; j < ROWS; ++j) {
        const float d = j < n ? to_f32(v[j].v[i]) - mean : 0.f;
        sq = __builtin_fmaf(d, d, sq);
      }
      m[i].join(float(n), mean, sq);
    }
  };
  const int64_t step = int64_t(per) * ROWS;
  load(a[0], first);
  for (int64_t r = first; r < end; r += 2 * step) {
    load(a[1], r + step);
    use(a[0], r);
    load(a[0], r + 2 * step);
    use(a[1], r + step);
  }
}

// Channel c's moments over the workgroup's `per` rows of threads, from LDS [per][L V].
__device__ __forceinline__ Moments column_moments(const float2* lds, const float* counts, int per,
                                                  int width, int c) {
  Moments m{0.f, 0.f, 0.f};
  for (int r = 0; r < per; ++r) {
    const float2 v = lds[r * width + c];
    m.join(counts[r], v.x, v.y);
  }
  return m;
}

template <typename T, typename P, int V>
__global__ __launch_bounds__(kNormThreads) void norm_moments(NormArgs<T, P> a) {
  __shared__ float2 lds[kNormThreads * V];
  __shared__ float counts[kNormThreads];
  const Tile t = find_tile(a.seqs, 1, int(a.s.chunk), blockIdx.x);
  if (t.at >= t.len || a.seqs.outside(t.part)) return;
  const int64_t end = t.at + a.s.chunk < t.len ? t.at + a.s.chunk : t.len;
  const NormLane l = norm_lane<V>(a.s, int(blockIdx.y));
  const int width = a.s.L * V;
  if (l.on) {
    Moments m[V];
    row_moments<kNormRows, T, V>(a.x + t.lo * a.ldx, a.ldx, t.at + l.row, end, a.s.per, l.c, m);
    const int at = l.c - int(blockIdx.y) * width;
#pragma unroll
    for (int i = 0; i < V; ++i) lds[l.row * width + at + i] = float2{m[i].mean, m[i].m2};
    if (at == 0) counts[l.row] = m[0].n;
  }
  __syncthreads();
  for (int c = int(threadIdx.x); c < width; c += kNormThreads) {
    const int channel = int(blockIdx.y) * width + c;
    if (channel >= a.s.C) break;
    const Moments m = column_moments(lds, counts, a.s.per, width, c);
    a.part[int64_t(blockIdx.x) * a.s.C + channel] = float2{m.mean, m.m2};
  }
}

// Sums of two values, or joined moments, over a workgroup, on every thread.
__device__ __forceinline__ Moments block_moments(Moments m, float* lds) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) {
    const float n = __shfl_xor(m.n, off, 64), mean = __shfl_xor(m.mean, off, 64);
    const float m2 = __shfl_xor(m.m2, off, 64);
    // (both partners join in one order, so that they agree)
    Moments lo = m, hi{n, mean, m2};
    if ((int(threadIdx.x) & off) != 0) {
      lo = hi;
      hi = m;
    }
    lo.join(hi.n, hi.mean, hi.m2);
    m = lo;
  }
  const int wave = int(threadIdx.x) >> 6;
  if ((threadIdx.x & 63) == 0) {
    lds[3 * wave] = m.n;
    lds[3 * wave + 1] = m.mean;
    lds[3 * wave + 2] = m.m2;
  }
  __syncthreads();
  Moments all{0.f, 0.f, 0.f};
#pragma unroll
  for (int w = 0; w < kNormThreads / 64; ++w) all.join(lds[3 * w], lds[3 * w + 1], lds[3 * w + 2]);
  return all;
}

// The chunks of part p: the first one's slot, and how many.
struct PartChunks {
  int64_t slot, n, len;
};
__device__ __forceinline__ PartChunks part_chunks(const Seqs& s, int64_t chunk, int p) {
  const int64_t lo = s.bound(p), hi = s.bound(p + 1), len = hi > lo ? hi - lo : 0;
  return PartChunks{lo / chunk + p, (len + chunk - 1) / chunk, len};
}

// A part's group: its chunks' and channels' moments joined.
template <typename T, typename P>
__global__ __launch_bounds__(kNormThreads) void norm_stats(NormArgs<T, P> a) {
  __shared__ float lds[3 * kNormThreads / 64];
  const int p = int(blockIdx.x) / a.s.groups, g = int(blockIdx.x) % a.s.groups;
  if (a.seqs.outside(p)) return;
  const PartChunks k = part_chunks(a.seqs, a.s.chunk, p);
  if (k.len == 0) return;
  Moments m{0.f, 0.f, 0.f};
  // (neighbouring threads take a chunk's channels)
  const int wide = a.s.cg < kNormThreads ? a.s.cg : kNormThreads, rows = kNormThreads / wide;
  const int row = int(threadIdx.x) / wide;
  if (row < rows)
    for (int c = int(threadIdx.x) - row * wide; c < a.s.cg; c += wide) {
      const float2* at = a.part + k.slot * a.s.C + g * a.s.cg + c;
      for (int j = row; j < int(k.n); j += kNormLoads * rows) {
        float2 v[kNormLoads];
#pragma unroll
        for (int i = 0; i < kNormLoads; ++i) {
          const int r = j + i * rows;
          v[i] = at[int64_t(r < k.n ? r : j) * a.s.C];
        }
#pragma unroll
        for (int i = 0; i < kNormLoads; ++i) {
          const int r = j + i * rows;
          if (r < k.n)
            m.join(float(r + 1 < k.n ? a.s.chunk : k.len - r * a.s.chunk), v[i].x, v[i].y);
        }
      }
    }
  m = block_moments(m, lds);
  if (threadIdx.x == 0)
    a.stats[blockIdx.x] = float2{m.mean, 1.f / sqrtf(m.m2 / m.n + a.eps)};
}

// What a thread needs of its channels.
template <int V>
struct NormChannels {
  float mean[V], inv[V], w[V], b[V];
  template <typename P>
  __device__ __forceinline__ NormChannels(const NormShape& s, const float2* stats, const P* wt,
                                          const P* bt, int c) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float2 st = stats[(c + i) / s.cg];
      mean[i] = st.x;
      inv[i] = st.y;
      w[i] = wt ? to_f32(wt[c + i]) : 1.f;
      b[i] = bt ? to_f32(bt[c + i]) : 0.f;
    }
  }
};

// f(pointer offset row) over a thread's rows, kNormRows at a time.
template <int ROWS, typename T, int V, int ACT>
__device__ __forceinline__ void norm_rows(const T* x, int64_t ldx, T* y, int64_t ldy, int64_t first,
                                          int64_t end, int per, int c, const NormChannels<V>& k) {
  using vec = NormPiece<T, V>;
  constexpr bool FAST = sizeof(T) == 2;
  for (int64_t r = first; r < end; r += int64_t(per) * ROWS) {
    vec a[ROWS];
#pragma unroll
    for (int j = 0; j < ROWS; ++j)
      if (r + int64_t(j) * per < end)
        a[j] = *reinterpret_cast<const vec*>(x + (r + int64_t(j) * per) * ldx + c);
#pragma unroll
    for (int j = 0; j < ROWS; ++j) {
      if (r + int64_t(j) * per >= end) break;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float u = (to_f32(a[j].v[i]) - k.mean[i]) * k.inv[i];
        float value, slope;
        norm_act<FAST, ACT>(__builtin_fmaf(u, k.w[i], k.b[i]), value, slope);
        a[j].v[i] = from_f32<T>(value);
      }
      *reinterpret_cast<vec*>(y + (r + int64_t(j) * per) * ldy + c) = a[j];
    }
  }
}

template <typename T, int V>
__device__ __forceinline__ void zero_rows(T* y, int64_t ld, int64_t first, int64_t end, int per,
                                          int c) {
  for (int64_t r = first; r < end; r += per)
    *reinterpret_cast<NormPiece<T, V>*>(y + r * ld + c) = NormPiece<T, V>{};
}

template <typename T, typename P, int V, int ACT>
__global__ __launch_bounds__(kNormThreads) void norm_apply(NormArgs<T, P> a) {
  const Tile t = find_tile(a.seqs, 1, int(a.s.chunk), blockIdx.x);
  if (t.at >= t.len) return;
  const int64_t end = t.at + a.s.chunk < t.len ? t.at + a.s.chunk : t.len;
  const NormLane l = norm_lane<V>(a.s, int(blockIdx.y));
  if (!l.on) return;
  T* y = a.y + t.lo * a.s.C;
  if (a.seqs.outside(t.part)) {
    zero_rows<T, V>(y, a.s.C, t.at + l.row, end, a.s.per, l.c);
    return;
  }
  const NormChannels<V> k(a.s, a.stats + int64_t(t.part) * a.s.groups, a.w, a.b, l.c);
  norm_rows<kNormRows, T, V, ACT>(a.x + t.lo * a.ldx, a.ldx, y, a.s.C, t.at + l.row, end, a.s.per, l.c, k);
}

// ---- gradients ---------------------------------------------------------------------
// Sums of dz and dz u of V channels over rows first, first + per, ...
template <int ROWS, typename T, int V, int ACT>
__device__ __forceinline__ void row_sums(const T* x, int64_t ldx, const T* dy, int64_t lddy,
                                         int64_t first, int64_t end, int per, int c,
                                         const NormChannels<V>& k, float (&s1)[V],
                                         float (&s2)[V]) {
  using vec = NormPiece<T, V>;
  constexpr bool FAST = sizeof(T) == 2;
#pragma unroll
  for (int i = 0; i < V; ++i) s1[i] = s2[i] = 0.f;
  vec a[2][ROWS], d[2][ROWS];
  auto load = [&](int s, int64_t r) {
#pragma unroll
    for (int j = 0; j < ROWS; ++j) {
      a[s][j] = d[s][j] = vec{};
      if (r + int64_t(j) * per < end) {
        a[s][j] = *reinterpret_cast<const vec*>(x + (r + int64_t(j) * per) * ldx + c);
        d[s][j] = *reinterpret_cast<const vec*>(dy + (r + int64_t(j) * per) * lddy + c);
      }
    }
  };
  auto use = [&](int s, int64_t r) {
#pragma unroll
    for (int j = 0; j < ROWS; ++j) {
      if (r + int64_t(j) * per >= end) break;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float u = (to_f32(a[s][j].v[i]) - k.mean[i]) * k.inv[i];
        float value, slope;
        norm_act<FAST, ACT>(__builtin_fmaf(u, k.w[i], k.b[i]), value, slope);
        const float dz = to_f32(d[s][j].v[i]) * slope;
        s1[i] += dz;
        s2[i] = __builtin_fmaf(dz, u, s2[i]);
      }
    }
  };
  const int64_t step = int64_t(per) * ROWS;
  load(0, first);
  for (int64_t r = first; r < end; r += 2 * step) {
    load(1, r + step);
    use(0, r);
    load(0, r + 2 * step);
    use(1, r + step);
  }
}

// a b - c with the product rounded, as it was when c was summed up: where c is the mean of one value, the
// difference is zero.
__device__ __forceinline__ float less(float a, float b, float c) {
#pragma clang fp contract(off)
  const float p = a * b;
  return p - c;
}

template <int ROWS, typename T, int V, int ACT>
__device__ __forceinline__ void grad_rows(const T* x, int64_t ldx, const T* dy, int64_t lddy, T* dx,
                                          int64_t lddx, int64_t first, int64_t end, int per, int c,
                                          const NormChannels<V>& k, const float (&m1)[V],
                                          const float (&m2)[V]) {
  using vec = NormPiece<T, V>;
  constexpr bool FAST = sizeof(T) == 2;
  for (int64_t r = first; r < end; r += int64_t(per) * ROWS) {
    vec a[ROWS], d[ROWS];
#pragma unroll
    for (int j = 0; j < ROWS; ++j)
      if (r + int64_t(j) * per < end) {
        a[j] = *reinterpret_cast<const vec*>(x + (r + int64_t(j) * per) * ldx + c);
        d[j] = *reinterpret_cast<const vec*>(dy + (r + int64_t(j) * per) * lddy + c);
      }
#pragma unroll
    for (int j = 0; j < ROWS; ++j) {
      if (r + int64_t(j) * per >= end) break;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float u = (to_f32(a[j].v[i]) - k.mean[i]) * k.inv[i];
        float value, slope;
        norm_act<FAST, ACT>(__builtin_fmaf(u, k.w[i], k.b[i]), value, slope);
        a[j].v[i] = from_f32<T>(
            k.inv[i] * __builtin_fmaf(-u, m2[i], less(to_f32(d[j].v[i]) * slope, k.w[i], m1[i])));
      }
      *reinterpret_cast<vec*>(dx + (r + int64_t(j) * per) * lddx + c) = a[j];
    }
  }
}

// (two rows a thread and twice as many on their way: with four, 194 registers, a CU holds half as many workgroups)
template <typename T, typename P, int V, int ACT>
__global__ __launch_bounds__(kNormThreads, 4) void norm_grad_sums(NormArgs<T, P> a) {
  __shared__ float2 lds[kNormThreads * V];
  const Tile t = find_tile(a.seqs, 1, int(a.s.chunk), blockIdx.x);
  if (t.at >= t.len || a.seqs.outside(t.part)) return;
  const int64_t end = t.at + a.s.chunk < t.len ? t.at + a.s.chunk : t.len;
  const NormLane l = norm_lane<V>(a.s, int(blockIdx.y));
  const int width = a.s.L * V;
  if (l.on) {
    const NormChannels<V> k(a.s, a.stats + int64_t(t.part) * a.s.groups, a.w, a.b, l.c);
    float s1[V], s2[V];
    row_sums<2, T, V, ACT>(a.x + t.lo * a.ldx, a.ldx, a.dy + t.lo * a.lddy, a.lddy, t.at + l.row, end,
                        a.s.per, l.c, k, s1, s2);
    const int at = l.c - int(blockIdx.y) * width;
#pragma unroll
    for (int i = 0; i < V; ++i) lds[l.row * width + at + i] = float2{s1[i], s2[i]};
  }
  __syncthreads();
  for (int c = int(threadIdx.x); c < width; c += kNormThreads) {
    const int channel = int(blockIdx.y) * width + c;
    if (channel >= a.s.C) break;
    float2 v{0.f, 0.f};
    for (int r = 0; r < a.s.per; ++r) {
      v.x += lds[r * width + c].x;
      v.y += lds[r * width + c].y;
    }
    a.part[int64_t(blockIdx.x) * a.s.C + channel] = v;
  }
}

// A part's group: its channels' sums over the chunks, and from them the group's means.  A wave a
// channel at a time.
template <typename T, typename P>
__global__ __launch_bounds__(kNormThreads) void norm_grad_join(NormArgs<T, P> a) {
  __shared__ float2 lds[kNormThreads / 64];
  const int p = int(blockIdx.x) / a.s.groups, g = int(blockIdx.x) % a.s.groups;
  const PartChunks k = part_chunks(a.seqs, a.s.chunk, p);
  const int64_t n = a.seqs.outside(p) ? 0 : k.n;
  const int wave = int(threadIdx.x) >> 6, lane = int(threadIdx.x) & 63;
  float2 mine{0.f, 0.f};
  for (int j = wave; j < a.s.cg; j += kNormThreads / 64) {
    const int c = g * a.s.cg + j;
    float2 v{0.f, 0.f};
    for (int64_t i = lane; i < n; i += 64 * kNormLoads) {
      float2 o[kNormLoads];
#pragma unroll
      for (int l = 0; l < kNormLoads; ++l)
        o[l] = a.part[(k.slot + (i + 64 * l < n ? i + 64 * l : i)) * a.s.C + c];
#pragma unroll
      for (int l = 0; l < kNormLoads; ++l) {
        v.x += i + 64 * l < n ? o[l].x : 0.f;
        v.y += i + 64 * l < n ? o[l].y : 0.f;
      }
    }
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) {
      v.x += __shfl_xor(v.x, off, 64);
      v.y += __shfl_xor(v.y, off, 64);
    }
    if (lane == 0) a.sums[int64_t(p) * a.s.C + c] = v;
    const float w = a.w ? to_f32(a.w[c]) : 1.f;
    mine.x = __builtin_fmaf(v.x, w, mine.x);
    mine.y = __builtin_fmaf(v.y, w, mine.y);
  }
  if (lane == 0) lds[wave] = mine;
  __syncthreads();
  if (threadIdx.x != 0) return;
  float2 all = lds[0];
#pragma unroll
  for (int w = 1; w < kNormThreads / 64; ++w) {
    all.x += lds[w].x;
    all.y += lds[w].y;
  }
  const float count = float(k.len) * float(a.s.cg);
  a.back[blockIdx.x] = n ? float2{all.x / count, all.y / count} : float2{0.f, 0.f};
}

// The sum of rows first .. end - 1 at 64 channels from c0 on, a channel a lane of the first wave.
__device__ __forceinline__ float2 sum_rows(const float2* rows, int64_t first, int64_t end, int C,
                                           int c0) {
  static_assert(kNormThreads == 256, "four runs");
  __shared__ float2 lds[4][64];
  const int lane = int(threadIdx.x) & 63, run = int(threadIdx.x) >> 6, c = c0 + lane;
  float2 v{0.f, 0.f};
  if (c < C) {
    const int64_t per = (end - first + 3) / 4, lo = first + run * per;
    const int64_t hi = lo + per < end ? lo + per : end;
    for (int64_t r = lo; r < hi; r += kNormLoads) {
      float2 o[kNormLoads];
#pragma unroll
      for (int i = 0; i < kNormLoads; ++i) o[i] = rows[(r + i < hi ? r + i : r) * C + c];
#pragma unroll
      for (int i = 0; i < kNormLoads; ++i) {
        v.x += r + i < hi ? o[i].x : 0.f;
        v.y += r + i < hi ? o[i].y : 0.f;
      }
    }
  }
  lds[run][lane] = v;
  __syncthreads();
#pragma unroll
  for (int k = 1; k < 4; ++k) {
    v.x += lds[k][lane].x;
    v.y += lds[k][lane].y;
  }
  return v;  // (of use to the first wave: its own run and the others in order)
}

// The sums of the slabs of rows [n][C], a row each.
__global__ __launch_bounds__(kNormThreads) void norm_slabs(const float2* __restrict__ rows, int n,
                                                           int C, float2* __restrict__ out) {
  const int blocks = (C + 63) / 64;
  const int64_t slab = blockIdx.x / blocks, first = slab * kNormSlab;
  const int c0 = int(blockIdx.x - slab * blocks) * 64;
  const float2 v = sum_rows(rows, first, first + kNormSlab < n ? first + kNormSlab : n, C, c0);
  const int c = c0 + int(threadIdx.x);
  if (threadIdx.x < 64 && c < C) out[slab * C + c] = v;
}

// The parameters' gradients of 64 channels.
template <typename T, typename P>
__device__ __forceinline__ void write_params(const NormArgs<T, P>& a, int c0) {
  const float2 v = sum_rows(a.rows, 0, a.n_rows, a.s.C, c0);
  const int c = c0 + int(threadIdx.x);
  if (threadIdx.x >= 64 || c >= a.s.C) return;
  if (a.dw) a.dw[c] = from_f32<P>(v.y);
  if (a.db) a.db[c] = from_f32<P>(v.x);
}

// dx; the workgroups from `slots` on sum the parameters' gradients.
template <typename T, typename P, int V, int ACT>
__global__ __launch_bounds__(kNormThreads) void norm_grad_apply(NormArgs<T, P> a, int64_t slots) {
  if (int64_t(blockIdx.x) >= slots) {
    if (blockIdx.y == 0) write_params(a, int(blockIdx.x - slots) * 64);
    return;
  }
  if (!a.dx) return;
  const Tile t = find_tile(a.seqs, 1, int(a.s.chunk), blockIdx.x);
  if (t.at >= t.len) return;
  const int64_t end = t.at + a.s.chunk < t.len ? t.at + a.s.chunk : t.len;
  const NormLane l = norm_lane<V>(a.s, int(blockIdx.y));
  if (!l.on) return;
  T* dx = a.dx + t.lo * a.s.C;
  if (a.seqs.outside(t.part)) {
    zero_rows<T, V>(dx, a.s.C, t.at + l.row, end, a.s.per, l.c);
    return;
  }
  const NormChannels<V> k(a.s, a.stats + int64_t(t.part) * a.s.groups, a.w, a.b, l.c);
  float m1[V], m2[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const float2 v = a.back[int64_t(t.part) * a.s.groups + (l.c + i) / a.s.cg];
    m1[i] = v.x;
    m2[i] = v.y;
  }
  grad_rows<kNormRows, T, V, ACT>(a.x + t.lo * a.ldx, a.ldx, a.dy + t.lo * a.lddy, a.lddy, dx, a.s.C,
                       t.at + l.row, end, a.s.per, l.c, k, m1, m2);
}

// ---- small calls: a workgroup a part -------------------------------------------------
template <typename T, typename P, int V, int ACT>
__global__ __launch_bounds__(kSmallThreads) void norm_small(NormArgs<T, P> a) {
  __shared__ float2 lds[kSmallThreads * V];
  __shared__ float counts[kSmallThreads];
  const NormLane l = norm_lane<V>(a.s, 0);
  const int width = a.s.L * V, p = int(blockIdx.x);
  const int64_t lo = a.seqs.bound(p), hi = a.seqs.bound(p + 1), len = hi > lo ? hi - lo : 0;
  if (len == 0) return;
  T* y = a.y + lo * a.s.C;
  if (a.seqs.outside(p)) {
    if (l.on) zero_rows<T, V>(y, a.s.C, l.row, len, a.s.per, l.c);
    return;
  }
  const T* x = a.x + lo * a.ldx;
  if (l.on) {
    Moments m[V];
    row_moments<2, T, V>(x, a.ldx, l.row, len, a.s.per, l.c, m);
#pragma unroll
    for (int i = 0; i < V; ++i) lds[l.row * width + l.c + i] = float2{m[i].mean, m[i].m2};
    if (l.c == 0) counts[l.row] = m[0].n;
  }
  __syncthreads();
  for (int c = int(threadIdx.x); c < a.s.C; c += kSmallThreads) {
    const Moments m = column_moments(lds, counts, a.s.per, width, c);
    lds[c] = float2{m.mean, m.m2};  // (its own column's first place)
  }
  __syncthreads();
  float2* stats = a.stats + int64_t(p) * a.s.groups;
  for (int g = int(threadIdx.x); g < a.s.groups; g += kSmallThreads) {
    Moments m{0.f, 0.f, 0.f};
    for (int c = g * a.s.cg; c < (g + 1) * a.s.cg; ++c) m.join(float(len), lds[c].x, lds[c].y);
    stats[g] = float2{m.mean, 1.f / sqrtf(m.m2 / m.n + a.eps)};
  }
  __syncthreads();  // (which makes the workgroup's own stores to memory visible to it)
  if (!l.on) return;
  const NormChannels<V> k(a.s, stats, a.w, a.b, l.c);
  norm_rows<2, T, V, ACT>(x, a.ldx, y, a.s.C, l.row, len, a.s.per, l.c, k);
}

template <typename T, typename P, int V, int ACT>
__global__ __launch_bounds__(kSmallThreads) void norm_grad_small(NormArgs<T, P> a) {
  __shared__ float2 lds[kSmallThreads * V];
  const NormLane l = norm_lane<V>(a.s, 0);
  const int width = a.s.L * V, p = int(blockIdx.x);
  const int64_t lo = a.seqs.bound(p), hi = a.seqs.bound(p + 1), len = hi > lo ? hi - lo : 0;
  const bool outside = a.seqs.outside(p);
  if (len == 0 || outside) {
    if (outside && l.on && a.dx)
      zero_rows<T, V>(a.dx + lo * a.s.C, a.s.C, l.row, len, a.s.per, l.c);
    if (a.seqs.parts > 1)
      for (int c = int(threadIdx.x); c < a.s.C; c += kSmallThreads)
        a.sums[int64_t(p) * a.s.C + c] = float2{0.f, 0.f};
    return;
  }
  const NormChannels<V> k(a.s, a.stats + int64_t(p) * a.s.groups, a.w, a.b, l.on ? l.c : 0);
  const T* x = a.x + lo * a.ldx;
  const T* dy = a.dy + lo * a.lddy;
  if (l.on) {
    float s1[V], s2[V];
    row_sums<2, T, V, ACT>(x, a.ldx, dy, a.lddy, l.row, len, a.s.per, l.c, k, s1, s2);
#pragma unroll
    for (int i = 0; i < V; ++i) lds[l.row * width + l.c + i] = float2{s1[i], s2[i]};
  }
  __syncthreads();
  for (int c = int(threadIdx.x); c < a.s.C; c += kSmallThreads) {
    float2 v{0.f, 0.f};
    for (int r = 0; r < a.s.per; ++r) {
      v.x += lds[r * width + c].x;
      v.y += lds[r * width + c].y;
    }
    lds[c] = v;  // (its own column's first place)
    if (a.seqs.parts > 1) {
      a.sums[int64_t(p) * a.s.C + c] = v;
    } else {
      if (a.dw) a.dw[c] = from_f32<P>(v.y);
      if (a.db) a.db[c] = from_f32<P>(v.x);
    }
  }
  __syncthreads();
  if (!l.on || !a.dx) return;
  const float count = float(len) * float(a.s.cg);
  float m1[V], m2[V];
  int at = -1;
  float2 all{0.f, 0.f};
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int g = (l.c + i) / a.s.cg;
    if (g != at) {
      all = float2{0.f, 0.f};
      for (int c = g * a.s.cg; c < (g + 1) * a.s.cg; ++c) {
        const float w = a.w ? to_f32(a.w[c]) : 1.f;
        all.x = __builtin_fmaf(lds[c].x, w, all.x);
        all.y = __builtin_fmaf(lds[c].y, w, all.y);
      }
      at = g;
    }
    m1[i] = all.x / count;
    m2[i] = all.y / count;
  }
  grad_rows<2, T, V, ACT>(x, a.ldx, dy, a.lddy, a.dx + lo * a.s.C, a.s.C, l.row, len, a.s.per, l.c, k,
                          m1, m2);
}

// The parameters' gradients from the parts' sums.
template <typename T, typename P>
__global__ __launch_bounds__(kNormThreads) void norm_grad_params(NormArgs<T, P> a) {
  write_params(a, int(blockIdx.x) * 64);
}

// ---- host ------------------------------------------------------------------------
static NormShape norm_shape(int64_t rows, int C, int groups, int V, int threads = kNormThreads) {
  NormShape s{};
  s.C = C;
  s.groups = groups;
  s.cg = C / groups;
  s.L = C / V < threads ? C / V : threads;
  s.per = threads / s.L;
  s.blocks = int(cdiv(C, s.L * V));
  const int64_t step = int64_t(s.per) * kNormRows;
  s.chunk = cdiv(cdiv(rows, kNormChunks), step) * step;
  return s;
}

// (a row that is wider than a workgroup goes by blocks of its channels)
static bool norm_is_small(int64_t rows, int64_t C, const Seqs& q, int V) {
  const int64_t samples = q.parts > 2 ? q.parts - 2 : 1, n = rows * C;
  return n <= kNormSmall && n <= kNormSmallPart * samples && C <= kSmallThreads * V;
}

static Seqs norm_seqs(const int32_t* off, int64_t rows, int64_t n) {
  return Seqs{off, rows, off ? int(n) + 2 : 1};
}

static size_t slabs_bytes(int64_t parts, int64_t C) {
  return parts > kNormSlab ? align_up(size_t(cdiv(parts, kNormSlab)) * C * sizeof(float2), 256) : 0;
}

constexpr int64_t kNormMaxGroups = max_groups(kNormThreads);

static int64_t slab_groups(int64_t parts, int64_t C) {
  return parts > kNormSlab ? cdiv(parts, kNormSlab) * cdiv(C, 64) : 0;
}

// At most kNormSlab rows that add up to those of the parts: a.rows, between a.sums and the workspace at `slabs`.
template <typename T, typename P>
static int join_parts(NormArgs<T, P>& a, char* slabs, hipStream_t st) {
  float2 *from = a.sums, *to = reinterpret_cast<float2*>(slabs);
  int64_t n = a.seqs.parts;
  while (n > kNormSlab && (a.dw || a.db)) {
    const int64_t next = cdiv(n, kNormSlab);
    norm_slabs<<<unsigned(slab_groups(n, a.s.C)), kNormThreads, 0, st>>>(from, int(n), a.s.C, to);
    SP_LAUNCHED();
    float2* const read = from;
    from = to;
    to = read;
    n = next;
  }
  a.rows = from;
  a.n_rows = int(n);
  return SP_OK;
}

// (the sizes do not depend on V, which the tensors' addresses decide)
static size_t norm_workspace(int64_t rows, int64_t C, int64_t groups, const Seqs& q, int V,
                             bool grad) {
  const size_t sums = align_up(size_t(q.parts) * C * sizeof(float2), 256) + slabs_bytes(q.parts, C);
  if (norm_is_small(rows, C, q, V)) return grad && q.parts > 1 ? sums : 0;
  const NormShape s = norm_shape(rows, int(C), int(groups), V);
  size_t n = align_up(size_t(tile_slots(q, 1, int(s.chunk))) * C * sizeof(float2), 256);
  if (grad)
    n += sums + align_up(size_t(q.parts) * groups * sizeof(float2), 256);
  return n;
}

template <typename F>
static int norm_act_of(int act, F&& f) {
  switch (act) {
    case kActSilu: return f(std::integral_constant<int, kActSilu>());
    case kActGelu: return f(std::integral_constant<int, kActGelu>());
    case kActRelu: return f(std::integral_constant<int, kActRelu>());
    default: return f(std::integral_constant<int, kActNone>());
  }
}

template <typename T, typename P, int V>
static int norm_forward(NormArgs<T, P> a, int act, char* ws, hipStream_t st) {
  if (norm_is_small(a.seqs.rows, a.s.C, a.seqs, V)) {
    SP_CHECK_ARG(a.seqs.parts <= max_groups(kSmallThreads),
                 "group_norm: too many samples for a launch");
    a.s = norm_shape(a.seqs.rows, a.s.C, a.s.groups, V, kSmallThreads);
    norm_act_of(act, [&](auto k) {
      norm_small<T, P, V, k.value><<<unsigned(a.seqs.parts), kSmallThreads, 0, st>>>(a);
      return 0;
    });
    SP_LAUNCHED();
    return SP_OK;
  }
  a.s = norm_shape(a.seqs.rows, a.s.C, a.s.groups, V);
  const int64_t slots = tile_slots(a.seqs, 1, int(a.s.chunk));
  const int64_t joins = int64_t(a.seqs.parts) * a.s.groups;
  SP_CHECK_ARG(slots * a.s.blocks <= kNormMaxGroups && joins <= kNormMaxGroups,
               "group_norm: too many samples for a launch");
  a.part = reinterpret_cast<float2*>(ws);
  const dim3 grid(unsigned(slots), unsigned(a.s.blocks));
  norm_moments<T, P, V><<<grid, kNormThreads, 0, st>>>(a);
  SP_LAUNCHED();
  norm_stats<T, P><<<unsigned(joins), kNormThreads, 0, st>>>(a);
  SP_LAUNCHED();
  norm_act_of(act, [&](auto k) {
    norm_apply<T, P, V, k.value><<<grid, kNormThreads, 0, st>>>(a);
    return 0;
  });
  SP_LAUNCHED();
  return SP_OK;
}

template <typename T, typename P, int V>
static int norm_backward(NormArgs<T, P> a, int act, char* ws, hipStream_t st) {
  if (norm_is_small(a.seqs.rows, a.s.C, a.seqs, V)) {
    SP_CHECK_ARG(a.seqs.parts <= max_groups(kSmallThreads) &&
                     slab_groups(a.seqs.parts, a.s.C) <= kNormMaxGroups,
                 "group_norm_bwd: too many samples for a launch");
    a.s = norm_shape(a.seqs.rows, a.s.C, a.s.groups, V, kSmallThreads);
    a.sums = reinterpret_cast<float2*>(ws);
    norm_act_of(act, [&](auto k) {
      norm_grad_small<T, P, V, k.value><<<unsigned(a.seqs.parts), kSmallThreads, 0, st>>>(a);
      return 0;
    });
    SP_LAUNCHED();
    if (a.seqs.parts == 1 || !(a.dw || a.db)) return SP_OK;
    ws += align_up(size_t(a.seqs.parts) * a.s.C * sizeof(float2), 256);
    if (int rc = join_parts(a, ws, st)) return rc;
    norm_grad_params<T, P><<<unsigned(cdiv(a.s.C, 64)), kNormThreads, 0, st>>>(a);
    SP_LAUNCHED();
    return SP_OK;
  }
  a.s = norm_shape(a.seqs.rows, a.s.C, a.s.groups, V);
  const int64_t slots = tile_slots(a.seqs, 1, int(a.s.chunk));
  const int64_t joins = int64_t(a.seqs.parts) * a.s.groups;
  const int64_t extra = a.dw || a.db ? cdiv(a.s.C, 64) : 0;
  SP_CHECK_ARG((slots + extra) * a.s.blocks <= kNormMaxGroups && joins <= kNormMaxGroups &&
                   slab_groups(a.seqs.parts, a.s.C) <= kNormMaxGroups,
               "group_norm_bwd: too many samples for a launch");
  a.part = reinterpret_cast<float2*>(ws);
  ws += align_up(size_t(slots) * a.s.C * sizeof(float2), 256);
  a.sums = reinterpret_cast<float2*>(ws);
  ws += align_up(size_t(a.seqs.parts) * a.s.C * sizeof(float2), 256);
  char* const slabs = ws;
  ws += slabs_bytes(a.seqs.parts, a.s.C);
  a.back = reinterpret_cast<float2*>(ws);
  const dim3 grid(unsigned(slots), unsigned(a.s.blocks));
  norm_act_of(act, [&](auto k) {
    norm_grad_sums<T, P, V, k.value><<<grid, kNormThreads, 0, st>>>(a);
    return 0;
  });
  SP_LAUNCHED();
  norm_grad_join<T, P><<<unsigned(joins), kNormThreads, 0, st>>>(a);
  SP_LAUNCHED();
  if (int rc = join_parts(a, slabs, st)) return rc;
  const dim3 last(unsigned(slots + extra), unsigned(a.s.blocks));
  norm_act_of(act, [&](auto k) {
    norm_grad_apply<T, P, V, k.value><<<last, kNormThreads, 0, st>>>(a, slots);
    return 0;
  });
  SP_LAUNCHED();
  return SP_OK;
}

static int check_norm(const char* what, int32_t dtype, int64_t rows, int64_t C, int64_t groups,
                      int32_t param_dtype, float eps, int32_t act, const int32_t* offsets,
                      int64_t samples) {
  SP_CHECK_ARG(dtype == SP_F16 || dtype == SP_BF16 || dtype == SP_F32,
               "%s: dtype %d not supported (f16/bf16/f32)", what, dtype);
  SP_CHECK_ARG(param_dtype == dtype || param_dtype == SP_F32,
               "%s: parameters of type %d for rows of type %d", what, param_dtype, dtype);
  SP_CHECK_ARG(rows >= 0 && rows < (int64_t(1) << 31) && C >= 1 && C < 65536,
               "%s: bad sizes rows=%lld C=%lld", what, (long long)rows, (long long)C);
  SP_CHECK_ARG(groups >= 1 && groups <= C && C % groups == 0, "%s: %lld channels in %lld groups",
               what, (long long)C, (long long)groups);
  SP_CHECK_ARG(eps >= 0.f && eps < __builtin_inff(), "%s: bad eps", what);
  SP_CHECK_ARG(act >= kActSilu && act <= kActNone, "%s: unknown activation %d", what, act);
  SP_CHECK_ARG(!offsets || (samples >= 0 && samples < (1 << 24)), "%s: bad number of samples %lld",
               what, (long long)samples);
  return SP_OK;
}

template <typename T, typename P, typename F>
static int norm_width(const NormArgs<T, P>& a, bool vec, F&& run) {
  constexpr int V = Mfma<T>::V;
  if (vec) return run(a, std::integral_constant<int, V>());
  return run(a, std::integral_constant<int, 1>());
}

template <typename F>
static int norm_types(int32_t dtype, int32_t param_dtype, F&& f) {
  if (dtype == SP_F32) return f(float(), float());
  if (dtype == SP_F16)
    return param_dtype == SP_F16 ? f(_Float16(), _Float16()) : f(_Float16(), float());
  return param_dtype == SP_BF16 ? f(__bf16(), __bf16()) : f(__bf16(), float());
}

}  // namespace sp

using namespace sp;

extern "C" size_t sp_group_norm_workspace(int32_t dtype, int64_t rows, int64_t C, int64_t groups,
                                          int64_t samples, int32_t backward) {
  if (check_norm("group_norm", dtype, rows, C, groups, dtype, 0.f, kActNone, nullptr, 0) != SP_OK ||
      rows == 0 || samples >= (1 << 24))
    return 0;
  const Seqs q{nullptr, rows, samples >= 0 ? int(samples) + 2 : 1};
  const size_t one = norm_workspace(rows, C, groups, q, 1, backward != 0);
  if (C % vec_of(dtype) != 0) return one;
  const size_t vec = norm_workspace(rows, C, groups, q, vec_of(dtype), backward != 0);
  return one > vec ? one : vec;
}

extern "C" int sp_group_norm(const void* x, int64_t ldx, int32_t dtype, int64_t rows, int64_t C,
                             int64_t groups, const void* weight, const void* bias,
                             int32_t param_dtype, float eps, int32_t act, const int32_t* offsets,
                             int64_t samples, void* y, float* stats, void* ws, size_t ws_bytes,
                             void* stream) {
  if (int rc = check_norm("group_norm", dtype, rows, C, groups, param_dtype, eps, act, offsets,
                          samples))
    return rc;
  if (rows == 0) return SP_OK;
  SP_CHECK_ARG(x && y && stats, "group_norm: null pointer");
  SP_CHECK_ARG(ldx >= C, "group_norm: rows overlap");
  const size_t need =
      sp_group_norm_workspace(dtype, rows, C, groups, offsets ? samples : -1, 0);
  if (ws_bytes < need)
    return set_error(SP_ERR_WORKSPACE, "group_norm: workspace of %zu bytes, needs %zu", ws_bytes,
                     need);
  SP_CHECK_ARG(!need || (ws && aligned(ws)), "group_norm: the workspace must be 16-byte aligned");
  return norm_types(dtype, param_dtype, [&](auto t, auto p) {
    using T = decltype(t);
    using P = decltype(p);
    NormArgs<T, P> a{};
    a.x = static_cast<const T*>(x);
    a.ldx = ldx;
    a.seqs = norm_seqs(offsets, rows, samples);
    a.s.C = int(C);
    a.s.groups = int(groups);
    a.w = static_cast<const P*>(weight);
    a.b = static_cast<const P*>(bias);
    a.eps = eps;
    a.y = static_cast<T*>(y);
    a.stats = reinterpret_cast<float2*>(stats);
    const int V = vec_of(dtype);
    const bool vec = C % V == 0 && ldx % V == 0 && aligned(x) && aligned(y);
    return norm_width(a, vec, [&](const auto& args, auto v) {
      return norm_forward<T, P, v.value>(args, act, static_cast<char*>(ws), as_stream(stream));
    });
  });
}

extern "C" int sp_group_norm_bwd(const void* dy, int64_t lddy, const void* x, int64_t ldx,
                                 int32_t dtype, int64_t rows, int64_t C, int64_t groups,
                                 const void* weight, const void* bias, int32_t param_dtype,
                                 int32_t act, const int32_t* offsets, int64_t samples,
                                 const float* stats, void* dx, void* dweight, void* dbias, void* ws,
                                 size_t ws_bytes, void* stream) {
  if (int rc = check_norm("group_norm_bwd", dtype, rows, C, groups, param_dtype, 0.f, act, offsets,
                          samples))
    return rc;
  if (rows == 0) return SP_OK;
  SP_CHECK_ARG(dy && x && stats, "group_norm_bwd: null pointer");
  SP_CHECK_ARG(ldx >= C && lddy >= C, "group_norm_bwd: rows overlap");
  const size_t need =
      sp_group_norm_workspace(dtype, rows, C, groups, offsets ? samples : -1, 1);
  if (ws_bytes < need)
    return set_error(SP_ERR_WORKSPACE, "group_norm_bwd: workspace of %zu bytes, needs %zu",
                     ws_bytes, need);
  SP_CHECK_ARG(!need || (ws && aligned(ws)),
               "group_norm_bwd: the workspace must be 16-byte aligned");
  return norm_types(dtype, param_dtype, [&](auto t, auto p) {
    using T = decltype(t);
    using P = decltype(p);
    NormArgs<T, P> a{};
    a.x = static_cast<const T*>(x);
    a.dy = static_cast<const T*>(dy);
    a.ldx = ldx;
    a.lddy = lddy;
    a.seqs = norm_seqs(offsets, rows, samples);
    a.s.C = int(C);
    a.s.groups = int(groups);
    a.w = static_cast<const P*>(weight);
    a.b = static_cast<const P*>(bias);
    a.dx = static_cast<T*>(dx);
    a.dw = static_cast<P*>(dweight);
    a.db = static_cast<P*>(dbias);
    a.stats = reinterpret_cast<float2*>(const_cast<float*>(stats));
    const int V = vec_of(dtype);
    const bool vec = C % V == 0 && ldx % V == 0 && lddy % V == 0 && aligned(x) && aligned(dy) &&
                     (!dx || aligned(dx));
    return norm_width(a, vec, [&](const auto& args, auto v) {
      return norm_backward<T, P, v.value>(args, act, static_cast<char*>(ws), as_stream(stream));
    });
  });
}
