// What the attention kernels share: sequences in packed rows, tiles of rows in LDS and the
// operands that the matrix instructions take from them.
#pragma once

#include "sp_ffn.h"  // LDS order, loads to LDS, batched operand reads

namespace sp {

constexpr int kAttnThreads = 256;
constexpr int kAttnWaves = kAttnThreads / 64;
constexpr int kAttnBatch = 2;  // operands read from LDS at a time, while as many are in use

// Rows [rows] in `parts` sequences, sequence p at bound(p) .. bound(p + 1).  With offsets the first and the
// last part are the rows before the first sequence and behind the last one: they have no keys, and
// no queries.  Whatever the offsets hold, a bound lies in the rows.
struct Seqs {
  const int32_t* off;
  int64_t rows;
  int parts;
  __device__ __forceinline__ int64_t bound(int p) const {
    if (p == 0) return 0;
    if (!off || p >= parts) return rows;
    const int64_t b = off[p - 1];
    return b < 0 ? 0 : b < rows ? b : rows;
  }
  __device__ __forceinline__ bool outside(int p) const { return off && (p == 0 || p + 1 == parts); }
};

// A sequence's tile of `tile` of its rows: `at` is the first one's place among the sequence's rows, lo the
// sequence's first row.  Each row counts `mult` times (the query heads that share a key head are rows of
// one tile).
struct Tile {
  int part;
  int64_t lo, len, at;  // len: the sequence's rows, times mult; at < len where there is a tile
};

// Tile number `slot` of start(p) = bound(p) mult / tile + p on: a sequence has at least as many slots
// as tiles, and no table of tiles is needed.  All lanes of a wave look 64 ways at a time.
__device__ __forceinline__ Tile find_tile(const Seqs& s, int mult, int tile, int64_t slot) {
  int lo = 0, size = s.parts;
  const int lane = int(threadIdx.x) & 63;
  while (size > 1) {
    const int step = (size + 63) >> 6, at = lane * step;
    const bool before = at < size && s.bound(lo + at) * mult / tile + lo + at <= slot;
    const int n = __popcll(__ballot(before));
    const int skip = n > 1 ? (n - 1) * step : 0;
    lo += skip;
    size = size - skip < step ? size - skip : step;
  }
  Tile t;
  t.part = lo;
  t.lo = s.bound(lo);
  const int64_t hi = s.bound(lo + 1);
  t.len = hi > t.lo ? (hi - t.lo) * mult : 0;
  t.at = (slot - (t.lo * mult / tile + lo)) * tile;
  if (t.at < 0) t.at = t.len;
  return t;
}

inline int64_t tile_slots(const Seqs& s, int mult, int tile) {
  return s.rows * mult / tile + s.parts;
}

// The keys of the queries of part p.
__device__ __forceinline__ int keys_of(const Seqs& q, const Seqs& k, int p, int64_t klo) {
  const int64_t n = q.outside(p) ? 0 : k.bound(p + 1) - klo;
  return n > 0 ? int(n) : 0;
}

// How many of Lk keys the i-th of Lq queries sees, causal: the last one sees all.
__device__ __forceinline__ int keys_seen(int64_t i, int Lq, int Lk) {
  const int64_t n = i + 1 + Lk - Lq;
  return n < 0 ? 0 : n < Lk ? int(n) : Lk;
}

// Rows of a head: row r, head h at p + r * row + h * head.
template <typename T>
struct Heads {
  T* p;
  int64_t row, head;
};

// ---- tiles in LDS ----------------------------------------------------------------
// ROWS rows of DP values (the head's, then zeros) in 16-byte pieces, permuted within a row so that neither
// whole pieces of 32 rows nor transposed reads meet on a bank.  Rows lie in their own order.
template <typename T, int DP, int ROWS>
struct HeadTile {
  using frag = typename Mfma<T>::frag;
  static constexpr int V = Mfma<T>::V, KSTEP = Mfma<T>::KSTEP;
  static constexpr int PIECES = DP / V, BYTES = ROWS * PIECES * 16;
  static constexpr int N = ROWS * PIECES / kAttnThreads;  // pieces of a thread
  static_assert(ROWS * PIECES % kAttnThreads == 0, "whole rounds");

  // The operand row that MFMA row m of a 32-row block takes: then the accumulator's register i of lane half
  // h is row 2 V (i / V) + V h + i % V, which is the order of the next product's operand.
  __device__ __forceinline__ static int row_of(int m) { return sizeof(T) == 2 ? unit_of(m) : m; }

  // rows r0 .. r0 + 31, values k .. k + KSTEP - 1 (step k of the reduction)
  __device__ __forceinline__ static frag read(const char* lds, int r0, int step) {
    const int lane = int(threadIdx.x) & 63, r = r0 + row_of(lane & 31);
    return *reinterpret_cast<const frag*>(
        lds + (r * PIECES + swizzled<PIECES>(r, 2 * step + (lane >> 5))) * 16);
  }
  // transposed: values c0 .. c0 + 31 (permuted as row_of) of rows r0 .. r0 + KSTEP - 1, which are
  // the reduction
  __device__ __forceinline__ static frag read_t(const char* lds, int r0, int c0) {
    const int lane = int(threadIdx.x) & 63, half = lane >> 5;
    if constexpr (sizeof(T) == 4) {
      frag f;
      const int c = c0 + (lane & 31);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int r = r0 + half * V + i;
        f[i] = *reinterpret_cast<const T*>(
            lds + (r * PIECES + swizzled<PIECES>(r, c / V)) * 16 + c % V * 4);
      }
      return f;
    } else {
      typedef short short4 __attribute__((ext_vector_type(4)));
      const int t = lane & 15;
      const int c = c0 + (lane & 16) + ((t & 1) << 3) + ((t & 2) << 1);
      union {
        short4 q[2];
        frag f;
      } u;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int r = r0 + 8 * half + 4 * j + (t >> 2);
        u.q[j] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) short4*)(lds + (r * PIECES +
                swizzled<PIECES>(r, c >> 3)) * 16 + (c & 7) * 2));
      }
      return u.f;
    }
  }
};

// The row (reduction index of the next product) of an accumulator's register i.
template <typename T>
__device__ __forceinline__ int acc_row(int i) {
  constexpr int V = Mfma<T>::V;
  return i / V * 2 * V + V * ((int(threadIdx.x) >> 5) & 1) + i % V;
}

// A pointer that is the same on all lanes, in scalar registers.
__device__ __forceinline__ const char* uniform(const char* p) {
  const uint64_t u = reinterpret_cast<uint64_t>(p);
  const uint32_t lo = __builtin_amdgcn_readfirstlane(uint32_t(u));
  const uint32_t hi = __builtin_amdgcn_readfirstlane(uint32_t(u >> 32));
  return reinterpret_cast<const char*>(uint64_t(hi) << 32 | lo);
}

// Loads of a thread's pieces of tiles of a head's rows.  Whole tiles take an address of the workgroup's and
// an offset of the lane's for good.  A tile that passes the last row, or whose head is narrower than DP, goes by
// piece, with zeros past the ends (0 times what lies there could be NaN).  Every lane loads, at a selected address:
// behind a branch that some lanes take the compiler once saved registers before the others were back.
template <typename T, int DP, int ROWS>
struct TileLoads {
  using L = HeadTile<T, DP, ROWS>;
  const T* p;  // the sequence's first row
  int64_t row;
  int len, D;
  unsigned off[L::N];  // of this thread's pieces, in bytes (rows of less than 2^23 values)

  __device__ __forceinline__ TileLoads(const T* p_, int64_t row_, int len_, int D_)
      : p(p_), row(row_), len(len_), D(D_) {
#pragma unroll
    for (int j = 0; j < L::N; ++j) off[j] = unsigned(at_row(j) * int(row) + at_value(j)) * unsigned(sizeof(T));
  }
  __device__ __forceinline__ static int at_row(int j) {
    return (j * kAttnThreads + int(threadIdx.x)) / L::PIECES;
  }
  __device__ __forceinline__ static int at_value(int j) {
    const int m = at_row(j);
    return swizzled<L::PIECES>(m, j * kAttnThreads + int(threadIdx.x) - m * L::PIECES) * L::V;
  }
  __device__ __forceinline__ void start(int at, char* lds) const {
    const char* base = uniform(reinterpret_cast<const char*>(p + at * row));
    if (DP == D && at + ROWS <= len) {
#pragma unroll
      for (int j = 0; j < L::N; ++j)
        copy_piece(base + off[j], lds + (j * kAttnThreads + wave_of() * 64) * 16);
      return;
    }
#pragma unroll
    for (int j = 0; j < L::N; ++j) {
      const bool in = (at_value(j) < D) & (at + at_row(j) < len);
      copy_piece(in ? static_cast<const void*>(base + off[j]) : &g_zero_piece,
                 lds + (j * kAttnThreads + wave_of() * 64) * 16);
    }
  }
};

// A row's operands for the whole head (zeros past D).
template <typename T, int DP>
__device__ __forceinline__ void load_head(const T* p, bool live, int D,
                                          typename Mfma<T>::frag (&f)[DP / Mfma<T>::KSTEP]) {
  using frag = typename Mfma<T>::frag;
  constexpr int V = Mfma<T>::V;
  const int half = (int(threadIdx.x) >> 5) & 1;
#pragma unroll
  for (int s = 0; s < DP / Mfma<T>::KSTEP; ++s) {
    const int c = (2 * s + half) * V;
    f[s] = frag{};
    if (live && c < D) f[s] = *reinterpret_cast<const frag*>(p + c);
  }
}

template <typename T>
struct Both {
  typename Mfma<T>::frag a, b;
};

__device__ __forceinline__ void zero(floatx16& a) {
#pragma unroll
  for (int i = 0; i < 16; ++i) a[i] = 0.f;
}

// Both halves' values of a row on each of them, joined by f.
template <typename F>
__device__ __forceinline__ float join_halves(float v, F&& f) {
  const auto r =
      __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return f(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float half_sum(float v) {
  return join_halves(v, [](float a, float b) { return a + b; });
}
__device__ __forceinline__ float half_max(float v) {
  return join_halves(v, [](float a, float b) { return __builtin_fmaxf(a, b); });
}

// N products whose operands come from LDS, AHEAD of them on their way: use(i, operand) issues the product and
// some vector instructions that run beside it.  The order is the one written here (the compiler's
// puts the products first, and then the matrix cores wait for the vector unit and the other way round).
template <typename F, int N, int AHEAD, typename Read, typename Use>
__device__ __forceinline__ void beside(Read&& read, Use&& use) {
  F f[AHEAD];
#pragma unroll
  for (int i = 0; i < AHEAD && i < N; ++i) f[i] = read(i);
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    use(i, f[i % AHEAD]);
    if (i + AHEAD < N) f[i % AHEAD] = read(i + AHEAD);
    __builtin_amdgcn_sched_barrier(0);
  }
}

// acc[t] += (values 32 t .. of rows r0 .. r0 + 31)' p: the second product of attention and of its gradients.
template <typename T, int DP, int ROWS, int B>
__device__ __forceinline__ void add_rows(const char* lds, int r0,
                                         const typename Mfma<T>::frag (&p)[32 / Mfma<T>::KSTEP],
                                         floatx16 (&acc)[DP / 32]) {
  using L = HeadTile<T, DP, ROWS>;
  constexpr int TILES = DP / 32, STEPS = 32 / Mfma<T>::KSTEP;
  // (neighbouring products go to different accumulators)
  auto read = [&](int i) {
    return L::read_t(lds, r0 + i / TILES * Mfma<T>::KSTEP, i % TILES * 32);
  };
  Batched<typename Mfma<T>::frag, TILES * STEPS, B> f;
  f.start(read);
  f.run(read, [&](int i, const typename Mfma<T>::frag& a) {
    Mfma<T>::mma(a, p[i / TILES], acc[i % TILES]);
  });
}

// The same where a lane sees the rows lo .. hi - 1 only and the others may hold infinities or NaN, which times
// the zeros of p would be NaN: one row at a time on the vector unit, added where it is seen.  Slow (32 rows of 128
// values are 4096 multiplications a lane for 32 matrix instructions), and run for tiles whose results came out not
// finite only; what counts is that it needs few registers, so one accumulator at a time goes through the rows.
template <typename T, int DP, int ROWS>
__device__ __forceinline__ void add_rows_seen(const char* lds, int r0, int lo, int hi,
                                              const typename Mfma<T>::frag (&p)[32 / Mfma<T>::KSTEP],
                                              floatx16 (&acc)[DP / 32]) {
  using L = HeadTile<T, DP, ROWS>;
  using frag = typename Mfma<T>::frag;
  constexpr int V = Mfma<T>::V, STEPS = 32 / Mfma<T>::KSTEP;
  const int half = (int(threadIdx.x) >> 5) & 1;
#pragma unroll
  for (int t = 0; t < DP / 32; ++t) {
#pragma unroll 1
    for (int k = 0; k < 16; ++k) {
      // weight k of either half is of row 2 V (k / V) + V half + k % V (acc_row); here both halves get both
      float mine = 0.f;
#pragma unroll
      for (int s = 0; s < STEPS; ++s)
#pragma unroll
        for (int i = 0; i < V; ++i) mine = s * V + i == k ? to_f32(p[s][i]) : mine;
      const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(mine),
                                                         __float_as_uint(mine), false, false);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float w = __uint_as_float(both[h]);
        const int r = r0 + k / V * 2 * V + V * h + k % V;
        const bool seen = r >= lo && r < hi;
#pragma unroll
        for (int b = 0; b < 16 / V; ++b) {
          const frag f = *reinterpret_cast<const frag*>(
              lds + (r * L::PIECES + swizzled<L::PIECES>(r, 32 / V * t + 2 * b + half)) * 16);
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const float v = to_f32(f[i]) * w;
            acc[t][V * b + i] += seen ? v : 0.f;
          }
        }
      }
    }
  }
}

// Whether any lane of the wave holds a value that is not finite.
template <int N>
__device__ __forceinline__ bool any_not_finite(const floatx16 (&acc)[N]) {
  bool bad = false;
#pragma unroll
  for (int t = 0; t < N; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i)
      bad |= !(__builtin_fabsf(acc[t][i]) < __builtin_inff());
  return __ballot(bad) != 0;
}

// The lane's row of results, value(t, i) for register i of tile t.
template <typename T, int DP, typename F>
__device__ __forceinline__ void store_head(T* p, int D, F&& value) {
  using frag = typename Mfma<T>::frag;
  constexpr int V = Mfma<T>::V;
  const int half = (int(threadIdx.x) >> 5) & 1;
#pragma unroll
  for (int t = 0; t < DP / 32; ++t)
#pragma unroll
    for (int b = 0; b < 16 / V; ++b) {
      const int c = 32 * t + 2 * V * b + V * half;
      if (c >= D) continue;
      frag f;
#pragma unroll
      for (int i = 0; i < V; ++i) f[i] = from_f32<T>(value(t, V * b + i));
      *reinterpret_cast<frag*>(p + c) = f;
    }
}

// fp32 partials of a share, D values a row.
template <int DP, int V, typename F>
__device__ __forceinline__ void store_part(float* p, int D, F&& value) {
  const int half = (int(threadIdx.x) >> 5) & 1;
#pragma unroll
  for (int t = 0; t < DP / 32; ++t)
#pragma unroll
    for (int b = 0; b < 16 / V; ++b) {
      const int c = 32 * t + 2 * V * b + V * half;
      if (c >= D) continue;
#pragma unroll
      for (int i = 0; i < V; i += 4)
        *reinterpret_cast<float4v*>(p + c + i) =
            float4v{value(t, V * b + i), value(t, V * b + i + 1), value(t, V * b + i + 2),
                    value(t, V * b + i + 3)};
    }
}

template <typename T>
struct AttnArgs {
  Heads<const T> q, k, v, o, dout;  // o: the forward pass's result, in the backward pass
  Heads<T> out, dq, dk, dv;
  Seqs qs, ks;
  int H, Hk, G, D, causal;
  float scale, scale2;  // of the scores, and times log2(e)
  float* lse;           // [H][rows of q], base 2; +inf for a row without keys
  const float* top;     // partial maxima of the rows' norms (fp16 gradients)
  int tops;
  int shares;
  float *part, *part_ml;
  int* again;  // causal: one a workgroup, whether its results are not finite
};

// Causal tiles run in two launches.  Where a query does not see a key, the product's operand is zero, but the
// key's value may be an infinity or NaN, and a result that is not finite may come from there. The first
// launch says which workgroups have such results, the second (STRICT) makes those again and adds
// only what is seen; it costs the time of a launch.
template <bool CAUSAL, bool STRICT>
__device__ __forceinline__ bool skips(const int* again) {
  return STRICT && !again[blockIdx.x];
}
template <bool CAUSAL, bool STRICT>
__device__ __forceinline__ void report(int* again, bool bad, int* lds) {
  if (!CAUSAL || STRICT) return;
  if (threadIdx.x == 0) *lds = 0;
  __syncthreads();
  if (bad) *lds = 1;
  __syncthreads();
  if (threadIdx.x == 0) again[blockIdx.x] = *lds;
}

// The workgroup's tile: slot, key head and share of the other axis.
struct Place {
  int64_t slot;
  int head, share;
};
// (an XCD's workgroups are an eighth of the places in a row: the tiles of a key head, or of a share of its keys,
// are neighbours and meet in its L2)
__device__ __forceinline__ bool find_place(int64_t slots, int heads, int shares, int64_t id,
                                           Place& p) {
  const int64_t total = slots * heads * shares, per = (total + 7) >> 3;
  const int64_t k = (id >> 3) < per ? (id & 7) * per + (id >> 3) : total;
  if (k >= total) return false;
  const int64_t a = k / slots;
  p.slot = k - a * slots;
  p.share = int(a / heads);
  p.head = int(a - int64_t(p.share) * heads);
  return true;
}

// ---- host ------------------------------------------------------------------------
constexpr int kAttnMaxDim = 128;
// (the kernels' 32-bit places go up to a whole tile past the last row)
constexpr int64_t kAttnMaxRows = (int64_t(1) << 31) - 128;
constexpr int kMostShares = 1024;

// Rows of a tile that passes through LDS.
template <typename T>
constexpr int attn_stage() { return sizeof(T) == 4 ? 32 : 64; }

// How many shares the other axis, of `len` rows on average, is cut into: where `tiles` tiles leave some of the
// `groups` workgroups that are resident at a time without work, as many as make one round of them (800
// rows of 4 heads of 64 over 2 x 30k keys: 864 workgroups for 768 places took 54 us, 768 of them, a share's tiles on
// one XCD, 38); where the tiles are one round and a part of another, two (12k keys of 4 heads of 128, causal, whole training
// step 1 113 us with one and 1 058 with two).  A share keeps 256 rows.
inline int attn_shares(int64_t tiles, int64_t len, int groups) {
  if (tiles < 1) tiles = 1;
  const int64_t want = tiles > groups && tiles < 2 * groups ? 2 : groups / tiles, most = len / 256;
  const int64_t n = want < most ? want : most;
  return n < 1 ? 1 : n < kMostShares ? int(n) : kMostShares;
}

inline int64_t attn_sequences(const Seqs& s) { return s.off && s.parts > 2 ? s.parts - 2 : 1; }

inline int64_t attn_tiles(const Seqs& s, int mult, int heads, int tile) {
  const int64_t n = attn_sequences(s);
  return cdiv(cdiv(s.rows, n) * mult, tile) * n * heads;
}

inline int64_t attn_length(const Seqs& s) { return s.rows / attn_sequences(s); }

// f(padded head width as a constant)
template <typename F>
int with_width(int D, F&& f) {
  if (D <= 32) return f(std::integral_constant<int, 32>());
  if (D <= 64) return f(std::integral_constant<int, 64>());
  if (D <= 96) return f(std::integral_constant<int, 96>());
  return f(std::integral_constant<int, 128>());
}

// The workgroups of a launch: whole eights (find_place).
inline int64_t attn_groups(int64_t slots, int heads, int shares) {
  return cdiv(slots * heads * shares, 8) * 8;
}

constexpr int64_t kAttnMaxGroups = max_groups(kAttnThreads);

struct AttnGradLayout {
  size_t nl, nd, tops, part, again, total;
  int dq_shares, dkv_shares;
};
AttnGradLayout attn_grad_layout(const Seqs& q, const Seqs& k, int H, int Hk, int D,
                                bool causal, int32_t dtype);
template <typename T>
int attn_backward(AttnArgs<T> a, const AttnGradLayout& l, char* ws, bool need_dq, bool need_dkv,
                  hipStream_t s);

}  // namespace sp
