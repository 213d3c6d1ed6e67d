// Gradients of softmax attention (sp_attention.hip) from that of its result, dO:
//
//   P = 2^(c S - lse), delta = sum(dO * O) over a head's values
//   dV = P' dO, dP = dO V', dS = P * (dP - delta), dQ = scale dS K, dK = scale dS' Q
//
// S and P are formed again from q, k and the forward pass's lse, in two kernels: one with a tile of
// queries a workgroup, which goes through the keys for dQ (S, dP, dQ), and one with a tile of keys, which
// goes through the queries for dK and dV (S, dP, dV, dK).  That is seven products for the five that one
// kernel would need, but no sums by atomics: two calls give the same gradients.
//
// P and dS are rounded to the rows' type as operands of the products that follow.  In fp16, P of a long
// row (1 / its keys) and dS would lie below the normal range: P goes in times 2^15 (it is at most 1), and dS times the
// power of two that the bound |dS| <= 2 |dO| max|v| (lengths of rows) leaves: for dQ from the
// query's own |dO|, for dK, whose sums are over queries, from the largest.
//
// Bound by the matrix cores and the vector unit in turn, as the forward pass is: self-attention of 8 heads of 64 bf16
// values, dQ 1 038 us (9.9e11 operations, 958 TFLOP/s), dK and dV 1 480 (1.33e12, 896); causal, 128 fp16 values, 427 and
// 508; 5 003 rows of 4 heads of 32 fp32 values 100 and 130 (77 and 79 TFLOP/s, where a product of 8192^3 reaches 154).
#include "sp_attention.h"

namespace sp {

constexpr int kGradLoads = 4;  // rows of a group of lanes at a time in attend_grad_rows
constexpr int kTops = 512;  // workgroups of attend_grad_rows at most

constexpr int kAhead = 3;  // operands on their way from LDS
constexpr int kStats = 64;  // places of a tile's statistics, of each kind

// Whether 32 rows' products are written beside the weights of the 32 rows before, with two tiles' scores in
// registers.  That pays where a SIMD has one wave in any case (128 values a head, causal, fp16: dQ 451 us
// and 415 so, dK and dV 563 and 442) and for dK and dV of 64 values (bf16, 1 520 and 1 470); elsewhere more waves are
// worth more (dQ of 64 values 1 032 and 1 130; of 32 values 460 and 475, dK and dV 581 and 670).
template <typename T>
constexpr bool dq_beside(int DP) { return DP > 64 || sizeof(T) == 4; }
template <typename T>
constexpr bool dkv_beside(int DP) { return DP >= 64 || sizeof(T) == 4; }

// Waves a SIMD (of a launch that makes results again: as few as leave it all registers).
template <typename T>
constexpr int dq_waves(int DP, bool strict = false) {
  if (strict) return 1;
  return sizeof(T) == 4 ? (DP <= 32 ? 4 : DP <= 64 ? 2 : 1) : DP <= 32 ? 4 : DP <= 64 ? 3 : 1;
}
template <typename T>
constexpr int grad_waves(int DP, bool strict = false) {
  if (strict) return 1;
  return sizeof(T) == 4 ? (DP <= 32 ? 3 : 1) : DP <= 32 ? 4 : DP <= 64 ? 2 : 1;
}

template <typename T>
constexpr float kLift = sizeof(T) == 2 && std::is_same<T, _Float16>::value ? 15.f : 0.f;

__device__ const float g_no_row[2] = {-__builtin_inff(), 0.f};  // of a row past the end: P = 0

// What both kernels need of each query and head: nl = lift - lse and nd = -delta, [H][rows].  In fp16 also
// the largest squares of |dO| and |v| over the rows of the sequences, one pair a workgroup (those that
// are not finite do not count: their rows' gradients are not finite either).
template <typename T>
__global__ __launch_bounds__(kAttnThreads) void attend_grad_rows(AttnArgs<T> a, int log_lanes,
                                                                 float* __restrict__ nl,
                                                                 float* __restrict__ nd,
                                                                 float* __restrict__ tops) {
  constexpr int V = Mfma<T>::V;
  using frag = typename Mfma<T>::frag;
  const int lanes = 1 << log_lanes, lane = int(threadIdx.x) & (lanes - 1);
  const int per = kAttnThreads >> log_lanes;
  const int64_t stride = int64_t(gridDim.x) * per;
  const int64_t start = int64_t(blockIdx.x) * per + (int(threadIdx.x) >> log_lanes);
  float top[2] = {0.f, 0.f};
  auto sum = [&](float v) {
    for (int off = lanes >> 1; off >= 1; off >>= 1) v += __shfl_xor(v, off, 64);
    return v;
  };
  // (kGradLoads rows' loads start before the first one's sum; the bounds are the workgroup's)
  const int64_t n = a.qs.rows * a.H;
  const int c = lane * V;
  for (int64_t b = start - (int(threadIdx.x) >> log_lanes); b < n; b += stride * kGradLoads) {
    frag x[kGradLoads], y[kGradLoads];
#pragma unroll
    for (int j = 0; j < kGradLoads; ++j) {
      const int64_t at = b + j * stride + (int(threadIdx.x) >> log_lanes), r = at / a.H;
      const int h = int(at - r * a.H);
      x[j] = y[j] = frag{};
      if (at < n && c < a.D) {
        x[j] = *reinterpret_cast<const frag*>(a.dout.p + r * a.dout.row + h * a.dout.head + c);
        y[j] = *reinterpret_cast<const frag*>(a.o.p + r * a.o.row + h * a.o.head + c);
      }
    }
#pragma unroll
    for (int j = 0; j < kGradLoads; ++j) {
      const int64_t at = b + j * stride + (int(threadIdx.x) >> log_lanes), r = at / a.H;
      const int h = int(at - r * a.H);
      float dot = 0.f, sq = 0.f;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        dot = __builtin_fmaf(to_f32(x[j][i]), to_f32(y[j][i]), dot);
        sq = __builtin_fmaf(to_f32(x[j][i]), to_f32(x[j][i]), sq);
      }
      dot = sum(dot);
      if (kLift<T> != 0.f) {
        sq = sum(sq);
        const bool in = !a.qs.off || (r >= a.qs.bound(1) && r < a.qs.bound(a.qs.parts - 1));
        if (at < n && in && sq < __builtin_inff()) top[0] = __builtin_fmaxf(top[0], sq);
      }
      if (at < n && lane == 0) {
        nl[h * a.qs.rows + r] = kLift<T> - a.lse[h * a.qs.rows + r];
        nd[h * a.qs.rows + r] = -dot;
      }
    }
  }
  if (kLift<T> == 0.f) return;
  const int64_t nv = a.ks.rows * a.Hk;
  for (int64_t b = start - (int(threadIdx.x) >> log_lanes); b < nv; b += stride * kGradLoads) {
    frag x[kGradLoads];
#pragma unroll
    for (int j = 0; j < kGradLoads; ++j) {
      const int64_t at = b + j * stride + (int(threadIdx.x) >> log_lanes), r = at / a.Hk;
      const int h = int(at - r * a.Hk);
      x[j] = frag{};
      if (at < nv && c < a.D)
        x[j] = *reinterpret_cast<const frag*>(a.v.p + r * a.v.row + h * a.v.head + c);
    }
#pragma unroll
    for (int j = 0; j < kGradLoads; ++j) {
      const int64_t at = b + j * stride + (int(threadIdx.x) >> log_lanes), r = at / a.Hk;
      float sq = 0.f;
#pragma unroll
      for (int i = 0; i < V; ++i) sq = __builtin_fmaf(to_f32(x[j][i]), to_f32(x[j][i]), sq);
      sq = sum(sq);
      const bool in = !a.ks.off || (r >= a.ks.bound(1) && r < a.ks.bound(a.ks.parts - 1));
      if (at < nv && in && sq < __builtin_inff()) top[1] = __builtin_fmaxf(top[1], sq);
    }
  }
  __shared__ float lds[2][kAttnWaves];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1)
      top[j] = __builtin_fmaxf(top[j], __shfl_xor(top[j], off, 64));
    if ((threadIdx.x & 63) == 0) lds[j][wave_of()] = top[j];
  }
  __syncthreads();
  if (threadIdx.x < 2) {
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < kAttnWaves; ++w) v = __builtin_fmaxf(v, lds[threadIdx.x][w]);
    tops[2 * blockIdx.x + threadIdx.x] = v;
  }
}

// The largest of the workgroups' pairs, on every lane of the wave.
__device__ __forceinline__ void read_tops(const float* tops, int n, float& grad, float& value) {
  grad = value = 0.f;
  for (int i = int(threadIdx.x) & 63; i < n; i += 64) {
    grad = __builtin_fmaxf(grad, tops[2 * i]);
    value = __builtin_fmaxf(value, tops[2 * i + 1]);
  }
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) {
    grad = __builtin_fmaxf(grad, __shfl_xor(grad, off, 64));
    value = __builtin_fmaxf(value, __shfl_xor(value, off, 64));
  }
}

// The exponent e with 2 |dO| |v| 2^e <= 2^15, from the squares of the lengths.
__device__ __forceinline__ float lift_of(float grad_sq, float value_sq) {
  const float e = __builtin_floorf(
      14.f - 0.5f * (__builtin_amdgcn_logf(grad_sq) + __builtin_amdgcn_logf(value_sq)));
  return e > -100.f ? (e < 100.f ? e : 100.f) : 0.f;  // (a length of 0 makes e infinite)
}

template <typename T, int DP, int BK, bool CAUSAL, bool STRICT>
__global__ __launch_bounds__(kAttnThreads, dq_waves<T>(DP, STRICT)) void attend_dq(
    AttnArgs<T> a, const float* __restrict__ nl, const float* __restrict__ nd, int64_t slots) {
  using frag = typename Mfma<T>::frag;
  using L = HeadTile<T, DP, BK>;
  constexpr int STEPS = DP / Mfma<T>::KSTEP, PS = 32 / Mfma<T>::KSTEP, V = Mfma<T>::V;
  constexpr int BQ = kAttnWaves * 32, TILES = DP / 32, NX = BK / 32;
  static_assert(NX <= 2, "a step holds one tile's weights while the next one's are formed");
  __shared__ __attribute__((aligned(16))) char lds[4 * L::BYTES];
  __shared__ int bad_lds;
  Place place;
  if (!find_place(slots, a.Hk, a.shares, blockIdx.x, place)) return;
  if (skips<CAUSAL, STRICT>(a.again)) return;
  if (CAUSAL) place.slot = slots - 1 - place.slot;
  const Tile t = find_tile(a.qs, a.G, BQ, place.slot);
  if (t.at >= t.len) {
    if (CAUSAL && !STRICT && threadIdx.x == 0) a.again[blockIdx.x] = 0;
    return;
  }
  const int64_t klo = a.ks.bound(t.part);
  const int Lk = keys_of(a.qs, a.ks, t.part, klo), Lq = int(t.len / a.G);
  const int wave = wave_of(), lane = int(threadIdx.x) & 31;
  float top_grad = 0.f, top_value = 0.f;
  if (kLift<T> != 0.f) read_tops(a.top, a.tops, top_grad, top_value);

  // this lane's query
  const int64_t r = t.at + wave * 32 + lane;
  const bool live = r < t.len;
  const int row = int(r / a.G), head = place.head * a.G + int(r - int64_t(row) * a.G);
  const int seen = a.causal ? keys_seen(row, Lq, Lk) : Lk;
  const int64_t at = t.lo + row;
  frag q[STEPS], g[STEPS];
  load_head<T, DP>(a.q.p + at * a.q.row + head * a.q.head, live, a.D, q);
  load_head<T, DP>(a.dout.p + at * a.dout.row + head * a.dout.head, live, a.D, g);
  float base = live ? nl[head * a.qs.rows + at] : -__builtin_inff();
  const float minus = live ? nd[head * a.qs.rows + at] : 0.f;
  float lift = 0.f;
  if (kLift<T> != 0.f) {
    float sq = 0.f;
#pragma unroll
    for (int s = 0; s < STEPS; ++s)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float v = to_f32(g[s][j]);
        sq = __builtin_fmaf(v, v, sq);
      }
    lift = lift_of(half_sum(sq), top_value);
    base += lift - kLift<T>;
  }
  int most = Lk, wave_most = Lk, wave_least = Lk;
  if (a.causal) {
    const int64_t last = t.at + BQ < t.len ? t.at + BQ : t.len, w = t.at + wave * 32;
    most = keys_seen((last - 1) / a.G, Lq, Lk);
    wave_least = keys_seen(w / a.G, Lq, Lk);
    wave_most = keys_seen((w + 31) / a.G, Lq, Lk);
    wave_most = wave_most < most ? wave_most : most;
  }
  const int tiles = (most + BK - 1) / BK, per = (tiles + a.shares - 1) / a.shares;
  const int first = place.share * per, end = first + per < tiles ? first + per : tiles;
  const TileLoads<T, DP, BK> lk(a.k.p + klo * a.k.row + place.head * a.k.head, a.k.row, Lk, a.D);
  const TileLoads<T, DP, BK> lv(a.v.p + klo * a.v.row + place.head * a.v.head, a.v.row, Lk, a.D);
  const float c = a.scale2;
  floatx16 acc[TILES];
#pragma unroll
  for (int d = 0; d < TILES; ++d) zero(acc[d]);
  // A tile of keys in buffer B, in the order of attend_dkv's step.
  auto step = [&](int n, auto buffer) {
    char* buf = lds + buffer.value * 2 * L::BYTES;
    loads_in_flight<0>();
    __syncthreads();
    if (n + 1 < end) {
      char* next = lds + (1 - buffer.value) * 2 * L::BYTES;
      lk.start((n + 1) * BK, next);
      lv.start((n + 1) * BK, next + L::BYTES);
    }
    const int key0 = n * BK;
    if (key0 >= wave_most) return;
    const bool edge = key0 + BK > wave_least;
    floatx16 s[NX], dp[NX];
    frag ds[NX][PS];
    auto read = [&](int x) {
      return [=](int i) { return L::read(buf + (i & 1) * L::BYTES, 32 * x, i >> 1); };
    };
    auto form = [&](int x, int i, const frag& f) {
      if (i & 1)
        Mfma<T>::mma(f, g[i >> 1], dp[x]);
      else
        Mfma<T>::mma(f, q[i >> 1], s[x]);
    };
    auto prepare = [&](int x) {
      if (!edge) return;
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (key0 + 32 * x + acc_row<T>(i) >= seen) {
          s[x][i] = -__builtin_inff();
          dp[x][i] = 0.f;  // (not what a NaN there makes of it)
        }
    };
    auto weigh = [&](int x, int lo, int hi) {
#pragma unroll
      for (int i = lo; i < hi; ++i) {
        const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[x][i], c, base));
        ds[x][i / V][i % V] = T(p * (dp[x][i] + minus));
      }
    };
    auto read_t = [&](int x) {
      return [=](int i) {
        return L::read_t(buf, 32 * x + i / TILES * Mfma<T>::KSTEP, 32 * (i % TILES));
      };
    };
    auto add = [&](int x, int i, const frag& f) {
      Mfma<T>::mma(f, ds[x][i / TILES], acc[i % TILES]);
    };
    constexpr int FORM = 2 * STEPS, ADD = PS * TILES;
    if constexpr (STRICT || !dq_beside<T>(DP)) {
#pragma unroll
      for (int x = 0; x < NX; ++x) {
        zero(s[x]);
        zero(dp[x]);
        beside<frag, FORM, kAhead>(read(x), [&](int i, const frag& f) { form(x, i, f); });
        prepare(x);
        weigh(x, 0, 16);
        if (STRICT && edge)
          add_rows_seen<T, DP, BK>(buf, 32 * x, 0, seen - key0, ds[x], acc);
        else
          beside<frag, ADD, kAhead>(read_t(x), [&](int i, const frag& f) { add(x, i, f); });
      }
      return;
    }
#pragma unroll
    for (int x = 0; x < NX; ++x) {
      zero(s[x]);
      zero(dp[x]);
    }
    beside<frag, FORM, kAhead>(read(0), [&](int i, const frag& f) { form(0, i, f); });
#pragma unroll
    for (int x = 0; x < NX; ++x) {
      prepare(x);
      if (x + 1 < NX) {
        beside<frag, FORM, kAhead>(read(x + 1), [&](int i, const frag& f) {
          form(x + 1, i, f);
          weigh(x, 16 * i / FORM, 16 * (i + 1) / FORM);
        });
      } else if (x > 0) {
        beside<frag, ADD, kAhead>(read_t(x - 1), [&](int i, const frag& f) {
          add(x - 1, i, f);
          weigh(x, 16 * i / ADD, 16 * (i + 1) / ADD);
        });
      } else {
        weigh(x, 0, 16);
      }
    }
    beside<frag, ADD, kAhead>(read_t(NX - 1), [&](int i, const frag& f) { add(NX - 1, i, f); });
  };
  if (first < end) {
    lk.start(first * BK, lds);
    lv.start(first * BK, lds + L::BYTES);
  }
  for (int n = first; n < end; n += 2) {
    step(n, std::integral_constant<int, 0>());
    if (n + 1 < end) step(n + 1, std::integral_constant<int, 1>());
  }
  bool bad = false;
  if (CAUSAL && !STRICT) bad = any_not_finite(acc);
  report<CAUSAL, STRICT>(a.again, bad, &bad_lds);
  if (!live) return;
  const float f = a.scale * __builtin_amdgcn_exp2f(-lift);
  if (a.shares > 1) {
    const int64_t i = (place.share * a.qs.rows + at) * a.H + head;
    store_part<DP, V>(a.part + i * a.D, a.D, [&](int d, int j) { return acc[d][j] * f; });
  } else {
    store_head<T, DP>(a.dq.p + at * a.dq.row + head * a.dq.head, a.D,
                      [&](int d, int j) { return acc[d][j] * f; });
  }
}

// A tile of keys goes through the queries of its head's G query heads, one head after the other.
template <typename T, int DP, int BQ, bool CAUSAL, bool STRICT>
__global__ __launch_bounds__(kAttnThreads, grad_waves<T>(DP, STRICT)) void attend_dkv(
    AttnArgs<T> a, const float* __restrict__ nl, const float* __restrict__ nd, int64_t slots) {
  using frag = typename Mfma<T>::frag;
  using L = HeadTile<T, DP, BQ>;
  constexpr int STEPS = DP / Mfma<T>::KSTEP, PS = 32 / Mfma<T>::KSTEP, V = Mfma<T>::V;
  constexpr int TILES = DP / 32, NX = BQ / 32;
  static_assert(NX <= 2, "a step holds one tile's weights while the next one's are formed");
  constexpr int BK = kAttnWaves * 32, STAGE = 2 * L::BYTES + 2 * kStats * 4;
  static_assert(BQ <= kStats, "a wave loads a tile's statistics at once");
  __shared__ __attribute__((aligned(16))) char lds[2 * STAGE];
  __shared__ int bad_lds;
  Place place;
  if (!find_place(slots, a.Hk, a.shares, blockIdx.x, place)) return;
  if (skips<CAUSAL, STRICT>(a.again)) return;
  const Tile t = find_tile(a.ks, 1, BK, place.slot);
  if (t.at >= t.len) {
    if (CAUSAL && !STRICT && threadIdx.x == 0) a.again[blockIdx.x] = 0;
    return;
  }
  const int64_t qlo = a.qs.bound(t.part);
  const int Lk = int(t.len), Lq = keys_of(a.ks, a.qs, t.part, qlo);
  const int wave = wave_of(), lane = int(threadIdx.x) & 31, lane64 = int(threadIdx.x) & 63;
  float g = 1.f, lift = 0.f;
  if (kLift<T> != 0.f) {
    float top_grad, top_value;
    read_tops(a.top, a.tops, top_grad, top_value);
    lift = lift_of(top_grad, top_value);
    g = __builtin_amdgcn_exp2f(lift - kLift<T>);
  }

  // this lane's key: its place in its sequence, its first query
  const int at = int(t.at) + wave * 32 + lane;
  const bool live = at < Lk;
  const int from = a.causal && at > Lk - Lq ? at - Lk + Lq : 0;
  frag k[STEPS], v[STEPS];
  load_head<T, DP>(a.k.p + (t.lo + at) * a.k.row + place.head * a.k.head, live, a.D, k);
  load_head<T, DP>(a.v.p + (t.lo + at) * a.v.row + place.head * a.v.head, live, a.D, v);
  // first queries: of the workgroup's keys, of the wave's, of its last key
  int least = 0, wave_least = 0, wave_most = 0;
  if (a.causal) {
    const int shift = Lq - Lk, j = int(t.at) + wave * 32;
    least = t.at + shift > 0 ? int(t.at) + shift : 0;
    wave_least = j + shift > 0 ? j + shift : 0;
    wave_most = j + 31 + shift > 0 ? j + 31 + shift : 0;
  }
  const int begin = least / BQ, last = (Lq + BQ - 1) / BQ;  // tiles of a head
  const int64_t tiles = last > begin ? int64_t(last - begin) * a.G : 0;
  const int64_t per = (tiles + a.shares - 1) / a.shares, first = place.share * per;
  const int64_t end = first + per < tiles ? first + per : tiles;
  const int64_t h0 = int64_t(place.head) * a.G;
  TileLoads<T, DP, BQ> lq(a.q.p + qlo * a.q.row, a.q.row, Lq, a.D);
  TileLoads<T, DP, BQ> lg(a.dout.p + qlo * a.dout.row, a.dout.row, Lq, a.D);
  const T *q0 = lq.p, *g0 = lg.p;
  auto start = [&](int head, int tile, char* to) {
    lq.p = q0 + (h0 + head) * a.q.head;
    lg.p = g0 + (h0 + head) * a.dout.head;
    lq.start(tile * BQ, to);
    lg.start(tile * BQ, to + L::BYTES);
    if (wave < 2) {
      // (a whole wave, each lane by a selected address: a branch of some lanes here had the compiler save registers
      // for those lanes only)
      // (the lane's part of the address is of this tile: a row's own times 4 would pass 32 bits)
      const int first_row = tile * BQ;
      const char* rows = uniform(reinterpret_cast<const char*>(
          (wave ? nd : nl) + (h0 + head) * a.qs.rows + qlo + first_row));
      const char* from_ = first_row + lane64 < Lq ? rows + unsigned(lane64) * 4
                                                  : reinterpret_cast<const char*>(&g_no_row[wave]);
      __builtin_amdgcn_global_load_lds(
          (const __attribute__((address_space(1))) void*)from_,
          (__attribute__((address_space(3))) void*)(to + 2 * L::BYTES + wave * (kStats * 4)), 4, 0,
          0);
    }
  };
  const float c = a.scale2;
  // A pass over the queries, for dk, dv or both.
  auto pass = [&](auto want_dk, auto want_dv) {
    constexpr bool DK = want_dk.value, DV = want_dv.value;
    floatx16 dk[DK ? TILES : 1], dv[DV ? TILES : 1];
#pragma unroll
    for (int d = 0; d < TILES; ++d) {
      if constexpr (DK) zero(dk[d]);
      if constexpr (DV) zero(dv[d]);
    }
    int64_t n = first;
    int qh = 0, qt = begin;  // the tile's head and place
    if (n < end) {
      qh = int(n / (last - begin));
      qt = begin + int(n - int64_t(qh) * (last - begin));
    }
    // A tile of queries in buffer B.  32 queries' scores and their gradients are formed beside the weights of the
    // 32 before, and these are multiplied beside the weights of the next.
    auto step = [&](auto buffer) {
      char* buf = lds + buffer.value * STAGE;
      loads_in_flight<0>();
      __syncthreads();
      const int query0 = qt * BQ;
      if (++qt == last) {
        qt = begin;
        ++qh;
      }
      if (n + 1 < end) start(qh, qt, lds + (1 - buffer.value) * STAGE);
      // (asked in either case: without these branches the compiler's order of the step takes more registers than
      // there are, 176 bytes of scratch at 64 values a head and half the speed)
      if (query0 + BQ <= wave_least) return;
      const bool edge = query0 < wave_most;
      const float* stats = reinterpret_cast<const float*>(buf + 2 * L::BYTES);
      floatx16 s[NX], dp[NX];
      frag p[NX][PS], ds[NX][PS];
      float4v base[2], minus[2];  // of four weights, and of the next four
      auto read = [&](int x) {
        return [=](int i) { return L::read(buf + (i & 1) * L::BYTES, 32 * x, i >> 1); };
      };
      auto form = [&](int x, int i, const frag& f) {
        if (i & 1)
          Mfma<T>::mma(f, v[i >> 1], dp[x]);
        else
          Mfma<T>::mma(f, k[i >> 1], s[x]);
      };
      // the weights of 32 queries: what they take, what of them is hidden, and weights lo .. hi - 1
      auto take = [&](int x, int i) {
        const int r = 32 * x + acc_row<T>(4 * i);
        base[i & 1] = *reinterpret_cast<const float4v*>(stats + r);
        minus[i & 1] = *reinterpret_cast<const float4v*>(stats + kStats + r);
      };
      auto prepare = [&](int x) {
        take(x, 0);
        if (!edge) return;
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (query0 + 32 * x + acc_row<T>(i) < from) {
            s[x][i] = -__builtin_inff();
            dp[x][i] = 0.f;  // (not what a NaN there makes of it)
          }
      };
      auto weigh = [&](int x, int lo, int hi) {
#pragma unroll
        for (int i = lo; i < hi; ++i) {
          if ((i & 3) == 0 && i < 12) take(x, (i >> 2) + 1);
          const float e =
              __builtin_amdgcn_exp2f(__builtin_fmaf(s[x][i], c, base[i >> 2 & 1][i & 3]));
          float d = dp[x][i] + minus[i >> 2 & 1][i & 3];
          if (kLift<T> != 0.f) d *= g;
          p[x][i / V][i % V] = T(e);
          ds[x][i / V][i % V] = T(e * d);
        }
      };
      auto read_t = [&](int x) {
        return [=](int i) {
          return L::read_t(buf + (i & 1 ? 0 : L::BYTES),
                           32 * x + (i >> 1) / TILES * Mfma<T>::KSTEP, 32 * ((i >> 1) % TILES));
        };
      };
      auto add = [&](int x, int i, const frag& f) {
        const int d = (i >> 1) % TILES, w = (i >> 1) / TILES;
        if (i & 1) {
          if constexpr (DK) Mfma<T>::mma(f, ds[x][w], dk[d]);
        } else {
          if constexpr (DV) Mfma<T>::mma(f, p[x][w], dv[d]);
        }
      };
      constexpr int FORM = 2 * STEPS, ADD = 2 * PS * TILES;
      if constexpr (STRICT || !dkv_beside<T>(DP)) {
#pragma unroll
        for (int x = 0; x < NX; ++x) {
          zero(s[x]);
          zero(dp[x]);
          beside<frag, FORM, kAhead>(read(x), [&](int i, const frag& f) { form(x, i, f); });
          prepare(x);
          weigh(x, 0, 16);
          if (STRICT && edge) {
            if constexpr (DV)
              add_rows_seen<T, DP, BQ>(buf + L::BYTES, 32 * x, from - query0, BQ, p[x], dv);
            if constexpr (DK)
              add_rows_seen<T, DP, BQ>(buf, 32 * x, from - query0, BQ, ds[x], dk);
          } else {
            beside<frag, ADD, kAhead>(read_t(x), [&](int i, const frag& f) { add(x, i, f); });
          }
        }
        return;
      }
#pragma unroll
      for (int x = 0; x < NX; ++x) {
        zero(s[x]);
        zero(dp[x]);
      }
      beside<frag, FORM, kAhead>(read(0), [&](int i, const frag& f) { form(0, i, f); });
#pragma unroll
      for (int x = 0; x < NX; ++x) {
        prepare(x);
        if (x + 1 < NX) {
          beside<frag, FORM, kAhead>(read(x + 1), [&](int i, const frag& f) {
            form(x + 1, i, f);
            weigh(x, 16 * i / FORM, 16 * (i + 1) / FORM);
          });
        } else if (x > 0) {
          beside<frag, ADD, kAhead>(read_t(x - 1), [&](int i, const frag& f) {
            add(x - 1, i, f);
            weigh(x, 16 * i / ADD, 16 * (i + 1) / ADD);
          });
        } else {
          weigh(x, 0, 16);
        }
      }
      beside<frag, ADD, kAhead>(read_t(NX - 1), [&](int i, const frag& f) { add(NX - 1, i, f); });
    };
    if (n < end) start(qh, qt, lds);
    while (n < end) {
      step(std::integral_constant<int, 0>());
      if (++n == end) break;
      step(std::integral_constant<int, 1>());
      ++n;
    }
    bool bad = false;
    if constexpr (CAUSAL && !STRICT) bad = any_not_finite(dk) || any_not_finite(dv);
    report<CAUSAL, STRICT>(a.again, bad, &bad_lds);
    if (!live) return;
    const float fk = a.scale * __builtin_amdgcn_exp2f(-lift), fv = __builtin_amdgcn_exp2f(-kLift<T>);
    const int64_t r = t.lo + at;
    if (a.shares > 1) {
      float* to = a.part + (((place.share * 2) * a.ks.rows + r) * a.Hk + place.head) * a.D;
      if constexpr (DK) store_part<DP, V>(to, a.D, [&](int d, int i) { return dk[d][i] * fk; });
      if constexpr (DV)
        store_part<DP, V>(to + a.ks.rows * a.Hk * a.D, a.D, [&](int d, int i) { return dv[d][i] * fv; });
      return;
    }
    if constexpr (DK)
      if (a.dk.p)
        store_head<T, DP>(a.dk.p + r * a.dk.row + place.head * a.dk.head, a.D,
                          [&](int d, int i) { return dk[d][i] * fk; });
    if constexpr (DV)
      if (a.dv.p)
        store_head<T, DP>(a.dv.p + r * a.dv.row + place.head * a.dv.head, a.D,
                          [&](int d, int i) { return dv[d][i] * fv; });
  };
  if constexpr (STRICT) {
    // (one after the other: both at once take more registers than there are, 1.3 KB of scratch a lane at 128 values)
    pass(std::true_type(), std::false_type());
    __syncthreads();  // (the last tile is read by all before the first one is loaded again)
    pass(std::false_type(), std::true_type());
  } else {
    pass(std::true_type(), std::true_type());
  }
}

// out[r][h] = the sum of the shares' partials, which lie `stride` values apart: four values a lane, four runs of
// the shares summed apart and then in order (one lane for all of 54 shares took 18 us for 20 MB).
template <typename T>
__global__ __launch_bounds__(kAttnThreads) void attend_sum(const float* __restrict__ part,
                                                           int64_t stride, int shares,
                                                           int64_t rows, int heads, int D,
                                                           Heads<T> out) {
  __shared__ float4v lds[4][64];
  const int lane = int(threadIdx.x) & 63, run = int(threadIdx.x) >> 6, quads = D / 4;
  const int64_t i = int64_t(blockIdx.x) * 64 + lane, n = rows * heads * quads;
  float4v v = {0.f, 0.f, 0.f, 0.f};
  if (i < n) {
    const int per = (shares + 3) / 4, end = (run + 1) * per < shares ? (run + 1) * per : shares;
#pragma unroll 8
    for (int s = run * per; s < end; ++s)
      v += *reinterpret_cast<const float4v*>(part + s * stride + i * 4);
  }
  lds[run][lane] = v;
  __syncthreads();
  if (run != 0 || i >= n) return;
  v = ((lds[0][lane] + lds[1][lane]) + lds[2][lane]) + lds[3][lane];
  const int64_t at = i / quads, r = at / heads;
  T* to = out.p + r * out.row + (at - r * heads) * out.head + (i - at * quads) * 4;
#pragma unroll
  for (int j = 0; j < 4; ++j) to[j] = from_f32<T>(v[j]);
}

// ---- host ------------------------------------------------------------------------
constexpr int kGradRows = kAttnWaves * 32;

AttnGradLayout attn_grad_layout(const Seqs& q, const Seqs& k, int H, int Hk, int D,
                                bool causal, int32_t dtype) {
  AttnGradLayout l{};
  with_width(D, [&](auto w) {
    const bool f32 = dtype == SP_F32;
    l.dq_shares = attn_shares(attn_tiles(q, H / Hk, Hk, kGradRows), attn_length(k),
                              256 * (f32 ? dq_waves<float>(w.value) : dq_waves<__bf16>(w.value)));
    l.dkv_shares =
        attn_shares(attn_tiles(k, 1, Hk, kGradRows), attn_length(q) * (H / Hk),
                    256 * (f32 ? grad_waves<float>(w.value) : grad_waves<__bf16>(w.value)));
    return 0;
  });
  size_t off = 0;
  auto take = [&](size_t floats) {
    const size_t at = off;
    off = align_up(off + floats * sizeof(float), 256);
    return at;
  };
  l.nl = take(size_t(q.rows) * H);
  l.nd = take(size_t(q.rows) * H);
  l.tops = take(2 * kTops);
  // (one after the other)
  const size_t dq = l.dq_shares > 1 ? size_t(l.dq_shares) * q.rows * H * D : 0;
  const size_t dkv = l.dkv_shares > 1 ? size_t(l.dkv_shares) * 2 * k.rows * Hk * D : 0;
  l.part = take(dq > dkv ? dq : dkv);
  if (causal) {
    const int64_t gq = attn_groups(tile_slots(q, H / Hk, kGradRows), Hk, l.dq_shares);
    const int64_t gk = attn_groups(tile_slots(k, 1, kGradRows), Hk, l.dkv_shares);
    l.again = take(size_t(gq > gk ? gq : gk));
  }
  l.total = off;
  return l;
}

template <typename T>
int attn_backward(AttnArgs<T> a, const AttnGradLayout& l, char* ws, bool need_dq, bool need_dkv,
                  hipStream_t s) {
  float* nl = reinterpret_cast<float*>(ws + l.nl);
  float* nd = reinterpret_cast<float*>(ws + l.nd);
  float* tops = reinterpret_cast<float*>(ws + l.tops);
  a.part = reinterpret_cast<float*>(ws + l.part);
  a.again = reinterpret_cast<int*>(ws + l.again);
  a.top = tops;
  if (!need_dq && !need_dkv) return SP_OK;
  const int64_t q_slots = tile_slots(a.qs, a.G, kGradRows), k_slots = tile_slots(a.ks, 1, kGradRows);
  const int64_t q_groups = attn_groups(q_slots, a.Hk, l.dq_shares);
  const int64_t k_groups = attn_groups(k_slots, a.Hk, l.dkv_shares);
  auto sums = [&](int shares, int64_t n) { return shares > 1 ? cdiv(n * (a.D / 4), 64) : 0; };
  SP_CHECK_ARG((!need_dq || (q_groups <= kAttnMaxGroups &&
                             sums(l.dq_shares, a.qs.rows * a.H) <= kAttnMaxGroups)) &&
                   (!need_dkv || (k_groups <= kAttnMaxGroups &&
                                  sums(l.dkv_shares, a.ks.rows * a.Hk) <= kAttnMaxGroups)),
               "attention_bwd: too many rows and sequences for a launch");
  int lanes = 0;
  while ((Mfma<T>::V << lanes) < a.D) ++lanes;
  const int64_t most = a.qs.rows * a.H > a.ks.rows * a.Hk ? a.qs.rows * a.H : a.ks.rows * a.Hk;
  const int64_t rows = cdiv(most, kAttnThreads >> lanes);
  a.tops = int(rows < kTops ? rows : kTops);
  attend_grad_rows<T><<<unsigned(a.tops), kAttnThreads, 0, s>>>(a, lanes, nl, nd, tops);
  SP_LAUNCHED();
  auto sum = [&](const float* part, int64_t stride, int shares, int64_t n, int heads,
                 const Heads<T>& out) -> int {
    if (!out.p) return SP_OK;
    attend_sum<T><<<unsigned(cdiv(n * heads * (a.D / 4), 64)), kAttnThreads, 0, s>>>(part, stride, shares, n, heads, a.D, out);
    SP_LAUNCHED();
    return SP_OK;
  };
  if (need_dq) {
    const int64_t slots = q_slots;
    a.shares = l.dq_shares;
    with_width(a.D, [&](auto w) {
      constexpr int DP = w.value, B = attn_stage<T>();
      const dim3 grid{unsigned(q_groups)}, block{kAttnThreads};
      if (!a.causal) {
        attend_dq<T, DP, B, false, false><<<grid, block, 0, s>>>(a, nl, nd, slots);
      } else {
        attend_dq<T, DP, B, true, false><<<grid, block, 0, s>>>(a, nl, nd, slots);
        attend_dq<T, DP, B, true, true><<<grid, block, 0, s>>>(a, nl, nd, slots);
      }
      return 0;
    });
    SP_LAUNCHED();
    if (a.shares > 1)
      if (int rc = sum(a.part, a.qs.rows * a.H * a.D, a.shares, a.qs.rows, a.H, a.dq)) return rc;
  }
  if (need_dkv) {
    const int64_t slots = k_slots;
    a.shares = l.dkv_shares;
    with_width(a.D, [&](auto w) {
      constexpr int DP = w.value, B = attn_stage<T>();
      const dim3 grid{unsigned(k_groups)}, block{kAttnThreads};
      if (!a.causal) {
        attend_dkv<T, DP, B, false, false><<<grid, block, 0, s>>>(a, nl, nd, slots);
      } else {
        attend_dkv<T, DP, B, true, false><<<grid, block, 0, s>>>(a, nl, nd, slots);
        attend_dkv<T, DP, B, true, true><<<grid, block, 0, s>>>(a, nl, nd, slots);
      }
      return 0;
    });
    SP_LAUNCHED();
    if (a.shares > 1) {
      const int64_t one = a.ks.rows * a.Hk * a.D;
      if (int rc = sum(a.part, 2 * one, a.shares, a.ks.rows, a.Hk, a.dk)) return rc;
      if (int rc = sum(a.part + one, 2 * one, a.shares, a.ks.rows, a.Hk, a.dv)) return rc;
    }
  }
  return SP_OK;
}

template int attn_backward<_Float16>(AttnArgs<_Float16>, const AttnGradLayout&, char*, bool, bool,
                                     hipStream_t);
template int attn_backward<__bf16>(AttnArgs<__bf16>, const AttnGradLayout&, char*, bool, bool,
                                   hipStream_t);
template int attn_backward<float>(AttnArgs<float>, const AttnGradLayout&, char*, bool, bool,
                                  hipStream_t);

}  // namespace sp
