// Softmax attention of packed sequences of rows, forward pass:
//
//   S = scale q k', P = softmax(S) over the keys that a query sees, O = P v
//
// Everything is computed transposed, with the queries as the MFMAs' columns: S' = K Q', O' += V' P'.
// A lane then holds one query, and the accumulators of the first product are the second one's operand:
// P exists in registers only.  Keys pass through LDS a tile at a time with the running maximum
// and sum of the softmax; the query heads that share a key head are rows of one tile.
//
// Statistics and sums are fp32.  P is rounded to the rows' type between the products, as the matrix
// instructions take it.  Weights are relative to a base at or below the largest score, and no weight exceeds 2^15.  fp16
// rounds weights below 2^-14 to multiples of 2^-24, so its base lies 2^8 below a maximum, and a weight is off by at most
// 2^-33 of the largest one: over 2^21 keys by half a step of the type.  (With the maximum itself as the base 2^18 keys
// 25 ln 2 below one other, 2^-7 of the sum, came out as twice as much.)
//
// Bound by the vector unit beside the matrix cores: a weight costs an exponential (8 cycles of a SIMD for 64 of them,
// 4 times an addition), its conversion and its sum, and a matrix instruction keeps the vector unit from
// issuing for half of its time.  Self-attention of 8 heads of 64 bf16 values, 6.6e11 operations:
// 846 us, 783 TFLOP/s (a library product of 8192^3 reaches 1 138 on the same card); causal, 128 fp16 values, 1.4e11:
// 223 us; 4 heads of 16 fp16 values in windows of 1024 rows, where half of the products are padding: 194 us for 8.2e8
// weights.  One query over 120k keys of 8 heads of 32 fp16 values: 41 us, 3.0 TB/s.
// Not faster: two query tiles a wave (945 us for 880 at 64 values), eight waves a workgroup (713 for 625),
// three key tiles in flight, the next tile's scores beside this tile's weights (892), four waves a SIMD (spills).
#include "sp_attention.h"

namespace sp {

// A lane's weights of a tile may sum up to this before they are put relative to a new maximum (fp16 holds
// weights up to 2^16).
constexpr float kMostWeight = 32768.f;

// The base of the weights below the maximum that sets it, in powers of two.
template <typename T>
constexpr float kBelow = std::is_same<T, _Float16>::value ? 8.f : 0.f;

// Waves a SIMD (of a launch that makes results again: as few as leave it all registers).
template <typename T>
constexpr int attend_waves(int DP, bool strict = false) {
  if (strict) return 1;
  return sizeof(T) == 4 ? (DP <= 32 ? 4 : DP <= 64 ? 2 : 1) : DP <= 32 ? 4 : DP <= 64 ? 3 : 2;
}

template <typename T, int DP, int BK, bool CAUSAL, bool STRICT>
__global__ __launch_bounds__(kAttnThreads, attend_waves<T>(DP, STRICT)) void attend(
    AttnArgs<T> a, int64_t slots) {
  using frag = typename Mfma<T>::frag;
  using L = HeadTile<T, DP, BK>;
  constexpr int STEPS = DP / Mfma<T>::KSTEP, PS = 32 / Mfma<T>::KSTEP, V = Mfma<T>::V;
  constexpr int NK = BK / 32, BQ = kAttnWaves * 32, TILES = DP / 32;
  __shared__ __attribute__((aligned(16))) char lds[4 * L::BYTES];
  __shared__ int bad_lds;
  Place place;
  if (!find_place(slots, a.Hk, a.shares, blockIdx.x, place)) return;
  if (skips<CAUSAL, STRICT>(a.again)) return;
  if (CAUSAL) place.slot = slots - 1 - place.slot;  // (the longest rows first)
  const Tile t = find_tile(a.qs, a.G, BQ, place.slot);
  if (t.at >= t.len) {
    if (CAUSAL && !STRICT && threadIdx.x == 0) a.again[blockIdx.x] = 0;
    return;
  }
  const int64_t klo = a.ks.bound(t.part);
  const int Lk = keys_of(a.qs, a.ks, t.part, klo), Lq = int(t.len / a.G);

  // this lane's query
  const int wave = wave_of(), lane = int(threadIdx.x) & 31, half = (int(threadIdx.x) >> 5) & 1;
  const int64_t r = t.at + wave * 32 + lane;
  const bool live = r < t.len;
  const int row = int(r / a.G), head = place.head * a.G + int(r - int64_t(row) * a.G);
  const int seen = CAUSAL ? keys_seen(row, Lq, Lk) : Lk;  // how many keys it sees
  frag q[STEPS];
  load_head<T, DP>(a.q.p + (t.lo + row) * a.q.row + head * a.q.head, live, a.D, q);
  // keys that some query of the workgroup or wave sees, and that every one of the wave sees
  int most = Lk, wave_most = Lk, wave_least = Lk;
  if (CAUSAL) {
    const int64_t last = t.at + BQ < t.len ? t.at + BQ : t.len, w = t.at + wave * 32;
    most = keys_seen((last - 1) / a.G, Lq, Lk);
    wave_least = keys_seen(w / a.G, Lq, Lk);
    wave_most = keys_seen((w + 31) / a.G, Lq, Lk);
    wave_most = wave_most < most ? wave_most : most;
  }

  // this share's tiles
  const int tiles = (most + BK - 1) / BK, per = (tiles + a.shares - 1) / a.shares;
  const int first = place.share * per, end = first + per < tiles ? first + per : tiles;
  const TileLoads<T, DP, BK> lk(a.k.p + klo * a.k.row + place.head * a.k.head, a.k.row, Lk, a.D);
  const TileLoads<T, DP, BK> lv(a.v.p + klo * a.v.row + place.head * a.v.head, a.v.row, Lk, a.D);
  const float c = a.scale2;
  floatx16 o[TILES];
  float m = -__builtin_inff(), neg = 0.f, l = 0.f;
#pragma unroll
  for (int d = 0; d < TILES; ++d) zero(o[d]);
  // Tile n, in buffer B (constants, so that the reads' addresses stay in registers).
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
    if (CAUSAL && key0 >= wave_most) return;
    const bool edge = key0 + BK > wave_least;
    floatx16 s[NK];
#pragma unroll
    for (int x = 0; x < NK; ++x) zero(s[x]);
    // (products of neighbouring keys in turn: one that adds to the result of the one before waits for it)
    auto read = [&](int i) { return L::read(buf, 32 * (i % NK), i / NK); };
    Batched<frag, STEPS * NK, kAttnBatch> f;
    f.start(read);
    f.run(read, [&](int i, const frag& kf) { Mfma<T>::mma(kf, q[i / NK], s[i % NK]); });
    if (edge) {
#pragma unroll
      for (int x = 0; x < NK; ++x)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (key0 + 32 * x + acc_row<T>(i) >= seen) s[x][i] = -__builtin_inff();
    }
    // Weights relative to the maximum so far.  Only where their sum grows out of hand (or there is no
    // maximum yet) is the tile's maximum found and everything put relative to it.
    frag p[NK][PS];
    float sum[2];
    auto weigh = [&]() {
      sum[0] = sum[1] = 0.f;
#pragma unroll
      for (int x = 0; x < NK; ++x)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(s[x][i], c, neg));
          sum[i & 1] += e;
          p[x][i / V][i % V] = T(e);
        }
      sum[0] += sum[1];
    };
    const bool fresh = __ballot(m == -__builtin_inff()) != 0;
    if (!fresh) weigh();
    if (fresh || __ballot(sum[0] > kMostWeight)) {
      float mx = s[0][0];
#pragma unroll
      for (int x = 0; x < NK; ++x)
#pragma unroll
        for (int i = 0; i < 16; ++i) mx = __builtin_fmaxf(mx, s[x][i]);
      const float now = __builtin_fmaxf(half_max(mx) * c - kBelow<T>, m);
      const float safe = now == -__builtin_inff() ? 0.f : now;
      const float down = __builtin_amdgcn_exp2f(m - safe);
      m = now;
      neg = -safe;
      l *= down;
#pragma unroll
      for (int d = 0; d < TILES; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d][i] *= down;
      weigh();
    }
    l += sum[0];
#pragma unroll
    for (int x = 0; x < NK; ++x) {
      if (STRICT && edge)
        add_rows_seen<T, DP, BK>(buf + L::BYTES, 32 * x, 0, seen - key0, p[x], o);
      else
        add_rows<T, DP, BK, kAttnBatch>(buf + L::BYTES, 32 * x, p[x], o);
    }
  };
  if (first < end) {
    lk.start(first * BK, lds);
    lv.start(first * BK, lds + L::BYTES);
  }
  for (int n = first; n < end; n += 2) {
    step(n, std::integral_constant<int, 0>());
    if (n + 1 < end) step(n + 1, std::integral_constant<int, 1>());
  }
  report<CAUSAL, STRICT>(a.again, CAUSAL && !STRICT && any_not_finite(o), &bad_lds);

  const float sum = half_sum(l);
  if (!live) return;
  const int64_t rows = a.qs.rows, at = t.lo + row;
  if (a.shares > 1) {
    const int64_t i = (place.share * rows + at) * a.H + head;
    store_part<DP, V>(a.part + i * a.D, a.D, [&](int d, int j) { return o[d][j]; });
    if (half == 0) {
      a.part_ml[2 * i] = m;
      a.part_ml[2 * i + 1] = sum;
    }
    return;
  }
  // (a row without keys is zeros)
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  store_head<T, DP>(a.out.p + at * a.out.row + head * a.out.head, a.D,
                    [&](int d, int j) { return o[d][j] * inv; });
  if (a.lse && half == 0)
    a.lse[head * rows + at] = sum == 0.f ? __builtin_inff() : m + __builtin_amdgcn_logf(sum);
}

// The shares' results of a row and head joined, a workgroup each.  Every thread weighs some shares, then adds
// up four values over some of them (one wave going through all shares by itself took 54 us for one
// query's 8 heads of 32 in 96 shares, where the pass over 120k keys took 45).
template <typename T>
__global__ __launch_bounds__(kAttnThreads) void attend_join(AttnArgs<T> a) {
  __shared__ float weight[kMostShares];
  __shared__ float4v lds[kAttnThreads];
  __shared__ float wave_max[kAttnWaves], wave_sum[kAttnWaves];
  const int64_t n = a.qs.rows * a.H, at = blockIdx.x;
  const int tid = int(threadIdx.x), lane = tid & 63, wave = wave_of();
  float m = -__builtin_inff();
  for (int s = tid; s < a.shares; s += kAttnThreads) {
    const float v = a.part_ml[2 * (s * n + at)];
    weight[s] = v;
    m = __builtin_fmaxf(m, v);
  }
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) m = __builtin_fmaxf(m, __shfl_xor(m, off, 64));
  if (lane == 0) wave_max[wave] = m;
  __syncthreads();
  m = wave_max[0];
#pragma unroll
  for (int w = 1; w < kAttnWaves; ++w) m = __builtin_fmaxf(m, wave_max[w]);
  const float safe = m == -__builtin_inff() ? 0.f : m;
  float sum = 0.f;
  for (int s = tid; s < a.shares; s += kAttnThreads) {
    const float w = __builtin_amdgcn_exp2f(weight[s] - safe);
    weight[s] = w;
    sum = __builtin_fmaf(w, a.part_ml[2 * (s * n + at) + 1], sum);
  }
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) sum += __shfl_xor(sum, off, 64);
  if (lane == 0) wave_sum[wave] = sum;
  __syncthreads();
  sum = 0.f;
#pragma unroll
  for (int w = 0; w < kAttnWaves; ++w) sum += wave_sum[w];
  const int quads = a.D / 4, runs = kAttnThreads / quads, run = tid / quads, c = tid - run * quads;
  float4v v = {0.f, 0.f, 0.f, 0.f};
  if (run < runs) {
#pragma unroll 4
    for (int s = run; s < a.shares; s += runs)
      v += weight[s] * *reinterpret_cast<const float4v*>(a.part + (s * n + at) * a.D + 4 * c);
  }
  lds[tid] = v;
  __syncthreads();
  if (run == 0) {
    for (int r = 1; r < runs; ++r) v += lds[r * quads + c];
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    const int64_t r = at / a.H;
    T* to = a.out.p + r * a.out.row + (at - r * a.H) * a.out.head + 4 * c;
#pragma unroll
    for (int i = 0; i < 4; ++i) to[i] = from_f32<T>(v[i] * inv);
  }
  if (a.lse && tid == 0) {
    const int64_t r = at / a.H;
    a.lse[(at - r * a.H) * a.qs.rows + r] =
        sum == 0.f ? __builtin_inff() : m + __builtin_amdgcn_logf(sum);
  }
}

// The same for few shares, four values a thread.
constexpr int kFewShares = 16;
template <typename T>
__global__ __launch_bounds__(kAttnThreads) void attend_join_few(AttnArgs<T> a) {
  const int quads = a.D / 4;
  const int64_t n = a.qs.rows * a.H, i = int64_t(blockIdx.x) * kAttnThreads + threadIdx.x;
  const int64_t at = i / quads;
  if (at >= n) return;
  const int c = int(i - at * quads) * 4;
  const float2* ml = reinterpret_cast<const float2*>(a.part_ml) + at;
  float m = -__builtin_inff();
  for (int s = 0; s < a.shares; ++s) m = __builtin_fmaxf(m, ml[s * n].x);
  const float safe = m == -__builtin_inff() ? 0.f : m;
  float sum = 0.f;
  float4v v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = 0; s < a.shares; ++s) {
    const float2 o = ml[s * n];
    const float w = __builtin_amdgcn_exp2f(o.x - safe);
    sum = __builtin_fmaf(w, o.y, sum);
    v += w * *reinterpret_cast<const float4v*>(a.part + (s * n + at) * a.D + c);
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  const int64_t r = at / a.H, h = at - r * a.H;
  T* to = a.out.p + r * a.out.row + h * a.out.head + c;
#pragma unroll
  for (int j = 0; j < 4; ++j) to[j] = from_f32<T>(v[j] * inv);
  if (a.lse && c == 0)
    a.lse[h * a.qs.rows + r] = sum == 0.f ? __builtin_inff() : m + __builtin_amdgcn_logf(sum);
}

// ---- host ------------------------------------------------------------------------
constexpr int kForwardRows = kAttnWaves * 32;

template <typename T>
static int launch_attend(AttnArgs<T> a, hipStream_t s) {
  const int64_t slots = tile_slots(a.qs, a.G, kForwardRows);
  const int64_t groups = attn_groups(slots, a.Hk, a.shares);
  const bool few = a.shares <= kFewShares;
  const int64_t rows = a.qs.rows * a.H;
  const int64_t joins =
      a.shares == 1 ? 0 : few ? cdiv(rows * (a.D / 4), kAttnThreads) : rows;
  SP_CHECK_ARG(groups <= kAttnMaxGroups && joins <= kAttnMaxGroups,
               "attention: too many rows and sequences for a launch");
  with_width(a.D, [&](auto w) {
    constexpr int DP = w.value, BK = attn_stage<T>();
    const dim3 grid{unsigned(groups)}, block{kAttnThreads};
    if (!a.causal) {
      attend<T, DP, BK, false, false><<<grid, block, 0, s>>>(a, slots);
    } else {
      attend<T, DP, BK, true, false><<<grid, block, 0, s>>>(a, slots);
      attend<T, DP, BK, true, true><<<grid, block, 0, s>>>(a, slots);
    }
    return 0;
  });
  SP_LAUNCHED();
  if (a.shares == 1) return SP_OK;
  if (few)
    attend_join_few<T><<<unsigned(joins), kAttnThreads, 0, s>>>(a);
  else
    attend_join<T><<<unsigned(joins), kAttnThreads, 0, s>>>(a);
  SP_LAUNCHED();
  return SP_OK;
}

static int check_heads(const char* what, const char* name, const void* p, int64_t row,
                       int64_t head, int64_t heads, int64_t dim, int V) {
  SP_CHECK_ARG(p, "%s: %s is null", what, name);
  SP_CHECK_ARG(aligned(p) && row % V == 0 && head % V == 0,
               "%s: heads of %s do not start at multiples of 16 bytes", what, name);
  SP_CHECK_ARG((heads == 1 || head >= dim) && row >= 0, "%s: heads of %s overlap", what, name);
  SP_CHECK_ARG(row < (1 << 23), "%s: %s has 2^23 values or more from row to row", what, name);
  return SP_OK;
}

static int check_call(const char* what, const sp_attn* a) {
  SP_CHECK_ARG(a, "%s: null arguments", what);
  SP_CHECK_ARG(a->dtype == SP_F16 || a->dtype == SP_BF16 || a->dtype == SP_F32,
               "%s: dtype %d not supported (f16/bf16/f32)", what, a->dtype);
  const int V = vec_of(a->dtype);
  SP_CHECK_ARG(a->heads >= 1 && a->kv_heads >= 1 && a->heads < 65536 &&
                   a->heads % a->kv_heads == 0,
               "%s: %lld query heads for %lld key heads", what, (long long)a->heads,
               (long long)a->kv_heads);
  SP_CHECK_ARG(a->dim >= 1 && a->dim % V == 0, "%s: head width %lld is no multiple of %d", what,
               (long long)a->dim, V);
  if (a->dim > kAttnMaxDim)
    return set_error(SP_ERR_UNSUPPORTED, "%s: heads wider than %d", what, kAttnMaxDim);
  SP_CHECK_ARG(a->nq >= 0 && a->nk >= 0 && a->nq <= kAttnMaxRows && a->nk <= kAttnMaxRows,
               "%s: bad row counts %lld and %lld (at most 2^31 - 128)", what, (long long)a->nq,
               (long long)a->nk);
  SP_CHECK_ARG((a->q_offsets == nullptr) == (a->k_offsets == nullptr),
               "%s: offsets of queries and keys go together", what);
  SP_CHECK_ARG(!a->q_offsets || (a->sequences >= 0 && a->sequences < (1 << 30)),
               "%s: bad number of sequences %lld", what, (long long)a->sequences);
  SP_CHECK_ARG(a->scale > 0.f && a->scale < __builtin_inff(), "%s: the scale must be positive",
               what);
  if (a->nq) {
    if (int rc = check_heads(what, "q", a->q, a->q_row, a->q_head, a->heads, a->dim, V)) return rc;
  }
  if (a->nk) {
    if (int rc = check_heads(what, "k", a->k, a->k_row, a->k_head, a->kv_heads, a->dim, V))
      return rc;
    if (int rc = check_heads(what, "v", a->v, a->v_row, a->v_head, a->kv_heads, a->dim, V))
      return rc;
  }
  return SP_OK;
}

static Seqs seqs(const int32_t* off, int64_t rows, int64_t n) {
  return Seqs{off, rows, off ? int(n) + 2 : 1};
}

template <typename T>
static AttnArgs<T> arguments(const sp_attn& c) {
  AttnArgs<T> a{};
  a.q = {static_cast<const T*>(c.q), c.q_row, c.q_head};
  a.k = {static_cast<const T*>(c.k), c.k_row, c.k_head};
  a.v = {static_cast<const T*>(c.v), c.v_row, c.v_head};
  a.qs = seqs(c.q_offsets, c.nq, c.sequences);
  a.ks = seqs(c.k_offsets, c.nk, c.sequences);
  a.H = int(c.heads);
  a.Hk = int(c.kv_heads);
  a.G = a.H / a.Hk;
  a.D = int(c.dim);
  a.causal = c.causal != 0;
  a.scale = c.scale;
  a.scale2 = c.scale * 1.4426950408889634f;
  a.shares = 1;
  return a;
}

// Workgroups that are resident at a time.
static int forward_groups(int32_t dtype, int dim) {
  return 256 * with_width(dim, [&](auto w) {
    return dtype == SP_F32 ? attend_waves<float>(w.value) : attend_waves<__bf16>(w.value);
  });
}

struct ForwardLayout {
  size_t part, ml, again, total;
  int shares;
};

static ForwardLayout forward_layout(const sp_attn& c) {
  const Seqs q = seqs(c.q_offsets, c.nq, c.sequences), k = seqs(c.k_offsets, c.nk, c.sequences);
  const int G = int(c.heads / c.kv_heads), Hk = int(c.kv_heads);
  ForwardLayout l{};
  l.shares = attn_shares(attn_tiles(q, G, Hk, kForwardRows), attn_length(k),
                         forward_groups(c.dtype, int(c.dim)));
  size_t off = 0;
  auto take = [&](size_t bytes) {
    const size_t at = off;
    off = align_up(off + bytes, 256);
    return at;
  };
  const size_t rows = l.shares > 1 ? size_t(l.shares) * c.nq * c.heads : 0;
  l.part = take(rows * c.dim * sizeof(float));
  l.ml = take(rows * 2 * sizeof(float));
  if (c.causal)
    l.again = take(size_t(attn_groups(tile_slots(q, G, kForwardRows), Hk, l.shares)) * sizeof(int));
  l.total = off;
  return l;
}

template <typename T>
static int run_forward(const sp_attn& c, void* out, int64_t row, int64_t head, float* lse,
                       char* ws, hipStream_t s) {
  AttnArgs<T> a = arguments<T>(c);
  a.out = {static_cast<T*>(out), row, head};
  a.lse = lse;
  const ForwardLayout l = forward_layout(c);
  a.shares = l.shares;
  a.part = reinterpret_cast<float*>(ws + l.part);
  a.part_ml = reinterpret_cast<float*>(ws + l.ml);
  a.again = reinterpret_cast<int*>(ws + l.again);
  return launch_attend(a, s);
}

template <typename T>
static int run_backward(const sp_attn& c, const sp_attn_grad& g, const AttnGradLayout& l, char* ws,
                        hipStream_t s) {
  AttnArgs<T> a = arguments<T>(c);
  a.o = {static_cast<const T*>(g.o), g.o_row, g.o_head};
  a.dout = {static_cast<const T*>(g.dout), g.dout_row, g.dout_head};
  a.lse = const_cast<float*>(g.lse);
  a.dq = {static_cast<T*>(g.dq), g.dq_row, g.dq_head};
  a.dk = {static_cast<T*>(g.dk), g.dk_row, g.dk_head};
  a.dv = {static_cast<T*>(g.dv), g.dv_row, g.dv_head};
  return attn_backward<T>(a, l, ws, g.dq != nullptr && c.nq > 0,
                          (g.dk != nullptr || g.dv != nullptr) && c.nk > 0, s);
}

}  // namespace sp

using namespace sp;

extern "C" size_t sp_attention_workspace(const sp_attn* c) {
  if (check_call("attention", c) != SP_OK || c->nq == 0) return 0;
  return forward_layout(*c).total;
}

extern "C" int sp_attention(const sp_attn* c, void* out, int64_t out_row, int64_t out_head,
                            float* lse, void* ws, size_t ws_bytes, void* stream) {
  if (int rc = check_call("attention", c)) return rc;
  if (c->nq == 0) return SP_OK;
  if (int rc = check_heads("attention", "out", out, out_row, out_head, c->heads, c->dim,
                           vec_of(c->dtype)))
    return rc;
  const size_t need = sp_attention_workspace(c);
  if (ws_bytes < need)
    return set_error(SP_ERR_WORKSPACE, "attention: workspace of %zu bytes, needs %zu", ws_bytes,
                     need);
  SP_CHECK_ARG(!need || (ws && aligned(ws)), "attention: the workspace must be 16-byte aligned");
  char* w = static_cast<char*>(ws);
  const hipStream_t s = as_stream(stream);
  if (c->dtype == SP_F16)
    return run_forward<_Float16>(*c, out, out_row, out_head, lse, w, s);
  if (c->dtype == SP_BF16) return run_forward<__bf16>(*c, out, out_row, out_head, lse, w, s);
  return run_forward<float>(*c, out, out_row, out_head, lse, w, s);
}

static AttnGradLayout grad_layout(const sp_attn* c) {
  return attn_grad_layout(seqs(c->q_offsets, c->nq, c->sequences),
                          seqs(c->k_offsets, c->nk, c->sequences), int(c->heads),
                          int(c->kv_heads), int(c->dim), c->causal != 0, c->dtype);
}

extern "C" size_t sp_attention_bwd_workspace(const sp_attn* c) {
  if (check_call("attention_bwd", c) != SP_OK || (c->nq == 0 && c->nk == 0)) return 0;
  return grad_layout(c).total;
}

extern "C" int sp_attention_bwd(const sp_attn* c, const sp_attn_grad* g, void* ws, size_t ws_bytes,
                                void* stream) {
  if (int rc = check_call("attention_bwd", c)) return rc;
  SP_CHECK_ARG(g, "attention_bwd: null arguments");
  if (c->nq == 0 && c->nk == 0) return SP_OK;
  const int V = vec_of(c->dtype);
  auto check = [&](const char* name, const void* p, int64_t row, int64_t head, int64_t heads) {
    return check_heads("attention_bwd", name, p, row, head, heads, c->dim, V);
  };
  if (c->nq) {
    if (int rc = check("o", g->o, g->o_row, g->o_head, c->heads)) return rc;
    if (int rc = check("dout", g->dout, g->dout_row, g->dout_head, c->heads)) return rc;
    SP_CHECK_ARG(g->lse, "attention_bwd: lse is null");
  }
  if (g->dq) {
    if (int rc = check("dq", g->dq, g->dq_row, g->dq_head, c->heads)) return rc;
  }
  if (g->dk) {
    if (int rc = check("dk", g->dk, g->dk_row, g->dk_head, c->kv_heads)) return rc;
  }
  if (g->dv) {
    if (int rc = check("dv", g->dv, g->dv_row, g->dv_head, c->kv_heads)) return rc;
  }
  const AttnGradLayout l = grad_layout(c);
  if (ws_bytes < l.total)
    return set_error(SP_ERR_WORKSPACE, "attention_bwd: workspace of %zu bytes, needs %zu",
                     ws_bytes, l.total);
  SP_CHECK_ARG(ws && aligned(ws), "attention_bwd: the workspace must be 16-byte aligned");
  char* w = static_cast<char*>(ws);
  const hipStream_t s = as_stream(stream);
  if (c->dtype == SP_F16) return run_backward<_Float16>(*c, *g, l, w, s);
  if (c->dtype == SP_BF16) return run_backward<__bf16>(*c, *g, l, w, s);
  return run_backward<float>(*c, *g, l, w, s);
}
