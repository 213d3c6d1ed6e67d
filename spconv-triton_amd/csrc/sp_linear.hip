// A linear layer of feature rows with its bias, activation and residual in the product's epilogue, and its
// gradients, on 32x32 MFMA tiles with fp32 accumulation:
//
//   z = x W' + b, y = act(z) + residual
//   dz = dy act'(z), dx = dz W, dW = dz' x, db = sum dz
//
// z is not kept: with an activation the backward pass forms it again, in a product whose epilogue writes dz
// (16-bit rows of up to some 400 channels read and write less than that product takes; keeping z
// would also hold rows x outputs of memory).  dz is rounded to the rows' type, as an operand of the
// products that follow; z, the activation and every sum are fp32.
//
// 75k x 256 -> 1024 bf16 with gelu and a residual, 3.9e10 operations a product: forward 132 us (346 MB of rows in and out are
// 70 at a copy's rate; then the activation, whose instructions come after the tile's four stages), dz 137, dx 74
// (531 TFLOP/s), dW and db 77 (510) and their shares' sums 12 (a library product of these operands: 66 forward,
// 53 for dx and 280 for dW).
#include "sp_tiles.h"

namespace sp {

enum { kActNone = 3 };  // beside the feed-forward block's activations

template <bool FAST, int ACT, typename F>
__device__ __forceinline__ void linear_act16(const floatx16& z, F&& f) {
  if constexpr (ACT == kActNone) {
#pragma unroll
    for (int i = 0; i < 16; ++i) f(i, z[i], 1.f);
  } else {
    gate16<FAST, ACT>(z, f);
  }
}

template <typename T>
struct LinearOut {
  const T *bias, *extra;  // extra: the residual, or dy
  int64_t lde, ldo;
  T* out;
  int n, columns;  // outputs; columns of `out`, zeros past n
  int act;
  int vec_b, vec_e, vec_o;
};

// A piece of V values from p on, of which `left` exist.
template <typename T>
__device__ __forceinline__ typename Mfma<T>::frag piece_at(const T* p, int left, bool vec) {
  constexpr int V = Mfma<T>::V;
  typename Mfma<T>::frag f = {};
  if (vec && left >= V) return *reinterpret_cast<const typename Mfma<T>::frag*>(p);
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (i < left) f[i] = p[i];
  return f;
}

// GRAD: out = extra * act'(z), else act(z) + extra.
template <typename T, typename S, bool ASYNC, bool GRAD>
__device__ __forceinline__ void linear_tile(const Rows<T>& x, const Rows<T>& w,
                                            const LinearOut<T>& o, int64_t x0, int n0, char* lds) {
  using frag = typename Mfma<T>::frag;
  constexpr int V = Mfma<T>::V;
  const int wave = int(threadIdx.x) >> 6, wm = wave / S::WW, wn = wave % S::WW;
  const int lane = int(threadIdx.x) & 31, half = (int(threadIdx.x) >> 5) & 1;
  const int xrow = wm * 32 * S::XT;
  floatx16 acc[S::XT][S::WT];
  clear(acc);
  int wrow[S::WT];
#pragma unroll
  for (int i = 0; i < S::WT; ++i) wrow[i] = (wn * S::WT + i) * 32;
  // Whole pieces of the bias and of the other input are loaded without a branch of lanes, behind which each load
  // would wait for the one before it: the bias, which the products are added to, while the first stage is on its way,
  // the other input in the smaller tiles before it.  What lies past the ends meets outputs that are not written.  The
  // epilogue is chosen once, not activation by activation within it (75k x 256 -> 1024 bf16, gelu, residual: 128 us,
  // 138 with branches and the bias added last).
  constexpr bool EARLY = ASYNC && S::XT * S::WT <= 2;
  const bool whole = (!o.bias || o.vec_b) && (!o.extra || o.vec_e) && o.n % V == 0;
  frag e[EARLY ? S::WT : 1][S::XT][16 / V];
  auto load = [&](int i, frag (&to)[S::XT][16 / V]) {
#pragma unroll
    for (int j = 0; j < S::XT; ++j) {
      const int64_t r = x0 + xrow + 32 * j + lane;
      const T* row = o.extra + (r < x.n ? r : x.n - 1) * o.lde;
#pragma unroll
      for (int p = 0; p < 16 / V; ++p) {
        const int c = n0 + wrow[i] + 2 * V * p + V * half;
        to[j][p] = *reinterpret_cast<const frag*>(row + (c < o.n ? c : o.n - V));
      }
    }
  };
  auto start = [&](auto get) {
    frag b[S::WT][16 / V];
#pragma unroll
    for (int i = 0; i < S::WT; ++i)
#pragma unroll
      for (int p = 0; p < 16 / V; ++p) b[i][p] = get(n0 + wrow[i] + 2 * V * p + V * half);
#pragma unroll
    for (int i = 0; i < S::WT; ++i)
#pragma unroll
      for (int j = 0; j < S::XT; ++j)
#pragma unroll
        for (int k = 0; k < 16; ++k) acc[j][i][k] = to_f32(b[i][k / V][k % V]);
  };
  if constexpr (EARLY)
    if (whole && o.extra) {
#pragma unroll
      for (int i = 0; i < S::WT; ++i) load(i, e[i]);
    }
  products<T, S, ASYNC, S::WT>(x, x0, w, nullptr, n0, wrow, xrow, lds, acc, [&] {
    if (!o.bias) return;
    if (whole)
      start([&](int c) { return *reinterpret_cast<const frag*>(o.bias + (c < o.n ? c : o.n - V)); });
    else
      start([&](int c) { return piece_at<T>(o.bias + c, o.n - c, o.vec_b); });
  });
  auto finish = [&](auto fast, auto act) {
    constexpr bool FAST = fast.value;
#pragma unroll
    for (int i = 0; i < S::WT; ++i) {
      const int c0 = n0 + wrow[i];
      if constexpr (FAST && !EARLY)
        if (o.extra) load(i, e[0]);
#pragma unroll
      for (int j = 0; j < S::XT; ++j) {
        const int64_t r = x0 + xrow + 32 * j + lane;
        frag own[16 / V];
#pragma unroll
        for (int p = 0; p < 16 / V; ++p) {
          const int c = c0 + 2 * V * p + V * half;
          own[p] = frag{};
          if constexpr (FAST)
            own[p] = o.extra ? e[EARLY ? i : 0][j][p] : frag{};
          else if (o.extra && r < x.n)
            own[p] = piece_at<T>(o.extra + r * o.lde + c, o.n - c, o.vec_e);
        }
        const floatx16 z = acc[j][i];
        linear_act16<sizeof(T) == 2, act.value>(z, [&](int k, float value, float slope) {
          const float v = to_f32(own[k / V][k % V]);
          acc[j][i][k] = GRAD ? v * slope : value + v;
        });
        write_piece_row<T>(o.out, o.ldo, r, x.n, c0, o.columns, o.vec_o, [&](int k, int c) {
          return GRAD && c >= o.n ? 0.f : acc[j][i][k];
        });
      }
    }
  };
  auto end = [&](auto act) {
    if (ASYNC && whole)
      finish(std::true_type(), act);
    else
      finish(std::false_type(), act);
  };
  if (o.act == kActNone)
    end(std::integral_constant<int, kActNone>());
  else
    with_act(o.act, end);
}

template <typename T, typename S, bool ASYNC, bool GRAD>
__global__ __launch_bounds__(S::THREADS, 2) void linear_rows(Rows<T> x, Rows<T> w,
                                                             LinearOut<T> o) {
  __shared__ __attribute__((aligned(16))) char lds[2 * S::BYTES];
  const int cols = (o.columns + S::W - 1) / S::W;
  const int64_t place = place_of((x.n + S::X - 1) / S::X * cols);
  if (place < 0) return;
  linear_tile<T, S, ASYNC, GRAD>(x, w, o, place / cols * S::X, int(place % cols) * S::W, lds);
}

// Up to four rows: a group of lanes an output, each weight read once.
template <typename T, int R>
__global__ __launch_bounds__(kFfnThreads) void linear_few(Rows<T> x, Rows<T> w, LinearOut<T> o,
                                                          int log_lanes) {
  constexpr int V = Mfma<T>::V;
  const int lanes = 1 << log_lanes, lane = int(threadIdx.x) & (lanes - 1);
  const int64_t c = int64_t(blockIdx.x) * (kFfnThreads >> log_lanes) + (int(threadIdx.x) >> log_lanes);
  float a[R];
#pragma unroll
  for (int i = 0; i < R; ++i) a[i] = 0.f;
  if (c < w.n)
    for (int k = lane * V; k < w.K; k += lanes * V) {
      const auto f = piece_of(w, c, k);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const auto v = piece_of(x, r < x.n ? r : x.n - 1, k);
#pragma unroll
        for (int i = 0; i < V; ++i) a[r] = __builtin_fmaf(to_f32(v[i]), to_f32(f[i]), a[r]);
      }
    }
  sum_lanes(a, lanes);
  if (c >= w.n || lane != 0) return;
  const float b = o.bias ? to_f32(o.bias[c]) : 0.f;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    if (r >= x.n) continue;
    const float z = a[r] + b;
    float value = z, slope;
    if (o.act != kActNone)
      with_act(o.act, [&](auto kind) { gate<false, kind.value>(z, value, slope); });
    if (o.extra) value += to_f32(o.extra[r * o.lde + c]);
    o.out[r * o.ldo + c] = from_f32<T>(value);
  }
}

// dst [cols][ldd] = src [rows][cols] transposed, zeros from rows to ldd.
template <typename T>
__global__ __launch_bounds__(kFfnThreads) void linear_transpose(const T* __restrict__ src, int rows,
                                                                int cols, T* __restrict__ dst,
                                                                int ldd) {
  __shared__ T tile[32][33];
  const int r0 = int(blockIdx.x) * 32, c0 = int(blockIdx.y) * 32;
  const int tx = int(threadIdx.x) & 31, ty = int(threadIdx.x) >> 5;
#pragma unroll
  for (int j = 0; j < 32; j += 8) {
    const int r = r0 + ty + j, c = c0 + tx;
    tile[ty + j][tx] = r < rows && c < cols ? src[int64_t(r) * cols + c] : T(0.f);
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < 32; j += 8) {
    const int c = c0 + ty + j, r = r0 + tx;
    if (c < cols && r < ldd) dst[int64_t(c) * ldd + r] = tile[tx][ty + j];
  }
}

// Partials of dW = dz' x over a share of the rows, TP x TQ a workgroup, and of db, which the workgroups of the
// first columns sum from what they stage.
template <typename T>
struct LinearGram {
  const T *a, *b;
  int64_t lda, ldb;
  int P, Q, tiles_q, tiles, vec_a, vec_b;
  float* part;           // [shares][P][Q], then P sums of rows, `stride` values a share
  int64_t stride;
  T *dw, *db;            // each nullable; written by the one share, where there is only one
  int bias;
};

template <typename T, int TP, int TQ>
__global__ __launch_bounds__(2 * TP, 2) void linear_gram(LinearGram<T> g, int64_t rows,
                                                         int64_t share, int shares) {
  constexpr int THREADS = 2 * TP, ROWS = gram_rows<T>();
  constexpr int NP = 2, NQ = TQ / 64;
  constexpr int STAGE = kGramStage * (TP + TQ);
  using SA = GramStage<T, TP, THREADS>;
  using SB = GramStage<T, TQ, THREADS>;
  __shared__ __attribute__((aligned(16))) char lds[2 * STAGE];
  const int64_t place = place_of(int64_t(g.tiles) * shares);
  if (place < 0) return;
  const int64_t lo = place / g.tiles * share;
  const int tile = int(place % g.tiles);
  const int p0 = tile / g.tiles_q * TP, q0 = tile % g.tiles_q * TQ;
  const int64_t hi = lo + share < rows ? lo + share : rows;
  const int wave = int(threadIdx.x) >> 6, wp = (wave >> 1) * 64, wq = (wave & 1) * (TQ / 2);
  const bool sums = g.bias && q0 == 0;
  constexpr int V = Mfma<T>::V;
  floatx16 acc[NP][NQ];
  clear(acc);
  float db[V] = {};
  SA sa;
  SB sb;
  auto fetch = [&](int64_t m) {
    sa.load(g.a, g.lda, g.vec_a, m, hi, p0, g.P);
    sb.load(g.b, g.ldb, g.vec_b, m, hi, q0, g.Q);
  };
  fetch(lo);
  int s = 0;
  for (int64_t m = lo; m < hi; m += ROWS, s ^= 1) {
    char* la = lds + s * STAGE;
    char* lb = la + kGramStage * TP;
    sa.store(la, hi - m);
    sb.store(lb, hi - m);
    if (sums) sa.sum(db);
    __syncthreads();  // (the other buffer's readers are past their previous barrier)
    if (m + ROWS < hi) fetch(m + ROWS);
    auto read = [&](int k) {
      Operands<T, NP, NQ> f;
#pragma unroll
      for (int i = 0; i < NP; ++i) f.x[i] = SA::read(la, k * 2 * Mfma<T>::V, wp + 32 * i);
#pragma unroll
      for (int i = 0; i < NQ; ++i) f.w[i] = SB::read(lb, k * 2 * Mfma<T>::V, wq + 32 * i);
      return f;
    };
    Batched<Operands<T, NP, NQ>, ROWS / (2 * Mfma<T>::V), 1> steps;
    steps.start(read);
    steps.run(read, [&](int, const Operands<T, NP, NQ>& f) {
#pragma unroll
      for (int i = 0; i < NP; ++i)
#pragma unroll
        for (int j = 0; j < NQ; ++j) Mfma<T>::mma(f.x[i], f.w[j], acc[i][j]);
    });
  }
  float* part = g.part + lo / share * g.stride;
  const int lane = int(threadIdx.x) & 31, half = (int(threadIdx.x) >> 5) & 1;
#pragma unroll
  for (int i = 0; i < NP; ++i)
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      const int p = p0 + wp + 32 * i + (k & 3) + 8 * (k >> 2) + 4 * half;
      if (p >= g.P) continue;
      const int64_t row = int64_t(p) * g.Q;
#pragma unroll
      for (int j = 0; j < NQ; ++j) {
        const int q = q0 + wq + 32 * j + lane;
        if (q >= g.Q) continue;
        if (shares > 1)
          part[row + q] = acc[i][j][k];
        else if (g.dw)
          g.dw[row + q] = from_f32<T>(acc[i][j][k]);
      }
    }
  if (!sums) return;
  __syncthreads();
  float* all = reinterpret_cast<float*>(lds);  // [THREADS / SA::PER][TP]
#pragma unroll
  for (int i = 0; i < V; ++i) all[int(threadIdx.x) * V + i] = db[i];
  __syncthreads();
  const int c = int(threadIdx.x);
  if (c >= TP || p0 + c >= g.P) return;
  float v = 0.f;
#pragma unroll
  for (int k = 0; k < THREADS / SA::PER; ++k) v += all[k * TP + c];
  if (shares > 1)
    part[int64_t(g.P) * g.Q + p0 + c] = v;
  else
    g.db[p0 + c] = from_f32<T>(v);
}

// dW (n values) and db (behind it, m) from their partials, V values a lane, four runs of the shares summed apart and
// then in order.
template <typename T, int V>
__global__ __launch_bounds__(kFfnThreads) void linear_reduce(const float* __restrict__ part,
                                                             int64_t stride, int64_t n, int m,
                                                             int shares, T* __restrict__ dw,
                                                             T* __restrict__ db) {
  typedef float vec __attribute__((ext_vector_type(V)));
  __shared__ vec lds[4][64];
  const int lane = int(threadIdx.x) & 63, run = int(threadIdx.x) >> 6;
  const int64_t i = (int64_t(blockIdx.x) * 64 + lane) * V;
  const bool in = i < n ? dw != nullptr : db && i < n + m;  // (V divides n)
  vec v = vec(0.f);
  if (in) {
    const int per = (shares + 3) / 4, end = (run + 1) * per < shares ? (run + 1) * per : shares;
#pragma unroll 8
    for (int s = run * per; s < end; ++s)
      v += *reinterpret_cast<const vec*>(part + int64_t(s) * stride + i);
  }
  lds[run][lane] = v;
  __syncthreads();
  if (run != 0 || !in) return;
  v = ((lds[0][lane] + lds[1][lane]) + lds[2][lane]) + lds[3][lane];
#pragma unroll
  for (int k = 0; k < V; ++k) {
    if (i < n)
      dw[i + k] = from_f32<T>(v[k]);
    else if (i + k < n + m)
      db[i - n + k] = from_f32<T>(v[k]);
  }
}

// ---- host ------------------------------------------------------------------------
struct LinearCall {
  const void *x, *w, *bias, *residual, *dy;
  int64_t ldx, ldr, lddy, rows;
  int C, Co, act;
  void *y, *dx, *dw, *db;
  char* ws;
  hipStream_t stream;
};

template <typename T, typename S, bool ASYNC, bool GRAD>
static int launch_linear(const Rows<T>& x, const Rows<T>& w, const LinearOut<T>& o,
                         hipStream_t s) {
  const int64_t groups = tile_groups<S>(x.n, cdiv(o.columns, S::W));
  SP_CHECK_ARG(groups <= max_groups(S::THREADS), "linear: too many rows for a launch");
  linear_rows<T, S, ASYNC, GRAD><<<unsigned(groups), S::THREADS, 0, s>>>(x, w, o);
  SP_LAUNCHED();
  return SP_OK;
}

template <typename T, bool GRAD>
static int run_linear(const Rows<T>& x, const Rows<T>& w, const LinearOut<T>& o, hipStream_t s) {
  if (!whole(x) || !whole(w)) return launch_linear<T, SmallTile, false, GRAD>(x, w, o, s);
  if (x.K <= 4 * kStagePieces * Mfma<T>::V && fills<QuickTile>(x.n, cdiv(o.columns, QuickTile::W)))
    return launch_linear<T, QuickTile, true, GRAD>(x, w, o, s);
  if (o.columns > 128 && fills<LargeTile>(x.n, cdiv(o.columns, LargeTile::W)))
    return launch_linear<T, LargeTile, true, GRAD>(x, w, o, s);
  if (fills<LongTile>(x.n, cdiv(o.columns, LongTile::W)))
    return launch_linear<T, LongTile, true, GRAD>(x, w, o, s);
  return launch_linear<T, ThinTile, true, GRAD>(x, w, o, s);
}

template <typename T>
static LinearOut<T> linear_out(const void* bias, const void* extra, int64_t lde, void* out,
                               int64_t ldo, int n, int columns, int act) {
  constexpr int V = Mfma<T>::V;
  return LinearOut<T>{static_cast<const T*>(bias), static_cast<const T*>(extra), lde, ldo,
                      static_cast<T*>(out), n, columns, act, bias && aligned(bias),
                      extra && aligned(extra) && lde % V == 0, aligned(out) && ldo % V == 0};
}

template <typename T>
static int linear_forward(const LinearCall& c) {
  const Rows<T> x = operand<T>(c.x, c.ldx, c.rows, c.C), w = operand<T>(c.w, c.C, c.Co, c.C);
  const LinearOut<T> o =
      linear_out<T>(c.bias, c.residual, c.ldr, c.y, c.Co, c.Co, c.Co, c.act);
  if (c.rows > kFewRows) return run_linear<T, false>(x, w, o, c.stream);
  const int l = few_lanes(c.C, Mfma<T>::V);
  const unsigned groups = unsigned(cdiv(c.Co, kFfnThreads >> l));
  if (c.rows == 1)
    linear_few<T, 1><<<groups, kFfnThreads, 0, c.stream>>>(x, w, o, l);
  else if (c.rows == 2)
    linear_few<T, 2><<<groups, kFfnThreads, 0, c.stream>>>(x, w, o, l);
  else
    linear_few<T, 4><<<groups, kFfnThreads, 0, c.stream>>>(x, w, o, l);
  SP_LAUNCHED();
  return SP_OK;
}

// The backward pass's workspace: dz, W transposed, the partials of dW and db.
struct LinearLayout {
  size_t dz, wt, part, total;
  int Cop;
  int64_t shares, stride;  // values of a share's partials
};

static int64_t linear_gram_tiles(int64_t Co, int64_t C, int t) { return cdiv(Co, t) * cdiv(C, t); }
// 256 x 256 where both widths fill it (each operand is read half as often), else 128 x 128.
static int linear_gram_tile(int64_t Co, int64_t C) { return Co > 128 && C > 128 ? 256 : 128; }

static LinearLayout linear_layout(int32_t dtype, int64_t rows, int64_t C, int64_t Co, int act) {
  LinearLayout l{};
  const int V = vec_of(dtype);
  const size_t z = size_of(dtype);
  l.Cop = int(cdiv(Co, V) * V);
  const int t = linear_gram_tile(Co, C);
  const int64_t want = (t == 256 ? 256 : 512) / linear_gram_tiles(Co, C, t), most = cdiv(rows, 256);
  l.shares = want < 1 ? 1 : want < most ? want : most;
  size_t off = 0;
  auto take = [&](size_t bytes) {
    const size_t at = off;
    off = align_up(off + bytes, 256);
    return at;
  };
  if (act != kActNone) l.dz = take(size_t(rows) * l.Cop * z);
  l.wt = take(size_t(C) * l.Cop * z);
  l.stride = cdiv(Co * C + Co, 4) * 4;
  if (l.shares > 1) l.part = take(size_t(l.shares) * l.stride * sizeof(float));
  l.total = off;
  return l;
}

template <typename T>
static int linear_backward(const LinearCall& c, const LinearLayout& l) {
  const Rows<T> x = operand<T>(c.x, c.ldx, c.rows, c.C);
  Rows<T> dz = operand<T>(c.dy, c.lddy, c.rows, c.Co);
  if (c.act != kActNone) {
    T* to = reinterpret_cast<T*>(c.ws + l.dz);
    const LinearOut<T> o = linear_out<T>(c.bias, c.dy, c.lddy, to, l.Cop, c.Co, l.Cop, c.act);
    if (int rc = run_linear<T, true>(x, operand<T>(c.w, c.C, c.Co, c.C), o, c.stream)) return rc;
    dz = operand<T>(to, l.Cop, c.rows, l.Cop);
  }
  if (c.dx) {
    T* wt = reinterpret_cast<T*>(c.ws + l.wt);
    linear_transpose<T><<<dim3(unsigned(cdiv(l.Cop, 32)), unsigned(cdiv(c.C, 32))), kFfnThreads, 0,
                          c.stream>>>(static_cast<const T*>(c.w), c.Co, c.C, wt, l.Cop);
    SP_LAUNCHED();
    const LinearOut<T> o = linear_out<T>(nullptr, nullptr, 0, c.dx, c.C, c.C, c.C, kActNone);
    // (W' has zeros past Co, as a stored dz does)
    if (int rc = run_linear<T, false>(dz, operand<T>(wt, l.Cop, c.C, dz.K), o, c.stream)) return rc;
  }
  if (!c.dw && !c.db) return SP_OK;
  const int t = linear_gram_tile(c.Co, c.C);
  LinearGram<T> g{dz.p, x.p, dz.ld, x.ld, c.Co, c.C, int(cdiv(c.C, t)),
                  int(linear_gram_tiles(c.Co, c.C, t)), dz.vec, x.vec,
                  reinterpret_cast<float*>(c.ws + l.part), l.stride, static_cast<T*>(c.dw),
                  static_cast<T*>(c.db), c.db != nullptr};
  constexpr int stage = gram_rows<T>();
  const int64_t share = cdiv(cdiv(c.rows, l.shares), stage) * stage, shares = cdiv(c.rows, share);
  const unsigned groups = unsigned(cdiv(shares * g.tiles, 8) * 8);
  if (t == 256)
    linear_gram<T, 256, 256><<<groups, 512, 0, c.stream>>>(g, c.rows, share, int(shares));
  else
    linear_gram<T, 128, 128><<<groups, 256, 0, c.stream>>>(g, c.rows, share, int(shares));
  SP_LAUNCHED();
  if (shares == 1) return SP_OK;
  const int64_t n = int64_t(c.Co) * c.C;
  auto reduce = [&](auto kernel, int V) {
    kernel<<<unsigned(cdiv(n + c.Co, 64 * V)), kFfnThreads, 0, c.stream>>>(
        g.part, l.stride, n, c.Co, int(shares), g.dw, g.db);
  };
  if (n % 4 == 0)
    reduce(linear_reduce<T, 4>, 4);
  else
    reduce(linear_reduce<T, 1>, 1);
  SP_LAUNCHED();
  return SP_OK;
}

static int check_linear(const char* what, int32_t dtype, int64_t rows, int64_t C, int64_t Co,
                        int32_t act) {
  SP_CHECK_ARG(dtype == SP_F16 || dtype == SP_BF16 || dtype == SP_F32,
               "%s: dtype %d not supported (f16/bf16/f32)", what, dtype);
  SP_CHECK_ARG(rows >= 0 && C >= 1 && Co >= 1 && C < 65536 && Co < 65536,
               "%s: bad sizes rows=%lld C=%lld Co=%lld", what, (long long)rows, (long long)C,
               (long long)Co);
  SP_CHECK_ARG(rows < (int64_t(1) << 31), "%s: 2^31 rows or more", what);
  SP_CHECK_ARG(act >= kActSilu && act <= kActNone, "%s: unknown activation %d", what, act);
  return SP_OK;
}

template <typename F>
static int linear_types(int32_t dtype, F&& f) {
  return dtype == SP_F16 ? f(_Float16()) : dtype == SP_BF16 ? f(__bf16()) : f(float());
}

}  // namespace sp

using namespace sp;

extern "C" int sp_linear(const void* x, int64_t ldx, int32_t dtype, int64_t rows, int64_t C,
                         const void* weight, int64_t Co, const void* bias, int32_t act,
                         const void* residual, int64_t ldr, void* y, void* stream) {
  if (int rc = check_linear("linear", dtype, rows, C, Co, act)) return rc;
  if (rows == 0) return SP_OK;
  SP_CHECK_ARG(x && weight && y, "linear: null pointer");
  SP_CHECK_ARG(ldx >= C && (!residual || ldr >= Co), "linear: rows overlap");
  LinearCall c{};
  c.x = x, c.w = weight, c.bias = bias, c.residual = residual;
  c.ldx = ldx, c.ldr = ldr, c.rows = rows;
  c.C = int(C), c.Co = int(Co), c.act = act;
  c.y = y, c.stream = as_stream(stream);
  return linear_types(dtype, [&](auto t) { return linear_forward<decltype(t)>(c); });
}

extern "C" size_t sp_linear_bwd_workspace(int32_t dtype, int64_t rows, int64_t C, int64_t Co,
                                          int32_t act) {
  if (check_linear("linear_bwd", dtype, rows, C, Co, act) != SP_OK || rows == 0) return 0;
  return linear_layout(dtype, rows, C, Co, act).total;
}

extern "C" int sp_linear_bwd(const void* dy, int64_t lddy, const void* x, int64_t ldx, int32_t dtype,
                             int64_t rows, int64_t C, const void* weight, int64_t Co,
                             const void* bias, int32_t act, void* dx, void* dweight, void* dbias,
                             void* ws, size_t ws_bytes, void* stream) {
  if (int rc = check_linear("linear_bwd", dtype, rows, C, Co, act)) return rc;
  if (rows == 0) return SP_OK;
  SP_CHECK_ARG(dy && x && weight && ws, "linear_bwd: null pointer");
  SP_CHECK_ARG(ldx >= C && lddy >= Co, "linear_bwd: rows overlap");
  SP_CHECK_ARG(aligned(ws), "linear_bwd: the workspace must be 16-byte aligned");
  const LinearLayout l = linear_layout(dtype, rows, C, Co, act);
  if (ws_bytes < l.total)
    return set_error(SP_ERR_WORKSPACE, "linear_bwd: workspace of %zu bytes, needs %zu", ws_bytes,
                     l.total);
  LinearCall c{};
  c.dy = dy, c.x = x, c.w = weight, c.bias = bias;
  c.ldx = ldx, c.lddy = lddy, c.rows = rows;
  c.C = int(C), c.Co = int(Co), c.act = act;
  c.dx = dx, c.dw = dweight, c.db = dbias;
  c.ws = static_cast<char*>(ws), c.stream = as_stream(stream);
  return linear_types(dtype, [&](auto t) { return linear_backward<decltype(t)>(c, l); });
}
