// The gated feed-forward block's backward pass for 16-bit rows of up to 128 channels, and of up to 192 the
// gradient of the hidden rows and of x in one kernel.  Nothing of the hidden width is in memory: both
// kernels form g, u and dh again from x, dy and the weights.
//
//   dh = dy Wd, dg = dh * u * act'(g), du = dh * act(g), h = act(g) * u
//   ffn_fused_dx:      dx = dg Wg + du Wu                       (a wave: 32 rows, all hidden units)
//   ffn_fused_weights: dWg = dg' x, dWu = du' x, dWd' = h' dy   (a wave: 32 hidden units, many rows)
//
// The first goes through the chunks of the weights like the forward pass (sp_ffn_fused.hip): all is transposed,
// values go from accumulators into operands within the lane.  Wd' and Wg', Wu' are the same chunks, read
// transposed (ds_read_b64_tr_b16: sixteen lanes take a 4 x 16 block, 8 bytes each, and get a
// column of it each).
//
// The second holds the weights of 32 hidden units as operands and their three gradients as accumulators in
// registers.  Rows pass through LDS 32 at a time; g, u and dh come out with a hidden unit a lane and
// 16 rows of the tile in its registers, which is an operand of the products over rows; the other one is
// the tile read transposed.
#include "sp_ffn_fused.h"

namespace sp {

typedef short short4v __attribute__((ext_vector_type(4)));

// Two transposed reads as one operand: four rows from `a` and four from `b` on, the lane's own
// addresses.
template <typename T>
__device__ __forceinline__ typename Mfma<T>::frag read_transposed(const char* a, const char* b) {
  union {
    short4v q[2];
    typename Mfma<T>::frag f;
  } u;
  u.q[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
      (__attribute__((address_space(3))) short4v*)(a));
  u.q[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
      (__attribute__((address_space(3))) short4v*)(b));
  return u.f;
}

// Operand whose rows are the columns of a chunk matrix: 32 columns from piece c0 on in the order
// unit_of, reduction index 16 k .. 16 k + 15 of the matrix's rows (which lie in that order
// too).  `at(row, piece)` is where a piece lies.
template <typename T, typename At>
__device__ __forceinline__ typename Mfma<T>::frag columns_of(At&& at, int k, int c0) {
  const int lane = int(threadIdx.x) & 63, half = lane >> 5, t = lane & 15;
  // lanes of a column group get columns unit_of(16 (lane >> 4 & 1)) + ..: groups of four in the
  // order 0, 2, 1, 3
  const int piece = c0 + 2 * ((lane >> 4) & 1) + (t & 1), off = ((t >> 1) & 1) * 8;
  const int row = 16 * k + 4 * half + (t >> 2);
  return read_transposed<T>(at(row, piece) + off, at(row + 8, piece) + off);
}

// A row's values kept in 8 bits (codes null: not kept so).
struct Kept {
  const int8_t* codes;
  const float* scales;
  int groups, vec;
};

template <typename T>
__device__ __forceinline__ typename Mfma<T>::frag kept_piece(const Kept& q, int64_t r, int c,
                                                             int n) {
  typename Mfma<T>::frag f = {};
  if (c >= n) return f;
  const int8_t* p = q.codes + r * n + c;
  const float step = q.scales[r * q.groups + (c >> 7)];
  if (q.vec) {
    const int2 w = *reinterpret_cast<const int2*>(p);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      f[i] = T(float(int8_t((i < 4 ? w.x : w.y) >> (8 * (i & 3)))) * step);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i < n) f[i] = T(float(p[i]) * step);
  }
  return f;
}

template <typename T>
struct GradArgs {
  Rows<T> x, dy;
  Kept kept;  // instead of x.p
  Weights<T> w;
  T *dx, *hid;   // hid [rows][3 Fp]: dg, du and h for a kernel that follows
  int vec_dx, Fp;
  float *part0, *part1;  // the weight gradients' partials, [shares][2 Fp][C] and [shares][F][Co]
  int64_t share;
};

template <typename T>
__device__ __forceinline__ typename Mfma<T>::frag x_piece(const GradArgs<T>& a, int64_t r, int c) {
  if (r >= a.x.n) return typename Mfma<T>::frag{};
  return a.kept.codes ? kept_piece<T>(a.kept, r, c, a.x.K)
                      : row_piece<T>(a.x.p + r * a.x.ld, c, a.x.K, a.x.vec);
}

// dg and du are rounded to the rows' type as operands of the last products.  240k x 64 -> 256 fp16 64 us: five
// products, 39 GFLOP, 615 TFLOP/s; bound as the forward pass, by the gate's instructions beside the
// MFMAs.  HIDDEN: writes dg, du and h as well, for rows whose weight gradients do not fit in registers.
template <typename T, int ACT, int CP, bool HIDDEN, int MINW>
__global__ __launch_bounds__(kFfnThreads, MINW) void ffn_fused_dx(GradArgs<T> a) {
  using frag = typename Mfma<T>::frag;
  using C = Chunk<CP>;
  __shared__ __attribute__((aligned(16))) char lds[2 * C::BYTES];
  const int wave = int(threadIdx.x) >> 6, lane = int(threadIdx.x) & 31;
  const int half = (int(threadIdx.x) >> 5) & 1;
  const int64_t r = (int64_t(blockIdx.x) * 4 + wave) * kFusedRows + lane;
  Chunks<T, CP> chunks(a.w, lds);
  frag x[CP / 16], dy[CP / 16];
#pragma unroll
  for (int k = 0; k < CP / 16; ++k) x[k] = x_piece(a, r, k * 16 + half * 8);
  load_rows<T, CP>(a.dy, r, dy);
  floatx16 dx[CP / 32];
  clear_rows(dx);
  for (int f0 = 0; f0 < a.w.F; f0 += 32) {
    const char* chunk = chunks.next();
    floatx16 g, u, dh;
    fused_up<T, CP>(chunk, x, g, u);
#pragma unroll
    for (int i = 0; i < 16; ++i) dh[i] = 0.f;
    auto down = [&](int k) {
      return columns_of<T>([&](int m, int c) { return C::down(chunk, m, c); }, k, 0);
    };
    Batched<frag, CP / 16, 4> wd;
    wd.start(down);
    wd.run(down, [&](int k, const frag& f) { Mfma<T>::mma(f, dy[k], dh); });
    auto up = [&](int i) {  // Wg's and Wu's 32 channels i / 2, 16 hidden units i % 2
      return FragPair<T>{
          columns_of<T>([&](int m, int c) { return C::up(chunk, 0, m, c); }, i & 1, 4 * (i >> 1)),
          columns_of<T>([&](int m, int c) { return C::up(chunk, 1, m, c); }, i & 1, 4 * (i >> 1))};
    };
    Batched<FragPair<T>, CP / 16, 2> wgu;
    wgu.start(up);
    frag dg[2], du[2], h[2];
    gate16<true, ACT>(g, [&](int i, float value, float slope) {
      dg[i >> 3][i & 7] = T(dh[i] * u[i] * slope);
      du[i >> 3][i & 7] = T(dh[i] * value);
      if (HIDDEN) h[i >> 3][i & 7] = T(value * u[i]);
    });
    if (f0 + 32 > a.w.F) {  // (h's are not read)
      end_units(dg, f0, a.w.F);
      end_units(du, f0, a.w.F);
    }
    wgu.run(up, [&](int i, const FragPair<T>& f) {
      Mfma<T>::mma(f.a, dg[i & 1], dx[i >> 1]);
      Mfma<T>::mma(f.b, du[i & 1], dx[i >> 1]);
    });
    if (HIDDEN && a.hid && r < a.x.n) {
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const int f = f0 + 16 * s + 8 * half;
        if (f < a.Fp) {
          T* to = a.hid + r * (3 * int64_t(a.Fp)) + f;
          *reinterpret_cast<frag*>(to) = dg[s];
          *reinterpret_cast<frag*>(to + a.Fp) = du[s];
          *reinterpret_cast<frag*>(to + 2 * a.Fp) = h[s];
        }
      }
    }
  }
  if (!a.dx || r >= a.x.n) return;
#pragma unroll
  for (int t = 0; t < CP / 32; ++t)
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int c = t * 32 + 16 * s + 8 * half;
      if (c >= a.x.K) continue;
      frag o;
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] = T(dx[t][8 * s + i]);
      T* to = a.dx + r * a.x.K + c;
      if (a.vec_dx) {
        *reinterpret_cast<frag*>(to) = o;
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (c + i < a.x.K) to[i] = o[i];
      }
    }
}

// A tile of ROWS rows of x and of dy on its way to LDS, [ROWS][CP] each.
template <typename T, int CP, int THREADS, int ROWS>
struct RowTile {
  using frag = typename Mfma<T>::frag;
  static constexpr int UP = CP / 8, PIECES = ROWS * UP, N = (PIECES + THREADS - 1) / THREADS;
  static constexpr int BYTES = PIECES * 16;
  frag x[N], dy[N];

  __device__ __forceinline__ void load(const GradArgs<T>& a, int64_t r0, int64_t hi) {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int i = j * THREADS + int(threadIdx.x), row = i / UP, c = (i - row * UP) * 8;
      const int64_t r = r0 + row;
      x[j] = frag{};
      dy[j] = frag{};
      if (i < PIECES && r < hi) {
        x[j] = x_piece(a, r, c);
        dy[j] = row_piece<T>(a.dy.p + r * a.dy.ld, c, a.dy.K, a.dy.vec);
      }
    }
  }
  __device__ __forceinline__ void store(char* lds) const {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int i = j * THREADS + int(threadIdx.x), row = i / UP;
      if (PIECES % THREADS != 0 && i >= PIECES) break;
      char* to = lds + (row * UP + swizzled<UP>(row, i - row * UP)) * 16;
      *reinterpret_cast<frag*>(to) = x[j];
      *reinterpret_cast<frag*>(to + BYTES) = dy[j];
    }
  }
};

// A workgroup: 128 hidden units (four waves of 32) and a share of the rows, HALVES tiles of 32 rows
// between barriers, one for each four waves.  240k x 64 -> 256 fp16 87 us: six products, 47 GFLOP, 543
// TFLOP/s.  Weights and gradients fill the registers of two waves a SIMD, so that little runs beside a
// wave's gate and its waits at the barrier; one wave a SIMD with two tiles was slower.  Storing the
// hidden rows and multiplying them instead moves 1.5 KB a row.
template <typename T, int ACT, int CP, int HALVES>
__global__ __launch_bounds__(kFfnThreads * HALVES) void ffn_fused_weights(GradArgs<T> a) {
  using frag = typename Mfma<T>::frag;
  constexpr int THREADS = kFfnThreads * HALVES, ROWS = kFusedRows * HALVES, UP = CP / 8;
  constexpr int K = CP / 16, TILES = CP / 32;
  using Tile = RowTile<T, CP, THREADS, ROWS>;
  constexpr int JOIN = HALVES > 1 ? 4 * TILES * 4096 : 0;  // a matrix of four waves
  __shared__ __attribute__((aligned(16))) char lds[4 * Tile::BYTES > JOIN ? 4 * Tile::BYTES : JOIN];
  const int wave = int(threadIdx.x) >> 6, lane = int(threadIdx.x) & 31;
  const int half = (int(threadIdx.x) >> 5) & 1;
  const int f = int(blockIdx.x) * 128 + (wave & 3) * 32 + lane;
  const int64_t lo = int64_t(blockIdx.y) * a.share;
  const int64_t hi = lo + a.share < a.x.n ? lo + a.share : a.x.n;
  Tile tile;
  tile.load(a, lo, hi);
  frag wg[K], wu[K], wd[K];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = 16 * k + 8 * half;
    wg[k] = wu[k] = wd[k] = frag{};
    if (f < a.w.Fw && c < a.w.C) {
      wg[k] = *reinterpret_cast<const frag*>(a.w.g + int64_t(f) * a.w.ldu + c);
      wu[k] = *reinterpret_cast<const frag*>(a.w.u + int64_t(f) * a.w.ldu + c);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (f < a.w.Fw && c + i < a.w.Cow) wd[k][i] = a.w.d[int64_t(c + i) * a.w.ldd + f];
  }
  floatx16 dwg[TILES], dwu[TILES], dwd[TILES];
  clear_rows(dwg);
  clear_rows(dwu);
  clear_rows(dwd);
  int buf = 0;
  for (int64_t m = lo; m < hi; m += ROWS, buf ^= 1) {
    char* at = lds + buf * (2 * Tile::BYTES);
    tile.store(at);
    __syncthreads();  // (the other buffer's readers are past their previous barrier)
    if (m + ROWS < hi) tile.load(a, m + ROWS, hi);
    const char* xs = at + (wave >> 2) * (kFusedRows * UP * 16);
    const char* ds = xs + Tile::BYTES;
    floatx16 g, u, dh;
#pragma unroll
    for (int i = 0; i < 16; ++i) g[i] = u[i] = dh[i] = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int piece = (lane * UP + swizzled<UP>(lane, 2 * k + half)) * 16;
      const frag fx = *reinterpret_cast<const frag*>(xs + piece);
      const frag fd = *reinterpret_cast<const frag*>(ds + piece);
      Mfma<T>::mma(fx, wg[k], g);
      Mfma<T>::mma(fx, wu[k], u);
      Mfma<T>::mma(fd, wd[k], dh);
    }
    // register 8 s + j of lane half b holds row 16 s + 8 (j >> 2) + 4 b + (j & 3) of the tile
    frag dg[2], du[2], h[2];
    gate16<true, ACT>(g, [&](int i, float value, float slope) {
      dg[i >> 3][i & 7] = T(dh[i] * u[i] * slope);
      du[i >> 3][i & 7] = T(dh[i] * value);
      h[i >> 3][i & 7] = T(value * u[i]);
    });
    if (m + ROWS > hi) {
      // rows past the end are zeros, of which an infinity in a weight makes NaN
      const int left = int(hi - m) - (wave >> 2) * kFusedRows;
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (16 * (i >> 3) + 8 * ((i >> 2) & 1) + 4 * half + (i & 3) >= left)
          dg[i >> 3][i & 7] = du[i >> 3][i & 7] = h[i >> 3][i & 7] = 0;
    }
#pragma unroll
    for (int t = 0; t < TILES; ++t)
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        // columns 32 t .. of those rows
        const int l = int(threadIdx.x) & 15;
        const int col = 4 * t + 2 * ((int(threadIdx.x) >> 4) & 1) + ((l >> 1) & 1);
        const int row = 16 * s + 4 * half + (l >> 2);
        const int p0 = (row * UP + swizzled<UP>(row, col)) * 16 + (l & 1) * 8;
        const int p1 = ((row + 8) * UP + swizzled<UP>(row + 8, col)) * 16 + (l & 1) * 8;
        const frag fx = read_transposed<T>(xs + p0, xs + p1);
        const frag fd = read_transposed<T>(ds + p0, ds + p1);
        Mfma<T>::mma(dg[s], fx, dwg[t]);
        Mfma<T>::mma(du[s], fx, dwu[t]);
        Mfma<T>::mma(h[s], fd, dwd[t]);
      }
  }
  // the second four waves' sums through LDS to the first's
  auto join = [&](floatx16(&d)[TILES]) {
    if constexpr (HALVES > 1) {
      float* at = reinterpret_cast<float*>(lds) + (wave & 3) * (TILES * 1024) +
                  (int(threadIdx.x) & 63);
      __syncthreads();
      if (wave >= 4)
#pragma unroll
        for (int t = 0; t < TILES; ++t)
#pragma unroll
          for (int i = 0; i < 16; ++i) at[(t * 16 + i) * 64] = d[t][i];
      __syncthreads();
      if (wave < 4)
#pragma unroll
        for (int t = 0; t < TILES; ++t)
#pragma unroll
          for (int i = 0; i < 16; ++i) d[t][i] += at[(t * 16 + i) * 64];
    }
  };
  join(dwg);
  join(dwu);
  join(dwd);
  if (wave >= 4) return;
  const int f1 = int(blockIdx.x) * 128 + (wave & 3) * 32;
  float* p0 = a.part0 + int64_t(blockIdx.y) * 2 * a.Fp * a.x.K;
  float* p1 = a.part1 + int64_t(blockIdx.y) * a.w.F * a.w.Co;
#pragma unroll
  for (int t = 0; t < TILES; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int fi = f1 + (i & 3) + 8 * (i >> 2) + 4 * half, c = t * 32 + lane;
      if (fi >= a.w.F) continue;
      if (c < a.x.K) {
        p0[int64_t(fi) * a.x.K + c] = dwg[t][i];
        p0[int64_t(a.Fp + fi) * a.x.K + c] = dwu[t][i];
      }
      if (c < a.w.Co) p1[int64_t(fi) * a.w.Co + c] = dwd[t][i];
    }
}

// ---- host ------------------------------------------------------------------------
static int64_t widest(int64_t C, int64_t Co) { return C > Co ? C : Co; }

// Rows of a tile of the weight gradients' kernel.
static int tile_rows(int64_t C, int64_t Co) { return widest(C, Co) <= 64 ? 64 : 32; }

// Measured, these kernels against the tiled ones (us, fp16): 64 -> 256 38 / 31 at 1 000 rows, 42 / 43 at 16 000,
// 50 / 57 at 32 000; 128 -> 344 54 / 37, 67 / 64, 79 / 88; 192 -> 512 68 / 49, 90 / 87, 112 / 133; 32 -> 128
// 24 / 27 at 1 000; 256 -> 688 bf16 at 75 000 rows 477 / 449.
bool fused_backward_takes(int32_t dtype, int64_t rows, int64_t C, int64_t Co) {
  const int64_t n = widest(C, Co);
  return dtype != SP_F32 && n <= kFusedWidth && (n <= 32 || rows >= 16384);
}

// Shares of the rows: one workgroup a CU, each with eight tiles at least.
int64_t fused_weights_shares(int64_t rows, int64_t C, int64_t F, int64_t Co) {
  const int64_t want = cdiv(256, cdiv(F, 128)), most = cdiv(rows, 8 * tile_rows(C, Co));
  return want < most ? want : most;
}

template <typename T, int CP, bool HIDDEN, int MINW>
static int launch_dx(const GradArgs<T>& a, int act, hipStream_t s) {
  const int64_t blocks = cdiv(a.x.n, 4 * kFusedRows);
  SP_CHECK_ARG(blocks <= kMaxGridX, "gated_ffn_bwd: too many rows");
  using Kern = void (*)(GradArgs<T>);
  const Kern kern = act == kActSilu   ? Kern(ffn_fused_dx<T, kActSilu, CP, HIDDEN, MINW>)
                    : act == kActGelu ? Kern(ffn_fused_dx<T, kActGelu, CP, HIDDEN, MINW>)
                                      : Kern(ffn_fused_dx<T, kActRelu, CP, HIDDEN, MINW>);
  kern<<<unsigned(blocks), kFfnThreads, 0, s>>>(a);
  SP_LAUNCHED();
  return SP_OK;
}

template <typename T, int CP, int HALVES>
static int launch_weights(const GradArgs<T>& a, int act, hipStream_t s) {
  using Kern = void (*)(GradArgs<T>);
  const Kern kern = act == kActSilu   ? Kern(ffn_fused_weights<T, kActSilu, CP, HALVES>)
                    : act == kActGelu ? Kern(ffn_fused_weights<T, kActGelu, CP, HALVES>)
                                      : Kern(ffn_fused_weights<T, kActRelu, CP, HALVES>);
  const dim3 grid(unsigned(cdiv(a.w.F, 128)), unsigned(cdiv(a.x.n, a.share)));
  kern<<<grid, kFfnThreads * HALVES, 0, s>>>(a);
  SP_LAUNCHED();
  return SP_OK;
}

template <typename T>
static int run_grad(const FfnCall& c, const FusedGrad& o, int64_t* shares) {
  GradArgs<T> a{};
  a.x = operand<T>(c.x, c.ldx, c.rows, c.C);
  a.dy = operand<T>(c.dy, c.lddy, c.rows, c.Co);
  if (c.codes) {
    a.kept = Kept{c.codes, c.scales, int(cdiv(c.C, 128)),
                  c.C % 8 == 0 && (reinterpret_cast<uintptr_t>(c.codes) & 7) == 0};
  }
  a.dx = static_cast<T*>(c.dx);
  a.hid = static_cast<T*>(o.hid);
  a.vec_dx = aligned(c.dx) && c.C % 8 == 0;
  a.Fp = o.Fp;
  a.part0 = o.part0, a.part1 = o.part1;
  if (int rc = fused_weights(c, static_cast<T*>(o.weights), a.w)) return rc;
  const int64_t n = widest(c.C, c.Co);
  if (a.dx || a.hid) {
    int rc;
    if (n > kFusedGramWidth)
      rc = n <= 160 ? launch_dx<T, 160, true, 1>(a, c.act, c.stream)
                    : launch_dx<T, 192, true, 1>(a, c.act, c.stream);
    else
      rc = n <= 32   ? launch_dx<T, 32, false, 4>(a, c.act, c.stream)
           : n <= 64 ? launch_dx<T, 64, false, 3>(a, c.act, c.stream)
           : n <= 96 ? launch_dx<T, 96, false, 2>(a, c.act, c.stream)
                     : launch_dx<T, 128, false, 2>(a, c.act, c.stream);
    if (rc) return rc;
  }
  if (!o.part0) return SP_OK;
  const int tile = tile_rows(c.C, c.Co);
  a.share = cdiv(cdiv(c.rows, o.shares), tile) * tile;
  *shares = cdiv(c.rows, a.share);
  return n <= 32   ? launch_weights<T, 32, 2>(a, c.act, c.stream)
         : n <= 64 ? launch_weights<T, 64, 2>(a, c.act, c.stream)
         : n <= 96 ? launch_weights<T, 96, 1>(a, c.act, c.stream)
                   : launch_weights<T, 128, 1>(a, c.act, c.stream);
}

int fused_backward(int32_t dtype, const FfnCall& a, const FusedGrad& o, int64_t* shares) {
  return dtype == SP_F16 ? run_grad<_Float16>(a, o, shares) : run_grad<__bf16>(a, o, shares);
}

}  // namespace sp
