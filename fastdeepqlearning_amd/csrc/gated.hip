// Gated linear unit (fdql_gated*):  y = f(x Wg^T + bg) * (x Wu^T + bu), forward and backward.
//
// Forward: one matrix product against both weights, with the activation, the product and the biases in its epilogue - a wave's accumulators
// hold the gate and the up column of the same 32 outputs, so both meet in one lane and neither is stored (training keeps them in
// float32 for the backward pass: rounded to 16 bits they would cost the gradients a bit more than their own rounding does).
// Backward: an elementwise pass forms dg = dy u f'(g), du = dy f(g) (rounded to the operand type the matrix instructions take) and
// their column sums; then dx = dg Wg + du Wu is one product over 2 F, and dWg = dg^T x, dWu = du^T x are one launch with the rows
// split over workgroups where the weights alone leave the card idle (float32 slabs, added in order).
//
// Tiles: BM x 128 per workgroup of four waves, K in slices of 128 bytes; LDS rows are one slice long, 16-byte chunk c of row n lies at
// c ^ swz(n), and both operands are kept contraction-contiguous: an operand that lies the other way in memory is transposed in
// registers on its way to LDS (16-byte rows of k against 4 columns: byte permutes for 16-bit types, renaming for float).  So one inner loop
// serves all three products: v_mfma_f32_32x32x16 (bf16, fp16) or four v_mfma_f32_32x32x2 (float) per pair of 16-byte fragments; which k
// a lane half holds is the same on both sides and does not matter.  Slices are double-buffered, the next one in flight in registers.
//
// Few rows (M <= 32) are bound by the weights' bytes and by latency: k_gated_rows gives 16 outputs to a workgroup, splits K over its
// four waves and reads fragments straight from memory.
#include "seq.h"

#include <algorithm>

namespace fdql {
namespace {

typedef float v16f __attribute__((ext_vector_type(16)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef int v4i __attribute__((ext_vector_type(4)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));

constexpr int BN = 128;

enum Mode { FWD, DX, DW };

struct Args {
  fdql_gated_t p;
  int Fp;                          // row length of d (F rounded up to 8)
  void *d;                         // [2][M][Fp] dg, du in the operand type, zeros behind column F
  float *colsum;                   // [row blocks][2][F]
  float *slab;                     // [ksplit][2][F][D] when ksplit > 1
  int ksplit, kper;                // DW: slices of the rows and their length (a multiple of the K slice)
  int tiles_m, tiles_n;
};

__device__ __forceinline__ int swz(int n) { return (n ^ (n >> 3)) & 7; }

template <typename T> struct Mma;
template <> struct Mma<bf16_t> {
  static __device__ __forceinline__ void mma32(v16f &c, v4i a, v4i b) {
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ void mma16(v4f &c, v4i a, v4i b) {
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
  }
};
template <> struct Mma<f16_t> {
  static __device__ __forceinline__ void mma32(v16f &c, v4i a, v4i b) {
    c = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ void mma16(v4f &c, v4i a, v4i b) {
    c = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
  }
};
template <> struct Mma<float> {
  static __device__ __forceinline__ void mma32(v16f &c, v4i a, v4i b) {
    const v4f fa = __builtin_bit_cast(v4f, a), fb = __builtin_bit_cast(v4f, b);
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(fa[i], fb[i], c, 0, 0, 0);
  }
  static __device__ __forceinline__ void mma16(v4f &c, v4i a, v4i b) {
    const v4f fa = __builtin_bit_cast(v4f, a), fb = __builtin_bit_cast(v4f, b);
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(fa[i], fb[i], c, 0, 0, 0);
  }
};

// f(g) and f'(g)
__device__ __forceinline__ float act_f(int act, float g) {
  if (act == FDQL_ACT_GELU) return 0.5f * g * erfcf(-0.70710678118654752f * g);
  const float s = sigmoid_f(g);
  return act == FDQL_ACT_SILU ? g * s : s;
}
__device__ __forceinline__ void act_df(int act, float g, float &f, float &df) {
  if (act == FDQL_ACT_GELU) {
    const float cdf = 0.5f * erfcf(-0.70710678118654752f * g);
    f = g * cdf;
    df = fmaf(g * 0.39894228040143268f, exp_acc(-0.5f * g * g), cdf);
  } else {
    const float s = sigmoid_f(g), r = s * (1.f - s);
    f = act == FDQL_ACT_SILU ? g * s : s;
    df = act == FDQL_ACT_SILU ? fmaf(g, r, s) : r;
  }
}

// 16 bytes of a contraction-contiguous row: elements [k, k + E) of `row`, zeros at and behind K.
template <typename T, bool VEC>
__device__ __forceinline__ v4i row_chunk(const T *row, int64_t k, int64_t K) {
  constexpr int E = 16 / sizeof(T);
  if constexpr (VEC) {
    v4i z = {0, 0, 0, 0};
    return k < K ? *reinterpret_cast<const v4i *>(row + k) : z;
  } else {
    typedef T vec __attribute__((ext_vector_type(E)));
    vec v;
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = k + e < K ? row[k + e] : T(0.f);
    return __builtin_bit_cast(v4i, v);
  }
}

// A K slice of `rows` LDS rows on its way: NCH 16-byte chunks per thread.
template <int NCH>
struct Flight { v4i c[NCH]; };

// rows_ptr(n) -> first element of operand row n or nullptr (zeros)
template <typename T, bool VEC, int NCH, typename F>
__device__ __forceinline__ void fetch_rows(Flight<NCH> &f, F row_ptr, int64_t k0, int64_t K) {
  constexpr int E = 16 / sizeof(T);
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    const int n = (threadIdx.x >> 3) + 32 * i, c = threadIdx.x & 7;
    const T *row = row_ptr(n);
    v4i z = {0, 0, 0, 0};
    f.c[i] = row ? row_chunk<T, VEC>(row, k0 + c * E, K) : z;
  }
}
template <int NCH>
__device__ __forceinline__ void put_rows(const Flight<NCH> &f, char *lds) {
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    const int n = (threadIdx.x >> 3) + 32 * i, c = threadIdx.x & 7;
    *reinterpret_cast<v4i *>(lds + n * 128 + ((c ^ swz(n)) << 4)) = f.c[i];
  }
}

// The other orientation: memory is [k][column] with row length ld; thread = 4 columns x E rows of k, transposed in registers to four chunks.
template <typename T, bool VEC>
__device__ __forceinline__ void fetch_cols(Flight<4> &f, const T *base, int64_t ld, int64_t k0, int64_t K, int64_t col0, int64_t cols) {
  constexpr int E = 16 / sizeof(T);
  typedef T vec4 __attribute__((ext_vector_type(4)));
  const int64_t col = col0 + (threadIdx.x & 31) * 4;
  const int64_t k = k0 + (threadIdx.x >> 5) * E;
  vec4 r[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
#pragma unroll
    for (int j = 0; j < 4; ++j) r[e][j] = T(0.f);
    if (k + e < K) {
      if constexpr (VEC) {
        if (col < cols) r[e] = *reinterpret_cast<const vec4 *>(base + (k + e) * ld + col);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (col + j < cols) r[e][j] = base[(k + e) * ld + col + j];
      }
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    typedef T vec __attribute__((ext_vector_type(E)));
    vec v;
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = r[e][j];
    f.c[j] = __builtin_bit_cast(v4i, v);
  }
}
__device__ __forceinline__ void put_cols(const Flight<4> &f, char *lds) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int n = (threadIdx.x & 31) * 4 + j, c = threadIdx.x >> 5;
    *reinterpret_cast<v4i *>(lds + n * 128 + ((c ^ swz(n)) << 4)) = f.c[j];
  }
}

// Workgroups are dealt to the eight XCDs in turn: give each XCD a contiguous run of tiles, row tiles innermost in groups of 8, so that the
// tiles that share operand rows meet in one L2.
__device__ __forceinline__ void tile_of(int bid, int tiles_m, int tiles_n, int &tm, int &tn) {
  const int n = tiles_m * tiles_n, q = n / 8, rem = n % 8, x = bid % 8;
  const int t = x * q + min(x, rem) + bid / 8;
  const int group = 8 * tiles_n, g0 = t / group * 8, in = t % group, h = min(8, tiles_m - g0);
  tm = g0 + in % h;
  tn = in / h;
}

template <typename T, int MODE, int BM, bool VEC>
__global__ __launch_bounds__(256, 2) void k_gated_tile(Args a) {
  constexpr int BK = 128 / sizeof(T), MT = BM / 64, NT = 2, NCA = BM / 32;
  __shared__ __align__(16) char lds[2][(BM + BN) * 128];
  const fdql_gated_t &p = a.p;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave >> 1, wn = wave & 1;
  int tm, tn;
  tile_of(blockIdx.x, a.tiles_m, a.tiles_n, tm, tn);
  const int64_t M = p.M, D = p.D, F = p.F, m0 = (int64_t)tm * BM;
  const int which = MODE == DW ? blockIdx.y : 0, ks = MODE == DW ? blockIdx.z : 0;
  const T *x = reinterpret_cast<const T *>(p.x), *wg = reinterpret_cast<const T *>(p.w_gate), *wu = reinterpret_cast<const T *>(p.w_up);
  const T *dd = reinterpret_cast<const T *>(a.d);
  const int64_t f0 = (int64_t)tn * (BN / 2), n0 = (int64_t)tn * BN;

  int64_t kbeg = 0, kend;                          // contraction range in elements; DX runs over both halves one after the other
  int steps;
  if (MODE == FWD) kend = D, steps = (int)((D + BK - 1) / BK);
  else if (MODE == DX) kend = F, steps = 2 * (int)((F + BK - 1) / BK);
  else kbeg = (int64_t)ks * a.kper, kend = min(M, kbeg + a.kper), steps = kend > kbeg ? (int)((kend - kbeg + BK - 1) / BK) : 0;
  const int half = steps / 2;

  Flight<NCA> fa;
  Flight<4> fb;
  const auto fetch = [&](int step) {
    if constexpr (MODE == FWD) {
      const int64_t k0 = (int64_t)step * BK;
      fetch_rows<T, VEC>(fa, [&](int n) { return m0 + n < M ? x + (m0 + n) * p.x_sr : (const T *)nullptr; }, k0, D);
      fetch_rows<T, VEC>(fb, [&](int n) {          // 32 gate rows, 32 up rows per wave column
        const int64_t f = f0 + (n >> 6) * 32 + (n & 31);
        return f < F ? (n & 32 ? wu : wg) + f * D : (const T *)nullptr;
      }, k0, D);
    } else if constexpr (MODE == DX) {
      const int up = step >= half;
      const int64_t k0 = (int64_t)(step - up * half) * BK;
      const T *src = dd + up * M * a.Fp;
      fetch_rows<T, true>(fa, [&](int n) { return m0 + n < M ? src + (m0 + n) * a.Fp : (const T *)nullptr; }, k0, a.Fp);
      fetch_cols<T, VEC>(fb, up ? wu : wg, D, k0, F, n0, D);
    } else {
      const int64_t k0 = kbeg + (int64_t)step * BK;
      fetch_cols<T, true>(reinterpret_cast<Flight<4> &>(fa), dd + which * M * a.Fp, a.Fp, k0, kend, m0, a.Fp);
      fetch_cols<T, VEC>(fb, x, p.x_sr, k0, kend, n0, D);
    }
  };
  const auto put = [&](int buf) {
    if constexpr (MODE == DW) put_cols(reinterpret_cast<const Flight<4> &>(fa), lds[buf]);
    else put_rows(fa, lds[buf]);
    if constexpr (MODE == FWD) put_rows(fb, lds[buf] + BM * 128);
    else put_cols(fb, lds[buf] + BM * 128);
  };

  v16f acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;

  if (steps > 0) {
    fetch(0);
    put(0);
  }
  __syncthreads();
  for (int step = 0; step < steps; ++step) {
    const int buf = step & 1;
    if (step + 1 < steps) fetch(step + 1);
    const char *la = lds[buf] + (wm * (BM / 2) + (lane & 31)) * 128, *lb = lds[buf] + (BM + wn * 64 + (lane & 31)) * 128;
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
      const int c = 2 * kk + (lane >> 5);
      v4i ra[MT], rb[NT];
#pragma unroll
      for (int i = 0; i < MT; ++i) ra[i] = *reinterpret_cast<const v4i *>(la + i * 32 * 128 + ((c ^ swz(wm * (BM / 2) + i * 32 + (lane & 31))) << 4));
#pragma unroll
      for (int j = 0; j < NT; ++j) rb[j] = *reinterpret_cast<const v4i *>(lb + j * 32 * 128 + ((c ^ swz(wn * 64 + j * 32 + (lane & 31))) << 4));
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) Mma<T>::mma32(acc[i][j], ra[i], rb[j]);
    }
    if (step + 1 < steps) put(buf ^ 1);
    __syncthreads();
  }

  // register r of a 32 x 32 tile: row 8 (r / 4) + 4 (lane / 32) + r % 4, column lane % 32
  const int64_t rows = MODE == DW ? F : M;
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    if constexpr (MODE == FWD) {
      const int64_t f = f0 + wn * 32 + (lane & 31);
      const float bg = p.b_gate && f < F ? to_f(reinterpret_cast<const T *>(p.b_gate)[f]) : 0.f;
      const float bu = p.b_up && f < F ? to_f(reinterpret_cast<const T *>(p.b_up)[f]) : 0.f;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int64_t m = m0 + wm * (BM / 2) + i * 32 + 8 * (r / 4) + 4 * (lane >> 5) + r % 4;
        if (m < M && f < F) {
          const float g = acc[i][0][r] + bg, u = acc[i][1][r] + bu;
          reinterpret_cast<T *>(p.y)[m * F + f] = from_f<T>(act_f(p.act, g) * u);
          if (p.pre) {
            p.pre[m * F + f] = g;
            p.pre[(M + m) * F + f] = u;
          }
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const int64_t n = n0 + wn * 64 + j * 32 + (lane & 31);
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int64_t m = m0 + wm * (BM / 2) + i * 32 + 8 * (r / 4) + 4 * (lane >> 5) + r % 4;
          if (m < rows && n < D) {
            if (MODE == DX) reinterpret_cast<T *>(p.dx)[m * D + n] = from_f<T>(acc[i][j][r]);
            else if (a.ksplit > 1) a.slab[(((int64_t)ks * 2 + which) * F + m) * D + n] = acc[i][j][r];
            else reinterpret_cast<T *>(which ? p.dw_up : p.dw_gate)[m * D + n] = from_f<T>(acc[i][j][r]);
          }
        }
      }
    }
  }
}

// M <= 32 rows: 16 outputs per workgroup, K split over its four waves.  MFMA 16x16: the outputs are the A side, the rows the B side, so
// a lane ends with four consecutive outputs of one row.
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void k_gated_rows(Args a) {
  constexpr int E = 16 / sizeof(T), KS = 4 * E;         // elements of k per fragment step
  __shared__ v4f red[3][2][2][64];
  const fdql_gated_t &p = a.p;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t f0 = (int64_t)blockIdx.x * 16, D = p.D, F = p.F;
  const int i = lane & 15, q = lane >> 4;
  const T *x = reinterpret_cast<const T *>(p.x);
  const int64_t f = min(f0 + i, F - 1);                 // rows past the ends repeat the last one and are not stored
  const T *wg = reinterpret_cast<const T *>(p.w_gate) + f * D, *wu = reinterpret_cast<const T *>(p.w_up) + f * D;
  const T *x0 = x + min((int64_t)i, p.M - 1) * p.x_sr, *x1 = x + min((int64_t)i + 16, p.M - 1) * p.x_sr;
  v4f acc[2][2];
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int w = 0; w < 2; ++w) acc[m][w] = v4f{0.f, 0.f, 0.f, 0.f};
  const bool two = p.M > 16;
  const int64_t steps = (D + KS - 1) / KS, per = (steps + 3) / 4, s1 = min(steps, (wave + 1) * per);
#pragma unroll 4
  for (int64_t st = wave * per; st < s1; ++st) {
    const int64_t k = st * KS + q * E;
    const v4i g = row_chunk<T, VEC>(wg, k, D), u = row_chunk<T, VEC>(wu, k, D), b0 = row_chunk<T, VEC>(x0, k, D);
    Mma<T>::mma16(acc[0][0], g, b0);
    Mma<T>::mma16(acc[0][1], u, b0);
    if (two) {
      const v4i b1 = row_chunk<T, VEC>(x1, k, D);
      Mma<T>::mma16(acc[1][0], g, b1);
      Mma<T>::mma16(acc[1][1], u, b1);
    }
  }
  if (wave) {
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int w = 0; w < 2; ++w) red[wave - 1][m][w][lane] = acc[m][w];
  }
  __syncthreads();
  if (wave) return;
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    const int64_t row = m * 16 + i;
#pragma unroll
    for (int w = 0; w < 2; ++w)
#pragma unroll
      for (int v = 0; v < 3; ++v) acc[m][w] += red[v][m][w][lane];
    if (row >= p.M) continue;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int64_t o = f0 + 4 * q + r;
      if (o < F) {
        const float g = acc[m][0][r] + (p.b_gate ? to_f(reinterpret_cast<const T *>(p.b_gate)[o]) : 0.f);
        const float u = acc[m][1][r] + (p.b_up ? to_f(reinterpret_cast<const T *>(p.b_up)[o]) : 0.f);
        reinterpret_cast<T *>(p.y)[row * F + o] = from_f<T>(act_f(p.act, g) * u);
        if (p.pre) {
          p.pre[row * F + o] = g;
          p.pre[(p.M + row) * F + o] = u;
        }
      }
    }
  }
}

// dg, du of 64 columns x RB rows and their sums over those rows.
constexpr int RB = 128;
template <typename T>
__global__ __launch_bounds__(256) void k_gated_grad(Args a) {
  __shared__ float red[3][2][64];
  const fdql_gated_t &p = a.p;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t f = (int64_t)blockIdx.x * 64 + lane, m0 = (int64_t)blockIdx.y * RB;
  const int64_t F = p.F, M = p.M, MF = M * F;
  T *d = reinterpret_cast<T *>(a.d);
  float sg = 0.f, su = 0.f;
  if (f < a.Fp) {
    for (int64_t m = m0 + wave; m < min(M, m0 + RB); m += 4) {
      float dg = 0.f, du = 0.f;
      if (f < F) {
        const float g = p.pre[m * F + f], u = p.pre[MF + m * F + f];
        const float dy = to_f(reinterpret_cast<const T *>(p.dy)[m * p.dy_sr + f]);
        float v, dv;
        act_df(p.act, g, v, dv);
        dg = dy * u * dv;
        du = dy * v;
      }
      sg += dg;
      su += du;
      d[m * a.Fp + f] = from_f<T>(dg);
      d[(M + m) * a.Fp + f] = from_f<T>(du);
    }
  }
  if (wave) {
    red[wave - 1][0][lane] = sg;
    red[wave - 1][1][lane] = su;
  }
  __syncthreads();
  if (wave || f >= F) return;
#pragma unroll
  for (int q = 0; q < 3; ++q) {
    sg += red[q][0][lane];
    su += red[q][1][lane];
  }
  a.colsum[((int64_t)blockIdx.y * 2) * F + f] = sg;
  a.colsum[((int64_t)blockIdx.y * 2 + 1) * F + f] = su;
}

// out[i] = sum over n parts, `stride` floats apart; blockIdx.y picks the gate's or the up side's.
template <typename T>
__global__ __launch_bounds__(256) void k_gated_sum(const float *part, int64_t n, int64_t stride, int64_t count, void *gate, void *up) {
  T *out = reinterpret_cast<T *>(blockIdx.y ? up : gate);
  if (!out) return;
  const float *src = part + blockIdx.y * count;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < count; i += (int64_t)gridDim.x * 256) {
    float v = 0.f;
    for (int64_t k = 0; k < n; ++k) v += src[k * stride + i];
    out[i] = from_f<T>(v);
  }
}

struct Plan {
  int Fp, bk, ksplit, kper;
  int64_t rblocks;
};
Plan plan_of(const fdql_gated_t &p) {
  Plan q;
  q.Fp = (p.F + 7) / 8 * 8;
  q.bk = p.dtype == FDQL_F32 ? 32 : 64;
  q.rblocks = (p.M + RB - 1) / RB;
  const int64_t tiles = 2ll * ((p.F + 127) / 128) * ((p.D + BN - 1) / BN), slices = std::max<int64_t>(1, (p.M + q.bk - 1) / q.bk);
  int64_t ks = std::max<int64_t>(1, std::min<int64_t>(512 / tiles, slices / 8));
  q.kper = (int)((slices + ks - 1) / ks * q.bk);
  q.ksplit = (int)std::max<int64_t>(1, (p.M + q.kper - 1) / q.kper);
  return q;
}
int64_t up16(int64_t n) { return (n + 15) / 16 * 16; }
bool al16(const void *q) { return ((uintptr_t)q & 15) == 0; }

template <typename T>
hipError_t fwd(const fdql_gated_t &p, hipStream_t s) {
  Args a = {};
  a.p = p;
  constexpr int E = 16 / sizeof(T);
  const bool vec = p.D % E == 0 && p.x_sr % E == 0 && al16(p.x) && al16(p.w_gate) && al16(p.w_up);
  if (p.M <= 32) {
    const dim3 grid((unsigned)((p.F + 15) / 16));
    if (vec) hipLaunchKernelGGL((k_gated_rows<T, true>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((k_gated_rows<T, false>), grid, dim3(256), 0, s, a);
    return hipGetLastError();
  }
  a.tiles_n = (p.F + BN / 2 - 1) / (BN / 2);
  const bool small = (p.M + 127) / 128 * a.tiles_n < 512;
  a.tiles_m = (int)(small ? (p.M + 63) / 64 : (p.M + 127) / 128);
  const dim3 grid((unsigned)(a.tiles_m * a.tiles_n));
  if (small) {
    if (vec) hipLaunchKernelGGL((k_gated_tile<T, FWD, 64, true>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((k_gated_tile<T, FWD, 64, false>), grid, dim3(256), 0, s, a);
  } else {
    if (vec) hipLaunchKernelGGL((k_gated_tile<T, FWD, 128, true>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((k_gated_tile<T, FWD, 128, false>), grid, dim3(256), 0, s, a);
  }
  return hipGetLastError();
}

template <typename T>
hipError_t bwd(const fdql_gated_t &p, hipStream_t s) {
  const Plan q = plan_of(p);
  Args a = {};
  a.p = p;
  a.Fp = q.Fp;
  char *ws = reinterpret_cast<char *>(p.workspace);
  a.d = ws;
  ws += up16(2 * p.M * q.Fp * (int64_t)sizeof(T));
  a.colsum = reinterpret_cast<float *>(ws);
  ws += up16(q.rblocks * 2 * p.F * 4);
  a.slab = reinterpret_cast<float *>(ws);
  a.ksplit = q.ksplit;
  a.kper = q.kper;
  hipLaunchKernelGGL((k_gated_grad<T>), dim3((unsigned)((q.Fp + 63) / 64), (unsigned)q.rblocks), dim3(256), 0, s, a);
  // a column group of 4 must not straddle a row's end and must lie on its own size in memory
  const auto ok = [](const void *v) { return ((uintptr_t)v & (4 * sizeof(T) - 1)) == 0; };
  a.tiles_n = (p.D + BN - 1) / BN;
  if (p.dx) {
    const bool vec = p.D % 4 == 0 && ok(p.w_gate) && ok(p.w_up);
    const bool small = (p.M + 127) / 128 * a.tiles_n < 512;
    a.tiles_m = (int)(small ? (p.M + 63) / 64 : (p.M + 127) / 128);
    const dim3 grid((unsigned)(a.tiles_m * a.tiles_n));
    if (small) {
      if (vec) hipLaunchKernelGGL((k_gated_tile<T, DX, 64, true>), grid, dim3(256), 0, s, a);
      else hipLaunchKernelGGL((k_gated_tile<T, DX, 64, false>), grid, dim3(256), 0, s, a);
    } else {
      if (vec) hipLaunchKernelGGL((k_gated_tile<T, DX, 128, true>), grid, dim3(256), 0, s, a);
      else hipLaunchKernelGGL((k_gated_tile<T, DX, 128, false>), grid, dim3(256), 0, s, a);
    }
  }
  if (p.dw_gate && p.dw_up) {
    const bool vec = p.D % 4 == 0 && p.x_sr % 4 == 0 && ok(p.x);
    a.tiles_m = (p.F + 127) / 128;
    const dim3 grid((unsigned)(a.tiles_m * a.tiles_n), 2, (unsigned)q.ksplit);
    if (vec) hipLaunchKernelGGL((k_gated_tile<T, DW, 128, true>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((k_gated_tile<T, DW, 128, false>), grid, dim3(256), 0, s, a);
    if (q.ksplit > 1) {
      const int64_t n = (int64_t)p.F * p.D;
      hipLaunchKernelGGL((k_gated_sum<T>), dim3((unsigned)std::min<int64_t>((n + 255) / 256, 4096), 2), dim3(256), 0, s, a.slab, (int64_t)q.ksplit, 2 * n, n,
                         p.dw_gate, p.dw_up);
    }
  }
  if (p.db_gate || p.db_up)
    hipLaunchKernelGGL((k_gated_sum<T>), dim3((unsigned)((p.F + 255) / 256), 2), dim3(256), 0, s, a.colsum, q.rblocks, 2ll * p.F, (int64_t)p.F, p.db_gate, p.db_up);
  return hipGetLastError();
}

}  // namespace

int64_t gated_workspace_bytes(const fdql_gated_t &p, bool backward) {
  if (!backward) return 0;
  const Plan q = plan_of(p);
  const int64_t esz = p.dtype == FDQL_F32 ? 4 : 2;
  return up16(2 * p.M * q.Fp * esz) + up16(q.rblocks * 2 * p.F * 4) + (q.ksplit > 1 ? (int64_t)q.ksplit * 2 * p.F * p.D * 4 : 0);
}
hipError_t gated_fwd_launch(const fdql_gated_t &p, hipStream_t s) {
  return p.dtype == FDQL_F32 ? fwd<float>(p, s) : p.dtype == FDQL_BF16 ? fwd<bf16_t>(p, s) : fwd<f16_t>(p, s);
}
hipError_t gated_bwd_launch(const fdql_gated_t &p, hipStream_t s) {
  return p.dtype == FDQL_F32 ? bwd<float>(p, s) : p.dtype == FDQL_BF16 ? bwd<bf16_t>(p, s) : bwd<f16_t>(p, s);
}

}  // namespace fdql
