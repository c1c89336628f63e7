// Gated linear unit (fdql_gated*):  y = f(x Wg^T + bg) * (x Wu^T + bu), forward and backward.
//
// Forward: one matrix product against both weights, with the activation, the product and the biases in its epilogue - a wave's accumulators
// hold the gate and the up column of the same 32 outputs, so both meet in one lane and neither is stored (training keeps them in
// float32 for the backward pass: rounded to 16 bits they would cost the gradients a bit more than their own rounding does).
// Backward: an elementwise pass forms dg = dy u f'(g), du = dy f(g) in the operand type the matrix instructions take (16-bit types: in two parts
// whose sum has twice the digits, see Plan) and their column sums; then dx = dg Wg + du Wu is one product over 2 F, and dWg = dg^T x, dWu = du^T x are one launch with the rows
// split over workgroups where the weights alone leave the card idle (float32 slabs, added in order).
//
// k_gated_mma serves all three products: tiles of BM x BN, slices of the contraction in an LDS ring filled by LDS-DMA (see there).  Rows that are
// not whole 16-byte chunks are copied into the workspace first (k_gated_pack); tensors that only start in the middle of a chunk, and calls without
// a workspace, take k_gated_any: the same tiles with element loads through registers.  Matrix instructions:
// v_mfma_f32_32x32x16 (bf16, fp16) or four v_mfma_f32_32x32x2 (float) per pair of 16-byte fragments; which k a lane half holds is the same on
// both sides and does not matter.
//
// Few rows (M <= 32) are bound by the weights' bytes and by latency: k_gated_rows gives 16 outputs to a workgroup, splits K over its
// eight waves and reads fragments straight from memory.
#include "seq.h"

#include <algorithm>
#include <type_traits>

namespace fdql {
namespace {

typedef float v16f __attribute__((ext_vector_type(16)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef int v4i __attribute__((ext_vector_type(4)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));

enum Mode { FWD, DX, DW };

struct Args {
  fdql_gated_t p;
  int Fp, parts;                   // row length of d (F rounded up to 8); 2: d in two parts whose sum has twice the digits
  void *d;                         // [2][parts][M][Fp] dg, du in the operand type, zeros behind column F
  float *colsum;                   // [row blocks][2][F]
  float *slab;                     // [ksplit][2][F][D] when ksplit > 1
  int ksplit, kper;                // DW: slices of the rows and their length (a multiple of the K slice)
  int tiles_m, tiles_n;
  int Dk, ldw;                     // length of x's and the weights' rows as they are multiplied (D, or up to whole chunks with zeros behind), of the weights' as they lie
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

// GELU's two pieces: e^(-g^2 / 2), the square's rounding undone, and the normal distribution P(g) = erfc(-g / sqrt 2) / 2.  The argument's rounding
// is off by up to g^2 steps of a small P: a float result adds its first order, -rest erfc'(x) / 2 = rest e^(-x^2) / sqrt pi (a 16-bit one does not see it:
// P is below float's range from g = -13 on, 2^-16 before).
__device__ __forceinline__ float gauss(float g) {
  const float sq = g * g, rest = fmaf(g, g, -sq);
  return exp_acc(-0.5f * sq) * (sq < 1e4f ? fmaf(-0.5f, rest, 1.f) : 1.f);
}
template <typename T>
__device__ __forceinline__ float normal_cdf(float g, float gauss_g) {
  constexpr float C = 0.70710678118654752f, C_REST = (float)(0.70710678118654752440 - (double)C);
  const float x = -C * g;
  float p = 0.5f * erfcf(x);
  if (sizeof(T) == 4 && fabsf(g) < 100.f) p = fmaf(fmaf(C, g, x) + C_REST * g, 0.56418958354775628f * gauss_g, p);
  return p;
}
// f(g) and f'(g)
template <typename T>
__device__ __forceinline__ float act_f(int act, float g) {
  if (act == FDQL_ACT_GELU) return g * normal_cdf<T>(g, sizeof(T) == 4 ? gauss(g) : 0.f);
  const float s = sigmoid_f<T>(g).s;
  return act == FDQL_ACT_SILU ? g * s : s;
}
template <typename T>
__device__ __forceinline__ void act_df(int act, float g, float &f, float &df) {
  if (act == FDQL_ACT_GELU) {
    const float e = gauss(g), cdf = normal_cdf<T>(g, e);
    f = g * cdf;
    df = fmaf(g * 0.39894228040143268f, e, cdf);
  } else {
    const Sigmoid v = sigmoid_f<T>(g);
    f = act == FDQL_ACT_SILU ? g * v.s : v.s;
    df = act == FDQL_ACT_SILU ? fmaf(g * v.s, v.c, v.s) : v.s * v.c;
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

// A slice of LDS rows on its way through registers: NCH 16-byte chunks per thread.
template <int NCH>
struct Flight { v4i c[NCH]; };

// row_ptr(n) -> first element of operand row n or nullptr (zeros)
template <typename T, int NCH, typename F>
__device__ __forceinline__ void fetch_rows(Flight<NCH> &f, F row_ptr, int64_t k0, int64_t K) {
  constexpr int E = 16 / sizeof(T);
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    const int n = (threadIdx.x >> 3) + 32 * i, c = threadIdx.x & 7;
    const T *row = row_ptr(n);
    v4i z = {0, 0, 0, 0};
    f.c[i] = row ? row_chunk<T, false>(row, k0 + c * E, K) : z;
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

// The other orientation: memory is [k][column] with row length ld; thread = NJ columns x E rows of k, transposed in registers.
template <typename T, int NJ>
__device__ __forceinline__ void fetch_cols(Flight<NJ> &f, const T *base, int64_t ld, int64_t k0, int64_t K, int64_t col0, int64_t cols) {
  constexpr int E = 16 / sizeof(T);
  typedef T vec __attribute__((ext_vector_type(E)));
  const int64_t col = col0 + (threadIdx.x & 31) * NJ;
  const int64_t k = k0 + (threadIdx.x >> 5) * E;
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    vec v;
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = k + e < K && col + j < cols ? base[(k + e) * ld + col + j] : T(0.f);
    f.c[j] = __builtin_bit_cast(v4i, v);
  }
}
template <int NJ>
__device__ __forceinline__ void put_cols(const Flight<NJ> &f, char *lds) {
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    const int n = (threadIdx.x & 31) * NJ + j, c = threadIdx.x >> 5;
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

// A wave's accumulators: rows wm of two, 64 columns wn.  Register r of a 32 x 32 tile: row 8 (r / 4) + 4 (lane / 32) + r % 4, column lane % 32.
// WHOLE: the tile lies inside the matrix.  An address is a running scalar part and one 32-bit offset per lane (rows are at most 2^24 long).
template <typename T, int MODE, int MT, int BM, bool WHOLE>
__device__ __forceinline__ void store_part(const Args &a, const v16f (&acc)[MT][2], int64_t m0, int64_t n0, int64_t f0, int wm, int wn, int which, int ks) {
  const fdql_gated_t &p = a.p;
  const int lane = threadIdx.x & 63;
  const int64_t ld = MODE == FWD ? p.F : p.D, rows = MODE == DW ? p.F : p.M, top = m0 + wm * (BM / 2);
  const unsigned at = (unsigned)(lane >> 5) * 4u * (unsigned)ld + (lane & 31);
  const int left = (int)min(rows - top, (int64_t)BM) - 4 * (lane >> 5);           // rows of this lane's that are there
  float bg = 0.f, bu = 0.f;
  if (MODE == FWD && p.b_gate && f0 + wn * 32 + (lane & 31) < p.F) {
    bg = to_f(reinterpret_cast<const T *>(p.b_gate)[f0 + wn * 32 + (lane & 31)]);
    bu = to_f(reinterpret_cast<const T *>(p.b_up)[f0 + wn * 32 + (lane & 31)]);
  }
  T *out = reinterpret_cast<T *>(MODE == FWD ? p.y : MODE == DX ? p.dx : which ? p.dw_up : p.dw_gate);
  float *slab = MODE == DW ? a.slab + ((int64_t)ks * 2 + which) * rows * ld : nullptr;
#pragma unroll
  for (int j = 0; j < (MODE == FWD ? 1 : 2); ++j) {
    const int64_t c0 = MODE == FWD ? f0 + wn * 32 : n0 + wn * 64 + j * 32;
    const bool col = WHOLE || c0 + (lane & 31) < ld;
    int64_t o = top * ld + c0;
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int row = i * 32 + 8 * (r / 4) + r % 4;
        if (WHOLE || (col && row < left)) {
          if constexpr (MODE == FWD) {
            const float g = acc[i][0][r] + bg, u = acc[i][1][r] + bu;
            (out + o)[at] = from_f<T>(act_f<T>(p.act, g) * u);
            if (p.pre) {
              (p.pre + o)[at] = g;
              (p.pre + p.M * ld + o)[at] = u;
            }
          } else if (MODE == DW && a.ksplit > 1) {
            (slab + o)[at] = acc[i][j][r];
          } else {
            (out + o)[at] = from_f<T>(acc[i][j][r]);
          }
        }
        o += r % 4 == 3 ? 5 * ld : ld;
        asm volatile("" : "+s"(o));         // (64 precomputed row addresses would spill)
      }
  }
}
template <typename T, int MODE, int MT, int BM, int BN>
__device__ __forceinline__ void store_tile(const Args &a, const v16f (&acc)[MT][2], int64_t m0, int64_t n0, int64_t f0, int wm, int wn, int which, int ks) {
  const int64_t rows = MODE == DW ? a.p.F : a.p.M, cols = MODE == FWD ? a.p.F : a.p.D, c1 = MODE == FWD ? f0 + BN / 2 : n0 + BN;
  if (m0 + BM <= rows && c1 <= cols) store_part<T, MODE, MT, BM, true>(a, acc, m0, n0, f0, wm, wn, which, ks);
  else store_part<T, MODE, MT, BM, false>(a, acc, m0, n0, f0, wm, wn, which, ks);
}

template <int MT>
__device__ __forceinline__ void clear(v16f (&acc)[MT][2]) {
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
}

// The backward products pass over their contraction once for each of d's PARTS, DX for the gate's side, then the up side's.
template <int MODE, int PARTS>
constexpr int passes_of() { return MODE == FWD ? 1 : MODE == DX ? 2 * PARTS : PARTS; }
template <int MODE, int PARTS>
__device__ __forceinline__ int pass_of(int step, int len) {
  constexpr int N = passes_of<MODE, PARTS>();
  return N == 1 ? 0 : N == 2 ? step >= len : (step >= len) + (step >= 2 * len) + (step >= 3 * len);
}
template <int MODE, int PARTS>
__device__ __forceinline__ int side_of(int pass) { return MODE == DX ? pass / PARTS : 0; }

// Float sums over a long contraction: RUN slices (512 products) at a time, the runs added up apart, so that the rounding error grows with the run's
// length and their number instead of the whole length (dx at F 2000: 1.2e-6 of its norm in one chain).  16-bit results round at 2^-12
// or 2^-9 and keep one chain.
template <typename T, int MT>
struct Runs {
  static constexpr bool ON = sizeof(T) == 4;
  static constexpr int RUN = 16;
  v16f sum[ON ? MT : 1][2];
  __device__ __forceinline__ Runs() {
    if constexpr (ON) clear(sum);
  }
  __device__ __forceinline__ void turn(v16f (&acc)[MT][2], int step) {       // behind a slice's products
    if constexpr (ON) {
      if (step % RUN == RUN - 1) {
        close(acc);
        clear(acc);
      }
    }
  }
  __device__ __forceinline__ void close(v16f (&acc)[MT][2]) {
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) sum[i][j] += acc[i][j];
  }
  __device__ __forceinline__ void total(v16f (&acc)[MT][2]) {
    if constexpr (ON) {
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] += sum[i][j];
    }
  }
};

// 64 x 128 tiles for any alignment: slices of 128 bytes through registers into two LDS buffers, operands that lie across the contraction
// transposed on the way.
template <typename T, int MODE, int PARTS>
__global__ __launch_bounds__(256, 2) void k_gated_any(Args a) {
  constexpr int BM = 64, BN = 128, BK = 128 / sizeof(T);
  __shared__ __align__(16) char lds[2][(BM + BN) * 128];
  const fdql_gated_t &p = a.p;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave >> 1, wn = wave & 1;
  int tm, tn;
  tile_of(blockIdx.x, a.tiles_m, a.tiles_n, tm, tn);
  const int64_t M = p.M, D = p.D, F = p.F, m0 = (int64_t)tm * BM, f0 = (int64_t)tn * (BN / 2), n0 = (int64_t)tn * BN;
  const int which = MODE == DW ? blockIdx.y : 0, ks = MODE == DW ? blockIdx.z : 0;
  const T *x = reinterpret_cast<const T *>(p.x), *wg = reinterpret_cast<const T *>(p.w_gate), *wu = reinterpret_cast<const T *>(p.w_up);
  const T *dd = reinterpret_cast<const T *>(a.d) + (MODE == DW ? which * PARTS * M * a.Fp : 0);
  const int64_t kbeg = MODE == DW ? (int64_t)ks * a.kper : 0, kend = MODE == FWD ? D : MODE == DX ? F : min(M, kbeg + a.kper);
  const int half = (int)((kend - kbeg + BK - 1) / BK), steps = passes_of<MODE, PARTS>() * half;

  Flight<2> fa;
  Flight<4> fb;
  const auto fetch = [&](int step) {
    if constexpr (MODE == FWD) {
      const int64_t k0 = (int64_t)step * BK;
      fetch_rows<T>(fa, [&](int n) { return m0 + n < M ? x + (m0 + n) * p.x_sr : (const T *)nullptr; }, k0, D);
      fetch_rows<T>(fb, [&](int n) {               // 32 gate rows, 32 up rows per wave column
        const int64_t f = f0 + (n >> 6) * 32 + (n & 31);
        return f < F ? (n & 32 ? wu : wg) + f * D : (const T *)nullptr;
      }, k0, D);
    } else if constexpr (MODE == DX) {
      const int pass = pass_of<MODE, PARTS>(step, half), up = side_of<MODE, PARTS>(pass);
      const int64_t k0 = (int64_t)(step - pass * half) * BK;
      const T *src = dd + pass * M * a.Fp;
      fetch_rows<T>(fa, [&](int n) { return m0 + n < M ? src + (m0 + n) * a.Fp : (const T *)nullptr; }, k0, F);
      fetch_cols<T>(fb, up ? wu : wg, D, k0, F, n0, D);
    } else {
      const int pass = pass_of<MODE, PARTS>(step, half);
      const int64_t k0 = kbeg + (int64_t)(step - pass * half) * BK;
      fetch_cols<T>(fa, dd + pass * M * a.Fp, a.Fp, k0, kend, m0, F);
      fetch_cols<T>(fb, x, p.x_sr, k0, kend, n0, D);
    }
  };
  const auto put = [&](int buf) {
    if constexpr (MODE == DW) put_cols(fa, lds[buf]);
    else put_rows(fa, lds[buf]);
    if constexpr (MODE == FWD) put_rows(fb, lds[buf] + BM * 128);
    else put_cols(fb, lds[buf] + BM * 128);
  };
  v16f acc[1][2];
  clear(acc);
  Runs<T, 1> runs;
  if (steps > 0) {
    fetch(0);
    put(0);
  }
  __syncthreads();
  for (int step = 0; step < steps; ++step) {
    const int buf = step & 1, n = lane & 31;
    if (step + 1 < steps) fetch(step + 1);
    const char *la = lds[buf] + (wm * 32 + n) * 128, *lb = lds[buf] + (BM + wn * 64 + n) * 128;
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
      const int c = 2 * kk + (lane >> 5);
      const v4i ra = *reinterpret_cast<const v4i *>(la + ((c ^ swz(wm * 32 + n)) << 4));
#pragma unroll
      for (int j = 0; j < 2; ++j) Mma<T>::mma32(acc[0][j], ra, *reinterpret_cast<const v4i *>(lb + j * 32 * 128 + ((c ^ swz(wn * 64 + j * 32 + n)) << 4)));
    }
    runs.turn(acc, step);
    if (step + 1 < steps) put(buf ^ 1);
    __syncthreads();
  }
  runs.total(acc);
  store_tile<T, MODE, 1, BM, BN>(a, acc, m0, n0, f0, wm, wn, which, ks);
}

// ---------------------------------------------------------------------------------------------------- rows of whole 16-byte chunks
// BM x BN tiles, two waves along the rows and BN / 64 along the columns.  LDS holds a ring of NBUF slices of KS along the contraction, filled by
// LDS-DMA (16 bytes per lane straight from memory, no registers in between): while one slice is multiplied the next ones are on their way, with
// one counted wait and one barrier per slice; a wave's requests go out in pieces between its products.  An operand whose rows run along the
// contraction lies in LDS as [row][slice] and is read 16 bytes at a time; one that runs across it lies as [k][column]: 16-bit types read it with
// ds_read_b64_tr_b16, which hands every lane four consecutive k of its column, float one value at a time (v_mfma_f32_32x32x2 wants no more).
// The DMA writes lanes in order, so the swizzles against bank conflicts are applied to the addresses that lanes read from memory.  Chunks past
// an edge come from a block of zeros.
// Shapes: 256 x 256 (KS 32, 4 slices) and 128 x 256 (KS 64, 3 slices) with one workgroup per CU for 16-bit types and many tiles; 64 x 128 for
// few tiles; 64 x 128 and 128 x 128 for float, whose matrix instructions take so long that the ring needs only two slices and three or two
// workgroups share a CU.
// Measured (bf16, 8192 rows, F 4096): forward 508 us at D 4096 = 1082 TFLOP/s, 156 at D 1024 (about 45 us of it outside the contraction: filling
// the ring, activations, stores); float 12800 x 2048 x 1024 115 TFLOP/s.  What bounds the 16-bit loop is the way from L2 into LDS (copies of the
// kernel that left one thing out: with every request at one address 80% of the time, with none 76%, with one slice's LDS reads for all 97%); 128 x 256 tiles,
// which need half as much again per product, lose a third to it.  Splitting each slice between two groups of four waves (a third fewer LDS reads)
// gave 172 us instead of 182 for dx, of d in one part, and lost as much on the weight gradients.
__device__ const v4i g_zeros = {0, 0, 0, 0};

template <typename T, int BM, int BN>
struct Ring {
  static constexpr int KS = sizeof(T) == 4 ? 32 : BM == 256 ? 32 : 64, NBUF = sizeof(T) == 4 ? 2 : BM == 256 ? 4 : 3;
  static constexpr int ABYTES = BM * KS * (int)sizeof(T), BBYTES = BN * KS * (int)sizeof(T), BYTES = NBUF * (ABYTES + BBYTES);
};

template <int RB>     // [row][RB bytes]: row and chunk of LDS byte `o`; sixteen rows that are read together use sixteen different 16-byte places of 256
struct RowTile {
  static __device__ __forceinline__ int turn(int n) { return RB == 128 ? swz(n) : n >> 2 & 3; }
  static __device__ __forceinline__ int row(int o) { return o / RB; }
  static __device__ __forceinline__ int chunk(int o) { return (o / 16 % (RB / 16)) ^ turn(row(o)); }
  static __device__ __forceinline__ int at(int n, int c) { return n * RB + ((c ^ turn(n)) << 4); }
};
template <typename T, int COLS>   // [k][COLS]: groups of 32 columns change places with k so that the rows one instruction reads lie in different banks
struct ColTile {
  static constexpr int RB = COLS * (int)sizeof(T), GC = 32 * (int)sizeof(T) / 16, GROUPS = COLS / 32;      // chunks of a group
  static __device__ __forceinline__ int turn(int k) {
    if (sizeof(T) == 4) return k >> 2 & 1;                             // lane halves read k and k + 4
    return COLS == 64 ? k >> 1 & 1 : ((k & 3) | (k >> 1 & 4)) & (GROUPS - 1);      // four k, and four more eight further
  }
  static __device__ __forceinline__ int row(int o) { return o / RB; }
  static __device__ __forceinline__ int chunk(int o) { return (o / 16 % (RB / 16)) ^ (turn(row(o)) * GC); }
};
__device__ __forceinline__ unsigned lds_addr(const char *p) { return (unsigned)(uintptr_t)(const __attribute__((address_space(3))) char *)p; }
// LDS-DMA of 16 bytes per lane, lane l to lds + 16 l.  Written out because the compiler, which knows the builtin, would wait for every DMA in
// flight in front of each transposing read; nothing comes back into a register but M0, and the kernel counts its own waits.
__device__ __forceinline__ void dma16(const void *src, unsigned lds) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(src), "s"(lds) : "memory", "m0");
}
typedef short v4s __attribute__((ext_vector_type(4)));
__device__ __forceinline__ int2 tr_read(const char *p) {
  return __builtin_bit_cast(int2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4s *)p));
}

template <typename T, int MODE, int BM, int BN, int PARTS>
__global__ __launch_bounds__(BN * 2, 2) void k_gated_mma(Args a) {
  typedef Ring<T, BM, BN> R;
  constexpr int KS = R::KS, NBUF = R::NBUF, ABYTES = R::ABYTES, BBYTES = R::BBYTES, E = 16 / sizeof(T), RB = KS * sizeof(T), WAVES = BN / 32;
  constexpr int MT = BM / 64, NT = 2, NA = ABYTES / (WAVES * 1024), NB = BBYTES / (WAVES * 1024), KSTEPS = RB / 32;
  typedef RowTile<RB> Rows;
  typedef ColTile<T, BM> ACols;
  typedef ColTile<T, BN> BCols;
  extern __shared__ __align__(16) char lds[];
  const fdql_gated_t &p = a.p;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave / (WAVES / 2), wn = wave % (WAVES / 2);
  int tm, tn;
  tile_of(blockIdx.x, a.tiles_m, a.tiles_n, tm, tn);
  const int64_t M = p.M, D = p.D, F = p.F, m0 = (int64_t)tm * BM, n0 = (int64_t)tn * BN, f0 = (int64_t)tn * (BN / 2);
  const int which = MODE == DW ? blockIdx.y : 0, ks = MODE == DW ? blockIdx.z : 0;
  const T *x = reinterpret_cast<const T *>(p.x), *wg = reinterpret_cast<const T *>(p.w_gate), *wu = reinterpret_cast<const T *>(p.w_up);
  const T *dd = reinterpret_cast<const T *>(a.d) + which * PARTS * M * a.Fp;
  // contraction [kbeg, K) of one pass
  const int64_t kbeg = MODE == DW ? (int64_t)ks * a.kper : 0, K = MODE == FWD ? a.Dk : MODE == DX ? a.Fp : min(M, kbeg + a.kper);
  const int half = (int)((K - kbeg + KS - 1) / KS), steps = passes_of<MODE, PARTS>() * half;

  // where this lane's chunks come from: an element offset from the operand's start for slice 0, and the chunk's place in the contraction
  int64_t oa[NA], ob[NB];
  int ka[NA], kb[NB];
  bool ina[NA], inb[NB];
#pragma unroll
  for (int q = 0; q < NA; ++q) {
    const int o = (wave * NA + q) * 1024 + lane * 16;
    if (MODE == DW) {
      ka[q] = ACols::row(o);
      const int64_t c = m0 + ACols::chunk(o) * E;
      ina[q] = c < a.Fp;
      oa[q] = (int64_t)ka[q] * a.Fp + c;
    } else {
      ka[q] = Rows::chunk(o) * E;
      const int64_t r = m0 + Rows::row(o);
      ina[q] = r < M;
      oa[q] = r * (MODE == FWD ? p.x_sr : a.Fp) + ka[q];
    }
  }
#pragma unroll
  for (int q = 0; q < NB; ++q) {
    const int o = (wave * NB + q) * 1024 + lane * 16;
    if (MODE == FWD) {                              // LDS row n: 32 gate rows, then 32 up rows for every wave column
      const int n = Rows::row(o);
      kb[q] = Rows::chunk(o) * E;
      const int64_t f = f0 + (n >> 6) * 32 + (n & 31);
      inb[q] = f < F;
      ob[q] = f * a.ldw + kb[q];
    } else {
      kb[q] = BCols::row(o);
      const int64_t c = n0 + BCols::chunk(o) * E;
      inb[q] = c < D;
      ob[q] = (int64_t)kb[q] * (MODE == DX ? a.ldw : p.x_sr) + c;
    }
  }
  // piece `piece` of `pieces` of a slice's DMA (a wave is held up while its requests are taken: in one go, with the other waves', that left the
  // matrix unit idle for a quarter of a step)
  const auto fetch = [&](int step, int buf, int piece, int pieces) {
    const int pass = pass_of<MODE, PARTS>(step, half), up = side_of<MODE, PARTS>(pass);
    const int64_t k0 = kbeg + (int64_t)(step - pass * half) * KS;
    const unsigned la = lds_addr(lds) + buf * (ABYTES + BBYTES) + wave * NA * 1024, lb = lds_addr(lds) + buf * (ABYTES + BBYTES) + ABYTES + wave * NB * 1024;
    const T *pa = MODE == FWD ? x + k0 : MODE == DX ? dd + pass * M * a.Fp + k0 : dd + pass * M * a.Fp + k0 * a.Fp;
    const int64_t kx = k0 * (MODE == DX ? a.ldw : p.x_sr);
#pragma unroll
    for (int q = 0; q < NA + NB; ++q) {
      if (q * pieces / (NA + NB) != piece) continue;
      if (q < NA) {
        const int i = q < NA ? q : 0;
        dma16(ina[i] && k0 + ka[i] < K ? (const void *)(pa + oa[i]) : (const void *)&g_zeros, la + i * 1024);
      } else {
        const int i = q < NA ? 0 : q - NA;
        const T *pb = MODE == FWD ? ((wave * NB + i) * (1024 / RB) & 32 ? wu : wg) + k0 : MODE == DX ? (up ? wu : wg) + kx : x + kx;
        dma16(inb[i] && k0 + kb[i] < (MODE == DX ? F : K) ? (const void *)(pb + ob[i]) : (const void *)&g_zeros, lb + i * 1024);
      }
    }
  };

  // where this lane reads its fragments: [row][slice] tiles at row lane % 32, chunk 2 kk + lane / 32; [k][column] tiles at the k and columns
  // that the transposing read collects from it, or that it multiplies itself
  const int tr_k = (lane >> 5) * (sizeof(T) == 4 ? 4 : 8) + (sizeof(T) == 4 ? 0 : lane >> 2 & 3);
  const int tr_c = sizeof(T) == 4 ? lane & 31 : (lane >> 4 & 1) * 16 + (lane & 3) * 4;
  int at_a[MT], at_b[NT];                           // byte offsets of the wave's 32-row / 32-column blocks, kk = 0
#pragma unroll
  for (int i = 0; i < MT; ++i)
    at_a[i] = MODE == DW ? tr_k * ACols::RB + ((wm * MT + i) ^ ACols::turn(tr_k)) * (32 * (int)sizeof(T)) + tr_c * (int)sizeof(T) : 0;
#pragma unroll
  for (int j = 0; j < NT; ++j)
    at_b[j] = MODE != FWD ? tr_k * BCols::RB + ((wn * 2 + j) ^ BCols::turn(tr_k)) * (32 * (int)sizeof(T)) + tr_c * (int)sizeof(T) : 0;
  const auto row_frag = [&](const char *t, int r0, int kk) { return *reinterpret_cast<const v4i *>(t + Rows::at(r0 + (lane & 31), 2 * kk + (lane >> 5))); };
  const auto col_frag = [&](const char *t, int kk, int rb) {
    if constexpr (sizeof(T) == 4) {
      v4i v;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = *reinterpret_cast<const int *>(t + (kk * 8 + e) * rb);
      return v;
    } else {
      const int2 lo = tr_read(t + kk * 16 * rb), hi = tr_read(t + (kk * 16 + 4) * rb);
      return v4i{lo.x, lo.y, hi.x, hi.y};
    }
  };

  v16f acc[MT][NT];
  clear(acc);
  Runs<T, MT> runs;
  // (s_barrier by itself: __syncthreads would wait for every DMA in flight)
  int issued = 0;
  for (; issued < min(NBUF - 1, steps); ++issued) fetch(issued, issued, 0, 1);
  if (issued == NBUF - 1) asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"i"((NBUF - 2) * (NA + NB)) : "memory");
  else asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
  // The next fragments are on their way while these are multiplied, across slices too: the wait and the barrier stand in front of a slice's
  // last products (behind them, every wave would start the next slice with the latency of its LDS reads).
  constexpr int PIECES = NBUF == 2 ? KSTEPS - 1 : KSTEPS;                 // two slices: the next one must be on its way whole by then
  constexpr int EARLY = ((KSTEPS - 1) * (NA + NB) + PIECES - 1) / PIECES; // requests of a slice that go out before the wait
  constexpr int FLYING = NBUF == 2 ? 0 : (NBUF - 3) * (NA + NB) + EARLY;  // ... and may be under way behind it
  int buf = 0;
  v4i ra[2][MT], rb[2][NT];
  const auto frags = [&](int of, int kk) {
    const char *ta = lds + of * (ABYTES + BBYTES), *tb = ta + ABYTES;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      if constexpr (MODE == FWD) rb[kk & 1][j] = row_frag(tb, wn * 64 + j * 32, kk);
      else rb[kk & 1][j] = col_frag(tb + at_b[j], kk, BCols::RB);
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      if constexpr (MODE == DW) ra[kk & 1][i] = col_frag(ta + at_a[i], kk, ACols::RB);
      else ra[kk & 1][i] = row_frag(ta, wm * (BM / 2) + i * 32, kk);
    }
  };
  if (steps > 0) frags(0, 0);
  for (int step = 0; step < steps; ++step) {
    const bool more = step + NBUF - 1 < steps;
    const int next = buf == NBUF - 1 ? 0 : buf + 1;
#pragma unroll
    for (int kk = 0; kk < KSTEPS; ++kk) {
      if (kk + 1 < KSTEPS) {
        frags(buf, kk + 1);
      } else if (step + 1 < steps) {
        if (more) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"i"(FLYING) : "memory");
        else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        frags(next, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) Mma<T>::mma32(acc[i][j], ra[kk & 1][i], rb[kk & 1][j]);
      __builtin_amdgcn_sched_barrier(0);
      if (more) fetch(step + NBUF - 1, buf ? buf - 1 : NBUF - 1, kk, PIECES);   // into the slice that the last step was done with
    }
    buf = next;
    runs.turn(acc, step);
  }
  runs.total(acc);
  store_tile<T, MODE, MT, BM, BN>(a, acc, m0, n0, f0, wm, wn, which, ks);
}

// M <= 32 rows: 16 outputs per workgroup, K split over its eight waves.  MFMA 16x16: the outputs are the A side, the rows the B side, so
// a lane ends with four consecutive outputs of one row.  Bound by the weights' bytes, and by latency where they are few.  Measured against
// 64 x 128 tiles: float 32 x 256 x 256 6.2 us (15.0), 32 x 1024 x 4096 13.4 us (52.8), bf16 32 x 4096 x 4096 22.9 us = 2.9 TB/s (34.3), float
// 8 x 4096 x 4096 27.4 us = 4.9 TB/s.  With four waves 6.5, 16.8, 26.6 and 34.1 us; with sixteen 6.4, 13.2, 21.0 and 26.8, but bf16 4 x 4096 x
// 14336 48.0 instead of 44.6.
constexpr int NW = 8;
template <typename T, bool VEC>
__global__ __launch_bounds__(NW * 64) void k_gated_rows(Args a) {
  constexpr int E = 16 / sizeof(T), KS = 4 * E;         // elements of k per fragment step
  __shared__ v4f red[NW - 1][2][2][64];
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
  float bg[4] = {}, bu[4] = {};                         // read now, added behind the sums
  if (wave == 0 && p.b_gate) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int64_t o = min(f0 + 4 * q + r, F - 1);
      bg[r] = to_f(reinterpret_cast<const T *>(p.b_gate)[o]);
      bu[r] = to_f(reinterpret_cast<const T *>(p.b_up)[o]);
    }
  }
  const int64_t steps = (D + KS - 1) / KS, per = (steps + NW - 1) / NW, s1 = min(steps, (wave + 1) * per);
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
      for (int v = 0; v < NW - 1; ++v) acc[m][w] += red[v][m][w][lane];
    if (row >= p.M) continue;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int64_t o = f0 + 4 * q + r;
      if (o < F) {
        const float g = acc[m][0][r] + bg[r];
        const float u = acc[m][1][r] + bu[r];
        reinterpret_cast<T *>(p.y)[row * F + o] = from_f<T>(act_f<T>(p.act, g) * u);
        if (p.pre) {
          p.pre[row * F + o] = g;
          p.pre[(p.M + row) * F + o] = u;
        }
      }
    }
  }
}

// what rounding v to its first part left over (nothing where that overflowed)
template <typename T>
__device__ __forceinline__ T rest_of(float v, T part) {
  const float p = to_f(part);
  return from_f<T>(fabsf(p) < INFINITY ? v - p : 0.f);
}
// dg, du of 64 columns x RB rows and their sums over those rows.  Memory bounds it: bf16 8192 x 4096 140 us = 4.3 TB/s with d in two parts, 110 = 4.3 in one.
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
        act_df<T>(p.act, g, v, dv);
        dg = dy * u * dv;
        du = dy * v;
      }
      sg += dg;
      su += du;
      const T hg = from_f<T>(dg), hu = from_f<T>(du);
      d[m * a.Fp + f] = hg;
      d[(a.parts * M + m) * a.Fp + f] = hu;
      if (a.parts == 2) {
        d[(M + m) * a.Fp + f] = rest_of(dg, hg);
        d[(3 * M + m) * a.Fp + f] = rest_of(du, hu);
      }
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

// Weight gradients from the row slices' slabs (blockIdx.z 0) and bias gradients from the row blocks' column sums (1), both sides (blockIdx.y):
// 64 neighbouring values per workgroup, the parts dealt to its four waves.
template <typename T>
__global__ __launch_bounds__(256) void k_gated_sum(Args a, int64_t rblocks) {
  __shared__ float red[3][64];
  const bool bias = blockIdx.z;
  const int64_t count = bias ? a.p.F : (int64_t)a.p.F * a.p.D, n = bias ? rblocks : a.ksplit;
  T *out = reinterpret_cast<T *>(bias ? (blockIdx.y ? a.p.db_up : a.p.db_gate) : (blockIdx.y ? a.p.dw_up : a.p.dw_gate));
  if (!out || (!bias && a.ksplit == 1)) return;
  const float *src = (bias ? a.colsum : a.slab) + blockIdx.y * count;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int64_t i0 = (int64_t)blockIdx.x * 64; i0 < count; i0 += (int64_t)gridDim.x * 64) {
    const int64_t i = min(i0 + lane, count - 1);
    float v = 0.f;
#pragma unroll 8
    for (int64_t k = wave; k < n; k += 4) v += src[k * 2 * count + i];
    if (wave) red[wave - 1][lane] = v;
    __syncthreads();
    if (wave == 0 && i0 + lane < count) out[i] = from_f<T>(v + red[0][lane] + red[1][lane] + red[2][lane]);
    __syncthreads();
  }
}

// Rows of whole chunks from rows that are not: x [M], then Wg and Wu [F], each of Dp elements with zeros behind D.  A thread copies one chunk.
struct Pack {
  const void *src[3];
  int64_t sr[3], first[4];         // row strides; rows in front of each tensor's
  void *dst;
  int D, Dp;
};
template <typename T>
__global__ __launch_bounds__(256) void k_gated_pack(Pack a) {
  constexpr int E = 16 / sizeof(T);
  const int64_t per = a.Dp / E, n = a.first[3] * per;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    const int64_t row = i / per, c = i % per * E;
    const int w = (row >= a.first[1]) + (row >= a.first[2]);
    const T *src = reinterpret_cast<const T *>(a.src[w]) + (row - a.first[w]) * a.sr[w] + c;
    typedef T vec __attribute__((ext_vector_type(E)));
    vec v;
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = c + e < a.D ? src[e] : T(0.f);
    reinterpret_cast<vec *>(a.dst)[i] = v;
  }
}

constexpr int CUS = 256;
// Tile shape of a product: rows x columns of tiles, and for the weight gradients the slices of the rows that fill the card.
struct Shape {
  int bm, bn;
  int64_t tiles_m, tiles_n;
};
enum Choice { SMALL, WIDE, FLOAT };        // which tiles there are: 64 x 128 alone; and 128, 256 x 256 of 16-bit types; and 128 x 128 of float
Shape shape_of(Choice choice, int64_t rows, int64_t cols, int tile_of_256, int copies) {     // tile_of_256: columns that a 256-wide tile covers
  const auto tiles = [&](int bm, int bn) { return (rows + bm - 1) / bm * ((cols + tile_of_256 * bn / 256 - 1) / (tile_of_256 * bn / 256)); };
  Shape s = {64, 128, 0, 0};
  const auto rounds = [&](int64_t n) { return (n * copies + CUS - 1) / CUS; };      // tiles on the CU that has most
  // float: two workgroups of 128 x 128 on a CU or three of 64 x 128, both near the rate of the matrix units while they share it and slow when the
  // last one is alone: the larger tile (fewer bytes through LDS) where it needs no more row-steps of the card.  Forward without `pre` at D 512, F 256:
  // 12800 rows 79 us -> 70 to 75 (800 tiles or 400), 8192 rows 43 either way; where it needs more, 20000 rows, it would take 113 us instead of 102.
  if (choice == FLOAT && tiles(128, 128) >= CUS && 2 * rounds(tiles(128, 128)) <= rounds(tiles(64, 128))) s.bm = 128;
  // 16 bits: up to half a tile of 128 x 256 per CU the small ones are faster (bf16, D 1024: 128 tiles 19.7 us, as 512 small ones 17.1; 136 tiles 19.2
  // against 24.5; 256 tiles 22.8 against 29.5)
  if (choice == WIDE && tiles(128, 256) * copies > CUS / 2) {
    // one workgroup per CU: the tile that needs fewer row-steps of the card, the larger one where they need the same
    s.bn = 256;
    s.bm = rounds(tiles(256, 256)) * 2 <= rounds(tiles(128, 256)) ? 256 : 128;
  }
  s.tiles_m = (rows + s.bm - 1) / s.bm;
  s.tiles_n = (cols + tile_of_256 * s.bn / 256 - 1) / (tile_of_256 * s.bn / 256);
  return s;
}

// Rounding d to 16 bits once would add as much to the gradients' error as rounding the results does (8192 x 1024 x 4096, bf16: 0.0023 of their norm
// instead of 0.0017), so it is kept in two parts, whatever the size, and each part has its pass in the products: 890 us a training pass there
// against 564, 12800 x 512 x 256 91 us of kernels against 71, 1024 x 512 x 512 66 against 53.  A caller who would rather have the time asks for one
// part (FDQL_GATED_ROUND_GRADS).
struct Plan {
  int Fp, parts, ksplit, kper;
  int64_t rblocks;
};
Plan plan_of(const fdql_gated_t &p) {
  Plan q;
  q.Fp = (p.F + 7) / 8 * 8;
  q.parts = p.dtype == FDQL_F32 || (p.act & FDQL_GATED_ROUND_GRADS) ? 1 : 2;
  q.rblocks = (p.M + RB - 1) / RB;
  // rows split for the 64 x 128 tiles of the weight gradients (larger tiles are chosen where there are enough of them): slices of 256 rows and
  // more, up to three workgroups per CU of float (backward of 4096 x 1024 x 1024 324 us, with two 330, one 369) and two of 16 bits, whose
  // products are over sooner (weight gradients of bf16 12800 x 512 x 256 27.9 us, with three 31.6, of 4096 x 1024 x 1024 53.1 and 58.5)
  const int64_t tiles = 2ll * ((p.F + 63) / 64) * ((p.D + 127) / 128);
  const int64_t ks = std::max<int64_t>(1, std::min<int64_t>((p.dtype == FDQL_F32 ? 3 : 2) * CUS / tiles, p.M / 256));
  q.kper = (int)(((p.M + ks - 1) / ks + 63) / 64 * 64);
  q.kper = std::max(q.kper, 64);
  q.ksplit = (int)std::max<int64_t>(1, (p.M + q.kper - 1) / q.kper);
  return q;
}
int64_t up16(int64_t n) { return (n + 15) / 16 * 16; }
bool al16(const void *q) { return ((uintptr_t)q & 15) == 0; }

// Rows that are not whole 16-byte chunks are copied into some that are, whatever the size; the same work with element loads (k_gated_any) took, for
// forward and backward of bf16 4097 x 1001 x 2730, 1906 us against 483, 1000 x 301 x 203 118 against 63, 64 x 101 x 99 50 against 34, float 12800 x 511 x
// 256 365 against 273, and only where rows are a few dozen elements long up to 2 us less (forward of 10000 x 17 x 61 7.3 against 8.3).
bool packs(const fdql_gated_t &p) {
  const int E = p.dtype == FDQL_F32 ? 4 : 8;
  return p.M > 32 && (p.D % E != 0 || p.x_sr % E != 0);
}
int64_t pack_bytes(const fdql_gated_t &p) {
  const int E = p.dtype == FDQL_F32 ? 4 : 8;
  return packs(p) ? (p.M + (p.D % E ? 2ll * p.F : 0)) * ((p.D + E - 1) / E * 16ll) : 0;
}
// a.p's x and weights become their packed copies at the workspace's start; without a workspace they stay as they are
template <typename T>
hipError_t pack(Args &a, hipStream_t s) {
  constexpr int E = 16 / sizeof(T);
  fdql_gated_t &p = a.p;
  a.Dk = a.ldw = p.D;
  if (!packs(p) || !p.workspace) return hipSuccess;
  const bool w = p.D % E != 0;
  const int Dp = (p.D + E - 1) / E * E;
  Pack k = {{p.x, p.w_gate, p.w_up}, {p.x_sr, p.D, p.D}, {0, p.M, p.M + (w ? p.F : 0), p.M + (w ? 2ll * p.F : 0)}, p.workspace, p.D, Dp};
  hipLaunchKernelGGL((k_gated_pack<T>), dim3((unsigned)std::min<int64_t>((k.first[3] * (Dp / E) + 255) / 256, 8 * CUS)), dim3(256), 0, s, k);
  const T *at = reinterpret_cast<const T *>(p.workspace);
  p.x = at;
  p.x_sr = Dp;
  if (w) {
    p.w_gate = at + k.first[1] * Dp;
    p.w_up = at + k.first[2] * Dp;
    a.Dk = a.ldw = Dp;
  }
  return hipGetLastError();
}

template <typename T, int MODE>
Choice choice_of(bool aligned) {
  if (!aligned) return SMALL;
  return sizeof(T) == 2 ? WIDE : MODE == DW ? SMALL : FLOAT;
}

template <typename T, int MODE, int BM, int BN, int PARTS>
hipError_t launch_mma(const Args &a, dim3 grid, hipStream_t s) {
  constexpr int bytes = Ring<T, BM, BN>::BYTES;
  const hipError_t e = hipFuncSetAttribute((const void *)k_gated_mma<T, MODE, BM, BN, PARTS>, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL((k_gated_mma<T, MODE, BM, BN, PARTS>), grid, dim3(BN * 2), bytes, s, a);
  return hipGetLastError();
}
template <typename T, int MODE, int PARTS>
hipError_t launch_tiles(const Args &a, const Shape &q, bool aligned, dim3 grid, hipStream_t s) {
  if (!aligned) {
    hipLaunchKernelGGL((k_gated_any<T, MODE, PARTS>), grid, dim3(256), 0, s, a);
    return hipGetLastError();
  }
  if constexpr (sizeof(T) == 2) {
    if (q.bm == 256) return launch_mma<T, MODE, 256, 256, PARTS>(a, grid, s);
    if (q.bm == 128) return launch_mma<T, MODE, 128, 256, PARTS>(a, grid, s);
  }
  if constexpr (sizeof(T) == 4 && MODE != DW) {
    if (q.bm == 128) return launch_mma<T, MODE, 128, 128, PARTS>(a, grid, s);
  }
  return launch_mma<T, MODE, 64, 128, PARTS>(a, grid, s);
}
// rows x cols of the product's result; aligned: every operand row is made of whole 16-byte chunks
template <typename T, int MODE>
hipError_t product(Args a, int64_t rows, int64_t cols, bool aligned, hipStream_t s) {
  const int copies = MODE == DW ? 2 : 1;
  const Shape q = shape_of(choice_of<T, MODE>(aligned), rows, cols, MODE == FWD ? 128 : 256, copies);
  a.tiles_m = (int)q.tiles_m;
  a.tiles_n = (int)q.tiles_n;
  if (MODE == DW && q.bn == 256) a.ksplit = 1, a.kper = (int)((a.p.M + 63) / 64 * 64);
  const dim3 grid((unsigned)(q.tiles_m * q.tiles_n), copies, MODE == DW ? (unsigned)a.ksplit : 1);
  if constexpr (sizeof(T) == 2 && MODE != FWD) {
    if (a.parts == 2) return launch_tiles<T, MODE, 2>(a, q, aligned, grid, s);
  }
  return launch_tiles<T, MODE, 1>(a, q, aligned, grid, s);
}

template <typename T>
hipError_t fwd(const fdql_gated_t &p, hipStream_t s) {
  Args a = {};
  a.p = p;
  a.p.act &= ~FDQL_GATED_ROUND_GRADS;
  constexpr int E = 16 / sizeof(T);
  const hipError_t e = pack<T>(a, s);
  if (e != hipSuccess) return e;
  const bool vec = a.ldw % E == 0 && a.p.x_sr % E == 0 && al16(a.p.x) && al16(a.p.w_gate) && al16(a.p.w_up);
  if (p.M > 32) return product<T, FWD>(a, p.M, p.F, vec, s);
  const dim3 grid((unsigned)((p.F + 15) / 16));
  if (vec) hipLaunchKernelGGL((k_gated_rows<T, true>), grid, dim3(NW * 64), 0, s, a);
  else hipLaunchKernelGGL((k_gated_rows<T, false>), grid, dim3(NW * 64), 0, s, a);
  return hipGetLastError();
}

template <typename T>
hipError_t bwd(const fdql_gated_t &p, hipStream_t s) {
  constexpr int E = 16 / sizeof(T);
  const Plan q = plan_of(p);
  Args a = {};
  a.p = p;
  a.p.act &= ~FDQL_GATED_ROUND_GRADS;
  a.Fp = q.Fp;
  a.parts = q.parts;
  hipError_t e = pack<T>(a, s);
  if (e != hipSuccess) return e;
  char *ws = reinterpret_cast<char *>(p.workspace) + pack_bytes(p);
  a.d = ws;
  ws += up16(2 * q.parts * p.M * q.Fp * (int64_t)sizeof(T));
  a.colsum = reinterpret_cast<float *>(ws);
  ws += up16(q.rblocks * 2 * p.F * 4);
  a.slab = reinterpret_cast<float *>(ws);
  a.ksplit = q.ksplit;
  a.kper = q.kper;
  hipLaunchKernelGGL((k_gated_grad<T>), dim3((unsigned)((q.Fp + 63) / 64), (unsigned)q.rblocks), dim3(256), 0, s, a);
  e = hipGetLastError();
  if (e == hipSuccess && p.dx) e = product<T, DX>(a, p.M, p.D, a.ldw % E == 0 && al16(a.p.w_gate) && al16(a.p.w_up), s);
  const bool w = p.dw_gate && p.dw_up, vec = a.ldw % E == 0 && a.p.x_sr % E == 0 && al16(a.p.x);
  if (w && shape_of(choice_of<T, DW>(vec), p.F, p.D, 256, 2).bn == 256) a.ksplit = 1;
  if (e == hipSuccess && w) e = product<T, DW>(a, p.F, p.D, vec, s);
  const bool sum_w = w && a.ksplit > 1;
  if (e == hipSuccess && (sum_w || p.db_gate || p.db_up)) {
    const int64_t n = sum_w ? (int64_t)p.F * p.D : p.F;
    hipLaunchKernelGGL((k_gated_sum<T>), dim3((unsigned)std::min<int64_t>((n + 63) / 64, 4096), 2, 2), dim3(256), 0, s, a, q.rblocks);
    e = hipGetLastError();
  }
  return e;
}

}  // namespace

int64_t gated_workspace_bytes(const fdql_gated_t &p, bool backward) {
  if (!backward) return pack_bytes(p);
  const Plan q = plan_of(p);
  const int64_t esz = p.dtype == FDQL_F32 ? 4 : 2;
  return pack_bytes(p) + up16(2 * q.parts * p.M * q.Fp * esz) + up16(q.rblocks * 2 * p.F * 4) + (q.ksplit > 1 ? (int64_t)q.ksplit * 2 * p.F * p.D * 4 : 0);
}
hipError_t gated_fwd_launch(const fdql_gated_t &p, hipStream_t s) {
  return p.dtype == FDQL_F32 ? fwd<float>(p, s) : p.dtype == FDQL_BF16 ? fwd<bf16_t>(p, s) : fwd<f16_t>(p, s);
}
hipError_t gated_bwd_launch(const fdql_gated_t &p, hipStream_t s) {
  return p.dtype == FDQL_F32 ? bwd<float>(p, s) : p.dtype == FDQL_BF16 ? bwd<bf16_t>(p, s) : bwd<f16_t>(p, s);
}

}  // namespace fdql
