// Newton-Schulz orthogonalisation and the Muon server step (gfx950).
//
// For a matrix G (rows x cols) with m = min, n = max of the two sides, X is
// the m x n orientation of G / max(|G|_F, eps) and each step takes
//     A = X X^T,   Q = bA + cA^2,   X <- aX + QX,
// an odd polynomial of X's singular values (X = U s V^T gives U p(s) V^T).
//
// Numbers.  The iterates are kept as two fp16 limbs of 2^12·x: h = fp16(v),
// l = fp16(v - h), 22 bits of v and an absolute floor of 2^-37.  A product
// takes the three limb products hh + hl + lh on the matrix cores, each exact
// in its fp32 accumulator (the dropped ll is 2^-24 relative).  aX is added
// outside of the product in fp32: folded into Q its rounding would be
// amplified with the small singular values (x a = 3.44 a step), three times
// the error.  So the result is as exact as a chain of fp32 products (relative
// error 1e-6 .. 8e-6 against 64 bits by spectrum, both) at 3/16 of the cost
// per product: 16-bit limbs run at 16 times the fp32 matrix rate.
// The result's type does not matter to this: a 16-bit result is the fp32 one,
// rounded once.
//
// A = X X^T and A^2 are products C = P R^T with both operands contiguous along
// k; A and Q are symmetric: the tiles on and above the diagonal are computed
// and stored twice.  QX is computed as (QX)^T = X^T Q with X's fragments read
// transposed from LDS, so that X is kept in one orientation and a lane's
// results lie side by side in it (against X kept both ways: 4096 x 8192
// 7.36 -> 7.18 ms, 12 matrices' Muon step 2.23 -> 2.09).
//
// What bounds it: large matrices the matrix cores (4096 x 8192, QX 0.69 ms =
// 1.2 PFLOP/s of limb products, a library fp16 product of 8192^3 reaches
// 1.24) and, where the short side is 1024, the tiles' ends, which move 8 B a
// value through the caches with no product to hide them; middle ones the
// reads from L2 and three to five launches a step; narrow ones the latency
// of a chain of one launch a step.
#include "common.h"

#include <hip/hip_fp16.h>

#include <cmath>
#include <initializer_list>
#include <type_traits>

namespace fsagg {
namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef _Float16 half2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kMaxGroup = 24;     // matrices per launch (kernel arguments)
constexpr int kNormBlock = 256;
constexpr int kMaxNorm = 1024;    // norm workgroups per matrix
constexpr int kBK = 32;           // k per LDS stage
constexpr float kS = 4096.0f;     // limb scale
constexpr float kInvS = 1.0f / 4096.0f;

// One entry: `batch` matrices of one shape.
struct Mat {
  const void *g;       // update (newton_schulz); parameter average (muon)
  void *out;           // result (newton_schulz); parameter (muon)
  float *buf;          // momentum (muon)
  char *ws;            // workspace of matrix 0; matrix z at ws + z * wstride
  int64_t wstride;
  int64_t sz, si, sj;  // update strides, elements
  int32_t rows, cols, batch;
  int32_t m, n, mp, np;  // short and long side, and padded
  int32_t nb;            // norm workgroups per matrix
  int32_t slabs, each;   // narrow matrices: slabs, and 64-column chunks of one
  int32_t vec;           // 8 results side by side may be stored at once
  int16_t dt, odt;
};

// Workspace of one matrix: X limbs twice (a step reads one and writes the
// other), A limbs, Q limbs, norm partials.  The fp32 update lies in the
// second X until the first step writes it.
struct Planes {
  _Float16 *x, *ah, *al, *qh, *ql;
  int64_t e;
  double *norm;
  // (selected by arithmetic: an array indexed at run time would live in
  // scratch memory)
  __device__ __forceinline__ _Float16 *xh(int k) const {
    return x + 2 * k * e;
  }
  __device__ __forceinline__ _Float16 *xl(int k) const {
    return x + (2 * k + 1) * e;
  }
};

__host__ __device__ inline int64_t ws_elems(int64_t mp, int64_t np) {
  return 4 * mp * np + 4 * mp * mp;
}
__host__ __device__ inline int64_t ws_bytes_of(int64_t mp, int64_t np) {
  return 2 * ws_elems(mp, np) + 8 * kMaxNorm;
}
__device__ __forceinline__ Planes planes_of(const Mat &M, int z) {
  _Float16 *p = reinterpret_cast<_Float16 *>(M.ws + z * M.wstride);
  const int64_t e = int64_t(M.mp) * M.np, s = int64_t(M.mp) * M.mp;
  Planes P;
  P.x = p;
  P.e = e;
  P.ah = p + 4 * e;
  P.al = P.ah + s;
  P.qh = P.ah + 2 * s;
  P.ql = P.ah + 3 * s;
  P.norm = reinterpret_cast<double *>(P.ah + 4 * s);
  return P;
}

// A narrow matrix (m <= kNarrow) keeps the iterate as fp32, a column's 64
// rows together, and the slabs' shares of the Gram matrix, of this step and
// the next.
constexpr int kNarrow = 64;
constexpr int kNarrowLong = 16384;
constexpr int kMaxEach = 4, kMaxWhole = 4;
constexpr int kGramElems = kNarrow * kNarrow;
struct Narrow {
  double *norm;
  float *u, *x, *gram;
};
__device__ __forceinline__ Narrow narrow_of(const Mat &M, int z) {
  char *p = M.ws + z * M.wstride;
  Narrow N;
  N.norm = reinterpret_cast<double *>(p);
  N.x = reinterpret_cast<float *>(p + 8 * kMaxNorm);
  N.gram = N.x + int64_t(M.np) * kNarrow;
  N.u = N.gram + 2 * int64_t(M.slabs) * kGramElems;
  return N;
}

struct Group {
  int nmat;
  int start[kMaxGroup + 1];  // first workgroup of each entry
  Mat mat[kMaxGroup];
};

// entry and workgroup within it of workgroup b
__device__ __forceinline__ int find_mat(const Group &G, int b, int &rel) {
  int i = 0;
  while (i + 1 < G.nmat && b >= G.start[i + 1]) ++i;
  rel = b - G.start[i];
  return i;
}

struct MuonScalars {
  float keep, mu, lr, decay;  // 1 - momentum, momentum, lr, 1 - lr * wd
  int nesterov, maximize, adjust;
};

// the matrix's own learning rate
__device__ __forceinline__ float muon_lr(const Mat &M, const MuonScalars &S) {
  const float r = float(M.rows), k = float(M.cols);
  if (S.adjust == FSAGG_MUON_MATCH_RMS)
    return S.lr * (0.2f * __fsqrt_rn(r > k ? r : k));
  return r > k ? S.lr * __fsqrt_rn(__fdiv_rn(r, k)) : S.lr;
}

template <int DT>
__device__ __forceinline__ float load_as_f32(const void *p, int64_t i) {
  if constexpr (DT == FSAGG_F32) return static_cast<const float *>(p)[i];
  else if constexpr (DT == FSAGG_F16)
    return float(static_cast<const _Float16 *>(p)[i]);
  else
    return __uint_as_float(uint32_t(static_cast<const uint16_t *>(p)[i])
                           << 16);
}

// round to nearest even, NaN kept (quieted)
__device__ __forceinline__ uint16_t to_bf16(float v) {
  const uint32_t u = __float_as_uint(v);
  if ((u & 0x7FFFFFFFu) > 0x7F800000u) return uint16_t((u >> 16) | 0x40u);
  return uint16_t((u + 0x7FFFu + ((u >> 16) & 1u)) >> 16);
}

template <int DT>
__device__ __forceinline__ void store_from_f32(void *p, int64_t i, float v) {
  if constexpr (DT == FSAGG_F32) static_cast<float *>(p)[i] = v;
  else if constexpr (DT == FSAGG_F16)
    static_cast<_Float16 *>(p)[i] = _Float16(v);
  else
    static_cast<uint16_t *>(p)[i] = to_bf16(v);
}

// N = 4 or 8 results y of matrix z (m x n orientation) from (i, j) on, as
// type DT: rows i, i + 1, .. of column j (DOWN) or columns j, j + 1, .. of
// row i.  They lie side by side if the matrix is tall, or not, respectively;
// the first is then a multiple of N.
template <bool MUON, int DT, int N, bool DOWN>
__device__ __forceinline__ void store_result(const Mat &M,
                                             const MuonScalars &S, int z,
                                             int i, int j, const float *y) {
  if (j >= M.n || i >= M.m) return;
  const bool tall = M.rows > M.cols;
  const int64_t o = (MUON ? 0 : int64_t(z) * M.rows * M.cols) +
                    (tall ? int64_t(j) * M.cols + i
                          : int64_t(i) * M.cols + j);
  if (tall == DOWN && M.vec) {
    if constexpr (MUON) {
      f32x4 *p = reinterpret_cast<f32x4 *>(static_cast<float *>(M.out) + o);
      const float lr = muon_lr(M, S);
      f32x4 v[N / 4];
#pragma unroll
      for (int q = 0; q < N / 4; ++q) v[q] = p[q];
#pragma unroll
      for (int q = 0; q < N / 4; ++q) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          v[q][e] = __builtin_fmaf(-lr, y[4 * q + e],
                                   __fmul_rn(v[q][e], S.decay));
        p[q] = v[q];
      }
    } else if constexpr (DT == FSAGG_F32) {
      f32x4 *p = reinterpret_cast<f32x4 *>(static_cast<float *>(M.out) + o);
#pragma unroll
      for (int q = 0; q < N / 4; ++q)
        p[q] = f32x4{y[4 * q], y[4 * q + 1], y[4 * q + 2], y[4 * q + 3]};
    } else {
      typedef uint32_t un __attribute__((ext_vector_type(N / 2)));
      un v;
#pragma unroll
      for (int e = 0; e < N; e += 2) {
        uint32_t h[2];
#pragma unroll
        for (int d = 0; d < 2; ++d)
          h[d] = DT == FSAGG_F16
                     ? __builtin_bit_cast(uint16_t, _Float16(y[e + d]))
                     : to_bf16(y[e + d]);
        v[e / 2] = h[0] | (h[1] << 16);
      }
      *reinterpret_cast<un *>(static_cast<uint16_t *>(M.out) + o) = v;
    }
    return;
  }
  const int64_t step = tall == DOWN ? 1 : M.cols;
  const int have = DOWN ? M.m - i : M.n - j;
  if constexpr (MUON) {
    float *const out = static_cast<float *>(M.out) + o;
    const float lr = muon_lr(M, S);
    float v[N];
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = out[(e < have ? e : have - 1) * step];
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (e < have)
        out[e * step] = __builtin_fmaf(-lr, y[e], __fmul_rn(v[e], S.decay));
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (e < have) store_from_f32<DT>(M.out, o + e * step, y[e]);
  }
}

// Limbs of two values (one conversion instruction rounds both).
__device__ __forceinline__ void split2(float v0, float v1, half2 &h,
                                       half2 &l) {
  h = __builtin_convertvector((f32x2){v0, v1}, half2);
  l = __builtin_convertvector((f32x2){v0 - float(h[0]), v1 - float(h[1])},
                              half2);
}
// Limbs of N values, side by side.
template <int N, typename H>
__device__ __forceinline__ void split_n(const float *v, H &h, H &l) {
#pragma unroll
  for (int e = 0; e < N; e += 2) {
    half2 x, y;
    split2(v[e], v[e + 1], x, y);
    h[e] = x[0];
    h[e + 1] = x[1];
    l[e] = y[0];
    l[e + 1] = y[1];
  }
}

// What the update at a place is made of: the loads, apart from what follows
// them so that those of several places go out together.
struct Taken {
  float g, p, o;  // update or average; parameter, momentum (muon)
};
template <bool MUON, int DT>
__device__ __forceinline__ Taken take_at(const Mat &M, int z, int64_t e,
                                         int64_t i, int64_t j) {
  if constexpr (!MUON)
    return {load_as_f32<DT>(M.g, z * M.sz + i * M.si + j * M.sj), 0.0f, 0.0f};
  return {static_cast<const float *>(M.g)[e],
          static_cast<const float *>(M.out)[e], M.buf[e]};
}

// The update at element e: the input's own, or the momentum step from
// parameter - average, whose new momentum is stored.
template <bool MUON>
__device__ __forceinline__ float update_of(const Mat &M, const MuonScalars &S,
                                           int64_t e, const Taken &t) {
  if constexpr (!MUON) return t.g;
  float g = __fsub_rn(t.p, t.g);
  if (S.maximize) g = -g;
  // the torch.lerp forms: exact at both ends (mu = 0 gives g)
  const float d = __fsub_rn(g, t.o);
  const float n = S.keep < 0.5f
                      ? __builtin_fmaf(S.keep, d, t.o)
                      : __fsub_rn(g, __fmul_rn(d, 1.0f - S.keep));
  M.buf[e] = n;
  return S.nesterov ? __builtin_fmaf(S.mu, __fsub_rn(n, g), g) : n;
}

// f(integral constant): the update's type as a template argument
template <bool MUON, typename F>
__device__ __forceinline__ void with_update_type(const Mat &M, F f) {
  if (!MUON && M.dt == FSAGG_F16) f(std::integral_constant<int, FSAGG_F16>());
  else if (!MUON && M.dt == FSAGG_BF16)
    f(std::integral_constant<int, FSAGG_BF16>());
  else f(std::integral_constant<int, FSAGG_F32>());
}

// Sum of the workgroup's kThreads values, in a fixed order, in every thread.
template <int kThreads>
__device__ __forceinline__ double block_sum(double v, double *part) {
  part[threadIdx.x] = v;
  __syncthreads();
  for (int s = kThreads / 2; s > 0; s >>= 1) {
    if (int(threadIdx.x) < s) part[threadIdx.x] += part[threadIdx.x + s];
    __syncthreads();
  }
  return part[0];
}

// The sum of the norm workgroups' shares.
__device__ __forceinline__ double norm_sum(const double *norm, int nb,
                                           double *part) {
  double v = 0.0;
  for (int i = threadIdx.x; i < nb; i += 256) v += norm[i];
  return block_sum<256>(v, part);
}

// kS / max(norm, eps); NaN for a NaN norm, as dividing by it would give
__device__ __forceinline__ double limb_scale(double sq, double eps) {
  const double norm = sqrt(sq);
  return double(kS) / (norm < eps ? eps : norm);
}

// Pass 1: the fp32 update u, rows x cols contiguous, and a workgroup's sum
// of u^2 in fp64 (squares of fp32 neither overflow nor vanish there).
template <bool MUON, bool NARROW>
__global__ __launch_bounds__(kNormBlock) void ns_update_kernel(
    Group G, MuonScalars S) {
  int rel;
  const Mat &M = G.mat[find_mat(G, blockIdx.x, rel)];
  const int z = rel / M.nb, b = rel % M.nb;
  float *u;
  double *norm;
  if constexpr (NARROW) {
    const Narrow N = narrow_of(M, z);
    u = N.u;
    norm = N.norm;
  } else {
    const Planes P = planes_of(M, z);
    u = reinterpret_cast<float *>(P.xh(1));
    norm = P.norm;
  }
  const uint32_t total = uint32_t(M.rows) * uint32_t(M.cols);
  const uint32_t step = uint32_t(M.nb) * kNormBlock;
  double sq = 0.0;
  constexpr int kAhead = 8;
  with_update_type<MUON>(M, [&](auto dt) {
    for (uint32_t e0 = uint32_t(b) * kNormBlock + threadIdx.x; e0 < total;
         e0 += kAhead * step) {
      Taken t[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const uint32_t e = e0 + k * step < total ? e0 + k * step : total - 1;
        const uint32_t i = MUON ? 0u : e / uint32_t(M.cols);
        t[k] = take_at<MUON, decltype(dt)::value>(
            M, z, e, i, e - i * uint32_t(M.cols));
      }
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const uint32_t e = e0 + k * step;
        if (e >= total) break;
        const float v = update_of<MUON>(M, S, e, t[k]);
        u[e] = v;
        sq += double(v) * double(v);
      }
    }
  });
  __shared__ double part[kNormBlock];
  sq = block_sum<kNormBlock>(sq, part);
  if (threadIdx.x == 0) norm[b] = sq;
}

// Pass 2: X limbs of u / max(|u|, eps), zero in the padding.  One workgroup
// per 64 x 64 tile of the padded m x n orientation; the tile goes through LDS
// so that it is read and written in rows, whichever way u lies.
__global__ __launch_bounds__(256) void ns_prepare_kernel(Group G,
                                                         double eps) {
  int rel;
  const Mat &M = G.mat[find_mat(G, blockIdx.x, rel)];
  const int tn = M.np / 64, tiles = (M.mp / 64) * tn;
  const int z = rel / tiles, t = rel % tiles;
  const Planes P = planes_of(M, z);
  const float *u = reinterpret_cast<const float *>(P.xh(1));
  __shared__ double part[256];
  __shared__ float tile[64][65];
  const int i0 = (t / tn) * 64, j0 = (t % tn) * 64;
  const bool tall = M.rows > M.cols;
  // u's own rows r and columns c of this tile
  const int r0 = tall ? j0 : i0, c0 = tall ? i0 : j0;
  // (all on their way before the norm is waited for; places past the matrix
  // read its last row or column: a load under a condition is waited for
  // before the next one goes out)
  const int c = threadIdx.x % 64;
  float u0[16];
#pragma unroll
  for (int k = 0; k < 16; ++k) {
    const int r = r0 + k * 4 + int(threadIdx.x) / 64;
    u0[k] = u[int64_t(r < M.rows ? r : M.rows - 1) * M.cols +
              (c0 + c < M.cols ? c0 + c : M.cols - 1)];
  }
  const double scale = limb_scale(norm_sum(P.norm, M.nb, part), eps);
#pragma unroll
  for (int k = 0; k < 16; ++k) {
    const int r = k * 4 + int(threadIdx.x) / 64;
    // (a place past the matrix stays zero under a scale of infinity or NaN)
    const bool in = r0 + r < M.rows && c0 + c < M.cols;
    const float v = in ? float(double(u0[k]) * scale) : 0.0f;
    if (tall) tile[c][r] = v;
    else tile[r][c] = v;
  }
  __syncthreads();
  // 8 values a thread
  for (int k = threadIdx.x; k < 64 * 8; k += 256) {
    const int r = k / 8, c8 = k % 8 * 8;
    float v[8];
    half8 h, l;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = tile[r][c8 + e];
    split_n<8>(v, h, l);
    const int64_t x = int64_t(i0 + r) * M.np + j0 + c8;
    *reinterpret_cast<half8 *>(P.xh(0) + x) = h;
    *reinterpret_cast<half8 *>(P.xl(0) + x) = l;
  }
}

// A transposing read of LDS: of the 16 lanes of a group, lane i is given 4
// values of row i / 4, columns 4 (i % 4) on, and gets those of column i.
__device__ __forceinline__ half4 read_tr(const _Float16 *p) {
  typedef short s4 __attribute__((ext_vector_type(4)));
  return __builtin_bit_cast(
      half4, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                 (__attribute__((address_space(3))) s4 *)(uintptr_t)p));
}
__device__ __forceinline__ half8 join4(half4 x, half4 y) {
  return __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
}

enum Mode { kGram, kSquare, kApply, kLast, kLastMuon };

constexpr bool symmetric(int mode) { return mode == kGram || mode == kSquare; }

// Tiles of one matrix and stages (of kBK) of a tile.
template <int MODE, int BM, int BN>
__host__ __device__ __forceinline__ int mode_tiles(const Mat &M) {
  const int tm = M.mp / BM;
  return symmetric(MODE) ? tm * (tm + 1) / 2 : tm * (M.np / BN);
}
template <int MODE>
__host__ __device__ __forceinline__ int mode_stages(const Mat &M) {
  return (MODE == kGram ? M.np : M.mp) / kBK;
}

// Tile t of a matrix.  Neighbours in t share operands, so that the
// workgroups of one XCD read few rows: bands of kBand tile rows, column by
// column.  A symmetric product has the tiles with ti <= tj only.
constexpr int kBand = 4;
template <int MODE, int BM, int BN>
__device__ __forceinline__ void tile_of(const Mat &M, int t, int &ti,
                                        int &tj) {
  const int tm = M.mp / BM;
  if constexpr (symmetric(MODE)) {
    int b = 0;  // first tile row of the band
    for (;;) {
      const int h = tm - b < kBand ? tm - b : kBand;
      // a triangle of h rows, then full columns
      const int tri = h * (h + 1) / 2, n = tri + h * (tm - b - h);
      if (t >= n) {
        t -= n;
        b += h;
        continue;
      }
      if (t < tri) {
        int c = 0;
        while (t > c) {
          t -= c + 1;
          ++c;
        }
        ti = b + t;
        tj = b + c;
      } else {
        t -= tri;
        ti = b + t % h;
        tj = b + h + t / h;
      }
      return;
    }
  } else {
    const int tn = M.np / BN;
    const int b = t / (kBand * tn) * kBand;
    const int h = tm - b < kBand ? tm - b : kBand;
    t -= b * tn;
    ti = b + t % h;
    tj = t / h;
  }
}

// The stages of a group's product in one line: entry after entry, tile after
// tile.  Each of `workers` workgroups takes `each` of them, the first `more`
// one more (no division: in 64 bits it costs the join more than its sums).
struct Line {
  int workers, each, more;
  float *partial;  // [workers][first, later][BM * BN]
};
__device__ __forceinline__ int line_at(const Line &L, int q) {
  return q * L.each + (q < L.more ? q : L.more);
}

// One tile of C = P R^T (k contiguous in both), from stage k0 to stage k1.  A
// stage is kBK of k of both operands' limbs, written to LDS by 16-byte direct
// loads: 64-byte rows, the four 16-byte slots of row r permuted by (r / 4) %
// 4 so that a fragment read of 16 rows touches all 64 banks once.  NBUF
// stages of LDS: one is multiplied while NBUF - 1 are on their way.
//
// With TR the left operand lies the other way, P^T with rows along k: a stage
// is kBK rows of BM, and transposing reads (a group of 16 lanes takes 4 rows
// of 16 columns, lane i the 4 values of column i) make the same fragments.
// 32 lanes read 64 bytes of each of 4 rows, so the rows' 64-byte pieces are
// permuted by the row, and again every bank is touched once.
//
// Rows and columns of the padding are zero in every plane (the prepare pass
// writes them, products of zero rows are zero), so no tile is ragged inside
// the workspace; only the last step checks its stores against the matrix.
template <int BM, int BN, int WM, int WN, int NBUF>
struct Tile {
  static constexpr int kBM = BM, kBN = BN;
  static constexpr int kWaves = (BM / WM) * (BN / WN);
  static constexpr int kThreads = kWaves * 64;
  static constexpr int MI = WM / 32, NJ = WN / 32;
  static constexpr int kLoads = (BM + BN) * 2 * kBK * 2 / 1024;  // 1 KiB
  static constexpr int kPer = kLoads / kWaves;
  static constexpr int kStage = (BM + BN) * 2 * kBK;  // halfs
  static constexpr int kLds = NBUF * kStage;
  static_assert(kPer * kWaves == kLoads, "loads divide over the waves");
  static_assert(BM % (kPer * 16) == 0 && BN % (kPer * 16) == 0,
                "a wave loads one plane's rows");

  f32x16 acc[MI][NJ];
  int lane, wave, wm, wn;

  __device__ __forceinline__ Tile() {
    lane = threadIdx.x & 63;
    wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) >> 6);
    wm = (wave % (BM / WM)) * WM;
    wn = (wave / (BM / WM)) * WN;
  }

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;
  }

  // which 64-byte piece of row k of a transposed stage piece 0 goes to (rows
  // of 64 have two pieces, and two rows fill the banks)
  static __device__ __forceinline__ int piece(int k) {
    return BM >= 128 ? k & 3 : (k >> 1) & 1;
  }

  template <bool TR>
  __device__ __forceinline__ void multiply(_Float16 *lds, const _Float16 *ph,
                                           const _Float16 *pl, int ldp,
                                           const _Float16 *rh,
                                           const _Float16 *rl, int ldr,
                                           int i0, int j0, int k0, int k1,
                                           int depth) {
    // this wave's loads of a stage: LDS order is [P.h][P.l][R.h][R.l] rows
    // of 64 bytes, 16 rows per instruction, one plane per wave
    const int row0 = wave * (kPer * 16);
    const bool right = row0 >= 2 * BM;
    const int in = right ? row0 - 2 * BM : row0;
    const int side = right ? BN : BM;
    const _Float16 *base = in < side ? (right ? rh : ph) : (right ? rl : pl);
    const int g0 = (right ? j0 : i0) + (in < side ? in : in - side);
    // (a buffer descriptor: one 32-bit offset per lane instead of a 64-bit
    // address per load)
    const int lr = lane >> 2;
    const int ld = right ? ldr : ldp;
    const _Float16 *first = base + int64_t(g0) * ld;
    uint32_t extent = uint32_t(kPer * 16 * ld) * 2u;
    // lane offsets of even and odd loads, bytes from load to load and from
    // stage to stage
    uint32_t goff0 = uint32_t(lr * ld + ((lane & 3) ^ ((lr >> 2) & 3)) * 8) *
                     2u;
    uint32_t goff1 = goff0, dload = uint32_t(16 * ld) * 2u, dstage = kBK * 2;
    if constexpr (TR) {
      if (!right) {
        constexpr int kSlots = BM / 8;        // 16-byte slots of a row
        constexpr int kRows = 64 / kSlots;    // rows of a load
        const int r0 = (in < side ? in : in - side) / 16 * kRows;
        const int r = lane / kSlots, slot = lane % kSlots;
        first = base + int64_t(r0) * ld + i0;
        extent = uint32_t(depth - r0) * uint32_t(ld) * 2u - uint32_t(i0) * 2u;
        goff0 = uint32_t(r * ld + (slot ^ (piece(r0 + r) << 2)) * 8) * 2u;
        goff1 = uint32_t(r * ld + (slot ^ (piece(r0 + kRows + r) << 2)) * 8) *
                2u;
        dload = uint32_t(kRows * ld) * 2u;
        dstage = uint32_t(kBK * ld) * 2u;
      }
    }
    __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<_Float16 *>(first), short(0), int(extent), 0x00020000);
    // (past the last stage: an offset outside the descriptor, which fetches
    // nothing; so every stage has as many loads on their way, and the loop
    // has no branch.  A plane has at most 2.7 GB: FSAGG_NS_MAX_ELEMS halfs,
    // and a quarter more of padding)
    constexpr uint32_t kPast = 0xF0000000u;
    auto issue = [&](int k) {
      _Float16 *st = lds + (k % NBUF) * kStage + row0 * kBK;
      const uint32_t off0 = k < k1 ? goff0 : kPast;
      const uint32_t off1 = k < k1 ? goff1 : kPast;
      const uint32_t at = k < k1 ? uint32_t(k) * dstage : 0u;
#pragma unroll
      for (int q = 0; q < kPer; ++q)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(
            rsrc,
            (__attribute__((address_space(3))) void *)(uintptr_t)(
                st + q * 16 * kBK),
            16, int(q & 1 ? off1 : off0), int(uint32_t(q) * dload + at), 0, 0);
    };
    const int fr = lane & 31, fk = lane >> 5;
    struct Frags {
      half8 a[2][MI], b[2][NJ];
    };
    auto read = [&](Frags &f, int k, int kk) {
      const _Float16 *st = lds + (k % NBUF) * kStage;
#pragma unroll
      for (int i = 0; i < MI; ++i) {
        if constexpr (TR) {
          const int r = kk * 16 + fk * 8 + (lane & 15) / 4;
          const int col = wm + i * 32 + (fr & 16) + (lane & 3) * 4;
          const int o =
              r * BM + (((col / 8) ^ (piece(r) << 2)) * 8) + col % 8;
#pragma unroll
          for (int l = 0; l < 2; ++l) {
            const _Float16 *p = st + l * BM * kBK + o;
            f.a[l][i] = join4(read_tr(p), read_tr(p + 4 * BM));
          }
          continue;
        }
        const int r = wm + i * 32 + fr;
        const int o = r * kBK + (((kk * 2 + fk) ^ ((r >> 2) & 3)) * 8);
#pragma unroll
        for (int l = 0; l < 2; ++l)
          f.a[l][i] = *reinterpret_cast<const half8 *>(st + l * BM * kBK + o);
      }
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const int r = wn + j * 32 + fr;
        const int o = r * kBK + (((kk * 2 + fk) ^ ((r >> 2) & 3)) * 8);
#pragma unroll
        for (int l = 0; l < 2; ++l)
          f.b[l][j] = *reinterpret_cast<const half8 *>(
              st + (2 * BM + l * BN) * kBK + o);
      }
    };
    // l h, h l, h h (the small terms first)
    auto mul = [&](const Frags &f) {
#pragma unroll
      for (int t = 0; t < 3; ++t)
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
          for (int j = 0; j < NJ; ++j)
            acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(
                f.a[t == 0 ? 1 : 0][i], f.b[t == 1 ? 1 : 0][j], acc[i][j], 0, 0,
                0);
    };
    clear();
    // nothing of the previous tile is on its way, and every wave has read its
    // last stage
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
    for (int n = 0; n < NBUF; ++n) issue(k0 + n);
    // The fragments of the next half stage are read while the present one is
    // multiplied.  In the middle of stage k every wave has read all of it:
    // past that barrier its buffer takes stage k + NBUF.
    Frags f0, f1;
    wait_and_meet<(NBUF - 1) * kPer>();
    read(f0, k0, 0);
    for (int k = k0; k + 1 < k1; ++k) {
      read(f1, k, 1);
      mul(f0);
      spread<0, TR>();
      __builtin_amdgcn_sched_barrier(0);
      wait_and_meet<(NBUF - 2) * kPer>();
      read(f0, k + 1, 0);
      issue(k + NBUF);
      mul(f1);
      spread<kPer, TR>();
      __builtin_amdgcn_sched_barrier(0);
    }
    read(f1, k1 - 1, 1);
    __builtin_amdgcn_sched_barrier(0);
    mul(f0);
    mul(f1);
    // (nothing may be on its way to LDS when the workgroup ends)
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  }

  // Order of a half stage: the fragment reads, then LOADS direct loads, one
  // at a time between the matrix instructions, so that the waves do not queue
  // for the LDS and the memory pipe while the matrix cores wait.
  template <int LOADS, bool TR>
  static __device__ __forceinline__ void spread() {
    constexpr int kMfma = MI * NJ * 3;
    constexpr int kReads = 2 * ((TR ? 2 : 1) * MI + NJ);
    constexpr int kEach = kMfma > kReads + LOADS ? kMfma / (kReads + LOADS)
                                                 : 1;
#pragma unroll
    for (int n = 0; n < kReads; ++n) {
      __builtin_amdgcn_sched_group_barrier(0x008, kEach, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
#pragma unroll
    for (int n = 0; n < LOADS; ++n) {
      __builtin_amdgcn_sched_group_barrier(0x008, kEach, 0);
      __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, kMfma, 0);
  }

  // all but the last N of this wave's direct loads have landed, and every
  // wave says so; LDS reads before it are done
  template <int N>
  static __device__ __forceinline__ void wait_and_meet() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N)
                 : "memory");
  }

  // block (i, j) of the accumulators as it lies in the threads, 16 bytes at
  // a time
  __device__ __forceinline__ void put_partial(float *p) const {
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          f32x4 v;
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = acc[i][j][4 * q + e];
          reinterpret_cast<f32x4 *>(
              p)[((i * NJ + j) * 4 + q) * kThreads + threadIdx.x] = v;
        }
  }
  static __device__ __forceinline__ void get_partial(f32x4 (&v)[4],
                                                     const float *p,
                                                     int block) {
#pragma unroll
    for (int q = 0; q < 4; ++q)
      v[q] = reinterpret_cast<const f32x4 *>(
          p)[(block * 4 + q) * kThreads + threadIdx.x];
  }

  // f(integral constant): the result's type as a template argument
  template <int MODE, typename F>
  static __device__ __forceinline__ void with_result_type(const Mat &M, F f) {
    if constexpr (MODE == kLast) {
      if (M.odt == FSAGG_BF16) f(std::integral_constant<int, FSAGG_BF16>());
      else if (M.odt == FSAGG_F16)
        f(std::integral_constant<int, FSAGG_F16>());
      else f(std::integral_constant<int, FSAGG_F32>());
    } else {
      f(std::integral_constant<int, FSAGG_F32>());
    }
  }

  template <int MODE, int DT>
  __device__ __forceinline__ void finish_as(const Mat &M, const Planes &P,
                                            int z, int ti, int tj, int src,
                                            float a, float b, float c,
                                            const MuonScalars &S) const {
    // (what is added is read kAhead blocks before its turn)
    constexpr int kBlocks = MI * NJ, kAhead = kBlocks < 2 ? kBlocks : 2;
    Addend add[kAhead];
#pragma unroll
    for (int n = 0; n < kAhead; ++n)
      add[n] = addend<MODE>(M, P, ti, tj, n / NJ, n % NJ, src);
#pragma unroll
    for (int n = 0; n < kBlocks; ++n) {
      const Addend now = add[n % kAhead];
      if (n + kAhead < kBlocks)
        add[n % kAhead] = addend<MODE>(M, P, ti, tj, (n + kAhead) / NJ,
                                       (n + kAhead) % NJ, src);
      finish_block<MODE, DT>(acc[n / NJ][n % NJ], now, M, P, z, ti, tj, n / NJ,
                             n % NJ, src, a, b, c, S);
    }
  }
  template <int MODE>
  __device__ __forceinline__ void finish(const Mat &M, const Planes &P, int z,
                                         int ti, int tj, int src, float a,
                                         float b, float c,
                                         const MuonScalars &S) const {
    with_result_type<MODE>(M, [&](auto dt) {
      finish_as<MODE, decltype(dt)::value>(M, P, z, ti, tj, src, a, b, c, S);
    });
  }

  // Block (i, j) of the accumulators: the matrix cores leave a lane column gj
  // and four runs of 4 rows; lanes l and l + 32 exchange two of them, so that
  // a lane has two runs of 8 rows (gi .. gi + 7, + 16).  Of (QX)^T these are
  // 8 columns of X, 16 bytes a lane.
  template <int MODE>
  __device__ __forceinline__ int block_row(int ti, int tj, int i) const {
    return (symmetric(MODE) ? ti : tj) * BM + wm + i * 32 + 8 * (lane >> 5);
  }
  template <int MODE>
  __device__ __forceinline__ int block_column(int ti, int tj, int j) const {
    return (symmetric(MODE) ? tj : ti) * BN + wn + j * 32 + (lane & 31);
  }

  // A or X where the block's results lie (A is symmetric: its column gj is
  // row gj)
  struct Addend {
    half8 h[2], l[2];
  };
  template <int MODE>
  __device__ __forceinline__ Addend addend(const Mat &M, const Planes &P,
                                           int ti, int tj, int i, int j,
                                           int src) const {
    Addend v;
    if constexpr (MODE != kGram) {
      const _Float16 *bh = MODE == kSquare ? P.ah : P.xh(src);
      const _Float16 *bl = MODE == kSquare ? P.al : P.xl(src);
      const int64_t o = int64_t(block_column<MODE>(ti, tj, j)) *
                            (MODE == kSquare ? M.mp : M.np) +
                        block_row<MODE>(ti, tj, i);
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        v.h[p] = *reinterpret_cast<const half8 *>(bh + o + 16 * p);
        v.l[p] = *reinterpret_cast<const half8 *>(bl + o + 16 * p);
      }
    }
    return v;
  }

  // what the product is for, for one block.  DT: the result's type.
  template <int MODE, int DT>
  __device__ __forceinline__ void finish_block(
      const f32x16 &acc16, const Addend &add, const Mat &M, const Planes &P,
      int z, int ti, int tj, int i, int j, int src, float a, float b, float c,
      const MuonScalars &S) const {
    constexpr bool kX = !symmetric(MODE);
    const int gi0 = block_row<MODE>(ti, tj, i);
    const int gj = block_column<MODE>(ti, tj, j);
    const int ld = kX ? M.np : M.mp;
    f32x16 x = acc16;
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const auto s = __builtin_amdgcn_permlane32_swap(
            __float_as_uint(x[8 * p + e]), __float_as_uint(x[8 * p + 4 + e]),
            false, false);
        x[8 * p + e] = __uint_as_float(s[0]);
        x[8 * p + 4 + e] = __uint_as_float(s[1]);
      }
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const int gi = gi0 + 16 * p;
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[e] = x[8 * p + e] * kInvS;
        if constexpr (MODE == kSquare)
          v[e] = b * (float(add.h[p][e]) + float(add.l[p][e])) + c * v[e];
        else if constexpr (MODE != kGram)
          v[e] = a * (float(add.h[p][e]) + float(add.l[p][e])) + v[e];
      }
      if constexpr (MODE == kLast || MODE == kLastMuon) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] *= kInvS;
        store_result<MODE == kLastMuon, DT, 8, false>(M, S, z, gj, gi, v);
      } else {
        half8 h, l;
        split_n<8>(v, h, l);
        _Float16 *ch = kX ? P.xh(src ^ 1) : MODE == kGram ? P.ah : P.qh;
        _Float16 *cl = kX ? P.xl(src ^ 1) : MODE == kGram ? P.al : P.ql;
        // C's other half, unless the tile is its own transpose
        if (!kX && ti != tj) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int64_t o = int64_t(gi + e) * ld + gj;
            ch[o] = h[e];
            cl[o] = l[e];
          }
        }
        const int64_t o = int64_t(gj) * ld + gi;
        *reinterpret_cast<half8 *>(ch + o) = h;
        *reinterpret_cast<half8 *>(cl + o) = l;
      }
    }
  }
};

// Tile (ti, tj) of the mode's product, stages k0 to k1.
template <int MODE, class T>
__device__ __forceinline__ void multiply_of(T &tile, _Float16 *lds,
                                            const Mat &M, const Planes &P,
                                            int src, int ti, int tj, int k0,
                                            int k1) {
  if constexpr (MODE == kGram)
    tile.template multiply<false>(lds, P.xh(src), P.xl(src), M.np, P.xh(src),
                                  P.xl(src), M.np, ti * T::kBM, tj * T::kBN,
                                  k0, k1, 0);
  else if constexpr (MODE == kSquare)
    tile.template multiply<false>(lds, P.ah, P.al, M.mp, P.ah, P.al, M.mp,
                                  ti * T::kBM, tj * T::kBN, k0, k1, 0);
  else
    tile.template multiply<true>(lds, P.xh(src), P.xl(src), M.np, P.qh, P.ql,
                                 M.mp, tj * T::kBM, ti * T::kBN, k0, k1,
                                 M.mp);
}

// Workgroup b's place when the workgroups, which go round robin over the 8
// XCDs, shall take a contiguous stretch of the work per XCD.
__device__ __forceinline__ int xcd_place(int b, int n) {
  const int per = n / 8, more = n % 8, x = b % 8;
  return x * per + (x < more ? x : more) + b / 8;
}

// A product, one workgroup per tile (G.start counts tiles).
template <class T, int MODE>
__global__ __launch_bounds__(T::kThreads) void ns_gemm_kernel(
    Group G, int src, float a, float b, float c, MuonScalars S) {
  __shared__ __attribute__((aligned(1024))) _Float16 lds[T::kLds];
  int rel;
  const Mat &M =
      G.mat[find_mat(G, xcd_place(int(blockIdx.x), int(gridDim.x)), rel)];
  const int tiles = mode_tiles<MODE, T::kBM, T::kBN>(M);
  const int z = rel / tiles;
  int ti, tj;
  tile_of<MODE, T::kBM, T::kBN>(M, rel % tiles, ti, tj);
  const Planes P = planes_of(M, z);
  T tile;
  multiply_of<MODE>(tile, lds, M, P, src, ti, tj, 0, mode_stages<MODE>(M));
  tile.template finish<MODE>(M, P, z, ti, tj, src, a, b, c, S);
}

// A product over the line of stages (G.start counts stages): whole tiles are
// finished here, a tile that two or more workgroups share leaves its parts
// in `partial`.
template <class T, int MODE>
__global__ __launch_bounds__(T::kThreads) void ns_line_kernel(
    Group G, Line L, int src, float a, float b, float c, MuonScalars S) {
  __shared__ __attribute__((aligned(1024))) _Float16 lds[T::kLds];
  const int q = xcd_place(int(blockIdx.x), L.workers);
  int at = line_at(L, q);
  const int end = line_at(L, q + 1);
  T tile;
  for (int seg = 0; at < end; ++seg) {
    int rel;
    const Mat &M = G.mat[find_mat(G, at, rel)];
    const int stages = mode_stages<MODE>(M);
    const int tiles = mode_tiles<MODE, T::kBM, T::kBN>(M);
    const int t = rel / stages, k0 = rel % stages;
    const int left = end - at;
    const int k1 = stages - k0 < left ? stages : k0 + left;
    const int z = t / tiles;
    int ti, tj;
    tile_of<MODE, T::kBM, T::kBN>(M, t % tiles, ti, tj);
    const Planes P = planes_of(M, z);
    multiply_of<MODE>(tile, lds, M, P, src, ti, tj, k0, k1);
    if (k0 == 0 && k1 == stages)
      tile.template finish<MODE>(M, P, z, ti, tj, src, a, b, c, S);
    else
      tile.put_partial(L.partial +
                       (int64_t(q) * 2 + (seg > 0)) * (T::kBM * T::kBN));
    at += k1 - k0;
  }
}

// Tiles that workgroups shared: workgroup (w, block) looks at the boundary
// between workers w and w + 1 and, when it is the first one inside a tile,
// adds the tile's parts in order, one 32 x 32 block of every wave.
template <class T, int MODE>
__global__ __launch_bounds__(T::kThreads) void ns_join_kernel(
    Group G, Line L, int src, float a, float b, float c, MuonScalars S) {
  int w = int(blockIdx.x);
  const int block = int(blockIdx.y);
  const int cut = line_at(L, w + 1);
  int rel;
  const Mat &M = G.mat[find_mat(G, cut, rel)];
  const int stages = mode_stages<MODE>(M);
  const int tiles = mode_tiles<MODE, T::kBM, T::kBN>(M);
  const int t = rel / stages, first = cut - rel % stages;
  if (cut == first || line_at(L, w) > first) return;
  const int z = t / tiles;
  int ti, tj;
  tile_of<MODE, T::kBM, T::kBN>(M, t % tiles, ti, tj);
  const T tile;
  const Planes P = planes_of(M, z);
  const int i = block / T::NJ, j = block % T::NJ;
  const auto add = tile.template addend<MODE>(M, P, ti, tj, i, j, src);
  f32x16 x;
#pragma unroll
  for (int r = 0; r < 16; ++r) x[r] = 0.0f;
  constexpr int kAhead = 4;
  for (bool more = true; more; w += kAhead) {
    f32x4 v[kAhead][4];
    bool in[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      in[u] = w + u < L.workers && line_at(L, w + u) < first + stages;
      if (in[u])
        T::get_partial(v[u],
                       L.partial + (int64_t(w + u) * 2 +
                                    (line_at(L, w + u) < first)) *
                                       (T::kBM * T::kBN),
                       block);
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (in[u]) {
#pragma unroll
        for (int r = 0; r < 16; ++r) x[r] = __fadd_rn(x[r], v[u][r / 4][r % 4]);
      }
    more = in[kAhead - 1];
  }
  T::template with_result_type<MODE>(M, [&](auto dt) {
    tile.template finish_block<MODE, decltype(dt)::value>(
        x, add, M, P, z, ti, tj, i, j, src, a, b, c, S);
  });
}

// -- narrow matrices ---------------------------------------------------------
// m <= 64: A and Q are one 64 x 64 tile, and what a step costs is latency:
// reading the columns, three small products one after the other, and handing
// the Gram matrix over.  A group of 4 waves owns up to kMaxEach chunks of 64
// columns, a wave one 32 x 32 block of every product; the columns stay in
// its registers for the step.  Up to kMaxWhole chunks are the groups of one
// workgroup, which takes all steps in one launch (the Gram shares meet in
// LDS).  Beyond that a workgroup is one group: a launch sums the slabs' Gram
// shares of the step before (every workgroup the same, in order), forms Q,
// applies it and leaves its share of the next one, so a step is one launch
// where the tiled products take three (us: 62 x 2048 66, of which a launch
// 11; tiled 109; one launch of all steps: 5 x 9 14.5, 50 x 60 18.4, 60 x 250
// 31).
__device__ __forceinline__ int swz(int r, int chunk) {
  return r * 64 + ((chunk ^ ((r >> 1) & 7)) * 8);
}

struct Slab {
  int lane, fr, fk, bi, bj;
  __device__ __forceinline__ Slab() {
    lane = threadIdx.x & 63;
    fr = lane & 31;
    fk = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) >> 6);
    bi = (wave & 1) * 32;
    bj = (wave & 2) * 16;
  }
  // rows of quad q of this lane, and its column
  __device__ __forceinline__ int row(int q) const {
    return bi + 8 * q + 4 * fk;
  }
  __device__ __forceinline__ int col() const { return bj + fr; }

  // x += the products of K times 16 of k, of the fragments that left(kk, limb)
  // and right(kk, limb) read.  The small limb products go to an accumulator of
  // their own (a chain of dependent matrix instructions is what a product this
  // small waits for).
  template <int K, typename P, typename R>
  static __device__ __forceinline__ void chain(P left, R right, f32x16 &x) {
    f32x16 s;
#pragma unroll
    for (int e = 0; e < 16; ++e) s[e] = 0.0f;
#pragma unroll
    for (int kk = 0; kk < K; ++kk) {
      const half8 ph = left(kk, 0), pl = left(kk, 4096);
      const half8 rh = right(kk, 0), rl = right(kk, 4096);
      s = __builtin_amdgcn_mfma_f32_32x32x16_f16(pl, rh, s, 0, 0, 0);
      x = __builtin_amdgcn_mfma_f32_32x32x16_f16(ph, rh, x, 0, 0, 0);
      s = __builtin_amdgcn_mfma_f32_32x32x16_f16(ph, rl, s, 0, 0, 0);
    }
#pragma unroll
    for (int e = 0; e < 16; ++e) x[e] = __fadd_rn(x[e], s[e]);
  }

  // x += P R^T over the first 16 K of k (the rest is zero); planes [64][64],
  // limbs l at + 4096
  template <int K>
  __device__ __forceinline__ void multiply(const _Float16 *p,
                                           const _Float16 *r,
                                           f32x16 &x) const {
    const auto rows = [&](const _Float16 *q, int b) {
      return [=](int kk, int limb) {
        return *reinterpret_cast<const half8 *>(
            q + limb + swz(b + fr, kk * 2 + fk));
      };
    };
    chain<K>(rows(p, bi), rows(r, bj), x);
  }
  // x += X X^T over the first 16 K columns, of the plane as put_columns leaves
  // it (row j: column j of X): fragments by transposing reads of rows j .. j + 3
  // and j + 4 .. j + 7
  template <int K>
  __device__ __forceinline__ void gram_of(const _Float16 *p,
                                          f32x16 &x) const {
    const int l = lane & 15, j = fk * 8 + (l >> 2);
    const auto rows = [&](int b) {
      const int i = b + (fr & 16) + 4 * (l & 3);
      const _Float16 *lo = p + swz(j, i >> 3) + (i & 7);
      const _Float16 *hi = p + swz(j + 4, i >> 3) + (i & 7);
      // (16 rows on, the slots are permuted alike)
      return [=](int kk, int limb) {
        return join4(read_tr(lo + limb + kk * 16 * 64),
                     read_tr(hi + limb + kk * 16 * 64));
      };
    };
    chain<K>(rows(bi), rows(bj), x);
  }
  // limbs of the block's values (times kS), transposed: row col(), the rows
  // of a quad side by side
  __device__ __forceinline__ void put_columns(_Float16 *p,
                                              const f32x16 &x) const {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const float v[4] = {x[4 * q], x[4 * q + 1], x[4 * q + 2], x[4 * q + 3]};
      half4 h, l;
      split_n<4>(v, h, l);
      const int o = swz(col(), row(q) >> 3) + (row(q) & 7);
      *reinterpret_cast<half4 *>(p + o) = h;
      *reinterpret_cast<half4 *>(p + 4096 + o) = l;
    }
  }
};

// The scaled update of chunk `ch` (kS times), zero in the padding whatever
// the scale; raw: the update itself.
template <bool MUON, bool WHOLE>
__device__ __forceinline__ void load_update(const Mat &M, const Narrow &N,
                                            const Slab &W,
                                            const MuonScalars &S, int z,
                                            int ch, f32x16 &x) {
  const bool tall = M.rows > M.cols;
  const int j = ch * 64 + W.col();
  // (places past the matrix read its last row or column)
  const int lj = j < M.n ? j : M.n - 1;
  const auto place = [&](int i, int jj) {
    return int64_t(tall ? jj : i) * M.cols + (tall ? i : jj);
  };
  if constexpr (!WHOLE) {
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int i = W.row(r / 4) + r % 4;
      x[r] = N.u[place(i < M.m ? i : M.m - 1, lj)];
    }
  } else {
    with_update_type<MUON>(M, [&](auto dt) {
      // (4 at a time, and the addresses of 4: with 1024 threads there are no
      // registers for all)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        int i0 = W.row(q);
        asm volatile("" : "+v"(i0));
        Taken t[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int li = i0 + r < M.m ? i0 + r : M.m - 1;
          t[r] = take_at<MUON, decltype(dt)::value>(
              M, z, place(li, lj), tall ? lj : li, tall ? li : lj);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (i0 + r < M.m && j < M.n)
            x[4 * q + r] = update_of<MUON>(M, S, place(i0 + r, j), t[r]);
      }
    });
  }
#pragma unroll
  for (int r = 0; r < 16; ++r)
    if (W.row(r / 4) + r % 4 >= M.m || j >= M.n) x[r] = 0.0f;
}
__device__ __forceinline__ void scale_update(const Mat &M, const Slab &W,
                                             int ch, double scale,
                                             f32x16 &x) {
  const int j = ch * 64 + W.col();
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const int i = W.row(r / 4) + r % 4;
    x[r] = i < M.m && j < M.n ? float(double(x[r]) * scale) : 0.0f;
  }
}
template <bool MUON, int DT>
__device__ __forceinline__ void store_chunk_as(const Mat &M, const Slab &W,
                                               const MuonScalars &S, int z,
                                               int ch, const f32x16 &x) {
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    float y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = x[4 * q + e] * kInvS;
    store_result<MUON, DT, 4, true>(M, S, z, W.row(q), ch * 64 + W.col(), y);
  }
}
template <bool MUON>
__device__ __forceinline__ void store_chunk(const Mat &M, const Slab &W,
                                            const MuonScalars &S, int z,
                                            int ch, const f32x16 &x) {
  if (!MUON && M.odt == FSAGG_BF16)
    store_chunk_as<MUON, FSAGG_BF16>(M, W, S, z, ch, x);
  else if (!MUON && M.odt == FSAGG_F16)
    store_chunk_as<MUON, FSAGG_F16>(M, W, S, z, ch, x);
  else
    store_chunk_as<MUON, FSAGG_F32>(M, W, S, z, ch, x);
}
__device__ __forceinline__ void clear16(f32x16 &v) {
#pragma unroll
  for (int r = 0; r < 16; ++r) v[r] = 0.0f;
}
// A whole matrix of up to kMaxWhole chunks, group g the chunk g.
template <bool MUON>
__global__ __launch_bounds__(256 * kMaxWhole) void ns_whole_kernel(
    Group G, int steps, float a, float b, float c, double eps,
    MuonScalars S) {
  // Q, and per group the columns' limbs and its Gram share
  __shared__ __attribute__((aligned(1024)))
  _Float16 lds[8192 * (1 + 2 * kMaxWhole)];
  __shared__ double part[256 * kMaxWhole];
  int z;
  const Mat &M = G.mat[find_mat(G, blockIdx.x, z)];
  const Narrow N = {};
  Slab W;
  const int g = __builtin_amdgcn_readfirstlane(int(threadIdx.x) >> 8);
  const int t256 = threadIdx.x & 255;
  const int chunks = M.np / 64;
  _Float16 *const lq = lds, *const lt = lds + 8192 * (1 + 2 * g);
  _Float16 *const lx = lt + 8192;
  f32x16 x, gram, t;
  double sq = 0.0;
  load_update<MUON, true>(M, N, W, S, z, g, x);
#pragma unroll
  for (int r = 0; r < 16; ++r) sq += double(x[r]) * double(x[r]);
  scale_update(M, W, g,
               limb_scale(block_sum<256 * kMaxWhole>(sq, part), eps), x);
  // (16 M16 rows and, of a chunk, 16 N16 columns are all there are)
  const auto run = [&](auto m16, auto n16) {
    constexpr int M16 = decltype(m16)::value, N16 = decltype(n16)::value;
    for (int step = 1; step <= steps; ++step) {
      // (addresses are worked out anew: there are no registers to keep them)
      asm volatile("" : "+v"(W.lane), "+v"(W.fr));
      clear16(gram);
      if (g < chunks) W.put_columns(lt, x);
      __syncthreads();
      if (g < chunks) W.gram_of<N16>(lt, gram);
      // the groups' shares, in order
      if (chunks > 1) {
        f32x4 *mine = reinterpret_cast<f32x4 *>(lx);
        if (g < chunks) {
#pragma unroll
          for (int q = 0; q < 4; ++q)
            mine[q * 256 + t256] = f32x4{gram[4 * q], gram[4 * q + 1],
                                         gram[4 * q + 2], gram[4 * q + 3]};
        }
        __syncthreads();
        if (g == 0) clear16(gram);
        for (int k = 0; g == 0 && k < chunks; ++k) {
          const f32x4 *other = reinterpret_cast<const f32x4 *>(
              lds + 8192 * (2 + 2 * k));
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const f32x4 v = other[q * 256 + t256];
#pragma unroll
            for (int e = 0; e < 4; ++e)
              gram[4 * q + e] = __fadd_rn(gram[4 * q + e], v[e]);
          }
        }
      }
      // Q by the first group, which others wait for: all of them at it would
      // share the one CU's vector units
      if (g == 0) {
#pragma unroll
        for (int r = 0; r < 16; ++r) gram[r] *= kInvS;
        W.put_columns(lq, gram);
      }
      __syncthreads();
      if (g == 0) {
        clear16(t);
        W.multiply<M16>(lq, lq, t);
#pragma unroll
        for (int r = 0; r < 16; ++r) t[r] = b * gram[r] + c * (t[r] * kInvS);
      }
      __syncthreads();
      if (g == 0) W.put_columns(lq, t);
      __syncthreads();
      if (g < chunks) {
        clear16(t);
        W.multiply<M16>(lq, lt, t);
#pragma unroll
        for (int r = 0; r < 16; ++r) x[r] = a * x[r] + t[r] * kInvS;
      }
      __syncthreads();  // lt and lq have been read
    }
  };
  using One = std::integral_constant<int, 1>;
  using Four = std::integral_constant<int, 4>;
  if (M.n <= 16) run(One(), One());
  else if (M.m <= 16) run(One(), Four());
  else run(Four(), Four());
  if (g < chunks) store_chunk<MUON>(M, W, S, z, g, x);
}

// Launch k of a narrow matrix in slabs: 0 scales the update; k = 1 .. steps
// is step k, the last of which stores the result.
template <bool MUON>
__global__ __launch_bounds__(256) void ns_narrow_kernel(
    Group G, int k, int steps, float a, float b, float c, double eps,
    MuonScalars S) {
  __shared__ __attribute__((aligned(1024))) _Float16 lds[3 * 8192];
  __shared__ double part[256];
  _Float16 *const lq = lds, *const lt = lds + 8192, *const lx = lds + 16384;
  int rel;
  const Mat &M = G.mat[find_mat(G, blockIdx.x, rel)];
  const int slabs = M.slabs;
  const int z = rel / slabs, slab = rel % slabs;
  const int chunk0 = slab * M.each, chunks = M.np / 64;
  const int have = chunks - chunk0 < M.each ? chunks - chunk0 : M.each;
  const Narrow N = narrow_of(M, z);
  const Slab W;
  f32x16 x[kMaxEach];  // kS times the columns
  f32x16 gram, t;
  clear16(gram);
  if (k == 0) {
#pragma unroll
    for (int ch = 0; ch < kMaxEach; ++ch)
      if (ch < have)
        load_update<MUON, false>(M, N, W, S, z, chunk0 + ch, x[ch]);
    const double scale = limb_scale(norm_sum(N.norm, M.nb, part), eps);
#pragma unroll
    for (int ch = 0; ch < kMaxEach; ++ch) {
      if (ch >= have) break;
      scale_update(M, W, chunk0 + ch, scale, x[ch]);
      W.put_columns(lx, x[ch]);
      __syncthreads();
      W.gram_of<4>(lx, gram);
      __syncthreads();
    }
  } else {
#pragma unroll
    for (int ch = 0; ch < kMaxEach; ++ch) {
      if (ch >= have) break;
      const float *p = N.x + (int64_t(chunk0 + ch) * 64 + W.col()) * kNarrow;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const f32x4 v = *reinterpret_cast<const f32x4 *>(p + W.row(q));
#pragma unroll
        for (int e = 0; e < 4; ++e) x[ch][4 * q + e] = v[e];
      }
    }
    // every slab's share of the Gram matrix, in order
    const f32x4 *g = reinterpret_cast<const f32x4 *>(
        N.gram + int64_t((k - 1) & 1) * slabs * kGramElems);
    constexpr int kAhead = 8;
    for (int s0 = 0; s0 < slabs; s0 += kAhead) {
      f32x4 v[kAhead][4];
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (s0 + u < slabs)
            v[u][q] = g[(s0 + u) * (kGramElems / 4) + q * 256 + threadIdx.x];
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        if (s0 + u < slabs) {
#pragma unroll
          for (int r = 0; r < 16; ++r)
            gram[r] = __fadd_rn(gram[r], v[u][r / 4][r % 4]);
        }
    }
    // (16 M16 rows are all there are)
    const auto run = [&](auto m16) {
      constexpr int M16 = decltype(m16)::value;
      // kS Q = b kS A + c kS A^2 from kS^2 A
#pragma unroll
      for (int r = 0; r < 16; ++r) gram[r] *= kInvS;
      W.put_columns(lt, gram);
      __syncthreads();
      clear16(t);
      W.multiply<M16>(lt, lt, t);
#pragma unroll
      for (int r = 0; r < 16; ++r) t[r] = b * gram[r] + c * (t[r] * kInvS);
      W.put_columns(lq, t);
      clear16(gram);
      __syncthreads();
#pragma unroll
      for (int ch = 0; ch < kMaxEach; ++ch) {
        if (ch >= have) break;
        W.put_columns(lt, x[ch]);
        __syncthreads();
        clear16(t);
        W.multiply<M16>(lq, lt, t);
#pragma unroll
        for (int r = 0; r < 16; ++r) x[ch][r] = a * x[ch][r] + t[r] * kInvS;
        if (k < steps) {
          W.put_columns(lx, x[ch]);
          __syncthreads();
          W.gram_of<4>(lx, gram);
        } else {
          __syncthreads();
        }
      }
    };
    if (M.m <= 16) run(std::integral_constant<int, 1>());
    else run(std::integral_constant<int, 4>());
  }
  if (k < steps) {
#pragma unroll
    for (int ch = 0; ch < kMaxEach; ++ch) {
      if (ch >= have) break;
      float *p = N.x + (int64_t(chunk0 + ch) * 64 + W.col()) * kNarrow;
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *reinterpret_cast<f32x4 *>(p + W.row(q)) =
            f32x4{x[ch][4 * q], x[ch][4 * q + 1], x[ch][4 * q + 2],
                  x[ch][4 * q + 3]};
    }
    f32x4 *g = reinterpret_cast<f32x4 *>(
        N.gram + (int64_t(k & 1) * slabs + slab) * kGramElems);
#pragma unroll
    for (int q = 0; q < 4; ++q)
      g[q * 256 + threadIdx.x] = f32x4{gram[4 * q], gram[4 * q + 1],
                                       gram[4 * q + 2], gram[4 * q + 3]};
    return;
  }
#pragma unroll
  for (int ch = 0; ch < kMaxEach; ++ch)
    if (ch < have) store_chunk<MUON>(M, W, S, z, chunk0 + ch, x[ch]);
}

// -- host --------------------------------------------------------------------
// Tiles: 256 x 256 keeps a CU's matrix cores at up to 95 % of what a large
// library product reaches, where there is work for all of them; 128 x 128,
// two workgroups to a CU, is bound by its reads (of LDS, and twice the L2
// traffic), but takes products that leave the last round of large ones too
// empty (below); 64 x 64 is for matrices too small for that, where a tile's
// latency counts.
using BigTile = Tile<256, 256, 128, 64, 2>;
using HalfTile = Tile<128, 128, 64, 64, 2>;
using MidTile = Tile<64, 64, 32, 32, 4>;
// workgroups that the GPU holds: one of a 256 x 256 tile per CU, two of the
// others
constexpr int kBigPlaces = 256, kMidPlaces = 512;
constexpr int kBigSide = 256, kMidSide = 64;

// How an entry is computed: in one launch, by slabs, or by tiled products.
enum Way { kWhole, kNarrowSlabs, kMid, kBig, kWays };

int64_t round_to(int64_t v, int64_t p) { return (v + p - 1) / p * p; }

// Checks the sizes and fills in what does not depend on the other entries.
int size_mat(Mat &M, int64_t rows, int64_t cols, int64_t batch,
             const char *what) {
  if (rows < 0 || cols < 0 || batch < 0) {
    set_error("%s: negative size", what);
    return FSAGG_EINVAL;
  }
  const int64_t m = rows < cols ? rows : cols, n = rows < cols ? cols : rows;
  if (m > FSAGG_NS_MAX_SHORT || n > FSAGG_NS_MAX_LONG ||
      m * n > FSAGG_NS_MAX_ELEMS || batch > 65535) {
    set_error("%s: a %lld x %lld matrix (batch %lld) is outside the limits "
              "(short side %d, long side %d, %d elements, batch 65535)",
              what, (long long)rows, (long long)cols, (long long)batch,
              FSAGG_NS_MAX_SHORT, FSAGG_NS_MAX_LONG, FSAGG_NS_MAX_ELEMS);
    return FSAGG_EINVAL;
  }
  M.rows = int32_t(rows);
  M.cols = int32_t(cols);
  M.batch = int32_t(batch);
  M.m = int32_t(m);
  M.n = int32_t(n);
  // a launch counts its work items in 32 bits: workgroups of the update pass
  // and 64 x 64 tiles of all entries of a group (where one workgroup takes a
  // whole matrix, a batch has few enough)
  if (!(m <= kNarrow && n <= 64 * kMaxWhole) &&
      batch * (round_to(m, kBigSide) / 64) * (round_to(n, kBigSide) / 64) >
          (int64_t(1) << 24) / kMaxGroup) {
    set_error("%s: a batch of %lld %lld x %lld matrices is too large for one "
              "call", what, (long long)batch, (long long)rows,
              (long long)cols);
    return FSAGG_EINVAL;
  }
  return FSAGG_OK;
}

bool empty(const Mat &M) { return M.m == 0 || M.batch == 0; }

// What big tiles gain over 64 x 64 ones, in multiplications of an m x m by an
// m x n matrix: 7 of the entry's own to 4 of its padded one, less what the
// shorter pipelines of small tiles save (kBigGain, for all of the group).
// Fitted to both sides of 35 shapes; big against small tiles, us:
// 512 x 16384 594 / 559, 512 x 32768 941 / 1022, 1024 x 4096 573 / 488,
// 1024 x 8192 807 / 875, 1280 x 2560 677 / 518, 1280 x 5120 860 / 907,
// 2048 x 2048 917 / 942, 2 x (1500 x 1500) 807 / 909, 12 x (1024 x 1024)
// 1018 / 1335; a short side of 384 loses at any length (384 x 32768 879 /
// 682).
constexpr int kBigShort = 512;
constexpr int64_t kBigGain = 17500000000;
int64_t big_gain(const Mat &M) {
  if (empty(M) || M.m < kBigShort) return 0;
  const int64_t m = M.m, n = M.n, mp = round_to(m, kBigSide),
                np = round_to(n, kBigSide);
  const int64_t gain = 7 * (m * m * n) - 4 * (mp * mp * np);
  return gain > 0 ? gain * M.batch : 0;
}

Way way_of(const Mat &M, int64_t gain) {
  // narrow against 64 x 64 tiles, us: 50 x 1024 53 / 87, 50 x 16384 150 / 199
  if (M.m <= kNarrow && M.n <= kNarrowLong)
    return M.n <= 64 * kMaxWhole ? kWhole : kNarrowSlabs;
  return big_gain(M) > 0 && gain >= kBigGain ? kBig : kMid;
}

// The derived fields of an entry computed that way.
void plan_mat(Mat &M, Way way) {
  const int64_t total = int64_t(M.rows) * M.cols;
  int64_t bytes;
  M.slabs = M.each = 1;
  // update workgroups of a matrix: 4 elements a thread while all of the batch
  // are few, else 16 (no more of them than of 64 x 64 tiles)
  const auto blocks = [&](int64_t each) {
    const int64_t nb = (total + each - 1) / each;
    return int32_t(nb > kMaxNorm ? kMaxNorm : nb);
  };
  M.nb = blocks(4 * kNormBlock);
  if (int64_t(M.batch) * M.nb > 8 * kMaxNorm) M.nb = blocks(16 * kNormBlock);
  if (way == kWhole || way == kNarrowSlabs) {
    M.mp = kNarrow;
    M.np = int32_t(round_to(M.n, 64));
    const int chunks = M.np / 64;
    // a launch reads 16 KiB of Gram shares per slab into every workgroup,
    // and works its chunks one after the other: 8 slabs' shares cost about
    // what a chunk does (1 / 2 / 4 chunks a slab, us: 50 x 1500 62 / 64 / -,
    // 50 x 1984 70 / 67 / -, 50 x 4096 106 / 85 / 95, 50 x 8192 178 / - / 113)
    M.each = way == kWhole ? 1 : chunks <= 28 ? 1 : chunks <= 96 ? 2 : 4;
    M.slabs = (chunks + M.each - 1) / M.each;
    bytes = way == kWhole ? 0
                          : 8 * kMaxNorm +
                                4 * (int64_t(M.np) * kNarrow +
                                     2 * int64_t(M.slabs) * kGramElems +
                                     total);
  } else {
    const int side = way == kMid ? kMidSide : kBigSide;
    M.mp = int32_t(round_to(M.m, side));
    M.np = int32_t(round_to(M.n, side));
    bytes = ws_bytes_of(M.mp, M.np);
  }
  M.wstride = round_to(bytes, 1024);
}

// Parts that the workgroups of one product may leave.
int64_t partial_bytes(Way way) {
  switch (way) {
    case kBig:
      return int64_t(2) * kBigPlaces * kBigSide * kBigSide * 4;
    case kMid:
      return int64_t(2) * kMidPlaces * kMidSide * kMidSide * 4;
    default:
      return 0;
  }
}

// The largest |x|, |x|^2 and |q| that the iteration's limbs have to hold,
// from the scalar iteration on the interval of the singular values, [0, 1] at
// the start: all have to stay under 2^16 / 2^12.  (In closed form: a grid of
// 4096 points took the host 72 us a call.)
bool coefficients_fit(double a, double b, double c, int steps) {
  if (!std::isfinite(a) || !std::isfinite(b) || !std::isfinite(c))
    return false;
  double hi = 1.0;  // bound on the singular values entering the step
  for (int s = 0; s < steps; ++s) {
    // With l = x^2 in [0, hi^2]: q = b l + c l^2 turns at l = -b / 2c, and
    // x (a + q) where a + 3 b l + 5 c l^2 = 0.
    const double end = hi * hi;
    if (!(end <= 15.0)) return false;
    const auto q = [&](double l) { return std::fabs(b * l + c * l * l); };
    const auto p = [&](double l) {
      return std::sqrt(l) * std::fabs(a + b * l + c * l * l);
    };
    const auto inside = [&](double l) { return l > 0.0 && l < end; };
    double top = q(end), next = p(end);
    if (c != 0.0) {
      if (inside(-b / (2 * c))) top = std::fmax(top, q(-b / (2 * c)));
      const double d = 9 * b * b - 20 * a * c;
      if (d >= 0.0)
        for (const double r : {std::sqrt(d), -std::sqrt(d)})
          if (inside((r - 3 * b) / (10 * c)))
            next = std::fmax(next, p((r - 3 * b) / (10 * c)));
    } else if (b != 0.0 && inside(-a / (3 * b))) {
      next = std::fmax(next, p(-a / (3 * b)));
    }
    hi = next * (1.0 + 1.0 / 1024);  // what the step's own rounding may add
    if (!(top <= 15.0 && hi <= 15.0)) return false;
  }
  return true;
}

struct Step {
  float a, b, c;
  double eps;
  int steps;
  MuonScalars S;
  hipStream_t stream;
};

// The tiles of a group's product, its stages, and those of the longest tile.
struct Count {
  int64_t tiles = 0, stages = 0;
  int longest = 0;
};
template <class T, int MODE>
Count count_tiles(const Group &G) {
  Count c;
  for (int i = 0; i < G.nmat; ++i) {
    const Mat &M = G.mat[i];
    const int64_t t = int64_t(M.batch) * mode_tiles<MODE, T::kBM, T::kBN>(M);
    c.tiles += t;
    c.stages += t * mode_stages<MODE>(M);
    if (mode_stages<MODE>(M) > c.longest) c.longest = mode_stages<MODE>(M);
  }
  return c;
}

// Sets the entries' first workgroups (a workgroup per tile) or first stages.
template <class T, int MODE>
int place_tiles(Group &G, bool share) {
  int total = 0;
  for (int i = 0; i < G.nmat; ++i) {
    const Mat &M = G.mat[i];
    G.start[i] = total;
    total += M.batch * mode_tiles<MODE, T::kBM, T::kBN>(M) *
             (share ? mode_stages<MODE>(M) : 1);
  }
  G.start[G.nmat] = total;
  return total;
}

template <class T, int MODE>
void launch_whole(Group &G, int src, const Step &st) {
  const int total = place_tiles<T, MODE>(G, false);
  hipLaunchKernelGGL((ns_gemm_kernel<T, MODE>), dim3(total),
                     dim3(T::kThreads), 0, st.stream, G, src, st.a, st.b,
                     st.c, st.S);
}

// One product of the whole group: one workgroup per tile, of either size, or
// the line of stages shared by as many workgroups as the GPU holds (`places`),
// each with at least kMinStages of them.  Whole tiles leave places idle in
// the last round; sharing fills them, but its workgroups walk the operands
// at different stages, so less of what they read is in the caches, and a join
// writes parts and reads them again.  What is expected to take least is
// taken, by times fitted to some 30 shapes with either way measured
// (us: A of 4096 x 4096 whole 251, shared 276, halved 284; A of 2048 x 3136
// 175 / 70 / 87; QX there 136 / 112 / 91; A^2 of 12 matrices of 1024 79 / 89 /
// 54; 64 x 64 tiles, A of 1000 x 1000 12 / 20, of 512 x 3136 31 / 21):
//   s0, s1  a stage, with none of the places taken and what all add (clocks
//           and caches are shared; half of it grows with the square),
//   e0, e1  a tile's end, as much,
//   l0, l1  a stage of the line,  j0, j1  the join;  kPart each part of a tile.
struct Cost {
  double s0, s1, e0, e1, l0, l1, j0, j1;
};
template <class T>
constexpr Cost cost_of() {
  if (T::kBM == 256)
    return Cost{1.5, 0.9, 7, 20, 1.8, 1.6, 8, 22};
  if (T::kBM == 128) return Cost{0.65, 0.75, 4, 9, 0, 0, 0, 0};
  return Cost{0.25, 0.31, 4, 4, 0.3, 0.4, 8, 8};
}
constexpr int kMinStages = 8;
constexpr double kPart = 0.3;

double whole_time(const Count &n, int places, const Cost &c) {
  const auto round = [&](double f, double stages) {
    return stages * (c.s0 + c.s1 * (f + f * f) / 2) + c.e0 + c.e1 * f;
  };
  const double each = double(n.stages) / double(n.tiles);
  const int64_t left = n.tiles % places;
  const double t = double(n.tiles / places) * round(1.0, each) +
                   (left ? round(double(left) / places, each) : 0.0);
  const double most =
      round(n.tiles < places ? double(n.tiles) / places : 1.0, n.longest);
  return t > most ? t : most;
}
double line_time(const Count &n, int64_t workers, int places, const Cost &c) {
  const double f = double(workers) / places,
               each = double(n.stages) / double(workers);
  return each * (c.l0 + c.l1 * f) + c.j0 + c.j1 * f +
         double(n.tiles / workers) * (c.e0 + c.e1) +
         kPart * double(n.longest) / each;
}

template <class T, int MODE, class H = void>
void launch_product(Group &G, int places, float *partial, int src,
                    const Step &st) {
  const Count n = count_tiles<T, MODE>(G);
  int64_t w = n.stages / kMinStages;
  if (w > places) w = places;
  const double whole = whole_time(n, places, cost_of<T>());
  const double line =
      w > 1 ? line_time(n, w, places, cost_of<T>()) : whole;
  if constexpr (!std::is_void<H>::value) {
    const double half =
        whole_time(count_tiles<H, MODE>(G), 2 * places, cost_of<H>());
    if (half < whole && half < line) {
      launch_whole<H, MODE>(G, src, st);
      return;
    }
  }
  if (whole <= line) {
    launch_whole<T, MODE>(G, src, st);
    return;
  }
  Line L;
  L.workers = int(w);
  L.partial = partial;
  const int total = place_tiles<T, MODE>(G, true);
  L.each = total / L.workers;
  L.more = total % L.workers;
  hipLaunchKernelGGL((ns_line_kernel<T, MODE>), dim3(L.workers),
                     dim3(T::kThreads), 0, st.stream, G, L, src, st.a, st.b,
                     st.c, st.S);
  hipLaunchKernelGGL((ns_join_kernel<T, MODE>),
                     dim3(L.workers - 1, T::MI * T::NJ), dim3(T::kThreads), 0,
                     st.stream, G, L, src, st.a, st.b, st.c, st.S);
}

template <class T, bool MUON, class H = void>
void run_products(Group &G, int places, float *partial, const Step &st) {
  int total = 0;
  for (int i = 0; i < G.nmat; ++i) {
    G.start[i] = total;
    total += G.mat[i].batch * G.mat[i].nb;
  }
  G.start[G.nmat] = total;
  hipLaunchKernelGGL((ns_update_kernel<MUON, false>), dim3(total),
                     dim3(kNormBlock), 0, st.stream, G, st.S);
  total = 0;
  for (int i = 0; i < G.nmat; ++i) {
    G.start[i] = total;
    total += G.mat[i].batch * (G.mat[i].mp / 64) * (G.mat[i].np / 64);
  }
  G.start[G.nmat] = total;
  hipLaunchKernelGGL(ns_prepare_kernel, dim3(total), dim3(256), 0, st.stream,
                     G, st.eps);
  int src = 0;
  for (int k = 0; k < st.steps; ++k, src ^= 1) {
    launch_product<T, kGram, H>(G, places, partial, src, st);
    launch_product<T, kSquare, H>(G, places, partial, src, st);
    if (k + 1 < st.steps)
      launch_product<T, kApply, H>(G, places, partial, src, st);
    else
      launch_product<T, MUON ? kLastMuon : kLast, H>(G, places, partial, src,
                                                     st);
  }
}

template <bool MUON>
void run_narrow(Group &G, const Step &st) {
  int total = 0;
  for (int i = 0; i < G.nmat; ++i) {
    G.start[i] = total;
    total += G.mat[i].batch * G.mat[i].nb;
  }
  G.start[G.nmat] = total;
  hipLaunchKernelGGL((ns_update_kernel<MUON, true>), dim3(total),
                     dim3(kNormBlock), 0, st.stream, G, st.S);
  total = 0;
  for (int i = 0; i < G.nmat; ++i) {
    G.start[i] = total;
    total += G.mat[i].batch * G.mat[i].slabs;
  }
  G.start[G.nmat] = total;
  for (int k = 0; k <= st.steps; ++k)
    hipLaunchKernelGGL(ns_narrow_kernel<MUON>, dim3(total), dim3(256), 0,
                       st.stream, G, k, st.steps, st.a, st.b, st.c, st.eps,
                       st.S);
}

template <bool MUON>
void run_whole(Group &G, const Step &st) {
  int total = 0;
  for (int i = 0; i < G.nmat; ++i) {
    G.start[i] = total;
    total += G.mat[i].batch;
  }
  G.start[G.nmat] = total;
  hipLaunchKernelGGL(ns_whole_kernel<MUON>, dim3(total),
                     dim3(256 * kMaxWhole), 0, st.stream, G, st.steps, st.a,
                     st.b, st.c, st.eps, st.S);
}

template <bool MUON>
void run_group(Group &G, Way way, float *partial, const Step &st) {
  if (way == kWhole) run_whole<MUON>(G, st);
  else if (way == kNarrowSlabs) run_narrow<MUON>(G, st);
  else if (way == kMid)
    run_products<MidTile, MUON>(G, kMidPlaces, partial, st);
  else
    run_products<BigTile, MUON, HalfTile>(G, kBigPlaces, partial, st);
}

// f(group, way, bytes of its entries) for every group of entries, in turn;
// entries of one way go together.  `fill(i, M)` sets entry i's sizes, types
// and pointers.
template <typename Fill, typename F>
int each_group(int nmat, Fill fill, Group &G, F f) {
  int64_t gain = 0;
  for (int i = 0; i < nmat; ++i) {
    Mat M;
    const int rc = fill(i, M);
    if (rc != FSAGG_OK) return rc;
    gain += big_gain(M);
  }
  for (int way = 0; way < kWays; ++way) {
    G.nmat = 0;
    size_t bytes = 0;
    for (int i = 0; i < nmat; ++i) {
      Mat &M = G.mat[G.nmat];
      fill(i, M);
      if (empty(M) || way_of(M, gain) != way) continue;
      plan_mat(M, Way(way));
      bytes += size_t(M.wstride) * M.batch;
      if (++G.nmat == kMaxGroup) {
        f(G, Way(way), bytes);
        G.nmat = 0;
        bytes = 0;
      }
    }
    if (G.nmat) f(G, Way(way), bytes);
  }
  return FSAGG_OK;
}

// The groups run one after the other, so they share the workspace.
template <typename Fill>
int workspace_of(int nmat, Fill fill, size_t &need) {
  Group G;
  need = 0;
  return each_group(nmat, fill, G, [&](Group &, Way way, size_t bytes) {
    const size_t b = bytes + partial_bytes(way);
    if (b > need) need = b;
  });
}

template <typename Fill>
bool nothing(int nmat, Fill fill) {
  for (int i = 0; i < nmat; ++i) {
    Mat M;
    fill(i, M);
    if (!empty(M)) return false;
  }
  return true;
}

// What a call may be refused for, its sizes, pointers and workspace apart.
int check_settings(int steps, const double *coef, double eps,
                   const char *what) {
  if (steps < 1 || steps > 99) {
    set_error("%s: steps must be in [1, 99], got %d", what, steps);
    return FSAGG_EINVAL;
  }
  if (!(eps > 0.0) || !std::isfinite(eps)) {
    set_error("%s: eps must be positive and finite", what);
    return FSAGG_EINVAL;
  }
  if (!coef || !coefficients_fit(coef[0], coef[1], coef[2], steps)) {
    set_error("%s: these coefficients let the iterates grow past what the "
              "limbs hold", what);
    return FSAGG_EINVAL;
  }
  return FSAGG_OK;
}

template <bool MUON, typename Fill>
int run_all(int nmat, Fill fill, int steps, const double *coef, double eps,
            const MuonScalars &S, void *ws, size_t ws_bytes,
            hipStream_t stream, const char *what) {
  int rc = check_settings(steps, coef, eps, what);
  if (rc != FSAGG_OK) return rc;
  // everything is checked before anything is launched
  size_t need = 0;
  rc = workspace_of(nmat, fill, need);
  if (rc != FSAGG_OK) return rc;
  if (need > 0 && (!ws || ws_bytes < need)) {
    set_error("%s: workspace of %zu bytes, %zu needed", what,
              ws ? ws_bytes : size_t(0), need);
    return FSAGG_ESPACE;
  }
  if (!aligned16(ws)) {
    set_error("%s: workspace must be 16-byte aligned", what);
    return FSAGG_EINVAL;
  }
  if (need == 0 && nothing(nmat, fill)) return FSAGG_OK;
  // (the norm of an fp32 matrix is zero or over 1e-45, so a divisor below
  // 1e-300 meets zeros only; kS / eps has to stay finite for them)
  const double least = eps > 1e-300 ? eps : 1e-300;
  const Step st = {float(coef[0]), float(coef[1]), float(coef[2]), least,
                   steps,          S,              stream};
  Group G;
  each_group(nmat, fill, G, [&](Group &g, Way way, size_t bytes) {
    char *at = static_cast<char *>(ws);
    for (int i = 0; i < g.nmat; ++i) {
      g.mat[i].ws = at;
      at += size_t(g.mat[i].wstride) * g.mat[i].batch;
    }
    run_group<MUON>(g, way,
                    reinterpret_cast<float *>(static_cast<char *>(ws) + bytes),
                    st);
  });
  return check_launch(what);
}

bool float_dtype(int dt) {
  return dt == FSAGG_F32 || dt == FSAGG_F16 || dt == FSAGG_BF16;
}

// Entry i of either table: sizes and types, and (for a run) its pointers.
auto ns_fill(const fsagg_ns_mat *mats, bool pointers, const char *what) {
  return [=](int i, Mat &M) {
    const fsagg_ns_mat &d = mats[i];
    const int rc = size_mat(M, d.rows, d.cols, d.batch, what);
    if (rc != FSAGG_OK) return rc;
    if (!float_dtype(d.dtype) || !float_dtype(d.out_dtype) ||
        (pointers && !empty(M) && (!d.g || !d.out))) {
      set_error("%s: matrix %d: null pointer or unknown dtype", what, i);
      return int(FSAGG_EINVAL);
    }
    M.g = d.g;
    M.out = d.out;
    M.vec = aligned16(d.out) && d.cols % 8 == 0;
    M.buf = nullptr;
    M.ws = nullptr;
    M.sz = d.batch_stride;
    M.si = d.row_stride;
    M.sj = d.col_stride;
    M.dt = int16_t(d.dtype);
    M.odt = int16_t(d.out_dtype);
    return int(FSAGG_OK);
  };
}

auto muon_fill(const fsagg_muon_mat *mats, bool pointers, const char *what) {
  return [=](int i, Mat &M) {
    const fsagg_muon_mat &d = mats[i];
    const int rc = size_mat(M, d.rows, d.cols, 1, what);
    if (rc != FSAGG_OK) return rc;
    if (pointers && !empty(M) && (!d.param || !d.avg || !d.momentum)) {
      set_error("%s: matrix %d: null pointer", what, i);
      return int(FSAGG_EINVAL);
    }
    M.g = d.avg;
    M.out = d.param;
    M.vec = aligned16(d.param) && d.cols % 8 == 0;
    M.buf = d.momentum;
    M.ws = nullptr;
    M.sz = M.si = M.sj = 0;
    M.dt = M.odt = FSAGG_F32;
    return int(FSAGG_OK);
  };
}

}  // namespace
}  // namespace fsagg

using namespace fsagg;

extern "C" size_t fsagg_newton_schulz_workspace_bytes(
    const fsagg_ns_mat *mats, int nmat) {
  const char *what = "fsagg_newton_schulz_workspace_bytes";
  size_t need = 0;
  if (nmat <= 0 || !mats ||
      workspace_of(nmat, ns_fill(mats, false, what), need) != FSAGG_OK)
    return 0;
  return need;
}

extern "C" int fsagg_newton_schulz(const fsagg_ns_mat *mats, int nmat,
                                   int steps, const double *coefficients,
                                   double eps, void *workspace,
                                   size_t workspace_bytes,
                                   fsagg_stream_t stream) {
  const char *what = "fsagg_newton_schulz";
  if (nmat < 0 || (nmat > 0 && !mats)) {
    set_error("%s: invalid argument", what);
    return FSAGG_EINVAL;
  }
  return run_all<false>(nmat, ns_fill(mats, true, what), steps, coefficients,
                        eps, MuonScalars{}, workspace, workspace_bytes,
                        as_stream(stream), what);
}

extern "C" size_t fsagg_muon_workspace_bytes(const fsagg_muon_mat *mats,
                                             int nmat) {
  const char *what = "fsagg_muon_workspace_bytes";
  size_t need = 0;
  if (nmat <= 0 || !mats ||
      workspace_of(nmat, muon_fill(mats, false, what), need) != FSAGG_OK)
    return 0;
  return need;
}

namespace {
// the arguments that both calls below take
int muon_arguments(const fsagg_muon_mat *mats, int nmat,
                   const fsagg_muon_params *hp, const char *what) {
  if (nmat < 0 || (nmat > 0 && !mats) || !hp) {
    set_error("%s: invalid argument", what);
    return FSAGG_EINVAL;
  }
  if (hp->adjust != FSAGG_MUON_ORIGINAL &&
      hp->adjust != FSAGG_MUON_MATCH_RMS) {
    set_error("%s: unknown learning-rate adjustment %d", what, hp->adjust);
    return FSAGG_EINVAL;
  }
  return FSAGG_OK;
}
}  // namespace

extern "C" int fsagg_muon_check(const fsagg_muon_mat *mats, int nmat,
                                const fsagg_muon_params *hp) {
  const char *what = "fsagg_muon_check";
  int rc = muon_arguments(mats, nmat, hp, what);
  if (rc != FSAGG_OK) return rc;
  const double coef[3] = {hp->a, hp->b, hp->c};
  rc = check_settings(hp->steps, coef, hp->eps, what);
  if (rc != FSAGG_OK) return rc;
  size_t need = 0;
  return workspace_of(nmat, muon_fill(mats, false, what), need);
}

extern "C" int fsagg_muon_step_f32(const fsagg_muon_mat *mats, int nmat,
                                   const fsagg_muon_params *hp,
                                   void *workspace, size_t workspace_bytes,
                                   fsagg_stream_t stream) {
  const char *what = "fsagg_muon_step_f32";
  const int rc = muon_arguments(mats, nmat, hp, what);
  if (rc != FSAGG_OK) return rc;
  MuonScalars S;
  S.keep = float(1.0 - hp->momentum);
  S.mu = float(hp->momentum);
  S.lr = float(hp->lr);
  S.decay = float(1.0 - hp->lr * hp->weight_decay);
  S.nesterov = hp->nesterov;
  S.maximize = hp->maximize;
  S.adjust = hp->adjust;
  const double coef[3] = {hp->a, hp->b, hp->c};
  return run_all<true>(nmat, muon_fill(mats, true, what), hp->steps, coef,
                       hp->eps, S, workspace, workspace_bytes,
                       as_stream(stream), what);
}
