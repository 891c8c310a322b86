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
//
// Every product is C = P R^T with both operands contiguous along k, so X is
// kept as X (for A) and as T = X^T (for QX); A and Q are symmetric: the
// tiles on and above the diagonal are computed and stored twice.
#include "common.h"

#include <hip/hip_fp16.h>

#include <cmath>

namespace fsagg {
namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kMaxGroup = 24;     // matrices per launch (kernel arguments)
constexpr int kNormBlock = 256;
constexpr int kNormElems = 8192;  // update elements per norm workgroup
constexpr int kMaxNorm = 256;     // norm workgroups per matrix
constexpr int kPad = 128;         // workspace sides are multiples of this
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
  int16_t dt, odt;
};

// Workspace of one matrix: X limbs, T limbs twice (a step reads one and
// writes the other), A limbs, Q limbs, norm partials.  The fp32 update lies
// in the second T until the first step writes it.
struct Planes {
  _Float16 *xh, *xl, *t, *ah, *al, *qh, *ql;
  int64_t e;
  double *norm;
  // (selected by arithmetic: an array indexed at run time would live in
  // scratch memory)
  __device__ __forceinline__ _Float16 *th(int k) const {
    return t + 2 * k * e;
  }
  __device__ __forceinline__ _Float16 *tl(int k) const {
    return t + (2 * k + 1) * e;
  }
};

__host__ __device__ inline int64_t ws_elems(int64_t mp, int64_t np) {
  return 6 * mp * np + 4 * mp * mp;
}
__host__ __device__ inline int64_t ws_bytes_of(int64_t mp, int64_t np) {
  return 2 * ws_elems(mp, np) + 8 * kMaxNorm;
}
__device__ __forceinline__ Planes planes_of(const Mat &M, int z) {
  _Float16 *p = reinterpret_cast<_Float16 *>(M.ws + z * M.wstride);
  const int64_t e = int64_t(M.mp) * M.np, s = int64_t(M.mp) * M.mp;
  Planes P;
  P.xh = p;
  P.xl = p + e;
  P.t = p + 2 * e;
  P.e = e;
  P.ah = p + 6 * e;
  P.al = P.ah + s;
  P.qh = P.ah + 2 * s;
  P.ql = P.ah + 3 * s;
  P.norm = reinterpret_cast<double *>(P.ah + 4 * s);
  return P;
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

__device__ __forceinline__ float load_as_f32(const void *p, int64_t i,
                                             int dt) {
  if (dt == FSAGG_F32) return static_cast<const float *>(p)[i];
  if (dt == FSAGG_F16)
    return float(static_cast<const _Float16 *>(p)[i]);
  return __uint_as_float(uint32_t(static_cast<const uint16_t *>(p)[i]) << 16);
}

// round to nearest even, NaN kept (quieted)
__device__ __forceinline__ uint16_t to_bf16(float v) {
  const uint32_t u = __float_as_uint(v);
  if ((u & 0x7FFFFFFFu) > 0x7F800000u) return uint16_t((u >> 16) | 0x40u);
  return uint16_t((u + 0x7FFFu + ((u >> 16) & 1u)) >> 16);
}

__device__ __forceinline__ void store_from_f32(void *p, int64_t i, int dt,
                                               float v) {
  if (dt == FSAGG_F32) static_cast<float *>(p)[i] = v;
  else if (dt == FSAGG_F16) static_cast<_Float16 *>(p)[i] = _Float16(v);
  else static_cast<uint16_t *>(p)[i] = to_bf16(v);
}

__device__ __forceinline__ void split(float v, _Float16 &h, _Float16 &l) {
  h = _Float16(v);
  l = _Float16(v - float(h));
}

// Pass 1: the fp32 update u, rows x cols contiguous, and a workgroup's sum
// of u^2 in fp64 (squares of fp32 neither overflow nor vanish there).
//   MUON: g = p - avg (negated for maximize); buf += (1 - mu)(g - buf);
//         u = nesterov ? g + mu (buf - g) : buf.
template <bool MUON>
__global__ __launch_bounds__(kNormBlock) void ns_update_kernel(
    Group G, MuonScalars S) {
  int rel;
  const Mat &M = G.mat[find_mat(G, blockIdx.x, rel)];
  const int z = rel / M.nb, b = rel % M.nb;
  const Planes P = planes_of(M, z);
  float *u = reinterpret_cast<float *>(P.th(1));
  const int64_t total = int64_t(M.rows) * M.cols;
  double sq = 0.0;
  for (int64_t e = int64_t(b) * kNormBlock + threadIdx.x; e < total;
       e += int64_t(M.nb) * kNormBlock) {
    float v;
    if constexpr (MUON) {
      const float p = static_cast<const float *>(M.out)[e];
      float g = __fsub_rn(p, static_cast<const float *>(M.g)[e]);
      if (S.maximize) g = -g;
      const float o = M.buf[e];
      // the torch.lerp forms: exact at both ends (mu = 0 gives g)
      const float d = __fsub_rn(g, o);
      const float n = S.keep < 0.5f
                          ? __builtin_fmaf(S.keep, d, o)
                          : __fsub_rn(g, __fmul_rn(d, 1.0f - S.keep));
      M.buf[e] = n;
      v = S.nesterov ? __builtin_fmaf(S.mu, __fsub_rn(n, g), g) : n;
    } else {
      const int64_t i = e / M.cols, j = e - i * M.cols;
      v = load_as_f32(M.g, z * M.sz + i * M.si + j * M.sj, M.dt);
    }
    u[e] = v;
    sq += double(v) * double(v);
  }
  __shared__ double part[kNormBlock];
  part[threadIdx.x] = sq;
  __syncthreads();
  for (int s = kNormBlock / 2; s > 0; s >>= 1) {
    if (int(threadIdx.x) < s) part[threadIdx.x] += part[threadIdx.x + s];
    __syncthreads();
  }
  if (threadIdx.x == 0) P.norm[b] = part[0];
}

// Pass 2: X and T limbs of u / max(|u|, eps), zero in the padding.  One
// workgroup per 64 x 64 tile of the padded m x n orientation; the tile goes
// through LDS so that both orientations are written in rows.
__global__ __launch_bounds__(256) void ns_prepare_kernel(Group G,
                                                         double eps) {
  int rel;
  const Mat &M = G.mat[find_mat(G, blockIdx.x, rel)];
  const int tn = M.np / 64, tiles = (M.mp / 64) * tn;
  const int z = rel / tiles, t = rel % tiles;
  const Planes P = planes_of(M, z);
  const float *u = reinterpret_cast<const float *>(P.th(1));
  __shared__ double part[256];
  __shared__ float tile[64][65];
  part[threadIdx.x] = int(threadIdx.x) < M.nb ? P.norm[threadIdx.x] : 0.0;
  __syncthreads();
  for (int s = 128; s > 0; s >>= 1) {
    if (int(threadIdx.x) < s) part[threadIdx.x] += part[threadIdx.x + s];
    __syncthreads();
  }
  const double norm = sqrt(part[0]);
  // NaN norm: every value becomes NaN, as dividing by it would
  const double scale = double(kS) / (norm < eps ? eps : norm);
  const int i0 = (t / tn) * 64, j0 = (t % tn) * 64;
  const bool tall = M.rows > M.cols;
  // u's own rows r and columns c of this tile
  const int r0 = tall ? j0 : i0, c0 = tall ? i0 : j0;
  for (int k = threadIdx.x; k < 64 * 64; k += 256) {
    const int r = k / 64, c = k % 64;
    float v = 0.0f;
    if (r0 + r < M.rows && c0 + c < M.cols)
      v = float(double(u[int64_t(r0 + r) * M.cols + c0 + c]) * scale);
    if (tall) tile[c][r] = v;
    else tile[r][c] = v;
  }
  __syncthreads();
  for (int k = threadIdx.x; k < 64 * 64; k += 256) {
    const int r = k / 64, c = k % 64;
    _Float16 h, l;
    split(tile[r][c], h, l);
    const int64_t x = int64_t(i0 + r) * M.np + j0 + c;
    P.xh[x] = h;
    P.xl[x] = l;
    split(tile[c][r], h, l);
    const int64_t y = int64_t(j0 + r) * M.mp + i0 + c;
    P.th(0)[y] = h;
    P.tl(0)[y] = l;
  }
}

enum Mode { kGram, kSquare, kApply, kLast, kLastMuon };

// One BM x BN tile of C = P R^T (k contiguous in both) in limbs, 4 waves of
// WM x WN.  A stage is kBK of k of both operands' limbs, written to LDS by
// 16-byte direct loads: 64-byte rows, the four 16-byte slots of row r
// permuted by (r / 4) % 4 so that a fragment read of 16 rows touches all 64
// banks once.  Two stages: one is loaded while the other is multiplied.
//
// Rows and columns of the padding are zero in every plane (the prepare pass
// writes them, products of zero rows are zero), so no tile is ragged inside
// the workspace; only the last step checks its stores against the matrix.
template <int BM, int BN, int WM, int WN, int MODE>
__global__ __launch_bounds__((BM / WM) * (BN / WN) * 64) void ns_gemm_kernel(
    Group G, int src, float b, float c, float a, MuonScalars S) {
  constexpr int kWaves = (BM / WM) * (BN / WN);
  constexpr int kLoads = (BM + BN) * 2 * kBK * 2 / 1024;  // 1 KiB each
  constexpr int kPer = kLoads / kWaves;
  static_assert(kPer * kWaves == kLoads, "loads divide over the waves");
  constexpr int MI = WM / 32, NJ = WN / 32;
  constexpr int kStage = (BM + BN) * 2 * kBK;  // halfs
  __shared__ __attribute__((aligned(1024))) _Float16 lds[2 * kStage];

  int rel;
  const Mat &M = G.mat[find_mat(G, blockIdx.x, rel)];
  const int tm = M.mp / BM;
  int z, ti, tj;
  if constexpr (MODE == kGram || MODE == kSquare) {
    static_assert(BM == BN || (MODE != kGram && MODE != kSquare),
                  "square tiles of a symmetric product");
    const int tiles = tm * (tm + 1) / 2;
    z = rel / tiles;
    int t = rel % tiles;
    ti = 0;
    while (t >= tm - ti) {
      t -= tm - ti;
      ++ti;
    }
    tj = ti + t;
  } else {
    const int tn = M.np / BN, tiles = tm * tn;
    z = rel / tiles;
    const int t = rel % tiles;
    ti = t % tm;
    tj = t / tm;
  }
  const Planes P = planes_of(M, z);
  const _Float16 *ph, *pl, *rh, *rl;
  int ld, K;
  if constexpr (MODE == kGram) {
    ph = rh = P.xh;
    pl = rl = P.xl;
    ld = K = M.np;
  } else if constexpr (MODE == kSquare) {
    ph = rh = P.ah;
    pl = rl = P.al;
    ld = K = M.mp;
  } else {
    ph = P.qh;
    pl = P.ql;
    rh = P.th(src);
    rl = P.tl(src);
    ld = K = M.mp;
  }
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) >> 6);
  const int i0 = ti * BM, j0 = tj * BN;

  // this wave's loads of a stage: LDS order is [P.h][P.l][R.h][R.l] rows of
  // 64 bytes, 16 rows per instruction
  const _Float16 *gsrc[kPer];
  int ldst[kPer];
#pragma unroll
  for (int q = 0; q < kPer; ++q) {
    const int k = wave * kPer + q;
    const int row16 = k * 16;
    const bool right = row16 >= 2 * BM;
    const int in = right ? row16 - 2 * BM : row16;
    const int side = right ? BN : BM;
    const _Float16 *base =
        in < side ? (right ? rh : ph) : (right ? rl : pl);
    const int g0 = (right ? j0 : i0) + (in < side ? in : in - side);
    const int r = lane >> 2, slot = (lane & 3) ^ ((r >> 2) & 3);
    gsrc[q] = base + int64_t(g0 + r) * ld + slot * 8;
    ldst[q] = row16 * kBK;
  }
  auto issue = [&](int k0, int buf) {
#pragma unroll
    for (int q = 0; q < kPer; ++q)
      __builtin_amdgcn_global_load_lds(
          (__attribute__((address_space(1))) void *)(gsrc[q] + k0),
          (__attribute__((address_space(3))) void *)(uintptr_t)(
              lds + buf * kStage + ldst[q]),
          16, 0, 0);
  };

  const int wm = (wave % (BM / WM)) * WM, wn = (wave / (BM / WM)) * WN;
  const int fr = lane & 31, fk = lane >> 5;
  f32x16 acc[MI][NJ];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;

  issue(0, 0);
  for (int k0 = 0, buf = 0; k0 < K; k0 += kBK, buf ^= 1) {
    // this stage has landed for every wave, and the other is read out
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (k0 + kBK < K) issue(k0 + kBK, buf ^ 1);
    const _Float16 *st = lds + buf * kStage;
#pragma unroll
    for (int kk = 0; kk < kBK / 16; ++kk) {
      half8 fah[MI], fal[MI], fbh[NJ], fbl[NJ];
#pragma unroll
      for (int i = 0; i < MI; ++i) {
        const int r = wm + i * 32 + fr;
        const int o = r * kBK + (((kk * 2 + fk) ^ ((r >> 2) & 3)) * 8);
        fah[i] = *reinterpret_cast<const half8 *>(st + o);
        fal[i] = *reinterpret_cast<const half8 *>(st + BM * kBK + o);
      }
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const int r = wn + j * 32 + fr;
        const int o = r * kBK + (((kk * 2 + fk) ^ ((r >> 2) & 3)) * 8);
        fbh[j] = *reinterpret_cast<const half8 *>(st + 2 * BM * kBK + o);
        fbl[j] =
            *reinterpret_cast<const half8 *>(st + (2 * BM + BN) * kBK + o);
      }
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(
              fal[i], fbh[j], acc[i][j], 0, 0, 0);
          acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(
              fah[i], fbl[j], acc[i][j], 0, 0, 0);
          acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(
              fah[i], fbh[j], acc[i][j], 0, 0, 0);
        }
    }
  }

  // a lane holds column j and rows i .. i + 3 of each quad
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int gi = i0 + wm + i * 32 + 8 * q + 4 * fk;
        const int gj = j0 + wn + j * 32 + fr;
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = acc[i][j][4 * q + e] * kInvS;
        if constexpr (MODE == kSquare) {
          // A is symmetric: its column gj is row gj
          const int64_t o = int64_t(gj) * M.mp + gi;
          const half4 h = *reinterpret_cast<const half4 *>(P.ah + o);
          const half4 l = *reinterpret_cast<const half4 *>(P.al + o);
#pragma unroll
          for (int e = 0; e < 4; ++e)
            v[e] = b * (float(h[e]) + float(l[e])) + c * v[e];
        }
        if constexpr (MODE == kApply || MODE == kLast || MODE == kLastMuon) {
          const int64_t o = int64_t(gj) * M.mp + gi;
          const half4 h = *reinterpret_cast<const half4 *>(P.th(src) + o);
          const half4 l = *reinterpret_cast<const half4 *>(P.tl(src) + o);
#pragma unroll
          for (int e = 0; e < 4; ++e)
            v[e] = a * (float(h[e]) + float(l[e])) + v[e];
        }
        if constexpr (MODE == kLast || MODE == kLastMuon) {
          if (gj >= M.n) continue;
          const bool tall = M.rows > M.cols;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if (gi + e >= M.m) continue;
            const int64_t o = tall ? int64_t(gj) * M.cols + gi + e
                                   : int64_t(gi + e) * M.cols + gj;
            const float y = v[e] * kInvS;
            if constexpr (MODE == kLast) {
              store_from_f32(M.out, int64_t(z) * M.rows * M.cols + o, M.odt,
                             y);
            } else {
              const float r = float(M.rows), k = float(M.cols);
              const float lr =
                  S.lr * (S.adjust == FSAGG_MUON_MATCH_RMS
                              ? 0.2f * __fsqrt_rn(r > k ? r : k)
                              : (r > k ? __fsqrt_rn(__fdiv_rn(r, k)) : 1.0f));
              float *p = static_cast<float *>(M.out) + o;
              *p = __builtin_fmaf(-lr, y, __fmul_rn(*p, S.decay));
            }
          }
        } else {
          half4 h, l;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            _Float16 x, y;
            split(v[e], x, y);
            h[e] = x;
            l[e] = y;
          }
          _Float16 *ch, *cl, *dh, *dl;  // C by rows, and C^T
          int ldc, ldd;
          if constexpr (MODE == kApply) {
            ch = P.xh;
            cl = P.xl;
            ldc = M.np;
            dh = P.th(src ^ 1);
            dl = P.tl(src ^ 1);
            ldd = M.mp;
          } else {
            ch = MODE == kGram ? P.ah : P.qh;
            cl = MODE == kGram ? P.al : P.ql;
            ldc = ldd = M.mp;
            dh = ch;
            dl = cl;
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int64_t o = int64_t(gi + e) * ldc + gj;
            ch[o] = h[e];
            cl[o] = l[e];
          }
          if (MODE == kApply || ti != tj) {
            const int64_t o = int64_t(gj) * ldd + gi;
            *reinterpret_cast<half4 *>(dh + o) = h;
            *reinterpret_cast<half4 *>(dl + o) = l;
          }
        }
      }
}

int64_t round_pad(int64_t v) { return (v + kPad - 1) / kPad * kPad; }

// Fills the derived fields; 0 on success.
int plan_mat(Mat &M, int64_t rows, int64_t cols, int64_t batch,
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
  M.mp = int32_t(round_pad(m));
  M.np = int32_t(round_pad(n));
  int64_t nb = (rows * cols + kNormElems - 1) / kNormElems;
  M.nb = int32_t(nb < 1 ? 1 : nb > kMaxNorm ? kMaxNorm : nb);
  M.wstride = (ws_bytes_of(M.mp, M.np) + 1023) / 1024 * 1024;
  return FSAGG_OK;
}

bool empty(const Mat &M) { return M.m == 0 || M.batch == 0; }

// The largest |x|, |x|^2 and |q| that the iteration's limbs have to hold,
// from the scalar iteration on a grid of the singular values in [0, 1]
// (any start is one of these): all have to stay under 2^16 / 2^12.
bool coefficients_fit(double a, double b, double c, int steps) {
  if (!std::isfinite(a) || !std::isfinite(b) || !std::isfinite(c))
    return false;
  constexpr int kGrid = 4096;
  double hi = 1.0;  // bound on the singular values entering the step
  for (int s = 0; s < steps; ++s) {
    if (hi * hi > 15.0) return false;
    double next = 0.0;
    for (int i = 0; i <= kGrid; ++i) {
      const double x = hi * i / kGrid, l = x * x, q = b * l + c * l * l;
      if (!(std::fabs(q) <= 15.0)) return false;
      next = std::fmax(next, std::fabs(a * x + q * x));
    }
    // the grid misses a maximum by at most half a cell's slope
    hi = next * (1.0 + 1.0 / 1024);
    if (!(hi <= 15.0)) return false;
  }
  return true;
}

template <int MODE>
void launch_gemm(Group &G, int src, float a, float b, float c,
                 const MuonScalars &S, hipStream_t s) {
  constexpr int B = 128, W = 64;
  int total = 0;
  for (int i = 0; i < G.nmat; ++i) {
    const Mat &M = G.mat[i];
    const int tm = M.mp / B;
    G.start[i] = total;
    total += M.batch * (MODE == kGram || MODE == kSquare
                            ? tm * (tm + 1) / 2
                            : tm * (M.np / B));
  }
  G.start[G.nmat] = total;
  hipLaunchKernelGGL((ns_gemm_kernel<B, B, W, W, MODE>), dim3(total),
                     dim3(256), 0, s, G, src, b, c, a, S);
}

template <bool MUON>
int run_group(Group &G, int steps, float a, float b, float c, double eps,
              const MuonScalars &S, hipStream_t s, const char *what) {
  int total = 0;
  for (int i = 0; i < G.nmat; ++i) {
    G.start[i] = total;
    total += G.mat[i].batch * G.mat[i].nb;
  }
  G.start[G.nmat] = total;
  hipLaunchKernelGGL(ns_update_kernel<MUON>, dim3(total), dim3(kNormBlock), 0,
                     s, G, S);
  total = 0;
  for (int i = 0; i < G.nmat; ++i) {
    G.start[i] = total;
    total += G.mat[i].batch * (G.mat[i].mp / 64) * (G.mat[i].np / 64);
  }
  G.start[G.nmat] = total;
  hipLaunchKernelGGL(ns_prepare_kernel, dim3(total), dim3(256), 0, s, G, eps);
  int src = 0;
  for (int k = 0; k < steps; ++k) {
    launch_gemm<kGram>(G, src, a, b, c, S, s);
    launch_gemm<kSquare>(G, src, a, b, c, S, s);
    if (k + 1 < steps) launch_gemm<kApply>(G, src, a, b, c, S, s);
    else if (MUON) launch_gemm<kLastMuon>(G, src, a, b, c, S, s);
    else launch_gemm<kLast>(G, src, a, b, c, S, s);
    src ^= 1;
  }
  return check_launch(what);
}

// Workgroups of the widest launch: the prepare pass, 64 x 64 tiles.
int64_t most_blocks(const Mat &M) {
  return int64_t(M.batch) * (M.mp / 64) * (M.np / 64) +
         int64_t(M.batch) * M.nb;
}

// Entries in order, up to kMaxGroup per run.
template <bool MUON, typename Fill>
int run_all(int nmat, Fill fill, int steps, const double *coef, double eps,
            const MuonScalars &S, void *ws, size_t ws_bytes, hipStream_t s,
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
  // everything is checked before anything is launched
  size_t need = 0;
  for (int i = 0; i < nmat; ++i) {
    Mat M;
    const int rc = fill(i, M);
    if (rc != FSAGG_OK) return rc;
    if (empty(M)) continue;
    need += size_t(M.wstride) * M.batch;
    // a launch counts its work items in 32 bits
    if (most_blocks(M) > (int64_t(1) << 24) / kMaxGroup) {
      set_error("%s: matrix %d: a batch of %d is too large for one call",
                what, i, M.batch);
      return FSAGG_EINVAL;
    }
  }
  if (need == 0) return FSAGG_OK;
  if (!ws || ws_bytes < need) {
    set_error("%s: workspace of %zu bytes, %zu needed", what,
              ws ? ws_bytes : size_t(0), need);
    return FSAGG_ESPACE;
  }
  if (!aligned16(ws)) {
    set_error("%s: workspace must be 16-byte aligned", what);
    return FSAGG_EINVAL;
  }
  char *at = static_cast<char *>(ws);
  Group G;
  G.nmat = 0;
  for (int i = 0; i < nmat; ++i) {
    Mat &M = G.mat[G.nmat];
    fill(i, M);
    if (empty(M)) continue;
    M.ws = at;
    at += size_t(M.wstride) * M.batch;
    if (++G.nmat == kMaxGroup) {
      const int rc = run_group<MUON>(G, steps, float(coef[0]), float(coef[1]),
                                     float(coef[2]), eps, S, s, what);
      if (rc != FSAGG_OK) return rc;
      G.nmat = 0;
    }
  }
  if (G.nmat == 0) return FSAGG_OK;
  return run_group<MUON>(G, steps, float(coef[0]), float(coef[1]),
                         float(coef[2]), eps, S, s, what);
}

bool float_dtype(int dt) {
  return dt == FSAGG_F32 || dt == FSAGG_F16 || dt == FSAGG_BF16;
}

}  // namespace
}  // namespace fsagg

using namespace fsagg;

extern "C" size_t fsagg_newton_schulz_workspace_bytes(int64_t rows,
                                                      int64_t cols,
                                                      int64_t batch) {
  Mat M;
  if (plan_mat(M, rows, cols, batch, "fsagg_newton_schulz_workspace_bytes") !=
          FSAGG_OK ||
      empty(M))
    return 0;
  return size_t(M.wstride) * M.batch;
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
  auto fill = [&](int i, Mat &M) {
    const fsagg_ns_mat &d = mats[i];
    const int rc = plan_mat(M, d.rows, d.cols, d.batch, what);
    if (rc != FSAGG_OK) return rc;
    if (empty(M)) return int(FSAGG_OK);
    if (!d.g || !d.out || !float_dtype(d.dtype) || !float_dtype(d.out_dtype)) {
      set_error("%s: matrix %d: null pointer or unknown dtype", what, i);
      return int(FSAGG_EINVAL);
    }
    M.g = d.g;
    M.out = d.out;
    M.buf = nullptr;
    M.sz = d.batch_stride;
    M.si = d.row_stride;
    M.sj = d.col_stride;
    M.dt = int16_t(d.dtype);
    M.odt = int16_t(d.out_dtype);
    return int(FSAGG_OK);
  };
  return run_all<false>(nmat, fill, steps, coefficients, eps, MuonScalars{},
                        workspace, workspace_bytes, as_stream(stream), what);
}

extern "C" int fsagg_muon_step_f32(const fsagg_muon_mat *mats, int nmat,
                                   const fsagg_muon_params *hp,
                                   void *workspace, size_t workspace_bytes,
                                   fsagg_stream_t stream) {
  const char *what = "fsagg_muon_step_f32";
  if (nmat < 0 || (nmat > 0 && !mats) || !hp) {
    set_error("%s: invalid argument", what);
    return FSAGG_EINVAL;
  }
  if (hp->adjust != FSAGG_MUON_ORIGINAL && hp->adjust != FSAGG_MUON_MATCH_RMS) {
    set_error("%s: unknown learning-rate adjustment %d", what, hp->adjust);
    return FSAGG_EINVAL;
  }
  auto fill = [&](int i, Mat &M) {
    const fsagg_muon_mat &d = mats[i];
    const int rc = plan_mat(M, d.rows, d.cols, 1, what);
    if (rc != FSAGG_OK) return rc;
    if (empty(M)) return int(FSAGG_OK);
    if (!d.param || !d.avg || !d.momentum) {
      set_error("%s: matrix %d: null pointer", what, i);
      return int(FSAGG_EINVAL);
    }
    M.g = d.avg;
    M.out = d.param;
    M.buf = d.momentum;
    M.sz = M.si = M.sj = 0;
    M.dt = M.odt = FSAGG_F32;
    return int(FSAGG_OK);
  };
  MuonScalars S;
  S.keep = float(1.0 - hp->momentum);
  S.mu = float(hp->momentum);
  S.lr = float(hp->lr);
  S.decay = float(1.0 - hp->lr * hp->weight_decay);
  S.nesterov = hp->nesterov;
  S.maximize = hp->maximize;
  S.adjust = hp->adjust;
  const double coef[3] = {hp->a, hp->b, hp->c};
  return run_all<true>(nmat, fill, hp->steps, coef, hp->eps, S, workspace,
                       workspace_bytes, as_stream(stream), what);
}
