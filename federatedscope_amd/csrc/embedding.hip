// Embedding rows: the lookup with a scale, and its gradient — the weighted
// sum of many clients' rows by token (gfx950).
//
//   lookup:   out[t] = round(scale * E[ids[t]])
//   gradient: out[v] = [out[v] +] sum over the tokens t with ids[t] = v, in
//             token order, of coef(part of t) * rows[t], in fp32, rounded
//             once.
//
// A token number outside [0, V) is padding: the lookup gives a zero row, the
// gradient does not read its row at all.
//
// The gradient sorts the tokens by row (a stable radix sort, so a row's
// tokens stay in token order and the result does not depend on timing), then
// walks the sorted list in chunks of at most 64 tokens.  A wave owns a chunk
// and 64 vectors of columns: it loads the rows of its chunk and keeps one
// running sum in registers, written out where the token number changes.  A
// row whose tokens cross chunks leaves one partial sum per chunk, added up
// in order by a last pass; the split is fixed by the sizes alone.  Both
// operators are bound by memory where they are large: they read each token's
// row once and write each result row once (65536 x 2048 bf16 into 128000
// rows, 0.79 GB, 183 us = 4.3 TB/s, the sum alone 142 us; 100 clients' 400
// rows of 1024 fp32 added into 50000, 0.26 GB, 88 us, of which the sum is
// 52 and the sort 27; a lookup of 16384 x 4096 bf16 34 us).  Small calls are
// bound by the host and their launches (7 rows 5 us, 48 tokens 7, 5001 22).
#include "common.h"

#include <hip/hip_fp16.h>

namespace fsagg {
namespace {

constexpr int kBlock = 256;
constexpr int kWaves = kBlock / kWave;
constexpr int kMaxParts = 112;    // parts per key launch (kernel arguments)
// Sorting: a thread holds kRounds tokens.  Up to kOneTile tokens are one
// workgroup's (4096 tokens of 4000 rows of 300, the whole call 25 us, in
// tiles 30; 1000 tokens 16, 25); else tiles of 1024 tokens, small enough that
// many sort at once.
constexpr int kRounds = 4;
constexpr int kOneThreads = 1024, kOneTile = kOneThreads * kRounds;
constexpr int kTileThreads = 256, kTile = kTileThreads * kRounds;
// Tiles whose counts a tile adds up itself; more are scanned first by a launch
// of their own (40 tiles: 92 us with the scan, 96 without; 64 tiles 182, 203).
constexpr int kSumBlocks = 8;
constexpr int kFew = kBlock;      // tokens that every workgroup sorts itself
constexpr int kMaxDigit = 10;     // bits per radix pass
// a launch counts its work items in 32 bits
constexpr int64_t kMaxGrid = (int64_t(1) << 32) / kBlock - 1;

// -- element types -----------------------------------------------------------
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

template <int DT>
struct Elem;
template <>
struct Elem<FSAGG_F32> {
  using type = float;
  static constexpr int kVec = 4;
  __device__ static float get(float x) { return x; }
  __device__ static float put(float x) { return x; }
};
template <>
struct Elem<FSAGG_F16> {
  using type = _Float16;
  static constexpr int kVec = 8;
  __device__ static float get(_Float16 x) { return float(x); }
  __device__ static _Float16 put(float x) { return _Float16(x); }
};
template <>
struct Elem<FSAGG_BF16> {
  using type = uint16_t;
  static constexpr int kVec = 8;
  __device__ static float get(uint16_t x) {
    return __uint_as_float(uint32_t(x) << 16);
  }
  // round to nearest even, NaN kept (quieted)
  __device__ static uint16_t put(float v) {
    const uint32_t u = __float_as_uint(v);
    if ((u & 0x7FFFFFFFu) > 0x7F800000u) return uint16_t((u >> 16) | 0x40u);
    return uint16_t((u + 0x7FFFu + ((u >> 16) & 1u)) >> 16);
  }
};

// VEC elements as they lie: one 16-byte load (or less), or a single element
template <int DT, int VEC>
struct Raw {
  typedef typename Elem<DT>::type type __attribute__((ext_vector_type(VEC)));
};
template <int DT>
struct Raw<DT, 1> {
  using type = typename Elem<DT>::type;
};
template <int DT, int VEC>
__device__ __forceinline__ typename Raw<DT, VEC>::type load_raw(
    const void *p) {
  return gld(static_cast<const typename Raw<DT, VEC>::type *>(p));
}
template <int DT, int VEC>
__device__ __forceinline__ void widen(
    const typename Raw<DT, VEC>::type &x, float (&v)[VEC]) {
  if constexpr (VEC == 1) {
    v[0] = Elem<DT>::get(x);
  } else {
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] = Elem<DT>::get(x[e]);
  }
}
template <int DT, int VEC>
__device__ __forceinline__ void load_vec(const void *p, float (&v)[VEC]) {
  widen<DT, VEC>(load_raw<DT, VEC>(p), v);
}
// (rows that go by once bypass the caches, NT here and gld_nt: a lookup of
// 16384 x 4096 bf16 45 -> 35 us, the rows of 100 x 400 tokens of 1024 fp32
// 108 -> 92; the sums' own rows lost by it, 65536 x 2048 bf16 183 -> 196)
template <int DT, int VEC, bool NT = false>
__device__ __forceinline__ void store_vec(void *p, const float (&v)[VEC]) {
  typename Raw<DT, VEC>::type x;
  if constexpr (VEC == 1) {
    x = Elem<DT>::put(v[0]);
  } else {
#pragma unroll
    for (int e = 0; e < VEC; ++e) x[e] = Elem<DT>::put(v[e]);
  }
  if constexpr (NT)
    __builtin_nontemporal_store(x,
                                static_cast<typename Raw<DT, VEC>::type *>(p));
  else
    *static_cast<typename Raw<DT, VEC>::type *>(p) = x;
}

__device__ __forceinline__ int64_t load_id(const void *ids, int64_t t,
                                           int ids64) {
  return ids64 ? static_cast<const int64_t *>(ids)[t]
               : int64_t(static_cast<const int32_t *>(ids)[t]);
}

// -- lookup ------------------------------------------------------------------
constexpr int kLookVecs = 4;  // vectors of a row per lane

// One wave per token and stretch of 64 * kLookVecs vectors of its row.
template <int DT, int VEC>
__global__ __launch_bounds__(kBlock) void embed_lookup_kernel(
    const char *__restrict__ table, int64_t row_bytes, int64_t vocab,
    const void *__restrict__ ids, int ids64, int64_t tokens, int64_t dim,
    int stretches, float scale, char *__restrict__ out) {
  constexpr int kE = sizeof(typename Elem<DT>::type);
  const int lane = threadIdx.x & (kWave - 1);
  const int wave =
      __builtin_amdgcn_readfirstlane(int(threadIdx.x) / kWave);
  const int64_t unit = int64_t(blockIdx.x) * kWaves + wave;
  if (unit >= tokens * stretches) return;
  const int64_t t = unit / stretches;
  const int64_t c0 = (unit % stretches) * (kWave * kLookVecs * VEC);
  const int64_t id = load_id(ids, t, ids64);
  const bool ok = id >= 0 && id < vocab;
  const char *src = table + (ok ? id : 0) * row_bytes;
  char *dst = out + t * dim * kE;
  float v[kLookVecs][VEC] = {};
  if (ok) {
    // (lanes past the row read its start: a load under a condition is waited
    // for before the next one goes out)
    typename Raw<DT, VEC>::type raw[kLookVecs];
#pragma unroll
    for (int k = 0; k < kLookVecs; ++k) {
      const int64_t c = c0 + (k * kWave + lane) * VEC;
      raw[k] = load_raw<DT, VEC>(src + (c < dim ? c : 0) * kE);
    }
#pragma unroll
    for (int k = 0; k < kLookVecs; ++k) widen<DT, VEC>(raw[k], v[k]);
  }
#pragma unroll
  for (int k = 0; k < kLookVecs; ++k) {
    const int64_t c = c0 + (k * kWave + lane) * VEC;
    if (c < dim) {
      if (ok) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[k][e] = __fmul_rn(v[k][e], scale);
      }
      store_vec<DT, VEC, true>(dst + c * kE, v[k]);
    }
  }
}

// -- gradient: keys and sort ---------------------------------------------------
struct Part {
  const void *ids;
  const char *rows;
  uint32_t start;   // first token of the part
  uint32_t stride;  // elements between rows; the top bit: int64 ids
  float coef;
};
struct Parts {
  int n, elem;
  uint32_t end;  // tokens up to the end of the last part here
  Part part[kMaxParts];
};
constexpr uint32_t kIds64 = 0x80000000u;

// Arrays of a call, in its workspace.
struct Sort {
  uint32_t *key[2];
  uint32_t *tok[2];
  const char **row, **srow;  // by token, and as sorted
  float *coef, *scoef;
  uint32_t *hist;    // [digits][blocks]
  uint32_t *total;   // [digits]
  float *partial;    // [chunk][head, tail][dim]
};

// Keys of N tokens (each its row, or V for padding), their rows of values
// and factors; the N chains of loads go side by side.
template <int N>
__device__ __forceinline__ void token_keys(const Parts &P,
                                           const uint32_t *starts,
                                           const uint32_t (&t)[N],
                                           uint32_t vocab, uint32_t (&key)[N],
                                           const char *(&row)[N],
                                           float (&coef)[N]) {
  static_assert(kMaxParts <= 128, "steps of the search");
  int at[N];
#pragma unroll
  for (int k = 0; k < N; ++k) at[k] = 0;
#pragma unroll
  for (int step = 64; step > 0; step >>= 1)
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int next = at[k] + step;
      const uint32_t first = starts[next < P.n ? next : 0];
      at[k] = next < P.n && first <= t[k] ? next : at[k];
    }
  Part p[N];
#pragma unroll
  for (int k = 0; k < N; ++k) p[k] = P.part[at[k]];
  // (both halves of an int64 id as words, so that one kind of load serves
  // both types)
  uint32_t lo[N], hi[N];
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const int64_t i = t[k] - p[k].start;
    const bool wide = (p[k].stride & kIds64) != 0;
    const uint32_t *q = static_cast<const uint32_t *>(p[k].ids) +
                        (wide ? 2 * i : i);
    lo[k] = gld(q);
    hi[k] = gld(q + (wide ? 1 : 0));
  }
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const int64_t i = t[k] - p[k].start;
    const bool wide = (p[k].stride & kIds64) != 0;
    row[k] = p[k].rows + i * int64_t(p[k].stride & ~kIds64) * P.elem;
    coef[k] = p[k].coef;
    // (a negative int32 id is above any row, too)
    key[k] = (!wide || hi[k] == 0) && lo[k] < vocab ? lo[k] : vocab;
  }
}

// The parts' first tokens, for token_keys, in LDS (the caller synchronises).
__device__ __forceinline__ void stage_starts(const Parts &P,
                                             uint32_t *starts) {
  if (int(threadIdx.x) < P.n) starts[threadIdx.x] = P.part[threadIdx.x].start;
}

__device__ __forceinline__ void note_token(const Sort &W, uint32_t t,
                                           uint32_t key, const char *row,
                                           float coef) {
  W.key[0][t] = key;
  W.tok[0][t] = t;
  W.row[t] = row;
  W.coef[t] = coef;
}

// Keys of these parts' tokens (a call of more parts than fit one launch).
__global__ __launch_bounds__(kBlock) void embed_key_kernel(Parts P, Sort W,
                                                           uint32_t vocab) {
  __shared__ uint32_t starts[kMaxParts];
  stage_starts(P, starts);
  __syncthreads();
  for (int64_t t = int64_t(P.part[0].start) +
                   int64_t(blockIdx.x) * kBlock + threadIdx.x;
       t < P.end; t += int64_t(gridDim.x) * kBlock) {
    const uint32_t at[1] = {uint32_t(t)};
    uint32_t key[1];
    const char *row[1];
    float coef[1];
    token_keys<1>(P, starts, at, vocab, key, row, coef);
    note_token(W, at[0], key[0], row[0], coef[0]);
  }
}

// token k of this thread's `rounds` in the tile at `base`: a wave owns
// neighbouring tokens, in rounds of 64
__device__ __forceinline__ int64_t tile_token(int64_t base, int k,
                                              int rounds = kRounds) {
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  return base + wave * (rounds * kWave) + k * kWave + lane;
}

// Rank of every token of a workgroup's tile among the tile's tokens of the
// same digit in the same wave, in order; cnt[digit][wave] ends as the wave's
// count of the digit.
template <int TH>
__device__ __forceinline__ void tile_ranks(const uint32_t (&key)[kRounds],
                                           const bool (&in)[kRounds],
                                           int rounds, int shift, int bits,
                                           uint16_t *cnt,
                                           uint32_t (&rank)[kRounds]) {
  constexpr int kW = TH / kWave;
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const uint32_t mask = (1u << bits) - 1u;
  u32x4 *cnt4 = reinterpret_cast<u32x4 *>(cnt);
  for (int i = threadIdx.x; i < (kW << bits) / 8; i += TH)
    cnt4[i] = u32x4{0, 0, 0, 0};
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kRounds; ++k) {
    if (k >= rounds) break;
    const uint32_t d = (key[k] >> shift) & mask;
    uint64_t same = __ballot(in[k]);
    for (int b = 0; b < bits; ++b) {
      const uint64_t m = __ballot((d >> b) & 1u);
      same &= ((d >> b) & 1u) ? m : ~m;
    }
    uint16_t *c = cnt + d * kW + wave;
    const uint32_t before = in[k] ? *c : 0u;
    rank[k] = before + __popcll(same & ((1ull << lane) - 1ull));
    // the whole wave has read its counters (one instruction stream); the
    // digit's last lane leaves the new count
    __builtin_amdgcn_wave_barrier();
    if (in[k] && (same >> lane) == 1ull)
      *c = uint16_t(before + __popcll(same));
    __builtin_amdgcn_wave_barrier();
  }
  __syncthreads();
}

// Turns digit d's counts by wave into the counts of the waves before; the
// digit's total.
template <int TH>
__device__ __forceinline__ uint32_t wave_prefix(uint16_t *cnt, int d) {
  constexpr int kW = TH / kWave;
  uint16_t n[kW];
#pragma unroll
  for (int w = 0; w < kW; ++w) n[w] = cnt[d * kW + w];
  uint32_t total = 0;
#pragma unroll
  for (int w = 0; w < kW; ++w) {
    cnt[d * kW + w] = uint16_t(total);
    total += n[w];
  }
  return total;
}

// Exclusive sums over digits: at[d] = v(0) + .. + v(d - 1), 1 << kMaxDigit
// digits at most.  A thread has neighbouring digits, so that their counts
// are read together and one scan does.
template <int TH, typename F>
__device__ __forceinline__ void digit_starts(int digits, F v, uint32_t *at,
                                             uint32_t *scratch) {
  constexpr int kEach = (1 << kMaxDigit) / TH;
  static_assert(kEach * TH == 1 << kMaxDigit, "digits divide over threads");
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const int each = (digits + TH - 1) / TH;
  const int d0 = int(threadIdx.x) * each;
  uint32_t n[kEach], own = 0;
#pragma unroll
  for (int i = 0; i < kEach; ++i)
    n[i] = i < each && d0 + i < digits ? v(d0 + i) : 0u;
#pragma unroll
  for (int i = 0; i < kEach; ++i) own += n[i];
  uint32_t s = own;
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) {
    const uint32_t u = __shfl_up(s, o);
    if (lane >= o) s += u;
  }
  if (lane == kWave - 1) scratch[wave] = s;
  __syncthreads();
  s -= own;
  for (int w = 0; w < wave; ++w) s += scratch[w];
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    if (i < each && d0 + i < digits) at[d0 + i] = s;
    s += n[i];
  }
  __syncthreads();
}

// The result, and how it is cut.
struct Out {
  char *out;
  int64_t row_bytes, dim, vocab, tokens;
  int chunk, slices, accumulate, elem;
  int zero_nt, zero_rows;  // rows per zero workgroup
  int64_t chunks;
  const uint32_t *key;
};

// Zeros into the rows [r0, r1) that are not named (null: into all), by the
// whole workgroup: `g` lanes a row, 16 bytes a lane whatever the row's
// alignment, 2 bytes at a time before and behind.
template <int TH>
__device__ __forceinline__ void zero_rows_of(const Out &O, int64_t r0,
                                             int64_t r1,
                                             const uint8_t *named) {
  const int lane = threadIdx.x & (kWave - 1);
  const int wave =
      __builtin_amdgcn_readfirstlane(int(threadIdx.x) / kWave);
  const int64_t bytes = O.dim * O.elem;
  int g = kWave;
  while (g > 1 && bytes <= int64_t(g / 2) * 16) g /= 2;
  const int l = lane & (g - 1), sub = lane / g, rows = kWave / g;
  for (int64_t r = r0 + wave * rows + sub; r < r1;
       r += TH / kWave * rows) {
    if (named && named[r - r0]) continue;
    char *p = O.out + r * O.row_bytes;
    const int64_t before = -reinterpret_cast<uint64_t>(p) & 15;
    const int64_t head = before < bytes ? before : bytes;
    const int64_t body = head + ((bytes - head) & ~int64_t(15));
    if (O.zero_nt)
      for (int64_t c = head + l * 16; c < body; c += g * 16)
        __builtin_nontemporal_store(u32x4{0, 0, 0, 0},
                                    reinterpret_cast<u32x4 *>(p + c));
    else
      for (int64_t c = head + l * 16; c < body; c += g * 16)
        *reinterpret_cast<u32x4 *>(p + c) = u32x4{0, 0, 0, 0};
    for (int64_t c = l * 2; c < head; c += g * 2)
      *reinterpret_cast<uint16_t *>(p + c) = 0;
    for (int64_t c = body + l * 2; c < bytes; c += g * 2)
      *reinterpret_cast<uint16_t *>(p + c) = 0;
  }
}

// hist[digit][block], of the keys as they are (P.n = 0) or as they are made
// here.
__global__ __launch_bounds__(kTileThreads) void embed_hist_kernel(
    Parts P, Sort W, int src, int64_t tokens, uint32_t vocab, int shift,
    int bits, int blocks) {
  __shared__ uint32_t h[1 << kMaxDigit];
  __shared__ uint32_t starts[kMaxParts];
  const int digits = 1 << bits;
  for (int i = threadIdx.x; i < digits; i += kTileThreads) h[i] = 0;
  stage_starts(P, starts);
  __syncthreads();
  const int64_t base = int64_t(blockIdx.x) * kTile;
  uint32_t t[kRounds], key[kRounds];
  bool in[kRounds];
#pragma unroll
  for (int k = 0; k < kRounds; ++k) {
    const int64_t at = tile_token(base, k);
    in[k] = at < tokens;
    t[k] = uint32_t(in[k] ? at : tokens - 1);
  }
  if (P.n > 0) {
    const char *row[kRounds];
    float coef[kRounds];
    token_keys<kRounds>(P, starts, t, vocab, key, row, coef);
#pragma unroll
    for (int k = 0; k < kRounds; ++k)
      if (in[k]) note_token(W, t[k], key[k], row[k], coef[k]);
  } else {
#pragma unroll
    for (int k = 0; k < kRounds; ++k) key[k] = W.key[src][t[k]];
  }
#pragma unroll
  for (int k = 0; k < kRounds; ++k)
    if (in[k]) atomicAdd(&h[(key[k] >> shift) & (digits - 1)], 1u);
  __syncthreads();
  for (int i = threadIdx.x; i < digits; i += kTileThreads)
    W.hist[int64_t(i) * blocks + blockIdx.x] = h[i];
}

// Where there are many tiles: a digit's counts become the counts of the
// tiles before, and its total is noted (one workgroup per digit).
__global__ __launch_bounds__(kTileThreads) void embed_scan_kernel(
    Sort W, int blocks) {
  __shared__ uint32_t scratch[kTileThreads / kWave];
  uint32_t *h = W.hist + int64_t(blockIdx.x) * blocks;
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  uint32_t before = 0;
  for (int b0 = 0; b0 < blocks; b0 += kTileThreads) {
    const int b = b0 + int(threadIdx.x);
    const uint32_t n = b < blocks ? h[b] : 0u;
    uint32_t s = n;
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
      const uint32_t u = __shfl_up(s, o);
      if (lane >= o) s += u;
    }
    if (lane == kWave - 1) scratch[wave] = s;
    __syncthreads();
    uint32_t sum = before;
    for (int w = 0; w < kTileThreads / kWave; ++w) {
      if (w == wave && b < blocks) h[b] = sum + s - n;
      sum += scratch[w];
    }
    before = sum;
    __syncthreads();
  }
  if (threadIdx.x == 0) W.total[blockIdx.x] = before;
}

// One stable pass: every token of tile b goes to the digit's start plus the
// digit's tokens in earlier tiles and waves plus its rank.  The last pass
// takes the rows and factors along.
__global__ __launch_bounds__(kTileThreads) void embed_scatter_kernel(
    Sort W, int src, int64_t tokens, int shift, int bits, int blocks,
    int scanned, int last) {
  constexpr int kW = kTileThreads / kWave;
  __shared__ __attribute__((aligned(16))) uint16_t cnt[kW << kMaxDigit];
  __shared__ uint32_t at[1 << kMaxDigit], mine[1 << kMaxDigit];
  __shared__ uint32_t scratch[kW];
  uint32_t key[kRounds], tok[kRounds], rank[kRounds];
  bool in[kRounds];
  const int64_t base = int64_t(blockIdx.x) * kTile;
#pragma unroll
  for (int k = 0; k < kRounds; ++k) {
    const int64_t t = tile_token(base, k);
    in[k] = t < tokens;
    key[k] = W.key[src][in[k] ? t : tokens - 1];
    tok[k] = W.tok[src][in[k] ? t : tokens - 1];
  }
  const int digits = 1 << bits;
  // a digit's total and its tokens in earlier tiles
  digit_starts<kTileThreads>(
      digits,
      [&](int d) {
        const uint32_t *h = W.hist + int64_t(d) * blocks;
        if (scanned) {
          mine[d] = h[blockIdx.x];
          return W.total[d];
        }
        uint32_t total = 0, m = 0;
        constexpr int kAhead = 8;
        for (int b0 = 0; b0 < blocks; b0 += kAhead) {
          uint32_t n[kAhead];
#pragma unroll
          for (int u = 0; u < kAhead; ++u)
            n[u] = b0 + u < blocks ? h[b0 + u] : 0u;
#pragma unroll
          for (int u = 0; u < kAhead; ++u) {
            if (b0 + u == int(blockIdx.x)) m = total;
            total += n[u];
          }
        }
        mine[d] = m;
        return total;
      },
      at, scratch);
  tile_ranks<kTileThreads>(key, in, kRounds, shift, bits, cnt, rank);
  for (int d = threadIdx.x; d < digits; d += kTileThreads) {
    at[d] += mine[d];
    wave_prefix<kTileThreads>(cnt, d);
  }
  __syncthreads();
  const int wave = threadIdx.x / kWave;
  const char *row[kRounds];
  float coef[kRounds];
  if (last) {
#pragma unroll
    for (int k = 0; k < kRounds; ++k) {
      row[k] = W.row[tok[k]];
      coef[k] = W.coef[tok[k]];
    }
  }
#pragma unroll
  for (int k = 0; k < kRounds; ++k) {
    if (!in[k]) continue;
    const uint32_t d = (key[k] >> shift) & (digits - 1);
    const uint32_t o = at[d] + cnt[d * kW + wave] + rank[k];
    W.key[src ^ 1][o] = key[k];
    if (last) {
      W.srow[o] = row[k];
      W.scoef[o] = coef[k];
    } else {
      W.tok[src ^ 1][o] = tok[k];
    }
  }
}

// Keys and sort of one workgroup's tokens in one launch, through LDS; the
// other workgroups, if any, zero all rows.
__global__ __launch_bounds__(kOneThreads) void embed_sort_kernel(
    Parts P, Sort W, int src, int64_t tokens, uint32_t vocab, int passes,
    int bits, Out O) {
  if (blockIdx.x > 0) {
    const int64_t r0 = int64_t(blockIdx.x - 1) * O.zero_rows;
    const int64_t r1 =
        r0 + O.zero_rows < O.vocab ? r0 + O.zero_rows : O.vocab;
    zero_rows_of<kOneThreads>(O, r0, r1, nullptr);
    return;
  }
  constexpr int kW = kOneThreads / kWave;
  __shared__ __attribute__((aligned(16))) uint16_t cnt[kW << kMaxDigit];
  __shared__ uint32_t at[1 << kMaxDigit];
  __shared__ uint32_t scratch[kW];
  __shared__ uint32_t skey[kOneTile];
  __shared__ uint16_t stok[kOneTile];
  __shared__ const char *srow[kOneTile];
  __shared__ float scoef[kOneTile];
  __shared__ uint32_t starts[kMaxParts];
  stage_starts(P, starts);
  __syncthreads();
  uint32_t key[kRounds], tok[kRounds], rank[kRounds];
  bool in[kRounds];
  const int wave = threadIdx.x / kWave;
  // (as few rounds as hold the tokens: all waves are at it)
  const int rounds = int((tokens + kOneThreads - 1) / kOneThreads);
#pragma unroll
  for (int k = 0; k < kRounds; ++k) {
    const int t = int(tile_token(0, k, rounds));
    in[k] = k < rounds && t < tokens;
    tok[k] = uint32_t(in[k] ? t : int(tokens) - 1);
  }
  const char *row[kRounds];
  float coef[kRounds];
  if (P.n > 0) {
    token_keys<kRounds>(P, starts, tok, vocab, key, row, coef);
  } else {
#pragma unroll
    for (int k = 0; k < kRounds; ++k) {
      key[k] = W.key[0][tok[k]];
      row[k] = W.row[tok[k]];
      coef[k] = W.coef[tok[k]];
    }
  }
#pragma unroll
  for (int k = 0; k < kRounds; ++k)
    if (in[k]) {
      srow[tok[k]] = row[k];
      scoef[tok[k]] = coef[k];
    }
  const int digits = 1 << bits;
  for (int p = 0; p < passes; ++p) {
    const int shift = p * bits;
    tile_ranks<kOneThreads>(key, in, rounds, shift, bits, cnt, rank);
    digit_starts<kOneThreads>(
        digits, [&](int d) { return wave_prefix<kOneThreads>(cnt, d); }, at,
        scratch);
#pragma unroll
    for (int k = 0; k < kRounds; ++k) {
      if (!in[k]) continue;
      const uint32_t d = (key[k] >> shift) & (digits - 1);
      const uint32_t o = at[d] + cnt[d * kW + wave] + rank[k];
      skey[o] = key[k];
      stok[o] = uint16_t(tok[k]);
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kRounds; ++k) {
      const int t = int(tile_token(0, k, rounds));
      if (in[k]) {
        key[k] = skey[t];
        tok[k] = stok[t];
      }
    }
  }
#pragma unroll
  for (int k = 0; k < kRounds; ++k) {
    const int64_t t = tile_token(0, k, rounds);
    if (in[k]) {
      W.key[src][t] = key[k];
      W.srow[t] = srow[tok[k]];
      W.scoef[t] = scoef[tok[k]];
    }
  }
}

// -- gradient: sums ------------------------------------------------------------
// lanes from the first on that say yes
__device__ __forceinline__ int run_length(bool yes) {
  const uint64_t m = __ballot(yes);
  return m == ~0ull ? kWave : __builtin_ctzll(~m);
}

// first positions a and b in key[0, n) with key >= x and key >= y, by the
// whole wave: 64 probes a round for each, both on their way together
__device__ __forceinline__ void wave_bounds(const uint32_t *key, int64_t n,
                                            uint32_t x, uint32_t y,
                                            int64_t &a, int64_t &b) {
  const int lane = threadIdx.x & (kWave - 1);
  int64_t lo[2] = {0, 0}, hi[2] = {n, n};
  while (lo[0] < hi[0] || lo[1] < hi[1]) {
    int64_t step[2];
    bool below[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      step[i] = (hi[i] - lo[i] + kWave - 1) / kWave;
      const int64_t p = lo[i] + lane * step[i];
      below[i] = false;
      if (p < hi[i]) below[i] = key[p] < (i ? y : x);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      // probes whose key is below: all before the answer
      const int c = __popcll(__ballot(below[i]));
      if (c == 0) {
        hi[i] = lo[i];
        continue;
      }
      const int64_t nhi = lo[i] + c * step[i];
      lo[i] += (c - 1) * step[i] + 1;
      hi[i] = nhi < hi[i] ? nhi : hi[i];
    }
  }
  a = lo[0];
  b = lo[1];
}

constexpr int kZeroRows = kBlock;  // most rows of a zero workgroup

// (keys of a stretch that are looked at one by one: 15003 of 4 stretches save
// 0.5 us against the search, 65536 of 2 would lose 7)
constexpr int64_t kScanKeys = 32 * kBlock;

// Row sums of one chunk of sorted tokens and one slice of columns per wave;
// workgroups past those write the zero rows that no token names.
template <int GT, int OT, int VEC>
__global__ __launch_bounds__(kBlock) void embed_sum_kernel(Out O, Sort W,
                                                           int sum_blocks) {
  constexpr int kOE = sizeof(typename Elem<OT>::type);
  const int lane = threadIdx.x & (kWave - 1);
  const int wave =
      __builtin_amdgcn_readfirstlane(int(threadIdx.x) / kWave);
  if (int(blockIdx.x) >= sum_blocks) {
    // the rows of this stretch that a token names, from the stretch's own
    // tokens: all of them where they are few, else one search per thread
    __shared__ uint8_t named[kZeroRows];
    const int64_t r0 = int64_t(blockIdx.x - sum_blocks) * O.zero_rows;
    const int64_t r1 =
        r0 + O.zero_rows < O.vocab ? r0 + O.zero_rows : O.vocab;
    int64_t a, b;
    wave_bounds(O.key, O.tokens, uint32_t(r0), uint32_t(r1), a, b);
    named[threadIdx.x] = 0;
    __syncthreads();
    if (b - a <= kScanKeys) {
      constexpr int kAhead = 8;
      for (int64_t i0 = a + threadIdx.x; i0 < b; i0 += kAhead * kBlock) {
        uint32_t r[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
          r[u] = i0 + u * kBlock < b ? O.key[i0 + u * kBlock] : 0u;
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
          if (i0 + u * kBlock < b) named[r[u] - uint32_t(r0)] = 1;
      }
    } else if (r0 + int64_t(threadIdx.x) < r1) {
      const uint32_t r = uint32_t(r0) + threadIdx.x;
      int64_t lo = a, hi = b;
      while (lo < hi) {
        const int64_t mid = (lo + hi) >> 1;
        if (O.key[mid] < r) lo = mid + 1;
        else hi = mid;
      }
      named[threadIdx.x] = lo < b && O.key[lo] == r;
    }
    __syncthreads();
    zero_rows_of<kBlock>(O, r0, r1, named);
    return;
  }
  const int64_t unit = int64_t(blockIdx.x) * kWaves + wave;
  if (unit >= O.chunks * O.slices) return;
  const int64_t chunk = unit / O.slices;
  const int64_t c = ((unit % O.slices) * kWave + lane) * VEC;
  const bool mine = c < O.dim;
  // (lanes past the row read its start: a load under a condition is waited
  // for before the next one goes out)
  const int64_t lc = mine ? c / VEC : 0;
  const int64_t p0 = chunk * O.chunk;
  const int64_t left = O.tokens - p0;
  const int cnt = int(left < O.chunk ? left : O.chunk);
  // lane i holds token i of the chunk
  const uint32_t none = uint32_t(O.vocab);
  uint32_t k = none;
  const char *row = nullptr;
  float coef = 0.0f;
  if (lane < cnt) {
    k = O.key[p0 + lane];
    row = W.srow[p0 + lane];
    coef = W.scoef[p0 + lane];
  }
  // padding sorts last
  const int valid = __popcll(__ballot(k != none));
  if (valid == 0) return;
  const uint32_t prev = p0 > 0 ? O.key[p0 - 1] : none;
  const uint32_t next =
      valid == cnt && p0 + cnt < O.tokens ? O.key[p0 + cnt] : none;
  float acc[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) acc[e] = 0.0f;
  bool head = __builtin_amdgcn_readlane(k, 0) == prev;
  constexpr int kAhead = 16;
  for (int i0 = 0; i0 < valid; i0 += kAhead) {
    typename Raw<GT, VEC>::type raw[kAhead];
    typename Raw<OT, VEC>::type old[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int i = i0 + u < valid ? i0 + u : valid - 1;
      const uint64_t a = reinterpret_cast<uint64_t>(row);
      const uint32_t alo = __builtin_amdgcn_readlane(uint32_t(a), i);
      const uint32_t ahi = __builtin_amdgcn_readlane(uint32_t(a >> 32), i);
      const char *src =
          reinterpret_cast<const char *>((uint64_t(ahi) << 32) | alo);
      raw[u] = gld_nt(
          reinterpret_cast<const typename Raw<GT, VEC>::type *>(src) + lc);
    }
    // what the rows hold (of those that end here it is needed)
    if (O.accumulate) {
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int i = i0 + u < valid ? i0 + u : valid - 1;
        old[u] = load_raw<OT, VEC>(
            O.out + int64_t(__builtin_amdgcn_readlane(k, i)) * O.row_bytes +
            lc * (VEC * kOE));
      }
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int i = i0 + u;
      if (i >= valid) break;
      const float w =
          __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(coef), i));
      float v[VEC];
      widen<GT, VEC>(raw[u], v);
#pragma unroll
      for (int e = 0; e < VEC; ++e) acc[e] = __builtin_fmaf(v[e], w, acc[e]);
      const uint32_t key = __builtin_amdgcn_readlane(k, i);
      const uint32_t after =
          i + 1 < valid ? __builtin_amdgcn_readlane(k, i + 1) : next;
      const bool open = i + 1 == valid && after == key;  // goes on
      if (after == key && !open) continue;
      if (mine) {
        if (head || open) {
          float *dst = W.partial + (chunk * 2 + (head ? 0 : 1)) * O.dim + c;
          store_vec<FSAGG_F32, VEC>(dst, acc);
        } else {
          char *dst = O.out + int64_t(key) * O.row_bytes + c * kOE;
          if (O.accumulate) {
            float o[VEC];
            widen<OT, VEC>(old[u], o);
#pragma unroll
            for (int e = 0; e < VEC; ++e) acc[e] = __fadd_rn(o[e], acc[e]);
          }
          store_vec<OT, VEC>(dst, acc);
        }
      }
      head = false;
#pragma unroll
      for (int e = 0; e < VEC; ++e) acc[e] = 0.0f;
    }
  }
}

// A call of few tokens, in one launch: every workgroup sorts them itself (a
// token's place is the number of tokens that come before it), then a wave
// adds up one row's tokens in one slice of columns; workgroups past those
// write the zero rows.  Against the sort's launches, us: 64 tokens of 4000
// rows of 300 6.6 / 14.4, 256 tokens 11.4 / 17.2, 256 of 100 rows of 64
// 13.7 / 15.2 (of 10 rows, which are long, 19.5 / 14.6); it grows with the
// tokens' square.
template <int GT, int OT, int VEC>
__global__ __launch_bounds__(kBlock) void embed_few_kernel(Parts P, Out O,
                                                           int sum_blocks) {
  constexpr int kGE = sizeof(typename Elem<GT>::type);
  constexpr int kOE = sizeof(typename Elem<OT>::type);
  __shared__ uint32_t starts[kMaxParts];
  __shared__ uint32_t key[kFew], skey[kFew];
  __shared__ const char *srow[kFew];
  __shared__ float scoef[kFew];
  __shared__ uint8_t named[kZeroRows];
  const int lane = threadIdx.x & (kWave - 1);
  const int wave =
      __builtin_amdgcn_readfirstlane(int(threadIdx.x) / kWave);
  const int tokens = int(O.tokens), t = threadIdx.x;
  const uint32_t none = uint32_t(O.vocab);
  stage_starts(P, starts);
  named[t] = 0;
  __syncthreads();
  const char *rows[1];
  float coefs[1];
  uint32_t k = ~0u;
  if (tokens > 0) {  // (else there is no part to look into)
    const uint32_t at[1] = {uint32_t(t < tokens ? t : tokens - 1)};
    uint32_t keys[1];
    token_keys<1>(P, starts, at, none, keys, rows, coefs);
    if (t < tokens) k = keys[0];
  }
  key[t] = k;
  __syncthreads();
  if (int(blockIdx.x) >= sum_blocks) {
    const int64_t r0 = int64_t(blockIdx.x - sum_blocks) * O.zero_rows;
    const int64_t r1 =
        r0 + O.zero_rows < O.vocab ? r0 + O.zero_rows : O.vocab;
    if (t < tokens && int64_t(k) >= r0 && int64_t(k) < r1) named[k - r0] = 1;
    __syncthreads();
    zero_rows_of<kBlock>(O, r0, r1, named);
    return;
  }
  if (t < tokens) {
    int place = 0;
    for (int j = 0; j < tokens; ++j)
      place += key[j] < k || (key[j] == k && j < t);
    skey[place] = k;
    srow[place] = rows[0];
    scoef[place] = coefs[0];
  }
  __syncthreads();
  const int64_t unit = int64_t(blockIdx.x) * kWaves + wave;
  const int p = int(unit / O.slices);
  if (p >= tokens) return;
  const uint32_t mine = skey[p];
  if (mine == none || (p > 0 && skey[p - 1] == mine)) return;
  int end = p;
  for (;;) {
    const int q = end + lane;
    const int n = run_length(q < tokens && skey[q] == mine);
    end += n;
    if (n < kWave) break;
  }
  const int64_t c = ((unit % O.slices) * kWave + lane) * VEC;
  if (c >= O.dim) return;
  float acc[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) acc[e] = 0.0f;
  constexpr int kAhead = 8;
  for (int i0 = p; i0 < end; i0 += kAhead) {
    typename Raw<GT, VEC>::type raw[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      raw[u] = load_raw<GT, VEC>(srow[i0 + u < end ? i0 + u : end - 1] +
                                 c * kGE);
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (i0 + u < end) {
        const float w = scoef[i0 + u];
        float v[VEC];
        widen<GT, VEC>(raw[u], v);
#pragma unroll
        for (int e = 0; e < VEC; ++e)
          acc[e] = __builtin_fmaf(v[e], w, acc[e]);
      }
  }
  char *dst = O.out + int64_t(mine) * O.row_bytes + c * kOE;
  if (O.accumulate) {
    float o[VEC];
    load_vec<OT, VEC>(dst, o);
#pragma unroll
    for (int e = 0; e < VEC; ++e) acc[e] = __fadd_rn(o[e], acc[e]);
  }
  store_vec<OT, VEC>(dst, acc);
}

// Rows whose tokens cross chunks: the wave of the chunk in which the row
// begins adds the later chunks' partial sums in order.
template <int OT, int VEC>
__global__ __launch_bounds__(kBlock) void embed_join_kernel(Out O, Sort W) {
  constexpr int kOE = sizeof(typename Elem<OT>::type);
  const int lane = threadIdx.x & (kWave - 1);
  const int wave =
      __builtin_amdgcn_readfirstlane(int(threadIdx.x) / kWave);
  const int64_t unit = int64_t(blockIdx.x) * kWaves + wave;
  if (unit >= (O.chunks - 1) * O.slices) return;
  const int64_t chunk = unit / O.slices;
  const int64_t c = ((unit % O.slices) * kWave + lane) * VEC;
  const int64_t end = (chunk + 1) * O.chunk;  // < tokens: not the last chunk
  const uint32_t key = O.key[end - 1];
  if (key == uint32_t(O.vocab) || O.key[end] != key) return;
  // the row began here unless it fills the chunk and began before
  if (O.key[chunk * O.chunk] == key && chunk > 0 &&
      O.key[chunk * O.chunk - 1] == key)
    return;
  // chunks after this one that the row reaches: those that begin with it
  // (a lane looks at one)
  int64_t last = chunk;
  for (;;) {
    const int64_t q = last + 1 + lane;
    const int n = run_length(q < O.chunks && O.key[q * O.chunk] == key);
    last += n;
    if (n < kWave) break;
  }
  if (c >= O.dim) return;
  float acc[VEC];
  load_vec<FSAGG_F32, VEC>(W.partial + (chunk * 2 + 1) * O.dim + c, acc);
  constexpr int kAhead = VEC > 4 ? 8 : 16;
  for (int64_t q0 = chunk + 1; q0 <= last; q0 += kAhead) {
    float v[kAhead][VEC];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int64_t q = q0 + u <= last ? q0 + u : last;
      load_vec<FSAGG_F32, VEC>(W.partial + q * 2 * O.dim + c, v[u]);
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (q0 + u <= last) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) acc[e] = __fadd_rn(acc[e], v[u][e]);
      }
  }
  char *dst = O.out + int64_t(key) * O.row_bytes + c * kOE;
  if (O.accumulate) {
    float o[VEC];
    load_vec<OT, VEC>(dst, o);
#pragma unroll
    for (int e = 0; e < VEC; ++e) acc[e] = __fadd_rn(o[e], acc[e]);
  }
  store_vec<OT, VEC>(dst, acc);
}

// -- host ----------------------------------------------------------------------
int elem_bytes(int dt) { return dt == FSAGG_F32 ? 4 : 2; }
bool float_dtype(int dt) {
  return dt == FSAGG_F32 || dt == FSAGG_F16 || dt == FSAGG_BF16;
}

// f(integral constant): the element type as a template argument
template <typename F>
void with_dtype(int dt, F f) {
  if (dt == FSAGG_F32) f(std::integral_constant<int, FSAGG_F32>());
  else if (dt == FSAGG_F16) f(std::integral_constant<int, FSAGG_F16>());
  else f(std::integral_constant<int, FSAGG_BF16>());
}

// Tokens per chunk: long chunks leave fewer partial sums of a row with many
// tokens to add up, short ones make enough waves where tokens are few.
// Shorter chunks below 2048 / 512 / 256 / 128 waves, us: 15003 tokens of 777
// rows of 129 41 / 33 / 30 / 33, 6000 of 90 of 64 33 / 33 / 26 / 24, 6000 of
// 90 of 1024 36 / 26 / 30 / 30, 65536 of 60 of 64 68 / 52 / 53 / 52.
constexpr int64_t kManyWaves = 256;
int chunk_tokens(int64_t tokens, int64_t dim) {
  const int64_t slices = (dim + 255) / 256;
  int chunk = kWave;
  while (chunk > 8 && tokens * slices < int64_t(chunk) * kManyWaves) chunk /= 2;
  return chunk;
}

struct Sizes {
  int64_t tokens, dim, chunk, chunks, blocks;
  int bits, passes, digit;
  size_t key, row, coef, hist, digits, partial, total;
};

Sizes sizes_of(int64_t tokens, int64_t dim, int64_t vocab) {
  Sizes Z;
  auto up = [](size_t b) { return (b + 255) / 256 * 256; };
  Z.tokens = tokens;
  Z.dim = dim;
  Z.chunk = chunk_tokens(tokens, dim);
  Z.chunks = (tokens + Z.chunk - 1) / Z.chunk;
  Z.blocks = (tokens + kTile - 1) / kTile;
  Z.bits = 1;
  while (Z.bits < 32 && (vocab >> Z.bits)) ++Z.bits;  // keys 0 .. vocab
  Z.passes = (Z.bits + kMaxDigit - 1) / kMaxDigit;
  Z.digit = (Z.bits + Z.passes - 1) / Z.passes;
  Z.key = up(4 * tokens);
  Z.row = up(8 * tokens);
  Z.coef = up(4 * tokens);
  Z.hist = up(size_t(4) * Z.blocks << Z.digit);
  Z.partial = Z.chunks > 1 ? up(size_t(8) * Z.chunks * dim) : 0;
  Z.digits = up(size_t(4) << Z.digit);
  Z.total = 4 * Z.key + 2 * Z.row + 2 * Z.coef + Z.hist + Z.digits +
            Z.partial;
  return Z;
}

}  // namespace
}  // namespace fsagg

using namespace fsagg;

extern "C" int fsagg_embed_lookup(const void *table, int64_t vocab,
                                  int64_t dim, int64_t row_stride, int dtype,
                                  const void *ids, int ids64, int64_t tokens,
                                  float scale, void *out,
                                  fsagg_stream_t stream) {
  const char *what = "fsagg_embed_lookup";
  if (vocab < 0 || dim < 0 || tokens < 0 || row_stride < 0 ||
      !float_dtype(dtype) ||
      (tokens > 0 && dim > 0 && (!ids || !out || (vocab > 0 && !table)))) {
    set_error("%s: invalid argument", what);
    return FSAGG_EINVAL;
  }
  if (tokens == 0 || dim == 0) return FSAGG_OK;
  const int e = elem_bytes(dtype);
  // 16 bytes a lane, else an element (65536 tokens of 1024 / 1025, us: bf16
  // 38 / 69, fp32 75 / 94; the gradient 87 / 133, 116 / 143)
  const bool vec = (dim * e) % 16 == 0 && (row_stride * e) % 16 == 0 &&
                   aligned16(table) && aligned16(out);
  const int v = vec ? 16 / e : 1;
  const int64_t per = int64_t(kWave) * kLookVecs * v;
  const int64_t stretches = (dim + per - 1) / per;
  const int64_t grid = (tokens * stretches + kWaves - 1) / kWaves;
  if (stretches > INT32_MAX || tokens > kMaxGrid * kWaves ||
      grid > kMaxGrid) {
    set_error("%s: %lld tokens of %lld columns are too many for one call",
              what, (long long)tokens, (long long)dim);
    return FSAGG_EINVAL;
  }
  with_dtype(dtype, [&](auto dt) {
    constexpr int D = decltype(dt)::value;
    if (vec)
      hipLaunchKernelGGL((embed_lookup_kernel<D, Elem<D>::kVec>), dim3(grid),
                         dim3(kBlock), 0, as_stream(stream),
                         static_cast<const char *>(table), row_stride * e,
                         vocab, ids, ids64, tokens, dim, int(stretches),
                         scale, static_cast<char *>(out));
    else
      hipLaunchKernelGGL((embed_lookup_kernel<D, 1>), dim3(grid),
                         dim3(kBlock), 0, as_stream(stream),
                         static_cast<const char *>(table), row_stride * e,
                         vocab, ids, ids64, tokens, dim, int(stretches),
                         scale, static_cast<char *>(out));
  });
  return check_launch(what);
}

extern "C" size_t fsagg_embed_grad_workspace_bytes(int64_t tokens,
                                                   int64_t dim,
                                                   int64_t vocab) {
  if (tokens <= 0 || tokens > FSAGG_EMBED_MAX_TOKENS || dim <= 0 ||
      dim > FSAGG_EMBED_MAX_COLS || vocab < 0 ||
      vocab > FSAGG_EMBED_MAX_ROWS)
    return 0;
  return sizes_of(tokens, dim, vocab).total;
}

extern "C" int fsagg_embed_grad(const fsagg_embed_part *parts, int nparts,
                                int dtype, int64_t vocab, int64_t dim,
                                void *out, int out_dtype, int64_t out_stride,
                                int accumulate, void *workspace,
                                size_t workspace_bytes,
                                fsagg_stream_t stream) {
  const char *what = "fsagg_embed_grad";
  if (nparts < 0 || (nparts > 0 && !parts) || vocab < 0 || dim < 0 ||
      !float_dtype(dtype) || !float_dtype(out_dtype) ||
      (vocab > 0 && dim > 0 && !out)) {
    set_error("%s: invalid argument", what);
    return FSAGG_EINVAL;
  }
  if (vocab > FSAGG_EMBED_MAX_ROWS || dim > FSAGG_EMBED_MAX_COLS) {
    set_error("%s: %lld rows of %lld columns, at most %d of %d", what,
              (long long)vocab, (long long)dim, FSAGG_EMBED_MAX_ROWS,
              FSAGG_EMBED_MAX_COLS);
    return FSAGG_EINVAL;
  }
  if (out_stride < 0 || (vocab > 1 && out_stride < dim)) {
    set_error("%s: result rows of %lld columns, %lld apart, overlap", what,
              (long long)dim, (long long)out_stride);
    return FSAGG_EINVAL;
  }
  const int e = elem_bytes(dtype), oe = elem_bytes(out_dtype);
  // the vector width is the narrower type's: 16 bytes of gradients, and the
  // same number of result elements
  const int vec_elems = dtype == FSAGG_F32 ? 4 : 8;
  bool vec = dim % vec_elems == 0 && (out_stride * oe) % 16 == 0 &&
             aligned16(out);
  int64_t tokens = 0;
  for (int i = 0; i < nparts; ++i) {
    const fsagg_embed_part &p = parts[i];
    if (p.tokens < 0 || (p.tokens > 0 && dim > 0 && (!p.ids || !p.rows)) ||
        p.row_stride < 0 || p.row_stride >= int64_t(kIds64)) {
      set_error("%s: part %d: invalid argument", what, i);
      return FSAGG_EINVAL;
    }
    if (p.tokens > 0)
      vec = vec && (p.row_stride * e) % 16 == 0 && aligned16(p.rows);
    tokens += p.tokens;
    if (tokens > FSAGG_EMBED_MAX_TOKENS) {
      set_error("%s: more than %d tokens", what, FSAGG_EMBED_MAX_TOKENS);
      return FSAGG_EINVAL;
    }
  }
  if (vocab == 0 || dim == 0 || (tokens == 0 && accumulate)) return FSAGG_OK;
  hipStream_t s = as_stream(stream);
  const Sizes Z = sizes_of(tokens, dim, vocab);
  if (tokens > 0 && (!workspace || workspace_bytes < Z.total)) {
    set_error("%s: workspace of %zu bytes, %zu needed", what,
              workspace ? workspace_bytes : size_t(0), Z.total);
    return FSAGG_ESPACE;
  }
  if (!aligned16(workspace)) {
    set_error("%s: workspace must be 16-byte aligned", what);
    return FSAGG_EINVAL;
  }
  Sort W = {};
  char *at = static_cast<char *>(workspace);
  auto take = [&](size_t b) {
    char *p = at;
    at += b;
    return p;
  };
  if (tokens > 0) {
    for (int i = 0; i < 2; ++i) {
      W.key[i] = reinterpret_cast<uint32_t *>(take(Z.key));
      W.tok[i] = reinterpret_cast<uint32_t *>(take(Z.key));
    }
    W.row = reinterpret_cast<const char **>(take(Z.row));
    W.srow = reinterpret_cast<const char **>(take(Z.row));
    W.coef = reinterpret_cast<float *>(take(Z.coef));
    W.scoef = reinterpret_cast<float *>(take(Z.coef));
    W.hist = reinterpret_cast<uint32_t *>(take(Z.hist));
    W.total = reinterpret_cast<uint32_t *>(take(Z.digits));
    W.partial = reinterpret_cast<float *>(take(Z.partial));
  }
  // the parts that hold tokens, up to kMaxParts at a time
  Parts P;
  P.n = 0;
  P.elem = e;
  P.end = 0;
  int nonempty = 0;
  for (int i = 0; i < nparts; ++i) nonempty += parts[i].tokens > 0;
  const bool one_launch = nonempty <= kMaxParts;
  for (int i = 0; i < nparts; ++i) {
    const fsagg_embed_part &p = parts[i];
    if (p.tokens == 0) continue;
    Part &q = P.part[P.n++];
    q.ids = p.ids;
    q.rows = static_cast<const char *>(p.rows);
    q.start = P.end;
    q.stride = uint32_t(p.row_stride) | (p.ids64 ? kIds64 : 0u);
    q.coef = p.coef;
    P.end += uint32_t(p.tokens);
    if (!one_launch && (P.n == kMaxParts || P.end == uint32_t(tokens))) {
      hipLaunchKernelGGL(embed_key_kernel,
                         dim3(stream_grid(P.end - P.part[0].start, kBlock,
                                          2048)),
                         dim3(kBlock), 0, s, P, W, uint32_t(vocab));
      P.n = 0;
    }
  }
  Out O;
  O.out = static_cast<char *>(out);
  O.row_bytes = out_stride * oe;
  O.dim = dim;
  O.vocab = vocab;
  O.tokens = tokens;
  O.elem = oe;
  O.chunk = int(Z.chunk);
  O.chunks = Z.chunks;
  O.accumulate = accumulate;
  // zeros go past the caches where they would fill the last one (256 MiB) and
  // many rows are read meanwhile (past / through, us: 128000 rows of 1024
  // fp32, 65536 tokens 180 / 196; of 2048, 32768 tokens 271 / 282, 8192 238 /
  // 235, 48 184 / 180; of 300, 32768 tokens 80 / 74)
  O.zero_nt = vocab * dim * oe >> 28 && tokens >= vocab / 8;
  const int v = vec ? vec_elems : 1;
  O.slices = int((dim + int64_t(kWave) * v - 1) / (int64_t(kWave) * v));
  const bool few = tokens <= kFew && one_launch;
  const int64_t sum_units = few ? tokens : Z.chunks;
  const int64_t sum_blocks = (sum_units * O.slices + kWaves - 1) / kWaves;
  // rows per zero workgroup: about 64 KiB, or 256 KiB where that leaves
  // enough of them (128000 rows of 2048 fp32, 48 tokens: 191 / 180 us), or
  // 16 KiB where they would be few (4000 rows of 300, 48 tokens 7.6 / 5.9,
  // 700 tokens 22.7 / 20.6)
  const int64_t total = vocab * dim * oe;
  const int64_t most =
      (total >> 29 ? 262144 : total >> 24 ? 65536 : 16384) / (dim * oe);
  O.zero_rows = int(most < kWaves      ? kWaves
                    : most > kZeroRows ? kZeroRows
                                       : most);
  const int64_t zero_blocks =
      accumulate ? 0 : (vocab + O.zero_rows - 1) / O.zero_rows;
  // Where few rows are named, all of them are zeroed while one workgroup
  // sorts, and the named ones written again (zeros after / before, us: 700
  // tokens of 128000 rows of 2048 fp32 201 / 186, of 100000 of 1025 97 / 86;
  // a sort in tiles hides no more than it costs, 5000 tokens there 117 / 119).
  const bool zero_first =
      !few && tokens <= kOneTile && tokens < vocab / 8 &&
      zero_blocks < kMaxGrid / (kOneThreads / kBlock);
  const unsigned first = unsigned(zero_first ? zero_blocks : 0);
  const int64_t join_blocks =
      Z.chunks > 1 && !few
          ? ((Z.chunks - 1) * O.slices + kWaves - 1) / kWaves
          : 0;
  if (sum_blocks + zero_blocks > kMaxGrid) {
    set_error("%s: %lld tokens of %lld columns are too many for one call",
              what, (long long)tokens, (long long)dim);
    return FSAGG_EINVAL;
  }
  if (few) {
    with_dtype(dtype, [&](auto gt) {
      with_dtype(out_dtype, [&](auto ot) {
        constexpr int D = decltype(gt)::value, Q = decltype(ot)::value;
        const dim3 grid(unsigned(sum_blocks + zero_blocks)), block(kBlock);
        if (vec)
          hipLaunchKernelGGL((embed_few_kernel<D, Q, Elem<D>::kVec>), grid,
                             block, 0, s, P, O, int(sum_blocks));
        else
          hipLaunchKernelGGL((embed_few_kernel<D, Q, 1>), grid, block, 0, s,
                             P, O, int(sum_blocks));
      });
    });
    return check_launch(what);
  }
  int src = 0;
  if (tokens <= kOneTile) {
    src = 1;
    hipLaunchKernelGGL(embed_sort_kernel, dim3(1 + first), dim3(kOneThreads),
                       0, s, P, W, src, tokens, uint32_t(vocab), Z.passes,
                       Z.digit, O);
  } else {
    const int scanned = Z.blocks > kSumBlocks;
    for (int p = 0; p < Z.passes; ++p, src ^= 1) {
      hipLaunchKernelGGL(embed_hist_kernel, dim3(Z.blocks),
                         dim3(kTileThreads), 0, s, P, W, src, tokens,
                         uint32_t(vocab), p * Z.digit, Z.digit,
                         int(Z.blocks));
      P.n = 0;  // the keys are there
      if (scanned)
        hipLaunchKernelGGL(embed_scan_kernel, dim3(1 << Z.digit),
                           dim3(kTileThreads), 0, s, W, int(Z.blocks));
      hipLaunchKernelGGL(embed_scatter_kernel, dim3(Z.blocks),
                         dim3(kTileThreads), 0, s, W, src, tokens,
                         p * Z.digit, Z.digit, int(Z.blocks), scanned,
                         int(p + 1 == Z.passes));
    }
  }
  O.key = W.key[src];
  with_dtype(dtype, [&](auto gt) {
    with_dtype(out_dtype, [&](auto ot) {
      constexpr int D = decltype(gt)::value, Q = decltype(ot)::value;
      constexpr int V = Elem<D>::kVec;
      const dim3 grid(unsigned(sum_blocks) +
                      unsigned(zero_first ? 0 : zero_blocks)),
          block(kBlock);
      if (vec)
        hipLaunchKernelGGL((embed_sum_kernel<D, Q, V>), grid, block, 0, s, O,
                           W, int(sum_blocks));
      else
        hipLaunchKernelGGL((embed_sum_kernel<D, Q, 1>), grid, block, 0, s, O,
                           W, int(sum_blocks));
      if (join_blocks == 0) return;
      const dim3 jg{unsigned(join_blocks)};
      if (vec)
        hipLaunchKernelGGL((embed_join_kernel<Q, V>), jg, block, 0, s, O, W);
      else
        hipLaunchKernelGGL((embed_join_kernel<Q, 1>), jg, block, 0, s, O, W);
    });
  });
  return check_launch(what);
}
