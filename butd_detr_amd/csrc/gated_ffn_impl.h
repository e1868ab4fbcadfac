// gated_ffn_impl.h -- the gated feed-forward block for one tensor type T (include/butd_gated_ffn.h): the kernels around the
// tile product (ffn_tile.h) and the host-side plan.  Instantiated by gated_ffn_f32 / _bf16 / _f16.hip.
#pragma once
#include "../../include/butd_gated_ffn.h"
#include "ffn_tile.h"
#include "zero_fill.h"

#include <cmath>

namespace ffn {

// ---- few rows -----------------------------------------------------------------------------------------------------------
// Up to 16 rows, and up to 64 with small weights: the product reads every weight once and little else, so it is a stream of
// weights with 16 rows (a matrix instruction's width) per accumulator tile.  A workgroup owns 16 output columns; its waves
// share out the contraction in 128-byte pieces (whole lines of the weights' rows), load straight into fragments -- nothing is
// reused between waves, LDS would only add a trip -- and join their sums in LDS.  Bound by the weights' stream: 1 row of 4096 ->
// 11264 bf16 37.7 + 19.2 us, 4.9 TB/s; 13 rows of 2048 -> 5632 fp16 15.1 + 11.1 us, of which 3 us are a launch's and a quarter
// the rows themselves, read again for every 16 columns.  16 waves a workgroup, where there are fewer workgroups than CUs, change
// nothing for large weights and cost up to a quarter for small ones.
template <typename T, bool AL> __device__ inline u32x4 load_unit(const T *p, int left) {
  u32x4 v;
  if constexpr (AL) {
    v = left > 0 ? *(const u32x4 *)p : u32x4{0, 0, 0, 0};
  } else {
    if (left >= Num<T>::kVec) {
      __builtin_memcpy(&v, p, 16);                       // rows at odd addresses: unaligned vector loads
    } else {
      T e[Num<T>::kVec];
#pragma unroll
      for (int i = 0; i < Num<T>::kVec; ++i) e[i] = i < left ? p[i] : (T)0.f;
      __builtin_memcpy(&v, e, 16);
    }
  }
  return v;
}

struct FewRows {
  const void *x, *w0, *w1;     // ld in elements
  long ldx, ldw0, ldw1;
  int M, N, K, act;
  void *c;
  long ldc;
  int pad;
  const void *bias0, *bias1;
  float *out0, *out1;
  long ldaux;
};

template <typename T, int PARTS, int MT, bool AL>
__global__ __launch_bounds__(512) void few_rows_kernel(const FewRows P) {
  constexpr int NW = 8, kVec = Num<T>::kVec, kStep = 8 * kVec;   // 128 bytes of a row
  __shared__ f32x4 part[NW][PARTS * MT][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * 16;
  const int nrow = min(n0 + i, P.N - 1);                 // rows behind the last repeat it; their results are not stored
  const T *w[PARTS];
  w[0] = (const T *)P.w0 + (long)nrow * P.ldw0 + g * kVec;
  if constexpr (PARTS == 2) w[1] = (const T *)P.w1 + (long)nrow * P.ldw1 + g * kVec;
  const T *x[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) x[t] = (const T *)P.x + (long)min(16 * t + i, P.M - 1) * P.ldx + g * kVec;
  f32x4 acc[PARTS][MT];
#pragma unroll
  for (int p = 0; p < PARTS; ++p)
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[p][t] = f32x4{0.f, 0.f, 0.f, 0.f};
  // kAhead pieces' loads are issued before the first of them is used (units past the contraction's end arrive as zeros)
  // (more rows: fewer registers a piece and a second workgroup on the CU instead; 64 rows of 288 -> 256 fp32 15.4 -> 12.6 us)
  constexpr int kAhead = MT == 1 ? 4 : MT == 2 ? 2 : 1;
  for (int k = wave * kStep; k < P.K; k += kAhead * NW * kStep) {
    u32x4 fw[kAhead][2][PARTS], fx[kAhead][2][MT];
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const int kk = k + u * NW * kStep + s * 4 * kVec, left = P.K - kk - g * kVec;
#pragma unroll
        for (int p = 0; p < PARTS; ++p) fw[u][s][p] = load_unit<T, AL>(w[p] + kk, left);
#pragma unroll
        for (int t = 0; t < MT; ++t) fx[u][s][t] = load_unit<T, AL>(x[t] + kk, left);
      }
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int p = 0; p < PARTS; ++p)
#pragma unroll
          for (int t = 0; t < MT; ++t) acc[p][t] = mma(fw[u][s][p], fx[u][s][t], acc[p][t], (const T *)nullptr);
  }
#pragma unroll
  for (int p = 0; p < PARTS; ++p)
#pragma unroll
    for (int t = 0; t < MT; ++t) part[wave][p * MT + t][lane] = acc[p][t];
  __syncthreads();
  if (wave >= MT) return;
  const int t = wave, m = 16 * t + i, n = n0 + 4 * g;
  f32x4 sum[PARTS];
#pragma unroll
  for (int p = 0; p < PARTS; ++p) {
    sum[p] = part[0][p * MT + t][lane];
    for (int v = 1; v < NW; ++v) sum[p] += part[v][p * MT + t][lane];
  }
  if (m >= P.M) return;
  float v[PARTS][4];
#pragma unroll
  for (int p = 0; p < PARTS; ++p)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const void *bias = p ? P.bias1 : P.bias0;
      v[p][e] = sum[p][e] + (bias && n + e < P.N ? (float)((const T *)bias)[n + e] : 0.f);
    }
  T *row = (T *)P.c + (long)m * P.ldc;
  const bool whole = (P.ldc & 3) == 0 && ((uintptr_t)P.c & 15) == 0;
  if constexpr (PARTS == 2) {
    float h[4], slope[4];
    activations<4>(P.act, v[0], h, slope);
#pragma unroll
    for (int e = 0; e < 4; ++e) h[e] *= v[1][e];
    put<T>(row, n, P.N, P.pad, whole, h);
    if (P.out0) {
      put<float>(P.out0 + (long)m * P.ldaux, n, P.N, 0, true, v[0]);
      put<float>(P.out1 + (long)m * P.ldaux, n, P.N, 0, true, v[1]);
    }
  } else {
    put<T>(row, n, P.N, 0, whole, v[0]);
  }
}

// ---- rows that direct loads cannot take -----------------------------------------------------------------------------------
// One pass over the operand, in the launch before the product (x and the three weights of 1003 x 777 -> 2051 fp16: 6 us).
struct Copy {
  const void *src;
  void *dst;
  long rows, ld_src, ld_dst;   // elements
  int cols;
  long first;                  // first block
};
constexpr int kMaxCopies = 5;
struct Copies {
  Copy c[kMaxCopies];
  int count;
};
// 16-byte units of the destination, zeros behind the last column
template <typename T> __global__ __launch_bounds__(256) void copy_rows_kernel(const Copies L) {
  int ci = 0;
#pragma unroll
  for (int i = 1; i < kMaxCopies; ++i)
    if (i < L.count && (long)blockIdx.x >= L.c[i].first) ci = i;
  const Copy C = L.c[ci];
  const long unit = ((long)blockIdx.x - C.first) * 256 + threadIdx.x;
  const int per_row = (int)(C.ld_dst / Num<T>::kVec);
  const long row = unit / per_row;
  if (row >= C.rows) return;
  const int col = (int)(unit - row * per_row) * Num<T>::kVec;
  *(u32x4 *)((T *)C.dst + row * C.ld_dst + col) = load_unit<T, false>((const T *)C.src + row * C.ld_src + col, C.cols - col);
}

// ---- slabs of a split contraction -----------------------------------------------------------------------------------------
// Memory bound: every slab once (2 slabs of 2048 x 4096 and a bf16 result, 84 MB: 13.9 us).  Atomics into one slab would
// change the order of the sums from run to run.
struct Fold {
  const float *slab;
  long stride;                 // elements between slices
  int ld;                      // ... and rows of a slice
  int split, M, N;
  void *c;
  long ldc;
  const void *bias;
  long first;
};
constexpr int kMaxFolds = 2 * kMaxProblems + 1;
struct Folds {
  Fold f[kMaxFolds];
  int count;
  long blocks;
};
template <typename T> __global__ __launch_bounds__(256) void fold_kernel(const Folds L) {
  int fi = 0;
#pragma unroll
  for (int i = 1; i < kMaxFolds; ++i)
    if (i < L.count && (long)blockIdx.x >= L.f[i].first) fi = i;
  const Fold F = L.f[fi];
  const long quads = (F.N + 3) / 4, q = ((long)blockIdx.x - F.first) * 256 + threadIdx.x;
  const long m = q / quads;
  if (m >= F.M) return;
  const int n = (int)(q - m * quads) * 4;
  const float *src = F.slab + m * F.ld + n;
  float v[4] = {0.f, 0.f, 0.f, 0.f};
  if (((F.ld | F.stride) & 3) == 0) {                    // (rows padded to vectors: a column behind the last is read, not stored)
    f32x4 s = *(const f32x4 *)src;
#pragma unroll 8
    for (int i = 1; i < F.split; ++i) s += *(const f32x4 *)(src + i * F.stride);      // in slice order: reproducible
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = s[e];
  } else {
#pragma unroll 4
    for (int i = 0; i < F.split; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (n + e < F.N) v[e] += src[i * F.stride + e];
  }
  if (F.bias) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (n + e < F.N) v[e] += (float)((const T *)F.bias)[n + e];
  }
  put<T>((T *)F.c + m * F.ldc, n, F.N, 0, (F.ldc & 3) == 0 && ((uintptr_t)F.c & 15) == 0, v);
}

// ---- bias gradients: sums over chunks of rows, folded like slabs -------------------------------------------------------------
// Of dy itself, and of the column sums over each wave's rows that the product before took of da and db in 32 bits (from the
// rounded da and db the sums' error is 1.57 times that of one rounding at the end, 8192 rows).  2048 x 288 -> 2048 fp32: 4.7 us,
// a launch's.
struct ColumnSum {
  const void *src;
  long rows, ld;               // ld in elements
  int f32, cols, chunks;
  float *part;                 // (chunks, cols)
  void *out;
  int first;                   // first column block
};
struct ColumnSums {
  ColumnSum c[3];
  int count;
};
template <typename T> __device__ inline float column_sum(const T *p, long ld, long r0, long r1) {
  float s = 0.f;
#pragma unroll 8
  for (long r = r0; r < r1; r += 4) s += (float)p[r * ld];
  return s;
}
template <typename T> __global__ __launch_bounds__(256) void column_sum_kernel(const ColumnSums L) {
  int ci = 0;
#pragma unroll
  for (int i = 1; i < 3; ++i)
    if (i < L.count && (int)blockIdx.x >= L.c[i].first) ci = i;
  const ColumnSum C = L.c[ci];
  if ((int)blockIdx.y >= C.chunks) return;               // (the whole workgroup)
  const int col = ((int)blockIdx.x - C.first) * 64 + (threadIdx.x & 63), sub = threadIdx.x >> 6;
  const long per = (C.rows + C.chunks - 1) / C.chunks, r0 = blockIdx.y * per, r1 = min(C.rows, r0 + per);
  float s = 0.f;
  if (col < C.cols) {
    if (C.f32) s = column_sum((const float *)C.src + col, C.ld, r0 + sub, r1);
    else s = column_sum((const T *)C.src + col, C.ld, r0 + sub, r1);
  }
  __shared__ float sums[4][64];
  sums[sub][threadIdx.x & 63] = s;
  __syncthreads();
  if (sub == 0 && col < C.cols)
    C.part[(long)blockIdx.y * C.cols + col] = (sums[0][threadIdx.x] + sums[1][threadIdx.x]) + (sums[2][threadIdx.x] + sums[3][threadIdx.x]);
}
// ---- plan -----------------------------------------------------------------------------------------------------------------
constexpr int kCUs = 256;
constexpr long kMaxThreads = 0xffffffffL;            // a launch has to stay below 2^32 threads
constexpr long kMaxBlocks = kMaxThreads / 256;
constexpr long kMaxLd = 1L << 22;      // bytes between rows: 256 rows of a tile stay within a buffer descriptor's 2 GB

// what butd_gated_ffn_set_tile asks for, read once a call: a plan is counted and carried out with one setting.  0: the rule
struct Forced {
  int tile, split;
};

struct Arena {                         // carves the workspace; with a null base it only counts
  char *base;
  Forced forced;
  long used = 0;
  void *take(long bytes) {
    char *p = base ? base + used : nullptr;
    used += (bytes + 255) / 256 * 256;
    return p;
  }
};

enum Layout { kNT, kNN, kTN };         // A and B K-contiguous; B K-strided; both K-strided

struct TileChoice {
  int size, split;                     // 256, 128 or 64
  double us;                           // modelled
};

// Which tile, and into how many slices the contraction is cut (products whose slabs can be folded only): the smallest of the
// modelled times.  The tiles go round the chip in batches of 256 CUs x as many workgroups as a CU holds.  A step of a batch
// takes what one workgroup's step takes alone (latency) or what the multiplications of all workgroups of a CU take,
// whichever is more; `fill` steps pass before the first and behind the last; the epilogue's bytes take the memory's time,
// hidden in part where another workgroup of the CU computes meanwhile.  Slabs are written and read once, plus a launch.
// The operands' bytes at 5.5 TB/s overlap with that in part (root of the squares' sum).  Constants fitted to 120 measured launches of 16 shapes
// (1 .. 8192 rows x 200 .. 4096 x 256 .. 11264, both widths of types): the chosen tile was the fastest one in 3 of 4 and at
// most 18 % slower in the rest.
struct Shape {
  long M, N;
};
struct TileModel {
  int size;
  double latency_us, rate, fill;       // rate: multiply-adds per CU and microsecond with all CUs at work
  int resident;                        // workgroups of a CU
};
template <typename T> inline TileChoice choose(Forced forced, const Shape *shapes, int count, long k, int segments, bool can_split, double epilogue_bytes) {
  if (forced.tile) return TileChoice{sizeof(T) == 4 && forced.tile == 256 ? 128 : forced.tile, can_split ? forced.split : 1, 0.0};
  static const TileModel models16[3] = {{64, 0.49, 1.15e6, 2.0, 4}, {128, 0.65, 1.75e6, 3.0, 2}, {256, 1.2, 2.4e6, 3.0, 1}};
  static const TileModel models32[2] = {{64, 0.60, 0.245e6, 1.5, 4}, {128, 2.0, 0.258e6, 1.5, 2}};
  static const int splits[] = {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64};
  const TileModel *models = sizeof(T) == 2 ? models16 : models32;
  constexpr int bk = Num<T>::kBK;
  const long steps = (k + bk - 1) / bk * segments;
  TileChoice best{64, 1, 1e30};
  double operands = 0;
  for (int i = 0; i < count; ++i) operands += (double)(shapes[i].M + shapes[i].N) * (double)k * segments * sizeof(T);
  for (int c = 0; c < (sizeof(T) == 2 ? 3 : 2); ++c) {
    const TileModel &m = models[c];
    // (a tile with twice the rows that there are: 24 rows of 11264 -> 4096 bf16 24 us with the 128 tile, 18 with the 64)
    if (count == 1 && shapes[0].M * 2 <= m.size && m.size > 64) break;
    const double area = (double)m.size * m.size, resident = kCUs * m.resident;
    double tiles = 0, elems = 0;
    for (int i = 0; i < count; ++i) {
      tiles += (double)((shapes[i].M + m.size - 1) / m.size) * (double)((shapes[i].N + m.size - 1) / m.size);
      elems += (double)shapes[i].M * (double)shapes[i].N;
    }
    if (m.size < 256 && tiles * 256.0 > (double)kMaxThreads) continue;       // (only a larger tile's launch has room for them)
    for (int s : splits) {
      if (s > 1 && (!can_split || steps < 3L * s)) break;
      const double turn = (double)((steps + s - 1) / s) + m.fill, bytes = s == 1 ? epilogue_bytes : 4.0;
      const double all = tiles * s, full = (double)(long)(all / resident);
      auto batch = [&](double workgroups) {
        // a CU with one workgroup more than the others sets the time; with part of the chip idle the 16-bit matrix cores
        // clock higher
        const double per_cu = workgroups / kCUs, most = (double)(long)(per_cu + 0.999);
        const double step = most * area * bk / m.rate * (sizeof(T) == 4 ? 1.0 : 0.6 + 0.4 * per_cu / most);
        return turn * (step > m.latency_us ? step : m.latency_us) + per_cu * area * bytes / 2e4 * (m.resident == 1 ? 1.2 : 0.6);
      };
      double us = full * batch(resident);
      if (all > full * resident) us += batch(all - full * resident);
      us = 3.0 + sqrt(us * us + operands / 5.5e6 * (operands / 5.5e6));
      if (s > 1) us += 3.5 + elems * (4.0 * s + sizeof(T)) / 4.5e6;
      if (us < best.us) best = TileChoice{m.size, s, us};
    }
  }
  return best;
}

// The streaming kernel's time: the weights once and the rows again for every 16 columns (from L2; padded to 32 or 64), but
// not less than one workgroup's way along the contraction, 128 bytes a wave at a time.
template <typename T> inline double few_rows_us(long M, long N, long K, int parts) {
  const double tiles = M <= 32 ? 2 : 4, weights = (double)N * K * sizeof(T);
  const double all = weights * parts / 5.6e6 + tiles * weights / 6.5e6;
  const double one = (double)((K * (long)sizeof(T) + 1023) / 1024) * (0.25 + 0.45 * tiles);
  return 3.0 + (all > one ? all : one);
}

// run == false, here and below: only what would be refused
template <class C> inline hipError_t launch_tiles(Launch &L, bool run, hipStream_t stream) {
  constexpr int nw = C::kind == kGateUp ? C::TN / 2 : C::TN, bk = Num<typename C::type>::kBK;
  long total = 0;
  int slices = 1;
  for (int i = 0; i < L.count; ++i) {
    Problem &p = L.p[i];
    if constexpr (C::kind != kPlain) {                   // the epilogue of h, a, b, da and db knows whole vectors only
      const uintptr_t at = (uintptr_t)p.c | (uintptr_t)p.c2 | (uintptr_t)p.aux0 | (uintptr_t)p.aux1 |
                           (C::kind == kGateUp ? (uintptr_t)p.out0 | (uintptr_t)p.out1 : 0);
      if (p.pad < p.N || (p.pad | p.ldc | p.ldaux) & 3 || at & 15) return hipErrorInvalidValue;
    }
    const long tm = ((long)p.M + C::TM - 1) / C::TM, tn = ((long)p.N + nw - 1) / nw;
    if (tm * tn > kMaxThreads / C::kThreads - total) return hipErrorInvalidValue;
    p.tiles_m = (int)tm;
    p.tiles_n = (int)tn;
    p.first = (int)total;
    p.steps = (int)(((long)p.K + bk - 1) / bk) * p.segments;
    p.per_slice = (p.steps + p.split - 1) / p.split;
    p.group_magic = (uint32_t)((1ULL << 32) / (8ULL * (uint64_t)tn)) + 1;
    total += tm * tn;
    if (p.split > slices) slices = p.split;
  }
  L.total = (int)total;
  if (!run) return hipSuccess;
  hipLaunchKernelGGL((tile_kernel<C>), dim3((unsigned)total, (unsigned)slices), dim3(C::kThreads), 0, stream, L);
  return hipGetLastError();
}

// The tile kernels of one type.  (Named here: from the launches alone hipcc leaves the host side of some of them out.)
#define BUTD_FFN_TILES(T, TM, WM, WN, WM1, WN1)                                                \
  template __global__ void tile_kernel<Config<T, kGateUp, true, true, TM, TM, WM1, WN1>>(const Launch); \
  template __global__ void tile_kernel<Config<T, kPlain, true, true, TM, TM, WM, WN>>(const Launch);   \
  template __global__ void tile_kernel<Config<T, kPlain, true, false, TM, TM, WM, WN>>(const Launch);  \
  template __global__ void tile_kernel<Config<T, kPlain, false, false, TM, TM, WM, WN>>(const Launch); \
  template __global__ void tile_kernel<Config<T, kGrad, true, false, TM, TM, WM, WN>>(const Launch);

// The three tiles of every kind.  The smallest of kGateUp has its waves stacked along m: a wave holds both parts of its columns.
template <typename T, int KIND, Layout LAY> inline hipError_t run_tiles(Launch &L, int size, bool run, hipStream_t stream) {
  constexpr bool ak = LAY != kTN, bk = LAY == kNT;
  if constexpr (sizeof(T) == 2) {
    if (size == 256) return launch_tiles<Config<T, KIND, ak, bk, 256, 256, 2, 4>>(L, run, stream);
  }
  if (size == 128) return launch_tiles<Config<T, KIND, ak, bk, 128, 128, 2, 2>>(L, run, stream);
  if constexpr (KIND == kGateUp) return launch_tiles<Config<T, KIND, ak, bk, 64, 64, 4, 1>>(L, run, stream);
  else return launch_tiles<Config<T, KIND, ak, bk, 64, 64, 2, 2>>(L, run, stream);
}

template <typename T> struct Block {
  static constexpr int kVec = Num<T>::kVec;
  static constexpr long kFewRows = 64;

  // an operand as the tile product takes it: itself, or a copy with aligned rows in the workspace
  struct Operand {
    const void *p;
    long ld;                                             // elements
  };
  struct Packer {
    Arena &ws;
    Copies L;
    long blocks = 0;
    explicit Packer(Arena &a) : ws(a) { L.count = 0; }
    static bool direct(const void *p, long ld, int cols) {
      return ((uintptr_t)p & 15) == 0 && ld % kVec == 0 && cols % kVec == 0 && ld * (long)sizeof(T) <= kMaxLd;
    }
    Operand pack(const void *p, long ld, long rows, int cols) {
      const long ld_dst = (cols + kVec - 1) / kVec * kVec;
      void *dst = ws.take(rows * ld_dst * (long)sizeof(T));
      L.c[L.count++] = Copy{p, dst, rows, ld, ld_dst, cols, blocks};
      blocks += (rows * (ld_dst / kVec) + 255) / 256;
      return Operand{dst, ld_dst};
    }
    Operand take(const void *p, long ld, long rows, int cols) {
      return direct(p, ld, cols) ? Operand{p, ld} : pack(p, ld, rows, cols);
    }
    hipError_t launch(bool run, hipStream_t stream) {
      if (!L.count) return hipSuccess;
      if (blocks > kMaxBlocks) return hipErrorInvalidValue;
      if (!run) return hipSuccess;
      hipLaunchKernelGGL((copy_rows_kernel<T>), dim3((unsigned)blocks), dim3(256), 0, stream, L);
      return hipGetLastError();
    }
  };
  static bool direct_pair(const butd_gated_ffn_args &A) {
    return A.ld_gate == A.ld_up && Packer::direct(A.w_gate, A.ld_gate, A.width) && Packer::direct(A.w_up, A.ld_up, A.width);
  }
  static bool direct_in(const butd_gated_ffn_args &A) { return direct_pair(A) && Packer::direct(A.x, A.ld_x, A.width); }
  // the two projections share one row stride in the product
  static void take_pair(Packer &pk, const butd_gated_ffn_args &A, Operand &gate, Operand &up) {
    if (direct_pair(A)) {
      gate = Operand{A.w_gate, A.ld_gate};
      up = Operand{A.w_up, A.ld_up};
    } else {
      gate = pk.pack(A.w_gate, A.ld_gate, A.hidden, A.width);
      up = pk.pack(A.w_up, A.ld_up, A.hidden, A.width);
    }
  }
  static void operands(Problem &p, Operand a, Operand b) {
    p.a[0] = p.a[1] = a.p;
    p.b[0] = p.b[1] = b.p;
    p.lda = a.ld * (long)sizeof(T);
    p.ldb = b.ld * (long)sizeof(T);
    p.segments = 1;
    p.split = 1;
  }
  static void add_fold(Folds &F, const float *slab, long stride, int ld, int split, int M, int N, void *c, long ldc, const void *bias) {
    F.f[F.count++] = Fold{slab, stride, ld, split, M, N, c, ldc, bias, F.blocks};
    F.blocks += ((long)M * ((N + 3) / 4) + 255) / 256;
  }
  static void add_folds(Folds &F, const Launch &L) {
    for (int i = 0; i < L.count; ++i) {
      const Problem &p = L.p[i];
      if (p.split > 1) add_fold(F, p.slab, p.slab_stride, slab_ld(p.N), p.split, p.M, p.N, p.c, p.ldc, p.bias0);
    }
  }
  static hipError_t run_folds(const Folds &F, bool run, hipStream_t stream) {
    if (!F.count) return hipSuccess;
    if (F.blocks > kMaxBlocks) return hipErrorInvalidValue;
    if (!run) return hipSuccess;
    hipLaunchKernelGGL((fold_kernel<T>), dim3((unsigned)F.blocks), dim3(256), 0, stream, F);
    return hipGetLastError();
  }
  static hipError_t fold(const Launch &L, bool run, hipStream_t stream) {
    Folds F{};
    add_folds(F, L);
    return run_folds(F, run, stream);
  }
  static void slabs(Launch &L, int split, Arena &ws) {
    for (int i = 0; i < L.count; ++i) {
      Problem &p = L.p[i];
      const int steps = (p.K + Num<T>::kBK - 1) / Num<T>::kBK * p.segments;
      const int per = (steps + split - 1) / split;
      p.split = (steps + per - 1) / per;                 // every slice owns at least one step
      if (p.split > 1) {
        p.slab_stride = (long)p.M * slab_ld(p.N);
        p.slab = (float *)ws.take(p.slab_stride * p.split * 4);
      }
    }
  }

  template <int PARTS> static hipError_t few_rows(const FewRows &P, bool run, hipStream_t stream) {
    if (!run) return hipSuccess;
    const bool al = (((uintptr_t)P.x | (uintptr_t)P.w0 | (uintptr_t)P.w1) & 15) == 0 && P.ldx % kVec == 0 && P.ldw0 % kVec == 0 &&
                    P.ldw1 % kVec == 0 && P.K % kVec == 0;
    const dim3 grid((unsigned)((P.N + 15) / 16));
#define BUTD_FEW_ROWS(MT, AL) hipLaunchKernelGGL((few_rows_kernel<T, PARTS, MT, AL>), grid, dim3(512), 0, stream, P)
    if (P.M <= 16) {
      if (al) BUTD_FEW_ROWS(1, true); else BUTD_FEW_ROWS(1, false);
    } else if (P.M <= 32) {
      if (al) BUTD_FEW_ROWS(2, true); else BUTD_FEW_ROWS(2, false);
    } else {
      if (al) BUTD_FEW_ROWS(4, true); else BUTD_FEW_ROWS(4, false);
    }
#undef BUTD_FEW_ROWS
    return hipGetLastError();
  }

  // run == false: count the workspace and refuse what a launch cannot hold; nothing is launched
  static hipError_t forward(const butd_gated_ffn_args &A, Arena &ws, bool run, hipStream_t stream) {
    const int M = (int)A.rows, E = A.width, F = A.hidden;
    if (M == 0) return hipSuccess;
    hipError_t err;
    // Each product of up to 16 rows is streamed, and of 17 to 64 rows where tiles would be modelled slower or need copies
    // (bf16, 4096 -> 11264 -> 4096, streamed / tiles: 16 rows 64 / 73 us, 24 rows 81 / 73, 64 rows 132 / 79;
    // 512 -> 2048 -> 512: 24 rows 10.9 / 14.2, 64 rows 16.8 / 14.4; 288 -> 256 -> 288: 64 rows 7.6 / 9.3; fp32, 512 -> 2048
    // -> 512, 64 rows 32.5 / 24.4, the first product streamed and the second on tiles 21.6)
    const Shape gs{M, 2L * F}, ds{M, E};
    const TileChoice gc = choose<T>(ws.forced, &gs, 1, E, 1, false, (A.a ? 8 + sizeof(T) : sizeof(T)) / 2.0),
                     dc = choose<T>(ws.forced, &ds, 1, F, 1, true, sizeof(T));
    const bool few = M <= kFewRows && !ws.forced.tile;
    const bool stream_in = few && (M <= 16 || !direct_in(A) || few_rows_us<T>(M, F, E, 2) <= gc.us);
    const bool stream_out = few && (M <= 16 || !Packer::direct(A.w_down, A.ld_down, F) || few_rows_us<T>(M, E, F, 1) <= dc.us);
    Packer pk(ws);
    Launch G{}, D{};
    if (!stream_in) {
      Operand x = pk.take(A.x, A.ld_x, M, E), gate, up;
      take_pair(pk, A, gate, up);
      G.count = 1;
      G.act = A.activation;
      Problem &g = G.p[0];
      operands(g, x, gate);
      g.b[1] = up.p;
      g.M = M; g.N = F; g.K = E;
      g.c = A.h; g.ldc = A.ld_h; g.pad = (int)A.ld_h;
      g.bias0 = A.b_gate; g.bias1 = A.b_up;
      g.out0 = A.a; g.out1 = A.b; g.ldaux = A.ld_h;
    }
    if (!stream_out) {
      Operand down = pk.take(A.w_down, A.ld_down, E, F);
      D.count = 1;
      Problem &d = D.p[0];
      operands(d, Operand{A.h, A.ld_h}, down);
      d.M = M; d.N = E; d.K = F;
      d.c = A.y; d.ldc = A.ld_y; d.bias0 = A.b_down;
      slabs(D, dc.split, ws);
    }
    if ((err = pk.launch(run, stream)) != hipSuccess) return err;
    if (stream_in) {
      FewRows P{A.x, A.w_gate, A.w_up, A.ld_x, A.ld_gate, A.ld_up, M, F, E, A.activation, A.h, A.ld_h, (int)A.ld_h,
                A.b_gate, A.b_up, A.a, A.b, A.ld_h};
      err = few_rows<2>(P, run, stream);
    } else {
      err = run_tiles<T, kGateUp, kNT>(G, gc.size, run, stream);
    }
    if (err != hipSuccess) return err;
    if (stream_out) {
      FewRows P{A.h, A.w_down, A.w_down, A.ld_h, A.ld_down, A.ld_down, M, E, F, A.activation, A.y, A.ld_y, 0,
                A.b_down, nullptr, nullptr, nullptr, 0};
      return few_rows<1>(P, run, stream);
    }
    if ((err = run_tiles<T, kPlain, kNT>(D, dc.size, run, stream)) != hipSuccess) return err;
    return fold(D, run, stream);
  }

  static hipError_t backward(const butd_gated_ffn_args &A, Arena &ws, bool run, hipStream_t stream) {
    const int M = (int)A.rows, E = A.width, F = A.hidden;
    hipError_t err;
    const bool inner = A.dx || A.dw_gate || A.dw_up || A.db_gate || A.db_up;    // da, db wanted
    if (M == 0) {                                        // sums over nothing
      if (!run) return hipSuccess;
      void *const w[3] = {A.dw_gate, A.dw_up, A.dw_down}, *const b[3] = {A.db_gate, A.db_up, A.db_down};
      for (int i = 0; i < 3; ++i) {
        if (w[i] && (err = butd_zero_async(w[i], (size_t)E * F * sizeof(T), stream)) != hipSuccess) return err;
        if (b[i] && (err = butd_zero_async(b[i], (size_t)(i == 2 ? E : F) * sizeof(T), stream)) != hipSuccess) return err;
      }
      return hipSuccess;
    }
    Packer pk(ws);
    Operand x{}, gate{}, up{}, down{}, dy{};
    if (inner || A.dw_down) dy = pk.take(A.dy, A.ld_dy, M, E);
    if (A.dw_gate || A.dw_up) x = pk.take(A.x, A.ld_x, M, E);
    if (A.dx) take_pair(pk, A, gate, up);
    Operand da{}, db{};
    Launch G{}, X{}, W{};
    TileChoice gc{}, xc{}, wc{};
    if (inner) {
      down = pk.take(A.w_down, A.ld_down, E, F);
      da = Operand{ws.take(A.ld_h * (long)M * (long)sizeof(T)), A.ld_h};
      db = Operand{ws.take(A.ld_h * (long)M * (long)sizeof(T)), A.ld_h};
      G.count = 1;
      G.act = A.activation;
      Problem &g = G.p[0];
      operands(g, dy, down);
      g.M = M; g.N = F; g.K = E;
      g.c = (void *)da.p; g.c2 = (void *)db.p; g.ldc = A.ld_h; g.pad = (int)A.ld_h;
      g.aux0 = A.a; g.aux1 = A.b; g.ldaux = A.ld_h;
      const Shape s{M, F};
      gc = choose<T>(ws.forced, &s, 1, E, 1, false, 8 + 2 * sizeof(T));
    }
    if (A.dx) {
      X.count = 1;
      Problem &p = X.p[0];
      operands(p, da, gate);
      p.a[1] = db.p; p.b[1] = up.p;
      p.segments = 2;
      p.M = M; p.N = E; p.K = F;
      p.c = A.dx; p.ldc = A.ld_dx;
      const Shape s{M, E};
      xc = choose<T>(ws.forced, &s, 1, F, 2, true, sizeof(T));
      slabs(X, xc.split, ws);
    }
    Shape ws_shapes[3];
    auto weight = [&](Operand a, Operand b, int m, int n, void *c) {
      ws_shapes[W.count] = Shape{m, n};
      Problem &p = W.p[W.count++];
      operands(p, a, b);
      p.M = m; p.N = n; p.K = M;
      p.c = c; p.ldc = n;
    };
    if (A.dw_gate) weight(da, x, F, E, A.dw_gate);
    if (A.dw_up) weight(db, x, F, E, A.dw_up);
    if (A.dw_down) weight(dy, Operand{A.h, A.ld_h}, E, F, A.dw_down);
    if (W.count) {
      wc = choose<T>(ws.forced, ws_shapes, W.count, M, 1, true, sizeof(T));
      slabs(W, wc.split, ws);
    }
    // bias gradients: column sums of da, db, dy in row chunks
    ColumnSums S;
    S.count = 0;
    int blocks = 0, chunks = 0;
    auto column = [&](const void *src, bool f32, long rows, long ld, int cols, void *out) {
      S.c[S.count++] = ColumnSum{src, rows, ld, f32, cols, 0, nullptr, out, blocks};
      blocks += (cols + 63) / 64;
    };
    if (A.db_gate || A.db_up) {
      const long parts = ((long)M + gc.size - 1) / gc.size * kWavesM;
      Problem &g = G.p[0];
      if (A.db_gate) column(g.out0 = (float *)ws.take(parts * F * 4), true, parts, F, F, A.db_gate);
      if (A.db_up) column(g.out1 = (float *)ws.take(parts * F * 4), true, parts, F, F, A.db_up);
    }
    if (A.db_down) column(A.dy, sizeof(T) == 4, M, A.ld_dy, E, A.db_down);
    for (int i = 0; i < S.count; ++i) {
      // about four workgroups per CU, at least 32 rows each, few enough for one thread to fold
      ColumnSum &c = S.c[i];
      const long want = (4L * kCUs + blocks - 1) / blocks, rows = (c.rows + 31) / 32, most = rows < 48 ? rows : 48;
      c.chunks = (int)(want > most ? most : want);
      c.part = (float *)ws.take((long)c.chunks * c.cols * 4);
      if (c.chunks > chunks) chunks = c.chunks;
    }
    if ((err = pk.launch(run, stream)) != hipSuccess) return err;
    if (inner && (err = run_tiles<T, kGrad, kNN>(G, gc.size, run, stream)) != hipSuccess) return err;
    if (S.count && run) {
      hipLaunchKernelGGL((column_sum_kernel<T>), dim3((unsigned)blocks, (unsigned)chunks), dim3(256), 0, stream, S);
      if ((err = hipGetLastError()) != hipSuccess) return err;
    }
    if (A.dx && (err = run_tiles<T, kPlain, kNN>(X, xc.size, run, stream)) != hipSuccess) return err;
    if (W.count && (err = run_tiles<T, kPlain, kTN>(W, wc.size, run, stream)) != hipSuccess) return err;
    // the slabs of dx and of the weight gradients and the bias gradients' row chunks in one launch
    Folds last{};
    add_folds(last, X);
    add_folds(last, W);
    for (int i = 0; i < S.count; ++i) add_fold(last, S.c[i].part, S.c[i].cols, S.c[i].cols, S.c[i].chunks, 1, S.c[i].cols, S.c[i].out, S.c[i].cols, nullptr);
    return run_folds(last, run, stream);
  }
};

}  // namespace ffn
