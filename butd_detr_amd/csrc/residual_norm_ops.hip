// residual_norm_ops.hip -- norms before and after a block with its gate and residual scale (include/butd_residual_norm.h).
//
// Memory bound: forward reads x and residual and writes stream and normed, backward reads x, residual and the two arriving
// gradients and writes two.  A row's values stay in registers from the load to the last use (both norms' statistics are
// sums over registers, the deviations taken around the mean, not as a difference of squares), so each tensor is touched
// once.  Measured (16384 rows of 4096, bf16 on a 32-bit stream, RMSNorm on both sides, a gate per channel): forward 146 us,
// backward 239 us, sums of the parameters' gradients 4.7 us -- 5.5, 5.1 TB/s (a large copy: 5.15); 8192 rows of 8192 bf16 forward
// 98 us, 5.5 TB/s.  2048 rows of 288 fp32, the layers' own: 5.6, 9.6 and 4.1 us, launches more than bytes.
// Rows of up to 512 elements belong to ONE wave and are reduced inside it; wider rows to a workgroup.  Rows of any
// width and address, 16 bytes a lane.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/butd_residual_norm.h"
#include "zero_fill.h"

#ifndef BUTD_MAIN_PRIO
#define BUTD_MAIN_PRIO 0
#endif

namespace {

typedef butd_residual_norm_args Args;
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int N = 8;           // consecutive elements of a row in a thread: 16 bytes of a 16-bit tensor, two loads of a 32-bit one

// How threads share a row out, N elements each, the first `left` of them existing.
//   kWhole     a length that is a multiple of N: all of a thread's elements exist, or none
//   kOverlap   any other length above N: the last unit is moved back to end with the row, so every access is a whole unit.
//              The first `twice` elements of it are its neighbour's too: both threads compute and write the same values, and
//              the row's sums take the neighbour's.  (1537 fp16 columns, 3003 rows: backward 24 us; 35 with the last
//              unit element by element, whose eight predicates for every tensor spill scalar registers.)
//   kElements  rows shorter than N
enum Mode { kWhole, kOverlap, kElements };

// ---- N consecutive elements of type T at any address, `left` of them existing --------------------------------------------
template <Mode MODE, typename T> __device__ inline void load(const T *p, int left, float *v) {
  if (MODE != kElements ? left > 0 : left >= N) {
    T e[N];
    __builtin_memcpy(e, p, N * sizeof(T));
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = (float)e[i];
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = MODE == kElements && i < left ? (float)p[i] : 0.f;
  }
}
template <Mode MODE, typename T> __device__ inline void store(T *p, int left, const float *v) {
  if (MODE != kElements ? left > 0 : left >= N) {
    T e[N];
#pragma unroll
    for (int i = 0; i < N; ++i) e[i] = (T)v[i];
    __builtin_memcpy(p, e, N * sizeof(T));
  } else if (MODE == kElements) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < left) p[i] = (T)v[i];
  }
}
// the same elements as they lie in memory, loaded now and widened later.  (Held in 32-bit words: 16-bit elements that are
// loaded on one side of a branch and zero on the other are packed there, which waits for the load.)
template <Mode MODE, typename T> struct Raw {
  static constexpr int kWords = N * sizeof(T) / 4;
  uint32_t words[kWords];
  __device__ inline void load(const T *p, int left) {
#pragma unroll
    for (int i = 0; i < kWords; ++i) words[i] = 0;
    if (MODE != kElements ? left > 0 : left >= N) {
      __builtin_memcpy(words, p, sizeof(words));
    } else if (MODE == kElements) {
      T e[N];
#pragma unroll
      for (int i = 0; i < N; ++i) e[i] = i < left ? p[i] : (T)0.f;
      __builtin_memcpy(words, e, sizeof(words));
    }
  }
  __device__ inline void widen(float *v) const {
    T e[N];
    __builtin_memcpy(e, words, sizeof(words));
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = (float)e[i];
  }
};
// parameters: the type of x or 32 bits; one that is not there is `value`.  Behind the row's end: zeros, which keeps the
// elements there out of every sum without a test.
template <Mode MODE, typename T> __device__ inline void load_param(const void *p, bool f32, long at, int left, float value, float *v) {
  if (!p) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = (MODE != kElements ? 0 : i) < left ? value : 0.f;
  } else if (f32) {
    load<MODE, float>((const float *)p + at, left, v);
  } else {
    load<MODE, T>((const T *)p + at, left, v);
  }
}

// sum over the wave, in every lane (data-parallel primitives: no LDS)
template <int CTRL, int ROWS> __device__ inline float dpp_add(float v) {
  return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, ROWS, 0xf, false));
}
__device__ inline float wave_sum(float v) {
  v = dpp_add<0x111, 0xf>(v);                            // row_shr 1, 2, 4, 8: lane 15 of a row has the row's sum
  v = dpp_add<0x112, 0xf>(v);
  v = dpp_add<0x114, 0xf>(v);
  v = dpp_add<0x118, 0xf>(v);
  v = dpp_add<0x142, 0xa>(v);                            // row_bcast 15 into rows 1 and 3
  v = dpp_add<0x143, 0xc>(v);                            // row_bcast 31 into rows 2 and 3
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}
// sums of K values over the TPR threads of a row.  Two buffers in turn: one barrier a call.
template <int TPR, int K> struct RowSum {
  static constexpr int kWaves = TPR / 64;
  float (*buf)[kWaves][K];                               // [2][waves][K]
  int turn = 0;
  __device__ inline void operator()(float *v) {
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = wave_sum(v[k]);
    if constexpr (TPR > 64) {
      const int wave = threadIdx.x >> 6;
      if ((threadIdx.x & 63) == 0) {
#pragma unroll
        for (int k = 0; k < K; ++k) buf[turn][wave][k] = v[k];
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < K; ++k) {
        float s = buf[turn][0][k];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) s += buf[turn][w][k];
        v[k] = s;
      }
      turn ^= 1;
    }
  }
};

// A workgroup: kRows rows side by side (one wave each), or one row on all its threads
template <int TPR> struct Group {
  static constexpr int kThreads = TPR == 64 ? 256 : TPR;
  static constexpr int kRows = kThreads / TPR;
};

template <typename T, typename R, int TPR, Mode MODE>
__global__ __launch_bounds__(Group<TPR>::kThreads, TPR == 1024 ? 8 : 1) void forward_kernel(const Args A, const long row0) {
  __shared__ float sums[2][TPR / 64][1];
  __builtin_amdgcn_s_setprio(BUTD_MAIN_PRIO);
  RowSum<TPR, 1> row_sum{sums};
  const int sub = threadIdx.x / TPR, th = threadIdx.x % TPR, cols = A.cols;
  const int twice = MODE == kOverlap && th * N < cols ? max(th * N + N - cols, 0) : 0;
  const int c = th * N - twice, left = cols - c;
  const long row = row0 + (long)blockIdx.x * Group<TPR>::kRows + sub, at = row * cols + c;
  if (row >= A.rows) return;                             // (whole waves, or the whole workgroup)
  // everything the row needs is on its way before the first sum
  float x[N], r[N], w1[N], b1[N], g[N];
  load<MODE, T>((const T *)A.x + at, left, x);
  if (A.residual) load<MODE, R>((const R *)A.residual + at, left, r);
  const long gate_row = A.gate_kind == BUTD_GATE_ELEMENT ? row : A.gate_kind == BUTD_GATE_SAMPLE ? row / A.rows_per_sample : 0;
  load_param<MODE, T>(A.gate, A.gate_dtype == BUTD_NORM_F32, gate_row * cols + c, left, 1.f, g);
  if (A.post_kind) {
    load_param<MODE, T>(A.post_weight, A.post_dtype == BUTD_NORM_F32, c, left, 1.f, w1);
    load_param<MODE, T>(A.post_bias, A.post_dtype == BUTD_NORM_F32, c, left, 0.f, b1);
  }
  // v -> (v - mean) / deviation
  auto normalise = [&](float *v, int kind, float eps, float *stats) {
    float mean = 0.f;
    if (kind == BUTD_NORM_LAYER) {
      float s[1] = {0.f};
#pragma unroll
      for (int i = 0; i < N; ++i) s[0] += i >= twice ? v[i] : 0.f;
      row_sum(s);
      mean = s[0] / (float)cols;
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = (MODE != kElements ? 0 : i) < left ? v[i] - mean : 0.f;
    }
    float s[1] = {0.f};
#pragma unroll
    for (int i = 0; i < N; ++i) s[0] += i >= twice ? v[i] * v[i] : 0.f;
    row_sum(s);
    const float rstd = 1.f / sqrtf(s[0] / (float)cols + eps);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] *= rstd;
    if (stats && th == 0) {
      stats[row] = mean;
      stats[A.rows + row] = rstd;
    }
  };
  if (A.post_kind) {
    normalise(x, A.post_kind, A.post_eps, A.stats);
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = x[i] * w1[i] + b1[i];
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    x[i] *= g[i];
    if (A.residual) x[i] += A.residual_scale * r[i];
  }
  if (A.stream) store<MODE, R>((R *)A.stream + at, left, x);
  if (!A.pre_kind) return;
  float w2[N], b2[N];                                    // on their way during the second norm's sums
  load_param<MODE, T>(A.pre_weight, A.pre_dtype == BUTD_NORM_F32, c, left, 1.f, w2);
  load_param<MODE, T>(A.pre_bias, A.pre_dtype == BUTD_NORM_F32, c, left, 0.f, b2);
  normalise(x, A.pre_kind, A.pre_eps, A.stats ? A.stats + 2 * A.rows : nullptr);
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = x[i] * w2[i] + b2[i];
  store<MODE, T>((T *)A.normed + at, left, x);
}

// ---- backward --------------------------------------------------------------------------------------------------------------
// 180 to 220 registers a thread (four or five column sums of eight elements each, parameters, a row), so two waves a SIMD and
// nobody to cover for a row's loads: the next row's are issued first (16384 rows of 4096: 307 -> 255 us).
// A workgroup owns consecutive rows, [first, last) of one run of samples, and keeps its threads' column sums in registers:
//   part[workgroup][4][cols]: d_post_weight, d_post_bias, d_pre_weight, d_pre_bias;   gate_part[slot][cols]
// Gate per sample: the rows of a workgroup are either whole samples (slot = sample, written as each sample ends) or part of
// one sample (slot = workgroup, `share` of them a sample).  Gate per channel: slot = workgroup.
struct Plan {
  long per;                    // rows of a workgroup
  long share;                  // workgroups of a run
  long run;                    // rows of a run: rows_per_sample where samples are cut up, else all rows
  long blocks, slots;
  float *part, *gate_part;
};

enum { kPostW = 0, kPostB, kPreW, kPreB };

template <typename T, typename R, int TPR, Mode MODE>
__global__ __launch_bounds__(Group<TPR>::kThreads) void backward_kernel(const Args A, const Plan P) {
  constexpr int kRows = Group<TPR>::kRows;
  __shared__ float sums[2][TPR / 64][2];
  __shared__ float joined[kRows > 1 ? kRows : 1][kRows > 1 ? 64 * N : 1];
  __builtin_amdgcn_s_setprio(BUTD_MAIN_PRIO);
  RowSum<TPR, 2> row_sum{sums};
  const int sub = threadIdx.x / TPR, th = threadIdx.x % TPR, cols = A.cols;
  const int twice = MODE == kOverlap && th * N < cols ? max(th * N + N - cols, 0) : 0;
  const int c = th * N - twice, left = cols - c;
  const float inv_cols = 1.f / (float)cols;
  const long run = blockIdx.x / P.share, piece = blockIdx.x - run * P.share;
  const long first = run * P.run + piece * P.per, last = min(first + P.per, min((run + 1) * P.run, A.rows));
  const bool post = A.post_kind != 0, pre = A.pre_kind != 0 && A.d_normed != nullptr;
  // a segment: rows that share a slot of the gate's sums
  const bool by_sample = A.gate_kind == BUTD_GATE_SAMPLE, by_element = A.gate_kind == BUTD_GATE_ELEMENT;
  const long segment = by_sample ? A.rows_per_sample : A.rows;

  float w1[N], b1[N], w2[N], g[N];
  load_param<MODE, T>(post ? A.post_weight : nullptr, A.post_dtype == BUTD_NORM_F32, c, left, 1.f, w1);
  load_param<MODE, T>(post ? A.post_bias : nullptr, A.post_dtype == BUTD_NORM_F32, c, left, 0.f, b1);
  load_param<MODE, T>(pre ? A.pre_weight : nullptr, A.pre_dtype == BUTD_NORM_F32, c, left, 1.f, w2);
  // column sums: a thread's own, in registers; those of a row on 1024 threads (128 registers each) in LDS
  constexpr bool kInLds = TPR == 1024;
  constexpr int kSums = kInLds ? 1 : 4;
  __shared__ f32x4 shared_sums[kInLds ? 4 : 1][2][kInLds ? TPR : 1];
  float sum[kSums][N], sum_g[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
#pragma unroll
    for (int k = 0; k < kSums; ++k) sum[k][i] = 0.f;
    sum_g[i] = 0.f;
  }
  if constexpr (kInLds) {
#pragma unroll
    for (int k = 0; k < 4; ++k) shared_sums[k][0][th] = shared_sums[k][1][th] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  auto add = [&](int k, const float *v) {
    if constexpr (kInLds) {
      shared_sums[k][0][th] += f32x4{v[0], v[1], v[2], v[3]};
      shared_sums[k][1][th] += f32x4{v[4], v[5], v[6], v[7]};
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) sum[k][i] += v[i];
    }
  };
  auto total = [&](int k, float *v) {
    if constexpr (kInLds) {
      __builtin_memcpy(v, &shared_sums[k][0][th], 16);
      __builtin_memcpy(v + 4, &shared_sums[k][1][th], 16);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = sum[k][i];
    }
  };

  // column sums of the workgroup: over its rows side by side through LDS, then out
  auto flush = [&](const float *own, float *dst) {
    if constexpr (kRows > 1) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < N; ++i) joined[sub][i * 64 + th] = own[i];
      __syncthreads();
      if (sub == 0) {
        float v[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
          v[i] = joined[0][i * 64 + th];
#pragma unroll
          for (int s = 1; s < kRows; ++s) v[i] += joined[s][i * 64 + th];
        }
        store<MODE, float>(dst + c, left, v);
      }
    } else {
      store<MODE, float>(dst + c, left, own);
    }
  };

  // a row's tensors and statistics, loaded while the row before is worked on (not with 128 registers a thread)
  constexpr bool kAhead = TPR < 1024;
  struct Ahead {
    Raw<MODE, T> x, u;
    Raw<MODE, R> n, d;
    float stats[4];
  };
  auto fetch = [&](Ahead &h, long row) {
    const long at = row * cols + c;
    h.x.load((const T *)A.x + at, left);
    h.n.load((const R *)A.residual + at, pre && A.residual ? left : 0);
    h.u.load((const T *)A.d_normed + at, pre ? left : 0);
    h.d.load((const R *)A.d_stream + at, A.d_stream ? left : 0);
    h.stats[0] = post ? A.stats[row] : 0.f;
    h.stats[1] = post ? A.stats[A.rows + row] : 1.f;
    h.stats[2] = pre ? A.stats[2 * A.rows + row] : 0.f;
    h.stats[3] = pre ? A.stats[3 * A.rows + row] : 1.f;
  };
  for (long s0 = first; s0 < last;) {
    const long s1 = by_sample ? min(last, (s0 / segment + 1) * segment) : last;
    if (!by_element) load_param<MODE, T>(A.gate, A.gate_dtype == BUTD_NORM_F32, (by_sample ? s0 / segment : 0) * cols + c, left, 1.f, g);
    Ahead ahead;
    if (kAhead && s0 + sub < s1) fetch(ahead, s0 + sub);
    for (long row = s0 + sub; row < s1; row += kRows) {  // (several rows: each is one wave's, nothing below waits for another wave)
      const long at = row * cols + c;
      float x[N], n[N], u[N], d[N];
      if (!kAhead) fetch(ahead, row);
      ahead.x.widen(x);
      ahead.n.widen(n);
      ahead.u.widen(u);
      ahead.d.widen(d);
      const float mean1 = ahead.stats[0], rstd1 = ahead.stats[1], mean2 = ahead.stats[2], rstd2 = ahead.stats[3];
      if (by_element) load_param<MODE, T>(A.gate, A.gate_dtype == BUTD_NORM_F32, at, left, 1.f, g);
      if (kAhead && row + kRows < s1) fetch(ahead, row + kRows);   // on its way while this row is worked on
      if (post) {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = (x[i] - mean1) * rstd1;
      }
      float s[2];
      if (pre) {
        // the stream again, normalised: n;  d += rstd2 (u - mean(u) - n mean(u n)),  u = d_normed * weight
        float v[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
          float t = g[i] * (x[i] * w1[i] + b1[i]);
          if (A.residual) t += A.residual_scale * n[i];
          n[i] = (t - mean2) * rstd2;
          v[i] = u[i] * n[i];
        }
        add(kPreW, v);
        add(kPreB, u);
        s[0] = s[1] = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) {
          u[i] *= w2[i];
          s[0] += i >= twice ? u[i] : 0.f;
          s[1] += i >= twice ? u[i] * n[i] : 0.f;
        }
        row_sum(s);
        const float m0 = A.pre_kind == BUTD_NORM_LAYER ? s[0] * inv_cols : 0.f, m1 = s[1] * inv_cols;
#pragma unroll
        for (int i = 0; i < N; ++i) d[i] += rstd2 * (u[i] - m0 - n[i] * m1);
      }
      if (A.d_residual) {
        float v[N];
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = A.residual_scale * d[i];
        store<MODE, R>((R *)A.d_residual + at, left, v);
      }
#pragma unroll
      for (int i = 0; i < N; ++i) {
        u[i] = d[i] * (x[i] * w1[i] + b1[i]);            // the gate's gradient
        sum_g[i] += u[i];
        d[i] *= g[i];
        n[i] = d[i] * x[i];
      }
      if (by_element && A.d_gate) {
        if (A.gate_dtype == BUTD_NORM_F32) store<MODE, float>((float *)A.d_gate + at, left, u);
        else store<MODE, T>((T *)A.d_gate + at, left, u);
      }
      if (post) {
        add(kPostW, n);
        add(kPostB, d);
        s[0] = s[1] = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) {
          s[0] += i >= twice ? d[i] * w1[i] : 0.f;
          s[1] += i >= twice ? n[i] * w1[i] : 0.f;
          d[i] *= w1[i];
        }
        row_sum(s);
        const float m0 = A.post_kind == BUTD_NORM_LAYER ? s[0] * inv_cols : 0.f, m1 = s[1] * inv_cols;
#pragma unroll
        for (int i = 0; i < N; ++i) d[i] = rstd1 * (d[i] - m0 - x[i] * m1);
      }
      if (A.d_x) store<MODE, T>((T *)A.d_x + at, left, d);
    }
    if (by_sample && P.gate_part) {
      flush(sum_g, P.gate_part + (P.run == segment ? (long)blockIdx.x : s0 / segment) * cols);
#pragma unroll
      for (int i = 0; i < N; ++i) sum_g[i] = 0.f;
    }
    s0 = s1;
  }
  if (A.gate_kind == BUTD_GATE_CHANNEL && P.gate_part) flush(sum_g, P.gate_part + (long)blockIdx.x * cols);
  if (P.part) {
    float *dst = P.part + (long)blockIdx.x * 4 * cols;
    float v[N];
    void *const wanted[4] = {A.d_post_weight, A.d_post_bias, A.d_pre_weight, A.d_pre_bias};
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (wanted[k]) {
        total(k, v);
        flush(v, dst + k * (long)cols);
      }
  }
}

// out[o][c] = sum over `count` partial rows, in a fixed order; 64 columns x 16 rows at a time (256 partial rows of 4 x 4096:
// 4.4 us)
struct Fold {
  const float *part;           // row k of output o at part + (o * count + k) * stride
  long stride;
  long count, outputs;
  void *out;                   // (outputs, cols)
  int f32;
  long first;                  // first workgroup
};
struct Folds {
  Fold f[5];
  int n, cols, col_blocks;
  long items;
};
template <typename T> __global__ __launch_bounds__(1024) void fold_kernel(const Folds L) {
  __shared__ float sums[16][64];
  for (long at = blockIdx.x; at < L.items; at += gridDim.x) {
    int fi = 0;
#pragma unroll
    for (int i = 1; i < 5; ++i)
      if (i < L.n && at >= L.f[i].first) fi = i;
    const Fold F = L.f[fi];
    const long item = at - F.first, o = item / L.col_blocks;
    const int c = (int)(item - o * L.col_blocks) * 64 + (threadIdx.x & 63), sub = threadIdx.x >> 6;
    float s = 0.f;
    if (c < L.cols) {
      const float *p = F.part + o * F.count * F.stride + c;
#pragma unroll 4
      for (long k = sub; k < F.count; k += 16) s += p[k * F.stride];
    }
    __syncthreads();                                       // (the sums of the item before have been read)
    sums[sub][threadIdx.x & 63] = s;
    __syncthreads();
    if (sub == 0 && c < L.cols) {
      for (int k = 1; k < 16; ++k) s += sums[k][threadIdx.x];
      if (F.f32) ((float *)F.out)[o * L.cols + c] = s;
      else ((T *)F.out)[o * L.cols + c] = (T)s;
    }
  }
}

// ---- host --------------------------------------------------------------------------------------------------------------------
size_t size_of(int dtype) { return dtype == BUTD_NORM_F32 ? 4 : 2; }

bool valid(const Args *a, bool backward) {
  if (!a || a->x_dtype < BUTD_NORM_F32 || a->x_dtype > BUTD_NORM_F16) return false;
  for (int d : {a->stream_dtype, a->post_dtype, a->pre_dtype, a->gate_dtype})
    if (d != a->x_dtype && d != BUTD_NORM_F32) return false;
  if (a->post_kind < 0 || a->post_kind > BUTD_NORM_LAYER || a->pre_kind < 0 || a->pre_kind > BUTD_NORM_LAYER) return false;
  if (a->gate_kind < 0 || a->gate_kind > BUTD_GATE_ELEMENT) return false;
  if (a->cols < 1 || a->cols > BUTD_NORM_MAX_COLS || a->rows < 0 || a->rows > 0x7fffffffL) return false;
  if (a->gate_kind == BUTD_GATE_SAMPLE && a->rows && (a->rows_per_sample < 1 || a->rows % a->rows_per_sample)) return false;
  const size_t x = size_of(a->x_dtype), r = size_of(a->stream_dtype), post = size_of(a->post_dtype), pre = size_of(a->pre_dtype),
               gate = size_of(a->gate_dtype);
  const struct { const void *p; size_t size; } typed[] = {
      {a->x, x}, {a->normed, x}, {a->d_x, x}, {a->d_normed, x}, {a->residual, r}, {a->stream, r}, {a->d_residual, r}, {a->d_stream, r},
      {a->gate, gate}, {a->d_gate, gate}, {a->post_weight, post}, {a->post_bias, post}, {a->d_post_weight, post}, {a->d_post_bias, post},
      {a->pre_weight, pre}, {a->pre_bias, pre}, {a->d_pre_weight, pre}, {a->d_pre_bias, pre}, {a->stats, 4}};
  for (const auto &t : typed)
    if ((uintptr_t)t.p % t.size) return false;
  if (a->rows == 0) return true;
  if (!a->x || (a->gate_kind && !a->gate)) return false;
  const bool plain = !a->residual && !a->gate_kind && !a->post_kind;      // the stream is x
  if (!backward) return (a->stream || plain) && (!a->pre_kind || a->normed);
  if ((a->post_kind || (a->pre_kind && a->d_normed)) && !a->stats) return false;
  return true;
}

constexpr long kMaxBlocks = 1L << 21;

// threads of a row: the smallest power of two of them that holds it, eight elements each
template <typename F> hipError_t by_width(int cols, F &&f) {
  if (cols <= 64 * N) return f.template operator()<64>();
  if (cols <= 128 * N) return f.template operator()<128>();
  if (cols <= 256 * N) return f.template operator()<256>();
  if (cols <= 512 * N) return f.template operator()<512>();
  return f.template operator()<1024>();
}

template <typename T, typename R> struct Forward {
  const Args &A;
  hipStream_t stream;
  template <int TPR> hipError_t operator()() {
    auto *kernel = A.cols % N == 0 ? &forward_kernel<T, R, TPR, kWhole> : &forward_kernel<T, R, TPR, kOverlap>;
    if constexpr (TPR == 64)
      if (A.cols < N) kernel = &forward_kernel<T, R, TPR, kElements>;
    // (a launch has to stay below 2^32 threads)
    hipError_t err = hipSuccess;
    for (long row0 = 0; row0 < A.rows && err == hipSuccess; row0 += kMaxBlocks * Group<TPR>::kRows) {
      const long blocks = (A.rows - row0 + Group<TPR>::kRows - 1) / Group<TPR>::kRows;
      hipLaunchKernelGGL(kernel, dim3((unsigned)(blocks < kMaxBlocks ? blocks : kMaxBlocks)), dim3(Group<TPR>::kThreads), 0, stream, A,
                         row0);
      err = hipGetLastError();
    }
    return err;
  }
};

// the rows' shares: about `target` workgroups, whole samples each where the gate is one of the sample's.  As many as run at
// once, two waves a SIMD of the 180 to 220 registers: each workgroup more costs five partial rows, written and read again
// (16384 rows of 4096 with both norms: 256 workgroups 237 + 4 us for the sums, 512 247 + 8, 768 251 + 12)
Plan plan_of(const Args &A, char *ws, long *bytes) {
  Plan P{};
  const bool wave_rows = A.cols <= 64 * N;
  const int threads = A.cols <= 64 * N ? 256 : A.cols <= 128 * N ? 128 : A.cols <= 256 * N ? 256 : 512;
  const long step = wave_rows ? 4 : 1, target = 256 * (512 / threads);
  long per = (A.rows + target - 1) / target;
  per = (per + step - 1) / step * step;
  const long least = wave_rows ? 8 : 2;
  if (per < least) per = least;
  P.run = A.rows;
  P.share = (A.rows + per - 1) / per;
  P.slots = P.share;
  if (A.gate_kind == BUTD_GATE_SAMPLE) {
    if (A.rows_per_sample >= per) {
      P.run = A.rows_per_sample;
      P.share = (P.run + per - 1) / per;
      per = (P.run + P.share - 1) / P.share;
      P.slots = (A.rows / P.run) * P.share;
    } else {
      per = per / A.rows_per_sample * A.rows_per_sample;
      P.share = (A.rows + per - 1) / per;
      P.slots = A.rows / A.rows_per_sample;
    }
  }
  P.per = per;
  P.blocks = (A.rows / P.run) * P.share;
  long used = 0;
  if (A.d_post_weight || A.d_post_bias || A.d_pre_weight || A.d_pre_bias) {
    P.part = (float *)(ws ? ws + used : nullptr);
    used += (P.blocks * 4 * A.cols * 4 + 255) / 256 * 256;
  }
  if (A.d_gate && (A.gate_kind == BUTD_GATE_CHANNEL || A.gate_kind == BUTD_GATE_SAMPLE)) {
    P.gate_part = (float *)(ws ? ws + used : nullptr);
    used += (P.slots * A.cols * 4 + 255) / 256 * 256;
  }
  *bytes = used;
  return P;
}

template <typename T, typename R> struct Backward {
  const Args &A;
  const Plan &P;
  hipStream_t stream;
  template <int TPR> hipError_t operator()() {
    auto *kernel = A.cols % N == 0 ? &backward_kernel<T, R, TPR, kWhole> : &backward_kernel<T, R, TPR, kOverlap>;
    if constexpr (TPR == 64)
      if (A.cols < N) kernel = &backward_kernel<T, R, TPR, kElements>;
    hipLaunchKernelGGL(kernel, dim3((unsigned)P.blocks), dim3(Group<TPR>::kThreads), 0, stream, A, P);
    hipError_t err = hipGetLastError();
    if (err != hipSuccess) return err;
    Folds L;
    L.n = 0;
    L.cols = A.cols;
    L.col_blocks = (A.cols + 63) / 64;
    long first = 0;
    auto add = [&](const float *part, long stride, long count, long outputs, void *out, int dtype) {
      L.f[L.n++] = Fold{part, stride, count, outputs, out, dtype == BUTD_NORM_F32, first};
      first += outputs * L.col_blocks;
    };
    const long stride = 4L * A.cols;
    if (A.d_post_weight) add(P.part + kPostW * (long)A.cols, stride, P.blocks, 1, A.d_post_weight, A.post_dtype);
    if (A.d_post_bias) add(P.part + kPostB * (long)A.cols, stride, P.blocks, 1, A.d_post_bias, A.post_dtype);
    if (A.d_pre_weight) add(P.part + kPreW * (long)A.cols, stride, P.blocks, 1, A.d_pre_weight, A.pre_dtype);
    if (A.d_pre_bias) add(P.part + kPreB * (long)A.cols, stride, P.blocks, 1, A.d_pre_bias, A.pre_dtype);
    if (P.gate_part) {
      const long outputs = A.gate_kind == BUTD_GATE_SAMPLE ? A.rows / A.rows_per_sample : 1;
      add(P.gate_part, A.cols, P.slots / outputs, outputs, A.d_gate, A.gate_dtype);
    }
    if (!L.n) return hipSuccess;
    L.items = first;
    const long most = 1L << 16;
    hipLaunchKernelGGL((fold_kernel<T>), dim3((unsigned)(first < most ? first : most)), dim3(1024), 0, stream, L);
    return hipGetLastError();
  }
};

template <typename T, typename R> hipError_t forward(const Args &A, hipStream_t stream) {
  return by_width(A.cols, Forward<T, R>{A, stream});
}
template <typename T, typename R> hipError_t backward(const Args &A, const Plan &P, hipStream_t stream) {
  return by_width(A.cols, Backward<T, R>{A, P, stream});
}

// gate of a one-row sample: an element's gate
Args simplified(const Args &a) {
  Args A = a;
  if (A.gate_kind == BUTD_GATE_SAMPLE && A.rows_per_sample == 1) A.gate_kind = BUTD_GATE_ELEMENT;
  // gradients of what is not there
  if (!A.post_kind || !A.post_weight) A.d_post_weight = nullptr;
  if (!A.post_kind || !A.post_bias) A.d_post_bias = nullptr;
  if (!A.pre_kind || !A.pre_weight) A.d_pre_weight = nullptr;
  if (!A.pre_kind || !A.pre_bias) A.d_pre_bias = nullptr;
  if (!A.gate_kind) A.gate = nullptr, A.d_gate = nullptr;
  return A;
}

}  // namespace

extern "C" {

long butd_residual_norm_args_size(void) { return (long)sizeof(butd_residual_norm_args); }

int butd_residual_norm_fwd(const butd_residual_norm_args *args, butd_stream_t stream) {
  if (!valid(args, false)) return (int)hipErrorInvalidValue;
  if (args->rows == 0) return 0;
  const Args A = simplified(*args);
  const hipStream_t s = (hipStream_t)stream;
  const bool wide = A.stream_dtype == BUTD_NORM_F32;
  switch (A.x_dtype) {
    case BUTD_NORM_F32: return (int)forward<float, float>(A, s);
    case BUTD_NORM_BF16: return (int)(wide ? forward<__bf16, float>(A, s) : forward<__bf16, __bf16>(A, s));
    default: return (int)(wide ? forward<_Float16, float>(A, s) : forward<_Float16, _Float16>(A, s));
  }
}

long butd_residual_norm_bwd_workspace(const butd_residual_norm_args *args) {
  if (!valid(args, true)) return -(long)hipErrorInvalidValue;
  if (args->rows == 0) return 0;
  long bytes = 0;
  plan_of(simplified(*args), nullptr, &bytes);
  return bytes;
}

int butd_residual_norm_bwd(const butd_residual_norm_args *args, void *workspace, long workspace_bytes, butd_stream_t stream) {
  if (!valid(args, true)) return (int)hipErrorInvalidValue;
  const Args A = simplified(*args);
  const hipStream_t s = (hipStream_t)stream;
  if (A.rows == 0) {                                     // sums over nothing
    const struct { void *p; int dtype; } sums[] = {{A.d_post_weight, A.post_dtype}, {A.d_post_bias, A.post_dtype},
                                                   {A.d_pre_weight, A.pre_dtype}, {A.d_pre_bias, A.pre_dtype},
                                                   {A.gate_kind == BUTD_GATE_CHANNEL ? A.d_gate : nullptr, A.gate_dtype}};
    for (const auto &o : sums) {
      const hipError_t err = o.p ? butd_zero_async(o.p, (size_t)A.cols * size_of(o.dtype), s) : hipSuccess;
      if (err != hipSuccess) return (int)err;
    }
    return 0;
  }
  long need = 0;
  const Plan P = plan_of(A, (char *)workspace, &need);
  if (need > 0 && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15))) return (int)hipErrorInvalidValue;
  const bool wide = A.stream_dtype == BUTD_NORM_F32;
  // a null d_normed: d_pre_* are sums over nothing
  if (!A.d_normed) {
    Args B = A;
    for (void **p : {&B.d_pre_weight, &B.d_pre_bias}) {
      const hipError_t err = *p ? butd_zero_async(*p, (size_t)A.cols * size_of(A.pre_dtype), s) : hipSuccess;
      if (err != hipSuccess) return (int)err;
      *p = nullptr;
    }
    switch (B.x_dtype) {
      case BUTD_NORM_F32: return (int)backward<float, float>(B, P, s);
      case BUTD_NORM_BF16: return (int)(wide ? backward<__bf16, float>(B, P, s) : backward<__bf16, __bf16>(B, P, s));
      default: return (int)(wide ? backward<_Float16, float>(B, P, s) : backward<_Float16, _Float16>(B, P, s));
    }
  }
  switch (A.x_dtype) {
    case BUTD_NORM_F32: return (int)backward<float, float>(A, P, s);
    case BUTD_NORM_BF16: return (int)(wide ? backward<__bf16, float>(A, P, s) : backward<__bf16, __bf16>(A, P, s));
    default: return (int)(wide ? backward<_Float16, float>(A, P, s) : backward<_Float16, _Float16>(A, P, s));
  }
}

}  // extern "C"
