// ffn_tile.h -- the matrix-product core of the gated feed-forward block (include/butd_gated_ffn.h), gfx950.
//
// One kernel template computes   C(m, n) = sum_k A(m, k) B(n, k)   for every product of the block; what differs is how an
// operand lies in memory (its contraction index contiguous, "K-contiguous", or its row index contiguous, "K-strided") and
// what happens to the accumulators:
//   kGateUp   A = x, B = W_gate | W_up side by side: h = act(a + b_gate) * (b + b_up) leaves the kernel, not a and b
//   kPlain    y = h W_down^T + b_down;  dx = da W_gate + db W_up (two contraction segments);  the three weight gradients
//   kGrad     dh = dy W_down: da = dh * b * act'(a) and db = dh * act(a) leave the kernel, not dh
//
// A tile of C is computed by 4 or 8 waves.  Global -> LDS goes by direct loads (16 bytes a lane, no registers), two LDS
// stages, the next stage in flight while the matrix cores work on the present one.  A 1 KB direct load writes LDS linearly,
// so bank swizzles are made on the SOURCE side: each lane picks which 16 bytes of the row it fetches.
//   K-contiguous tile: rows of 128 bytes; 16-byte unit u of row r stands at u ^ key(r): eight rows read at one unit touch
//     eight different unit columns.
//   K-strided tile, 16-bit: row k holds all m (or n) of the tile; the transposing LDS read hands each lane four k of its
//     column; 32-byte granules are XORed with a key of k so that the four rows of a 16-lane block do not share banks.
//   K-strided tile, 32-bit: one 16-byte read serves four MFMA tiles whose columns are interleaved (n = 4 i + t).
// Out-of-range rows read as zero through the buffer descriptor's bound; a contraction tail inside a row is masked per lane.
//
// The accumulators are computed transposed (B as the first MFMA operand): a lane then holds consecutive columns of one row
// of C and stores vectors.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#ifndef BUTD_MAIN_PRIO
#define BUTD_MAIN_PRIO 0
#endif

namespace ffn {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

enum Kind { kGateUp = 0, kPlain = 1, kGrad = 2 };
enum Act { kSilu = 0, kGelu = 1, kGeluTanh = 2, kRelu = 3, kSigmoid = 4 };

// ---- types ------------------------------------------------------------------------------------------------------------
template <typename T> struct Num {                       // 16-bit types
  static constexpr int kVec = 8;                         // elements of 16 bytes
  static constexpr int kBK = 64;                         // contraction depth of a stage: 128 bytes
};
template <> struct Num<float> {
  static constexpr int kVec = 4;
  static constexpr int kBK = 32;
};

__device__ inline f32x4 mma(u32x4 b, u32x4 a, f32x4 c, const __bf16 *) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, b), __builtin_bit_cast(bf16x8, a), c, 0, 0, 0);
}
__device__ inline f32x4 mma(u32x4 b, u32x4 a, f32x4 c, const _Float16 *) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, b), __builtin_bit_cast(f16x8, a), c, 0, 0, 0);
}
// 32-bit: element j of the two 16-byte fragments is one 16x16x4 step.  Lane group g holds k = 4 g + j of either operand, so
// step j sums k = j, 4 + j, 8 + j, 12 + j: together the sixteen k of the fragment, each once.
__device__ inline f32x4 mma(u32x4 b, u32x4 a, f32x4 c, const float *) {
  const f32x4 fb = __builtin_bit_cast(f32x4, b), fa = __builtin_bit_cast(f32x4, a);
#pragma unroll
  for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(fb[j], fa[j], c, 0, 0, 0);
  return c;
}

// ---- activation -------------------------------------------------------------------------------------------------------
// 1 / (1 + e^-a) from the hardware exponential and reciprocal (about one unit in the last place of 32 bits each)
__device__ inline float logistic(float a) { return __builtin_amdgcn_rcpf(1.f + __expf(-a)); }

// value and slope of the activation.  gelu_tanh: 0.5 a (1 + tanh u) = a * logistic(2 u), which does not cancel for u << 0.
template <int KIND> __device__ inline void activation(float a, float &v, float &d) {
  if constexpr (KIND == kSilu) {
    const float s = logistic(a);
    v = a * s;
    d = s * (1.f + a * (1.f - s));
  } else if constexpr (KIND == kGelu) {
    const float cdf = 0.5f * (1.f + erff(a * 0.70710678118654752f));
    v = a * cdf;
    d = cdf + a * (0.39894228040143268f * __expf(-0.5f * a * a));
  } else if constexpr (KIND == kGeluTanh) {
    const float k = 0.79788456080286536f, c = 0.044715f;
    const float s = logistic(2.f * k * (a + c * a * a * a));
    v = a * s;
    d = s + a * s * (1.f - s) * (2.f * k * (1.f + 3.f * c * a * a));
  } else if constexpr (KIND == kRelu) {
    v = a < 0.f ? 0.f : a;                               // (not fmaxf: a NaN stays one)
    d = a > 0.f ? 1.f : 0.f;
  } else {
    const float s = logistic(a);
    v = s;
    d = s * (1.f - s);
  }
}
template <int KIND> __device__ inline void activation4_of(const float *a, float *v, float *d) {
#pragma unroll
  for (int e = 0; e < 4; ++e) activation<KIND>(a[e], v[e], d[e]);
}
// four elements behind one uniform branch
__device__ inline void activation4(int kind, const float *a, float *v, float *d) {
  switch (kind) {
    case kSilu: activation4_of<kSilu>(a, v, d); break;
    case kGelu: activation4_of<kGelu>(a, v, d); break;
    case kGeluTanh: activation4_of<kGeluTanh>(a, v, d); break;
    case kRelu: activation4_of<kRelu>(a, v, d); break;
    default: activation4_of<kSigmoid>(a, v, d);
  }
}

// ---- a launch ---------------------------------------------------------------------------------------------------------
struct Problem {
  // operands of up to two contraction segments (same shapes and strides); ld in BYTES
  const void *a[2], *b[2];
  long lda, ldb;
  int M, N, K;                 // K: of one segment
  int segments;
  // kGateUp: b[0] / b[1] are W_gate / W_up of the ONE segment; c = h, aux0 / aux1 = a, b (32-bit) or null
  // kGrad:   c = da, c2 = db, aux0 / aux1 = a, b
  // kPlain:  c, or the 32-bit slab of slice s at slab + s * slab_stride (elements) when split > 1
  void *c, *c2;
  long ldc;                    // elements
  int pad;                     // columns N .. pad - 1 of c / c2 are written as zeros (the rows' padding)
  const float *aux0, *aux1;
  float *out0, *out1;
  long ldaux;                  // elements
  const void *bias0, *bias1;
  float *slab;
  long slab_stride;
  int split;
  int tiles_m, tiles_n, first; // first block of this problem
};
constexpr int kMaxProblems = 3;
struct Launch {
  Problem p[kMaxProblems];
  int count, act, total;
};

// blockIdx -> work item: the chip deals consecutive workgroups to its 8 dies in turn; the dies' L2 caches are separate, so
// each die is given a consecutive run of tiles instead
__device__ inline int die_local(int b, int n) {
  const int die = b & 7, q = n >> 3, r = n & 7;
  return die * q + (die < r ? die : r) + (b >> 3);
}

__device__ inline int key_natural(int row) { return row & 7; }
__device__ inline int key_pair(int row) { return (row & 3) | ((row >> 1) & 4); }

template <typename T, int KIND, bool AK, bool BK_, int TM_, int TN_, int WM_, int WN_>
struct Config {
  using type = T;
  static constexpr int kind = KIND, TM = TM_, TN = TN_, WM = WM_, WN = WN_, NW = WM_ * WN_;
  static constexpr bool a_kc = AK, b_kc = BK_;
  static constexpr int FM = TM / WM / 16, FN = TN / WN / 16;
  static constexpr int kA = TM * 128, kB = TN * 128;     // bytes of a stage
  static constexpr int kThreads = NW * 64;
};

// direct load of one operand's stage.  EXT: rows of the tile (m or n extent); KC: K-contiguous; PAIR: swizzle key
template <typename T, int EXT, int NW, bool KC, bool PAIR>
struct Loader {
  static constexpr int kChunks = EXT * 128 / 1024 / NW;  // 1 KB direct loads of a wave
  static_assert(kChunks >= 1, "tile too small for the workgroup");
  static constexpr int kRowBytes = EXT * (int)sizeof(T);
  uint32_t voff[kChunks];
  int kunit;                                             // K-contiguous: first k of the lane's unit
  __device__ inline void init(int wave, int lane, long ld) {
#pragma unroll
    for (int j = 0; j < kChunks; ++j) {
      const int c = j * NW + wave;
      if constexpr (KC) {
        const int row = 8 * c + (lane >> 3);
        const int unit = (lane & 7) ^ (PAIR ? key_pair(row) : key_natural(row));
        voff[j] = (uint32_t)(row * ld) + unit * 16;
      } else {
        constexpr int kUnits = kRowBytes / 16;
        const int k = c * (64 / kUnits) + lane / kUnits;
        int unit = lane % kUnits;
        if constexpr (sizeof(T) == 2) unit = ((((unit >> 1) ^ (key_pair(k) & (kUnits / 2 - 1)))) << 1) | (unit & 1);
        voff[j] = (uint32_t)(k * ld) + unit * 16;
      }
    }
    if constexpr (KC) {      // (NW * 8 rows between a wave's chunks, a multiple of 16: the unit is the same in all of them)
      static_assert(NW % 2 == 0, "the swizzle key must not change between a wave's chunks");
      const int row = 8 * wave + (lane >> 3);
      kunit = ((lane & 7) ^ (PAIR ? key_pair(row) : key_natural(row))) * Num<T>::kVec;
    }
  }
  // base: address of (first row, k0) resp. (k0, first row); bytes: what is readable from there; klimit = K - k0
  __device__ inline void issue(char *lds, int wave, const char *base, long bytes, int klimit, int j0 = 0, int j1 = kChunks) const {
    const uint32_t records = bytes > 0x7fffffffL ? 0x7fffffffu : (bytes < 0 ? 0u : (uint32_t)bytes);
    __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc((void *)base, 0, records, 0x00020000);
    const bool live = !KC || kunit < klimit;             // a masked unit points past the bound and arrives as zeros
#pragma unroll
    for (int j = 0; j < kChunks; ++j) {
      if (j < j0 || j >= j1) continue;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          rsrc, (__attribute__((address_space(3))) void *)(lds + (j * NW + wave) * 1024), 16,
          live ? voff[j] : 0x80000000u, 0, 0, 0);
    }
  }
};

// fragment reads of one operand: tile t (16 rows of C's m or n), step s (half of the stage)
template <typename T, int EXT, int F, bool KC, bool PAIR>
struct Reader {
  static constexpr int kRowBytes = EXT * (int)sizeof(T);
  static constexpr int kGroup = (!KC && sizeof(T) == 4) ? (F >= 4 ? 4 : F) : 1;
  static_assert(F % kGroup == 0, "");
  int base;
  int key;
  __device__ inline void init(int lane, int first) {     // first: first row of the wave's part of the tile
    const int i = lane & 15, g = lane >> 4;
    if constexpr (KC) {
      const int row = PAIR ? 8 * (i >> 2) + (i & 3) : i;
      key = (PAIR ? key_pair(row) : key_natural(row));
      base = (first + row) * 128 + ((g ^ key) << 4);     // step 1 flips bit 2 of the unit: address ^ 64
    } else if constexpr (sizeof(T) == 2) {
      const int k = 8 * g + (i >> 2);
      key = key_pair(k) & (kRowBytes / 32 - 1);
      base = k * kRowBytes + (i & 3) * 8;
    } else {
      base = 4 * g * kRowBytes + (first + kGroup * i) * 4;
      key = 0;
    }
  }
  __device__ inline void read(const char *lds, int first, int s, u32x4 *frag) const {
    if constexpr (KC) {
#pragma unroll
      for (int t = 0; t < F; ++t) {
        // PAIR: tiles 2 G, 2 G + 1 cover the rows 32 G + 8 (i / 4) + 4 (t % 2) + i % 4
        const int off = PAIR ? (t >> 1) * (32 * 128) + (t & 1) * (4 * 128) : t * (16 * 128);
        frag[t] = *(const u32x4 *)(lds + (base ^ (s << 6)) + off);
      }
    } else if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int t = 0; t < F; ++t) {
        const int addr = base + ((((first >> 4) + t) ^ key) << 5);
        u32x4 f;
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const s16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (__attribute__((address_space(3))) s16x4 *)(lds + addr + (32 * s + 4 * q) * kRowBytes));
          const uint2 w = __builtin_bit_cast(uint2, v);
          f[2 * q] = w.x;
          f[2 * q + 1] = w.y;
        }
        frag[t] = f;
      }
    } else {
#pragma unroll
      for (int G = 0; G < F / kGroup; ++G) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const char *p = lds + base + (16 * s + j) * kRowBytes + G * (16 * kGroup * 4);
          if constexpr (kGroup == 4) {
            const u32x4 v = *(const u32x4 *)p;
#pragma unroll
            for (int t = 0; t < 4; ++t) frag[4 * G + t][j] = v[t];
          } else if constexpr (kGroup == 2) {
            const uint2 v = *(const uint2 *)p;
            frag[2 * G][j] = v.x;
            frag[2 * G + 1][j] = v.y;
          } else {
            frag[G][j] = *(const uint32_t *)p;
          }
        }
      }
    }
  }
};

// ---- stores -----------------------------------------------------------------------------------------------------------
template <typename T> __device__ inline void store_quad(T *p, const float *v);
template <> __device__ inline void store_quad<float>(float *p, const float *v) { *(f32x4 *)p = f32x4{v[0], v[1], v[2], v[3]}; }
template <> __device__ inline void store_quad<__bf16>(__bf16 *p, const float *v) {
  typedef __bf16 v4 __attribute__((ext_vector_type(4)));
  *(v4 *)p = v4{(__bf16)v[0], (__bf16)v[1], (__bf16)v[2], (__bf16)v[3]};
}
template <> __device__ inline void store_quad<_Float16>(_Float16 *p, const float *v) {
  typedef _Float16 v4 __attribute__((ext_vector_type(4)));
  *(v4 *)p = v4{(_Float16)v[0], (_Float16)v[1], (_Float16)v[2], (_Float16)v[3]};
}

// four consecutive columns n .. n + 3 of a row; `whole`: rows of this matrix start at vector boundaries
template <typename T> __device__ inline void put(T *row, int n, int N, int pad, bool whole, const float *v) {
  if (whole && n + 4 <= N) {
    store_quad<T>(row + n, v);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (n + e < N) row[n + e] = (T)v[e];
      else if (n + e < pad) row[n + e] = (T)0.f;
  }
}

// ---- the kernel -------------------------------------------------------------------------------------------------------
template <class C> __global__ __launch_bounds__(C::kThreads) void tile_kernel(const Launch L) {
  using T = typename C::type;
  constexpr int BK = Num<T>::kBK;
  constexpr bool kPairB = C::b_kc && sizeof(T) == 2;     // (needs an even number of tiles of each B part in a wave)
  constexpr int FM = C::FM, FN = C::FN;
  constexpr int kParts = C::kind == kGateUp ? 2 : 1;
  constexpr int FP = FN / kParts;                        // tiles of one part in a wave
  static_assert(!kPairB || FP % 2 == 0, "");
  // two stages as separate objects: the compiler then knows that a read of one does not depend on loads into the other
  __shared__ __attribute__((aligned(1024))) char a_lds0[C::kA], b_lds0[C::kB], a_lds1[C::kA], b_lds1[C::kB];
  __builtin_amdgcn_s_setprio(BUTD_MAIN_PRIO);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

  // ---- which tile
  const int item = die_local(blockIdx.x, L.total);
  int pi = 0;
#pragma unroll
  for (int i = 1; i < kMaxProblems; ++i)
    if (i < L.count && item >= L.p[i].first) pi = i;
  const Problem P = L.p[pi];                             // (a copy: scalar registers, not reloads behind every barrier)
  const int local = item - P.first, tiles = P.tiles_m * P.tiles_n;
  const int slice = local / tiles, idx = local - slice * tiles;
  constexpr int kGroupM = 8;                             // 8 x n blocks of tiles: neighbours share both operands in L2
  const int width = kGroupM * P.tiles_n, grp = idx / width, first_m = grp * kGroupM;
  const int gsz = min(P.tiles_m - first_m, kGroupM), in = idx - grp * width;
  const int m0 = (first_m + in % gsz) * C::TM, n0 = (in / gsz) * (C::TN / kParts);

  const int per_seg = (P.K + BK - 1) / BK, steps = per_seg * P.segments;
  const int per_slice = (steps + P.split - 1) / P.split;
  const int it0 = slice * per_slice, it1 = min(steps, it0 + per_slice);

  const int wm = wave / C::WN, wn = wave % C::WN;
  const int a_first = wm * (FM * 16), b_first = wn * (FP * 16);

  Loader<T, C::TM, C::NW, C::a_kc, false> la;
  Loader<T, C::TN, C::NW, C::b_kc, kPairB> lb;
  la.init(wave, lane, P.lda);
  if constexpr (kParts == 2) {
    // rows TN/2 .. TN - 1 of the tile are W_up's rows 0 .. TN/2 - 1
    lb.init(wave, lane, P.ldb);
#pragma unroll
    for (int j = lb.kChunks / 2; j < lb.kChunks; ++j) lb.voff[j] -= (uint32_t)(C::TN / 2 * P.ldb);
  } else {
    lb.init(wave, lane, P.ldb);
  }
  Reader<T, C::TM, FM, C::a_kc, false> ra;
  Reader<T, C::TN, FP, C::b_kc, kPairB> rb;
  ra.init(lane, a_first);
  rb.init(lane, b_first);

  // next stage to be loaded: its addresses, what is left of the contraction segment
  int fetched = it0, left;
  const char *pa, *pb, *pb2 = nullptr;
  long a_bytes, b_bytes;                                 // readable from there on
  constexpr long kStepA = C::a_kc ? 128 : 0, kStepB = C::b_kc ? 128 : 0;
  const long step_a = C::a_kc ? kStepA : BK * P.lda, step_b = C::b_kc ? kStepB : BK * P.ldb;
  // a row's last 16-byte unit counts whole: rows that direct loads take end in one, or in padding (zeros where K ends in it)
  constexpr int kVec = Num<T>::kVec;
  const long unit_m = (P.M - m0 + kVec - 1) / kVec * 16L, unit_n = (P.N - n0 + kVec - 1) / kVec * 16L;
  auto seek = [&](int seg, int k0) {
    left = P.K - k0;
    const long unit_k = (left + kVec - 1) / kVec * 16L;
    if constexpr (C::a_kc) {
      pa = (const char *)P.a[seg] + (long)m0 * P.lda + (long)k0 * (int)sizeof(T);
      a_bytes = (long)(P.M - m0 - 1) * P.lda + unit_k;
    } else {
      pa = (const char *)P.a[seg] + (long)k0 * P.lda + (long)m0 * (int)sizeof(T);
      a_bytes = (long)(left - 1) * P.lda + unit_m;
    }
    if constexpr (C::b_kc) {
      const long off = (long)n0 * P.ldb + (long)k0 * (int)sizeof(T);
      pb = (const char *)P.b[seg] + off;
      if constexpr (kParts == 2) pb2 = (const char *)P.b[1] + off;
      b_bytes = (long)(P.N - n0 - 1) * P.ldb + unit_k;
    } else {
      pb = (const char *)P.b[seg] + (long)k0 * P.ldb + (long)n0 * (int)sizeof(T);
      b_bytes = (long)(left - 1) * P.ldb + unit_n;
    }
  };
  seek(it0 >= per_seg ? 1 : 0, (it0 >= per_seg ? it0 - per_seg : it0) * BK);
  auto issue = [&](char *al, char *bl) {
    la.issue(al, wave, pa, a_bytes, left);
    if constexpr (kParts == 2) {
      lb.issue(bl, wave, pb, b_bytes, left, 0, lb.kChunks / 2);
      lb.issue(bl, wave, pb2, b_bytes, left, lb.kChunks / 2, lb.kChunks);
      pb2 += step_b;
    } else {
      lb.issue(bl, wave, pb, b_bytes, left);
    }
    pa += step_a; pb += step_b; a_bytes -= step_a; b_bytes -= step_b; left -= BK;
    if (++fetched == per_seg) seek(1, 0);
  };

  f32x4 acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  // Two sets of fragments: while the matrix cores work on one half of a stage, the other half is read.  The barrier of a
  // stage stands BETWEEN its halves: the second half's operands are in registers by then, so the loads that overwrite the
  // stage go out, and the next stage is read, under the second half's matrix instructions.
  u32x4 fa[2][FM], fb[2][FN];
  auto read = [&](const char *al, const char *bl, int s) {
#pragma unroll
    for (int q = 0; q < kParts; ++q) rb.read(bl + q * (C::TN / 2 * 128), b_first, s, fb[s] + q * FP);
    ra.read(al, a_first, s, fa[s]);
  };
  auto multiply = [&](int s) {
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j) acc[i][j] = mma(fb[s][j], fa[s][i], acc[i][j], (const T *)nullptr);
  };
  // what the barrier orders: the next stage's direct loads of ALL waves have landed (each waits for its own first), and all
  // waves hold the present stage's operands in registers
  auto fence = [&]() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(0x0070);                  // vmcnt(0) lgkmcnt(0)
    asm volatile("s_barrier" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };
  if (it0 < it1) {
    issue(a_lds0, b_lds0);
    fence();
    if (it0 + 1 < it1) issue(a_lds1, b_lds1);
    read(a_lds0, b_lds0, 0);
  }
  // (one exit: a break behind the first half made the compiler keep a second copy of the accumulators)
  for (int it = it0; it < it1; it += 2) {
    read(a_lds0, b_lds0, 1);
    multiply(0);
    fence();
    if (it + 2 < it1) issue(a_lds0, b_lds0);
    if (it + 1 < it1) read(a_lds1, b_lds1, 0);
    multiply(1);
    if (it + 1 < it1) {
      read(a_lds1, b_lds1, 1);
      multiply(0);
      fence();
      if (it + 3 < it1) issue(a_lds1, b_lds1);
      if (it + 2 < it1) read(a_lds0, b_lds0, 0);
      multiply(1);
    }
  }

  // ---- epilogue.  The accumulators pass through LDS, a wave's own part of it, up to 64 of its rows at a time: behind that a
  // lane has four consecutive columns, 16 (or 8) lanes a row, so that global accesses are whole lines and the element-wise
  // work is a short loop (unrolled over the accumulators it needs more registers than there are).
  constexpr int WA = decltype(ra)::kGroup, WB = decltype(rb)::kGroup;
  constexpr int CT = FM < 4 ? FM : 4, kCols = FN * 16, kQuads = kCols / 4;      // m tiles of a chunk; columns of the wave
  constexpr int kChunkBytes = CT * 16 * kCols * 4;
  static_assert(C::kA == C::kB && C::kA % kChunkBytes == 0 && kChunkBytes * C::NW <= 4 * C::kA, "");
  static_assert(FM % CT == 0 && CT % WA == 0 && (kQuads & (kQuads - 1)) == 0, "");
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");               // the last stage has been read by every wave
  const int slot = wave * kChunkBytes / C::kA;
  char *mine = (slot == 0 ? a_lds0 : slot == 1 ? b_lds0 : slot == 2 ? a_lds1 : b_lds1) + wave * kChunkBytes % C::kA;
  const int i16 = lane & 15, g = lane >> 4;
  const bool whole = (P.ldc % 4 == 0) && ((uintptr_t)P.c & 15) == 0 && ((uintptr_t)P.c2 & 15) == 0;
  const bool to_slab = C::kind == kPlain && P.split > 1;
#pragma unroll
  for (int chunk = 0; chunk < FM / CT; ++chunk) {
#pragma unroll
    for (int tt = 0; tt < CT; ++tt) {
      const int row = 16 * WA * (tt / WA) + WA * i16 + tt % WA;
#pragma unroll
      for (int q = 0; q < FN; ++q) {
        const int part = q / FP, qq = q % FP;
        // quad q of the lane: four consecutive columns of the wave's part
        int col;
        if constexpr (kPairB) col = 32 * (qq >> 1) + 8 * g + 4 * (qq & 1);
        else col = 16 * WB * (qq / WB) + 4 * WB * g + 4 * (qq % WB);
        f32x4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int c = 4 * (qq % WB) + e;               // column c = WB * r + tile of the group (WB == 1: the tile's own rows r)
          v[e] = acc[chunk * CT + tt][part * FP + (qq / WB) * WB + c % WB][c / WB];
        }
        const int quad = part * (FP * 4) + (col >> 2);
        *(f32x4 *)(mine + row * (kCols * 4) + ((quad ^ (row & (kQuads - 1))) << 4)) = v;
      }
    }
    // (a wave's own LDS traffic is in order: the reads below see the writes above without a barrier)
    asm volatile("" ::: "memory");
    constexpr int kLanes = kQuads / kParts, kRows = 64 / kLanes;                  // lanes of a row, rows of a step
    const int quad = lane % kLanes;
    const int n = n0 + b_first + 4 * quad;
#pragma unroll 2
    for (int r = lane / kLanes; r < CT * 16; r += kRows) {
      float v[kParts][4];
#pragma unroll
      for (int part = 0; part < kParts; ++part) {
        const f32x4 w = *(const f32x4 *)(mine + r * (kCols * 4) + (((part * kLanes + quad) ^ (r & (kQuads - 1))) << 4));
#pragma unroll
        for (int e = 0; e < 4; ++e) v[part][e] = w[e];
      }
      const int m = m0 + a_first + chunk * (CT * 16) + r;
      if (m >= P.M) continue;
      if (to_slab) {
        put<float>(P.slab + (long)slice * P.slab_stride + (long)m * P.N, n, P.N, 0, (P.N & 3) == 0, v[0]);
        continue;
      }
      T *row = (T *)P.c + (long)m * P.ldc;
      if constexpr (C::kind == kGateUp) {
        float h[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (P.bias0 && n + e < P.N) v[0][e] += (float)((const T *)P.bias0)[n + e];
          if (P.bias1 && n + e < P.N) v[1][e] += (float)((const T *)P.bias1)[n + e];
        }
        float slope[4];
        activation4(L.act, v[0], h, slope);
#pragma unroll
        for (int e = 0; e < 4; ++e) h[e] *= v[1][e];
        put<T>(row, n, P.N, P.pad, whole, h);
        if (P.out0) {
          // kept in 32 bits: rounded to the operands' 16 bits here, the gradients of x and W_gate would carry two
          // roundings more than the product's own operands do
          put<float>(P.out0 + (long)m * P.ldaux, n, P.N, 0, true, v[0]);
          put<float>(P.out1 + (long)m * P.ldaux, n, P.N, 0, true, v[1]);
        }
      } else if constexpr (C::kind == kGrad) {
        f32x4 a4 = {0.f, 0.f, 0.f, 0.f}, b4 = a4;
        if (n + 4 <= P.N) {
          a4 = *(const f32x4 *)(P.aux0 + (long)m * P.ldaux + n);
          b4 = *(const f32x4 *)(P.aux1 + (long)m * P.ldaux + n);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (n + e < P.N) {
              a4[e] = P.aux0[(long)m * P.ldaux + n + e];
              b4[e] = P.aux1[(long)m * P.ldaux + n + e];
            }
        }
        float a[4] = {a4[0], a4[1], a4[2], a4[3]}, value[4], slope[4], da[4], db[4];
        activation4(L.act, a, value, slope);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          da[e] = v[0][e] * b4[e] * slope[e];
          db[e] = v[0][e] * value[e];
        }
        put<T>(row, n, P.N, P.pad, whole, da);
        put<T>((T *)P.c2 + (long)m * P.ldc, n, P.N, P.pad, whole, db);
      } else {
        if (P.bias0) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (n + e < P.N) v[0][e] += (float)((const T *)P.bias0)[n + e];
        }
        put<T>(row, n, P.N, P.pad, whole, v[0]);
      }
    }
    asm volatile("" ::: "memory");
  }
}

}  // namespace ffn
