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
// Bound by the matrix cores and the LDS at large sizes (8192 x 4096 -> 11264 bf16, a pass: x W_gate | W_up 1252 us and 1208
// TFLOP/s, h W_down^T 593 and 1275, dh 800 and 945 -- its epilogue reads a and b -- dx 1168 and 1294, the weight gradients 1915
// and 1184; library products of this card 1490), by latency at small ones (8192 x 288 -> 256: 7 to 15 us a launch).
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
template <int KIND, int N> __device__ inline void activations_of(const float *a, float *v, float *d) {
#pragma unroll
  for (int e = 0; e < N; ++e) activation<KIND>(a[e], v[e], d[e]);
}
// N elements behind one uniform branch
template <int N> __device__ inline void activations(int kind, const float *a, float *v, float *d) {
  switch (kind) {
    case kSilu: activations_of<kSilu, N>(a, v, d); break;
    case kGelu: activations_of<kGelu, N>(a, v, d); break;
    case kGeluTanh: activations_of<kGeluTanh, N>(a, v, d); break;
    case kRelu: activations_of<kRelu, N>(a, v, d); break;
    default: activations_of<kSigmoid, N>(a, v, d);
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
  // kGrad:   c = da, c2 = db, aux0 / aux1 = a, b; out0 / out1 = column sums of da and db over each wave's rows,
  //          (tiles_m * kWavesM, N), or null
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
  // filled in by the launch: tiles, the first block's x of this problem, steps of the contraction in all and of a slice,
  // and 2^32 / (8 tiles_n) + 1
  int tiles_m, tiles_n, first, steps, per_slice;
  uint32_t group_magic;
};
// rows of a slab are whole vectors
__host__ __device__ inline int slab_ld(int n) { return (n + 3) & ~3; }
constexpr int kWavesM = 2;                               // waves along m of every kGrad and kPlain tile
constexpr int kMaxProblems = 3;
struct Launch {
  Problem p[kMaxProblems];
  int count, act, total;       // total: blocks in x; the slices are blocks in y
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
  static constexpr bool kMulti = KIND == kPlain && !AK;           // the weight gradients: several problems in a launch
  static constexpr bool kSegments = KIND == kPlain && AK && !BK_; // dx: two contraction segments
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
  // base: address of (first row, k0) resp. (k0, first row); records: bytes that are readable from there; klimit = K - k0
  __device__ inline void issue(char *lds, int wave, const char *base, uint32_t records, int klimit, int j0 = 0, int j1 = kChunks) const {
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
  static constexpr int kReads = KC ? F : sizeof(T) == 2 ? 2 * F : 4 * F / kGroup;      // LDS instructions of one read()
  static_assert(F % kGroup == 0, "");
  int base;
  __device__ inline void init(int lane, int first) {     // first: first row of the wave's part of the tile
    const int i = lane & 15, g = lane >> 4;
    if constexpr (KC) {
      const int row = PAIR ? 8 * (i >> 2) + (i & 3) : i;
      base = (first + row) * 128 + ((g ^ (PAIR ? key_pair(row) : key_natural(row))) << 4);     // step 1 flips bit 2 of the unit: address ^ 64
    } else if constexpr (sizeof(T) == 2) {
      // granule of tile t: ((first >> 4) + t) ^ key, = ((first >> 4) ^ key) ^ t since t stays below the alignment of first
      const int k = 8 * g + (i >> 2);
      base = k * kRowBytes + (i & 3) * 8 + (((first >> 4) ^ (key_pair(k) & (kRowBytes / 32 - 1))) << 5);
    } else {
      base = 4 * g * kRowBytes + (first + kGroup * i) * 4;
    }
  }
  __device__ inline void read(const char *lds, int s, u32x4 *frag) const {
    if constexpr (KC) {
      int b = base ^ (s << 6);
#pragma unroll
      for (int t = 0; t < F; ++t) {
        // PAIR: tiles 2 G, 2 G + 1 cover the rows 32 G + 8 (i / 4) + 4 (t % 2) + i % 4
        const int off = PAIR ? (t >> 1) * (32 * 128) + (t & 1) * (4 * 128) : t * (16 * 128);
        frag[t] = *(const u32x4 *)(lds + b + off);
      }
    } else if constexpr (sizeof(T) == 2) {
      int b = base;
      asm volatile("" : "+v"(b));                        // (one XOR a tile here, not a register a tile across the loop)
#pragma unroll
      for (int t = 0; t < F; ++t) {
        const int addr = b ^ (t << 5);
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

// ... through a buffer descriptor: dropped where the offset is out of its bound
template <typename T> __device__ inline void store_buffer(__amdgpu_buffer_rsrc_t r, uint32_t off, const float *v) {
  if constexpr (sizeof(T) == 4) {
    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, f32x4{v[0], v[1], v[2], v[3]}), r, off, 0, 0);
  } else {
    typedef T v4 __attribute__((ext_vector_type(4)));
    typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
    __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, v4{(T)v[0], (T)v[1], (T)v[2], (T)v[3]}), r, off, 0, 0);
  }
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

  // ---- which tile.  (Divisions by run-time numbers cost hundreds of cycles each before the first load: the host's share of
  // them comes with the arguments.)
  const int item = die_local(blockIdx.x, L.total), slice = blockIdx.y;
  int pi = 0;
  if constexpr (C::kMulti) {
#pragma unroll
    for (int i = 1; i < kMaxProblems; ++i)
      if (i < L.count && item >= L.p[i].first) pi = i;
  }
  const Problem P = L.p[C::kMulti ? pi : 0];             // (a copy: scalar registers, not reloads behind every barrier)
  if (C::kMulti && slice >= P.split) return;
  const int idx = item - P.first;
  constexpr int kGroupM = 8;                             // 8 x n blocks of tiles: neighbours share both operands in L2
  const int width = kGroupM * P.tiles_n;
  int grp = (int)(((uint64_t)(uint32_t)idx * P.group_magic) >> 32);              // idx / width, or one more
  if (grp * width > idx) --grp;
  const int first_m = grp * kGroupM, gsz = min(P.tiles_m - first_m, kGroupM), in = idx - grp * width;
  int tn = in >> 3;                                      // in / gsz
  if (gsz != kGroupM) {
    tn = __builtin_amdgcn_readfirstlane((int)((float)in * __builtin_amdgcn_rcpf((float)gsz)));
    const int rest = in - tn * gsz;
    tn += rest < 0 ? -1 : rest >= gsz ? 1 : 0;
  }
  const int tm = first_m + in - tn * gsz, m0 = tm * C::TM, n0 = tn * (C::TN / kParts);

  const int per_seg = (P.K + BK - 1) / BK;
  const int it0 = slice * P.per_slice, it1 = min(P.steps, it0 + P.per_slice);

  const int wm = wave / C::WN, wn = wave % C::WN;
  const int a_first = wm * (FM * 16), b_first = wn * (FP * 16);

  Loader<T, C::TM, C::NW, C::a_kc, false> la;
  Loader<T, C::TN, C::NW, C::b_kc, kPairB> lb;
  la.init(wave, lane, P.lda);
  lb.init(wave, lane, P.ldb);
  if constexpr (kParts == 2) {
    // rows TN/2 .. TN - 1 of the tile are W_up's rows 0 .. TN/2 - 1
#pragma unroll
    for (int j = lb.kChunks / 2; j < lb.kChunks; ++j) lb.voff[j] -= (uint32_t)(C::TN / 2 * P.ldb);
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
  if constexpr (C::kSegments) seek(it0 >= per_seg ? 1 : 0, (it0 >= per_seg ? it0 - per_seg : it0) * BK);
  else seek(0, it0 * BK);
  // (no branch around it: behind the last step nothing is readable, the stage arrives as zeros and costs no memory traffic)
  uint32_t records_a, records_b;
  auto prepare = [&]() {                                 // masks and selects: no branch
    const uint32_t live = fetched < it1 ? 0xffffffffu : 0u;
    records_a = (uint32_t)min(max(a_bytes, 0L), 0x7fffffffL) & live;
    records_b = (uint32_t)min(max(b_bytes, 0L), 0x7fffffffL) & live;
  };
  auto issue = [&](char *al, char *bl) {
    la.issue(al, wave, pa, records_a, left);
    if constexpr (kParts == 2) {
      lb.issue(bl, wave, pb, records_b, left, 0, lb.kChunks / 2);
      lb.issue(bl, wave, pb2, records_b, left, lb.kChunks / 2, lb.kChunks);
      pb2 += step_b;
    } else {
      lb.issue(bl, wave, pb, records_b, left);
    }
    pa += step_a;
    pb += step_b;
    a_bytes -= step_a;
    b_bytes -= step_b;
    left -= BK;
    ++fetched;
    if constexpr (C::kSegments) {
      // the second segment has the first one's shape: back to its k = 0 on the other pointers
      const bool over = fetched == per_seg;
      const long back = (long)per_seg * BK;
      pa = over ? (const char *)P.a[1] + (long)m0 * P.lda : pa;
      pb = over ? (const char *)P.b[1] + (long)n0 * (int)sizeof(T) : pb;
      a_bytes += over ? back * (int)sizeof(T) : 0;
      b_bytes += over ? back * P.ldb : 0;
      left += over ? (int)back : 0;
    }
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
    for (int q = 0; q < kParts; ++q) rb.read(bl + q * (C::TN / 2 * 128), s, fb[s] + q * FP);
    ra.read(al, s, fa[s]);
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
  // The order of a half's instructions: a wave issues in order, and a run of LDS reads in front of the matrix instructions
  // holds those back while the LDS works the run off.  One direct load or read behind every matrix instruction hides both:
  // 3150 -> 2720 cycles a stage (4096^3, 256 tile; 2048 are the matrix instructions'), whichever side is K-strided.  Two
  // workgroups of the 128 tile share a CU and cover for each other; ordered like this they lose 10 %.
  constexpr bool kInterleave = C::NW == 8;
  constexpr int kReads = decltype(ra)::kReads + kParts * decltype(rb)::kReads, kLoads = decltype(la)::kChunks + decltype(lb)::kChunks;
  auto interleave = [&](int loads) {
    if constexpr (kInterleave) {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        if (i >= loads) break;
        __builtin_amdgcn_sched_group_barrier(0x020, 1, 0); // direct load
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0); // matrix instruction
      }
#pragma unroll
      for (int i = 0; i < kReads; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0); // LDS read
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      }
    }
  };
  // both halves of the stage in (al, bl); (an, bn): the other stage, which is on its way
  auto stage = [&](char *al, char *bl, const char *an, const char *bn) {
    read(al, bl, 1);
    multiply(0);
    interleave(0);
    prepare();                                           // (not behind the barrier, where everything waits for it)
    fence();
    issue(al, bl);
    read(an, bn, 0);
    multiply(1);
    interleave(kLoads);
  };
  prepare();
  issue(a_lds0, b_lds0);
  prepare();
  fence();
  issue(a_lds1, b_lds1);
  read(a_lds0, b_lds0, 0);
  // (one exit: a break behind the first stage made the compiler keep a second copy of the accumulators)
  for (int it = it0; it < it1; it += 2) {
    stage(a_lds0, b_lds0, a_lds1, b_lds1);
    if (it + 1 < it1) stage(a_lds1, b_lds1, a_lds0, b_lds0);
  }

  // ---- epilogue.  The accumulators pass through LDS, a wave's own part of it, up to 64 of its rows at a time: behind that a
  // lane has four consecutive columns, 16 (or 8) lanes a row, so that global accesses are whole lines and the element-wise
  // work is a short loop (unrolled over the accumulators it needs more registers than there are).
  constexpr int WA = decltype(ra)::kGroup, WB = decltype(rb)::kGroup;
  constexpr int CT = FM < 4 ? FM : 4, kCols = FN * 16, kQuads = kCols / 4;      // m tiles of a chunk; columns of the wave
  constexpr int kChunkBytes = CT * 16 * kCols * 4;
  static_assert(C::kA == C::kB && C::kA % kChunkBytes == 0 && kChunkBytes * C::NW <= 4 * C::kA, "");
  static_assert(FM % CT == 0 && CT % WA == 0 && (kQuads & (kQuads - 1)) == 0, "");
  fence();                                               // every wave has read its last stage; no direct load is in flight
  const int slot = wave * kChunkBytes / C::kA;
  char *mine = (slot == 0 ? a_lds0 : slot == 1 ? b_lds0 : slot == 2 ? a_lds1 : b_lds1) + wave * kChunkBytes % C::kA;
  const int i16 = lane & 15, g = lane >> 4;
  const bool whole = (P.ldc % 4 == 0) && ((uintptr_t)P.c & 15) == 0;
  const bool to_slab = C::kind == kPlain && P.split > 1;
  constexpr int kLanes = kQuads / kParts, kRows = 64 / kLanes;                    // lanes of a row, rows of a step
  constexpr int kSteps = CT * 16 / kRows, U = kSteps < 4 ? kSteps : 4;            // steps of a chunk, of a batch
  static_assert(kSteps % U == 0, "");
  static_assert((U * kRows) % 8 == 0, "a batch must not change the swizzle (quad ^ row % 8)");
  const int quad = lane % kLanes, r_lane = lane / kLanes;
  const int n = n0 + b_first + 4 * quad;
  const uint32_t row_step = kRows;
  // LDS address of step u of a batch (rows that are a multiple of the swizzle apart share it)
  int place[U][kParts];
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int part = 0; part < kParts; ++part) {
      const int r = u * kRows + r_lane;
      place[u][part] = r * (kCols * 4) + (((part * kLanes + quad) ^ (r & 7)) << 4);
    }
  float bias0[4], bias1[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    bias0[e] = P.bias0 && n + e < P.N && !to_slab ? (float)((const T *)P.bias0)[n + e] : 0.f;
    bias1[e] = kParts == 2 && P.bias1 && n + e < P.N ? (float)((const T *)P.bias1)[n + e] : 0.f;
  }
  // Whole rows of vectors (every column in one, the rows' padding counted, and rows at vector boundaries): buffer stores with
  // 32-bit offsets; rows behind the last and columns behind the padding fall outside the descriptor's bound and are dropped.
  // Of h, a, b, da and db that is every case (the launch checks it); y, dx and weight gradients of other widths or addresses go
  // element by element through put().  (1003 x 777 -> 2051, whose h, a, b, da and db are padded, fp16
  // trained: element by element 143 us, like this 130.)
  using OutT = T;
  const int cols = to_slab ? slab_ld(P.N) : max(P.N, P.pad);
  const bool vectors = C::kind != kPlain || ((cols & 3) == 0 && (to_slab || whole));
  const long ld_out = to_slab ? slab_ld(P.N) : P.ldc;
  const int size_out = to_slab ? 4 : (int)sizeof(OutT);
  const int m_base = m0 + a_first;
  const auto bound = [&](long ld, int size) -> uint32_t {               // bytes from (m_base, 0) to the last column of the last row
    const long bytes = ((long)(P.M - m_base - 1) * ld + cols) * size;
    return P.M <= m_base ? 0u : bytes > 0x7fffffffL ? 0x7fffffffu : (uint32_t)bytes;
  };
  const auto resource = [&](const void *base, long ld, int size) {
    return __builtin_amdgcn_make_buffer_rsrc((void *)((const char *)base + (long)m_base * ld * size), 0, bound(ld, size), 0x00020000);
  };
  const __amdgpu_buffer_rsrc_t rc = to_slab ? resource(P.slab + (long)slice * P.slab_stride, ld_out, 4) : resource(P.c, ld_out, size_out);
  __amdgpu_buffer_rsrc_t rc2 = rc, rx0 = rc, rx1 = rc;
  if constexpr (C::kind == kGrad) {
    rc2 = resource(P.c2, P.ldc, sizeof(T));
    rx0 = resource(P.aux0, P.ldaux, 4);
    rx1 = resource(P.aux1, P.ldaux, 4);
  } else if constexpr (C::kind == kGateUp) {
    rx0 = resource(P.out0, P.ldaux, 4);
    rx1 = resource(P.out1, P.ldaux, 4);
  }
  const bool exists = n < cols;
  const uint32_t step_out = row_step * (uint32_t)(ld_out * size_out), step_aux = row_step * (uint32_t)(P.ldaux * 4);
  const uint32_t off_out = exists ? (uint32_t)(r_lane * ld_out + n) * size_out : 0x80000000u;
  const uint32_t off_aux = exists ? (uint32_t)(r_lane * P.ldaux + n) * 4 : 0x80000000u;

  // what a batch reads from memory (kGrad: a and b); fetched one batch ahead, the first before the accumulators are staged
  struct Aux {
    f32x4 a[U], b[U];
  };
  auto fetch = [&](int step, Aux &x) {                   // step: counted over all chunks
    if constexpr (C::kind == kGrad) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const uint32_t off = off_aux + (step + u) * step_aux;
        x.a[u] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rx0, off, 0, 0));
        x.b[u] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rx1, off, 0, 0));
      }
    }
  };
  // kGrad: the lane's column sums of da and db, taken before their rounding (they are no operand of a product)
  float sum0[4] = {0.f, 0.f, 0.f, 0.f}, sum1[4] = {0.f, 0.f, 0.f, 0.f};
  // element-wise part of a batch: v (kParts x 4 of each step) -> o0, o1
  auto combine = [&](float (&v)[U][kParts][4], const Aux &x, float (&o0)[U][4], float (&o1)[U][4]) {
    if constexpr (C::kind == kPlain) {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) o0[u][e] = v[u][0][e] + bias0[e];
    } else {
      float a[U * 4], value[U * 4], slope[U * 4];
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if constexpr (C::kind == kGateUp) {
            v[u][0][e] += bias0[e];
            v[u][kParts - 1][e] += bias1[e];
            a[u * 4 + e] = v[u][0][e];
          } else {
            a[u * 4 + e] = x.a[u][e];
          }
        }
      activations<U * 4>(L.act, a, value, slope);
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if constexpr (C::kind == kGateUp) {
            // (zeros behind the last column also where a row of x is infinite: the next product reads them)
            o0[u][e] = n + e < P.N ? value[u * 4 + e] * v[u][kParts - 1][e] : 0.f;
          } else {
            // (W_down's rows follow each other: behind the last column there is the next row's first)
            o0[u][e] = n + e < P.N ? v[u][0][e] * x.b[u][e] * slope[u * 4 + e] : 0.f;
            o1[u][e] = n + e < P.N ? v[u][0][e] * value[u * 4 + e] : 0.f;
          }
        }
    }
  };
#pragma unroll
  for (int chunk = 0; chunk < FM / CT; ++chunk) {
    Aux next;
    fetch(chunk * kSteps, next);
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
        const int at = part * (FP * 4) + (col >> 2);
        *(f32x4 *)(mine + row * (kCols * 4) + ((at ^ (row & 7)) << 4)) = v;
      }
    }
    // (a wave's own LDS traffic is in order: the reads below see the writes above without a barrier)
    asm volatile("" ::: "memory");
#pragma unroll 1
    for (int step = 0; step < kSteps; step += U) {
      const Aux now = next;
      if (step + U < kSteps) fetch(chunk * kSteps + step + U, next);
      float v[U][kParts][4], o0[U][4], o1[U][4];
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int part = 0; part < kParts; ++part) {
          const f32x4 w = *(const f32x4 *)(mine + place[u][part] + step * (kRows * kCols * 4));
#pragma unroll
          for (int e = 0; e < 4; ++e) v[u][part][e] = w[e];
        }
      combine(v, now, o0, o1);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int done = chunk * kSteps + step + u;
        if constexpr (C::kind == kGrad) {
          if (m_base + done * kRows + r_lane < P.M) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              sum0[e] += o0[u][e];
              sum1[e] += o1[u][e];
            }
          }
        }
        if (vectors) {
          const uint32_t off = off_out + done * step_out;
          if (to_slab) store_buffer<float>(rc, off, o0[u]);
          else store_buffer<T>(rc, off, o0[u]);
          if constexpr (C::kind == kGrad) store_buffer<T>(rc2, off, o1[u]);
          if constexpr (C::kind == kGateUp) {
            if (P.out0) {
              // kept in 32 bits: rounded to the operands' 16 bits here, the gradients of x and W_gate would carry two
              // roundings more than the product's own operands do
              const uint32_t aux = off_aux + done * step_aux;
              store_buffer<float>(rx0, aux, v[u][0]);
              store_buffer<float>(rx1, aux, v[u][kParts - 1]);
            }
          }
        } else if constexpr (C::kind == kPlain) {
          const int m = m_base + done * kRows + r_lane;
          if (m < P.M) put<T>((T *)P.c + (long)m * P.ldc, n, P.N, 0, whole, o0[u]);
        }
      }
    }
    asm volatile("" ::: "memory");
  }
  if constexpr (C::kind == kGrad) {
    static_assert(C::WM == kWavesM, "");
    if (P.out0 || P.out1) {
      // over the lanes that hold the same columns, in a fixed order
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int apart = kLanes; apart < 64; apart *= 2) {
          sum0[e] += __shfl_xor(sum0[e], apart);
          sum1[e] += __shfl_xor(sum1[e], apart);
        }
      const long at = ((long)tm * kWavesM + wm) * P.N + n;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (r_lane == 0 && n + e < P.N) {
          if (P.out0) P.out0[at + e] = sum0[e];
          if (P.out1) P.out1[at + e] = sum1[e];
        }
    }
  }
}

}  // namespace ffn
