// Products of the feed-forward block on the matrix cores: the 8-bit product with token and channel
// scales, the gated projections h = act(x Wg^T) * (x Wu^T), and the products of their backward pass.
//
// All of them are C[m, n] = sum_k A[m, k] B[n, k] with both operands' rows contiguous in k, and one
// kernel body serves every type because it works on 16-byte pieces of rows: a lane's operand of an
// MFMA is 16 bytes of one row whatever the type (16 int8, 8 bf16 / fp16, 4 fp32), and the order in
// which the k of a product are summed over lanes is free as long as A and B agree on it.  (The backward
// pass's products read operands whose rows are rows of k across, see below.)
//
// Large products are bound by the MFMAs and, as closely, by LDS: a 256 x 256 tile reads 96 KB a run of 64
// bytes of k and is handed 32, which takes as long as its MFMAs; they are busy 59 % of the time at about
// 2.0 GHz.  Small ones are bound by the weights' bytes (few_rows) or by a launch's start and its one burst of
// stores.  Measured: 8 bits 8192^3 to bf16 450 us = 2.44 PTOP/s; bf16 forward 8192 x 8192 (two weights)
// over 2048 490 us, 590 with g and u kept (537 MB of stores more); dx and dw 475 each = 1.15 PFLOP/s;
// fp32 13312 x 1024 over 256 157, 156 and 130 us for three times 14 GFLOP; 8 bits 1 x 4096 over 4096
// 5.3 us = 3.2 TB/s of weights; 4 rows against a bf16 pair of 5632 x 2048 4.1 TB/s.
#include "common.h"

#include <type_traits>

namespace sage {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(1))) const void* gptr_t;
typedef __attribute__((address_space(3))) void* lptr_t;

// ------------------------------------------------------------------------------- types
// Frag: 16 bytes of a row.  mma: 16 x 16 outputs, all k of the two 64-byte row pieces held by the wave.
template <typename T>
struct Mma;
template <>
struct Mma<int8_t> {
  using Acc = i32x4;
  __device__ static Acc mma(const i32x4& a, const i32x4& b, const Acc& c) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0);
  }
};
template <>
struct Mma<__bf16> {
  using Acc = f32x4;
  __device__ static Acc mma(const i32x4& a, const i32x4& b, const Acc& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
};
template <>
struct Mma<_Float16> {
  using Acc = f32x4;
  __device__ static Acc mma(const i32x4& a, const i32x4& b, const Acc& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
};
template <>
struct Mma<float> {
  using Acc = f32x4;
  // four products of one k a lane: lane group q supplies k = 4 q + e of the 16 that the piece holds
  __device__ static Acc mma(const i32x4& a, const i32x4& b, Acc c) {
    const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[e], y[e], c, 0, 0, 0);
    return c;
  }
};

// ------------------------------------------------------------------------------- epilogues
// kExact: full-precision exponential and division (fp32 outputs); else the hardware's: the reciprocal is within
// 2^-23, the exponential's error grows with its argument (2^-24 |g| for the change of base, and a few 2^-24), and
// both vanish in a 16-bit rounding.  SiLU is 0 from about g = -87 on, where its value is below 1e-36.
template <bool kExact>
__device__ inline float sigmoid(float g) {
  if constexpr (kExact) return 1.f / (1.f + expf(-g));
  else return __builtin_amdgcn_rcpf(1.f + __expf(-g));
}
// Phi(g), the normal distribution, and exp(-g^2 / 2).  With a = |g| and t = 1 / (1 + p a), Phi(-a) = exp(-a^2 / 2) t P(t):
// P is of degree 8, fitted to erfcx(a / sqrt 2) / (2 t) on a <= 14 (where the exponential leaves the type) with the
// least relative error, 2^-26; evaluated, 8 * 2^-24 besides the exponential's.  From 1 + erf(g / sqrt 2) the values of
// negative g would be the difference of near-equal terms (4 % off at g = -5, nothing left from -5.5 on).
template <bool kExact>
__device__ inline float normal_below(float g, float* bell) {
  *bell = kExact ? expf(-0.5f * g * g) : __expf(-0.5f * g * g);
  const float t = __builtin_amdgcn_rcpf(fmaf(0.26521662f, fabsf(g), 1.f));
  float sum = 0.030827843f;
  sum = fmaf(sum, t, -0.14384112f);
  sum = fmaf(sum, t, 0.21640144f);
  sum = fmaf(sum, t, -0.11497585f);
  sum = fmaf(sum, t, 0.13705088f);
  sum = fmaf(sum, t, 0.060669467f);
  sum = fmaf(sum, t, 0.10269817f);
  sum = fmaf(sum, t, 0.10534162f);
  sum = fmaf(sum, t, 0.10582755f);
  const float below = *bell * (sum * t);
  return g < 0.f ? below : 1.f - below;
}
template <bool kExact>
__device__ inline float act_value(float g, int act) {
  if (act == SAGE_ACT_SILU) return g * sigmoid<kExact>(g);
  if (act == SAGE_ACT_GELU) {
    float bell;
    return g * normal_below<kExact>(g, &bell);
  }
  return g < 0.f ? 0.f : g;
}
template <bool kExact>
__device__ inline float act_slope(float g, int act) {
  if (act == SAGE_ACT_SILU) {
    const float p = sigmoid<kExact>(g);
    return p * (1.f + g * (1.f - p));
  }
  if (act == SAGE_ACT_GELU) {
    float bell;
    const float below = normal_below<kExact>(g, &bell);
    return fmaf(g * 0.39894228040143268f, bell, below);
  }
  return g > 0.f ? 1.f : 0.f;
}

struct Product {
  const char* a;        // A rows (bytes)
  const char* b0;       // B rows
  const char* b1;       // second B of a gated product
  int64_t lda, ldb0, ldb1;   // row strides in bytes
  int64_t m, n;         // outputs (n: of each B)
  int64_t kbytes;       // rows along k: their length in bytes, a multiple of 16
  int64_t depth;        // rows of k: how many (of each B, where b1 follows b0)
  void* out;
  int64_t ldo;          // in elements
  int out_dtype;
  int act;
  const float* sa;      // int8: scales of A's and B's rows
  const float* sb0;
  const float* sb1;
  const float* bias;
  int64_t fold, fold_rows;   // two outputs below each other: row fold + r is row fold_rows + r, fold_rows .. fold - 1 none
  float* saved;         // gated, training: pre-activations [2, m, n] in fp32
  // k in runs of 64 bytes: all of it; before b1's begin; before the first that k does not fill; of a slice
  int64_t runs, part_runs, whole_runs, slice_runs;
  i32x4* partial;       // k split over blockIdx.y: the slices' sums, as the waves hold them
};

template <int n, typename T>
struct __attribute__((packed, aligned(sizeof(T)))) Run {
  T v[n];
};

template <int n, typename T>
__device__ inline void store_run(T* p, int64_t left, const float (&v)[n]) {
  if (left >= n) {
    Run<n, T> r;
#pragma unroll
    for (int i = 0; i < n; ++i) r.v[i] = static_cast<T>(v[i]);
    *reinterpret_cast<Run<n, T>*>(p) = r;
  } else {
#pragma unroll
    for (int i = 0; i < n; ++i)
      if (i < left) p[i] = static_cast<T>(v[i]);
  }
}
template <int n>
__device__ inline void store_out(const Product& p, int64_t row, int64_t col, const float (&v)[n]) {
  const int64_t at = row * p.ldo + col, left = p.n - col;
  if (p.out_dtype == SAGE_BF16) store_run<n>(static_cast<__bf16*>(p.out) + at, left, v);
  else if (p.out_dtype == SAGE_F16) store_run<n>(static_cast<_Float16*>(p.out) + at, left, v);
  else store_run<n>(static_cast<float*>(p.out) + at, left, v);
}

// two values in T's 16 bits, the first in the low half
template <typename T>
__device__ inline uint32_t pack16(float a, float b) {
  const T r[2] = {static_cast<T>(a), static_cast<T>(b)};
  return __builtin_bit_cast(uint32_t, r);
}

// n values, zeros behind the `left` that are there
template <int n>
__device__ inline void load_run(const float* p, int64_t left, float (&v)[n]) {
  if (left >= n) {
    const Run<n, float> r = *reinterpret_cast<const Run<n, float>*>(p);
#pragma unroll
    for (int i = 0; i < n; ++i) v[i] = r.v[i];
  } else {
#pragma unroll
    for (int i = 0; i < n; ++i) v[i] = i < left ? p[i] : 0.f;
  }
}

// n consecutive columns of one row, from the sums of one B (8 bits: the other types' products with few rows are pairs)
template <typename T, int n, typename S>
__device__ inline void finish(const Product& p, int64_t row, int64_t col, const S (&c)[n]) {
  static_assert(std::is_same<T, int8_t>::value, "the form that is used");
  if (row >= p.m || col >= p.n) return;
  float v[n];
  const float sa = p.sa[row];
#pragma unroll
  for (int i = 0; i < n; ++i) {
    const int64_t at = col + i < p.n ? col + i : p.n - 1;
    v[i] = static_cast<float>(c[i]) * (sa * p.sb0[at]) + (p.bias != nullptr ? p.bias[at] : 0.f);
  }
  store_out<n>(p, row, col, v);
}

// the same from the sums of both Bs
template <typename T, int n, typename S>
__device__ inline void finish_gated(const Product& p, int64_t row, int64_t col, const S (&cg)[n], const S (&cu)[n]) {
  if (row >= p.m || col >= p.n) return;
  float g[n], u[n], v[n];
  if constexpr (std::is_same<T, int8_t>::value) {
    const float sa = p.sa[row];
#pragma unroll
    for (int i = 0; i < n; ++i) {
      const int64_t at = col + i < p.n ? col + i : p.n - 1;
      g[i] = static_cast<float>(cg[i]) * (sa * p.sb0[at]);
      u[i] = static_cast<float>(cu[i]) * (sa * p.sb1[at]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < n; ++i) {
      g[i] = cg[i];
      u[i] = cu[i];
    }
    if (p.saved != nullptr) {
      store_run<n>(p.saved + row * p.n + col, p.n - col, g);
      store_run<n>(p.saved + (p.m + row) * p.n + col, p.n - col, u);
    }
  }
  if (p.out_dtype == SAGE_F32) {
#pragma unroll
    for (int i = 0; i < n; ++i) v[i] = act_value<true>(g[i], p.act) * u[i];
  } else {
#pragma unroll
    for (int i = 0; i < n; ++i) v[i] = act_value<false>(g[i], p.act) * u[i];
  }
  store_out<n>(p, row, col, v);
}

// 16 zero bytes that lanes read whose piece lies behind the row's end
__device__ const i32x4 kZeroPiece = {0, 0, 0, 0};

// ------------------------------------------------------------------------------- tiles
// kTile x kTile outputs a block (gated: kTile / 2 of each B), 2 x 4 waves at 256 and 2 x 2 at 128, so that a wave
// has 64 slots of B and 128 or 64 rows of A.
//
// An operand's rows lie along k (its tile: kTile rows of 64 bytes of k a run), or they are rows of k whose elements
// are the outputs' rows or columns (kAT, kBT: 64 / sizeof(T) rows of kTile elements a run), as the weights' gradients
// and dx want them; both fill kTile * 64 bytes of LDS a run.  Tiles go straight from memory to LDS
// (global_load_lds, 16 bytes a lane, no registers); LDS holds four runs in a ring, separate arrays so that the
// compiler's waits for one do not cover the others.
//
// LDS order: rows along k: piece c (of 4) of row r lies at c ^ ((r >> 2) & 3), so that the 16 rows of an MFMA operand
// fall on all banks.  Rows of k, 16 bits: the operand is read with the transposing read (a group of 16 lanes takes
// 4 rows x 16 elements and each lane leaves with a column's 4), and the 32 bytes c of row r lie at c ^ f,
// f = r & 3 | (r >> 3 & 1) << 2, so that the 8 rows of half a wave fall on all banks.  fp32: four plain reads, and the
// 64 bytes c of row r lie at c ^ (r >> 2 & 3).
//
// A wave's 64 slots of B are 64 columns, gated 32 of the first B and the same 32 of the second.  Where B's rows lie
// along k, any column may be any slot: slot 16 j + i is column 4 i + j (gated 2 i + j % 2 of B j / 2), so that the 16
// lanes that the MFMA leaves a row of C in hold 4 (2) consecutive columns each.
template <int kTile, bool kGated>
struct TileShape {
  static constexpr int kThreads = kTile == 256 ? 512 : 256;
  static constexpr int WM = 2, WN = kTile / 64;
  static constexpr int kMI = kTile / WM / 16, kNI = 4;
  static constexpr int kColsOut = kGated ? kTile / 2 : kTile;
};

template <bool kGated>
__device__ inline int slot_column(int s, int* which) {
  const int wn = s >> 6, j = (s >> 4) & 3, i = s & 15;
  *which = kGated ? j >> 1 : 0;
  return kGated ? wn * 32 + 2 * i + (j & 1) : wn * 64 + 4 * i + j;
}

// The tile of a block: each XCD (blockIdx modulo 8) takes a contiguous run of them, so that its L2 holds what
// they share.
__device__ inline int xcd_tile(int block, int total) {
  const int per = total / 8, rest = total % 8, xcd = block % 8;
  return xcd * per + (xcd < rest ? xcd : rest) + block / 8;
}

// Tile t's place: runs of tiles go down groups of 8 tile rows, so that the blocks of a run share operands.
__device__ inline void tile_place(int tile, int tiles_m, int tiles_n, int* tm, int* tn) {
  constexpr int kGroup = 8;
  const int group = tile / (kGroup * tiles_n);
  const int first_m = group * kGroup;
  const int rows = tiles_m - first_m < kGroup ? tiles_m - first_m : kGroup;
  const int in = tile - group * kGroup * tiles_n;
  *tm = first_m + in % rows;
  *tn = in / rows;
}

// 16 rows of C from one wave's sums, B along k.  The MFMA's rows are A's: lane l holds, of slot group j, slot l & 15 of
// rows 4 (l >> 4) + 0..3, which the slot order makes consecutive columns over j: a store is 256 bytes of a row in fp32
// and 128 in 16 bits (gated 128 and 64).  kFull: all of the block's rows and columns are there; kAct, kOut: the
// activation and the output's type, or -1: known at run time.
template <typename T, bool kGated, bool kFull, int kAct, int kOut, typename Acc>
__device__ inline void finish_along(const Product& p, int64_t r0, int64_t col, const Acc (&acc)[4]) {
  constexpr int n = kGated ? 2 : 4;
  const int64_t left = kFull ? n : p.n - col;
  if (!kFull && left <= 0) return;
  const int act = kAct < 0 ? p.act : kAct, out_dtype = kOut < 0 ? p.out_dtype : kOut;
  float s0[n], s1[n], bias[n];
  if constexpr (std::is_same<T, int8_t>::value) {
    load_run<n>(p.sb0 + col, left, s0);
    if constexpr (kGated) load_run<n>(p.sb1 + col, left, s1);
    if (p.bias != nullptr) load_run<n>(p.bias + col, left, bias);
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int64_t r = r0 + e;
    if (!kFull && r >= p.m) continue;
    float v[n], u[n];
    if constexpr (std::is_same<T, int8_t>::value) {
      const float sa = p.sa[r];
#pragma unroll
      for (int j = 0; j < n; ++j) {
        v[j] = static_cast<float>(acc[j][e]) * (sa * s0[j]) + (p.bias != nullptr ? bias[j] : 0.f);
        if constexpr (kGated) u[j] = static_cast<float>(acc[2 + j][e]) * (sa * s1[j]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < n; ++j) {
        v[j] = acc[j][e];
        if constexpr (kGated) u[j] = acc[2 + j][e];
      }
      if constexpr (kGated) {
        if (p.saved != nullptr) {
          store_run<n>(p.saved + r * p.n + col, left, v);
          store_run<n>(p.saved + (p.m + r) * p.n + col, left, u);
        }
      }
    }
    if constexpr (kGated) {
#pragma unroll
      for (int j = 0; j < n; ++j)
        v[j] = (out_dtype == SAGE_F32 ? act_value<true>(v[j], act) : act_value<false>(v[j], act)) * u[j];
    }
    const int64_t at = r * p.ldo + col;
    if (out_dtype == SAGE_BF16) store_run<n>(static_cast<__bf16*>(p.out) + at, left, v);
    else if (out_dtype == SAGE_F16) store_run<n>(static_cast<_Float16*>(p.out) + at, left, v);
    else store_run<n>(static_cast<float*>(p.out) + at, left, v);
  }
}

// The same where B's rows are rows of k, whose slots are columns in order.  There B's slots are the MFMA's rows: lane l
// holds row l & 15, and of slot group j slots 4 q + 0..3, q = l >> 4.  In 16 bits two groups trade halves between the
// lanes of odd and even q first, and lane q stores 8 consecutive columns, 8 (q >> 1) and on, of group j + (q & 1)
// (dx and dw of 8192 x 8192 over 2048 in bf16 486 -> 436 us).
template <typename T, typename Acc>
__device__ inline void finish_across(const Product& p, int64_t m0, int64_t n0, int row, int wn, int lane, const Acc (&acc)[4]) {
  const int q = lane >> 4;
  int64_t r = m0 + row + (lane & 15);
  bool kept = r < p.m;
  const int64_t col0 = n0 + wn * 64;
  if (p.fold > p.fold_rows) {
    if (r >= p.fold) r -= p.fold - p.fold_rows;
    else kept = kept && r < p.fold_rows;
  }
  if constexpr (std::is_same<T, float>::value) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t col = col0 + j * 16 + q * 4;
      const float v[4] = {acc[j][0], acc[j][1], acc[j][2], acc[j][3]};
      if (kept && col < p.n) store_run<4>(static_cast<float*>(p.out) + r * p.ldo + col, p.n - col, v);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; j += 2) {
      uint32_t all[4];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const auto t = __builtin_amdgcn_permlane16_swap(pack16<T>(acc[j][2 * e], acc[j][2 * e + 1]),
                                                        pack16<T>(acc[j + 1][2 * e], acc[j + 1][2 * e + 1]), false, false);
        all[e] = t[0];
        all[2 + e] = t[1];
      }
      const int64_t col = col0 + (j + (q & 1)) * 16 + (q >> 1) * 8, left = p.n - col;
      uint16_t* to = static_cast<uint16_t*>(p.out) + r * p.ldo + col;
      if (kept && left >= 8) {
        Run<8, uint16_t> run;
#pragma unroll
        for (int e = 0; e < 8; ++e) run.v[e] = static_cast<uint16_t>(all[e >> 1] >> (16 * (e & 1)));
        *reinterpret_cast<Run<8, uint16_t>*>(to) = run;
      } else if (kept) {
#pragma unroll
        for (int e = 0; e < 7; ++e)
          if (e < left) to[e] = static_cast<uint16_t>(all[e >> 1] >> (16 * (e & 1)));
      }
    }
  }
}

// kMI groups of 16 rows by 64 slots of C from a wave's sums.  The common activation and output types are compiled by
// themselves, and blocks that are all there: the choices, made for every run of columns, took longer than the values
// (the forward pass of 8192 x 8192 over 2048 in bf16 that keeps its sums 728 -> 598 us).
template <typename T, bool kGated, bool kBT, int kMI, typename Acc>
__device__ inline void finish_rows(const Product& p, int64_t m0, int64_t n0, int row, int wn, int lane, bool full, const Acc (&acc)[kMI][4]) {
  if constexpr (kBT) {
#pragma unroll
    for (int i = 0; i < kMI; ++i) finish_across<T>(p, m0, n0, row + i * 16, wn, lane, acc[i]);
  } else {
    constexpr int n = kGated ? 2 : 4;
    const int64_t r0 = m0 + row + (lane >> 4) * 4, col = n0 + (wn * 16 + (lane & 15)) * n;
    auto all = [&](auto is_full, auto act, auto out) {
#pragma unroll
      for (int i = 0; i < kMI; ++i)
        finish_along<T, kGated, decltype(is_full)::value, decltype(act)::value, decltype(out)::value>(p, r0 + i * 16, col, acc[i]);
    };
    using any = std::integral_constant<int, -1>;
    using silu = std::integral_constant<int, SAGE_ACT_SILU>;
    if constexpr (std::is_same<T, int8_t>::value) {
      using bf16 = std::integral_constant<int, SAGE_BF16>;
      using f32 = std::integral_constant<int, SAGE_F32>;
      const int out = kGated && p.act != SAGE_ACT_SILU ? -1 : p.out_dtype;
      if (out == SAGE_BF16 && full) all(std::true_type{}, silu{}, bf16{});
      else if (out == SAGE_BF16) all(std::false_type{}, silu{}, bf16{});
      else if (out == SAGE_F32 && full) all(std::true_type{}, silu{}, f32{});
      else if (out == SAGE_F32) all(std::false_type{}, silu{}, f32{});
      else all(std::false_type{}, any{}, any{});
    } else {
      using out = std::integral_constant<int, std::is_same<T, float>::value ? SAGE_F32 : std::is_same<T, __bf16>::value ? SAGE_BF16 : SAGE_F16>;
      if (full && p.act == SAGE_ACT_SILU) all(std::true_type{}, silu{}, out{});
      else if (p.act == SAGE_ACT_SILU) all(std::false_type{}, silu{}, out{});
      else all(std::false_type{}, any{}, out{});
    }
  }
}

// Where a lane's two loads of an operand's run come from, as offsets of 32 bits from the tile's first row (strides are
// below 2^23 bytes), and which of them lie behind the end of k.
template <typename T, int kTile, bool kTransposed>
struct Lanes {
  static constexpr int kThreads = kTile == 256 ? 512 : 256;
  uint32_t off[2];
  int at[2];      // rows along k: byte of the run; rows of k: row of the run

  // rows along k: `of(r)` is the operand's row for LDS row r
  template <typename F>
  __device__ void along(int wave, int lane, uint32_t ld, F&& of) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      at[j] = ((lane & 3) ^ ((lane >> 4) & 3)) * 16;
      off[j] = static_cast<uint32_t>(of(j * (kThreads / 4) + wave * 16 + (lane >> 2))) * ld + at[j];
    }
  }
  // rows of k; `last`: the last piece of 16 bytes that the row has (what is behind it is not stored)
  __device__ void across(int wave, int lane, uint32_t ld, int last) {
    constexpr int kPieces = kTile * static_cast<int>(sizeof(T)) / 16;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int index = j * kThreads + wave * kWave + lane, r = index / kPieces, to = index % kPieces;
      int from;
      if constexpr (sizeof(T) == 2) from = ((to >> 1) ^ ((r & 3) | ((r >> 3 & 1) << 2))) << 1 | (to & 1);
      else from = to ^ ((r >> 2 & 3) << 2);
      at[j] = r;
      off[j] = static_cast<uint32_t>(r) * ld + (from < last ? from : last) * 16;
    }
  }
};

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4* lds16_t;

// An MFMA operand: 16 rows or slots (those of the 16 that begin at 16 * c) by 64 bytes of k
template <typename T, int kTile, bool kTransposed>
__device__ inline i32x4 operand(const char* tile, int c, int lane) {
  const int l15 = lane & 15, q = lane >> 4;
  if constexpr (!kTransposed) {
    return *reinterpret_cast<const i32x4*>(tile + (c * 16 + l15) * 64 + (q ^ ((l15 >> 2) & 3)) * 16);
  } else if constexpr (sizeof(T) == 2) {
    constexpr int kRow = kTile * 2;
    const int r = l15 >> 2;            // rows 8 q + r and 8 q + 4 + r
    const char* at = tile + (8 * q + r) * kRow + ((c ^ (r | ((q & 1) << 2))) * 32 + (l15 & 3) * 8);
    union {
      s16x4 half[2];
      i32x4 whole;
    } v;
    v.half[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds16_t)(at));
    v.half[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds16_t)(at + 4 * kRow));
    return v.whole;
  } else {
    constexpr int kRow = kTile * 4;
    const char* at = tile + 4 * q * kRow + ((c ^ q) * 64 + l15 * 4);
    i32x4 v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = *reinterpret_cast<const int*>(at + e * kRow);
    return v;
  }
}

// The ring: run u lies in stage u % 4.  Before run u is read, run u + 3 is fetched into the place of run u - 1, whose
// readers have met since; at most 8 loads a wave (runs u + 2 and u + 3) are under way when run u + 1 is next.
//
// At 256, two waves share a SIMD, one of each half of the block (wave / 4), and the halves run half a phase apart:
// while one half's waves read their operands from LDS, the other's multiply.  Run u is read in phase 2 u by the first
// half and in phase 2 u + 1 by the second, and multiplied in the phase after; every phase ends at a barrier of the
// whole block (the second half passes one more before its first phase, the first half one more behind its last).
// Run u - 1 was last read in phase 2 u - 1, and its reads had landed (lgkmcnt(0)) before the barrier that ended it, so
// run u + 3 may be fetched from phase 2 u on; run u + 1 is first read in phase 2 u + 2, and at the end of their reading
// phases 2 u and 2 u + 1 both halves have waited for their loads of it.
//
// At 128, two blocks share a CU instead, and a run is one phase: wait, meet, fetch, read, multiply.
template <typename T, int kTile, bool kGated, bool kAT, bool kBT>
__global__ void __launch_bounds__(kTile == 256 ? 512 : 256, 2) tile_kernel(Product p, int tiles_m, int tiles_n) {
  using S = TileShape<kTile, kGated>;
  using Acc = typename Mma<T>::Acc;
  constexpr int kHalf = kTile * 64, kRows = 64 / static_cast<int>(sizeof(T));
  static_assert(!(kGated && (kAT || kBT)) && (!kAT || kBT), "the forms that are used");
  __shared__ __attribute__((aligned(1024))) char stage0[2 * kHalf];
  __shared__ __attribute__((aligned(1024))) char stage1[2 * kHalf];
  __shared__ __attribute__((aligned(1024))) char stage2[2 * kHalf];
  __shared__ __attribute__((aligned(1024))) char stage3[2 * kHalf];
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int total = tiles_m * tiles_n;
  const int tile = xcd_tile(blockIdx.x, total);
  int tm, tn;
  tile_place(tile, tiles_m, tiles_n, &tm, &tn);
  const int64_t m0 = static_cast<int64_t>(tm) * kTile, n0 = static_cast<int64_t>(tn) * S::kColsOut;

  const int64_t first = static_cast<int64_t>(blockIdx.y) * p.slice_runs;         // runs of this block
  const int64_t runs = p.runs - first < p.slice_runs ? p.runs - first : p.slice_runs;
  const bool up = kGated && ((wave >> 1) & 1);          // slots 32 to 63 of each 64 are the second B's
  const uint32_t lda = static_cast<uint32_t>(p.lda), ldb = static_cast<uint32_t>(up ? p.ldb1 : p.ldb0);
  const int rows_left = p.m - m0 < kTile ? static_cast<int>(p.m - m0) : kTile;
  const int cols_left = p.n - n0 < S::kColsOut ? static_cast<int>(p.n - n0) : S::kColsOut;
  Lanes<T, kTile, kAT> la;
  Lanes<T, kTile, kBT> lb;
  // rows and columns behind the last repeat it: their outputs are not stored
  if constexpr (kAT) la.across(wave, lane, lda, (rows_left * static_cast<int>(sizeof(T)) - 1) / 16);
  else la.along(wave, lane, lda, [&](int r) { return r < rows_left ? r : rows_left - 1; });
  if constexpr (kBT) {
    lb.across(wave, lane, ldb, (cols_left * static_cast<int>(sizeof(T)) - 1) / 16);
  } else {
    lb.along(wave, lane, ldb, [&](int r) {
      int which;
      const int c = slot_column<kGated>(r, &which);
      return c < cols_left ? c : cols_left - 1;
    });
  }
  const char* a_base = kAT ? p.a + m0 * sizeof(T) : p.a + m0 * p.lda;
  const char* b_base = kBT ? p.b0 + n0 * sizeof(T) : up ? p.b1 + n0 * p.ldb1 : p.b0 + n0 * p.ldb0;
  const char* b_base1 = kBT ? p.b1 + n0 * sizeof(T) : nullptr;
  const char* zero = reinterpret_cast<const char*>(&kZeroPiece);
  // kWhole: every element of the run is there; else pieces and rows behind the end of k are zeros (and runs behind
  // the last are all zeros: the number of loads under way is always the same)
  auto fetch = [&](char* stage, int64_t run, auto whole) {
    constexpr bool kWhole = decltype(whole)::value;
    const int64_t u = first + run;
    const bool second = kBT && u >= p.part_runs;
    const int64_t ub = second ? u - p.part_runs : u;
    const char* a = a_base + (kAT ? u * kRows * p.lda : u * 64);
    const char* b = (second ? b_base1 : b_base) + (kBT ? ub * kRows * p.ldb0 : u * 64);
    const int64_t left_a = kAT ? p.depth - u * kRows : p.kbytes - u * 64, left_b = kBT ? p.depth - ub * kRows : p.kbytes - u * 64;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const bool in_a = kWhole || la.at[j] < left_a, in_b = kWhole || lb.at[j] < left_b;
      char* to = stage + (j * S::kThreads + wave * kWave) * 16;
      __builtin_amdgcn_global_load_lds((gptr_t)(in_a ? a + la.off[j] : zero), (lptr_t)(to), 16, 0, 0);
      __builtin_amdgcn_global_load_lds((gptr_t)(in_b ? b + lb.off[j] : zero), (lptr_t)(to + kHalf), 16, 0, 0);
    }
  };

  Acc acc[S::kMI][S::kNI];
#pragma unroll
  for (int i = 0; i < S::kMI; ++i)
#pragma unroll
    for (int j = 0; j < S::kNI; ++j) acc[i][j] = Acc{};
  const int wm = wave / S::WN, wn = wave % S::WN;
  i32x4 a[S::kMI], b[S::kNI];
  auto read = [&](const char* stage) {
#pragma unroll
    for (int j = 0; j < S::kNI; ++j) b[j] = operand<T, kTile, kBT>(stage + kHalf, wn * S::kNI + j, lane);
#pragma unroll
    for (int i = 0; i < S::kMI; ++i) a[i] = operand<T, kTile, kAT>(stage, wm * S::kMI + i, lane);
  };
  auto multiply = [&]() {
#pragma unroll
    for (int i = 0; i < S::kMI; ++i)
#pragma unroll
      for (int j = 0; j < S::kNI; ++j) acc[i][j] = kBT ? Mma<T>::mma(b[j], a[i], acc[i][j]) : Mma<T>::mma(a[i], b[j], acc[i][j]);
  };
  auto meet = [&]() {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };
  // Until a wave's LDS reads have landed and no more than the loads of two runs are under way.  (The builtin,
  // whose counts the compiler takes into account: it adds no waits of its own.)
  auto wait_loads = [&]() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0078);        // vmcnt(8) lgkmcnt(0)
    asm volatile("" ::: "memory");
  };
  const int half = wave >> 2;
  auto run_step = [&](const char* now, char* then, int64_t u, auto whole) {
    if constexpr (kTile == 256) {
      fetch(then, u + 3, whole);
      read(now);
      wait_loads();
      meet();
      __builtin_amdgcn_s_setprio(1);
      multiply();
      __builtin_amdgcn_s_setprio(0);
      meet();
    } else {
      wait_loads();
      meet();
      fetch(then, u + 3, whole);
      read(now);
      multiply();
    }
  };
  fetch(stage0, 0, std::false_type{});
  fetch(stage1, 1, std::false_type{});
  fetch(stage2, 2, std::false_type{});
  if constexpr (kTile == 256) {
    wait_loads();
    meet();
    if (half) meet();
  }
  int64_t u = 0;
  const int64_t whole = p.whole_runs - first < runs ? p.whole_runs - first : runs;     // runs before the first that is not
  for (; u + 7 <= whole; u += 4) {
    run_step(stage0, stage3, u, std::true_type{});
    run_step(stage1, stage0, u + 1, std::true_type{});
    run_step(stage2, stage1, u + 2, std::true_type{});
    run_step(stage3, stage2, u + 3, std::true_type{});
  }
  for (; runs - u > 7; u += 4) {
    run_step(stage0, stage3, u, std::false_type{});
    run_step(stage1, stage0, u + 1, std::false_type{});
    run_step(stage2, stage1, u + 2, std::false_type{});
    run_step(stage3, stage2, u + 3, std::false_type{});
  }
  // the last one to seven, in a row: left early from inside a loop, the compiler would see ways back to its head on
  // which loads are under way that are not, and wait for them
  do {
    run_step(stage0, stage3, u, std::false_type{});
    if (u + 1 >= runs) break;
    run_step(stage1, stage0, u + 1, std::false_type{});
    if (u + 2 >= runs) break;
    run_step(stage2, stage1, u + 2, std::false_type{});
    if (u + 3 >= runs) break;
    run_step(stage3, stage2, u + 3, std::false_type{});
    if (u + 4 >= runs) break;
    run_step(stage0, stage3, u + 4, std::false_type{});
    if (u + 5 >= runs) break;
    run_step(stage1, stage0, u + 5, std::false_type{});
    if (u + 6 >= runs) break;
    run_step(stage2, stage1, u + 6, std::false_type{});
  } while (false);
  if (kTile == 256 && !half) meet();
  __builtin_amdgcn_s_waitcnt(0x0070);        // no load is under way into LDS when the block gives it back

  if (p.partial != nullptr) {
    i32x4* to = p.partial + ((static_cast<int64_t>(blockIdx.y) * total + tile) * (S::WM * S::WN) + wave) * (S::kMI * S::kNI) * kWave + lane;
#pragma unroll
    for (int i = 0; i < S::kMI; ++i)
#pragma unroll
      for (int j = 0; j < S::kNI; ++j) to[(i * S::kNI + j) * kWave] = __builtin_bit_cast(i32x4, acc[i][j]);
    return;
  }
  finish_rows<T, kGated, kBT, S::kMI>(p, m0, n0, wm * S::kMI * 16, wn, lane, rows_left == kTile && cols_left == S::kColsOut, acc);
}

// The slices' sums of a split product, added in order by waves that each take the 16 rows that one wave
// of the tile kernel holds in acc[i], and finished as there.
template <typename T, int kTile, bool kGated, bool kBT>
__global__ void __launch_bounds__(256) join_kernel(Product p, int tiles_m, int tiles_n, int slices) {
  using S = TileShape<kTile, kGated>;
  using Acc = typename Mma<T>::Acc;
  const int lane = threadIdx.x & (kWave - 1);
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * 4 + threadIdx.x / kWave;   // (tile, wave, i)
  const int64_t total = static_cast<int64_t>(tiles_m) * tiles_n, per_tile = S::WM * S::WN * S::kMI;
  if (unit >= total * per_tile) return;
  const int tile = static_cast<int>(unit / per_tile), in_tile = static_cast<int>(unit - tile * per_tile);
  const int wave = in_tile / S::kMI, i = in_tile - wave * S::kMI;
  int tm, tn;
  tile_place(tile, tiles_m, tiles_n, &tm, &tn);
  const i32x4* from = p.partial + ((static_cast<int64_t>(tile) * (S::WM * S::WN) + wave) * S::kMI + i) * S::kNI * kWave + lane;
  const int64_t stride = total * (S::WM * S::WN) * S::kMI * S::kNI * kWave;
  Acc acc[1][S::kNI];
#pragma unroll
  for (int j = 0; j < S::kNI; ++j) acc[0][j] = __builtin_bit_cast(Acc, from[j * kWave]);
  constexpr int kAhead = 4;      // slices under way at once (48 slices 17 -> 11 us; with 8, whose places behind the last load it again, 2 or 3 slices cost a microsecond more)
  for (int s = 1; s < slices; s += kAhead) {
    i32x4 part[kAhead][S::kNI];
#pragma unroll
    for (int t = 0; t < kAhead; ++t) {
      const int of = s + t < slices ? s + t : s;
#pragma unroll
      for (int j = 0; j < S::kNI; ++j) part[t][j] = from[of * stride + j * kWave];
    }
    asm volatile("" ::: "memory");      // the loads stay in front of the first sum
#pragma unroll
    for (int t = 0; t < kAhead; ++t) {
      if (s + t >= slices) break;
#pragma unroll
      for (int j = 0; j < S::kNI; ++j) acc[0][j] += __builtin_bit_cast(Acc, part[t][j]);
    }
  }
  const int64_t m0 = static_cast<int64_t>(tm) * kTile, n0 = static_cast<int64_t>(tn) * S::kColsOut;
  finish_rows<T, kGated, kBT, 1>(p, m0, n0, (wave / S::WN * S::kMI + i) * 16, wave % S::WN, lane,
                                 m0 + kTile <= p.m && n0 + S::kColsOut <= p.n, acc);
}

// ------------------------------------------------------------------------------- few rows
// 16 * MT rows of A (grid y: more of them) against the whole of B: B goes straight into the registers that
// the MFMAs take, so the kernel is as fast as B's bytes arrive.  A block owns 16 * NT columns (gated: of
// each B); its waves take k in runs of 256 bytes in turn and add their sums in LDS, in wave order.
constexpr int kFewWaves = 8;

// 16 bytes of a row of T at `at`, zeros behind its end.  kRagged: rows of any length and alignment (at least 16 bytes).
// In a wave's last turn a row's last piece is its last 16 bytes moved down.  Rows that start inside a 4-byte word are read
// as the words that hold them (at most the 3 bytes before and behind them that share a word with theirs), shifted into
// place: bf16, 4 rows against a pair of 5632 x 2047 23 us, 40 as loads that cross words, 32 through padded copies.
template <typename T, bool kRagged>
__device__ inline i32x4 load_piece(const char* row, int64_t at, int64_t kbytes, bool last) {
  const i32x4 none = {0, 0, 0, 0};
  if constexpr (!kRagged) return at < kbytes ? *reinterpret_cast<const i32x4*>(row + at) : none;
  struct __attribute__((packed, aligned(4))) Words {
    i32x4 v;
  };
  const int64_t from = at + 16 <= kbytes ? at : kbytes - 16;
  i32x4 v;
  if constexpr (sizeof(T) == 4) {
    v = reinterpret_cast<const Words*>(row + from)->v;
  } else {
    const int off = static_cast<int>(reinterpret_cast<uintptr_t>(row + from) & 3);
    const char* word = row + from - off;
    const i32x4 lo = reinterpret_cast<const Words*>(word)->v;
    const uint32_t next = *reinterpret_cast<const uint32_t*>(word + (off ? 16 : 12));   // no word behind a row that ends with one
    const uint32_t w[5] = {static_cast<uint32_t>(lo[0]), static_cast<uint32_t>(lo[1]), static_cast<uint32_t>(lo[2]), static_cast<uint32_t>(lo[3]), next};
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = static_cast<int>(__builtin_amdgcn_alignbyte(w[i + 1], w[i], off));
  }
  if (last) {
    unsigned __int128 bits = __builtin_bit_cast(unsigned __int128, v);
    const int64_t over = at - from;
    bits = over < 16 ? bits >> (over * 8) : 0;
    v = __builtin_bit_cast(i32x4, bits);
  }
  return v;
}

template <typename T, int MT, bool kGated, int NT, bool kRagged>
__global__ void __launch_bounds__(kFewWaves* kWave) few_rows_kernel(Product p) {
  using Acc = typename Mma<T>::Acc;
  constexpr int NB = kGated ? 2 : 1, NC = NB * NT, U = 4;
  __shared__ Acc lds[kFewWaves][MT * NC][kWave];
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const int l15 = lane & 15, q = lane >> 4;
  const int64_t n0 = static_cast<int64_t>(blockIdx.x) * (16 * NT), m0 = static_cast<int64_t>(blockIdx.y) * (16 * MT);
  const char* b[NC];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int64_t col = n0 + t * 16 + l15 < p.n ? n0 + t * 16 + l15 : p.n - 1;
    b[t * NB] = p.b0 + col * p.ldb0;
    if constexpr (kGated) b[t * NB + 1] = p.b1 + col * p.ldb1;
  }
  const char* a[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int64_t row = m0 + i * 16 + l15 < p.m ? m0 + i * 16 + l15 : p.m - 1;
    a[i] = p.a + row * p.lda;
  }
  Acc acc[MT][NC];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NC; ++j) acc[i][j] = Acc{};
  // U pieces of 64 bytes a turn: contiguous bytes of a row, all loads before the first product
  for (int64_t k = wave * (U * 64); k < p.kbytes; k += kFewWaves * U * 64) {
    const bool last = k + U * 64 > p.kbytes;
    i32x4 bv[U][NC], av[U][MT];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < NC; ++j) bv[u][j] = load_piece<T, kRagged>(b[j], k + u * 64 + q * 16, p.kbytes, last);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < MT; ++i) av[u][i] = load_piece<T, kRagged>(a[i], k + u * 64 + q * 16, p.kbytes, last);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NC; ++j) acc[i][j] = Mma<T>::mma(bv[u][j], av[u][i], acc[i][j]);
  }
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NC; ++j) lds[wave][i * NC + j][lane] = acc[i][j];
  __syncthreads();
  using E = std::conditional_t<std::is_same<T, int8_t>::value, int, float>;
  for (int o = wave; o < MT * NT; o += kFewWaves) {
    const int i = o / NT, t = o % NT;
    Acc sum[NB];
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      const int at = i * NC + t * NB + j;
      sum[j] = lds[0][at][lane];
#pragma unroll
      for (int w = 1; w < kFewWaves; ++w) sum[j] += lds[w][at][lane];
    }
    const int64_t row = m0 + i * 16 + l15, at = n0 + t * 16 + q * 4;
    E c[4], d[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      c[e] = sum[0][e];
      d[e] = sum[NB - 1][e];
    }
    if constexpr (kGated) finish_gated<T, 4>(p, row, at, c, d);
    else finish<T, 4>(p, row, at, c);
  }
}

// Up to 16 rows against a pair of Bs: a block owns 8 columns of each, whose rows are the 16 slots of one MFMA operand
// (0 to 7 the first B's, 8 to 15 the second's), so that there are twice as many blocks to share out over the CUs.
template <typename T, int U, bool kRagged>
__global__ void __launch_bounds__(kFewWaves* kWave) few_rows_pair_kernel(Product p) {
  using Acc = typename Mma<T>::Acc;
  __shared__ Acc lds[kFewWaves][kWave];
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const int l15 = lane & 15, q = lane >> 4;
  const int64_t n0 = static_cast<int64_t>(blockIdx.x) * 8;
  const int64_t col = n0 + (l15 & 7) < p.n ? n0 + (l15 & 7) : p.n - 1, row = l15 < p.m ? l15 : p.m - 1;
  const char* b = l15 < 8 ? p.b0 + col * p.ldb0 : p.b1 + col * p.ldb1;
  const char* a = p.a + row * p.lda;
  Acc acc = Acc{};
  for (int64_t k = wave * (U * 64); k < p.kbytes; k += kFewWaves * U * 64) {
    const bool last = k + U * 64 > p.kbytes;
    i32x4 bv[U], av[U];
#pragma unroll
    for (int u = 0; u < U; ++u) bv[u] = load_piece<T, kRagged>(b, k + u * 64 + q * 16, p.kbytes, last);
#pragma unroll
    for (int u = 0; u < U; ++u) av[u] = load_piece<T, kRagged>(a, k + u * 64 + q * 16, p.kbytes, last);
#pragma unroll
    for (int u = 0; u < U; ++u) acc = Mma<T>::mma(bv[u], av[u], acc);
  }
  lds[wave][lane] = acc;
  __syncthreads();
  if (threadIdx.x >= 32) return;      // lane: row l15, slots 4 q + 0..3 of the first B; 32 lanes on the second's
  Acc g = lds[0][lane], u = lds[0][lane + 32];
#pragma unroll
  for (int w = 1; w < kFewWaves; ++w) {
    g += lds[w][lane];
    u += lds[w][lane + 32];
  }
  using E = std::conditional_t<std::is_same<T, int8_t>::value, int, float>;
  const E c[4] = {g[0], g[1], g[2], g[3]}, d[4] = {u[0], u[1], u[2], u[3]};
  finish_gated<T, 4>(p, l15, n0 + q * 4, c, d);
}

// Up to 8 rows against one B in blocks of 8 columns: an MFMA operand's slots 8 to 15 are the rows and columns of slots 0
// to 7 again, at later bytes of k, so that C's two diagonal quarters add up to the 8 x 8 outputs.
template <typename T, int U, bool kRagged>
__global__ void __launch_bounds__(kFewWaves* kWave) few_rows_half_kernel(Product p) {
  using Acc = typename Mma<T>::Acc;
  __shared__ Acc lds[kFewWaves][kWave];
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const int l15 = lane & 15, q = lane >> 4;
  const int64_t n0 = static_cast<int64_t>(blockIdx.x) * 8;
  const int64_t col = n0 + (l15 & 7) < p.n ? n0 + (l15 & 7) : p.n - 1, row = (l15 & 7) < p.m ? l15 & 7 : p.m - 1;
  const char* b = p.b0 + col * p.ldb0;
  const char* a = p.a + row * p.lda;
  const int64_t from = (l15 >> 3) * (U * 64) + q * 16;
  Acc acc = Acc{};
  for (int64_t k = wave * (2 * U * 64); k < p.kbytes; k += kFewWaves * 2 * U * 64) {
    const bool last = k + 2 * U * 64 > p.kbytes;
    i32x4 bv[U], av[U];
#pragma unroll
    for (int u = 0; u < U; ++u) bv[u] = load_piece<T, kRagged>(b, k + from + u * 64, p.kbytes, last);
#pragma unroll
    for (int u = 0; u < U; ++u) av[u] = load_piece<T, kRagged>(a, k + from + u * 64, p.kbytes, last);
#pragma unroll
    for (int u = 0; u < U; ++u) acc = Mma<T>::mma(bv[u], av[u], acc);
  }
  lds[wave][lane] = acc;
  __syncthreads();
  if (threadIdx.x >= 32 || l15 >= 8) return;      // lane: row l15, columns 4 q + 0..3; 40 lanes on those of the later k
  Acc sum = lds[0][lane] + lds[0][lane + 40];
#pragma unroll
  for (int w = 1; w < kFewWaves; ++w) sum += lds[w][lane] + lds[w][lane + 40];
  using E = std::conditional_t<std::is_same<T, int8_t>::value, int, float>;
  E c[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) c[e] = sum[e];
  finish<T, 4>(p, l15, n0 + q * 4, c);
}

// ------------------------------------------------------------------------------- launch
inline bool rows16(const void* p, int64_t ld_bytes) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (ld_bytes & 15) == 0 && ld_bytes >= 0;
}
constexpr int64_t kMaxRowBytes = int64_t{1} << 23;     // the tile loads' offsets: 256 rows in 31 bits

// How a product is cut: blocks of 64 rows and 16 columns (tile 0: few_rows_kernel), or tiles of `tile` x `tile`
// (gated: `tile` / 2 columns), k in `slices`.
struct Plan {
  int tile, slices;
  int64_t slice_runs;
  size_t workspace;
};

// The cut with the least estimated time.  The estimate, in microseconds, is fitted to measurements of every cut (slices
// in powers of two, up to 32) at m 24 to 8000 against weights of 256 x 256 to 8192 x 2048 and 2048 x 8192 in 8 bits, bf16
// pairs and fp32 pairs: its choice is 0.4 % slower than the best cut there in the geometric mean, and 18 % at most.  The
// other numbers of slices that it tries (3, 5, 6, 10, 12, 24, and 48 and 64) take the same formula; they were measured on
// a few products only (fp32 training pass 1216 x 615 over 969 177 -> 146 us).
//   few rows: a block's bytes of k at 2.2 us a thousand (more with two Bs), blocks in turns of one a CU;
//   tiles: a step of 128 bytes of k takes a CU 1.5 us at 256 x 256 (1.4 while half of the chip is idle), at
//     128 x 128 0.57 us alone and 1.2 us for the two that share a CU; fp32 is bound by its MFMAs (8, 2.15, 4.4 us);
//   slices: one more launch, and their sums written and read.
inline Plan plan_product(int64_t m, int64_t n, int64_t kbytes, bool gated, bool fp32, bool few) {
  Plan best{0, 1, cdiv(kbytes, 64), 0};
  if (few && m <= 16) return best;
  const int64_t steps = cdiv(kbytes, 128);
  double least = 1e300;
  if (few && m <= 512) {
    const double byte = 0.0022 * (gated ? (fp32 ? 1.9 : 1.4) : 1.0) * (m <= 32 ? 0.61 : 1.0);
    least = 4.1 + cdiv(cdiv(n, 16) * cdiv(m, 64), 256) * kbytes * byte;
  }
  for (int tile : {128, 256}) {
    const int64_t tiles = cdiv(m, tile) * cdiv(n, gated ? tile / 2 : tile);
    for (const int slices : {1, 2, 3, 4, 5, 6, 8, 10, 12, 16, 24, 32, 48, 64}) {
      if (2 * slices > steps + 1) break;
      const int64_t each = cdiv(steps, slices), blocks = tiles * slices;
      if (cdiv(steps, each) != slices) continue;
      double time;
      if (tile == 128) {
        const double alone = fp32 ? 2.15 : blocks <= 128 ? 0.56 : 0.58, pair = fp32 ? 4.4 : 1.2;
        const int64_t turns = blocks / 512, rest = blocks % 512;
        time = each * (turns * pair + (rest == 0 ? 0.0 : rest <= 256 ? alone : pair)) + 7.7 + 2.0 * (turns - (rest == 0 ? 1 : 0));
      } else {
        const int64_t turns = cdiv(blocks, 256);
        time = each * turns * (fp32 ? 8.0 : blocks <= 128 ? 1.4 : 1.5) + 12.0 + 7.5 * (turns - 1);
      }
      const double bytes = static_cast<double>(blocks) * tile * tile * 4;
      if (slices > 1) time += 4.2 + 2.0 * bytes / 7.5e6;
      if (time < least) {
        least = time;
        best = Plan{tile, slices, each * 2, slices > 1 ? static_cast<size_t>(bytes) : 0};
      }
    }
  }
  return best;
}

template <typename T, int kTile, bool kGated, bool kAT, bool kBT>
void launch_tiles(const Product& p, const Plan& plan, int64_t tm, int64_t tn, hipStream_t stream) {
  hipLaunchKernelGGL((tile_kernel<T, kTile, kGated, kAT, kBT>), dim3(static_cast<unsigned>(tm * tn), plan.slices),
                     dim3(TileShape<kTile, kGated>::kThreads), 0, stream, p, static_cast<int>(tm), static_cast<int>(tn));
  if (plan.slices > 1) {
    const int64_t units = tm * tn * (kTile * kTile / (16 * 64));
    hipLaunchKernelGGL((join_kernel<T, kTile, kGated, kBT>), dim3(static_cast<unsigned>(cdiv(units, 4))), dim3(256), 0, stream, p,
                       static_cast<int>(tm), static_cast<int>(tn), plan.slices);
  }
}

template <typename T, bool kGated, bool kAT, bool kBT>
int launch_planned(Product p, const Plan& plan, void* ws, size_t ws_bytes, hipStream_t stream, const char* what) {
  SAGE_REQUIRE(p.lda < kMaxRowBytes && p.ldb0 < kMaxRowBytes && p.ldb1 < kMaxRowBytes, SAGE_ELIMIT, "%s: rows more than %ld bytes apart",
               what, (long)kMaxRowBytes);
  SAGE_REQUIRE(plan.workspace <= ws_bytes && (plan.workspace == 0 || rows16(ws, 0)), SAGE_EWORKSPACE,
               "%s: workspace of %zu bytes, %zu needed", what, ws_bytes, plan.workspace);
  const int64_t tm = cdiv(p.m, plan.tile), tn = cdiv(p.n, kGated ? plan.tile / 2 : plan.tile);
  SAGE_REQUIRE(tm * tn < (int64_t{1} << 23), SAGE_ELIMIT, "%s: %ld output tiles", what, (long)(tm * tn));
  p.slice_runs = plan.slice_runs;
  p.partial = plan.slices > 1 ? static_cast<i32x4*>(ws) : nullptr;
  if (plan.tile == 256) launch_tiles<T, 256, kGated, kAT, kBT>(p, plan, tm, tn, stream);
  else launch_tiles<T, 128, kGated, kAT, kBT>(p, plan, tm, tn, stream);
  SAGE_CHECK_LAUNCH(what);
  return SAGE_OK;
}

template <typename T, bool kGated, bool kRagged>
void launch_few_rows(const Product& p, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>(cdiv(p.n, 16)), static_cast<unsigned>(cdiv(p.m, 64))), threads(kFewWaves * kWave);   // m <= 512
  if constexpr (kGated) {
    // 8 columns a block where the busiest CU then gets fewer of them (bf16, 4 rows: 5632 x 2048 14.6 -> 12.8 us, 1024 x 1024
    // 5.0 -> 4.2, 1000 x 4000 9.7 -> 7.0; 8192 x 2048, where it does not, 16.4 -> 16.7)
    if (p.m <= 16 && cdiv(cdiv(p.n, 8), 256) < 2 * cdiv(cdiv(p.n, 16), 256)) {
      const dim3 eight(static_cast<unsigned>(cdiv(p.n, 8)));
      if (p.kbytes >= kFewWaves * 512) hipLaunchKernelGGL((few_rows_pair_kernel<T, 8, kRagged>), eight, threads, 0, stream, p);
      else hipLaunchKernelGGL((few_rows_pair_kernel<T, 4, kRagged>), eight, threads, 0, stream, p);
      return;
    }
  }
  if constexpr (!kGated) {
    // the same, for up to 8 rows (8 bits, 1 row: 2048 x 8192 8.0 -> 6.5 us, 5120 x 13824 22.0 -> 18.4, 64 x 65536 36.6 -> 19.5)
    if (p.m <= 8 && cdiv(cdiv(p.n, 8), 256) < 2 * cdiv(cdiv(p.n, 16), 256)) {
      const dim3 eight(static_cast<unsigned>(cdiv(p.n, 8)));
      hipLaunchKernelGGL((few_rows_half_kernel<T, 4, kRagged>), eight, threads, 0, stream, p);
      return;
    }
  }
  // 32 columns a block where 17 to 32 rows would otherwise be read for every 16 (8-bit pair of 8192 x 2048 against 24
  // rows 10.9 -> 10.3 us, bf16 pair of 5632 x 2048 against 20 rows 19.1 -> 16.9; more or fewer pieces a turn and 32
  // columns for other row counts measured the same or slower)
  if (p.m <= 16) hipLaunchKernelGGL((few_rows_kernel<T, 1, kGated, 1, kRagged>), grid, threads, 0, stream, p);
  else if (p.m <= 32 && p.n >= 4096)
    hipLaunchKernelGGL((few_rows_kernel<T, 2, kGated, 2, kRagged>), dim3(static_cast<unsigned>(cdiv(p.n, 32))), threads, 0, stream, p);
  else if (p.m <= 32) hipLaunchKernelGGL((few_rows_kernel<T, 2, kGated, 1, kRagged>), grid, threads, 0, stream, p);
  else hipLaunchKernelGGL((few_rows_kernel<T, 4, kGated, 1, kRagged>), grid, threads, 0, stream, p);
}

// rows of both operands along k
template <typename T, bool kGated>
int launch_product(Product p, void* ws, size_t ws_bytes, hipStream_t stream, const char* what) {
  const Plan plan = plan_product(p.m, p.n, p.kbytes, kGated, std::is_same<T, float>::value, true);
  p.runs = cdiv(p.kbytes, 64);
  p.part_runs = p.runs;
  p.whole_runs = p.kbytes / 64;
  if (plan.tile != 0) return launch_planned<T, kGated, false, false>(p, plan, ws, ws_bytes, stream, what);
  SAGE_REQUIRE(p.n < (int64_t{1} << 26), SAGE_ELIMIT, "%s: %ld columns", what, (long)p.n);
  const bool whole = p.kbytes % 16 == 0 && rows16(p.a, p.lda) && rows16(p.b0, p.ldb0) && rows16(p.b1, p.ldb1);
  if (whole) launch_few_rows<T, kGated, false>(p, stream);
  else launch_few_rows<T, kGated, true>(p, stream);
  SAGE_CHECK_LAUNCH(what);
  return SAGE_OK;
}

inline int size_of(int dtype) { return dtype == SAGE_F32 ? 4 : 2; }
inline bool known_dtype(int d) { return d == SAGE_F32 || d == SAGE_BF16 || d == SAGE_F16; }
inline bool known_act(int a) { return a == SAGE_ACT_SILU || a == SAGE_ACT_GELU || a == SAGE_ACT_RELU; }

template <bool kGated>
int product_by_type(const Product& p, int dtype, void* ws, size_t ws_bytes, hipStream_t stream, const char* what) {
  if (dtype == SAGE_F32) return launch_product<float, kGated>(p, ws, ws_bytes, stream, what);
  if (dtype == SAGE_BF16) return launch_product<__bf16, kGated>(p, ws, ws_bytes, stream, what);
  return launch_product<_Float16, kGated>(p, ws, ws_bytes, stream, what);
}

// ------------------------------------------------------------------------------- backward pass
// dg = dh * u * act'(g), du = dh * act(g), each rounded once to the operands' type (the matrix cores take no wider
// one; in fp16 its range too: above 65504 they are infinite, below 3e-8 zero, as a loss scale has to allow for), as the rows [dg, zeros to wide, du, zeros to wide] that both products read: along h for dx, across for the
// weights' gradients.  Bound by HBM: 8 bytes of g and u and one element of dh read, two elements written.
template <typename T, int kAct>
__global__ void __launch_bounds__(256) gate_bwd_kernel(const T* dh, int64_t ld_dh, const float* saved, int64_t m,
                                                       int64_t h, int64_t wide, T* out) {
  constexpr int act = kAct;
  constexpr bool kExact = std::is_same<T, float>::value;
  const int64_t per = wide / 4, total = m * per;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < total; i += static_cast<int64_t>(gridDim.x) * 256) {
    const int64_t row = i / per, col = (i - row * per) * 4;
    float g[4], u[4], d[4];
    if (col + 4 <= h) {
      const Run<4, float> rg = *reinterpret_cast<const Run<4, float>*>(saved + row * h + col);
      const Run<4, float> ru = *reinterpret_cast<const Run<4, float>*>(saved + (m + row) * h + col);
      const Run<4, T> rd = *reinterpret_cast<const Run<4, T>*>(dh + row * ld_dh + col);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        g[e] = rg.v[e];
        u[e] = ru.v[e];
        d[e] = static_cast<float>(rd.v[e]);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const bool in = col + e < h;
        g[e] = in ? saved[row * h + col + e] : 0.f;
        u[e] = in ? saved[(m + row) * h + col + e] : 0.f;
        d[e] = in ? static_cast<float>(dh[row * ld_dh + col + e]) : 0.f;
      }
    }
    Run<4, T> dg, du;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      dg.v[e] = static_cast<T>(d[e] * u[e] * act_slope<kExact>(g[e], act));
      du.v[e] = static_cast<T>(d[e] * act_value<kExact>(g[e], act));
    }
    T* to = out + row * 2 * wide + col;
    *reinterpret_cast<Run<4, T>*>(to) = dg;
    *reinterpret_cast<Run<4, T>*>(to + wide) = du;
  }
}

struct PadArgs {
  const uint8_t* in[3];
  int64_t ld[3];          // bytes
  int64_t first[3];       // output row of the first row
};
// A piece of 16 bytes a thread.  The matrices of a product come in one launch: most are small, and a call's launches cost
// more than the bytes (8 bits, 1411 x 470 over 634: a launch and an output for each 24.0 us a call, one for both 18.7).
__global__ void __launch_bounds__(256) pad_rows_kernel(PadArgs a, int64_t row_bytes, uint8_t* out, int64_t ld_out, int64_t pieces,
                                                       int64_t total) {
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < total; i += static_cast<int64_t>(gridDim.x) * 256) {
    const int64_t row = i / pieces, at = (i - row * pieces) * 16;
    const int of = row >= a.first[2] ? 2 : row >= a.first[1] ? 1 : 0;
    const uint8_t* p = (of == 2 ? a.in[2] : of == 1 ? a.in[1] : a.in[0]) +
                       (row - (of == 2 ? a.first[2] : of == 1 ? a.first[1] : 0)) * (of == 2 ? a.ld[2] : of == 1 ? a.ld[1] : a.ld[0]) + at;
    struct __attribute__((packed, aligned(1))) P {
      uint8_t v[16];
    } k;
    if (at + 16 <= row_bytes) {
      k = *reinterpret_cast<const P*>(p);
    } else {
#pragma unroll
      for (int e = 0; e < 16; ++e) k.v[e] = at + e < row_bytes ? p[e] : 0;
    }
    *reinterpret_cast<i32x4*>(out + row * ld_out + at) = __builtin_bit_cast(i32x4, k);
  }
}

// The backward pass's workspace: [m, 2 wide] of dg and du, and the room for slices, which its two products, one
// after the other, share.
struct BwdLayout {
  int64_t wide;                // h in whole runs
  Plan dx, dw;
  size_t part, part_bytes, bytes;
};
inline BwdLayout bwd_layout(int64_t m, int64_t h, int64_t k, int dtype) {
  const int64_t size = size_of(dtype), each = 64 / size;
  BwdLayout l;
  l.wide = cdiv(h, each) * each;
  l.dx = plan_product(m, k, 2 * l.wide * size, false, dtype == SAGE_F32, false);
  l.dw = plan_product(l.wide + h, k, m * size, false, dtype == SAGE_F32, false);
  l.part = align_up(static_cast<size_t>(m * 2 * l.wide * size), 256);
  l.part_bytes = l.dx.workspace > l.dw.workspace ? l.dx.workspace : l.dw.workspace;
  l.bytes = l.part + l.part_bytes;
  return l;
}

template <typename T>
int gated_bwd(const void* dh, int64_t ld_dh, const void* x, int64_t ld_x, const void* wg, const void* wu, int64_t ld_w,
              const float* saved, int act, int64_t m, int64_t h, int64_t k, int dtype, void* dx, int64_t ld_dx, void* dw,
              char* ws, hipStream_t st, const char* what) {
  const BwdLayout l = bwd_layout(m, h, k, dtype);
  constexpr int64_t kRows = 64 / sizeof(T);
  const int64_t units = cdiv(m * (l.wide / 4), 256);
  const auto gate = act == SAGE_ACT_SILU ? gate_bwd_kernel<T, SAGE_ACT_SILU>
                    : act == SAGE_ACT_GELU ? gate_bwd_kernel<T, SAGE_ACT_GELU> : gate_bwd_kernel<T, SAGE_ACT_RELU>;
  hipLaunchKernelGGL(gate, dim3(static_cast<unsigned>(units < 16384 ? units : 16384)), dim3(256), 0, st,
                     static_cast<const T*>(dh), ld_dh, saved, m, h, l.wide, reinterpret_cast<T*>(ws));
  SAGE_CHECK_LAUNCH(what);
  if (dx != nullptr) {
    // dx[m, k]: k runs over dg's columns against w_gate's rows, then over du's against w_up's
    Product p{};
    p.a = ws; p.lda = 2 * l.wide * sizeof(T);
    p.b0 = static_cast<const char*>(wg); p.b1 = static_cast<const char*>(wu); p.ldb0 = p.ldb1 = ld_w * sizeof(T);
    p.m = m; p.n = k; p.kbytes = 2 * l.wide * sizeof(T); p.depth = h;
    p.part_runs = l.wide / kRows; p.runs = 2 * p.part_runs;
    p.whole_runs = h % kRows == 0 ? p.runs : h / kRows;
    p.out = dx; p.ldo = ld_dx; p.out_dtype = dtype;
    const int rc = launch_planned<T, false, false, true>(p, l.dx, ws + l.part, l.part_bytes, st, what);
    if (rc != SAGE_OK) return rc;
  }
  if (dw != nullptr) {
    // [dw_gate; dw_up]: dg's and du's columns at once; the rows of those between h and wide are not stored, and the
    // last row is du's last column, wide + h - 1
    Product p{};
    p.a = ws; p.lda = 2 * l.wide * sizeof(T);
    p.b0 = static_cast<const char*>(x); p.ldb0 = ld_x * sizeof(T);
    p.m = l.wide + h; p.n = k; p.depth = m; p.fold = l.wide; p.fold_rows = h;
    p.runs = cdiv(m, kRows); p.part_runs = INT64_MAX; p.whole_runs = m / kRows;
    p.out = dw; p.ldo = k; p.out_dtype = dtype;
    return launch_planned<T, false, true, true>(p, l.dw, ws + l.part, l.part_bytes, st, what);
  }
  return SAGE_OK;
}

}  // namespace
}  // namespace sage

using namespace sage;

extern "C" int sage_pad_rows(const void* in0, sage_i64 ld0_bytes, sage_i64 rows0, const void* in1, sage_i64 ld1_bytes, sage_i64 rows1,
                             const void* in2, sage_i64 ld2_bytes, sage_i64 rows2, sage_i64 row_bytes, void* out,
                             sage_i64 ld_out_bytes, void* stream) {
  SAGE_REQUIRE(rows0 >= 0 && rows1 >= 0 && rows2 >= 0 && row_bytes > 0, SAGE_EINVAL, "sage_pad_rows: bad shape [%ld + %ld + %ld, %ld]",
               (long)rows0, (long)rows1, (long)rows2, (long)row_bytes);
  const int64_t rows = rows0 + rows1 + rows2;
  if (rows == 0) return SAGE_OK;
  SAGE_REQUIRE((in0 || rows0 == 0) && (in1 || rows1 == 0) && (in2 || rows2 == 0) && out, SAGE_EINVAL, "sage_pad_rows: NULL pointer");
  SAGE_REQUIRE(rows16(out, ld_out_bytes) && ld_out_bytes >= row_bytes && ld0_bytes >= 0 && ld1_bytes >= 0 && ld2_bytes >= 0, SAGE_EINVAL,
               "sage_pad_rows: output rows start on 16 bytes and hold the input's");
  const PadArgs a = {{static_cast<const uint8_t*>(in0), static_cast<const uint8_t*>(in1), static_cast<const uint8_t*>(in2)},
                     {ld0_bytes, ld1_bytes, ld2_bytes}, {0, rows0, rows0 + rows1}};
  const int64_t pieces = cdiv(row_bytes, 16), total = rows * pieces;
  const int64_t blocks = cdiv(total, 256) < (1 << 20) ? cdiv(total, 256) : 1 << 20;
  hipLaunchKernelGGL(pad_rows_kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, static_cast<hipStream_t>(stream),
                     a, row_bytes, static_cast<uint8_t*>(out), ld_out_bytes, pieces, total);
  SAGE_CHECK_LAUNCH("sage_pad_rows");
  return SAGE_OK;
}

extern "C" int sage_product_any_rows(sage_i64 m, sage_i64 n, sage_i64 row_bytes, int gated, int fp32) {
  return m > 0 && n > 0 && row_bytes >= 16 && plan_product(m, n, row_bytes, gated != 0, fp32 != 0, true).tile == 0;
}

extern "C" size_t sage_product_workspace_bytes(sage_i64 m, sage_i64 n, sage_i64 row_bytes, int gated, int fp32) {
  if (m <= 0 || n <= 0 || row_bytes <= 0) return 0;
  return plan_product(m, n, row_bytes, gated != 0, fp32 != 0, true).workspace;
}

extern "C" int sage_product_cut(sage_i64 m, sage_i64 n, sage_i64 row_bytes, int gated, int fp32, int few_rows, int* tile_host,
                                int* slices_host) {
  SAGE_REQUIRE(m > 0 && n > 0 && row_bytes > 0, SAGE_EINVAL, "sage_product_cut: bad shape m %ld n %ld, rows of %ld bytes", (long)m,
               (long)n, (long)row_bytes);
  SAGE_REQUIRE(tile_host != nullptr && slices_host != nullptr, SAGE_EINVAL, "sage_product_cut: NULL pointer");
  const Plan plan = plan_product(m, n, row_bytes, gated != 0, fp32 != 0, few_rows != 0);
  *tile_host = plan.tile;
  *slices_host = plan.slices;
  return SAGE_OK;
}

#define SAGE_INT8_CHECKS(what)                                                                                          \
  SAGE_REQUIRE(known_dtype(out_dtype), SAGE_EINVAL, what ": unknown output dtype %d", out_dtype);                       \
  SAGE_REQUIRE(m >= 0 && n > 0 && k > 0, SAGE_EINVAL, what ": bad shape m %ld n %ld k %ld", (long)m, (long)n, (long)k); \
  SAGE_REQUIRE(k <= SAGE_INT8_MAX_K, SAGE_ELIMIT, what ": k = %ld: a sum of k products could leave 32 bits", (long)k)

extern "C" int sage_int8_linear(const int8_t* x, sage_i64 ld_x, const float* x_scale, const int8_t* w, sage_i64 ld_w,
                                const float* w_scale, const float* bias, sage_i64 m, sage_i64 n, sage_i64 k, int out_dtype,
                                void* out, sage_i64 ld_out, void* workspace, size_t workspace_bytes, void* stream) {
  SAGE_INT8_CHECKS("sage_int8_linear");
  if (m == 0) return SAGE_OK;
  SAGE_REQUIRE(x && x_scale && w && w_scale && out, SAGE_EINVAL, "sage_int8_linear: NULL pointer");
  SAGE_REQUIRE(((k % 16 == 0 && rows16(x, ld_x) && rows16(w, ld_w)) || sage_product_any_rows(m, n, k, 0, 0)) && ld_x >= 0 &&
                   ld_w >= 0 && ld_out >= n, SAGE_EINVAL, "sage_int8_linear: rows are whole pieces of 16 bytes (sage_pad_rows) and outputs do not overlap");
  Product p{};
  p.a = reinterpret_cast<const char*>(x); p.lda = ld_x;
  p.b0 = reinterpret_cast<const char*>(w); p.ldb0 = ld_w;
  p.m = m; p.n = n; p.kbytes = k;
  p.out = out; p.ldo = ld_out; p.out_dtype = out_dtype;
  p.sa = x_scale; p.sb0 = w_scale; p.bias = bias;
  return launch_product<int8_t, false>(p, workspace, workspace_bytes, static_cast<hipStream_t>(stream), "sage_int8_linear");
}

extern "C" int sage_int8_gated_linear(const int8_t* x, sage_i64 ld_x, const float* x_scale, const int8_t* w_gate, sage_i64 ld_g,
                                      const float* gate_scale, const int8_t* w_up, sage_i64 ld_u, const float* up_scale,
                                      int activation, sage_i64 m, sage_i64 n, sage_i64 k, int out_dtype, void* out,
                                      sage_i64 ld_out, void* workspace, size_t workspace_bytes, void* stream) {
  SAGE_INT8_CHECKS("sage_int8_gated_linear");
  SAGE_REQUIRE(known_act(activation), SAGE_EINVAL, "sage_int8_gated_linear: unknown activation %d", activation);
  if (m == 0) return SAGE_OK;
  SAGE_REQUIRE(x && x_scale && w_gate && gate_scale && w_up && up_scale && out, SAGE_EINVAL, "sage_int8_gated_linear: NULL pointer");
  SAGE_REQUIRE(((k % 16 == 0 && rows16(x, ld_x) && rows16(w_gate, ld_g) && rows16(w_up, ld_u)) || sage_product_any_rows(m, n, k, 1, 0)) &&
                   ld_x >= 0 && ld_g >= 0 && ld_u >= 0 && ld_out >= n, SAGE_EINVAL, "sage_int8_gated_linear: rows are whole pieces of 16 bytes (sage_pad_rows) and outputs do not overlap");
  Product p{};
  p.a = reinterpret_cast<const char*>(x); p.lda = ld_x;
  p.b0 = reinterpret_cast<const char*>(w_gate); p.ldb0 = ld_g;
  p.b1 = reinterpret_cast<const char*>(w_up); p.ldb1 = ld_u;
  p.m = m; p.n = n; p.kbytes = k;
  p.out = out; p.ldo = ld_out; p.out_dtype = out_dtype; p.act = activation;
  p.sa = x_scale; p.sb0 = gate_scale; p.sb1 = up_scale;
  return launch_product<int8_t, true>(p, workspace, workspace_bytes, static_cast<hipStream_t>(stream), "sage_int8_gated_linear");
}

extern "C" int sage_gated_linear_fwd(const void* x, sage_i64 ld_x, const void* w_gate, sage_i64 ld_g, const void* w_up,
                                     sage_i64 ld_u, int activation, sage_i64 m, sage_i64 h, sage_i64 k, int dtype, void* out,
                                     sage_i64 ld_out, float* saved, void* workspace, size_t workspace_bytes, void* stream) {
  SAGE_REQUIRE(known_dtype(dtype), SAGE_EINVAL, "sage_gated_linear_fwd: unknown dtype %d", dtype);
  SAGE_REQUIRE(known_act(activation), SAGE_EINVAL, "sage_gated_linear_fwd: unknown activation %d", activation);
  SAGE_REQUIRE(m >= 0 && h > 0 && k > 0, SAGE_EINVAL, "sage_gated_linear_fwd: bad shape m %ld h %ld k %ld", (long)m, (long)h, (long)k);
  if (m == 0) return SAGE_OK;
  SAGE_REQUIRE(x && w_gate && w_up && out, SAGE_EINVAL, "sage_gated_linear_fwd: NULL pointer");
  const int size = size_of(dtype);
  SAGE_REQUIRE(((k * size % 16 == 0 && rows16(x, ld_x * size) && rows16(w_gate, ld_g * size) && rows16(w_up, ld_u * size)) ||
                sage_product_any_rows(m, h, k * size, 1, dtype == SAGE_F32)) && ld_x >= 0 && ld_g >= 0 && ld_u >= 0 && ld_out >= h,
               SAGE_EINVAL, "sage_gated_linear_fwd: rows are whole pieces of 16 bytes (sage_pad_rows) and outputs do not overlap");
  Product p{};
  p.a = static_cast<const char*>(x); p.lda = ld_x * size;
  p.b0 = static_cast<const char*>(w_gate); p.ldb0 = ld_g * size;
  p.b1 = static_cast<const char*>(w_up); p.ldb1 = ld_u * size;
  p.m = m; p.n = h; p.kbytes = k * size;
  p.out = out; p.ldo = ld_out; p.out_dtype = dtype; p.act = activation; p.saved = saved;
  return product_by_type<true>(p, dtype, workspace, workspace_bytes, static_cast<hipStream_t>(stream), "sage_gated_linear_fwd");
}

extern "C" size_t sage_gated_linear_bwd_workspace_bytes(sage_i64 m, sage_i64 h, sage_i64 k, int dtype) {
  if (m <= 0 || h <= 0 || k <= 0 || !known_dtype(dtype)) return 0;
  return bwd_layout(m, h, k, dtype).bytes;
}

extern "C" int sage_gated_linear_bwd(const void* dh, sage_i64 ld_dh, const void* x, sage_i64 ld_x, const void* w_gate,
                                     sage_i64 ld_g, const void* w_up, sage_i64 ld_u, const float* saved, int activation,
                                     sage_i64 m, sage_i64 h, sage_i64 k, int dtype, void* dx, sage_i64 ld_dx, void* dw,
                                     void* workspace, size_t workspace_bytes, void* stream) {
  SAGE_REQUIRE(known_dtype(dtype), SAGE_EINVAL, "sage_gated_linear_bwd: unknown dtype %d", dtype);
  SAGE_REQUIRE(known_act(activation), SAGE_EINVAL, "sage_gated_linear_bwd: unknown activation %d", activation);
  SAGE_REQUIRE(m > 0 && h > 0 && k > 0, SAGE_EINVAL, "sage_gated_linear_bwd: bad shape m %ld h %ld k %ld", (long)m, (long)h, (long)k);
  SAGE_REQUIRE(dh && x && w_gate && w_up && saved && (dx || dw), SAGE_EINVAL, "sage_gated_linear_bwd: NULL pointer");
  const int64_t size = size_of(dtype), row_bytes = static_cast<int64_t>(align_up(static_cast<size_t>(k * size), 16));
  SAGE_REQUIRE(ld_dh >= 0 && (dx == nullptr || ld_dx >= k), SAGE_EINVAL, "sage_gated_linear_bwd: row stride below the width");
  SAGE_REQUIRE(rows16(x, ld_x * size) && rows16(w_gate, ld_g * size) && rows16(w_up, ld_u * size) && ld_x * size >= row_bytes &&
                   ld_g * size >= row_bytes && ld_g == ld_u,
               SAGE_EINVAL, "sage_gated_linear_bwd: rows are whole pieces of 16 bytes (sage_pad_rows), both weights' strides the same");
  SAGE_REQUIRE(workspace != nullptr && (reinterpret_cast<uintptr_t>(workspace) & 255) == 0 &&
                   workspace_bytes >= sage_gated_linear_bwd_workspace_bytes(m, h, k, dtype),
               SAGE_EWORKSPACE, "sage_gated_linear_bwd: workspace of %zu bytes", workspace_bytes);
  char* ws = static_cast<char*>(workspace);
  hipStream_t st = static_cast<hipStream_t>(stream);
  const char* what = "sage_gated_linear_bwd";
  if (dtype == SAGE_F32)
    return gated_bwd<float>(dh, ld_dh, x, ld_x, w_gate, w_up, ld_g, saved, activation, m, h, k, dtype, dx, ld_dx, dw, ws, st, what);
  if (dtype == SAGE_BF16)
    return gated_bwd<__bf16>(dh, ld_dh, x, ld_x, w_gate, w_up, ld_g, saved, activation, m, h, k, dtype, dx, ld_dx, dw, ws, st, what);
  return gated_bwd<_Float16>(dh, ld_dh, x, ld_x, w_gate, w_up, ld_g, saved, activation, m, h, k, dtype, dx, ld_dx, dw, ws, st, what);
}
