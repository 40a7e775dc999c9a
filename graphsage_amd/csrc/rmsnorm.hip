// Root-mean-square norm with the residual's addition, forward (own type or 8 bits with one scale a
// row) and backward, and the reading back of 8-bit rows.
//
//   s = x + r,  rstd = 1 / sqrt(mean(s^2) + eps),  y = s * rstd * w
//   8 bits:   t = s * w, a = max|t|, q = rint(t * 127 / a), scale = a * rstd / 127
//             (the row's factor rstd cancels in q: 127 t rstd / (a rstd), so q does not wait for it)
//   backward: xh = s * rstd, c = mean(dy * w * xh), dx = rstd * (dy * w - xh * c) + ds,
//             dw = sum over rows of dy * xh
//
// Bound by HBM: every array is read or written once.  A row stays in registers between the
// reduction and the output (kNV vectors of 16 bytes a thread), so there is no second pass over
// memory; rows longer than the registers hold are read twice (the long kernels, the second time
// mostly from L2).  Sums, maxima and rstd are fp32 whatever the type of the rows, and the forward
// pass norms the fp32 sum s; the s that is stored, and that the backward pass reads, is rounded once
// to the rows' type, as a residual stream in that type is.
//
// Measured (a large copy runs at 5.16 TB/s): forward to 8 bits, 8192 x 5120 bf16 with a residual 70 us
// = 4.2 TB/s; forward, 16381 x 2047 bf16 59 us = 4.5 TB/s; its backward pass 64 us = 4.2 TB/s and 7 us
// for dw's join.
//
// Rows start at any address: vectors are loaded and stored with the element's alignment (gfx950
// splits a misaligned 16-byte access itself), so odd widths need no other kernel; a row's last
// partial vector goes element by element.
#include "common.h"

#include <type_traits>

namespace sage {
namespace {

constexpr int kRowBlock = 256;   // threads of a block that holds several rows

template <typename T>
struct VecOf {
  static constexpr int n = 16 / static_cast<int>(sizeof(T));
};

// 16 bytes of T with T's own alignment
template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) Pack {
  T v[VecOf<T>::n];
};

template <typename T>
__device__ inline float to_f(T v) { return static_cast<float>(v); }
template <typename T>
__device__ inline T from_f(float v) { return static_cast<T>(v); }   // round to nearest even

// A vector of a row, zeros behind its end.  The last, partial one is the row's last n elements moved down (one
// load; element by element where the row is shorter than a vector).
template <typename T>
__device__ inline Pack<T> load_pack(const T* p, int64_t at, int64_t dim) {
  constexpr int n = VecOf<T>::n;
  Pack<T> k;
  if (at + n <= dim) {
    k = *reinterpret_cast<const Pack<T>*>(p + at);
  } else if (at < dim && dim >= n) {
    k = *reinterpret_cast<const Pack<T>*>(p + (dim - n));
    unsigned __int128 bits;
    __builtin_memcpy(&bits, &k, 16);
    bits >>= (at + n - dim) * (8 * sizeof(T));
    __builtin_memcpy(&k, &bits, 16);
  } else {
#pragma unroll
    for (int i = 0; i < n; ++i) k.v[i] = at + i < dim ? p[at + i] : static_cast<T>(0.f);
  }
  return k;
}
template <typename T>
__device__ inline void load_vec(const T* p, int64_t at, int64_t dim, float (&v)[VecOf<T>::n]) {
  const Pack<T> k = load_pack<T>(p, at, dim);
#pragma unroll
  for (int i = 0; i < VecOf<T>::n; ++i) v[i] = to_f(k.v[i]);
}

template <typename T>
__device__ inline void store_vec(T* p, int64_t at, int64_t dim, const float (&v)[VecOf<T>::n]) {
  constexpr int n = VecOf<T>::n;
  if (at + n <= dim) {
    Pack<T> k;
#pragma unroll
    for (int i = 0; i < n; ++i) k.v[i] = from_f<T>(v[i]);
    *reinterpret_cast<Pack<T>*>(p + at) = k;
  } else {
#pragma unroll
    for (int i = 0; i < n; ++i)
      if (at + i < dim) p[at + i] = from_f<T>(v[i]);
  }
}

template <int N>
struct __attribute__((packed, aligned(1))) Bytes {
  int8_t v[N];
};

// The norm's weight in the rows' type or in fp32 (w32), or none at all (both NULL: ones)
template <typename T>
__device__ inline void load_weight(const T* w, const float* w32, int64_t at, int64_t dim, float (&v)[VecOf<T>::n]) {
  constexpr int n = VecOf<T>::n;
  if (w != nullptr) {
    load_vec<T>(w, at, dim, v);
  } else if (w32 != nullptr) {
    if (at + n <= dim) {
#pragma unroll
      for (int h = 0; h < n; h += 4) {
        const Pack<float> k = *reinterpret_cast<const Pack<float>*>(w32 + at + h);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[h + i] = k.v[i];
      }
    } else {
#pragma unroll
      for (int i = 0; i < n; ++i) v[i] = at + i < dim ? w32[at + i] : 0.f;
    }
  } else {
#pragma unroll
    for (int i = 0; i < n; ++i) v[i] = 1.f;
  }
}

__device__ inline float wave_add(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}
__device__ inline uint32_t wave_umax(uint32_t v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = max(v, static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), o)));
  return v;
}

// Sum and maximum over the threads of a row (a wave, or the block), given to all of them.  The order of the additions
// is fixed (lanes, then waves in order), so a row's result does not depend on the launch.
template <bool kWaveRow>
__device__ inline void row_reduce(float& sum, uint32_t& top, float* lds_sum, uint32_t* lds_top) {
  sum = wave_add(sum);
  top = wave_umax(top);
  if constexpr (!kWaveRow) {
    const int waves = blockDim.x / kWave;
    const int wave = threadIdx.x / kWave;
    if ((threadIdx.x & (kWave - 1)) == 0) {
      lds_sum[wave] = sum;
      lds_top[wave] = top;
    }
    __syncthreads();
    sum = 0.f;
    top = 0;
    for (int i = 0; i < waves; ++i) {
      sum += lds_sum[i];
      top = max(top, lds_top[i]);
    }
  }
}

// |t| as an unsigned whole number: the order of the magnitudes, infinities above them and NaN above
// all, so that the maximum of a row that holds one is not finite (fmaxf would drop a NaN).
__device__ inline uint32_t magnitude(float t) { return __float_as_uint(t) & 0x7fffffffu; }

// What 8-bit rows are made with: q = rint(t * lift * inv), value = q * scale
struct RowScale {
  float lift, inv, scale;
};
__device__ inline RowScale row_scale(uint32_t top_bits, float rstd) {
  const float top = __uint_as_float(top_bits);
  RowScale r;
  if (top_bits >= 0x7f800000u || !(rstd == rstd)) {   // an infinity or NaN in the row: all of it is NaN
    r.lift = r.inv = 0.f;
    r.scale = __uint_as_float(0x7fc00000u);
  } else if (top_bits == 0) {
    r.lift = r.inv = r.scale = 0.f;
  } else {
    // 127 / top overflows below 2^-121: such rows are lifted by 2^64 first, which is exact
    r.lift = top < 1e-30f ? 18446744073709551616.f : 1.f;
    r.inv = 127.f / (top * r.lift);
    r.scale = top * rstd / 127.f;
  }
  return r;
}
__device__ inline int8_t to_q(float t, const RowScale& s) {
  const float v = rintf(t * s.lift * s.inv);
  return s.lift == 0.f ? static_cast<int8_t>(0) : static_cast<int8_t>(static_cast<int>(v));
}

struct NormArgs {
  const void* x;
  const void* r;
  const void* w;        // weight in the rows' type
  const float* w32;     // or in fp32
  void* y;
  void* sum;
  int8_t* q;
  float* scale;
  int64_t ld_x, ld_r, ld_y, ld_sum, ld_q;
  int64_t rows, dim;
  int64_t q_cols;       // columns of q written: dim, or more with zeros behind it
  float eps;
  int normalise;        // 0: rstd = 1 (quantisation alone)
};

// Which of a launch's blocks this is: their number may pass what one dimension of a grid takes (2^32 threads).
inline dim3 block_grid(int64_t blocks) {
  const int64_t x = blocks < (1 << 20) ? blocks : 1 << 20;
  return dim3(static_cast<unsigned>(x), static_cast<unsigned>(cdiv(blocks, x)));
}
__device__ inline int64_t block_index() { return static_cast<int64_t>(blockIdx.y) * gridDim.x + blockIdx.x; }

// A row to a wave (four rows a block) or to the block; kNV vectors of 16 bytes a thread hold it.
template <typename T, bool kInt8, bool kWaveRow, int kNV>
__global__ void __launch_bounds__(kWaveRow ? kRowBlock : 1024) rms_norm_kernel(NormArgs a) {
  constexpr int n = VecOf<T>::n;
  __shared__ float lds_sum[16];
  __shared__ uint32_t lds_top[16];
  const int threads = kWaveRow ? kWave : blockDim.x;       // of a row
  const int t = kWaveRow ? threadIdx.x % kWave : threadIdx.x;
  const int64_t row = kWaveRow ? block_index() * (kRowBlock / kWave) + threadIdx.x / kWave : block_index();
  if (row >= a.rows) return;     // whole waves, and never part of a block that meets at a barrier
  const T* x = static_cast<const T*>(a.x) + row * a.ld_x;
  const T* r = a.r ? static_cast<const T*>(a.r) + row * a.ld_r : nullptr;
  float s[kNV][n];
  float w[kNV][n];
  float ss = 0.f;
  uint32_t top = 0;
  {
    Pack<T> px[kNV], pr[kNV];     // all of a row's loads before the first use
#pragma unroll
    for (int j = 0; j < kNV; ++j) px[j] = load_pack<T>(x, static_cast<int64_t>(j * threads + t) * n, a.dim);
    if (r != nullptr) {
#pragma unroll
      for (int j = 0; j < kNV; ++j) pr[j] = load_pack<T>(r, static_cast<int64_t>(j * threads + t) * n, a.dim);
    }
#pragma unroll
    for (int j = 0; j < kNV; ++j)
      load_weight<T>(static_cast<const T*>(a.w), a.w32, static_cast<int64_t>(j * threads + t) * n, a.dim, w[j]);
#pragma unroll
    for (int j = 0; j < kNV; ++j)
#pragma unroll
      for (int i = 0; i < n; ++i) s[j][i] = r != nullptr ? to_f(px[j].v[i]) + to_f(pr[j].v[i]) : to_f(px[j].v[i]);
  }
#pragma unroll
  for (int j = 0; j < kNV; ++j) {
#pragma unroll
    for (int i = 0; i < n; ++i) {
      ss += s[j][i] * s[j][i];
      if constexpr (kInt8) top = max(top, magnitude(s[j][i] * w[j][i]));
    }
  }
  if (a.sum != nullptr) {
    T* out = static_cast<T*>(a.sum) + row * a.ld_sum;
#pragma unroll
    for (int j = 0; j < kNV; ++j) store_vec<T>(out, static_cast<int64_t>(j * threads + t) * n, a.dim, s[j]);
  }
  row_reduce<kWaveRow>(ss, top, lds_sum, lds_top);
  const float rstd = a.normalise ? 1.f / sqrtf(ss / static_cast<float>(a.dim) + a.eps) : 1.f;
  if constexpr (kInt8) {
    const RowScale k = row_scale(top, rstd);
    if (t == 0) a.scale[row] = k.scale;
    int8_t* q = a.q + row * a.ld_q;
#pragma unroll
    for (int j = 0; j < kNV; ++j) {
      const int64_t at = static_cast<int64_t>(j * threads + t) * n;
      Bytes<n> o;
#pragma unroll
      for (int i = 0; i < n; ++i) o.v[i] = to_q(s[j][i] * w[j][i], k);
      if (at + n <= a.q_cols) {
        *reinterpret_cast<Bytes<n>*>(q + at) = o;
      } else {
#pragma unroll
        for (int i = 0; i < n; ++i)
          if (at + i < a.q_cols) q[at + i] = o.v[i];
      }
    }
  } else {
    T* y = static_cast<T*>(a.y) + row * a.ld_y;
#pragma unroll
    for (int j = 0; j < kNV; ++j) {
      float o[n];
#pragma unroll
      for (int i = 0; i < n; ++i) o[i] = s[j][i] * rstd * w[j][i];
      store_vec<T>(y, static_cast<int64_t>(j * threads + t) * n, a.dim, o);
    }
  }
}

// Rows longer than the registers hold: 1024 threads go over the row twice.
template <typename T, bool kInt8>
__global__ void __launch_bounds__(1024) rms_norm_long_kernel(NormArgs a) {
  constexpr int n = VecOf<T>::n;
  __shared__ float lds_sum[16];
  __shared__ uint32_t lds_top[16];
  const int64_t row = block_index();
  if (row >= a.rows) return;
  const T* x = static_cast<const T*>(a.x) + row * a.ld_x;
  const T* r = a.r ? static_cast<const T*>(a.r) + row * a.ld_r : nullptr;
  float ss = 0.f;
  uint32_t top = 0;
  float s[n], b[n], w[n];
  auto sum_at = [&](int64_t at) {
    load_vec<T>(x, at, a.dim, s);
    if (r != nullptr) {
      load_vec<T>(r, at, a.dim, b);
#pragma unroll
      for (int i = 0; i < n; ++i) s[i] += b[i];
    }
  };
  for (int64_t at = static_cast<int64_t>(threadIdx.x) * n; at < a.dim; at += 1024 * n) {
    sum_at(at);
    if constexpr (kInt8) load_weight<T>(static_cast<const T*>(a.w), a.w32, at, a.dim, w);
#pragma unroll
    for (int i = 0; i < n; ++i) {
      ss += s[i] * s[i];
      if constexpr (kInt8) top = max(top, magnitude(s[i] * w[i]));
    }
  }
  row_reduce<false>(ss, top, lds_sum, lds_top);
  const float rstd = a.normalise ? 1.f / sqrtf(ss / static_cast<float>(a.dim) + a.eps) : 1.f;
  RowScale k{};
  if constexpr (kInt8) {
    k = row_scale(top, rstd);
    if (threadIdx.x == 0) a.scale[row] = k.scale;
  }
  for (int64_t at = static_cast<int64_t>(threadIdx.x) * n; at < (kInt8 ? a.q_cols : a.dim); at += 1024 * n) {
    sum_at(at);
    load_weight<T>(static_cast<const T*>(a.w), a.w32, at, a.dim, w);
    if (a.sum != nullptr) store_vec<T>(static_cast<T*>(a.sum) + row * a.ld_sum, at, a.dim, s);
    if constexpr (kInt8) {
#pragma unroll
      for (int i = 0; i < n; ++i)
        if (at + i < a.q_cols) a.q[row * a.ld_q + at + i] = to_q(s[i] * w[i], k);
    } else {
#pragma unroll
      for (int i = 0; i < n; ++i) s[i] = s[i] * rstd * w[i];
      store_vec<T>(static_cast<T*>(a.y) + row * a.ld_y, at, a.dim, s);
    }
  }
}

struct NormBwdArgs {
  const void* dy;
  const void* s;
  const void* w;
  const float* w32;
  const void* ds;
  void* dx;
  float* part;          // [blocks, dim] column sums of dy * xh, or NULL
  int64_t ld_dy, ld_s, ld_ds, ld_dx;
  int64_t rows, dim;
  float eps;
};

// A block goes over rows r, r + step, ...; dw's column sums stay in registers until its last row and are
// written once, as the block's partial row (dweight_sum_kernel adds those in a fixed order).  The next
// row's three inputs are under way while a row is computed, and they and the weight are kept in their own type
// and widened where they are used: with the widened values kept as well a wave of 4 vectors a lane needs 241
// registers, and half as many waves fit a CU.
template <typename T>
__device__ inline void narrow(Pack<T>& p) {
  uint32_t w[4];
  __builtin_memcpy(w, &p, 16);
  asm volatile("" : "+v"(w[0]), "+v"(w[1]), "+v"(w[2]), "+v"(w[3]));   // what was widened from it is not kept
  __builtin_memcpy(&p, w, 16);
}

template <typename T, typename W, bool kWaveRow, int kNV>
__global__ void __launch_bounds__(kWaveRow ? kRowBlock : 1024, 4) rms_norm_bwd_kernel(NormBwdArgs a) {
  constexpr int n = VecOf<T>::n;
  constexpr int kRows = kWaveRow ? kRowBlock / kWave : 1;
  const int threads = kWaveRow ? kWave : blockDim.x, waves = blockDim.x / kWave;
  __shared__ float lds_a[2][16];
  __shared__ float lds_b[2][16];
  const int t = kWaveRow ? threadIdx.x % kWave : threadIdx.x;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kRows;
  constexpr int nw = VecOf<W>::n, kW = n / nw;         // an fp32 weight of 16-bit rows is two vectors
  Pack<W> w[kNV][kW];
  float acc[kNV][n];
  // a lane's vectors begin at `at`; the row's last is its last n elements, of which the first `skip` are the lane
  // before's as well: both store the same dx there, one counts them (vectors behind the row: skip = n)
  int64_t at[kNV];
  int skip[kNV];
#pragma unroll
  for (int j = 0; j < kNV; ++j) {
    at[j] = static_cast<int64_t>(j * threads + t) * n;
    const int64_t over = at[j] + n - a.dim;
    skip[j] = over <= 0 ? 0 : over < n ? static_cast<int>(over) : n;
    if (skip[j] > 0) at[j] = a.dim - n;
  }
  const W* wp = std::is_same<T, W>::value ? static_cast<const W*>(a.w) : reinterpret_cast<const W*>(a.w32);
#pragma unroll
  for (int j = 0; j < kNV; ++j) {
#pragma unroll
    for (int h = 0; h < kW; ++h) w[j][h] = *reinterpret_cast<const Pack<W>*>(wp + at[j] + h * nw);
#pragma unroll
    for (int i = 0; i < n; ++i) acc[j][i] = 0.f;
  }
  auto weight = [&](int j, int i) { return to_f(w[j][i / nw].v[i % nw]); };
  int flip = 0;
  Pack<T> s[kNV], g[kNV], d[kNV], s_next[kNV], g_next[kNV], d_next[kNV];
  auto load_row = [&](int64_t row) {
    const T* sp = static_cast<const T*>(a.s) + row * a.ld_s;
    const T* yp = static_cast<const T*>(a.dy) + row * a.ld_dy;
#pragma unroll
    for (int j = 0; j < kNV; ++j) {
      if (skip[j] == n) continue;
      s_next[j] = *reinterpret_cast<const Pack<T>*>(sp + at[j]);
      g_next[j] = *reinterpret_cast<const Pack<T>*>(yp + at[j]);
    }
    if (a.ds != nullptr) {
      const T* dsp = static_cast<const T*>(a.ds) + row * a.ld_ds;
#pragma unroll
      for (int j = 0; j < kNV; ++j)
        if (skip[j] < n) d_next[j] = *reinterpret_cast<const Pack<T>*>(dsp + at[j]);
    }
  };
  int64_t row = kWaveRow ? static_cast<int64_t>(blockIdx.x) * kRows + threadIdx.x / kWave : blockIdx.x;
  constexpr bool kAhead = kNV == 1;     // two rows of two vectors a thread would not fit the registers
  if (kAhead && row < a.rows) load_row(row);
  for (; row < a.rows; row += step) {
    if (!kAhead) load_row(row);
#pragma unroll
    for (int j = 0; j < kNV; ++j) {
      s[j] = s_next[j];
      g[j] = g_next[j];
      d[j] = d_next[j];
    }
    if (kAhead && row + step < a.rows) load_row(row + step);      // under way while this row is computed
    float ss = 0.f, dot = 0.f;
#pragma unroll
    for (int j = 0; j < kNV; ++j) {
#pragma unroll
      for (int i = 0; i < n; ++i) {
        const float v = i < skip[j] ? 0.f : to_f(s[j].v[i]);
        ss += v * v;
        dot += i < skip[j] ? 0.f : to_f(g[j].v[i]) * weight(j, i) * v;
      }
    }
#pragma unroll
    for (int j = 0; j < kNV; ++j) {
      narrow(s[j]);
      narrow(g[j]);
#pragma unroll
      for (int h = 0; h < kW; ++h) narrow(w[j][h]);
    }
    ss = wave_add(ss);
    dot = wave_add(dot);
    if constexpr (!kWaveRow) {
      // two sets of slots in turn: a wave that is a row ahead writes the other one
      const int wave = threadIdx.x / kWave;
      if ((threadIdx.x & (kWave - 1)) == 0) {
        lds_a[flip][wave] = ss;
        lds_b[flip][wave] = dot;
      }
      __syncthreads();
      ss = 0.f;
      dot = 0.f;
      for (int i = 0; i < waves; ++i) {
        ss += lds_a[flip][i];
        dot += lds_b[flip][i];
      }
      flip ^= 1;
    }
    const float rstd = 1.f / sqrtf(ss / static_cast<float>(a.dim) + a.eps);
    const float c = dot * rstd / static_cast<float>(a.dim);          // mean(dy * w * xh)
    T* dxp = static_cast<T*>(a.dx) + row * a.ld_dx;
#pragma unroll
    for (int j = 0; j < kNV; ++j) {
      float o[n];
#pragma unroll
      for (int i = 0; i < n; ++i) {
        const float xh = to_f(s[j].v[i]) * rstd, gy = to_f(g[j].v[i]);
        acc[j][i] += gy * xh;
        o[i] = rstd * (gy * weight(j, i) - xh * c) + (a.ds != nullptr ? to_f(d[j].v[i]) : 0.f);
      }
      if (a.dx != nullptr && skip[j] < n) store_vec<T>(dxp, at[j], a.dim, o);
    }
  }
  if (a.part == nullptr) return;
  float* part = a.part + static_cast<int64_t>(blockIdx.x) * a.dim;
  if constexpr (kRows > 1) {
    // the block's rows' sums, added in wave order
    __shared__ float lds[kWave * kNV * n];
    for (int wave = 0; wave < kRows; ++wave) {
      if (static_cast<int>(threadIdx.x) / kWave == wave) {
#pragma unroll
        for (int j = 0; j < kNV; ++j)
#pragma unroll
          for (int i = 0; i < n; ++i) {
            float* to = lds + (j * n + i) * kWave + t;
            *to = (wave == 0 ? 0.f : *to) + acc[j][i];
          }
      }
      __syncthreads();
    }
    for (int e = threadIdx.x; e < kWave * kNV * n; e += kRowBlock) {
      const int place = e / n, over = static_cast<int>((place + 1) * n - a.dim);       // > 0 for the row's last vector
      if (e < a.dim) part[e] = lds[(place / kWave * n + e % n + (over > 0 ? over : 0)) * kWave + place % kWave];
    }
  } else {
#pragma unroll
    for (int j = 0; j < kNV; ++j) {
#pragma unroll
      for (int i = 0; i < n; ++i)
        if (i >= skip[j]) part[at[j] + i] = acc[j][i];
    }
  }
}

// Long rows: three passes over the row (statistics, dx, and dw's share into the block's partial row).
template <typename T>
__global__ void __launch_bounds__(1024) rms_norm_bwd_long_kernel(NormBwdArgs a) {
  constexpr int n = VecOf<T>::n;
  __shared__ float lds_a[16];
  __shared__ float lds_b[16];
  float* part = a.part ? a.part + static_cast<int64_t>(blockIdx.x) * a.dim : nullptr;
  bool first = true;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* sp = static_cast<const T*>(a.s) + row * a.ld_s;
    const T* yp = static_cast<const T*>(a.dy) + row * a.ld_dy;
    const T* dsp = a.ds ? static_cast<const T*>(a.ds) + row * a.ld_ds : nullptr;
    float ss = 0.f, dot = 0.f;
    float s[n], g[n], w[n], o[n];
    for (int64_t at = static_cast<int64_t>(threadIdx.x) * n; at < a.dim; at += 1024 * n) {
      load_vec<T>(sp, at, a.dim, s);
      load_vec<T>(yp, at, a.dim, g);
      load_weight<T>(static_cast<const T*>(a.w), a.w32, at, a.dim, w);
#pragma unroll
      for (int i = 0; i < n; ++i) {
        ss += s[i] * s[i];
        dot += g[i] * w[i] * s[i];
      }
    }
    ss = wave_add(ss);
    dot = wave_add(dot);
    __syncthreads();          // the row before has read its sums
    if ((threadIdx.x & (kWave - 1)) == 0) {
      lds_a[threadIdx.x / kWave] = ss;
      lds_b[threadIdx.x / kWave] = dot;
    }
    __syncthreads();
    ss = 0.f;
    dot = 0.f;
    for (int i = 0; i < 16; ++i) {
      ss += lds_a[i];
      dot += lds_b[i];
    }
    const float rstd = 1.f / sqrtf(ss / static_cast<float>(a.dim) + a.eps);
    const float c = dot * rstd / static_cast<float>(a.dim);
    for (int64_t at = static_cast<int64_t>(threadIdx.x) * n; at < a.dim; at += 1024 * n) {
      load_vec<T>(sp, at, a.dim, s);
      load_vec<T>(yp, at, a.dim, g);
      load_weight<T>(static_cast<const T*>(a.w), a.w32, at, a.dim, w);
      if (dsp != nullptr) {
        load_vec<T>(dsp, at, a.dim, o);
      } else {
#pragma unroll
        for (int i = 0; i < n; ++i) o[i] = 0.f;
      }
#pragma unroll
      for (int i = 0; i < n; ++i) {
        const float xh = s[i] * rstd;
        o[i] += rstd * (g[i] * w[i] - xh * c);
        if (part != nullptr && at + i < a.dim)      // the same thread owns these columns in every row
          part[at + i] = (first ? 0.f : part[at + i]) + g[i] * xh;
      }
      if (a.dx != nullptr) store_vec<T>(static_cast<T*>(a.dx) + row * a.ld_dx, at, a.dim, o);
    }
    first = false;
  }
}

// dw[c] = sum of the partial rows: 64 threads a column take every 64th of them, then one adds the 64 in order.
template <typename T>
__global__ void __launch_bounds__(1024) dweight_sum_kernel(const float* part, int64_t parts, int64_t dim, T* dw) {
  __shared__ float lds[64][17];
  const int c = threadIdx.x & 15, g = threadIdx.x >> 4;
  const int64_t col = static_cast<int64_t>(blockIdx.x) * 16 + c;
  float v = 0.f;
  if (col < dim) {
#pragma unroll 8
    for (int64_t p = g; p < parts; p += 64) v += part[p * dim + col];
  }
  lds[g][c] = v;
  __syncthreads();
  if (g == 0 && col < dim) {
    v = 0.f;
#pragma unroll
    for (int i = 0; i < 64; ++i) v += lds[i][c];
    dw[col] = from_f<T>(v);
  }
}

template <typename T>
__global__ void __launch_bounds__(256) dequantize_kernel(const int8_t* q, int64_t ld_q, const float* scale, int64_t rows,
                                                         int64_t dim, T* out, int64_t ld_out) {
  constexpr int n = 8;
  const int64_t per = (dim + n - 1) / n;
  const int64_t total = rows * per;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < total; i += static_cast<int64_t>(gridDim.x) * 256) {
    const int64_t row = i / per, at = (i - row * per) * n;
    const float s = scale[row];
    const int8_t* p = q + row * ld_q + at;
    T* o = out + row * ld_out + at;
    if (at + n <= dim) {
      const Bytes<n> b = *reinterpret_cast<const Bytes<n>*>(p);
      struct __attribute__((packed, aligned(sizeof(T)))) Out {
        T v[n];
      } k;
#pragma unroll
      for (int e = 0; e < n; ++e) k.v[e] = from_f<T>(static_cast<float>(b.v[e]) * s);
      *reinterpret_cast<Out*>(o) = k;
    } else {
      for (int e = 0; at + e < dim; ++e) o[e] = from_f<T>(static_cast<float>(p[e]) * s);
    }
  }
}

// How a row of v vectors is split: a wave (four rows a block) or a block of `threads` to a row, and vectors a
// thread; no vectors: longer than the registers hold.
struct RowShape {
  int threads, vectors;
  bool wave;
};
inline RowShape block_row(int64_t v, int vectors) {
  return {static_cast<int>(cdiv(v, kWave * vectors)) * kWave, vectors, false};
}
// With many rows a wave takes a row of up to 256 vectors alone: no barrier, and 4 KB of each input under way
// a wave.  With few (fewer than the chip's waves) a row's latency counts: one vector a thread.
inline RowShape row_shape(int64_t dim, int n, int64_t rows) {
  const int64_t v = cdiv(dim, n);
  if (v <= (rows >= 2048 ? 256 : 64)) return {kWave, static_cast<int>(cdiv(v, 64)), true};
  if (v <= 1024 && rows < 2048) return block_row(v, 1);
  if (v <= 2048) return block_row(v, 2);
  if (v <= 4096) return block_row(v, 4);
  return {1024, 0, false};
}
template <typename F>
inline bool with_row_shape(const RowShape& s, F&& f) {
  using std::integral_constant;
#define SAGE_SHAPE(WAVE, NV) \
  if (s.wave == WAVE && s.vectors == NV) { f(integral_constant<bool, WAVE>{}, integral_constant<int, NV>{}); return true; }
  SAGE_SHAPE(true, 1) SAGE_SHAPE(true, 2) SAGE_SHAPE(true, 3) SAGE_SHAPE(true, 4)
  SAGE_SHAPE(false, 1) SAGE_SHAPE(false, 2) SAGE_SHAPE(false, 4)
#undef SAGE_SHAPE
  return false;
}

template <typename T, bool kInt8>
void launch_norm(const NormArgs& a, hipStream_t stream) {
  const RowShape shape = row_shape(kInt8 ? a.q_cols : a.dim, VecOf<T>::n, a.rows);
  const bool held = with_row_shape(shape, [&](auto wave, auto nv) {
    constexpr bool kWaveRow = decltype(wave)::value;
    const dim3 grid = block_grid(kWaveRow ? cdiv(a.rows, kRowBlock / kWave) : a.rows);
    hipLaunchKernelGGL((rms_norm_kernel<T, kInt8, kWaveRow, decltype(nv)::value>), grid,
                       dim3(kWaveRow ? kRowBlock : shape.threads), 0, stream, a);
  });
  if (!held)
    hipLaunchKernelGGL((rms_norm_long_kernel<T, kInt8>), block_grid(a.rows), dim3(1024), 0, stream, a);
}

template <bool kInt8>
int norm_by_type(const NormArgs& a, int dtype, hipStream_t stream, const char* what) {
  if (dtype == SAGE_F32) launch_norm<float, kInt8>(a, stream);
  else if (dtype == SAGE_BF16) launch_norm<__bf16, kInt8>(a, stream);
  else launch_norm<_Float16, kInt8>(a, stream);
  SAGE_CHECK_LAUNCH(what);
  return SAGE_OK;
}

// The backward pass: one vector a thread with the next row's under way (16381 x 2047 bf16, all of it: four vectors
// a lane of a wave 90 us; with the next row under way as well they leave one wave a SIMD, 147; two vectors
// a thread 102, their registers spill), two where a block is too short; rows of over 2048 vectors go through the
// long kernel.  As many blocks as run at once (20 waves a CU in 16 bits, 32 in fp32), so that none is left over.
inline RowShape bwd_shape(int64_t dim, int dtype) {
  const int n = dtype == SAGE_F32 ? 4 : 8;
  const int64_t v = cdiv(dim, n);
  if (dim < n) return {1024, 0, false};
  if (v <= 64) return {kWave, 1, true};
  if (v <= 1024) return block_row(v, 1);
  if (v <= 2048) return block_row(v, 2);
  return {1024, 0, false};
}
inline int64_t bwd_blocks(int64_t rows, int64_t dim, int dtype) {
  const RowShape s = bwd_shape(dim, dtype);
  const int64_t blocks = s.wave ? cdiv(rows, kRowBlock / kWave) : rows;
  const int64_t most = 256 * ((dtype == SAGE_F32 ? 32 : 20) / (s.wave ? kRowBlock / kWave : s.threads / kWave));
  return blocks < most ? blocks : most;
}

template <typename T>
void launch_norm_bwd(const NormBwdArgs& a, int dtype, hipStream_t stream) {
  const unsigned blocks = static_cast<unsigned>(bwd_blocks(a.rows, a.dim, dtype));
  const RowShape shape = bwd_shape(a.dim, dtype);
  const bool held = with_row_shape(shape, [&](auto wave, auto nv) {
    constexpr bool kWaveRow = decltype(wave)::value;
    constexpr int kNV = decltype(nv)::value;
    const dim3 threads(kWaveRow ? kRowBlock : shape.threads);
    if constexpr (kNV == 1 || (kNV == 2 && !kWaveRow)) {
      if (a.w32 == nullptr)
        hipLaunchKernelGGL((rms_norm_bwd_kernel<T, T, kWaveRow, kNV>), dim3(blocks), threads, 0, stream, a);
      else if constexpr (!std::is_same<T, float>::value)
        hipLaunchKernelGGL((rms_norm_bwd_kernel<T, float, kWaveRow, kNV>), dim3(blocks), threads, 0, stream, a);
    }
  });
  if (!held) hipLaunchKernelGGL((rms_norm_bwd_long_kernel<T>), dim3(blocks), dim3(1024), 0, stream, a);
}

inline bool known_dtype(int d) { return d == SAGE_F32 || d == SAGE_BF16 || d == SAGE_F16; }

}  // namespace
}  // namespace sage

using namespace sage;

extern "C" int sage_rms_norm_fwd(const void* x, sage_i64 ld_x, const void* residual, sage_i64 ld_r, const void* weight,
                                 int weight_dtype, sage_i64 rows, sage_i64 dim, int dtype, float eps, void* y,
                                 sage_i64 ld_y, void* sum, sage_i64 ld_sum, void* stream) {
  SAGE_REQUIRE(known_dtype(dtype), SAGE_EINVAL, "sage_rms_norm_fwd: unknown dtype %d", dtype);
  SAGE_REQUIRE(rows >= 0 && dim > 0, SAGE_EINVAL, "sage_rms_norm_fwd: bad shape [%ld, %ld]", (long)rows, (long)dim);
  SAGE_REQUIRE(rows < (int64_t{1} << 31), SAGE_ELIMIT, "sage_rms_norm_fwd: %ld rows", (long)rows);
  SAGE_REQUIRE(weight_dtype == dtype || weight_dtype == SAGE_F32, SAGE_EINVAL,
               "sage_rms_norm_fwd: the weight is in the rows' type or in fp32");
  if (rows == 0) return SAGE_OK;
  SAGE_REQUIRE(x != nullptr && weight != nullptr && y != nullptr, SAGE_EINVAL, "sage_rms_norm_fwd: NULL pointer");
  SAGE_REQUIRE(ld_y >= dim && (sum == nullptr || ld_sum >= dim) && ld_x >= 0 && ld_r >= 0, SAGE_EINVAL,
               "sage_rms_norm_fwd: row stride below the width");
  NormArgs a{};
  a.x = x; a.r = residual; a.y = y; a.sum = sum;
  if (weight_dtype == dtype) a.w = weight; else a.w32 = static_cast<const float*>(weight);
  a.ld_x = ld_x; a.ld_r = ld_r; a.ld_y = ld_y; a.ld_sum = ld_sum;
  a.rows = rows; a.dim = dim; a.eps = eps; a.normalise = 1;
  return norm_by_type<false>(a, dtype, static_cast<hipStream_t>(stream), "sage_rms_norm_fwd");
}

extern "C" int sage_rms_norm_int8(const void* x, sage_i64 ld_x, const void* residual, sage_i64 ld_r, const void* weight,
                                  int weight_dtype, sage_i64 rows, sage_i64 dim, int dtype, float eps, int normalise,
                                  int8_t* q, sage_i64 ld_q, sage_i64 q_cols, float* scale, void* sum, sage_i64 ld_sum,
                                  void* stream) {
  SAGE_REQUIRE(known_dtype(dtype), SAGE_EINVAL, "sage_rms_norm_int8: unknown dtype %d", dtype);
  SAGE_REQUIRE(rows >= 0 && dim > 0, SAGE_EINVAL, "sage_rms_norm_int8: bad shape [%ld, %ld]", (long)rows, (long)dim);
  SAGE_REQUIRE(rows < (int64_t{1} << 31), SAGE_ELIMIT, "sage_rms_norm_int8: %ld rows", (long)rows);
  SAGE_REQUIRE(weight_dtype == dtype || weight_dtype == SAGE_F32, SAGE_EINVAL,
               "sage_rms_norm_int8: the weight is in the rows' type or in fp32");
  if (rows == 0) return SAGE_OK;
  SAGE_REQUIRE(x != nullptr && q != nullptr && scale != nullptr, SAGE_EINVAL, "sage_rms_norm_int8: NULL pointer");
  SAGE_REQUIRE(q_cols >= dim && ld_q >= q_cols && (sum == nullptr || ld_sum >= dim) && ld_x >= 0 && ld_r >= 0, SAGE_EINVAL,
               "sage_rms_norm_int8: row stride below the width");
  NormArgs a{};
  a.x = x; a.r = residual; a.sum = sum; a.q = q; a.scale = scale;
  if (weight_dtype == dtype) a.w = weight; else a.w32 = static_cast<const float*>(weight);
  a.ld_x = ld_x; a.ld_r = ld_r; a.ld_q = ld_q; a.q_cols = q_cols; a.ld_sum = ld_sum;
  a.rows = rows; a.dim = dim; a.eps = eps; a.normalise = normalise;
  return norm_by_type<true>(a, dtype, static_cast<hipStream_t>(stream), "sage_rms_norm_int8");
}

extern "C" int sage_dequantize_rows(const int8_t* q, sage_i64 ld_q, const float* scale, sage_i64 rows, sage_i64 dim,
                                    int dtype, void* out, sage_i64 ld_out, void* stream) {
  SAGE_REQUIRE(known_dtype(dtype), SAGE_EINVAL, "sage_dequantize_rows: unknown dtype %d", dtype);
  SAGE_REQUIRE(rows >= 0 && dim > 0, SAGE_EINVAL, "sage_dequantize_rows: bad shape [%ld, %ld]", (long)rows, (long)dim);
  if (rows == 0) return SAGE_OK;
  SAGE_REQUIRE(q != nullptr && scale != nullptr && out != nullptr, SAGE_EINVAL, "sage_dequantize_rows: NULL pointer");
  SAGE_REQUIRE(ld_out >= dim && ld_q >= 0, SAGE_EINVAL, "sage_dequantize_rows: row stride below the width");
  const int64_t want = cdiv(rows * cdiv(dim, 8), 256);
  const dim3 grid(static_cast<unsigned>(want < 8192 ? want : 8192));
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == SAGE_F32)
    hipLaunchKernelGGL((dequantize_kernel<float>), grid, dim3(256), 0, st, q, ld_q, scale, rows, dim, static_cast<float*>(out), ld_out);
  else if (dtype == SAGE_BF16)
    hipLaunchKernelGGL((dequantize_kernel<__bf16>), grid, dim3(256), 0, st, q, ld_q, scale, rows, dim, static_cast<__bf16*>(out), ld_out);
  else
    hipLaunchKernelGGL((dequantize_kernel<_Float16>), grid, dim3(256), 0, st, q, ld_q, scale, rows, dim, static_cast<_Float16*>(out), ld_out);
  SAGE_CHECK_LAUNCH("sage_dequantize_rows");
  return SAGE_OK;
}

extern "C" size_t sage_rms_norm_bwd_workspace_bytes(sage_i64 rows, sage_i64 dim, int dtype) {
  if (rows <= 0 || dim <= 0) return 0;
  return static_cast<size_t>(bwd_blocks(rows, dim, dtype)) * static_cast<size_t>(dim) * sizeof(float);
}

extern "C" int sage_rms_norm_bwd(const void* dy, sage_i64 ld_dy, const void* sum, sage_i64 ld_sum, const void* weight,
                                 int weight_dtype, const void* dsum, sage_i64 ld_dsum, sage_i64 rows, sage_i64 dim,
                                 int dtype, float eps, void* dx, sage_i64 ld_dx, void* dweight, void* workspace,
                                 size_t workspace_bytes, void* stream) {
  SAGE_REQUIRE(known_dtype(dtype), SAGE_EINVAL, "sage_rms_norm_bwd: unknown dtype %d", dtype);
  SAGE_REQUIRE(rows > 0 && dim > 0, SAGE_EINVAL, "sage_rms_norm_bwd: bad shape [%ld, %ld]", (long)rows, (long)dim);
  SAGE_REQUIRE(weight_dtype == dtype || weight_dtype == SAGE_F32, SAGE_EINVAL,
               "sage_rms_norm_bwd: the weight is in the rows' type or in fp32");
  SAGE_REQUIRE(dy != nullptr && sum != nullptr && weight != nullptr && (dx != nullptr || dweight != nullptr), SAGE_EINVAL,
               "sage_rms_norm_bwd: NULL pointer");
  SAGE_REQUIRE(ld_dy >= 0 && ld_sum >= 0 && ld_dsum >= 0 && (dx == nullptr || ld_dx >= dim), SAGE_EINVAL,
               "sage_rms_norm_bwd: row stride below the width");
  SAGE_REQUIRE(dweight == nullptr || (workspace != nullptr && workspace_bytes >= sage_rms_norm_bwd_workspace_bytes(rows, dim, dtype)),
               SAGE_EWORKSPACE, "sage_rms_norm_bwd: workspace of %zu bytes", workspace_bytes);
  NormBwdArgs a{};
  a.dy = dy; a.s = sum; a.ds = dsum; a.dx = dx;
  if (weight_dtype == dtype) a.w = weight; else a.w32 = static_cast<const float*>(weight);
  a.part = dweight != nullptr ? static_cast<float*>(workspace) : nullptr;
  a.ld_dy = ld_dy; a.ld_s = ld_sum; a.ld_ds = ld_dsum; a.ld_dx = ld_dx;
  a.rows = rows; a.dim = dim; a.eps = eps;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == SAGE_F32) launch_norm_bwd<float>(a, dtype, st);
  else if (dtype == SAGE_BF16) launch_norm_bwd<__bf16>(a, dtype, st);
  else launch_norm_bwd<_Float16>(a, dtype, st);
  SAGE_CHECK_LAUNCH("sage_rms_norm_bwd");
  if (dweight != nullptr) {
    const int64_t parts = bwd_blocks(rows, dim, dtype);
    const dim3 grid(static_cast<unsigned>(cdiv(dim, 16)));
    if (weight_dtype == SAGE_F32)
      hipLaunchKernelGGL((dweight_sum_kernel<float>), grid, dim3(1024), 0, st, a.part, parts, dim, static_cast<float*>(dweight));
    else if (weight_dtype == SAGE_BF16)
      hipLaunchKernelGGL((dweight_sum_kernel<__bf16>), grid, dim3(1024), 0, st, a.part, parts, dim, static_cast<__bf16*>(dweight));
    else
      hipLaunchKernelGGL((dweight_sum_kernel<_Float16>), grid, dim3(1024), 0, st, a.part, parts, dim, static_cast<_Float16*>(dweight));
    SAGE_CHECK_LAUNCH("sage_rms_norm_bwd");
  }
  return SAGE_OK;
}
