// Device pieces shared by the operators of policies over tokens: values of float32 or bfloat16
// rows four at a time at any address, sums over lanes, exponentials, and the sums of a matrix's
// columns in a fixed order.
#pragma once

#include "hipenvs_device.h"

namespace hipenvs {
namespace rows {

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
// four values at whatever address they lie: the card reads and writes them at any alignment
typedef f32x4 __attribute__((aligned(4))) f32x4_any;
typedef bf16x4 __attribute__((aligned(2))) bf16x4_any;

// A launch's threads stay below 2^32, the most a grid's axis takes.
constexpr int64_t kMostThreads = (int64_t)1 << 31;

constexpr float kLog2e = 0x1.715476p+0f, kLog2eLow = 0x1.4ae0cp-26f, kLn2 = 0x1.62e43p-1f;

template <class T>
__device__ __forceinline__ f32x4 load4(const T* p) {
  if constexpr (sizeof(T) == 2)
    return __builtin_convertvector(*(const bf16x4_any*)p, f32x4);
  else
    return *(const f32x4_any*)p;
}

// The first `n` of four values, zeros for the others; n may be 0 or less.
template <class T>
__device__ __forceinline__ f32x4 load_upto(const T* p, int64_t n) {
  if (n >= 4) return load4(p);
  f32x4 x = {0.0f, 0.0f, 0.0f, 0.0f};
  if (n > 0) x[0] = (float)p[0];
  if (n > 1) x[1] = (float)p[1];
  if (n > 2) x[2] = (float)p[2];
  return x;
}

// Four values as they lie in memory: a conversion where they are loaded would wait for each load by
// itself.
template <class T>
struct Raw;
template <>
struct Raw<float> {
  typedef f32x4 type;
  typedef f32x4_any any;
};
template <>
struct Raw<__bf16> {
  typedef bf16x4 type;
  typedef bf16x4_any any;
};

// Four values from `c` (a multiple of 4 below d) on of a row of d; at a ragged end the row's last four,
// which values() puts in their place. No branch depends on the lane, so a caller's loads are all in
// flight at once.
template <class T>
__device__ __forceinline__ typename Raw<T>::type fetch4(const T* row, int c, int d) {
  if (d >= 4) return *(const typename Raw<T>::any*)(row + (c < d - 4 ? c : d - 4));
  return typename Raw<T>::type{row[0], row[d > 1 ? 1 : 0], row[d > 2 ? 2 : 0], row[0]};
}

// What fetch4 read, as float32; zeros past the row.
template <class T>
__device__ __forceinline__ f32x4 values(typename Raw<T>::type raw, int c, int d) {
  const f32x4 x = __builtin_convertvector(raw, f32x4);
  const int left = d - c;
  if (__builtin_amdgcn_ballot_w64(left < 4) == 0) return x;   // no lane of the wave at the row's end
  const int by = d >= 4 && left < 4 ? 4 - left : 0;
  f32x4 y;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    y[e] = x[e];
#pragma unroll
    for (int k = 1; e + k < 4; ++k) y[e] = by == k ? x[e + k] : y[e];
    y[e] = e < left ? y[e] : 0.0f;
  }
  return y;
}

// The same for a thread that walks down a column of rows: where its four values lie is worked out once.
// kWide: rows of four values and more.
template <class T, bool kWide>
struct FourOf {
  int from, by, left;   // the first read, how far the values lie behind it, and how many there are
  bool ragged;          // of any lane of the wave

  __device__ __forceinline__ FourOf(int c, int d) {
    left = d - c;
    from = kWide && left < 4 ? d - 4 : c;
    by = kWide && left < 4 ? 4 - left : 0;
    ragged = __builtin_amdgcn_ballot_w64(left < 4) != 0;
  }

  __device__ __forceinline__ typename Raw<T>::type fetch(const T* row) const {   // row: from `from` on
    if constexpr (kWide)
      return *(const typename Raw<T>::any*)row;
    else
      return typename Raw<T>::type{row[0], row[left > 1 ? 1 : 0], row[left > 2 ? 2 : 0], row[0]};
  }

  __device__ __forceinline__ f32x4 value(typename Raw<T>::type raw) const {
    const f32x4 x = __builtin_convertvector(raw, f32x4);
    if (!ragged) return x;
    f32x4 y;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      y[e] = x[e];
#pragma unroll
      for (int k = 1; e + k < 4; ++k) y[e] = by == k ? x[e + k] : y[e];
      y[e] = e < left ? y[e] : 0.0f;
    }
    return y;
  }
};

template <class T>
__device__ __forceinline__ void store_upto(T* p, f32x4 x, int64_t n) {
  if (n >= 4) {
    if constexpr (sizeof(T) == 2)
      *(bf16x4_any*)p = __builtin_convertvector(x, bf16x4);   // to nearest even
    else
      *(f32x4_any*)p = x;
    return;
  }
  if (n > 0) p[0] = (T)x[0];
  if (n > 1) p[1] = (T)x[1];
  if (n > 2) p[2] = (T)x[2];
}

template <int kControl>
__device__ __forceinline__ float moved(float v) {
  return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), kControl, 0xF, 0xF, true));
}

// Lane l's value from lane l ^ kXor, within 16 lanes.
template <int kXor>
__device__ __forceinline__ float from_xor(float v) {
  if constexpr (kXor == 1) return moved<0xB1>(v);              // [1, 0, 3, 2] of four
  if constexpr (kXor == 2) return moved<0x4E>(v);              // [2, 3, 0, 1] of four
  if constexpr (kXor == 4) return moved<0x141>(moved<0x1B>(v));   // mirrored in four, then in eight
  if constexpr (kXor == 8) return moved<0x128>(v);             // turned by eight of sixteen
}

// The sum over kLanes neighbouring lanes (a power of two), the same bits in each of them.
template <int kLanes>
__device__ __forceinline__ float lanes_sum(float v) {
  if constexpr (kLanes >= 2) v += from_xor<1>(v);
  if constexpr (kLanes >= 4) v += from_xor<2>(v);
  if constexpr (kLanes >= 8) v += from_xor<4>(v);
  if constexpr (kLanes >= 16) v += from_xor<8>(v);
  if constexpr (kLanes >= 32) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  if constexpr (kLanes >= 64) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  return v;
}

__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }

// exp(-|x|), the rounding of x log2(e) made good; 0 below exp(-104).
__device__ __forceinline__ float exp_negative(float x) {
  const float a = __builtin_fabsf(x), n = a > 104.0f ? -104.0f : -a;
  const float hi = n * kLog2e, lo = __builtin_fmaf(n, kLog2eLow, __builtin_fmaf(n, kLog2e, -hi));
  const float e = exp2_of(hi);
  return __builtin_fmaf(e, lo * kLn2, e);
}

__device__ __forceinline__ float sigmoid(float x) {
  const float e = exp_negative(x), r = __builtin_amdgcn_rcpf(1.0f + e);
  return x >= 0.0f ? r : e * r;
}

// A sigmoid for results of type T. The short form's exponent is rounded once, by half a unit of 1.44 |x|:
// within 2^-16 of itself for the |x| <= 87 where it is a normal number, and zero from -88.8 on, far
// below a bfloat16's half unit; half the instructions.
template <class T>
__device__ __forceinline__ float sigmoid_for(float x) {
  if constexpr (sizeof(T) == 2)
    return __builtin_amdgcn_rcpf(1.0f + exp2_of(-kLog2e * x));
  else
    return sigmoid(x);
}

// log(1 + exp(x)) = max(x, 0) + log(1 + e), e = exp(-|x|), and its slope, the sigmoid. The rounding of
// u = 1 + e is made good by (e - (u - 1)) / u, the slope of the logarithm there.
struct Softplus {
  float value, slope;

  __device__ __forceinline__ explicit Softplus(float x) {
    const float e = exp_negative(x), u = 1.0f + e, r = __builtin_amdgcn_rcpf(u);
    const float l = __builtin_fmaf(e - (u - 1.0f), r, __builtin_amdgcn_logf(u) * kLn2);
    value = __builtin_amdgcn_fmed3f(x, 0.0f, __builtin_inff()) + l;   // a NaN is in l
    slope = x >= 0.0f ? r : e * r;
  }
};

__device__ __forceinline__ float softplus(float x) { return Softplus(x).value; }

// Sums of the columns of `from` (count, width) f32, in an order that depends on the sizes alone:
// block (i, j) sums rows i * each .. of 64 columns, four rows at once, into row i of `to`.
template <class Out>
__global__ __launch_bounds__(kBlock) void column_sums_kernel(const float* __restrict__ from, int64_t count,
                                                             int64_t width, int64_t each, float scale,
                                                             Out* __restrict__ to) {
  __shared__ float share[4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t column = (int64_t)blockIdx.x * 64 + lane, row0 = (int64_t)blockIdx.y * each;
  const int64_t rows_end = row0 + each < count ? row0 + each : count;
  float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  if (column < width) {
    int64_t r = row0 + wave;
    for (; r + 12 < rows_end; r += 16) {
#pragma unroll
      for (int k = 0; k < 4; ++k) sum[k] += from[(r + 4 * k) * width + column];
    }
    for (; r < rows_end; r += 4) sum[0] += from[r * width + column];
  }
  share[wave][lane] = (sum[0] + sum[1]) + (sum[2] + sum[3]);
  __syncthreads();
  if (wave == 0 && column < width)
    to[(int64_t)blockIdx.y * width + column] =
        (Out)(scale * ((share[0][lane] + share[1][lane]) + (share[2][lane] + share[3][lane])));
}

// Rows that the first of two launches leaves: enough blocks to fill the card, at least 32 rows each.
inline int64_t column_sums_rows(int64_t count, int64_t width) {
  const int64_t wide = (width + 63) / 64, most = (2048 + wide - 1) / wide, least = (count + 31) / 32;
  const int64_t rows = most < least ? most : least;
  return rows < 1 ? 1 : rows > 1024 ? 1024 : rows;
}

inline int64_t column_sums_bytes(int64_t count, int64_t width) {
  const int64_t rows = column_sums_rows(count, width);
  return rows > 1 ? rows * width * (int64_t)sizeof(float) : 0;
}

// to (width) = scale * the column sums of from (count, width); `between` has column_sums_bytes.
template <class Out>
int column_sums(const float* from, int64_t count, int64_t width, float scale, Out* to, float* between, hipStream_t s) {
  if (width <= 0) return HIPENVS_OK;
  const int64_t rows = column_sums_rows(count, width);
  const unsigned wide = (unsigned)((width + 63) / 64);
  if (rows == 1) {
    hipLaunchKernelGGL(column_sums_kernel<Out>, dim3(wide), dim3(kBlock), 0, s, from, count, width, count, scale, to);
    return launch_status();
  }
  const int64_t each = (count + rows - 1) / rows;
  hipLaunchKernelGGL(column_sums_kernel<float>, dim3(wide, (unsigned)rows), dim3(kBlock), 0, s, from, count, width, each,
                     1.0f, between);
  const int status = launch_status();
  if (status != HIPENVS_OK) return status;
  hipLaunchKernelGGL(column_sums_kernel<Out>, dim3(wide), dim3(kBlock), 0, s, (const float*)between, rows, width, rows,
                     scale, to);
  return launch_status();
}

}  // namespace rows
}  // namespace hipenvs
