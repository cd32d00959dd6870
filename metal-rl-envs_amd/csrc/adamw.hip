// One AdamW step over many tensors at once, moments in 32 bits or in 8 bits with a scale for
// every 256 values, and the read-back of 8-bit moments. No reference counterpart: the
// reference's learners call their array library's optimizer.
//
//   m' = b1 m + (1 - b1) g          v' = b2 v + (1 - b2) g^2
//   p' = keep p - (rate m') / (sqrt(v') root + eps),
//   keep = 1 - lr wd, rate = lr / (1 - b1^t), root = 1 / sqrt(1 - b2^t)
//
// All arithmetic is float32, each operation rounded on its own (the library's
// -ffp-contract=off), with correctly rounded division and square root, so the result is a
// function of the inputs bit for bit. Parameters and gradients are float32 or bfloat16;
// a bfloat16 parameter is rounded once, to nearest even, when it is written.
#include "hipenvs_device.h"

namespace hipenvs {
namespace adamw {

constexpr int kQuant = 256;          // values that share one scale, and the grain of the flat moments
constexpr int kTile = 1024;          // values a block takes: four quant blocks, one for each wave
constexpr int kMaxTensors = 64;      // of one launch: its descriptors are kernel arguments, below 4 KiB
// A launch's threads stay below 2^32, the most a grid's axis takes: a tensor goes in pieces of
// kPiece values, at most kMostTiles tiles to a launch.
constexpr int64_t kPiece = (int64_t)1 << 32;
constexpr uint64_t kMostTiles = (uint64_t)1 << 23;
constexpr uint32_t kParamBf16 = 1, kGradBf16 = 2, kWide = 4;

struct Tensor {
  void* param;
  const void* grad;
  int64_t n;
  int64_t at;       // where its moments begin, a multiple of kQuant
  uint32_t tile0;   // the first of its tiles in this launch
  uint32_t types;   // kParamBf16 | kGradBf16 | kWide: every pointer can take four values at once
  float rate, root;
};

struct Batch {
  Tensor t[kMaxTensors];
  int32_t count;
  float beta1, rest1, beta2, rest2, eps, keep;
};

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));

// Four values at `i` of a float32 or bfloat16 array of n; beyond n they are zero. `whole`: they
// are all there, and lie where four are read at once (the same for a wave).
__device__ __forceinline__ void load4(const void* base, int64_t i, int64_t n, bool bf16, bool whole, float (&x)[4]) {
  if (whole) {
    f32x4 w;
    if (bf16)
      w = __builtin_convertvector(*(const bf16x4*)((const __bf16*)base + i), f32x4);
    else
      w = *(const f32x4*)((const float*)base + i);
    x[0] = w.x, x[1] = w.y, x[2] = w.z, x[3] = w.w;
    return;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    x[e] = 0.0f;
    if (i + e < n) x[e] = bf16 ? (float)((const __bf16*)base)[i + e] : ((const float*)base)[i + e];
  }
}

__device__ __forceinline__ void store4(void* base, int64_t i, int64_t n, bool bf16, bool whole, const float (&x)[4]) {
  const f32x4 w = {x[0], x[1], x[2], x[3]};
  if (whole) {
    if (bf16)
      *(bf16x4*)((__bf16*)base + i) = __builtin_convertvector(w, bf16x4);   // to nearest even
    else
      *(f32x4*)((float*)base + i) = w;
    return;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (i + e < n) {
      if (bf16)
        ((__bf16*)base)[i + e] = (__bf16)x[e];
      else
        ((float*)base)[i + e] = x[e];
    }
}

__device__ __forceinline__ float moved(float p, float m, float v, const Batch& b, const Tensor& t) {
  return p * b.keep - (m * t.rate) / (sqrt_rn(v) * t.root + b.eps);
}

// The tensor whose tiles hold `tile`: the last one that begins at or before it. Uniform over
// the block, over at most 64 descriptors in the kernel's arguments.
__device__ __forceinline__ int find(const Batch& b, uint32_t tile) {
  int lo = 0, hi = b.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (b.t[mid].tile0 <= tile)
      lo = mid;
    else
      hi = mid - 1;
  }
  return lo;
}

// 32-bit moments: 28 bytes a float32 value, four values a thread, bound by memory (184 million
// values in 950 us, 5.4 TB/s). A block finds its tensor in the kernel's arguments: no table to
// upload, and one launch for 64 tensors.
__global__ __launch_bounds__(kBlock) void step32_kernel(Batch b, float* __restrict__ m_all, float* __restrict__ v_all) {
  const Tensor& t = b.t[find(b, blockIdx.x)];
  const int64_t first = (int64_t)(blockIdx.x - t.tile0) * kTile, i = first + 4 * threadIdx.x;
  if (i >= t.n) return;
  const bool wide = (t.types & kWide) && first + kTile <= t.n, pb = t.types & kParamBf16, gb = t.types & kGradBf16;
  float* m_at = m_all + t.at;
  float* v_at = v_all + t.at;
  float p[4], g[4], m[4], v[4];
  load4(t.param, i, t.n, pb, wide, p);
  load4(t.grad, i, t.n, gb, wide, g);
  load4(m_at, i, t.n, false, wide, m);
  load4(v_at, i, t.n, false, wide, v);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    m[e] = m[e] * b.beta1 + g[e] * b.rest1;
    v[e] = v[e] * b.beta2 + (g[e] * g[e]) * b.rest2;
    p[e] = moved(p[e], m[e], v[e], b, t);
  }
  store4(t.param, i, t.n, pb, wide, p);
  store4(m_at, i, t.n, false, wide, m);
  store4(v_at, i, t.n, false, wide, v);
}

// ---- 8-bit moments -------------------------------------------------------------------
// A block of 256 values keeps its largest magnitude A (float32) and a code for each value:
// of m, c in [-127, 127] for A t |t| with t = c / 127; of v, c in [0, 255] for A t^4 with
// t = c / 255, so sqrt(v), which divides the update, is held as a square like m. Rounding is
// to the nearest code of the root. No v above zero gets code 0: a denominator would fall to
// eps, and the update would grow by orders of magnitude. A block with a NaN or an infinity
// has that as its scale and reads back as no number; one whose largest magnitude is subnormal has
// the smallest normal number as its scale, whose reciprocal is finite.

__device__ __forceinline__ float decode_m(int c, float scale) {
  const float t = (float)c * (float)(1.0 / 127.0);
  return (t * __builtin_fabsf(t)) * scale;
}

__device__ __forceinline__ float decode_v(uint32_t c, float scale) {
  float t = (float)c * (float)(1.0 / 255.0);
  t = t * t;
  return (t * t) * scale;
}

// The largest of a wave's magnitudes, as bits, which order like the magnitudes with the
// infinities and NaN above every number.
__device__ __forceinline__ float wave_scale(const float (&x)[4]) {
  uint32_t u = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const uint32_t a = __float_as_uint(x[e]) & 0x7FFFFFFFu;
    u = a > u ? a : u;
  }
  // within 16 lanes by data-parallel moves, between the four rows by scalars
  const auto larger = [](uint32_t a, uint32_t b) { return a > b ? a : b; };
  u = larger(u, (uint32_t)__builtin_amdgcn_mov_dpp((int)u, 0xB1, 0xF, 0xF, true));    // the neighbour of two
  u = larger(u, (uint32_t)__builtin_amdgcn_mov_dpp((int)u, 0x4E, 0xF, 0xF, true));    // of four
  u = larger(u, (uint32_t)__builtin_amdgcn_mov_dpp((int)u, 0x141, 0xF, 0xF, true));   // mirrored in eight
  u = larger(u, (uint32_t)__builtin_amdgcn_mov_dpp((int)u, 0x140, 0xF, 0xF, true));   // mirrored in sixteen
  u = larger(larger((uint32_t)__builtin_amdgcn_readlane((int)u, 0), (uint32_t)__builtin_amdgcn_readlane((int)u, 16)),
             larger((uint32_t)__builtin_amdgcn_readlane((int)u, 32), (uint32_t)__builtin_amdgcn_readlane((int)u, 48)));
  return __uint_as_float(u != 0 && u < 0x00800000u ? 0x00800000u : u);
}

// A code: the nearest whole number in 0 .. top of root * top. The roots that
// decide are the correctly rounded ones, but only a product next to the border of two codes
// depends on their last bits. The hardware's root is within 1 ulp, and a root of such a root
// within 1.5; the exact ones within 0.5 and 0.75: so the products differ by at most
// 255 * 2.25 * 2^-23 and their own roundings, 2^-16, together below 8.5e-5, and give the same
// code unless they lie within kBorder of a half. A wave that holds such a one (about one in
// ten) takes the exact roots for all of it. Three exact roots for every value took 322 us for
// 87 million, bound by their float64 instructions.
constexpr float kBorder = 1e-4f;

__device__ __forceinline__ bool near_border(float product) {
  return __builtin_fabsf(__builtin_amdgcn_fractf(product) - 0.5f) < kBorder;
}

// 8-bit moments: a wave for a quant block, its largest magnitudes by moves within the wave.
// 88 million bfloat16 values in 242 us (10 bytes each, 3.6 TB/s), bound by its instructions, about
// 85 for a value: the exact root and quotient of the update and the codes. More quant blocks a
// wave did not help (251 us with two in flight, 275 with four).
__global__ __launch_bounds__(kBlock) void step8_kernel(Batch b, uint32_t* __restrict__ m_codes,
                                                       uint32_t* __restrict__ v_codes, float* __restrict__ m_scales,
                                                       float* __restrict__ v_scales) {
  const Tensor& t = b.t[find(b, blockIdx.x)];
  const int64_t first = (int64_t)(blockIdx.x - t.tile0) * kTile;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  if (first + wave * kQuant >= t.n) return;   // the whole wave: its quant block is past the tensor
  const int64_t i = first + 4 * threadIdx.x;
  const bool inside = first + (wave + 1) * kQuant <= t.n;
  const bool wide = (t.types & kWide) && inside, pb = t.types & kParamBf16, gb = t.types & kGradBf16;
  const int64_t word = (t.at + i) >> 2, block = (t.at + first) / kQuant + wave;
  float p[4], g[4], m[4], v[4];
  load4(t.param, i, t.n, pb, wide, p);
  load4(t.grad, i, t.n, gb, wide, g);
  const uint32_t mc = m_codes[word], vc = v_codes[word];
  const float ms = m_scales[block], vs = v_scales[block];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    m[e] = decode_m((int)(int8_t)(mc >> (8 * e)), ms) * b.beta1 + g[e] * b.rest1;
    v[e] = decode_v((vc >> (8 * e)) & 0xFFu, vs) * b.beta2 + (g[e] * g[e]) * b.rest2;
  }
  if (!inside) {   // the padding stays zero, also in a block that does not read back as numbers
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (i + e >= t.n) m[e] = v[e] = 0.0f;
  }
  const float new_ms = wave_scale(m), new_vs = wave_scale(v);
  const float m_inv = new_ms > 0.0f ? 1.0f / new_ms : 0.0f, v_inv = new_vs > 0.0f ? 1.0f / new_vs : 0.0f;
  float of_m[4], of_v[4];
  bool unsure = false;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    of_m[e] = __builtin_amdgcn_sqrtf(__builtin_fabsf(m[e]) * m_inv) * 127.0f;
    of_v[e] = __builtin_amdgcn_sqrtf(__builtin_amdgcn_sqrtf(v[e] * v_inv)) * 255.0f;
    unsure = unsure || near_border(of_m[e]) || near_border(of_v[e]);
  }
  if (__builtin_amdgcn_ballot_w64(unsure)) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      of_m[e] = sqrt_rn(__builtin_fabsf(m[e]) * m_inv) * 127.0f;
      of_v[e] = sqrt_rn(sqrt_rn(v[e] * v_inv)) * 255.0f;
    }
  }
  // the codes as float32 and into their bytes: a code of m below zero as 256 more, its two's
  // complement
  uint32_t new_mc = 0, new_vc = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float cm = __builtin_copysignf(__builtin_fminf(__builtin_rintf(of_m[e]), 127.0f), m[e]);
    const float cv = __builtin_fmaxf(__builtin_fminf(__builtin_rintf(of_v[e]), 255.0f), v[e] > 0.0f ? 1.0f : 0.0f);
    new_mc = __builtin_amdgcn_cvt_pk_u8_f32(cm < 0.0f ? cm + 256.0f : cm, e, new_mc);
    new_vc = __builtin_amdgcn_cvt_pk_u8_f32(cv, e, new_vc);
    p[e] = moved(p[e], m[e], v[e], b, t);
  }
  store4(t.param, i, t.n, pb, wide, p);
  m_codes[word] = new_mc;
  v_codes[word] = new_vc;
  if (lane == 0) {
    m_scales[block] = new_ms;
    v_scales[block] = new_vs;
  }
}

// The values of 8-bit moments: 2 bytes in, 8 out; 88 million in 137 us, 6.4 TB/s.
__global__ __launch_bounds__(kBlock) void decode_kernel(const uint32_t* __restrict__ m_codes,
                                                        const uint32_t* __restrict__ v_codes,
                                                        const float* __restrict__ m_scales,
                                                        const float* __restrict__ v_scales, int64_t word0,
                                                        int64_t words, float* __restrict__ m,
                                                        float* __restrict__ v) {
  const int64_t word = word0 + (int64_t)blockIdx.x * kBlock + threadIdx.x;
  if (word >= words) return;
  const int64_t block = word / (kQuant / 4);
  const uint32_t mc = m_codes[word], vc = v_codes[word];
  const float ms = m_scales[block], vs = v_scales[block];
  float x[4], y[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    x[e] = decode_m((int)(int8_t)(mc >> (8 * e)), ms);
    y[e] = decode_v((vc >> (8 * e)) & 0xFFu, vs);
  }
  store4(m, 4 * word, 4 * words, false, true, x);
  store4(v, 4 * word, 4 * words, false, true, y);
}

bool aligned(const void* p, uintptr_t to) { return ((uintptr_t)p & (to - 1)) == 0; }

}  // namespace adamw
}  // namespace hipenvs

using namespace hipenvs;
using namespace hipenvs::adamw;

extern "C" int hipenvs_adamw_step(int32_t bits, int32_t count, void* const* params, const void* const* grads,
                                  const int64_t* sizes, const int32_t* types, const double* rates,
                                  const double* roots, double beta1, double beta2, double eps, double keep, void* m,
                                  void* v, float* m_scales, float* v_scales, hipenvs_stream_t stream) {
  if ((bits != 32 && bits != 8) || count < 0) return HIPENVS_E_ARG;
  if (count == 0) return HIPENVS_OK;
  if (!params || !grads || !sizes || !types || !rates || !roots) return HIPENVS_E_ARG;
  int64_t total = 0;
  for (int32_t k = 0; k < count; ++k) {
    if (sizes[k] < 0 || sizes[k] > (int64_t)1 << 40 || (types[k] & ~3)) return HIPENVS_E_ARG;
    if (sizes[k] > 0 && !params[k]) return HIPENVS_E_ARG;
    total += sizes[k];
  }
  if (total == 0) return HIPENVS_OK;
  if (!m || !v || !aligned(m, 4) || !aligned(v, 4)) return HIPENVS_E_ARG;
  if (bits == 8 && (!m_scales || !v_scales)) return HIPENVS_E_ARG;
  const bool moments_wide = bits == 8 || (aligned(m, 16) && aligned(v, 16));
  Batch b;
  b.beta1 = (float)beta1, b.rest1 = (float)(1.0 - beta1);
  b.beta2 = (float)beta2, b.rest2 = (float)(1.0 - beta2);
  b.eps = (float)eps, b.keep = (float)keep;
  b.count = 0;
  int64_t at = 0;
  uint64_t tiles = 0;
  const auto launch = [&]() {
    const dim3 grid((unsigned)tiles), block(kBlock);
    if (bits == 32)
      hipLaunchKernelGGL(step32_kernel, grid, block, 0, as_stream(stream), b, (float*)m, (float*)v);
    else
      hipLaunchKernelGGL(step8_kernel, grid, block, 0, as_stream(stream), b, (uint32_t*)m, (uint32_t*)v, m_scales,
                         v_scales);
    b.count = 0;
    tiles = 0;
    return launch_status();
  };
  for (int32_t k = 0; k < count; ++k) {
    const int64_t n = grads[k] ? sizes[k] : 0;   // a tensor without a gradient keeps its parameters and its moments
    const int64_t p_size = (types[k] & 1) ? 2 : 4, g_size = (types[k] & 2) ? 2 : 4;
    for (int64_t done = 0; done < n; done += kPiece) {
      char* param = (char*)params[k] + done * p_size;
      const char* grad = (const char*)grads[k] + done * g_size;
      const int64_t own_n = n - done < kPiece ? n - done : kPiece;
      const uint64_t own = (uint64_t)((own_n + kTile - 1) / kTile);
      if (b.count == kMaxTensors || tiles + own > kMostTiles) {
        const int status = b.count ? launch() : HIPENVS_OK;
        if (status != HIPENVS_OK) return status;
      }
      const bool wide = moments_wide && aligned(param, 4 * p_size) && aligned(grad, 4 * g_size);
      b.t[b.count++] = {param, grad, own_n, at + done, (uint32_t)tiles, (uint32_t)types[k] | (wide ? kWide : 0u),
                        (float)rates[k], (float)roots[k]};
      tiles += own;
    }
    at += (sizes[k] + kQuant - 1) / kQuant * kQuant;
  }
  return b.count ? launch() : HIPENVS_OK;
}

extern "C" int hipenvs_adamw_decode(const void* m_codes, const void* v_codes, const float* m_scales,
                                    const float* v_scales, int64_t blocks, float* m, float* v,
                                    hipenvs_stream_t stream) {
  if (blocks < 0 || blocks > (int64_t)1 << 32) return HIPENVS_E_ARG;
  if (blocks == 0) return HIPENVS_OK;
  if (!m_codes || !v_codes || !m_scales || !v_scales || !m || !v) return HIPENVS_E_ARG;
  if (!aligned(m_codes, 4) || !aligned(v_codes, 4) || !aligned(m, 16) || !aligned(v, 16)) return HIPENVS_E_ARG;
  const int64_t words = blocks * (kQuant / 4);
  constexpr int64_t kMostWords = (int64_t)1 << 30;
  for (int64_t word0 = 0; word0 < words; word0 += kMostWords) {
    const int64_t own = words - word0 < kMostWords ? words - word0 : kMostWords;
    hipLaunchKernelGGL(decode_kernel, dim3(grid_for(own)), dim3(kBlock), 0, as_stream(stream),
                       (const uint32_t*)m_codes, (const uint32_t*)v_codes, m_scales, v_scales, word0, words, m, v);
    const int status = launch_status();
    if (status != HIPENVS_OK) return status;
  }
  return HIPENVS_OK;
}
