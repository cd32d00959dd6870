// The short causal convolution in front of a selective scan, channel by channel, with its
// gradients, and one token of every environment. No reference counterpart.
//
//   pre_t = bias + sum_{i < W} weight[W - 1 - i] x_{t-i}        out = pre silu'd, or pre itself
//
// where taps that reach before the first token of t's episode are left out, and those before the
// row's first token come from `state`, the W - 1 values before it.
//
// A thread walks a run of tokens of four channels with the last W - 1 values in registers, so each
// value is read once but for the W - 1 at a run's borders. A block's threads walk the same tokens, so
// what depends on the token alone is scalar. 64 x 1,000 tokens of 501 channels, bfloat16 at odd addresses: 41 us,
// 3.1 TB/s, and 76 + 10 backwards, 2.5 TB/s, bound by vector instructions (about 55 and 60 % of the time) and
// by the latency that two waves a SIMD leave backwards (204 registers; three waves spill: 180 us). In float32, with
// 248 registers backwards, 61 us, and 170 for both.
#include "row_ops.h"

namespace hipenvs {
namespace conv {

using namespace rows;

constexpr int kMaxTaps = 4;
constexpr int kAhead = 4;   // tokens whose loads are in flight

struct Conv {
  const void *x, *dout;
  int64_t x_sb, x_st, dout_sb, dout_st, reset_sb, reset_st;
  const float *weight, *bias, *state, *dfinal;
  const uint8_t* reset;
  void *out, *dx;
  float *final_state, *dstate, *dparams;   // dparams (runs b, d (W + 1)): weight (d, W), then bias
  int64_t b, t, run, runs, across, item0;   // across: blocks that hold a run of every row
  int32_t d, quads;
  bool silu;
};

template <int W>
struct Taps {
  f32x4 w[W], bias;

  __device__ __forceinline__ Taps(const Conv& s, int c) {
    const int left = s.d - c;
    bias = s.bias ? load_upto(s.bias + c, left) : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < W; ++j) {
      w[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (e < left) w[j][e] = s.weight[(int64_t)(c + e) * W + j];
    }
  }

  // hist[i]: the value i tokens back
  __device__ __forceinline__ f32x4 apply(const f32x4 (&hist)[W]) const {
    f32x4 pre = bias;
#pragma unroll
    for (int i = W - 1; i >= 0; --i)
#pragma unroll
      for (int e = 0; e < 4; ++e) pre[e] = __builtin_fmaf(w[W - 1 - i][e], hist[i][e], pre[e]);
    return pre;
  }
};

// The new value in front of those before it, which end where an episode begins.
template <int W>
__device__ __forceinline__ void push(f32x4 (&hist)[W], f32x4 x, bool begins) {
#pragma unroll
  for (int i = W - 1; i > 0; --i) hist[i] = hist[i - 1];
  hist[0] = x;
  if (__builtin_amdgcn_ballot_w64(begins)) {   // seldom
#pragma unroll
    for (int i = 1; i < W; ++i) hist[i] = begins ? f32x4{0.0f, 0.0f, 0.0f, 0.0f} : hist[i];
  }
}

// A thread's place: a run of tokens, the same for its block, and four channels of a row.
struct Place {
  int64_t run, t0, t1, b;
  int c;
  bool there;

  __device__ __forceinline__ explicit Place(const Conv& s) {
    const int64_t block = s.item0 + blockIdx.x;
    run = block / s.across;
    t0 = run * s.run;
    t1 = t0 + s.run < s.t ? t0 + s.run : s.t;
    const int64_t item = (block - run * s.across) * kBlock + threadIdx.x;
    b = item / s.quads;
    there = b < s.b;
    c = (int)(item - b * s.quads) * 4;
  }
};

// A row's tokens for four channels, fetched kAhead at once; those past `end` are the last one again.
template <class T, bool kWide, bool kBack>
struct Tokens {
  const T *x, *dout;
  const uint8_t* reset;
  int64_t x_st, dout_st, reset_st;
  FourOf<T, kWide> four;

  struct Piece {
    typename Raw<T>::type x[kAhead], dout[kAhead];
    uint8_t begins[kAhead];
  };

  __device__ __forceinline__ Tokens(const Conv& s, int64_t b, int c) : four(c, s.d) {
    x = (const T*)s.x + b * s.x_sb + four.from;
    dout = kBack ? (const T*)s.dout + b * s.dout_sb + four.from : nullptr;
    reset = s.reset ? s.reset + b * s.reset_sb : nullptr;
    x_st = s.x_st, dout_st = s.dout_st, reset_st = s.reset_st;
  }

  __device__ __forceinline__ void fetch(Piece& to, int64_t first, int64_t end) const {
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int64_t t = first + k < end ? first + k : end - 1;   // the same for every lane
      to.x[k] = four.fetch(x + t * x_st);
      if (kBack) to.dout[k] = four.fetch(dout + t * dout_st);
      to.begins[k] = reset ? reset[t * reset_st] : 0;
    }
  }
};

// hist as it is before token t0: hist[i] then holds the value of token t0 - 1 - i. A run has more tokens
// than a window: windows of all runs but the first lie within the row. Returns the tokens from the episode's
// first to t0 - 1, W where it lies before the window.
template <class T, int W, bool kWide, bool kBack>
__device__ __forceinline__ int before(const Conv& s, const Tokens<T, kWide, kBack>& of, int64_t b, int64_t t0, int c,
                                       f32x4 (&hist)[W]) {
#pragma unroll
  for (int i = 0; i < W; ++i) hist[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  if (t0 == 0) {
#pragma unroll
    for (int k = 0; k < W - 1; ++k) {
      f32x4 x = {0.0f, 0.0f, 0.0f, 0.0f};
      if (s.state) x = load_upto(s.state + (b * (W - 1) + k) * s.d + c, s.d - c);
      push(hist, x, false);
    }
    return W;
  }
  typename Raw<T>::type x[W];
  uint8_t begins[W];
#pragma unroll
  for (int k = 0; k < W - 1; ++k) {
    const int64_t t = t0 - (W - 1) + k;
    x[k] = of.four.fetch(of.x + t * of.x_st);
    begins[k] = of.reset ? of.reset[t * of.reset_st] : 0;
  }
  int since = W;
#pragma unroll
  for (int k = 0; k < W - 1; ++k) {
    push(hist, of.four.value(x[k]), begins[k]);
    since = begins[k] ? 0 : since < W ? since + 1 : W;
  }
  return since;
}

template <class T, int W, bool kWide>
__global__ __launch_bounds__(kBlock) void forward_kernel(Conv s) {
  const Place at(s);
  if (!at.there) return;
  const int left = s.d - at.c;
  const Taps<W> taps(s, at.c);
  const Tokens<T, kWide, false> of(s, at.b, at.c);
  f32x4 hist[W];
  before(s, of, at.b, at.t0, at.c, hist);
  typename Tokens<T, kWide, false>::Piece next;
  if (at.t0 < at.t1) of.fetch(next, at.t0, at.t1);
  T* out = (T*)s.out + at.b * s.t * s.d + at.c;
  for (int64_t first = at.t0; first < at.t1; first += kAhead) {
    const auto now = next;
    if (first + kAhead < at.t1) of.fetch(next, first + kAhead, at.t1);
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      if (first + k >= at.t1) break;
      push(hist, of.four.value(now.x[k]), now.begins[k]);
      f32x4 pre = taps.apply(hist);
      if (s.silu)
#pragma unroll
        for (int e = 0; e < 4; ++e) pre[e] *= sigmoid_for<T>(pre[e]);
      store_upto(out + (first + k) * s.d, pre, left);
    }
  }
  if (at.t1 == s.t)
#pragma unroll
    for (int k = 0; k < W - 1; ++k)
      store_upto(s.final_state + (at.b * (W - 1) + k) * s.d + at.c, hist[W - 2 - k], left);
}

// Gradients of a run: token t's reaches the W tokens up to t, as far as its episode does. A run's own
// tokens wait in `late` for those behind them, W - 1 past its end; the first run has the state's
// values among its own, and what a row's last values leave in the final state comes last.
template <class T, int W, bool kWide>
__global__ __launch_bounds__(kBlock, 2) void backward_kernel(Conv s) {
  const Place at(s);
  if (!at.there) return;
  const int left = s.d - at.c;
  const int64_t t0 = at.t0, t1 = at.t1, past = t1 + W - 1 < s.t ? t1 + W - 1 : s.t;
  const int64_t first_own = t0 == 0 ? -(W - 1) : t0;
  const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
  const Taps<W> taps(s, at.c);
  const Tokens<T, kWide, true> of(s, at.b, at.c);
  f32x4 hist[W], late[W], dweight[W], dbias = zero;   // late[i]: the gradient of token t - i
  int since = before(s, of, at.b, t0, at.c, hist);   // tokens since the episode's first
#pragma unroll
  for (int i = 0; i < W; ++i) late[i] = dweight[i] = zero;
  T* dx = (T*)s.dx + at.b * s.t * s.d + at.c;
  float* dstate = s.dstate + at.b * (W - 1) * s.d + at.c;
  const auto emit = [&](int64_t u, f32x4 grad) {   // u is the same for every lane
    if (u < first_own || u >= t1) return;
    if (u < 0)
      store_upto(dstate + (u + W - 1) * s.d, grad, left);
    else
      store_upto(dx + u * s.d, grad, left);
  };
  typename Tokens<T, kWide, true>::Piece next;
  if (t0 < past) of.fetch(next, t0, past);
  for (int64_t first = t0; first < past; first += kAhead) {
    const auto now = next;
    if (first + kAhead < past) of.fetch(next, first + kAhead, past);
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int64_t t = first + k;
      if (t >= past) break;
      push(hist, of.four.value(now.x[k]), now.begins[k]);
      since = now.begins[k] ? 0 : since < W ? since + 1 : W;
      f32x4 grad = of.four.value(now.dout[k]);
      if (s.silu) {
        const f32x4 pre = taps.apply(hist);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float one = sigmoid_for<T>(pre[e]);
          grad[e] *= one * __builtin_fmaf(pre[e], 1.0f - one, 1.0f);
        }
      }
#pragma unroll
      for (int i = W - 1; i > 0; --i) late[i] = late[i - 1];
      late[0] = zero;
      if (t < t1 && __builtin_amdgcn_ballot_w64(since < W - 1) == 0) {   // whole windows of own tokens
#pragma unroll
        for (int i = 0; i < W; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            late[i][e] = __builtin_fmaf(taps.w[W - 1 - i][e], grad[e], late[i][e]);
            dweight[i][e] = __builtin_fmaf(hist[i][e], grad[e], dweight[i][e]);
          }
        dbias += grad;
      } else {
#pragma unroll
        for (int i = 0; i < W; ++i)
          if (i <= since)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              late[i][e] = __builtin_fmaf(taps.w[W - 1 - i][e], grad[e], late[i][e]);
              if (t < t1) dweight[i][e] = __builtin_fmaf(hist[i][e], grad[e], dweight[i][e]);
            }
        if (t < t1) dbias += grad;
      }
      emit(t - (W - 1), late[W - 1]);
    }
  }
  if (past == s.t)   // what the final state takes of the last W - 1 tokens
#pragma unroll
    for (int i = W - 2; i >= 0; --i) {
      f32x4 grad = late[i];
      if (s.dfinal && i <= since) grad += load_upto(s.dfinal + (at.b * (W - 1) + (W - 2 - i)) * s.d + at.c, left);
      emit(s.t - 1 - i, grad);
    }
  float* params = s.dparams + (at.run * s.b + at.b) * ((int64_t)s.d * (W + 1));
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (e < left) {
#pragma unroll
      for (int j = 0; j < W; ++j) params[(int64_t)(at.c + e) * W + j] = dweight[W - 1 - j][e];
      params[(int64_t)s.d * W + at.c + e] = dbias[e];
    }
}

// One token of every environment; next may be state itself: a thread writes only what it has read.
struct Step {
  const void* x;
  int64_t x_s, reset_s;
  const float *weight, *bias, *state;
  const uint8_t* reset;
  void* out;
  float* next;
  int64_t n, item0;
  int32_t d, quads;
  bool silu;
};

template <class T, int W>
__global__ __launch_bounds__(kBlock) void step_kernel(Step s) {
  const int64_t item = (s.item0 + blockIdx.x) * kBlock + threadIdx.x, env = item / s.quads;
  if (env >= s.n) return;
  const int c = (int)(item - env * s.quads) * 4, left = s.d - c;
  Conv of = {};
  of.weight = s.weight, of.bias = s.bias, of.d = s.d;
  const Taps<W> taps(of, c);
  const bool begins = s.reset && s.reset[env * s.reset_s];
  f32x4 hist[W];
#pragma unroll
  for (int i = 0; i < W - 1; ++i) hist[i] = load_upto(s.state + (env * (W - 1) + (W - 2 - i)) * s.d + c, left);
  push(hist, load_upto((const T*)s.x + env * s.x_s + c, left), begins);
  f32x4 pre = taps.apply(hist);
  if (s.silu)
#pragma unroll
    for (int e = 0; e < 4; ++e) pre[e] *= sigmoid_for<T>(pre[e]);
  store_upto((T*)s.out + env * s.d + c, pre, left);
#pragma unroll
  for (int k = 0; k < W - 1; ++k) store_upto(s.next + (env * (W - 1) + k) * s.d + c, hist[W - 2 - k], left);
}

namespace {
bool dims_ok(int32_t dtype, int64_t d, int64_t w) {
  return (dtype == 0 || dtype == 1) && d >= 1 && d <= 65536 && w >= 1 && w <= kMaxTaps;
}

bool sequence_ok(int32_t dtype, int64_t b, int64_t t, int32_t d, int32_t w) {
  return dims_ok(dtype, d, w) && b >= 0 && b <= 0x7FFFFFFF && t >= 0 && t <= 0x7FFFFFFF && b * d <= 0x7FFFFFFF;
}

// Runs of 64 tokens, shorter (down to 8) while the card has fewer waves than it holds: eight a CU
// forwards, and half of that backwards, where a run costs a row of partial sums (64 x 1,000 x 501
// bfloat16: 84 + 13 us with runs of 32, 76 + 10 with 64). By this rule, with runs of 64 and of 8 throughout, in us,
// bfloat16: 64 x 1,000 x 501 41, 45 and 54 (both passes 120, 120, 194), 16 x 1,000 x 501 21, 33 and 21 (55, 91, 66),
// 1 x 16,381 x 512 18, 30 and 20 (57, 83, 79), 128 x 64 x 64 9, 26 and 9 (26, 75, 26).
int plan(Conv* s, int64_t b, int64_t t, int32_t d, bool back) {
  int cus = 0;
  const int status = device_cus(&cus);
  if (status != HIPENVS_OK) return status;
  s->b = b, s->t = t, s->d = d, s->quads = (d + 3) / 4;
  s->run = 64;
  while (s->run > 8 && b * s->quads * ((t + s->run - 1) / s->run) < (int64_t)cus * (back ? 4 : 8) * 64)
    s->run /= 2;
  s->runs = t > 0 ? (t + s->run - 1) / s->run : 1;
  s->across = (b * s->quads + kBlock - 1) / kBlock;
  return HIPENVS_OK;
}

template <class F>
int for_taps(int w, const F& f) {
  switch (w) {
    case 1: return f(std::integral_constant<int, 1>());
    case 2: return f(std::integral_constant<int, 2>());
    case 3: return f(std::integral_constant<int, 3>());
    default: return f(std::integral_constant<int, 4>());
  }
}

template <class S, class F>
int in_launches(S s, int64_t blocks, const F& launch) {
  constexpr int64_t kMost = kMostThreads / kBlock;
  for (s.item0 = 0; s.item0 < blocks; s.item0 += kMost) {
    launch(s, dim3((unsigned)(blocks - s.item0 < kMost ? blocks - s.item0 : kMost)));
    const int status = launch_status();
    if (status != HIPENVS_OK) return status;
  }
  return HIPENVS_OK;
}
}  // namespace

}  // namespace conv
}  // namespace hipenvs

using namespace hipenvs;
using namespace hipenvs::conv;

extern "C" int64_t hipenvs_causal_conv_workspace_bytes(int64_t b, int64_t t, int32_t d, int32_t w) {
  if (!sequence_ok(0, b, t, d, w)) return -1;
  if (b == 0) return 0;
  Conv s = {};
  if (plan(&s, b, t, d, true) != HIPENVS_OK) return -1;
  const int64_t rows = b * s.runs, width = (int64_t)d * (w + 1);
  return rows * width * (int64_t)sizeof(float) + column_sums_bytes(rows, width);
}

extern "C" int hipenvs_causal_conv(int32_t dtype, const void* x, const float* weight, const float* bias,
                                   const float* state, const uint8_t* reset, const int64_t* strides, int32_t silu,
                                   void* out, float* final_state, int64_t b, int64_t t, int32_t d, int32_t w,
                                   hipenvs_stream_t stream) {
  if (!sequence_ok(dtype, b, t, d, w)) return HIPENVS_E_ARG;
  if (b == 0) return HIPENVS_OK;
  if (!weight || (w > 1 && !final_state) || (t > 0 && (!x || !out || !strides))) return HIPENVS_E_ARG;
  Conv s = {};
  const int status = plan(&s, b, t, d, false);
  if (status != HIPENVS_OK) return status;
  s.x = x, s.weight = weight, s.bias = bias, s.state = state, s.reset = reset, s.silu = silu != 0;
  s.out = out, s.final_state = final_state;
  if (t > 0) s.x_sb = strides[0], s.x_st = strides[1], s.reset_sb = strides[2], s.reset_st = strides[3];
  return for_taps(w, [&](auto taps) {
    constexpr int W = decltype(taps)::value;
    return in_launches(s, s.runs * s.across, [&](const Conv& a, dim3 grid) {
      const bool wide = d >= 4;
      if (dtype == 1 && wide)
        hipLaunchKernelGGL((forward_kernel<__bf16, W, true>), grid, dim3(kBlock), 0, as_stream(stream), a);
      else if (dtype == 1)
        hipLaunchKernelGGL((forward_kernel<__bf16, W, false>), grid, dim3(kBlock), 0, as_stream(stream), a);
      else if (wide)
        hipLaunchKernelGGL((forward_kernel<float, W, true>), grid, dim3(kBlock), 0, as_stream(stream), a);
      else
        hipLaunchKernelGGL((forward_kernel<float, W, false>), grid, dim3(kBlock), 0, as_stream(stream), a);
    });
  });
}

extern "C" int hipenvs_causal_conv_backward(int32_t dtype, const void* x, const float* weight, const float* bias,
                                            const float* state, const uint8_t* reset, const void* dout,
                                            const float* dfinal, const int64_t* strides, int32_t silu, void* dx,
                                            float* dparams, float* dstate, int64_t b, int64_t t, int32_t d, int32_t w,
                                            void* workspace, int64_t workspace_bytes, hipenvs_stream_t stream) {
  if (!sequence_ok(dtype, b, t, d, w) || !dparams) return HIPENVS_E_ARG;
  const int64_t width = (int64_t)d * (w + 1);
  if (b == 0) return column_sums<float>(nullptr, 0, width, 1.0f, dparams, nullptr, as_stream(stream));
  if (!weight || (w > 1 && !dstate) || (t > 0 && (!x || !dout || !dx || !strides))) return HIPENVS_E_ARG;
  Conv s = {};
  int status = plan(&s, b, t, d, true);
  if (status != HIPENVS_OK) return status;
  const int64_t rows = b * s.runs, partial = rows * width * (int64_t)sizeof(float);
  if (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < partial + column_sums_bytes(rows, width))
    return HIPENVS_E_ARG;
  s.x = x, s.weight = weight, s.bias = bias, s.state = state, s.reset = reset, s.silu = silu != 0;
  s.dout = dout, s.dfinal = dfinal, s.dx = dx, s.dstate = dstate, s.dparams = (float*)workspace;
  if (t > 0)
    s.x_sb = strides[0], s.x_st = strides[1], s.reset_sb = strides[2], s.reset_st = strides[3], s.dout_sb = strides[4],
    s.dout_st = strides[5];
  status = for_taps(w, [&](auto taps) {
    constexpr int W = decltype(taps)::value;
    return in_launches(s, s.runs * s.across, [&](const Conv& a, dim3 grid) {
      const bool wide = d >= 4;
      if (dtype == 1 && wide)
        hipLaunchKernelGGL((backward_kernel<__bf16, W, true>), grid, dim3(kBlock), 0, as_stream(stream), a);
      else if (dtype == 1)
        hipLaunchKernelGGL((backward_kernel<__bf16, W, false>), grid, dim3(kBlock), 0, as_stream(stream), a);
      else if (wide)
        hipLaunchKernelGGL((backward_kernel<float, W, true>), grid, dim3(kBlock), 0, as_stream(stream), a);
      else
        hipLaunchKernelGGL((backward_kernel<float, W, false>), grid, dim3(kBlock), 0, as_stream(stream), a);
    });
  });
  if (status != HIPENVS_OK) return status;
  return column_sums<float>(s.dparams, rows, width, 1.0f, dparams, (float*)((char*)workspace + partial), as_stream(stream));
}

extern "C" int hipenvs_causal_conv_step(int32_t dtype, const void* x, int64_t x_sn, const float* weight,
                                        const float* bias, const float* state, const uint8_t* reset, int64_t reset_sn,
                                        int32_t silu, void* out, float* next_state, int64_t n, int32_t d, int32_t w,
                                        hipenvs_stream_t stream) {
  if (!dims_ok(dtype, d, w) || n < 0 || n > 0x7FFFFFFF || n * d > 0x7FFFFFFF) return HIPENVS_E_ARG;
  if (n == 0) return HIPENVS_OK;
  if (!x || !weight || !out || (w > 1 && (!state || !next_state))) return HIPENVS_E_ARG;
  Step s = {x, x_sn, reset_sn, weight, bias, state, reset, out, next_state, n, 0, d, (d + 3) / 4, silu != 0};
  return for_taps(w, [&](auto taps) {
    constexpr int W = decltype(taps)::value;
    return in_launches(s, (n * s.quads + kBlock - 1) / kBlock, [&](const Step& a, dim3 grid) {
      if (dtype == 1)
        hipLaunchKernelGGL((step_kernel<__bf16, W>), grid, dim3(kBlock), 0, as_stream(stream), a);
      else
        hipLaunchKernelGGL((step_kernel<float, W>), grid, dim3(kBlock), 0, as_stream(stream), a);
    });
  });
}
