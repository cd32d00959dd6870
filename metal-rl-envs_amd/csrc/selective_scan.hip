// The selective state space scan over trajectories, its gradients, and one token of every
// environment. No reference counterpart.
#include "selective_scan.h"

namespace hipenvs {
namespace scan {

// What a tile's walk has to leave out. States past n have no write and no read, but zero times an
// infinity is no number: where there are any, they are kept at zero, by whole lanes that see neither delta x
// nor dy (n a multiple of four) or one by one. 64 x 1,000 tokens of 500 channels of 12 states, bfloat16:
// 264 and 635 us forwards and backwards with every tile as kAny, 230 and 575 so.
// kFull: n is all the lanes' states, and there are none past it.
enum Kind { kPlain, kLanes, kBegins, kAny };   // nothing; lanes without states; beginnings; single states too

template <bool kFull, class F>
__device__ __forceinline__ void for_kind(uint32_t begins, int n, const F& walk) {
  if constexpr (kFull) {
    if (begins)
      walk(std::integral_constant<int, kBegins>());
    else
      walk(std::integral_constant<int, kPlain>());
  } else {
    if (begins || n % 4 != 0)
      walk(std::integral_constant<int, kAny>());
    else
      walk(std::integral_constant<int, kLanes>());
  }
}

// A rate times log2(e). An infinite one is as good as float32's largest, and times a delta of zero, which stands
// for that of an episode's first token in a walk, it is a number.
__device__ __forceinline__ float rate_of(float rate) {
  constexpr float kMost = 0x1.fffffep+127f;
  const float x = rate * kLog2e;
  return x > kMost ? kMost : x < -kMost ? -kMost : x;   // a NaN stays
}

// Four states' rates; those past n decay, so that an infinite delta leaves them at zero.
__device__ __forceinline__ f32x4 rates_of(const float* from, int left) {
  f32x4 rate = load_upto(from, left);
#pragma unroll
  for (int e = 0; e < 4; ++e) rate[e] = rate_of(e < left ? rate[e] : -1.0f);
  return rate;
}

// x, or 0 where `bits` is 0 and not ~0. A selection of the backward pass's values by a scalar condition became
// branches, across which 60 to 110 registers of decays and states spilled: 1,190 -> 2,000 us at 4,096 x 128 tokens of
// 128 channels, float32.
__device__ __forceinline__ float masked(float x, uint32_t bits) { return __uint_as_float(__float_as_uint(x) & bits); }

// One part of a row's tokens for a block of channels: LPC lanes hold a channel, four states each,
// and walk token by token; delta, x, write and read come through LDS, a tile of 16 tokens at a
// time, computed once each and fetched a tile ahead. kOut: outputs, from the states before the
// part; otherwise the part's own state alone, from zeros, for rows walked in parts.
//
// Bound by its vector instructions, which issue all of the time at 4,096 x 128 tokens of 128 channels, float32:
// 44 a token for 16 channels of 16 states, 22 of them the walk (two for each exponential), the rest what a
// tile's elements take: softplus, the gate, addresses, and reading back the scalars that spill into vector lanes
// (53 to 82 with outputs, 21 to 41 without; none in the walks). 340 to 370 us there, 2.5 TB/s and more; 16,381
// tokens of 512 channels in parts 36 + 15 + 51 us. n counts as the 8, 16, 32 or 64 states that the lanes hold:
// 1,024 x 128 x 128, bfloat16, 62 us for n = 8, 96 for 9, 86 for 16, 178 for 17, 160 for 32, 352 for 33, 318 for 64.
// Tiles of eight tokens took 442, of one row in fewer parts (eight waves a CU instead of 16) 41 + 9 + 64. Loads
// that a branch or a conversion separates wait for each other: 73 us for the 51 before they went.
template <class T, int LPC, bool kFew, bool kFull, bool kOut>
__global__ __launch_bounds__((Shape<LPC, kFew>::kThreads)) void forward_kernel(Scan s) {
  using S = Shape<LPC, kFew>;
  using At = Slots<LPC, kFew>;
  __shared__ __attribute__((aligned(16))) f32x2 steps[kTile][S::CH];      // delta, delta x; then y
  __shared__ __attribute__((aligned(16))) float mix[kTile][2 * S::NP];
  const int parts = kOut ? s.parts : s.parts - 1;
  const Place at = place_of(s, s.item0 + blockIdx.x, parts, S::CH);
  const int ch = threadIdx.x / LPC, n0 = (threadIdx.x % LPC) * 4;
  const bool live = at.first + ch < s.dg;
  const int64_t c = (int64_t)at.group * s.dg + at.first + ch;
  const int64_t start = at.p * s.part, end = start + s.part < s.t ? start + s.part : s.t;
  const int left = live ? s.n - n0 : 0;
  const f32x4 rate = rates_of(s.rate + c * s.n + n0, left);
  f32x4 h = {0.0f, 0.0f, 0.0f, 0.0f};
  if (kOut) {
    if (s.parts > 1)
      h = load_upto(s.carry + ((at.b * s.parts + at.p) * s.d + c) * s.n + n0, left);
    else if (s.state)
      h = load_upto(s.state + (at.b * s.d + c) * s.n + n0, left);
  }
  const int own = at.first + At::channel();   // the channels this thread fetches
  const f32x4 bias = per_channel(s.bias, (int64_t)at.group * s.dg + own, s.dg - own, 0.0f);
  const f32x4 skip = per_channel(s.skip, (int64_t)at.group * s.dg + own, s.dg - own, 0.0f);
  const int64_t checks = (s.t + kTile - 1) / kTile;
  float span = 0.0f;
  uint32_t begun = 0;
  Sources<T, kOut, false> of(s, at, start);
  Fetched<T, LPC, kFew, kOut, false> next;
  if (start < end) next.fetch(s, of, at.first, end - start);
  for (int64_t tile = start; tile < end; tile += kTile) {
    const int64_t t0 = anew(tile);
    const Fetched<T, LPC, kFew, kOut, false> now = next;
    const uint32_t begins = now.begun(t0, end);
    const int k = At::channel();
    f32x4 x[S::kSlots];
#pragma unroll
    for (int i = 0; i < S::kSlots; ++i) {
      const int tok = At::token(i);
      if (tok >= kTile) break;
      const bool there = t0 + tok < end && at.first + k < s.dg;   // past the end the state stays
      x[i] = values<T>(now.x[i], there ? at.first + k : 0, s.dg);
      const f32x4 dt = values<T>(now.dt[i], there ? at.first + k : 0, s.dg);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float delta = softplus(dt[e] + bias[e]);
        steps[tok][k + e] = there ? f32x2{delta, delta * x[i][e]} : f32x2{0.0f, 0.0f};
      }
    }
    now.put_mix(s, t0, end, mix);
    __syncthreads();
    if (t0 + kTile < end) {
      of.move(kTile);
      next.fetch(s, of, at.first, end - t0 - kTile);
    }
    if (kOut && s.checks)
      store_upto(s.checks + ((at.b * checks + t0 / kTile) * s.d + c) * s.n + n0, h, left);
    begun |= begins;
    const auto walk = [&](auto kind) {
      constexpr int kKind = decltype(kind)::value;
#pragma unroll
      for (int tok = 0; tok < kTile; ++tok) {
        f32x2 st = steps[tok][ch];
        const f32x4 w = *(const f32x4*)&mix[tok][n0];
        if (kKind == kLanes) st.y = left > 0 ? st.y : 0.0f;
        if (kKind >= kBegins) {   // no state before, and no decay that could be infinite and make zero no number
          const bool first = begins >> tok & 1;
          if (first) h = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
          st.x = masked(st.x, first ? 0u : ~0u);
        }
        float y = 0.0f;
        f32x4 r = {0.0f, 0.0f, 0.0f, 0.0f};
        if (kOut) r = *(const f32x4*)&mix[tok][S::NP + n0];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          h[e] = __builtin_fmaf(exp2_of(st.x * rate[e]), h[e], st.y * w[e]);
          if (kKind == kAny) h[e] = e < left ? h[e] : 0.0f;
          if (kOut) y = e ? __builtin_fmaf(r[e], h[e], y) : r[e] * h[e];
        }
        if (kOut)
          steps[tok][ch].x = lanes_sum<LPC>(y);   // the same from each of the channel's lanes
        else
          span += st.x;
      }
    };
    for_kind<kFull>(begins, s.n, walk);
    __syncthreads();
    if (kOut) {
      next.arrive();
#pragma unroll
      for (int i = 0; i < S::kSlots; ++i) {
        const int tok = At::token(i);
        if (tok >= kTile || t0 + tok >= end || at.first + k >= s.dg) continue;
        f32x4 o, z = {0.0f, 0.0f, 0.0f, 0.0f};
        if (s.gate.data) z = values<T>(now.gate[i], at.first + k, s.dg);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          o[e] = steps[tok][k + e].x;
          if (s.skip) o[e] = __builtin_fmaf(skip[e], x[i][e], o[e]);
          if (s.gate.data) o[e] *= z[e] * sigmoid_for<T>(z[e]);
        }
        T* out = (T*)s.out + (at.b * s.t + t0) * s.d + (int64_t)at.group * s.dg + at.first;
        store_upto(const_cast<T*>(row_at(out, tok, anew(s.d))) + k, o, s.dg - at.first - k);
      }
      __syncthreads();
    }
  }
  if (kOut) {
    if (at.p == s.parts - 1) store_upto(s.final_state + (at.b * s.d + c) * s.n + n0, h, left);
  } else {
    const int64_t at_part = at.b * s.parts + at.p;
    store_upto(s.carry + (at_part * s.d + c) * s.n + n0, h, left);
    if (live && n0 == 0) s.spans[at_part * s.d + c] = span;
    if (threadIdx.x == 0 && at.group == 0 && at.first == 0) s.begun[at_part] = begun != 0;
  }
}

// A state carried over a part: exp(rate * the part's sum of delta) of it, `rate` times log2(e), and nothing
// over an episode's beginning. Token by token, an infinite state and a zero one stay what they are, which
// their product with a decay that leaves float32's range would not.
__device__ __forceinline__ float carried(float rate, float span, float state) {
  const float decay = exp2_of(span * rate);
  return state == 0.0f || __builtin_isinf(state) ? state : decay * state;
}

// The states before each part (kBack: the gradients behind it) from the parts' own: a thread for
// each state of a row, over the parts in order.
template <bool kBack>
__global__ __launch_bounds__(kBlock) void join_kernel(Scan s) {
  const int64_t each = (int64_t)s.d * s.n, i = s.item0 + (int64_t)blockIdx.x * kBlock + threadIdx.x;
  if (i >= s.b * each) return;
  const int64_t b = i / each, x = i - b * each, c = x / s.n;
  const float* first = kBack ? s.dfinal : s.state;
  float state = first ? first[i] : 0.0f;
  const float rate = rate_of(s.rate[x]);
  constexpr int kAhead = 32;
  for (int p0 = 0; p0 < s.parts; p0 += kAhead) {
    float own[kAhead], span[kAhead];
    bool begun[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {   // past the last but one, that one again: all loads in flight
      const int at = p0 + k < s.parts - 1 ? p0 + k : s.parts - 2, p = kBack ? s.parts - 1 - at : at;
      own[k] = s.carry[(b * s.parts + p) * each + x];
      span[k] = s.spans[(b * s.parts + p) * s.d + c];
      begun[k] = s.begun[b * s.parts + p];
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int at = p0 + k, p = kBack ? s.parts - 1 - at : at;
      if (at < s.parts) s.carry[(b * s.parts + p) * each + x] = state;
      state = (begun[k] ? 0.0f : carried(rate, span[k], state)) + own[k];
    }
  }
}

// The gradient that a part passes to the states before it where none reaches it from behind.
template <class T, int LPC, bool kFew>
__global__ __launch_bounds__((Shape<LPC, kFew>::kThreads)) void passed_kernel(Scan s) {
  using S = Shape<LPC, kFew>;
  using At = Slots<LPC, kFew>;
  __shared__ __attribute__((aligned(16))) f32x2 steps[kTile][S::CH];      // delta, dy
  __shared__ __attribute__((aligned(16))) float mix[kTile][2 * S::NP];
  Place at = place_of(s, s.item0 + blockIdx.x, s.parts - 1, S::CH);
  at.p += 1;
  const int ch = threadIdx.x / LPC, n0 = (threadIdx.x % LPC) * 4;
  const bool live = at.first + ch < s.dg;
  const int64_t c = (int64_t)at.group * s.dg + at.first + ch;
  const int64_t start = at.p * s.part, end = start + s.part < s.t ? start + s.part : s.t;
  const int left = live ? s.n - n0 : 0;
  const f32x4 rate = rates_of(s.rate + c * s.n + n0, left);
  f32x4 g = {0.0f, 0.0f, 0.0f, 0.0f};
  const int own = at.first + At::channel();
  const f32x4 bias = per_channel(s.bias, (int64_t)at.group * s.dg + own, s.dg - own, 0.0f);
  float span = 0.0f;
  uint32_t begun = 0;
  int64_t t0 = start + (end - start - 1) / kTile * kTile;
  Sources<T, true, true> of(s, at, t0);
  Fetched<T, LPC, kFew, true, true> next;
  next.fetch(s, of, at.first, end - t0);
  for (int64_t tile = t0; tile >= start; tile -= kTile) {
    const int64_t t0 = anew(tile);
    const Fetched<T, LPC, kFew, true, true> now = next;
    const uint32_t begins = now.begun(t0, end);
    const int k = At::channel();
#pragma unroll
    for (int i = 0; i < S::kSlots; ++i) {
      const int tok = At::token(i);
      if (tok >= kTile) break;
      const bool there = t0 + tok < end && at.first + k < s.dg;
      const int c0 = there ? at.first + k : 0;
      const f32x4 dt = values<T>(now.dt[i], c0, s.dg);
      f32x4 dy = values<T>(now.dout[i], c0, s.dg);
      if (s.gate.data) {
        const f32x4 z = values<T>(now.gate[i], c0, s.dg);
#pragma unroll
        for (int e = 0; e < 4; ++e) dy[e] *= z[e] * sigmoid_for<T>(z[e]);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e)
        steps[tok][k + e] = there ? f32x2{softplus(dt[e] + bias[e]), dy[e]} : f32x2{0.0f, 0.0f};
    }
    now.put_mix(s, t0, end, mix);
    __syncthreads();
    if (t0 - kTile >= start) {
      of.move(-kTile);
      next.fetch(s, of, at.first, end - t0 + kTile);
    }
    begun |= begins;
#pragma unroll
    for (int tok = kTile - 1; tok >= 0; --tok) {
      const f32x2 st = steps[tok][ch];
      const f32x4 r = *(const f32x4*)&mix[tok][S::NP + n0];
#pragma unroll
      for (int e = 0; e < 4; ++e) g[e] = exp2_of(st.x * rate[e]) * __builtin_fmaf(r[e], st.y, g[e]);
      if (begins >> tok & 1) g = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      span += st.x;
    }
    __syncthreads();
  }
  const int64_t at_part = at.b * s.parts + at.p;
  store_upto(s.carry + (at_part * s.d + c) * s.n + n0, g, left);
  if (live && n0 == 0) s.spans[at_part * s.d + c] = span;
  if (threadIdx.x == 0 && at.group == 0 && at.first == 0) s.begun[at_part] = begun != 0;
}

// The gradients of one part for a block of channels, tile by tile from its end: the tile's states
// again from the one kept before it, decays and what they leave in registers, then back through them.
//
//   g_t = read dy + a_{t+1} g_{t+1}     dread = sum_c h dy        dwrite = sum_c g delta x
//   dx = skip dy + delta sum_n g write  ddelta = sum_n g (rate a h_{t-1} + x write)
//   drate = sum g a h_{t-1} delta       ddt = ddelta sigmoid(dt + bias)
//
// Sums over a channel's states stay within its lanes; sums over channels go lane by lane within the
// wave, then through LDS, then (dmix) over the blocks of a group.
//
// Bound by instruction issue at the two waves a SIMD that 128 registers of decays and states leave (a vector
// one 81 % of the time, 120 a token for 16 channels of 16 states): 1,100 to 1,200 us for 4,096 x 128 tokens of 128
// channels, float32, of which the sums over channels take some 190, the exponentials 155 and the outputs 165. Among
// them are the reads of 134 to 181 scalars that spill into vector lanes, none in the walks. Vector registers spill
// in float32 with two lanes a channel, 6 to 12 of them, and 2 with eight or 16 lanes, few channels and all states:
// 1,024 x 128 x 128 forwards and backwards 326 us for n = 8 where bfloat16, without, takes 246.
// Before the next tile's loads were waited for ahead of the outputs' stores, and its addresses kept from tile to
// tile, it took 1,290; then, three waves with the decays computed again instead of held 1,340, tiles of
// eight tokens with three waves 1,620.
template <class T, int LPC, bool kFew, bool kFull>
__global__ __launch_bounds__((Shape<LPC, kFew>::kThreads), 2) void backward_kernel(Scan s) {
  using S = Shape<LPC, kFew>;
  using At = Slots<LPC, kFew>;
  // delta, delta x, dy; then delta, sum g write, sum g rate a h_{t-1} / ln 2, sum read h
  __shared__ __attribute__((aligned(16))) f32x4 steps[kTile][S::CH];
  // of each slot, for its outputs: x, dy, the slope of softplus, dout times that of the gate's silu
  __shared__ __attribute__((aligned(16))) f32x4 held[4][kTile * S::CH / 4];
  __shared__ __attribute__((aligned(16))) float mix[kTile][2 * S::NP];
  __shared__ __attribute__((aligned(16))) float sums[S::kWaves][kTile][2 * S::NP];
  const Place at = place_of(s, s.item0 + blockIdx.x, s.parts, S::CH);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int ch = threadIdx.x / LPC, n0 = (threadIdx.x % LPC) * 4;
  const bool live = at.first + ch < s.dg;
  const int64_t c = (int64_t)at.group * s.dg + at.first + ch;
  const int64_t start = at.p * s.part, end = start + s.part < s.t ? start + s.part : s.t;
  const int left = live ? s.n - n0 : 0;
  const f32x4 rate = rates_of(s.rate + c * s.n + n0, left);
  f32x4 g = {0.0f, 0.0f, 0.0f, 0.0f}, drate = g;
  if (s.parts > 1)
    g = load_upto(s.carry + ((at.b * s.parts + at.p) * s.d + c) * s.n + n0, left);
  else if (s.dfinal)
    g = load_upto(s.dfinal + (at.b * s.d + c) * s.n + n0, left);
  const int own = at.first + At::channel();   // the channels this thread fetches
  // out of the registers: of those channels dt_bias and skip, and of this thread the sums of their gradients
  __shared__ __attribute__((aligned(16))) f32x4 params[2][S::CH / 4], grads[2][S::kThreads];
  if (threadIdx.x < S::CH / 4) {
    params[0][threadIdx.x] = per_channel(s.bias, (int64_t)at.group * s.dg + own, s.dg - own, 0.0f);
    params[1][threadIdx.x] = per_channel(s.skip, (int64_t)at.group * s.dg + own, s.dg - own, 0.0f);
  }
  grads[0][threadIdx.x] = grads[1][threadIdx.x] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  __syncthreads();
  const int64_t checks = (s.t + kTile - 1) / kTile;
  const int64_t t0 = end > start ? start + (end - start - 1) / kTile * kTile : start;
  Sources<T, true, true> of(s, at, t0);
  Fetched<T, LPC, kFew, true, true> next;
  // the states before each tile, of the last ones where there are none
  const int c_in = at.first + ch < s.dg ? at.first + ch : 0, n_in = n0 < s.n ? n0 : 0;
  const float* check = s.checks + ((at.b * checks + t0 / kTile) * s.d + (int64_t)at.group * s.dg) * s.n;
  const auto fetch_check = [&]() { return fetch4(check + c_in * s.n, n_in, s.n); };
  f32x4 h_next = {0.0f, 0.0f, 0.0f, 0.0f};
  if (end > start) {
    next.fetch(s, of, at.first, end - t0);
    h_next = fetch_check();
  }
  for (int64_t tile = t0; end > start && tile >= start; tile -= kTile) {
    const int64_t t0 = anew(tile);
    uint32_t begun;
    const int k = At::channel();
    {
      const Fetched<T, LPC, kFew, true, true>& now = next;
      begun = now.begun(t0, end);
      const f32x4 bias = params[0][k / 4];
#pragma unroll
      for (int i = 0; i < S::kSlots; ++i) {
        const int tok = At::token(i), slot = tok * (S::CH / 4) + k / 4;
        if (tok >= kTile) break;
        const bool there = t0 + tok < end && at.first + k < s.dg;
        const int c0 = there ? at.first + k : 0;
        const f32x4 x = values<T>(now.x[i], c0, s.dg), dt = values<T>(now.dt[i], c0, s.dg);
        const f32x4 dout = values<T>(now.dout[i], c0, s.dg);
        f32x4 dy = dout, slope, of_gate;
        if (s.gate.data) {
          const f32x4 z = values<T>(now.gate[i], c0, s.dg);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float one = sigmoid_for<T>(z[e]);
            dy[e] = dout[e] * (z[e] * one);
            of_gate[e] = dout[e] * (one * __builtin_fmaf(z[e], 1.0f - one, 1.0f));
          }
          held[3][slot] = of_gate;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const Softplus delta(dt[e] + bias[e]);
          slope[e] = delta.slope;
          steps[tok][k + e] = there ? f32x4{delta.value, delta.value * x[e], dy[e], 0.0f} : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }
        held[0][slot] = x, held[1][slot] = dy, held[2][slot] = slope;
      }
      now.put_mix(s, t0, end, mix);
    }
    f32x4 h = values<float>(h_next, n_in, s.n);
    if (left <= 0) h = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    __syncthreads();
    if (t0 - kTile >= start) {
      of.move(-kTile);
      check -= (int64_t)s.d * s.n;
      next.fetch(s, of, at.first, end - t0 + kTile);
      h_next = fetch_check();
    }
    const auto walk = [&](auto kind) {
      constexpr int kKind = decltype(kind)::value;
      f32x4 a[kTile], kept[kTile];   // of the state before: its decay, and what is left of it
#pragma unroll
      for (int tok = 0; tok < kTile; ++tok) {
        f32x2 st = *(const f32x2*)&steps[tok][ch];
        const f32x4 w = *(const f32x4*)&mix[tok][n0];
        const bool begins = kKind >= kBegins && (begun >> tok & 1);
        if (kKind == kLanes) st.y = left > 0 ? st.y : 0.0f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          a[tok][e] = exp2_of(st.x * rate[e]);
          kept[tok][e] = begins ? 0.0f : a[tok][e] * h[e];
          h[e] = __builtin_fmaf(st.y, w[e], kept[tok][e]);
          if (kKind == kAny) h[e] = e < left ? h[e] : 0.0f;
        }
        if (tok % 4 == 3) __builtin_amdgcn_sched_barrier(0);   // loads moved further ahead would spill
      }
#pragma unroll
      for (int tok = kTile - 1; tok >= 0; --tok) {
        f32x4 st = steps[tok][ch];
        const f32x4 w = *(const f32x4*)&mix[tok][n0], r = *(const f32x4*)&mix[tok][S::NP + n0];
        float y = 0.0f, into = 0.0f, dd = 0.0f, v[8];
        const bool begins = kKind >= kBegins && (begun >> tok & 1);
        const uint32_t owing = begins ? 0u : ~0u;   // the state before owes nothing where an episode begins
        const float delta = masked(st.x, owing);
        if (kKind == kLanes) st.y = left > 0 ? st.y : 0.0f, st.z = left > 0 ? st.z : 0.0f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float state = __builtin_fmaf(st.y, w[e], kept[tok][e]);
          g[e] = __builtin_fmaf(r[e], st.z, g[e]);
          if (kKind == kAny) state = e < left ? state : 0.0f, g[e] = e < left ? g[e] : 0.0f;
          y = e ? __builtin_fmaf(r[e], state, y) : r[e] * state;
          into = e ? __builtin_fmaf(g[e], w[e], into) : g[e] * w[e];
          v[e] = g[e] * st.y;
          v[4 + e] = state * st.z;
          // of what is left of the state before, whose size may be far below the state's: kept by itself,
          // as their difference would lose its last bits. That is zero where an episode begins, but zero
          // times an infinite g or delta is no number
          const float through = masked(g[e], owing) * kept[tok][e];
          drate[e] = __builtin_fmaf(through, delta, drate[e]);
          dd = e ? __builtin_fmaf(through, rate[e], dd) : through * rate[e];
          g[e] = begins ? 0.0f : g[e] * a[tok][e];
        }
        y = lanes_sum<LPC>(y);
        into = lanes_sum<LPC>(into);
        dd = lanes_sum<LPC>(dd);
        steps[tok][ch] = f32x4{st.x, into, dd, y};
        Across<LPC>::sum(v, lane);
#pragma unroll
        for (int kk = 0; kk < Across<LPC>::kLeft; ++kk) {
          const int id = Across<LPC>::id(lane, kk);
          sums[wave][tok][(id >> 2) * S::NP + n0 + (id & 3)] = v[kk];
        }
        if (tok % 4 == 0) __builtin_amdgcn_sched_barrier(0);
      }
    };
    for_kind<kFull>(begun, s.n, walk);
    __syncthreads();
    next.arrive();
    settle(h_next);
#pragma unroll
    for (int i = 0; i < S::kSlots; ++i) {
      const int tok = At::token(i), slot = tok * (S::CH / 4) + k / 4;
      if (tok >= kTile || t0 + tok >= end || at.first + k >= s.dg) continue;
      const f32x4 x = held[0][slot], dy = held[1][slot], slope = held[2][slot], skip = params[1][k / 4];
      f32x4 dx, ddt, dgate, dskip = grads[0][threadIdx.x];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const f32x4 st = steps[tok][k + e];
        dx[e] = st.x * st.y, dgate[e] = st.w;
        if (s.skip) {
          dx[e] = __builtin_fmaf(skip[e], dy[e], dx[e]);
          dgate[e] = __builtin_fmaf(skip[e], x[e], dgate[e]);
        }
        ddt[e] = __builtin_fmaf(st.z, kLn2, st.y * x[e]) * slope[e];
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) dskip[e] = __builtin_fmaf(dy[e], x[e], dskip[e]);
      grads[0][threadIdx.x] = dskip;
      grads[1][threadIdx.x] += ddt;
      const int64_t col = (int64_t)at.group * s.dg + at.first;
      const int64_t row = (at.b * s.t + t0) * s.d + col;
      const int own_left = s.dg - at.first - k;
      const int64_t to = (int64_t)tok * anew(s.d) + row + k;
      store_upto((T*)s.dx + to, dx, own_left);
      store_upto((T*)s.ddt + to, ddt, own_left);
      if (s.gate.data) {
        const f32x4 of_gate = held[3][slot];
        store_upto((T*)s.dgate + to, dgate * of_gate, own_left);
      }
    }
#pragma unroll
    for (int i = 0; i < S::kMixSlots; ++i) {
      const int tok = At::mix_token(i), part = At::mix_part(), n = At::mix_state();
      if (tok >= kTile || t0 + tok >= end) continue;
      f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int w = 0; w < S::kWaves; ++w) sum += *(const f32x4*)&sums[w][tok][part * 4];
      const int64_t row = (at.b * s.t + t0) * s.g + at.group;
      if (s.tiles > 1) {
        float* to = s.dmix + ((int64_t)(at.first / S::CH) * (s.b * s.t * s.g) + row) * (2 * S::NP);
        *(f32x4*)(to + (int64_t)tok * anew(s.g * (2 * S::NP)) + part * 4) = sum;
      } else {
        T* to = (T*)(part < LPC ? s.dwrite : s.dread) + row * s.n;
        store_upto(to + (int64_t)tok * anew(s.g * s.n) + n, sum, s.n - n);
      }
    }
    __syncthreads();
  }
  const int64_t at_part = at.b * s.parts + at.p;
  if (at.p == 0) store_upto(s.dstate + (at.b * s.d + c) * s.n + n0, g, left);
  float* params_to = s.dparams + at_part * ((int64_t)s.d * (s.n + 2));
  store_upto(params_to + c * s.n + n0, drate, left);
  // the threads of the same four channels, one after another
  constexpr int kQuads = S::CH / 4;
  if (threadIdx.x < 2 * kQuads) {
    const int which = threadIdx.x / kQuads, quad = threadIdx.x % kQuads, of = at.first + quad * 4;
    f32x4 sum = grads[which][quad];
    for (int i = 1; i < S::kThreads / kQuads; ++i) sum += grads[which][quad + i * kQuads];
    store_upto(params_to + (int64_t)s.d * (s.n + which) + (int64_t)at.group * s.dg + of, sum, s.dg - of);
  }
}

// The sums over a group's blocks of channels, rounded to the result's type: four values a thread.
template <class T, int LPC>
__global__ __launch_bounds__(kBlock) void mix_sums_kernel(Scan s) {
  constexpr int NP = 4 * LPC;
  const int64_t rows = s.b * s.t * s.g, i = s.item0 + (int64_t)blockIdx.x * kBlock + threadIdx.x, row = i / (2 * LPC);
  if (row >= rows) return;
  const int part = (int)(i % (2 * LPC)), n = part % LPC * 4;
  f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int k0 = 0; k0 < s.tiles; k0 += 4) {
    f32x4 x[4];
#pragma unroll
    for (int k = 0; k < 4; ++k)
      x[k] = *(const f32x4*)(s.dmix + ((int64_t)(k0 + k < s.tiles ? k0 + k : k0) * rows + row) * (2 * NP) + part * 4);
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (k0 + k < s.tiles) sum += x[k];
  }
  store_upto((T*)(part < LPC ? s.dwrite : s.dread) + row * s.n + n, sum, s.n - n);
}

// One token of every environment: LPC lanes a channel, each with four states, which are read once and
// written once, bound by that. A thread takes its channel of kEnvs environments, so that as many states are
// in flight. Medians over replays of a graph, states in turn, one environment a thread and four: 4,096 x 512 x 16
// with bfloat16 rows 82.3 and 79.0 us (285 MB, 3.6 TB/s), 8,192 of them 158.7 and 146.8; with float32 rows, where
// registers for four leave fewer waves, 91.8 and 97.7 (302 MB, 3.3 TB/s), 179.8 and 186.4. next may be state itself:
// a thread writes only what it has read.
struct Step {
  const void *x, *dt, *gate, *write, *read;
  int64_t x_s, dt_s, gate_s, write_s, write_sg, read_s, read_sg, reset_s;
  const float *rate, *skip, *bias, *state;
  const uint8_t* reset;
  void* out;
  float* next;
  int64_t count, items, item0;   // count: environments; items: channels of groups of kEnvs
  int32_t d, n, dg;
};

template <class T, int LPC, int kEnvs>
__global__ __launch_bounds__(kBlock) void step_kernel(Step s) {
  const int64_t item = s.item0 + (int64_t)blockIdx.x * (kBlock / LPC) + threadIdx.x / LPC;
  if (item >= s.items) return;   // all of a channel's lanes
  const int64_t env0 = (int64_t)((uint32_t)item / (uint32_t)s.d) * kEnvs;
  const int c = (int)(item % (uint32_t)s.d), group = c / s.dg, n0 = (threadIdx.x % LPC) * 4, left = s.n - n0;
  f32x4 h[kEnvs];
  typename Raw<T>::type w[kEnvs], r[kEnvs];
  T x[kEnvs], dt[kEnvs], z[kEnvs];
  uint8_t begins[kEnvs];
  const int from = n0 < s.n ? n0 : 0;
#pragma unroll
  for (int k = 0; k < kEnvs; ++k) {   // past the last environment, that one again: all loads in flight
    const int64_t env = env0 + k < s.count ? env0 + k : s.count - 1;
    h[k] = fetch4(s.state + (env * s.d + c) * s.n, from, s.n);
    w[k] = fetch4((const T*)s.write + env * s.write_s + group * s.write_sg, from, s.n);
    r[k] = fetch4((const T*)s.read + env * s.read_s + group * s.read_sg, from, s.n);
    x[k] = ((const T*)s.x)[env * s.x_s + c];
    dt[k] = ((const T*)s.dt)[env * s.dt_s + c];
    z[k] = s.gate ? ((const T*)s.gate)[env * s.gate_s + c] : (T)0.0f;
    begins[k] = s.reset ? s.reset[env * s.reset_s] : 0;
  }
  const f32x4 rate = rates_of(s.rate + (int64_t)c * s.n + n0, left);
  const float bias = s.bias ? s.bias[c] : 0.0f, skip = s.skip ? s.skip[c] : 0.0f;
#pragma unroll
  for (int k = 0; k < kEnvs; ++k) {
    if (env0 + k >= s.count) break;
    const float delta = softplus((float)dt[k] + bias), du = delta * (float)x[k];
    f32x4 state = values<float>(h[k], from, s.n), wk = values<T>(w[k], from, s.n), rk = values<T>(r[k], from, s.n);
    if (n0 >= s.n) wk = rk = state = f32x4{0.0f, 0.0f, 0.0f, 0.0f};   // a lane without states
    float y = 0.0f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float own = du * wk[e];
      state[e] = begins[k] ? own : __builtin_fmaf(exp2_of(delta * rate[e]), state[e], own);
      state[e] = e < left ? state[e] : 0.0f;   // zero times an infinity
      y = __builtin_fmaf(rk[e], state[e], y);
    }
    store_upto(s.next + ((env0 + k) * s.d + c) * s.n + n0, state, left);
    y = lanes_sum<LPC>(y);
    if (n0 == 0) {
      if (s.skip) y = __builtin_fmaf(skip, (float)x[k], y);
      if (s.gate) y *= (float)z[k] * sigmoid_for<T>((float)z[k]);
      ((T*)s.out)[(env0 + k) * s.d + c] = (T)y;
    }
  }
}

namespace {
bool dims_ok(int32_t dtype, int64_t d, int64_t n, int64_t g) {
  return (dtype == 0 || dtype == 1) && d >= 1 && d <= 65536 && n >= 1 && n <= kMaxStates && g >= 1 && g <= d && d % g == 0;
}

bool sequence_ok(int32_t dtype, int64_t b, int64_t t, int32_t d, int32_t n, int32_t g) {
  return dims_ok(dtype, d, n, g) && b >= 0 && b <= 0x7FFFFFFF && t >= 0 && t <= 0x7FFFFFFF && b * d <= 0x7FFFFFFF;
}

int64_t blocks_of(const Scan& s, int64_t parts) { return s.b * parts * s.g * s.tiles; }

// Sizes, and the parts of a row: as many as fill the card with the waves that a CU holds of the pass, 16
// forwards and 8 backwards, no part below 64 tokens; none from more than four waves a CU on, where every token is
// walked twice to fill what little of the card is free. Rows of 2,048 x 512 x 16, bfloat16, in parts and without, in us:
// 32 rows, the last in parts, 277 and 331 (forwards and backwards 1,000 and 1,150); 33 rows, the first without, 371
// and 407 (1,459 and 1,507), 48 rows 428 and 409 (1,533 and 1,524), 64 rows 495 and 411 (1,610 and 1,535).
int plan(Scan* s, int64_t b, int64_t t, int32_t d, int32_t n, int32_t g, bool back) {
  int cus = 0;
  const int status = device_cus(&cus);
  if (status != HIPENVS_OK) return status;
  const int lpc = lanes_of(n), ch = channels_of(lpc, few_channels(d / g));
  s->b = b, s->t = t, s->d = d, s->n = n, s->g = g, s->dg = d / g;
  s->tiles = (s->dg + ch - 1) / ch;
  const int64_t waves = b * g * s->tiles * (ch * lpc / 64), want = (int64_t)cus * (back ? 8 : 16);
  int64_t parts = 1;
  if (waves > 0 && waves <= (int64_t)cus * 4) {
    parts = want / waves;
    if (parts > t / 64) parts = t / 64;
    if (parts < 1) parts = 1;
  }
  s->part = ((t + parts - 1) / parts + kTile - 1) / kTile * kTile;
  if (s->part < kTile) s->part = kTile;
  s->parts = t > 0 ? (int32_t)((t + s->part - 1) / s->part) : 1;
  return HIPENVS_OK;
}

int64_t round16(int64_t x) { return (x + 15) / 16 * 16; }

// Where the states between the parts lie in `workspace`; the bytes used.
int64_t lay_parts(Scan* s, char* at) {
  if (s->parts <= 1) return 0;
  const int64_t carry = round16(s->b * s->parts * s->d * s->n * 4), spans = round16(s->b * s->parts * s->d * 4);
  s->carry = (float*)at;
  s->spans = (float*)(at + carry);
  s->begun = (uint8_t*)(at + carry + spans);
  return carry + spans + round16(s->b * s->parts);
}

// The same of the backward pass, with its partial sums; *between is what the columns' sums need.
int64_t lay_back(Scan* s, char* at, float** between) {
  int64_t used = lay_parts(s, at);
  const int np = 4 * lanes_of(s->n);
  s->dmix = (float*)(at + used);
  if (s->tiles > 1) used += round16(s->tiles * s->b * s->t * s->g * 2 * np * 4);
  s->dparams = (float*)(at + used);
  const int64_t rows = s->b * s->parts, width = (int64_t)s->d * (s->n + 2);
  used += round16(rows * width * 4);
  *between = (float*)(at + used);
  return used + column_sums_bytes(rows, width);
}

template <class F>
int in_launches(Scan s, int64_t blocks, int threads, const F& launch) {
  const int64_t most = kMostThreads / threads;
  for (s.item0 = 0; s.item0 < blocks; s.item0 += most) {
    launch(s, dim3((unsigned)(blocks - s.item0 < most ? blocks - s.item0 : most)));
    const int status = launch_status();
    if (status != HIPENVS_OK) return status;
  }
  return HIPENVS_OK;
}

template <class F>
int for_lanes(int lpc, const F& f) {
  switch (lpc) {
    case 2: return f(std::integral_constant<int, 2>());
    case 4: return f(std::integral_constant<int, 4>());
    case 8: return f(std::integral_constant<int, 8>());
    default: return f(std::integral_constant<int, 16>());
  }
}

// f(lanes of a channel, whether groups have few channels, whether n is all of the lanes' states)
template <class F>
int for_shape(const Scan& s, const F& f) {
  return for_lanes(lanes_of(s.n), [&](auto lanes) {
    const bool full = s.n == 4 * decltype(lanes)::value;
    if (few_channels(s.dg))
      return full ? f(lanes, std::true_type(), std::true_type()) : f(lanes, std::true_type(), std::false_type());
    return full ? f(lanes, std::false_type(), std::true_type()) : f(lanes, std::false_type(), std::false_type());
  });
}

template <bool kBack>
int join(const Scan& s, hipStream_t stream) {
  Scan one = s;
  const int64_t items = s.b * s.d * s.n;
  for (one.item0 = 0; one.item0 < items; one.item0 += kMostThreads) {
    const int64_t own = items - one.item0 < kMostThreads ? items - one.item0 : kMostThreads;
    hipLaunchKernelGGL(join_kernel<kBack>, dim3(grid_for(own)), dim3(kBlock), 0, stream, one);
    const int status = launch_status();
    if (status != HIPENVS_OK) return status;
  }
  return HIPENVS_OK;
}

template <class T>
int forward(const Scan& s, hipStream_t stream) {
  return for_shape(s, [&](auto lanes, auto few, auto full) {
    constexpr int LPC = decltype(lanes)::value;
    constexpr bool kFew = decltype(few)::value, kFull = decltype(full)::value;
    constexpr int kThreads = Shape<LPC, kFew>::kThreads;
    if (s.parts > 1) {
      int status = in_launches(s, blocks_of(s, s.parts - 1), kThreads, [&](const Scan& a, dim3 grid) {
        hipLaunchKernelGGL((forward_kernel<T, LPC, kFew, kFull, false>), grid, dim3(kThreads), 0, stream, a);
      });
      if (status == HIPENVS_OK) status = join<false>(s, stream);
      if (status != HIPENVS_OK) return status;
    }
    return in_launches(s, blocks_of(s, s.parts), kThreads, [&](const Scan& a, dim3 grid) {
      hipLaunchKernelGGL((forward_kernel<T, LPC, kFew, kFull, true>), grid, dim3(kThreads), 0, stream, a);
    });
  });
}

template <class T>
int backward(const Scan& s, hipStream_t stream) {
  const int walked = for_shape(s, [&](auto lanes, auto few, auto full) {
    constexpr int LPC = decltype(lanes)::value;
    constexpr bool kFew = decltype(few)::value, kFull = decltype(full)::value;
    constexpr int kThreads = Shape<LPC, kFew>::kThreads;
    if (s.parts > 1) {
      int status = in_launches(s, blocks_of(s, s.parts - 1), kThreads, [&](const Scan& a, dim3 grid) {
        hipLaunchKernelGGL((passed_kernel<T, LPC, kFew>), grid, dim3(kThreads), 0, stream, a);
      });
      if (status == HIPENVS_OK) status = join<true>(s, stream);
      if (status != HIPENVS_OK) return status;
    }
    return in_launches(s, blocks_of(s, s.parts), kThreads, [&](const Scan& a, dim3 grid) {
      hipLaunchKernelGGL((backward_kernel<T, LPC, kFew, kFull>), grid, dim3(kThreads), 0, stream, a);
    });
  });
  if (walked != HIPENVS_OK || s.tiles <= 1 || s.t == 0) return walked;
  return for_lanes(lanes_of(s.n), [&](auto lanes) {
    constexpr int LPC = decltype(lanes)::value;
    Scan one = s;
    const int64_t items = s.b * s.t * s.g * 2 * LPC;
    for (one.item0 = 0; one.item0 < items; one.item0 += kMostThreads) {
      const int64_t own = items - one.item0 < kMostThreads ? items - one.item0 : kMostThreads;
      hipLaunchKernelGGL((mix_sums_kernel<T, LPC>), dim3(grid_for(own)), dim3(kBlock), 0, stream, one);
      const int status = launch_status();
      if (status != HIPENVS_OK) return status;
    }
    return (int)HIPENVS_OK;
  });
}

// Whether the strides of t (of dout too, where `back`) fit the kernels' 32 bits.
bool near(const int64_t* st, bool back) {
  for (const int i : {1, 3, 5, 7, 10, 13, 15})
    if ((i < 15 || back) && (st[i] > 0x7FFFFFFF || st[i] < -0x7FFFFFFF)) return false;
  return true;
}

// x, dt, gate (and dout): b, t of each; write, read: b, t, g of each; reset: b, t.
void strided(Scan* s, const int64_t* st, bool back) {
  s->x.sb = st[0], s->x.st = st[1], s->dt.sb = st[2], s->dt.st = st[3], s->gate.sb = st[4], s->gate.st = st[5];
  s->write.sb = st[6], s->write.st = st[7], s->write.sg = st[8];
  s->read.sb = st[9], s->read.st = st[10], s->read.sg = st[11];
  s->reset_sb = st[12], s->reset_st = st[13];
  if (back) s->dout.sb = st[14], s->dout.st = st[15];
}
}  // namespace

}  // namespace scan
}  // namespace hipenvs

using namespace hipenvs;
using namespace hipenvs::scan;

extern "C" int64_t hipenvs_selective_scan_workspace_bytes(int32_t which, int64_t b, int64_t t, int32_t d, int32_t n,
                                                          int32_t g) {
  if (!sequence_ok(0, b, t, d, n, g) || which < 0 || which > 2) return -1;
  if (b == 0) return 0;
  if (which == 1) return b * ((t + kTile - 1) / kTile) * d * n * (int64_t)sizeof(float);
  Scan s = {};
  if (plan(&s, b, t, d, n, g, which == 2) != HIPENVS_OK) return -1;
  float* between = nullptr;
  return which == 0 ? lay_parts(&s, nullptr) : lay_back(&s, nullptr, &between);
}

extern "C" int hipenvs_selective_scan(int32_t dtype, const void* x, const void* dt, const float* rate,
                                      const void* write, const void* read, const float* skip, const void* gate,
                                      const float* dt_bias, const float* state, const uint8_t* reset,
                                      const int64_t* strides, void* out, float* final_state, float* checks, int64_t b,
                                      int64_t t, int32_t d, int32_t n, int32_t g, void* workspace,
                                      int64_t workspace_bytes, hipenvs_stream_t stream) {
  if (!sequence_ok(dtype, b, t, d, n, g)) return HIPENVS_E_ARG;
  if (b == 0) return HIPENVS_OK;
  if (!rate || !final_state || (t > 0 && (!x || !dt || !write || !read || !out || !strides))) return HIPENVS_E_ARG;
  Scan s = {};
  const int status = plan(&s, b, t, d, n, g, false);
  if (status != HIPENVS_OK) return status;
  const int64_t need = lay_parts(&s, (char*)workspace);
  if (need > 0 && (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < need)) return HIPENVS_E_ARG;
  if (t > 0 && !near(strides, false)) return HIPENVS_E_ARG;
  static const int64_t none[14] = {};
  s.x.data = x, s.dt.data = dt, s.gate.data = t > 0 ? gate : nullptr, s.write.data = write, s.read.data = read;
  strided(&s, t > 0 ? strides : none, false);
  s.rate = rate, s.skip = skip, s.bias = dt_bias, s.state = state, s.reset = reset;
  s.out = out, s.final_state = final_state, s.checks = checks;
  return dtype == 1 ? forward<__bf16>(s, as_stream(stream)) : forward<float>(s, as_stream(stream));
}

extern "C" int hipenvs_selective_scan_backward(int32_t dtype, const void* x, const void* dt, const float* rate,
                                               const void* write, const void* read, const float* skip,
                                               const void* gate, const float* dt_bias, const uint8_t* reset,
                                               const void* dout, const float* dfinal, const float* checks,
                                               const int64_t* strides, void* dx, void* ddt, void* dwrite, void* dread,
                                               void* dgate, float* dparams, float* dstate, int64_t b, int64_t t,
                                               int32_t d, int32_t n, int32_t g, void* workspace,
                                               int64_t workspace_bytes, hipenvs_stream_t stream) {
  if (!sequence_ok(dtype, b, t, d, n, g)) return HIPENVS_E_ARG;
  if (!dparams) return HIPENVS_E_ARG;
  const int64_t width = (int64_t)d * (n + 2);
  if (b == 0) return column_sums<float>(nullptr, 0, width, 1.0f, dparams, nullptr, as_stream(stream));
  if (!rate || !dstate || (t > 0 && (!x || !dt || !write || !read || !dout || !checks || !dx || !ddt || !dwrite ||
                                     !dread || !strides || (gate && !dgate))))
    return HIPENVS_E_ARG;
  Scan s = {};
  int status = plan(&s, b, t, d, n, g, true);
  if (status != HIPENVS_OK) return status;
  float* between = nullptr;
  const int64_t need = lay_back(&s, (char*)workspace, &between);
  if (need > 0 && (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < need)) return HIPENVS_E_ARG;
  if (t > 0 && !near(strides, true)) return HIPENVS_E_ARG;
  static const int64_t none[16] = {};
  s.x.data = x, s.dt.data = dt, s.gate.data = t > 0 ? gate : nullptr, s.write.data = write, s.read.data = read;
  s.dout.data = dout;
  strided(&s, t > 0 ? strides : none, true);
  s.rate = rate, s.skip = skip, s.bias = dt_bias, s.reset = reset, s.dfinal = dfinal;
  s.checks = const_cast<float*>(checks);
  s.dx = dx, s.ddt = ddt, s.dwrite = dwrite, s.dread = dread, s.dgate = dgate, s.dstate = dstate;
  const hipStream_t on = as_stream(stream);
  status = dtype == 1 ? backward<__bf16>(s, on) : backward<float>(s, on);
  if (status != HIPENVS_OK) return status;
  return column_sums<float>(s.dparams, b * s.parts, width, 1.0f, dparams, between, on);
}

extern "C" int hipenvs_selective_scan_step(int32_t dtype, const void* x, const void* dt, const float* rate,
                                           const void* write, const void* read, const float* skip, const void* gate,
                                           const float* dt_bias, const float* state, const uint8_t* reset,
                                           const int64_t* strides, void* out, float* next_state, int64_t count,
                                           int32_t d, int32_t n, int32_t g, hipenvs_stream_t stream) {
  if (!dims_ok(dtype, d, n, g) || count < 0 || count > 0x7FFFFFFF || count * d > 0x7FFFFFFF) return HIPENVS_E_ARG;
  if (count == 0) return HIPENVS_OK;
  if (!x || !dt || !rate || !write || !read || !state || !strides || !out || !next_state) return HIPENVS_E_ARG;
  int cus = 0;
  const int status = device_cus(&cus);
  if (status != HIPENVS_OK) return status;
  Step s = {x,          dt,         gate,       write,      read,       strides[0], strides[1], strides[2], strides[3],
            strides[4], strides[5], strides[6], strides[7], rate,       skip,       dt_bias,    state,      reset,
            out,        next_state, count,      0,          0,          d,          n,          d / g};
  return for_lanes(lanes_of(n), [&](auto lanes) {
    constexpr int LPC = decltype(lanes)::value, kChannels = kBlock / LPC;
    // four environments a thread for bfloat16 rows where that leaves 32 blocks a CU
    const bool many = dtype == 1 && count * d / 4 >= (int64_t)cus * 32 * kChannels;
    s.items = (many ? (count + 3) / 4 : count) * d;
    const int64_t most = kMostThreads / kBlock * kChannels;
    for (s.item0 = 0; s.item0 < s.items; s.item0 += most) {
      const int64_t own = s.items - s.item0 < most ? s.items - s.item0 : most;
      const dim3 grid((unsigned)((own + kChannels - 1) / kChannels)), block(kBlock);
      if (dtype == 1 && many)
        hipLaunchKernelGGL((step_kernel<__bf16, LPC, 4>), grid, block, 0, as_stream(stream), s);
      else if (dtype == 1)
        hipLaunchKernelGGL((step_kernel<__bf16, LPC, 1>), grid, block, 0, as_stream(stream), s);
      else
        hipLaunchKernelGGL((step_kernel<float, LPC, 1>), grid, block, 0, as_stream(stream), s);
      const int launched = launch_status();
      if (launched != HIPENVS_OK) return launched;
    }
    return (int)HIPENVS_OK;
  });
}
