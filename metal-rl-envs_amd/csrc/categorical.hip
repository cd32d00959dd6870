// Log probabilities of given tokens under rows of logits, with entropies, the most likely tokens, and
// the gradient of the logits. No reference counterpart.
//
//   m = max x, s = sum exp(x - m), w = sum exp(x - m) (x - m)
//   log p(token) = x[token] - m - log s        H = log s - w / s
//   dx_j = dlog_prob ([j = token] - p_j) - dentropy p_j (log p_j + H)
//
// A logit of -inf is a token that is not allowed: it adds nothing to any sum. A row of nothing else
// has log probabilities of -inf, entropy 0 and a gradient of zeros; a row with a NaN or +inf is no
// number throughout. A negative token is none: log probability 0, no gradient of its own.
// Everything is float32 but the logits, which may be bfloat16, and their gradient.
#include "row_ops.h"

namespace hipenvs {
namespace categorical {

using namespace rows;

constexpr int kMaxTop = 64;

struct LogProbs {
  const void* logits;
  const int64_t* tokens;
  int64_t logits_s, rows, v, part;   // part: values of a row that one block takes
  float *log_prob, *entropy, *stats;   // stats (rows, 2): m and log2 s
  float* top_log_prob;               // (rows, top)
  int64_t* top_index;
  float* partial;                    // (rows, parts, 4): m, s, w
  uint64_t* tops;                    // (rows, parts, top)
  int32_t parts, top;
  int64_t item0;
};

// Differences of logits reach -inf, and a zero times that is no number; exp(-160) and
// 2^-160 are 0 in float32. The median of three is one instruction, with a NaN's others where one is a
// NaN; the exponential beside it keeps the NaN.
__device__ __forceinline__ float at_least(float x) { return __builtin_amdgcn_fmed3f(x, -160.0f, __builtin_inff()); }

__device__ __forceinline__ float larger(float a, float b) { return __builtin_amdgcn_fmed3f(a, b, __builtin_inff()); }

// m, s and w of some of a row's values.
struct Sums {
  float m, s, w;

  __device__ __forceinline__ void raise(float to) {
    if (to > m) {
      const float step = at_least(m - to), k = exp2_of(step * kLog2e);
      if (m != -__builtin_inff()) {
        w = k * __builtin_fmaf(s, step, w);
        s *= k;
      }
      m = to;
    }
  }

  // after raise(x): values of which none is above m. The exponential of a NaN keeps it in both sums.
  template <int kCount>
  __device__ __forceinline__ void add(const float (&x)[kCount]) {
    const float base = m == -__builtin_inff() ? 0.0f : m;
#pragma unroll
    for (int i = 0; i < kCount; ++i) {
      const float t = x[i] - base, e = exp2_of(t * kLog2e);
      s += e;
      w = __builtin_fmaf(e, at_least(t), w);
    }
  }

  __device__ __forceinline__ void join(Sums o) {
    raise(o.m);
    o.raise(m);
    s += o.s;
    w += o.w;
  }
};

__device__ __forceinline__ Sums none() { return {-__builtin_inff(), 0.0f, 0.0f}; }

template <int kXor>
__device__ __forceinline__ float from_lane_xor(float v) {
  if constexpr (kXor < 16) return from_xor<kXor>(v);
  else return __shfl_xor(v, kXor);
}

template <int kLanes>
__device__ __forceinline__ Sums joined(Sums a) {
  const auto with = [&](auto step) {
    constexpr int kXor = decltype(step)::value;
    if constexpr (kXor < kLanes)
      a.join({from_lane_xor<kXor>(a.m), from_lane_xor<kXor>(a.s), from_lane_xor<kXor>(a.w)});
  };
  with(std::integral_constant<int, 1>()), with(std::integral_constant<int, 2>()), with(std::integral_constant<int, 4>());
  with(std::integral_constant<int, 8>()), with(std::integral_constant<int, 16>()), with(std::integral_constant<int, 32>());
  return a;
}

// A value and its place as one number: larger ones first, NaN before all, of equals the lowest place.
__device__ __forceinline__ uint64_t ranked(float x, uint32_t index) {
  const uint32_t u = __float_as_uint(x + 0.0f);   // -0 as 0
  const uint32_t key = x != x ? 0xFFFFFFFFu : u & 0x80000000u ? ~u : u | 0x80000000u;
  return (uint64_t)key << 32 | (0xFFFFFFFFu - index);
}

__device__ __forceinline__ uint32_t place_in(uint64_t r) { return 0xFFFFFFFFu - (uint32_t)r; }

__device__ __forceinline__ float value_in(uint64_t r) {
  const uint32_t key = (uint32_t)(r >> 32);
  if (key == 0xFFFFFFFFu) return __builtin_nanf("");
  return __uint_as_float(key & 0x80000000u ? key & 0x7FFFFFFFu : ~key);
}

__device__ __forceinline__ uint64_t lane_value(uint64_t v, int lane) {
  return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32 |
         (uint32_t)__builtin_amdgcn_readlane((int)v, lane);
}

template <int kXor>
__device__ __forceinline__ uint32_t key_from_xor(uint32_t v, int lane) {
  if constexpr (kXor == 32) {
    const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return lane & 32 ? r[0] : r[1];
  } else if constexpr (kXor == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return lane & 16 ? r[0] : r[1];
  } else {
    return __float_as_uint(from_xor<kXor>(__uint_as_float(v)));
  }
}

// One step of a bitonic sort over the wave, largest first in runs of kRun.
template <int kRun, int kXor>
__device__ __forceinline__ void sort_step(uint32_t& v, int lane) {
  const uint32_t o = key_from_xor<kXor>(v, lane);
  const bool larger = ((lane & kXor) == 0) == (kRun == 64 || (lane & kRun) == 0);
  v = larger ? (v > o ? v : o) : (v < o ? v : o);
  if constexpr (kXor > 1) sort_step<kRun, kXor / 2>(v, lane);
}

__device__ __forceinline__ void sort_wave(uint32_t& v, int lane) {
  sort_step<2, 1>(v, lane), sort_step<4, 2>(v, lane), sort_step<8, 4>(v, lane);
  sort_step<16, 8>(v, lane), sort_step<32, 16>(v, lane), sort_step<64, 32>(v, lane);
}

// The lane before's value; 0 in the first.
__device__ __forceinline__ uint64_t from_before(uint64_t v) {
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(v >> 32), 0x138, 0xF, 0xF, false);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x138, 0xF, 0xF, false);
  return (uint64_t)hi << 32 | lo;
}

// The most likely so far, one a lane, in order; empty places are 0.
struct Best {
  uint64_t own, least;   // least: the last that is kept, in all lanes

  // takes each lane's candidate, if it is among the best
  __device__ __forceinline__ void offer(uint64_t candidate, int top, int lane) {
    uint64_t better = __builtin_amdgcn_ballot_w64(candidate > least);
    while (better) {
      const uint64_t v = lane_value(candidate, __builtin_ctzll(better));
      const int at = __popcll(__builtin_amdgcn_ballot_w64(own > v));
      const uint64_t before = from_before(own);
      own = lane < at ? own : lane == at ? v : before;
      least = lane_value(own, top - 1);
      better &= better - 1;
      better &= __builtin_amdgcn_ballot_w64(candidate > least);
    }
  }

  // A batch of candidates, a lane's largest given. At least `top` candidates reach the top-th of the
  // lanes' largest, so the rest of the first batch need no look. The 20 best of 16 rows of 131,071: 13 + 6 us
  // for the parts and their joining, 21 + 12 without this bound.
  template <class F>
  __device__ __forceinline__ void offer_batch(uint64_t largest, int count, int top, int lane, const F& candidate) {
    uint32_t bound = (uint32_t)(least >> 32);
    if (__builtin_amdgcn_ballot_w64((uint32_t)(largest >> 32) >= bound && largest != 0) == 0) return;
    if (least == 0) {
      uint32_t sorted = (uint32_t)(largest >> 32);
      sort_wave(sorted, lane);
      bound = (uint32_t)__builtin_amdgcn_readlane((int)sorted, top - 1);
    }
#pragma unroll
    for (int e = 0; e < count; ++e) {
      const uint64_t c = candidate(e);
      offer((uint32_t)(c >> 32) >= bound ? c : 0, top, lane);
    }
  }
};

// What a row's sums say: its outputs, by one lane.
__device__ __forceinline__ void write_row(const LogProbs& p, int64_t row, Sums a, float chosen, int64_t token) {
  const bool empty = a.m == -__builtin_inff() && a.s == 0.0f;
  const float log_s = __builtin_amdgcn_logf(a.s);   // to the base of 2
  const float l = log_s * kLn2;
  float lp = empty ? -__builtin_inff() : (chosen - a.m) - l;
  if (token >= p.v) lp = __builtin_nanf("");
  p.log_prob[row] = token < 0 ? 0.0f : lp;
  p.entropy[row] = empty ? 0.0f : l - a.w / a.s;
  if (p.stats) {
    p.stats[2 * row] = empty ? 0.0f : a.m;
    p.stats[2 * row + 1] = empty ? __builtin_inff() : log_s;   // every p = 0
  }
}

__device__ __forceinline__ float top_log_prob(uint64_t ranked, Sums a) {
  const float x = value_in(ranked);
  if (a.m == -__builtin_inff() && a.s == 0.0f) return x;   // every token is out: -inf
  return (x - a.m) - __builtin_amdgcn_logf(a.s) * kLn2;
}

// Short rows: G lanes hold a row in registers, E values each, four next to each other of every 4 G, all loaded
// before any is used. Bound by memory: 2^28 values, forwards and backwards, in rows of 1,000 in 628 us as float32
// (5.1 TB/s) and 338 as bfloat16, in rows of 64 in 611 and 395. Values loaded one by one, each behind a
// comparison and a conversion, took 729 and 749, 904 and 759.
template <class T, int G, int E>
__global__ __launch_bounds__(kBlock) void short_kernel(LogProbs p) {
  const int64_t row = p.item0 + (int64_t)blockIdx.x * (kBlock / G) + threadIdx.x / G;
  const int lane = threadIdx.x % G;
  if (row >= p.rows) return;   // all of a row's lanes
  const T* x = (const T*)p.logits + row * p.logits_s;
  const int v = (int)p.v;
  const int64_t token = p.tokens[row];
  const auto place = [&](int e) { return (e / 4 * G + lane) * 4 + e % 4; };
  typename Raw<T>::type raw[E / 4];
#pragma unroll
  for (int k = 0; k < E / 4; ++k) raw[k] = fetch4(x, place(4 * k), v);
  const bool has = token >= 0 && token < v;
  const T chosen = x[has ? token : 0];
  float own[E];
  Sums a = none();
#pragma unroll
  for (int k = 0; k < E / 4; ++k) {
    const f32x4 y = values<T>(raw[k], place(4 * k), v);
#pragma unroll
    for (int e = 0; e < 4; ++e) own[4 * k + e] = place(4 * k + e) < v ? y[e] : -__builtin_inff();
  }
#pragma unroll
  for (int e = 0; e < E; ++e) a.m = larger(own[e], a.m);
  a.add(own);
  a = joined<G>(a);
  if (lane == 0) write_row(p, row, a, has ? (float)chosen : 0.0f, token);
  uint32_t taken = 0;
  for (int k = 0; k < p.top; ++k) {
    uint64_t best = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const uint64_t r = place(e) < v && !(taken >> e & 1) ? ranked(own[e], place(e)) : 0;
      best = r > best ? r : best;
    }
    uint64_t all = best;
#pragma unroll
    for (int step = 1; step < G; step *= 2) {
      const uint64_t other = __shfl_xor(all, step);
      all = other > all ? other : all;
    }
    const uint32_t at = place_in(all);
    if (at / 4 % G == (uint32_t)lane) taken |= 1u << (at / (4 * G) * 4 + at % 4);
    if (lane == 0) {
      p.top_log_prob[row * p.top + k] = top_log_prob(all, a);
      p.top_index[row * p.top + k] = at;
    }
  }
}

// Four values from i on of a row of at least four, at its end or past it the last four: no branch before
// the load.
template <class T>
__device__ __forceinline__ typename Raw<T>::type fetch_piece(const T* x, uint32_t i, uint32_t v) {
  return *(const typename Raw<T>::any*)(x + (i < v - 4 ? i : v - 4));
}

// What fetch_piece read, kEnd: where the row's end may be among it.
template <class T, bool kEnd>
__device__ __forceinline__ f32x4 piece_values(typename Raw<T>::type raw, uint32_t i, uint32_t v) {
  f32x4 x = __builtin_convertvector(raw, f32x4);
  if (kEnd && i > v - 4) {   // only a row's last thread
    const uint32_t by = i - (v - 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = by == 1 && e < 3 ? x[(e + 1) & 3] : by == 2 && e < 2 ? x[(e + 2) & 3] : by == 3 ? x[3] : x[e];
  }
  return x;
}

// Long rows: a block takes a part of a row, every wave with its own sums and its own best, in batches of
// 16 values a lane, the next one's loads in flight. Bound by memory: 16,384 rows of 40,064 bfloat16 read at
// 5.8 TB/s, rows of odd length, which lie at odd addresses, at 4.5.
template <class T, bool kTop>
__global__ __launch_bounds__(kBlock, kTop ? 4 : 8) void long_kernel(LogProbs p) {
  __shared__ Sums sums[4];
  __shared__ uint64_t best[4][kTop ? kMaxTop : 1];
  constexpr uint32_t kLoads = 4, kStep = kBlock * 4, kBatch = kLoads * kStep;
  const int64_t item = p.item0 + blockIdx.x, row = item / p.parts;
  const int part = (int)(item - row * p.parts), lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const T* x = (const T*)p.logits + row * p.logits_s;
  const uint32_t v = (uint32_t)p.v, first = part * (uint32_t)p.part;
  const uint32_t end = v - first > (uint32_t)p.part ? first + (uint32_t)p.part : v;
  Sums a = none();
  Best b = {0, 0};
  typename Raw<T>::type next[kLoads];
#pragma unroll
  for (uint32_t k = 0; k < kLoads; ++k) next[k] = fetch_piece(x, first + k * kStep + threadIdx.x * 4, v);
  const auto batch = [&](uint32_t at, auto last) {
    constexpr bool kEnd = decltype(last)::value;   // some of the batch may lie past the part
    const uint32_t i = at + threadIdx.x * 4;
    float own[kLoads * 4];
#pragma unroll
    for (uint32_t k = 0; k < kLoads; ++k) {
      const f32x4 y = piece_values<T, kEnd>(next[k], i + k * kStep, v);
#pragma unroll
      for (uint32_t e = 0; e < 4; ++e) own[k * 4 + e] = kEnd && i + k * kStep + e >= end ? -__builtin_inff() : y[e];
    }
    if (!kEnd)
#pragma unroll
      for (uint32_t k = 0; k < kLoads; ++k) next[k] = fetch_piece(x, i + kBatch + k * kStep, v);
    float m = own[0];
#pragma unroll
    for (uint32_t e = 1; e < kLoads * 4; ++e) m = larger(own[e], m);
    a.raise(m);
    a.add(own);
    if constexpr (kTop) {
      const auto candidate = [&](int e) {
        const uint32_t j = i + (uint32_t)(e / 4) * kStep + (uint32_t)(e % 4);
        return !kEnd || j < end ? ranked(own[e], j) : 0;
      };
      uint64_t largest = 0;
#pragma unroll
      for (int e = 0; e < (int)kLoads * 4; ++e) largest = candidate(e) > largest ? candidate(e) : largest;
      b.offer_batch(largest, kLoads * 4, p.top, lane, candidate);
    }
  };
  uint32_t at = first;   // rows end below 2^31
  for (; end - at >= kBatch; at += kBatch) batch(at, std::false_type());
  if (at < end) batch(at, std::true_type());
  a = joined<64>(a);
  if (lane == 0) sums[wave] = a;
  if (kTop && lane < p.top) best[wave][kTop ? lane : 0] = b.own;
  __syncthreads();
  if (wave != 0) return;
  for (int k = 1; k < 4; ++k) {
    a.join(sums[k]);
    if constexpr (kTop) b.offer(lane < p.top ? best[k][lane] : 0, p.top, lane);
  }
  if (p.parts == 1) {
    const int64_t token = p.tokens[row];
    if (lane == 0) write_row(p, row, a, token >= 0 && token < p.v ? (float)x[token] : 0.0f, token);
    if (kTop && lane < p.top) {
      p.top_log_prob[row * p.top + lane] = top_log_prob(b.own, a);
      p.top_index[row * p.top + lane] = place_in(b.own);
    }
    return;
  }
  if (lane == 0) {
    float* to = p.partial + item * 4;
    to[0] = a.m, to[1] = a.s, to[2] = a.w;
  }
  if (kTop && lane < p.top) p.tops[item * p.top + lane] = b.own;
}

// The parts of a row together, a wave for each.
template <class T>
__global__ __launch_bounds__(64) void join_kernel(LogProbs p) {
  const int64_t row = p.item0 + blockIdx.x;
  const int lane = threadIdx.x;
  Sums a = none();
  Best b = {0, 0};
  for (int k0 = 0; k0 < p.parts; k0 += 64) {
    const int k = k0 + lane;
    if (k < p.parts) {
      const float* from = p.partial + (row * p.parts + k) * 4;
      a.join({from[0], from[1], from[2]});
    }
  }
  a = joined<64>(a);
  if (p.top) {
    constexpr int kLoads = 16;
    const int64_t count = (int64_t)p.parts * p.top;
    const uint64_t* from = p.tops + row * count;
    for (int64_t k0 = lane; k0 - lane < count; k0 += kLoads * 64) {
      uint64_t own[kLoads], largest = 0;
#pragma unroll
      for (int e = 0; e < kLoads; ++e) own[e] = from[k0 + e * 64 < count ? k0 + e * 64 : count - 1];
#pragma unroll
      for (int e = 0; e < kLoads; ++e) {
        own[e] = k0 + e * 64 < count ? own[e] : 0;
        largest = own[e] > largest ? own[e] : largest;
      }
      b.offer_batch(largest, kLoads, p.top, lane, [&](int e) { return own[e]; });
    }
  }
  const int64_t token = p.tokens[row];
  if (lane == 0)
    write_row(p, row, a, token >= 0 && token < p.v ? (float)((const T*)p.logits)[row * p.logits_s + token] : 0.0f, token);
  if (lane < p.top) {
    p.top_log_prob[row * p.top + lane] = top_log_prob(b.own, a);
    p.top_index[row * p.top + lane] = place_in(b.own);
  }
}

struct Gradient {
  const void* logits;
  const int64_t* tokens;
  const float *stats, *entropy, *dlog_prob, *dentropy;
  void* dlogits;   // (rows, v) contiguous
  int64_t logits_s, rows, v, item0;
  int32_t pieces;
};

// What a row's gradient takes: dx = chosen dlog_prob - p (dlog_prob + dentropy (log p + H)), the bracket as
// one product and a sum of log2 p.
struct RowGradient {
  float m, log_s, slope, level, dlp;
  int64_t token;

  __device__ __forceinline__ RowGradient(const Gradient& g, int64_t row) {
    m = g.stats[2 * row], log_s = g.stats[2 * row + 1];
    token = g.tokens[row];
    dlp = g.dlog_prob && token >= 0 && log_s != __builtin_inff() ? g.dlog_prob[row] : 0.0f;
    const float dh = g.dentropy ? g.dentropy[row] : 0.0f;
    slope = dh * kLn2;
    level = __builtin_fmaf(dh, g.entropy[row], dlp);
  }

  // a token that is not allowed owes nothing, to an infinite slope or level neither
  __device__ __forceinline__ float of(float x) const {
    const float log2_p = __builtin_fmaf(x - m, kLog2e, -log_s), p = exp2_of(log2_p);
    return p == 0.0f ? 0.0f : -p * __builtin_fmaf(at_least(log2_p), slope, level);
  }
};

template <class T, int G, int E>
__global__ __launch_bounds__(kBlock) void short_gradient_kernel(Gradient g) {
  const int64_t row = g.item0 + (int64_t)blockIdx.x * (kBlock / G) + threadIdx.x / G;
  const int lane = threadIdx.x % G;
  if (row >= g.rows) return;
  const T* x = (const T*)g.logits + row * g.logits_s;
  T* dx = (T*)g.dlogits + row * g.v;
  const int v = (int)g.v;
  typename Raw<T>::type raw[E / 4];
#pragma unroll
  for (int k = 0; k < E / 4; ++k) raw[k] = fetch4(x, (k * G + lane) * 4, v);
  const RowGradient of(g, row);
  const uint32_t token = of.token >= 0 && of.token < v ? (uint32_t)of.token : 0xFFFFFFFFu;
#pragma unroll
  for (int k = 0; k < E / 4; ++k) {
    const int j = (k * G + lane) * 4;
    f32x4 own = values<T>(raw[k], j, v);
#pragma unroll
    for (int e = 0; e < 4; ++e) own[e] = of.of(own[e]);
    const uint32_t at = token - (uint32_t)j;
    if (at < 4)   // one thread of the row
#pragma unroll
      for (uint32_t e = 0; e < 4; ++e) own[e] += at == e ? of.dlp : 0.0f;
    store_upto(dx + j, own, v - j);
  }
}

constexpr int kPiece = 4096;   // values of a row that a block takes

// Bound by memory: 4,093 rows of 40,009 bfloat16 in and out in 98 us, 6.7 TB/s (part of what is read is still
// in the cache from the forward pass). The token's own term is added by the one thread that has it: a
// comparison for every value took 115.

template <class T>
__global__ __launch_bounds__(kBlock) void long_gradient_kernel(Gradient g) {
  const int64_t item = g.item0 + blockIdx.x, row = item / g.pieces, first = (item - row * g.pieces) * kPiece;
  const T* x = (const T*)g.logits + row * g.logits_s;
  T* dx = (T*)g.dlogits + row * g.v;
  const RowGradient of(g, row);
  // a token that is none or past the row is no thread's: they begin below 2^31 + 4096
  const uint32_t token = of.token >= 0 && of.token < g.v ? (uint32_t)of.token : 0xFFFFFFFFu;
  constexpr uint32_t kLoads = kPiece / (kBlock * 4), kStep = kBlock * 4;
  const uint32_t v = (uint32_t)g.v, j0 = (uint32_t)first + threadIdx.x * 4;
  typename Raw<T>::type pieces[kLoads];
#pragma unroll
  for (uint32_t k = 0; k < kLoads; ++k) pieces[k] = fetch_piece(x, j0 + k * kStep, v);
  const auto put = [&](auto last) {
    constexpr bool kEnd = decltype(last)::value;
#pragma unroll
    for (uint32_t k = 0; k < kLoads; ++k) {
      const uint32_t j = j0 + k * kStep;
      if (kEnd && j >= v) break;
      f32x4 own = piece_values<T, kEnd>(pieces[k], j, v);
#pragma unroll
      for (int e = 0; e < 4; ++e) own[e] = of.of(own[e]);
      const uint32_t at = token - j;
      if (at < 4)   // one thread of the row
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e) own[e] += at == e ? of.dlp : 0.0f;
      store_upto(dx + j, own, kEnd ? (int64_t)v - j : 4);
    }
  };
  if (v - (uint32_t)first >= (uint32_t)kPiece)
    put(std::false_type());
  else
    put(std::true_type());
}

namespace {
constexpr int64_t kShort = 1024;   // values of a row that a wave holds in registers

bool sizes_ok(int32_t dtype, int64_t rows, int64_t v, int64_t top) {
  return (dtype == 0 || dtype == 1) && rows >= 0 && rows <= 0x7FFFFFFF && v >= 1 && v <= 0x7FFFFFFF && top >= 0 &&
         top <= kMaxTop && top <= v;
}

// The parts of a long row: as many as give the card eight waves a CU, none below 4,096 values.
int plan(LogProbs* p, int64_t rows, int64_t v) {
  int cus = 0;
  const int status = device_cus(&cus);
  if (status != HIPENVS_OK) return status;
  p->rows = rows, p->v = v;
  int64_t parts = 1;
  if (v > kShort && rows < cus * 2) {
    parts = (cus * 2 + rows - 1) / rows;
    if (parts > (v + 4095) / 4096) parts = (v + 4095) / 4096;
  }
  p->part = ((v + parts - 1) / parts + 3) / 4 * 4;
  p->parts = (int32_t)((v + p->part - 1) / p->part);
  return HIPENVS_OK;
}

int64_t round16(int64_t x) { return (x + 15) / 16 * 16; }

int64_t lay(LogProbs* p, char* at, int32_t top) {
  if (p->parts <= 1) return 0;
  const int64_t partial = round16(p->rows * p->parts * 16);
  p->partial = (float*)at;
  p->tops = (uint64_t*)(at + partial);
  return partial + p->rows * p->parts * top * 8;
}

template <class S, class F>
int in_launches(S s, int64_t blocks, int threads, const F& launch) {
  const int64_t most = kMostThreads / threads;
  for (int64_t done = 0; done < blocks; done += most) {
    launch(s, done, dim3((unsigned)(blocks - done < most ? blocks - done : most)));
    const int status = launch_status();
    if (status != HIPENVS_OK) return status;
  }
  return HIPENVS_OK;
}

// f(lanes of a row, values a lane) for rows of up to kShort values: the fewer lanes, the more rows a wave's
// joins serve, but the further apart lie the values that a load fetches. 2^28 values, forwards and backwards, in
// us, at four a lane, eight and 16, float32 and then bfloat16: rows of 32 747, 676, 914 and 603, 397, 482; of 64
// 761, 611, 650 and 626, 395, 451; of 128 766, 590, 601 and 630, 397, 327; of 256 779, 601, 581 and 654, 404, 311.
template <class F>
int for_short(int64_t v, const F& f) {
  using std::integral_constant;
  if (v <= 4) return f(integral_constant<int, 1>(), integral_constant<int, 4>());
  if (v <= 8) return f(integral_constant<int, 1>(), integral_constant<int, 8>());
  if (v <= 16) return f(integral_constant<int, 2>(), integral_constant<int, 8>());
  if (v <= 32) return f(integral_constant<int, 4>(), integral_constant<int, 8>());
  if (v <= 64) return f(integral_constant<int, 8>(), integral_constant<int, 8>());
  if (v <= 128) return f(integral_constant<int, 8>(), integral_constant<int, 16>());
  if (v <= 256) return f(integral_constant<int, 16>(), integral_constant<int, 16>());
  if (v <= 512) return f(integral_constant<int, 32>(), integral_constant<int, 16>());
  return f(integral_constant<int, 64>(), integral_constant<int, 16>());
}

template <class T>
int forward(const LogProbs& p, hipStream_t stream) {
  if (p.v <= kShort)
    return for_short(p.v, [&](auto lanes, auto values) {
      constexpr int G = decltype(lanes)::value, E = decltype(values)::value, kRows = kBlock / G;
      return in_launches(p, (p.rows + kRows - 1) / kRows, kBlock, [&](LogProbs a, int64_t done, dim3 grid) {
        a.item0 = done * kRows;
        hipLaunchKernelGGL((short_kernel<T, G, E>), grid, dim3(kBlock), 0, stream, a);
      });
    });
  const int status = in_launches(p, p.rows * p.parts, kBlock, [&](LogProbs a, int64_t done, dim3 grid) {
    a.item0 = done;
    if (p.top > 0)
      hipLaunchKernelGGL((long_kernel<T, true>), grid, dim3(kBlock), 0, stream, a);
    else
      hipLaunchKernelGGL((long_kernel<T, false>), grid, dim3(kBlock), 0, stream, a);
  });
  if (status != HIPENVS_OK || p.parts == 1) return status;
  return in_launches(p, p.rows, 64, [&](LogProbs a, int64_t done, dim3 grid) {
    a.item0 = done;
    hipLaunchKernelGGL(join_kernel<T>, grid, dim3(64), 0, stream, a);
  });
}

template <class T>
int gradient(const Gradient& g, hipStream_t stream) {
  if (g.v <= kShort)
    return for_short(g.v, [&](auto lanes, auto values) {
      constexpr int G = decltype(lanes)::value, E = decltype(values)::value, kRows = kBlock / G;
      return in_launches(g, (g.rows + kRows - 1) / kRows, kBlock, [&](Gradient a, int64_t done, dim3 grid) {
        a.item0 = done * kRows;
        hipLaunchKernelGGL((short_gradient_kernel<T, G, E>), grid, dim3(kBlock), 0, stream, a);
      });
    });
  return in_launches(g, g.rows * g.pieces, kBlock, [&](Gradient a, int64_t done, dim3 grid) {
    a.item0 = done;
    hipLaunchKernelGGL(long_gradient_kernel<T>, grid, dim3(kBlock), 0, stream, a);
  });
}
}  // namespace

}  // namespace categorical
}  // namespace hipenvs

using namespace hipenvs;
using namespace hipenvs::categorical;

extern "C" int64_t hipenvs_log_probs_workspace_bytes(int64_t rows, int64_t v, int32_t top) {
  if (!sizes_ok(0, rows, v, top)) return -1;
  if (rows == 0) return 0;
  LogProbs p = {};
  return plan(&p, rows, v) == HIPENVS_OK ? lay(&p, nullptr, top) : -1;
}

extern "C" int hipenvs_log_probs(int32_t dtype, const void* logits, int64_t logits_s, const int64_t* tokens,
                                 float* log_prob, float* entropy, float* stats, int32_t top, float* top_log_prob,
                                 int64_t* top_index, int64_t rows, int64_t v, void* workspace,
                                 int64_t workspace_bytes, hipenvs_stream_t stream) {
  if (!sizes_ok(dtype, rows, v, top)) return HIPENVS_E_ARG;
  if (rows == 0) return HIPENVS_OK;
  if (!logits || !tokens || !log_prob || !entropy || (top > 0 && (!top_log_prob || !top_index))) return HIPENVS_E_ARG;
  LogProbs p = {};
  const int status = plan(&p, rows, v);
  if (status != HIPENVS_OK) return status;
  const int64_t need = lay(&p, (char*)workspace, top);
  if (need > 0 && (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < need)) return HIPENVS_E_ARG;
  p.logits = logits, p.logits_s = logits_s, p.tokens = tokens, p.log_prob = log_prob, p.entropy = entropy;
  p.stats = stats, p.top = top, p.top_log_prob = top_log_prob, p.top_index = top_index;
  return dtype == 1 ? forward<__bf16>(p, as_stream(stream)) : forward<float>(p, as_stream(stream));
}

extern "C" int hipenvs_log_probs_backward(int32_t dtype, const void* logits, int64_t logits_s, const int64_t* tokens,
                                          const float* stats, const float* entropy, const float* dlog_prob,
                                          const float* dentropy, void* dlogits, int64_t rows, int64_t v,
                                          hipenvs_stream_t stream) {
  if (!sizes_ok(dtype, rows, v, 0)) return HIPENVS_E_ARG;
  if (rows == 0) return HIPENVS_OK;
  if (!logits || !tokens || !stats || !entropy || !dlogits) return HIPENVS_E_ARG;
  const Gradient g = {logits,   tokens,   stats,    entropy, dlog_prob, dentropy,
                      dlogits,  logits_s, rows,     v,       0,         (int32_t)((v + kPiece - 1) / kPiece)};
  return dtype == 1 ? gradient<__bf16>(g, as_stream(stream)) : gradient<float>(g, as_stream(stream));
}
