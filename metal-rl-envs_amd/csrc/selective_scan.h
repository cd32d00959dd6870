// The selective state space scan: what its kernels and its entry points share.
//
//   delta = softplus(dt + dt_bias)          h_t[n] = exp(delta rate[n]) h_{t-1}[n] + delta x write_t[n]
//   y = sum_n read_t[n] h_t[n] + skip x     out = y silu(gate)
//
// for each channel of each row, with h_{t-1} left out where an episode begins at t. Channels lie
// in g groups of dg, each with rows of write and read of its own.
#pragma once

#include "row_ops.h"

namespace hipenvs {
namespace scan {

using namespace rows;

constexpr int kTile = 16;        // tokens staged at once; the states before each are kept for the backward pass
constexpr int kMaxStates = 64;

struct Rows {      // (b, t, channels)
  const void* data;
  int64_t sb, st;
};

struct Mix {       // (b, t, g, n)
  const void* data;
  int64_t sb, st, sg;
};

struct Scan {
  Rows x, dt, gate, dout;
  Mix write, read;
  const float *rate, *skip, *bias, *state, *dfinal;
  const uint8_t* reset;
  int64_t reset_sb, reset_st;
  void* out;
  float *final_state, *checks;     // checks (b, ceil(t / kTile), d, n), or null
  void *dx, *ddt, *dgate, *dwrite, *dread;
  float *dstate, *dmix, *dparams;  // dmix (tiles, b t g, 2 NP) where tiles > 1; dparams (b parts, d (n + 2))
  float *carry, *spans;            // (b, parts, d, n): the states between the parts; (b, parts, d): their sums of delta
  uint8_t* begun;                  // (b, parts): whether an episode begins in the part
  int64_t b, t, part;              // part: tokens of a part, whole tiles
  int32_t d, n, g, dg, tiles, parts;
  int64_t item0;
};

// LPC lanes a channel, four states each. A block has 64 channels (32 at 16 lanes) of one group, or where a
// group has no more than 32, as few as fill its waves: lanes without a channel cost as much as others. 128
// channels in four groups, 1,024 x 128 tokens, forwards and backwards: 714 us in blocks of 64, 511 so; in 128
// groups 25,300 and 6,900.
constexpr int channels_of(int lpc, bool few) { return few ? (lpc == 2 ? 32 : 16) : lpc == 16 ? 32 : 64; }
inline int lanes_of(int n) { return n <= 8 ? 2 : n <= 16 ? 4 : n <= 32 ? 8 : 16; }
inline bool few_channels(int dg) { return dg <= 32; }

template <int LPC, bool kFew>
struct Shape {
  static constexpr int CH = channels_of(LPC, kFew), kThreads = CH * LPC, kWaves = kThreads / 64, NP = 4 * LPC;
  static constexpr int kSlots = (kTile * CH / 4 + kThreads - 1) / kThreads;   // four channels of a token each
  static constexpr int kMixSlots = (kTile * 2 * LPC + kThreads - 1) / kThreads;
};

// Where a block is: row b, part p, group and the first of its channels within the group.
struct Place {
  int64_t b;
  int p, group, first;
};

__device__ __forceinline__ Place place_of(const Scan& s, int64_t item, int parts, int channels) {
  const int tile = (int)(item % s.tiles);
  item /= s.tiles;
  const int group = (int)(item % s.g);
  item /= s.g;
  return {item / parts, (int)(item % parts), group, tile * channels};
}

// What a thread fetches of every tile: its slots of four channels of a token, and of four states of write or
// read. Rows lie at a block's own address plus token times stride, one instruction: strides of t are
// below 2^31. Channels and states past theirs read the last four, and whoever uses them leaves them out.
template <int LPC, bool kFew>
struct Slots {
  using S = Shape<LPC, kFew>;

  static __device__ __forceinline__ int token(int i) {   // of slot i; kTile and more: none
    return (threadIdx.x + i * S::kThreads) / (S::CH / 4);
  }
  static __device__ __forceinline__ int channel() { return threadIdx.x % (S::CH / 4) * 4; }   // within the block
  static __device__ __forceinline__ int mix_token(int i) { return (threadIdx.x + i * S::kThreads) / (2 * LPC); }
  static __device__ __forceinline__ int mix_part() { return threadIdx.x % (2 * LPC); }   // below LPC: write
  static __device__ __forceinline__ int mix_state() { return threadIdx.x % LPC * 4; }
};

// The same number, about which the compiler knows nothing: addresses that it works out once for all of a
// loop's rounds would take the registers of the states.
__device__ __forceinline__ int32_t anew(int32_t x) {
  asm volatile("" : "+s"(x));
  return x;
}

__device__ __forceinline__ int64_t anew(int64_t x) {
  const uint32_t lo = (uint32_t)anew((int32_t)x), hi = (uint32_t)anew((int32_t)(x >> 32));
  return (int64_t)((uint64_t)hi << 32 | lo);
}

// A use of a loaded value: the wait for it comes here, and not behind the stores that follow, which a later
// one would wait for as well.
template <class V>
__device__ __forceinline__ void settle(V& x) {
  static_assert(sizeof(V) == 8 || sizeof(V) == 16, "four values");
  typedef uint32_t bits __attribute__((ext_vector_type(sizeof(V) / 4)));
  bits held = __builtin_bit_cast(bits, x);
  asm volatile("" : "+v"(held));
  x = __builtin_bit_cast(V, held);
}

template <class T>
__device__ __forceinline__ const T* row_at(const T* base, int token, int32_t stride) {
  return (const T*)((const char*)base + (int64_t)(token * (int)sizeof(T)) * (int64_t)stride);
}

// Where a tile's first token lies, and how far apart tokens are.
template <class T>
struct Source {
  const T* at;
  int32_t st;

  __device__ __forceinline__ void set(const void* data, int64_t offset, int64_t t0, int64_t stride) {
    at = (const T*)data + offset + t0 * stride;
    st = (int32_t)stride;
  }
  __device__ __forceinline__ void move(int tokens) { at = row_at(at, tokens, st); }
};

// A block's sources, a tile after another. Without a gate its place is x, read again and not used: a
// branch would keep the loads behind it from being in flight with those before.
template <class T, bool kGate, bool kBack>
struct Sources {
  Source<T> x, dt, gate, dout, write, read;
  Source<uint8_t> reset;

  __device__ __forceinline__ Sources(const Scan& s, const Place& at, int64_t t0) {
    const int64_t col = (int64_t)at.group * s.dg;
    x.set(s.x.data, at.b * s.x.sb + col, t0, s.x.st);
    dt.set(s.dt.data, at.b * s.dt.sb + col, t0, s.dt.st);
    const Rows& z = s.gate.data ? s.gate : s.x;
    if (kGate) gate.set(z.data, at.b * z.sb + col, t0, z.st);
    if (kBack) dout.set(s.dout.data, at.b * s.dout.sb + col, t0, s.dout.st);
    write.set(s.write.data, at.b * s.write.sb + at.group * s.write.sg, t0, s.write.st);
    read.set(s.read.data, at.b * s.read.sb + at.group * s.read.sg, t0, s.read.st);
    reset.at = nullptr, reset.st = 0;
    if (s.reset) reset.set(s.reset, at.b * s.reset_sb, t0, s.reset_st);
  }

  __device__ __forceinline__ void move(int tokens) {
    x.move(tokens), dt.move(tokens), write.move(tokens), read.move(tokens);
    if (kGate) gate.move(tokens);
    if (kBack) dout.move(tokens);
    reset.move(tokens);
  }
};

template <class T, int LPC, bool kFew, bool kGate, bool kBack>
struct Fetched {
  using S = Shape<LPC, kFew>;
  using At = Slots<LPC, kFew>;
  typename Raw<T>::type x[S::kSlots], dt[S::kSlots], gate[S::kSlots], dout[S::kSlots], mix[S::kMixSlots];
  uint8_t begins;   // of the token of this lane

  // kWhole: four channels and four states at least, and `count`, the tokens from the tile's first on, a whole
  // tile; otherwise tokens past the end are the last one again
  template <bool kWhole>
  __device__ __forceinline__ void load(const Scan& s, const Sources<T, kGate, kBack>& of, int first, int64_t count) {
    const int last = kWhole || count > kTile ? kTile - 1 : (int)count - 1;
    int c = first + At::channel();
    c = c < s.dg ? c : 0;
    if (kWhole) c = c < s.dg - 4 ? c : s.dg - 4;
    const auto four = [&](const Source<T>& source, int token) {
      const T* row = row_at(source.at, token < last ? token : last, anew(source.st));
      if constexpr (kWhole)
        return *(const typename Raw<T>::any*)(row + c);
      else
        return fetch4(row, c, s.dg);
    };
#pragma unroll
    for (int i = 0; i < S::kSlots; ++i) {
      x[i] = four(of.x, At::token(i));
      dt[i] = four(of.dt, At::token(i));
      if (kGate) gate[i] = four(of.gate, At::token(i));
      if (kBack) dout[i] = four(of.dout, At::token(i));
    }
    const bool writes = At::mix_part() < LPC;
    const T* mix0 = writes ? of.write.at : of.read.at;
    const int32_t mix_st = writes ? anew(of.write.st) : anew(of.read.st);
    int n0 = At::mix_state();
    n0 = n0 < s.n ? n0 : 0;
    if (kWhole) n0 = n0 < s.n - 4 ? n0 : s.n - 4;
#pragma unroll
    for (int i = 0; i < S::kMixSlots; ++i) {
      const T* row = row_at(mix0, At::mix_token(i) < last ? At::mix_token(i) : last, mix_st);
      if constexpr (kWhole)
        mix[i] = *(const typename Raw<T>::any*)(row + n0);
      else
        mix[i] = fetch4(row, n0, s.n);
    }
    begins = 0;
    if (of.reset.at) {
      const int tok = threadIdx.x & 63;
      begins = *row_at(of.reset.at, tok < last ? tok : last, anew(of.reset.st));
    }
  }

  __device__ __forceinline__ void fetch(const Scan& s, const Sources<T, kGate, kBack>& of, int first, int64_t count) {
    if (count >= kTile && s.dg >= 4 && s.n >= 4)
      load<true>(s, of, first, count);
    else
      load<false>(s, of, first, count);
  }

  __device__ __forceinline__ void arrive() {
#pragma unroll
    for (int i = 0; i < S::kSlots; ++i) {
      settle(x[i]), settle(dt[i]);
      if (kGate) settle(gate[i]);
      if (kBack) settle(dout[i]);
    }
#pragma unroll
    for (int i = 0; i < S::kMixSlots; ++i) settle(mix[i]);
    uint32_t held = begins;
    asm volatile("" : "+v"(held));
    begins = (uint8_t)held;
  }

  // a bit for each token of the tile that begins an episode
  __device__ __forceinline__ uint32_t begun(int64_t t0, int64_t end) const {
    const int tok = threadIdx.x & 63;
    return (uint32_t)__builtin_amdgcn_ballot_w64(tok < kTile && t0 + tok < end && begins != 0);
  }

  // write and read to LDS, zeros past the end and past the states
  __device__ __forceinline__ void put_mix(const Scan& s, int64_t t0, int64_t end, float (*to)[8 * LPC]) const {
    const int n0 = At::mix_state();
#pragma unroll
    for (int i = 0; i < S::kMixSlots; ++i) {
      const int tok = At::mix_token(i);
      f32x4 m = values<T>(mix[i], n0 < s.n ? n0 : 0, s.n);
      if (t0 + tok >= end || n0 >= s.n) m = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      if (tok < kTile) *(f32x4*)&to[tok][At::mix_part() * 4] = m;
    }
  }
};

__device__ __forceinline__ f32x4 per_channel(const float* of, int64_t c, int left, float otherwise) {
  f32x4 r = {otherwise, otherwise, otherwise, otherwise};
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (of && e < left) r[e] = of[c + e];
  return r;
}

// Sums 8 values of a lane over the channels of its wave: the lanes whose bits from log2(LPC) on
// differ. Each step halves the values a lane keeps, until one is left; lane l then has value
// id(l) of its states, twice over where fewer channel bits than that are left.
template <int LPC>
struct Across {
  static constexpr int kLeft = LPC == 16 ? 2 : 1;

  static __device__ __forceinline__ void sum(float (&v)[8], int lane) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {   // bit 5
      const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v[i]), __float_as_uint(v[i + 4]), false, false);
      v[i] = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {   // bit 4
      const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v[i]), __float_as_uint(v[i + 2]), false, false);
      v[i] = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    if constexpr (LPC <= 8) {       // bit 3
      const bool upper = lane & 8;
      const float keep = upper ? v[1] : v[0], give = upper ? v[0] : v[1];
      v[0] = keep + from_xor<8>(give);
    }
    if constexpr (LPC <= 4) v[0] += from_xor<4>(v[0]);
    if constexpr (LPC <= 2) v[0] += from_xor<2>(v[0]);
  }

  // which of the eight values `kept` of this lane is
  static __device__ __forceinline__ int id(int lane, int kept) {
    return ((lane >> 5) & 1) * 4 + ((lane >> 4) & 1) * 2 + (LPC <= 8 ? (lane >> 3) & 1 : kept);
  }
};

}  // namespace scan
}  // namespace hipenvs
