// Linear attention with a decay for each head and episodes inside its rows (see
// include/hipenvs.h): the walk over whole sequences, in chunks on the matrix cores. No
// reference counterpart: the reference's policies have no memory.
//
//   S_t = (reset_t ? 0 : lambda S_{t-1}) + k_t v_t^T        o_t = scale S_t^T q_t
//
// One walk gives the outputs and every gradient. Forwards, it decays the state, adds
// add * k v^T and reads read * S^T q; backwards, it adds and reads first and decays after. With
// G_t = dL/dS_t = scale q_t do_t^T + (reset_{t+1} ? 0 : lambda G_{t+1}):
//
//   o  = walk(q, k, v) on S        dq = walk(do, v, k) on S^T            forwards
//   dv = walk(k, q, do) on G       dk = walk(v, do, q) on G^T            backwards
//
// A chunk of n tokens with S before it, i and j counted within it:
//
//   o_i = read lambda^{i+1} S^T q_i [no reset in 0..i]
//         + add read sum_{j <= i, no reset in j+1..i} lambda^{i-j} (q_i . k_j) v_j
//   S'  = lambda^n S [no reset] + add sum_{j: no reset in j+1..n-1} lambda^{n-1-j} k_j v_j^T
//
// and mirrored backwards (lambda^{n-1-i} and lambda^{j+1} change places). Whatever is left out
// is chosen out, never multiplied by zero, except inside the matrix products over a chunk's
// tokens, where a zero weight meets whatever its token holds; see `serial`.
#pragma once

#include "hipenvs_device.h"

namespace hipenvs {
namespace da {

constexpr int kMaxDim = 128;

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

template <class T>
__device__ __forceinline__ float to_f32(T x) {
  return (float)x;
}
template <class T>
__device__ __forceinline__ T from_f32(float x) {
  return (T)x;  // bfloat16: to nearest even
}

struct Rows {
  const void* data;
  int64_t sb, st, sh;  // strides in elements of a row's batch, token and head; the last is 1
};

struct Walk {
  Rows q, k, v;            // roles: read with q, add k v^T
  int32_t dk, dv;          // of these roles
  const float* log_decay;  // (h)
  const uint8_t* reset;    // (b, t) or null
  int64_t reset_sb, reset_st;
  const float* state_in;   // (b, h, dk, dv), or (b, h, dv, dk) when flipped; null: zeros
  float* state_out;        // null: not wanted
  bool flipped, backwards;
  float read, add;
  void* out;               // (b, t, h, dv) contiguous
  int64_t b, t;
  int32_t h;
  // the axis in parts of `part` tokens (a multiple of the chunk), each walked by a block of its
  // own from the state before it; one part: states and flags are not used
  int32_t parts;
  int64_t part;
  float* states;           // (b h, parts, dk, dv), or (b h, parts, dv, dk) when turned
  uint8_t* flags;          // (b h, parts): a reset in the part
  bool turned;
  uint32_t row0;           // the first row of this launch
};

// Threads of a launch stay below 2^32, the most a grid's axis takes.
constexpr int64_t kMostThreads = 0xFFFFFFFFll;

// One walk, or two of the same kind over the same rows: their blocks for a row lie side by side
// on one XCD and read what they share (q and dout, for the gradients of k and v) once.
struct Walks {
  Walk w[2];
  int32_t count;
};

// Values of a state in its caller's layout.
__device__ __forceinline__ int64_t state_index(const Walk& w, int64_t row, int r, int c) {
  return row * w.dk * w.dv + (w.flipped ? (int64_t)c * w.dk + r : (int64_t)r * w.dv + c);
}

// Tokens [t0, t1) of a row one after another, for the 16 columns of one wave, four at a time:
// column c of the four in each 16 lanes, an eighth of 128 rows of the state in each lane. The
// chunked form meets zero weights with whatever their tokens hold, and 0 * NaN is not 0; so a
// wave that finds anything but finite numbers in its outputs or its state walks its part
// again here, where a token takes part only where it counts, from the state that the chunked
// form started from: `from`, with its strides of rows and columns (null: zeros). A path for
// data that has gone wrong: small in registers, not fast.
template <class T, bool kOut>
__device__ __forceinline__ void serial(const Walk& w, int64_t row, int col0, int64_t t0, int64_t t1,
                                       const float* from, int on_row, int on_col, float* to, bool last) {
  constexpr int N = kMaxDim / 16;
  const int lane = threadIdx.x & 63, l = lane & 15;
  const int64_t b = row / w.h, h = row - b * w.h;
  const float lambda = expf(w.log_decay[h]);
  const T* q = (const T*)w.q.data + b * w.q.sb + h * w.q.sh;
  const T* k = (const T*)w.k.data + b * w.k.sb + h * w.k.sh;
  const T* v = (const T*)w.v.data + b * w.v.sb + h * w.v.sh;
  for (int four = 0; four < 16; four += 4) {
    const int col = col0 + four + (lane >> 4);
    const bool live = col < w.dv;
    float s[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int r = 16 * i + l;
      s[i] = 0.0f;
      if (from && r < w.dk && live) s[i] = from[r * on_row + col * on_col];
    }
    for (int64_t n = 0; n < t1 - t0; ++n) {
      const int64_t t = w.backwards ? t1 - 1 - n : t0 + n;
      const bool fresh = w.reset && w.reset[b * w.reset_sb + t * w.reset_st];
      const float x = live ? w.add * to_f32<T>(v[t * w.v.st + col]) : 0.0f;
      float o = 0.0f;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int r = 16 * i + l;
        if (r < w.dk) {
          if (!w.backwards) s[i] = fresh ? 0.0f : s[i] * lambda;
          s[i] = __builtin_fmaf(to_f32<T>(k[t * w.k.st + r]), x, s[i]);
          if (kOut) o = __builtin_fmaf(to_f32<T>(q[t * w.q.st + r]), s[i], o);
          if (w.backwards) s[i] = fresh ? 0.0f : s[i] * lambda;
        }
      }
      if (kOut) {
#pragma unroll
        for (int m = 8; m > 0; m >>= 1) o += __shfl_xor(o, m);
        if (l == 0 && live) ((T*)w.out)[((b * w.t + t) * w.h + h) * w.dv + col] = from_f32<T>(w.read * o);
      }
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int r = 16 * i + l;
      if (r < w.dk && live) {
        if (to) to[(int64_t)r * w.dv + col] = s[i];
        if (last && w.state_out) w.state_out[state_index(w, row, r, col)] = s[i];
      }
    }
  }
}

// ---- the chunked walk -------------------------------------------------------------------

// Tokens a chunk holds and the padding of LDS rows of `width` values: 16 rows read at one column
// in 16 bytes lie on different banks, and so do, nearly, the 8 bytes of 8 rows that the
// transposing reads of bfloat16 take at once (rows 12, 28, 36 or 52 banks apart).
template <class T>
struct Chunk;
template <>
struct Chunk<__bf16> {
  static constexpr int kTokens = 64;
  static constexpr int pad(int width) { return width == 32 || width == 128 ? 24 : 8; }
};
template <>
struct Chunk<float> {
  static constexpr int kTokens = 32;
  static constexpr int pad(int) { return 4; }
};

// What P is stored as: float32, or T's parts.
template <bool kSplit, class T>
struct Stored {
  typedef float type;
  static constexpr int kPad = Chunk<float>::pad(0);
};
template <class T>
struct Stored<true, T> {
  typedef T type;
  static constexpr int kPad = Chunk<T>::pad(Chunk<T>::kTokens);
};

// 16 bytes at any address that is a multiple of the value's size.
typedef u32x4 __attribute__((aligned(2))) piece_at_2;
template <class T>
struct Fours;   // four values
template <>
struct Fours<__bf16> {
  typedef u32x2 type;
};
template <>
struct Fours<float> {
  typedef u32x4 type;
};

// A token's row of `dim` values is read in 16-byte pieces. The last one may be short: then the
// row's last 16 bytes are read, which begin piece_begin(col) values into the row, and moved
// down by `settled` once they are there (where they are written to LDS, so that no load waits
// for another). A row shorter than a piece is read one value after another.
template <class T>
__device__ __forceinline__ int piece_begin(int col, int dim) {
  constexpr int E = 16 / sizeof(T);
  return dim < E ? 0 : col + E <= dim ? col : dim - E;
}

template <class T>
__device__ __forceinline__ u32x4 load_short_row(const T* at, int col, int dim) {
  constexpr int E = 16 / sizeof(T);
  u32x4 x = {0, 0, 0, 0};
  if (col >= dim) return x;
  if (dim >= E) return *(const piece_at_2*)at;
#pragma unroll 1
  for (int e = dim - 1; e >= 0; --e) {
    if (sizeof(T) == 4)
      x = u32x4{((const uint32_t*)at)[e], x[0], x[1], x[2]};
    else
      x = u32x4{(x[0] << 16) | ((const uint16_t*)at)[e], (x[1] << 16) | (x[0] >> 16), (x[2] << 16) | (x[1] >> 16),
                (x[3] << 16) | (x[2] >> 16)};
  }
  return x;
}

template <class T>
__device__ __forceinline__ u32x4 settled(u32x4 x, int col, int dim) {
  constexpr int E = 16 / sizeof(T);
  if (dim % E != 0 && dim > E) {
    const int over = col + E > dim ? col + E - dim : 0, bytes = over * (int)sizeof(T);
    if (bytes & 8) x = u32x4{x[2], x[3], 0, 0};
    if (bytes & 4) x = u32x4{x[1], x[2], x[3], 0};
    if (bytes & 2)
      x = u32x4{(x[0] >> 16) | (x[1] << 16), (x[1] >> 16) | (x[2] << 16), (x[2] >> 16) | (x[3] << 16), x[3] >> 16};
  }
  return x;
}

__device__ __forceinline__ bf16x8 join(i16x4 a, i16x4 b) {
  const bf16x4 x = __builtin_bit_cast(bf16x4, a), y = __builtin_bit_cast(bf16x4, b);
  return __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
}

// Columns col .. col + 15 of rows row .. row + 3 and row + 16 .. row + 19 of a bfloat16 tile,
// rows differing between the four groups of 16 lanes: lane l of a group gets column col + l. A
// transposing read gives a group 16 columns of 4 rows, each of its lanes addressing 4 values.
__device__ __forceinline__ bf16x8 read_columns(const __bf16* tile, int stride, int row, int col) {
  const int l = threadIdx.x & 15;
  const __bf16* p = tile + (row + (l >> 2)) * stride + col + 4 * (l & 3);
  typedef __attribute__((address_space(3))) i16x4* lds4;
  return join(__builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)p),
              __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(p + 16 * stride)));
}

// Four values and the four 16 further on: an operand whose summed axis is ordered like
// read_columns' and like a result's rows.
__device__ __forceinline__ bf16x8 read_pair(const __bf16* p) {
  return __builtin_shufflevector(*(const bf16x4*)p, *(const bf16x4*)(p + 16), 0, 1, 2, 3, 4, 5, 6, 7);
}

// A lane's index, in a branch that few chunks take: what is computed from it there is computed
// there. Otherwise the compiler computes it all before the loop and holds it in registers that
// the loop itself needs (248 of 256 at bfloat16 heads of 64, its reads waiting for each other).
__device__ __forceinline__ int here(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

// The bfloat16 parts of N (even) float32 values: of each, the rounding of what is left. Three
// parts of 8 bits hold all 24.
constexpr int kParts = 3;
template <int N>
__device__ __forceinline__ void split(float (&rest)[N], __bf16 (&parts)[kParts][N]) {
#pragma unroll
  for (int m = 0; m < kParts; ++m)
#pragma unroll
    for (int e = 0; e < N; e += 2) {
      const f32x2 x = {rest[e], rest[e + 1]};
      const bf16x2 y = __builtin_convertvector(x, bf16x2);
      parts[m][e] = y[0], parts[m][e + 1] = y[1];
      rest[e] -= (float)y[0], rest[e + 1] -= (float)y[1];
    }
}

// Waves a SIMD holds at once, which bounds their registers (512 over that many): three where
// that many registers suffice without spilling, two elsewhere.
template <class T>
constexpr int waves_of(int dk, int nw) {
  return sizeof(T) == 4 && (dk == 32 || (dk == 64 && nw >= 4)) ? 3 : 2;
}

constexpr int power_of_two(int n) {   // the least that is not below n
  int p = 1;
  while (p < n) p *= 2;
  return p;
}

// A wave takes 16 columns of the state, all of its rows: S[a][r] is row 16 a + 4 g + r, column
// l, for lane 16 g + l. That is both a matrix instruction's result and, its rows
// taken as the summed axis in that order, an operand of the read S^T q, so the state never
// leaves its registers. The block's NW waves share a chunk's q, k, v (in LDS; while one
// chunk is computed the next is on its way to registers) and its masked products
// P[i][j], computed once.
//
// bfloat16 rows: the inputs are exact operands. P, the S that is read and the lambda^n v_j that
// is added are float32, split for the matrix instructions into three bfloat16 parts, each the
// rounding of what the parts before it leave: all 24 bits, so nothing but a result is rounded to
// fewer. float32 rows use the float32 matrix instructions throughout.
//
// What bounds it: with many rows of 128 tokens memory, at 4.8 TB/s (float32 heads of 32), 4.3 (of
// 64), 3.6 and 3.8 (bfloat16 heads of 32 and 64), where `step` reaches 5.8; in heads of 128 the
// chain of a chunk's loads, barriers and products, eight waves being all that 239 registers
// leave a CU (3.2 TB/s bfloat16, 3.0 float32, there mostly float32 products). A chunk of 64
// tokens takes a block of four waves 3.4 us alone on a CU and 4.2 beside another (bfloat16
// heads of 64), of eight waves 5.8 (heads of 128). Parts of 24 bits, where two (16 bits) would be
// within a result's own rounding, cost 1 to 13 % (sequence of 8 heads of 64 x 16,381 41.7 -> 43.5 us,
// 512 rows of 1,000 with gradients 272 -> 294). Chunks of 64 are one wave's reset mask and
// two products' depth; float32's 32 keep a block's q, k, v and P below 56 KB of LDS.
template <class T, int DK, int NW, bool kOut, bool kBack>
__global__ __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(waves_of<T>(DK, NW)))) void chunk_kernel(Walks walks) {
  constexpr bool kHalf = sizeof(T) == 2;
  constexpr int C = Chunk<T>::kTokens, E = 16 / sizeof(T), TH = 64 * NW, DV = 16 * NW, NT = C / 16;
  constexpr int SQ = DK + Chunk<T>::pad(DK), SV = DV + Chunk<T>::pad(DV);
  constexpr int QP = power_of_two(DK / E), VP = power_of_two(DV / E);      // pieces of a row, rounded up
  constexpr int NQ = (C * QP + TH - 1) / TH, NV = (C * VP + TH - 1) / TH;  // pieces of a thread
  __shared__ __attribute__((aligned(16))) T Qs[kOut ? C * SQ : 8];
  __shared__ __attribute__((aligned(16))) T Ks[C * SQ];
  __shared__ __attribute__((aligned(16))) T Vs[C * SV];
  // Where dv <= 16 the block is one wave, which has all of P, and P's tiles are operands as they lie
  // in its registers: no copy in shared memory, no wait for it, and the smaller block (17.7 kB, not
  // 45, in bf16 with dk = 32) runs more often per CU. 2^24 values of q, k and v by 16 x 16 heads,
  // 128 tokens: bf16 145 -> 55 us, with gradients 588 -> 217; f32 113 -> 76 and 376 -> 287; at
  // dk = 128 56 -> 41 and 75 -> 48. With more waves each has a share of P only and reads the rest:
  // two that make all of P each took 21 % less to 9 % more by shape and length (bf16 in two parts),
  // and spilled at dk = 128 in bf16 (45 -> 74 us).
  constexpr bool kOwnP = NW == 1;
  // bfloat16's parts of P are made once, by the wave that made its tile, but in blocks of two waves
  // and at most 32 rows: these read P as float32 and split it themselves, so that four of them fit a CU's
  // LDS (39 kB, not 49). 32 x 32 heads, 2^24 values each of q, k and v, 128 tokens: 58 us, not 67,
  // with gradients 213, not 256; 1,000 tokens 66, not 64, and 237, not 248. With more rows three fit
  // either way (64 x 32: 50 and 49 us).
  constexpr bool kSplitP = kHalf && !kOwnP && !(NW == 2 && DK == 32);
  typedef Stored<kSplitP, T> P;
  constexpr int SP = C + P::kPad, kPs = kSplitP ? kParts : 1;
  __shared__ __attribute__((aligned(16))) typename P::type Ps[kOut && !kOwnP ? kPs * C * SP : 8];
  __shared__ float pw[C + 1];

  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, g = lane >> 4, l = lane & 15;
  // blocks of one XCD (every eighth) take neighbouring rows, whose tokens share cache lines
  const uint32_t blocks = gridDim.x;
  const uint32_t at = blocks % 8 == 0 ? (blockIdx.x % 8) * (blocks / 8) + blockIdx.x / 8 : blockIdx.x;
  const uint32_t id = walks.count == 2 ? at / 2 : at;
  const Walk& w = walks.w[walks.count == 2 ? at % 2 : 0];
  const uint32_t piece = id / (uint32_t)w.parts, part = id - piece * (uint32_t)w.parts, row = w.row0 + piece;
  const int64_t b = row / (uint32_t)w.h, h = row - (uint32_t)b * (uint32_t)w.h;
  const int64_t t0 = part * w.part, t1 = t0 + w.part < w.t ? t0 + w.part : w.t;
  const int chunks = (int)((t1 - t0 + C - 1) / C);
  const bool last = part == (kBack ? 0 : (uint32_t)w.parts - 1);
  const int tokens_of_last = (int)(t1 - t0) - (chunks - 1) * C;
  float* local = w.parts > 1 ? w.states + ((int64_t)row * w.parts + part) * w.dk * w.dv : nullptr;

  // where this thread's pieces of the first chunk lie, and how far on the next chunk's do
  const int64_t start = t0 + (kBack ? (int64_t)(chunks - 1) * C : 0);
  static_assert(TH % QP == 0 && TH % VP == 0, "a thread's pieces lie in one column of a chunk");
  const int qx = tid % QP * E, qr = tid / QP, vx = tid % VP * E, vr = tid / VP;
  constexpr int QR = TH / QP, VR = TH / VP;   // rows between a thread's pieces
  const int ky = piece_begin<T>(qx, w.dk);
  const T* kp = (const T*)w.k.data + b * w.k.sb + h * w.k.sh + (start + qr) * w.k.st + ky;
  const T* qp = kOut ? (const T*)w.q.data + b * w.q.sb + h * w.q.sh + (start + qr) * w.q.st + ky : nullptr;
  const T* vp = (const T*)w.v.data + b * w.v.sb + h * w.v.sh + (start + vr) * w.v.st + piece_begin<T>(vx, w.dv);
  const uint8_t* rp = w.reset ? w.reset + b * w.reset_sb + (start + lane) * w.reset_st : nullptr;
  const int64_t q_on = (kBack ? -C : C) * w.q.st, k_on = (kBack ? -C : C) * w.k.st, v_on = (kBack ? -C : C) * w.v.st;

  u32x4 xq[kOut ? NQ : 1], xk[NQ], xv[NV];
  uint32_t xr = 0;
  const bool tiny = w.dk < E || w.dv < E;
  const bool filled = w.dk == DK && w.dv == DV && QP * E == DK && VP * E == DV && C % QR == 0 && C % VR == 0;
  const auto load = [&](int n) {
    if (filled && n == C) {
#pragma unroll
      for (int m = 0; m < NQ; ++m) {
        xk[m] = *(const piece_at_2*)(kp + m * QR * w.k.st);
        if constexpr (kOut) xq[m] = *(const piece_at_2*)(qp + m * QR * w.q.st);
      }
#pragma unroll
      for (int m = 0; m < NV; ++m) xv[m] = *(const piece_at_2*)(vp + m * VR * w.v.st);
    } else {
      const u32x4 none = {0, 0, 0, 0};
#pragma unroll
      for (int m = 0; m < NQ; ++m) {
        xk[m] = none;
        if constexpr (kOut) xq[m] = none;
      }
#pragma unroll
      for (int m = 0; m < NV; ++m) xv[m] = none;
      if (!tiny) {
#pragma unroll
        for (int m = 0; m < NQ; ++m)
          if (qr + m * QR < n && qx < w.dk) {
            xk[m] = *(const piece_at_2*)(kp + m * QR * w.k.st);
            if constexpr (kOut) xq[m] = *(const piece_at_2*)(qp + m * QR * w.q.st);
          }
#pragma unroll
        for (int m = 0; m < NV; ++m)
          if (vr + m * VR < n && vx < w.dv) xv[m] = *(const piece_at_2*)(vp + m * VR * w.v.st);
      } else {
#pragma unroll
        for (int m = 0; m < NQ; ++m)
          if (qr + m * QR < n) {
            xk[m] = load_short_row<T>(kp + m * QR * w.k.st, qx, w.dk);
            if constexpr (kOut) xq[m] = load_short_row<T>(qp + m * QR * w.q.st, qx, w.dk);
          }
#pragma unroll
        for (int m = 0; m < NV; ++m)
          if (vr + m * VR < n) xv[m] = load_short_row<T>(vp + m * VR * w.v.st, vx, w.dv);
      }
    }
    kp += k_on;
    if constexpr (kOut) qp += q_on;
    vp += v_on;
    xr = 0;
    if (rp) {
      if (lane < n) xr = *rp;
      rp += (kBack ? -C : C) * w.reset_st;
    }
  };
  if (chunks > 0) load(kBack || chunks == 1 ? tokens_of_last : C);

  const float ld = w.log_decay[h];
  for (int n = tid; n <= C; n += TH) pw[n] = n == 0 ? 1.0f : expf(ld * (float)n);
  f32x4 S[DK / 16];
  const int col = 16 * wave + l;
#pragma unroll
  for (int a = 0; a < DK / 16; ++a) S[a] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  // where the state before the first token lies, and its strides of rows and columns
  const float* from = !kOut ? nullptr : local ? local : w.state_in ? w.state_in + (int64_t)row * w.dk * w.dv : nullptr;
  const bool turned = local ? w.turned : w.flipped;
  const int on_row = turned ? 1 : w.dv, on_col = turned ? w.dk : 1;
  if (from) {   // every value in flight at once: none behind a condition of its own
    const int c = col < w.dv ? col : 0;
#pragma unroll
    for (int a = 0; a < DK / 16; ++a)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int k = 16 * a + 4 * g + r;
        S[a][r] = from[(k < w.dk ? k : 0) * on_row + c * on_col];
      }
#pragma unroll
    for (int a = 0; a < DK / 16; ++a)
#pragma unroll
      for (int r = 0; r < 4; ++r) S[a][r] = 16 * a + 4 * g + r < w.dk && col < w.dv ? S[a][r] : 0.0f;
  }
  __syncthreads();   // pw

  // The tiles of P, 16 queries x 16 keys, that some product uses, dealt to the waves: tile x of
  // this wave is pair_of(x) = (query tile, key tile). bfloat16's products run over 32 keys, so
  // the tiles beside the diagonal are among them, with decays of zero.
  constexpr int kPairs = kHalf ? 12 : 4, kOwn = (kPairs + NW - 1) / NW;
  const auto pair_of = [&](int x) {
    const int y = kOwnP ? x : wave + NW * x;
    const int it = y < 4 ? y >> 1 : y < 8 ? 2 : 3, jt = y < 4 ? y & 1 : y & 3;
    return kBack ? make_int2(NT - 1 - it, NT - 1 - jt) : make_int2(it, jt);
  };

  // and the other way round, where one wave has them all
  const auto own_of = [](int it, int jt) {
    const int i = kBack ? NT - 1 - it : it, j = kBack ? NT - 1 - jt : jt;
    return i < 2 ? 2 * i + j : 4 * (i - 1) + j;
  };

  // The decays of a whole chunk. of_pair[x][r]: of tile x of P, zero where the key is not yet
  // there; of_read[it]: of the state, for query 16 it + l; of_add[x]: of the x-th token that
  // this lane holds of v, which is held(x).
  const auto held = [](int x, int g) { return 16 * (x / 4) + 4 * g + x % 4; };
  constexpr int NH = C / 4;
  float of_pair[kOut ? kOwn : 1][4], of_read[kOut ? NT : 1], of_add[NH];
  if constexpr (kOut) {
#pragma unroll
    for (int x = 0; x < kOwn; ++x) {
      const int2 tile = pair_of(x);
      const int ahead = 16 * (tile.x - tile.y) + l - 4 * g;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int gap = kBack ? r - ahead : ahead - r;
        of_pair[x][r] = gap >= 0 && gap < C ? w.read * w.add * pw[gap] : 0.0f;
      }
    }
#pragma unroll
    for (int it = 0; it < NT; ++it) of_read[it] = w.read * pw[kBack ? C - 1 - (16 * it + l) : 16 * it + l + 1];
  }
#pragma unroll
  for (int x = 0; x < NH; ++x) of_add[x] = w.add * pw[kBack ? held(x, g) + 1 : C - 1 - held(x, g)];
  const float of_chunk = pw[C];

  T* op = nullptr;   // this lane's first output of the chunk
  const int64_t o_row = (int64_t)w.h * w.dv;
  if constexpr (kOut) op = (T*)w.out + (b * w.t + start + l) * o_row + h * w.dv + 16 * wave + 4 * g;

  // The outputs of a chunk are stored while the next one is on its way to LDS: after the wait
  // for that one's loads, which would otherwise be a wait for the stores as well.
  typedef typename Fours<T>::type Four;
  Four done[kOut ? NT : 1];
  int done_n = 0;
  const auto store = [&]() {
    typedef Four __attribute__((aligned(2))) at_2;
    if (done_n == C && 16 * wave + 16 <= w.dv) {
#pragma unroll
      for (int it = 0; it < NT; ++it) *(at_2*)(op + it * 16 * o_row) = done[it];
    } else {
      const int lh = here(l), c0 = here(16 * wave + 4 * g);
#pragma unroll
      for (int it = 0; it < NT; ++it) {
        T* to = op + it * 16 * o_row;
        if (16 * it + lh < done_n) {
          if (c0 + 4 <= w.dv) {
            *(at_2*)to = done[it];
          } else if (w.dv % 4 != 0) {
            T y[4];
            __builtin_memcpy(y, &done[it], sizeof(y));
#pragma unroll
            for (int r = 0; r < 3; ++r)
              if (c0 + r < w.dv) to[r] = y[r];
          }
        }
      }
    }
    if (done_n > 0) op += (kBack ? -C : C) * o_row;
  };

  const bool idle = 16 * wave >= w.dv;   // no columns: this wave only moves and shares
  uint64_t any = 0;
  float bad = 0.0f;   // becomes NaN with the first value that is not finite
  for (int step = 0; step < chunks; ++step) {
    const int n = (kBack ? step == 0 : step == chunks - 1) ? tokens_of_last : C;
    if (step > 0) __syncthreads();   // the chunk before has been read
    if (w.dk % E != 0 || w.dv % E != 0) {
#pragma unroll
      for (int m = 0; m < NQ; ++m) {
        xk[m] = settled<T>(xk[m], qx, w.dk);
        if constexpr (kOut) xq[m] = settled<T>(xq[m], qx, w.dk);
      }
#pragma unroll
      for (int m = 0; m < NV; ++m) xv[m] = settled<T>(xv[m], vx, w.dv);
    }
#pragma unroll
    for (int m = 0; m < NQ; ++m)
      if ((C % QR == 0 || qr + m * QR < C) && (QP * E == DK || qx < DK)) {
        *(u32x4*)(Ks + (qr + m * QR) * SQ + qx) = xk[m];
        if constexpr (kOut) *(u32x4*)(Qs + (qr + m * QR) * SQ + qx) = xq[m];
      }
#pragma unroll
    for (int m = 0; m < NV; ++m)
      if ((C % VR == 0 || vr + m * VR < C) && (VP * E == DV || vx < DV)) *(u32x4*)(Vs + (vr + m * VR) * SV + vx) = xv[m];
    if constexpr (kOut) store();
    // the chunk's resets, bit i for token i; the first and the last of them
    const uint64_t mask = __builtin_amdgcn_ballot_w64(xr != 0);
    any |= mask;
    const int r_first = mask ? __builtin_ctzll(mask) : C, r_last = mask ? 63 - __builtin_clzll(mask) : -1;
    __syncthreads();
    if (step + 1 < chunks) load(!kBack && step + 2 == chunks ? tokens_of_last : C);

    f32x4 o[kOut ? NT : 1];
    f32x4 own_p[kOut && kOwnP ? kOwn : 1];
    if constexpr (kOut) {
      f32x4 p[kOwn];
#pragma unroll
      for (int x = 0; x < kOwn; ++x) {
        const int2 tile = pair_of(x);
        p[x] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        if (kPairs % NW != 0 && wave + NW * x >= kPairs) break;
        const T* kt = Ks + (16 * tile.y + l) * SQ;
        const T* qt = Qs + (16 * tile.x + l) * SQ;
        if constexpr (kHalf) {
#pragma unroll
          for (int m = 0; m < DK / 32; ++m)
            p[x] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(*(const bf16x8*)(kt + 32 * m + 8 * g),
                                                           *(const bf16x8*)(qt + 32 * m + 8 * g), p[x], 0, 0, 0);
        } else {
#pragma unroll
          for (int m = 0; m < DK / 16; ++m) {
            const f32x4 kf = *(const f32x4*)(kt + 16 * m + 4 * g), qf = *(const f32x4*)(qt + 16 * m + 4 * g);
#pragma unroll
            for (int e = 0; e < 4; ++e) p[x] = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[e], qf[e], p[x], 0, 0, 0);
          }
        }
      }
#pragma unroll
      for (int x = 0; x < kOwn; ++x)
#pragma unroll
        for (int r = 0; r < 4; ++r) p[x][r] *= of_pair[x][r];
      if (mask) {
        const int lh = here(l), gh = here(g);
#pragma unroll
        for (int x = 0; x < kOwn; ++x) {
          const int2 tile = pair_of(x);
          const int i = 16 * tile.x + lh;
          const uint64_t upto = mask & ((2ull << i) - 1), after = i < 63 ? mask >> (i + 1) : 0;
          const int from = upto ? 63 - __builtin_clzll(upto) : 0, until = after ? i + 1 + __builtin_ctzll(after) : C;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int j = 16 * tile.y + 4 * gh + r;
            p[x][r] = (kBack ? j < until : j >= from) ? p[x][r] : 0.0f;
          }
        }
      }
#pragma unroll
      for (int x = 0; x < kOwn; ++x) {
        const int2 tile = pair_of(x);
        if (kPairs % NW != 0 && wave + NW * x >= kPairs) break;
        typename P::type* to = Ps + (16 * tile.x + l) * SP + 16 * tile.y + 4 * g;
        if constexpr (kOwnP) {
          own_p[x] = p[x];
        } else if constexpr (kSplitP) {
          float rest[4] = {p[x][0], p[x][1], p[x][2], p[x][3]};
          __bf16 of[kParts][4];
          split(rest, of);
#pragma unroll
          for (int m = 0; m < kParts; ++m) *(bf16x4*)(to + m * C * SP) = __builtin_bit_cast(bf16x4, of[m]);
        } else {
          *(f32x4*)to = p[x];
        }
      }

      // what the state gives
      if (!idle) {
        if constexpr (kHalf) {
#pragma unroll
          for (int a = 0; a < DK / 32; ++a) {
            float rest[8];
            __bf16 of[kParts][8];
#pragma unroll
            for (int e = 0; e < 8; ++e) rest[e] = S[2 * a + e / 4][e % 4];
            split(rest, of);
#pragma unroll
            for (int it = 0; it < NT; ++it) {
              const bf16x8 qf = read_pair(Qs + (16 * it + l) * SQ + 32 * a + 4 * g);
              const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
              for (int m = 0; m < kParts; ++m)
                o[it] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, of[m]), qf,
                                                                a == 0 && m == 0 ? zero : o[it], 0, 0, 0);
            }
          }
        } else {
#pragma unroll
          for (int a = 0; a < DK / 16; ++a) {
            f32x4 qf[NT];
#pragma unroll
            for (int it = 0; it < NT; ++it) qf[it] = *(const f32x4*)(Qs + (16 * it + l) * SQ + 16 * a + 4 * g);
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
              for (int it = 0; it < NT; ++it) {
                const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
                o[it] = __builtin_amdgcn_mfma_f32_16x16x4f32(S[a][e], qf[it][e], a == 0 && e == 0 ? zero : o[it], 0, 0,
                                                             0);
              }
          }
        }
        if (!kBack || n == C) {
#pragma unroll
          for (int it = 0; it < NT; ++it)
#pragma unroll
            for (int r = 0; r < 4; ++r) o[it][r] *= of_read[it];
        } else {
          const int lh = here(l);
#pragma unroll
          for (int it = 0; it < NT; ++it) {
            const float f = 16 * it + lh < n ? w.read * pw[n - 1 - (16 * it + lh)] : 0.0f;
#pragma unroll
            for (int r = 0; r < 4; ++r) o[it][r] *= f;
          }
        }
        if (mask) {
          const int lh = here(l);
#pragma unroll
          for (int it = 0; it < NT; ++it) {
            const bool sees = kBack ? 16 * it + lh >= r_last : 16 * it + lh < r_first;
#pragma unroll
            for (int r = 0; r < 4; ++r) o[it][r] = sees ? o[it][r] : 0.0f;
          }
        }
      }
      if constexpr (!kOwnP) __syncthreads();
    }
    if (idle) continue;

    // this wave's columns of v, and its share of the products
    bf16x8 vh[kHalf ? C / 32 : 1];
    float vf[kHalf ? 1 : NH];
    if constexpr (kHalf) {
#pragma unroll
      for (int s = 0; s < C / 32; ++s) vh[s] = read_columns(Vs, SV, 32 * s + 4 * g, 16 * wave);
    } else {
#pragma unroll
      for (int x = 0; x < NH; ++x) vf[x] = Vs[held(x, g) * SV + col];
    }

    if constexpr (kOut) {
      if constexpr (kHalf) {
#pragma unroll
        for (int s = 0; s < C / 32; ++s)
#pragma unroll
          for (int it = 0; it < NT; ++it)
            if (kBack ? 2 * s + 1 >= it : 2 * s <= it) {
              const typename P::type* p = Ps + (16 * it + l) * SP + 32 * s + 4 * g;
              __bf16 of[kParts][8];
              if constexpr (!kSplitP) {
                float rest[8];
#pragma unroll
                for (int e = 0; e < 8; e += 4) {
                  f32x4 four;
                  if constexpr (kOwnP)
                    four = own_p[own_of(it, 2 * s + e / 4)];
                  else
                    four = *(const f32x4*)(p + 4 * e);
                  rest[e] = four[0], rest[e + 1] = four[1], rest[e + 2] = four[2], rest[e + 3] = four[3];
                }
                split(rest, of);
              }
#pragma unroll
              for (int m = 0; m < kParts; ++m) {
                bf16x8 pf;
                if constexpr (kSplitP)
                  pf = read_pair(p + m * C * SP);
                else
                  pf = __builtin_bit_cast(bf16x8, of[m]);
                o[it] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vh[s], pf, o[it], 0, 0, 0);
              }
            }
      } else {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int it = 0; it < NT; ++it)
            if (kBack ? t >= it : t <= it) {
              f32x4 p;
              if constexpr (kOwnP)
                p = own_p[own_of(it, t)];
              else
                p = *(const f32x4*)(Ps + (16 * it + l) * SP + 16 * t + 4 * g);
#pragma unroll
              for (int e = 0; e < 4; ++e)
                o[it] = __builtin_amdgcn_mfma_f32_16x16x4f32(vf[4 * t + e], p[e], o[it], 0, 0, 0);
            }
      }
    }

    // the state after the chunk
    float add[NH];
    if (n == C) {
#pragma unroll
      for (int x = 0; x < NH; ++x) add[x] = of_add[x];
    } else {
      const int gh = here(g);
#pragma unroll
      for (int x = 0; x < NH; ++x) {
        const int j = held(x, gh);
        add[x] = j < n ? w.add * pw[kBack ? j + 1 : n - 1 - j] : 0.0f;
      }
    }
    const float keep = n == C ? of_chunk : pw[n];
    if (mask) {
      const int gh = here(g);
#pragma unroll
      for (int x = 0; x < NH; ++x) add[x] = (kBack ? held(x, gh) < r_first : held(x, gh) >= r_last) ? add[x] : 0.0f;
#pragma unroll
      for (int a = 0; a < DK / 16; ++a) S[a] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    } else {
#pragma unroll
      for (int a = 0; a < DK / 16; ++a)
#pragma unroll
        for (int r = 0; r < 4; ++r) S[a][r] *= keep;
    }
    if constexpr (kHalf) {
#pragma unroll
      for (int s = 0; s < C / 32; ++s) {
        float rest[8];
        __bf16 of[kParts][8];
#pragma unroll
        for (int e = 0; e < 8; ++e) rest[e] = (float)vh[s][e] * add[8 * s + e];
        split(rest, of);
        bf16x8 kf[DK / 16];
#pragma unroll
        for (int a = 0; a < DK / 16; ++a) kf[a] = read_columns(Ks, SQ, 32 * s + 4 * g, 16 * a);
#pragma unroll
        for (int m = 0; m < kParts; ++m)
#pragma unroll
          for (int a = 0; a < DK / 16; ++a)
            S[a] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[a], __builtin_bit_cast(bf16x8, of[m]), S[a], 0, 0, 0);
      }
    } else {
#pragma unroll
      for (int x = 0; x < NH; ++x) {
        const float y = vf[x] * add[x];
#pragma unroll
        for (int a = 0; a < DK / 16; ++a)
          S[a] = __builtin_amdgcn_mfma_f32_16x16x4f32(Ks[held(x, g) * SQ + 16 * a + l], y, S[a], 0, 0, 0);
      }
    }

    if constexpr (kOut) {
#pragma unroll
      for (int it = 0; it < NT; ++it) {
#pragma unroll
        for (int r = 0; r < 4; ++r) bad = __builtin_fmaf(o[it][r], 0.0f, bad);
        if constexpr (kHalf)
          done[it] = __builtin_bit_cast(Four, __builtin_convertvector(o[it], bf16x4));
        else
          done[it] = __builtin_bit_cast(Four, o[it]);
      }
      done_n = n;
    }
  }
  if constexpr (kOut) store();

#pragma unroll
  for (int a = 0; a < DK / 16; ++a)
#pragma unroll
    for (int r = 0; r < 4; ++r) bad = __builtin_fmaf(S[a][r], 0.0f, bad);
  if (!kOut && tid == 0) w.flags[(int64_t)row * w.parts + part] = any != 0;
  if (16 * wave >= w.dv) return;
  if (__builtin_amdgcn_ballot_w64(bad != bad)) {
    serial<T, kOut>(w, row, 16 * wave, t0, t1, from, on_row, on_col, kOut ? nullptr : local, kOut && last);
    return;
  }
#pragma unroll
  for (int a = 0; a < DK / 16; ++a)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int k = 16 * a + 4 * g + r;
      if (k < w.dk && col < w.dv) {
        if (!kOut) local[(int64_t)k * w.dv + col] = S[a][r];
        if (kOut && last && w.state_out) w.state_out[state_index(w, row, k, col)] = S[a][r];
      }
    }
}

template <class T, int DK, int NW>
int launch_sized(Walks walks, bool out, hipStream_t s) {
  const Walk& w = walks.w[0];
  const int64_t rows = w.b * w.h, per = (int64_t)w.parts * walks.count, most = kMostThreads / (64 * NW) / per;
  for (int64_t row0 = 0; row0 < rows; row0 += most) {
    walks.w[0].row0 = walks.w[1].row0 = (uint32_t)row0;
    const dim3 grid((unsigned)((rows - row0 < most ? rows - row0 : most) * per)), block(64 * NW);
    if (out && w.backwards)
      hipLaunchKernelGGL((chunk_kernel<T, DK, NW, true, true>), grid, block, 0, s, walks);
    else if (out)
      hipLaunchKernelGGL((chunk_kernel<T, DK, NW, true, false>), grid, block, 0, s, walks);
    else if (w.backwards)
      hipLaunchKernelGGL((chunk_kernel<T, DK, NW, false, true>), grid, block, 0, s, walks);
    else
      hipLaunchKernelGGL((chunk_kernel<T, DK, NW, false, false>), grid, block, 0, s, walks);
    const int status = launch_status();
    if (status != HIPENVS_OK) return status;
  }
  return HIPENVS_OK;
}

// The kernel that takes dk rows and dv columns of a state: its rows, and its waves.
inline int rows_of(int dk) { return dk <= 32 ? 32 : dk <= 64 ? 64 : dk <= 96 ? 96 : 128; }
inline int waves_for(int dv) {
  const int waves = (dv + 15) / 16;
  return waves == 7 ? 8 : waves;
}

template <class T, int DK>
int of_rows(const Walks& walks, bool out, hipStream_t s) {
  switch (waves_for(walks.w[0].dv)) {
    case 1: return launch_sized<T, DK, 1>(walks, out, s);
    case 2: return launch_sized<T, DK, 2>(walks, out, s);
    case 3: return launch_sized<T, DK, 3>(walks, out, s);
    case 4: return launch_sized<T, DK, 4>(walks, out, s);
    case 5: return launch_sized<T, DK, 5>(walks, out, s);
    case 6: return launch_sized<T, DK, 6>(walks, out, s);
    default: return launch_sized<T, DK, 8>(walks, out, s);
  }
}

// These walks, all of one size of kernel: with outputs, or each part's own state alone.
template <class T>
int launch_walks(const Walks& walks, bool out, hipStream_t s) {
  switch (rows_of(walks.w[0].dk)) {
    case 32: return of_rows<T, 32>(walks, out, s);
    case 64: return of_rows<T, 64>(walks, out, s);
    case 96: return of_rows<T, 96>(walks, out, s);
    default: return of_rows<T, 128>(walks, out, s);
  }
}

// Each in a file of its own, which compile side by side.
#define HIPENVS_DA_ROWS(of, T, DK) of template int of_rows<T, DK>(const Walks&, bool, hipStream_t);
#ifndef HIPENVS_DA_DEFINE
HIPENVS_DA_ROWS(extern, __bf16, 32)
HIPENVS_DA_ROWS(extern, __bf16, 64)
HIPENVS_DA_ROWS(extern, __bf16, 96)
HIPENVS_DA_ROWS(extern, __bf16, 128)
HIPENVS_DA_ROWS(extern, float, 32)
HIPENVS_DA_ROWS(extern, float, 64)
HIPENVS_DA_ROWS(extern, float, 96)
HIPENVS_DA_ROWS(extern, float, 128)
#endif

}  // namespace da
}  // namespace hipenvs
