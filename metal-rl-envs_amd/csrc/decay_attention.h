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
  bool wide;           // every row begins at a multiple of 16 bytes and is whole 16-byte pieces
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
  float* states;           // (b h, parts, dk, dv)
  uint8_t* flags;          // (b h, parts): a reset in the part
};

// Values of a state in its caller's layout.
__device__ __forceinline__ int64_t state_index(const Walk& w, int64_t row, int r, int c) {
  return row * w.dk * w.dv + (w.flipped ? (int64_t)c * w.dk + r : (int64_t)r * w.dv + c);
}

// Tokens [t0, t1) of a row one after another, for the 16 columns of one wave, four at a time:
// column c of the four in each 16 lanes, an eighth of 128 rows of the state in each lane. The
// chunked form meets zero weights with whatever their tokens hold, and 0 * NaN is not 0; so a
// wave that finds anything but finite numbers in its outputs or its state walks its part
// again here, where a token takes part only where it counts. It starts from what the
// chunked form started from: `from` (rows, columns), else the caller's state, or zeros. A path
// for data that has gone wrong: small in registers, not fast.
template <class T, bool kOut>
__device__ __forceinline__ void serial(const Walk& w, int64_t row, int col0, int64_t t0, int64_t t1, const float* from,
                                    bool zero, float* to, bool last) {
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
      if (!zero && r < w.dk && live)
        s[i] = from ? from[(int64_t)r * w.dv + col] : w.state_in ? w.state_in[state_index(w, row, r, col)] : 0.0f;
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

// Tokens a chunk holds and the padding of its LDS rows, which keeps 16 rows read at one column
// on different banks.
template <class T>
struct Chunk;
template <>
struct Chunk<__bf16> {
  static constexpr int kTokens = 64, kPad = 8;
};
template <>
struct Chunk<float> {
  static constexpr int kTokens = 32, kPad = 4;
};

// One 16-byte piece of a token's row, zeros where the row has ended.
template <class T>
__device__ __forceinline__ u32x4 load_piece(const T* row, int col, int dim, bool wide) {
  constexpr int E = 16 / sizeof(T);
  u32x4 x = {0, 0, 0, 0};
  if (wide) {
    if (col < dim) x = *(const u32x4*)(row + col);
  } else {
    T* y = (T*)&x;
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (col + e < dim) y[e] = row[col + e];
  }
  return x;
}

__device__ __forceinline__ bf16x8 join(i16x4 a, i16x4 b) {
  const bf16x4 x = __builtin_bit_cast(bf16x4, a), y = __builtin_bit_cast(bf16x4, b);
  return __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
}

// Columns col .. col + 15 of rows row .. row + 7 of a bfloat16 tile, rows differing between
// the four groups of 16 lanes: lane l of a group gets column col + l, its 8 rows in order. A
// transposing read gives a group 16 columns of 4 rows, each of its lanes addressing 4 values.
__device__ __forceinline__ bf16x8 read_columns(const __bf16* tile, int stride, int row, int col) {
  const int l = threadIdx.x & 15;
  const __bf16* p = tile + (row + (l >> 2)) * stride + col + 4 * (l & 3);
  typedef __attribute__((address_space(3))) i16x4* lds4;
  return join(__builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)p),
              __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(p + 4 * stride)));
}

// The bfloat16 parts of N (even) float32 values: of each, the rounding of what is left.
template <int M, int N>
__device__ __forceinline__ void split(float (&rest)[N], __bf16 (&parts)[M][N]) {
#pragma unroll
  for (int m = 0; m < M; ++m)
#pragma unroll
    for (int e = 0; e < N; e += 2) {
      const f32x2 x = {rest[e], rest[e + 1]};
      const bf16x2 y = __builtin_convertvector(x, bf16x2);
      parts[m][e] = y[0], parts[m][e + 1] = y[1];
      rest[e] -= (float)y[0], rest[e + 1] -= (float)y[1];
    }
}

// A wave takes 16 columns of the state, all of its rows: S[a][r] is row 16 a + 4 g + r, column
// l, for lane 16 g + l. That is both a matrix instruction's result and, its rows
// taken as the summed axis in that order, an operand of the read S^T q, so the state never
// leaves its registers. The block's NW waves share a chunk's q, k, v (LDS, two buffers: while
// one chunk is computed the next is on its way to registers) and its masked products
// P[i][j], computed once.
//
// bfloat16 rows: the inputs are exact operands. P, the S that is read and the lambda^n v_j that
// is added are float32, split for the matrix instructions into bfloat16 parts, each the
// rounding of what the parts before it leave: two parts for P and S (16 bits, so a result's
// error is that of its own rounding to bfloat16), three for what enters a state (all 24 bits: a
// state is a float32 result). float32 rows use the float32 matrix instructions throughout.
template <class T, int DK, int NW, bool kOut>
__global__ __launch_bounds__(64 * NW) void chunk_kernel(Walk w) {
  constexpr bool kHalf = sizeof(T) == 2;
  constexpr int C = Chunk<T>::kTokens, PAD = Chunk<T>::kPad, E = 16 / sizeof(T), TH = 64 * NW, DV = 16 * NW;
  constexpr int SQ = DK + PAD, SV = DV + PAD, SP = C + PAD, NT = C / 16;
  constexpr int QP = DK / E, VP = DV / E;                               // pieces of a row
  constexpr int NQ = (C * QP + TH - 1) / TH, NV = (C * VP + TH - 1) / TH;  // pieces of a thread
  __shared__ __attribute__((aligned(16))) T Qs[kOut ? 2 * C * SQ : 8];
  __shared__ __attribute__((aligned(16))) T Ks[2 * C * SQ];
  __shared__ __attribute__((aligned(16))) T Vs[2 * C * SV];
  __shared__ __attribute__((aligned(16))) T Ps[kOut ? (kHalf ? 2 : 1) * C * SP : 8];
  __shared__ float pw[C + 1];
  __shared__ __attribute__((aligned(16))) float wu[2 * C];

  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, g = lane >> 4, l = lane & 15;
  // blocks of one XCD (every eighth) take neighbouring rows, whose tokens share cache lines
  const int64_t blocks = gridDim.x;
  const int64_t id = blocks % 8 == 0 ? (int64_t)(blockIdx.x % 8) * (blocks / 8) + blockIdx.x / 8 : blockIdx.x;
  const int64_t row = id / w.parts;
  const int part = (int)(id - row * w.parts);
  const int64_t b = row / w.h, h = row - b * w.h;
  const int64_t t0 = part * w.part, t1 = t0 + w.part < w.t ? t0 + w.part : w.t;
  const int64_t chunks = (t1 - t0 + C - 1) / C;
  const bool back = w.backwards;
  const bool first = part == (back ? w.parts - 1 : 0), last = part == (back ? 0 : w.parts - 1);
  const float ld = w.log_decay[h];
  const T* qrow = (const T*)w.q.data + b * w.q.sb + h * w.q.sh;
  const T* krow = (const T*)w.k.data + b * w.k.sb + h * w.k.sh;
  const T* vrow = (const T*)w.v.data + b * w.v.sb + h * w.v.sh;
  float* local = w.parts > 1 ? w.states + (row * w.parts + part) * w.dk * w.dv : nullptr;

  for (int n = tid; n <= C; n += TH) pw[n] = n == 0 ? 1.0f : expf(ld * (float)n);

  f32x4 S[DK / 16];
  const int col = 16 * wave + l;
#pragma unroll
  for (int a = 0; a < DK / 16; ++a)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int k = 16 * a + 4 * g + r;
      float x = 0.0f;
      if (kOut && k < w.dk && col < w.dv)
        x = local ? local[(int64_t)k * w.dv + col] : w.state_in ? w.state_in[state_index(w, row, k, col)] : 0.0f;
      S[a][r] = x;
    }

  u32x4 xq[kOut ? NQ : 1], xk[NQ], xv[NV];
  uint32_t xr = 0;
  const auto load = [&](int64_t c) {
    const int64_t at = t0 + c * C;
    const int n = (int)(t1 - at < C ? t1 - at : C);
#pragma unroll
    for (int m = 0; m < NQ; ++m) {
      const int p = tid + m * TH, r = p / QP, x = (p - r * QP) * E;
      const u32x4 none = {0, 0, 0, 0};
      xk[m] = none;
      if constexpr (kOut) xq[m] = none;
      if (r < n) {
        xk[m] = load_piece<T>(krow + (at + r) * w.k.st, x, w.dk, w.k.wide);
        if constexpr (kOut) xq[m] = load_piece<T>(qrow + (at + r) * w.q.st, x, w.dk, w.q.wide);
      }
    }
#pragma unroll
    for (int m = 0; m < NV; ++m) {
      const int p = tid + m * TH, r = p / VP, x = (p - r * VP) * E;
      const u32x4 none = {0, 0, 0, 0};
      xv[m] = none;
      if (r < n) xv[m] = load_piece<T>(vrow + (at + r) * w.v.st, x, w.dv, w.v.wide);
    }
    xr = 0;
    if (w.reset && lane < n) xr = w.reset[b * w.reset_sb + (at + lane) * w.reset_st];
  };

  uint64_t any = 0;
  float bad = 0.0f;   // becomes NaN with the first value that is not finite
  if (chunks > 0) load(back ? chunks - 1 : 0);
  for (int64_t step = 0; step < chunks; ++step) {
    const int64_t c = back ? chunks - 1 - step : step, at = t0 + c * C;
    const int n = (int)(t1 - at < C ? t1 - at : C);
    const int buf = (int)(step & 1);
    T* Kb = Ks + buf * C * SQ;
    T* Vb = Vs + buf * C * SV;
    T* Qb = kOut ? Qs + buf * C * SQ : Qs;
    float* wb = wu + buf * C;
#pragma unroll
    for (int m = 0; m < NQ; ++m) {
      const int p = tid + m * TH, r = p / QP, x = (p - r * QP) * E;
      if (r < C) {
        *(u32x4*)(Kb + r * SQ + x) = xk[m];
        if constexpr (kOut) *(u32x4*)(Qb + r * SQ + x) = xq[m];
      }
    }
#pragma unroll
    for (int m = 0; m < NV; ++m) {
      const int p = tid + m * TH, r = p / VP, x = (p - r * VP) * E;
      if (r < C) *(u32x4*)(Vb + r * SV + x) = xv[m];
    }
    // the chunk's resets, bit i for token i; the first and the last of them
    const uint64_t mask = __builtin_amdgcn_ballot_w64(xr != 0);
    any |= mask;
    const int r_first = mask ? __builtin_ctzll(mask) : C, r_last = mask ? 63 - __builtin_clzll(mask) : -1;
    if (step == 0) __syncthreads();   // pw
    if (tid < C) {
      const int j = tid;
      float x = 0.0f;
      if (j < n) x = back ? (j < r_first ? w.add * pw[j + 1] : 0.0f) : (j >= r_last ? w.add * pw[n - 1 - j] : 0.0f);
      wb[j] = x;
    }
    __syncthreads();
    if (step + 1 < chunks) load(back ? chunks - 2 - step : step + 1);

    if constexpr (kOut) {
      // P[i][j], the tiles of 16 queries x 16 keys dealt to the waves
      constexpr int H = NW > NT ? NW / NT : 1;
      const int it0 = wave % NT, jt0 = wave / NT;
      for (int it = it0; it < NT && jt0 < H; it += NW) {
        const int i = 16 * it + l;
        const uint64_t upto = mask & ((2ull << i) - 1), after = i < 63 ? mask >> (i + 1) : 0;
        const int from = upto ? 63 - __builtin_clzll(upto) : 0, until = after ? i + 1 + __builtin_ctzll(after) : C;
#pragma unroll
        for (int jt = 0; jt < NT; ++jt) {
          if (jt % H != jt0) continue;
          T* to = Ps + i * SP + 16 * jt + 4 * g;
          if (back ? jt < it : jt > it) {
            if constexpr (kHalf) {
              if ((jt ^ it) == 1) {   // the other half of a 32-key product
                const u32x2 none = {0, 0};
                *(u32x2*)to = none;
                *(u32x2*)(to + C * SP) = none;
              }
            }
            continue;
          }
          f32x4 p = {0.0f, 0.0f, 0.0f, 0.0f};
          if constexpr (kHalf) {
#pragma unroll
            for (int s = 0; s < DK / 32; ++s) {
              const bf16x8 kf = *(const bf16x8*)(Kb + (16 * jt + l) * SQ + 32 * s + 8 * g);
              const bf16x8 qf = *(const bf16x8*)(Qb + i * SQ + 32 * s + 8 * g);
              p = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qf, p, 0, 0, 0);
            }
          } else {
#pragma unroll
            for (int s = 0; s < DK / 16; ++s) {
              const f32x4 kf = *(const f32x4*)(Kb + (16 * jt + l) * SQ + 16 * s + 4 * g);
              const f32x4 qf = *(const f32x4*)(Qb + i * SQ + 16 * s + 4 * g);
#pragma unroll
              for (int e = 0; e < 4; ++e) p = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[e], qf[e], p, 0, 0, 0);
            }
          }
          f32x4 y;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int j = 16 * jt + 4 * g + r, gap = back ? j - i : i - j;
            const bool seen = back ? j < until : j >= from;
            y[r] = gap >= 0 && seen ? p[r] * (w.read * w.add * pw[gap < 0 ? 0 : gap]) : 0.0f;
          }
          if constexpr (kHalf) {
            float rest[4] = {y[0], y[1], y[2], y[3]};
            __bf16 of[2][4];
            split(rest, of);
            *(bf16x4*)to = __builtin_bit_cast(bf16x4, of[0]);
            *(bf16x4*)(to + C * SP) = __builtin_bit_cast(bf16x4, of[1]);
          } else {
            *(f32x4*)to = y;
          }
        }
      }
      __syncthreads();
    }

    // this wave's columns of v, and its share of the products
    bf16x8 vh[kHalf ? C / 32 : 1];
    float vf[kHalf ? 1 : C / 4];
    if constexpr (kHalf) {
#pragma unroll
      for (int s = 0; s < C / 32; ++s) vh[s] = read_columns(Vb, SV, 32 * s + 8 * g, 16 * wave);
    } else {
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) vf[4 * t + e] = Vb[(16 * t + 4 * g + e) * SV + col];
    }

    if constexpr (kOut) {
      bf16x8 sh[kHalf ? DK / 32 : 1][2];
      if constexpr (kHalf) {
#pragma unroll
        for (int a = 0; a < DK / 32; ++a) {
          float rest[8];
          __bf16 of[2][8];
#pragma unroll
          for (int e = 0; e < 8; ++e) rest[e] = S[2 * a + e / 4][e % 4];
          split(rest, of);
          sh[a][0] = __builtin_bit_cast(bf16x8, of[0]), sh[a][1] = __builtin_bit_cast(bf16x8, of[1]);
        }
      }
#pragma unroll
      for (int it = 0; it < NT; ++it) {
        if (16 * it >= n) continue;
        const int i = 16 * it + l;
        f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
        if (back ? r_last < 16 * it + 16 : r_first > 16 * it) {   // some token of the tile sees S
          if constexpr (kHalf) {
#pragma unroll
            for (int a = 0; a < DK / 32; ++a) {
              const __bf16* at_q = Qb + i * SQ + 32 * a + 4 * g;
              const bf16x8 qf = __builtin_shufflevector(*(const bf16x4*)at_q, *(const bf16x4*)(at_q + 16), 0, 1, 2, 3,
                                                        4, 5, 6, 7);
              o = __builtin_amdgcn_mfma_f32_16x16x32_bf16(sh[a][0], qf, o, 0, 0, 0);
              o = __builtin_amdgcn_mfma_f32_16x16x32_bf16(sh[a][1], qf, o, 0, 0, 0);
            }
          } else {
#pragma unroll
            for (int a = 0; a < DK / 16; ++a) {
              const f32x4 qf = *(const f32x4*)(Qb + i * SQ + 16 * a + 4 * g);
#pragma unroll
              for (int e = 0; e < 4; ++e) o = __builtin_amdgcn_mfma_f32_16x16x4f32(S[a][e], qf[e], o, 0, 0, 0);
            }
          }
          const bool sees = back ? i >= r_last : i < r_first;
          const int gap = back ? n - 1 - i : i + 1;
          const float f = w.read * pw[gap < 0 ? 0 : gap];
#pragma unroll
          for (int r = 0; r < 4; ++r) o[r] = sees ? o[r] * f : 0.0f;
        }
        if constexpr (kHalf) {
#pragma unroll
          for (int s = 0; s < C / 32; ++s)
            if (back ? 2 * s + 1 >= it : 2 * s <= it) {
              const T* p = Ps + i * SP + 32 * s + 8 * g;
              o = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vh[s], *(const bf16x8*)p, o, 0, 0, 0);
              o = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vh[s], *(const bf16x8*)(p + C * SP), o, 0, 0, 0);
            }
        } else {
#pragma unroll
          for (int t = 0; t < NT; ++t)
            if (back ? t >= it : t <= it) {
              const f32x4 p = *(const f32x4*)(Ps + i * SP + 16 * t + 4 * g);
#pragma unroll
              for (int e = 0; e < 4; ++e) o = __builtin_amdgcn_mfma_f32_16x16x4f32(vf[4 * t + e], p[e], o, 0, 0, 0);
            }
        }
        if (i < n) {
          const int c0 = 16 * wave + 4 * g;
          T* to = (T*)w.out + ((b * w.t + at + i) * w.h + h) * w.dv + c0;
#pragma unroll
          for (int r = 0; r < 4; ++r) bad = __builtin_fmaf(o[r], 0.0f, bad);
          if (w.dv % 4 == 0) {
            if (c0 < w.dv) {
              if constexpr (kHalf)
                *(bf16x4*)to = __builtin_convertvector(o, bf16x4);
              else
                *(f32x4*)to = o;
            }
          } else {
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (c0 + r < w.dv) to[r] = from_f32<T>(o[r]);
          }
        }
      }
    }

    // the state after the chunk
    const float keep = pw[n];
#pragma unroll
    for (int a = 0; a < DK / 16; ++a)
#pragma unroll
      for (int r = 0; r < 4; ++r) S[a][r] = mask ? 0.0f : S[a][r] * keep;
    if constexpr (kHalf) {
#pragma unroll
      for (int s = 0; s < C / 32; ++s) {
        if (32 * s >= n) continue;
        const f32x4 w0 = *(const f32x4*)(wb + 32 * s + 8 * g), w1 = *(const f32x4*)(wb + 32 * s + 8 * g + 4);
        float rest[8];
        __bf16 of[3][8];
#pragma unroll
        for (int e = 0; e < 8; ++e) rest[e] = (float)vh[s][e] * (e < 4 ? w0[e & 3] : w1[e & 3]);
        split(rest, of);
#pragma unroll
        for (int a = 0; a < DK / 16; ++a) {
          const bf16x8 kf = read_columns(Kb, SQ, 32 * s + 8 * g, 16 * a);
#pragma unroll
          for (int m = 0; m < 3; ++m)
            S[a] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, __builtin_bit_cast(bf16x8, of[m]), S[a], 0, 0, 0);
        }
      }
    } else {
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        if (16 * t >= n) continue;
        const f32x4 x = *(const f32x4*)(wb + 16 * t + 4 * g);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float y = vf[4 * t + e] * x[e];
#pragma unroll
          for (int a = 0; a < DK / 16; ++a)
            S[a] = __builtin_amdgcn_mfma_f32_16x16x4f32(Kb[(16 * t + 4 * g + e) * SQ + 16 * a + l], y, S[a], 0, 0, 0);
        }
      }
    }
  }

#pragma unroll
  for (int a = 0; a < DK / 16; ++a)
#pragma unroll
    for (int r = 0; r < 4; ++r) bad = __builtin_fmaf(S[a][r], 0.0f, bad);
  if (!kOut && tid == 0) w.flags[row * w.parts + part] = any != 0;
  if (16 * wave >= w.dv) return;
  if (__builtin_amdgcn_ballot_w64(bad != bad)) {
    serial<T, kOut>(w, row, 16 * wave, t0, t1, kOut ? local : nullptr, !kOut, kOut ? nullptr : local, kOut && last);
    return;
  }
  (void)first;
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
int launch_sized(const Walk& w, bool out, hipStream_t s) {
  const dim3 grid((unsigned)(w.b * w.h * w.parts)), block(64 * NW);
  if (out)
    hipLaunchKernelGGL((chunk_kernel<T, DK, NW, true>), grid, block, 0, s, w);
  else
    hipLaunchKernelGGL((chunk_kernel<T, DK, NW, false>), grid, block, 0, s, w);
  return launch_status();
}

template <class T, int DK>
int launch_rows(const Walk& w, bool out, hipStream_t s) {
  if (w.dv <= 32) return launch_sized<T, DK, 2>(w, out, s);
  if (w.dv <= 64) return launch_sized<T, DK, 4>(w, out, s);
  return launch_sized<T, DK, 8>(w, out, s);
}

// The walk's kernel for w.dk and w.dv: with outputs, or each part's own state alone.
template <class T>
int launch_chunks(const Walk& w, bool out, hipStream_t s) {
  if (w.dk <= 32) return launch_rows<T, 32>(w, out, s);
  if (w.dk <= 64) return launch_rows<T, 64>(w, out, s);
  return launch_rows<T, 128>(w, out, s);
}

extern template int launch_chunks<__bf16>(const Walk&, bool, hipStream_t);
extern template int launch_chunks<float>(const Walk&, bool, hipStream_t);

}  // namespace da
}  // namespace hipenvs
