// Linear attention with a decay for each head and episodes inside its rows: over whole
// sequences, with its gradients, and for one token of every environment. No reference
// counterpart: the reference's policies have no memory.
//
//   S_t = (reset_t ? 0 : lambda S_{t-1}) + k_t v_t^T        o_t = scale S_t^T q_t
//
// lambda = exp(log_decay[h]); S is (dk, dv) in float32 for every row (b, h).
//
// One walk gives the outputs and every gradient. Forwards, it decays the state, adds
// add * k v^T and reads read * S^T q; backwards, it adds and reads first and decays after. With
// G_t = dL/dS_t = scale q_t do_t^T + (reset_{t+1} ? 0 : lambda G_{t+1}):
//
//   o  = walk(q, k, v) on S        dq = walk(do, v, k) on S^T            forwards
//   dv = walk(k, q, do) on G       dk = walk(v, do, q) on G^T            backwards
#include "hipenvs_device.h"

namespace hipenvs {
namespace da {

constexpr int kMaxDim = 128;

template <class T>
__device__ __forceinline__ float to_f32(T x);
template <>
__device__ __forceinline__ float to_f32<float>(float x) {
  return x;
}
template <>
__device__ __forceinline__ float to_f32<uint16_t>(uint16_t x) {
  return __uint_as_float((uint32_t)x << 16);
}

// Nearest even; a NaN stays a NaN.
__device__ __forceinline__ uint16_t bf16_of(float x) {
  const uint32_t u = __float_as_uint(x);
  return (uint16_t)(x != x ? ((u >> 16) | 0x40u) : (u + 0x7FFFu + ((u >> 16) & 1u)) >> 16);
}
template <class T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) {
  return x;
}
template <>
__device__ __forceinline__ uint16_t from_f32<uint16_t>(float x) {
  return bf16_of(x);
}

struct Rows {
  const void* data;
  int64_t sb, st, sh;   // strides in elements of a row's batch, token and head; the last is 1
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
  int64_t t;
  int32_t h;
};

// The walk, token by token: one wave for 16 columns of a row's state, a quarter of the rows of
// the state in each 16 lanes.
template <class T>
__global__ __launch_bounds__(64) void walk_kernel(Walk w) {
  const int col = blockIdx.y * 16 + (threadIdx.x & 15), part = threadIdx.x >> 4;
  const int64_t row = blockIdx.x;
  const int64_t b = row / w.h, h = row - b * w.h;
  const int per = (w.dk + 3) / 4, r0 = part * per;
  const bool live = col < w.dv;
  const float lambda = expf(w.log_decay[h]);
  const T* q = (const T*)w.q.data + b * w.q.sb + h * w.q.sh;
  const T* k = (const T*)w.k.data + b * w.k.sb + h * w.k.sh;
  const T* v = (const T*)w.v.data + b * w.v.sb + h * w.v.sh;
  float s[kMaxDim / 4];
#pragma unroll
  for (int i = 0; i < kMaxDim / 4; ++i) {
    const int r = r0 + i;
    s[i] = 0.0f;
    if (w.state_in && i < per && r < w.dk && live)
      s[i] = w.state_in[row * w.dk * w.dv + (w.flipped ? (int64_t)col * w.dk + r : (int64_t)r * w.dv + col)];
  }
  for (int64_t n = 0; n < w.t; ++n) {
    const int64_t t = w.backwards ? w.t - 1 - n : n;
    const bool fresh = w.reset && w.reset[b * w.reset_sb + t * w.reset_st];
    const float x = live ? w.add * to_f32<T>(v[t * w.v.st + col]) : 0.0f;
    float o = 0.0f;
#pragma unroll
    for (int i = 0; i < kMaxDim / 4; ++i) {
      const int r = r0 + i;
      if (i < per && r < w.dk) {
        if (!w.backwards) s[i] = fresh ? 0.0f : s[i] * lambda;
        s[i] = __builtin_fmaf(to_f32<T>(k[t * w.k.st + r]), x, s[i]);
        o = __builtin_fmaf(to_f32<T>(q[t * w.q.st + r]), s[i], o);
        if (w.backwards) s[i] = fresh ? 0.0f : s[i] * lambda;
      }
    }
    o += __shfl_xor(o, 16);
    o += __shfl_xor(o, 32);
    if (part == 0 && live) ((T*)w.out)[((b * w.t + t) * w.h + h) * w.dv + col] = from_f32<T>(w.read * o);
  }
  if (!w.state_out || !live) return;
#pragma unroll
  for (int i = 0; i < kMaxDim / 4; ++i) {
    const int r = r0 + i;
    if (i < per && r < w.dk)
      w.state_out[row * w.dk * w.dv + (w.flipped ? (int64_t)col * w.dk + r : (int64_t)r * w.dv + col)] = s[i];
  }
}

// One token of every environment: a block for each (n, h), the state read once and written
// once. `V` values of a state row at a time: L = ceil(dv / V) threads hold a row, 256 / L
// rows at a time; the rows' shares of the output meet in LDS. next may be state itself: a
// thread writes only what it has read.
struct Step {
  Rows q, k, v;   // sb: stride of the environment; st is not read
  const float* log_decay;
  const uint8_t* reset;
  int64_t reset_sn;
  const float* state;
  float* next;
  void* out;      // (n, h, dv) contiguous
  float scale;
  int32_t h, dk, dv;
};

template <class T, int V>
__global__ __launch_bounds__(kBlock) void step_kernel(Step s) {
  typedef float vec __attribute__((ext_vector_type(V)));
  __shared__ float share[kBlock * V];
  const int64_t item = blockIdx.x, n = item / s.h, h = item - n * s.h;
  const int L = (s.dv + V - 1) / V, R = kBlock / L;
  const int r0 = threadIdx.x / L, c = (threadIdx.x - r0 * L) * V;
  const T* q = (const T*)s.q.data + n * s.q.sb + h * s.q.sh;
  const T* k = (const T*)s.k.data + n * s.k.sb + h * s.k.sh;
  const T* v = (const T*)s.v.data + n * s.v.sb + h * s.v.sh;
  const bool fresh = s.reset && s.reset[n * s.reset_sn];
  const float lambda = expf(s.log_decay[h]);
  float x[V], o[V];
#pragma unroll
  for (int e = 0; e < V; ++e) o[e] = 0.0f;
  if (r0 < R) {
#pragma unroll
    for (int e = 0; e < V; ++e) x[e] = to_f32<T>(v[c + e]);
    const int64_t base = item * s.dk * s.dv + c;
    for (int r = r0; r < s.dk; r += R) {
      const float kr = to_f32<T>(k[r]), qr = to_f32<T>(q[r]);
      vec y = 0.0f;
      if (!fresh) y = *(const vec*)(s.state + base + (int64_t)r * s.dv);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float kept = fresh ? 0.0f : y[e] * lambda;
        y[e] = __builtin_fmaf(kr, x[e], kept);
        o[e] = __builtin_fmaf(qr, y[e], o[e]);
      }
      *(vec*)(s.next + base + (int64_t)r * s.dv) = y;
    }
#pragma unroll
    for (int e = 0; e < V; ++e) share[r0 * L * V + c + e] = o[e];
  }
  __syncthreads();
  for (int j = threadIdx.x; j < s.dv; j += kBlock) {
    float sum = 0.0f;
    const int rows = R < s.dk ? R : s.dk;
    for (int r = 0; r < rows; ++r) sum += share[r * L * V + j];
    ((T*)s.out)[item * s.dv + j] = from_f32<T>(s.scale * sum);
  }
}

bool dims_ok(int32_t dtype, int64_t h, int64_t dk, int64_t dv) {
  return (dtype == 0 || dtype == 1) && h >= 1 && h <= 65536 && dk >= 1 && dk <= kMaxDim && dv >= 1 && dv <= kMaxDim;
}

int launch_walk(int32_t dtype, const Walk& w, int64_t b, hipStream_t s) {
  const dim3 grid((unsigned)(b * w.h), (unsigned)((w.dv + 15) / 16)), block(64);
  if (dtype == 0)
    hipLaunchKernelGGL(walk_kernel<float>, grid, block, 0, s, w);
  else
    hipLaunchKernelGGL(walk_kernel<uint16_t>, grid, block, 0, s, w);
  return launch_status();
}

}  // namespace da
}  // namespace hipenvs

using namespace hipenvs;
using namespace hipenvs::da;

namespace {
// Rows of (b, h) within a grid, and a sequence whose contiguous outputs stay within 63 bits.
bool sequence_ok(int32_t dtype, int64_t b, int64_t t, int64_t h, int64_t dk, int64_t dv) {
  return dims_ok(dtype, h, dk, dv) && b >= 0 && t >= 0 && b * h <= 0x7FFFFFFF && b <= 0x7FFFFFFF && t <= 0x7FFFFFFF;
}

Rows rows(const void* data, const int64_t* strides) { return {data, strides[0], strides[1], strides[2]}; }
}  // namespace

extern "C" int hipenvs_decay_attention(int32_t dtype, const void* q, const void* k, const void* v,
                                       const int64_t* strides, const float* log_decay, const float* state,
                                       const uint8_t* reset, float scale, void* out, float* final_state, int64_t b,
                                       int64_t t, int32_t h, int32_t dk, int32_t dv, hipenvs_stream_t stream) {
  if (!sequence_ok(dtype, b, t, h, dk, dv)) return HIPENVS_E_ARG;
  if (b == 0) return HIPENVS_OK;
  if (!log_decay || !final_state || (t > 0 && (!q || !k || !v || !out || !strides))) return HIPENVS_E_ARG;
  static const int64_t none[11] = {};
  const int64_t* st = t > 0 ? strides : none;
  Walk w = {rows(q, st), rows(k, st + 3), rows(v, st + 6), dk, dv, log_decay, reset, st[9], st[10],
            state, final_state, false, false, scale, 1.0f, out, t, h};
  return launch_walk(dtype, w, b, as_stream(stream));
}

extern "C" int hipenvs_decay_attention_backward(int32_t dtype, const void* q, const void* k, const void* v,
                                                const void* dout, const int64_t* strides, const float* log_decay,
                                                const float* state, const uint8_t* reset, const float* dfinal,
                                                float scale, void* dq, void* dk_out, void* dv_out, float* dstate,
                                                int64_t b, int64_t t, int32_t h, int32_t dk, int32_t dv,
                                                hipenvs_stream_t stream) {
  if (!sequence_ok(dtype, b, t, h, dk, dv)) return HIPENVS_E_ARG;
  if (b == 0) return HIPENVS_OK;
  if (!log_decay || !dstate || (t > 0 && (!q || !k || !v || !dout || !dq || !dk_out || !dv_out || !strides)))
    return HIPENVS_E_ARG;
  static const int64_t none[14] = {};
  const int64_t* st = t > 0 ? strides : none;
  const Rows rq = rows(q, st), rk = rows(k, st + 3), rv = rows(v, st + 6), rdo = rows(dout, st + 9);
  const hipStream_t s = as_stream(stream);
  const Walk by_q = {rdo, rv, rk, dv, dk, log_decay, reset, st[12], st[13], state, nullptr, true, false, scale, 1.0f,
                     dq, t, h};
  const Walk by_v = {rk, rq, rdo, dk, dv, log_decay, reset, st[12], st[13], dfinal, dstate, false, true, 1.0f, scale,
                     dv_out, t, h};
  const Walk by_k = {rv, rdo, rq, dv, dk, log_decay, reset, st[12], st[13], dfinal, nullptr, true, true, 1.0f, scale,
                     dk_out, t, h};
  int status = launch_walk(dtype, by_q, b, s);
  if (status == HIPENVS_OK) status = launch_walk(dtype, by_v, b, s);
  if (status == HIPENVS_OK) status = launch_walk(dtype, by_k, b, s);
  return status;
}

extern "C" int hipenvs_decay_attention_step(int32_t dtype, const void* q, int64_t q_sn, int64_t q_sh, const void* k,
                                            int64_t k_sn, int64_t k_sh, const void* v, int64_t v_sn, int64_t v_sh,
                                            const float* log_decay, const float* state, const uint8_t* reset,
                                            int64_t reset_sn, float scale, void* out, float* next_state, int64_t n,
                                            int32_t h, int32_t dk, int32_t dv, hipenvs_stream_t stream) {
  if (!dims_ok(dtype, h, dk, dv) || n < 0 || n > 0x7FFFFFFF || n * h > 0x7FFFFFFF) return HIPENVS_E_ARG;
  if (n == 0) return HIPENVS_OK;
  if (!q || !k || !v || !log_decay || !state || !out || !next_state) return HIPENVS_E_ARG;
  const Step s = {{q, q_sn, 0, q_sh}, {k, k_sn, 0, k_sh}, {v, v_sn, 0, v_sh}, log_decay, reset, reset_sn,
                  state, next_state, out, scale, h, dk, dv};
  const bool wide = dv % 4 == 0 && (((uintptr_t)state | (uintptr_t)next_state) & 15) == 0;
  const dim3 grid((unsigned)(n * h)), block(kBlock);
  const hipStream_t at = as_stream(stream);
  if (dtype == 0 && wide) hipLaunchKernelGGL((step_kernel<float, 4>), grid, block, 0, at, s);
  if (dtype == 0 && !wide) hipLaunchKernelGGL((step_kernel<float, 1>), grid, block, 0, at, s);
  if (dtype == 1 && wide) hipLaunchKernelGGL((step_kernel<uint16_t, 4>), grid, block, 0, at, s);
  if (dtype == 1 && !wide) hipLaunchKernelGGL((step_kernel<uint16_t, 1>), grid, block, 0, at, s);
  return launch_status();
}
