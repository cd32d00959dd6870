// Linear attention with a decay for each head (decay_attention.h): the C entry points, the
// joining of a sequence's parts, and one token of every environment.
#include "decay_attention.h"

namespace hipenvs {
namespace da {

// From each part's own state (what its tokens alone leave behind) to the state before each
// part, in the order of the walk: carry' = lambda^tokens carry [no reset] + own. A thread for
// each value of a row's state, eight parts' values read ahead of their use.
__global__ __launch_bounds__(kBlock) void join_kernel(Walk w) {
  const int size = w.dk * w.dv, at = blockIdx.y * kBlock + threadIdx.x;
  if (at >= size) return;
  const int64_t row = blockIdx.x, h = row % w.h;
  const float ld = w.log_decay[h];
  float* states = w.states + row * w.parts * size + at;
  const uint8_t* flags = w.flags + row * w.parts;
  float carry = w.state_in ? w.state_in[state_index(w, row, at / w.dv, at % w.dv)] : 0.0f;
  constexpr int kAhead = 8;
  for (int n0 = 0; n0 < w.parts; n0 += kAhead) {
    float own[kAhead];
    bool reset[kAhead];
#pragma unroll
    for (int e = 0; e < kAhead; ++e) {
      const int n = n0 + e, p = w.backwards ? w.parts - 1 - n : n;
      own[e] = n < w.parts ? states[(int64_t)p * size] : 0.0f;
      reset[e] = n < w.parts ? flags[p] != 0 : false;
    }
#pragma unroll
    for (int e = 0; e < kAhead; ++e) {
      const int n = n0 + e, p = w.backwards ? w.parts - 1 - n : n;
      if (n >= w.parts) break;
      states[(int64_t)p * size] = carry;
      const int64_t left = w.t - (int64_t)p * w.part, tokens = left < w.part ? left : w.part;
      carry = (reset[e] ? 0.0f : carry * expf(ld * (float)tokens)) + own[e];
    }
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

// A block walks a row, or a part of one where the rows are too few to fill the card: then a first
// pass leaves each part's own state, the second joins them, the third walks every part from
// the state before it.
void divide(int64_t rows, int64_t t, int32_t chunk, int64_t cus, int32_t* parts, int64_t* part) {
  const int64_t chunks = (t + chunk - 1) / chunk;
  const int64_t want = (2 * cus + rows - 1) / rows, most = chunks / 4;
  int64_t n = want < most ? want : most;
  if (n < 2) n = 1;
  const int64_t per = n > 1 ? (chunks + n - 1) / n : chunks;
  *parts = n > 1 ? (int32_t)((chunks + per - 1) / per) : 1;
  *part = (per > 0 ? per : 1) * chunk;
}

int32_t chunk_of(int32_t dtype) { return dtype == 1 ? Chunk<__bf16>::kTokens : Chunk<float>::kTokens; }

int launch_walk(int32_t dtype, Walk w, hipStream_t s) {
  if (w.parts > 1) {
    int status = dtype == 1 ? launch_chunks<__bf16>(w, false, s) : launch_chunks<float>(w, false, s);
    if (status != HIPENVS_OK) return status;
    hipLaunchKernelGGL(join_kernel, dim3((unsigned)(w.b * w.h), grid_for(w.dk * w.dv)), dim3(kBlock), 0, s, w);
    status = launch_status();
    if (status != HIPENVS_OK) return status;
  }
  return dtype == 1 ? launch_chunks<__bf16>(w, true, s) : launch_chunks<float>(w, true, s);
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

// `d` values a row of `size` bytes each.
Rows rows(const void* data, const int64_t* strides, int64_t size, int64_t d) {
  const bool wide = (((uintptr_t)data | (uintptr_t)(strides[0] * size) | (uintptr_t)(strides[1] * size) |
                      (uintptr_t)(strides[2] * size) | (uintptr_t)(d * size)) & 15) == 0;
  return {data, strides[0], strides[1], strides[2], wide};
}

// The parts of a sequence and where in `workspace` their states and flags lie; the bytes used.
int plan(int32_t dtype, int64_t b, int64_t t, int32_t h, int32_t dk, int32_t dv, void* workspace, Walk* w,
         int64_t* bytes) {
  int cus = 0;
  const int status = device_cus(&cus);
  if (status != HIPENVS_OK) return status;
  divide(b * h, t, chunk_of(dtype), cus, &w->parts, &w->part);
  const int64_t states = w->parts > 1 ? b * h * w->parts * dk * dv * (int64_t)sizeof(float) : 0;
  w->states = (float*)workspace;
  w->flags = (uint8_t*)workspace + states;
  *bytes = w->parts > 1 ? states + b * h * w->parts : 0;
  return HIPENVS_OK;
}
}  // namespace

extern "C" int64_t hipenvs_decay_attention_workspace_bytes(int32_t dtype, int64_t b, int64_t t, int32_t h, int32_t dk,
                                                           int32_t dv) {
  if (!sequence_ok(dtype, b, t, h, dk, dv)) return -1;
  if (b == 0) return 0;
  Walk w = {};
  int64_t bytes = 0;
  return plan(dtype, b, t, h, dk, dv, nullptr, &w, &bytes) == HIPENVS_OK ? bytes : -1;
}

extern "C" int hipenvs_decay_attention(int32_t dtype, const void* q, const void* k, const void* v,
                                       const int64_t* strides, const float* log_decay, const float* state,
                                       const uint8_t* reset, float scale, void* out, float* final_state, int64_t b,
                                       int64_t t, int32_t h, int32_t dk, int32_t dv, void* workspace,
                                       int64_t workspace_bytes, hipenvs_stream_t stream) {
  if (!sequence_ok(dtype, b, t, h, dk, dv)) return HIPENVS_E_ARG;
  if (b == 0) return HIPENVS_OK;
  if (!log_decay || !final_state || (t > 0 && (!q || !k || !v || !out || !strides))) return HIPENVS_E_ARG;
  static const int64_t none[11] = {};
  const int64_t* st = t > 0 ? strides : none;
  const int64_t e = dtype == 1 ? 2 : 4;
  Walk w = {};
  int64_t need = 0;
  const int status = plan(dtype, b, t, h, dk, dv, workspace, &w, &need);
  if (status != HIPENVS_OK) return status;
  if (need > 0 && (!workspace || workspace_bytes < need)) return HIPENVS_E_ARG;
  w.q = rows(q, st, e, dk), w.k = rows(k, st + 3, e, dk), w.v = rows(v, st + 6, e, dv);
  w.dk = dk, w.dv = dv, w.log_decay = log_decay, w.reset = reset, w.reset_sb = st[9], w.reset_st = st[10];
  w.state_in = state, w.state_out = final_state, w.read = scale, w.add = 1.0f;
  w.out = out, w.b = b, w.t = t, w.h = h;
  return launch_walk(dtype, w, as_stream(stream));
}

extern "C" int hipenvs_decay_attention_backward(int32_t dtype, const void* q, const void* k, const void* v,
                                                const void* dout, const int64_t* strides, const float* log_decay,
                                                const float* state, const uint8_t* reset, const float* dfinal,
                                                float scale, void* dq, void* dk_out, void* dv_out, float* dstate,
                                                int64_t b, int64_t t, int32_t h, int32_t dk, int32_t dv,
                                                void* workspace, int64_t workspace_bytes, hipenvs_stream_t stream) {
  if (!sequence_ok(dtype, b, t, h, dk, dv)) return HIPENVS_E_ARG;
  if (b == 0) return HIPENVS_OK;
  if (!log_decay || !dstate || (t > 0 && (!q || !k || !v || !dout || !dq || !dk_out || !dv_out || !strides)))
    return HIPENVS_E_ARG;
  static const int64_t none[14] = {};
  const int64_t* st = t > 0 ? strides : none;
  const int64_t e = dtype == 1 ? 2 : 4;
  Walk w = {};
  int64_t need = 0;
  int status = plan(dtype, b, t, h, dk, dv, workspace, &w, &need);
  if (status != HIPENVS_OK) return status;
  if (need > 0 && (!workspace || workspace_bytes < need)) return HIPENVS_E_ARG;
  const Rows rq = rows(q, st, e, dk), rk = rows(k, st + 3, e, dk), rv = rows(v, st + 6, e, dv),
             rdo = rows(dout, st + 9, e, dv);
  const hipStream_t s = as_stream(stream);
  w.log_decay = log_decay, w.reset = reset, w.reset_sb = st[12], w.reset_st = st[13], w.b = b, w.t = t, w.h = h;
  // dq: forwards over the transposed states
  w.q = rdo, w.k = rv, w.v = rk, w.dk = dv, w.dv = dk, w.state_in = state, w.state_out = nullptr;
  w.flipped = true, w.backwards = false, w.read = scale, w.add = 1.0f, w.out = dq;
  status = launch_walk(dtype, w, s);
  if (status != HIPENVS_OK) return status;
  // dv, and the gradient of the first state: backwards over the states' gradients
  w.q = rk, w.k = rq, w.v = rdo, w.dk = dk, w.dv = dv, w.state_in = dfinal, w.state_out = dstate;
  w.flipped = false, w.backwards = true, w.read = 1.0f, w.add = scale, w.out = dv_out;
  status = launch_walk(dtype, w, s);
  if (status != HIPENVS_OK) return status;
  // dk: the same, transposed
  w.q = rv, w.k = rdo, w.v = rq, w.dk = dv, w.dv = dk, w.state_out = nullptr, w.flipped = true, w.out = dk_out;
  return launch_walk(dtype, w, s);
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
  if (dtype == 1 && wide) hipLaunchKernelGGL((step_kernel<__bf16, 4>), grid, block, 0, at, s);
  if (dtype == 1 && !wide) hipLaunchKernelGGL((step_kernel<__bf16, 1>), grid, block, 0, at, s);
  return launch_status();
}
