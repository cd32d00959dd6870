// Linear attention with a decay for each head (decay_attention.h): the C entry points, the
// joining of a sequence's parts, and one token of every environment.
#include "decay_attention.h"

namespace hipenvs {
namespace da {

// From each part's own state (what its tokens alone leave behind) to the state before each
// part, in the order of the walk: carry' = lambda^tokens carry [no reset] + own. `groups`
// threads (1 to 8) take one value of a row's state, eight parts each: a thread reads its parts at
// once and composes them into one step of the same form; the steps before it give it its
// carry, and it writes its parts' states. One load's latency for up to 64 parts, and every
// state read and written once. (A thread with all parts one after another took 31 us at
// 64 parts of 8 rows of 64 x 64; eight threads for a value whatever the parts, 28 us at 4
// parts of 150 rows of 48 x 80.)
constexpr int kEach = 8, kGroups = 8;
__global__ __launch_bounds__(kBlock) void join_kernel(Walk w, int groups) {
  __shared__ float keeps[kBlock], owns[kBlock];
  const int values = kBlock / groups, size = w.dk * w.dv;
  const int group = threadIdx.x / values, x = threadIdx.x - group * values, at = blockIdx.y * values + x;
  const int64_t row = blockIdx.x, h = row % w.h;
  const bool live = at < size;
  const float ld = w.log_decay[h];
  float* states = w.states + row * w.parts * size + (live ? at : 0);
  const uint8_t* flags = w.flags + row * w.parts;
  // A part's step; a keep below zero drops the state before it, whatever that holds. lambda^n over
  // a part's n tokens may underflow or overflow where lambda does not: token by token an
  // infinity stays what it is under any lambda above zero, and zero under any.
  const bool lasting = expf(ld) > 0.0f;
  const auto stepped = [lasting](float keep, float before, float own) {
    const float kept = lasting && __builtin_isinf(before) ? before : before * keep;
    return (keep < 0.0f || before == 0.0f ? 0.0f : kept) + own;
  };
  float carry = w.state_in && live ? w.state_in[state_index(w, row, at / w.dv, at % w.dv)] : 0.0f;
  const float whole = expf(ld * (float)w.part);
  for (int base = 0; base < w.parts; base += groups * kEach) {
    const int n0 = base + group * kEach;
    float own[kEach], of[kEach];
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      own[e] = 0.0f, of[e] = 1.0f;
      if (n0 + e < w.parts) {
        const int p = w.backwards ? w.parts - 1 - n0 - e : n0 + e;
        own[e] = states[(int64_t)p * size];
        of[e] = flags[p] ? -1.0f : p < w.parts - 1 ? whole : expf(ld * (float)(w.t - (int64_t)p * w.part));
      }
    }
    float mid = carry;
    if (groups > 1) {
      float keep = 1.0f, sum = 0.0f;
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
        sum = stepped(of[e], sum, own[e]);
        keep = of[e] < 0.0f || keep < 0.0f ? -1.0f : keep * of[e];
      }
      __syncthreads();   // the round before has been read
      keeps[threadIdx.x] = keep;
      owns[threadIdx.x] = sum;
      __syncthreads();
      for (int e = 0; e < groups; ++e) {
        if (e == group) mid = carry;
        carry = stepped(keeps[e * values + x], carry, owns[e * values + x]);
      }
    }
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      if (n0 + e < w.parts && live) {
        const int p = w.backwards ? w.parts - 1 - n0 - e : n0 + e;
        states[(int64_t)p * size] = mid;
      }
      mid = stepped(of[e], mid, own[e]);
    }
    if (groups == 1) carry = mid;
  }
}

// One token of every environment: a block for each (n, h), the state read once and written
// once, bound by that. Four values of a state row at a time, at whatever address they lie:
// L = ceil(dv / 4) threads hold a row (the last one its one to four last values), 256 / L rows at a
// time; the rows' shares of the output meet in LDS. next may be state itself: a thread writes
// only what it has read. 4,096 environments x 8 heads of 64: 188 us, 5.8 TB/s. (One value at a
// time where dv is no multiple of four: 39 us at 8,364 states of 16 x 127, where this takes
// 30.)
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
  int64_t item0;  // the first state of this launch
};

template <class T>
__global__ __launch_bounds__(kBlock) void step_kernel(Step s) {
  typedef f32x4 __attribute__((aligned(4))) four;
  __shared__ __attribute__((aligned(16))) float share[kBlock * 4];
  const int64_t item = s.item0 + blockIdx.x, n = item / s.h, h = item - n * s.h;
  const int L = (s.dv + 3) / 4, R = kBlock / L;
  const int r0 = threadIdx.x / L, c = (threadIdx.x - r0 * L) * 4;
  const int left = s.dv - c;   // values of the row from c on
  const T* q = (const T*)s.q.data + n * s.q.sb + h * s.q.sh;
  const T* k = (const T*)s.k.data + n * s.k.sb + h * s.k.sh;
  const T* v = (const T*)s.v.data + n * s.v.sb + h * s.v.sh;
  const bool fresh = s.reset && s.reset[n * s.reset_sn];
  const float lambda = expf(s.log_decay[h]);
  f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
  if (r0 < R) {
    float x[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = to_f32<T>(v[e < left ? c + e : c]);
    const int64_t base = item * s.dk * s.dv + c;
    constexpr int kAhead = 4;   // rows in flight: next may be state, so no read passes a write by itself
    for (int first = r0; first < s.dk; first += kAhead * R) {
      f32x4 y[kAhead];
      float kr[kAhead], qr[kAhead];
#pragma unroll
      for (int m = 0; m < kAhead; ++m) {
        const int r = first + m * R;
        y[m] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        kr[m] = qr[m] = 0.0f;
        if (r < s.dk) {
          kr[m] = to_f32<T>(k[r]), qr[m] = to_f32<T>(q[r]);
          const float* from = s.state + base + (int64_t)r * s.dv;
          if (!fresh) {
            if (left >= 4)
              y[m] = *(const four*)from;
            else
              y[m] = f32x4{from[0], from[left > 1 ? 1 : 0], from[left > 2 ? 2 : 0], 0.0f};
          }
        }
      }
#pragma unroll
      for (int m = 0; m < kAhead; ++m) {
        const int r = first + m * R;
        if (r < s.dk) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            y[m][e] = __builtin_fmaf(kr[m], x[e], fresh ? 0.0f : y[m][e] * lambda);
            o[e] = __builtin_fmaf(qr[m], y[m][e], o[e]);
          }
          float* to = s.next + base + (int64_t)r * s.dv;
          if (left >= 4) {
            *(four*)to = y[m];
          } else {
            to[0] = y[m][0];
            if (left > 1) to[1] = y[m][1];
            if (left > 2) to[2] = y[m][2];
          }
        }
      }
    }
    *(f32x4*)(share + (r0 * L * 4 + c)) = o;
  }
  __syncthreads();
  for (int j = threadIdx.x; j < s.dv; j += kBlock) {
    float sum = 0.0f;
    const int rows = R < s.dk ? R : s.dk;
    for (int r = 0; r < rows; ++r) sum += share[r * L * 4 + j];
    ((T*)s.out)[item * s.dv + j] = from_f32<T>(s.scale * sum);
  }
}

bool dims_ok(int32_t dtype, int64_t h, int64_t dk, int64_t dv) {
  return (dtype == 0 || dtype == 1) && h >= 1 && h <= 65536 && dk >= 1 && dk <= kMaxDim && dv >= 1 && dv <= kMaxDim;
}

int launch(int32_t dtype, const Walks& walks, bool out, hipStream_t s) {
  return dtype == 1 ? launch_walks<__bf16>(walks, out, s) : launch_walks<float>(walks, out, s);
}

// A block walks a row, or a part of one where the rows are too few to fill the card: then a first
// pass leaves each part's own state, the second joins them, the third walks every part from
// the state before it. The card is full at eight waves a CU: two blocks of four waves take
// 4.2 us a chunk where one takes 3.4 (bfloat16 heads of 64), two of eight waves as long as one
// after the other (heads of 128: 228 us at 512 rows, 117 at 256). As many parts as fill it
// once are the fastest (32 rows of 8,192 tokens in heads of 128: 158 us in 8 parts, 173 in
// 16, 724 in one; 8 rows of 16,381 in heads of 64: 46 us in 64 parts, 81 in 16), of two
// chunks at least, where they save more than the passes cost: the first pass takes about 0.45 of
// the third, joining and launching about five chunks.
int divide(int32_t dtype, int64_t rows, int64_t t, int32_t widest, int32_t* parts, int64_t* part) {
  int cus = 0;
  const int status = device_cus(&cus);
  if (status != HIPENVS_OK) return status;
  const int64_t chunk = dtype == 1 ? Chunk<__bf16>::kTokens : Chunk<float>::kTokens;
  const int64_t chunks = (t + chunk - 1) / chunk, waves = waves_for(widest);
  const int64_t fill = cus * (waves > 4 ? 1 : 8 / waves) / rows, most = chunks / 2;
  int64_t n = fill < most ? fill : most;
  if (n < 2 || chunks * (20 * n - 29) <= 100 * n) n = 1;
  const int64_t per = n > 1 ? (chunks + n - 1) / n : chunks;
  *parts = n > 1 ? (int32_t)((chunks + per - 1) / per) : 1;
  *part = (per > 0 ? per : 1) * chunk;
  return HIPENVS_OK;
}

// The states before the parts of a walk whose rows are walked in parts.
int launch_states(int32_t dtype, const Walk& w, hipStream_t s) {
  if (w.parts == 1) return HIPENVS_OK;
  const int status = launch(dtype, {{w, w}, 1}, false, s);
  if (status != HIPENVS_OK) return status;
  int groups = 1;
  while (groups < kGroups && groups * kEach < w.parts) groups *= 2;
  hipLaunchKernelGGL(join_kernel, dim3((unsigned)(w.b * w.h), grid_for(w.dk * w.dv, kBlock / groups)), dim3(kBlock), 0,
                     s, w, groups);
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

// The parts of a sequence and where in `workspace` their states and flags lie; the bytes used.
int plan(int32_t dtype, int64_t b, int64_t t, int32_t h, int32_t dk, int32_t dv, void* workspace, Walk* w,
         int64_t* bytes) {
  const int status = divide(dtype, b * h, t, dk < dv ? dv : dk, &w->parts, &w->part);
  if (status != HIPENVS_OK) return status;
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
  Walk w = {};
  int64_t need = 0;
  const int status = plan(dtype, b, t, h, dk, dv, workspace, &w, &need);
  if (status != HIPENVS_OK) return status;
  if (need > 0 && (!workspace || ((uintptr_t)workspace & 3) || workspace_bytes < need)) return HIPENVS_E_ARG;
  w.q = rows(q, st), w.k = rows(k, st + 3), w.v = rows(v, st + 6);
  w.dk = dk, w.dv = dv, w.log_decay = log_decay, w.reset = reset, w.reset_sb = st[9], w.reset_st = st[10];
  w.state_in = state, w.state_out = final_state, w.read = scale, w.add = 1.0f;
  w.out = out, w.b = b, w.t = t, w.h = h;
  const int walked = launch_states(dtype, w, as_stream(stream));
  return walked == HIPENVS_OK ? launch(dtype, {{w, w}, 1}, true, as_stream(stream)) : walked;
}

extern "C" int hipenvs_decay_attention_backward(int32_t dtype, const void* q, const void* k, const void* v,
                                                const void* dout, const int64_t* strides, const float* log_decay,
                                                const float* state, const uint8_t* reset, const float* dfinal,
                                                const float* states, float scale, void* dq, void* dk_out, void* dv_out, float* dstate,
                                                int64_t b, int64_t t, int32_t h, int32_t dk, int32_t dv,
                                                void* workspace, int64_t workspace_bytes, hipenvs_stream_t stream) {
  if (!sequence_ok(dtype, b, t, h, dk, dv)) return HIPENVS_E_ARG;
  if (b == 0) return HIPENVS_OK;
  if (!log_decay || !dstate || (t > 0 && (!q || !k || !v || !dout || !dq || !dk_out || !dv_out || !strides)))
    return HIPENVS_E_ARG;
  if ((uintptr_t)states & 3) return HIPENVS_E_ARG;
  static const int64_t none[14] = {};
  const int64_t* st = t > 0 ? strides : none;
  Walk w = {};
  int64_t need = 0;
  int status = plan(dtype, b, t, h, dk, dv, workspace, &w, &need);
  if (status != HIPENVS_OK) return status;
  if (need > 0 && (!workspace || ((uintptr_t)workspace & 3) || workspace_bytes < need)) return HIPENVS_E_ARG;
  float* own_states = w.states;
  const Rows rq = rows(q, st), rk = rows(k, st + 3), rv = rows(v, st + 6),
             rdo = rows(dout, st + 9);
  const hipStream_t s = as_stream(stream);
  w.log_decay = log_decay, w.reset = reset, w.reset_sb = st[12], w.reset_st = st[13], w.b = b, w.t = t, w.h = h;
  // dq: forwards over the transposed states, which the forward pass has left, or are computed
  // again (transposed) where it has not
  w.q = rdo, w.k = rv, w.v = rk, w.dk = dv, w.dv = dk, w.state_in = state, w.state_out = nullptr;
  w.flipped = true, w.backwards = false, w.read = scale, w.add = 1.0f, w.out = dq;
  if (states) {
    w.states = const_cast<float*>(states);
    w.turned = true;
  } else {
    status = launch_states(dtype, w, s);
    if (status != HIPENVS_OK) return status;
  }
  status = launch(dtype, {{w, w}, 1}, true, s);
  if (status != HIPENVS_OK) return status;
  // dv, and the gradient of the first state: backwards over the states' gradients
  w.q = rk, w.k = rq, w.v = rdo, w.dk = dk, w.dv = dv, w.state_in = dfinal, w.state_out = dstate;
  w.states = own_states, w.turned = false;
  w.flipped = false, w.backwards = true, w.read = 1.0f, w.add = scale, w.out = dv_out;
  status = launch_states(dtype, w, s);
  if (status != HIPENVS_OK) return status;
  // dk: the same, transposed
  Walk u = w;
  u.q = rv, u.k = rdo, u.v = rq, u.dk = dv, u.dv = dk, u.state_out = nullptr, u.flipped = true;
  u.turned = true, u.out = dk_out;
  if (rows_of(dk) == rows_of(dv) && waves_for(dk) == waves_for(dv)) return launch(dtype, {{w, u}, 2}, true, s);
  status = launch(dtype, {{w, w}, 1}, true, s);
  return status == HIPENVS_OK ? launch(dtype, {{u, u}, 1}, true, s) : status;
}

extern "C" int hipenvs_decay_attention_step(int32_t dtype, const void* q, int64_t q_sn, int64_t q_sh, const void* k,
                                            int64_t k_sn, int64_t k_sh, const void* v, int64_t v_sn, int64_t v_sh,
                                            const float* log_decay, const float* state, const uint8_t* reset,
                                            int64_t reset_sn, float scale, void* out, float* next_state, int64_t n,
                                            int32_t h, int32_t dk, int32_t dv, hipenvs_stream_t stream) {
  if (!dims_ok(dtype, h, dk, dv) || n < 0 || n > 0x7FFFFFFF || n * h > 0x7FFFFFFF) return HIPENVS_E_ARG;
  if (n == 0) return HIPENVS_OK;
  if (!q || !k || !v || !log_decay || !state || !out || !next_state) return HIPENVS_E_ARG;
  Step s = {{q, q_sn, 0, q_sh}, {k, k_sn, 0, k_sh}, {v, v_sn, 0, v_sh}, log_decay, reset, reset_sn,
            state, next_state, out, scale, h, dk, dv, 0};
  const int64_t items = n * h, most = kMostThreads / kBlock;
  for (s.item0 = 0; s.item0 < items; s.item0 += most) {
    const dim3 grid((unsigned)(items - s.item0 < most ? items - s.item0 : most)), block(kBlock);
    if (dtype == 1)
      hipLaunchKernelGGL(step_kernel<__bf16>, grid, block, 0, as_stream(stream), s);
    else
      hipLaunchKernelGGL(step_kernel<float>, grid, block, 0, as_stream(stream), s);
    const int status = launch_status();
    if (status != HIPENVS_OK) return status;
  }
  return HIPENVS_OK;
}
