// Rows of a table for tokens, scaled, and the gradient of the table by sorted tokens. No reference
// counterpart.
//
//   out_i = scale table[token_i]        dtable[v] = scale sum_{i: token_i = v} dout_i
//
// A negative token is none: a row of zeros, no gradient. One past the table is a mistake: a row
// that is no number, no gradient. Sums are float32, in an order that depends on the tokens alone.
#include "row_ops.h"

namespace hipenvs {
namespace embedding {

using namespace rows;

struct Tokens {
  const void* data;
  bool wide;   // int64, otherwise int32

  __device__ __forceinline__ int64_t operator[](int64_t i) const {
    return wide ? ((const int64_t*)data)[i] : ((const int32_t*)data)[i];
  }
};

// Four values a thread; bound by the output's writes.
template <class T>
__global__ __launch_bounds__(kBlock) void lookup_kernel(Tokens tokens, const T* __restrict__ table, int64_t table_sv,
                                                        float scale, T* __restrict__ out, int64_t count, int64_t v,
                                                        int32_t d, int32_t quads, int64_t item0) {
  const int64_t item = item0 + (int64_t)blockIdx.x * kBlock + threadIdx.x, i = item / quads;
  if (i >= count) return;
  const int c = (int)(item - i * quads) * 4;
  const int64_t token = tokens[i];
  const bool there = token >= 0 && token < v;
  const f32x4 row = values<T>(fetch4(table + (there ? token : 0) * table_sv, c, d), c, d);
  f32x4 x;
#pragma unroll
  for (int e = 0; e < 4; ++e) x[e] = there ? row[e] * scale : token < 0 ? 0.0f : __builtin_nanf("");
  store_upto(out + i * d + c, x, d - c);
}

// ---- sorting the tokens ---------------------------------------------------------------
// Least digit first, 8 bits a pass, each pass stable, so a token's places stay in their order. Keys
// are tokens, v where there is none. A pass counts the digits of each tile of 4,096, sums the
// counts up, digit by digit and tile by tile, and moves each key with its place.

constexpr int kDigit = 256, kRounds = 16, kSortTile = kBlock * kRounds;

struct Sort {
  Tokens tokens;
  const uint32_t *keys, *places;   // null in the first pass: the tokens as they come
  uint32_t *keys_out, *places_out, *counts;
  int64_t count, v, tiles;
  int shift;

  __device__ __forceinline__ uint32_t key(int64_t i) const {
    if (keys) return keys[i];
    const int64_t t = tokens[i];
    return t < 0 || t >= v ? (uint32_t)v : (uint32_t)t;
  }
};

__global__ __launch_bounds__(kBlock) void count_kernel(Sort s) {
  __shared__ uint32_t counts[kDigit];
  counts[threadIdx.x] = 0;
  __syncthreads();
  const int64_t first = (int64_t)blockIdx.x * kSortTile;
  for (int r = 0; r < kRounds; ++r) {
    const int64_t i = first + r * kBlock + threadIdx.x;
    if (i < s.count) atomicAdd(&counts[(s.key(i) >> s.shift) & 255], 1u);
  }
  __syncthreads();
  s.counts[threadIdx.x * s.tiles + blockIdx.x] = counts[threadIdx.x];
}

// counts -> the sums of those before, in place; one block.
__global__ __launch_bounds__(1024) void sum_up_kernel(uint32_t* counts, int64_t n) {
  __shared__ uint32_t totals[16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t before = 0;
  for (int64_t first = 0; first < n; first += 4096) {
    const int64_t i = first + threadIdx.x * 4;
    uint32_t x[4], sum = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      x[k] = i + k < n ? counts[i + k] : 0u;
      sum += x[k];
    }
    uint32_t upto = sum;
#pragma unroll
    for (int step = 1; step < 64; step *= 2) {
      const uint32_t other = __shfl_up(upto, step);
      if (lane >= step) upto += other;
    }
    if (lane == 63) totals[wave] = upto;
    __syncthreads();
    uint32_t at = before + upto - sum, all = 0;
    for (int k = 0; k < 16; ++k) {
      if (k < wave) at += totals[k];
      all += totals[k];
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (i + k < n) counts[i + k] = at;
      at += x[k];
    }
    before += all;
    __syncthreads();
  }
}

__global__ __launch_bounds__(kBlock) void move_kernel(Sort s) {
  __shared__ uint32_t at[4][kDigit];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int k = 0; k < 4; ++k) at[k][threadIdx.x] = 0;
  __syncthreads();
  // a wave moves 1,024 neighbouring keys, so that the order of the places holds across waves
  const int64_t first = (int64_t)blockIdx.x * kSortTile + wave * (kRounds * 64) + lane;
  uint32_t keys[kRounds];
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const int64_t i = first + r * 64;
    keys[r] = i < s.count ? s.key(i) : 0u;
    if (i < s.count) atomicAdd(&at[wave][(keys[r] >> s.shift) & 255], 1u);
  }
  __syncthreads();
  uint32_t base = s.counts[threadIdx.x * s.tiles + blockIdx.x];
  for (int k = 0; k < 4; ++k) {
    const uint32_t own = at[k][threadIdx.x];
    at[k][threadIdx.x] = base;
    base += own;
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const int64_t i = first + r * 64;
    const uint32_t digit = (keys[r] >> s.shift) & 255;
    uint64_t same = __builtin_amdgcn_ballot_w64(i < s.count);   // the lanes with this digit
#pragma unroll
    for (int bit = 0; bit < 8; ++bit) {
      const uint64_t set = __builtin_amdgcn_ballot_w64(digit >> bit & 1);
      same &= digit >> bit & 1 ? set : ~set;
    }
    const uint64_t below = same & ((1ull << lane) - 1);
    if (i < s.count) {
      const uint32_t to = at[wave][digit] + (uint32_t)__popcll(below);
      s.keys_out[to] = keys[r];
      s.places_out[to] = s.places ? s.places[i] : (uint32_t)i;
    }
    __builtin_amdgcn_wave_barrier();
    if (i < s.count && below == 0) at[wave][digit] += (uint32_t)__popcll(same);
    __builtin_amdgcn_wave_barrier();
  }
}

// ---- sums over equal keys --------------------------------------------------------------
// A group of lanes, one for every four columns, walks a chunk of the sorted keys and adds up the rows
// that they name. A run of equal keys within the chunk is finished; the sum of one that reaches over
// the chunk's beginning or end goes to `firsts` or `lasts`, which a second kernel adds in order.

constexpr int kChunk = 64;

struct Sums {
  const uint32_t *keys, *places;
  const void* dout;   // (count, d) rows, dout_s apart
  void* dtable;       // (v, d)
  float *firsts, *lasts;   // (chunks, d)
  int64_t count, v, chunks, dout_s, item0;
  int32_t d, quads, group, columns;   // group: lanes that share a chunk; columns: groups for a row
  float scale;
};

template <class T>
__global__ __launch_bounds__(kBlock) void clear_kernel(T* x, int64_t n, int64_t item0) {
  const int64_t i = (item0 + (int64_t)blockIdx.x * kBlock + threadIdx.x) * 4;
  if (i < n) store_upto(x + i, f32x4{0.0f, 0.0f, 0.0f, 0.0f}, n - i);
}

template <class T>
__global__ __launch_bounds__(kBlock) void chunks_kernel(Sums s) {
  const int64_t item = (s.item0 + (int64_t)blockIdx.x * kBlock + threadIdx.x) / s.group;
  const int64_t chunk = item / s.columns;
  const int quad = (int)(item - chunk * s.columns) * s.group + threadIdx.x % s.group;
  if (chunk >= s.chunks || quad >= s.quads) return;
  const int c = quad * 4, left = s.d - c;
  const int64_t first = chunk * kChunk, end = first + kChunk < s.count ? first + kChunk : s.count;
  const uint32_t none = (uint32_t)s.v;
  const uint32_t before = first > 0 ? s.keys[first - 1] : none, behind = end < s.count ? s.keys[end] : none;
  uint32_t current = s.keys[first];
  bool opened = first == 0 || before != current;   // the current run begins in this chunk
  f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
  const auto close = [&](bool last) {
    if (current == none) return;
    if (!opened)
      store_upto(s.firsts + chunk * s.d + c, sum, left);
    else if (last && end < s.count && behind == current)
      store_upto(s.lasts + chunk * s.d + c, sum, left);
    else
      store_upto((T*)s.dtable + (int64_t)current * s.d + c, sum * s.scale, left);
  };
  constexpr int kAhead = 8;
  for (int64_t i0 = first; i0 < end; i0 += kAhead) {
    uint32_t key[kAhead];
    typename Raw<T>::type x[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {   // past the end, the last one: all loads in flight
      const int64_t i = i0 + k < end ? i0 + k : end - 1;
      key[k] = s.keys[i];
      x[k] = fetch4((const T*)s.dout + (int64_t)s.places[i] * s.dout_s, c, s.d);
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      if (i0 + k >= end) break;
      if (key[k] != current) {
        close(false);
        current = key[k], opened = true;
        sum = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      }
      sum += values<T>(x[k], c, s.d);
    }
  }
  close(true);
}

// The runs that reach over chunks, each by the group of the chunk where it begins.
template <class T>
__global__ __launch_bounds__(kBlock) void across_kernel(Sums s) {
  const int64_t item = (s.item0 + (int64_t)blockIdx.x * kBlock + threadIdx.x) / s.group;
  const int64_t chunk = item / s.columns;
  const int quad = (int)(item - chunk * s.columns) * s.group + threadIdx.x % s.group;
  if (chunk >= s.chunks || quad >= s.quads) return;
  const int c = quad * 4, left = s.d - c;
  const int64_t first = chunk * kChunk, end = first + kChunk;
  if (end >= s.count) return;
  const uint32_t key = s.keys[end - 1];
  if (key == (uint32_t)s.v || s.keys[end] != key) return;
  if (first > 0 && s.keys[first - 1] == key) return;   // it began before this chunk
  // the last of its chunks: the one that holds the last key not above it
  int64_t low = end, high = s.count;                    // keys[low] == key, keys[high] > key
  while (high - low > 1) {
    const int64_t mid = (low + high) / 2;
    if (s.keys[mid] == key) low = mid;
    else high = mid;
  }
  const int64_t last = low / kChunk;
  f32x4 sum = load_upto(s.lasts + chunk * s.d + c, left);
  constexpr int kAhead = 8;
  for (int64_t k0 = chunk + 1; k0 <= last; k0 += kAhead) {
    f32x4 x[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) x[k] = fetch4(s.firsts + (k0 + k < last ? k0 + k : last) * s.d, c, s.d);
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      if (k0 + k <= last) sum += values<float>(x[k], c, s.d);
  }
  store_upto((T*)s.dtable + (int64_t)key * s.d + c, sum * s.scale, left);
}

namespace {
bool sizes_ok(int32_t dtype, int64_t count, int64_t v, int32_t d) {
  return (dtype == 0 || dtype == 1) && count >= 0 && count <= 0x7FFFFFFF && v >= 1 && v <= 0x7FFFFFFF && d >= 1 &&
         d <= 65536;
}

int64_t round16(int64_t x) { return (x + 15) / 16 * 16; }

struct Laid {
  int64_t keys, counts, partial, bytes;
};

// keys and places twice, the digits' counts, the chunks' partial sums
Laid lay(int64_t count, int32_t d) {
  const int64_t tiles = (count + kSortTile - 1) / kSortTile, chunks = (count + kChunk - 1) / kChunk;
  Laid l = {round16(count * 4), round16(tiles * kDigit * 4), round16(chunks * d * 4), 0};
  l.bytes = 4 * l.keys + l.counts + 2 * l.partial;
  return l;
}

template <class F>
int in_launches(int64_t items, const F& launch) {
  for (int64_t item0 = 0; item0 < items; item0 += kMostThreads) {
    const int64_t own = items - item0 < kMostThreads ? items - item0 : kMostThreads;
    launch(item0, dim3(grid_for(own)));
    const int status = launch_status();
    if (status != HIPENVS_OK) return status;
  }
  return HIPENVS_OK;
}

template <class T>
int gradient(Tokens tokens, const void* dout, int64_t dout_s, float scale, void* dtable, int64_t count, int64_t v,
             int32_t d, char* workspace, hipStream_t stream) {
  const int64_t values = v * d;
  int status = in_launches((values + 3) / 4, [&](int64_t item0, dim3 grid) {
    hipLaunchKernelGGL(clear_kernel<T>, grid, dim3(kBlock), 0, stream, (T*)dtable, values, item0);
  });
  if (status != HIPENVS_OK || count == 0) return status;
  const Laid l = lay(count, d);
  uint32_t* keys[2] = {(uint32_t*)workspace, (uint32_t*)(workspace + l.keys)};
  uint32_t* places[2] = {(uint32_t*)(workspace + 2 * l.keys), (uint32_t*)(workspace + 3 * l.keys)};
  Sort sort = {tokens, nullptr, nullptr, nullptr, nullptr, (uint32_t*)(workspace + 4 * l.keys), count, v,
               (count + kSortTile - 1) / kSortTile, 0};
  int to = 0;
  for (; (v >> sort.shift) > 0; sort.shift += 8, to ^= 1) {
    sort.keys_out = keys[to], sort.places_out = places[to];
    const dim3 tiles((unsigned)sort.tiles);
    hipLaunchKernelGGL(count_kernel, tiles, dim3(kBlock), 0, stream, sort);
    hipLaunchKernelGGL(sum_up_kernel, dim3(1), dim3(1024), 0, stream, sort.counts, sort.tiles * kDigit);
    hipLaunchKernelGGL(move_kernel, tiles, dim3(kBlock), 0, stream, sort);
    status = launch_status();
    if (status != HIPENVS_OK) return status;
    sort.keys = keys[to], sort.places = places[to];
  }
  char* partial = workspace + 4 * l.keys + l.counts;
  const int quads = (d + 3) / 4;
  int group = 1;
  while (group < 64 && group < quads) group *= 2;
  Sums s = {sort.keys, sort.places, dout, dtable, (float*)partial, (float*)(partial + l.partial), count, v,
            (count + kChunk - 1) / kChunk, dout_s, 0, d, quads, group, (quads + group - 1) / group, scale};
  const int64_t items = s.chunks * s.columns * group;
  status = in_launches(items, [&](int64_t item0, dim3 grid) {
    s.item0 = item0;
    hipLaunchKernelGGL(chunks_kernel<T>, grid, dim3(kBlock), 0, stream, s);
  });
  if (status != HIPENVS_OK || s.chunks == 1) return status;
  return in_launches(items, [&](int64_t item0, dim3 grid) {
    s.item0 = item0;
    hipLaunchKernelGGL(across_kernel<T>, grid, dim3(kBlock), 0, stream, s);
  });
}
}  // namespace

}  // namespace embedding
}  // namespace hipenvs

using namespace hipenvs;
using namespace hipenvs::embedding;

extern "C" int hipenvs_embedding(int32_t dtype, const void* tokens, int32_t token_bytes, const void* table,
                                 int64_t table_sv, float scale, void* out, int64_t count, int64_t v, int32_t d,
                                 hipenvs_stream_t stream) {
  if (!sizes_ok(dtype, count, v, d) || (token_bytes != 4 && token_bytes != 8)) return HIPENVS_E_ARG;
  if (count == 0) return HIPENVS_OK;
  if (!tokens || !table || !out) return HIPENVS_E_ARG;
  const Tokens of = {tokens, token_bytes == 8};
  const int quads = (d + 3) / 4;
  return in_launches(count * quads, [&](int64_t item0, dim3 grid) {
    if (dtype == 1)
      hipLaunchKernelGGL(lookup_kernel<__bf16>, grid, dim3(kBlock), 0, as_stream(stream), of, (const __bf16*)table,
                         table_sv, scale, (__bf16*)out, count, v, d, quads, item0);
    else
      hipLaunchKernelGGL(lookup_kernel<float>, grid, dim3(kBlock), 0, as_stream(stream), of, (const float*)table,
                         table_sv, scale, (float*)out, count, v, d, quads, item0);
  });
}

extern "C" int64_t hipenvs_embedding_workspace_bytes(int64_t count, int64_t v, int32_t d) {
  if (!sizes_ok(0, count, v, d)) return -1;
  return count == 0 ? 0 : lay(count, d).bytes;
}

extern "C" int hipenvs_embedding_backward(int32_t dtype, const void* tokens, int32_t token_bytes, const void* dout,
                                          int64_t dout_s, float scale, void* dtable, int64_t count, int64_t v,
                                          int32_t d, void* workspace, int64_t workspace_bytes,
                                          hipenvs_stream_t stream) {
  if (!sizes_ok(dtype, count, v, d) || (token_bytes != 4 && token_bytes != 8) || !dtable) return HIPENVS_E_ARG;
  if (count > 0 && (!tokens || !dout || !workspace || ((uintptr_t)workspace & 15) ||
                    workspace_bytes < lay(count, d).bytes))
    return HIPENVS_E_ARG;
  const Tokens of = {tokens, token_bytes == 8};
  return dtype == 1 ? gradient<__bf16>(of, dout, dout_s, scale, dtable, count, v, d, (char*)workspace, as_stream(stream))
                    : gradient<float>(of, dout, dout_s, scale, dtable, count, v, d, (char*)workspace, as_stream(stream));
}
