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

// Four values a thread; bound by the output's writes (134 MB of float32 in 27 us, 5 TB/s).
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
// are tokens, v where there is none. A pass counts the digits of each tile of kRounds x 256 keys,
// sums each digit's counts up over the tiles (where they are few, in every block that moves) and
// moves each key with its place.

constexpr int kDigit = 256, kFewTiles = 64;

struct Sort {
  Tokens tokens;
  const uint32_t *keys, *places;   // null in the first pass: the tokens as they come
  uint32_t *keys_out, *places_out, *counts;   // counts (tiles, 256), then the digits' totals (256)
  int64_t count, v, tiles;
  int shift;
  bool summed;   // counts are those of the tiles before; otherwise of the tile itself, at most kFewTiles of them
  void* clear;   // in the first pass, what becomes zeros: the gradient, of `words` 32-bit words and a half of one
  int64_t words;
  bool half;

  __device__ __forceinline__ uint32_t key(int64_t i) const {
    if (keys) return keys[i];
    const int64_t t = tokens[i];
    return t < 0 || t >= v ? (uint32_t)v : (uint32_t)t;
  }
};

// The tile's digits; and in the first pass zeros over the gradient, by as many blocks as that takes.
template <int kRounds>
__global__ __launch_bounds__(kBlock) void count_kernel(Sort s) {
  __shared__ uint32_t counts[kDigit];
  if (s.clear) {
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    const int64_t step = (int64_t)gridDim.x * kBlock, first = (int64_t)blockIdx.x * kBlock + threadIdx.x;
    for (int64_t i = first; i < s.words / 4; i += step) ((u32x4*)s.clear)[i] = u32x4{0, 0, 0, 0};
    if (first < s.words % 4) ((uint32_t*)s.clear)[s.words / 4 * 4 + first] = 0;
    if (first == 0 && s.half) ((uint16_t*)s.clear)[2 * s.words] = 0;
  }
  if (blockIdx.x >= s.tiles) return;
  counts[threadIdx.x] = 0;
  __syncthreads();
  const int64_t first = (int64_t)blockIdx.x * (kBlock * kRounds) + threadIdx.x;
  uint32_t keys[kRounds];
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const int64_t i = first + r * kBlock;
    keys[r] = s.key(i < s.count ? i : s.count - 1);
  }
#pragma unroll
  for (int r = 0; r < kRounds; ++r)
    if (first + r * kBlock < s.count) atomicAdd(&counts[(keys[r] >> s.shift) & 255], 1u);
  __syncthreads();
  s.counts[blockIdx.x * kDigit + threadIdx.x] = counts[threadIdx.x];
}

// A block for each digit: its tiles' counts -> the sums of those before, in place; and its total.
__global__ __launch_bounds__(kBlock) void sum_up_kernel(Sort s) {
  __shared__ uint32_t totals[4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t* counts = s.counts + blockIdx.x;
  uint32_t before = 0;
  for (int64_t first = 0; first < s.tiles; first += kBlock) {
    const int64_t i = first + threadIdx.x;
    const uint32_t own = i < s.tiles ? counts[i * kDigit] : 0u;
    uint32_t upto = own;
#pragma unroll
    for (int step = 1; step < 64; step *= 2) {
      const uint32_t other = __shfl_up(upto, step);
      if (lane >= step) upto += other;
    }
    if (lane == 63) totals[wave] = upto;
    __syncthreads();
    uint32_t at = before + upto - own;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (k < wave) at += totals[k];
      before += totals[k];
    }
    if (i < s.tiles) counts[i * kDigit] = at;
    __syncthreads();
  }
  if (threadIdx.x == 0) s.counts[kDigit * s.tiles + blockIdx.x] = before;
}

template <int kRounds>
__global__ __launch_bounds__(kBlock) void move_kernel(Sort s) {
  __shared__ uint32_t at[4][kDigit], totals[4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  // a wave moves kRounds x 64 neighbouring keys, so that the order of the places holds across waves
  const int64_t first = (int64_t)blockIdx.x * (kBlock * kRounds) + wave * (kRounds * 64) + lane;
  uint32_t keys[kRounds], places[kRounds];
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const int64_t i = first + r * 64 < s.count ? first + r * 64 : s.count - 1;
    keys[r] = s.key(i);
    places[r] = s.places ? s.places[i] : (uint32_t)i;
  }
  // the keys of lower digits, by the digits' totals
  uint32_t total = 0, base = 0;
  if (s.summed) {
    total = s.counts[kDigit * s.tiles + threadIdx.x];
    base = s.counts[blockIdx.x * kDigit + threadIdx.x];
  } else {
    const int tiles = (int)s.tiles;
    for (int k0 = 0; k0 < tiles; k0 += 16) {
      uint32_t own[16];
#pragma unroll
      for (int k = 0; k < 16; ++k) own[k] = s.counts[(k0 + k < tiles ? k0 + k : tiles - 1) * kDigit + threadIdx.x];
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        if (k0 + k < tiles) total += own[k];
        if (k0 + k < (int)blockIdx.x) base += own[k];
      }
    }
  }
  uint32_t upto = total;
#pragma unroll
  for (int step = 1; step < 64; step *= 2) {
    const uint32_t other = __shfl_up(upto, step);
    if (lane >= step) upto += other;
  }
  if (lane == 63) totals[wave] = upto;
  for (int k = 0; k < 4; ++k) at[k][threadIdx.x] = 0;
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kRounds; ++r)
    if (first + r * 64 < s.count) atomicAdd(&at[wave][(keys[r] >> s.shift) & 255], 1u);
  base += upto - total;
  for (int k = 0; k < wave; ++k) base += totals[k];
  __syncthreads();
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
      s.places_out[to] = places[r];
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

constexpr int kChunk = 32;

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

// The runs that reach over chunks, each by the block of the chunk where it begins: its groups of lanes
// add up every so many of its chunks, and their sums meet in LDS.
template <class T>
__global__ __launch_bounds__(kBlock) void across_kernel(Sums s) {
  __shared__ f32x4 share[kBlock];
  const int64_t item = s.item0 + blockIdx.x, chunk = item / s.columns;
  const int rows = kBlock / s.group, row = threadIdx.x / s.group, lane = threadIdx.x % s.group;
  const int quad = (int)(item - chunk * s.columns) * s.group + lane, c = (quad < s.quads ? quad : 0) * 4;
  const int64_t first = chunk * kChunk, end = first + kChunk;
  if (end >= s.count) return;   // the conditions are the block's
  const uint32_t key = s.keys[end - 1];
  if (key == (uint32_t)s.v || s.keys[end] != key) return;
  if (first > 0 && s.keys[first - 1] == key) return;   // it began before this chunk
  int64_t low = end, high = s.count;   // keys[low] == key, keys[high] is above it: 256 probes a round
  while (high - low > 1) {
    const int64_t step = (high - low + kBlock - 1) / kBlock, at = low + (threadIdx.x + 1) * step;
    low += __syncthreads_count(at < high && s.keys[at] == key) * step;
    high = low + step < high ? low + step : high;
  }
  const int64_t last = low / kChunk;   // of the run's chunks
  f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
  if (row == 0) sum = values<float>(fetch4(s.lasts + chunk * s.d, c, s.d), c, s.d);
  constexpr int kAhead = 8;
  for (int64_t k0 = chunk + 1 + row; k0 <= last; k0 += kAhead * rows) {
    f32x4 x[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int64_t at = k0 + k * rows;
      x[k] = fetch4(s.firsts + (at < last ? at : last) * s.d, c, s.d);
    }
    f32x4 some = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const f32x4 y = values<float>(x[k], c, s.d);
#pragma unroll
      for (int e = 0; e < 4; ++e) some[e] += k0 + k * rows <= last ? y[e] : 0.0f;
    }
    sum += some;
  }
  share[threadIdx.x] = sum;
  __syncthreads();
  for (int half = rows / 2; half > 0; half /= 2) {
    if (row < half) share[threadIdx.x] += share[threadIdx.x + half * s.group];
    __syncthreads();
  }
  if (row == 0 && quad < s.quads) store_upto((T*)s.dtable + (int64_t)key * s.d + c, share[threadIdx.x] * s.scale, s.d - c);
}

// ---- small tables ----------------------------------------------------------------------
// A table of at most kSmall rows is summed without sorting: each group of lanes of a block takes every
// so many of its tokens and adds their rows to sums of its own in LDS; a block's groups then meet, and the
// blocks' sums are the rows of a matrix whose columns are added up. 524,288 tokens of 3 x 64 float32, 134 MB:
// 27 + 8 us, 4.9 TB/s. The lookup and its gradient, so and sorted: that 60 and 156 us, of 8 rows 61 and 122, of
// 16, which leave LDS for two blocks a CU, 88 and 114; 64,000 tokens of 2 x 512 bfloat16 46 and 106, of 8 53 and 72,
// of 16 69 and 66; 3,000 of 16 x 64 float32 16 and 28. A thread's sums are its own, so their order is that of the tokens.

constexpr int kSmall = 16;

struct Small {
  Tokens tokens;
  const void* dout;
  float* partial;   // (blocks, v d)
  int64_t count, each, dout_s;   // each: tokens of a block
  int32_t v, d, quads, group;
};

template <class T>
__global__ __launch_bounds__(kBlock) void small_kernel(Small s) {
  extern __shared__ __attribute__((aligned(16))) f32x4 sums[];   // (v, 256)
  const int rows = kBlock / s.group, row = threadIdx.x / s.group;
  const int quad = blockIdx.y * s.group + threadIdx.x % s.group, c = (quad < s.quads ? quad : 0) * 4;
  for (int k = 0; k < s.v; ++k) sums[k * kBlock + threadIdx.x] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  const int64_t first = blockIdx.x * s.each, end = first + s.each < s.count ? first + s.each : s.count;
  constexpr int kAhead = 8;
  for (int64_t i0 = first + row; i0 < end; i0 += kAhead * rows) {
    int64_t token[kAhead];
    typename Raw<T>::type x[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int64_t i = i0 + k * rows < end ? i0 + k * rows : end - 1;
      token[k] = s.tokens[i];
      x[k] = fetch4((const T*)s.dout + i * s.dout_s, c, s.d);
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const f32x4 y = values<T>(x[k], c, s.d);
      if (i0 + k * rows < end && token[k] >= 0 && token[k] < s.v) sums[token[k] * kBlock + threadIdx.x] += y;
    }
  }
  __syncthreads();
  for (int half = rows / 2; half > 0; half /= 2) {
    if (row < half)
      for (int k = 0; k < s.v; ++k) sums[k * kBlock + threadIdx.x] += sums[k * kBlock + threadIdx.x + half * s.group];
    __syncthreads();
  }
  if (row == 0 && quad < s.quads)
    for (int k = 0; k < s.v; ++k)
      store_upto(s.partial + ((int64_t)blockIdx.x * s.v + k) * s.d + c, sums[k * kBlock + threadIdx.x], s.d - c);
}

namespace {
bool sizes_ok(int32_t dtype, int64_t count, int64_t v, int32_t d) {
  return (dtype == 0 || dtype == 1) && count >= 0 && count <= 0x7FFFFFFF && v >= 1 && v <= 0x7FFFFFFF && d >= 1 &&
         d <= 65536;
}

int64_t round16(int64_t x) { return (x + 15) / 16 * 16; }

int group_of(int quads) {
  int group = 1;
  while (group < 64 && group < quads) group *= 2;
  return group;
}

// Blocks of a small table's sums: four a CU of 256 (from 11 rows on LDS holds fewer at once), but no fewer than
// eight tokens for a group of lanes.
int64_t small_blocks(int64_t count, int32_t d) {
  const int64_t least = 8 * (kBlock / group_of((d + 3) / 4)), blocks = (count + least - 1) / least;
  return blocks < 1024 ? blocks : 1024;
}

int rounds_of(int64_t count) { return count <= 4 * kBlock * kFewTiles ? 4 : 16; }

struct Laid {
  int64_t keys, counts, partial, bytes;
};

// keys and places twice, the digits' counts, the chunks' partial sums; or a small table's partial sums
Laid lay(int64_t count, int64_t v, int32_t d) {
  if (v <= kSmall) {
    const int64_t blocks = small_blocks(count, d), partial = round16(blocks * v * d * 4);
    return {0, 0, partial, partial + column_sums_bytes(blocks, v * d)};
  }
  const int64_t tile = kBlock * rounds_of(count), tiles = (count + tile - 1) / tile;
  const int64_t chunks = (count + kChunk - 1) / kChunk;
  Laid l = {round16(count * 4), round16((tiles + 1) * kDigit * 4), round16(chunks * d * 4), 0};
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
int small_gradient(Tokens tokens, const void* dout, int64_t dout_s, float scale, void* dtable, int64_t count, int64_t v,
                   int32_t d, char* workspace, hipStream_t stream) {
  const Laid l = lay(count, v, d);
  const int quads = (d + 3) / 4, group = group_of(quads);
  const int64_t blocks = small_blocks(count, d);
  const Small s = {tokens, dout, (float*)workspace, count, (count + blocks - 1) / blocks, dout_s, (int32_t)v, d, quads,
                   group};
  hipLaunchKernelGGL(small_kernel<T>, dim3((unsigned)blocks, (unsigned)((quads + group - 1) / group)), dim3(kBlock),
                     (size_t)v * kBlock * sizeof(f32x4), stream, s);
  const int status = launch_status();
  if (status != HIPENVS_OK) return status;
  return column_sums<T>(s.partial, blocks, v * d, scale, (T*)dtable, (float*)(workspace + l.partial), stream);
}

template <class T>
int gradient(Tokens tokens, const void* dout, int64_t dout_s, float scale, void* dtable, int64_t count, int64_t v,
             int32_t d, char* workspace, hipStream_t stream) {
  if (v <= kSmall && count > 0)
    return small_gradient<T>(tokens, dout, dout_s, scale, dtable, count, v, d, workspace, stream);
  const int64_t bytes = v * d * (int64_t)sizeof(T);
  // 16 KiB a block, at most eight blocks a CU
  const unsigned clears = (unsigned)(bytes / 16384 < 2047 ? bytes / 16384 + 1 : 2048);
  const int rounds = rounds_of(count);
  if (count == 0) {
    Sort nothing = {};
    nothing.clear = dtable, nothing.words = bytes / 4, nothing.half = bytes % 4 != 0;
    hipLaunchKernelGGL(count_kernel<4>, dim3(clears), dim3(kBlock), 0, stream, nothing);
    return launch_status();
  }
  int status = HIPENVS_OK;
  const Laid l = lay(count, v, d);
  uint32_t* keys[2] = {(uint32_t*)workspace, (uint32_t*)(workspace + l.keys)};
  uint32_t* places[2] = {(uint32_t*)(workspace + 2 * l.keys), (uint32_t*)(workspace + 3 * l.keys)};
  Sort sort = {tokens, nullptr, nullptr, nullptr, nullptr, (uint32_t*)(workspace + 4 * l.keys), count, v,
               (count + kBlock * rounds - 1) / (kBlock * rounds), 0, false, dtable, bytes / 4, bytes % 4 != 0};
  sort.summed = sort.tiles > kFewTiles;
  int to = 0;
  for (; (v >> sort.shift) > 0; sort.shift += 8, to ^= 1) {
    sort.keys_out = keys[to], sort.places_out = places[to];
    const dim3 tiles((unsigned)sort.tiles), block(kBlock);
    const dim3 counting(sort.clear && clears > tiles.x ? clears : tiles.x);
    if (rounds == 4)
      hipLaunchKernelGGL(count_kernel<4>, counting, block, 0, stream, sort);
    else
      hipLaunchKernelGGL(count_kernel<16>, counting, block, 0, stream, sort);
    sort.clear = nullptr;
    if (sort.summed) hipLaunchKernelGGL(sum_up_kernel, dim3(kDigit), block, 0, stream, sort);
    if (rounds == 4)
      hipLaunchKernelGGL(move_kernel<4>, tiles, block, 0, stream, sort);
    else
      hipLaunchKernelGGL(move_kernel<16>, tiles, block, 0, stream, sort);
    status = launch_status();
    if (status != HIPENVS_OK) return status;
    sort.keys = keys[to], sort.places = places[to];
  }
  char* partial = workspace + 4 * l.keys + l.counts;
  const int quads = (d + 3) / 4, group = group_of(quads);
  Sums s = {sort.keys, sort.places, dout, dtable, (float*)partial, (float*)(partial + l.partial), count, v,
            (count + kChunk - 1) / kChunk, dout_s, 0, d, quads, group, (quads + group - 1) / group, scale};
  status = in_launches(s.chunks * s.columns * group, [&](int64_t item0, dim3 grid) {
    s.item0 = item0;
    hipLaunchKernelGGL(chunks_kernel<T>, grid, dim3(kBlock), 0, stream, s);
  });
  if (status != HIPENVS_OK || s.chunks == 1) return status;
  const int64_t blocks = s.chunks * s.columns, most = kMostThreads / kBlock;
  for (s.item0 = 0; s.item0 < blocks; s.item0 += most) {
    const dim3 grid((unsigned)(blocks - s.item0 < most ? blocks - s.item0 : most));
    hipLaunchKernelGGL(across_kernel<T>, grid, dim3(kBlock), 0, stream, s);
    status = launch_status();
    if (status != HIPENVS_OK) return status;
  }
  return HIPENVS_OK;
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
  return count == 0 ? 0 : lay(count, v, d).bytes;
}

extern "C" int hipenvs_embedding_backward(int32_t dtype, const void* tokens, int32_t token_bytes, const void* dout,
                                          int64_t dout_s, float scale, void* dtable, int64_t count, int64_t v,
                                          int32_t d, void* workspace, int64_t workspace_bytes,
                                          hipenvs_stream_t stream) {
  if (!sizes_ok(dtype, count, v, d) || (token_bytes != 4 && token_bytes != 8) || !dtable) return HIPENVS_E_ARG;
  if (count > 0 && (!tokens || !dout || !workspace || ((uintptr_t)workspace & 15) ||
                    workspace_bytes < lay(count, v, d).bytes))
    return HIPENVS_E_ARG;
  if ((uintptr_t)dtable & 15) return HIPENVS_E_ARG;
  const Tokens of = {tokens, token_bytes == 8};
  return dtype == 1 ? gradient<__bf16>(of, dout, dout_s, scale, dtable, count, v, d, (char*)workspace, as_stream(stream))
                    : gradient<float>(of, dout, dout_s, scale, dtable, count, v, d, (char*)workspace, as_stream(stream));
}
