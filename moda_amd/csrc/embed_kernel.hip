// Rows of an embedding by their tokens, y[n] = s E[t_n], and the gradient, dE[v] = s * (the sum of dy[n] over n with t_n = v).
//
// The gradient has one writer for every row and adds in the order of n, so that it has the same bits every time: the tokens are put in
// the order of their words first (a stable sort by digits), after which the rows of a word are neighbours in that order.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/moda_hip.h"
#include "paged.h"
#include "vocab.h"

namespace moda {
namespace {

// Elements as vectors of VEC: 16 bytes, or one element where rows do not lie on that grid.
template <int DT>
struct Element;
template <>
struct Element<MODA_HIP_BF16> {
  typedef uint16_t bits;
  __device__ static float widen(bits x) { return __uint_as_float((uint32_t)x << 16); }
  __device__ static bits narrow(float x) { return __builtin_bit_cast(uint16_t, (__bf16)x); }
};
template <>
struct Element<MODA_HIP_FP16> {
  typedef uint16_t bits;
  __device__ static float widen(bits x) { return (float)__builtin_bit_cast(_Float16, x); }
  __device__ static bits narrow(float x) { return __builtin_bit_cast(uint16_t, (_Float16)x); }
};
template <>
struct Element<MODA_HIP_FP32> {
  typedef uint32_t bits;
  __device__ static float widen(bits x) { return __uint_as_float(x); }
  __device__ static bits narrow(float x) { return __float_as_uint(x); }
};

constexpr int kChunks = 4;  // vectors of a row that a lane has at once

template <typename E, int VEC>
struct Vectors {
  typedef typename E::bits bits;
  typedef bits vec __attribute__((ext_vector_type(VEC)));
};

// 2^lane_shift lanes share a row (kChunks vectors of it each in one go), a wave has 64 >> lane_shift rows.
//
// Bound by the bytes: 64 K rows of 2048 bf16 elements, words as in text, 73 us, 3.7 TB/s written (60 where the rows read are in the caches;
// two or four rows a group: the same; stores through the caches: 78).  Small calls are a launch and two loads, one after the other: 4.6 us.
template <typename E, int VEC, bool STREAM>
__global__ __launch_bounds__(256) void embed_rows_kernel(const EmbedArgs a) {
  typedef typename Vectors<E, VEC>::vec vec;
  typedef typename E::bits bits;
  const int lanes = 1 << a.lane_shift, sub = threadIdx.x & (lanes - 1);
  const int64_t n = ((int64_t)workgroup() * 256 + threadIdx.x) >> a.lane_shift;
  if (n >= a.words.n) return;
  const int word = a.words.of(n);
  const bits* x = (const bits*)a.weight + (int64_t)word * a.ld_in;
  bits* y = (bits*)a.y + n * a.ld_out;
  for (int64_t c0 = sub; c0 * VEC < a.width; c0 += lanes * kChunks) {
    vec v[kChunks];
#pragma unroll
    for (int i = 0; i < kChunks; i++) {
      const int64_t c = c0 + i * lanes;
      v[i] = vec{};
      if (word >= 0 && c * VEC < a.width) v[i] = *(const vec*)(x + c * VEC);
    }
#pragma unroll
    for (int i = 0; i < kChunks; i++) {
      const int64_t c = c0 + i * lanes;
      if (c * VEC >= a.width) break;
      if (a.scale != 1.f)  // (a product with one is the element itself, but for the bits of a NaN)
#pragma unroll
        for (int j = 0; j < VEC; j++) v[i][j] = E::narrow(E::widen(v[i][j]) * a.scale);
      if (STREAM)
        __builtin_nontemporal_store(v[i], (vec*)(y + c * VEC));
      else
        *(vec*)(y + c * VEC) = v[i];
    }
  }
}

// ---------------------------------------------------------------------------------------------------------------------
// the order of words
// ---------------------------------------------------------------------------------------------------------------------
struct Entry {
  uint32_t key, place;
};
__device__ __forceinline__ Entry entry(const SortArgs& a, int64_t i) {
  if (a.keys) return {a.keys[i], a.places[i]};
  const int w = a.words.of(i);
  return {w < 0 ? (uint32_t)a.words.vocab : (uint32_t)w, (uint32_t)i};
}

// (The first pass clears the words' ranges besides: to look whether a range is one costs 64 K tokens on 128 K words 7 us.)
__global__ __launch_bounds__(kSortThreads) void count_digits_kernel(const SortArgs a) {
  __shared__ uint32_t count[kDigits];
  if (!a.keys)
    for (int64_t v = (int64_t)blockIdx.x * kSortThreads + threadIdx.x; v < a.words.vocab; v += (int64_t)a.blocks * kSortThreads) a.range[v] = int2{0, 0};
  for (int d = threadIdx.x; d < kDigits; d += kSortThreads) count[d] = 0;
  __syncthreads();
  const int64_t first = (int64_t)blockIdx.x * kSortThreads * a.rounds;
  for (int r = 0; r < a.rounds; r++) {
    const int64_t i = first + (int64_t)r * kSortThreads + threadIdx.x;
    if (i < a.words.n) atomicAdd(&count[entry(a, i).key >> a.shift & (kDigits - 1)], 1u);
  }
  __syncthreads();
  for (int d = threadIdx.x; d < kDigits; d += kSortThreads) a.counts[(int64_t)blockIdx.x * kDigits + d] = count[d];
}

// How many lanes below this one have its digit, among those that are `there`; same: how many have it in all.
__device__ __forceinline__ int rank_in_wave(int digit, bool there, int& same) {
  uint64_t mask = __ballot(there);
  for (int b = 0; b < kDigitBits; b++) {
    const uint64_t set = __ballot(digit >> b & 1);
    mask &= digit >> b & 1 ? set : ~set;
  }
  same = __popcll(mask);
  return __popcll(mask & ((1ull << (threadIdx.x & 63)) - 1));
}

// Sum over the digits below that of a thread of the first kDigits; total: LDS of a number for each of their waves.
__device__ __forceinline__ uint32_t sum_below(uint32_t count, uint32_t* total) {
  const int tid = threadIdx.x, lane = tid & 63;
  uint32_t upto = count;  // of the digits of this wave up to this one
  for (int s = 1; s < 64; s <<= 1) {
    const uint32_t o = __shfl_up(upto, s, 64);
    upto += lane >= s ? o : 0;
  }
  if (tid < kDigits && lane == 63) total[tid >> 6] = upto;
  __syncthreads();
  uint32_t lower = upto - count;
  if (tid < kDigits)
    for (int w = 0; w < tid >> 6; w++) lower += total[w];
  return lower;
}

// Up to kFewTokens of them: all passes, and the words' ranges, in one workgroup: 3063 tokens 16 us, where five launches took 24.
__global__ __launch_bounds__(kSortThreads) void sort_few_kernel(const SortArgs a, int passes) {
  constexpr int W = kSortThreads / 64;
  __shared__ uint32_t key[kFewTokens], base[kDigits], total[kDigits / 64];
  __shared__ uint16_t place[kFewTokens], in_wave[W][kDigits];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = (int)a.words.n;
  Entry e[kFewRounds];
#pragma unroll
  for (int r = 0; r < kFewRounds; r++) {
    const int i = r * kSortThreads + tid;
    e[r] = i < n ? entry(a, i) : Entry{0, 0};
  }
  for (int p = 0; p < passes; p++) {
    const int shift = p * kDigitBits;
    if (tid < kDigits) base[tid] = 0;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kFewRounds; r++)
      if (r * kSortThreads + tid < n) atomicAdd(&base[e[r].key >> shift & (kDigits - 1)], 1u);
    __syncthreads();
    const uint32_t lower = sum_below(tid < kDigits ? base[tid] : 0, total);
    if (tid < kDigits) base[tid] = lower;
    int to[kFewRounds];
#pragma unroll
    for (int r = 0; r < kFewRounds; r++) {
      if (r * kSortThreads >= n) break;
      for (int d = lane; d < kDigits; d += 64) in_wave[wave][d] = 0;
      const bool there = r * kSortThreads + tid < n;
      const int digit = e[r].key >> shift & (kDigits - 1);
      int same;
      const int rank = rank_in_wave(digit, there, same);
      __syncthreads();
      if (there && rank == 0) in_wave[wave][digit] = (uint16_t)same;
      __syncthreads();
      if (tid < kDigits) {  // counts of the waves -> where each begins
        uint32_t at = base[tid];
#pragma unroll
        for (int w = 0; w < W; w++) {
          const uint32_t c = in_wave[w][tid];
          in_wave[w][tid] = (uint16_t)at;
          at += c;
        }
        base[tid] = at;
      }
      __syncthreads();
      to[r] = in_wave[wave][digit] + rank;
      __syncthreads();
    }
#pragma unroll
    for (int r = 0; r < kFewRounds; r++)
      if (r * kSortThreads + tid < n) {
        key[to[r]] = e[r].key;
        place[to[r]] = (uint16_t)e[r].place;
      }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kFewRounds; r++) {
      const int i = r * kSortThreads + tid;
      if (i < n) e[r] = {key[i], place[i]};
    }
  }
#pragma unroll
  for (int r = 0; r < kFewRounds; r++) {
    const int i = r * kSortThreads + tid;
    if (i >= n) break;
    a.keys_out[i] = e[r].key;
    a.places_out[i] = e[r].place;
    if (e[r].key >= (uint32_t)a.words.vocab) continue;
    if (i == 0 || key[i - 1] != e[r].key) a.range[e[r].key].x = i;
    if (i == n - 1 || key[i + 1] != e[r].key) a.range[e[r].key].y = i + 1;
  }
}

// Where an entry goes: behind all with a lower digit, those with its own of the blocks and rounds before, and those with its own of the
// waves and lanes before it in this round.
__global__ __launch_bounds__(kSortThreads) void place_digits_kernel(const SortArgs a) {
  constexpr int W = kSortThreads / 64;
  static_assert(kSortThreads == 2 * kDigits, "two threads a digit");
  __shared__ uint32_t base[kDigits], in_wave[W][kDigits], total[kDigits / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  uint32_t before = 0, all = 0;
  {
    uint32_t* other = &in_wave[0][0];  // what the second thread of a digit has counted
    const int d = tid & (kDigits - 1), half = (a.blocks + 1) / 2, from = tid < kDigits ? 0 : half, to = tid < kDigits ? half : a.blocks;
#pragma unroll 16
    for (int b = from; b < to; b++) {
      const uint32_t c = a.counts[b * kDigits + d];
      all += c;
      before += b < (int)blockIdx.x ? c : 0;
    }
    if (tid >= kDigits) {
      other[2 * d] = all;
      other[2 * d + 1] = before;
    }
    __syncthreads();
    if (tid < kDigits) {
      all += other[2 * d];
      before += other[2 * d + 1];
    }
  }
  const uint32_t lower = sum_below(tid < kDigits ? all : 0, total);
  if (tid < kDigits) base[tid] = lower + before;
  const int64_t first = (int64_t)blockIdx.x * kSortThreads * a.rounds;
  for (int r = 0; r < a.rounds; r++) {
    for (int d = lane; d < kDigits; d += 64) in_wave[wave][d] = 0;
    __syncthreads();
    const int64_t i = first + (int64_t)r * kSortThreads + tid;
    const bool there = i < a.words.n;
    const Entry e = there ? entry(a, i) : Entry{0, 0};
    const int digit = e.key >> a.shift & (kDigits - 1);
    int same;
    const int rank = rank_in_wave(digit, there, same);
    if (there && rank == 0) in_wave[wave][digit] = (uint32_t)same;
    __syncthreads();
    if (tid < kDigits) {  // counts of the waves -> where each begins
      uint32_t at = base[tid];
      for (int w = 0; w < W; w++) {
        const uint32_t c = in_wave[w][tid];
        in_wave[w][tid] = at;
        at += c;
      }
      base[tid] = at;
    }
    __syncthreads();
    const uint32_t to = in_wave[wave][digit] + rank;
    if (there && to < (uint64_t)a.words.n) {  // (tokens that change during the call make wrong results, no access out of place)
      a.keys_out[to] = e.key;
      a.places_out[to] = e.place;
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------------------------------------------------
// sums of the rows of a word
// ---------------------------------------------------------------------------------------------------------------------

__global__ __launch_bounds__(256) void word_ranges_kernel(const SortArgs a) {
  const int i = (int)(workgroup() * 256 + threadIdx.x), n = (int)a.words.n;
  if (i >= n) return;
  const uint32_t k = a.keys[i];
  if (k >= (uint32_t)a.words.vocab) return;
  if (i == 0 || a.keys[i - 1] != k) a.range[k].x = i;
  if (i == n - 1 || a.keys[i + 1] != k) a.range[k].y = i + 1;
}

// The sum of the rows at places[first .. last), in their order, of a lane's kChunks vectors from c0 on; `lanes` neighbouring lanes share the
// rows, have a place of theirs each and hand them round.
template <typename E, int VEC>
__device__ __forceinline__ void add_rows(const EmbedArgs& a, int first, int last, int64_t c0, int lanes, float (&sum)[kChunks][VEC]) {
  typedef typename Vectors<E, VEC>::vec vec;
  typedef typename E::bits bits;
  constexpr int ROWS = 4;  // in flight
  const int lane = threadIdx.x & 63, sub = lane & (lanes - 1), group = lane - sub;
#pragma unroll
  for (int i = 0; i < kChunks; i++)
#pragma unroll
    for (int j = 0; j < VEC; j++) sum[i][j] = 0.f;
  const bits* x = (const bits*)a.weight;
  for (int b = first; b < last; b += lanes) {
    const uint32_t there = b + sub < last ? a.places[b + sub] : 0;
    const int place = there < (uint32_t)a.words.n ? (int)there : 0, count = min(lanes, last - b);
    for (int r = 0; r < count; r += ROWS) {
      vec v[ROWS][kChunks];
#pragma unroll
      for (int k = 0; k < ROWS; k++) {
        const bits* row = x + (int64_t)__shfl(place, group + r + k, 64) * a.ld_in;
#pragma unroll
        for (int i = 0; i < kChunks; i++) {
          const int64_t c = c0 + i * lanes;
          v[k][i] = vec{};
          if (r + k < count && c * VEC < a.width) v[k][i] = *(const vec*)(row + c * VEC);
        }
      }
#pragma unroll
      for (int k = 0; k < ROWS; k++)
#pragma unroll
        for (int i = 0; i < kChunks; i++)
#pragma unroll
          for (int j = 0; j < VEC; j++) sum[i][j] += E::widen(v[k][i][j]);  // (a row past the end is zeros: nothing is added)
    }
  }
}

// Bound by the bytes: 64 K rows into 128 K words of 2048 bf16 elements, 805 MB in and out, 157 us, 5.1 TB/s (276 with two rows in flight, each behind
// its place's load, eight words a wave and the long runs last); sorting 27, joining 10.
// Blocks below chunk_blocks: pieces of kRunRows sorted places, of which those of longer runs are added up into parts.  Such a run covers
// the first or the last place of each piece that it reaches into, so that there are two at most.
// Blocks behind: words, kWordsOfGroup for each group of lanes: a word's rows added up where they are at most kRunRows, zeros where it has none.
constexpr int kWordsOfGroup = 2;
constexpr int kLeastShift = 3;  // eight lanes a row at least
template <typename E, int VEC, bool STREAM>
__global__ __launch_bounds__(256) void embed_grad_kernel(const EmbedArgs a) {
  typedef typename Vectors<E, VEC>::vec vec;
  typedef typename E::bits bits;
  const int lanes = 1 << a.lane_shift, sub = threadIdx.x & (lanes - 1), groups = 256 >> a.lane_shift, group = threadIdx.x >> a.lane_shift;
  const unsigned block = workgroup();
  const int n = (int)a.words.n, vocab = (int)a.words.vocab;
  float sum[kChunks][VEC];
  if (block < a.chunk_blocks) {
    const int chunk = (int)block * groups + group, p0 = chunk * kRunRows, p1 = min(p0 + kRunRows, n);
    if (chunk >= a.chunks) return;
    const uint32_t k[2] = {a.keys[p0], a.keys[p1 - 1]};
#pragma unroll
    for (int s = 0; s < 2; s++) {
      if (k[s] >= (uint32_t)vocab || (s == 1 && k[1] == k[0])) break;
      const int2 run = a.range[k[s]];
      if (run.y - run.x <= kRunRows) continue;
      float* part = a.parts + (2ll * chunk + s) * a.part_ld;
      for (int64_t c0 = sub; (c0 - sub) * VEC < a.width; c0 += lanes * kChunks) {  // (by all lanes: they hand places round)
        add_rows<E, VEC>(a, max(run.x, p0), min(run.y, p1), c0, lanes, sum);
#pragma unroll
        for (int i = 0; i < kChunks; i++) {
          const int64_t c = c0 + i * lanes;
          if (c * VEC >= a.width) break;
#pragma unroll
          for (int j = 0; j < VEC; j++) part[c * VEC + j] = sum[i][j];
        }
      }
    }
    return;
  }
  const int64_t w0 = ((int64_t)(block - a.chunk_blocks) * groups + group) * kWordsOfGroup;
  int2 run[kWordsOfGroup];
#pragma unroll
  for (int w = 0; w < kWordsOfGroup; w++) {
    run[w] = w0 + w < vocab ? a.range[w0 + w] : int2{0, 0x7fffffff};
    // what the memory of a word's range held that is not there names no place of it
    if (!a.cleared && w0 + w < vocab && ((unsigned)run[w].x >= (unsigned)n || a.keys[run[w].x] != (uint32_t)(w0 + w))) run[w] = int2{0, 0};
  }
#pragma unroll
  for (int w = 0; w < kWordsOfGroup; w++) {
    if (run[w].y - run[w].x > kRunRows) continue;
    bits* y = (bits*)a.y + (w0 + w) * a.ld_out;
    for (int64_t c0 = sub; (c0 - sub) * VEC < a.width; c0 += lanes * kChunks) {  // (by all lanes: they hand places round)
      add_rows<E, VEC>(a, run[w].x, run[w].y, c0, lanes, sum);
#pragma unroll
      for (int i = 0; i < kChunks; i++) {
        const int64_t c = c0 + i * lanes;
        if (c * VEC >= a.width) break;
        vec v;
#pragma unroll
        for (int j = 0; j < VEC; j++) v[j] = E::narrow(run[w].y > run[w].x ? sum[i][j] * a.scale : 0.f);
        if (STREAM)
          __builtin_nontemporal_store(v, (vec*)(y + c * VEC));
        else
          *(vec*)(y + c * VEC) = v;
      }
    }
  }
}

// Runs longer than kRunRows, by the piece that they begin in (one at most; they reach its last place): the sum of their parts, four columns
// a thread.
template <typename E>
__global__ __launch_bounds__(256) void embed_join_kernel(const EmbedArgs a) {
  typedef float f32x4 __attribute__((ext_vector_type(4)));
  const unsigned of_row = (unsigned)((a.part_ld + 1023) / 1024), block = workgroup();
  const int chunk = (int)(block / of_row), p0 = chunk * kRunRows, p1 = min(p0 + kRunRows, (int)a.words.n);
  if (chunk >= a.chunks) return;
  const uint32_t k = a.keys[p1 - 1];
  if (k >= (uint32_t)a.words.vocab) return;
  const int2 run = a.range[k];
  if (run.x < p0 || run.y - run.x <= kRunRows) return;
  const int end = (run.y + kRunRows - 1) / kRunRows;  // pieces
  const int64_t c = (int64_t)(block % of_row) * 1024 + threadIdx.x * 4;
  if (c >= a.width) return;
  const float* part = a.parts + (2ll * chunk + (run.x > p0)) * a.part_ld + c;
  f32x4 s = *(const f32x4*)part;
  part = a.parts + 2ll * (chunk + 1) * a.part_ld + c;
  int q = chunk + 1;
  for (; q + 16 <= end; q += 16, part += 32 * a.part_ld) {
    f32x4 v[16];
#pragma unroll
    for (int i = 0; i < 16; i++) v[i] = *(const f32x4*)(part + 2 * i * a.part_ld);
#pragma unroll
    for (int i = 0; i < 16; i++) s += v[i];
  }
  for (; q < end; q++, part += 2 * a.part_ld) s += *(const f32x4*)part;
  typename E::bits* y = (typename E::bits*)a.y + (int64_t)k * a.ld_out;
#pragma unroll
  for (int i = 0; i < 4; i++)
    if (c + i < a.width) y[c + i] = E::narrow(s[i] * a.scale);
}

template <typename E, int VEC>
hipError_t rows_as(const EmbedArgs& a, bool through, int64_t blocks, hipStream_t stream) {
  through ? embed_rows_kernel<E, VEC, true><<<grid_of(blocks), 256, 0, stream>>>(a) : embed_rows_kernel<E, VEC, false><<<grid_of(blocks), 256, 0, stream>>>(a);
  return hipGetLastError();
}
template <typename E, int VEC>
hipError_t grad_as(const EmbedArgs& a, bool through, int64_t blocks, hipStream_t stream) {
  through ? embed_grad_kernel<E, VEC, true><<<grid_of(blocks), 256, 0, stream>>>(a) : embed_grad_kernel<E, VEC, false><<<grid_of(blocks), 256, 0, stream>>>(a);
  hipError_t e = hipGetLastError();
  if (e == hipSuccess && a.chunks > 1) {
    embed_join_kernel<E><<<grid_of(a.chunks * ((a.part_ld + 1023) / 1024)), 256, 0, stream>>>(a);
    e = hipGetLastError();
  }
  return e;
}
int lane_shift_of(int64_t width, int vec, int least) {
  int s = least;
  while (s < 6 && (int64_t)vec << s < width) s++;
  return s;
}

}  // namespace

// `vec`: rows lie on the 16-byte grid
hipError_t launch_embed_rows(EmbedArgs& a, int dtype, bool vec, hipStream_t stream) {
  const int es = dtype == MODA_HIP_FP32 ? 4 : 2, v = vec ? 16 / es : 1;
  a.lane_shift = lane_shift_of(a.width, v, 0);
  const int64_t blocks = ((a.words.n << a.lane_shift) + 255) / 256;
  const bool through = a.words.n * a.width * es * 2 > 256ll << 20;  // what does not fit the memory-side cache passes it by
  if (dtype == MODA_HIP_FP32)
    return vec ? rows_as<Element<MODA_HIP_FP32>, 4>(a, through, blocks, stream) : rows_as<Element<MODA_HIP_FP32>, 1>(a, through, blocks, stream);
  if (dtype == MODA_HIP_FP16)
    return vec ? rows_as<Element<MODA_HIP_FP16>, 8>(a, through, blocks, stream) : rows_as<Element<MODA_HIP_FP16>, 1>(a, through, blocks, stream);
  return vec ? rows_as<Element<MODA_HIP_BF16>, 8>(a, through, blocks, stream) : rows_as<Element<MODA_HIP_BF16>, 1>(a, through, blocks, stream);
}

hipError_t launch_embed_grad(EmbedArgs& a, int dtype, bool vec, char* work, hipStream_t stream) {
  const EmbedGradPlan p = plan_embed_grad(a.words.n, a.words.vocab, a.width);
  SortArgs s = {};
  s.words = a.words;
  s.counts = (uint32_t*)(work + p.counts);
  s.range = (int2*)(work + p.range);
  s.rounds = p.rounds;
  s.blocks = p.blocks;
  hipError_t e = hipSuccess;
  if (a.words.n <= kFewTokens) {
    s.keys_out = (uint32_t*)(work + p.keys[0]);
    s.places_out = (uint32_t*)(work + p.places[0]);
    if (a.words.n > 0) sort_few_kernel<<<1, kSortThreads, 0, stream>>>(s, p.passes);
    if ((e = hipGetLastError()) != hipSuccess) return e;
    a.keys = s.keys_out;
    a.places = s.places_out;
  } else {
    for (int i = 0; i < p.passes; i++) {
      s.shift = i * kDigitBits;
      s.keys = i == 0 ? nullptr : (const uint32_t*)(work + p.keys[(i - 1) & 1]);
      s.places = i == 0 ? nullptr : (const uint32_t*)(work + p.places[(i - 1) & 1]);
      s.keys_out = (uint32_t*)(work + p.keys[i & 1]);
      s.places_out = (uint32_t*)(work + p.places[i & 1]);
      count_digits_kernel<<<p.blocks, kSortThreads, 0, stream>>>(s);
      if ((e = hipGetLastError()) != hipSuccess) return e;
      place_digits_kernel<<<p.blocks, kSortThreads, 0, stream>>>(s);
      if ((e = hipGetLastError()) != hipSuccess) return e;
    }
    a.keys = s.keys = (const uint32_t*)(work + p.keys[(p.passes - 1) & 1]);
    a.places = (const uint32_t*)(work + p.places[(p.passes - 1) & 1]);
    word_ranges_kernel<<<grid_of((a.words.n + 255) / 256), 256, 0, stream>>>(s);
    if ((e = hipGetLastError()) != hipSuccess) return e;
  }
  a.range = s.range;
  a.cleared = a.words.n > kFewTokens;
  a.parts = (float*)(work + p.parts);
  a.part_ld = p.part_ld;
  a.chunks = (int)p.chunks;
  const int es = dtype == MODA_HIP_FP32 ? 4 : 2, v = vec ? 16 / es : 1;
  a.lane_shift = lane_shift_of(a.width, v, kLeastShift);
  const int64_t groups = 256 >> a.lane_shift, of_block = groups * kWordsOfGroup;
  a.chunk_blocks = (unsigned)((p.chunks + groups - 1) / groups);
  const int64_t blocks = a.chunk_blocks + (a.words.vocab + of_block - 1) / of_block;
  const bool through = (a.words.n + a.words.vocab) * a.width * es > 256ll << 20;
  if (dtype == MODA_HIP_FP32)
    return vec ? grad_as<Element<MODA_HIP_FP32>, 4>(a, through, blocks, stream) : grad_as<Element<MODA_HIP_FP32>, 1>(a, through, blocks, stream);
  if (dtype == MODA_HIP_FP16)
    return vec ? grad_as<Element<MODA_HIP_FP16>, 8>(a, through, blocks, stream) : grad_as<Element<MODA_HIP_FP16>, 1>(a, through, blocks, stream);
  return vec ? grad_as<Element<MODA_HIP_BF16>, 8>(a, through, blocks, stream) : grad_as<Element<MODA_HIP_BF16>, 1>(a, through, blocks, stream);
}

}  // namespace moda
