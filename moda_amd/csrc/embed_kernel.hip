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
// Bound by the bytes: 64 K rows of 2048 bf16 elements.  Small calls are a launch and two loads, one after the other.
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

__global__ __launch_bounds__(kSortThreads) void count_digits_kernel(const SortArgs a) {
  __shared__ uint32_t count[kDigits];
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

// Where an entry goes: behind all with a lower digit, those with its own of the blocks and rounds before, and those with its own of the
// waves and lanes before it in this round.
__global__ __launch_bounds__(kSortThreads) void place_digits_kernel(const SortArgs a) {
  constexpr int W = kSortThreads / 64;
  __shared__ uint32_t base[kDigits], in_wave[W][kDigits], total[kDigits / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  uint32_t before = 0, all = 0, upto = 0;
  if (tid < kDigits) {
    for (int b = 0; b < a.blocks; b++) {
      const uint32_t c = a.counts[(int64_t)b * kDigits + tid];
      all += c;
      before += b < (int)blockIdx.x ? c : 0;
    }
    upto = all;  // of the digits of this wave up to this one
    for (int s = 1; s < 64; s <<= 1) {
      const uint32_t o = __shfl_up(upto, s, 64);
      upto += lane >= s ? o : 0;
    }
    if (lane == 63) total[wave] = upto;
  }
  __syncthreads();
  if (tid < kDigits) {
    uint32_t lower = upto - all;
    for (int w = 0; w < wave; w++) lower += total[w];
    base[tid] = lower + before;
  }
  const int64_t first = (int64_t)blockIdx.x * kSortThreads * a.rounds;
  for (int r = 0; r < a.rounds; r++) {
    for (int d = lane; d < kDigits; d += 64) in_wave[wave][d] = 0;
    __syncthreads();
    const int64_t i = first + (int64_t)r * kSortThreads + tid;
    const bool there = i < a.words.n;
    const Entry e = there ? entry(a, i) : Entry{0, 0};
    const int digit = e.key >> a.shift & (kDigits - 1);
    uint64_t same = __ballot(there);
    for (int b = 0; b < kDigitBits; b++) {
      const uint64_t set = __ballot(digit >> b & 1);
      same &= digit >> b & 1 ? set : ~set;
    }
    const int rank = __popcll(same & ((1ull << lane) - 1));
    if (there && rank == 0) in_wave[wave][digit] = (uint32_t)__popcll(same);
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
    if (there) {
      const uint32_t to = in_wave[wave][digit] + rank;
      a.keys_out[to] = e.key;
      a.places_out[to] = e.place;
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------------------------------------------------
// sums of the rows of a word
// ---------------------------------------------------------------------------------------------------------------------

// How many of the places lo .. hi - 1 satisfy `holds`, which none does behind one that does not; by a wave, 64 places in one go.  (In 32 bits:
// a loop of this form over 64-bit uniform values was compiled to selects by a stale condition.)
template <typename Holds>
__device__ __forceinline__ int count_while(int lo, int hi, Holds holds) {
  const int lane = threadIdx.x & 63, first = lo;
  while (hi > lo) {
    const int step = (hi - lo + 63) >> 6, at = lo + (lane + 1) * step - 1;  // the last place of this lane's piece
    const int from = lo + __popcll(__ballot(at < hi && holds(at))) * step;  // pieces that hold altogether
    hi = min(from + step - 1, hi);
    lo = min(from, hi);
  }
  return lo - first;
}

// the sum of the rows at places[first .. last), in their order, of a lane's kChunks vectors from c0 on
template <typename E, int VEC>
__device__ __forceinline__ void add_rows(const EmbedArgs& a, int first, int last, int64_t c0, int lanes, float (&sum)[kChunks][VEC]) {
  typedef typename Vectors<E, VEC>::vec vec;
  typedef typename E::bits bits;
#pragma unroll
  for (int i = 0; i < kChunks; i++)
#pragma unroll
    for (int j = 0; j < VEC; j++) sum[i][j] = 0.f;
  const bits* x = (const bits*)a.weight;
  constexpr int ROWS = 2;  // in flight
  for (int r = first; r < last; r += ROWS) {
    vec v[ROWS][kChunks];
#pragma unroll
    for (int k = 0; k < ROWS; k++) {
      const bool there = r + k < last;
      const bits* row = x + (int64_t)(there ? a.places[r + k] : 0) * a.ld_in;
#pragma unroll
      for (int i = 0; i < kChunks; i++) {
        const int64_t c = c0 + i * lanes;
        v[k][i] = vec{};
        if (there && c * VEC < a.width) v[k][i] = *(const vec*)(row + c * VEC);
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

// Blocks below word_blocks: kWordsOfBlock words each, a word's rows added up where they are at most kRunRows, zeros where there are none.
// Blocks behind: pieces of kRunRows sorted places, of which those of longer runs (two at most: each is longer than a piece) are added up
// into parts.
constexpr int kWordsOfBlock = 32;
constexpr int kLeastShift = 3;  // eight lanes a row at least
template <typename E, int VEC, bool STREAM>
__global__ __launch_bounds__(256) void embed_grad_kernel(const EmbedArgs a) {
  typedef typename Vectors<E, VEC>::vec vec;
  typedef typename E::bits bits;
  const int lanes = 1 << a.lane_shift, lane = threadIdx.x & 63, sub = lane & (lanes - 1), wave = threadIdx.x >> 6;
  const unsigned block = workgroup();
  const int n = (int)a.words.n, vocab = (int)a.words.vocab;
  float sum[kChunks][VEC];
  if (block < a.word_blocks) {
    __shared__ int from[kWordsOfBlock], upto[kWordsOfBlock], range[2];
    const int w0 = (int)block * kWordsOfBlock;
    if (threadIdx.x < kWordsOfBlock) from[threadIdx.x] = upto[threadIdx.x] = 0;
    if (wave < 2) {
      const uint32_t w = (uint32_t)min(wave == 0 ? w0 : w0 + min(kWordsOfBlock, vocab - w0), vocab);
      const int at = count_while(0, n, [&](int i) { return a.keys[i] < w; });
      if (lane == 0) range[wave] = at;
    }
    __syncthreads();
    const int lo = range[0], hi = range[1];
    for (int i = lo + (int)threadIdx.x; i < hi; i += 256) {
      const uint32_t k = a.keys[i];
      if (i == lo || a.keys[i - 1] != k) from[k - w0] = i;
      if (i == hi - 1 || a.keys[i + 1] != k) upto[k - w0] = i + 1;
    }
    __syncthreads();
    const int rows = 256 >> a.lane_shift;  // words at once
    for (int w = threadIdx.x >> a.lane_shift; w < kWordsOfBlock; w += rows) {
      if (w >= vocab - w0) break;
      const int first = from[w], last = upto[w];
      if (last - first > kRunRows) continue;
      bits* y = (bits*)a.y + (int64_t)(w0 + w) * a.ld_out;
      for (int64_t c0 = sub; c0 * VEC < a.width; c0 += lanes * kChunks) {
        add_rows<E, VEC>(a, first, last, c0, lanes, sum);
#pragma unroll
        for (int i = 0; i < kChunks; i++) {
          const int64_t c = c0 + i * lanes;
          if (c * VEC >= a.width) break;
          vec v;
#pragma unroll
          for (int j = 0; j < VEC; j++) v[j] = E::narrow(last > first ? sum[i][j] * a.scale : 0.f);
          if (STREAM)
            __builtin_nontemporal_store(v, (vec*)(y + c * VEC));
          else
            *(vec*)(y + c * VEC) = v;
        }
      }
    }
    return;
  }
  // the keys of this block's pieces, and of kRunRows places on either side
  __shared__ uint32_t near[(256 >> kLeastShift) * kRunRows + 2 * kRunRows];
  const int of_block = 256 >> a.lane_shift, group = threadIdx.x >> a.lane_shift;
  const int chunk0 = (int)(block - a.word_blocks) * of_block, chunk = chunk0 + group;
  for (int i = threadIdx.x; i < (of_block + 2) * kRunRows; i += 256) {
    const int at = (chunk0 - 1) * kRunRows + i;
    near[i] = at >= 0 && at < n ? a.keys[at] : 0xffffffffu;  // (no key is as large)
  }
  __syncthreads();
  const uint32_t* keys = near + (group + 1) * kRunRows;
  for (int first = 0; first < kRunRows;) {
    const uint32_t k = keys[first];
    if (k >= (uint32_t)vocab) return;  // no words from here on
    int last = first + 1;
    while (last < kRunRows && keys[last] == k) last++;
    // longer than kRunRows?  A run that is has more than that many places within that many of this one's ends.
    int b = first, e = last;
    while (b > -kRunRows && keys[b - 1] == k) b--;
    while (e < 2 * kRunRows && keys[e] == k) e++;
    if (e - b > kRunRows) {
      float* part = a.parts + (2ll * chunk + (first > 0)) * a.part_ld;
      for (int64_t c0 = sub; c0 * VEC < a.width; c0 += lanes * kChunks) {
        add_rows<E, VEC>(a, chunk * kRunRows + first, chunk * kRunRows + last, c0, lanes, sum);
#pragma unroll
        for (int i = 0; i < kChunks; i++) {
          const int64_t c = c0 + i * lanes;
          if (c * VEC >= a.width) break;
#pragma unroll
          for (int j = 0; j < VEC; j++) part[c * VEC + j] = sum[i][j];
        }
      }
    }
    first = last;
  }
}

// Runs longer than kRunRows, by the piece that they begin in (one at most): the sum of their parts.
template <typename E>
__global__ __launch_bounds__(256) void embed_join_kernel(const EmbedArgs a) {
  const int chunk = (int)workgroup(), n = (int)a.words.n, p0 = chunk * kRunRows, p1 = min(p0 + kRunRows, n);
  if (p0 >= n) return;
  // the last run that begins here, if it reaches past kRunRows places
  int first = p1 - 1;
  const uint32_t k = a.keys[first];
  if (k >= (uint32_t)a.words.vocab) return;  // (a run that ends before the piece does is no long one)
  while (first > p0 && a.keys[first - 1] == k) first--;
  if (first == p0 && p0 > 0 && a.keys[p0 - 1] == k) return;  // begins earlier
  if (first + kRunRows >= n || a.keys[first + kRunRows] != k) return;
  const int last = first + kRunRows + count_while(first + kRunRows, n, [&](int i) { return a.keys[i] == k; });
  const int end = (last + kRunRows - 1) / kRunRows;  // pieces
  typename E::bits* y = (typename E::bits*)a.y + (int64_t)k * a.ld_out;
  for (int64_t c = threadIdx.x; c < a.width; c += 256) {
    const float* part = a.parts + (2ll * chunk + (first > p0)) * a.part_ld + c;
    float s = *part;
    part = a.parts + 2ll * (chunk + 1) * a.part_ld + c;
    int q = chunk + 1;
    for (; q + 8 <= end; q += 8, part += 16 * a.part_ld) {
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; i++) v[i] = part[2 * i * a.part_ld];
#pragma unroll
      for (int i = 0; i < 8; i++) s += v[i];
    }
    for (; q < end; q++, part += 2 * a.part_ld) s += *part;
    y[c] = E::narrow(s * a.scale);
  }
}

template <typename E, int VEC>
hipError_t rows_as(const EmbedArgs& a, bool through, int64_t blocks, hipStream_t stream) {
  through ? embed_rows_kernel<E, VEC, true><<<grid_of(blocks), 256, 0, stream>>>(a) : embed_rows_kernel<E, VEC, false><<<grid_of(blocks), 256, 0, stream>>>(a);
  return hipGetLastError();
}
template <typename E, int VEC>
hipError_t grad_as(const EmbedArgs& a, bool through, int64_t blocks, int64_t chunks, hipStream_t stream) {
  through ? embed_grad_kernel<E, VEC, true><<<grid_of(blocks), 256, 0, stream>>>(a) : embed_grad_kernel<E, VEC, false><<<grid_of(blocks), 256, 0, stream>>>(a);
  hipError_t e = hipGetLastError();
  if (e == hipSuccess && chunks > 1) {
    embed_join_kernel<E><<<grid_of(chunks), 256, 0, stream>>>(a);
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
  s.rounds = p.rounds;
  s.blocks = p.blocks;
  for (int i = 0; i < p.passes && a.words.n > 0; i++) {
    s.shift = i * kDigitBits;
    s.keys = i == 0 ? nullptr : (const uint32_t*)(work + p.keys[(i - 1) & 1]);
    s.places = i == 0 ? nullptr : (const uint32_t*)(work + p.places[(i - 1) & 1]);
    s.keys_out = (uint32_t*)(work + p.keys[i & 1]);
    s.places_out = (uint32_t*)(work + p.places[i & 1]);
    count_digits_kernel<<<p.blocks, kSortThreads, 0, stream>>>(s);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    place_digits_kernel<<<p.blocks, kSortThreads, 0, stream>>>(s);
    if ((e = hipGetLastError()) != hipSuccess) return e;
  }
  a.keys = (const uint32_t*)(work + p.keys[(p.passes - 1) & 1]);
  a.places = (const uint32_t*)(work + p.places[(p.passes - 1) & 1]);
  a.parts = (float*)(work + p.parts);
  a.part_ld = p.part_ld;
  const int es = dtype == MODA_HIP_FP32 ? 4 : 2, v = vec ? 16 / es : 1;
  a.lane_shift = lane_shift_of(a.width, v, kLeastShift);
  a.word_blocks = (unsigned)((a.words.vocab + kWordsOfBlock - 1) / kWordsOfBlock);
  const int64_t of_block = 256 >> a.lane_shift, blocks = a.word_blocks + (p.chunks + of_block - 1) / of_block;
  const bool through = (a.words.n + a.words.vocab) * a.width * es > 256ll << 20;
  if (dtype == MODA_HIP_FP32)
    return vec ? grad_as<Element<MODA_HIP_FP32>, 4>(a, through, blocks, p.chunks, stream) : grad_as<Element<MODA_HIP_FP32>, 1>(a, through, blocks, p.chunks, stream);
  if (dtype == MODA_HIP_FP16)
    return vec ? grad_as<Element<MODA_HIP_FP16>, 8>(a, through, blocks, p.chunks, stream) : grad_as<Element<MODA_HIP_FP16>, 1>(a, through, blocks, p.chunks, stream);
  return vec ? grad_as<Element<MODA_HIP_BF16>, 8>(a, through, blocks, p.chunks, stream) : grad_as<Element<MODA_HIP_BF16>, 1>(a, through, blocks, p.chunks, stream);
}

}  // namespace moda
