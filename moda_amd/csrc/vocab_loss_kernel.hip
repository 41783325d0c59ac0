// The cross entropy of rows over a vocabulary without keeping the logits, z[n][v] = s x[n] W[v]:
//   lse[n] = log sum_v exp z[n][v],  l[n] = lse[n] - z[n][t_n]
//   dz[n][v] = g[n] (exp(z[n][v] - lse[n]) - [v = t_n]),  dx = s dz W,  dW = s dz^T x
// Rows without a target are left out from the start: the others are laid one behind the other first (gather_rows_kernel), so that what is
// in the rows left out, NaN included, reaches nothing and costs nothing.  The logits leave the registers as a largest value and a sum of
// exponentials for every tile of words, which a second launch joins in the words' order, behind what the pieces of the vocabulary before have
// come to.  The backward pass computes them once more, a piece of the vocabulary at a time, and keeps that piece's gradient in 16 bits (fp32: 48)
// for the two products that read it.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/moda_hip.h"
#include "paged.h"
#include "product.h"
#include "vocab.h"

namespace moda {
namespace {

constexpr float kLn2 = 0.69314718055994531f;

// Eight elements of a row from column c on (zeros behind its end), on their way to the products' planes.
template <int DT>
struct Eight {
  static constexpr int SIZE = DT == MODA_HIP_FP32 ? 2 : 1;
  i32x4 v[SIZE];
  __device__ __forceinline__ void load(const char* row, int64_t c, int64_t width, bool vec) {
    if (vec && c + 8 <= width) {
#pragma unroll
      for (int i = 0; i < SIZE; i++) v[i] = *(const i32x4*)(row + c * 2 * SIZE + 16 * i);
      return;
    }
#pragma unroll
    for (int i = 0; i < SIZE; i++) v[i] = i32x4{0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 8; i++) {
      if (c + i >= width) break;
      if constexpr (SIZE == 2)
        v[i >> 2][i & 3] = ((const int*)row)[c + i];
      else
        v[0][i >> 1] |= (int)((uint32_t)((const uint16_t*)row)[c + i] << (16 * (i & 1)));
    }
  }
  __device__ __forceinline__ void store(uint16_t* to, int64_t plane) const {
    if constexpr (SIZE == 2) {
      uint16_t piece[8][3];
#pragma unroll
      for (int i = 0; i < 8; i++) three_pieces(__int_as_float(v[i >> 2][i & 3]), piece[i]);
#pragma unroll
      for (int k = 0; k < 3; k++) {
        i32x4 w;
#pragma unroll
        for (int i = 0; i < 4; i++) w[i] = piece[2 * i][k] | piece[2 * i + 1][k] << 16;
        *(i32x4*)(to + k * plane) = w;
      }
    } else {
      *(i32x4*)to = v[0];
    }
  }
};

// Sums of the workgroup's 256 threads, and their largest.
__device__ __forceinline__ void over_block(int& a, int& b, int& largest) {
  __shared__ int sums[3][4];
#pragma unroll
  for (int s = 32; s > 0; s >>= 1) {
    a += __shfl_xor(a, s, 64);
    b += __shfl_xor(b, s, 64);
    largest = max(largest, __shfl_xor(largest, s, 64));
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 0) {
    sums[0][threadIdx.x >> 6] = a;
    sums[1][threadIdx.x >> 6] = b;
    sums[2][threadIdx.x >> 6] = largest;
  }
  __syncthreads();
  a = sums[0][0] + sums[0][1] + sums[0][2] + sums[0][3];
  b = sums[1][0] + sums[1][1] + sums[1][2] + sums[1][3];
  largest = max(max(sums[2][0], sums[2][1]), max(sums[2][2], sums[2][3]));
}

// the size of a row's upstream gradient as the bits of a float, which order as it does; zero where it is not finite
__device__ __forceinline__ int size_of(const GatherArgs& a, int64_t i) {
  const int bits = a.d_loss ? (int)(__float_as_uint(a.d_loss[i * a.d_loss_stride]) & 0x7fffffffu) : 0;
  return bits < 0x7f800000 ? bits : 0;
}

// Where every workgroup of the gather would otherwise look at more than kScanMost targets: rows with one of each kCountBlock.
__global__ __launch_bounds__(256) void count_rows_kernel(const GatherArgs a) {
  const int64_t first = (int64_t)workgroup() * kCountBlock;
  int live = 0, unused = 0, e = 0;
  for (int64_t i = first + threadIdx.x; i < first + kCountBlock && i < a.words.n; i += 256)
    if (a.words.of(i) >= 0) {
      live++;
      e = max(e, size_of(a, i));
    }
  over_block(live, unused, e);
  if (threadIdx.x == 0) {
    a.counts[workgroup()] = live;
    a.largest[workgroup()] = e;
  }
}

// A workgroup has kGatherBlock rows; it counts those with a target before them, and all, by itself.  Bound by latency, then by the bytes: 8192 rows of
// 2048 bf16 elements 17 us (67 MB), 509 of 1000 6 us; with 32 rows a workgroup 46 and 15.
template <int DT>
__global__ __launch_bounds__(256) void gather_rows_kernel(const GatherArgs a) {
  __shared__ int to[kGatherBlock];  // where a row goes, or -1
  const int tid = threadIdx.x;
  const int64_t n = a.words.n, first = (int64_t)workgroup() * kGatherBlock;
  int before = 0, all = 0, e = 0;
  int64_t from = 0, upto = n;
  if (a.counts) {
    const int64_t own = first / kCountBlock, blocks = (n + kCountBlock - 1) / kCountBlock;
    for (int64_t i = tid; i < blocks; i += 256) {
      const int c = a.counts[i];
      all += c;
      before += i < own ? c : 0;
      e = max(e, a.largest[i]);
    }
    from = own * kCountBlock;
    upto = first;
  }
  constexpr int AHEAD = 8;  // targets in flight
  for (int64_t i0 = from + tid; i0 < upto; i0 += 256 * AHEAD) {
    int word[AHEAD], size[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; k++) {
      const int64_t i = i0 + 256 * k;
      word[k] = i < upto ? a.words.of(i) : -1;
      size[k] = i < upto && a.d_loss_stride ? size_of(a, i) : 0;
    }
#pragma unroll
    for (int k = 0; k < AHEAD; k++) {
      before += word[k] >= 0 && i0 + 256 * k < first;
      if (!a.counts && word[k] >= 0) {
        all++;
        e = max(e, size[k]);
      }
    }
  }
  if (a.d_loss && !a.d_loss_stride) e = size_of(a, 0);
  over_block(before, all, e);
  // The gradient of a logit is rounded to 16 bits.  The factor that rows share stays out of that, or its own rounding would be in all of them,
  // the same way: it is kept relative to the largest upstream gradient, which the products multiply by at their end.
  const float most = e > 0 ? __uint_as_float((uint32_t)e) : 1.f;
  if (first == 0 && tid < 64) {
    // How the words are split for the gradient of so many rows: the time of each choice, a lane a choice (choose_tiling's estimate).
    int splits = tid + 1;
    float us = __builtin_huge_valf();
    if (a.rule.steps > 0 && (int64_t)splits * all <= a.rule.most * n && (splits == 1 || a.rule.steps >= 4 * splits)) {
      const int items = (all + a.rule.tile_p - 1) / a.rule.tile_p * a.rule.tiles_f * splits;
      us = (float)((items + a.rule.at_once - 1) / a.rule.at_once) * ((float)((a.rule.steps + splits - 1) / splits) * a.rule.step_us + a.rule.end_us) +
           (float)splits * (float)all * a.rule.split_us;
    }
    for (int s = 32; s > 0; s >>= 1) {
      const float other_us = __shfl_xor(us, s, 64);
      const int other = __shfl_xor(splits, s, 64);
      if (other_us < us || (other_us == us && other < splits)) {
        us = other_us;
        splits = other;
      }
    }
    if (us == __builtin_huge_valf()) splits = 1;
    if (tid == 0) *a.head = LossHead{all, splits, a.d_loss ? most / (a.mean ? (float)max(all, 1) : 1.f) / a.up : 1.f};
  }
  if (tid < 64) {
    const int64_t i = first + tid;
    const int word = tid < kGatherBlock && i < n ? a.words.of(i) : -1;
    const uint64_t mask = __ballot(word >= 0);
    const int at = before + __popcll(mask & ((1ull << tid) - 1));
    if (tid < kGatherBlock) to[tid] = word >= 0 ? at : -1;
    if (word >= 0) {
      a.row_of[at] = (int)i;
      a.target[at] = word;
      if (a.d_loss) {
        a.factor[at] = a.d_loss[i * a.d_loss_stride] / most * a.up;
        a.lse[at] = a.lse_in[i];
      }
    } else if (tid < kGatherBlock && i < n && a.loss) {
      a.loss[i] = 0.f;
      a.lse_out[i] = 0.f;
    }
  }
  __syncthreads();
  constexpr int ES = DT == MODA_HIP_FP32 ? 4 : 2, COPIES = 4;  // (in flight)
  const int chunks = (int)(a.rows_ld / 8), lane = tid & 63;
  for (int r = tid >> 6; r < kGatherBlock && first + r < n; r += 4) {
    const int64_t i = first + r;
    if (to[r] >= 0) {
      const char* row = a.x + i * a.ld_x * ES;
      uint16_t* out = a.rows + to[r] * a.rows_ld;
      for (int c0 = lane; c0 < chunks; c0 += 64 * COPIES) {
        Eight<DT> x[COPIES];
#pragma unroll
        for (int k = 0; k < COPIES; k++)
          if (c0 + 64 * k < chunks) x[k].load(row, (c0 + 64 * k) * 8, a.width, a.vec_x);
#pragma unroll
        for (int k = 0; k < COPIES; k++)
          if (c0 + 64 * k < chunks) x[k].store(out + (c0 + 64 * k) * 8, a.rows_plane);
      }
    } else if (a.dx) {
      const float zeros[4] = {0.f, 0.f, 0.f, 0.f};
      for (int64_t c = 4 * lane; c < a.width; c += 256)
        store_four<BF16, DT == MODA_HIP_FP32>(a.dx + i * a.ld_dx * ES, c, zeros, (int)min(a.width - c, (int64_t)4), a.vec_dx);
    }
  }
}

template <int DT>
__global__ __launch_bounds__(256) void lay_rows_kernel(const LayArgs a) {
  const int64_t chunks = a.to_ld / 8, w = (int64_t)workgroup() * 256 + threadIdx.x, r = w / chunks, c = w - r * chunks;
  if (r >= a.rows) return;
  Eight<DT> x;
  x.load(a.x + r * a.ld_x * (DT == MODA_HIP_FP32 ? 4 : 2), c * 8, a.width, a.vec);
  x.store(a.to + r * a.to_ld + c * 8, a.to_plane);
}

// Bound by latency: one row of 250 tiles 4 us, 4096 rows of 256 tiles 9.
// LANES lanes a row take every LANES-th tile of words each and meet in LDS, in a fixed order.
template <int LANES>
__global__ __launch_bounds__(256) void join_stats_kernel(const JoinStatsArgs a) {
  constexpr int ROWS = 256 / LANES, AHEAD = 4;
  __shared__ float largest[LANES][ROWS + 1], sum[LANES][ROWS + 1];
  const int r = threadIdx.x % ROWS, part = threadIdx.x / ROWS;
  const int rows = a.head ? a.head->live : (int)a.words.n;
  const int64_t p = (int64_t)workgroup() * ROWS + r;
  float m = kNegInf, s = 0.f;
  if (part == 0 && p < rows && !a.first) {
    const float2 before = a.carry[p];
    m = before.x;
    s = before.y;
  }
  const auto add = [](float& m, float& s, float xm, float xs) {  // (a sum of no logit above minus infinity is zero, or NaN)
    if (xm > m) {
      s = (m == kNegInf ? s : s * fast_exp2(m - xm)) + xs;
      m = xm;
    } else {
      s += xm == kNegInf ? xs : xs * fast_exp2(xm - m);
    }
  };
  if (p < rows)
    for (int64_t t0 = part; t0 < a.tiles; t0 += LANES * AHEAD) {
      float2 x[AHEAD];
#pragma unroll
      for (int k = 0; k < AHEAD; k++) x[k] = t0 + LANES * k < a.tiles ? a.stats[(t0 + LANES * k) * a.stats_ld + p] : float2{kNegInf, 0.f};
#pragma unroll
      for (int k = 0; k < AHEAD; k++) add(m, s, x[k].x, x[k].y);
    }
  for (int half = LANES / 2; half > 0; half >>= 1) {
    largest[part][r] = m;
    sum[part][r] = s;
    __syncthreads();
    if (part < half) add(m, s, largest[part + half][r], sum[part + half][r]);
    __syncthreads();
  }
  if (part != 0 || p >= rows) return;
  if (!a.last) {
    a.carry[p] = float2{m, s};
    return;
  }
  const float log_sum = log2f(s);
  float lse = m + log_sum;
  const int word = a.head ? 0 : a.words.of(p);
  float loss = (m - a.target_logit[p] + log_sum) * kLn2;  // (a target that is the likeliest word: log_sum alone, with all its bits)
  if (word < 0) lse = loss = 0.f;
  const int64_t row = a.head ? a.row_of[p] : p;
  if ((uint64_t)row >= (uint64_t)a.words.n) return;  // (targets that change during the call)
  a.loss[row] = loss;
  a.lse[row] = lse;
}

__global__ __launch_bounds__(1024) void loss_total_kernel(const LossTotalArgs a) {
  __shared__ double part[16];
  __shared__ int count[16];
  double s = 0.;
  int live = 0;
  for (int64_t i = threadIdx.x; i < a.words.n; i += 1024) {
    s += (double)a.rows[i];
    if (!a.head) live += a.words.of(i) >= 0;
  }
  for (int k = 32; k > 0; k >>= 1) {
    s += __shfl_xor(s, k, 64);
    live += __shfl_xor(live, k, 64);
  }
  if ((threadIdx.x & 63) == 0) {
    part[threadIdx.x >> 6] = s;
    count[threadIdx.x >> 6] = live;
  }
  __syncthreads();
  if (threadIdx.x != 0) return;
  for (int i = 1; i < 16; i++) {
    s += part[i];
    live += count[i];
  }
  if (a.head) live = a.head->live;
  *a.total = (float)(a.mean ? s / (double)max(live, 1) : s);
}

// Sums of a split summation axis, in its order.
template <typename T, bool FP32_OUT>
__global__ __launch_bounds__(256) void join_sums_kernel(const JoinSumsArgs a) {
  const int64_t chunks = (a.width + 3) / 4, w = (int64_t)workgroup() * 256 + threadIdx.x, p = w / chunks, f = (w - p * chunks) * 4;
  const int64_t rows = a.head && a.by_head ? a.head->live : a.rows;
  if (p >= rows) return;
  const int splits = a.by_head ? a.head->splits : a.splits;
  const int64_t acc_split = a.by_head ? rows * a.acc_ld : a.acc_split;
  const float* from = a.acc + p * a.acc_ld + f;
  f32x4 s = {0.f, 0.f, 0.f, 0.f};
  int i = 0;
  for (; i + 8 <= splits; i += 8) {
    f32x4 v[8];
#pragma unroll
    for (int k = 0; k < 8; k++) v[k] = *(const f32x4*)(from + (i + k) * acc_split);
#pragma unroll
    for (int k = 0; k < 8; k++) s += v[k];
  }
#pragma unroll 4
  for (; i < splits; i++) s += *(const f32x4*)(from + i * acc_split);
  const float scale = a.scale * a.head->down;
  const float v[4] = {s[0] * scale, s[1] * scale, s[2] * scale, s[3] * scale};
  const int64_t row = a.by_head ? a.row_of[p] : p;
  if ((uint64_t)row >= (uint64_t)a.rows) return;  // (targets that change during the call)
  store_four<T, FP32_OUT>(a.out, row * a.out_ld + f, v, (int)min(a.width - f, (int64_t)4), a.out_vec);
}

int64_t blocks_for(int64_t items) { return (items + 255) / 256; }

#define MODA_BY_TYPE(kernel, dtype, blocks, a)                                     \
  (dtype) == MODA_HIP_FP32   ? kernel<MODA_HIP_FP32><<<grid_of(blocks), 256, 0, stream>>>(a) \
  : (dtype) == MODA_HIP_FP16 ? kernel<MODA_HIP_FP16><<<grid_of(blocks), 256, 0, stream>>>(a) \
                             : kernel<MODA_HIP_BF16><<<grid_of(blocks), 256, 0, stream>>>(a)

}  // namespace

hipError_t launch_gather_rows(const GatherArgs& a, int dtype, hipStream_t stream) {
  if (a.counts) {
    count_rows_kernel<<<grid_of((a.words.n + kCountBlock - 1) / kCountBlock), 256, 0, stream>>>(a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  const int64_t blocks = (a.words.n + kGatherBlock - 1) / kGatherBlock;
  MODA_BY_TYPE(gather_rows_kernel, dtype, blocks > 0 ? blocks : 1, a);  // (one, for the head)
  return hipGetLastError();
}
hipError_t launch_lay_rows(const LayArgs& a, int dtype, hipStream_t stream) {
  MODA_BY_TYPE(lay_rows_kernel, dtype, blocks_for(a.rows * (a.to_ld / 8)), a);
  return hipGetLastError();
}
hipError_t launch_stats(const ProductArgs& a, int dtype, ProductTile tile, int compute_units, hipStream_t stream) { return launch_product<kStats>(a, dtype, tile, compute_units, stream); }
hipError_t launch_grad_logits(const ProductArgs& a, int dtype, ProductTile tile, int compute_units, hipStream_t stream) {
  return launch_product<kGradLogits>(a, dtype, tile, compute_units, stream);
}
hipError_t launch_join_stats(const JoinStatsArgs& a, hipStream_t stream) {
  // lanes enough for one round of loads where there are few rows, coalesced loads where there are many
  if (a.words.n <= 512)
    join_stats_kernel<256><<<grid_of(a.words.n), 256, 0, stream>>>(a);
  else if (a.words.n <= 8192)
    join_stats_kernel<64><<<grid_of((a.words.n + 3) / 4), 256, 0, stream>>>(a);
  else
    join_stats_kernel<16><<<grid_of((a.words.n + 15) / 16), 256, 0, stream>>>(a);
  return hipGetLastError();
}
hipError_t launch_loss_total(const LossTotalArgs& a, hipStream_t stream) {
  loss_total_kernel<<<1, 1024, 0, stream>>>(a);
  return hipGetLastError();
}
hipError_t launch_join_sums(const JoinSumsArgs& a, int dtype, hipStream_t stream) {
  const dim3 grid = grid_of(blocks_for(a.rows * ((a.width + 3) / 4)));
  dtype == MODA_HIP_FP32   ? join_sums_kernel<BF16, true><<<grid, 256, 0, stream>>>(a)
  : dtype == MODA_HIP_FP16 ? join_sums_kernel<FP16, false><<<grid, 256, 0, stream>>>(a)
                           : join_sums_kernel<BF16, false><<<grid, 256, 0, stream>>>(a);
  return hipGetLastError();
}

}  // namespace moda
