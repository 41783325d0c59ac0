// The cross entropy of rows over a vocabulary without keeping the logits, z[n][v] = s x[n] W[v]:
//   lse[n] = log sum_v exp z[n][v],  l[n] = lse[n] - z[n][t_n]
//   dz[n][v] = g[n] (exp(z[n][v] - lse[n]) - [v = t_n]),  dx = s dz W,  dW = s dz^T x
// Rows without a target are left out from the start: the others are laid one behind the other first (gather_rows_kernel), so that what is
// in the rows left out, NaN included, reaches nothing and costs nothing.  The logits leave the registers as a largest value and a sum of
// exponentials for every tile of words, which a second launch joins in the words' order.  The backward pass computes them once more, a piece
// of the vocabulary at a time, and keeps that piece's gradient in 16 bits (fp32: 48) for the two products that read it.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/moda_hip.h"
#include "paged.h"
#include "product.h"
#include "vocab.h"

namespace moda {
namespace {

constexpr float kLn2 = 0.69314718055994531f;

// Eight elements of a row from column c on (zeros behind its end) -> the products' planes.
template <int DT>
__device__ __forceinline__ void lay_eight(const char* row, int64_t c, int64_t width, bool vec, uint16_t* to, int64_t plane) {
  if constexpr (DT == MODA_HIP_FP32) {
    float v[8];
    const float* x = (const float*)row + c;
    if (vec && c + 8 <= width) {
      const f32x4 lo = *(const f32x4*)x, hi = *(const f32x4*)(x + 4);
#pragma unroll
      for (int i = 0; i < 4; i++) {
        v[i] = lo[i];
        v[4 + i] = hi[i];
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; i++) v[i] = c + i < width ? x[i] : 0.f;
    }
    uint16_t piece[8][3];
#pragma unroll
    for (int i = 0; i < 8; i++) three_pieces(v[i], piece[i]);
#pragma unroll
    for (int k = 0; k < 3; k++) {
      i32x4 w;
#pragma unroll
      for (int i = 0; i < 4; i++) w[i] = piece[2 * i][k] | piece[2 * i + 1][k] << 16;
      *(i32x4*)(to + k * plane + c) = w;
    }
  } else {
    const uint16_t* x = (const uint16_t*)row + c;
    i32x4 w = {0, 0, 0, 0};
    if (vec && c + 8 <= width) {
      w = *(const i32x4*)x;
    } else {
#pragma unroll
      for (int i = 0; i < 8; i++)
        if (c + i < width) w[i >> 1] |= (int)((uint32_t)x[i] << (16 * (i & 1)));
    }
    *(i32x4*)(to + c) = w;
  }
}

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

// A workgroup has kGatherBlock rows; it counts those with a target before them, and all, by itself.
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
  for (int64_t i = from + tid; i < upto; i += 256) {
    const bool live = a.words.of(i) >= 0;
    before += live && i < first;
    if (!a.counts && live) {
      all++;
      e = max(e, size_of(a, i));
    }
  }
  over_block(before, all, e);
  // The gradient of a logit is rounded to 16 bits.  The factor that rows share stays out of that, or its own rounding would be in all of them,
  // the same way: it is kept relative to the largest upstream gradient, which the products multiply by at their end.
  const float most = e > 0 ? __uint_as_float((uint32_t)e) : 1.f;
  if (first == 0 && tid == 0) *a.head = LossHead{all, a.d_loss ? most / (a.mean ? (float)max(all, 1) : 1.f) / a.up : 1.f};
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
  const int64_t chunks = a.rows_ld / 8, out_chunks = (a.width + 7) / 8;
  for (int64_t w = tid; w < kGatherBlock * chunks; w += 256) {
    const int r = (int)(w / chunks);
    const int64_t c = w - r * chunks, i = first + r;
    if (i >= n) break;
    if (to[r] >= 0) {
      lay_eight<DT>(a.x + i * a.ld_x * (DT == MODA_HIP_FP32 ? 4 : 2), c * 8, a.width, a.vec_x, a.rows + to[r] * a.rows_ld, a.rows_plane);
    } else if (a.dx && c < out_chunks) {
      char* row = a.dx + i * a.ld_dx * (DT == MODA_HIP_FP32 ? 4 : 2);
      const float zeros[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int h = 0; h < 2; h++) store_four<BF16, DT == MODA_HIP_FP32>(row, c * 8 + 4 * h, zeros, (int)min(a.width - c * 8 - 4 * h, (int64_t)4), a.vec_dx);
    }
  }
}

template <int DT>
__global__ __launch_bounds__(256) void lay_rows_kernel(const LayArgs a) {
  const int64_t chunks = a.to_ld / 8, w = (int64_t)workgroup() * 256 + threadIdx.x, r = w / chunks, c = w - r * chunks;
  if (r < a.rows) lay_eight<DT>(a.x + r * a.ld_x * (DT == MODA_HIP_FP32 ? 4 : 2), c * 8, a.width, a.vec, a.to + r * a.to_ld, a.to_plane);
}

// Sixteen lanes a row take every sixteenth tile of words each and meet in LDS, in a fixed order.
__global__ __launch_bounds__(256) void join_stats_kernel(const JoinStatsArgs a) {
  __shared__ float largest[16][17], sum[16][17];
  const int r = threadIdx.x & 15, part = threadIdx.x >> 4;
  const int rows = a.head ? a.head->live : (int)a.words.n;
  const int64_t p = (int64_t)workgroup() * 16 + r;
  float m = kNegInf, s = 0.f;
  if (p < rows)
    for (int64_t t = part; t < a.tiles; t += 16) {
      const float2 x = a.stats[t * a.stats_ld + p];
      if (x.x > m) {
        s = s * fast_exp2(m - x.x) + x.y;
        m = x.x;
      } else {
        s += x.x == kNegInf ? x.y : x.y * fast_exp2(x.x - m);  // (a sum of no logit above minus infinity is zero, or NaN)
      }
    }
  largest[part][r] = m;
  sum[part][r] = s;
  __syncthreads();
  if (part != 0 || p >= rows) return;
  for (int i = 1; i < 16; i++) m = fmaxf(m, largest[i][r]);
  s = 0.f;
  for (int i = 0; i < 16; i++) s += largest[i][r] == kNegInf ? sum[i][r] : sum[i][r] * fast_exp2(largest[i][r] - m);
  const float log_sum = log2f(s);
  float lse = m + log_sum;
  const int word = a.head ? 0 : a.words.of(p);
  float loss = (m - a.target_logit[p] + log_sum) * kLn2;  // (a target that is the likeliest word: log_sum alone, with all its bits)
  if (word < 0) lse = loss = 0.f;
  const int64_t row = a.head ? a.row_of[p] : p;
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
  const float* from = a.acc + p * a.acc_ld + f;
  f32x4 s = *(const f32x4*)from;
  for (int i = 1; i < a.splits; i++) s += *(const f32x4*)(from + i * a.acc_split);
  const float scale = a.scale * a.head->down;
  const float v[4] = {s[0] * scale, s[1] * scale, s[2] * scale, s[3] * scale};
  store_four<T, FP32_OUT>(a.out, (a.by_head ? a.row_of[p] : p) * a.out_ld + f, v, (int)min(a.width - f, (int64_t)4), a.out_vec);
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
  MODA_BY_TYPE(gather_rows_kernel, dtype, a.words.n > 0 ? (a.words.n + kGatherBlock - 1) / kGatherBlock : 1, a);  // (one, for the head)
  return hipGetLastError();
}
hipError_t launch_lay_rows(const LayArgs& a, int dtype, hipStream_t stream) {
  MODA_BY_TYPE(lay_rows_kernel, dtype, blocks_for(a.rows * (a.to_ld / 8)), a);
  return hipGetLastError();
}
hipError_t launch_stats(const ProductArgs& a, int dtype, ProductTile tile, hipStream_t stream) { return launch_product<kStats>(a, dtype, tile, stream); }
hipError_t launch_grad_logits(const ProductArgs& a, int dtype, ProductTile tile, hipStream_t stream) {
  return launch_product<kGradLogits>(a, dtype, tile, stream);
}
hipError_t launch_join_stats(const JoinStatsArgs& a, hipStream_t stream) {
  join_stats_kernel<<<grid_of((a.words.n + 15) / 16), 256, 0, stream>>>(a);
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
