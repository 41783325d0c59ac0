// Rows of query and key heads rotated by their token's position, and the same on the way into a paged cache.
//
// Pair i of a row at position p turns by the angle 2 pi frac(p * rate_i): product and fraction in 64 bits (a position of
// 10^6 leaves 32-bit angles with four correct digits), sine and cosine of the rest in 32 bits, once for all heads that
// a thread has of its token.  y0 = A (x0 cos - x1 sin), y1 = A (x0 sin + x1 cos); the gradient of x is the rotation of
// the gradient of y by the opposite angle, so the backward pass is this kernel with the other sign.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "paged.h"
#include "../../include/moda_hip.h"

namespace moda {

struct Bf16 {
  typedef uint16_t bits;
  __device__ static float widen(bits x) { return __uint_as_float((uint32_t)x << 16); }
  __device__ static bits narrow(float x) { return __builtin_bit_cast(uint16_t, (__bf16)x); }
};
struct Fp16 {
  typedef uint16_t bits;
  __device__ static float widen(bits x) { return (float)__builtin_bit_cast(_Float16, x); }
  __device__ static bits narrow(float x) { return __builtin_bit_cast(uint16_t, (_Float16)x); }
};
struct Fp32 {
  typedef uint32_t bits;
  __device__ static float widen(bits x) { return __uint_as_float(x); }
  __device__ static bits narrow(float x) { return __float_as_uint(x); }
};

// sequence of token n of a packed axis (B: behind the last one); any offsets at all leave it within 0 .. B
__device__ __forceinline__ int sequence_of(const int32_t* cu, int B, int64_t n) {
  int lo = 0, hi = B;  // cu[lo] <= n < cu[hi], hi = B standing for any
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid + 1] <= n)
      lo = mid + 1;
    else
      hi = mid;
  }
  return lo;
}

// A thread has chunk c of VEC pairs (or, past the rotated elements, of VEC elements) of every `groups`-th (row, head) item of
// one token.  VEC elements are 16 bytes, or one where rows do not lie on that grid.  STREAM: nontemporal accesses.
//
// Bound by the bytes: 64 K tokens of 16 + 4 heads of 128 (671 MB in and out) take 114 us, 5.9 TB/s, where a copy of 4 GiB
// reaches 4.7.  Small calls by loads that are sent one after the other, counts, page, rates and last the rows, which need none of
// them: 4.4 us for one token, 5.5 into a cache.
template <typename E, int VEC, bool INTER, bool PAGED, bool STREAM>
__global__ __launch_bounds__(256) void rows_kernel(const RowArgs a) {
  typedef typename E::bits bits;
  typedef bits vec __attribute__((ext_vector_type(VEC)));
  auto get = [](const bits* p) { return STREAM ? __builtin_nontemporal_load((const vec*)p) : *(const vec*)p; };
  auto put = [](vec x, bits* p) {
    if (STREAM)
      __builtin_nontemporal_store(x, (vec*)p);
    else
      *(vec*)p = x;
  };
  const int64_t id = (int64_t)workgroup() * 256 + threadIdx.x, unit = id >> a.lane_shift;
  const int c0 = (int)(id & ((1 << a.lane_shift) - 1));
  const int64_t n = unit / a.groups;
  if (n >= a.tokens) return;
  const int group = (int)(unit - n * a.groups);

  int64_t tb = n / a.T, tt = n - tb * a.T;  // batch and token of the tensors
  int64_t pos = tt;
  int page = -1, b = (int)tb;
  bool turn = true, stored = false;  // whether the token is of a sequence; whether it goes to the cache
  if (PAGED) {
    if (a.cache.cu) {
      b = sequence_of(a.cache.cu, a.cache.B, n);
      pos = b < a.cache.B ? n - a.cache.cu[b] : -1;
      turn = pos >= 0;  // (below zero: before the first sequence, or offsets out of order)
      stored = turn;
    } else {
      stored = tt < a.cache.new_of(b);
    }
    if (!turn) {  // a token of no sequence: q as it is, infinities and signs of zero with it
      for (int p = 0; p < a.n_parts; p++) {
        const RowPart& part = a.part[p];
        if (!part.y) continue;
        for (int item = group; item < part.rows * part.heads; item += a.groups) {
          const int r = part.heads_magic ? (int)__umulhi((unsigned)item, part.heads_magic) : item, h = item - r * part.heads;
          const bits* x = (const bits*)part.x + tb * part.sx[0] + (tt * part.rows + r) * part.sx[1] + h * part.sx[2];
          bits* y = (bits*)part.y + tb * part.sy[0] + (tt * part.rows + r) * part.sy[1] + h * part.sy[2];
          for (int e = c0 * VEC; e < part.dim; e += VEC << a.lane_shift) put(get(x + e), y + e);
        }
      }
      return;
    }
    pos += a.cache.past_of(b);
    if (stored && pos < a.cache.capacity()) page = a.cache.page_of(b, (int)pos);
  } else if (a.positions) {
    const int64_t at = tb * a.position_stride + tt;
    pos = a.positions64 ? ((const int64_t*)a.positions)[at] : ((const int32_t*)a.positions)[at];
  }

  const int n_rot = a.rot / (2 * VEC);
  float cs[VEC], sn[VEC];
  if (c0 < n_rot) {
#pragma unroll
    for (int i = 0; i < VEC; i++) {
      const double t = (double)pos * a.rates[c0 * VEC + i];
      float s, c;
      sincospif(2.f * (float)(t - rint(t)), &s, &c);
      cs[i] = c * a.amplitude;
      sn[i] = s * a.amplitude * a.sign;
    }
  }

  int first = 0;
  for (int p = 0; p < a.n_parts; p++) {
    const RowPart& part = a.part[p];
    const int count = part.rows * part.heads, rot = part.rotated ? n_rot : 0, rot_elems = rot * 2 * VEC;
    const int chunks = rot + (part.dim - rot_elems) / VEC;
    const bits* x = (const bits*)part.x + tb * part.sx[0] + tt * part.rows * part.sx[1];
    bits *y = nullptr, *depth = nullptr;
    if (part.y) {
      y = (bits*)part.y + tb * part.sy[0] + tt * part.rows * part.sy[1];
    } else if (PAGED) {
      if (page >= 0)
        y = part.values ? (bits*)a.cache.v + a.cache.offset(a.cache.sv, page, (int)pos, 0)
                        : (bits*)a.cache.k + a.cache.offset(a.cache.sk, page, (int)pos, 0);
      if (part.depth && stored) depth = (bits*)part.depth + tb * part.sd[0] + (tt * a.L + a.slot) * part.sd[1];
    }
    const int64_t y_head = part.y ? part.sy[2] : part.values ? a.cache.sv[2] : a.cache.sk[2];
    // the items of all parts are dealt out in turn: a part goes on where the one before it stopped
    int item = group - first % a.groups;
    if (item < 0) item += a.groups;
    first += count;
    if (!y && !depth) continue;
    for (; item < count; item += a.groups) {
      const int r = part.heads_magic ? (int)__umulhi((unsigned)item, part.heads_magic) : item, h = item - r * part.heads;
      const bits* xr = x + r * part.sx[1] + h * part.sx[2];
      bits* yr = y + (part.y ? r * part.sy[1] : 0) + h * y_head;
      bits* dr = depth + h * part.sd[2];
      for (int c = c0; c < chunks; c += 1 << a.lane_shift) {
        if (c < rot) {
          const int e0 = INTER ? 2 * c * VEC : c * VEC, e1 = INTER ? e0 + VEC : a.rot / 2 + e0;
          const vec u = get(xr + e0), v = get(xr + e1);
          vec yu, yv;
#pragma unroll
          for (int i = 0; i < VEC; i++) {
            // interleaved: pair i is elements 2i, 2i + 1 of the two vectors together
            const float x0 = E::widen(!INTER ? u[i] : 2 * i < VEC ? u[2 * i % VEC] : v[2 * i % VEC]);
            const float x1 = E::widen(!INTER ? v[i] : 2 * i + 1 < VEC ? u[(2 * i + 1) % VEC] : v[(2 * i + 1) % VEC]);
            const bits y0 = E::narrow(x0 * cs[i] - x1 * sn[i]), y1 = E::narrow(x0 * sn[i] + x1 * cs[i]);
            if (!INTER) {
              yu[i] = y0;
              yv[i] = y1;
            } else {
              (2 * i < VEC ? yu : yv)[2 * i % VEC] = y0;
              (2 * i + 1 < VEC ? yu : yv)[(2 * i + 1) % VEC] = y1;
            }
          }
          if (y) {
            put(yu, yr + e0);
            put(yv, yr + e1);
          }
          if (PAGED && depth) {
            put(yu, dr + e0);
            put(yv, dr + e1);
          }
        } else {
          const int e = rot_elems + (c - rot) * VEC;
          const vec u = get(xr + e);
          if (y) put(u, yr + e);
          if (PAGED && depth) put(u, dr + e);
        }
      }
    }
  }
}

template <typename E, int VEC, bool PAGED>
static void launch_rows_as(const RowArgs& a, bool inter, bool stream_through, int64_t blocks, hipStream_t stream) {
  const dim3 grid = grid_of(blocks);
  if (VEC > 1 && stream_through) {
    inter ? rows_kernel<E, VEC, true, PAGED, VEC != 1><<<grid, 256, 0, stream>>>(a) : rows_kernel<E, VEC, false, PAGED, VEC != 1><<<grid, 256, 0, stream>>>(a);
    return;
  }
  inter ? rows_kernel<E, VEC, true, PAGED, false><<<grid, 256, 0, stream>>>(a) : rows_kernel<E, VEC, false, PAGED, false><<<grid, 256, 0, stream>>>(a);
}

// `vec`: all rows lie on the 16-byte grid and the rotated elements are whole vectors of pairs
hipError_t launch_rows(RowArgs& a, int dtype, bool vec, bool inter, bool paged, hipStream_t stream) {
  const int v = !vec ? 1 : dtype == MODA_HIP_FP32 ? 4 : 8;
  int most = 1;
  int64_t bytes = 0;  // in and out, of a token
  a.items = 0;
  for (int p = 0; p < a.n_parts; p++) {
    RowPart& part = a.part[p];
    const int rot = part.rotated ? a.rot / (2 * v) : 0, chunks = rot + (part.dim - 2 * rot * v) / v;
    most = max(most, part.rotated ? chunks : (chunks + 1) / 2);  // copies: two chunks a thread, as many bytes as a rotated one
    part.heads_magic = part.heads == 1 ? 0 : (unsigned)((1ull << 32) / part.heads) + 1;
    a.items += part.rows * part.heads;
    bytes += 2ll * part.rows * part.heads * part.dim * (dtype == MODA_HIP_FP32 ? 4 : 2);
  }
  a.lane_shift = 0;
  while ((1 << a.lane_shift) < most && a.lane_shift < 8) a.lane_shift++;
  // One item a thread until there are two waves a SIMD, then up to five, which share the angles.  With up to 3, 4, 5, 8 and 10 items a thread,
  // 64 K tokens, bf16: 16 items of 128 elements 89, 92, 92, 98, 98 us; 20: 111, 112, 112, 118, 125; 40: 220, 218, 219, 226, 232; 72 of 64
  // elements 238, 241, 246, 248, 244; fp32: 40 items 443, 455, 465, 471, 482.  4 K tokens, bf16: 20 items 10.8, 10.5, 10.4, 10.4, 10.5; 40: 16.9,
  // 16.5, 16.2, 17.0, 18.4.  Below nine items it makes no difference.
  const int64_t full = 256 * 512, lanes = a.tokens << a.lane_shift;
  a.groups = (int)max((int64_t)(a.items + 4) / 5, min((int64_t)a.items, full / max(lanes, (int64_t)1)));
  // What does not fit the 256 MB memory-side cache passes it by (115 us instead of 126); what does is found there by whoever reads it next.
  const bool stream_through = a.tokens * bytes > 256ll << 20;
  const int64_t blocks = (lanes * a.groups + 255) / 256;
  if (blocks >= (1ll << 31)) return hipErrorInvalidValue;
#define MODA_ROWS(E, V) paged ? launch_rows_as<E, V, true>(a, inter, stream_through, blocks, stream) : launch_rows_as<E, V, false>(a, inter, stream_through, blocks, stream)
  if (dtype == MODA_HIP_FP32)
    vec ? (MODA_ROWS(Fp32, 4)) : (MODA_ROWS(Fp32, 1));
  else if (dtype == MODA_HIP_FP16)
    vec ? (MODA_ROWS(Fp16, 8)) : (MODA_ROWS(Fp16, 1));
  else
    vec ? (MODA_ROWS(Bf16, 8)) : (MODA_ROWS(Bf16, 1));
#undef MODA_ROWS
  return hipGetLastError();
}

}  // namespace moda
