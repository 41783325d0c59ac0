// Attention of new tokens over their sequence's pages of a key/value cache and over their own depth slots.
//
// Row (t, g) of sequence b sees positions j <= past[b] + t and slots l < Lv of its token:
//   s = scale <q, key>,  o = sum 2^(s - m) value / sum 2^(s - m),  lse = m + log2(sum)
// with the running maximum m and both sums in 32 bits.  A row that sees nothing has o = 0 and lse = -inf.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "paged.h"
#include "../../include/moda_hip.h"

namespace moda {

namespace {

__device__ __forceinline__ float load_as_float(const char* p, int64_t i, int dtype) {
  if (dtype == MODA_HIP_FP32) return ((const float*)p)[i];
  const uint16_t x = ((const uint16_t*)p)[i];
  return dtype == MODA_HIP_FP16 ? (float)__builtin_bit_cast(_Float16, x) : __uint_as_float((uint32_t)x << 16);
}

// One wave per query row and head, a lane every 64th element of the head.
__global__ __launch_bounds__(64) void paged_attend_kernel(const PagedAttendArgs a, int dtype) {
  const PagedKV& c = a.cache;
  const int lane = threadIdx.x;
  int64_t at = blockIdx.x;
  const int h = (int)(at % c.H);
  at /= c.H;
  const int g = (int)(at % a.G);
  at /= a.G;
  const int t = (int)(at % c.T), b = (int)(at / c.T);

  float q[4], o[4] = {0.f, 0.f, 0.f, 0.f}, m = -INFINITY, l = 0.f;
  const int64_t q0 = b * a.sq[0] + t * a.sq[1] + g * a.sq[2] + h * a.sq[3];
  for (int i = 0; i < 4; i++) q[i] = lane + 64 * i < a.D ? load_as_float(a.q, q0 + lane + 64 * i, dtype) : 0.f;
  auto see = [&](const char* kp, int64_t k0, const char* vp, int64_t v0) {
    float s = 0.f;
    for (int i = 0; i < 4; i++)
      if (lane + 64 * i < a.D) s += q[i] * load_as_float(kp, k0 + lane + 64 * i, dtype);
    for (int d = 32; d > 0; d >>= 1) s += __shfl_xor(s, d, 64);
    s *= a.scale;
    const float top = fmaxf(m, s), from = top == -INFINITY ? 0.f : top;
    const float shrink = exp2f(m - from), p = exp2f(s - from);
    m = top;
    l = l * shrink + p;
    for (int i = 0; i < 4; i++)
      if (lane + 64 * i < a.Dv) o[i] = o[i] * shrink + p * load_as_float(vp, v0 + lane + 64 * i, dtype);
  };
  if (t < c.new_of(b)) {
    const int end = min(c.past_of(b) + t + 1, c.capacity());
    for (int j = 0; j < end; j++) {
      const int page = c.page_of(b, j);
      if (page >= 0) see(c.k, c.offset(c.sk, page, j, h), c.v, c.offset(c.sv, page, j, h));
    }
    for (int s = 0; s < a.Lv; s++) {
      const int64_t row = (int64_t)t * a.L + s;
      see(a.kd, b * a.skd[0] + row * a.skd[1] + h * a.skd[2], a.vd, b * a.svd[0] + row * a.svd[1] + h * a.svd[2]);
    }
  }
  const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
  const int64_t o0 = b * a.so[0] + t * a.so[1] + g * a.so[2] + h * a.so[3];
  for (int i = 0; i < 4; i++)
    if (lane + 64 * i < a.Dv) {
      const float x = o[i] * inv;
      if (dtype == MODA_HIP_FP32)
        ((float*)a.o)[o0 + lane + 64 * i] = x;
      else
        ((uint16_t*)a.o)[o0 + lane + 64 * i] =
            dtype == MODA_HIP_FP16 ? __builtin_bit_cast(uint16_t, (_Float16)x) : __builtin_bit_cast(uint16_t, (__bf16)x);
    }
  if (lane == 0) a.lse[b * a.slse[0] + t * a.slse[1] + g * a.slse[2] + h * a.slse[3]] = l > 0.f || l != l ? m + log2f(l) : -INFINITY;
}

}  // namespace

hipError_t launch_paged_attend(const PagedAttendArgs& a, int dtype, hipStream_t stream) {
  const int64_t rows = (int64_t)a.cache.B * a.cache.T * a.G * a.cache.H;
  paged_attend_kernel<<<(unsigned)rows, 64, 0, stream>>>(a, dtype);
  return hipGetLastError();
}

}  // namespace moda
