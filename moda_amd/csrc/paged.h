// Argument blocks of the rotation of rows by their position, of appending to a paged key/value cache and of the attention
// that reads it, and where a position of a sequence lies in such a cache.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace moda {

// Pages [n_pages][2^page_shift tokens][heads][dim] of keys and values (strides in elements), the table of every sequence's
// pages, and how many tokens are there.  Nothing of what the device arrays hold is known to the host: counts are bounded
// and page numbers checked where they are read.
struct PagedKV {
  char *k, *v;
  int64_t sk[3], sv[3];  // page, token in the page, head
  const int32_t* table;
  int64_t table_stride;
  const int32_t* past;      // tokens of each sequence before the call
  const int32_t* new_lens;  // new tokens of each sequence, or NULL: T
  const int32_t* cu;        // packed new tokens: offsets, or NULL
  int B, T, H;
  int n_pages, page_shift, max_pages;

  __device__ __forceinline__ int past_of(int b) const { return min(max(past[b], 0), capacity()); }
  __device__ __forceinline__ int new_of(int b) const { return new_lens ? min(max(new_lens[b], 0), T) : T; }
  __device__ __forceinline__ int capacity() const { return max_pages << page_shift; }
  // page of position `pos` < capacity(), or -1: a number outside the cache names no page
  __device__ __forceinline__ int page_of(int b, int pos) const {
    const int p = table[b * table_stride + (pos >> page_shift)];
    return (unsigned)p < (unsigned)n_pages ? p : -1;
  }
  __device__ __forceinline__ int64_t offset(const int64_t (&s)[3], int page, int pos, int head) const {
    return page * s[0] + (pos & ((1 << page_shift) - 1)) * s[1] + head * s[2];
  }
};

// One tensor of a launch that rotates or copies rows: its rows [batch][token * rows + r][head] go to y, to the cache or both
// to the cache and to a depth slot.
struct RowPart {
  const char* x;
  char* y;                // NULL: the pages (and depth, unless NULL)
  char* depth;
  int64_t sx[3], sy[3], sd[3];  // batch, row, head
  int rows, heads, dim;
  unsigned heads_magic;   // item / heads = umulhi(item, heads_magic); 0: heads is 1
  int rotated;            // whether the first `rot` elements are rotated (else copied)
  int values;             // of the cache: its v (else its k)
};

struct RowArgs {
  RowPart part[3];
  int n_parts, items;  // rows * heads of all parts
  int64_t tokens;      // B * T, or the packed axis
  int T;
  // rotation: turns per position of each pair, position of each token
  const double* rates;
  int rot;
  float amplitude, sign;
  const void* positions;  // NULL: 0, 1, .. (of a cache: past, past + 1, ..)
  int64_t position_stride;
  int positions64;
  // destination
  PagedKV cache;
  int L, slot;
  // launch
  int lane_shift, groups;  // 2^lane_shift lanes share a token's heads with groups - 1 others
};

struct PagedAttendArgs {
  PagedKV cache;
  const char *q, *kd, *vd;
  char* o;
  float* lse;
  int64_t sq[4], so[4];    // batch, token, row of the group, head
  int64_t skd[3], svd[3];  // batch, row, head
  int64_t slse[4];
  int G, D, Dv, L, Lv;
  float scale;  // of logits in base 2
  float* work;
  // how the work is cut (plan_paged_attend)
  int waves, row_tiles, part_rows, part_width;
  int slot_blocks;  // sixteens of a token's depth slots
  float blocks_inverse;
  unsigned group_magic;
};

// A launch of n workgroups: an axis has less than 2^32 threads, so the second one counts runs of 2^20 (a constant, so that kernels need not load
// the launch's shape).  The last run may reach past n.
constexpr unsigned kGridRun = 1 << 20;
inline dim3 grid_of(int64_t n) { return dim3((unsigned)(n < kGridRun ? n : kGridRun), (unsigned)((n + kGridRun - 1) / kGridRun)); }
__device__ __forceinline__ unsigned workgroup() { return blockIdx.y * kGridRun + blockIdx.x; }

}  // namespace moda
