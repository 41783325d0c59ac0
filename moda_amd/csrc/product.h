// The matrix products of the cross entropy over a vocabulary, out[p][f] = sum_k P(p, k) F(f, k), and what is done with a result before it
// leaves the registers:
//   kStats        logits (f: words, p: rows, k: columns): their largest and the sum of their exponentials a row, a target's own
//   kGradLogits   logits once more: their gradient, rounded to 16 bits (fp32: three of them).  In the tensors' own type, so that the two products
//                 that read it are ones of 16 bits: in three pieces they would be three each.  8192 x 32000 x 2048, bf16: gradients 0.0019 from 64
//                 bits (norms), where the rounding of the results alone leaves 0.0017
//   kGradRows     f: columns, p: rows, k: words: the gradient of the rows
//   kGradWeight   f: columns, p: words, k: rows: the gradient of the weight
// An operand lies in memory either with k innermost (a tile of 64 k and as many rows as the result's tile has) or with f or p innermost
// (64 rows of k), and is read from LDS by row or transposed (tile16.h).  The transposed read takes k slots 0 .. 3 and 4 .. 7 of a lane from rows
// slot_base(q) and 16 + slot_base(q) on; the loader puts row k = 8 q + j there, so that both kinds of operand have k slot j of lane group q at
// k = 8 q + j.
//
// f sits on the matrix instruction's A side: a lane has four neighbouring f of one p.
//
// Bound by the matrix pipe at the clock that the power limit leaves: 8192 rows, 32000 words, width 2048, bf16: statistics 836 us (1284
// TFLOP/s), gradient of the logits 880, of the rows 804, of the weight 865, once the clock has settled (sixty passes in a row, the last twenty), the
// pipe busy 55 to 62 % of the cycles at 2.0 to 2.1 GHz; plain library products of these shapes 754, 754, 796 and 1104.  What it took (us of the four, one after the other): a workgroup for each tile, operands read
// and then multiplied 926, 1010, 822, 934; workgroups that stay, so that the first loads of a tile are on their way during the end of the one
// before; operands of the next half step read among the products of this one (861, 964, 836, 850: fewer cycles at a lower clock); the loads'
// addresses advanced on the scalar unit among the products and the loads sent right behind the barrier.  Stages of 32 k, four of them: 4 - 8 %
// slower (a barrier for half the products).  Without the tile loads at all the products took 595 to 727: what is left is there.
//
// fp32 (PLANES): each operand as the sum of three bf16 (exact: 24 bits), of whose nine products the six largest are added up, the small
// ones first; the others are below 2^-24 of the whole.  Six products of 16 bits at 1300 TFLOP/s are faster than one of the fp32 matrix
// instruction (150).  An infinite element is its own first piece, with zeros behind, and what it makes of the small products is no number; what it
// is worth, infinite or NaN, is the product of the first pieces, so that sums of small products that are not finite are dropped before that one.
#pragma once
#include "../../include/moda_hip.h"
#include "tile.h"
#include "tile16.h"
#include "vocab.h"

namespace moda {

enum Product { kStats, kGradLogits, kGradRows, kGradWeight };

// x as the sum of three bf16.  An x that is not finite has itself, NaN or infinite, as the first and zeros behind.
__device__ __forceinline__ void three_pieces(float x, uint16_t (&piece)[3]) {
  auto bits = [](float v) { return __builtin_bit_cast(uint16_t, (__bf16)v); };
  auto widen = [](uint16_t v) { return __builtin_bit_cast(float, (uint32_t)v << 16); };
  piece[0] = bits(x);
  const bool finite = fabsf(x) < __builtin_huge_valf();
  if (finite && (piece[0] & 0x7f80) == 0x7f80) piece[0]--;  // rounded past the largest: the largest
  const float rest = finite ? x - widen(piece[0]) : 0.f;
  piece[1] = bits(rest);
  piece[2] = bits(rest - widen(piece[1]));
}

// the planes of the i-th pair of an fp32 product, small ones first
__device__ __forceinline__ int plane_f(int i) { return (0x201100 >> (4 * (5 - i))) & 15; }
__device__ __forceinline__ int plane_p(int i) { return (0x021010 >> (4 * (5 - i))) & 15; }

__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// Rows of k of a tile whose columns are f or p: in LDS row r of a sixteen lies the k that the transposed read takes from there.
template <int COLS, int NT>
struct ColumnLoader {
  typedef AsyncTileLoader<COLS, 64, NT> Loader;
  static constexpr int N = Loader::N;
  static constexpr int PASS = Loader::RPW * Loader::NW;  // rows
  static_assert(PASS == 16 || PASS == 32, "sixteens of rows, the second of two with the four k behind");
  Loader l;
  i32x4 rs;
  int voff, stride;
  uint64_t at;   // of the next step's first row
  int64_t step;  // bytes
  __device__ __forceinline__ void begin(int tid, int64_t ld) {
    l.init(tid);
    stride = (int)ld * 2;
    step = 64 * (int64_t)stride;
  }
  // columns f0 .. of `cols`, rows from k0 on
  __device__ __forceinline__ void open(const uint16_t* p, int f0, int cols, int64_t ld, int k0) {
    const int r = l.row_in_pass, k = 8 * ((0x9C >> (2 * ((r >> 2) & 3))) & 3) + (r & 3) + 4 * (r >> 4);  // slot_base(q) = 4 j  <=>  q = 0x9C >> 2 j
    voff = l.pads(cols - f0) ? kPadOffset : k * stride + l.gchunk * 16;
    at = (uint64_t)(p + f0 + k0 * ld);
  }
  // the next 64 rows, of which `left` are there
  __device__ __forceinline__ void aim(int left) {
    rs = rsrc_words((const void*)at, (uint32_t)max(min(left, 64), 0) * (uint32_t)stride);
    at += step;
  }
  __device__ __forceinline__ void load(lds_ptr tile, int i) const {  // the i-th of a wave's N
    lds_dma<16>(rs, lds_addr(tile + l.lds_elems(i)), voff, (PASS == 32 ? 32 * i : 32 * (i >> 1) + 4 * (i & 1)) * stride);
  }
};

// Rows of f or p, 64 k of each.
template <int ROWS, int NT>
struct RowLoader {
  typedef AsyncTileLoader<64, ROWS, NT> Loader;
  static constexpr int N = Loader::N;
  Loader l;
  i32x4 rs;
  int voff, now, stride, bytes;
  uint64_t at;
  __device__ __forceinline__ void begin(int tid, int64_t ld) {
    l.init(tid);
    stride = (int)ld * 2;
    voff = l.row_in_pass * stride + l.gchunk * 16;
  }
  // rows f0 .. of `rows`, columns from k0 on
  __device__ __forceinline__ void open(const uint16_t* p, int f0, int rows, int64_t ld, int k0) {
    bytes = max(min(rows - f0, ROWS), 0) * stride;
    at = (uint64_t)(p + f0 * ld + k0);
  }
  // the next 64 columns, of which `left` are there
  __device__ __forceinline__ void aim(int left) {
    rs = rsrc_words((const void*)at, left > 0 ? (uint32_t)bytes : 0u);
    now = l.pads(left) ? kPadOffset : voff;
    at += 128;
  }
  __device__ __forceinline__ void load(lds_ptr tile, int i) const { lds_dma<16>(rs, lds_addr(tile + l.lds_elems(i)), now, l.rows_before(i) * stride); }
};

template <bool COLUMNS, int SIZE, int NT>
struct OperandLoader : RowLoader<SIZE, NT> {};
template <int SIZE, int NT>
struct OperandLoader<true, SIZE, NT> : ColumnLoader<SIZE, NT> {};

// A wave's MFMA operands from such a tile, by blocks of sixteen f or p from `first` on.
template <int SIZE, int BLOCKS>
struct RowOperand {
  Operand16<64> o;
  int first;
  __device__ __forceinline__ void init(int lane, int first_block) {
    o.init(lane);
    first = first_block * 16 * 64;
  }
  __device__ __forceinline__ i32x4 read(lds_cptr tile, int ks, int block) const { return o.row_operand(tile + first, block * 16, ks); }
};
template <int SIZE, int BLOCKS>
struct ColumnOperand {
  int at[BLOCKS];
  __device__ __forceinline__ void init(int lane, int first_block) {
    const int n = lane & 15, q = lane >> 4, r = slot_base(q) + (n >> 2);
#pragma unroll
    for (int b = 0; b < BLOCKS; b++) {
      const int col = 16 * (first_block + b) + 4 * (n & 3);
      at[b] = Tile<SIZE>::off(r, col >> 3) + (col & 7);
    }
  }
  __device__ __forceinline__ i32x4 read(lds_cptr tile, int ks, int block) const {
    const i32x2 lo = __builtin_bit_cast(i32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((MODA_LDS s16x4*)(tile + at[block] + 32 * ks * SIZE)));
    const i32x2 hi = __builtin_bit_cast(i32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((MODA_LDS s16x4*)(tile + at[block] + (32 * ks + 16) * SIZE)));
    return i32x4{lo[0], lo[1], hi[0], hi[1]};
  }
};
template <bool COLUMNS, int SIZE, int BLOCKS>
struct TileOperand : RowOperand<SIZE, BLOCKS> {};
template <int SIZE, int BLOCKS>
struct TileOperand<true, SIZE, BLOCKS> : ColumnOperand<SIZE, BLOCKS> {};

// four neighbouring results, rounded, n of them inside the row
template <typename T, bool FP32_OUT>
__device__ __forceinline__ void store_four(char* out, int64_t at, const float (&v)[4], int n, bool vec) {
  if (FP32_OUT) {
    float* o = (float*)out + at;
    if (vec && n >= 4) {
      *(f32x4*)o = f32x4{v[0], v[1], v[2], v[3]};
    } else {
#pragma unroll
      for (int i = 0; i < 4; i++)
        if (i < n) o[i] = v[i];
    }
  } else {
    uint16_t* o = (uint16_t*)out + at;
    const i32x2 w = {pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3])};
    if (vec && n >= 4) {
      *(i32x2*)o = w;
    } else {
#pragma unroll
      for (int i = 0; i < 4; i++)
        if (i < n) o[i] = (uint16_t)(w[i >> 1] >> (16 * (i & 1)));
    }
  }
}

// The results of two neighbouring blocks of sixteen f, four f a lane as they leave the matrix instruction, rounded -> eight neighbouring f a lane:
// those of block q >> 1 from 8 (q & 1) on.  A store then writes 64 bytes of a row, not 32 (8192 rows, 32000 words, forward and
// backward: 3.54 -> 3.49 ms).  COLUMNS: lane group q had f 4 q .., else slot_base(q) ..
template <bool COLUMNS>
__device__ __forceinline__ i32x4 eight_of(i32x2 a, i32x2 b, int q) {
  i32x4 r;
#if defined(__HIP_DEVICE_COMPILE__)
#pragma unroll
  for (int i = 0; i < 2; i++) {
    const auto half = __builtin_amdgcn_permlane32_swap(a[i], b[i], false, false);  // {a 0, a 1, b 0, b 1}, {a 2, a 3, b 2, b 3}
    if (COLUMNS) {
      const auto row = __builtin_amdgcn_permlane16_swap(half[0], half[1], false, false);  // {a 0, a 2, b 0, b 2}, {a 1, a 3, b 1, b 3}
      r[i] = row[0];
      r[2 + i] = row[1];
    } else {  // a 0 and a 3 are neighbours, a 1 and a 2
      const auto row = __builtin_amdgcn_permlane16_swap(half[1], half[1], false, false);
      r[i] = half[0];
      r[2 + i] = q & 1 ? row[0] : row[1];
    }
  }
#endif
  return r;
}

// What is done with a tile's result.  `part`: LDS of [WF][BP] pairs (kStats).
template <typename T, int BF, int BP, int WF, int WP, Product PROD, bool PLANES>
__device__ __forceinline__ void finish(const ProductArgs& a, f32x4 (&acc)[BF / WF / 16][BP / WP / 16], MODA_LDS float* part, int f0, int p0, int split,
                                       int64_t acc_split, int p_count, float down, int wf, int wp, int tid) {
  constexpr int NT = 64 * WF * WP, MB = BF / WF / 16, NB = BP / WP / 16;
  constexpr bool FC = PROD == kGradRows || PROD == kGradWeight, PC = PROD == kGradWeight;
  const int lane = tid & 63, n = lane & 15, q = lane >> 4;
  // four f from f_of(mb) on of p_of(nb)
  const int f_wave = f0 + wf * MB * 16;
  auto f_of = [&](int mb) { return f_wave + mb * 16 + (FC ? 4 * q : slot_base(q)); };
  auto p_of = [&](int nb) { return p0 + (wp * NB + nb) * 16 + (PC ? n : slot_base(n >> 2) + (n & 3)); };
  const bool last_f = f_wave + MB * 16 > a.f_count;  // some of the wave's f may be past the end

  if constexpr (PROD == kStats) {
#pragma unroll
    for (int nb = 0; nb < NB; nb++) {
      const int p = p_of(nb);
      int target = p < p_count ? (a.head ? a.target[p] : a.words.of(p)) - a.first_word : -1;
      if (target >= a.f_count) target = -1;  // of a later piece
#pragma unroll
      for (int mb = 0; mb < MB; mb++) acc[mb][nb] *= a.c;
      if (last_f) {
#pragma unroll
        for (int mb = 0; mb < MB; mb++)
#pragma unroll
          for (int i = 0; i < 4; i++)
            if (f_of(mb) + i >= a.f_count) acc[mb][nb][i] = kNegInf;
      }
      if (__any((unsigned)(target - f_wave) < (unsigned)(MB * 16))) {
#pragma unroll
        for (int mb = 0; mb < MB; mb++)
#pragma unroll
          for (int i = 0; i < 4; i++)
            if (f_of(mb) + i == target) a.target_logit[p] = acc[mb][nb][i];
      }
      float m = kNegInf;
#pragma unroll
      for (int mb = 0; mb < MB; mb++)
        m = fmaxf(fmaxf(fmaxf(m, acc[mb][nb][0]), acc[mb][nb][1]), fmaxf(acc[mb][nb][2], acc[mb][nb][3]));
      m = quad_max(m);
      const float ref = m == kNegInf ? 0.f : m;
      float s = 0.f;
#pragma unroll
      for (int mb = 0; mb < MB; mb++)
#pragma unroll
        for (int i = 0; i < 4; i++) s += fast_exp2(acc[mb][nb][i] - ref);
      s = quad_sum(s);
      if (q == 0) {
        const int at = wf * BP + p - p0;
        part[2 * at] = m;
        part[2 * at + 1] = s;
      }
    }
    __syncthreads();
    for (int r = tid; r < BP; r += NT) {
      if (p0 + r >= p_count) break;
      float m = kNegInf, s = 0.f;
#pragma unroll
      for (int w = 0; w < WF; w++) m = fmaxf(m, part[2 * (w * BP + r)]);
      const float ref = m == kNegInf ? 0.f : m;
#pragma unroll
      for (int w = 0; w < WF; w++) s += part[2 * (w * BP + r) + 1] * fast_exp2((part[2 * (w * BP + r)] == kNegInf ? ref : part[2 * (w * BP + r)]) - ref);
      a.stats[(int64_t)(f0 / BF) * a.stats_ld + p0 + r] = float2{m, s};
    }
    __syncthreads();  // (an item without steps brings no barrier of its own before `part` is written again)
  }
  if constexpr (PROD == kGradLogits) {
#pragma unroll
    for (int nb = 0; nb < NB; nb++) {
      const int p = p_of(nb);
      const bool there = p < p_count;
      const int target = there ? a.target[p] - a.first_word : -1;
      const float factor = there ? a.factor[p] : 0.f, lse = there ? a.lse[p] : 0.f;
#pragma unroll
      for (int mb = 0; mb < MB; mb++)
#pragma unroll
        for (int i = 0; i < 4; i++) acc[mb][nb][i] = fast_exp2(acc[mb][nb][i] * a.c - lse);
      if (__any((unsigned)(target - f_wave) < (unsigned)(MB * 16))) {
#pragma unroll
        for (int mb = 0; mb < MB; mb++)
#pragma unroll
          for (int i = 0; i < 4; i++) acc[mb][nb][i] -= f_of(mb) + i == target ? 1.f : 0.f;
      }
#pragma unroll
      for (int mb = 0; mb < MB; mb += 2) {
        i32x2 w[2][PLANES ? 3 : 1];
#pragma unroll
        for (int h = 0; h < 2; h++) {
          const int f = f_of(mb + h);
          float v[4];
#pragma unroll
          for (int i = 0; i < 4; i++) v[i] = last_f && f + i >= a.f_count ? 0.f : factor * acc[mb + h][nb][i];
          if constexpr (PLANES) {
            uint16_t piece[4][3];
#pragma unroll
            for (int i = 0; i < 4; i++) three_pieces(v[i], piece[i]);
#pragma unroll
            for (int k = 0; k < 3; k++) w[h][k] = i32x2{piece[0][k] | piece[1][k] << 16, piece[2][k] | piece[3][k] << 16};
          } else {
            w[h][0] = i32x2{pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3])};
          }
        }
        const int f = f_wave + (mb + (q >> 1)) * 16 + 8 * (q & 1);
        uint16_t* to = a.dz + (int64_t)p * a.dz_ld + f;
#pragma unroll
        for (int k = 0; k < (PLANES ? 3 : 1); k++) {
          const i32x4 x = eight_of<false>(w[0][k], w[1][k], q);
          if (there && f < a.dz_ld) *(i32x4*)(to + k * a.dz_plane) = x;
        }
      }
    }
  }
  if constexpr (PROD == kGradRows || PROD == kGradWeight) {
    const float scale = a.scale * down;
#pragma unroll
    for (int nb = 0; nb < NB; nb++) {
      const int p = p_of(nb);
      bool there = p < p_count;
      if (a.acc) {
#pragma unroll
        for (int mb = 0; mb < MB; mb++) {
          if (!there || f_of(mb) >= a.f_count) continue;
          f32x4* to = (f32x4*)(a.acc + split * acc_split + p * a.acc_ld + f_of(mb));
          *to = a.add ? *to + acc[mb][nb] : acc[mb][nb];
        }
        continue;
      }
      int r = p;
      if (PROD == kGradRows && there) {
        r = a.row_of[p];
        there = (unsigned)r < (unsigned)a.rows;  // (targets that change during the call make wrong results, no access out of place)
      }
      const int64_t row = r * a.out_ld;
#pragma unroll
      for (int mb = 0; mb < MB; mb++) acc[mb][nb] *= scale;
      if (!PLANES && a.out_by_eight) {
#pragma unroll
        for (int mb = 0; mb < MB; mb += 2) {
          const i32x2 w[2] = {{pack2<T>(acc[mb][nb][0], acc[mb][nb][1]), pack2<T>(acc[mb][nb][2], acc[mb][nb][3])},
                              {pack2<T>(acc[mb + 1][nb][0], acc[mb + 1][nb][1]), pack2<T>(acc[mb + 1][nb][2], acc[mb + 1][nb][3])}};
          const i32x4 x = eight_of<true>(w[0], w[1], q);
          const int f = f_wave + (mb + (q >> 1)) * 16 + 8 * (q & 1);
          if (there && f < a.f_count) *(i32x4*)(a.out + (row + f) * 2) = x;
        }
        continue;
      }
#pragma unroll
      for (int mb = 0; mb < MB; mb++) {
        const int f = f_of(mb);
        const float v[4] = {acc[mb][nb][0], acc[mb][nb][1], acc[mb][nb][2], acc[mb][nb][3]};
        if (there && f < a.f_count) store_four<T, PLANES>(a.out, row + f, v, a.f_count - f, a.out_vec);
      }
    }
  }
}

// WF x WP waves share a tile of BF x BP, NST stages of LDS hold 64 k of both operands each.  A workgroup stays and takes tile after tile (and
// part after part of a split summation axis), so that the first loads of the next are on their way while a result leaves the registers: a
// product of 32 steps otherwise spends a fifth of its time on starts and ends.
template <typename T, int BF, int BP, int WF, int WP, int NST, Product PROD, bool PLANES>
__global__ __launch_bounds__(64 * WF * WP, 2) void product_kernel(const ProductArgs a) {
  constexpr int NT = 64 * WF * WP, MB = BF / WF / 16, NB = BP / WP / 16, STAGE = (BF + BP) * 64;
  constexpr bool FC = PROD == kGradRows || PROD == kGradWeight, PC = PROD == kGradWeight;  // operands with f or p innermost
  extern __shared__ __align__(16) unsigned char smem_raw[];
  lds_ptr smem = (lds_ptr)smem_raw;
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wf = wave % WF, wp = wave / WF;

  int p_count = a.p_count, k_count = a.k_count, splits = a.splits;
  float down = 1.f;
  if (a.head) {
    const int live = __builtin_amdgcn_readfirstlane(a.head->live);
    if (PROD == kGradWeight)
      k_count = live;
    else
      p_count = live;
    if (PROD == kGradRows || PROD == kGradWeight) down = a.head->down;
    if (PROD == kGradRows && a.acc) splits = uniform(a.head->splits);
  }
  const int64_t acc_split = PROD == kGradRows ? p_count * a.acc_ld : a.acc_split;  // (sums of the live rows alone)
  // The workgroups of one XCD (every eighth) have neighbouring tiles at a time, of columns of eight tiles of p through all f.
  const int tiles_f = (a.f_count + BF - 1) / BF, tiles_p = (p_count + BP - 1) / BP, tiles = tiles_f * tiles_p;
  const int of_xcd = (tiles * splits + 7) >> 3, xcd = blockIdx.x & 7, at_once = gridDim.x >> 3;
  const int item_end = min((xcd + 1) * of_xcd, tiles * splits), item_first = xcd * of_xcd + (int)(blockIdx.x >> 3);
  if (item_first >= item_end) return;
  const int steps_all = (k_count + 63) >> 6, steps_of_split = splits == 1 ? steps_all : uniform(steps_all / splits);

  struct Item {
    int f0, p0, split, first, steps;  // of the summation axis: its first step and how many (for each pair of planes)
  };
  auto item_of = [&](int item) {
    Item t;
    t.split = splits == 1 ? 0 : uniform(item / tiles);
    const int id = item - t.split * tiles, band = uniform(id / (8 * tiles_f)), in_band = id - band * 8 * tiles_f;
    const int band_p = min(tiles_p - 8 * band, 8), f = uniform(in_band / band_p);
    t.f0 = f * BF;
    t.p0 = (8 * band + in_band - f * band_p) * BP;
    const int part = steps_of_split, more = steps_all - part * splits;  // the first `more` parts have a step more
    t.first = t.split * part + min(t.split, more);
    t.steps = part + (t.split < more);
    return t;
  };

  // the loads' side: NST steps ahead
  OperandLoader<FC, BF, NT> lf;
  OperandLoader<PC, BP, NT> lp;
  lf.begin(tid, a.f_ld);
  lp.begin(tid, a.p_ld);
  int ld_st = 0, ld_item = item_first - at_once, ld_pair = 5, ld_steps = 0, ld_left = 0;  // steps of the item (or pair of planes) to come, k that are there
  // The next step's loads are aimed; behind the last step at nothing, which fills their place with zeros: no branch in what is timed.
  auto aim = [&]() {
    while (ld_steps == 0 && ld_item < item_end) {  // (an item may have no steps at all)
      ld_pair++;
      if (!PLANES || ld_pair == 6) {
        ld_pair = 0;
        ld_item += at_once;
        if (ld_item >= item_end) break;
      }
      const Item t = item_of(ld_item);
      const int k0 = t.first * 64;
      lf.open(a.f + (PLANES ? plane_f(ld_pair) * a.f_plane : 0), t.f0, a.f_count, a.f_ld, k0);
      lp.open(a.p + (PLANES ? plane_p(ld_pair) * a.p_plane : 0), t.p0, p_count, a.p_ld, k0);
      ld_steps = t.steps;
      ld_left = k_count - k0;
    }
    if (ld_item >= item_end) ld_left = 0;
    lf.aim(ld_left);
    lp.aim(ld_left);
    ld_left -= 64;
    ld_steps--;
  };
  constexpr int LOADS_F = decltype(lf)::N, LOADS = LOADS_F + decltype(lp)::N;
  auto send = [&](int i) {
    lds_ptr to = smem + ld_st * STAGE;
    if (i < LOADS_F)
      lf.load(to, i);
    else
      lp.load(to + BF * 64, i - LOADS_F);
  };
  auto sent = [&]() { ld_st = (ld_st + 1 == NST) ? 0 : ld_st + 1; };
  typedef AsyncTileLoader<64, 64, 256> Wait;

  TileOperand<FC, BF, MB> of;
  TileOperand<PC, BP, NB> op;
  of.init(lane, wf * MB);
  op.init(lane, wp * NB);
  // A wave's operands of half a step (32 k), read from LDS while the products of the half before are on the matrix pipe: one read between two
  // products, in the order of use.
  struct Half {
    i32x4 f[MB], p[NB];
  };
  auto read = [&](Half& h, lds_cptr tile, int ks, int i) {
    if (i == 0)
      h.p[0] = op.read(tile + BF * 64, ks, 0);
    else if (i <= MB)
      h.f[i - 1] = of.read(tile, ks, i - 1);
    else
      h.p[i - MB] = op.read(tile + BF * 64, ks, i - MB);
  };
  constexpr int READS = MB + NB, PRODUCTS = MB * NB, APART = PRODUCTS / READS > 2 ? 2 : 1, APART2 = PRODUCTS >= 2 * LOADS ? 2 : 1;
  f32x4 acc[MB][NB];
  // products of `now`, reads of `next` among them, and `others(j)` behind the j-th product
  auto half_step = [&](const Half& now, Half& next, lds_cptr tile, int ks, auto others) {
#pragma unroll
    for (int j = 0; j < PRODUCTS; j++) {
      if (j % APART == 0 && j / APART < READS) read(next, tile, ks, j / APART);
      if (j == PRODUCTS - 1)
#pragma unroll
        for (int i = (PRODUCTS + APART - 1) / APART; i < READS; i++) read(next, tile, ks, i);
      acc[j % MB][j / MB] = mfma16<T>(now.f[j % MB], now.p[j / MB], acc[j % MB][j / MB]);
      __builtin_amdgcn_sched_barrier(0);
      others(j);
    }
  };

#pragma unroll 1  // (code that runs once comes from memory)
  for (int j = 0; j < NST; j++) {
    aim();
#pragma unroll
    for (int i = 0; i < LOADS; i++) send(i);
    sent();
  }
  Wait::wait_all();
  __syncthreads();
  int st = 0;
  Half h0, h1;
#pragma unroll
  for (int i = 0; i < READS; i++) read(h0, smem, 0, i);
  for (int item = item_first; item < item_end; item += at_once) {
    const Item t = item_of(item);
    const int n_steps = PLANES ? 6 * t.steps : t.steps;
#pragma unroll
    for (int mb = 0; mb < MB; mb++)
#pragma unroll
      for (int nb = 0; nb < NB; nb++) acc[mb][nb] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int it = 0; it < n_steps; it++) {
      lds_cptr tile = smem + st * STAGE;
      if (PLANES && it == 5 * t.steps) {  // the first pieces are next
#pragma unroll
        for (int mb = 0; mb < MB; mb++)
#pragma unroll
          for (int nb = 0; nb < NB; nb++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
              const float small = acc[mb][nb][i];
              acc[mb][nb][i] = fabsf(small) < __builtin_huge_valf() ? small : 0.f;
            }
      }
      half_step(h0, h1, tile, 1, [&](int j) {
        if (j == PRODUCTS * 3 / 4) aim();
      });
      st = (st + 1 == NST) ? 0 : st + 1;
      // the loads of the next step have landed (of those behind it too where stores of the result before are counted with them)
      if (NST > 2 && it > 0)
        Wait::template wait_but<(NST - 2) * LOADS>();
      else
        Wait::wait_all();
      __syncthreads();  // every wave has read this step's tile, whose place the loads may have now, and sees the next one
      lds_cptr next = smem + st * STAGE;  // (behind the last step: what is there, for nothing)
      half_step(h1, h0, next, 0, [&](int j) {  // the loads: as early as may be
#pragma unroll
        for (int i = 0; i < LOADS; i++)
          if (j == (i * APART2 < PRODUCTS ? i * APART2 : PRODUCTS - 1)) send(i);
        __builtin_amdgcn_sched_barrier(0);
      });
      sent();
    }
    finish<T, BF, BP, WF, WP, PROD, PLANES>(a, acc, (MODA_LDS float*)(smem + NST * STAGE), t.f0, t.p0, t.split, acc_split, p_count, down, wf, wp, tid);
  }
  Wait::wait_all();  // no load outlives its workgroup's LDS
}

template <typename T, int BF, int BP, int WF, int WP, int NST, Product PROD, bool PLANES>
hipError_t launch_product_as(const ProductArgs& a, int compute_units, hipStream_t stream) {
  static LdsAttrState state;
  const auto kernel = &product_kernel<T, BF, BP, WF, WP, NST, PROD, PLANES>;
  const size_t lds = (size_t)NST * (BF + BP) * 128 + (PROD == kStats ? WF * BP * 8 : 0);
  hipError_t e = allow_dynamic_lds(state, (const void*)kernel, lds);
  if (e != hipSuccess) return e;
  const int64_t tiles = (int64_t)((a.f_count + BF - 1) / BF) * ((a.p_count + BP - 1) / BP) * a.splits;
  if (tiles == 0) return hipSuccess;
  if (tiles >= (1ll << 28)) return hipErrorInvalidValue;
  const int64_t room = (int64_t)compute_units * (160 * 1024 / lds < 1 ? 1 : 160 * 1024 / lds) / 8 * 8, blocks = (tiles + 7) / 8 * 8;
  kernel<<<(unsigned)(blocks < room || room == 0 ? blocks : room), 64 * WF * WP, lds, stream>>>(a);
  return hipGetLastError();
}
template <Product PROD, typename T, bool PLANES>
hipError_t launch_product_of(const ProductArgs& a, ProductTile tile, int compute_units, hipStream_t stream) {
  if (tile == kTileLarge) return launch_product_as<T, 256, 256, 2, 4, 2, PROD, PLANES>(a, compute_units, stream);
  if (tile == kTileMedium) return launch_product_as<T, 128, 128, 2, 2, 2, PROD, PLANES>(a, compute_units, stream);
  if (tile == kTileSmall) return launch_product_as<T, 64, 64, 2, 2, 3, PROD, PLANES>(a, compute_units, stream);
  if constexpr (PROD == kGradWeight)
    return hipErrorInvalidValue;  // (choose_tiling: its p are words)
  else
    return launch_product_as<T, 128, 32, 4, 1, 3, PROD, PLANES>(a, compute_units, stream);
}
template <Product PROD>
hipError_t launch_product(const ProductArgs& a, int dtype, ProductTile tile, int compute_units, hipStream_t stream) {
  if (dtype == MODA_HIP_FP32) return launch_product_of<PROD, BF16, true>(a, tile, compute_units, stream);
  if (dtype == MODA_HIP_FP16) return launch_product_of<PROD, FP16, false>(a, tile, compute_units, stream);
  return launch_product_of<PROD, BF16, false>(a, tile, compute_units, stream);
}

}  // namespace moda
