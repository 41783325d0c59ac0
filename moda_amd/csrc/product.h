// The matrix products of the cross entropy over a vocabulary, out[p][f] = sum_k P(p, k) F(f, k), and what is done with a result before it
// leaves the registers:
//   kStats        logits (f: words, p: rows, k: columns): their largest and the sum of their exponentials a row, a target's own
//   kGradLogits   logits once more: their gradient, rounded to 16 bits (fp32: three of them)
//   kGradRows     f: columns, p: rows, k: words: the gradient of the rows
//   kGradWeight   f: columns, p: words, k: rows: the gradient of the weight
// An operand lies in memory either with k innermost (a tile of 64 k and as many rows as the result's tile has) or with f or p innermost
// (64 rows of k), and is read from LDS by row or transposed (tile16.h).  The transposed read takes k slots 0 .. 3 and 4 .. 7 of a lane from rows
// slot_base(q) and 16 + slot_base(q) on; the loader puts row k = 8 q + j there, so that both kinds of operand have k slot j of lane group q at
// k = 8 q + j.
//
// f sits on the matrix instruction's A side: a lane has four neighbouring f of one p.
//
// fp32 (PLANES): each operand as the sum of three bf16 (exact: 24 bits), of whose nine products the six largest are added up, the small
// ones first; the others are below 2^-24 of the whole.  Six products of 16 bits are faster than one of the fp32 matrix instruction.
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

// Rows of k of a tile whose columns are f or p: in LDS row r of a sixteen lies the k that the transposed read takes from there.
template <int COLS, int NT>
struct ColumnLoader {
  typedef AsyncTileLoader<COLS, 64, NT> Loader;
  static constexpr int N = Loader::N;
  static_assert(Loader::RPW * Loader::NW == 16, "a pass of the loads is sixteen rows");
  Loader l;
  int voff;
  __device__ __forceinline__ void init(int tid, int stride_bytes, int cols) {
    l.init(tid);
    const int r = l.row_in_pass, k = 8 * ((0x9C >> (2 * (r >> 2))) & 3) + (r & 3);  // slot_base(q) = 4 j  <=>  q = 0x9C >> 2 j
    voff = l.pads(cols) ? kPadOffset : k * stride_bytes + l.gchunk * 16;
  }
  // rows [k0, k0 + 64) of `rows`, at `base`
  __device__ __forceinline__ void load(lds_ptr tile, const uint16_t* base, int64_t ld, int k0, int rows) const {
    const int left = rows - k0 < 64 ? rows - k0 : 64, stride_bytes = (int)ld * 2;
    const i32x4 rs = rsrc_words(base + (int64_t)k0 * ld, left <= 0 ? 0u : (uint32_t)left * (uint32_t)stride_bytes);
#pragma unroll
    for (int i = 0; i < N; i++) lds_dma<16>(rs, lds_addr(tile + l.lds_elems(i)), voff, (32 * (i >> 1) + 4 * (i & 1)) * stride_bytes);
  }
};

// Rows of f or p, 64 k of each.
template <int ROWS, int NT>
struct RowLoader {
  typedef AsyncTileLoader<64, ROWS, NT> Loader;
  static constexpr int N = Loader::N;
  Loader l;
  int voff, rows_bytes;
  __device__ __forceinline__ void init(int tid, int stride_bytes, int rows) {  // rows from the tile's first on
    l.init(tid);
    voff = l.row_in_pass * stride_bytes + l.gchunk * 16;
    rows_bytes = (rows < ROWS ? (rows < 0 ? 0 : rows) : ROWS) * stride_bytes;
  }
  // columns [k0, k0 + 64) of `cols`, of the rows at `base`
  __device__ __forceinline__ void load(lds_ptr tile, const uint16_t* base, int64_t ld, int k0, int cols) const {
    const i32x4 rs = rsrc_words(base + k0, (uint32_t)rows_bytes);
    const int v = l.pads(cols - k0) ? kPadOffset : voff;
#pragma unroll
    for (int i = 0; i < N; i++) lds_dma<16>(rs, lds_addr(tile + l.lds_elems(i)), v, l.rows_before(i) * (int)ld * 2);
  }
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

// WF x WP waves share a tile of BF x BP, NST stages of LDS hold 64 k of both operands each.
template <typename T, int BF, int BP, int WF, int WP, int NST, Product PROD, bool PLANES>
__global__ __launch_bounds__(64 * WF * WP, 2) void product_kernel(const ProductArgs a) {
  constexpr int NT = 64 * WF * WP, MB = BF / WF / 16, NB = BP / WP / 16, DIST = NST - 1, STAGE = (BF + BP) * 64;
  constexpr bool FC = PROD == kGradRows || PROD == kGradWeight, PC = PROD == kGradWeight;  // operands with f or p innermost
  extern __shared__ __align__(16) unsigned char smem_raw[];
  lds_ptr smem = (lds_ptr)smem_raw;
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wf = wave % WF, wp = wave / WF;

  int p_count = a.p_count, k_count = a.k_count;
  float down = 1.f;
  if (a.head) {
    const int live = __builtin_amdgcn_readfirstlane(a.head->live);
    if (PROD == kGradWeight)
      k_count = live;
    else
      p_count = live;
    if (PROD == kGradRows || PROD == kGradWeight) down = a.head->down;
  }
  // Which tile: the workgroups of one XCD (every eighth) have neighbouring ones, in columns of eight tiles of p through all f.
  const int tiles_f = (a.f_count + BF - 1) / BF, tiles_p = (p_count + BP - 1) / BP;
  const int split = blockIdx.y;
  const int64_t tiles = (int64_t)tiles_f * tiles_p, of_xcd = (tiles + 7) / 8;
  const int64_t id = (int64_t)(blockIdx.x & 7) * of_xcd + (blockIdx.x >> 3);
  if ((int64_t)(blockIdx.x >> 3) >= of_xcd || id >= tiles) return;
  const int band = (int)(id / (8ll * tiles_f)), in_band = (int)(id - band * 8ll * tiles_f);
  const int band_p = tiles_p - 8 * band < 8 ? tiles_p - 8 * band : 8;
  const int f0 = in_band / band_p * BF, p0 = (8 * band + in_band % band_p) * BP;

  const int steps_all = (k_count + 63) / 64;
  const int first = (int)((int64_t)steps_all * split / a.splits), steps = (int)((int64_t)steps_all * (split + 1) / a.splits) - first;
  const int n_steps = PLANES ? 6 * steps : steps;

  OperandLoader<FC, BF, NT> lf;
  OperandLoader<PC, BP, NT> lp;
  lf.init(tid, (int)a.f_ld * 2, a.f_count - f0);
  lp.init(tid, (int)a.p_ld * 2, p_count - p0);
  const uint16_t* fb = a.f + (FC ? (int64_t)f0 : (int64_t)f0 * a.f_ld);
  const uint16_t* pb = a.p + (PC ? (int64_t)p0 : (int64_t)p0 * a.p_ld);

  int ld_st = 0, ld_pair = 0, ld_step = 0;
  auto issue = [&]() {
    lds_ptr fs = smem + ld_st * STAGE;
    const int k0 = (first + ld_step) * 64;
    lf.load(fs, fb + (PLANES ? plane_f(ld_pair) * a.f_plane : 0), a.f_ld, k0, k_count);
    lp.load(fs + BF * 64, pb + (PLANES ? plane_p(ld_pair) * a.p_plane : 0), a.p_ld, k0, k_count);
    ld_st = (ld_st + 1 == NST) ? 0 : ld_st + 1;
    if (++ld_step == steps && PLANES) {
      ld_step = 0;
      ld_pair++;
    }
  };
  constexpr int LOADS = decltype(lf)::N + decltype(lp)::N;
  typedef AsyncTileLoader<64, 64, 256> Wait;
  auto wait_tile = [&](int next) {  // the loads of step `next` have landed
    const int behind = n_steps - 1 - next;  // of later steps, up to DIST - 1 of which are on their way
    if (DIST >= 3 && behind >= 2)
      Wait::template wait_but<2 * LOADS <= 60 ? 2 * LOADS : 0>();
    else if (DIST >= 2 && behind >= 1)
      Wait::template wait_but<LOADS <= 60 ? LOADS : 0>();
    else
      Wait::wait_all();
  };

  TileOperand<FC, BF, MB> of;
  TileOperand<PC, BP, NB> op;
  of.init(lane, wf * MB);
  op.init(lane, wp * NB);
  f32x4 acc[MB][NB];
#pragma unroll
  for (int mb = 0; mb < MB; mb++)
#pragma unroll
    for (int nb = 0; nb < NB; nb++) acc[mb][nb] = f32x4{0.f, 0.f, 0.f, 0.f};

#pragma unroll
  for (int j = 0; j < DIST; j++)
    if (j < n_steps) issue();
  wait_tile(0);
  __syncthreads();
  int st = 0;
  for (int it = 0; it < n_steps; it++) {
    if (it + DIST < n_steps) issue();
    lds_cptr fs = smem + st * STAGE, ps = fs + BF * 64;
#pragma unroll
    for (int ks = 0; ks < 2; ks++) {
      i32x4 fo[MB], po[NB];
#pragma unroll
      for (int mb = 0; mb < MB; mb++) fo[mb] = of.read(fs, ks, mb);
#pragma unroll
      for (int nb = 0; nb < NB; nb++) po[nb] = op.read(ps, ks, nb);
#pragma unroll
      for (int nb = 0; nb < NB; nb++)
#pragma unroll
        for (int mb = 0; mb < MB; mb++) acc[mb][nb] = mfma16<T>(fo[mb], po[nb], acc[mb][nb]);
    }
    st = (st + 1 == NST) ? 0 : st + 1;
    wait_tile(it + 1);
    __syncthreads();
  }

  // four f from f_of(mb) on of p_of(nb)
  auto f_of = [&](int mb) { return f0 + (wf * MB + mb) * 16 + (FC ? 4 * q : slot_base(q)); };
  auto p_of = [&](int nb) { return p0 + (wp * NB + nb) * 16 + (PC ? n : slot_base(n >> 2) + (n & 3)); };

  if constexpr (PROD == kStats) {
    MODA_LDS float* part = (MODA_LDS float*)smem;  // [WF][BP] pairs
#pragma unroll
    for (int nb = 0; nb < NB; nb++) {
      const int p = p_of(nb);
      int target = p < p_count ? (a.head ? a.target[p] : a.words.of(p)) - a.first_word : -1;
      if (target >= a.f_count) target = -1;  // of a later piece
      float m = kNegInf;
#pragma unroll
      for (int mb = 0; mb < MB; mb++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const int f = f_of(mb) + i;
          const float z = f < a.f_count ? acc[mb][nb][i] * a.c : kNegInf;
          if (f == target) a.target_logit[p] = z;
          acc[mb][nb][i] = z;
          m = fmaxf(m, z);
        }
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
  }
  if constexpr (PROD == kGradLogits) {
#pragma unroll
    for (int nb = 0; nb < NB; nb++) {
      const int p = p_of(nb);
      const bool there = p < p_count;
      const int target = there ? a.target[p] - a.first_word : -1;
      const float factor = there ? a.factor[p] : 0.f, lse = there ? a.lse[p] : 0.f;
#pragma unroll
      for (int mb = 0; mb < MB; mb++) {
        const int f = f_of(mb);
        float v[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const float prob = fast_exp2(acc[mb][nb][i] * a.c - lse);
          v[i] = f + i < a.f_count ? factor * (prob - (f + i == target ? 1.f : 0.f)) : 0.f;
        }
        if (!there || f >= a.dz_ld) continue;
        uint16_t* to = a.dz + (int64_t)p * a.dz_ld + f;
        if (PLANES) {
          uint16_t piece[4][3];
#pragma unroll
          for (int i = 0; i < 4; i++) three_pieces(v[i], piece[i]);
#pragma unroll
          for (int k = 0; k < 3; k++)
            *(i32x2*)(to + k * a.dz_plane) = i32x2{piece[0][k] | piece[1][k] << 16, piece[2][k] | piece[3][k] << 16};
        } else {
          *(i32x2*)to = i32x2{pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3])};
        }
      }
    }
  }
  if constexpr (PROD == kGradRows || PROD == kGradWeight) {
    const float scale = a.scale * down;
#pragma unroll
    for (int nb = 0; nb < NB; nb++) {
      const int p = p_of(nb);
      if (p >= p_count) continue;
      const int64_t row = PROD == kGradRows && !a.acc ? a.row_of[p] : p;
#pragma unroll
      for (int mb = 0; mb < MB; mb++) {
        const int f = f_of(mb);
        if (f >= a.f_count) continue;
        if (a.acc) {
          f32x4* to = (f32x4*)(a.acc + split * a.acc_split + p * a.acc_ld + f);
          *to = a.add ? *to + acc[mb][nb] : acc[mb][nb];
        } else {
          const float v[4] = {acc[mb][nb][0] * scale, acc[mb][nb][1] * scale, acc[mb][nb][2] * scale, acc[mb][nb][3] * scale};
          store_four<T, PLANES>(a.out, row * a.out_ld + f, v, a.f_count - f, a.out_vec);
        }
      }
    }
  }
}

template <typename T, int BF, int BP, int WF, int WP, int NST, Product PROD, bool PLANES>
hipError_t launch_product_as(const ProductArgs& a, hipStream_t stream) {
  static LdsAttrState state;
  const auto kernel = &product_kernel<T, BF, BP, WF, WP, NST, PROD, PLANES>;
  const size_t lds = (size_t)NST * (BF + BP) * 128;
  hipError_t e = allow_dynamic_lds(state, (const void*)kernel, lds);
  if (e != hipSuccess) return e;
  const int64_t tiles = (int64_t)((a.f_count + BF - 1) / BF) * ((a.p_count + BP - 1) / BP), blocks = (tiles + 7) / 8 * 8;
  if (blocks == 0) return hipSuccess;
  if (blocks >= (1ll << 23)) return hipErrorInvalidValue;
  kernel<<<dim3((unsigned)blocks, (unsigned)a.splits), 64 * WF * WP, lds, stream>>>(a);
  return hipGetLastError();
}
template <Product PROD, typename T, bool PLANES>
hipError_t launch_product_of(const ProductArgs& a, ProductTile tile, hipStream_t stream) {
  if (tile == kTileLarge) return launch_product_as<T, 256, 256, 2, 4, 2, PROD, PLANES>(a, stream);
  if (tile == kTileMedium) return launch_product_as<T, 128, 128, 2, 2, 2, PROD, PLANES>(a, stream);
  if constexpr (PROD == kGradWeight)
    return hipErrorInvalidValue;  // (choose_tiling: its p are words)
  else
    return launch_product_as<T, 128, 32, 4, 1, 3, PROD, PLANES>(a, stream);
}
template <Product PROD>
hipError_t launch_product(const ProductArgs& a, int dtype, ProductTile tile, hipStream_t stream) {
  if (dtype == MODA_HIP_FP32) return launch_product_of<PROD, BF16, true>(a, tile, stream);
  if (dtype == MODA_HIP_FP16) return launch_product_of<PROD, FP16, false>(a, tile, stream);
  return launch_product_of<PROD, BF16, false>(a, tile, stream);
}

}  // namespace moda
