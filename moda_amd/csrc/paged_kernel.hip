// Attention of new tokens over their sequence's pages of a key/value cache and over their own depth slots.
//
// Row (t, g) of sequence b sees positions j <= past[b] + t and slots l < Lv of its token:
//   s = scale <q, key>,  o = sum 2^(s - m) value / sum 2^(s - m),  lse = m + log2(sum)
// in one pass over keys and values with the running maximum m, the sum and o in 32 bits.  A row that sees nothing has
// o = 0 and lse = -inf.
//
// What bounds it is the stream of keys and values from HBM: each is read once for 16 (32) rows of its key/value head, four rows
// make 4 FLOP of a byte, the matrix instruction does a hundred times that.  So the work is cut for the stream alone.  All
// tiles of 32 keys -- of every sequence, key/value head and 16 (32) rows of the call, whether or not the sequence has new tokens
// in them -- stand on one axis, sequences with
// their lengths as they are on the device; each of a fixed number of waves, as many as keep the card's loads in flight, takes an equal
// run of it, whatever the lengths are, and the host needs to know none of them (a captured launch follows them as they grow).
// A wave is a workgroup by itself: it fetches its tiles into a ring of its own and waits for nobody.  Runs that begin or end
// inside a segment (one sequence, head and row tile) leave maximum, sum and o in the workspace, at most two of them a
// wave; a second launch joins them in the order of the axis, so that results do not depend on who came first.
//
// Measured (bf16, head dim 128, four rows a head; a copy of 4 GiB reaches 4.7 TB/s in and out, reading alone more): 256 sequences
// of 12 - 24 K tokens, 4 heads (9.4 GB) 1.59 ms, 5.9 TB/s; one sequence of 1 M tokens 359 us + 8 for joining, 6.0 TB/s; 64 of 1 - 8 K
// 117 + 5.4 us, 5.2 TB/s; one of 101 tokens 6.6 + 4.4 us, the chain counts -> table -> rows -> keys -> products and a second
// launch.  More than 16 rows a head are bound by the vector instructions of a wave's tile (some 500), and by the tiles of rows that are
// not there: five drafted tokens of eight rows, two row tiles, of sequences that have up to five, 34 + 6 us, 36 % of the tiles for
// padded tokens alone.
#include "paged.h"
#include "tile16.h"
#include "../../include/moda_hip.h"

namespace moda {

namespace {

constexpr int kTileKeys = 32;

// what invalid rows and chunks past a head dim read
__device__ __align__(64) uint32_t zero_line[16];

// The kernel's arguments, read again where they are used: kept from the start they take every scalar register there is, and the main
// loop's own move to vector lanes and back.  (They begin the kernel's argument segment, which only a kernel knows: in a function that is
// called, not inlined, its address is zero.  Whoever calls this is forced inline.)
__device__ __forceinline__ PagedAttendArgs reload() {
  PagedAttendArgs a;
#if defined(__HIP_DEVICE_COMPILE__)
  auto p = __builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  __builtin_memcpy(&a, (const void*)p, sizeof(a));
#endif
  return a;
}

// Sum over lanes 0 .. l in lane l.
__device__ __forceinline__ int wave_scan(int x) {
#if defined(__HIP_DEVICE_COMPILE__)
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // row_shr:1, 2, 4, 8: within 16 lanes
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // row_bcast:15 to rows 1 and 3
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // row_bcast:31 to rows 2 and 3
#endif
  return x;
}

// Pointers out of the argument block are global memory; read from a copy of it the compiler does not know.
template <typename V>
__device__ __forceinline__ const __attribute__((address_space(1))) V* in_global(const void* p) {
  return (const __attribute__((address_space(1))) V*)(uint64_t)p;
}
template <typename V>
__device__ __forceinline__ __attribute__((address_space(1))) V* out_global(void* p) {
  return (__attribute__((address_space(1))) V*)(uint64_t)p;
}

// Sequence b on the axis: positions that its last new token sees, tiles of them and of its new tokens' depth slots.  The slots of
// a token begin a sixteen of their own: slot l of token t has index 16 blocks t + l.
struct Seq {
  int past, fresh, len, seq_tiles, tiles;
  __device__ __forceinline__ Seq(const PagedAttendArgs& a, int b) : Seq(a, a.cache.past_of(b), a.cache.new_of(b)) {}
  __device__ __forceinline__ Seq(const PagedAttendArgs& a, int past_, int fresh_) : past(past_), fresh(fresh_) {
    len = fresh > 0 ? min(past + fresh, a.cache.capacity()) : 0;
    seq_tiles = (len + kTileKeys - 1) / kTileKeys;
    tiles = seq_tiles + (fresh * a.slot_blocks + 1) / 2;
  }
};

// of one sequence for the whole wave, in scalar registers
__device__ __forceinline__ Seq uniform_seq(const PagedAttendArgs& a, int b) {
  return Seq(a, __builtin_amdgcn_readfirstlane(a.cache.past_of(b)), __builtin_amdgcn_readfirstlane(a.cache.new_of(b)));
}

// x / d for whole numbers of a wave, d > 0: an estimate in 32-bit floating point, put right (a division of integers is forty
// instructions one after the other, which a wave by itself waits for).
__device__ __forceinline__ int uniform_div(int x, int d) {
  int q = __builtin_amdgcn_readfirstlane((int)((float)x * __builtin_amdgcn_rcpf((float)d)));
  while ((int64_t)q * d > x) q--;
  while ((int64_t)(q + 1) * d <= x) q++;
  return q;
}

// Tiles on the whole axis, and how many of them a wave takes.  The host has made sure that they fit 32 bits.
struct Plan {
  int total, per;
  __device__ __forceinline__ Plan(const PagedAttendArgs& a, int tiles_of_one_head) {
    total = tiles_of_one_head * (a.cache.H * a.row_tiles);
    per = uniform_div(total + a.waves - 1, a.waves);
  }
};

// One 16-byte piece a lane, global -> LDS, lane l to lds + l * 16, from an address of its own; inline assembly for the reason
// lds_dma (tile.h) gives: the compiler puts no waits between these loads and later LDS reads, whoever reads the tile waits by count.
__device__ __forceinline__ void global_to_lds(uint32_t lds, uint64_t address) {
  const uint32_t m0v = (uint32_t)__builtin_amdgcn_readfirstlane((int)lds);
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tglobal_load_lds_dwordx4 %1, off" : : "s"(m0v), "v"(address) : "memory", "m0");
}
template <int K>
__device__ __forceinline__ void wait_but() {
  WaveTileLoader<64>::wait_but<K>();
}

// The workspace: for each segment the slot of its first part and the wave of its last (written by the waves that have its first and
// its last tile; a segment without tiles has none), then statistics and sums by slot.
__device__ __forceinline__ int64_t segments(const PagedAttendArgs& a) {
  return ((int64_t)a.cache.B * a.cache.H * a.row_tiles + 1) & ~1ll;  // even: what follows stays on 16 bytes
}

// A part of a segment that a wave has: its row statistics (m, sum) and sums, row n of 16 (NR times) on lane n = lane & 15, elements
// 16 c + 4 q + i of o[c] on lane group q = lane >> 4 (MAP: 64 (c / 4) + 16 q + 4 i + c % 4, the order of the fp32 kernel).
struct PartAt {
  float *ml, *o;
  __device__ __forceinline__ PartAt(const PagedAttendArgs& a, int64_t slot) {
    float* first = a.work + segments(a) * 2;
    ml = first + slot * a.part_rows * 2;
    o = first + (int64_t)2 * a.waves * a.part_rows * 2 + slot * a.part_rows * a.part_width;
  }
};

// four elements from a multiple of four on (rows lie on 16-byte boundaries)
template <typename E>
__device__ __forceinline__ void store_four(char* p, int64_t i, const f32x4& x) {
  typedef typename E::elem elem4 __attribute__((ext_vector_type(4)));
  elem4 y;
#pragma unroll
  for (int e = 0; e < 4; e++) y[e] = (typename E::elem)x[e];
  *out_global<elem4>((typename E::elem*)p + i) = y;
}
// token that a sixteen of depth slots belongs to (at most 2^22 slots: off by less than 1 / 16 blocks, the estimate is exact)
__device__ __forceinline__ int token_of_block(const PagedAttendArgs& a, int block) { return (int)(((float)block + 0.5f) * a.blocks_inverse); }
struct FP32 {
  typedef float elem;
};

// What a row's exponents are taken against is its running maximum `top`, for fp16 less 15: probabilities up to 2^15 leave the type
// 2^-39 of the largest one as its last bit, not 2^-24.  (Maxima of 2^24 and more, whose neighbours are further apart, stay as they are: no
// probability may pass 2^16.)
template <typename E>
constexpr float kLead = __is_same(E, FP16) ? 15.f : 0.f;
template <typename E>
__device__ __forceinline__ float base_of(float top) {
  if (kLead<E> == 0.f) return top;
  const float y = top - kLead<E>;
  return top - y > kLead<E> + 0.5f ? top : y;
}
// log2 of a row's sum l of probabilities against m
template <typename E>
__device__ __forceinline__ float log_sum(float m, float l) {
  return kLead<E> == 0.f ? m + __builtin_amdgcn_logf(l) : (m + kLead<E>) + __builtin_amdgcn_logf(l * (1.f / (float)(1 << (int)kLead<E>)));
}

// the row of the call that row r of a row tile is
struct RowOf {
  int t, g;
  bool real;
  __device__ __forceinline__ RowOf(const PagedAttendArgs& a, int rt, int rows, int r) {
    const int row = rt * rows + r;
    real = row < a.cache.T * a.G;
    t = a.group_magic ? (int)__umulhi((unsigned)row, a.group_magic) : row;
    g = row - t * a.G;
  }
};

template <typename E, int W, int NR, bool MAP>
__device__ __forceinline__ void store_part(const Seq& seq, int b, int h, int rt, bool whole, int slot, const f32x4 (&o)[W / 16][NR],
                           const float (&m)[NR], const float (&l_lane)[NR], int lane) {
  const PagedAttendArgs a = reload();
  const int n = lane & 15, q = lane >> 4;
#pragma unroll
  for (int nr = 0; nr < NR; nr++) {
    const RowOf row(a, rt, 16 * NR, 16 * nr + n);
    const float l = quad_sum(l_lane[nr]);
    if (!row.real) continue;
    const bool padded = row.t >= seq.fresh;
    if (!whole) {
      const PartAt part(a, slot);
      const int r = 16 * nr + n;
      if (q == 0) {
        out_global<float>(part.ml)[2 * r] = padded ? kNegInf : m[nr];
        out_global<float>(part.ml)[2 * r + 1] = padded ? 0.f : l;
      }
#pragma unroll
      for (int c = 0; c < W / 16; c++) {
        float* to = part.o + (int64_t)r * W;
        if (!MAP) {
          *out_global<f32x4>(to + 16 * c + 4 * q) = o[c][nr];
        } else if (c % 4 == 0) {
#pragma unroll
          for (int i = 0; i < 4; i++) *out_global<f32x4>(to + 16 * c + 16 * q + 4 * i) = f32x4{o[c][nr][i], o[c + 1][nr][i], o[c + 2][nr][i], o[c + 3][nr][i]};
        }
      }
      continue;
    }
    const bool empty = padded || l == 0.f;
    const float inv = empty ? 0.f : 1.f / l;
    const int64_t to = b * a.so[0] + row.t * a.so[1] + row.g * a.so[2] + h * a.so[3];
#pragma unroll
    for (int c = 0; c < W / 16; c++) {
      const int e = MAP ? 64 * (c / 4) + 16 * q + 4 * (c % 4) : 16 * c + 4 * q;
      f32x4 x;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const float v = MAP ? o[c / 4 * 4 + i][nr][c % 4] : o[c][nr][i];
        x[i] = empty ? 0.f : v * inv;
      }
      if (e < a.Dv) store_four<E>(a.o, to + e, x);
    }
    if (q == 0)
      out_global<float>(a.lse)[b * a.slse[0] + row.t * a.slse[1] + row.g * a.slse[2] + h * a.slse[3]] =
          empty ? kNegInf : log_sum<E>(m[nr], l);
  }
}

// Logits from the sums of a matrix product, in the product's own basic block: the compiler's hazard pass leaves out the wait
// states that a result needs where its first reader comes behind a branch (seen as element 3 of some logits holding an
// earlier sum, where a skipped branch led straight from the last product to v_accvgpr_read).
template <int N>
__device__ __forceinline__ void scaled(float* x, const f32x4 (&s)[N], float scale) {
#pragma unroll
  for (int i = 0; i < 4 * N; i++) {
    x[i] = s[i >> 2][i & 3] * scale;
    asm volatile("" : "+v"(x[i]));
  }
}
// ... and before the results of the last products are read behind a loop or a branch: 32 wait states
__device__ __forceinline__ void products_done() { asm volatile("s_nop 15\n\ts_nop 15" ::: "memory"); }

// Maximum over the four lanes of a row.
__device__ __forceinline__ float row_max(float x) {
#if defined(__HIP_DEVICE_COMPILE__)
  const int xi = __builtin_bit_cast(int, x);
  const auto r = __builtin_amdgcn_permlane16_swap(xi, xi, false, false);
  x = fmaxf(__builtin_bit_cast(float, (int)r[0]), __builtin_bit_cast(float, (int)r[1]));
#endif
  return pair_max(x);
}

// Which keys row `nr` of a lane sees in a tile: indices [lo, hi) of the sequence's positions, or of its depth columns.
struct Window {
  int lo, hi;
  // key `key` of a tile that begins at index `first` and holds the keys `there`
  __device__ __forceinline__ bool sees(uint32_t there, int first, int key) const {
    return (there >> key & 1) & (first + key >= lo) & (first + key < hi);
  }
};

// The running softmax of one tile: x = logits in base 2 (what is not seen: -inf) -> probabilities against m (base_of the new maximum);
// the sums so far are brought to it.  In lanes of one row (four) m agrees, the sum is the lane's own.  Returns, for the wave, whether one of them is
// small (PagedWave::add_small).
template <typename E, int N, int MB, int NR>
__device__ __forceinline__ bool softmax_step(float (&x)[N], float& m, float& l, f32x4 (&o)[MB][NR], int nr) {
  float top = x[0], least = x[0];
#pragma unroll
  for (int i = 1; i < N; i++) {
    top = fmaxf(top, x[i]);
    if (kLead<E> != 0.f) least = fminf(least, x[i]);
  }
  top = fmaxf(m, base_of<E>(row_max(top)));
  const float from = top == kNegInf ? 0.f : top, small_below = from - 10.f;
  bool small = false;
  if (__any((top != m) | (kLead<E> != 0.f && least < small_below))) {  // (a NaN never equals itself: the sums become NaN with it)
    if (kLead<E> != 0.f) {
      bool here = false;
#pragma unroll
      for (int i = 0; i < N; i++) here |= (x[i] < small_below) & (x[i] > kNegInf);
      small = __any(here);
    }
    const float shrink = fast_exp2(m - from);
    l *= shrink;
#pragma unroll
    for (int c = 0; c < MB; c++)
#pragma unroll
      for (int i = 0; i < 4; i++) o[c][nr][i] *= shrink;
    m = top;
  }
#pragma unroll
  for (int i = 0; i < N; i++) {
    x[i] = fast_exp2(x[i] - from);
    l += x[i];
  }
  return small;
}

// ------------------------------------------------------------------------------------------------------------------
// 16-bit types
// ------------------------------------------------------------------------------------------------------------------

// LDS of a wave: NS stages of a K and a V tile; table entries of the tiles to come (2 NS tiles); addresses of the rows of one
// tile; which keys of a tile are there.
template <int W, int NS>
struct WaveLds {
  static constexpr int kTile = kTileKeys * W * 2, kStage = 2 * kTile;
  static constexpr int kTable = NS * kStage, kRows = kTable + 2 * NS * 256, kMask = kRows + kTileKeys * 16, kBytes = kMask + 16 * NS;
};

template <typename T, int W, int NR, int NS>
struct PagedWave {
  typedef WaveLds<W, NS> Lds;
  static constexpr int CH = W / 8, RPW = 64 / CH, NL = kTileKeys / RPW, KS = W / 32, MB = W / 16;
  const PagedAttendArgs& a;
  const int lane;
  const uint32_t lds;  // byte address
  Operand16<W> oa;
  i32x4 q[NR][KS];
  f32x4 o[MB][NR];
  float m[NR], l[NR];
  // the segment
  int b, h, rt;
  Seq seq;
  __device__ __forceinline__ PagedWave(const PagedAttendArgs& args, int lane_, uint32_t lds_) : a(args), lane(lane_), lds(lds_), seq(args, 0, 0) {}
  __device__ __forceinline__ void init() { oa.init(lane); }
  template <typename P>
  __device__ __forceinline__ MODA_LDS P* at(int byte) const {
    return (MODA_LDS P*)(uintptr_t)(lds + byte);
  }

  // table entries of a tile's positions (lanes r and r + 32: row r); past the sequence's pages: zeros
  __device__ __forceinline__ void fetch_table(int tile, int ring) const {
    const int pages = (seq.len + (1 << a.cache.page_shift) - 1) >> a.cache.page_shift;
    const i32x4 rs = rsrc_words(a.cache.table + b * a.cache.table_stride, (uint32_t)pages * 4);
    const unsigned page = ((unsigned)tile * kTileKeys + (lane & 31)) >> a.cache.page_shift;
    lds_dma<4>(rs, lds + Lds::kTable + ring * 256, tile < seq.seq_tiles ? (int)(page * 4) : kPadOffset, 0);
  }
  // Where the rows of a tile lie, every row for itself (two base addresses a tile for pages of 16 tokens and more, in scalar
  // registers, made no case faster by more than 1 % and the largest slower by 2): lane r's address of row r; zero: nowhere.
  __device__ __forceinline__ void find_rows(int tile, int ring, int stage) const {
    const PagedAttendArgs a = reload();
    const int r = lane & 31;
    uint64_t kp = 0, vp = 0;
    if (tile < seq.seq_tiles) {
      const int j = tile * kTileKeys + r, page = *at<int>(Lds::kTable + ring * 256 + 4 * lane);
      if (j < seq.len && (unsigned)page < (unsigned)a.cache.n_pages) {
        kp = (uint64_t)(a.cache.k + 2 * a.cache.offset(a.cache.sk, page, j, h));
        vp = (uint64_t)(a.cache.v + 2 * a.cache.offset(a.cache.sv, page, j, h));
      }
    } else {
      const int block = 2 * (tile - seq.seq_tiles) + (r >> 4), t = token_of_block(a, block), slot = 16 * (block - t * a.slot_blocks) + (r & 15);
      if (t < seq.fresh && slot < a.Lv) {
        const int64_t row = (int64_t)t * a.L + slot;
        kp = (uint64_t)(a.kd + 2 * (b * a.skd[0] + row * a.skd[1] + h * a.skd[2]));
        vp = (uint64_t)(a.vd + 2 * (b * a.svd[0] + row * a.svd[1] + h * a.svd[2]));
      }
    }
    const uint32_t there = (uint32_t)__ballot(kp != 0);
    if (lane < 32) {
      *at<uint64_t>(Lds::kRows + 16 * r) = kp;
      *at<uint64_t>(Lds::kRows + 16 * r + 8) = vp;
    }
    if (lane == 0) *at<uint32_t>(Lds::kMask + 4 * stage) = there;
  }
  // a K (0) or V (1) tile, from the rows found last (all addresses first: a load's assembly block is a barrier to the reads behind it)
  __device__ __forceinline__ void fetch_tile(int which, int stage) const {
    const uint32_t to = lds + stage * Lds::kStage + which * Lds::kTile;
    const int prow = lane / CH, pch = lane % CH, dim = which ? a.Dv : a.D;
    const uint64_t zero = (uint64_t)&zero_line[0];
    uint64_t from[NL];
#pragma unroll
    for (int i = 0; i < NL; i++) from[i] = *at<uint64_t>(Lds::kRows + 16 * (i * RPW + prow) + 8 * which);
#pragma unroll
    for (int i = 0; i < NL; i++) {
      const int chunk = pch ^ Tile<W>::swz(i * RPW + prow);
      global_to_lds(to + i * 1024, from[i] != 0 && chunk * 8 < dim ? from[i] + chunk * 16 : zero);
    }
  }

  // the K tile of step i + NS, the tile's rows, and the table entries of the tile NS steps further
  __device__ __forceinline__ void send(int tile, int i, int stage) const {
    fetch_table(tile + 2 * NS, (i + 2 * NS) % (2 * NS));
    find_rows(tile + NS, (i + NS) % (2 * NS), stage);
    fetch_tile(0, stage);
  }

  // Probabilities w times a tile's values.  They go to the matrix instruction in pieces, each the rounding of what those before it left:
  // three of bf16 hold all 24 bits, two of fp16 hold 22 (but see add_small).  With two of bf16, 16 bits, 0.2 % of the results were rounded the
  // other way than the exact ones, with three 0.01 %, as many as where everything is in 32 bits; the third costs drafted tokens 4 % and one token
  // nothing.
  static constexpr int kPieces = __is_same(T, BF16) ? 3 : 2;
  __device__ __forceinline__ void add_products(float (&w)[NR][8], lds_cptr tile) {
    i32x4 piece[kPieces][NR];
#pragma unroll
    for (int nr = 0; nr < NR; nr++) {
#pragma unroll
      for (int k = 0; k < kPieces; k++) {
#pragma unroll
        for (int i = 0; i < 4; i++) piece[k][nr][i] = pack2<T>(w[nr][2 * i], w[nr][2 * i + 1]);
        if (k + 1 == kPieces) continue;
#pragma unroll
        for (int i = 0; i < 4; i++) {
          float x0, x1;
          unpack2<T>(piece[k][nr][i], x0, x1);
          w[nr][2 * i] -= x0;
          w[nr][2 * i + 1] -= x1;
        }
      }
    }
    constexpr int DEPTH = 4;
    i32x4 ops[MB];
#pragma unroll
    for (int c = 0; c < DEPTH && c < MB; c++) ops[c] = oa.tr_operand(tile, 0, c);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int c = 0; c < MB; c++) {
      if (c + DEPTH < MB) ops[c + DEPTH] = oa.tr_operand(tile, 0, c + DEPTH);
#pragma unroll
      for (int k = 0; k < kPieces; k++)
#pragma unroll
        for (int nr = 0; nr < NR; nr++) o[c][nr] = mfma16<T>(ops[c], piece[k][nr], o[c][nr]);
      __builtin_amdgcn_sched_barrier(0);
    }
  }

  // fp16: probabilities below 2^-10 -- 2^-25 of the row's largest -- would be left fewer than 14 bits above the type's last one, 2^-24, and
  // in the end none, while the sum under them counts them.  They take a product of their own, 2^25 times as large, o with them; what they
  // lose then is 2^-64 of the largest.  (Asking for them and the code for them cost drafted tokens 6 % at head dim 64, 12 at 128, one token
  // nothing; a second pass over the runs that have them, instead, twice the time where there are some.)
  static constexpr float kUp = 0x1p25f;
  __device__ __forceinline__ void scale_sums(float by) {
#pragma unroll
    for (int c = 0; c < MB; c++)
#pragma unroll
      for (int nr = 0; nr < NR; nr++)
#pragma unroll
        for (int i = 0; i < 4; i++) o[c][nr][i] *= by;
  }
  __device__ __forceinline__ void add_small(float (&p)[NR][8], lds_cptr tile) {
    float w[NR][8];
#pragma unroll
    for (int nr = 0; nr < NR; nr++)
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const bool small = p[nr][i] < 0x1p-10f;
        w[nr][i] = small ? p[nr][i] * kUp : 0.f;
        p[nr][i] = small ? 0.f : p[nr][i];
      }
    scale_sums(kUp);
    add_products(w, tile);
    scale_sums(1.f / kUp);
  }

  // Values of a tile, one of them not finite: each row adds up what it sees, key by key.  0 x inf would reach rows that do not see it, and of
  // an infinite value that a row sees the pieces of its probability would make inf and, the second being zero or negative, NaN.  p: the
  // lane's probabilities (zero where unseen, and where they underflow 32 bits: NaN then, as in any 32-bit sum).
  __device__ __forceinline__ void add_key_by_key(const float (&p)[8], int nr, Window win, int first, uint32_t there, lds_cptr tile) {
    const int n = lane & 15, g = lane >> 4;
#pragma unroll 1
    for (int key = 0; key < kTileKeys; key++) {
      const int low = key & 15, from = (low >> 2) == 0 ? 0 : (low >> 2) == 1 ? 3 : (low >> 2) == 2 ? 1 : 2;  // slot_base(from) = low & 12
      float x = p[0];
#pragma unroll
      for (int i = 1; i < 8; i++) x = i == (key >> 4) * 4 + (key & 3) ? p[i] : x;
      x = __shfl(x, n + 16 * from, 64);
      if (!win.sees(there, first, key)) continue;
#pragma unroll
      for (int c = 0; c < MB; c++) {
        const int e = 16 * c + 4 * g;
        const i32x2 v = *(MODA_LDS const i32x2*)(tile + Tile<W>::off(key, e >> 3) + (e & 7));
        float v0, v1, v2, v3;
        unpack2<T>(v[0], v0, v1);
        unpack2<T>(v[1], v2, v3);
        o[c][nr][0] += x * v0;
        o[c][nr][1] += x * v1;
        o[c][nr][2] += x * v2;
        o[c][nr][3] += x * v3;
      }
    }
  }

  // Tiles [t0, t1) of the segment.  `careful`: every tile's values are looked at, not only those that some row does not see.
  __device__ __forceinline__ void run(int t0, int t1, bool careful) {
    const int n = lane & 15, g = lane >> 4, tiles = t1 - t0;
    const bool one_token = a.cache.T == 1;
    Window seq_win[NR], depth_win[NR];
    int first_t;  // of the row tile's tokens
    {
    const PagedAttendArgs a = reload();
    first_t = RowOf(a, rt, 16 * NR, 0).t;
#pragma unroll
    for (int nr = 0; nr < NR; nr++) {
      const RowOf row(a, rt, 16 * NR, 16 * nr + n);
      const int64_t from = b * a.sq[0] + row.t * a.sq[1] + row.g * a.sq[2] + h * a.sq[3];
#pragma unroll
      for (int ks = 0; ks < KS; ks++) {
        const int e = 32 * ks + 8 * g;
        i32x4 x = {0, 0, 0, 0};
        if (row.real && e < a.D) x = *in_global<i32x4>(a.q + 2 * (from + e));
        q[nr][ks] = x;
      }
      seq_win[nr] = {0, seq.past + row.t + 1};
      depth_win[nr] = {row.t * a.slot_blocks * 16, row.t * a.slot_blocks * 16 + a.Lv};
      m[nr] = kNegInf;
      l[nr] = 0.f;
#pragma unroll
      for (int c = 0; c < MB; c++) o[c][nr] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    }
    // the table's entries and the rows have to be here before the tiles are sent for: the compiler would wait for everything
    // behind the rows as well
#pragma unroll
    for (int j = 0; j < NS; j++) fetch_table(t0 + j, j);
#pragma unroll
    for (int nr = 0; nr < NR; nr++)
#pragma unroll
      for (int ks = 0; ks < KS; ks++) asm volatile("" : "+v"(q[nr][ks]));
    wait_but<0>();
    // loads behind a tile's K when NS - 1 more tiles are on their way, and behind its V when the next K is as well
    constexpr int kBehindK = NL + (NS - 1) * (2 * NL + 1), kBehindV = (NS - 1) * (2 * NL + 1) + NL + 1;
    // step i sends for tile i + NS and works on tile i (the first NS steps only send: one copy of the code)
#pragma unroll 1
    for (int i = -NS; i < tiles; i++) {
      const int stage = (i + NS) % NS, tile = t0 + i;
      const bool more = i + NS < tiles;
      if (i < 0) {
        if (more) {
          send(tile, i, stage);
          fetch_tile(1, stage);
        }
        continue;
      }
      if (i + NS <= tiles)
        wait_but<kBehindK>();
      else
        wait_but<0>();
      const uint32_t there = (uint32_t)__builtin_amdgcn_readfirstlane((int)*at<uint32_t>(Lds::kMask + 4 * stage));
      const lds_cptr kt = at<uint16_t>(stage * Lds::kStage), vt = at<uint16_t>(stage * Lds::kStage + Lds::kTile);
      f32x4 s[2][NR];
      mfma16_rows<T, W, 2, NR, 4>(oa, kt, q, s);
      float p[NR][8];
#pragma unroll
      for (int nr = 0; nr < NR; nr++) {
        const f32x4 both[2] = {s[0][nr], s[1][nr]};
        scaled(p[nr], both, a.scale);
      }
      WaveTileLoader<64>::reads_done();
      if (more) send(tile, i, stage);
      const bool depth = tile >= seq.seq_tiles;
      const int first = (depth ? tile - seq.seq_tiles : tile) * kTileKeys;
      const bool all_seen = there == ~0u && (depth ? one_token : first + kTileKeys - 1 <= seq.past + first_t);
      if (!all_seen) {
#pragma unroll
        for (int nr = 0; nr < NR; nr++) {
          const Window win = depth ? depth_win[nr] : seq_win[nr];
#pragma unroll
          for (int i8 = 0; i8 < 8; i8++) {
            const int key = 16 * (i8 >> 2) + slot_base(g) + (i8 & 3);
            p[nr][i8] = win.sees(there, first, key) ? p[nr][i8] : kNegInf;
          }
        }
      }
      bool small = false;
#pragma unroll
      for (int nr = 0; nr < NR; nr++) small |= softmax_step<T, 8>(p[nr], m[nr], l[nr], o, nr);
      if (more)
        wait_but<kBehindV>();
      else
        wait_but<0>();
      bool odd = false;
      if (careful || (!all_seen && !one_token)) {
        const int top = __is_same(T, BF16) ? 0x7f80 : 0x7c00;
#pragma unroll 2
        for (int c = lane; c < kTileKeys * CH; c += 64) {
          const i32x4 v = *(MODA_LDS const i32x4*)(vt + 8 * c);
#pragma unroll
          for (int i4 = 0; i4 < 4; i4++) odd = odd || (v[i4] & top) == top || (v[i4] >> 16 & top) == top;
        }
      }
      if (__builtin_expect(__any(odd), false)) {
#pragma unroll
        for (int nr = 0; nr < NR; nr++) add_key_by_key(p[nr], nr, depth ? depth_win[nr] : seq_win[nr], first, there, vt);
      } else {
        if (__builtin_expect(small, false)) add_small(p, vt);
        add_products(p, vt);
      }
      WaveTileLoader<64>::reads_done();
      if (more) fetch_tile(1, stage);
    }
    products_done();
  }
  // Whether a result is NaN and its row's sum is not: from a value that is not finite.  (Asked of all elements of a row together: infinities of
  // both signs among them run once more for nothing.)
  __device__ __forceinline__ bool spoiled() const {
    bool bad = false;
#pragma unroll
    for (int nr = 0; nr < NR; nr++) {
      f32x4 all = o[0][nr];
#pragma unroll
      for (int c = 1; c < MB; c++) all += o[c][nr];
      const float sum = (all[0] + all[1]) + (all[2] + all[3]);
      bad |= (sum != sum) & (l[nr] == l[nr]);
    }
    return __any(bad);
  }
};

// Walks a wave's run of the axis: part(seq, b, h, rt, t0, t1, whole, slot) for each segment in it.
// `meanwhile` runs while the counts are on their way.
template <typename G, typename F>
__device__ __forceinline__ void walk(const PagedAttendArgs& a, int lane, G&& meanwhile, F&& part) {
  const int heads = a.cache.H * a.row_tiles;
  // Up to 64 sequences are read once; of more the first pass over the others is for the total alone.  Counts that somebody
  // changes meanwhile make wrong results; places stay within the arrays and loops end all the same.
  Seq own(a, 0, 0);
  if (lane < a.cache.B) own = Seq(a, lane);
  int sum = own.tiles;
  for (int b = lane + 64; b < a.cache.B; b += 64) sum += Seq(a, b).tiles;
  meanwhile();
  const Plan plan(a, __builtin_amdgcn_readlane(wave_scan(sum), 63));
  const int wave = blockIdx.x;
  if ((int64_t)wave * plan.per >= plan.total) return;
  const int s = wave * plan.per, e = min(s + plan.per, plan.total);
  int b = 0, start = 0, first_lane = 0;  // start of sequence b, in tiles
  for (int b0 = 0;;) {
    const int upto = wave_scan(own.tiles);
    const uint64_t behind = __ballot(start + upto * heads > s);
    first_lane = behind ? __builtin_ctzll(behind) : 63;
    start += __builtin_amdgcn_readlane(behind ? upto - own.tiles : upto, first_lane) * heads;
    if (behind) {
      b = b0 + first_lane;
      break;
    }
    if ((b0 += 64) >= a.cache.B) return;
    own = b0 + lane < a.cache.B ? Seq(a, b0 + lane) : Seq(a, 0, 0);
  }
  Seq seq(a, __builtin_amdgcn_readlane(own.past, first_lane), __builtin_amdgcn_readlane(own.fresh, first_lane));
  const int rest = __builtin_amdgcn_readfirstlane(s - start);
  int hr = uniform_div(rest, seq.tiles), tile = rest - hr * seq.tiles;
  int h = a.row_tiles == 1 ? hr : uniform_div(hr, a.row_tiles), rt = hr - h * a.row_tiles;
  for (int at = s; at < e;) {
    const int upto = min(seq.tiles, tile + (e - at)), slot = 2 * wave + (at == s ? 0 : 1);
    const bool first = tile == 0, last = upto == seq.tiles;
    if (lane == 0) {
      int* info = (int*)a.work + 2 * ((int64_t)b * heads + h * a.row_tiles + rt);
      if (first) info[0] = slot;
      if (last) info[1] = wave;
    }
    part(seq, b, h, rt, tile, upto, first && last, slot);
    at += upto - tile;
    tile = 0;
    if (++rt < a.row_tiles) continue;
    rt = 0;
    if (++h < a.cache.H || at >= e) continue;
    h = 0;
    do {
      if (++b >= a.cache.B) return;
      seq = uniform_seq(a, b);
    } while (seq.tiles == 0);
  }
}

// Stages of a wave's ring and waves of a compute unit (four at one a SIMD).  With several waves a SIMD one stage does: K of the next
// tile is sent for once the scores are formed, V once it is used, and while a wave waits the others work.  Measured: 128 sequences of
// 4 - 8 K tokens, 64 query heads of 64 on 8, with 2 stages and 8 waves 304 us, 1 and 12: 286, 1 and 16: 299 (registers for
// four waves a SIMD leave none over); head dim 128, 2 stages and 4 waves against 1 and 8: 2048 short sequences 145 -> 121
// us, 8 of 2 K tokens 15.3 -> 13.2, a million tokens 356 -> 361.
template <int W, int NR>
struct Shape {
  static constexpr int kStages = NR == 2 ? 2 : 1;
  static constexpr int kWaves = NR == 2 ? (W == 64 ? 8 : 4) : W == 64 ? 12 : W == 128 ? 8 : 4;
};

template <typename T, int W, int NR>
__global__ __launch_bounds__(64, (Shape<W, NR>::kWaves + 3) / 4) void paged_kernel(const PagedAttendArgs a) {
  extern __shared__ __attribute__((aligned(16))) char lds_raw[];
  const int lane = threadIdx.x;
  PagedWave<T, W, NR, Shape<W, NR>::kStages> w(a, lane, (uint32_t)(uintptr_t)(MODA_LDS char*)lds_raw);
  walk(a, lane, [&] { w.init(); }, [&](const Seq& seq, int b, int h, int rt, int t0, int t1, bool whole, int slot) {
    w.seq = seq;
    w.b = b;
    w.h = h;
    w.rt = rt;
    for (bool careful = false;; careful = true) {
      w.run(t0, t1, careful);
      if (careful || __builtin_expect(!w.spoiled(), true)) break;
    }
    store_part<T, W, NR, false>(seq, b, h, rt, whole, slot, w.o, w.m, w.l, lane);
  });
}

// ------------------------------------------------------------------------------------------------------------------
// fp32: operands from global memory into the registers of v_mfma_f32_16x16x4_f32 (see fp32_kernels.hip for the layout)
// ------------------------------------------------------------------------------------------------------------------

template <int W>
__global__ __launch_bounds__(64, 1) void paged_fp32_kernel(const PagedAttendArgs a) {
  constexpr int MB = W / 16;
  const int lane = threadIdx.x, n = lane & 15, g = lane >> 4;
  const bool one_token = a.cache.T == 1;
  walk(a, lane, [] {}, [&](const Seq& seq, int b, int h, int rt, int t0, int t1, bool whole, int slot) {
    const RowOf row(a, rt, 16, n);
    const float* qp = (const float*)a.q + b * a.sq[0] + row.t * a.sq[1] + row.g * a.sq[2] + h * a.sq[3];
    f32x4 q[MB], o[MB][1];
    float m[1] = {kNegInf}, l[1] = {0.f};
#pragma unroll
    for (int s = 0; s < MB; s++) {
      q[s] = f32x4{0.f, 0.f, 0.f, 0.f};
      if (row.real && 16 * s + 4 * g < a.D) q[s] = *(const f32x4*)(qp + 16 * s + 4 * g);
      o[s][0] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    const int first_t = RowOf(a, rt, 16, 0).t;
    // 16 keys at a time, up to head dim 128 with the next ones on their way while these are worked on
    struct Keys {
      f32x4 k[MB], v[4][MB / 4];
      uint64_t vp;  // of key n
      uint32_t there;
    };
    auto fetch = [&](int half, Keys& x) {
      const bool depth = half >= 2 * seq.seq_tiles;
      const int key = (depth ? half - 2 * seq.seq_tiles : half) * 16 + n;
      const float *kp = nullptr, *vp = nullptr;  // (read as global memory below: a choice between them and zeros would make flat loads)
      if (!depth) {
        const int page = key < seq.len ? a.cache.page_of(b, key) : -1;
        if (page >= 0) {
          kp = (const float*)a.cache.k + a.cache.offset(a.cache.sk, page, key, h);
          vp = (const float*)a.cache.v + a.cache.offset(a.cache.sv, page, key, h);
        }
      } else {
        const int t = token_of_block(a, key >> 4), slot = key - 16 * t * a.slot_blocks;
        if (t < seq.fresh && slot < a.Lv) {
          const int64_t r = (int64_t)t * a.L + slot;
          kp = (const float*)a.kd + b * a.skd[0] + r * a.skd[1] + h * a.skd[2];
          vp = (const float*)a.vd + b * a.svd[0] + r * a.svd[1] + h * a.svd[2];
        }
      }
      x.vp = (uint64_t)vp;
      x.there = (uint32_t)__ballot(kp != nullptr) & 0xffffu;
      // a row that is not there, and pieces past the head dim: zeros
      typedef const __attribute__((address_space(1))) f32x4* global_f32x4;
      const float* zeros = (const float*)zero_line;
#pragma unroll
      for (int s = 0; s < MB; s++) {
        const bool in = kp && 16 * s + 4 * g < a.D;
        x.k[s] = *(global_f32x4)(uint64_t)(in ? kp + 16 * s + 4 * g : zeros);
      }
#pragma unroll
      for (int r = 0; r < 4; r++) {
        const float* row_v = (const float*)__shfl((unsigned long long)x.vp, 4 * g + r, 64);
#pragma unroll
        for (int c = 0; c < MB / 4; c++) x.v[r][c] = *(global_f32x4)(uint64_t)(row_v && 64 * c + 4 * n < a.Dv ? row_v + 64 * c + 4 * n : zeros);
      }
    };
    auto work = [&](int half, const Keys& x) {
      const bool depth = half >= 2 * seq.seq_tiles;
      const int first = (depth ? half - 2 * seq.seq_tiles : half) * 16;
      const uint32_t there = x.there;
      const auto& k = x.k;
      const auto& v = x.v;
      f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < MB; c++)
#pragma unroll
        for (int i = 0; i < 4; i++) s = __builtin_amdgcn_mfma_f32_16x16x4f32(k[c][i], q[c][i], s, 0, 0, 0);
      float p[4];
      const f32x4 sums[1] = {s};
      scaled(p, sums, a.scale);
      const Window win = depth ? Window{row.t * a.slot_blocks * 16, row.t * a.slot_blocks * 16 + a.Lv} : Window{0, seq.past + row.t + 1};
      const bool all_seen = there == 0xffffu && (depth ? one_token : first + 15 <= seq.past + first_t);
#pragma unroll
      for (int i = 0; i < 4; i++) p[i] = (all_seen | win.sees(there, first, 4 * g + i)) ? p[i] : kNegInf;
      softmax_step<FP32, 4>(p, m[0], l[0], o, 0);
      bool odd = false;
      if (!all_seen && !one_token) {
#pragma unroll
        for (int r = 0; r < 4; r++)
#pragma unroll
          for (int c = 0; c < MB / 4; c++)
#pragma unroll
            for (int i = 0; i < 4; i++) odd = odd || !(__builtin_fabsf(v[r][c][i]) < __builtin_huge_valf());
      }
      if (__any(odd)) {  // see PagedWave::add_key_by_key
#pragma unroll 1
        for (int j = 0; j < 16; j++) {
          const int i = j & 3;
          const float w = __shfl(i == 0 ? p[0] : i == 1 ? p[1] : i == 2 ? p[2] : p[3], n + 16 * (j >> 2), 64);
          const float* from = (const float*)__shfl((unsigned long long)x.vp, j, 64);
          if (!win.sees(there, first, j)) continue;
#pragma unroll
          for (int c = 0; c < MB; c++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
              const int at = 64 * (c / 4) + 16 * g + 4 * e + c % 4;
              if (at < a.Dv) o[c][0][e] += w * from[at];
            }
        }
      } else {
#pragma unroll
        for (int c = 0; c < MB; c++)
#pragma unroll
          for (int r = 0; r < 4; r++) o[c][0] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[r][c / 4][c % 4], p[r], o[c][0], 0, 0, 0);
      }
    };
    if constexpr (W == 256) {  // two sets of keys and values do not fit beside q and o: 451 us spilled, 388 one after the other (32 x 1 - 8 K tokens)
      Keys x;
#pragma unroll 1
      for (int half = 2 * t0; half < 2 * t1; half++) {
        fetch(half, x);
        work(half, x);
      }
    } else {
      Keys x[2];
      fetch(2 * t0, x[0]);
      for (int half = 2 * t0; half < 2 * t1; half += 2) {
        fetch(half + 1, x[1]);
        work(half, x[0]);
        if (half + 2 < 2 * t1) fetch(half + 2, x[0]);
        work(half + 1, x[1]);
      }
    }
    products_done();
    store_part<FP32, W, 1, true>(seq, b, h, rt, whole, slot, o, m, l, lane);
  });
}

// ------------------------------------------------------------------------------------------------------------------
// joining
// ------------------------------------------------------------------------------------------------------------------

// A workgroup per query row, head and WC of its W elements: the parts of its segment, in the order of the axis.  WC / 4 threads have four
// elements each of every (NT * 4 / WC)-th part.
template <typename E, int W, int WC, int NT>
__global__ __launch_bounds__(NT) void paged_join_kernel(const PagedAttendArgs a, int rows_per_tile) {
  constexpr int LANES = WC / 4, GROUPS = NT / LANES, WAVES = NT / 64;
  __shared__ f32x4 sums[WAVES][LANES];
  __shared__ float lsum[WAVES], tops[WAVES];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, x = tid % LANES, group = tid / LANES;
  unsigned at = workgroup();  // (rows are below 2^31)
  const int e0 = W == WC ? 0 : (int)(at % (W / WC)) * WC;  // the workgroup's first element
  at /= W / WC;
  const int h = (int)(at % (unsigned)a.cache.H);
  at /= (unsigned)a.cache.H;
  const int rows = a.cache.T * a.G, row = (int)(at % (unsigned)rows), b = (int)(at / (unsigned)rows);
  if (b >= a.cache.B) return;
  const int rt = row / rows_per_tile, r = row - rt * rows_per_tile, t = row / a.G, g = row - t * a.G;
  const int64_t seg = ((int64_t)b * a.cache.H + h) * a.row_tiles + rt;
  const int first = ((const int*)a.work)[2 * seg], last = ((const int*)a.work)[2 * seg + 1];
  const int parts = Seq(a, b).tiles && (unsigned)first < 2u * a.waves && (unsigned)last < (unsigned)a.waves ? last - (first >> 1) + 1 : 0;
  if (parts == 1) return;  // one wave had all of it and has stored the row
  auto slot = [&](int p) { return p == 0 ? first : (first & ~1) + 2 * p; };
  float top = kNegInf;
  for (int p = tid; p < parts; p += NT) top = fmaxf(top, PartAt(a, slot(p)).ml[2 * r]);
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor(top, d, 64));
  if (WAVES > 1) {
    if (lane == 0) tops[wave] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < WAVES; i++) top = fmaxf(top, tops[i]);
  }
  const float from = top == kNegInf ? 0.f : top;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  float l = 0.f;
#pragma unroll 4
  for (int p = group; p < parts; p += GROUPS) {
    const PartAt part(a, slot(p));
    const float w = fast_exp2(part.ml[2 * r] - from);
    const f32x4 v = *(const f32x4*)(part.o + (int64_t)r * W + e0 + 4 * x);
    l += w * part.ml[2 * r + 1];
#pragma unroll
    for (int i = 0; i < 4; i++) o[i] += w * v[i];
  }
#pragma unroll
  for (int d = LANES; d < 64; d <<= 1) {  // groups of one wave, then waves
    l += __shfl_xor(l, d, 64);
#pragma unroll
    for (int i = 0; i < 4; i++) o[i] += __shfl_xor(o[i], d, 64);
  }
  if (WAVES > 1) {
    if (lane < LANES) sums[wave][x] = o;
    if (lane == 0) lsum[wave] = l;
    __syncthreads();
    if (wave > 0) return;
    l = lsum[0];
    o = sums[0][x];
#pragma unroll
    for (int i = 1; i < WAVES; i++) {
      l += lsum[i];
      const f32x4 v = sums[i][x];
#pragma unroll
      for (int e = 0; e < 4; e++) o[e] += v[e];
    }
  }
  if (lane >= LANES) return;
  const bool empty = l == 0.f;
  const float inv = empty ? 0.f : 1.f / l;
  const int64_t to = b * a.so[0] + t * a.so[1] + g * a.so[2] + h * a.so[3];
#pragma unroll
  for (int e = 0; e < 4; e++) o[e] = empty ? 0.f : o[e] * inv;
  if (e0 + 4 * x < a.Dv) store_four<E>(a.o, to + e0 + 4 * x, o);
  if (e0 + x == 0) a.lse[b * a.slse[0] + t * a.slse[1] + g * a.slse[2] + h * a.slse[3]] = empty ? kNegInf : log_sum<E>(top, l);
}

int tile_width(const PagedAttendArgs& a) {
  const int d = a.D > a.Dv ? a.D : a.Dv;
  return d <= 64 ? 64 : d <= 128 ? 128 : 256;
}

// rows of a row tile, in sixteens: as many as a wave's registers hold without spilling
int row_blocks(const PagedAttendArgs& a, int dtype) {
  const int rows = a.cache.T * a.G, width = tile_width(a);
  return dtype == MODA_HIP_FP32 || rows <= 16 || width == 256 ? 1 : 2;
}

template <typename T, int W, int NR>
hipError_t launch_waves(const PagedAttendArgs& a, hipStream_t stream) {
  constexpr int bytes = WaveLds<W, Shape<W, NR>::kStages>::kBytes;
  static_assert(bytes * Shape<W, NR>::kWaves <= 160 << 10 && bytes <= 64 << 10, "the rings of a compute unit");
  paged_kernel<T, W, NR><<<a.waves, 64, bytes, stream>>>(a);
  return hipGetLastError();
}
template <typename T>
hipError_t launch_waves_as(const PagedAttendArgs& a, int width, int blocks, hipStream_t stream) {
  if (width == 256) return launch_waves<T, 256, 1>(a, stream);
  if (width == 128) return blocks == 1 ? launch_waves<T, 128, 1>(a, stream) : launch_waves<T, 128, 2>(a, stream);
  return blocks == 1 ? launch_waves<T, 64, 1>(a, stream) : launch_waves<T, 64, 2>(a, stream);
}
int waves_of_a_unit(int width, int blocks) {
  if (width == 256) return Shape<256, 1>::kWaves;
  if (width == 128) return blocks == 1 ? Shape<128, 1>::kWaves : Shape<128, 2>::kWaves;
  return blocks == 1 ? Shape<64, 1>::kWaves : Shape<64, 2>::kWaves;
}

// Threads of a row's workgroup: parts of one row are read side by side, and many rows keep the card busy by themselves.  Few rows of many
// parts are spread by elements as well (16 rows of 512 parts 12.5 -> 8.6 us; 128 rows of 130 parts: 6.8 spread, 4.5 not).
template <typename E, int W>
hipError_t launch_join_of(const PagedAttendArgs& a, int per_tile, hipStream_t stream) {
  const int64_t rows = (int64_t)a.cache.B * a.cache.T * a.G * a.cache.H;
  if (rows >= 2048)
    paged_join_kernel<E, W, W, 64><<<grid_of(rows), 64, 0, stream>>>(a, per_tile);
  else if (rows >= 256)
    paged_join_kernel<E, W, W, 256><<<grid_of(rows), 256, 0, stream>>>(a, per_tile);
  else if (rows >= 64)
    paged_join_kernel<E, W, W, 1024><<<grid_of(rows), 1024, 0, stream>>>(a, per_tile);
  else
    paged_join_kernel<E, W, 32, 1024><<<grid_of(rows * (W / 32)), 1024, 0, stream>>>(a, per_tile);
  return hipGetLastError();
}
template <typename E>
hipError_t launch_join(const PagedAttendArgs& a, int width, int blocks, hipStream_t stream) {
  if (width == 64) return launch_join_of<E, 64>(a, 16 * blocks, stream);
  return width == 128 ? launch_join_of<E, 128>(a, 16 * blocks, stream) : launch_join_of<E, 256>(a, 16 * blocks, stream);
}

}  // namespace

// How the work is cut: waves on the axis, row tiles, the workspace's rows.  Nothing here depends on what the device arrays hold.
size_t plan_paged_attend(PagedAttendArgs& a, int dtype) {
  const int width = tile_width(a), blocks = row_blocks(a, dtype), rows = a.cache.T * a.G;
  a.row_tiles = (rows + 16 * blocks - 1) / (16 * blocks);
  a.part_rows = rows < 16 * blocks ? rows : 16 * blocks;
  a.part_width = width;
  // waves of the whole card: what holds its rings in the 160 KB of a compute unit, fp32 by its registers
  const int per_unit = dtype == MODA_HIP_FP32 ? (width == 64 ? 8 : 4) : waves_of_a_unit(width, blocks);
  a.slot_blocks = (a.Lv + 15) / 16;
  a.blocks_inverse = 1.f / (float)(a.slot_blocks > 0 ? a.slot_blocks : 1);
  const int64_t capacity = (int64_t)a.cache.max_pages << a.cache.page_shift;
  const int64_t most = (int64_t)a.cache.B * a.cache.H * a.row_tiles *
                       ((capacity + kTileKeys - 1) / kTileKeys + ((int64_t)a.cache.T * a.slot_blocks + 1) / 2);
  if (most >= 1ll << 30) return 0;  // the axis is counted in 32 bits
  a.group_magic = a.G == 1 ? 0 : (unsigned)((1ull << 32) / a.G) + 1;  // row / G = umulhi(row, magic): rows are below 2^16
  a.waves = (int)(most < 256 * per_unit ? (most > 0 ? most : 1) : 256 * per_unit);
  const size_t segments = ((size_t)a.cache.B * a.cache.H * a.row_tiles + 1) / 2 * 2;
  return (segments * 2 + (size_t)2 * a.waves * a.part_rows * (a.part_width + 2)) * sizeof(float);
}

hipError_t launch_paged_attend(const PagedAttendArgs& a, int dtype, hipStream_t stream) {
  const int width = tile_width(a), blocks = row_blocks(a, dtype);
  hipError_t e;
  if (dtype == MODA_HIP_FP32) {
    if (width == 64)
      paged_fp32_kernel<64><<<a.waves, 64, 0, stream>>>(a);
    else if (width == 128)
      paged_fp32_kernel<128><<<a.waves, 64, 0, stream>>>(a);
    else
      paged_fp32_kernel<256><<<a.waves, 64, 0, stream>>>(a);
    e = hipGetLastError();
    if (e == hipSuccess) e = launch_join<FP32>(a, width, blocks, stream);
  } else if (dtype == MODA_HIP_FP16) {
    e = launch_waves_as<FP16>(a, width, blocks, stream);
    if (e == hipSuccess) e = launch_join<FP16>(a, width, blocks, stream);
  } else {
    e = launch_waves_as<BF16>(a, width, blocks, stream);
    if (e == hipSuccess) e = launch_join<BF16>(a, width, blocks, stream);
  }
  return e;
}

}  // namespace moda
