// Attention of a chunk of new tokens per sequence over the [num_blocks, Hkv*D/16, block_size, 16] fp16 caches: the kernel,
// a template over head_dim.
//
//   row (token i, head h) of sequence b sits at position p = L_b - n_b + i and sees keys max(0, p - window + 1) .. p:
//   o = sum_j softmax_j(scale q.k_j) v_j,   lse = log sum_j exp(scale q.k_j)
//
// Work.  The query heads of a kv head share its K and V, so a kv head's rows are (token, head of the group) pairs, token
// by token, and a tile is up to 256 of them (head_dim above 128: 128) from one sequence.  A workgroup of eight (four) waves,
// one per CU, runs over the keys a tile sees, once, with the running maximum and sum of its softmax in registers.
//
//  * More than 32 rows ("tile"): wave w owns rows 32w .. 32w+31, in two blocks of 16 columns; the waves
//    share K and V tiles of kTile tokens in LDS, which are on their way while others are computed.  Tiles of at most half the
//    rows may give each half of the waves one half of every tile's keys instead (chunk_run).
//  * Fewer ("stream", the decode-like case): every wave owns all rows and its own 32 tokens of every 256 (128); K goes from
//    memory straight into the operand registers, V through the wave's own piece of LDS, no barriers in the loop, and the
//    eight waves are joined through LDS at the end.
//
// Operands.  The cache layout is the operand layout of v_mfma_f32_16x16x32_f16: lane (n = lane%16, kg = lane/16) takes for
// token n the 16 bytes that hold d = 32s + 8kg ..+7, so S^T[token][row] = K . Q^T needs no shuffling, in LDS or out of it (a
// tile keeps the cache's [chunk of 16 d][token][16], and every fragment read covers contiguous bytes).  S^T leaves lane
// (row n, kg) with tokens 4kg ..+3 of each group of 16; two groups packed to fp16 are the operand P^T of O^T += V^T . P^T, with
// the 32 tokens of a step in the order 16g + 4kg + i.  V^T in that order is what ds_read_b64_tr_b16 returns from the same
// layout: 16 lanes read 4 tokens x 16 d, 128 contiguous bytes, and lane n receives d = n of the four.
//
// Softmax.  In log2 units, fp32.  The reference value of a row moves only when the maximum has grown by more than
// 2^kSlack over it, so accumulators are rarely rescaled; weights are exp2(s - ref + kLift), which keeps those up to 2^-20 of
// the largest normal numbers when they are rounded to fp16 for the product, at most 2^(kLift + kSlack) = 2^14.  Their sum is
// taken before that rounding.  It is the only one to fewer than 32 bits in front of the result's: the matrix core takes both operands in
// 16 bits, and weights in two halves would double the second product.  It costs 2.6-2.9e-4 of the result against 64 bits instead of
// 2.1e-4.  A row whose reference value is beyond kChunkFar has its scores rounded before that is taken off (chunk_softmax).
//
// Masked places.  Scores out of sight are replaced, not added to, so their K may hold anything.  V rows behind the context
// are zeroed on the way in; a V row that some rows of the tile see and others must not, and that holds an infinity or NaN,
// would spread through the product as 0 * inf, so tiles at an edge of the mask are searched for such values, which are left out
// of the products and added to the results (chunk_add_not_finite).
//
// What it measured (MI355X; 32 query and 8 kv heads of 128 elements, pages of 128 tokens unless said otherwise):
//    4096 tokens over 32768 keys   1720-1820 us over the cards seen, 1.13-1.20 PFLOP/s (a library matrix product of 8192^3 reached
//                                  1.47): bound by the matrix core under the power limit (1.9 GHz; busy 0.59 of the cycles; the same
//                                  loop with the softmax left out takes 1250 us)
//    16 tokens over 131079 keys    98 us, 5.5 TB/s of K and V (a copy of 1 GiB reached 5.0 read and written): bound by HBM, 90 us,
//                                  and by joining partial results
//    24 sequences, 14 of one token and 10 of 253 to 470, window 1024, 16 + 16 heads of 80, pages of 16 tokens
//                                  87-90 us: 304 tiles and 224 single rows on 256 CUs, two rounds of about 40 us of 20 steps each,
//                                  because a tile has up to 256 rows whatever the batch
//    first prompts of 1000, 2000 and 4000 tokens   33, 58 and 140 us, 0.17, 0.38 and 0.64 of the library product's rate: 128, 256
//                                  and 512 tiles of that height on 256 CUs
//    4 sequences of 2 to 5 tokens over up to 704 keys   12.7 us: latency, four steps of about 1.2 us on 32 CUs between 3 us that
//                                  find and load the rows and 3 us that join and store them
#pragma once

#include <type_traits>

#include "aops_common.h"

namespace aops {

// Waves of a workgroup, 32 rows of a tile each: eight with 256 registers, or, for heads whose accumulators and operands take
// more, four with 512.
__host__ __device__ constexpr int chunk_waves(int head_dim) { return head_dim <= 128 ? 8 : 4; }
__host__ __device__ constexpr int chunk_rows(int head_dim) { return 32 * chunk_waves(head_dim); }
constexpr int kChunkUnit = 256;    // tokens per unit of the balanced partition
constexpr int kChunkWorth = 8;     // what cutting tiles costs, in units
constexpr int kChunkPlanHead = 4;  // ints in front of the plan: units per share
constexpr int kChunkMaxTiles = 1024;  // of the balanced partition
constexpr float kChunkNegBig = -1.0e30f;
constexpr float kChunkMaxScale = 0x1p56f;  // a score of up to 256 elements of fp16 (below 2^40) then stays above kChunkNegBig
constexpr float kChunkLog2e = 1.4426950408889634f;
constexpr float kChunkLn2 = 0.6931471805599453f;
constexpr float kChunkLift = 6.0f, kChunkSlack = 8.0f;
constexpr float kChunkFar = 1024.0f;  // up to here kChunkLift - ref is off by 2^-14 at most, a weight by an eighth of its rounding to fp16

struct ChunkArgs {
  const f16 *q, *key_cache, *value_cache;
  const int32_t *block_tables, *context_lens, *query_starts;
  f16* out;
  float* lse;            // may be null
  float *part_o, *part_ml;  // partial results: [kv head][2 * shares][part_rows][D] and [..][2]
  int32_t* plan;         // head; units in front of each tile (max_tiles + 1), sequence and number of each tile, tiles to join
  int32_t tokens, seqs, num_heads, num_kv_heads, group, block_size, max_pages, num_blocks, window;
  int32_t max_tiles, tile_rows, shares, part_rows;  // shares: of the balanced partition, per kv head; 0: one workgroup per tile
  uint32_t block_magic, block_shift;  // x / block_size = x * magic >> shift, x < 2^31
  float scale_log2;
};

// The arguments where the kernel was given them, to be read by scalar loads when they are needed.  chunk_reread: the same, but
// the compiler does not know, so what the end of a tile needs is not held in registers through its loop.
typedef const __attribute__((address_space(4))) ChunkArgs ChunkArgsMem;
typedef ChunkArgsMem& ChunkArgsRef;
__device__ __forceinline__ ChunkArgsRef chunk_args() { return *(ChunkArgsMem*)__builtin_amdgcn_kernarg_segment_ptr(); }
__device__ __forceinline__ ChunkArgsRef chunk_reread(ChunkArgsRef a) {
  ChunkArgsMem* p = &a;
  asm volatile("" : "+s"(p));
  return *p;
}

// A tile: rows row0 + rows - 1 of sequence b's (token, head) rows.
struct ChunkTile {
  int b, q0, row0, rows;
  bool alone;           // the only one of its sequence
  int p_first, p_last;  // positions of its first and last row's tokens (may be negative: sees nothing)
  int ctx;              // keys there are
  int lo, hi;           // keys seen by any of its rows
  int unit0, units;     // in units of kChunkUnit tokens, at least one
};

// First row and number of rows between two bounds.
__device__ __forceinline__ void chunk_rows_between(ChunkArgsRef a, int start, int end, int& q0, int& n) {
  q0 = min(max(start, 0), a.tokens);
  n = min(max(end, q0), a.tokens) - q0;
}

__device__ __forceinline__ void chunk_seq(ChunkArgsRef a, int b, int& q0, int& n) {
  chunk_rows_between(a, a.query_starts[b], a.query_starts[b + 1], q0, n);
}

__device__ __forceinline__ int chunk_tiles(ChunkArgsRef a, int n) {
  return (n * a.group + a.tile_rows - 1) >> __builtin_ctz(a.tile_rows);  // (a power of two)
}

// First key that the row at position p sees through the window (a row at a negative position sees nothing anyway).
__device__ __forceinline__ int chunk_window_start(int p, int window) { return max(p, 0) - window + 1; }

__device__ __forceinline__ ChunkTile chunk_geometry(ChunkArgsRef a, int b, int index) {
  ChunkTile t;
  int n;
  t.b = b;
  chunk_seq(a, b, t.q0, n);
  // the sequence's rows in even tiles (whole waves of 32): a nearly empty last one would take as long as a full one
  const int tiles = chunk_tiles(a, n), per = ((n * a.group + tiles - 1) / tiles + 31) & ~31;
  t.alone = tiles == 1;
  t.row0 = index * per;
  t.rows = min(n * a.group - t.row0, per);
  const int len = max(a.context_lens[b], 0);
  t.ctx = (int)min((int64_t)len, (int64_t)a.max_pages * a.block_size);
  t.p_first = len - n + t.row0 / a.group;
  t.p_last = len - n + (t.row0 + t.rows - 1) / a.group;
  t.lo = a.window > 0 ? min(max(chunk_window_start(t.p_first, a.window), 0), t.ctx) : 0;
  t.hi = min(max(t.p_last + 1, 0), t.ctx);
  t.unit0 = t.lo / kChunkUnit;
  t.units = max((t.hi - 1) / kChunkUnit + 1 - t.unit0, 1);
  return t;
}

// How a head of D elements is cut up for the matrix core.
template <int D>
struct ChunkDims {
  static_assert(D % 16 == 0 && D >= 16 && D <= 256, "head_dim: a multiple of 16 up to 256");
  static constexpr int kFull = D / 32;         // slices of 32 d of the score product
  static constexpr int kTail = (D % 32) / 16;  // and a half slice: 16 d in the lanes kg < 2, zeros in the others, in Q and K
  static constexpr int kSlices = kFull + kTail;
  static constexpr int kBlocks = D / 16;       // chunks of the cache, blocks of 16 d of O^T
  static constexpr int kWaves = chunk_waves(D), kThreads = kWaves * kWave;
  static constexpr int kTile = D <= 176 ? 64 : 32;        // tokens of a shared tile: what LDS has room for
  static constexpr int kStreamBlocks = 2;                 // column blocks of the stream path
  static constexpr int kStages = 16 * kTile * D <= 128 * 1024 ? 4 : 3;  // tiles of K, and of V, in LDS
  static constexpr int kPagesLds = kThreads * 4 * 4;      // page numbers of the tokens that a thread copies, four tiles
  static constexpr int kLds = 2 * kStages * kTile * D * 2 + kPagesLds;
  static constexpr int kStreamLds = kWaves * 32 * D * 2;
  static constexpr int kJoinBlocks = 4;                   // blocks of O^T joined at a time: 64 KiB of LDS, or 32
  static constexpr int kJoinLds = kWaves * 16 * kStreamBlocks * kJoinBlocks * 16 * 4;
  static constexpr int kMain = kLds > kStreamLds ? (kLds > kJoinLds ? kLds : kJoinLds) : (kStreamLds > kJoinLds ? kStreamLds : kJoinLds);
  static constexpr int kSmall = 2 * kWaves * 32 * 4 + 16;         // joined maxima and sums, flags
  static constexpr int kPlan = (3 * kChunkMaxTiles + 1 + kThreads + kWaves) * 4;
  static_assert(kMain + kSmall + kPlan <= 160 * 1024, "LDS of a CU");
};

__device__ __forceinline__ uint32_t chunk_lds_address(const void* p) {
  return __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void*)p);
}

// 16 bytes per lane from memory to LDS, lane l's to to + 16 l.  M0 carries the address; nothing else in these kernels uses it.
// ONCE: of lines that nobody else will read, which need not stay in the caches.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
template <bool ONCE>
__device__ __forceinline__ void chunk_copy16(const f16* from, uint32_t to) {
  if constexpr (ONCE)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off nt" ::"s"(to), "v"(from) : "m0");
  else
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(to), "v"(from) : "m0");
}
__device__ __forceinline__ void chunk_copy4(const int32_t* from, uint32_t to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(to), "v"(from) : "m0");
}
#pragma clang diagnostic pop

// f(0), ..., f(N-1) with the numbers as types
template <int N, int I = 0, typename F>
__device__ __forceinline__ void chunk_for(F&& f) {
  if constexpr (I < N) {
    f(std::integral_constant<int, I>{});
    chunk_for<N, I + 1>(f);
  }
}

// All but the last N copies have arrived, and LDS reads and writes are done.
template <int N>
__device__ __forceinline__ void chunk_wait_copies() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
}
__device__ __forceinline__ void chunk_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

typedef __fp16 ChunkTr __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) ChunkTr ChunkTrLds;

__device__ __forceinline__ f16x4 chunk_read_tr(const f16* lds) {
  return __builtin_bit_cast(f16x4, __builtin_amdgcn_ds_read_tr16_b64_v4f16((ChunkTrLds*)lds));
}

// Maxima in assembly: fmaxf would first quiet each operand that comes from the matrix core or from assembly, an instruction
// more for each of them.
__device__ __forceinline__ float chunk_max3(float a, float b, float c) {
  asm("v_max3_f32 %0, %0, %1, %2" : "+v"(a) : "v"(b), "v"(c));
  return a;
}
__device__ __forceinline__ float chunk_max2(float a, float b) {
  asm("v_max_f32 %0, %0, %1" : "+v"(a) : "v"(b));
  return a;
}
// Largest of the four lanes n, n + 16, n + 32, n + 48, in all four, of two values.  (The swaps exchange halves and quarters of
// the wave between two registers; in assembly because the compiler folds the builtins' two results into one when both operands
// are the same value.  Their two wait states are part of it.)
__device__ __forceinline__ void chunk_max4(float& a, float& b) {
  float c = a, d = b;
  asm("s_nop 1\n\tv_permlane32_swap_b32 %0, %1\n\tv_permlane32_swap_b32 %2, %3" : "+v"(a), "+v"(c), "+v"(b), "+v"(d));
  a = chunk_max2(a, c), b = chunk_max2(b, d);
  c = a, d = b;
  asm("s_nop 1\n\tv_permlane16_swap_b32 %0, %1\n\tv_permlane16_swap_b32 %2, %3" : "+v"(a), "+v"(c), "+v"(b), "+v"(d));
  a = chunk_max2(a, c), b = chunk_max2(b, d);
}
__device__ __forceinline__ float chunk_sum4(float x) {
  x += __shfl_xor(x, 16);
  return x + __shfl_xor(x, 32);
}

// Zero times a number is zero, times an infinity or NaN it is NaN.
__device__ __forceinline__ bool chunk_not_finite(f16x8 v) {
  const f16x2 zero = {0, 0};
  f16x2 z = __builtin_shufflevector(v, v, 0, 1) * zero;
  z += __builtin_shufflevector(v, v, 2, 3) * zero;
  z += __builtin_shufflevector(v, v, 4, 5) * zero;
  z += __builtin_shufflevector(v, v, 6, 7) * zero;
  const f16 both = z[0] + z[1];
  return both != both;
}

// Offset (in halfs) of token tok of the tile's sequence, from the start of the cache's kv head 0; entries outside the cache
// read the nearest page.
__device__ __forceinline__ int chunk_block(ChunkArgsRef a, int tok) {
  return (int)((uint64_t)(uint32_t)tok * a.block_magic >> a.block_shift);  // tok / block_size
}
__device__ __forceinline__ int64_t chunk_page_offset(ChunkArgsRef a, int entry, int tok, int blk, int64_t page_elems) {
  return min(max(entry, 0), a.num_blocks - 1) * page_elems + (int64_t)(tok - blk * a.block_size) * 16;
}
__device__ __forceinline__ int64_t chunk_token_offset(ChunkArgsRef a, const int32_t* table, int tok, int64_t page_elems) {
  const int blk = chunk_block(a, tok);
  return chunk_page_offset(a, table[blk], tok, blk, page_elems);
}

template <int D, int CB>
struct ChunkState {
  f32x4 o[CB][ChunkDims<D>::kBlocks];  // O^T: lane (row n, kg), element i <-> d = 16 block + 4kg + i
  float ref[CB];                       // reference value of the row's weights, log2 units
  float sum[CB];                       // this lane's share of the sum of weights
  uint64_t far;                        // not 0: a row of the wave has its reference value far from zero
};

template <int D, int CB>
struct ChunkQuery {
  f16x8 d[CB][ChunkDims<D>::kSlices];
  int pos[CB];  // position of this lane's row; a row that is none: -1
};

template <int D, int CB>
__device__ __forceinline__ void chunk_load_query(ChunkArgsRef a, const ChunkTile& t, int head, int first_row, int n, int kg,
                                                 ChunkQuery<D, CB>& q) {
  using Dims = ChunkDims<D>;
#pragma unroll
  for (int c = 0; c < CB; ++c) {
    const int r = first_row + 16 * c + n;
    const bool live = r < t.rows;
    const int row = t.row0 + (live ? r : 0);
    const int token = row / a.group;
    q.pos[c] = live ? max(t.p_first + token - t.row0 / a.group, -1) : -1;
    const f16* src = a.q + ((int64_t)(t.q0 + token) * a.num_heads + head * a.group + (row - token * a.group)) * D;
    const f16x8 zero8 = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
    for (int s = 0; s < Dims::kSlices; ++s) {
      q.d[c][s] = zero8;
      if (live && (s < Dims::kFull || kg < 2)) q.d[c][s] = ld128(src + 32 * s + 8 * kg);
    }
  }
}

template <int D, int CB>
__device__ __forceinline__ void chunk_init(ChunkState<D, CB>& st) {
#pragma unroll
  for (int c = 0; c < CB; ++c) {
#pragma unroll
    for (int db = 0; db < ChunkDims<D>::kBlocks; ++db) st.o[c][db] = f32x4{0.f, 0.f, 0.f, 0.f};
    st.ref[c] = kChunkNegBig;
    st.sum[c] = 0.f;
  }
  st.far = 0;
}

// Scores out of sight become -inf.  Lane (row n, kg) has tokens token0 + 16g + 4kg + i.
template <int CB, int KG>
__device__ __forceinline__ void chunk_mask(f32x4 (&s)[CB][KG], const int (&pos)[CB], int token0, int ctx, int window, int kg) {
#pragma unroll
  for (int c = 0; c < CB; ++c) {
    const int last = min(pos[c], ctx - 1), first = window > 0 ? max(pos[c] - window + 1, 0) : 0;
    const bool any = last >= first;
    // tokens first .. last, in one unsigned comparison; where there are none, no token
    const uint32_t span = any ? (uint32_t)(last - first) : 0u;
    const uint32_t at = any ? (uint32_t)(token0 + 4 * kg - first) : 0x40000000u;
#pragma unroll
    for (int g = 0; g < KG; ++g)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (at + (16 * g + i) > span) s[c][g][i] = -__builtin_inff();
  }
}

// Scores as the matrix core left them.  Its results may be read only some wait states after it (four passes and a few); the
// compiler cannot tell for the assembly that reads them below, so the wait is part of handing them over.
template <int CB, int KG>
__device__ __forceinline__ void chunk_settle(f32x4 (&acc)[CB][KG]) {
  static_assert(CB == 2 && (KG == 2 || KG == 4), "operands are listed");
  if constexpr (KG == 4)
    asm volatile("s_nop 7" : "+v"(acc[0][0]), "+v"(acc[0][1]), "+v"(acc[0][2]), "+v"(acc[0][3]), "+v"(acc[1][0]), "+v"(acc[1][1]), "+v"(acc[1][2]), "+v"(acc[1][3]));
  else
    asm volatile("s_nop 7" : "+v"(acc[0][0]), "+v"(acc[0][1]), "+v"(acc[1][0]), "+v"(acc[1][1]));
}

// Online softmax over settled scores; returns the weights packed as P^T operands of 32 tokens each.
template <int D, int CB, int KG>
__device__ __forceinline__ void chunk_softmax(f32x4 (&s)[CB][KG], float scale, ChunkState<D, CB>& st, f16x8 (&p)[CB][KG / 2]) {
  float top[CB];
  bool moved = false;
#pragma unroll
  for (int c = 0; c < CB; ++c) {
    float m[2];  // two chains: a wave computes its softmax alone on its SIMD's vector unit
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      m[h] = chunk_max3(s[c][h][0], s[c][h][1], s[c][h][2]);
      if constexpr (KG == 4) {
        m[h] = chunk_max3(m[h], s[c][h][3], s[c][h + 2][0]);
        m[h] = chunk_max3(m[h], s[c][h + 2][1], s[c][h + 2][2]);
      }
    }
    m[0] = chunk_max3(m[0], s[c][KG - 2][3], s[c][KG - 1][3]);
    top[c] = chunk_max2(m[0], m[1]);
  }
  chunk_max4(top[0], top[1]);
#pragma unroll
  for (int c = 0; c < CB; ++c) {
    top[c] *= scale;
    moved |= top[c] > st.ref[c] + kChunkSlack;
  }
  if (__builtin_amdgcn_ballot_w64(moved)) {
#pragma unroll
    for (int c = 0; c < CB; ++c) {
      const float ref = fmaxf(st.ref[c], top[c]);
      const float alpha = __builtin_amdgcn_exp2f(st.ref[c] - ref);
      st.ref[c] = ref;
      st.sum[c] *= alpha;
#pragma unroll
      for (int db = 0; db < ChunkDims<D>::kBlocks; ++db)
#pragma unroll
        for (int i = 0; i < 4; ++i) st.o[c][db][i] *= alpha;
    }
    bool far = false;
#pragma unroll
    for (int c = 0; c < CB; ++c) far |= __builtin_fabsf(st.ref[c]) > kChunkFar && st.ref[c] > kChunkNegBig;
    st.far = __builtin_amdgcn_ballot_w64(far);
  }
  // A weight is exp2(s scale + (kChunkLift - ref)), with one rounding of the bracket and one of the sum: where the reference value is
  // so large that these are not small, the score is rounded first, as the reference value was, so that the largest one's distance
  // from it is what it is, down to 0 (else scores of 2^25 and more left infinite weights, or none).
  float base[CB];
#pragma unroll
  for (int c = 0; c < CB; ++c) base[c] = kChunkLift - st.ref[c];
  if (__builtin_expect(st.far != 0, 0)) {
#pragma clang fp contract(off)
#pragma unroll
    for (int c = 0; c < CB; ++c) {
      base[c] = kChunkLift;
#pragma unroll
      for (int g = 0; g < KG; ++g)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[c][g][i] = s[c][g][i] * scale - st.ref[c];
    }
    scale = 1.0f;
  }
#pragma unroll
  for (int c = 0; c < CB; ++c) {
    float sum[KG];
#pragma unroll
    for (int g = 0; g < KG; ++g) {
#pragma unroll
      for (int i = 0; i < 4; ++i) s[c][g][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[c][g][i], scale, base[c]));
      sum[g] = (s[c][g][0] + s[c][g][1]) + (s[c][g][2] + s[c][g][3]);
    }
    float all = KG == 4 ? (sum[0] + sum[1]) + (sum[KG - 2] + sum[KG - 1]) : sum[0] + sum[1];
    asm volatile("" : "+v"(all));  // added up here, not when the registers of all the weights have been held for long
    st.sum[c] += all;
#pragma unroll
    for (int h = 0; h < KG / 2; ++h)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        p[c][h][i] = (f16)s[c][2 * h][i];
        p[c][h][4 + i] = (f16)s[c][2 * h + 1][i];
      }
  }
}

// O^T += V^T . P^T for 16 * KG tokens of a V tile in LDS whose chunks are `stride` halfs apart; v: this wave's first token.
template <int D, int CB, int KG>
__device__ __forceinline__ void chunk_pv(const f16* v, int stride, int lane, const f16x8 (&p)[CB][KG / 2], ChunkState<D, CB>& st) {
#pragma unroll
  for (int h = 0; h < KG / 2; ++h)
#pragma unroll
    for (int db = 0; db < ChunkDims<D>::kBlocks; ++db) {
      const f16* at = v + db * stride + 2 * h * 256 + lane * 4;
      const f16x4 lo = chunk_read_tr(at), hi = chunk_read_tr(at + 256);
      const f16x8 vt = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
      for (int c = 0; c < CB; ++c) st.o[c][db] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vt, p[c][h], st.o[c][db], 0, 0, 0);
    }
}

// v with zeros in the place of infinities and NaN
__device__ __forceinline__ f16x8 chunk_finite(f16x8 v) {
  u32x4 u = __builtin_bit_cast(u32x4, v);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if ((u[i] & 0x7c00u) == 0x7c00u) u[i] &= 0xffff0000u;
    if ((u[i] & 0x7c000000u) == 0x7c000000u) u[i] &= 0x0000ffffu;
  }
  return __builtin_bit_cast(f16x8, u);
}

// Where a row's result goes: the outputs (part < 0) or slot `part` of the partial results.
template <int D>
__device__ __forceinline__ int64_t chunk_out_row(ChunkArgsRef a, const ChunkTile& t, int head, int r) {
  const int row = t.row0 + r, token = row / a.group;
  return (int64_t)(t.q0 + token) * a.num_heads + head * a.group + (row - token * a.group);
}
__device__ __forceinline__ int64_t chunk_part_row(ChunkArgsRef a, int head, int part, int r) {
  return ((int64_t)head * 2 * a.shares + part) * a.part_rows + r;
}
// log-sum-exp (natural) of weights exp2(s - ref + kChunkLift) that add up to sum
__device__ __forceinline__ float chunk_lse(float ref, float sum) {
  return sum > 0.f || sum != sum ? (ref - kChunkLift + __builtin_amdgcn_logf(sum)) * kChunkLn2 : -__builtin_inff();
}

// Rows that see only a part of the `width` tokens from token0 on: those in front of the last of them, those whose window begins
// behind the first; and tokens behind the context.
__device__ __forceinline__ bool chunk_at_edge(ChunkArgsRef a, int token0, int width, int p_first, int p_last, int ctx) {
  return token0 + width - 1 > p_first || token0 + width > ctx ||
         (a.window > 0 && token0 < chunk_window_start(p_last, a.window));
}

// Adds to results that have been stored what their rows see of infinities and NaN in V at the edges, where these were left out
// of the products.  Rare, and outside of the loops, whose registers it must not cost: a thread takes an element of the head.
template <int D>
__device__ void chunk_add_not_finite(ChunkArgsRef a, const ChunkTile& t, int head, int k0, int k1, int width, int part) {
  __syncthreads();  // the results are stored
  const int64_t page_elems = (int64_t)a.num_kv_heads * D * a.block_size;
  const int32_t* table = a.block_tables + (int64_t)t.b * a.max_pages;
  for (int d = threadIdx.x; d < D; d += ChunkDims<D>::kThreads)
    for (int tok = k0; tok < k1; ++tok) {
      if (!chunk_at_edge(a, k0 + (tok - k0) / width * width, width, t.p_first, t.p_last, t.ctx)) continue;
      const f16 v = a.value_cache[chunk_token_offset(a, table, tok, page_elems) + ((int64_t)head * D + d / 16 * 16) * a.block_size + d % 16];
      if ((__builtin_bit_cast(uint16_t, v) & 0x7c00u) != 0x7c00u) continue;
      for (int r = 0; r < t.rows; ++r) {
        const int p = t.p_first + (t.row0 + r) / a.group - t.row0 / a.group;
        if (tok > p || (a.window > 0 && tok <= p - a.window)) continue;
        if (part < 0) {
          f16* o = a.out + chunk_out_row<D>(a, t, head, r) * D + d;
          *o = (f16)((float)*o + (float)v);
        } else {
          a.part_o[chunk_part_row(a, head, part, r) * D + d] += (float)v;
        }
      }
    }
}

// Keys k0 .. k1-1 (k0 a multiple of the tile) for a tile of many rows.  ONCE: no other tile reads these keys.  SPLIT, for at most
// half of the rows that a tile may have: the second half of the waves has the rows of the first one again, and every wave takes
// one half of each tile's keys.
template <int D, bool ONCE, bool SPLIT>
__device__ __forceinline__ void chunk_run_tile(ChunkArgsRef a, const ChunkTile& t, int head, int k0, int k1, int part,
                                               unsigned char* lds, int* flags) {
  using Dims = ChunkDims<D>;
  constexpr int KT = Dims::kTile, KG = KT / (SPLIT ? 32 : 16), CB = 2;  // KG: a wave's groups of 16 keys per tile
  constexpr int kRowWaves = Dims::kWaves / (SPLIT ? 2 : 1);
  constexpr int kPieces = 2 * KT;                       // 16-byte pieces of one chunk of a tile
  constexpr int kStep = Dims::kThreads / kPieces;       // chunks per round of the workgroup
  constexpr int kRounds = (Dims::kBlocks + kStep - 1) / kStep;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int lane = threadIdx.x & (kWave - 1), n = lane & 15, kg = lane >> 4;
  const int first_row = 32 * (wave % kRowWaves);
  const int key0 = wave / kRowWaves * (KT / 2);  // first key of a tile that is this wave's (not SPLIT: 0)
  const bool live = first_row < t.rows;

  ChunkQuery<D, CB> q;
  ChunkState<D, CB> st;
  chunk_load_query<D, CB>(a, t, head, first_row, n, kg, q);
  chunk_init<D, CB>(st);
  const int wp_first = t.p_first + ((t.row0 + first_row) / a.group - t.row0 / a.group);
  const int wp_last = t.p_first + ((t.row0 + min(first_row + 31, t.rows - 1)) / a.group - t.row0 / a.group);

  // Copies: this thread's 16-byte pieces are piece threadIdx.x of every kStep chunks, all of one token.
  const int my_token = (threadIdx.x >> 1) & (KT - 1), my_chunk = __builtin_amdgcn_readfirstlane(threadIdx.x / kPieces);
  const int64_t page_elems = (int64_t)a.num_kv_heads * D * a.block_size;
  const int64_t chunk_elems = (int64_t)a.block_size * 16;
  const int64_t lane_off = (int64_t)head * D * a.block_size + (threadIdx.x & 1) * 8 + my_chunk * chunk_elems;
  const int32_t* table = a.block_tables + (int64_t)t.b * a.max_pages;
  f16* const k_ring = reinterpret_cast<f16*>(lds);
  f16* const v_ring = k_ring + Dims::kStages * KT * D;
  const uint32_t lds_base = chunk_lds_address(lds);
  const uint32_t k_to = lds_base + wave * (kWave * 16), v_to = k_to + Dims::kStages * KT * D * 2;  // this wave's pieces of a tile
  auto token_of = [&](int tile) { return min(k0 + tile * KT + my_token, t.ctx - 1); };
  // Page numbers come through LDS too (a wave's own, tile i in slot i % 4): waiting for an ordinary load would be waiting for all
  // copies issued in front of it.
  constexpr int kPagesAt = Dims::kLds - Dims::kPagesLds;
  const int32_t* const my_pages = reinterpret_cast<const int32_t*>(lds + kPagesAt) + wave * (4 * kWave);
  auto copy_page = [&](int tile) { chunk_copy4(table + chunk_block(a, token_of(tile)), lds_base + kPagesAt + wave * (4 * kWave * 4) + (tile & 3) * (kWave * 4)); };
  auto offset_of = [&](int tile) {
    const int tok = token_of(tile);
    return chunk_page_offset(a, my_pages[(tile & 3) * kWave + lane], tok, chunk_block(a, tok), page_elems) + lane_off;
  };
  auto copy_round = [&](const f16* cache, int64_t off, uint32_t ring, int slot, int r) {
    if ((Dims::kBlocks % kStep == 0) || my_chunk + r * kStep < Dims::kBlocks)
      chunk_copy16<ONCE>(cache + off + r * kStep * chunk_elems, ring + slot * (KT * D * 2) + r * (Dims::kThreads * 16));
  };
  auto copy = [&](const f16* cache, int64_t off, uint32_t ring, int slot) {
#pragma unroll
    for (int r = 0; r < kRounds; ++r) copy_round(cache, off, ring, slot, r);
  };
  // V rows behind the context become zeros, infinities and NaN at an edge too (and are noted): by the thread that copied them
  auto patch = [&](int tile, int slot) {
    const int kt = k0 + tile * KT;
    if (!chunk_at_edge(a, kt, KT, t.p_first, t.p_last, t.ctx)) return;
    const bool beyond = kt + my_token >= t.ctx;
#pragma unroll
    for (int r = 0; r < kRounds; ++r)
      if ((Dims::kBlocks % kStep == 0) || my_chunk + r * kStep < Dims::kBlocks) {
        f16* at = v_ring + slot * KT * D + (threadIdx.x + r * Dims::kThreads) * 8;
        const f16x8 x = ld128(at);
        const bool bad = chunk_not_finite(x);
        if (beyond) st128(at, f16x8{0, 0, 0, 0, 0, 0, 0, 0});
        if (bad && !beyond) {
          st128(at, chunk_finite(x));
          flags[0] = 1;
        }
      }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // written before the barrier that follows, which waits for nothing itself
  };

  // A step is work for the matrix core (P V of the tile before, then the scores of this one) and then for the vector units (the
  // softmax), with one barrier: waves 0-3 meet it behind their softmax, waves 4-7, which share their SIMDs with these, behind
  // their products, so that they run half a step behind them: while one wave of a SIMD keeps the matrix core busy the other one
  // computes weights (4096 tokens over 32768 keys: 1787 us, 1883 with a barrier behind each half, 2935 in a first
  // version, whose waves all did the same at the same time).
  // K and V go straight to LDS, in rings of n = kStages tiles each.  At the start of its step for tile j a wave issues its copies
  // for K(j+n-1) and V(j+n-2), into the slots of K(j-1) and V(j-2), which all waves have read in front of the barrier that they
  // met last, and for the page numbers of tile j+2n-2.  In front of its barrier it waits for all but those of the last n-2
  // tiles: K(j+1) and V(j), which waves read in their step j+1, and the page numbers of tile j+n, read at that step's start, have then
  // arrived.
  // The copies are assembly that the compiler does not count (it would turn every wait for an LDS read into a wait for all of
  // them); a wave issues at least kCopies per tile.
  constexpr int kAhead = Dims::kStages - 1, kCopies = 2 * (Dims::kBlocks / kStep) + 1;
  const int tiles = k0 < k1 ? (k1 - k0 + KT - 1) / KT : 0;
  const bool second = wave >= 4;
  __syncthreads();  // the last item's reads of LDS are done
  if (threadIdx.x == 0) flags[0] = 0;
  int64_t off_v = 0;  // of V(j+n-2)
  for (int i = 0; i < min(tiles, kAhead); ++i) {
    off_v = chunk_token_offset(a, table, token_of(i), page_elems) + lane_off;
    copy(a.key_cache, off_v, k_to, i);
    if (i + 1 < kAhead) copy(a.value_cache, off_v, v_to, i);
  }
  for (int i = kAhead; i < min(tiles, 2 * kAhead); ++i) copy_page(i);
  chunk_wait_copies<0>();
  chunk_barrier();

  f16x8 p[CB][KG / 2];
  int j = 0, slot = 0, last_slot = Dims::kStages - 1;  // of K(j) and V(j), and of K(j-1) and V(j-1)
  constexpr int kFragments = Dims::kBlocks * (KG / 2) + Dims::kSlices * KG;  // of a step
  constexpr int kEvery = kFragments >= 4 * kRounds + 4 ? 2 : 1;              // a copy behind each so many-th
  const f16* const k_lane = k_ring + (kg >> 1) * KT * 16 + (key0 + n) * 16 + (kg & 1) * 8;  // fragment s, group g: + s * 2 * KT * 16 + g * 256
  const f16* const k_half = k_ring + Dims::kFull * 2 * KT * 16 + (key0 + n) * 16 + (kg & 1) * 8;
  const f16* const v_lane = v_ring + key0 * 16 + lane * 4;
  // steady: in the middle of an item, where every step issues all of its copies; inner: where no row's view begins or ends
  auto step = [&](auto pv, auto score, auto steady, auto inner) {
    constexpr bool kPv = decltype(pv)::value, kScore = decltype(score)::value, kSteady = decltype(steady)::value;
    constexpr bool kInner = decltype(inner)::value;
    // slot j+n-1 = slot j-1; slot j+n-2 = slot j-2
    const int v_slot = last_slot > 0 ? last_slot - 1 : kAhead;
    if constexpr (!kSteady) {
      if (j + kAhead - 1 < tiles) copy(a.value_cache, off_v, v_to, v_slot);
      if (j + kAhead < tiles) {
        off_v = offset_of(j + kAhead);
        copy(a.key_cache, off_v, k_to, last_slot);
        copy_page(j + 2 * kAhead);  // (behind the last tile: of the last token, and not used)
      }
    }
    const int kt = k0 + j * KT + key0;
    f32x4 acc[CB][KG];
    // Fragments of V (two reads each), then of K (one), each for CB products; a fragment is read kRing fragments before its
    // products, and a steady step issues a copy behind every second one (or, if they are too few, every one), where the matrix core
    // is busy.  The order is the one written here: left to itself the compiler reads each fragment right in front of its products and waits for LDS, and
    // copies in front of them all would leave the matrix core idle.
    constexpr int kRing = 4, kV = kPv ? Dims::kBlocks * (KG / 2) : 0, kK = kScore ? Dims::kSlices * KG : 0;
    f16x8 ring[kRing];
    const int v_at = last_slot * KT * D, k_at = slot * KT * D;
    auto read = [&](auto at) {
      constexpr int I = decltype(at)::value;
      if constexpr (I < kV) {
        const f16* from = v_lane + v_at + (I % Dims::kBlocks) * KT * 16 + 2 * (I / Dims::kBlocks) * 256;
        const f16x4 lo = chunk_read_tr(from), hi = chunk_read_tr(from + 256);
        ring[I % kRing] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
      } else if constexpr (I < kV + kK) {
        constexpr int S = (I - kV) / KG, G = (I - kV) % KG;
        ring[I % kRing] = ld128((S < Dims::kFull ? k_lane + S * 2 * KT * 16 : k_half) + k_at + G * 256);
      }
    };
    auto products = [&](auto at) {
      constexpr int I = decltype(at)::value;
      if constexpr (I < kV) {
#pragma unroll
        for (int c = 0; c < CB; ++c)
          st.o[c][I % Dims::kBlocks] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ring[I % kRing], p[c][I / Dims::kBlocks], st.o[c][I % Dims::kBlocks], 0, 0, 0);
      } else {
        constexpr int S = (I - kV) / KG, G = (I - kV) % KG;
        f16x8 kf = ring[I % kRing];
        if constexpr (S >= Dims::kFull)
          if (kg >= 2) kf = f16x8{0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
        for (int c = 0; c < CB; ++c)
          acc[c][G] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, q.d[c][S], S > 0 ? acc[c][G] : f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
      }
    };
    auto copies = [&](auto at) {
      constexpr int I = decltype(at)::value;
      if constexpr (kSteady && I % kEvery == kEvery - 1) {
        constexpr int R = I / kEvery;
        if constexpr (R < kRounds) copy_round(a.value_cache, off_v, v_to, v_slot, R);
        if constexpr (R == kRounds) off_v = offset_of(j + kAhead);
        if constexpr (R > kRounds && R <= 2 * kRounds) copy_round(a.key_cache, off_v, k_to, last_slot, R - kRounds - 1);
        if constexpr (R == 2 * kRounds + 1) copy_page(j + 2 * kAhead);
      }
    };
    __builtin_amdgcn_s_setprio(1);
    chunk_for<kRing>([&](auto i) { read(i); });
    __builtin_amdgcn_sched_barrier(0);
    chunk_for<kV + kK>([&](auto i) {
      products(i);
      copies(i);
      read(std::integral_constant<int, decltype(i)::value + kRing>{});
      __builtin_amdgcn_sched_barrier(0);
    });
    if constexpr (kScore) chunk_settle<CB, KG>(acc);
    __builtin_amdgcn_s_setprio(0);
    if (kSteady || j + kAhead < tiles) {
      chunk_wait_copies<(kAhead - 1) * kCopies>();
    } else {
      chunk_wait_copies<0>();
    }
    if (!kInner && j < tiles) patch(j, slot);
    if (second) chunk_barrier();
    if constexpr (kScore) {
      if (!kInner && chunk_at_edge(a, kt, 16 * KG, wp_first, wp_last, t.ctx)) chunk_mask<CB, KG>(acc, q.pos, kt, t.ctx, a.window, kg);
      chunk_softmax<D, CB, KG>(acc, a.scale_log2, st, p);
    }
    if (!second) chunk_barrier();
    ++j;
    last_slot = slot;
    slot = slot < kAhead ? slot + 1 : 0;
  };
  // A wave computes where one of its rows sees a tile, and only helps with the copies in front of that and behind it: loops of
  // their own, because accumulators changed under a condition inside a loop are copied in it.
  const std::true_type yes;
  const std::false_type no;
  const int w_first = a.window > 0 ? max(chunk_window_start(wp_first, a.window) - k0, 0) / KT : 0;
  const int w_end = live && wp_last >= k0 ? min(tiles, (wp_last - k0) / KT + 1) : 0;
  while (j <= tiles && j < min(w_first, w_end)) step(no, no, no, no);
  if (j < w_end) {
    step(no, yes, no, no);
    const int inner = a.window > 0 ? (max(chunk_window_start(t.p_last, a.window) - k0, 0) + KT - 1) / KT : 0;
    const int outer = max(min(t.p_first + 1, t.ctx) - k0, 0) / KT, steady = min(w_end, tiles - kAhead);
    if constexpr (kFragments >= 2 * kRounds + 2) {  // (else no room for all copies)
      while (j < min(steady, inner)) step(yes, yes, yes, no);
      while (j < min(steady, outer)) step(yes, yes, yes, yes);
      while (j < steady) step(yes, yes, yes, no);
    }
    while (j < w_end) step(yes, yes, no, no);
    step(yes, no, no, no);
  }
  while (j <= tiles) step(no, no, no, no);

  ChunkArgsRef e = chunk_reread(a);
  static_assert(!SPLIT || (KG == 2 && kRowWaves * CB * (Dims::kBlocks + 1) * kWave * 16 <= Dims::kMain), "halves of a tile, and room");
  if constexpr (SPLIT) {  // the second half's results join those of the wave with the same rows
    f32x4* const out = reinterpret_cast<f32x4*>(lds) + (wave % kRowWaves) * (CB * (Dims::kBlocks + 1) * kWave) + lane;
    __syncthreads();  // the last tile has been read
    if (wave >= kRowWaves) {
#pragma unroll
      for (int c = 0; c < CB; ++c) {
#pragma unroll
        for (int db = 0; db < Dims::kBlocks; ++db) out[(c * (Dims::kBlocks + 1) + db) * kWave] = st.o[c][db];
        out[(c * (Dims::kBlocks + 1) + Dims::kBlocks) * kWave] = f32x4{st.ref[c], st.sum[c], 0.f, 0.f};
      }
    }
    __syncthreads();
    if (wave < kRowWaves) {
#pragma unroll
      for (int c = 0; c < CB; ++c) {
        const f32x4 other = out[(c * (Dims::kBlocks + 1) + Dims::kBlocks) * kWave];
        const float ref = fmaxf(st.ref[c], other[0]);
        const float mine = __builtin_amdgcn_exp2f(st.ref[c] - ref), theirs = __builtin_amdgcn_exp2f(other[0] - ref);
        st.ref[c] = ref;
        st.sum[c] = st.sum[c] * mine + other[1] * theirs;
#pragma unroll
        for (int db = 0; db < Dims::kBlocks; ++db) st.o[c][db] = st.o[c][db] * mine + out[(c * (Dims::kBlocks + 1) + db) * kWave] * theirs;
      }
    }
  }
#pragma unroll
  for (int c = 0; c < CB; ++c) {
    const int r = first_row + 16 * c + n;
    const float sum = chunk_sum4(st.sum[c]);
    if (r >= t.rows || (SPLIT && wave >= kRowWaves)) continue;
    if (part < 0) {
      const int64_t row = chunk_out_row<D>(e, t, head, r);
      const float inv = sum == 0.f ? 0.f : 1.0f / sum;
#pragma unroll
      for (int db = 0; db < Dims::kBlocks; ++db) {
        f16x4 v;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = (f16)(st.o[c][db][i] * inv);
        *reinterpret_cast<f16x4*>(e.out + row * D + 16 * db + 4 * kg) = v;
      }
      if (e.lse && kg == 0) e.lse[row] = chunk_lse(st.ref[c], sum);
    } else {
      const int64_t row = chunk_part_row(e, head, part, r);
#pragma unroll
      for (int db = 0; db < Dims::kBlocks; ++db)
        *reinterpret_cast<f32x4*>(e.part_o + row * D + 16 * db + 4 * kg) = st.o[c][db];
      if (kg == 0) {
        e.part_ml[2 * row] = st.ref[c];
        e.part_ml[2 * row + 1] = sum;
      }
    }
  }
  if (flags[0]) chunk_add_not_finite<D>(e, t, head, k0, k1, KT, part);
}

// Keys k0 .. k1-1 (k0 a multiple of the unit) for a tile of at most 16 * kStreamBlocks rows.
template <int D>
__device__ __forceinline__ void chunk_run_stream(ChunkArgsRef a, const ChunkTile& t, int head, int k0, int k1, int part,
                                                 unsigned char* lds, float* small) {
  using Dims = ChunkDims<D>;
  constexpr int CB = Dims::kStreamBlocks, KG = 2, kStep = 32 * Dims::kWaves;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int lane = threadIdx.x & (kWave - 1), n = lane & 15, kg = lane >> 4;
  ChunkQuery<D, CB> q;
  ChunkState<D, CB> st;
  chunk_load_query<D, CB>(a, t, head, 0, n, kg, q);
  chunk_init<D, CB>(st);
  const int64_t page_elems = (int64_t)a.num_kv_heads * D * a.block_size;
  const int64_t chunk_elems = (int64_t)a.block_size * 16;
  const int64_t head_off = (int64_t)head * D * a.block_size;
  const int32_t* table = a.block_tables + (int64_t)t.b * a.max_pages;
  f16* mine = reinterpret_cast<f16*>(lds) + wave * 32 * D;  // [chunk][32 tokens][16]
  __syncthreads();  // the last item's reads of LDS are done

  // K operand registers: token n of group g, d = 32s + 8kg ..+7.  V: 16-byte piece `lane` of every chunk's 32 tokens.
  f16x8 kreg[KG][Dims::kSlices], vreg[Dims::kBlocks];
  int64_t koff[KG], voff;
  auto offsets = [&](int token0) {
#pragma unroll
    for (int g = 0; g < KG; ++g)
      koff[g] = chunk_token_offset(a, table, min(token0 + 16 * g + n, t.ctx - 1), page_elems) + head_off;
    voff = chunk_token_offset(a, table, min(token0 + (lane >> 1), t.ctx - 1), page_elems) + head_off + (lane & 1) * 8;
  };
  auto load_k = [&]() {
#pragma unroll
    for (int g = 0; g < KG; ++g) {
      const f16* src = a.key_cache + koff[g] + (kg >> 1) * chunk_elems + (kg & 1) * 8;
#pragma unroll
      for (int s = 0; s < Dims::kSlices; ++s) {
        if (s < Dims::kFull) {
          kreg[g][s] = ld128_stream(src + 2 * s * chunk_elems);
        } else {
          kreg[g][s] = f16x8{0, 0, 0, 0, 0, 0, 0, 0};
          if (kg < 2) kreg[g][s] = ld128_stream(src + 2 * s * chunk_elems);
        }
      }
    }
  };
  auto load_v = [&]() {
#pragma unroll
    for (int db = 0; db < Dims::kBlocks; ++db) vreg[db] = ld128_stream(a.value_cache + voff + db * chunk_elems);
  };
  bool not_finite = false;
  int token0 = k0 + 32 * wave;
  if (token0 < k1) {
    offsets(token0);
    load_k();
    load_v();
  }
  for (; token0 < k1; token0 += kStep) {
    const bool more = token0 + kStep < k1;
    if (more) offsets(token0 + kStep);
    f32x4 acc[CB][KG];
#pragma unroll
    for (int c = 0; c < CB; ++c)
#pragma unroll
      for (int g = 0; g < KG; ++g) {
        acc[c][g] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < Dims::kSlices; ++s)
          acc[c][g] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kreg[g][s], q.d[c][s], acc[c][g], 0, 0, 0);
      }
    chunk_settle<CB, KG>(acc);
    if (more) load_k();
    const f16x8 zero8 = {0, 0, 0, 0, 0, 0, 0, 0};
    if (chunk_at_edge(a, token0, 32, t.p_first, t.p_last, t.ctx)) {
      chunk_mask<CB, KG>(acc, q.pos, token0, t.ctx, a.window, kg);
      bool bad = false;
#pragma unroll
      for (int db = 0; db < Dims::kBlocks; ++db) {
        if (token0 + (lane >> 1) >= t.ctx) vreg[db] = zero8;
        bad |= chunk_not_finite(vreg[db]);
        vreg[db] = chunk_finite(vreg[db]);
      }
      not_finite |= bad;
    }
#pragma unroll
    for (int db = 0; db < Dims::kBlocks; ++db) st128(mine + db * 512 + lane * 8, vreg[db]);
    if (more) load_v();
    f16x8 p[CB][KG / 2];
    chunk_softmax<D, CB, KG>(acc, a.scale_log2, st, p);
    chunk_pv<D, CB, KG>(mine, 512, lane, p, st);
  }

  // Join the waves: common reference and total of every row, then the accumulators, kJoinBlocks blocks of 16 d at a time.
  ChunkArgsRef e = chunk_reread(a);
  float* refs = small;                        // [wave][row]
  float* sums = small + Dims::kWaves * 32;
#pragma unroll
  for (int c = 0; c < CB; ++c) {
    const float sum = chunk_sum4(st.sum[c]);
    if (kg == 0) {
      refs[wave * 32 + 16 * c + n] = st.ref[c];
      sums[wave * 32 + 16 * c + n] = sum;
    }
  }
  const bool add_not_finite = __syncthreads_or(not_finite);
  float factor[CB];
#pragma unroll
  for (int c = 0; c < CB; ++c) {
    float ref = kChunkNegBig;
#pragma unroll
    for (int w = 0; w < Dims::kWaves; ++w) ref = fmaxf(ref, refs[w * 32 + 16 * c + n]);
    factor[c] = __builtin_amdgcn_exp2f(st.ref[c] - ref);
  }
  // [wave][row][four d], the groups of four d in an order that depends on the row: rows are as long as the banks are wide, so
  // the same group of 16 rows, which a wave writes together, would fall into the same banks (12.7 us instead of 15.6 for four
  // sequences of 2 to 5 tokens over up to 704 keys)
  f32x4* acc = reinterpret_cast<f32x4*>(lds);
  constexpr int kRow = Dims::kJoinBlocks * 4;
  static_assert((kRow & (kRow - 1)) == 0, "groups of a row are told apart by their bits");
  auto at = [&](int w, int r, int g) { return (w * (16 * CB) + r) * kRow + (g ^ (r & (kRow - 1))); };
  for (int db0 = 0; db0 < Dims::kBlocks; db0 += Dims::kJoinBlocks) {
    __syncthreads();  // LDS is free: V was read, or the blocks in front of these were joined
#pragma unroll
    for (int c = 0; c < CB; ++c)
      if (16 * c < t.rows)
#pragma unroll
        for (int db = 0; db < Dims::kBlocks; ++db)
          if (db >= db0 && db < db0 + Dims::kJoinBlocks) acc[at(wave, 16 * c + n, (db - db0) * 4 + kg)] = st.o[c][db] * factor[c];
    __syncthreads();
    const int width = min(Dims::kBlocks - db0, Dims::kJoinBlocks) * 4;  // groups of four d
    for (int i = threadIdx.x; i < t.rows * width; i += Dims::kThreads) {
      const int r = i / width, d4 = i - r * width;
      f32x4 v = {0.f, 0.f, 0.f, 0.f};
      float ref = kChunkNegBig, sum = 0.f;
#pragma unroll
      for (int w = 0; w < Dims::kWaves; ++w) {
        v += acc[at(w, r, d4)];
        ref = fmaxf(ref, refs[w * 32 + r]);
      }
#pragma unroll
      for (int w = 0; w < Dims::kWaves; ++w) sum += sums[w * 32 + r] * __builtin_amdgcn_exp2f(refs[w * 32 + r] - ref);
      const int d = db0 * 16 + 4 * d4;
      if (part < 0) {
        const int64_t row = chunk_out_row<D>(e, t, head, r);
        const float inv = sum == 0.f ? 0.f : 1.0f / sum;
        f16x4 o;
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] = (f16)(v[j] * inv);
        *reinterpret_cast<f16x4*>(e.out + row * D + d) = o;
        if (e.lse && d == 0) e.lse[row] = chunk_lse(ref, sum);
      } else {
        const int64_t row = chunk_part_row(e, head, part, r);
        *reinterpret_cast<f32x4*>(e.part_o + row * D + d) = v;
        if (d == 0) {
          e.part_ml[2 * row] = ref;
          e.part_ml[2 * row + 1] = sum;
        }
      }
    }
  }
  if (add_not_finite) chunk_add_not_finite<D>(e, t, head, k0, k1, 32, part);
}

template <int D>
__device__ __forceinline__ void chunk_run(ChunkArgsRef a, const ChunkTile& t, int head, int unit, int units, int part,
                                          unsigned char* lds, float* small) {
  const int k0 = (t.unit0 + unit) * kChunkUnit, k1 = min(t.hi, (t.unit0 + unit + units) * kChunkUnit);
  if (t.rows <= 16 * ChunkDims<D>::kStreamBlocks) {
    chunk_run_stream<D>(a, t, head, k0, k1, part, lds, small);
  } else {
    const int first = max(k0, t.lo / ChunkDims<D>::kTile * ChunkDims<D>::kTile);
    int* const flags = reinterpret_cast<int*>(small);
    // Keys that one tile reads go past the caches (64 rows over 131079 keys: 100 us instead of 112; those that four tiles
    // read 318 instead of 294).  Halves of the waves with a half of the keys each where a whole tile is one workgroup's, whose
    // time is that of its steps (16 sequences of 100 rows over 3000 keys, 8 heads: 60 us instead of 73), not where tiles are cut
    // and all CUs wait for memory (8 of 128 rows over 8000 keys: 84 us, not split 74-79).
    if (!t.alone) {
      chunk_run_tile<D, false, false>(a, t, head, first, k1, part, lds, flags);
      return;
    }
    if constexpr (ChunkDims<D>::kTile == 64) {
      if (part < 0 && t.rows <= chunk_rows(D) / 2) {
        chunk_run_tile<D, true, true>(a, t, head, first, k1, part, lds, flags);
        return;
      }
    }
    chunk_run_tile<D, true, false>(a, t, head, first, k1, part, lds, flags);
  }
}

// Sequence and number of tile `tile` (the same in all lanes), counting the sequences' tiles one after the other, PER sequences a
// lane at a time; false where there are fewer.  Every wave counts alone where its lanes suffice for all sequences; where not, the
// waves share them (8000 decoding sequences of 245 keys on average: 9.4 ms with 64 sequences at a time, 5.3 with 512, 2.7 so).
// `shared`: an int of LDS per wave and two more.
template <int PER, int WAVES>
__device__ __forceinline__ bool chunk_find(ChunkArgsRef a, int tile, int* shared, int& b, int& index) {
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const bool alone = a.seqs <= PER * kWave;
  int running = 0;  // tiles of the sequences in front
  for (uint32_t base = 0; base < (uint32_t)a.seqs; base += PER * kWave * WAVES) {
    const uint32_t own = base + (alone ? lane : threadIdx.x) * PER, first = min(own, (uint32_t)(a.seqs - PER));
    // A lane's bounds lie next to each other and are on their way at once (a pair for each sequence, under a condition of its own, was
    // waited for: 512 decoding sequences 169 us instead of 164, 8000 2.74 ms instead of 2.66).  The last lanes with sequences read the
    // last PER and leave out those in front of their own.
    int bounds[PER + 1], tiles[PER], mine = 0;
#pragma unroll
    for (int i = 0; i <= PER; ++i) bounds[i] = a.query_starts[first + i];
#pragma unroll
    for (int i = 0; i <= PER; ++i) asm volatile("" : "+v"(bounds[i]));  // (else the compiler moves the first load into a branch)
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      int q0, n;
      chunk_rows_between(a, bounds[i], bounds[i + 1], q0, n);
      tiles[i] = first + i >= own ? chunk_tiles(a, n) : 0;
      mine += tiles[i];
    }
    mine = min(mine, a.max_tiles);  // (bounds that overlap count tokens again and again: what is behind max_tiles is not looked for)
    int upto = mine;
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
      const int o = __shfl_up(upto, d);
      if (lane >= d) upto += o;
    }
    int in_front = running;
    if (!alone) {
      __syncthreads();
      if (lane == kWave - 1) shared[wave] = min(upto, a.max_tiles);
      __syncthreads();
#pragma unroll
      for (int w = 0; w < WAVES; ++w) {
        in_front += w < wave ? shared[w] : 0;
        running += shared[w];
      }
      in_front = __builtin_amdgcn_readfirstlane(in_front);
      running = __builtin_amdgcn_readfirstlane(running);
    }
    const uint64_t behind = __builtin_amdgcn_ballot_w64(in_front + upto > tile);
    if (behind && in_front <= tile) {
      int rest = tile - in_front - (upto - mine), i = 0;  // of this lane's tiles; meant where it is the first one behind
#pragma unroll
      for (int k = 0; k < PER - 1; ++k)
        if (i == k && rest >= tiles[k]) rest -= tiles[k], ++i;
      const int at = __builtin_ctzll(behind);
      b = __builtin_amdgcn_readlane((int)first + i, at);
      index = __builtin_amdgcn_readlane(rest, at);
      if (alone) return true;
      shared[WAVES] = b, shared[WAVES + 1] = index;
    }
    if (!alone && running > tile) {
      __syncthreads();
      b = shared[WAVES], index = shared[WAVES + 1];
      return true;
    }
  }
  return false;
}

// One workgroup per (tile, kv head), kv heads next to each other so that a kv head's tiles run on one XCD (or few) and share
// its K and V in that L2.  The last tiles of the sequences, which see the most keys, come first.
template <int D>
__global__ __launch_bounds__(ChunkDims<D>::kThreads, ChunkDims<D>::kWaves / 4) void chunk_tiles_kernel(ChunkArgs) {
  ChunkArgsRef a = chunk_args();
  extern __shared__ __attribute__((aligned(16))) unsigned char chunk_lds[];
  const int head = blockIdx.x % a.num_kv_heads;
  int b, index;
  float* small = reinterpret_cast<float*>(chunk_lds + ChunkDims<D>::kMain);
  const int tile = a.max_tiles - 1 - (int)(blockIdx.x / a.num_kv_heads);
  int* const shared = reinterpret_cast<int*>(small);
  constexpr int kWaves = ChunkDims<D>::kWaves;
  // (one sequence a lane is 0.5 us faster than eight for a few sequences)
  if (!(a.seqs <= kWave ? chunk_find<1, kWaves>(a, tile, shared, b, index) : chunk_find<8, kWaves>(a, tile, shared, b, index))) return;
  const ChunkTile t = chunk_geometry(a, __builtin_amdgcn_readfirstlane(b), __builtin_amdgcn_readfirstlane(index));
  chunk_run<D>(a, t, head, 0, t.units, -1, chunk_lds, small);
}

// The same where tiles may have to be cut, which depends on the lengths: every workgroup looks at all tiles first.  Either the
// tiles stay whole, and workgroup i of a kv head takes one of them; or their keys, in units of 256 tokens, are laid end to end
// and cut into `shares` equal shares per kv head, one for each of the CUs.  A tile inside one share is then written directly;
// of the others every share leaves a partial result, in slot 2w of share w if the tile began in front of the share and in slot
// 2w + 1 if it began in it, which chunk_merge_kernel joins in the order of the keys.  The shares take kChunkWorth units longer
// than the keys of an even distribution (30 us for full tiles: partial results, several tiles' starts and ends, the join), whole
// tiles as long as their longest, or as their average times the rounds that the CUs need for all.
template <int D>
__global__ __launch_bounds__(ChunkDims<D>::kThreads, ChunkDims<D>::kWaves / 4) void chunk_shares_kernel(ChunkArgs) {
  ChunkArgsRef a = chunk_args();
  using Dims = ChunkDims<D>;
  extern __shared__ __attribute__((aligned(16))) unsigned char chunk_lds[];
  float* small = reinterpret_cast<float*>(chunk_lds + Dims::kMain);
  int* before = reinterpret_cast<int*>(chunk_lds + Dims::kMain + Dims::kSmall);
  int* seq = before + kChunkMaxTiles + 1;
  int* number = seq + kChunkMaxTiles;
  int* starts = number + kChunkMaxTiles;  // first tile of each of kThreads sequences
  int* sums = starts + Dims::kThreads;    // of the waves
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const int head = blockIdx.x % a.num_kv_heads, index = blockIdx.x / a.num_kv_heads;
  int count = 0;  // tiles
  for (int64_t s0 = 0; s0 < a.seqs && count < a.max_tiles; s0 += Dims::kThreads) {
    int q0, n = 0;
    if (s0 + threadIdx.x < a.seqs) chunk_seq(a, (int)(s0 + threadIdx.x), q0, n);
    const int mine = chunk_tiles(a, n);
    int upto = mine;
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
      const int o = __shfl_up(upto, d);
      if (lane >= d) upto += o;
    }
    // (sums of bounds that overlap are cut off: nothing behind max_tiles is looked at)
    if (lane == kWave - 1) sums[wave] = min(upto, a.max_tiles);
    __syncthreads();
    int in_front = 0, total = 0;
#pragma unroll
    for (int w = 0; w < Dims::kWaves; ++w) {
      in_front += w < wave ? sums[w] : 0;
      total += sums[w];
    }
    starts[threadIdx.x] = min(in_front + upto - mine, total);
    __syncthreads();
    const int end = min(count + total, a.max_tiles);
    for (int tile = count + threadIdx.x; tile < end; tile += Dims::kThreads) {
      int k = 0;  // the last sequence that starts at or in front of the tile (those without tiles start with the next one)
#pragma unroll
      for (int step = Dims::kThreads / 2; step > 0; step >>= 1)
        if (starts[k + step] <= tile - count) k += step;
      seq[tile] = (int)s0 + k;
      number[tile] = tile - count - starts[k];
      before[tile + 1] = chunk_geometry(a, (int)s0 + k, tile - count - starts[k]).units;
    }
    count = end;
    __syncthreads();
  }
  if (threadIdx.x < kWave) {  // running sums
    int running = 0;
    if (lane == 0) before[0] = 0;
    for (int base = 0; base < count; base += kWave) {
      int upto = base + lane < count ? before[base + lane + 1] : 0;
#pragma unroll
      for (int d = 1; d < kWave; d <<= 1) {
        const int o = __shfl_up(upto, d);
        if (lane >= d) upto += o;
      }
      if (base + lane < count) before[base + lane + 1] = running + upto;
      running += __shfl(upto, kWave - 1);
    }
  }
  __syncthreads();
  count = __builtin_amdgcn_readfirstlane(count);
  if (count == 0) {  // no sequence has a token: nothing to do, and to join
    if (head == 0 && index < a.shares && threadIdx.x == 0) a.plan[kChunkPlanHead + 3 * a.max_tiles + 1 + index] = -1;
    return;
  }
  const int total = __builtin_amdgcn_readfirstlane(before[count]);
  const int share = (total + a.shares - 1) / a.shares;
  int longest = 0;
  for (int i = lane; i < count; i += kWave) longest = max(longest, before[i + 1] - before[i]);
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) longest = max(longest, __shfl_xor(longest, d));
  const int rounds = (count + a.shares - 1) / a.shares;
  const bool whole = __builtin_amdgcn_readfirstlane(max(longest, rounds * (total / count)) <= share + kChunkWorth);
  int tile, begin, end;
  if (whole) {
    tile = count - 1 - index;  // the last tiles of the sequences, which see the most keys, first
    begin = tile >= 0 ? before[tile] : 0;
    end = tile >= 0 ? before[tile + 1] : 0;
  } else {
    begin = (int)min((int64_t)index * share, (int64_t)total);
    end = index < a.shares ? min(begin + share, total) : begin;
    tile = 0;
#pragma unroll
    for (int step = kChunkMaxTiles / 2; step > 0; step >>= 1)  // the last tile that begins at or in front of `begin`
      if (tile + step < count && before[tile + step] <= begin) tile += step;
  }
  begin = __builtin_amdgcn_readfirstlane(begin);
  end = __builtin_amdgcn_readfirstlane(end);
  tile = __builtin_amdgcn_readfirstlane(tile);
  if (head == 0) {  // for the join: the plan, and for each share the tile that it continues, if it is the first one to do so
    if (index == 0) {
      for (int i = threadIdx.x; i <= count; i += Dims::kThreads) a.plan[kChunkPlanHead + i] = before[i];
      for (int i = threadIdx.x; i < count; i += Dims::kThreads) {
        a.plan[kChunkPlanHead + a.max_tiles + 1 + i] = seq[i];
        a.plan[kChunkPlanHead + 2 * a.max_tiles + 1 + i] = number[i];
      }
      if (threadIdx.x == 0) a.plan[0] = share;
    }
    if (index < a.shares && threadIdx.x == 0)
      a.plan[kChunkPlanHead + 3 * a.max_tiles + 1 + index] =
          !whole && begin < end && begin > before[tile] && before[tile] / share + 1 == index ? tile : -1;
  }
  while (begin < end) {
    const int from = __builtin_amdgcn_readfirstlane(before[tile]), to = __builtin_amdgcn_readfirstlane(before[tile + 1]);
    const int upto = min(end, to);
    const int part = begin == from && upto == to ? -1 : 2 * index + (begin == from ? 1 : 0);
    ChunkArgsRef e = chunk_reread(a);
    const ChunkTile t = chunk_geometry(e, __builtin_amdgcn_readfirstlane(seq[tile]), __builtin_amdgcn_readfirstlane(number[tile]));
    chunk_run<D>(e, t, head, begin - from, upto - begin, part, chunk_lds, small);
    begin = upto;
    ++tile;
  }
}

template <int D>
hipError_t chunk_launch(const ChunkArgs& a, hipStream_t stream) {
  using Dims = ChunkDims<D>;
  static std::atomic<uint64_t> tiles_done{0}, shares_done{0};
  if (a.shares > 0) {
    constexpr int lds = Dims::kMain + Dims::kSmall + Dims::kPlan;
    if (const hipError_t e = allow_dynamic_lds((const void*)chunk_shares_kernel<D>, lds, shares_done)) return e;
    chunk_shares_kernel<D><<<(unsigned)((a.shares > a.max_tiles ? a.shares : a.max_tiles) * a.num_kv_heads), Dims::kThreads, lds, stream>>>(a);
  } else {
    constexpr int lds = Dims::kMain + Dims::kSmall;
    if (const hipError_t e = allow_dynamic_lds((const void*)chunk_tiles_kernel<D>, lds, tiles_done)) return e;
    chunk_tiles_kernel<D><<<(unsigned)((int64_t)a.max_tiles * a.num_kv_heads), Dims::kThreads, lds, stream>>>(a);
  }
  return hipGetLastError();
}

#define AOPS_CHUNK_DIMS(X) \
  X(16) X(32) X(48) X(64) X(80) X(96) X(112) X(128) X(144) X(160) X(176) X(192) X(208) X(224) X(240) X(256)
#define AOPS_CHUNK_EXTERN(D) extern template hipError_t chunk_launch<D>(const ChunkArgs&, hipStream_t);

}  // namespace aops
