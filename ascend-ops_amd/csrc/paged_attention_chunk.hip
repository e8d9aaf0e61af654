// Entry points of the attention of a chunk of new tokens per sequence over the paged caches, the choice between the two
// partitions of its work, and the kernel that joins partial results.  The kernels proper: paged_attention_chunk.h.
#include <algorithm>

#include "paged_attention_chunk.h"

namespace aops {

AOPS_CHUNK_DIMS(AOPS_CHUNK_EXTERN)

// Joins the partial results of a tile, in the order of their keys, whatever order they were made in: a wave per row.  The wave
// first finds the row's common reference and total, a lane per partial result; then `lanes` lanes (a power of two from a
// quarter of head_dim on) take four elements each, and the 64 / lanes groups of them every so many-th partial result, so that
// the many partial results of a few rows are read side by side (one after the other they took 36 us of 127 for 32 rows of
// 32 partial results).
constexpr int kMergeWaves = 8;
__global__ __launch_bounds__(kMergeWaves* kWave) void chunk_merge_kernel(ChunkArgs, int head_dim, int lanes, int rows) {
  ChunkArgsRef a = chunk_args();
  const int32_t* plan = a.plan + kChunkPlanHead;
  const int tile = plan[3 * a.max_tiles + 1 + blockIdx.z], head = blockIdx.x;
  if (tile < 0) return;
  const int from = plan[tile], to = plan[tile + 1], share = a.plan[0];
  const ChunkTile t = chunk_geometry(a, plan[a.max_tiles + 1 + tile], plan[2 * a.max_tiles + 1 + tile]);
  const int lane = threadIdx.x & (kWave - 1);
  const int s0 = from / share, parts = (to - 1) / share - s0 + 1;
  const int first = blockIdx.y * rows;
  for (int r = first + threadIdx.x / kWave; r < min(first + rows, t.rows); r += kMergeWaves) {
    // the first share's part begins in that share, all others' in front of theirs
    auto slot = [&](int i) { return chunk_part_row(a, head, 2 * (s0 + i) + (i == 0 ? 1 : 0), r); };
    float ref = kChunkNegBig;
    for (int i = lane; i < parts; i += kWave) ref = fmaxf(ref, a.part_ml[2 * slot(i)]);
#pragma unroll
    for (int m = 1; m < kWave; m <<= 1) ref = fmaxf(ref, __shfl_xor(ref, m));
    float sum = 0.f;
    for (int i = lane; i < parts; i += kWave) {
      const int64_t at = slot(i);
      sum += a.part_ml[2 * at + 1] * __builtin_amdgcn_exp2f(a.part_ml[2 * at] - ref);
    }
    sum = wave_sum(sum);
    const int l = lane & (lanes - 1), groups = kWave / lanes;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    if (4 * l < head_dim) {
#pragma unroll 4
      for (int i = lane / lanes; i < parts; i += groups) {
        const int64_t at = slot(i);
        v += *reinterpret_cast<const f32x4*>(a.part_o + at * head_dim + 4 * l) * __builtin_amdgcn_exp2f(a.part_ml[2 * at] - ref);
      }
    }
    for (int m = lanes; m < kWave; m <<= 1)
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] += __shfl_xor(v[j], m);
    if (lane >= lanes || 4 * l >= head_dim) continue;
    const float inv = sum == 0.f ? 0.f : 1.0f / sum;
    const int64_t row = chunk_out_row<0>(a, t, head, r);
    f16x4 o;
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = (f16)(v[j] * inv);
    *reinterpret_cast<f16x4*>(a.out + row * head_dim + 4 * l) = o;
    if (a.lse && l == 0) a.lse[row] = chunk_lse(ref, sum);
  }
}

struct ChunkPlan {
  int64_t max_tiles, shares, part_rows;
  size_t bytes;
};

static bool chunk_sizes_ok(int64_t tokens, int64_t seqs, int64_t num_heads, int64_t num_kv_heads, int64_t head_dim,
                           int64_t block_size, int64_t max_pages) {
  return tokens >= 0 && tokens <= 0x7fffffff && seqs >= 0 && seqs < 0x7fffffff && num_heads > 0 && num_heads <= 0x7fffffff &&
         num_kv_heads > 0 && num_heads % num_kv_heads == 0 && head_dim >= 16 && head_dim <= 256 && head_dim % 16 == 0 &&
         block_size > 0 && block_size <= 0x7fffffff && max_pages >= 0 && max_pages <= 0x7fffffff &&
         tokens <= 0x3fffffff / (num_heads / num_kv_heads) && max_pages <= 0x7ffffe00 / block_size;
}

// Where contexts may be longer than kChunkWorth units (by what a row of the block table can hold) the kernel that can cut tiles is
// taken, which looks at the lengths: it costs a small call 4.5 us (4 sequences of 2 to 5 tokens over up to 1004 keys: 14.4 and 19.0 us,
// of which the launch that finds nothing to join is most), and where contexts are long it saves much more (16 tokens over 131079
// keys: 1700 and 98 us).  All tiles' units together are counted in 32 bits, and every workgroup plans all tiles in its LDS, which has room
// for kChunkMaxTiles: beyond that tiles stay whole, and one long context among many short ones is what the call waits for (one token
// each of 999 sequences of 100 keys and 4 tokens over 131072 keys 576 us, of 1014 sequences and the same 1230).
static ChunkPlan chunk_plan(int64_t tokens, int64_t seqs, int64_t num_heads, int64_t num_kv_heads, int64_t head_dim,
                            int64_t block_size, int64_t max_pages) {
  const int64_t group = num_heads / num_kv_heads, cus = device_cu_count(), tile_rows = chunk_rows((int)head_dim);
  ChunkPlan p = {(tokens * group + tile_rows - 1) / tile_rows + std::min(seqs, tokens), 0, 0, 16};
  const int64_t longest = max_pages * block_size / kChunkUnit + 1;
  if (p.max_tiles <= kChunkMaxTiles && num_kv_heads <= cus && longest > kChunkWorth + 1 && longest * p.max_tiles <= 0x3fffffff) {
    p.shares = cus / num_kv_heads;
    p.part_rows = std::min<int64_t>(tile_rows, (tokens * group + 15) / 16 * 16);
    const size_t rows = (size_t)(num_kv_heads * 2 * p.shares * p.part_rows);
    p.bytes = rows * (size_t)(head_dim + 2) * sizeof(float) + (size_t)(kChunkPlanHead + 3 * p.max_tiles + 1 + p.shares) * sizeof(int32_t);
  }
  return p;
}

}  // namespace aops

extern "C" size_t aops_paged_attention_chunk_workspace(int64_t tokens, int64_t seqs, int64_t num_heads, int64_t num_kv_heads,
                                                       int64_t head_dim, int64_t block_size, int64_t max_pages) {
  using namespace aops;
  if (!chunk_sizes_ok(tokens, seqs, num_heads, num_kv_heads, head_dim, block_size, max_pages)) return 0;
  return chunk_plan(tokens, seqs, num_heads, num_kv_heads, head_dim, block_size, max_pages).bytes;
}

extern "C" int aops_paged_attention_chunk_f16(const void* q, const void* key_cache, const void* value_cache,
                                              const int32_t* block_tables, const int32_t* context_lens,
                                              const int32_t* query_starts, void* out, float* lse, float scale, int64_t window,
                                              void* workspace, size_t workspace_bytes, int64_t tokens, int64_t seqs,
                                              int64_t num_heads, int64_t num_kv_heads, int64_t head_dim, int64_t block_size,
                                              int64_t max_pages, int64_t num_blocks, void* stream) {
  using namespace aops;
  if (!chunk_sizes_ok(tokens, seqs, num_heads, num_kv_heads, head_dim, block_size, max_pages) || num_blocks < 0 ||
      num_blocks > 0x7fffffff || window < 0 || !(scale > 0.f) || !(scale <= kChunkMaxScale))
    return AOPS_ERR_INVALID_ARGUMENT;
  if (tokens == 0 || seqs == 0) return AOPS_OK;
  if (!q || !out || !context_lens || !query_starts) return AOPS_ERR_INVALID_ARGUMENT;
  // with no pages there are no keys: every row sees nothing, and no address is formed from the null pointers
  if (num_blocks == 0 || max_pages == 0) num_blocks = max_pages = 0;
  if (max_pages > 0 && (!key_cache || !value_cache || !block_tables)) return AOPS_ERR_INVALID_ARGUMENT;
  const ChunkPlan p = chunk_plan(tokens, seqs, num_heads, num_kv_heads, head_dim, block_size, max_pages);
  if (!workspace || workspace_bytes < p.bytes) return AOPS_ERR_WORKSPACE;
  if (!grid_fits(p.max_tiles * num_kv_heads, kWave * chunk_waves((int)head_dim))) return AOPS_ERR_INVALID_ARGUMENT;
  // with 2^s the power of two at or above block_size, floor(2^(31+s) / block_size) + 1 is off by at most 2^s parts in
  // 2^(31+s): too little to change the quotient of a number below 2^31
  uint32_t s = 0;
  while (((int64_t)1 << s) < block_size) ++s;
  ChunkArgs a = {};
  a.q = static_cast<const f16*>(q);
  a.key_cache = static_cast<const f16*>(key_cache);
  a.value_cache = static_cast<const f16*>(value_cache);
  a.block_tables = block_tables;
  a.context_lens = context_lens;
  a.query_starts = query_starts;
  a.out = static_cast<f16*>(out);
  a.lse = lse;
  a.tokens = (int32_t)tokens;
  a.seqs = (int32_t)seqs;
  a.num_heads = (int32_t)num_heads;
  a.num_kv_heads = (int32_t)num_kv_heads;
  a.group = (int32_t)(num_heads / num_kv_heads);
  a.block_size = (int32_t)block_size;
  a.block_magic = (uint32_t)(((uint64_t)1 << (31 + s)) / (uint64_t)block_size + 1);
  a.block_shift = 31 + s;
  a.max_pages = (int32_t)max_pages;
  a.num_blocks = (int32_t)num_blocks;
  a.window = (int32_t)std::min<int64_t>(window, 0x7fffffff);
  a.max_tiles = (int32_t)p.max_tiles;
  a.tile_rows = chunk_rows((int)head_dim);
  a.shares = (int32_t)p.shares;
  a.part_rows = (int32_t)p.part_rows;
  a.scale_log2 = scale * kChunkLog2e;
  if (p.shares > 0) {
    a.part_o = static_cast<float*>(workspace);
    const size_t rows = (size_t)(num_kv_heads * 2 * p.shares * p.part_rows);
    a.part_ml = a.part_o + rows * (size_t)head_dim;
    a.plan = reinterpret_cast<int32_t*>(a.part_ml + 2 * rows);
  }
  const hipStream_t st = static_cast<hipStream_t>(stream);
  hipError_t e = hipErrorInvalidValue;
  switch (head_dim) {
#define AOPS_CHUNK_CASE(D) \
  case D:                  \
    e = chunk_launch<D>(a, st); \
    break;
    AOPS_CHUNK_DIMS(AOPS_CHUNK_CASE)
#undef AOPS_CHUNK_CASE
  }
  if (e != hipSuccess || p.shares == 0) return record_launch_status(e);
  int lanes = 4;
  while (4 * lanes < head_dim) lanes *= 2;
  // One row per wave where there are few and so, as a rule, many partial results of each (64 rows of 33: 8 us, 21 with four rows
  // per wave), else four (80 rows, of which few need it: 6.3 us instead of 7.9, spent on workgroups that find nothing to do).
  const int rows = p.part_rows <= 64 ? kMergeWaves : 4 * kMergeWaves;
  // (kv heads vary fastest, so that the few tiles of a small call are joined on all XCDs)
  chunk_merge_kernel<<<dim3((unsigned)num_kv_heads, (unsigned)((p.part_rows + rows - 1) / rows), (unsigned)p.shares),
                       kMergeWaves * kWave, 0, st>>>(a, (int)head_dim, lanes, rows);
  return record_launch_status(hipGetLastError());
}
