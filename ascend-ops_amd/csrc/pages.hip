// Pages of the paged caches [num_blocks, row_elems/16, block_size, 16]: copied, shared between sequences, given out,
// taken back and packed, for all layers' caches at once and without a word to the host.
//
// The state of a pool is one count per page: how many sequences hold it; a page is free where that is not positive.
// Pages are given out lowest first in the order of the requests, so every result is determined by its inputs.  All
// operators read their tables and counts and write new ones; only the caches are written in place, and only in pages
// that no sequence held before.
//
// An allocation is two launches.  `pages_plan` is one workgroup that adds up the requests, lists the lowest free
// pages, and copies the counts: a scan with one running total, a tile of 8192 counts in registers at a time (ranks
// inside a wave from ballots).  The second launch has a workgroup per row of the tables and, for forks and packing,
// workgroups that copy page data, each thread with several 128-bit loads in flight.  Small pools take one launch.
//
// Bound: the copies by HBM, the rest by the launches.  MI355X: 301 pages of 256 KiB in eight caches (1262 MB read and written)
// 218-241 us, 5.2-5.8 TB/s over the cards seen; packing a pool of 1024 such pages (1071 MB) 183-214 us; 128 forks from
// 64 sequences (294 MB) 70 us, 4.2 TB/s: the used tokens of a page are runs of 2 KiB on average, 4 KiB apart.
#include <algorithm>

#include "aops_common.h"

namespace aops {

constexpr int kMaxCaches = 256;
struct Caches {
  f16* at[kMaxCaches];
};

// Copies n 16-byte pieces, which `piece(i)` gives the offset (in halfs) of, between two pages of one cache; called by
// a workgroup of 256 threads.  Four loads of a thread are in flight before its first store.
template <typename F>
__device__ __forceinline__ void copy_pieces(const f16* __restrict__ src, f16* __restrict__ dst, uint32_t begin,
                                            uint32_t end, F piece) {
  constexpr uint32_t kDeep = 4;
  for (uint32_t i = begin + threadIdx.x; i < end; i += 256 * kDeep) {
    f16x8 v[kDeep];
#pragma unroll
    for (uint32_t j = 0; j < kDeep; ++j)
      if (i + 256 * j < end) v[j] = ld128_stream(src + piece(i + 256 * j));
#pragma unroll
    for (uint32_t j = 0; j < kDeep; ++j)
      if (i + 256 * j < end) st128_stream(dst + piece(i + 256 * j), v[j]);
  }
}

constexpr uint32_t kCopyPieces = 1024;  // 16 KiB per workgroup

__global__ __launch_bounds__(256) void copy_pages_kernel(Caches caches, const int32_t* __restrict__ src_pages,
                                                         const int32_t* __restrict__ dst_pages, uint32_t chunks,
                                                         int32_t num_blocks, int64_t page_elems) {
  const uint32_t pair = blockIdx.x / chunks, chunk = blockIdx.x - pair * chunks;
  const int32_t src = src_pages[pair], dst = dst_pages[pair];
  if (src < 0 || src >= num_blocks || dst < 0 || dst >= num_blocks || src == dst) return;
  f16* cache = caches.at[blockIdx.y];
  const uint32_t begin = chunk * kCopyPieces;
  const uint32_t end = (uint32_t)min((int64_t)begin + kCopyPieces, page_elems / 8);
  copy_pieces(cache + src * page_elems, cache + dst * page_elems, begin, end, [](uint32_t i) { return (int64_t)i * 8; });
}

// ------------------------------------------------------------------------------------------- plans
// What the planning workgroup leaves for the second launch, in the caller's workspace.
struct PlanOut {
  int32_t* head;    // [0]: free pages; packing: [1] = pages that move
  int32_t* before;  // per request: pages asked for by the requests in front of it
  int32_t* list;    // the free pages, lowest first, as many as are asked for; packing: the holes
  int32_t* movers;  // packing: the pages that move, and for every page its place among them
  int32_t* place;
};

constexpr int kPlanWaves = 16;  // of a planning workgroup
constexpr int kRowWaves = 4;    // of the others

// Exclusive sum over the waves of a workgroup and the total; `sums`: WAVES ints of LDS.
template <int WAVES>
__device__ __forceinline__ int waves_before(int mine, int* sums, int& total) {
  const int wave = threadIdx.x / kWave;
  __syncthreads();  // the last round's values have been read
  if ((threadIdx.x & (kWave - 1)) == 0) sums[wave] = mine;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    const int n = sums[w];
    before += w < wave ? n : 0;
    total += n;
  }
  return before;
}

// Sum over a workgroup.
template <int WAVES>
__device__ __forceinline__ int workgroup_sum(int mine, int* sums) {
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) mine += __shfl_xor(mine, d);
  int total;
  waves_before<WAVES>(mine, sums, total);
  return total;
}

// One pass over the counts in page order: visit(page, count, is_free, free pages in front of it).  Returns the free pages.
template <int WAVES, typename F>
__device__ __forceinline__ int scan_counts(const int32_t* __restrict__ counts, int num_blocks, int* sums, F visit) {
  const int wave = threadIdx.x / kWave, lane = threadIdx.x & (kWave - 1);
  const uint64_t below = lane == 0 ? 0 : ~uint64_t(0) >> (kWave - lane);
  constexpr int kPer = 8;  // counts per lane and tile
  int running = 0;
  for (int64_t tile = 0; tile < num_blocks; tile += WAVES * kWave * kPer) {
    const int first = wave * (kWave * kPer) + lane, left = (int)min((int64_t)num_blocks - tile, (int64_t)(WAVES * kWave * kPer));
    int32_t c[kPer];
    uint64_t free[kPer];
    int mine = 0;
    // (Behind the pool the last count is read, not nothing: of loads that are each under a condition of their own, the compiler
    // waits for one before it issues the next.)
    if (left == WAVES * kWave * kPer) {
#pragma unroll
      for (int j = 0; j < kPer; ++j) c[j] = counts[tile + first + j * kWave];
    } else {
#pragma unroll
      for (int j = 0; j < kPer; ++j) c[j] = counts[tile + min(first + j * kWave, left - 1)];
#pragma unroll
      for (int j = 0; j < kPer; ++j) c[j] = first + j * kWave < left ? c[j] : 1;
    }
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      free[j] = __builtin_amdgcn_ballot_w64(c[j] <= 0);
      mine += __builtin_popcountll(free[j]);
    }
    int total;
    int rank = running + waves_before<WAVES>(mine, sums, total);
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      if (first + j * kWave < left)
        visit((int)(tile + first + j * kWave), c[j], c[j] <= 0, rank + __builtin_popcountll(free[j] & below));
      rank += __builtin_popcountll(free[j]);
    }
    running += total;
  }
  return running;
}

struct Tables {
  const int32_t* tables;
  const int32_t* lens;
  int32_t seqs, width, block_size;
};

// Tokens of a sequence as far as its row of the table can hold them; 0 for a row that is none.
__device__ __forceinline__ int seq_tokens(const Tables& t, int seq) {
  if (seq < 0 || seq >= t.seqs) return 0;
  return (int)min((int64_t)max(t.lens[seq], 0), (int64_t)t.width * t.block_size);
}
__device__ __forceinline__ int pages_of(int64_t tokens, int block_size) {
  return (int)((tokens + block_size - 1) / block_size);
}

// Requests: fork asks for one page where the parent's last page is not full, extend for the pages that are missing.
// `who`: parents, or the wanted lengths.
template <bool FORK>
__device__ __forceinline__ int plan_request(const Tables& t, const int32_t* who, int i) {
  if constexpr (FORK) {
    return seq_tokens(t, who[i]) % t.block_size != 0;
  } else {
    const int have = seq_tokens(t, i), want = who[i];
    if (want <= have || (int64_t)want > (int64_t)t.width * t.block_size) return 0;
    return pages_of(want, t.block_size) - pages_of(have, t.block_size);
  }
}

template <bool FORK>
__global__ __launch_bounds__(kPlanWaves* kWave) void pages_plan_kernel(Tables t, const int32_t* __restrict__ who,
                                                                       int32_t requests,
                                                                       const int32_t* __restrict__ counts,
                                                                       int32_t num_blocks, int32_t* __restrict__ new_counts,
                                                                       PlanOut out) {
  __shared__ int sums[kPlanWaves];
  const int lane = threadIdx.x & (kWave - 1);
  // Sums of requests stop at num_blocks + 1: what is beyond is refused all the same, and nothing overflows.
  const int cap = num_blocks == 0x7fffffff ? num_blocks : num_blocks + 1;
  int asked = 0;
  for (int64_t tile = 0; tile < requests; tile += kPlanWaves * kWave) {
    const int64_t i = tile + threadIdx.x;
    const int need = i < requests ? plan_request<FORK>(t, who, (int)i) : 0;
    int64_t upto = need;
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
      const int64_t o = __shfl_up(upto, d);
      if (lane >= d) upto += o;
    }
    const int wave_total = (int)min(__shfl(upto, kWave - 1), (int64_t)cap);
    int64_t before = 0, total = 0;
    {
      const int wave = threadIdx.x / kWave;
      __syncthreads();
      if (lane == 0) sums[wave] = wave_total;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < kPlanWaves; ++w) {
        before += w < wave ? sums[w] : 0;
        total += sums[w];
      }
    }
    if (i < requests) out.before[i] = (int)min((int64_t)asked + before + (upto - need), (int64_t)cap);
    asked = (int)min((int64_t)asked + total, (int64_t)cap);
  }
  const int free = scan_counts<kPlanWaves>(counts, num_blocks, sums, [&](int page, int32_t c, bool is_free, int rank) {
    new_counts[page] = max(c, 0);
    if (is_free && rank < asked) out.list[rank] = page;
  });
  if (threadIdx.x == 0) out.head[0] = free;
}

// ------------------------------------------------------------------------------------------- fork
// Copies the first `part` tokens of page src to page dst: workgroup y - 1 = cache * slices + slice, its slice of them.
__device__ __forceinline__ void copy_last_page(const Tables& t, int32_t src, int32_t dst, int part, const Caches& caches,
                                               uint32_t slices, int32_t num_blocks, uint32_t granules) {
  if (src < 0 || src >= num_blocks) return;
  const int64_t page_elems = (int64_t)granules * t.block_size * 16;
  const uint32_t per_granule = 2u * part;  // 16-byte pieces of the used tokens; a page has `granules` such runs
  const uint32_t pieces = granules * per_granule;
  const uint32_t cache = (blockIdx.y - 1) / slices, slice = (blockIdx.y - 1) - cache * slices;
  f16* base = caches.at[cache];
  const uint32_t begin = (uint32_t)((uint64_t)pieces * slice / slices);
  const uint32_t end = (uint32_t)((uint64_t)pieces * (slice + 1) / slices);
  // i / per_granule by its reciprocal, rounded down: at most one too small
  const uint32_t inverse = 0xffffffffu / per_granule;
  copy_pieces(base + src * page_elems, base + dst * page_elems, begin, end, [&](uint32_t i) {
    uint32_t c = __umulhi(i, inverse), rest = i - c * per_granule;
    if (rest >= per_granule) ++c, rest -= per_granule;
    return ((int64_t)c * t.block_size * 2 + rest) * 8;
  });
}

// Workgroup (child, y): y == 0 writes the child's row; y - 1 = cache * slices + slice copies a slice of the used tokens
// of the parent's last page.
__global__ __launch_bounds__(256) void fork_kernel(Tables t, const int32_t* __restrict__ parents, Caches caches,
                                                   uint32_t slices, int32_t num_blocks, uint32_t granules,
                                                   int32_t* __restrict__ child_tables, int32_t* __restrict__ child_lens,
                                                   int32_t* __restrict__ new_counts, PlanOut plan) {
  const int child = blockIdx.x;
  const int parent = parents[child];
  const int tokens = seq_tokens(t, parent);
  const int full = tokens / t.block_size, part = tokens - full * t.block_size;
  const int rank = plan.before[child];
  const bool ok = part == 0 || rank < plan.head[0];
  const int32_t* row = t.tables + (int64_t)(tokens > 0 ? parent : 0) * t.width;
  if (blockIdx.y == 0) {
    int32_t* out = child_tables + (int64_t)child * t.width;
    for (int j = threadIdx.x; j < t.width; j += 256) {
      int32_t page = -1;
      if (ok && j < full) page = row[j];
      if (ok && j == full && part > 0) page = plan.list[rank];
      out[j] = page;
      if (ok && j < full + (part > 0) && page >= 0 && page < num_blocks) atomicAdd(new_counts + page, 1);
    }
    if (threadIdx.x == 0) child_lens[child] = ok ? tokens : 0;
    return;
  }
  if (!ok || part == 0) return;
  copy_last_page(t, row[full], plan.list[rank], part, caches, slices, num_blocks, granules);
}

// ------------------------------------------------------------------------------------------- extend
__global__ __launch_bounds__(256) void extend_kernel(Tables t, const int32_t* __restrict__ wanted,
                                                     int32_t* __restrict__ new_tables, int32_t* __restrict__ granted,
                                                     int32_t* __restrict__ new_counts, PlanOut plan) {
  const int seq = blockIdx.x;
  const int have_tokens = seq_tokens(t, seq), want = wanted[seq];
  const int have = pages_of(have_tokens, t.block_size);
  const int need = plan_request<false>(t, wanted, seq);
  const int before = plan.before[seq];
  const bool ok = want > have_tokens && (int64_t)want <= (int64_t)t.width * t.block_size &&
                  (need == 0 || (int64_t)before + need <= plan.head[0]);
  const int32_t* row = t.tables + (int64_t)seq * t.width;
  int32_t* out = new_tables + (int64_t)seq * t.width;
  for (int j = threadIdx.x; j < t.width; j += 256) {
    int32_t page = row[j];
    if (ok && j >= have && j < have + need) {
      page = plan.list[before + j - have];
      atomicAdd(new_counts + page, 1);
    }
    out[j] = page;
  }
  if (threadIdx.x == 0) granted[seq] = ok ? want : have_tokens;
}

// ------------------------------------------------------------------------------------------- free
__global__ __launch_bounds__(256) void counts_copy_kernel(const int32_t* __restrict__ counts, int32_t num_blocks,
                                                          int32_t* __restrict__ new_counts) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i < num_blocks) new_counts[i] = max(counts[i], 0);
}

// A count never falls below zero: a decrement that finds none left is taken back.  As many succeed as there were
// counts, in whatever order they come: one fails only after all have been taken.
__global__ __launch_bounds__(256) void free_kernel(Tables t, const int32_t* __restrict__ rows, int32_t num_blocks,
                                                   int32_t* __restrict__ new_counts) {
  const int seq = rows[blockIdx.x];
  const int pages = pages_of(seq_tokens(t, seq), t.block_size);
  const int32_t* row = t.tables + (int64_t)(pages > 0 ? seq : 0) * t.width;
  for (int j = threadIdx.x; j < pages; j += 256) {
    const int32_t page = row[j];
    if (page < 0 || page >= num_blocks) continue;
    if (atomicSub(new_counts + page, 1) <= 0) atomicAdd(new_counts + page, 1);
  }
}

// ------------------------------------------------------------------------------------------- compact
__global__ __launch_bounds__(kPlanWaves* kWave) void compact_plan_kernel(const int32_t* __restrict__ counts,
                                                                         int32_t num_blocks, int32_t* __restrict__ used_out,
                                                                         PlanOut out) {
  __shared__ int sums[kPlanWaves];
  const int free = scan_counts<kPlanWaves>(counts, num_blocks, sums, [](int, int32_t, bool, int) {});
  const int used = num_blocks - free;
  __shared__ int free_below;  // free pages in front of page `used`: the holes
  if (threadIdx.x == 0) free_below = used == num_blocks ? free : -1;
  scan_counts<kPlanWaves>(counts, num_blocks, sums, [&](int page, int32_t, bool is_free, int rank) {
    if (page == used) free_below = rank;
    if (is_free && page < used) out.list[rank] = page;
    // used pages in front of this one: page - rank; the ones behind `used` come after used - free_below others
    if (!is_free && page >= used) out.place[page] = page - rank;
  });
  __syncthreads();
  const int holes = free_below, stay = used - holes;
  for (int64_t p = (int64_t)used + threadIdx.x; p < num_blocks; p += kPlanWaves * kWave) {
    if (counts[p] <= 0) continue;
    const int k = out.place[p] - stay;
    out.place[p] = k;
    out.movers[k] = (int)p;
  }
  if (threadIdx.x == 0) {
    out.head[0] = used;
    out.head[1] = holes;
    used_out[0] = used;
  }
}

// Workgroup `wg` of `wgs` copies its share of the pages that move, a piece of one page in one cache at a time.
template <typename FROM, typename TO>
__device__ __forceinline__ void copy_moves(uint32_t wg, uint32_t wgs, int moves, const Caches& caches, int num_caches,
                                           uint32_t chunks, int64_t page_elems, FROM from, TO to) {
  const uint64_t per_move = (uint64_t)num_caches * chunks;
  const uint64_t items = per_move * moves;
  for (uint64_t i = wg; i < items; i += wgs) {
    const uint32_t move = (uint32_t)(i / per_move), rest = (uint32_t)(i - move * per_move);
    const uint32_t cache = rest / chunks, chunk = rest - cache * chunks;
    const uint32_t begin = chunk * kCopyPieces;
    const uint32_t end = (uint32_t)min((int64_t)begin + kCopyPieces, page_elems / 8);
    f16* base = caches.at[cache];
    copy_pieces(base + from(move) * page_elems, base + to(move) * page_elems, begin, end,
                [](uint32_t j) { return (int64_t)j * 8; });
  }
}

// Workgroups 0 .. row_wgs-1 rewrite the tables and counts, the others copy pages.
__global__ __launch_bounds__(256) void compact_kernel(Tables t, const int32_t* __restrict__ counts, int32_t num_blocks,
                                                      Caches caches, int32_t num_caches, uint32_t chunks,
                                                      int64_t page_elems, uint32_t row_wgs, int32_t* __restrict__ new_tables,
                                                      int32_t* __restrict__ new_counts, PlanOut plan) {
  const int used = plan.head[0], moves = plan.head[1];
  if (blockIdx.x < row_wgs) {
    const int64_t stride = (int64_t)row_wgs * 256, first = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t entries = (int64_t)t.seqs * t.width;
    for (int64_t i = first; i < entries; i += stride) {
      const int seq = (int)(i / t.width), j = (int)(i - (int64_t)seq * t.width);
      int32_t page = t.tables[i];
      if (page >= used && page < num_blocks && j < pages_of(seq_tokens(t, seq), t.block_size) && counts[page] > 0)
        page = plan.list[plan.place[page]];
      new_tables[i] = page;
    }
    for (int64_t p = first; p < num_blocks; p += stride) {
      const int32_t c = counts[p];
      if (p >= used) {
        new_counts[p] = 0;
        if (c > 0) new_counts[plan.list[plan.place[p]]] = c;
      } else if (c > 0) {
        new_counts[p] = c;
      }
    }
    return;
  }
  copy_moves(blockIdx.x - row_wgs, gridDim.x - row_wgs, moves, caches, num_caches, chunks, page_elems,
             [&](int k) { return (int64_t)plan.movers[k]; }, [&](int k) { return (int64_t)plan.list[k]; });
}

// ------------------------------------------------------------------------------------------- small pools
// The same operators in one launch, for pools of up to kSmallPool pages, up to kSmallRequests requests (one per thread) and
// tables of up to kSmallEntries entries, kSmallWalked where one workgroup walks them all: a decode step's calls, where each launch
// counts (about 2 us on the host and as much between two kernels).  Every workgroup finds what it
// needs of the plan itself, from counts that are a few KiB in the L2, and one workgroup makes the new counts, in LDS.
constexpr int kSmallPool = 4096;
constexpr int kSmallRequests = kRowWaves * kWave;
constexpr int64_t kSmallEntries = 16384, kSmallWalked = 4096;

// Pages asked for by the requests in front of request i; called by a workgroup of kRowWaves waves.
template <bool FORK>
__device__ __forceinline__ int asked_before(const Tables& t, const int32_t* who, int i, int* sums) {
  const int k = threadIdx.x;
  return workgroup_sum<kRowWaves>(k < i ? min(plan_request<FORK>(t, who, k), kSmallPool + 1) : 0, sums);
}

// Pages asked for by this thread's request and those in front of it.
template <bool FORK>
__device__ __forceinline__ int asked_upto(const Tables& t, const int32_t* who, int requests, int* sums) {
  const int i = threadIdx.x, lane = threadIdx.x & (kWave - 1);
  int upto = i < requests ? min(plan_request<FORK>(t, who, i), kSmallPool + 1) : 0;
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
    const int o = __shfl_up(upto, d);
    if (lane >= d) upto += o;
  }
  int total;
  const int mine = __shfl(upto, kWave - 1);
  return upto + waves_before<kRowWaves>(mine, sums, total);
}

// Largest value of a workgroup of kRowWaves waves; none is negative.
__device__ __forceinline__ int workgroup_max(int mine, int* sums) {
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) mine = max(mine, __shfl_xor(mine, d));
  __syncthreads();
  if ((threadIdx.x & (kWave - 1)) == 0) sums[threadIdx.x / kWave] = mine;
  __syncthreads();
  int most = 0;
#pragma unroll
  for (int w = 0; w < kRowWaves; ++w) most = max(most, sums[w]);
  return most;
}

// Pages given out: the largest sum of leading requests that the free pages suffice for; `upto`: asked_upto.
__device__ __forceinline__ int given_out(int upto, int free, int* sums) { return workgroup_max(upto <= free ? upto : 0, sums); }

// Counts in `held` (LDS) the pages that children share with their parents: the first `full` pages of row `row` for the child
// that each thread stands for (row 0 where full is 0).  A thread takes (child, page) pairs, eight at a time, whose loads are in
// flight together: a thread per child, which walks its pages one after the other, took 304 us for one child of 4000 pages and
// 81 for 1000; so they take 8.5 and 7.4, in two launches, with a workgroup per child, 12.4 and 9.1.
__device__ __forceinline__ void hold_shared_pages(const Tables& t, int row, int full, int children, int32_t num_blocks, int* rows,
                                                  int* fulls, int* held, int* sums) {
  constexpr int kDeep = 8, kThreads = kRowWaves * kWave;
  rows[threadIdx.x] = row;
  fulls[threadIdx.x] = full;
  const int longest = workgroup_max(full, sums);
  const int pairs = children * longest;
  const uint32_t inverse = longest > 0 ? 0xffffffffu / longest : 0;  // pair / longest, rounded down: at most one too small
  for (int first = threadIdx.x; first < pairs; first += kThreads * kDeep) {
    int32_t page[kDeep];
    bool is[kDeep];
#pragma unroll
    for (int k = 0; k < kDeep; ++k) {
      const int pair = min(first + k * kThreads, pairs - 1);
      int child = __umulhi(pair, inverse), j = pair - child * longest;
      if (j >= longest) ++child, j -= longest;
      is[k] = first + k * kThreads < pairs && j < fulls[child];
      page[k] = t.tables[(int64_t)rows[child] * t.width + j];
    }
#pragma unroll
    for (int k = 0; k < kDeep; ++k)
      if (is[k] && page[k] >= 0 && page[k] < num_blocks) atomicAdd(held + page[k], 1);
  }
}

// Workgroup (child, y) as in fork_kernel; workgroup (children, 0) makes the counts and lengths.
__global__ __launch_bounds__(kRowWaves* kWave) void fork_small_kernel(Tables t, const int32_t* __restrict__ parents,
                                                                       int32_t children, Caches caches, uint32_t slices,
                                                                       const int32_t* __restrict__ counts, int32_t num_blocks,
                                                                       uint32_t granules, int32_t* __restrict__ child_tables,
                                                                       int32_t* __restrict__ child_lens,
                                                                       int32_t* __restrict__ new_counts) {
  __shared__ int sums[kRowWaves];
  __shared__ int fresh;
  __shared__ int held[kSmallPool];
  __shared__ int rows[kSmallRequests], fulls[kSmallRequests];
  const int child = blockIdx.x;
  if (child == children) {
    if (blockIdx.y > 0) return;
    const int free = scan_counts<kRowWaves>(counts, num_blocks, sums, [&](int page, int32_t c, bool, int) { held[page] = max(c, 0); });
    const int upto = asked_upto<true>(t, parents, children, sums);
    const int given = given_out(upto, free, sums);
    scan_counts<kRowWaves>(counts, num_blocks, sums, [&](int page, int32_t, bool is_free, int rank) {
      if (is_free && rank < given) atomicAdd(held + page, 1);
    });
    // shared pages, of the children whose own page (if they need one) is among those given out
    const int i = threadIdx.x;
    int full = 0;
    if (i < children) {
      const int tokens = seq_tokens(t, parents[i]);
      const bool ok = tokens % t.block_size == 0 || upto <= free;
      child_lens[i] = ok ? tokens : 0;
      if (ok) full = tokens / t.block_size;
    }
    hold_shared_pages(t, full > 0 ? parents[i] : 0, full, children, num_blocks, rows, fulls, held, sums);
    __syncthreads();
    for (int p = threadIdx.x; p < num_blocks; p += kRowWaves * kWave) new_counts[p] = held[p];
    return;
  }
  const int parent = parents[child];
  const int tokens = seq_tokens(t, parent);
  const int full = tokens / t.block_size, part = tokens - full * t.block_size;
  const int32_t* row = t.tables + (int64_t)(tokens > 0 ? parent : 0) * t.width;
  bool ok = true;
  if (part > 0) {
    const int rank = asked_before<true>(t, parents, child, sums);
    const int free = scan_counts<kRowWaves>(counts, num_blocks, sums, [&](int page, int32_t, bool is_free, int r) {
      if (is_free && r == rank) fresh = page;
    });
    ok = rank < free;
    __syncthreads();
  }
  if (blockIdx.y == 0) {
    int32_t* out = child_tables + (int64_t)child * t.width;
    for (int j = threadIdx.x; j < t.width; j += 256) out[j] = !ok ? -1 : j < full ? row[j] : j == full && part > 0 ? fresh : -1;
    return;
  }
  if (!ok || part == 0) return;
  copy_last_page(t, row[full], fresh, part, caches, slices, num_blocks, granules);
}

// Workgroup `seq` writes the row of a sequence, workgroup `seqs` the counts.
__global__ __launch_bounds__(kRowWaves* kWave) void extend_small_kernel(Tables t, const int32_t* __restrict__ wanted,
                                                                         const int32_t* __restrict__ counts, int32_t num_blocks,
                                                                         int32_t* __restrict__ new_tables,
                                                                         int32_t* __restrict__ granted,
                                                                         int32_t* __restrict__ new_counts) {
  __shared__ int sums[kRowWaves];
  const int seq = blockIdx.x;
  if (seq == t.seqs) {
    const int free = scan_counts<kRowWaves>(counts, num_blocks, sums, [](int, int32_t, bool, int) {});
    const int given = given_out(asked_upto<false>(t, wanted, t.seqs, sums), free, sums);
    scan_counts<kRowWaves>(counts, num_blocks, sums, [&](int page, int32_t c, bool is_free, int rank) {
      new_counts[page] = is_free ? (rank < given ? 1 : 0) : c;
    });
    return;
  }
  const int have_tokens = seq_tokens(t, seq), want = wanted[seq];
  const int have = pages_of(have_tokens, t.block_size);
  const int need = plan_request<false>(t, wanted, seq);
  const int32_t* row = t.tables + (int64_t)seq * t.width;
  int32_t* out = new_tables + (int64_t)seq * t.width;
  bool ok = want > have_tokens && (int64_t)want <= (int64_t)t.width * t.block_size;
  if (ok && need > 0) {
    const int before = asked_before<false>(t, wanted, seq, sums);
    const int free = scan_counts<kRowWaves>(counts, num_blocks, sums, [](int, int32_t, bool, int) {});
    ok = before + need <= free;
    if (ok)
      scan_counts<kRowWaves>(counts, num_blocks, sums, [&](int page, int32_t, bool is_free, int r) {
        if (is_free && r >= before && r < before + need) out[have + r - before] = page;
      });
  }
  for (int j = threadIdx.x; j < t.width; j += 256)
    if (!ok || j < have || j >= have + need) out[j] = row[j];
  if (threadIdx.x == 0) granted[seq] = ok ? want : have_tokens;
}

__global__ __launch_bounds__(kPlanWaves* kWave) void free_small_kernel(Tables t, const int32_t* __restrict__ rows,
                                                                       int32_t num_rows, const int32_t* __restrict__ counts,
                                                                       int32_t num_blocks, int32_t* __restrict__ new_counts) {
  __shared__ int named[kSmallPool];
  for (int p = threadIdx.x; p < num_blocks; p += kPlanWaves * kWave) named[p] = 0;
  __syncthreads();
  for (int64_t i = threadIdx.x; i < (int64_t)num_rows * t.width; i += kPlanWaves * kWave) {
    const int k = (int)(i / t.width), j = (int)(i - (int64_t)k * t.width), seq = rows[k];
    if (j >= pages_of(seq_tokens(t, seq), t.block_size)) continue;
    const int32_t page = t.tables[(int64_t)seq * t.width + j];
    if (page >= 0 && page < num_blocks) atomicAdd(named + page, 1);
  }
  __syncthreads();
  for (int p = threadIdx.x; p < num_blocks; p += kPlanWaves * kWave) new_counts[p] = max(max(counts[p], 0) - named[p], 0);
}

// As compact_kernel, with the plan in every workgroup's LDS.
__global__ __launch_bounds__(kRowWaves* kWave) void compact_small_kernel(Tables t, const int32_t* __restrict__ counts,
                                                                         int32_t num_blocks, Caches caches,
                                                                         int32_t num_caches, uint32_t chunks,
                                                                         int64_t page_elems, uint32_t row_wgs,
                                                                         int32_t* __restrict__ new_tables,
                                                                         int32_t* __restrict__ new_counts,
                                                                         int32_t* __restrict__ used_out) {
  __shared__ int sums[kRowWaves];
  __shared__ uint16_t holes[kSmallPool / 2], movers[kSmallPool / 2];  // movers: the last one first
  __shared__ uint16_t place[kSmallPool];                              // of a page that moves, in movers
  __shared__ int free_below;
  const int free = scan_counts<kRowWaves>(counts, num_blocks, sums, [](int, int32_t, bool, int) {});
  const int used = num_blocks - free;
  if (threadIdx.x == 0) free_below = 0;
  scan_counts<kRowWaves>(counts, num_blocks, sums, [&](int page, int32_t, bool is_free, int rank) {
    if (page == used) free_below = rank;
    if (is_free && page < used) holes[rank] = (uint16_t)page;
    if (!is_free && page >= used) {
      const int from_end = used - 1 - (page - rank);  // used pages behind this one
      movers[from_end] = (uint16_t)page;
      place[page] = (uint16_t)from_end;
    }
  });
  __syncthreads();
  const int moves = free_below;
  auto hole_of = [&](int from_end) { return (int)holes[moves - 1 - from_end]; };
  if (blockIdx.x < row_wgs) {
    const int64_t stride = (int64_t)row_wgs * 256, first = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t entries = (int64_t)t.seqs * t.width;
    for (int64_t i = first; i < entries; i += stride) {
      const int seq = (int)(i / t.width), j = (int)(i - (int64_t)seq * t.width);
      int32_t page = t.tables[i];
      if (page >= used && page < num_blocks && j < pages_of(seq_tokens(t, seq), t.block_size) && counts[page] > 0)
        page = hole_of(place[page]);
      new_tables[i] = page;
    }
    for (int64_t p = first; p < num_blocks; p += stride) {
      const int32_t c = counts[p];
      if (p >= used) {
        new_counts[p] = 0;
        if (c > 0) new_counts[hole_of(place[p])] = c;
      } else if (c > 0) {
        new_counts[p] = c;
      }
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) used_out[0] = used;
    return;
  }
  copy_moves(blockIdx.x - row_wgs, gridDim.x - row_wgs, moves, caches, num_caches, chunks, page_elems,
             [&](int k) { return (int64_t)movers[k]; }, [&](int k) { return (int64_t)hole_of(k); });
}

// ------------------------------------------------------------------------------------------- host side
static int fill(Caches& c, void* const* caches, int64_t num_caches) {
  if (!caches) return AOPS_ERR_INVALID_ARGUMENT;
  for (int64_t i = 0; i < num_caches; ++i) {
    if (!caches[i]) return AOPS_ERR_INVALID_ARGUMENT;
    c.at[i] = static_cast<f16*>(caches[i]);
  }
  return AOPS_OK;
}

static bool geometry_ok(int64_t num_caches, int64_t num_blocks, int64_t row_elems, int64_t block_size) {
  return num_caches >= 1 && num_caches <= kMaxCaches && num_blocks >= 0 && num_blocks < 0x7fffffff && row_elems > 0 &&
         row_elems % 16 == 0 && row_elems <= 0x7fffffff && block_size > 0 && block_size <= 0x7fffffff &&
         row_elems * block_size / 8 <= 0x7fffffff;  // 16-byte pieces of a page are counted in 32 bits
}

// (A workgroup counts the columns of a row in 32 bits, 256 at a time: behind 2^31 - 256 of them the last step would wrap.)
static bool tables_ok(int64_t seqs, int64_t max_pages, int64_t block_size) {
  return seqs >= 0 && seqs <= 0x7fffffff && max_pages >= 0 && max_pages <= 0x7fffff00 && block_size > 0 &&
         block_size <= 0x7fffffff;
}

static PlanOut plan_layout(void* workspace, int64_t num_blocks) {
  int32_t* w = static_cast<int32_t*>(workspace);
  PlanOut p;
  p.head = w;
  p.list = w + 4;
  p.before = p.list + num_blocks;
  p.movers = p.before;  // packing has no requests
  p.place = p.movers + num_blocks;
  return p;
}

// Sides of the rule (us, one launch and two): a beam step of 4 sequences in a pool of 96 pages, three calls, 17 and 23; 128 children of
// short sequences in a pool of 4096 pages 7.5 and 9.0, 256 7.9 and 9.1, 512 17-22 and 14, 2000 91 and 33: every
// workgroup looks at all requests and all counts.  Extending 256 sequences 6.0 and 8.3.
// `most` entries of the requests' rows: the pages of forks and of sequences that end are counted by one workgroup, 4000 of them in 8.5
// and 9.0-12.4 (fork), 5.0 and 6.5-10.0 (free), 16000 in 15.7 and 9.3, 11.6 and 6.6; rows are extended by a workgroup each, 16000
// entries in 6.0-7.9 and 8.2-8.6.
static bool small_pool(int64_t num_blocks, int64_t requests, int64_t max_pages, int64_t most) {
  return num_blocks <= kSmallPool && requests <= kSmallRequests && requests * max_pages <= most;
}

static uint32_t page_chunks(int64_t page_elems) { return (uint32_t)((page_elems / 8 + kCopyPieces - 1) / kCopyPieces); }

}  // namespace aops

extern "C" size_t aops_pages_workspace(int64_t requests, int64_t num_blocks) {
  if (requests < 0 || num_blocks < 0 || requests > 0x7fffffff || num_blocks >= 0x7fffffff) return 0;
  const int64_t ints = 4 + num_blocks + std::max(requests, 2 * num_blocks);
  return (size_t)ints * sizeof(int32_t);
}

extern "C" int aops_copy_pages_f16(void* const* caches, int64_t num_caches, const int32_t* src_pages,
                                   const int32_t* dst_pages, int64_t pairs, int64_t num_blocks, int64_t row_elems,
                                   int64_t block_size, void* stream) {
  using namespace aops;
  if (!geometry_ok(num_caches, num_blocks, row_elems, block_size) || pairs < 0) return AOPS_ERR_INVALID_ARGUMENT;
  if (pairs == 0 || num_blocks == 0) return AOPS_OK;
  const uint32_t chunks = page_chunks(row_elems * block_size);
  if (pairs > 0x7fffffff || !grid_fits(pairs * chunks, 256) || !src_pages || !dst_pages) return AOPS_ERR_INVALID_ARGUMENT;
  Caches c;
  if (const int e = fill(c, caches, num_caches)) return e;
  copy_pages_kernel<<<dim3((unsigned)(pairs * chunks), (unsigned)num_caches), 256, 0, static_cast<hipStream_t>(stream)>>>(
      c, src_pages, dst_pages, chunks, (int32_t)num_blocks, row_elems * block_size);
  return record_launch_status(hipGetLastError());
}

extern "C" int aops_fork_sequences_f16(const int32_t* block_tables, const int32_t* context_lens, int64_t seqs,
                                       int64_t max_pages, const int32_t* parents, int64_t children,
                                       const int32_t* ref_counts, int64_t num_blocks, void* const* caches,
                                       int64_t num_caches, int64_t row_elems, int64_t block_size, int32_t* child_tables,
                                       int32_t* child_lens, int32_t* new_ref_counts, void* workspace,
                                       size_t workspace_bytes, void* stream) {
  using namespace aops;
  if (!geometry_ok(num_caches, num_blocks, row_elems, block_size) || !tables_ok(seqs, max_pages, block_size) ||
      children < 0 || children > 0x7fffffff || !grid_fits(children + 1, 256))
    return AOPS_ERR_INVALID_ARGUMENT;
  if (children == 0 && num_blocks == 0) return AOPS_OK;
  if ((num_blocks > 0 && (!ref_counts || !new_ref_counts)) ||
      (children > 0 && (!parents || !child_lens || (max_pages > 0 && !child_tables))) ||
      (seqs > 0 && (!context_lens || (max_pages > 0 && !block_tables))))
    return AOPS_ERR_INVALID_ARGUMENT;
  Caches c;
  if (const int e = fill(c, caches, num_caches)) return e;
  if (!workspace || workspace_bytes < aops_pages_workspace(children, num_blocks)) return AOPS_ERR_WORKSPACE;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const Tables t = {block_tables, context_lens, (int32_t)seqs, (int32_t)max_pages, (int32_t)block_size};
  // a slice is at most four rounds of a workgroup's copy loop, unless a page is larger than 64 of them
  const uint32_t slices = (uint32_t)std::min<int64_t>((row_elems * block_size / 8 + 4 * kCopyPieces - 1) / (4 * kCopyPieces), 64);
  if (small_pool(num_blocks, children, max_pages, kSmallWalked)) {
    fork_small_kernel<<<dim3((unsigned)children + 1, 1 + (unsigned)num_caches * slices), kRowWaves * kWave, 0, st>>>(
        t, parents, (int32_t)children, c, slices, ref_counts, (int32_t)num_blocks, (uint32_t)(row_elems / 16), child_tables,
        child_lens, new_ref_counts);
    return record_launch_status(hipGetLastError());
  }
  const PlanOut plan = plan_layout(workspace, num_blocks);
  pages_plan_kernel<true><<<1, kPlanWaves * kWave, 0, st>>>(t, parents, (int32_t)children, ref_counts,
                                                            (int32_t)num_blocks, new_ref_counts, plan);
  if (children > 0)
    fork_kernel<<<dim3((unsigned)children, 1 + (unsigned)num_caches * slices), 256, 0, st>>>(
        t, parents, c, slices, (int32_t)num_blocks, (uint32_t)(row_elems / 16), child_tables, child_lens, new_ref_counts,
        plan);
  return record_launch_status(hipGetLastError());
}

extern "C" int aops_extend_sequences(const int32_t* block_tables, const int32_t* context_lens,
                                     const int32_t* wanted_lens, int64_t seqs, int64_t max_pages, int64_t block_size,
                                     const int32_t* ref_counts, int64_t num_blocks, int32_t* new_tables,
                                     int32_t* granted_lens, int32_t* new_ref_counts, void* workspace,
                                     size_t workspace_bytes, void* stream) {
  using namespace aops;
  if (!tables_ok(seqs, max_pages, block_size) || !grid_fits(seqs + 1, 256) || num_blocks < 0 || num_blocks >= 0x7fffffff)
    return AOPS_ERR_INVALID_ARGUMENT;
  if (seqs == 0 && num_blocks == 0) return AOPS_OK;
  if ((num_blocks > 0 && (!ref_counts || !new_ref_counts)) ||
      (seqs > 0 && (!context_lens || !wanted_lens || !granted_lens || (max_pages > 0 && (!block_tables || !new_tables)))))
    return AOPS_ERR_INVALID_ARGUMENT;
  if (!workspace || workspace_bytes < aops_pages_workspace(seqs, num_blocks)) return AOPS_ERR_WORKSPACE;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const Tables t = {block_tables, context_lens, (int32_t)seqs, (int32_t)max_pages, (int32_t)block_size};
  if (small_pool(num_blocks, seqs, max_pages, kSmallEntries)) {
    extend_small_kernel<<<(unsigned)seqs + 1, kRowWaves * kWave, 0, st>>>(t, wanted_lens, ref_counts, (int32_t)num_blocks,
                                                                           new_tables, granted_lens, new_ref_counts);
    return record_launch_status(hipGetLastError());
  }
  const PlanOut plan = plan_layout(workspace, num_blocks);
  pages_plan_kernel<false><<<1, kPlanWaves * kWave, 0, st>>>(t, wanted_lens, (int32_t)seqs, ref_counts,
                                                             (int32_t)num_blocks, new_ref_counts, plan);
  if (seqs > 0)
    extend_kernel<<<(unsigned)seqs, 256, 0, st>>>(t, wanted_lens, new_tables, granted_lens, new_ref_counts, plan);
  return record_launch_status(hipGetLastError());
}

extern "C" int aops_free_sequences(const int32_t* block_tables, const int32_t* context_lens, int64_t seqs,
                                   int64_t max_pages, int64_t block_size, const int32_t* rows, int64_t num_rows,
                                   const int32_t* ref_counts, int64_t num_blocks, int32_t* new_ref_counts, void* stream) {
  using namespace aops;
  if (!tables_ok(seqs, max_pages, block_size) || num_rows < 0 || !grid_fits(num_rows, 256) || num_blocks < 0 ||
      num_blocks >= 0x7fffffff)
    return AOPS_ERR_INVALID_ARGUMENT;
  if (num_blocks == 0) return AOPS_OK;
  if (!ref_counts || !new_ref_counts || (num_rows > 0 && !rows) ||
      (seqs > 0 && (!context_lens || (max_pages > 0 && !block_tables))))
    return AOPS_ERR_INVALID_ARGUMENT;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const Tables t = {block_tables, context_lens, (int32_t)seqs, (int32_t)max_pages, (int32_t)block_size};
  if (small_pool(num_blocks, seqs > 0 ? num_rows : 0, max_pages, kSmallWalked)) {
    free_small_kernel<<<1, kPlanWaves * kWave, 0, st>>>(t, rows, (int32_t)(seqs > 0 ? num_rows : 0), ref_counts,
                                                        (int32_t)num_blocks, new_ref_counts);
    return record_launch_status(hipGetLastError());
  }
  counts_copy_kernel<<<(unsigned)((num_blocks + 255) / 256), 256, 0, st>>>(ref_counts, (int32_t)num_blocks, new_ref_counts);
  if (num_rows > 0 && seqs > 0 && max_pages > 0)
    free_kernel<<<(unsigned)num_rows, 256, 0, st>>>(t, rows, (int32_t)num_blocks, new_ref_counts);
  return record_launch_status(hipGetLastError());
}

extern "C" int aops_compact_pages_f16(const int32_t* block_tables, const int32_t* context_lens, int64_t seqs,
                                      int64_t max_pages, const int32_t* ref_counts, int64_t num_blocks,
                                      void* const* caches, int64_t num_caches, int64_t row_elems, int64_t block_size,
                                      int32_t* new_tables, int32_t* new_ref_counts, int32_t* num_used, void* workspace,
                                      size_t workspace_bytes, void* stream) {
  using namespace aops;
  if (!geometry_ok(num_caches, num_blocks, row_elems, block_size) || !tables_ok(seqs, max_pages, block_size))
    return AOPS_ERR_INVALID_ARGUMENT;
  if (!num_used || (num_blocks > 0 && (!ref_counts || !new_ref_counts)) ||
      (seqs > 0 && (!context_lens || (max_pages > 0 && (!block_tables || !new_tables)))))
    return AOPS_ERR_INVALID_ARGUMENT;
  Caches c;
  if (const int e = fill(c, caches, num_caches)) return e;
  if (!workspace || workspace_bytes < aops_pages_workspace(0, num_blocks)) return AOPS_ERR_WORKSPACE;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const Tables t = {block_tables, context_lens, (int32_t)seqs, (int32_t)max_pages, (int32_t)block_size};
  const int64_t page_elems = row_elems * block_size;
  const uint32_t chunks = page_chunks(page_elems);
  const int64_t ints = std::max(seqs * max_pages, num_blocks);
  const int64_t row_wgs = std::min<int64_t>(std::max<int64_t>((ints + 1023) / 1024, 1), device_cu_count());
  const int64_t most = num_blocks / 2 * num_caches * (int64_t)chunks;  // at most half of the pages move
  const int64_t copy_wgs = std::min<int64_t>(most, 8 * (int64_t)device_cu_count());
  // (one launch and two, pools of 1025, 2048, 3000 and 4096 pages: 6.9 and 9.4 us, 6.9 and 9.3, 10.0 and 9.4, 9.5 and 9.4; with counts
  // that were waited for one by one 14.4 at 4096)
  if (num_blocks <= kSmallPool) {
    compact_small_kernel<<<(unsigned)(row_wgs + std::max<int64_t>(copy_wgs, 1)), kRowWaves * kWave, 0, st>>>(
        t, ref_counts, (int32_t)num_blocks, c, (int32_t)num_caches, chunks, page_elems, (uint32_t)row_wgs, new_tables,
        new_ref_counts, num_used);
    return record_launch_status(hipGetLastError());
  }
  const PlanOut plan = plan_layout(workspace, num_blocks);
  compact_plan_kernel<<<1, kPlanWaves * kWave, 0, st>>>(ref_counts, (int32_t)num_blocks, num_used, plan);
  compact_kernel<<<(unsigned)(row_wgs + std::max<int64_t>(copy_wgs, 1)), 256, 0, st>>>(
      t, ref_counts, (int32_t)num_blocks, c, (int32_t)num_caches, chunks, page_elems, (uint32_t)row_wgs, new_tables,
      new_ref_counts, plan);
  return record_launch_status(hipGetLastError());
}
