// Operations on whole pages (blocks) of the paged KV cache for NVIDIA B200 (sm_100a), and their C ABI.
//
//   kvc_copy_blocks     page dst <- page src in every cache of a list (all layers, keys and values)
//   kvc_fork_blocks     a new sequence shares its parent's full pages and gets a copy of the last, partly filled one
//   kvc_free_blocks     a finished sequence gives its pages back
//   kvc_compact_blocks  the highest pages in use move into the lowest free ones
//
// State, all of it in device memory and owned by the caller:
//   block_table [num_seqs][width] int32   page of tokens [j * block_size, (j + 1) * block_size) of a sequence
//   seq_lens    [num_seqs] int32          cached tokens; 0 = the row is empty
//   ref_counts  [num_blocks] int32        sequences that hold the page; 0 = the page is free
// There is no free list: the pages a call hands out are the lowest ones whose count is 0, so the result depends on
// the state alone and not on the order in which threads or earlier calls ran.  Nothing is read on the host, so every
// call may be captured into a graph; what a call could not do is told in device memory (`made`, `block_mapping`).
//
// The copies are pure HBM traffic and carry nearly all of the time; the bookkeeping before them is one CTA over the
// page counts (fork, compact) and one pass over the table rows concerned.
#include "kvc_common.cuh"

namespace kvc {

// ---------------------------------------------------------------------------------------------
// bookkeeping
// ---------------------------------------------------------------------------------------------
struct PageTable {
  int32_t* block_table;
  int32_t* seq_lens;
  int32_t* ref_counts;
  int64_t table_stride;
  int64_t num_blocks;
  int32_t num_seqs, width, block_size;
};

constexpr int kPlanThreads = 1024;
constexpr int kPlanWarps = kPlanThreads / 32;
// The bookkeeping CTA holds one bit per page in shared memory.
constexpr int64_t kMaxPages = 200 * 1024 * 8;

// Exclusive prefix sum of `v` over the CTA in thread order; `total` gets the sum.  `part` is kPlanWarps + 1 words.
__device__ __forceinline__ uint32_t cta_prefix(uint32_t v, uint32_t* part, uint32_t& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t sum = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t up = __shfl_up_sync(0xFFFFFFFFu, sum, o);
    if (lane >= o) sum += up;
  }
  __syncthreads();  // the words of an earlier call have been read
  if (lane == 31) part[warp] = sum;
  __syncthreads();
  if (warp == 0) {
    const uint32_t mine = part[lane];
    uint32_t s = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t up = __shfl_up_sync(0xFFFFFFFFu, s, o);
      if (lane >= o) s += up;
    }
    part[lane] = s - mine;
    if (lane == 31) part[kPlanWarps] = s;
  }
  __syncthreads();
  total = part[kPlanWarps];
  return part[warp] + sum - v;
}

// bits[w] bit b = page 32 w + b is in use; bits past the last page are 0.  Eight loads per thread in flight.
__device__ __forceinline__ void load_used_bits(const PageTable& t, uint32_t* bits, uint32_t words) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  constexpr int kDepth = 8;
  for (uint32_t w0 = warp * kDepth; w0 < words; w0 += kPlanWarps * kDepth) {
    int32_t c[kDepth];
#pragma unroll
    for (int i = 0; i < kDepth; ++i) {
      const int64_t page = static_cast<int64_t>(w0 + i) * 32 + lane;
      c[i] = page < t.num_blocks ? __ldcg(t.ref_counts + page) : 0;
    }
#pragma unroll
    for (int i = 0; i < kDepth; ++i) {
      const uint32_t b = __ballot_sync(0xFFFFFFFFu, c[i] > 0);
      if (lane == 0 && w0 + i < words) bits[w0 + i] = b;
    }
  }
}

__device__ __forceinline__ uint32_t mask_below(int64_t n) {  // bits 0 .. n-1
  return n >= 32 ? 0xFFFFFFFFu : n <= 0 ? 0u : (1u << n) - 1u;
}

struct ForkParams {
  PageTable t;
  const int32_t* parents;
  const int32_t* children;
  int64_t* mapping;  // [num_forks][2]
  int32_t* made;     // [num_forks]
  int32_t num_forks;
};

// One CTA decides every fork: whether it can be made, and the page its copy goes to.
//  1. made[i] = the parent's length, or -1 when an index is out of range, the child's row is not empty or the
//     parent's length does not fit the table.  Lengths are read before any of them is changed.
//  2. A child that is named more than once belongs to the first fork that names it: its length, 0 until now, is
//     lowered to -(num_forks - i), and the fork that finds its own mark afterwards has it.
//  3. Forks whose parent ends inside a page are ranked in order; rank r gets the r-th lowest free page.
//  4. Results: lengths, mapping, made.
// mapping doubles as scratch: column 0 of row r holds the fork of rank r until step 4.
__global__ void __launch_bounds__(kPlanThreads) fork_plan_kernel(const ForkParams p) {
  extern __shared__ uint32_t bits[];
  __shared__ uint32_t part[kPlanWarps + 1];
  const PageTable& t = p.t;
  const int n = p.num_forks;
  pdl_prologue();
  const uint32_t words = static_cast<uint32_t>((t.num_blocks + 31) / 32);
  load_used_bits(t, bits, words);
  for (int i = threadIdx.x; i < n; i += kPlanThreads) {
    const int32_t parent = p.parents[i], child = p.children[i];
    int32_t len = -1;
    if (parent >= 0 && parent < t.num_seqs && child >= 0 && child < t.num_seqs) {
      const int32_t l = __ldcg(t.seq_lens + parent);
      const int64_t pages = (static_cast<int64_t>(l) + t.block_size - 1) / t.block_size;
      if (l >= 0 && pages <= t.width && __ldcg(t.seq_lens + child) == 0) len = l;
    }
    p.made[i] = len;
    p.mapping[2 * static_cast<int64_t>(i) + 1] = -1;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kPlanThreads)
    if (p.made[i] > 0) atomicMin(t.seq_lens + p.children[i], i - n);
  __syncthreads();
  uint32_t ranked = 0;
  for (int i0 = 0; i0 < n; i0 += kPlanThreads) {
    const int i = i0 + threadIdx.x;
    bool needs = false;
    if (i < n && p.made[i] > 0) {
      if (__ldcg(t.seq_lens + p.children[i]) != i - n) p.made[i] = -1;
      else needs = p.made[i] % t.block_size != 0;
    }
    uint32_t total;
    const uint32_t rank = ranked + cta_prefix(needs ? 1u : 0u, part, total);
    if (needs) p.mapping[2 * static_cast<int64_t>(rank)] = i;
    ranked += total;
  }
  __syncthreads();
  // every thread owns a run of words: count its free pages, then hand them out in order
  const uint32_t per = (words + kPlanThreads - 1) / kPlanThreads;
  const uint32_t w0 = min(threadIdx.x * per, words), w1 = min(w0 + per, words);
  uint32_t mine = 0, total;
  for (uint32_t w = w0; w < w1; ++w) mine += __popc(~bits[w] & mask_below(t.num_blocks - static_cast<int64_t>(w) * 32));
  uint32_t rank = cta_prefix(mine, part, total);
  for (uint32_t w = w0; w < w1 && rank < ranked; ++w) {
    uint32_t free_bits = ~bits[w] & mask_below(t.num_blocks - static_cast<int64_t>(w) * 32);
    for (; free_bits && rank < ranked; free_bits &= free_bits - 1, ++rank) {
      const int32_t page = static_cast<int32_t>(w * 32 + __ffs(free_bits) - 1);
      const int64_t i = p.mapping[2 * static_cast<int64_t>(rank)];
      p.mapping[2 * i + 1] = page;
      t.ref_counts[page] = 1;
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kPlanThreads) {
    const int32_t len = p.made[i];
    int64_t* pair = p.mapping + 2 * static_cast<int64_t>(i);
    pair[0] = -1;
    if (len <= 0) continue;
    const int32_t child = p.children[i];
    if (len % t.block_size == 0) {
      t.seq_lens[child] = len;
    } else if (pair[1] < 0) {  // no page was left for it
      t.seq_lens[child] = 0;
      p.made[i] = -1;
    } else {
      t.seq_lens[child] = len;
      pair[0] = t.block_table[p.parents[i] * t.table_stride + len / t.block_size];
    }
  }
}

constexpr int kRowThreads = 256;

// By the kRowThreads threads of a CTA: the child's row of fork i, and one more holder for each full page.
__device__ __forceinline__ void fork_row(const ForkParams& p, int i) {
  const PageTable& t = p.t;
  const int32_t len = p.made[i];
  if (len <= 0) return;
  const int32_t full = len / t.block_size;
  const int32_t* from = t.block_table + p.parents[i] * t.table_stride;
  int32_t* to = t.block_table + p.children[i] * t.table_stride;
  for (int32_t j = threadIdx.x; j < full; j += kRowThreads) {
    const int32_t page = from[j];
    to[j] = page;
    if (page >= 0 && page < t.num_blocks) atomicAdd(t.ref_counts + page, 1);
  }
  if (threadIdx.x == 0 && len % t.block_size != 0) to[full] = static_cast<int32_t>(p.mapping[2 * static_cast<int64_t>(i) + 1]);
}

struct FreeParams {
  PageTable t;
  const int32_t* sequences;
};

// One CTA per sequence.  Whoever exchanges the length for 0 frees the pages, so a sequence that is named twice is
// freed once.
__global__ void __launch_bounds__(kRowThreads) free_rows_kernel(const FreeParams p) {
  __shared__ int32_t len;
  const PageTable& t = p.t;
  pdl_prologue();
  const int32_t seq = p.sequences[blockIdx.x];
  if (seq < 0 || seq >= t.num_seqs) return;
  if (threadIdx.x == 0) len = atomicExch(t.seq_lens + seq, 0);
  __syncthreads();
  const int64_t pages = (static_cast<int64_t>(len) + t.block_size - 1) / t.block_size;
  int32_t* row = t.block_table + seq * t.table_stride;
  for (int64_t j = threadIdx.x; j < pages && j < t.width; j += kRowThreads) {
    const int32_t page = row[j];
    if (page >= 0 && page < t.num_blocks) atomicSub(t.ref_counts + page, 1);
    row[j] = -1;
  }
}

struct CompactParams {
  PageTable t;
  int64_t* mapping;  // [max_moves][2]
  int32_t max_moves;
};

// One CTA: with U pages in use, move k takes the k-th highest page in use at or above U to the k-th lowest free page
// below U (there are as many of the one as of the other).  Counts move with the pages; unused rows become -1.
__global__ void __launch_bounds__(kPlanThreads) compact_plan_kernel(const CompactParams p) {
  extern __shared__ uint32_t bits[];
  __shared__ uint32_t part[kPlanWarps + 1];
  const PageTable& t = p.t;
  pdl_prologue();
  const uint32_t words = static_cast<uint32_t>((t.num_blocks + 31) / 32);
  load_used_bits(t, bits, words);
  __syncthreads();
  const uint32_t per = (words + kPlanThreads - 1) / kPlanThreads;
  const uint32_t w0 = min(threadIdx.x * per, words), w1 = min(w0 + per, words);
  uint32_t used = 0, border;
  for (uint32_t w = w0; w < w1; ++w) used += __popc(bits[w]);
  cta_prefix(used, part, border);
  uint32_t holes = 0, strays = 0, moves, same;
  for (uint32_t w = w0; w < w1; ++w) {
    const uint32_t below = mask_below(static_cast<int64_t>(border) - static_cast<int64_t>(w) * 32);
    holes += __popc(~bits[w] & below);
    strays += __popc(bits[w] & ~below);
  }
  uint32_t hole = cta_prefix(holes, part, moves);
  const uint32_t stray = cta_prefix(strays, part, same);
  const uint32_t limit = min(moves, static_cast<uint32_t>(p.max_moves));
  for (uint32_t w = w0; w < w1 && hole < limit; ++w) {
    uint32_t b = ~bits[w] & mask_below(static_cast<int64_t>(border) - static_cast<int64_t>(w) * 32);
    for (; b && hole < limit; b &= b - 1, ++hole) p.mapping[2 * static_cast<int64_t>(hole) + 1] = w * 32 + __ffs(b) - 1;
  }
  uint32_t k = moves - stray;  // the stray of ascending rank s is move moves - 1 - s
  for (uint32_t w = w0; w < w1; ++w) {
    uint32_t b = bits[w] & ~mask_below(static_cast<int64_t>(border) - static_cast<int64_t>(w) * 32);
    for (; b; b &= b - 1) {
      --k;
      if (k < limit) p.mapping[2 * static_cast<int64_t>(k)] = w * 32 + __ffs(b) - 1;
    }
  }
  __syncthreads();
  for (uint32_t r = threadIdx.x; r < static_cast<uint32_t>(p.max_moves); r += kPlanThreads) {
    int64_t* pair = p.mapping + 2 * static_cast<int64_t>(r);
    if (r < limit) {
      t.ref_counts[pair[1]] = t.ref_counts[pair[0]];
      t.ref_counts[pair[0]] = 0;
    } else {
      pair[0] = pair[1] = -1;
    }
  }
}

// By the kRowThreads threads of a CTA: table row i.  The sources of the mapping fall from row to row (the -1 of unused
// rows included), so a page's move, if it has one, is found by bisection.
__device__ __forceinline__ void compact_row(const CompactParams& p, int i) {
  const PageTable& t = p.t;
  int32_t* row = t.block_table + i * t.table_stride;
  const int32_t lowest = static_cast<int32_t>(p.mapping[2 * static_cast<int64_t>(p.max_moves) - 2]);  // -1 unless all rows are in use
  for (int32_t j = threadIdx.x; j < t.width; j += kRowThreads) {
    const int32_t page = row[j];
    if (page < 0 || page < lowest) continue;
    int32_t lo = 0, hi = p.max_moves;  // the first row whose source is <= page
    while (lo < hi) {
      const int32_t mid = (lo + hi) >> 1;
      if (p.mapping[2 * static_cast<int64_t>(mid)] > page) lo = mid + 1;
      else hi = mid;
    }
    if (lo < p.max_moves && p.mapping[2 * static_cast<int64_t>(lo)] == page)
      row[j] = static_cast<int32_t>(p.mapping[2 * static_cast<int64_t>(lo) + 1]);
  }
}

// ---------------------------------------------------------------------------------------------
// copies
// ---------------------------------------------------------------------------------------------
// A launch carries the base addresses of up to kMaxCaches caches in its parameters: nothing has to be uploaded, and a
// captured launch keeps them.
constexpr int kMaxCaches = 256;
constexpr int kCopyThreads = 256;
constexpr int kCopyUnroll = 4;
static_assert(kCopyThreads == kRowThreads, "a CTA of the copy kernel can take a table row");

struct NoRows {};
struct PageCopy {
  void* caches[kMaxCaches];
  const int64_t* mapping;  // (source, destination) per pair
  int64_t num_blocks;
  int64_t block_stride;    // bytes
  int64_t row_stride;      // bytes, between the rows of one page
  int64_t row_vectors;     // vectors of VB bytes per row
  uint32_t n_units;        // pairs * units_per_pair
  uint32_t units_per_pair; // caches * segments
  uint32_t segments;       // rows * segments_per_row
  uint32_t segments_per_row;
  FastDiv div_pair, div_cache, div_row;
  bool packed;             // the pairs in use come first: the first negative one ends the list
  uint32_t table_rows;     // CTAs that follow up the table instead: rows of Rows
};
template <typename Rows>
struct PageCopyParams {
  PageCopy c;
  Rows rows;
};

// The first table_rows CTAs take a row of the table each.  The others stride over units: one segment (kCopyThreads *
// kCopyUnroll vectors) of one page of one cache.  A thread has kCopyUnroll loads in flight before its first store, and the
// next unit's pair of pages is asked for while this one is copied.
template <int VB, typename Rows>
__global__ void __launch_bounds__(kCopyThreads) copy_pages_kernel(const __grid_constant__ PageCopyParams<Rows> params) {
  const PageCopy& p = params.c;
  pdl_prologue();
  if constexpr (!std::is_same_v<Rows, NoRows>) {
    if (blockIdx.x < p.table_rows) {
      if constexpr (std::is_same_v<Rows, ForkParams>) fork_row(params.rows, blockIdx.x);
      else compact_row(params.rows, blockIdx.x);
      return;
    }
  }
  const uint32_t stride = gridDim.x - p.table_rows;
  uint32_t u = blockIdx.x - p.table_rows;
  if (u >= p.n_units) return;
  uint32_t pair = p.div_pair.div(u);
  longlong2 pages = *reinterpret_cast<const longlong2*>(p.mapping + 2 * static_cast<int64_t>(pair));
  while (true) {
    const uint32_t rest = u - pair * p.units_per_pair;
    const int64_t src = pages.x, dst = pages.y;
    const uint32_t next = u + stride;
    if (next < p.n_units) {
      pair = p.div_pair.div(next);
      pages = *reinterpret_cast<const longlong2*>(p.mapping + 2 * static_cast<int64_t>(pair));
    }
    const bool none = src < 0 || dst < 0;
    if (none && p.packed) return;
    if (!none && src != dst && src < p.num_blocks && dst < p.num_blocks) {
      const uint32_t cache = p.div_cache.div(rest);
      const uint32_t segment = rest - cache * p.segments;
      const uint32_t row = p.div_row.div(segment);
      const int64_t first =
          static_cast<int64_t>(segment - row * p.segments_per_row) * (kCopyThreads * kCopyUnroll) + threadIdx.x;
      char* base = static_cast<char*>(p.caches[cache]) + static_cast<int64_t>(row) * p.row_stride;
      const char* from = base + src * p.block_stride;
      char* to = base + dst * p.block_stride;
      Chunk<VB> v[kCopyUnroll];
#pragma unroll
      for (int i = 0; i < kCopyUnroll; ++i)
        if (first + i * kCopyThreads < p.row_vectors) load_chunk_inplace(v[i], from + (first + i * kCopyThreads) * VB);
#pragma unroll
      for (int i = 0; i < kCopyUnroll; ++i)
        if (first + i * kCopyThreads < p.row_vectors) store_chunk(to + (first + i * kCopyThreads) * VB, v[i], VB == 32);
    }
    if (next >= p.n_units) return;
    u = next;
  }
}

// ---------------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------------
namespace {

struct PageGeometry {
  void* const* caches;
  int64_t num_caches, num_blocks, block_stride, rows, row_bytes, row_stride;  // strides in bytes
};

int check_geometry(const char* op, const PageGeometry& g) {
  const std::string name(op);
  if (g.num_caches < 0 || g.num_blocks < 0 || g.rows < 0 || g.row_bytes < 0)
    return fail(KVC_ERR_INVALID_ARG, name + ": negative size");
  if (g.num_caches > 0 && !g.caches) return fail(KVC_ERR_INVALID_ARG, name + ": the list of caches must be non-NULL");
  for (int64_t i = 0; i < g.num_caches; ++i)
    if (!g.caches[i] && g.num_blocks > 0 && g.rows > 0 && g.row_bytes > 0)
      return fail(KVC_ERR_INVALID_ARG, name + ": a cache of the list is NULL");
  return KVC_OK;
}

// How the pages are cut into units: the widest access that every address and length allows, segments per row, and units per
// pair of pages.  Refuses what does not fit a launch; fork and compact ask before their plan changes the state.
struct PageCut {
  int vb;
  int64_t per_row, per_cache;
};
int cut_pages(const char* op, const PageGeometry& g, PageCut& cut) {
  cut = PageCut{32, 1, 1};
  if (g.num_caches == 0 || g.num_blocks == 0 || g.rows == 0 || g.row_bytes == 0) return KVC_OK;  // nothing to copy
  for (; cut.vb > 1; cut.vb >>= 1) {
    const int vb = cut.vb;
    bool ok = g.row_bytes % vb == 0 && g.block_stride % vb == 0 && (g.rows == 1 || g.row_stride % vb == 0);
    for (int64_t i = 0; ok && i < g.num_caches; ++i) ok = aligned(g.caches[i], vb);
    if (ok) break;
  }
  cut.per_row = (g.row_bytes / cut.vb - 1) / (kCopyThreads * kCopyUnroll) + 1;
  const int64_t caches = g.num_caches < kMaxCaches ? g.num_caches : kMaxCaches, most = ((1ll << 30) - 1) / caches;
  if (g.rows > most || cut.per_row > most || g.rows * cut.per_row > most)
    return fail(KVC_ERR_TOO_LARGE, std::string(op) + ": a page is too large");
  cut.per_cache = g.rows * cut.per_row;
  return KVC_OK;
}

// Copies the pages of `pairs` rows of `mapping` in all caches, and follows up `table_rows` rows of the table beside them.
template <typename Rows>
int copy_pages(const char* op, const PageGeometry& g, const int64_t* mapping, int64_t pairs, bool packed, int64_t table_rows,
               const Rows& rows, cudaStream_t st) {
  if (g.num_caches == 0 || g.num_blocks == 0 || g.rows == 0 || g.row_bytes == 0) pairs = 0;  // nothing to copy
  PageCut cut{1, 1, 1};
  if (pairs > 0)
    if (int rc = cut_pages(op, g, cut)) return rc;
  const int vb = cut.vb;
  PageCopyParams<Rows> params{};
  params.rows = rows;
  PageCopy& p = params.c;
  p.num_blocks = g.num_blocks;
  p.block_stride = g.block_stride;
  p.row_stride = g.row_stride;
  p.row_vectors = g.row_bytes / vb;
  p.packed = packed;
  int64_t c0 = 0;
  do {
    const int64_t nc = g.num_caches - c0 < kMaxCaches ? g.num_caches - c0 : kMaxCaches;
    for (int64_t i = 0; i < nc; ++i) p.caches[i] = g.caches[c0 + i];
    const int64_t per_pair = pairs > 0 ? nc * cut.per_cache : 1;
    p.units_per_pair = static_cast<uint32_t>(per_pair);
    p.segments = static_cast<uint32_t>(cut.per_cache);
    p.segments_per_row = static_cast<uint32_t>(cut.per_row);
    p.div_pair = FastDiv(p.units_per_pair);
    p.div_cache = FastDiv(p.segments);
    p.div_row = FastDiv(p.segments_per_row);
    const int64_t step = ((1ll << 31) - (1 << 20)) / per_pair;
    int64_t i0 = 0;
    do {
      const int64_t np = pairs - i0 < step ? pairs - i0 : step;
      p.mapping = mapping + 2 * i0;
      p.n_units = static_cast<uint32_t>(np * per_pair);
      p.table_rows = c0 == 0 && i0 == 0 ? static_cast<uint32_t>(table_rows) : 0;
      const dim3 grid(p.table_rows + (p.n_units < 148u * 8u ? p.n_units : 148u * 8u));
      if (grid.x > 0) {
        cudaError_t e;
        switch (vb) {
          case 32: e = launch_pdl(copy_pages_kernel<32, Rows>, grid, kCopyThreads, params, st); break;
          case 16: e = launch_pdl(copy_pages_kernel<16, Rows>, grid, kCopyThreads, params, st); break;
          case 8: e = launch_pdl(copy_pages_kernel<8, Rows>, grid, kCopyThreads, params, st); break;
          case 4: e = launch_pdl(copy_pages_kernel<4, Rows>, grid, kCopyThreads, params, st); break;
          case 2: e = launch_pdl(copy_pages_kernel<2, Rows>, grid, kCopyThreads, params, st); break;
          default: e = launch_pdl(copy_pages_kernel<1, Rows>, grid, kCopyThreads, params, st); break;
        }
        if (e != cudaSuccess)
          return fail(KVC_ERR_CUDA, std::string(op) + " launch failed: " + cudaGetErrorString(e));
      }
      i0 += step;
    } while (i0 < pairs);
    c0 += kMaxCaches;
  } while (c0 < g.num_caches);
  return KVC_OK;
}

int check_table(const char* op, const PageTable& t, int64_t num_seqs, int64_t width, int64_t block_size, bool lens = true) {
  const std::string name(op);
  if (num_seqs < 0 || width < 0 || t.num_blocks < 0) return fail(KVC_ERR_INVALID_ARG, name + ": negative size");
  if (block_size <= 0) return fail(KVC_ERR_INVALID_ARG, name + ": block_size must be positive");
  if (num_seqs > 0x7FFFFFFFll || width > 0x7FFFFFFFll || block_size > 0x7FFFFFFFll)
    return fail(KVC_ERR_INVALID_ARG, name + ": sizes out of range");
  if (t.num_blocks > kMaxPages)
    return fail(KVC_ERR_TOO_LARGE, name + ": more than " + std::to_string(kMaxPages) + " pages");
  if ((num_seqs > 0 && ((lens && !t.seq_lens) || (width > 0 && !t.block_table))) || (t.num_blocks > 0 && !t.ref_counts))
    return fail(KVC_ERR_INVALID_ARG, name + ": block_table, seq_lens and ref_counts must be non-NULL");
  if (!aligned(t.block_table, 4) || !aligned(t.seq_lens, 4) || !aligned(t.ref_counts, 4))
    return fail(KVC_ERR_INVALID_ARG, name + ": block_table, seq_lens and ref_counts must be 4-byte aligned");
  return KVC_OK;
}

PageTable make_table(int32_t* block_table, int32_t* seq_lens, int32_t* ref_counts, int64_t num_seqs, int64_t width,
                     int64_t table_stride, int64_t num_blocks, int64_t block_size) {
  return PageTable{block_table, seq_lens, ref_counts, table_stride, num_blocks, static_cast<int32_t>(num_seqs),
                   static_cast<int32_t>(width), static_cast<int32_t>(block_size)};
}

// The bookkeeping CTA: its bits are dynamic shared memory, beyond the default limit for many pages.  The limit is raised to
// the same value by every call: two threads' calls, or a captured one and a later one, may need different amounts.
template <typename Params>
int launch_plan(const char* op, void (*kernel)(const Params), const Params& p, cudaStream_t st) {
  const size_t smem = static_cast<size_t>((p.t.num_blocks + 31) / 32) * 4;
  if (smem > 40 * 1024)
    KVC_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kMaxPages / 8)));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(1);
  cfg.blockDim = dim3(kPlanThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p);
  if (e != cudaSuccess) return fail(KVC_ERR_CUDA, std::string(op) + " launch failed: " + cudaGetErrorString(e));
  return KVC_OK;
}

template <typename Params>
int launch_rows(const char* op, void (*kernel)(const Params), int64_t rows, const Params& p, cudaStream_t st) {
  const cudaError_t e = launch_pdl(kernel, dim3(static_cast<unsigned>(rows)), kRowThreads, p, st);
  if (e != cudaSuccess) return fail(KVC_ERR_CUDA, std::string(op) + " launch failed: " + cudaGetErrorString(e));
  return KVC_OK;
}

}  // namespace
}  // namespace kvc

// ---------------------------------------------------------------------------------------------
// C ABI
// ---------------------------------------------------------------------------------------------
extern "C" {

KVC_API int kvc_copy_blocks(void* const* caches, int64_t num_caches, const int64_t* block_mapping, int64_t num_pairs,
                            int64_t num_blocks, int64_t block_stride, int64_t rows_per_block, int64_t row_bytes,
                            int64_t row_stride, void* stream) {
  constexpr const char* op = "copy_blocks";
  const kvc::PageGeometry g{caches, num_caches, num_blocks, block_stride, rows_per_block, row_bytes, row_stride};
  if (int rc = kvc::check_geometry(op, g)) return rc;
  if (num_pairs < 0) return kvc::fail(KVC_ERR_INVALID_ARG, "copy_blocks: negative size");
  if (num_pairs > 0 && !block_mapping)
    return kvc::fail(KVC_ERR_INVALID_ARG, "copy_blocks: block_mapping must be non-NULL");
  if (!kvc::aligned(block_mapping, 16))
    return kvc::fail(KVC_ERR_INVALID_ARG, "copy_blocks: block_mapping must be 16-byte aligned");
  return kvc::copy_pages(op, g, block_mapping, num_pairs, false, 0, kvc::NoRows{}, static_cast<cudaStream_t>(stream));
}

KVC_API int kvc_fork_blocks(int32_t* block_table, int32_t* seq_lens, int32_t* ref_counts, const int32_t* parents,
                            const int32_t* children, int64_t num_forks, int64_t num_seqs, int64_t table_width,
                            int64_t table_stride, int64_t num_blocks, int64_t block_size, void* const* caches,
                            int64_t num_caches, int64_t block_stride, int64_t rows_per_block, int64_t row_bytes,
                            int64_t row_stride, int64_t* block_mapping, int32_t* made, void* stream) {
  constexpr const char* op = "fork_blocks";
  const kvc::PageGeometry g{caches, num_caches, num_blocks, block_stride, rows_per_block, row_bytes, row_stride};
  if (int rc = kvc::check_geometry(op, g)) return rc;
  kvc::ForkParams p{};
  p.t = kvc::make_table(block_table, seq_lens, ref_counts, num_seqs, table_width, table_stride, num_blocks, block_size);
  if (int rc = kvc::check_table(op, p.t, num_seqs, table_width, block_size)) return rc;
  if (num_forks < 0 || num_forks > 0x3FFFFFFFll) return kvc::fail(KVC_ERR_INVALID_ARG, "fork_blocks: bad number of forks");
  if (num_forks == 0) return KVC_OK;
  if (!parents || !children || !block_mapping || !made)
    return kvc::fail(KVC_ERR_INVALID_ARG, "fork_blocks: parents, children, block_mapping and made must be non-NULL");
  if (!kvc::aligned(parents, 4) || !kvc::aligned(children, 4) || !kvc::aligned(made, 4) || !kvc::aligned(block_mapping, 16))
    return kvc::fail(KVC_ERR_INVALID_ARG, "fork_blocks: index arrays must be aligned to their rows (4 and 16 bytes)");
  p.parents = parents;
  p.children = children;
  p.mapping = block_mapping;
  p.made = made;
  p.num_forks = static_cast<int32_t>(num_forks);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  kvc::PageCut cut;
  if (int rc = kvc::cut_pages(op, g, cut)) return rc;
  if (int rc = kvc::launch_plan(op, kvc::fork_plan_kernel, p, st)) return rc;
  return kvc::copy_pages(op, g, block_mapping, num_forks, false, num_forks, p, st);
}

KVC_API int kvc_free_blocks(int32_t* block_table, int32_t* seq_lens, int32_t* ref_counts, const int32_t* sequences,
                            int64_t num_sequences, int64_t num_seqs, int64_t table_width, int64_t table_stride,
                            int64_t num_blocks, int64_t block_size, void* stream) {
  constexpr const char* op = "free_blocks";
  kvc::FreeParams p{};
  p.t = kvc::make_table(block_table, seq_lens, ref_counts, num_seqs, table_width, table_stride, num_blocks, block_size);
  if (int rc = kvc::check_table(op, p.t, num_seqs, table_width, block_size)) return rc;
  if (num_sequences < 0 || num_sequences > 0x7FFFFFFFll)
    return kvc::fail(KVC_ERR_INVALID_ARG, "free_blocks: bad number of sequences");
  if (num_sequences == 0) return KVC_OK;
  if (!sequences || !kvc::aligned(sequences, 4))
    return kvc::fail(KVC_ERR_INVALID_ARG, "free_blocks: sequences must be non-NULL and 4-byte aligned");
  p.sequences = sequences;
  return kvc::launch_rows(op, kvc::free_rows_kernel, num_sequences, p, static_cast<cudaStream_t>(stream));
}

KVC_API int kvc_compact_blocks(int32_t* block_table, int32_t* ref_counts, int64_t num_seqs, int64_t table_width,
                               int64_t table_stride, int64_t num_blocks, void* const* caches, int64_t num_caches,
                               int64_t block_stride, int64_t rows_per_block, int64_t row_bytes, int64_t row_stride,
                               int64_t* block_mapping, int64_t max_moves, void* stream) {
  constexpr const char* op = "compact_blocks";
  const kvc::PageGeometry g{caches, num_caches, num_blocks, block_stride, rows_per_block, row_bytes, row_stride};
  if (int rc = kvc::check_geometry(op, g)) return rc;
  kvc::CompactParams p{};
  p.t = kvc::make_table(block_table, nullptr, ref_counts, num_seqs, table_width, table_stride, num_blocks, 1);
  if (int rc = kvc::check_table(op, p.t, num_seqs, table_width, 1, false)) return rc;
  if (num_seqs > 0x3FFFFFFFll) return kvc::fail(KVC_ERR_INVALID_ARG, "compact_blocks: sizes out of range");  // a CTA per row
  if (max_moves < 0 || max_moves > 0x3FFFFFFFll)
    return kvc::fail(KVC_ERR_INVALID_ARG, "compact_blocks: bad number of moves");
  if (max_moves == 0) return KVC_OK;
  if (!block_mapping || !kvc::aligned(block_mapping, 16))
    return kvc::fail(KVC_ERR_INVALID_ARG, "compact_blocks: block_mapping must be non-NULL and 16-byte aligned");
  p.mapping = block_mapping;
  p.max_moves = static_cast<int32_t>(max_moves);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  kvc::PageCut cut;
  if (int rc = kvc::cut_pages(op, g, cut)) return rc;
  if (int rc = kvc::launch_plan(op, kvc::compact_plan_kernel, p, st)) return rc;
  return kvc::copy_pages(op, g, block_mapping, max_moves, true, table_width > 0 ? num_seqs : 0, p, st);
}

}  // extern "C"
