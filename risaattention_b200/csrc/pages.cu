// Pages of a cache shared, handed out, given back and moved together: what belongs to the page tables rather than to the
// tokens.  `references` counts for each page how many entries of page tables lead to it; a page with none is free.  All of it
// happens on the device in a fixed order, so results do not depend on timing: the lowest free pages go first, to the sequences
// in their order.
#include "serving_plan.cuh"

#include <algorithm>

namespace risa_b200 {
namespace serving {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kPlanEach = 16;  // pages that a planning thread looks at in a round

// Exclusive prefix of the block's values and their total.
__device__ __forceinline__ int block_prefix(int v, int* warp_sums, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int through = v;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int below = __shfl_up_sync(0xffffffffu, through, off);
    if (lane >= off) through += below;
  }
  __syncthreads();  // an earlier round's sums are read
  if (lane == 31) warp_sums[warp] = through;
  __syncthreads();
  const int mine = lane < int(blockDim.x >> 5) ? warp_sums[lane] : 0;
  total = __reduce_add_sync(0xffffffffu, mine);
  return __reduce_add_sync(0xffffffffu, lane < warp ? mine : 0) + through - v;
}

__device__ __forceinline__ int pages_for(int tokens, int page_shift) { return (tokens >> page_shift) + ((tokens & ((1 << page_shift) - 1)) != 0); }

// ---- fork ---------------------------------------------------------------------------------------------------
struct ForkArgs {
  StepView step;
  int32_t* references;
  const int32_t* parents;
  int32_t* table;
  int32_t* lengths;
  int pages;
  unsigned int* status;
};

// A thread per entry of a child's row (grid y over them).
__global__ __launch_bounds__(256) void fork_kernel(const ForkArgs a) {
  chain_wait();
  chain_release();
  const int child = blockIdx.x, column = blockIdx.y * 256 + threadIdx.x;
  const int parent = __ldg(a.parents + child);
  int length = 0;
  if (parent >= 0 && parent < a.step.batch) length = min(max(__ldg(a.step.lengths + parent), 0), a.step.width << a.step.page_shift);
  if (column == 0) a.lengths[child] = length;
  if (column >= a.step.width) return;
  int page = -1;
  if (column < pages_for(length, a.step.page_shift)) {
    page = __ldg(a.step.table + int64_t(parent) * a.step.width + column);
    if (page >= 0 && page < a.pages) atomicAdd(a.references + page, 1);
    else atomicCAS(a.status, 0u, unsigned(parent) + 1u);
  }
  a.table[int64_t(child) * a.step.width + column] = page;
}

// ---- resize -------------------------------------------------------------------------------------------------
// A sequence on its way from `length` to `wanted` tokens.
struct Change {
  int length, wanted, held, needed;  // tokens, pages
  int shared;                        // a last page that must not be written to, or -1
  __device__ __forceinline__ int need() const { return wanted > length ? (shared >= 0) + max(needed - held, 0) : 0; }
};
struct ResizeArgs {
  int32_t* table;
  const int32_t* lengths;
  const int32_t* wanted;
  int32_t* granted;
  int32_t* references;
  int batch, width, page_shift, pages;
  // the plan: both lengths of each sequence as they were (`granted` may lie over them), pages that sequences in front of it need,
  // the shared page that it leaves, and the pages handed out
  int32_t* was;
  int32_t* asked;
  int32_t* before;
  int32_t* left;
  int32_t* fresh;
  int32_t* counts;  // of pages needed and found
  char* keys;
  char* values;
  char* key_scales;
  char* value_scales;
  int kv_heads, row_bytes, token_scales, group_scales;  // bytes: of a row, of a token's scale, of its groups' scales beside that
  unsigned int* status;
};

__device__ __forceinline__ Change change_of(const ResizeArgs& a, int length, int wanted, int shared) {
  return {length, wanted, pages_for(length, a.page_shift), pages_for(wanted, a.page_shift), shared};
}
// As planned.
__device__ __forceinline__ Change planned_change(const ResizeArgs& a, int s) { return change_of(a, a.was[s], a.asked[s], a.left[s]); }

// One CTA: what each sequence needs, added up in order; then free pages, lowest first, until there are enough (16 K a round); then
// what each sequence is granted.
struct PlanShared {
  BlockScan<kPlanThreads> scan;  // needs can add up past 32 bits
  int warp_sums[32];
};
__device__ __forceinline__ void plan_resize(const ResizeArgs& a, PlanShared& shared) {
  int needed = 0;
  for (int s0 = 0; s0 < a.batch; s0 += kPlanThreads) {
    const int s = s0 + threadIdx.x;
    int need = 0;
    if (s < a.batch) {
      const int most = a.width << a.page_shift;
      Change c = change_of(a, min(max(a.lengths[s], 0), most), min(max(a.wanted[s], 0), most), -1);
      if (c.wanted > c.length && (c.length & ((1 << a.page_shift) - 1)) != 0) {
        const int last = a.table[int64_t(s) * a.width + c.held - 1];
        if (last < 0 || last >= a.pages) atomicCAS(a.status, 0u, unsigned(s) + 1u);
        else if (a.references[last] > 1) c.shared = last;
      }
      need = c.need();
      a.was[s] = c.length;
      a.asked[s] = c.wanted;
      a.left[s] = c.shared;
    }
    int64_t total;
    const int64_t before = needed + block_inclusive_scan<kPlanThreads>(need, shared.scan, total) - need;
    if (s < a.batch) a.before[s] = int(min(before, int64_t(a.pages)));
    needed = int(min(needed + total, int64_t(a.pages)));  // more than there are: nobody behind gets any
  }
  int found = 0;
  for (int p0 = 0; p0 < a.pages && found < needed; p0 += kPlanThreads * kPlanEach) {
    const int first = p0 + threadIdx.x * kPlanEach;
    uint32_t free_pages = 0;
#pragma unroll
    for (int i = 0; i < kPlanEach; ++i)
      if (first + i < a.pages && a.references[first + i] == 0) free_pages |= 1u << i;
    int total, rank = found + block_prefix(__popc(free_pages), shared.warp_sums, total);
    for (; free_pages != 0 && rank < needed; free_pages &= free_pages - 1) a.fresh[rank++] = first + __ffs(free_pages) - 1;
    found += total;
  }
  if (threadIdx.x == 0) a.counts[0] = min(found, needed);
  found = min(found, needed);
  for (int s = threadIdx.x; s < a.batch; s += kPlanThreads) {
    const Change c = planned_change(a, s);
    const int need = c.need(), given = max(min(found - a.before[s], need), 0);
    int length = c.wanted;
    if (given < need) {
      // a shared page that could not be replaced must not be written to; else as far as the pages reach
      const int whole = (c.held + given - (c.shared >= 0 ? 1 : 0)) << a.page_shift;
      length = given == 0 && c.shared >= 0 ? c.length : min(c.wanted, whole);
    }
    a.granted[s] = length;
  }
}

// By `step` threads, of which this is the `first`-th: entries and counts, then the rows of a page that was shared.
__device__ __forceinline__ void apply_resize(const ResizeArgs& a, int s, int first, int step) {
  const Change c = planned_change(a, s);
  const int found = a.counts[0], before = a.before[s], given = max(min(found - before, c.need()), 0);
  const bool copies = c.shared >= 0 && given > 0;
  int32_t* row = a.table + int64_t(s) * a.width;
  for (int i = first; i < given; i += step) {
    const int page = a.fresh[before + i], column = copies ? c.held - 1 + i : c.held + i;
    a.references[page] = 1;
    row[column] = page;
  }
  if (copies && first == 0) atomicAdd(a.references + c.shared, -1);
  for (int i = c.needed + first; i < c.held; i += step) {  // given back
    const int page = row[i];
    if (page >= 0 && page < a.pages) atomicAdd(a.references + page, -1);
    else atomicCAS(a.status, 0u, unsigned(s) + 1u);
    row[i] = -1;
  }
  if (!copies) return;
  const int64_t from = int64_t(c.shared) * a.kv_heads, to = int64_t(a.fresh[before]) * a.kv_heads;
  const int rows = c.length & ((1 << a.page_shift) - 1), pieces = a.row_bytes >> 4, each = rows * pieces;  // of a head
  for (int i = first; i < a.kv_heads * each; i += step) {
    const int h = i / each;
    const int64_t in_head = int64_t(i - h * each) * 16, head_bytes = int64_t(a.row_bytes) << a.page_shift;
    const uint4 k = *reinterpret_cast<const uint4*>(a.keys + (from + h) * head_bytes + in_head);
    const uint4 v = *reinterpret_cast<const uint4*>(a.values + (from + h) * head_bytes + in_head);
    *reinterpret_cast<uint4*>(a.keys + (to + h) * head_bytes + in_head) = k;
    *reinterpret_cast<uint4*>(a.values + (to + h) * head_bytes + in_head) = v;
  }
  if (a.token_scales == 0) return;
  // scales byte by byte: of the tokens, then (behind those of all the page's tokens) of their groups (256 shared pages of 31 tokens of
  // 8 heads of 128: 10.5 us of INT8 and 4-bit rows, 12.7 of bf16 ones, which are two and four times as many bytes)
  const int64_t block = int64_t(a.token_scales + a.group_scales) << a.page_shift;
  const int of_tokens = rows * a.token_scales, of_head = of_tokens + rows * a.group_scales;
  for (int i = first; i < a.kv_heads * of_head; i += step) {
    const int h = i / of_head, j = i - h * of_head;
    const int64_t at = j < of_tokens ? j : (int64_t(a.token_scales) << a.page_shift) + j - of_tokens;
    a.key_scales[(to + h) * block + at] = a.key_scales[(from + h) * block + at];
    a.value_scales[(to + h) * block + at] = a.value_scales[(from + h) * block + at];
  }
}

__global__ __launch_bounds__(kPlanThreads) void resize_plan_kernel(const ResizeArgs a) {
  __shared__ PlanShared shared;
  chain_wait();
  chain_release();
  plan_resize(a, shared);
}
__global__ __launch_bounds__(256) void resize_apply_kernel(const ResizeArgs a) {
  chain_wait();
  chain_release();
  apply_resize(a, blockIdx.x, blockIdx.y * blockDim.x + threadIdx.x, gridDim.y * blockDim.x);
}
// Both in one launch where there is little to do: a cluster of eight CTAs, of which the first one plans.  Its warps are dealt to
// the sequences, so that the chains of look-ups of as many run side by side (64 sequences that grow within their pages 5.0 us on
// the GPU, 4.5 as two launches; calls in a row, which the host bounds, 8.3 and 10.4).  More sequences than warps, and more bytes
// than this that all together can have copied, are for two launches: 4096 sequences 20.7 and 15.9 us, 256 with 4 MB to copy 21.8
// and 8.9, with 1 MB 10.2 and 8.0.
constexpr int kResizeCtas = 8, kResizeWarps = kResizeCtas * kPlanThreads / 32;
constexpr int64_t kLittle = 4 << 20;
__global__ __cluster_dims__(kResizeCtas, 1, 1) __launch_bounds__(kPlanThreads) void resize_kernel(const ResizeArgs a) {
  __shared__ PlanShared shared;
  chain_wait();
  chain_release();
  if (blockIdx.x == 0) plan_resize(a, shared);
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  const int thread = blockIdx.x * kPlanThreads + threadIdx.x, each = kResizeWarps / a.batch * 32, s = thread / each;
  if (s < a.batch) apply_resize(a, s, thread - s * each, each);
}

// ---- compact ------------------------------------------------------------------------------------------------
struct CompactArgs {
  StepView step;
  const int32_t* references;
  int32_t* place;   // of each page in the target, -1: nowhere
  int32_t* source;  // the page that goes to each place, -1: none
  int32_t* table;
  int32_t* target_references;
  int32_t* used;
  int pages, target_pages;
  const char* from[4];  // keys, values, their scales
  char* to[4];
  int units[2];         // of a page: 16-byte pieces of rows, 4-byte pieces of scales
  int pages_each;       // pages that a copying CTA takes where they are small
  unsigned int parts[2], copies[2];  // CTAs of such a group of pages, CTAs in all, of rows and of scales
  unsigned int* status;
};

// The place of a page is the number of pages in use in front of it.  A CTA places 16 K pages; it counts those in front of them by
// itself (256 KB of counters for a pool of 64 K pages, from L2).
__global__ __launch_bounds__(kPlanThreads) void compact_plan_kernel(const CompactArgs a) {
  __shared__ int warp_sums[32];
  chain_wait();
  chain_release();
  const int p0 = blockIdx.x * (kPlanThreads * kPlanEach), first = p0 + threadIdx.x * kPlanEach;
  int in_front = 0;
#pragma unroll 8
  for (int p = threadIdx.x; p < p0; p += kPlanThreads) in_front += __ldg(a.references + p) > 0;
  int base, total;
  block_prefix(in_front, warp_sums, base);
  uint32_t in_use = 0;
#pragma unroll
  for (int i = 0; i < kPlanEach; ++i)
    if (first + i < a.pages && __ldg(a.references + first + i) > 0) in_use |= 1u << i;
  int rank = base + block_prefix(__popc(in_use), warp_sums, total);
#pragma unroll 1
  for (int i = 0; i < kPlanEach && first + i < a.pages; ++i) {
    const bool moves = (in_use >> i & 1) && rank < a.target_pages;
    a.place[first + i] = moves ? rank : -1;
    if (moves) {
      a.source[rank] = first + i;
      a.target_references[rank] = __ldg(a.references + first + i);
    }
    rank += in_use >> i & 1;
  }
  if (blockIdx.x == gridDim.x - 1) {
    if (threadIdx.x == 0) *a.used = base + total;
    for (int p = base + total + threadIdx.x; p < a.target_pages; p += kPlanThreads) {
      a.source[p] = -1;
      a.target_references[p] = 0;
    }
  }
}

// CTAs that copy rows to places of the target, then those that copy scales, then those that rewrite the tables.  Eight loads of a
// thread are on their way at once.  (CTAs of pages that stand empty, and as many for the tables as for rows: 32 requests in half
// of a pool, 671 MB, 256 us.)
constexpr int kCopyAhead = 4;
template <typename V>
__device__ __forceinline__ void copy_pages(const CompactArgs& a, int kind, unsigned int block) {
  const int units = a.units[kind];
  const unsigned int group = block / a.parts[kind], part = block - group * a.parts[kind];
  const int64_t place0 = int64_t(group) * a.pages_each;
  // units of the places [place0, place0 + pages_each), 256 * kCopyAhead of them for each part
  const V* from_k = reinterpret_cast<const V*>(a.from[2 * kind]);
  const V* from_v = reinterpret_cast<const V*>(a.from[2 * kind + 1]);
  V* to_k = reinterpret_cast<V*>(a.to[2 * kind]);
  V* to_v = reinterpret_cast<V*>(a.to[2 * kind + 1]);
  V k[kCopyAhead], v[kCopyAhead];
  int64_t to[kCopyAhead];
#pragma unroll
  for (int i = 0; i < kCopyAhead; ++i) {
    const int64_t u = (int64_t(part) * kCopyAhead + i) * 256 + threadIdx.x;
    to[i] = -1;
    const int64_t in_group = a.pages_each == 1 ? 0 : u / units, place = place0 + in_group;
    const int64_t in_page = u - in_group * units;
    if (in_group < a.pages_each && in_page < units && place < a.target_pages) {
      const int64_t page = __ldg(a.source + place);
      if (page >= 0) {
        to[i] = place * units + in_page;
        k[i] = __ldg(from_k + page * units + in_page);
        v[i] = __ldg(from_v + page * units + in_page);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < kCopyAhead; ++i)
    if (to[i] >= 0) {
      to_k[to[i]] = k[i];
      to_v[to[i]] = v[i];
    }
}
__global__ __launch_bounds__(256) void compact_copy_kernel(const CompactArgs a) {
  chain_wait();
  chain_release();
  if (blockIdx.x < a.copies[0]) return copy_pages<uint4>(a, 0, blockIdx.x);
  const unsigned int behind = blockIdx.x - a.copies[0];
  if (behind < a.copies[1]) return copy_pages<uint32_t>(a, 1, behind);
  const int64_t entries = int64_t(a.step.batch) * a.step.width, threads = int64_t(gridDim.x - a.copies[0] - a.copies[1]) * 256;
  for (int64_t i = int64_t(behind - a.copies[1]) * 256 + threadIdx.x; i < entries; i += threads) {
    const int s = int(i / a.step.width), column = int(i - int64_t(s) * a.step.width);
    const int length = min(max(__ldg(a.step.lengths + s), 0), a.step.width << a.step.page_shift);
    int place = -1;
    if (column < pages_for(length, a.step.page_shift)) {
      const int page = __ldg(a.step.table + i);
      if (page >= 0 && page < a.pages) place = a.place[page];
      else atomicCAS(a.status, 0u, unsigned(s) + 1u);
    }
    a.table[i] = place;
  }
}

int check_table(const void* table, const void* lengths, int batch, int width, const risa_b200_cache* cache, const char* what) {
  RISA_REQUIRE(table && lengths && batch > 0 && batch <= 65535 && width > 0, "%s: null table, or batch not in 1..65535", what);
  RISA_REQUIRE(int64_t(width) * cache->page_size < RISA_B200_CACHE_MOST_SLOTS, "%s: a sequence may hold fewer than 2^31 - 8192 keys", what);
  return RISA_B200_OK;
}
int shift_of(int page_size) {
  int shift = 4;
  while ((1 << shift) < page_size) ++shift;
  return shift;
}
// Bytes of a token's scale (of one head and pool) and of its groups' scales.
int token_scale_of(const risa_b200_cache& c) { return c.dtype_code == kInt8 ? 4 : c.dtype_code == kInt4 ? 1 : 0; }
int group_scales_of(const risa_b200_cache& c) { return c.dtype_code == kInt4 ? c.head_dim / 16 : 0; }

}  // namespace
}  // namespace serving
}  // namespace risa_b200

using namespace risa_b200;
using namespace risa_b200::serving;

extern "C" int risa_b200_fork_sequences(const risa_b200_cache* cache, int32_t* references, const risa_b200_step* step, const int32_t* parents,
                                        int children, int32_t* table, int32_t* lengths, void* stream_ptr) {
  if (const int bad = check_cache(cache, "fork")) return bad;
  RISA_REQUIRE(step != nullptr, "fork: null step");
  if (const int bad = check_table(step->page_table, step->lengths, step->batch, step->table_width, cache, "fork")) return bad;
  RISA_REQUIRE(references && parents && table && lengths, "fork: null tensor");
  RISA_REQUIRE(children > 0, "fork: no children");
  RISA_REQUIRE((step->table_width + 255) / 256 <= 65535, "fork: the page table is too wide");
  unsigned int* status = status_word();
  if (status == nullptr) return RISA_B200_CUDA;
  const ForkArgs a{{step->page_table, step->lengths, nullptr, step->batch, step->table_width, 0, shift_of(cache->page_size)},
                   references, parents, table, lengths, cache->pages, status};
  return launched(launch_chained(fork_kernel, dim3(children, (step->table_width + 255) / 256), dim3(256), 0, static_cast<cudaStream_t>(stream_ptr), a), "fork");
}

extern "C" size_t risa_b200_resize_scratch_size(const risa_b200_cache* cache, int batch) {
  if (cache == nullptr || batch <= 0) return 0;
  return sizeof(int32_t) * (4 * size_t(batch) + size_t(std::max(cache->pages, 0)) + 1);
}

extern "C" int risa_b200_resize_sequences(const risa_b200_cache* cache, int32_t* references, int32_t* page_table, int table_width,
                                          const int32_t* lengths, const int32_t* new_lengths, int batch, int32_t* granted, void* scratch,
                                          size_t scratch_bytes, void* stream_ptr) {
  if (const int bad = check_cache(cache, "resize")) return bad;
  if (const int bad = check_table(page_table, lengths, batch, table_width, cache, "resize")) return bad;
  RISA_REQUIRE(references && new_lengths && granted, "resize: null tensor");
  RISA_REQUIRE(scratch != nullptr && reinterpret_cast<uintptr_t>(scratch) % 4 == 0 && scratch_bytes >= risa_b200_resize_scratch_size(cache, batch),
               "resize: the scratch is too small");
  const int row_bytes = cache->head_dim * bits_of(*cache) / 8;
  // what is copied of a page is counted in 32 bits
  RISA_REQUIRE(int64_t(cache->kv_heads) * cache->page_size * row_bytes < (int64_t(1) << 31), "resize: a page is too large");
  unsigned int* status = status_word();
  if (status == nullptr) return RISA_B200_CUDA;
  int32_t* words = static_cast<int32_t*>(scratch);
  const ResizeArgs a{page_table, lengths, new_lengths, granted, references, batch, table_width, shift_of(cache->page_size), cache->pages,
                     words + 1, words + 1 + batch, words + 1 + 2 * int64_t(batch), words + 1 + 3 * int64_t(batch), words + 1 + 4 * int64_t(batch), words,
                     static_cast<char*>(cache->keys), static_cast<char*>(cache->values), reinterpret_cast<char*>(cache->key_scales),
                     reinterpret_cast<char*>(cache->value_scales), cache->kv_heads, row_bytes, token_scale_of(*cache), group_scales_of(*cache), status};
  const cudaStream_t stream = static_cast<cudaStream_t>(stream_ptr);
  if (batch <= kResizeWarps && 2 * int64_t(batch) * cache->kv_heads * cache->page_size * row_bytes <= kLittle)
    return launched(launch_chained(resize_kernel, dim3(kResizeCtas), dim3(kPlanThreads), 0, stream, a), "resize");
  if (const int bad = launched(launch_chained(resize_plan_kernel, dim3(1), dim3(kPlanThreads), 0, stream, a), "resize")) return bad;
  // parts: 16 bytes of keys and values for each thread in turn, as many as fill the SMs and as a page has work for
  const int64_t work = (int64_t(cache->kv_heads) * cache->page_size * row_bytes / 16 + 255) / 256;
  const int parts = int(std::max<int64_t>(1, std::min<int64_t>(work, (148 * 8 + batch - 1) / batch)));
  return launched(launch_chained(resize_apply_kernel, dim3(batch, parts), dim3(256), 0, stream, a), "resize");
}

extern "C" size_t risa_b200_compact_scratch_size(const risa_b200_cache* cache, const risa_b200_cache* target) {
  if (cache == nullptr || target == nullptr) return 0;
  return sizeof(int32_t) * (size_t(std::max(cache->pages, 0)) + size_t(std::max(target->pages, 0)));
}

extern "C" int risa_b200_cache_compact(const risa_b200_cache* cache, const int32_t* references, const risa_b200_step* step, const risa_b200_cache* target,
                                       int32_t* table, int32_t* target_references, int32_t* used, void* scratch, size_t scratch_bytes, void* stream_ptr) {
  if (const int bad = check_cache(cache, "compact")) return bad;
  if (const int bad = check_cache(target, "compact")) return bad;
  RISA_REQUIRE(step != nullptr, "compact: null step");
  if (const int bad = check_table(step->page_table, step->lengths, step->batch, step->table_width, cache, "compact")) return bad;
  RISA_REQUIRE(references && table && target_references && used, "compact: null tensor");
  RISA_REQUIRE(cache->kv_heads == target->kv_heads && cache->page_size == target->page_size && cache->head_dim == target->head_dim &&
                   cache->dtype_code == target->dtype_code, "compact: both caches must have pages of the same kind");
  RISA_REQUIRE(cache->keys != target->keys && cache->values != target->values, "compact: the target must be another pool");
  RISA_REQUIRE(scratch != nullptr && reinterpret_cast<uintptr_t>(scratch) % 4 == 0 && scratch_bytes >= risa_b200_compact_scratch_size(cache, target),
               "compact: the scratch is too small");
  const int64_t rows = int64_t(cache->kv_heads) * cache->page_size;
  const int64_t row_units = rows * cache->head_dim * bits_of(*cache) / 8 / 16, scale_units = rows * (token_scale_of(*cache) + group_scales_of(*cache)) / 4;
  const int per_plan = kPlanThreads * kPlanEach, per_copy = 256 * kCopyAhead;
  const int64_t pages_each = std::max<int64_t>(1, per_copy / std::max(row_units, scale_units)), groups = (target->pages + pages_each - 1) / pages_each;
  const int64_t row_parts = (row_units * pages_each + per_copy - 1) / per_copy, scale_parts = (scale_units * pages_each + per_copy - 1) / per_copy;
  const int64_t table_blocks = std::min<int64_t>((int64_t(step->batch) * step->table_width + 2047) / 2048, 1024);
  RISA_REQUIRE(std::max(row_units, scale_units) < (int64_t(1) << 31) && groups * (row_parts + scale_parts) + table_blocks < (int64_t(1) << 31),
               "compact: the target has too many pages, or too large ones");
  unsigned int* status = status_word();
  if (status == nullptr) return RISA_B200_CUDA;
  const CompactArgs a{{step->page_table, step->lengths, nullptr, step->batch, step->table_width, 0, shift_of(cache->page_size)},
                references, static_cast<int32_t*>(scratch), static_cast<int32_t*>(scratch) + cache->pages, table, target_references, used, cache->pages, target->pages,
                {static_cast<const char*>(cache->keys), static_cast<const char*>(cache->values), reinterpret_cast<const char*>(cache->key_scales),
                 reinterpret_cast<const char*>(cache->value_scales)},
                {static_cast<char*>(target->keys), static_cast<char*>(target->values), reinterpret_cast<char*>(target->key_scales),
                 reinterpret_cast<char*>(target->value_scales)},
                {int(row_units), int(scale_units)}, int(pages_each), {unsigned(row_parts), unsigned(std::max<int64_t>(scale_parts, 1))},
                {unsigned(groups * row_parts), unsigned(groups * scale_parts)}, status};
  const cudaStream_t stream = static_cast<cudaStream_t>(stream_ptr);
  if (const int bad = launched(launch_chained(compact_plan_kernel, dim3((cache->pages + per_plan - 1) / per_plan), dim3(kPlanThreads), 0, stream, a), "compact"))
    return bad;
  return launched(launch_chained(compact_copy_kernel, dim3(unsigned(a.copies[0] + a.copies[1] + table_blocks)), dim3(256), 0, stream, a), "compact");
}
