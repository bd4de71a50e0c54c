// Pages of a cache: copied, forked (and freed), compacted.  No counterpart in
// the reference, whose block tables are fixed (ops/paged_kv_ops.py:99-115).
//
// The bookkeeping -- block tables, lengths, reference counts -- stays on the
// device, so that a step whose parents come from a device (beams, samples)
// needs no host: a page is free when its count is 0, and pages are handed out
// by ascending id to rows in order, so every result is determined by the
// inputs.  Counts change by integer atomics, whose order does not matter.
//
// The moves are bound by memory: a page is read and written once, 16 bytes a
// lane, by a workgroup per (page, tensor).
#include "common.h"

namespace {

constexpr int kMaxTensors = 128;  // tensors of one launch: their addresses travel as kernel arguments

struct PageTensors {
  uint8_t* base[kMaxTensors];
  int64_t bytes[kMaxTensors];  // of a page
};

// one page, by a workgroup
__device__ __forceinline__ void copy_page(uint8_t* base, int64_t bytes, int64_t src, int64_t dst) {
  const uint8_t* from = base + src * bytes;
  uint8_t* to = base + dst * bytes;
  if (((reinterpret_cast<uintptr_t>(base) | (uintptr_t)bytes) & 15) == 0) {
    for (int64_t o = 16 * (int64_t)threadIdx.x; o < bytes; o += 16 * 256)
      *reinterpret_cast<u32x4*>(to + o) = ldg128_stream(from + o);
  } else {
    for (int64_t o = threadIdx.x; o < bytes; o += 256) to[o] = from[o];
  }
}

// pages src[i] -> dst[i] in every tensor; entries outside [0, num_pages) and
// pages onto themselves are skipped
__global__ __launch_bounds__(256) void copy_pages_kernel(PageTensors t, const int32_t* __restrict__ src,
                                                         const int32_t* __restrict__ dst, int n,
                                                         int64_t num_pages) {
  for (int i = blockIdx.x; i < n; i += gridDim.x) {
    const int64_t a = src[i], b = dst[i];
    if (a < 0 || a >= num_pages || b < 0 || b >= num_pages || a == b) continue;
    copy_page(t.base[blockIdx.y], t.bytes[blockIdx.y], a, b);
  }
}

// ---------------------------------------------------------------------------
// sums over a workgroup
// ---------------------------------------------------------------------------

// exclusive prefix sum of v over 1024 threads; *total: over all of them
__device__ __forceinline__ int block_scan(int v, int* total, int* lds) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int s = v;
#pragma unroll
  for (int o = 1; o < MK_WAVE; o <<= 1) {
    const int up = __shfl_up(s, o, MK_WAVE);
    if (lane >= o) s += up;
  }
  __syncthreads();  // the last call's sums are read
  if (lane == 63) lds[wave] = s;
  __syncthreads();
  int before = 0, all = 0;
  for (int w = 0; w < 16; ++w) {
    if (w < wave) before += lds[w];
    all += lds[w];
  }
  *total = all;
  return before + s - v;
}

// counts are changed by atomics, which go to the L2: reads that have to see them do too
__device__ __forceinline__ int load_count(const int32_t* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void store_count(int32_t* p, int v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void add_count(int32_t* p, int v) {
  __hip_atomic_fetch_add(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// ---------------------------------------------------------------------------
// fork
// ---------------------------------------------------------------------------

constexpr int kForkRows = 4096;   // rows of the new table
constexpr int kForkPerThread = kForkRows / 1024;

struct ForkArgs {
  const int32_t* table;    // [B, blocks]
  const int32_t* lengths;  // [B]
  const int32_t* refs;     // [pages]
  const int32_t* parents;  // [n]
  int32_t* new_table;      // [n, blocks]
  int32_t* new_lengths;    // [n]
  int32_t* new_refs;       // [pages]
  uint8_t* ready;          // [n]
  int32_t* moves;          // [2, n]: source and destination of each row's copied page, -1 for none
  int32_t* ids;            // [max_new]: the pages handed out
  int64_t B, blocks, pages, page_size, reserve, max_new;
  int n;
};

__device__ __forceinline__ int64_t fork_length(const ForkArgs& a, int r, int64_t* parent) {
  const int64_t p = a.parents[r];
  *parent = p;
  if (p < 0 || p >= a.B) return 0;
  const int64_t l = a.lengths[p], most = a.blocks * a.page_size;
  return l < 0 ? 0 : (l > most ? most : l);
}

// counts as they are, then the old rows' references off and the kept ones on
__device__ __forceinline__ void fork_init(const ForkArgs& a, int64_t i0, int64_t step) {
  for (int64_t i = i0; i < a.pages; i += step) store_count(a.new_refs + i, a.refs[i]);
}
__device__ __forceinline__ void fork_rows(const ForkArgs& a, int64_t i0, int64_t step) {
  for (int64_t i = i0; i < a.B * a.blocks; i += step) {
    const int64_t p = a.table[i];
    if (p >= 0 && p < a.pages) add_count(a.new_refs + p, -1);
  }
  for (int64_t i = i0; i < a.n * a.blocks; i += step) {
    const int r = (int)(i / a.blocks);
    const int64_t j = i - r * a.blocks;
    int64_t parent;
    const int64_t len = fork_length(a, r, &parent);
    int64_t p = -1;
    if (j * a.page_size < len) {
      p = a.table[parent * a.blocks + j];
      if (p < 0 || p >= a.pages) p = -1;
    }
    a.new_table[i] = (int32_t)p;
    if (p >= 0) add_count(a.new_refs + p, 1);
    if (j == 0) a.new_lengths[r] = (int32_t)len;
  }
}

// New pages for the rows, by one workgroup of 1024 threads.  A partly filled
// last page stays with the longest of its rows (the first of those) if nobody
// else holds it; every other row gets a copy.  Row r of thread t is
// t * per + k, so that a thread's rows and the threads are in order.
__device__ void fork_allot(const ForkArgs& a, int* scan) {
  __shared__ int last[kForkRows];           // partly filled last page, -1 for none
  __shared__ int key[kForkRows];            // values in it
  const int tid = threadIdx.x;
  const int per = (a.n + 1023) / 1024;
  const int64_t P = a.page_size;
  int64_t len[kForkPerThread];
  int need[kForkPerThread];
  bool copies[kForkPerThread], fits[kForkPerThread];
#pragma unroll
  for (int k = 0; k < kForkPerThread; ++k) {
    const int r = tid * per + k;
    len[k] = 0;
    need[k] = 0;
    copies[k] = false;
    fits[k] = true;
    if (k >= per || r >= a.n) continue;
    int64_t parent;
    len[k] = fork_length(a, r, &parent);
    const int part = (int)(len[k] % P);
    int64_t page = -1;
    if (part) {
      page = a.table[parent * a.blocks + len[k] / P];
      if (page < 0 || page >= a.pages) page = -1;
    }
    last[r] = (int)page;
    key[r] = part;
    a.moves[r] = a.moves[a.n + r] = -1;
    fits[k] = parent < 0 || parent >= a.B || len[k] + a.reserve <= a.blocks * P;
    need[k] = parent < 0 || parent >= a.B || !fits[k]
                  ? 0 : (int)((len[k] + a.reserve + P - 1) / P - (len[k] + P - 1) / P);
  }
  __syncthreads();
  int mine = 0;
#pragma unroll
  for (int k = 0; k < kForkPerThread; ++k) {
    const int r = tid * per + k;
    if (k >= per || r >= a.n) continue;
    const int page = last[r];
    int64_t parent = a.parents[r];
    if (page >= 0 && fits[k] && parent >= 0 && parent < a.B) {
      int same = 0;
      bool best = true;
      for (int o = 0; o < a.n; ++o) {
        const bool s = last[o] == page;
        same += s;
        best &= !s || key[o] < key[r] || (key[o] == key[r] && o >= r);
      }
      copies[k] = !(best && load_count(a.new_refs + page) == same);
      need[k] += copies[k];
    }
    mine += need[k];
  }
  int wanted;
  int off = block_scan(mine, &wanted, scan);
  __syncthreads();
  // ids of the first free pages; stops where there are enough
  int found = 0;
  for (int64_t base = 0; base < a.pages && found < wanted; base += 8 * 1024) {
    int ok = 0, cnt = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int64_t i = base + 8 * tid + e;
      const bool f = i < a.pages && load_count(a.new_refs + i) == 0;
      ok |= (int)f << e;
      cnt += f;
    }
    int total;
    int at = found + block_scan(cnt, &total, scan);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if ((ok >> e) & 1) {
        if (at < wanted && at < a.max_new) a.ids[at] = (int32_t)(base + 8 * tid + e);
        ++at;
      }
    found += total;
  }
  __syncthreads();  // ids are written, counts are read
#pragma unroll
  for (int k = 0; k < kForkPerThread; ++k) {
    const int r = tid * per + k;
    if (k >= per || r >= a.n) continue;
    const bool got = fits[k] && (need[k] == 0 || off + need[k] <= found);
    a.ready[r] = got;
    if (got && need[k] > 0) {
      int i = off;
      const int end = off + need[k];
      int64_t j = (len[k] + P - 1) / P;
      if (copies[k]) {
        a.moves[r] = last[r];
        a.moves[a.n + r] = a.ids[i];
        add_count(a.new_refs + last[r], -1);
        --j;
      }
      for (; i < end; ++i, ++j) {
        a.new_table[(int64_t)r * a.blocks + j] = a.ids[i];
        add_count(a.new_refs + a.ids[i], 1);
      }
    }
    off += need[k];
  }
}

__global__ __launch_bounds__(1024) void fork_kernel(ForkArgs a) {
  __shared__ int scan[16];
  fork_init(a, threadIdx.x, 1024);
  __syncthreads();
  fork_rows(a, threadIdx.x, 1024);
  __syncthreads();
  if (a.reserve > 0) {
    fork_allot(a, scan);
  } else {
    for (int r = threadIdx.x; r < a.n; r += 1024) a.ready[r] = 1;
  }
}

// ---------------------------------------------------------------------------
// compact
// ---------------------------------------------------------------------------

struct CompactArgs {
  const int32_t* table;  // [entries]
  const int32_t* refs;   // [pages]
  int32_t* new_table;
  int32_t* new_refs;
  int32_t* page_map;  // [pages]: where a page went, -1 for a free one
  int32_t* counts;    // [2]: live pages, moved ones
  int32_t* list;      // [2 * (pages / 2)]: free pages below the live count, then live ones from it on
  int64_t entries, pages;
};

// With n live pages, the i-th live page at or past n moves to the i-th free
// one below n: as many of the one as of the other, and no page is both.
__global__ __launch_bounds__(1024) void compact_kernel(CompactArgs a) {
  __shared__ int scan[16];
  const int tid = threadIdx.x;
  int mine = 0;
  for (int64_t i = tid; i < a.pages; i += 1024) mine += a.refs[i] > 0;
  int n;
  block_scan(mine, &n, scan);
  __syncthreads();
  int found = 0;
  for (int64_t base = 0; base < a.pages; base += 8 * 1024) {
    int ok = 0, cnt = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int64_t i = base + 8 * tid + e;
      if (i >= a.pages) continue;
      const int c = a.refs[i];
      const bool f = i < n ? c <= 0 : c > 0;
      ok |= (int)f << e;
      cnt += f;
      a.page_map[i] = c > 0 && i < n ? (int32_t)i : -1;
      a.new_refs[i] = i < n ? c : 0;
    }
    int total;
    int at = found + block_scan(cnt, &total, scan);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if ((ok >> e) & 1) a.list[at++] = (int32_t)(base + 8 * tid + e);
    found += total;
  }
  __syncthreads();
  const int m = found / 2;
  if (tid == 0) {
    a.counts[0] = n;
    a.counts[1] = m;
  }
  for (int i = tid; i < m; i += 1024) {
    const int to = a.list[i], from = a.list[m + i];
    a.page_map[from] = to;
    a.new_refs[to] = a.refs[from];
  }
  __syncthreads();
  for (int64_t i = tid; i < a.entries; i += 1024) {
    const int64_t p = a.table[i];
    a.new_table[i] = p >= 0 && p < a.pages ? a.page_map[p] : -1;
  }
}

__global__ __launch_bounds__(256) void copy_compacted_kernel(PageTensors t, const int32_t* __restrict__ list,
                                                             const int32_t* __restrict__ counts) {
  const int m = counts[1];
  for (int i = blockIdx.x; i < m; i += gridDim.x)
    copy_page(t.base[blockIdx.y], t.bytes[blockIdx.y], list[m + i], list[i]);
}

inline PageTensors page_tensors(void* const* tensors, const int64_t* bytes, int k) {
  PageTensors t;
  for (int i = 0; i < kMaxTensors; ++i) {
    t.base[i] = i < k ? reinterpret_cast<uint8_t*>(tensors[i]) : nullptr;
    t.bytes[i] = i < k ? bytes[i] : 0;
  }
  return t;
}

}  // namespace

extern "C" {

int mk_copy_kv_pages(void* const* tensors, const int64_t* page_bytes, int64_t num_tensors, const int32_t* src,
                     const int32_t* dst, int64_t n, int64_t num_pages, void* stream) {
  MK_REQUIRE(num_tensors >= 0 && n >= 0 && n < (1LL << 31) && num_pages >= 0 && num_pages < (1LL << 31));
  MK_REQUIRE(num_tensors == 0 || (tensors && page_bytes));
  MK_REQUIRE(n == 0 || (src && dst));
  for (int64_t i = 0; i < num_tensors; ++i) MK_REQUIRE(tensors[i] && page_bytes[i] >= 0);
  if (n == 0) return MK_OK;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  for (int64_t at = 0; at < num_tensors; at += kMaxTensors) {
    const int k = (int)(num_tensors - at < kMaxTensors ? num_tensors - at : kMaxTensors);
    const PageTensors t = page_tensors(tensors + at, page_bytes + at, k);
    copy_pages_kernel<<<dim3((unsigned)(n < 65536 ? n : 65536), (unsigned)k), 256, 0, st>>>(t, src, dst, (int)n,
                                                                                          num_pages);
    MK_CHECK_LAUNCH();
  }
  return MK_OK;
}

int mk_fork_kv_sequences(void* const* tensors, const int64_t* page_bytes, int64_t num_tensors,
                         const int32_t* block_table, const int32_t* lengths, const int32_t* ref_counts,
                         const int32_t* parents, int32_t* new_table, int32_t* new_lengths, int32_t* new_ref_counts,
                         uint8_t* ready, int32_t* workspace, int64_t workspace_ints, int64_t B, int64_t n,
                         int64_t max_blocks, int64_t page_size, int64_t num_pages, int64_t reserve, void* stream) {
  MK_REQUIRE(B >= 0 && n >= 0 && n <= kForkRows && max_blocks > 0 && page_size > 0 && num_pages > 0 && reserve >= 0);
  MK_REQUIRE(max_blocks < (1LL << 31) && page_size < (1LL << 31) && num_pages < (1LL << 31) && reserve < (1LL << 31));
  MK_REQUIRE(max_blocks * page_size < (1LL << 31) && n * (max_blocks + 1) < (1LL << 31) && B < (1LL << 31));
  MK_REQUIRE(ref_counts && new_ref_counts && (B == 0 || (block_table && lengths)));
  MK_REQUIRE(n == 0 || (parents && new_table && new_lengths && ready));
  const int64_t most = n * (1 + (reserve + page_size - 1) / page_size);  // pages that the rows can need
  const int64_t max_new = reserve == 0 ? 0 : (most < num_pages ? most : num_pages);
  MK_REQUIRE(reserve == 0 || n == 0 || (workspace && workspace_ints >= 2 * n + max_new));
  MK_REQUIRE(num_tensors >= 0 && (num_tensors == 0 || (tensors && page_bytes)));
  for (int64_t i = 0; i < num_tensors; ++i) MK_REQUIRE(tensors[i] && page_bytes[i] >= 0);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const ForkArgs a = {block_table, lengths, ref_counts, parents, new_table, new_lengths, new_ref_counts, ready,
                      workspace, workspace ? workspace + 2 * n : nullptr, B, max_blocks, num_pages, page_size, reserve,
                      max_new, (int)n};
  fork_kernel<<<1, 1024, 0, st>>>(a);
  MK_CHECK_LAUNCH();
  if (reserve == 0 || n == 0) return MK_OK;
  return mk_copy_kv_pages(tensors, page_bytes, num_tensors, workspace, workspace + n, n, num_pages, stream);
}

int mk_compact_kv_pages(void* const* tensors, const int64_t* page_bytes, int64_t num_tensors,
                        const int32_t* block_table, const int32_t* ref_counts, int32_t* new_table,
                        int32_t* new_ref_counts, int32_t* page_map, int32_t* counts, int32_t* workspace,
                        int64_t workspace_ints, int64_t entries, int64_t num_pages, void* stream) {
  MK_REQUIRE(entries >= 0 && num_pages > 0 && num_pages < (1LL << 31) && ref_counts && new_ref_counts && page_map);
  MK_REQUIRE(counts && workspace && workspace_ints >= num_pages && (entries == 0 || (block_table && new_table)));
  MK_REQUIRE(num_tensors >= 0 && (num_tensors == 0 || (tensors && page_bytes)));
  for (int64_t i = 0; i < num_tensors; ++i) MK_REQUIRE(tensors[i] && page_bytes[i] >= 0);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const CompactArgs a = {block_table, ref_counts, new_table, new_ref_counts, page_map, counts, workspace, entries,
                         num_pages};
  compact_kernel<<<1, 1024, 0, st>>>(a);
  MK_CHECK_LAUNCH();
  for (int64_t at = 0; at < num_tensors && num_pages > 1; at += kMaxTensors) {
    const int k = (int)(num_tensors - at < kMaxTensors ? num_tensors - at : kMaxTensors);
    const PageTensors t = page_tensors(tensors + at, page_bytes + at, k);
    const int64_t most = num_pages / 2;  // moved pages: no more than free ones, and no more than live ones
    copy_compacted_kernel<<<dim3((unsigned)(most < 1024 ? most : 1024), (unsigned)k), 256, 0, st>>>(t, workspace,
                                                                                                  counts);
    MK_CHECK_LAUNCH();
  }
  return MK_OK;
}

}  // extern "C"
