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
// lane.  509 pages of 16 KB in 64 arrays take 202 us (5.28 TB/s, a large copy's
// rate); with stores kept in the L2 215.
#include "common.h"

namespace {

constexpr int kMaxTensors = 128;  // tensors of one launch: their addresses travel as kernel arguments
constexpr int kClasses = 5;       // lanes that move a page: 16, 32, .. 256

struct PageTensors {
  uint8_t* base[kMaxTensors];
  int64_t bytes[kMaxTensors];  // of a page
  int first[kClasses + 1];     // class c has the tensors from first[c] to first[c + 1]
};

// Pages src[i] -> dst[i], i < m, in every array: m = *count (n where count is
// NULL), src = dst + m where src is NULL.  Entries outside [0, num_pages) and
// pages onto themselves are skipped.  A page is moved by lanes of 16 bytes, at
// most 256 of them, and a workgroup takes several small pages of an array (509
// pages of 256 bytes in 64 arrays: 5.7 us, 19 with a workgroup a page); the
// large pages come first.  Where the device knows their number, workgroups go
// round until all are done: those of empty entries would cost a trip to memory
// each (11 pages of 64 arrays in a list of 32: 16 us).
__global__ __launch_bounds__(256) void copy_pages_kernel(PageTensors t, const int32_t* __restrict__ src,
                                                         const int32_t* __restrict__ dst,
                                                         const int32_t* __restrict__ count, int n,
                                                         int64_t num_pages) {
  const int m = count ? min(*count, n) : n;
  if (!src) src = dst + m;
  for (int64_t w = blockIdx.x;; w += gridDim.x) {
    int c = kClasses - 1, tensors = 0, lgl = 0;
    int64_t rest = w;
    for (; c >= 0; --c) {
      lgl = 4 + c;
      tensors = t.first[c + 1] - t.first[c];
      const int64_t work = (int64_t)((m + (256 >> lgl) - 1) >> (8 - lgl)) * tensors;
      if (rest < work) break;
      rest -= work;
    }
    if (c < 0) return;
    const int lane = threadIdx.x & ((1 << lgl) - 1), lanes = 1 << lgl;
    const int batch = (int)(rest / tensors), k = t.first[c] + (int)(rest - (int64_t)batch * tensors);
    const int i = (batch << (8 - lgl)) + ((int)threadIdx.x >> lgl);
    if (i >= m) continue;
    const int64_t a = src[i], b = dst[i];
    if (a < 0 || a >= num_pages || b < 0 || b >= num_pages || a == b) continue;
    uint8_t* base = t.base[k];
    const int64_t bytes = t.bytes[k];
    const uint8_t* from = base + a * bytes;
    uint8_t* to = base + b * bytes;
    if (((reinterpret_cast<uintptr_t>(base) | (uintptr_t)bytes) & 15) == 0) {
      constexpr int UN = 4;  // loads in flight before the first store
      for (int64_t o = 16 * (int64_t)lane; o < bytes; o += 16 * (int64_t)lanes * UN) {
        u32x4 v[UN];
#pragma unroll
        for (int u = 0; u < UN; ++u)
          if (o + 16 * lanes * u < bytes) v[u] = ldg128_stream(from + o + 16 * lanes * u);
#pragma unroll
        for (int u = 0; u < UN; ++u)
          if (o + 16 * lanes * u < bytes)
            __builtin_nontemporal_store(v[u], reinterpret_cast<u32x4*>(to + o + 16 * lanes * u));
      }
    } else {
      for (int64_t o = lane; o < bytes; o += lanes) to[o] = from[o];
    }
  }
}

// class of a page of so many bytes
inline int page_class(int64_t bytes) {
  int c = 0;
  while (c < kClasses - 1 && (256 << c) < bytes) ++c;
  return c;
}

// The moves of all arrays, kMaxTensors of them in a launch, whatever their pages'
// sizes (4 to 44 pages of 46 arrays of codes and 46 of scales: 35.8 us a call,
// 39.5 with a launch for each size); n: the most pairs that there can be.
int copy_pages(void* const* tensors, const int64_t* page_bytes, int64_t num_tensors, const int32_t* src,
               const int32_t* dst, const int32_t* count, int64_t n, int64_t num_pages, hipStream_t st) {
  for (int64_t at = 0; at < num_tensors; at += kMaxTensors) {
    const int64_t end = at + kMaxTensors < num_tensors ? at + kMaxTensors : num_tensors;
    PageTensors t = {};
    int k = 0;
    int64_t work = 0;
    for (int c = 0; c < kClasses; ++c) {
      t.first[c] = k;
      for (int64_t i = at; i < end; ++i) {
        if (page_bytes[i] == 0 || page_class(page_bytes[i]) != c) continue;
        t.base[k] = reinterpret_cast<uint8_t*>(tensors[i]);
        t.bytes[k++] = page_bytes[i];
      }
      work += ((n + (16 >> c) - 1) / (16 >> c)) * (k - t.first[c]);
    }
    t.first[kClasses] = k;
    if (k == 0) continue;
    // a workgroup for each piece of a known number of pages (64 x 509 pages of
    // 16 KB: 202 us, 225 with 2048 workgroups going round), else as many as
    // the CUs hold at a time
    const int64_t most = count ? 2048 : 1 << 20;
    copy_pages_kernel<<<(unsigned)(work < most ? work : most), 256, 0, st>>>(t, src, dst, count, (int)n, num_pages);
    MK_CHECK_LAUNCH();
  }
  return MK_OK;
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
__device__ __forceinline__ void add_count(int32_t* p, int v) {
  __hip_atomic_fetch_add(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// ---------------------------------------------------------------------------
// fork
// ---------------------------------------------------------------------------

constexpr int kForkRows = 4096;  // rows of the new table
// What one workgroup does with the counts in LDS: a step of 32 beams over 700
// pages in 9.2 us (16.6 with counts in memory, whose atomics and reads go to the
// L2 one after another).  Beyond, launches over all CUs count the references.
constexpr int kSmallPages = 8192, kSmallRows = 1024, kSmallNew = 2048, kSmallEntries = 1 << 16;

struct ForkArgs {
  const int32_t* table;    // [B, blocks]
  const int32_t* lengths;  // [B]
  const int32_t* refs;     // [pages]
  const int32_t* parents;  // [n]
  int32_t* new_table;      // [n, blocks]
  int32_t* new_lengths;    // [n]
  int32_t* new_refs;       // [pages]
  uint8_t* ready;          // [n]
  int32_t* moves;          // [2, n] + 1: sources and destinations of the copied pages, and their number
  int32_t* ids;            // [max_new]: the pages handed out
  int64_t B, blocks, pages, page_size, reserve, max_new;
  int n;
};

// counts and pages handed out: in LDS, or in memory
template <bool SMALL>
struct ForkCounts {
  int32_t* count;
  int32_t* ids;
  __device__ __forceinline__ int load(int64_t p) const {
    if constexpr (SMALL) return count[p];
    else return load_count(count + p);
  }
  __device__ __forceinline__ void add(int64_t p, int v) const {
    if constexpr (SMALL) atomicAdd(count + p, v);
    else add_count(count + p, v);
  }
};

// the old rows' references off, entries i0, i0 + step, ..., eight of them on their way together
template <bool SMALL>
__device__ __forceinline__ void fork_drop(const ForkArgs& a, const ForkCounts<SMALL>& c, int64_t i0, int64_t step) {
  const int64_t all = a.B * a.blocks;
  for (int64_t i = i0; i < all; i += 8 * step) {
    int p[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) p[u] = i + u * step < all ? a.table[i + u * step] : -1;
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (p[u] >= 0 && p[u] < a.pages) c.add(p[u], -1);
  }
}

// positions of new row r, and its parent (-1: an empty row)
__device__ __forceinline__ int fork_length(const ForkArgs& a, int r, int* parent) {
  const int p = a.parents[r];
  *parent = p < 0 || p >= a.B ? -1 : p;
  if (*parent < 0) return 0;
  const int l = a.lengths[p], most = (int)(a.blocks * a.page_size);  // < 2^31
  return l < 0 ? 0 : (l > most ? most : l);
}

// New row r: its length, the kept entries and their references; threads j0,
// j0 + step, ...  Gives the partly filled last page to the thread that has it.
template <bool SMALL>
__device__ __forceinline__ void fork_row(const ForkArgs& a, const ForkCounts<SMALL>& c, int r, int j0, int step,
                                         int parent, int len, int* last) {
  const int P = (int)a.page_size, blocks = (int)a.blocks;
  const int used = (len + P - 1) / P, part = len % P;
  const int32_t* old = a.table + (int64_t)(parent < 0 ? 0 : parent) * blocks;
  int32_t* now = a.new_table + (int64_t)r * blocks;
  for (int64_t jb = j0; jb < blocks; jb += 4 * step) {
    int p[4];  // on their way together
#pragma unroll
    for (int u = 0; u < 4; ++u) p[u] = jb + u * step < used ? old[jb + u * step] : -1;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int64_t j = jb + u * step;
      if (j >= blocks) break;
      if (p[u] >= a.pages) p[u] = -1;
      if (p[u] < 0) p[u] = -1;
      else c.add(p[u], 1);
      if (part && j == used - 1 && last) *last = p[u];
      now[j] = p[u];
    }
  }
  if (j0 == 0) {
    a.new_lengths[r] = len;
    if (!part && last) *last = -1;
  }
}

// New pages for the rows, by one workgroup of 1024 threads.  A partly filled
// last page stays with the longest of its rows (the first of those) if nobody
// else holds it; every other row gets a copy.  Row k of thread t is
// t * per + k, so that a thread's rows and the threads are in order.
// parts: positions on each row's last page, -1 for a row without a parent.
// paired: the rows that get a copy are marked in a.ready already.
template <bool SMALL, int PER>
__device__ void fork_allot(const ForkArgs& a, const ForkCounts<SMALL>& c, const int* last, const int* lens,
                           const int* parts, int* scan, bool paired) {
  const int tid = threadIdx.x;
  const int per = (a.n + 1023) / 1024;
  const int P = (int)a.page_size, blocks = (int)a.blocks;
  int need[PER];
  bool copies[PER], fits[PER];
  int mine = 0;
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int r = tid * per + k;
    need[k] = 0;
    copies[k] = false;
    fits[k] = true;
    if (k >= per || r >= a.n) continue;
    const int len = lens[r], page = last[r], part = parts[r];
    if (part < 0) continue;
    const int64_t end = len + a.reserve;
    fits[k] = end <= (int64_t)blocks * P;
    if (!fits[k]) continue;
    need[k] = (int)((end + P - 1) / P) - (len + P - 1) / P;
    if (paired) {
      copies[k] = a.ready[r];
    } else if (page >= 0) {
      int same = 0;
      bool best = true;
#pragma unroll 8
      for (int o = 0; o < a.n; ++o) {
        const bool s = last[o] == page;
        const int other = parts[o];
        same += s;
        best &= !s || other < part || (other == part && o >= r);
      }
      copies[k] = !(best && c.load(page) == same);
    }
    need[k] += copies[k];
    mine += need[k];
  }
  int wanted;
  int off = block_scan(mine, &wanted, scan);
  // ids of the first free pages; stops where there are enough (the counts of the next 8192 on their way)
  int found = 0;
  int next[8];
  auto read = [&](int64_t base) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int64_t i = base + 8 * tid + e;
      next[e] = i < a.pages ? c.load(i) : 1;
    }
  };
  if (wanted > 0) read(0);
  for (int64_t base = 0; base < a.pages && found < wanted; base += 8 * 1024) {
    int ok = 0, cnt = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const bool f = next[e] == 0;
      ok |= (int)f << e;
      cnt += f;
    }
    if (base + 8 * 1024 < a.pages) read(base + 8 * 1024);
    int total;
    int at = found + block_scan(cnt, &total, scan);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if ((ok >> e) & 1) {
        if (at < wanted && at < a.max_new) c.ids[at] = (int32_t)(base + 8 * tid + e);
        ++at;
      }
    found += total;
  }
  __syncthreads();  // ids are written, counts are read
  int moved = 0, moves;
  {
    int o = off;
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      copies[k] = copies[k] && o + need[k] <= found;
      moved += copies[k];
      o += need[k];
    }
  }
  moved = block_scan(moved, &moves, scan);
  if (tid == 0) a.moves[2 * a.n] = moves;
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int r = tid * per + k;
    if (k >= per || r >= a.n) continue;
    const bool got = fits[k] && (need[k] == 0 || off + need[k] <= found);
    a.ready[r] = got;
    if (got && need[k] > 0) {
      int i = off;
      const int end = off + need[k];
      int j = (lens[r] + P - 1) / P;
      if (copies[k]) {
        a.moves[moved] = last[r];
        a.moves[a.n + moved++] = c.ids[i];
        c.add(last[r], -1);
        --j;
      }
      for (; i < end; ++i, ++j) {
        a.new_table[(int64_t)r * blocks + j] = c.ids[i];
        c.add(c.ids[i], 1);
      }
    }
    off += need[k];
  }
}

__global__ __launch_bounds__(1024) void fork_small_kernel(ForkArgs a) {
  __shared__ int32_t count[kSmallPages], ids[kSmallNew];
  __shared__ int last[kSmallRows], lens[kSmallRows], parts[kSmallRows], parents[kSmallRows], scan[16];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const ForkCounts<true> c = {count, ids};
  for (int i = tid; i < (int)a.pages; i += 1024) count[i] = a.refs[i];
  for (int r = tid; r < a.n; r += 1024) {
    lens[r] = fork_length(a, r, &parents[r]);
    parts[r] = parents[r] < 0 ? -1 : lens[r] % (int)a.page_size;
  }
  __syncthreads();
  fork_drop(a, c, tid, 1024);
  for (int r = wave; r < a.n; r += 16) fork_row(a, c, r, lane, MK_WAVE, parents[r], lens[r], &last[r]);
  __syncthreads();
  if (a.reserve > 0) {
    fork_allot<true, 1>(a, c, last, lens, parts, scan, false);
  } else {
    for (int r = tid; r < a.n; r += 1024) a.ready[r] = 1;
  }
  __syncthreads();
  for (int i = tid; i < (int)a.pages; i += 1024) a.new_refs[i] = count[i];
}

__global__ __launch_bounds__(256) void fork_init_kernel(ForkArgs a) {
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < a.pages; i += gridDim.x * 256ll) a.new_refs[i] = a.refs[i];
}

// workgroup r < n: new row r, its last page and the positions on it to the
// workspace (which the moves take later); the others: the old table
__global__ __launch_bounds__(256) void fork_rows_kernel(ForkArgs a) {
  const ForkCounts<false> c = {a.new_refs, nullptr};
  const int r = blockIdx.x;
  if (r < a.n) {
    int parent;
    const int len = fork_length(a, r, &parent);
    fork_row(a, c, r, threadIdx.x, 256, parent, len, a.reserve > 0 ? a.moves + r : nullptr);
    if (threadIdx.x == 0) {
      if (a.reserve > 0) a.moves[a.n + r] = parent < 0 ? -1 : len % (int)a.page_size;
      else a.ready[r] = 1;
    }
  } else {
    fork_drop(a, c, (r - a.n) * 256ll + threadIdx.x, (gridDim.x - a.n) * 256ll);
  }
}

// Workgroup r: whether row r gets a copy of its last page, to a.ready.  Up to
// kPairRows rows the next kernel looks for itself (4096 rows: the fork in 50 us,
// 1010 without this launch).
constexpr int kPairRows = 256;
__global__ __launch_bounds__(256) void fork_pairs_kernel(ForkArgs a) {
  const int r = blockIdx.x, page = a.moves[r], part = a.moves[a.n + r];
  int same = 0, better = 0;
  if (page >= 0) {
    for (int o = threadIdx.x; o < a.n; o += 256) {
      const bool s = a.moves[o] == page;
      const int other = a.moves[a.n + o];
      same += s;
      better |= s && (other > part || (other == part && o < r));
    }
  }
  __shared__ int all;
  if (threadIdx.x == 0) all = 0;
  better = __syncthreads_or(better);
  if (same) atomicAdd(&all, same);
  __syncthreads();
  if (threadIdx.x == 0) a.ready[r] = page >= 0 && (better || load_count(a.new_refs + page) != all);
}

__global__ __launch_bounds__(1024) void fork_allot_kernel(ForkArgs a, bool paired) {
  __shared__ int last[kForkRows], lens[kForkRows], parts[kForkRows], scan[16];
  const ForkCounts<false> c = {a.new_refs, a.ids};
  for (int r = threadIdx.x; r < a.n; r += 1024) {
    lens[r] = a.new_lengths[r];
    last[r] = a.moves[r];
    parts[r] = a.moves[a.n + r];
  }
  __syncthreads();
  fork_allot<false, kForkRows / 1024>(a, c, last, lens, parts, scan, paired);
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
  int32_t* live;      // [pages / 8192, rounded up]
  int64_t entries, pages;
};

// With n live pages, the i-th live page at or past n moves to the i-th free
// one below n: as many of the one as of the other, and no page is both.
// list: those free pages, then from m on the live ones, m = how many they are.

// page i of count c, with `live` live ones before it and `below` live ones below n
__device__ __forceinline__ void place_page(const CompactArgs& a, int64_t i, int c, int n, int live, int below) {
  if (i < n && c <= 0) a.list[i - live] = (int32_t)i;
  if (i >= n && c > 0) a.list[n - below + live - below] = (int32_t)i;
  a.page_map[i] = c > 0 && i < n ? (int32_t)i : -1;
  a.new_refs[i] = i < n ? c : 0;
}

// how many of the 8 pages from i on are live and below n
__device__ __forceinline__ int live_below(const int (&c)[8], int64_t i, int n) {
  int k = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) k += c[e] > 0 && i + e < n;
  return k;
}
__device__ __forceinline__ void read_counts(const CompactArgs& a, int64_t i, int (&c)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) c[e] = i + e < a.pages ? a.refs[i + e] : 0;
}

// entries of pairs i0, i0 + step, ... of m: where a page went, its count there
__device__ __forceinline__ void move_pages(const CompactArgs& a, int m, int i0, int step) {
  for (int i = i0; i < m; i += step) {
    const int to = a.list[i], from = a.list[m + i];
    a.page_map[from] = to;
    a.new_refs[to] = a.refs[from];
  }
}

// Table entries renamed, i0, i0 + step, ..., eight of them on their way together
__device__ __forceinline__ void rename_entries(const CompactArgs& a, int64_t i0, int64_t step) {
  for (int64_t i = i0; i < a.entries; i += 8 * step) {
    int p[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) p[u] = i + u * step < a.entries ? a.table[i + u * step] : -1;
#pragma unroll
    for (int u = 0; u < 8; ++u) p[u] = p[u] >= 0 && p[u] < a.pages ? a.page_map[p[u]] : -1;
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (i + u * step < a.entries) a.new_table[i + u * step] = p[u];
  }
}

// up to 8192 pages: all by one workgroup
__global__ __launch_bounds__(1024) void compact_small_kernel(CompactArgs a) {
  __shared__ int scan[16];
  const int tid = threadIdx.x;
  const int64_t i = 8 * tid;
  int c[8], n, below;
  read_counts(a, i, c);
  int live = block_scan(live_below(c, i, INT32_MAX), &n, scan);
  block_scan(live_below(c, i, n), &below, scan);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    if (i + e < a.pages) place_page(a, i + e, c[e], n, live, below);
    live += c[e] > 0;
  }
  if (tid == 0) {
    a.counts[0] = n;
    a.counts[1] = n - below;
  }
  __syncthreads();
  move_pages(a, n - below, tid, 1024);
  __syncthreads();
  rename_entries(a, tid, 1024);
}

// Larger pools: 8192 pages a workgroup, four launches.
__global__ __launch_bounds__(1024) void compact_count_kernel(CompactArgs a) {
  __shared__ int scan[16];
  const int64_t i = blockIdx.x * 8192ll + 8 * threadIdx.x;
  int c[8], n;
  read_counts(a, i, c);
  block_scan(live_below(c, i, INT32_MAX), &n, scan);
  if (threadIdx.x == 0) a.live[blockIdx.x] = n;
}

__global__ __launch_bounds__(1024) void compact_place_kernel(CompactArgs a) {
  __shared__ int scan[16];
  const int tid = threadIdx.x;
  const int64_t i = blockIdx.x * 8192ll + 8 * tid;
  int c[8], v, n, before, below, part;
  read_counts(a, i, c);
  v = 0;
  for (int k = tid; k < (int)gridDim.x; k += 1024) v += a.live[k];
  block_scan(v, &n, scan);
  v = 0;
  for (int k = tid; k < (int)blockIdx.x; k += 1024) v += a.live[k];
  block_scan(v, &before, scan);
  const int cut = n / 8192;  // the workgroup that page n is in (there may be none)
  v = 0;
  for (int k = tid; k < cut; k += 1024) v += a.live[k];
  int at[8];
  read_counts(a, cut * 8192ll + 8 * tid, at);
  v += live_below(at, cut * 8192ll + 8 * tid, n);
  block_scan(v, &below, scan);
  int live = before + block_scan(live_below(c, i, INT32_MAX), &part, scan);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    if (i + e < a.pages) place_page(a, i + e, c[e], n, live, below);
    live += c[e] > 0;
  }
  if (blockIdx.x == 0 && tid == 0) {
    a.counts[0] = n;
    a.counts[1] = n - below;
  }
}

__global__ __launch_bounds__(256) void compact_move_kernel(CompactArgs a) {
  move_pages(a, a.counts[1], (int)(blockIdx.x * 256 + threadIdx.x), (int)(gridDim.x * 256));
}

__global__ __launch_bounds__(256) void compact_rename_kernel(CompactArgs a) {
  rename_entries(a, blockIdx.x * 256ll + threadIdx.x, gridDim.x * 256ll);
}

}  // namespace

extern "C" {

int mk_copy_kv_pages(void* const* tensors, const int64_t* page_bytes, int64_t num_tensors, const int32_t* src,
                     const int32_t* dst, int64_t n, int64_t num_pages, void* stream) {
  MK_REQUIRE(num_tensors >= 0 && n >= 0 && n < (1LL << 30) && num_pages >= 0 && num_pages < (1LL << 31));
  MK_REQUIRE(num_tensors == 0 || (tensors && page_bytes));
  MK_REQUIRE(n == 0 || (src && dst));
  for (int64_t i = 0; i < num_tensors; ++i) MK_REQUIRE(tensors[i] && page_bytes[i] >= 0);
  if (n == 0) return MK_OK;
  return copy_pages(tensors, page_bytes, num_tensors, src, dst, nullptr, n, num_pages,
                    reinterpret_cast<hipStream_t>(stream));
}

int mk_fork_kv_sequences(void* const* tensors, const int64_t* page_bytes, int64_t num_tensors,
                         const int32_t* block_table, const int32_t* lengths, const int32_t* ref_counts,
                         const int32_t* parents, int32_t* new_table, int32_t* new_lengths, int32_t* new_ref_counts,
                         uint8_t* ready, int32_t* workspace, int64_t workspace_ints, int64_t B, int64_t n,
                         int64_t max_blocks, int64_t page_size, int64_t num_pages, int64_t reserve, void* stream) {
  MK_REQUIRE(B >= 0 && n >= 0 && n <= kForkRows && max_blocks > 0 && page_size > 0 && num_pages > 0 && reserve >= 0);
  MK_REQUIRE(max_blocks < (1LL << 31) && page_size < (1LL << 31) && num_pages < (1LL << 31) && reserve < (1LL << 31));
  MK_REQUIRE((max_blocks + 1) * page_size < (1LL << 31) && n * (max_blocks + 1) < (1LL << 31) && B < (1LL << 31));
  MK_REQUIRE(B * max_blocks < (1LL << 40));
  MK_REQUIRE(ref_counts && new_ref_counts && (B == 0 || (block_table && lengths)));
  MK_REQUIRE(n == 0 || (parents && new_table && new_lengths && ready));
  if (n == 0) reserve = 0;  // no row takes pages: nothing below may touch the workspace, which may be NULL
  const int64_t most = n * (1 + (reserve + page_size - 1) / page_size);  // pages that the rows can need
  const int64_t max_new = reserve == 0 ? 0 : (most < num_pages ? most : num_pages);
  MK_REQUIRE(reserve == 0 || (workspace && workspace_ints >= 2 * n + 1 + max_new));
  MK_REQUIRE(num_tensors >= 0 && (num_tensors == 0 || (tensors && page_bytes)));
  for (int64_t i = 0; i < num_tensors; ++i) MK_REQUIRE(tensors[i] && page_bytes[i] >= 0);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const ForkArgs a = {block_table, lengths, ref_counts, parents, new_table, new_lengths, new_ref_counts, ready,
                      workspace, workspace ? workspace + 2 * n + 1 : nullptr, B, max_blocks, num_pages, page_size,
                      reserve, max_new, (int)n};
  if (num_pages <= kSmallPages && n <= kSmallRows && max_new <= kSmallNew && (B + n) * max_blocks <= kSmallEntries) {
    fork_small_kernel<<<1, 1024, 0, st>>>(a);
  } else {
    const int64_t init = (num_pages + 255) / 256;
    fork_init_kernel<<<(unsigned)(init < 1024 ? init : 1024), 256, 0, st>>>(a);
    const int64_t drop = (B * max_blocks + 255) / 256;
    if (n + drop > 0) fork_rows_kernel<<<(unsigned)(n + (drop < 1024 ? drop : 1024)), 256, 0, st>>>(a);
    if (reserve > 0) {
      if (n > kPairRows) fork_pairs_kernel<<<(unsigned)n, 256, 0, st>>>(a);
      fork_allot_kernel<<<1, 1024, 0, st>>>(a, n > kPairRows);
    }
  }
  MK_CHECK_LAUNCH();
  if (reserve == 0) return MK_OK;
  return copy_pages(tensors, page_bytes, num_tensors, workspace, workspace + n, workspace + 2 * n, n, num_pages, st);
}

int mk_compact_kv_pages(void* const* tensors, const int64_t* page_bytes, int64_t num_tensors,
                        const int32_t* block_table, const int32_t* ref_counts, int32_t* new_table,
                        int32_t* new_ref_counts, int32_t* page_map, int32_t* counts, int32_t* workspace,
                        int64_t workspace_ints, int64_t entries, int64_t num_pages, void* stream) {
  MK_REQUIRE(entries >= 0 && num_pages > 0 && num_pages < (1LL << 31) && ref_counts && new_ref_counts && page_map);
  const int64_t chunks = (num_pages + 8191) / 8192;
  MK_REQUIRE(counts && workspace && workspace_ints >= num_pages + chunks);
  MK_REQUIRE(entries == 0 || (block_table && new_table));
  MK_REQUIRE(num_tensors >= 0 && (num_tensors == 0 || (tensors && page_bytes)));
  for (int64_t i = 0; i < num_tensors; ++i) MK_REQUIRE(tensors[i] && page_bytes[i] >= 0);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const CompactArgs a = {block_table, ref_counts, new_table, new_ref_counts, page_map, counts, workspace,
                         workspace + num_pages, entries, num_pages};
  // One launch of one workgroup, or four over all CUs, us a call: 8000 pages and
  // 16384 entries 20 / 32; 40000 pages and 32768 entries 69 / 32; 300000 pages
  // 470 / 33.
  if (num_pages <= 8192 && entries <= 16384) {
    compact_small_kernel<<<1, 1024, 0, st>>>(a);
  } else {
    const int64_t moves = (num_pages / 2 + 255) / 256, names = (entries + 2047) / 2048;
    compact_count_kernel<<<(unsigned)chunks, 1024, 0, st>>>(a);
    compact_place_kernel<<<(unsigned)chunks, 1024, 0, st>>>(a);
    compact_move_kernel<<<(unsigned)(moves < 1024 ? moves : 1024), 256, 0, st>>>(a);
    if (names > 0) compact_rename_kernel<<<(unsigned)(names < 1024 ? names : 1024), 256, 0, st>>>(a);
  }
  MK_CHECK_LAUNCH();
  // no more pages move than are free, and than are live
  return num_pages > 1 ? copy_pages(tensors, page_bytes, num_tensors, nullptr, workspace, counts + 1, num_pages / 2,
                                    num_pages, st)
                       : MK_OK;
}

}  // extern "C"
