// kv_pages.hip -- the pages of the paged KV cache: taken, given back, shared by forked
// sequences, moved together.  prichs_hip.h has what each call does; kv_cache.hpp the
// page's layout, which nothing here looks into.
//
// Free pages are taken lowest first, so every result is that of the items done one after
// the other, in whatever order workgroups run.  Counts and tables are some bytes a page:
// launches and round trips to memory are the cost, until data is copied, which runs at the
// rate of the memory.  Up to kSmallPages pages and kSmallRows rows one workgroup of 1024
// threads finds the free pages (16 of them a thread in one round trip) and ranks them in one
// launch; beyond, workgroups count them in blocks of kBlockPages and a second launch ranks
// them behind the blocks before.  MI355X: the kernels that plan and write tables take 3 to
// 9 us each; fork_apply 4.4 us for 7 items and 6.0 for 224; compact_apply 39 us where 3661
// pages of three heads move (191 MB read and written, 4.9 TB/s); kv_cache_copy of 600 pages of
// three heads 5.8 us in a graph (7.0 a call from Python), of 16384 174 (856 MB, 4.9 TB/s).
#include "kv_cache.hpp"

#include <climits>

namespace prichs {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256;
constexpr int kSteps = 16;                          // pages of a lane
constexpr int kBlockPages = kThreads * kSteps;      // pages of a workgroup
constexpr int kCopyUnroll = 4;
// A page in equal chunks of at most so many 16-byte pieces, one for a copying workgroup.
constexpr int kChunk = kThreads * kCopyUnroll;
struct Chunks {
  int pieces, chunks, chunk;  // of a page; of a chunk
  explicit Chunks(size_t n_kv_heads)
      : pieces((int)(n_kv_heads * kKvPart / 16)),
        chunks((int)cdiv(pieces, kChunk)),
        chunk((int)cdiv(pieces, chunks)) {}
};
constexpr size_t kMaxPages = (size_t)1 << 24, kMaxRows = (size_t)1 << 20;
constexpr int kPlanThreads = 1024, kPlanWaves = kPlanThreads / 64;
// What one workgroup plans for: the pages that it has in registers.  A call in a captured
// graph, us, one workgroup and many, none of the pages free (the longest scan), 32 rows:
//                     reserve      fork, 16 items   compact, nothing moves
//      1024 pages    6.4, 11.3      8.5,  9.4           6.9, 8.3
//     16384          6.5, 11.3      8.4,  9.4           7.9, 9.0
//     65536         15.0, 11.0     17.0,  9.8          26.0, 9.3 (one workgroup: four rounds)
//     16384 pages, 1024 rows: 7.8, 12.1 and 13.8, 17.6; 4096: 15.9, 18.6 and 33.8, 45.1.
constexpr size_t kSmallPages = kPlanThreads * kSteps, kSmallRows = 4 * kPlanThreads;

// The workspace, in int32: block counts; what the first page list holds; then by call.
struct Work {
  int32_t *counts;   // [blocks] free pages of each block
  int32_t *head;     // [4]: free pages in all, moves
  int32_t *free_of;  // [n_pages] page of each rank among the free
  int32_t *a, *b;    // reserve: wanted [batch], offset [batch]; fork: owner [batch], slot [n];
                     // compact: pages to move, highest first [n_pages], rank [n_pages]
};
size_t blocks_of(size_t n_pages) { return cdiv(n_pages, (size_t)kBlockPages); }
size_t work_words(size_t n_pages, size_t rows) {
  const size_t a = n_pages > rows ? n_pages : rows;
  return roundup(blocks_of(n_pages), 4) + 4 + n_pages + 2 * a;
}
Work work_of(void *ws, size_t n_pages, size_t rows) {
  const size_t a = n_pages > rows ? n_pages : rows;
  Work w;
  w.counts = static_cast<int32_t *>(ws);
  w.head = w.counts + roundup(blocks_of(n_pages), 4);
  w.free_of = w.head + 4;
  w.a = w.free_of + n_pages;
  w.b = w.a + a;
  return w;
}

__device__ __forceinline__ int wave_sum(int v) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) v += __shfl_xor(v, m);
  return v;
}
// Sum over the workgroup, in every thread (s: an int of LDS for each of its waves).
template <int WAVES>
__device__ __forceinline__ int block_sum(int v, int *s) {
  v = wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
  __syncthreads();
  int all = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) all += s[w];
  return all;
}
// Sum of v over the threads before this one; *all: over the workgroup.
template <int WAVES>
__device__ __forceinline__ int block_before(int v, int *s, int *all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int x = v;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int y = __shfl_up(x, d);
    if (lane >= d) x += y;
  }
  __syncthreads();
  if (lane == 63) s[wave] = x;
  __syncthreads();
  int before = 0, sum = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    before += w < wave ? s[w] : 0;
    sum += s[w];
  }
  *all = sum;
  return before + x - v;
}

// Which of a wave's pages p0 + 64 i + lane are free, as one mask a step.
__device__ __forceinline__ int free_masks(const int32_t *refs, int n_pages, int p0,
                                          uint64_t (&mask)[kSteps]) {
  const int lane = threadIdx.x & 63;
  int r[kSteps];
#pragma unroll
  for (int i = 0; i < kSteps; ++i) {
    r[i] = refs[min(p0 + 64 * i + lane, n_pages - 1)];  // all loads at once
  }
  int n = 0;
#pragma unroll
  for (int i = 0; i < kSteps; ++i) {
    mask[i] = __ballot(r[i] <= 0 && p0 + 64 * i + lane < n_pages);
    n += __popcll(mask[i]);
  }
  return n;
}
__device__ __forceinline__ int first_page() {
  return blockIdx.x * kBlockPages + (threadIdx.x >> 6) * 64 * kSteps;
}
__device__ __forceinline__ void count_block(const int32_t *refs, int n_pages, int32_t *counts) {
  __shared__ int s[4];
  uint64_t mask[kSteps];
  const int n = free_masks(refs, n_pages, first_page(), mask);
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = n;
  __syncthreads();
  if (threadIdx.x == 0) counts[blockIdx.x] = s[0] + s[1] + s[2] + s[3];
}
// Free pages before this block, and in all.
__device__ __forceinline__ int free_before(const int32_t *counts, int blocks, int at, int *all,
                                           int *s) {
  int before = 0, total = 0;
  for (int i = threadIdx.x; i < blocks; i += kThreads) {
    const int c = counts[i];
    total += c;
    before += i < at ? c : 0;
  }
  *all = block_sum<4>(total, s);
  return block_sum<4>(before, s);
}

// The table entries of row b that hold positions from .. from + n - 1 (clipped to the
// table), and how many more pages the positions would need.
__device__ __forceinline__ bool entries_of(const int32_t *lens, const int32_t *counts, int b,
                                           int max_pages, int *e0, int *e1, long long *beyond) {
  const long long len = max(lens[b], 0), n = counts[b];
  *beyond = 0;
  if (n <= 0) return false;
  const long long first = len / kKvPage, last = (len + n - 1) / kKvPage;
  *e0 = (int)min(first, (long long)max_pages);
  *e1 = (int)min(last + 1, (long long)max_pages);
  *beyond = last + 1 - max(first, (long long)max_pages);
  if (*beyond < 0) *beyond = 0;
  return true;
}
__device__ __forceinline__ bool names(int p, int n_pages) { return p >= 0 && p < n_pages; }

// ------------------------------------------------------------------ reserve --
// Entries of a lane that are in flight at a time: a row may want thousands.  One row of 2048
// entries 14 us, of 8192 35; one entry after the other took a thread 418 and 1631.
constexpr int kEntrySteps = 8;
// One wave: how many of a row's entries e0 .. e1 - 1 name no page.
__device__ __forceinline__ int row_wants(const int32_t *row, int e0, int e1, int n_pages) {
  const int lane = threadIdx.x & 63;
  int n = 0;
  for (int e = e0; e < e1; e += 64 * kEntrySteps) {
    int32_t v[kEntrySteps];
#pragma unroll
    for (int i = 0; i < kEntrySteps; ++i) v[i] = row[min(e + 64 * i + lane, e1 - 1)];
#pragma unroll
    for (int i = 0; i < kEntrySteps; ++i)
      n += e + 64 * i + lane < e1 && !names(v[i], n_pages);
  }
  return wave_sum(n);
}
// One wave: those entries take the free pages from rank `at`, -1 where there are no more.
__device__ __forceinline__ void row_takes(int32_t *row, int e0, int e1, int at, int n_free,
                                          const int32_t *free_of, int32_t *refs, int n_pages) {
  const int lane = threadIdx.x & 63;
  for (int e = e0; e < e1; e += 64 * kEntrySteps) {
    int32_t v[kEntrySteps];
    int k[kEntrySteps];
#pragma unroll
    for (int i = 0; i < kEntrySteps; ++i) v[i] = row[min(e + 64 * i + lane, e1 - 1)];
#pragma unroll
    for (int i = 0; i < kEntrySteps; ++i) {
      const bool want = e + 64 * i + lane < e1 && !names(v[i], n_pages);
      const uint64_t mask = __ballot(want);
      k[i] = want ? at + __popcll(mask & ((1ull << lane) - 1)) : -1;
      at += __popcll(mask);
    }
#pragma unroll
    for (int i = 0; i < kEntrySteps; ++i)
      v[i] = k[i] >= 0 && k[i] < n_free ? free_of[k[i]] : -1;
#pragma unroll
    for (int i = 0; i < kEntrySteps; ++i) {
      if (k[i] < 0) continue;
      row[e + 64 * i + lane] = v[i];
      if (v[i] >= 0) refs[v[i]] = 1;
    }
  }
}
// Workgroups past the blocks of pages: a wave counts what a row of the table wants.
__global__ __launch_bounds__(kThreads) void reserve_count_kernel(
    const int32_t *refs, int n_pages, int blocks, const int32_t *table, int max_pages,
    const int32_t *lens, const int32_t *counts, int batch, Work w) {
  if ((int)blockIdx.x < blocks) {
    count_block(refs, n_pages, w.counts);
    return;
  }
  const int b = (blockIdx.x - blocks) * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (b >= batch) return;
  int e0, e1, n = 0;
  long long beyond;
  if (entries_of(lens, counts, b, max_pages, &e0, &e1, &beyond))
    n = row_wants(table + (size_t)b * max_pages, e0, e1, n_pages);
  if (lane == 0) w.a[b] = n;
}

// A wave's free pages take their ranks, those below `most`.
__device__ __forceinline__ void list_wave(const uint64_t (&mask)[kSteps], int p0, int rank,
                                          int most, int32_t *free_of) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int i = 0; i < kSteps; ++i) {
    const int k = rank + __popcll(mask[i] & ((1ull << lane) - 1));
    if (((mask[i] >> lane) & 1) && k < most) free_of[k] = p0 + 64 * i + lane;
    rank += __popcll(mask[i]);
  }
}
// One workgroup of kPlanThreads, at most kSmallPages: the lowest `want` free pages into
// free_of; returns how many are free.
__device__ __forceinline__ int list_free(const int32_t *refs, int n_pages, int want,
                                         int32_t *free_of, int *s) {
  if (n_pages == 0 || want == 0) return 0;
  const int wave = threadIdx.x >> 6, p0 = wave * 64 * kSteps;
  uint64_t mask[kSteps];
  const int n = free_masks(refs, n_pages, p0, mask);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s[wave] = n;
  __syncthreads();
  int rank = 0, found = 0;
#pragma unroll
  for (int v = 0; v < kPlanWaves; ++v) {
    rank += v < wave ? s[v] : 0;
    found += s[v];
  }
  list_wave(mask, p0, rank, want, free_of);
  return found;
}
// Ranks the free pages of its block.
__device__ __forceinline__ void list_block(const int32_t *refs, int n_pages, int blocks,
                                           const Work &w) {
  __shared__ int s[4], s_wave[4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, p0 = first_page();
  uint64_t mask[kSteps];
  const int n = free_masks(refs, n_pages, p0, mask);
  int all, rank = free_before(w.counts, blocks, blockIdx.x, &all, s);
  if (lane == 0) s_wave[wave] = n;
  __syncthreads();
  for (int v = 0; v < wave; ++v) rank += s_wave[v];
  list_wave(mask, p0, rank, INT_MAX, w.free_of);
}
// Writes the free pages in all and what of `wanted` (and of pages past the table) is missing.
__device__ __forceinline__ void tell(long long wanted, long long beyond, int blocks,
                                     const Work &w, int32_t *shortfall, int *s) {
  int all;
  (void)free_before(w.counts, blocks, 0, &all, s);
  if (threadIdx.x != 0) return;
  w.head[0] = all;
  const long long missing = beyond + (wanted > all ? wanted - all : 0);
  if (shortfall != nullptr) *shortfall = (int32_t)min(missing, (long long)INT_MAX);
}

__global__ __launch_bounds__(kThreads) void reserve_list_kernel(
    const int32_t *refs, int n_pages, int blocks, int max_pages, const int32_t *lens,
    const int32_t *counts, int batch, int32_t *shortfall, Work w) {
  if ((int)blockIdx.x < blocks) {
    list_block(refs, n_pages, blocks, w);
    return;
  }
  // The last workgroup scans the rows' wants, 8 rows a thread.
  __shared__ int s[4];
  __shared__ long long s_beyond[kThreads];
  constexpr int kRows = 8;
  int base = 0;  // at most the table's entries: below 2^31 (host check)
  long long beyond = 0;
  for (int b0 = 0; b0 < batch; b0 += kThreads * kRows) {
    int v[kRows], sum = 0;
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const int b = b0 + kRows * threadIdx.x + i;
      v[i] = b < batch ? w.a[b] : 0;
      sum += v[i];
      if (b < batch) {
        int e0, e1;
        long long more;
        (void)entries_of(lens, counts, b, max_pages, &e0, &e1, &more);
        beyond += more;
      }
    }
    int all, at = base + block_before<4>(sum, s, &all);
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const int b = b0 + kRows * threadIdx.x + i;
      if (b < batch) w.b[b] = at;
      at += v[i];
    }
    base += all;
  }
  s_beyond[threadIdx.x] = beyond;
  __syncthreads();
  if (threadIdx.x == 0) {
    beyond = 0;
    for (int i = 0; i < kThreads; ++i) beyond += s_beyond[i];
  }
  tell(base, beyond, blocks, w, shortfall, s);
}

__global__ __launch_bounds__(kThreads) void reserve_apply_kernel(
    int32_t *refs, int n_pages, int32_t *table, int max_pages, const int32_t *lens,
    const int32_t *counts, int batch, Work w) {
  const int b = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (b >= batch || w.a[b] == 0) return;
  int e0, e1;
  long long beyond;
  if (!entries_of(lens, counts, b, max_pages, &e0, &e1, &beyond)) return;
  row_takes(table + (size_t)b * max_pages, e0, e1, w.b[b], w.head[0], w.free_of, refs, n_pages);
}

// All of it in one workgroup: a thread for each row, a wave for one of more than kShortRow
// entries.
constexpr int kShortRow = 4;
__global__ __launch_bounds__(kPlanThreads) void reserve_small_kernel(
    int32_t *refs, int n_pages, int32_t *table, int max_pages, const int32_t *lens,
    const int32_t *counts, int batch, int32_t *shortfall, Work w) {
  // Of each row what it wants, then the rank of its first page; the rows with many entries.
  __shared__ int s[kPlanWaves], s_row[kSmallRows], s_long[kSmallRows], n_long;
  __shared__ unsigned long long s_beyond;
  const int wave = threadIdx.x >> 6;
  if (threadIdx.x == 0) {
    s_beyond = 0;
    n_long = 0;
  }
  __syncthreads();
  int e0, e1;
  long long beyond;
  for (int b = threadIdx.x; b < batch; b += kPlanThreads) {
    int n = 0;
    if (entries_of(lens, counts, b, max_pages, &e0, &e1, &beyond)) {
      if (beyond) atomicAdd(&s_beyond, (unsigned long long)beyond);
      if (e1 - e0 > kShortRow) {
        s_long[atomicAdd(&n_long, 1)] = b;  // in any order: each is counted by itself
      } else {
        for (int e = e0; e < e1; ++e) n += !names(table[(size_t)b * max_pages + e], n_pages);
      }
    }
    s_row[b] = n;
  }
  __syncthreads();
  for (int i = wave; i < n_long; i += kPlanWaves) {
    const int b = s_long[i];
    (void)entries_of(lens, counts, b, max_pages, &e0, &e1, &beyond);
    const int n = row_wants(table + (size_t)b * max_pages, e0, e1, n_pages);
    if ((threadIdx.x & 63) == 0) s_row[b] = n;
  }
  __syncthreads();
  int base = 0;
  for (int b0 = 0; b0 < batch; b0 += kPlanThreads) {
    const int b = b0 + threadIdx.x, n = b < batch ? s_row[b] : 0;
    int all;
    const int at = base + block_before<kPlanWaves>(n, s, &all);
    if (b < batch) s_row[b] = at;
    base += all;
  }
  const int found = list_free(refs, n_pages, base, w.free_of, s);
  __syncthreads();  // the list is written
  if (threadIdx.x == 0 && shortfall != nullptr) {
    const long long missing = (long long)s_beyond + (base > found ? base - found : 0);
    *shortfall = (int32_t)min(missing, (long long)INT_MAX);
  }
  for (int i = wave; i < n_long; i += kPlanWaves) {
    const int b = s_long[i];
    (void)entries_of(lens, counts, b, max_pages, &e0, &e1, &beyond);
    row_takes(table + (size_t)b * max_pages, e0, e1, s_row[b], found, w.free_of, refs, n_pages);
  }
  for (int b = threadIdx.x; b < batch; b += kPlanThreads) {
    if (!entries_of(lens, counts, b, max_pages, &e0, &e1, &beyond) || e1 - e0 > kShortRow)
      continue;
    int at = s_row[b];
    for (int e = e0; e < e1; ++e) {
      int32_t *entry = table + (size_t)b * max_pages + e;
      if (names(*entry, n_pages)) continue;
      const int p = at < found ? w.free_of[at] : -1;
      ++at;
      *entry = p;
      if (p >= 0) refs[p] = 1;
    }
  }
}

// --------------------------------------------------------------------- fork --
__global__ __launch_bounds__(kThreads) void count_kernel(const int32_t *refs, int n_pages,
                                                         Work w) {
  count_block(refs, n_pages, w.counts);
}

// The first item that names a row as its child has it: owners of rows in LDS, or, past
// kSmallRows, in memory, where atomics and accesses beside them have to meet.
struct LdsOwners {
  int *at;
  __device__ void clear(int r) { at[r] = INT_MAX; }
  __device__ void claim(int r, int i) { atomicMin(at + r, i); }
  __device__ int of(int r) { return at[r]; }
  __device__ void join() { __syncthreads(); }
};
struct MemoryOwners {
  int32_t *at;
  __device__ void clear(int r) {
    __hip_atomic_store(at + r, INT_MAX, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __device__ void claim(int r, int i) { atomicMin(at + r, i); }
  __device__ int of(int r) {
    return __hip_atomic_load(at + r, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __device__ void join() {
    __threadfence();
    __syncthreads();
  }
};

// One workgroup: of each item the rank of its new page among the free ones, -1 where it
// needs none, -2 where the item is left out.  Returns how many want a page.
template <int WAVES, typename Owners>
__device__ __forceinline__ int fork_items(Owners own, int n_pages, const int32_t *table,
                                          int max_pages,
                                          const int32_t *lens, int batch, const int32_t *parents,
                                          const int32_t *children, int n, const Work &w, int *s) {
  constexpr int kT = 64 * WAVES;
  for (int r = threadIdx.x; r < batch; r += kT) own.clear(r);
  own.join();
  for (int i = threadIdx.x; i < n; i += kT) {
    const int c = children[i];
    if (c >= 0 && c < batch) own.claim(c, i);
  }
  own.join();
  int base = 0;
  for (int i0 = 0; i0 < n; i0 += kT) {
    const int i = i0 + threadIdx.x;
    bool ok = false, want = false;
    if (i < n) {
      const int c = children[i], p = parents[i];
      ok = c >= 0 && c < batch && p >= 0 && p < batch && own.of(c) == i &&
           own.of(p) == INT_MAX;
      if (ok) {
        const int L = min(max(lens[p], 0), max_pages * kKvPage);
        want = L % kKvPage != 0 &&
               names(table[(size_t)p * max_pages + L / kKvPage], n_pages);
      }
    }
    int all;
    const int at = base + block_before<WAVES>(want ? 1 : 0, s, &all);
    if (i < n) w.b[i] = !ok ? -2 : want ? at : -1;
    base += all;
  }
  return base;
}

__global__ __launch_bounds__(kThreads) void fork_list_kernel(
    const int32_t *refs, int n_pages, int blocks, const int32_t *table, int max_pages,
    const int32_t *lens, int batch, const int32_t *parents, const int32_t *children, int n,
    int32_t *shortfall, Work w) {
  if ((int)blockIdx.x < blocks) {
    list_block(refs, n_pages, blocks, w);
    return;
  }
  __shared__ int s[4];
  const int want =
      fork_items<4>(MemoryOwners{w.a}, n_pages, table, max_pages, lens, batch, parents, children,
                    n, w, s);
  tell(want, 0, blocks, w, shortfall, s);
}
__global__ __launch_bounds__(kPlanThreads) void fork_small_kernel(
    const int32_t *refs, int n_pages, const int32_t *table, int max_pages, const int32_t *lens,
    int batch, const int32_t *parents, const int32_t *children, int n, int32_t *shortfall,
    Work w) {
  __shared__ int s[kPlanWaves], s_owner[kSmallRows];
  const int want = fork_items<kPlanWaves>(LdsOwners{s_owner}, n_pages, table, max_pages, lens,
                                          batch, parents, children, n, w, s);
  const int found = list_free(refs, n_pages, want, w.free_of, s);
  if (threadIdx.x != 0) return;
  w.head[0] = found;
  if (shortfall != nullptr) *shortfall = want > found ? want - found : 0;
}

// Chunk `ch` of a page.
__device__ __forceinline__ void copy_chunk(const uint8_t *cache_from, int from, uint8_t *cache_to,
                                           int to, const Chunks &c, int ch) {
  const size_t bytes = (size_t)c.pieces * 16;
  const u32x4 *src = reinterpret_cast<const u32x4 *>(cache_from + from * bytes) + ch * c.chunk;
  u32x4 *dst = reinterpret_cast<u32x4 *>(cache_to + to * bytes) + ch * c.chunk;
  const int n = min(c.chunk, c.pieces - ch * c.chunk);
  u32x4 v[kCopyUnroll];
#pragma unroll
  for (int j = 0; j < kCopyUnroll; ++j)  // without a branch: all loads at once
    v[j] = src[min(j * kThreads + (int)threadIdx.x, n - 1)];
#pragma unroll
  for (int j = 0; j < kCopyUnroll; ++j) {
    const int x = j * kThreads + threadIdx.x;
    if (x < n) dst[x] = v[j];
  }
}

// Grid (items, chunks of a page): the first chunk's workgroups write the table too.
__global__ __launch_bounds__(kThreads) void fork_apply_kernel(
    uint8_t *cache, int32_t *refs, int n_pages, int32_t *table, int max_pages, int32_t *lens,
    const int32_t *parents, const int32_t *children, Chunks c16, Work w) {
  const int i = blockIdx.x, slot = w.b[i];
  if (slot == -2) return;
  const int c = children[i], p = parents[i];
  const int L = min(max(lens[p], 0), max_pages * kKvPage), full = L / kKvPage;
  const int32_t *from = table + (size_t)p * max_pages;
  const int fresh = slot >= 0 && slot < w.head[0] ? w.free_of[slot] : -1;
  if (fresh >= 0) copy_chunk(cache, from[full], cache, fresh, c16, blockIdx.y);
  if (blockIdx.y != 0) return;
  int32_t *to = table + (size_t)c * max_pages;
  for (int e = threadIdx.x; e < max_pages; e += kThreads) {
    int v = e < full ? from[e] : e == full ? fresh : -1;
    if (!names(v, n_pages)) v = -1;
    to[e] = v;
    if (e < full && v >= 0) atomicAdd(refs + v, 1);
  }
  if (threadIdx.x == 0) {
    lens[c] = L;
    if (fresh >= 0) refs[fresh] = 1;
  }
}

// ------------------------------------------------------------------ release --
// An entry is taken out of the table by an exchange, so rows named twice give a page back
// once; a count is not taken below 0.
__global__ __launch_bounds__(kThreads) void release_kernel(int32_t *refs, int n_pages,
                                                           int32_t *table, int max_pages,
                                                           int batch, const int32_t *rows,
                                                           const int32_t *keep) {
  const int i = blockIdx.x, row = rows[i];
  if (row < 0 || row >= batch) return;
  const int kept = keep == nullptr ? 0 : max(keep[i], 0);
  const int first = kept / kKvPage + (kept % kKvPage != 0);
  for (int e = first + blockIdx.y * kThreads + threadIdx.x; e < max_pages;
       e += gridDim.y * kThreads) {
    int32_t *entry = table + (size_t)row * max_pages + e;
    if (*entry == -1) continue;
    const int p = atomicExch(entry, -1);
    if (names(p, n_pages) && atomicAdd(refs + p, -1) <= 0) atomicAdd(refs + p, 1);
  }
}

// ------------------------------------------------------------------ compact --
// With n_live pages in use, those at n_live and above move to the free ones below; both
// are equally many (head[1]).  a: the moving pages, highest first; b: of every page its
// index in a, -1 where it is in use and stays, -2 where it is free.
__device__ __forceinline__ void compact_wave(const uint64_t (&mask)[kSteps], int p0, int rank,
                                             int n_pages, int live, const Work &w) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int i = 0; i < kSteps; ++i) {
    const int p = p0 + 64 * i + lane, f = rank + __popcll(mask[i] & ((1ull << lane) - 1));
    if (p < n_pages) {
      const bool is_free = (mask[i] >> lane) & 1;
      int b = is_free ? -2 : -1;
      if (is_free && p < live) w.free_of[f] = p;
      if (!is_free && p >= live) {
        b = live - 1 - (p - f);  // p - f pages in use are below p
        w.a[b] = p;
      }
      if (p == live) w.head[1] = f;
      w.b[p] = b;
    }
    rank += __popcll(mask[i]);
  }
}
__global__ __launch_bounds__(kThreads) void compact_list_kernel(const int32_t *refs, int n_pages,
                                                                int blocks, int32_t *n_live,
                                                                Work w) {
  __shared__ int s[4], s_wave[4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, p0 = first_page();
  uint64_t mask[kSteps];
  const int n = free_masks(refs, n_pages, p0, mask);
  int all, rank = free_before(w.counts, blocks, blockIdx.x, &all, s);
  if (lane == 0) s_wave[wave] = n;
  __syncthreads();
  for (int v = 0; v < wave; ++v) rank += s_wave[v];
  const int live = n_pages - all;
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    *n_live = live;
    if (live == n_pages) w.head[1] = 0;
  }
  compact_wave(mask, p0, rank, n_pages, live, w);
}
__global__ __launch_bounds__(kPlanThreads) void compact_small_kernel(const int32_t *refs,
                                                                     int n_pages,
                                                                     int32_t *n_live, Work w) {
  __shared__ int s[kPlanWaves];
  const int wave = threadIdx.x >> 6, p0 = wave * 64 * kSteps;
  uint64_t mask[kSteps];
  const int n = n_pages == 0 ? 0 : free_masks(refs, n_pages, p0, mask);
  if ((threadIdx.x & 63) == 0) s[wave] = n;
  __syncthreads();
  int rank = 0, all = 0;
#pragma unroll
  for (int v = 0; v < kPlanWaves; ++v) {
    rank += v < wave ? s[v] : 0;
    all += s[v];
  }
  const int live = n_pages - all;
  if (threadIdx.x == 0) {
    *n_live = live;
    if (live == n_pages) w.head[1] = 0;
  }
  if (n_pages != 0) compact_wave(mask, p0, rank, n_pages, live, w);
}

__global__ __launch_bounds__(kThreads) void compact_apply_kernel(
    uint8_t *cache, int32_t *refs, int n_pages, int32_t *table, size_t entries, Chunks c16,
    int32_t *new_page, Work w) {
  const int moves = w.head[1];
  const long long units = (long long)moves * c16.chunks;
  for (long long u = blockIdx.x; u < units; u += gridDim.x) {
    const int r = (int)(u / c16.chunks), ch = (int)(u - (long long)r * c16.chunks);
    copy_chunk(cache, w.a[moves - 1 - r], cache, w.free_of[r], c16, ch);
  }
  const size_t first = (size_t)blockIdx.x * kThreads + threadIdx.x,
               step = (size_t)gridDim.x * kThreads;
  for (size_t p = first; p < (size_t)n_pages; p += step) {
    const int b = w.b[p];
    int to = b == -2 ? -1 : (int)p;
    if (b >= 0) {
      to = w.free_of[moves - 1 - b];
      refs[to] = refs[p];
      refs[p] = 0;
    }
    new_page[p] = to;
  }
  for (size_t e = first; e < entries; e += step) {
    const int p = table[e];
    if (!names(p, n_pages)) continue;
    const int b = w.b[p];
    if (b != -1) table[e] = b == -2 ? -1 : w.free_of[moves - 1 - b];
  }
}

// --------------------------------------------------------------------- copy --
// Grid (chunks of a page, items).
__global__ __launch_bounds__(kThreads) void copy_kernel(uint8_t *dst, int dst_pages,
                                                        const uint8_t *src, int src_pages,
                                                        const int32_t *to, const int32_t *from,
                                                        int n, Chunks c16) {
  for (int i = blockIdx.y; i < n; i += gridDim.y) {
    const int t = to[i], f = from[i];
    if (names(t, dst_pages) && names(f, src_pages))
      copy_chunk(src, f, dst, t, c16, blockIdx.x);
  }
}

// Checks that the calls share; `ws_rows`: what the workspace holds rows for.
int pages_check(const char *who, const int32_t *refs, size_t n_pages, const int32_t *table,
                size_t max_pages, size_t batch) {
  PRICHS_REQUIRE(n_pages <= kMaxPages && batch <= kMaxRows &&
                     max_pages <= (size_t)INT32_MAX / kKvPage &&
                     (batch == 0 || max_pages <= (size_t)INT32_MAX / batch),
                 "%s: shape too large", who);
  PRICHS_REQUIRE((refs || n_pages == 0) && (table || batch * max_pages == 0),
                 "%s: null pointer argument", who);
  return PRICHS_OK;
}
int work_check(const char *who, const void *ws, size_t bytes, size_t need) {
  if (bytes < need)
    return fail(PRICHS_ERR_CAPACITY, "%s: workspace of %zu bytes, %zu needed", who, bytes, need);
  PRICHS_REQUIRE(ws != nullptr && reinterpret_cast<uintptr_t>(ws) % 16 == 0,
                 "%s: the workspace must be 16-byte aligned device memory", who);
  return PRICHS_OK;
}
int page_check(const char *who, const void *cache, size_t n_pages, size_t n_kv_heads) {
  PRICHS_REQUIRE(n_kv_heads >= 1 && n_kv_heads <= 65535, "%s: n_kv_heads=%zu", who, n_kv_heads);
  PRICHS_REQUIRE(cache || n_pages == 0, "%s: null pointer argument", who);
  PRICHS_REQUIRE(reinterpret_cast<uintptr_t>(cache) % 16 == 0,
                 "%s: the cache must be 16-byte aligned", who);
  return PRICHS_OK;
}

}  // namespace
}  // namespace prichs

using namespace prichs;

extern "C" size_t prichs_kv_pages_workspace(size_t n_pages, size_t batch, size_t n) {
  if (n_pages > kMaxPages || batch > kMaxRows || n > kMaxRows) return 0;
  return work_words(n_pages, batch > n ? batch : n) * sizeof(int32_t);
}

extern "C" int prichs_kv_pages_reserve(int32_t *refs, size_t n_pages, int32_t *page_table,
                                       size_t max_pages, const int32_t *lens,
                                       const int32_t *counts, size_t batch, int32_t *shortfall,
                                       void *workspace, size_t workspace_bytes, void *stream) {
  const char *who = "kv_pages_reserve";
  PRICHS_TRY(pages_check(who, refs, n_pages, page_table, max_pages, batch));
  PRICHS_REQUIRE(batch == 0 || (lens && counts), "%s: null pointer argument", who);
  if (batch == 0 && shortfall == nullptr) return PRICHS_OK;
  PRICHS_TRY(work_check(who, workspace, workspace_bytes,
                        prichs_kv_pages_workspace(n_pages, batch, 0)));
  const Work w = work_of(workspace, n_pages, batch);
  const hipStream_t s = as_stream(stream);
  if (n_pages <= kSmallPages && batch <= kSmallRows) {
    hipLaunchKernelGGL(reserve_small_kernel, dim3(1), dim3(kPlanThreads), 0, s, refs, (int)n_pages,
                       page_table, (int)max_pages, lens, counts, (int)batch, shortfall, w);
    PRICHS_LAUNCH_CHECK("kv_pages_reserve launch");
    return PRICHS_OK;
  }
  const unsigned blocks = (unsigned)blocks_of(n_pages), rows = (unsigned)cdiv(batch, 4);
  if (blocks + rows > 0) {
    hipLaunchKernelGGL(reserve_count_kernel, dim3(blocks + rows), dim3(kThreads), 0, s, refs,
                       (int)n_pages, (int)blocks, page_table, (int)max_pages, lens, counts,
                       (int)batch, w);
    PRICHS_LAUNCH_CHECK("kv_pages_reserve count launch");
  }
  hipLaunchKernelGGL(reserve_list_kernel, dim3(blocks + 1), dim3(kThreads), 0, s, refs,
                     (int)n_pages, (int)blocks, (int)max_pages, lens, counts, (int)batch,
                     shortfall, w);
  PRICHS_LAUNCH_CHECK("kv_pages_reserve list launch");
  if (rows > 0) {
    hipLaunchKernelGGL(reserve_apply_kernel, dim3(rows), dim3(kThreads), 0, s, refs, (int)n_pages,
                       page_table, (int)max_pages, lens, counts, (int)batch, w);
    PRICHS_LAUNCH_CHECK("kv_pages_reserve launch");
  }
  return PRICHS_OK;
}

extern "C" int prichs_kv_pages_fork(void *cache, int32_t *refs, size_t n_pages,
                                    int32_t *page_table, size_t max_pages, int32_t *lens,
                                    size_t batch, const int32_t *parents,
                                    const int32_t *children, size_t n, size_t n_kv_heads,
                                    int32_t *shortfall, void *workspace, size_t workspace_bytes,
                                    void *stream) {
  const char *who = "kv_pages_fork";
  PRICHS_TRY(pages_check(who, refs, n_pages, page_table, max_pages, batch));
  PRICHS_TRY(page_check(who, cache, n_pages, n_kv_heads));
  PRICHS_REQUIRE(n <= kMaxRows, "%s: shape too large", who);
  PRICHS_REQUIRE((batch == 0 || lens) && (n == 0 || (parents && children)),
                 "%s: null pointer argument", who);
  if (n == 0 && shortfall == nullptr) return PRICHS_OK;
  PRICHS_TRY(work_check(who, workspace, workspace_bytes,
                        prichs_kv_pages_workspace(n_pages, batch, n)));
  const Work w = work_of(workspace, n_pages, batch > n ? batch : n);
  const hipStream_t s = as_stream(stream);
  if (n_pages <= kSmallPages && batch <= kSmallRows && n <= kSmallRows) {
    hipLaunchKernelGGL(fork_small_kernel, dim3(1), dim3(kPlanThreads), 0, s, refs, (int)n_pages,
                       page_table, (int)max_pages, lens, (int)batch, parents, children, (int)n,
                       shortfall, w);
  } else {
    const unsigned blocks = (unsigned)blocks_of(n_pages);
    if (blocks > 0) {
      hipLaunchKernelGGL(count_kernel, dim3(blocks), dim3(kThreads), 0, s, refs, (int)n_pages, w);
      PRICHS_LAUNCH_CHECK("kv_pages_fork count launch");
    }
    hipLaunchKernelGGL(fork_list_kernel, dim3(blocks + 1), dim3(kThreads), 0, s, refs,
                       (int)n_pages, (int)blocks, page_table, (int)max_pages, lens, (int)batch,
                       parents, children, (int)n, shortfall, w);
  }
  PRICHS_LAUNCH_CHECK("kv_pages_fork list launch");
  if (n > 0) {
    const Chunks c16(n_kv_heads);
    hipLaunchKernelGGL(fork_apply_kernel, dim3((unsigned)n, (unsigned)c16.chunks),
                       dim3(kThreads), 0, s, static_cast<uint8_t *>(cache), refs, (int)n_pages,
                       page_table, (int)max_pages, lens, parents, children, c16, w);
    PRICHS_LAUNCH_CHECK("kv_pages_fork launch");
  }
  return PRICHS_OK;
}

extern "C" int prichs_kv_pages_release(int32_t *refs, size_t n_pages, int32_t *page_table,
                                       size_t max_pages, size_t batch, const int32_t *rows,
                                       const int32_t *keep, size_t n, void *stream) {
  const char *who = "kv_pages_release";
  PRICHS_TRY(pages_check(who, refs, n_pages, page_table, max_pages, batch));
  PRICHS_REQUIRE(n <= kMaxRows, "%s: shape too large", who);
  PRICHS_REQUIRE(n == 0 || rows, "%s: null pointer argument", who);
  if (n == 0 || batch == 0 || max_pages == 0) return PRICHS_OK;
  const size_t parts = cdiv(max_pages, (size_t)kThreads);
  hipLaunchKernelGGL(release_kernel, dim3((unsigned)n, (unsigned)(parts < 1024 ? parts : 1024)),
                     dim3(kThreads), 0, as_stream(stream), refs, (int)n_pages, page_table,
                     (int)max_pages, (int)batch, rows, keep);
  PRICHS_LAUNCH_CHECK("kv_pages_release launch");
  return PRICHS_OK;
}

extern "C" int prichs_kv_pages_compact(void *cache, int32_t *refs, size_t n_pages,
                                       int32_t *page_table, size_t max_pages, size_t batch,
                                       size_t n_kv_heads, int32_t *new_page, int32_t *n_live,
                                       void *workspace, size_t workspace_bytes, void *stream) {
  const char *who = "kv_pages_compact";
  PRICHS_TRY(pages_check(who, refs, n_pages, page_table, max_pages, batch));
  PRICHS_TRY(page_check(who, cache, n_pages, n_kv_heads));
  PRICHS_REQUIRE((new_page || n_pages == 0) && n_live, "%s: null pointer argument", who);
  PRICHS_TRY(work_check(who, workspace, workspace_bytes,
                        prichs_kv_pages_workspace(n_pages, 0, 0)));
  const Work w = work_of(workspace, n_pages, 0);
  const hipStream_t s = as_stream(stream);
  if (n_pages <= kSmallPages) {
    hipLaunchKernelGGL(compact_small_kernel, dim3(1), dim3(kPlanThreads), 0, s, refs,
                       (int)n_pages, n_live, w);
  } else {
    const unsigned blocks = (unsigned)blocks_of(n_pages);
    hipLaunchKernelGGL(count_kernel, dim3(blocks), dim3(kThreads), 0, s, refs, (int)n_pages, w);
    PRICHS_LAUNCH_CHECK("kv_pages_compact count launch");
    hipLaunchKernelGGL(compact_list_kernel, dim3(blocks), dim3(kThreads), 0, s, refs,
                       (int)n_pages, (int)blocks, n_live, w);
  }
  PRICHS_LAUNCH_CHECK("kv_pages_compact list launch");
  if (n_pages == 0) return PRICHS_OK;
  const Chunks c16(n_kv_heads);
  const size_t entries = batch * max_pages;
  // At most half of the pages move; workgroups loop over what there is.
  size_t grid = cdiv(n_pages, 2) * c16.chunks;
  const size_t small = cdiv(n_pages > entries ? n_pages : entries, (size_t)kThreads);
  grid = grid > small ? grid : small;
  hipLaunchKernelGGL(compact_apply_kernel, dim3((unsigned)(grid < 2048 ? grid : 2048)),
                     dim3(kThreads), 0, s, static_cast<uint8_t *>(cache), refs, (int)n_pages,
                     page_table, entries, c16, new_page, w);
  PRICHS_LAUNCH_CHECK("kv_pages_compact launch");
  return PRICHS_OK;
}

extern "C" int prichs_kv_cache_copy(void *dst, size_t dst_pages, const void *src,
                                    size_t src_pages, const int32_t *to, const int32_t *from,
                                    size_t n, size_t n_kv_heads, void *stream) {
  const char *who = "kv_cache_copy";
  PRICHS_TRY(page_check(who, dst, dst_pages, n_kv_heads));
  PRICHS_TRY(page_check(who, src, src_pages, n_kv_heads));
  PRICHS_REQUIRE(dst_pages <= (size_t)INT32_MAX && src_pages <= (size_t)INT32_MAX &&
                     n <= (size_t)INT32_MAX / 2,
                 "%s: shape too large", who);
  PRICHS_REQUIRE(n == 0 || (to && from), "%s: null pointer argument", who);
  if (n == 0 || dst_pages == 0 || src_pages == 0) return PRICHS_OK;
  const Chunks c16(n_kv_heads);
  hipLaunchKernelGGL(copy_kernel, dim3((unsigned)c16.chunks, (unsigned)(n < 65535 ? n : 65535)),
                     dim3(kThreads), 0, as_stream(stream), static_cast<uint8_t *>(dst),
                     (int)dst_pages, static_cast<const uint8_t *>(src), (int)src_pages, to, from,
                     (int)n, c16);
  PRICHS_LAUNCH_CHECK("kv_cache_copy launch");
  return PRICHS_OK;
}
