// kv_shared_attention.hip -- attention of each sequence's last tokens over the paged 4-bit
// KV cache where groups of sequences share their first pages: the shared pages are read
// and multiplied once for all rows of a group, each sequence's own pages once for its
// rows, and the parts are joined.  With o_p, m_p, l_p the sums, maximum and sum of
// exponentials over part p of the keys,
//   o = sum_p exp(m_p - m) o_p / sum_p exp(m_p - m) l_p,  m = max_p m_p.
// kv_attend.hpp has the tiles and the join.
//
// MI355X, 12 + 3 heads, us from Python (kernels): 8 sequences of one prompt of 1000
// positions 11 (10 captured), 16 prompts of 2048 with 4 sequences each 15, 24 x 6 tokens
// behind 8000 shared positions 25, 256 sequences behind 32768 80: 52 GFLOP, 650 TFLOP/s.
//
// Where little is saved, attention of each sequence by itself (kv_attention.hip) is the faster
// call for rows of the table that name their shared pages, as those of a fork do: it deals all
// of a sequence's pages to as many workgroups as the chip holds, this one its own pages to at
// most eight.  One token each, us captured, this call and that one, by sequences:
//   positions shared + own   1           4           8           16          64
//   1000 + 200               9.2, 7.2    9.3, 7.3    9.4, 7.5    9.5, 7.7    10.0, 11.8
//   1000 + 8000              11.4, 7.8   12.0, 9.5   14.7, 12.2  19.2, 17.7  55.6, 38.3
//   1000 + 30000             24.8, 10.4  31.1, 16.8  31.6, 23.6  44.6, 37.0  233, 144
//   8000 + 1000              9.4, 7.7    10.2, 9.5   11.2, 12.2  14.2, 14.4  19.8, 30.8
//   8000 + 8000              12.4, 7.9   14.6, 11.3  17.7, 13.7  19.5, 19.4  57.5, 49.6
//   30000 + 1000             12.6, 10.4  14.5, 13.5  15.8, 18.5  17.7, 27.9  32.1, 82.3
//   30000 + 8000             15.1, 11.0  17.2, 15.7  19.7, 21.3  23.0, 33.0  63.8, 100
#include "kv_attend.hpp"

namespace prichs {
namespace {

constexpr int kWaves = 4, kRowWaves = 8;

// Workgroups over shared pages, with tiles of 16 NB rows, then those over own pages.
template <int NB, bool LSE>
__global__ __launch_bounds__(64 * kWaves, NB == 1 ? 3 : 2) void kv_shared_kernel(
    const bf16_t *__restrict__ q, size_t ldq, const uint8_t *__restrict__ cache,
    const int32_t *__restrict__ table, const int32_t *__restrict__ lens,
    float *__restrict__ part_o, float2 *__restrict__ part_ml, AttendShape sh, Groups gr) {
  __shared__ JoinLds<kWaves> s;
  if ((int)blockIdx.x < shared_workgroups(sh, gr))
    kv_attend<kWaves, LSE, kSharedRole, NB>(q, ldq, cache, table, lens, nullptr, 0, nullptr,
                                            part_o, part_ml, sh, s, gr);
  else
    kv_attend<kWaves, LSE, kOwnRole>(q, ldq, cache, table, lens, nullptr, 0, nullptr, part_o,
                                     part_ml, sh, s, gr);
}
// Few pages: a workgroup for each tile of a sequence, and no second kernel.
template <bool LSE>
__global__ __launch_bounds__(64 * kRowWaves, 2) void kv_shared_rows_kernel(
    const bf16_t *__restrict__ q, size_t ldq, const uint8_t *__restrict__ cache,
    const int32_t *__restrict__ table, const int32_t *__restrict__ lens, bf16_t *__restrict__ o,
    size_t ldo, float *__restrict__ lse, AttendShape sh, Groups gr) {
  __shared__ JoinLds<kRowWaves> s;
  kv_attend<kRowWaves, LSE, kRowRole>(q, ldq, cache, table, lens, o, ldo, lse, nullptr, nullptr,
                                      sh, s, gr);
}
template <int KG, bool LSE>
__global__ __launch_bounds__(256) void kv_shared_join_kernel(
    const float *__restrict__ part_o, const float2 *__restrict__ part_ml, bf16_t *__restrict__ o,
    size_t ldo, float *__restrict__ lse, AttendShape sh, Groups gr) {
  kv_join<KG, LSE, true>(part_o, part_ml, o, ldo, lse, sh, gr);
}

// How a call is cut.  For 256 CUs whatever the current device has: a workspace's size may
// be asked for on another.  12 + 3 heads, us of a captured call (kernel and join):
//   sequences x shared positions   8 x 1000  20 x 4096  64 x 8192  256 x 8192  256 x 32768
//   tiles of 16 rows, 512            10.1      11.4       20.4        41.5        132
//   tiles of 32 rows, 256            12.3      13.5       20.2        38.2        118
//   tiles of 32 rows, 512            12.3      13.6       24.6        37.2         91
// (the second number: workgroups that the shared pages are dealt to).  24 x 8000 with six
// tokens each 26.2, 24.7, 30.5; 128 x 16384 36.3, 34.5, 38.1; 200 x 16384 52, 48, 45.
// Dealt by die (kv_attend.hpp) the last three are 24.5, 32.7 and 44.2.
// With tiles of 16 rows three workgroups fit a CU: half of that round for shared and half
// for own pages instead of 512 and 256: 16 prompts of 2048 x 4 sequences 15.4 -> 14.3, with
// some 2000 positions of their own each 23.8 -> 19.0, 32 x 8000 with 1000 each 17.1 -> 16.0, but
// 20 x 4096 11.5 -> 12.0 and 8 x 8 x 4096 16.5 -> 17.2.
// What bounds a large call is the vector instructions of a page, some 460 for 32 rows (128
// conversions, 64 permutes, the softmax), which two waves a SIMD issue 56% of the time.
// Measured and not kept, at 256 x 32768: tiles of 48 and 64 rows, one wave a SIMD, 140 and
// 166 us; each page converted once into LDS for 128 rows, whose waves wait for each other at
// every page, 95 to 101 (and 36 to 39 at 24 x 8000); queries in LDS, which leaves registers
// for a third wave, 98 to 109; own pages first 98; wave priorities, the same to 1%.  K's codes
// in products without a conversion (queries as sums of two e4m3 parts, scores of the next
// page formed between the products with V): 80.4 -> 77.8, but 64 x 8192 19.7 -> 20.4, and 24
// registers in memory where lse is wanted.
struct Plan {
  int blocks;               // of 16 rows in a tile over shared pages
  size_t tiles_p, split_p;  // tiles over shared pages of a kv head at most, splits of each
  size_t tiles_s, split_s;  // the same of a sequence's own pages
  bool rows;                // few pages: tiles_s tiles over all of a sequence's pages, one launch
};
// Up to so many pages, and a CU for each tile of a sequence, one launch takes each sequence by
// itself.  Captured, us (from Python in brackets), so and apart with a join, in turn: 8 sequences
// of 8 pages 6.4, 8.7 (10.7, 14.5), 16 pages 8.1, 8.9 (10.6, 14.4), 20 pages 9.6, 9.3, 24 pages 9.6,
// 9.4 (10.7, 14.5), 32 pages 11.2, 9.4 (11.4, 14.5); one of 16 pages 7.8, 8.2, of 24 9.5, 8.6; 80 of
// 24 10.5, 14.4; 20 of 24 with eight tokens each 10.2, 14.7.  So a few sequences of 20 to 24 pages
// lose up to 0.9 us in a graph; the bound is where calls from Python, which gain 4, still do, and
// batches do either way.  100 sequences, more tiles than CUs, in graphs of ten calls: 8 pages
// 11.8, 10.7 (11.3, 14.9), 24 pages 18.6, 13.7.
constexpr size_t kFewPages = 24;
constexpr size_t kHalfRound = 384;
constexpr size_t kManySteps = 4096, kMoreSteps = 32768;  // pages of all tiles of 16 rows
// `pages`: that a sequence's tile sees at most.
Plan plan_of(size_t batch, size_t n_q, size_t n_heads, size_t n_kv_heads, size_t max_pages,
             size_t n_groups, size_t pages) {
  const size_t rows = n_q * (n_heads / n_kv_heads);  // of a sequence
  const size_t most = std::max<size_t>(cdiv(max_pages, (size_t)kWaves), 1);
  // Only groups of some sequence have tiles, and the last of each may be short.
  const size_t groups = std::min(n_groups, batch);
  const size_t steps = cdiv(batch * rows, (size_t)kRows) * n_kv_heads * max_pages;
  Plan p;
  p.blocks = batch * rows >= 2 * kRows * groups && steps >= kManySteps ? 2 : 1;
  const size_t per = (size_t)kRows * p.blocks;
  p.tiles_p = p.split_p = 0;
  if (groups > 0) {
    p.tiles_p = (batch * rows + groups * (per - 1)) / per;
    const size_t wgs = p.blocks == 1 ? kHalfRound : steps >= kMoreSteps ? 512 : 256;
    p.split_p = std::max<size_t>(std::min(wgs / (n_kv_heads * p.tiles_p), most), 1);
  }
  // Own pages: as a rule few, of a number that only the device knows.
  p.tiles_s = cdiv(rows, (size_t)kRows);
  p.rows = pages <= kFewPages && batch * n_kv_heads * p.tiles_s <= 256;
  const size_t own = p.blocks == 1 ? kHalfRound : 256;
  p.split_s = std::max<size_t>(
      std::min({own / (batch * n_kv_heads * p.tiles_s), most, (size_t)8}), 1);
  return p;
}
size_t workspace_of(const Plan &p, size_t rows) {
  if (p.rows) return 0;
  return rows * (p.split_p + p.split_s) * (kKvHd + 3) * sizeof(float);
}

}  // namespace
}  // namespace prichs

using namespace prichs;

extern "C" size_t prichs_kv_cache_shared_attention_workspace(size_t batch, size_t n_q,
                                                             size_t n_heads, size_t n_kv_heads,
                                                             size_t max_pages, size_t n_groups) {
  if (n_kv_heads == 0 || n_heads < n_kv_heads || batch == 0 || n_q == 0) return 0;
  return workspace_of(plan_of(batch, n_q, n_heads, n_kv_heads, max_pages, n_groups, max_pages),
                      batch * n_q * n_heads);
}

extern "C" int prichs_kv_cache_shared_attention(
    const void *q, size_t ldq, const void *cache, size_t n_pages, const int32_t *page_table,
    size_t max_pages, const int32_t *lens, const int32_t *group_start, const int32_t *shared,
    size_t n_groups, void *o, size_t ldo, float *lse, size_t batch, size_t n_q, size_t n_heads,
    size_t n_kv_heads, size_t head_dim, size_t window, size_t sinks, int dtype, void *workspace,
    size_t workspace_bytes, void *stream) {
  const char *who = "kv_cache_shared_attention";
  PRICHS_REQUIRE(dtype == PRICHS_DTYPE_BF16, "%s: only bf16 is supported (dtype=%d)", who, dtype);
  if (head_dim != (size_t)kKvHd)
    return fail(PRICHS_ERR_UNSUPPORTED, "%s: head_dim=%zu (only %d is supported)", who, head_dim,
                kKvHd);
  PRICHS_REQUIRE(n_heads >= 1 && n_kv_heads >= 1 && n_heads % n_kv_heads == 0,
                 "%s: n_heads=%zu must be a positive multiple of n_kv_heads=%zu", who, n_heads,
                 n_kv_heads);
  PRICHS_REQUIRE(n_heads <= 65535 && batch <= 65535 && n_q <= (size_t)1 << 21 &&
                     n_groups <= 65535 && n_pages <= (size_t)INT32_MAX &&
                     max_pages <= ((size_t)1 << 30) / kKvPage &&
                     batch * n_q * n_heads <= (size_t)1 << 26,
                 "%s: shape too large", who);
  PRICHS_REQUIRE(ldq >= n_heads * head_dim && ldo >= n_heads * head_dim && ldq % 8 == 0 &&
                     ldo % 8 == 0,
                 "%s: ldq and ldo must be multiples of 8 elements that hold all heads", who);
  if (batch == 0 || n_q == 0) return PRICHS_OK;
  const size_t cap = max_pages * kKvPage;
  PRICHS_REQUIRE(q && o && lens && (cap == 0 || page_table) && (n_pages == 0 || cache) &&
                     (n_groups == 0 || (group_start && shared)),
                 "%s: null pointer argument", who);
  PRICHS_REQUIRE((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(o) |
                  reinterpret_cast<uintptr_t>(cache)) % 16 == 0,
                 "%s: q, o and the cache must be 16-byte aligned", who);
  // A window past the table hides nothing.
  const size_t w = window >= cap ? 0 : window, sk = std::min(sinks, cap);
  const size_t pages =
      w == 0 ? max_pages : std::min(max_pages, cdiv(w + n_q, kKvPage) + 1 + cdiv(sk, kKvPage));
  const Plan p = plan_of(batch, n_q, n_heads, n_kv_heads, max_pages, n_groups, pages);
  // Workgroups of 256 threads, fewer than 2^32 in a launch.
  const size_t wgs = roundup(n_kv_heads * p.tiles_p * p.split_p, 8) +
                     n_kv_heads * batch * p.tiles_s * p.split_s;
  PRICHS_REQUIRE(wgs < (size_t)1 << 24, "%s: shape too large", who);
  const size_t rows = batch * n_q * n_heads, need = workspace_of(p, rows);
  if (workspace_bytes < need)
    return fail(PRICHS_ERR_CAPACITY, "%s: workspace of %zu bytes, %zu needed", who,
                workspace_bytes, need);
  PRICHS_REQUIRE(need == 0 ||
                     (workspace != nullptr && reinterpret_cast<uintptr_t>(workspace) % 16 == 0),
                 "%s: the workspace must be 16-byte aligned device memory", who);
  const AttendShape sh{(int)n_pages,
                       (int)max_pages,
                       (int)n_q,
                       (int)n_heads,
                       (int)n_kv_heads,
                       (int)w,
                       (int)sk,
                       (int)p.tiles_s,
                       1,
                       (1.0f / sqrtf((float)head_dim)) * 1.4426950408889634f};
  const Groups gr{group_start,    shared,         (int)n_groups, (int)batch,
                  (int)p.tiles_p, (int)p.split_p, (int)p.split_s};
  if (p.rows) {
    hipLaunchKernelGGL(lse == nullptr ? kv_shared_rows_kernel<false> : kv_shared_rows_kernel<true>,
                       dim3((unsigned)(n_kv_heads * p.tiles_s), 1, (unsigned)batch),
                       dim3(64 * kRowWaves), 0, as_stream(stream), static_cast<const bf16_t *>(q),
                       ldq, static_cast<const uint8_t *>(cache), page_table, lens,
                       static_cast<bf16_t *>(o), ldo, lse, sh, gr);
    PRICHS_LAUNCH_CHECK("kv_cache_shared_attention launch");
    return PRICHS_OK;
  }
  float *part_o = static_cast<float *>(workspace);
  float2 *part_ml =
      reinterpret_cast<float2 *>(part_o + rows * (p.split_p + p.split_s) * kKvHd);
  const hipStream_t s = as_stream(stream);
  auto kern = p.blocks == 2
                  ? (lse == nullptr ? kv_shared_kernel<2, false> : kv_shared_kernel<2, true>)
                  : (lse == nullptr ? kv_shared_kernel<1, false> : kv_shared_kernel<1, true>);
  hipLaunchKernelGGL(kern, dim3((unsigned)wgs), dim3(64 * kWaves), 0, s,
                     static_cast<const bf16_t *>(q), ldq, static_cast<const uint8_t *>(cache),
                     page_table, lens, part_o, part_ml, sh, gr);
  PRICHS_LAUNCH_CHECK("kv_cache_shared_attention launch");
  // Eight groups of threads a row where it has more parts than one can load at once.
  const bool wide = p.split_p + p.split_s > 8;
  auto join = lse == nullptr
                  ? (wide ? kv_shared_join_kernel<8, false> : kv_shared_join_kernel<1, false>)
                  : (wide ? kv_shared_join_kernel<8, true> : kv_shared_join_kernel<1, true>);
  hipLaunchKernelGGL(join, dim3((unsigned)(wide ? rows : cdiv(rows, 8))), dim3(256), 0, s, part_o,
                     part_ml, static_cast<bf16_t *>(o), ldo, lse, sh, gr);
  PRICHS_LAUNCH_CHECK("kv_cache_shared_attention join launch");
  return PRICHS_OK;
}
