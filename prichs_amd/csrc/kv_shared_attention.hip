// kv_shared_attention.hip -- attention of each sequence's last tokens over the paged 4-bit
// KV cache where groups of sequences share their first pages: the shared pages are read
// and multiplied once for all rows of a group, each sequence's own pages once for its
// rows, and the parts are joined.  With o_p, m_p, l_p the sums, maximum and sum of
// exponentials over part p of the keys,
//   o = sum_p exp(m_p - m) o_p / sum_p exp(m_p - m) l_p,  m = max_p m_p.
// kv_attend.hpp has the tiles and the join.
#include "kv_attend.hpp"

namespace prichs {
namespace {

constexpr int kPartWaves = 4;

template <bool LSE>
__global__ __launch_bounds__(64 * kPartWaves, 3) void kv_shared_kernel(
    const bf16_t *__restrict__ q, size_t ldq, const uint8_t *__restrict__ cache,
    const int32_t *__restrict__ table, const int32_t *__restrict__ lens,
    float *__restrict__ part_o, float2 *__restrict__ part_ml, AttendShape sh, Groups gr) {
  kv_attend<kPartWaves, LSE, Groups>(q, ldq, cache, table, lens, nullptr, 0, nullptr, part_o,
                                     part_ml, sh, gr);
}
template <int KG, bool LSE>
__global__ __launch_bounds__(256) void kv_shared_join_kernel(
    const float *__restrict__ part_o, const float2 *__restrict__ part_ml, bf16_t *__restrict__ o,
    size_t ldo, float *__restrict__ lse, AttendShape sh, Groups gr) {
  kv_join<KG, LSE, Groups>(part_o, part_ml, o, ldo, lse, sh, gr);
}

// How a call is cut.  For 256 CUs whatever the current device has: a workspace's size may
// be asked for on another.
struct Plan {
  size_t tiles_p, split_p;  // tiles over shared pages of a kv head at most, splits of each
  size_t tiles_s, split_s;  // the same of a sequence's own pages
};
Plan plan_of(size_t batch, size_t n_q, size_t n_heads, size_t n_kv_heads, size_t max_pages,
             size_t n_groups) {
  const size_t rows = n_q * (n_heads / n_kv_heads);  // of a sequence
  const size_t most = std::max<size_t>(cdiv(max_pages, 4), 1);
  Plan p;
  // The last tile of each group may be short; only groups of some sequence have tiles.
  p.tiles_p = n_groups == 0
                  ? 0
                  : (batch * rows + std::min(n_groups, batch) * (kRows - 1)) / kRows;
  p.split_p = n_groups == 0
                  ? 0
                  : std::max<size_t>(std::min(768 / (n_kv_heads * p.tiles_p), most), 1);
  p.tiles_s = cdiv(rows, (size_t)kRows);
  p.split_s =
      std::max<size_t>(std::min(768 / (batch * n_kv_heads * p.tiles_s), std::min<size_t>(most, 8)), 1);
  return p;
}
size_t workspace_of(const Plan &p, size_t rows) {
  return rows * (p.split_p + p.split_s) * (kKvHd + 3) * sizeof(float);
}

}  // namespace
}  // namespace prichs

using namespace prichs;

extern "C" size_t prichs_kv_cache_shared_attention_workspace(size_t batch, size_t n_q,
                                                             size_t n_heads, size_t n_kv_heads,
                                                             size_t max_pages, size_t n_groups) {
  if (n_kv_heads == 0 || n_heads < n_kv_heads || batch == 0 || n_q == 0) return 0;
  return workspace_of(plan_of(batch, n_q, n_heads, n_kv_heads, max_pages, n_groups),
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
  const Plan p = plan_of(batch, n_q, n_heads, n_kv_heads, max_pages, n_groups);
  // Workgroups of 256 threads, fewer than 2^32 in a launch.
  const size_t wgs = n_kv_heads * (p.tiles_p * p.split_p + batch * p.tiles_s * p.split_s);
  PRICHS_REQUIRE(wgs < (size_t)1 << 24, "%s: shape too large", who);
  const size_t rows = batch * n_q * n_heads, need = workspace_of(p, rows);
  if (workspace_bytes < need)
    return fail(PRICHS_ERR_CAPACITY, "%s: workspace of %zu bytes, %zu needed", who,
                workspace_bytes, need);
  PRICHS_REQUIRE(workspace != nullptr && reinterpret_cast<uintptr_t>(workspace) % 16 == 0,
                 "%s: the workspace must be 16-byte aligned device memory", who);
  // A window past the table hides nothing.
  const AttendShape sh{(int)n_pages,
                       (int)max_pages,
                       (int)n_q,
                       (int)n_heads,
                       (int)n_kv_heads,
                       (int)(window >= cap ? 0 : window),
                       (int)std::min(sinks, cap),
                       (int)p.tiles_s,
                       1,
                       (1.0f / sqrtf((float)head_dim)) * 1.4426950408889634f};
  const Groups gr{group_start,    shared,          (int)n_groups,  (int)batch,
                  (int)p.tiles_p, (int)p.split_p, (int)p.split_s};
  float *part_o = static_cast<float *>(workspace);
  float2 *part_ml =
      reinterpret_cast<float2 *>(part_o + rows * (p.split_p + p.split_s) * kKvHd);
  const hipStream_t s = as_stream(stream);
  const dim3 grid((unsigned)wgs);
  auto kern = lse == nullptr ? kv_shared_kernel<false> : kv_shared_kernel<true>;
  hipLaunchKernelGGL(kern, grid, dim3(64 * kPartWaves), 0, s, static_cast<const bf16_t *>(q), ldq,
                     static_cast<const uint8_t *>(cache), page_table, lens, part_o, part_ml, sh,
                     gr);
  PRICHS_LAUNCH_CHECK("kv_cache_shared_attention launch");
  const bool wide = p.split_p + p.split_s > 8;
  auto join = lse == nullptr
                  ? (wide ? kv_shared_join_kernel<8, false> : kv_shared_join_kernel<1, false>)
                  : (wide ? kv_shared_join_kernel<8, true> : kv_shared_join_kernel<1, true>);
  hipLaunchKernelGGL(join, dim3((unsigned)(wide ? rows : cdiv(rows, 8))), dim3(256), 0, s, part_o,
                     part_ml, static_cast<bf16_t *>(o), ldo, lse, sh, gr);
  PRICHS_LAUNCH_CHECK("kv_cache_shared_attention join launch");
  return PRICHS_OK;
}
