// kv_attention.hip -- GQA attention of a sequence's last tokens over its paged
// 4-bit KV cache (kv_cache.hpp has the layout and the number format).
// kv_attend.hpp has the tiles and the join; here is how a call is cut into them.
#include "kv_attend.hpp"

namespace prichs {
namespace {

template <int kWaves>
__global__ __launch_bounds__(64 * kWaves, kWaves == 4 ? 3 : 2) void kv_attend_kernel(
    const bf16_t *__restrict__ q, size_t ldq, const uint8_t *__restrict__ cache,
    const int32_t *__restrict__ table, const int32_t *__restrict__ lens, bf16_t *__restrict__ o,
    size_t ldo, float *__restrict__ lse, float *__restrict__ part_o, float2 *__restrict__ part_ml,
    AttendShape sh) {
  __shared__ JoinLds<kWaves> s;
  kv_attend<kWaves, false>(q, ldq, cache, table, lens, o, ldo, lse, part_o, part_ml, sh, s, Groups{});
}
// With lse: up to 0.8 us a call (one token over 8192 positions 8.2 -> 8.8 us, 32 x 3000 15.5
// -> 15.9, 8 x 5 over 4096 13.8 -> 14.6, 2 x 256 over 4352 34.6 -> 35.1).
template <int kWaves>
__global__ __launch_bounds__(64 * kWaves, kWaves == 4 ? 3 : 2) void kv_attend_lse_kernel(
    const bf16_t *__restrict__ q, size_t ldq, const uint8_t *__restrict__ cache,
    const int32_t *__restrict__ table, const int32_t *__restrict__ lens, bf16_t *__restrict__ o,
    size_t ldo, float *__restrict__ lse, float *__restrict__ part_o, float2 *__restrict__ part_ml,
    AttendShape sh) {
  __shared__ JoinLds<kWaves> s;
  kv_attend<kWaves, true>(q, ldq, cache, table, lens, o, ldo, lse, part_o, part_ml, sh, s, Groups{});
}

template <int KG>
__global__ __launch_bounds__(256) void kv_join_kernel(
    const float *__restrict__ part_o, const float2 *__restrict__ part_ml, bf16_t *__restrict__ o,
    size_t ldo, float *__restrict__ lse, AttendShape sh) {
  kv_join<KG, false>(part_o, part_ml, o, ldo, lse, sh, Groups{});
}
template <int KG>
__global__ __launch_bounds__(256) void kv_join_lse_kernel(
    const float *__restrict__ part_o, const float2 *__restrict__ part_ml, bf16_t *__restrict__ o,
    size_t ldo, float *__restrict__ lse, AttendShape sh) {
  kv_join<KG, true>(part_o, part_ml, o, ldo, lse, sh, Groups{});
}

// Pages up to which one workgroup of 8 waves takes a tile without a second kernel:
// a page costs a wave some 2 us, the second kernel 2.5 on the device and 4 on the
// host.  Captured, us (from Python in brackets), one kernel and two, in turn: one token over
// 8 pages 5.7, 6.7 (9.6, 13.3), over 16 pages 7.3, 6.7 (9.6, 13.4), over 32 pages 10.5, 7.0
// (10.6, 13.5); 32 and 80 sequences over 8 pages 5.9, 7.0 and 6.1, 8.4, over 16 pages 7.6,
// 8.4 and 8.6, 12.9, over 32 pages 11.6, 10.4 and 14.9, 18.9.
constexpr size_t kShortPages = 16;

// How a call is cut: n_split workgroups of `waves` waves over a tile's pages.  For 256
// CUs whatever the current device has: a workspace's size may be asked for on another.
struct Plan {
  int waves;
  size_t tiles, n_split;
};
Plan plan_of(size_t batch, size_t n_q, size_t n_heads, size_t n_kv_heads, size_t pages) {
  const size_t rows = n_q * (n_heads / n_kv_heads);
  Plan p;
  p.waves = 4;
  p.tiles = cdiv(rows, (size_t)kRows);
  const size_t wgs = std::max<size_t>(batch * n_kv_heads * p.tiles, 1);
  // Few pages and a CU for every tile: one workgroup of 8 waves a tile, and no
  // second kernel.
  if (pages > 4 && pages <= kShortPages && wgs <= 256) {
    p.waves = 8;
    p.n_split = 1;
    return p;
  }
  // As many workgroups as fit the chip at once (three a CU), and a page for each
  // wave of a workgroup.
  p.n_split = std::max<size_t>(std::min(768 / wgs, cdiv(pages, 4)), 1);
  return p;
}
size_t workspace_of(const Plan &p, size_t batch, size_t n_kv_heads) {
  if (p.n_split <= 1) return 0;
  return batch * n_kv_heads * p.tiles * p.n_split * kRows * (kKvHd + 3) * sizeof(float);
}

}  // namespace
}  // namespace prichs

using namespace prichs;

extern "C" size_t prichs_kv_cache_attention_workspace(size_t batch, size_t n_q, size_t n_heads,
                                                      size_t n_kv_heads, size_t max_pages) {
  if (n_kv_heads == 0 || n_heads < n_kv_heads || batch == 0 || n_q == 0) return 0;
  return workspace_of(plan_of(batch, n_q, n_heads, n_kv_heads, max_pages), batch, n_kv_heads);
}

extern "C" int prichs_kv_cache_attention(const void *q, size_t ldq, const void *cache,
                                         size_t n_pages, const int32_t *page_table,
                                         size_t max_pages, const int32_t *lens, void *o,
                                         size_t ldo, float *lse, size_t batch, size_t n_q,
                                         size_t n_heads, size_t n_kv_heads, size_t head_dim,
                                         size_t window, size_t sinks, int dtype, void *workspace,
                                         size_t workspace_bytes, void *stream) {
  const char *who = "kv_cache_attention";
  PRICHS_REQUIRE(dtype == PRICHS_DTYPE_BF16, "%s: only bf16 is supported (dtype=%d)", who, dtype);
  if (head_dim != (size_t)kKvHd)
    return fail(PRICHS_ERR_UNSUPPORTED, "%s: head_dim=%zu (only %d is supported)", who, head_dim,
                kKvHd);
  PRICHS_REQUIRE(n_heads >= 1 && n_kv_heads >= 1 && n_heads % n_kv_heads == 0,
                 "%s: n_heads=%zu must be a positive multiple of n_kv_heads=%zu", who, n_heads,
                 n_kv_heads);
  PRICHS_REQUIRE(n_heads <= 65535 && batch <= 65535 && n_q <= (size_t)1 << 21 &&
                     batch * n_q <= (size_t)INT32_MAX / 2 && n_pages <= (size_t)INT32_MAX &&
                     max_pages <= ((size_t)1 << 30) / kKvPage,
                 "%s: shape too large", who);
  PRICHS_REQUIRE(ldq >= n_heads * head_dim && ldo >= n_heads * head_dim && ldq % 8 == 0 &&
                     ldo % 8 == 0,
                 "%s: ldq and ldo must be multiples of 8 elements that hold all heads", who);
  const size_t cap = max_pages * kKvPage;
  if (batch == 0 || n_q == 0) return PRICHS_OK;
  PRICHS_REQUIRE(q && o && lens && (cap == 0 || page_table) && (n_pages == 0 || cache),
                 "%s: null pointer argument", who);
  PRICHS_REQUIRE((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(o) |
                  reinterpret_cast<uintptr_t>(cache)) % 16 == 0,
                 "%s: q, o and the cache must be 16-byte aligned", who);
  const size_t need =
      prichs_kv_cache_attention_workspace(batch, n_q, n_heads, n_kv_heads, max_pages);
  if (workspace_bytes < need)
    return fail(PRICHS_ERR_CAPACITY, "%s: workspace of %zu bytes, %zu needed", who,
                workspace_bytes, need);
  PRICHS_REQUIRE(need == 0 ||
                     (workspace != nullptr && reinterpret_cast<uintptr_t>(workspace) % 16 == 0),
                 "%s: the workspace must be 16-byte aligned device memory", who);
  // Pages that a tile can see at most: those of the window and of the sinks (a
  // window past the table hides nothing).
  const size_t w = window >= cap ? 0 : window, sk = std::min(sinks, cap);
  const size_t pages =
      w == 0 ? max_pages
             : std::min(max_pages, cdiv(w + n_q, kKvPage) + 1 + cdiv(sk, kKvPage));
  const Plan p = plan_of(batch, n_q, n_heads, n_kv_heads, pages);
  PRICHS_REQUIRE(n_kv_heads * p.tiles <= (size_t)1 << 23, "%s: shape too large", who);
  const AttendShape sh{(int)n_pages,
                       (int)max_pages,
                       (int)n_q,
                       (int)n_heads,
                       (int)n_kv_heads,
                       (int)w,
                       (int)sk,
                       (int)p.tiles,
                       (int)p.n_split,
                       (1.0f / sqrtf((float)head_dim)) * 1.4426950408889634f};
  const size_t part_rows = batch * n_kv_heads * p.tiles * p.n_split * kRows;
  float *part_o = static_cast<float *>(workspace);
  float2 *part_ml = reinterpret_cast<float2 *>(part_o + (p.n_split > 1 ? part_rows * kKvHd : 0));
  const dim3 grid((unsigned)(n_kv_heads * p.tiles), (unsigned)p.n_split, (unsigned)batch);
  auto kern = lse == nullptr ? (p.waves == 8 ? kv_attend_kernel<8> : kv_attend_kernel<4>)
                             : (p.waves == 8 ? kv_attend_lse_kernel<8> : kv_attend_lse_kernel<4>);
  hipLaunchKernelGGL(kern, grid, dim3((unsigned)(64 * p.waves)), 0, as_stream(stream),
                     static_cast<const bf16_t *>(q), ldq, static_cast<const uint8_t *>(cache),
                     page_table, lens, static_cast<bf16_t *>(o), ldo, lse, part_o, part_ml, sh);
  PRICHS_LAUNCH_CHECK("kv_cache_attention launch");
  if (p.n_split > 1) {
    const size_t rows = n_q * (n_heads / n_kv_heads);
    // Eight threads groups a row where a row has more splits than one can load at
    // once.
    const bool wide = p.n_split > 8;
    const dim3 join((unsigned)(wide ? rows : cdiv(rows, 8)), (unsigned)n_kv_heads,
                    (unsigned)batch);
    auto join_kern = lse == nullptr ? (wide ? kv_join_kernel<8> : kv_join_kernel<1>)
                                    : (wide ? kv_join_lse_kernel<8> : kv_join_lse_kernel<1>);
    hipLaunchKernelGGL(join_kern, join, dim3(256), 0, as_stream(stream), part_o, part_ml,
                       static_cast<bf16_t *>(o), ldo, lse, sh);
    PRICHS_LAUNCH_CHECK("kv_cache_attention join launch");
  }
  return PRICHS_OK;
}
