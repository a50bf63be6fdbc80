// kv_attention.hip -- GQA attention of a sequence's last tokens over its paged
// 4-bit KV cache (kv_cache.hpp has the layout and the number format).
#include "kv_cache.hpp"

namespace prichs {
namespace {

struct AttendShape {
  int n_pages, max_pages, n_q, Hq, Hkv, window, sinks;
  float scale;
};

// One wave per (query row, query head), the lane holding dims 2 lane, 2 lane + 1.
__global__ __launch_bounds__(64) void kv_attend_row_kernel(
    const bf16_t *q, size_t ldq, const uint8_t *cache, const int32_t *table, const int32_t *lens,
    bf16_t *o, size_t ldo, float *lse, AttendShape sh) {
  const int lane = threadIdx.x, h = blockIdx.y;
  const int b = blockIdx.x / sh.n_q, iq = blockIdx.x - b * sh.n_q;
  const int kvh = h / (sh.Hq / sh.Hkv);
  const int L = min(max(lens[b], 0), sh.max_pages * kKvPage);
  const int i = L - sh.n_q + iq;
  const size_t c = (size_t)h * kKvHd + 2 * lane;
  const float q0 = bf16_to_f32(q[(size_t)blockIdx.x * ldq + c]),
              q1 = bf16_to_f32(q[(size_t)blockIdx.x * ldq + c + 1]);
  const int lo = sh.window == 0 ? 0 : max(0, i - sh.window + 1);
  float m = -INFINITY, l = 0.f, a0 = 0.f, a1 = 0.f;
  bool any = false;
  for (int j = 0; j <= i; ++j) {
    if (j >= min(sh.sinks, lo) && j < lo) j = lo;
    const int page = table[(size_t)b * sh.max_pages + j / kKvPage];
    if (page < 0 || page >= sh.n_pages) continue;
    any = true;
    const uint8_t *part = cache + ((size_t)page * sh.Hkv + kvh) * kKvPart;
    const int t = j % kKvPage;
    const float ks = kv_scale(part[kKvKScale + 4 * t + lane / 16]),
                vs = kv_scale(part[kKvVScale + 4 * t + lane / 16]);
    const auto kk = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(
        part[kKvK + t * (kKvHd / 2) + lane], 1.0f, 0);
    const auto vv = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(
        part[kv_v_off(t, lane >> 2) + (lane & 3)], 1.0f, 0);
    float s = q0 * (kk[0] * ks) + q1 * (kk[1] * ks);
    for (int x = 1; x < 64; x <<= 1) s += __shfl_xor(s, x);
    s *= sh.scale;
    const float m2 = __builtin_elementwise_maximum(m, s);
    const float r = m2 == m ? 1.f : expf(m - m2), p = m2 == -INFINITY ? 0.f : expf(s - m2);
    l = l * r + p;
    a0 = a0 * r + p * (vv[0] * vs);
    a1 = a1 * r + p * (vv[1] * vs);
    m = m2;
  }
  *reinterpret_cast<uint32_t *>(o + (size_t)blockIdx.x * ldo + c) =
      any ? pack_bf16x2(a0 / l, a1 / l) : 0u;
  if (lse != nullptr && lane == 0)
    lse[((size_t)b * sh.Hq + h) * sh.n_q + iq] = any ? m + logf(l) : -INFINITY;
}

}  // namespace
}  // namespace prichs

using namespace prichs;

extern "C" size_t prichs_kv_cache_attention_workspace(size_t batch, size_t n_q, size_t n_heads,
                                                      size_t n_kv_heads, size_t max_pages) {
  (void)batch, (void)n_q, (void)n_heads, (void)n_kv_heads, (void)max_pages;
  return 0;
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
  PRICHS_REQUIRE(ldq >= n_heads * head_dim && ldo >= n_heads * head_dim && ldq % 8 == 0 &&
                     ldo % 8 == 0,
                 "%s: ldq and ldo must be multiples of 8 elements that hold all heads", who);
  const size_t cap = max_pages * kKvPage;
  PRICHS_REQUIRE(n_heads <= 65535 && batch <= 65535 && n_q <= (size_t)1 << 21 &&
                     batch * n_q <= (size_t)INT32_MAX / 2 && n_pages <= (size_t)INT32_MAX &&
                     max_pages <= ((size_t)1 << 30) / kKvPage,
                 "%s: shape too large", who);
  if (batch == 0 || n_q == 0) return PRICHS_OK;
  PRICHS_REQUIRE(q && o && lens && (cap == 0 || (cache && page_table)),
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
  const AttendShape sh{(int)n_pages,
                       (int)max_pages,
                       (int)n_q,
                       (int)n_heads,
                       (int)n_kv_heads,
                       (int)(window >= cap ? 0 : window),
                       (int)(sinks < cap ? sinks : cap),
                       1.0f / sqrtf((float)head_dim)};
  hipLaunchKernelGGL(kv_attend_row_kernel, dim3((unsigned)(batch * n_q), (unsigned)n_heads),
                     dim3(64), 0, as_stream(stream), static_cast<const bf16_t *>(q), ldq,
                     static_cast<const uint8_t *>(cache), page_table, lens,
                     static_cast<bf16_t *>(o), ldo, lse, sh);
  PRICHS_LAUNCH_CHECK("kv_cache_attention launch");
  return PRICHS_OK;
}
