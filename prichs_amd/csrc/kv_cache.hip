// kv_cache.hip -- tokens quantised into the paged 4-bit KV cache, and read
// back.  kv_cache.hpp has the layout and the number format.
#include "kv_cache.hpp"

namespace prichs {
namespace {

// Page of position pos of sequence b, or -1 where the table has none.
__device__ __forceinline__ int page_of(const int32_t *table, int max_pages, int n_pages, int b,
                                       long long pos) {
  if (pos < 0 || pos >= (long long)max_pages * kKvPage) return -1;
  const int p = table[(long long)b * max_pages + (int)(pos / kKvPage)];
  return p >= 0 && p < n_pages ? p : -1;
}

// One 64-thread workgroup per (row, kv head): lanes 0..31 quantise k, lanes
// 32..63 v; a lane holds 4 values, 8 lanes a group of 32.
template <typename T>
__global__ __launch_bounds__(64) void kv_write_kernel(
    const T *__restrict__ k, size_t ldk, const T *__restrict__ v, size_t ldv, uint8_t *cache,
    int n_pages, const int32_t *table, int max_pages, const int32_t *start, const int32_t *counts,
    int n, int kv_heads) {
  const int row = blockIdx.x, h = blockIdx.y, lane = threadIdx.x;
  const int b = row / n, i = row - b * n;
  if (counts != nullptr && i >= counts[b]) return;
  const long long pos = (long long)start[b] + i;
  const int page = page_of(table, max_pages, n_pages, b, pos);
  if (page < 0) return;
  const bool is_v = lane >= 32;
  const int c = lane & 31;
  const T *src = (is_v ? v + (size_t)row * ldv : k + (size_t)row * ldk) + (size_t)h * kKvHd + 4 * c;
  float x[4];
  uint32_t amax = 0;
  for (int e = 0; e < 4; ++e) {
    x[e] = Elem<T>::load(src + e);
    amax = max(amax, __float_as_uint(x[e]) & 0x7fffffffu);
  }
  for (int m = 1; m < 8; m <<= 1) amax = max(amax, (uint32_t)__shfl_xor((int)amax, m));
  const uint32_t s = kv_scale_byte(amax);
  uint32_t code = 0;
  if (s != 255) {
    const float sc = kv_scale(s);
    code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, x[0], x[1], sc, 0);
    code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, x[2], x[3], sc, 1);
  }
  uint8_t *part = cache + ((size_t)page * kv_heads + h) * kKvPart;
  const int t = (int)(pos % kKvPage);
  const int off = is_v ? kv_v_off(t, c >> 1) + 2 * (c & 1) : kKvK + t * (kKvHd / 2) + 2 * c;
  *reinterpret_cast<uint16_t *>(part + off) = (uint16_t)code;
  if ((c & 7) == 0) part[(is_v ? kKvVScale : kKvKScale) + 4 * t + (c >> 3)] = (uint8_t)s;
}

template <typename T>
__global__ __launch_bounds__(64) void kv_read_kernel(
    T *__restrict__ k, size_t ldk, T *__restrict__ v, size_t ldv, const uint8_t *cache,
    int n_pages, const int32_t *table, int max_pages, const int32_t *start, const int32_t *counts,
    int n, int kv_heads) {
  const int row = blockIdx.x, h = blockIdx.y, lane = threadIdx.x;
  const int b = row / n, i = row - b * n;
  if (counts != nullptr && i >= counts[b]) return;
  const long long pos = (long long)start[b] + i;
  const int page = page_of(table, max_pages, n_pages, b, pos);
  const bool is_v = lane >= 32;
  const int c = lane & 31;
  uint32_t code = 0, s = 127;
  if (page >= 0) {
    const uint8_t *part = cache + ((size_t)page * kv_heads + h) * kKvPart;
    const int t = (int)(pos % kKvPage);
    const int off = is_v ? kv_v_off(t, c >> 1) + 2 * (c & 1) : kKvK + t * (kKvHd / 2) + 2 * c;
    code = *reinterpret_cast<const uint16_t *>(part + off);
    s = part[(is_v ? kKvVScale : kKvKScale) + 4 * t + (c >> 3)];
  }
  const float sc = kv_scale(s);
  const auto lo = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code, sc, 0);
  const auto hi = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code, sc, 1);
  T *dst = (is_v ? v + (size_t)row * ldv : k + (size_t)row * ldk) + (size_t)h * kKvHd + 4 * c;
  const float x[4] = {lo[0], lo[1], hi[0], hi[1]};
  for (int e = 0; e < 4; ++e) Elem<T>::store(dst + e, s == 255 ? sc : x[e]);
}

// Checks shared by the write and the read entry point; PRICHS_OK with *work =
// false where there is nothing to do.
int kv_check(const char *who, const void *k, size_t ldk, const void *v, size_t ldv,
             const void *cache, size_t n_pages, const int32_t *page_table, size_t max_pages,
             const int32_t *start, size_t batch, size_t n, size_t n_kv_heads, size_t head_dim,
             int dtype, bool *work) {
  *work = false;
  PRICHS_REQUIRE(dtype_ok(dtype), "%s: bad dtype %d", who, dtype);
  if (head_dim != (size_t)kKvHd)
    return fail(PRICHS_ERR_UNSUPPORTED, "%s: head_dim=%zu (only %d is supported)", who, head_dim,
                kKvHd);
  PRICHS_REQUIRE(n_kv_heads >= 1 && n_kv_heads <= 65535, "%s: n_kv_heads=%zu", who, n_kv_heads);
  PRICHS_REQUIRE(ldk >= n_kv_heads * head_dim && ldv >= n_kv_heads * head_dim,
                 "%s: leading dimensions too small", who);
  PRICHS_REQUIRE(ldk % 8 == 0 && ldv % 8 == 0,
                 "%s: leading dimensions must be multiples of 8 elements", who);
  PRICHS_REQUIRE(batch <= (size_t)INT32_MAX && n <= (size_t)INT32_MAX &&
                     (n == 0 || batch <= (size_t)INT32_MAX / n) && n_pages <= (size_t)INT32_MAX &&
                     max_pages <= (size_t)INT32_MAX / kKvPage,
                 "%s: shape too large", who);
  if (batch == 0 || n == 0) return PRICHS_OK;
  PRICHS_REQUIRE(k && v && cache && page_table && start, "%s: null pointer argument", who);
  const uintptr_t al = reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) |
                       reinterpret_cast<uintptr_t>(cache);
  PRICHS_REQUIRE(al % 16 == 0, "%s: k, v and the cache must be 16-byte aligned", who);
  *work = true;
  return PRICHS_OK;
}

}  // namespace
}  // namespace prichs

using namespace prichs;

extern "C" int prichs_kv_cache_write(void *cache, size_t n_pages, const int32_t *page_table,
                                     size_t max_pages, const int32_t *start,
                                     const int32_t *counts, const void *k, size_t ldk,
                                     const void *v, size_t ldv, size_t batch, size_t n,
                                     size_t n_kv_heads, size_t head_dim, int dtype,
                                     void *stream) {
  bool work;
  const int rc = kv_check("kv_cache_write", k, ldk, v, ldv, cache, n_pages, page_table, max_pages,
                          start, batch, n, n_kv_heads, head_dim, dtype, &work);
  if (rc != PRICHS_OK || !work) return rc;
  const dim3 grid((unsigned)(batch * n), (unsigned)n_kv_heads);
  if (dtype == PRICHS_DTYPE_BF16)
    hipLaunchKernelGGL(kv_write_kernel<bf16_t>, grid, dim3(64), 0, as_stream(stream),
                       static_cast<const bf16_t *>(k), ldk, static_cast<const bf16_t *>(v), ldv,
                       static_cast<uint8_t *>(cache), (int)n_pages, page_table, (int)max_pages,
                       start, counts, (int)n, (int)n_kv_heads);
  else
    hipLaunchKernelGGL(kv_write_kernel<float>, grid, dim3(64), 0, as_stream(stream),
                       static_cast<const float *>(k), ldk, static_cast<const float *>(v), ldv,
                       static_cast<uint8_t *>(cache), (int)n_pages, page_table, (int)max_pages,
                       start, counts, (int)n, (int)n_kv_heads);
  PRICHS_LAUNCH_CHECK("kv_cache_write launch");
  return PRICHS_OK;
}

extern "C" int prichs_kv_cache_read(const void *cache, size_t n_pages, const int32_t *page_table,
                                    size_t max_pages, const int32_t *start,
                                    const int32_t *counts, void *k, size_t ldk, void *v,
                                    size_t ldv, size_t batch, size_t n, size_t n_kv_heads,
                                    size_t head_dim, int dtype, void *stream) {
  bool work;
  const int rc = kv_check("kv_cache_read", k, ldk, v, ldv, cache, n_pages, page_table, max_pages,
                          start, batch, n, n_kv_heads, head_dim, dtype, &work);
  if (rc != PRICHS_OK || !work) return rc;
  const dim3 grid((unsigned)(batch * n), (unsigned)n_kv_heads);
  if (dtype == PRICHS_DTYPE_BF16)
    hipLaunchKernelGGL(kv_read_kernel<bf16_t>, grid, dim3(64), 0, as_stream(stream),
                       static_cast<bf16_t *>(k), ldk, static_cast<bf16_t *>(v), ldv,
                       static_cast<const uint8_t *>(cache), (int)n_pages, page_table,
                       (int)max_pages, start, counts, (int)n, (int)n_kv_heads);
  else
    hipLaunchKernelGGL(kv_read_kernel<float>, grid, dim3(64), 0, as_stream(stream),
                       static_cast<float *>(k), ldk, static_cast<float *>(v), ldv,
                       static_cast<const uint8_t *>(cache), (int)n_pages, page_table,
                       (int)max_pages, start, counts, (int)n, (int)n_kv_heads);
  PRICHS_LAUNCH_CHECK("kv_cache_read launch");
  return PRICHS_OK;
}
