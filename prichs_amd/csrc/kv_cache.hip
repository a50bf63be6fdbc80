// kv_cache.hip -- tokens quantised into the paged 4-bit KV cache, and read
// back.  kv_cache.hpp has the layout and the number format.
#include "kv_cache.hpp"

namespace prichs {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

// Both kernels are bound by HBM (a read of 512 bytes and a write of 136 per
// position and kv head in bf16, or the reverse; 1024 and 136 in f32).  32 sequences x
// 6000 positions x 3 heads: 373 MB in bf16, written in 81 us and read in 93 back to
// back (92 and 86 alone), 668 MB in f32, 137 and 175 (165 and 162): 4.0 to 4.9 TB/s.
// 4 x 2048 positions: 5.2 and 5.5 us, f32 5.7 and 8.9; one new token of 32 sequences
// 3.3 us, which is the launch.  16 lanes hold one (position, kv
// head), 8 values each: one 16-byte access in bf16, one dword of codes.  Items run
// over (sequence, head, row) with the row fastest, so that a wave's four items are
// as a rule four positions of one head, whose V dwords are neighbours in the cache
// -- and four heads where every sequence has one new token.
constexpr int kItems = 16;  // items per workgroup of 256 threads
// Whole workgroups of items whose lanes (16 an item) stay below 2^32 in a launch.
constexpr size_t kMaxItems = ((size_t)1 << 28) - kItems;

struct Item {
  int row, h, c, page, t;  // row of k / v; dword c; page (-1: none) and slot
  bool live;               // not past its sequence's count
};
__device__ __forceinline__ bool item_of(Item &it, const int32_t *table, int max_pages, int n_pages,
                                        const int32_t *start, const int32_t *counts, int n,
                                        int kv_heads, uint32_t items) {
  const uint32_t x = blockIdx.x * (uint32_t)kItems + threadIdx.x / 16;
  if (x >= items) return false;
  const uint32_t bh = x / (uint32_t)n;
  const int i = (int)(x - bh * (uint32_t)n), b = (int)(bh / (uint32_t)kv_heads);
  it.h = (int)(bh - (uint32_t)b * (uint32_t)kv_heads);
  it.row = b * n + i;
  it.c = threadIdx.x & 15;
  it.live = counts == nullptr || i < counts[b];
  const long long pos = (long long)start[b] + i;
  it.page = kv_page_of(table, max_pages, n_pages, b, pos);
  it.t = (int)(pos & (kKvPage - 1));
  return true;
}

__device__ __forceinline__ void load8(const float *p, float (&x)[8]) {
  const f32x4 a = *reinterpret_cast<const f32x4 *>(p), b = *reinterpret_cast<const f32x4 *>(p + 4);
#pragma unroll
  for (int e = 0; e < 4; ++e) x[e] = a[e], x[4 + e] = b[e];
}
__device__ __forceinline__ void load8(const bf16_t *p, float (&x)[8]) {
  const u32x4 u = *reinterpret_cast<const u32x4 *>(p);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    x[2 * e] = __uint_as_float(u[e] << 16);
    x[2 * e + 1] = __uint_as_float(u[e] & 0xffff0000u);
  }
}

// 8 values of a group of 32 that 4 neighbouring lanes hold: their codes, and the
// group's scale byte.
__device__ __forceinline__ uint32_t quantise8(const float (&x)[8], uint32_t *scale) {
  uint32_t amax = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) amax = max(amax, __float_as_uint(x[e]) & 0x7fffffffu);
  amax = max(amax, (uint32_t)__shfl_xor((int)amax, 1));
  amax = max(amax, (uint32_t)__shfl_xor((int)amax, 2));
  *scale = kv_scale_byte(amax);
  if (*scale == 255) return 0;
  const float sc = kv_scale(*scale);
  uint32_t code = 0;
  code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, x[0], x[1], sc, 0);
  code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, x[2], x[3], sc, 1);
  code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, x[4], x[5], sc, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, x[6], x[7], sc, 3);
}

template <typename T>
__global__ __launch_bounds__(256) void kv_write_kernel(
    const T *__restrict__ k, size_t ldk, const T *__restrict__ v, size_t ldv, uint8_t *cache,
    int n_pages, const int32_t *table, int max_pages, const int32_t *start, const int32_t *counts,
    int n, int kv_heads, uint32_t items) {
  Item it;
  if (!item_of(it, table, max_pages, n_pages, start, counts, n, kv_heads, items)) return;
  if (!it.live || it.page < 0) return;  // the 16 lanes of an item agree
  const size_t col = (size_t)it.h * kKvHd + 8 * it.c;
  float xk[8], xv[8];
  load8(k + (size_t)it.row * ldk + col, xk);
  load8(v + (size_t)it.row * ldv + col, xv);
  uint32_t sk, sv;
  const uint32_t ck = quantise8(xk, &sk), cv = quantise8(xv, &sv);
  uint8_t *part = cache + ((size_t)it.page * kv_heads + it.h) * kKvPart;
  *reinterpret_cast<uint32_t *>(part + kKvK + it.t * (kKvHd / 2) + 4 * it.c) = ck;
  *reinterpret_cast<uint32_t *>(part + kv_v_off(it.t, it.c)) = cv;
  if ((it.c & 3) == 0) {
    part[kv_k_scale_off(it.t, it.c >> 2)] = (uint8_t)sk;
    part[kv_v_scale_off(it.t, it.c >> 2)] = (uint8_t)sv;
  }
}

__device__ __forceinline__ void store8(bf16_t *p, uint32_t code, float sc) {
  u32x4 u;
  u[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(code, sc, 0));
  u[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(code, sc, 1));
  u[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(code, sc, 2));
  u[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(code, sc, 3));
  *reinterpret_cast<u32x4 *>(p) = u;
}
__device__ __forceinline__ void store8(float *p, uint32_t code, float sc) {
  const auto a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code, sc, 0);
  const auto b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code, sc, 1);
  const auto c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code, sc, 2);
  const auto d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code, sc, 3);
  *reinterpret_cast<f32x4 *>(p) = f32x4{a[0], a[1], b[0], b[1]};
  *reinterpret_cast<f32x4 *>(p + 4) = f32x4{c[0], c[1], d[0], d[1]};
}

template <typename T>
__global__ __launch_bounds__(256) void kv_read_kernel(
    T *__restrict__ k, size_t ldk, T *__restrict__ v, size_t ldv, const uint8_t *cache,
    int n_pages, const int32_t *table, int max_pages, const int32_t *start, const int32_t *counts,
    int n, int kv_heads, uint32_t items) {
  Item it;
  if (!item_of(it, table, max_pages, n_pages, start, counts, n, kv_heads, items)) return;
  if (!it.live) return;
  uint32_t ck = 0, cv = 0, sk = 127, sv = 127;  // zeros where there is no page
  if (it.page >= 0) {
    const uint8_t *part = cache + ((size_t)it.page * kv_heads + it.h) * kKvPart;
    ck = *reinterpret_cast<const uint32_t *>(part + kKvK + it.t * (kKvHd / 2) + 4 * it.c);
    cv = *reinterpret_cast<const uint32_t *>(part + kv_v_off(it.t, it.c));
    sk = part[kv_k_scale_off(it.t, it.c >> 2)];
    sv = part[kv_v_scale_off(it.t, it.c >> 2)];
  }
  const size_t col = (size_t)it.h * kKvHd + 8 * it.c;
  store8(k + (size_t)it.row * ldk + col, ck, kv_scale(sk));
  store8(v + (size_t)it.row * ldv + col, cv, kv_scale(sv));
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
                     (n == 0 || batch <= kMaxItems / n / n_kv_heads) && n_pages <= (size_t)INT32_MAX &&
                     max_pages <= (size_t)INT32_MAX / kKvPage,
                 "%s: shape too large", who);
  if (batch == 0 || n == 0) return PRICHS_OK;
  PRICHS_REQUIRE(k && v && start && (n_pages == 0 || cache) && (max_pages == 0 || page_table),
                 "%s: null pointer argument", who);
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
  const uint32_t items = (uint32_t)(batch * n * n_kv_heads);
  const dim3 grid((unsigned)cdiv(items, kItems));
  if (dtype == PRICHS_DTYPE_BF16)
    hipLaunchKernelGGL(kv_write_kernel<bf16_t>, grid, dim3(256), 0, as_stream(stream),
                       static_cast<const bf16_t *>(k), ldk, static_cast<const bf16_t *>(v), ldv,
                       static_cast<uint8_t *>(cache), (int)n_pages, page_table, (int)max_pages,
                       start, counts, (int)n, (int)n_kv_heads, items);
  else
    hipLaunchKernelGGL(kv_write_kernel<float>, grid, dim3(256), 0, as_stream(stream),
                       static_cast<const float *>(k), ldk, static_cast<const float *>(v), ldv,
                       static_cast<uint8_t *>(cache), (int)n_pages, page_table, (int)max_pages,
                       start, counts, (int)n, (int)n_kv_heads, items);
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
  const uint32_t items = (uint32_t)(batch * n * n_kv_heads);
  const dim3 grid((unsigned)cdiv(items, kItems));
  if (dtype == PRICHS_DTYPE_BF16)
    hipLaunchKernelGGL(kv_read_kernel<bf16_t>, grid, dim3(256), 0, as_stream(stream),
                       static_cast<bf16_t *>(k), ldk, static_cast<bf16_t *>(v), ldv,
                       static_cast<const uint8_t *>(cache), (int)n_pages, page_table,
                       (int)max_pages, start, counts, (int)n, (int)n_kv_heads, items);
  else
    hipLaunchKernelGGL(kv_read_kernel<float>, grid, dim3(256), 0, as_stream(stream),
                       static_cast<float *>(k), ldk, static_cast<float *>(v), ldv,
                       static_cast<const uint8_t *>(cache), (int)n_pages, page_table,
                       (int)max_pages, start, counts, (int)n, (int)n_kv_heads, items);
  PRICHS_LAUNCH_CHECK("kv_cache_read launch");
  return PRICHS_OK;
}
