// window_attention.hip -- causal GQA attention with a sliding window and sinks,
// and its backward.
#include "common.hpp"

namespace prichs {
namespace {

constexpr int kHd = 128;

// Rows of sequence b.
__device__ __forceinline__ int rows_of(const int32_t *seq_lens, int b, int S) {
  return seq_lens == nullptr ? S : min(max(seq_lens[b], 0), S);
}
__device__ __forceinline__ float wave_sum(float x) {
  for (int m = 1; m < 64; m <<= 1) x += __shfl_xor(x, m);
  return x;
}
__device__ __forceinline__ float2 load2(const bf16_t *p) {
  return make_float2(bf16_to_f32(p[0]), bf16_to_f32(p[1]));
}
__device__ __forceinline__ void store2(bf16_t *p, float a, float b) {
  *reinterpret_cast<uint32_t *>(p) = pack_bf16x2(a, b);
}

struct Shape {
  int S, Hq, Hkv, window, sinks;
  float scale;
};

// delta[b][h][i] = d_o . o, one wave per (row, query head).
__global__ __launch_bounds__(64) void window_delta_kernel(const bf16_t *d_o, size_t ldd,
                                                          const bf16_t *o, size_t ldo,
                                                          const int32_t *seq_lens, float *delta,
                                                          Shape sh) {
  const int lane = threadIdx.x, h = blockIdx.y;
  const int b = blockIdx.x / sh.S, i = blockIdx.x - b * sh.S;
  if (i >= rows_of(seq_lens, b, sh.S)) return;
  const size_t c = (size_t)h * kHd + 2 * lane;
  const float2 x = load2(d_o + (size_t)blockIdx.x * ldd + c),
               y = load2(o + (size_t)blockIdx.x * ldo + c);
  const float s = wave_sum(x.x * y.x + x.y * y.y);
  if (lane == 0) delta[((size_t)b * sh.Hq + h) * sh.S + i] = s;
}

// One wave per (row, query head): d_q.
__global__ __launch_bounds__(64) void window_dq_row_kernel(
    const bf16_t *d_o, size_t ldd, const bf16_t *q, size_t ldq, const bf16_t *k, size_t ldk,
    const bf16_t *v, size_t ldv, const float *lse, const float *delta, const int32_t *seq_lens,
    bf16_t *dq, size_t lddq, Shape sh) {
  const int lane = threadIdx.x, h = blockIdx.y;
  const int b = blockIdx.x / sh.S, i = blockIdx.x - b * sh.S;
  const int kvh = h / (sh.Hq / sh.Hkv);
  const size_t row0 = (size_t)b * sh.S, hc = (size_t)h * kHd + 2 * lane;
  bf16_t *out = dq + (row0 + i) * lddq + hc;
  if (i >= rows_of(seq_lens, b, sh.S)) {
    store2(out, 0.f, 0.f);
    return;
  }
  const float2 qv = load2(q + (row0 + i) * ldq + hc), dv = load2(d_o + (row0 + i) * ldd + hc);
  const size_t st = ((size_t)b * sh.Hq + h) * sh.S + i;
  const int lo = sh.window == 0 ? 0 : max(0, i - sh.window + 1);
  float a0 = 0.f, a1 = 0.f;
  for (int j = 0; j <= i; ++j) {
    if (j >= min(sh.sinks, lo) && j < lo) j = lo;
    const size_t c = (size_t)kvh * kHd + 2 * lane;
    const float2 kv = load2(k + (row0 + j) * ldk + c), vv = load2(v + (row0 + j) * ldv + c);
    const float p = expf(wave_sum(qv.x * kv.x + qv.y * kv.y) * sh.scale - lse[st]);
    const float ds = p * (wave_sum(dv.x * vv.x + dv.y * vv.y) - delta[st]) * sh.scale;
    a0 += ds * kv.x;
    a1 += ds * kv.y;
  }
  store2(out, a0, a1);
}

// One wave per (key, kv head): d_k and d_v over the rows and query heads that
// see the key.
__global__ __launch_bounds__(64) void window_dkv_row_kernel(
    const bf16_t *d_o, size_t ldd, const bf16_t *q, size_t ldq, const bf16_t *k, size_t ldk,
    const bf16_t *v, size_t ldv, const float *lse, const float *delta, const int32_t *seq_lens,
    bf16_t *dk, size_t lddk, bf16_t *dv, size_t lddv, Shape sh) {
  const int lane = threadIdx.x, kvh = blockIdx.y;
  const int b = blockIdx.x / sh.S, j = blockIdx.x - b * sh.S;
  const int L = rows_of(seq_lens, b, sh.S), G = sh.Hq / sh.Hkv;
  const size_t row0 = (size_t)b * sh.S, c = (size_t)kvh * kHd + 2 * lane;
  float k0 = 0.f, k1 = 0.f, v0 = 0.f, v1 = 0.f;
  if (j < L) {
    const float2 kv = load2(k + (row0 + j) * ldk + c), vv = load2(v + (row0 + j) * ldv + c);
    const bool far = sh.window == 0 || j < sh.sinks || sh.window > L - j;
    const int end = far ? L : j + sh.window;
    for (int h = kvh * G; h < (kvh + 1) * G; ++h)
      for (int i = j; i < end; ++i) {
        const size_t st = ((size_t)b * sh.Hq + h) * sh.S + i, hc = (size_t)h * kHd + 2 * lane;
        const float2 qv = load2(q + (row0 + i) * ldq + hc),
                     gv = load2(d_o + (row0 + i) * ldd + hc);
        const float p = expf(wave_sum(qv.x * kv.x + qv.y * kv.y) * sh.scale - lse[st]);
        const float ds = p * (wave_sum(gv.x * vv.x + gv.y * vv.y) - delta[st]) * sh.scale;
        k0 += ds * qv.x;
        k1 += ds * qv.y;
        v0 += p * gv.x;
        v1 += p * gv.y;
      }
  }
  store2(dk + (row0 + j) * lddk + c, k0, k1);
  store2(dv + (row0 + j) * lddv + c, v0, v1);
}

// Checks shared by both directions; PRICHS_OK with *work = false where there is
// nothing to do.
int check_shape(const char *who, size_t batch, size_t seq_len, size_t n_heads, size_t n_kv_heads,
                size_t head_dim, int dtype, size_t window, size_t sinks, Shape *sh, bool *work) {
  *work = false;
  PRICHS_REQUIRE(dtype == PRICHS_DTYPE_BF16, "%s: only bf16 is supported (dtype=%d)", who, dtype);
  if (head_dim != (size_t)kHd)
    return fail(PRICHS_ERR_UNSUPPORTED, "%s: head_dim=%zu (only %d is supported)", who, head_dim,
                kHd);
  PRICHS_REQUIRE(n_heads >= 1 && n_kv_heads >= 1 && n_heads % n_kv_heads == 0,
                 "%s: n_heads=%zu must be a positive multiple of n_kv_heads=%zu", who, n_heads,
                 n_kv_heads);
  PRICHS_REQUIRE(n_heads <= 65535 && batch <= 65535 && seq_len <= (size_t)1 << 21 &&
                     batch * seq_len <= (size_t)INT32_MAX / 2,
                 "%s: shape too large", who);
  // A window past the sequence hides nothing.
  *sh = Shape{(int)seq_len,
              (int)n_heads,
              (int)n_kv_heads,
              (int)(window >= seq_len ? 0 : window),
              (int)(sinks < seq_len ? sinks : seq_len),
              1.0f / sqrtf((float)head_dim)};
  *work = batch != 0 && seq_len != 0;
  return PRICHS_OK;
}

// A row operand: its leading dimension holds its heads, and rows and base are
// 16-byte aligned.
int check_rows(const char *who, const char *name, const void *p, size_t ld, size_t cols) {
  PRICHS_REQUIRE(p != nullptr, "%s: null pointer argument %s", who, name);
  PRICHS_REQUIRE(ld >= cols && ld % 8 == 0 && ld < ((size_t)1 << 25),
                 "%s: the leading dimension %zu of %s must be a multiple of 8 elements, at least "
                 "%zu and below 2^25",
                 who, ld, name, cols);
  PRICHS_REQUIRE(reinterpret_cast<uintptr_t>(p) % 16 == 0, "%s: %s must be 16-byte aligned", who,
                 name);
  return PRICHS_OK;
}

}  // namespace
}  // namespace prichs

using namespace prichs;

#define WINDOW_TRY(expr)                     \
  do {                                       \
    const int _rc = (expr);                  \
    if (_rc != PRICHS_OK) return _rc;        \
  } while (0)

extern "C" int prichs_window_attention_forward(
    const void *q, size_t ldq, const void *k, size_t ldk, const void *v, size_t ldv, void *o,
    size_t ldo, float *lse, const int32_t *seq_lens, size_t batch, size_t seq_len, size_t n_heads,
    size_t n_kv_heads, size_t head_dim, size_t window, size_t sinks, int dtype, void *stream) {
  const char *who = "window_attention";
  Shape sh;
  bool work;
  WINDOW_TRY(check_shape(who, batch, seq_len, n_heads, n_kv_heads, head_dim, dtype, window, sinks,
                         &sh, &work));
  if (!work) return PRICHS_OK;
  const size_t H = n_heads * head_dim, K = n_kv_heads * head_dim;
  WINDOW_TRY(check_rows(who, "q", q, ldq, H));
  WINDOW_TRY(check_rows(who, "k", k, ldk, K));
  WINDOW_TRY(check_rows(who, "v", v, ldv, K));
  WINDOW_TRY(check_rows(who, "o", o, ldo, H));
  return window_attention_launch(q, ldq, k, ldk, v, ldv, o, ldo, lse, seq_lens, batch, seq_len,
                                 n_heads, n_kv_heads, (size_t)sh.window, (size_t)sh.sinks, stream);
}

extern "C" size_t prichs_window_attention_backward_workspace(size_t batch, size_t seq_len,
                                                             size_t n_heads, size_t n_kv_heads) {
  (void)n_kv_heads;
  return roundup(batch * seq_len * n_heads * sizeof(float), 256);
}

extern "C" int prichs_window_attention_backward(
    const void *d_o, size_t ldd, const void *q, size_t ldq, const void *k, size_t ldk,
    const void *v, size_t ldv, const void *o, size_t ldo, const float *lse,
    const int32_t *seq_lens, void *d_q, size_t lddq, void *d_k, size_t lddk, void *d_v,
    size_t lddv, size_t batch, size_t seq_len, size_t n_heads, size_t n_kv_heads, size_t head_dim,
    size_t window, size_t sinks, int dtype, void *workspace, size_t workspace_bytes,
    void *stream) {
  const char *who = "window_attention_backward";
  Shape sh;
  bool work;
  WINDOW_TRY(check_shape(who, batch, seq_len, n_heads, n_kv_heads, head_dim, dtype, window, sinks,
                         &sh, &work));
  if (!work) return PRICHS_OK;
  const size_t H = n_heads * head_dim, K = n_kv_heads * head_dim;
  WINDOW_TRY(check_rows(who, "d_o", d_o, ldd, H));
  WINDOW_TRY(check_rows(who, "q", q, ldq, H));
  WINDOW_TRY(check_rows(who, "k", k, ldk, K));
  WINDOW_TRY(check_rows(who, "v", v, ldv, K));
  WINDOW_TRY(check_rows(who, "o", o, ldo, H));
  WINDOW_TRY(check_rows(who, "d_q", d_q, lddq, H));
  WINDOW_TRY(check_rows(who, "d_k", d_k, lddk, K));
  WINDOW_TRY(check_rows(who, "d_v", d_v, lddv, K));
  PRICHS_REQUIRE(lse != nullptr, "%s: null pointer argument lse", who);
  const size_t need =
      prichs_window_attention_backward_workspace(batch, seq_len, n_heads, n_kv_heads);
  if (workspace_bytes < need)
    return fail(PRICHS_ERR_CAPACITY, "%s: workspace of %zu bytes, %zu needed", who,
                workspace_bytes, need);
  PRICHS_REQUIRE(workspace != nullptr && reinterpret_cast<uintptr_t>(workspace) % 16 == 0,
                 "%s: the workspace must be 16-byte aligned device memory", who);
  float *delta = static_cast<float *>(workspace);
  const dim3 rows_q((unsigned)(batch * seq_len), (unsigned)n_heads),
      rows_kv((unsigned)(batch * seq_len), (unsigned)n_kv_heads);
  const auto *bd = static_cast<const bf16_t *>(d_o), *bq = static_cast<const bf16_t *>(q),
             *bk = static_cast<const bf16_t *>(k), *bv = static_cast<const bf16_t *>(v),
             *bo = static_cast<const bf16_t *>(o);
  hipLaunchKernelGGL(window_delta_kernel, rows_q, dim3(64), 0, as_stream(stream), bd, ldd, bo, ldo,
                     seq_lens, delta, sh);
  PRICHS_LAUNCH_CHECK("window_attention_backward delta launch");
  hipLaunchKernelGGL(window_dq_row_kernel, rows_q, dim3(64), 0, as_stream(stream), bd, ldd, bq,
                     ldq, bk, ldk, bv, ldv, lse, delta, seq_lens, static_cast<bf16_t *>(d_q), lddq,
                     sh);
  PRICHS_LAUNCH_CHECK("window_attention_backward d_q launch");
  hipLaunchKernelGGL(window_dkv_row_kernel, rows_kv, dim3(64), 0, as_stream(stream), bd, ldd, bq,
                     ldq, bk, ldk, bv, ldv, lse, delta, seq_lens, static_cast<bf16_t *>(d_k), lddk,
                     static_cast<bf16_t *>(d_v), lddv, sh);
  PRICHS_LAUNCH_CHECK("window_attention_backward d_k / d_v launch");
  return PRICHS_OK;
}
