// qk_norm_rope.hip -- queries and keys normed per head and rotated to their
// positions in one pass, and the gradients.
//
// A head x of d values, with xh = x inv, inv = 1 / sqrt(mean(x^2) + eps):
//   o = R(pos) (xh w)        R rotates the pairs (2i, 2i + 1) by cos / sin [pos][i];
//   g = R(pos)^T d_o, t = g w:
//   d_x = inv (t - xh mean(t xh)),   d_w = sum over rows and heads of g xh.
// Everything is f32 between the load and the one rounding of a result.
//
// `LANES` lanes hold one head of one row, 8 values (4 whole pairs) each, so sums over a
// head are a few lane exchanges.  Such a group of lanes takes up to kHeads heads of its
// row, kHeads loads in flight, with one load of the position's cos and sin (32 bytes a
// lane against 16 of a bf16 head).
#include "common.hpp"

namespace prichs {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256;
constexpr int kHeads = 4;  // heads of a group of lanes

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
__device__ __forceinline__ void store8(float *p, const float (&x)[8]) {
  *reinterpret_cast<f32x4 *>(p) = f32x4{x[0], x[1], x[2], x[3]};
  *reinterpret_cast<f32x4 *>(p + 4) = f32x4{x[4], x[5], x[6], x[7]};
}
__device__ __forceinline__ void store8(bf16_t *p, const float (&x)[8]) {
  *reinterpret_cast<u32x4 *>(p) = u32x4{pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]),
                                        pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7])};
}

template <int LANES>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
  for (int m = LANES / 2; m >= 1; m >>= 1) v += __shfl_xor(v, m);
  return v;
}

// The operands of a call.  Heads 0 .. Hq - 1 are q's, then k's.
template <typename T>
struct Args {
  const T *x[2];   // q, k
  const T *d[2];   // backward: gradients of the outputs
  T *out[2];       // outputs, or gradients of q and k
  size_t ldx[2], ldd[2], ldo[2];
  const float *w[2], *cs, *sn;
  const int32_t *positions;
  long long rows, cache_rows, pos_offset, seq_len;
  int Hq, H, hd, per_row;  // per_row: groups of lanes of a row
  float inv_hd, eps;
};

// Position of a row, or -1 outside the tables.
template <typename T>
__device__ __forceinline__ long long position(const Args<T> &a, long long row) {
  const long long p =
      a.positions != nullptr ? (long long)a.positions[row] : row % a.seq_len + a.pos_offset;
  return p < a.cache_rows ? p : -1;
}

// Head h of a row in q (or k) and its like.
template <typename T>
__device__ __forceinline__ T *head_at(T *const (&p)[2], const size_t (&ld)[2], long long row,
                                      int h, int Hq, int hd) {
  const bool isk = h >= Hq;
  return (isk ? p[1] : p[0]) + (size_t)row * (isk ? ld[1] : ld[0]) +
         (size_t)(h - (isk ? Hq : 0)) * hd;
}

// Unit u: row u / per_row; heads u % per_row + per_row j, so that neighbouring groups of
// lanes read neighbouring heads.
template <typename T, int LANES>
__global__ __launch_bounds__(kThreads) void qk_norm_rope_kernel(Args<T> a) {
  constexpr int kGroups = kThreads / LANES;
  const int c = threadIdx.x % LANES;
  const bool lane = 8 * c < a.hd;  // of the lanes' 8 LANES values hd are the head's
  const long long units = a.rows * a.per_row;
  for (long long u = (long long)blockIdx.x * kGroups + threadIdx.x / LANES; u < units;
       u += (long long)gridDim.x * kGroups) {
    const long long row = u / a.per_row;
    const int s = (int)(u - row * a.per_row);
    const long long pos = position(a, row);
    if (pos < 0) continue;  // the lanes of a group agree
    float x[kHeads][8], w[2][8], cs[4], sn[4];
#pragma unroll
    for (int j = 0; j < kHeads; ++j) {
      const int h = s + a.per_row * j;
#pragma unroll
      for (int e = 0; e < 8; ++e) x[j][e] = 0.f;
      if (lane && h < a.H) load8(head_at(a.x, a.ldx, row, h, a.Hq, a.hd) + 8 * c, x[j]);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) cs[e] = sn[e] = 0.f;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) w[i][e] = 0.f;
    if (lane) {
      const size_t at = (size_t)pos * (a.hd / 2) + 4 * c;
      const f32x4 c4 = *reinterpret_cast<const f32x4 *>(a.cs + at);
      const f32x4 s4 = *reinterpret_cast<const f32x4 *>(a.sn + at);
#pragma unroll
      for (int e = 0; e < 4; ++e) cs[e] = c4[e], sn[e] = s4[e];
      if (a.Hq > 0) load8(a.w[0] + 8 * c, w[0]);
      if (a.H > a.Hq) load8(a.w[1] + 8 * c, w[1]);
    }
#pragma unroll
    for (int j = 0; j < kHeads; ++j) {
      const int h = s + a.per_row * j;
      const bool isk = h >= a.Hq;
      float ss = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) ss = fmaf(x[j][e], x[j][e], ss);
      ss = lanes_sum<LANES>(ss);
      const float inv = 1.0f / sqrtf(fmaf(ss, a.inv_hd, a.eps));
      float o[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float y0 = x[j][2 * i] * inv * (isk ? w[1][2 * i] : w[0][2 * i]);
        const float y1 = x[j][2 * i + 1] * inv * (isk ? w[1][2 * i + 1] : w[0][2 * i + 1]);
        o[2 * i] = y0 * cs[i] - y1 * sn[i];
        o[2 * i + 1] = y0 * sn[i] + y1 * cs[i];
      }
      if (lane && h < a.H) store8(head_at(a.out, a.ldo, row, h, a.Hq, a.hd) + 8 * c, o);
    }
  }
}

// The gradients.  part: f32 [gridDim.x][2][hd], each workgroup's sums of d_wq and d_wk.
template <typename T, int LANES>
__global__ __launch_bounds__(kThreads) void qk_norm_rope_bwd_kernel(Args<T> a,
                                                                    float *__restrict__ part) {
  constexpr int kGroups = kThreads / LANES;
  __shared__ float s_dw[kGroups][2][8 * LANES];
  const int c = threadIdx.x % LANES, grp = threadIdx.x / LANES;
  const bool lane = 8 * c < a.hd;
  float w[2][8], dw[2][8];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) w[i][e] = dw[i][e] = 0.f;
  if (lane && a.Hq > 0) load8(a.w[0] + 8 * c, w[0]);
  if (lane && a.H > a.Hq) load8(a.w[1] + 8 * c, w[1]);
  const long long units = a.rows * a.per_row;
  for (long long u = (long long)blockIdx.x * kGroups + grp; u < units;
       u += (long long)gridDim.x * kGroups) {
    const long long row = u / a.per_row;
    const int s = (int)(u - row * a.per_row);
    const long long pos = position(a, row);
    const bool live = lane && pos >= 0;
    float x[kHeads][8], d[kHeads][8], cs[4], sn[4];
#pragma unroll
    for (int j = 0; j < kHeads; ++j) {
      const int h = s + a.per_row * j;
#pragma unroll
      for (int e = 0; e < 8; ++e) x[j][e] = d[j][e] = 0.f;
      if (live && h < a.H) {
        load8(head_at(a.x, a.ldx, row, h, a.Hq, a.hd) + 8 * c, x[j]);
        load8(head_at(a.d, a.ldd, row, h, a.Hq, a.hd) + 8 * c, d[j]);
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) cs[e] = sn[e] = 0.f;
    if (live) {
      const size_t at = (size_t)pos * (a.hd / 2) + 4 * c;
      const f32x4 c4 = *reinterpret_cast<const f32x4 *>(a.cs + at);
      const f32x4 s4 = *reinterpret_cast<const f32x4 *>(a.sn + at);
#pragma unroll
      for (int e = 0; e < 4; ++e) cs[e] = c4[e], sn[e] = s4[e];
    }
#pragma unroll
    for (int j = 0; j < kHeads; ++j) {
      const int h = s + a.per_row * j;
      const bool isk = h >= a.Hq;
      float g[8], t[8], ss = 0.f, tx = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        g[2 * i] = d[j][2 * i] * cs[i] + d[j][2 * i + 1] * sn[i];
        g[2 * i + 1] = d[j][2 * i + 1] * cs[i] - d[j][2 * i] * sn[i];
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        t[e] = g[e] * (isk ? w[1][e] : w[0][e]);
        ss = fmaf(x[j][e], x[j][e], ss);
        tx = fmaf(t[e], x[j][e], tx);
      }
      ss = lanes_sum<LANES>(ss);
      tx = lanes_sum<LANES>(tx);
      const float inv = 1.0f / sqrtf(fmaf(ss, a.inv_hd, a.eps));
      const float m = tx * inv * a.inv_hd;  // mean(t xh)
      float o[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float xh = x[j][e] * inv;
        o[e] = inv * (t[e] - xh * m);
        // A group without a position or past the last head adds nothing, whatever inv is.
        const float p = live && h < a.H ? g[e] * xh : 0.f;
        dw[0][e] += isk ? 0.f : p;
        dw[1][e] += isk ? p : 0.f;
      }
      if (lane && h < a.H) {
        if (pos < 0)
#pragma unroll
          for (int e = 0; e < 8; ++e) o[e] = 0.f;
        store8(head_at(a.out, a.ldo, row, h, a.Hq, a.hd) + 8 * c, o);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) s_dw[grp][i][8 * c + e] = dw[i][e];
  __syncthreads();
  for (int v = threadIdx.x; v < 2 * a.hd; v += kThreads) {
    const int i = v >= a.hd, e = v - (i ? a.hd : 0);
    float sum = 0.f;
#pragma unroll
    for (int q = 0; q < kGroups; ++q) sum += s_dw[q][i][e];
    part[(size_t)blockIdx.x * 2 * a.hd + v] = sum;
  }
}

// d_w[v] (+)= the workgroups' sums, added in a fixed order: 32 columns a workgroup, 32
// threads a column, whose loads are all in flight.
__global__ __launch_bounds__(1024) void qk_norm_dw_kernel(const float *__restrict__ part, int n,
                                                          int hd, float *d_wq, float *d_wk,
                                                          int beta) {
  __shared__ float s[32][33];
  const int col = threadIdx.x & 31, r = threadIdx.x >> 5, v = blockIdx.x * 32 + col;
  float sum = 0.f;
  if (v < 2 * hd) {
#pragma unroll 8
    for (int i = r; i < n; i += 32) sum += part[(size_t)i * 2 * hd + v];
  }
  s[r][col] = sum;
  __syncthreads();
  if (r != 0 || v >= 2 * hd) return;
  sum = 0.f;
#pragma unroll
  for (int i = 0; i < 32; ++i) sum += s[i][col];
  float *out = v < hd ? d_wq : d_wk;
  if (out == nullptr) return;  // a call without queries or without keys
  out += v < hd ? v : v - hd;
  *out = beta ? *out + sum : sum;
}

// Workgroups of the backward: the sums of the weights' gradients end in one row of `part`
// each.
constexpr size_t kBwdBlocks = 1024;
int lanes_of(size_t hd) { return hd <= 32 ? 4 : hd <= 64 ? 8 : hd <= 128 ? 16 : 32; }
size_t per_row_of(size_t heads) { return cdiv(heads, (size_t)kHeads); }
size_t bwd_blocks(size_t rows, size_t heads, size_t hd) {
  const size_t blocks = cdiv(rows * per_row_of(heads), (size_t)(kThreads / lanes_of(hd)));
  return blocks < kBwdBlocks ? blocks : kBwdBlocks;
}

bool al16(const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// Checks and operands of both directions; *work = false where there is nothing to do.
struct Call {
  const void *x[2], *d[2];
  void *out[2];
  size_t ldx[2], ldd[2], ldo[2];
  const float *w[2], *cs, *sn;
  size_t cache_rows;
  const int32_t *positions;
  size_t seq_len, pos_offset, rows, heads[2], hd;
  float eps;
  int dtype;
};
int check(const char *who, const Call &c, bool backward, bool *work) {
  *work = false;
  PRICHS_REQUIRE(dtype_ok(c.dtype), "%s: bad dtype %d", who, c.dtype);
  if (c.hd < 8 || c.hd > 256 || c.hd % 8 != 0)
    return fail(PRICHS_ERR_UNSUPPORTED, "%s: head_dim=%zu (multiples of 8 up to 256)", who, c.hd);
  PRICHS_REQUIRE(c.heads[0] <= 65535 && c.heads[1] <= 65535 && c.heads[0] + c.heads[1] >= 1,
                 "%s: n_heads=%zu, n_kv_heads=%zu", who, c.heads[0], c.heads[1]);
  PRICHS_REQUIRE(c.rows <= (size_t)INT32_MAX && c.cache_rows <= (size_t)INT32_MAX,
                 "%s: shape too large", who);
  PRICHS_REQUIRE(c.eps >= 0.f, "%s: eps must not be negative", who);
  if (c.positions == nullptr) {
    PRICHS_REQUIRE(c.seq_len >= 1, "%s: without positions seq_len must be positive", who);
    PRICHS_REQUIRE(c.seq_len <= c.cache_rows && c.pos_offset <= c.cache_rows - c.seq_len,
                   "%s: positions up to %zu + %zu exceed the tables (%zu rows)", who, c.seq_len,
                   c.pos_offset, c.cache_rows);
  }
  for (int i = 0; i < 2; ++i) {
    const size_t width = c.heads[i] * c.hd;
    if (width == 0) continue;
    PRICHS_REQUIRE(c.ldx[i] >= width && c.ldo[i] >= width && (!backward || c.ldd[i] >= width) &&
                       c.ldx[i] % 8 == 0 && c.ldo[i] % 8 == 0 && (!backward || c.ldd[i] % 8 == 0),
                   "%s: leading dimensions must be multiples of 8 elements that hold all heads",
                   who);
  }
  if (c.rows == 0 && !backward) return PRICHS_OK;
  for (int i = 0; i < 2; ++i) {
    if (c.heads[i] == 0) continue;
    if (c.rows > 0) {
      PRICHS_REQUIRE(c.x[i] && c.out[i] && c.w[i] && (!backward || c.d[i]),
                     "%s: null pointer argument", who);
      PRICHS_REQUIRE(al16(c.x[i]) && al16(c.out[i]) && al16(c.w[i]) && (!backward || al16(c.d[i])),
                     "%s: operands must be 16-byte aligned", who);
    }
  }
  if (c.rows > 0) {
    PRICHS_REQUIRE(c.cs && c.sn, "%s: null pointer argument", who);
    PRICHS_REQUIRE(al16(c.cs) && al16(c.sn), "%s: the tables must be 16-byte aligned", who);
  }
  *work = true;
  return PRICHS_OK;
}

template <typename T>
Args<T> args_of(const Call &c) {
  Args<T> a;
  for (int i = 0; i < 2; ++i) {
    a.x[i] = static_cast<const T *>(c.x[i]);
    a.d[i] = static_cast<const T *>(c.d[i]);
    a.out[i] = static_cast<T *>(c.out[i]);
    a.ldx[i] = c.ldx[i], a.ldd[i] = c.ldd[i], a.ldo[i] = c.ldo[i];
    a.w[i] = c.w[i];
  }
  a.cs = c.cs, a.sn = c.sn, a.positions = c.positions;
  a.rows = (long long)c.rows, a.cache_rows = (long long)c.cache_rows;
  a.pos_offset = (long long)c.pos_offset, a.seq_len = (long long)(c.positions ? 1 : c.seq_len);
  a.Hq = (int)c.heads[0], a.H = (int)(c.heads[0] + c.heads[1]), a.hd = (int)c.hd;
  a.per_row = (int)per_row_of(c.heads[0] + c.heads[1]);
  a.inv_hd = 1.0f / (float)c.hd, a.eps = c.eps;
  return a;
}

template <typename T>
void launch_forward(const Call &c, hipStream_t s) {
  const int lanes = lanes_of(c.hd);
  const size_t units = c.rows * per_row_of(c.heads[0] + c.heads[1]);
  const size_t blocks = cdiv(units, (size_t)(kThreads / lanes));
  const dim3 grid((unsigned)(blocks < (1u << 20) ? blocks : 1u << 20));
  auto kern = lanes == 4    ? qk_norm_rope_kernel<T, 4>
              : lanes == 8  ? qk_norm_rope_kernel<T, 8>
              : lanes == 16 ? qk_norm_rope_kernel<T, 16>
                            : qk_norm_rope_kernel<T, 32>;
  hipLaunchKernelGGL(kern, grid, dim3(kThreads), 0, s, args_of<T>(c));
}
template <typename T>
void launch_backward(const Call &c, size_t blocks, float *part, hipStream_t s) {
  const int lanes = lanes_of(c.hd);
  auto kern = lanes == 4    ? qk_norm_rope_bwd_kernel<T, 4>
              : lanes == 8  ? qk_norm_rope_bwd_kernel<T, 8>
              : lanes == 16 ? qk_norm_rope_bwd_kernel<T, 16>
                            : qk_norm_rope_bwd_kernel<T, 32>;
  hipLaunchKernelGGL(kern, dim3((unsigned)blocks), dim3(kThreads), 0, s, args_of<T>(c), part);
}

}  // namespace
}  // namespace prichs

using namespace prichs;

extern "C" int prichs_qk_norm_rope_forward(const void *q, size_t ldq, const void *k, size_t ldk,
                                           const float *w_q, const float *w_k,
                                           const float *cos_cache, const float *sin_cache,
                                           size_t cache_rows, const int32_t *positions,
                                           size_t seq_len, size_t pos_offset, void *q_out,
                                           size_t ldqo, void *k_out, size_t ldko, size_t rows,
                                           size_t n_heads, size_t n_kv_heads, size_t head_dim,
                                           float eps, int dtype, void *stream) {
  const Call c{{q, k},
               {nullptr, nullptr},
               {q_out, k_out},
               {ldq, ldk},
               {0, 0},
               {ldqo, ldko},
               {w_q, w_k},
               cos_cache,
               sin_cache,
               cache_rows,
               positions,
               seq_len,
               pos_offset,
               rows,
               {n_heads, n_kv_heads},
               head_dim,
               eps,
               dtype};
  bool work;
  const int rc = check("qk_norm_rope_forward", c, false, &work);
  if (rc != PRICHS_OK || !work) return rc;
  if (dtype == PRICHS_DTYPE_BF16)
    launch_forward<bf16_t>(c, as_stream(stream));
  else
    launch_forward<float>(c, as_stream(stream));
  PRICHS_LAUNCH_CHECK("qk_norm_rope_forward launch");
  return PRICHS_OK;
}

extern "C" size_t prichs_qk_norm_rope_backward_workspace(size_t rows, size_t n_heads,
                                                         size_t n_kv_heads, size_t head_dim) {
  if (rows == 0 || rows > (size_t)INT32_MAX || head_dim == 0 || head_dim > 256 ||
      n_heads > 65535 || n_kv_heads > 65535)
    return 0;
  return bwd_blocks(rows, n_heads + n_kv_heads, head_dim) * 2 * head_dim * sizeof(float);
}

extern "C" int prichs_qk_norm_rope_backward(
    const void *d_q_out, size_t lddqo, const void *d_k_out, size_t lddko, const void *q,
    size_t ldq, const void *k, size_t ldk, const float *w_q, const float *w_k,
    const float *cos_cache, const float *sin_cache, size_t cache_rows, const int32_t *positions,
    size_t seq_len, size_t pos_offset, void *d_q, size_t lddq, void *d_k, size_t lddk,
    float *d_wq, float *d_wk, int beta, size_t rows, size_t n_heads, size_t n_kv_heads,
    size_t head_dim, float eps, int dtype, void *workspace, size_t workspace_bytes,
    void *stream) {
  const char *who = "qk_norm_rope_backward";
  const Call c{{q, k},
               {d_q_out, d_k_out},
               {d_q, d_k},
               {ldq, ldk},
               {lddqo, lddko},
               {lddq, lddk},
               {w_q, w_k},
               cos_cache,
               sin_cache,
               cache_rows,
               positions,
               seq_len,
               pos_offset,
               rows,
               {n_heads, n_kv_heads},
               head_dim,
               eps,
               dtype};
  bool work;
  const int rc = check(who, c, true, &work);
  if (rc != PRICHS_OK) return rc;
  PRICHS_REQUIRE(beta == 0 || beta == 1, "%s: beta must be 0 or 1", who);
  PRICHS_REQUIRE((n_heads == 0 || d_wq) && (n_kv_heads == 0 || d_wk),
                 "%s: null pointer argument", who);
  const size_t need =
      prichs_qk_norm_rope_backward_workspace(rows, n_heads, n_kv_heads, head_dim);
  if (workspace_bytes < need)
    return fail(PRICHS_ERR_CAPACITY, "%s: workspace of %zu bytes, %zu needed", who,
                workspace_bytes, need);
  PRICHS_REQUIRE(need == 0 || (workspace != nullptr && al16(workspace)),
                 "%s: the workspace must be 16-byte aligned device memory", who);
  const hipStream_t s = as_stream(stream);
  float *part = static_cast<float *>(workspace);
  // No rows: no sums, and d_w is zero (or stays what it was).
  const size_t blocks = rows == 0 ? 0 : bwd_blocks(rows, n_heads + n_kv_heads, head_dim);
  if (blocks > 0) {
    if (dtype == PRICHS_DTYPE_BF16)
      launch_backward<bf16_t>(c, blocks, part, s);
    else
      launch_backward<float>(c, blocks, part, s);
    PRICHS_LAUNCH_CHECK("qk_norm_rope_backward launch");
  }
  hipLaunchKernelGGL(qk_norm_dw_kernel, dim3((unsigned)cdiv(2 * head_dim, 32)), dim3(1024), 0, s,
                     part, (int)blocks, (int)head_dim, n_heads ? d_wq : nullptr,
                     n_kv_heads ? d_wk : nullptr, beta);
  PRICHS_LAUNCH_CHECK("qk_norm_rope_backward weights launch");
  return PRICHS_OK;
}
