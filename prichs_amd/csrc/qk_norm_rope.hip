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
// head are a few lane exchanges.  Such a group of lanes takes kHeads heads of its row, whose
// loads are all in flight, with one load of the position's cos and sin (32 bytes a lane
// against 16 of a bf16 head).  Bound by HBM where there are many rows: 4 x 2048 of 12 + 3
// heads in bf16 (64 MB; MI355X) 12.6 us forward, 5.1 TB/s, and 18.4 backward (98 MB, 5.3);
// by the launch where there are few (32 rows 3.7 us).  Heads a group, us of a captured
// forward, and of a forward and backward: 1 13.6 and 35.6, 2 12.6 and 34.1, 3 12.2 and 33.3,
// 4 12.2 and 36.2, 5 12.6 and 44.8 (registers).
#include "common.hpp"

namespace prichs {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256;
constexpr int kHeads = 3;  // heads of a group of lanes

// 8 values as they were loaded; taken apart where they are used, which keeps the registers
// of loads in flight few.
template <typename T> struct Raw8;
template <> struct Raw8<float> {
  f32x4 a, b;
  __device__ __forceinline__ void load(const float *p) {
    a = *reinterpret_cast<const f32x4 *>(p), b = *reinterpret_cast<const f32x4 *>(p + 4);
  }
  __device__ __forceinline__ void clear() { a = b = f32x4{0.f, 0.f, 0.f, 0.f}; }
  __device__ __forceinline__ float operator[](int e) const { return e < 4 ? a[e] : b[e - 4]; }
};
template <> struct Raw8<bf16_t> {
  u32x4 u;
  __device__ __forceinline__ void load(const bf16_t *p) { u = *reinterpret_cast<const u32x4 *>(p); }
  __device__ __forceinline__ void clear() { u = u32x4{0, 0, 0, 0}; }
  __device__ __forceinline__ float operator[](int e) const {
    return __uint_as_float(e & 1 ? u[e / 2] & 0xffff0000u : u[e / 2] << 16);
  }
};
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
  uint32_t rows, cache_rows, pos_offset, seq_len;
  int Hq, H, hd;
  uint32_t per_row;  // groups of lanes of a row
  float inv_hd, eps;
};

// Position of a row; cache_rows or more outside the tables.
template <typename T>
__device__ __forceinline__ uint32_t position(const Args<T> &a, uint32_t row) {
  return a.positions != nullptr ? (uint32_t)a.positions[row] : row % a.seq_len + a.pos_offset;
}
// Row and first head of a group of lanes: the `at`-th of workgroup `block`, `groups` a workgroup.
template <typename T>
__device__ __forceinline__ void unit_of(const Args<T> &a, uint64_t block, int groups, int at,
                                        uint64_t *row, int *s) {
  const uint64_t u0 = block * groups, r0 = u0 / a.per_row;  // the same for the workgroup
  const uint32_t x = (uint32_t)(u0 - r0 * a.per_row) + at, r = x / a.per_row;
  *row = r0 + r;
  *s = (int)(x - r * a.per_row);
}

// A lane's values of the heads s, s + per_row, .. of a row: in q (or its like) up to Hq, then
// in k, which gets an address of its own that lies Hq heads before k's row.
template <typename T> struct Heads {
  T *q, *k;
  __device__ __forceinline__ Heads(T *const (&p)[2], const size_t (&ld)[2], uint64_t row, int at,
                                   int Hq, int hd)
      : q(p[0] + row * ld[0] + at), k(p[1] + row * ld[1] + (at - Hq * hd)) {}
  __device__ __forceinline__ T *at(bool isk, int step) const { return (isk ? k : q) + step; }
};

// Unit u: row u / per_row; heads u % per_row + per_row j, so that neighbouring groups of
// lanes read neighbouring heads.
// Lanes past the head's end and heads past the last load what the group's first ones do,
// so that all loads are in flight without a branch between them.
// ZEROS: rows outside the tables become zeros (otherwise they stay as they were), by way of
// the others' loads and products, at no cost (4 x 2048 rows by position 12.8 us either way): a
// branch of their own took nine registers a lane from all rows and 3% of the time.
template <typename T, int LANES, bool ZEROS>
__device__ __forceinline__ void norm_rope(const Args<T> &a, uint64_t blocks) {
  constexpr int kGroups = kThreads / LANES;
  const int c = threadIdx.x % LANES;
  const bool lane = 8 * c < a.hd;  // of the lanes' 8 LANES values hd are the head's
  const int col = lane ? 8 * c : 0;
  for (uint64_t block = blockIdx.x; block < blocks; block += gridDim.x) {
    uint64_t row;
    int s;
    unit_of(a, block, kGroups, threadIdx.x / LANES, &row, &s);
    if (row >= a.rows) continue;  // the lanes of a group agree
    const uint32_t pos = position(a, (uint32_t)row);
    const bool live = pos < a.cache_rows;
    if (!ZEROS && !live) continue;
    const int step = (int)a.per_row * a.hd;  // from a head to the next of the group
    const Heads<const T> xs(a.x, a.ldx, row, s * a.hd + col, a.Hq, a.hd);
    Raw8<T> x[kHeads];
#pragma unroll
    for (int j = 0; j < kHeads; ++j) {
      const int h = s + a.per_row * j, jj = h < a.H ? j : 0;
      x[j].load(xs.at(s + (int)a.per_row * jj >= a.Hq, jj * step));
    }
    const size_t at = (size_t)(!ZEROS || live ? pos : 0) * (a.hd / 2) + col / 2;
    f32x4 cs = f32x4{0.f, 0.f, 0.f, 0.f}, sn = cs;
    if (!ZEROS || a.cache_rows > 0) {
      cs = *reinterpret_cast<const f32x4 *>(a.cs + at);
      sn = *reinterpret_cast<const f32x4 *>(a.sn + at);
    }
    Raw8<float> wq, wk;
    wq.load(a.w[0] + col), wk.load(a.w[1] + col);
    const Heads<T> os(a.out, a.ldo, row, s * a.hd + col, a.Hq, a.hd);
#pragma unroll
    for (int j = 0; j < kHeads; ++j) {
      const int h = s + a.per_row * j;
      const bool isk = h >= a.Hq;
      float ss = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) ss = fmaf(x[j][e], x[j][e], ss);
      ss = lanes_sum<LANES>(lane ? ss : 0.f);
      const float inv = rsqrtf(fmaf(ss, a.inv_hd, a.eps));
      float o[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float y0 = x[j][2 * i] * inv * (isk ? wk[2 * i] : wq[2 * i]);
        const float y1 = x[j][2 * i + 1] * inv * (isk ? wk[2 * i + 1] : wq[2 * i + 1]);
        o[2 * i] = y0 * cs[i] - y1 * sn[i];
        o[2 * i + 1] = y0 * sn[i] + y1 * cs[i];
      }
      if constexpr (ZEROS) {
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = live ? o[e] : 0.f;
      }
      if (lane && h < a.H) store8(os.at(isk, j * step), o);
    }
  }
}
template <typename T, int LANES>
__global__ __launch_bounds__(kThreads) void qk_norm_rope_kernel(Args<T> a, uint64_t blocks) {
  norm_rope<T, LANES, false>(a, blocks);
}
template <typename T, int LANES>
__global__ __launch_bounds__(kThreads) void qk_norm_rope_zeros_kernel(Args<T> a, uint64_t blocks) {
  norm_rope<T, LANES, true>(a, blocks);
}

// The gradients.  part: f32 [gridDim.x][2][hd], each workgroup's sums of d_wq and d_wk.
template <typename T, int LANES>
__global__ __launch_bounds__(kThreads, 4) void qk_norm_rope_bwd_kernel(Args<T> a, uint64_t blocks,
                                                                       float *__restrict__ part) {
  constexpr int kGroups = kThreads / LANES;
  __shared__ float s_dw[kGroups][2][8 * LANES];
  const int c = threadIdx.x % LANES, grp = threadIdx.x / LANES;
  const bool lane = 8 * c < a.hd;
  const int col = lane ? 8 * c : 0;
  Raw8<float> wq, wk;
  wq.load(a.w[0] + col), wk.load(a.w[1] + col);
  float dw[2][8];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) dw[i][e] = 0.f;
  for (uint64_t block = blockIdx.x; block < blocks; block += gridDim.x) {
    uint64_t row;
    int s;
    unit_of(a, block, kGroups, grp, &row, &s);
    if (row >= a.rows) continue;
    const uint32_t pos = position(a, (uint32_t)row);
    const bool live = pos < a.cache_rows;
    const int step = (int)a.per_row * a.hd;  // from a head to the next of the group
    const Heads<const T> xs(a.x, a.ldx, row, s * a.hd + col, a.Hq, a.hd);
    const Heads<const T> ds(a.d, a.ldd, row, s * a.hd + col, a.Hq, a.hd);
    Raw8<T> x[kHeads], d[kHeads];
#pragma unroll
    for (int j = 0; j < kHeads; ++j) {
      const int h = s + a.per_row * j, jj = h < a.H ? j : 0;
      const bool isk = s + (int)a.per_row * jj >= a.Hq;
      x[j].load(xs.at(isk, jj * step));
      d[j].load(ds.at(isk, jj * step));
    }
    const size_t at = (size_t)(live ? pos : 0) * (a.hd / 2) + col / 2;
    f32x4 cs = f32x4{0.f, 0.f, 0.f, 0.f}, sn = cs;
    if (a.cache_rows > 0) {
      cs = *reinterpret_cast<const f32x4 *>(a.cs + at);
      sn = *reinterpret_cast<const f32x4 *>(a.sn + at);
    }
    const Heads<T> os(a.out, a.ldo, row, s * a.hd + col, a.Hq, a.hd);
#pragma unroll
    for (int j = 0; j < kHeads; ++j) {
      const int h = s + a.per_row * j;
      const bool isk = h >= a.Hq;
      float g[8], ss = 0.f, tx = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        g[2 * i] = d[j][2 * i] * cs[i] + d[j][2 * i + 1] * sn[i];
        g[2 * i + 1] = d[j][2 * i + 1] * cs[i] - d[j][2 * i] * sn[i];
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        ss = fmaf(x[j][e], x[j][e], ss);
        tx = fmaf(g[e] * (isk ? wk[e] : wq[e]), x[j][e], tx);
      }
      ss = lanes_sum<LANES>(lane ? ss : 0.f);
      tx = lanes_sum<LANES>(lane ? tx : 0.f);
      const float inv = rsqrtf(fmaf(ss, a.inv_hd, a.eps));
      const float m = tx * inv * a.inv_hd;  // mean(t xh)
      float o[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float xh = x[j][e] * inv;
        o[e] = inv * (g[e] * (isk ? wk[e] : wq[e]) - xh * m);
        // A group without a position or past the last head adds nothing, whatever inv is.
        const float p = live && h < a.H ? g[e] * xh : 0.f;
        dw[0][e] += isk ? 0.f : p;
        dw[1][e] += isk ? p : 0.f;
      }
      if (lane && h < a.H) {
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = live ? o[e] : 0.f;
        store8(os.at(isk, j * step), o);
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

// d_w[v] (+)= the workgroups' sums, added in a fixed order: kCols columns a workgroup, the
// other threads of which share the rows of a column and have all their loads in flight.
constexpr int kCols = 8;
__global__ __launch_bounds__(1024) void qk_norm_dw_kernel(const float *__restrict__ part, int n,
                                                          int hd, float *d_wq, float *d_wk,
                                                          int beta) {
  constexpr int kParts = 1024 / kCols;
  __shared__ float s[16][kCols];
  const int col = threadIdx.x % kCols, r = threadIdx.x / kCols, v = blockIdx.x * kCols + col;
  float sum = 0.f;
#pragma unroll 8
  for (int i = r; i < n; i += kParts) sum += part[(size_t)i * 2 * hd + v];
  // The 8 parts of a column that a wave holds, then the 16 waves'.
#pragma unroll
  for (int m = kCols; m < 64; m <<= 1) sum += __shfl_xor(sum, m);
  if ((threadIdx.x & 63) < kCols) s[threadIdx.x >> 6][col] = sum;
  __syncthreads();
  if (threadIdx.x >= kCols) return;
  sum = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) sum += s[i][col];
  float *out = v < hd ? d_wq : d_wk;
  if (out == nullptr) return;  // a call without queries or without keys
  out += v < hd ? v : v - hd;
  *out = beta ? *out + sum : sum;
}

// Workgroups of the backward: the sums of the weights' gradients end in one row of `part`
// each.  1024 are all resident (four a CU); 256, 512 and 2048 take 40.4, 34.1 and 35.7 us where
// these take 33.3 (4 x 2048 rows, a captured forward and backward).
constexpr size_t kBwdBlocks = 1024;
int lanes_of(size_t hd) { return hd <= 32 ? 4 : hd <= 64 ? 8 : hd <= 128 ? 16 : 32; }
size_t per_row_of(size_t heads) { return cdiv(heads, (size_t)kHeads); }
size_t blocks_of(size_t rows, size_t heads, size_t hd) {
  return cdiv(rows * per_row_of(heads), (size_t)(kThreads / lanes_of(hd)));
}
size_t bwd_blocks(size_t rows, size_t heads, size_t hd) {
  const size_t blocks = blocks_of(rows, heads, hd);
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
  bool zeros;  // forward: in rows outside the tables
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
    // A side without heads is never stored; its weights are loaded from the other's.
    a.w[i] = c.heads[i] ? c.w[i] : c.w[1 - i];
  }
  a.cs = c.cs, a.sn = c.sn, a.positions = c.positions;
  a.rows = (uint32_t)c.rows, a.cache_rows = (uint32_t)c.cache_rows;
  a.pos_offset = (uint32_t)c.pos_offset, a.seq_len = (uint32_t)(c.positions ? 1 : c.seq_len);
  a.Hq = (int)c.heads[0], a.H = (int)(c.heads[0] + c.heads[1]), a.hd = (int)c.hd;
  a.per_row = (uint32_t)per_row_of(c.heads[0] + c.heads[1]);
  a.inv_hd = 1.0f / (float)c.hd, a.eps = c.eps;
  return a;
}

template <typename T, int LANES>
auto forward_kernel(bool zeros) {
  return zeros ? qk_norm_rope_zeros_kernel<T, LANES> : qk_norm_rope_kernel<T, LANES>;
}
template <typename T>
void launch_forward(const Call &c, hipStream_t s) {
  const int lanes = lanes_of(c.hd);
  const size_t blocks = blocks_of(c.rows, c.heads[0] + c.heads[1], c.hd);
  const dim3 grid((unsigned)(blocks < (1u << 20) ? blocks : 1u << 20));
  const bool zeros = c.zeros && c.positions != nullptr;  // without them no row is outside
  auto kern = lanes == 4    ? forward_kernel<T, 4>(zeros)
              : lanes == 8  ? forward_kernel<T, 8>(zeros)
              : lanes == 16 ? forward_kernel<T, 16>(zeros)
                            : forward_kernel<T, 32>(zeros);
  hipLaunchKernelGGL(kern, grid, dim3(kThreads), 0, s, args_of<T>(c),
                     (uint64_t)blocks);
}
template <typename T>
void launch_backward(const Call &c, size_t grid, float *part, hipStream_t s) {
  const int lanes = lanes_of(c.hd);
  auto kern = lanes == 4    ? qk_norm_rope_bwd_kernel<T, 4>
              : lanes == 8  ? qk_norm_rope_bwd_kernel<T, 8>
              : lanes == 16 ? qk_norm_rope_bwd_kernel<T, 16>
                            : qk_norm_rope_bwd_kernel<T, 32>;
  hipLaunchKernelGGL(kern, dim3((unsigned)grid), dim3(kThreads), 0, s, args_of<T>(c),
                     (uint64_t)blocks_of(c.rows, c.heads[0] + c.heads[1], c.hd), part);
}

int forward(const char *who, const Call &c, void *stream) {
  bool work;
  const int rc = check(who, c, false, &work);
  if (rc != PRICHS_OK || !work) return rc;
  if (c.dtype == PRICHS_DTYPE_BF16)
    launch_forward<bf16_t>(c, as_stream(stream));
  else
    launch_forward<float>(c, as_stream(stream));
  PRICHS_LAUNCH_CHECK("qk_norm_rope_forward launch");
  return PRICHS_OK;
}

}  // namespace
}  // namespace prichs

using namespace prichs;

extern "C" int prichs_qk_norm_rope_forward(
    const void *q, size_t ldq, const void *k, size_t ldk, const float *w_q, const float *w_k,
    const float *cos_cache, const float *sin_cache, size_t cache_rows, const int32_t *positions,
    size_t seq_len, size_t pos_offset, void *q_out, size_t ldqo, void *k_out, size_t ldko,
    size_t rows, size_t n_heads, size_t n_kv_heads, size_t head_dim, float eps, int dtype,
    void *stream) {
  return forward("qk_norm_rope_forward",
                 {{q, k},
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
                  dtype,
                  false},
                 stream);
}

extern "C" int prichs_qk_norm_rope_forward_zeros(
    const void *q, size_t ldq, const void *k, size_t ldk, const float *w_q, const float *w_k,
    const float *cos_cache, const float *sin_cache, size_t cache_rows, const int32_t *positions,
    size_t seq_len, size_t pos_offset, void *q_out, size_t ldqo, void *k_out, size_t ldko,
    size_t rows, size_t n_heads, size_t n_kv_heads, size_t head_dim, float eps, int dtype,
    void *stream) {
  return forward("qk_norm_rope_forward_zeros",
                 {{q, k},
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
                  dtype,
                  true},
                 stream);
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
               dtype,
               false};
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
  hipLaunchKernelGGL(qk_norm_dw_kernel, dim3((unsigned)(2 * head_dim / kCols)), dim3(1024), 0, s,
                     part, (int)blocks, (int)head_dim, n_heads ? d_wq : nullptr,
                     n_kv_heads ? d_wk : nullptr, beta);
  PRICHS_LAUNCH_CHECK("qk_norm_rope_backward weights launch");
  return PRICHS_OK;
}
