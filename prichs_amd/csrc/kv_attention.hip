// kv_attention.hip -- GQA attention of a sequence's last tokens over its paged
// 4-bit KV cache (kv_cache.hpp has the layout and the number format).
//
// All query rows that read one kv head (n_q tokens x G heads, row = token * G +
// head) form tiles of 16 rows.  A wave takes whole pages of 64 keys:
//   S^T = K Q^T     v_mfma_f32_16x16x32_bf16: a lane holds 32 head dims (16 bytes
//                   of codes, one scale) of a key, converted two at a time with
//                   their scale -- exact in bf16 -- straight into the operand; the
//                   products' k index runs over dims 32 g + 8 kk .. + 7 (g = lane /
//                   16) on both sides;
//   O^T += V^T P^T  P comes from the softmax registers: a lane holds keys 16 c +
//                   4 g .. + 3 of its query, two quads of each 32-key step, and
//                   reads dword lane % 16 of the same quads of V.  A converted pair
//                   holds two dims of one key; a byte permute of two keys' pairs
//                   gives both dims' operands, and the product's row m of block jd
//                   is dim 8 m + jd.
// Nothing goes through LDS before the waves join, there is no lane exchange but the
// row maximum, and a page is read once per row tile: 8704 bytes against 32 KB in
// bf16.  Bound by HBM where the caches are long (MI355X, 12 + 3 heads, 64 sequences
// of 16384 positions: 428 MB, more than the last-level cache holds, in 89 us, 4.8
// TB/s; 32 sequences, which it does hold, 41 us), by the latency of a page (about 2
// us from its table entry to its last product) where they are short (one token over
// 8192 positions: 8.6 us, 3.3 MB).  Some 80 scalar registers are spilled to lanes of
// vector registers (none to memory), and about 80 of a page's 650 instructions move
// them.  Three workgroups a CU hide each other's loads: a
// second set of registers for a wave's next page cost the third and was no faster
// (32 x 3000 positions 15.2 -> 16.1 us).  Tiles of 32 rows share the conversions of
// two row blocks but leave half the waves (8 x 8 queries over 4096: 15.7 us against
// 14.7; 1 x 8: 10.9 against 8.7; only 32 x 6 over 2000 gains, 18.9 to 17.6).
//
// The visible pages of a tile are dealt evenly to the waves of n_split workgroups in
// contiguous runs; the waves of a workgroup join in LDS, workgroups through the
// workspace and a second kernel (n_split > 1).  The order of both is fixed, so
// results are reproducible.
#include "attention_tile.hpp"
#include "kv_cache.hpp"

#include <algorithm>

namespace prichs {
namespace {

constexpr int kRows = 16;          // query rows of a tile
constexpr int kLdRow = kKvHd + 4;  // LDS row of joined outputs: 16 rows on distinct banks
constexpr float kLazy = 8.0f;      // log2 headroom of the lazily raised softmax max

struct AttendShape {
  int n_pages, max_pages, n_q, Hq, Hkv, window, sinks, tiles, n_split;
  float scale_log2;
};

__device__ __forceinline__ f32x4 mfma_u32(u32x4 a, u32x4 b, f32x4 c) {
  return mfma_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c);
}
// Values 2 BYTE and 2 BYTE + 1 of a dword of codes, in bf16.
template <int BYTE>
__device__ __forceinline__ uint32_t pair(uint32_t codes, float scale) {
  return __builtin_bit_cast(uint32_t,
                            __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, BYTE));
}
__device__ __forceinline__ u32x4 eight(uint32_t codes, float scale) {
  return u32x4{pair<0>(codes, scale), pair<1>(codes, scale), pair<2>(codes, scale),
               pair<3>(codes, scale)};
}

// A page of one kv head as a lane holds it.
struct PageRegs {
  u32x4 k[4];  // key 16 c + lane % 16, dims 32 g ..
  u32x4 v[4];  // quad 4 q + g, dword lane % 16 of its four keys
  uint32_t ks; // scales of k[0..3]
  u32x4 vs;    // scales of v[0..3]
};

// The workspace, where a tile's pages are split: the parts of each row's output (kKvHd
// floats), maximum and sum (2), then from here the sums of unrounded P (1).
__device__ __forceinline__ size_t sums_at(const AttendShape &sh) {
  return (size_t)gridDim.z * sh.Hkv * sh.tiles * sh.n_split * kRows * (kKvHd + 2);
}

// A part of a row (maximum mw, sum lw) joined to the row's maximum m: its weight, and
// its share of the sum.
__device__ __forceinline__ float part_weight(float mw, float m) {
  return mw == m ? 1.f : fast_exp2(mw - m);
}
__device__ __forceinline__ float part_sum(float mw, float lw, float m) {
  return mw == -INFINITY && m != -INFINITY ? 0.f : lw * part_weight(mw, m);
}

template <int kWaves, bool LSE>
__device__ __forceinline__ void kv_attend(
    const bf16_t *__restrict__ q, size_t ldq, const uint8_t *__restrict__ cache,
    const int32_t *__restrict__ table, const int32_t *__restrict__ lens, bf16_t *__restrict__ o,
    size_t ldo, float *__restrict__ lse, float *__restrict__ part_o, float2 *__restrict__ part_ml,
    const AttendShape &sh) {
  constexpr int kThreads = 64 * kWaves;
  __shared__ float s_ml[LSE ? 3 : 2][kWaves][kRows];
  __shared__ float s_o[kWaves][kRows * kLdRow];

  const int split = blockIdx.y;
  const int kvh = blockIdx.x / sh.tiles, tile = blockIdx.x - kvh * sh.tiles;
  const int b = blockIdx.z;
  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, l16 = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int G = sh.Hq / sh.Hkv, rows = sh.n_q * G;

  const int L = min(max(lens[b], 0), sh.max_pages * kKvPage);
  // Positions of the tile's first and last row, and of this lane's rows.
  const int r0 = tile * kRows, r1 = min(r0 + kRows, rows) - 1;
  const int p0 = L - sh.n_q + r0 / G, p1 = L - sh.n_q + r1 / G;
  u32x4 qf[4];
  const int lrow = min(r0 + l16, rows - 1), lq = lrow / G;
  const int pos = L - sh.n_q + lq;
  const bf16_t *qrow = q + ((size_t)b * sh.n_q + lq) * ldq +
                       (size_t)(kvh * G + lrow - lq * G) * kKvHd + 32 * g;
#pragma unroll
  for (int kk = 0; kk < 4; ++kk) qf[kk] = *reinterpret_cast<const u32x4 *>(qrow + 8 * kk);

  // The pages that some row sees: those of the sinks, then from the first row's
  // window on.
  const int first = sh.window == 0 ? 0 : max(0, p0 - sh.window + 1) / kKvPage;
  const int n_sink = min((sh.sinks + kKvPage - 1) / kKvPage, first);
  const int skip = first - n_sink;
  const int n_vis = p1 < 0 ? 0 : p1 / kKvPage + 1 - skip;
  const int64_t worker = split * kWaves + wave, workers = sh.n_split * kWaves;
  const int begin = (int)(n_vis * worker / workers), end = (int)(n_vis * (worker + 1) / workers);
  auto block_of = [&](int i) { return i >= n_sink ? i + skip : i; };
  const int32_t *row_table = table + (size_t)b * sh.max_pages;
  // Page of the i-th visible block (-1: none); the same for the whole wave.
  auto page_at = [&](int i) {
    if (i >= end) return -1;
    const int p = __builtin_amdgcn_readfirstlane(row_table[block_of(i)]);
    return p >= 0 && p < sh.n_pages ? p : -1;
  };

  f32x4 oacc[8], lsum = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int jd = 0; jd < 8; ++jd) oacc[jd] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m_ref = -INFINITY;
  // LSE: the lane's share of the sum of P before its rounding, for lse.  The output is
  // divided by the sum of the rounded P, lsum, whose errors its own cancel with.
  float psum = 0.f;
  bool seen = false;
  const u32x4 ones = u32x4{0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};

  auto part_of = [&](int page) { return cache + ((size_t)page * sh.Hkv + kvh) * kKvPart; };
  // A lane's offsets within a page; the page's address is the wave's.
  const uint32_t ko = kKvK + 64 * l16 + 16 * g, vo = kKvV + 256 * g + 16 * l16,
                 kso = kKvKScale + kKvPage * g + 4 * l16,
                 vso = kKvVScale + kKvPage * (l16 >> 2) + 16 * g;
  auto load = [&](PageRegs &x, int page) {
    if (page < 0) return;
    const uint8_t *p = part_of(page);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      x.k[c] = *reinterpret_cast<const u32x4 *>(p + ko + 1024 * c);
      x.v[c] = *reinterpret_cast<const u32x4 *>(p + vo + 1024 * c);
    }
    x.ks = *reinterpret_cast<const uint32_t *>(p + kso);
    x.vs = *reinterpret_cast<const u32x4 *>(p + vso);
  };

  auto compute = [&](PageRegs &x, int i, int page) {
    if (page < 0) return;
    const int kv0 = block_of(i) * kKvPage;
    f32x4 s[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const float sc = kv_scale((x.ks >> (8 * c)) & 255u);
      s[c] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) {
        const u32x4 kf = eight(x.k[c][kk], sc);
        s[c] = mfma_u32(kf, qf[kk], s[c]);
      }
    }
    // s[c][r]: query row l16 of the tile, key kv0 + 16 c + 4 g + r.
    const bool whole = kv0 + kKvPage - 1 <= p0 &&
                       (sh.window == 0 || p1 - kv0 < sh.window || kv0 + kKvPage <= sh.sinks);
    bool nans = false;  // a V group without finite values in a page that not all rows see
    if (!whole) {
      const int lim = pos - kv0 - 4 * g;
      const int old = sh.window == 0 ? -64 : lim - sh.window;
      const int sink = sh.sinks - kv0 - 4 * g;
      bool any = false;
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int e = 16 * c + r;
          const bool hidden = (e > lim) | ((e <= old) & (e >= sink));
          any |= !hidden;
          s[c][r] = hidden ? -INFINITY : s[c][r];
        }
      seen |= any;
      // A key that a row does not see has p = 0 there, but 0 times an infinity or
      // NaN of V is NaN: such groups (slots never written among them) count as
      // zeros here, and as NaN after the product for the rows that see them.
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (((x.vs[c] >> (8 * j)) & 255u) > 252u) {
            x.vs[c] &= ~(255u << (8 * j));
            nans = true;
          }
    } else {
      seen = true;
    }

    u32x4 pf[2];
    float mloc = -INFINITY;
#pragma unroll
    for (int c = 0; c < 4; ++c)
      mloc = vmax(vmax(vmax(mloc, s[c][0]), s[c][1]), vmax(s[c][2], s[c][3]));
    mloc = max_across_groups(mloc);
    // The reference max is raised only when a page's passes it by 2^8 in p.
    const float m_blk = mloc * sh.scale_log2;
    const bool raise = m_blk > m_ref + kLazy;
    const float m_new = raise ? m_blk : m_ref;
    const float alpha = raise ? fast_exp2(m_ref - m_new) : 1.0f;
    m_ref = m_new;
    const float neg_m = m_new == -INFINITY ? 0.f : -m_new;
    if constexpr (LSE) psum *= alpha;
#pragma unroll
    for (int ks2 = 0; ks2 < 2; ++ks2) {
      float p[8];
#pragma unroll
      for (int h2 = 0; h2 < 2; ++h2)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          p[4 * h2 + r] = fast_exp2(fmaf(s[2 * ks2 + h2][r], sh.scale_log2, neg_m));
      if constexpr (LSE)
        psum += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
      // P rounded to bf16 for the product; its sum is that of the rounded values.
      pf[ks2] = u32x4{pack_bf16x2(p[0], p[1]), pack_bf16x2(p[2], p[3]),
                      pack_bf16x2(p[4], p[5]), pack_bf16x2(p[6], p[7])};
    }
    if (__any(raise)) {
#pragma unroll
      for (int jd = 0; jd < 8; ++jd) oacc[jd] = oacc[jd] * alpha;
      lsum = lsum * alpha;
    }
    auto v_block = [&](auto byte_c, int ks2, const float (&sa)[4], const float (&sb)[4]) {
      constexpr int BYTE = decltype(byte_c)::value;
      uint32_t w[8];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        w[j] = pair<BYTE>(x.v[2 * ks2][j], sa[j]);
        w[4 + j] = pair<BYTE>(x.v[2 * ks2 + 1][j], sb[j]);
      }
      u32x4 lo, hi;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        lo[j] = __builtin_amdgcn_perm(w[2 * j + 1], w[2 * j], 0x05040100);
        hi[j] = __builtin_amdgcn_perm(w[2 * j + 1], w[2 * j], 0x07060302);
      }
      oacc[2 * BYTE] = mfma_u32(lo, pf[ks2], oacc[2 * BYTE]);
      oacc[2 * BYTE + 1] = mfma_u32(hi, pf[ks2], oacc[2 * BYTE + 1]);
    };
#pragma unroll
    for (int ks2 = 0; ks2 < 2; ++ks2) {
      float sa[4], sb[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        sa[j] = kv_scale((x.vs[2 * ks2] >> (8 * j)) & 255u);
        sb[j] = kv_scale((x.vs[2 * ks2 + 1] >> (8 * j)) & 255u);
      }
      v_block(std::integral_constant<int, 0>{}, ks2, sa, sb);
      v_block(std::integral_constant<int, 1>{}, ks2, sa, sb);
      v_block(std::integral_constant<int, 2>{}, ks2, sa, sb);
      v_block(std::integral_constant<int, 3>{}, ks2, sa, sb);
      lsum = mfma_u32(ones, pf[ks2], lsum);
    }
    if (!whole && __any(nans)) {
      // The lane's dims 8 (4 g + r) + jd are group g's.
      const uint8_t *p = part_of(page);
      bool hit = false;
#pragma unroll 1
      for (int t = 0; t < kKvPage; ++t) {
        const bool off = p[kv_v_scale_off(t, g)] > 252;
        const int key = kv0 + t;
        hit |= off & (key <= pos) &
               ((sh.window == 0) | (pos - key < sh.window) | (key < sh.sinks));
      }
#pragma unroll
      for (int jd = 0; jd < 8; ++jd)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          oacc[jd][r] = hit ? __uint_as_float(0x7fc00000u) : oacc[jd][r];
    }
  };

#pragma unroll 1
  for (int i = begin; i < end; ++i) {
    const int page = page_at(i);
    PageRegs x;
    load(x, page);
    compute(x, i, page);
  }

  // The waves join.  A score that is NaN makes the row's maximum NaN.  A row that saw
  // keys but no score above -inf has no softmax: its sum is NaN, and counts where no
  // other part of the row has a score (part_sum).
  if constexpr (LSE) {
    psum += __shfl_xor(psum, 16);
    psum += __shfl_xor(psum, 32);
  }
  if (lsum[0] != lsum[0]) m_ref = lsum[0];
  int lost = seen && m_ref == -INFINITY;
  lost |= __shfl_xor(lost, 16);
  lost |= __shfl_xor(lost, 32);
  if (g == 0) {
    s_ml[0][wave][l16] = m_ref;
    s_ml[1][wave][l16] = lost ? __uint_as_float(0x7fc00000u) : lsum[0];
    if constexpr (LSE) s_ml[2][wave][l16] = lost ? __uint_as_float(0x7fc00000u) : psum;
  }
  __syncthreads();
  float m = -INFINITY;
  for (int w = 0; w < kWaves; ++w) m = vmax(m, s_ml[0][w][l16]);
  const float f = part_weight(m_ref, m);
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int j4 = 0; j4 < 2; ++j4) {
      f32x4 t;
#pragma unroll
      for (int e = 0; e < 4; ++e) t[e] = oacc[4 * j4 + e][r] * f;
      *reinterpret_cast<f32x4 *>(&s_o[wave][l16 * kLdRow + 8 * (4 * g + r) + 4 * j4]) = t;
    }
  __syncthreads();
  for (int x = tid; x < kRows * kKvHd / 4; x += kThreads) {
    const int row = x / (kKvHd / 4), d = 4 * (x - row * (kKvHd / 4));
    if (r0 + row > r1) break;
    float m = -INFINITY, l = 0.f, ls = 0.f;
    for (int w = 0; w < kWaves; ++w) m = vmax(m, s_ml[0][w][row]);
    f32x4 t = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int w = 0; w < kWaves; ++w) {
      const float mw = s_ml[0][w][row];
      l += part_sum(mw, s_ml[1][w][row], m);
      if constexpr (LSE) ls += part_sum(mw, s_ml[2][w][row], m);
      t = t + *reinterpret_cast<const f32x4 *>(&s_o[w][row * kLdRow + d]);
    }
    if (sh.n_split > 1) {
      const size_t at =
          ((((size_t)b * sh.Hkv + kvh) * sh.tiles + tile) * sh.n_split + split) * kRows + row;
      *reinterpret_cast<f32x4 *>(part_o + at * kKvHd + d) = t;
      if (d == 0) part_ml[at] = make_float2(m, l);
      if (LSE && d == 0) part_o[sums_at(sh) + at] = ls;
      continue;
    }
    const int r = r0 + row, iq = r / G, h = kvh * G + r - iq * G;
    const float inv = l == 0.f ? 0.f : 1.0f / l;  // l = 0: no key seen
    uint2 u;
    u.x = pack_bf16x2(t[0] * inv, t[1] * inv);
    u.y = pack_bf16x2(t[2] * inv, t[3] * inv);
    *reinterpret_cast<uint2 *>(o + ((size_t)b * sh.n_q + iq) * ldo + (size_t)h * kKvHd + d) = u;
    if (LSE && d == 0)
      lse[((size_t)b * sh.Hq + h) * sh.n_q + iq] = (m + log2f(ls)) * 0.6931471805599453f;
  }
}

template <int kWaves>
__global__ __launch_bounds__(64 * kWaves, kWaves == 4 ? 3 : 2) void kv_attend_kernel(
    const bf16_t *__restrict__ q, size_t ldq, const uint8_t *__restrict__ cache,
    const int32_t *__restrict__ table, const int32_t *__restrict__ lens, bf16_t *__restrict__ o,
    size_t ldo, float *__restrict__ lse, float *__restrict__ part_o, float2 *__restrict__ part_ml,
    AttendShape sh) {
  kv_attend<kWaves, false>(q, ldq, cache, table, lens, o, ldo, lse, part_o, part_ml, sh);
}
// With lse: 10 registers more, and 0.2 to 1 us a call (one token over 8192 positions 8.6 ->
// 9.1 us, 32 x 3000 16.1 -> 16.6, 8 x 5 over 4096 14.7 -> 15.3, 2 x 256 over 4352 35.9 -> 36.9).
template <int kWaves>
__global__ __launch_bounds__(64 * kWaves, kWaves == 4 ? 3 : 2) void kv_attend_lse_kernel(
    const bf16_t *__restrict__ q, size_t ldq, const uint8_t *__restrict__ cache,
    const int32_t *__restrict__ table, const int32_t *__restrict__ lens, bf16_t *__restrict__ o,
    size_t ldo, float *__restrict__ lse, float *__restrict__ part_o, float2 *__restrict__ part_ml,
    AttendShape sh) {
  kv_attend<kWaves, true>(q, ldq, cache, table, lens, o, ldo, lse, part_o, part_ml, sh);
}

// Joins the splits of a query row: KG groups of 32 threads, thread d4 of group k
// taking dims 4 d4 .. + 3 of splits k, k + KG, ..; all loads of up to 8 splits are
// in flight at once (the partial results come from other dies' caches).
template <int KG, bool LSE>
__device__ __forceinline__ void kv_join(
    const float *__restrict__ part_o, const float2 *__restrict__ part_ml, bf16_t *__restrict__ o,
    size_t ldo, float *__restrict__ lse, const AttendShape &sh) {
  __shared__ f32x4 s_o[8][32];
  __shared__ float2 s_ml[8];
  __shared__ float s_s[8];
  const int G = sh.Hq / sh.Hkv, rows = sh.n_q * G;
  const int d4 = threadIdx.x & 31, slot = threadIdx.x >> 5, k = slot % KG;
  const int r = blockIdx.x * (8 / KG) + slot / KG;
  const int kvh = blockIdx.y, b = blockIdx.z;
  if (KG == 1 && r >= rows) return;  // with KG = 8 the grid is the rows
  const int tile = r / kRows, row = r - tile * kRows;
  const size_t base = (((size_t)b * sh.Hkv + kvh) * sh.tiles + tile) * sh.n_split * kRows + row;
  float m = -INFINITY, l = 0.f, ls = 0.f;
  f32x4 t = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int s0 = k; s0 < sh.n_split; s0 += 8 * KG) {
    f32x4 p[8];
    float2 ml[8];
    float ps[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int s = s0 + j * KG;
      ml[j] = make_float2(-INFINITY, 0.f);
      p[j] = f32x4{0.f, 0.f, 0.f, 0.f};
      ps[j] = 0.f;
      if (s < sh.n_split) {
        const size_t at = base + (size_t)s * kRows;
        ml[j] = part_ml[at];
        if constexpr (LSE) ps[j] = part_o[sums_at(sh) + at];
        p[j] = *reinterpret_cast<const f32x4 *>(part_o + at * kKvHd + 4 * d4);
      }
    }
    float m2 = m;
#pragma unroll
    for (int j = 0; j < 8; ++j) m2 = vmax(m2, ml[j].x);
    l = part_sum(m, l, m2);
    ls = part_sum(m, ls, m2);
    t = t * part_weight(m, m2);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      l += part_sum(ml[j].x, ml[j].y, m2);
      ls += part_sum(ml[j].x, ps[j], m2);
      t = t + p[j] * part_weight(ml[j].x, m2);
    }
    m = m2;
  }
  if (KG > 1) {
    s_o[slot][d4] = t;
    if (d4 == 0) s_ml[slot] = make_float2(m, l);
    if (LSE && d4 == 0) s_s[slot] = ls;
    __syncthreads();
    if (k != 0) return;
    m = -INFINITY;
#pragma unroll
    for (int j = 0; j < KG; ++j) m = vmax(m, s_ml[j].x);
    l = ls = 0.f;
    t = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < KG; ++j) {
      l += part_sum(s_ml[j].x, s_ml[j].y, m);
      ls += part_sum(s_ml[j].x, s_s[j], m);
      t = t + s_o[j][d4] * part_weight(s_ml[j].x, m);
    }
  }
  const int iq = r / G, h = kvh * G + r - iq * G;
  const float inv = l == 0.f ? 0.f : 1.0f / l;  // l = 0: no key seen
  uint2 u;
  u.x = pack_bf16x2(t[0] * inv, t[1] * inv);
  u.y = pack_bf16x2(t[2] * inv, t[3] * inv);
  *reinterpret_cast<uint2 *>(o + ((size_t)b * sh.n_q + iq) * ldo + (size_t)h * kKvHd + 4 * d4) = u;
  if (LSE && d4 == 0)
    lse[((size_t)b * sh.Hq + h) * sh.n_q + iq] = (m + log2f(ls)) * 0.6931471805599453f;
}
template <int KG>
__global__ __launch_bounds__(256) void kv_join_kernel(
    const float *__restrict__ part_o, const float2 *__restrict__ part_ml, bf16_t *__restrict__ o,
    size_t ldo, float *__restrict__ lse, AttendShape sh) {
  kv_join<KG, false>(part_o, part_ml, o, ldo, lse, sh);
}
template <int KG>
__global__ __launch_bounds__(256) void kv_join_lse_kernel(
    const float *__restrict__ part_o, const float2 *__restrict__ part_ml, bf16_t *__restrict__ o,
    size_t ldo, float *__restrict__ lse, AttendShape sh) {
  kv_join<KG, true>(part_o, part_ml, o, ldo, lse, sh);
}

// Pages up to which one workgroup of 8 waves takes a tile without a second kernel:
// a page costs a wave some 2 us, the second kernel 2.5 on the device and 4 on the
// host.  One token over 8 pages 7.4 -> 6.1 us (graph), over 16 pages 7.4 -> 8.2
// (called from Python 15.2 -> 11), 32 and 80 sequences over 16 pages 9.2 -> 8.4 and
// 14.6 -> 10.6, 32 over 32 pages 11.1 -> 13.3.
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
