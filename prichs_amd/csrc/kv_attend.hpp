// kv_attend.hpp -- the tiles of attention over the paged 4-bit KV cache: rows that share
// keys, and the join of their parts.  kv_attention.hip calls them for each sequence by
// itself, kv_shared_attention.hip for groups of sequences that share pages.
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
// of 16384 positions: 428 MB, more than the last-level cache holds, in 87 us, 4.9
// TB/s; 32 sequences, which it does hold, 40 us), by the latency of a page where they
// are short (one token over 8192 positions: 8.2 us, 3.3 MB).  K and V of a wave's next
// page take the registers of this one's as soon as its products are formed (32 x 6000
// windowed 17.5 -> 16 us, 2 x 256 over 4352 26 -> 24, with what follows); a second set of
// registers cost the third workgroup a CU and was no faster.  Masks are bit fields: as
// comparisons their results took so many scalar registers that some 80 others were held
// in lanes of vector registers, which 80 of a page's 650 instructions moved.  19 to 27 are
// held so now, none of which is read back among a page's products.  The kernels of two kinds of
// workgroup (kv_shared_kernel) hold 48 to 54 with tiles of 16 rows, whose loop over shared pages
// reads some 24 back a page, and 79 to 90 with tiles of 32, whose loop reads hardly any.
//
// The visible pages of a tile are dealt evenly to the waves of n_split workgroups in
// contiguous runs; the waves of a workgroup join in LDS, workgroups through the
// workspace and a second kernel (n_split > 1).  The order of both is fixed, so
// results are reproducible.
#pragma once

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

// Bit e: whether a row sees key e from some first key on, for a row at position `lim` from
// that key, and sinks up to key `sink` (exclusive).
__device__ __forceinline__ uint64_t bits_below(int n) {
  return n >= 64 ? ~0ull : (1ull << max(n, 0)) - 1;
}
__device__ __forceinline__ uint64_t visible_keys(int lim, int window, int sink) {
  const uint64_t old = window == 0 ? 0 : bits_below(lim - window + 1) & ~bits_below(sink);
  return bits_below(lim + 1) & ~old;
}
// The score, or -inf where bit e of `vis` is not set: without comparisons, whose results
// would take a pair of scalar registers each.
__device__ __forceinline__ float or_hidden(uint64_t vis, int e, float s) {
  const uint32_t half = e < 32 ? (uint32_t)vis : (uint32_t)(vis >> 32);
  const uint32_t m = (uint32_t)__builtin_amdgcn_sbfe((int)half, e & 31, 1);
  return __uint_as_float((m & __float_as_uint(s)) | (~m & 0xff800000u));
}
// The top bit of each byte of x that is greater than 252.
__device__ __forceinline__ uint32_t bytes_past_252(uint32_t x) {
  return ((x & 0x7f7f7f7fu) + 0x03030303u) & x & 0x80808080u;
}

// A page of one kv head as a lane holds it.
struct PageRegs {
  u32x4 k[4];  // key 16 c + lane % 16, dims 32 g ..
  u32x4 v[4];  // quad 4 q + g, dword lane % 16 of its four keys
  uint32_t ks; // scales of k[0..3]
  u32x4 vs;    // scales of v[0..3]
};

// Groups of sequences that share their first pages (prichs_kv_cache_shared_attention).  A
// launch then has two kinds of workgroup: splits of a group's tiles over its shared pages,
// and splits of each sequence's tiles over its own.  Each writes the parts of its rows
// into a slot of its own, split_p slots for shared and split_s for own pages.  Or, where
// there are few pages, one kind: a sequence's tile over all its pages, the shared ones
// where its group's first sequence names them.
enum { kWholeRole, kSharedRole, kOwnRole, kRowRole };  // a call without groups; these kinds
struct Groups {
  const int32_t *start, *shared;
  int n, batch;
  int tiles_p, split_p, split_s;  // tiles over shared pages at most, of one kv head
};
// Workgroups over shared pages: an equal number on each of the eight dies, on which
// workgroup `id` runs by id % 8, so that tiles that read the same pages (of one kv head and
// split) do so through one L2.
__host__ __device__ __forceinline__ int on_a_die(int kv_heads, const Groups &gr) {
  return (kv_heads * gr.tiles_p * gr.split_p + 7) / 8;
}
__device__ __forceinline__ int shared_workgroups(const AttendShape &sh, const Groups &gr) {
  return 8 * on_a_die(sh.Hkv, gr);
}

// Whole pages that `positions` cover.
__device__ __forceinline__ int whole_pages(int positions, int max_pages) {
  return min(max(positions, 0) / kKvPage, max_pages);
}
// A start counts as no less than those before it and lies in 0 .. batch, so that groups
// never overlap, whatever the arrays hold.
//
// Shared pages of sequence b: its group ends at the first start past b.  Without groups
// there may be no starts.  *first (where wanted): the group's first sequence.
__device__ __forceinline__ int shared_pages_of(const Groups &gr, int b, int max_pages,
                                               int *first = nullptr) {
  if (gr.n == 0) return 0;
  const int lane = threadIdx.x & 63;
  int low = 0;  // the group starts at the greatest start up to b
  for (int base = 0; base <= gr.n; base += 64) {
    const int i = base + lane;
    const int start = i <= gr.n ? gr.start[i] : 0x7fffffff;
    const int before = i >= 1 && i <= gr.n ? gr.shared[i - 1] : 0;  // of the group that ends here
    const uint64_t past = __ballot(start > b);
    const int at = past == 0 ? 64 : __ffsll((unsigned long long)past) - 1;
    if (first != nullptr) {
      int s = lane < at ? start : 0;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) s = max(s, __shfl_xor(s, d));
      low = max(low, s);
      *first = __builtin_amdgcn_readfirstlane(low);
    }
    if (past != 0) return whole_pages(__builtin_amdgcn_readlane(before, at), max_pages);
  }
  return 0;
}
// The group of the `tile`-th tile of `per` rows over shared pages (seq_rows rows a
// sequence): its first sequence, its rows, its shared pages and the tile's number in it.
// false: there are fewer tiles.
__device__ __forceinline__ bool shared_tile(const Groups &gr, int tile, int per, int seq_rows,
                                            int max_pages, int *first, int *rows, int *pages,
                                            int *nth) {
  const int lane = threadIdx.x & 63;
  int before = 0, low = 0;
  for (int base = 0; base < gr.n; base += 64) {
    const int i = base + lane;
    int s = i < gr.n ? min(max(gr.start[i], 0), gr.batch) : 0;
    int e = i < gr.n ? min(max(gr.start[i + 1], 0), gr.batch) : 0;
    const int P = i < gr.n ? whole_pages(gr.shared[i], max_pages) : 0;
    s = max(s, low);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int y = __shfl_up(s, d);
      if (lane >= d) s = max(s, y);
    }
    e = max(e, s);
    const int n = i < gr.n ? (e - s) * seq_rows : 0, t = P > 0 ? (n + per - 1) / per : 0;
    int c = t;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int y = __shfl_up(c, d);
      if (lane >= d) c += y;
    }
    const uint64_t past = __ballot(before + c > tile);
    if (past != 0) {
      const int j = __ffsll((unsigned long long)past) - 1;
      *first = __builtin_amdgcn_readlane(s, j);
      *rows = __builtin_amdgcn_readlane(n, j);
      *pages = __builtin_amdgcn_readlane(P, j);
      *nth = tile - (before + __builtin_amdgcn_readlane(c - t, j));
      return true;
    }
    before += __builtin_amdgcn_readlane(c, 63);
    low = __builtin_amdgcn_readlane(e, 63);
  }
  return false;
}
// Rows of a call: the distance of two slots.
__device__ __forceinline__ size_t all_rows(const AttendShape &sh, const Groups &gr) {
  return (size_t)gr.batch * sh.n_q * sh.Hq;
}

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

// LDS that the waves of a workgroup join in, 16 rows at a time.
template <int kWaves> struct JoinLds {
  float o[kWaves][kRows * kLdRow];
  float ml[3][kWaves][kRows];
};

// A workgroup's tile of 16 NB rows; NB > 1 (with groups) shares a page's conversions among
// more rows.
template <int kWaves, bool LSE, int ROLE = kWholeRole, int NB = 1>
__device__ __forceinline__ void kv_attend(
    const bf16_t *__restrict__ q, size_t ldq, const uint8_t *__restrict__ cache,
    const int32_t *__restrict__ table, const int32_t *__restrict__ lens, bf16_t *__restrict__ o,
    size_t ldo, float *__restrict__ lse, float *__restrict__ part_o, float2 *__restrict__ part_ml,
    const AttendShape &sh, JoinLds<kWaves> &s, const Groups &gr) {
  constexpr bool kGroups = ROLE == kSharedRole || ROLE == kOwnRole;
  static_assert(NB == 1 || kGroups, "whole sequences have tiles of 16 rows");
  constexpr int kThreads = 64 * kWaves, kTileRows = 16 * NB;
  auto &s_ml = s.ml;
  auto &s_o = s.o;

  int split = blockIdx.y, n_split = sh.n_split;
  int kvh = blockIdx.x / sh.tiles, tile = blockIdx.x - kvh * sh.tiles;
  int b = blockIdx.z;  // with groups: the first sequence of the tile's rows
  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, l16 = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int G = sh.Hq / sh.Hkv;
  int rows = sh.n_q * G;
  const int seq_rows = rows;
  // With groups: the pages that count, and the slot of the parts.
  int lo = 0, hi = sh.max_pages, slot = 0;
  bool alone = false;  // no workgroup writes the slots for shared pages of these rows
  if constexpr (ROLE == kSharedRole) {
    const int id = (blockIdx.x & 7) * on_a_die(sh.Hkv, gr) + (blockIdx.x >> 3);
    const int pages = id / gr.tiles_p;  // kv head and split
    kvh = pages / gr.split_p, split = pages - kvh * gr.split_p;
    if (kvh >= sh.Hkv || !shared_tile(gr, id - pages * gr.tiles_p, kTileRows, seq_rows,
                                      sh.max_pages, &b, &rows, &hi, &tile))
      return;
    n_split = gr.split_p;
    slot = split;
  } else if constexpr (ROLE == kOwnRole) {
    int id = blockIdx.x - shared_workgroups(sh, gr);
    split = id % gr.split_s, id /= gr.split_s;
    tile = id % sh.tiles, id /= sh.tiles;
    b = id / sh.Hkv;
    kvh = id - b * sh.Hkv;
    lo = shared_pages_of(gr, b, sh.max_pages);
    alone = lo == 0 && split == 0;
    n_split = gr.split_s;
    slot = gr.split_p + split;
  }

  // Positions of the tile's first and last row (with groups the least and the greatest),
  // and of this lane's rows.
  const int r0 = tile * kTileRows, r1 = min(r0 + kTileRows, rows) - 1;
  u32x4 qf[NB][4];
  int pos[NB], p0, p1;
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    const int lrow = min(r0 + 16 * nb + l16, rows - 1);
    const int lseq = ROLE == kSharedRole ? lrow / seq_rows : 0,
              lq = (lrow - lseq * seq_rows) / G;
    const int L = min(max(lens[b + lseq], 0), sh.max_pages * kKvPage);
    pos[nb] = L - sh.n_q + lq;
    if constexpr (ROLE == kSharedRole) {
      p0 = nb == 0 ? pos[0] : min(p0, pos[nb]);
      p1 = nb == 0 ? pos[0] : max(p1, pos[nb]);
    } else {
      p0 = L - sh.n_q + r0 / G, p1 = L - sh.n_q + r1 / G;
    }
    const bf16_t *qrow = q + ((size_t)(b + lseq) * sh.n_q + lq) * ldq +
                         (size_t)(kvh * G + lrow - lseq * seq_rows - lq * G) * kKvHd + 32 * g;
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) qf[nb][kk] = *reinterpret_cast<const u32x4 *>(qrow + 8 * kk);
  }
  if constexpr (ROLE == kSharedRole) {
#pragma unroll
    for (int d = 1; d < 16; d <<= 1) {
      p0 = min(p0, __shfl_xor(p0, d));
      p1 = max(p1, __shfl_xor(p1, d));
    }
    p0 = __builtin_amdgcn_readfirstlane(p0);
    p1 = __builtin_amdgcn_readfirstlane(p1);
  }

  // The pages that some row sees: those of the sinks, then from the first row's
  // window on.
  const int first = sh.window == 0 ? 0 : max(0, p0 - sh.window + 1) / kKvPage;
  int n_sink = min((sh.sinks + kKvPage - 1) / kKvPage, first);
  int skip = first - n_sink;
  int n_vis = p1 < 0 ? 0 : p1 / kKvPage + 1 - skip;
  if constexpr (kGroups) {
    // Of both runs of pages what lies in lo .. hi - 1.
    const int from = max(first, lo), to = min(p1 < 0 ? 0 : p1 / kKvPage + 1, hi);
    n_sink = max(min(n_sink, hi) - lo, 0);
    skip = from - n_sink;
    n_vis = n_sink + max(to - from, 0);
  }
  // Without a window the shared pages are dealt whatever the rows' positions, whose loads
  // they then need not wait for; a row that ends before them sees none of the rest.
  if (ROLE == kSharedRole && sh.window == 0) n_sink = skip = 0, n_vis = hi;
  const int64_t worker = split * kWaves + wave, workers = n_split * kWaves;
  const int begin = (int)(n_vis * worker / workers), end = (int)(n_vis * (worker + 1) / workers);
  auto block_of = [&](int i) { return i >= n_sink ? i + skip : i + lo; };
  const int32_t *row_table = table + (size_t)b * sh.max_pages, *first_table = row_table;
  int n_shared = 0;  // kRowRole: pages that stand in first_table
  if constexpr (ROLE == kRowRole) {
    int first_b = 0;
    n_shared = shared_pages_of(gr, b, sh.max_pages, &first_b);
    if (n_shared > 0) first_table = table + (size_t)first_b * sh.max_pages;
  }
  auto entry = [&](int block) {
    return ROLE == kRowRole && block < n_shared ? first_table[block] : row_table[block];
  };
  // The wave's next visible block whose page exists (end: none), and its page.  It holds 64
  // entries of the table at a time, and a bit for each that names a page.
  int ids = -1, base = begin - 64;
  uint64_t left = 0;
  auto next_page = [&](int *page) {
    while (left == 0) {
      base += 64;
      if (base >= end) return end;
      ids = base + lane < end ? entry(block_of(base + lane)) : -1;
      left = __ballot(ids >= 0 && ids < sh.n_pages);
    }
    const int at = __ffsll((unsigned long long)left) - 1;
    left &= left - 1;
    *page = __builtin_amdgcn_readlane(ids, at);
    return base + at;
  };

  f32x4 oacc[8][NB], lsum[NB];
  float m_ref[NB];
  // LSE: the lane's share of the sum of P before its rounding, for lse.  The output is
  // divided by the sum of the rounded P, lsum, whose errors its own cancel with.
  float psum[NB];
  bool seen[NB];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
    for (int jd = 0; jd < 8; ++jd) oacc[jd][nb] = f32x4{0.f, 0.f, 0.f, 0.f};
    lsum[nb] = f32x4{0.f, 0.f, 0.f, 0.f};
    m_ref[nb] = -INFINITY;
    psum[nb] = 0.f;
    seen[nb] = false;
  }
  const u32x4 ones = u32x4{0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};

  auto part_of = [&](int page) { return cache + ((size_t)page * sh.Hkv + kvh) * kKvPart; };
  // A lane's offsets within a page; the page's address is the wave's.
  const uint32_t ko = kKvK + 64 * l16 + 16 * g, vo = kKvV + 256 * g + 16 * l16,
                 kso = kKvKScale + kKvPage * g + 4 * l16,
                 vso = kKvVScale + kKvPage * (l16 >> 2) + 16 * g;
  auto load_k = [&](PageRegs &x, int page) {
    const uint8_t *p = part_of(page);
#pragma unroll
    for (int c = 0; c < 4; ++c) x.k[c] = *reinterpret_cast<const u32x4 *>(p + ko + 1024 * c);
    x.ks = *reinterpret_cast<const uint32_t *>(p + kso);
  };
  auto load_v = [&](PageRegs &x, int page) {
    const uint8_t *p = part_of(page);
#pragma unroll
    for (int c = 0; c < 4; ++c) x.v[c] = *reinterpret_cast<const u32x4 *>(p + vo + 1024 * c);
    x.vs = *reinterpret_cast<const u32x4 *>(p + vso);
  };

  // K and V of a page each take the registers of the page before as soon as its products
  // are formed, so that they are on their way during the other half of a page's work.
  auto compute = [&](PageRegs &x, int i, int page, int next) {
    const int kv0 = block_of(i) * kKvPage;
    f32x4 s[4][NB];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const float sc = kv_scale((x.ks >> (8 * c)) & 255u);
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) s[c][nb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) {
        const u32x4 kf = eight(x.k[c][kk], sc);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) s[c][nb] = mfma_u32(kf, qf[nb][kk], s[c][nb]);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    if (next >= 0) load_k(x, next);
    __builtin_amdgcn_sched_barrier(0);
    // s[c][nb][r]: query row 16 nb + l16 of the tile, key kv0 + 16 c + 4 g + r.
    const bool whole = kv0 + kKvPage - 1 <= p0 &&
                       (sh.window == 0 || p1 - kv0 < sh.window || kv0 + kKvPage <= sh.sinks);
    bool nans = false;  // a V group without finite values in a page that not all rows see
    if (!whole) {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        const uint64_t vis = visible_keys(pos[nb] - kv0 - 4 * g, sh.window, sh.sinks - kv0 - 4 * g);
        seen[nb] |= (vis & 0x000f000f000f000full) != 0;  // the lane's keys are 16 c + r, r < 4
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int r = 0; r < 4; ++r) s[c][nb][r] = or_hidden(vis, 16 * c + r, s[c][nb][r]);
      }
      // A key that a row does not see has p = 0 there, but 0 times an infinity or
      // NaN of V is NaN: such groups (slots never written among them) count as
      // zeros here, and as NaN after the product for the rows that see them (past the last
      // row's position there are none).
      uint32_t bad[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) bad[c] = bytes_past_252(x.vs[c]);
      if (__any((bad[0] | bad[1] | bad[2] | bad[3]) != 0)) {
        const int last = p1 - kv0 - 4 * g;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          x.vs[c] &= ~((bad[c] >> 7) * 255u);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            nans |= ((bad[c] >> (8 * j + 7)) & 1) != 0 && 16 * c + j <= last;
        }
      }
    } else {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) seen[nb] = true;
    }

    u32x4 pf[NB][2];
    float alpha[NB];
    bool any_raise = false;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      float mloc = -INFINITY;
#pragma unroll
      for (int c = 0; c < 4; ++c)
        mloc = vmax(vmax(vmax(mloc, s[c][nb][0]), s[c][nb][1]), vmax(s[c][nb][2], s[c][nb][3]));
      mloc = max_across_groups(mloc);
      // The reference max is raised only when a page's passes it by 2^8 in p.
      const float m_blk = mloc * sh.scale_log2;
      const bool raise = m_blk > m_ref[nb] + kLazy;
      any_raise |= raise;
      const float m_new = raise ? m_blk : m_ref[nb];
      alpha[nb] = raise ? fast_exp2(m_ref[nb] - m_new) : 1.0f;
      m_ref[nb] = m_new;
      const float neg_m = m_new == -INFINITY ? 0.f : -m_new;
      if constexpr (LSE) psum[nb] *= alpha[nb];
#pragma unroll
      for (int ks2 = 0; ks2 < 2; ++ks2) {
        float p[8];
#pragma unroll
        for (int h2 = 0; h2 < 2; ++h2)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            p[4 * h2 + r] = fast_exp2(fmaf(s[2 * ks2 + h2][nb][r], sh.scale_log2, neg_m));
        if constexpr (LSE)
          psum[nb] += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
        // P rounded to bf16 for the product, whose other operand is exact in bf16; its sum is
        // that of the rounded values.  With the output's rounding (0.0017 of the norm) outputs
        // are off by 0.0021 to 0.0023.  P in two parts would take half as many products again.
        pf[nb][ks2] = u32x4{pack_bf16x2(p[0], p[1]), pack_bf16x2(p[2], p[3]),
                            pack_bf16x2(p[4], p[5]), pack_bf16x2(p[6], p[7])};
      }
    }
    if (__any(any_raise)) {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
        for (int jd = 0; jd < 8; ++jd) oacc[jd][nb] = oacc[jd][nb] * alpha[nb];
        lsum[nb] = lsum[nb] * alpha[nb];
      }
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
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        oacc[2 * BYTE][nb] = mfma_u32(lo, pf[nb][ks2], oacc[2 * BYTE][nb]);
        oacc[2 * BYTE + 1][nb] = mfma_u32(hi, pf[nb][ks2], oacc[2 * BYTE + 1][nb]);
      }
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
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) lsum[nb] = mfma_u32(ones, pf[nb][ks2], lsum[nb]);
    }
    __builtin_amdgcn_sched_barrier(0);
    if (next >= 0) load_v(x, next);
    __builtin_amdgcn_sched_barrier(0);
    if (!whole && __any(nans)) {
      // The lane's dims 8 (4 g + r) + jd are group g's.
      const uint8_t *p = part_of(page);
      bool hit[NB] = {};
#pragma unroll 1
      for (int t = 0; t < kKvPage; ++t) {
        const bool off = p[kv_v_scale_off(t, g)] > 252;
        const int key = kv0 + t;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
          hit[nb] |= off & (key <= pos[nb]) &
                     ((sh.window == 0) | (pos[nb] - key < sh.window) | (key < sh.sinks));
      }
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int jd = 0; jd < 8; ++jd)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            oacc[jd][nb][r] = hit[nb] ? __uint_as_float(0x7fc00000u) : oacc[jd][nb][r];
    }
  };

  int page = -1;
  int i = next_page(&page);
  if (i < end) {
    PageRegs x;
    load_k(x, page);
    load_v(x, page);
#pragma unroll 1
    while (i < end) {
      int page2 = -1;
      const int j = next_page(&page2);
      compute(x, i, page, page2);
      i = j, page = page2;
    }
  }

  // The waves join.  A score that is NaN makes the row's maximum NaN.  A row that saw
  // keys but no score above -inf has no softmax: its sum is NaN, and counts where no
  // other part of the row has a score (part_sum).
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    if (nb > 0) __syncthreads();  // the rows before have been read
    if constexpr (LSE) {
      psum[nb] += __shfl_xor(psum[nb], 16);
      psum[nb] += __shfl_xor(psum[nb], 32);
    }
    float mr = m_ref[nb];
    if (lsum[nb][0] != lsum[nb][0]) mr = lsum[nb][0];
    int lost = seen[nb] && mr == -INFINITY;
    lost |= __shfl_xor(lost, 16);
    lost |= __shfl_xor(lost, 32);
    if (g == 0) {
      s_ml[0][wave][l16] = mr;
      s_ml[1][wave][l16] = lost ? __uint_as_float(0x7fc00000u) : lsum[nb][0];
      if constexpr (LSE) s_ml[2][wave][l16] = lost ? __uint_as_float(0x7fc00000u) : psum[nb];
    }
    __syncthreads();
    float m = -INFINITY;
    for (int w = 0; w < kWaves; ++w) m = vmax(m, s_ml[0][w][l16]);
    const float f = part_weight(mr, m);
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int j4 = 0; j4 < 2; ++j4) {
        f32x4 t;
#pragma unroll
        for (int e = 0; e < 4; ++e) t[e] = oacc[4 * j4 + e][nb][r] * f;
        *reinterpret_cast<f32x4 *>(&s_o[wave][l16 * kLdRow + 8 * (4 * g + r) + 4 * j4]) = t;
      }
    __syncthreads();
    for (int x = tid; x < kRows * kKvHd / 4; x += kThreads) {
      const int row = x / (kKvHd / 4), d = 4 * (x - row * (kKvHd / 4));
      const int r = r0 + 16 * nb + row;
      if (r > r1) break;
      float m = -INFINITY, l = 0.f, ls = 0.f;
      for (int w = 0; w < kWaves; ++w) m = vmax(m, s_ml[0][w][row]);
      f32x4 t = f32x4{0.f, 0.f, 0.f, 0.f};
      for (int w = 0; w < kWaves; ++w) {
        const float mw = s_ml[0][w][row];
        l += part_sum(mw, s_ml[1][w][row], m);
        if constexpr (LSE) ls += part_sum(mw, s_ml[2][w][row], m);
        t = t + *reinterpret_cast<const f32x4 *>(&s_o[w][row * kLdRow + d]);
      }
      const int iq = r / G, h = kvh * G + r - iq * G;  // iq: token from b's first
      if constexpr (kGroups) {
        const size_t n = all_rows(sh, gr), id = ((size_t)b * sh.n_q + iq) * sh.Hq + h;
        const size_t at = slot * n + id;
        // A part without keys is known by its maximum and sum.
        if (m != -INFINITY || l != 0.f)
          *reinterpret_cast<f32x4 *>(part_o + at * kKvHd + d) = t;
        if (d == 0) {
          float *sums = part_o + n * (gr.split_p + gr.split_s) * (kKvHd + 2);
          part_ml[at] = make_float2(m, l);
          if (LSE) sums[at] = ls;
          if (alone)
            for (int s = 0; s < gr.split_p; ++s) {
              part_ml[s * n + id] = make_float2(-INFINITY, 0.f);
              if (LSE) sums[s * n + id] = 0.f;
            }
        }
        continue;
      }
      if (sh.n_split > 1) {
        const size_t at =
            ((((size_t)b * sh.Hkv + kvh) * sh.tiles + tile) * sh.n_split + split) * kRows + row;
        *reinterpret_cast<f32x4 *>(part_o + at * kKvHd + d) = t;
        if (d == 0) part_ml[at] = make_float2(m, l);
        if (LSE && d == 0) part_o[sums_at(sh) + at] = ls;
        continue;
      }
      const float inv = l == 0.f ? 0.f : 1.0f / l;  // l = 0: no key seen
      uint2 u;
      u.x = pack_bf16x2(t[0] * inv, t[1] * inv);
      u.y = pack_bf16x2(t[2] * inv, t[3] * inv);
      *reinterpret_cast<uint2 *>(o + ((size_t)b * sh.n_q + iq) * ldo + (size_t)h * kKvHd + d) = u;
      if (LSE && d == 0)
        lse[((size_t)b * sh.Hq + h) * sh.n_q + iq] = (m + log2f(ls)) * 0.6931471805599453f;
    }
  }
}

// Joins the splits of a query row: KG groups of 32 threads, thread d4 of group k
// taking dims 4 d4 .. + 3 of splits k, k + KG, ..; all loads of up to 8 splits are
// in flight at once (the partial results come from other dies' caches).
template <int KG, bool LSE, bool GROUPS = false>
__device__ __forceinline__ void kv_join(
    const float *__restrict__ part_o, const float2 *__restrict__ part_ml, bf16_t *__restrict__ o,
    size_t ldo, float *__restrict__ lse, const AttendShape &sh, const Groups &gr) {
  __shared__ f32x4 s_o[8][32];
  __shared__ float2 s_ml[8];
  __shared__ float s_s[8];
  const int d4 = threadIdx.x & 31, slot = threadIdx.x >> 5, k = slot % KG;
  const int r = blockIdx.x * (8 / KG) + slot / KG;
  // The row's parts: the first, and the distance to the next.
  size_t base, step = kRows, sums;
  int b = blockIdx.z, iq, h, n_split = sh.n_split;
  if constexpr (GROUPS) {
    step = all_rows(sh, gr);
    if ((size_t)r >= step) return;  // with KG = 8 the grid is the rows
    iq = r / sh.Hq, h = r - iq * sh.Hq;
    b = iq / sh.n_q, iq -= b * sh.n_q;
    n_split = gr.split_p + gr.split_s;
    base = r;
    sums = step * n_split * (kKvHd + 2);
  } else {
    const int G = sh.Hq / sh.Hkv, rows = sh.n_q * G, kvh = blockIdx.y;
    if (KG == 1 && r >= rows) return;  // with KG = 8 the grid is the rows
    const int tile = r / kRows, row = r - tile * kRows;
    base = (((size_t)b * sh.Hkv + kvh) * sh.tiles + tile) * sh.n_split * kRows + row;
    iq = r / G, h = kvh * G + r - iq * G;
    sums = sums_at(sh);
  }
  float m = -INFINITY, l = 0.f, ls = 0.f;
  f32x4 t = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int s0 = k; s0 < n_split; s0 += 8 * KG) {
    f32x4 p[8];
    float2 ml[8];
    float ps[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int s = s0 + j * KG;
      ml[j] = make_float2(-INFINITY, 0.f);
      p[j] = f32x4{0.f, 0.f, 0.f, 0.f};
      ps[j] = 0.f;
      if (s < n_split) {
        const size_t at = base + (size_t)s * step;
        ml[j] = part_ml[at];
        if constexpr (LSE) ps[j] = part_o[sums + at];
        p[j] = *reinterpret_cast<const f32x4 *>(part_o + at * kKvHd + 4 * d4);
      }
    }
    if constexpr (GROUPS)  // parts without keys were not written
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (ml[j].x == -INFINITY && ml[j].y == 0.f) p[j] = f32x4{0.f, 0.f, 0.f, 0.f};
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
  const float inv = l == 0.f ? 0.f : 1.0f / l;  // l = 0: no key seen
  uint2 u;
  u.x = pack_bf16x2(t[0] * inv, t[1] * inv);
  u.y = pack_bf16x2(t[2] * inv, t[3] * inv);
  *reinterpret_cast<uint2 *>(o + ((size_t)b * sh.n_q + iq) * ldo + (size_t)h * kKvHd + 4 * d4) = u;
  if (LSE && d4 == 0)
    lse[((size_t)b * sh.Hq + h) * sh.n_q + iq] = (m + log2f(ls)) * 0.6931471805599453f;
}
}  // namespace
}  // namespace prichs
