// window_attention.hip -- causal GQA attention with a sliding window and sinks,
// and its backward.
#include "attention_tile.hpp"

#include <algorithm>

namespace prichs {
namespace {

constexpr int kHd = 128;

// Rows of sequence b.
__device__ __forceinline__ int rows_of(const int32_t *seq_lens, int b, int S) {
  return seq_lens == nullptr ? S : min(max(seq_lens[b], 0), S);
}
struct Shape {
  int S, Hq, Hkv, window, sinks;
  float scale, scale_log2;  // 1 / sqrt(128), and times log2(e)
};

constexpr float kLog2e = 1.4426950408889634f;

// Chunk key of a row of a [rows][128] tile in LDS: its 16-byte chunk c is stored at
// c ^ tile_key(row).  One key serves both kinds of read without a bank conflict
// (counted: SQ_LDS_BANK_CONFLICT 0; the row's bits rotated by one double every
// fragment read): a transposing read takes two neighbouring chunks of 8 rows at a
// time, whose keys differ above bit 0; a fragment read is served in quarters of 16
// lanes that pair rows 0-3 and 12-15 of one chunk with rows 4-7 and 8-11 of the
// next, and each of the two sets of keys is closed under exclusive or with 1.
__device__ __forceinline__ int tile_key(int row) {
  return (((row & 7) ^ ((row & 8) >> 1)) << 1) | ((row >> 3) & 1);
}
__device__ __forceinline__ int tile_off(int row, int c) { return row * kHd + ((c ^ tile_key(row)) << 3); }

// A copy of 16 (or 4) bytes a lane to LDS, as dma_16b, in a form whose target the
// compiler does not see: it would wait for all copies in flight before every
// transposing read.  There are no result registers; callers wait by vmcnt.
__device__ __forceinline__ void copy_16b(__amdgpu_buffer_rsrc_t r, uint32_t voff, uint32_t lds_at) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds_at),
               "v"(voff), "s"(r)
               : "memory", "m0");
}
__device__ __forceinline__ void copy_4b(__amdgpu_buffer_rsrc_t r, uint32_t voff, uint32_t lds_at) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds" ::"s"(lds_at),
               "v"(voff), "s"(r)
               : "memory", "m0");
}
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
// A transposing fragment: both halves of a 32-row step.
__device__ __forceinline__ u32x4 read_tr(uint32_t lds_at) {
  typedef __attribute__((address_space(3))) bf16x4 *at_t;
  const bf16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((at_t)(uintptr_t)lds_at);
  const bf16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((at_t)(uintptr_t)(lds_at + 2 * 16 * kHd));
  return __builtin_bit_cast(u32x4, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
}

__device__ __forceinline__ void finite_frags(u32x4 (&f)[4]) {
#pragma unroll
  for (int t = 0; t < 4; ++t)
#pragma unroll
    for (int e = 0; e < 4; ++e) f[t][e] = finite_bf16x2(f[t][e]);
}
// 0 where every element is finite, NaN otherwise.
__device__ __forceinline__ float not_finite(f32x4 x, float z) {
#pragma unroll
  for (int r = 0; r < 4; ++r) z = fmaf(x[r], 0.f, z);
  return z;
}

// The lane's number, formed anew where it is asked for: what a loop derives from
// it then holds no register over the loop.
__device__ __forceinline__ int lane_here() {
  int x;
  asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=&v"(x));
  return x;
}

struct BwdArgs {
  const bf16_t *d_o, *q, *k, *v, *o;
  const float *lse;
  const int32_t *seq_lens;
  bf16_t *dq, *dk, *dv;
  int ldd, ldq, ldk, ldv, ldo, lddq, lddk, lddv;
  // Per (sequence, head), per 32 rows: lse * log2(e) of the rows, then delta =
  // d_o . o of the rows; a row past the sequence has +inf and 0 (p = 0).
  float *rows;
  int row_tiles;  // 32-row tiles of a (sequence, head) there
  float *part;    // f32 partial d_k, d_v (window_dkv_kernel)
  int budget;     // steps of a workgroup there
  int items;      // items of a (sequence, kv head) there
  int slots;      // of them, the first ones, those that have a place in part
  // For workgroups dealt by die: row blocks of window_dq_kernel, and the (sequence,
  // head set) pairs there and (sequence, kv head) pairs in window_dkv_kernel.
  int dq_blocks, dq_pairs, dkv_pairs;
  Shape sh;
};

// ---------------------------------------------------------------- d_q --------
// As the forward (attention.hip): a wave owns NB blocks of 16 query rows of one
// head, HPW heads of a kv group share the K / V tiles that the workgroup streams
// through LDS (64 keys, two stages).
//   S^T = K Q^T, dP^T = V d_o^T   both operands' rows straight from LDS / registers
//   dS^T = exp2(S scale log2(e) - lse) (dP - delta)   in the accumulator layout,
//                   which is the operand layout of
//   dQ^T += K^T dS^T              K^T by transposing LDS reads
// The kernel also forms delta of its rows and leaves it, with lse, to
// window_dkv_kernel.  12 + 3 heads: 4 x 2048, window 512, 66 us; 1 x 4096 whole 116
// us (670 TFLOP/s); 3 x 500, window 128, 21 us.  Long windows are bound by the matrix
// cores (busy 55% of the time) and the vector instructions between their products,
// which the two waves of a SIMD overlap little; short ones by the latency of a block
// (load, barrier, two dependent products: 1.5 us), twice for rows of few blocks.
// Eight waves of 16 rows a workgroup on the same tiles were no faster (170 -> 167,
// 1481 -> 1552 us for the whole backward of 4 x 2048 and of 1 x 16384, window 4096).
constexpr int kTr = 32;  // rows of a step of window_dkv_kernel
constexpr int kKeys = 64;
constexpr int kQStage = 2 * kKeys * kHd;  // elements: K, then V
constexpr int kExactBlocks = 4;  // delta in a sweep of its own up to so many blocks
constexpr size_t kQLds = 2 * (size_t)kQStage * sizeof(bf16_t);

// NB: 16-row blocks of a wave.  DIE: workgroups dealt by die (attention_tile.hpp).
template <int HPW, int NB, bool DIE = false>
__global__ __launch_bounds__(256, 2) void window_dq_kernel(BwdArgs a) {
  constexpr int kRowsWg = 64 * NB / HPW;
  extern __shared__ __attribute__((aligned(16))) bf16_t lds[];
  const Shape &sh = a.sh;
  const int group = sh.Hq / sh.Hkv, sets = group / HPW;
  int x = blockIdx.x, b = blockIdx.y, qb = (int)(gridDim.z - 1 - blockIdx.z);  // long rows first
  if constexpr (DIE) {
    int pair, rank;
    if (!die_rank(blockIdx.x, a.dq_pairs, a.dq_blocks, &pair, &rank)) return;
    b = pair / (sh.Hq / HPW), x = pair - b * (sh.Hq / HPW), qb = a.dq_blocks - 1 - rank;
  }
  const int kvh = x / sets;
  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, l16 = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int h = kvh * group + (x - kvh * sets) * HPW + wave % HPW;
  const int q0 = qb * kRowsWg + (wave / HPW) * 16 * NB;
  const int L = rows_of(a.seq_lens, b, sh.S);
  const size_t seq0 = (size_t)b * sh.S;

  // This wave's rows: fragments of q and d_o, lse, delta.
  bf16x8 qf[NB][4], df[NB][4];
  float lse2[NB], delta[NB];
  float *rows = a.rows + (((size_t)b * sh.Hq + h) * a.row_tiles + q0 / kTr) * 2 * kTr + q0 % kTr;
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    const int row = q0 + 16 * nb + l16;
    const size_t r = seq0 + min(row, sh.S - 1);
    const size_t c = (size_t)h * kHd + 8 * g;
    float s = 0.f;
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
      qf[nb][kk] = *reinterpret_cast<const bf16x8 *>(a.q + r * a.ldq + c + 32 * kk);
      df[nb][kk] = *reinterpret_cast<const bf16x8 *>(a.d_o + r * a.ldd + c + 32 * kk);
      const u32x4 x = __builtin_bit_cast(u32x4, df[nb][kk]);
      const u32x4 y = *reinterpret_cast<const u32x4 *>(a.o + r * a.ldo + c + 32 * kk);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s += __uint_as_float(x[e] << 16) * __uint_as_float(y[e] << 16);
        s += __uint_as_float(x[e] & 0xffff0000u) * __uint_as_float(y[e] & 0xffff0000u);
      }
    }
    s += __shfl_xor(s, 16);
    s += __shfl_xor(s, 32);
    const bool live = row < L;
    lse2[nb] = live ? a.lse[((size_t)b * sh.Hq + h) * sh.S + row] * kLog2e : INFINITY;
    delta[nb] = live ? s : 0.f;
  }
  f32x4 acc[8][NB];
#pragma unroll
  for (int jd = 0; jd < 8; ++jd)
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) acc[jd][nb] = f32x4{0.f, 0.f, 0.f, 0.f};

  // Blocks of 64 keys: the sinks', then from the first row's window on.
  const int q_last = min(L, (qb + 1) * kRowsWg) - 1;
  const int first = sh.window == 0 ? 0 : max(0, qb * kRowsWg - sh.window + 1) / kKeys;
  const int n_sink = min((sh.sinks + kKeys - 1) / kKeys, first), skip = first - n_sink;
  const int n_blk = qb * kRowsWg >= L ? 0 : q_last / kKeys + 1 - skip;
  auto block_of = [&](int i) { return i >= n_sink ? i + skip : i; };

  const bf16_t *kbase = a.k + seq0 * a.ldk + (size_t)kvh * kHd;
  const bf16_t *vbase = a.v + seq0 * a.ldv + (size_t)kvh * kHd;
  const uint32_t lds_base =
      (uint32_t)(size_t)(const __attribute__((address_space(3))) bf16_t *)lds;
  auto issue_tile = [&](int i, const bf16_t *src, int ld, int tile) {
    const int blk = block_of(i);
    const uint64_t bytes = (uint64_t)(L - 1 - blk * kKeys) * 2 * (uint64_t)ld + 2 * kHd;
    const __amdgpu_buffer_rsrc_t r = buffer_rsrc(
        src + (size_t)blk * kKeys * ld, bytes > 0xffffffffull ? 0xffffffffu : (uint32_t)bytes);
    const uint32_t dst = lds_base + 2u * (uint32_t)((i & 1) * kQStage + tile * kKeys * kHd);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int row = 16 * wave + 4 * j + g;
      copy_16b(r, 2u * ((uint32_t)row * (uint32_t)ld + 8u * (uint32_t)(l16 ^ tile_key(row))),
               dst + (uint32_t)(2 * (16 * wave + 4 * j) * kHd));
    }
  };
  auto issue = [&](int i) {
    issue_tile(i, kbase, a.ldk, 0);
    issue_tile(i, vbase, a.ldv, 1);
  };
  const uint32_t row_addr = 2u * (uint32_t)tile_off(l16, g);
  const uint32_t tr_addr =
      lds_base + 2u * (uint32_t)(tile_off(4 * g + (l16 >> 2), (l16 & 3) >> 1) + 4 * (l16 & 1));

  // One sweep over the blocks: f(half, stage, first key, S^T, dP^T, rare) for each half
  // block that some row of the wave sees, hidden elements at -inf and 0.
  auto sweep = [&](auto &&f) {
    if (n_blk > 0) issue(0);
#pragma unroll 1
    for (int i = 0; i < n_blk; ++i) {
      const int kv0 = block_of(i) * kKeys;
      // Block i has landed for every wave, and every wave is done with block i - 1.
      asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
      if (i + 1 < n_blk) issue(i + 1);
      // Every row of the wave sees the whole block, or none of it.
      const bool whole = kv0 + kKeys <= min(q0 + 1, L) &&
                         (sh.window == 0 || q0 + 16 * NB - 1 - kv0 < sh.window || kv0 + kKeys <= sh.sinks);
      const bool none = kv0 > q0 + 16 * NB - 1 || (sh.window != 0 && q0 - (kv0 + kKeys - 1) >= sh.window &&
                                          kv0 >= sh.sinks);
      if (none) continue;
      const uint32_t stage = (uint32_t)(i & 1) * (uint32_t)(kQStage * sizeof(bf16_t));
      const char *kt = reinterpret_cast<const char *>(lds) + stage;
      static_for<2>([&](auto half_c) {
        constexpr int half = decltype(half_c)::value;  // keys 32 half ..
        f32x4 s[2][NB], dp[2][NB];
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) s[c][nb] = dp[c][nb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const char *p = kt + (row_addr ^ (uint32_t)(64 * kk)) + 2 * kHd * (32 * half + 16 * c);
            const bf16x8 kf = *reinterpret_cast<const bf16x8 *>(p);
            const bf16x8 vf = *reinterpret_cast<const bf16x8 *>(p + 2 * kKeys * kHd);
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
              s[c][nb] = mfma_bf16(kf, qf[nb][kk], s[c][nb]);
              dp[c][nb] = mfma_bf16(vf, df[nb][kk], dp[c][nb]);
            }
          }
        bool rare = false;
        if (!whole) {
          // What a row does not see must not reach it: hidden elements become p = 0,
          // and an infinity or NaN in K^T, which 0 would turn into NaN, is taken out
          // of the product (see rare below).  Rows past the sequence need no mask: they
          // reach no other row.  The wave's rows decide which of the rules a block needs.
          float z = 0.f;
          const bool ahead = kv0 + kKeys - 1 > q0;
          const bool behind = sh.window != 0 && q0 + 16 * NB - 1 - kv0 >= sh.window &&
                              kv0 + kKeys > sh.sinks;
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) z = not_finite(s[c][nb], z);
          const int first_key = kv0 + 32 * half + 4 * g - (q0 + l16);
          if (ahead) {
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
              for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                  const bool hidden = first_key > 16 * nb - 16 * c - r;
                  s[c][nb][r] = hidden ? -INFINITY : s[c][nb][r];
                  dp[c][nb][r] = hidden ? 0.f : dp[c][nb][r];
                }
          }
          if (behind) {
            const int old = first_key + sh.window, sink = sh.sinks - (kv0 + 32 * half + 4 * g);
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
              for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                  const bool hidden = (old <= 16 * nb - 16 * c - r) & (sink <= 16 * c + r);
                  s[c][nb][r] = hidden ? -INFINITY : s[c][nb][r];
                  dp[c][nb][r] = hidden ? 0.f : dp[c][nb][r];
                }
          }
          rare = __any(!(z == 0.f)) != 0;
        }
        f(half_c, stage, kv0 + 32 * half, s, dp, rare);
      });
    }
  };

  // delta = d_o . o, from an o that was rounded to bf16, is off by some 2^-9 of the
  // terms' root sum of squares: little beside dP where a row sees many keys, but half
  // again the error of d_q and d_k where it sees few (0.0038 instead of 0.0024 of
  // their norm at 2 keys, 0.0027 at 8, 0.0025 at 64).  Rows of few blocks form it as
  // sum p dP / sum p instead, in a sweep of their own (2 of the 3 products again).
  if (n_blk > 0 && n_blk <= kExactBlocks) {
    float num[NB] = {}, den[NB] = {};
    sweep([&](auto, uint32_t, int, f32x4 (&s)[2][NB], f32x4 (&dp)[2][NB], bool) {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float p = fast_exp2(fmaf(s[c][nb][r], sh.scale_log2, -lse2[nb]));
            num[nb] = fmaf(p, dp[c][nb][r], num[nb]);
            den[nb] += p;
          }
    });
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      num[nb] += __shfl_xor(num[nb], 16);
      den[nb] += __shfl_xor(den[nb], 16);
      num[nb] += __shfl_xor(num[nb], 32);
      den[nb] += __shfl_xor(den[nb], 32);
      if (q0 + 16 * nb + l16 < L) delta[nb] = num[nb] / den[nb];
    }
    asm volatile("s_barrier" ::: "memory");  // the last block's readers, before it is refilled
  }
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
    if (g == 0 && q0 < a.row_tiles * kTr) {
      rows[16 * nb + l16] = lse2[nb];
      rows[kTr + 16 * nb + l16] = delta[nb];
    }

  sweep([&](auto half_c, uint32_t stage, int key0, f32x4 (&s)[2][NB], f32x4 (&dp)[2][NB],
            bool rare) {
    constexpr int half = decltype(half_c)::value;
    u32x4 ds[NB];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      float e[8];
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          e[4 * c + r] = fast_exp2(fmaf(s[c][nb][r], sh.scale_log2, -lse2[nb])) *
                         (dp[c][nb][r] - delta[nb]);
      // dS rounded to bf16 for the product.
      ds[nb] = u32x4{pack_bf16(e[0], e[1]), pack_bf16(e[2], e[3]), pack_bf16(e[4], e[5]),
                     pack_bf16(e[6], e[7])};
    }
#pragma unroll
    for (int j0 = 0; j0 < 8; j0 += 4) {
      u32x4 f[4];
#pragma unroll
      for (int t = 0; t < 4; ++t)
        f[t] = read_tr(((tr_addr + stage) ^ (uint32_t)(32 * (j0 + t))) + 2 * 32 * half * kHd);
      if (rare) finite_frags(f);
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
          acc[j0 + t][nb] = mfma_bf16(__builtin_bit_cast(bf16x8, f[t]),
                                      __builtin_bit_cast(bf16x8, ds[nb]), acc[j0 + t][nb]);
    }
    if (rare) {
      // A row that sees a key that is not finite: 0 (of a score of -inf) or NaN times
      // what was taken out is NaN, in that element.
      const char *kt = reinterpret_cast<const char *>(lds) + stage;
#pragma unroll 1
      for (int x = 0; x < 32; ++x) {
        const int key = key0 + x;
#pragma unroll
        for (int jd = 0; jd < 8; ++jd) {
          asm volatile("" ::: "memory");  // one load after the other: registers
          const u32x2 raw = *reinterpret_cast<const u32x2 *>(
              kt + ((uint32_t)(2 * (tile_off(32 * half + x, g >> 1) + 4 * (g & 1))) ^ (32u * jd)));
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) {
            const int row = q0 + 16 * nb + l16;
            const bool seen = (key <= row) & ((sh.window == 0) | (row - key < sh.window) |
                                              (key < sh.sinks));
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const uint32_t u = r & 1 ? raw[r / 2] & 0xffff0000u : raw[r / 2] << 16;
              const bool off = (u & 0x7f800000u) == 0x7f800000u;
              acc[jd][nb][r] = (off & seen) ? __uint_as_float(0x7fc00000u) : acc[jd][nb][r];
            }
          }
        }
      }
    }
  });

#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    const int row = q0 + 16 * nb + l16;
    if (row >= sh.S) continue;
    bf16_t *out = a.dq + (seq0 + row) * a.lddq + (size_t)h * kHd + 4 * g;
    const bool live = row < L;
#pragma unroll
    for (int jd = 0; jd < 8; ++jd) {
      const f32x4 t = acc[jd][nb] * sh.scale;
      const u32x2 u = u32x2{pack_bf16(t[0], t[1]), pack_bf16(t[2], t[3])};
      *reinterpret_cast<u32x2 *>(out + 16 * jd) = live ? u : u32x2{0, 0};
    }
  }
}

// ------------------------------------------------------------ d_k, d_v -------
// A workgroup owns 128 keys of one kv head and runs over the (query head, 32-row
// tile) steps that see them.  16 waves: 8 key groups of 16 keys, whose K fragments
// and f32 gradients stay in registers and V in LDS, times 2 step groups, which take
// every second step and join in LDS at the end.
//   S = Q K^T, dP = d_o V^T       rows of the q and d_o tiles straight from LDS
//   P, dS                         in the accumulator layout, which is the operand
//                                 layout (a lane holds one key and 8 of 32 rows) of
//   dV^T += d_o^T P, dK^T += Q^T dS   by transposing LDS reads
// Tiles come in three stages, so that a step's copies have the time of two steps.
// 12 + 3 heads: 4 x 2048, window 512, 97 us; 1 x 4096 whole 156 us (660 TFLOP/s), 1 x
// 16384, window 4096, 900 us (800); 3 x 500, window 128, 21 us.  No single unit bounds it: without the copies it takes
// 2 to 7% less, without the transposing reads 2 to 7%, without the exponentials 1.5%;
// the matrix cores are busy 40% of the time, LDS 50%, and what is left is the latency of a step
// (reads, four dependent products, exponentials, products) that four waves a SIMD,
// held together by a barrier a step, do not hide.  With 32 keys a wave (two waves a
// SIMD, half the LDS reads) the whole backward of 4 x 2048 takes 187 us instead of 157
// and that of 1 x 16384, window 4096, 1390 instead of 1413; 64-key blocks, two
// workgroups a CU, 195 and 1740.  No register may spill in the loop: a reload waits for
// all copies in flight (7%).
// Steps are cut into items of at most `budget` (a block that holds sinks is seen by
// every later row); the items of one block meet in f32 partial sums that
// window_dkv_join_kernel adds in order.
constexpr int kBlk = 128;           // keys of a workgroup
constexpr int kKg = kBlk / 16;      // key groups
constexpr int kStages = 3;
constexpr int kStepElems = 2 * kTr * kHd + 128;  // q, d_o, then lse / delta (64 floats)
constexpr size_t kKvLds = (2 * kStages * (size_t)kStepElems + kBlk * kHd) * sizeof(bf16_t);
static_assert(kKvLds >= kKg * 8 * 64 * sizeof(f32x4), "the join of the step groups fits");

// Steps of key block j over sequences of S rows.
__host__ __device__ inline int steps_of(const Shape &sh, int rows, int j) {
  const int left = rows - j * kBlk;
  const bool far = sh.window == 0 || j * kBlk < sh.sinks;
  const int n = far || left < kBlk + sh.window - 1 ? left : kBlk + sh.window - 1;
  return n <= 0 ? 0 : (n + kTr - 1) / kTr * (sh.Hq / sh.Hkv);
}
__host__ __device__ inline int splits_of(const Shape &sh, int budget, int j) {
  const int n = (steps_of(sh, sh.S, j) + budget - 1) / budget;
  return n < 1 ? 1 : n;
}
// The block and split of an item (the same in every lane).
__device__ __forceinline__ void item_at(const Shape &sh, int budget, int item, int *block,
                                        int *split) {
  const int lane = threadIdx.x & 63, blocks = (sh.S + kBlk - 1) / kBlk;
  for (int base = 0; base < blocks; base += 64) {
    const int n = base + lane < blocks ? splits_of(sh, budget, base + lane) : 0;
    int end = n;
    for (int d = 1; d < 64; d <<= 1) {
      const int up = __shfl_up(end, d);
      if (lane >= d) end += up;
    }
    const unsigned long long in = __ballot(item < end);
    if (in != 0) {
      const int at = __ffsll((long long)in) - 1;
      *block = base + at;
      *split = __builtin_amdgcn_readfirstlane(item - (__shfl(end, at) - __shfl(n, at)));
      return;
    }
    item -= __shfl(end, 63);
  }
  *block = blocks - 1, *split = 0;  // not reached: the grid holds the items
}

template <bool DIE>
__global__ __launch_bounds__(128 * kKg, 4) void window_dkv_kernel(BwdArgs a) {
  extern __shared__ __attribute__((aligned(16))) bf16_t lds[];
  const Shape &sh = a.sh;
  const int G = sh.Hq / sh.Hkv;
  int item = blockIdx.x, kvh = blockIdx.y, b = blockIdx.z;
  if constexpr (DIE) {
    int pair;
    if (!die_rank(blockIdx.x, a.dkv_pairs, a.items, &pair, &item)) return;
    b = pair / sh.Hkv, kvh = pair - b * sh.Hkv;
  }
  int blk, split;
  item_at(sh, a.budget, item, &blk, &split);
  blk = __builtin_amdgcn_readfirstlane(blk);
  const int n_split = splits_of(sh, a.budget, blk);
  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, l16 = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kg = wave % kKg, sg = wave / kKg;
  const int L = rows_of(a.seq_lens, b, sh.S);
  const size_t seq0 = (size_t)b * sh.S;
  const int k0 = blk * kBlk + 16 * kg;  // this wave's first key

  bf16x8 kf[4];
  f32x4 dk[8], dv[8];
  {
    const int key = k0 + l16;
    const size_t r = seq0 + min(key, sh.S - 1), c = (size_t)kvh * kHd + 8 * g;
    const bool live = key < L;
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
      u32x4 x = *reinterpret_cast<const u32x4 *>(a.k + r * a.ldk + c + 32 * kk);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = live ? x[e] : 0u;
      kf[kk] = __builtin_bit_cast(bf16x8, x);
    }
  }
#pragma unroll
  for (int jd = 0; jd < 8; ++jd) dk[jd] = dv[jd] = f32x4{0.f, 0.f, 0.f, 0.f};

  // This item's steps: step x is head x / tiles, row tile t_lo + x % tiles.
  const int steps = steps_of(sh, L, blk), tiles = steps / G;
  const int begin = (int)((int64_t)steps * split / n_split),
            end = (int)((int64_t)steps * (split + 1) / n_split);
  const int t_lo = blk * (kBlk / kTr);
  const int n_it = (end - begin + 1) / 2;

  // The step to compute next: its number and row tile.
  int cx = begin + sg, ct = tiles > 0 ? cx % tiles : 0;
  // Every wave of a step group moves kRowsEach of the step's rows of q and of d_o, and
  // all of lse / delta (the same bytes).
  constexpr int kRowsEach = kTr / kKg, kCopies = 3;
  static_assert(kRowsEach == 4, "one copy of 16 bytes a lane each");
  // The step to fetch next: where the wave's rows of q and d_o start, how many rows
  // the sequence has from there on, and the step's statistics.
  int fx = cx, ft = ct, fh = tiles > 0 ? cx / tiles : 0, left;
  const char *pq, *pd;
  const float *pr;
  auto seek = [&]() {
    const int h = kvh * G + fh, t0 = (t_lo + ft) * kTr + kRowsEach * kg;
    pq = reinterpret_cast<const char *>(a.q + (seq0 + t0) * a.ldq + (size_t)h * kHd);
    pd = reinterpret_cast<const char *>(a.d_o + (seq0 + t0) * a.ldd + (size_t)h * kHd);
    pr = a.rows + (((size_t)b * sh.Hq + h) * a.row_tiles + t_lo + ft) * 64;
    left = L - t0;
  };
  seek();
  const uint32_t lds_base =
      (uint32_t)(size_t)(const __attribute__((address_space(3))) bf16_t *)lds;
  // V of the block, behind the steps' tiles.
  const uint32_t v_tile = 2 * kStages * kStepElems * 2u;
  {
    const int left = L - blk * kBlk;  // rows of V
    const uint64_t bytes = (uint64_t)(left - 1) * 2 * (uint64_t)a.ldv + 2 * kHd;
    const __amdgpu_buffer_rsrc_t r = buffer_rsrc(
        a.v + (seq0 + (left > 0 ? blk * kBlk : 0)) * a.ldv + (size_t)kvh * kHd,
        left <= 0 ? 0u : bytes > 0xffffffffull ? 0xffffffffu : (uint32_t)bytes);
#pragma unroll
    for (int j = 0; j < kBlk / (8 * kKg); ++j) {
      const int x = kBlk / (2 * kKg) * wave + 4 * j + g;
      copy_16b(r, 2u * ((uint32_t)x * (uint32_t)a.ldv + 8u * (uint32_t)(l16 ^ tile_key(x))),
               lds_base + v_tile + (uint32_t)(2 * (kBlk / (2 * kKg) * wave + 4 * j) * kHd));
    }
  }
  // Row 4 kg + g of a step's tile has the key 2 g ^ `turn`.  A step past the end copies
  // nothing (an empty buffer: zeros), so that the count of copies in flight stays known;
  // rows past the sequence are zeros too.
  const uint32_t turn = (uint32_t)tile_key(kRowsEach * kg);
  auto fetch = [&](int slot) {
    const uint32_t dst = lds_base + (uint32_t)((sg * kStages + slot) * kStepElems) * 2u;
    const int ln = lane_here(), n = fx < end ? min(left, kRowsEach) : 0;
    const uint32_t gg = (uint32_t)ln >> 4, at = (((uint32_t)ln & 15) ^ (2 * gg) ^ turn) << 4;
    auto rows = [&](const char *src, int pitch, int tile) {
      copy_16b(buffer_rsrc(src, n <= 0 ? 0u : (uint32_t)(n - 1) * 2u * (uint32_t)pitch + 2 * kHd),
               (2 * gg) * ((uint32_t)pitch & 0xffffffu) + at,
               dst + (uint32_t)(2 * (tile + kRowsEach * kg * kHd)));
    };
    rows(pq, a.ldq, 0);
    rows(pd, a.ldd, kTr * kHd);
    copy_4b(buffer_rsrc(pr, fx < end ? 256u : 0u), 4u * (uint32_t)ln, dst + 4 * kTr * kHd);
    fx += 2;
    ft += 2;
    if (ft < tiles) {
      pq += 4 * kTr * (int64_t)a.ldq;
      pd += 4 * kTr * (int64_t)a.ldd;
      pr += 2 * 64;
      left -= 2 * kTr;
    } else if (tiles > 0) {
      while (ft >= tiles) ft -= tiles, ++fh;
      seek();
    }
  };

  const uint32_t ra0 = 2u * (uint32_t)tile_off(l16, g);
  const uint32_t ta0 = 2u * (uint32_t)(tile_off(4 * g + (l16 >> 2), (l16 & 3) >> 1) + 4 * (l16 & 1));
  const uint32_t g16 = 16u * (uint32_t)g;
  auto compute = [&](int slot) {
    const int t0 = (t_lo + ct) * kTr;
    const bool none = cx >= end || k0 >= L || t0 + kTr - 1 < k0 ||
                      (sh.window != 0 && t0 - (k0 + 16 - 1) >= sh.window && k0 >= sh.sinks);
    if (none) return;
    const bool whole = t0 >= k0 + 16 - 1 && (sh.window == 0 || t0 + kTr - 1 - k0 < sh.window ||
                                         k0 + 16 <= sh.sinks);
    // Rows past the sequence are zeros in the tiles, and p is 0 by their lse -- but not
    // with a key that is not finite: their scores are NaN, and their dP.
    const bool past = t0 + kTr > L;
    const uint32_t at = (uint32_t)((sg * kStages + slot) * kStepElems) * 2u;
    const char *tile = reinterpret_cast<const char *>(lds) + at;
    const uint32_t ra = lds_base + at + ra0, ta = lds_base + at + ta0;
    auto frag_at = [&](uint32_t lane_at, int kk, uint32_t off) {
      typedef const __attribute__((address_space(3))) bf16x8 *at_t;
      return *(at_t)(uintptr_t)((lane_at ^ (uint32_t)(64 * kk)) + off);
    };
    auto stat_at = [&](uint32_t off) {
      typedef const __attribute__((address_space(3))) f32x4 *at_t;
      return *(at_t)(uintptr_t)(lds_base + at + 4 * kTr * kHd + g16 + off);
    };
    // x is 0 where the key's row does not see it.
    auto hide = [&](int qb, f32x4 &x) {
      int row = t0 + 16 * qb + 4 * g;
      asm volatile("" : "+v"(row));  // keeps this in the branches that call it
      const int key = k0 + l16;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const bool seen = (key <= row + r) & ((sh.window == 0) | (row + r - key < sh.window) |
                                              (key < sh.sinks));
        x[r] = seen ? x[r] : 0.f;
      }
    };
    auto hide_past = [&](int qb, f32x4 &x) {
      int row = t0 + 16 * qb + 4 * g;
      asm volatile("" : "+v"(row));
#pragma unroll
      for (int r = 0; r < 4; ++r) x[r] = row + r < L ? x[r] : 0.f;
    };
    // Softmax and first products before the other waves' last ones: 1 x 16384 window
    // 4096 1411 -> 1390 us, 4 x 2048 158.7 -> 156.
    __builtin_amdgcn_s_setprio(1);
    u32x4 pf, ds;  // P and dS rounded to bf16 for the products
    float z = 0.f;
    f32x4 p[2], x[2];  // of 16 rows each
    x[0] = x[1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int kk = 0; kk < 4; ++kk)
#pragma unroll
      for (int qb = 0; qb < 2; ++qb)
        x[qb] = mfma_bf16(frag_at(ra, kk, 2 * kHd * 16 * qb), kf[kk], x[qb]);
#pragma unroll
    for (int qb = 0; qb < 2; ++qb) {
      const f32x4 lse2 = stat_at(64 * qb);
#pragma unroll
      for (int r = 0; r < 4; ++r) p[qb][r] = fast_exp2(fmaf(x[qb][r], sh.scale_log2, -lse2[r]));
    }
    // What a key's row does not see must not reach the key, whatever the row holds: p
    // and dS are 0 there, and see rare below.
    if (!whole) {
#pragma unroll
      for (int qb = 0; qb < 2; ++qb) {
        z = not_finite(x[qb], z);
        hide(qb, p[qb]);
      }
    }
    if (past) {
#pragma unroll
      for (int qb = 0; qb < 2; ++qb) hide_past(qb, p[qb]);
    }
    x[0] = x[1] = f32x4{0.f, 0.f, 0.f, 0.f};
    uint32_t va = lds_base + ra0 + v_tile + 2 * kHd * 16 * kg;
    asm volatile("" : "+v"(va));  // its fragments' addresses are not kept over the steps
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
      const bf16x8 vf = frag_at(va, kk, 0);
#pragma unroll
      for (int qb = 0; qb < 2; ++qb)
        x[qb] = mfma_bf16(frag_at(ra, kk, 2 * kTr * kHd + 2 * kHd * 16 * qb), vf, x[qb]);
    }
    f32x4 e[2];
#pragma unroll
    for (int qb = 0; qb < 2; ++qb) {
      const f32x4 delta = stat_at(4 * kTr + 64 * qb);
#pragma unroll
      for (int r = 0; r < 4; ++r) e[qb][r] = p[qb][r] * (x[qb][r] - delta[r]);
    }
    if (!whole) {
#pragma unroll
      for (int qb = 0; qb < 2; ++qb) {
        z = not_finite(x[qb], z);
        hide(qb, e[qb]);
      }
    }
    if (past) {
#pragma unroll
      for (int qb = 0; qb < 2; ++qb) hide_past(qb, e[qb]);
    }
#pragma unroll
    for (int qb = 0; qb < 2; ++qb) {
      pf[2 * qb] = pack_bf16(p[qb][0], p[qb][1]), pf[2 * qb + 1] = pack_bf16(p[qb][2], p[qb][3]);
      ds[2 * qb] = pack_bf16(e[qb][0], e[qb][1]), ds[2 * qb + 1] = pack_bf16(e[qb][2], e[qb][3]);
    }
    // An infinity or NaN of q or d_o, which 0 would turn into NaN, is taken out of
    // the products of a step that not every key's row sees.
    const bool rare = !whole && __any(!(z == 0.f)) != 0;
    constexpr int kDo = 2 * kTr * kHd;  // bytes to the d_o tile
    __builtin_amdgcn_s_setprio(0);
#pragma unroll
    for (int j0 = 0; j0 < 8; j0 += 4) {
      u32x4 f[4];
#pragma unroll
      for (int t = 0; t < 4; ++t) f[t] = read_tr((ta ^ (uint32_t)(32 * (j0 + t))) + kDo);
      if (rare) finite_frags(f);
#pragma unroll
      for (int t = 0; t < 4; ++t)
        dv[j0 + t] = mfma_bf16(__builtin_bit_cast(bf16x8, f[t]), __builtin_bit_cast(bf16x8, pf),
                               dv[j0 + t]);
#pragma unroll
      for (int t = 0; t < 4; ++t) f[t] = read_tr(ta ^ (uint32_t)(32 * (j0 + t)));
      if (rare) finite_frags(f);
#pragma unroll
      for (int t = 0; t < 4; ++t)
        dk[j0 + t] = mfma_bf16(__builtin_bit_cast(bf16x8, f[t]), __builtin_bit_cast(bf16x8, ds),
                               dk[j0 + t]);
    }
    if (rare) {
      // The infinities and NaN of d_o that were taken out, for the keys that their
      // rows see (p > 0: an infinity keeps its sign).  A row with such a q has NaN
      // in P and dS already.
#pragma unroll 1
      for (int x = 0; x < kTr; ++x) {
        const int row = t0 + x;
#pragma unroll
        for (int jd = 0; jd < 8; ++jd) {
          asm volatile("" ::: "memory");  // one load after the other: registers
          const u32x2 raw = *reinterpret_cast<const u32x2 *>(
              tile + kDo + ((uint32_t)(2 * (tile_off(x, g >> 1) + 4 * (g & 1))) ^ (32u * jd)));
          const int key = k0 + l16;
          const bool seen = (key <= row) & ((sh.window == 0) | (row - key < sh.window) |
                                            (key < sh.sinks));
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const uint32_t u = r & 1 ? raw[r / 2] & 0xffff0000u : raw[r / 2] << 16;
            const bool off = (u & 0x7f800000u) == 0x7f800000u;
            dv[jd][r] += (off & seen) ? __uint_as_float(u) : 0.f;
          }
        }
      }
    }
  };

#pragma unroll
  for (int x = 0; x < kStages - 1; ++x) fetch(x);
  int slot = 0;
#pragma unroll 1
  for (int it = 0; it < n_it; ++it) {
    // Of the copies in flight only the newest kStages - 2 steps' may be missing;
    // every wave is done with the slot that is fetched into next.
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(kCopies * (kStages - 2)) : "memory");
    fetch(slot == 0 ? kStages - 1 : slot - 1);
    compute(slot);
    cx += 2, ct += 2;
    while (ct >= tiles) ct -= tiles;
    slot = slot + 1 == kStages ? 0 : slot + 1;
  }
  // The copies past the end write zeros: they must land before LDS is used again.
  asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");

  // The second step group's sums join the first's, d_k then d_v.
  const int le = lane_here(), ge = le >> 4, l16e = le & 15;
  f32x4 *join = reinterpret_cast<f32x4 *>(lds);
  auto joined = [&](f32x4 (&x)[8]) {
    if (sg == 1) {
#pragma unroll
      for (int jd = 0; jd < 8; ++jd) join[(jd * kKg + kg) * 64 + le] = x[jd];
    }
    __syncthreads();
    if (sg == 0) {
#pragma unroll
      for (int jd = 0; jd < 8; ++jd) x[jd] = x[jd] + join[(jd * kKg + kg) * 64 + le];
    }
    __syncthreads();
  };
  joined(dk);
  joined(dv);
  if (sg != 0) return;
  if (n_split > 1) {
    float *part = a.part + ((((size_t)b * sh.Hkv + kvh) * a.slots + item) * 2) * kBlk * kHd;
    float *row = part + (16 * kg + l16e) * kHd + 4 * ge;
#pragma unroll
    for (int jd = 0; jd < 8; ++jd) {
      *reinterpret_cast<f32x4 *>(row + 16 * jd) = dk[jd];
      *reinterpret_cast<f32x4 *>(row + kBlk * kHd + 16 * jd) = dv[jd];
    }
    return;
  }
  const int key = k0 + l16e;
  if (key >= sh.S) return;
  bf16_t *ok = a.dk + (seq0 + key) * a.lddk + (size_t)kvh * kHd + 4 * ge;
  bf16_t *ov = a.dv + (seq0 + key) * a.lddv + (size_t)kvh * kHd + 4 * ge;
  const bool live = key < L;
#pragma unroll
  for (int jd = 0; jd < 8; ++jd) {
    const f32x4 x = dk[jd] * sh.scale, y = dv[jd];
    const u32x2 ux = u32x2{pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3])};
    const u32x2 uy = u32x2{pack_bf16(y[0], y[1]), pack_bf16(y[2], y[3])};
    *reinterpret_cast<u32x2 *>(ok + 16 * jd) = live ? ux : u32x2{0, 0};
    *reinterpret_cast<u32x2 *>(ov + 16 * jd) = live ? uy : u32x2{0, 0};
  }
}

// Adds the items of the blocks that were cut, in the items' order: a workgroup per
// (block, kv head, sequence) and 16 of its keys.  Bound by the latency of its loads
// (3 x 500, window 128: 6 us).
__global__ __launch_bounds__(256) void window_dkv_join_kernel(BwdArgs a) {
  const Shape &sh = a.sh;
  const int blk = blockIdx.x / (kBlk / 16), kvh = blockIdx.y, b = blockIdx.z;
  const int n_split = splits_of(sh, a.budget, blk);
  if (n_split == 1) return;
  int item = 0;  // the block's first
  const int lane = threadIdx.x & 63;
  for (int j = lane; j < blk; j += 64) item += splits_of(sh, a.budget, j);
  for (int m = 1; m < 64; m <<= 1) item += __shfl_xor(item, m);
  const int key = 16 * (blockIdx.x % (kBlk / 16)) + (threadIdx.x >> 4), d = 8 * (threadIdx.x & 15);
  const int row = blk * kBlk + key;
  if (row >= sh.S) return;
  const bool live = row < rows_of(a.seq_lens, b, sh.S);
  const float *part =
      a.part + ((((size_t)b * sh.Hkv + kvh) * a.slots + item) * 2) * kBlk * kHd + key * kHd + d;
  f32x4 t[2][2];
#pragma unroll
  for (int w = 0; w < 2; ++w) t[w][0] = t[w][1] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < n_split; ++s)
#pragma unroll
    for (int w = 0; w < 2; ++w)
#pragma unroll
      for (int e = 0; e < 2; ++e)
        t[w][e] = t[w][e] + *reinterpret_cast<const f32x4 *>(
                                part + (size_t)(2 * s + w) * kBlk * kHd + 4 * e);
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    bf16_t *out = (w == 0 ? a.dk + ((size_t)b * sh.S + row) * a.lddk
                          : a.dv + ((size_t)b * sh.S + row) * a.lddv) +
                  (size_t)kvh * kHd + d;
    const float f = w == 0 ? sh.scale : 1.0f;
    u32x4 u;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      u[2 * e] = pack_bf16(t[w][e][0] * f, t[w][e][1] * f);
      u[2 * e + 1] = pack_bf16(t[w][e][2] * f, t[w][e][3] * f);
    }
    *reinterpret_cast<u32x4 *>(out) = live ? u : u32x4{0, 0, 0, 0};
  }
}

// How the key blocks are cut: items of at most `budget` steps.  No block has more steps
// than the one before it (the sinks' come first, and a window or the rows left are the
// same or fewer from block to block), so the items of cut blocks are the first `cut`.
struct BwdPlan {
  int budget = 0;
  size_t items = 0;
  size_t cut = 0;
};
BwdPlan plan_bwd(const Shape &sh, size_t batch) {
  const int blocks = (int)cdiv((size_t)sh.S, (size_t)kBlk);
  int64_t total = 0, most = 1;
  for (int j = 0; j < blocks; ++j) {
    const int n = steps_of(sh, sh.S, j);
    total += n;
    most = std::max<int64_t>(most, n);
  }
  // One workgroup fits a CU, of which 256 are counted on every device (a workspace's
  // size may be asked for on another).  The time is about that of the longest item
  // where all items are resident, and the average load and half an item more beyond; an
  // item of a cut block costs about 8 steps more (its sums go through memory), and has 8
  // steps at least (whole backward with at least 4, 8, 12, us: 3 x 500 46.9, 46.4, 49.6;
  // 2 x 1000 47.2, 45.6, 48.6; 1 x 200 30.9, 33.0, 35.6).
  const int64_t wgs = (int64_t)batch * sh.Hkv, cus = 256;
  BwdPlan best;
  double best_cost = 0;
  for (int64_t n = 1; n <= 64; n += n < 8 ? 1 : n / 4) {
    const int budget = (int)std::max<int64_t>((most + n - 1) / n, 8);
    int64_t items = 0, extra = 0;
    for (int j = 0; j < blocks; ++j) {
      const int x = splits_of(sh, budget, j);
      items += x;
      if (x > 1) extra += x;
    }
    const double load = double(total + 8 * extra) * wgs / cus, item = budget + (extra ? 8 : 0);
    const double cost = items * wgs <= cus ? item : std::max(load + item / 2, item);
    if (best.budget == 0 || cost < best_cost) {
      best_cost = cost;
      best.budget = budget;
      best.items = (size_t)items;
      best.cut = (size_t)extra;
    }
    if (budget == 8) break;
  }
  return best;
}
// Items of a (sequence, kv head) that have a place among the partial sums: those of cut
// blocks.  Up to 32 MiB all items have one, which is the size that callers of shapes
// so small have known; where batches are large the uncut blocks' places are most of it
// (16 x 8192 rows, 32 + 8 heads, window 512, 4 sinks: 1200 MiB with them, 192 without).
size_t part_slots(const Shape &sh, size_t batch, const BwdPlan &p) {
  constexpr size_t kSmall = (size_t)32 << 20;
  const size_t all = batch * sh.Hkv * p.items * 2 * kBlk * kHd * sizeof(float);
  return p.cut == 0 || all <= kSmall ? p.items : p.cut;
}
// Bytes of the row statistics and of the partial sums.
size_t stat_bytes(const Shape &sh, size_t batch) {
  return roundup(batch * sh.Hq * cdiv((size_t)sh.S, (size_t)kTr) * 64 * sizeof(float), 256);
}
size_t part_bytes(const Shape &sh, size_t batch, const BwdPlan &p) {
  return p.cut == 0 ? 0
                    : batch * sh.Hkv * part_slots(sh, batch, p) * 2 * kBlk * kHd * sizeof(float);
}

Shape shape_of(size_t seq_len, size_t n_heads, size_t n_kv_heads, size_t window, size_t sinks) {
  // A window past the sequence hides nothing.
  return Shape{(int)seq_len,
               (int)n_heads,
               (int)n_kv_heads,
               (int)(window >= seq_len ? 0 : window),
               (int)(sinks < seq_len ? sinks : seq_len),
               1.0f / sqrtf((float)kHd),
               1.0f / sqrtf((float)kHd) * kLog2e};
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
                     batch * seq_len <= (size_t)INT32_MAX / 2 &&
                     (seq_len + 128) * (n_heads / n_kv_heads) <= (size_t)INT32_MAX,
                 "%s: shape too large", who);
  *sh = shape_of(seq_len, n_heads, n_kv_heads, window, sinks);
  *work = batch != 0 && seq_len != 0;
  return PRICHS_OK;
}

// A row operand: its leading dimension holds its heads, and rows and base are
// 16-byte aligned.
int check_rows(const char *who, const char *name, const void *p, size_t ld, size_t cols) {
  PRICHS_REQUIRE(p != nullptr, "%s: null pointer argument %s", who, name);
  // The kernels address up to 128 rows with 32-bit byte offsets.
  PRICHS_REQUIRE(ld >= cols && ld % 8 == 0 && ld < ((size_t)1 << 24),
                 "%s: the leading dimension %zu of %s must be a multiple of 8 elements, at least "
                 "%zu and below 2^24",
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
                                                             size_t n_heads, size_t n_kv_heads,
                                                             size_t window, size_t sinks) {
  Shape sh;
  bool work;
  if (check_shape("window_attention_backward_workspace", batch, seq_len, n_heads, n_kv_heads, kHd,
                  PRICHS_DTYPE_BF16, window, sinks, &sh, &work) != PRICHS_OK ||
      !work)
    return 0;
  return stat_bytes(sh, batch) + part_bytes(sh, batch, plan_bwd(sh, batch));
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
  const BwdPlan plan = plan_bwd(sh, batch);
  const size_t stats = stat_bytes(sh, batch), need = stats + part_bytes(sh, batch, plan);
  if (workspace_bytes < need)
    return fail(PRICHS_ERR_CAPACITY, "%s: workspace of %zu bytes, %zu needed", who,
                workspace_bytes, need);
  PRICHS_REQUIRE(workspace != nullptr && reinterpret_cast<uintptr_t>(workspace) % 16 == 0,
                 "%s: the workspace must be 16-byte aligned device memory", who);
  const int hpw = window_heads(n_heads / n_kv_heads, seq_len);
  const size_t blocks = cdiv(seq_len, (size_t)kBlk), n_qb32 = cdiv(seq_len, (size_t)(128 / hpw));
  const bool few = few_workgroups((n_heads / hpw) * batch * n_qb32);
  // Rows of a wave of the d_q kernel, by the forward's rule.  Whole
  // backward, 32 -> 16 rows, us: 1 x 777 52 -> 46, 3 x 500 56 -> 50, 1 x 4096 277 ->
  // 260, 4 x 1024 (384 workgroups) 81.6 -> 81.9, 4 x 2048 169 -> 173, 1 x 16384 1499 ->
  // 1671.
  // The d_q kernel writes the statistics of whole 32-row tiles, so its rows go to the
  // end of the last one.
  const size_t n_qb = few ? cdiv(roundup(seq_len, (size_t)kTr), (size_t)(64 / hpw)) : n_qb32;
  const size_t dq_pairs = n_heads / hpw * batch, dkv_pairs = n_kv_heads * batch;
  const bool dq_dies = !few && by_die(seq_len, sh.window, dq_pairs, n_qb),
             dkv_dies = by_die(seq_len, sh.window, dkv_pairs, plan.items);
  // Before the first launch: a call that fails leaves nothing half done.
  static LdsLimit limits[2];
  auto dkv_kern = dkv_dies ? window_dkv_kernel<true> : window_dkv_kernel<false>;
  WINDOW_TRY(raise_lds_limit(limits[dkv_dies], reinterpret_cast<const void *>(dkv_kern), kKvLds, who));
  const auto bf = [](const void *p) { return static_cast<const bf16_t *>(p); };
  const auto out = [](void *p) { return static_cast<bf16_t *>(p); };
  BwdArgs a{bf(d_o), bf(q), bf(k), bf(v), bf(o), lse, seq_lens, out(d_q), out(d_k), out(d_v),
            (int)ldd, (int)ldq, (int)ldk, (int)ldv, (int)ldo, (int)lddq, (int)lddk, (int)lddv,
            static_cast<float *>(workspace), (int)cdiv(seq_len, (size_t)kTr),
            reinterpret_cast<float *>(static_cast<char *>(workspace) + stats), plan.budget,
            (int)plan.items, (int)part_slots(sh, batch, plan), (int)n_qb, (int)dq_pairs,
            (int)dkv_pairs, sh};
  auto dq_kern = few ? (hpw == 4   ? window_dq_kernel<4, 1>
                        : hpw == 2 ? window_dq_kernel<2, 1>
                                   : window_dq_kernel<1, 1>)
                 : dq_dies ? (hpw == 4   ? window_dq_kernel<4, 2, true>
                              : hpw == 2 ? window_dq_kernel<2, 2, true>
                                         : window_dq_kernel<1, 2, true>)
                           : (hpw == 4   ? window_dq_kernel<4, 2>
                              : hpw == 2 ? window_dq_kernel<2, 2>
                                         : window_dq_kernel<1, 2>);
  hipLaunchKernelGGL(dq_kern,
                     dq_dies ? dim3((unsigned)die_grid(dq_pairs, n_qb))
                             : dim3((unsigned)(n_heads / hpw), (unsigned)batch, (unsigned)n_qb),
                     dim3(256), kQLds, as_stream(stream), a);
  PRICHS_LAUNCH_CHECK("window_attention_backward d_q launch");
  hipLaunchKernelGGL(dkv_kern,
                     dkv_dies ? dim3((unsigned)die_grid(dkv_pairs, plan.items))
                              : dim3((unsigned)plan.items, (unsigned)n_kv_heads, (unsigned)batch),
                     dim3(128 * kKg),
                     kKvLds, as_stream(stream), a);
  PRICHS_LAUNCH_CHECK("window_attention_backward d_k / d_v launch");
  if (plan.cut != 0) {
    hipLaunchKernelGGL(window_dkv_join_kernel,
                       dim3((unsigned)(kBlk / 16 * blocks), (unsigned)n_kv_heads, (unsigned)batch),
                       dim3(256), 0, as_stream(stream), a);
    PRICHS_LAUNCH_CHECK("window_attention_backward join launch");
  }
  return PRICHS_OK;
}
