// attention.hip -- causal GQA self-attention forward (flash-style) on CDNA4
// MFMA, for the PrichsBlock attention sub-layer.
//
// Semantics: crates/prichs-model/src/attention.rs:94-149 -- per head h with
// kv head h / (Hq / Hkv): scores = (q . k) * scale over j <= i, softmax over
// the causal row, out = sum_j p_j v_j.  The T x T score matrix is never
// materialised: each workgroup streams 64-row K/V blocks through LDS and
// keeps an online softmax per query row: a reference max m, raised only when
// a block's max passes it by more than 2^8 in p (so the output is rescaled a
// few times per row), and the row sum l = sum p, accumulated by MFMA as P
// times a ones fragment next to O += P V.
//
// Layout per workgroup: 4 wave64s, each owning 32 query rows (two 16-row
// MFMA blocks) of one query head.  With HPW heads per workgroup the 4 waves
// are HPW heads of one kv group x (4 / HPW) row blocks, so the workgroup
// covers 128 / HPW queries and every K/V tile it stages in LDS serves HPW
// query heads (HPW = 4 at 12 Q / 3 KV heads: the whole group shares a tile).
//   S^T = K Q^T     v_mfma_f32_16x16x32_bf16(K frag, Q frag): the lane owning
//                   query column q = lane % 16 holds the scores of kv rows
//                   4*(lane/16) + r of every 16-row kv block;
//   O^T += V^T P^T  v_mfma_f32_16x16x32_bf16(V^T frag, P frag): P (bf16) is
//                   taken straight from the softmax registers -- the MFMA's
//                   k index runs over kv rows {4g..4g+3, 16+4g..16+4g+3} of
//                   each 32-row step (g = lane / 16), and the V^T fragment
//                   reads the same kv rows -- so no lane exchange is needed,
//                   and the lane that owns query q also owns its output row.
// K and V go straight from global memory to LDS (global_load_lds, no VGPR
// round trip) into two stage buffers, so the next block's tiles stream in
// while this block is computed.  Both tiles are row-major [64 kv][128 d] with
// their 16-byte chunks XOR-swizzled per row (the DMA lane for LDS slot s of
// row r fetches logical chunk s ^ key(r)): K fragments are plain 16-byte
// reads, and the V^T fragments of the P.V product come from the transposing
// LDS read ds_read_b64_tr_b16 -- within each 16-lane group it hands lane i
// element j = M[4j + i/4][i % 4] of the group's 16 x 4 loaded elements, so
// lanes reading rows r0 + m/4, columns 4 (m % 4).. of a 16-column block give
// lane i that column's 4 consecutive kv values.
#include "attention_tile.hpp"

namespace prichs {
namespace {

constexpr int kHd = 128;      // head dim supported by this kernel
constexpr int kBKV = 64;      // kv rows per block
constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kTileElems = kBKV * kHd;                   // one K or V tile [64][128]
constexpr int kStageElems = 2 * kTileElems;              // K then V
constexpr size_t kLdsBytes = 2 * (size_t)kStageElems * sizeof(bf16_t);  // two stages
// Arguments of window attention alone (prichs_hip.h).
struct WindowArgs {
  float *lse;
  const int32_t *seq_lens;
  int window, sinks;
  int pairs;  // head sets times sequences
};
constexpr size_t kWinLdsBytes = kLdsBytes + 16;  // and a flag
constexpr float kLazy = 8.0f;  // log2 headroom of the lazily raised softmax max

// Chunk keys: K fragment reads (16 kv rows, one chunk) and V transposing
// reads (4 rows x 2 chunks per 16-lane group) both land on distinct banks.
__device__ __forceinline__ int k_key(int kv) { return kv & 15; }
__device__ __forceinline__ int v_key(int kv) { return (2 * kv) & 15; }
// Element offset of (kv row, logical 16-byte chunk c) in a K / V tile.
__device__ __forceinline__ int k_off(int kv, int c) { return kv * kHd + ((c ^ k_key(kv)) << 3); }
__device__ __forceinline__ int v_off(int kv, int c) { return kv * kHd + ((c ^ v_key(kv)) << 3); }

constexpr uint32_t kTileBytes = kTileElems * sizeof(bf16_t);
constexpr uint32_t kStageBytes = kStageElems * sizeof(bf16_t);

// q/k/v/o: row r of sequence b is row b*S + r; head h of q/o starts at column
// h*128, kv head j of k/v at column j*128 (leading dimensions ldq/ldk/ldv/ldo;
// 64 rows of k or v span less than 4 GiB).
// RoPE of one Q fragment (8 consecutive head dims 8 c .. 8 c + 7, 4 pairs)
// with the cos / sin of its pairs: the reference's rotation with each
// product and each sum rounded (crates/prichs-core/src/backward.rs:175-184),
// then bf16 -- the same operations and rounding as rope_kernel, so the result
// is the bf16 value that kernel would have stored.
__device__ __forceinline__ bf16x8 rope_frag(bf16x8 f, float4 c4, float4 s4) {
#pragma clang fp contract(off)
  u32x4 u = __builtin_bit_cast(u32x4, f);
  const float c[4] = {c4.x, c4.y, c4.z, c4.w}, sn[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float q0 = __uint_as_float(u[j] << 16), q1 = __uint_as_float(u[j] & 0xffff0000u);
    const float a0 = q0 * c[j], b0 = q1 * sn[j];
    const float a1 = q0 * sn[j], b1 = q1 * c[j];
    u[j] = pack_bf16(a0 - b0, a1 + b1);
  }
  return __builtin_bit_cast(bf16x8, u);
}

// NB: 16-row query blocks per wave.  WIN: window attention -- a sliding window,
// sinks and sequences of their own lengths (the arguments in wa); row i of a
// sequence then sees the keys j <= i with i - j < window (0: all) or j < sinks.
// DIE: workgroups dealt by die (attention_tile.hpp).  LSE: the log-sum-exp is written.
// 12 + 3 heads with a window, without lse: 1 x 16384 of 4096 367 us
// (980 TFLOP/s), 4 x 2048 of 512 48 us (470), 1 x 4096 whole 74 us (700), bound as
// without one; a block of keys that some rows do not see costs its masks and a scan
// of V (a whole causal 4 x 2048 takes 65 us here and 60 there).  1 x 777 of 256 13 us:
// the latency of its five blocks of keys.
template <int HPW, int NB, bool WIN, bool DIE, bool LSE>
__device__ __forceinline__ void attn_fwd(
    const bf16_t *__restrict__ q, int ldq, const bf16_t *__restrict__ k, int ldk,
    const bf16_t *__restrict__ v, int ldv, bf16_t *__restrict__ o, int ldo, int S, int Hq,
    int group, float scale_log2, const float *__restrict__ rcos, const float *__restrict__ rsin,
    int pos_offset, WindowArgs wa) {
  static_assert(kWaves % HPW == 0, "whole row blocks per head");
  constexpr int kRowsWg = 16 * NB * kWaves / HPW;  // query rows per workgroup
  extern __shared__ __attribute__((aligned(16))) bf16_t lds[];

  // Grid (head set, sequence, query block): blocks are dispatched x-fastest,
  // so every head set's longest causal rows (the last query block) go first.
  const int n_qb = (S + kRowsWg - 1) / kRowsWg;
  const int sets = group / HPW;  // head sets per kv group
  int x = blockIdx.x, b = blockIdx.y, qb = n_qb - 1 - (int)blockIdx.z;
  if constexpr (DIE) {
    int pair, rank;
    if (!die_rank(blockIdx.x, wa.pairs, n_qb, &pair, &rank)) return;
    b = pair / (Hq / HPW), x = pair - b * (Hq / HPW), qb = n_qb - 1 - rank;
  }
  const int kvh = x / sets;
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int h = kvh * group + (x - kvh * sets) * HPW + wave % HPW;
  const int g = lane >> 4;    // 0..3
  const int l16 = lane & 15;  // 0..15

  const size_t seq0 = (size_t)b * S;
  // Rows of this sequence; those past them are padding.
  int L = S;
  if constexpr (WIN) {
    if (wa.seq_lens != nullptr) L = min(max(wa.seq_lens[b], 0), S);
  }
  const bf16_t *kbase = k + seq0 * ldk + (size_t)kvh * kHd;
  const bf16_t *vbase = v + seq0 * ldv + (size_t)kvh * kHd;

  // Query rows of this wave: q0 + 16*nb + l16 (nb < NB).
  const int q0 = qb * kRowsWg + (wave / HPW) * 16 * NB;
  if constexpr (WIN) {
    if (qb * kRowsWg >= L) {  // padding only
      for (int nb = 0; nb < NB; ++nb) {
        const int qrow = q0 + 16 * nb + l16;
        if (qrow >= S) continue;
        bf16_t *orow = o + (seq0 + qrow) * ldo + (size_t)h * kHd + 4 * g;
        for (int jd = 0; jd < 8; ++jd) *reinterpret_cast<u32x2 *>(orow + 16 * jd) = u32x2{0, 0};
        if (LSE && g == 0) wa.lse[((size_t)b * Hq + h) * S + qrow] = -INFINITY;
      }
      return;
    }
  }

  // Q fragments (B operand of S^T = K Q^T): lane holds Q[q][32kk + 8g .. +8].
  bf16x8 qf[NB][4];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    int qr = q0 + 16 * nb + l16;
    qr = qr < S ? qr : S - 1;
    const bf16_t *qrow = q + (seq0 + qr) * ldq + (size_t)h * kHd + 8 * g;
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) qf[nb][kk] = *reinterpret_cast<const bf16x8 *>(qrow + 32 * kk);
    if (rcos != nullptr) {
      // q as projected: rotate it here (the fragment's pairs are 16 kk + 4 g ..).
      const size_t cbase = (size_t)(qr + pos_offset) * (kHd / 2) + 4 * g;
#pragma unroll
      for (int kk = 0; kk < 4; ++kk)
        qf[nb][kk] = rope_frag(qf[nb][kk], *reinterpret_cast<const float4 *>(rcos + cbase + 16 * kk),
                               *reinterpret_cast<const float4 *>(rsin + cbase + 16 * kk));
    }
  }

  f32x4 oacc[8][NB];  // O^T blocks: d block jd, query block nb
#pragma unroll
  for (int jd = 0; jd < 8; ++jd)
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) oacc[jd][nb] = f32x4{0.f, 0.f, 0.f, 0.f};
  // Reference max (log2 units) of row q: p = exp2(s - m_ref).  It is only
  // raised when a block's max exceeds it by more than kLazy, so p <= 2^kLazy
  // and the output rows are rescaled a few times per row, not per block.
  float m_ref[NB];
  // Row sums of P, accumulated by MFMA against a ones fragment (every element
  // of lsum[nb] holds the sum of query row q0 + 16 nb + lane % 16).
  f32x4 lsum[NB];
  // LSE: this lane's share of the sum of P before its rounding, for lse.  The output is
  // divided by the sum of the rounded P, whose errors its own cancel with.
  float psum[NB];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    m_ref[nb] = -INFINITY;
    lsum[nb] = f32x4{0.f, 0.f, 0.f, 0.f};
    psum[nb] = 0.f;
  }
  const bf16x8 ones = __builtin_bit_cast(bf16x8, u32x4{0x3f803f80u, 0x3f803f80u, 0x3f803f80u,
                                                        0x3f803f80u});

  // kv blocks up to the last query row of the workgroup (causal).
  const int q_last = min(L, (qb + 1) * kRowsWg) - 1;
  int n_kvb = q_last / kBKV + 1;
  // With a window: the blocks that hold sinks (n_sink of them), then those from
  // the first row's window on; block_of maps an iteration to its block.
  int n_sink = 0, skip = 0;
  if constexpr (WIN) {
    const int first = wa.window == 0 ? 0 : max(0, qb * kRowsWg - wa.window + 1) / kBKV;
    n_sink = min((wa.sinks + kBKV - 1) / kBKV, first);
    skip = first - n_sink;
    n_kvb -= skip;
  }
  // The last iteration (+ 1) whose V held an infinity or NaN (behind the tiles).
  volatile int *scan_flag = reinterpret_cast<volatile int *>(lds + 2 * kStageElems);
  if constexpr (WIN) {
    if (tid == 0) *scan_flag = 0;
  }
  auto block_of = [&](int i) { return WIN && i >= n_sink ? i + skip : i; };

  // Loop-invariant LDS byte addresses of this lane's fragment reads within a
  // stage; rows 16c (K) and 32 ks2 / +16 (V) on share the chunk key and
  // become the instructions' immediate offsets, the stage a register add.
  //   K fragment: kv row l16 (+16c), logical chunk 4kk + g.
  //   V^T read:   kv row 4g + l16/4 (+32 ks2, +16), column 16 jd + 4 (l16 % 4).
  uint32_t k_addr[4], v_addr[8];
  const uint32_t lds_base =
      (uint32_t)(size_t)(const __attribute__((address_space(3))) bf16_t *)lds;
#pragma unroll
  for (int kk = 0; kk < 4; ++kk) k_addr[kk] = 2u * (uint32_t)k_off(l16, 4 * kk + g);
#pragma unroll
  for (int jd = 0; jd < 8; ++jd) {
    const int col = 16 * jd + 4 * (l16 & 3);
    v_addr[jd] = lds_base + 2u * (uint32_t)(v_off(4 * g + (l16 >> 2), col >> 3) + (col & 7));
  }
  // Loop-invariant byte offsets of this lane's DMA sources within a 64-row
  // block: wave w moves rows 16 w .. 16 w + 15 of each tile, 4 rows
  // (1 KiB) per instruction, and the lane for LDS slot (row, s) fetches
  // logical chunk s ^ key(row).
  uint32_t dk[4], dv[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = 16 * wave + 4 * i + g;
    dk[i] = 2u * ((uint32_t)row * (uint32_t)ldk + 8u * (uint32_t)(l16 ^ k_key(row)));
    dv[i] = 2u * ((uint32_t)row * (uint32_t)ldv + 8u * (uint32_t)(l16 ^ v_key(row)));
  }
  // The window's masks need registers: there all but the first of each of these
  // addresses are formed where they are used.  4 kk, 2 jd and 4 i (8 i) only reach
  // bits of the chunk index that are exclusive-ored anyway.
  auto k_at = [&](int kk) { return WIN ? k_addr[0] ^ (uint32_t)(64 * kk) : k_addr[kk]; };
  auto v_at = [&](int jd, uint32_t stage) {
    return WIN ? (v_addr[0] + stage) ^ (uint32_t)(32 * jd) : v_addr[jd] + stage;
  };
  const uint32_t xk = 16u * (uint32_t)(l16 ^ k_key(g)), rk = dk[0] - xk;
  const uint32_t xv = 16u * (uint32_t)(l16 ^ v_key(g)), rv = dv[0] - xv;

  // Block kb's K tile lives in stage buffer kb & 1 of K, its V tile in stage
  // buffer kb & 1 of V.  K runs one block ahead of V: iteration kb computes
  // S for block kb + 1 (MFMA) while the softmax of block kb (VALU) and then
  // its P.V product run, so the matrix and vector pipes overlap within a wave.
  // The buffer resources end after the sequence's last row, so rows past it
  // (last block only) load as zeros; their scores are masked.
  auto issue_tile = [&](int kb, const bf16_t *src, int ld, const uint32_t (&off)[4], uint32_t x,
                        uint32_t row, int tile) {
    bf16_t *dst = lds + (kb & 1) * kStageElems + tile * kTileElems;
    const int blk = block_of(kb);
    const uint64_t bytes = (uint64_t)(L - 1 - blk * kBKV) * 2 * (uint64_t)ld + 2 * kHd;
    const __amdgpu_buffer_rsrc_t r = buffer_rsrc(
        src + (size_t)blk * kBKV * ld, bytes > 0xffffffffull ? 0xffffffffu : (uint32_t)bytes);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t key = tile == 0 ? 64u * i : 128u * (i & 1);
      dma_16b(r, WIN ? (x ^ key) + (row + 8u * i * (uint32_t)ld) : off[i],
              dst + (16 * wave + 4 * i) * kHd);
    }
  };
  auto issue_k = [&](int kb) { issue_tile(kb, kbase, ldk, dk, xk, rk, 0); };
  auto issue_v = [&](int kb) { issue_tile(kb, vbase, ldv, dv, xv, rv, 1); };
  // Every wave's DMAs issued so far have landed (each wave waits for its own,
  // the barrier for the others'), and every wave is past the reads before it.
  // s_waitcnt vmcnt(0) (gfx9 encoding: vmcnt[3:0] | expcnt 7 << 4 |
  // lgkmcnt 15 << 8 | vmcnt[5:4] << 14).
  auto sync_tiles = [&]() {
    __builtin_amdgcn_s_waitcnt((7 << 4) | (15 << 8));
    __syncthreads();
  };

  // S^T = K Q^T of block kb: 4 kv blocks x NB query blocks; sacc[c][nb][r] =
  // raw score of (query q0 + 16nb + l16, kv 64 kb + 16c + 4g + r).
  auto compute_s = [&](int kb, f32x4 (&sacc)[4][NB]) {
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) sacc[c][nb] = f32x4{0.f, 0.f, 0.f, 0.f};
    const char *kbytes = reinterpret_cast<const char *>(lds) + (uint32_t)(kb & 1) * kStageBytes;
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
      bf16x8 kf[4];
#pragma unroll
      for (int c = 0; c < 4; ++c)
        kf[c] = *reinterpret_cast<const bf16x8 *>(kbytes + 16 * kHd * 2 * c + k_at(kk));
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) sacc[c][nb] = mfma_bf16(kf[c], qf[nb][kk], sacc[c][nb]);
    }
  };

  // Masks block kv0's scores of query block nb.
  auto hide = [&](int nb, int kv0, f32x4 (&scur)[4][NB]) {
    // Valid iff kv <= query row and kv < L, i.e. 16c + r <= lim.
    const int lim = min(q0 + 16 * nb + l16, L - 1) - kv0 - 4 * g;
    // Behind the window: 16c + r <= old, unless a sink (16c + r < sink).
    const int old = WIN && wa.window != 0 ? q0 + 16 * nb + l16 - wa.window - kv0 - 4 * g : -64;
    const int sink = WIN ? wa.sinks - kv0 - 4 * g : 0;
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        bool hidden = 16 * c + r > lim;
        if constexpr (WIN) hidden |= (16 * c + r <= old) & (16 * c + r >= sink);
        scur[c][nb][r] = hidden ? -INFINITY : scur[c][nb][r];
      }
  };
  // Whether every row of the workgroup sees all of iteration i's block.
  auto whole = [&](int i) {
    const int kv0 = block_of(i) * kBKV;
    return kv0 + kBKV <= min(qb * kRowsWg + 1, L) &&
           (wa.window == 0 || (qb + 1) * kRowsWg - 1 - kv0 < wa.window ||
            kv0 + kBKV <= wa.sinks);
  };

  // Iteration kb: S of block kb + 1 into snext (past the last block the
  // stale tile it reads gives a result nobody uses), then the softmax and
  // P.V of block kb from scur.  MASKED applies the causal / length mask
  // (blocks reaching past this wave's first query row or the sequence end).
  auto run_iter = [&](int kb, auto masked_c, f32x4 (&scur)[4][NB], f32x4 (&snext)[4][NB]) {
    constexpr bool kMasked = decltype(masked_c)::value;
    const int kv0 = block_of(kb) * kBKV;
    // K of block kb + 1 and V of block kb have landed; the buffers of K kb
    // and V kb - 1 are free for K kb + 2 and V kb + 1.
    sync_tiles();
    if (kb + 2 < n_kvb) issue_k(kb + 2);
    if (kb + 1 < n_kvb) issue_v(kb + 1);

    // Window attention decides by block, in one body, whether it is masked (the
    // waves of a workgroup agree: a masked block has one barrier more).
    bool masked = kMasked;
    if constexpr (WIN) masked = !whole(kb);
    if (WIN && masked) {
      // This block holds keys that some rows of the workgroup do not see.  Their p
      // is 0, but 0 times an infinity or NaN of V is NaN: those elements are set to
      // 0 in the tile, and added after the product to the rows that see them.  (A
      // half of u has all exponent bits set where adding one to its exponent
      // carries into the sign.)
      char *vt = reinterpret_cast<char *>(lds) + (uint32_t)(kb & 1) * kStageBytes + kTileBytes;
      uint32_t bad = 0;
#pragma unroll 1
      for (int i = 0; i < 4; ++i) {
        const u32x4 u = *reinterpret_cast<const u32x4 *>(vt + 16 * (i * kThreads + tid));
#pragma unroll
        for (int e = 0; e < 4; ++e) bad |= (u[e] & 0x7f807f80u) + 0x00800080u;
      }
      if (bad & 0x80008000u) {
#pragma unroll 1
        for (int i = 0; i < 4; ++i) {
          u32x4 u = *reinterpret_cast<const u32x4 *>(vt + 16 * (i * kThreads + tid));
#pragma unroll
          for (int e = 0; e < 4; ++e) u[e] = finite_bf16x2(u[e]);
          *reinterpret_cast<u32x4 *>(vt + 16 * (i * kThreads + tid)) = u;
        }
        *scan_flag = kb + 1;
      }
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) hide(nb, kv0, scur);
    }

    compute_s(kb + 1, snext);

    // Online softmax.  The block max is taken on raw scores (the scale is
    // positive, and rounding is monotone, so max(fl(s * c)) = fl(max(s) * c))
    // and p = exp2(s * scale_log2 - m_ref) is one fma per score.
    u32x4 pf[NB][2];  // P fragments: [nb][32-row kv step]
    float alpha[NB];
    bool raise[NB];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      if constexpr (kMasked && !WIN) hide(nb, kv0, scur);
      float mloc = -INFINITY;
#pragma unroll
      for (int c = 0; c < 4; ++c)
        mloc = vmax(vmax(vmax(mloc, scur[c][nb][0]), scur[c][nb][1]),
                    vmax(scur[c][nb][2], scur[c][nb][3]));
      mloc = max_across_groups(mloc);
      const float m_blk = mloc * scale_log2;
      // -inf + kLazy stays -inf: a row's first valid score always raises it.
      raise[nb] = m_blk > m_ref[nb] + kLazy;
      const float m_new = raise[nb] ? m_blk : m_ref[nb];
      alpha[nb] = raise[nb] ? fast_exp2(m_ref[nb] - m_new) : 1.0f;
      m_ref[nb] = m_new;
      float m_use = m_new;
      // Rows with no valid score yet keep m = -inf; exp2(-inf - -inf) would
      // be NaN.  Only a masked block can leave a row without one.
      if constexpr (kMasked || WIN) m_use = m_new == -INFINITY ? 0.f : m_new;
      const float neg_m = -m_use;
      float part[2];
#pragma unroll
      for (int ks2 = 0; ks2 < 2; ++ks2) {
        // k slots 0..3: kv block 2 ks2 (rows 4g + r); slots 4..7: block 2 ks2 + 1.
        float p[8];
#pragma unroll
        for (int h2 = 0; h2 < 2; ++h2)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            p[4 * h2 + r] = fast_exp2(fmaf(scur[2 * ks2 + h2][nb][r], scale_log2, neg_m));
        if constexpr (LSE)
          part[ks2] = ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
        pf[nb][ks2] = u32x4{pack_bf16(p[0], p[1]), pack_bf16(p[2], p[3]), pack_bf16(p[4], p[5]),
                            pack_bf16(p[6], p[7])};
      }
      if constexpr (LSE) psum[nb] = fmaf(psum[nb], alpha[nb], part[0] + part[1]);
    }
    // Pin the P fragments here: otherwise the compiler sinks the exp work
    // past the branch below, out of reach of the S MFMAs it should overlap.
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      asm volatile("" ::"v"(pf[nb][0]), "v"(pf[nb][1]));
      if constexpr (LSE) asm volatile("" : "+v"(psum[nb]));  // P need not live on for it
    }
    // Rescale the output rows where the reference max was raised (rare).
    if (__any(raise[0] || raise[NB - 1])) {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
        for (int jd = 0; jd < 8; ++jd) oacc[jd][nb] = oacc[jd][nb] * alpha[nb];
        lsum[nb] = lsum[nb] * alpha[nb];
      }
    }

    // O^T += V^T P^T: d blocks jd, 32-row kv steps ks2.  Lane m of each
    // 16-lane group reads row 32 ks2 + 4g + m/4 (and 16 rows on for the
    // upper half), columns 16 jd + 4 (m % 4) .. + 3; four d blocks per batch
    // of transposing reads.
    const uint32_t v_stage = (uint32_t)(kb & 1) * kStageBytes;
    if (WIN && masked) lds_write_barrier();  // the scan's zeros
    static_for<2>([&](auto ks2_c) {
      constexpr int ks2 = decltype(ks2_c)::value;
      constexpr int kLo = (int)kTileBytes + 2 * 32 * ks2 * kHd;  // rows 32 ks2 + ...
      constexpr int kHi = kLo + 2 * 16 * kHd;                    // rows 32 ks2 + 16 + ...
#pragma unroll
      for (int j0 = 0; j0 < 8; j0 += 4) {
        u32x2 lo[4], hi[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const uint32_t a = v_at(j0 + t, v_stage);
          lo[t] = ds_read_tr16<kLo>(a);
          hi[t] = ds_read_tr16<kHi>(a);
        }
        lds_wait_tied(lo[0], hi[0], lo[1], hi[1], lo[2], hi[2], lo[3], hi[3]);
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const bf16x8 vf = __builtin_bit_cast(bf16x8, u32x4{lo[t][0], lo[t][1], hi[t][0], hi[t][1]});
#pragma unroll
          for (int nb = 0; nb < NB; ++nb)
            oacc[j0 + t][nb] =
                mfma_bf16(vf, __builtin_bit_cast(bf16x8, pf[nb][ks2]), oacc[j0 + t][nb]);
        }
      }
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
        lsum[nb] = mfma_bf16(ones, __builtin_bit_cast(bf16x8, pf[nb][ks2]), lsum[nb]);
    });
    if (WIN && masked) {
      // The infinities and NaN that the scan took out, for the rows that see
      // them (p > 0 there: an infinity keeps its sign).
      if (*scan_flag == kb + 1) {
#pragma unroll 1
        for (int j = 0; j < kBKV && kv0 + j < L; ++j) {
          const int key = kv0 + j;
          const bf16_t *vrow = vbase + (size_t)key * ldv + 4 * g;
          bool sees[NB];
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) {
            const int row = q0 + 16 * nb + l16;
            sees[nb] = (key <= row) &
                       ((wa.window == 0) | (row - key < wa.window) | (key < wa.sinks));
          }
#pragma unroll
          for (int jd = 0; jd < 8; ++jd) {
            const u32x2 raw = *reinterpret_cast<const u32x2 *>(vrow + 16 * jd);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const uint32_t x = r & 1 ? raw[r / 2] & 0xffff0000u : raw[r / 2] << 16;
              const bool off = (x & 0x7f800000u) == 0x7f800000u;
#pragma unroll
              for (int nb = 0; nb < NB; ++nb)
                oacc[jd][nb][r] += (off & sees[nb]) ? __uint_as_float(x) : 0.f;
            }
          }
        }
      }
    }
  };

  // Blocks whose kv rows all lie at or before this wave's first query row
  // and inside the sequence run unmasked (two per loop trip, so the score
  // registers swap roles without copies); the rest (the diagonal and the
  // ragged tail) run masked.
  const int n_full = min(min(q0 + 1, S) / kBKV, n_kvb);
  f32x4 sa[4][NB], sb[4][NB];
  issue_k(0);
  sync_tiles();
  issue_v(0);
  if (n_kvb > 1) issue_k(1);
  compute_s(0, sa);
  int kb = 0;
  auto take_next = [&]() {
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) sa[c][nb] = sb[c][nb];
  };
  if constexpr (WIN) {
    for (; kb < n_kvb; kb += 2) {
      run_iter(kb, bool_c<false>{}, sa, sb);
      if (kb + 1 < n_kvb) run_iter(kb + 1, bool_c<false>{}, sb, sa);
    }
  } else {
    for (; kb + 2 <= n_full; kb += 2) {
      run_iter(kb, bool_c<false>{}, sa, sb);
      run_iter(kb + 1, bool_c<false>{}, sb, sa);
    }
    if (kb < n_full) {
      run_iter(kb, bool_c<false>{}, sa, sb);
      take_next();
      ++kb;
    }
    for (; kb < n_kvb; ++kb) {
      run_iter(kb, bool_c<true>{}, sa, sb);
      take_next();
    }
  }

  // Normalise by the row sum and store: lane holds O[q][16 jd + 4g + r].
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    // (A row of window attention sees itself at least: a sum of 0 means that
    // every score is -inf, and 0 / 0 is the softmax of that.)
    const float inv = 1.0f / (WIN ? lsum[nb][0] : fmaxf(lsum[nb][0], 1e-30f));
    const int qrow = q0 + 16 * nb + l16;
    if constexpr (LSE) {
      float l = psum[nb] + __shfl_xor(psum[nb], 16);
      l += __shfl_xor(l, 32);
      if (g == 0 && qrow < S)
        wa.lse[((size_t)b * Hq + h) * S + qrow] =
            qrow < L ? (m_ref[nb] + log2f(l)) * 0.6931471805599453f : -INFINITY;
    }
    if constexpr (WIN) {
      if (qrow >= L && qrow < S) {
        bf16_t *orow = o + (seq0 + qrow) * ldo + (size_t)h * kHd + 4 * g;
#pragma unroll
        for (int jd = 0; jd < 8; ++jd) *reinterpret_cast<u32x2 *>(orow + 16 * jd) = u32x2{0, 0};
      }
    }
    if (qrow < L) {
      bf16_t *orow = o + (seq0 + qrow) * ldo + (size_t)h * kHd + 4 * g;
#pragma unroll
      for (int jd = 0; jd < 8; ++jd) {
        const f32x4 a = oacc[jd][nb];
        *reinterpret_cast<u32x2 *>(orow + 16 * jd) =
            u32x2{pack_bf16(a[0] * inv, a[1] * inv), pack_bf16(a[2] * inv, a[3] * inv)};
      }
    }
  }
}

// The whole attention, or (WIN) window attention with lse.
template <int HPW, int NB, bool WIN, bool DIE = false>
__global__ __launch_bounds__(kThreads, 2) void attn_fwd_kernel(
    const bf16_t *__restrict__ q, int ldq, const bf16_t *__restrict__ k, int ldk,
    const bf16_t *__restrict__ v, int ldv, bf16_t *__restrict__ o, int ldo, int S, int Hq,
    int group, float scale_log2, const float *__restrict__ rcos, const float *__restrict__ rsin,
    int pos_offset, WindowArgs wa) {
  attn_fwd<HPW, NB, WIN, DIE, WIN>(q, ldq, k, ldk, v, ldv, o, ldo, S, Hq, group, scale_log2, rcos,
                                   rsin, pos_offset, wa);
}
// Window attention without lse, whose sum costs 17 vector instructions for each 64 keys and
// 16 rows (1 x 777 window 256 12.8 -> 13.0 us, 4 x 2048 window 512 48.3 -> 49.9, 1 x 16384
// window 4096 365 -> 387).
template <int HPW, int NB, bool DIE = false>
__global__ __launch_bounds__(kThreads, 2) void window_fwd_kernel(
    const bf16_t *__restrict__ q, int ldq, const bf16_t *__restrict__ k, int ldk,
    const bf16_t *__restrict__ v, int ldv, bf16_t *__restrict__ o, int ldo, int S, int Hq,
    int group, float scale_log2, const float *__restrict__ rcos, const float *__restrict__ rsin,
    int pos_offset, WindowArgs wa) {
  attn_fwd<HPW, NB, true, DIE, false>(q, ldq, k, ldk, v, ldv, o, ldo, S, Hq, group, scale_log2,
                                      rcos, rsin, pos_offset, wa);
}

}  // namespace
}  // namespace prichs

using namespace prichs;

namespace prichs {
int attention_forward_impl(const void *q, size_t ldq, const void *k, size_t ldk, const void *v,
                           size_t ldv, void *o, size_t ldo, size_t batch, size_t seq_len,
                           size_t n_heads, size_t n_kv_heads, size_t head_dim, int dtype,
                           const float *rope_cos, const float *rope_sin, size_t cache_rows,
                           size_t pos_offset, void *stream) {
  PRICHS_REQUIRE(dtype == PRICHS_DTYPE_BF16, "attention: only bf16 is supported (dtype=%d)", dtype);
  if (head_dim != (size_t)kHd)
    return fail(PRICHS_ERR_UNSUPPORTED, "attention: head_dim=%zu (only %d is supported)",
                head_dim, kHd);
  PRICHS_REQUIRE(n_heads >= 1 && n_kv_heads >= 1 && n_heads % n_kv_heads == 0,
                 "attention: n_heads=%zu must be a positive multiple of n_kv_heads=%zu",
                 n_heads, n_kv_heads);
  PRICHS_REQUIRE(ldq >= n_heads * head_dim && ldo >= n_heads * head_dim &&
                     ldk >= n_kv_heads * head_dim && ldv >= n_kv_heads * head_dim,
                 "attention: leading dimensions too small");
  PRICHS_REQUIRE(ldq % 8 == 0 && ldk % 8 == 0 && ldv % 8 == 0 && ldo % 8 == 0,
                 "attention: leading dimensions must be multiples of 8 elements");
  PRICHS_REQUIRE(batch * seq_len <= (size_t)INT32_MAX && n_heads <= 65535 && batch <= 65535 &&
                     ldq <= (size_t)INT32_MAX && ldo <= (size_t)INT32_MAX,
                 "attention: shape too large");
  // The kernel addresses a 64-row K/V block with 32-bit byte offsets.
  PRICHS_REQUIRE(ldk < ((size_t)1 << 25) && ldv < ((size_t)1 << 25),
                 "attention: ldk / ldv must be below 2^25 elements");
  if (batch == 0 || seq_len == 0) return PRICHS_OK;
  PRICHS_REQUIRE(rope_cos == nullptr || (rope_sin != nullptr && seq_len + pos_offset <= cache_rows &&
                                         pos_offset <= (size_t)INT32_MAX),
                 "attention: rope cache of %zu rows does not cover positions %zu + %zu",
                 cache_rows, pos_offset, seq_len);
  PRICHS_REQUIRE(q && k && v && o, "attention: null pointer argument");
  const uintptr_t al = reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) |
                       reinterpret_cast<uintptr_t>(v) | reinterpret_cast<uintptr_t>(o);
  PRICHS_REQUIRE(al % 16 == 0, "attention: q/k/v/o must be 16-byte aligned");
  const int group = (int)(n_heads / n_kv_heads);
  // Heads per workgroup: the largest of 4, 2, 1 dividing the GQA group.
  const int hpw = group % 4 == 0 ? 4 : group % 2 == 0 ? 2 : 1;
  int n_qb = (int)cdiv(seq_len, (size_t)(32 * kWaves / hpw));
  const float scale_log2 = (1.0f / sqrtf((float)head_dim)) * 1.4426950408889634f;
  PRICHS_REQUIRE(n_qb <= 65535, "attention: seq_len too large");
  // 16 query rows per wave instead of 32 where the workgroups would all be
  // resident with room to spare (two fit a CU): each walks its causal K / V
  // blocks one after the other, and half the products and exponentials per
  // block shorten that chain; beyond, they only read every K / V tile twice as
  // often.  The same operations per row, so the same bits.  MI355X, 12 + 3
  // heads, 32 -> 16 rows, us: 1 x 333 11.2 -> 9.1, 1 x 777 19.1 -> 13.5, 1 x
  // 2048 41.2 -> 31.0, 4 x 1024 (384 workgroups) 26.6 -> 24.1, 4 x 2048 (768)
  // 60.3 -> 69.8.
  const bool few = few_workgroups((n_heads / hpw) * batch * (size_t)n_qb);
  if (few) n_qb = (int)cdiv(seq_len, (size_t)(16 * kWaves / hpw));
  const dim3 grid((unsigned)(n_heads / hpw), (unsigned)batch, (unsigned)n_qb);
  auto kern = few ? (hpw == 4   ? attn_fwd_kernel<4, 1, false>
                     : hpw == 2 ? attn_fwd_kernel<2, 1, false>
                                : attn_fwd_kernel<1, 1, false>)
                  : (hpw == 4   ? attn_fwd_kernel<4, 2, false>
                     : hpw == 2 ? attn_fwd_kernel<2, 2, false>
                                : attn_fwd_kernel<1, 2, false>);
  hipLaunchKernelGGL(kern, grid, dim3(kThreads), kLdsBytes, as_stream(stream),
                     static_cast<const bf16_t *>(q), (int)ldq, static_cast<const bf16_t *>(k),
                     (int)ldk, static_cast<const bf16_t *>(v), (int)ldv,
                     static_cast<bf16_t *>(o), (int)ldo, (int)seq_len, (int)n_heads, group,
                     scale_log2, rope_cos, rope_sin, (int)pos_offset, WindowArgs{});
  PRICHS_LAUNCH_CHECK("attention launch");
  return PRICHS_OK;
}

int window_attention_launch(const void *q, size_t ldq, const void *k, size_t ldk, const void *v,
                            size_t ldv, void *o, size_t ldo, float *lse, const int32_t *seq_lens,
                            size_t batch, size_t seq_len, size_t n_heads, size_t n_kv_heads,
                            size_t window, size_t sinks, void *stream) {
  const int group = (int)(n_heads / n_kv_heads);
  const int hpw = window_heads((size_t)group, seq_len);
  const size_t n_qb32 = cdiv(seq_len, (size_t)(32 * kWaves / hpw));
  // 16 query rows per wave by attention's rule.  32 -> 16 rows, us: 1 x 777 window 256
  // 17.7 -> 12.8, 3 x 500 window 128 15.4 -> 11.6, 1 x 4096 whole 95.6 -> 76.0, 1 x 2048
  // window 512 23.8 -> 22.0, 4 x 1024 window 256 (384 workgroups) 25.5 -> 26.4, 4 x 2048
  // window 512 48.8 -> 52.6, 1 x 16384 window 4096 414 -> 493.
  const bool few = few_workgroups((n_heads / hpw) * batch * n_qb32);
  const size_t n_qb = few ? cdiv(seq_len, (size_t)(16 * kWaves / hpw)) : n_qb32;
  const float scale_log2 = (1.0f / sqrtf((float)kHd)) * 1.4426950408889634f;
  const size_t pairs = n_heads / hpw * batch;
  const bool dies = !few && by_die(seq_len, window, pairs, n_qb);
  const dim3 grid = dies ? dim3((unsigned)die_grid(pairs, n_qb))
                         : dim3((unsigned)(n_heads / hpw), (unsigned)batch, (unsigned)n_qb);
  static const struct {
    decltype(&attn_fwd_kernel<4, 2, true>) with_lse, without;
    int hpw;
    bool few, dies;
  } kinds[] = {{attn_fwd_kernel<4, 1, true>, window_fwd_kernel<4, 1>, 4, true, false},
               {attn_fwd_kernel<2, 1, true>, window_fwd_kernel<2, 1>, 2, true, false},
               {attn_fwd_kernel<1, 1, true>, window_fwd_kernel<1, 1>, 1, true, false},
               {attn_fwd_kernel<4, 2, true>, window_fwd_kernel<4, 2>, 4, false, false},
               {attn_fwd_kernel<2, 2, true>, window_fwd_kernel<2, 2>, 2, false, false},
               {attn_fwd_kernel<1, 2, true>, window_fwd_kernel<1, 2>, 1, false, false},
               {attn_fwd_kernel<4, 2, true, true>, window_fwd_kernel<4, 2, true>, 4, false, true},
               {attn_fwd_kernel<2, 2, true, true>, window_fwd_kernel<2, 2, true>, 2, false, true},
               {attn_fwd_kernel<1, 2, true, true>, window_fwd_kernel<1, 2, true>, 1, false, true}};
  static LdsLimit limits[9][2];
  int i = 0;
  while (kinds[i].hpw != hpw || kinds[i].few != few || kinds[i].dies != dies) ++i;
  const auto kern = lse != nullptr ? kinds[i].with_lse : kinds[i].without;
  if (int rc = raise_lds_limit(limits[i][lse != nullptr], reinterpret_cast<const void *>(kern),
                               kWinLdsBytes, "window_attention"))
    return rc;
  hipLaunchKernelGGL(kern, grid, dim3(kThreads), kWinLdsBytes, as_stream(stream),
                     static_cast<const bf16_t *>(q), (int)ldq, static_cast<const bf16_t *>(k),
                     (int)ldk, static_cast<const bf16_t *>(v), (int)ldv,
                     static_cast<bf16_t *>(o), (int)ldo, (int)seq_len, (int)n_heads, group,
                     scale_log2, nullptr, nullptr, 0,
                     WindowArgs{lse, seq_lens, (int)window, (int)sinks, (int)pairs});
  PRICHS_LAUNCH_CHECK("window_attention launch");
  return PRICHS_OK;
}
}  // namespace prichs

extern "C" int prichs_attention_forward(const void *q, size_t ldq, const void *k, size_t ldk,
                                        const void *v, size_t ldv, void *o, size_t ldo,
                                        size_t batch, size_t seq_len, size_t n_heads,
                                        size_t n_kv_heads, size_t head_dim, int dtype,
                                        void *stream) {
  return attention_forward_impl(q, ldq, k, ldk, v, ldv, o, ldo, batch, seq_len, n_heads,
                                n_kv_heads, head_dim, dtype, nullptr, nullptr, 0, 0, stream);
}

extern "C" int prichs_attention_forward_rope_q(const void *q, size_t ldq, const void *k,
                                               size_t ldk, const void *v, size_t ldv, void *o,
                                               size_t ldo, size_t batch, size_t seq_len,
                                               size_t n_heads, size_t n_kv_heads,
                                               size_t head_dim, int dtype, const float *rope_cos,
                                               const float *rope_sin, size_t cache_rows,
                                               size_t pos_offset, void *stream) {
  PRICHS_REQUIRE(rope_cos && rope_sin, "attention_rope_q: null RoPE table");
  return attention_forward_impl(q, ldq, k, ldk, v, ldv, o, ldo, batch, seq_len, n_heads,
                                n_kv_heads, head_dim, dtype, rope_cos, rope_sin, cache_rows,
                                pos_offset, stream);
}

// ---------------------------------------------------------------------------
// f32 causal attention with materialised probabilities: the computation of
// the reference's per-head CPU attention (crates/prichs-model/src/
// attention.rs:96-149) for one sequence, keeping the [H, T, T] probability
// matrix that the reference's host-slice GPU method returns
// (gpu_batched_attention_forward, crates/prichs-cuda/src/engine.rs:1181-1405).
// One wave per (query row i, head h):
//   s_j = (sum_c q[i][c] k[j][c]) * scale for j <= i (each a sequential sum
//   over c, lanes over j), written into the probability row;
//   m = max_j s_j (exact in any order); e_j = expf(s_j - m);
//   sum of e_j by a fixed wave-tree order; p_j = e_j * (1 / max(sum, 1e-9));
//   zeros past the diagonal; ctx[i][h][c] = sum_j p_j v[j][c] with j
//   ascending (lanes over c).
// ---------------------------------------------------------------------------
namespace prichs {
namespace {
__global__ __launch_bounds__(64) void attn_probs_f32_kernel(
    const float *__restrict__ q, const float *__restrict__ k, const float *__restrict__ v,
    float *__restrict__ probs, float *__restrict__ ctx, int T, int H, int group, int hd,
    float scale) {
#pragma clang fp contract(off)
  extern __shared__ float srow[];  // the row's scores, then probabilities [T]
  const int i = blockIdx.x, h = blockIdx.y, lane = threadIdx.x;
  const int kvh = h / group;
  const long long ldq = (long long)H * hd, ldk = (long long)(H / group) * hd;
  const float *qr = q + (long long)i * ldq + (long long)h * hd;
  float mx = -INFINITY;
  for (int j = lane; j <= i; j += 64) {
    const float *kr = k + (long long)j * ldk + (long long)kvh * hd;
    float dot = 0.0f;
    for (int c = 0; c < hd; ++c) {
      const float p = qr[c] * kr[c];
      dot = dot + p;
    }
    const float s = dot * scale;
    srow[j] = s;
    mx = fmaxf(mx, s);
  }
  for (int m = 32; m >= 1; m >>= 1) mx = fmaxf(mx, __shfl_xor(mx, m));
  float sum = 0.0f;
  for (int j = lane; j <= i; j += 64) {
    const float e = expf(srow[j] - mx);
    srow[j] = e;
    sum = sum + e;
  }
  for (int m = 1; m < 64; m <<= 1) sum = sum + __shfl_xor(sum, m);
  const float inv = 1.0f / fmaxf(sum, 1e-9f);
  float *row = probs + ((long long)h * T + i) * T;
  for (int j = lane; j < T; j += 64) {
    const float p = j <= i ? srow[j] * inv : 0.0f;
    if (j <= i) srow[j] = p;
    row[j] = p;
  }
  __syncthreads();  // every lane's probabilities are in LDS
  for (int c = lane; c < hd; c += 64) {
    float acc = 0.0f;
    for (int j = 0; j <= i; ++j) {
      const float p = srow[j] * v[(long long)j * ldk + (long long)kvh * hd + c];
      acc = acc + p;
    }
    ctx[(long long)i * ldq + (long long)h * hd + c] = acc;
  }
}
}  // namespace
}  // namespace prichs

extern "C" int prichs_attention_probs_f32(const float *q, const float *k, const float *v,
                                          float *probs, float *ctx, size_t seq_len,
                                          size_t n_heads, size_t n_kv_heads, size_t head_dim,
                                          void *stream) {
  PRICHS_REQUIRE(n_heads >= 1 && n_kv_heads >= 1 && n_heads % n_kv_heads == 0,
                 "attention_probs: n_heads=%zu must be a positive multiple of n_kv_heads=%zu",
                 n_heads, n_kv_heads);
  PRICHS_REQUIRE(head_dim >= 1 && head_dim <= 65536 && n_heads <= 65535,
                 "attention_probs: shape too large");
  if (seq_len > 16384)
    return fail(PRICHS_ERR_UNSUPPORTED, "attention_probs: seq_len=%zu above 16384 (one row of "
                "scores is kept in LDS)", seq_len);
  if (seq_len == 0) return PRICHS_OK;
  PRICHS_REQUIRE(q && k && v && probs && ctx, "attention_probs: null pointer argument");
  const float scale = 1.0f / sqrtf((float)head_dim);
  hipLaunchKernelGGL(attn_probs_f32_kernel, dim3((unsigned)seq_len, (unsigned)n_heads), dim3(64),
                     seq_len * sizeof(float), as_stream(stream), q, k, v, probs, ctx,
                     (int)seq_len, (int)n_heads,
                     (int)(n_heads / n_kv_heads), (int)head_dim, scale);
  PRICHS_LAUNCH_CHECK("attention_probs launch");
  return PRICHS_OK;
}
