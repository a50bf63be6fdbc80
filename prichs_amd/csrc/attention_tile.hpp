// attention_tile.hpp -- what the attention kernels share: matrix and transposing
// reads, copies straight into LDS, exchanges between a query's lanes.
#pragma once

#include <algorithm>
#include <type_traits>
#include <utility>

#include "common.hpp"

namespace prichs {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ f32x4 mfma_bf16(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// Buffer resource over `bytes` bytes from `base` (raw: stride 0, gfx9 word 3).
// Loads at offsets at or past `bytes` return zeros instead of reading memory.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_rsrc(const void *base, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(base), (short)0, (int)bytes,
                                           0x00020000);
}
// 16 bytes per lane from buffer offset voff straight into LDS at lds_dst +
// 16 * lane (lds_dst wave-uniform).
__device__ __forceinline__ void dma_16b(__amdgpu_buffer_rsrc_t r, uint32_t voff, bf16_t *lds_dst) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(
      r, (__attribute__((address_space(3))) void *)lds_dst, 16, voff, 0, 0, 0);
}
// ds_read_b64_tr_b16 as inline asm: the builtin form makes the compiler wait
// for every DMA in flight (it cannot tell the read from the DMA's target).
// OFF is the instruction's immediate byte offset.  The result is pending
// until lds_wait_tied() below, which takes the registers as operands so no
// use can be scheduled before the wait.
template <int OFF>
__device__ __forceinline__ u32x2 ds_read_tr16(uint32_t lds_byte_addr) {
  static_assert(OFF >= 0 && OFF < 65536, "ds offset is 16 bits");
  u32x2 r;
  asm volatile("ds_read_b64_tr_b16 %0, %1 offset:%2" : "=v"(r) : "v"(lds_byte_addr), "n"(OFF));
  return r;
}
__device__ __forceinline__ void lds_wait_tied(u32x2 &a, u32x2 &b, u32x2 &c, u32x2 &d, u32x2 &e,
                                              u32x2 &f, u32x2 &g, u32x2 &h) {
  asm volatile("s_waitcnt lgkmcnt(0)"
               : "+v"(a), "+v"(b), "+v"(c), "+v"(d), "+v"(e), "+v"(f), "+v"(g), "+v"(h)
               :
               : "memory");
}

__device__ __forceinline__ uint32_t pack_bf16(float a, float b) { return pack_bf16x2(a, b); }

// Max over lanes l, l ^ 16, l ^ 32, l ^ 48 (the four 16-lane groups
// sharing a query column): v_permlane16_swap exchanges odd and even 16-lane
// rows, v_permlane32_swap the two wave halves.
// The maxima are IEEE 754-2019 maximum (v_maximum3_f32 on gfx950: NaN
// propagates, so no operand needs the canonicalising pass that fmaxf's
// maxNum semantics put before each raw MFMA result).
__device__ __forceinline__ float vmax(float a, float b) { return __builtin_elementwise_maximum(a, b); }
__device__ __forceinline__ float max_across_groups(float x) {
  const uint32_t u = __float_as_uint(x);
  const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  x = vmax(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const uint32_t w = __float_as_uint(x);
  const auto b = __builtin_amdgcn_permlane32_swap(w, w, false, false);
  return vmax(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
template <bool B> using bool_c = std::integral_constant<bool, B>;
template <int I> using int_c = std::integral_constant<int, I>;
template <typename F, int... I>
__device__ __forceinline__ void static_for_impl(F &&f, std::integer_sequence<int, I...>) {
  (f(int_c<I>{}), ...);
}
// f(int_c<0>), ..., f(int_c<N - 1>): loop indices usable as template arguments.
template <int N, typename F>
__device__ __forceinline__ void static_for(F &&f) {
  static_for_impl(f, std::make_integer_sequence<int, N>{});
}

// Two bf16 with an infinity or NaN replaced by 0.
__device__ __forceinline__ uint32_t finite_bf16x2(uint32_t u) {
  if ((u & 0x7f80u) == 0x7f80u) u &= 0xffff0000u;
  if ((u & 0x7f800000u) == 0x7f800000u) u &= 0xffffu;
  return u;
}

// Query heads that share the K / V tiles of a window attention workgroup (128 / heads
// rows of each): the largest of 4, 2, 1 that divides the GQA group and leaves at most
// 65535 row blocks, a grid's third dimension (of four heads up to 2^21 - 32 rows).
inline int window_heads(size_t group, size_t seq_len) {
  int heads = group % 4 == 0 ? 4 : group % 2 == 0 ? 2 : 1;
  while (heads > 1 && cdiv(seq_len, (size_t)(128 / heads)) > 65535) heads /= 2;
  return heads;
}

// Whether a wave takes 16 query rows instead of 32: where the workgroups of 32 would
// all be resident with room to spare (two fit a CU).  attention.hip and
// window_attention.hip have what either takes.
inline bool few_workgroups(size_t wgs32) {
  return 2 * wgs32 <= 3 * (size_t)std::max(device_cu_count(), 0);
}

// Workgroups whose keys (or query rows) are their neighbours' too, on one die: of the
// eight dies, each with an L2 of its own, workgroup `id` runs on die id % 8.  A launch
// of die_grid(pairs, n) workgroups covers the ranks 0 .. n - 1 of `pairs` sequences'
// heads in runs of kDieRun neighbouring ranks, low ranks first; false: none left.
constexpr int kDieRun = 8;
__device__ __forceinline__ bool die_rank(unsigned id, int pairs, int n, int *pair, int *rank) {
  const int j = id >> 3, run = j / kDieRun * 8 + (id & 7), c = run / pairs;
  *pair = run - c * pairs;
  *rank = c * kDieRun + j % kDieRun;
  return *rank < n;
}
inline size_t die_grid(size_t pairs, size_t n) {
  return 8 * kDieRun * cdiv(pairs * cdiv(n, (size_t)kDieRun), (size_t)8);
}
// With a window, from this many rows on; below, neighbours mostly run at the same time
// on all dies, and without one the longest rows would not all come first.  In launch
// order -> by die, us: forward 1 x 16384 window 4096 393 -> 367, 1 x 8192 window 1024 79.1
// -> 73.4, window 128 31.7 -> 29.4, 1 x 4096 window 512 34.2 -> 34.4, 2 x 8192 whole 389 ->
// 395; backward 1 x 16384 1378 -> 1353, 1 x 8192 window 128 92.5 -> 88.7, 1 x 4096 104 -> 105.6.
constexpr size_t kDieRows = 8192;
inline bool by_die(size_t seq_len, size_t window, size_t pairs, size_t n) {
  constexpr size_t kMost = (size_t)1 << 21;  // workgroups, of 1024 threads at most
  return seq_len >= kDieRows && window != 0 && pairs <= kMost && die_grid(pairs, n) <= kMost;
}

}  // namespace prichs
