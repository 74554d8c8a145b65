// What the attention sources share: the formats' sizes, MFMA operands and LDS DMA (gfx950, wave64).
#pragma once

#include "nkv_common.h"

namespace nkv {

constexpr int D = 128;
constexpr int GT = 64;              // tokens per ruler group == ring slots
constexpr int CODE_BYTES = GT * D;                        // one tensor's codes of one group
constexpr int RULER_BYTES = 4 * D * 2;                    // kst, kmn, vst, vmn of one group
// paged layout: one page = one 64-token group of one KV head, K codes | V codes | kst | kmn | vst | vmn
constexpr int PAGE_BYTES = 2 * CODE_BYTES + RULER_BYTES;  // 17 KiB, a multiple of 128
// paged per-token symmetric layout: one page = 64 tokens of one KV head, K codes | V codes |
// K scales (64 fp16) | V scales
constexpr int PAGE_TOK_BYTES = 2 * CODE_BYTES + 2 * GT * 2;  // 16640, a multiple of 128
constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;
constexpr float NEG_INF = -__builtin_huge_valf();

typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) void lds_void_t;
typedef int v2i_t __attribute__((vector_size(8)));
typedef __attribute__((address_space(3))) v2i_t lds_v2i_t;

// XOR key of the 16-byte chunk positions of LDS row `row` (a token within its group).
// K reads (16 consecutive rows, one chunk) and V transpose reads (rows 4g + {0..3} of
// two 16-row blocks, one chunk) both hit 16 distinct bank positions per 16 lanes.
__device__ __forceinline__ int swz(int row) { return ((row >> 1) & 7) ^ (((row >> 4) & 1) << 2); }

__device__ __forceinline__ float sum4rows(float v) {
  auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

__device__ __forceinline__ float4_t mfma32(half8_t a, half8_t b, float4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ half8_t as_h8(uint4 w) { return __builtin_bit_cast(half8_t, w); }

// The thread index for code that runs seldom (the tails, the chained step's merger, a softmax's slow path):
// read through an opaque move, so that values derived from it are recomputed where they are used
// rather than hoisted out of the surrounding loop and kept live across it (which exhausts the
// register file there).
__device__ __forceinline__ int tail_tid() {
  int t;
  asm volatile("v_mov_b32 %0, %1" : "=v"(t) : "v"((int)__builtin_amdgcn_workitem_id_x()));
  return t;
}

// ---------------------------------------------------------------- HBM -> LDS

__device__ __forceinline__ uint32_t lds_addr(const void* p) {
  return (uint32_t)(uintptr_t)(const lds_void_t*)p;
}

// A pointer the wave holds in common, moved to scalar registers.
__device__ __forceinline__ const void* uniform_ptr(const void* p) {
  const uint64_t v = reinterpret_cast<uint64_t>(p);
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v);
  const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)(v >> 32));
  return reinterpret_cast<const void*>(((uint64_t)hi << 32) | lo);
}

// One `global_load_lds_dwordx4`: lane L's 16 bytes at sbase + voff land at LDS byte
// address lds + 16 * L (sbase and lds are wave-uniform).
__device__ __forceinline__ void dma16(const void* sbase, uint32_t voff, uint32_t lds) {
  lds = __builtin_amdgcn_readfirstlane(lds);
  asm volatile("s_mov_b32 m0, %2\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(voff), "s"(sbase), "s"(lds) : "memory");
}

// The same, nontemporal: for the decode prefix's codes and rulers, which a step reads once
// (about 3-5% faster than the default policy on the 32k decode step).
__device__ __forceinline__ void dma16_stream(const void* sbase, uint32_t voff, uint32_t lds) {
  lds = __builtin_amdgcn_readfirstlane(lds);
  asm volatile("s_mov_b32 m0, %2\n\tglobal_load_lds_dwordx4 %0, %1 nt" ::"v"(voff), "s"(sbase), "s"(lds) : "memory");
}

__device__ __forceinline__ void wait_groups_all() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

}  // namespace nkv
