// What the attention sources share: the formats' sizes, MFMA operands, LDS DMA and the online softmax of
// a row block (gfx950, wave64).
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
constexpr float PF_TAU = 8.0f;                       // lazy softmax rescaling threshold (log2)

typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) void lds_void_t;
typedef int v2i_t __attribute__((vector_size(8)));
typedef __attribute__((address_space(3))) v2i_t lds_v2i_t;
typedef short v4s_t __attribute__((vector_size(8)));
typedef __attribute__((address_space(3))) v4s_t lds_v4s_t;

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

// Online-softmax state of one wave. m, l: head (lane & 15), log2 domain; m is a reference
// maximum (at least every score seen so far, times sl2), the weights are 2^(s sl2 - m + 15).
// acc[cb][i]: head 4*(lane>>4) + i, dim 16*cb + (lane&15), in the same scale.
struct WaveState {
  float m, l;
  float4_t acc[8];
};

__device__ __forceinline__ void state_init(WaveState& st) {
  st.m = NEG_INF;
  st.l = 0.0f;
#pragma unroll
  for (int cb = 0; cb < 8; ++cb) st.acc[cb] = float4_t{0.f, 0.f, 0.f, 0.f};
}

__device__ __forceinline__ float4_t mfma32(half8_t a, half8_t b, float4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ half8_t as_h8(uint4 w) { return __builtin_bit_cast(half8_t, w); }

// The thread index for code that runs once per layer (the tails, the chained step's merger):
// read through an opaque move, so that values derived from it are recomputed where they are used
// rather than hoisted out of the chained kernel's layer loop and kept live across it (which
// exhausts the register file there).
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

// ---------------------------------------------------------------- codes to fp16

// fp16(code * scale) for 8 signed codes sharing one fp16 scale, and for 8 codes with one
// scale each: the product of an 8-bit integer and an fp16 is exact in fp32, so the packed
// fp16 multiply rounds it once, as fp16(fp32(code) * fp32(scale)) does.
__device__ __forceinline__ half8_t dq8_sym(uint32_t w0, uint32_t w1, half2_t s) {
  const half2_t a = scodes_to_h2(w0, kSelB01) * s;
  const half2_t b = scodes_to_h2(w0, kSelB23) * s;
  const half2_t c = scodes_to_h2(w1, kSelB01) * s;
  const half2_t d = scodes_to_h2(w1, kSelB23) * s;
  return half8_t{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}
__device__ __forceinline__ half8_t dq8_sym_v(uint32_t w0, uint32_t w1, uint4 s) {
  const half2_t a = scodes_to_h2(w0, kSelB01) * as_h2(s.x);
  const half2_t b = scodes_to_h2(w0, kSelB23) * as_h2(s.y);
  const half2_t c = scodes_to_h2(w1, kSelB01) * as_h2(s.z);
  const half2_t d = scodes_to_h2(w1, kSelB23) * as_h2(s.w);
  return half8_t{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}

// ---------------------------------------------------------------- softmax

// Online softmax of one 16-row block over 64 tokens, from the raw scores S[b][i] (token
// 16b + 4g + i, row c; -inf where masked): m is a reference maximum in the log2 domain, within
// PF_TAU below the row's maximum of S * sl2, and P comes out as exp2(S sl2 - m + 15 - PF_TAU)
// <= 2^15 in two fp16 A operands (tokens of blocks 0,1 and 2,3). The row sums of P are taken on
// the matrix core by the caller (P times a ones operand, in the accumulator layout), which leaves
// the VALU the maximum, the exponentials and the conversions; the caller rescales the
// accumulators and those sums by alpha, only when m moves.
__device__ __forceinline__ void pf_softmax(WaveState& st, const float (&S)[4][4], float sl2, half8_t (&ph)[2],
                                           float& alpha_out, bool& moved_out) {
  float smax = NEG_INF;
#pragma unroll
  for (int b = 0; b < 4; ++b)
#pragma unroll
    for (int i = 0; i < 4; ++i) smax = fmaxf(smax, S[b][i]);
  smax = max4rows(smax);
  const float m_cand = fmaxf(st.m, smax * sl2);
  const float m_new = m_cand > st.m + PF_TAU ? m_cand : st.m;
  const float m_use = m_new == NEG_INF ? 0.0f : m_new;
  const float alpha = __builtin_amdgcn_exp2f(st.m - m_use);
  const float off = 15.0f - PF_TAU - m_use;
  _Float16 p16[2][8];
#pragma unroll
  for (int b = 0; b < 4; ++b)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      p16[b >> 1][4 * (b & 1) + i] = (_Float16)__builtin_amdgcn_exp2f(__builtin_fmaf(S[b][i], sl2, off));
#pragma unroll
  for (int B = 0; B < 2; ++B)
    ph[B] = half8_t{p16[B][0], p16[B][1], p16[B][2], p16[B][3], p16[B][4], p16[B][5], p16[B][6], p16[B][7]};
  moved_out = st.m != m_new;
  alpha_out = alpha;
  st.m = m_new;
}

}  // namespace nkv
