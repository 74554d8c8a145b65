// The 4-bit format of weights and cache (gfx950, wave64).
//
// 32 consecutive values of a row share a scale: with amax their largest magnitude, s = max(amax / 7, 2^-24) rounded to 8
// significant bits and held in fp16, code = clamp(rint(x / s), -7, 7), value = code * s. A code has 3 significant bits
// beside its sign and the scale 8, so that every value is an fp16 number (denormals among them: their codes' multiples of
// 2^-24, too): the matrix cores' fp16 operands are the values themselves, with no rounding. A scale whose sevenfold passes
// fp16's range is infinite, that of a group with a NaN is NaN.
//
// A weight is blocks of 16 rows and 128 columns, 1152 bytes: first 64 lanes' codes, 16 bytes each, then their scales. Lane c +
// 16 g holds row c, columns 32 g .. + 31: word k columns 8 k .. + 7 of those, nibble p code + 8 of column 2 p, nibble
// p + 4 of column 2 p + 1, so that unpack4 gives them in order. The blocks of a tile of 16 rows follow each other; rows
// and columns behind the last hold zeros. A wave's load is a block's 1024 bytes in a row: with rows of in / 2 bytes, 16
// pieces of 64 bytes, the q/k/v product of one token took 6.7 us instead of 5.5.
//
// In the cache a row is a token's 128 channels of one KV head, 64 bytes: nibble e of word w holds code + 8 of channel 8 w + e,
// K's words 4 j + g and 4 g + j in each other's place (j, g < 4), so that 16 bytes hold eight channels of each group.
// A page of the cache is 64 tokens of one KV head: K codes [64][64 bytes], V codes, K scales, V scales (256 fp16 each). The
// scales lie as the attention's lanes take them (k_scale_at, v_scale_at).
#pragma once

#include "nkv_mfma.h"

namespace nkv {

constexpr int Q4_GROUP = 32;
constexpr int Q4_ROW = D / 2;                      // bytes of a token's codes
constexpr int Q4_CODES = GT * Q4_ROW;              // one tensor's codes of a page
constexpr int Q4_SCALES = GT * (D / Q4_GROUP) * 2;  // one tensor's scales
constexpr int PAGE_Q4_BYTES = 2 * (Q4_CODES + Q4_SCALES);
static_assert(PAGE_Q4_BYTES == 9216 && PAGE_Q4_BYTES % 128 == 0, "a page is a multiple of 128 bytes");

// Where the scale of token t (0 .. 63 of its page), channels 32 grp .. + 31, stands among its tensor's. In the products
// lane c + 16 g of tile b holds token 16 (c / 4) + 4 b + c % 4 of K, so that its scores are of tokens 16 g + 4 b ..
// + 3 and the 16 tokens of a lane's scores follow each other.
// K: in order, so that the four tokens of a tile's scores follow each other.
__host__ __device__ __forceinline__ constexpr int k_scale_at(int t, int grp) { return grp * GT + t; }
// The place of word w (channels 8 w .. + 7) in a row of K's (which 0) or V's codes.
__host__ __device__ __forceinline__ constexpr int word_at(int which, int w) { return which ? w : 4 * (w & 3) + (w >> 2); }
// V: tokens r and r + 4 of eight follow each other, as the two halves of a register do after unpack4.
__host__ __device__ __forceinline__ constexpr int v_scale_at(int t, int grp) {
  return grp * GT + (t & ~7) + 2 * (t & 3) + ((t >> 2) & 1);
}

// The scale's bits for a group whose largest magnitude has the bits `amax` (of fp32; NaN above infinity).
__device__ __forceinline__ uint16_t q4_scale(uint32_t amax) {
  if (amax > 0x7f800000u) return 0x7e00u;
  const float s = bf2f(f2bf(fmaxf(__fdiv_rn(__uint_as_float(amax), 7.0f), 0x1p-24f)));
  return 7.0f * s <= 65504.0f ? f2h(s) : 0x7c00u;
}

constexpr int W4_ROWS = 16, W4_COLS = 128;
constexpr int W4_CODES = W4_ROWS * W4_COLS / 2, W4_BLOCK = W4_CODES + W4_ROWS * (W4_COLS / Q4_GROUP) * 2;
static_assert(W4_BLOCK == 1152 && W4_BLOCK % 128 == 0, "a block is a multiple of 128 bytes");

// Where row `row` (of a weight with nb blocks a row), columns 128 kb + 32 g .. + 31 are: codes, and from them the scale.
__host__ __device__ __forceinline__ int64_t w4_at(int64_t row, int64_t nb, int64_t kb, int g) {
  return ((row >> 4) * nb + kb) * W4_BLOCK + ((row & 15) + 16 * g) * 16;
}
__host__ __device__ __forceinline__ int w4_scale_from(int lane) { return W4_CODES + 2 * lane - 16 * lane; }

__device__ __forceinline__ uint32_t bias1024() {
  uint32_t b;
  asm("v_mov_b32 %0, 0x64006400" : "=v"(b));
  return b;
}

// Eight values of a lane; the four lanes 4 k .. 4 k + 3 hold a group. The packed codes, and the scale's bits in all four.
// (The quotient as a product unless it is near a half, as sym_code does.)
// ORDER: nibble e / 2 + 4 (e % 2) for value e (a weight's), else nibble e.
template <bool ORDER = false>
__device__ __forceinline__ uint32_t q4_quant8(const float (&v)[8], uint16_t& scale) {
  uint32_t m = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) m = max(m, __float_as_uint(v[e]) & 0x7fffffffu);
  m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0xB1, 0xf, 0xf, false));
  m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x4E, 0xf, 0xf, false));
  scale = q4_scale(m);
  const float s = h2f(scale), inv = __builtin_amdgcn_rcpf(s);
  uint32_t w = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float q = __fmul_rn(v[e], inv);
    float r = __builtin_rintf(q);
    if (__builtin_fabsf(q - r) > 0.5f - 0x1p-12f) r = __builtin_rintf(__fdiv_rn(v[e], s));
    w |= (uint32_t)((int)fminf(fmaxf(r, -7.0f), 7.0f) + 8) << (4 * (ORDER ? e / 2 + 4 * (e % 2) : e));
  }
  return w;
}

// Value e of a packed word (fp32).
__device__ __forceinline__ float q4_value(uint32_t w, int e, float s) { return (float)((int)((w >> (4 * e)) & 15u) - 8) * s; }

// The eight values of a packed word as fp16, in the order 0 4 1 5 2 6 3 7 of its nibbles; s: their scales (a pair's two
// halves may differ). A nibble becomes the mantissa's end of 1024 + n, or the middle of 1024 + 16 n: exact throughout. bias:
// bias1024(), in a register, so that the mask and the bias are one instruction.
__device__ __forceinline__ half8_t unpack4(uint32_t w, const half2_t (&s)[4], uint32_t bias) {
  const half2_t lo = {(_Float16)-1032.0f, (_Float16)-1032.0f}, hi = {(_Float16)-72.0f, (_Float16)-72.0f};
  const half2_t by = {(_Float16)0.0625f, (_Float16)0.0625f};
  const uint32_t x = w >> 8;
  const half2_t a = (as_h2((w & 0x000f000fu) | bias) + lo) * s[0];
  const half2_t b = (as_h2((w & 0x00f000f0u) | bias) * by + hi) * s[1];
  const half2_t c = (as_h2((x & 0x000f000fu) | bias) + lo) * s[2];
  const half2_t d = (as_h2((x & 0x00f000f0u) | bias) * by + hi) * s[3];
  return half8_t{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}
__device__ __forceinline__ half8_t unpack4(uint32_t w, half2_t s, uint32_t bias) {
  const half2_t four[4] = {s, s, s, s};
  return unpack4(w, four, bias);
}
// The codes + 8 of a packed word as fp16 denormals, in the same order: n 2^-24, in the second and fourth pair 16 n 2^-24.
__device__ __forceinline__ half8_t tiny4(uint32_t w) {
  const uint32_t x = w >> 8;
  return as_h8(uint4{w & 0x000f000fu, w & 0x00f000f0u, x & 0x000f000fu, x & 0x00f000f0u});
}
// Eight consecutive fp16 values in unpack4's order.
__device__ __forceinline__ half8_t paired(uint4 w) {
  return as_h8(uint4{perm(w.z, w.x, 0x05040100u), perm(w.z, w.x, 0x07060302u), perm(w.w, w.y, 0x05040100u),
                     perm(w.w, w.y, 0x07060302u)});
}

}  // namespace nkv
