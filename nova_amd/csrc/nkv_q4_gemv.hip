// The decode step's projections with 4-bit weights (nkv_q4.h) for one token or a few: y = W xn (+ residual), and the
// first half of a SwiGLU block, xn = x or its RMSNorm.
//
// On the matrix cores: tiles of 16 rows of W times tiles of 16 columns. Lane c + 16 g takes row c's group g of a block's 128
// inputs, 16 bytes. xn is held in fp16 (parts_of it), scaled by a power of two of the token's own, so that bf16's range
// and large gammas stay within fp16's. The waves of a workgroup cut the inputs among them, a block in turn; everything else in fp32,
// with one rounding at the end. Bound by the weights' bytes, and by a launch's chain of loads that wait for each other.
//
// Three forms, by the tokens and by what is to be done to x:
// - product4_few_kernel: up to 4 tokens with a norm (or bf16), more for small weights (few_each), one launch;
// - product4_kernel: up to 16 tokens of fp16 as they are, one launch;
// - product4_many_kernel: the rest, after xn_kernel has laid xn out as the products take it.

#include <algorithm>
#include <type_traits>

#include "nkv_paged.h"
#include "nkv_q4.h"

namespace nkv {

namespace {

constexpr int PB = 128;       // inputs of a block: four products deep
constexpr int P_IN = 1 << 20;  // inputs, at most
constexpr int64_t P_TOKENS = (int64_t(1) << 20) - 16;
constexpr int XCDS = 8;       // workgroups are dealt to them in turn

struct ProductArgs {
  const uint8_t* x;        // [tokens][in]
  const uint8_t* gamma;    // [in] or NULL
  float eps;
  const uint8_t* w4;       // blocks of 16 rows and 128 inputs
  int64_t out;             // outputs a token (SwiGLU: half the rows)
  int in;
  const uint8_t* residual;  // [tokens][out] or NULL
  uint8_t* y;
  int64_t tokens;
  const float* unit;  // [tokens], or NULL: 1
};

template <int DT>
__device__ __forceinline__ float load1(const uint8_t* p, int64_t i) {
  const uint16_t b = reinterpret_cast<const uint16_t*>(p)[i];
  return DT == NKV_F16 ? h2f(b) : bf2f(b);
}

// ---------------------------------------------------------------- xn

// A token's norm factor and the power of two that its xn is held in: the largest comes to 2^14 (not finite: 1).
struct Factor {
  float norm, inverse, unit;
};
__device__ __forceinline__ Factor factor_of(float ss, float top, bool norm, int in, float eps) {
  const float r = norm ? rsqrtf(ss / (float)in + eps) : 1.0f;
  top *= r;
  const int ex = top > 0.0f && top < 3e38f ? max((int)(__float_as_uint(top) >> 23) - 127 - 14, -100) : 0;
  return {r, __uint_as_float((uint32_t)(127 - ex) << 23), __uint_as_float((uint32_t)(127 + ex) << 23)};
}
// What eight values add to a token's sum of squares and largest product with gamma.
__device__ __forceinline__ void measure8(const float (&v)[8], const float (&gv)[8], float& ss, float& top) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    ss = __builtin_fmaf(v[e], v[e], ss);
    top = fmaxf(top, __builtin_fabsf(v[e] * gv[e]));
  }
}
// xn of eight inputs as fp16, and what that leaves off (lo).
__device__ __forceinline__ uint4 xn8(const float (&v)[8], const float (&gv)[8], const Factor& f, uint4& lo) {
  uint32_t h[4], l[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float a = v[2 * e] * f.norm * gv[2 * e] * f.inverse, b = v[2 * e + 1] * f.norm * gv[2 * e + 1] * f.inverse;
    const uint16_t ha = f2h(a), hb = f2h(b);
    h[e] = (uint32_t)ha | ((uint32_t)hb << 16);
    l[e] = (uint32_t)f2h(a - h2f(ha)) | ((uint32_t)f2h(b - h2f(hb)) << 16);
  }
  lo = uint4{l[0], l[1], l[2], l[3]};
  return uint4{h[0], h[1], h[2], h[3]};
}

// The fp16 parts that xn is held in: two where a norm made it of fp16 inputs, whose product would else have 1.4 to 1.6 times
// the error of a result that is rounded once, a SwiGLU's 1.8 times; in bf16's error nothing of it shows.
constexpr int parts_of(int dt, bool norm) { return dt == NKV_F16 && norm ? 2 : 1; }
// xn once for all workgroups of a product, one token a workgroup, as operands: piece (block kb, k, tile n, lane c + 16 g) of 16
// bytes holds token 16 n + c's inputs 128 kb + 32 g + 8 k .. + 7 (zeros behind the last). Tiles are counted in passes of
// NT, each of which lies together. P: parts of xn (parts_of), the second of tile n as tile NT + n.
template <int DT, int P>
__global__ __launch_bounds__(256) void xn_kernel(ProductArgs a, int nt, uint8_t* xn, float* unit) {
  __shared__ float part[2][4];
  const int tid = threadIdx.x;
  const int64_t t = blockIdx.x;
  const uint8_t* x = a.x + t * a.in * 2;
  float ss = 0.0f, top = 0.0f, v[8], gv[8];
  constexpr int KEEP = 2;  // chunks held from the first pass to the second
  Raw8<DT> r[KEEP], gr[KEEP];
  const auto load = [&](int i, Raw8<DT>& xr, Raw8<DT>& g8) {
    xr.load(x + 2 * i);
    if (a.gamma) g8.load(a.gamma + 2 * i);
  };
  const auto get = [&](const Raw8<DT>& xr, const Raw8<DT>& g8) {
    xr.get(v);
    if (a.gamma) {
      g8.get(gv);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) gv[e] = 1.0f;
    }
  };
#pragma unroll
  for (int k = 0; k < KEEP; ++k)
    if (const int i = 8 * tid + 2048 * k; i < a.in) load(i, r[k], gr[k]);
#pragma unroll
  for (int k = 0; k < KEEP; ++k)
    if (8 * tid + 2048 * k < a.in) {
      get(r[k], gr[k]);
      measure8(v, gv, ss, top);
    }
  for (int i = 8 * tid + 2048 * KEEP; i < a.in; i += 2048) {
    Raw8<DT> x8, g8;
    load(i, x8, g8);
    get(x8, g8);
    measure8(v, gv, ss, top);
  }
  ss = sum4rows(row16_sum(ss));
  top = max4rows(row16_max(top));
  if ((tid & 63) == 0) part[0][tid >> 6] = ss, part[1][tid >> 6] = top;
  __syncthreads();
  ss = (part[0][0] + part[0][1]) + (part[0][2] + part[0][3]);
  top = fmaxf(fmaxf(part[1][0], part[1][1]), fmaxf(part[1][2], part[1][3]));
  const Factor f = factor_of(ss, top, a.gamma, a.in, a.eps);
  const int blocks = (a.in + PB - 1) / PB, tile = (int)(t / 16), n = tile % nt;
  uint8_t* to = xn + (int64_t)(tile - n) * (P * blocks) * 4096 + n * 1024 + (int)(t & 15) * 16;
  const auto store = [&](int i, uint4 u, uint4 lo) {  // input i: block i / 128, g, k
    uint8_t* at = to + ((int64_t)(i >> 7) * 4 + ((i >> 3) & 3)) * (P * nt * 1024) + ((i >> 5) & 3) * 256;
    *reinterpret_cast<uint4*>(at) = u;
    if constexpr (P == 2) *reinterpret_cast<uint4*>(at + nt * 1024) = lo;
  };
  uint4 lo = {0, 0, 0, 0};
#pragma unroll
  for (int k = 0; k < KEEP; ++k)
    if (const int i = 8 * tid + 2048 * k; i < a.in) {
      get(r[k], gr[k]);
      const uint4 hi = xn8(v, gv, f, lo);
      store(i, hi, lo);
    }
  for (int i = 8 * tid + 2048 * KEEP; i < a.in; i += 2048) {
    Raw8<DT> x8, g8;
    load(i, x8, g8);
    get(x8, g8);
    const uint4 hi = xn8(v, gv, f, lo);
    store(i, hi, lo);
  }
  for (int i = a.in + 8 * tid; i < blocks * PB; i += 2048) store(i, uint4{0, 0, 0, 0}, uint4{0, 0, 0, 0});
  if (tid == 0) unit[t] = f.unit;
}

// ---------------------------------------------------------------- the weights of a wave

// RT: tiles of 16 rows; GATED: the first half of them are gates, the others their up rows. W: the workgroup's waves.
template <int RT, bool GATED, int W, int AHEAD>
struct Weights {
  static constexpr int TILES = GATED ? RT / 2 : RT;  // of 16 outputs
  const uint8_t* wp[RT];
  uint4 w[AHEAD][RT];
  uint16_t s[AHEAD][RT];
  int from[RT];
  uint32_t bias = bias1024();
  __device__ __forceinline__ Weights(const ProductArgs& a, int64_t o0, int lane, int blocks) {
#pragma unroll
    for (int r = 0; r < RT; ++r) {  // (outputs behind the last: the last, not stored)
      const int64_t row = min(o0 + 16 * (r % TILES) + (lane & 15), a.out - 1) + (r >= TILES ? a.out : 0);
      wp[r] = a.w4 + w4_at(row, blocks, 0, lane >> 4);
      from[r] = w4_scale_from((int)(row & 15) + (lane & 48));
    }
  }
  __device__ __forceinline__ void load(int e, int kb) {
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      const uint8_t* p = wp[r] + (int64_t)kb * W4_BLOCK;
      const u32x4_t v = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(p));
      w[e][r] = uint4{v.x, v.y, v.z, v.w};
      s[e][r] = *reinterpret_cast<const uint16_t*>(p + from[r]);
    }
  }
  __device__ __forceinline__ half8_t operand(int e, int r, int k) const {
    const half2_t sc = as_h2((uint32_t)s[e][r] * 0x10001u);
    const uint4& x = w[e][r];
    return unpack4(k == 0 ? x.x : k == 1 ? x.y : k == 2 ? x.z : x.w, sc, bias);
  }
};

// The waves' sums into one, and out, a tile of outputs at a time: tokens t0 .. t0 + nt - 1, outputs o0 ... red: room for
// red_floats. PER: columns of a token.
constexpr int red_floats(int nt, bool gated, int w) { return w * (gated ? 2 : 1) * nt * 16 * 17; }
template <int DT, int RT, int NT, bool GATED, int W, int PER = 1>
__device__ __forceinline__ void finish(const ProductArgs& a, const float4_t (&acc)[RT][NT], float* red, int64_t t0, int nt,
                                       int64_t o0, const float* unit) {
  constexpr int HALVES = GATED ? 2 : 1, TILES = RT / HALVES;
  const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4, wave = tid >> 6;
#pragma unroll
  for (int r = 0; r < TILES; ++r) {
    if (r) __syncthreads();
#pragma unroll
    for (int h = 0; h < HALVES; ++h)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) red[(((wave * HALVES + h) * NT + n) * 16 + 4 * g + i) * 17 + c] = acc[r + h * TILES][n][i];
    __syncthreads();
    for (int i = tid; i < NT * 256; i += 64 * W) {
      const int row = i & 15, t16 = (i >> 4) & 15, n = i >> 8, t = (16 * n + t16) / PER;
      const int64_t o = o0 + 16 * r + row;
      if (t >= nt || o >= a.out || t16 % PER) continue;
      float v[2] = {0.0f, 0.0f};
#pragma unroll
      for (int h = 0; h < HALVES; ++h)
#pragma unroll
        for (int q = 0; q < W; ++q) v[h] += red[(((q * HALVES + h) * NT + n) * 16 + row) * 17 + t16];
      const float f = unit ? unit[t] : 1.0f;
      v[0] *= f;
      v[1] *= f;
      if constexpr (GATED) v[0] = v[0] / (1.0f + expf(-v[0])) * v[1];
      const int64_t at = (t0 + t) * a.out + o;
      if (a.residual) v[0] += load1<DT>(a.residual, at);
      reinterpret_cast<uint16_t*>(a.y)[at] = DT == NKV_F16 ? f2h(v[0]) : f2bf(v[0]);
    }
  }
}

// ---------------------------------------------------------------- a few tokens: one launch
//
// Passes of up to 4 tokens, which leave most of a product's 16 columns free: column 4 t + j takes token t's group j of a block alone (its
// other inputs are 0), so that a group's sum comes out by itself and the scales are applied to it, 4 products' results
// instead of 32 operands. The codes then need no arithmetic: n = code + 8 is an fp16 denormal, n 2^-24 (a nibble at the
// mantissa's end) or 16 n 2^-24 (the next one; its inputs are held over 16), which the matrix cores take as they are: 5
// instructions for 8 codes instead of 13. The offset's share, -8 2^-24 sum(x), starts the sums.
// Each workgroup makes its tokens' xn itself, in LDS, while its weights are on the way; the waves are shared out to the tokens
// (a power of two of them, `each` waves a token), a lane takes up to KX chunks of eight inputs.

constexpr int FEW_W = 4, FEW_KX = 5, FEW_AHEAD = 5;

// M: the products that xn's parts take. One is enough for two tokens' two parts: a part is a token to the columns.

template <int DT, int RT, int M>
__global__ __launch_bounds__(64 * FEW_W, RT == 1 ? 4 : 3) void product4_few_kernel(ProductArgs a, int each) {
  constexpr int W = FEW_W, KX = FEW_KX, AHEAD = FEW_AHEAD, P = parts_of(DT, true);
  extern __shared__ __attribute__((aligned(16))) uint8_t xs[];  // [tokens][P][in + 8] fp16, the groups' offsets; sums, at the end
  __shared__ float2 part[W];
  __shared__ float unit[4];
  __shared__ __attribute__((aligned(16))) uint4 zeros[4];
  const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t t0 = W / each * (int64_t)blockIdx.y;
  const int nt = (int)min<int64_t>(W / each, a.tokens - t0), n8 = a.in / 8, blocks = (a.in + PB - 1) / PB;
  const int token = wave / each, at0 = 64 * (wave % each) + lane;  // this lane's chunks: at0 + 64 each k

  Raw8<DT> xr[KX], gr[KX];
  const uint8_t* x = a.x + (t0 + token) * a.in * 2;
#pragma unroll
  for (int k = 0; k < KX; ++k) {
    const int i = at0 + 64 * each * k;
    xr[k].zero();
    gr[k].zero();
    if (token < nt && i < n8) {
      xr[k].load(x + 16 * i);
      if (a.gamma) gr[k].load(a.gamma + 16 * i);
    }
  }
  // tile r of the workgroup (RT 2: the up rows of the first's gates): codes as the lanes lie, and the scales of rows
  // 4 g .. + 3, group c % 4, as their sums come out
  const uint8_t* wp[RT];
  uint4 w[AHEAD][RT];
  uint2 s[AHEAD][RT];
#pragma unroll
  for (int r = 0; r < RT; ++r) wp[r] = a.w4 + ((int64_t)blockIdx.x + r * (a.out / 16)) * blocks * W4_BLOCK;
  auto load = [&](int e, int kb) {
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      const uint8_t* p = wp[r] + (int64_t)kb * W4_BLOCK;
      const u32x4_t v = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(p + 16 * lane));
      w[e][r] = uint4{v.x, v.y, v.z, v.w};
      s[e][r] = *reinterpret_cast<const uint2*>(p + W4_CODES + 8 * g + 32 * (c & 3));
    }
  };
#pragma unroll
  for (int e = 0; e < AHEAD; ++e)
    if (wave + W * e < blocks) load(e, wave + W * e);

  const int part_size = 2 * (blocks * PB) + 16;  // (the rows' chunks fall on different banks)
  const int stride = P * part_size;              // bytes of a token
  float* offset = reinterpret_cast<float*>(xs + nt * stride);  // [tokens][P][4 blocks]
  float v[8], gv[8];
  auto values = [&](int k) {
    xr[k].get(v);
    if (a.gamma) {
      gr[k].get(gv);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) gv[e] = 1.0f;
    }
  };
  float ss = 0.0f, top = 0.0f;
#pragma unroll
  for (int k = 0; k < KX; ++k)
    if (64 * (wave % each + each * k) < n8) {  // (the wave agrees)
      values(k);
      measure8(v, gv, ss, top);
    }
  ss = sum4rows(row16_sum(ss));
  top = max4rows(row16_max(top));
  if (lane == 0) part[wave] = float2{ss, top};
  if (tid < 4) zeros[tid] = uint4{0, 0, 0, 0};
  __syncthreads();
#pragma unroll
  for (int k = 0; k < KX; ++k)  // (converted again below, for want of registers)
    asm volatile("" : "+v"(xr[k].w[0].x), "+v"(xr[k].w[0].y), "+v"(xr[k].w[0].z), "+v"(xr[k].w[0].w),
                 "+v"(gr[k].w[0].x), "+v"(gr[k].w[0].y), "+v"(gr[k].w[0].z), "+v"(gr[k].w[0].w));
  ss = top = 0.0f;
  for (int q = token * each; q < (token + 1) * each; ++q) ss += part[q].x, top = fmaxf(top, part[q].y);
  const Factor f = factor_of(ss, top, a.gamma, a.in, a.eps);
  if (wave % each == 0 && lane == 0) unit[token] = f.unit * 0x1p24f;
  if (token < nt) {
#pragma unroll
    for (int k = 0; k < KX; ++k) {
      const int i = at0 + 64 * each * k;
      if (64 * (wave % each + each * k) >= blocks * (PB / 8)) break;  // (the wave agrees)
      values(k);  // (behind the inputs: zeros)
      uint32_t h[P][4];
      float sum[P] = {};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float by = e & 1 ? f.inverse * 0.0625f : f.inverse;
        float a0 = v[2 * e] * f.norm * gv[2 * e] * by, a1 = v[2 * e + 1] * f.norm * gv[2 * e + 1] * by;
#pragma unroll
        for (int p = 0; p < P; ++p) {
          const uint16_t h0 = f2h(a0), h1 = f2h(a1);
          h[p][e] = (uint32_t)h0 | ((uint32_t)h1 << 16);
          sum[p] = __builtin_fmaf(h2f(h0) + h2f(h1), e & 1 ? 16.0f : 1.0f, sum[p]);
          a0 -= h2f(h0);
          a1 -= h2f(h1);
        }
      }
#pragma unroll
      for (int p = 0; p < P; ++p) {
        sum[p] += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(sum[p]), 0xB1, 0xf, 0xf, false));
        sum[p] += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(sum[p]), 0x4E, 0xf, 0xf, false));
        if (i < blocks * (PB / 8)) {
          *reinterpret_cast<uint4*>(xs + token * stride + p * part_size + 16 * i) = uint4{h[p][0], h[p][1], h[p][2], h[p][3]};
          if (i % 4 == 0) offset[(token * P + p) * 4 * blocks + i / 4] = sum[p] * (-8.0f * 0x1p-24f);
        }
      }
    }
  }
  __syncthreads();

  float4_t acc[RT];
#pragma unroll
  for (int r = 0; r < RT; ++r) acc[r] = float4_t{0.f, 0.f, 0.f, 0.f};
  // column 4 v + j: group j of row v of xs (token v, or, where a part is a token, v / P of its part v % P)
  constexpr int ROWS = P / M;  // of xs, a token
  const int mine = min(c >> 2, ROWS * nt - 1);
  const bool own = (c & 3) == g;
  const uint8_t* xp = own ? xs + mine * (M * part_size) + 64 * g : reinterpret_cast<const uint8_t*>(zeros);
  const int step = own ? 2 * PB : 0, part_step = own ? part_size : 0;
  const float* op = offset + mine * (M * 4 * blocks) + (c & 3);
  for (int kb0 = wave; kb0 < blocks; kb0 += W * AHEAD) {
#pragma unroll
    for (int e = 0; e < AHEAD; ++e) {
      const int kb = kb0 + W * e;
      if (kb < blocks) {  // (the wave's lanes agree)
        half8_t b[4 * M];
#pragma unroll
        for (int k = 0; k < 4 * M; ++k)
          b[k] = *reinterpret_cast<const half8_t*>(xp + kb * step + (k / 4) * part_step + 16 * (k % 4));
        float start = op[4 * kb];
        if constexpr (M == 2) start += op[4 * (blocks + kb)];
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          const uint32_t words[4] = {w[e][r].x, w[e][r].y, w[e][r].z, w[e][r].w};
          float4_t d = {start, start, start, start};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const half8_t n = tiny4(words[k]);
#pragma unroll
            for (int p = 0; p < M; ++p) d = mfma32(n, b[4 * p + k], d);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const half2_t h = as_h2(i < 2 ? s[e][r].x : s[e][r].y);
            acc[r][i] = __builtin_fmaf((float)(i & 1 ? h.y : h.x), d[i], acc[r][i]);
          }
        }
        if (kb + W * AHEAD < blocks) load(e, kb + W * AHEAD);
      }
    }
  }
  __syncthreads();  // xn is read
  // the four groups' columns into the token's
  float4_t y[RT][1];
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float q = acc[r][i];
      q += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(q), 0xB1, 0xf, 0xf, false));
      q += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(q), 0x4E, 0xf, 0xf, false));
      if constexpr (ROWS == 2) q += shfl_xor(q, 4);  // and the token's two parts
      y[r][0][i] = q;
    }
  finish<DT, RT, 1, RT == 2, W, 4 * ROWS>(a, y, reinterpret_cast<float*>(xs), t0, nt, 16 * (int64_t)blockIdx.x, unit);
}

// ---------------------------------------------------------------- up to 16 tokens of fp16 as they are: one launch
//
// Each wave brings its own blocks of x to LDS, 256 bytes a token, in rows that 16 lanes load together, and takes them from
// there as operands: no workgroup barrier in the loop.

template <int RT, bool GATED, int W>
__global__ __launch_bounds__(64 * W, W == 16 ? 1 : 8 / W) void product4_kernel(ProductArgs a) {
  constexpr int AHEAD = 5, ROW = 2 * PB + 16, SLOT = 16 * ROW, RED = 4 * red_floats(1, GATED, W);
  __shared__ __attribute__((aligned(16))) uint8_t lds[RED > W * SLOT ? RED : W * SLOT];
  const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int nt = (int)a.tokens, blocks = (a.in + PB - 1) / PB;
  const int64_t o0 = 16 * (int64_t)blockIdx.x;

  uint4 xr[4];  // the next block: token 4 e + g, inputs 8 c ..
  const uint8_t* xp = a.x + (int64_t)g * a.in * 2 + 16 * c;
  auto load_x = [&](int kb) {
    const bool in = kb * PB + 8 * c < a.in;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      xr[e] = uint4{0, 0, 0, 0};
      if (in && 4 * e + g < nt) xr[e] = *reinterpret_cast<const uint4*>(xp + ((int64_t)(4 * e) * a.in + (int64_t)kb * PB) * 2);
    }
  };
  load_x(wave);
  Weights<RT, GATED, W, AHEAD> wt(a, o0, lane, blocks);
#pragma unroll
  for (int e = 0; e < AHEAD; ++e)
    if (wave + W * e < blocks) wt.load(e, wave + W * e);

  float4_t acc[RT][1];
#pragma unroll
  for (int r = 0; r < RT; ++r) acc[r][0] = float4_t{0.f, 0.f, 0.f, 0.f};
  uint8_t* slot = lds + wave * SLOT;
  for (int kb0 = wave; kb0 < blocks; kb0 += W * AHEAD) {
#pragma unroll
    for (int e = 0; e < AHEAD; ++e) {
      const int kb = kb0 + W * e;
      if (kb < blocks) {  // (the wave's lanes agree)
#pragma unroll
        for (int i = 0; i < 4; ++i) *reinterpret_cast<uint4*>(slot + (4 * i + g) * ROW + 16 * c) = xr[i];
        if (kb + W < blocks) load_x(kb + W);
        __builtin_amdgcn_wave_barrier();  // (the wave's own LDS operations stay in order)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const half8_t b = *reinterpret_cast<const half8_t*>(slot + c * ROW + 64 * g + 16 * k);
#pragma unroll
          for (int r = 0; r < RT; ++r) acc[r][0] = mfma32(wt.operand(e, r, k), b, acc[r][0]);
        }
        __builtin_amdgcn_wave_barrier();
        if (kb + W * AHEAD < blocks) wt.load(e, kb + W * AHEAD);
      }
    }
  }
  __syncthreads();
  finish<NKV_F16, RT, 1, GATED, W>(a, acc, reinterpret_cast<float*>(lds), 0, nt, o0, nullptr);
}

// ---------------------------------------------------------------- many tokens
//
// xn lies as operands (xn_kernel): a wave's loads of it are 1024 bytes in a row, from the XCD's L2 where the workgroups of
// other rows have it, too. A pass is 16 NT tokens; the passes of the same rows are dealt to one XCD, next to each other, so
// that all but the first find the weights in its L2 (64 tokens over 2560 x 9728 in passes of 16: 25.2 us, so 20.9).

template <int DT, int P, int RT, int NT, bool GATED, int W, int AHEAD>
__global__ __launch_bounds__(64 * W, 8 / W) void product4_many_kernel(ProductArgs a) {
  constexpr int XT = P * NT;
  __shared__ __attribute__((aligned(16))) float red[red_floats(NT, GATED, W)];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t id = blockIdx.y * gridDim.x + blockIdx.x;  // (gridDim.x: a multiple of the XCDs)
  const uint32_t pass = (id / XCDS) % gridDim.y, rows = id / (XCDS * gridDim.y) * XCDS + id % XCDS;
  const int64_t t0 = (int64_t)pass * (16 * NT);
  const int nt = (int)min<int64_t>(16 * NT, a.tokens - t0), blocks = (a.in + PB - 1) / PB;
  const int64_t o0 = (int64_t)rows * (16 * Weights<RT, GATED, W, AHEAD>::TILES);
  if (o0 >= a.out) return;

  half8_t b[4][XT];  // the next block's
  const uint8_t* xp = a.x + (int64_t)pass * XT * blocks * 4096 + 16 * lane;
  auto load_x = [&](int kb, int k) {
#pragma unroll
    for (int n = 0; n < XT; ++n) b[k][n] = *reinterpret_cast<const half8_t*>(xp + ((int64_t)(4 * kb + k) * XT + n) * 1024);
  };
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (wave < blocks) load_x(wave, k);
  Weights<RT, GATED, W, AHEAD> wt(a, o0, lane, blocks);
#pragma unroll
  for (int e = 0; e < AHEAD; ++e)
    if (wave + W * e < blocks) wt.load(e, wave + W * e);

  float4_t acc[RT][NT];
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[r][n] = float4_t{0.f, 0.f, 0.f, 0.f};
  for (int kb0 = wave; kb0 < blocks; kb0 += W * AHEAD) {
#pragma unroll
    for (int e = 0; e < AHEAD; ++e) {
      const int kb = kb0 + W * e;
      if (kb < blocks) {  // (the wave's lanes agree)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
#pragma unroll
          for (int r = 0; r < RT; ++r) {
            const half8_t w = wt.operand(e, r, k);
#pragma unroll
            for (int n = 0; n < XT; ++n) acc[r][n % NT] = mfma32(w, b[k][n], acc[r][n % NT]);
          }
          if (kb + W < blocks) load_x(kb + W, k);
        }
        if (kb + W * AHEAD < blocks) wt.load(e, kb + W * AHEAD);
      }
    }
  }
  finish<DT, RT, NT, GATED, W>(a, acc, red, t0, nt, o0, a.unit + t0);
}

// ---------------------------------------------------------------- host side

// How many waves share a token in product4_few_kernel, whose pass is 4 / each tokens; 0: another form is taken. (Gates and ups
// must be in tiles of their own.)
// Passes, all in one launch, are less than the launch of xn as long as their workgroups do not fill the card
// (us, passes / xn and product: 5 to 16 tokens over 1024 x 2560 7.2 / 7.4 fp16, 6.1 / 6.9 bf16; over 512 x 1024 4.7 / 5.9 and
// 4.2 / 5.5; over 2560 x 2560, 320 workgroups and more, 9.2 / 7.5 and 7.5 / 6.9). One product's worth, 2 tokens in two parts or 4
// in one, always is: 4 bf16 tokens over 6144 x 2560 7.5 / 8.1; with two products (fp16) 9.3 / 8.8. More inputs than a token's
// waves hold take more waves a token, and passes of fewer: of two 7.9 / 8.6 (fp16, 4 tokens over 1000 x 4096; bf16 7.4 / 7.9),
// of one 14.0 / 15.9 and 12.1 / 13.7 (fp16, 512 x 9728 and 1024 x 8192; bf16 13.2 / 13.1, 11.4 / 11.7, and 333 x 9728 14.4 / 13.2:
// not for bf16).
int few_each(int dtype, int64_t tokens, int64_t out, int64_t in, bool norm, bool gated) {
  if ((gated && out % 16) || (!norm && dtype == NKV_F16)) return 0;
  int each = tokens == 1 ? 4 : tokens == 2 ? 2 : 1;
  while (each < 4 && cdiv(in, PB) * PB > each * FEW_KX * 512) each *= 2;
  if (cdiv(in, PB) * PB > each * FEW_KX * 512) return 0;
  const int64_t pass = 4 / each, passes = cdiv(tokens, pass);
  const int parts = parts_of(dtype, true);
  if (parts == 1 && pass == 1 && tokens > 1) return 0;
  return (passes == 1 && tokens * parts <= 4) || passes * cdiv(out, 16) <= CUS ? each : 0;
}

// A cut of product4_many_kernel's work: the token tiles of a pass, and the tiles of 16 outputs of a workgroup.
struct Cut {
  int nt, rt;
};
// A workgroup's time goes with the operands that it makes of the codes and those of xn that it loads (from the L2, which is
// what it waits for), rt + parts nt a step; the launch's with that and the rounds of workgroups. us, xn's launch among it, 17 /
// 32 / 48 / 64 tokens, (nt, rt): 2560 x 9728 (2, 1) 16.3 / 16.8, (3, 1) 20.8, (1, 2) 16.3 / 16.9 / 17.4 / 24, (2, 2) 19.3 / 20.0 /
// 20.0 / 20.6, (4, 1) 23.4, (1, 4) 22.4 / 23.0 / 23.4 / 23.7; 6144 x 2560 fp16 (2, 2) 11.0 / 11.4, (1, 3) 10.4 / 10.7, (3, 2) 13.8,
// (2, 3) 12.4 / 12.7 / 13.1 / 13.9, (4, 2) 15.7; 10240 x 2560 fp16 with rt 2 16.7 / 17.4 / 21.8 / 24.7, with 3 12.9 / 13.7 /
// 16.4 / 18.3; 16384 x 2560 with 2 17.7 / 18.4 / 22.8, with 4 15.2 / 16.3 / 19.8. (32000 x 2560 bf16 with 2 19.4 / 20.2 / 29.2
// / 32.7, with 4 20.8 / 21.3 / 26.2 / 28.4: there the weights' bytes count, too.) Of the same the one with fewer passes.
// Gates and ups: three tiles of each, up to 32 tokens, where that is one round of workgroups (17 tokens, as one / as three:
// 9728 of 2560 fp16 22.0 / 17.5, bf16 14.9 / 14.5; 11008 of 4096 31.6 / 24.5 and 22.3 / 20.6) or where xn is as much as four
// operands (18944 of 2560 fp16 33.9 / 29.7; bf16 22.4 / 25.0). More tokens' sums take the registers: one tile of each.
Cut many_cut(int parts, int64_t tokens, int64_t out, bool gated) {
  const int64_t tiles = cdiv(out, 16), t16 = cdiv(tokens, 16);
  const int most = (int)std::min<int64_t>(t16, 4);
  if (gated) return {most, most <= 2 && tiles > 2 * CUS && (tiles <= 3 * CUS || parts * most == 4) ? 3 : 1};
  Cut best = {0, 0};
  int64_t least = 0;
  for (int nt = most; nt >= 1; --nt)
    for (int rt = 1; rt <= 4; ++rt) {
      if (parts * nt == 8 && rt == 4) continue;  // (no registers for it)
      const int64_t time = cdiv(cdiv(tiles, rt) * cdiv(t16, nt), CUS) * (rt + parts * nt);
      if (best.nt == 0 || time < least) best = {nt, rt}, least = time;
    }
  return best;
}

int64_t product_workspace(int dtype, int64_t tokens, int64_t out, int64_t in, bool norm, bool gated) {
  if (few_each(dtype, tokens, out, in, norm, gated) || (tokens <= 16 && dtype == NKV_F16 && !norm)) return 0;
  const int parts = parts_of(dtype, norm), nt = many_cut(parts, tokens, out, gated).nt;
  return cdiv(tokens, 16 * nt) * nt * cdiv(in, PB) * 4096 * parts + 4 * tokens;
}

template <int DT, bool GATED>
int launch_product(const char* what, ProductArgs a, uint8_t* ws, int64_t ws_bytes, hipStream_t s) {
  constexpr int R1 = GATED ? 2 : 1;
  const int blocks = (int)cdiv(a.in, PB);
  const int64_t tiles = cdiv(a.out, 16);
  const bool norm = a.gamma != nullptr;
  if (const int each = few_each(DT, a.tokens, a.out, a.in, norm, GATED)) {
    const int64_t pass = std::min<int64_t>(a.tokens, FEW_W / each);
    const size_t xn = pass * (parts_of(DT, true) * (2 * blocks * PB + 16 + 16 * blocks));
    const size_t lds = std::max(xn, (size_t)4 * red_floats(1, GATED, FEW_W));
    const dim3 grid((unsigned)tiles, (unsigned)cdiv(a.tokens, FEW_W / each)), block(64 * FEW_W);
    constexpr int P = parts_of(DT, true);
    if (pass <= 2) hipLaunchKernelGGL((product4_few_kernel<DT, R1, 1>), grid, block, lds, s, a, each);
    else hipLaunchKernelGGL((product4_few_kernel<DT, R1, P>), grid, block, lds, s, a, each);
    return check_launch(what);
  }
  if constexpr (DT == NKV_F16) {
    if (a.tokens <= 16 && !norm) {
      if (blocks <= 24) hipLaunchKernelGGL((product4_kernel<R1, GATED, 4>), dim3((unsigned)tiles), dim3(256), 0, s, a);
      else hipLaunchKernelGGL((product4_kernel<R1, GATED, 16>), dim3((unsigned)tiles), dim3(1024), 0, s, a);
      return check_launch(what);
    }
  }
  const int64_t need = product_workspace(DT, a.tokens, a.out, a.in, norm, GATED);
  if (!ws || ws_bytes < need)
    return fail(NKV_ERR_INVALID, "%s: workspace of %lld bytes, %lld needed", what, (long long)ws_bytes, (long long)need);
  const Cut cut = many_cut(parts_of(DT, norm), a.tokens, a.out, GATED);
  const int nt = cut.nt;
  float* unit = reinterpret_cast<float*>(ws + need - 4 * a.tokens);
  const dim3 each_token((unsigned)a.tokens);
  if (parts_of(DT, norm) == 2) hipLaunchKernelGGL((xn_kernel<DT, 2>), each_token, dim3(256), 0, s, a, nt, ws, unit);
  else hipLaunchKernelGGL((xn_kernel<DT, 1>), each_token, dim3(256), 0, s, a, nt, ws, unit);
  if (int rc = check_launch(what)) return rc;
  a.x = ws;
  a.unit = unit;
  const int64_t passes = cdiv(a.tokens, 16 * nt), groups = cdiv(cdiv(tiles, cut.rt), XCDS) * XCDS;
  if (groups * passes >= (int64_t(1) << 31))
    return fail(NKV_ERR_INVALID, "%s: sizes out=%lld tokens=%lld (less than 2^31 workgroups)", what, (long long)a.out, (long long)a.tokens);
  const auto go = [&](auto kernel, int waves) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)groups, (unsigned)passes), dim3(64 * waves), 0, s, a);
  };
  const auto pass = [&](auto n, auto p) {
    constexpr int NT = decltype(n)::value, P = decltype(p)::value;
    if constexpr (GATED && NT > 2) {  // (as 4 waves 19.3 and 21.3 us of 48 and 64 tokens, as 8 21.0 and 24.0)
      go(product4_many_kernel<DT, P, 2, NT, true, 4, 5>, 4);
    } else if constexpr (GATED) {
      if (cut.rt == 3) go(product4_many_kernel<DT, P, 6, NT, true, 8, 2>, 8);
      else go(product4_many_kernel<DT, P, 2, NT, true, 8, 3>, 8);
    } else {
      if (cut.rt == 1) return go(product4_many_kernel<DT, P, 1, NT, false, 8, 5>, 8);
      if (cut.rt == 2) return go(product4_many_kernel<DT, P, 2, NT, false, 8, 3>, 8);
      if (cut.rt == 3) return go(product4_many_kernel<DT, P, 3, NT, false, 8, 2>, 8);
      if constexpr (P * NT < 8) go(product4_many_kernel<DT, P, 4, NT, false, 8, 2>, 8);
    }
  };
  const auto with_tiles = [&](auto p) {
    if (nt == 1) pass(std::integral_constant<int, 1>{}, p);
    else if (nt == 2) pass(std::integral_constant<int, 2>{}, p);
    else if (nt == 3) pass(std::integral_constant<int, 3>{}, p);
    else pass(std::integral_constant<int, 4>{}, p);
  };
  if constexpr (DT == NKV_F16) {
    if (norm) with_tiles(std::integral_constant<int, 2>{});
    else with_tiles(std::integral_constant<int, 1>{});
  } else {
    with_tiles(std::integral_constant<int, 1>{});
  }
  return check_launch(what);
}

int product(const char* what, const void* x, int dtype, int64_t tokens, const void* gamma, float eps, const uint8_t* w4, int64_t out,
            int64_t in, const void* residual, void* y, bool gated, void* workspace, int64_t workspace_bytes, void* stream) {
  set_error("");
  if (dtype != NKV_F16 && dtype != NKV_BF16) return fail(NKV_ERR_INVALID, "%s: dtype %d (fp16 or bf16)", what, dtype);
  if (out <= 0 || out >= (int64_t(1) << 27) || in <= 0 || in % Q4_GROUP || in > P_IN || tokens < 0 || tokens > P_TOKENS)
    return fail(NKV_ERR_INVALID, "%s: sizes out=%lld in=%lld tokens=%lld (out in [1, 2^27), in a positive multiple of 32, at most %d, "
                "tokens at most %lld)", what, (long long)out, (long long)in, (long long)tokens, P_IN, (long long)P_TOKENS);
  if (tokens == 0) return NKV_OK;
  if (!x || !w4 || !y) return fail(NKV_ERR_INVALID, "%s: null pointer argument", what);
  if (!al16(x) || !al16(w4) || !al16(gamma) || !al16(workspace))
    return fail(NKV_ERR_UNSUPPORTED, "%s: x, gamma, the weight and the workspace must be 16-byte aligned", what);
  ProductArgs a{static_cast<const uint8_t*>(x), static_cast<const uint8_t*>(gamma), eps, w4, out, (int)in,
                static_cast<const uint8_t*>(residual), static_cast<uint8_t*>(y), tokens, nullptr};
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == NKV_F16) {
    return gated ? launch_product<NKV_F16, true>(what, a, ws, workspace_bytes, s)
                 : launch_product<NKV_F16, false>(what, a, ws, workspace_bytes, s);
  }
  return gated ? launch_product<NKV_BF16, true>(what, a, ws, workspace_bytes, s)
               : launch_product<NKV_BF16, false>(what, a, ws, workspace_bytes, s);
}

}  // namespace

}  // namespace nkv

using namespace nkv;

extern "C" int64_t nkv_gemv_q4_workspace_bytes(int dtype, int64_t tokens, int64_t out_features, int64_t in_features, int norm,
                                                int swiglu) {
  return tokens > 0 && out_features > 0 && in_features > 0
             ? product_workspace(dtype, tokens, out_features, in_features, norm != 0, swiglu != 0) : 0;
}

extern "C" int nkv_gemv_q4(const void* x, int dtype, int64_t tokens, const void* gamma, float eps, const uint8_t* w4,
                           int64_t out_features, int64_t in_features, const void* residual, void* y,
                           void* workspace, int64_t workspace_bytes, void* stream) {
  return product("gemv_q4", x, dtype, tokens, gamma, eps, w4, out_features, in_features, residual, y, false,
                 workspace, workspace_bytes, stream);
}

extern "C" int nkv_swiglu_gemv_q4(const void* x, int dtype, int64_t tokens, const void* gamma, float eps, const uint8_t* w4,
                                  int64_t intermediate, int64_t in_features, void* act, void* workspace,
                                  int64_t workspace_bytes, void* stream) {
  return product("swiglu_gemv_q4", x, dtype, tokens, gamma, eps, w4, intermediate, in_features, nullptr, act, true,
                 workspace, workspace_bytes, stream);
}
