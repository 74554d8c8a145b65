// The decode step's projections with 4-bit weights (nkv_q4.h) for one token or a few: y = W xn (+ residual), and the
// first half of a SwiGLU block, xn = x or its RMSNorm.
//
// On the matrix cores: 16 rows of W times up to 16 tokens. The weights become exact fp16 operands; lane c + 16 g takes
// row c's group g of every 128 inputs, 16 bytes, one scale. xn is rounded once to fp16, scaled by a power of two of the
// token's own, so that bf16's range and large gammas stay within fp16's. The waves of a workgroup cut the inputs among them;
// everything else in fp32, with one rounding at the end. Bound by the weights' bytes.

#include <algorithm>
#include <type_traits>

#include "nkv_paged.h"
#include "nkv_q4.h"

namespace nkv {

namespace {

constexpr int PW = 4;             // waves of a workgroup
constexpr int PB = 128;           // inputs of a block: four products deep
constexpr int PT = 16;            // tokens of a workgroup, at most
constexpr int PX = 48 * 1024;     // bytes of LDS for xn
constexpr int P_IN = 1 << 20;     // inputs, at most

struct ProductArgs {
  const uint8_t* x;        // [tokens][in]
  const uint8_t* gamma;    // [in] or NULL
  float eps;
  const uint8_t* codes;    // [rows][in / 2]
  const uint16_t* scales;  // [rows][in / 32]
  int64_t out;             // outputs a token (SwiGLU: half the rows)
  int in;
  const uint8_t* residual;  // [tokens][out] or NULL
  uint8_t* y;
  int64_t tokens;
  int chunk;               // inputs whose xn is in LDS at a time, a multiple of PW * PB
};

// A few values of element type DT.
template <int DT>
__device__ __forceinline__ float load1(const uint8_t* p, int64_t i) {
  const uint16_t b = reinterpret_cast<const uint16_t*>(p)[i];
  return DT == NKV_F16 ? h2f(b) : bf2f(b);
}

// RT: tiles of 16 rows a workgroup takes; GATED: the second is the up rows of the first's gates.
template <int DT, int RT, bool GATED>
__global__ __launch_bounds__(64 * PW, 4) void product4_kernel(ProductArgs a) {
  extern __shared__ __attribute__((aligned(16))) uint8_t xs[];  // [tokens][chunk + 8] fp16; the sums at the end
  __shared__ float unit[PT], inverse[PT];  // of a token: xn = x * norm * gamma, held times inverse, unit = 1 / inverse
  __shared__ float norm[PT];
  const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t t0 = (int64_t)blockIdx.y * PT;
  const int nt = (int)min<int64_t>(PT, a.tokens - t0);
  const int64_t o0 = (int64_t)blockIdx.x * (GATED ? 16 : 16 * RT);
  const int blocks = (a.in + PB - 1) / PB, groups = a.in / Q4_GROUP;

  // this lane's rows (rows behind the last: the last, not stored)
  const uint8_t* wp[RT];
  const uint16_t* sp[RT];
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    const int64_t row = GATED ? r * a.out + min(o0 + c, a.out - 1) : min(o0 + 16 * r + c, a.out - 1);
    wp[r] = a.codes + row * (a.in / 2) + 16 * g;
    sp[r] = a.scales + row * groups + g;
  }
  constexpr int AHEAD = 4;
  uint4 w[AHEAD][RT];
  uint16_t s[AHEAD][RT];
  auto load = [&](int e, int kb) {
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      const bool ok = 4 * kb + g < groups;
      const u32x4_t* p = reinterpret_cast<const u32x4_t*>(wp[r] + (int64_t)kb * (PB / 2));
      u32x4_t v = {0, 0, 0, 0};
      if (ok) v = __builtin_nontemporal_load(p);
      w[e][r] = uint4{v.x, v.y, v.z, v.w};
      s[e][r] = ok ? sp[r][4 * kb] : 0;
    }
  };
#pragma unroll
  for (int e = 0; e < AHEAD; ++e) load(e, wave + PW * e);

  // the tokens' norms and units
  if (a.gamma || DT != NKV_F16) {
    for (int t = wave; t < nt; t += PW) {
      const uint8_t* x = a.x + (t0 + t) * a.in * 2;
      float ss = 0.0f, top = 0.0f;
      for (int i = 8 * lane; i < a.in; i += 512) {
        Raw8<DT> r, gr;
        r.load(x + 2 * i);
        float v[8], gv[8];
        r.get(v);
        if (a.gamma) {
          gr.load(a.gamma + 2 * i);
          gr.get(gv);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          ss = __builtin_fmaf(v[e], v[e], ss);
          top = fmaxf(top, __builtin_fabsf(a.gamma ? v[e] * gv[e] : v[e]));
        }
      }
      ss = hsum64(ss);
#pragma unroll
      for (int o = 32; o >= 1; o >>= 1) top = fmaxf(top, shfl_xor(top, o));
      const float r = a.gamma ? rsqrtf(ss / (float)a.in + a.eps) : 1.0f;
      top *= r;
      // the power of two that brings the largest to 2^14
      const int ex = top > 0.0f && top < 3e38f ? max((int)(__float_as_uint(top) >> 23) - 127 - 14, -100) : 0;
      if (lane == 0) {
        norm[t] = r;
        inverse[t] = __uint_as_float((uint32_t)(127 - ex) << 23);
        unit[t] = __uint_as_float((uint32_t)(127 + ex) << 23);
      }
    }
  } else if (tid < PT) {
    norm[tid] = inverse[tid] = unit[tid] = 1.0f;
  }

  const int stride = 2 * a.chunk + 16;  // bytes of a token's row: 16 tokens' chunks fall on different banks
  float4_t acc[RT];
#pragma unroll
  for (int r = 0; r < RT; ++r) acc[r] = float4_t{0.f, 0.f, 0.f, 0.f};
  const uint8_t* xp = xs + min(c, nt - 1) * stride + 64 * g;
  int kb = wave;
  for (int k0 = 0; k0 < a.in; k0 += a.chunk) {
    __syncthreads();  // norms are there; the chunk before is read
    const int n8 = min(a.chunk, (blocks * PB) - k0) / 8;
    for (int i = tid; i < nt * n8; i += 64 * PW) {
      const int t = i / n8, k = 8 * (i - t * n8), at = k0 + k;
      Raw8<DT> r, gr;
      r.zero();
      float v[8], gv[8];
      if (at < a.in) r.load(a.x + ((t0 + t) * a.in + at) * 2);
      uint4 u;
      if (!a.gamma && DT == NKV_F16) {
        u = r.w[0];
      } else {
        r.get(v);
        const float f = inverse[t];
        if (a.gamma) {
          gr.zero();
          if (at < a.in) gr.load(a.gamma + 2 * at);
          gr.get(gv);
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = v[e] * norm[t] * gv[e];
        }
        uint32_t h[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) h[e] = (uint32_t)f2h(v[2 * e] * f) | ((uint32_t)f2h(v[2 * e + 1] * f) << 16);
        u = uint4{h[0], h[1], h[2], h[3]};
      }
      *reinterpret_cast<half8_t*>(xs + t * stride + 2 * k) = paired(u);
    }
    __syncthreads();
    const int end = min(blocks, (k0 + a.chunk) / PB), base = k0 / PB;
    while (kb < end) {
#pragma unroll
      for (int e = 0; e < AHEAD; ++e) {
        if (kb < end) {  // (the waves differ, their lanes agree)
          const uint8_t* p = xp + (kb - base) * (2 * PB);
          half8_t b[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) b[k] = *reinterpret_cast<const half8_t*>(p + 16 * k);
#pragma unroll
          for (int r = 0; r < RT; ++r) {
            const half2_t sc = as_h2((uint32_t)s[0][r] * 0x10001u);
            acc[r] = mfma32(unpack4(w[0][r].x, sc), b[0], acc[r]);
            acc[r] = mfma32(unpack4(w[0][r].y, sc), b[1], acc[r]);
            acc[r] = mfma32(unpack4(w[0][r].z, sc), b[2], acc[r]);
            acc[r] = mfma32(unpack4(w[0][r].w, sc), b[3], acc[r]);
          }
          // the registers move up: chunks may end anywhere
#pragma unroll
          for (int f = 0; f + 1 < AHEAD; ++f)
#pragma unroll
            for (int r = 0; r < RT; ++r) w[f][r] = w[f + 1][r], s[f][r] = s[f + 1][r];
          load(AHEAD - 1, kb + PW * AHEAD);
          kb += PW;
        }
      }
    }
  }

  // ---- the waves' sums into one
  __syncthreads();
  float* red = reinterpret_cast<float*>(xs);  // [wave][tile][row 16][token 16 + 1]
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int i = 0; i < 4; ++i) red[((wave * RT + r) * 16 + 4 * g + i) * 17 + c] = acc[r][i];
  __syncthreads();
  const int t = tid >> 4, row = tid & 15;
  if (t >= nt) return;
  float v[RT];
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    v[r] = 0.0f;
#pragma unroll
    for (int q = 0; q < PW; ++q) v[r] += red[((q * RT + r) * 16 + row) * 17 + t];
    v[r] *= unit[t];
  }
  auto store = [&](int64_t o, float f) {
    const int64_t at = (t0 + t) * a.out + o;
    if (a.residual) f += load1<DT>(a.residual, at);
    reinterpret_cast<uint16_t*>(a.y)[at] = DT == NKV_F16 ? f2h(f) : f2bf(f);
  };
  if constexpr (GATED) {
    if (o0 + row < a.out) store(o0 + row, v[0] / (1.0f + expf(-v[0])) * v[1]);
  } else {
#pragma unroll
    for (int r = 0; r < RT; ++r)
      if (o0 + 16 * r + row < a.out) store(o0 + 16 * r + row, v[r]);
  }
}

template <int DT>
void launch_product(const ProductArgs& a, bool gated, hipStream_t s) {
  const int nt = (int)std::min<int64_t>(a.tokens, PT);
  ProductArgs b = a;
  const int whole = (int)cdiv(a.in, PW * PB) * (PW * PB);
  b.chunk = std::min(whole, std::max(PW * PB, PX / (2 * nt) / (PW * PB) * (PW * PB)));
  const int rt = gated ? 2 : 1;
  const size_t lds = std::max((size_t)nt * (2 * b.chunk + 16), (size_t)PW * rt * 16 * 17 * 4);
  const dim3 grid((unsigned)cdiv(a.out, 16), (unsigned)cdiv(a.tokens, PT));
  if (gated) hipLaunchKernelGGL((product4_kernel<DT, 2, true>), grid, dim3(64 * PW), lds, s, b);
  else hipLaunchKernelGGL((product4_kernel<DT, 1, false>), grid, dim3(64 * PW), lds, s, b);
}

int product(const char* what, const void* x, int dtype, int64_t tokens, const void* gamma, float eps, const uint8_t* codes,
            const uint16_t* scales, int64_t out, int64_t in, const void* residual, void* y, bool gated, void* stream) {
  set_error("");
  if (dtype != NKV_F16 && dtype != NKV_BF16) return fail(NKV_ERR_INVALID, "%s: dtype %d (fp16 or bf16)", what, dtype);
  if (out <= 0 || out >= (int64_t(1) << 27) || in <= 0 || in % Q4_GROUP || in > P_IN || tokens < 0 || tokens > 65535 * PT)
    return fail(NKV_ERR_INVALID, "%s: sizes out=%lld in=%lld tokens=%lld (out in [1, 2^27), in a positive multiple of 32, at most %d, "
                "tokens at most %d)", what, (long long)out, (long long)in, (long long)tokens, P_IN, 65535 * PT);
  if (tokens == 0) return NKV_OK;
  if (!x || !codes || !scales || !y) return fail(NKV_ERR_INVALID, "%s: null pointer argument", what);
  if (!al16(x) || !al16(codes) || !al16(gamma)) return fail(NKV_ERR_UNSUPPORTED, "%s: x, gamma and the codes must be 16-byte aligned", what);
  ProductArgs a{static_cast<const uint8_t*>(x), static_cast<const uint8_t*>(gamma), eps, codes, scales, out, (int)in,
                static_cast<const uint8_t*>(residual), static_cast<uint8_t*>(y), tokens, 0};
  if (dtype == NKV_F16) launch_product<NKV_F16>(a, gated, static_cast<hipStream_t>(stream));
  else launch_product<NKV_BF16>(a, gated, static_cast<hipStream_t>(stream));
  return check_launch(what);
}

}  // namespace

}  // namespace nkv

using namespace nkv;

extern "C" int nkv_gemv_q4(const void* x, int dtype, int64_t tokens, const void* gamma, float eps, const uint8_t* codes,
                           const uint16_t* scales, int64_t out_features, int64_t in_features, const void* residual, void* y,
                           void* stream) {
  return product("gemv_q4", x, dtype, tokens, gamma, eps, codes, scales, out_features, in_features, residual, y, false, stream);
}

extern "C" int nkv_swiglu_gemv_q4(const void* x, int dtype, int64_t tokens, const void* gamma, float eps, const uint8_t* codes,
                                  const uint16_t* scales, int64_t intermediate, int64_t in_features, void* act, void* stream) {
  return product("swiglu_gemv_q4", x, dtype, tokens, gamma, eps, codes, scales, intermediate, in_features, nullptr, act, true,
                 stream);
}
