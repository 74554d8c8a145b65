// The new tokens of a paged batch: a step in which every sequence brings any number of tokens (a prompt's
// chunk, drafted tokens, one decode token, none), packed one after another.
//
// - append_chunks: the head norms and the rotary embedding of the stacked q/k/v projections, and the
//   quantized store of the keys and values into their pages (per-token symmetric format);
// - attn_chunks: the new tokens' causal attention over everything their sequence has in its pages;
// - read: spans of cached tokens back to fp16 / bf16 / fp32, from either page format.
//
// Token t of the packed batch belongs to sequence seq_of[t] and is its new token t - cu[seq]; its position is
// start[seq] + that. Lengths and positions are read on the device, so a captured graph follows them.

#include <type_traits>

#include "nkv_mfma.h"

namespace nkv {

namespace {

// ---------------------------------------------------------------- the packed batch

struct Batch {
  const int32_t* seq_of;   // [tokens]
  const int32_t* cu;       // [nseq + 1]
  const int64_t* start;    // [nseq]
  const int32_t* table;    // [nseq][table_stride]
  int64_t table_stride, num_pages;
  int nseq, hkv;
};

// The page of group `grp` of sequence b, -1 where the table holds none.
__device__ __forceinline__ int64_t page_at(const Batch& a, int b, int64_t grp) {
  if (grp < 0 || grp >= a.table_stride) return -1;
  const int32_t page = a.table[(int64_t)b * a.table_stride + grp];
  return page >= 0 && page < a.num_pages ? page : -1;
}

struct TokenAt {
  int64_t pos, page;  // position in its sequence; page -1: none
  int seq;
};

__device__ __forceinline__ TokenAt token_at(const Batch& a, int64_t t) {
  const int b = a.seq_of[t];
  if (b < 0 || b >= a.nseq) return {-1, -1, -1};
  const int64_t pos = a.start[b] + (t - a.cu[b]);
  return {pos, page_at(a, b, pos < 0 ? -1 : pos / GT), b};
}

// ---------------------------------------------------------------- eight values of a row

template <int DT>
struct Elem;
template <>
struct Elem<NKV_F16> {
  static constexpr int SIZE = 2;
};
template <>
struct Elem<NKV_BF16> {
  static constexpr int SIZE = 2;
};
template <>
struct Elem<NKV_F32> {
  static constexpr int SIZE = 4;
};

template <int DT>
struct Raw8 {  // eight consecutive values as loaded
  uint4 w[Elem<DT>::SIZE / 2];
  __device__ __forceinline__ void load(const uint8_t* p) {
#pragma unroll
    for (int i = 0; i < Elem<DT>::SIZE / 2; ++i) w[i] = *reinterpret_cast<const uint4*>(p + 16 * i);
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < Elem<DT>::SIZE / 2; ++i) w[i] = uint4{0, 0, 0, 0};
  }
  __device__ __forceinline__ void get(float (&v)[8]) const {
    const uint32_t u[4] = {w[0].x, w[0].y, w[0].z, w[0].w};
    if constexpr (DT == NKV_F32) {
      const uint32_t u2[4] = {w[1].x, w[1].y, w[1].z, w[1].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(u[i]), v[4 + i] = __uint_as_float(u2[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (DT == NKV_F16) {
          v[2 * i] = h2f((uint16_t)(u[i] & 0xffffu));
          v[2 * i + 1] = h2f((uint16_t)(u[i] >> 16));
        } else {
          v[2 * i] = bf2f((uint16_t)(u[i] & 0xffffu));
          v[2 * i + 1] = bf2f((uint16_t)(u[i] >> 16));
        }
      }
    }
  }
};

template <bool NT>
__device__ __forceinline__ void store16(uint8_t* p, u32x4_t w) {
  if constexpr (NT) __builtin_nontemporal_store(w, reinterpret_cast<u32x4_t*>(p));
  else *reinterpret_cast<u32x4_t*>(p) = w;
}
template <int DT, bool NT>
__device__ __forceinline__ void store8(uint8_t* p, const float (&v)[8]) {
  if constexpr (DT == NKV_F32) {
#pragma unroll
    for (int i = 0; i < 8; i += 4)
      store16<NT>(p + 4 * i, u32x4_t{__float_as_uint(v[i]), __float_as_uint(v[i + 1]), __float_as_uint(v[i + 2]), __float_as_uint(v[i + 3])});
  } else {
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t lo = DT == NKV_F16 ? f2h(v[2 * i]) : f2bf(v[2 * i]);
      const uint32_t hi = DT == NKV_F16 ? f2h(v[2 * i + 1]) : f2bf(v[2 * i + 1]);
      u[i] = lo | (hi << 16);
    }
    store16<NT>(p, u32x4_t{u[0], u[1], u[2], u[3]});
  }
}

// ---------------------------------------------------------------- append

// Sum over the 16 lanes of each 16-lane row (DPP only; every lane gets it).
__device__ __forceinline__ float row16_sum(float v) {
  v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0xB1, 0xf, 0xf, false));
  v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x4E, 0xf, 0xf, false));
  v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x124, 0xf, 0xf, false));
  v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x128, 0xf, 0xf, false));
  return v;
}

__device__ __forceinline__ float row16_max(float v) {
  v = fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0xB1, 0xf, 0xf, false)));
  v = fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x4E, 0xf, 0xf, false)));
  v = fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x124, 0xf, 0xf, false)));
  v = fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x128, 0xf, 0xf, false)));
  return v;
}

// The value of lane l ^ 8 of the same 16-lane row (a rotation by 8).
__device__ __forceinline__ float row16_other_half(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x128, 0xf, 0xf, false));
}

struct AppendArgs {
  Batch b;
  const uint8_t* x;  // [tokens][hq + 2 hkv][128], row stride x_rs elements
  int64_t x_rs, tokens;
  uint8_t* pages;
  const uint8_t* q_gamma;  // [128] of x's type; NULL: no head norms
  const uint8_t* k_gamma;
  float eps;
  const float* inv_freq;   // [64]; NULL: no rotation
  uint16_t* q_out;         // token t, head i at q_out + t * q_rs + i * 128
  int64_t q_rs;
  int hq, heads_per_wg;
};

// A workgroup takes one token and heads_per_wg of its hq + 2 hkv heads: a head row of 128 values to 16 lanes, 8
// values each, 16 rows at a time. Everything in fp32, rounded once (q to fp16, k and v to codes). The angle position *
// inv_freq is exact in fp64 and reduced there to a part of a turn, so that far positions lose nothing; one lane
// computes it for each frequency, for all heads. The rows ahead are loaded while one is worked on, the first ones
// before the angles and the page are known.
// Bound by memory: 4112 tokens of 32 q and 8 KV heads (93 MB) in 20.6 us, 4.5 TB/s (a large copy reaches 4.9); four
// tokens a workgroup without the loads ahead took 25.8 us. 1029 bf16 tokens of 28 q and 4 KV heads 7.3
// us (21 MB, 2.9 TB/s: a workgroup's chain takes about as long as its data); 12 tokens 3.7 us, the time of the chain
// sequence, position and table, angles, rows. NT: nontemporal q stores.
template <int DT, bool NT>
__global__ __launch_bounds__(256) void append_chunks_kernel(AppendArgs a) {
  __shared__ __attribute__((aligned(16))) float turn[2][D / 2];  // cos, sin
  __shared__ int64_t row_of;  // byte offset of KV head 0's page, or -1
  __shared__ int slot_of;
  const int tid = threadIdx.x, j = tid & 15, first = tid >> 4;
  const int64_t t = blockIdx.x;
  const int heads = a.hq + 2 * a.b.hkv, h0 = blockIdx.y * a.heads_per_wg, h1 = min(h0 + a.heads_per_wg, heads);
  const bool norm = a.q_gamma != nullptr, rotate = a.inv_freq != nullptr;
  constexpr int SIZE = Elem<DT>::SIZE, AHEAD = DT == NKV_F32 ? 2 : 4;

  const uint8_t* x = a.x + (t * a.x_rs + 8 * j) * SIZE;
  Raw8<DT> ahead[AHEAD];
#pragma unroll
  for (int e = 0; e < AHEAD; ++e)
    if (h0 + first + 16 * e < h1) ahead[e].load(x + (int64_t)(h0 + first + 16 * e) * (D * SIZE));
  float gq[8], gk[8];
  if (norm) {
    Raw8<DT> r;
    r.load(a.q_gamma + 8 * j * SIZE);
    r.get(gq);
    r.load(a.k_gamma + 8 * j * SIZE);
    r.get(gk);
  }
  if (tid < D / 2) {
    const TokenAt at = token_at(a.b, t);
    if (tid == 0) {
      row_of = at.page < 0 ? -1 : at.page * a.b.hkv * (int64_t)PAGE_TOK_BYTES;
      slot_of = (int)(at.pos & (GT - 1));
    }
    if (rotate) {
      const double turns = (double)at.pos * (double)a.inv_freq[tid] * 0.15915494309189533577;  // 1 / 2 pi
      const float part = (float)(turns - __builtin_rint(turns));
      turn[0][tid] = cospif(2.0f * part);
      turn[1][tid] = sinpif(2.0f * part);
    }
  }
  __syncthreads();
  // the lane's angles: elements i and i + 64 share one
  float cs[8], sn[8];
  if (rotate) {
#pragma unroll
    for (int e = 0; e < 8; e += 4) {
      const float4 c4 = *reinterpret_cast<const float4*>(&turn[0][(8 * j + e) & (D / 2 - 1)]);
      const float4 s4 = *reinterpret_cast<const float4*>(&turn[1][(8 * j + e) & (D / 2 - 1)]);
      cs[e] = c4.x, cs[e + 1] = c4.y, cs[e + 2] = c4.z, cs[e + 3] = c4.w;
      // element i < 64 becomes x_i cos - x_(i + 64) sin, element i + 64 x_(i + 64) cos + x_i sin
      const float side = j < 8 ? -1.0f : 1.0f;
      sn[e] = side * s4.x, sn[e + 1] = side * s4.y, sn[e + 2] = side * s4.z, sn[e + 3] = side * s4.w;
    }
  }

  for (int h = h0 + first; h < h1; h += 16) {  // (16 lanes agree)
    float v[8];
    ahead[0].get(v);
#pragma unroll
    for (int e = 0; e + 1 < AHEAD; ++e) ahead[e] = ahead[e + 1];
    if (h + 16 * AHEAD < h1) ahead[AHEAD - 1].load(x + (int64_t)(h + 16 * AHEAD) * (D * SIZE));
    const bool is_q = h < a.hq, is_v = h >= a.hq + a.b.hkv;
    if (!is_v) {
      if (norm) {
        float ss = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = __builtin_fmaf(v[e], v[e], ss);
        const float r = rsqrtf(row16_sum(ss) * (1.0f / D) + a.eps);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = v[e] * r * (is_q ? gq[e] : gk[e]);
      }
      if (rotate) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = __builtin_fmaf(v[e], cs[e], row16_other_half(v[e]) * sn[e]);
      }
    }
    if (is_q) {
      store8<NKV_F16, NT>(reinterpret_cast<uint8_t*>(a.q_out + t * a.q_rs + (int64_t)h * D + 8 * j), v);
    } else if (row_of >= 0) {
      const int kv = is_v ? h - a.hq - a.b.hkv : h - a.hq, which = is_v ? 1 : 0;
      float scale;
      const uint2 codes = sym_quant8<true>(v, scale);
      uint8_t* page = a.pages + row_of + (int64_t)kv * PAGE_TOK_BYTES;
      *reinterpret_cast<uint2*>(page + which * CODE_BYTES + slot_of * D + 8 * j) = codes;
      if (j == 0) *reinterpret_cast<uint16_t*>(page + 2 * CODE_BYTES + which * (2 * GT) + 2 * slot_of) = f2h(scale);
    }
  }
}

// ---------------------------------------------------------------- read

struct ReadArgs {
  Batch b;
  int64_t tokens;
  const uint8_t* pages;
  const uint16_t* rings;   // int8t64: [nseq][hkv][2][64][128]
  const int64_t* length;   // int8t64: [nseq] tokens written
  uint8_t* k_out;          // [tokens][hkv][128]
  uint8_t* v_out;
};

// TOK tokens of one workgroup; 16 lanes to a row of 128, 8 values each, four rows of every lane in flight (two of
// int8t64, whose steps and minima are 32 bytes a lane more). Bound by memory: 70000 tokens of 8 KV heads to bf16 (431 MB)
// in 92 us, 4.7 TB/s; 275 tokens 3.0 us, a chain of three loads.
template <int DT, bool T64, int TOK>
__global__ __launch_bounds__(256) void read_kernel(ReadArgs a) {
  __shared__ int64_t page_of[TOK];  // the token's page; -1: none, -2: in its sequence's ring
  __shared__ int slot_of[TOK], seq_of[TOK];
  const int tid = threadIdx.x, j = tid & 15;
  const int64_t t0 = (int64_t)blockIdx.x * TOK;
  const int nt = (int)min<int64_t>(TOK, a.tokens - t0);
  if (tid < nt) {
    const TokenAt at = token_at(a.b, t0 + tid);
    int64_t page = at.page;
    if (T64 && at.seq >= 0) {
      const int64_t len = a.length[at.seq];
      if (at.pos >= len) page = -1;
      else if (at.pos >= len / GT * GT) page = -2;
    }
    page_of[tid] = page;
    slot_of[tid] = (int)(at.pos & (GT - 1));
    seq_of[tid] = at.seq;
  }
  __syncthreads();
  constexpr int SIZE = Elem<DT>::SIZE, FLY = T64 ? 2 : 4;
  const int rows = 2 * a.b.hkv * nt;
  // item `it`: token it % nt, tensor and KV head it / nt (neighbouring rows of a page, first)
  for (int it0 = tid >> 4; it0 < rows; it0 += 16 * FLY) {
    uint2 codes[FLY];
    uint16_t scale[FLY];
    Raw8<NKV_F16> st[FLY], mn[FLY];  // (st: the ring's values, too)
#pragma unroll
    for (int f = 0; f < FLY; ++f) {
      const int it = it0 + 16 * f;
      if (it >= rows) break;
      const int k = it % nt, hw = it / nt, h = hw >> 1, which = hw & 1, slot = slot_of[k];
      const int64_t page = page_of[k];
      if (T64 && page == -2) {
        st[f].load(reinterpret_cast<const uint8_t*>(a.rings + ((((int64_t)seq_of[k] * a.b.hkv + h) * 2 + which) * GT + slot) * D + 8 * j));
      } else if (page >= 0) {
        const uint8_t* p = a.pages + (page * a.b.hkv + h) * (T64 ? PAGE_BYTES : PAGE_TOK_BYTES);
        codes[f] = *reinterpret_cast<const uint2*>(p + which * CODE_BYTES + slot * D + 8 * j);
        if constexpr (T64) {
          st[f].load(p + 2 * CODE_BYTES + which * (4 * D) + 16 * j);
          mn[f].load(p + 2 * CODE_BYTES + which * (4 * D) + 2 * D + 16 * j);
        } else {
          scale[f] = *reinterpret_cast<const uint16_t*>(p + 2 * CODE_BYTES + which * (2 * GT) + 2 * slot);
        }
      }
    }
#pragma unroll
    for (int f = 0; f < FLY; ++f) {
      const int it = it0 + 16 * f;
      if (it >= rows) break;
      const int k = it % nt, hw = it / nt, h = hw >> 1, which = hw & 1;
      const int64_t page = page_of[k];
      float v[8];
      if (page == -1) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = 0.0f;
      } else if (T64 && page == -2) {
        st[f].get(v);
      } else if constexpr (T64) {
        float s8[8], m8[8];
        st[f].get(s8);
        mn[f].get(m8);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint32_t code = ((e < 4 ? codes[f].x : codes[f].y) >> (8 * (e & 3))) & 0xffu;
          v[e] = __builtin_fmaf((float)code, s8[e], m8[e]);  // (the product is exact)
        }
      } else {
        const float s = h2f(scale[f]);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = (float)(int8_t)((e < 4 ? codes[f].x : codes[f].y) >> (8 * (e & 3))) * s;
      }
      store8<DT, (TOK > 4)>((which ? a.v_out : a.k_out) + (((t0 + k) * a.b.hkv + h) * D + 8 * j) * SIZE, v);
    }
  }
}

// ---------------------------------------------------------------- attention
//
// The rows of KV head h in sequence b: row R = (new token R / gq, q head h gq + R % gq), gq = hq / hkv. They
// are cut into tiles; a tile attends the 64-token groups up to its last token (steps 0 .. S - 1), and its
// steps are cut into parts, unit = one part of one tile. Part p of P takes steps [S p / P, S (p + 1) / P),
// from the S of the device's lengths: the plan stays valid while sequences grow.
//
// softmax(q K^T / sqrt(128)) V with K = code * scale and V likewise: K's scale multiplies the scores and V's the
// weights, so that the codes are exact operands, and only P (weight times V's scale) and the output are rounded to fp16.
//
// Units of up to 32 rows (small): the waves of a workgroup take the part's groups in turn, each wave its own
// group against all the rows, and their states are merged in LDS at the end. K codes go from memory to the
// registers of S^T = K Q^T's A operand; V codes and both scales go to LDS, where the transposing read gives
// the operand of O = P V. Bound by memory: one token of each of 32 sequences of 64 to 8155 tokens (274 MB) in 50 us
// and 4 for the merge, 5.5 TB/s; 64 sequences of 2048 in 45 us, 6.1 TB/s.

constexpr int CH_WAVES = 8, CH_THREADS = 64 * CH_WAVES;
constexpr int CH_VSLOT = CODE_BYTES + 4 * GT;            // V codes, K scales, V scales: the rest of a page after K
constexpr int CH_PART = D + 4;                           // floats of a row's partial: acc[128], m, l, pad
static_assert(CODE_BYTES + CH_VSLOT == PAGE_TOK_BYTES, "a page is K codes and a slot");
static_assert(16 * CH_PART * 4 <= CH_VSLOT, "a wave's 16 rows fit one of its slots at the merge");
constexpr int CH_LDS = 2 * CH_WAVES * CH_VSLOT;          // 132 KiB: two slots a wave

enum UnitKind : int { ROWS16 = 0, ROWS32 = 1, ROWS256 = 2 };

struct Unit {  // (int32 each, as the plan lays them out)
  int seq, row0, rows, part, parts, slot, kind, alone;  // slot: partial row of part 0 of the tile; alone: of its sequence
};
struct Merge {
  int first, row0, rows, parts, slot, stride, pad0, pad1;  // first: the sequence's first packed token; up to 8 rows;
                                                           // part p's partial of row r: slot + p * stride + r
};

struct ChunkArgs {
  Batch b;
  const uint16_t* q;  // token t, head i at q + t * q_ts + i * q_hs
  int64_t q_ts, q_hs, tokens;
  const uint8_t* pages;
  const Unit* units;
  int hq, gq;
  float sl2;
  uint16_t* out;
  int64_t o_ts, o_hs;
  float* lse;  // [tokens][hq] or NULL
  float* ws;   // partial rows [ws_rows][hkv][CH_PART]
  int64_t ws_rows;
};

// Where a tile of sequence b stands.
struct TileAt {
  int64_t start, first_token;  // position of the sequence's first new token; packed index of it
  int rows;                    // rows of the tile (no more than the sequence has)
  int64_t steps;               // groups up to the tile's last token
};
__device__ __forceinline__ TileAt tile_at(const ChunkArgs& a, int seq, int row0, int rows) {
  TileAt t;
  const int64_t c0 = a.b.cu[seq], c1 = a.b.cu[seq + 1];
  const int64_t have = max<int64_t>(0, min(c1, a.tokens) - c0) * a.gq - row0;
  t.rows = c0 < 0 ? 0 : (int)max<int64_t>(0, min<int64_t>(rows, have));
  t.start = a.b.start[seq];
  t.first_token = c0;
  t.steps = t.rows == 0 || t.start < 0 ? 0 : min((t.start + (row0 + t.rows - 1) / a.gq) / GT + 1, a.b.table_stride);
  return t;
}

constexpr float W_TAU = 4.0f;  // (RowState; log2 of the weights that a lane sums at a time)

// A row's sums, 32 lanes a row, 4 dims each: l of the weights 2^(score - m), scores in the log2 domain, acc of weight
// times V.
struct RowSum {
  float m, l;
  float4 acc;
};
__device__ __forceinline__ void write_row(const ChunkArgs& a, int h, int64_t token, int head, const RowSum& r, int l32) {
  const float inv = r.l > 0.0f || r.l != r.l ? 1.0f / r.l : 0.0f;
  const int i = h * a.gq + head;
  *reinterpret_cast<uint2*>(a.out + token * a.o_ts + i * a.o_hs + 4 * l32) =
      uint2{(uint32_t)f2h(r.acc.x * inv) | ((uint32_t)f2h(r.acc.y * inv) << 16),
            (uint32_t)f2h(r.acc.z * inv) | ((uint32_t)f2h(r.acc.w * inv) << 16)};
  if (a.lse && l32 == 0) a.lse[token * a.hq + i] = r.l == 0.0f ? NEG_INF : (r.m + __builtin_amdgcn_logf(r.l)) * LN2;
}

// The pages of a wave's groups first, first + stride, .., n of them, held 64 at a time, one a lane. (Scalar loads
// of the table would share their counter with LDS: every wait for an operand would be one for the table, too.)
struct Pages {
  const int32_t* row;
  int64_t num_pages;
  int stride, n, base;
  int page;  // lane l: that of group base + l, -1: none
  __device__ __forceinline__ Pages(const Batch& b, int seq, int64_t first, int stride_, int n_)
      : row(b.table + (int64_t)seq * b.table_stride + first), num_pages(b.num_pages), stride(stride_), n(n_), base(0) {
    fetch();
  }
  __device__ __forceinline__ void fetch() {
    const int i = base + ((int)threadIdx.x & 63);
    page = i < n ? row[(int64_t)i * stride] : -1;
    if (page >= num_pages) page = -1;
  }
  // i: not decreasing from call to call
  __device__ __forceinline__ int at(int i) {
    if (i >= base + 64) {
      base = i;
      fetch();
    }
    return __builtin_amdgcn_readlane(page, i - base);
  }
};

__device__ __forceinline__ bool finite_h(uint32_t bits) { return (bits & 0x7c00u) != 0x7c00u; }

// Eight signed codes as the fp16 values 2^-24 (code + 128): denormals, which the matrix core takes as they are, so
// that a code becomes an operand with a byte's move alone.
__device__ __forceinline__ half8_t tiny8(uint32_t w0, uint32_t w1) {
  w0 ^= 0x80808080u;
  w1 ^= 0x80808080u;
  return as_h8(uint4{perm(0u, w0, 0x0c010c00u), perm(0u, w0, 0x0c030c02u), perm(0u, w1, 0x0c010c00u), perm(0u, w1, 0x0c030c02u)});
}

__device__ __forceinline__ _Float16 half_at(uint2 w, int i) {
  const half2_t h = as_h2(i < 2 ? w.x : w.y);
  return i & 1 ? h.y : h.x;
}

// Eight signed codes as fp16 whole numbers.
__device__ __forceinline__ half8_t whole8(uint32_t w0, uint32_t w1) {
  const half2_t a = scodes_to_h2(w0, kSelB01), b = scodes_to_h2(w0, kSelB23);
  const half2_t c = scodes_to_h2(w1, kSelB01), d = scodes_to_h2(w1, kSelB23);
  return half8_t{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}

// The state of a row block. Weights are at most 2^top: with the largest V scale so far (as bits at most vs, which has
// all of its exponent) P = weight times scale is 65504 at most, and no lower than that asks, so that small V lose
// nothing to fp16's denormals. In a group that some row does not see whole, the largest scale differs from row to row:
// there each row goes by those that it attends, for that group, and top stays. Of row c: off, what turns a score (log2
// domain) into a weight's exponent, and l, the sum of weights over the lane's tokens. Of rows 4 g + i: acc, the sum of
// P code (small units: 2^-24 P (code + 128), and psum that of P). A row's largest score so far has an exponent of its
// top - W_TAU at least; before its first score off is NO_SCORE, with which any score passes top.
constexpr float NO_SCORE = 3e38f;
struct RowState {
  float top, cap;  // (the wave's lanes agree on top, cap = 2^top, and vs)
  uint32_t vs;
  float off, l;
  float4_t psum, acc[8];
};
__device__ __forceinline__ void state_init(RowState& x) {
  x.top = 30.0f;
  x.cap = 0x1p30f;
  x.vs = 0x3ff;
  x.off = NO_SCORE;
  x.l = 0.0f;
  x.psum = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int cb = 0; cb < 8; ++cb) x.acc[cb] = float4_t{0.f, 0.f, 0.f, 0.f};
}
// The score (log2 domain) whose weight is 1; -inf: no token yet.
__device__ __forceinline__ float reference(const RowState& x) { return x.off == NO_SCORE ? NEG_INF : -x.off; }

// The bits of the largest of the V scales (one token's a lane) up to token `reach` of the group.
__device__ __forceinline__ uint32_t largest_up_to(uint32_t vs, int reach) {
  int m = (int)(vs & 0x7fffu);
#pragma unroll
  for (int o = 1; o < 64; o *= 2) m = max(m, __shfl_up(m, o));
  m = __shfl(m, min(max(reach, 0), 63));
  return reach < 0 ? 0u : (uint32_t)m;
}

// Whether a group has a V scale (its bits, one token's a lane) that lowers top.
__device__ __forceinline__ bool larger_scale(const RowState& x, uint32_t vs) {
  return __builtin_amdgcn_ballot_w64((vs & 0x7fffu) > x.vs) != 0;
}
__device__ __forceinline__ float uniform(float v) { return __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(v))); }

// Where the accumulators of Q K^T start: the share of the codes' offset, -128 2^-24 sum(q), of row c.
__device__ __forceinline__ float4_t offset_share(const half8_t (&qb)[4]) {
  float sum = 0.0f;
#pragma unroll
  for (int k = 0; k < 4; ++k)
#pragma unroll
    for (int e = 0; e < 8; ++e) sum += (float)qb[k][e];
  sum = sum4rows(sum) * (-128.0f * 0x1p-24f);
  return float4_t{sum, sum, sum, sum};
}

// The online softmax of a row block over 64 tokens. exponent(b, i, off): the weight's exponent of token 16 b + 4 g + i
// and row c, its score plus off (-inf where masked); vs: the tokens' V scales; ph: the weights times those, in fp16,
// as the operands of O = P V. The weights are taken with the off there is, without a maximum; only if a lane's sum
// passes 2^top (16 weights of 2^(top - W_TAU) do not), or the group has a larger V scale than top allows (`larger`, of
// the wave; scale(): the lane's token's), is off moved, what was summed up scaled, and the pass made again. masked:
// some row does not see the group whole; reach(): the last token that row c attends, counted in the group (any
// integer).
template <class M, class F, class V, class R>
__device__ __forceinline__ void weigh(RowState& x, bool larger, M masked, V&& scale, R&& reach, F&& exponent,
                                      const uint2 (&vs)[4], half8_t (&ph)[2], int g) {
  float sum;
  auto pass = [&]() {
    float part[4];
    _Float16 p16[2][8];
#pragma unroll
    for (int b = 0; b < 4; ++b)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float p = __builtin_amdgcn_exp2f(exponent(b, i, x.off));
        part[i] = b ? part[i] + p : p;
        p16[b >> 1][4 * (b & 1) + i] = (_Float16)__builtin_fmaf(p, (float)half_at(vs[b], i), 0.0f);
      }
    sum = (part[0] + part[1]) + (part[2] + part[3]);
#pragma unroll
    for (int B = 0; B < 2; ++B)
      ph[B] = half8_t{p16[B][0], p16[B][1], p16[B][2], p16[B][3], p16[B][4], p16[B][5], p16[B][6], p16[B][7]};
  };
  pass();
  asm volatile("" : "+v"(ph[0]), "+v"(ph[1]));  // (P is made here, not sunk past the branch)
  // (one comparison for both)
  if (__builtin_amdgcn_ballot_w64(sum > (larger ? -1.0f : x.cap)) != 0) {
    float cap = x.cap, top = x.top, by = 0.0f;
    if (masked && larger) {
      const uint32_t m = max(largest_up_to(scale(), reach()), x.vs);
      top = 30.0f - (float)(m >> 10);
      cap = __builtin_amdgcn_exp2f(top);
    }
    const bool own = max4rows(sum) > cap;  // (a row's result does not hang on its neighbours')
    if (!masked && larger) {
      const float all = max4rows(row16_max((float)(scale() & 0x7fffu)));
      // (this row block may be ahead of the one that `larger` was taken from)
      const uint32_t m = max((uint32_t)__builtin_amdgcn_readfirstlane((int)all), x.vs);
      const float to = 30.0f - (float)(m >> 10);  // 2^15 over the power of two in the scale
      by = x.top - to;
      x.top = uniform(to);
      x.cap = uniform(__builtin_amdgcn_exp2f(to));
      x.vs = m | 0x3ffu;
      top = x.top;
    }
    const bool first = x.off == NO_SCORE;
    float off = first ? 0.0f : x.off, t = NEG_INF;
    asm volatile("" : "+v"(off));  // (all of it in this branch: few groups come here)
#pragma unroll
    for (int b = 0; b < 4; ++b)
#pragma unroll
      for (int i = 0; i < 4; ++i) t = fmaxf(t, exponent(b, i, off));
    t = max4rows(t);
    const float moved = t - (top - W_TAU);
    const float delta = first ? moved : fmaxf(own ? moved : 0.0f, by);
    const float alpha = first ? 1.0f : __builtin_amdgcn_exp2f(-delta);
    x.off = first && t == NEG_INF ? NO_SCORE : off - delta;
    x.l *= alpha;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float ai = shfl(alpha, 4 * g + i);
#pragma unroll
      for (int cb = 0; cb < 8; ++cb) x.acc[cb][i] *= ai;
      x.psum[i] *= ai;
    }
    pass();
  }
  x.l += sum;
}
// Takes the offset's share off the sum of V, every FOLD groups of a wave: left there it would grow with the tokens, and
// with it what each addition loses (of 262144 tokens with V codes of 1, weighed alike: 12%, a multiple of the output's
// half step already from 32768).
constexpr int FOLD = 16;
__device__ __forceinline__ void fold_offset(RowState& x) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
#pragma unroll
    for (int cb = 0; cb < 8; ++cb) x.acc[cb][i] = __builtin_fmaf(x.psum[i], -128.0f * 0x1p-24f, x.acc[cb][i]);
    x.psum[i] = 0.0f;
  }
}
// Element (row 4 g + i, dim 16 cb + c) of the weighted sum of V.
__device__ __forceinline__ float value_sum(const RowState& x, int cb, int i) {
  return __builtin_fmaf(x.acc[cb][i], 0x1p24f, -128.0f * x.psum[i]);
}

// W: waves of the workgroup.
template <int RB, int W>
__device__ __forceinline__ void attend_small(const ChunkArgs& a, const Unit& u, int h, uint8_t* lds) {
  const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const TileAt at = tile_at(a, u.seq, u.row0, u.rows);
  const int fresh = a.b.cu[u.seq + 1] - a.b.cu[u.seq];  // the sequence's new tokens
  constexpr bool LATE = RB > 1;  // K's next loads after this group's scores: no registers for both
  // (whole rounds of the waves, so that no wave idles in a part's last one)
  const int64_t rounds = (at.steps + W - 1) / W;
  const int64_t s0 = rounds * u.part / u.parts * W, s1 = min(rounds * (u.part + 1) / u.parts * W, at.steps);
  const uint8_t* pages = a.pages + (int64_t)h * PAGE_TOK_BYTES;
  const int64_t page_stride = (int64_t)a.b.hkv * PAGE_TOK_BYTES;

  uint4 kn[4][2];  // the next group's K codes: token 16 b + c, bytes 16 g + 64 hh ..
  // The pages of a sequence with one tile are read once in the launch, and not kept in the caches (nontemporal); those
  // of several tiles are left there for the others.
  auto issue_k = [&](int page) {
    const uint8_t* p = reinterpret_cast<const uint8_t*>(uniform_ptr(pages + page * page_stride)) + c * D + 16 * g;
#pragma unroll
    for (int b = 0; b < 4; ++b)
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        const u32x4_t* from = reinterpret_cast<const u32x4_t*>(p + 16 * b * D + 64 * hh);
        const u32x4_t x = u.alone ? __builtin_nontemporal_load(from) : *from;
        kn[b][hh] = uint4{x.x, x.y, x.z, x.w};
      }
  };
  auto issue_v = [&](int page, int sb) {
    const uint8_t* p = reinterpret_cast<const uint8_t*>(uniform_ptr(pages + page * page_stride));
    const uint32_t slot = __builtin_amdgcn_readfirstlane(lds_addr(lds)) + (2 * wave + sb) * CH_VSLOT;
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // earlier reads of this slot are done
    auto load = [&](auto dma) {
      const int lane = tail_tid() & 63;  // (opaque: the offsets are made again at each use, for want of registers)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int row = 8 * e + (lane >> 3);
        dma(p, (uint32_t)(CODE_BYTES + row * D + (((lane & 7) ^ swz(row)) << 4)), slot + 1024 * e);
      }
      if (lane < 16) dma(p, (uint32_t)(2 * CODE_BYTES + 16 * lane), slot + CODE_BYTES);
    };
    if (u.alone) load([](const void* b, uint32_t off, uint32_t to) { dma16_stream(b, off, to); });
    else load([](const void* b, uint32_t off, uint32_t to) { dma16(b, off, to); });
  };

  int64_t s = s0 + wave;
  const int mine = s < s1 ? (int)((s1 - s + W - 1) / W) : 0;  // groups of this wave
  Pages pg(a.b, u.seq, s, W, mine);
  half8_t qb[RB][4];
  int tq[RB];  // the token of row c: the last one that it attends
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    const int r = 16 * rb + c, row = u.row0 + r;
    const bool ok = r < at.rows;
    const int tk = ok ? row / a.gq : 0, hd = h * a.gq + (ok ? row % a.gq : 0);
    tq[rb] = tk;
    const uint16_t* qr = a.q + (at.first_token + tk) * a.q_ts + hd * a.q_hs;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      uint4 w = {0, 0, 0, 0};
      if (ok) w = *reinterpret_cast<const uint4*>(qr + 16 * g + 64 * (k >> 1) + 8 * (k & 1));
      qb[rb][k] = as_h8(w);
    }
  }
  int page = pg.at(0);
  if (page >= 0) {
    issue_k(page);
    issue_v(page, 0);
  }

  const int64_t whole = (at.start + u.row0 / a.gq + 1) / GT;  // steps that every row of the tile sees whole
  const _Float16 one = (_Float16)1.0f;
  const half8_t ones = half8_t{one, one, one, one, one, one, one, one};
  float4_t start[RB];
  RowState st[RB];
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    start[rb] = offset_share(qb[rb]);
    state_init(st[rb]);
  }
  const float sl2 = a.sl2 * 0x1p24f;

  for (int t = 0; t < mine; ++t, s += W) {
    const int sb = t & 1;
    const bool here = page >= 0;
    uint4 kc[4][2];
    wait_groups_all();
#pragma unroll
    for (int b = 0; b < 4; ++b)
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) kc[b][hh] = kn[b][hh];
    page = pg.at(t + 1);
    if (page >= 0) {
      issue_v(page, sb ^ 1);
      if (!LATE || !here) issue_k(page);
    }
    if (t % FOLD == 0) {
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) fold_offset(st[rb]);
    }
    if (!here) continue;  // a group without a page takes no part

    const uint8_t* slot = lds + (2 * wave + sb) * CH_VSLOT;
    // the scales of tokens 16 b + 4 g .. + 3, as the lane's scores have them
    uint2 ks[4], vs[4];
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      ks[b] = *reinterpret_cast<const uint2*>(slot + CODE_BYTES + 2 * (16 * b + 4 * g));
      vs[b] = *reinterpret_cast<const uint2*>(slot + CODE_BYTES + 2 * GT + 2 * (16 * b + 4 * g));
    }
    // (places behind the sequence's last token hold anything)
    auto own_scale = [&]() -> uint32_t {
      const int l = tail_tid() & 63;
      const uint32_t v = *reinterpret_cast<const uint16_t*>(slot + CODE_BYTES + 2 * GT + 2 * l);
      return s >= whole && (!finite_h(v) || (int)(s * GT - at.start) + l >= fresh) ? 0u : v;
    };
    const bool larger = larger_scale(st[0], own_scale());
    float S[RB][4][4];  // scores, times 2^-24, in the natural domain
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      half8_t kop[4];
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        kop[2 * hh] = tiny8(kc[b][hh].x, kc[b][hh].y);
        kop[2 * hh + 1] = tiny8(kc[b][hh].z, kc[b][hh].w);
      }
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) {
        float4_t x = start[rb];
#pragma unroll
        for (int k = 0; k < 4; ++k) x = mfma32(kop[k], qb[rb][k], x);
#pragma unroll
        for (int i = 0; i < 4; ++i) S[rb][b][i] = __builtin_fmaf(x[i], (float)half_at(ks[b], i), 0.0f);
      }
    }
    if (LATE && page >= 0) issue_k(page);
    if (s >= whole) {
      // Masked positions: tokens behind a row's own, and the page's rows behind the sequence's last token, which
      // hold anything. Their weight is 0, but 0 times a V that is not finite is NaN, so such scales become 0;
      // where a row does attend such a token, its score becomes NaN instead. (Positions count from the sequence's
      // first new token: they fit there.)
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        int tok = (int)(s * GT - at.start) + 16 * b + 4 * g;
        asm volatile("" : "+v"(tok), "+v"(vs[b].x), "+v"(vs[b].y));  // (all of it in this branch: few groups come here)
        uint32_t v16[4] = {vs[b].x & 0xffffu, vs[b].x >> 16, vs[b].y & 0xffffu, vs[b].y >> 16};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const bool fin = finite_h(v16[i]);
#pragma unroll
          for (int rb = 0; rb < RB; ++rb) S[rb][b][i] = tok + i > tq[rb] ? NEG_INF : fin ? S[rb][b][i] : __builtin_nanf("");
          if (!fin || tok + i >= fresh) v16[i] = 0;
        }
        vs[b] = uint2{v16[0] | (v16[1] << 16), v16[2] | (v16[3] << 16)};
      }
    }
    half8_t ph[RB][2];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb)
      weigh(st[rb], larger, s >= whole, own_scale,
            [&]() { return tq[rb] - (int)(s * GT - at.start); },
            [&](int b, int i, float off) { return __builtin_fmaf(S[rb][b][i], sl2, off); }, vs, ph[rb], g);
    const int vl = tail_tid() & 63, vc = vl & 1, vr = (vl & 15) >> 1, vg = vl >> 4;
#pragma unroll
    for (int B = 0; B < 2; ++B) {
      const int vrow = 16 * (2 * B + (vr >> 2)) + 4 * vg + (vr & 3);
#pragma unroll
      for (int cb = 0; cb < 8; ++cb) {
        const u32x2 vw = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr8_b64_v2i32(
            (lds_v2i_t*)(const lds_void_t*)(slot + vrow * D + 8 * vc + ((cb ^ swz(vrow)) << 4))));
        const half8_t vop = tiny8(vw.x, vw.y);
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) st[rb].acc[cb] = mfma32(ph[rb][B], vop, st[rb].acc[cb]);
      }
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) st[rb].psum = mfma32(ph[rb][B], ones, st[rb].psum);
    }
  }

  // ---- the waves' states into one, row by row
  wait_groups_all();
  __syncthreads();  // every wave is done with its slots
  float* state = reinterpret_cast<float*>(lds) + wave * (RB * 16 * CH_PART);
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    const float l = sum4rows(st[rb].l);
    if (g == 0) {
      state[(16 * rb + c) * CH_PART + D] = reference(st[rb]);
      state[(16 * rb + c) * CH_PART + D + 1] = l;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int cb = 0; cb < 8; ++cb) state[(16 * rb + 4 * g + i) * CH_PART + 16 * cb + c] = value_sum(st[rb], cb, i);
  }
  __syncthreads();
  const int l32 = tid & 31;
#pragma unroll
  for (int p = 0; p < RB * 8 / W; ++p) {
    const int r = 2 * W * p + (tid >> 5);
    if (r >= at.rows) continue;
    const float* base = reinterpret_cast<const float*>(lds) + r * CH_PART;
    RowSum sum = {NEG_INF, 0.0f, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
    for (int w = 0; w < W; ++w) sum.m = fmaxf(sum.m, base[w * (RB * 16 * CH_PART) + D]);
    const float mu = sum.m == NEG_INF ? 0.0f : sum.m;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float* x = base + w * (RB * 16 * CH_PART);
      const float wt = __builtin_amdgcn_exp2f(x[D] - mu);
      const float4 v = *reinterpret_cast<const float4*>(x + 4 * l32);
      sum.acc.x += v.x * wt; sum.acc.y += v.y * wt; sum.acc.z += v.z * wt; sum.acc.w += v.w * wt;
      sum.l += x[D + 1] * wt;
    }
    const int row = u.row0 + r;
    if (u.parts == 1) {
      write_row(a, h, at.first_token + row / a.gq, row % a.gq, sum, l32);
    } else {
      const int64_t pr = (int64_t)u.slot + (int64_t)u.part * u.rows + r;
      if (pr >= a.ws_rows) continue;
      float* dst = a.ws + (pr * a.b.hkv + h) * CH_PART;
      *reinterpret_cast<float4*>(dst + 4 * l32) = sum.acc;
      if (l32 == 0) *reinterpret_cast<float2*>(dst + D) = float2{sum.m, sum.l};
    }
  }
}

// Units of up to 256 rows (big): wave w takes rows 32 w .. 32 w + 31 as two row blocks, and every wave every
// group. The waves turn a group's codes once into fp16 LDS tiles (whole8): K row-major (rows of 256 bytes, their
// 16-byte chunk x at x ^ (row & 15)), V transposed in the tokens' order of P's operand (rows of 128 bytes, chunk x at
// x ^ (row & 7)), the scales beside. (These swizzles read without conflicts: 5 cycles a wave's 16 bytes a lane, padded
// rows of 272 and 144 bytes take 8.)
// One barrier a step: in step t, before it, the conversion of group t + 1 into the tiles that step t - 1 read and the
// wait for the loads of group t + 2; after it the loads of group t + 4 into the stage of group t + 1.
// Bound by the vector and matrix instructions' issue: a step of a wave has 64 matrix (16 cycles each on the SIMD that
// two waves share), 32 exponentials and about 215 other instructions; 2048 tokens over 14336, 32 q and 8 KV heads (515
// GFLOP) in 591 us, 872 TFLOP/s, where a large fp16 matrix product of the library reaches 1092; 2.3 us a step, and a
// unit of one step takes 15 us (8 of them its queries' and outputs' traffic when 256 units run). Keys and values rounded
// to fp16 instead of exact codes: 578 us, and twice the error. Slower were: waves of 64 rows, for want of registers;
// the conversion at the start of the step in half of the waves (600 us); the largest score taken before the weights
// (622 us); 32 x 32 x 16 products (606 us: half as many, twice the accumulators' traffic).
constexpr int BG_RB = 2, BG_ROWS = CH_WAVES * BG_RB * 16, BG_STAGES = 3;
constexpr int BG_TILE = GT * D * 2, BG_SCALES = 8 * GT;  // a tile's scales, 32 bytes for 4 tokens: K's in fp32, V's, 0
constexpr int BG_KT = 2 * BG_SCALES, BG_VT = BG_KT + 2 * BG_TILE;  // scales, K tiles, V tiles, stages: what is read most
constexpr int BG_ST = BG_VT + 2 * BG_TILE;                         // in the range of an instruction's offset
constexpr int BG_LDS = BG_ST + BG_STAGES * PAGE_TOK_BYTES;
static_assert(BG_LDS <= CH_LDS, "both kinds of unit share the LDS");
static_assert(BG_ROWS * D * 2 <= BG_LDS, "the output of a tile fits");

__device__ __forceinline__ void attend_big(const ChunkArgs& a, const Unit& u, int h, uint8_t* lds) {
  const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const TileAt at = tile_at(a, u.seq, u.row0, u.rows);
  const int s0 = (int)(at.steps * u.part / u.parts), n = (int)(at.steps * (u.part + 1) / u.parts) - s0;
  const int64_t len = at.start + (a.b.cu[u.seq + 1] - a.b.cu[u.seq]);
  const uint8_t* pages = a.pages + (int64_t)h * PAGE_TOK_BYTES;
  const int64_t page_stride = (int64_t)a.b.hkv * PAGE_TOK_BYTES;
  const uint32_t stages = __builtin_amdgcn_readfirstlane(lds_addr(lds)) + BG_ST;
  Pages pg(a.b, u.seq, s0, 1, n);
  // wave w's loads of a group: K and V rows 8 w .. 8 w + 7, wave 0 the scales, too
  int loads = 0;  // in flight of the newest group
  auto issue = [&](int page, int slot) {
    loads = 0;
    if (page < 0) return;
    loads = wave == 0 ? 3 : 2;
    const void* p = uniform_ptr(pages + page * page_stride);
    const uint32_t dst = stages + slot * PAGE_TOK_BYTES;
    const int row = 8 * wave + (lane >> 3);
    const uint32_t off = (uint32_t)(row * D + (((lane & 7) ^ swz(row)) << 4));
    dma16(p, off, dst + 1024 * wave);
    dma16(p, off + CODE_BYTES, dst + CODE_BYTES + 1024 * wave);
    if (wave == 0 && lane < 16) dma16(p, (uint32_t)(2 * CODE_BYTES + 16 * lane), dst + 2 * CODE_BYTES);
  };
  // steps that some row of the tile does not see whole: masked places may hold anything there (attend_small)
  const int tile_whole = (int)((at.start + u.row0 / a.gq + 1) / GT) - s0;
  // Group t from its stage into its tiles: lane l of wave w takes K row l, dims 16 w .. + 15, and V dims 16 w .. + 15;
  // and the scales, with the rules for masked places where `check`. `here`: the group has a page.
  auto convert = [&](int t, int slot, auto check, bool here) {
    const uint8_t* sg = lds + BG_ST + slot * PAGE_TOK_BYTES;
    const int lane = tail_tid() & 63, c = lane & 15, g = lane >> 4, r = c >> 1;
    const uint4 kw = *reinterpret_cast<const uint4*>(sg + lane * D + ((wave ^ swz(lane)) << 4));
    const int vrow = 16 * (r >> 2) + 4 * g + (r & 3);  // and 32 further, swizzled alike
    const uint8_t* vp = sg + CODE_BYTES + vrow * D + 8 * (c & 1) + ((wave ^ swz(vrow)) << 4);
    const uint16_t* sc = reinterpret_cast<const uint16_t*>(sg + 2 * CODE_BYTES);
    uint32_t ks = sc[lane], vs = sc[GT + lane];
    if constexpr (decltype(check)::value) {
      if (!finite_h(vs)) ks = 0x7e00u, vs = 0;  // NaN
      if (!here || (int64_t)(s0 + t) * GT + lane >= len) vs = 0;
    }
    u32x2 vw[2];
#pragma unroll
    for (int B = 0; B < 2; ++B)
      vw[B] = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_v2i_t*)(const lds_void_t*)(vp + 32 * D * B)));
    uint8_t* kt = lds + BG_KT + (t & 1) * BG_TILE + lane * (2 * D);
    uint8_t* vt = lds + BG_VT + (t & 1) * BG_TILE + (16 * wave + c) * (2 * GT);
    const int kx = ((2 * wave) ^ (lane & 15)) << 4, vx = (g ^ (c & 7)) << 4;
    *reinterpret_cast<half8_t*>(kt + kx) = whole8(kw.x, kw.y);
    *reinterpret_cast<half8_t*>(kt + (kx ^ 16)) = whole8(kw.z, kw.w);
    *reinterpret_cast<half8_t*>(vt + vx) = whole8(vw[0].x, vw[0].y);
    *reinterpret_cast<half8_t*>(vt + (vx ^ 64)) = whole8(vw[1].x, vw[1].y);
    // (every wave writes the scales, the same ones: a branch would end the block that the products are mixed with)
    uint8_t* to = lds + (t & 1) * BG_SCALES + 32 * (lane >> 2);
    *reinterpret_cast<float*>(to + 4 * (lane & 3)) = h2f((uint16_t)ks) * a.sl2;
    *reinterpret_cast<uint16_t*>(to + 16 + 2 * (lane & 3)) = (uint16_t)vs;
    return vs;
  };

  const int row0 = u.row0 + wave * (BG_RB * 16);  // first row of this wave
  const int rows = u.row0 + at.rows;
  half8_t qb[BG_RB][4];  // (loaded beside the page ids)
#pragma unroll
  for (int rb = 0; rb < BG_RB; ++rb) {
    const int row = row0 + 16 * rb + c;
    const bool ok = row < rows;
    const int tk = ok ? row / a.gq : 0, hd = h * a.gq + (ok ? row % a.gq : 0);
    const uint16_t* qr = a.q + (at.first_token + tk) * a.q_ts + hd * a.q_hs;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      uint4 w = {0, 0, 0, 0};
      if (ok) w = *reinterpret_cast<const uint4*>(qr + 16 * g + 64 * (k >> 1) + 8 * (k & 1));
      qb[rb][k] = as_h8(w);
    }
  }
  int p0 = pg.at(0), p1 = pg.at(1), p2 = pg.at(2), p3 = pg.at(3);  // the pages of steps t .. t + 3
  issue(p0, 0);
  issue(p1, 1);

  RowState st[BG_RB];  // (codes are whole numbers here: acc is the sum of P code, psum stays 0)
#pragma unroll
  for (int rb = 0; rb < BG_RB; ++rb) state_init(st[rb]);
  bool larger = false;  // the next group has a larger V scale
  // this wave's rows attend steps t < mine
  const int last = min(row0 + BG_RB * 16, rows) - 1;
  const int mine = row0 < rows ? min(n, (int)((at.start + last / a.gq) / GT) + 1 - s0) : 0;

  half8_t op[16];  // the operands of the products: K's, then V's
  // where this lane reads the tiles and scales of step t: kept, opaque to the compiler so that it makes the few others
  // (an exclusive or each) at their use, for want of registers
  uint32_t ka = c * (2 * D) + (((2 * g) ^ c) << 4), va = c * (2 * GT) + ((g ^ (c & 7)) << 4), sa = 32 * g;
  auto load_k = [&]() {
    asm volatile("" : "+v"(ka));
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int b = 0; b < 4; ++b)
        op[4 * k + b] = *reinterpret_cast<const half8_t*>(lds + (ka ^ (128 * (k >> 1) + 16 * (k & 1))) +
                                                          (BG_KT + 16 * b * (2 * D)));
  };
  auto load_v = [&]() {
    asm volatile("" : "+v"(va));
#pragma unroll
    for (int B = 0; B < 2; ++B)
#pragma unroll
      for (int cb = 0; cb < 8; ++cb)
        op[8 * B + cb] = *reinterpret_cast<const half8_t*>(lds + (va ^ (64 * B)) + (BG_VT + 16 * cb * (2 * GT)));
  };
  float4_t S[BG_RB][4];
  half8_t ph[BG_RB][2];
  auto qk = [&](int rb) {
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int b = 0; b < 4; ++b)
        S[rb][b] = mfma32(op[4 * k + b], qb[rb][k], k ? S[rb][b] : float4_t{0.f, 0.f, 0.f, 0.f});
  };
  auto softmax = [&](int rb, auto masked, int t) {
    // the scales of tokens 16 b + 4 g .. + 3, K's with the softmax's factor (read again by each row block: kept for
    // both, they would not fit)
    asm volatile("" : "+v"(sa));
    float4_t ks[4];
    uint2 vs[4];
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      ks[b] = *reinterpret_cast<const float4_t*>(lds + sa + 128 * b);
      vs[b] = *reinterpret_cast<const uint2*>(lds + sa + (128 * b + 16));
    }
    const int l = tail_tid() & 63;
    const int tok0 = (int)((int64_t)(s0 + t) * GT - at.start) + 4 * (l >> 4);  // (masked: near the sequence's end, it fits)
    const int tq = (row0 + 16 * rb + (l & 15)) / a.gq;
    auto scale = [&]() { return *reinterpret_cast<const uint16_t*>(lds + (t & 1) * BG_SCALES + 32 * (l >> 2) + 16 + 2 * (l & 3)); };
    auto reach = [&]() { return tq - (int)((int64_t)(s0 + t) * GT - at.start); };
    const bool part = decltype(masked)::value && __builtin_amdgcn_readfirstlane(reach()) < GT - 1;  // (the first row's)
    weigh(st[rb], larger, part, scale, reach, [&](int b, int i, float off) {
      const float e = __builtin_fmaf(S[rb][b][i], ks[b][i], off);
      return decltype(masked)::value && tok0 + 16 * b + i > tq ? NEG_INF : e;
    }, vs, ph[rb], l >> 4);
  };
  auto pv = [&](int rb) {
#pragma unroll
    for (int B = 0; B < 2; ++B)
#pragma unroll
      for (int cb = 0; cb < 8; ++cb) st[rb].acc[cb] = mfma32(ph[rb][B], op[8 * B + cb], st[rb].acc[cb]);
  };

  wait_groups_all();
  __syncthreads();
  if (n > 0) larger = larger_scale(st[0], convert(0, 0, std::true_type{}, p0 >= 0));
  __syncthreads();
  issue(p2, 2);
  issue(p3, 0);
  int r1 = 1;  // (t + 1) mod 3

  // One step. `fast`: every row sees groups t and t + 1 whole, and both have a page. A wave issues in order, so
  // the products of one row block are placed between the softmax instructions of the other: QK(1) beside softmax(0),
  // PV(0) beside softmax(1), PV(1) beside the conversion.
  auto step = [&](int t, auto fast_) {
    constexpr bool fast = decltype(fast_)::value;
    using masked = std::integral_constant<bool, !fast>;
    const int p4 = pg.at(t + 4);
    const bool go = fast || (t < mine && p0 >= 0);
    if (go) {
      load_k();
      qk(0);
      qk(1);
      softmax(0, masked{}, t);
      load_v();
      pv(0);
      softmax(1, masked{}, t);
    }
    uint32_t vs = 0;
    if constexpr (fast) vs = convert(t + 1, r1, std::false_type{}, true);
    else if (t + 1 < n) vs = convert(t + 1, r1, std::true_type{}, p1 >= 0);
    if (go) pv(1);
    larger = larger_scale(st[0], vs);
    // tile t + 1 is written, tile t is read, group t + 2 has landed
    if (loads == 2) asm volatile("s_waitcnt vmcnt(2) lgkmcnt(0)" ::: "memory");
    else if (loads == 3) asm volatile("s_waitcnt vmcnt(3) lgkmcnt(0)" ::: "memory");
    else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    asm volatile("s_barrier" ::: "memory");
    issue(p4, r1);
    r1 = r1 == 2 ? 0 : r1 + 1;
    p0 = p1; p1 = p2; p2 = p3; p3 = p4;
    ka ^= BG_TILE; va ^= BG_TILE; sa ^= BG_SCALES;
  };
  int t = 0;
  for (; t + 1 < min(n, tile_whole) && p0 >= 0 && p1 >= 0; ++t) step(t, std::true_type{});
  for (; t < n; ++t) step(t, std::false_type{});
  wait_groups_all();
  float rl[BG_RB];  // row c's sum of weights
#pragma unroll
  for (int rb = 0; rb < BG_RB; ++rb) rl[rb] = sum4rows(st[rb].l);

  if (u.parts == 1) {
    // ---- out = the sum of V / l, through LDS so that 16 lanes store a row's 256 bytes (the 2-byte values
    // at chunk ^ 2 ((row >> 2) & 3))
    __syncthreads();  // every wave is past its last read of the tiles
    const int lane = tail_tid() & 63, c = lane & 15, g = lane >> 4;  // (made again, for want of registers in the loop)
    uint8_t* ow = lds + wave * (BG_RB * 16 * D * 2);
#pragma unroll
    for (int rb = 0; rb < BG_RB; ++rb)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float l = shfl(rl[rb], 4 * g + i), inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
        const float m = shfl(reference(st[rb]), 4 * g + i);
        const int r = 16 * rb + 4 * g + i, row = row0 + r;
#pragma unroll
        for (int cb = 0; cb < 8; ++cb)
          *reinterpret_cast<uint16_t*>(ow + r * (2 * D) + (((2 * cb + (c >> 3)) ^ (((r >> 2) & 3) << 1)) << 4) + 2 * (c & 7)) =
              f2h(st[rb].acc[cb][i] * inv);
        if (a.lse && c == 0 && row < rows)
          a.lse[(at.first_token + row / a.gq) * a.hq + h * a.gq + row % a.gq] =
              l == 0.0f ? NEG_INF : (m + __builtin_amdgcn_logf(l)) * LN2;
      }
#pragma unroll
    for (int k = 0; k < BG_RB * 4; ++k) {
      const int r = 4 * k + g, row = row0 + r;
      const uint4 v = *reinterpret_cast<const uint4*>(ow + r * (2 * D) + ((c ^ (((r >> 2) & 3) << 1)) << 4));
      if (row < rows)
        *reinterpret_cast<uint4*>(a.out + (at.first_token + row / a.gq) * a.o_ts + (h * a.gq + row % a.gq) * a.o_hs + 8 * c) = v;
    }
  } else {
    const int64_t pr0 = (int64_t)u.slot + (int64_t)u.part * u.rows + wave * (BG_RB * 16);
#pragma unroll
    for (int rb = 0; rb < BG_RB; ++rb) {
      if (g == 0 && row0 + 16 * rb + c < rows && pr0 + 16 * rb + c < a.ws_rows)
        *reinterpret_cast<float2*>(a.ws + ((pr0 + 16 * rb + c) * a.b.hkv + h) * CH_PART + D) = float2{reference(st[rb]), rl[rb]};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = 16 * rb + 4 * g + i;
        if (row0 + r >= rows || pr0 + r >= a.ws_rows) continue;
        float* dst = a.ws + ((pr0 + r) * a.b.hkv + h) * CH_PART;
#pragma unroll
        for (int cb = 0; cb < 8; ++cb) dst[16 * cb + c] = st[rb].acc[cb][i];
      }
    }
  }
}

__global__ __launch_bounds__(CH_THREADS, 1) void attn_chunks_kernel(ChunkArgs a) {
  __shared__ __attribute__((aligned(16))) uint8_t lds[CH_LDS];
  const int h = blockIdx.x % a.b.hkv;
  const Unit u = a.units[blockIdx.x / a.b.hkv];
  if (u.seq < 0 || u.seq >= a.b.nseq || u.row0 < 0 || u.rows <= 0 || u.rows > BG_ROWS || u.part < 0 || u.part >= u.parts ||
      u.slot < 0)
    return;
  if (u.kind == ROWS256) attend_big(a, u, h, lds);
  else if (u.rows > 32) return;
  else if (u.rows <= 16) attend_small<1, CH_WAVES>(a, u, h, lds);
  else attend_small<2, CH_WAVES>(a, u, h, lds);
}

// A launch without units of more than 32 rows: workgroups of four waves, two on a CU, so that one's start and end (a
// chain of loads that wait for each other, the merge of its waves) pass beside the other's stream.
constexpr int SM_WAVES = 4;
__global__ __launch_bounds__(64 * SM_WAVES, 2) void attn_small_chunks_kernel(ChunkArgs a) {
  __shared__ __attribute__((aligned(16))) uint8_t lds[2 * SM_WAVES * CH_VSLOT];
  const int h = blockIdx.x % a.b.hkv;
  const Unit u = a.units[blockIdx.x / a.b.hkv];
  if (u.seq < 0 || u.seq >= a.b.nseq || u.row0 < 0 || u.rows <= 0 || u.rows > 32 || u.part < 0 || u.part >= u.parts || u.slot < 0)
    return;
  if (u.rows <= 16) attend_small<1, SM_WAVES>(a, u, h, lds);
  else attend_small<2, SM_WAVES>(a, u, h, lds);
}

// The parts of a tile's rows into one: 32 lanes a row, 8 rows a workgroup. The entry holds all that it needs, and the
// columns of 8 parts are in flight beside the weights' loads: two waits for memory in a row for up to 8 parts. 2.7 us
// for few rows, 7 us for 45760 partial rows (24 MB, 3.4 TB/s).
__global__ __launch_bounds__(256) void merge_chunks_kernel(ChunkArgs a, const Merge* merges) {
  const int h = blockIdx.x % a.b.hkv;
  const Merge g = merges[blockIdx.x / a.b.hkv];
  const int r = threadIdx.x >> 5, l32 = threadIdx.x & 31, row = g.row0 + r;
  const int64_t token = (int64_t)g.first + row / a.gq;
  if (r >= g.rows || g.first < 0 || g.row0 < 0 || token >= a.tokens || g.slot < 0 || g.stride < 0 || g.parts <= 0 ||
      g.slot + (int64_t)(g.parts - 1) * g.stride + r >= a.ws_rows)
    return;  // (32 lanes agree)
  const float* base = a.ws + (((int64_t)g.slot + r) * a.b.hkv + h) * CH_PART;
  const int64_t step = (int64_t)g.stride * a.b.hkv * CH_PART;
  RowSum sum = {NEG_INF, 0.0f, {0.f, 0.f, 0.f, 0.f}};
  constexpr int FLY = 8;
  float4 v[FLY];
  auto columns = [&](int p0) {
#pragma unroll
    for (int e = 0; e < FLY; ++e) v[e] = *reinterpret_cast<const float4*>(base + min(p0 + e, g.parts - 1) * step + 4 * l32);
  };
  columns(0);
  float2 ml = {NEG_INF, 0.0f};
  if (l32 < g.parts) ml = *reinterpret_cast<const float2*>(base + l32 * step + D);
  sum.m = ml.x;
  for (int p = l32 + 32; p < g.parts; p += 32) sum.m = fmaxf(sum.m, base[p * step + D]);
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) sum.m = fmaxf(sum.m, __shfl_xor(sum.m, o, 32));
  const float mu = sum.m == NEG_INF ? 0.0f : sum.m;
  for (int p0 = 0; p0 < g.parts; p0 += FLY) {
    if (p0) columns(p0);
    if (p0 % 32 == 0 && p0) {
      ml = float2{NEG_INF, 0.0f};
      if (p0 + l32 < g.parts) ml = *reinterpret_cast<const float2*>(base + (p0 + l32) * step + D);
    }
    const float wt = __builtin_amdgcn_exp2f(ml.x - mu);
#pragma unroll
    for (int e = 0; e < FLY; ++e) {
      const int from = (p0 + e) & 31;
      const float we = __shfl(wt, from, 32), le = __shfl(ml.y, from, 32);
      if (p0 + e < g.parts) {
        sum.acc.x += v[e].x * we; sum.acc.y += v[e].y * we; sum.acc.z += v[e].z * we; sum.acc.w += v[e].w * we;
        sum.l += le * we;
      }
    }
  }
  write_row(a, h, token, row % a.gq, sum, l32);
}

// ---------------------------------------------------------------- host side

bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

int batch_args(const char* what, Batch& b, const int32_t* seq_of, bool need_seq_of, const int32_t* cu, const int64_t* start,
               const int32_t* table, int64_t table_stride, int64_t num_pages, int64_t nseq, int64_t hkv, int64_t head_dim,
               int64_t tokens) {
  if (head_dim != D) return fail(NKV_ERR_UNSUPPORTED, "%s: head_dim %lld: the HIP kernels are built for head_dim 128", what, (long long)head_dim);
  if (nseq <= 0 || nseq > 32767 || hkv <= 0 || hkv > 1024 || table_stride <= 0 || num_pages <= 0 || num_pages > (int64_t(1) << 31))
    return fail(NKV_ERR_INVALID, "%s: bad sizes nseq=%lld hkv=%lld table_stride=%lld num_pages=%lld", what, (long long)nseq,
                (long long)hkv, (long long)table_stride, (long long)num_pages);
  if (tokens < 0 || tokens >= (int64_t(1) << 24))  // (a launch has less than 2^32 threads)
    return fail(NKV_ERR_INVALID, "%s: %lld tokens outside [0, 2^24)", what, (long long)tokens);
  if (tokens > 0 && ((need_seq_of && !seq_of) || !cu || !start || !table)) return fail(NKV_ERR_INVALID, "%s: null pointer argument", what);
  b = Batch{seq_of, cu, start, table, table_stride, num_pages, (int)nseq, (int)hkv};
  return NKV_OK;
}

// The heads of few tokens are spread over workgroups (12 tokens: 3.7 us, all 48 heads in one 4.6 us), those of many
// are not (1029 tokens: 7.3 us, spread 8.6 us; 4112 tokens 20.6 and 25.8 us: each workgroup makes the angles). From 2048
// tokens the queries are stored past the caches (us nontemporal / ordinary, 32 q and 8 KV heads): 2048 tokens 12.0 /
// 12.8, 4112 20.1 / 20.7; 8 and 2 heads, 4112 tokens 9.6 / 10.3; 4 and 2, 16000 26.1 / 26.5. With a kernel that reads
// the queries next, both: 19.7 / 20.1, 31.9 / 31.1, 14.9 / 16.1, 33.3 / 32.6. Few tokens gain nothing (300: 5.1 / 5.1).
// In between it would gain, too (1029 tokens 7.9 / 8.9, with the reader 12.7 / 15.0).
template <int DT>
void launch_append(const AppendArgs& a, hipStream_t s) {
  const int heads = a.hq + 2 * a.b.hkv;
  AppendArgs c = a;
  c.heads_per_wg = a.tokens < CUS ? 16 : heads;
  const dim3 grid((unsigned)a.tokens, (unsigned)cdiv(heads, c.heads_per_wg));
  if (a.tokens >= 8 * CUS) hipLaunchKernelGGL((append_chunks_kernel<DT, true>), grid, dim3(256), 0, s, c);
  else hipLaunchKernelGGL((append_chunks_kernel<DT, false>), grid, dim3(256), 0, s, c);
}

template <bool T64, int TOK>
void launch_read_as(const ReadArgs& a, int dtype, hipStream_t s) {
  const dim3 grid((unsigned)cdiv(a.tokens, TOK));
  if (dtype == NKV_F16) hipLaunchKernelGGL((read_kernel<NKV_F16, T64, TOK>), grid, dim3(256), 0, s, a);
  else if (dtype == NKV_BF16) hipLaunchKernelGGL((read_kernel<NKV_BF16, T64, TOK>), grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((read_kernel<NKV_F32, T64, TOK>), grid, dim3(256), 0, s, a);
}

// Few tokens want all the workgroups that there are, many tokens few waits for the chain at a workgroup's start. Tokens a
// workgroup 1 / 4 / 16, 8 KV heads: 275 tokens 3.3 / 4.5 / 9.5 us, 5418 tokens of int8t64 16.1 / 14.4 / 19.6 us, 70000
// tokens 16: 98 us, 4: 101 us. Stores of the long ones pass the caches (store8).
template <bool T64>
void launch_read(const ReadArgs& a, int dtype, hipStream_t s) {
  if (a.tokens * a.b.hkv <= 16 * CUS) launch_read_as<T64, 1>(a, dtype, s);
  else if (a.tokens * a.b.hkv <= 512 * CUS) launch_read_as<T64, 4>(a, dtype, s);
  else launch_read_as<T64, 16>(a, dtype, s);
}

int read_tokens(const char* what, bool t64, const uint8_t* pages, const int32_t* page_table, int64_t table_stride,
                int64_t num_pages, const uint16_t* rings, const int64_t* length_dev, const int32_t* seq_of,
                const int32_t* cu, const int64_t* start_dev, int64_t tokens, int64_t nseq, int64_t hkv, int64_t head_dim,
                void* k_out, void* v_out, int out_dtype, void* stream) {
  set_error("");
  ReadArgs a{};
  if (int rc = batch_args(what, a.b, seq_of, true, cu, start_dev, page_table, table_stride, num_pages, nseq, hkv, head_dim, tokens))
    return rc;
  if (out_dtype != NKV_F16 && out_dtype != NKV_BF16 && out_dtype != NKV_F32)
    return fail(NKV_ERR_INVALID, "%s: unknown dtype %d", what, out_dtype);
  if (tokens == 0) return NKV_OK;
  if (!pages || !k_out || !v_out || (t64 && (!rings || !length_dev))) return fail(NKV_ERR_INVALID, "%s: null pointer argument", what);
  if (!al16(pages) || !al16(k_out) || !al16(v_out) || (t64 && !al16(rings)))
    return fail(NKV_ERR_UNSUPPORTED, "%s: buffers must be 16-byte aligned", what);
  a.tokens = tokens;
  a.pages = pages; a.rings = rings; a.length = length_dev;
  a.k_out = static_cast<uint8_t*>(k_out); a.v_out = static_cast<uint8_t*>(v_out);
  if (t64) launch_read<true>(a, out_dtype, static_cast<hipStream_t>(stream));
  else launch_read<false>(a, out_dtype, static_cast<hipStream_t>(stream));
  return check_launch(what);
}

}  // namespace

}  // namespace nkv

using namespace nkv;

extern "C" int nkv_paged_append_chunks_tok(const void* qkv, int qkv_dtype, int64_t row_stride, int64_t tokens,
                                           uint8_t* pages, const int32_t* page_table, int64_t table_stride,
                                           int64_t num_pages, const int32_t* seq_of, const int32_t* cu,
                                           const int64_t* start_dev, int64_t nseq, int64_t hq, int64_t hkv,
                                           int64_t head_dim, const void* q_gamma, const void* k_gamma, float eps,
                                           const float* inv_freq, uint16_t* q_out, int64_t q_row_stride, void* stream) {
  set_error("");
  const char* what = "paged_append_chunks_tok";
  AppendArgs a{};
  if (int rc = batch_args(what, a.b, seq_of, true, cu, start_dev, page_table, table_stride, num_pages, nseq, hkv, head_dim, tokens))
    return rc;
  if (qkv_dtype != NKV_F16 && qkv_dtype != NKV_BF16 && qkv_dtype != NKV_F32)
    return fail(NKV_ERR_INVALID, "%s: unknown dtype %d", what, qkv_dtype);
  if (hq <= 0 || hq > 16 * hkv || hq % hkv) return fail(NKV_ERR_INVALID, "%s: heads hq=%lld hkv=%lld", what, (long long)hq, (long long)hkv);
  if (row_stride < (hq + 2 * hkv) * D || q_row_stride < hq * D)
    return fail(NKV_ERR_INVALID, "%s: row strides %lld and %lld for %lld q and %lld KV heads", what, (long long)row_stride,
                (long long)q_row_stride, (long long)hq, (long long)hkv);
  if (tokens == 0) return NKV_OK;
  if (!qkv || !pages || !q_out || (!q_gamma != !k_gamma)) return fail(NKV_ERR_INVALID, "%s: null pointer argument", what);
  if (!al16(qkv) || !al16(pages) || !al16(q_out) || !al16(q_gamma) || !al16(k_gamma) || row_stride % 8 || q_row_stride % 8)
    return fail(NKV_ERR_UNSUPPORTED, "%s: rows and buffers must be 16-byte aligned", what);
  a.x = static_cast<const uint8_t*>(qkv); a.x_rs = row_stride; a.tokens = tokens; a.pages = pages;
  a.q_gamma = static_cast<const uint8_t*>(q_gamma); a.k_gamma = static_cast<const uint8_t*>(k_gamma);
  a.eps = eps; a.inv_freq = inv_freq; a.q_out = q_out; a.q_rs = q_row_stride; a.hq = (int)hq;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (qkv_dtype == NKV_F16) launch_append<NKV_F16>(a, s);
  else if (qkv_dtype == NKV_BF16) launch_append<NKV_BF16>(a, s);
  else launch_append<NKV_F32>(a, s);
  return check_launch(what);
}

extern "C" int nkv_paged_read_tok(const uint8_t* pages, const int32_t* page_table, int64_t table_stride, int64_t num_pages,
                                  const int32_t* seq_of, const int32_t* cu, const int64_t* start_dev, int64_t tokens,
                                  int64_t nseq, int64_t hkv, int64_t head_dim, void* k_out, void* v_out, int out_dtype,
                                  void* stream) {
  return read_tokens("paged_read_tok", false, pages, page_table, table_stride, num_pages, nullptr, nullptr, seq_of, cu,
                     start_dev, tokens, nseq, hkv, head_dim, k_out, v_out, out_dtype, stream);
}

extern "C" int nkv_paged_read_t64(const uint8_t* pages, const int32_t* page_table, int64_t table_stride, int64_t num_pages,
                                  const uint16_t* rings, const int64_t* length_dev, const int32_t* seq_of,
                                  const int32_t* cu, const int64_t* start_dev, int64_t tokens, int64_t nseq, int64_t hkv,
                                  int64_t head_dim, void* k_out, void* v_out, int out_dtype, void* stream) {
  return read_tokens("paged_read_t64", true, pages, page_table, table_stride, num_pages, rings, length_dev, seq_of, cu,
                     start_dev, tokens, nseq, hkv, head_dim, k_out, v_out, out_dtype, stream);
}

extern "C" int64_t nkv_paged_chunks_workspace_bytes(int64_t hkv, int64_t partial_rows) {
  return hkv > 0 && partial_rows > 0 ? partial_rows * hkv * CH_PART * (int64_t)sizeof(float) : 0;
}

extern "C" int nkv_paged_attn_chunks_tok(const uint16_t* q, int64_t q_token_stride, int64_t q_head_stride, int64_t tokens,
                                         const uint8_t* pages, const int32_t* page_table, int64_t table_stride,
                                         int64_t num_pages, const int32_t* cu, const int64_t* start_dev, int64_t nseq,
                                         int64_t hq, int64_t hkv, int64_t head_dim, const int32_t* units, int64_t n_units, int wide,
                                         const int32_t* merges, int64_t n_merges, uint16_t* out, int64_t out_token_stride,
                                         int64_t out_head_stride, float* lse_out, void* workspace, int64_t workspace_bytes,
                                         void* stream) {
  set_error("");
  const char* what = "paged_attn_chunks_tok";
  ChunkArgs a{};
  if (int rc = batch_args(what, a.b, nullptr, false, cu, start_dev, page_table, table_stride, num_pages, nseq, hkv, head_dim, tokens))
    return rc;
  if (hq <= 0 || hq > 16 * hkv || hq % hkv) return fail(NKV_ERR_INVALID, "%s: heads hq=%lld hkv=%lld", what, (long long)hq, (long long)hkv);
  constexpr int64_t MOST = (int64_t(1) << 23) - 1;  // workgroups: a launch has less than 2^32 threads
  if (n_units < 0 || n_merges < 0 || n_units > MOST / hkv || n_merges > MOST / hkv)
    return fail(NKV_ERR_INVALID, "%s: %lld units and %lld merges of %lld KV heads", what, (long long)n_units,
                (long long)n_merges, (long long)hkv);
  if (tokens == 0 || n_units == 0) return NKV_OK;
  if (!q || !pages || !units || !out || (n_merges && (!merges || !workspace)))
    return fail(NKV_ERR_INVALID, "%s: null pointer argument", what);
  if (!al16(q) || !al16(pages) || !al16(out) || !al16(units) || (n_merges && (!al16(merges) || !al16(workspace))) ||
      q_token_stride % 8 || q_head_stride % 8 || out_token_stride % 8 || out_head_stride % 8)
    return fail(NKV_ERR_UNSUPPORTED, "%s: rows and buffers must be 16-byte aligned", what);
  a.q = q; a.q_ts = q_token_stride; a.q_hs = q_head_stride; a.tokens = tokens; a.pages = pages;
  a.units = reinterpret_cast<const Unit*>(units);
  a.hq = (int)hq; a.gq = (int)(hq / hkv);
  a.sl2 = LOG2E / sqrtf((float)D);
  a.out = out; a.o_ts = out_token_stride; a.o_hs = out_head_stride; a.lse = lse_out;
  a.ws = static_cast<float*>(workspace);
  a.ws_rows = workspace && workspace_bytes > 0 ? workspace_bytes / (hkv * CH_PART * (int64_t)sizeof(float)) : 0;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const dim3 grid((unsigned)(n_units * hkv));
  if (wide) hipLaunchKernelGGL(attn_chunks_kernel, grid, dim3(CH_THREADS), 0, s, a);
  else hipLaunchKernelGGL(attn_small_chunks_kernel, grid, dim3(64 * SM_WAVES), 0, s, a);
  if (int rc = check_launch(what)) return rc;
  if (n_merges) {
    hipLaunchKernelGGL(merge_chunks_kernel, dim3((unsigned)(n_merges * hkv)), dim3(256), 0, s, a,
                       reinterpret_cast<const Merge*>(merges));
    return check_launch(what);
  }
  return NKV_OK;
}
