// What the calls over a packed batch share (gfx950, wave64): where its tokens are, eight values of a row in any
// element type, the units of its attention and the joining of their parts.
//
// Token t of the packed batch belongs to sequence seq_of[t] and is its new token t - cu[seq]; its position is
// start[seq] + that. Lengths and positions are read on the device, so a captured graph follows them.
#pragma once

#include "nkv_mfma.h"

namespace nkv {

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

// Sum over the 16 lanes of each 16-lane row (DPP only; every lane gets it).
__device__ __forceinline__ float row16_sum(float v) {
  v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0xB1, 0xf, 0xf, false));
  v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x4E, 0xf, 0xf, false));
  v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x124, 0xf, 0xf, false));
  v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x128, 0xf, 0xf, false));
  return v;
}

// ---------------------------------------------------------------- attention
//
// The rows of KV head h in sequence b: row R = (new token R / gq, q head h gq + R % gq), gq = hq / hkv. They
// are cut into tiles; a tile attends the 64-token groups up to its last token (steps 0 .. S - 1), and its
// steps are cut into parts, unit = one part of one tile. Part p of P takes steps [S p / P, S (p + 1) / P),
// from the S of the device's lengths: the plan stays valid while sequences grow.

constexpr int CH_PART = D + 4;                           // floats of a row's partial: acc[128], m, l, pad

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

// Joins the parts of cut tiles (n_merges entries): defined once, for every page format.
int launch_merges(const char* what, const ChunkArgs& a, const Merge* merges, int64_t n_merges, hipStream_t s);

// ---------------------------------------------------------------- host side

inline bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

inline int batch_args(const char* what, Batch& b, const int32_t* seq_of, bool need_seq_of, const int32_t* cu, const int64_t* start,
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

// The attention calls' arguments, checked. any: there is something to launch.
inline int chunk_args(const char* what, ChunkArgs& a, bool& any, const uint16_t* q, int64_t q_token_stride,
                      int64_t q_head_stride, int64_t tokens, const uint8_t* pages, const int32_t* page_table,
                      int64_t table_stride, int64_t num_pages, const int32_t* cu, const int64_t* start_dev, int64_t nseq,
                      int64_t hq, int64_t hkv, int64_t head_dim, const int32_t* units, int64_t n_units, const int32_t* merges,
                      int64_t n_merges, uint16_t* out, int64_t out_token_stride, int64_t out_head_stride, float* lse_out,
                      void* workspace, int64_t workspace_bytes) {
  set_error("");
  if (int rc = batch_args(what, a.b, nullptr, false, cu, start_dev, page_table, table_stride, num_pages, nseq, hkv, head_dim, tokens))
    return rc;
  if (hq <= 0 || hq > 16 * hkv || hq % hkv) return fail(NKV_ERR_INVALID, "%s: heads hq=%lld hkv=%lld", what, (long long)hq, (long long)hkv);
  constexpr int64_t MOST = (int64_t(1) << 23) - 1;  // workgroups: a launch has less than 2^32 threads
  if (n_units < 0 || n_merges < 0 || n_units > MOST / hkv || n_merges > MOST / hkv)
    return fail(NKV_ERR_INVALID, "%s: %lld units and %lld merges of %lld KV heads", what, (long long)n_units,
                (long long)n_merges, (long long)hkv);
  any = tokens > 0 && n_units > 0;
  if (!any) return NKV_OK;
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
  return NKV_OK;
}

}  // namespace nkv
