// The 4-bit format (nkv_q4.h): quantizers of weights and of a prompt's keys and values, and the attention of a packed
// batch's new tokens over 4-bit pages. (The packed batch's append and read: nkv_chunks.hip; the products with 4-bit weights:
// nkv_q4_gemv.hip.)

#include <algorithm>
#include <type_traits>

#include "nkv_paged.h"
#include "nkv_q4.h"

namespace nkv {

namespace {

// ---------------------------------------------------------------- quantizers

struct Quant4Args {
  const uint8_t* x;
  int64_t head_stride;   // pages: elements from head to head
  int64_t chunks;        // of eight values, all rows'
  uint8_t* codes;        // a word a chunk
  uint16_t* scales;      // one for four chunks
  // pages: row r of head h is token first + r of a sequence, of tensor `which`; tokens whose table entry is outside
  // [0, num_pages) are skipped
  uint8_t* pages;
  const int32_t* table;
  int64_t n, hkv, first, num_pages;
  int which;
};

// Eight values a lane, a group to four lanes, both ways bound by memory.
template <int DT, bool PAGES>
__global__ __launch_bounds__(256) void quant4_kernel(Quant4Args a) {
  const int64_t step = (int64_t)gridDim.x * 256;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < a.chunks; i += step) {  // (four lanes agree: chunks % 4 == 0)
    Raw8<DT> r;
    float v[8];
    uint16_t scale;
    if constexpr (PAGES) {
      const int64_t row = i >> 4, h = row / a.n, t = row % a.n, tok = a.first + t;
      const int j = (int)(i & 15), slot = (int)(tok % GT);
      r.load(a.x + (h * a.head_stride + t * D + 8 * j) * Elem<DT>::SIZE);
      const int32_t page = a.table[tok / GT];
      r.get(v);
      const uint32_t w = q4_quant8(v, scale);
      if (page < 0 || page >= a.num_pages) continue;
      uint8_t* p = a.pages + ((int64_t)page * a.hkv + h) * PAGE_Q4_BYTES;
      *reinterpret_cast<uint32_t*>(p + a.which * Q4_CODES + slot * Q4_ROW + 4 * j) = w;
      const int to = a.which ? v_scale_at(slot, j / 4) : k_scale_at(slot, j / 4);
      if (j % 4 == 0) *reinterpret_cast<uint16_t*>(p + 2 * Q4_CODES + a.which * Q4_SCALES + 2 * to) = scale;
    } else {
      r.load(a.x + i * (8 * Elem<DT>::SIZE));
      r.get(v);
      const uint32_t w = q4_quant8(v, scale);
      reinterpret_cast<uint32_t*>(a.codes)[i] = w;
      if (i % 4 == 0) a.scales[i / 4] = scale;
    }
  }
}

template <int DT>
__global__ __launch_bounds__(256) void dequant4_kernel(const uint32_t* codes, const uint16_t* scales, int64_t chunks, uint8_t* out) {
  const int64_t step = (int64_t)gridDim.x * 256;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < chunks; i += step) {
    const uint32_t w = codes[i];
    const float s = h2f(scales[i / 4]);
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = q4_value(w, e, s);
    store8<DT, false>(out + i * (8 * Elem<DT>::SIZE), v);
  }
}

// ---------------------------------------------------------------- attention
//
// softmax(q K^T / sqrt(128)) V. K and V are exact fp16 operands (nkv_q4.h); what is rounded to fp16 is the softmax's weights
// and the output. The units of up to 32 rows ("small"): a workgroup's waves take the part's pages in turn, each its own
// page against all the rows, and their states are merged in LDS at the end. K's codes go from memory to registers: lane
// c + 16 g of tile b takes the 16 bytes of channels 32 g .. + 31 of token 16 (c / 4) + 4 b + c % 4, one scale's codes.
// V's codes and the scales go to LDS, where the transposing read gives lane c + 16 g channel 16 cb + c of tokens 16 g ..
// + 15: those that its scores are of.

constexpr uint32_t Q4_LARGEST = 0x7090;  // the largest scale that is held (9344): beyond it values are not finite in fp16
constexpr int Q4_WAVES = 8, Q4_THREADS = 64 * Q4_WAVES;
constexpr int Q4_SLOT = Q4_CODES + 2 * Q4_SCALES;  // V codes, K scales, V scales: the rest of a page after K's codes
static_assert(16 * CH_PART * 4 <= 2 * Q4_SLOT, "a wave's 16 rows fit its slots at the merge");

// XOR key of the 16-byte chunks of V row `row` in LDS: the 16 rows of a transposing read hit 16 places.
__device__ __forceinline__ int swz4(int row) { return (row >> 2) & 3; }

// The state of a row block: of row c the offset that turns a score (log2 domain) into a weight's exponent, and l, the sum
// of weights over the lane's tokens; of rows 4 g + i acc, the sum of weight times V. A lane's weights sum up to at most
// CAP = 2^15, so that fp16 holds them; a row's largest score so far has a weight of 2^11 at least, so that weights down to
// 2^-36 of the largest are held.
constexpr float Q4_NO_SCORE = 3e38f, Q4_CAP = 0x1p15f, Q4_FIRST = 11.0f;
struct Sum4 {
  float off, l;
  float4_t acc[8];
};
__device__ __forceinline__ void init(Sum4& x) {
  x.off = Q4_NO_SCORE;
  x.l = 0.0f;
#pragma unroll
  for (int cb = 0; cb < 8; ++cb) x.acc[cb] = float4_t{0.f, 0.f, 0.f, 0.f};
}
// The score (log2 domain) whose weight is 1; -inf: no token yet.
__device__ __forceinline__ float reference(const Sum4& x) { return x.off == Q4_NO_SCORE ? NEG_INF : -x.off; }

// The online softmax of a row block over 64 tokens: S[b][i] the score of token 16 g + 4 b + i and row c (-inf where masked), ph
// the weights as the operands of P V, in unpack4's order. The weights are taken with the offset there is, without a maximum;
// only if a lane's sum passes CAP is the offset moved, what was summed up scaled, and the pass made again.
__device__ __forceinline__ void weigh(Sum4& x, const float4_t (&S)[4], float sl2, half8_t (&ph)[2], int g) {
  float sum;
  auto pass = [&]() {
    float part[4];
    _Float16 p16[4][4];
#pragma unroll
    for (int b = 0; b < 4; ++b)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(S[b][i], sl2, x.off));
        part[i] = b ? part[i] + p : p;
        p16[b][i] = (_Float16)p;
      }
    sum = (part[0] + part[1]) + (part[2] + part[3]);
#pragma unroll
    for (int w = 0; w < 2; ++w)
      ph[w] = half8_t{p16[2 * w][0], p16[2 * w + 1][0], p16[2 * w][1], p16[2 * w + 1][1],
                      p16[2 * w][2], p16[2 * w + 1][2], p16[2 * w][3], p16[2 * w + 1][3]};
  };
  pass();
  if (__builtin_amdgcn_ballot_w64(sum > Q4_CAP) != 0) {
    const bool own = max4rows(sum) > Q4_CAP;  // (a row's result does not hang on its neighbours')
    const bool first = x.off == Q4_NO_SCORE;
    const float off = first ? 0.0f : x.off;
    float t = NEG_INF;
#pragma unroll
    for (int b = 0; b < 4; ++b)
#pragma unroll
      for (int i = 0; i < 4; ++i) t = fmaxf(t, __builtin_fmaf(S[b][i], sl2, off));
    t = max4rows(t);
    const float delta = first ? t - Q4_FIRST : own ? t - Q4_FIRST : 0.0f;
    const float alpha = first ? 1.0f : __builtin_amdgcn_exp2f(-delta);
    x.off = first && t == NEG_INF ? Q4_NO_SCORE : off - delta;
    x.l *= alpha;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float ai = shfl(alpha, 4 * g + i);
#pragma unroll
      for (int cb = 0; cb < 8; ++cb) x.acc[cb][i] *= ai;
    }
    pass();
  }
  x.l += sum;
}

__device__ __forceinline__ half2_t twice(uint32_t bits) { return as_h2(bits | (bits << 16)); }

// W: waves of the workgroup.
template <int RB, int W>
__device__ __forceinline__ void attend4_small(const ChunkArgs& a, const Unit& u, int h, uint8_t* lds) {
  const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const TileAt at = tile_at(a, u.seq, u.row0, u.rows);
  const int fresh = a.b.cu[u.seq + 1] - a.b.cu[u.seq];  // the sequence's new tokens
  // (whole rounds of the waves, so that no wave idles in a part's last one)
  const int64_t rounds = (at.steps + W - 1) / W;
  const int64_t s0 = rounds * u.part / u.parts * W, s1 = min(rounds * (u.part + 1) / u.parts * W, at.steps);
  const uint8_t* pages = a.pages + (int64_t)h * PAGE_Q4_BYTES;
  const int64_t page_stride = (int64_t)a.b.hkv * PAGE_Q4_BYTES;

  uint4 kn[4];  // the next page's K codes
  auto issue = [&](int page, int sb) {
    const uint8_t* p = reinterpret_cast<const uint8_t*>(uniform_ptr(pages + page * page_stride));
    const uint8_t* k = p + (16 * (c >> 2) + (c & 3)) * Q4_ROW + 16 * g;
#pragma unroll
    for (int b = 0; b < 4; ++b) kn[b] = *reinterpret_cast<const uint4*>(k + 4 * b * Q4_ROW);
    const uint32_t slot = __builtin_amdgcn_readfirstlane(lds_addr(lds)) + (2 * wave + sb) * Q4_SLOT;
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // earlier reads of this slot are done
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int row = 16 * e + (lane >> 2);
      dma16(p, (uint32_t)(Q4_CODES + row * Q4_ROW + (((lane & 3) ^ swz4(row)) << 4)), slot + 1024 * e);
    }
    dma16(p, (uint32_t)(2 * Q4_CODES + 16 * lane), slot + Q4_CODES);
  };

  int64_t s = s0 + wave;
  const int mine = s < s1 ? (int)((s1 - s + W - 1) / W) : 0;  // pages of this wave
  Pages pg(a.b, u.seq, s, W, mine);
  half8_t qb[RB][4];  // channels 32 g + 8 k ..
  int tq[RB];         // the token of row c: the last one that it attends
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    const int r = 16 * rb + c, row = u.row0 + r;
    const bool ok = r < at.rows;
    const int tk = ok ? row / a.gq : 0, hd = h * a.gq + (ok ? row % a.gq : 0);
    tq[rb] = tk;
    const uint16_t* qr = a.q + (at.first_token + tk) * a.q_ts + hd * a.q_hs + 32 * g;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      uint4 w = {0, 0, 0, 0};
      if (ok) w = *reinterpret_cast<const uint4*>(qr + 8 * k);
      qb[rb][k] = paired(w);
    }
  }
  int page = pg.at(0);
  if (page >= 0) issue(page, 0);

  const int64_t whole = (at.start + u.row0 / a.gq + 1) / GT;  // steps that every row of the tile sees whole
  Sum4 st[RB];
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) init(st[rb]);

  for (int t = 0; t < mine; ++t, s += W) {
    const int sb = t & 1;
    const bool here = page >= 0;
    uint4 kc[4];
    wait_groups_all();
#pragma unroll
    for (int b = 0; b < 4; ++b) kc[b] = kn[b];
    page = pg.at(t + 1);
    if (page >= 0) issue(page, sb ^ 1);
    if (!here) continue;  // a group without a page takes no part

    uint8_t* slot = lds + (2 * wave + sb) * Q4_SLOT;
    const uint2 ks = *reinterpret_cast<const uint2*>(slot + Q4_CODES + 8 * (4 * c + g));
    float4_t S[RB][4];
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      const half2_t sc = twice(b < 2 ? (b & 1 ? ks.x >> 16 : ks.x & 0xffffu) : (b & 1 ? ks.y >> 16 : ks.y & 0xffffu));
      const half8_t kop[4] = {unpack4(kc[b].x, sc), unpack4(kc[b].y, sc), unpack4(kc[b].z, sc), unpack4(kc[b].w, sc)};
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) {
        float4_t x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < 4; ++k) x = mfma32(kop[k], qb[rb][k], x);
        S[rb][b] = x;
      }
    }
    uint16_t* vsc = reinterpret_cast<uint16_t*>(slot + Q4_CODES + Q4_SCALES);
    if (s >= whole) {
      // Masked places: tokens behind a row's own, and the page's rows behind the sequence's last token, which hold
      // anything. Their weight is 0, but 0 times a V that is not finite is NaN, so such scales become 0; where a row does
      // attend such a token, its score becomes NaN instead. (Positions count from the sequence's first new token: they fit.)
      const int l = tail_tid() & 63, first = (int)(s * GT - at.start);
      bool bad = false;
#pragma unroll
      for (int grp = 0; grp < 4; ++grp) bad |= (vsc[v_scale_at(l, grp)] & 0x7fffu) > Q4_LARGEST;
      if (bad || first + l >= fresh) {
#pragma unroll
        for (int grp = 0; grp < 4; ++grp) vsc[v_scale_at(l, grp)] = 0;
      }
      const uint64_t bads = __builtin_amdgcn_ballot_w64(bad);
      const uint32_t mine16 = (uint32_t)(bads >> (16 * (l >> 4)));
#pragma unroll
      for (int rb = 0; rb < RB; ++rb)
#pragma unroll
        for (int b = 0; b < 4; ++b)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if ((mine16 >> (4 * b + i)) & 1) S[rb][b][i] = __builtin_nanf("");
            if (first + 16 * (l >> 4) + 4 * b + i > tq[rb]) S[rb][b][i] = NEG_INF;
          }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the scales that were cleared, before they are read
    }
    half8_t ph[RB][2];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) weigh(st[rb], S[rb], a.sl2, ph[rb], g);
    const int vrow = 16 * g + c;
    const uint8_t* vp = slot + vrow * Q4_ROW;
#pragma unroll
    for (int grp = 0; grp < 4; ++grp) {
      const uint4* sp = reinterpret_cast<const uint4*>(slot + Q4_CODES + Q4_SCALES + 2 * (grp * GT + 16 * g));
      const uint4 s0w = sp[0], s1w = sp[1];
      const half2_t sv[2][4] = {{as_h2(s0w.x), as_h2(s0w.y), as_h2(s0w.z), as_h2(s0w.w)},
                                {as_h2(s1w.x), as_h2(s1w.y), as_h2(s1w.z), as_h2(s1w.w)}};
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int cb = 2 * grp + e;
        const u32x2 vw = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr4_b64_v2i32(
            (lds_v2i_t*)(const lds_void_t*)(vp + 8 * e + ((grp ^ swz4(vrow)) << 4))));
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          const half8_t vop = unpack4(w ? vw.y : vw.x, sv[w]);
#pragma unroll
          for (int rb = 0; rb < RB; ++rb) st[rb].acc[cb] = mfma32(ph[rb][w], vop, st[rb].acc[cb]);
        }
      }
    }
  }

  // ---- the waves' states into one, row by row
  wait_groups_all();
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    __syncthreads();  // every wave is done with its slots (or with the row block before)
    float* state = reinterpret_cast<float*>(lds) + wave * (16 * CH_PART);
    const float l = sum4rows(st[rb].l);
    if (g == 0) {
      state[c * CH_PART + D] = reference(st[rb]);
      state[c * CH_PART + D + 1] = l;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int cb = 0; cb < 8; ++cb) state[(4 * g + i) * CH_PART + 16 * cb + c] = st[rb].acc[cb][i];
    __syncthreads();
    const int l32 = tid & 31;
#pragma unroll
    for (int p = 0; p < 8 / W; ++p) {
      const int r16 = 2 * W * p + (tid >> 5), r = 16 * rb + r16;
      if (r >= at.rows) continue;
      const float* base = reinterpret_cast<const float*>(lds) + r16 * CH_PART;
      RowSum sum = {NEG_INF, 0.0f, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
      for (int w = 0; w < W; ++w) sum.m = fmaxf(sum.m, base[w * (16 * CH_PART) + D]);
      const float mu = sum.m == NEG_INF ? 0.0f : sum.m;
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const float* x = base + w * (16 * CH_PART);
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
}

constexpr int Q4_SMALL = 4;  // waves of a workgroup in a launch of small units alone
__global__ __launch_bounds__(64 * Q4_SMALL, 2) void attn_q4_small_kernel(ChunkArgs a) {
  __shared__ __attribute__((aligned(16))) uint8_t lds[2 * Q4_SMALL * Q4_SLOT];
  const int h = blockIdx.x % a.b.hkv;
  const Unit u = a.units[blockIdx.x / a.b.hkv];
  if (u.seq < 0 || u.seq >= a.b.nseq || u.row0 < 0 || u.rows <= 0 || u.rows > 32 || u.part < 0 || u.part >= u.parts || u.slot < 0)
    return;
  if (u.rows <= 16) attend4_small<1, Q4_SMALL>(a, u, h, lds);
  else attend4_small<2, Q4_SMALL>(a, u, h, lds);
}

// ---------------------------------------------------------------- host side

int dtype_ok(const char* what, int dtype) {
  return dtype == NKV_F16 || dtype == NKV_BF16 || dtype == NKV_F32 ? NKV_OK : fail(NKV_ERR_INVALID, "%s: unknown dtype %d", what, dtype);
}

unsigned blocks_of(int64_t chunks) { return (unsigned)std::min<int64_t>(cdiv(chunks, 256), 1 << 20); }

template <bool PAGES>
int launch_quant4(const char* what, const Quant4Args& a, int dtype, hipStream_t s) {
  const dim3 grid(blocks_of(a.chunks)), block(256);
  if (dtype == NKV_F16) hipLaunchKernelGGL((quant4_kernel<NKV_F16, PAGES>), grid, block, 0, s, a);
  else if (dtype == NKV_BF16) hipLaunchKernelGGL((quant4_kernel<NKV_BF16, PAGES>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((quant4_kernel<NKV_F32, PAGES>), grid, block, 0, s, a);
  return check_launch(what);
}

}  // namespace

}  // namespace nkv

using namespace nkv;

extern "C" int nkv_quantize_q4(const void* x, int x_dtype, int64_t rows, int64_t n, uint8_t* codes, uint16_t* scales,
                               void* stream) {
  set_error("");
  const char* what = "quantize_q4";
  if (int rc = dtype_ok(what, x_dtype)) return rc;
  if (rows < 0 || n <= 0 || n % Q4_GROUP || (rows && n > (int64_t(1) << 40) / rows))
    return fail(NKV_ERR_INVALID, "%s: sizes rows=%lld n=%lld (n a positive multiple of 32)", what, (long long)rows, (long long)n);
  if (rows == 0) return NKV_OK;
  if (!x || !codes || !scales) return fail(NKV_ERR_INVALID, "%s: null pointer argument", what);
  if (!al16(x) || !al16(codes)) return fail(NKV_ERR_UNSUPPORTED, "%s: x and codes must be 16-byte aligned", what);
  Quant4Args a{};
  a.x = static_cast<const uint8_t*>(x);
  a.chunks = rows * (n / 8);
  a.codes = codes;
  a.scales = scales;
  return launch_quant4<false>(what, a, x_dtype, static_cast<hipStream_t>(stream));
}

extern "C" int nkv_dequantize_q4(const uint8_t* codes, const uint16_t* scales, int64_t rows, int64_t n, void* out,
                                 int out_dtype, void* stream) {
  set_error("");
  const char* what = "dequantize_q4";
  if (int rc = dtype_ok(what, out_dtype)) return rc;
  if (rows < 0 || n <= 0 || n % Q4_GROUP || (rows && n > (int64_t(1) << 40) / rows))
    return fail(NKV_ERR_INVALID, "%s: sizes rows=%lld n=%lld (n a positive multiple of 32)", what, (long long)rows, (long long)n);
  if (rows == 0) return NKV_OK;
  if (!codes || !scales || !out) return fail(NKV_ERR_INVALID, "%s: null pointer argument", what);
  if (!al16(codes) || !al16(out)) return fail(NKV_ERR_UNSUPPORTED, "%s: codes and out must be 16-byte aligned", what);
  const int64_t chunks = rows * (n / 8);
  const dim3 grid(blocks_of(chunks)), block(256);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const uint32_t* words = reinterpret_cast<const uint32_t*>(codes);
  uint8_t* to = static_cast<uint8_t*>(out);
  if (out_dtype == NKV_F16) hipLaunchKernelGGL(dequant4_kernel<NKV_F16>, grid, block, 0, s, words, scales, chunks, to);
  else if (out_dtype == NKV_BF16) hipLaunchKernelGGL(dequant4_kernel<NKV_BF16>, grid, block, 0, s, words, scales, chunks, to);
  else hipLaunchKernelGGL(dequant4_kernel<NKV_F32>, grid, block, 0, s, words, scales, chunks, to);
  return check_launch(what);
}

extern "C" int nkv_paged_quantize_q4(const void* x, int x_dtype, int64_t x_head_stride, int64_t hkv, int64_t n, int which,
                                     uint8_t* pages, const int32_t* table_row, int64_t first_token, int64_t num_pages,
                                     void* stream) {
  set_error("");
  const char* what = "paged_quantize_q4";
  if (int rc = dtype_ok(what, x_dtype)) return rc;
  if (hkv <= 0 || hkv > 1024 || n < 0 || n > (int64_t(1) << 31) || first_token < 0 || (which != 0 && which != 1) || num_pages <= 0)
    return fail(NKV_ERR_INVALID, "%s: bad sizes hkv=%lld n=%lld first_token=%lld which=%d num_pages=%lld", what, (long long)hkv,
                (long long)n, (long long)first_token, which, (long long)num_pages);
  if (n == 0) return NKV_OK;
  if (!x || !pages || !table_row) return fail(NKV_ERR_INVALID, "%s: null pointer argument", what);
  if (!al16(x) || !al16(pages) || x_head_stride % 8 || x_head_stride < n * D)
    return fail(NKV_ERR_UNSUPPORTED, "%s: x and pages must be 16-byte aligned, the head stride a multiple of 8 and >= n * 128", what);
  Quant4Args a{};
  a.x = static_cast<const uint8_t*>(x);
  a.head_stride = x_head_stride;
  a.chunks = hkv * n * (D / 8);
  a.pages = pages;
  a.table = table_row;
  a.n = n; a.hkv = hkv; a.first = first_token; a.num_pages = num_pages; a.which = which;
  return launch_quant4<true>(what, a, x_dtype, static_cast<hipStream_t>(stream));
}

extern "C" int nkv_paged_attn_chunks_q4(const uint16_t* q, int64_t q_token_stride, int64_t q_head_stride, int64_t tokens,
                                        const uint8_t* pages, const int32_t* page_table, int64_t table_stride,
                                        int64_t num_pages, const int32_t* cu, const int64_t* start_dev, int64_t nseq,
                                        int64_t hq, int64_t hkv, int64_t head_dim, const int32_t* units, int64_t n_units, int wide,
                                        const int32_t* merges, int64_t n_merges, uint16_t* out, int64_t out_token_stride,
                                        int64_t out_head_stride, float* lse_out, void* workspace, int64_t workspace_bytes,
                                        void* stream) {
  const char* what = "paged_attn_chunks_q4";
  ChunkArgs a{};
  bool any = false;
  if (int rc = chunk_args(what, a, any, q, q_token_stride, q_head_stride, tokens, pages, page_table, table_stride, num_pages, cu,
                          start_dev, nseq, hq, hkv, head_dim, units, n_units, merges, n_merges, out, out_token_stride,
                          out_head_stride, lse_out, workspace, workspace_bytes))
    return rc;
  if (!any) return NKV_OK;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const dim3 grid((unsigned)(n_units * hkv));
  hipLaunchKernelGGL(attn_q4_small_kernel, grid, dim3(64 * Q4_SMALL), 0, s, a);
  if (int rc = check_launch(what)) return rc;
  return launch_merges(what, a, reinterpret_cast<const Merge*>(merges), n_merges, s);
}
