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
  int64_t head_stride;  // elements from head to head
  int64_t chunks;       // of eight values, all rows'
  // row r of head h is token first + r of a sequence, of tensor `which`; tokens whose table entry is outside
  // [0, num_pages) are skipped
  uint8_t* pages;
  const int32_t* table;
  int64_t n, hkv, first, num_pages;
  int which;
};

// A prompt's keys or values into their pages: eight values a lane, a group to four lanes; bound by memory.
template <int DT>
__global__ __launch_bounds__(256) void quant4_pages_kernel(Quant4Args a) {
  const int64_t step = (int64_t)gridDim.x * 256;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < a.chunks; i += step) {  // (16 lanes agree)
    Raw8<DT> r;
    float v[8];
    uint16_t scale;
    const int64_t row = i >> 4, h = row / a.n, t = row % a.n, tok = a.first + t;
    const int j = (int)(i & 15), slot = (int)(tok % GT);
    r.load(a.x + (h * a.head_stride + t * D + 8 * j) * Elem<DT>::SIZE);
    const int32_t page = a.table[tok / GT];
    r.get(v);
    const uint32_t w = q4_quant8(v, scale);
    if (page < 0 || page >= a.num_pages) continue;
    uint8_t* p = a.pages + ((int64_t)page * a.hkv + h) * PAGE_Q4_BYTES;
    *reinterpret_cast<uint32_t*>(p + a.which * Q4_CODES + slot * Q4_ROW + 4 * word_at(a.which, j)) = w;
    const int to = a.which ? v_scale_at(slot, j / 4) : k_scale_at(slot, j / 4);
    if (j % 4 == 0) *reinterpret_cast<uint16_t*>(p + 2 * Q4_CODES + a.which * Q4_SCALES + 2 * to) = scale;
  }
}

// A weight [rows][n] into blocks: a workgroup takes one, four lanes a row's group of 32, four groups a lane.
template <int DT>
__global__ __launch_bounds__(64) void quant4_weight_kernel(const uint8_t* x, int64_t rows, int64_t n, uint8_t* out) {
  const int64_t nb = (n + W4_COLS - 1) / W4_COLS, kb = blockIdx.x % nb, tile = blockIdx.x / nb;
  const int lane = threadIdx.x, c = lane >> 2, k = lane & 3;
  const int64_t row = tile * W4_ROWS + c;
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const int64_t col = kb * W4_COLS + 32 * g + 8 * k;
    const bool in = row < rows && col < n;  // (four lanes agree)
    Raw8<DT> r;
    float v[8];
    uint16_t scale;
    r.zero();
    if (in) r.load(x + (row * n + col) * Elem<DT>::SIZE);
    r.get(v);
    const uint32_t w = q4_quant8<true>(v, scale);
    uint8_t* to = out + w4_at(row, nb, kb, g);
    *reinterpret_cast<uint32_t*>(to + 4 * k) = w;
    if (k == 0) *reinterpret_cast<uint16_t*>(to + w4_scale_from(c + 16 * g)) = in ? scale : (uint16_t)0;
  }
}

template <int DT>
__global__ __launch_bounds__(64) void dequant4_weight_kernel(const uint8_t* w4, int64_t rows, int64_t n, uint8_t* out) {
  const int64_t nb = (n + W4_COLS - 1) / W4_COLS, kb = blockIdx.x % nb, tile = blockIdx.x / nb;
  const int lane = threadIdx.x, c = lane >> 2, k = lane & 3;
  const int64_t row = tile * W4_ROWS + c;
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const int64_t col = kb * W4_COLS + 32 * g + 8 * k;
    if (row >= rows || col >= n) continue;
    const uint8_t* at = w4 + w4_at(row, nb, kb, g);
    const uint32_t w = *reinterpret_cast<const uint32_t*>(at + 4 * k);
    const float s = h2f(*reinterpret_cast<const uint16_t*>(at + w4_scale_from(c + 16 * g)));
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = q4_value(w, e / 2 + 4 * (e % 2), s);
    store8<DT, false>(out + (row * n + col) * Elem<DT>::SIZE, v);
  }
}

// ---------------------------------------------------------------- attention
//
// softmax(q K^T / sqrt(128)) V. K and V are exact fp16 operands (nkv_q4.h); what is rounded to fp16 is the softmax's weights
// and the output. The units of up to 32 rows ("small"): a workgroup's waves take the part's pages in turn, each its own
// page against all the rows, and their states are merged in LDS at the end. K's codes go from memory to registers: lane
// c + 16 g of tile b takes 16 bytes of token 16 (c / 4) + 4 b + c % 4, channels 32 j + 8 g .. + 7 of each group j. A product
// is of one group's 32 channels, so that the scale multiplies its results and the codes need no arithmetic (tiny4; the
// offset's share, -8 2^-24 sum(q), starts the sum): 5 instructions for 8 codes instead of 17 and a scale.
// V's codes and the scales go to LDS, where the transposing read gives lane c + 16 g channel 16 cb + c of tokens 16 g ..
// + 15: those that its scores are of.
//
// Measured (32 query and 8 KV heads): 64 sequences of one token over 2000, 151 MB in 31 us; 32 over 64 to 8155 35 us with the
// second launch: 610 vector instructions a page and wave, which is about half of that, and memory's 22 us, neither of
// them alone. Pages that one unit reads alone are loaded past the caches (37 to 31 us).

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

// 16 bytes of global memory, named as such: a flat load shares LDS's counter, and every wait for LDS would be one for it.
__device__ __forceinline__ uint4 load_global16(const uint8_t* p, bool once) {
  const auto* from = reinterpret_cast<const __attribute__((address_space(1))) u32x4_t*>(reinterpret_cast<uintptr_t>(p));
  const u32x4_t v = once ? __builtin_nontemporal_load(from) : *from;
  return uint4{v.x, v.y, v.z, v.w};
}

// n part / parts, without the 64-bit division that it looks like (parts: 2^15 at most).
__device__ __forceinline__ int cut_at(int n, int part, int parts) {
  return n / parts * part + n % parts * part / parts;
}

// W: waves of the workgroup.
template <int RB, int W>
__device__ __forceinline__ void attend4_small(const ChunkArgs& a, const Unit& u, int h, uint8_t* lds) {
  const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const TileAt at = tile_at(a, u.seq, u.row0, u.rows);
  const int fresh = a.b.cu[u.seq + 1] - a.b.cu[u.seq];  // the sequence's new tokens
  // (whole rounds of the waves, so that no wave idles in a part's last one)
  const int rounds = (int)((at.steps + W - 1) / W);
  const int64_t s0 = (int64_t)cut_at(rounds, u.part, u.parts) * W, s1 = min((int64_t)cut_at(rounds, u.part + 1, u.parts) * W, at.steps);
  const uint8_t* pages = a.pages + (int64_t)h * PAGE_Q4_BYTES;
  const int64_t page_stride = (int64_t)a.b.hkv * PAGE_Q4_BYTES;

  uint4 kn[4];  // the next page's K codes
  // (a group without a page: any page's bytes, all of them masked)
  auto issue = [&](int page, int sb) {
    page = max(page, 0);
    const int lane = tail_tid() & 63;  // (opaque: the offsets are made again at each use, for want of registers)
    const uint8_t* p = reinterpret_cast<const uint8_t*>(uniform_ptr(pages + page * page_stride));
    const uint32_t k = (uint32_t)((16 * ((lane >> 2) & 3) + (lane & 3)) * Q4_ROW + 16 * (lane >> 4));
#pragma unroll
    for (int b = 0; b < 4; ++b) kn[b] = load_global16(p + (k + 4 * b * Q4_ROW), u.alone);
    const uint32_t slot = __builtin_amdgcn_readfirstlane(lds_addr(lds)) + (2 * wave + sb) * Q4_SLOT;
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // earlier reads of this slot are done
    const uint32_t v = (uint32_t)(Q4_CODES + (lane >> 2) * Q4_ROW + (((lane & 3) ^ swz4(lane >> 2)) << 4));
#pragma unroll
    for (int e = 0; e < 4; ++e) {  // (rows 16 e + lane / 4: the key is theirs)
      if (u.alone) dma16_stream(p, v + 1024 * e, slot + 1024 * e);
      else dma16(p, v + 1024 * e, slot + 1024 * e);
    }
    if (u.alone) dma16_stream(p, (uint32_t)(2 * Q4_CODES + 16 * lane), slot + Q4_CODES);
    else dma16(p, (uint32_t)(2 * Q4_CODES + 16 * lane), slot + Q4_CODES);
  };

  int64_t s = s0 + wave;
  const int mine = s < s1 ? (int)((s1 - s + W - 1) / W) : 0;  // pages of this wave
  Pages pg(a.b, u.seq, s, W, mine);
  half8_t qb[RB][4];  // channels 32 k + 8 g ..; the pairs that meet 16 n are held over 16, all times a power of two
  float4_t start[RB][4];  // the offset's share of group k
  float sl2[RB];       // what turns row c's sums into scores (log2 domain)
  int tq[RB];          // the token of row c: the last one that it attends
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    const int r = 16 * rb + c, row = u.row0 + r;
    const bool ok = r < at.rows;
    const int tk = ok ? row / a.gq : 0, hd = h * a.gq + (ok ? row % a.gq : 0);
    tq[rb] = tk;
    const uint16_t* qr = a.q + (at.first_token + tk) * a.q_ts + hd * a.q_hs + 8 * g;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      uint4 w = {0, 0, 0, 0};
      if (ok) w = *reinterpret_cast<const uint4*>(qr + 32 * k);
      qb[rb][k] = paired(w);
    }
  }
  int page = pg.at(0);
  if (mine > 0) issue(page, 0);
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    // (the row's largest comes to 2^14, so that over 16 what is lost is 2^-35 of it, at most; not finite: as it is)
    float top = 0.0f;
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int e = 0; e < 8; ++e) top = fmaxf(top, __builtin_fabsf((float)qb[rb][k][e]));
    top = max4rows(top);
    const int up = top > 0.0f && top < 65536.0f ? 127 + 14 - (int)(__float_as_uint(top) >> 23) : 0;
    const float by = __uint_as_float((uint32_t)(127 + up) << 23);
    sl2[rb] = a.sl2 * 0x1p24f * __uint_as_float((uint32_t)(127 - up) << 23);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      float sum = 0.0f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float f = e & 2 ? 0.0625f : 1.0f;  // (pairs of two)
        qb[rb][k][e] = (_Float16)((float)qb[rb][k][e] * (by * f));
        sum = __builtin_fmaf((float)qb[rb][k][e], 1.0f / f, sum);
      }
      sum = sum4rows(sum) * (-8.0f * 0x1p-24f);
      start[rb][k] = float4_t{sum, sum, sum, sum};
    }
  }

  const int64_t whole = (at.start + u.row0 / a.gq + 1) / GT;  // steps that every row of the tile sees whole
  Sum4 st[RB];
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) init(st[rb]);
  const uint32_t bias = bias1024();

  for (int t = 0; t < mine; ++t, s += W) {
    const int sb = t & 1;
    const bool here = page >= 0;  // a group without a page takes no part
    wait_groups_all();
    uint4 kc[4];
#pragma unroll
    for (int b = 0; b < 4; ++b) kc[b] = kn[b];
    page = pg.at(t + 1);
    if (t + 1 < mine) issue(page, sb ^ 1);  // (a whole step ahead: 64 x 2000 tokens 36 us; issued after K's products 45)

    uint8_t* slot = lds + (2 * wave + sb) * Q4_SLOT;
    const uint8_t* ksc = slot + Q4_CODES + 32 * (tail_tid() >> 4 & 3);
    float4_t S[RB][4];
    uint2 ks[2][4];  // of tokens 16 g + 4 b .. + 3, group k; the next tile's on the way
    auto load_ks = [&](int b) {
#pragma unroll
      for (int k = 0; k < 4; ++k) ks[b & 1][k] = *reinterpret_cast<const uint2*>(ksc + 2 * GT * k + 8 * b);
    };
    load_ks(0);
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      // (a tile after the other, for want of registers: what is opaque stays in order)
      asm volatile("" : "+v"(kc[b].x), "+v"(kc[b].y), "+v"(kc[b].z), "+v"(kc[b].w));
      if (b < 3) load_ks(b + 1);
      const uint32_t words[4] = {kc[b].x, kc[b].y, kc[b].z, kc[b].w};
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) S[rb][b] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const half8_t kop = tiny4(words[k]);
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
          const float4_t d = mfma32(kop, qb[rb][k], start[rb][k]);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const half2_t h = as_h2(i < 2 ? ks[b & 1][k].x : ks[b & 1][k].y);
            S[rb][b][i] = __builtin_fmaf((float)(i & 1 ? h.y : h.x), d[i], S[rb][b][i]);
          }
        }
      }
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) asm volatile("" : "+v"(S[rb][b]));
    }
    uint16_t* vsc = reinterpret_cast<uint16_t*>(slot + Q4_CODES + Q4_SCALES);
    if (s >= whole || !here) {
      // Masked places: tokens behind a row's own, and the page's rows behind the sequence's last token, which hold
      // anything. Their weight is 0, but 0 times a V that is not finite is NaN, so such scales become 0; where a row does
      // attend such a token, its score becomes NaN instead. (Positions count from the sequence's first new token: they fit.)
      const int l = tail_tid() & 63, first = here ? (int)(s * GT - at.start) : 1 << 30;
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
    for (int rb = 0; rb < RB; ++rb) weigh(st[rb], S[rb], sl2[rb], ph[rb], g);
    const int vl = tail_tid() & 63;
    const uint8_t* vp = slot + vl * Q4_ROW;  // (row 16 g + c)
#pragma unroll
    for (int grp = 0; grp < 4; ++grp) {
      asm volatile("" : "+v"(vp));  // (as above)
      const uint4* sp = reinterpret_cast<const uint4*>(slot + Q4_CODES + Q4_SCALES + 2 * (grp * GT + 16 * (vl >> 4)));
      const uint4 s0w = sp[0], s1w = sp[1];
      const half2_t sv[2][4] = {{as_h2(s0w.x), as_h2(s0w.y), as_h2(s0w.z), as_h2(s0w.w)},
                                {as_h2(s1w.x), as_h2(s1w.y), as_h2(s1w.z), as_h2(s1w.w)}};
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int cb = 2 * grp + e;
        const u32x2 vw = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr4_b64_v2i32(
            (lds_v2i_t*)(const lds_void_t*)(vp + 8 * e + ((grp ^ swz4(vl)) << 4))));
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          const half8_t vop = unpack4(w ? vw.y : vw.x, sv[w], bias);
#pragma unroll
          for (int rb = 0; rb < RB; ++rb) st[rb].acc[cb] = mfma32(ph[rb][w], vop, st[rb].acc[cb]);
        }
      }
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) asm volatile("" : "+v"(st[rb].acc[2 * grp]), "+v"(st[rb].acc[2 * grp + 1]));
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
    for (int p = 0; p < (8 + W - 1) / W; ++p) {
      const int r16 = 2 * W * p + (tid >> 5), r = 16 * rb + r16;
      if (r16 >= 16 || r >= at.rows) continue;
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

// Units of up to 256 rows ("wide"): wave w takes rows 32 w .. 32 w + 31 as two row blocks, and every wave every page. A page's
// codes come to one of three stages in LDS; its operands are made once for all waves, a sixteenth of K's and of V's by each, and
// laid out as the products take them, 16 bytes a lane: tile t & 1 while the other one is read. One barrier a step: in step
// t, before it, the conversion of page t + 1 into the tile that step t - 1 read and the wait for the loads of page t + 2;
// after it the loads of page t + 4 into the stage of page t + 1. A step is 64 matrix and 206 vector instructions a wave, 1.85
// us: 2048 tokens over 14336 487 us, 1060 TFLOP/s (made by each wave for itself, the operands took 784 us); a unit's start and end
// are 10 us, of which the chain unit - page ids - first page - operands is 4.
constexpr int WD_RB = 2, WD_ROWS = Q4_WAVES * WD_RB * 16, WD_STAGES = 3;
constexpr int WD_TILE = GT * D * 2;                   // an operand tile: [16][64 lanes][16 bytes]
constexpr int WD_VT = 2 * WD_TILE, WD_ST = 4 * WD_TILE;  // K tiles, V tiles, stages
constexpr int WD_LDS = WD_ST + WD_STAGES * PAGE_Q4_BYTES;
static_assert(WD_ROWS * D * 2 <= WD_LDS && 2 * Q4_WAVES * Q4_SLOT <= WD_LDS, "the output of a tile, and the small units, fit");

__device__ __forceinline__ void attend4_wide(const ChunkArgs& a, const Unit& u, int h, uint8_t* lds) {
  const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const TileAt at = tile_at(a, u.seq, u.row0, u.rows);
  const int s0 = cut_at((int)at.steps, u.part, u.parts), n = cut_at((int)at.steps, u.part + 1, u.parts) - s0;
  const int64_t len = at.start + (a.b.cu[u.seq + 1] - a.b.cu[u.seq]);
  const uint8_t* pages = a.pages + (int64_t)h * PAGE_Q4_BYTES;
  const int64_t page_stride = (int64_t)a.b.hkv * PAGE_Q4_BYTES;
  const uint32_t stages = __builtin_amdgcn_readfirstlane(lds_addr(lds)) + WD_ST;
  Pages pg(a.b, u.seq, s0, 1, n);
  // wave w's loads of a page: 16 rows of K's (0 .. 3) or V's codes, wave 0 the scales, too. The 16-byte chunks of a row are
  // moved by a key, so that the conversion's reads fall on different banks: K's by row / 16, V's by row / 4.
  int loads = 0;  // in flight of the newest page
  auto issue = [&](int page, int slot) {
    loads = 0;
    if (page < 0) return;
    loads = wave == 0 ? 2 : 1;
    const void* p = uniform_ptr(pages + page * page_stride);
    const uint32_t dst = stages + slot * PAGE_Q4_BYTES;
    const int key = wave < 4 ? wave : lane >> 4;
    dma16(p, (uint32_t)(1024 * wave + (lane >> 2) * Q4_ROW + (((lane & 3) ^ key) << 4)), dst + 1024 * wave);
    if (wave == 0) dma16(p, (uint32_t)(2 * Q4_CODES + 16 * lane), dst + 2 * Q4_CODES);
  };
  // steps that some row of the tile does not see whole: masked places may hold anything there (attend4_small)
  const int tile_whole = (int)((at.start + u.row0 / a.gq + 1) / GT) - s0;
  // Page t from its stage into its tiles; with the rules for masked places where `check` (a token whose V is not finite
  // gets a K that is not). Wave w: K's tile b = w / 2, groups 2 (w % 2) and the next; V's channels 16 w .. + 15.
  const uint32_t bias = bias1024();
  auto convert = [&](int t, int slot, auto check) {
    const uint8_t* sg = lds + WD_ST + slot * PAGE_Q4_BYTES;
    const int lane = tail_tid() & 63, c = lane & 15, g = lane >> 4, b = wave >> 1;
    const int krow = 16 * (c >> 2) + 4 * b + (c & 3), vrow = 16 * g + c;
    const uint2 kw = *reinterpret_cast<const uint2*>(sg + krow * Q4_ROW + ((g ^ (c >> 2)) << 4) + 8 * (wave & 1));
    const u32x2 vw = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr4_b64_v2i32(
        (lds_v2i_t*)(const lds_void_t*)(sg + Q4_CODES + vrow * Q4_ROW + 8 * (wave & 1) + (((wave >> 1) ^ (c >> 2)) << 4))));
    const uint16_t* sc = reinterpret_cast<const uint16_t*>(sg + 2 * Q4_CODES);
    uint32_t k0 = sc[2 * (wave & 1) * GT + krow], k1 = sc[(2 * (wave & 1) + 1) * GT + krow];
    const uint4* vp = reinterpret_cast<const uint4*>(sc + Q4_SCALES / 2 + (wave >> 1) * GT + 16 * g);
    const uint4 v0 = vp[0], v1 = vp[1];
    uint32_t vs[8] = {v0.x, v0.y, v0.z, v0.w, v1.x, v1.y, v1.z, v1.w};
    if constexpr (decltype(check)::value) {
#pragma unroll
      for (int grp = 0; grp < 4; ++grp)
        if ((sc[Q4_SCALES / 2 + v_scale_at(krow, grp)] & 0x7fffu) > Q4_LARGEST) k0 = k1 = 0x7e00u;
      const int left = (int)min<int64_t>(GT, len - (int64_t)(s0 + t) * GT);  // tokens that the page has
#pragma unroll
      for (int e = 0; e < 8; ++e) {  // the pair of tokens 16 g + 8 (e / 4) + e % 4 and 4 further
        const int tok = 16 * g + 8 * (e >> 2) + (e & 3);
        if ((vs[e] & 0x7fffu) > Q4_LARGEST || tok >= left) vs[e] &= 0xffff0000u;
        if (((vs[e] >> 16) & 0x7fffu) > Q4_LARGEST || tok + 4 >= left) vs[e] &= 0xffffu;
      }
    }
    const half2_t va[4] = {as_h2(vs[0]), as_h2(vs[1]), as_h2(vs[2]), as_h2(vs[3])};
    const half2_t vb[4] = {as_h2(vs[4]), as_h2(vs[5]), as_h2(vs[6]), as_h2(vs[7])};
    uint8_t* kt = lds + (t & 1) * WD_TILE + 16 * lane + 2048 * wave;  // (operand 4 b + k of wave 2 b + k / 2)
    uint8_t* vt = lds + WD_VT + (t & 1) * WD_TILE + 16 * lane + 1024 * wave;
    *reinterpret_cast<half8_t*>(kt) = unpack4(kw.x, twice(k0), bias);
    *reinterpret_cast<half8_t*>(kt + 1024) = unpack4(kw.y, twice(k1), bias);
    *reinterpret_cast<half8_t*>(vt) = unpack4(vw.x, va, bias);
    *reinterpret_cast<half8_t*>(vt + 8192) = unpack4(vw.y, vb, bias);
  };

  int p0 = pg.at(0), p1 = pg.at(1), p2 = pg.at(2), p3 = pg.at(3);  // the pages of steps t .. t + 3
  issue(p0, 0);
  issue(p1, 1);
  const int row0 = u.row0 + wave * (WD_RB * 16);  // first row of this wave
  const int rows = u.row0 + at.rows;
  half8_t qb[WD_RB][4];
#pragma unroll
  for (int rb = 0; rb < WD_RB; ++rb) {
    const int row = row0 + 16 * rb + c;
    const bool ok = row < rows;
    const int tk = ok ? row / a.gq : 0, hd = h * a.gq + (ok ? row % a.gq : 0);
    const uint16_t* qr = a.q + (at.first_token + tk) * a.q_ts + hd * a.q_hs + 8 * g;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      uint4 w = {0, 0, 0, 0};
      if (ok) w = *reinterpret_cast<const uint4*>(qr + 32 * k);
      qb[rb][k] = paired(w);
    }
  }
  Sum4 st[WD_RB];
#pragma unroll
  for (int rb = 0; rb < WD_RB; ++rb) init(st[rb]);
  // this wave's rows attend steps t < mine
  const int last = min(row0 + WD_RB * 16, rows) - 1;
  const int mine = row0 < rows ? min(n, (int)((at.start + last / a.gq) / GT) + 1 - s0) : 0;

  half8_t op[16];  // the operands of the products: K's, then V's
  const uint8_t* tile = lds + 16 * lane;
  auto load_k = [&](int t) {
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int b = 0; b < 4; ++b) op[4 * k + b] = *reinterpret_cast<const half8_t*>(tile + (t & 1) * WD_TILE + 1024 * (4 * b + k));
  };
  auto load_v = [&](int t) {
#pragma unroll
    for (int e = 0; e < 16; ++e) op[e] = *reinterpret_cast<const half8_t*>(tile + (t & 1) * WD_TILE + WD_VT + 1024 * e);
  };
  float4_t S[WD_RB][4];
  half8_t ph[WD_RB][2];
  auto qk = [&](int rb) {
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int b = 0; b < 4; ++b)
        S[rb][b] = mfma32(op[4 * k + b], qb[rb][k], k ? S[rb][b] : float4_t{0.f, 0.f, 0.f, 0.f});
  };
  auto softmax = [&](int rb, auto masked, int t) {
    const int l = tail_tid() & 63;
    if constexpr (decltype(masked)::value) {
      const int tok0 = (int)((int64_t)(s0 + t) * GT - at.start) + 16 * (l >> 4);  // (near the sequence's end, it fits)
      const int tq = (row0 + 16 * rb + (l & 15)) / a.gq;
#pragma unroll
      for (int b = 0; b < 4; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (tok0 + 4 * b + i > tq) S[rb][b][i] = NEG_INF;
    }
    weigh(st[rb], S[rb], a.sl2, ph[rb], l >> 4);
  };
  auto pv = [&](int rb) {
#pragma unroll
    for (int w = 0; w < 2; ++w)
#pragma unroll
      for (int cb = 0; cb < 8; ++cb) st[rb].acc[cb] = mfma32(ph[rb][w], op[8 * w + cb], st[rb].acc[cb]);
  };

  wait_groups_all();
  __syncthreads();
  if (n > 0) convert(0, 0, std::true_type{});
  __syncthreads();
  issue(p2, 2);
  issue(p3, 0);
  int r1 = 1;  // (t + 1) mod 3

  // One step. `fast`: every row sees pages t and t + 1 whole, and both are there.
  auto step = [&](int t, auto fast_) {
    constexpr bool fast = decltype(fast_)::value;
    using masked = std::integral_constant<bool, !fast>;
    const int p4 = pg.at(t + 4);
    const bool go = fast || (t < mine && p0 >= 0);
    if (go) {
      load_k(t);
      qk(0);
      qk(1);
      softmax(0, masked{}, t);
      load_v(t);
      pv(0);
      softmax(1, masked{}, t);
    }
    if constexpr (fast) convert(t + 1, r1, std::false_type{});
    else if (t + 1 < n) convert(t + 1, r1, std::true_type{});
    if (go) pv(1);
    // tile t + 1 is written, tile t is read, page t + 2 has landed
    if (loads == 1) asm volatile("s_waitcnt vmcnt(1) lgkmcnt(0)" ::: "memory");
    else if (loads == 2) asm volatile("s_waitcnt vmcnt(2) lgkmcnt(0)" ::: "memory");
    else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    asm volatile("s_barrier" ::: "memory");
    issue(p4, r1);
    r1 = r1 == 2 ? 0 : r1 + 1;
    p0 = p1; p1 = p2; p2 = p3; p3 = p4;
  };
  int t = 0;
  for (; t + 1 < min(n, tile_whole) && p0 >= 0 && p1 >= 0; ++t) step(t, std::true_type{});
  for (; t < n; ++t) step(t, std::false_type{});
  wait_groups_all();
  float rl[WD_RB];  // row c's sum of weights
#pragma unroll
  for (int rb = 0; rb < WD_RB; ++rb) rl[rb] = sum4rows(st[rb].l);

  if (u.parts == 1) {
    // out = the sum of V / l, through LDS so that 16 lanes store a row's 256 bytes (the 2-byte values at chunk ^ 2 ((row >> 2) & 3))
    __syncthreads();  // every wave is past its last read of the tiles
    const int lane = tail_tid() & 63, c = lane & 15, g = lane >> 4;
    uint8_t* ow = lds + wave * (WD_RB * 16 * D * 2);
#pragma unroll
    for (int rb = 0; rb < WD_RB; ++rb)
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
    for (int k = 0; k < WD_RB * 4; ++k) {
      const int r = 4 * k + g, row = row0 + r;
      const uint4 v = *reinterpret_cast<const uint4*>(ow + r * (2 * D) + ((c ^ (((r >> 2) & 3) << 1)) << 4));
      if (row < rows)
        *reinterpret_cast<uint4*>(a.out + (at.first_token + row / a.gq) * a.o_ts + (h * a.gq + row % a.gq) * a.o_hs + 8 * c) = v;
    }
  } else {
    const int64_t pr0 = (int64_t)u.slot + (int64_t)u.part * u.rows + wave * (WD_RB * 16);
#pragma unroll
    for (int rb = 0; rb < WD_RB; ++rb) {
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

__device__ __forceinline__ bool unit_ok(const ChunkArgs& a, const Unit& u, int most) {
  return u.seq >= 0 && u.seq < a.b.nseq && u.row0 >= 0 && u.rows > 0 && u.rows <= most && u.part >= 0 && u.part < u.parts &&
         u.parts <= (1 << 15) && u.slot >= 0;
}

__global__ __launch_bounds__(Q4_THREADS, 1) void attn_q4_kernel(ChunkArgs a) {
  __shared__ __attribute__((aligned(16))) uint8_t lds[WD_LDS];
  const int h = blockIdx.x % a.b.hkv;
  const Unit u = a.units[blockIdx.x / a.b.hkv];
  if (!unit_ok(a, u, u.kind == ROWS256 ? WD_ROWS : 32)) return;
  if (u.kind == ROWS256) attend4_wide(a, u, h, lds);
  else if (u.rows <= 16) attend4_small<1, Q4_WAVES>(a, u, h, lds);
  else attend4_small<2, Q4_WAVES>(a, u, h, lds);
}

constexpr int Q4_SMALL = 4;  // waves of a workgroup in a launch of small units alone
template <int RB>
__global__ __launch_bounds__(64 * Q4_SMALL, RB == 1 ? 3 : 2) void attn_q4_small_kernel(ChunkArgs a) {
  __shared__ __attribute__((aligned(16))) uint8_t lds[2 * Q4_SMALL * Q4_SLOT];
  const int h = blockIdx.x % a.b.hkv;
  const Unit u = a.units[blockIdx.x / a.b.hkv];
  if (!unit_ok(a, u, 16 * RB)) return;
  if (RB == 1 || u.rows <= 16) attend4_small<1, Q4_SMALL>(a, u, h, lds);
  else attend4_small<RB, Q4_SMALL>(a, u, h, lds);
}

// ---------------------------------------------------------------- host side

int dtype_ok(const char* what, int dtype) {
  return dtype == NKV_F16 || dtype == NKV_BF16 || dtype == NKV_F32 ? NKV_OK : fail(NKV_ERR_INVALID, "%s: unknown dtype %d", what, dtype);
}

// The arguments of the weights' quantizers, and the blocks of a launch.
int weight_args(const char* what, const void* x, int dtype, int64_t rows, int64_t n, const void* w4, int64_t& blocks) {
  set_error("");
  blocks = 0;
  if (int rc = dtype_ok(what, dtype)) return rc;
  if (rows < 0 || n <= 0 || n % Q4_GROUP || rows >= (int64_t(1) << 40) || n >= (int64_t(1) << 40))
    return fail(NKV_ERR_INVALID, "%s: sizes rows=%lld n=%lld (n a positive multiple of 32)", what, (long long)rows, (long long)n);
  const int64_t tiles = cdiv(rows, W4_ROWS), nb = cdiv(n, W4_COLS);
  if (tiles && nb > ((int64_t(1) << 26) - 1) / tiles)  // (a launch has less than 2^32 threads)
    return fail(NKV_ERR_INVALID, "%s: rows=%lld n=%lld: more than 2^37 values", what, (long long)rows, (long long)n);
  if (rows == 0) return NKV_OK;
  if (!x || !w4) return fail(NKV_ERR_INVALID, "%s: null pointer argument", what);
  if (!al16(x) || !al16(w4)) return fail(NKV_ERR_UNSUPPORTED, "%s: buffers must be 16-byte aligned", what);
  blocks = tiles * nb;
  return NKV_OK;
}

}  // namespace

}  // namespace nkv

using namespace nkv;

extern "C" int64_t nkv_q4_weight_bytes(int64_t rows, int64_t n) {
  return rows > 0 && n > 0 ? cdiv(rows, W4_ROWS) * cdiv(n, W4_COLS) * W4_BLOCK : 0;
}

extern "C" int nkv_quantize_q4(const void* x, int x_dtype, int64_t rows, int64_t n, uint8_t* w4, void* stream) {
  int64_t blocks;
  if (int rc = weight_args("quantize_q4", x, x_dtype, rows, n, w4, blocks)) return rc;
  if (!blocks) return NKV_OK;
  const dim3 grid((unsigned)blocks), block(64);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const uint8_t* from = static_cast<const uint8_t*>(x);
  if (x_dtype == NKV_F16) hipLaunchKernelGGL(quant4_weight_kernel<NKV_F16>, grid, block, 0, s, from, rows, n, w4);
  else if (x_dtype == NKV_BF16) hipLaunchKernelGGL(quant4_weight_kernel<NKV_BF16>, grid, block, 0, s, from, rows, n, w4);
  else hipLaunchKernelGGL(quant4_weight_kernel<NKV_F32>, grid, block, 0, s, from, rows, n, w4);
  return check_launch("quantize_q4");
}

extern "C" int nkv_dequantize_q4(const uint8_t* w4, int64_t rows, int64_t n, void* out, int out_dtype, void* stream) {
  int64_t blocks;
  if (int rc = weight_args("dequantize_q4", out, out_dtype, rows, n, w4, blocks)) return rc;
  if (!blocks) return NKV_OK;
  const dim3 grid((unsigned)blocks), block(64);
  hipStream_t s = static_cast<hipStream_t>(stream);
  uint8_t* to = static_cast<uint8_t*>(out);
  if (out_dtype == NKV_F16) hipLaunchKernelGGL(dequant4_weight_kernel<NKV_F16>, grid, block, 0, s, w4, rows, n, to);
  else if (out_dtype == NKV_BF16) hipLaunchKernelGGL(dequant4_weight_kernel<NKV_BF16>, grid, block, 0, s, w4, rows, n, to);
  else hipLaunchKernelGGL(dequant4_weight_kernel<NKV_F32>, grid, block, 0, s, w4, rows, n, to);
  return check_launch("dequantize_q4");
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
  const dim3 grid((unsigned)std::min<int64_t>(cdiv(a.chunks, 256), 1 << 20)), block(256);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (x_dtype == NKV_F16) hipLaunchKernelGGL(quant4_pages_kernel<NKV_F16>, grid, block, 0, s, a);
  else if (x_dtype == NKV_BF16) hipLaunchKernelGGL(quant4_pages_kernel<NKV_BF16>, grid, block, 0, s, a);
  else hipLaunchKernelGGL(quant4_pages_kernel<NKV_F32>, grid, block, 0, s, a);
  return check_launch(what);
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
  if (wide == ROWS256) hipLaunchKernelGGL(attn_q4_kernel, grid, dim3(Q4_THREADS), 0, s, a);
  else if (wide == ROWS16) hipLaunchKernelGGL(attn_q4_small_kernel<1>, grid, dim3(64 * Q4_SMALL), 0, s, a);
  else hipLaunchKernelGGL(attn_q4_small_kernel<2>, grid, dim3(64 * Q4_SMALL), 0, s, a);
  if (int rc = check_launch(what)) return rc;
  return launch_merges(what, a, reinterpret_cast<const Merge*>(merges), n_merges, s);
}
