// attn_masked.hip - attention of rows of queries over the f16 cache, with capped scores, a bias by distance and a
// span of keys for each row (documents packed side by side, sliding windows, prompts that see themselves whole, a
// prefix that all rows share), for one row as for a chunk.
//
// For row t at position p_t, q head h and a key j that the row sees (j < hi_t, and j >= lo_t or j < prefix):
//   s = scale q_t . k_j;  with a cap s = cap tanh(s / cap);  with slopes s -= slope_h |p_t - j|
//   out_t = sum_j e^s v_j / sum_j e^s, zeros for a row that sees no key.
// Scores are formed in base 2, y = s log2(e). cap tanh(x / cap) = cap - 2 cap / (e^(2 x / cap) + 1), which costs an
// exponential, a reciprocal and two fused operations and is off by 2^-22 cap at most, where f16 weights are off by 2^-11.
// A column (a row and one of its q heads) keeps a reference r and forms its weights as 2^(y - r); r is raised, and the
// accumulators rescaled, only when a score passes it by more than 15, and then to 7 below that score: the weights
// are f16 numbers up to 2^15, and 2^-24 of the largest is still an f16 number to eight bits, so that the many small weights of
// a long cache are not lost. q is taken as f16 high and low parts, so scores carry fp32's error of the sum alone;
// the weights are rounded to f16 once (2^-11 of each weight, as much as the output's own rounding).
//
// A key that a row does not see has weight 0, but 0 times an infinity or a NaN of its V row is a NaN. A block whose
// result is not finite is therefore formed again, key by key, over the keys that each row sees.
#include <algorithm>

#include "mi_capi_internal.h"
#include "mi_common.h"

namespace mi {
namespace {

constexpr float kNoKey = -1e30f, kLog2e = 1.4426950408889634f;
constexpr float kRaise = 15.f, kBelow = 7.f;
constexpr uint32_t kTile = 32;      // keys per step of a wave
constexpr uint32_t kMaxRows = 128;  // rows of a block at most

struct MaskedArgs {
  const float* q;        // [T][q_heads][HD]
  const uint16_t *k, *v;
  const uint32_t* pages;
  const uint32_t *lo, *hi, *pos;
  const float* slopes;
  uint16_t* out;         // [T][q_heads][HD]
  float* part;           // splits > 1: see part_at
  uint32_t* flag;
  size_t row_stride, head_stride;
  uint32_t page, page_shift, n_pages, kv_len, T, pos0, prefix, q_heads, kv_heads, gqa, rows, splits, act;
  float c, c2, cap;      // y = c s, or cap - 2 cap / (2^(c2 s) + 1) (cap here in base 2)
};

// What a block's rows see, and the 32-key tiles that hold it: tiles [0, n_a) of the prefix, then from b0 on.
struct Block {
  uint32_t lo[kMaxRows], hi[kMaxRows], pos[kMaxRows];  // hi 0: the row sees nothing
  uint32_t min_lo, max_lo, min_hi, max_hi;
  int again;
};
struct Tiles {
  uint32_t n_a, b0, n;
  __device__ __forceinline__ uint32_t key(uint32_t i) const { return kTile * (i < n_a ? i : b0 + (i - n_a)); }
};
__device__ __forceinline__ uint32_t row_pos(const MaskedArgs& a, uint32_t t) { return a.pos ? a.pos[t] : a.pos0 + t; }

// every thread of the work-group; rows_here <= its threads
__device__ __forceinline__ Tiles block_begin(const MaskedArgs& a, Block& b, uint32_t t0, uint32_t rows_here) {
  const uint32_t t = threadIdx.x;
  if (t == 0) {
    b.min_lo = b.min_hi = 0xFFFFFFFFu;
    b.max_lo = b.max_hi = 0u;
    b.again = 0;
  }
  __syncthreads();
  if (t < rows_here) {
    const uint32_t p = row_pos(a, t0 + t);
    uint32_t hi = min(a.hi ? a.hi[t0 + t] : p + 1u, a.kv_len), lo = min(a.lo ? a.lo[t0 + t] : 0u, hi);
    if (lo == hi && min(a.prefix, hi) == 0u) lo = hi = 0u;  // nothing
    b.lo[t] = lo;
    b.hi[t] = hi;
    b.pos[t] = p;
    if (hi) {
      atomicMin(&b.min_lo, lo);
      atomicMax(&b.max_lo, lo);
      atomicMin(&b.min_hi, hi);
      atomicMax(&b.max_hi, hi);
    }
  }
  __syncthreads();
  Tiles w{0u, 0u, 0u};
  if (b.max_hi) {
    w.n_a = (min(a.prefix, b.max_hi) + kTile - 1u) / kTile;
    w.b0 = max(b.min_lo / kTile, w.n_a);
    const uint32_t end = (b.max_hi + kTile - 1u) / kTile;
    w.n = w.n_a + (end > w.b0 ? end - w.b0 : 0u);
  }
  return w;
}

// the cache row of a key below kv_len
__device__ __forceinline__ uint32_t cache_row(const MaskedArgs& a, uint32_t key) {
  if (!a.pages) return key;
  const uint32_t at = a.page_shift < 32u ? key >> a.page_shift : key / a.page;
  uint32_t pg = a.pages[at];
  if (pg >= a.n_pages) {
    if (a.flag) *a.flag = MI_STATUS_BAD_PAGE;
    pg = 0u;
  }
  return pg * a.page + (key - at * a.page);
}

// A column of a wave's 16 x CT: its span and what its scores take.
struct Column {
  uint32_t lo, hi, pos;
  float slope;
  bool live;  // a row and a head, and the row sees something
};
__device__ __forceinline__ Column column(const MaskedArgs& a, const Block& b, uint32_t j, uint32_t row, uint32_t g,
                                         uint32_t rows_here) {
  Column c{0u, 0xFFFFFFFFu, 0u, 0.f, row < rows_here && b.hi[min(row, kMaxRows - 1u)] != 0u};
  if (row < rows_here) c.pos = b.pos[row];
  if (c.live) {  // (any other column sees every key and is not written)
    c.lo = b.lo[row];
    c.hi = b.hi[row];
  }
  if (a.slopes) c.slope = a.slopes[j * a.gqa + g] * kLog2e;
  return c;
}
__device__ __forceinline__ bool sees(const MaskedArgs& a, const Column& c, uint32_t key) {
  return key < c.hi && (key >= c.lo || key < a.prefix);
}
// The scores of keys key0 + 16 (e / 4) + e % 4 (e < 8) in base 2, -inf for a key that the column does not see.
__device__ __forceinline__ void scores(const MaskedArgs& a, const Column& c, uint32_t key0, bool masked, float (&w)[8]) {
  if (a.cap != 0.f) {
#pragma unroll
    for (uint32_t e = 0; e < 8; ++e)
      w[e] = __builtin_fmaf(-2.f * a.cap, __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(w[e] * a.c2) + 1.f), a.cap);
  } else {
#pragma unroll
    for (uint32_t e = 0; e < 8; ++e) w[e] *= a.c;
  }
  if (a.slopes) {
    const float d = (float)(int)(c.pos - key0);
#pragma unroll
    for (uint32_t e = 0; e < 8; ++e) w[e] = __builtin_fmaf(-c.slope, fabsf(d - (float)(16u * (e / 4) + e % 4)), w[e]);
  }
  if (masked) {
#pragma unroll
    for (uint32_t e = 0; e < 8; ++e) w[e] = sees(a, c, key0 + 16u * (e / 4) + e % 4) ? w[e] : -INFINITY;
  }
}
// whether some column of the block does not see some key of the tile (uniform)
__device__ __forceinline__ bool tile_masked(const MaskedArgs& a, const Block& b, uint32_t key) {
  return key + kTile > b.min_hi || (key < b.max_lo && key + kTile > a.prefix);
}

// where a split leaves column `col` of its block: HD values (sums of weight times V), then r and the weights' sum
template <int HD>
__device__ __forceinline__ float* part_at(const MaskedArgs& a, uint32_t j, uint32_t t, uint32_t g, uint32_t split) {
  return a.part + ((size_t)(t * a.q_heads + j * a.gqa + g) * a.splits + split) * (HD + 4);
}

// The columns of a block one by one, over the keys that they see only: a lane holds dims lane + 64 i.
template <int HD>
__device__ __forceinline__ void slow_block(const MaskedArgs& a, const Block& b, const Tiles& tiles, uint32_t j, uint32_t t0,
                                           uint32_t rows_here, uint32_t from, uint32_t to, uint32_t split) {
  constexpr uint32_t D = HD / 64;
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
  const size_t hoff = (size_t)j * a.head_stride;
#pragma unroll 1
  for (uint32_t p = wave; p < rows_here * a.gqa; p += blockDim.x / 64u) {
    const uint32_t row = p / a.gqa, g = p % a.gqa;
    const Column c = column(a, b, j, row, g, rows_here);
    const float* q = a.q + ((size_t)(t0 + row) * a.q_heads + j * a.gqa + g) * HD + lane;
    float r = kNoKey, l = 0.f, acc[D];
#pragma unroll
    for (uint32_t i = 0; i < D; ++i) acc[i] = 0.f;
    if (c.live) {
#pragma unroll 1
      for (uint32_t i = from; i < to; ++i) {
        const uint32_t k0 = tiles.key(i);
#pragma unroll 1
        for (uint32_t key = k0; key < k0 + kTile; ++key) {
          if (!sees(a, c, key)) continue;
          const size_t at = (size_t)cache_row(a, key) * a.row_stride + hoff + lane;
          float s = 0.f;
#pragma unroll
          for (uint32_t d = 0; d < D; ++d) s = __builtin_fmaf(q[64u * d], h2f(a.k[at + 64u * d]), s);
          float w[8] = {wave_sum(s), 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
          scores(a, c, key, false, w);
          if (w[0] > r + kRaise) {
            const float to_r = w[0] - kBelow, alpha = __builtin_amdgcn_exp2f(r - to_r);
            r = to_r;
            l *= alpha;
#pragma unroll
            for (uint32_t d = 0; d < D; ++d) acc[d] *= alpha;
          }
          const float pw = __builtin_amdgcn_exp2f(w[0] - r);
          l += pw;
#pragma unroll
          for (uint32_t d = 0; d < D; ++d) acc[d] = __builtin_fmaf(pw, h2f(a.v[at + 64u * d]), acc[d]);
        }
      }
    }
    if (a.splits > 1) {
      float* o = part_at<HD>(a, j, t0 + row, g, split);
#pragma unroll
      for (uint32_t d = 0; d < D; ++d) o[lane + 64u * d] = acc[d];
      if (lane == 0) {
        o[HD] = r;
        o[HD + 1] = l;
      }
    } else {
      uint16_t* o = a.out + ((size_t)(t0 + row) * a.q_heads + j * a.gqa + g) * HD + lane;
#pragma unroll
      for (uint32_t d = 0; d < D; ++d) o[64u * d] = act_enc(l == 0.f ? 0.f : acc[d] / l, a.act);
    }
  }
}

// q of a column as the B operand, f16 high and low parts: k = 32 kk + 8 qq + e
template <int HD>
__device__ __forceinline__ void load_q(const float* qp, h8_t (&qh)[HD / 32], h8_t (&ql)[HD / 32]) {
  float neg1 = -1.f;
  asm("" : "+s"(neg1));
#pragma unroll
  for (uint32_t kk = 0; kk < HD / 32; ++kk) {
    const f4_t q0 = *reinterpret_cast<const f4_any*>(qp + 32u * kk), q1 = *reinterpret_cast<const f4_any*>(qp + 32u * kk + 4);
    u4_t h, l;
    uint32_t hh, ll;
    f16_parts(q0.x, q0.y, neg1, hh, ll); h.x = hh; l.x = ll;
    f16_parts(q0.z, q0.w, neg1, hh, ll); h.y = hh; l.y = ll;
    f16_parts(q1.x, q1.y, neg1, hh, ll); h.z = hh; l.z = ll;
    f16_parts(q1.z, q1.w, neg1, hh, ll); h.w = hh; l.w = ll;
    qh[kk] = __builtin_bit_cast(h8_t, h);
    ql[kk] = __builtin_bit_cast(h8_t, l);
  }
}

// One step of a column's softmax: the scores w become weights (in place and as the B operand of P V).
template <uint32_t NT>
__device__ __forceinline__ h8_t weigh(float (&w)[8], uint32_t qi, float& r, float& l, f4_t (&acc)[NT]) {
  const float mx = max3(max3(w[0], w[1], w[2]), max3(w[3], w[4], w[5]), max3(w[6], w[7], w[7]));
  if (const uint64_t over = __ballot(mx > r + kRaise)) {
    // (each column by its own four lanes, whatever its neighbours need)
    const uint32_t o = (uint32_t)over | (uint32_t)(over >> 32);
    const float cm = col_max(mx), to = ((o | o >> 16) >> qi) & 1u ? fmaxf(r, cm - kBelow) : r;
    const float alpha = __builtin_amdgcn_exp2f(r - to);
    r = to;
    l *= alpha;
#pragma unroll
    for (uint32_t tt = 0; tt < NT; ++tt) acc[tt] *= alpha;
  }
#pragma unroll
  for (uint32_t e = 0; e < 8; ++e) w[e] = __builtin_amdgcn_exp2f(w[e] - r);
  l += ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
  u4_t b;
#pragma unroll
  for (uint32_t e = 0; e < 4; ++e) b[e] = h2_bits(__builtin_convertvector((f2_t{w[2 * e], w[2 * e + 1]}), h2_t));
  return __builtin_bit_cast(h8_t, b);
}
typedef short v4s_t __attribute__((ext_vector_type(4)));
typedef v4s_t __attribute__((address_space(3)))* v4s_lds;
// V^T of a 32-key tile as the A operand: the k of the product are the keys 4 qq + e of the two 16-key groups, which is
// how the lanes hold the weights; 4 keys' dims come from one transposing read
template <uint32_t VROW>
__device__ __forceinline__ h8_t v_operand(const uint16_t* vb, uint32_t tt) {
  const v4s_t a0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((v4s_lds)(vb + 16u * tt));
  const v4s_t a1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((v4s_lds)(vb + 16u * VROW + 16u * tt));
  return __builtin_bit_cast(h8_t, __builtin_shufflevector(a0, a1, 0, 1, 2, 3, 4, 5, 6, 7));
}
// the sum over the four lanes of a column
__device__ __forceinline__ float col_sum(float x) {
  float a0 = x, a1 = x;
  lane_swap16(a0, a1);
  float b0 = a0 + a1, b1 = b0;
  lane_swap32(b0, b1);
  return b0 + b1;
}
template <int HD>
__device__ __forceinline__ void store_part(const MaskedArgs& a, uint32_t j, uint32_t t, uint32_t g, uint32_t split, uint32_t qq,
                                           uint32_t tt, f4_t v) {
  *reinterpret_cast<f4_t*>(part_at<HD>(a, j, t, g, split) + 16u * tt + 4u * qq) = v;
}
template <int HD>
__device__ __forceinline__ void store_out(const MaskedArgs& a, uint32_t j, uint32_t t, uint32_t g, uint32_t qq, uint32_t tt, f4_t v) {
  const u2_t h = {(uint32_t)act_enc(v[0], a.act) | ((uint32_t)act_enc(v[1], a.act) << 16),
                  (uint32_t)act_enc(v[2], a.act) | ((uint32_t)act_enc(v[3], a.act) << 16)};
  *reinterpret_cast<h4_any*>(a.out + ((size_t)t * a.q_heads + j * a.gqa + g) * HD + 16u * tt + 4u * qq) = h;
}
__device__ __forceinline__ float not_finite(f4_t v) {  // 0, or NaN
  return ((v[0] - v[0]) + (v[1] - v[1])) + ((v[2] - v[2]) + (v[3] - v[3]));
}

// Few rows (16 columns per block): grid (kv_heads, row blocks, splits), 4 waves. A wave walks its own 32-key tiles,
// every fourth of the split's: K from memory as the A operand, V through its own part of LDS for the transposing
// reads, the next tile's rows in registers meanwhile. The waves' sums join through LDS.
template <int HD>
__global__ __launch_bounds__(256, HD == 128 ? 2 : 1) void attn_masked_few_kernel(MaskedArgs a) {
  constexpr uint32_t KK = HD / 32, NT = HD / 16, VROW = HD + 16;
  constexpr uint32_t PPR = HD / 8, RPP = 64 / PPR, NV = kTile / RPP;  // 16-byte pieces per V row, rows per load, loads per tile
  __shared__ Block b;
  __shared__ __align__(16) union Slab {
    uint16_t v[kTile * VROW];
    struct {
      float acc[NT * 4][64], r[64], l[64];
    } part;
  } slab[4];
  const uint32_t j = blockIdx.x, t0 = blockIdx.y * a.rows, split = blockIdx.z;
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, qi = lane & 15u, qq = lane >> 4;
  const uint32_t rows_here = min(a.rows, a.T - t0);
  const Tiles tiles = block_begin(a, b, t0, rows_here);
  const uint32_t from = (uint32_t)((uint64_t)tiles.n * split / a.splits), to = (uint32_t)((uint64_t)tiles.n * (split + 1u) / a.splits);
  const uint32_t row = qi / a.gqa, g = qi % a.gqa;
  const Column col = column(a, b, j, row, g, rows_here);
  h8_t qh[KK], ql[KK];
  load_q<HD>(a.q + ((size_t)(t0 + (row < rows_here ? row : 0u)) * a.q_heads + j * a.gqa + g) * HD + 8u * qq, qh, ql);
  float r = kNoKey, l = 0.f;
  f4_t acc[NT];
#pragma unroll
  for (uint32_t tt = 0; tt < NT; ++tt) acc[tt] = f4_t{0.f, 0.f, 0.f, 0.f};

  const size_t hoff = (size_t)j * a.head_stride;
  const uint32_t last = b.max_hi - 1u;
  u4_t kr[2][KK], vr[NV];
  // a lane's cache row: of key 16 (lane / 16 % 2) + lane % 16 of the tile (keys behind the last one read it again)
  auto rows_of = [&](uint32_t i) { return cache_row(a, min(tiles.key(i) + (lane & 31u), last)); };
  auto load = [&](uint32_t crow) {
#pragma unroll
    for (uint32_t gg = 0; gg < 2; ++gg) {
      const uint16_t* p = a.k + (size_t)(uint32_t)__shfl((int)crow, (int)(16u * gg + qi), 64) * a.row_stride + hoff + 8u * qq;
#pragma unroll
      for (uint32_t kk = 0; kk < KK; ++kk) kr[gg][kk] = *reinterpret_cast<const u4_t*>(p + 32u * kk);
    }
#pragma unroll
    for (uint32_t i = 0; i < NV; ++i) {
      const uint32_t cr = (uint32_t)__shfl((int)crow, (int)(RPP * i + lane / PPR), 64);
      vr[i] = *reinterpret_cast<const u4_t*>(a.v + (size_t)cr * a.row_stride + hoff + 8u * (lane % PPR));
    }
  };
  uint32_t i = from + wave, crow = 0;
  if (i < to) {
    load(rows_of(i));
    if (i + 4u < to) crow = rows_of(i + 4u);
  }
  uint16_t* vs = slab[wave].v;
  const uint16_t* vb = vs + (4u * qq + (qi >> 2)) * VROW + 4u * (qi & 3u);
  for (; i < to; i += 4u) {
    const uint32_t key = tiles.key(i);
    f4_t d[2] = {f4_t{0.f, 0.f, 0.f, 0.f}, f4_t{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
    for (uint32_t kk = 0; kk < KK; ++kk)
#pragma unroll
      for (uint32_t gg = 0; gg < 2; ++gg) {
        d[gg] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8_t, kr[gg][kk]), qh[kk], d[gg], 0, 0, 0);
        d[gg] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8_t, kr[gg][kk]), ql[kk], d[gg], 0, 0, 0);
      }
    wave_lds_sync();
#pragma unroll
    for (uint32_t n = 0; n < NV; ++n) *reinterpret_cast<u4_t*>(vs + (RPP * n + lane / PPR) * VROW + 8u * (lane % PPR)) = vr[n];
    wave_lds_sync();
    if (i + 4u < to) {
      load(crow);
      if (i + 8u < to) crow = rows_of(i + 8u);
    }
    float w[8];
#pragma unroll
    for (uint32_t e = 0; e < 8; ++e) w[e] = d[e / 4][e % 4];
    scores(a, col, key + 4u * qq, tile_masked(a, b, key), w);
    const h8_t p = weigh<NT>(w, qi, r, l, acc);
#pragma unroll
    for (uint32_t tt = 0; tt < NT; ++tt) acc[tt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v_operand<VROW>(vb, tt), p, acc[tt], 0, 0, 0);
  }
  l = col_sum(l);
  float bad = 0.f;
#pragma unroll
  for (uint32_t tt = 0; tt < NT; ++tt) bad += not_finite(acc[tt]);
  if (col.live && (bad != 0.f || l - l != 0.f)) b.again = 1;
  wave_lds_sync();
  auto& mine = slab[wave].part;
#pragma unroll
  for (uint32_t tt = 0; tt < NT; ++tt)
#pragma unroll
    for (uint32_t e = 0; e < 4; ++e) mine.acc[4u * tt + e][lane] = acc[tt][e];
  mine.r[lane] = r;
  mine.l[lane] = l;
  __syncthreads();
  if (b.again) {
    slow_block<HD>(a, b, tiles, j, t0, rows_here, from, to, split);
    return;
  }
  // wave w joins the dims 16 tt + .. of its quarter of the tiles
  float top = slab[0].part.r[lane], f[4], sum = 0.f;
#pragma unroll
  for (uint32_t w = 1; w < 4; ++w) top = fmaxf(top, slab[w].part.r[lane]);
#pragma unroll
  for (uint32_t w = 0; w < 4; ++w) {
    f[w] = __builtin_amdgcn_exp2f(slab[w].part.r[lane] - top);
    sum = __builtin_fmaf(slab[w].part.l[lane], f[w], sum);
  }
  if (row >= rows_here) return;
  const float inv = col.live && sum != 0.f ? 1.0f / sum : 0.f;
#pragma unroll
  for (uint32_t n = 0; n < NT / 4; ++n) {
    const uint32_t tt = wave * (NT / 4) + n;
    f4_t v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (uint32_t w = 0; w < 4; ++w)
#pragma unroll
      for (uint32_t e = 0; e < 4; ++e) v[e] = __builtin_fmaf(slab[w].part.acc[4u * tt + e][lane], f[w], v[e]);
    if (a.splits > 1) store_part<HD>(a, j, t0 + row, g, split, qq, tt, v);
    else store_out<HD>(a, j, t0 + row, g, qq, tt, v * inv);
  }
  if (a.splits > 1 && wave == 0 && qq == 0) {
    float* o = part_at<HD>(a, j, t0 + row, g, split);
    o[HD] = top;
    o[HD + 1] = col.live ? sum : 0.f;
  }
}

// A chunk: grid (kv_heads, row blocks, splits); 4 waves side by side of CT column tiles each walk the same 32-key tiles,
// staged in LDS for all of them, the next tile's rows in registers meanwhile.
template <int HD, int CT>
__global__ __launch_bounds__(256, 2) void attn_masked_kernel(MaskedArgs a) {
  constexpr uint32_t KK = HD / 32, NT = HD / 16, KROW = HD + 8, VROW = HD + 16;
  constexpr uint32_t PPR = HD / 8, RPP = 256 / PPR, CH = kTile / RPP;  // 16-byte pieces per row, rows per pass, passes
  struct Stage {
    uint16_t k[kTile * KROW], v[kTile * VROW];
  };
  __shared__ Block b;
  __shared__ __align__(16) Stage st[2];
  // the last row blocks of a causal chunk see the most keys: they are dispatched first
  const uint32_t j = blockIdx.x, t0 = (gridDim.y - 1u - blockIdx.y) * a.rows, split = blockIdx.z;
  const uint32_t t = threadIdx.x, lane = t & 63u, wave = t >> 6, qi = lane & 15u, qq = lane >> 4;
  const uint32_t rows_here = min(a.rows, a.T - t0);
  const Tiles tiles = block_begin(a, b, t0, rows_here);
  const uint32_t from = (uint32_t)((uint64_t)tiles.n * split / a.splits), to = (uint32_t)((uint64_t)tiles.n * (split + 1u) / a.splits);
  const size_t hoff = (size_t)j * a.head_stride;
  const uint32_t last = b.max_hi - 1u, srow = t / PPR, sp = 8u * (t % PPR);
  u4_t kr[CH], vr[CH];
  uint32_t crow[CH];
  auto rows_of = [&](uint32_t i) {
#pragma unroll
    for (uint32_t n = 0; n < CH; ++n) crow[n] = cache_row(a, min(tiles.key(i) + RPP * n + srow, last));
  };
  auto load = [&]() {
#pragma unroll
    for (uint32_t n = 0; n < CH; ++n) {
      const size_t at = (size_t)crow[n] * a.row_stride + hoff + sp;
      kr[n] = *reinterpret_cast<const u4_t*>(a.k + at);
      vr[n] = *reinterpret_cast<const u4_t*>(a.v + at);
    }
  };
  auto store = [&](Stage& s) {
#pragma unroll
    for (uint32_t n = 0; n < CH; ++n) {
      *reinterpret_cast<u4_t*>(s.k + (RPP * n + srow) * KROW + sp) = kr[n];
      *reinterpret_cast<u4_t*>(s.v + (RPP * n + srow) * VROW + sp) = vr[n];
    }
  };
  if (from < to) {
    rows_of(from);
    load();
    if (from + 1u < to) rows_of(from + 1u);
  }
  const bool computes = 16u * CT * wave < rows_here * a.gqa;  // a wave without a live column only stages
  uint32_t row[CT], g[CT];
  Column col[CT];
  h8_t qh[CT][KK], ql[CT][KK];
  float r[CT], l[CT];
  f4_t acc[CT][NT];
#pragma unroll
  for (uint32_t ct = 0; ct < CT; ++ct) {
    const uint32_t p = 16u * (CT * wave + ct) + qi;
    row[ct] = p / a.gqa;
    g[ct] = p % a.gqa;
    col[ct] = column(a, b, j, row[ct], g[ct], rows_here);
    load_q<HD>(a.q + ((size_t)(t0 + (row[ct] < rows_here ? row[ct] : 0u)) * a.q_heads + j * a.gqa + g[ct]) * HD + 8u * qq, qh[ct],
               ql[ct]);
    r[ct] = kNoKey;
    l[ct] = 0.f;
#pragma unroll
    for (uint32_t tt = 0; tt < NT; ++tt) acc[ct][tt] = f4_t{0.f, 0.f, 0.f, 0.f};
  }
  if (from < to) {
    store(st[0]);
    if (from + 1u < to) {
      load();
      if (from + 2u < to) rows_of(from + 2u);
    }
  }
  lds_barrier();
  for (uint32_t i = from; i < to; ++i) {
    const Stage& s = st[(i - from) & 1u];
    if (computes) {
      const uint32_t key = tiles.key(i);
      f4_t d[CT][2];
#pragma unroll
      for (uint32_t ct = 0; ct < CT; ++ct) d[ct][0] = d[ct][1] = f4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (uint32_t kk = 0; kk < KK; ++kk)
#pragma unroll
        for (uint32_t gg = 0; gg < 2; ++gg) {
          const h8_t kh = *reinterpret_cast<const h8_t*>(s.k + (16u * gg + qi) * KROW + 32u * kk + 8u * qq);
#pragma unroll
          for (uint32_t ct = 0; ct < CT; ++ct) d[ct][gg] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kh, qh[ct][kk], d[ct][gg], 0, 0, 0);
#pragma unroll
          for (uint32_t ct = 0; ct < CT; ++ct) d[ct][gg] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kh, ql[ct][kk], d[ct][gg], 0, 0, 0);
        }
      const bool masked = tile_masked(a, b, key);
      h8_t p[CT];
#pragma unroll
      for (uint32_t ct = 0; ct < CT; ++ct) {
        float w[8];
#pragma unroll
        for (uint32_t e = 0; e < 8; ++e) w[e] = d[ct][e / 4][e % 4];
        scores(a, col[ct], key + 4u * qq, masked, w);
        p[ct] = weigh<NT>(w, qi, r[ct], l[ct], acc[ct]);
      }
      const uint16_t* vb = s.v + (4u * qq + (qi >> 2)) * VROW + 4u * (qi & 3u);
#pragma unroll
      for (uint32_t tt = 0; tt < NT; ++tt) {
        const h8_t av = v_operand<VROW>(vb, tt);
#pragma unroll
        for (uint32_t ct = 0; ct < CT; ++ct) acc[ct][tt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(av, p[ct], acc[ct][tt], 0, 0, 0);
      }
    }
    // (the other buffer was last read before the previous barrier)
    if (i + 1u < to) {
      store(st[(i + 1u - from) & 1u]);
      if (i + 2u < to) {
        load();
        if (i + 3u < to) rows_of(i + 3u);
      }
    }
    lds_barrier();
  }
  float sum[CT];
#pragma unroll
  for (uint32_t ct = 0; ct < CT; ++ct) {
    sum[ct] = col_sum(l[ct]);
    float bad = 0.f;
#pragma unroll
    for (uint32_t tt = 0; tt < NT; ++tt) bad += not_finite(acc[ct][tt]);
    if (col[ct].live && (bad != 0.f || sum[ct] - sum[ct] != 0.f)) b.again = 1;
  }
  __syncthreads();
  if (b.again) {
    slow_block<HD>(a, b, tiles, j, t0, rows_here, from, to, split);
    return;
  }
#pragma unroll
  for (uint32_t ct = 0; ct < CT; ++ct) {
    if (row[ct] >= rows_here) continue;
    if (a.splits > 1) {
#pragma unroll
      for (uint32_t tt = 0; tt < NT; ++tt) store_part<HD>(a, j, t0 + row[ct], g[ct], split, qq, tt, acc[ct][tt]);
      if (qq == 0) {
        float* o = part_at<HD>(a, j, t0 + row[ct], g[ct], split);
        o[HD] = r[ct];
        o[HD + 1] = col[ct].live ? sum[ct] : 0.f;
      }
    } else {
      const float inv = col[ct].live && sum[ct] != 0.f ? 1.0f / sum[ct] : 0.f;
#pragma unroll
      for (uint32_t tt = 0; tt < NT; ++tt) store_out<HD>(a, j, t0 + row[ct], g[ct], qq, tt, inv == 0.f ? f4_t{0.f, 0.f, 0.f, 0.f} : acc[ct][tt] * inv);
    }
  }
}

// grid (q_heads, T): one column's splits, a thread per dim
template <int HD>
__global__ __launch_bounds__(HD) void attn_masked_join_kernel(MaskedArgs a) {
  const uint32_t h = blockIdx.x, t = blockIdx.y, d = threadIdx.x;
  const float* p = a.part + (size_t)(t * a.q_heads + h) * a.splits * (HD + 4);
  float top = kNoKey, sum = 0.f, v = 0.f;
  for (uint32_t s = 0; s < a.splits; ++s)
    if (p[s * (HD + 4) + HD + 1] != 0.f) top = fmaxf(top, p[s * (HD + 4) + HD]);
  for (uint32_t s = 0; s < a.splits; ++s) {
    const float l = p[s * (HD + 4) + HD + 1];
    if (l == 0.f) continue;  // (no key of the row in that part)
    const float f = __builtin_amdgcn_exp2f(p[s * (HD + 4) + HD] - top);
    sum = __builtin_fmaf(l, f, sum);
    v = __builtin_fmaf(p[s * (HD + 4) + d], f, v);
  }
  a.out[((size_t)t * a.q_heads + h) * HD + d] = act_enc(sum == 0.f ? 0.f : v / sum, a.act);
}

// The launch: few columns per block, or a chunk's, and the parts that the keys are split in.
struct Pick {
  bool few;
  uint32_t ct, rows, splits;
};
constexpr uint32_t kCus = 256;
Pick pick(uint32_t T, uint32_t keys, uint32_t kv_heads, uint32_t gqa, uint32_t hd) {
  Pick p;
  p.few = gqa <= 16 && T * gqa <= 16;
  p.ct = !p.few && hd == 128 && (uint64_t)kv_heads * ((T + 128 / gqa - 1) / (128 / gqa)) > kCus ? 2 : 1;
  p.rows = (p.few ? 16u : 64u * p.ct) / gqa;
  const uint64_t blocks = (uint64_t)kv_heads * ((T + p.rows - 1) / p.rows);
  const uint64_t want = p.few ? (4 * kCus + blocks - 1) / blocks : (2 * kCus + blocks - 1) / blocks;
  const uint64_t most = (keys + 255u) / 256u;  // (at least 256 keys each)
  p.splits = blocks >= kCus ? 1u : (uint32_t)std::max<uint64_t>(1, std::min(want, most));
  return p;
}
size_t part_bytes(const Pick& p, uint32_t T, uint32_t q_heads, uint32_t hd) {
  return p.splits == 1 ? 0 : (size_t)T * q_heads * p.splits * (hd + 4) * 4;
}
bool shape_ok(const mi_attn_shape* s) {
  return s && s->kv_heads && s->q_heads && s->q_heads % s->kv_heads == 0 && s->q_heads / s->kv_heads <= 64 &&
         s->q_heads <= 1024 && (s->head_dim == 128 || s->head_dim == 256);
}

}  // namespace
}  // namespace mi

using namespace mi;

extern "C" {

size_t mi_attn_masked_ws(uint32_t T, uint32_t kv_len, const mi_attn_shape* shape) {
  if (T == 0 || kv_len == 0 || !shape_ok(shape)) return 0;
  return part_bytes(pick(T, kv_len, shape->kv_heads, shape->q_heads / shape->kv_heads, shape->head_dim), T, shape->q_heads,
                    shape->head_dim);
}

int mi_attn_masked(const float* attn_q, const uint16_t* kv_k, const uint16_t* kv_v, size_t row_stride, size_t head_stride,
                   const uint32_t* pages, uint32_t page, uint32_t n_pages, uint32_t kv_len, uint32_t T,
                   const mi_attn_shape* shape, const mi_attn_mask* mask, void* ws, size_t ws_bytes, uint16_t* attn_out,
                   uint32_t* flag, void* stream) {
  if (!attn_q || !kv_k || !kv_v || !attn_out || !shape || !mask) return mi_fail(MI_ERR_ARG, "attn_masked: null pointer");
  if (!shape_ok(shape))
    return mi_fail(MI_ERR_SHAPE, "attn_masked: head_dim 128 or 256, q_heads a multiple of kv_heads, up to 64 of them each");
  if (shape->gated) return mi_fail(MI_ERR_SHAPE, "attn_masked: gated shapes are not supported");
  if (shape->act > 1) return mi_fail(MI_ERR_ARG, "attn_masked: act is 0 or 1");
  if (T == 0 || T > 65535 || kv_len == 0 || kv_len > 1u << 30) return mi_fail(MI_ERR_SHAPE, "attn_masked: T 1..65535, kv_len 1..2^30");
  if (pages && (page == 0 || n_pages == 0)) return mi_fail(MI_ERR_ARG, "attn_masked: page size or page count 0");
  if (pages && (uint64_t)page * n_pages > 0xFFFFFFFFull) return mi_fail(MI_ERR_SHAPE, "attn_masked: above 2^32 cache rows");
  if (row_stride % 8 || head_stride % 8) return mi_fail(MI_ERR_ARG, "attn_masked: KV strides must keep 8-element alignment");
  auto off = [](const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1u)) != 0; };
  if (off(kv_k, 16) || off(kv_v, 16) || off(attn_q, 4) || off(attn_out, 2))
    return mi_fail(MI_ERR_ARG, "attn_masked: misaligned pointer (K and V 16 bytes)");
  if (!(mask->cap >= 0.f) || mask->cap > 1e30f) return mi_fail(MI_ERR_ARG, "attn_masked: cap is 0 (none) or positive and finite");
  const uint32_t gqa = shape->q_heads / shape->kv_heads;
  const Pick p = pick(T, kv_len, shape->kv_heads, gqa, shape->head_dim);
  const size_t need = part_bytes(p, T, shape->q_heads, shape->head_dim);
  if (need && (!ws || off(ws, 16) || ws_bytes < need))
    return mi_fail(MI_ERR_ARG, "attn_masked: the workspace is null, misaligned (16 bytes) or below mi_attn_masked_ws");
  MaskedArgs a{};
  a.q = attn_q;
  a.k = kv_k;
  a.v = kv_v;
  a.pages = pages;
  a.lo = mask->lo;
  a.hi = mask->hi;
  a.pos = mask->pos;
  a.slopes = mask->slopes;
  a.out = attn_out;
  a.part = static_cast<float*>(ws);
  a.flag = flag;
  a.row_stride = row_stride;
  a.head_stride = head_stride;
  a.page = page;
  a.page_shift = pages && (page & (page - 1u)) == 0 ? (uint32_t)__builtin_ctz(page) : 32u;
  a.n_pages = n_pages;
  a.kv_len = kv_len;
  a.T = T;
  a.pos0 = mask->pos0;
  a.prefix = mask->prefix;
  a.q_heads = shape->q_heads;
  a.kv_heads = shape->kv_heads;
  a.gqa = gqa;
  a.rows = p.rows;
  a.splits = p.splits;
  a.act = shape->act;
  a.c = shape->scale * kLog2e;
  a.cap = mask->cap * kLog2e;
  a.c2 = mask->cap != 0.f ? 2.f * a.c / mask->cap : 0.f;
  hipStream_t st = (hipStream_t)stream;
  const dim3 grid(shape->kv_heads, (T + p.rows - 1u) / p.rows, p.splits);
  const bool narrow = shape->head_dim == 128;
  if (p.few) {
    if (narrow) attn_masked_few_kernel<128><<<grid, 256, 0, st>>>(a);
    else attn_masked_few_kernel<256><<<grid, 256, 0, st>>>(a);
  } else if (narrow) {
    if (p.ct == 2) attn_masked_kernel<128, 2><<<grid, 256, 0, st>>>(a);
    else attn_masked_kernel<128, 1><<<grid, 256, 0, st>>>(a);
  } else {
    attn_masked_kernel<256, 1><<<grid, 256, 0, st>>>(a);
  }
  if (p.splits > 1) {
    if (narrow) attn_masked_join_kernel<128><<<dim3(shape->q_heads, T), 128, 0, st>>>(a);
    else attn_masked_join_kernel<256><<<dim3(shape->q_heads, T), 256, 0, st>>>(a);
  }
  return mi_hip((int)hipGetLastError(), "attn_masked");
}

}  // extern "C"
