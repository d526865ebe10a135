// attn_rows.h - what attention of rows of queries over the f16 cache shares, whatever the rows see: the kernel of a few columns (a
// column is a row and one of its q heads), the softmax's steps, operands, stores, and the way out where a result is not finite. What a
// row sees, where a work-group's rows and keys are and where a key lies in the cache is the caller's type A (MaskedRows in
// attn_masked.hip, TreeRows in attn_tree.hip), the kernels' argument:
//   Place place(bool chunk)      kv head j, the rows t0 .. t0 + rows - 1, and which of `splits` parts of their keys it takes
//                                (kItems: each_item instead, for the places of a work-group one behind another)
//   Block block(Place)           the 32-key tiles that the rows see: n of them, the first key of each, the last key that a row sees
//   uint32_t part_begin(...)     the first tile of a part
//   Column column(...)           what a column sees; bool masked(Block, key): whether some column does not see some key of a tile
//   bool sees(Column, key), bias_and_mask, scores_by_form: of products the scores in base 2
//   row_of, cache_row            the cache rows of keys, with whether a page's entry is outside the cache; report_pages
//   part_at                      where a part's sums go: HD values (sums of weight times V), then the reference and the weights' sum
//
// For a column with scores y_j in base 2: out = sum_j 2^y_j v_j / sum_j 2^y_j.
// A column keeps a reference r and forms its weights as 2^(y - r); r is raised, and the accumulators rescaled, only when a
// score passes it by more than 15, and then to 7 below that score: the weights are f16 numbers up to 2^15, and 2^-24 of the
// largest is still an f16 number to eight bits, so that the many small weights of a long cache are not lost. q is taken as f16
// high and low parts, so scores carry fp32's error of the sum alone. The few-rows kernel takes the weights so too (it is bound
// by the cache's bytes, not by products); the kernels of many columns round each to f16 once (2^-11 of it, as much as the output's
// own rounding; the weights' sum is taken before).
//
// A key that a row does not see has weight 0, but 0 times an infinity or a NaN of its V row is a NaN. A block whose
// result is not finite is therefore formed again, key by key, over the keys that each row sees. That is slow, and a call lasts as long
// as its slowest block: with one NaN among the keys that one of 48 texts' next tokens sees they take 2.3 ms (0.27), 8 trees of up to 61
// rows 36 ms (0.09).
#pragma once
#include <type_traits>

#include "mi_pieces.h"

namespace mi {
namespace {

constexpr float kNoKey = -0x1.fffffep127f;  // the reference before the first key: no finite score is below it
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kRaise = 15.f, kBelow = 7.f;
constexpr uint32_t kTile = 32;      // keys per step of a wave

template <typename F>
__device__ __forceinline__ uint32_t wave_fold(uint32_t v, F f) {
  auto swap = [](uint32_t x, auto c) { return (uint32_t)__builtin_amdgcn_mov_dpp((int)x, decltype(c)::value, 0xF, 0xF, false); };
  v = f(v, swap(v, std::integral_constant<int, 0xB1>{}));
  v = f(v, swap(v, std::integral_constant<int, 0x4E>{}));
  v = f(v, swap(v, std::integral_constant<int, 0x141>{}));
  v = f(v, swap(v, std::integral_constant<int, 0x140>{}));
  auto at = [&](int lane) { return (uint32_t)__builtin_amdgcn_readlane((int)v, lane); };
  return f(f(at(0), at(16)), f(at(32), at(48)));
}

// The cache's order: contiguous, pages that hold whole tiles (one table entry for a tile's 32 keys), any pages.
enum Order { kContiguous, kWholeTiles, kAnyPages };

// The columns of a block one by one, over the keys that they see only: a lane holds dims lane + 64 i. `capped` makes scores in
// base 2 of products.
template <int HD, typename A, typename F>
__device__ __forceinline__ void slow_block(const A& a, const typename A::Place& p, const typename A::Block& b, uint32_t from,
                                           uint32_t to, F capped) {
  constexpr uint32_t D = HD / 64;
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
  const size_t hoff = (size_t)p.j * a.head_stride;
#pragma unroll 1
  for (uint32_t i = wave; i < p.rows * a.gqa; i += blockDim.x / 64u) {
    const uint32_t row = i / a.gqa, g = i % a.gqa;
    const auto c = a.column(p, b, row, g);
    const float* q = a.q + ((size_t)(p.t0 + row) * a.q_heads + p.j * a.gqa + g) * HD + lane;
    float r = kNoKey, l = 0.f, acc[D];
#pragma unroll
    for (uint32_t i = 0; i < D; ++i) acc[i] = 0.f;
    if (c.live) {
#pragma unroll 1
      for (uint32_t n = from; n < to; ++n) {
        const uint32_t k0 = b.key(n);
#pragma unroll 1
        for (uint32_t key = k0; key < k0 + kTile; ++key) {
          if (!a.sees(c, key)) continue;
          bool outside;  // (the block's walk has reported it)
          const size_t at = (size_t)a.cache_row(b, key, outside) * a.row_stride + hoff + lane;
          float s = 0.f;
#pragma unroll
          for (uint32_t d = 0; d < D; ++d) s = __builtin_fmaf(q[64u * d], h2f(a.k[at + 64u * d]), s);
          float w[8] = {wave_sum(s), 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
          capped(w);
          a.bias_and_mask(c, key, false, w);
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
    if (p.splits > 1) {
      float* o = a.template part_at<HD>(p, row, g);
#pragma unroll
      for (uint32_t d = 0; d < D; ++d) o[lane + 64u * d] = acc[d];
      if (lane == 0) {
        o[HD] = r;
        o[HD + 1] = l;
      }
    } else {
      uint16_t* o = a.out + ((size_t)(p.t0 + row) * a.q_heads + p.j * a.gqa + g) * HD + lane;
#pragma unroll
      for (uint32_t d = 0; d < D; ++d) o[64u * d] = act_enc(l == 0.f ? 0.f : acc[d] / l, a.act);
    }
  }
}

// KK x 32 dims of a column's q as the B operand, f16 high and low parts: k = 32 kk + 8 qq + e
template <uint32_t KK>
__device__ __forceinline__ void split_q(const f4_t (&q)[2 * KK], h8_t (&qh)[KK], h8_t (&ql)[KK]) {
  float neg1 = -1.f;
  asm("" : "+s"(neg1));
#pragma unroll
  for (uint32_t kk = 0; kk < KK; ++kk) {
    u4_t h, l;
#pragma unroll
    for (uint32_t x = 0; x < 4; ++x) {
      uint32_t hh, ll;
      f16_parts(q[2 * kk + x / 2][2 * (x % 2)], q[2 * kk + x / 2][2 * (x % 2) + 1], neg1, hh, ll);
      h[x] = hh;
      l[x] = ll;
    }
    qh[kk] = __builtin_bit_cast(h8_t, h);
    ql[kk] = __builtin_bit_cast(h8_t, l);
  }
}
template <uint32_t KK>
__device__ __forceinline__ void load_q(const float* qp, h8_t (&qh)[KK], h8_t (&ql)[KK]) {
  f4_t q[2 * KK];
#pragma unroll
  for (uint32_t x = 0; x < 2 * KK; ++x) q[x] = *as_global(reinterpret_cast<const f4_any*>(qp + 32u * (x / 2) + 4u * (x % 2)));
  split_q<KK>(q, qh, ql);
}

__device__ __forceinline__ float most_of(const float (&w)[8]) {
  return max3(max3(w[0], w[1], w[2]), max3(w[3], w[4], w[5]), max3(w[6], w[7], w[7]));
}
// One step of the softmax of a wave's CT column tiles, whose lanes' largest scores are mx. The references first: raised, with what
// was formed by them, where a score passes one (each column by its own four lanes, whatever its neighbours need). NT 0: the
// accumulators are left to the caller, with their factor.
template <uint32_t CT, uint32_t NT, uint32_t N, uint32_t M>
__device__ __forceinline__ void raise_to(const float (&mx)[N], uint32_t qi, float (&r)[M], float (&l)[M], f4_t (*acc)[NT ? NT : 1],
                                         float* factor) {
  bool over = false;
#pragma unroll
  for (uint32_t ct = 0; ct < CT; ++ct) over |= mx[ct] > r[ct] + kRaise;
  if (!__ballot(over)) return;
#pragma unroll
  for (uint32_t ct = 0; ct < CT; ++ct) {
    const uint64_t lanes = __ballot(mx[ct] > r[ct] + kRaise);
    const uint32_t o = (uint32_t)lanes | (uint32_t)(lanes >> 32);
    const float cm = col_max(mx[ct]), to = ((o | o >> 16) >> qi) & 1u ? fmaxf(r[ct], cm - kBelow) : r[ct];
    const float alpha = __builtin_amdgcn_exp2f(r[ct] - to);
    r[ct] = to;
    l[ct] *= alpha;
#pragma unroll
    for (uint32_t tt = 0; tt < NT; ++tt) acc[ct][tt] *= alpha;
    if constexpr (NT == 0) *factor = alpha;
  }
}
template <uint32_t CT, uint32_t NT>
__device__ __forceinline__ void raise(const float (&w)[CT][8], uint32_t qi, float (&r)[CT], float (&l)[CT], f4_t (*acc)[NT ? NT : 1],
                                      float* factor) {
  float mx[CT];
#pragma unroll
  for (uint32_t ct = 0; ct < CT; ++ct) mx[ct] = most_of(w[ct]);
  raise_to<CT, NT>(mx, qi, r, l, acc, factor);
}
// Then the weights, as the B operands of P V in f16 high and low parts; their sum goes to l.
__device__ __forceinline__ void weights(float (&w)[8], float r, float& l, h8_t& hi, h8_t& lo) {
#pragma unroll
  for (uint32_t e = 0; e < 8; ++e) w[e] = __builtin_amdgcn_exp2f(w[e] - r);
  l += ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
  float neg1 = -1.f;
  asm("" : "+s"(neg1));
  u4_t h, m;
#pragma unroll
  for (uint32_t e = 0; e < 4; ++e) {
    uint32_t hh, mm;
    f16_parts(w[2 * e], w[2 * e + 1], neg1, hh, mm);
    h[e] = hh;
    m[e] = mm;
  }
  hi = __builtin_bit_cast(h8_t, h);
  lo = __builtin_bit_cast(h8_t, m);
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
template <int HD, typename A>
__device__ __forceinline__ void store_part(const A& a, const typename A::Place& p, uint32_t row, uint32_t g, uint32_t qq,
                                           uint32_t tt, f4_t v) {
  *reinterpret_cast<f4_t*>(a.template part_at<HD>(p, row, g) + 16u * tt + 4u * qq) = v;
}
template <int HD, typename A>
__device__ __forceinline__ void store_out(const A& a, uint32_t j, uint32_t t, uint32_t g, uint32_t qq, uint32_t tt, f4_t v) {
  const u2_t h = {(uint32_t)act_enc(v[0], a.act) | ((uint32_t)act_enc(v[1], a.act) << 16),
                  (uint32_t)act_enc(v[2], a.act) | ((uint32_t)act_enc(v[3], a.act) << 16)};
  *reinterpret_cast<h4_any*>(a.out + ((size_t)t * a.q_heads + j * a.gqa + g) * HD + 16u * tt + 4u * qq) = h;
}
__device__ __forceinline__ float not_finite(float z, f4_t v) {  // 0 (a zero z), or NaN
#pragma unroll
  for (uint32_t e = 0; e < 4; ++e) z = __builtin_fmaf(v[e], 0.f, z);
  return z;
}

// 16 bytes of a row that the caches need not keep (a batch's cache is read once a step: 48 sequences of up to 16000 keys, 1.58 GB,
// 267 us, 5.9 TB/s, and 293 with loads that they keep; eight of 4000 keys, which the last cache holds from call to call, 31 and 29).
template <bool ONCE>
__device__ __forceinline__ u4_t load_row(const uint16_t* p) {
  if constexpr (ONCE) return __builtin_nontemporal_load(as_global(reinterpret_cast<const u4_t*>(p)));
  else return *reinterpret_cast<const u4_t*>(p);
}
// Few rows (16 columns per block): grid (kv_heads, row blocks, splits), or with kItems work-groups that take such places one behind
// another; 4 waves. A wave walks its own 32-key tiles, every fourth of the split's: K from memory as the A operand, V through its own
// part of LDS for the transposing reads, the next tile's rows in registers meanwhile. The waves' sums join through LDS.
template <int HD, typename A>
__device__ __forceinline__ void few_rows_of(const A& a, const typename A::Place& p) {
  constexpr uint32_t KK = HD / 32, NT = HD / 16, VROW = HD + 16;
  constexpr uint32_t PPR = HD / 8, RPP = 64 / PPR, NV = kTile / RPP;  // 16-byte pieces per V row, rows per load, loads per tile
  __shared__ __align__(16) union Slab {
    uint16_t v[kTile * VROW];
    struct {
      float acc[NT * 4][64], r[64], l[64];
    } part;
  } slab[4];
  uint32_t thread = threadIdx.x;
  if constexpr (A::kItems) asm volatile("" : "+v"(thread));  // (what follows from it is formed anew in each item, not kept)
  const uint32_t lane = thread & 63u, wave = thread >> 6, qi = lane & 15u, qq = lane >> 4;
  const uint32_t j = p.j, t0 = p.t0, rows_here = p.rows;
  const uint32_t row = qi / a.gqa, g = qi % a.gqa;
  const typename A::Block b = a.block(p);
  const auto col = a.column(p, b, row, g);
  const uint32_t from = a.part_begin(p, b, p.split), to = a.part_begin(p, b, p.split + 1u);
  const float* qp = a.q + ((size_t)(t0 + (row < rows_here ? row : 0u)) * a.q_heads + j * a.gqa + g) * HD + 8u * qq;
  float r[1] = {kNoKey}, l[1] = {0.f};
  f4_t acc[1][NT];
#pragma unroll
  for (uint32_t tt = 0; tt < NT; ++tt) acc[0][tt] = f4_t{0.f, 0.f, 0.f, 0.f};

  const size_t hoff = (size_t)j * a.head_stride;
  u4_t kr[2][KK], vr[NV];
  // a lane's cache row: of key 16 (lane / 16 % 2) + lane % 16 of the tile
  bool outside = false;
  auto rows_of = [&](uint32_t i) {
    const uint32_t key = b.key(i) + (lane & 31u);
    return a.row_of(b, i, key, outside);
  };
  auto load = [&](uint32_t crow) {
#pragma unroll
    for (uint32_t gg = 0; gg < 2; ++gg) {
      const uint16_t* p = a.k + (size_t)(uint32_t)__shfl((int)crow, (int)(16u * gg + qi), 64) * a.row_stride + hoff + 8u * qq;
#pragma unroll
      for (uint32_t kk = 0; kk < KK; ++kk) kr[gg][kk] = load_row<A::kItems>(p + 32u * kk);
    }
#pragma unroll
    for (uint32_t i = 0; i < NV; ++i) {
      const uint32_t cr = (uint32_t)__shfl((int)crow, (int)(RPP * i + lane / PPR), 64);
      vr[i] = load_row<A::kItems>(a.v + (size_t)cr * a.row_stride + hoff + 8u * (lane % PPR));
    }
  };
  uint32_t i = from + wave, crow = 0;
  if (i < to) {
    load(rows_of(i));
    if (i + 4u < to) crow = rows_of(i + 4u);
  }
  h8_t qh[KK], ql[KK];
  load_q<KK>(qp, qh, ql);
  uint16_t* vs = slab[wave].v;
  const uint16_t* vb = vs + (4u * qq + (qi >> 2)) * VROW + 4u * (qi & 3u);
  for (; i < to; i += 4u) {
    const uint32_t key = b.key(i);
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
      const uint32_t now = crow;  // (the next rows' page is asked for before these rows are)
      if (i + 8u < to) crow = rows_of(i + 8u);
      load(now);
    }
    float w[1][8];
#pragma unroll
    for (uint32_t e = 0; e < 8; ++e) w[0][e] = d[e / 4][e % 4];
    a.scores_by_form(w[0]);
    a.bias_and_mask(col, key + 4u * qq, a.masked(b, key), w[0]);
    raise<1, NT>(w, qi, r, l, acc, nullptr);
    h8_t ph, pl;
    weights(w[0], r[0], l[0], ph, pl);
#pragma unroll
    for (uint32_t tt = 0; tt < NT; ++tt) {
      const h8_t av = v_operand<VROW>(vb, tt);
      acc[0][tt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(av, ph, acc[0][tt], 0, 0, 0);
      acc[0][tt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(av, pl, acc[0][tt], 0, 0, 0);
    }
  }
  if (__ballot(outside)) a.report_pages(p, b, from + wave, to, 4u);
  l[0] = col_sum(l[0]);
  float bad = 0.f;
#pragma unroll
  for (uint32_t tt = 0; tt < NT; ++tt) bad = not_finite(bad, acc[0][tt]);
  bad += l[0] - l[0];
  wave_lds_sync();
  auto& mine = slab[wave].part;
#pragma unroll
  for (uint32_t tt = 0; tt < NT; ++tt)
#pragma unroll
    for (uint32_t e = 0; e < 4; ++e) mine.acc[4u * tt + e][lane] = acc[0][tt][e];
  mine.r[lane] = r[0];
  mine.l[lane] = l[0];
  if (__syncthreads_or(col.live && bad != 0.f)) {
    slow_block<HD>(a, p, b, from, to, [&](float(&w)[8]) { a.scores_by_form(w); });
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
    if (!col.live) v = f4_t{0.f, 0.f, 0.f, 0.f};  // (what it summed may be a NaN, which no factor makes a zero)
    if (p.splits > 1) store_part<HD>(a, p, row, g, qq, tt, v);
    else store_out<HD>(a, j, t0 + row, g, qq, tt, v * inv);
  }
  if (p.splits > 1 && wave == 0 && qq == 0) {
    float* o = a.template part_at<HD>(p, row, g);
    o[HD] = top;
    o[HD + 1] = col.live ? sum : 0.f;
  }
}
template <int HD, typename A>
__global__ __launch_bounds__(256, HD == 128 ? 2 : 1) void attn_rows_few_kernel(A a) {
  if constexpr (A::kItems) {
    a.each_item([&](const typename A::Place& p) { few_rows_of<HD>(a, p); });
  } else {
    few_rows_of<HD>(a, a.place(false));
  }
}

}  // namespace
}  // namespace mi
