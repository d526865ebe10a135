// attn_masked.hip - attention of rows of queries over the f16 cache, with capped scores, a bias by distance and a
// span of keys for each row (documents packed side by side, sliding windows, prompts that see themselves whole, a
// prefix that all rows share), for one row as for a chunk.
//
// For row t at position p_t, q head h and a key j that the row sees (j < hi_t, and j >= lo_t or j < prefix):
//   s = scale q_t . k_j;  with a cap s = cap tanh(s / cap);  with slopes s -= slope_h |p_t - j|
//   out_t = sum_j e^s v_j / sum_j e^s, zeros for a row that sees no key.
// Scores are formed in base 2, y = s log2(e). cap tanh(x / cap) = cap - 2 cap / (e^(2 x / cap) + 1), which costs an
// exponential, a reciprocal and two fused operations and is off by 2^-21 cap at most; caps above 256, where that error would come
// near the weights' rounding, take a form whose error goes with the score.
// The kernels, and how their softmax and its roundings go, are attn_rows.h's.
//
// What bounds it (MI355X): one row the cache's bytes, 131072 keys of 8 heads of 128 99 us, 5.4 TB/s; a chunk the matrix
// cores, whose products are 3 per score-and-value pair (q in two parts): 2048 rows causal over 2048, 40 / 8 heads of 128,
// 83 us; where rows see little (7 documents in 2048 rows 35.4 us, 14 of it the bytes of q and the outputs) a work-group's
// chain of loads before its first tile, the tiles' unseen parts, and CUs that are done before the longest document's.
//
// A key that a row does not see has weight 0, but 0 times an infinity or a NaN of its V row is a NaN. A block whose
// result is not finite is therefore formed again, key by key, over the keys that each row sees. That is slow: a NaN in an unseen V row
// of one part in 64 takes one row over 131072 keys from 100 us to 2.5 ms, one between 7 documents 2048 rows from 38 to 1560.
#include <algorithm>

#include "attn_rows.h"
#include "mi_capi_internal.h"

namespace mi {
namespace {

constexpr uint32_t kMaxRows = 65535, kMaxKeys = 1u << 30;

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
  uint32_t form;         // a Cap
};

// A row's span: lo <= hi <= kv_len; lo == hi: it sees the prefix alone, up to hi; hi 0: it sees nothing.
struct Span {
  uint32_t lo, hi, pos;
};
__device__ __forceinline__ Span row_span(const MaskedArgs& a, uint32_t t) {
  Span s;
  s.pos = a.pos ? a.pos[t] : a.pos0 + t;
  s.hi = min(a.hi ? a.hi[t] : s.pos + 1u, a.kv_len);
  s.lo = min(a.lo ? a.lo[t] : 0u, s.hi);
  if (s.lo == s.hi) s.lo = s.hi = min(a.prefix, s.hi);
  return s;
}
// What a block's rows see, and the 32-key tiles that hold it: tiles [0, n_a) of the prefix, then from b0 on. Every wave
// forms it by itself from the rows' spans, a row (or two) per lane: no barrier stands before the first loads.
struct Block {
  uint32_t min_hi, max_lo, last;  // the last key that a row sees
  uint32_t prefix, gap;           // the prefix's end as far as a row sees it, and how many keys behind it no row sees
  uint32_t n_a, b0, n;
  __device__ __forceinline__ uint32_t key(uint32_t i) const { return kTile * (i < n_a ? i : b0 + (i - n_a)); }
  // A key of tile i, or where it lies outside what the rows see one of that tile that does not: a page that holds such keys alone
  // may not be there.
  __device__ __forceinline__ uint32_t within(uint32_t i, uint32_t k) const {
    k = min(k, last);
    return k - prefix < gap ? (i < n_a ? prefix - 1u : prefix + gap) : k;
  }
};
__device__ __forceinline__ Block block_of(const MaskedArgs& a, uint32_t t0, uint32_t rows_here) {
  const uint32_t lane = threadIdx.x & 63u;
  uint32_t min_lo = 0xFFFFFFFFu, min_hi = 0xFFFFFFFFu, max_lo = 0u, max_hi = 0u;
  for (uint32_t r = lane; r < rows_here; r += 64u) {
    const Span s = row_span(a, t0 + r);
    if (s.hi) {
      if (s.lo < s.hi) min_lo = min(min_lo, s.lo);
      max_lo = max(max_lo, s.lo);
      min_hi = min(min_hi, s.hi);
      max_hi = max(max_hi, s.hi);
    }
  }
  auto lesser = [](uint32_t x, uint32_t y) { return min(x, y); };
  auto greater = [](uint32_t x, uint32_t y) { return max(x, y); };
  min_lo = wave_fold(min_lo, lesser);
  max_hi = wave_fold(max_hi, greater);
  Block b{wave_fold(min_hi, lesser), wave_fold(max_lo, greater), max_hi - 1u, min(a.prefix, max_hi), 0u, 0u, 0u, 0u};
  if (max_hi) {
    b.gap = max(min_lo, b.prefix) - b.prefix;
    b.n_a = (b.prefix + kTile - 1u) / kTile;
    b.b0 = max(min_lo / kTile, b.n_a);
    const uint32_t end = (max_hi + kTile - 1u) / kTile;
    b.n = b.n_a + (end > b.b0 ? end - b.b0 : 0u);
  }
  return b;
}

__device__ __forceinline__ uint32_t page_of(const MaskedArgs& a, uint32_t key) {
  return a.page_shift < 32u ? key >> a.page_shift : key / a.page;
}
// the cache row of a key below kv_len; `outside`: its page's entry is not the cache's, and the row is the first page's
__device__ __forceinline__ uint32_t cache_row(const MaskedArgs& a, uint32_t key, bool& outside) {
  if (!a.pages) return key;
  const uint32_t at = page_of(a, key);
  uint32_t pg = a.pages[at];
  if (pg >= a.n_pages) {
    outside = true;
    pg = 0u;
  }
  return pg * a.page + (key - at * a.page);
}
// A wave that met such an entry among the tiles from, from + step .. of its block reports it if a row sees one of the keys: the
// tiles between the rows' spans (far apart documents in one block) are walked too.
__device__ __forceinline__ void report_pages(const MaskedArgs& a, const Block& b, uint32_t t0, uint32_t rows_here, uint32_t from,
                                             uint32_t to, uint32_t step) {
  if (!a.flag) return;
#pragma unroll 1
  for (uint32_t i = from; i < to; i += step) {
    const uint32_t key = b.key(i) + (threadIdx.x & (kTile - 1u));
    if (key > b.last || a.pages[page_of(a, key)] < a.n_pages) continue;
#pragma unroll 1
    for (uint32_t r = 0; r < rows_here; ++r) {
      const Span s = row_span(a, t0 + r);
      if (key < s.hi && (key >= s.lo || key < a.prefix)) *a.flag = MI_STATUS_BAD_PAGE;
    }
  }
}

// A column of a wave's 16 x CT: its span and what its scores take.
struct Column {
  uint32_t lo, hi, pos;
  float slope;
  bool live;  // a row and a head, and the row sees something
};
__device__ __forceinline__ Column column(const MaskedArgs& a, uint32_t j, uint32_t t0, uint32_t row, uint32_t g, uint32_t rows_here) {
  const Span s = row_span(a, t0 + min(row, rows_here - 1u));
  Column c{s.lo, s.hi, s.pos, 0.f, row < rows_here && s.hi != 0u};
  if (!c.live) {  // (it sees every key, so no tile is masked for it; zeros are stored in place of what it sums)
    c.lo = 0u;
    c.hi = 0xFFFFFFFFu;
  }
  if (a.slopes) c.slope = a.slopes[j * a.gqa + g] * kLog2e;
  return c;
}
__device__ __forceinline__ bool sees(const MaskedArgs& a, const Column& c, uint32_t key) {
  return key < c.hi && (key >= c.lo || key < a.prefix);
}
// The scores' cap: none; one up to kPlainCap, by one exponential; any, by a form that leaves the scores their bits where the cap is
// far above them.
enum Cap { kNoCap, kPlain, kAnyCap };
// The plain form's error is the cap's, 2^-21 of it: at 256 2^-13 of a weight, below their own rounding to f16.
constexpr float kPlainCap = 256.f;
// A score in base 2, the cap applied.
template <Cap CAP>
__device__ __forceinline__ float score(const MaskedArgs& a, float s) {
  if constexpr (CAP == kNoCap) return s * a.c;
  if constexpr (CAP == kPlain)
    return __builtin_fmaf(-2.f * a.cap, __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(s * a.c2) + 1.f), a.cap);
  // With u = x / cap and t = 2 u log2(e): from |u| = 1/4 on the same form at |t|, with the sign of t, its error 2^-20 of the score;
  // below, x (1 - u^2 / 3 + 2 u^4 / 15 - 17 u^6 / 315), off by 62 u^8 / 2835 < 2^-21 of it.
  constexpr float kU2 = 0.25f * 0.4804530139182014f;  // u^2 = (ln 2 / 2)^2 t^2
  const float t = s * a.c2, v = t * t;
  const float far = __builtin_fmaf(-2.f * a.cap, __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(fabsf(t)) + 1.f), a.cap);
  const float f = __builtin_fmaf(v, __builtin_fmaf(v, -17.f / 315.f * kU2 * kU2 * kU2, 2.f / 15.f * kU2 * kU2), -1.f / 3.f * kU2);
  return v < 0.0625f / kU2 ? s * a.c * __builtin_fmaf(v, f, 1.f) : copysignf(far, t);
}
// The rest for the scores of keys key0 + 16 (e / 4) + e % 4 (e < 8): the bias, and -inf for a key that the column does not
// see.
__device__ __forceinline__ void bias_and_mask(const MaskedArgs& a, const Column& c, uint32_t key0, bool masked, float (&w)[8]) {
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
// (where the cap's form is not the kernel's own)
__device__ __forceinline__ void scores_by_form(const MaskedArgs& a, float (&w)[8]) {
  if (a.form == kAnyCap) {
#pragma unroll
    for (uint32_t e = 0; e < 8; ++e) w[e] = score<kAnyCap>(a, w[e]);
  } else if (a.form == kPlain) {
#pragma unroll
    for (uint32_t e = 0; e < 8; ++e) w[e] = score<kPlain>(a, w[e]);
  } else {
#pragma unroll
    for (uint32_t e = 0; e < 8; ++e) w[e] = score<kNoCap>(a, w[e]);
  }
}
// The kernels' argument (attn_rows.h).
struct Place {
  uint32_t j, t0, rows, split, splits;
};
struct MaskedRows : MaskedArgs {
  using Place = mi::Place;
  using Block = mi::Block;
  using Column = mi::Column;
  static constexpr bool kItems = false;
  // grid (kv_heads, row blocks, splits); the last row blocks of a causal chunk see the most keys: they are dispatched first
  __device__ __forceinline__ Place place(bool chunk) const {
    const uint32_t t0 = (chunk ? gridDim.y - 1u - blockIdx.y : blockIdx.y) * rows;
    return {blockIdx.x, t0, min(rows, T - t0), blockIdx.z, splits};
  }
  __device__ __forceinline__ Block block(const Place& p) const { return block_of(*this, p.t0, p.rows); }
  __device__ __forceinline__ uint32_t part_begin(const Place& p, const Block& b, uint32_t split) const {
    return (uint32_t)((uint64_t)b.n * split / p.splits);
  }
  __device__ __forceinline__ Column column(const Place& p, const Block&, uint32_t row, uint32_t g) const {
    return mi::column(*this, p.j, p.t0, row, g, p.rows);
  }
  __device__ __forceinline__ bool masked(const Block& b, uint32_t key) const {
    return key + kTile > b.min_hi || (key < b.max_lo && key + kTile > prefix);
  }
  __device__ __forceinline__ bool sees(const Column& c, uint32_t key) const { return mi::sees(*this, c, key); }
  template <Cap CAP>
  __device__ __forceinline__ float score(float s) const {
    return mi::score<CAP>(*this, s);
  }
  __device__ __forceinline__ void scores_by_form(float (&w)[8]) const { mi::scores_by_form(*this, w); }
  __device__ __forceinline__ void bias_and_mask(const Column& c, uint32_t key0, bool masked, float (&w)[8]) const {
    mi::bias_and_mask(*this, c, key0, masked, w);
  }
  __device__ __forceinline__ uint32_t first_row(const Block&, uint32_t key) const { return key; }
  __device__ __forceinline__ uint32_t cache_row(const Block&, uint32_t key, bool& outside) const {
    return mi::cache_row(*this, key, outside);
  }
  __device__ __forceinline__ uint32_t row_of(const Block& b, uint32_t i, uint32_t key, bool& outside) const {
    return pages ? mi::cache_row(*this, b.within(i, key), outside) : min(key, b.last);
  }
  __device__ __forceinline__ void report_pages(const Place& p, const Block& b, uint32_t from, uint32_t to, uint32_t step) const {
    mi::report_pages(*this, b, p.t0, p.rows, from, to, step);
  }
  template <int HD>
  __device__ __forceinline__ float* part_at(const Place& p, uint32_t row, uint32_t g) const {
    return part + ((size_t)((p.t0 + row) * q_heads + p.j * gqa + g) * splits + p.split) * (HD + 4);
  }
};

// A chunk: grid (kv_heads, row blocks, splits). Four waves side by side take CT column tiles each and 128 of the dims; at
// rows of 256 four more take the other half (a wave's registers hold 32 columns of 128 dims with two waves per SIMD, and
// every LDS read then serves 32 columns). All walk the same 32-key tiles, K and V staged in LDS for all of them, the rows
// after them in registers meanwhile. A step i has two halves with a barrier between them:
//   the products of tile i + 1's scores, dealt out among the exponentials that make tile i's weights;
//   P V of tile i, dealt out among the scaling (and the tanh) of tile i + 1's scores, whose maxima follow.
// So the matrix core has products while the vector ALUs work in the same wave. The halves of the dims exchange their parts
// of the scores through LDS across the barrier. With two column tiles each of the two waves takes the softmax of one, its
// tile 0 (the other wave's 1): the parts of the other's scores go over, and a step later the weights and the factor of a raised
// reference come back (777 rows over 3778 keys, 16 / 2 heads, with distances, in 5 parts: 125 -> 110 us).
template <int HD, int CT, Cap CAP, Order ORDER>
__global__ __launch_bounds__(2 * HD, 2) void attn_masked_kernel(MaskedRows a) {
  constexpr uint32_t DS = HD / 128, KK = 4, NT = 8, KROW = HD + 8, VROW = HD + 16, THREADS = 2 * HD;
  constexpr uint32_t PPR = HD / 8, RPP = THREADS / PPR, CH = kTile / RPP;  // 16-byte pieces per row, rows per pass, passes
  constexpr bool OWN = DS == 2 && CT == 2;
  constexpr uint32_t SC = OWN ? 1 : CT;  // column tiles whose softmax the wave takes
  __shared__ __align__(16) struct {
    uint16_t k[2][kTile * KROW], v[2][kTile * VROW];
    f4_t s[DS > 1 ? 2 : 1][DS > 1 ? 4 * DS : 1][2 * SC][DS > 1 ? 64 : 1];
    h8_t p[OWN ? 2 : 1][OWN ? 8 : 1][OWN ? 64 : 1];
    float f[OWN ? 2 : 1][OWN ? 8 : 1][OWN ? 64 : 1];  // the references' factors; the sums at the end
  } st;
  const uint32_t t = threadIdx.x, lane = t & 63u, wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(t >> 6)), qi = lane & 15u, qq = lane >> 4;
  const uint32_t cw = wave % 4u, ds = wave / 4u;
  const Place pl = a.place(true);
  const uint32_t j = pl.j, t0 = pl.t0, rows_here = pl.rows;
  const Block b = a.block(pl);
  uint32_t row[CT], g[CT];
  Column col[SC];
  bool live[CT];
  f4_t qraw[CT][2 * KK];  // (converted behind the first tiles' loads)
#pragma unroll
  for (uint32_t ct = 0; ct < CT; ++ct) {
    const uint32_t p = 16u * (CT * cw + (OWN ? ct ^ ds : ct)) + qi;
    row[ct] = p / a.gqa;
    g[ct] = p % a.gqa;
    const auto c = a.column(pl, b, row[ct], g[ct]);
    live[ct] = c.live;
    if (ct < SC) col[ct] = c;
    const float* qp = a.q + ((size_t)(t0 + (row[ct] < rows_here ? row[ct] : 0u)) * a.q_heads + j * a.gqa + g[ct]) * HD + 128u * ds + 8u * qq;
#pragma unroll
    for (uint32_t x = 0; x < 2 * KK; ++x) qraw[ct][x] = *as_global(reinterpret_cast<const f4_any*>(qp + 32u * (x / 2) + 4u * (x % 2)));
  }
  const uint32_t from = a.part_begin(pl, b, pl.split), n = a.part_begin(pl, b, pl.split + 1u) - from;
  auto uniform = [](uint32_t v) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)v); };
  const size_t hoff = (size_t)j * a.head_stride;
  const uint32_t srow = t / PPR, sp = 8u * (t % PPR);
  u4_t kr[CH], vr[CH];
  // the cache rows of tile i: its first (r[0]) where they follow one another, else those that the thread loads
  struct Rows {
    uint32_t r[CH];
  };
  bool outside = false;
  auto rows_of = [&](uint32_t i) {
    Rows w;
    const uint32_t tile = from + min(i, n - 1u), key0 = b.key(tile);
    if constexpr (ORDER == kContiguous) {
      w.r[0] = a.first_row(b, key0);
    } else if constexpr (ORDER == kWholeTiles) {
      w.r[0] = a.cache_row(b, key0, outside);
    } else {
#pragma unroll
      for (uint32_t c = 0; c < CH; ++c) w.r[c] = a.cache_row(b, b.within(tile, key0 + RPP * c + srow), outside);
    }
    return w;
  };
  // (a tile behind the last is that one again, and its loads are not used)
  auto load = [&](const uint16_t* cache, uint32_t i, const Rows& w, u4_t (&to)[CH]) {
    const uint32_t left = b.last - b.key(from + min(i, n - 1u));
#pragma unroll
    for (uint32_t c = 0; c < CH; ++c) {
      const uint32_t r = ORDER == kAnyPages ? w.r[c] : uniform(w.r[0]) + min(RPP * c + srow, left);
      to[c] = *as_global(reinterpret_cast<const u4_t*>(cache + (size_t)r * a.row_stride + hoff + sp));
    }
  };
  auto store = [&](uint16_t* to, uint32_t pitch, const u4_t (&v)[CH]) {
#pragma unroll
    for (uint32_t c = 0; c < CH; ++c) *reinterpret_cast<u4_t*>(to + (RPP * c + srow) * pitch + sp) = v[c];
  };
  // the rows of the tiles i + 1 .. i + 3 of a step i: V of the first and K of the last are loaded in it (a page's entry is
  // fetched a step before the loads that need it)
  Rows r1, r2, r3;
  u4_t k1[CH];
  if (n) {
    const Rows r0 = rows_of(0);
    r1 = rows_of(1);
    r2 = rows_of(2);
    r3 = rows_of(3);
    load(a.k, 0, r0, kr);
    load(a.v, 0, r0, vr);
    load(a.k, 1, r1, k1);
  }
  float r[SC], l[SC], factor = 1.f;
  f4_t acc[CT][NT], d[CT][2];
  h8_t qh[CT][KK], ql[CT][KK];
#pragma unroll
  for (uint32_t ct = 0; ct < CT; ++ct) {
    split_q<KK>(qraw[ct], qh[ct], ql[ct]);
    if (ct < SC) {
      r[ct] = kNoKey;
      l[ct] = 0.f;
    }
#pragma unroll
    for (uint32_t tt = 0; tt < NT; ++tt) acc[ct][tt] = f4_t{0.f, 0.f, 0.f, 0.f};
  }
  // One K operand (16 keys x 32 dims, number s = 2 kk + gg) and its products: this wave's part of the scores
  // S^T[key 16 gg + 4 qq + e][column qi].
  auto k_operand = [&](uint32_t buf, uint32_t s) {
    return *reinterpret_cast<const h8_t*>(st.k[buf] + (16u * (s % 2u) + qi) * KROW + 128u * ds + 8u * qq + 32u * (s / 2u));
  };
  auto product = [&](h8_t kh, uint32_t s, uint32_t part) {  // part < 2 CT: the columns' high parts, then the low ones
    const uint32_t ct = part % CT;
    d[ct][s % 2] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kh, part < CT ? qh[ct][s / 2] : ql[ct][s / 2], d[ct][s % 2], 0, 0, 0);
  };
  auto clear = [&]() {
#pragma unroll
    for (uint32_t ct = 0; ct < CT; ++ct) d[ct][0] = d[ct][1] = f4_t{0.f, 0.f, 0.f, 0.f};
  };
  auto hand_over = [&](uint32_t buf) {
    if constexpr (DS > 1) {
#pragma unroll
      for (uint32_t ct = 0; ct < SC; ++ct)
#pragma unroll
        for (uint32_t gg = 0; gg < 2; ++gg) st.s[buf][wave][2 * ct + gg][lane] = d[OWN ? 1 : ct][gg];
    }
  };
  auto take_over = [&](uint32_t buf) {
    if constexpr (DS > 1) {
#pragma unroll
      for (uint32_t ct = 0; ct < SC; ++ct)
#pragma unroll
        for (uint32_t gg = 0; gg < 2; ++gg) d[ct][gg] += st.s[buf][wave ^ 4u][2 * ct + gg][lane];
    }
  };
  float w[SC][8];
  // the scores w of tile i: bias, mask, and the columns' references
  auto settle = [&](uint32_t i) {
    const uint32_t key = b.key(from + i);
    const bool masked = a.masked(b, key);
#pragma unroll
    for (uint32_t ct = 0; ct < SC; ++ct) a.bias_and_mask(col[ct], key + 4u * qq, masked, w[ct]);
    if constexpr (OWN) raise<1, 0>(w, qi, r, l, nullptr, &factor);
    else raise<CT, NT>(w, qi, r, l, acc, nullptr);
  };
  if (n) {
    store(st.k[0], KROW, kr);
    store(st.k[1], KROW, k1);
    load(a.k, 2, r2, kr);
    lds_barrier();
    clear();
#pragma unroll
    for (uint32_t s = 0; s < 2 * KK; ++s) {
      const h8_t kh = k_operand(0, s);
#pragma unroll
      for (uint32_t part = 0; part < 2 * CT; ++part) product(kh, s, part);
    }
    hand_over(0);
    lds_barrier();
    take_over(0);
#pragma unroll
    for (uint32_t ct = 0; ct < SC; ++ct)
#pragma unroll
      for (uint32_t e = 0; e < 8; ++e) w[ct][e] = a.score<CAP>(d[ct][e / 4][e % 4]);
    settle(0);
  }
  for (uint32_t i = 0; i < n; ++i) {
    const uint32_t cur = i & 1u, nxt = cur ^ 1u;
    // V of tile i and K of tile i + 2 into the buffers that were last read before the barrier behind us; then the loads of
    // the next step's
    store(st.v[cur], VROW, vr);
    store(st.k[cur], KROW, kr);
    const Rows r4 = rows_of(i + 4u);
    load(a.v, i + 1u, r1, vr);
    load(a.k, i + 3u, r3, kr);
    r1 = r2;
    r2 = r3;
    r3 = r4;
    h8_t p[CT];
    {  // (behind the last tile the products are of a tile that is not used)
      constexpr uint32_t S = 2 * KK, AHEAD = 3;
      h8_t kh[S];
      clear();
#pragma unroll
      for (uint32_t s = 0; s < AHEAD; ++s) kh[s] = k_operand(nxt, s);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (uint32_t s = 0; s < S; ++s) {
        if (s + AHEAD < S) kh[s + AHEAD] = k_operand(nxt, s + AHEAD);
#pragma unroll
        for (uint32_t h = 0; h < CT; ++h) {  // two products, one weight (or a weight for every four)
          product(kh[s], s, 2 * h);
          product(kh[s], s, 2 * h + 1);
          if (h >= SC) continue;
          const uint32_t x = s * SC + h, ct = x / 8, e = x % 8;
          w[ct][e] = __builtin_amdgcn_exp2f(w[ct][e] - r[ct]);
          l[ct] += w[ct][e];
          if (e % 2) {
            u4_t pk = __builtin_bit_cast(u4_t, p[ct]);
            pk[e / 2] = h2_bits(__builtin_convertvector((f2_t{w[ct][e - 1], w[ct][e]}), h2_t));
            p[ct] = __builtin_bit_cast(h8_t, pk);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      hand_over(nxt);
      if constexpr (OWN) {
        st.p[cur][wave][lane] = p[0];
        st.f[cur][wave][lane] = factor;
      }
    }
    lds_barrier();
    {
      const uint16_t* vb = st.v[cur] + (4u * qq + (qi >> 2)) * VROW + 128u * ds + 4u * (qi & 3u);
      constexpr uint32_t AHEAD = 3;
      h8_t av[NT];
#pragma unroll
      for (uint32_t tt = 0; tt < AHEAD; ++tt) av[tt] = v_operand<VROW>(vb, tt);
      if constexpr (OWN) {
        p[1] = st.p[cur][wave ^ 4u][lane];
        const float other = st.f[cur][wave ^ 4u][lane];
        if (__ballot(factor != 1.f || other != 1.f)) {
#pragma unroll
          for (uint32_t tt = 0; tt < NT; ++tt) {
            acc[0][tt] *= factor;
            acc[1][tt] *= other;
          }
        }
        factor = 1.f;
      }
      take_over(nxt);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (uint32_t tt = 0; tt < NT; ++tt) {
        if (tt + AHEAD < NT) av[tt + AHEAD] = v_operand<VROW>(vb, tt + AHEAD);
#pragma unroll
        for (uint32_t ct = 0; ct < CT; ++ct) acc[ct][tt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(av[tt], p[ct], acc[ct][tt], 0, 0, 0);
#pragma unroll
        for (uint32_t ct = 0; ct < SC; ++ct) w[ct][tt] = a.score<CAP>(d[ct][tt / 4][tt % 4]);
        __builtin_amdgcn_sched_barrier(0);
      }
      if (i + 1u < n) settle(i + 1u);
    }
  }
  if (ORDER != kContiguous && __ballot(outside)) a.report_pages(pl, b, from, from + n, 1u);
  float sum[CT];
  bool bad = false;
#pragma unroll
  for (uint32_t ct = 0; ct < CT; ++ct) {
    float z = 0.f;
    if (ct < SC) {
      sum[ct] = col_sum(l[ct]);
      z = sum[ct] - sum[ct];
    }
#pragma unroll
    for (uint32_t tt = 0; tt < NT; ++tt) z = not_finite(z, acc[ct][tt]);
    bad |= live[ct] && z != 0.f;
  }
  if constexpr (OWN) st.f[n & 1u][wave][lane] = sum[0];  // (the last step's are in the other half)
  if (__syncthreads_or(bad)) {
    slow_block<HD>(a, pl, b, from, from + n, [&](float(&w)[8]) { w[0] = a.score<CAP>(w[0]); });
    return;
  }
  if constexpr (OWN) sum[1] = st.f[n & 1u][wave ^ 4u][lane];
#pragma unroll
  for (uint32_t ct = 0; ct < CT; ++ct) {
    if (row[ct] >= rows_here) continue;
    if (pl.splits > 1) {
#pragma unroll
      for (uint32_t tt = 0; tt < NT; ++tt)
        store_part<HD>(a, pl, row[ct], g[ct], qq, 8u * ds + tt, live[ct] ? acc[ct][tt] : f4_t{0.f, 0.f, 0.f, 0.f});
      if (qq == 0 && (OWN ? ct == 0 : ds == 0)) {
        float* o = a.part_at<HD>(pl, row[ct], g[ct]);
        o[HD] = r[ct < SC ? ct : 0];
        o[HD + 1] = live[ct] ? sum[ct] : 0.f;
      }
    } else {
      const float inv = live[ct] && sum[ct] != 0.f ? 1.0f / sum[ct] : 0.f;
#pragma unroll
      for (uint32_t tt = 0; tt < NT; ++tt)
        store_out<HD>(a, j, t0 + row[ct], g[ct], qq, 8u * ds + tt, inv == 0.f ? f4_t{0.f, 0.f, 0.f, 0.f} : acc[ct][tt] * inv);
    }
  }
}
template <int HD, int CT, Cap CAP>
void launch_order(const MaskedRows& a, const dim3& grid, hipStream_t st) {
  if (!a.pages) attn_masked_kernel<HD, CT, CAP, kContiguous><<<grid, 2 * HD, 0, st>>>(a);
  else if (a.page % kTile == 0) attn_masked_kernel<HD, CT, CAP, kWholeTiles><<<grid, 2 * HD, 0, st>>>(a);
  else attn_masked_kernel<HD, CT, CAP, kAnyPages><<<grid, 2 * HD, 0, st>>>(a);
}
// Caps above kPlainCap take one column tile (two do not fit the registers), in one kernel for every order of the cache: they are
// the rare ones. Measured (us; cap 257, then 30): 2048 rows causal, 40 / 8 heads of 128 117, 93; 7 documents in them 41, 38; 500
// rows causal over 4500 keys, 32 / 8 101, 79; 777 over 3778, 16 / 2 of 256 159, 107. A single row over 131072 keys 99.6, 99.5.
template <int HD, int CT>
void launch_chunk(const MaskedRows& a, const dim3& grid, hipStream_t st) {
  if constexpr (CT == 1)
    if (a.form == kAnyCap) return attn_masked_kernel<HD, 1, kAnyCap, kAnyPages><<<grid, 2 * HD, 0, st>>>(a);
  if (a.form == kPlain) launch_order<HD, CT, kPlain>(a, grid, st);
  else launch_order<HD, CT, kNoCap>(a, grid, st);
}

// grid (q_heads, T): one column's splits. Each split's factor first, a thread each; then HD / 4 threads side by side take
// four dims each, of every G-th split.
constexpr uint32_t kMaxSplits = 256;
template <int HD>
__global__ __launch_bounds__(256) void attn_masked_join_kernel(MaskedArgs a) {
  constexpr uint32_t G = 256 / (HD / 4);
  __shared__ float factor[kMaxSplits], most[4], total[4];
  __shared__ __align__(16) f4_t sums[G][HD / 4];
  const uint32_t h = blockIdx.x, t = blockIdx.y, i = threadIdx.x, lane = i & 63u, wave = i >> 6;
  const float* p = a.part + (size_t)(t * a.q_heads + h) * a.splits * (HD + 4);
  float r = kNoKey, l = 0.f;
  if (i < a.splits) {
    r = p[i * (HD + 4) + HD];
    l = p[i * (HD + 4) + HD + 1];
  }
  if (l == 0.f) r = kNoKey;  // (no key of the row in that part)
  const float m = wave_max(r);
  if (lane == 0) most[wave] = m;
  __syncthreads();
  const float f = l == 0.f ? 0.f : __builtin_amdgcn_exp2f(r - fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3])));
  if (i < a.splits) factor[i] = f;
  const float sum = wave_sum(l * f);
  if (lane == 0) total[wave] = sum;
  __syncthreads();
  const uint32_t g = i / (HD / 4), d = i % (HD / 4);
  f4_t v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (uint32_t s = g; s < a.splits; s += G) {
    const float w = factor[s];
    const f4_t x = *reinterpret_cast<const f4_t*>(p + s * (HD + 4) + 4u * d);
#pragma unroll
    for (uint32_t e = 0; e < 4; ++e) v[e] = __builtin_fmaf(x[e], w, v[e]);
  }
  sums[g][d] = v;
  __syncthreads();
  if (i >= HD / 4) return;
#pragma unroll
  for (uint32_t k = 1; k < G; ++k) v += sums[k][d];
  const float all = (total[0] + total[1]) + (total[2] + total[3]), inv = all == 0.f ? 0.f : 1.0f / all;
  const u2_t o = {(uint32_t)act_enc(v[0] * inv, a.act) | ((uint32_t)act_enc(v[1] * inv, a.act) << 16),
                  (uint32_t)act_enc(v[2] * inv, a.act) | ((uint32_t)act_enc(v[3] * inv, a.act) << 16)};
  *reinterpret_cast<h4_any*>(a.out + ((size_t)t * a.q_heads + h) * HD + 4u * d) = o;
}

// The same for few splits: HD / 4 threads take a column, each four dims of all its splits; several columns per work-group.
constexpr uint32_t kFewSplits = 8;
template <int HD>
__global__ __launch_bounds__(256) void attn_masked_join_few_kernel(MaskedArgs a, uint32_t columns) {
  constexpr uint32_t C = 256 / (HD / 4);
  const uint32_t c = blockIdx.x * C + threadIdx.x / (HD / 4), d = threadIdx.x % (HD / 4);
  if (c >= columns) return;
  const float* p = a.part + (size_t)c * a.splits * (HD + 4);
  f4_t v[kFewSplits];
  float r[kFewSplits], l[kFewSplits], top = kNoKey;
#pragma unroll
  for (uint32_t s = 0; s < kFewSplits; ++s) {
    const float* q = p + (s < a.splits ? s : 0u) * (HD + 4);
    v[s] = *reinterpret_cast<const f4_t*>(q + 4u * d);
    r[s] = q[HD];
    l[s] = s < a.splits ? q[HD + 1] : 0.f;
  }
#pragma unroll
  for (uint32_t s = 0; s < kFewSplits; ++s) top = l[s] == 0.f ? top : fmaxf(top, r[s]);
  f4_t o = {0.f, 0.f, 0.f, 0.f};
  float sum = 0.f;
#pragma unroll
  for (uint32_t s = 0; s < kFewSplits; ++s) {
    const float f = l[s] == 0.f ? 0.f : __builtin_amdgcn_exp2f(r[s] - top);  // (no key of the row in that part)
    sum = __builtin_fmaf(l[s], f, sum);
#pragma unroll
    for (uint32_t e = 0; e < 4; ++e) o[e] = __builtin_fmaf(v[s][e], f, o[e]);
  }
  const float inv = sum == 0.f ? 0.f : 1.0f / sum;
  const u2_t h = {(uint32_t)act_enc(o[0] * inv, a.act) | ((uint32_t)act_enc(o[1] * inv, a.act) << 16),
                  (uint32_t)act_enc(o[2] * inv, a.act) | ((uint32_t)act_enc(o[3] * inv, a.act) << 16)};
  *reinterpret_cast<h4_any*>(a.out + (size_t)c * HD + 4u * d) = h;
}

// The launch: the few-rows kernel up to 16 columns, else the chunk's with CT column tiles, and the parts that the keys are
// split in.
//   few: as many parts as fill the CUs (two work-groups each at rows of 128, one at 256), of 128 keys at least. Measured
//   (us): one row, 40 / 8 heads of 128, 4099 keys 17.7 / 13.5 / 12.0 / 11.8 / 11.8 in 4 / 8 / 16 / 32 / 64 parts; 131072 keys
//   97 / 99 / 102 / 106 in 32 / 64 / 128 / 256; 16 / 2 heads of 256, 65536 keys 40 / 34 / 42 in 64 / 128 / 256.
//   chunk: the least modelled time over both CT and the parts s, in us. With `same` keys that all rows see and up to `own` keys
//   more, a work-group has between same / 32 and (same + own) / 32 tiles:
//     the longest, start + most / s tau, or all of them over the CUs, rounds (start + mean / s tau), and for s > 1
//     join = 3 + T q_heads s (head_dim + 4) 8 bytes at 3.5 TB/s
//   with cap the work-groups that a CU holds, tau a tile's time with that many on it, and rounds between w / (256 cap), where
//   short work-groups fill up behind long ones, and the next whole number, where all are alike. What the rows see is the
//   device's. Without `lo` the model takes them for the last T of the cache and causal (own = T). With it (documents, a
//   window) they see less, how much is not known: the least product of that time and the one at own = 512 behind the
//   prefix, so that neither is far from its best, with no more parts than the first's. Measured
//   (us; CT 1 then 2, in 1 / 2 / 3 / 4 parts): 500 rows over 4500 keys, 32 / 8 heads of 128: 105 / 84 / 80 / 82, 140 / 84 / 79 / 71;
//   777 over 3778, 16 / 2 of 256: 128 / 128 / 134 / 139, 172 / 104 / 125 / 112 (104 in 5); 2048 over 2048, 40 / 8 of 128:
//   99 / 127, 81 / 112, 16 / 2 of 256: 85 / 115, 100 / 94; 333 over 333, 40 / 8 of 128: 14 / 19 / 20, 20 / 21 / 23; 20 over 4020:
//   87 / 49 / 35 / 29 (16 parts 16), 126 / 69 / 49 / 40. With `lo`, over 45 shapes (2 to 12 documents, windows of 256 and
//   1024) 3 % off the best on average, 27 % by the causal time alone: 2048 rows, 12 documents, 16 / 16 heads of 128 20.2 us (43.8 in
//   3 parts of CT 2), 1000 rows behind 4000, 3 documents, 40 / 8 23.5 (45.1).
struct Pick {
  bool few;
  uint32_t ct, rows, splits;
};
constexpr uint32_t kCus = 256;
// A chunk's columns times its parts, each of at least four tiles: so many in a workspace at most (138 MB at rows of 128). Where more
// would be chosen the work-groups fill the CUs many times over without them: up to 3000 rows over 16384 keys the limit is never met.
constexpr uint32_t kMostColumns = 1u << 18;
uint32_t most_parts(uint32_t keys) { return std::min(64u, std::max(1u, (keys + kTile - 1u) / kTile / 4u)); }
Pick pick(uint32_t T, uint32_t keys, uint32_t kv_heads, uint32_t gqa, uint32_t hd, const mi_attn_mask* mask = nullptr) {
  Pick p{gqa <= 16 && (uint64_t)T * gqa <= 16, 1, 0, 1};
  if (p.few) {
    p.rows = 16u / gqa;
    const uint32_t slots = hd == 128 ? 2 * kCus : kCus;
    p.splits = std::max(1u, std::min({slots / kv_heads, (keys + 127u) / 128u, kMaxSplits}));
    return p;
  }
  static constexpr double kTau[2][2][3] = {{{0.73, 1.15, 1.53}, {1.05, 1.45, 1.45}}, {{1.2, 1.2, 1.2}, {1.5, 1.5, 1.5}}};
  static constexpr double kStart[2][2] = {{4.0, 8.0}, {6.0, 6.0}};
  auto time = [&](uint32_t ct, uint32_t s, uint32_t same, uint32_t own) {
    const uint32_t rows = 64u * ct / gqa, cap = hd == 128 ? 4u - ct : 1u;
    const double most = (same + own + kTile - 1u) / kTile, mean = most - own / (2.0 * kTile), alike = (double)same / (same + own);
    const uint64_t w = (uint64_t)kv_heads * ((T + rows - 1u) / rows) * s;
    const double tau = kTau[hd == 256][ct - 1][std::min<uint64_t>((w + kCus - 1u) / kCus, cap) - 1u], start = kStart[hd == 256][ct - 1];
    const double turns = (double)w / (kCus * cap), whole = (double)((w + kCus * cap - 1u) / (kCus * cap));
    const double us = std::max(start + most / s * tau, (turns + (whole - turns) * alike) * (start + mean / s * tau));
    return s == 1 ? us : us + 3.0 + (double)T * (kv_heads * gqa) * s * (hd + 4) * 8.0 / 3.5e6;
  };
  const uint32_t own = std::min(T, keys);
  auto choose = [&](uint32_t most, auto cost) {
    double least = 1e300;
    for (uint32_t ct = 1; ct <= 2; ++ct)
      for (uint32_t s = 1; s <= most; ++s) {
        const double c = cost(ct, s);
        if (c >= least) continue;
        least = c;
        p = Pick{false, ct, 64u * ct / gqa, s};
      }
  };
  const uint32_t parts = std::min(most_parts(keys), std::max(1u, kMostColumns / (T * kv_heads * gqa)));
  choose(parts, [&](uint32_t ct, uint32_t s) { return time(ct, s, keys - own, own); });
  if (mask && mask->lo) {
    const uint32_t same = std::min(mask->prefix, keys), near = std::min(keys - same, 512u);
    choose(p.splits, [&](uint32_t ct, uint32_t s) { return time(ct, s, keys - own, own) * time(ct, s, same, near); });
  }
  return p;
}
size_t part_bytes(uint32_t columns, uint32_t hd) { return (size_t)columns * (hd + 4) * 4; }
bool shape_ok(const mi_attn_shape* s) {
  return s && s->kv_heads && s->q_heads && s->q_heads % s->kv_heads == 0 && s->q_heads / s->kv_heads <= 64 &&
         s->q_heads <= 1024 && (s->head_dim == 128 || s->head_dim == 256);
}

}  // namespace
}  // namespace mi

using namespace mi;

extern "C" {

// What a call of up to T rows over up to kv_len keys takes at most: of as many rows as the few-rows kernel takes, or of a chunk.
size_t mi_attn_masked_ws(uint32_t T, uint32_t kv_len, const mi_attn_shape* shape) {
  if (T == 0 || T > kMaxRows || kv_len == 0 || kv_len > kMaxKeys || !shape_ok(shape)) return 0;
  const uint32_t gqa = shape->q_heads / shape->kv_heads, few = std::min(T, 16u / gqa), parts = most_parts(kv_len);
  uint32_t columns = 0;
  if (few) {
    const Pick p = pick(few, kv_len, shape->kv_heads, gqa, shape->head_dim);
    if (p.splits > 1) columns = few * shape->q_heads * p.splits;
  }
  if (T > few && parts > 1)
    columns = std::max(columns, (uint32_t)std::min<uint64_t>((uint64_t)T * shape->q_heads * parts, kMostColumns));
  return part_bytes(columns, shape->head_dim);
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
  if (T == 0 || T > kMaxRows || kv_len == 0 || kv_len > kMaxKeys) return mi_fail(MI_ERR_SHAPE, "attn_masked: T 1..65535, kv_len 1..2^30");
  if (pages && (page == 0 || n_pages == 0)) return mi_fail(MI_ERR_ARG, "attn_masked: page size or page count 0");
  if (pages && (uint64_t)page * n_pages > 0xFFFFFFFFull) return mi_fail(MI_ERR_SHAPE, "attn_masked: above 2^32 cache rows");
  if (row_stride % 8 || head_stride % 8) return mi_fail(MI_ERR_ARG, "attn_masked: KV strides must keep 8-element alignment");
  auto off = [](const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1u)) != 0; };
  if (off(kv_k, 16) || off(kv_v, 16) || off(attn_q, 4) || off(attn_out, 2))
    return mi_fail(MI_ERR_ARG, "attn_masked: misaligned pointer (K and V 16 bytes)");
  if (off(pages, 4) || off(mask->lo, 4) || off(mask->hi, 4) || off(mask->pos, 4) || off(mask->slopes, 4) || off(flag, 4))
    return mi_fail(MI_ERR_ARG, "attn_masked: misaligned pages, spans, positions, slopes or flag (4 bytes)");
  if (!(mask->cap == 0.f || (mask->cap >= 1e-20f && mask->cap <= 1e30f)))  // (2 c / cap stays finite)
    return mi_fail(MI_ERR_ARG, "attn_masked: cap is 0 (none) or between 1e-20 and 1e30");
  if (!mask->pos && (uint64_t)mask->pos0 + T > 1u << 31)  // (distances are int32)
    return mi_fail(MI_ERR_SHAPE, "attn_masked: positions are below 2^31");
  const uint32_t gqa = shape->q_heads / shape->kv_heads;
  Pick p = pick(T, kv_len, shape->kv_heads, gqa, shape->head_dim, mask);
  const Cap form = mask->cap == 0.f ? kNoCap : mask->cap <= kPlainCap ? kPlain : kAnyCap;
  if (form == kAnyCap && !p.few) p = Pick{false, 1, 64u / gqa, p.splits};
  const size_t need = p.splits == 1 ? 0 : part_bytes(T * shape->q_heads * p.splits, shape->head_dim);
  if (need && (!ws || off(ws, 16) || ws_bytes < need))
    return mi_fail(MI_ERR_ARG, "attn_masked: the workspace is null, misaligned (16 bytes) or below mi_attn_masked_ws");
  MaskedRows a{};
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
  a.form = form;
  hipStream_t st = (hipStream_t)stream;
  const dim3 grid(shape->kv_heads, (T + p.rows - 1u) / p.rows, p.splits);
  const bool narrow = shape->head_dim == 128;
  if (p.few) {
    if (narrow) attn_rows_few_kernel<128><<<grid, 256, 0, st>>>(a);
    else attn_rows_few_kernel<256><<<grid, 256, 0, st>>>(a);
  } else if (narrow) {
    if (p.ct == 2) launch_chunk<128, 2>(a, grid, st);
    else launch_chunk<128, 1>(a, grid, st);
  } else {
    if (p.ct == 2) launch_chunk<256, 2>(a, grid, st);
    else launch_chunk<256, 1>(a, grid, st);
  }
  const uint32_t columns = T * shape->q_heads;
  if (p.splits > kFewSplits) {
    if (narrow) attn_masked_join_kernel<128><<<dim3(shape->q_heads, T), 256, 0, st>>>(a);
    else attn_masked_join_kernel<256><<<dim3(shape->q_heads, T), 256, 0, st>>>(a);
  } else if (p.splits > 1) {
    if (narrow) attn_masked_join_few_kernel<128><<<(columns + 7u) / 8u, 256, 0, st>>>(a, columns);
    else attn_masked_join_few_kernel<256><<<(columns + 3u) / 4u, 256, 0, st>>>(a, columns);
  }
  return mi_hip((int)hipGetLastError(), "attn_masked");
}

}  // extern "C"
