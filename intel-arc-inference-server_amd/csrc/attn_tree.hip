// attn_tree.hip - attention of the rows of several sequences over their own pages of the f16 cache: a token each, a tree of
// drafted tokens each, or stretches of prompts.
//
// Row i of sequence b (its node i) stands behind cached_b keys and sees them all, and of the step's own keys cached_b + c those
// whose bit c is set in its mask: the ancestors of a node and the node itself; without masks c <= i. With y_j = scale q . k_j
// log2(e):  out = sum_j 2^y_j v_j / sum_j 2^y_j, zeros for a row that sees nothing.
// The kernels, and how their softmax and its roundings go, are attn_rows.h's.
//
// How the work is dealt out: a sequence's rows are cut into blocks of `rows`, its 32-key tiles into parts of `per` tiles, the same
// for all sequences (a sequence's parts then as even as may be). A block, a part and a kv head are an item, and a work-group's.
// Lengths are the device's: every wave reads them all, forms `per` and finds its item by itself. Items that read the same keys (a sequence's blocks) follow one another
// and run on one XCD. Sequences of several parts leave sums, which a second launch joins.
#include <algorithm>

#include "attn_rows.h"
#include "mi_capi_internal.h"

namespace mi {
namespace {

constexpr uint32_t kMaxRows = 65535, kMaxKeys = 1u << 30, kMaxSequences = 1024, kMaxWords = 64, kMaxSplits = 1024, kXcds = 8, kNone = 0xFFFFFFFFu;
constexpr uint32_t kNoTree = 0x7FFFFFFFu;  // a column's `first` where it is none: every key lies before it

struct TreeArgs {
  const float* q;  // [T][q_heads][HD]
  const uint16_t *k, *v;
  const uint32_t *tables, *row_start, *cached, *mask;
  uint16_t* out;  // [T][q_heads][HD]
  u4_t* info;     // [T]: a row's first item, its sequence's blocks and parts, its place in the block
  float* part;    // items of several parts: see part_at
  uint32_t* flag;
  size_t row_stride, head_stride;
  uint32_t table_stride, page, page_shift, n_pages, kv_len, T, sequences, words, q_heads, kv_heads, gqa, rows, columns, slots,
      share, least, most_blocks, act;
  float c;  // y = c q . k
};

// A sequence's rows, keys and tiles, whatever the arrays hold.
struct Sequence {
  uint32_t start, rows, cached, keys, blocks, tiles;
};
__device__ __forceinline__ Sequence sequence(const TreeArgs& a, uint32_t b) {
  Sequence s{0u, 0u, 0u, 0u, 0u, 0u};
  if (b < a.sequences) {
    s.start = a.row_start[b];
    const uint32_t end = min(a.row_start[b + 1u], a.T);
    s.cached = min(a.cached[b], a.kv_len);
    s.rows = end > s.start ? end - s.start : 0u;
    s.keys = s.cached + min(s.rows, a.kv_len - s.cached);
    s.blocks = (s.rows + a.rows - 1u) / a.rows;
    s.tiles = s.rows ? (s.keys + kTile - 1u) / kTile : 0u;
  }
  return s;
}

struct TreeRows : TreeArgs {
  struct Place {
    uint32_t j, t0, rows, split, splits;
    uint32_t b, own, cached, keys, per, part;  // the sequence, its index of the first row, where the part's sums go
  };
  struct Block {
    uint32_t last, n, free, base;  // free: so many keys every row of the block sees
    const uint32_t* pages;
    __device__ __forceinline__ uint32_t key(uint32_t i) const { return kTile * i; }
    __device__ __forceinline__ uint32_t within(uint32_t, uint32_t k) const { return min(k, last); }
  };
  struct Column {
    const uint32_t* bits;
    uint32_t own, first, count;  // its index, the first of the step's own keys and how many they are
    bool live;
  };
  static constexpr bool kMayIdle = true;

  static __device__ __forceinline__ uint32_t parts(const Sequence& s, uint32_t per) { return (s.tiles + per - 1u) / per; }
  // Tiles of a part at most. With `even` tiles in each of the work-groups that run at once, and parts of `per` tiles that make `items`
  // items, the call lasts per + 3 where all run at once, else even + per / 2 + 3 items / slots (in tiles; 3: an item's start).
  // Few sequences of uneven lengths are near `even` in one round or none: of the candidates the least is taken. None is below
  // total / share, so there are no more items than share and one for each block.
  __device__ __forceinline__ uint32_t part_tiles(const Sequence& first, float total) const {
    const uint32_t lane = threadIdx.x & 63u;
    constexpr uint32_t N = 8;
    constexpr float kOf[N] = {2.f, 1.5f, 1.25f, 1.125f, 1.f, 0.5f, 0.33f, 0.25f};
    const float even = total * (float)kv_heads / (float)slots;
    float items[N];
    uint32_t per[N];
#pragma unroll
    for (uint32_t n = 0; n < N; ++n) {
      per[n] = max(least, (uint32_t)fminf(fmaxf(even * kOf[n], total * 1.0001f / (float)share), (float)kMaxKeys) + 1u);
      items[n] = 0.f;
    }
    for (uint32_t b = 0; b < sequences; b += 64u) {
      const Sequence s = b ? sequence(*this, b + lane) : first;
#pragma unroll
      for (uint32_t n = 0; n < N; ++n)
        items[n] += (float)s.blocks * ceilf((float)s.tiles * __builtin_amdgcn_rcpf((float)per[n]));
    }
    uint32_t best = 0;
    float cost = INFINITY;
#pragma unroll
    for (uint32_t n = 0; n < N; ++n) {
      const float turns = wave_sum(items[n]) * (float)kv_heads / (float)slots;
      const float c = turns <= 1.f ? (float)per[n] + 3.f : even + 0.5f * (float)per[n] + 3.f * turns;
      if (c < cost) {
        cost = c;
        best = per[n];
      }
    }
    return best;
  }
  __device__ __forceinline__ Place place(bool) const {
    const uint32_t lane = threadIdx.x & 63u;
    auto plus = [](uint32_t x, uint32_t y) { return x + y; };
    Place p{};
    if (sequences == 1u) {
      const Sequence s = sequence(*this, 0u);
      p.per = max(least, max(s.blocks, s.tiles) < 65536u ? (s.blocks * s.tiles + share - 1u) / share
                                                         : (uint32_t)((float)s.blocks * (float)s.tiles * 1.0001f / (float)share) + 1u);
      const uint32_t n = parts(s, p.per), item = item_of(s.blocks * n * kv_heads);
      if (item == kNone) return p;
      return inside(p, s, 0u, n, item, 0u);
    }
    Sequence s = sequence(*this, lane);
    float total = (float)s.blocks * (float)s.tiles, blocks = (float)s.blocks;
    for (uint32_t b = 64u; b < sequences; b += 64u) {
      const Sequence o = sequence(*this, b + lane);
      total += (float)o.blocks * (float)o.tiles;
      blocks += (float)o.blocks;
    }
    if (wave_sum(blocks) > (float)most_blocks) {  // (sequences that overlap: their items would be more than are counted with)
      if (flag) *flag = MI_STATUS_BAD_ROWS;
      return p;
    }
    p.per = part_tiles(s, wave_sum(total));
    uint32_t items = s.blocks * parts(s, p.per);
    for (uint32_t b = 64u; b < sequences; b += 64u) {
      const Sequence o = sequence(*this, b + lane);
      items += o.blocks * parts(o, p.per);
    }
    uint32_t item = item_of(wave_fold(items, plus) * kv_heads);
    if (item == kNone) return p;
    uint32_t part = 0;
    for (uint32_t b0 = 0; b0 < sequences; b0 += 64u) {
      if (b0) s = sequence(*this, b0 + lane);
      const uint32_t n = parts(s, p.per), mine = s.blocks * n * kv_heads;
      uint32_t sum = mine;  // of the lanes up to this one
#pragma unroll
      for (uint32_t d = 1; d < 64u; d *= 2) {
        const uint32_t o = (uint32_t)__shfl_up((int)sum, d, 64);
        sum += lane >= d ? o : 0u;
      }
      const uint64_t behind = __ballot(sum > item);
      const uint32_t found = behind ? (uint32_t)__builtin_ctzll(behind) : 64u;
      part += wave_fold(lane < found && n > 1u ? mine : 0u, plus);
      if (found == 64u) {
        item -= (uint32_t)__builtin_amdgcn_readlane((int)sum, 63);
        continue;
      }
      auto of = [&](uint32_t v) { return (uint32_t)__builtin_amdgcn_readlane((int)v, (int)found); };
      const Sequence f = {of(s.start), of(s.rows), of(s.cached), of(s.keys), of(s.blocks), of(s.tiles)};
      return inside(p, f, b0 + found, of(n), item - of(sum - mine), part);
    }
    return p;
  }
  // This work-group's of `items` items: XCD x (every eighth work-group is its) has those from x / 8 of them on.
  __device__ __forceinline__ uint32_t item_of(uint32_t items) const {
    const uint32_t each = (items + kXcds - 1u) / kXcds, at = blockIdx.x / kXcds, item = (blockIdx.x % kXcds) * each + at;
    return at < each && item < items ? item : kNone;
  }
  // The place of item `item` of sequence b, of n parts, whose first item's sums are number `part`.
  __device__ __forceinline__ Place inside(Place p, const Sequence& s, uint32_t b, uint32_t n, uint32_t item, uint32_t part) const {
    const uint32_t each = s.blocks * kv_heads, split = item / each, rest = item - split * each;
    p.j = rest / s.blocks;
    p.own = (rest - p.j * s.blocks) * rows;
    p.rows = min(rows, s.rows - p.own);
    p.t0 = s.start + p.own;
    p.split = split;
    p.splits = n;
    p.b = b;
    p.cached = s.cached;
    p.keys = s.keys;
    p.part = part + item;
    if (split == 0u && p.j == 0u && threadIdx.x < p.rows)
      info[p.t0 + threadIdx.x] = u4_t{p.part, s.blocks, p.splits, threadIdx.x};
    return p;
  }
  __device__ __forceinline__ Block block(const Place& p) const {
    Block b{};
    // (without masks a block sees no key behind its last row's)
    const uint32_t end = mask ? p.keys : min(p.keys, p.cached + p.own + p.rows);
    b.last = end - 1u;
    b.n = (end + kTile - 1u) / kTile;
    b.free = mask ? p.cached : min(p.keys, p.cached + p.own + 1u);
    b.base = tables ? 0u : p.b * table_stride;
    b.pages = tables ? tables + (size_t)p.b * table_stride : nullptr;
    return b;
  }
  __device__ __forceinline__ uint32_t part_begin(const Place& p, const Block& b, uint32_t split) const {
    return (uint32_t)((uint64_t)b.n * split / p.splits);
  }
  __device__ __forceinline__ Column column(const Place& p, const Block& b, uint32_t row, uint32_t) const {
    Column c{nullptr, p.own + row, p.cached, p.keys - p.cached, row < p.rows};
    if (mask) c.bits = mask + (size_t)(p.t0 + min(row, p.rows - 1u)) * words;
    if (!c.live) c.first = kNoTree;  // (it sees every key, so no tile is masked for it; what it sums is not stored)
    return c;
  }
  __device__ __forceinline__ bool masked(const Block& b, uint32_t key) const { return key + kTile > b.free; }
  // bits 32 i .. of which of the step's own keys the column sees
  __device__ __forceinline__ uint32_t word(const Column& c, int32_t i) const {
    if (i < 0) return 0xFFFFFFFFu;
    const uint32_t seen = mask ? c.count : min(c.count, c.own + 1u), from = 32u * (uint32_t)i;
    const uint32_t bits = mask ? ((uint32_t)i < words ? c.bits[i] : 0u) : 0xFFFFFFFFu;
    return seen <= from ? 0u : seen - from >= 32u ? bits : bits & ((1u << (seen - from)) - 1u);
  }
  __device__ __forceinline__ bool sees(const Column& c, uint32_t key) const {
    const int32_t n = (int32_t)(key - c.first);
    return (word(c, n >> 5) >> (n & 31)) & 1u;
  }
  template <Cap>
  __device__ __forceinline__ float score(float s) const {
    return s * c;
  }
  __device__ __forceinline__ void scores_by_form(float (&w)[8]) const {
#pragma unroll
    for (uint32_t e = 0; e < 8; ++e) w[e] *= c;
  }
  // -inf for a key that the column does not see, of keys key0 + 16 (e / 4) + e % 4 (e < 8)
  __device__ __forceinline__ void bias_and_mask(const Column& c, uint32_t key0, bool masked, float (&w)[8]) const {
    if (!masked) return;
    const int32_t n = (int32_t)(key0 - c.first), i = n >> 5;
    const uint32_t lo = word(c, i), hi = word(c, i + 1), bits = (uint32_t)(((uint64_t)hi << 32 | lo) >> (n & 31));
#pragma unroll
    for (uint32_t e = 0; e < 8; ++e) w[e] = (bits >> (16u * (e / 4) + e % 4)) & 1u ? w[e] : -INFINITY;
  }
  __device__ __forceinline__ uint32_t first_row(const Block& b, uint32_t key) const { return b.base + key; }
  // the cache row of a key of the sequence; `outside`: its page's entry is not the cache's, and the row is the first page's
  __device__ __forceinline__ uint32_t cache_row(const Block& b, uint32_t key, bool& outside) const {
    if (!b.pages) return b.base + key;
    const uint32_t at = page_shift < 32u ? key >> page_shift : key / page;
    uint32_t pg = b.pages[at];
    if (pg >= n_pages) {
      outside = true;
      pg = 0u;
    }
    return pg * page + (key - at * page);
  }
  __device__ __forceinline__ uint32_t row_of(const Block& b, uint32_t, uint32_t key, bool& outside) const {
    return cache_row(b, min(key, b.last), outside);
  }
  __device__ __forceinline__ void report_pages(const Place&, const Block&, uint32_t, uint32_t, uint32_t) const {
    if (flag) *flag = MI_STATUS_BAD_PAGE;
  }
  template <int HD>
  __device__ __forceinline__ float* part_at(const Place& p, uint32_t row, uint32_t g) const {
    return part + ((size_t)p.part * columns + row * gqa + g) * (HD + 4);
  }
};

// Joins the parts of columns: HD / 4 threads side by side take a column, each four dims of all its parts, eight parts at a time; a
// work-group `C` columns of one row (C 1: all its threads one column's, which then share the parts out).
template <int HD, bool MANY>
__global__ __launch_bounds__(256) void attn_tree_join_kernel(TreeArgs a, uint32_t most) {
  constexpr uint32_t L = HD / 4, G = 256 / L, U = 8;
  const uint32_t t = blockIdx.y, g = threadIdx.x / L, d = threadIdx.x % L;
  const uint32_t h = MANY ? blockIdx.x : blockIdx.x * G + g;
  if (t < a.row_start[0] || t >= min(a.row_start[a.sequences], a.T)) return;  // (uniform: no sequence's row)
  const u4_t info = a.info[t];
  const uint32_t splits = min(info[2], kMaxSplits);
  if (splits < 2u) return;  // (uniform: its work-group stored it)
  if (!MANY && h >= a.q_heads) return;
  const uint32_t j = h / a.gqa, col = info[3] * a.gqa + h % a.gqa;
  auto part = [&](uint32_t s) {  // (within the workspace whatever row_start held)
    return a.part + ((size_t)min(info[0] + (s * a.kv_heads + j) * info[1], most) * a.columns + min(col, a.columns - 1u)) * (HD + 4);
  };
  f4_t o = {0.f, 0.f, 0.f, 0.f};
  float top = kNoKey, sum = 0.f;
  for (uint32_t s0 = MANY ? g : 0u; s0 < splits; s0 += U * (MANY ? G : 1u)) {
    f4_t v[U];
    float r[U], l[U], now = top;
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) {
      const uint32_t s = s0 + u * (MANY ? G : 1u);
      const float* p = part(s < splits ? s : s0);
      v[u] = *as_global(reinterpret_cast<const f4_t*>(p + 4u * d));
      r[u] = *as_global(p + HD);
      l[u] = s < splits ? *as_global(p + HD + 1) : 0.f;
    }
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) now = l[u] == 0.f ? now : fmaxf(now, r[u]);
    const float f = __builtin_amdgcn_exp2f(top - now);
    sum *= f;
    o *= f;
    top = now;
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) {
      const float w = l[u] == 0.f ? 0.f : __builtin_amdgcn_exp2f(r[u] - top);  // (no key of the row in that part)
      sum = __builtin_fmaf(l[u], w, sum);
#pragma unroll
      for (uint32_t e = 0; e < 4; ++e) o[e] = __builtin_fmaf(v[u][e], w, o[e]);
    }
  }
  if constexpr (MANY) {
    __shared__ __align__(16) f4_t sums[G][L];
    __shared__ float tops[G], totals[G];
    sums[g][d] = o;
    if (d == 0) {
      tops[g] = top;
      totals[g] = sum;
    }
    __syncthreads();
    if (g) return;
#pragma unroll
    for (uint32_t n = 1; n < G; ++n) top = fmaxf(top, tops[n]);
    const float f = __builtin_amdgcn_exp2f(tops[0] - top);
    sum *= f;
    o *= f;
#pragma unroll
    for (uint32_t n = 1; n < G; ++n) {
      const float w = __builtin_amdgcn_exp2f(tops[n] - top);
      const f4_t x = sums[n][d];
      sum = __builtin_fmaf(totals[n], w, sum);
#pragma unroll
      for (uint32_t e = 0; e < 4; ++e) o[e] = __builtin_fmaf(x[e], w, o[e]);
    }
  }
  const float inv = sum == 0.f ? 0.f : 1.0f / sum;
  store_out<HD>(a, j, t, h % a.gqa, d % 4u, d / 4u, o * inv);
}

struct Pick {
  bool few;
  uint32_t ct, rows, columns, slots;
};
constexpr uint32_t kCus = 256;
Pick few_rows(uint32_t gqa, uint32_t hd) { return Pick{true, 1, 16u / gqa, 16, (hd == 128 ? 2u : 1u) * kCus}; }
Pick chunk(uint32_t ct, uint32_t gqa, uint32_t hd) {
  return Pick{false, ct, 64u * ct / gqa, 64u * ct, hd == 128 ? (4u - ct) * kCus : kCus};
}
Pick pick(uint32_t T, uint32_t sequences, uint32_t gqa, uint32_t hd) {
  const uint32_t each = (T + sequences - 1u) / sequences * gqa;  // columns
  if (each <= 16u) return few_rows(gqa, hd);
  return chunk(each <= 64u ? 1u : 2u, gqa, hd);
}
// The parts of all sequences at most, one for each block aside: as many as make every work-group that runs at once busy, where there
// are several sequences some times as many.
uint32_t share_of(const Pick& p, uint32_t kv_heads, uint32_t sequences) {
  return std::min(kMaxSplits - 1u, std::max(1u, p.slots * (sequences == 1u ? 1u : p.few ? 4u : 2u) / kv_heads));
}
// The items of sequences of several parts: such a sequence has at most twice tiles / per parts.
size_t part_floats(const Pick& p, uint32_t kv_heads, uint32_t sequences, uint32_t hd) {
  return (size_t)2u * share_of(p, kv_heads, sequences) * kv_heads * p.columns * (hd + 4u);
}
bool shape_ok(const mi_attn_shape* s) {
  return s && s->kv_heads && s->q_heads && s->q_heads % s->kv_heads == 0 && s->q_heads / s->kv_heads <= 64 &&
         s->q_heads <= 1024 && (s->head_dim == 128 || s->head_dim == 256);
}
template <int HD, int CT>
void launch_chunk(const TreeRows& a, uint32_t grid, hipStream_t st) {
  if (!a.tables) attn_rows_kernel<HD, CT, kNoCap, kContiguous><<<grid, 2 * HD, 0, st>>>(a);
  else if (a.page % kTile == 0) attn_rows_kernel<HD, CT, kNoCap, kWholeTiles><<<grid, 2 * HD, 0, st>>>(a);
  else attn_rows_kernel<HD, CT, kNoCap, kAnyPages><<<grid, 2 * HD, 0, st>>>(a);
}

}  // namespace
}  // namespace mi

using namespace mi;

extern "C" {

size_t mi_attn_tree_ws(uint32_t T, uint32_t sequences, const mi_attn_shape* shape) {
  if (T == 0 || T > kMaxRows || sequences == 0 || sequences > kMaxSequences || !shape_ok(shape)) return 0;
  const uint32_t gqa = shape->q_heads / shape->kv_heads, hd = shape->head_dim;
  // the most that any call of up to T rows takes
  size_t floats = gqa <= 16u ? part_floats(few_rows(gqa, hd), shape->kv_heads, 2u, hd) : 0u;
  for (uint32_t ct = 1; ct <= 2; ++ct)
    if (T * gqa > (ct == 1u ? 16u : 64u)) floats = std::max(floats, part_floats(chunk(ct, gqa, hd), shape->kv_heads, 2u, hd));
  return (size_t)T * sizeof(u4_t) + floats * 4u;
}

int mi_attn_tree(const float* attn_q, const uint16_t* kv_k, const uint16_t* kv_v, size_t row_stride, size_t head_stride,
                 uint32_t T, const mi_attn_shape* shape, const mi_attn_batch* batch, void* ws, size_t ws_bytes,
                 uint16_t* attn_out, uint32_t* flag, void* stream) {
  if (!attn_q || !kv_k || !kv_v || !attn_out || !shape || !batch) return mi_fail(MI_ERR_ARG, "attn_tree: null pointer");
  if (!batch->row_start || !batch->cached) return mi_fail(MI_ERR_ARG, "attn_tree: row_start and cached are needed");
  if (!shape_ok(shape))
    return mi_fail(MI_ERR_SHAPE, "attn_tree: head_dim 128 or 256, q_heads a multiple of kv_heads, up to 64 of them each");
  if (shape->gated) return mi_fail(MI_ERR_SHAPE, "attn_tree: gated shapes are not supported");
  if (shape->act > 1) return mi_fail(MI_ERR_ARG, "attn_tree: act is 0 or 1");
  const uint32_t kv_len = batch->kv_len, n = batch->sequences;
  if (T == 0 || T > kMaxRows || kv_len == 0 || kv_len > kMaxKeys || n == 0 || n > kMaxSequences)
    return mi_fail(MI_ERR_SHAPE, "attn_tree: T 1..65535, kv_len 1..2^30, 1..1024 sequences");
  if (batch->tables) {
    if (batch->page == 0 || batch->n_pages == 0) return mi_fail(MI_ERR_ARG, "attn_tree: page size or page count 0");
    if ((uint64_t)batch->page * batch->n_pages > 0xFFFFFFFFull) return mi_fail(MI_ERR_SHAPE, "attn_tree: above 2^32 cache rows");
    if ((uint64_t)batch->table_stride * batch->page < kv_len)
      return mi_fail(MI_ERR_ARG, "attn_tree: table_stride pages hold fewer than kv_len keys");
  } else {
    if (n > 1 && batch->table_stride < kv_len) return mi_fail(MI_ERR_ARG, "attn_tree: table_stride rows hold fewer than kv_len keys");
    if ((uint64_t)batch->table_stride * (n - 1u) + kv_len > 0xFFFFFFFFull)
      return mi_fail(MI_ERR_SHAPE, "attn_tree: above 2^32 cache rows");
  }
  if (batch->mask ? batch->words == 0 || batch->words > kMaxWords : batch->words != 0)
    return mi_fail(MI_ERR_ARG, "attn_tree: 1..64 words go with masks, 0 with none");
  if (row_stride % 8 || head_stride % 8) return mi_fail(MI_ERR_ARG, "attn_tree: KV strides must keep 8-element alignment");
  auto off = [](const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1u)) != 0; };
  if (off(kv_k, 16) || off(kv_v, 16) || off(attn_q, 4) || off(attn_out, 2))
    return mi_fail(MI_ERR_ARG, "attn_tree: misaligned pointer (K and V 16 bytes)");
  if (off(batch->row_start, 4) || off(batch->cached, 4) || off(batch->tables, 4) || off(batch->mask, 4) || off(flag, 4))
    return mi_fail(MI_ERR_ARG, "attn_tree: misaligned row_start, cached, tables, mask or flag (4 bytes)");
  const uint32_t gqa = shape->q_heads / shape->kv_heads;
  const Pick p = pick(T, n, gqa, shape->head_dim);
  const size_t floats = part_floats(p, shape->kv_heads, n, shape->head_dim);
  if (!ws || off(ws, 16) || ws_bytes < (size_t)T * sizeof(u4_t) + floats * 4u)
    return mi_fail(MI_ERR_ARG, "attn_tree: the workspace is null, misaligned (16 bytes) or below mi_attn_tree_ws");
  TreeRows a{};
  a.q = attn_q;
  a.k = kv_k;
  a.v = kv_v;
  a.tables = batch->tables;
  a.row_start = batch->row_start;
  a.cached = batch->cached;
  a.mask = batch->mask;
  a.out = attn_out;
  a.info = static_cast<u4_t*>(ws);
  a.part = reinterpret_cast<float*>(a.info + T);
  a.flag = flag;
  a.row_stride = row_stride;
  a.head_stride = head_stride;
  a.table_stride = n > 1 || batch->tables ? batch->table_stride : 0u;
  a.page = batch->page;
  a.page_shift = batch->tables && (batch->page & (batch->page - 1u)) == 0 ? (uint32_t)__builtin_ctz(batch->page) : 32u;
  a.n_pages = batch->n_pages;
  a.kv_len = kv_len;
  a.T = T;
  a.sequences = n;
  a.words = batch->words;
  a.q_heads = shape->q_heads;
  a.kv_heads = shape->kv_heads;
  a.gqa = gqa;
  a.rows = p.rows;
  a.columns = p.columns;
  a.slots = p.slots;
  a.share = share_of(p, shape->kv_heads, n);
  a.least = 4;
  a.act = shape->act;
  a.c = shape->scale * kLog2e;
  hipStream_t st = (hipStream_t)stream;
  a.most_blocks = T / p.rows + n;
  // as many work-groups as there are items at most: share and one more for each block, of each kv head, no more than the blocks have
  // parts of the least size
  const uint64_t least_parts = ((uint64_t)kv_len + a.least * kTile - 1u) / (a.least * kTile);
  const uint32_t items = shape->kv_heads * (uint32_t)std::min<uint64_t>(a.share + a.most_blocks, a.most_blocks * least_parts);
  const uint32_t grid = (items + kXcds - 1u) / kXcds * kXcds;
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
  if (kv_len > a.least * kTile) {  // (there may be several parts)
    const uint32_t most = 2u * a.share * shape->kv_heads - 1u;
    if (a.most_blocks * 8u <= a.share) {
      if (narrow) attn_tree_join_kernel<128, true><<<dim3(shape->q_heads, T), 256, 0, st>>>(a, most);
      else attn_tree_join_kernel<256, true><<<dim3(shape->q_heads, T), 256, 0, st>>>(a, most);
    } else {
      if (narrow) attn_tree_join_kernel<128, false><<<dim3((shape->q_heads + 7u) / 8u, T), 256, 0, st>>>(a, most);
      else attn_tree_join_kernel<256, false><<<dim3((shape->q_heads + 3u) / 4u, T), 256, 0, st>>>(a, most);
    }
  }
  return mi_hip((int)hipGetLastError(), "attn_tree");
}

}  // extern "C"
