// attn_tree.hip - attention of the rows of several sequences over their own pages of the f16 cache: a token each, a tree of
// drafted tokens each, or stretches of prompts.
//
// Row i of sequence b (its node i) stands behind cached_b keys and sees them all, and of the step's own keys cached_b + c those
// whose bit c is set in its mask: the ancestors of a node and the node itself; without masks c <= i. With y_j = scale q . k_j
// log2(e):  out = sum_j 2^y_j v_j / sum_j 2^y_j, zeros for a row that sees nothing.
// The kernels, and how their softmax and its roundings go, are attn_rows.h's.
//
// How the work is dealt out: a sequence's rows are cut into blocks of `rows`, its 32-key tiles into parts of `per` tiles, the same
// for all sequences (a sequence's parts then as even as may be). A block, a part and a kv head are an item; as many work-groups as run
// at once take them. Lengths are the device's: every wave reads them all, forms `per` and finds its items by itself. The items
// of a kv head follow one another, those that read the same keys (a sequence's blocks) side by side, and an XCD takes an even stretch
// of all: with 8 kv heads one head, so that the XCDs' loads are alike whatever the lengths are. Sequences of several parts leave
// sums, which a second launch joins. Code is short here and its loops are not unrolled: every work-group fetches it anew (sixteen
// candidates of `per` in unrolled code took 5 us more than eight; the 64 of part_tiles are a lane each).
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
      share, least, act;
  float c;  // y = c q . k
};

// A sequence's rows, keys and tiles, whatever the arrays hold.
struct Sequence {
  uint32_t start, rows, cached, keys, blocks, tiles;
  bool falls;  // it ends before it starts: where none does, no two share a row
};
__device__ __forceinline__ Sequence sequence(const TreeArgs& a, uint32_t b) {
  Sequence s{0u, 0u, 0u, 0u, 0u, 0u, false};
  if (b < a.sequences) {
    s.start = a.row_start[b];
    const uint32_t next = a.row_start[b + 1u], end = min(next, a.T);
    s.falls = next < s.start;
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
    uint32_t b, own, cached, keys, part;  // the sequence, its index of the first row, where the part's sums go
  };
  struct Block {
    uint32_t last, n, free, base;  // free: so many keys every row of the block sees
    const uint32_t* pages;
    __device__ __forceinline__ uint32_t key(uint32_t i) const { return kTile * i; }
  };
  struct Column {
    const uint32_t* bits;
    uint32_t own, first, count;  // its index, the first of the step's own keys and how many they are
    bool live;
  };
  static constexpr bool kItems = true;

  static __device__ __forceinline__ uint32_t parts(const Sequence& s, uint32_t per) { return (s.tiles + per - 1u) / per; }
  // Tiles of a part at most, for several sequences of `total` tiles in all blocks. With `even` tiles in each of the work-groups that
  // run at once, and parts of `per` tiles that make `items` items, the call lasts per + 3 where all run at once, else
  // even + per / 2 + 3 items / slots (in tiles; 3: an item's start). Few sequences of uneven lengths are near `even` in one round or
  // none: of 64 candidates, a lane each, the least is taken. Of many sequences items / slots is near even / per, and the second
  // form is least at per = sqrt(6 even). None is below total / share, so there are no more items than share and one for each block.
  __device__ __forceinline__ uint32_t part_tiles(const Sequence& first, float total) const {
    const uint32_t lane = threadIdx.x & 63u;
    const float even = total * (float)kv_heads / (float)slots, floor = total * 1.0001f / (float)share;
    auto from = [&](float tiles) { return max(least, (uint32_t)fminf(fmaxf(tiles, floor), (float)kMaxKeys) + 1u); };
    if (sequences > 64u) return from(sqrtf(6.f * even));
    const uint32_t per = from(even * (lane < 48u ? 1.f + (float)lane * (1.f / 48.f) : (float)(lane - 46u) * (1.f / 18.f)));
    const float one = __builtin_amdgcn_rcpf((float)per);
    float items = 0.f;
#pragma unroll 1
    for (uint32_t b = 0; b < sequences; ++b) {
      const float tiles = (float)__builtin_amdgcn_readlane((int)first.tiles, (int)b);
      items += (float)__builtin_amdgcn_readlane((int)first.blocks, (int)b) * ceilf(tiles * one);
    }
    const float turns = items * (float)kv_heads / (float)slots;
    const float c = turns <= 1.f ? (float)per + 3.f : even + 0.5f * (float)per + 3.f * turns;
    const uint32_t cost = __builtin_bit_cast(uint32_t, c);  // (above 0: the bits are in the numbers' order)
    const uint64_t least_cost = __ballot(cost == wave_fold(cost, [](uint32_t x, uint32_t y) { return min(x, y); }));
    return (uint32_t)__builtin_amdgcn_readlane((int)per, (int)__builtin_ctzll(least_cost));
  }
  // All items of a work-group, blockIdx.x and every gridDim.x-th behind it: of(place).
  template <typename F>
  __device__ __forceinline__ void each_item(F of) const {
    const uint32_t lane = threadIdx.x & 63u;
    const bool one = sequences == 1u;
    auto plus = [](uint32_t x, uint32_t y) { return x + y; };
    Sequence s = sequence(*this, one ? 0u : lane);
    uint32_t per, items;  // (items of a kv head)
    bool falls = s.falls;
    for (uint32_t b = 64u; b < sequences; b += 64u) falls |= sequence(*this, b + lane).falls;
    if (__ballot(falls)) {  // (sequences may share rows: two work-groups would store one)
      if (flag) *flag = MI_STATUS_BAD_ROWS;
      if (blockIdx.x == 0u)
        for (uint32_t t = threadIdx.x; t < T; t += blockDim.x) info[t] = u4_t{0u, 0u, 0u, 0u};  // (nothing to join)
      return;
    }
    if (one) {
      per = max(least, max(s.blocks, s.tiles) < 65536u ? (s.blocks * s.tiles + share - 1u) / share
                                                       : (uint32_t)((float)s.blocks * (float)s.tiles * 1.0001f / (float)share) + 1u);
      items = s.blocks * parts(s, per);
    } else {
      float total = (float)s.blocks * (float)s.tiles;
      for (uint32_t b = 64u; b < sequences; b += 64u) {
        const Sequence o = sequence(*this, b + lane);
        total += (float)o.blocks * (float)o.tiles;
      }
      per = part_tiles(s, wave_sum(total));
      items = s.blocks * parts(s, per);
      for (uint32_t b = 64u; b < sequences; b += 64u) {
        const Sequence o = sequence(*this, b + lane);
        items += o.blocks * parts(o, per);
      }
      items = wave_fold(items, plus);
    }
#pragma unroll 1
    for (uint32_t at = blockIdx.x;; at += gridDim.x) {
      uint32_t item = item_of(items * kv_heads, at), part = 0, b = 0;
      if (item == kNone) return;
      const uint32_t j = item / items;
      item -= j * items;
      uint32_t found = 0;
      if (one) {
        if (at != blockIdx.x) s = sequence(*this, 0u);
      } else {
#pragma unroll 1
        for (;; b += 64u) {
          if (at != blockIdx.x || b) s = sequence(*this, b + lane);
          const uint32_t n = parts(s, per), mine = s.blocks * n;
          uint32_t sum = mine;  // of the lanes up to this one
#pragma unroll
          for (uint32_t d = 1; d < 64u; d *= 2) {
            const uint32_t o = (uint32_t)__shfl_up((int)sum, d, 64);
            sum += lane >= d ? o : 0u;
          }
          const uint64_t behind = __ballot(sum > item);
          found = behind ? (uint32_t)__builtin_ctzll(behind) : 64u;
          part += wave_fold(lane < found && n > 1u ? mine : 0u, plus);
          if (found < 64u) {
            item -= (uint32_t)__builtin_amdgcn_readlane((int)(sum - mine), (int)found);
            break;
          }
          if (b + 64u >= sequences) return;  // (not reached: item is below the sum of all)
          item -= (uint32_t)__builtin_amdgcn_readlane((int)sum, 63);
        }
      }
      auto of_found = [&](uint32_t v) { return (uint32_t)__builtin_amdgcn_readlane((int)v, (int)found); };
      const Sequence f = {of_found(s.start),  of_found(s.rows),  of_found(s.cached), of_found(s.keys),
                          of_found(s.blocks), of_found(s.tiles), false};
      b += found;
      s = Sequence{};  // (not kept in registers meanwhile)
      of(inside(f, b, parts(f, per), j, item, part));
      __syncthreads();
    }
  }
  // Work-group `group`'s of `items` items: XCD x (every eighth work-group is its) has those from x / 8 of them on.
  __device__ __forceinline__ uint32_t item_of(uint32_t items, uint32_t group) const {
    const uint32_t each = (items + kXcds - 1u) / kXcds, at = group / kXcds, item = (group % kXcds) * each + at;
    return at < each && item < items ? item : kNone;
  }
  // The place of kv head j's item `item` of sequence b, of n parts; behind `part` items of a head that leave sums.
  __device__ __forceinline__ Place inside(const Sequence& s, uint32_t b, uint32_t n, uint32_t j, uint32_t item, uint32_t part) const {
    Place p{};
    const uint32_t split = item / s.blocks, block = item - split * s.blocks;
    p.j = j;
    p.own = block * rows;
    p.rows = min(rows, s.rows - p.own);
    p.t0 = s.start + p.own;
    p.split = split;
    p.splits = n;
    p.b = b;
    p.cached = s.cached;
    p.keys = s.keys;
    p.part = part * kv_heads + (split * kv_heads + j) * s.blocks + block;
    if (split == 0u && j == 0u && threadIdx.x < p.rows)
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

// 16 bytes per lane from base + off straight into LDS [lds, lds + 1024), lane L at lds + 16 L. The compiler neither sees what this
// writes nor counts the load: the kernel waits by vmcnt itself (the compiler's own loads only make such a wait stricter).
__device__ __forceinline__ void load_lds(uint32_t lds, const uint16_t* base, uint32_t off) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(off), "s"(base) : "memory");
}
__device__ __forceinline__ void load_lds(uint32_t lds, const uint16_t* from) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds), "v"(from) : "memory");
}
template <uint32_t N>
__device__ __forceinline__ void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// Blocks of more than 16 columns: four waves side by side, CT column tiles and all dims each, all walking the same 32-key tiles. K and V
// go straight into LDS, into rings of three and four tiles: a tile's loads have two steps. A step i:
//   the products of tile i + 1's scores, dealt out among the exponentials that make tile i's weights;
//   the barrier: behind it every wave has read K of tile i + 1 and V of tile i - 1, whose places take K of tile i + 4 and V of
//   tile i + 3, and the loads of two steps ago (K of i + 2, V of i + 1) are there;
//   P V of tile i, dealt out among tile i + 1's masks and maxima.
// A wave's column tiles are every fourth, and those behind the block's columns are left out: each wave walks with as many as it
// has. The first operands of each half are read in the one before. Rows of a tile lie 2 HD bytes apart in LDS, the 16-byte pieces of row r
// in the order p ^ (r % 16): the 16 rows of a read fall on distinct banks.
template <int HD, int CT, Order ORDER>
__device__ __forceinline__ void rows_of_block(const TreeRows& a, const TreeRows::Place& p) {
  constexpr uint32_t KK = HD / 32, NT = HD / 16, S = 2 * KK, ROW = 2 * HD, TILE = kTile * ROW;
  constexpr uint32_t NI = TILE / 4096, RPI = 1024 / ROW, PPR = ROW / 16;  // a wave's loads of a tile, rows of each, pieces of a row
  constexpr uint32_t AK = 3, AV = 3, PER = KK / 2;  // operands read ahead; products for each weight
  __shared__ __align__(1024) uint8_t ring[7 * TILE];
  uint32_t thread = threadIdx.x;
  asm volatile("" : "+v"(thread));  // (what follows from it is formed anew in each item, not kept)
  const TreeRows::Block b = a.block(p);
  const uint32_t lane = thread & 63u, wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(thread >> 6)), qi = lane & 15u,
                 qq = lane >> 4;
  auto uniform = [](uint32_t v) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)v); };
  const uint32_t from = uniform(a.part_begin(p, b, p.split)), n = uniform(a.part_begin(p, b, p.split + 1u)) - from;
  const uint32_t last = uniform(b.last);
  uint32_t row[CT], g[CT];
  h8_t qh[CT][KK], ql[CT][KK];
  // ---- the loads ----
  const uint32_t lds = (uint32_t)(uintptr_t)ring;
  const size_t hoff = (size_t)uniform(p.j) * a.head_stride;
  // a load's row of the tile, its piece's elements, and its bytes behind the tile's first row, in the last tile too
  uint32_t place[NI], piece[NI], off[NI], off_last[NI];
#pragma unroll
  for (uint32_t c = 0; c < NI; ++c) {
    place[c] = (4u * c + wave) * RPI + lane / PPR;
    piece[c] = 8u * ((lane % PPR) ^ (place[c] & 15u));
    off[c] = 2u * (place[c] * (uint32_t)a.row_stride + piece[c]);
    off_last[c] = 2u * (min(place[c], (last - b.key(from + n - 1u))) * (uint32_t)a.row_stride + piece[c]);
  }
  bool outside = false;
  struct Rows {
    uint32_t r[ORDER == kAnyPages ? NI : 1];  // the cache rows of a tile: its first, or each load's
  };
  // (whole tiles) 64 entries of the page table from that of tile i on, a lane each, and the first's number
  uint32_t entries = 0, entries_at = 0;
  auto fetch = [&](uint32_t i) {
    entries_at = b.key(from + min(i, n - 1u)) >> a.page_shift;
    entries = b.pages[min(entries_at + lane, last >> a.page_shift)];
  };
  auto rows_of = [&](uint32_t i) {
    const uint32_t key = b.key(from + min(i, n - 1u));
    Rows w;
    if constexpr (ORDER == kContiguous) {
      w.r[0] = b.base + key;
    } else if constexpr (ORDER == kWholeTiles) {
      const uint32_t at = key >> a.page_shift, pg = (uint32_t)__builtin_amdgcn_readlane((int)entries, (int)(at - entries_at));
      outside |= pg >= a.n_pages;
      w.r[0] = (pg < a.n_pages ? pg << a.page_shift : 0u) + (key - (at << a.page_shift));
    } else {
#pragma unroll
      for (uint32_t c = 0; c < NI; ++c) w.r[c] = a.cache_row(b, min(key + place[c], b.last), outside);
    }
    return w;
  };
  auto load = [&](const uint16_t* cache, uint32_t to, uint32_t i, const Rows& w) {
    if constexpr (ORDER == kAnyPages) {
#pragma unroll
      for (uint32_t c = 0; c < NI; ++c)
        load_lds(lds + to + (4u * c + wave) * 1024u, cache + ((size_t)w.r[c] * a.row_stride + hoff + piece[c]));
    } else {
      const uint16_t* base = cache + ((size_t)uniform(w.r[0]) * a.row_stride + hoff);
#pragma unroll
      for (uint32_t c = 0; c < NI; ++c)
        load_lds(lds + to + (4u * c + wave) * 1024u, base, i + 1u < n ? off[c] : off_last[c]);
    }
  };
  auto k_at = [](uint32_t i) { return i % 3u * TILE; };
  auto v_at = [](uint32_t i) { return (3u + i % 4u) * TILE; };
  // the page table's entries and the columns' queries, asked for together; then the first tiles; then, meanwhile, the queries as the B
  // operand, scaled, in f16 high and low parts: k = 32 kk + 8 qq + e
  if constexpr (ORDER == kWholeTiles) fetch(0);
  f4_t q[CT][2 * KK];
#pragma unroll
  for (uint32_t ct = 0; ct < CT; ++ct) {
    const uint32_t col = 16u * (4u * ct + wave) + qi;
    row[ct] = col / a.gqa;
    g[ct] = col % a.gqa;
    const float* qp = a.q + ((size_t)(p.t0 + (row[ct] < p.rows ? row[ct] : 0u)) * a.q_heads + p.j * a.gqa + g[ct]) * HD + 8u * qq;
#pragma unroll
    for (uint32_t x = 0; x < 2 * KK; ++x) q[ct][x] = *as_global(reinterpret_cast<const f4_any*>(qp + 32u * (x / 2) + 4u * (x % 2)));
  }
  Rows r2{}, r3{};
  if (n) {
    asm volatile("" ::"v"(entries));
    const Rows r0 = rows_of(0), r1 = rows_of(1);
    r2 = rows_of(2);
    r3 = rows_of(3);
#pragma unroll
    for (uint32_t ct = 0; ct < CT; ++ct)
#pragma unroll
      for (uint32_t x = 0; x < 2 * KK; ++x) asm volatile("" : "+v"(q[ct][x]));  // (waited for here: behind the tiles' loads it would be for them too)
    load(a.k, k_at(0), 0, r0);
    load(a.k, k_at(1), 1, r1);
    load(a.v, v_at(0), 0, r0);
    load(a.k, k_at(2), 2, r2);
    load(a.v, v_at(1), 1, r1);
  }
#pragma unroll
  for (uint32_t ct = 0; ct < CT; ++ct) {
#pragma unroll
    for (uint32_t x = 0; x < 2 * KK; ++x) q[ct][x] *= a.c;
    split_q<KK>(q[ct], qh[ct], ql[ct]);
    if constexpr (HD * CT > 256) {  // (in accumulation registers, which the products read too: the others are the vector ALUs')
#pragma unroll
      for (uint32_t kk = 0; kk < KK; ++kk) asm volatile("" : "+a"(qh[ct][kk]), "+a"(ql[ct][kk]));
    }
  }
  if (n) {
    wait_loads<2 * NI>();
    lds_barrier();
    // V of tile 2 and K of tile 3 follow behind the first scores
  }
  float r[CT], l[CT], w[CT][8];
  f4_t acc[CT][NT], d[CT][2];
#pragma unroll
  for (uint32_t ct = 0; ct < CT; ++ct) {
    r[ct] = kNoKey;
    l[ct] = 0.f;
#pragma unroll
    for (uint32_t tt = 0; tt < NT; ++tt) acc[ct][tt] = f4_t{0.f, 0.f, 0.f, 0.f};
  }
  // K operand s = 2 kk + gg: 16 keys x 32 dims
  auto k_operand = [&](uint32_t to, uint32_t s) {
    const uint32_t at = qi * ROW + 16u * ((4u * (s / 2u) + qq) ^ qi);
    return *reinterpret_cast<const h8_t*>(ring + to + at + (s % 2u) * 16u * ROW);
  };
  // V^T of 32 keys x 16 dims: the k of the product are the keys 4 qq + e of the two 16-key groups, which is how the lanes hold the
  // weights
  auto v_operand_at = [&](uint32_t to, uint32_t tt) {
    const uint32_t vrow = 4u * qq + (qi >> 2), at = vrow * ROW + 16u * ((2u * tt + ((qi >> 1) & 1u)) ^ vrow) + 8u * (qi & 1u);
    const v4s_t a0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((v4s_lds)(reinterpret_cast<const uint16_t*>(ring + to + at)));
    const v4s_t a1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((v4s_lds)(reinterpret_cast<const uint16_t*>(ring + to + at + 16u * ROW)));
    return __builtin_bit_cast(h8_t, __builtin_shufflevector(a0, a1, 0, 1, 2, 3, 4, 5, 6, 7));
  };
  // the walk of a wave with NC column tiles that hold columns
  auto walk = [&](auto tiles) {
    constexpr uint32_t NC = decltype(tiles)::value;
    auto product = [&](h8_t kh, uint32_t s, uint32_t part) {  // part < 2 NC: the columns' high parts, then the low ones
      const uint32_t ct = part % NC;
      d[ct][s % 2] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kh, part < NC ? qh[ct][s / 2] : ql[ct][s / 2], d[ct][s % 2], 0, 0, 0);
    };
    auto clear = [&]() {
#pragma unroll
      for (uint32_t ct = 0; ct < NC; ++ct) d[ct][0] = d[ct][1] = f4_t{0.f, 0.f, 0.f, 0.f};
    };
    // a tile's scores of column tile ct and the largest of them; behind that tile i's masks and the references
    float mx[NC ? NC : 1];
    auto scores = [&](uint32_t ct) {
#pragma unroll
      for (uint32_t e = 0; e < 8; ++e) w[ct][e] = d[ct][e / 4][e % 4];
      mx[ct] = most_of(w[ct]);
      asm volatile("" : "+v"(mx[ct]));  // (formed here, between the products, not where it is used)
    };
    auto settle = [&](uint32_t i) {
      const uint32_t key = b.key(from + i);
      if (a.masked(b, key)) {
#pragma unroll
        for (uint32_t ct = 0; ct < NC; ++ct) {
          a.bias_and_mask(a.column(p, b, row[ct], g[ct]), key + 4u * qq, true, w[ct]);
          mx[ct] = most_of(w[ct]);
        }
      }
      if constexpr (NC != 0) raise_to<NC, NT>(mx, qi, r, l, acc, nullptr);
    };
    h8_t kh[S], av[NT];
    if (n) {
      clear();
#pragma unroll
      for (uint32_t s = 0; s < S; ++s) {
        const h8_t k0 = k_operand(k_at(0), s);
#pragma unroll
        for (uint32_t part = 0; part < 2 * NC; ++part) product(k0, s, part);
      }
#pragma unroll
      for (uint32_t ct = 0; ct < NC; ++ct) scores(ct);
      settle(0);
      lds_barrier();
      load(a.k, k_at(3), 3, r3);
      load(a.v, v_at(2), 2, r2);
#pragma unroll
      for (uint32_t s = 0; s < AK; ++s) kh[s] = k_operand(k_at(1), s);
    }
    uint32_t k1 = TILE, k2 = 2u * TILE, k3 = 0u, v0 = 3u * TILE, v1 = 4u * TILE, v2 = 5u * TILE, v3 = 6u * TILE;  // of tiles i + ..
#pragma unroll 1
    for (uint32_t i = 0; i < n; ++i) {
      if constexpr (ORDER == kWholeTiles)
        if (i % 32u == 0u) {  // (pages hold a tile at least: 64 entries serve 64 steps)
          fetch(i + 4u);
          asm volatile("" ::"v"(entries));  // (waited for here, not in the loop)
        }
      h8_t pw[NC ? NC : 1];
      {  // (behind the last tile the products are of a tile that is not used)
        clear();
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (uint32_t s = 0; s < S; ++s) {
          if (s + AK < S) kh[s + AK] = k_operand(k1, s + AK);
          if (s + AV >= S) av[s + AV - S] = v_operand_at(v0, s + AV - S);
#pragma unroll
          for (uint32_t part = 0; part < 2 * NC; ++part) {
            product(kh[s], s, part);
            const uint32_t done = s * 2 * NC + part + 1u;
            if (done % PER) continue;
            const uint32_t x = done / PER - 1u, ct = x / 8, e = x % 8;
            w[ct][e] = __builtin_amdgcn_exp2f(w[ct][e] - r[ct]);
            l[ct] += w[ct][e];
            asm volatile("" : "+v"(l[ct]));
            if (e % 2) {
              u4_t pk = __builtin_bit_cast(u4_t, pw[ct]);
              pk[e / 2] = h2_bits(__builtin_convertvector((f2_t{w[ct][e - 1], w[ct][e]}), h2_t));
              pw[ct] = __builtin_bit_cast(h8_t, pk);
            }
            __builtin_amdgcn_sched_barrier(0);
          }
        }
      }
      wait_loads<2 * NI>();
      lds_barrier();
      {
        const Rows r4 = rows_of(i + 4u);
        load(a.k, k1, i + 4u, r4);
        load(a.v, v3, i + 3u, r3);
        r3 = r4;
      }
      {
#pragma unroll
        for (uint32_t tt = 0; tt < NT; ++tt) {
          if (tt + AV < NT) av[tt + AV] = v_operand_at(v0, tt + AV);
          if (tt + AK >= NT) kh[tt + AK - NT] = k_operand(k2, tt + AK - NT);
#pragma unroll
          for (uint32_t ct = 0; ct < NC; ++ct) acc[ct][tt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(av[tt], pw[ct], acc[ct][tt], 0, 0, 0);
          if (tt >= 1 && tt <= NC) scores(tt - 1);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      if (NC != 0 && i + 1u < n) settle(i + 1u);
      const uint32_t k = k1, v = v0;
      k1 = k2;
      k2 = k3;
      k3 = k;
      v0 = v1;
      v1 = v2;
      v2 = v3;
      v3 = v;
    }
  };
  const uint32_t used = (p.rows * a.gqa + 15u) / 16u, live = uniform(used > wave ? (used - wave + 3u) / 4u : 0u);
  auto walk_if = [&](auto tiles) {
    if constexpr (decltype(tiles)::value <= CT)
      if (live == tiles) walk(tiles);
  };
  walk_if(std::integral_constant<uint32_t, 0>{});
  walk_if(std::integral_constant<uint32_t, 1>{});
  walk_if(std::integral_constant<uint32_t, 2>{});
  walk_if(std::integral_constant<uint32_t, 3>{});
  walk_if(std::integral_constant<uint32_t, 4>{});
  wait_loads<0>();
  if (ORDER != kContiguous && __ballot(outside)) a.report_pages(p, b, from, from + n, 1u);
  float sum[CT];
  bool bad = false;
#pragma unroll
  for (uint32_t ct = 0; ct < CT; ++ct) {
    sum[ct] = col_sum(l[ct]);
    float z = sum[ct] - sum[ct];
#pragma unroll
    for (uint32_t tt = 0; tt < NT; ++tt) z = not_finite(z, acc[ct][tt]);
    bad |= row[ct] < p.rows && z != 0.f;
  }
  if (__syncthreads_or(bad)) {
    slow_block<HD>(a, p, b, from, from + n, [&](float(&w)[8]) { a.scores_by_form(w); });
    return;
  }
#pragma unroll
  for (uint32_t ct = 0; ct < CT; ++ct) {
    if (row[ct] >= p.rows) continue;
    if (p.splits > 1) {
#pragma unroll
      for (uint32_t tt = 0; tt < NT; ++tt) store_part<HD>(a, p, row[ct], g[ct], qq, tt, acc[ct][tt]);
      if (qq == 0) {
        float* o = a.template part_at<HD>(p, row[ct], g[ct]);
        o[HD] = r[ct];
        o[HD + 1] = sum[ct];
      }
    } else {
      const float inv = sum[ct] != 0.f ? 1.0f / sum[ct] : 0.f;
#pragma unroll
      for (uint32_t tt = 0; tt < NT; ++tt)
        store_out<HD>(a, p.j, p.t0 + row[ct], g[ct], qq, tt, inv == 0.f ? f4_t{0.f, 0.f, 0.f, 0.f} : acc[ct][tt] * inv);
    }
  }
}

template <int HD, int CT, Order ORDER>
__global__ __launch_bounds__(256, HD * CT <= 256 ? 2 : 1) void attn_tree_kernel(TreeRows a) {
  a.each_item([&](const TreeRows::Place& p) { rows_of_block<HD, CT, ORDER>(a, p); });
}

// The sums of a column's parts s0, s0 + step .., four dims of them, U parts at a time.
struct Sums {
  f4_t o = {0.f, 0.f, 0.f, 0.f};
  float top = kNoKey, sum = 0.f;
  __device__ __forceinline__ void turn(float to) {
    const float f = __builtin_amdgcn_exp2f(top - to);
    sum *= f;
    o *= f;
    top = to;
  }
  __device__ __forceinline__ void add(f4_t v, float r, float l) {  // (r up to top)
    const float w = l == 0.f ? 0.f : __builtin_amdgcn_exp2f(r - top);  // (0: no key of the row in that part)
    sum = __builtin_fmaf(l, w, sum);
#pragma unroll
    for (uint32_t e = 0; e < 4; ++e) o[e] = __builtin_fmaf(v[e], w, o[e]);
  }
};
template <int HD, uint32_t U, typename F>
__device__ __forceinline__ Sums join_parts(uint32_t s0, uint32_t step, uint32_t splits, uint32_t d, F part) {
  Sums a;
  for (; s0 < splits; s0 += U * step) {
    f4_t v[U];
    float r[U], l[U], now = a.top;
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) {
      const uint32_t s = s0 + u * step;
      const float* p = part(s < splits ? s : s0);
      v[u] = *as_global(reinterpret_cast<const f4_t*>(p + 4u * d));
      r[u] = *as_global(p + HD);
      l[u] = s < splits ? *as_global(p + HD + 1) : 0.f;
    }
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) now = l[u] == 0.f ? now : fmaxf(now, r[u]);
    a.turn(now);
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) a.add(v[u], r[u], l[u]);
  }
  return a;
}
// Joins the parts of row blockIdx.y: HD / 4 threads side by side take a column, four dims each. MANY: all threads of a work-group are
// one column's and share its parts out; else each HD / 4 take columns in turn.
template <int HD, bool MANY>
__global__ __launch_bounds__(256) void attn_tree_join_kernel(TreeArgs a, uint32_t most) {
  constexpr uint32_t L = HD / 4, G = 256 / L;
  const uint32_t t = blockIdx.y, g = threadIdx.x / L, d = threadIdx.x % L;
  const u4_t info = *as_global(a.info + t);
  const uint32_t first = a.row_start[0], end = min(a.row_start[a.sequences], a.T), splits = min(info[2], kMaxSplits);
  asm volatile("" ::"v"(info), "s"(first), "s"(end));  // (one round trip for all three)
  if (t < first || t >= end || splits < 2u) return;  // (uniform: no sequence's row, or its work-group stored it)
  auto part_of = [&](uint32_t h) {
    const uint32_t j = h / a.gqa, col = info[3] * a.gqa + h % a.gqa;
    return [&a, info, j, col, most](uint32_t s) {  // (within the workspace whatever row_start held)
      return a.part + ((size_t)min(info[0] + (s * a.kv_heads + j) * info[1], most) * a.columns + min(col, a.columns - 1u)) * (HD + 4);
    };
  };
  auto store = [&](uint32_t h, const Sums& s) {
    const float inv = s.sum == 0.f ? 0.f : 1.0f / s.sum;
    store_out<HD>(a, h / a.gqa, t, h % a.gqa, d % 4u, d / 4u, s.o * inv);
  };
  if constexpr (MANY) {
    __shared__ __align__(16) f4_t sums[G][L];
    __shared__ float tops[G], totals[G];
    Sums s = join_parts<HD, 8>(g, G, splits, d, part_of(blockIdx.x));
    sums[g][d] = s.o;
    if (d == 0) {
      tops[g] = s.top;
      totals[g] = s.sum;
    }
    __syncthreads();
    if (g) return;
    float top = s.top;
#pragma unroll
    for (uint32_t n = 1; n < G; ++n) top = fmaxf(top, tops[n]);
    s.turn(top);
#pragma unroll
    for (uint32_t n = 1; n < G; ++n) s.add(sums[n][d], tops[n], totals[n]);
    store(blockIdx.x, s);
  } else {
    for (uint32_t h = blockIdx.x * G + g; h < a.q_heads; h += gridDim.x * G) store(h, join_parts<HD, 4>(0u, 1u, splits, d, part_of(h)));
  }
}

// The launch: the few-rows kernel up to 16 columns a sequence, else the other with CT column tiles a wave (64 CT columns a
// work-group; two work-groups a CU of rows of 128 with CT 2).
//   rows of 256: CT 1 up to 64 columns, else 2. Measured (us): 6 ragged sequences up to 8200 keys, 16 / 2 heads, 8 rows 28.5
//   against 32.7; 8 sequences, 30 rows 57.4 against 55.8; one of 131072, 60 rows 254 against 204.
//   rows of 128: one sequence's rows make blocks / CT work-groups of a known number: the least modelled time of 2, 3 and 4, a
//   block's tile 1.1, 1.375 and 1.7 us of a CU. Measured (us; CT 2, 3, 4; 40 / 8 heads; 25, 38, 51 and 64 rows): over 65536 keys
//   83 / 82 / 82, 111 / 97 / 97, 184 / 151 / 117, 193 / 155 / 185; over 8192 29 / 27 / 27, 33 / 32 / 32, 37 / 38 / 38, 39 / 40 / 46;
//   over 4096 27 / 23 / 23, 28 / 27 / 28, 31 / 30 / 32, 32 / 31 / 36. Of several sequences only the mean is known: CT 2, which
//   loses least where they are ragged (8 trees of 38 to 61 rows 93 / 105 / 125; of 51 each, 4000 keys, 93 / 85 / 72).
// The mean says little of single tokens beside a stretch of a prompt, 40 / 8 heads, taken as one call / as two (us): 48 tokens up to 16000
// keys and 100 rows behind 2000 329 / 301, and 512 rows 351 / 337; 63 tokens up to 4000 and 128 rows behind 4000 187 / 155; 300 and
// 300 rows 665 / 560; 31 and 512 rows behind none 88 / 91.
struct Pick {
  bool few;
  uint32_t ct, rows, columns, slots;
};
constexpr uint32_t kCus = 256;
Pick few_rows(uint32_t gqa, uint32_t hd) { return Pick{true, 1, 16u / gqa, 16, (hd == 128 ? 2u : 1u) * kCus}; }
Pick chunk(uint32_t ct, uint32_t gqa, uint32_t hd) {
  return Pick{false, ct, 64u * ct / gqa, 64u * ct, hd == 128 && ct == 2u ? 2u * kCus : kCus};
}
Pick pick(uint32_t T, uint32_t sequences, uint32_t gqa, uint32_t hd) {
  const uint32_t each = (T + sequences - 1u) / sequences * gqa;  // columns
  if (each <= 16u) return few_rows(gqa, hd);
  if (hd == 256) return chunk(each <= 64u ? 1u : 2u, gqa, hd);
  Pick best = chunk(2u, gqa, hd);
  if (sequences > 1u) return best;
  static constexpr double kTau[5] = {0.0, 0.0, 1.1, 1.375, 1.7};
  double least = 1e300;
  for (uint32_t ct = 2; ct <= 4; ++ct) {
    const Pick p = chunk(ct, gqa, hd);
    const double c = ((T + p.rows - 1u) / p.rows) * kTau[ct];
    if (c >= least) continue;
    least = c;
    best = p;
  }
  return best;
}
// The parts of all sequences at most, one for each block aside: as many as make every work-group that runs at once busy, where there
// are several sequences some times as many, which its work-groups take one behind another.
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
  const bool near = a.row_stride <= 1u << 25;  // (a tile's rows by a 32-bit offset)
  if (!a.tables && near) attn_tree_kernel<HD, CT, kContiguous><<<grid, 256, 0, st>>>(a);
  else if (a.tables && a.page >= kTile && a.page_shift < 32u && near) attn_tree_kernel<HD, CT, kWholeTiles><<<grid, 256, 0, st>>>(a);
  else attn_tree_kernel<HD, CT, kAnyPages><<<grid, 256, 0, st>>>(a);
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
  if (T * gqa > 16u)
    for (uint32_t ct = 1; ct <= 4; ++ct)
      floats = std::max(floats, part_floats(chunk(ct, gqa, hd), shape->kv_heads, ct <= 2u ? 2u : 1u, hd));
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
  const uint32_t most_blocks = T / p.rows + n;  // (no two sequences share a row)
  // as many work-groups as run at once, and as there are items at most: share and one more for each block, of each kv head, no more
  // than the blocks have parts of the least size
  const uint64_t least_parts = ((uint64_t)kv_len + a.least * kTile - 1u) / (a.least * kTile);
  const uint32_t items = shape->kv_heads * (uint32_t)std::min<uint64_t>(a.share + most_blocks, most_blocks * least_parts);
  const uint32_t grid = std::min((items + kXcds - 1u) / kXcds * kXcds, p.slots);
  const bool narrow = shape->head_dim == 128;
  if (p.few) {
    if (narrow) attn_rows_few_kernel<128><<<grid, 256, 0, st>>>(a);
    else attn_rows_few_kernel<256><<<grid, 256, 0, st>>>(a);
  } else if (narrow) {
    if (p.ct == 2) launch_chunk<128, 2>(a, grid, st);
    else if (p.ct == 3) launch_chunk<128, 3>(a, grid, st);
    else launch_chunk<128, 4>(a, grid, st);
  } else {
    if (p.ct == 2) launch_chunk<256, 2>(a, grid, st);
    else launch_chunk<256, 1>(a, grid, st);
  }
  if (kv_len > a.least * kTile) {  // (there may be several parts)
    const uint32_t most = 2u * a.share * shape->kv_heads - 1u;
    if (most_blocks * 8u <= a.share) {
      if (narrow) attn_tree_join_kernel<128, true><<<dim3(shape->q_heads, T), 256, 0, st>>>(a, most);
      else attn_tree_join_kernel<256, true><<<dim3(shape->q_heads, T), 256, 0, st>>>(a, most);
    } else {  // (of many rows most have one part: few work-groups a row)
      const uint32_t heads = narrow ? 8u : 4u, x = std::min((shape->q_heads + heads - 1u) / heads, std::max(1u, 4096u / T));
      if (narrow) attn_tree_join_kernel<128, false><<<dim3(x, T), 256, 0, st>>>(a, most);
      else attn_tree_join_kernel<256, false><<<dim3(x, T), 256, 0, st>>>(a, most);
    }
  }
  return mi_hip((int)hipGetLastError(), "attn_tree");
}

}  // extern "C"
