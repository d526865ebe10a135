// paged.hip - the bookkeeping of several sequences over one paged cache, on the GPU: block tables and slot maps from the requests'
// lengths (mi_block_tables), and moves of cache rows (mi_kv_move).
//
// A step's plan. Request b holds held_b pages and cached_b keys and adds added_b rows:
//   need_b = ceil((cached_b + added_b) / page);  it takes max(need_b - held_b, 0) pages from a ring of free ones, the first request
//   first, and gives back max(held_b - need_b, 0) behind the ring's last
//   row t = row_start_b + i (row_start: the sums of added): key cached_b + i, cache row table_b[key / page] page + key % page
//   a tree's node i: mask_t the bits of i and its ancestors, position cached_b + their number; else position = key
// One work-group does the requests, a thread each; a thread does a row. Bound by chains of loads, not by bytes: 8 trees of 61 nodes
// (10 KB) 5.6 us, a launch that does nothing 3.5; 509 requests with 10000 rows 8.3 in two launches. More rows than kOneGroup are
// more than one work-group's loads hide.
#include <algorithm>

#include "mi_capi_internal.h"
#include "mi_pieces.h"

namespace mi {
namespace {

constexpr uint32_t kMaxRequests = 1024, kMaxRows = 65535, kMaxKeys = 1u << 30, kMaxWords = 64, kMaxTable = 1u << 21, kMaxPage = 1u << 20, kNone = 0xFFFFFFFFu;
constexpr uint32_t kOneGroup = 4096;  // rows that the requests' work-group does itself

struct PlanArgs {
  mi_block_plan p;
  uint32_t* ws;  // [0] whether there is a plan, [1] the ring's first page, then (held, first taken) of each request
};

// The sums of three values over the threads before each one, and over all of them.
struct Three {
  uint32_t a, b, c;
};
__device__ __forceinline__ Three sums_before(Three v, Three& all) {
  __shared__ Three of[kMaxRequests / 64];
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
  Three s = v;
#pragma unroll
  for (uint32_t d = 1; d < 64u; d *= 2) {
    const Three o = {(uint32_t)__shfl_up((int)s.a, d, 64), (uint32_t)__shfl_up((int)s.b, d, 64), (uint32_t)__shfl_up((int)s.c, d, 64)};
    if (lane >= d) s = Three{s.a + o.a, s.b + o.b, s.c + o.c};
  }
  if (lane == 63u) of[wave] = s;
  __syncthreads();
  Three before = {s.a - v.a, s.b - v.b, s.c - v.c};
  all = Three{0u, 0u, 0u};
  for (uint32_t w = 0; w < blockDim.x / 64u; ++w) {
    const Three o = of[w];
    if (w < wave) before = Three{before.a + o.a, before.b + o.b, before.c + o.c};
    all = Three{all.a + o.a, all.b + o.b, all.c + o.c};
  }
  return before;
}

// What the rows of a work-group need of the requests, in LDS.
struct Requests {
  uint32_t start[kMaxRequests + 1];  // row_start
  uint32_t cached[kMaxRequests], held[kMaxRequests], taken[kMaxRequests];
};
// the last of n + 1 ascending sums that is not above i, which is below the last one
__device__ __forceinline__ uint32_t find(const uint32_t* sums, uint32_t n, uint32_t i) {
  uint32_t lo = 0, hi = n;
  while (hi - lo > 1u) {
    const uint32_t mid = (lo + hi) / 2u;
    if (sums[mid] <= i) lo = mid;
    else hi = mid;
  }
  return lo;
}
// The rows begin .. end - 1, and their parents in LDS.
__device__ __forceinline__ void plan_rows(const PlanArgs& a, const Requests& r, bool planned, uint32_t head, uint32_t begin, uint32_t end,
                                          const uint32_t* parents) {
  const mi_block_plan& p = a.p;
  const uint32_t total = planned ? r.start[p.requests] : 0u;
  for (uint32_t t = begin + threadIdx.x; t < end; t += blockDim.x) {
    if (t >= total) {
      p.seq[t] = p.slot[t] = kNone;
      p.pos[t] = 0u;
      if (p.mask)
        for (uint32_t w = 0; w < p.words; ++w) p.mask[(size_t)t * p.words + w] = 0u;
      continue;
    }
    const uint32_t b = find(r.start, p.requests, t), start = r.start[b], i = t - start, key = r.cached[b] + i;
    const uint32_t held = r.held[b], at = key / p.page, in = key - at * p.page;
    uint32_t* table = p.tables + (size_t)b * p.table_stride;
    const bool fresh = at >= held;
    const uint32_t page = fresh ? p.ring[(uint32_t)(((uint64_t)head + r.taken[b] + (at - held)) % p.ring_len)] : table[at];
    if (fresh && in == 0u) table[at] = page;  // (its first key is one of the step's: the cached ones have their pages)
    if (page >= p.n_pages && p.flag) *p.flag = MI_STATUS_BAD_PAGE;
    p.seq[t] = b;
    p.slot[t] = page < p.n_pages ? page * p.page + in : kNone;
    if (!p.parent) {
      p.pos[t] = key;
      continue;
    }
    // up the tree: a parent's number is below its child's, so the words of the mask come one after another
    uint32_t* mask = p.mask + (size_t)t * p.words;
    uint32_t w = i / 32u, bits = 1u << (i % 32u), depth = 0, node = i;
    for (uint32_t x = p.words - 1u; x > w; --x) mask[x] = 0u;
    for (;;) {
      const uint32_t row = start + node, up = row >= begin ? parents[row - begin] : p.parent[row];
      if (up >= node) {
        if (up != kNone && p.flag) *p.flag = MI_STATUS_BAD_ROWS;
        break;
      }
      for (; w > up / 32u; --w) {
        mask[w] = bits;
        bits = 0u;
      }
      bits |= 1u << (up % 32u);
      node = up;
      ++depth;
    }
    for (mask[w] = bits; w; --w) mask[w - 1u] = 0u;
    p.pos[t] = r.cached[b] + depth;
  }
}

// One work-group: the requests, a thread each; ROWS: then the rows too.
template <bool ROWS>
__global__ __launch_bounds__(kMaxRequests) void plan_kernel(PlanArgs a) {
  const mi_block_plan& p = a.p;
  __shared__ Requests r;
  __shared__ uint32_t back_at[kMaxRequests + 1], need_of[kMaxRequests], parents[ROWS ? kOneGroup : 1];
  const uint32_t b = threadIdx.x;
  const bool request = b < p.requests;
  const uint32_t head = p.ring_at[0], count = p.ring_at[1];
  uint32_t cached = 0, added = 0, held = 0, need = 0, before_held = 0;
  bool ok = true;
  if (request) {
    cached = p.cached[b];
    added = p.added[b];
    before_held = held = p.held[b];
    const uint64_t keys = (uint64_t)cached + added;
    ok = keys <= kMaxKeys && held <= p.table_stride && (uint64_t)held * p.page >= cached && added <= p.rows &&
         (!p.parent || added <= 32u * p.words);
    need = ok ? ((uint32_t)keys + p.page - 1u) / p.page : 0u;
    ok = ok && need <= p.table_stride;
  }
  if constexpr (ROWS)
    if (p.parent)
      for (uint32_t t = b; t < p.rows; t += blockDim.x) parents[t] = p.parent[t];
  if (!ok) {  // (one request that cannot be makes the sum of the rows too large)
    added = kMaxRows + 1u;
    need = held = 0u;
  }
  Three all;  // (1024 requests of 2^21 pages at most: none of the sums wraps)
  const Three before = sums_before(Three{added, need > held ? need - held : 0u, held > need ? held - need : 0u}, all);
  const bool sound = all.a <= p.rows && head < p.ring_len && count <= p.ring_len && (uint64_t)count + all.c <= p.ring_len;
  const bool planned = sound && all.b <= count;
  if (request) {
    r.start[b] = p.row_start[b] = planned ? before.a : 0u;
    r.cached[b] = cached;
    r.held[b] = held;
    r.taken[b] = before.b;
    back_at[b] = before.c;
    need_of[b] = need;
    p.held_out[b] = planned ? need : before_held;
    if constexpr (!ROWS) {
      a.ws[2u + 2u * b] = held;
      a.ws[3u + 2u * b] = before.b;
    }
  }
  if (b == 0) {
    r.start[p.requests] = p.row_start[p.requests] = planned ? all.a : 0u;
    back_at[p.requests] = all.c;
    p.ring_at_out[0] = planned ? (uint32_t)(((uint64_t)head + all.b) % p.ring_len) : head;
    p.ring_at_out[1] = planned ? count - all.b + all.c : count;
    if constexpr (!ROWS) {
      a.ws[0] = planned ? 1u : 0u;
      a.ws[1] = head;
    }
    if (!planned && p.flag) *p.flag = sound ? MI_STATUS_NO_PAGES : MI_STATUS_BAD_ROWS;
  }
  __syncthreads();
  if (planned)  // what goes back, a thread a page
    for (uint32_t i = b; i < all.c; i += blockDim.x) {
      const uint32_t of = find(back_at, p.requests, i), page = p.tables[(size_t)of * p.table_stride + need_of[of] + (i - back_at[of])];
      p.ring[(uint32_t)(((uint64_t)head + count + i) % p.ring_len)] = page;
    }
  if constexpr (ROWS) plan_rows(a, r, planned, head, 0u, p.rows, parents);
}
__global__ __launch_bounds__(256) void plan_rows_kernel(PlanArgs a) {
  const mi_block_plan& p = a.p;
  __shared__ Requests r;
  __shared__ uint32_t parents[256];
  const uint32_t begin = blockIdx.x * 256u, end = min(begin + 256u, p.rows);
  if (p.parent && begin + threadIdx.x < end) parents[threadIdx.x] = p.parent[begin + threadIdx.x];
  for (uint32_t b = threadIdx.x; b < p.requests; b += 256u) {
    r.start[b] = p.row_start[b];
    r.cached[b] = p.cached[b];
    r.held[b] = a.ws[2u + 2u * b];
    r.taken[b] = a.ws[3u + 2u * b];
  }
  if (threadIdx.x == 0) r.start[p.requests] = p.row_start[p.requests];
  const bool planned = a.ws[0] != 0u;
  const uint32_t head = a.ws[1];
  __syncthreads();
  plan_rows(a, r, planned, head, begin, end, parents);
}

struct MoveArgs {
  uint16_t *k, *v;
  const uint32_t *from, *to;
  uint32_t* flag;
  size_t layer_stride, row_stride, head_stride;
  uint32_t rows, per;
};
// grid (groups, kv_heads, layers): a work-group takes one group's rows of one head, K and V, into registers, and stores them when
// all are there: rows may move onto one another. 16 bytes a thread and piece, U pieces of each. Bound by the bytes: 32 pages of 64 rows
// of 2 heads of 256 in 40 layers (171 MB in, as many out) 37.5 us, 4.6 TB/s (a copy 4.9; with loads that the caches keep 42.7; with
// such stores also passed by the caches 39.2).
template <int HD, int U>
__global__ __launch_bounds__(256) void kv_move_kernel(MoveArgs a) {
  constexpr uint32_t PPR = HD / 8;
  const size_t base = blockIdx.z * a.layer_stride + blockIdx.y * a.head_stride;
  const uint32_t* from = a.from + (size_t)blockIdx.x * a.per;
  const uint32_t* to = a.to + (size_t)blockIdx.x * a.per;
  u4_t k[U], v[U];
  uint32_t whence[U], at[U];
  // (all of the lists' entries first: loads come back in order, and an entry asked for behind rows would wait for them)
#pragma unroll
  for (uint32_t u = 0; u < U; ++u) {
    const uint32_t i = min((256u * u + threadIdx.x) / PPR, a.per - 1u);
    whence[u] = from[i];
    at[u] = to[i];
  }
  bool outside = false;
#pragma unroll
  for (uint32_t u = 0; u < U; ++u) {
    if ((256u * u + threadIdx.x) / PPR >= a.per) at[u] = kNone;
    const bool moves = whence[u] < a.rows && at[u] < a.rows;
    outside |= !moves && at[u] != kNone;
    if (!moves) at[u] = kNone;
    // (what does not move loads row 0: a branch would wait for what was loaded in it)
    const size_t o = base + (size_t)(moves ? whence[u] : 0u) * a.row_stride + 8u * (threadIdx.x % PPR);
    k[u] = __builtin_nontemporal_load(as_global(reinterpret_cast<const u4_t*>(a.k + o)));
    v[u] = __builtin_nontemporal_load(as_global(reinterpret_cast<const u4_t*>(a.v + o)));
  }
  if (outside && a.flag) *a.flag = MI_STATUS_BAD_PAGE;
  wait_memory();
  __syncthreads();
#pragma unroll
  for (uint32_t u = 0; u < U; ++u)
    if (at[u] != kNone) {
      const size_t o = base + (size_t)at[u] * a.row_stride + 8u * (threadIdx.x % PPR);
      *as_global(reinterpret_cast<u4_t*>(a.k + o)) = k[u];
      *as_global(reinterpret_cast<u4_t*>(a.v + o)) = v[u];
    }
}
template <int HD>
void launch_move(const MoveArgs& a, const dim3& grid, hipStream_t st) {
  const uint32_t pieces = (a.per * (HD / 8u) + 255u) / 256u;
  if (pieces <= 1u) kv_move_kernel<HD, 1><<<grid, 256, 0, st>>>(a);
  else if (pieces <= 2u) kv_move_kernel<HD, 2><<<grid, 256, 0, st>>>(a);
  else if (pieces <= 4u) kv_move_kernel<HD, 4><<<grid, 256, 0, st>>>(a);
  else kv_move_kernel<HD, 8><<<grid, 256, 0, st>>>(a);
}
bool off(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1u)) != 0; }

}  // namespace
}  // namespace mi

using namespace mi;

extern "C" {

size_t mi_block_tables_ws(uint32_t requests) {
  return requests == 0 || requests > kMaxRequests ? 0 : (size_t)(2u + 2u * requests) * 4u;
}

int mi_block_tables(const mi_block_plan* plan, void* ws, size_t ws_bytes, void* stream) {
  if (!plan) return mi_fail(MI_ERR_ARG, "block_tables: null pointer");
  const mi_block_plan& p = *plan;
  for (const void* q : {(const void*)p.cached, (const void*)p.added, (const void*)p.held, (const void*)p.held_out, (const void*)p.tables,
                        (const void*)p.ring, (const void*)p.ring_at, (const void*)p.ring_at_out, (const void*)p.row_start,
                        (const void*)p.seq, (const void*)p.slot, (const void*)p.pos})
    if (!q || off(q, 4)) return mi_fail(MI_ERR_ARG, "block_tables: null or misaligned array (4 bytes)");
  if (off(p.parent, 4) || off(p.mask, 4) || off(p.flag, 4))
    return mi_fail(MI_ERR_ARG, "block_tables: misaligned parent, mask or flag (4 bytes)");
  if (p.requests == 0 || p.requests > kMaxRequests || p.rows == 0 || p.rows > kMaxRows)
    return mi_fail(MI_ERR_SHAPE, "block_tables: 1..1024 requests, 1..65535 rows");
  if (p.page == 0 || p.n_pages == 0 || p.table_stride == 0 || p.ring_len == 0)
    return mi_fail(MI_ERR_ARG, "block_tables: page size, page count, table_stride or ring_len 0");
  if ((uint64_t)p.page * p.n_pages > 0xFFFFFFFFull) return mi_fail(MI_ERR_SHAPE, "block_tables: above 2^32 cache rows");
  if (p.table_stride > kMaxTable || p.ring_len > 1u << 31 || p.page > kMaxPage)
    return mi_fail(MI_ERR_SHAPE, "block_tables: pages of 2^20 positions, tables of 2^21 pages, a ring of 2^31 at most");
  if (p.parent ? !p.mask || p.words == 0 || p.words > kMaxWords : p.mask || p.words)
    return mi_fail(MI_ERR_ARG, "block_tables: masks of 1..64 words go with parents");
  if (!ws || off(ws, 4) || ws_bytes < mi_block_tables_ws(p.requests))
    return mi_fail(MI_ERR_ARG, "block_tables: the workspace is null, misaligned (4 bytes) or below mi_block_tables_ws");
  const PlanArgs a{p, static_cast<uint32_t*>(ws)};
  hipStream_t st = (hipStream_t)stream;
  // a thread a request, and some for the rows
  const uint32_t threads = std::max((p.requests + 63u) / 64u * 64u, p.rows <= 256u ? 256u : 1024u);
  if (p.rows <= kOneGroup) {
    plan_kernel<true><<<1, threads, 0, st>>>(a);
  } else {
    plan_kernel<false><<<1, threads, 0, st>>>(a);
    plan_rows_kernel<<<(p.rows + 255u) / 256u, 256, 0, st>>>(a);
  }
  return mi_hip((int)hipGetLastError(), "block_tables");
}

int mi_kv_move(uint16_t* kv_k, uint16_t* kv_v, uint32_t layers, size_t layer_stride, size_t row_stride, size_t head_stride,
               uint32_t kv_heads, uint32_t head_dim, uint32_t rows, const uint32_t* from, const uint32_t* to, uint32_t groups,
               uint32_t per, uint32_t* flag, void* stream) {
  if (!kv_k || !kv_v || !from || !to) return mi_fail(MI_ERR_ARG, "kv_move: null pointer");
  if (off(kv_k, 16) || off(kv_v, 16) || off(from, 4) || off(to, 4) || off(flag, 4))
    return mi_fail(MI_ERR_ARG, "kv_move: misaligned pointer (K and V 16 bytes)");
  if (row_stride % 8 || head_stride % 8 || layer_stride % 8)
    return mi_fail(MI_ERR_ARG, "kv_move: strides must keep 8-element alignment");
  if (head_dim != 128 && head_dim != 256) return mi_fail(MI_ERR_SHAPE, "kv_move: head_dim 128 or 256");
  if (layers == 0 || layers > 65535 || kv_heads == 0 || kv_heads > 65535 || rows == 0 || groups == 0 || groups > 1u << 20 || per == 0 ||
      per > 64)
    return mi_fail(MI_ERR_SHAPE, "kv_move: layers and kv_heads 1..65535, rows from 1, groups 1..2^20 of 1..64 rows");
  const MoveArgs a{kv_k, kv_v, from, to, flag, layer_stride, row_stride, head_stride, rows, per};
  const dim3 grid(groups, kv_heads, layers);
  if (head_dim == 128) launch_move<128>(a, grid, (hipStream_t)stream);
  else launch_move<256>(a, grid, (hipStream_t)stream);
  return mi_hip((int)hipGetLastError(), "kv_move");
}

}  // extern "C"
