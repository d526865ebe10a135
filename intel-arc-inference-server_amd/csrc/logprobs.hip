// logprobs.hip - what a row of logits says about given tokens: log probability and rank of one token, the
// distribution's entropy, the most likely tokens.
//
// With m = max_i x_i, d_i = x_i - m, Z = sum_i e^(d_i), T = sum_i e^(d_i) d_i over the vocabulary:
//   log p_i = d_i - log Z,   entropy = log Z - T / Z,   rank(t) = #{i : x_i > x_t, or x_i = x_t and i < t}
// One pass: a lane keeps its own running maximum with its Z and T (a maximum that rises by -delta turns them into
// Z e^delta and (T + delta Z) e^delta), a wave its 64 best tokens sorted over its lanes, best first. A token is
// better than another when its logit is larger, or equal with the lower index. Whatever beats the wave's k-th best is
// put in: few at once by a shift of the lanes behind its place, many at once as a sorted 64 merged with the list.
#include <algorithm>
#include <type_traits>

#include "mi_capi_internal.h"
#include "mi_common.h"

namespace mi {
namespace {

constexpr uint32_t kMaxTop = 64, kNone = 0xFFFFFFFFu;
constexpr float kLog2e = 1.4426950408889634f;

struct LogprobArgs {
  const float* logits;
  size_t row_stride;
  const uint32_t* tokens;
  uint32_t vocab, top, slices, slice;  // `slice` tokens each, a multiple of 4
  float *logprob, *entropy, *top_logprobs;
  uint32_t *rank, *top_ids;
  // per (row, slice): (m, Z, T, count) and `top` (value, id) pairs
  f4_t* stats;
  u2_t* lists;
};

// ---- the statistics ----
struct Stats {
  float m = -INFINITY, z = 0.f, t = 0.f;
  // the maximum rises to `to` (not NaN)
  __device__ __forceinline__ void raise(float to) {
    if (to > m) {
      if (z != 0.f) {  // (a NaN stays one)
        const float delta = fmaxf(m - to, -1e30f), a = __builtin_amdgcn_exp2f(delta * kLog2e);
        t = __builtin_fmaf(delta, z, t) * a;
        z *= a;
      }
      m = to;
    }
  }
  __device__ __forceinline__ void merge(Stats o) {
    raise(o.m);
    o.raise(m);
    z += o.z;
    t += o.t;
  }
};
template <uint32_t X>
__device__ __forceinline__ uint32_t xor_lane(uint32_t v) {
  auto dpp = [](uint32_t x, auto c) { return (uint32_t)__builtin_amdgcn_mov_dpp((int)x, decltype(c)::value, 0xF, 0xF, false); };
  if constexpr (X == 1) return dpp(v, std::integral_constant<int, 0xB1>{});        // quad_perm 1, 0, 3, 2
  else if constexpr (X == 2) return dpp(v, std::integral_constant<int, 0x4E>{});   // quad_perm 2, 3, 0, 1
  else if constexpr (X == 4)                                                       // half mirror (^ 7), then quad ^ 3
    return dpp(dpp(v, std::integral_constant<int, 0x141>{}), std::integral_constant<int, 0x1B>{});
  else if constexpr (X == 8) return dpp(v, std::integral_constant<int, 0x128>{});  // rotated by 8 in the row of 16
  else {
    float a = __builtin_bit_cast(float, v), b = a;
    if constexpr (X == 16) lane_swap16(a, b);
    else lane_swap32(a, b);
    return __builtin_bit_cast(uint32_t, (threadIdx.x & X) ? a : b);
  }
}
template <uint32_t X>
__device__ __forceinline__ void merge_lanes(Stats& s) {
  const auto f = [](float x) { return __builtin_bit_cast(float, xor_lane<X>(__builtin_bit_cast(uint32_t, x))); };
  Stats o;
  o.m = f(s.m);
  o.z = f(s.z);
  o.t = f(s.t);
  s.merge(o);
}

// ---- the best tokens ----
struct Entry {
  float v = -INFINITY;
  uint32_t id = kNone;  // (no token: behind every token)
};
__device__ __forceinline__ bool better(Entry a, Entry b) { return a.v > b.v || (a.v == b.v && a.id < b.id); }
template <uint32_t X>
__device__ __forceinline__ Entry xor_entry(Entry e) {
  return {__builtin_bit_cast(float, xor_lane<X>(__builtin_bit_cast(uint32_t, e.v))), xor_lane<X>(e.id)};
}
// the better or the worse of this lane's and its partner's
template <uint32_t X>
__device__ __forceinline__ void exchange(Entry& e, bool keep_better) {
  const Entry o = xor_entry<X>(e);
  if (better(o, e) == keep_better) e = o;
}
template <uint32_t X>
__device__ __forceinline__ void half_clean(Entry& e, uint32_t lane, bool best_first) {  // strides X .. 1
  exchange<X>(e, ((lane & X) == 0) == best_first);
  if constexpr (X > 1) half_clean<X / 2>(e, lane, best_first);
}
// 64 entries sorted, best first (or last)
__device__ __forceinline__ void sort64(Entry& e, uint32_t lane, bool best_first) {
  half_clean<1>(e, lane, (lane & 2u) == 0);
  half_clean<2>(e, lane, (lane & 4u) == 0);
  half_clean<4>(e, lane, (lane & 8u) == 0);
  half_clean<8>(e, lane, (lane & 16u) == 0);
  half_clean<16>(e, lane, (lane & 32u) == 0);
  half_clean<32>(e, lane, best_first);
}
// the best 64 of a list (best first) and another (best last)
__device__ __forceinline__ void merge64(Entry& list, Entry rising, uint32_t lane) {
  if (better(rising, list)) list = rising;
  half_clean<32>(list, lane, true);
}
__device__ __forceinline__ Entry entry_at(Entry e, uint32_t lane) {
  return {lane_f(e.v, (int)lane), (uint32_t)__builtin_amdgcn_readlane((int)e.id, (int)lane)};
}
__device__ __forceinline__ void insert(Entry& list, Entry e, uint32_t lane) {
  const uint32_t at = (uint32_t)__popcll(__ballot(better(list, e)));
  const Entry up = {__builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, list.v), 0x138, 0xF, 0xF, false)),
                    (uint32_t)__builtin_amdgcn_update_dpp(0, (int)list.id, 0x138, 0xF, 0xF, false)};  // (the lane below's)
  if (lane == at) list = e;
  else if (lane > at) list = up;
}
// puts in the lanes' entries that beat the list's k-th
__device__ __forceinline__ void put(Entry& list, Entry& last, Entry e, uint32_t k, uint32_t lane) {
  const bool in = better(e, last);
  uint64_t who = __ballot(in);
  if (!who) return;
  if (__popcll(who) > 8) {
    if (!in) e = Entry{};
    sort64(e, lane, false);
    merge64(list, e, lane);
  } else {
    for (; who; who &= who - 1u) insert(list, entry_at(e, (uint32_t)__builtin_ctzll(who)), lane);
  }
  last = entry_at(list, k - 1u);
}

// the row's answers, from its whole statistics and list (one wave)
__device__ __forceinline__ void answer(const LogprobArgs& a, uint32_t row, const Stats& s, uint32_t count, Entry list,
                                       uint32_t lane) {
  const float log_z = logf(s.z);
  if (lane == 0) {
    if (a.entropy) a.entropy[row] = log_z - s.t / s.z;
    if (a.tokens) {
      const uint32_t t = a.tokens[row];
      const float x = t < a.vocab ? a.logits[(size_t)row * a.row_stride + t] : __builtin_bit_cast(float, kNanBits);
      if (a.logprob) a.logprob[row] = (x - s.m) - log_z;
      if (a.rank) a.rank[row] = x != x ? kNone : count;
    }
  }
  if (lane < a.top) {
    a.top_ids[(size_t)row * a.top + lane] = list.id;
    a.top_logprobs[(size_t)row * a.top + lane] = list.id == kNone ? -INFINITY : (list.v - s.m) - log_z;
  }
}

// grid (slices, rows): 4 waves walk a slice of the row's tokens, each 256 at a time
__global__ __launch_bounds__(256) void logprobs_kernel(LogprobArgs a) {
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, row = blockIdx.y;
  const float* x = a.logits + (size_t)row * a.row_stride;
  const uint32_t begin = blockIdx.x * a.slice, end = min(begin + a.slice, a.vocab);
  const uint32_t t = a.tokens ? a.tokens[row] : kNone;
  const float xt = t < a.vocab ? x[t] : INFINITY;
  const uint32_t ahead = min(t, end);  // equal logits count up to here
  Stats s;
  uint32_t count = 0;
  Entry list, last;
  constexpr uint32_t U = 4;
  for (uint32_t i0 = begin + 4u * threadIdx.x; i0 - 4u * lane < end; i0 += 1024u * U) {
    f4_t v[U];
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) {
      const uint32_t i = i0 + 1024u * u;
      v[u] = f4_t{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
      if (i + 4u <= end) v[u] = *reinterpret_cast<const f4_any*>(x + i);
      else
#pragma unroll
        for (uint32_t r = 0; r < 4; ++r)
          if (i + r < end) v[u][r] = x[i + r];
    }
    float most[U], all = -INFINITY;
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) {
      most[u] = fmaxf(fmaxf(v[u][0], v[u][1]), fmaxf(v[u][2], v[u][3]));
      all = fmaxf(all, most[u]);
    }
    s.raise(all);
    const float ref = s.m == -INFINITY ? 0.f : s.m;
#pragma unroll
    for (uint32_t u = 0; u < U; ++u)
#pragma unroll
      for (uint32_t r = 0; r < 4; ++r) {
        const float d = v[u][r] - ref, e = __builtin_amdgcn_exp2f(d * kLog2e);
        s.z += e;
        s.t = __builtin_fmaf(e, fmaxf(d, -1e30f), s.t);  // (-inf counts nothing)
        count += v[u][r] > xt || (v[u][r] == xt && i0 + 1024u * u + r < ahead) ? 1u : 0u;
      }
    if (a.top) {
      uint32_t hit = 0;  // the pieces with a logit that may be among the best
#pragma unroll
      for (uint32_t u = 0; u < U; ++u) hit |= __ballot(most[u] >= last.v) ? 1u << u : 0u;
      while (hit) {
        const uint32_t u = (uint32_t)__builtin_ctz(hit);
        hit &= hit - 1u;
        const f4_t w = u == 0 ? v[0] : u == 1 ? v[1] : u == 2 ? v[2] : v[3];
#pragma unroll 1
        for (uint32_t r = 0; r < 4; ++r) {
          const uint32_t i = i0 + 1024u * u + r;
          put(list, last, Entry{r == 0 ? w[0] : r == 1 ? w[1] : r == 2 ? w[2] : w[3], i < end ? i : kNone}, a.top, lane);
        }
      }
    }
  }
  merge_lanes<1>(s);
  merge_lanes<2>(s);
  merge_lanes<4>(s);
  merge_lanes<8>(s);
  merge_lanes<16>(s);
  merge_lanes<32>(s);
  count = (uint32_t)wave_sum((float)count);  // (below 2^24: exact)
  __shared__ float sm[4], sz[4], stt[4];
  __shared__ uint32_t sc[4];
  __shared__ float sv[4][64];
  __shared__ uint32_t si[4][64];
  if (lane == 0) {
    sm[wave] = s.m;
    sz[wave] = s.z;
    stt[wave] = s.t;
    sc[wave] = count;
  }
  sv[wave][lane] = list.v;
  si[wave][lane] = list.id;
  __syncthreads();
  if (wave) return;
#pragma unroll 1
  for (uint32_t w = 1; w < 4; ++w) {
    Stats o;
    o.m = sm[w];
    o.z = sz[w];
    o.t = stt[w];
    s.merge(o);
    count += sc[w];
    if (a.top) merge64(list, Entry{sv[w][63u - lane], si[w][63u - lane]}, lane);
  }
  if (a.slices == 1) {
    answer(a, row, s, count, list, lane);
    return;
  }
  const size_t at = (size_t)row * a.slices + blockIdx.x;
  if (lane == 0) a.stats[at] = f4_t{s.m, s.z, s.t, (float)count};
  if (lane < a.top) a.lists[at * a.top + lane] = u2_t{__builtin_bit_cast(uint32_t, list.v), list.id};
}

// one work-group per row: its slices' statistics and lists
__global__ __launch_bounds__(256) void logprobs_join_kernel(LogprobArgs a) {
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, row = blockIdx.x;
  const f4_t* stats = a.stats + (size_t)row * a.slices;
  const u2_t* lists = a.lists + (size_t)row * a.slices * a.top;
  Stats s;
  float count = 0.f;
  for (uint32_t i = threadIdx.x; i < a.slices; i += 256u) {
    const f4_t p = stats[i];
    Stats o;
    o.m = p[0];
    o.z = p[1];
    o.t = p[2];
    s.merge(o);
    count += p[3];
  }
  merge_lanes<1>(s);
  merge_lanes<2>(s);
  merge_lanes<4>(s);
  merge_lanes<8>(s);
  merge_lanes<16>(s);
  merge_lanes<32>(s);
  count = wave_sum(count);
  Entry list;
  if (a.top)
    for (uint32_t i = wave; i < a.slices; i += 4u) {
      Entry e;
      if (63u - lane < a.top) {
        const u2_t p = lists[(size_t)i * a.top + 63u - lane];
        e = Entry{__builtin_bit_cast(float, p.x), p.y};
      }
      merge64(list, e, lane);
    }
  __shared__ float sm[4], sz[4], stt[4], sc[4];
  __shared__ float sv[4][64];
  __shared__ uint32_t si[4][64];
  if (lane == 0) {
    sm[wave] = s.m;
    sz[wave] = s.z;
    stt[wave] = s.t;
    sc[wave] = count;
  }
  sv[wave][lane] = list.v;
  si[wave][lane] = list.id;
  __syncthreads();
  if (wave) return;
#pragma unroll 1
  for (uint32_t w = 1; w < 4; ++w) {
    Stats o;
    o.m = sm[w];
    o.z = sz[w];
    o.t = stt[w];
    s.merge(o);
    count += sc[w];
    if (a.top) merge64(list, Entry{sv[w][63u - lane], si[w][63u - lane]}, lane);
  }
  answer(a, row, s, (uint32_t)count, list, lane);
}

// The slices of a row: one where the rows alone fill the chip.
void pick_slices(uint32_t M, uint32_t vocab, uint32_t* slices, uint32_t* slice) {
  const uint32_t want = std::max(1u, 1024u / M), most = (vocab + 2047u) / 2048u;
  const uint32_t n = std::min(want, most);
  *slice = ((vocab + n - 1u) / n + 3u) / 4u * 4u;
  *slices = (vocab + *slice - 1u) / *slice;
}

}  // namespace
}  // namespace mi

using namespace mi;

extern "C" {

size_t mi_logprobs_ws(uint32_t M, uint32_t vocab_used, uint32_t top) {
  if (M == 0 || vocab_used == 0) return 0;
  uint32_t slices, slice;
  pick_slices(M, vocab_used, &slices, &slice);
  return slices == 1 ? 0 : (size_t)M * slices * (16u + 8u * (size_t)top);
}

int mi_logprobs(const float* logits, size_t row_stride, const uint32_t* tokens, uint32_t M, uint32_t vocab_used,
                uint32_t top, float* logprob, uint32_t* rank, float* entropy, uint32_t* top_ids, float* top_logprobs,
                void* ws, size_t ws_bytes, void* stream) {
  if (!logits || (reinterpret_cast<uintptr_t>(logits) & 3u)) return mi_fail(MI_ERR_ARG, "logprobs: null or misaligned logits");
  if (M == 0 || M > 65535 || vocab_used == 0 || vocab_used > 1u << 23)
    return mi_fail(MI_ERR_SHAPE, "logprobs: M 1..65535, vocab_used 1..2^23");
  if (row_stride < vocab_used) return mi_fail(MI_ERR_ARG, "logprobs: row_stride below vocab_used");
  if (top > kMaxTop) return mi_fail(MI_ERR_SHAPE, "logprobs: at most 64 top tokens");
  if ((logprob || rank) && !tokens) return mi_fail(MI_ERR_ARG, "logprobs: logprob and rank need tokens");
  if (top ? !top_ids || !top_logprobs : top_ids || top_logprobs)
    return mi_fail(MI_ERR_ARG, "logprobs: top_ids and top_logprobs go with top > 0");
  if (!logprob && !rank && !entropy && !top) return mi_fail(MI_ERR_ARG, "logprobs: nothing is asked");
  const size_t need = mi_logprobs_ws(M, vocab_used, top);
  if (need && (!ws || (reinterpret_cast<uintptr_t>(ws) & 15u) || ws_bytes < need))
    return mi_fail(MI_ERR_ARG, "logprobs: the workspace is null, misaligned (16 bytes) or below mi_logprobs_ws");
  LogprobArgs a{logits, row_stride, tokens, vocab_used, top, 1, vocab_used, logprob, entropy, top_logprobs, rank, top_ids,
                nullptr, nullptr};
  pick_slices(M, vocab_used, &a.slices, &a.slice);
  if (need) {
    a.stats = static_cast<f4_t*>(ws);
    a.lists = reinterpret_cast<u2_t*>(a.stats + (size_t)M * a.slices);
  }
  hipStream_t st = (hipStream_t)stream;
  logprobs_kernel<<<dim3(a.slices, M), 256, 0, st>>>(a);
  if (a.slices > 1) logprobs_join_kernel<<<M, 256, 0, st>>>(a);
  return mi_hip((int)hipGetLastError(), "logprobs");
}

}  // extern "C"
