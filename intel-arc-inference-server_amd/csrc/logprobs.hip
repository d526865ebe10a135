// logprobs.hip - what a row of logits says about given tokens: log probability and rank of one token, the
// distribution's entropy, the most likely tokens.
//
// With m = max_i x_i, d_i = x_i - m, Z = sum_i e^(d_i), T = sum_i e^(d_i) d_i over the vocabulary:
//   log p_i = d_i - log Z,   entropy = log Z - T / Z,   rank(t) = #{i : x_i > x_t, or x_i = x_t and i < t}
// One pass: a lane keeps its own running maximum with its Z and T in base 2 (a maximum that rises by -delta turns them into
// Z 2^delta and (T + delta Z) 2^delta), a wave its 64 best tokens sorted over its lanes, best first. A token is better than
// another when its logit is larger, or equal with the lower index. What beats the wave's k-th best and reaches the
// work-group's bound is put in: few at once by a shift of the lanes behind its place, many at once as a sorted 64 merged
// with the list. The bound: with W waves each publishes its ceil(k / W)-th best, and k logits reach the least of these,
// which is close to the k-th best of all. In the first step a wave takes it from its lanes' maxima, so that of the first
// 4096 tokens hardly more than k go into a list (each wave by its own k-th best alone put in four times as many).
// What bounds it: the memory's stream, with the vector ALUs close behind (about ten instructions per logit); few rows are
// bound by their two launches' chains of loads. Each wave's next 4 KiB are loaded ahead of the work on the present ones.
// Measured (MI355X, vocabulary 151936): 2048 rows with the 20 best 323 -> 271 us by the bound (-30) and the loads ahead (-22), 246
// with the 5 best, 234 with none (5.3 TB/s; a plain read of those bytes 6.7); 333 rows with 5 66 -> 55; one row with 20
// 33 -> 18.7 in 149 slices (the lanes' statistics by one wave maximum, eight waves in the join, its loads all at its start).
#include <algorithm>
#include <type_traits>

#include "mi_capi_internal.h"
#include "mi_common.h"

namespace mi {
namespace {

constexpr uint32_t kMaxTop = 64, kNone = 0xFFFFFFFFu;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

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
// m: the maximum; z = sum of e^(x - m) = 2^d, t = sum of 2^d d
struct Stats {
  float m = -INFINITY, z = 0.f, t = 0.f;
  // the maximum rises to `to` (not NaN)
  __device__ __forceinline__ void raise(float to) {
    if (to > m) {
      if (z != 0.f) {  // (a NaN stays one)
        const float delta = fmaxf((m - to) * kLog2e, -1e30f), a = __builtin_amdgcn_exp2f(delta);
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
// the lanes' into one, by the wave's maximum
__device__ __forceinline__ void merge_lanes(Stats& s) {
  s.raise(wave_max(s.m));
  s.z = wave_sum(s.z);
  s.t = wave_sum(s.t);
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
// puts in the lanes' entries that beat the list's k-th and reach `cut`
__device__ __forceinline__ void put(Entry& list, Entry& last, Entry e, float cut, uint32_t k, uint32_t lane) {
  const bool in = better(e, last) && e.v >= cut;
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
// W waves' bound: k entries that any of them has seen reach it
template <uint32_t W>
struct Bound {
  float share[W];  // each wave's ceil(k / W)-th best
  __device__ __forceinline__ void publish(uint32_t wave, uint32_t lane, float v) {
    if (lane == 0) __hip_atomic_store(&share[wave], v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
  }
  __device__ __forceinline__ float get() const {
    float v = INFINITY;
#pragma unroll
    for (uint32_t w = 0; w < W; ++w) v = fminf(v, __hip_atomic_load(&share[w], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP));
    return v;
  }
};
// the k-th largest of the lanes' values (NaN counts as -inf), by taking the largest away
__device__ __forceinline__ float kth_largest(float v, uint32_t k, uint32_t lane) {
  float m = wave_max(v);
#pragma unroll 1
  for (uint32_t i = 1; i < k; ++i) {
    if (lane == (uint32_t)__builtin_ctzll(__ballot(v == m) | 1ull << 63)) v = -INFINITY;
    m = wave_max(v);
  }
  return fmaxf(m, -INFINITY);
}

// W waves' statistics and lists into the first's: halves of the waves into the other half
template <uint32_t W>
struct Joint {
  float m[W], z[W], t[W], v[W][64];
  uint32_t count[W], id[W][64];
};
template <uint32_t W>  // whether this wave holds the joint ones
__device__ __forceinline__ bool join_waves(Joint<W>& j, Stats& s, uint32_t& count, Entry& list, uint32_t top, uint32_t wave, uint32_t lane) {
  merge_lanes(s);
#pragma unroll 1
  for (uint32_t step = W / 2; step; step /= 2) {
    if (lane == 0) {
      j.m[wave] = s.m;
      j.z[wave] = s.z;
      j.t[wave] = s.t;
      j.count[wave] = count;
    }
    j.v[wave][lane] = list.v;
    j.id[wave][lane] = list.id;
    __syncthreads();
    if (wave >= step) return false;
    Stats o;
    o.m = j.m[wave + step];
    o.z = j.z[wave + step];
    o.t = j.t[wave + step];
    s.merge(o);
    count += j.count[wave + step];
    if (top) merge64(list, Entry{j.v[wave + step][63u - lane], j.id[wave + step][63u - lane]}, lane);
  }
  return true;
}
// the given token's logit, NaN for none
__device__ __forceinline__ float token_logit(const LogprobArgs& a, uint32_t row, uint32_t* token) {
  const uint32_t t = *token = a.tokens ? a.tokens[row] : kNone;
  return t < a.vocab ? a.logits[(size_t)row * a.row_stride + t] : __builtin_bit_cast(float, kNanBits);
}
// the row's answers, from its whole statistics and list and its token's logit (one wave)
__device__ __forceinline__ void answer(const LogprobArgs& a, uint32_t row, const Stats& s, uint32_t count, Entry list, float xt,
                                       uint32_t lane) {
  const float log_z = logf(s.z);
  if (lane == 0) {
    if (a.entropy) a.entropy[row] = log_z - s.t / s.z * kLn2;
    if (a.logprob) a.logprob[row] = (xt - s.m) - log_z;
    if (a.rank) a.rank[row] = xt != xt ? kNone : count;
  }
  if (lane < a.top) {
    a.top_ids[(size_t)row * a.top + lane] = list.id;
    a.top_logprobs[(size_t)row * a.top + lane] = list.id == kNone ? -INFINITY : (list.v - s.m) - log_z;
  }
}

// grid (slices, rows): 4 waves walk a slice of the row's tokens, each 256 at a time
__global__ __launch_bounds__(256, 5) void logprobs_kernel(LogprobArgs a) {
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, row = blockIdx.y;
  const float* x = a.logits + (size_t)row * a.row_stride;
  const uint32_t begin = blockIdx.x * a.slice, end = min(begin + a.slice, a.vocab);
  uint32_t token, ahead = 0;
  float xt = 0.f;  // (loaded behind the first step's tokens, whose use it must not delay)
  Stats s;
  uint32_t count = 0;  // (of the wave)
  Entry list, last;
  __shared__ Bound<4> bound;
  const uint32_t share = (a.top + 3u) / 4u;
  constexpr uint32_t U = 4;
  auto load = [&](f4_t (&to)[U], uint32_t i0) {
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) {
      const uint32_t i = i0 + 1024u * u;
      to[u] = f4_t{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
      if (i + 4u <= end) to[u] = *as_global(reinterpret_cast<const f4_any*>(x + i));
      else if (i < end)
#pragma unroll
        for (uint32_t r = 0; r < 4; ++r)
          if (i + r < end) to[u][r] = *as_global(x + i + r);
    }
  };
  f4_t next[U];
  load(next, begin + 4u * threadIdx.x);
  // (the first step is every wave's, tokens or not: they meet in it)
  for (uint32_t i0 = begin + 4u * threadIdx.x, first = 1; first || i0 - 4u * lane < end; i0 += 1024u * U, first = 0) {
    f4_t v[U];
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) v[u] = next[u];
    load(next, i0 + 1024u * U);
    if (first) {
      xt = token_logit(a, row, &token);
      ahead = min(token, end);  // equal logits count up to here
    }
    float most[U];
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) most[u] = fmaxf(fmaxf(v[u][0], v[u][1]), fmaxf(v[u][2], v[u][3]));
    const float all = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3]));
    s.raise(all);
    const float ref = s.m == -INFINITY ? 0.f : s.m;
#pragma unroll
    for (uint32_t u = 0; u < U; ++u)
#pragma unroll
      for (uint32_t r = 0; r < 4; ++r) {
        const float d = (v[u][r] - ref) * kLog2e, e = __builtin_amdgcn_exp2f(d);
        s.z += e;
        s.t = __builtin_fmaf(e, __builtin_elementwise_maximum(d, -1e30f), s.t);  // (-inf counts nothing)
      }
    if (a.top) {
      if (first) {
        bound.publish(wave, lane, kth_largest(all, share, lane));
        __syncthreads();
      }
      const float cut = fmaxf(last.v, bound.get());
      uint32_t hit = 0;  // the pieces with a logit that may be among the best
      if (__ballot(all >= cut)) {
#pragma unroll
        for (uint32_t u = 0; u < U; ++u) hit |= __ballot(most[u] >= cut) ? 1u << u : 0u;
      }
      if (hit) {
        while (hit) {
          const uint32_t u = (uint32_t)__builtin_ctz(hit);
          hit &= hit - 1u;
          const f4_t w = u == 0 ? v[0] : u == 1 ? v[1] : u == 2 ? v[2] : v[3];
          uint32_t of = 0;
#pragma unroll
          for (uint32_t r = 0; r < 4; ++r) of |= __ballot(w[r] >= cut) ? 1u << r : 0u;
          for (; of; of &= of - 1u) {
            const uint32_t r = (uint32_t)__builtin_ctz(of), i = i0 + 1024u * u + r;
            put(list, last, Entry{r == 0 ? w[0] : r == 1 ? w[1] : r == 2 ? w[2] : w[3], i < end ? i : kNone}, cut, a.top, lane);
          }
        }
        // (a list that holds fewer entries than the share keeps the first step's value, which is no larger)
        const float mine = lane_f(list.v, (int)(share - 1u));
        if (mine > -INFINITY) bound.publish(wave, lane, mine);
      }
    }
    // the tokens before t count where they are equal too; t lies within one step of one wave
    const uint32_t w0 = i0 - 4u * lane;
    if (w0 + 1024u * (U - 1u) + 256u <= ahead) {
#pragma unroll
      for (uint32_t u = 0; u < U; ++u)
#pragma unroll
        for (uint32_t r = 0; r < 4; ++r) count += (uint32_t)__popcll(__ballot(v[u][r] >= xt));
    } else if (w0 >= ahead) {
#pragma unroll
      for (uint32_t u = 0; u < U; ++u)
#pragma unroll
        for (uint32_t r = 0; r < 4; ++r) count += (uint32_t)__popcll(__ballot(v[u][r] > xt));
    } else {
#pragma unroll
      for (uint32_t u = 0; u < U; ++u)
#pragma unroll
        for (uint32_t r = 0; r < 4; ++r)
          count += (uint32_t)__popcll(__ballot(v[u][r] > xt || (v[u][r] == xt && i0 + 1024u * u + r < ahead)));
    }
  }
  __shared__ Joint<4> joint;
  if (!join_waves<4>(joint, s, count, list, a.top, wave, lane)) return;
  if (a.slices == 1) {
    answer(a, row, s, count, list, xt, lane);
    return;
  }
  const size_t at = (size_t)row * a.slices + blockIdx.x;
  if (lane == 0) a.stats[at] = f4_t{s.m, s.z, s.t, (float)count};
  if (lane < a.top) a.lists[at * a.top + lane] = u2_t{__builtin_bit_cast(uint32_t, list.v), list.id};
}

// one work-group of W waves per row: its slices' statistics, and their lists as one set of entries, 4 per lane at a time
template <uint32_t W>
__global__ __launch_bounds__(64 * W) void logprobs_join_kernel(LogprobArgs a) {
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, row = blockIdx.x, n = a.slices * a.top;
  const f4_t* stats = a.stats + (size_t)row * a.slices;
  const u2_t* entries = a.lists + (size_t)row * n;
  Stats s;
  uint32_t count = 0, token;
  Entry list, last;
  constexpr uint32_t U = 4;
  __shared__ Bound<W> bound;
  __shared__ Joint<W> joint;
  const uint32_t share = (a.top + W - 1u) / W;
  float xt = 0.f;
  for (uint32_t i0 = 0, first = 1; first || i0 < n; i0 += 64u * W * U, first = 0) {
    u2_t p[U];
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) {
      const uint32_t i = i0 + 64u * W * u + threadIdx.x;
      p[u] = i < n ? entries[i] : u2_t{0xFF800000u, kNone};
    }
    if (first) {  // (every load that the answers wait for is out before the first entry is looked at)
      f4_t q = {-INFINITY, 0.f, 0.f, 0.f};
      if (threadIdx.x < a.slices) q = stats[threadIdx.x];
      xt = token_logit(a, row, &token);
      float all = -INFINITY;
#pragma unroll
      for (uint32_t u = 0; u < U; ++u) all = fmaxf(all, __builtin_bit_cast(float, p[u].x));
      if (a.top) {
        bound.publish(wave, lane, kth_largest(all, share, lane));
        if constexpr (W > 1) __syncthreads();
      }
      s.m = q[0];
      s.z = q[1];
      s.t = q[2];
      count = (uint32_t)q[3];  // (below 2^24: exact)
    }
    if (a.top) {
      const float cut = fmaxf(last.v, bound.get());
#pragma unroll 1
      for (uint32_t u = 0; u < U; ++u) {
        const u2_t q = u == 0 ? p[0] : u == 1 ? p[1] : u == 2 ? p[2] : p[3];
        put(list, last, Entry{__builtin_bit_cast(float, q.x), q.y}, cut, a.top, lane);
      }
    }
  }
  for (uint32_t i = threadIdx.x + 64u * W; i < a.slices; i += 64u * W) {
    const f4_t p = stats[i];
    Stats o;
    o.m = p[0];
    o.z = p[1];
    o.t = p[2];
    s.merge(o);
    count += (uint32_t)p[3];
  }
  count = (uint32_t)wave_sum((float)count);
  if (join_waves<W>(joint, s, count, list, a.top, wave, lane)) answer(a, row, s, count, list, xt, lane);
}

// The slices of a row: one where the rows alone fill the chip.
void pick_slices(uint32_t M, uint32_t vocab, uint32_t* slices, uint32_t* slice) {
  const uint32_t want = std::max(1u, 1024u / M), most = (vocab + 1023u) / 1024u;
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
  if (a.slices > 8) logprobs_join_kernel<8><<<M, 512, 0, st>>>(a);
  else if (a.slices > 1) logprobs_join_kernel<1><<<M, 64, 0, st>>>(a);
  return mi_hip((int)hipGetLastError(), "logprobs");
}

}  // extern "C"
