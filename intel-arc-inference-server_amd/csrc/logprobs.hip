// logprobs.hip - what a row of logits says about given tokens: log probability and rank of one token, the
// distribution's entropy, the most likely tokens.
//
// With m = max_i x_i, d_i = x_i - m, Z = sum_i e^(d_i), T = sum_i e^(d_i) d_i over the vocabulary:
//   log p_i = d_i - log Z,   entropy = log Z - T / Z,   rank(t) = #{i : x_i > x_t, or x_i = x_t and i < t}
// One pass: a lane keeps its own running maximum with its Z and T in base 2 (a maximum that rises by -delta turns them into
// Z 2^delta and (T + delta Z) 2^delta). A token is better than another when its logit is larger, or equal with the lower
// index.
// Many rows, one work-group each: a wave keeps its 64 best tokens sorted over its lanes, best first. What beats the wave's
// k-th best and reaches the work-group's bound is put in: few at once by a shift of the lanes behind its place, many at once
// as a sorted 64 merged with the list. The bound: with W waves each publishes its ceil(k / W)-th best, and k logits reach
// the least of these, which is close to the k-th best of all. In the first step a wave takes it from its lanes' maxima, so
// that of the first 4096 tokens hardly more than k go into a list (each wave by its own k-th best alone put in four times
// as many). Few rows are cut into slices, which leave their statistics and the largest logit of each 256 tokens; a second
// launch joins them and reads again the few runs that can hold one of the k best.
// What bounds it: the memory's stream, with the vector ALUs close behind (about ten instructions per logit); few rows are
// bound by their two launches' chains of loads. Each wave's next 4 KiB are loaded ahead of the work on the present ones.
// Measured (MI355X, vocabulary 151936): 2048 rows with the 20 best 257 us (323 without the bound, which takes 30 off, and the
// loads ahead, 22), 244 with the 5 best, 232 with none (5.4 TB/s; a plain read of those bytes 6.7); 333 rows with 5 53 (66); one
// row with 20 11.6 in 149 slices (33 in one).
#include <algorithm>
#include <type_traits>

#include "mi_capi_internal.h"
#include "mi_pieces.h"

namespace mi {
namespace {

constexpr uint32_t kMaxRows = 65535, kMaxVocab = 1u << 23, kMaxTop = 64, kNone = 0xFFFFFFFFu;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct LogprobArgs {
  const float* logits;
  size_t row_stride;
  const uint32_t* tokens;
  uint32_t vocab, top, slices, slice;  // `slice` tokens each; a multiple of 1024 where there are several
  float *logprob, *entropy, *top_logprobs;
  uint32_t *rank, *top_ids;
  // where a row has several slices: (m, Z, T, count) per (row, slice), the largest logit per (row, 256 tokens)
  f4_t* stats;
  float* peaks;
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
    if (top) {
      j.v[wave][lane] = list.v;
      j.id[wave][lane] = list.id;
    }
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
// the row's answers, from its whole statistics (log_z = logf(s.z)) and its token's logit
__device__ __forceinline__ void answer(const LogprobArgs& a, uint32_t row, const Stats& s, uint32_t count, float log_z, float xt,
                                       uint32_t lane) {
  if (lane != 0) return;
  if (a.entropy) a.entropy[row] = log_z - s.t / s.z * kLn2;
  if (a.logprob) a.logprob[row] = (xt - s.m) - log_z;
  if (a.rank) a.rank[row] = xt != xt ? kNone : count;
}
__device__ __forceinline__ void answer_top(const LogprobArgs& a, uint32_t row, uint32_t place, Entry e, const Stats& s, float log_z) {
  a.top_ids[(size_t)row * a.top + place] = e.id;
  a.top_logprobs[(size_t)row * a.top + place] = e.id == kNone ? -INFINITY : (e.v - s.m) - log_z;
}

// four values' maxima over the wave: lane 0 the first's, 32 the second's, 16 the third's, 48 the fourth's
__device__ __forceinline__ float wave_max4(float a, float b, float c, float d) {
  lane_swap32(a, b);
  lane_swap32(c, d);
  float m = fmaxf(a, b), n = fmaxf(c, d);
  lane_swap16(m, n);
  m = fmaxf(m, n);
  auto with = [&](auto x) { m = fmaxf(m, __builtin_bit_cast(float, xor_lane<decltype(x)::value>(__builtin_bit_cast(uint32_t, m)))); };
  with(std::integral_constant<uint32_t, 1>{});
  with(std::integral_constant<uint32_t, 2>{});
  with(std::integral_constant<uint32_t, 4>{});
  with(std::integral_constant<uint32_t, 8>{});
  return m;
}

// grid (slices, rows): 4 waves walk a slice of the row's tokens, each 256 at a time. LISTS: the slice is the whole row, and
// the waves keep its best tokens; otherwise they leave the largest logit of each 256.
template <bool LISTS>
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
    if (LISTS && a.top) {
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
    const uint32_t w0 = i0 - 4u * lane;
    if (!LISTS && a.top) {
      const float peak = wave_max4(most[0], most[1], most[2], most[3]);
      const uint32_t at = w0 + 1024u * ((lane >> 5) + ((lane >> 3) & 2u));
      if ((lane & 15u) == 0 && at < end) a.peaks[(size_t)row * ((a.vocab + 255u) / 256u) + at / 256u] = peak;
    }
    // the tokens before t count where they are equal too; t lies within one step of one wave
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
  if (!join_waves<4>(joint, s, count, list, LISTS ? a.top : 0u, wave, lane)) return;
  if constexpr (LISTS) {
    const float log_z = logf(s.z);
    answer(a, row, s, count, log_z, xt, lane);
    if (lane < a.top) answer_top(a, row, lane, list, s, log_z);
  } else if (lane == 0) a.stats[(size_t)row * a.slices + blockIdx.x] = f4_t{s.m, s.z, s.t, (float)count};
}

// A work-group per row of several slices: joins their statistics, and finds the best tokens among the runs of 256 whose
// largest logit reaches a bound that k runs' reach, which it reads again: about 50 runs and 60 tokens at 151936 tokens and
// k = 20. The bound: of runs by their largest logit, equal ones by their place, the worst of the waves' ceil(k / W)-th best
// (k runs have a token at least as good as any token of a run behind it). A token's place among the best is the number of
// those read that are better. Where more tokens reach the bound than fit (equal logits, or fewer finite ones than k), the
// waves keep lists. One row of 151936 with the 20 best takes 11.6 us, 16 rows 15.2, 333 with the 5 best 53 (lists from
// every slice, as a row in one has them: 18.6, 23 and 54.2); one row of equal logits 21.6 (20.9).
__global__ __launch_bounds__(512) void logprobs_join_kernel(LogprobArgs a) {
  constexpr uint32_t W = 8, U = 4, B = 8, kFit = 1024;  // waves; a lane's runs looked at together; runs read together; tokens
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, row = blockIdx.x, runs = (a.vocab + 255u) / 256u;
  const float* x = a.logits + (size_t)row * a.row_stride;
  const f4_t* stats = a.stats + (size_t)row * a.slices;
  const float* peaks = a.peaks + (size_t)row * runs;
  __shared__ union {
    Joint<W> joint;
    struct {
      float v[kFit];
      uint32_t id[kFit];
    } fit;
  } sm;
  __shared__ float m[W], z[W], t[W];
  __shared__ uint32_t counts[W], fits, place[W];
  __shared__ float least[W];
  const uint32_t share = (a.top + W - 1u) / W;
  // (every load that the answers wait for goes out at once)
  f4_t q = {-INFINITY, 0.f, 0.f, 0.f};
  if (threadIdx.x < a.slices) q = stats[threadIdx.x];
  float p[U];
  auto load = [&](uint32_t r0) {  // run r is wave r % W's
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) {
      const uint32_t r = r0 + W * (64u * u + lane) + wave;
      p[u] = r < runs ? peaks[r] : -INFINITY;
    }
  };
  if (a.top) load(0);
  uint32_t token;
  const float xt = token_logit(a, row, &token);
  if (threadIdx.x == 0) fits = 0;
  if (a.top) {  // this wave's share of the bound, from the best run of each lane
    float v = p[0];
    uint32_t run = W * lane + wave;
#pragma unroll
    for (uint32_t u = 1; u < U; ++u)
      if (p[u] > v || v != v) {
        v = p[u];
        run = W * (64u * u + lane) + wave;
      }
    // its value, and of the lanes that have just that one as many as the share takes, the lowest: the last of their runs
    const float low = kth_largest(v, share, lane);
    const uint64_t with = __ballot(run < runs && v == low), above = __ballot(run < runs && v > low);
    const uint32_t need = share - min(share, (uint32_t)__popcll(above));
    const bool mine = ((with >> lane) & 1u) && (uint32_t)__popcll(with & ((1ull << lane) - 1u)) < need;
    const float last_of = wave_max(mine ? (float)run : 0.f);
    if (lane == 0) {
      least[wave] = low;
      place[wave] = (uint32_t)__popcll(with) < need ? kNone : (uint32_t)last_of;  // (too few: every token reaches it)
    }
  }
  __syncthreads();
  float cut = INFINITY;
  uint32_t last_run = 0;  // of runs whose largest logit is `cut`
  if (a.top)
#pragma unroll
    for (uint32_t w = 0; w < W; ++w) {
      last_run = least[w] < cut ? place[w] : least[w] == cut ? max(last_run, place[w]) : last_run;
      cut = fminf(cut, least[w]);
    }
  // `take` gets this wave's runs that reach `cut`, each lane 4 tokens from `at` of every one
  auto walk = [&](auto take) {
    for (uint32_t r0 = 0;;) {
#pragma unroll 1
      for (uint32_t u = 0; u < U; ++u) {
        const float peak = u == 0 ? p[0] : u == 1 ? p[1] : u == 2 ? p[2] : p[3];
        const uint32_t run = r0 + W * (64u * u + lane) + wave;
        for (uint64_t who = __ballot(run < runs && (peak > cut || (peak == cut && run <= last_run))); who;) {
          f4_t v[B];
          uint32_t at[B] = {}, n = 0;
#pragma unroll
          for (uint32_t b = 0; b < B; ++b) {
            v[b] = f4_t{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
            if (!who) continue;
            at[b] = 256u * (r0 + W * (64u * u + (uint32_t)__builtin_ctzll(who)) + wave) + 4u * lane;
            who &= who - 1u;
            n = b + 1u;
            if (at[b] + 4u <= a.vocab) v[b] = *as_global(reinterpret_cast<const f4_any*>(x + at[b]));
            else
#pragma unroll
              for (uint32_t i = 0; i < 4; ++i)
                if (at[b] + i < a.vocab) v[b][i] = *as_global(x + at[b] + i);
          }
          take(v, at, n);
        }
      }
      r0 += 64u * W * U;
      if (r0 >= runs) break;
      load(r0);
    }
  };
  if (a.top)
    walk([&](f4_t(&v)[B], uint32_t(&at)[B], uint32_t n) {
#pragma unroll
      for (uint32_t b = 0; b < B; ++b) {
        if (b >= n) break;
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i)
          if (v[b][i] >= cut && at[b] + i < a.vocab) {
            const uint32_t to = atomicAdd(&fits, 1u);
            if (to < kFit) {
              sm.fit.v[to] = v[b][i];
              sm.fit.id[to] = at[b] + i;
            }
          }
      }
    });
  Stats s;
  s.m = q[0];
  s.z = q[1];
  s.t = q[2];
  uint32_t count = (uint32_t)q[3];  // (below 2^24: exact)
  for (uint32_t i = threadIdx.x + 64u * W; i < a.slices; i += 64u * W) {
    const f4_t r = stats[i];
    Stats o;
    o.m = r[0];
    o.z = r[1];
    o.t = r[2];
    s.merge(o);
    count += (uint32_t)r[3];
  }
  merge_lanes(s);
  count = (uint32_t)wave_sum((float)count);
  if (lane == 0) {
    m[wave] = s.m;
    z[wave] = s.z;
    t[wave] = s.t;
    counts[wave] = count;
  }
  __syncthreads();
  s = Stats{};
  if (lane < W) {
    s.m = m[lane];
    s.z = z[lane];
    s.t = t[lane];
  }
  merge_lanes(s);
  count = (uint32_t)wave_sum(lane < W ? (float)counts[lane] : 0.f);
  const float log_z = logf(s.z);
  if (wave == 0) answer(a, row, s, count, log_z, xt, lane);
  const uint32_t n = fits;
  if (n <= kFit) {
    for (uint32_t i0 = 0; i0 < n; i0 += 8u * W) {  // 8 lanes for each
      const uint32_t i = i0 + threadIdx.x / 8u, at = min(i, n - 1u);
      const Entry e = {sm.fit.v[at], sm.fit.id[at]};
      uint32_t place = 0;
#pragma unroll 4
      for (uint32_t o = lane & 7u; o < n; o += 8u) place += better(Entry{sm.fit.v[o], sm.fit.id[o]}, e) ? 1u : 0u;
      place += xor_lane<1>(place);
      place += xor_lane<2>(place);
      place += xor_lane<4>(place);
      if (i < n && place < a.top && (lane & 7u) == 0) answer_top(a, row, place, e, s, log_z);
    }
    for (uint32_t i = n + threadIdx.x; i < a.top; i += 64u * W) answer_top(a, row, i, Entry{}, s, log_z);  // (no such token)
    return;
  }
  Entry list, last;
  load(0);
  walk([&](f4_t(&v)[B], uint32_t(&at)[B], uint32_t n) {
#pragma unroll 1
    for (uint32_t b = 0; b < n; ++b) {  // (the first; the others move up)
#pragma unroll 1
      for (uint32_t i = 0; i < 4; ++i) {
        const float e = i == 0 ? v[0][0] : i == 1 ? v[0][1] : i == 2 ? v[0][2] : v[0][3];
        put(list, last, Entry{e, at[0] + i < a.vocab ? at[0] + i : kNone}, cut, a.top, lane);
      }
#pragma unroll
      for (uint32_t c = 0; c + 1u < B; ++c) {
        v[c] = v[c + 1u];
        at[c] = at[c + 1u];
      }
      cut = fmaxf(cut, last.v);
    }
  });
  __syncthreads();  // (the waves have read `fits`; what it counted is written over)
  Stats none;
  if (!join_waves<W>(sm.joint, none, count, list, a.top, wave, lane)) return;
  if (lane < a.top) answer_top(a, row, lane, list, s, log_z);
}

// The slices of a row: one where the rows alone fill the chip.
void pick_slices(uint32_t M, uint32_t vocab, uint32_t* slices, uint32_t* slice) {
  const uint32_t want = std::max(1u, 1024u / M), most = (vocab + 1023u) / 1024u;
  const uint32_t n = std::min(want, most);
  *slice = n == 1 ? vocab : ((vocab + n - 1u) / n + 1023u) / 1024u * 1024u;
  *slices = (vocab + *slice - 1u) / *slice;
}

}  // namespace
}  // namespace mi

using namespace mi;

extern "C" {

size_t mi_logprobs_ws(uint32_t M, uint32_t vocab_used, uint32_t top) {
  if (M == 0 || M > kMaxRows || vocab_used == 0 || vocab_used > kMaxVocab) return 0;
  uint32_t slices, slice;
  pick_slices(M, vocab_used, &slices, &slice);
  return slices == 1 ? 0 : (size_t)M * (16u * (size_t)slices + (top ? (vocab_used + 255u) / 256u * 4u : 0u));
}

int mi_logprobs(const float* logits, size_t row_stride, const uint32_t* tokens, uint32_t M, uint32_t vocab_used,
                uint32_t top, float* logprob, uint32_t* rank, float* entropy, uint32_t* top_ids, float* top_logprobs,
                void* ws, size_t ws_bytes, void* stream) {
  if (!logits || (reinterpret_cast<uintptr_t>(logits) & 3u)) return mi_fail(MI_ERR_ARG, "logprobs: null or misaligned logits");
  if (M == 0 || M > kMaxRows || vocab_used == 0 || vocab_used > kMaxVocab)
    return mi_fail(MI_ERR_SHAPE, "logprobs: M 1..65535, vocab_used 1..2^23");
  if (row_stride < vocab_used) return mi_fail(MI_ERR_ARG, "logprobs: row_stride below vocab_used");
  if (top > kMaxTop) return mi_fail(MI_ERR_SHAPE, "logprobs: at most 64 top tokens");
  if ((logprob || rank) && !tokens) return mi_fail(MI_ERR_ARG, "logprobs: logprob and rank need tokens");
  if (top ? !top_ids || !top_logprobs : top_ids || top_logprobs)
    return mi_fail(MI_ERR_ARG, "logprobs: top_ids and top_logprobs go with top > 0");
  for (const void* p : {(const void*)tokens, (const void*)logprob, (const void*)rank, (const void*)entropy, (const void*)top_ids,
                        (const void*)top_logprobs})
    if (reinterpret_cast<uintptr_t>(p) & 3u) return mi_fail(MI_ERR_ARG, "logprobs: misaligned tokens or outputs (4 bytes)");
  if (!logprob && !rank && !entropy && !top) return mi_fail(MI_ERR_ARG, "logprobs: nothing is asked");
  const size_t need = mi_logprobs_ws(M, vocab_used, top);
  if (need && (!ws || (reinterpret_cast<uintptr_t>(ws) & 15u) || ws_bytes < need))
    return mi_fail(MI_ERR_ARG, "logprobs: the workspace is null, misaligned (16 bytes) or below mi_logprobs_ws");
  LogprobArgs a{logits, row_stride, tokens, vocab_used, top, 1, vocab_used, logprob, entropy, top_logprobs, rank, top_ids,
                nullptr, nullptr};
  pick_slices(M, vocab_used, &a.slices, &a.slice);
  if (need) {
    a.stats = static_cast<f4_t*>(ws);
    a.peaks = reinterpret_cast<float*>(a.stats + (size_t)M * a.slices);
  }
  hipStream_t st = (hipStream_t)stream;
  if (a.slices == 1) {
    logprobs_kernel<true><<<dim3(1, M), 256, 0, st>>>(a);
  } else {
    logprobs_kernel<false><<<dim3(a.slices, M), 256, 0, st>>>(a);
    logprobs_join_kernel<<<M, 512, 0, st>>>(a);
  }
  return mi_hip((int)hipGetLastError(), "logprobs");
}

}  // extern "C"
