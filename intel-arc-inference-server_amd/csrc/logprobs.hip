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
  // of beams: the rows' (m, Z) (top_logprobs are then the logits themselves); NULL, or rows (not 0) of which nothing is asked
  f2_t* sums;
  const uint32_t* skip;
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
template <bool BEAMS>
__device__ __forceinline__ void answer(const LogprobArgs& a, uint32_t row, const Stats& s, uint32_t count, float log_z, float xt,
                                       uint32_t lane) {
  if (lane != 0) return;
  if (a.entropy) a.entropy[row] = log_z - s.t / s.z * kLn2;
  if (a.logprob) a.logprob[row] = (xt - s.m) - log_z;
  if (a.rank) a.rank[row] = xt != xt ? kNone : count;
  if constexpr (BEAMS) a.sums[row] = f2_t{s.m, s.z};
}
template <bool BEAMS>
__device__ __forceinline__ void answer_top(const LogprobArgs& a, uint32_t row, uint32_t place, Entry e, const Stats& s, float log_z) {
  a.top_ids[(size_t)row * a.top + place] = e.id;
  a.top_logprobs[(size_t)row * a.top + place] = e.id == kNone ? -INFINITY : BEAMS ? e.v : (e.v - s.m) - log_z;
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
// the waves keep its best tokens; otherwise they leave the largest logit of each 256. BEAMS: by loads that the caches need not keep
// (128 texts of 4 67.5 us in all, 77.5 with the others), and with `sums` and `skip` (asked for when the kernel runs they took one row of
// 151936 tokens of mi_logprobs from 11.6 to 11.9 us, 333 rows from 53.8 to 54.6).
template <bool LISTS, bool BEAMS>
__global__ __launch_bounds__(256, 5) void logprobs_kernel(LogprobArgs a) {
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, row = blockIdx.y;
  if constexpr (BEAMS)
    if (a.skip && a.skip[row]) return;
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
      if (i + 4u <= end) {
        const auto* from = as_global(reinterpret_cast<const f4_any*>(x + i));
        if constexpr (BEAMS) to[u] = __builtin_nontemporal_load(from);
        else to[u] = *from;
      } else if (i < end)
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
    answer<BEAMS>(a, row, s, count, log_z, xt, lane);
    if (lane < a.top) answer_top<BEAMS>(a, row, lane, list, s, log_z);
  } else if (lane == 0) a.stats[(size_t)row * a.slices + blockIdx.x] = f4_t{s.m, s.z, s.t, (float)count};
}

// A work-group per row of several slices: joins their statistics, and finds the best tokens among the runs of 256 whose
// largest logit reaches a bound that k runs' reach, which it reads again: about 50 runs and 60 tokens at 151936 tokens and
// k = 20. The bound: of runs by their largest logit, equal ones by their place, the worst of the waves' ceil(k / W)-th best
// (k runs have a token at least as good as any token of a run behind it). A token's place among the best is the number of
// those read that are better. Where more tokens reach the bound than fit (equal logits, or fewer finite ones than k), the
// waves keep lists. One row of 151936 with the 20 best takes 11.6 us, 16 rows 15.2, 333 with the 5 best 53 (lists from
// every slice, as a row in one has them: 18.6, 23 and 54.2); one row of equal logits 21.6 (20.9).
template <bool BEAMS>
__global__ __launch_bounds__(512) void logprobs_join_kernel(LogprobArgs a) {
  constexpr uint32_t W = 8, U = 4, B = 8, kFit = 1024;  // waves; a lane's runs looked at together; runs read together; tokens
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, row = blockIdx.x, runs = (a.vocab + 255u) / 256u;
  if constexpr (BEAMS)
    if (a.skip && a.skip[row]) return;
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
  if (wave == 0) answer<BEAMS>(a, row, s, count, log_z, xt, lane);
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
      if (i < n && place < a.top && (lane & 7u) == 0) answer_top<BEAMS>(a, row, place, e, s, log_z);
    }
    for (uint32_t i = n + threadIdx.x; i < a.top; i += 64u * W) answer_top<BEAMS>(a, row, i, Entry{}, s, log_z);  // (no such token)
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
  if (lane < a.top) answer_top<BEAMS>(a, row, lane, list, s, log_z);
}

// ---- the best continuations of beams ----
// A candidate: a token of a beam with the score cum + (x - m) - log Z, in 64 bits, so that candidates of different beams are
// told apart as far as Z (in 32 bits) tells them. A beam's candidates stand in the order of their logits; equal scores go to the
// lower beam, then to the lower place.
struct Candidate {
  double score = -INFINITY;
  uint32_t at = kNone;  // 64 beam + place; kNone: none
};
__device__ __forceinline__ bool better(const Candidate& a, const Candidate& b) {
  return a.score > b.score || (a.score == b.score && a.at < b.at);
}
template <uint32_t X>
__device__ __forceinline__ void half_clean(Candidate& e, uint32_t lane) {  // strides X .. 1, best first
  const uint64_t s = __builtin_bit_cast(uint64_t, e.score);
  const Candidate o = {__builtin_bit_cast(double, (uint64_t)xor_lane<X>((uint32_t)(s >> 32)) << 32 | xor_lane<X>((uint32_t)s)),
                       xor_lane<X>(e.at)};
  if (better(o, e) == ((lane & X) == 0)) e = o;
  if constexpr (X > 1) half_clean<X / 2>(e, lane);
}

struct BeamArgs {
  const float* cum;
  const uint32_t* done;
  const f2_t* sums;         // [rows]
  const uint32_t* top_ids;  // [rows][k]
  const float* top;         // [rows][k], logits
  uint32_t eos, beams, k;
  uint32_t *ids, *from;
  float* scores;
};
// what a beam's logits are added to, of its maximum and sum
__device__ __forceinline__ double beam_base(float cum, float m, float z) { return (double)cum - (double)m - log((double)z); }
__device__ __forceinline__ void take_best(Candidate& list, const Candidate& c, uint32_t lane) {  // (c: the best last)
  if (better(c, list)) list = c;
  half_clean<32>(list, lane);
}
// W waves' lists into the first's: whether this wave holds the joint one
template <uint32_t W>
struct JointCandidates {
  double score[W][64];
  uint32_t at[W][64];
};
template <uint32_t W>
__device__ __forceinline__ bool join_candidates(JointCandidates<W>& j, Candidate& list, uint32_t wave, uint32_t lane) {
#pragma unroll 1
  for (uint32_t step = W / 2; step; step /= 2) {
    j.score[wave][lane] = list.score;
    j.at[wave][lane] = list.at;
    __syncthreads();
    if (wave >= step) return false;
    take_best(list, Candidate{j.score[wave + step][63u - lane], j.at[wave + step][63u - lane]}, lane);
  }
  return true;
}
__device__ __forceinline__ void answer_beam(const BeamArgs& a, uint32_t batch, uint32_t place, bool none, uint32_t id, uint32_t w,
                                            double score) {
  const size_t to = (size_t)batch * a.k + place;
  a.ids[to] = none ? kNone : id;
  a.from[to] = none ? kNone : w;
  a.scores[to] = none ? -INFINITY : (float)score;
}
// Behind lists of every row's best. grid (batch), four waves: a wave merges every fourth beam's candidates, 64 at a time over its
// lanes, then the waves' join. Bound by its chain: two rounds of loads, a logarithm, six exchanges a beam.
__global__ __launch_bounds__(256) void beam_select_kernel(BeamArgs a) {
  __shared__ JointCandidates<4> joint;
  constexpr uint32_t U = 4;  // beams whose candidates are loaded at once
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, batch = blockIdx.x, n = 63u - lane;  // (the best come last)
  const uint32_t mine = batch * a.beams + min(lane, a.beams - 1u);
  uint32_t id[U];
  float top[U];
  auto load = [&](uint32_t w0) {
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) {
      const size_t at = (size_t)(batch * a.beams + min(w0 + 4u * u, a.beams - 1u)) * a.k + min(n, a.k - 1u);
      id[u] = *as_global(a.top_ids + at);
      top[u] = *as_global(a.top + at);
    }
  };
  load(wave);
  // a lane a beam
  const float cum = *as_global(a.cum + mine);
  const f2_t s = *as_global(a.sums + mine);
  const uint64_t done = __ballot(a.done && a.done[mine]);
  const uint64_t of = __builtin_bit_cast(uint64_t, (done >> lane) & 1u ? (double)cum : beam_base(cum, s.x, s.y));
  Candidate list;
  for (uint32_t w0 = wave; w0 < a.beams; w0 += 4u * U) {
    if (w0 != wave) load(w0);
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) {
      const uint32_t w = w0 + 4u * u;
      if (w >= a.beams) break;
      const double base = __builtin_bit_cast(double, (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(of >> 32), (int)w) << 32 |
                                                         (uint32_t)__builtin_amdgcn_readlane((int)of, (int)w));
      const bool ends = (done >> w) & 1u;
      const double sum = ends ? base : base + (double)top[u];
      Candidate c;
      if ((ends ? n == 0u : n < a.k && id[u] != kNone) && sum > -INFINITY) c = Candidate{sum, 64u * w + n};  // (nor a NaN)
      take_best(list, c, lane);
    }
  }
  if (!join_candidates<4>(joint, list, wave, lane) || lane >= a.k) return;
  const uint32_t w = list.at / 64u, row = batch * a.beams + w;
  const bool none = list.at == kNone;
  answer_beam(a, batch, lane, none, none ? kNone : a.done && a.done[row] ? a.eos : a.top_ids[(size_t)row * a.k + list.at % 64u], w,
              list.score);
}

// Behind slices, in place of logprobs_join_kernel and beam_select_kernel: grid (batch), sixteen waves. They join each beam's
// statistics; form a bound that k runs of 256 tokens reach by the score of their largest logit (as logprobs_join_kernel's); read again
// the runs that reach it, of all beams about k; and a token's place is the number of those read that are better. Where more tokens reach
// the bound than fit, the waves keep a list of every beam. One text of 4 beams with k = 8 takes 13.4 us in all, 16 of 8 with k = 16
// 28.7 (16.0 and 32 with the rows' lists first); equal logits 45, rising ones 104. Bound by its chain of loads. A wave with fewer runs
// than its share of k leaves no bound (all vocabularies of 1025 to 3840 tokens; one beam of 8000 with k = 64): the lists then do it all
// again, one text of 16 beams of 3800 tokens 59 us with k = 20 and 84 with 64, where 8000 tokens take 13 and 22.
constexpr uint32_t kFit = 1024, kMaxBeams = 64;
constexpr uint32_t kJoinWaves = 16, kJoinRuns = 8;  // a lane's runs
uint32_t runs_of_wave(uint32_t vocab) { return ((vocab + 255u) / 256u + kJoinWaves - 1u) / kJoinWaves; }
__global__ __launch_bounds__(64 * kJoinWaves) void beam_join_kernel(LogprobArgs a, BeamArgs o) {
  constexpr uint32_t W = kJoinWaves, U = kJoinRuns, B = 4;  // B: runs read together
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, batch = blockIdx.x, runs = (a.vocab + 255u) / 256u;
  const uint32_t row0 = batch * o.beams;
  __shared__ double base[kMaxBeams];  // what a beam's logits are added to; NaN: it has no candidates among them
  __shared__ float m[kMaxBeams], z[kMaxBeams], least[W];
  __shared__ uint32_t fits, hit_runs[W][64 * U];  // beam, run (below 2^15)
  __shared__ union {
    struct {
      double score[kFit];
      float v[kFit];
      uint32_t id[kFit], w[kFit];
    } fit;
    struct {
      JointCandidates<W> joint;
      uint32_t id[kMaxBeams][64];
    } lists;
  } sm;
  // (every load that the bound waits for goes out at once; a wave has every W-th run of every beam)
  float p[U];
  uint32_t run[U], beam_of[U];
  const uint32_t each = (runs + W - 1u) / W;
#pragma unroll
  for (uint32_t u = 0; u < U; ++u) {
    const uint32_t i = lane + 64u * u;
    beam_of[u] = i / each;
    run[u] = (i - beam_of[u] * each) * W + wave;
    p[u] = beam_of[u] < o.beams && run[u] < runs ? a.peaks[(size_t)(row0 + beam_of[u]) * runs + run[u]] : -INFINITY;
  }
  const uint32_t mine = min(lane, o.beams - 1u);
  const float cum = *as_global(o.cum + row0 + mine);
  const bool ends = o.done && o.done[row0 + mine];
  if (threadIdx.x == 0) fits = 0;
  for (uint32_t w = wave; w < o.beams; w += W) {
    const f4_t* stats = a.stats + (size_t)(row0 + w) * a.slices;
    Stats s;
    for (uint32_t i0 = 0; i0 < a.slices; i0 += 256u) {
      f4_t r[4];
#pragma unroll
      for (uint32_t j = 0; j < 4; ++j) {
        const uint32_t i = i0 + 64u * j + lane;
        r[j] = i < a.slices ? stats[i] : f4_t{-INFINITY, 0.f, 0.f, 0.f};
      }
#pragma unroll
      for (uint32_t j = 0; j < 4; ++j) {
        Stats of;
        of.m = r[j][0];
        of.z = r[j][1];
        s.merge(of);
      }
    }
    merge_lanes(s);
    if (lane == 0) {
      m[w] = s.m;
      z[w] = s.z;
    }
  }
  __syncthreads();
  if (wave == 0 && lane < o.beams) base[lane] = ends ? __builtin_bit_cast(double, 0x7FF8000000000000ull) : beam_base(cum, m[lane], z[lane]);
  __syncthreads();
  // `see` gets the score of each run's largest logit, -inf where there is none
  auto walk = [&](auto see) {
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) {
      if (64u * u >= o.beams * each) break;
      const double of = beam_of[u] < o.beams ? base[beam_of[u]] + (double)p[u] : -INFINITY;
      see(of > -INFINITY ? of : -INFINITY, beam_of[u], run[u]);  // (nor a NaN)
    }
  };
  float top = -INFINITY;
  walk([&](double of, uint32_t, uint32_t) { top = fmaxf(top, __double2float_rd(of)); });
  const uint32_t share = (o.k + W - 1u) / W;
  const float low = kth_largest(top, share, lane);
  if (lane == 0) least[wave] = low;
  __syncthreads();
  float cut = INFINITY;
#pragma unroll
  for (uint32_t w = 0; w < W; ++w) cut = fminf(cut, least[w]);
  auto put_in = [&](double score, float v, uint32_t id, uint32_t w) {
    const uint32_t to = atomicAdd(&fits, 1u);
    if (to < kFit) {
      sm.fit.score[to] = score;
      sm.fit.v[to] = v;
      sm.fit.id[to] = id;
      sm.fit.w[to] = w;
    }
  };
  // the wave's runs that reach it, then their tokens
  uint32_t hits = 0;
  walk([&](double of, uint32_t w, uint32_t r) {
    const bool hit = of > -INFINITY && of >= (double)cut;
    const uint64_t who = __ballot(hit);
    if (hit) hit_runs[wave][hits + (uint32_t)__popcll(who & ((1ull << lane) - 1u))] = w << 16 | r;
    hits += (uint32_t)__popcll(who);
  });
  wave_lds_sync();
#pragma unroll 1
  for (uint32_t h = 0; h < hits; h += B) {
    f4_t v[B];
    uint32_t at[B], beam[B];
    const uint32_t n = min(B, hits - h);
#pragma unroll
    for (uint32_t b = 0; b < B; ++b) {
      const uint32_t r = hit_runs[wave][min(h + b, hits - 1u)];
      beam[b] = r >> 16;
      at[b] = 256u * (r & 0xFFFFu) + 4u * lane;
      const float* x = a.logits + (size_t)(row0 + beam[b]) * a.row_stride;
      v[b] = f4_t{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
      if (at[b] + 4u <= a.vocab) v[b] = *as_global(reinterpret_cast<const f4_any*>(x + at[b]));
      else
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i)
          if (at[b] + i < a.vocab) v[b][i] = *as_global(x + at[b] + i);
    }
#pragma unroll
    for (uint32_t b = 0; b < B; ++b) {
      if (b >= n) break;
      const double of_beam = base[beam[b]];
#pragma unroll
      for (uint32_t i = 0; i < 4; ++i) {
        const double s = of_beam + (double)v[b][i];
        if (s > -INFINITY && s >= (double)cut) put_in(s, v[b][i], at[b] + i, beam[b]);
      }
    }
  }
  if (wave == 0 && lane < o.beams && ends && cum > -INFINITY) put_in((double)cum, 0.f, o.eos, lane);
  __syncthreads();
  const uint32_t n = fits;
  if (n <= kFit) {
    for (uint32_t i0 = 0; i0 < n; i0 += 8u * W) {  // 8 lanes for each
      const uint32_t i = i0 + threadIdx.x / 8u, at = min(i, n - 1u);
      const double score = sm.fit.score[at];
      const Entry e = {sm.fit.v[at], sm.fit.id[at]};
      const uint32_t w = sm.fit.w[at];
      uint32_t place = 0;
#pragma unroll 2
      for (uint32_t j = lane & 7u; j < n; j += 8u) {
        const double other = sm.fit.score[j];
        const uint32_t ow = sm.fit.w[j];
        place += other > score || (other == score && (ow < w || (ow == w && better(Entry{sm.fit.v[j], sm.fit.id[j]}, e)))) ? 1u : 0u;
      }
      place += xor_lane<1>(place);
      place += xor_lane<2>(place);
      place += xor_lane<4>(place);
      if (i < n && place < o.k && (lane & 7u) == 0) answer_beam(o, batch, place, false, e.id, w, score);
    }
    for (uint32_t i = n + threadIdx.x; i < o.k; i += 64u * W) answer_beam(o, batch, i, true, 0u, 0u, 0.0);
    return;
  }
  __syncthreads();  // (the waves have read `fits`; what it counted is written over)
  Candidate list;
  for (uint32_t w = wave; w < o.beams; w += W) {
    const double of = base[w];
    Entry best, last;
    const float* x = a.logits + (size_t)(row0 + w) * a.row_stride;
    const float* peaks = a.peaks + (size_t)(row0 + w) * runs;
    const bool over = o.done && o.done[row0 + w];
    for (uint32_t r0 = 0; !over && of == of && r0 < runs; r0 += 64u) {
      const float peak = r0 + lane < runs ? peaks[r0 + lane] : -INFINITY;
      // (in the runs' order: an equal logit behind a full list's last is not better)
      for (uint64_t who = __ballot(peak > last.v && of + (double)peak >= (double)cut); who; who &= who - 1u) {
        const int r = __builtin_ctzll(who);
        if (!(lane_f(peak, r) > last.v)) continue;
        const uint32_t i = 256u * (r0 + (uint32_t)r) + lane;
#pragma unroll
        for (uint32_t q = 0; q < 4; ++q)  // (64 ids at a time, ascending)
          put(best, last, i + 64u * q < a.vocab ? Entry{x[i + 64u * q], i + 64u * q} : Entry{}, -INFINITY, o.k, lane);
      }
    }
    sm.lists.id[w][lane] = best.id;
    const float v = __shfl(best.v, (int)(63u - lane), 64);
    const uint32_t id = (uint32_t)__shfl((int)best.id, (int)(63u - lane), 64), place = 63u - lane;
    const double score = over ? (double)o.cum[row0 + w] : of + (double)v;
    Candidate c;
    if ((over ? place == 0u : place < o.k && id != kNone) && score > -INFINITY) c = Candidate{score, 64u * w + place};
    take_best(list, c, lane);
  }
  if (!join_candidates<W>(sm.lists.joint, list, wave, lane) || lane >= o.k) return;
  const uint32_t w = list.at / 64u;
  const bool none = list.at == kNone;
  answer_beam(o, batch, lane, none, none ? kNone : o.done && o.done[row0 + w] ? o.eos : sm.lists.id[w][list.at % 64u], w, list.score);
}

// The slices of a row: one where the rows alone fill the chip.
void pick_slices(uint32_t M, uint32_t vocab, uint32_t* slices, uint32_t* slice) {
  const uint32_t want = std::max(1u, 1024u / M), most = (vocab + 1023u) / 1024u;
  const uint32_t n = std::min(want, most);
  *slice = n == 1 ? vocab : ((vocab + n - 1u) / n + 1023u) / 1024u * 1024u;
  *slices = (vocab + *slice - 1u) / *slice;
}

// (beams: the rows' slices are joined by texts, and nothing is left to do)
bool launch(LogprobArgs a, uint32_t M, void* ws, hipStream_t st, const BeamArgs* beams = nullptr) {
  pick_slices(M, a.vocab, &a.slices, &a.slice);
  if (a.slices == 1) {
    if (beams) logprobs_kernel<true, true><<<dim3(1, M), 256, 0, st>>>(a);
    else logprobs_kernel<true, false><<<dim3(1, M), 256, 0, st>>>(a);
    return false;
  }
  a.stats = static_cast<f4_t*>(ws);
  a.peaks = reinterpret_cast<float*>(a.stats + (size_t)M * a.slices);
  if (beams) logprobs_kernel<false, true><<<dim3(a.slices, M), 256, 0, st>>>(a);
  else logprobs_kernel<false, false><<<dim3(a.slices, M), 256, 0, st>>>(a);
  const bool whole = beams && beams->beams * runs_of_wave(a.vocab) <= 64u * kJoinRuns;
  if (whole) beam_join_kernel<<<M / beams->beams, 64 * kJoinWaves, 0, st>>>(a, *beams);
  else if (beams) logprobs_join_kernel<true><<<M, 512, 0, st>>>(a);
  else logprobs_join_kernel<false><<<M, 512, 0, st>>>(a);
  return whole;
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
  const LogprobArgs a{logits, row_stride, tokens, vocab_used, top, 1, vocab_used, logprob, entropy, top_logprobs, rank, top_ids,
                      nullptr, nullptr, nullptr, nullptr};
  launch(a, M, ws, (hipStream_t)stream);
  return mi_hip((int)hipGetLastError(), "logprobs");
}

size_t mi_beam_select_ws(uint32_t batch, uint32_t beams, uint32_t vocab_used, uint32_t k) {
  if (batch == 0 || beams == 0 || beams > kMaxBeams || (uint64_t)batch * beams > kMaxRows || vocab_used == 0 ||
      vocab_used > kMaxVocab || k == 0 || k > kMaxTop)
    return 0;
  const uint32_t rows = batch * beams;
  return (size_t)rows * (8u + 8u * k) + 16u + mi_logprobs_ws(rows, vocab_used, k);
}

int mi_beam_select(const float* logits, size_t row_stride, const float* cum, const uint32_t* done, uint32_t eos, uint32_t batch,
                   uint32_t beams, uint32_t vocab_used, uint32_t k, uint32_t* ids, uint32_t* from, float* scores, void* ws,
                   size_t ws_bytes, void* stream) {
  for (const void* p : {(const void*)logits, (const void*)cum, (const void*)ids, (const void*)from, (const void*)scores})
    if (!p || (reinterpret_cast<uintptr_t>(p) & 3u)) return mi_fail(MI_ERR_ARG, "beam_select: null or misaligned pointer (4 bytes)");
  if (reinterpret_cast<uintptr_t>(done) & 3u) return mi_fail(MI_ERR_ARG, "beam_select: misaligned done (4 bytes)");
  if (batch == 0 || beams == 0 || beams > kMaxBeams || (uint64_t)batch * beams > kMaxRows)
    return mi_fail(MI_ERR_SHAPE, "beam_select: 1..64 beams, batch * beams 1..65535");
  if (vocab_used == 0 || vocab_used > kMaxVocab || k == 0 || k > kMaxTop)
    return mi_fail(MI_ERR_SHAPE, "beam_select: vocab_used 1..2^23, k 1..64");
  if (row_stride < vocab_used) return mi_fail(MI_ERR_ARG, "beam_select: row_stride below vocab_used");
  if (!ws || (reinterpret_cast<uintptr_t>(ws) & 15u) || ws_bytes < mi_beam_select_ws(batch, beams, vocab_used, k))
    return mi_fail(MI_ERR_ARG, "beam_select: the workspace is null, misaligned (16 bytes) or below mi_beam_select_ws");
  const uint32_t rows = batch * beams;
  f2_t* sums = static_cast<f2_t*>(ws);
  float* top = reinterpret_cast<float*>(sums + rows);
  uint32_t* top_ids = reinterpret_cast<uint32_t*>(top + (size_t)rows * k);
  const uintptr_t end = (reinterpret_cast<uintptr_t>(top_ids + (size_t)rows * k) + 15u) & ~(uintptr_t)15u;
  const LogprobArgs a{logits, row_stride, nullptr, vocab_used, k, 1, vocab_used, nullptr, nullptr, top, nullptr, top_ids,
                      nullptr, nullptr, sums, done};
  hipStream_t st = (hipStream_t)stream;
  const BeamArgs o{cum, done, sums, top_ids, top, eos, beams, k, ids, from, scores};
  if (!launch(a, rows, reinterpret_cast<void*>(end), st, &o)) beam_select_kernel<<<batch, 256, 0, st>>>(o);
  return mi_hip((int)hipGetLastError(), "beam_select");
}

}  // extern "C"
