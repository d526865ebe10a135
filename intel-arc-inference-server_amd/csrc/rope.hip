// rope.hip - rotary positions: the table of cosines and sines with frequencies scaled for long contexts (mi_rope_table), and rows
// of q||k||v, normed, rotated at their own positions and stored, q in 32 bits, k and v into cache rows (mi_rope_rows).
//
// Pair i of r / 2 turns by p f_i at position p, f_i = theta^(-2 i / r), scaled (mi_rope). A rotation takes (x, y) to
// (x cos - y sin, y cos + x sin), the pairs being (i, i + r / 2) or the neighbours (2 i, 2 i + 1).
#include <algorithm>
#include <cmath>

#include "mi_capi_internal.h"
#include "mi_pieces.h"

namespace mi {
namespace {

constexpr uint32_t kMaxRot = 256, kMaxRows = 65535, kNone = 0xFFFFFFFFu;

struct TableArgs {
  float* table;
  uint32_t pos0, n, half;
  double much;
  double f[kMaxRot / 2], cos_f[kMaxRot / 2], sin_f[kMaxRot / 2];  // a pair's angle from a position to the next
};
// A thread takes four pairs of kStep positions. The first position's angle is formed in 64 bits, off by 2^-52 of itself (f_i, which
// the host forms in more bits, and the product p f_i are rounded once each), and brought to |r| <= pi / 4 by pi / 2 in two parts, off
// by 2^-53 of r; the series of sine and cosine there go to r^15 and r^14 (off by 2^-49). Every position behind it turns by f_i, four
// products of 64 bits in place of some thirty operations, off by 2^-52 more each. Bound by the stores: 131072 positions of 64 pairs
// (67 MB) 12.3 us (16.0 with each angle's own series, bound by the 64-bit operations; steps of 2 / 4 / 8 positions 12.6 / 12.3 / 14.2;
// a plain fill 11.2).
constexpr uint32_t kStep = 4;
__global__ __launch_bounds__(256) void rope_table_kernel(TableArgs a) {
  const uint32_t per = a.half / 4u, i = blockIdx.x * 256u + threadIdx.x;
  const uint32_t step = i / per, at = 4u * (i - step * per), row = step * kStep;
  if (row >= a.n) return;
  const double p = (double)((uint64_t)a.pos0 + row);
  double c[4], s[4], cf[4], sf[4];
#pragma unroll
  for (uint32_t e = 0; e < 4; ++e) {
    cf[e] = a.cos_f[at + e];
    sf[e] = a.sin_f[at + e];
    const double x = p * a.f[at + e], k = __builtin_rint(x * 0.6366197723675814);  // 2 / pi
    const double r = __builtin_fma(-k, 6.123233995736766e-17, __builtin_fma(-k, 1.5707963267948966, x)), z = r * r;
    double sn = -1.0 / 1307674368000.0, cs = -1.0 / 87178291200.0;  // 1 / 15!, 1 / 14!
    sn = __builtin_fma(sn, z, 1.0 / 6227020800.0);
    cs = __builtin_fma(cs, z, 1.0 / 479001600.0);
    sn = __builtin_fma(sn, z, -1.0 / 39916800.0);
    cs = __builtin_fma(cs, z, -1.0 / 3628800.0);
    sn = __builtin_fma(sn, z, 1.0 / 362880.0);
    cs = __builtin_fma(cs, z, 1.0 / 40320.0);
    sn = __builtin_fma(sn, z, -1.0 / 5040.0);
    cs = __builtin_fma(cs, z, -1.0 / 720.0);
    sn = __builtin_fma(sn, z, 1.0 / 120.0);
    cs = __builtin_fma(cs, z, 1.0 / 24.0);
    sn = __builtin_fma(sn, z, -1.0 / 6.0);
    cs = __builtin_fma(cs, z, -0.5);
    sn = __builtin_fma(sn * z, r, r);
    cs = __builtin_fma(cs, z, 1.0);
    const uint32_t q = (uint32_t)(int64_t)k & 3u;
    c[e] = (q & 1u) ? sn : cs;
    s[e] = (q & 1u) ? cs : sn;
    if (q == 1u || q == 2u) c[e] = -c[e];
    if (q & 2u) s[e] = -s[e];
  }
  float* to = a.table + (size_t)row * 2u * a.half + at;
#pragma unroll
  for (uint32_t k = 0; k < kStep; ++k, to += 2u * a.half) {
    if (row + k >= a.n) return;
    *as_global(reinterpret_cast<f4_any*>(to)) =
        f4_t{(float)(c[0] * a.much), (float)(c[1] * a.much), (float)(c[2] * a.much), (float)(c[3] * a.much)};
    *as_global(reinterpret_cast<f4_any*>(to + a.half)) =
        f4_t{(float)(s[0] * a.much), (float)(s[1] * a.much), (float)(s[2] * a.much), (float)(s[3] * a.much)};
#pragma unroll
    for (uint32_t e = 0; e < 4; ++e) {
      const double x = c[e];
      c[e] = __builtin_fma(x, cf[e], -(s[e] * sf[e]));
      s[e] = __builtin_fma(s[e], cf[e], x * sf[e]);
    }
  }
}

typedef f2_t f2_any __attribute__((aligned(4)));
struct RowsArgs {
  const void* qkv;
  const uint32_t *pos, *slots;
  const float *q_norm, *k_norm, *rope;
  float* attn_q;
  uint16_t *k, *v;
  uint32_t* flag;
  size_t in_stride, row_stride, head_stride;
  uint32_t T, pos0, rows, rope_len, q_heads, kv_heads, rot, act;
  float eps;
};
template <bool F16>
__device__ __forceinline__ f4_t load4(const void* base, size_t at) {
  if constexpr (F16) {
    const u2_t h = __builtin_nontemporal_load(as_global(reinterpret_cast<const h4_any*>(static_cast<const uint16_t*>(base) + at)));
    return f4_t{h2f((uint16_t)h[0]), h2f((uint16_t)(h[0] >> 16)), h2f((uint16_t)h[1]), h2f((uint16_t)(h[1] >> 16))};
  } else {
    return __builtin_nontemporal_load(as_global(reinterpret_cast<const f4_any*>(static_cast<const float*>(base) + at)));
  }
}
// HD / 8 threads take a head of a row, two pieces of four elements each: with pairs of halves the two pieces that turn together (and
// two of those behind the rotated part that do not turn), with pairs of neighbours any two. The norm's sum goes over these threads.
// Nothing is rounded before the stores. Bound by the bytes: 2048 rows of 40 / 8 heads of 128 (110 MB) 23.3 us, 4.7 TB/s (a copy
// 4.9; with loads that the caches keep 24.3). Four heads a thread took 2 us more at 256 and 512 rows and little less at 2048.
template <int HD, bool F16, bool PAIRED>
__global__ __launch_bounds__(256) void rope_rows_kernel(RowsArgs a) {
  constexpr uint32_t L = HD / 8;
  const uint32_t heads = a.q_heads + 2u * a.kv_heads, unit = blockIdx.x * (256u / L) + threadIdx.x / L, l = threadIdx.x % L;
  const uint32_t t = unit / heads, head = unit - t * heads;
  if (t >= a.T) return;
  const uint32_t turning = a.rot / 8u;  // threads whose pieces turn
  const uint32_t c0 = PAIRED ? 4u * l : l < turning ? 4u * l : a.rot + 8u * (l - turning);
  const uint32_t c1 = PAIRED ? 4u * (l + L) : l < turning ? 4u * l + a.rot / 2u : c0 + 4u;
  const bool is_q = head < a.q_heads, is_v = head >= a.q_heads + a.kv_heads;
  const uint32_t pos = a.pos ? a.pos[t] : a.pos0 + t, slot = a.slots ? a.slots[t] : pos;
  const size_t src = (size_t)t * a.in_stride + (size_t)head * HD;
  f4_t x = load4<F16>(a.qkv, src + c0), y = load4<F16>(a.qkv, src + c1);
  if (pos >= a.rope_len || (!is_q && slot != kNone && slot >= a.rows)) {
    if (l == 0 && a.flag) *a.flag = pos >= a.rope_len ? 0xDEAD0002u : MI_STATUS_BAD_PAGE;
    return;
  }
  if (!is_q && slot == kNone) return;
  if (!is_v) {
    const float* w = is_q ? a.q_norm : a.k_norm;
    if (w) {
      const f4_t z = x * x + y * y;
      float sum = (z[0] + z[1]) + (z[2] + z[3]);
#pragma unroll
      for (uint32_t d = 1; d < L; d *= 2) sum += __shfl_xor(sum, (int)d, 64);
      const float rstd = 1.0f / sqrtf(sum / (float)HD + a.eps);
      x = x * rstd * *as_global(reinterpret_cast<const f4_any*>(w + c0));
      y = y * rstd * *as_global(reinterpret_cast<const f4_any*>(w + c1));
    }
    const float* cs = a.rope + (size_t)pos * a.rot;
    if constexpr (PAIRED) {
      auto turn = [&](f4_t& e, uint32_t c) {
        if (c >= a.rot) return;
        const f2_t co = *as_global(reinterpret_cast<const f2_any*>(cs + c / 2u)),
                   si = *as_global(reinterpret_cast<const f2_any*>(cs + a.rot / 2u + c / 2u));
        e = f4_t{__builtin_fmaf(e[0], co[0], -(e[1] * si[0])), __builtin_fmaf(e[1], co[0], e[0] * si[0]),
                 __builtin_fmaf(e[2], co[1], -(e[3] * si[1])), __builtin_fmaf(e[3], co[1], e[2] * si[1])};
      };
      turn(x, c0);
      turn(y, c1);
    } else if (l < turning) {
      const f4_t co = *as_global(reinterpret_cast<const f4_any*>(cs + c0)), si = *as_global(reinterpret_cast<const f4_any*>(cs + c1));
      const f4_t u = x;
#pragma unroll
      for (uint32_t e = 0; e < 4; ++e) {
        x[e] = __builtin_fmaf(u[e], co[e], -(y[e] * si[e]));
        y[e] = __builtin_fmaf(y[e], co[e], u[e] * si[e]);
      }
    }
  }
  if (is_q) {
    float* to = a.attn_q + ((size_t)t * a.q_heads + head) * HD;
    *as_global(reinterpret_cast<f4_any*>(to + c0)) = x;
    *as_global(reinterpret_cast<f4_any*>(to + c1)) = y;
  } else {
    const uint32_t h = head - a.q_heads - (is_v ? a.kv_heads : 0u);
    uint16_t* to = (is_v ? a.v : a.k) + (size_t)slot * a.row_stride + (size_t)h * a.head_stride;
    auto store = [&](uint32_t c, f4_t e) {
      const u2_t o = {(uint32_t)act_enc(e[0], a.act) | ((uint32_t)act_enc(e[1], a.act) << 16),
                      (uint32_t)act_enc(e[2], a.act) | ((uint32_t)act_enc(e[3], a.act) << 16)};
      *as_global(reinterpret_cast<h4_any*>(to + c)) = o;
    };
    store(c0, x);
    store(c1, y);
  }
}
template <int HD>
void launch_rows(const RowsArgs& a, bool f16, bool paired, hipStream_t st) {
  constexpr uint32_t units = 256u / (HD / 8u);
  const uint32_t grid = (a.T * (a.q_heads + 2u * a.kv_heads) + units - 1u) / units;
  if (f16 && paired) rope_rows_kernel<HD, true, true><<<grid, 256, 0, st>>>(a);
  else if (f16) rope_rows_kernel<HD, true, false><<<grid, 256, 0, st>>>(a);
  else if (paired) rope_rows_kernel<HD, false, true><<<grid, 256, 0, st>>>(a);
  else rope_rows_kernel<HD, false, false><<<grid, 256, 0, st>>>(a);
}
bool off(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1u)) != 0; }

}  // namespace
}  // namespace mi

using namespace mi;

extern "C" {

int mi_rope_table(const mi_rope* rope, uint32_t pos0, uint32_t n, float* table, void* stream) {
  if (!rope || !table || off(table, 4)) return mi_fail(MI_ERR_ARG, "rope_table: null or misaligned pointer (4 bytes)");
  const uint32_t r = rope->rot_dim;
  if (r == 0 || r > kMaxRot || r % 8) return mi_fail(MI_ERR_SHAPE, "rope_table: rot_dim a multiple of 8 up to 256");
  if (n == 0 || n > 1u << 24 || (uint64_t)pos0 + n > 1ull << 31)
    return mi_fail(MI_ERR_SHAPE, "rope_table: 1..2^24 positions below 2^31");
  if (!(rope->theta > 1.0f && rope->theta <= 1e30f)) return mi_fail(MI_ERR_ARG, "rope_table: theta above 1");
  if (rope->scaling > MI_ROPE_YARN) return mi_fail(MI_ERR_ARG, "rope_table: an MI_ROPE_* scaling");
  const bool scaled = rope->scaling != MI_ROPE_NONE;
  if (scaled && !(rope->factor > 0.0f && rope->factor <= 1e6f)) return mi_fail(MI_ERR_ARG, "rope_table: factor above 0 up to 1e6");
  if (!(rope->attention >= 0.0f && rope->attention <= 1e6f)) return mi_fail(MI_ERR_ARG, "rope_table: attention 0 (its default) or above");
  const bool ranged = rope->scaling == MI_ROPE_WAVELENGTH || rope->scaling == MI_ROPE_YARN;
  if (ranged && !(rope->original && rope->low > 0.0f && rope->high > rope->low && rope->high <= 1e9f))
    return mi_fail(MI_ERR_ARG, "rope_table: original from 1, 0 < low < high turns");
  TableArgs a{table, pos0, n, r / 2u, 1.0, {}, {}, {}};
  // (in 64 bits the exponent's rounding alone would take a frequency ln(theta) 2^-53 of itself off)
  using wide = long double;
  const wide by = rope->factor, pi = 3.14159265358979323846L;
  wide theta = rope->theta, lo = 0, hi = 0;
  if (rope->scaling == MI_ROPE_BASE) theta *= std::pow(by, (wide)r / (wide)(r - 2u));
  if (rope->scaling == MI_ROPE_YARN) {
    auto pair = [&](wide turns) { return r * std::log(rope->original / (turns * 2 * pi)) / (2 * std::log(theta)); };
    lo = std::max(std::floor(pair(rope->high)), (wide)0);
    hi = std::min(std::ceil(pair(rope->low)), (wide)(r - 1u));
    a.much = by > 1 ? (double)(0.1L * std::log(by) + 1) : 1.0;
  }
  if (rope->attention != 0.0f) a.much = rope->attention;
  // theta^(-2 i / r), from those whose i is a power of two (a power of each took the host 31 us a call, these 7, of 64 bits 6)
  wide plain[kMaxRot / 2] = {1};
  for (uint32_t i = 1; i < a.half; ++i) {
    const uint32_t low = i & (0u - i);
    plain[i] = i == low ? std::pow(theta, (wide)-2 * i / r) : plain[i - low] * plain[low];
  }
  for (uint32_t i = 0; i < a.half; ++i) {
    wide f = plain[i];
    if (rope->divisors) {
      if (!(rope->divisors[i] > 0.0f)) return mi_fail(MI_ERR_ARG, "rope_table: divisors above 0");
      f /= rope->divisors[i];
    }
    wide part = 1;  // of the frequency as it is; the rest of it divided by the factor
    if (rope->scaling == MI_ROPE_LINEAR) part = 0;
    if (rope->scaling == MI_ROPE_WAVELENGTH) part = (rope->original * f / (2 * pi) - rope->low) / ((wide)rope->high - rope->low);
    if (rope->scaling == MI_ROPE_YARN) part = 1 - (i - lo) / std::max(hi - lo, (wide)0.001);
    part = std::min(std::max(part, (wide)0), (wide)1);
    a.f[i] = (double)(part == 1 ? f : part * f + (1 - part) * f / by);
    // (so that a position's angle stays below 2^51, where its number of quarter turns is a whole number of 64 bits)
    if (!(a.f[i] <= 1048576.0)) return mi_fail(MI_ERR_ARG, "rope_table: a frequency above 2^20");
    a.cos_f[i] = std::cos(a.f[i]);
    a.sin_f[i] = std::sin(a.f[i]);
  }
  const uint32_t threads = (n + kStep - 1u) / kStep * (a.half / 4u);
  rope_table_kernel<<<(threads + 255u) / 256u, 256, 0, (hipStream_t)stream>>>(a);
  return mi_hip((int)hipGetLastError(), "rope_table");
}

int mi_rope_rows(const void* qkv, uint32_t in_kind, size_t in_stride, uint32_t T, const uint32_t* pos, uint32_t pos0,
                 const uint32_t* slots, uint32_t rows, const mi_attn_shape* shape, uint32_t paired, const float* q_norm,
                 const float* k_norm, const float* rope, uint32_t rope_len, float* attn_q, uint16_t* kv_k, uint16_t* kv_v,
                 size_t row_stride, size_t head_stride, uint32_t* flag, void* stream) {
  if (!qkv || !shape || !rope || !attn_q || !kv_k || !kv_v) return mi_fail(MI_ERR_ARG, "rope_rows: null pointer");
  if (in_kind > MI_OUT_F16 || paired > 1u || shape->act > 1u) return mi_fail(MI_ERR_ARG, "rope_rows: in_kind, paired and act are 0 or 1");
  const uint32_t hd = shape->head_dim, qh = shape->q_heads, kvh = shape->kv_heads;
  if (hd != 128 && hd != 256) return mi_fail(MI_ERR_SHAPE, "rope_rows: head_dim 128 or 256");
  if (qh == 0 || kvh == 0 || qh > 1024 || kvh > 1024) return mi_fail(MI_ERR_SHAPE, "rope_rows: 1..1024 q and kv heads");
  if (shape->gated || shape->k_off != qh * hd || shape->v_off != (qh + kvh) * hd || shape->qkv_n != (qh + 2u * kvh) * hd)
    return mi_fail(MI_ERR_SHAPE, "rope_rows: a plain q||k||v layout (not gated)");
  if (shape->rot_dim > hd || shape->rot_dim % 8 || shape->rot_dim == 0)
    return mi_fail(MI_ERR_SHAPE, "rope_rows: rot_dim a multiple of 8 up to head_dim");
  if (T == 0 || T > kMaxRows || rows == 0 || rope_len == 0)
    return mi_fail(MI_ERR_SHAPE, "rope_rows: T 1..65535, rows and rope_len from 1");
  if ((uint64_t)T * (qh + 2u * kvh) > 1u << 26) return mi_fail(MI_ERR_SHAPE, "rope_rows: 2^26 heads of rows at most");
  if (!pos && (uint64_t)pos0 + T > 0xFFFFFFFFull) return mi_fail(MI_ERR_SHAPE, "rope_rows: positions are below 2^32");
  if (in_stride < shape->qkv_n) return mi_fail(MI_ERR_ARG, "rope_rows: in_stride below qkv_n");
  if (off(qkv, in_kind == MI_OUT_F16 ? 2 : 4) || off(attn_q, 4) || off(kv_k, 2) || off(kv_v, 2) || off(rope, 4) || off(q_norm, 4) ||
      off(k_norm, 4) || off(pos, 4) || off(slots, 4) || off(flag, 4))
    return mi_fail(MI_ERR_ARG, "rope_rows: misaligned pointer (its elements' size)");
  const RowsArgs a{qkv, pos, slots, q_norm, k_norm, rope, attn_q, kv_k, kv_v, flag, in_stride, row_stride, head_stride, T, pos0, rows,
                   rope_len, qh, kvh, shape->rot_dim, shape->act, shape->eps};
  if (hd == 128) launch_rows<128>(a, in_kind == MI_OUT_F16, paired != 0, (hipStream_t)stream);
  else launch_rows<256>(a, in_kind == MI_OUT_F16, paired != 0, (hipStream_t)stream);
  return mi_hip((int)hipGetLastError(), "rope_rows");
}

}  // extern "C"
