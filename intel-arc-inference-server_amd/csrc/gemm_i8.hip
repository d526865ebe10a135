// gemm_i8.hip - the linear in 8-bit integers (W8A8): rows of f16 activations quantised with a scale each,
// a product of int8 matrices on the matrix cores, a scale for each output column.
//
//   s_m = max_k |x[m][k]| / 127 (fp32),  q[m][k] = rne(x[m][k] / s_m)
//   out[m][n] = ((float)(sum_k q[m][k] w[n][k]) * s_m) * ws[n]
//
// The sum is an int32 and exact (K <= 131072: 131072 * 127 * 127 < 2^31), so an output's bits depend neither on
// the tile that computes it nor on the other rows: a row among 2048 is bitwise that row alone.
//
// Both operands are held in mi_i8w_index's layout, [rows / 16][K / 64][64 lanes][16 bytes], which is the order in
// which v_mfma_i32_16x16x64_i8 takes them: lane l holds row l % 16 at 16 of the chunk's 64 k, the same 16 in both
// operands (which 16 is free, the sum runs over all of them). A fragment of 16 rows x 64 k is 1 KiB, contiguous.
//
// What bounds it (MI355X): few rows the weights' bytes (13 rows 5120 -> 34816: 30.4 us, 5.9 TB/s), a single one of few
// columns also the row's own chain (maximum, quotients, then the products: 5120 -> 7168 9.4 us, 3.9 TB/s); many rows the
// matrix cores with the reads of their operands from LDS close behind (2048 rows 5120 -> 34816: 318 us, 2.3 PTOP/s; the
// largest library product on the card 2.06); some hundred rows the operands' way into LDS and out again, 192 rows and columns
// for 64 x 128 products per k (333 rows 17408 -> 5120: 51 us, 60 with the quantiser).
#include <cstdio>

#include "mi_capi_internal.h"
#include "mi_pieces.h"

namespace mi {
namespace {

typedef int i4_t __attribute__((ext_vector_type(4)));
typedef unsigned short us2_t __attribute__((ext_vector_type(2)));

constexpr uint32_t kMaxK = 131072;  // the int32 sums stay below 2^31
constexpr uint32_t kFusedK = 32768;  // the longest single row that a product quantises for itself, one byte of LDS for each k

__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
  return __builtin_bit_cast(uint32_t,
                            __builtin_elementwise_max(__builtin_bit_cast(us2_t, a), __builtin_bit_cast(us2_t, b)));
}
// the larger magnitude's bits of 8 f16 values and `m`, in pairs
__device__ __forceinline__ uint32_t max_abs8(uint32_t m, u4_t v) {
  const uint32_t a = max_u16x2(v.x & 0x7FFF7FFFu, v.y & 0x7FFF7FFFu), b = max_u16x2(v.z & 0x7FFF7FFFu, v.w & 0x7FFF7FFFu);
  return max_u16x2(m, max_u16x2(a, b));
}
// rne(x / s) as the low byte, |x / s| <= 127: 1.5 * 2^23 + r rounds r to an integer in the sum's low bits. The
// quotient is the fp32 one of the definition wherever that matters: x times the rounded 1 / s is within 2^-15 of it,
// so only a product nearer than 2^-13 to a border between integers (one in 4096) is divided.
__device__ __forceinline__ uint32_t quant_word(uint32_t p0, uint32_t p1, float s, float inv) {
  constexpr float kMagic = 12582912.0f;
  uint32_t b[4];
  bool near = false;
  float v[4];
#pragma unroll
  for (uint32_t i = 0; i < 4; ++i) {
    v[i] = h2f((uint16_t)((i < 2 ? p0 : p1) >> (16u * (i & 1u))));
    const float r = v[i] * inv, m = r + kMagic;
    near |= fabsf(r - (m - kMagic)) > 0.5f - 0x1p-13f;
    b[i] = __builtin_bit_cast(uint32_t, m);
  }
  if (near) {
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) b[i] = __builtin_bit_cast(uint32_t, v[i] / s + kMagic);
  }
  const uint32_t lo = __builtin_amdgcn_perm(b[1], b[0], 0x0C0C0400u), hi = __builtin_amdgcn_perm(b[3], b[2], 0x0C0C0400u);
  return lo | (hi << 16);
}
// A unit is 16 of a row's values, the 16 bytes of one lane of a fragment: unit u = 4 c + q holds
// k = 64 c + 8 q .. + 7 (a) and 64 c + 32 + 8 q .. + 7 (b).
struct Unit {
  u4_t a, b;
};
__device__ __forceinline__ Unit load_unit(const uint16_t* row, uint32_t u) {
  const u4_t* p = reinterpret_cast<const u4_t*>(row + 64u * (u >> 2) + 8u * (u & 3u));
  return {p[0], p[4]};
}
// the row's scale from its largest magnitude's bits (f16 magnitudes are ordered as their bits; an infinity or a NaN is at
// or above 0x7C00)
struct Scale {
  float s, inv;
  bool zero;  // the row's integers are zeros: a zero row, or one that is not finite
};
__device__ __forceinline__ Scale row_scale(uint32_t bits) {
  const bool finite = bits < 0x7C00u;
  const float s = finite ? h2f((uint16_t)bits) / 127.0f : __builtin_bit_cast(float, kNanBits);
  return {s, 1.0f / s, !finite || bits == 0u};
}
__device__ __forceinline__ u4_t quant_unit(const Unit& v, const Scale& s) {
  const u4_t w = {quant_word(v.a.x, v.a.y, s.s, s.inv), quant_word(v.a.z, v.a.w, s.s, s.inv), quant_word(v.b.x, v.b.y, s.s, s.inv),
                  quant_word(v.b.z, v.b.w, s.s, s.inv)};
  return s.zero ? u4_t{0u, 0u, 0u, 0u} : w;
}
__device__ __forceinline__ uint32_t max_bits(uint32_t m) { return (uint32_t)wave_max((float)max(m & 0xFFFFu, m >> 16)); }

// A work-group of W waves per row, up to U units per lane held in registers between the maximum and the quotients. A row
// writes 16 bytes in each 256 of its fragments, so a fragment's 16 rows go to one XCD, whose L2 makes whole lines of them:
// 333 rows of 17408 7.0 us (8.9 with the rows dealt out in order), 2048 of 5120 7.7 (9.9; 4.1 TB/s), 2048 of 17408 20.6
// (35.3; 5.2 TB/s).
template <uint32_t W, uint32_t U>
__global__ __launch_bounds__(64 * W) void quant_rows_kernel(const uint16_t* __restrict__ x, size_t x_stride, uint32_t M, uint32_t K,
                                                            int8_t* __restrict__ q_tiled, float* __restrict__ scales) {
  const uint32_t wave = threadIdx.x >> 6, t = threadIdx.x, units = K / 16u;
  const uint32_t tile = blockIdx.x / 128u * 8u + blockIdx.x % 8u, m = tile * 16u + blockIdx.x / 8u % 16u;
  if (tile * 16u >= M) return;
  u4_t* to = reinterpret_cast<u4_t*>(q_tiled + (size_t)(m / 16u) * 16u * K) + m % 16u;
  if (m >= M) {  // the last fragment's rows behind the matrix
    for (uint32_t u = t; u < units; u += 64u * W) to[16u * u] = u4_t{0u, 0u, 0u, 0u};
    return;
  }
  const uint16_t* row = x + (size_t)m * x_stride;
  Unit v[U];
  uint32_t mx = 0;
#pragma unroll
  for (uint32_t i = 0; i < U; ++i)
    if (t + 64u * W * i < units) v[i] = load_unit(row, t + 64u * W * i);
#pragma unroll
  for (uint32_t i = 0; i < U; ++i)
    if (t + 64u * W * i < units) mx = max_abs8(max_abs8(mx, v[i].a), v[i].b);
  uint32_t bits = max_bits(mx);
  __shared__ uint32_t part[W];
  if ((threadIdx.x & 63u) == 0) part[wave] = bits;
  __syncthreads();
#pragma unroll
  for (uint32_t i = 0; i < W; ++i) bits = max(bits, part[i]);
  const Scale s = row_scale(bits);
  if (t == 0) scales[m] = s.s;
#pragma unroll
  for (uint32_t i = 0; i < U; ++i)
    if (t + 64u * W * i < units) to[16u * (t + 64u * W * i)] = quant_unit(v[i], s);
}
// As many waves as the units take; more of them for the same rows are no faster (16 for 333 rows of 17408: 7.1 us, 8 7.0), nor is
// one wave for each of 2048 rows of 5120 (9.5).
void launch_quant(const uint16_t* x, size_t x_stride, uint32_t M, uint32_t K, int8_t* q, float* s, hipStream_t st) {
  const uint32_t rows = (M + 127u) / 128u * 128u;
  if (K <= 8192) quant_rows_kernel<4, 2><<<rows, 256, 0, st>>>(x, x_stride, M, K, q, s);
  else if (K <= 32768) quant_rows_kernel<8, 4><<<rows, 512, 0, st>>>(x, x_stride, M, K, q, s);
  else quant_rows_kernel<16, 8><<<rows, 1024, 0, st>>>(x, x_stride, M, K, q, s);
}

struct GemmArgs {
  const u4_t* q;       // [ceil(M / 16)][K / 64][64] fragments' lanes
  const float* qs;     // [M]
  const u4_t* w;       // [N / 16][K / 64][64]
  const float* ws;     // [N]
  void* out;
  size_t out_stride;
  uint32_t M, K, N;
};

// the four outputs n .. n + 3 of row m
template <bool F32>
__device__ __forceinline__ void store4(const GemmArgs& a, float s, uint32_t m, uint32_t n, i4_t acc) {
  const f4_t ws = *reinterpret_cast<const f4_any*>(a.ws + n);
  f4_t v;
#pragma unroll
  for (uint32_t r = 0; r < 4; ++r) v[r] = ((float)acc[r] * s) * ws[r];
  const size_t o = (size_t)m * a.out_stride + n;
  if constexpr (F32) {
    *reinterpret_cast<f4_any*>(static_cast<float*>(a.out) + o) = v;
  } else {
    const u2_t h = {(uint32_t)f2h(v[0]) | ((uint32_t)f2h(v[1]) << 16), (uint32_t)f2h(v[2]) | ((uint32_t)f2h(v[3]) << 16)};
    *reinterpret_cast<h4_any*>(static_cast<uint16_t*>(a.out) + o) = h;
  }
}

// Few rows: MT x 16 rows and NT x 16 columns per work-group, whose W waves deal the chunks of k out among them, U at a
// time each. Both operands come straight from memory (a lane without a row loads none); A is the weights, so a lane ends
// with four adjacent columns of a row. The waves' sums join through LDS.
// FUSED (MT 1, a single row): the row is the f16 one, which every work-group quantises for itself into LDS behind its
// first weights' loads, in place of a launch whose 4 us the weights wait for. Against the two launches: 5120 -> 7168
// 9.4 us (12.3), 17408 -> 5120 20.4 (23.7), 1024 -> 512 3.6 (6.6), 5120 -> 151936 111.8 (114.4), 32768 -> 4096 24.5
// (27.6). More rows cost each work-group more of that work: two are 33.6 (30.3) at 5120 -> 34816, four 14.8 (12.4) at
// 5120 -> 7168, so they take the two launches.
template <bool F32, uint32_t MT, uint32_t NT, uint32_t W, uint32_t U, bool FUSED>
__global__ __launch_bounds__(64 * W) void gemm_w8a8_few_kernel(GemmArgs a, const uint16_t* x) {
  static_assert(!FUSED || MT == 1);
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
  const uint32_t nc = a.K / 64u, nt = a.N / 16u;
  const uint32_t n0 = blockIdx.x * NT, m0 = blockIdx.y * MT;
  const u4_t* wp[NT];
  const u4_t* qp[MT];
  bool have[MT];
#pragma unroll
  for (uint32_t i = 0; i < NT; ++i) wp[i] = a.w + (size_t)min(n0 + i, nt - 1u) * nc * 64u + lane;
#pragma unroll
  for (uint32_t j = 0; j < MT; ++j) {
    have[j] = (m0 + j) * 16u + (lane & 15u) < a.M;
    qp[j] = FUSED ? nullptr : a.q + (size_t)(have[j] ? m0 + j : 0u) * nc * 64u + lane;
  }
  u4_t wv[U][NT];
  auto load_w = [&](uint32_t c0) {
#pragma unroll
    for (uint32_t u = 0; u < U; ++u)
#pragma unroll
      for (uint32_t i = 0; i < NT; ++i)
        wv[u][i] = load_stream16(reinterpret_cast<const uint32_t*>(wp[i] + (size_t)min(c0 + u, nc - 1u) * 64u));
  };
  uint32_t c0 = wave * U;
  if constexpr (FUSED) load_w(c0);
  extern __shared__ __align__(16) u4_t row_units[];  // FUSED: the row's K bytes, as [K / 64][4][16]
  __shared__ uint32_t top[W];
  Scale row{};
  if constexpr (FUSED) {
    const uint32_t units = a.K / 16u;
    uint32_t mx = 0;
    for (uint32_t u = threadIdx.x; u < units; u += 64u * W) {
      const Unit v = load_unit(x, u);
      mx = max_abs8(max_abs8(mx, v.a), v.b);
    }
    mx = max_bits(mx);
    if (lane == 0) top[wave] = mx;
    lds_barrier();
    uint32_t bits = top[0];
#pragma unroll
    for (uint32_t i = 1; i < W; ++i) bits = max(bits, top[i]);
    row = row_scale(bits);
    for (uint32_t u = threadIdx.x; u < units; u += 64u * W) row_units[u] = quant_unit(load_unit(x, u), row);
    lds_barrier();
  }
  i4_t acc[MT][NT];
#pragma unroll
  for (uint32_t j = 0; j < MT; ++j)
#pragma unroll
    for (uint32_t i = 0; i < NT; ++i) acc[j][i] = i4_t{0, 0, 0, 0};
  auto multiply = [&](uint32_t at) {
    u4_t qv[U][MT];
#pragma unroll
    for (uint32_t u = 0; u < U; ++u)
#pragma unroll
      for (uint32_t j = 0; j < MT; ++j) {
        qv[u][j] = u4_t{0u, 0u, 0u, 0u};
        if (have[j] && at + u < nc) {
          if constexpr (FUSED) qv[u][j] = row_units[4u * (at + u) + (lane >> 4)];
          else qv[u][j] = *as_global(qp[j] + (size_t)(at + u) * 64u);
        }
      }
#pragma unroll
    for (uint32_t u = 0; u < U; ++u)
#pragma unroll
      for (uint32_t j = 0; j < MT; ++j)
#pragma unroll
        for (uint32_t i = 0; i < NT; ++i)
          acc[j][i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i4_t, wv[u][i]), __builtin_bit_cast(i4_t, qv[u][j]),
                                                            acc[j][i], 0, 0, 0);
  };
  if constexpr (FUSED) {
    multiply(c0);
    c0 += W * U;
  }
#pragma unroll 1
  for (; c0 < nc; c0 += W * U) {
    load_w(c0);
    multiply(c0);
  }
  __shared__ __align__(16) i4_t part[W][MT * NT][64];
#pragma unroll
  for (uint32_t j = 0; j < MT; ++j)
#pragma unroll
    for (uint32_t i = 0; i < NT; ++i) part[wave][j * NT + i][lane] = acc[j][i];
  __syncthreads();
  for (uint32_t t = wave; t < MT * NT; t += W) {
    const uint32_t m = (m0 + t / NT) * 16u + (lane & 15u), tile = n0 + t % NT;
    if (m >= a.M || tile >= nt) continue;
    i4_t sum = part[0][t][lane];
#pragma unroll
    for (uint32_t p = 1; p < W; ++p) sum += part[p][t][lane];
    store4<F32>(a, FUSED ? row.s : a.qs[m], m, tile * 16u + 4u * (lane >> 4), sum);
  }
}

// One fragment (1 KiB, 16 bytes per lane) from memory straight into LDS. The compiler does not see what this writes, nor
// count the load: a kernel that uses it leaves no load of its own in flight and waits by vmcnt itself.
__device__ __forceinline__ void load_fragment(uint32_t lds, const u4_t* from, uint32_t lane16) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(lane16), "s"(from) : "memory");
}

// Many rows: WM x WN waves of 16 RM rows x 16 CN columns, KS times over the parts of k. Both operands go into LDS in
// fragment order, by direct loads into a ring of NS chunks, and from there into registers a chunk ahead of the products.
// A is the weights: a lane ends with four adjacent columns of a row.
template <uint32_t RM, uint32_t CN, uint32_t WM, uint32_t WN, uint32_t KS, uint32_t NS>
struct Stage {
  static constexpr uint32_t TM = RM * WM, TN = CN * WN, TT = TM + TN;  // 16-row and 16-column tiles of the work-group
  union {
    u4_t stage[KS][NS][TT][64];
    i4_t sums[KS > 1 ? (KS - 1) * RM * CN * WM * WN * 64 : 1];  // the other parts' sums
  };
};
// the work-group's share from the 16-row tile m0 and the 16-column tile n0 on
template <bool F32, uint32_t RM, uint32_t CN, uint32_t WM, uint32_t WN, uint32_t KS, uint32_t NS>
__device__ __forceinline__ void multiply_tile(const GemmArgs& a, Stage<RM, CN, WM, WN, KS, NS>& sm, uint32_t m0, uint32_t n0) {
  constexpr uint32_t TM = RM * WM, TN = CN * WN, TT = TM + TN;
  constexpr uint32_t PW = WM * WN;            // waves of a part
  constexpr uint32_t L = (TT + PW - 1) / PW;  // fragments a wave loads per chunk
  const uint32_t nt = a.N / 16u, mt = (a.M + 15u) / 16u, nc = a.K / 64u;
  const uint32_t lane = threadIdx.x & 63u, wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const uint32_t ks = wave / PW, pw = wave % PW, wm = pw / WN, wn = pw % WN;
  // this wave's fragments of a chunk: tile ft of the rows, then the columns (a tile behind the matrix is its last one, and
  // a wave without a fragment loads the last once more)
  const u4_t* from[L];
  uint32_t at[L];
#pragma unroll
  for (uint32_t i = 0; i < L; ++i) {
    const uint32_t ft = min(pw + PW * i, TT - 1u);
    from[i] = ft < TM ? a.q + (size_t)min(m0 + ft, mt - 1u) * nc * 64u : a.w + (size_t)min(n0 + ft - TM, nt - 1u) * nc * 64u;
    at[i] = (uint32_t)(uintptr_t)&sm.stage[ks][0][ft][0];
  }
  // this part's i-th chunk is KS i + ks (one behind the last is that one again, times zeros)
  const uint32_t steps = (nc + KS - 1u) / KS;
  auto load = [&](uint32_t k, uint32_t i, uint32_t slot) {
    load_fragment(at[k] + slot * (TT * 1024u), from[k] + (size_t)min(KS * i + ks, nc - 1u) * 64u, 16u * lane);
  };
  struct Operands {
    i4_t w[CN], x[RM];
  } f0, f1;
  auto read = [&](uint32_t k, Operands& f, uint32_t slot) {
    const u4_t(*st)[64] = sm.stage[ks][slot];
    if (k < CN) f.w[k] = __builtin_bit_cast(i4_t, st[TM + wn * CN + k][lane]);
    else f.x[k - CN] = __builtin_bit_cast(i4_t, st[wm * RM + k - CN][lane]);
  };
  i4_t acc[RM][CN];
#pragma unroll
  for (uint32_t j = 0; j < RM; ++j)
#pragma unroll
    for (uint32_t i = 0; i < CN; ++i) acc[j][i] = i4_t{0, 0, 0, 0};
#pragma unroll
  for (uint32_t i = 0; i < NS; ++i)
#pragma unroll
    for (uint32_t k = 0; k < L; ++k) load(k, i, i);
  asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((NS - 1u) * L) : "memory");
#pragma unroll
  for (uint32_t k = 0; k < RM + CN; ++k) read(k, f0, 0);
  uint32_t slot = 0;
  auto step = [&](uint32_t i, Operands& now, Operands& next) {
    // the next chunk is in LDS once every wave's fragments are, and this one's slot is free once every wave has read it
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((NS - 2u) * L) : "memory");
    const uint32_t freed = slot;
    slot = slot + 1u == NS ? 0u : slot + 1u;
    // The reads of the next chunk's operands and the loads of a later chunk's fragments, dealt out between the products:
    // one behind the other they would leave the matrix core idle for as long as they take to issue.
    constexpr uint32_t OPS = RM + CN + L, PER = RM * CN >= OPS ? RM * CN / OPS : 1, MORE = (OPS + RM * CN / PER - 1) / (RM * CN / PER);
    if (KS > 1 && KS * i + ks >= nc) {
#pragma unroll
      for (uint32_t k = 0; k < CN; ++k) now.w[k] = i4_t{0, 0, 0, 0};
    }
#pragma unroll
    for (uint32_t p = 0; p < RM * CN; ++p) {
      if (p % PER == 0) {
#pragma unroll
        for (uint32_t o = p / PER * MORE; o < (p / PER + 1u) * MORE; ++o) {
          if (o < RM + CN) read(o, next, slot);
          else if (o < OPS) load(o - RM - CN, i + NS, freed);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      acc[p / CN][p % CN] = __builtin_amdgcn_mfma_i32_16x16x64_i8(now.w[p % CN], now.x[p / CN], acc[p / CN][p % CN], 0, 0, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  uint32_t i = 0;
  for (; i + 2u <= steps; i += 2u) {
    step(i, f0, f1);
    step(i + 1u, f1, f0);
  }
  if (i < steps) step(i, f0, f1);
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
  if constexpr (KS > 1) {
    // the other parts hand their sums to the first
    i4_t* sums = sm.sums + pw * RM * CN * 64u + lane;
    constexpr uint32_t kPart = PW * RM * CN * 64;
    if (ks)
#pragma unroll
      for (uint32_t j = 0; j < RM; ++j)
#pragma unroll
        for (uint32_t k = 0; k < CN; ++k) sums[(ks - 1u) * kPart + (j * CN + k) * 64u] = acc[j][k];
    __syncthreads();
    if (ks) return;
#pragma unroll
    for (uint32_t p = 0; p + 1u < KS; ++p)
#pragma unroll
      for (uint32_t j = 0; j < RM; ++j)
#pragma unroll
        for (uint32_t k = 0; k < CN; ++k) acc[j][k] += sums[p * kPart + (j * CN + k) * 64u];
  }
#pragma unroll
  for (uint32_t j = 0; j < RM; ++j) {
    const uint32_t m = (m0 + wm * RM + j) * 16u + (lane & 15u);
    if (m >= a.M) continue;
    const float s = a.qs[m];
#pragma unroll
    for (uint32_t k = 0; k < CN; ++k) {
      const uint32_t tile = n0 + wn * CN + k;
      if (tile < nt) store4<F32>(a, s, m, tile * 16u + 4u * (lane >> 4), acc[j][k]);
    }
  }
}

// An XCD takes a run of column tiles with all their row tiles (the rows fastest): what it holds in its L2 at a time is
// shared by the work-groups it runs at a time. The id-th of `count` (a multiple of 8) work-groups' place in these runs:
__device__ __forceinline__ uint32_t in_runs(uint32_t id, uint32_t count) { return (id & 7u) * (count / 8u) + (id >> 3); }
template <bool F32, uint32_t RM, uint32_t CN, uint32_t WM, uint32_t WN, uint32_t KS, uint32_t NS>
__global__ __launch_bounds__(64 * WM * WN * KS, 2) void gemm_w8a8_kernel(GemmArgs a, uint32_t m_tiles) {
  __shared__ __align__(16) Stage<RM, CN, WM, WN, KS, NS> sm;
  const uint32_t id = in_runs(blockIdx.x, gridDim.x), n0 = id / m_tiles * (CN * WN);
  if (n0 < a.N / 16u) multiply_tile<F32, RM, CN, WM, WN, KS, NS>(a, sm, id % m_tiles * (RM * WM), n0);
}
// 256 x 256 where half a round of the CUs' tiles or less is left behind the whole rounds: those are cut into quarters of
// 128 x 128, which take half a tile's time, all CUs at once. Measured (us; without): 1000 rows 5120 -> 34816, 544 tiles, 168
// (194); 2048 rows 5120 -> 34816, 1088 tiles, 318 (344); 1000 rows 5120 -> 22528, 352 tiles, 123 (127); 500 rows
// 5120 -> 151936, 1188 tiles with 164 behind the whole rounds, 390 (381).
template <bool F32>
__global__ __launch_bounds__(512, 2) void gemm_w8a8_quarters_kernel(GemmArgs a, uint32_t m_tiles, uint32_t whole) {
  __shared__ __align__(16) union {
    Stage<8, 4, 2, 4, 1, 4> whole;
    Stage<4, 2, 2, 4, 1, 8> quarter;
  } sm;
  if (blockIdx.x < whole) {
    const uint32_t id = in_runs(blockIdx.x, whole);
    multiply_tile<F32, 8, 4, 2, 4, 1, 4>(a, sm.whole, id % m_tiles * 16u, id / m_tiles * 16u);
  } else {
    const uint32_t q = in_runs(blockIdx.x - whole, gridDim.x - whole), id = whole + q / 4u;
    const uint32_t m0 = id % m_tiles * 16u + 8u * (q & 1u), n0 = id / m_tiles * 16u + 4u * (q & 2u);
    if (n0 < a.N / 16u && 16u * m0 < a.M) multiply_tile<F32, 4, 2, 2, 4, 1, 8>(a, sm.quarter, m0, n0);
  }
}

template <bool F32, uint32_t RM, uint32_t CN, uint32_t WM, uint32_t WN, uint32_t KS, uint32_t NS>
void launch_tiles(const GemmArgs& a, hipStream_t st) {
  const uint32_t m_tiles = (a.M + 16u * RM * WM - 1u) / (16u * RM * WM), n_tiles = (a.N + 16u * CN * WN - 1u) / (16u * CN * WN);
  gemm_w8a8_kernel<F32, RM, CN, WM, WN, KS, NS><<<(m_tiles * n_tiles + 7u) / 8u * 8u, 64 * WM * WN * KS, 0, st>>>(a, m_tiles);
}
uint32_t tiles_256(uint32_t M, uint32_t N) { return (M + 255u) / 256u * ((N + 255u) / 256u); }
bool in_quarters(uint32_t tiles) { return tiles >= 256u && tiles % 256u != 0 && tiles % 256u <= 128u; }
template <bool F32>
void launch_256(const GemmArgs& a, hipStream_t st) {
  const uint32_t tiles = tiles_256(a.M, a.N), rest = tiles % 256u;
  if (!in_quarters(tiles)) return launch_tiles<F32, 8, 4, 2, 4, 1, 4>(a, st);
  gemm_w8a8_quarters_kernel<F32><<<tiles - rest + (4u * rest + 7u) / 8u * 8u, 512, 0, st>>>(a, (a.M + 255u) / 256u, tiles - rest);
}
template <bool F32, uint32_t MT, uint32_t NT, uint32_t W, uint32_t U>
void launch_few(const GemmArgs& a, hipStream_t st) {
  gemm_w8a8_few_kernel<F32, MT, NT, W, U, false>
      <<<dim3((a.N + 16u * NT - 1u) / (16u * NT), (a.M + 16u * MT - 1u) / (16u * MT)), 64 * W, 0, st>>>(a, nullptr);
}
template <uint32_t NT, uint32_t W, uint32_t U>
void launch_fused(const GemmArgs& a, uint32_t out_kind, const uint16_t* x, hipStream_t st) {
  const uint32_t wgs = (a.N + 16u * NT - 1u) / (16u * NT);
  if (out_kind == MI_OUT_F32) gemm_w8a8_few_kernel<true, 1, NT, W, U, true><<<wgs, 64 * W, a.K, st>>>(a, x);
  else gemm_w8a8_few_kernel<false, 1, NT, W, U, true><<<wgs, 64 * W, a.K, st>>>(a, x);
}

// The work-group's shape by the least modelled time in ns,
//   launch + turn r + step s c + work w s / 256 + weights K N / 10^6 + out M N / 10^6
// with w work-groups, s = K / (64 parts) steps of each, c = ceil(w / 256) work-groups a CU runs and r of them one after
// another (`occ` fit a CU at once); a last round in quarters counts 0.52 in c for up to 64 tiles, 0.95 for up to 128. The
// constants were fitted to every shape's times at 790 random sizes (1..2048 rows, K 256..17408, N 256..151936; a fifth of
// them this library's layers): the choice is 2.8 % off the best shape on average.
// Measured (us; the chosen shape, then others) at K -> N:
//   5120 -> 7168:   1 row 7.4 (16 x 16, 16 parts), 16 x 32 8.3, 64 x 64 10.3; 128 rows 12.3 (64 x 64, 4 parts), 64 x 32 18.8, 128 x 128 21.6;
//                   1000 rows 38.8 (128 x 256), 128 x 128 41.0, 256 x 256 55.6
//   5120 -> 34816:  13 rows 30.4 (16 x 32), 16 x 16 32.7; 128 rows 54.3 (128 x 256), 64 x 128 69.5; 2048 rows 318 (256 x 256), 128 x 256 381
//   17408 -> 5120:  333 rows 53.8 (64 x 128), 64 x 64 67.0, 128 x 256 107; 1000 rows 106 (192 x 256), 128 x 256 111
//   5120 -> 151936: 500 rows 374 (256 x 256), 128 x 256 453
enum Shape { kFew16x16, kFew16x16w, kFew16x32, kFew32x32, kFew64x16, kTile64p4, kTile64, kTile64x128, kTile128, kTile128x256, kTile192x256, kTile256 };
Shape pick(uint32_t M, uint32_t K, uint32_t N) {
  static constexpr struct {
    Shape shape;
    uint32_t rows, cols, parts, occ, most;  // most: rows it is meant for
    double launch, turn, step, work, weights, out;
  } kShapes[] = {{kFew16x16, 16, 16, 4, 8, 64u, 3757, 0, 89, 54, 0, 429},
                  {kFew16x16w, 16, 16, 16, 2, 64u, 3837, 0, 251, 294, 0, 2498},
                  {kFew16x32, 16, 32, 4, 8, 64u, 3475, 209, 187, 72, 1, 0},
                  {kFew32x32, 32, 32, 4, 6, 128u, 3634, 0, 221, 67, 0, 641},
                  {kFew64x16, 64, 16, 8, 4, 256u, 3666, 0, 263, 65, 0, 2705},
                  {kTile64p4, 64, 64, 4, 1, ~0u, 1859, 2180, 291, 140, 45, 1213},
                  {kTile64, 64, 64, 2, 2, ~0u, 2417, 1485, 162, 32, 54, 833},
                  {kTile64x128, 64, 128, 2, 1, ~0u, 1702, 2425, 195, 113, 80, 615},
                  {kTile128, 128, 128, 1, 2, ~0u, 3826, 118, 167, 51, 55, 871},
                  {kTile128x256, 128, 256, 1, 1, ~0u, 2392, 1775, 291, 97, 61, 797},
                  {kTile192x256, 192, 256, 1, 1, ~0u, 1798, 2791, 401, 125, 41, 830},
                  {kTile256, 256, 256, 1, 1, ~0u, 1714, 2879, 491, 146, 35, 871}};
  Shape best = kTile128;
  double least = 1e300;
  for (const auto& s : kShapes) {
    if (M > s.most) continue;
    const uint64_t w = (uint64_t)((M + s.rows - 1u) / s.rows) * ((N + s.cols - 1u) / s.cols);
    const double steps = (K / 64u + s.parts - 1u) / s.parts;
    const double rounds = s.shape == kTile256 && in_quarters((uint32_t)w) ? (double)(w / 256u) + (w % 256u <= 64u ? 0.52 : 0.95)
                                                                          : (double)((w + 255u) / 256u);
    const double t = s.launch + s.turn * (double)((w + 256u * s.occ - 1u) / (256u * s.occ)) + s.step * steps * rounds +
                     s.work * steps * (double)w / 256.0 + s.weights * 1e-6 * K * N + s.out * 1e-6 * M * N;
    if (t < least) {
      least = t;
      best = s.shape;
    }
  }
  return best;
}

template <bool F32>
void launch_shape(Shape p, const GemmArgs& a, hipStream_t st) {
  switch (p) {
    case kFew16x16: return launch_few<F32, 1, 1, 4, 8>(a, st);
    case kFew16x16w: return launch_few<F32, 1, 1, 16, 4>(a, st);
    case kFew16x32: return launch_few<F32, 1, 2, 4, 4>(a, st);
    case kFew32x32: return launch_few<F32, 2, 2, 4, 4>(a, st);
    case kFew64x16: return launch_few<F32, 4, 1, 8, 2>(a, st);
    case kTile64p4: return launch_tiles<F32, 4, 2, 1, 2, 4, 4>(a, st);
    case kTile64: return launch_tiles<F32, 4, 2, 1, 2, 2, 5>(a, st);
    case kTile64x128: return launch_tiles<F32, 2, 4, 2, 2, 2, 6>(a, st);
    case kTile128: return launch_tiles<F32, 4, 4, 2, 2, 1, 5>(a, st);
    case kTile128x256: return launch_tiles<F32, 4, 4, 2, 4, 1, 6>(a, st);
    case kTile192x256: return launch_tiles<F32, 6, 4, 2, 4, 1, 5>(a, st);
    case kTile256: return launch_256<F32>(a, st);
  }
}
int launch_gemm(const GemmArgs& a, uint32_t out_kind, hipStream_t st) {
  const Shape p = pick(a.M, a.K, a.N);
  if (out_kind == MI_OUT_F32) launch_shape<true>(p, a, st);
  else launch_shape<false>(p, a, st);
  return mi_hip((int)hipGetLastError(), "gemm_w8a8");
}

bool misaligned(const void* p, size_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1u)) != 0; }

int check_product(const char* name, uint32_t M, uint32_t K, uint32_t N, uint32_t out_kind, const void* out,
                  size_t out_stride, const int8_t* w, const float* w_scales) {
  static thread_local char msg[160];
  auto refuse = [&](int code, const char* what) {
    std::snprintf(msg, sizeof msg, "%s: %s", name, what);
    return mi_fail(code, msg);
  };
  if (!w || !w_scales || !out) return refuse(MI_ERR_ARG, "null pointer");
  if (M == 0 || M > 1u << 20 || K == 0 || K % 64 || K > kMaxK || N == 0 || N % 16 || N > 1u << 22)
    return refuse(MI_ERR_SHAPE, "M 1..2^20, K a multiple of 64 up to 131072, N a multiple of 16 up to 2^22");
  if (out_kind != MI_OUT_F32 && out_kind != MI_OUT_F16) return refuse(MI_ERR_ARG, "out_kind is MI_OUT_F32 or MI_OUT_F16");
  if (out_stride < N) return refuse(MI_ERR_ARG, "out_stride below N");
  if (misaligned(w, 16) || misaligned(w_scales, 4) || misaligned(out, out_kind == MI_OUT_F32 ? 4 : 2))
    return refuse(MI_ERR_ARG, "misaligned pointer (weights 16 bytes, scales 4, out its elements)");
  return 0;
}

size_t tiled_bytes(uint32_t M, uint32_t K) { return ((size_t)M + 15u) / 16u * 16u * K; }

int check_rows(const char* name, const uint16_t* x, size_t x_stride, uint32_t M, uint32_t K) {
  static thread_local char msg[160];
  const char* what = nullptr;
  int code = MI_ERR_ARG;
  if (!x) what = "null pointer";
  else if (M == 0 || M > 1u << 20 || K == 0 || K % 64 || K > kMaxK) {
    what = "M 1..2^20, K a multiple of 64 up to 131072";
    code = MI_ERR_SHAPE;
  } else if (misaligned(x, 16) || x_stride % 8 || x_stride < K) what = "x 16-byte aligned, its stride a multiple of 8 and at least K";
  if (!what) return 0;
  std::snprintf(msg, sizeof msg, "%s: %s", name, what);
  return mi_fail(code, msg);
}

}  // namespace
}  // namespace mi

using namespace mi;

extern "C" {

int mi_quant_rows_i8(const uint16_t* x, size_t x_stride, uint32_t M, uint32_t K, int8_t* q_tiled, float* row_scales,
                     void* stream) {
  if (int e = check_rows("quant_rows_i8", x, x_stride, M, K)) return e;
  if (!q_tiled || !row_scales || misaligned(q_tiled, 16) || misaligned(row_scales, 4))
    return mi_fail(MI_ERR_ARG, "quant_rows_i8: null or misaligned output (the rows 16 bytes, the scales 4)");
  launch_quant(x, x_stride, M, K, q_tiled, row_scales, (hipStream_t)stream);
  return mi_hip((int)hipGetLastError(), "quant_rows_i8");
}

int mi_gemm_w8a8(const int8_t* q_tiled, const float* row_scales, const int8_t* w_tiled, const float* w_scales, void* out,
                 uint32_t out_kind, size_t out_stride, uint32_t M, uint32_t K, uint32_t N, void* stream) {
  if (int e = check_product("gemm_w8a8", M, K, N, out_kind, out, out_stride, w_tiled, w_scales)) return e;
  if (!q_tiled || !row_scales || misaligned(q_tiled, 16) || misaligned(row_scales, 4))
    return mi_fail(MI_ERR_ARG, "gemm_w8a8: null or misaligned rows (16 bytes) or row scales (4)");
  const GemmArgs a{reinterpret_cast<const u4_t*>(q_tiled), row_scales, reinterpret_cast<const u4_t*>(w_tiled), w_scales,
                   out, out_stride, M, K, N};
  return launch_gemm(a, out_kind, (hipStream_t)stream);
}

size_t mi_linear_w8a8_ws(uint32_t M, uint32_t K) { return tiled_bytes(M, K) + (size_t)M * 4u; }

int mi_linear_w8a8(const uint16_t* x, size_t x_stride, const int8_t* w_tiled, const float* w_scales, void* ws,
                   size_t ws_bytes, void* out, uint32_t out_kind, size_t out_stride, uint32_t M, uint32_t K, uint32_t N,
                   void* stream) {
  if (int e = check_rows("linear_w8a8", x, x_stride, M, K)) return e;
  if (int e = check_product("linear_w8a8", M, K, N, out_kind, out, out_stride, w_tiled, w_scales)) return e;
  if (!ws || misaligned(ws, 16) || ws_bytes < mi_linear_w8a8_ws(M, K))
    return mi_fail(MI_ERR_ARG, "linear_w8a8: the workspace is null, misaligned (16 bytes) or below mi_linear_w8a8_ws");
  int8_t* q = static_cast<int8_t*>(ws);
  float* qs = reinterpret_cast<float*>(q + tiled_bytes(M, K));
  if (M == 1 && K <= kFusedK) {
    const GemmArgs a{nullptr, nullptr, reinterpret_cast<const u4_t*>(w_tiled), w_scales, out, out_stride, M, K, N};
    // 16 waves where all work-groups run at once, two to a CU: 24.5 us (4 waves 27.1) at 32768 -> 4096; where they take
    // turns each turn waits for its row again: 30.7 (28.1) at 5120 -> 34816
    const Shape p = pick(M, K, N);
    if (p == kFew16x32) launch_fused<2, 4, 4>(a, out_kind, x, (hipStream_t)stream);
    else if (p == kFew16x16w && N <= 8192u) launch_fused<1, 16, 4>(a, out_kind, x, (hipStream_t)stream);
    else launch_fused<1, 4, 8>(a, out_kind, x, (hipStream_t)stream);
    return mi_hip((int)hipGetLastError(), "linear_w8a8");
  }
  if (int e = mi_quant_rows_i8(x, x_stride, M, K, q, qs, stream)) return e;
  const GemmArgs a{reinterpret_cast<const u4_t*>(q), qs, reinterpret_cast<const u4_t*>(w_tiled), w_scales, out,
                   out_stride, M, K, N};
  return launch_gemm(a, out_kind, (hipStream_t)stream);
}

}  // extern "C"
