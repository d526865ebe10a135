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
#include <cstdio>

#include "mi_capi_internal.h"
#include "mi_common.h"

namespace mi {
namespace {

typedef int i4_t __attribute__((ext_vector_type(4)));
typedef unsigned short us2_t __attribute__((ext_vector_type(2)));

constexpr uint32_t kMaxK = 131072;  // the int32 sums stay below 2^31

__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
  return __builtin_bit_cast(uint32_t,
                            __builtin_elementwise_max(__builtin_bit_cast(us2_t, a), __builtin_bit_cast(us2_t, b)));
}
// the larger magnitude's bits of 8 f16 values and `m`, in pairs
__device__ __forceinline__ uint32_t max_abs8(uint32_t m, u4_t v) {
  const uint32_t a = max_u16x2(v.x & 0x7FFF7FFFu, v.y & 0x7FFF7FFFu), b = max_u16x2(v.z & 0x7FFF7FFFu, v.w & 0x7FFF7FFFu);
  return max_u16x2(m, max_u16x2(a, b));
}
// rne(x / s) as the low byte: |x / s| < 2^22, and 1.5 * 2^23 + r rounds r to an integer in the sum's low bits
__device__ __forceinline__ uint32_t quant_word(uint32_t p0, uint32_t p1, float s) {
  uint32_t b[4];
#pragma unroll
  for (uint32_t i = 0; i < 4; ++i) {
    const float v = h2f((uint16_t)((i < 2 ? p0 : p1) >> (16u * (i & 1u))));
    b[i] = __builtin_bit_cast(uint32_t, v / s + 12582912.0f);
  }
  const uint32_t lo = __builtin_amdgcn_perm(b[1], b[0], 0x0C0C0400u), hi = __builtin_amdgcn_perm(b[3], b[2], 0x0C0C0400u);
  return lo | (hi << 16);
}

// One wave per row, four rows per work-group; a unit is 16 of the row's values, the 16 bytes of one lane of a
// fragment: k = 64 c + 8 q .. + 7 and 64 c + 32 + 8 q .. + 7.
__global__ __launch_bounds__(256) void quant_rows_kernel(const uint16_t* __restrict__ x, size_t x_stride, uint32_t M,
                                                         uint32_t K, int8_t* __restrict__ q_tiled,
                                                         float* __restrict__ scales) {
  const uint32_t lane = threadIdx.x & 63u, m = blockIdx.x * 4u + (threadIdx.x >> 6), units = K / 16u;
  u4_t* to = reinterpret_cast<u4_t*>(q_tiled + (size_t)(m / 16u) * 16u * K) + m % 16u;
  if (m >= M) {  // the last fragment's rows behind the matrix
    for (uint32_t u = lane; u < units; u += 64u) to[16u * u] = u4_t{0u, 0u, 0u, 0u};
    return;
  }
  const uint16_t* row = x + (size_t)m * x_stride;
  auto piece = [&](uint32_t u, uint32_t half) {
    return *reinterpret_cast<const u4_t*>(row + 64u * (u >> 2) + 32u * half + 8u * (u & 3u));
  };
  uint32_t mx = 0;
  for (uint32_t u = lane; u < units; u += 64u) mx = max_abs8(max_abs8(mx, piece(u, 0)), piece(u, 1));
  // (f16 magnitudes are ordered as their bits; an infinity or a NaN is at or above 0x7C00)
  const uint32_t bits = (uint32_t)wave_max((float)max(mx & 0xFFFFu, mx >> 16));
  const bool finite = bits < 0x7C00u;
  const float s = finite ? h2f((uint16_t)bits) / 127.0f : __builtin_bit_cast(float, kNanBits);
  if (lane == 0) scales[m] = s;
  const bool zero = !finite || bits == 0;
  for (uint32_t u = lane; u < units; u += 64u) {
    const u4_t a = piece(u, 0), b = piece(u, 1);
    u4_t w = {quant_word(a.x, a.y, s), quant_word(a.z, a.w, s), quant_word(b.x, b.y, s), quant_word(b.z, b.w, s)};
    if (zero) w = u4_t{0u, 0u, 0u, 0u};
    to[16u * u] = w;
  }
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
__device__ __forceinline__ void store4(const GemmArgs& a, uint32_t m, uint32_t n, i4_t acc) {
  const float s = a.qs[m];
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

// 2 x 2 waves of 64 x 64 outputs each, operands straight from memory. A is the weights, so a lane ends with four
// adjacent columns of one row.
template <bool F32>
__global__ __launch_bounds__(256) void gemm_w8a8_kernel(GemmArgs a) {
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
  const uint32_t nc = a.K / 64u, nt = a.N / 16u, mt = (a.M + 15u) / 16u;
  const uint32_t n0 = (blockIdx.x * 2u + (wave & 1u)) * 4u, m0 = (blockIdx.y * 2u + (wave >> 1)) * 4u;
  const u4_t *wp[4], *qp[4];
#pragma unroll
  for (uint32_t i = 0; i < 4; ++i) {  // (a tile behind the matrix reads its last one and stores nothing)
    wp[i] = a.w + (size_t)min(n0 + i, nt - 1u) * nc * 64u + lane;
    qp[i] = a.q + (size_t)min(m0 + i, mt - 1u) * nc * 64u + lane;
  }
  i4_t acc[4][4];
#pragma unroll
  for (uint32_t i = 0; i < 4; ++i)
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) acc[i][j] = i4_t{0, 0, 0, 0};
  for (uint32_t c = 0; c < nc; ++c) {
    i4_t wv[4], qv[4];
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
      wv[i] = __builtin_bit_cast(i4_t, wp[i][(size_t)c * 64u]);
      qv[i] = __builtin_bit_cast(i4_t, qp[i][(size_t)c * 64u]);
    }
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i)
#pragma unroll
      for (uint32_t j = 0; j < 4; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wv[i], qv[j], acc[i][j], 0, 0, 0);
  }
#pragma unroll
  for (uint32_t j = 0; j < 4; ++j) {
    const uint32_t m = (m0 + j) * 16u + (lane & 15u);
    if (m >= a.M) continue;
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i)
      if (n0 + i < nt) store4<F32>(a, m, (n0 + i) * 16u + 4u * (lane >> 4), acc[i][j]);
  }
}

int launch_gemm(const GemmArgs& a, uint32_t out_kind, hipStream_t st) {
  const dim3 grid((a.N + 127u) / 128u, (a.M + 127u) / 128u);
  if (out_kind == MI_OUT_F32) gemm_w8a8_kernel<true><<<grid, 256, 0, st>>>(a);
  else gemm_w8a8_kernel<false><<<grid, 256, 0, st>>>(a);
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
  quant_rows_kernel<<<(M + 15u) / 16u * 4u, 256, 0, (hipStream_t)stream>>>(x, x_stride, M, K, q_tiled, row_scales);
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
  if (int e = mi_quant_rows_i8(x, x_stride, M, K, q, qs, stream)) return e;
  const GemmArgs a{reinterpret_cast<const u4_t*>(q), qs, reinterpret_cast<const u4_t*>(w_tiled), w_scales, out,
                   out_stride, M, K, N};
  return launch_gemm(a, out_kind, (hipStream_t)stream);
}

}  // extern "C"
