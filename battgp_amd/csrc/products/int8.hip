// Products in 8-bit integers with one scale per row of either operand (bgp_int8_gemm), and what makes their operands
// (bgp_quantize_rows).
#include <stdarg.h>
#include <stdio.h>

#include "entry.h"
#include "tile.h"

namespace {

thread_local char g_error[512] = "";

template <class T> __device__ __forceinline__ double widen(T v);
template <> __device__ __forceinline__ double widen<double>(double v) { return v; }
template <> __device__ __forceinline__ double widen<float>(float v) { return (double)v; }
template <> __device__ __forceinline__ double widen<bf16_t>(bf16_t v) {
  const uint32_t u = (uint32_t)v.v << 16;
  float f;
  __builtin_memcpy(&f, &u, 4);
  return (double)f;
}
template <> __device__ __forceinline__ double widen<f16_t>(f16_t v) {
  _Float16 h;
  __builtin_memcpy(&h, &v, 2);
  return (double)(float)h;
}
// to 16 bits by way of an fp32 number rounded to odd, so that the two roundings are one
template <class T> __device__ __forceinline__ T narrow(double v) {
  float f = (float)v;
  const double back = (double)f;
  if (back != v && v - v == 0.0) {
    uint32_t u;
    __builtin_memcpy(&u, &f, 4);
    u = (fabs(back) > fabs(v) ? u - 1 : u) | 1;
    __builtin_memcpy(&f, &u, 4);
  }
  return round_to<T, float>(f);
}
template <> __device__ __forceinline__ double narrow<double>(double v) { return v; }
template <> __device__ __forceinline__ float narrow<float>(double v) { return (float)v; }

template <class T> struct ScaleOf { using type = float; };
template <> struct ScaleOf<double> { using type = double; };

struct QuantArgs {
  const void* x;
  int8_t* q;
  void *scale, *rest;
  int64_t M, K, ldx, ldq, ldr;
  int pow2;
};

// One workgroup per row: the largest magnitude, then the codes.  The second pass finds the row in the caches.
template <class T> __global__ __launch_bounds__(256) void quantize_rows_kernel(QuantArgs p) {
  using S = typename ScaleOf<T>::type;
  __shared__ double part[4];
  for (int64_t row = blockIdx.x; row < p.M; row += gridDim.x) {
    const T* x = static_cast<const T*>(p.x) + row * p.ldx;
    double top = 0.0;
    for (int64_t k = threadIdx.x; k < p.K; k += 256) {
      const double v = fabs(widen(x[k]));
      top = v > top || v != v ? v : top;  // a NaN stays
      if (top != top) break;
    }
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) {
      const double v = __shfl_xor(top, d);
      top = v > top || v != v ? v : top;
    }
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = top;
    __syncthreads();
    top = part[0];
#pragma unroll
    for (int w = 1; w < 4; ++w) top = part[w] > top || part[w] != part[w] ? part[w] : top;
    constexpr double tiny = sizeof(S) == 8 ? 0x1p-1022 : 0x1p-126;
    double scale;
    const bool finite = top - top == 0.0;
    if (!finite) {
      scale = top;
    } else if (p.pow2) {
      int e;
      const double m = frexp(top, &e);  // top = m 2^e, 1/2 <= m < 1
      scale = top > 0.0 ? ldexp(1.0, e - 7 + (m > 127.0 / 128.0)) : 0.0;
    } else {
      scale = (double)(S)(top / 127.0);
    }
    if (finite && scale < tiny) scale = tiny;
    if (threadIdx.x == 0) static_cast<S*>(p.scale)[row] = (S)scale;
    for (int64_t k = threadIdx.x; k < p.K; k += 256) {
      const double v = widen(x[k]);
      double q = finite ? rint(v / scale) : 0.0;
      q = fmin(fmax(q, -127.0), 127.0);
      p.q[row * p.ldq + k] = (int8_t)q;
      if (p.rest) static_cast<T*>(p.rest)[row * p.ldr + k] = narrow<T>(v - q * scale);
    }
    __syncthreads();  // the next row's maxima overwrite part[]
  }
}

struct Int8Args {
  const int8_t *a, *b;
  const void *sa, *sb, *c;
  void* y;
  int64_t M, N, K, lda, ldb, ldc, ldy;
  int tiles_n;
};

// Y[i, j] = (C[i, j] +) sa[i] sb[j] sum_k A[i, k] B[j, k]: the sum exact in 32 bits, the rest in 64, one rounding
template <class T, class P, int BM, int BN> __device__ __forceinline__ void int8_tile(const Int8Args& p, char* lds) {
  using S = typename ScaleOf<T>::type;
  // each XCD takes a run of tiles, 8 row tiles deep (workgroups go to the 8 XCDs in turn; each has an L2 of its own)
  constexpr int XCDS = 8, DEEP = 8;
  const int tiles_m = (int)((p.M + BM - 1) / BM);
  const int64_t total = (int64_t)tiles_m * p.tiles_n, run = (total + XCDS - 1) / XCDS, at = blockIdx.x / XCDS, t = blockIdx.x % XCDS * run + at;
  if (at >= run || t >= total) return;
  const int64_t strip = t / (DEEP * p.tiles_n);
  const int in = (int)(t - strip * DEEP * p.tiles_n), deep = tiles_m - strip * DEEP < DEEP ? (int)(tiles_m - strip * DEEP) : DEEP;
  const int64_t m0 = (strip * DEEP + in % deep) * BM, n0 = (int64_t)(in / deep) * BN;
  P tile;
  tile.run(Operand<int8_t>{p.a + m0 * p.lda, p.lda, p.M - m0}, Operand<int8_t>{p.b + n0 * p.ldb, p.ldb, p.N - n0}, p.K, lds);
  tile.each([&](int i, int j, int step, const v4i& v) {
    const int64_t row = m0 + i;
    if (row >= p.M) return;
    const double si = (double)static_cast<const S*>(p.sa)[row];
    T* y = static_cast<T*>(p.y) + row * p.ldy;
    const T* c = p.c ? static_cast<const T*>(p.c) + row * p.ldc : nullptr;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int64_t col = n0 + j + e * step;
      if (col >= p.N) break;
      double r = (double)v[e] * (si * (double)static_cast<const S*>(p.sb)[col]);
      if (c) r += widen(c[col]);
      y[col] = narrow<T>(r);
    }
  });
}

// any operands, through registers
template <class T, int BM, int BN> __global__ __launch_bounds__(256, 2) void int8_gemm_kernel(Int8Args p) {
  using P = Tile<int8_t, BM, BN, 2, 2, true, true, false>;
  __shared__ __attribute__((aligned(16))) char lds[P::LDS_BYTES];
  int8_tile<T, P, BM, BN>(p, lds);
}

// operands in whole chunks, pipelined
template <class T, int BM, int BN> __global__ __launch_bounds__(BM == 256 ? 512 : 256, 2) void int8_gemm_pipe_kernel(Int8Args p) {
  using P = PipeTile<int8_t, BM, BN, 2, BM == 256 ? 4 : 2, true, true>;
  __shared__ __attribute__((aligned(16))) char lds[P::LDS_BYTES];
  int8_tile<T, P, BM, BN>(p, lds);
}

template <class T, int B, bool PIPE> int run_int8(const Int8Args& p0, hipStream_t st) {
  Int8Args p = p0;
  p.tiles_n = (int)((p.N + B - 1) / B);
  const int64_t tiles = (p.M + B - 1) / B * p.tiles_n + 7;
  if (tiles > MAX_WORKGROUPS / 2) return bgp_products_fail(-1, "bgp_int8_gemm: %lld tiles are more than one launch holds", (long long)tiles);
  const dim3 grid((unsigned)tiles);
  if constexpr (PIPE) return launch("bgp_int8_gemm", int8_gemm_pipe_kernel<T, B, B>, grid, dim3(B == 256 ? 512 : 256), st, p);
  else return launch("bgp_int8_gemm", int8_gemm_kernel<T, B, B>, grid, dim3(256), st, p);
}

template <class T> int int8_by_type(const Int8Args& p, hipStream_t st) {
  const bool vec = reinterpret_cast<uintptr_t>(p.a) % 16 == 0 && reinterpret_cast<uintptr_t>(p.b) % 16 == 0 && p.lda % 16 == 0 && p.ldb % 16 == 0 &&
                   p.K % 16 == 0 && pipe_fits(p.lda, 1, true, 256) && pipe_fits(p.ldb, 1, true, 256);
  const int64_t tiles = ((p.M + 127) / 128) * ((p.N + 127) / 128);
  if (!vec) return tiles < 256 ? run_int8<T, 64, false>(p, st) : run_int8<T, 128, false>(p, st);
  if (tiles >= 1024) return run_int8<T, 256, true>(p, st);
  return tiles < 256 ? run_int8<T, 64, true>(p, st) : run_int8<T, 128, true>(p, st);
}

}  // namespace

int bgp_products_fail(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_error, sizeof(g_error), fmt, ap);
  va_end(ap);
  return code;
}

extern "C" const char* bgp_products_last_error(void) { return g_error; }

extern "C" int bgp_quantize_rows(int device, void* stream, int dtype, int64_t M, int64_t K, const void* x, int64_t ldx, int8_t* q, int64_t ldq, void* scale,
                                 int pow2, void* rest, int64_t ldr) {
  const char* what = "bgp_quantize_rows";
  if (dtype < BGP_F64 || dtype > BGP_F16) return bgp_products_fail(-1, "%s: unknown type %d", what, dtype);
  if (M < 0 || K < 0) return bgp_products_fail(-1, "%s: bad sizes M=%lld K=%lld", what, (long long)M, (long long)K);
  if (M == 0) return 0;
  if (!scale || (K > 0 && (!x || !q))) return bgp_products_fail(-1, "%s: null pointer", what);
  if (ldx < K || ldq < K || (rest && ldr < K)) return bgp_products_fail(-1, "%s: bad strides ldx=%lld ldq=%lld ldr=%lld", what, (long long)ldx, (long long)ldq, (long long)ldr);
  DeviceScope scope(device);
  if (int rc = scope.check(what)) return rc;
  const QuantArgs p{x, q, scale, rest, M, K, ldx, ldq, ldr, pow2 != 0};
  const dim3 grid((unsigned)(M < MAX_WORKGROUPS ? M : MAX_WORKGROUPS)), block(256);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case BGP_F64: return launch(what, quantize_rows_kernel<double>, grid, block, st, p);
    case BGP_F32: return launch(what, quantize_rows_kernel<float>, grid, block, st, p);
    case BGP_BF16: return launch(what, quantize_rows_kernel<bf16_t>, grid, block, st, p);
    default: return launch(what, quantize_rows_kernel<f16_t>, grid, block, st, p);
  }
}

extern "C" int bgp_int8_gemm(int device, void* stream, int dtype, int64_t M, int64_t N, int64_t K, const int8_t* A, int64_t lda, const int8_t* B, int64_t ldb,
                             const void* scale_a, const void* scale_b, const void* C, int64_t ldc, void* Y, int64_t ldy) {
  const char* what = "bgp_int8_gemm";
  if (dtype < BGP_F64 || dtype > BGP_F16) return bgp_products_fail(-1, "%s: unknown type %d", what, dtype);
  if (M < 0 || N < 0 || K < 0 || K > BGP_INT8_MAX_K)
    return bgp_products_fail(-1, "%s: bad sizes M=%lld N=%lld K=%lld (K <= %d: a longer sum can pass 32 bits)", what, (long long)M, (long long)N, (long long)K, BGP_INT8_MAX_K);
  if (M == 0 || N == 0) return 0;
  if (!Y || !scale_a || !scale_b || (K > 0 && (!A || !B))) return bgp_products_fail(-1, "%s: null pointer", what);
  if (lda < K || ldb < K || ldy < N || (C && ldc < N))
    return bgp_products_fail(-1, "%s: bad strides lda=%lld ldb=%lld ldc=%lld ldy=%lld", what, (long long)lda, (long long)ldb, (long long)ldc, (long long)ldy);
  DeviceScope scope(device);
  if (int rc = scope.check(what)) return rc;
  const Int8Args p{A, B, scale_a, scale_b, C, Y, M, N, K, lda, ldb, ldc, ldy, 0};
  const hipStream_t st = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case BGP_F64: return int8_by_type<double>(p, st);
    case BGP_F32: return int8_by_type<float>(p, st);
    case BGP_BF16: return int8_by_type<bf16_t>(p, st);
    default: return int8_by_type<f16_t>(p, st);
  }
}
