// Products in 8-bit integers with one scale per row of either operand (bgp_int8_gemm), and what makes their operands
// (bgp_quantize_rows).
//
// Whole calls with the quantisation of A before them, from the host's side, on an MI355X: 8192^3 to bf16 0.49 ms (quantise 47 us:
// 202 MB at 4.3 TB/s; product 455 us: 2400 TOP/s, where clocks fall under the load); one row to 4096 x 4096 9.2 us, two launches
// at 3.8 us each from the host; an fp64 slice of 8192 x 1024 x 1024 added to fp64 79 us (36 + 38 us for 143 + 143 MB, bound by memory).
#include <stdarg.h>
#include <stdio.h>

#include <type_traits>

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
};

// Quantisation computes in fp32 for the types up to 32 bits and in fp64 for fp64.  The largest magnitude is found on the
// bit patterns without their sign, where an infinity is above every number and a NaN above that.
template <class T> struct Quant {
  using F = float;
  using B = uint32_t;
  static constexpr F tiny = 0x1p-126f;
  static constexpr B inf = 0x7f800000u;
};
template <> struct Quant<double> {
  using F = double;
  using B = uint64_t;
  static constexpr F tiny = 0x1p-1022;
  static constexpr B inf = 0x7ff0000000000000ull;
};
template <class A, class C> __device__ __forceinline__ A bits_as(C v) {
  static_assert(sizeof(A) == sizeof(C), "same size");
  A r;
  __builtin_memcpy(&r, &v, sizeof(A));
  return r;
}
template <class T> __device__ __forceinline__ typename Quant<T>::B magnitude(typename Quant<T>::F v) {
  using B = typename Quant<T>::B;
  return bits_as<B>(v) & (~(B)0 >> 1);
}

// the largest of the 64 lanes' values: inside rows of 16 lanes, then across them; it ends up in lane 63
template <int CTRL, int ROWS> __device__ __forceinline__ uint32_t dpp(uint32_t v) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false); }
template <int CTRL, int ROWS> __device__ __forceinline__ uint64_t dpp(uint64_t v) {
  return (uint64_t)dpp<CTRL, ROWS>((uint32_t)(v >> 32)) << 32 | dpp<CTRL, ROWS>((uint32_t)v);
}
template <int CTRL, int ROWS, class B> __device__ __forceinline__ B max_step(B v) {
  const B o = dpp<CTRL, ROWS>(v);
  return o > v ? o : v;
}
template <class B> __device__ __forceinline__ B wave_max(B v) {
  v = max_step<0x111, 0xf>(v);
  v = max_step<0x112, 0xf>(v);
  v = max_step<0x114, 0xf>(v);
  v = max_step<0x118, 0xf>(v);
  v = max_step<0x142, 0xa>(v);
  v = max_step<0x143, 0xc>(v);
  const uint32_t lo = __builtin_amdgcn_readlane((int)v, 63);
  if constexpr (sizeof(B) == 4) return lo;
  else return (B)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), 63) << 32 | lo;
}

// A row by TPR threads, U units of 8 elements each: the row stays in registers between the search for its scale and the
// codes, so x is read once.  With one unit the code is short, and fetching code is what short kernels wait for (16384 x 1024
// bf16 numbers: 25 us with four units a thread, 15 with one; 16 rows: 7.8 and 3.8); large matrices of long rows have
// fewer waves to start with four (8192 x 8192: 44 us against 51).  LONG: rows of more than 8 U TPR elements, read twice
// (the second time out of the caches).
template <class T, bool POW2, int TPR, int U, bool LONG> __global__ __launch_bounds__(TPR > 256 ? TPR : 256) void quantize_rows_kernel(QuantArgs p) {
  using F = typename Quant<T>::F;
  using B = typename Quant<T>::B;
  constexpr int NT = TPR > 256 ? TPR : 256, RPW = NT / TPR, WPR = TPR / 64;
  __shared__ B part[NT / 64];
  const int lane = threadIdx.x % TPR;
  const int64_t row = (int64_t)blockIdx.x * RPW + threadIdx.x / TPR;
  const bool mine = row < p.M;
  const T* x = static_cast<const T*>(p.x) + (mine ? row : 0) * p.ldx;
  const int64_t K = mine ? p.K : 0;
  F v[U][8];
  auto load = [&](int64_t k, F* f) {
    T e[8] = {};
    if (k + 8 <= K) {
      constexpr int N = (int)sizeof(T) / 2;  // 16-byte chunks
#pragma unroll
      for (int c = 0; c < N; ++c) {
        const chunk_t u = load_any(x + k + c * CHE<T>);
        __builtin_memcpy(e + c * CHE<T>, &u, 16);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (k + j < K) e[j] = x[k + j];
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = (F)widen(e[j]);
  };
  B top = 0;
  auto look = [&](const F* f) {
#pragma unroll
    for (int j = 0; j < 8; ++j) top = magnitude<T>(f[j]) > top ? magnitude<T>(f[j]) : top;
  };
#pragma unroll
  for (int u = 0; u < U; ++u) {
    load((u * TPR + lane) * 8, v[u]);
    look(v[u]);
  }
  if (LONG)
    for (int64_t k = (U * TPR + lane) * 8; k < K; k += TPR * 8) {
      F f[8];
      load(k, f);
      look(f);
    }
  top = wave_max(top);
  if (WPR > 1) {
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = top;
    __syncthreads();
    const int first = threadIdx.x / TPR * WPR;
#pragma unroll
    for (int w = 0; w < WPR; ++w) top = part[first + w] > top ? part[first + w] : top;
  }
  const bool finite = top < Quant<T>::inf;
  F scale = bits_as<F>(top);
  if (finite) {
    if (POW2) {
      // top = m 2^e with 1/2 <= m < 1: the smallest p with top <= 127 p is 2^(e - 7) or twice that
      int e;
      const F m = sizeof(F) == 8 ? (F)frexp((double)scale, &e) : (F)frexpf((float)scale, &e);
      scale = scale > 0 ? (F)ldexp(1.0, e - 7 + (m > (F)(127.0 / 128.0))) : (F)0;
    } else {
      scale = scale / (F)127;
    }
    if (scale < Quant<T>::tiny) scale = Quant<T>::tiny;
  }
  if (lane == 0 && mine) static_cast<F*>(p.scale)[row] = scale;
  const F inv = (F)1 / scale;
  auto put = [&](int64_t k, const F* f) {
    int8_t q[8];
    T r[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      F t = 0, left = f[j];
      if (finite) {
        // The product with the reciprocal is a hair off the quotient, so t may be the wrong neighbour where the quotient
        // lies next to a half; what is left over says so, and it is exact: a multiple of half the last place of
        // the scale, not larger than the scale.  (A power of two: the product is exact, and t right.)
        t = rint(f[j] * inv);
        left = fma(-t, scale, f[j]);
        if (!POW2) {
          const F twice = fabs(left) * 2;
          if (twice > scale || (twice == scale && ((int)t & 1))) {
            const F up = left > 0 ? (F)1 : (F)-1;
            t += up;
            left = fma(-up, scale, left);
          }
        }
      } else {
        left = f[j] - f[j] + bits_as<F>(~(B)0);  // no number
      }
      q[j] = (int8_t)t;
      r[j] = round_to<T, F>(left);
    }
    int8_t* out = p.q + row * p.ldq + k;
    T* rest = p.rest ? static_cast<T*>(p.rest) + row * p.ldr + k : nullptr;
    if (k + 8 <= K) {
      struct __attribute__((packed, aligned(1))) Eight { int8_t e[8]; } o;
      __builtin_memcpy(&o, q, 8);
      *reinterpret_cast<Eight*>(out) = o;
      if (rest) {
        constexpr int N = (int)sizeof(T) / 2;
#pragma unroll
        for (int c = 0; c < N; ++c) {
          Chunk<sizeof(T)> u;
          __builtin_memcpy(&u, r + c * CHE<T>, 16);
          *reinterpret_cast<Chunk<sizeof(T)>*>(rest + c * CHE<T>) = u;
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (k + j < K) {
          out[j] = q[j];
          if (rest) rest[j] = r[j];
        }
    }
  };
#pragma unroll
  for (int u = 0; u < U; ++u) put((u * TPR + lane) * 8, v[u]);
  if (LONG)
    for (int64_t k = (U * TPR + lane) * 8; k < K; k += TPR * 8) {
      F f[8];
      load(k, f);
      put(k, f);
    }
}

template <class T, bool POW2, int TPR, int U, bool LONG> int run_quantize(const QuantArgs& p, hipStream_t st) {
  constexpr int NT = TPR > 256 ? TPR : 256, RPW = NT / TPR;
  constexpr int64_t MOST = max_workgroups(NT) * RPW;
  for (int64_t from = 0; from < p.M; from += MOST) {
    QuantArgs q = p;
    q.M = p.M - from < MOST ? p.M - from : MOST;
    q.x = static_cast<const T*>(p.x) + from * p.ldx;
    q.q = p.q + from * p.ldq;
    q.scale = static_cast<typename Quant<T>::F*>(p.scale) + from;
    q.rest = p.rest ? static_cast<T*>(p.rest) + from * p.ldr : nullptr;
    if (int rc = launch("bgp_quantize_rows", quantize_rows_kernel<T, POW2, TPR, U, LONG>, dim3((unsigned)((q.M + RPW - 1) / RPW)), dim3(NT), st, q)) return rc;
  }
  return 0;
}

template <class T, bool POW2> int quantize_by_length(const QuantArgs& p, hipStream_t st) {
  if (p.K <= 512) return run_quantize<T, POW2, 64, 1, false>(p, st);
  if (p.K <= 1024) return run_quantize<T, POW2, 128, 1, false>(p, st);
  if (p.K <= 2048) return run_quantize<T, POW2, 256, 1, false>(p, st);
  if (p.K <= 4096) return run_quantize<T, POW2, 512, 1, false>(p, st);
  if (p.K <= 8192 && p.M >= 8 * CUS) return run_quantize<T, POW2, 256, 4, false>(p, st);
  if (p.K <= 8192) return run_quantize<T, POW2, 1024, 1, false>(p, st);
  return run_quantize<T, POW2, 1024, 1, true>(p, st);
}

template <class T> int quantize_by_type(const QuantArgs& p, int pow2, hipStream_t st) {
  return pow2 ? quantize_by_length<T, true>(p, st) : quantize_by_length<T, false>(p, st);
}

struct Int8Args {
  const int8_t *a, *b;
  const void *sa, *sb, *c;
  void* y;
  int64_t M, N, K, lda, ldb, ldc, ldy;
  int tiles_n;
};

// N neighbours of a row, at the alignment of one
template <class T, int N> struct __attribute__((packed, aligned(sizeof(T)))) Few { T e[N]; };

// scaled sums to D's rows, 16 bytes at a time; C is fetched for AHEAD units before the first is stored (the compiler may
// not do that: C can be D)
template <class T, bool ADD> struct ScaledRows {
  using S = typename ScaleOf<T>::type;
  static constexpr int E = 16 / (int)sizeof(T), AHEAD = ADD && sizeof(T) >= 4 ? 4 : 2;
  T* y;
  const T* c;
  const S *sa, *sb;
  int64_t ldy, ldc, cols;
  struct Other {
    Few<T, ADD ? E : 1> add;
  };
  __device__ __forceinline__ Other other(int i, int j) const {
    Other o;
    if constexpr (ADD)
      if (j + E <= cols) o.add = *reinterpret_cast<const Few<T, E>*>(c + i * ldc + j);
    return o;
  }
  __device__ __forceinline__ void single(int i, int j, int v) const {
    if (j >= cols) return;
    const double r = (double)v * ((double)sa[i] * (double)sb[j]);
    y[i * ldy + j] = narrow<T>(ADD ? r + widen(c[i * ldc + j]) : r);
  }
  __device__ __forceinline__ void operator()(int i, int j, const int* v, const Other& t) const {
    if (j + E <= cols) {
      const Few<S, E> s = *reinterpret_cast<const Few<S, E>*>(sb + j);
      const double si = (double)sa[i];
      Few<T, E> o;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        double r = (double)v[e] * (si * (double)s.e[e]);
        if constexpr (ADD) r += widen(t.add.e[e]);
        o.e[e] = narrow<T>(r);
      }
      *reinterpret_cast<Few<T, E>*>(y + i * ldy + j) = o;
    } else {
#pragma unroll 1
      for (int e = 0; e < E; ++e) single(i, j + e, v[e]);
    }
  }
};

// Y[i, j] = (C[i, j] +) sa[i] sb[j] sum_k A[i, k] B[j, k]: the sum exact in 32 bits, the rest in 64, one rounding
template <class T, class P, int BM, int BN> __device__ __forceinline__ void int8_tile(const Int8Args& p, int64_t m0, int64_t n0, char* lds) {
  using S = typename ScaleOf<T>::type;
  P tile;
  tile.run(Operand<int8_t>{p.a + m0 * p.lda, p.lda, p.M - m0, p.K >= 16}, Operand<int8_t>{p.b + n0 * p.ldb, p.ldb, p.N - n0, p.K >= 16}, p.K, lds);
  const S *sa = static_cast<const S*>(p.sa) + m0, *sb = static_cast<const S*>(p.sb) + n0;
  T* y = static_cast<T*>(p.y) + m0 * p.ldy + n0;
  const T* c = p.c ? static_cast<const T*>(p.c) + m0 * p.ldc + n0 : nullptr;
  const int64_t rows = p.M - m0, cols = p.N - n0;
  if (c) tile.template out<ScaledRows<T, true>::E>(lds, rows, ScaledRows<T, true>{y, c, sa, sb, p.ldy, p.ldc, cols});
  else tile.template out<ScaledRows<T, false>::E>(lds, rows, ScaledRows<T, false>{y, c, sa, sb, p.ldy, p.ldc, cols});
}

template <class T, class P, int BM, int BN> __device__ __forceinline__ void int8_workgroup(const Int8Args& p, char* lds) {
  const int tiles_m = (int)((p.M + BM - 1) / BM);
  const int i = place_runs(tiles_m * p.tiles_n);
  if (i < 0) return;
  const TileAt at = tile_at(i, tiles_m, p.tiles_n);
  int8_tile<T, P, BM, BN>(p, (int64_t)at.m * BM, (int64_t)at.n * BN, lds);
}

// 8 waves on 256 x 256
template <class T> __global__ __launch_bounds__(512, 2) void int8_gemm_pipe256_kernel(Int8Args p) {
  using P = PipeTile<int8_t, 256, 256, 2, 4, true, true>;
  __shared__ __attribute__((aligned(16))) char lds[P::LDS_BYTES];
  const int tiles_m = (int)((p.M + 255) / 256);
  const Place place = place_256(tiles_m * p.tiles_n);
  if (place.tile < 0) return;
  const TileAt at = tile_at(place.tile, tiles_m, p.tiles_n);
  int64_t m0 = (int64_t)at.m * 256, n0 = (int64_t)at.n * 256;
  if (place.parts == 1) {
    int8_tile<T, P, 256, 256>(p, m0, n0, lds);
    return;
  }
  m0 += (place.parts == 4 ? place.part >> 1 : place.part) * 128;
  if (place.parts == 4) n0 += (place.part & 1) * 128;
  if (m0 >= p.M || n0 >= p.N) return;
  if (place.parts == 4) int8_tile<T, PipeTile<int8_t, 128, 128, 2, 4, true, true>, 128, 128>(p, m0, n0, lds);
  else int8_tile<T, PipeTile<int8_t, 128, 256, 2, 4, true, true>, 128, 256>(p, m0, n0, lds);
}

// any operands, through registers
template <class T, int BM, int BN> __global__ __launch_bounds__(256, 2) void int8_gemm_kernel(Int8Args p) {
  using P = Tile<int8_t, BM, BN, 2, 2, true, true>;
  __shared__ __attribute__((aligned(16))) char lds[P::LDS_BYTES];
  int8_workgroup<T, P, BM, BN>(p, lds);
}

// operands in whole chunks, pipelined
template <class T, int BM, int BN, int SETS> __global__ __launch_bounds__(SETS * tile_threads(BM, 1), 2) void int8_gemm_pipe_kernel(Int8Args p) {
  using P = PipeTile<int8_t, BM, BN, 2, waves_w(BM, 1), true, true, SETS>;
  __shared__ __attribute__((aligned(16))) char lds[P::LDS_BYTES];
  int8_workgroup<T, P, BM, BN>(p, lds);
}

// small ones, straight from memory
template <class T, int F, bool ODD> __global__ __launch_bounds__(256) void int8_gemm_direct_kernel(Int8Args p) {
  using P = DirectTile<int8_t, F, F, true, true, ODD>;
  __shared__ __attribute__((aligned(16))) char lds[P::LDS_BYTES];
  int8_workgroup<T, P, 16 * F, 16 * F>(p, lds);
}

template <class T, int CUT> int run_int8(const Int8Args& p0, hipStream_t st) {
  const char* what = "bgp_int8_gemm";
  constexpr int B = tile_of(CUT), SETS = CUT == TWIN64 ? 2 : 1;
  Int8Args p = p0;
  p.tiles_n = (int)((p.N + B - 1) / B);
  const int64_t tiles = (p.M + B - 1) / B * p.tiles_n + (B == 256 ? CUS : 7);
  const dim3 grid((unsigned)tiles);
  if constexpr (CUT <= DIRECT32) {
    if (off_words(p.a, p.lda, 0, 1) || off_words(p.b, p.ldb, 0, 1))
      return launch(what, int8_gemm_direct_kernel<T, B / 16, true>, grid, dim3(256), st, p);
    return launch(what, int8_gemm_direct_kernel<T, B / 16, false>, grid, dim3(256), st, p);
  } else if constexpr (CUT <= PLAIN128) {
    return launch(what, int8_gemm_kernel<T, B, B>, grid, dim3(256), st, p);
  } else if constexpr (CUT == PIPE256) {
    return launch(what, int8_gemm_pipe256_kernel<T>, grid, dim3(512), st, p);
  } else {
    return launch(what, int8_gemm_pipe_kernel<T, B, B, SETS>, grid, dim3(SETS * tile_threads(B, 1)), st, p);
  }
}

template <class T> int run_int8_cut(const Int8Args& p, int cut, hipStream_t st) {
  switch (cut) {
    case DIRECT16: return run_int8<T, DIRECT16>(p, st);
    case DIRECT32: return run_int8<T, DIRECT32>(p, st);
    case PLAIN64: return run_int8<T, PLAIN64>(p, st);
    case PLAIN128: return run_int8<T, PLAIN128>(p, st);
    case PIPE64: return run_int8<T, PIPE64>(p, st);
    case PIPE128: return run_int8<T, PIPE128>(p, st);
    case TWIN64: return run_int8<T, TWIN64>(p, st);
    default: return run_int8<T, PIPE256>(p, st);
  }
}

template <int SIZE> __global__ __launch_bounds__(256) void pack_kernel(PackJob a, PackJob b) {
  using T = typename std::conditional<SIZE == 1, int8_t, typename std::conditional<SIZE == 2, bf16_t, typename std::conditional<SIZE == 4, float, double>::type>::type>::type;
  const PackJob& p = blockIdx.z ? b : a;
  const int64_t c = ((int64_t)blockIdx.x * 64 + threadIdx.x) * CHE<T>;
  if (c >= p.ld_to) return;
  for (int64_t r = (int64_t)blockIdx.y * 4 + threadIdx.y; r < p.rows; r += (int64_t)gridDim.y * 4) {
    const T* from = static_cast<const T*>(p.from) + r / p.per * p.stride + r % p.per * p.ld + c;
    *reinterpret_cast<chunk_t*>(static_cast<T*>(p.to) + r * p.ld_to + c) = p.extent - c >= CHE<T> ? load_any(from) : load_few(from, p.extent - c);
  }
}

}  // namespace

int bgp_products_fail(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_error, sizeof(g_error), fmt, ap);
  va_end(ap);
  return code;
}

int launch_pack(const char* what, int size, const PackJob* jobs, int count, hipStream_t st) {
  int64_t chunks = 0, rows = 0;
  for (int i = 0; i < count; ++i) {
    chunks = jobs[i].ld_to * size / 16 > chunks ? jobs[i].ld_to * size / 16 : chunks;
    rows = jobs[i].rows > rows ? jobs[i].rows : rows;
  }
  if (!chunks || !rows) return 0;
  const int64_t y = (rows + 3) / 4;
  const dim3 grid((unsigned)((chunks + 63) / 64), (unsigned)(y < 65535 ? y : 65535), (unsigned)count), block(64, 4);
  const PackJob a = jobs[0], b = jobs[count - 1];
  switch (size) {
    case 1: return launch(what, pack_kernel<1>, grid, block, st, a, b);
    case 2: return launch(what, pack_kernel<2>, grid, block, st, a, b);
    case 4: return launch(what, pack_kernel<4>, grid, block, st, a, b);
    default: return launch(what, pack_kernel<8>, grid, block, st, a, b);
  }
}

extern "C" const char* bgp_products_last_error(void) { return g_error; }

extern "C" int bgp_quantize_rows(int device, void* stream, int dtype, int64_t M, int64_t K, const void* x, int64_t ldx, int8_t* q, int64_t ldq, void* scale,
                                 int pow2, void* rest, int64_t ldr) {
  const char* what = "bgp_quantize_rows";
  if (dtype < BGP_F64 || dtype > BGP_F16) return bgp_products_fail(-1, "%s: unknown type %d", what, dtype);
  if (M < 0 || K < 0) return bgp_products_fail(-1, "%s: bad sizes M=%lld K=%lld", what, (long long)M, (long long)K);
  if (M == 0) return 0;
  if (!scale || (K > 0 && (!x || !q))) return bgp_products_fail(-1, "%s: null pointer", what);
  if (ldx < K || ldq < K || (rest && (ldr < K || (rest == x && ldr != ldx && M > 1))))
    return bgp_products_fail(-1, "%s: bad strides ldx=%lld ldq=%lld ldr=%lld", what, (long long)ldx, (long long)ldq, (long long)ldr);
  DeviceScope scope(device);
  if (int rc = scope.check(what)) return rc;
  const QuantArgs p{x, q, scale, rest, M, K, ldx, ldq, ldr};
  const hipStream_t st = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case BGP_F64: return quantize_by_type<double>(p, pow2, st);
    case BGP_F32: return quantize_by_type<float>(p, pow2, st);
    case BGP_BF16: return quantize_by_type<bf16_t>(p, pow2, st);
    default: return quantize_by_type<f16_t>(p, pow2, st);
  }
}

extern "C" int64_t bgp_int8_gemm(int device, void* stream, int dtype, int64_t M, int64_t N, int64_t K, const int8_t* A, int64_t lda, const int8_t* B,
                                 int64_t ldb, const void* scale_a, const void* scale_b, const void* C, int64_t ldc, void* Y, int64_t ldy, void* workspace,
                                 int64_t workspace_bytes) {
  const char* what = "bgp_int8_gemm";
  if (dtype < BGP_F64 || dtype > BGP_F16) return bgp_products_fail(-1, "%s: unknown type %d", what, dtype);
  if (M < 0 || N < 0 || K < 0 || K > BGP_INT8_MAX_K)
    return bgp_products_fail(-1, "%s: bad sizes M=%lld N=%lld K=%lld (K <= %d: a longer sum can pass 32 bits)", what, (long long)M, (long long)N, (long long)K, BGP_INT8_MAX_K);
  if (M == 0 || N == 0) return 0;
  if (!Y || !scale_a || !scale_b || (K > 0 && (!A || !B))) return bgp_products_fail(-1, "%s: null pointer", what);
  if (lda < K || ldb < K || ldy < N || (C && ldc < N) || (C == Y && ldc != ldy))
    return bgp_products_fail(-1, "%s: bad strides lda=%lld ldb=%lld ldc=%lld ldy=%lld", what, (long long)lda, (long long)ldb, (long long)ldc, (long long)ldy);
  const int64_t to = padded_row(K, 1);
  const bool a_ok = reinterpret_cast<uintptr_t>(A) % 16 == 0 && lda % 16 == 0 && pipe_fits(lda, 1, true, 256);
  const bool b_ok = reinterpret_cast<uintptr_t>(B) % 16 == 0 && ldb % 16 == 0 && pipe_fits(ldb, 1, true, 256);
  const Plan plan = plan_int8((dtype == BGP_F64 ? 8 : dtype == BGP_F32 ? 4 : 2) * (C ? 2 : 1), M, N, K,
                              Operands{a_ok && b_ok, (a_ok ? 0.0 : (double)M * to) + (b_ok ? 0.0 : (double)N * to)});
  if (plan.cut == CUTS) return bgp_products_fail(-1, "%s: M=%lld N=%lld are more tiles than one launch holds", what, (long long)M, (long long)N);
  Int8Args p{A, B, scale_a, scale_b, C, Y, M, N, K, lda, ldb, ldc, ldy, 0};
  Workspace ws(workspace);
  PackJob jobs[2];
  int count = 0;
  if (plan.pack && !a_ok) {
    p.a = static_cast<int8_t*>(ws.take(M * to));
    p.lda = to;
    jobs[count++] = PackJob{A, const_cast<int8_t*>(p.a), M, M, 0, lda, K, to};
  }
  if (plan.pack && !b_ok) {
    p.b = static_cast<int8_t*>(ws.take(N * to));
    p.ldb = to;
    jobs[count++] = PackJob{B, const_cast<int8_t*>(p.b), N, N, 0, ldb, K, to};
  }
  if (ws.short_of(workspace_bytes)) return ws.used();
  if (!ws.aligned()) return bgp_products_fail(-1, "%s: the workspace is not aligned to 16 bytes", what);
  DeviceScope scope(device);
  if (int rc = scope.check(what)) return rc;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (count)
    if (int rc = launch_pack(what, 1, jobs, count, st)) return rc;
  switch (dtype) {
    case BGP_F64: return run_int8_cut<double>(p, plan.cut, st);
    case BGP_F32: return run_int8_cut<float>(p, plan.cut, st);
    case BGP_BF16: return run_int8_cut<bf16_t>(p, plan.cut, st);
    default: return run_int8_cut<f16_t>(p, plan.cut, st);
  }
}
