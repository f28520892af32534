// Matrix products grouped by expert (bgp_grouped_gemm, bgp_grouped_gemm_dw): the rows of one matrix, sorted by group,
// against each group's own weights, in one launch.  The group bounds are read on the device, so nothing waits for them;
// the host sizes the grid by what they can be at most and the workgroups beyond the last tile leave at once.
#include "entry.h"
#include "tile.h"

namespace {

// The group of the `want`-th tile of BM rows.  Groups count their own tiles (a tile never crosses a bound); with
// `rest` != 0 the rows before the first and behind the last group follow as groups G and G + 1.  Bounds are clamped to
// [0, T], so wrong ones can name wrong rows but none outside the matrix.  Every wave of the workgroup works it out
// for itself: 64 groups at a time, one prefix sum over the lanes.
struct RowTile {
  int g;
  int64_t row0, rows;
};

__device__ __forceinline__ int64_t clamp64(int64_t v, int64_t lo, int64_t hi) { return v < lo ? lo : (v > hi ? hi : v); }

__device__ __forceinline__ RowTile find_row_tile(const int64_t* off, int G, int64_t T, int BM, int want, int rest) {
  const int lane = threadIdx.x & 63, total = rest ? G + 2 : G;
  for (int base = 0; base < total; base += 64) {
    const int g = base + lane;
    int64_t a = 0, b = 0;
    if (g < G) {
      a = clamp64(off[g], 0, T);
      b = clamp64(off[g + 1], a, T);
    } else if (g == G && rest) {
      b = G > 0 ? clamp64(off[0], 0, T) : T;
    } else if (g == G + 1 && rest && G > 0) {
      a = clamp64(off[G], 0, T);
      b = T;
    }
    const int tiles = (int)((b - a + BM - 1) / BM);
    int sum = tiles;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int v = __shfl_up(sum, d);
      if (lane >= d) sum += v;
    }
    const unsigned long long past = __ballot(sum > want);
    if (past) {
      const int at = __ffsll(past) - 1;
      const int64_t row0 = a + (int64_t)(want - (sum - tiles)) * BM;
      RowTile t;
      t.g = __builtin_amdgcn_readfirstlane(base + at);
      t.row0 = __shfl(row0, at);
      t.rows = __shfl(b - row0 < BM ? b - row0 : (int64_t)BM, at);
      return t;
    }
    want -= __shfl(sum, 63);
  }
  return RowTile{-1, 0, 0};
}

struct GroupedArgs {
  const void *x, *w;
  void* y;
  const int64_t* off;
  int64_t T, N, K, ldx, ldw, sw, ldy;
  int G, rest, tiles_n;
};

// Y[rows of g, :] = X[rows of g, :] W_g^T;  WK: W_g[n, k] = w[g sw + n ldw + k], else w[g sw + k ldw + n]
template <class T, int BM, int BN, bool WK, bool VEC>
__global__ __launch_bounds__(256, 2) void grouped_rows_kernel(GroupedArgs p) {
  using P = Tile<T, BM, BN, 2, 2, true, WK, VEC>;
  __shared__ __attribute__((aligned(16))) char lds[P::LDS_BYTES];
  const int tn = blockIdx.x % p.tiles_n, tm = blockIdx.x / p.tiles_n;
  const RowTile t = find_row_tile(p.off, p.G, p.T, BM, tm, p.rest);
  if (t.g < 0) return;
  const int64_t n0 = (int64_t)tn * BN;
  T* y = static_cast<T*>(p.y) + t.row0 * p.ldy + n0;
  P tile;
  const Operand<T> x{static_cast<const T*>(p.x) + t.row0 * p.ldx, p.ldx, t.rows};
  Operand<T> w{static_cast<const T*>(p.w), p.ldw, p.N - n0};
  if (t.g < p.G) w.p += t.g * p.sw + (WK ? n0 * p.ldw : n0);
  tile.run(x, w, t.g < p.G ? p.K : 0, lds);
  tile.each([&](int i, int j, int step, const typename P::acc_t& v) {
    if (i < t.rows) store_row(y + i * p.ldy, j, step, v, p.N - n0);
  });
}

// dW_g[n, k] = sum over the rows t of g of dY[t, n] X[t, k]
template <class T, int BM, int BN, bool VEC>
__global__ __launch_bounds__(256, 2) void grouped_dw_kernel(GroupedArgs p) {
  using P = Tile<T, BM, BN, 2, 2, false, false, VEC>;
  __shared__ __attribute__((aligned(16))) char lds[P::LDS_BYTES];
  const int tiles_k = (int)((p.K + BN - 1) / BN), tiles = p.tiles_n * tiles_k;
  const int g = blockIdx.x / tiles, i = blockIdx.x % tiles;
  const int64_t n0 = (int64_t)(i / tiles_k) * BM, k0 = (int64_t)(i % tiles_k) * BN;
  const int64_t a = clamp64(p.off[g], 0, p.T), b = clamp64(p.off[g + 1], a, p.T);
  P tile;
  const Operand<T> dy{static_cast<const T*>(p.y) + a * p.ldy + n0, p.ldy, p.N - n0};
  const Operand<T> x{static_cast<const T*>(p.x) + a * p.ldx + k0, p.ldx, p.K - k0};
  tile.run(dy, x, b - a, lds);
  T* dw = static_cast<T*>(const_cast<void*>(p.w)) + g * p.sw + n0 * p.ldw + k0;
  tile.each([&](int r, int j, int step, const typename P::acc_t& v) {
    if (r < p.N - n0) store_row(dw + r * p.ldw, j, step, v, p.K - k0);
  });
}

int size_of(int dtype) {
  switch (dtype) {
    case BGP_F64: return 8;
    case BGP_F32: return 4;
    case BGP_BF16:
    case BGP_F16: return 2;
  }
  return 0;
}

// whole 16-byte chunks: base, leading dimension and contiguous extent are multiples of 16 bytes
bool chunked(const void* p, int64_t ld, int64_t extent, int size) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && (ld * size) % 16 == 0 && (extent * size) % 16 == 0;
}

template <class T, int B, bool WK> int run_rows(const GroupedArgs& p0, bool vec, hipStream_t st) {
  GroupedArgs p = p0;
  p.tiles_n = (int)((p.N + B - 1) / B);
  const int64_t tiles = (p.T / B + p.G + (p.rest ? 2 : 0)) * p.tiles_n;
  if (tiles > MAX_WORKGROUPS) return bgp_products_fail(-1, "bgp_grouped_gemm: %lld tiles are more than one launch holds", (long long)tiles);
  return launch("bgp_grouped_gemm", vec ? grouped_rows_kernel<T, B, B, WK, true> : grouped_rows_kernel<T, B, B, WK, false>, dim3((unsigned)tiles),
                dim3(256), st, p);
}

template <class T> int rows_by_type(const GroupedArgs& p, bool trans, bool vec, hipStream_t st) {
  const bool small = p.T < (int64_t)p.G * 96;
  if (small) return trans ? run_rows<T, 64, false>(p, vec, st) : run_rows<T, 64, true>(p, vec, st);
  return trans ? run_rows<T, 128, false>(p, vec, st) : run_rows<T, 128, true>(p, vec, st);
}

template <class T> int dw_by_type(const GroupedArgs& p0, bool vec, hipStream_t st) {
  GroupedArgs p = p0;
  constexpr int B = 128;
  p.tiles_n = (int)((p.N + B - 1) / B);
  const int64_t tiles = (int64_t)p.G * p.tiles_n * ((p.K + B - 1) / B);
  if (tiles > MAX_WORKGROUPS) return bgp_products_fail(-1, "bgp_grouped_gemm_dw: %lld tiles are more than one launch holds", (long long)tiles);
  return launch("bgp_grouped_gemm_dw", vec ? grouped_dw_kernel<T, B, B, true> : grouped_dw_kernel<T, B, B, false>, dim3((unsigned)tiles), dim3(256), st, p);
}

int check_sizes(const char* what, int dtype, int64_t T, int64_t N, int64_t K, int64_t G, const void* off) {
  if (!size_of(dtype)) return bgp_products_fail(-1, "%s: unknown type %d", what, dtype);
  if (T < 0 || N < 0 || K < 0 || G < 0 || G > BGP_MAX_GROUPS)
    return bgp_products_fail(-1, "%s: bad sizes T=%lld N=%lld K=%lld G=%lld", what, (long long)T, (long long)N, (long long)K, (long long)G);
  if (G > 0 && !off) return bgp_products_fail(-1, "%s: no offsets", what);
  return 0;
}

}  // namespace

extern "C" int bgp_grouped_gemm(int device, void* stream, int dtype, int64_t T, int64_t N, int64_t K, int64_t G, const void* X, int64_t ldx, const void* W,
                                int64_t strideW, int64_t ldw, int w_trans, const int64_t* offsets, void* Y, int64_t ldy, int zero_rest) {
  const char* what = "bgp_grouped_gemm";
  if (int rc = check_sizes(what, dtype, T, N, K, G, offsets)) return rc;
  if (T == 0 || N == 0 || (G == 0 && !zero_rest)) return 0;
  if (!Y || (K > 0 && G > 0 && (!X || !W))) return bgp_products_fail(-1, "%s: null pointer", what);
  if (ldx < K || ldy < N || ldw < (w_trans ? N : K) || strideW < 0)
    return bgp_products_fail(-1, "%s: bad strides ldx=%lld ldw=%lld strideW=%lld ldy=%lld", what, (long long)ldx, (long long)ldw, (long long)strideW, (long long)ldy);
  DeviceScope scope(device);
  if (int rc = scope.check(what)) return rc;
  GroupedArgs p{X, W, Y, offsets, T, N, K, ldx, ldw, strideW, ldy, (int)G, zero_rest != 0, 0};
  const int size = size_of(dtype);
  const bool vec = chunked(X, ldx, K, size) && chunked(W, ldw, w_trans ? N : K, size) && (strideW * size) % 16 == 0;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case BGP_F64: return rows_by_type<double>(p, w_trans, vec, st);
    case BGP_F32: return rows_by_type<float>(p, w_trans, vec, st);
    case BGP_BF16: return rows_by_type<bf16_t>(p, w_trans, vec, st);
    default: return rows_by_type<f16_t>(p, w_trans, vec, st);
  }
}

extern "C" int bgp_grouped_gemm_dw(int device, void* stream, int dtype, int64_t T, int64_t N, int64_t K, int64_t G, const void* dY, int64_t lddy,
                                   const void* X, int64_t ldx, const int64_t* offsets, void* dW, int64_t strideW, int64_t ldw) {
  const char* what = "bgp_grouped_gemm_dw";
  if (int rc = check_sizes(what, dtype, T, N, K, G, offsets)) return rc;
  if (N == 0 || K == 0 || G == 0) return 0;
  if (!dW || (T > 0 && (!dY || !X))) return bgp_products_fail(-1, "%s: null pointer", what);
  if (lddy < N || ldx < K || ldw < K || strideW < N * ldw)
    return bgp_products_fail(-1, "%s: bad strides lddy=%lld ldx=%lld ldw=%lld strideW=%lld", what, (long long)lddy, (long long)ldx, (long long)ldw, (long long)strideW);
  DeviceScope scope(device);
  if (int rc = scope.check(what)) return rc;
  GroupedArgs p{X, dW, const_cast<void*>(dY), offsets, T, N, K, ldx, ldw, strideW, lddy, (int)G, 0, 0};
  const int size = size_of(dtype);
  const bool vec = chunked(dY, lddy, N, size) && chunked(X, ldx, K, size);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case BGP_F64: return dw_by_type<double>(p, vec, st);
    case BGP_F32: return dw_by_type<float>(p, vec, st);
    case BGP_BF16: return dw_by_type<bf16_t>(p, vec, st);
    default: return dw_by_type<f16_t>(p, vec, st);
  }
}
