// The tile product that the kernels of libbattgp_products.so share (gfx950 only).
//
// One workgroup forms D[i, j] = sum_k X(i, k) W(j, k) for BM rows i and BN rows j.  Both operands go through LDS in
// stages of 128 bytes of k (16 fp64, 32 fp32, 64 bf16 / fp16, 128 int8).  An operand is stored either with k contiguous
// ("along k") or with its row index contiguous ("along rows"); the LDS tile keeps the order of the memory, so that every
// global load and LDS store is a whole 16-byte chunk, and what transposing there is happens in the LDS read:
//   along k     a fragment is one ds_read_b128: lane (r, q) = (lane % 16, lane / 16) holds row r, 16-byte chunk 4 s + q
//               of the stage's half s.  For fp32 / fp64 a chunk feeds 4 / 2 matrix instructions that each take one
//               element per lane: the order of k inside a half is permuted, for both operands alike.
//   along rows  the same elements, gathered: fp64 / fp32 element by element, 16-bit types by two transposing reads
//               (ds_read_b64_tr_b16), which hand lane r column r of a 4 x 16 block of k x rows.
// Chunks are XOR-swizzled inside their LDS row so that the lanes that read together hit different banks.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

typedef double v4d __attribute__((ext_vector_type(4)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef int v4i __attribute__((ext_vector_type(4)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));

struct bf16_t { uint16_t v; };
struct f16_t { uint16_t v; };

#define BGP_LDS __attribute__((address_space(3)))

// a 16-byte chunk at the alignment of one element (gfx950 loads it in one instruction at any byte address)
template <int A>
struct __attribute__((packed, aligned(A))) Chunk { uint32_t a, b, c, d; };

template <class T> struct Num;
template <> struct Num<double> {
  using acc = v4d;
  static __device__ __forceinline__ acc mma(const uint4& a, const uint4& b, acc c) {
    double x[2], y[2];
    __builtin_memcpy(x, &a, 16);
    __builtin_memcpy(y, &b, 16);
    c = __builtin_amdgcn_mfma_f64_16x16x4f64(x[0], y[0], c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f64_16x16x4f64(x[1], y[1], c, 0, 0, 0);
  }
};
template <> struct Num<float> {
  using acc = v4f;
  static __device__ __forceinline__ acc mma(const uint4& a, const uint4& b, acc c) {
    float x[4], y[4];
    __builtin_memcpy(x, &a, 16);
    __builtin_memcpy(y, &b, 16);
#pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[j], y[j], c, 0, 0, 0);
    return c;
  }
};
template <> struct Num<bf16_t> {
  using acc = v4f;
  static __device__ __forceinline__ acc mma(const uint4& a, const uint4& b, acc c) {
    v8bf x, y;
    __builtin_memcpy(&x, &a, 16);
    __builtin_memcpy(&y, &b, 16);
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, y, c, 0, 0, 0);
  }
};
template <> struct Num<f16_t> {
  using acc = v4f;
  static __device__ __forceinline__ acc mma(const uint4& a, const uint4& b, acc c) {
    v8h x, y;
    __builtin_memcpy(&x, &a, 16);
    __builtin_memcpy(&y, &b, 16);
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(x, y, c, 0, 0, 0);
  }
};
template <> struct Num<int8_t> {
  using acc = v4i;
  static __device__ __forceinline__ acc mma(const uint4& a, const uint4& b, acc c) {
    v4i x, y;
    __builtin_memcpy(&x, &a, 16);
    __builtin_memcpy(&y, &b, 16);
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(x, y, c, 0, 0, 0);
  }
};

// one rounding to the nearest, ties to even, of what was summed in 32 (64) bits
template <class T, class A> __device__ __forceinline__ T round_to(A v);
template <> __device__ __forceinline__ double round_to<double, double>(double v) { return v; }
template <> __device__ __forceinline__ float round_to<float, float>(float v) { return v; }
template <> __device__ __forceinline__ bf16_t round_to<bf16_t, float>(float v) {
  const __bf16 b = (__bf16)v;
  bf16_t r;
  __builtin_memcpy(&r, &b, 2);
  return r;
}
template <> __device__ __forceinline__ f16_t round_to<f16_t, float>(float v) {
  const _Float16 b = (_Float16)v;
  f16_t r;
  __builtin_memcpy(&r, &b, 2);
  return r;
}

// element (r, k) = p[r ld + k] (along k) or p[k ld + r] (along rows); rows: how many from p on may be read
template <class T> struct Operand {
  const T* p;
  int64_t ld;
  int64_t rows;
};

template <class T> constexpr int CHE = 16 / (int)sizeof(T);        // elements in a chunk
template <class T> constexpr int KSTAGE = 128 / (int)sizeof(T);    // k per stage

// logical chunk <-> place inside an LDS row of `cpr` chunks (an involution)
template <class T, bool ALONG_K> __device__ __forceinline__ int swizzle(int row, int chunk, int cpr) {
  if (ALONG_K) return chunk ^ (row & 7);                                              // 8 chunks a row
  if (sizeof(T) == 2) return chunk ^ (((row & 3) << 1) & (cpr - 1));                  // 4 k-rows of a transposing read
  if (sizeof(T) == 4) return chunk ^ ((((row >> 2) & 1) << 2) & (cpr - 1));           // k-rows 4 q + j of the 4 lane groups
  return chunk;
}

// up to CHE elements (n of them exist, the others are 0)
template <class T, bool VEC> __device__ __forceinline__ uint4 load_chunk(const T* p, int64_t n) {
  uint4 v = make_uint4(0, 0, 0, 0);
  if (n >= CHE<T>) {
    if (VEC) return *reinterpret_cast<const uint4*>(p);
    const Chunk<sizeof(T)> c = *reinterpret_cast<const Chunk<sizeof(T)>*>(p);
    return make_uint4(c.a, c.b, c.c, c.d);
  }
  if (n > 0) {
    T e[CHE<T>] = {};
#pragma unroll
    for (int j = 0; j < CHE<T>; ++j)
      if (j < n) e[j] = p[j];
    __builtin_memcpy(&v, e, 16);
  }
  return v;
}

// one operand's share of a stage: ROWS x 128 bytes, fetched into registers by all NT threads, then stored to LDS
template <class T, int ROWS, bool ALONG_K, bool VEC, int NT> struct Stage {
  static constexpr int CHUNKS = ROWS * 8, NL = CHUNKS / NT;
  static constexpr int CPR = ALONG_K ? 8 : ROWS / CHE<T>;  // chunks per LDS row
  static_assert(CHUNKS % NT == 0, "every thread loads the same number of chunks");
  uint4 r[NL];

  __device__ __forceinline__ void fetch(const Operand<T>& o, int64_t k0, int64_t klen) {
#pragma unroll
    for (int l = 0; l < NL; ++l) {
      const int i = threadIdx.x + l * NT, row = i / CPR, c = swizzle<T, ALONG_K>(row, i % CPR, CPR);
      if (ALONG_K) {
        const int64_t k = k0 + c * CHE<T>;
        r[l] = load_chunk<T, VEC>(o.p + row * o.ld + k, row < o.rows ? klen - k : 0);
      } else {
        const int64_t k = k0 + row;
        r[l] = load_chunk<T, VEC>(o.p + k * o.ld + c * CHE<T>, k < klen ? o.rows - c * CHE<T> : 0);
      }
    }
  }
  __device__ __forceinline__ void store(char* lds) const {
#pragma unroll
    for (int l = 0; l < NL; ++l) *reinterpret_cast<uint4*>(lds + (threadIdx.x + l * NT) * 16) = r[l];
  }
};

// the 16 bytes of row r0 + lane % 16 that lane / 16 holds of half s of a stage
template <class T, int ROWS, bool ALONG_K> __device__ __forceinline__ uint4 fragment(const char* lds, int r0, int s) {
  const int lane = threadIdx.x & 63, q = s * 4 + (lane >> 4), r = lane & 15;
  uint4 v;
  if constexpr (ALONG_K) {
    v = *reinterpret_cast<const uint4*>(lds + (r0 + r) * 128 + swizzle<T, true>(r0 + r, q, 8) * 16);
  } else {
    constexpr int CPR = ROWS / CHE<T>, LROW = CPR * 16;
    if constexpr (sizeof(T) == 2) {
      v4s h[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int k = q * 8 + j * 4 + (r >> 2), col = r0 + (r & 3) * 4;  // this lane's 4 elements of the 4 x 16 block
        const char* a = lds + k * LROW + swizzle<T, false>(k, col / 8, CPR) * 16 + (col % 8) * 2;
        h[j] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((BGP_LDS v4s*)a);
      }
      __builtin_memcpy(&v, h, 16);
    } else {
      T e[CHE<T>];
#pragma unroll
      for (int j = 0; j < CHE<T>; ++j) {
        const int k = q * CHE<T> + j, col = r0 + r;
        e[j] = *reinterpret_cast<const T*>(lds + k * LROW + swizzle<T, false>(k, col / CHE<T>, CPR) * 16 + (col % CHE<T>) * (int)sizeof(T));
      }
      __builtin_memcpy(&v, e, 16);
    }
  }
  return v;
}

// The workgroup's tile: WX x WW waves, each (BM / WX) x (BN / WW).  acc[b][a] is the 16 x 16 block of X rows 16 a and
// W rows 16 b of the wave's part.
template <class T, int BM, int BN, int WX, int WW, bool XK, bool WK, bool VEC> struct Tile {
  static constexpr int NT = 64 * WX * WW, FA = BM / WX / 16, FB = BN / WW / 16;
  static constexpr int LDS_BYTES = 2 * (BM + BN) * 128;
  using acc_t = typename Num<T>::acc;
  acc_t acc[FB][FA];

  __device__ __forceinline__ int x0() const { return (int)(threadIdx.x >> 6) / WW * (BM / WX); }
  __device__ __forceinline__ int w0() const { return (int)(threadIdx.x >> 6) % WW * (BN / WW); }

  __device__ __forceinline__ void run(const Operand<T>& x, const Operand<T>& w, int64_t klen, char* lds) {
#pragma unroll
    for (int b = 0; b < FB; ++b)
#pragma unroll
      for (int a = 0; a < FA; ++a) acc[b][a] = acc_t{};
    if (klen <= 0) return;
    Stage<T, BM, XK, VEC, NT> sx;
    Stage<T, BN, WK, VEC, NT> sw;
    sx.fetch(x, 0, klen);
    sw.fetch(w, 0, klen);
    sx.store(lds);
    sw.store(lds + BM * 128);
    __syncthreads();
    int buf = 0;
    for (int64_t k0 = 0; k0 < klen; k0 += KSTAGE<T>) {
      const bool more = k0 + KSTAGE<T> < klen;
      if (more) {
        sx.fetch(x, k0 + KSTAGE<T>, klen);
        sw.fetch(w, k0 + KSTAGE<T>, klen);
      }
      const char *lx = lds + buf * (BM + BN) * 128, *lw = lx + BM * 128;
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        uint4 fx[FA], fw[FB];
#pragma unroll
        for (int a = 0; a < FA; ++a) fx[a] = fragment<T, BM, XK>(lx, x0() + a * 16, s);
#pragma unroll
        for (int b = 0; b < FB; ++b) fw[b] = fragment<T, BN, WK>(lw, w0() + b * 16, s);
#pragma unroll
        for (int b = 0; b < FB; ++b)
#pragma unroll
          for (int a = 0; a < FA; ++a) acc[b][a] = Num<T>::mma(fw[b], fx[a], acc[b][a]);
      }
      buf ^= 1;
      if (more) {
        sx.store(lds + buf * (BM + BN) * 128);
        sw.store(lds + buf * (BM + BN) * 128 + BM * 128);
      }
      __syncthreads();
    }
  }

  // f(i, j, values, first, step): X row i, W rows j + first + step * e for e < 4
  template <class F> __device__ __forceinline__ void each(F&& f) const {
    const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
#pragma unroll
    for (int a = 0; a < FA; ++a)
#pragma unroll
      for (int b = 0; b < FB; ++b) {
        if (sizeof(T) == 8) f(x0() + a * 16 + r, w0() + b * 16 + q, 4, acc[b][a]);
        else f(x0() + a * 16 + r, w0() + b * 16 + q * 4, 1, acc[b][a]);
      }
  }
};

// D[j .. j + 3 step] = values where they are inside n columns
template <class T, class A> __device__ __forceinline__ void store_row(T* row, int64_t j, int step, const A& v, int64_t n) {
  if (sizeof(T) <= 4 && step == 1 && j + 3 < n && (reinterpret_cast<uintptr_t>(row + j) % (4 * sizeof(T))) == 0) {
    struct alignas(4 * sizeof(T)) Four { T e[4]; } o;
#pragma unroll
    for (int e = 0; e < 4; ++e) o.e[e] = round_to<T>(v[e]);
    *reinterpret_cast<Four*>(row + j) = o;
    return;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (j + e * step < n) row[j + e * step] = round_to<T>(v[e]);
}
