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

#include <type_traits>

typedef double v2d __attribute__((ext_vector_type(2)));
typedef double v4d __attribute__((ext_vector_type(4)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef int v4i __attribute__((ext_vector_type(4)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));

typedef uint32_t chunk_t __attribute__((ext_vector_type(4)));  // 16 bytes, what every load and LDS access moves
__device__ __forceinline__ chunk_t chunk_of(uint32_t a, uint32_t b, uint32_t c, uint32_t d) { return chunk_t{a, b, c, d}; }

struct bf16_t { uint16_t v; };
struct f16_t { uint16_t v; };

#define BGP_LDS __attribute__((address_space(3)))

// a 16-byte chunk at the alignment of one element (gfx950 loads it in one instruction at any byte address)
template <int A>
struct __attribute__((packed, aligned(A))) Chunk { uint32_t a, b, c, d; };

template <class T> struct Num;
template <> struct Num<double> {
  using acc = v4d;
  static __device__ __forceinline__ acc mma(const chunk_t& a, const chunk_t& b, acc c) {
    const v2d x = __builtin_bit_cast(v2d, a), y = __builtin_bit_cast(v2d, b);
    c = __builtin_amdgcn_mfma_f64_16x16x4f64(x[0], y[0], c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f64_16x16x4f64(x[1], y[1], c, 0, 0, 0);
  }
};
template <> struct Num<float> {
  using acc = v4f;
  static __device__ __forceinline__ acc mma(const chunk_t& a, const chunk_t& b, acc c) {
    const v4f x = __builtin_bit_cast(v4f, a), y = __builtin_bit_cast(v4f, b);
#pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[j], y[j], c, 0, 0, 0);
    return c;
  }
};
template <> struct Num<bf16_t> {
  using acc = v4f;
  static __device__ __forceinline__ acc mma(const chunk_t& a, const chunk_t& b, acc c) {
    const v8bf x = __builtin_bit_cast(v8bf, a), y = __builtin_bit_cast(v8bf, b);
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, y, c, 0, 0, 0);
  }
};
template <> struct Num<f16_t> {
  using acc = v4f;
  static __device__ __forceinline__ acc mma(const chunk_t& a, const chunk_t& b, acc c) {
    const v8h x = __builtin_bit_cast(v8h, a), y = __builtin_bit_cast(v8h, b);
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(x, y, c, 0, 0, 0);
  }
};
template <> struct Num<int8_t> {
  using acc = v4i;
  static __device__ __forceinline__ acc mma(const chunk_t& a, const chunk_t& b, acc c) {
    const v4i x = __builtin_bit_cast(v4i, a), y = __builtin_bit_cast(v4i, b);
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(x, y, c, 0, 0, 0);
  }
};

// what sums of a type are held in
template <class T> struct Sum { using type = float; };
template <> struct Sum<double> { using type = double; };

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

// element (r, k) = p[r ld + k] (along k) or p[k ld + r] (along rows); rows: how many from p on may be read; wide: the
// matrix's rows (in memory) are 16 bytes long at least
template <class T> struct Operand {
  const T* p;
  int64_t ld;
  int64_t rows;
  bool wide;
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

// A chunk at any alignment, as it is loaded and as it is used.  Loads of 16 bytes are as fast at any multiple of 4 but take
// up to three times as long off it, which a tile straight from memory waits for (a product of 707 x 144 x 6467 8-bit
// integers: 35 us, of 6464: 12).  ODD: such a chunk is loaded from the word that its first element lies in, with
// the word behind, and moved down when it is used (21 us; but 23 for the 6464).  Words that hold no element of it are
// not touched.
template <class T, bool ODD = false> struct Piece {
  chunk_t c;
  static __device__ __forceinline__ Piece load(const T* p) {
    const Chunk<sizeof(T)> c = *reinterpret_cast<const Chunk<sizeof(T)>*>(p);
    return Piece{chunk_of(c.a, c.b, c.c, c.d)};
  }
  __device__ __forceinline__ chunk_t value() const { return c; }
};
template <class T> struct Piece<T, true> {
  chunk_t c;
  uint32_t next, off;
  static __device__ __forceinline__ Piece load(const T* p) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(p);
    const uint32_t off = (uint32_t)at & 3;
    const char* word = reinterpret_cast<const char*>(at - off);
    const Chunk<4> c = *reinterpret_cast<const Chunk<4>*>(word);
    return Piece{chunk_of(c.a, c.b, c.c, c.d), *reinterpret_cast<const uint32_t*>(word + (off ? 16 : 12)), off};
  }
  __device__ __forceinline__ chunk_t value() const {
    return chunk_of(__builtin_amdgcn_alignbyte(c.y, c.x, off), __builtin_amdgcn_alignbyte(c.z, c.y, off), __builtin_amdgcn_alignbyte(c.w, c.z, off),
                    __builtin_amdgcn_alignbyte(next, c.w, off));
  }
};
template <class T> __device__ __forceinline__ chunk_t load_any(const T* p) { return Piece<T>::load(p).value(); }

// the first n elements of a chunk, then zeros, one by one
template <class T> __device__ __forceinline__ chunk_t load_few(const T* p, int64_t n) {
  T e[CHE<T>] = {};
#pragma unroll
  for (int j = 0; j < CHE<T>; ++j)
    if (j < n) e[j] = p[j];
  chunk_t v;
  __builtin_memcpy(&v, e, 16);
  return v;
}

// The same without a branch, where the chunk that ends at p + n (0 < n < CHE) lies in the same row: it is loaded whole, and
// later (`settle`: not before it is needed, so that many loads are in flight) moved down.  n <= 0: zeros, and `home`
// is read instead.
template <class T> __device__ __forceinline__ int kept(int64_t n) { return n >= CHE<T> ? CHE<T> : n > 0 ? (int)n : 0; }
template <class T, bool ODD = false> __device__ __forceinline__ Piece<T, ODD> load_edge(const T* p, int64_t n, const T* home) {
  const int keep = kept<T>(n);
  return Piece<T, ODD>::load(keep ? p - (CHE<T> - keep) : home);
}
template <class T, bool ODD> __device__ __forceinline__ chunk_t settle(const Piece<T, ODD>& piece, int64_t n) {
  const int keep = kept<T>(n);
  const chunk_t c = piece.value();
  uint64_t lo = (uint64_t)c.y << 32 | c.x, hi = (uint64_t)c.w << 32 | c.z;
  int bits = (CHE<T> - keep) * 8 * (int)sizeof(T);
  if (bits >= 64) {
    lo = hi;
    hi = 0;
    bits -= 64;
  }
  lo = lo >> (bits & 63) | hi << 1 << (63 - (bits & 63));
  hi >>= bits & 63;
  if (!keep) lo = hi = 0;
  return chunk_of((uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32));
}

// a value that all lanes hold, in scalar registers
__device__ __forceinline__ int64_t scalar64(int64_t v) {
  const uint32_t lo = __builtin_amdgcn_readfirstlane((int)v), hi = __builtin_amdgcn_readfirstlane((int)(v >> 32));
  return (int64_t)((uint64_t)hi << 32 | lo);
}

// one operand's share of a stage: ROWS x 128 bytes, fetched into registers by all NT threads, then stored to LDS
template <class T, int ROWS, bool ALONG_K, int NT> struct Stage {
  static constexpr int CHUNKS = ROWS * 8, NL = CHUNKS / NT;
  static constexpr int CPR = ALONG_K ? 8 : ROWS / CHE<T>;  // chunks per LDS row
  static_assert(CHUNKS % NT == 0, "every thread loads the same number of chunks");
  Piece<T> r[NL];

  // A stage of which all k exist.  EDGE: not all rows do; along k the last one is repeated (it only reaches elements of D
  // that are not stored), along rows what does not exist is 0.
  template <bool EDGE> __device__ __forceinline__ void fetch(const Operand<T>& o, int64_t k0) {
    if (EDGE && !o.wide) return;
    const int last = EDGE && o.rows < ROWS ? (int)o.rows - 1 : ROWS - 1;
#pragma unroll
    for (int l = 0; l < NL; ++l) {
      const int i = threadIdx.x + l * NT, row = i / CPR, c = swizzle<T, ALONG_K>(row, i % CPR, CPR);
      if (ALONG_K) {
        r[l] = Piece<T>::load(o.p + (EDGE && row > last ? last : row) * o.ld + k0 + c * CHE<T>);
      } else {
        const T* p = o.p + (k0 + row) * o.ld + c * CHE<T>;
        r[l] = EDGE ? load_edge(p, o.rows - c * CHE<T>, o.rows >= CHE<T> ? o.p : o.p + o.rows - CHE<T>) : Piece<T>::load(p);
      }
    }
  }
  template <bool EDGE> __device__ __forceinline__ void store(char* lds, const Operand<T>& o, int64_t k0) const {
    if (EDGE && !o.wide) {
      store_narrow(lds, o, k0, k0 + KSTAGE<T>);
      return;
    }
#pragma unroll
    for (int l = 0; l < NL; ++l) {
      const int i = threadIdx.x + l * NT, row = i / CPR, c = swizzle<T, ALONG_K>(row, i % CPR, CPR);
      *reinterpret_cast<chunk_t*>(lds + i * 16) = EDGE && !ALONG_K ? settle(r[l], o.rows - c * CHE<T>) : r[l].value();
    }
  }

  // the stage in which k ends
  __device__ __forceinline__ void fetch_store_end(char* lds, const Operand<T>& o, int64_t k0, int64_t klen) {
    if (!o.wide) {
      store_narrow(lds, o, k0, klen);
      return;
    }
    const int last = o.rows < ROWS ? (int)o.rows - 1 : ROWS - 1;
    const T* home = ALONG_K || o.rows >= CHE<T> ? o.p : o.p + o.rows - CHE<T>;
    if (ALONG_K && klen < CHE<T>) home -= CHE<T> - klen;  // a part of k that is not the first
    auto exist = [&](int row, int c) { return ALONG_K ? klen - k0 - c * CHE<T> : k0 + row < klen ? o.rows - c * CHE<T> : 0; };
#pragma unroll
    for (int l = 0; l < NL; ++l) {
      const int i = threadIdx.x + l * NT, row = i / CPR, c = swizzle<T, ALONG_K>(row, i % CPR, CPR);
      r[l] = load_edge(ALONG_K ? o.p + (row < last ? row : last) * o.ld + k0 + c * CHE<T> : o.p + (k0 + row) * o.ld + c * CHE<T>, exist(row, c), home);
    }
#pragma unroll
    for (int l = 0; l < NL; ++l) {
      const int i = threadIdx.x + l * NT, row = i / CPR, c = swizzle<T, ALONG_K>(row, i % CPR, CPR);
      *reinterpret_cast<chunk_t*>(lds + i * 16) = settle(r[l], exist(row, c));
    }
  }

  // rows of less than 16 bytes, element by element
  static __device__ __forceinline__ void store_narrow(char* lds, const Operand<T>& o, int64_t k0, int64_t klen) {
#pragma unroll 1
    for (int i = threadIdx.x; i < CHUNKS; i += NT) {
      const int row = i / CPR, c = swizzle<T, ALONG_K>(row, i % CPR, CPR);
      const int64_t n = ALONG_K ? (row < o.rows ? klen - k0 - c * CHE<T> : 0) : (k0 + row < klen ? o.rows - c * CHE<T> : 0);
      *reinterpret_cast<chunk_t*>(lds + i * 16) = load_few(ALONG_K ? o.p + row * o.ld + k0 + c * CHE<T> : o.p + (k0 + row) * o.ld + c * CHE<T>, n);
    }
  }
};

// the 16 bytes of row r0 + lane % 16 that lane / 16 holds of half s of a stage
template <class T, int ROWS, bool ALONG_K> __device__ __forceinline__ chunk_t fragment(const char* lds, int r0, int s) {
  const int lane = threadIdx.x & 63, q = s * 4 + (lane >> 4), r = lane & 15;
  chunk_t v;
  if constexpr (ALONG_K) {
    v = *reinterpret_cast<const chunk_t*>(lds + (r0 + r) * 128 + swizzle<T, true>(r0 + r, q, 8) * 16);
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

// Hands the wave's part of D out in units of E neighbours of a row, through LDS: a matrix instruction leaves 4 neighbours in
// a lane, whose stores would touch 16 rows at 8 to 32 bytes each.  f(i, j, sums): X row i, W rows j .. j + E - 1; only
// i < rows.  Each wave has a region of LDS to itself, whose operations happen in order: no barrier.  Rows are
// handed out in a loop of few instructions: unrolled over the accumulators the same work was bound by fetching
// its code (8192 x 2048 bf16 results: 13 us instead of 4).
template <class T, int C, int E, int REGION, int FA, int FB, class ACC, class F>
__device__ __forceinline__ void hand_out(const ACC (&acc)[FB][FA], char* mine, int x0, int w0, int64_t rows, F&& f) {
  using S = typename std::remove_reference<decltype(acc[0][0][0] + acc[0][0][0])>::type;
  constexpr int LROW = C * (int)sizeof(S), FIT = REGION / LROW / 16;                       // 16-row blocks in the region
  constexpr int AT_ONCE = FIT >= FA ? FA : FIT >= 8 ? 8 : FIT >= 4 ? 4 : FIT >= 2 ? 2 : FIT;
  static_assert(AT_ONCE >= 1 && FA % AT_ONCE == 0, "a wave's region holds whole blocks");
  constexpr int UNITS = LROW / 16;  // 16-byte pieces of a row, swizzled by the row
  const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
  auto place = [&](int row, int col) {
    const int byte = col * (int)sizeof(S);
    return mine + row * LROW + (((byte >> 4) ^ row) & (UNITS - 1)) * 16 + (byte & 15);
  };
#pragma unroll
  for (int first = 0; first < FA; first += AT_ONCE) {
    if (x0 + first * 16 >= rows) return;
#pragma unroll
    for (int a = 0; a < AT_ONCE; ++a)
#pragma unroll
      for (int b = 0; b < FB; ++b) {
        if (sizeof(T) == 8) {
#pragma unroll
          for (int e = 0; e < 4; ++e) *reinterpret_cast<S*>(place(a * 16 + r, b * 16 + q + 4 * e)) = acc[b][first + a][e];
        } else {
          *reinterpret_cast<ACC*>(place(a * 16 + r, b * 16 + q * 4)) = acc[b][first + a];
        }
      }
    __builtin_amdgcn_wave_barrier();
    constexpr int PER_ROW = C / E, ALL = AT_ONCE * 16 * PER_ROW / 64;
    constexpr int AHEAD = std::remove_reference<F>::type::AHEAD < ALL ? std::remove_reference<F>::type::AHEAD : ALL;
    static_assert(ALL % AHEAD == 0, "whole rounds");
#pragma unroll 1
    for (int u0 = lane; u0 < 64 * ALL; u0 += 64 * AHEAD) {
      typename std::remove_reference<F>::type::Other other[AHEAD];  // what a unit takes from memory, before any is stored
#pragma unroll
      for (int n = 0; n < AHEAD; ++n) {
        const int u = u0 + 64 * n, i = x0 + first * 16 + u / PER_ROW;
        other[n] = f.other(i < rows ? i : (int)rows - 1, w0 + u % PER_ROW * E);
      }
#pragma unroll
      for (int n = 0; n < AHEAD; ++n) {
        const int u = u0 + 64 * n, row = u / PER_ROW, j = u % PER_ROW * E;
        S v[E];
        if constexpr (E * sizeof(S) < 16) {
          __builtin_memcpy(v, place(row, j), E * sizeof(S));
        } else {
#pragma unroll
          for (int c = 0; c < (int)(E * sizeof(S) / 16); ++c) {
            const chunk_t one = *reinterpret_cast<const chunk_t*>(place(row, j + c * 16 / (int)sizeof(S)));
            __builtin_memcpy(reinterpret_cast<char*>(v) + c * 16, &one, 16);
          }
        }
        const int i = x0 + first * 16 + row;
        if (i < rows) f(i, w0 + j, v, other[n]);
      }
    }
    __builtin_amdgcn_wave_barrier();
  }
}

// The workgroup's tile: WX x WW waves, each (BM / WX) x (BN / WW).  acc[b][a] is the 16 x 16 block of X rows 16 a and
// W rows 16 b of the wave's part.  For operands at any alignment: a stage waits in registers while the one before it is
// multiplied, and its 16-byte loads off the 4-byte words are what bounds it (3000 x 5000 x 300 8-bit integers to bf16: 25 us
// in tiles of 64); 7000 x 4096 x 2048 aligned numbers in bf16 take 138 us in tiles of 128, the pipeline below 111.
template <class T, int BM, int BN, int WX, int WW, bool XK, bool WK> struct Tile {
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
    if (x.rows >= BM && w.rows >= BN && x.wide && w.wide) loop<false>(x, w, klen, lds);
    else loop<true>(x, w, klen, lds);
  }

  // two buffers: while a stage is multiplied the next is fetched into registers.  If k ends inside a stage, that one
  // comes first.
  template <bool EDGE> __device__ __forceinline__ void loop(const Operand<T>& x, const Operand<T>& w, int64_t klen, char* lds) {
    constexpr int BUF = (BM + BN) * 128;
    Stage<T, BM, XK, NT> sx;
    Stage<T, BN, WK, NT> sw;
    const int whole = (int)(klen / KSTAGE<T>), stages = whole + (klen % KSTAGE<T> != 0);
    if (stages > whole) {
      sx.fetch_store_end(lds, x, (int64_t)whole * KSTAGE<T>, klen);
      sw.fetch_store_end(lds + BM * 128, w, (int64_t)whole * KSTAGE<T>, klen);
    } else {
      sx.template fetch<EDGE>(x, 0);
      sw.template fetch<EDGE>(w, 0);
      sx.template store<EDGE>(lds, x, 0);
      sw.template store<EDGE>(lds + BM * 128, w, 0);
    }
    int64_t k0 = stages > whole ? 0 : KSTAGE<T>;  // the next stage's
    __syncthreads();
    for (int s = 0; s < stages; ++s) {
      const char *lx = lds + (s & 1) * BUF, *lw = lx + BM * 128;
      char* next = lds + (~s & 1) * BUF;
      const bool more = s + 1 < stages;
      if (more) {
        sx.template fetch<EDGE>(x, k0);
        sw.template fetch<EDGE>(w, k0);
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        chunk_t fx[FA], fw[FB];
#pragma unroll
        for (int a = 0; a < FA; ++a) fx[a] = fragment<T, BM, XK>(lx, x0() + a * 16, h);
#pragma unroll
        for (int b = 0; b < FB; ++b) fw[b] = fragment<T, BN, WK>(lw, w0() + b * 16, h);
#pragma unroll
        for (int b = 0; b < FB; ++b)
#pragma unroll
          for (int a = 0; a < FA; ++a) acc[b][a] = Num<T>::mma(fw[b], fx[a], acc[b][a]);
      }
      if (more) {
        sx.template store<EDGE>(next, x, k0);
        sw.template store<EDGE>(next + BM * 128, w, k0);
        k0 += KSTAGE<T>;
      }
      __syncthreads();
    }
  }

  template <int E, class F> __device__ __forceinline__ void out(char* lds, int64_t rows, F&& f) const {
    constexpr int C = BN / WW, REGION = LDS_BYTES / (WX * WW);
    hand_out<T, C, E, REGION, FA, FB>(acc, lds + (threadIdx.x >> 6) * REGION, x0(), w0(), rows, f);
  }
};

// The same tile for operands whose rows start on 16 bytes and lie in whole chunks, as a pipeline: two buffers of a stage
// each, filled by loads that write LDS themselves (global_load_lds, 16 bytes a lane: no registers, no LDS stores, one 32-bit
// offset per lane and load against a scalar base) and issued a whole stage ahead; the fragments of the next half stage
// are read while the matrix instructions of this one run.
//   first half of stage b:   read the fragments of its second half; multiply those of the first.
//   second half:             wait until stage b + 1 has arrived and this wave's own fragment reads of stage b are done;
//                            barrier: both hold for every wave, so b's buffer is free; issue stage b + 2 into it; read
//                            the fragments of b + 1's first half; multiply those of b's second.
// A stage is 128 bytes of k, a whole cache line.  If k ends inside a stage, that last part comes first, through
// registers and filled up with zeros; all others are whole.  Rows (columns) past the operand's end repeat its last one:
// they only reach elements of D that are not stored.
// Bound by the matrix cores where there is much to do: 8192^3 in tiles of 256 takes 0.77 ms in bf16 (1430 TFLOP/s, the
// library's product 1477) and 0.42 ms in 8 bits (2590 TOP/s, the library's 2046); 8192 x 4096 x 2048 in fp64 1.89 ms (72.7 of 77
// TFLOP/s).  With few stages to a tile, by filling the pipeline and by the results of one round of tiles, which go to
// memory all at once: 18000 x 512 x 500 in fp64 runs at 60 TFLOP/s.  Workgroups of one CU at unlike wave priorities, to
// pull those apart, were no faster (159 us against 154).
// SETS = 2: two sets of waves halve k between them, each a pipeline of three buffers, and add up in LDS: for few tiles of
// long k, where a CU has one workgroup and one set of 4 waves waits for its loads, LDS reads and barriers in turn
// (1000 x 1024 x 4096 in bf16: 21 us against 32, and 27 with k cut over workgroups; where tiles fill the chip one set is
// faster, 700 rows of 2 groups, 4096 x 4096: 43 us against 61).  32- and 64-bit types have enough to multiply in a stage
// and gain nothing.
// Offsets inside a stage have 32 bits: pipe_fits() says whether an operand's do.
template <class T, int BM, int BN, int WX, int WW, bool XK, bool WK, int SETS = 1> struct PipeTile {
  static constexpr int NBUF = SETS == 1 ? 2 : 3;
  static constexpr int NW = WX * WW, NT = 64 * NW, FA = BM / WX / 16, FB = BN / WW / 16;
  static constexpr int KE = KSTAGE<T>;
  static constexpr int XL = BM / 8 / NW, WL = BN / 8 / NW;  // loads of a wave per stage
  static constexpr int BUF = (BM + BN) * 128, LDS_BYTES = SETS * NBUF * BUF, L = XL + WL;
  static_assert(BM / 8 % NW == 0 && BN / 8 % NW == 0, "every wave loads the same share of either operand");
  using acc_t = typename Num<T>::acc;
  acc_t acc[FB][FA];

  __device__ __forceinline__ int set() const { return SETS == 1 ? 0 : __builtin_amdgcn_readfirstlane((int)(threadIdx.x / NT)); }
  __device__ __forceinline__ int wave() const { return __builtin_amdgcn_readfirstlane((int)(SETS == 1 ? threadIdx.x >> 6 : threadIdx.x % NT >> 6)); }
  __device__ __forceinline__ int x0() const { return wave() / WW * (BM / WX); }
  __device__ __forceinline__ int w0() const { return wave() % WW * (BN / WW); }

  // a wave's loads of one operand: load l brings the 64 chunks from (wave + l NW) 64 on
  template <int ROWS, bool ALONG_K> struct Source {
    static constexpr int L = ROWS / 8 / NW;
    const char* p;  // the stage's first byte
    int64_t step;
    uint32_t at[L];
    __device__ __forceinline__ void start(const Operand<T>& o, int wave) {
      constexpr int CPR = ALONG_K ? 8 : ROWS / CHE<T>;
      p = reinterpret_cast<const char*>(scalar64(reinterpret_cast<int64_t>(o.p)));
      step = scalar64((ALONG_K ? (int64_t)KE : KE * o.ld) * (int)sizeof(T));
#pragma unroll
      for (int l = 0; l < L; ++l) {
        const int i = (wave + l * NW) * 64 + (int)(threadIdx.x & 63), row = i / CPR, c = swizzle<T, ALONG_K>(row, i % CPR, CPR);
        const int last = o.rows < ROWS ? (int)o.rows - 1 : ROWS - 1;
        if (ALONG_K) at[l] = (uint32_t)(row < last ? row : last) * (uint32_t)(o.ld * (int)sizeof(T)) + c * 16;
        else at[l] = (uint32_t)row * (uint32_t)(o.ld * (int)sizeof(T)) + (c < last / CHE<T> ? c : last / CHE<T>) * 16;
      }
    }
    // m0, where the load takes its LDS address from, is a reserved register: the compiler keeps nothing in it, and a clobber
    // list may not name it.  No other instruction of these kernels uses it (the static test of their assembly looks).
    __device__ __forceinline__ void issue(uint32_t lds) {
      const int64_t from = scalar64(reinterpret_cast<int64_t>(p));
#pragma unroll
      for (int l = 0; l < L; ++l)
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds + l * NW * 1024), "v"(at[l]), "s"(from) : "memory");
      p += step;
    }
  };

  __device__ __forceinline__ void run(const Operand<T>& x, const Operand<T>& w, int64_t k_length, char* lds) {
#pragma unroll
    for (int b = 0; b < FB; ++b)
#pragma unroll
      for (int a = 0; a < FA; ++a) acc[b][a] = acc_t{};
    const int64_t klen = scalar64(k_length);
    if (klen <= 0) return;
    const int64_t whole = klen / KE * KE;
    // every set's share of the stages, the part that k ends with counted as the first
    const int all = (int)(klen / KE) + (whole < klen), most = (all + SETS - 1) / SETS;
    const int before = set() * most, stages = all - before < most ? all - before : most;  // < 1: none
    const bool tail = whole < klen && set() == 0;
    char* mine = lds + set() * (NBUF * BUF);
    const uint32_t base = (uint32_t)(uintptr_t)(BGP_LDS char*)mine + wave() * 1024;
    Source<BM, XK> sx;
    Source<BN, WK> sw;
    sx.start(x, wave());
    sw.start(w, wave());
    if (set() > 0) {
      sx.p += (before - (whole < klen)) * sx.step;
      sw.p += (before - (whole < klen)) * sw.step;
    }
    auto issue = [&](int buf) {
      sx.issue(base + buf * BUF);
      sw.issue(base + buf * BUF + BM * 128);
    };
    if (tail) {
      Stage<T, BM, XK, NT> tx;
      Stage<T, BN, WK, NT> tw;
      tx.fetch_store_end(lds, x, whole, klen);
      tw.fetch_store_end(lds + BM * 128, w, whole, klen);
    } else if (SETS == 1 || stages > 0) {
      issue(0);
    }
#pragma unroll
    for (int i = 1; i < NBUF; ++i)
      if (i < stages) issue(i);
    // stage 0 is there for every wave
    if (stages >= NBUF && !tail) asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((NBUF - 1) * L) : "memory");
    else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    // stage s + 1 is, and this wave's reads of stage s are done
    auto arrive = [&](int s) {
      if (NBUF > 2 && s + NBUF <= stages) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((NBUF - 2) * L) : "memory");
      else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    };
    auto after = [](int buf) { return NBUF == 2 ? buf ^ 1 : buf + 1 == NBUF ? 0 : buf + 1; };
    chunk_t fx[2][FA], fw[2][FB];
    auto read = [&](int buf, int half) {
      const char* at = mine + buf * BUF;
#pragma unroll
      for (int a = 0; a < FA; ++a) fx[half][a] = fragment<T, BM, XK>(at, x0() + a * 16, half);
#pragma unroll
      for (int b = 0; b < FB; ++b) fw[half][b] = fragment<T, BN, WK>(at + BM * 128, w0() + b * 16, half);
    };
    auto multiply = [&](int half) {
#pragma unroll
      for (int b = 0; b < FB; ++b)
#pragma unroll
        for (int a = 0; a < FA; ++a) acc[b][a] = Num<T>::mma(fw[half][b], fx[half][a], acc[b][a]);
      interleave();
      __builtin_amdgcn_sched_barrier(0);
    };
    if (x0() >= x.rows || w0() >= w.rows) {  // none of this wave's elements exist: it only loads
      for (int s = 0, buf = 0; s < stages; ++s, buf = after(buf)) {
        arrive(s);
        if (s + NBUF < stages) issue(buf);
      }
      if constexpr (SETS == 1) {
        asm volatile("s_barrier" ::: "memory");
        return;
      }
    } else {
      if (SETS == 1 || stages > 0) read(0, 0);
      for (int s = 0, buf = 0; s < stages; ++s, buf = after(buf)) {
        __builtin_amdgcn_sched_barrier(0);
        read(buf, 1);
        multiply(0);
        arrive(s);
        if (s + NBUF < stages) issue(buf);
        __builtin_amdgcn_sched_barrier(0);
        read(after(buf), 0);  // behind the last stage: whatever is there, not used
        multiply(1);
      }
    }
    if (SETS > 1)
      for (int s = stages > 0 ? stages : 0; s < most; ++s) asm volatile("s_barrier" ::: "memory");
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (SETS > 1) add_sets(lds + LDS_BYTES / 2);
  }

  // the other sets' sums to the first's; `lds`: half of it, whose other half is free for `out`
  __device__ __forceinline__ void add_sets(char* lds) {
    static_assert(SETS == 1 || (SETS - 1) * NT * FA * FB * (int)sizeof(acc_t) <= LDS_BYTES / 2, "the sets' sums fit");
    acc_t* at = reinterpret_cast<acc_t*>(lds) + (threadIdx.x & (NT - 1));
#pragma unroll
    for (int b = 0; b < FB; ++b)
#pragma unroll
      for (int a = 0; a < FA; ++a)
        if (set() > 0) at[(((set() - 1) * FB + b) * FA + a) * NT] = acc[b][a];
    __syncthreads();
    if (set() == 0)
#pragma unroll
      for (int o = 0; o < SETS - 1; ++o)
#pragma unroll
        for (int b = 0; b < FB; ++b)
#pragma unroll
          for (int a = 0; a < FA; ++a) acc[b][a] += at[((o * FB + b) * FA + a) * NT];
  }

  // the order the scheduler is to give an iteration: the LDS reads spread evenly over the matrix instructions
  static constexpr int reads_of(bool along_k) { return along_k ? 1 : sizeof(T) == 2 ? 2 : CHE<T>; }
  __device__ __forceinline__ void interleave() const {
    constexpr int R = FA * reads_of(XK) + FB * reads_of(WK), M = FA * FB * (sizeof(T) == 8 ? 2 : sizeof(T) == 4 ? 4 : 1);
    constexpr int EACH = M / R > 0 ? M / R : 1;
#pragma unroll
    for (int i = 0; i < (R < M ? R : M); ++i) {
      __builtin_amdgcn_sched_group_barrier(0x100, R > M ? (R + M - 1) / M : 1, 0);  // LDS reads
      __builtin_amdgcn_sched_group_barrier(0x008, EACH, 0);                         // matrix instructions
    }
  }

  template <int E, class F> __device__ __forceinline__ void out(char* lds, int64_t rows, F&& f) const {
    constexpr int C = BN / WW, REGION = LDS_BYTES / (SETS > 1 ? 2 * NW : NW);
    if (set() == 0) hand_out<T, C, E, REGION, FA, FB>(acc, lds + wave() * REGION, x0(), w0(), rows, f);
  }
};

// The tile for small problems, where a wait for every stage costs more than what is multiplied: 16 FA x 16 FB elements of D
// by 4 waves that split k between them (8 were no faster) and add up in LDS at the end.  Fragments come straight from
// memory, several in flight, without a barrier; operands of any alignment (ODD: not of 4 bytes).  Along rows the elements
// are gathered one by one, which suits 32- and 64-bit types (16 lanes read 64 or 128 consecutive bytes).
// Bound by the launch and one or two waits for memory (8 single rows of 64 groups, 2048 x 1024 weights in bf16: 11.9 us for
// 34 MB; one row of 8-bit integers, 4096 x 4096: 6 us for 17 MB), by the loads' issue where rows are many (4096 x 2048 x 1024 in
// bf16: 128 us, and the model takes the pipeline at 30).
template <class T, int FA, int FB, bool XK, bool WK, bool ODD> struct DirectTile {
  static constexpr int NW = 4, BM = 16 * FA, BN = 16 * FB;
  static constexpr int KE = KSTAGE<T>, FLIGHT = FA * FB == 1 ? 4 : 2;  // stages of 128 bytes of k whose loads are in flight
  using acc_t = typename Num<T>::acc;
  static constexpr int LDS_BYTES = NW * FA * FB * 64 * (int)sizeof(acc_t);
  static_assert((XK && WK) || sizeof(T) >= 4, "16-bit types along rows need the transposing reads of the LDS tiles");
  acc_t acc[FB][FA];

  // this lane's 16 bytes of one 16-row block and half stage
  template <bool ALONG_K> struct Source {
    const T* p;
    int64_t ld;
    __device__ __forceinline__ void start(const Operand<T>& o, int r0) {
      const int lane = threadIdx.x & 63, r = r0 + (lane & 15), k = (lane >> 4) * CHE<T>;
      const int64_t row = r < o.rows ? r : o.rows - 1;  // past the end: the last one again, for elements that are not stored
      ld = o.ld;
      p = ALONG_K ? o.p + row * o.ld + k : o.p + row + k * o.ld;
    }
    __device__ __forceinline__ Piece<T, ODD> load(int64_t k) const {
      if constexpr (ALONG_K) {
        return Piece<T, ODD>::load(p + k);
      } else {
        T e[CHE<T>];
#pragma unroll
        for (int j = 0; j < CHE<T>; ++j) e[j] = p[(k + j) * ld];
        return gathered(e);
      }
    }
    // where k ends: loaded now, settled when it is multiplied
    __device__ __forceinline__ Piece<T, ODD> load_end(int64_t k, int64_t klen) const {
      const int first = ((threadIdx.x & 63) >> 4) * CHE<T>;
      const int64_t left = klen - k - first;
      if constexpr (ALONG_K) {
        return load_edge<T, ODD>(p + k, left, p - first);
      } else {
        T e[CHE<T>];
#pragma unroll
        for (int j = 0; j < CHE<T>; ++j) e[j] = p[(j < left ? k + j : -first) * ld];  // past the end: row 0, settled to 0
        return gathered(e);
      }
    }
    __device__ __forceinline__ chunk_t settle_end(const Piece<T, ODD>& v, int64_t k, int64_t klen) const {
      const int64_t left = klen - k - ((threadIdx.x & 63) >> 4) * CHE<T>;
      if constexpr (ALONG_K) {
        return settle(v, left);
      } else {
        T e[CHE<T>];
        __builtin_memcpy(e, &v.c, 16);
#pragma unroll
        for (int j = 0; j < CHE<T>; ++j) e[j] = j < left ? e[j] : (T)0;
        return gathered(e).c;
      }
    }
    static __device__ __forceinline__ Piece<T, ODD> gathered(const T (&e)[CHE<T>]) {
      Piece<T, ODD> v;
      __builtin_memcpy(&v.c, e, 16);
      return v;
    }
  };

  __device__ __forceinline__ void run(const Operand<T>& x, const Operand<T>& w, int64_t klen, char* lds) {
#pragma unroll
    for (int b = 0; b < FB; ++b)
#pragma unroll
      for (int a = 0; a < FA; ++a) acc[b][a] = acc_t{};
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int64_t share = ((klen + KE - 1) / KE + NW - 1) / NW * KE, end = (wave + 1) * share < klen ? (wave + 1) * share : klen;
    int64_t k = wave * share;
    if (k < end) {
      Source<XK> sx[FA];
      Source<WK> sw[FB];
#pragma unroll
      for (int a = 0; a < FA; ++a) sx[a].start(x, a * 16);
#pragma unroll
      for (int b = 0; b < FB; ++b) sw[b].start(w, b * 16);
      Piece<T, ODD> fx[2 * FLIGHT][FA], fw[2 * FLIGHT][FB];
      for (; k + FLIGHT * KE <= end; k += FLIGHT * KE) {
#pragma unroll
        for (int s = 0; s < 2 * FLIGHT; ++s) {
#pragma unroll
          for (int b = 0; b < FB; ++b) fw[s][b] = sw[b].load(k + s * (KE / 2));
#pragma unroll
          for (int a = 0; a < FA; ++a) fx[s][a] = sx[a].load(k + s * (KE / 2));
        }
#pragma unroll
        for (int s = 0; s < 2 * FLIGHT; ++s)
#pragma unroll
          for (int b = 0; b < FB; ++b)
#pragma unroll
            for (int a = 0; a < FA; ++a) acc[b][a] = Num<T>::mma(fw[s][b].value(), fx[s][a].value(), acc[b][a]);
      }
#pragma unroll
      for (int s = 0; s < 2 * FLIGHT; ++s)
        if (k + s * (KE / 2) < end) {
#pragma unroll
          for (int b = 0; b < FB; ++b) fw[s][b] = sw[b].load_end(k + s * (KE / 2), end);
#pragma unroll
          for (int a = 0; a < FA; ++a) fx[s][a] = sx[a].load_end(k + s * (KE / 2), end);
        }
#pragma unroll
      for (int s = 0; s < 2 * FLIGHT; ++s)
        if (k + s * (KE / 2) < end) {
#pragma unroll
          for (int b = 0; b < FB; ++b) {
            const chunk_t w = sw[b].settle_end(fw[s][b], k + s * (KE / 2), end);
#pragma unroll
            for (int a = 0; a < FA; ++a) acc[b][a] = Num<T>::mma(w, sx[a].settle_end(fx[s][a], k + s * (KE / 2), end), acc[b][a]);
          }
        }
    }
    acc_t* part = reinterpret_cast<acc_t*>(lds) + (threadIdx.x & 63);
#pragma unroll
    for (int b = 0; b < FB; ++b)
#pragma unroll
      for (int a = 0; a < FA; ++a) part[((wave * FB + b) * FA + a) * 64] = acc[b][a];
    __syncthreads();
    sums = part;
  }
  const acc_t* sums;

  // every wave adds up its share of the 16 x 16 blocks and hands it out
  template <int E, class F> __device__ __forceinline__ void out(char* lds, int64_t rows, F&& f) const {
    using S = typename std::remove_reference<decltype(acc[0][0][0] + acc[0][0][0])>::type;
    const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
    for (int i = threadIdx.x >> 6; i < FA * FB; i += NW) {
      acc_t v = sums[i * 64];
#pragma unroll
      for (int w = 1; w < NW; ++w) v += sums[(w * FA * FB + i) * 64];
      const int a = i % FA * 16 + r, b = i / FA * 16;
      if (a < rows) {
        // a lane's 4 sums: neighbours, or (fp64) every fourth column
        if (sizeof(T) == 8) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const S one = v[e];
            f.single(a, b + q + 4 * e, one);
          }
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const S one = v[e];
            f.single(a, b + q * 4 + e, one);
          }
        }
      }
    }
  }
};

// D's rows as they are: E = 16 bytes of them at a time
template <class O> struct PlainRows {
  O* d;
  int64_t ld, cols;
  static constexpr int E = 16 / (int)sizeof(O), AHEAD = 2;
  struct Other {};
  __device__ __forceinline__ Other other(int, int) const { return {}; }
  template <class S> __device__ __forceinline__ void single(int i, int j, S v) const {
    if (j < cols) d[i * ld + j] = round_to<O>(v);
  }
  template <class S> __device__ __forceinline__ void operator()(int i, int j, const S* v, const Other&) const {
    O e[E];
#pragma unroll
    for (int c = 0; c < E; ++c) e[c] = round_to<O>(v[c]);
    O* to = d + i * ld + j;
    if (j + E <= cols) {
      Chunk<sizeof(O)> u;
      __builtin_memcpy(&u, e, 16);
      *reinterpret_cast<Chunk<sizeof(O)>*>(to) = u;
    } else {
#pragma unroll 1
      for (int c = 0; c < E; ++c)
        if (j + c < cols) to[c] = round_to<O>(v[c]);
    }
  }
};

// row[j .. j + 3] = the values that are inside n columns
template <class T, class A> __device__ __forceinline__ void store_row(T* row, int64_t j, const A* v, int64_t n) {
  if (sizeof(T) <= 4 && j + 3 < n && reinterpret_cast<uintptr_t>(row + j) % (4 * sizeof(T)) == 0) {
    struct alignas(4 * sizeof(T)) Four { T e[4]; } o;
#pragma unroll
    for (int e = 0; e < 4; ++e) o.e[e] = round_to<T>(v[e]);
    *reinterpret_cast<Four*>(row + j) = o;
    return;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (j + e < n) row[j + e] = round_to<T>(v[e]);
}
