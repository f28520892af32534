// Matrix products grouped by expert (bgp_grouped_gemm, bgp_grouped_gemm_dw): the rows of one matrix, sorted by group,
// against each group's own weights, in one launch.  The group bounds are read on the device, so nothing waits for them;
// the host sizes the grid by what they can be at most and the workgroups beyond the last tile leave at once.
//
// Whole calls, from the host's side, on an MI355X: 16384 rows of 16 uneven groups, 4096 x 4096 in bf16 0.53 ms (1040 TFLOP/s: the
// groups' last tiles are part empty and the last round part full; one even group 1430); 2700 rows of 9 groups, 1000 x 1000 in
// fp64 101 us (54 TFLOP/s; 720 tiles of 64 are 2.8 rounds); both gradients of 8192 rows of 16 uneven groups, 2048 x 2048 in bf16 203 us
// (677 TFLOP/s: dW has 8 stages to a tile on the average, and 134 MB of results that go out round by round).
#include "entry.h"
#include "tile.h"

namespace {

// The rows are cut into tiles of BM rows, group by group (a tile never crosses a bound); with `rest` != 0 the rows before
// the first and behind the last group follow as groups G and G + 1.  Bounds are clamped to [0, T], so wrong ones can
// name wrong rows but none outside the matrix.  Every wave of a workgroup works its own tile out for itself: 64 groups
// at a time, one prefix sum over the lanes.
struct RowTile {
  int g;
  int64_t row0, rows;
};

__device__ __forceinline__ int64_t clamp64(int64_t v, int64_t lo, int64_t hi) { return v < lo ? lo : (v > hi ? hi : v); }

// one lane's value, in scalar registers
__device__ __forceinline__ int64_t lane_value(int64_t v, int lane) {
  const uint32_t lo = __builtin_amdgcn_readlane((int)v, lane), hi = __builtin_amdgcn_readlane((int)(v >> 32), lane);
  return (int64_t)((uint64_t)hi << 32 | lo);
}

struct GroupedArgs {
  const void *x, *w;
  void* y;
  const int64_t* off;
  int64_t T, N, K, ldx, ldw, sw, ldy;
  int G, rest, tiles_n;
  int most_m;  // row tiles that the launch was sized for: offsets that do not ascend can ask for more
  int split;   // k is cut in this many parts,
  void* part;  // whose sums go here: [split][rows of D][columns of D], fp32 (fp64)
};

// one part of k: from `from` on, `length` long
struct Part {
  int64_t from, length;
};
__device__ __forceinline__ Part part_of(int64_t k, int stage, int split, int i) {
  if (split == 1) return Part{0, k};
  const uint32_t stages = (uint32_t)((k + stage - 1) / stage);
  const int64_t each = (int64_t)((stages + split - 1) / split) * stage, from = i * each;
  return Part{from, from >= k ? 0 : k - from < each ? k - from : each};
}

// the sum over the lanes up to and with this one: inside rows of 16 lanes, then the last of a row to the rows behind it
__device__ __forceinline__ int lane_sum(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);  // row_shr:1
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row_bcast:15 to the second and fourth row
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // row_bcast:31 to the upper half
  return v;
}

struct Bounds {
  int64_t a, b;
  int sum;  // row tiles up to and with this lane's group, of this batch of 64 groups
};

__device__ __forceinline__ Bounds lane_bounds(const GroupedArgs& p, int BM, int g) {
  const int G = p.G;
  Bounds r{0, 0, 0};
  if (g < G) {
    r.a = clamp64(p.off[g], 0, p.T);
    r.b = clamp64(p.off[g + 1], r.a, p.T);
  } else if (g == G && p.rest) {
    r.b = G > 0 ? clamp64(p.off[0], 0, p.T) : p.T;
  } else if (g == G + 1 && p.rest && G > 0) {
    r.a = clamp64(p.off[G], 0, p.T);
    r.b = p.T;
  }
  r.sum = lane_sum((int)((uint64_t)(r.b - r.a + BM - 1) / (unsigned)BM));
  return r;
}

// all groups' row tiles; with them the bounds of this lane's first group
__device__ __forceinline__ int count_row_tiles(const GroupedArgs& p, int BM, Bounds* first) {
  const int lane = threadIdx.x & 63, groups = p.rest ? p.G + 2 : p.G;
  *first = lane_bounds(p, BM, lane);
  int tiles = __builtin_amdgcn_readlane(first->sum, 63);
  for (int base = 64; base < groups && tiles < p.most_m; base += 64) tiles += __builtin_amdgcn_readlane(lane_bounds(p, BM, base + lane).sum, 63);
  return tiles < p.most_m ? tiles : p.most_m;
}

// the want-th of them
__device__ __forceinline__ RowTile find_row_tile(const GroupedArgs& p, int BM, Bounds r, int want) {
  const int lane = threadIdx.x & 63, groups = p.rest ? p.G + 2 : p.G;
  for (int base = 0; base < groups;) {
    const unsigned long long past = __ballot(r.sum > want);
    if (past) {
      const int j = __ffsll(past) - 1;
      const int tiles = (int)((uint64_t)(r.b - r.a + BM - 1) / (unsigned)BM);
      const int64_t row0 = r.a + (int64_t)(want - (r.sum - tiles)) * BM;
      return RowTile{base + j, lane_value(row0, j), lane_value(r.b - row0 < BM ? r.b - row0 : (int64_t)BM, j)};
    }
    want -= __builtin_amdgcn_readlane(r.sum, 63);
    base += 64;
    r = lane_bounds(p, BM, base + lane);
  }
  return RowTile{-1, 0, 0};
}

// Y[rows of g, :] = X[rows of g, :] W_g^T;  WK: W_g[n, k] = w[g sw + n ldw + k], else w[g sw + k ldw + n]
template <class T, class P, bool WK> __device__ __forceinline__ void rows_tile(const GroupedArgs& p, const RowTile& t, int64_t n0, char* lds) {
  using A = typename Sum<T>::type;
  const bool some = t.g < p.G;
  if (t.g < 0 || (p.split > 1 && !some)) return;
  const Part k = some ? part_of(p.K, KSTAGE<T>, p.split, blockIdx.y) : Part{0, 0};
  const Operand<T> x{static_cast<const T*>(p.x) + t.row0 * p.ldx + k.from, p.ldx, t.rows, p.K >= CHE<T>};
  const Operand<T> w{static_cast<const T*>(p.w) + (some ? t.g * p.sw + (WK ? n0 * p.ldw + k.from : n0 + k.from * p.ldw) : 0), p.ldw, p.N - n0,
                     (WK ? p.K : p.N) >= CHE<T>};
  P tile;
  tile.run(x, w, k.length, lds);
  if (p.split == 1) {
    tile.template out<PlainRows<T>::E>(lds, t.rows, PlainRows<T>{static_cast<T*>(p.y) + t.row0 * p.ldy + n0, p.ldy, p.N - n0});
  } else {
    A* y = static_cast<A*>(p.part) + (blockIdx.y * p.T + t.row0) * p.N + n0;
    tile.template out<PlainRows<A>::E>(lds, t.rows, PlainRows<A>{y, p.N, p.N - n0});
  }
}

template <class T, class P, int BM, int BN, bool WK> __device__ __forceinline__ void rows_workgroup(const GroupedArgs& p, char* lds) {
  Bounds first;
  const int tiles_m = count_row_tiles(p, BM, &first);
  const int i = place_runs(tiles_m * p.tiles_n);
  if (i < 0) return;
  const TileAt at = tile_at(i, tiles_m, p.tiles_n);
  rows_tile<T, P, WK>(p, find_row_tile(p, BM, first, at.m), (int64_t)at.n * BN, lds);
}

// any operands, through registers
template <class T, int BM, int BN, bool WK> __global__ __launch_bounds__(tile_threads(BM, sizeof(T)), 2) void grouped_rows_kernel(GroupedArgs p) {
  using P = Tile<T, BM, BN, 2, waves_w(BM, sizeof(T)), true, WK>;
  __shared__ __attribute__((aligned(16))) char lds[P::LDS_BYTES];
  rows_workgroup<T, P, BM, BN, WK>(p, lds);
}

// operands in whole chunks, pipelined
template <class T, int BM, int BN, bool WK, int SETS> __global__ __launch_bounds__(SETS * tile_threads(BM, sizeof(T)), 2) void grouped_rows_pipe_kernel(GroupedArgs p) {
  using P = PipeTile<T, BM, BN, 2, waves_w(BM, sizeof(T)), true, WK, SETS>;
  __shared__ __attribute__((aligned(16))) char lds[P::LDS_BYTES];
  rows_workgroup<T, P, BM, BN, WK>(p, lds);
}

// 8 waves on 256 x 256
template <class T, bool WK> __global__ __launch_bounds__(512, 2) void grouped_rows_pipe256_kernel(GroupedArgs p) {
  using P = PipeTile<T, 256, 256, 2, 4, true, WK>;
  __shared__ __attribute__((aligned(16))) char lds[P::LDS_BYTES];
  Bounds first;
  const int tiles_m = count_row_tiles(p, 256, &first);
  const Place place = place_256(tiles_m * p.tiles_n);
  if (place.tile < 0) return;
  const TileAt at = tile_at(place.tile, tiles_m, p.tiles_n);
  RowTile t = find_row_tile(p, 256, first, at.m);
  int64_t n0 = (int64_t)at.n * 256;
  if (place.parts == 1) {
    rows_tile<T, P, WK>(p, t, n0, lds);
    return;
  }
  const int down = place.parts == 4 ? place.part >> 1 : place.part;
  t.row0 += down * 128;
  t.rows = t.rows - down * 128 < 128 ? t.rows - down * 128 : 128;
  if (place.parts == 4) n0 += (place.part & 1) * 128;
  if (t.rows <= 0 || n0 >= p.N) return;
  if (place.parts == 4) rows_tile<T, PipeTile<T, 128, 128, 2, 4, true, WK>, WK>(p, t, n0, lds);
  else rows_tile<T, PipeTile<T, 128, 256, 2, 4, true, WK>, WK>(p, t, n0, lds);
}

// small ones, straight from memory
template <class T, int F, bool WK, bool ODD> __global__ __launch_bounds__(256) void grouped_rows_direct_kernel(GroupedArgs p) {
  using P = DirectTile<T, F, F, true, WK, ODD>;
  __shared__ __attribute__((aligned(16))) char lds[P::LDS_BYTES];
  rows_workgroup<T, P, 16 * F, 16 * F, WK>(p, lds);
}

// dW_g[n, k] = sum over the rows t of g of dY[t, n] X[t, k]
template <class T, class P> __device__ __forceinline__ void dw_tile(const GroupedArgs& p, int g, int64_t n0, int64_t k0, char* lds) {
  using A = typename Sum<T>::type;
  const int64_t a = clamp64(p.off[g], 0, p.T), b = clamp64(p.off[g + 1], a, p.T);
  const Part t = part_of(b - a, KSTAGE<T>, p.split, blockIdx.y);
  const Operand<T> dy{static_cast<const T*>(p.y) + (a + t.from) * p.ldy + n0, p.ldy, p.N - n0, p.N >= CHE<T>};
  const Operand<T> x{static_cast<const T*>(p.x) + (a + t.from) * p.ldx + k0, p.ldx, p.K - k0, p.K >= CHE<T>};
  P tile;
  tile.run(dy, x, t.length, lds);
  if (p.split == 1) {
    T* dw = static_cast<T*>(const_cast<void*>(p.w)) + g * p.sw + n0 * p.ldw + k0;
    tile.template out<PlainRows<T>::E>(lds, p.N - n0, PlainRows<T>{dw, p.ldw, p.K - k0});
  } else {
    A* dw = static_cast<A*>(p.part) + (((int64_t)blockIdx.y * p.G + g) * p.N + n0) * p.K + k0;
    tile.template out<PlainRows<A>::E>(lds, p.N - n0, PlainRows<A>{dw, p.K, p.K - k0});
  }
}

// The group with the n-th most rows (up to 64 groups; more are taken as they come).  A tile's time is its group's rows:
// with 2880 of 8192 rows in one of 16 groups the long tiles at the end of an XCD's run made it 207 us.  Where groups are
// short on average the order matters less than the 0.5 us that finding it takes.
__device__ __forceinline__ int group_by_length(const GroupedArgs& p, int n) {
  if (p.G > 64 || p.T < 256 * (int64_t)p.G) return n;
  const int lane = threadIdx.x & 63;
  int key = -1;  // rows (2^25 and more are alike), then the earlier group
  if (lane < p.G) {
    const int64_t a = clamp64(p.off[lane], 0, p.T), rows = clamp64(p.off[lane + 1], a, p.T) - a;
    key = (int)(rows < 33554431 ? rows : 33554431) << 6 | (63 - lane);
  }
  int before = 0;
  for (int j = 0; j < p.G; ++j) before += __builtin_amdgcn_readlane(key, j) > key;
  return __ffsll((unsigned long long)__ballot(lane < p.G && before == n)) - 1;
}

// A group without rows: its zeros, where they lie in one piece, as one of `parts` shares of it.  True if that was it.
template <class T> __device__ __forceinline__ bool dw_empty(const GroupedArgs& p, int g, int part, int parts) {
  const int64_t a = clamp64(p.off[g], 0, p.T), total = p.N * p.K;
  if (clamp64(p.off[g + 1], a, p.T) > a || p.split > 1 || p.ldw != p.K) return false;
  const int64_t share = ((total + parts - 1) / parts + 63) / 64 * 64, from = part * share, to = from + share < total ? from + share : total;
  T* d = static_cast<T*>(const_cast<void*>(p.w)) + g * p.sw;
  const int64_t lead = from + (16 - reinterpret_cast<uintptr_t>(d + from) % 16) % 16 / sizeof(T);  // the first whole 16 bytes
  for (int64_t i = lead + (int64_t)threadIdx.x * CHE<T>; i + CHE<T> <= to; i += (int64_t)blockDim.x * CHE<T>) *reinterpret_cast<chunk_t*>(d + i) = chunk_of(0, 0, 0, 0);
  if (threadIdx.x < CHE<T>) {
    const int64_t i = from + threadIdx.x, j = (to - lead) / CHE<T> * CHE<T> + lead + threadIdx.x;
    if (i < lead && i < to) d[i] = T{};
    if (lead <= to && j < to) d[j] = T{};
  }
  return true;
}

template <class T, class P, int BM, int BN> __device__ __forceinline__ void dw_workgroup(const GroupedArgs& p, char* lds) {
  const int tiles_k = (int)((p.K + BN - 1) / BN), tiles = p.tiles_n * tiles_k;
  const int i = deal(blockIdx.x);
  if (i >= tiles * p.G) return;
  const int g = group_by_length(p, i / tiles);
  if (dw_empty<T>(p, g, i % tiles, tiles)) return;
  const TileAt at = tile_at<4>(i % tiles, p.tiles_n, tiles_k);
  dw_tile<T, P>(p, g, (int64_t)at.m * BM, (int64_t)at.n * BN, lds);
}

template <class T, int BM, int BN> __global__ __launch_bounds__(tile_threads(BM, sizeof(T)), 2) void grouped_dw_kernel(GroupedArgs p) {
  using P = Tile<T, BM, BN, 2, waves_w(BM, sizeof(T)), false, false>;
  __shared__ __attribute__((aligned(16))) char lds[P::LDS_BYTES];
  dw_workgroup<T, P, BM, BN>(p, lds);
}

template <class T, int BM, int BN, int SETS> __global__ __launch_bounds__(SETS * tile_threads(BM, sizeof(T)), 2) void grouped_dw_pipe_kernel(GroupedArgs p) {
  using P = PipeTile<T, BM, BN, 2, waves_w(BM, sizeof(T)), false, false, SETS>;
  __shared__ __attribute__((aligned(16))) char lds[P::LDS_BYTES];
  dw_workgroup<T, P, BM, BN>(p, lds);
}

template <class T> __global__ __launch_bounds__(512, 2) void grouped_dw_pipe256_kernel(GroupedArgs p) {
  using P = PipeTile<T, 256, 256, 2, 4, false, false>;
  __shared__ __attribute__((aligned(16))) char lds[P::LDS_BYTES];
  const int tiles_k = (int)((p.K + 255) / 256), tiles = p.tiles_n * tiles_k;
  Place place = place_256(tiles * p.G);
  if (place.tile < 0) return;
  if (place.parts == 1 && (int)blockIdx.x < tiles * p.G / CUS * CUS) place.tile = deal(blockIdx.x);
  const int g = group_by_length(p, place.tile / tiles);
  if (dw_empty<T>(p, g, place.tile % tiles * 4 + place.part, tiles * 4)) {  // in quarters: all four of a whole tile
    if (place.parts < 4)
      for (int q = place.parts; q < 4; q += place.parts) dw_empty<T>(p, g, place.tile % tiles * 4 + q + place.part, tiles * 4);
    return;
  }
  const TileAt at = tile_at<4>(place.tile % tiles, p.tiles_n, tiles_k);
  int64_t n0 = (int64_t)at.m * 256, k0 = (int64_t)at.n * 256;
  if (place.parts == 1) {
    dw_tile<T, P>(p, g, n0, k0, lds);
    return;
  }
  n0 += (place.parts == 4 ? place.part >> 1 : place.part) * 128;
  if (place.parts == 4) k0 += (place.part & 1) * 128;
  if (n0 >= p.N || k0 >= p.K) return;
  if (place.parts == 4) dw_tile<T, PipeTile<T, 128, 128, 2, 4, false, false>>(p, g, n0, k0, lds);
  else dw_tile<T, PipeTile<T, 128, 256, 2, 4, false, false>>(p, g, n0, k0, lds);
}

template <class T, int F> __global__ __launch_bounds__(256) void grouped_dw_direct_kernel(GroupedArgs p) {
  using P = DirectTile<T, F, F, false, false, false>;
  __shared__ __attribute__((aligned(16))) char lds[P::LDS_BYTES];
  dw_workgroup<T, P, 16 * F, 16 * F>(p, lds);
}

// out[r, c] = the parts' sum, in their order; rows of no group (off != NULL) as bgp_grouped_gemm leaves them
struct JoinArgs {
  const void* part;
  void* out;
  int64_t rows, cols, per, stride, ld;  // row r of `out` is at (r / per) stride + (r % per) ld
  int split;
  const int64_t* off;
  int G, rest;
};
template <class T> __global__ __launch_bounds__(256) void join_kernel(JoinArgs p) {
  using A = typename Sum<T>::type;
  const int64_t c = ((int64_t)blockIdx.x * 64 + threadIdx.x) * 4;
  if (c >= p.cols) return;
  const A* part = static_cast<const A*>(p.part);
  for (int64_t r = (int64_t)blockIdx.y * 4 + threadIdx.y; r < p.rows; r += (int64_t)gridDim.y * 4) {
    A sum[4] = {0, 0, 0, 0};
    const bool none = p.off && (r < p.off[0] || r >= p.off[p.G]);
    if (none && !p.rest) continue;
    if (!none)
      for (int s = 0; s < p.split; s += 4) {  // four parts to a wait for memory (18000 x 500 x 512 fp64 in 4: 181 -> 165 us)
        A one[4][4];
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
          for (int e = 0; e < 4; ++e) one[u][e] = s + u < p.split && c + e < p.cols ? part[((s + u) * p.rows + r) * p.cols + c + e] : (A)0;
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
          for (int e = 0; e < 4; ++e) sum[e] += one[u][e];
      }
    store_row(static_cast<T*>(p.out) + r / p.per * p.stride + r % p.per * p.ld, c, sum, p.cols);
  }
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

// rows that start on 16 bytes, and for an operand along rows no chunk that reaches past a row's end
bool aligned(const void* p, int64_t ld, int64_t stride, int size, bool along_k, int64_t extent) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld * size % 16 == 0 && stride * size % 16 == 0 && (along_k || extent * size % 16 == 0) &&
         pipe_fits(ld, size, along_k, 256);
}

// one operand: what it is now, and what it would be in the workspace
struct Laid {
  const void* p;
  int64_t stride, ld, rows, per, extent;
  bool along_k, ok;
  Laid(const void* at, int64_t batches, int64_t stride_, int64_t per_, int64_t ld_, int64_t extent_, int size, bool along)
      : p(at), stride(stride_), ld(ld_), rows(batches * per_), per(per_), extent(extent_), along_k(along), ok(aligned(at, ld_, stride_, size, along, extent_)) {}
  double bytes(int size) const { return ok ? 0 : (double)rows * padded_row(extent, size) * size; }
  void move(Workspace& ws, int size, PackJob* jobs, int* count) {
    if (ok) return;
    const int64_t to = padded_row(extent, size);
    void* at = ws.take(rows * to * size);
    jobs[(*count)++] = PackJob{p, at, rows, per, stride, ld, extent, to};
    p = at;
    ld = to;
    stride = per * to;
  }
};

template <class T> int join(const char* what, const JoinArgs& j, hipStream_t st) {
  const int64_t y = (j.rows + 3) / 4;
  return launch(what, join_kernel<T>, dim3((unsigned)((j.cols + 255) / 256), (unsigned)(y < 65535 ? y : 65535)), dim3(64, 4), st, j);
}

template <class T, bool WK, int CUT> int run_rows(const GroupedArgs& p0, hipStream_t st) {
  const char* what = "bgp_grouped_gemm";
  constexpr int B = tile_of(CUT), SETS = CUT == TWIN64 ? 2 : 1;
  GroupedArgs p = p0;
  p.tiles_n = (int)((p.N + B - 1) / B);
  // row tiles there can be at most: a group adds less than one to its share of the rows
  const int64_t most_m = p.T / B + p.G + (p.rest ? 2 : 0), tiles = most_m * p.tiles_n + (B == 256 ? CUS : 7);
  p.most_m = (int)most_m;
  const dim3 grid((unsigned)tiles, p.split);
  if constexpr (CUT <= DIRECT32) {
    if constexpr (sizeof(T) < 4)
      if (off_words(p.x, p.ldx, 0, sizeof(T)) || off_words(p.w, p.ldw, p.sw, sizeof(T)))
        return launch(what, grouped_rows_direct_kernel<T, B / 16, WK, true>, grid, dim3(256), st, p);
    return launch(what, grouped_rows_direct_kernel<T, B / 16, WK, false>, grid, dim3(256), st, p);
  } else if constexpr (CUT <= PLAIN128) {
    return launch(what, grouped_rows_kernel<T, B, B, WK>, grid, dim3(tile_threads(B, sizeof(T))), st, p);
  } else if constexpr (CUT == PIPE256) {
    return launch(what, grouped_rows_pipe256_kernel<T, WK>, grid, dim3(512), st, p);
  } else {
    return launch(what, grouped_rows_pipe_kernel<T, B, B, WK, SETS>, grid, dim3(SETS * tile_threads(B, sizeof(T))), st, p);
  }
}

template <class T, bool WK> int rows_by_cut(const GroupedArgs& p, int cut, hipStream_t st) {
  if constexpr (WK || sizeof(T) >= 4) {
    if (cut == DIRECT16) return run_rows<T, WK, DIRECT16>(p, st);
    if (cut == DIRECT32) return run_rows<T, WK, DIRECT32>(p, st);
  }
  if (cut == PLAIN64) return run_rows<T, WK, PLAIN64>(p, st);
  if (cut == PLAIN128) return run_rows<T, WK, PLAIN128>(p, st);
  if constexpr (sizeof(T) == 2) {
    if (cut == PIPE256) return run_rows<T, WK, PIPE256>(p, st);
    if (cut == TWIN64) return run_rows<T, WK, TWIN64>(p, st);
  }
  return cut == PIPE64 ? run_rows<T, WK, PIPE64>(p, st) : run_rows<T, WK, PIPE128>(p, st);
}

template <class T> int run_rows_plan(const GroupedArgs& p, bool trans, const Plan& plan, hipStream_t st) {
  const int rc = trans ? rows_by_cut<T, false>(p, plan.cut, st) : rows_by_cut<T, true>(p, plan.cut, st);
  if (rc || p.split == 1) return rc;
  return join<T>("bgp_grouped_gemm", JoinArgs{p.part, p.y, p.T, p.N, p.T, 0, p.ldy, p.split, p.off, p.G, p.rest}, st);
}

template <class T, int CUT> int run_dw(const GroupedArgs& p0, hipStream_t st) {
  const char* what = "bgp_grouped_gemm_dw";
  constexpr int B = tile_of(CUT), SETS = CUT == TWIN64 ? 2 : 1;
  GroupedArgs p = p0;
  p.tiles_n = (int)((p.N + B - 1) / B);
  const int64_t tiles = (int64_t)p.G * p.tiles_n * ((p.K + B - 1) / B) + (B == 256 ? CUS : 8 * DEALT - 1);
  const dim3 grid((unsigned)tiles, p.split);
  if constexpr (CUT <= DIRECT32) return launch(what, grouped_dw_direct_kernel<T, B / 16>, grid, dim3(256), st, p);
  else if constexpr (CUT <= PLAIN128) return launch(what, grouped_dw_kernel<T, B, B>, grid, dim3(tile_threads(B, sizeof(T))), st, p);
  else if constexpr (CUT == PIPE256) return launch(what, grouped_dw_pipe256_kernel<T>, grid, dim3(512), st, p);
  else return launch(what, grouped_dw_pipe_kernel<T, B, B, SETS>, grid, dim3(SETS * tile_threads(B, sizeof(T))), st, p);
}

template <class T> int dw_by_cut(const GroupedArgs& p, int cut, hipStream_t st) {
  if constexpr (sizeof(T) >= 4) {
    if (cut == DIRECT16) return run_dw<T, DIRECT16>(p, st);
    if (cut == DIRECT32) return run_dw<T, DIRECT32>(p, st);
  }
  if (cut == PLAIN64) return run_dw<T, PLAIN64>(p, st);
  if (cut == PLAIN128) return run_dw<T, PLAIN128>(p, st);
  if constexpr (sizeof(T) == 2) {
    if (cut == PIPE256) return run_dw<T, PIPE256>(p, st);
    if (cut == TWIN64) return run_dw<T, TWIN64>(p, st);
  }
  return cut == PIPE64 ? run_dw<T, PIPE64>(p, st) : run_dw<T, PIPE128>(p, st);
}

template <class T> int run_dw_plan(const GroupedArgs& p, const Plan& plan, hipStream_t st) {
  const int rc = dw_by_cut<T>(p, plan.cut, st);
  if (rc || p.split == 1) return rc;
  return join<T>("bgp_grouped_gemm_dw", JoinArgs{p.part, const_cast<void*>(p.w), p.G * p.N, p.K, p.N, p.sw, p.ldw, p.split, nullptr, p.G, 0}, st);
}

int check_sizes(const char* what, int dtype, int64_t T, int64_t N, int64_t K, int64_t G, const void* off) {
  if (!size_of(dtype)) return bgp_products_fail(-1, "%s: unknown type %d", what, dtype);
  if (T < 0 || N < 0 || K < 0 || G < 0 || G > BGP_MAX_GROUPS)
    return bgp_products_fail(-1, "%s: bad sizes T=%lld N=%lld K=%lld G=%lld", what, (long long)T, (long long)N, (long long)K, (long long)G);
  if (G > 0 && !off) return bgp_products_fail(-1, "%s: no offsets", what);
  return 0;
}

}  // namespace

extern "C" int64_t bgp_grouped_gemm(int device, void* stream, int dtype, int64_t T, int64_t N, int64_t K, int64_t G, const void* X, int64_t ldx,
                                    const void* W, int64_t strideW, int64_t ldw, int w_trans, const int64_t* offsets, void* Y, int64_t ldy, int zero_rest,
                                    void* workspace, int64_t workspace_bytes) {
  const char* what = "bgp_grouped_gemm";
  if (int rc = check_sizes(what, dtype, T, N, K, G, offsets)) return rc;
  if (T == 0 || N == 0 || (G == 0 && !zero_rest)) return 0;
  if (!Y || (K > 0 && G > 0 && (!X || !W))) return bgp_products_fail(-1, "%s: null pointer", what);
  if (ldx < K || ldy < N || ldw < (w_trans ? N : K) || strideW < 0)
    return bgp_products_fail(-1, "%s: bad strides ldx=%lld ldw=%lld strideW=%lld ldy=%lld", what, (long long)ldx, (long long)ldw, (long long)strideW, (long long)ldy);
  const int size = size_of(dtype);
  if (G == 0) K = 0;  // no row has weights: zeros, and neither operand is read (or copied): X and W may be NULL
  Laid x(X, 1, 0, T, ldx, K, size, true), w(W, strideW ? G : 1, strideW, w_trans ? K : N, ldw, w_trans ? N : K, size, !w_trans);
  const Plan plan = plan_rows(size, T, N, K, G, w_trans, Operands{x.ok && w.ok, x.bytes(size) + w.bytes(size)});
  if (plan.cut == CUTS) return bgp_products_fail(-1, "%s: T=%lld N=%lld are more tiles than one launch holds", what, (long long)T, (long long)N);
  Workspace ws(workspace);
  PackJob jobs[2];
  int count = 0;
  if (plan.pack) {
    x.move(ws, size, jobs, &count);
    w.move(ws, size, jobs, &count);
    if (strideW == 0) w.stride = 0;
  }
  void* part = plan.split > 1 ? ws.take(plan.split * T * N * (size == 8 ? 8 : 4)) : nullptr;
  if (ws.short_of(workspace_bytes)) return ws.used();
  if (!ws.aligned()) return bgp_products_fail(-1, "%s: the workspace is not aligned to 16 bytes", what);
  DeviceScope scope(device);
  if (int rc = scope.check(what)) return rc;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (count)
    if (int rc = launch_pack(what, size, jobs, count, st)) return rc;
  const GroupedArgs p{x.p, w.p, Y, offsets, T, N, K, x.ld, w.ld, w.stride, ldy, (int)G, zero_rest != 0, 0, 0, plan.split, part};
  switch (dtype) {
    case BGP_F64: return run_rows_plan<double>(p, w_trans, plan, st);
    case BGP_F32: return run_rows_plan<float>(p, w_trans, plan, st);
    case BGP_BF16: return run_rows_plan<bf16_t>(p, w_trans, plan, st);
    default: return run_rows_plan<f16_t>(p, w_trans, plan, st);
  }
}

extern "C" int64_t bgp_grouped_gemm_dw(int device, void* stream, int dtype, int64_t T, int64_t N, int64_t K, int64_t G, const void* dY, int64_t lddy,
                                       const void* X, int64_t ldx, const int64_t* offsets, void* dW, int64_t strideW, int64_t ldw, void* workspace,
                                       int64_t workspace_bytes) {
  const char* what = "bgp_grouped_gemm_dw";
  if (int rc = check_sizes(what, dtype, T, N, K, G, offsets)) return rc;
  if (N == 0 || K == 0 || G == 0) return 0;
  if (!dW || (T > 0 && (!dY || !X))) return bgp_products_fail(-1, "%s: null pointer", what);
  if (lddy < N || ldx < K || ldw < K || strideW < N * ldw)
    return bgp_products_fail(-1, "%s: bad strides lddy=%lld ldx=%lld ldw=%lld strideW=%lld", what, (long long)lddy, (long long)ldx, (long long)ldw, (long long)strideW);
  const int size = size_of(dtype);
  Laid y(dY, 1, 0, T, lddy, N, size, false), x(X, 1, 0, T, ldx, K, size, false);
  const Plan plan = plan_dw(size, T, N, K, G, Operands{x.ok && y.ok, x.bytes(size) + y.bytes(size)});
  if (plan.cut == CUTS)
    return bgp_products_fail(-1, "%s: G=%lld N=%lld K=%lld are more tiles than one launch holds", what, (long long)G, (long long)N, (long long)K);
  Workspace ws(workspace);
  PackJob jobs[2];
  int count = 0;
  if (plan.pack) {
    y.move(ws, size, jobs, &count);
    x.move(ws, size, jobs, &count);
  }
  void* part = plan.split > 1 ? ws.take(plan.split * G * N * K * (size == 8 ? 8 : 4)) : nullptr;
  if (ws.short_of(workspace_bytes)) return ws.used();
  if (!ws.aligned()) return bgp_products_fail(-1, "%s: the workspace is not aligned to 16 bytes", what);
  DeviceScope scope(device);
  if (int rc = scope.check(what)) return rc;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (count)
    if (int rc = launch_pack(what, size, jobs, count, st)) return rc;
  const GroupedArgs p{x.p, dW, const_cast<void*>(y.p), offsets, T, N, K, x.ld, ldw, strideW, y.ld, (int)G, 0, 0, 0, plan.split, part};
  switch (dtype) {
    case BGP_F64: return run_dw_plan<double>(p, plan, st);
    case BGP_F32: return run_dw_plan<float>(p, plan, st);
    case BGP_BF16: return run_dw_plan<bf16_t>(p, plan, st);
    default: return run_dw_plan<f16_t>(p, plan, st);
  }
}
