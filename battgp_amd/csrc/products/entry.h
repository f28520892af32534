// What the C entry points of libbattgp_products.so share: errors, the device of a call, launches.
#pragma once

#include <hip/hip_runtime.h>

#include "../../../include/battgp_products.h"
#include "plan.h"

// the threads of a launch are counted in 32 bits
constexpr int64_t max_workgroups(int threads) { return ((int64_t)1 << 32) / threads - 1; }

int bgp_products_fail(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));

// makes `device` the current one for the length of a call
class DeviceScope {
  int before_ = -1;
  hipError_t err_;

 public:
  explicit DeviceScope(int device) {
    err_ = hipGetDevice(&before_);
    if (err_ == hipSuccess && before_ != device) err_ = hipSetDevice(device);
    else if (err_ == hipSuccess) before_ = -1;
  }
  ~DeviceScope() {
    if (before_ >= 0) (void)hipSetDevice(before_);
  }
  int check(const char* what) const {
    if (err_ == hipSuccess) return 0;
    (void)hipGetLastError();
    return bgp_products_fail(-2, "%s: %s", what, hipGetErrorString(err_));
  }
};

template <class... A> int launch(const char* what, void (*kernel)(A...), dim3 grid, dim3 block, hipStream_t stream, A... args) {
  void* ptrs[] = {(void*)&args...};
  const hipError_t e = hipLaunchKernel(reinterpret_cast<const void*>(kernel), grid, block, ptrs, 0, stream);
  if (e == hipSuccess) return 0;
  (void)hipGetLastError();  // reported here: not by whoever asks next
  return bgp_products_fail(-2, "%s: launch failed: %s", what, hipGetErrorString(e));
}

// Waves of a tile in LDS: 2 x 4 of 128 x 64 on 256 x 256; 2 x 2 below, but 2 x 4 of 64 x 32 for fp64 on 128 x 128, whose
// accumulators take twice the registers.
constexpr int waves_w(int tile, int size) { return tile == 256 || (size == 8 && tile == 128) ? 4 : 2; }
constexpr int tile_threads(int tile, int size) { return 128 * waves_w(tile, size); }

#ifdef __HIPCC__
// Tiles of 256 x 256 fill a CU each, so the last round of 256 workgroups may have few: its tiles are cut into 2 or 4 parts
// (128 x 256, 128 x 128) where that still is one round.  4099 rows of 8 groups to 2816 columns (k = 1000, bf16), about 270
// tiles: 34.2 us, without it 39.7.  Workgroups go to the 8 XCDs in turn, and each XCD has an L2 of its own: whole rounds are
// dealt in runs, one for each XCD.
// (A launch has less than 2^23 tiles: 32 bits do.)
struct Place {
  int tile;  // -1: nothing to do
  int parts, part;
};
__device__ __forceinline__ Place place_256(int total) {
  constexpr int XCDS = 8;
  const int whole = total / CUS * CUS, left = total - whole, i = blockIdx.x;
  if (i < whole) return Place{i % XCDS * (whole / XCDS) + i / XCDS, 1, 0};
  const int parts = left * 4 <= CUS ? 4 : left * 2 <= CUS ? 2 : 1;
  const int j = i - whole;
  return j < left * parts ? Place{whole + j / parts, parts, j % parts} : Place{-1, 1, 0};
}
// smaller tiles: all of them in runs
__device__ __forceinline__ int place_runs(int total) {
  constexpr int XCDS = 8;
  const int run = (total + XCDS - 1) / XCDS, at = blockIdx.x / XCDS, i = blockIdx.x % XCDS * run + at;
  return at < run && i < total ? i : -1;
}
// Tiles of uneven length, the longest first: dealt to the XCDs 8 at a time, so that each has its share of the long ones.
constexpr int DEALT = 8;
__device__ __forceinline__ int deal(int i) {
  constexpr int XCDS = 8;
  const int at = i / XCDS;
  return (at / DEALT * XCDS + i % XCDS) * DEALT + at % DEALT;
}
// inside a run 8 row tiles are gone through before the next column tile, so that workgroups that run together share rows
// of both operands
struct TileAt {
  int m, n;
};
template <int DEEP = 8> __device__ __forceinline__ TileAt tile_at(int i, int tiles_m, int tiles_n) {
  const int strip = i / (DEEP * tiles_n), in = i - strip * DEEP * tiles_n, deep = tiles_m - strip * DEEP < DEEP ? tiles_m - strip * DEEP : DEEP;
  return TileAt{strip * DEEP + in % deep, in / deep};
}
#endif

// ---- what a call lays out in the caller's workspace ----

// rows of `extent` elements, `per` of them to a batch, copied to rows of ld_to elements (16-byte aligned) back to back
struct PackJob {
  const void* from;
  void* to;
  int64_t rows, per, stride, ld, extent, ld_to;
};
// at most two operands in one launch
int launch_pack(const char* what, int size, const PackJob* jobs, int count, hipStream_t st);

// whether rows start off the 4-byte words
inline bool off_words(const void* p, int64_t ld, int64_t stride, int size) {
  return (reinterpret_cast<uintptr_t>(p) | (uintptr_t)(ld * size) | (uintptr_t)(stride * size)) % 4 != 0;
}

// Takes pieces of the workspace, or only adds up what they come to.
class Workspace {
  char* at_;
  int64_t used_ = 0;

 public:
  explicit Workspace(void* at) : at_(static_cast<char*>(at)) {}
  void* take(int64_t bytes) {
    void* p = at_ ? at_ + used_ : nullptr;
    used_ += (bytes + 255) / 256 * 256;
    return p;
  }
  int64_t used() const { return used_; }
  // whether `bytes` of it, as the caller gave them, do not hold what was taken
  bool short_of(int64_t bytes) const { return used_ > 0 && (!at_ || bytes < used_); }
  bool aligned() const { return reinterpret_cast<uintptr_t>(at_) % 16 == 0; }
};
