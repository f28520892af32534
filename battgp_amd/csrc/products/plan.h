// How a product is cut, chosen by a model of its time.
#pragma once

#include <math.h>
#include <stdint.h>

// Straight from memory in tiles of 16 or 32, through registers (any operands) or pipelined (16-byte aligned rows) in tiles
// of 64, 128 or 256, or of 64 with k halved between two sets of waves.
enum Cut { DIRECT16, DIRECT32, PLAIN64, PLAIN128, PIPE64, PIPE128, PIPE256, TWIN64, CUTS };
constexpr int tile_of(int cut) {
  return cut == DIRECT16 ? 16 : cut == DIRECT32 ? 32 : cut == PLAIN64 || cut == PIPE64 || cut == TWIN64 ? 64 : cut == PIPE256 ? 256 : 128;
}
constexpr int kind_of(int size) { return size == 1 ? 0 : size == 2 ? 1 : size == 4 ? 2 : 3; }

// Measured on an MI355X, in us for one stage (128 bytes of k) of one tile: on a CU that is full of such tiles, and the time
// from stage to stage of a tile that has its CU to itself.  {int8, 16 bits, fp32, fp64}, by Cut.  In TFLOP/s of the whole
// chip the first row of e.g. PIPE128 is 2138, 925, 148 and 71, of DIRECT32 271, 190, 65 and 41; PLAIN* were measured
// on operands that are not aligned, since the others are pipelined.  DIRECT* were measured on operands along k: along rows (fp32 and
// fp64) they load element by element, and the model is short (fp32, 1237 rows of 5 groups, 333 x 513: dX predicted 12.2 us,
// kernel 13.6; dW 12.1 and 17.8).
constexpr float STAGE_US[4][CUTS] = {{0.115f, 0.247f, 0.40f, 0.95f, 0.187f, 0.50f, 1.68f, 0.24f},
                                     {0.075f, 0.177f, 0.39f, 0.87f, 0.228f, 0.58f, 1.78f, 0.25f},
                                     {0.090f, 0.260f, 0.61f, 2.20f, 0.476f, 1.82f, 9e9f, 9e9f},
                                     {0.075f, 0.200f, 0.60f, 2.20f, 0.470f, 1.90f, 9e9f, 9e9f}};
constexpr float ALONE_US[4][CUTS] = {{0.12f, 0.22f, 0.52f, 1.0f, 0.30f, 0.62f, 1.7f, 0.24f},
                                     {0.10f, 0.20f, 0.68f, 1.1f, 0.47f, 0.59f, 1.8f, 0.25f},
                                     {0.12f, 0.27f, 0.85f, 2.5f, 0.61f, 2.06f, 9e9f, 9e9f},
                                     {0.10f, 0.23f, 0.88f, 2.5f, 0.59f, 1.95f, 9e9f, 9e9f}};
constexpr float TWIN_US = 0.3f;  // filling its buffers and adding up
constexpr float LAUNCH_US = 3.0f, PACK_US = 2.0f, COPY_BYTES_US = 3.5e6f;
constexpr float OUT_BYTES_US = 20e3f;  // a CU's results to memory and back, with more than 4 waves at it
constexpr int CUS = 256;
constexpr int64_t MOST_TILES = (1 << 23) - 1 - CUS;  // the threads of a launch (512 to a workgroup) are counted in 32 bits

struct Plan {
  int cut = CUTS, split = 1;  // CUTS: more tiles than one launch holds, however it is cut
  bool pack = false;
};

// Rounds of a chip full of tiles.  The last round of 256 x 256 tiles is cut into parts where its tiles are few (entry.h,
// place_256): by their stages a quarter takes 0.35 and a half 0.6 of a whole one (16 groups of 512 rows, 2048 x 2048 in bf16, 320
// tiles expected: 62 us against 68 in tiles of 128, which two whole rounds would say to take).
inline double rounds_of(int cut, double units) {
  if (cut != PIPE256) return ceil(units / CUS);
  const double whole = floor(units / CUS), left = (units - whole * CUS) / CUS;
  return whole + (left == 0 ? 0 : left <= 0.25 ? 0.35 : left <= 0.5 ? 0.6 : 1);
}

// What the model is asked: D in tiles of b x b has tiles(b) of them; k bytes of k each.
struct Question {
  int size;                // of an element
  bool direct, pipe;       // which cuts the operands allow as they are
  bool packable;           // the pipelined ones after unaligned operands have been copied into aligned rows
  double k, pack_bytes;    // length of k; bytes of the operands that would be copied
  double outputs;          // elements of D
  int out_bytes;           // written (and read, if D is added to) for each
  int most_split;          // 1: k is not cut
};

// double(int b), of tiles: how many are expected, and how many there may be at most
template <class F, class M> Plan make_plan(const Question& q, F&& tiles, M&& most) {
  Plan best;
  double least = 1e30;
  const int kind = kind_of(q.size);
  const double stages = ceil(q.k * q.size / 128.0);
  for (int cut = 0; cut < CUTS; ++cut) {
    if (STAGE_US[kind][cut] > 1e8f || (cut <= DIRECT32 && !q.direct)) continue;
    const bool pipe = cut >= PIPE64, pack = pipe && !q.pipe;
    if (pack && !q.packable) continue;
    if ((cut == PLAIN64 || cut == PLAIN128) && q.pipe) continue;
    if (most(tile_of(cut)) > MOST_TILES) continue;
    const double unit = tiles(tile_of(cut));
    for (int split = 1; split <= (cut <= DIRECT32 ? 1 : q.most_split); split *= 2) {
      if (split > 1 && stages < 4.0 * split) break;
      if (cut == TWIN64 && unit * split > CUS) break;  // a CU holds one of these: two of PIPE64 would overlap
      const double each = rounds_of(cut, unit * split), sets = cut == TWIN64 ? 2 : 1, deep = sets * ceil(ceil(stages / split) / sets);
      double stage = each * STAGE_US[kind][cut];
      if (stage < ALONE_US[kind][cut]) stage = ALONE_US[kind][cut];
      const double tile_bytes = each * tile_of(cut) * tile_of(cut) * (split > 1 ? (q.size == 8 ? 8 : 4) : q.out_bytes);
      double us = LAUNCH_US + deep * stage + tile_bytes / (each > 1 || cut == PIPE256 ? OUT_BYTES_US : OUT_BYTES_US / 2);
      if (cut == TWIN64) us += TWIN_US;
      if (split > 1) us += LAUNCH_US + (split + 1) * q.outputs * (q.size == 8 ? 8 : 4) / COPY_BYTES_US;
      if (pack) us += PACK_US + 2 * q.pack_bytes / COPY_BYTES_US;
      if (us < least) {
        least = us;
        best.cut = cut;
        best.split = split;
        best.pack = pack;
      }
    }
  }
  return best;
}

// ---- the three products' questions ----

// rows of a copy that start on whole cache lines
constexpr int64_t padded_row(int64_t extent, int size) { return (extent * size + 127) / 128 * 128 / size; }

// whether an operand's offsets inside a stage fit 32 bits: up to `rows` rows of it along k, a stage's rows of k otherwise
inline bool pipe_fits(int64_t ld, int size, bool along_k, int rows) {
  return (along_k ? rows : 128 / size) * ld * size < (int64_t)1 << 32;
}

// Row tiles of b rows that are expected: every group with rows has one at least and half of one to spare, a single one is
// taken to hold all rows.
inline double expected_tiles(int64_t T, int64_t G, int b) {
  if (G == 1) return ceil((double)T / b);
  const double used = (double)(G < T ? G : T), even = (double)T / b + 0.5 * used;
  return even > used ? even : used;
}

// What a call's two operands are like: those that do not suit the pipelined cuts as they lie would be copied, `bytes` of them.
struct Operands {
  bool ok;
  double bytes;
};

// Y[T, N] of G groups' rows against W[K] along k, or (w_trans) along N
inline Plan plan_rows(int size, int64_t T, int64_t N, int64_t K, int64_t G, bool w_trans, const Operands& o) {
  const bool wide = K * size >= 16 && (!w_trans || N * size >= 16);
  const Question q{size, wide && (!w_trans || size >= 4), o.ok,
                   G > 0 && pipe_fits(padded_row(K, size), size, true, 256) && pipe_fits(padded_row(w_trans ? N : K, size), size, !w_trans, 256), (double)K, o.bytes,
                   (double)T * N, size, G > 0 ? 16 : 1};
  return make_plan(
      q, [&](int b) { return expected_tiles(T, G, b) * ((N + b - 1) / b); }, [&](int b) { return ((double)(T / b) + G + 2) * ((N + b - 1) / b); });
}

// dW[G, N, K] of T rows.  A group's rows are its length of k: their mean is taken, as if groups with rows were even.
inline Plan plan_dw(int size, int64_t T, int64_t N, int64_t K, int64_t G, const Operands& o) {
  const double used = (double)(G < T ? G : T > 0 ? T : 1);
  const Question q{size, size >= 4, o.ok, pipe_fits(padded_row(N, size), size, false, 256) && pipe_fits(padded_row(K, size), size, false, 256),
                   ceil(T / used), o.bytes, (double)G * N * K, size, 16};
  const auto tiles = [&](int b) { return (double)G * ((N + b - 1) / b) * ((K + b - 1) / b); };
  return make_plan(q, tiles, tiles);
}

// Y[M, N] in 8 bits, `out_bytes` written (and read) for each element
inline Plan plan_int8(int out_bytes, int64_t M, int64_t N, int64_t K, const Operands& o) {
  const Question q{1, K >= 16, o.ok, true, (double)K, o.bytes, (double)M * N, out_bytes, 1};
  const auto tiles = [&](int b) { return (double)((M + b - 1) / b) * ((N + b - 1) / b); };
  return make_plan(q, tiles, tiles);
}
