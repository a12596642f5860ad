// mi_fp8_table.hpp -- the compiled tile configs of the 8-bit products (kernels:
// mi_mm_fp8.hpp) and their launchers.
#pragma once
#include "mi_mm_fp8.hpp"

// block_m, block_n, waves, lds_stages, rhs read non-temporally; then what the
// library's choice goes by, terms of an estimate in microseconds: a K tile of a
// block alone on its compute unit with scales for 128 rows of rhs, for each row,
// and with powers of two, a K tile of one of several that share the unit, a
// block's beginning and end; how many of its blocks a unit holds; and TB/s of
// all of them together where rhs comes from HBM.  Of the two kinds of K tiles
// the one that makes the longer time counts.  Where one block fills a unit that
// is the larger of two terms, and the other is where the fit began, 0.350, which
// says nothing of a K tile.
//
// Fitted (least squares of the logarithm, near the fastest config of each
// shape) to all of them with up to 16 parts, timed in graphs at 42 shapes from
// 1 x 4096 x 4096 to 8192^3 with each kind of scales, and at 30 of 1 to 300
// rows and rhs of 64 to 235 MB, three operands in turn: the choice is within
// 1.03 of the fastest on average and 1.23 at most (48 x 20000 x 5000).  A large
// block alone is faster per flop but leaves units idle in its last round:
// 256x256 takes 62 us at 4096^3 where 128x128 takes 101, and at 1024^3, 6.2 in
// 64x64, the products' time is that of a block's eight K tiles one after the
// other.  For few rows non-temporal reads of rhs pay: 16 x 28672 x 8192 takes
// 43 us with them and 48 without, both in 64x64; 16 x 8192 x 28672 40 in 32x128
// and four parts, 78 unsplit.
#define MI_FP8_CONFIGS(X)                                                              \
  X(256, 256, 8, 2, 0, 1.543f, 2.009f, 1.428f, 0.350f, 6.452f, 1, 27.75f)              \
  X(256, 128, 8, 3, 0, 0.840f, 1.042f, 0.350f, 0.750f, 5.318f, 1, 15.18f)              \
  X(128, 256, 8, 3, 0, 0.842f, 1.024f, 0.766f, 0.350f, 5.507f, 1, 6.15f)               \
  X(128, 128, 4, 4, 0, 0.674f, 0.816f, 0.350f, 0.536f, 3.639f, 1, 6.34f)               \
  X(64, 128, 4, 3, 0, 0.506f, 0.548f, 0.368f, 0.355f, 3.489f, 2, 5.75f)                \
  X(128, 64, 4, 3, 0, 0.540f, 0.596f, 0.408f, 0.342f, 3.142f, 2, 7.08f)                \
  X(64, 64, 4, 4, 0, 0.343f, 0.365f, 0.313f, 0.259f, 3.022f, 2, 7.05f)                 \
  X(64, 64, 4, 4, 1, 0.361f, 0.385f, 0.335f, 0.303f, 2.978f, 2, 12.11f)                \
  X(32, 128, 4, 3, 1, 0.434f, 0.447f, 0.396f, 0.393f, 2.636f, 2, 6.28f)

namespace mi {

struct Fp8Entry {
  mi_tile_cfg cfg;  // split_k, group_m aside
  float alone[3], shared, ends;  // alone: by kScaleSquare, kScaleRows, kScalePow2
  int per_cu;
  float stream;
  void (*launch)(const Fp8MM&, const Fp8Out&, float* ws, int ldw, hipStream_t);
};

// The table, in the order of MI_FP8_CONFIGS, for a way of scaling and lhs's
// type (0: e4m3, 1: e5m2).
const Fp8Entry* fp8_table_square_e4m3(int* n);
const Fp8Entry* fp8_table_square_e5m2(int* n);
const Fp8Entry* fp8_table_rows_e4m3(int* n);
const Fp8Entry* fp8_table_rows_e5m2(int* n);
const Fp8Entry* fp8_table_pow2_e4m3(int* n);
const Fp8Entry* fp8_table_pow2_e5m2(int* n);

template <int BM, int BN, int WAVES, int STAGES, int MODE, int LA, bool NTB>
void fp8_launch(const Fp8MM& p, const Fp8Out& e, float* ws, int ldw, hipStream_t s) {
  const unsigned tiles = (unsigned)((p.M + BM - 1) / BM) * (unsigned)((p.N + BN - 1) / BN);
  mm_fp8_kernel<BM, BN, WAVES, STAGES, MODE, LA, NTB>
      <<<dim3(tiles * (unsigned)p.parts), dim3(WAVES * 64), 0, s>>>(p, e, ws, ldw);
}

// Two products in one launch, in 64 x 64 blocks of three stages: three to a unit.
#define MI_FP8_TWO 64, 64, 4, 3
void fp8_two_rows_e4m3(const Fp8Two& two, unsigned blocks, hipStream_t s);
void fp8_two_rows_e5m2(const Fp8Two& two, unsigned blocks, hipStream_t s);
void fp8_two_pow2_e4m3(const Fp8Two& two, unsigned blocks, hipStream_t s);
void fp8_two_pow2_e5m2(const Fp8Two& two, unsigned blocks, hipStream_t s);

}  // namespace mi

#define MI_FP8_ROW(BM, BN, W, S, NT, SQUARE, ROWS, POW2, SHARED, ENDS, PER_CU, STREAM)                       \
  Fp8Entry{mi_tile_cfg{BM, BN, 128, W, S, 1, 8, NT}, {SQUARE, ROWS, POW2}, SHARED, ENDS, PER_CU, STREAM,       \
           &fp8_launch<BM, BN, W, S, MI_FP8_MODE, MI_FP8_LHS, NT != 0>},
