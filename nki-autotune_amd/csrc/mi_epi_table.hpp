// mi_epi_table.hpp -- the compiled tile configs of the epilogue products
// (kernels: mi_mm_epi.hpp) and their launchers.
#pragma once
#include "mi_mm_epi.hpp"

// block_m, block_n, block_k, waves, lds_stages, rhs read non-temporally;
// then what the library's choice goes by: in microseconds a K tile of a block
// alone on its compute unit, a K tile of one of several that share it, a
// block's beginning and end; how many of its blocks a unit holds; and, for a
// rhs that the last-level cache does not hold, microseconds of a K tile of a
// block alone and TB/s of all of them together, rhs[K,N] and rhs[N,K].
//
// The first are fitted (least squares of the logarithm, near the fastest
// config of each shape) to these and eight more configs with up to 16 parts,
// timed at 44 shapes from 1 x 1024 x 1024 to 8192^3 in both layouts with bias
// and gelu_tanh: the choice is within 1.014 of the fastest on average and 1.15
// at most (8 x 1024 x 4096, 1.1 us).  A large block alone is faster per flop
// but leaves units idle in its last round, and a small one reads its operands
// more often: 256x256 takes 102 us at 4096^3 where 128x128 takes 125; at
// 1024^3 64x64 takes 6.9 us and 128x128 11.
//
// The last are fitted so to 19 shapes of 1 to 500 rows and rhs of 300 MB to 1
// GB: within 1.013 on average and 1.17 at most (64 x 8192 x 28672, rhs[N,K]);
// 4 other shapes within 1.09.
// There non-temporal reads pay, and wide rows of rhs[K,N] in one load, in
// whole rounds of blocks: 16 x 28672 x 8192 takes 79 us with 64x256 blocks in
// two parts and 91 with the 128x128 that the first figures alone prefer, 16 x
// 8192 x 28672 81 with 128x128 in four parts and 134 with 64x64 unsplit.
// rhs[N,K] goes non-temporally in 64x64: 80 us unsplit and 90 temporally, 78
// in four parts and 128 temporally unsplit.
//
// A smaller rhs is taken to be in the last-level cache, as in a loop over one
// product; where it comes from HBM, as in a decode over many layers, other
// configs are faster (a set of weights of 1.5 GB in turn: 16 x 8192 x 8192 41
// us and 30, 16 x 4096 x 14336 39 and 26, 32 x 10240 x 8192 59 and 36; a
// caller's cfg reaches them).
#define MI_EPI_CONFIGS(X)                                                     \
  X(256, 256, 64, 8, 2, 0, 0.564f, 1.304f, 11.831f, 1, 1.09f, 19.1f, 6.65f)   \
  X(256, 128, 64, 8, 3, 0, 0.720f, 0.413f, 6.953f, 1, 0.55f, 8.26f, 5.58f)    \
  X(128, 256, 64, 8, 3, 0, 0.719f, 0.667f, 6.492f, 1, 0.80f, 6.79f, 5.52f)    \
  X(128, 128, 64, 4, 4, 0, 0.457f, 0.294f, 5.173f, 1, 0.50f, 6.75f, 5.66f)    \
  X(64, 128, 64, 4, 3, 0, 0.316f, 0.275f, 4.365f, 2, 0.39f, 5.57f, 5.23f)     \
  X(128, 64, 64, 4, 3, 0, 0.318f, 0.264f, 4.439f, 2, 0.27f, 5.37f, 5.30f)     \
  X(64, 64, 64, 4, 2, 0, 0.176f, 0.206f, 3.076f, 4, 0.36f, 5.10f, 5.46f)      \
  X(64, 64, 64, 4, 4, 0, 0.144f, 0.186f, 3.255f, 2, 0.25f, 5.19f, 5.52f)      \
  X(32, 128, 64, 4, 4, 1, 0.171f, 0.376f, 1.655f, 2, 0.38f, 6.37f, 5.92f)     \
  X(128, 128, 64, 4, 3, 1, 0.575f, 0.350f, 4.790f, 1, 0.55f, 11.8f, 6.74f)    \
  X(64, 256, 64, 8, 3, 1, 0.600f, 0.600f, 4.500f, 1, 0.74f, 7.11f, 5.92f)     \
  X(64, 64, 64, 4, 4, 1, 0.260f, 0.230f, 3.200f, 2, 0.29f, 6.10f, 6.88f)

namespace mi {

struct EpiEntry {
  mi_tile_cfg cfg;  // split_k, group_m aside
  float alone, shared, ends;
  int per_cu;
  float cold, stream;  // of a rhs past the last-level cache
  void (*direct)(const EpiMM&, const EpiOut&, hipStream_t);
  void (*split)(const EpiMM&, float* ws, int ldw, hipStream_t);
};

// Tables in the order of MI_EPI_CONFIGS: rhs[K,N], rhs[N,K].
const EpiEntry* epi_table_nn(int* n);
const EpiEntry* epi_table_nt(int* n);

template <int BM, int BN, int BK, int WAVES, int STAGES, bool BT, bool NTB>
void epi_direct(const EpiMM& p, const EpiOut& e, hipStream_t s) {
  const unsigned tiles = (unsigned)((p.M + BM - 1) / BM) * (unsigned)((p.N + BN - 1) / BN);
  mm_epi_kernel<BM, BN, BK, WAVES, STAGES, BT, NTB><<<dim3(tiles), dim3(WAVES * 64), 0, s>>>(p, e);
}
template <int BM, int BN, int BK, int WAVES, int STAGES, bool BT, bool NTB>
void epi_split(const EpiMM& p, float* ws, int ldw, hipStream_t s) {
  const unsigned tiles = (unsigned)((p.M + BM - 1) / BM) * (unsigned)((p.N + BN - 1) / BN);
  mm_epi_split_kernel<BM, BN, BK, WAVES, STAGES, BT, NTB>
      <<<dim3(tiles * (unsigned)p.parts), dim3(WAVES * 64), 0, s>>>(p, ws, ldw);
}

}  // namespace mi

#define MI_EPI_ROW(BM, BN, BK, W, S, NT, ALONE, SHARED, ENDS, PER_CU, COLD, STREAM_KN, STREAM_NK)               \
  EpiEntry{mi_tile_cfg{BM, BN, BK, W, S, 1, 8, NT}, ALONE, SHARED, ENDS, PER_CU, COLD,                          \
           MI_EPI_BT ? STREAM_NK : STREAM_KN,                                                                   \
           &epi_direct<BM, BN, BK, W, S, MI_EPI_BT, NT != 0>, &epi_split<BM, BN, BK, W, S, MI_EPI_BT, NT != 0>},
