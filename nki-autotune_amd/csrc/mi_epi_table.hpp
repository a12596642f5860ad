// mi_epi_table.hpp -- the compiled tile configs of the epilogue products
// (kernels: mi_mm_epi.hpp) and their launchers.
#pragma once
#include "mi_mm_epi.hpp"

// block_m, block_n, block_k, waves, lds_stages, rhs read non-temporally
#define MI_EPI_CONFIGS(X)   \
  X(256, 256, 64, 8, 2, 0)  \
  X(256, 128, 64, 8, 3, 0)  \
  X(256, 128, 64, 4, 2, 0)  \
  X(256, 128, 64, 8, 2, 0)  \
  X(128, 256, 64, 8, 3, 0)  \
  X(128, 256, 64, 4, 2, 0)  \
  X(128, 128, 64, 4, 2, 0)  \
  X(128, 128, 64, 4, 4, 0)  \
  X(64, 128, 64, 4, 2, 0)   \
  X(64, 128, 64, 4, 3, 0)   \
  X(128, 64, 64, 4, 2, 0)   \
  X(128, 64, 64, 4, 3, 0)   \
  X(64, 64, 64, 4, 2, 0)    \
  X(64, 64, 64, 4, 4, 0)    \
  X(32, 64, 64, 2, 4, 0)    \
  X(32, 128, 64, 4, 4, 1)   \
  X(64, 128, 64, 4, 4, 1)   \
  X(128, 128, 64, 4, 2, 1)  \
  X(128, 128, 64, 4, 3, 1)

namespace mi {

struct EpiEntry {
  mi_tile_cfg cfg;  // split_k, group_m aside
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

#define MI_EPI_ROW(BM, BN, BK, W, S, NT)                                                   \
  EpiEntry{mi_tile_cfg{BM, BN, BK, W, S, 1, 8, NT}, &epi_direct<BM, BN, BK, W, S, MI_EPI_BT, NT != 0>, \
           &epi_split<BM, BN, BK, W, S, MI_EPI_BT, NT != 0>},
