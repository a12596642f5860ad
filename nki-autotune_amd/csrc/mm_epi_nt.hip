// Instances of the epilogue products with rhs[N,K].
#include "mi_epi_table.hpp"

namespace mi {
#define MI_EPI_BT true
const EpiEntry* epi_table_nt(int* n) {
  static const EpiEntry t[] = {MI_EPI_CONFIGS(MI_EPI_ROW)};
  *n = (int)(sizeof(t) / sizeof(t[0]));
  return t;
}
}  // namespace mi
