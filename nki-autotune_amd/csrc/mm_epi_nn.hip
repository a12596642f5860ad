// Instances of the epilogue products with rhs[K,N].
#include "mi_epi_table.hpp"

namespace mi {
#define MI_EPI_BT false
const EpiEntry* epi_table_nn(int* n) {
  static const EpiEntry t[] = {MI_EPI_CONFIGS(MI_EPI_ROW)};
  *n = (int)(sizeof(t) / sizeof(t[0]));
  return t;
}
}  // namespace mi
