// mi_capi_internal.hpp -- pieces of the C ABI implementation (mi_capi.hip)
// shared with the other translation units of libmi_kernels.so.
#pragma once
#include <stddef.h>

#include "mi_registry.hpp"

namespace mi {
namespace capi {

// Limits of a call: split-K parts, and bytes of device workspace.
constexpr int kMaxSplit = 16;
constexpr unsigned long long kMaxWorkspace = 1ull << 31;
constexpr unsigned long long kMaxOffset = 0xFFFFFFFFull;  // 32-bit buffer offsets

// Bytes that fp32 variant 3 addresses in an operand [K][cols] with blocks of
// `block` columns: a K chunk's rows (at most 32) and a block's width from
// each chunk's descriptor.
inline unsigned long long f32_kw_span(int cols, int K, int block) {
  const unsigned long long rows = (unsigned long long)(K > 32 ? K : 32);
  return (rows * (unsigned long long)cols + (unsigned long long)block) * 4ull;
}

// Tile rows of a raster group: a config's group_m (0: 8), at most those that M
// has.  More are the same one group of all, but the kernels multiply the group
// by the tile columns in 32 bits, where a group of 2^30 wraps to a width of 0
// or less and tiles far outside the output.
inline int raster_group(int group_m, int M, int block_m) {
  const int rows = (int)(((long long)M + block_m - 1) / block_m), group = group_m > 0 ? group_m : 8;
  return group < rows ? group : rows;
}

// Records the message of a failure for mi_last_error on this thread and
// returns `code`.
int fail(int code, const char* fmt, ...);

// Bytes that a call reads or writes.  No output (NULL or empty: none) shares
// one with an input or another output.
struct Range {
  const void* p;
  size_t n;
};
inline bool overlap(const Range& a, const Range& b) {
  return a.p && b.p && a.n && b.n && (uintptr_t)a.p < (uintptr_t)b.p + b.n && (uintptr_t)b.p < (uintptr_t)a.p + a.n;
}
template <size_t NO, size_t NI>
int check_overlap(const Range (&out)[NO], const Range (&in)[NI]) {
  for (size_t i = 0; i < NO; ++i) {
    for (const Range& q : in)
      if (overlap(out[i], q)) return fail(MI_E_ARGS, "an output overlaps an input");
    for (size_t j = 0; j < i; ++j)
      if (overlap(out[i], out[j])) return fail(MI_E_ARGS, "two outputs overlap");
  }
  return MI_OK;
}

// The prebuilt instance of `kernel_id` for cfg's tile parameters and
// variant (split_k and group_m aside), or NULL.
const MiEntry* find(int kernel_id, const mi_tile_cfg& cfg);

// Compute units of the current device (the stream-K grid); kDefaultCus,
// MI355X's count, when no device is visible.
constexpr int kDefaultCus = 256;
int device_cus();

// Whether `variant` of `kernel_id` takes split_k > 1.
bool splittable(int kernel_id, int variant);

// The library default config at a shape (mi_default_config without its
// argument checks; mi_defaults.hip).
int pick_default(int kernel_id, int M, int N, int K, mi_tile_cfg* cfg);
// The fused kernel's default for a call without gamma (mi_defaults.hip).
int pick_default_no_gamma(int M, int N, int K, mi_tile_cfg* cfg);

// The body of mi_matmul_lhsT_rhs_bf16.  fixed_ws == NULL: a call that needs
// device workspace takes it from the library's stream-ordered pool;
// otherwise fixed_ws (fixed_cap bytes, 256-byte aligned) is the workspace
// and a config needing more is rejected with MI_E_RANGE.  fixed_zeroed: the
// stream-K counters at its start are known to be 0.
int matmul_lhsT_rhs_bf16(const void* lhsT, const void* rhs, void* out, int M, int N, int K, const mi_tile_cfg* cfg,
                         void* stream, char* fixed_ws, size_t fixed_cap, bool fixed_zeroed = true);

}  // namespace capi
}  // namespace mi
