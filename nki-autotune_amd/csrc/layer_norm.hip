// layer_norm.hip -- mi_layer_norm and mi_layer_norm_backward: argument
// checks, the kernel a call takes, and its launch (kernels: mi_norm.hpp).
#include "mi_capi_internal.hpp"
#include "mi_norm.hpp"

namespace {

using mi::Bf16;
using mi::ColumnSum;
using mi::Fp16;
using mi::LnBwd;
using mi::LnFwd;
using mi::capi::check_overlap;
using mi::capi::fail;
using mi::capi::Range;

constexpr long long kMaxGrid = 1 << 20;  // blocks of one launch; they walk over the rows
constexpr int kLongChunks = 256;         // row chunks of the column sums of long rows

size_t elem_size(int dtype) { return dtype == MI_DTYPE_F32 ? 4 : 2; }

// Bytes from the first to past the last element of `rows` rows of D, a row stride of ld.
size_t span(long long rows, long long ld, int D, size_t elem) {
  return rows > 0 ? ((size_t)(rows - 1) * (size_t)ld + (size_t)D) * elem : 0;
}

int launched(const char* what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? MI_OK : fail(-(int)e, "%s: %s", what, hipGetErrorString(e));
}

// Threads of a block, and as many blocks as the chip holds with the rows'
// values, parameters and next row in registers: each walks over the rows.
template <class T, int E, int L>
void fwd(const LnFwd& p, hipStream_t s) {
  constexpr int ROWS = L <= 64 ? 256 / L : 1, PER_CU = L <= 256 ? 4 : 1024 / L;
  const long long need = (p.rows + ROWS - 1) / ROWS, most = (long long)mi::capi::device_cus() * PER_CU;
  const dim3 grid((unsigned)(need < most ? need : most)), block(ROWS * L);
  if (p.D == E * L) mi::layer_norm_kernel<T, E, L, ROWS, true, (E < 32)><<<grid, block, 0, s>>>(p);
  else mi::layer_norm_kernel<T, E, L, ROWS, false, (E < 32)><<<grid, block, 0, s>>>(p);
}

// Values of a lane and lanes of a row.  16 values a lane past 128: fewer lanes
// to sum over, and a second 16-byte load of bf16 in flight (us of 256 MB of
// rows in and out, 16 values and 8 on twice the lanes: bf16 D = 256 100 and
// 107, 512 101 and 112, 1024 99 and 130, 2048 97 and 120; 4096 108 and 116;
// fp32 within 4 either way).  Up to 64, 8 lanes of 8: 99 and 151 with 16 lanes
// at bf16 D = 64, 154 and 260 at 32; at 128 16 lanes of 8 take 96, 8 of 16 102.
// Past 8192 the values still fit 1024 lanes and the row is read once: 16384
// 110 and 186 in three passes, 28672 143 and 197.
template <class T>
void fwd_run(const LnFwd& p, hipStream_t s) {
  constexpr int V = 16 / (int)sizeof(T);
  const int D = p.D;
  const unsigned rows = (unsigned)(p.rows < kMaxGrid ? p.rows : kMaxGrid);
  if (D < V) mi::layer_norm_long_kernel<T, 64, 1><<<dim3(rows), dim3(64), 0, s>>>(p);
  else if (D <= 64) fwd<T, 8, 8>(p, s);
  else if (D <= 128) fwd<T, 8, 16>(p, s);
  else if (D <= 256) fwd<T, 16, 16>(p, s);
  else if (D <= 512) fwd<T, 16, 32>(p, s);
  else if (D <= 1024) fwd<T, 16, 64>(p, s);
  else if (D <= 2048) fwd<T, 16, 128>(p, s);
  else if (D <= 4096) fwd<T, 16, 256>(p, s);
  else if (D <= 8192) fwd<T, 16, 512>(p, s);
  else if (D <= 16384) fwd<T, 16, 1024>(p, s);
  else if (D <= 32768) fwd<T, 32, 1024>(p, s);
  else mi::layer_norm_long_kernel<T, 1024, V><<<dim3(rows), dim3(1024), 0, s>>>(p);
}

// Rows longer than this, or shorter than 16 bytes, are read more than once
// (bf16 D = 8192 152 us against 282, 16384 168 against 296, of 256 MB each of
// x, dout and dx).
int bwd_most(int dtype) { return dtype == MI_DTYPE_F32 ? 8192 : 16384; }

// Lanes of a row and blocks of the gradient's kernel; each block leaves a row
// of partial sums.  8 values a lane wherever they do: a lane holds their column
// sums beside them (16 on half the lanes: bf16 D = 256 to 4096 5 % slower, fp32
// up to twice, and with 64 rows 9 us for 6).  Rows of up to 128 bytes take 8
// lanes: bf16 D = 32 191 us and 333 with 16, 64 161 and 193; fp32 32 163 and 217,
// but 64 162 and 158.
struct BwdPlan {
  int lanes, blocks;
  bool is_long;
};
BwdPlan bwd_plan(long long rows, int D, int dtype) {
  BwdPlan b;
  const bool f32 = dtype == MI_DTYPE_F32;
  b.is_long = D > bwd_most(dtype) || D < (f32 ? 4 : 8);
  b.lanes = D <= (f32 ? 32 : 64) ? 8 : D <= 128 ? 16 : D <= 256 ? 32 : D <= 512 ? 64 : D <= 1024 ? 128 : D <= 2048 ? 256 : D <= 4096 ? 512 : 1024;
  const int per_block = b.is_long ? 1 : 1024 / b.lanes;
  const long long need = (rows + per_block - 1) / per_block, most = b.is_long ? kLongChunks : mi::capi::device_cus();
  b.blocks = (int)(need < most ? (need > 0 ? need : 1) : most);
  return b;
}

template <class T, int E, int L>
void bwd(const LnBwd& p, const BwdPlan& b, hipStream_t s) {
  const dim3 grid((unsigned)b.blocks), block(1024);
  if (p.D == E * L) mi::layer_norm_bwd_kernel<T, E, L, 1024 / L, true><<<grid, block, 0, s>>>(p);
  else mi::layer_norm_bwd_kernel<T, E, L, 1024 / L, false><<<grid, block, 0, s>>>(p);
}

template <class T>
void bwd_run(const LnBwd& p, const BwdPlan& b, hipStream_t s) {
  const int D = p.D;
  if (b.is_long) {
    const unsigned rows = (unsigned)(p.rows < kMaxGrid ? p.rows : kMaxGrid);
    constexpr int V = 16 / (int)sizeof(T);
    const unsigned chunks = (unsigned)b.blocks;
    if (D < V) {
      if (p.dx) mi::layer_norm_bwd_long_kernel<T, 64, 1><<<dim3(rows), dim3(64), 0, s>>>(p);
      if (p.part) mi::layer_norm_columns_kernel<T, 1><<<dim3(1, chunks), dim3(256), 0, s>>>(p);
    } else {
      if (p.dx) mi::layer_norm_bwd_long_kernel<T, 1024, V><<<dim3(rows), dim3(1024), 0, s>>>(p);
      if (p.part)
        mi::layer_norm_columns_kernel<T, V><<<dim3((unsigned)((D + 256 * V - 1) / (256 * V)), chunks), dim3(256), 0, s>>>(p);
    }
  } else if (D <= 128 / (int)sizeof(T)) bwd<T, 8, 8>(p, b, s);
  else if (D <= 128) bwd<T, 8, 16>(p, b, s);
  else if (D <= 256) bwd<T, 8, 32>(p, b, s);
  else if (D <= 512) bwd<T, 8, 64>(p, b, s);
  else if (D <= 1024) bwd<T, 8, 128>(p, b, s);
  else if (D <= 2048) bwd<T, 8, 256>(p, b, s);
  else if (D <= 4096) bwd<T, 8, 512>(p, b, s);
  else if (D <= 8192) bwd<T, 8, 1024>(p, b, s);
  else if constexpr (sizeof(T) == 2) bwd<T, 16, 1024>(p, b, s);
}

int check_common(long long rows, int D, long long ldx, int dtype) {
  if (rows < 0 || D <= 0) return fail(MI_E_ARGS, "bad size rows=%lld D=%d (D must be positive)", rows, D);
  if (D > 1 << 28) return fail(MI_E_RANGE, "D=%d over %d", D, 1 << 28);  // indexes run a block's stride past D in 32 bits
  if (ldx < 0) return fail(MI_E_ARGS, "negative row stride %lld", ldx);
  if (dtype != MI_DTYPE_BF16 && dtype != MI_DTYPE_F16 && dtype != MI_DTYPE_F32)
    return fail(MI_E_ARGS, "unknown dtype %d", dtype);
  return MI_OK;
}

}  // namespace

extern "C" {

int mi_layer_norm(const mi_layer_norm_args* a, void* stream) {
  if (!a) return fail(MI_E_ARGS, "null arguments");
  const int rc = check_common(a->rows, a->D, a->ldx, a->dtype);
  if (rc != MI_OK) return rc;
  if (!(a->eps >= 0.0f) || a->eps > 3.0e38f) return fail(MI_E_ARGS, "eps must be finite and >= 0");
  if (a->rows == 0) return MI_OK;
  if (!a->x || !a->y) return fail(MI_E_ARGS, "null pointer");
  const size_t es = elem_size(a->dtype), ps = a->params_f32 ? 4 : es;
  const size_t D = (size_t)a->D;
  if ((uintptr_t)a->x % es || (uintptr_t)a->y % es || (uintptr_t)a->weight % ps || (uintptr_t)a->bias % ps ||
      (uintptr_t)a->mean % 4 || (uintptr_t)a->rstd % 4)
    return fail(MI_E_ALIGN, "a pointer is not aligned to its elements");
  const size_t yb = (size_t)a->rows * D * es, sb = (size_t)a->rows * 4;
  const Range in[] = {{a->x, span(a->rows, a->ldx, a->D, es)}, {a->weight, D * ps}, {a->bias, D * ps}},
              out[] = {{a->y, yb}, {a->mean, sb}, {a->rstd, sb}};
  const int orc = check_overlap(out, in);
  if (orc != MI_OK) return orc;
  const LnFwd p = {a->x, a->weight, a->bias, a->y, a->mean, a->rstd, a->rows, a->ldx, a->D, a->eps, a->params_f32 != 0};
  const hipStream_t s = (hipStream_t)stream;
  if (a->dtype == MI_DTYPE_BF16) fwd_run<Bf16>(p, s);
  else if (a->dtype == MI_DTYPE_F16) fwd_run<Fp16>(p, s);
  else fwd_run<float>(p, s);
  return launched("layer norm");
}

int mi_layer_norm_backward_workspace(const mi_layer_norm_grad_args* a, unsigned long long* bytes) {
  if (!a || !bytes) return fail(MI_E_ARGS, "null arguments");
  const int rc = check_common(a->rows, a->D, a->ldx, a->dtype);
  if (rc != MI_OK) return rc;
  const BwdPlan b = bwd_plan(a->rows, a->D, a->dtype);
  *bytes = a->rows > 0 && (a->dweight || a->dbias) ? 2ull * (unsigned long long)b.blocks * (unsigned long long)a->D * 4ull : 0ull;
  return MI_OK;
}

int mi_layer_norm_backward(const mi_layer_norm_grad_args* a, void* workspace, unsigned long long workspace_bytes,
                           void* stream) {
  unsigned long long need = 0;
  const int rc = mi_layer_norm_backward_workspace(a, &need);
  if (rc != MI_OK) return rc;
  if (a->lddout < 0) return fail(MI_E_ARGS, "negative row stride %lld", a->lddout);
  if (!a->dx && !a->dweight && !a->dbias) return MI_OK;
  if (a->rows > 0 && (!a->dout || !a->x || !a->mean || !a->rstd)) return fail(MI_E_ARGS, "null pointer");
  if (need && (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16))
    return fail(MI_E_ARGS, "the call needs %llu bytes of workspace, 16-byte aligned", need);
  const size_t es = elem_size(a->dtype), ps = a->params_f32 ? 4 : es;
  if ((uintptr_t)a->x % es || (uintptr_t)a->dout % es || (uintptr_t)a->dx % es || (uintptr_t)a->weight % ps ||
      (uintptr_t)a->dweight % ps || (uintptr_t)a->dbias % ps || (uintptr_t)a->mean % 4 || (uintptr_t)a->rstd % 4)
    return fail(MI_E_ALIGN, "a pointer is not aligned to its elements");
  const size_t D = (size_t)a->D, sb = (size_t)a->rows * 4;
  const Range in[] = {{a->x, span(a->rows, a->ldx, a->D, es)}, {a->dout, span(a->rows, a->lddout, a->D, es)},
                      {a->weight, D * ps}, {a->mean, sb}, {a->rstd, sb}},
              out[] = {{a->dx, (size_t)a->rows * D * es}, {a->dweight, D * ps}, {a->dbias, D * ps}, {workspace, (size_t)need}};
  const int orc = check_overlap(out, in);
  if (orc != MI_OK) return orc;
  const hipStream_t s = (hipStream_t)stream;
  if (a->rows == 0) {
    // No row to read (the kernels take at least one): the sums are 0.
    for (void* g : {a->dweight, a->dbias}) {
      if (!g) continue;
      const size_t n = D * ps / 2;
      mi::fill_zero_kernel<<<dim3((unsigned)((n + 255) / 256 < 1024 ? (n + 255) / 256 : 1024)), dim3(256), 0, s>>>((uint16_t*)g, n);
      const int zrc = launched("zero gradient");
      if (zrc != MI_OK) return zrc;
    }
    return MI_OK;
  }
  const bool f32 = a->dtype == MI_DTYPE_F32;
  const BwdPlan b = bwd_plan(a->rows, a->D, a->dtype);
  const LnBwd p = {a->dout, a->x,         a->weight, a->mean, a->rstd, a->dx, need ? (float*)workspace : nullptr,
                   a->rows, a->lddout, a->ldx,    a->D,    a->params_f32 != 0};
  if (a->dtype == MI_DTYPE_BF16) bwd_run<Bf16>(p, b, s);
  else if (a->dtype == MI_DTYPE_F16) bwd_run<Fp16>(p, b, s);
  else bwd_run<float>(p, b, s);
  const int lrc = launched("layer norm gradient");
  if (lrc != MI_OK || !need) return lrc;
  const ColumnSum c = {(const float*)workspace, {a->dweight, a->dbias}, b.blocks, a->D, 0};
  if (f32 || a->params_f32) mi::column_sum<float>(c, 2, s);
  else if (a->dtype == MI_DTYPE_BF16) mi::column_sum<Bf16>(c, 2, s);
  else mi::column_sum<Fp16>(c, 2, s);
  return launched("layer norm parameter gradients");
}

}  // extern "C"
