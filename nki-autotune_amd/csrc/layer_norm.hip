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
using mi::capi::fail;

constexpr long long kMaxGrid = 1 << 20;  // blocks of one launch; they walk over the rows
constexpr int kLongChunks = 64;          // row chunks of the column sums of long rows

size_t elem_size(int dtype) { return dtype == MI_DTYPE_F32 ? 4 : 2; }

bool overlap(const void* p, size_t pb, const void* q, size_t qb) {
  return p && q && pb && qb && (uintptr_t)p < (uintptr_t)q + qb && (uintptr_t)q < (uintptr_t)p + pb;
}

// Bytes from the first to past the last element of `rows` rows of D, a row stride of ld.
size_t span(long long rows, long long ld, int D, size_t elem) {
  return rows > 0 ? ((size_t)(rows - 1) * (size_t)ld + (size_t)D) * elem : 0;
}

// Every row of p starts on 16 bytes (or there is no p).
bool rows_16(const void* p, long long ld, size_t elem) {
  return !p || ((uintptr_t)p % 16 == 0 && (size_t)ld * elem % 16 == 0);
}

int launched(const char* what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? MI_OK : fail(-(int)e, "%s: %s", what, hipGetErrorString(e));
}

template <class T, int VW, int E, int WPR>
void fwd(const LnFwd& p, hipStream_t s) {
  constexpr int RPB = WPR == 1 ? 4 : 1;
  const long long blocks = (p.rows + RPB - 1) / RPB;
  mi::layer_norm_kernel<T, VW, E, WPR>
      <<<dim3((unsigned)(blocks < kMaxGrid ? blocks : kMaxGrid)), dim3(WPR == 1 ? 256 : WPR * 64), 0, s>>>(p);
}

template <class T, int VW>
void fwd_pick(const LnFwd& p, hipStream_t s) {
  const int D = p.D;
  if (D <= 512) fwd<T, VW, 8, 1>(p, s);
  else if (D <= 1024) fwd<T, VW, 16, 1>(p, s);
  else if (D <= 2048) fwd<T, VW, 8, 4>(p, s);
  else if (D <= 4096) fwd<T, VW, 16, 4>(p, s);
  else if (VW == 1 && D <= 8192) fwd<T, 1, 8, 16>(p, s);
  else if (VW > 1 && D <= 8192) fwd<T, 16 / sizeof(T), 32, 4>(p, s);
  else if (VW > 1 && D <= 16384) fwd<T, 16 / sizeof(T), 16, 16>(p, s);
  else if (VW > 1 && D <= 32768) fwd<T, 16 / sizeof(T), 32, 16>(p, s);
  else mi::layer_norm_long_kernel<T><<<dim3((unsigned)(p.rows < kMaxGrid ? p.rows : kMaxGrid)), dim3(1024), 0, s>>>(p);
}

template <class T>
void fwd_run(const LnFwd& p, bool vec, hipStream_t s) {
  if (vec) fwd_pick<T, 16 / sizeof(T)>(p, s);
  else fwd_pick<T, 1>(p, s);
}

// Blocks of the gradient's kernel: each leaves a row of partial sums.
struct BwdPlan {
  int rows_per_block, blocks;
  bool is_long;
};
BwdPlan bwd_plan(long long rows, int D, int dtype, bool vec) {
  BwdPlan b;
  b.is_long = D > (vec ? 16384 : 8192);
  b.rows_per_block = D <= (vec && dtype == MI_DTYPE_BF16 ? 4096 : 2048) ? 8 : 1;
  const long long most = b.is_long ? kLongChunks : b.rows_per_block == 8 ? 256 : 512;
  const long long need = (rows + b.rows_per_block - 1) / b.rows_per_block;
  b.blocks = (int)(need < most ? (need > 0 ? need : 1) : most);
  return b;
}

template <class T, int VW, int E, int WPR>
void bwd(const LnBwd& p, const BwdPlan& b, hipStream_t s) {
  constexpr int WAVES = WPR == 1 ? 8 : WPR;
  mi::layer_norm_bwd_kernel<T, VW, E, WPR, WAVES><<<dim3((unsigned)b.blocks), dim3(WAVES * 64), 0, s>>>(p);
}

template <class T, int VW>
void bwd_pick(const LnBwd& p, const BwdPlan& b, hipStream_t s) {
  const int D = p.D;
  if (b.is_long) {
    if (p.dx)
      mi::layer_norm_bwd_long_kernel<T><<<dim3((unsigned)(p.rows < kMaxGrid ? p.rows : kMaxGrid)), dim3(1024), 0, s>>>(p);
    if (p.part)
      mi::layer_norm_columns_kernel<T><<<dim3((unsigned)((D + 255) / 256), (unsigned)b.blocks), dim3(256), 0, s>>>(p);
  } else if (b.rows_per_block == 8) {
    if (D <= 512) bwd<T, VW, 8, 1>(p, b, s);
    else if (D <= 1024) bwd<T, VW, 16, 1>(p, b, s);
    else if (D <= 2048) bwd<T, VW, 32, 1>(p, b, s);
    else if constexpr (VW > 1 && std::is_same_v<T, Bf16>) bwd<T, VW, 64, 1>(p, b, s);
  } else {
    if (D <= 4096) {
      if constexpr (VW == 1 || !std::is_same_v<T, Bf16>) bwd<T, VW, 8, 8>(p, b, s);
    } else if (D <= 8192) bwd<T, VW, 16, 8>(p, b, s);
    else if constexpr (VW > 1) bwd<T, VW, 32, 8>(p, b, s);
  }
}

template <class T>
void bwd_run(const LnBwd& p, const BwdPlan& b, bool vec, hipStream_t s) {
  if (vec) bwd_pick<T, 16 / sizeof(T)>(p, b, s);
  else bwd_pick<T, 1>(p, b, s);
}

// Whether every row of the gradient's operands can be read 16 bytes at a time.
bool bwd_vec(const mi_layer_norm_grad_args* a) {
  const size_t es = elem_size(a->dtype), ps = a->params_f32 ? 4 : es;
  return rows_16(a->x, a->ldx, es) && rows_16(a->dout, a->lddout, es) && rows_16(a->dx, a->D, es) &&
         rows_16(a->weight, 0, ps) && (size_t)a->D * es % 16 == 0;
}

int check_common(long long rows, int D, long long ldx, int dtype) {
  if (rows < 0 || D <= 0) return fail(MI_E_ARGS, "bad size rows=%lld D=%d (D must be positive)", rows, D);
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
  if (overlap(a->y, yb, a->x, span(a->rows, a->ldx, a->D, es)) || overlap(a->y, yb, a->weight, D * ps) ||
      overlap(a->y, yb, a->bias, D * ps) || overlap(a->y, yb, a->mean, sb) || overlap(a->y, yb, a->rstd, sb))
    return fail(MI_E_ARGS, "y overlaps another operand");
  const LnFwd p = {a->x, a->weight, a->bias, a->y, a->mean, a->rstd, a->rows, a->ldx, a->D, a->eps, a->params_f32 != 0};
  const bool vec = rows_16(a->x, a->ldx, es) && rows_16(a->y, a->D, es) && rows_16(a->weight, 0, ps) &&
                   rows_16(a->bias, 0, ps);
  const hipStream_t s = (hipStream_t)stream;
  if (a->dtype == MI_DTYPE_BF16) fwd_run<Bf16>(p, vec, s);
  else if (a->dtype == MI_DTYPE_F16) fwd_run<Fp16>(p, vec, s);
  else fwd_run<float>(p, vec, s);
  return launched("layer norm");
}

int mi_layer_norm_backward_workspace(const mi_layer_norm_grad_args* a, unsigned long long* bytes) {
  if (!a || !bytes) return fail(MI_E_ARGS, "null arguments");
  const int rc = check_common(a->rows, a->D, a->ldx, a->dtype);
  if (rc != MI_OK) return rc;
  const BwdPlan b = bwd_plan(a->rows, a->D, a->dtype, bwd_vec(a));
  *bytes = a->dweight || a->dbias ? 2ull * (unsigned long long)b.blocks * (unsigned long long)a->D * 4ull : 0ull;
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
  const struct {
    const void* p;
    size_t n;
  } in[] = {{a->x, span(a->rows, a->ldx, a->D, es)},
            {a->dout, span(a->rows, a->lddout, a->D, es)},
            {a->weight, D * ps},
            {a->mean, sb},
            {a->rstd, sb}},
    out[] = {{a->dx, (size_t)a->rows * D * es}, {a->dweight, D * ps}, {a->dbias, D * ps}, {workspace, (size_t)need}};
  for (int i = 0; i < 4; ++i) {
    for (const auto& q : in)
      if (overlap(out[i].p, out[i].n, q.p, q.n)) return fail(MI_E_ARGS, "an output overlaps an input");
    for (int j = 0; j < i; ++j)
      if (overlap(out[i].p, out[i].n, out[j].p, out[j].n)) return fail(MI_E_ARGS, "two outputs overlap");
  }
  const bool f32 = a->dtype == MI_DTYPE_F32;
  const bool vec = bwd_vec(a);
  const BwdPlan b = bwd_plan(a->rows, a->D, a->dtype, vec);
  const LnBwd p = {a->dout, a->x,         a->weight, a->mean, a->rstd, a->rows > 0 ? a->dx : nullptr, need ? (float*)workspace : nullptr,
                   a->rows, a->lddout, a->ldx,    a->D,    a->params_f32 != 0};
  const hipStream_t s = (hipStream_t)stream;
  if (a->dtype == MI_DTYPE_BF16) bwd_run<Bf16>(p, b, vec, s);
  else if (a->dtype == MI_DTYPE_F16) bwd_run<Fp16>(p, b, vec, s);
  else bwd_run<float>(p, b, vec, s);
  const int lrc = launched("layer norm gradient");
  if (lrc != MI_OK || !need) return lrc;
  const ColumnSum c = {(const float*)workspace, {a->dweight, a->dbias}, b.blocks, a->D};
  const dim3 grid((unsigned)((a->D + 63) / 64), 2);
  if (f32 || a->params_f32) mi::column_sum_kernel<float><<<grid, dim3(1024), 0, s>>>(c);
  else if (a->dtype == MI_DTYPE_BF16) mi::column_sum_kernel<Bf16><<<grid, dim3(1024), 0, s>>>(c);
  else mi::column_sum_kernel<Fp16><<<grid, dim3(1024), 0, s>>>(c);
  return launched("layer norm parameter gradients");
}

}  // extern "C"
