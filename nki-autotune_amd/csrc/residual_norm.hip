// residual_norm.hip -- mi_residual_norm and mi_residual_norm_backward:
// argument checks, the kernel a call takes, and its launch (kernels:
// mi_residual.hpp; instances: residual_norm_{fwd,bwd}.hip).
#include "mi_capi_internal.hpp"
#include "mi_residual_run.hpp"

namespace {

using mi::RnBwd;
using mi::RnColumns;
using mi::RnFwd;
using mi::capi::check_overlap;
using mi::capi::fail;
using mi::capi::Range;

size_t elem_size(int dtype) { return dtype == MI_DTYPE_F32 ? 4 : 2; }

// Bytes from the first to past the last element of `rows` rows of D, a row stride of ld.
size_t span(long long rows, long long ld, int D, size_t elem) {
  return rows > 0 ? ((size_t)(rows - 1) * (size_t)ld + (size_t)D) * elem : 0;
}

int launched(const char* what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? MI_OK : fail(-(int)e, "%s: %s", what, hipGetErrorString(e));
}

int check_common(long long rows, int D, int dtype, long long gates) {
  if (rows < 0 || D <= 0) return fail(MI_E_ARGS, "bad size rows=%lld D=%d (D must be positive)", rows, D);
  if (D > 1 << 28) return fail(MI_E_RANGE, "D=%d over %d", D, 1 << 28);  // indexes run a block's stride past D in 32 bits
  if (rows >= 1ll << 31) return fail(MI_E_RANGE, "rows=%lld over 32 bits", rows);
  if (dtype != MI_DTYPE_BF16 && dtype != MI_DTYPE_F16 && dtype != MI_DTYPE_F32)
    return fail(MI_E_ARGS, "unknown dtype %d", dtype);
  if (gates < 0 || (gates > 0 && rows % gates)) return fail(MI_E_ARGS, "%lld gates do not divide %lld rows", gates, rows);
  return MI_OK;
}
int check_factors(float scale, float eps) {
  if (!(eps >= 0.0f) || eps > 3.0e38f) return fail(MI_E_ARGS, "eps must be finite and >= 0");
  if (!(scale >= -3.0e38f && scale <= 3.0e38f)) return fail(MI_E_ARGS, "scale must be finite");
  return MI_OK;
}

// What the gradient's kernels take of a call.
struct Plan {
  mi::RnBwdPlan k;
  long long gates;            // of the gate (1: for all rows); 0: no gate
  bool own_rows, needs_x;     // a gate of one row each; x is read
  bool sum_w, sum_c;          // the column sums wanted
  size_t part, dots, total;   // bytes of one array of partial sums, of the rows' dots; of the workspace
};
Plan plan_of(const mi_residual_norm_grad_args* a) {
  Plan p = {};
  p.gates = a->gate ? (a->gates > 1 ? a->gates : 1) : 0;
  p.own_rows = p.gates > 1 && p.gates == a->rows;
  p.needs_x = a->gate || a->post_rstd;
  p.sum_w = a->dweight != nullptr;
  p.sum_c = a->dpost_weight || (a->dgate && !p.own_rows);
  // Sums of c are those of one gate's rows each, whichever of the two gradients they are for.
  p.k = mi::rn_bwd_plan(a->rows, a->D, a->dtype, p.gates > 1 && !p.own_rows && p.sum_c ? p.gates : 1);
  const size_t D = (size_t)a->D;
  p.part = (size_t)p.k.blocks * D * 4;
  p.dots = p.k.is_long && p.sum_c ? ((size_t)a->rows * 4 + 15) / 16 * 16 : 0;
  p.total = a->rows > 0 ? p.part * (size_t)(p.sum_w + p.sum_c) + p.dots : 0;
  return p;
}

}  // namespace

extern "C" {

int mi_residual_norm(const mi_residual_norm_args* a, void* stream) {
  if (!a) return fail(MI_E_ARGS, "null arguments");
  int rc = check_common(a->rows, a->D, a->dtype, a->gates);
  if (rc == MI_OK) rc = check_factors(a->scale, a->eps);
  if (rc != MI_OK) return rc;
  if (a->ldx < 0 || a->ldresidual < 0) return fail(MI_E_ARGS, "negative row stride (%lld, %lld)", a->ldx, a->ldresidual);
  if (a->post_weight && !a->post_norm) return fail(MI_E_ARGS, "post_weight without post_norm");
  if (a->rows == 0) return MI_OK;
  if (!a->x || !a->residual || !a->y || !a->hidden) return fail(MI_E_ARGS, "null pointer");
  const size_t es = elem_size(a->dtype), hs = a->stream_f32 ? 4 : es, ps = a->params_f32 ? 4 : es, gs = a->gate_f32 ? 4 : es;
  if ((uintptr_t)a->x % es || (uintptr_t)a->y % es || (uintptr_t)a->residual % hs || (uintptr_t)a->hidden % hs ||
      (uintptr_t)a->weight % ps || (uintptr_t)a->post_weight % ps || (uintptr_t)a->gate % gs || (uintptr_t)a->rstd % 4 ||
      (uintptr_t)a->post_rstd % 4)
    return fail(MI_E_ALIGN, "a pointer is not aligned to its elements");
  const size_t D = (size_t)a->D, n = (size_t)a->rows * D, sb = (size_t)a->rows * 4;
  const size_t gates = a->gates > 1 ? (size_t)a->gates : 1;
  const Range in[] = {{a->x, span(a->rows, a->ldx, a->D, es)}, {a->residual, span(a->rows, a->ldresidual, a->D, hs)},
                      {a->weight, D * ps}, {a->post_weight, D * ps}, {a->gate, gates * D * gs}},
              out[] = {{a->y, n * es}, {a->hidden, n * hs}, {a->rstd, sb}, {a->post_rstd, sb}};
  const int orc = check_overlap(out, in);
  if (orc != MI_OK) return orc;
  const RnFwd p = {a->x, a->residual, a->weight, a->gate, a->post_weight, a->y, a->hidden, a->rstd,
                   a->post_norm ? a->post_rstd : nullptr, a->rows, a->ldx, a->ldresidual, a->D,
                   a->gates > 1 ? (int)(a->rows / a->gates) : 0, a->scale, a->eps, a->params_f32 != 0, a->gate_f32 != 0,
                   a->post_norm != 0};
  mi::rn_fwd_run(p, a->dtype, a->stream_f32 != 0, (hipStream_t)stream);
  return launched("residual norm");
}

int mi_residual_norm_backward_workspace(const mi_residual_norm_grad_args* a, unsigned long long* bytes) {
  if (!a || !bytes) return fail(MI_E_ARGS, "null arguments");
  const int rc = check_common(a->rows, a->D, a->dtype, a->gates);
  if (rc != MI_OK) return rc;
  if (a->gate && a->gates > 1 << 20 && a->gates < a->rows)
    return fail(MI_E_RANGE, "%lld gates of several rows each, over %d", a->gates, 1 << 20);
  *bytes = (unsigned long long)plan_of(a).total;
  return MI_OK;
}

int mi_residual_norm_backward(const mi_residual_norm_grad_args* a, void* workspace, unsigned long long workspace_bytes,
                              void* stream) {
  unsigned long long need = 0;
  int rc = mi_residual_norm_backward_workspace(a, &need);
  if (rc == MI_OK) rc = check_factors(a->scale, 0.0f);
  if (rc != MI_OK) return rc;
  if (a->lddy < 0 || a->lddhidden < 0 || a->ldx < 0 || a->ldhidden < 0) return fail(MI_E_ARGS, "negative row stride");
  if ((a->post_weight || a->dpost_weight) && !a->post_rstd && a->rows > 0)
    return fail(MI_E_ARGS, "post_weight without post_rstd");
  if (a->dgate && !a->gate) return fail(MI_E_ARGS, "dgate without gate");
  if (a->dpost_weight && !a->post_weight) return fail(MI_E_ARGS, "dpost_weight without post_weight");
  const Plan plan = plan_of(a);
  if (a->rows > 0 && (!a->dy || !a->hidden || !a->rstd || !a->dresidual || (plan.needs_x && !a->x)))
    return fail(MI_E_ARGS, "null pointer");
  if (need && (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16))
    return fail(MI_E_ARGS, "the call needs %llu bytes of workspace, 16-byte aligned", need);
  const size_t es = elem_size(a->dtype), hs = a->stream_f32 ? 4 : es, ps = a->params_f32 ? 4 : es, gs = a->gate_f32 ? 4 : es;
  if ((uintptr_t)a->dy % es || (uintptr_t)a->x % es || (uintptr_t)a->dx % es || (uintptr_t)a->dhidden % hs ||
      (uintptr_t)a->hidden % hs || (uintptr_t)a->dresidual % hs || (uintptr_t)a->weight % ps || (uintptr_t)a->dweight % ps ||
      (uintptr_t)a->post_weight % ps || (uintptr_t)a->dpost_weight % ps || (uintptr_t)a->gate % gs ||
      (uintptr_t)a->dgate % gs || (uintptr_t)a->rstd % 4 || (uintptr_t)a->post_rstd % 4)
    return fail(MI_E_ALIGN, "a pointer is not aligned to its elements");
  const size_t D = (size_t)a->D, n = (size_t)a->rows * D, sb = (size_t)a->rows * 4;
  const size_t gates = (size_t)(a->gates > 1 ? a->gates : 1);
  const Range in[] = {{a->dy, span(a->rows, a->lddy, a->D, es)}, {a->dhidden, span(a->rows, a->lddhidden, a->D, hs)},
                      {plan.needs_x ? a->x : nullptr, span(a->rows, a->ldx, a->D, es)},
                      {a->hidden, span(a->rows, a->ldhidden, a->D, hs)}, {a->weight, D * ps}, {a->post_weight, D * ps},
                      {a->gate, gates * D * gs}, {a->rstd, sb}, {a->post_rstd, sb}},
              out[] = {{a->dx, n * es}, {a->dresidual, n * hs}, {a->dweight, D * ps}, {a->dpost_weight, D * ps},
                       {a->dgate, gates * D * gs}, {workspace, (size_t)need}};
  const int orc = check_overlap(out, in);
  if (orc != MI_OK) return orc;
  const hipStream_t s = (hipStream_t)stream;
  if (a->rows == 0) {
    // No row to read (the kernels take at least one): the sums are 0.
    const Range zero[] = {{a->dweight, D * ps}, {a->dpost_weight, D * ps}, {a->dgate, gates * D * gs}};
    for (const Range& z : zero) {
      const size_t halves = z.p ? z.n / 2 : 0;
      if (!halves) continue;
      mi::fill_zero_kernel<<<dim3((unsigned)((halves + 255) / 256 < 1024 ? (halves + 255) / 256 : 1024)), dim3(256), 0, s>>>(
          (uint16_t*)z.p, halves);
      const int zrc = launched("zero gradient");
      if (zrc != MI_OK) return zrc;
    }
    return MI_OK;
  }
  char* ws = (char*)workspace;
  RnBwd p = {};
  p.dy = a->dy;
  p.dhidden = a->dhidden;
  p.x = plan.needs_x ? a->x : nullptr;
  p.hidden = a->hidden;
  p.weight = a->weight;
  p.gate = a->gate;
  p.post_weight = a->post_weight;
  p.rstd = a->rstd;
  p.post_rstd = a->post_rstd;
  p.dx = a->dx;
  p.dresidual = a->dresidual;
  p.dgate = plan.own_rows ? a->dgate : nullptr;
  p.part_w = plan.sum_w ? (float*)ws : nullptr;
  p.part_c = plan.sum_c ? (float*)(ws + (plan.sum_w ? plan.part : 0)) : nullptr;
  p.row_dot = plan.dots ? (float*)(ws + plan.part * (size_t)(plan.sum_w + plan.sum_c)) : nullptr;
  p.rows = a->rows;
  p.lddy = a->lddy;
  p.lddh = a->lddhidden;
  p.ldx = a->ldx;
  p.ldh = a->ldhidden;
  p.D = a->D;
  p.per_gate = plan.gates > 1 ? (int)(a->rows / plan.gates) : 0;
  p.runs = plan.k.runs;
  p.per_run = (int)(a->rows / plan.k.runs);
  p.scale = a->scale;
  p.params_f32 = a->params_f32 != 0;
  p.gate_f32 = a->gate_f32 != 0;
  p.own_gates = plan.own_rows;
  mi::rn_bwd_run(p, plan.k, a->dtype, a->stream_f32 != 0, s);
  const int lrc = launched("residual norm gradient");
  if (lrc != MI_OK || (!plan.sum_w && !plan.sum_c)) return lrc;
  RnColumns c = {p.part_w, p.part_c, a->gate, a->post_weight, a->dweight, a->dpost_weight,
                 plan.own_rows ? nullptr : a->dgate, plan.k.blocks, plan.k.runs, a->D, 0, a->params_f32 != 0,
                 a->gate_f32 != 0, !plan.own_rows, plan.k.runs > 1};
  mi::rn_parameters(c, a->dtype, s);
  return launched("residual norm parameter gradients");
}

}  // extern "C"
