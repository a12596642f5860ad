// newton_schulz.hip -- mi_newton_schulz: argument checks, workspace, and the
// launches of its products (mi_ns.hpp).
#include "mi_capi_internal.hpp"
#include "mi_norm.hpp"
#include "mi_ns.hpp"

namespace {

using mi::Bf16;
using mi::NsMM;
using mi::NsOut;
using mi::capi::fail;

constexpr int kNormBlocks = 256;  // blocks of one matrix's sum of squares

// part[z][block] = the sum of squares of a share of G_z, in 64 bits (the
// squares of small gradients leave fp32's range).  16 bytes a load, at any
// address; block 0 also has the last n % V values.  4096 x 4096 bf16: 15 us
// (value by value 61).
template <class T>
__global__ __launch_bounds__(256) void ns_square_kernel(const T* __restrict__ g, double* __restrict__ part, long long n) {
  __shared__ double xs[4];
  constexpr int V = mi::Pack<T>::V, U = 4;
  const T* p = g + (size_t)blockIdx.y * (size_t)n;
  const long long packs = n / V, step = (long long)gridDim.x * 256;
  double s = 0.0;
  for (long long i0 = (long long)blockIdx.x * 256 + threadIdx.x; i0 < packs; i0 += U * step) {
    mi::Pack<T> v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = mi::load_pack(p + (i0 + u * step < packs ? i0 + u * step : i0) * V);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i0 + u * step >= packs) break;
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const double x = (double)mi::to_f32(v[u].v[k]);
        s += x * x;
      }
    }
  }
  const long long rest = packs * V + threadIdx.x;
  if (blockIdx.x == 0 && rest < n) {
    const double x = (double)mi::to_f32(p[rest]);
    s += x * x;
  }
#pragma unroll
  for (int k = 32; k > 0; k >>= 1) s += __shfl_xor(s, k);
  if ((threadIdx.x & 63) == 0) xs[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) part[(size_t)blockIdx.y * gridDim.x + blockIdx.x] = ((xs[0] + xs[1]) + xs[2]) + xs[3];
}

// X_0 = G / (||G|| + eps), or of G^T: 64 x 64 pieces, turned in LDS.  G
// [m][n]; X [s][2 * lp] (hi and lo by 32), s x l of it G's or G^T's, the rest
// zeros.
struct NsInit {
  const void* g;
  uint16_t* x;
  const double* part;
  int parts, m, n, s, l, lp;
  float eps;
  bool turn;
};
template <class T>
__global__ __launch_bounds__(256) void ns_init_kernel(const NsInit p) {
  __shared__ float tile[64][65];
  __shared__ double scale_lds;
  const int tid = (int)threadIdx.x, z = (int)blockIdx.z;
  const T* g = (const T*)p.g + (size_t)z * (size_t)p.m * (size_t)p.n;
  const int r0 = (int)blockIdx.y * 64, c0 = (int)blockIdx.x * 64;  // of X
  const int row0 = p.turn ? c0 : r0, col0 = p.turn ? r0 : c0;      // of G
  // 8 values a load, at any address: two a thread, on their way while the
  // parts are added up.
  mi::Pack<T, 8> in[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int row = row0 + tid / 8 + 32 * j, col = col0 + tid % 8 * 8;
    const T* at = g + (size_t)row * (size_t)p.n + col;
    in[j] = mi::Pack<T, 8>{};
    if (row < p.m && col + 8 <= p.n) {
      in[j] = mi::load_pack<T, 8>(at);
    } else if (row < p.m) {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (col + k < p.n) in[j].v[k] = at[k];
    }
  }
  if (tid < 64) {
    // The parts' sum, in an order fixed by their number.
    double t[kNormBlocks / 64];
#pragma unroll
    for (int i = 0; i < kNormBlocks / 64; ++i)
      t[i] = tid + 64 * i < p.parts ? p.part[(size_t)z * p.parts + tid + 64 * i] : 0.0;
    double sum = (t[0] + t[1]) + (t[2] + t[3]);
    for (int k = 32; k > 0; k >>= 1) sum += __shfl_xor(sum, k);
    if (tid == 0) scale_lds = 1.0 / (__builtin_sqrt(sum) + (double)p.eps);
  }
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int a = tid / 8 + 32 * j, b = tid % 8 * 8 + k;
      const float v = mi::to_f32(in[j].v[k]);
      if (p.turn) tile[b][a] = v;
      else tile[a][b] = v;
    }
  __syncthreads();
  // A scale that fp32 holds in full, or, of a norm under 2^-128 or past 2^126,
  // one that it does not, in 64 bits.
  const double exact = scale_lds;
  const float scale = (float)exact;
  const bool held = scale >= 0x1p-126f && scale <= 0x1.fffffep127f;
  uint16_t* x = p.x + (size_t)z * (size_t)p.s * (size_t)(2 * p.lp);
  for (int i = tid; i < 64 * 8; i += 256) {
    const int r = i / 8, c = (i % 8) * 8;
    if (r0 + r >= p.s || c0 + c >= p.lp) continue;
    float v[8], t[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = held ? tile[r][c + k] * scale : (float)((double)tile[r][c + k] * exact);
    const mi::u32x4_t hi = mi::pack8(v);
    mi::unpack8(hi, t);
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] -= t[k];
    uint16_t* at = x + (size_t)(r0 + r) * (size_t)(2 * p.lp) + mi::ns_at(c0 + c);
    *(mi::u32x4_t*)at = hi;
    *(mi::u32x4_t*)(at + 32) = mi::pack8(v);
  }
}

// A [s][2 * sp] = the sum of ns_split_kernel's parts, in their order: a block
// of 64 x 64 on or above the diagonal, and the same turned below it.
__global__ __launch_bounds__(256) void ns_sum_kernel(const float* __restrict__ ws, uint16_t* __restrict__ a, int parts,
                                                     int s, int sp) {
  __shared__ float tile[64][65];
  const int tid = (int)threadIdx.x, w = (int)blockIdx.x;
  int tn = (int)((__builtin_sqrtf(8.0f * (float)w + 1.0f) - 1.0f) * 0.5f);
  while (tn * (tn + 1) / 2 > w) --tn;
  while ((tn + 1) * (tn + 2) / 2 <= w) ++tn;
  const int m0 = (w - tn * (tn + 1) / 2) * 64, n0 = tn * 64;
  const size_t stride = (size_t)s * (size_t)sp;
  const float* part = ws + (size_t)blockIdx.y * (size_t)parts * stride;
  uint16_t* out = a + (size_t)blockIdx.y * 2 * stride;
  const auto store = [&](int row, int col, const float(&v)[8]) __attribute__((always_inline)) {
    float t[8];
    const mi::u32x4_t hi = mi::pack8(v);
    mi::unpack8(hi, t);
#pragma unroll
    for (int k = 0; k < 8; ++k) t[k] = v[k] - t[k];
    uint16_t* at = out + (size_t)row * (size_t)(2 * sp) + mi::ns_at(col);
    *(mi::u32x4_t*)at = hi;
    *(mi::u32x4_t*)(at + 32) = mi::pack8(t);
  };
  const int c = tid % 8 * 8;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int r = tid / 8 + 32 * j;
    float v[8] = {};
    if (m0 + r < s && n0 + c < sp) {
      const float* at = part + (size_t)(m0 + r) * (size_t)sp + n0 + c;
      const mi::f32x4_t lo = mi::sum_in_order<0>((const mi::f32x4_t*)at, stride, parts);
      const mi::f32x4_t hi = mi::sum_in_order<0>((const mi::f32x4_t*)(at + 4), stride, parts);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        v[k] = lo[k];
        v[4 + k] = hi[k];
      }
      store(m0 + r, n0 + c, v);
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) tile[r][c + k] = v[k];
  }
  if (m0 == n0) return;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int r = tid / 8 + 32 * j;
    float v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = tile[c + k][r];
    if (n0 + r < s && m0 + c < sp) store(n0 + r, m0 + c, v);
  }
}

// out [m][n] from the hi values of X [s][2 * lp], turned back where G was: hi
// is the value rounded to bf16.
__global__ __launch_bounds__(256) void ns_last_kernel(const uint16_t* __restrict__ x, uint16_t* __restrict__ out, int m,
                                                      int n, int s, int lp, bool turn) {
  __shared__ uint16_t tile[64][66];
  const int tid = (int)threadIdx.x, z = (int)blockIdx.z;
  const int r0 = (int)blockIdx.y * 64, c0 = (int)blockIdx.x * 64;  // of out
  const uint16_t* src = x + (size_t)z * (size_t)s * (size_t)(2 * lp);
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int a = tid / 8 + 32 * j, b = tid % 8 * 8;
    const int row = (turn ? c0 : r0) + a, col = (turn ? r0 : c0) + b;  // of X
    mi::Pack<uint16_t> v = {};
    if (row < s && col < lp) v = mi::load_pack(src + (size_t)row * (size_t)(2 * lp) + mi::ns_at(col));
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if (turn) tile[b + k][a] = v.v[k];
      else tile[a][b + k] = v.v[k];
    }
  }
  __syncthreads();
  uint16_t* dst = out + (size_t)z * (size_t)m * (size_t)n;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int a = tid / 8 + 32 * j, b = tid % 8 * 8, r = r0 + a, c = c0 + b;
    if (r >= m || c >= n) continue;
    uint16_t* to = dst + (size_t)r * (size_t)n + c;
    mi::Pack<uint16_t> v;
#pragma unroll
    for (int k = 0; k < 8; ++k) v.v[k] = tile[a][b + k];
    if (c + 8 <= n) {
      *(mi::Pack<uint16_t>*)to = v;
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (c + k < n) to[k] = v.v[k];
    }
  }
}

int launched(const char* what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? MI_OK : fail(-(int)e, "%s: %s", what, hipGetErrorString(e));
}

size_t up256(size_t v) { return (v + 255) / 256 * 256; }

struct Plan {
  int s, l, sp, lp, parts;
  int split;  // parts of X X^T (1: none)
  bool turn;
  size_t x1, a, b, part, gram, bytes;
};
int gram_parts(int s, int sp, int lp, int batch);
int ns_plan(const mi_newton_schulz_args* p, Plan* q) {
  if (p->batch < 0 || p->m < 0 || p->n < 0) return fail(MI_E_ARGS, "negative size batch=%d m=%d n=%d", p->batch, p->m, p->n);
  if (p->steps < 0) return fail(MI_E_ARGS, "steps=%d negative", p->steps);
  if (p->dtype != MI_DTYPE_BF16 && p->dtype != MI_DTYPE_F32) return fail(MI_E_ARGS, "grad must be bf16 or fp32");
  if (!(p->eps >= 0.0f) || p->eps > 3.0e38f) return fail(MI_E_ARGS, "eps must be finite and >= 0");
  if (p->batch > 65535) return fail(MI_E_RANGE, "batch=%d over 65535", p->batch);
  *q = Plan{};
  if (p->batch == 0 || p->m == 0 || p->n == 0) return MI_OK;
  q->turn = p->m > p->n;
  q->s = q->turn ? p->n : p->m;
  q->l = q->turn ? p->m : p->n;
  // A matrix's planes, and a block of rows past them, within 32-bit offsets.
  const unsigned long long lp = ((unsigned long long)q->l + 31) / 32 * 32;
  if (((unsigned long long)q->s + 512) * lp * 4 > mi::capi::kMaxOffset)
    return fail(MI_E_RANGE, "the planes of a %d x %d matrix exceed 32-bit buffer offsets", p->m, p->n);
  if (q->l > 1 << 20) return fail(MI_E_RANGE, "a side of %d exceeds %d", q->l, 1 << 20);
  q->lp = (int)lp;
  q->sp = (q->s + 31) / 32 * 32;
  const long long n = (long long)p->m * p->n;
  q->parts = (int)(n / 2048 < 1 ? 1 : n / 2048 > kNormBlocks ? kNormBlocks : n / 2048);
  const size_t x = up256((size_t)p->batch * q->s * q->lp * 4), a = up256((size_t)p->batch * q->s * q->sp * 4);
  q->x1 = x;
  q->a = 2 * x;
  q->b = q->a + a;
  q->part = q->b + a;
  q->gram = q->part + up256((size_t)p->batch * q->parts * 8);
  q->split = p->steps > 0 ? gram_parts(q->s, q->sp, q->lp, p->batch) : 1;
  q->bytes = q->gram + (q->split > 1 ? up256((size_t)p->batch * q->split * q->s * q->sp * 4) : 0);
  return MI_OK;
}

template <int BM, int BN, int W, int S, bool BT, bool SYM>
int product(const NsMM& p, const NsOut& o, int batch, hipStream_t s) {
  const unsigned tm = (unsigned)((p.M + BM - 1) / BM), tn = (unsigned)((p.N + BN - 1) / BN);
  mi::ns_product_kernel<BM, BN, W, S, BT, SYM>
      <<<dim3(SYM ? tn * (tn + 1) / 2 : tm * tn, (unsigned)batch), dim3(W * 64), 0, s>>>(p, o);
  return launched("Newton-Schulz product");
}
// Which block a product takes: the least estimated time, a K tile of a block
// alone on its unit (`alone`) or of one of several (`shared`), and a block's
// ends, in microseconds, fitted to five steps timed at 15 sizes from 128 x 128
// to 4096 x 4096 and 32 of 512 x 512.  Small blocks fill the chip where there
// are few (1024 x 1024: 182 us with 64-wide blocks, 301 with 128), large ones
// read their operands less often (4096 x 4096: 5.55 ms with 64, 4.05 with 192
// and 256).  The choice was within 1.06 of the fastest of each size.
struct NsBlock {
  int bm, per_cu;
  double alone, shared, ends;
};
double estimate(const NsBlock& b, long long blocks, int kts, int cus) {
  const long long each = (blocks + cus - 1) / cus, rounds = (each + b.per_cu - 1) / b.per_cu;
  const double in_line = (double)each * b.shared * kts, alone = (double)rounds * b.alone * kts;
  return (in_line > alone ? in_line : alone) + (double)rounds * b.ends;
}
template <size_t N>
int fastest(const NsBlock (&b)[N], const NsMM& p, bool sym, int batch) {
  const int cus = mi::capi::device_cus();
  int best = 0;
  double least = 1e30;
  for (size_t i = 0; i < N; ++i) {
    const long long tm = (p.M + b[i].bm - 1) / b[i].bm, tn = (p.N + b[i].bm - 1) / b[i].bm;
    const double us = estimate(b[i], batch * (sym ? tn * (tn + 1) / 2 : tm * tn), p.kw / 32, cus);
    if (us < least) {
      least = us;
      best = b[i].bm;
    }
  }
  return best;
}
constexpr NsBlock kSymmetric[] = {
    {64, 2, 0.205, 0.235, 3.875}, {128, 1, 0.538, 0.467, 6.619}, {192, 1, 0.949, 1.036, 12.722}};
// How many parts X X^T is split into: as many as the least estimated time
// takes, a part of at least 4 K tiles; parts cost a second launch and their
// products written and read.  Five steps of 640 x 6000 take 227 us in 4 parts
// and 319 unsplit, 64 x 2048 77 in 8 and 109, 2001 x 777 185 in 2 and 195; of
// 1024 x 4096, whose blocks take more than half the units, 331 in 4 and 328,
// 1000 x 3000 303 and 287.
int gram_parts(int s, int sp, int lp, int batch) {
  const int cus = mi::capi::device_cus(), kts = lp / 32;
  double least = 1e30;
  for (const NsBlock& b : kSymmetric) {
    const long long t = (sp + b.bm - 1) / b.bm;
    const double us = estimate(b, batch * (t * (t + 1) / 2), kts, cus);
    if (us < least) least = us;
  }
  int best = 1;
  const long long t = (sp + 63) / 64, tri = t * (t + 1) / 2;
  for (const int parts : {2, 4, 8}) {
    const int each = (kts + parts - 1) / parts;
    const double bytes = (double)batch * parts * s * sp * 4.0;
    if (each < 4 || (parts - 1) * each >= kts || bytes > (double)mi::capi::kMaxWorkspace) break;
    const double us = estimate(kSymmetric[0], batch * tri * parts, each, cus) + 5.0 + bytes / 2.5e6;
    if (us < least) {
      least = us;
      best = parts;
    }
  }
  return best;
}
int split_gram(const NsMM& p, uint16_t* a, float* ws, int parts, int batch, hipStream_t s) {
  const unsigned t = (unsigned)((p.N + 63) / 64), tri = t * (t + 1) / 2;
  mi::ns_split_kernel<64, 4, 4><<<dim3(tri * (unsigned)parts, (unsigned)batch), dim3(256), 0, s>>>(p, ws, parts);
  const int rc = launched("parts of a Newton-Schulz product");
  if (rc != MI_OK) return rc;
  ns_sum_kernel<<<dim3(tri, (unsigned)batch), dim3(256), 0, s>>>(ws, a, parts, p.M, p.N);
  return launched("sum of the parts");
}
int symmetric(const NsMM& p, const NsOut& o, int batch, hipStream_t s) {
  switch (fastest(kSymmetric, p, true, batch)) {
    case 64: return product<64, 64, 4, 4, true, true>(p, o, batch, s);
    case 128: return product<128, 128, 4, 4, true, true>(p, o, batch, s);
    default: return product<192, 192, 4, 3, true, true>(p, o, batch, s);
  }
}
int update(const NsMM& p, const NsOut& o, int batch, hipStream_t s) {
  static constexpr NsBlock blocks[] = {
      {64, 2, 0.219, 0.178, 6.251}, {128, 2, 0.543, 0.597, 6.950}, {256, 1, 1.478, 1.533, 11.596}};
  switch (fastest(blocks, p, false, batch)) {
    case 64: return product<64, 64, 4, 4, false, false>(p, o, batch, s);
    case 128: return product<128, 128, 4, 2, false, false>(p, o, batch, s);
    default: return product<256, 256, 8, 2, false, false>(p, o, batch, s);
  }
}

}  // namespace

extern "C" {

int mi_newton_schulz_workspace(const mi_newton_schulz_args* args, unsigned long long* bytes) {
  if (!args || !bytes) return fail(MI_E_ARGS, "null arguments");
  Plan q;
  const int rc = ns_plan(args, &q);
  *bytes = rc == MI_OK ? q.bytes : 0;
  return rc;
}

int mi_newton_schulz(const mi_newton_schulz_args* args, void* workspace, unsigned long long workspace_bytes, void* stream) {
  if (!args) return fail(MI_E_ARGS, "null arguments");
  Plan q;
  int rc = ns_plan(args, &q);
  if (rc != MI_OK || q.bytes == 0) return rc;
  const int m = args->m, n = args->n, batch = args->batch;
  const size_t es = args->dtype == MI_DTYPE_F32 ? 4 : 2, total = (size_t)batch * m * n;
  if (!args->grad || !args->out) return fail(MI_E_ARGS, "null pointer");
  if (!workspace || workspace_bytes < q.bytes || (uintptr_t)workspace % 16)
    return fail(MI_E_ARGS, "the call needs %zu bytes of workspace, 16-byte aligned", q.bytes);
  if ((uintptr_t)args->grad % es || (uintptr_t)args->out % 2) return fail(MI_E_ALIGN, "a pointer is not aligned to its elements");
  const mi::capi::Range in[] = {{args->grad, total * es}}, outs[] = {{args->out, total * 2}, {workspace, q.bytes}};
  if ((rc = mi::capi::check_overlap(outs, in)) != MI_OK) return rc;
  const hipStream_t st = (hipStream_t)stream;
  char* ws = (char*)workspace;
  double* part = (double*)(ws + q.part);
  uint16_t *x = (uint16_t*)ws, *next = (uint16_t*)(ws + q.x1), *A = (uint16_t*)(ws + q.a), *B = (uint16_t*)(ws + q.b);
  const long long per = (long long)m * n;
  const dim3 sq((unsigned)q.parts, (unsigned)batch);
  const NsInit init = {args->grad, x, part, q.parts, m, n, q.s, q.l, q.lp, args->eps, q.turn};
  const dim3 ig((unsigned)((q.lp + 63) / 64), (unsigned)((q.s + 63) / 64), (unsigned)batch);
  if (args->dtype == MI_DTYPE_F32) {
    ns_square_kernel<float><<<sq, dim3(256), 0, st>>>((const float*)args->grad, part, per);
    if ((rc = launched("sum of squares")) != MI_OK) return rc;
    ns_init_kernel<float><<<ig, dim3(256), 0, st>>>(init);
  } else {
    ns_square_kernel<Bf16><<<sq, dim3(256), 0, st>>>((const Bf16*)args->grad, part, per);
    if ((rc = launched("sum of squares")) != MI_OK) return rc;
    ns_init_kernel<Bf16><<<ig, dim3(256), 0, st>>>(init);
  }
  if ((rc = launched("first iterate")) != MI_OK) return rc;
  const int s = q.s, sp = q.sp, lp = q.lp;
  const uint32_t xb = (uint32_t)((size_t)s * lp * 4), ab = (uint32_t)((size_t)s * sp * 4);
  const long long xz = (long long)s * lp * 2, az = (long long)s * sp * 2;
  const bool direct = !q.turn && n == lp && (uintptr_t)args->out % 16 == 0;  // the last product stores out itself
  for (int k = 0; k < args->steps; ++k) {
    const NsMM gram = {x, x, xb, xb, s, sp, lp, lp, lp, xz, xz};
    const NsOut to_a = {nullptr, A, nullptr, s, sp, 1.0f, 0.0f, 0, az, 0};
    rc = q.split > 1 ? split_gram(gram, A, (float*)(ws + q.gram), q.split, batch, st) : symmetric(gram, to_a, batch, st);
    if (rc != MI_OK) return rc;
    const NsMM square = {A, A, ab, ab, s, sp, sp, sp, sp, az, az};
    const NsOut to_b = {A, B, nullptr, s, sp, args->c, args->b, az, az, 0};
    if ((rc = symmetric(square, to_b, batch, st)) != MI_OK) return rc;
    const NsMM by_b = {B, x, ab, xb, s, lp, sp, sp, lp, az, xz};
    const bool last = direct && k + 1 == args->steps;
    const NsOut to_x = {x, last ? nullptr : next, last ? (uint16_t*)args->out : nullptr, s, lp, 1.0f, args->a, xz, xz, per};
    if ((rc = update(by_b, to_x, batch, st)) != MI_OK) return rc;
    uint16_t* t = x;
    x = next;
    next = t;
    if (last) return MI_OK;
  }
  const dim3 lg((unsigned)((n + 63) / 64), (unsigned)((m + 63) / 64), (unsigned)batch);
  ns_last_kernel<<<lg, dim3(256), 0, st>>>(x, (uint16_t*)args->out, m, n, s, lp, q.turn);
  return launched("last iterate");
}

}  // extern "C"
