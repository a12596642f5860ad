// matmul_epilogue.hip -- mi_matmul_epilogue_bf16 and its gradient: argument
// checks, the config a call takes, workspaces and launches (products:
// mi_mm_epi.hpp).
#include <cmath>

#include "mi_capi_internal.hpp"
#include "mi_epi_table.hpp"
#include "mi_mm_any.hpp"
#include "mi_norm.hpp"

namespace {

using mi::AnyMM;
using mi::EpiEntry;
using mi::EpiMM;
using mi::EpiOut;
using mi::capi::check_overlap;
using mi::capi::fail;
using mi::capi::kMaxOffset;
using mi::capi::kMaxSplit;
using mi::capi::Range;

// ---- kernels beside the products --------------------------------------

// dst[r][0, cp) = src[r][0, c), then zeros: rows that start on 16 bytes.  One
// launch for both operands of a product (blockIdx.y).
struct PadRows {
  const uint16_t* src;
  uint16_t* dst;  // NULL: nothing to do
  long long rows;
  int c, cp;
};
struct PadBoth {
  PadRows op[2];
};
__global__ __launch_bounds__(256) void pad_rows_kernel(const PadBoth both) {
  const PadRows p = both.op[blockIdx.y];
  if (!p.dst) return;
  const int groups = p.cp / 8;
  const long long n = p.rows * groups;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) {
    const long long r = i / groups;
    const int d = (int)(i - r * groups) * 8;
    const uint16_t* s = p.src + (size_t)r * (size_t)p.c;
    uint16_t* t = p.dst + (size_t)r * (size_t)p.cp + d;
    if (d + 8 <= p.c) {
      *(mi::Pack<uint16_t>*)t = mi::load_pack(s + d);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) t[k] = d + k < p.c ? s[d + k] : (uint16_t)0;
    }
  }
}

// dst[r][0, c) = src[r][0, c) of rows cp apart (dst rows c apart): the way back.
__global__ __launch_bounds__(256) void unpad_rows_kernel(const uint16_t* __restrict__ src, uint16_t* __restrict__ dst,
                                                         long long rows, int c, int cp) {
  const int groups = cp / 8;
  const long long n = rows * groups;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) {
    const long long r = i / groups;
    const int d = (int)(i - r * groups) * 8;
    const uint16_t* s = src + (size_t)r * (size_t)cp + d;
    uint16_t* t = dst + (size_t)r * (size_t)c + d;
    if (d + 8 <= c) {
      *(mi::Pack<uint16_t>*)t = mi::load_pack(s);
    } else {
      for (int k = 0; d + k < c; ++k) t[k] = s[k];
    }
  }
}

// dst[c][0, rp) = src[0, rows)[c], then zeros: an operand whose rows are
// contracted, turned.  64 x 64 pieces through LDS.
__global__ __launch_bounds__(256) void turn_rows_kernel(const uint16_t* __restrict__ src, uint16_t* __restrict__ dst,
                                                        int rows, int cols, int ld, int rp) {
  __shared__ uint16_t tile[64][66];
  const int tid = (int)threadIdx.x, c0 = (int)blockIdx.x * 64;
  for (int r0 = (int)blockIdx.y * 64; r0 < rp; r0 += (int)gridDim.y * 64) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int r = r0 + (tid >> 6) + 4 * i, c = c0 + (tid & 63);
      tile[tid & 63][(tid >> 6) + 4 * i] = r < rows && c < cols ? src[(size_t)r * (size_t)ld + c] : (uint16_t)0;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int c = (tid >> 3) + 32 * i, r = (tid & 7) * 8;
      if (c0 + c >= cols || r0 + r >= rp) continue;
      mi::Pack<uint16_t> v;
#pragma unroll
      for (int k = 0; k < 8; ++k) v.v[k] = tile[c][r + k];
      *(mi::Pack<uint16_t>*)(dst + (size_t)(c0 + c) * (size_t)rp + r0 + r) = v;
    }
  }
}

// out = act(sum over parts of ws[part][M][ldw] + bias) + residual, parts in
// order (parts == 0: a product of 0); 8 columns of one row a thread.
__global__ __launch_bounds__(256) void epi_sum_kernel(const float* __restrict__ ws, int parts, int ldw, EpiOut e) {
  const int groups = ldw / 8;
  const long long n = (long long)e.M * groups;
  const size_t stride = (size_t)e.M * (size_t)ldw;
  e.m0 = 0;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) {
    const int m = (int)(i / groups), c = (int)(i - (long long)m * groups) * 8;
    e.columns(c);
    float v[8] = {};
    if (parts > 0) {
      const float* at = ws + (size_t)m * (size_t)ldw + c;
      const mi::f32x4_t lo = mi::sum_in_order<0>((const mi::f32x4_t*)at, stride, parts);
      const mi::f32x4_t hi = mi::sum_in_order<0>((const mi::f32x4_t*)(at + 4), stride, parts);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        v[k] = lo[k];
        v[4 + k] = hi[k];
      }
    }
    e.apply(0, m, c, v);
  }
}

// dpre[m][0, np) = bf16(dout * act'(pre)) with zeros past N, and the column
// sums of the unrounded values over this block's rows: blockIdx.x takes 64 W
// columns, the block's 4 waves rows 4 * blockIdx.y + wave, + 4 * gridDim.y, ...
// A lane has W columns (8; 1 where N < 8); past the row's end the last W, of
// which own .. W - 1 are its own.  dpre is rounded because the matrix cores
// take bf16: the products' error against float64 is then 2.35e-3, where their
// own rounding alone leaves 1.66e-3 (1000 x 1501 x 777 and 4096^3); keeping a
// second half as well would double both products (107 us each at 4096^3).
// Bound by its bytes: 22 us for 4096 x 4096
// (100 MB) on one MI355X, 4.6 TB/s.
struct ActGrad {
  const uint16_t *dout, *pre;
  uint16_t* dpre;  // NULL: not wanted
  float* part;     // [gridDim.y][N], NULL: not wanted
  int M, N, np, act;
};
template <int W>
__global__ __launch_bounds__(256) void act_grad_kernel(const ActGrad p) {
  __shared__ float xs[4][64 * W + 8];
  const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
  const int first = (int)blockIdx.x * 64 * W, c = first + lane * W;
  const int at = c + W <= p.N ? c : p.N - W, own = c - at;
  float sum[W];
  mi::fill(sum, 0.0f);
  const int step = 4 * (int)gridDim.y;
  constexpr int U = 4;
  for (int m0 = 4 * (int)blockIdx.y + wave; m0 < p.M; m0 += U * step) {
    mi::Pack<uint16_t, W> dq[U], xq[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int m = m0 + u * step < p.M ? m0 + u * step : p.M - 1;
      dq[u] = mi::load_pack<uint16_t, W>(p.dout + (size_t)m * (size_t)p.N + at);
    }
    if (p.pre) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int m = m0 + u * step < p.M ? m0 + u * step : p.M - 1;
        xq[u] = mi::load_pack<uint16_t, W>(p.pre + (size_t)m * (size_t)p.N + at);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int m = m0 + u * step;
      if (m >= p.M) break;
      float d[W];
#pragma unroll
      for (int i = 0; i < W; ++i) d[i] = mi::bf16lo((uint32_t)dq[u].v[i]);
      if (p.pre)
        mi::with_act(p.act, [&](auto a_c) __attribute__((always_inline)) {
#pragma unroll
          for (int i = 0; i < W; ++i) d[i] *= mi::act_slope<decltype(a_c)::value>(mi::bf16lo((uint32_t)xq[u].v[i]));
        });
#pragma unroll
      for (int i = 0; i < W; ++i) sum[i] += d[i];
      if (!p.dpre || c >= p.N) continue;
      uint16_t* row = p.dpre + (size_t)m * (size_t)p.np;
      if (own == 0) {
        if constexpr (W == 8) *(mi::u32x4_t*)(row + c) = mi::pack8(d);
        else row[c] = (uint16_t)mi::pack_bf16x2(d[0], 0.0f);
      } else {
#pragma unroll
        for (int i = 0; i < W; ++i)
          if (i >= own) row[at + i] = (uint16_t)mi::pack_bf16x2(d[i], 0.0f);
      }
      if (c + W >= p.N)  // the row's last lane
        for (int n = p.N; n < p.np; ++n) row[n] = 0;
    }
  }
  if (!p.part) return;
  if (c < p.N) {
#pragma unroll
    for (int i = 0; i < W; ++i)
      if (i >= own) xs[wave][at + i - first] = sum[i];
  }
  __syncthreads();
  for (int k = (int)threadIdx.x; k < 64 * W; k += 256) {
    const int n = first + k;
    if (n < p.N) p.part[(size_t)blockIdx.y * (size_t)p.N + n] = ((xs[0][k] + xs[1][k]) + xs[2][k]) + xs[3][k];
  }
}

// ---- host ----------------------------------------------------------------

int launched(const char* what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? MI_OK : fail(-(int)e, "%s: %s", what, hipGetErrorString(e));
}

unsigned blocks_for(long long items) {
  const long long b = (items + 255) / 256;
  return (unsigned)(b < 1 ? 1 : b > 8192 ? 8192 : b);
}

// Columns of an output whose block rows (256 of 4 bytes a column) stay within
// 32-bit offsets with room to spare: wider ones are stored element by element
// and not split.
constexpr int kWide = 1 << 20;

// A launch holds fewer than 2^32 threads.
bool launches(long long blocks, int threads) { return blocks * threads < 1ll << 32; }

int up8(int v) { return (v + 7) / 8 * 8; }
size_t up256(size_t v) { return (v + 255) / 256 * 256; }
bool at16(const void* p) { return (uintptr_t)p % 16 == 0; }

const EpiEntry* table(bool bt, int* n) { return bt ? mi::epi_table_nt(n) : mi::epi_table_nn(n); }

const EpiEntry* find(bool bt, const mi_tile_cfg& c) {
  int n = 0;
  const EpiEntry* t = table(bt, &n);
  for (int i = 0; i < n; ++i) {
    const mi_tile_cfg& x = t[i].cfg;
    if (x.block_m == c.block_m && x.block_n == c.block_n && x.block_k == c.block_k && x.waves == c.waves &&
        x.lds_stages == c.lds_stages && x.variant == c.variant)
      return &t[i];
  }
  return nullptr;
}

// The library's choice of a config for a product of these sizes: the least
// estimated time (mi_epi_table.hpp) over the configs and part counts.  The
// busiest unit's blocks run one after the other, or share it; no product is
// faster than its bytes at 5.4 TB/s, and one whose rhs the last-level cache
// does not hold nears the larger of its blocks' time and its bytes' as the two
// part; parts cost a second launch and their fp32 products written and read.
mi_tile_cfg pick(int M, int N, int K, bool bt) {
  int n = 0;
  const EpiEntry* t = table(bt, &n);
  const int cus = mi::capi::device_cus();
  const double bytes = 2.0 * ((double)N * K + (double)M * K + (double)M * N);
  const bool streamed = 2.0 * (double)N * K > 256.0 * (1 << 20);
  const int kt = (K + 63) / 64;
  mi_tile_cfg best = t[0].cfg;
  double least = 1e30;
  for (int i = 0; i < n; ++i) {
    const EpiEntry& e = t[i];
    const long long tiles =
        (long long)((M + e.cfg.block_m - 1) / e.cfg.block_m) * ((N + e.cfg.block_n - 1) / e.cfg.block_n);
    if (!launches(tiles, e.cfg.waves * 64)) continue;  // small blocks of an output past 128 GB
    for (const int parts : {1, 2, 3, 4, 6, 8, 12, 16}) {
      const int each = (kt + parts - 1) / parts;
      // Parts of at least three K tiles, none empty, in at most four blocks a
      // unit.  The first count that does not fit ends the search: at 61 to 64,
      // 76, 77, 109, 110 and 121 K tiles 12 parts leave one empty and 16 do
      // not, but those take 1.07 times what is chosen so (40 shapes of 1 to
      // 512 rows, 0.98 to 1.19).
      if (parts > 1 && (N > kWide || kt / parts < 3 || (parts - 1) * each >= kt || tiles * parts > 4ll * cus ||
                        (double)parts * M * N * 4.0 > (double)mi::capi::kMaxWorkspace))
        break;
      const long long blocks = (tiles * parts + cus - 1) / cus, rounds = (blocks + e.per_cu - 1) / e.per_cu;
      const double in_line = (double)blocks * e.shared * each, alone = (double)rounds * e.alone * each;
      double us = (in_line > alone ? in_line : alone) + (double)rounds * e.ends;
      if (streamed) {
        const double cold = (double)rounds * ((double)each * e.cold + e.ends), blocks_us = us > cold ? us : cold;
        const double mem = bytes / (e.stream * 1e6);
        us = std::cbrt(blocks_us * blocks_us * blocks_us + mem * mem * mem);
      } else if (us < bytes / 5.4e6) {
        us = bytes / 5.4e6;
      }
      if (parts > 1) us += 3.0 + (double)parts * M * N * 2e-6;
      if (us < least) {
        least = us;
        best = e.cfg;
        best.split_k = parts;
      }
    }
  }
  return best;
}

// One product A . B or A . B^T with an epilogue: of operands in rows of 16
// bytes, or (any) as they are.
struct Product {
  EpiMM mm;
  const EpiEntry* e;
  int ldw;
  size_t ws_bytes;
  bool any, bt;
  AnyMM as_is;
};
int plan(const uint16_t* a, int lda, const uint16_t* b, int ldb, long long b_rows, int M, int N, int K, bool bt,
         const mi_tile_cfg* cfg, Product* out) {
  mi_tile_cfg c = cfg ? *cfg : pick(M, N, K, bt);
  if (c.split_k < 1 || c.split_k > kMaxSplit) return fail(MI_E_SPLIT, "split_k=%d outside [1, %d]", c.split_k, kMaxSplit);
  if (c.group_m < 0) return fail(MI_E_ARGS, "group_m=%d negative", c.group_m);
  const EpiEntry* e = find(bt, c);
  if (!e)
    return fail(MI_E_NO_INSTANCE, "no compiled instance for the epilogue product with bm=%d bn=%d bk=%d waves=%d stages=%d variant=%d",
                c.block_m, c.block_n, c.block_k, c.waves, c.lds_stages, c.variant);
  const long long kt = ((long long)K + c.block_k - 1) / c.block_k, each = (kt + c.split_k - 1) / c.split_k;
  if ((long long)(c.split_k - 1) * each >= kt && c.split_k > 1)
    return fail(MI_E_SPLIT, "split_k=%d leaves a K part empty at K=%d, block_k=%d", c.split_k, K, c.block_k);
  if (c.split_k > 1 && N > kWide) return fail(MI_E_SPLIT, "split_k=%d takes at most %d columns", c.split_k, kWide);
  // Loads run up to a block past the last row and a K tile past the last column.
  const unsigned long long a_span = ((unsigned long long)M + c.block_m) * lda * 2ull + 16ull * c.block_k;
  const unsigned long long b_span = bt ? ((unsigned long long)N + c.block_n) * ldb * 2ull + 16ull * c.block_k
                                       : ((unsigned long long)K + c.block_k) * ldb * 2ull + 2ull * c.block_n;
  if (a_span > kMaxOffset || b_span > kMaxOffset)
    return fail(MI_E_RANGE, "operand spans exceed 32-bit buffer offsets (%llu, %llu bytes)", a_span, b_span);
  const long long tiles = ((long long)M + c.block_m - 1) / c.block_m * (((long long)N + c.block_n - 1) / c.block_n);
  if (!launches(tiles * c.split_k, c.waves * 64))
    return fail(MI_E_RANGE, "%lld blocks of %d threads are over a launch's 2^32 threads", tiles * c.split_k, c.waves * 64);
  out->any = false;
  out->e = e;
  out->ldw = up8(N);
  out->ws_bytes = c.split_k > 1 ? (size_t)c.split_k * (size_t)M * (size_t)out->ldw * 4 : 0;
  if (out->ws_bytes > mi::capi::kMaxWorkspace)
    return fail(MI_E_RANGE, "split-K workspace of %zu bytes exceeds %llu", out->ws_bytes, mi::capi::kMaxWorkspace);
  out->mm = EpiMM{a, b, (uint32_t)((size_t)M * lda * 2), (uint32_t)((size_t)b_rows * ldb * 2), M, N, K, lda, ldb,
                  mi::capi::raster_group(c.group_m, M, c.block_m), c.split_k};
  return MI_OK;
}
// The blocks of the products of operands as they are: 32 x 128, or 64 x 64
// past 32 rows.
int any_bm(int M) { return M <= 32 ? 32 : 64; }
int any_bn(int M) { return M <= 32 ? 128 : 64; }
template <int BM, int BN, bool BT>
void any_launch(const AnyMM& p, const EpiOut& o, float* ws, int ldw, hipStream_t s) {
  const unsigned tiles = (unsigned)((p.M + BM - 1) / BM) * (unsigned)((p.N + BN - 1) / BN);
  if (p.parts > 1) mi::mm_any_split_kernel<BM, BN, BT><<<dim3(tiles * (unsigned)p.parts), dim3(256), 0, s>>>(p, ws, ldw);
  else mi::mm_any_kernel<BM, BN, BT><<<dim3(tiles), dim3(256), 0, s>>>(p, o);
}
// A product of operands as they are: as many parts as fill the chip four
// blocks a unit.
void plan_any(const uint16_t* a, int lda, const uint16_t* b, int ldb, int M, int N, int K, bool bt, Product* out) {
  const long long tiles = (long long)((M + any_bm(M) - 1) / any_bm(M)) * ((N + any_bn(M) - 1) / any_bn(M));
  const int kt = (K + 63) / 64, cus = mi::capi::device_cus();
  int parts = 1;
  if (N <= kWide)
    while (parts < 8 && tiles * parts * 2 <= 4ll * cus && kt / (parts * 2) >= 4) parts *= 2;
  const int each = (kt + parts - 1) / parts;
  parts = (kt + each - 1) / each;
  out->any = true;
  out->bt = bt;
  out->as_is = AnyMM{a, b, M, N, K, lda, ldb, 8, parts};
  out->ldw = up8(N);
  out->ws_bytes = parts > 1 ? (size_t)parts * (size_t)M * (size_t)out->ldw * 4 : 0;
}
int run(const Product& p, const EpiOut& o, float* ws, hipStream_t s) {
  const int parts = p.any ? p.as_is.parts : p.mm.parts;
  if (p.any) {
    if (p.as_is.M <= 32) p.bt ? any_launch<32, 128, true>(p.as_is, o, ws, p.ldw, s) : any_launch<32, 128, false>(p.as_is, o, ws, p.ldw, s);
    else p.bt ? any_launch<64, 64, true>(p.as_is, o, ws, p.ldw, s) : any_launch<64, 64, false>(p.as_is, o, ws, p.ldw, s);
  } else if (parts > 1) {
    p.e->split(p.mm, ws, p.ldw, s);
  } else {
    p.e->direct(p.mm, o, s);
  }
  const int rc = launched("epilogue product");
  if (rc != MI_OK || parts == 1) return rc;
  epi_sum_kernel<<<dim3(blocks_for((long long)o.M * (p.ldw / 8))), dim3(256), 0, s>>>(ws, parts, p.ldw, o);
  return launched("sum of the parts");
}
// Whether a product some of whose operands would need padded copies takes them
// as they are instead.  A copy reads and writes its operand once more, which
// for few rows is most of the work: 16 x 8001 x 12345 takes 39 us as it is and
// 153 with copies (198 MB: 5 TB/s and 1.3), 200 x 4001 x 4001 37 and 38.  Past
// that the padded kernels' larger blocks win: 500 x 2001 x 3001 31 and 25 us,
// 1000 x 5001 x 4001 110 and 78.
bool better_as_is(int M, int N, int K, bool bt) {
  if (M > 256 || K < 8 || (!bt && N < 8)) return false;
  return launches((long long)((M + any_bm(M) - 1) / any_bm(M)) * ((N + any_bn(M) - 1) / any_bn(M)), 256);
}

// An operand that needs padded rows: its copy's place in the workspace.
struct Padded {
  bool on;
  int ld;
  size_t at, bytes;
};
Padded padded(const void* p, long long rows, int c, size_t* ws) {
  Padded q = {c % 8 != 0 || !at16(p), up8(c), 0, 0};
  if (q.on) {
    q.at = *ws;
    q.bytes = (size_t)rows * (size_t)q.ld * 2;
    *ws += up256(q.bytes);
  }
  return q;
}
PadRows pad_of(const void* src, char* ws, const Padded& q, long long rows, int c) {
  return PadRows{(const uint16_t*)src, q.on ? (uint16_t*)(ws + q.at) : nullptr, rows, c, q.ld};
}
int pad(const PadRows& a, const PadRows& b, hipStream_t s) {
  if (!a.dst && !b.dst) return MI_OK;
  const long long na = a.dst ? a.rows * (a.cp / 8) : 0, nb = b.dst ? b.rows * (b.cp / 8) : 0;
  pad_rows_kernel<<<dim3(blocks_for(na > nb ? na : nb), b.dst ? 2 : 1), dim3(256), 0, s>>>(PadBoth{{a, b}});
  return launched("padded copy");
}
const uint16_t* placed(const void* src, char* ws, const Padded& q) {
  return (const uint16_t*)(q.on ? ws + q.at : src);
}

int check_sizes(int M, int N, int K, int act) {
  if (M < 0 || N < 0 || K < 0) return fail(MI_E_ARGS, "negative size M=%d N=%d K=%d", M, N, K);
  constexpr int most = 0x7FFFFFFF - (1 << 20);  // indexes run a grid's stride past a size in 32 bits
  if (M > most || N > most || K > most) return fail(MI_E_RANGE, "a size over %d (M=%d N=%d K=%d)", most, M, N, K);
  if (act < MI_ACT_NONE || act > MI_ACT_SILU) return fail(MI_E_ARGS, "unknown activation %d", act);
  const unsigned long long lim = kMaxOffset / 2;
  if ((unsigned long long)M * K > lim || (unsigned long long)K * N > lim || (unsigned long long)M * N > 1ull << 40)
    return fail(MI_E_RANGE, "operand spans exceed 32-bit buffer offsets (M=%d N=%d K=%d)", M, N, K);
  return MI_OK;
}

// Everything that a forward call decides before it launches.
struct Fwd {
  Padded lhs, rhs;
  Product mm;
  size_t part_at, bytes;
};
int fwd_plan(const mi_epilogue_args* a, const mi_tile_cfg* cfg, char* ws, Fwd* f) {
  const int rc = check_sizes(a->M, a->N, a->K, a->activation);
  if (rc != MI_OK) return rc;
  *f = Fwd{};
  if (a->M == 0 || a->N == 0 || a->K == 0) return MI_OK;
  const bool bt = a->rhs_transposed != 0;
  const int b_rows = bt ? a->N : a->K, b_cols = bt ? a->K : a->N;
  f->lhs = padded(a->lhs, a->M, a->K, &f->bytes);
  f->rhs = padded(a->rhs, b_rows, b_cols, &f->bytes);
  if (f->bytes && !cfg && better_as_is(a->M, a->N, a->K, bt)) {
    *f = Fwd{};
    plan_any((const uint16_t*)a->lhs, a->K, (const uint16_t*)a->rhs, b_cols, a->M, a->N, a->K, bt, &f->mm);
    f->bytes = f->mm.ws_bytes;
    return MI_OK;
  }
  f->part_at = f->bytes;
  const int prc = plan(placed(a->lhs, ws, f->lhs), f->lhs.ld, placed(a->rhs, ws, f->rhs), f->rhs.ld, b_rows, a->M, a->N,
                       f->lhs.ld, bt, cfg, &f->mm);
  f->bytes += f->mm.ws_bytes;
  return prc;
}

// Whether a weight's gradient whose rows do not start on 16 bytes comes from
// a product of the turned operand, which stores where it belongs, rather than
// from padded rows and a copy of them.  Of rhs [K,N] it always does: lhs is
// turned and not padded (us turned and copied, M x N x K: 16 x 8001 x 12345 71
// and 127, 1000 x 1501 x 777 23.4 and 23.6, 4000 x 3001 x 2001 80 and 88).  Of
// rhs [N,K] dpre is turned next to lhs's padded copy, which only a result
// larger than its operands pays for: 75 and 126, 31 and 23, 94 and 83; 100 x
// 5001 x 1503 23.3 and 25.4, 16 x 1001 x 1001 13.6 and 12.
bool better_turned(int M, int N, int K, bool bt) { return !bt || (M <= 256 && (long long)N * K >= 4 << 20); }

struct Bwd {
  Padded dout, lhs, rhs;      // dout: dpre's place, or dout's padded copy
  bool dpre;                  // dout * act'(pre) goes to that place
  Product dlhs, drhs;
  bool turned;                // drhs by a product of its turned operand (else mi_matmul_lhsT_rhs_bf16)
  bool copied;                // that product's result goes through padded rows
  mi_tile_cfg lhsT;           // its config, and the workspace of it
  size_t lhsT_bytes;
  size_t dlhs_part, drhs_part, turn_at, drhs_at, bias_at, bytes;
  int chunks, rp, kp;
};
int bwd_plan(const mi_epilogue_grad_args* a, char* ws, Bwd* b) {
  const int rc = check_sizes(a->M, a->N, a->K, a->activation);
  if (rc != MI_OK) return rc;
  *b = Bwd{};
  if (a->M == 0 || a->N == 0) return MI_OK;
  const bool bt = a->rhs_transposed != 0;
  const long long M = a->M;
  const int N = a->N, K = a->K;
  const auto take = [&](size_t n) {
    const size_t at = b->bytes;
    b->bytes += up256(n);
    return at;
  };
  if (a->dbias) {
    if (N > 1 << 28) return fail(MI_E_RANGE, "dbias of %d columns, over %d", N, 1 << 28);  // the same limit as layer norm's
    const int xb = (up8(N) + 511) / 512;
    const int rows4 = (a->M + 3) / 4, want = 2048 / xb;
    b->chunks = want < 1 ? 1 : want > 256 ? 256 : want;
    if (b->chunks > rows4) b->chunks = rows4;
    b->bias_at = take((size_t)b->chunks * N * 4);
  }
  if (K == 0 || (!a->dlhs && !a->drhs)) return MI_OK;
  b->dpre = a->activation != MI_ACT_NONE;
  b->dout = Padded{b->dpre || N % 8 != 0 || !at16(a->dout), up8(N), 0, 0};
  if (b->dout.on) {
    b->dout.bytes = (size_t)M * b->dout.ld * 2;
    b->dout.at = take(b->dout.bytes);
  }
  const uint16_t* dpre = placed(a->dout, ws, b->dout);
  if (a->dlhs) {
    // dlhs[M,K] = dpre[M,N] . rhs^T: rhs[K,N] is K-contiguous for it, rhs[N,K] is not.
    const int rows = bt ? N : K, cols = bt ? K : N;
    const bool copies = cols % 8 != 0 || !at16(a->rhs);
    if (copies && better_as_is(a->M, K, N, !bt)) {
      plan_any(dpre, b->dout.ld, (const uint16_t*)a->rhs, cols, a->M, K, N, !bt, &b->dlhs);
    } else {
      b->rhs = padded(a->rhs, rows, cols, &b->bytes);
      const int prc = plan(dpre, b->dout.ld, placed(a->rhs, ws, b->rhs), b->rhs.ld, rows, a->M, K, b->dout.ld, !bt,
                           nullptr, &b->dlhs);
      if (prc != MI_OK) return prc;
    }
    b->dlhs_part = take(b->dlhs.ws_bytes);
  }
  if (a->drhs) {
    // The lhsT.rhs product stores whole 16-byte pieces of rows.  Other results
    // go through padded rows and are copied from there, or take the operand
    // whose columns are the result's rows turned and the epilogue product of
    // it: drhs[K,N] = (lhs^T) . dpre, drhs[N,K] = (dpre^T) . lhs.
    const bool odd = K % 8 != 0 || N % 8 != 0 || !at16(a->drhs);
    b->turned = odd && better_turned(a->M, N, K, bt);
    b->copied = odd && !b->turned;
    b->kp = up8(K);
    if (!b->turned || bt) b->lhs = padded(a->lhs, M, K, &b->bytes);
    const uint16_t* lhs = placed(a->lhs, ws, b->lhs);
    if (b->turned) {
      b->rp = up8(a->M);
      b->turn_at = take((size_t)(bt ? N : K) * b->rp * 2);
      const int prc = plan((const uint16_t*)(ws + b->turn_at), b->rp, bt ? lhs : dpre, bt ? b->lhs.ld : b->dout.ld, M,
                           bt ? N : K, bt ? K : N, b->rp, false, nullptr, &b->drhs);
      if (prc != MI_OK) return prc;
      b->drhs_part = take(b->drhs.ws_bytes);
    } else {
      // Its operands, and its loads past their ends.
      const unsigned long long span = ((unsigned long long)M + 1024) * (unsigned long long)up8(K > N ? K : N) * 2ull;
      if (span > kMaxOffset) return fail(MI_E_RANGE, "operand spans exceed 32-bit buffer offsets (%llu bytes)", span);
      if (b->copied) b->drhs_at = take((size_t)b->kp * up8(N) * 2);
      const int rows = bt ? up8(N) : b->kp, cols = bt ? b->kp : up8(N);
      mi::capi::pick_default(MI_KERNEL_MATMUL_LHST_RHS_BF16, rows, cols, a->M, &b->lhsT);
      b->lhsT_bytes = mi::workspace_bytes(MI_KERNEL_MATMUL_LHST_RHS_BF16, b->lhsT, rows, cols, a->M, mi::capi::device_cus());
      if (b->lhsT_bytes) b->drhs_part = take(b->lhsT_bytes + 256);  // 256: it starts on so many
    }
  }
  return MI_OK;
}

}  // namespace

extern "C" {

int mi_epilogue_num_configs(void) {
  int n = 0;
  (void)table(false, &n);
  return n;
}

int mi_epilogue_config(int idx, mi_tile_cfg* cfg) {
  int n = 0;
  const EpiEntry* t = table(false, &n);
  if (!cfg) return fail(MI_E_ARGS, "null config");
  if (idx < 0 || idx >= n) return fail(MI_E_ARGS, "config index %d out of range for the epilogue product", idx);
  *cfg = t[idx].cfg;
  return MI_OK;
}

int mi_epilogue_default_config(int M, int N, int K, int rhs_transposed, mi_tile_cfg* cfg) {
  if (!cfg) return fail(MI_E_ARGS, "null config");
  const int rc = check_sizes(M, N, K, MI_ACT_NONE);
  if (rc != MI_OK) return rc;
  *cfg = pick(M, N, up8(K), rhs_transposed != 0);
  return MI_OK;
}

int mi_matmul_epilogue_workspace(const mi_epilogue_args* a, const mi_tile_cfg* cfg, unsigned long long* bytes) {
  if (!a || !bytes) return fail(MI_E_ARGS, "null arguments");
  Fwd f;
  const int rc = fwd_plan(a, cfg, nullptr, &f);
  *bytes = rc == MI_OK ? f.bytes : 0;
  return rc;
}

int mi_matmul_epilogue_bf16(const mi_epilogue_args* a, const mi_tile_cfg* cfg, void* workspace,
                            unsigned long long workspace_bytes, void* stream) {
  if (!a) return fail(MI_E_ARGS, "null arguments");
  Fwd f;
  int rc = fwd_plan(a, cfg, (char*)workspace, &f);
  if (rc != MI_OK) return rc;
  const int M = a->M, N = a->N, K = a->K;
  if (M == 0 || N == 0) return MI_OK;
  if (!a->out || (K > 0 && (!a->lhs || !a->rhs))) return fail(MI_E_ARGS, "null pointer");
  if (f.bytes && (!workspace || workspace_bytes < f.bytes || !at16(workspace)))
    return fail(MI_E_ARGS, "the call needs %zu bytes of workspace, 16-byte aligned", f.bytes);
  if ((uintptr_t)a->lhs % 2 || (uintptr_t)a->rhs % 2 || (uintptr_t)a->out % 2 || (uintptr_t)a->residual % 2 ||
      (uintptr_t)a->pre % 2 || (uintptr_t)a->bias % (a->bias_f32 ? 4 : 2))
    return fail(MI_E_ALIGN, "a pointer is not aligned to its elements");
  const size_t ob = (size_t)M * N * 2;
  const Range in[] = {{a->lhs, (size_t)M * K * 2}, {a->rhs, (size_t)K * N * 2}, {a->bias, (size_t)N * (a->bias_f32 ? 4 : 2)},
                      {a->residual, ob}};
  const Range outs[] = {{a->out, ob}, {a->pre, ob}, {workspace, f.bytes}};
  if ((rc = check_overlap(outs, in)) != MI_OK) return rc;
  const hipStream_t s = (hipStream_t)stream;
  EpiOut o = {};
  o.bias = a->bias;
  o.residual = (const uint16_t*)a->residual;
  o.pre = (uint16_t*)a->pre;
  o.out = (uint16_t*)a->out;
  o.M = M;
  o.N = N;
  o.act = a->activation;
  o.bias_f32 = a->bias_f32 != 0;
  o.vec = N % 8 == 0 && N <= kWide && at16(a->bias) && at16(a->residual) && at16(a->pre) && at16(a->out);
  if (K == 0) {
    epi_sum_kernel<<<dim3(blocks_for((long long)M * (up8(N) / 8))), dim3(256), 0, s>>>(nullptr, 0, up8(N), o);
    return launched("epilogue of an empty product");
  }
  char* ws = (char*)workspace;
  const bool bt = a->rhs_transposed != 0;
  rc = pad(pad_of(a->lhs, ws, f.lhs, M, K), pad_of(a->rhs, ws, f.rhs, bt ? N : K, bt ? K : N), s);
  if (rc != MI_OK) return rc;
  return run(f.mm, o, (float*)(ws + f.part_at), s);
}

int mi_matmul_epilogue_backward_workspace(const mi_epilogue_grad_args* a, unsigned long long* bytes) {
  if (!a || !bytes) return fail(MI_E_ARGS, "null arguments");
  Bwd b;
  const int rc = bwd_plan(a, nullptr, &b);
  *bytes = rc == MI_OK ? b.bytes : 0;
  return rc;
}

int mi_matmul_epilogue_backward_bf16(const mi_epilogue_grad_args* a, void* workspace,
                                     unsigned long long workspace_bytes, void* stream) {
  if (!a) return fail(MI_E_ARGS, "null arguments");
  Bwd b;
  int rc = bwd_plan(a, (char*)workspace, &b);
  if (rc != MI_OK) return rc;
  const int M = a->M, N = a->N, K = a->K;
  const bool bt = a->rhs_transposed != 0, act = a->activation != MI_ACT_NONE;
  const bool any = M > 0 && N > 0;
  if (any && (!a->dout || (act && !a->pre) || (K > 0 && ((a->dlhs && !a->rhs) || (a->drhs && !a->lhs)))))
    return fail(MI_E_ARGS, "null pointer");
  if (b.bytes && (!workspace || workspace_bytes < b.bytes || !at16(workspace)))
    return fail(MI_E_ARGS, "the call needs %zu bytes of workspace, 16-byte aligned", b.bytes);
  if ((uintptr_t)a->dout % 2 || (uintptr_t)a->lhs % 2 || (uintptr_t)a->rhs % 2 || (uintptr_t)a->pre % 2 ||
      (uintptr_t)a->dlhs % 2 || (uintptr_t)a->drhs % 2 || (uintptr_t)a->dbias % (a->bias_f32 ? 4 : 2))
    return fail(MI_E_ALIGN, "a pointer is not aligned to its elements");
  const size_t mn = (size_t)M * N * 2, mk = (size_t)M * K * 2, kn = (size_t)K * N * 2;
  const Range in[] = {{a->dout, mn}, {a->pre, mn}, {a->lhs, mk}, {a->rhs, kn}};
  const Range outs[] = {{a->dlhs, mk}, {a->drhs, kn}, {a->dbias, (size_t)N * (a->bias_f32 ? 4 : 2)}, {workspace, b.bytes}};
  if ((rc = check_overlap(outs, in)) != MI_OK) return rc;
  const hipStream_t s = (hipStream_t)stream;
  char* ws = (char*)workspace;
  // Gradients of an empty product or of no rows are zeros; so is dlhs where
  // rhs has no columns.
  const auto zeros = [&](void* p, size_t n) {
    if (!p || n == 0) return (int)MI_OK;
    mi::fill_zero_kernel<<<dim3(blocks_for((long long)n)), dim3(256), 0, s>>>((uint16_t*)p, n);
    return launched("zero gradient");
  };
  if (!any) {
    if ((rc = zeros(a->dlhs, (size_t)M * K)) != MI_OK || (rc = zeros(a->drhs, (size_t)K * N)) != MI_OK) return rc;
    return zeros(a->dbias, (size_t)N * (a->bias_f32 ? 2 : 1));
  }
  const uint16_t* dout = (const uint16_t*)a->dout;
  const uint16_t* dpre = placed(a->dout, ws, b.dout);
  const int np = up8(N);
  if (a->dbias || b.dpre) {
    ActGrad g = {dout, act ? (const uint16_t*)a->pre : nullptr, b.dpre ? (uint16_t*)dpre : nullptr,
                 a->dbias ? (float*)(ws + b.bias_at) : nullptr, M, N, np, a->activation};
    const int xb = (np + 511) / 512, rows4 = (M + 3) / 4;
    int chunks = a->dbias ? b.chunks : 4096 / xb;
    chunks = chunks < 1 ? 1 : chunks > rows4 ? rows4 : chunks;
    const dim3 grid((unsigned)xb, (unsigned)chunks);
    if (N < 8) act_grad_kernel<1><<<grid, dim3(256), 0, s>>>(g);
    else act_grad_kernel<8><<<grid, dim3(256), 0, s>>>(g);
    if ((rc = launched("activation gradient")) != MI_OK) return rc;
    if (a->dbias) {
      const mi::ColumnSum c = {g.part, {a->dbias, nullptr}, chunks, N, 0};
      if (a->bias_f32) mi::column_sum<float>(c, 1, s);
      else mi::column_sum<mi::Bf16>(c, 1, s);
      if ((rc = launched("bias gradient")) != MI_OK) return rc;
    }
  }
  if (K == 0) return MI_OK;
  const PadRows none = {nullptr, nullptr, 0, 0, 0};
  if (!b.dpre && (a->dlhs || a->drhs) && (rc = pad(pad_of(a->dout, ws, b.dout, M, N), none, s)) != MI_OK) return rc;
  rc = pad(pad_of(a->lhs, ws, b.lhs, M, K), pad_of(a->rhs, ws, b.rhs, bt ? N : K, bt ? K : N), s);
  if (rc != MI_OK) return rc;
  const auto store_to = [](void* p, int rows, int cols) {
    EpiOut o = {};
    o.out = (uint16_t*)p;
    o.M = rows;
    o.N = cols;
    o.vec = cols % 8 == 0 && cols <= kWide && at16(p);
    return o;
  };
  if (a->dlhs && (rc = run(b.dlhs, store_to(a->dlhs, M, K), (float*)(ws + b.dlhs_part), s)) != MI_OK) return rc;
  if (a->drhs && b.turned) {
    const int cols = bt ? N : K;
    turn_rows_kernel<<<dim3((unsigned)((cols + 63) / 64), (unsigned)((M + 63) / 64 < 4096 ? (M + 63) / 64 : 4096)), dim3(256), 0, s>>>(
        bt ? dpre : (const uint16_t*)a->lhs, (uint16_t*)(ws + b.turn_at), M, cols, bt ? b.dout.ld : K, b.rp);
    if ((rc = launched("turned operand")) != MI_OK) return rc;
    return run(b.drhs, store_to(a->drhs, cols, bt ? K : N), (float*)(ws + b.drhs_part), s);
  }
  if (a->drhs) {
    // drhs[K,N] = lhs^T . dpre, or drhs[N,K] = dpre^T . lhs: rows M contracted.
    const uint16_t* lhs = placed(a->lhs, ws, b.lhs);
    void* out = b.copied ? (void*)(ws + b.drhs_at) : a->drhs;
    char* part = b.lhsT_bytes ? (char*)(((uintptr_t)ws + b.drhs_part + 255) / 256 * 256) : nullptr;
    rc = bt ? mi::capi::matmul_lhsT_rhs_bf16(dpre, lhs, out, np, b.kp, M, &b.lhsT, stream, part, b.lhsT_bytes, false)
            : mi::capi::matmul_lhsT_rhs_bf16(lhs, dpre, out, b.kp, np, M, &b.lhsT, stream, part, b.lhsT_bytes, false);
    if (rc != MI_OK || !b.copied) return rc;
    const long long rows = bt ? N : K;
    const int c = bt ? K : N;
    unpad_rows_kernel<<<dim3(blocks_for(rows * (up8(c) / 8))), dim3(256), 0, s>>>((const uint16_t*)out, (uint16_t*)a->drhs, rows, c, up8(c));
    return launched("gradient's copy");
  }
  return MI_OK;
}

}  // extern "C"
