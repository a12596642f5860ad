// matmul_fp8.hip -- mi_quantize_fp8, mi_matmul_fp8 and its gradients: argument
// checks, the config a call takes, workspaces and launches (kernels:
// mi_quant.hpp, mi_mm_fp8.hpp).
#include <cmath>

#include "mi_capi_internal.hpp"
#include "mi_fp8_table.hpp"
#include "mi_quant.hpp"

namespace {

using mi::Fp8Entry;
using mi::Fp8MM;
using mi::Fp8Out;
using mi::Quant;
using mi::capi::check_overlap;
using mi::capi::fail;
using mi::capi::kMaxOffset;
using mi::capi::kMaxSplit;
using mi::capi::Range;

// ---- kernels beside the products ------------------------------------------

using mi::PadAll;

// One launch for all operands of a call (blockIdx.y).
__global__ __launch_bounds__(256) void pad_bytes_kernel(const PadAll all) {
  mi::pad_bytes(all.op[blockIdx.y], (long long)blockIdx.x * 256 + threadIdx.x, (long long)gridDim.x * 256);
}

// dst[block][row] = src at row `row` and block `block`, of any strides: scales
// with their rows consecutive, as the products read them fastest.  64 x 64
// pieces through LDS; T: a scale's bits.
struct TurnScales {
  const void* src;
  void* dst;  // NULL: nothing to do
  long long row, k;
  int rows, blocks;
};
struct TurnBoth {
  TurnScales op[2];
};
template <class T>
__global__ __launch_bounds__(256) void turn_scales_kernel(const TurnBoth both) {
  __shared__ T tile[64][65];
  const TurnScales p = both.op[blockIdx.z];
  const int r0 = (int)blockIdx.x * 64, b0 = (int)blockIdx.y * 64;
  if (!p.dst || r0 >= p.rows || b0 >= p.blocks) return;
  const int x = (int)threadIdx.x & 63, y = (int)threadIdx.x >> 6;
  T v[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int r = r0 + y + 4 * i < p.rows ? r0 + y + 4 * i : p.rows - 1, b = b0 + x < p.blocks ? b0 + x : p.blocks - 1;
    v[i] = ((const T*)p.src)[(size_t)r * (size_t)p.row + (size_t)b * (size_t)p.k];
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) tile[y + 4 * i][x] = v[i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int b = b0 + y + 4 * i, r = r0 + x;
    if (r < p.rows && b < p.blocks) ((T*)p.dst)[(size_t)b * (size_t)p.rows + r] = tile[x][y + 4 * i];
  }
}

// out = the sum over parts of ws[part][M][ldw], parts in order (parts == 0: a
// product of 0); 8 columns of one row a thread.
__global__ __launch_bounds__(256) void fp8_sum_kernel(const float* __restrict__ ws, int parts, int ldw, const Fp8Out e) {
  const int groups = ldw / 8;
  const long long n = (long long)e.M * groups;
  const size_t stride = (size_t)e.M * (size_t)ldw;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) {
    const int m = (int)(i / groups), c = (int)(i - (long long)m * groups) * 8;
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
    e.put(m, c, v);
  }
}

// ---- host -----------------------------------------------------------------

int launched(const char* what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? MI_OK : fail(-(int)e, "%s: %s", what, hipGetErrorString(e));
}

unsigned blocks_for(long long items) {
  const long long b = (items + 255) / 256;
  return (unsigned)(b < 1 ? 1 : b > 8192 ? 8192 : b);
}

// Columns of an output whose block rows (256 of 4 bytes a column) stay within
// 32-bit offsets with room to spare: wider ones are stored with 64-bit ones
// and not split.
constexpr int kWide = 1 << 20;
constexpr int kMostSize = 0x7FFFFFFF - (1 << 20);  // indexes run a block past a size in 32 bits

// A launch holds fewer than 2^32 threads.
bool launches(long long blocks, int threads) { return blocks * threads < 1ll << 32; }

long long up(long long v, int to) { return (v + to - 1) / to * to; }
long long blocks128(long long v) { return (v + 127) / 128; }
size_t up256(size_t v) { return (v + 255) / 256 * 256; }
bool at16(const void* p) { return (uintptr_t)p % 16 == 0; }
// Bytes from the first to past the last of `rows` rows of `n` elements, `ld` apart.
size_t span(long long rows, long long ld, long long n, size_t elem) {
  return rows > 0 && n > 0 ? ((size_t)(rows - 1) * (size_t)ld + (size_t)n) * elem : 0;
}

const Fp8Entry* table(int mode, bool e5m2, int* n) {
  if (mode == mi::kScaleSquare) return e5m2 ? mi::fp8_table_square_e5m2(n) : mi::fp8_table_square_e4m3(n);
  if (mode == mi::kScaleRows) return e5m2 ? mi::fp8_table_rows_e5m2(n) : mi::fp8_table_rows_e4m3(n);
  return e5m2 ? mi::fp8_table_pow2_e5m2(n) : mi::fp8_table_pow2_e4m3(n);
}

const Fp8Entry* find(int mode, bool e5m2, const mi_tile_cfg& c) {
  int n = 0;
  const Fp8Entry* t = table(mode, e5m2, &n);
  for (int i = 0; i < n; ++i) {
    const mi_tile_cfg& x = t[i].cfg;
    if (x.block_m == c.block_m && x.block_n == c.block_n && x.block_k == c.block_k && x.waves == c.waves &&
        x.lds_stages == c.lds_stages && x.variant == c.variant)
      return &t[i];
  }
  return nullptr;
}

// The library's choice of a config for a product of these sizes: the least
// estimated time (mi_fp8_table.hpp) over the configs and part counts.  The
// busiest unit's blocks run one after the other, or share it; no product is
// faster than its bytes at 5.4 TB/s, and one whose rhs comes from HBM nears the
// larger of its blocks' time and its bytes' as the two part; parts cost a second
// launch and their fp32 products written and read.  A rhs of 64 MB and more is
// taken to come from HBM, as it does where several such take turns.
mi_tile_cfg pick(int M, int N, int K, int mode, double* estimate) {
  int n = 0;
  const Fp8Entry* t = table(mode, false, &n);
  const int cus = mi::capi::device_cus();
  const double bytes = (double)N * K + (double)M * K + 2.0 * (double)M * N;
  const bool streamed = (double)N * K >= 64.0 * (1 << 20);
  const int kt = (int)blocks128(K);
  mi_tile_cfg best = t[0].cfg;
  double least = 1e30;
  for (int i = 0; i < n; ++i) {
    const Fp8Entry& e = t[i];
    const long long tiles =
        (long long)((M + e.cfg.block_m - 1) / e.cfg.block_m) * ((N + e.cfg.block_n - 1) / e.cfg.block_n);
    if (!launches(tiles, e.cfg.waves * 64)) continue;  // small blocks of an output past 128 GB
    for (const int parts : {1, 2, 3, 4, 6, 8, 12, 16}) {
      const int each = (kt + parts - 1) / parts;
      // Parts of at least two K tiles, none empty, in at most six blocks a unit.
      if (parts > 1 && (N > kWide || kt / parts < 2 || (parts - 1) * each >= kt || tiles * parts > 6ll * cus ||
                        (double)parts * M * N * 4.0 > (double)mi::capi::kMaxWorkspace))
        break;
      const long long blocks = (tiles * parts + cus - 1) / cus, rounds = (blocks + e.per_cu - 1) / e.per_cu;
      const double in_line = (double)blocks * e.shared * each, alone = (double)rounds * e.alone[mode] * each;
      double us = (in_line > alone ? in_line : alone) + (double)rounds * e.ends;
      if (streamed) {
        const double mem = bytes / (e.stream * 1e6);
        us = std::cbrt(us * us * us + mem * mem * mem);
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
  *estimate = least;
  return best;
}

// An operand in memory: rows of K bytes with their scales.
struct Operand {
  const uint8_t* p;
  const void* scale;
  long long ld, scale_row, scale_k;
};

// An operand whose rows do not start on 16 bytes: its copy's place in the workspace.
struct Padded {
  bool on;
  long long ld;
  size_t at;
};
Padded padded(const Operand& o, long long rows, int K, size_t* ws) {
  Padded q = {o.ld % 16 != 0 || !at16(o.p), o.ld, 0};
  if (rows == 1 && at16(o.p)) q = {false, up(K, 16), 0};  // one row: no stride is used
  if (q.on) {
    q.ld = up(K, 16);
    q.at = *ws;
    *ws += up256((size_t)rows * (size_t)q.ld);
  }
  return q;
}

constexpr double kTurnFrom = 50.0;  // us of a product that scales are turned for (three times that, powers of two)

// Scales whose rows are copied to where they are consecutive: the place.
struct Turned {
  bool on;
  size_t at;
};

// One product: its copies, its config and its parts.
struct Product {
  Padded a, b;
  Turned ls, rs;
  Fp8MM mm;
  const Fp8Entry* e;
  bool pow2;
  int ldw;
  size_t part_at;
};
int plan(const Operand& a, const Operand& b, int M, int N, int K, int mode, bool e5m2, bool rs_square,
         const mi_tile_cfg* cfg, size_t* ws, Product* out, double* estimate = nullptr) {
  double us = 0.0;
  const mi_tile_cfg chosen = pick(M, N, K, mode, &us), c = cfg ? *cfg : chosen;
  if (estimate) *estimate = us;
  if (c.split_k < 1 || c.split_k > kMaxSplit) return fail(MI_E_SPLIT, "split_k=%d outside [1, %d]", c.split_k, kMaxSplit);
  if (c.group_m < 0) return fail(MI_E_ARGS, "group_m=%d negative", c.group_m);
  const Fp8Entry* e = find(mode, e5m2, c);
  if (!e)
    return fail(MI_E_NO_INSTANCE, "no compiled instance for the 8-bit product with bm=%d bn=%d bk=%d waves=%d stages=%d variant=%d",
                c.block_m, c.block_n, c.block_k, c.waves, c.lds_stages, c.variant);
  const long long kt = blocks128(K), each = (kt + c.split_k - 1) / c.split_k;
  if ((long long)(c.split_k - 1) * each >= kt && c.split_k > 1)
    return fail(MI_E_SPLIT, "split_k=%d leaves a K part empty at K=%d", c.split_k, K);
  if (c.split_k > 1 && N > kWide) return fail(MI_E_SPLIT, "split_k=%d takes at most %d columns", c.split_k, kWide);
  out->a = padded(a, M, K, ws);
  out->b = padded(b, N, K, ws);
  // Loads run up to a block past the last row and a K tile past the last column.
  const unsigned long long a_span = ((unsigned long long)M + c.block_m) * (unsigned long long)out->a.ld + 256ull;
  const unsigned long long b_span = ((unsigned long long)N + c.block_n) * (unsigned long long)out->b.ld + 256ull;
  if (a_span > kMaxOffset || b_span > kMaxOffset)
    return fail(MI_E_RANGE, "operand spans exceed 32-bit buffer offsets (%llu, %llu bytes)", a_span, b_span);
  const long long tiles = ((long long)M + c.block_m - 1) / c.block_m * (((long long)N + c.block_n - 1) / c.block_n);
  if (!launches(tiles * c.split_k, c.waves * 64))
    return fail(MI_E_RANGE, "%lld blocks of %d threads are over a launch's 2^32 threads", tiles * c.split_k, c.waves * 64);
  out->e = e;
  out->pow2 = mode == mi::kScalePow2;
  out->ldw = (int)up(N, 8);
  const size_t parts = c.split_k > 1 ? (size_t)c.split_k * (size_t)M * (size_t)out->ldw * 4 : 0;
  if (parts > mi::capi::kMaxWorkspace)
    return fail(MI_E_RANGE, "split-K workspace of %zu bytes exceeds %llu", parts, mi::capi::kMaxWorkspace);
  out->part_at = *ws;
  *ws += up256(parts);
  Fp8MM& m = out->mm;
  m = Fp8MM{};
  m.ls = a.scale;
  m.rs = b.scale;
  m.ls_row = a.scale_row;
  m.ls_k = a.scale_k;
  m.rs_row = b.scale_row;
  m.rs_k = b.scale_k;
  // Scales whose rows are apart cost a line a row in every K tile: 8192^3 takes
  // 435 us with consecutive ones and 475 so, 4096^3 64 and 68, 1024 x 8192 x 8192
  // 66 and 67.  The copy takes 3 to 4 us.
  const bool worth = us > (mode == mi::kScalePow2 ? 3.0 : 1.0) * kTurnFrom && kt >= 16 && kt < 65536;
  const size_t es = mode == mi::kScalePow2 ? 1 : 4;
  const auto turn = [&](const Operand& o, int rows, bool whole, Turned* t, const void** scale, long long* row, long long* k) {
    *t = Turned{worth && whole && o.scale_row != 1 && rows >= 1024, *ws};
    if (!t->on) return;
    *ws += up256((size_t)rows * (size_t)kt * es);
    *scale = nullptr;  // (in the workspace)
    *row = 1;
    *k = rows;
  };
  turn(a, M, true, &out->ls, &m.ls, &m.ls_row, &m.ls_k);
  turn(b, N, !rs_square, &out->rs, &m.rs, &m.rs_row, &m.rs_k);
  // (The last row's end rounded up to its 16 bytes, which lie in the same page: a dword past K is cleared in the kernel.)
  m.a_bytes = (uint32_t)up((long long)span(M, out->a.ld, K, 1), 16);
  m.b_bytes = (uint32_t)up((long long)span(N, out->b.ld, K, 1), 16);
  m.M = M;
  m.N = N;
  m.K = K;
  m.lda = (int)out->a.ld;
  m.ldb = (int)out->b.ld;
  m.group_m = mi::capi::raster_group(c.group_m, M, c.block_m);
  m.parts = c.split_k;
  m.rs_shift = rs_square ? 7 : 0;
  return MI_OK;
}

// The copies of the operands of a call's products, in one launch.
struct Copies {
  PadAll all;
  int count;
  long long most;
  void add(const Padded& q, const Operand& o, long long rows, int K, char* ws) {
    if (!q.on) return;
    all.op[count++] = {o.p, (uint8_t*)ws + q.at, rows, o.ld, K, (int)q.ld};
    const long long n = rows * (q.ld / 16);
    most = n > most ? n : most;
  }
  void add(const Product& p, const Operand& a, const Operand& b, char* ws) {
    add(p.a, a, p.mm.M, p.mm.K, ws);
    add(p.b, b, p.mm.N, p.mm.K, ws);
  }
  int run(hipStream_t s) const {
    if (!count) return MI_OK;
    pad_bytes_kernel<<<dim3(blocks_for(most), (unsigned)count), dim3(256), 0, s>>>(all);
    return launched("padded copies");
  }
};

// A product with its operands where they are, or their copies.
Fp8MM placed(const Product& p, const Operand& a, const Operand& b, char* ws) {
  Fp8MM m = p.mm;
  m.a = p.a.on ? (const uint8_t*)ws + p.a.at : a.p;
  m.b = p.b.on ? (const uint8_t*)ws + p.b.at : b.p;
  return m;
}
Fp8Out result(const Fp8MM& m, void* out) {
  return Fp8Out{(mi::Bf16*)out, m.M, m.N, m.N % 8 == 0 && at16(out) && m.N <= kWide};
}

int run(const Product& p, const Operand& a, const Operand& b, void* out, char* ws, hipStream_t s) {
  Fp8MM m = placed(p, a, b, ws);
  if (p.ls.on || p.rs.on) {
    const int kt = (int)blocks128(m.K);
    const TurnBoth t = {{{a.scale, p.ls.on ? ws + p.ls.at : nullptr, a.scale_row, a.scale_k, m.M, kt},
                         {b.scale, p.rs.on ? ws + p.rs.at : nullptr, b.scale_row, b.scale_k, m.N, kt}}};
    const int rows = p.ls.on && (m.M > m.N || !p.rs.on) ? m.M : m.N;
    const dim3 grid((unsigned)((rows + 63) / 64), (unsigned)((kt + 63) / 64), 2);
    if (p.pow2) turn_scales_kernel<uint8_t><<<grid, dim3(256), 0, s>>>(t);
    else turn_scales_kernel<float><<<grid, dim3(256), 0, s>>>(t);
    const int trc = launched("scales");
    if (trc != MI_OK) return trc;
    if (p.ls.on) m.ls = ws + p.ls.at;
    if (p.rs.on) m.rs = ws + p.rs.at;
  }
  const Fp8Out o = result(m, out);
  float* part = (float*)(ws + p.part_at);
  p.e->launch(m, o, part, p.ldw, s);
  const int rc = launched("8-bit product");
  if (rc != MI_OK || m.parts == 1) return rc;
  fp8_sum_kernel<<<dim3(blocks_for((long long)m.M * (p.ldw / 8))), dim3(256), 0, s>>>(part, m.parts, p.ldw, o);
  return launched("sum of the parts");
}

// The blocks of a pair of products in one launch.
constexpr mi_tile_cfg kTwo = {64, 64, 128, 4, 4, 1, 8, 0};
long long two_blocks(int M, int N) { return (long long)((M + 63) / 64) * ((N + 63) / 64); }

// Whether two products of these estimated times, each of a launch, take less
// time in one: by the same estimate of 64 x 64 blocks, all of them together,
// and 2 us that a launch costs behind another (1000 x 1501 x 777 with fp32
// scales: 8.4 and 9.5 us, in one launch 14.6).
bool better_as_one(double us, long long blocks, int K, int mode) {
  const Fp8Entry* e = find(mode, false, kTwo);
  const int cus = mi::capi::device_cus();
  const long long each = blocks128(K), in_line = (blocks + cus - 1) / cus, rounds = (in_line + 2) / 3;
  const double shared = (double)in_line * e->shared * each, alone = (double)rounds * e->alone[mode] * each;
  return (shared > alone ? shared : alone) + (double)rounds * e->ends < us + 2.0;
}

int zero(void* p, size_t bytes, hipStream_t s) {
  const size_t n = bytes / 2;
  if (!n) return MI_OK;
  mi::fill_zero_kernel<<<dim3((unsigned)((n + 255) / 256 < 8192 ? (n + 255) / 256 : 8192)), dim3(256), 0, s>>>((uint16_t*)p, n);
  return launched("a product of 0");
}

int check_sizes(int M, int N, int K) {
  if (M < 0 || N < 0 || K < 0) return fail(MI_E_ARGS, "negative size M=%d N=%d K=%d", M, N, K);
  if (M > kMostSize || N > kMostSize || K > kMostSize)
    return fail(MI_E_RANGE, "a size over %d (M=%d N=%d K=%d)", kMostSize, M, N, K);
  if ((unsigned long long)M * N > 1ull << 40) return fail(MI_E_RANGE, "an output of %d x %d", M, N);
  return MI_OK;
}
bool fp8_type(int t) { return t == MI_FP8_E4M3 || t == MI_FP8_E5M2; }

// An operand's scales: [rows or row blocks, K blocks], any strides of at least 0.
int check_operand(const char* what, const Operand& o, bool e8m0) {
  if (o.ld < 0 || o.scale_row < 0 || o.scale_k < 0) return fail(MI_E_ARGS, "negative stride of %s", what);
  if (!o.p || !o.scale) return fail(MI_E_ARGS, "null pointer (%s)", what);
  if (!e8m0 && (uintptr_t)o.scale % 4) return fail(MI_E_ALIGN, "%s's scales are not aligned to their elements", what);
  return MI_OK;
}
Range data_range(const Operand& o, long long rows, int K) { return {o.p, span(rows, o.ld, K, 1)}; }
Range scale_range(const Operand& o, long long rows, long long blocks, bool e8m0) {
  const size_t es = e8m0 ? 1 : 4;
  return {o.scale, rows > 0 && blocks > 0 ? ((size_t)(rows - 1) * (size_t)o.scale_row + (size_t)(blocks - 1) * (size_t)o.scale_k + 1) * es : 0};
}

// A matrix's 8-bit form: grids of 128 x 128 values.
int check_quant(long long M, long long K) {
  if (M < 0 || K < 0) return fail(MI_E_ARGS, "negative size M=%lld K=%lld", M, K);
  if (M > kMostSize || K > kMostSize) return fail(MI_E_RANGE, "a size over %d (M=%lld K=%lld)", kMostSize, M, K);
  if (!launches(blocks128(M) * blocks128(K), mi::kQuantThreads)) return fail(MI_E_RANGE, "a matrix of %lld x %lld", M, K);
  return MI_OK;
}
// Whether a matrix's two forms are taken by a block each: few tiles, whose time
// is that of a block's arithmetic and not of reading the values (both forms,
// bf16, in graphs, 300 x 700 6.5 us and 4.7, 1000 x 5000 9.2 and 7.8, 4096 x 2560
// 12.5 and 11.3, 4096 x 4096 17.6 and 18.2; fp32 1000 x 1501 6.4 and 5.0, 2048 x
// 4096 11.4 and 11.4).
bool in_halves(const Quant& p, bool light) {
  return p.q && p.q_t && blocks128(p.M) * blocks128(p.K) <= (light ? 3 : 1) * mi::capi::device_cus();
}

template <class T>
void quant_launch(const Quant& p, bool square, hipStream_t s) {
  const dim3 grid((unsigned)(blocks128(p.M) * blocks128(p.K)), in_halves(p, sizeof(T) == 2 && !square) ? 2 : 1), block(mi::kQuantThreads);
  if (square) {
    if (p.q_t) mi::quantize_fp8_kernel<T, true, true><<<grid, block, 0, s>>>(p);
    else mi::quantize_fp8_kernel<T, true, false><<<grid, block, 0, s>>>(p);
  } else {
    if (p.q_t) mi::quantize_fp8_kernel<T, false, true><<<grid, block, 0, s>>>(p);
    else mi::quantize_fp8_kernel<T, false, false><<<grid, block, 0, s>>>(p);
  }
}
int quantize(const Quant& p, int dtype, bool square, hipStream_t s) {
  if (p.M == 0 || p.K == 0) return MI_OK;
  if (dtype == MI_DTYPE_BF16) quant_launch<mi::Bf16>(p, square, s);
  else if (dtype == MI_DTYPE_F16) quant_launch<mi::Fp16>(p, square, s);
  else quant_launch<float>(p, square, s);
  return launched("8-bit form");
}

// The same of a gradient that is turned, with its products' padded copies in the
// same launch (1000 x 1501 x 777 with its products 26.5 us and 23.6).
bool joined(const Quant& q, const Copies& c) { return q.q_t && c.count > 0 && c.count <= 2; }
int quantize_with(const Quant& q, const Copies& c, hipStream_t s) {
  mi::QuantPad p = {q, {c.all.op[0], c.all.op[1]}, (unsigned)(blocks128(q.M) * blocks128(q.K)), 0, 0};
  p.quant_blocks = in_halves(q, true) ? 2 * p.tiles : p.tiles;
  const long long pad = (c.most + mi::kQuantThreads - 1) / mi::kQuantThreads;
  p.pad_blocks = (unsigned)(pad > 4096 ? 4096 : pad);
  const unsigned blocks = p.quant_blocks + p.pad_blocks * (unsigned)c.count;
  mi::quantize_pad_kernel<mi::Bf16><<<dim3(blocks), dim3(mi::kQuantThreads), 0, s>>>(p);
  return launched("8-bit form and padded copies");
}

struct Fwd {
  Operand a, b;
  Product mm;
  size_t bytes;
  int mode;
};
int fwd_plan(const mi_matmul_fp8_args* a, const mi_tile_cfg* cfg, Fwd* f) {
  const int rc = check_sizes(a->M, a->N, a->K);
  if (rc != MI_OK) return rc;
  if (!fp8_type(a->lhs_dtype)) return fail(MI_E_ARGS, "unknown 8-bit type %d", a->lhs_dtype);
  *f = Fwd{};
  f->a = Operand{(const uint8_t*)a->lhs, a->lhs_scale, a->ldlhs, a->lhs_scale_row, a->lhs_scale_k};
  f->b = Operand{(const uint8_t*)a->rhs, a->rhs_scale, a->ldrhs, a->rhs_scale_row, a->rhs_scale_k};
  if (a->ldlhs < 0 || a->ldrhs < 0) return fail(MI_E_ARGS, "negative row stride");
  f->mode = a->scale_e8m0 ? mi::kScalePow2 : a->rhs_square ? mi::kScaleSquare : mi::kScaleRows;
  if (a->M == 0 || a->N == 0 || a->K == 0) return MI_OK;
  return plan(f->a, f->b, a->M, a->N, a->K, f->mode, a->lhs_dtype == MI_FP8_E5M2, a->rhs_square != 0, cfg, &f->bytes, &f->mm);
}

// The gradient's 8-bit forms in the workspace, then its two products.
struct Bwd {
  Quant q;
  Operand d, d_t, rhs_t, lhs_t;
  Product dlhs, drhs;
  bool want_l, want_r, two;  // two: both products in one launch
  size_t bytes;
};
int bwd_plan(const mi_matmul_fp8_grad_args* a, char* ws, Bwd* b) {
  int rc = check_sizes(a->M, a->N, a->K);
  if (rc == MI_OK) rc = check_sizes(a->N, a->K, a->M);
  if (rc == MI_OK) rc = check_quant(a->M, a->N);
  if (rc != MI_OK) return rc;
  if (!fp8_type(a->dtype)) return fail(MI_E_ARGS, "unknown 8-bit type %d", a->dtype);
  if (a->ldlhs_t < 0 || a->ldrhs_t < 0 || a->lddout < 0) return fail(MI_E_ARGS, "negative row stride");
  *b = Bwd{};
  b->want_l = a->dlhs && a->M > 0 && a->K > 0;
  b->want_r = a->drhs && a->N > 0 && a->K > 0;
  if (a->M == 0 || a->N == 0 || a->K == 0 || (!b->want_l && !b->want_r)) return MI_OK;
  const bool e8m0 = a->scale_e8m0 != 0, e5m2 = a->dtype == MI_FP8_E5M2;
  const size_t es = e8m0 ? 1 : 4;
  Quant& q = b->q;
  q = Quant{};
  q.x = a->dout;
  q.ldx = a->lddout;
  q.M = a->M;
  q.K = a->N;
  q.e5m2 = e5m2;
  q.e8m0 = e8m0;
  size_t at = 0;
  const auto take = [&](size_t bytes) {
    char* p = ws + at;
    at += up256(bytes);
    return p;
  };
  if (b->want_l) {
    q.ldq = up(a->N, 16);
    q.q = (uint8_t*)take((size_t)a->M * (size_t)q.ldq);
    q.scale = take((size_t)a->M * (size_t)blocks128(a->N) * es);
    b->d = Operand{q.q, q.scale, q.ldq, 1, a->M};
    b->rhs_t = Operand{(const uint8_t*)a->rhs_t, a->rhs_t_scale, a->ldrhs_t, a->rhs_t_scale_row, a->rhs_t_scale_k};
  }
  if (b->want_r) {
    q.ldq_t = up(a->M, 16);
    q.q_t = (uint8_t*)take((size_t)a->N * (size_t)q.ldq_t);
    q.scale_t = take((size_t)a->N * (size_t)blocks128(a->M) * es);
    b->d_t = Operand{q.q_t, q.scale_t, q.ldq_t, 1, a->N};
    b->lhs_t = Operand{(const uint8_t*)a->lhs_t, a->lhs_t_scale, a->ldlhs_t, a->lhs_t_scale_row, a->lhs_t_scale_k};
  }
  b->bytes = at;
  const int l_mode = e8m0 ? mi::kScalePow2 : a->rhs_square ? mi::kScaleSquare : mi::kScaleRows;
  const int r_mode = e8m0 ? mi::kScalePow2 : mi::kScaleRows;
  double l_us = 0.0, r_us = 0.0;
  if (b->want_l)
    rc = plan(b->d, b->rhs_t, a->M, a->K, a->N, l_mode, e5m2, a->rhs_square != 0, nullptr, &b->bytes, &b->dlhs, &l_us);
  if (rc == MI_OK && b->want_r)
    rc = plan(b->d_t, b->lhs_t, a->N, a->K, a->M, r_mode, e5m2, false, nullptr, &b->bytes, &b->drhs, &r_us);
  if (rc != MI_OK || !b->want_l || !b->want_r) return rc;
  // (Long ones have their scales turned first, which a pair has not.)
  const long long blocks = two_blocks(a->M, a->K) + two_blocks(a->N, a->K);
  if (l_us + r_us > kTurnFrom || !launches(blocks, 256) || !better_as_one(l_us + r_us, blocks, a->M > a->N ? a->M : a->N, r_mode)) return rc;
  b->two = true;
  b->bytes = at;
  rc = plan(b->d, b->rhs_t, a->M, a->K, a->N, r_mode, e5m2, a->rhs_square != 0, &kTwo, &b->bytes, &b->dlhs);
  if (rc == MI_OK) rc = plan(b->d_t, b->lhs_t, a->N, a->K, a->M, r_mode, e5m2, false, &kTwo, &b->bytes, &b->drhs);
  return rc;
}

}  // namespace

extern "C" {

int mi_quantize_fp8(const mi_quantize_fp8_args* a, void* stream) {
  if (!a) return fail(MI_E_ARGS, "null arguments");
  const int rc = check_quant(a->M, a->K);
  if (rc != MI_OK) return rc;
  if (a->x_dtype != MI_DTYPE_BF16 && a->x_dtype != MI_DTYPE_F16 && a->x_dtype != MI_DTYPE_F32)
    return fail(MI_E_ARGS, "unknown dtype %d", a->x_dtype);
  if (!fp8_type(a->dtype)) return fail(MI_E_ARGS, "unknown 8-bit type %d", a->dtype);
  if (a->ldx < 0) return fail(MI_E_ARGS, "negative row stride %lld", a->ldx);
  if (a->M == 0 || a->K == 0) return MI_OK;
  if (!a->x || !a->q || !a->scale || (a->q_t && !a->scale_t)) return fail(MI_E_ARGS, "null pointer");
  const size_t xs = a->x_dtype == MI_DTYPE_F32 ? 4 : 2, ss = a->scale_e8m0 ? 1 : 4;
  if (a->ldq < up(a->K, 16) || (a->q_t && a->ldq_t < up(a->M, 16)))
    return fail(MI_E_ARGS, "rows of the 8-bit form hold %d values, rounded up to 16", a->K);
  if ((uintptr_t)a->x % xs || !at16(a->q) || a->ldq % 16 || (a->q_t && (!at16(a->q_t) || a->ldq_t % 16)) ||
      (uintptr_t)a->scale % ss || (a->q_t && (uintptr_t)a->scale_t % ss))
    return fail(MI_E_ALIGN, "a pointer is not aligned to its elements, or rows of the 8-bit form to 16 bytes");
  const bool square = a->square != 0;
  const size_t mb = (size_t)(square ? blocks128(a->M) : a->M), kb = (size_t)blocks128(a->K);
  const size_t kt = (size_t)(square ? blocks128(a->K) : a->K), mt = (size_t)blocks128(a->M);
  const Range in[] = {{a->x, span(a->M, a->ldx, a->K, xs)}},
              out[] = {{a->q, span(a->M, a->ldq, up(a->K, 16), 1)}, {a->scale, mb * kb * ss},
                       {a->q_t, a->q_t ? span(a->K, a->ldq_t, up(a->M, 16), 1) : 0}, {a->scale_t, a->q_t ? kt * mt * ss : 0}};
  const int orc = check_overlap(out, in);
  if (orc != MI_OK) return orc;
  const Quant p = {a->x,   (uint8_t*)a->q, (uint8_t*)a->q_t, a->scale, a->scale_t, a->ldx, a->ldq,
                   a->ldq_t, a->M,         a->K,             a->dtype == MI_FP8_E5M2,  a->scale_e8m0 != 0};
  return quantize(p, a->x_dtype, square, (hipStream_t)stream);
}

int mi_fp8_num_configs(void) {
  int n = 0;
  table(mi::kScaleSquare, false, &n);
  return n;
}

int mi_fp8_config(int idx, mi_tile_cfg* cfg) {
  int n = 0;
  const Fp8Entry* t = table(mi::kScaleSquare, false, &n);
  if (!cfg || idx < 0 || idx >= n) return fail(MI_E_ARGS, "config %d of %d", idx, n);
  *cfg = t[idx].cfg;
  return MI_OK;
}

int mi_matmul_fp8_workspace(const mi_matmul_fp8_args* a, const mi_tile_cfg* cfg, unsigned long long* bytes) {
  if (!a || !bytes) return fail(MI_E_ARGS, "null arguments");
  *bytes = 0;
  Fwd f;
  const int rc = fwd_plan(a, cfg, &f);
  if (rc == MI_OK) *bytes = (unsigned long long)f.bytes;
  return rc;
}

int mi_matmul_fp8(const mi_matmul_fp8_args* a, const mi_tile_cfg* cfg, void* workspace, unsigned long long workspace_bytes,
                  void* stream) {
  if (!a) return fail(MI_E_ARGS, "null arguments");
  Fwd f;
  const int rc = fwd_plan(a, cfg, &f);
  if (rc != MI_OK) return rc;
  if (a->M == 0 || a->N == 0) return MI_OK;
  if (!a->out) return fail(MI_E_ARGS, "null pointer (out)");
  const size_t ob = (size_t)a->M * (size_t)a->N * 2;
  if ((uintptr_t)a->out % 2) return fail(MI_E_ALIGN, "out is not aligned to its elements");
  const hipStream_t s = (hipStream_t)stream;
  if (a->K == 0) return zero(a->out, ob, s);
  const bool e8m0 = a->scale_e8m0 != 0;
  int orc = check_operand("lhs", f.a, e8m0);
  if (orc == MI_OK) orc = check_operand("rhs", f.b, e8m0);
  if (orc != MI_OK) return orc;
  if (f.bytes && (!workspace || workspace_bytes < f.bytes || !at16(workspace)))
    return fail(MI_E_ARGS, "the call needs %zu bytes of workspace, 16-byte aligned", f.bytes);
  const long long kb = blocks128(a->K);
  const Range in[] = {data_range(f.a, a->M, a->K), data_range(f.b, a->N, a->K), scale_range(f.a, a->M, kb, e8m0),
                      scale_range(f.b, a->rhs_square ? blocks128(a->N) : a->N, kb, e8m0)},
              out[] = {{a->out, ob}, {workspace, f.bytes}};
  orc = check_overlap(out, in);
  if (orc != MI_OK) return orc;
  Copies copies = {};
  copies.add(f.mm, f.a, f.b, (char*)workspace);
  const int prc = copies.run(s);
  return prc == MI_OK ? run(f.mm, f.a, f.b, a->out, (char*)workspace, s) : prc;
}

int mi_matmul_fp8_backward_workspace(const mi_matmul_fp8_grad_args* a, unsigned long long* bytes) {
  if (!a || !bytes) return fail(MI_E_ARGS, "null arguments");
  *bytes = 0;
  Bwd b;
  const int rc = bwd_plan(a, nullptr, &b);
  if (rc == MI_OK) *bytes = (unsigned long long)b.bytes;
  return rc;
}

int mi_matmul_fp8_backward(const mi_matmul_fp8_grad_args* a, void* workspace, unsigned long long workspace_bytes,
                           void* stream) {
  if (!a) return fail(MI_E_ARGS, "null arguments");
  Bwd b;
  const int rc = bwd_plan(a, (char*)workspace, &b);
  if (rc != MI_OK) return rc;
  const hipStream_t s = (hipStream_t)stream;
  const size_t lb = (size_t)a->M * (size_t)a->K * 2, rb = (size_t)a->N * (size_t)a->K * 2;
  if ((uintptr_t)a->dlhs % 2 || (uintptr_t)a->drhs % 2 || (uintptr_t)a->dout % 2)
    return fail(MI_E_ALIGN, "a pointer is not aligned to its elements");
  if (!b.want_l && !b.want_r) return MI_OK;
  if (a->M == 0 || a->N == 0) {
    const int zrc = b.want_l ? zero(a->dlhs, lb, s) : MI_OK;
    return zrc == MI_OK && b.want_r ? zero(a->drhs, rb, s) : zrc;
  }
  const bool e8m0 = a->scale_e8m0 != 0;
  if (!a->dout) return fail(MI_E_ARGS, "null pointer (dout)");
  int orc = b.want_l ? check_operand("rhs_t", b.rhs_t, e8m0) : MI_OK;
  if (orc == MI_OK && b.want_r) orc = check_operand("lhs_t", b.lhs_t, e8m0);
  if (orc != MI_OK) return orc;
  if (b.bytes && (!workspace || workspace_bytes < b.bytes || !at16(workspace)))
    return fail(MI_E_ARGS, "the call needs %zu bytes of workspace, 16-byte aligned", b.bytes);
  const Range in[] = {{a->dout, span(a->M, a->lddout, a->N, 2)},
                      b.want_l ? data_range(b.rhs_t, a->K, a->N) : Range{},
                      b.want_l ? scale_range(b.rhs_t, a->rhs_square ? blocks128(a->K) : a->K, blocks128(a->N), e8m0) : Range{},
                      b.want_r ? data_range(b.lhs_t, a->K, a->M) : Range{},
                      b.want_r ? scale_range(b.lhs_t, a->K, blocks128(a->M), e8m0) : Range{}},
              out[] = {{a->dlhs, lb}, {a->drhs, rb}, {workspace, b.bytes}};
  orc = check_overlap(out, in);
  if (orc != MI_OK) return orc;
  Copies copies = {};
  if (b.want_l) copies.add(b.dlhs, b.d, b.rhs_t, (char*)workspace);
  if (b.want_r) copies.add(b.drhs, b.d_t, b.lhs_t, (char*)workspace);
  const unsigned long long tiles = (unsigned long long)blocks128(a->M) * (unsigned long long)blocks128(a->N);
  if (joined(b.q, copies) && launches((long long)(tiles + 8192), mi::kQuantThreads)) {
    orc = quantize_with(b.q, copies, s);
  } else {
    orc = copies.run(s);
    if (orc == MI_OK) orc = quantize(b.q, MI_DTYPE_BF16, false, s);
  }
  if (orc == MI_OK && b.two) {
    const Fp8MM l = placed(b.dlhs, b.d, b.rhs_t, (char*)workspace), r = placed(b.drhs, b.d_t, b.lhs_t, (char*)workspace);
    const long long first = two_blocks(l.M, l.N);
    const mi::Fp8Two two = {{l, r}, {result(l, a->dlhs), result(r, a->drhs)}, (int)first};
    const unsigned blocks = (unsigned)(first + two_blocks(r.M, r.N));
    const bool e5m2 = a->dtype == MI_FP8_E5M2;
    if (e8m0) e5m2 ? mi::fp8_two_pow2_e5m2(two, blocks, s) : mi::fp8_two_pow2_e4m3(two, blocks, s);
    else e5m2 ? mi::fp8_two_rows_e5m2(two, blocks, s) : mi::fp8_two_rows_e4m3(two, blocks, s);
    return launched("8-bit products");
  }
  if (orc == MI_OK && b.want_l) orc = run(b.dlhs, b.d, b.rhs_t, a->dlhs, (char*)workspace, s);
  if (orc == MI_OK && b.want_r) orc = run(b.drhs, b.d_t, b.lhs_t, a->drhs, (char*)workspace, s);
  return orc;
}

}  // extern "C"
