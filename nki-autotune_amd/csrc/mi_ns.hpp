// mi_ns.hpp -- a matrix orthogonalised by Newton-Schulz products.
//
//   X_0 = G / (||G||_F + eps)          (G^T where G has more rows than columns)
//   A = X X^T;  B = b A + c A A;  X <- a X + B X
//
// Each step maps every singular value s to a s + b s^3 + c s^5.  With the
// usual coefficients (slope 3.44 at 0) five steps multiply what rounding
// leaves next to a small singular value by up to 480, so iterates of one bf16
// each end about 1e-2 off.  X, A and B are therefore held as two bf16, hi =
// bf16(v) and lo = bf16(v - hi) (together within 2^-18 of v), and a product
// is hi.hi + hi.lo + lo.hi in one fp32 accumulator (lo.lo is under 2^-18 of it
// and left out): 16 bits of each factor for three bf16 MFMAs, where the fp32
// MFMA gives 24 for sixteen times the work.
//
// Layout: rows of 32 hi, 32 lo, 32 hi, ...  A K tile of the product core (64
// elements, one 128-byte line of a row) is then 32 k's of both, so panels,
// loads and LDS are those of mi_mm_epi.hpp, and the fragments of a tile, read
// once, feed three MFMAs each pair instead of two: an 8-wave 256x256 block
// reads its LDS for two thirds of the time its MFMAs take, where the plain
// product's reads and loads fill all of it.  Widths are padded to 32 with
// zeros, which stay zeros: rows past a matrix read as zeros, so padded
// columns are products with 0.
//
// A and A A are symmetric: only blocks on and above the diagonal are
// computed, and each one above is stored twice, the second time turned.  X X^T
// of few rows of a long X has few blocks of many K tiles: it is split over K
// (ns_split_kernel).
#pragma once
#include "mi_mm_epi.hpp"

namespace mi {

// alpha * acc + beta * c, as hi and lo (out), or rounded once to bf16 (last).
// N: the padded width of c and out.
struct NsOut {
  const uint16_t* c;  // NULL: 0
  uint16_t* out;      // NULL where last is given
  uint16_t* last;     // [M][N]
  int M, N;
  float alpha, beta;
  long long batch_c, batch_out, batch_last;
};

// The operands: a's and b's rows of 2 * lda, 2 * ldb elements; kw: the padded
// contraction.
struct NsMM {
  const uint16_t *a, *b;
  uint32_t a_bytes, b_bytes;
  int M, N, kw, lda, ldb;
  long long batch_a, batch_b;
};

// Element 8 j of a row's hi values (its lo: 32 further on).
__device__ __forceinline__ uint32_t ns_at(int n) { return (uint32_t)((n >> 5) * 64 + (n & 31)); }

struct NsRows {
  EpiRows c, out, last, turned;
  int M, N, n0;  // n0: first row of `turned`
  float alpha, beta;
  u32x4_t nhi[4], nlo[4], hi[4], lo[4];

  // (m0, bm): the block's rows; (n0, bn): its columns, rows of the turned copy (bn == 0: none).
  __device__ __forceinline__ void init(const NsOut& o, long long z, int m0, int bm, int first_n, int bn) {
    const long long rows = o.M - m0 < bm ? o.M - m0 : bm, row = (long long)o.N * 4;
    c.init(o.c ? o.c + z * o.batch_c : nullptr, m0 * row, rows * row);
    uint16_t* p = o.out ? o.out + z * o.batch_out : nullptr;
    out.init(p, m0 * row, rows * row);
    last.init(o.last ? o.last + z * o.batch_last : nullptr, (long long)m0 * o.N * 2, rows * o.N * 2);
    long long cols = o.M - first_n < bn ? o.M - first_n : bn;
    if (cols < 0) cols = 0;
    turned.init(bn ? p : nullptr, first_n * row, cols * row);
    M = o.M;
    N = o.N;
    n0 = first_n;
    alpha = o.alpha;
    beta = o.beta;
  }
  __device__ __forceinline__ uint32_t at(int r, int n) const {
    return n < N ? ((uint32_t)r * (uint32_t)(2 * N) + ns_at(n)) * 2u : kEpiNowhere;
  }
  __device__ __forceinline__ void columns(int) {}
  __device__ __forceinline__ void fetch(int it, int r, int n) {
    nhi[it] = c.load(at(r, n));
    nlo[it] = c.load(n < N ? at(r, n) + 64u : kEpiNowhere);
  }
  __device__ __forceinline__ void arrived() {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      hi[i] = nhi[i];
      lo[i] = nlo[i];
    }
  }
  __device__ __forceinline__ void apply(int it, int r, int n, float (&v)[8]) {
    float h[8], l[8];
    unpack8(hi[it], h);
    unpack8(lo[it], l);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = alpha * v[i] + beta * (h[i] + l[i]);
    const u32x4_t top = store(out, at(r, n), n < N, v);
    last.store(n < N ? ((uint32_t)r * (uint32_t)N + (uint32_t)n) * 2u : kEpiNowhere, top);
  }
  // v's halves to offset off, and what the first one was.
  __device__ __forceinline__ u32x4_t store(const EpiRows& to, uint32_t off, bool in, const float (&v)[8]) const {
    const u32x4_t top = pack8(v);
    float h[8];
    unpack8(top, h);
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = v[i] - h[i];
    to.store(off, top);
    to.store(in ? off + 64u : kEpiNowhere, pack8(h));
    return top;
  }
  // Columns m .. m + 7 of row n of the turned copy.
  __device__ __forceinline__ void apply_turned(int n, int m, const float (&v)[8]) const {
    store(turned, at(n - n0, m), m < N, v);
  }
};

// acc = the product over kt K tiles of 32.
template <int BM, int BN, int WAVES, int STAGES, bool BT, int TM, int TN>
__device__ __forceinline__ void ns_main(const NsMM& p, const uint16_t* a, const uint16_t* b, char* smem, int tmi, int tni,
                                        f32x4_t (&acc)[TM][TN]) {
  using C = EpiCfg<BM, BN, 64, WAVES, STAGES>;
  using G = typename C::G;
  static_assert(TM == C::TM && TN == C::TN, "accumulators of the wave's part");
  using LA = EpiKLoad<BM, WAVES>;
  using LB = std::conditional_t<BT, EpiKLoad<BN, WAVES>, EpiNLoad<2 * BN, WAVES, 32>>;
  constexpr int LPT = LA::LOADS + LB::LOADS, NM = TM * TN;
  static_assert(C::LDS_BYTES <= kLdsBytesMax && (STAGES - 1) * LPT < 64, "LDS, vmcnt");

  const int tid = (int)threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int m0 = tmi * BM, n0 = tni * BN;
  const int wm0 = (wave / G::WN) * G::WTM, wn0 = (wave % G::WN) * G::WTN;
  const int kts = p.kw / 32;
  LA la;
  LB lb;
  la.init(wave, lane, m0, 2 * p.lda, 64);
  lb.init(wave, lane, BT ? n0 : 2 * n0, 2 * p.ldb, 64);
  const int row = lane & 15, chunk = lane >> 4;
  const int arow = (wm0 + row) * 128, brow = C::B_OFF + (wn0 + row) * 128;
  int koff[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) koff[h] = 16 * ((4 * h + chunk) ^ k_swz<64>(row));
  // N-contiguous B: rows of k, 2 * BN elements; lo is 4 chunks past hi, which
  // the swizzle (an exclusive or) turns into bit 6 of the address.
  constexpr int ROWB = BN * 4;
  int boff[TN];
  if constexpr (!BT) {
    const int krow = 8 * chunk + (row >> 2);
#pragma unroll
    for (int t = 0; t < TN; ++t) {
      const int col = (int)ns_at(wn0 + 16 * t + 4 * (row & 3));
      boff[t] = C::B_OFF + krow * ROWB + 16 * ((col >> 3) ^ mn_swz<ROWB>(krow)) + (col & 7) * 2;
    }
  }
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = f32x4_t{};

  bf16x8_t af[2][TM], bf[2][TN];  // [hi, lo]
  auto read_a = [&](int stage, int h, int t) __attribute__((always_inline)) {
    af[h][t] = __builtin_bit_cast(
        bf16x8_t, *(MI_LDS u32x4_t*)((MI_LDS char*)smem + stage * C::A_BYTES + arow + t * 2048 + koff[h]));
  };
  auto read_b = [&](int stage, int h, int t) __attribute__((always_inline)) {
    if constexpr (BT) {
      bf[h][t] = __builtin_bit_cast(
          bf16x8_t, *(MI_LDS u32x4_t*)((MI_LDS char*)smem + stage * C::B_BYTES + brow + t * 2048 + koff[h]));
    } else {
      const int at = (boff[t] ^ (64 * h)) + stage * C::B_BYTES;
      bf[h][t] = read_tr_frag(smem, at, at + 4 * ROWB);
    }
  };
  auto issue_one = [&](int q, int t, int stage) __attribute__((always_inline)) {
    if (q < LA::LOADS)
      la.template issue<false>(q, a, p.a_bytes, (uint32_t)t * 128u, smem + stage * C::A_BYTES, false);
    else
      lb.template issue<false>(q - LA::LOADS, b, p.b_bytes, (uint32_t)t * (BT ? 128u : 128u * (uint32_t)p.ldb),
                               smem + C::B_OFF + stage * C::B_BYTES, false);
  };
  auto clamp = [&](int t) { return t < kts ? t : kts - 1; };
  // MFMAs [lo, hi) of A half ha with B half hb, column by column.
  auto mfmas = [&](int ha, int hb, int lo, int hi) __attribute__((always_inline)) {
#pragma unroll
    for (int x = lo; x < hi; ++x)
      acc[x % TM][x / TM] =
          __builtin_amdgcn_mfma_f32_16x16x32_bf16(bf[hb][x / TM], af[ha][x % TM], acc[x % TM][x / TM], 0, 0, 0);
  };
  constexpr int B_READS = BT ? 1 : 2, READS = TM + B_READS * TN;

#pragma unroll
  for (int s = 0; s < STAGES; ++s)
#pragma unroll
    for (int q = 0; q < LPT; ++q) issue_one(q, clamp(s), s);
  vm_wait<(STAGES - 1) * LPT>();
  __syncthreads();
#pragma unroll
  for (int i = 0; i < TM; ++i) read_a(0, 0, i);
#pragma unroll
  for (int j = 0; j < TN; ++j) read_b(0, 0, j);

  // hi.hi, with lo's fragments read in its first half, then hi.lo.  Then tile
  // t+1 has landed, and its hi fragments are read over lo.hi, A's at once
  // (nobody needs this tile's any more), B's column by column as this tile's
  // are done with.
  //
  // The loads of tile t+STAGES go out once every wave has this tile's
  // fragments.  Two stages (large blocks) have a barrier of their own for it
  // three quarters into hi.hi, so the loads are in flight for the rest of it,
  // hi.lo and lo.hi and the next tile's first two; more stages (small blocks)
  // do with the one that tile t+1 needs (1024 x 1024: 182 -> 174 us).
  //
  // Small blocks are bound by what one unit draws from L2, about 100 GB/s (16
  // KB a tile in 0.15 us): a second group of waves taking every other tile
  // left 512 x 512 at 121 us (127 with it).
  constexpr int HM = NM / 2, QM = NM / 4, SLOTS = NM - HM - QM + NM;
  constexpr bool EARLY = STAGES == 2;
  auto tile = [&](int t, auto cur_c) __attribute__((always_inline)) {
    constexpr int cur = decltype(cur_c)::value, nxt = (cur + 1) % STAGES;
    const int t_new = clamp(t + STAGES);
#pragma unroll
    for (int i = 0; i < TM; ++i) read_a(cur, 1, i);
#pragma unroll
    for (int j = 0; j < TN; ++j) read_b(cur, 1, j);
    if constexpr (EARLY) {
      mfmas(0, 0, 0, HM);
      interleave_mfma_ds<HM, READS>();
      mfmas(0, 0, HM, HM + QM);
      __builtin_amdgcn_sched_barrier(0);
      __syncthreads();
      static_for<SLOTS>([&](auto x_c) __attribute__((always_inline)) {
        constexpr int x = decltype(x_c)::value;
#pragma unroll
        for (int q = x * LPT / SLOTS; q < (x + 1) * LPT / SLOTS; ++q) issue_one(q, t_new, cur);
        if constexpr (x < NM - HM - QM) mfmas(0, 0, HM + QM + x, HM + QM + x + 1);
        else mfmas(0, 1, x - (NM - HM - QM), x - (NM - HM - QM) + 1);
        __builtin_amdgcn_sched_barrier(0);
      });
      vm_wait<LPT>();
    } else {
      mfmas(0, 0, 0, NM);
      interleave_mfma_ds<NM, READS>();
      mfmas(0, 1, 0, NM);
      __builtin_amdgcn_sched_barrier(0);
      vm_wait<(STAGES - 2) * LPT>();
    }
    __syncthreads();
    static_for<TN>([&](auto j_c) __attribute__((always_inline)) {
      constexpr int j = decltype(j_c)::value;
#pragma unroll
      for (int i = j * TM / TN; i < (j + 1) * TM / TN; ++i) read_a(nxt, 0, i);
      if constexpr (!EARLY) {
#pragma unroll
        for (int q = j * LPT / TN; q < (j + 1) * LPT / TN; ++q) issue_one(q, t_new, cur);
      }
      mfmas(1, 0, j * TM, (j + 1) * TM);
      read_b(nxt, 0, j);
      __builtin_amdgcn_sched_barrier(0);
    });
  };
  int t0 = 0;
  for (; t0 + STAGES < kts; t0 += STAGES)
    static_for<STAGES>([&](auto s_c) __attribute__((always_inline)) { tile(t0 + s_c(), s_c); });
  static_while<STAGES>([&](auto s_c) __attribute__((always_inline)) {
    if (t0 + s_c() + 1 >= kts) return false;
    tile(t0 + s_c(), s_c);
    return true;
  });
  const int cur = (kts - 1) % STAGES;
#pragma unroll
  for (int i = 0; i < TM; ++i) read_a(cur, 1, i);
#pragma unroll
  for (int j = 0; j < TN; ++j) read_b(cur, 1, j);
  mfmas(0, 0, 0, NM);
  mfmas(0, 1, 0, NM);
  mfmas(1, 0, 0, NM);
  wait_vmem();
  __syncthreads();  // the epilogue reuses the panel buffers
}

// One product, blockIdx.y the matrix of the batch.  SYM: blocks on and above
// the diagonal of a symmetric result.
template <int BM, int BN, int WAVES, int STAGES, bool BT, bool SYM>
__global__ __launch_bounds__(WAVES * 64) void ns_product_kernel(const NsMM p, const NsOut o) {
  static_assert(!SYM || (BM == BN && BT), "a symmetric product's blocks are square");
  using C = EpiCfg<BM, BN, 64, WAVES, STAGES>;
  using G = typename C::G;
  __shared__ __attribute__((aligned(1024))) char smem[C::LDS_BYTES];
  int tm, tn;
  if constexpr (SYM) {
    // Block w (renumbered so that an XCD owns a run of them) is the w-th of
    // the columns' upper parts: column tn begins at tn (tn + 1) / 2.
    const int nwg = (int)gridDim.x, per = nwg >> 3, rem = nwg & 7, xcd = (int)blockIdx.x & 7;
    const int w = xcd * per + (xcd < rem ? xcd : rem) + ((int)blockIdx.x >> 3);
    tn = (int)((__builtin_sqrtf(8.0f * (float)w + 1.0f) - 1.0f) * 0.5f);
    while (tn * (tn + 1) / 2 > w) --tn;
    while ((tn + 1) * (tn + 2) / 2 <= w) ++tn;
    tm = w - tn * (tn + 1) / 2;
    tm = __builtin_amdgcn_readfirstlane(tm);
    tn = __builtin_amdgcn_readfirstlane(tn);
  } else {
    tile_coords((p.M + BM - 1) / BM, (p.N + BN - 1) / BN, 8, tm, tn);
  }
  const long long z = blockIdx.y;
  f32x4_t acc[C::TM][C::TN];
  ns_main<BM, BN, WAVES, STAGES, BT>(p, p.a + z * p.batch_a, p.b + z * p.batch_b, smem, tm, tn, acc);
  const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int row0 = (wave / G::WN) * G::WTM, col0 = tn * BN + (wave % G::WN) * G::WTN;
  NsRows rows;
  rows.init(o, z, tm * BM, BM, tn * BN, SYM && tm != tn ? BN : 0);
  epi_rows<C::TM, C::TN, C::TURN_ROW, SYM>(acc, smem, wave, lane, row0, col0, rows, tm * BM);
}

// Parts of A = X X^T over ranges of K tiles: fp32 products of the blocks on
// and above the diagonal to ws[matrix][part][M][N]; ns_sum_kernel adds them.
// For few rows of a long X, whose blocks would leave most units idle.
template <int BM, int WAVES, int STAGES>
__global__ __launch_bounds__(WAVES * 64) void ns_split_kernel(const NsMM p, float* __restrict__ ws, int parts) {
  using C = EpiCfg<BM, BM, 64, WAVES, STAGES>;
  using G = typename C::G;
  __shared__ __attribute__((aligned(1024))) char smem[C::LDS_BYTES];
  const int w = (int)blockIdx.x / parts, part = (int)blockIdx.x - w * parts;
  int tn = (int)((__builtin_sqrtf(8.0f * (float)w + 1.0f) - 1.0f) * 0.5f);
  while (tn * (tn + 1) / 2 > w) --tn;
  while ((tn + 1) * (tn + 2) / 2 <= w) ++tn;
  const int tm = __builtin_amdgcn_readfirstlane(w - tn * (tn + 1) / 2);
  tn = __builtin_amdgcn_readfirstlane(tn);
  const int kts = p.kw / 32, each = (kts + parts - 1) / parts, kt0 = part * each;
  const long long z = blockIdx.y;
  NsMM q = p;
  q.kw = (kts - kt0 < each ? kts - kt0 : each) * 32;
  q.a_bytes -= (uint32_t)kt0 * 128u;
  q.b_bytes -= (uint32_t)kt0 * 128u;
  f32x4_t acc[C::TM][C::TN];
  ns_main<BM, BM, WAVES, STAGES, true>(q, p.a + z * p.batch_a + kt0 * 64, p.b + z * p.batch_b + kt0 * 64, smem, tm, tn, acc);
  const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  EpiPart f;
  f.init(ws + ((size_t)z * (size_t)parts + (size_t)part) * (size_t)p.M * (size_t)p.N, p.M, p.N, tm * BM, BM);
  epi_rows<C::TM, C::TN, C::TURN_ROW>(acc, smem, wave, lane, (wave / G::WN) * G::WTM, tn * BM + (wave % G::WN) * G::WTN, f);
}

}  // namespace mi
