// mi_mm_any.hpp -- the epilogue products for operands whose rows do not start
// on 16 bytes (K or N no multiple of 8, or a pointer off 16): the panels go
// through registers, loaded 16 bytes at a time from wherever they lie, where
// the kernels of mi_mm_epi.hpp need aligned rows for their LDS-direct loads.
//
// For few rows of a large weight, where a padded copy of the weight would be
// read, written and read again.  Two K tiles are in flight in registers while
// a third is multiplied from LDS, and several small blocks share a unit; the
// LDS layout, fragments and epilogue are those of mi_mm_epi.hpp.
//
// No load is in a branch or passes an operand's end: a 16-byte piece that
// would is the last one that does not, and its values are moved to their
// places (and zeros behind them) on their way to LDS, in the K tile or block
// that ends there only.
#pragma once
#include "mi_mm_epi.hpp"
#include "mi_norm.hpp"

namespace mi {

// A is [M][lda], B [K][ldb] or (BT) [N][ldb], row strides as they come; K >=
// 8, and N >= 8 where B is [K][N].
struct AnyMM {
  const uint16_t *a, *b;
  int M, N, K, lda, ldb, group_m, parts;
};

// v's elements own .. 7 moved to 0 .., zeros behind them.
__device__ __forceinline__ Pack<uint16_t> moved_down(const Pack<uint16_t>& v, int own) {
  Pack<uint16_t> r = v;
#pragma unroll
  for (int s = 1; s < 8; s *= 2) {
    const bool on = (own & s) != 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) r.v[i] = on ? (i + s < 8 ? r.v[i + s] : (uint16_t)0) : r.v[i];
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) r.v[i] = own < 8 ? r.v[i] : (uint16_t)0;
  return r;
}

// ROWS rows of 64 consecutive k of a K-contiguous operand, by 256 threads.
template <int ROWS>
struct AnyKPanel {
  static constexpr int N = ROWS * 8 / 256;
  const uint16_t* row[N];
  int k8, lds[N], K;
  __device__ __forceinline__ void init(const uint16_t* p, int tid, int row0, int rows, int ld, int K_) {
    K = K_;
    k8 = (tid & 7) * 8;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int r = (tid >> 3) + 32 * j, at = row0 + r < rows ? row0 + r : rows - 1;
      row[j] = p + (size_t)at * (size_t)ld;
      lds[j] = r * 128 + 16 * ((tid & 7) ^ k_swz<64>(r));
    }
  }
  __device__ __forceinline__ void load(int kt, Pack<uint16_t> (&v)[N]) const {
    const int k = kt * 64 + k8, at = k + 8 <= K ? k : K - 8;
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = load_pack(row[j] + at);
  }
  __device__ __forceinline__ void store(int kt, const Pack<uint16_t> (&v)[N], MI_LDS char* panel) const {
    const bool tail = kt * 64 + 64 > K;
    const int own = kt * 64 + k8 + 8 - K;  // > 0: so many of the piece's first values are not its own
#pragma unroll
    for (int j = 0; j < N; ++j) {
      Pack<uint16_t> x = v[j];
      if (tail) x = moved_down(x, own > 0 ? own : 0);
      *(MI_LDS u32x4_t*)(panel + lds[j]) = __builtin_bit_cast(u32x4_t, x);
    }
  }
};
// 64 rows of COLS consecutive n of an N-contiguous operand.
template <int COLS>
struct AnyNPanel {
  static constexpr int N = COLS * 8 / 256, LPR = COLS / 8, ROWB = COLS * 2;
  const uint16_t* col;
  int r0, own, lds[N], K, ld;
  __device__ __forceinline__ void init(const uint16_t* p, int tid, int col0, int cols, int ld_, int K_) {
    K = K_;
    ld = ld_;
    r0 = tid / LPR;
    const int n = col0 + tid % LPR * 8, at = n + 8 <= cols ? n : cols - 8;
    col = p + at;
    own = n - at;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int r = r0 + 256 / LPR * j;
      lds[j] = r * ROWB + 16 * ((tid % LPR) ^ mn_swz<ROWB>(r));
    }
  }
  __device__ __forceinline__ void load(int kt, Pack<uint16_t> (&v)[N]) const {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int k = kt * 64 + r0 + 256 / LPR * j;
      v[j] = load_pack(col + (size_t)(k < K ? k : K - 1) * (size_t)ld);
    }
  }
  __device__ __forceinline__ void store(int kt, const Pack<uint16_t> (&v)[N], MI_LDS char* panel) const {
    const bool tail = kt * 64 + 64 > K;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      Pack<uint16_t> x = v[j];
      if (own > 0) x = moved_down(x, own);
      if (tail && kt * 64 + r0 + 256 / LPR * j >= K) x = moved_down(x, 8);
      *(MI_LDS u32x4_t*)(panel + lds[j]) = __builtin_bit_cast(u32x4_t, x);
    }
  }
};

template <int BM, int BN>
struct AnyCfg {
  using C = EpiCfg<BM, BN, 64, 4, 2>;
  using G = typename C::G;
};

// acc = the products of K tiles [kt0, kt0 + kts) of block (tm, tn).
template <int BM, int BN, bool BT, int TM, int TN>
__device__ __forceinline__ void any_main(const AnyMM& p, char* smem_c, int tmi, int tni, int kt0, int kts,
                                         f32x4_t (&acc)[TM][TN]) {
  using C = typename AnyCfg<BM, BN>::C;
  using G = typename C::G;
  using PA = AnyKPanel<BM>;
  using PB = std::conditional_t<BT, AnyKPanel<BN>, AnyNPanel<BN>>;
  MI_LDS char* smem = (MI_LDS char*)smem_c;
  const int tid = (int)threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm0 = (wave / G::WN) * G::WTM, wn0 = (wave % G::WN) * G::WTN;
  PA pa;
  PB pb;
  pa.init(p.a, tid, tmi * BM, p.M, p.lda, p.K);
  pb.init(p.b, tid, tni * BN, p.N, p.ldb, p.K);
  const int row = lane & 15, chunk = lane >> 4;
  const int arow = (wm0 + row) * 128, brow = C::B_OFF + (wn0 + row) * 128;
  int koff[2];
#pragma unroll
  for (int kk = 0; kk < 2; ++kk) koff[kk] = 16 * ((4 * kk + chunk) ^ k_swz<64>(row));
  constexpr int ROWB = BN * 2;
  int boff[TN];
  if constexpr (!BT) {
    const int krow = 8 * chunk + (row >> 2);
#pragma unroll
    for (int t = 0; t < TN; ++t) {
      const int col = wn0 + 16 * t + 4 * (row & 3);
      boff[t] = C::B_OFF + krow * ROWB + 16 * ((col >> 3) ^ mn_swz<ROWB>(krow)) + (col & 7) * 2;
    }
  }
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = f32x4_t{};
  Pack<uint16_t> va[2][PA::N], vb[2][PB::N];
  auto clamp = [&](int t) { return t < kts ? t : kts - 1; };
  auto fetch = [&](int t, int set) __attribute__((always_inline)) {
    pa.load(kt0 + clamp(t), va[set]);
    pb.load(kt0 + clamp(t), vb[set]);
  };
  auto put = [&](int t, int set, int stage) __attribute__((always_inline)) {
    pa.store(kt0 + clamp(t), va[set], smem + stage * C::A_BYTES);
    pb.store(kt0 + clamp(t), vb[set], smem + C::B_OFF + stage * C::B_BYTES);
  };
  fetch(0, 0);
  fetch(1, 1);
  put(0, 0, 0);
  __syncthreads();
  // Tile t is in stage t % 2, tile t+1 on its way in registers, tile t+2 requested.
  auto tile = [&](int t, auto s_c) __attribute__((always_inline)) {
    constexpr int s = decltype(s_c)::value;
    fetch(t + 2, s);
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      bf16x8_t af[TM], bf[TN];
#pragma unroll
      for (int i = 0; i < TM; ++i)
        af[i] = __builtin_bit_cast(bf16x8_t, *(MI_LDS u32x4_t*)(smem + s * C::A_BYTES + arow + i * 2048 + koff[kk]));
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        if constexpr (BT)
          bf[j] = __builtin_bit_cast(bf16x8_t, *(MI_LDS u32x4_t*)(smem + s * C::B_BYTES + brow + j * 2048 + koff[kk]));
        else
          bf[j] = read_tr_frag(smem_c, s * C::B_BYTES + kk * 32 * ROWB + boff[j],
                               s * C::B_BYTES + (kk * 32 + 4) * ROWB + boff[j]);
      }
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bf[j], af[i], acc[i][j], 0, 0, 0);
    }
    put(t + 1, s ^ 1, s ^ 1);
    __syncthreads();
  };
  for (int t = 0; t < kts; t += 2) {
    tile(t, std::integral_constant<int, 0>{});
    if (t + 1 < kts) tile(t + 1, std::integral_constant<int, 1>{});
  }
}

template <int BM, int BN, bool BT>
__global__ __launch_bounds__(256) void mm_any_kernel(const AnyMM p, EpiOut e) {
  using C = typename AnyCfg<BM, BN>::C;
  using G = typename C::G;
  __shared__ __attribute__((aligned(1024))) char smem[C::LDS_BYTES];
  int tm, tn;
  tile_coords((p.M + BM - 1) / BM, (p.N + BN - 1) / BN, p.group_m, tm, tn);
  f32x4_t acc[C::TM][C::TN];
  any_main<BM, BN, BT>(p, smem, tm, tn, 0, (p.K + 63) / 64, acc);
  const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int row0 = (wave / G::WN) * G::WTM, col0 = tn * BN + (wave % G::WN) * G::WTN;
  if (e.vec) {
    EpiVec v;
    v.init(e, tm * BM, BM);
    epi_rows<C::TM, C::TN, C::TURN_ROW>(acc, smem, wave, lane, row0, col0, v);
  } else {
    e.m0 = tm * BM;
    epi_rows<C::TM, C::TN, C::TURN_ROW>(acc, smem, wave, lane, row0, col0, e);
  }
}

template <int BM, int BN, bool BT>
__global__ __launch_bounds__(256) void mm_any_split_kernel(const AnyMM p, float* __restrict__ ws, int ldw) {
  using C = typename AnyCfg<BM, BN>::C;
  using G = typename C::G;
  __shared__ __attribute__((aligned(1024))) char smem[C::LDS_BYTES];
  int tm, tn, part;
  tile_coords_split((p.M + BM - 1) / BM, (p.N + BN - 1) / BN, p.group_m, p.parts, tm, tn, part);
  const int KT = (p.K + 63) / 64, each = (KT + p.parts - 1) / p.parts, kt0 = part * each;
  f32x4_t acc[C::TM][C::TN];
  any_main<BM, BN, BT>(p, smem, tm, tn, kt0, KT - kt0 < each ? KT - kt0 : each, acc);
  const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  EpiPart f;
  f.init(ws + (size_t)part * (size_t)p.M * (size_t)ldw, p.M, ldw, tm * BM, BM);
  epi_rows<C::TM, C::TN, C::TURN_ROW>(acc, smem, wave, lane, (wave / G::WN) * G::WTM, tn * BN + (wave % G::WN) * G::WTN, f);
}

}  // namespace mi
