// mi_mm_epi.hpp -- products of a K-contiguous A[M,K] whose epilogue does more
// than store: bias, activation and residual (matmul_epilogue), and the two
// bf16 halves of the Newton-Schulz iterates.
//
//   BT = false: out = A . B, B[K,N] (N contiguous; transposing operand reads)
//   BT = true:  out = A . B^T, B[N,K] (K contiguous, like A)
//
// The main loop is pipelined as that of mi_gemm.hpp is (LDS-direct panel
// loads, STAGES K tiles in flight, operands of the next MFMA step read while
// this one runs); here K tiles are 64 wide, so that a row of a K-contiguous
// panel is a whole 128-byte line and each line is requested once, and the
// MFMAs are 16x16x32, which read and write half the accumulator registers per
// flop that 32x32x16 do (8192^3 with bias and gelu: 775 us and 834).  They
// compute out^T: a lane ends with 4 consecutive columns of one row.
//
// The epilogue turns each wave's accumulators in its own piece of LDS as
// fp32 (32 rows of 64 columns at a time, wave-private: no barrier), so that a
// lane then holds 8 consecutive columns and every access to bias, residual
// and outputs is a 16-byte piece of a whole line, and the values are rounded
// once, after the last operation.  Residual rows are requested before the
// turn and arrive behind it.
//
// Measured on one MI355X, where the plain products of this library reach 1470
// TFLOP/s at 8192^3: that size with bias, gelu_tanh and the kept
// pre-activation 793 us, 1390 TFLOP/s (MFMAs busy 74 % of the time, the rest
// mostly waits at the barriers); 1000 x 5000 x 4104 with a residual 57 us,
// where 160 blocks of 128x256 leave 96 units idle (blocks of 192x128 fill 240
// and take 61: four waves alone on a unit run its MFMAs slower); 16 x 28672 x
// 8192 with silu 78 us, 6.0 TB/s.
#pragma once
#include <type_traits>

#include "mi_act.hpp"
#include "mi_gemm.hpp"

namespace mi {

// Operands as the kernel reads them.  K, lda and ldb are multiples of 8;
// a_bytes, b_bytes: what lies behind the pointers (reads past it give 0).
struct EpiMM {
  const uint16_t *a, *b;
  uint32_t a_bytes, b_bytes;
  int M, N, K, lda, ldb, group_m, parts;
};

// TM x TN fragments of 16 rows and 16 columns a wave.
template <int BM, int BN, int BK, int WAVES, int STAGES>
struct EpiCfg {
  using G = WaveGrid<BM, BN, WAVES>;
  static constexpr int TM = G::WTM / 16, TN = G::WTN / 16;
  static constexpr int A_BYTES = BK * BM * 2;
  static constexpr int B_BYTES = BK * BN * 2;
  // The stages of A, then those of B: an LDS read's offset from a lane's
  // address then fits its 16 bits (with A and B of a stage together, the
  // second stage of a 256x256 block took a register per read).
  static constexpr int B_OFF = STAGES * A_BYTES;
  static constexpr int TURN_COLS = TN % 4 == 0 ? 64 : 32;
  static constexpr int TURN_ROW = TURN_COLS * 4 + 16;  // + 16: rows start in different banks
  static constexpr int TURN_BYTES = WAVES * 32 * TURN_ROW;
  static constexpr int MAIN_BYTES = STAGES * (A_BYTES + B_BYTES);
  static constexpr int LDS_BYTES = MAIN_BYTES > TURN_BYTES ? MAIN_BYTES : TURN_BYTES;
};

// Loaders of one K tile of 64: each wave load brings 1 KiB, lane l's 16 bytes
// landing at 16 l of its piece, so the lane fetches what the swizzle puts
// there.  Load j covers the rows j * WAVES loads further on; the swizzle
// repeats over that (every second load, N contiguous), so a lane keeps one
// or two offsets, and the rest rides in the scalar base address.
// Reads past `bytes` give 0.
//
// The descriptor must come out of scalar instructions: the load is inline
// assembly, so the compiler does not see that it reads scalar registers and
// leaves out the wait states that a vector instruction's write to one needs
// (a saturating subtraction is such an instruction; the empty asm keeps the
// minimum and the difference from becoming one).
__device__ __forceinline__ __amdgpu_buffer_rsrc_t epi_rsrc(const uint16_t* p, uint32_t bytes, uint32_t off) {
  off = __builtin_amdgcn_readfirstlane(off);
  uint32_t at = off < bytes ? off : bytes;
  asm("" : "+s"(at));
  return make_rsrc((const char*)p + at, bytes - at);
}
// ROWS rows of 64 consecutive k (K contiguous).
template <int ROWS, int WAVES>
struct EpiKLoad {
  static constexpr int LOADS = ROWS / 8 / WAVES;
  static_assert(LOADS >= 1 && ROWS % (8 * WAVES) == 0 && WAVES % 2 == 0, "whole loads, the same swizzle in each");
  uint32_t voff, voff_tail, first, step;
  int lds;
  __device__ __forceinline__ void init(int wave, int lane, int row0, int ld, int k_last) {
    const int r = wave * 8 + (lane >> 3), q = (lane & 7) ^ k_swz<64>(r);
    voff = ((uint32_t)r * (uint32_t)ld + (uint32_t)(8 * q)) * 2u;
    voff_tail = 8 * q < k_last ? voff : 0xFFFFFFF0u;
    first = (uint32_t)row0 * (uint32_t)ld * 2u;
    step = (uint32_t)(WAVES * 8) * (uint32_t)ld * 2u;
    lds = wave * 1024;
  }
  template <bool NT>
  __device__ __forceinline__ void issue(int j, const uint16_t* p, uint32_t bytes, uint32_t tile, char* panel,
                                        bool tail) const {
    lds_dma16<NT>(epi_rsrc(p, bytes, first + (uint32_t)j * step + tile), panel + lds + j * WAVES * 1024,
                  tail ? voff_tail : voff);
  }
};
// ROWS rows of COLS consecutive n (N contiguous).
template <int COLS, int WAVES, int ROWS>
struct EpiNLoad {
  static constexpr int LOADS = ROWS * COLS / 512 / WAVES, ROWB = COLS * 2, RPL = 1024 / ROWB;
  static_assert(LOADS >= 1 && ROWS * COLS % (512 * WAVES) == 0 && RPL >= 1 && 2 * WAVES * RPL % 16 == 0,
                "whole loads, two swizzles");
  uint32_t voff[2], first, step;
  int lds;
  __device__ __forceinline__ void init(int wave, int lane, int col0, int ld, int) {
    const int r = wave * RPL + lane / (COLS / 8), slot = lane % (COLS / 8);
#pragma unroll
    for (int i = 0; i < 2; ++i)
      voff[i] = ((uint32_t)r * (uint32_t)ld + (uint32_t)(8 * (slot ^ mn_swz<ROWB>(r + i * WAVES * RPL)))) * 2u;
    first = (uint32_t)col0 * 2u;
    step = (uint32_t)(WAVES * RPL) * (uint32_t)ld * 2u;
    lds = wave * 1024;
  }
  template <bool NT>
  __device__ __forceinline__ void issue(int j, const uint16_t* p, uint32_t bytes, uint32_t tile, char* panel, bool) const {
    lds_dma16<NT>(epi_rsrc(p, bytes, first + (uint32_t)j * step + tile), panel + lds + j * WAVES * 1024, voff[j & 1]);
  }
};

// acc = the products of K tiles [kt0, kt0 + kts) of block (tm, tn).  Lane l,
// register r of acc[i][j]: row 16 i + l % 16, column 16 j + 4 (l / 16) + r of
// the wave's part.
template <int BM, int BN, int BK, int WAVES, int STAGES, bool BT, bool NTB, int TM, int TN>
__device__ __forceinline__ void epi_main(const EpiMM& p, const uint16_t* a, const uint16_t* b, char* smem, int tmi,
                                         int tni, int kt0, int kts, f32x4_t (&acc)[TM][TN]) {
  using C = EpiCfg<BM, BN, BK, WAVES, STAGES>;
  using G = typename C::G;
  static_assert(G::ok && BK == 64 && STAGES >= 2 && STAGES <= 4, "tile config");
  static_assert(TM == C::TM && TN == C::TN, "accumulators of the wave's part");
  static_assert(C::LDS_BYTES <= kLdsBytesMax, "LDS over 160 KiB");
  constexpr int KS = BK / 32, NF = TM + TN, NM = TM * TN;
  using LA = EpiKLoad<BM, WAVES>;
  using LB = std::conditional_t<BT, EpiKLoad<BN, WAVES>, EpiNLoad<BN, WAVES, BK>>;
  constexpr int LPT = LA::LOADS + LB::LOADS;  // of every wave: vm_wait counts them
  static_assert((STAGES - 1) * LPT < 64, "loads in flight exceed the 6-bit vmcnt");

  const int tid = (int)threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int m0 = tmi * BM, n0 = tni * BN;
  const int wm0 = (wave / G::WN) * G::WTM, wn0 = (wave % G::WN) * G::WTN;
  const int KT1 = (p.K + BK - 1) / BK;
  const int k_last = p.K - (KT1 - 1) * BK;
  LA la;
  LB lb;
  la.init(wave, lane, m0, p.lda, k_last);
  lb.init(wave, lane, n0, p.ldb, k_last);
  // K-contiguous operands: lane l reads row l % 16 of a fragment, K chunk
  // 4 kk + l / 16 of the tile, at its k_swz slot (the same for every
  // fragment: the swizzle repeats every 16 rows).
  const int row = lane & 15, chunk = lane >> 4;
  const int arow = (wm0 + row) * (BK * 2), brow = C::B_OFF + (wn0 + row) * (BK * 2);
  int koff[KS];
#pragma unroll
  for (int kk = 0; kk < KS; ++kk) koff[kk] = 16 * ((4 * kk + chunk) ^ k_swz<BK>(row));
  // N-contiguous B: 16 lanes read 4 rows of 16 columns and each gets one
  // column of them; lanes 16 g .. 16 g + 15 take K rows 8 g .. 8 g + 7 in two
  // reads.
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

  bf16x8_t af[2][TM], bf[2][TN];
  // Operand f of step kk, in the order the MFMAs (row-major) take them: A0,
  // B0 .. B(TN-1), A1 .. A(TM-1).
  auto read_frag = [&](int stage, int kk, int buf, int f) __attribute__((always_inline)) {
    const int abase = stage * C::A_BYTES, bbase = stage * C::B_BYTES;
    if (f == 0 || f > TN) {
      const int t = f == 0 ? 0 : f - TN;
      af[buf][t] = __builtin_bit_cast(
          bf16x8_t, *(MI_LDS u32x4_t*)((MI_LDS char*)smem + abase + arow + t * 16 * (BK * 2) + koff[kk]));
    } else {
      const int t = f - 1;
      if constexpr (BT)
        bf[buf][t] = __builtin_bit_cast(
            bf16x8_t, *(MI_LDS u32x4_t*)((MI_LDS char*)smem + bbase + brow + t * 16 * (BK * 2) + koff[kk]));
      else
        bf[buf][t] = read_tr_frag(smem, bbase + (kk * 32) * ROWB + boff[t], bbase + (kk * 32 + 4) * ROWB + boff[t]);
    }
  };
  auto read_frags = [&](int stage, int kk, int buf) __attribute__((always_inline)) {
#pragma unroll
    for (int f = 0; f < NF; ++f) read_frag(stage, kk, buf, f);
  };
  // MFMAs [lo, hi) of the fragments in `buf`, row-major.
  auto mfmas = [&](int buf, int lo, int hi) __attribute__((always_inline)) {
#pragma unroll
    for (int x = lo; x < hi; ++x)
      acc[x / TN][x % TN] =
          __builtin_amdgcn_mfma_f32_16x16x32_bf16(bf[buf][x % TN], af[buf][x / TN], acc[x / TN][x % TN], 0, 0, 0);
  };
  constexpr int READS = TM + (BT ? TN : 2 * TN);  // LDS reads of one step
  // Load q (< LPT) of K tile t of this block's range into `stage`.
  auto issue_one = [&](int q, int t, int stage) __attribute__((always_inline)) {
    const int kt = kt0 + t;
    const bool tail = kt == KT1 - 1;
    if (q < LA::LOADS) {
      const uint32_t off = (uint32_t)kt * (uint32_t)(BK * 2);
      la.template issue<false>(q, a, p.a_bytes, off, smem + stage * C::A_BYTES, tail);
    } else {
      const uint32_t off = (uint32_t)kt * (BT ? (uint32_t)(BK * 2) : (uint32_t)BK * (uint32_t)p.ldb * 2u);
      lb.template issue<NTB>(q - LA::LOADS, b, p.b_bytes, off, smem + C::B_OFF + stage * C::B_BYTES, tail);
    }
  };
  // Tiles past the range are the last one again (into a buffer that nobody
  // reads): every group has the same number of loads.
  auto clamp = [&](int t) { return t < kts ? t : kts - 1; };

#pragma unroll
  for (int s = 0; s < STAGES; ++s)
#pragma unroll
    for (int q = 0; q < LPT; ++q) issue_one(q, clamp(s), s);
  vm_wait<(STAGES - 1) * LPT>();
  __syncthreads();
  read_frags(0, 0, 0);

  if constexpr (STAGES == 2) {
    // Two stages.  A stage is read within half a tile (both steps' fragments
    // are in registers from the middle of step 0 on), so the loads that
    // refill it are in flight for 1.4 tiles rather than 1:
    //   step 0: fragments of step 1 read in its first half; three quarters
    //           in, every wave has them, the stage is free and the loads of
    //           tile t+2 go out behind it, up to the middle of step 1;
    //   step 1: in its middle tile t+1 has landed, and the fragments of its
    //           step 0 are read.
    constexpr int HM = NM / 2, QM = NM / 4, SLOTS = NM / 2;
    auto tile = [&](int t, auto cur_c) __attribute__((always_inline)) {
      constexpr int cur = decltype(cur_c)::value;
      read_frags(cur, 1, 1);
      mfmas(0, 0, HM);
      interleave_mfma_ds<HM, READS>();
      mfmas(0, HM, HM + QM);
      __builtin_amdgcn_sched_barrier(0);
      __syncthreads();
      const int t_new = clamp(t + 2);
      static_for<SLOTS>([&](auto x_c) __attribute__((always_inline)) {
        constexpr int x = decltype(x_c)::value;
#pragma unroll
        for (int q = x * LPT / SLOTS; q < (x + 1) * LPT / SLOTS; ++q) issue_one(q, t_new, cur);
        if constexpr (x < NM - HM - QM) mfmas(0, HM + QM + x, HM + QM + x + 1);
        else mfmas(1, x - (NM - HM - QM), x - (NM - HM - QM) + 1);
        __builtin_amdgcn_sched_barrier(0);
      });
      constexpr int DONE = SLOTS - (NM - HM - QM);  // MFMAs of step 1 so far
      mfmas(1, DONE, HM);
      __builtin_amdgcn_sched_barrier(0);
      vm_wait<LPT>();
      __syncthreads();
      read_frags(cur ^ 1, 0, 0);
      mfmas(1, HM, NM);
      interleave_mfma_ds<NM - HM, READS>();
    };
    int t0 = 0;
    for (; t0 + 2 < kts; t0 += 2)
      static_for<2>([&](auto s_c) __attribute__((always_inline)) { tile(t0 + s_c(), s_c); });
    if (t0 + 1 < kts) tile(t0, std::integral_constant<int, 0>{});
    read_frags((kts - 1) & 1, 1, 1);
    mfmas(0, 0, NM);
    mfmas(1, 0, NM);
  } else {
    // At the last step of tile t the wave waits for its loads of tile t+1,
    // meets the workgroup (tile t+1 is whole, tile t's buffer free), reads
    // tile t+1's first operands and requests tile t+STAGES.
    auto tile = [&](int t, auto cur_c) __attribute__((always_inline)) {
      constexpr int cur = decltype(cur_c)::value, nxt = (cur + 1) % STAGES;
      read_frags(cur, 1, 1);
      mfmas(0, 0, NM);
      interleave_mfma_ds<NM, READS>();
      vm_wait<(STAGES - 2) * LPT>();
      __syncthreads();
      const int t_new = clamp(t + STAGES);
#pragma unroll
      for (int f = 0; f < NF; ++f) {
        read_frag(nxt, 0, 0, f);
#pragma unroll
        for (int q = f * LPT / NF; q < (f + 1) * LPT / NF; ++q) issue_one(q, t_new, cur);
      }
      mfmas(1, 0, NM);
      interleave_mfma_ds<NM, READS>();
    };
    int t0 = 0;
    for (; t0 + STAGES < kts; t0 += STAGES)
      static_for<STAGES>([&](auto s_c) __attribute__((always_inline)) { tile(t0 + s_c(), s_c); });
    static_while<STAGES>([&](auto s_c) __attribute__((always_inline)) {
      if (t0 + s_c() + 1 >= kts) return false;
      tile(t0 + s_c(), s_c);
      return true;
    });
    read_frags((kts - 1) % STAGES, 1, 1);
    mfmas(0, 0, NM);
    mfmas(1, 0, NM);
  }
  wait_vmem();
  __syncthreads();  // the epilogue reuses the panel buffers
}

// Hands each lane 8 consecutive columns of the wave's accumulators at a time.
// For each group of columns f.columns(n); then for each turn of 32 rows
// f.fetch(it, r, n) one turn ahead, f.arrived() and f.apply(it, r, n, v), it <
// IT rows a lane has in a turn, r counted from the block's first row.
//
// Both loops are run-time ones: the code after a turn stands once, and only
// the writes that name accumulator registers are there for each slice
// (unrolled, the epilogue of a 128x128 wave tile is 12000 instructions, and
// where the compiler leaves the loop to run time by itself it keeps the
// accumulators in memory).  Loads and stores share one counter and are
// counted off in order, so a wait for a load waits for every store before it:
// the rows of turn s+1 are requested before the stores of turn s, and f has
// no branch around a load or store, which would make the compiler wait for
// all of them.
//
// TURNED: f.apply_turned(n, m, v) also gets the values that apply left, 8 rows
// m .. m + 7 (from the result's first row on, block_row the block's first) of
// one column n.
template <int TM, int TN, int ROWB, bool TURNED = false, class F>
__device__ __forceinline__ void epi_rows(const f32x4_t (&acc)[TM][TN], char* smem, int wave, int lane, int row0,
                                         int col0, F& f, int block_row = 0) {
  constexpr int TW = TN % 4 == 0 ? 2 : 1, LPR = 4 * TW, RPI = 64 / LPR, IT = 32 / RPI, NP = TN / (2 * TW), MT = TM / 2;
  static_assert(TN % (2 * TW) == 0 && TM % 2 == 0 && ROWB == TW * 128 + 16 && IT <= 4, "turn layout");
  MI_LDS char* slot = (MI_LDS char*)smem + wave * (32 * ROWB);
  const int n0 = col0 + 8 * (lane % LPR), r0 = row0 + lane / LPR;
#pragma unroll
  for (int it = 0; it < IT; ++it) f.fetch(it, r0 + it * RPI, n0);
#pragma unroll 1
  for (int np = 0; np < NP; ++np) {
    const int n = n0 + np * (TW * 32);
    f.columns(n);
#pragma unroll 1
    for (int mt = 0; mt < MT; ++mt) {
      const int s = np * MT + mt;
      f.arrived();
      const int r_next = r0 + (mt + 1 < MT ? mt + 1 : 0) * 32, n_next = n + (mt + 1 < MT ? 0 : TW * 32);
#pragma unroll
      for (int it = 0; it < IT; ++it) f.fetch(it, r_next + it * RPI, n_next);
      static_for<NP * MT>([&](auto k_c) __attribute__((always_inline)) {
        constexpr int k = decltype(k_c)::value;
        if (s != k) return;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int j = 0; j < 2 * TW; ++j)
            *(MI_LDS f32x4_t*)(slot + (16 * i + (lane & 15)) * ROWB + 64 * j + 16 * (lane >> 4)) =
                acc[k % MT * 2 + i][k / MT * 2 * TW + j];
      });
      wave_lds_turn();
#pragma unroll
      for (int it = 0; it < IT; ++it) {
        MI_LDS char* at = slot + (it * RPI + lane / LPR) * ROWB + 32 * (lane % LPR);
        const f32x4_t lo = *(MI_LDS f32x4_t*)at, hi = *(MI_LDS f32x4_t*)(at + 16);
        float v[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
        f.apply(it, r0 + mt * 32 + it * RPI, n, v);
        if constexpr (TURNED) {
          *(MI_LDS f32x4_t*)at = f32x4_t{v[0], v[1], v[2], v[3]};
          *(MI_LDS f32x4_t*)(at + 16) = f32x4_t{v[4], v[5], v[6], v[7]};
        }
      }
      wave_lds_turn();
      if constexpr (TURNED) {
        // A lane per column: neighbours read neighbouring words of a row.
        constexpr int W = TW * 32, LANES = 64 / W;
        const int c = lane % W;
#pragma unroll
        for (int g = 0; g < 4 / LANES; ++g) {
          const int r = 8 * (g * LANES + lane / W);
          float v[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = *(MI_LDS float*)(slot + (r + i) * ROWB + 4 * c);
          f.apply_turned(col0 + np * W + c, block_row + row0 + mt * 32 + r, v);
        }
        wave_lds_turn();
      }
    }
  }
}

// 16-byte accesses to rows of a tensor, from the block's first row on:
// past `bytes` a load gives 0 and a store does nothing, without a branch.  A
// tensor that is not there has no bytes.
struct EpiRows {
  __amdgpu_buffer_rsrc_t rs;
  __device__ __forceinline__ void init(const void* p, long long first, long long count) {
    rs = make_rsrc(p ? (const char*)p + first : nullptr, p ? (uint32_t)count : 0u);
  }
  __device__ __forceinline__ u32x4_t load(uint32_t off) const {
    return __builtin_amdgcn_raw_buffer_load_b128(rs, (int)off, 0, 0);
  }
  __device__ __forceinline__ void store(uint32_t off, u32x4_t v) const {
    __builtin_amdgcn_raw_buffer_store_b128(v, rs, (int)off, 0, 0);
  }
};
constexpr uint32_t kEpiNowhere = 0xFFFFFFF0u;  // past every EpiRows

__device__ __forceinline__ u32x4_t pack8(const float (&v)[8]) {
  return u32x4_t{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7])};
}
__device__ __forceinline__ void unpack8(u32x4_t w, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = bf16lo(w[i]);
    v[2 * i + 1] = bf16hi(w[i]);
  }
}

// pre = v + bias; out = act(pre) + residual.  `vec`: N is a multiple of 8 and
// every pointer 16-byte aligned (EpiVec); otherwise as here.
struct EpiOut {
  const void* bias;
  const uint16_t* residual;
  uint16_t *pre, *out;
  int M, N, act;
  bool bias_f32, vec;

  float b[8];
  int m0;  // the block's first row

  __device__ __forceinline__ float bias_at(int n) const {
    return bias_f32 ? ((const float*)bias)[n] : bf16lo((uint32_t)((const uint16_t*)bias)[n]);
  }
  __device__ __forceinline__ void columns(int n) {
#pragma unroll
    for (int i = 0; i < 8; ++i) b[i] = bias && n + i < N ? bias_at(n + i) : 0.0f;
  }
  __device__ __forceinline__ void fetch(int, int, int) {}
  __device__ __forceinline__ void arrived() {}
  __device__ __forceinline__ void apply(int, int r, int n, float (&v)[8]) {
    const int m = m0 + r;
    if (m >= M || n >= N) return;
    const size_t at = (size_t)m * (size_t)N + n;
    const bool whole = n + 8 <= N;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] += b[i];
    if (pre) put(pre + at, n, whole, v);
    with_act(act, [&](auto a_c) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = act_value<decltype(a_c)::value>(v[i]);
    });
    if (residual) {
      if (whole) {
        float x[8];
        unpack8(((const Piece*)(residual + at))->v, x);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] += x[i];
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (n + i < N) v[i] += bf16lo((uint32_t)residual[at + i]);
      }
    }
    put(out + at, n, whole, v);
  }
  // 16 bytes at any address.
  struct __attribute__((packed, aligned(2))) Piece {
    u32x4_t v;
  };
  __device__ __forceinline__ void put(uint16_t* p, int n, bool whole, const float (&v)[8]) const {
    if (whole) {
      ((Piece*)p)->v = pack8(v);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (n + i < N) p[i] = (uint16_t)pack_bf16x2(v[i], 0.0f);
    }
  }
};

// EpiOut's function where `vec` holds, without a branch around a load or
// store.
struct EpiVec {
  EpiRows out, pre, residual, bias16, bias32;
  int N, act;
  float b[8];
  u32x4_t next[4], res[4];

  __device__ __forceinline__ void init(const EpiOut& e, int m0, int bm) {
    const long long first = (long long)m0 * e.N * 2, rows = e.M - m0 < bm ? e.M - m0 : bm;
    out.init(e.out, first, rows * e.N * 2);
    pre.init(e.pre, first, rows * e.N * 2);
    residual.init(e.residual, first, rows * e.N * 2);
    bias16.init(e.bias_f32 ? nullptr : e.bias, 0, (long long)e.N * 2);
    bias32.init(e.bias_f32 ? e.bias : nullptr, 0, (long long)e.N * 4);
    N = e.N;
    act = e.act;
  }
  __device__ __forceinline__ uint32_t at(int r, int n) const {
    return n < N ? ((uint32_t)r * (uint32_t)N + (uint32_t)n) * 2u : kEpiNowhere;
  }
  __device__ __forceinline__ void columns(int n) {
    const u32x4_t h = bias16.load(n < N ? (uint32_t)n * 2u : kEpiNowhere);
    const u32x4_t f0 = bias32.load(n < N ? (uint32_t)n * 4u : kEpiNowhere);
    const u32x4_t f1 = bias32.load(n < N ? (uint32_t)n * 4u + 16u : kEpiNowhere);
    unpack8(h, b);  // one of the two is 0
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      b[i] += __builtin_bit_cast(float, (uint32_t)f0[i]);
      b[4 + i] += __builtin_bit_cast(float, (uint32_t)f1[i]);
    }
  }
  __device__ __forceinline__ void fetch(int it, int r, int n) { next[it] = residual.load(at(r, n)); }
  __device__ __forceinline__ void arrived() {
#pragma unroll
    for (int i = 0; i < 4; ++i) res[i] = next[i];
  }
  __device__ __forceinline__ void apply(int it, int r, int n, float (&v)[8]) {
    const uint32_t off = at(r, n);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] += b[i];
    pre.store(off, pack8(v));
    with_act(act, [&](auto a_c) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = act_value<decltype(a_c)::value>(v[i]);
    });
    float x[8];
    unpack8(res[it], x);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] += x[i];
    out.store(off, pack8(v));
  }
};

// out = act(A . B + bias) + residual, one workgroup per block.
template <int BM, int BN, int BK, int WAVES, int STAGES, bool BT, bool NTB>
__global__ __launch_bounds__(WAVES * 64) void mm_epi_kernel(const EpiMM p, EpiOut e) {
  using C = EpiCfg<BM, BN, BK, WAVES, STAGES>;
  using G = typename C::G;
  __shared__ __attribute__((aligned(1024))) char smem[C::LDS_BYTES];
  int tm, tn;
  tile_coords((p.M + BM - 1) / BM, (p.N + BN - 1) / BN, p.group_m, tm, tn);
  f32x4_t acc[C::TM][C::TN];
  epi_main<BM, BN, BK, WAVES, STAGES, BT, NTB>(p, p.a, p.b, smem, tm, tn, 0, (p.K + BK - 1) / BK, acc);
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

// fp32 products of one part of K, rows ldw apart.
struct EpiPart {
  EpiRows ws;
  int ldw;
  __device__ __forceinline__ void init(const float* p, int M, int ld, int m0, int bm) {
    const long long rows = M - m0 < bm ? M - m0 : bm;
    ws.init(p, (long long)m0 * ld * 4, rows * ld * 4);
    ldw = ld;
  }
  __device__ __forceinline__ void columns(int) {}
  __device__ __forceinline__ void fetch(int, int, int) {}
  __device__ __forceinline__ void arrived() {}
  __device__ __forceinline__ void apply(int, int r, int n, float (&v)[8]) {
    const uint32_t off = n < ldw ? ((uint32_t)r * (uint32_t)ldw + (uint32_t)n) * 4u : kEpiNowhere;
    ws.store(off, __builtin_bit_cast(u32x4_t, f32x4_t{v[0], v[1], v[2], v[3]}));
    ws.store(n < ldw ? off + 16u : kEpiNowhere, __builtin_bit_cast(u32x4_t, f32x4_t{v[4], v[5], v[6], v[7]}));
  }
};

// The same over one of p.parts ranges of K tiles: fp32 products to
// ws[part][M][ldw], ldw = N rounded up to 8; epi_sum_kernel adds them.
template <int BM, int BN, int BK, int WAVES, int STAGES, bool BT, bool NTB>
__global__ __launch_bounds__(WAVES * 64) void mm_epi_split_kernel(const EpiMM p, float* __restrict__ ws, int ldw) {
  using C = EpiCfg<BM, BN, BK, WAVES, STAGES>;
  using G = typename C::G;
  __shared__ __attribute__((aligned(1024))) char smem[C::LDS_BYTES];
  int tm, tn, part;
  tile_coords_split((p.M + BM - 1) / BM, (p.N + BN - 1) / BN, p.group_m, p.parts, tm, tn, part);
  const int KT = (p.K + BK - 1) / BK, each = (KT + p.parts - 1) / p.parts, kt0 = part * each;
  f32x4_t acc[C::TM][C::TN];
  epi_main<BM, BN, BK, WAVES, STAGES, BT, NTB>(p, p.a, p.b, smem, tm, tn, kt0, KT - kt0 < each ? KT - kt0 : each,
                                                      acc);
  const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  EpiPart f;
  f.init(ws + (size_t)part * (size_t)p.M * (size_t)ldw, p.M, ldw, tm * BM, BM);
  epi_rows<C::TM, C::TN, C::TURN_ROW>(acc, smem, wave, lane, (wave / G::WN) * G::WTM, tn * BN + (wave % G::WN) * G::WTN, f);
}

}  // namespace mi
