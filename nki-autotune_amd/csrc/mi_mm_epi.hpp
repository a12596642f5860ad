// mi_mm_epi.hpp -- products of a K-contiguous A[M,K] whose epilogue does more
// than store: bias, activation and residual (matmul_epilogue), and the two
// bf16 halves of the Newton-Schulz iterates.
//
//   BT = false: out = A . B, B[K,N] (N contiguous; transposing operand reads)
//   BT = true:  out = A . B^T, B[N,K] (K contiguous, like A)
//
// The main loop is the pipelined core of mi_gemm.hpp (LDS-direct panel loads,
// STAGES K tiles in flight, operands of the next MFMA step read while this
// one runs, one barrier a K tile); here K tiles are 64 wide, so that a row of
// a K-contiguous panel is a whole 128-byte line and each line is requested
// once.  The MFMAs compute out^T per 32x32 tile: a lane ends with 4
// consecutive columns of one row.
//
// The epilogue turns each wave's accumulators in its own piece of LDS as
// fp32 (32 rows of 64 columns at a time, wave-private: no barrier), so that a
// lane then holds 8 consecutive columns and every access to bias, residual
// and outputs is a 16-byte piece of a whole line, and the values are rounded
// once, after the last operation.  Residual rows are requested before the
// turn and arrive behind it.
//
// SEG3: A and B are each two bf16 planes, hi + lo (lo `plane` elements after
// hi), and the K loop runs three times over: hi.hi, hi.lo, lo.hi.  lo.lo is
// under 2^-18 of the product and left out.
#pragma once
#include <type_traits>

#include "mi_act.hpp"
#include "mi_gemm.hpp"

namespace mi {

// Operands as the kernel reads them.  K is a multiple of 8 (SEG3: of BK), lda
// and ldb too; a_bytes, b_bytes: what lies behind the pointers (reads past it
// give 0).
struct EpiMM {
  const uint16_t *a, *b;
  uint32_t a_bytes, b_bytes;
  int M, N, K, lda, ldb, group_m, parts;
  uint32_t plane_a, plane_b;          // SEG3: bytes from hi to lo
  long long batch_a, batch_b;         // elements from one product's operand to the next's (blockIdx.y)
};

template <int BM, int BN, int BK, int WAVES, int STAGES>
struct EpiCfg {
  using G = WaveGrid<BM, BN, WAVES>;
  static constexpr int A_BYTES = BK * BM * 2;
  static constexpr int B_BYTES = BK * BN * 2;
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
  static constexpr int TURN_COLS = G::TN >= 2 ? 64 : 32;
  static constexpr int TURN_ROW = TURN_COLS * 4 + 16;  // + 16: rows start in different banks
  static constexpr int TURN_BYTES = WAVES * 32 * TURN_ROW;
  static constexpr int MAIN_BYTES = STAGES * STAGE_BYTES;
  static constexpr int LDS_BYTES = MAIN_BYTES > TURN_BYTES ? MAIN_BYTES : TURN_BYTES;
};

// acc = the products of K tiles [kt0, kt0 + kts) of block (tm, tn).
template <int BM, int BN, int BK, int WAVES, int STAGES, bool BT, bool NTB, bool SEG3>
__device__ __forceinline__ void epi_main(const EpiMM& p, const uint16_t* a, const uint16_t* b, char* smem, int tmi,
                                         int tni, int kt0, int kts,
                                         f32x16_t (&acc)[WaveGrid<BM, BN, WAVES>::TM][WaveGrid<BM, BN, WAVES>::TN]) {
  using C = EpiCfg<BM, BN, BK, WAVES, STAGES>;
  using G = typename C::G;
  static_assert(G::ok && BK % 32 == 0 && STAGES >= 2 && STAGES <= 4, "tile config");
  static_assert(C::LDS_BYTES <= kLdsBytesMax, "LDS over 160 KiB");
  constexpr int TM = G::TM, TN = G::TN, KS = BK / 16, NF = TM + TN;
  using LA = KPanelLoader<BK, BM, WAVES>;
  using LB = std::conditional_t<BT, KPanelLoader<BK, BN, WAVES>, PanelLoader<BK, BN, WAVES>>;
  constexpr int LPT = LA::LOADS_PER_TILE + LB::LOADS_PER_TILE;
  static_assert(LA::EVEN && LB::EVEN, "every wave issues the same number of loads (vm_wait counts them)");
  static_assert((STAGES - 1) * LPT < 64, "loads in flight exceed the 6-bit vmcnt");

  const int tid = (int)threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int m0 = tmi * BM, n0 = tni * BN;
  const int wm0 = (wave / G::WN) * G::WTM, wn0 = (wave % G::WN) * G::WTN;
  const int KT1 = (p.K + BK - 1) / BK;  // K tiles of one pass over K
  const int k_last = p.K - (KT1 - 1) * BK;
  LA la;
  LB lb;
  la.init(wave, lane, m0, p.lda, k_last, p.a_bytes);
  if constexpr (BT) lb.init(wave, lane, n0, p.ldb, k_last, p.b_bytes);
  else lb.init(wave, lane, n0, p.ldb);
  using FB = TrFrag<BN, TN, BK>;
  FB fb;
  if constexpr (!BT) fb.init(lane, wn0);
  // K-contiguous operands: lane l reads row l%32 of a fragment, K chunk
  // 2*kk + l/32 of the step, at its k_swz slot.
  const int arow = (wm0 + (lane & 31)) * (BK * 2), brow = (wn0 + (lane & 31)) * (BK * 2);
  int akoff[KS], bkoff[KS];
#pragma unroll
  for (int kk = 0; kk < KS; ++kk) {
    akoff[kk] = 16 * ((2 * kk + (lane >> 5)) ^ k_swz<BK>(wm0 + (lane & 31)));
    bkoff[kk] = 16 * ((2 * kk + (lane >> 5)) ^ k_swz<BK>(wn0 + (lane & 31)));
  }
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = f32x16_t{};

  bf16x8_t af[2][TM], bf[2][TN];
  auto read_frag = [&](int stage, int kk, int buf, int f) __attribute__((always_inline)) {
    const int abase = stage * C::STAGE_BYTES, bbase = abase + C::A_BYTES;
    if (f == 0 || f > TN) {
      const int t = f == 0 ? 0 : f - TN;
      af[buf][t] = __builtin_bit_cast(
          bf16x8_t, *(MI_LDS u32x4_t*)((MI_LDS char*)smem + abase + arow + t * 32 * (BK * 2) + akoff[kk]));
    } else {
      const int t = f - 1;
      if constexpr (BT)
        bf[buf][t] = __builtin_bit_cast(
            bf16x8_t, *(MI_LDS u32x4_t*)((MI_LDS char*)smem + bbase + brow + t * 32 * (BK * 2) + bkoff[kk]));
      else
        bf[buf][t] = read_tr_frag(smem, bbase + (kk * 16) * FB::ROWB + fb.off[t],
                                  bbase + (kk * 16 + 4) * FB::ROWB + fb.off[t]);
    }
  };
  auto read_frags = [&](int stage, int kk, int buf) __attribute__((always_inline)) {
#pragma unroll
    for (int f = 0; f < NF; ++f) read_frag(stage, kk, buf, f);
  };
  auto mfmas = [&](int buf) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j)
        acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(bf[buf][j], af[buf][i], acc[i][j], 0, 0, 0);
  };
  constexpr int READS = TM + (BT ? TN : 2 * TN);  // LDS reads of one step
  // Load q (< LPT) of K tile t of this block's range into `stage`.
  auto issue_one = [&](int q, int t, int stage) __attribute__((always_inline)) {
    const int kt = kt0 + t;
    int r = kt, hi_a = 0, hi_b = 0;
    if constexpr (SEG3) {
      hi_a = kt >= 2 * KT1;
      hi_b = kt >= KT1 && !hi_a;
      r = kt - (hi_a ? 2 * KT1 : hi_b ? KT1 : 0);
    }
    const bool tail = !SEG3 && kt == KT1 - 1;
    if (q < LA::LOADS_PER_TILE) {
      const uint32_t off = (uint32_t)r * (uint32_t)(BK * 2) + (SEG3 && hi_a ? p.plane_a : 0u);
      la.issue_at(q, make_rsrc_from(a, p.a_bytes, off), smem, stage * C::STAGE_BYTES, tail);
    } else {
      const uint32_t off = (uint32_t)r * (BT ? (uint32_t)(BK * 2) : (uint32_t)BK * (uint32_t)p.ldb * 2u) +
                           (SEG3 && hi_b ? p.plane_b : 0u);
      if constexpr (BT)
        lb.template issue_at<NTB>(q - LA::LOADS_PER_TILE, make_rsrc_from(b, p.b_bytes, off), smem,
                                  stage * C::STAGE_BYTES + C::A_BYTES, tail);
      else
        lb.template issue_at<NTB>(q - LA::LOADS_PER_TILE, make_rsrc_from(b, p.b_bytes, off), smem,
                                  stage * C::STAGE_BYTES + C::A_BYTES);
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

  // At the last step of tile t the wave waits for its loads of tile t+1,
  // meets the workgroup (tile t+1 is whole, tile t's buffer free), reads tile
  // t+1's first operands and requests tile t+STAGES.
  auto tile = [&](int t, auto cur_c) __attribute__((always_inline)) {
    constexpr int cur = decltype(cur_c)::value, nxt = (cur + 1) % STAGES;
#pragma unroll
    for (int kk = 0; kk + 1 < KS; ++kk) {
      read_frags(cur, kk + 1, (kk + 1) & 1);
      mfmas(kk & 1);
      interleave_mfma_ds<TM * TN, READS>();
    }
    vm_wait<(STAGES - 2) * LPT>();
    __syncthreads();
    const int t_new = clamp(t + STAGES);
#pragma unroll
    for (int f = 0; f < NF; ++f) {
      read_frag(nxt, 0, 0, f);
#pragma unroll
      for (int q = f * LPT / NF; q < (f + 1) * LPT / NF; ++q) issue_one(q, t_new, cur);
    }
    mfmas((KS - 1) & 1);
    interleave_mfma_ds<TM * TN, READS>();
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
  for (int kk = 0; kk < KS; ++kk) {
    if (kk + 1 < KS) read_frags(cur, kk + 1, (kk + 1) & 1);
    mfmas(kk & 1);
    interleave_mfma_ds<TM * TN, READS>();
  }
  wait_vmem();
  __syncthreads();  // the epilogue reuses the panel buffers
}

// Hands each lane 8 consecutive columns of the wave's accumulators at a time:
// f.columns(n) once per column group, f.fetch(it, m, n) before a turn and
// f.apply(it, m, n, v) after it, it < F::ROWS (rows a lane has per turn).
template <int TM, int TN, int ROWB, class F>
__device__ __forceinline__ void epi_rows(const f32x16_t (&acc)[TM][TN], char* smem, int wave, int lane, int row0,
                                         int col0, F& f) {
  constexpr int TW = TN >= 2 ? 2 : 1, LPR = 4 * TW, RPI = 64 / LPR, IT = 32 / RPI;
  static_assert(TN % TW == 0 && ROWB == TW * 128 + 16 && IT <= 4, "turn layout");
  MI_LDS char* slot = (MI_LDS char*)smem + wave * (32 * ROWB);
#pragma unroll
  for (int np = 0; np < TN / TW; ++np) {
    const int n = col0 + np * TW * 32 + 8 * (lane % LPR);
    f.columns(n);
#pragma unroll
    for (int mt = 0; mt < TM; ++mt) {
      const int m = row0 + mt * 32 + lane / LPR;
#pragma unroll
      for (int it = 0; it < IT; ++it) f.fetch(it, m + it * RPI, n);
#pragma unroll
      for (int h = 0; h < TW; ++h)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const f32x16_t& x = acc[mt][np * TW + h];
          const f32x4_t v = {x[4 * j], x[4 * j + 1], x[4 * j + 2], x[4 * j + 3]};
          *(MI_LDS f32x4_t*)(slot + (lane & 31) * ROWB + h * 128 + 32 * j + 16 * (lane >> 5)) = v;
        }
      wave_lds_turn();
#pragma unroll
      for (int it = 0; it < IT; ++it) {
        MI_LDS char* at = slot + (it * RPI + lane / LPR) * ROWB + 32 * (lane % LPR);
        const f32x4_t lo = *(MI_LDS f32x4_t*)at, hi = *(MI_LDS f32x4_t*)(at + 16);
        float v[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
        f.apply(it, m + it * RPI, n, v);
      }
      wave_lds_turn();
    }
  }
}

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
// every pointer 16-byte aligned; otherwise elements go one by one.
struct EpiOut {
  const void* bias;
  const uint16_t* residual;
  uint16_t *pre, *out;
  int M, N, act;
  bool bias_f32, vec;

  float b[8];
  u32x4_t res[4];

  __device__ __forceinline__ float bias_at(int n) const {
    return bias_f32 ? ((const float*)bias)[n] : bf16lo((uint32_t)((const uint16_t*)bias)[n]);
  }
  __device__ __forceinline__ void columns(int n) {
#pragma unroll
    for (int i = 0; i < 8; ++i) b[i] = 0.0f;
    if (!bias) return;
    if (vec && n < N) {
      if (bias_f32) {
        const f32x4_t lo = *(const f32x4_t*)((const float*)bias + n), hi = *(const f32x4_t*)((const float*)bias + n + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          b[i] = lo[i];
          b[4 + i] = hi[i];
        }
      } else {
        unpack8(*(const u32x4_t*)((const uint16_t*)bias + n), b);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (n + i < N) b[i] = bias_at(n + i);
    }
  }
  __device__ __forceinline__ void fetch(int it, int m, int n) {
    if (residual && vec && m < M && n < N) res[it] = *(const u32x4_t*)(residual + (size_t)m * (size_t)N + n);
  }
  __device__ __forceinline__ void apply(int it, int m, int n, float (&v)[8]) {
    if (m >= M || n >= N) return;
    const size_t at = (size_t)m * (size_t)N + n;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] += b[i];
    if (pre) {
      if (vec) {
        *(u32x4_t*)(pre + at) = pack8(v);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (n + i < N) pre[at + i] = (uint16_t)pack_bf16x2(v[i], 0.0f);
      }
    }
    with_act(act, [&](auto a_c) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = act_value<decltype(a_c)::value>(v[i]);
    });
    if (vec) {
      if (residual) {
        float r[8];
        unpack8(res[it], r);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] += r[i];
      }
      *(u32x4_t*)(out + at) = pack8(v);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (n + i < N) {
          if (residual) v[i] += bf16lo((uint32_t)residual[at + i]);
          out[at + i] = (uint16_t)pack_bf16x2(v[i], 0.0f);
        }
    }
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
  f32x16_t acc[G::TM][G::TN];
  epi_main<BM, BN, BK, WAVES, STAGES, BT, NTB, false>(p, p.a, p.b, smem, tm, tn, 0, (p.K + BK - 1) / BK, acc);
  const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  epi_rows<G::TM, G::TN, C::TURN_ROW>(acc, smem, wave, lane, tm * BM + (wave / G::WN) * G::WTM,
                                      tn * BN + (wave % G::WN) * G::WTN, e);
}

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
  f32x16_t acc[G::TM][G::TN];
  epi_main<BM, BN, BK, WAVES, STAGES, BT, NTB, false>(p, p.a, p.b, smem, tm, tn, kt0, KT - kt0 < each ? KT - kt0 : each,
                                                      acc);
  const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  constexpr int ROWS = partial_rows(WAVES, C::LDS_BYTES);
  store_partial<G::TM, G::TN, ROWS>(acc, ws + (size_t)part * (size_t)p.M * (size_t)ldw, smem, wave, lane, p.M, ldw,
                                    tm * BM + (wave / G::WN) * G::WTM, tn * BN + (wave % G::WN) * G::WTN);
}

}  // namespace mi
