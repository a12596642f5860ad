// mi_ns.hpp -- a matrix orthogonalised by Newton-Schulz products.
//
//   X_0 = G / (||G||_F + eps)          (G^T where G has more rows than columns)
//   A = X X^T;  B = b A + c A A;  X <- a X + B X
//
// Each step maps every singular value s to a s + b s^3 + c s^5.  With the
// usual coefficients (slope 3.44 at 0) five steps multiply what rounding
// leaves next to a small singular value by up to 480, so iterates of one bf16
// each end about 1e-2 off.  X, A and B are therefore held as two bf16 planes,
// hi = bf16(v) and lo = bf16(v - hi) (together within 2^-18 of v), and a
// product is three passes of the bf16 MFMA over K, hi.hi + hi.lo + lo.hi, in
// one fp32 accumulator (SEG3 of mi_mm_epi.hpp): 16 bits of each factor for
// three times the work, where the fp32 MFMA gives 24 for sixteen times.
//
// Rows of X, A and B are [hi | lo], each half padded to a multiple of 64
// columns.  The padding is zero and stays so: its columns are products with
// rows past the end, which read as zeros.
#pragma once
#include "mi_mm_epi.hpp"

namespace mi {

// alpha * acc + beta * (c_hi + c_lo), as planes (out), or rounded once to
// bf16 (last).  N: the padded width of the planes, a multiple of 64.
struct NsOut {
  const uint16_t* c;  // NULL: 0
  uint16_t* out;      // planes, NULL where last is given
  uint16_t* last;     // [M][N]
  int M, N, ld;       // ld of c and out
  float alpha, beta;
  long long batch_c, batch_out, batch_last;
};
struct NsRows {
  EpiRows c, out, last;
  int N, ld;
  float alpha, beta;
  u32x4_t nhi[4], nlo[4], hi[4], lo[4];

  __device__ __forceinline__ void init(const NsOut& o, long long z, int m0, int bm) {
    const long long rows = o.M - m0 < bm ? o.M - m0 : bm;
    c.init(o.c ? o.c + z * o.batch_c : nullptr, (long long)m0 * o.ld * 2, rows * o.ld * 2);
    out.init(o.out ? o.out + z * o.batch_out : nullptr, (long long)m0 * o.ld * 2, rows * o.ld * 2);
    last.init(o.last ? o.last + z * o.batch_last : nullptr, (long long)m0 * o.N * 2, rows * o.N * 2);
    N = o.N;
    ld = o.ld;
    alpha = o.alpha;
    beta = o.beta;
  }
  __device__ __forceinline__ uint32_t at(int r, int n, int width) const {
    return n < N ? ((uint32_t)r * (uint32_t)width + (uint32_t)n) * 2u : kEpiNowhere;
  }
  __device__ __forceinline__ void columns(int) {}
  __device__ __forceinline__ void fetch(int it, int r, int n) {
    nhi[it] = c.load(at(r, n, ld));
    nlo[it] = c.load(n < N ? at(r, n, ld) + (uint32_t)N * 2u : kEpiNowhere);
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
    const u32x4_t top = pack8(v);
    unpack8(top, h);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] -= h[i];
    const uint32_t off = at(r, n, ld);
    out.store(off, top);
    out.store(n < N ? off + (uint32_t)N * 2u : kEpiNowhere, pack8(v));
    last.store(at(r, n, N), top);
  }
};

// One product of planes, blockIdx.y the matrix of the batch.
template <int BM, int BN, int BK, int WAVES, int STAGES, bool BT>
__global__ __launch_bounds__(WAVES * 64) void ns_product_kernel(const EpiMM p, const NsOut o) {
  using C = EpiCfg<BM, BN, BK, WAVES, STAGES>;
  using G = typename C::G;
  __shared__ __attribute__((aligned(1024))) char smem[C::LDS_BYTES];
  int tm, tn;
  tile_coords((p.M + BM - 1) / BM, (p.N + BN - 1) / BN, p.group_m, tm, tn);
  const long long z = blockIdx.y;
  f32x4_t acc[C::TM][C::TN];
  epi_main<BM, BN, BK, WAVES, STAGES, BT, false, true>(p, p.a + z * p.batch_a, p.b + z * p.batch_b, smem, tm, tn, 0,
                                                       3 * (p.K / BK), acc);
  const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  NsRows rows;
  rows.init(o, z, tm * BM, BM);
  epi_rows<C::TM, C::TN, C::TURN_ROW>(acc, smem, wave, lane, (wave / G::WN) * G::WTM, tn * BN + (wave % G::WN) * G::WTN,
                                      rows);
}

}  // namespace mi
