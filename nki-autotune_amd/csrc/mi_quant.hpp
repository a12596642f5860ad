// mi_quant.hpp -- a matrix in 8-bit floating point with a scale for each block
// of 1 x 128 or 128 x 128 values, and the same of its transpose.
//
//   scale = max(fp32(max |x| / limit), 2^-100), limit 448 (e4m3) or 57344 (e5m2);
//           or the least power of two from max |x| / limit on (e8m0)
//   q = x / scale, rounded to fp32 and then to 8 bits, both to nearest even
//
// A block that holds an infinity or a NaN is NaN throughout, its scale too.
//
// A workgroup takes 128 x 128 values and reads them once: a lane keeps 8
// columns of 4 consecutive rows in registers (16 lanes read 128 values of a
// row), from which come the rows' maxima (over 16 lanes), the columns' (over
// the lanes and the 8 waves) or the block's.  q is written 8 bytes a lane; the
// transpose's bytes are turned in LDS, where a lane writes the 4 rows of a
// column at once, and written 16 bytes a lane.  (8 rows a lane of 256 threads:
// 1000 x 5000 with the transpose 12.7 us, so 9.2, 7.8 with a block for each of
// the two forms, in graphs; calls one after the other 8.7.)  Scales of 1 x 128 blocks lie with the rows consecutive, as
// the workgroup has them.
//
// Large matrices are bound by HBM (28672 x 8192 fp32 with the transpose 264 us,
// 5.3 TB/s), small ones by a block's arithmetic: 32 quotients a lane and form.
//
// The quotient: t = x inv with inv = fp32(1 / scale), then t + (x - t scale)
// inv in two fmas; a division's own sequence is 10 instructions.  t is within
// 1.5 units of x / scale, so what the last fma rounds is within 2^-22 of one of
// it, while a quotient of two fp32 numbers may be 2^-25 of one from halfway
// between two others.  The rest was checked by enumeration.  A last place that
// is off changes the 8-bit value only next to a border between two of them:
// for every significand of the scale, every border and the 9 fp32 numbers
// nearest to their product (1.2e9 pairs) the result is x / scale correctly
// rounded.  Exponents do not matter as long as no bit of the residual x - t
// scale falls below 2^-149.  Some do for scales under 2^-86 (e5m2; 2^-93 for
// e4m3), and values beside borders came out as their neighbours: blocks with
// scales below 2^-80 are divided with values and scale times 2^60 (but for the
// least scale, with which, a power of two, t is exact), behind branches of the
// wave, which cost 0.25 of 8.75 us for 1000 x 5000 bf16 with the transpose and
// 0.8 of 18.4 for 4096 x 4096.  (Values lifted in place behind one branch, or
// all quotients twice in the code behind one: as long for the first, 0.3 less
// for the second.)
//
// Maxima are taken of the bits without their sign, which order as the values
// do, with infinity and NaN above them.
#pragma once
#include "mi_norm.hpp"

namespace mi {

constexpr float kQuantMinScale = 0x1p-100f;
constexpr float kQuantSmall = 0x1p-80f, kQuantLift = 0x1p60f;
constexpr int kQuantThreads = 512;

struct Quant {
  const void* x;
  uint8_t *q, *q_t;      // rows ldq and ldq_t bytes apart, multiples of 16; NULL, and its scale too: not wanted
  void *scale, *scale_t;
  long long ldx, ldq, ldq_t;
  int M, K;
  bool e5m2, e8m0;
};

template <class T>
__device__ __forceinline__ uint32_t abs_bits(T x) {
  return __builtin_bit_cast(uint32_t, to_f32(x)) & 0x7FFFFFFFu;
}
__device__ __forceinline__ uint32_t max_bits(uint32_t a, uint32_t b) { return a > b ? a : b; }

// The scale of a block whose largest magnitude has these bits, and its
// reciprocal.
__device__ __forceinline__ void scale_of(uint32_t most, bool e5m2, bool e8m0, float& scale, float& inv) {
  if (most >= 0x7F800000u) {
    scale = inv = __builtin_nanf("");
    return;
  }
  if (e8m0) {
    // most = m 2^e, 1 <= m < 2; both limits are 1.75 times a power of two.
    int e = (int)(most >> 23) - 127 - (e5m2 ? 15 : 8) + ((most & 0x7FFFFFu) > 0x600000u ? 1 : 0);
    e = e < -100 ? -100 : e;
    scale = __builtin_bit_cast(float, (uint32_t)(e + 127) << 23);
    inv = __builtin_bit_cast(float, (uint32_t)(127 - e) << 23);
    return;
  }
  const float s = __builtin_bit_cast(float, most) / (e5m2 ? 57344.0f : 448.0f);
  scale = s > kQuantMinScale ? s : kQuantMinScale;
  inv = 1.0f / scale;
}
__device__ __forceinline__ float quotient(float x, float scale, float inv) {
  const float t = x * inv;
  return __builtin_fmaf(__builtin_fmaf(-t, scale, x), inv, t);
}
// Whether a lane of the wave has such a small scale.  (fp16 values have none but
// the least.)
template <class T>
__device__ __forceinline__ bool any_small(float scale) {
  return !std::is_same<T, Fp16>::value && __builtin_amdgcn_ballot_w64(scale < kQuantSmall && scale > kQuantMinScale) != 0;
}
template <int N>
__device__ __forceinline__ void divide(float (&t)[N], float scale, float inv, bool small) {
  if (small) {
    const bool own = scale < kQuantSmall;
    const float up = own ? kQuantLift : 1.0f;
    scale *= up;
    inv *= own ? 1.0f / kQuantLift : 1.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) t[i] *= up;
  }
#pragma unroll
  for (int i = 0; i < N; ++i) t[i] = quotient(t[i], scale, inv);
}
// Four values as bytes.
__device__ __forceinline__ uint32_t fp8x4(float a, float b, float c, float d, bool e5m2) {
  int v = 0;
  if (e5m2) {
    v = __builtin_amdgcn_cvt_pk_bf8_f32(a, b, v, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_bf8_f32(c, d, v, true);
  }
  v = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, v, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, v, true);
}
__device__ __forceinline__ void put_scale(void* p, size_t at, float scale, bool e8m0) {
  if (e8m0) ((uint8_t*)p)[at] = (uint8_t)(__builtin_bit_cast(uint32_t, scale) >> 23 & 0xFFu);
  else ((float*)p)[at] = scale;
}

// v shifted down by n places (0 to 7), zeros behind.
template <class T>
__device__ __forceinline__ void shift_down(Pack<T, 8>& v, int n) {
#pragma unroll
  for (int s = 4; s > 0; s >>= 1) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const T from = i + s < 8 ? v.v[i + s < 8 ? i + s : i] : T{};
      v.v[i] = n & s ? from : v.v[i];
    }
  }
}

// Keeps what was computed from v out of registers from here on: the compiler
// would hold 8 floats for each 4 registers of 16-bit values.
template <class T>
__device__ __forceinline__ void forget(Pack<T, 8>& v) {
  if constexpr (sizeof(T) == 2) {
    u32x4_t w = __builtin_bit_cast(u32x4_t, v);
    asm volatile("" : "+v"(w));
    v = __builtin_bit_cast(Pack<T, 8>, w);
  }
}

// Tile number `tile`; q where `rows`, q_t where `cols` (both the same for the
// whole block).
template <class T, bool SQUARE, bool TURNED>
__device__ __forceinline__ void quantize_tile(const Quant& p, unsigned tile, bool rows, bool cols) {
  constexpr int V = 8, R = 4, WAVES = kQuantThreads / 64;
  // A column's 128 bytes, its 16-byte pieces exchanged by column so that
  // writes of 16 columns spread over the banks.
  __shared__ __attribute__((aligned(16))) uint8_t turned[TURNED ? 128 * 128 : 16];
  __shared__ __attribute__((aligned(16))) uint32_t most_of[TURNED || SQUARE ? WAVES : 1][128];
  __shared__ __attribute__((aligned(16))) float col_scale[TURNED && !SQUARE ? 128 : 4], col_inv[TURNED && !SQUARE ? 128 : 4];
  __shared__ uint32_t half_most[2];  // or whether 64 columns' scales have a small one
  const int tid = (int)threadIdx.x, wave = tid >> 6;
  const int group = tid >> 4, in_row = tid & 15;  // rows 4 group .. 4 group + 3, columns 8 in_row ..
  const int tiles_k = (p.K + 127) / 128;
  const int tm = (int)(tile / (unsigned)tiles_k), tk = (int)(tile - (unsigned)tm * (unsigned)tiles_k);
  const int m0 = tm * 128 + group * R, k = tk * 128 + in_row * V;
  const T* x = (const T*)p.x;
  Pack<T, V> v[R];
  if (p.K >= V) {
    // (Past the row's end the last 8 values, of which those that are the
    // lane's own are kept; past the last row the last one.)
    const int at = k + V <= p.K ? k : p.K - V;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int m = m0 + r < p.M ? m0 + r : p.M - 1;
      v[r] = load_pack<T, V>(x + (size_t)m * (size_t)p.ldx + at);
    }
    if (at != k) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        if (k < p.K) shift_down(v[r], k - at);
        else v[r] = Pack<T, V>{};
      }
    }
    if (tm * 128 + 128 > p.M) {
#pragma unroll
      for (int r = 0; r < R; ++r)
        if (m0 + r >= p.M) v[r] = Pack<T, V>{};
    }
  } else {
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        v[r].v[i] = T{};
        if (m0 + r < p.M && k + i < p.K) v[r].v[i] = x[(size_t)(m0 + r) * (size_t)p.ldx + k + i];
      }
  }
  float all_scale = 0.0f, all_inv = 0.0f;
  if ((TURNED && cols) || SQUARE) {
    // The columns' maxima over the wave's 16 rows, then over the waves: a
    // thread to a column, which takes its scale (a division for each of the
    // 512 threads' 8 columns would be most of the kernel's work).
    uint32_t col[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      col[i] = 0;
#pragma unroll
      for (int r = 0; r < R; ++r) col[i] = max_bits(col[i], abs_bits(v[r].v[i]));
      col[i] = max_bits(col[i], __shfl_xor(col[i], 16));
      col[i] = max_bits(col[i], __shfl_xor(col[i], 32));
    }
    if ((tid & 63) < 16) {
      u32x4_t* to = (u32x4_t*)&most_of[wave][in_row * V];
      to[0] = u32x4_t{col[0], col[1], col[2], col[3]};
      to[1] = u32x4_t{col[4], col[5], col[6], col[7]};
    }
    __syncthreads();
    if (SQUARE || tid < 128) {
      const int c = tid & 127;
      uint32_t most = 0;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) most = max_bits(most, most_of[w][c]);
      if constexpr (SQUARE) {
        // (Each wave has 64 of the columns; the other half's maximum comes through LDS.)
#pragma unroll
        for (int s = 32; s > 0; s >>= 1) most = max_bits(most, __shfl_xor(most, s));
        if ((tid & 63) == 0 && tid < 128) half_most[tid >> 6] = most;
      } else {
        float scale, inv;
        scale_of(most, p.e5m2, p.e8m0, scale, inv);
        col_scale[c] = scale;
        col_inv[c] = inv;
        const bool small = any_small<T>(scale);
        if ((tid & 63) == 0) half_most[tid >> 6] = small;
        if (tk * 128 + c < p.K) put_scale(p.scale_t, (size_t)tm * (size_t)p.K + tk * 128 + c, scale, p.e8m0);
      }
    }
    if constexpr (SQUARE) {
      __syncthreads();
      scale_of(max_bits(half_most[0], half_most[1]), p.e5m2, p.e8m0, all_scale, all_inv);
      if (tid == 0) {
        if (rows) put_scale(p.scale, (size_t)tm * (size_t)tiles_k + tk, all_scale, p.e8m0);
        if (TURNED && cols) put_scale(p.scale_t, (size_t)tk * (size_t)((p.M + 127) / 128) + tm, all_scale, p.e8m0);
      }
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r) forget(v[r]);
  const int k_end = (p.K + 15) / 16 * 16, m_end = (p.M + 15) / 16 * 16;
  const bool edge_k = k + V > p.K;
  if (rows) {
    float scale[R], inv[R];
    bool small;
    if constexpr (!SQUARE) {
      uint32_t most[R];
#pragma unroll
      for (int r = 0; r < R; ++r) {
        most[r] = 0;
#pragma unroll
        for (int i = 0; i < V; ++i) most[r] = max_bits(most[r], abs_bits(v[r].v[i]));
      }
#pragma unroll
      for (int s = 8; s > 0; s >>= 1)
#pragma unroll
        for (int r = 0; r < R; ++r) most[r] = max_bits(most[r], __shfl_xor(most[r], s));
      // (Lane r of the row's 16 takes and writes row r's scale.)
      const int mine = in_row & 3;
      const uint32_t own = mine == 0 ? most[0] : mine == 1 ? most[1] : mine == 2 ? most[2] : most[3];
      float my_scale, my_inv;
      scale_of(own, p.e5m2, p.e8m0, my_scale, my_inv);
      small = any_small<T>(my_scale);
      if (in_row < R && m0 + in_row < p.M) put_scale(p.scale, (size_t)tk * (size_t)p.M + m0 + in_row, my_scale, p.e8m0);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        scale[r] = __shfl(my_scale, r, 16);
        inv[r] = __shfl(my_inv, r, 16);
      }
    } else {
      small = any_small<T>(all_scale);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        scale[r] = all_scale;
        inv[r] = all_inv;
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float t[V];
#pragma unroll
      for (int i = 0; i < V; ++i) t[i] = to_f32(v[r].v[i]);
      divide(t, scale[r], inv[r], small);
      if (edge_k) {
#pragma unroll
        for (int i = 0; i < V; ++i) t[i] = k + i < p.K ? t[i] : 0.0f;  // (a NaN scale leaves no zeros)
      }
      const u32x2_t w = {fp8x4(t[0], t[1], t[2], t[3], p.e5m2), fp8x4(t[4], t[5], t[6], t[7], p.e5m2)};
      if (m0 + r < p.M && k < k_end) *(u32x2_t*)(p.q + (size_t)(m0 + r) * (size_t)p.ldq + k) = w;
    }
  }
  if (TURNED && cols) {
    if constexpr (!SQUARE) __syncthreads();  // the columns' scales
    const bool edge_m = m0 + R > p.M;
#pragma unroll
    for (int r = 0; r < R; ++r) forget(v[r]);
    const bool small = SQUARE ? any_small<T>(all_scale)
                              : !std::is_same<T, Fp16>::value && __builtin_amdgcn_readfirstlane(half_most[0] | half_most[1]) != 0;
    f32x4_t scales = {}, invs = {};
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if constexpr (!SQUARE) {
        if (i % 4 == 0) {
          scales = *(const f32x4_t*)&col_scale[in_row * V + i];
          invs = *(const f32x4_t*)&col_inv[in_row * V + i];
        }
      }
      const float scale = SQUARE ? all_scale : scales[i % 4], inv = SQUARE ? all_inv : invs[i % 4];
      float t[R];
#pragma unroll
      for (int r = 0; r < R; ++r) t[r] = to_f32(v[r].v[i]);
      divide(t, scale, inv, small);
      if (edge_m) {
#pragma unroll
        for (int r = 0; r < R; ++r) t[r] = m0 + r < p.M ? t[r] : 0.0f;
      }
      *(uint32_t*)(turned + (in_row * V + i) * 128 + (((group >> 2) ^ (in_row & 7)) * 16 + (group & 3) * 4)) =
          fp8x4(t[0], t[1], t[2], t[3], p.e5m2);
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int c = j * 64 + (tid >> 3), piece = tid & 7, m = tm * 128 + piece * 16;
      const u32x4_t w = *(const u32x4_t*)(turned + c * 128 + (piece ^ ((c >> 3) & 7)) * 16);
      if (tk * 128 + c < p.K && m < m_end) *(u32x4_t*)(p.q_t + (size_t)(tk * 128 + c) * (size_t)p.ldq_t + m) = w;
    }
  }
}

// A grid of two rows: the first writes q, the second q_t.
template <class T, bool SQUARE, bool TURNED>
__global__ __launch_bounds__(kQuantThreads, sizeof(T) == 2 && !TURNED ? 8 : 6) void quantize_fp8_kernel(const Quant p) {
  const bool both = !TURNED || gridDim.y == 1;
  quantize_tile<T, SQUARE, TURNED>(p, blockIdx.x, p.q && (both || blockIdx.y == 0), both || blockIdx.y == 1);
}

// Rows of c bytes copied to rows of cp (a multiple of 16) with zeros behind:
// rows that start on 16 bytes.  (A row's last piece is 16 loads at once, of the
// last byte where they would pass it: a loop over the bytes that are there waits
// for each, 17 us for 1000 x 1501.)
struct PadBytes {
  const uint8_t* src;
  uint8_t* dst;
  long long rows, ld;
  int c, cp;
};
__device__ __forceinline__ void pad_bytes(const PadBytes& p, long long first, long long step) {
  const int groups = p.cp / 16;
  const long long n = p.rows * groups;
  for (long long i = first; i < n; i += step) {
    const long long r = n < 1ll << 31 ? (long long)((uint32_t)i / (uint32_t)groups) : i / groups;
    const int d = (int)(i - r * groups) * 16;
    const uint8_t* s = p.src + (size_t)r * (size_t)p.ld + d;
    Pack<uint8_t, 16> v;
    if (d + 16 <= p.c) {
      v = load_pack<uint8_t, 16>(s);
    } else {
#pragma unroll
      for (int k = 0; k < 16; ++k) v.v[k] = s[d + k < p.c ? k : p.c - 1 - d];
#pragma unroll
      for (int k = 0; k < 16; ++k) v.v[k] = d + k < p.c ? v.v[k] : (uint8_t)0;
    }
    *(u32x4_t*)(p.dst + (size_t)r * (size_t)p.cp + d) = __builtin_bit_cast(u32x4_t, v);
  }
}
struct PadAll {
  PadBytes op[4];
};

// The gradients' 8-bit form, and behind its blocks (`tiles`, or that many for
// each of q and q_t) the padded copies of up to two operands: pad_blocks each.
struct QuantPad {
  Quant q;
  PadBytes op[2];
  unsigned tiles, quant_blocks, pad_blocks;
};
template <class T>
__global__ __launch_bounds__(kQuantThreads, 6) void quantize_pad_kernel(const QuantPad p) {
  if (blockIdx.x < p.quant_blocks) {
    const bool both = p.quant_blocks == p.tiles, turn = blockIdx.x >= p.tiles;
    quantize_tile<T, false, true>(p.q, turn ? blockIdx.x - p.tiles : blockIdx.x, p.q.q && !turn, both || turn);
    return;
  }
  const unsigned at = blockIdx.x - p.quant_blocks;
  const bool second = at >= p.pad_blocks;
  pad_bytes(p.op[second], (long long)(second ? at - p.pad_blocks : at) * kQuantThreads + (long long)threadIdx.x,
            (long long)p.pad_blocks * kQuantThreads);
}

}  // namespace mi
