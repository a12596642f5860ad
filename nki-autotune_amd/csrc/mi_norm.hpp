// mi_norm.hpp -- layer norm over the rows of x[rows, D], and its gradients.
//
//   mean_r = sum_d x / D;  var_r = sum_d (x - mean_r)^2 / D;  rstd_r = 1 / sqrt(var_r + eps)
//   y = (x - mean_r) * rstd_r * weight_d + bias_d
//
//   xh = (x - mean_r) * rstd_r;  g = dout * weight_d
//   dx = rstd_r * (g - sum_d g / D - xh * sum_d (g * xh) / D)
//   dweight_d = sum_r dout * xh;  dbias_d = sum_r dout
//
// All sums are fp32 in an order fixed by the sizes, so results do not depend
// on timing; each output is rounded once.
//
// Both passes read every row once: its E values per lane stay in registers
// between the sums and the output, so the bytes that cross HBM are the
// tensors' own.  A row belongs to WPR waves (WPR * 64 lanes of E values).
// The gradient's blocks walk over many rows and keep the column sums of
// dweight and dbias in registers too (2 * E per lane); each block writes one
// row of partial sums, and column_sum_kernel adds those in block order.
//
// x, dout: bf16, fp16 or fp32 (T); weight and bias: T or fp32 (a run-time
// flag: a wave-uniform branch per group of loads).  VW consecutive values
// per load: 16 bytes (8, or 4 of fp32) where every row starts on 16 bytes,
// else 1, lanes next to each other either way.
#pragma once
#include <hip/hip_runtime.h>
#include <hip/hip_fp16.h>
#include <stdint.h>

#include "mi_gemm.hpp"

namespace mi {

struct Bf16 {
  uint16_t v;
};
struct Fp16 {
  uint16_t v;
};

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(Bf16 x) { return __builtin_bit_cast(float, (uint32_t)x.v << 16); }
__device__ __forceinline__ float to_f32(Fp16 x) { return (float)__builtin_bit_cast(_Float16, x.v); }
// Round to nearest even.
template <class T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ Bf16 from_f32<Bf16>(float x) { return Bf16{__builtin_bit_cast(uint16_t, (__bf16)x)}; }
template <>
__device__ __forceinline__ Fp16 from_f32<Fp16>(float x) { return Fp16{__builtin_bit_cast(uint16_t, (_Float16)x)}; }

// V consecutive values: one access where they fill 16 (or, fp32 by 8, 32)
// bytes.
template <class T, int V>
struct alignas(V * sizeof(T) < 16 ? V * sizeof(T) : 16) Pack {
  T v[V];
};
template <class T, int V>
__device__ __forceinline__ void load_f32(const T* __restrict__ p, float (&out)[V]) {
  const Pack<T, V> x = *(const Pack<T, V>*)p;
#pragma unroll
  for (int i = 0; i < V; ++i) out[i] = to_f32(x.v[i]);
}
template <class T, int V>
__device__ __forceinline__ void store_f32(T* __restrict__ p, const float (&in)[V]) {
  Pack<T, V> x;
#pragma unroll
  for (int i = 0; i < V; ++i) x.v[i] = from_f32<T>(in[i]);
  *(Pack<T, V>*)p = x;
}
// A row of parameters: T, or fp32 where `f32`.
template <class T, int V>
__device__ __forceinline__ void load_param(const void* p, bool f32, size_t at, float (&out)[V]) {
  if (f32) load_f32<float, V>((const float*)p + at, out);
  else load_f32<T, V>((const T*)p + at, out);
}

template <int V>
__device__ __forceinline__ void fill(float (&x)[V], float to) {
#pragma unroll
  for (int i = 0; i < V; ++i) x[i] = to;
}

// Sums a and b over the WPR waves of a row: every lane gets both.  `turn`
// counts the calls: with more than one wave the sums cross LDS in two places
// used by turns, so one barrier a call is enough (a wave can only be one
// call ahead of the others).
template <int WPR>
__device__ __forceinline__ void row_sum2(float& a, float& b, float (*xs)[WPR][2], int wave, int lane, int& turn) {
#pragma unroll
  for (int s = 32; s > 0; s >>= 1) {
    a += __shfl_xor(a, s);
    b += __shfl_xor(b, s);
  }
  if constexpr (WPR > 1) {
    if (lane == 0) {
      xs[turn & 1][wave][0] = a;
      xs[turn & 1][wave][1] = b;
    }
    __syncthreads();
    a = 0.0f;
    b = 0.0f;
#pragma unroll
    for (int w = 0; w < WPR; ++w) {
      a += xs[turn & 1][w][0];
      b += xs[turn & 1][w][1];
    }
    ++turn;
  }
}

// 1 / sqrt(var + eps); a variance that rounding left below 0 counts as 0, a
// NaN stays one.
__device__ __forceinline__ float norm_rstd(float var, float eps) {
  return 1.0f / __builtin_sqrtf((var < 0.0f ? 0.0f : var) + eps);
}

struct LnFwd {
  const void *x, *weight, *bias;  // weight, bias: NULL for 1 and 0
  void* y;
  float *mean, *rstd;  // NULL: not written
  long long rows, ldx;
  int D;
  float eps;
  bool params_f32;
};

// WPR == 1: blocks of 4 waves, a row each; otherwise a block per row.
template <class T, int VW, int E, int WPR>
__global__ __launch_bounds__(WPR == 1 ? 256 : WPR * 64) void layer_norm_kernel(const LnFwd p) {
  constexpr int G = E / VW, RPB = WPR == 1 ? 4 : 1;
  __shared__ float xs[2][WPR][2];
  const int tid = (int)threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int in_row = WPR == 1 ? lane : tid;
  const float inv_d = 1.0f / (float)p.D;
  int turn = 0;
  for (long long r = (long long)blockIdx.x * RPB + (WPR == 1 ? wave : 0); r < p.rows; r += (long long)gridDim.x * RPB) {
    const T* x = (const T*)p.x + (size_t)r * (size_t)p.ldx;
    float v[G][VW];
    float sum = 0.0f, none = 0.0f;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const int d = (g * WPR * 64 + in_row) * VW;
      if (d < p.D) load_f32<T, VW>(x + d, v[g]);
      else fill(v[g], 0.0f);
    }
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int i = 0; i < VW; ++i) sum += v[g][i];
    row_sum2<WPR>(sum, none, xs, wave, lane, turn);
    float mean = sum * inv_d;
    // The centred values' own sum is what rounding left in the mean: taken
    // out again, so rows far from zero keep their digits.
    float rest = 0.0f, sq = 0.0f;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const bool in = (g * WPR * 64 + in_row) * VW < p.D;
#pragma unroll
      for (int i = 0; i < VW; ++i) {
        v[g][i] = in ? v[g][i] - mean : 0.0f;
        rest += v[g][i];
        sq += v[g][i] * (v[g][i] * inv_d);  // a share of the mean each: the sum stays in range wherever the variance does
      }
    }
    row_sum2<WPR>(rest, sq, xs, wave, lane, turn);
    rest *= inv_d;
    mean += rest;
    const float rstd = norm_rstd(sq - rest * rest, p.eps);
    T* y = (T*)p.y + (size_t)r * (size_t)p.D;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const int d = (g * WPR * 64 + in_row) * VW;
      if (d >= p.D) continue;
      float w[VW], b[VW], o[VW];
      if (p.weight) load_param<T, VW>(p.weight, p.params_f32, d, w);
      else fill(w, 1.0f);
      if (p.bias) load_param<T, VW>(p.bias, p.params_f32, d, b);
      else fill(b, 0.0f);
#pragma unroll
      for (int i = 0; i < VW; ++i) o[i] = (v[g][i] - rest) * rstd * w[i] + b[i];
      store_f32<T, VW>(y + d, o);
    }
    if (in_row == 0) {
      if (p.mean) p.mean[r] = mean;
      if (p.rstd) p.rstd[r] = rstd;
    }
  }
}

// Rows longer than registers hold: a block of 1024 per row reads it three
// times (from L2 after the first).
template <class T>
__global__ __launch_bounds__(1024) void layer_norm_long_kernel(const LnFwd p) {
  __shared__ float xs[2][16][2];
  const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const float inv_d = 1.0f / (float)p.D;
  int turn = 0;
  for (long long r = blockIdx.x; r < p.rows; r += gridDim.x) {
    const T* x = (const T*)p.x + (size_t)r * (size_t)p.ldx;
    float sum = 0.0f, none = 0.0f;
    for (int d = tid; d < p.D; d += 1024) sum += to_f32(x[d]);
    row_sum2<16>(sum, none, xs, wave, lane, turn);
    float mean = sum * inv_d, rest = 0.0f, sq = 0.0f;
    for (int d = tid; d < p.D; d += 1024) {
      const float c = to_f32(x[d]) - mean;
      rest += c;
      sq += c * (c * inv_d);
    }
    row_sum2<16>(rest, sq, xs, wave, lane, turn);
    rest *= inv_d;
    const float rstd = norm_rstd(sq - rest * rest, p.eps);
    T* y = (T*)p.y + (size_t)r * (size_t)p.D;
    for (int d = tid; d < p.D; d += 1024) {
      float w[1] = {1.0f}, b[1] = {0.0f};
      if (p.weight) load_param<T, 1>(p.weight, p.params_f32, d, w);
      if (p.bias) load_param<T, 1>(p.bias, p.params_f32, d, b);
      y[d] = from_f32<T>((to_f32(x[d]) - mean - rest) * rstd * w[0] + b[0]);
    }
    if (tid == 0) {
      if (p.mean) p.mean[r] = mean + rest;
      if (p.rstd) p.rstd[r] = rstd;
    }
  }
}

struct LnBwd {
  const void *dout, *x, *weight;
  const float *mean, *rstd;
  void* dx;      // NULL: not wanted
  float* part;   // [2][gridDim.x][D] partial sums of dweight and dbias; NULL: not wanted
  long long rows, lddout, ldx;
  int D;
  bool weight_f32;
};

// WAVES waves a block, WPR of them to a row.
template <class T, int VW, int E, int WPR, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void layer_norm_bwd_kernel(const LnBwd p) {
  constexpr int G = E / VW, RPB = WAVES / WPR;
  static_assert(WPR == 1 || RPB == 1, "a block holds single-wave rows or one row");
  __shared__ float xs[2][WPR][2];
  const int tid = (int)threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int in_row = WPR == 1 ? lane : tid;
  const float inv_d = 1.0f / (float)p.D;
  float dw[G][VW], db[G][VW];
#pragma unroll
  for (int g = 0; g < G; ++g) {
    fill(dw[g], 0.0f);
    fill(db[g], 0.0f);
  }
  int turn = 0;
  for (long long r = (long long)blockIdx.x * RPB + (WPR == 1 ? wave : 0); r < p.rows; r += (long long)gridDim.x * RPB) {
    const T* x = (const T*)p.x + (size_t)r * (size_t)p.ldx;
    const T* dout = (const T*)p.dout + (size_t)r * (size_t)p.lddout;
    const float mean = p.mean[r], rstd = p.rstd[r];
    Pack<T, VW> xv[G], dv[G];
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const int d = (g * WPR * 64 + in_row) * VW;
      if (d < p.D) {
        xv[g] = *(const Pack<T, VW>*)(x + d);
        dv[g] = *(const Pack<T, VW>*)(dout + d);
      }
    }
    float sg = 0.0f, sgx = 0.0f;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const int d = (g * WPR * 64 + in_row) * VW;
      if (d >= p.D) continue;
      float w[VW];
      if (p.weight) load_param<T, VW>(p.weight, p.weight_f32, d, w);
      else fill(w, 1.0f);
#pragma unroll
      for (int i = 0; i < VW; ++i) {
        const float dy = to_f32(dv[g].v[i]), xh = (to_f32(xv[g].v[i]) - mean) * rstd;
        dw[g][i] += dy * xh;
        db[g][i] += dy;
        sg += dy * w[i];
        sgx += dy * w[i] * xh;
      }
    }
    if (!p.dx) continue;
    row_sum2<WPR>(sg, sgx, xs, wave, lane, turn);
    sg *= inv_d;
    sgx *= inv_d;
    T* dx = (T*)p.dx + (size_t)r * (size_t)p.D;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const int d = (g * WPR * 64 + in_row) * VW;
      if (d >= p.D) continue;
      float w[VW], o[VW];
      if (p.weight) load_param<T, VW>(p.weight, p.weight_f32, d, w);
      else fill(w, 1.0f);
#pragma unroll
      for (int i = 0; i < VW; ++i) {
        const float xh = (to_f32(xv[g].v[i]) - mean) * rstd;
        o[i] = rstd * (to_f32(dv[g].v[i]) * w[i] - sg - xh * sgx);
      }
      store_f32<T, VW>(dx + d, o);
    }
  }
  if (!p.part) return;
  float* part_w = p.part + (size_t)blockIdx.x * (size_t)p.D;
  float* part_b = part_w + (size_t)gridDim.x * (size_t)p.D;
  if constexpr (RPB == 1) {
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const int d = (g * WPR * 64 + in_row) * VW;
      if (d >= p.D) continue;
      store_f32<float, VW>(part_w + d, dw[g]);
      store_f32<float, VW>(part_b + d, db[g]);
    }
  } else {
    // The waves' sums, in wave order: one group of columns at a time in LDS.
    __shared__ __attribute__((aligned(16))) float ws[RPB][64 * VW + 4];
    for (int k = 0; k < 2; ++k) {
#pragma unroll
      for (int g = 0; g < G; ++g) {
        if (g * 64 * VW >= p.D) break;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < VW; ++i) ws[wave][lane * VW + i] = k ? db[g][i] : dw[g][i];
        __syncthreads();
        for (int c = tid; c < 64 * VW; c += WAVES * 64) {
          const int d = g * 64 * VW + c;
          if (d >= p.D) break;
          float s = ws[0][c];
#pragma unroll
          for (int w = 1; w < RPB; ++w) s += ws[w][c];
          (k ? part_b : part_w)[d] = s;
        }
      }
    }
  }
}

// Rows longer than registers hold: dx by a block per row, and the column
// sums by layer_norm_columns_kernel.
template <class T>
__global__ __launch_bounds__(1024) void layer_norm_bwd_long_kernel(const LnBwd p) {
  __shared__ float xs[2][16][2];
  const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const float inv_d = 1.0f / (float)p.D;
  int turn = 0;
  for (long long r = blockIdx.x; r < p.rows; r += gridDim.x) {
    const T* x = (const T*)p.x + (size_t)r * (size_t)p.ldx;
    const T* dout = (const T*)p.dout + (size_t)r * (size_t)p.lddout;
    const float mean = p.mean[r], rstd = p.rstd[r];
    float sg = 0.0f, sgx = 0.0f;
    for (int d = tid; d < p.D; d += 1024) {
      float w[1] = {1.0f};
      if (p.weight) load_param<T, 1>(p.weight, p.weight_f32, d, w);
      const float g = to_f32(dout[d]) * w[0];
      sg += g;
      sgx += g * ((to_f32(x[d]) - mean) * rstd);
    }
    row_sum2<16>(sg, sgx, xs, wave, lane, turn);
    sg *= inv_d;
    sgx *= inv_d;
    T* dx = (T*)p.dx + (size_t)r * (size_t)p.D;
    for (int d = tid; d < p.D; d += 1024) {
      float w[1] = {1.0f};
      if (p.weight) load_param<T, 1>(p.weight, p.weight_f32, d, w);
      const float xh = (to_f32(x[d]) - mean) * rstd;
      dx[d] = from_f32<T>(rstd * (to_f32(dout[d]) * w[0] - sg - xh * sgx));
    }
  }
}

// Column sums over the rows of one chunk: blockIdx.x takes 256 columns,
// blockIdx.y (of gridDim.y) every gridDim.y-th row.  part: [2][gridDim.y][D].
template <class T>
__global__ __launch_bounds__(256) void layer_norm_columns_kernel(const LnBwd p) {
  const int d = (int)blockIdx.x * 256 + (int)threadIdx.x;
  if (d >= p.D) return;
  float dw = 0.0f, db = 0.0f;
  for (long long r = blockIdx.y; r < p.rows; r += gridDim.y) {
    const float dy = to_f32(((const T*)p.dout)[(size_t)r * (size_t)p.lddout + d]);
    dw += dy * ((to_f32(((const T*)p.x)[(size_t)r * (size_t)p.ldx + d]) - p.mean[r]) * p.rstd[r]);
    db += dy;
  }
  float* part_w = p.part + (size_t)blockIdx.y * (size_t)p.D;
  part_w[d] = dw;
  part_w[(size_t)gridDim.y * (size_t)p.D + d] = db;
}

// (A kernel rather than a memset: memset nodes of a captured graph have given
// wrong results on replays.)
static __global__ __launch_bounds__(256) void fill_zero_kernel(uint16_t* __restrict__ p, size_t n) {
  for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (size_t)gridDim.x * 256) p[i] = 0;
}

// out_k[d] = sum_i part[k][i][d] over i < parts, for the gridDim.y arrays k:
// 64 columns a block, its 16 waves taking turns over the parts and their
// sums added in wave order.
struct ColumnSum {
  const float* part;
  void* out[2];  // NULL: not wanted
  int parts, D;
};
template <class T>
__global__ __launch_bounds__(1024) void column_sum_kernel(const ColumnSum p) {
  __shared__ float xs[16][64];
  T* out = (T*)p.out[blockIdx.y];
  if (!out) return;
  const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
  const int d = (int)blockIdx.x * 64 + lane;
  const float* part = p.part + (size_t)blockIdx.y * (size_t)p.parts * (size_t)p.D;
  float s = 0.0f;
  if (d < p.D) {
    constexpr int U = 8;
    for (int i0 = wave; i0 < p.parts; i0 += 16 * U) {
      float v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = i0 + 16 * u;
        v[u] = i < p.parts ? part[(size_t)i * (size_t)p.D + d] : 0.0f;
      }
#pragma unroll
      for (int u = 0; u < U; ++u) s += v[u];
    }
  }
  xs[wave][lane] = s;
  __syncthreads();
  if (wave == 0 && d < p.D) {
#pragma unroll
    for (int w = 1; w < 16; ++w) s += xs[w][lane];
    out[d] = from_f32<T>(s);
  }
}

}  // namespace mi
