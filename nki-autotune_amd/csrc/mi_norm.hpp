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
// tensors' own.  A row belongs to L lanes (8 of a wave to 16
// waves).  Blocks walk over the rows with the parameters in registers and the
// next row's loads in flight behind this row's work; the gradient's keep the
// column sums of dweight and dbias in registers too (2 E a lane), add their
// rows' through LDS at the end, and each leaves one row of partial sums, which
// column_sum_kernel adds in block order.
//
// Every load and store is 16 bytes (8 values, 4 of fp32), aligned or not (the
// hardware takes any address), and none is in a branch: a wait for a load
// would otherwise wait for all of them.  Where a lane's values would pass the
// row's end, it takes the row's last 16 bytes, computes what the lanes that
// own them compute, stores the same, and leaves them out of the row's sums;
// rows past the last are the last one again, left out of the column sums.
//
// Bound by HBM: on one MI355X, where a large copy runs at 4.9 TB/s, 16384 x
// 8192 bf16 takes 98 us forward (5.5 TB/s; caches hold the last writes) and
// 16384 x 4096 backward 77 us (5.2 TB/s); at most of the odd sizes 0.8 to 0.95
// of that.  Few rows are bound by latency: 8 x 4096 2.3 us.
// Rows of 64 or fewer values are bound by the instructions of their sums.
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

// W consecutive values (16 bytes of them) at any address.
template <class T, int W = 16 / sizeof(T)>
struct __attribute__((packed, aligned(sizeof(T)))) Pack {
  static constexpr int V = W;
  T v[V];
};
template <class T, int W = 16 / sizeof(T)>
__device__ __forceinline__ Pack<T, W> load_pack(const T* p) {
  return *(const Pack<T, W>*)p;
}
template <class T, int W>
__device__ __forceinline__ void store_pack(T* p, const float (&in)[W]) {
  Pack<T, W> x;
#pragma unroll
  for (int i = 0; i < W; ++i) x.v[i] = from_f32<T>(in[i]);
  *(Pack<T, W>*)p = x;
}
// Packs of a row of parameters, T or (`f32`) fp32; `other` where there is none.
template <class T, int G, int W>
__device__ __forceinline__ void load_params(const void* p, bool f32, const int (&at)[G], float other, float (&out)[G][W]) {
  if (!p) {
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int i = 0; i < W; ++i) out[g][i] = other;
  } else if (f32) {
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const Pack<float, W> x = load_pack<float, W>((const float*)p + at[g]);
#pragma unroll
      for (int i = 0; i < W; ++i) out[g][i] = x.v[i];
    }
  } else {
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const Pack<T, W> x = load_pack<T, W>((const T*)p + at[g]);
#pragma unroll
      for (int i = 0; i < W; ++i) out[g][i] = to_f32(x.v[i]);
    }
  }
}

// Sums a and b over the L lanes of a row: every lane gets both.  `turn`
// counts the calls: with more than one wave the sums cross LDS in two places
// used by turns, so one barrier a call is enough (a wave can only be one call
// ahead of the others).  wave: within the row.
template <int L>
__device__ __forceinline__ void row_sum2(float& a, float& b, float (*xs)[L < 64 ? 1 : L / 64][2], int wave, int lane,
                                         int& turn) {
#pragma unroll
  for (int s = (L < 64 ? L : 64) / 2; s > 0; s >>= 1) {
    a += __shfl_xor(a, s);
    b += __shfl_xor(b, s);
  }
  if constexpr (L > 64) {
    if (lane == 0) {
      xs[turn & 1][wave][0] = a;
      xs[turn & 1][wave][1] = b;
    }
    __syncthreads();
    a = 0.0f;
    b = 0.0f;
#pragma unroll
    for (int w = 0; w < L / 64; ++w) {
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

// Where a lane's packs of a row lie, and which of their values are its own.
template <int V, int G, int L, bool EXACT>
struct RowSplit {
  int at[G];   // first element of pack g
  int own[G];  // its own are elements own[g] .. V - 1 of it
  __device__ __forceinline__ void init(int in_row, int D) {
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const int d = (g * L + in_row) * V;
      at[g] = EXACT || d + V <= D ? d : D - V;
      own[g] = EXACT ? 0 : d - at[g];
    }
  }
  __device__ __forceinline__ float mine(int g, int i, float x) const { return EXACT || i >= own[g] ? x : 0.0f; }
};

template <int V>
__device__ __forceinline__ void fill(float (&x)[V], float to) {
#pragma unroll
  for (int i = 0; i < V; ++i) x[i] = to;
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

// GROUPS rows at a time in a block of GROUPS * L threads.  EXACT: D = E * L.
// KEEP: the parameters and the next row stay in registers (E = 32 of 1024
// threads leaves no room for them).
template <class T, int E, int L, int GROUPS, bool EXACT, bool KEEP>
__global__ __launch_bounds__(L* GROUPS) void layer_norm_kernel(const LnFwd p) {
  constexpr int V = Pack<T>::V, G = E / V;
  static_assert(L <= 64 || GROUPS == 1, "rows of several waves have their block to themselves");
  __shared__ float xs[2][L < 64 ? 1 : L / 64][2];
  const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int in_row = tid % L;
  const float inv_d = 1.0f / (float)p.D;
  RowSplit<V, G, L, EXACT> split;
  split.init(in_row, p.D);
  const auto row_of = [&](long long r) { return r < p.rows ? r : p.rows - 1; };
  const long long step = (long long)gridDim.x * GROUPS;
  long long r = (long long)blockIdx.x * GROUPS + tid / L;
  Pack<T> next[G];
  const auto fetch = [&](long long at) __attribute__((always_inline)) {
    const T* x = (const T*)p.x + (size_t)at * (size_t)p.ldx;
#pragma unroll
    for (int g = 0; g < G; ++g) next[g] = load_pack(x + split.at[g]);
  };
  float w[KEEP ? G : 1][V], b[KEEP ? G : 1][V];
  if constexpr (KEEP) {
    fetch(row_of(r));
    load_params<T>(p.weight, p.params_f32, split.at, 1.0f, w);
    load_params<T>(p.bias, p.params_f32, split.at, 0.0f, b);
  }
  int turn = 0;
  for (long long first = (long long)blockIdx.x * GROUPS; first < p.rows; first += step, r += step) {
    float v[G][V];
    if constexpr (!KEEP) fetch(row_of(r));
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int i = 0; i < V; ++i) v[g][i] = to_f32(next[g].v[i]);
    if constexpr (KEEP) fetch(row_of(r + step));
    float sum = 0.0f, none = 0.0f;
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int i = 0; i < V; ++i) sum += split.mine(g, i, v[g][i]);
    row_sum2<L>(sum, none, xs, wave, lane, turn);
    float mean = sum * inv_d;
    // The centred values' own sum is what rounding left in the mean: taken
    // out again, so rows far from zero keep their digits.
    float rest = 0.0f, sq = 0.0f;
#pragma unroll
    for (int g = 0; g < G; ++g) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        v[g][i] -= mean;
        const float c = split.mine(g, i, v[g][i]);
        rest += c;
        sq += c * (c * inv_d);  // a share of the mean each: the sum stays in range wherever the variance does
      }
    }
    row_sum2<L>(rest, sq, xs, wave, lane, turn);
    rest *= inv_d;
    mean += rest;
    const float rstd = norm_rstd(sq - rest * rest, p.eps);
    T* y = (T*)p.y + (size_t)row_of(r) * (size_t)p.D;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      constexpr int K = KEEP ? 1 : 0;
      if constexpr (!KEEP) {
        // (Read again for each row, not once and then spilled.)
        const void *weight = p.weight, *bias = p.bias;
        asm volatile("" : "+s"(weight), "+s"(bias));
        const int at[1] = {split.at[g]};
        load_params<T>(weight, p.params_f32, at, 1.0f, w);
        load_params<T>(bias, p.params_f32, at, 0.0f, b);
      }
      float o[V];
#pragma unroll
      for (int i = 0; i < V; ++i) o[i] = (v[g][i] - rest) * rstd * w[K * g][i] + b[K * g][i];
      store_pack(y + split.at[g], o);
    }
    if (in_row == 0 && r < p.rows) {
      if (p.mean) p.mean[r] = mean;
      if (p.rstd) p.rstd[r] = rstd;
    }
  }
}

// Rows longer than registers hold (W = 16 bytes), or shorter than 16 bytes (W
// = 1): a block of B threads per row reads it three times (from L2 after the
// first).  f(at, own) for each of a thread's packs.
template <int B, int W, class F>
__device__ __forceinline__ void each_pack(int tid, int D, F&& f) {
  for (int d = tid * W; d < D; d += B * W) {
    const int at = d + W <= D ? d : D - W;
    f(at, d - at);
  }
}
template <class T, int B, int W>
__global__ __launch_bounds__(B) void layer_norm_long_kernel(const LnFwd p) {
  __shared__ float xs[2][B / 64][2];
  const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const float inv_d = 1.0f / (float)p.D;
  int turn = 0;
  for (long long r = blockIdx.x; r < p.rows; r += gridDim.x) {
    const T* x = (const T*)p.x + (size_t)r * (size_t)p.ldx;
    float sum = 0.0f, none = 0.0f;
    each_pack<B, W>(tid, p.D, [&](int at, int own) __attribute__((always_inline)) {
      const Pack<T, W> v = load_pack<T, W>(x + at);
#pragma unroll
      for (int i = 0; i < W; ++i) sum += i >= own ? to_f32(v.v[i]) : 0.0f;
    });
    row_sum2<B>(sum, none, xs, wave, lane, turn);
    float mean = sum * inv_d, rest = 0.0f, sq = 0.0f;
    each_pack<B, W>(tid, p.D, [&](int at, int own) __attribute__((always_inline)) {
      const Pack<T, W> v = load_pack<T, W>(x + at);
#pragma unroll
      for (int i = 0; i < W; ++i) {
        const float c = i >= own ? to_f32(v.v[i]) - mean : 0.0f;
        rest += c;
        sq += c * (c * inv_d);
      }
    });
    row_sum2<B>(rest, sq, xs, wave, lane, turn);
    rest *= inv_d;
    const float rstd = norm_rstd(sq - rest * rest, p.eps);
    T* y = (T*)p.y + (size_t)r * (size_t)p.D;
    each_pack<B, W>(tid, p.D, [&](int at, int) __attribute__((always_inline)) {
      const Pack<T, W> v = load_pack<T, W>(x + at);
      float w[1][W], b[1][W], o[W];
      const int where[1] = {at};
      load_params<T>(p.weight, p.params_f32, where, 1.0f, w);
      load_params<T>(p.bias, p.params_f32, where, 0.0f, b);
#pragma unroll
      for (int i = 0; i < W; ++i) o[i] = (to_f32(v.v[i]) - mean - rest) * rstd * w[0][i] + b[0][i];
      store_pack(y + at, o);
    });
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

// GROUPS rows at a time in a block of GROUPS * L threads; EXACT: as above.
template <class T, int E, int L, int GROUPS, bool EXACT>
__global__ __launch_bounds__(L* GROUPS) void layer_norm_bwd_kernel(const LnBwd p) {
  constexpr int V = Pack<T>::V, G = E / V, WPR = L < 64 ? 1 : L / 64;
  __shared__ float xs[GROUPS][2][WPR][2];
  __shared__ float cols[GROUPS > 1 ? GROUPS : 1][GROUPS > 1 ? L * V : 1];
  const int tid = (int)threadIdx.x, lane = tid & 63;
  const int in_row = tid % L, group = tid / L, wave = in_row >> 6;
  const float inv_d = 1.0f / (float)p.D;
  RowSplit<V, G, L, EXACT> split;
  split.init(in_row, p.D);
  const auto row_of = [&](long long r) { return r < p.rows ? r : p.rows - 1; };
  const long long step = (long long)gridDim.x * GROUPS;
  long long r = (long long)blockIdx.x * GROUPS + group;
  Pack<T> nx[G], nd[G];
  float nmean, nrstd;
  const auto fetch = [&](long long at) __attribute__((always_inline)) {
    const T* x = (const T*)p.x + (size_t)at * (size_t)p.ldx;
    const T* dout = (const T*)p.dout + (size_t)at * (size_t)p.lddout;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      nx[g] = load_pack(x + split.at[g]);
      nd[g] = load_pack(dout + split.at[g]);
    }
    nmean = p.mean[at];
    nrstd = p.rstd[at];
  };
  float w[G][V], dw[G][V], db[G][V];
  fetch(row_of(r));
  load_params<T>(p.weight, p.weight_f32, split.at, 1.0f, w);
#pragma unroll
  for (int g = 0; g < G; ++g) {
    fill(dw[g], 0.0f);
    fill(db[g], 0.0f);
  }
  int turn = 0;
  for (long long first = (long long)blockIdx.x * GROUPS; first < p.rows; first += step, r += step) {
    Pack<T> xv[G], dv[G];
#pragma unroll
    for (int g = 0; g < G; ++g) {
      xv[g] = nx[g];
      dv[g] = nd[g];
    }
    const float mean = nmean, rstd = nrstd;
    fetch(row_of(r + step));
    const bool live = r < p.rows;
    float sg = 0.0f, sgx = 0.0f;
#pragma unroll
    for (int g = 0; g < G; ++g) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float dy = to_f32(dv[g].v[i]), xh = (to_f32(xv[g].v[i]) - mean) * rstd;
        const float counted = live ? dy : 0.0f;
        dw[g][i] += live ? dy * xh : 0.0f;
        db[g][i] += counted;
        const float gw = split.mine(g, i, dy * w[g][i]);
        sg += gw;
        sgx += split.mine(g, i, gw * xh);
      }
    }
    if (!p.dx) continue;
    row_sum2<L>(sg, sgx, xs[group], wave, lane, turn);
    sg *= inv_d;
    sgx *= inv_d;
    T* dx = (T*)p.dx + (size_t)row_of(r) * (size_t)p.D;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      float o[V];
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float xh = (to_f32(xv[g].v[i]) - mean) * rstd;
        o[i] = rstd * (to_f32(dv[g].v[i]) * w[g][i] - sg - xh * sgx);
      }
      store_pack(dx + split.at[g], o);
    }
  }
  if (!p.part) return;
  float* part_w = p.part + (size_t)blockIdx.x * (size_t)p.D;
  float* part_b = part_w + (size_t)gridDim.x * (size_t)p.D;
  if constexpr (GROUPS == 1) {
#pragma unroll
    for (int g = 0; g < G; ++g) {
      store_pack(part_w + split.at[g], dw[g]);
      store_pack(part_b + split.at[g], db[g]);
    }
  } else {
    // The groups' sums in their order, one pack of columns at a time.
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int g = 0; g < G; ++g) {
        if (g * L * V >= p.D) break;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < V; ++i) cols[group][in_row * V + i] = k ? db[g][i] : dw[g][i];
        __syncthreads();
        for (int c = tid; c < L * V; c += L * GROUPS) {
          const int d = g * L * V + c / V * V, at = d + V <= p.D ? d : p.D - V;
          float s = cols[0][c];
#pragma unroll
          for (int q = 1; q < GROUPS; ++q) s += cols[q][c];
          (k ? part_b : part_w)[at + c % V] = s;
        }
      }
  }
}

// Rows longer than registers hold, or shorter than 16 bytes: dx by a block of
// B threads per row, and the column sums by layer_norm_columns_kernel.
template <class T, int B, int W>
__global__ __launch_bounds__(B) void layer_norm_bwd_long_kernel(const LnBwd p) {
  __shared__ float xs[2][B / 64][2];
  const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const float inv_d = 1.0f / (float)p.D;
  int turn = 0;
  for (long long r = blockIdx.x; r < p.rows; r += gridDim.x) {
    const T* x = (const T*)p.x + (size_t)r * (size_t)p.ldx;
    const T* dout = (const T*)p.dout + (size_t)r * (size_t)p.lddout;
    const float mean = p.mean[r], rstd = p.rstd[r];
    // f(at, own, g, xh): a pack's dout * weight and normalised values.
    const auto each = [&](auto&& f) __attribute__((always_inline)) {
      each_pack<B, W>(tid, p.D, [&](int at, int own) __attribute__((always_inline)) {
        const Pack<T, W> v = load_pack<T, W>(x + at), d = load_pack<T, W>(dout + at);
        float w[1][W], g[W], xh[W];
        const int where[1] = {at};
        load_params<T>(p.weight, p.weight_f32, where, 1.0f, w);
#pragma unroll
        for (int i = 0; i < W; ++i) {
          g[i] = to_f32(d.v[i]) * w[0][i];
          xh[i] = (to_f32(v.v[i]) - mean) * rstd;
        }
        f(at, own, g, xh);
      });
    };
    float sg = 0.0f, sgx = 0.0f;
    each([&](int, int own, const float(&g)[W], const float(&xh)[W]) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < W; ++i) {
        sg += i >= own ? g[i] : 0.0f;
        sgx += i >= own ? g[i] * xh[i] : 0.0f;
      }
    });
    row_sum2<B>(sg, sgx, xs, wave, lane, turn);
    sg *= inv_d;
    sgx *= inv_d;
    T* dx = (T*)p.dx + (size_t)r * (size_t)p.D;
    each([&](int at, int, const float(&g)[W], const float(&xh)[W]) __attribute__((always_inline)) {
      float o[W];
#pragma unroll
      for (int i = 0; i < W; ++i) o[i] = rstd * (g[i] - sg - xh[i] * sgx);
      store_pack(dx + at, o);
    });
  }
}

// Column sums over the rows of one chunk: blockIdx.x takes 256 packs of
// columns, blockIdx.y (of gridDim.y) every gridDim.y-th row.  part:
// [2][gridDim.y][D].
template <class T, int W>
__global__ __launch_bounds__(256) void layer_norm_columns_kernel(const LnBwd p) {
  const int d = ((int)blockIdx.x * 256 + (int)threadIdx.x) * W;
  if (d >= p.D) return;
  const int at = d + W <= p.D ? d : p.D - W;
  float dw[W], db[W];
  fill(dw, 0.0f);
  fill(db, 0.0f);
#pragma unroll 4
  for (long long r = blockIdx.y; r < p.rows; r += gridDim.y) {
    const Pack<T, W> v = load_pack<T, W>((const T*)p.x + (size_t)r * (size_t)p.ldx + at);
    const Pack<T, W> g = load_pack<T, W>((const T*)p.dout + (size_t)r * (size_t)p.lddout + at);
    const float mean = p.mean[r], rstd = p.rstd[r];
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const float dy = to_f32(g.v[i]);
      dw[i] += dy * ((to_f32(v.v[i]) - mean) * rstd);
      db[i] += dy;
    }
  }
  float* part_w = p.part + (size_t)blockIdx.y * (size_t)p.D + at;
  store_pack(part_w, dw);
  store_pack(part_w + (size_t)gridDim.y * (size_t)p.D, db);
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
  int parts, D, first;  // first: of this launch's columns
};
template <class T>
__global__ __launch_bounds__(1024) void column_sum_kernel(const ColumnSum p) {
  __shared__ float xs[16][64];
  T* out = (T*)p.out[blockIdx.y];
  if (!out) return;
  const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
  const int d = p.first + (int)blockIdx.x * 64 + lane;
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
// The launches for `arrays` arrays: one, or, past 2^26 columns, one for each
// 2^26 (a launch holds under 2^32 threads, which are 2^28 - 64 columns here).
template <class T>
void column_sum(ColumnSum c, unsigned arrays, hipStream_t s) {
  constexpr int most = 1 << 26;
  for (c.first = 0; c.first < c.D; c.first += most) {
    const int n = c.D - c.first < most ? c.D - c.first : most;
    column_sum_kernel<T><<<dim3((unsigned)((n + 63) / 64), arrays), dim3(1024), 0, s>>>(c);
  }
}

}  // namespace mi
