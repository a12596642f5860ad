// mi_residual.hpp -- the residual stream between two blocks: the norm after a
// block, its gate and scale, the sum, and the norm before the next block, over
// rows of D values; and the gradients.
//
//   z = x * post_rstd_r * post_weight_d  (post_rstd_r = 1 / sqrt(sum_d x^2 / D + eps)), or x
//   hidden = residual + scale * gate * z
//   y = hidden * rstd_r * weight_d       (rstd_r = 1 / sqrt(sum_d hidden^2 / D + eps))
//
//   u = hidden * rstd, g = dy * weight;  dh = dhidden + rstd * (g - u * sum_d (g * u) / D)
//   dresidual = dh;  dweight_d = sum_r dy * u
//   t = x * post_rstd, or x;  dz = scale * gate * dh * post_weight
//   dx = post_rstd * (dz - t * sum_d (dz * t) / D), or dz
//   c = scale * dh * t:  dgate = post_weight * c and dpost_weight = gate * c, summed over the rows they serve
//
// A gate serves every row, each run of per_gate rows, or one row.  The first
// two need one column sum for both parameters: sums of c over each gate's
// rows, multiplied by post_weight for the gate's gradient and by the gate for
// post_weight's.  A gate of one row stores its gradient as it goes, and the
// column sum is that of gate * c.
//
// y is taken from the sum before hidden is rounded.  Statistics and sums are
// fp32 in an order fixed by the sizes (no atomics); each output is rounded
// once, to nearest even.
//
// One pass over the data, as in mi_norm.hpp: a row's values stay in the
// registers of L lanes between the two row sums and the outputs, blocks walk
// over the rows with the next row's loads in flight, and accesses are 16 bytes
// at any address.  Where a lane's values would pass the row's end it takes
// the row's last ones and leaves those of other lanes out of the sums.
//
// Bound by HBM: 16384 x 8192 bf16 with both norms 207 us (5.2 TB/s; a copy
// reaches 5.0), the gradients of 16384 x 4096 with an fp32 stream 218 us (5.6
// TB/s with the column sums' second launch, 5 us).  A gate for each row: 16384 x
// 8192 bf16 266 us forward (5.0 TB/s) and 364 back (5.9).  Few rows are bound by
// the launches: 8 x 4096 3.9 us of a kernel, 1000 x 1501 fp32 gradients 11.5 +
// 5.4.  Rows past 8192 wait for their own loads (8192 x 16384 bf16 with both
// norms 237 us, 4.5 TB/s), and longer ones, past 8192 in the gradients, are read
// two or three times, from the caches at best: 4096 x 32768 247 us without a
// norm after the block and 350 with, the gradients of 8192 x 16384 655 (2.5 TB/s
// of what has to move), their column sums' kernel among them.
#pragma once
#include "mi_norm.hpp"

namespace mi {

struct RnFwd {
  const void *x, *residual, *weight, *gate, *post_weight;  // weight, gate, post_weight: NULL for 1
  void *y, *hidden;
  float *rstd, *post_rstd;  // NULL: not written
  long long rows, ldx, ldr;
  int D, per_gate;  // per_gate 0: one gate for all rows
  float scale, eps;
  bool params_f32, gate_f32, post;
};

// A mean square whose value, and the squares that make it, are well within
// fp32; otherwise the row is summed again with its values times rms_factor,
// from which rms_rstd takes 1 / sqrt(mean square + eps).
__device__ __forceinline__ bool ms_in_range(float ms, float eps) { return ms < 1e37f && (ms > 1e-30f || eps > 1e-30f); }
__device__ __forceinline__ float rms_factor(float ms) { return ms < 1.0f ? 0x1p64f : 0x1p-64f; }
__device__ __forceinline__ float rms_rstd(float ms, float eps, float k) { return k / __builtin_sqrtf(ms + eps * k * k); }

// The gate of row r: its first value's index.
__device__ __forceinline__ size_t gate_row(long long r, int per_gate, int D) {
  return per_gate ? (size_t)((uint32_t)r / (uint32_t)per_gate) * (size_t)D : 0;
}
__device__ __forceinline__ const void* gate_at(const void* gate, bool f32, size_t elem, size_t at) {
  return (const char*)gate + at * (f32 ? 4 : elem);
}

// GROUPS rows at a time in a block of GROUPS * L threads.  KEEP: the
// parameters and the next row stay in registers (1024 threads leave no room).
template <class T, class R, int E, int L, int GROUPS, bool KEEP>
__global__ __launch_bounds__(L* GROUPS, 4) void residual_norm_kernel(const RnFwd p) {
  constexpr int V = Pack<T>::V, G = E / V, KG = KEEP ? G : 1;
  static_assert(L <= 64 || GROUPS == 1, "rows of several waves have their block to themselves");
  __shared__ float xs[2][L < 64 ? 1 : L / 64][2];
  const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6, in_row = tid % L;
  const float inv_d = 1.0f / (float)p.D;
  RowSplit<V, G, L, false> split;
  split.init(in_row, p.D);
  const auto row_of = [&](long long r) { return r < p.rows ? r : p.rows - 1; };
  const long long step = (long long)gridDim.x * GROUPS;
  long long r = (long long)blockIdx.x * GROUPS + tid / L;
  Pack<T> nx[G];
  Pack<R, V> nr[G];
  const auto fetch = [&](long long at) __attribute__((always_inline)) {
    const T* x = (const T*)p.x + (size_t)at * (size_t)p.ldx;
    const R* res = (const R*)p.residual + (size_t)at * (size_t)p.ldr;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      nx[g] = load_pack(x + split.at[g]);
      nr[g] = load_pack<R, V>(res + split.at[g]);
    }
  };
  float w[KG][V], pw[KG][V], gt[KG][V];
  if constexpr (KEEP) {
    fetch(row_of(r));
    load_params<T>(p.weight, p.params_f32, split.at, 1.0f, w);
    load_params<T>(p.post_weight, p.params_f32, split.at, 1.0f, pw);
#pragma unroll
    for (int g = 0; g < G; ++g) fill(gt[g], 1.0f);
  }
  long long gate_now = -1;
  int turn = 0;
  for (long long first = (long long)blockIdx.x * GROUPS; first < p.rows; first += step, r += step) {
    const long long row = row_of(r);
    if constexpr (!KEEP) fetch(row);
    if constexpr (KEEP) {
      if (p.gate) {
        const size_t at = gate_row(row, p.per_gate, p.D);
        if ((long long)at != gate_now) {
          load_params<T>(gate_at(p.gate, p.gate_f32, sizeof(T), at), p.gate_f32, split.at, 1.0f, gt);
          gate_now = (long long)at;
        }
      }
    }
    float v[G][V], h[G][V];
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        v[g][i] = to_f32(nx[g].v[i]);
        h[g][i] = to_f32(nr[g].v[i]);
      }
    if constexpr (KEEP) fetch(row_of(r + step));
    // 1 / sqrt(mean square + eps) of a row, which adds to `sq` its lane's part.
    const auto rstd_of = [&](float sq, const float(&row_v)[G][V]) __attribute__((always_inline)) {
      float none = 0.0f;
      row_sum2<L>(sq, none, xs, wave, lane, turn);
      if (ms_in_range(sq, p.eps)) return 1.0f / __builtin_sqrtf(sq + p.eps);
      const float k = rms_factor(sq);
      sq = none = 0.0f;
#pragma unroll
      for (int g = 0; g < G; ++g)
#pragma unroll
        for (int i = 0; i < V; ++i) sq += split.mine(g, i, row_v[g][i] * k * (row_v[g][i] * k * inv_d));
      row_sum2<L>(sq, none, xs, wave, lane, turn);
      return rms_rstd(sq, p.eps, k);
    };
    float post_rstd = 1.0f;
    if (p.post) {
      float sq = 0.0f;
#pragma unroll
      for (int g = 0; g < G; ++g)
#pragma unroll
        for (int i = 0; i < V; ++i) sq += split.mine(g, i, v[g][i] * (v[g][i] * inv_d));  // a share of the mean each
      post_rstd = rstd_of(sq, v);
    }
    float sq = 0.0f;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      constexpr int K = KEEP ? 1 : 0;
      if constexpr (!KEEP) {
        // (Read again for each row, not once and then spilled.)
        const void *weight = p.post_weight, *gate = p.gate;
        asm volatile("" : "+s"(weight), "+s"(gate));
        const int at[1] = {split.at[g]};
        load_params<T>(weight, p.params_f32, at, 1.0f, pw);
        load_params<T>(gate ? gate_at(gate, p.gate_f32, sizeof(T), gate_row(row, p.per_gate, p.D)) : nullptr, p.gate_f32,
                       at, 1.0f, gt);
      }
#pragma unroll
      for (int i = 0; i < V; ++i) {
        h[g][i] += v[g][i] * post_rstd * pw[K * g][i] * (gt[K * g][i] * p.scale);
        sq += split.mine(g, i, h[g][i] * (h[g][i] * inv_d));
      }
    }
    const float rstd = rstd_of(sq, h);
    T* y = (T*)p.y + (size_t)row * (size_t)p.D;
    R* hidden = (R*)p.hidden + (size_t)row * (size_t)p.D;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      constexpr int K = KEEP ? 1 : 0;
      if constexpr (!KEEP) {
        const void* weight = p.weight;
        asm volatile("" : "+s"(weight));
        const int at[1] = {split.at[g]};
        load_params<T>(weight, p.params_f32, at, 1.0f, w);
      }
      float o[V];
#pragma unroll
      for (int i = 0; i < V; ++i) o[i] = h[g][i] * rstd * w[K * g][i];
      store_pack<R>(hidden + split.at[g], h[g]);
      store_pack<T>(y + split.at[g], o);
    }
    if (in_row == 0 && r < p.rows) {
      if (p.rstd) p.rstd[r] = rstd;
      if (p.post_rstd) p.post_rstd[r] = post_rstd;
    }
  }
}

// Rows longer than registers hold (W = 16 bytes of T), or shorter than 16
// bytes (W = 1): a block of B threads per row reads it two or three times.
template <class T, class R, int B, int W>
__global__ __launch_bounds__(B) void residual_norm_long_kernel(const RnFwd p) {
  __shared__ float xs[2][B / 64][2];
  const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const float inv_d = 1.0f / (float)p.D;
  int turn = 0;
  for (long long r = blockIdx.x; r < p.rows; r += gridDim.x) {
    const T* x = (const T*)p.x + (size_t)r * (size_t)p.ldx;
    const R* res = (const R*)p.residual + (size_t)r * (size_t)p.ldr;
    const void* gate =
        p.gate ? gate_at(p.gate, p.gate_f32, sizeof(T), gate_row(r, p.per_gate, p.D)) : nullptr;
    // sum(k): the mean of the squares of k times the row's values.
    const auto rstd_of = [&](auto&& sum) __attribute__((always_inline)) {
      const float ms = sum(1.0f);
      if (ms_in_range(ms, p.eps)) return 1.0f / __builtin_sqrtf(ms + p.eps);
      const float k = rms_factor(ms);
      return rms_rstd(sum(k), p.eps, k);
    };
    float post_rstd = 1.0f;
    if (p.post) {
      post_rstd = rstd_of([&](float k) {
        float sq = 0.0f, none = 0.0f;
        each_pack<B, W>(tid, p.D, [&](int at, int own) __attribute__((always_inline)) {
          const Pack<T, W> v = load_pack<T, W>(x + at);
#pragma unroll
          for (int i = 0; i < W; ++i) {
            const float f = to_f32(v.v[i]) * k;
            sq += i >= own ? f * (f * inv_d) : 0.0f;
          }
        });
        row_sum2<B>(sq, none, xs, wave, lane, turn);
        return sq;
      });
    }
    const auto hidden_of = [&](int at, float (&h)[W]) __attribute__((always_inline)) {
      const Pack<T, W> v = load_pack<T, W>(x + at);
      const Pack<R, W> s = load_pack<R, W>(res + at);
      float pw[1][W], gt[1][W];
      const int where[1] = {at};
      load_params<T>(p.post_weight, p.params_f32, where, 1.0f, pw);
      load_params<T>(gate, p.gate_f32, where, 1.0f, gt);
#pragma unroll
      for (int i = 0; i < W; ++i) h[i] = to_f32(s.v[i]) + to_f32(v.v[i]) * post_rstd * pw[0][i] * (gt[0][i] * p.scale);
    };
    const float rstd = rstd_of([&](float k) {
      float sq = 0.0f, none = 0.0f;
      each_pack<B, W>(tid, p.D, [&](int at, int own) __attribute__((always_inline)) {
        float h[W];
        hidden_of(at, h);
#pragma unroll
        for (int i = 0; i < W; ++i) sq += i >= own ? h[i] * k * (h[i] * k * inv_d) : 0.0f;
      });
      row_sum2<B>(sq, none, xs, wave, lane, turn);
      return sq;
    });
    each_pack<B, W>(tid, p.D, [&](int at, int) __attribute__((always_inline)) {
      float h[W], w[1][W], o[W];
      hidden_of(at, h);
      const int where[1] = {at};
      load_params<T>(p.weight, p.params_f32, where, 1.0f, w);
#pragma unroll
      for (int i = 0; i < W; ++i) o[i] = h[i] * rstd * w[0][i];
      store_pack<R>((R*)p.hidden + (size_t)r * (size_t)p.D + at, h);
      store_pack<T>((T*)p.y + (size_t)r * (size_t)p.D + at, o);
    });
    if (tid == 0) {
      if (p.rstd) p.rstd[r] = rstd;
      if (p.post_rstd) p.post_rstd[r] = post_rstd;
    }
  }
}

struct RnBwd {
  const void *dy, *dhidden, *x, *hidden, *weight, *gate, *post_weight;  // dhidden: NULL for 0; x: NULL where nothing needs it
  const float *rstd, *post_rstd;  // post_rstd: NULL without a norm after the block
  void *dx, *dresidual, *dgate;   // dx: NULL: not wanted; dgate: of a gate of one row each (else, or not wanted: NULL)
  float *part_w, *part_c;         // [blocks][D] partial column sums; NULL: not wanted
  float* row_dot;                 // [rows] sum_d (g * u) / D, written and read by the kernels of long rows
  long long rows, lddy, lddh, ldx, ldh;
  int D, per_gate;                // per_gate 0: one gate for all rows
  int runs, per_run;              // the rows in runs of per_run, gridDim.x / runs blocks to each
  float scale;
  bool params_f32, gate_f32;
  bool own_gates;                 // a gate of one row each: part_c's sums are those of gate * c, wanted dgate or not
};

// GROUPS rows at a time in a block of GROUPS * L threads, which stays within
// one run of rows.  AHEAD: the next row's loads in flight.
template <class T, class R, int E, int L, int GROUPS, bool AHEAD>
__global__ __launch_bounds__(L* GROUPS) void residual_norm_bwd_kernel(const RnBwd p) {
  constexpr int V = Pack<T>::V, G = E / V, WPR = L < 64 ? 1 : L / 64;
  __shared__ float xs[GROUPS][2][WPR][2];
  __shared__ float cols[GROUPS > 1 ? GROUPS : 1][GROUPS > 1 ? L * V : 1];
  const int tid = (int)threadIdx.x, lane = tid & 63;
  const int in_row = tid % L, group = tid / L, wave = in_row >> 6;
  const float inv_d = 1.0f / (float)p.D;
  RowSplit<V, G, L, false> split;
  split.init(in_row, p.D);
  const int blocks = (int)gridDim.x / p.runs, run = (int)blockIdx.x / blocks, block = (int)blockIdx.x - run * blocks;
  const long long begin = (long long)run * p.per_run;
  const long long end = begin + p.per_run < p.rows ? begin + p.per_run : p.rows;
  const auto row_of = [&](long long r) { return r < end ? r : end - 1; };
  const long long step = (long long)blocks * GROUPS;
  long long r = begin + (long long)block * GROUPS + group;
  Pack<T> ny[G], nx[G];
  Pack<R, V> nd[G], nh[G];
  float nrstd, npost = 1.0f;
  // (What is not there is read as rows that are, x as dy and dhidden as hidden, and left out.)
  const T* xp = p.x ? (const T*)p.x : (const T*)p.dy;
  const size_t ldx = p.x ? (size_t)p.ldx : (size_t)p.lddy;
  const R* dhp = p.dhidden ? (const R*)p.dhidden : (const R*)p.hidden;
  const size_t lddh = p.dhidden ? (size_t)p.lddh : (size_t)p.ldh;
  const float has_dh = p.dhidden ? 1.0f : 0.0f;
  const float* post = p.post_rstd ? p.post_rstd : p.rstd;
  const auto fetch = [&](long long at) __attribute__((always_inline)) {
    const T *dy = (const T*)p.dy + (size_t)at * (size_t)p.lddy, *x = xp + (size_t)at * ldx;
    const R *h = (const R*)p.hidden + (size_t)at * (size_t)p.ldh, *dh = dhp + (size_t)at * lddh;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      ny[g] = load_pack(dy + split.at[g]);
      nh[g] = load_pack<R, V>(h + split.at[g]);
      nd[g] = load_pack<R, V>(dh + split.at[g]);
      nx[g] = load_pack(x + split.at[g]);
    }
    nrstd = p.rstd[at];
    npost = post[at];
  };
  float w[G][V], pw[G][V], gt[G][V], dw[G][V], c[G][V];
  if constexpr (AHEAD) fetch(row_of(r));
  load_params<T>(p.weight, p.params_f32, split.at, 1.0f, w);
  load_params<T>(p.post_weight, p.params_f32, split.at, 1.0f, pw);
#pragma unroll
  for (int g = 0; g < G; ++g) {
    fill(gt[g], 1.0f);
    fill(dw[g], 0.0f);
    fill(c[g], 0.0f);
  }
  long long gate_now = -1;
  int turn = 0;
  for (long long first = begin + (long long)block * GROUPS; first < end; first += step, r += step) {
    const long long row = row_of(r);
    if constexpr (!AHEAD) fetch(row);
    if (p.gate) {
      const size_t at = gate_row(row, p.per_gate, p.D);
      if ((long long)at != gate_now) {
        load_params<T>(gate_at(p.gate, p.gate_f32, sizeof(T), at), p.gate_f32, split.at, 1.0f, gt);
        gate_now = (long long)at;
      }
    }
    Pack<T> yv[G], xv[G];
    Pack<R, V> dv[G], hv[G];
#pragma unroll
    for (int g = 0; g < G; ++g) {
      yv[g] = ny[g];
      xv[g] = nx[g];
      dv[g] = nd[g];
      hv[g] = nh[g];
    }
    const float rstd = nrstd, post_rstd = p.post_rstd ? npost : 1.0f;
    if constexpr (AHEAD) fetch(row_of(r + step));
    const bool live = r < end;
    float dot = 0.0f, none = 0.0f;
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float dy = to_f32(yv[g].v[i]), u = to_f32(hv[g].v[i]) * rstd;
        dw[g][i] += live ? dy * u : 0.0f;
        dot += split.mine(g, i, dy * w[g][i] * (u * inv_d));
      }
    row_sum2<L>(dot, none, xs[group], wave, lane, turn);
    float dh[G][V], sum = 0.0f;
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float u = to_f32(hv[g].v[i]) * rstd;
        const float d = to_f32(dv[g].v[i]);
        dh[g][i] = (has_dh != 0.0f ? d : 0.0f) + rstd * (to_f32(yv[g].v[i]) * w[g][i] - u * dot);
      }
    R* dres = (R*)p.dresidual + (size_t)row * (size_t)p.D;
#pragma unroll
    for (int g = 0; g < G; ++g) store_pack<R>(dres + split.at[g], dh[g]);
    if (!p.x) {
      // No gate and no norm after the block: dx = scale * dh.
      if (p.dx) {
        T* dx = (T*)p.dx + (size_t)row * (size_t)p.D;
#pragma unroll
        for (int g = 0; g < G; ++g) {
          float o[V];
#pragma unroll
          for (int i = 0; i < V; ++i) o[i] = p.scale * dh[g][i];
          store_pack<T>(dx + split.at[g], o);
        }
      }
      continue;
    }
#pragma unroll
    for (int g = 0; g < G; ++g) {
      float each[V];
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float t = to_f32(xv[g].v[i]) * post_rstd, s = p.scale * dh[g][i];
        const float one = s * t;
        c[g][i] += live ? (p.own_gates ? one * gt[g][i] : one) : 0.0f;
        each[i] = one * pw[g][i];
        dh[g][i] = s * gt[g][i] * pw[g][i];  // dz from here on
        sum += split.mine(g, i, dh[g][i] * (t * inv_d));
      }
      if (p.dgate) {
        if (p.gate_f32) store_pack<float>((float*)p.dgate + (size_t)row * (size_t)p.D + split.at[g], each);
        else store_pack<T>((T*)p.dgate + (size_t)row * (size_t)p.D + split.at[g], each);
      }
    }
    if (!p.dx) continue;
    if (p.post_rstd) {
      none = 0.0f;
      row_sum2<L>(sum, none, xs[group], wave, lane, turn);
    } else {
      sum = 0.0f;
    }
    T* dx = (T*)p.dx + (size_t)row * (size_t)p.D;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      float o[V];
#pragma unroll
      for (int i = 0; i < V; ++i) o[i] = post_rstd * (dh[g][i] - to_f32(xv[g].v[i]) * post_rstd * sum);
      store_pack<T>(dx + split.at[g], o);
    }
  }
  float* part[2] = {p.part_w, p.part_c};
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    if (!part[k]) continue;
    float* to = part[k] + (size_t)blockIdx.x * (size_t)p.D;
    if constexpr (GROUPS == 1) {
#pragma unroll
      for (int g = 0; g < G; ++g) store_pack<float>(to + split.at[g], k ? c[g] : dw[g]);
    } else {
      // The groups' sums in their order, one pack of columns at a time.
#pragma unroll
      for (int g = 0; g < G; ++g) {
        if (g * L * V >= p.D) break;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < V; ++i) cols[group][in_row * V + i] = k ? c[g][i] : dw[g][i];
        __syncthreads();
        for (int e = tid; e < L * V; e += L * GROUPS) {
          const int d = g * L * V + e / V * V, at = d + V <= p.D ? d : p.D - V;
          float s = cols[0][e];
#pragma unroll
          for (int q = 1; q < GROUPS; ++q) s += cols[q][e];
          to[at + e % V] = s;
        }
      }
    }
  }
}

// Rows longer than registers hold, or shorter than 16 bytes: dresidual, dx
// and a gate of one row's gradient by a block of B threads per row (two or
// three reads of it), the column sums by residual_columns_kernel.
template <class T, class R, int B, int W>
__global__ __launch_bounds__(B) void residual_norm_bwd_long_kernel(const RnBwd p) {
  __shared__ float xs[2][B / 64][2];
  const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const float inv_d = 1.0f / (float)p.D;
  int turn = 0;
  for (long long r = blockIdx.x; r < p.rows; r += gridDim.x) {
    const T* dy = (const T*)p.dy + (size_t)r * (size_t)p.lddy;
    const R* h = (const R*)p.hidden + (size_t)r * (size_t)p.ldh;
    const float rstd = p.rstd[r], post_rstd = p.post_rstd ? p.post_rstd[r] : 1.0f;
    const void* gate =
        p.gate ? gate_at(p.gate, p.gate_f32, sizeof(T), gate_row(r, p.per_gate, p.D)) : nullptr;
    float dot = 0.0f, none = 0.0f;
    each_pack<B, W>(tid, p.D, [&](int at, int own) __attribute__((always_inline)) {
      const Pack<T, W> d = load_pack<T, W>(dy + at);
      const Pack<R, W> v = load_pack<R, W>(h + at);
      float w[1][W];
      const int where[1] = {at};
      load_params<T>(p.weight, p.params_f32, where, 1.0f, w);
#pragma unroll
      for (int i = 0; i < W; ++i) dot += i >= own ? to_f32(d.v[i]) * w[0][i] * (to_f32(v.v[i]) * rstd * inv_d) : 0.0f;
    });
    row_sum2<B>(dot, none, xs, wave, lane, turn);
    if (tid == 0 && p.row_dot) p.row_dot[r] = dot;
    // f(at, own, dh) for each of a thread's packs.
    const auto each = [&](auto&& f) __attribute__((always_inline)) {
      each_pack<B, W>(tid, p.D, [&](int at, int own) __attribute__((always_inline)) {
        const Pack<T, W> d = load_pack<T, W>(dy + at);
        const Pack<R, W> v = load_pack<R, W>(h + at);
        float w[1][W], dh[W];
        const int where[1] = {at};
        load_params<T>(p.weight, p.params_f32, where, 1.0f, w);
#pragma unroll
        for (int i = 0; i < W; ++i) dh[i] = rstd * (to_f32(d.v[i]) * w[0][i] - to_f32(v.v[i]) * rstd * dot);
        if (p.dhidden) {
          const Pack<R, W> e = load_pack<R, W>((const R*)p.dhidden + (size_t)r * (size_t)p.lddh + at);
#pragma unroll
          for (int i = 0; i < W; ++i) dh[i] += to_f32(e.v[i]);
        }
        f(at, own, dh);
      });
    };
    const auto turned = [&](int at, float (&t)[W]) __attribute__((always_inline)) {
      const Pack<T, W> v = load_pack<T, W>((const T*)p.x + (size_t)r * (size_t)p.ldx + at);
#pragma unroll
      for (int i = 0; i < W; ++i) t[i] = to_f32(v.v[i]) * post_rstd;
    };
    const auto dz_of = [&](int at, float (&dh)[W]) __attribute__((always_inline)) {
      float gt[1][W], pw[1][W];
      const int where[1] = {at};
      load_params<T>(gate, p.gate_f32, where, 1.0f, gt);
      load_params<T>(p.post_weight, p.params_f32, where, 1.0f, pw);
#pragma unroll
      for (int i = 0; i < W; ++i) dh[i] = p.scale * dh[i] * gt[0][i] * pw[0][i];
    };
    float sum = 0.0f;
    each([&](int at, int own, float(&dh)[W]) __attribute__((always_inline)) {
      store_pack<R>((R*)p.dresidual + (size_t)r * (size_t)p.D + at, dh);
      if (!p.post_rstd && !p.dgate) return;
      float t[W];
      turned(at, t);
      if (p.dgate) {
        float one[W], pw[1][W];
        const int where[1] = {at};
        load_params<T>(p.post_weight, p.params_f32, where, 1.0f, pw);
#pragma unroll
        for (int i = 0; i < W; ++i) one[i] = p.scale * dh[i] * t[i] * pw[0][i];
        if (p.gate_f32) store_pack<float>((float*)p.dgate + (size_t)r * (size_t)p.D + at, one);
        else store_pack<T>((T*)p.dgate + (size_t)r * (size_t)p.D + at, one);
      }
      if (!p.post_rstd) return;
      dz_of(at, dh);
#pragma unroll
      for (int i = 0; i < W; ++i) sum += i >= own ? dh[i] * (t[i] * inv_d) : 0.0f;
    });
    if (!p.dx) continue;
    if (p.post_rstd) {
      none = 0.0f;
      row_sum2<B>(sum, none, xs, wave, lane, turn);
    }
    each([&](int at, int, float(&dh)[W]) __attribute__((always_inline)) {
      dz_of(at, dh);
      if (p.post_rstd) {
        float t[W];
        turned(at, t);
#pragma unroll
        for (int i = 0; i < W; ++i) dh[i] = post_rstd * (dh[i] - t[i] * sum);
      }
      store_pack<T>((T*)p.dx + (size_t)r * (size_t)p.D + at, dh);
    });
  }
}

// Column sums of the chunks of the rows' runs, `chunks` of them over all:
// blockIdx.x takes 256 packs of columns, blockIdx.y (and those gridDim.y
// further on) a chunk, every so many-th row of its run.
template <class T, class R, int W>
__global__ __launch_bounds__(256) void residual_columns_kernel(const RnBwd p, int chunks) {
  const int d = ((int)blockIdx.x * 256 + (int)threadIdx.x) * W;
  if (d >= p.D) return;
  const int at = d + W <= p.D ? d : p.D - W;
  const int each = chunks / p.runs;
  float w[1][W], dw[W], c[W];
  const int where[1] = {at};
  load_params<T>(p.weight, p.params_f32, where, 1.0f, w);
  for (int chunk = (int)blockIdx.y; chunk < chunks; chunk += (int)gridDim.y) {
    const int run = chunk / each;
    const long long begin = (long long)run * p.per_run;
    const long long end = begin + p.per_run < p.rows ? begin + p.per_run : p.rows;
    fill(dw, 0.0f);
    fill(c, 0.0f);
    for (long long r = begin + (chunk - run * each); r < end; r += each) {
      const Pack<T, W> y = load_pack<T, W>((const T*)p.dy + (size_t)r * (size_t)p.lddy + at);
      const Pack<R, W> h = load_pack<R, W>((const R*)p.hidden + (size_t)r * (size_t)p.ldh + at);
      const float rstd = p.rstd[r];
  #pragma unroll
      for (int i = 0; i < W; ++i) dw[i] += to_f32(y.v[i]) * (to_f32(h.v[i]) * rstd);
      if (!p.part_c) continue;
      const float dot = p.row_dot[r], post_rstd = p.post_rstd ? p.post_rstd[r] : 1.0f;
      const Pack<T, W> x = load_pack<T, W>((const T*)p.x + (size_t)r * (size_t)p.ldx + at);
      float dh[W], gt[1][W];
  #pragma unroll
      for (int i = 0; i < W; ++i) dh[i] = rstd * (to_f32(y.v[i]) * w[0][i] - to_f32(h.v[i]) * rstd * dot);
      if (p.dhidden) {
        const Pack<R, W> e = load_pack<R, W>((const R*)p.dhidden + (size_t)r * (size_t)p.lddh + at);
  #pragma unroll
        for (int i = 0; i < W; ++i) dh[i] += to_f32(e.v[i]);
      }
      load_params<T>(p.own_gates ? gate_at(p.gate, p.gate_f32, sizeof(T), gate_row(r, p.per_gate, p.D)) : nullptr,
                     p.gate_f32, where, 1.0f, gt);
  #pragma unroll
      for (int i = 0; i < W; ++i) c[i] += p.scale * dh[i] * (to_f32(x.v[i]) * post_rstd) * gt[0][i];
    }
    if (p.part_w) store_pack<float>(p.part_w + (size_t)chunk * (size_t)p.D + at, dw);
    if (p.part_c) store_pack<float>(p.part_c + (size_t)chunk * (size_t)p.D + at, c);
  }
}

// The parameters' gradients from the partial sums, 64 columns a block, its 16
// waves taking turns over the parts and their sums added in wave order:
// role 0 (blockIdx.y, and those gridDim.y further on): dweight; 1:
// dpost_weight, each part times its run's gate; 2 + k: the k-th gate's, its
// run's parts times post_weight.
struct RnColumns {
  const float *part_w, *part_c;
  const void *gate, *post_weight;
  void *dweight, *dpost, *dgate;  // NULL: not wanted
  int parts, runs, D, first;      // parts: of all runs together
  bool params_f32, gate_f32;
  bool weigh, gate_rows;  // dpost's parts are not yet multiplied by the gate; which has a row for each run
};
template <class T>
__device__ __forceinline__ void put_param(void* out, bool f32, size_t at, float v) {
  if (f32) ((float*)out)[at] = v;
  else ((T*)out)[at] = from_f32<T>(v);
}
template <class T>
__device__ __forceinline__ float get_param(const void* p, bool f32, size_t at) {
  return f32 ? ((const float*)p)[at] : to_f32(((const T*)p)[at]);
}
template <class T>
__global__ __launch_bounds__(1024) void residual_parameters_kernel(const RnColumns p) {
  __shared__ float xs[16][64];
  const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
  const int d = p.first + (int)blockIdx.x * 64 + lane;
  const int each = p.parts / p.runs, roles = 2 + (p.dgate ? p.runs : 0);
  for (int role = (int)blockIdx.y; role < roles; role += (int)gridDim.y) {
    const int kind = role < 2 ? role : 2, run = role - 2;
    void* out = kind == 0 ? p.dweight : kind == 1 ? p.dpost : p.dgate;
    if (!out) continue;
    const int n = kind == 2 ? each : p.parts;
    const float* part = (kind == 0 ? p.part_w : p.part_c) + (kind == 2 ? (size_t)run * (size_t)each * (size_t)p.D : 0);
    const bool weigh = kind == 1 && p.weigh && p.gate;
    float s = 0.0f;
    if (d < p.D) {
      constexpr int U = 8;
      for (int i0 = wave; i0 < n; i0 += 16 * U) {
        float v[U], f[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int i = i0 + 16 * u;
          v[u] = i < n ? part[(size_t)i * (size_t)p.D + d] : 0.0f;
          f[u] = weigh && i < n ? get_param<T>(p.gate, p.gate_f32, p.gate_rows ? (size_t)(i / each) * (size_t)p.D + d : d)
                                : 1.0f;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) s += v[u] * f[u];
      }
    }
    __syncthreads();  // the sums of the role before are read
    xs[wave][lane] = s;
    __syncthreads();
    if (wave == 0 && d < p.D) {
#pragma unroll
      for (int w = 1; w < 16; ++w) s += xs[w][lane];
      if (kind == 2) {
        if (p.post_weight) s *= get_param<T>(p.post_weight, p.params_f32, d);
        put_param<T>(out, p.gate_f32, (size_t)run * (size_t)p.D + d, s);
      } else {
        put_param<T>(out, p.params_f32, d, s);
      }
    }
  }
}

}  // namespace mi
