// The short convolution along the tokens of each channel, causal, with its gradients and its step for one token.
//
//   pre_t = bias + sum_k w[k] x_{t - W + 1 + k},   y_t = pre_t or silu(pre_t);   x in front of the first token: the state, or 0
//   dpre_t = dy_t (silu'(pre_t)),   dx_t = sum_k w[k] dpre_{t + W - 1 - k} (+ the final state's gradient),   dw[k] = sum_t dpre_t x_{t - W + 1 + k},   dbias = sum_t dpre_t
//
// Memory bounds it: a thread slides over a run of tokens of a few channels, so that a row is read once but for the W - 1 rows on a run's edges, which come out of a
// cache.  Sixteen threads side by side take 128 bytes of a row.
#include "common.h"
#include "launch.h"

#include <algorithm>
#include <type_traits>

namespace vig {
namespace {

constexpr int kConvLanes = 16, kConvRuns = 256 / kConvLanes;  // of a workgroup: threads side by side along a row, runs of tokens

template <int V, typename T> __device__ __forceinline__ void load_vec(float (&x)[V], const T* from) {
  struct alignas(V * sizeof(T)) Whole { T v[V]; };
  const Whole w = *reinterpret_cast<const Whole*>(from);
#pragma unroll
  for (int i = 0; i < V; ++i) x[i] = Elem<T>::load(&w.v[i]);
}
template <int V, typename T> __device__ __forceinline__ void store_vec(T* to, const float (&x)[V]) {
  struct alignas(V * sizeof(T)) Whole { T v[V]; };
  Whole w;
#pragma unroll
  for (int i = 0; i < V; ++i) Elem<T>::store(&w.v[i], x[i]);
  *reinterpret_cast<Whole*>(to) = w;
}

// A thread's place: channels from c on, tokens of the walk from `first` to `end`
template <int V> struct Run {
  int b, c, first, end;
  bool has;
  __device__ __forceinline__ Run(const CausalConv& p) {
    unsigned id = blockIdx.x;
    const int block = (int)(id % (unsigned)p.blocks);
    id /= (unsigned)p.blocks;
    const int runs = (int)(id % (unsigned)p.groups) * kConvRuns + threadIdx.x / kConvLanes;
    b = (int)(id / (unsigned)p.groups);
    c = (block * kConvLanes + threadIdx.x % kConvLanes) * V;
    first = (int)min((long long)runs * p.run, (long long)p.L), end = min(first + p.run, p.L);
    has = c < p.D && first < end;
  }
};

// x of the walk's token t, in front of the first from the state
template <typename T, int V>
__device__ __forceinline__ void load_row(float (&x)[V], const CausalConv& p, int b, int c, int t) {
  const T* from = nullptr;
  if (t >= 0) from = static_cast<const T*>(p.x) + b * p.xb + (p.reverse ? p.L - 1 - t : t) * p.xl + c;
  else if (p.initial) from = static_cast<const T*>(p.initial) + ((long long)b * (p.W - 1) + t + p.W - 1) * p.D + c;
  if (from) {
    load_vec<V>(x, from);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = 0.f;
  }
}
__device__ __forceinline__ long long dense_row(const CausalConv& p, int b, int t) { return ((long long)b * p.L + (p.reverse ? p.L - 1 - t : t)) * p.D; }

template <int V, int W> struct Taps {
  float w[V][W], bias[V];
  __device__ __forceinline__ void load(const CausalConv& p, int c) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
#pragma unroll
      for (int k = 0; k < W; ++k) w[i][k] = p.weight[(long long)(c + i) * W + k];
      bias[i] = p.bias ? p.bias[c + i] : 0.f;
    }
  }
};

template <typename T, int V, int W>
__global__ __launch_bounds__(256) void causal_conv_kernel(CausalConv p) {
  const Run<V> at(p);
  if (!at.has) return;
  Taps<V, W> taps;
  taps.load(p, at.c);
  float rows[W][V];  // the last one is the newest
#pragma unroll
  for (int k = 1; k < W; ++k) load_row<T, V>(rows[k], p, at.b, at.c, at.first - W + k);
  T* const final = static_cast<T*>(p.final);
  const long long held = (long long)at.b * (W - 1);
  if (final && at.first == 0) {  // states of the state, where there are fewer tokens than it has rows
#pragma unroll
    for (int k = 1; k < W; ++k)
      if (k - 1 - p.L >= 0) store_vec<V>(final + (held + k - 1 - p.L) * p.D + at.c, rows[k]);
  }
#pragma unroll 4
  for (int t = at.first; t < at.end; ++t) {
#pragma unroll
    for (int k = 0; k + 1 < W; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) rows[k][i] = rows[k + 1][i];
    load_row<T, V>(rows[W - 1], p, at.b, at.c, t);
    float y[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float s = taps.bias[i];
#pragma unroll
      for (int k = 0; k < W; ++k) s = fmaf(taps.w[i][k], rows[k][i], s);
      y[i] = p.silu ? s * sigmoidf_(s) : s;
    }
    store_vec<V>(static_cast<T*>(p.y) + dense_row(p, at.b, t) + at.c, y);
    if (final && t >= p.L - (W - 1)) store_vec<V>(final + (held + t - (p.L - (W - 1))) * p.D + at.c, rows[W - 1]);
  }
}

// parts: a row of D (W + 1) sums for each group of runs
template <typename T, int V, int W>
__global__ __launch_bounds__(256) void causal_conv_bwd_kernel(CausalConv p) {
  __shared__ float sums[kConvRuns][kConvLanes * V + 1];
  const Run<V> at(p);
  Taps<V, W> taps;
  float dw[V][W], db[V], x[W][V], dpre[W][V];  // the last rows are the newest
#pragma unroll
  for (int i = 0; i < V; ++i) {
    db[i] = 0.f;
#pragma unroll
    for (int k = 0; k < W; ++k) dw[i][k] = 0.f, dpre[k][i] = 0.f;
  }
  if (at.has) {
    taps.load(p, at.c);
#pragma unroll
    for (int k = 1; k < W; ++k) load_row<T, V>(x[k], p, at.b, at.c, at.first - W + k);
    const T* const final = static_cast<const T*>(p.d_final);
    const long long held = (long long)at.b * (W - 1);
    // the gradient of token t is whole once dpre of t + W - 1 is there
    const int stop = at.end + W - 1;
#pragma unroll 2
    for (int t = at.first; t < stop; ++t) {
#pragma unroll
      for (int k = 0; k + 1 < W; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) x[k][i] = x[k + 1][i], dpre[k][i] = dpre[k + 1][i];
      if (t < p.L) {
        load_row<T, V>(x[W - 1], p, at.b, at.c, t);
        load_vec<V>(dpre[W - 1], static_cast<const T*>(p.dy) + dense_row(p, at.b, t) + at.c);
        if (p.silu) {
#pragma unroll
          for (int i = 0; i < V; ++i) {
            float s = taps.bias[i];
#pragma unroll
            for (int k = 0; k < W; ++k) s = fmaf(taps.w[i][k], x[k][i], s);
            const float g = sigmoidf_(s);
            dpre[W - 1][i] *= fmaf(s * g, 1.f - g, g);
          }
        }
        if (t < at.end) {
#pragma unroll
          for (int i = 0; i < V; ++i) {
            db[i] += dpre[W - 1][i];
#pragma unroll
            for (int k = 0; k < W; ++k) dw[i][k] = fmaf(dpre[W - 1][i], x[k][i], dw[i][k]);
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) dpre[W - 1][i] = 0.f;
      }
      const int to = t - (W - 1);  // (dpre[k] is of token to + k)
      if (to >= at.first || at.first == 0) {
        if (to < 0 && !p.d_initial) continue;
        float g[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
          g[i] = 0.f;
#pragma unroll
          for (int k = 0; k < W; ++k) g[i] = fmaf(taps.w[i][W - 1 - k], dpre[k][i], g[i]);
        }
        if (final && to >= p.L - (W - 1)) {
          float f[V];
          load_vec<V>(f, final + (held + to - (p.L - (W - 1))) * p.D + at.c);
#pragma unroll
          for (int i = 0; i < V; ++i) g[i] += f[i];
        }
        if (to >= 0) store_vec<V>(static_cast<T*>(p.dx) + dense_row(p, at.b, to) + at.c, g);
        else store_vec<V>(static_cast<T*>(p.d_initial) + (held + to + W - 1) * p.D + at.c, g);
      }
    }
  }
  if (!p.parts) return;
  // the sums of the workgroup's runs, one number a channel at a time
  const int run = threadIdx.x / kConvLanes, lane = threadIdx.x % kConvLanes;
  const int part = blockIdx.x / p.blocks, c0 = (int)(blockIdx.x % p.blocks) * kConvLanes * V;
#pragma unroll
  for (int k = 0; k <= W; ++k) {
#pragma unroll
    for (int i = 0; i < V; ++i) sums[run][lane * V + i] = k < W ? dw[i][k < W ? k : 0] : db[i];
    __syncthreads();
    for (int e = threadIdx.x; e < kConvLanes * V; e += 256) {
      float s = 0.f;
#pragma unroll
      for (int r = 0; r < kConvRuns; ++r) s += sums[r][e];
      const int c = c0 + e;
      if (c < p.D) p.parts[(long long)part * p.D * (W + 1) + (k < W ? (long long)c * W + k : (long long)p.D * W + c)] = s;
    }
    __syncthreads();
  }
}

template <typename T, int V, int W>
__global__ __launch_bounds__(256) void causal_conv_step_kernel(CausalConv p) {
  const unsigned nv = (unsigned)((p.D + V - 1) / V), id = blockIdx.x * 256u + threadIdx.x;
  const int b = (int)(id / nv), c = (int)(id - b * nv) * V;
  if (b >= p.B) return;
  Taps<V, W> taps;
  taps.load(p, c);
  float rows[W][V], y[V];
  T* const state = static_cast<T*>(p.final) + (long long)b * (W - 1) * p.D + c;
#pragma unroll
  for (int k = 0; k + 1 < W; ++k) load_vec<V>(rows[k], state + (long long)k * p.D);
  load_vec<V>(rows[W - 1], static_cast<const T*>(p.x) + b * p.xb + c);
#pragma unroll
  for (int i = 0; i < V; ++i) {
    float s = taps.bias[i];
#pragma unroll
    for (int k = 0; k < W; ++k) s = fmaf(taps.w[i][k], rows[k][i], s);
    y[i] = p.silu ? s * sigmoidf_(s) : s;
  }
#pragma unroll
  for (int k = 0; k + 1 < W; ++k) store_vec<V>(state + (long long)k * p.D, rows[k + 1]);
  store_vec<V>(static_cast<T*>(p.y) + (long long)b * p.D + c, y);
}

// Channels of a thread: as many as make `bytes`, where every row begins on that boundary; else one.
bool whole(const CausalConv& p, size_t bytes, size_t size) {
  const long long v = (long long)(bytes / size);
  for (const void* t : {p.x, p.initial, (const void*)p.y, (const void*)p.final, p.dy, p.d_final, (const void*)p.dx, (const void*)p.d_initial})
    if (reinterpret_cast<uintptr_t>(t) % bytes) return false;
  return p.D % v == 0 && p.xb % v == 0 && p.xl % v == 0;
}

template <typename F> int by_taps(int W, F f) {
  switch (W) {
    case 2: return f(std::integral_constant<int, 2>{});
    case 3: return f(std::integral_constant<int, 3>{});
    default: return f(std::integral_constant<int, 4>{});
  }
}
// f(type, channels a thread, taps)
template <int BYTES, typename F> int by_case(const CausalConv& p, int io_dtype, F f) {
  return by_taps(p.W, [&](auto w) {
    if (io_dtype == VIG_BF16)
      return whole(p, BYTES, 2) ? f(uint16_t{}, std::integral_constant<int, BYTES / 2>{}, w) : f(uint16_t{}, std::integral_constant<int, 1>{}, w);
    return whole(p, BYTES, 4) ? f(float{}, std::integral_constant<int, BYTES / 4>{}, w) : f(float{}, std::integral_constant<int, 1>{}, w);
  });
}
// Runs of tokens: as long as leaves four workgroups a compute unit, so that few rows on their edges are read twice.
void cut_runs(CausalConv& p, int V, int most) {
  p.blocks = (p.D + kConvLanes * V - 1) / (kConvLanes * V);
  const long long tokens = (long long)p.B * p.blocks * p.L / (kConvRuns * 1024);
  p.run = (int)std::max(4LL, std::min<long long>(most, tokens));
  p.groups = (int)(((p.L + p.run - 1) / p.run + kConvRuns - 1) / kConvRuns);
  p.run = std::max(1, (p.L + p.groups * kConvRuns - 1) / (p.groups * kConvRuns));  // (the runs of a group of alike length)
}
bool conv_fits(const CausalConv& p) { return (long long)p.B * p.groups * p.blocks <= 0xffffff; }  // (below 2^32 threads)
unsigned conv_grid(const CausalConv& p) { return (unsigned)((long long)p.B * p.groups * p.blocks); }
int launched() { return hipGetLastError() == hipSuccess ? 0 : -5; }

}  // namespace

int launch_causal_conv(CausalConv& p, int io_dtype, hipStream_t stream) {
  return by_case<16>(p, io_dtype, [&](auto t, auto v, auto w) {
    cut_runs(p, v, 16);
    if (!conv_fits(p)) return -95;
    hipLaunchKernelGGL((causal_conv_kernel<decltype(t), v, w>), dim3(conv_grid(p)), dim3(256), 0, stream, p);
    return launched();
  });
}

int launch_causal_conv_step(CausalConv& p, int io_dtype, hipStream_t stream) {
  return by_case<16>(p, io_dtype, [&](auto t, auto v, auto w) {
    const long long n = (long long)p.B * ((p.D + v - 1) / v);
    if (n > 0xffffff00LL) return -95;
    hipLaunchKernelGGL((causal_conv_step_kernel<decltype(t), v, w>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, stream, p);
    return launched();
  });
}

// (one channel a thread has the most groups; the room holds for both)
size_t causal_conv_bwd_workspace(int B, int L, int D, int W) {
  CausalConv p{};
  p.B = B, p.L = L, p.D = D, p.W = W;
  size_t most = 0;
  for (int v : {1, 2, 4}) {
    cut_runs(p, v, 64);
    most = std::max(most, sizeof(float) * (size_t)B * p.groups * D * (W + 1));
  }
  return most;
}

int launch_causal_conv_bwd(CausalConv& p, void* workspace, int io_dtype, hipStream_t stream) {
  const int rc = by_case<8>(p, io_dtype, [&](auto t, auto v, auto w) {
    cut_runs(p, v, 64);
    if (!conv_fits(p)) return -95;
    p.parts = p.dparams ? (float*)workspace : nullptr;
    hipLaunchKernelGGL((causal_conv_bwd_kernel<decltype(t), v, w>), dim3(conv_grid(p)), dim3(256), 0, stream, p);
    return launched();
  });
  if (rc || !p.dparams) return rc;
  vig_sum_jobs sums{};
  if (!put_off(sums, p.parts, p.dparams, p.B * p.groups, (long long)p.D * (p.W + 1), false)) return -22;
  return launch_sum_jobs(sums, stream);
}

}  // namespace vig
