// The short convolution along the tokens of each channel, causal, with its gradients and its step for one token.
//
//   pre_t = bias + sum_k w[k] x_{t - W + 1 + k},   y_t = pre_t or silu(pre_t);   x in front of the first token: the state, or 0
//   dpre_t = dy_t (silu'(pre_t)),   dx_t = sum_k w[k] dpre_{t + W - 1 - k} (+ the final state's gradient),   dw[k] = sum_t dpre_t x_{t - W + 1 + k},   dbias = sum_t dpre_t
//
// Memory bounds it: a thread slides over a run of tokens of a few channels, so that a row is read once but for the W - 1 rows on a run's edges, which come out of a
// cache.  Sixteen threads side by side take 256 bytes of a row (128 in the backward, which has twice the registers to hold).
//
// Measured, bf16, 4 taps, silu: 65536 x 1024 53 us, 5.1 TB/s (a large copy: 5.4); 128 x 196 x 768 forward 19, backward 33 (116 MB, part of it in the 256 MB cache; 35 operations an
// element beside it), sums of the weights' gradient 4.
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

typedef __amdgpu_buffer_rsrc_t rsrc_t;
constexpr unsigned kNowhere = 0x80000000u;  // byte offset behind every descriptor here

// V channels of a row as stored
template <typename T, int V> struct Piece {
  static constexpr int kBytes = V * sizeof(T);
  u32x4_t v;
  __device__ __forceinline__ void load(rsrc_t r, unsigned off) {
    if constexpr (kBytes == 16) v = __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0);
    else if constexpr (kBytes == 8) { const u32x2_t w = __builtin_amdgcn_raw_buffer_load_b64(r, off, 0, 0); v[0] = w[0], v[1] = w[1]; }
    else if constexpr (kBytes == 4) v[0] = __builtin_amdgcn_raw_buffer_load_b32(r, off, 0, 0);
    else v[0] = __builtin_amdgcn_raw_buffer_load_b16(r, off, 0, 0);
  }
  __device__ __forceinline__ void get(float (&x)[V]) const {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if constexpr (sizeof(T) == 4) x[i] = __uint_as_float(v[i]);
      else x[i] = i & 1 ? bf16hi_to_f32(v[i / 2]) : bf16lo_to_f32(v[i / 2]);
    }
  }
  __device__ __forceinline__ void set(const float (&x)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if constexpr (sizeof(T) == 4) v[i] = __float_as_uint(x[i]);
      else if constexpr (V == 1) v[0] = f32_to_bf16(x[0]);
      else if (i & 1) v[i / 2] = pack_bf16x2(x[i - 1], x[i]);
    }
  }
  __device__ __forceinline__ void store(rsrc_t r, unsigned off) const {
    if constexpr (kBytes == 16) __builtin_amdgcn_raw_buffer_store_b128(v, r, off, 0, 0);
    else if constexpr (kBytes == 8) __builtin_amdgcn_raw_buffer_store_b64(u32x2_t{v[0], v[1]}, r, off, 0, 0);
    else if constexpr (kBytes == 4) __builtin_amdgcn_raw_buffer_store_b32(v[0], r, off, 0, 0);
    else __builtin_amdgcn_raw_buffer_store_b16((uint16_t)v[0], r, off, 0, 0);
  }
};

// A thread's place: channels from c on, tokens of the walk from `first` to `end`; and the tokens that its workgroup reads, from `low` to `high`
template <int V> struct Run {
  int b, c, first, end, low, high;
  bool has;
  __device__ __forceinline__ Run(const CausalConv& p) {
    unsigned id = blockIdx.x;
    const int block = (int)(id % (unsigned)p.blocks);
    id /= (unsigned)p.blocks;
    const long long group = (long long)(id % (unsigned)p.groups) * kConvRuns * p.run;
    b = (int)(id / (unsigned)p.groups);
    c = (block * kConvLanes + threadIdx.x % kConvLanes) * V;
    first = (int)min(group + threadIdx.x / kConvLanes * p.run, (long long)p.L), end = min(first + p.run, p.L);
    low = (int)max(group - (p.W - 1), 0LL), high = (int)min(group + kConvRuns * p.run + p.W - 1, (long long)p.L);
    has = c < p.D && first < end;
  }
};
// The workgroup's rows of a tensor: the descriptor begins at the lowest in memory and ends behind the highest, so that rows in front of the first token and behind the last
// read as zeros and are not stored
template <typename T> struct RowsOf {
  rsrc_t r;
  unsigned pitch, offset;  // offset: of token 0 of the walk, for this thread
  bool reverse;
  template <int V> __device__ __forceinline__ RowsOf(const CausalConv& p, const Run<V>& at, const void* base, long long sb, long long sl) {
    reverse = p.reverse != 0;
    const long long lowest = p.reverse ? (long long)p.L - at.high : at.low;
    r = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(static_cast<const T*>(base)) + at.b * sb + lowest * sl, 0, (int)((at.high - at.low) * (unsigned)(sl * sizeof(T))), 0x00020000);
    pitch = (unsigned)sl * sizeof(T);
    offset = at.has ? at.c * (unsigned)sizeof(T) : kNowhere;
    low = at.low, high = at.high;
  }
  int low, high;
  // (rows that are not there wrap round to offsets behind the descriptor)
  __device__ __forceinline__ unsigned of(int t) const { return offset + (unsigned)(reverse ? high - 1 - t : t - low) * pitch; }
};

// Weights of V channels: in pieces of 16 bytes where they begin on one
template <int N> __device__ __forceinline__ void load_floats(float (&x)[N], const float* from) {
  if (N % 4 == 0 && reinterpret_cast<uintptr_t>(from) % 16 == 0) {
#pragma unroll
    for (int i = 0; i + 3 < N; i += 4) {
      const f32x4_t v = *reinterpret_cast<const f32x4_t*>(from + i);
      x[i] = v[0], x[i + 1] = v[1], x[i + 2] = v[2], x[i + 3] = v[3];
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = from[i];
  }
}
template <int V, int W> struct Taps {
  float w[V * W], bias[V];
  __device__ __forceinline__ void load(const CausalConv& p, int c) {
    load_floats(w, p.weight + (long long)c * W);
    if (p.bias) {
      load_floats(bias, p.bias + c);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) bias[i] = 0.f;
    }
  }
};
// the state's row of token t < 0, or zeros
template <typename T, int V>
__device__ __forceinline__ void state_row(float (&x)[V], const CausalConv& p, int b, int c, int t) {
  if (p.initial) {
    load_vec<V>(x, static_cast<const T*>(p.initial) + ((long long)b * (p.W - 1) + t + p.W - 1) * p.D + c);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = 0.f;
  }
}

// Tokens whose rows are on their way together: the next ones' while a thread works on these.  us, 65536 x 1024 forward / 128 x 196 x 768 backward: two 53 / 34, four 55 / 34, eight 59 / 42 (170
// registers, two waves a SIMD).
constexpr int kConvTokens = 2;

template <typename T, int V, int W>
__global__ __launch_bounds__(256) void causal_conv_kernel(CausalConv p) {
  const Run<V> at(p);
  const RowsOf<T> in(p, at, p.x, p.xb, p.xl), out(p, at, p.y, (long long)p.L * p.D, p.D);
  Piece<T, V> raw[2][kConvTokens];
  auto load = [&](Piece<T, V> (&to)[kConvTokens], int t) {
#pragma unroll
    for (int k = 0; k < kConvTokens; ++k) to[k].load(in.r, in.of(t + k));
  };
  Piece<T, V> edge[W - 1];
#pragma unroll
  for (int k = 0; k + 1 < W; ++k) edge[k].load(in.r, in.of(at.first - (W - 1) + k));
  load(raw[0], at.first);
  if (!at.has) return;
  Taps<V, W> taps;
  taps.load(p, at.c);
  float rows[W][V];  // the last one is the newest
#pragma unroll
  for (int k = 0; k + 1 < W; ++k) {
    if (at.first - (W - 1) + k < 0) state_row<T, V>(rows[k + 1], p, at.b, at.c, at.first - (W - 1) + k);
    else edge[k].get(rows[k + 1]);
  }
  auto work = [&](const Piece<T, V> (&from)[kConvTokens], int t) {
#pragma unroll
    for (int k = 0; k < kConvTokens; ++k) {
#pragma unroll
      for (int j = 0; j + 1 < W; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i) rows[j][i] = rows[j + 1][i];
      from[k].get(rows[W - 1]);
      float y[V];
#pragma unroll
      for (int i = 0; i < V; ++i) {
        float s = taps.bias[i];
#pragma unroll
        for (int j = 0; j < W; ++j) s = fmaf(taps.w[i * W + j], rows[j][i], s);
        y[i] = p.silu ? s * sigmoidf_(s) : s;
      }
      Piece<T, V> o;
      o.set(y);
      o.store(out.r, t + k < at.end ? out.of(t + k) : kNowhere);
    }
  };
  for (int t = at.first; t < at.end; t += 2 * kConvTokens) {
    load(raw[1], t + kConvTokens);
    work(raw[0], t);
    if (t + kConvTokens >= at.end) break;
    load(raw[0], t + 2 * kConvTokens);
    work(raw[1], t + kConvTokens);
  }
  if (!p.final || at.end != p.L) return;
  // the last rows, those of the state among them where there are few tokens
#pragma unroll
  for (int k = 0; k + 1 < W; ++k) {
    const int t = p.L - (W - 1) + k;
    float x[V];
    if (t < 0) {
      state_row<T, V>(x, p, at.b, at.c, t);
    } else {
      Piece<T, V> last;
      last.load(in.r, in.of(t));
      last.get(x);
    }
    store_vec<V>(static_cast<T*>(p.final) + ((long long)at.b * (W - 1) + k) * p.D + at.c, x);
  }
}

// parts: a row of D (W + 1) sums for each group of runs
template <typename T, int V, int W>
__global__ __launch_bounds__(256) void causal_conv_bwd_kernel(CausalConv p) {
  __shared__ float sums[kConvRuns][kConvLanes * V + 1];
  const Run<V> at(p);
  const RowsOf<T> in(p, at, p.x, p.xb, p.xl), grad(p, at, p.dy, (long long)p.L * p.D, p.D), out(p, at, p.dx, (long long)p.L * p.D, p.D);
  float dw[V][W], db[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    db[i] = 0.f;
#pragma unroll
    for (int k = 0; k < W; ++k) dw[i][k] = 0.f;
  }
  Piece<T, V> raw_x[kConvTokens], raw_dy[kConvTokens], edge[W - 1];
  auto load = [&](int t) {
#pragma unroll
    for (int k = 0; k < kConvTokens; ++k) raw_x[k].load(in.r, in.of(t + k)), raw_dy[k].load(grad.r, grad.of(t + k));
  };
#pragma unroll
  for (int k = 0; k + 1 < W; ++k) edge[k].load(in.r, in.of(at.first - (W - 1) + k));
  load(at.first);
  if (at.has) {
    Taps<V, W> taps;
    taps.load(p, at.c);
    float x[W][V], dpre[W][V];  // the last rows are the newest
#pragma unroll
    for (int k = 0; k + 1 < W; ++k) {
      if (at.first - (W - 1) + k < 0) state_row<T, V>(x[k + 1], p, at.b, at.c, at.first - (W - 1) + k);
      else edge[k].get(x[k + 1]);
    }
#pragma unroll
    for (int k = 0; k < W; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) dpre[k][i] = 0.f;
    const T* const final = static_cast<const T*>(p.d_final);
    const long long held = (long long)at.b * (W - 1);
    // the gradient of a token is whole once dpre of the token W - 1 behind it is there
    for (int t0 = at.first; t0 < at.end + W - 1; t0 += kConvTokens) {
      Piece<T, V> now_x[kConvTokens], now_dy[kConvTokens];
#pragma unroll
      for (int k = 0; k < kConvTokens; ++k) now_x[k] = raw_x[k], now_dy[k] = raw_dy[k];
      if (t0 + kConvTokens < at.end + W - 1) load(t0 + kConvTokens);
#pragma unroll
      for (int u = 0; u < kConvTokens; ++u) {
        const int t = t0 + u;
#pragma unroll
        for (int k = 0; k + 1 < W; ++k)
#pragma unroll
          for (int i = 0; i < V; ++i) x[k][i] = x[k + 1][i], dpre[k][i] = dpre[k + 1][i];
        now_x[u].get(x[W - 1]);
        now_dy[u].get(dpre[W - 1]);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          if (p.silu) {
            float s = taps.bias[i];
#pragma unroll
            for (int k = 0; k < W; ++k) s = fmaf(taps.w[i * W + k], x[k][i], s);
            const float g = sigmoidf_(s), d = dpre[W - 1][i] * fmaf(s * g, 1.f - g, g);
            dpre[W - 1][i] = t < p.L ? d : 0.f;
          }
          const float own = t < at.end ? dpre[W - 1][i] : 0.f;
          db[i] += own;
#pragma unroll
          for (int k = 0; k < W; ++k) dw[i][k] = fmaf(own, x[k][i], dw[i][k]);
        }
        const int to = t - (W - 1);  // (dpre[k] is of token to + k)
        float g[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
          g[i] = 0.f;
#pragma unroll
          for (int k = 0; k < W; ++k) g[i] = fmaf(taps.w[i * W + W - 1 - k], dpre[k][i], g[i]);
        }
        if (final && to >= p.L - (W - 1) && to < at.end) {
          float f[V];
          load_vec<V>(f, final + (held + to - (p.L - (W - 1))) * p.D + at.c);
#pragma unroll
          for (int i = 0; i < V; ++i) g[i] += f[i];
        }
        Piece<T, V> o;
        o.set(g);
        o.store(out.r, to >= at.first && to < at.end ? out.of(to) : kNowhere);
        if (to < 0 && at.first == 0 && p.d_initial) store_vec<V>(static_cast<T*>(p.d_initial) + (held + to + W - 1) * p.D + at.c, g);
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
    for (int k = 0; k < W; ++k) s = fmaf(taps.w[i * W + k], rows[k][i], s);
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
// Runs of tokens: as long as leaves two workgroups a compute unit (and `most`), so that few rows on their edges are read twice and few partial sums are left.  us, one / two / four a unit:
// forward of 128 x 196 x 768 17.9 / 18.0 / 19.7, of 4096 x 1024 6.6 / 7.0 / 7.0;  backward of 32 x 196 x 768 17.0 / 16.5 / 21.0, of 64 x 196 x 768 21.5 / 21.3 / 24.4, of 16384 x 1024
// 37.4 / 29.0 / 29.0.
void cut_runs(CausalConv& p, int V, int most) {
  p.blocks = (p.D + kConvLanes * V - 1) / (kConvLanes * V);
  const long long tokens = (long long)p.B * p.blocks * p.L / (kConvRuns * 512);
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
