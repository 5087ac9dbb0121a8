// Residual add and layer norm over the last axis, and its gradients.
//
//   sum = x + residual, as stored;   xhat = (sum - mean) rstd,   y = xhat w + b
//   g = dy w:   d_sum' = rstd (g - mean(g) - xhat mean(g xhat)) + d_sum  (to x and the residual, a buffer each),   dw = sum over rows of dy xhat,   db = ... of dy
//
// Memory bounds it: a row lies in the registers of 32, 64 or 256 threads between its sums.  The backward's threads keep their columns' sums of the rows
// that they come by, a workgroup adds up its threads' and leaves a row of partial sums.
//
// Measured, 25088 x 768, bf16 rows beside an fp32 residual stream: forward 45 us, 5.1 TB/s, backward 57, 5.4 (a large copy: 5.4), sums of the parameters' gradients 4.
// The same sizes with both streams in fp32, forward and backward: 148 where both summands want their gradient, 122 where they were given one buffer (bf16: 83, by the host's calls, either way).
#include "common.h"
#include "launch.h"

#include <algorithm>
#include <type_traits>

namespace vig {
namespace {

// V elements from p on, in pieces of 16 bytes where V is 8
template <int V, typename T> __device__ __forceinline__ void take(float (&x)[V], const T* p) {
  if constexpr (V == 8) {
    Raw8<T> r;
    r.load(p);
    r.unpack(x);
  } else {
    x[0] = Elem<T>::load(p);
  }
}
template <int V> __device__ __forceinline__ void give(uint16_t* p, const float (&x)[V]) {
  if constexpr (V == 8) *reinterpret_cast<u32x4_t*>(p) = u32x4_t{pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7])};
  else Elem<uint16_t>::store(p, x[0]);
}
template <int V> __device__ __forceinline__ void give(float* p, const float (&x)[V]) {
  if constexpr (V == 8) {
    *reinterpret_cast<f32x4_t*>(p) = f32x4_t{x[0], x[1], x[2], x[3]};
    *reinterpret_cast<f32x4_t*>(p + 4) = f32x4_t{x[4], x[5], x[6], x[7]};
  } else {
    *p = x[0];
  }
}
__device__ __forceinline__ float stored(float x, float) { return x; }
__device__ __forceinline__ float stored(float x, uint16_t) { return bf16_to_f32(f32_to_bf16(x)); }

// Sums over the G threads of a row, in all of them.  G 256: through `board` (two of them in turn, so that one barrier a sum does).
template <int G> struct Sum {
  float (*board)[8];
  int turn = 0;
  __device__ __forceinline__ void operator()(float& a, float& b) {
    constexpr int lanes = G < 64 ? G : 64;
#pragma unroll
    for (int k = 1; k < lanes; k *= 2) a += __shfl_xor(a, k), b += __shfl_xor(b, k);
    if constexpr (G > 64) {
      float* const s = board[turn];
      turn ^= 1;
      const int wave = threadIdx.x >> 6;
      if ((threadIdx.x & 63) == 0) s[2 * wave] = a, s[2 * wave + 1] = b;
      __syncthreads();
      a = (s[0] + s[2]) + (s[4] + s[6]), b = (s[1] + s[3]) + (s[5] + s[7]);
    }
  }
};

template <typename TX, typename TS, int V, int NV, int G>
__global__ __launch_bounds__(256) void add_norm_kernel(AddNorm p) {
  constexpr int kRows = 256 / G;
  __shared__ float board[2][8];
  Sum<G> sum{board};
  const int lane = threadIdx.x % G;
  const long long row = p.first + (long long)blockIdx.x * kRows + threadIdx.x / G;
  const bool is = row < p.rows;  // (lanes of a missing row still take part in the sums)
  const long long base = (is ? row : 0) * p.C;
  float s[NV][V], w[NV][V], b[NV][V];
  float total = 0.f, none = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {  // (up to four pieces of the parameters on their way with the row; more would cost registers)
    const int c = (lane + G * i) * V;
    if (NV > 4 || c >= p.C) continue;
    take<V>(w[i], p.weight + c);
    if (p.bias) take<V>(b[i], p.bias + c);
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (lane + G * i) * V;
    if (c >= p.C) continue;
    take<V>(s[i], static_cast<const TX*>(p.x) + base + c);
    if (p.residual) {
      float r[V];
      take<V>(r, static_cast<const TS*>(p.residual) + base + c);
#pragma unroll
      for (int e = 0; e < V; ++e) s[i][e] = stored(s[i][e] + r[e], TS{});
      if (is) give<V>(static_cast<TS*>(p.sum) + base + c, s[i]);
    }
#pragma unroll
    for (int e = 0; e < V; ++e) total += s[i][e];
  }
  sum(total, none);
  const float mean = total / (float)p.C;
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if ((lane + G * i) * V < p.C) {
#pragma unroll
      for (int e = 0; e < V; ++e) s[i][e] -= mean, ss = fmaf(s[i][e], s[i][e], ss);
    }
  sum(ss, none);
  const float rstd = 1.f / sqrtf(ss / (float)p.C + p.eps);
  if (!is) return;
  if (p.stats && lane == 0) p.stats[2 * row] = mean, p.stats[2 * row + 1] = rstd;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (lane + G * i) * V;
    if (c >= p.C) continue;
    if (NV > 4) {
      take<V>(w[i], p.weight + c);
      if (p.bias) take<V>(b[i], p.bias + c);
    }
#pragma unroll
    for (int e = 0; e < V; ++e) s[i][e] = fmaf(s[i][e] * rstd, w[i][e], p.bias ? b[i][e] : 0.f);
    give<V>(static_cast<TX*>(p.y) + base + c, s[i]);
  }
}

template <typename TX, typename TS, int V, int NV, int G>
__global__ __launch_bounds__(256) void add_norm_bwd_kernel(AddNorm p) {
  constexpr int kRows = 256 / G;
  __shared__ float board[2][8];
  __shared__ float sums[G == 256 ? 1 : kRows][G == 256 ? 1 : G * V];
  Sum<G> sum{board};
  const int lane = threadIdx.x % G, sub = threadIdx.x / G;
  float w[NV][V], dw[NV][V], db[NV][V];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (lane + G * i) * V;
    if (c < p.C) take<V>(w[i], p.weight + c);
#pragma unroll
    for (int e = 0; e < V; ++e) dw[i][e] = db[i][e] = 0.f;
  }
  const long long first = (long long)blockIdx.x * p.each;
  for (long long at = first; at < min(first + p.each, p.rows); at += kRows) {
    const long long row = at + sub;
    const bool is = row < min(first + p.each, p.rows);
    const long long base = (is ? row : at) * p.C;
    const float mean = p.stats[2 * (is ? row : at)], rstd = p.stats[2 * (is ? row : at) + 1];
    float x[NV][V], dy[NV][V];
    float g1 = 0.f, g2 = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (lane + G * i) * V;
      if (c >= p.C) continue;
      take<V>(x[i], static_cast<const TS*>(p.held) + base + c);
      take<V>(dy[i], static_cast<const TX*>(p.dy) + base + c);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if ((lane + G * i) * V >= p.C) continue;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        x[i][e] = (x[i][e] - mean) * rstd;
        if (is) dw[i][e] = fmaf(dy[i][e], x[i][e], dw[i][e]), db[i][e] += dy[i][e];
        dy[i][e] *= w[i][e];
        g1 += dy[i][e], g2 = fmaf(dy[i][e], x[i][e], g2);
      }
    }
    sum(g1, g2);
    g1 /= (float)p.C, g2 /= (float)p.C;
    if (!is) continue;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (lane + G * i) * V;
      if (c >= p.C) continue;
      float d[V];
#pragma unroll
      for (int e = 0; e < V; ++e) d[e] = 0.f;
      if (p.d_sum) take<V>(d, static_cast<const TS*>(p.d_sum) + base + c);
#pragma unroll
      for (int e = 0; e < V; ++e) d[e] = fmaf(rstd, dy[i][e] - g1 - x[i][e] * g2, d[e]);
      if (p.dx) give<V>(static_cast<TX*>(p.dx) + base + c, d);
      if (p.d_residual) give<V>(static_cast<TS*>(p.d_residual) + base + c, d);
    }
  }
  if (!p.parts) return;
  float* const part = p.parts + (long long)blockIdx.x * 2 * p.C;
  if constexpr (G == 256) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (lane + G * i) * V;
      if (c >= p.C) continue;
#pragma unroll
      for (int e = 0; e < V; ++e) part[c + e] = dw[i][e], part[p.C + c + e] = db[i][e];
    }
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        __syncthreads();
#pragma unroll
        for (int e = 0; e < V; ++e) sums[sub][lane * V + e] = k ? db[i][e] : dw[i][e];
        __syncthreads();
        for (int e = threadIdx.x; e < G * V; e += 256) {
          float s = 0.f;
#pragma unroll
          for (int r = 0; r < kRows; ++r) s += sums[r][e];
          const int c = G * V * i + e;
          if (c < p.C) part[k * (long long)p.C + c] = s;
        }
      }
  }
}

int launched() { return hipGetLastError() == hipSuccess ? 0 : -5; }

// Eight elements a thread at once where rows begin on 16 bytes, else one; as few threads a row as hold it.  LONE: a workgroup for each row, where a wave a row would leave the chip to few of
// them, each with several pieces to go through.  us of the forward, bf16, a wave / a workgroup: wide, 16 x 768 3.64 / 3.35, 512 x 768 3.90 / 3.70, 1024 x 768 4.09 / 4.19, 16 x 2048 5.08 / 3.38,
// 16 x 384 (one piece a lane) 3.04 / 3.30; narrow, 16 x 999 8.86 / 4.21, 1024 x 385 5.79 / 4.48, 4096 x 385 7.54 / 8.68, 16 x 100 3.22 / 3.26.  The backward's workgroups take eight rows,
// four at a time in waves: one at a time takes 11.1 for 6.4 (16 x 384), 11.9 for 7.8 (16 x 768).
template <bool LONE, typename F> int by_width(bool wide, long long rows, int C, F f) {
#define VIG_NORM_CASE(V, NV, G) f(std::integral_constant<int, V>{}, std::integral_constant<int, NV>{}, std::integral_constant<int, G>{})
  if (wide) {
    if (LONE && rows <= 512 && C > 512 && C <= 2048) return VIG_NORM_CASE(8, 1, 256);
    if (C <= 256) return VIG_NORM_CASE(8, 1, 32);
    if (C <= 512) return VIG_NORM_CASE(8, 1, 64);
    if (C <= 1024) return VIG_NORM_CASE(8, 2, 64);
    if (C <= 2048) return VIG_NORM_CASE(8, 4, 64);
    if (C <= 4096) return VIG_NORM_CASE(8, 2, 256);
    return VIG_NORM_CASE(8, 8, 256);
  }
  if (LONE && rows <= 1024 && C > 256 && C <= 1024) return VIG_NORM_CASE(1, 4, 256);
  if (C <= 256) return VIG_NORM_CASE(1, 4, 64);
  if (C <= 1024) return VIG_NORM_CASE(1, 16, 64);
  if (C <= 4096) return VIG_NORM_CASE(1, 16, 256);
  return VIG_NORM_CASE(1, 64, 256);
#undef VIG_NORM_CASE
}
template <typename F> int by_types(int io_dtype, int sum_dtype, F f) {
  if (io_dtype == VIG_F32) return f(float{}, float{});
  return sum_dtype == VIG_F32 ? f(uint16_t{}, float{}) : f(uint16_t{}, uint16_t{});
}
bool wide(const AddNorm& p) {
  for (const void* t : {p.x, p.residual, (const void*)p.weight, (const void*)p.bias, (const void*)p.sum, (const void*)p.y, p.held, p.dy, p.d_sum, (const void*)p.d_residual, (const void*)p.dx})
    if (reinterpret_cast<uintptr_t>(t) % 16) return false;
  return p.C % 8 == 0;
}

}  // namespace

int launch_add_norm(AddNorm& p, hipStream_t stream) {
  constexpr long long most = 1LL << 23;  // rows of a launch: below 2^32 threads where a row takes a workgroup
  return by_types(p.io_dtype, p.sum_dtype, [&](auto tx, auto ts) {
    return by_width<true>(wide(p), p.rows, p.C, [&](auto v, auto nv, auto g) {
      for (p.first = 0; p.first < p.rows; p.first += most) {
        const long long groups = (std::min(most, p.rows - p.first) + 256 / g - 1) / (256 / g);
        hipLaunchKernelGGL((add_norm_kernel<decltype(tx), decltype(ts), v, nv, g>), dim3((unsigned)groups), dim3(256), 0, stream, p);
        if (const int rc = launched()) return rc;
      }
      return 0;
    });
  });
}

// Workgroups of the backward: enough to fill the chip, few enough that their partial sums are little beside the rows.  us with 256 / 512 / 1024 of them, bf16:  8192 x 768 21.9 / 16.9 / 17.7,
// 25088 x 768 51.4 / 33.7 / 29.6, 65536 x 384 77.7 / 45.9 / 34.7, 30000 x 4096 394 / 235 / 179;  four pieces a lane, which leave room for half as many: 20000 x 2048 83.8 / 65.1 / 74.2;
// long rows: 9000 x 8192 248 / 263 / 294, 16384 x 16384 794 / 828 / 880;  one element at a time: 9000 x 999 69.8 / 45.3 / 36.1, 20000 x 1501 261 / 141 / 81.
static long long norm_groups(long long rows, int C, bool wide) {
  const long long most = C > 4096 ? 256 : wide && ((C > 1024 && C <= 2048) || rows < 12000) ? 512 : 1024;
  return std::max(1LL, std::min(most, rows / 8));
}
size_t add_norm_bwd_workspace(long long rows, int C) { return sizeof(float) * std::max(norm_groups(rows, C, true), norm_groups(rows, C, false)) * 2 * (size_t)C; }

int launch_add_norm_bwd(AddNorm& p, void* workspace, hipStream_t stream) {
  p.parts = p.dparams ? (float*)workspace : nullptr;
  const long long want = norm_groups(p.rows, p.C, wide(p));
  p.each = (p.rows + want - 1) / want;
  const long long groups = (p.rows + p.each - 1) / p.each;
  const int rc = by_types(p.io_dtype, p.sum_dtype, [&](auto tx, auto ts) {
    return by_width<false>(wide(p), p.rows, p.C, [&](auto v, auto nv, auto g) {
      hipLaunchKernelGGL((add_norm_bwd_kernel<decltype(tx), decltype(ts), v, nv, g>), dim3((unsigned)groups), dim3(256), 0, stream, p);
      return launched();
    });
  });
  if (rc || !p.dparams) return rc;
  vig_sum_jobs sums{};
  if (!put_off(sums, p.parts, p.dparams, (int)groups, 2LL * p.C, false)) return -22;
  return launch_sum_jobs(sums, stream);
}

}  // namespace vig
