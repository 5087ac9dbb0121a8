// The selective state space scan and its step for one token.
//
//   s_t = softplus(delta_t + bias)                                    (or delta_t + bias as it is)
//   h_t[n] = e^{s_t A[n]} h_{t-1}[n] + s_t x_t B_t[n]                  N numbers a channel; B, C of a token shared by the channels of a group
//   o_t = (sum_n C_t[n] h_t[n] + skip x_t) silu(z_t)
//
// Decays go by channel and state, so that no product of matrices is in it: for each number of state and token one exponential, four multiply-adds and a product.
#include "selective_scan.h"

namespace vig {
namespace {

// ---- forward.  FOLD: only what a chunk of tokens leaves from nothing, and the sum of its steps

template <typename S, int CN, bool FOLD>
__global__ __launch_bounds__(64 * kScanWaves) void selective_scan_kernel(SelScanArgs p) {
  constexpr int T = kTileTokens<CN>, R = T / 4, NP = 4 * CN;
  __shared__ __align__(16) Pass<CN, 2> lds[kScanWaves];
  const Stand at(p);
  Pass<CN, 2>& pass = lds[at.wave];
  const float bias = p.bias && at.has ? p.bias[at.c] : 0.f, skip = p.skip && at.has ? p.skip[at.c] : 0.f;
  float A[CN], h[CN];
  load_states(A, p.A, 0, p.D, p.N, p.N, at);
#pragma unroll
  for (int i = 0; i < CN; ++i) A[i] *= kLog2e;
  const size_t row = (size_t)at.b * p.chunks + at.chunk;
  if constexpr (FOLD) {
#pragma unroll
    for (int i = 0; i < CN; ++i) h[i] = 0.f;
  } else if (p.chunks > 1) {
    kept_states(h, p.ends, row, p.D, at);
  } else {
    load_states(h, p.h0, at.b, p.D, p.N, p.N, at);
  }
  const bool gated = !FOLD && p.z.at;
  float sum = 0.f;
  Channels<S, T> x, delta, z;
  Shared<S, CN> B, C;
  x.stand(p, p.x, at), delta.stand(p, p.delta, at), B.stand(p, p.B, at);
  if constexpr (!FOLD) C.stand(p, p.C, at), z.stand(p, p.z, at);
  const Line<S> out = dense_line<S>(p, p.o, at);
  auto load = [&](int first) {
    const Tile<T> tile(p, first, at.end);
    x.load(tile), delta.load(tile), B.load(tile);
    if constexpr (!FOLD) C.load(tile);
    if (gated) z.load(tile);
  };
  load(at.first);
  for (int first = at.first; first < at.end; first += T) {
    const Tile<T> tile(p, first, at.end);
    float xs[R], zs[R];
#pragma unroll
    for (int m = 0; m < R; ++m) {
      const float step = first + 4 * m + at.q < at.end ? step_of(delta.v[m] + bias, p.softplus) : 0.f;
      xs[m] = x.v[m], zs[m] = z.v[m];
      pass.of_channel[0][at.j][4 * m + at.q] = step;
      pass.of_channel[1][at.j][4 * m + at.q] = step * x.v[m];
      if constexpr (FOLD) sum += step;
    }
    B.pass(pass.of_token[0], at);
    if constexpr (!FOLD) C.pass(pass.of_token[1], at);
    passed();
    if (first + T < at.end) load(first + T);
    if constexpr (!FOLD)
      if (p.kept) keep_states(p.kept, h, (size_t)at.b * ((p.L + T - 1) / T) + first / T, p.D, at);
#pragma unroll
    for (int m = 0; m < R; ++m) {
      float step[4], u[4], s[4];
      read_lds(step, &pass.of_channel[0][at.j][4 * m]);
      read_lds(u, &pass.of_channel[1][at.j][4 * m]);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float b[CN], c[CN];
        read_lds(b, &pass.of_token[0][4 * m + k][at.q * CN]);
        if constexpr (!FOLD) read_lds(c, &pass.of_token[1][4 * m + k][at.q * CN]);
        s[k] = 0.f;
#pragma unroll
        for (int i = 0; i < CN; ++i) {
          h[i] = fmaf(u[k], b[i], __builtin_amdgcn_exp2f(step[k] * A[i]) * h[i]);
          if constexpr (!FOLD) s[k] = fmaf(c[i], h[i], s[k]);
        }
      }
      if constexpr (!FOLD) {
        float y = fmaf(skip, xs[m], of_rows(s[0], s[1], s[2], s[3]));
        if (gated) y *= zs[m] * sigmoidf_(zs[m]);
        out.store(tile, m, y);
      }
    }
    passed();
  }
  if constexpr (FOLD) {
    keep_states(p.ends, h, row, p.D, at);
    sum = of_all_rows(sum);
    if (at.q == 0 && at.has) p.sums[row * p.D + at.c] = sum;
  } else if (p.hT && at.chunk == p.chunks - 1) {
    store_states(p.hT, h, at.b, p.D, p.N, p.N, at);
  }
}

// What chunks leave -> what enters them, in place: along the walk (forward), or against it (backward, whose last chunk is entered by the end's gradient).
// A thread for each state of a channel.
template <bool BACK>
__global__ __launch_bounds__(256) void selective_join_kernel(SelScanArgs p, int np) {
  const long long n = (long long)p.D * np, id = (long long)blockIdx.x * 256 + threadIdx.x;
  if (id >= p.batch * n) return;
  const long long b = id / n, in = id - b * n;
  const int c = (int)(in / np), s = (int)(in - (long long)c * np);
  const float* from = BACK ? p.dhT : p.h0;
  float h = from && s < p.N ? from[(b * p.D + c) * p.N + s] : 0.f;
  const float A = s < p.N ? p.A[(long long)c * p.N + s] * kLog2e : 0.f;
  for (int k = 0; k < p.chunks; ++k) {
    const size_t row = (size_t)b * p.chunks + (BACK ? p.chunks - 1 - k : k);
    float* at = p.ends + row * n + in;
    const float leaves = *at, a = __builtin_amdgcn_exp2f(A * p.sums[row * p.D + c]);
    *at = h;
    h = fmaf(a, h, leaves);
  }
}

// ---- one token of every sequence.  NL lanes take a channel, four states each: side by side in pieces of 16 bytes (WHOLE), or NL apart.

template <typename S, int NL, bool WHOLE>
__global__ __launch_bounds__(256) void selective_step_kernel(SelScanStep p) {
  const long long id = ((long long)blockIdx.x * 256 + threadIdx.x) / NL;
  const int l = threadIdx.x % NL;
  const bool is = id < (long long)p.batch * p.D;  // (the others still take part in the sums)
  const long long at = is ? id : 0;
  const int b = (int)(at / p.D), c = (int)(at - (long long)b * p.D), g = c / (p.D / p.G);
  const float raw = Elem<S>::load(static_cast<const S*>(p.delta) + b * p.delta_stride + c) + (p.bias ? p.bias[c] : 0.f);
  const float x = Elem<S>::load(static_cast<const S*>(p.x) + b * p.x_stride + c);
  const S* const B = static_cast<const S*>(p.B) + b * p.B_strides[0] + g * p.B_strides[1];
  const S* const C = static_cast<const S*>(p.C) + b * p.C_strides[0] + g * p.C_strides[1];
  float* const state = p.state + at * p.N;
  const float* const decay = p.A + (long long)c * p.N;
  auto n = [&](int i) { return WHOLE ? 4 * l + i : l + NL * i; };
  float h[4], a[4];
  if constexpr (WHOLE) {
    if (4 * l < p.N) {
      const f32x4_t hv = *reinterpret_cast<const f32x4_t*>(state + 4 * l), av = *reinterpret_cast<const f32x4_t*>(decay + 4 * l);
#pragma unroll
      for (int i = 0; i < 4; ++i) h[i] = hv[i], a[i] = av[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n(i) < p.N) h[i] = state[n(i)], a[i] = decay[n(i)];
  }
  const float step = step_of(raw, p.softplus), u = step * x;
  float y = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (n(i) < p.N) {
      h[i] = fmaf(u, Elem<S>::load(B + n(i)), exp_fast(step * a[i]) * h[i]);
      y = fmaf(Elem<S>::load(C + n(i)), h[i], y);
    }
#pragma unroll
  for (int k = 1; k < NL; k *= 2) y += __shfl_xor(y, k);
  if (!is) return;
  if constexpr (WHOLE) {
    if (4 * l < p.N) *reinterpret_cast<f32x4_t*>(state + 4 * l) = f32x4_t{h[0], h[1], h[2], h[3]};
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n(i) < p.N) state[n(i)] = h[i];
  }
  if (l) return;
  if (p.skip) y = fmaf(p.skip[c], x, y);
  if (p.z) {
    const float z = Elem<S>::load(static_cast<const S*>(p.z) + b * p.z_stride + c);
    y *= z * sigmoidf_(z);
  }
  Elem<S>::store(static_cast<S*>(p.o) + at, y);
}

}  // namespace

int launch_selective_join(const SelScanArgs& p, int np, bool back, hipStream_t stream) {
  const long long n = (long long)p.batch * p.D * np;
  hipLaunchKernelGGL((back ? selective_join_kernel<true> : selective_join_kernel<false>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, stream, p, np);
  return hipGetLastError() == hipSuccess ? 0 : -5;
}

template <typename S, int CN>
static int run_forward(const SelScanArgs& p, hipStream_t stream) {
  const dim3 grid(scan_grid(p)), block(64 * kScanWaves);
  if (p.chunks > 1) {
    hipLaunchKernelGGL((selective_scan_kernel<S, CN, true>), grid, block, 0, stream, p);
    const int rc = launch_selective_join(p, 4 * CN, false, stream);
    if (rc) return rc;
  }
  hipLaunchKernelGGL((selective_scan_kernel<S, CN, false>), grid, block, 0, stream, p);
  return hipGetLastError() == hipSuccess ? 0 : -5;
}

template <typename S, int NL>
static int run_step(const SelScanStep& p, hipStream_t stream) {
  const long long groups = ((long long)p.batch * p.D * NL + 255) / 256;
  if (groups > 0xffffff) return -95;
  const bool whole = p.N % 4 == 0 && reinterpret_cast<uintptr_t>(p.state) % 16 == 0 && reinterpret_cast<uintptr_t>(p.A) % 16 == 0;
  hipLaunchKernelGGL((whole ? selective_step_kernel<S, NL, true> : selective_step_kernel<S, NL, false>), dim3((unsigned)groups), dim3(256), 0, stream, p);
  return hipGetLastError() == hipSuccess ? 0 : -5;
}

int launch_selective_scan_step(const SelScanStep& p, hipStream_t stream) {
  return by_states(scan_states(p.N), [&](auto nl) { return p.io_dtype == VIG_BF16 ? run_step<uint16_t, nl>(p, stream) : run_step<float, nl>(p, stream); });
}

int launch_selective_scan(SelScanArgs& p, void* workspace, int io_dtype, hipStream_t stream) {
  const int CN = scan_states(p.N);
  cut_chunks(p);
  if (!scan_fits(p)) return -95;
  p.ends = (float*)workspace;
  p.sums = p.ends + (size_t)p.batch * p.chunks * p.D * 4 * CN;
  return by_states(CN, [&](auto cn) { return io_dtype == VIG_BF16 ? run_forward<uint16_t, cn>(p, stream) : run_forward<float, cn>(p, stream); });
}

size_t selective_scan_workspace(int batch, int L, int D, int N, int G) {
  SelScanArgs p{};
  p.batch = batch, p.L = L, p.D = D, p.N = N, p.G = G;
  cut_chunks(p);
  return p.chunks > 1 ? sizeof(float) * (size_t)batch * p.chunks * D * (4 * scan_states(N) + 1) : 0;
}
size_t selective_scan_kept(int batch, int L, int D, int N) {
  const int CN = scan_states(N), T = scan_tile(CN);
  return sizeof(float) * (size_t)batch * ((L + T - 1) / T) * D * 4 * CN;
}

}  // namespace vig
