// The selective state space scan and its step for one token.
//
//   s_t = softplus(delta_t + bias)                                    (or delta_t + bias as it is)
//   h_t[n] = e^{s_t A[n]} h_{t-1}[n] + s_t x_t B_t[n]                  N numbers a channel; B, C of a token shared by the channels of a group
//   o_t = (sum_n C_t[n] h_t[n] + skip x_t) silu(z_t)
//
// Decays go by channel and state, so that no product of matrices is in it: for each number of state and token an exponential (two issue slots), a product for its exponent, one for
// the decay and two multiply-adds.  The vector pipe bounds it: 466 instructions a wave, tile of 16 tokens, 16 channels and 16 states, 320 of them these (64 of them double), the others
// the steps' softplus, gates, addresses and sums over the lane rows.  Sums over n stay in a lane for its four states, and h never leaves its registers.
//
// Sequences go through uncut where they give every compute unit a workgroup; else in chunks of tokens: a launch folds each (the state that it leaves from nothing, and the sum of its
// steps, which is all that a decay over it takes), and the chunks are joined by the walk itself or, many of them, by a launch in between.
//
// Measured, bf16, 16 states, gate: 128 x 196 x 768 83 us (3.7 M numbers of state a us; the rows alone, 156 MB, 29 at the rate of a copy; vector pipe 84 % busy, 6 waves a SIMD), 65536 x 1024
// fold 216, join 10, walk 295.  Tried: the products s x B as outer products of the matrix cores (16 blocks of 4 x 4): 88 to 90 cycles for 84 beside the arithmetic of a token,
// which they do not run beside.  A softplus of fewer instructions for bf16 rows: no gain, and states of less precision.
#include "selective_scan.h"

namespace vig {
namespace {

// ---- forward.  FOLD: only what a chunk of tokens leaves from nothing, and the sum of its steps

template <typename S, int CN, bool FOLD>
__global__ __launch_bounds__(64 * kScanWaves, CN > 4 ? 4 : FOLD ? 8 : 7) void selective_scan_kernel(SelScanArgs p) {
  constexpr int T = kTileTokens<CN>, R = T / 4, NP = 4 * CN;
  __shared__ __align__(16) Pass<CN> lds[kScanWaves];
  const Stand at(p);
  Pass<CN>& pass = lds[at.wave];
  const float bias = p.bias && at.has ? p.bias[at.c] : 0.f, skip = p.skip && at.has ? p.skip[at.c] : 0.f;
  float A[CN], h[CN];
  load_states(A, p.A, 0, p.D, p.N, p.N, at);
#pragma unroll
  for (int i = 0; i < CN; ++i) A[i] *= kLog2e;
  const size_t row = (size_t)at.b * p.chunks + at.chunk;
  const Kept<CN> kept(at);
  [[maybe_unused]] const int tiles = (p.L + T - 1) / T;
  if constexpr (FOLD) {
#pragma unroll
    for (int i = 0; i < CN; ++i) h[i] = 0.f;
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
  if constexpr (!FOLD) {  // (behind the first rows' loads, which are on their way meanwhile)
    if (p.chunks > kFewChunks) {
      kept.load(h, p.ends, row, p.D);
    } else {
      load_states(h, p.h0, at.b, p.D, p.N, p.N, at);
      entering<false>(h, A, p, at);
    }
  }
  for (int first = at.first; first < at.end; first += T) {
    const Tile<T> tile(p, first, at.end);
    float steps[R];
#pragma unroll
    for (int m = 0; m < R; ++m) steps[m] = step_of(delta[m] + bias, p.softplus);
    if (tile.rows < T) leave_out<R>(steps, tile.rows, at);
#pragma unroll
    for (int m = 0; m < R; ++m) {
      const float step = steps[m], xs = x[m];
      f32x4_t of = {step, step * xs, skip * xs, 1.f};
      if constexpr (!FOLD)
        if (gated) {
          const float zs = z[m];
          of[3] = zs * sigmoidf_(zs);
        }
      pass.of_channel[4 * m + at.q][at.j] = of;
      if constexpr (FOLD) sum += step;
    }
    B.pass(pass.of_token[0], at);
    if constexpr (!FOLD) C.pass(pass.of_token[1], at);
    passed();
    if (first + T < at.end) load(first + T);
    if constexpr (!FOLD)
      if (p.kept) kept.store(p.kept, (size_t)at.b * tiles + first / T, p.D, h);
    // a token's numbers are on their way while the one in front is worked on; the fences keep the compiler from reading further ahead, which would cost a wave a SIMD
    constexpr int kAhead = CN <= 8 ? 2 : 1;
    struct Token {
      f32x2_t of;
      float b[CN], c[CN];
    } ahead[kAhead];
    auto read = [&](int t) {
      Token& to = ahead[t % kAhead];
      to.of = *reinterpret_cast<const f32x2_t*>(&pass.of_channel[t][at.j]);
      read_lds(to.b, &pass.of_token[0][t][at.q * CN]);
      if constexpr (!FOLD) read_lds(to.c, &pass.of_token[1][t][at.q * CN]);
    };
    float s[4];
    if (kAhead > 1) read(0);
#pragma unroll
    for (int t = 0; t < T; ++t) {
      if (t % 4 == 0 && t >= tile.rows) break;  // (a last tile's tokens that are not there, by fours)
      __builtin_amdgcn_sched_barrier(0);
      if (kAhead == 1) read(t);
      else if (t + 1 < T) read(t + 1);
      const Token& now = ahead[t % kAhead];
      s[t % 4] = 0.f;
#pragma unroll
      for (int i = 0; i < CN; ++i) {
        h[i] = fmaf(now.of[1], now.b[i], __builtin_amdgcn_exp2f(now.of[0] * A[i]) * h[i]);
        if constexpr (!FOLD) s[t % 4] = fmaf(now.c[i], h[i], s[t % 4]);
      }
      if constexpr (!FOLD)
        if (t % 4 == 3) {
          const f32x4_t own = pass.of_channel[t - 3 + at.q][at.j];
          out.store(tile, t / 4, (of_rows(s[0], s[1], s[2], s[3]) + own[2]) * own[3]);
        }
    }
    passed();
  }
  if constexpr (FOLD) {
    kept.store(p.ends, row, p.D, h);
    sum = of_all_rows(sum);
    if (at.q == 0 && at.has) p.sums[row * p.D + at.c] = sum;
  } else if (p.hT && at.chunk == p.chunks - 1) {
    store_states(p.hT, h, at.b, p.D, p.N, p.N, at);
  }
}

// What chunks leave -> what enters them, in place: along the walk (forward), or against it (backward, whose last chunk is entered by the end's gradient).
// A thread for each state of a channel, eight chunks on their way together.
template <bool BACK>
__global__ __launch_bounds__(256) void selective_join_kernel(SelScanArgs p, int np) {
  constexpr int K = 8;
  const long long n = (long long)p.D * np, id = (long long)blockIdx.x * 256 + threadIdx.x;
  if (id >= p.batch * n) return;
  const long long b = id / n, in = id - b * n;
  const int c = (int)(in / np), s = (int)(in - (long long)c * np);
  const float* from = BACK ? p.dhT : p.h0;
  float h = from && s < p.N ? from[(b * p.D + c) * p.N + s] : 0.f;
  const float A = s < p.N ? p.A[(long long)c * p.N + s] * kLog2e : 0.f;
  auto row = [&](int k) { return (size_t)b * p.chunks + (BACK ? p.chunks - 1 - k : k); };
  for (int k0 = 0; k0 < p.chunks; k0 += K) {
    float leaves[K], sum[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const size_t r = row(min(k0 + k, p.chunks - 1));
      leaves[k] = p.ends[r * n + in], sum[k] = p.sums[r * p.D + c];
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (k0 + k >= p.chunks) break;
      p.ends[row(k0 + k) * n + in] = h;
      h = fmaf(__builtin_amdgcn_exp2f(A * sum[k]), h, leaves[k]);
    }
  }
}

// ---- one token of every sequence.  NL lanes take a channel, four states each: side by side in pieces of 16 bytes (WHOLE; B and C in whole fours then too), or NL apart.  A thread goes through
// ROWS sequences' states of the channel, all of them on their way together.

template <typename S> __device__ __forceinline__ void four(float (&v)[4], const S* from);
template <> __device__ __forceinline__ void four<uint16_t>(float (&v)[4], const uint16_t* from) {
  const u32x2_t w = *reinterpret_cast<const u32x2_t*>(from);
  v[0] = bf16lo_to_f32(w[0]), v[1] = bf16hi_to_f32(w[0]), v[2] = bf16lo_to_f32(w[1]), v[3] = bf16hi_to_f32(w[1]);
}
template <> __device__ __forceinline__ void four<float>(float (&v)[4], const float* from) {
  const f32x4_t w = *reinterpret_cast<const f32x4_t*>(from);
  v[0] = w[0], v[1] = w[1], v[2] = w[2], v[3] = w[3];
}

template <typename S, int NL, bool WHOLE, int ROWS>
__global__ __launch_bounds__(256) void selective_step_kernel(SelScanStep p) {
  constexpr int kChannels = 256 / NL;
  const int l = threadIdx.x % NL, c = (int)(blockIdx.x % (unsigned)p.blocks) * kChannels + threadIdx.x / NL, first = (int)(blockIdx.x / (unsigned)p.blocks) * ROWS;
  const bool is = c < p.D && (!WHOLE || 4 * l < p.N);
  auto n = [&](int i) { return WHOLE ? 4 * l + i : l + NL * i; };
  float a[4] = {0.f, 0.f, 0.f, 0.f}, h[ROWS][4], b[ROWS][4], g[ROWS][4], x[ROWS], raw[ROWS], z[ROWS];
  const int group = is ? c / (p.D / p.G) : 0;
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    const long long row = first + r;
    x[r] = raw[r] = z[r] = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) h[r][i] = b[r][i] = g[r][i] = 0.f;
    if (!is || row >= p.batch) continue;
    const float* const state = p.state + (row * p.D + c) * p.N;
    const S* const B = static_cast<const S*>(p.B) + row * p.B_strides[0] + group * p.B_strides[1];
    const S* const C = static_cast<const S*>(p.C) + row * p.C_strides[0] + group * p.C_strides[1];
    if constexpr (WHOLE) {
      four<float>(h[r], state + 4 * l), four<S>(b[r], B + 4 * l), four<S>(g[r], C + 4 * l);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (n(i) < p.N) h[r][i] = state[n(i)], b[r][i] = Elem<S>::load(B + n(i)), g[r][i] = Elem<S>::load(C + n(i));
    }
    x[r] = Elem<S>::load(static_cast<const S*>(p.x) + row * p.x_stride + c), raw[r] = Elem<S>::load(static_cast<const S*>(p.delta) + row * p.delta_stride + c);
    if (p.z) z[r] = Elem<S>::load(static_cast<const S*>(p.z) + row * p.z_stride + c);
  }
  float bias = 0.f, skip = 0.f;
  if (is) {
    const float* const decay = p.A + (long long)c * p.N;
    if constexpr (WHOLE) {
      four<float>(a, decay + 4 * l);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (n(i) < p.N) a[i] = decay[n(i)];
    }
    if (p.bias) bias = p.bias[c];
    if (p.skip) skip = p.skip[c];
  }
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    const float step = step_of(raw[r] + bias, p.softplus), u = step * x[r];
    float y = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      h[r][i] = fmaf(u, b[r][i], exp_fast(step * a[i]) * h[r][i]);
      // (a state that is not there may have become NaN of an infinite step)
      if (WHOLE || n(i) < p.N) y = fmaf(g[r][i], h[r][i], y);
    }
    if (!is) y = 0.f;
#pragma unroll
    for (int k = 1; k < NL; k *= 2) y += __shfl_xor(y, k);
    const long long row = first + r;
    if (!is || row >= p.batch) continue;
    float* const state = p.state + (row * p.D + c) * p.N;
    if constexpr (WHOLE) {
      *reinterpret_cast<f32x4_t*>(state + 4 * l) = f32x4_t{h[r][0], h[r][1], h[r][2], h[r][3]};
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (n(i) < p.N) state[n(i)] = h[r][i];
    }
    if (l) continue;
    y = fmaf(skip, x[r], y);
    if (p.z) y *= z[r] * sigmoidf_(z[r]);
    Elem<S>::store(static_cast<S*>(p.o) + row * p.D + c, y);
  }
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
    const int rc = p.chunks > kFewChunks ? launch_selective_join(p, 4 * CN, false, stream) : 0;
    if (rc) return rc;
  }
  hipLaunchKernelGGL((selective_scan_kernel<S, CN, false>), grid, block, 0, stream, p);
  return hipGetLastError() == hipSuccess ? 0 : -5;
}

template <typename S, int NL, bool WHOLE, int ROWS>
static int run_step(SelScanStep& p, hipStream_t stream) {
  p.blocks = (p.D + 256 / NL - 1) / (256 / NL);
  const long long groups = (long long)p.blocks * ((p.batch + ROWS - 1) / ROWS);
  if (groups > 0xffffff) return -95;
  hipLaunchKernelGGL((selective_step_kernel<S, NL, WHOLE, ROWS>), dim3((unsigned)groups), dim3(256), 0, stream, p);
  return hipGetLastError() == hipSuccess ? 0 : -5;
}
// Two sequences a thread once that leaves four workgroups a compute unit
template <typename S, int NL>
static int step_rows(SelScanStep& p, hipStream_t stream) {
  auto on = [](const void* t, size_t bytes) { return reinterpret_cast<uintptr_t>(t) % bytes == 0; };
  bool whole = p.N % 4 == 0 && on(p.state, 16) && on(p.A, 16) && on(p.B, 4 * sizeof(S)) && on(p.C, 4 * sizeof(S));
  for (int k = 0; k < 2; ++k) whole = whole && p.B_strides[k] % 4 == 0 && p.C_strides[k] % 4 == 0;
  const bool many = (long long)p.batch * p.D * NL / (2 * 256) >= 1024;
  if (whole) return many ? run_step<S, NL, true, 2>(p, stream) : run_step<S, NL, true, 1>(p, stream);
  return many ? run_step<S, NL, false, 2>(p, stream) : run_step<S, NL, false, 1>(p, stream);
}

int launch_selective_scan_step(SelScanStep& p, hipStream_t stream) {
  return by_states(scan_states(p.N), [&](auto nl) { return p.io_dtype == VIG_BF16 ? step_rows<uint16_t, nl>(p, stream) : step_rows<float, nl>(p, stream); });
}

int launch_selective_scan(SelScanArgs& p, void* workspace, int io_dtype, hipStream_t stream) {
  const int CN = scan_states(p.N);
  cut_chunks(p, false);
  p.ends = (float*)workspace;
  p.sums = p.ends + (size_t)p.batch * p.chunks * p.D * 4 * CN;
  return by_states(CN, [&](auto cn) { return io_dtype == VIG_BF16 ? run_forward<uint16_t, cn>(p, stream) : run_forward<float, cn>(p, stream); });
}

bool selective_scan_fits(int batch, int L, int D, int N, int G, bool back, bool training) {
  SelScanArgs p{};
  p.batch = batch, p.L = L, p.D = D, p.N = N, p.G = G;
  cut_chunks(p, back);
  return scan_fits(p, training);
}
size_t selective_scan_workspace(int batch, int L, int D, int N, int G) {
  SelScanArgs p{};
  p.batch = batch, p.L = L, p.D = D, p.N = N, p.G = G;
  cut_chunks(p, false);
  return p.chunks > 1 ? sizeof(float) * (size_t)batch * p.chunks * D * (4 * scan_states(N) + 1) : 0;
}
size_t selective_scan_kept(int batch, int L, int D, int N) {
  const int CN = scan_states(N), T = scan_tile(CN);
  return sizeof(float) * (size_t)batch * ((L + T - 1) / T) * D * 4 * CN;
}

}  // namespace vig
