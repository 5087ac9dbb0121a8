// The selective scan's gradients.
//
//   dy_t = do_t silu(z_t),  dz_t = do_t y_t silu'(z_t)                                     (y: the output in front of the gate)
//   dh_t[n] = C_t[n] dy_t + a_{t+1}[n] dh_{t+1}[n],  a_t[n] = e^{s_t A[n]},  behind the last token: the final state's gradient
//   with p_t = a_t h_{t-1}:   dA[n] = sum_t s_t dh_t p_t,   ds_t = sum_n A[n] dh_t p_t + x_t du_t,   dx_t = s_t du_t + skip dy_t,   du_t = sum_n B_t[n] dh_t[n]
//   dB_t[n] = sum over the group's channels of s_t x_t dh_t[n],   dC_t[n] = ... of dy_t h_t[n],   dskip = sum_t x_t dy_t,   dbias = sum_t of the steps' gradients
//
// The forward kept the states that enter each tile of tokens.  A wave goes through its tiles against the walk: from the kept state forward again, with a and p of all of the
// tile's tokens left in registers (one exponential a number of state, as in the forward), then back.
#include "selective_scan.h"

namespace vig {
namespace {

template <int CTRL> __device__ __forceinline__ float from_lane(float x) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, true));
}
// Sums of eight values over the sixteen channels of a lane row: lane j holds in out[i] those of value i + 2 (j >> 2 & 1) + 4 (j >> 3).
__device__ __forceinline__ void of_channels(const float (&v)[8], float (&out)[2], int j) {
  float w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = (j & 8 ? v[i + 4] : v[i]) + from_lane<0x128>(j & 8 ? v[i] : v[i + 4]);  // (row_ror:8)
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    // (row_half_mirror: the other four of eight, in some order)
    float s = (j & 4 ? w[i + 2] : w[i]) + from_lane<0x141>(j & 4 ? w[i] : w[i + 2]);
    s += from_lane<0xb1>(s);  // (quad_perm 1 0 3 2)
    out[i] = s + from_lane<0x4e>(s);  // (quad_perm 2 3 0 1)
  }
}

// A workgroup's sums of its waves' gradients of B (0) and C (1)
template <int CN> struct Board {
  float v[2][kTileTokens<CN>][4 * CN];
};

// FOLD: only what a chunk hands back to the one in front of it
template <typename S, int CN, bool FOLD>
__global__ __launch_bounds__(64 * kScanWaves, FOLD ? 4 : 2) void selective_scan_bwd_kernel(SelScanArgs p) {
  constexpr int T = kTileTokens<CN>, R = T / 4, NP = 4 * CN;
  __shared__ __align__(16) Pass<CN, 3> lds[kScanWaves];
  __shared__ __align__(16) Board<CN> boards[FOLD ? 1 : 2][FOLD ? 1 : kScanWaves];
  const Stand at(p);
  Pass<CN, 3>& pass = lds[at.wave];
  const float bias = p.bias && at.has ? p.bias[at.c] : 0.f, skip = p.skip && at.has ? p.skip[at.c] : 0.f;
  float A[CN], back[CN];  // back: a dh of the token behind
  load_states(A, p.A, 0, p.D, p.N, p.N, at);
#pragma unroll
  for (int i = 0; i < CN; ++i) A[i] *= kLog2e;
  const size_t row = (size_t)at.b * p.chunks + at.chunk;
  if constexpr (FOLD) {
#pragma unroll
    for (int i = 0; i < CN; ++i) back[i] = 0.f;
  } else if (p.chunks > kFewChunks) {
    kept_states(back, p.ends, row, p.D, at);
  } else {
    load_states(back, p.dhT, at.b, p.D, p.N, p.N, at);
    entering<true>(back, A, p, at);
  }
  const bool gated = p.z.at;
  float sum = 0.f, dskip = 0.f, dbias = 0.f, dA[CN];
#pragma unroll
  for (int i = 0; i < CN; ++i) dA[i] = 0.f;
  [[maybe_unused]] const Line<S> dx = dense_line<S>(p, p.dx, at), ddelta = dense_line<S>(p, p.ddelta, at), dz = dense_line<S>(p, p.dz, at);
  const int tiles = (p.L + T - 1) / T, last = at.first + (at.end - 1 - at.first) / T * T;
  Channels<S, T> x, delta, z, d_o;
  Shared<S, CN> B, C;
  delta.stand(p, p.delta, at), d_o.stand(p, p.d_o, at), C.stand(p, p.C, at), z.stand(p, p.z, at);
  if constexpr (!FOLD) x.stand(p, p.x, at), B.stand(p, p.B, at);
  auto load = [&](int first) {
    const Tile<T> tile(p, first, at.end);
    delta.load(tile), d_o.load(tile), C.load(tile);
    if (gated) z.load(tile);
    if constexpr (!FOLD) x.load(tile), B.load(tile);
  };
  load(last);
  for (int first = last, turn = 0; first >= at.first; first -= T, turn ^= 1) {
    [[maybe_unused]] const Tile<T> tile(p, first, at.end);
    float raw[R], xs[R], by_y[R];  // by_y: what makes dz of y
#pragma unroll
    for (int m = 0; m < R; ++m) {
      raw[m] = delta.v[m] + bias, xs[m] = x.v[m];
      const float step = first + 4 * m + at.q < at.end ? step_of(raw[m], p.softplus) : 0.f;
      float dy = d_o.v[m];
      if (gated) {
        const float s = sigmoidf_(z.v[m]), g = z.v[m] * s;
        by_y[m] = dy * fmaf(g, 1.f - s, s);
        dy *= g;
      }
      pass.of_channel[0][at.j][4 * m + at.q] = step;
      pass.of_channel[1][at.j][4 * m + at.q] = dy;
      if constexpr (FOLD) sum += step;
      else pass.of_channel[2][at.j][4 * m + at.q] = step * xs[m];
    }
    if constexpr (!FOLD) B.pass(pass.of_token[0], at);
    C.pass(pass.of_token[1], at);
    passed();
    if constexpr (FOLD) {
      if (first > at.first) load(first - T);
#pragma unroll
      for (int m = R - 1; m >= 0; --m) {
        float step[4], d[4];
        read_lds(step, &pass.of_channel[0][at.j][4 * m]);
        read_lds(d, &pass.of_channel[1][at.j][4 * m]);
#pragma unroll
        for (int k = 3; k >= 0; --k) {
          float c[CN];
          read_lds(c, &pass.of_token[1][4 * m + k][at.q * CN]);
#pragma unroll
          for (int i = 0; i < CN; ++i) back[i] = __builtin_amdgcn_exp2f(step[k] * A[i]) * fmaf(c[i], d[k], back[i]);
        }
      }
      passed();
    } else {
      Board<CN>& board = boards[turn][at.wave];
      // eight values of tokens and states at a time: of 8 / CN tokens behind one another, or of a token's states by eights
      constexpr int TT = CN >= 8 ? 1 : 8 / CN, NN = CN >= 8 ? 8 : CN;
      auto shared = [&](const float (&v)[8], int which, int token, int state) {
        float s[2];
        of_channels(v, s, at.j);
        const int i = at.j & 1, e = i + 2 * (at.j >> 2 & 1) + 4 * (at.j >> 3);
        board.v[which][token + e / NN][at.q * CN + state + e % NN] = i ? s[1] : s[0];
      };
      float h[CN], a[T][CN], ph[T][CN];
      kept_states(h, p.kept, (size_t)at.b * tiles + first / T, p.D, at);
      // forward again
      float few[8];
#pragma unroll
      for (int m = 0; m < R; ++m) {
        __builtin_amdgcn_sched_barrier(0);
        float step[4], d[4], u[4], s[4];
        read_lds(step, &pass.of_channel[0][at.j][4 * m]);
        read_lds(d, &pass.of_channel[1][at.j][4 * m]);
        read_lds(u, &pass.of_channel[2][at.j][4 * m]);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int t = 4 * m + k;
          if constexpr (CN >= 8) __builtin_amdgcn_sched_barrier(0);
          float b[CN], c[CN];
          read_lds(b, &pass.of_token[0][t][at.q * CN]);
          read_lds(c, &pass.of_token[1][t][at.q * CN]);
          s[k] = 0.f;
#pragma unroll
          for (int i = 0; i < CN; ++i) {
            a[t][i] = __builtin_amdgcn_exp2f(step[k] * A[i]);
            ph[t][i] = a[t][i] * h[i];
            h[i] = fmaf(u[k], b[i], ph[t][i]);
            s[k] = fmaf(c[i], h[i], s[k]);
            few[t % TT * NN + i % 8] = d[k] * h[i];
            if (t % TT == TT - 1 && i % 8 == NN - 1) shared(few, 1, t - (TT - 1), i - (NN - 1));
          }
        }
        if (gated) dz.store(tile, m, by_y[m] * fmaf(skip, xs[m], of_rows(s[0], s[1], s[2], s[3])));
      }
      // and back
#pragma unroll
      for (int m = R - 1; m >= 0; --m) {
        __builtin_amdgcn_sched_barrier(0);
        float step[4], d[4], u[4], du[4], dd[4];
        read_lds(step, &pass.of_channel[0][at.j][4 * m]);
        read_lds(d, &pass.of_channel[1][at.j][4 * m]);
        read_lds(u, &pass.of_channel[2][at.j][4 * m]);
#pragma unroll
        for (int k = 3; k >= 0; --k) {
          const int t = 4 * m + k;
          if constexpr (CN >= 8) __builtin_amdgcn_sched_barrier(0);
          float b[CN], c[CN];
          read_lds(b, &pass.of_token[0][t][at.q * CN]);
          read_lds(c, &pass.of_token[1][t][at.q * CN]);
          du[k] = dd[k] = 0.f;
#pragma unroll
          for (int i = 0; i < CN; ++i) {
            const float dh = fmaf(c[i], d[k], back[i]), e = dh * ph[t][i];
            du[k] = fmaf(b[i], dh, du[k]);
            dd[k] = fmaf(A[i], e, dd[k]);
            dA[i] = fmaf(step[k], e, dA[i]);
            back[i] = a[t][i] * dh;
            few[t % TT * NN + i % 8] = dh * u[k];
            if (t % TT == 0 && i % 8 == NN - 1) shared(few, 0, t, i - (NN - 1));
          }
        }
        const float du_m = of_rows(du[0], du[1], du[2], du[3]), dd_m = of_rows(dd[0], dd[1], dd[2], dd[3]);
        const float dy = pass.of_channel[1][at.j][4 * m + at.q];
        const float ds = fmaf(xs[m], du_m, dd_m * kLn2) * dstep_of(raw[m], p.softplus);
        dx.store(tile, m, fmaf(pass.of_channel[0][at.j][4 * m + at.q], du_m, skip * dy));
        ddelta.store(tile, m, ds);
        if (first + 4 * m + at.q < at.end) dbias += ds, dskip = fmaf(dy, xs[m], dskip);
        // (the next tile's rows, into registers that the last tokens' factors have left)
        if (m == R - 1 && first > at.first) load(first - T);
      }
      // the workgroup's sums (the other turn's are read until the next barrier)
      __syncthreads();
      const size_t rows = (((size_t)at.b * p.G + at.g) * p.blocks + at.block) * p.L;
      for (int e = threadIdx.x; e < 2 * T * NP; e += 64 * kScanWaves) {
        const int n = e % NP, which = e / NP % 2, t = first + e / (2 * NP);
        if (t >= at.end) break;
        float s = 0.f;
#pragma unroll
        for (int w = 0; w < kScanWaves; ++w) s += boards[turn][w].v[which][t - first][n];
        p.shared[((rows + (p.reverse ? p.L - 1 - t : t)) * 2 + which) * NP + n] = s;
      }
    }
  }
  if constexpr (FOLD) {
    keep_states(p.ends, back, row, p.D, at);
    sum = of_all_rows(sum);
    if (at.q == 0 && at.has) p.sums[row * p.D + at.c] = sum;
  } else {
    if (p.dh0 && at.chunk == 0) store_states(p.dh0, back, at.b, p.D, p.N, p.N, at);
    const size_t each = (size_t)p.D * (p.N + 2);
    store_states(p.params + row * each, dA, 0, p.D, p.N, p.N, at);
    dskip = of_all_rows(dskip), dbias = of_all_rows(dbias);
    if (at.q == 0 && at.has) {
      float* to = p.params + row * each + (size_t)p.D * p.N + at.c;
      to[0] = dskip, to[p.D] = dbias;
    }
  }
}

// dB, dC [B, L, G, N]: the sums over a group's workgroups
template <typename S>
__global__ __launch_bounds__(256) void selective_shared_kernel(SelScanArgs p, int np) {
  const long long each = (long long)p.L * 2 * np, id = (long long)blockIdx.x * 256 + threadIdx.x;  // a thread: group, token, which, state
  if (id >= each * p.batch * p.G) return;
  const long long bg = id / each, in = id - bg * each;
  const int n = (int)(in % np), which = (int)(in / np % 2);
  const long long t = in / (2 * np);
  if (n >= p.N) return;
  const float* from = p.shared + bg * p.blocks * each + in;
  float s = 0.f;
  for (int k = 0; k < p.blocks; ++k) s += from[k * each];
  const long long b = bg / p.G;
  Elem<S>::store(static_cast<S*>(which ? p.dC : p.dB) + ((b * p.L + t) * p.G + (bg - b * p.G)) * p.N + n, s);
}

}  // namespace

template <typename S, int CN>
static int run_backward(const SelScanArgs& p, hipStream_t stream) {
  const dim3 grid(scan_grid(p)), block(64 * kScanWaves);
  if (p.chunks > 1) {
    hipLaunchKernelGGL((selective_scan_bwd_kernel<S, CN, true>), grid, block, 0, stream, p);
    const int rc = p.chunks > kFewChunks ? launch_selective_join(p, 4 * CN, true, stream) : 0;
    if (rc) return rc;
  }
  hipLaunchKernelGGL((selective_scan_bwd_kernel<S, CN, false>), grid, block, 0, stream, p);
  const long long n = (long long)p.batch * p.G * p.L * 8 * CN;
  hipLaunchKernelGGL((selective_shared_kernel<S>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, stream, p, 4 * CN);
  if (hipGetLastError() != hipSuccess) return -5;
  vig_sum_jobs sums{};
  if (!put_off(sums, p.params, p.dparams, p.batch * p.chunks, (long long)p.D * (p.N + 2), false)) return -22;
  return launch_sum_jobs(sums, stream);
}

static size_t cut_workspace(SelScanArgs& p, void* workspace) {
  const int CN = scan_states(p.N);
  cut_chunks(p);
  const size_t rows = (size_t)p.batch * p.chunks;
  float* at = (float*)workspace;
  p.ends = at, at += p.chunks > 1 ? rows * p.D * 4 * CN : 0;
  p.shared = at, at += (size_t)p.batch * p.G * p.blocks * p.L * 8 * CN;
  p.sums = at, at += p.chunks > 1 ? rows * p.D : 0;
  p.params = at, at += rows * p.D * (p.N + 2);
  return (char*)at - (char*)workspace;
}

int launch_selective_scan_bwd(SelScanArgs& p, void* workspace, int io_dtype, hipStream_t stream) {
  cut_workspace(p, workspace);
  if (!scan_fits(p)) return -95;
  return by_states(scan_states(p.N), [&](auto cn) { return io_dtype == VIG_BF16 ? run_backward<uint16_t, cn>(p, stream) : run_backward<float, cn>(p, stream); });
}
size_t selective_scan_bwd_workspace(int batch, int L, int D, int N, int G) {
  SelScanArgs p{};
  p.batch = batch, p.L = L, p.D = D, p.N = N, p.G = G;
  return cut_workspace(p, nullptr);
}

}  // namespace vig
