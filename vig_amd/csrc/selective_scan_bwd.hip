// The selective scan's gradients.
//
//   dy_t = do_t silu(z_t),  dz_t = do_t y_t silu'(z_t)                                     (y: the output in front of the gate)
//   dh_t[n] = C_t[n] dy_t + a_{t+1}[n] dh_{t+1}[n],  a_t[n] = e^{s_t A[n]},  behind the last token: the final state's gradient
//   with p_t = a_t h_{t-1}:   dA[n] = sum_t s_t dh_t p_t,   ds_t = sum_n A[n] dh_t p_t + x_t du_t,   dx_t = s_t du_t + skip dy_t,   du_t = sum_n B_t[n] dh_t[n]
//   dB_t[n] = sum over the group's channels of s_t x_t dh_t[n],   dC_t[n] = ... of dy_t h_t[n],   dskip = sum_t x_t dy_t,   dbias = sum_t of the steps' gradients
//
// The forward kept the states that enter each tile of tokens.  A wave goes through its tiles against the walk: from the kept state forward again, with a and p of all of the
// tile's tokens left in registers (one exponential a number of state, as in the forward), then back.
// The vector pipe bounds it: 1424 instructions a tile of 16 tokens, 16 channels and 16 states, 830 of them the two walks, 256 the sums of dB and dC over the channels of a lane row, which
// go on over a workgroup's four waves through LDS and over workgroups by a launch behind (four waves: 2 bytes of partial sums a channel and token).  Two waves a SIMD have 256
// registers, 128 of them a and p.  Gradients of A, the skip and the bias stay in registers along the tokens; a launch adds up the sequences'.
//
// Measured, bf16, 16 states, gate: 128 x 196 x 768 266 to 302 us (the clock goes down under it), 50 at the rate of a copy for the rows; vector pipe 82 % busy.  Tiles of 8 tokens at three waves a
// SIMD: 359 for 345, kept states of twice the size.  Sums of the partial gradients 9, of the parameters' 6.
#include "selective_scan.h"

namespace vig {
namespace {

// Sums of eight values over the sixteen channels of a lane row: lane j is left in out[i] with that of value i + 2 (j >> 2 & 1) + 4 (j >> 3).
// Half the values stay with each half of the row, half of these with each half of it, and a sum over four lanes closes: 16 additions, each of them with its exchange of lanes, and the ones
// that only some lanes take behind the ones that all do.  In assembly, because the compiler makes a selection of each addition that only some lanes take (22 instructions).  An instruction
// that reads another lane's register stands two behind the one that wrote it: the compiler does not look in here.
__device__ __forceinline__ void of_channels(const float (&v)[8], float (&out)[2]) {
  float w0, w1, w2, w3;
  asm("s_nop 1\n\t"
      "v_add_f32_dpp %0, %6, %6 row_ror:8 row_mask:0xf bank_mask:0xf\n\t"
      "v_add_f32_dpp %1, %7, %7 row_ror:8 row_mask:0xf bank_mask:0xf\n\t"
      "v_add_f32_dpp %2, %8, %8 row_ror:8 row_mask:0xf bank_mask:0xf\n\t"
      "v_add_f32_dpp %3, %9, %9 row_ror:8 row_mask:0xf bank_mask:0xf\n\t"
      "v_add_f32_dpp %0, %10, %10 row_ror:8 row_mask:0xf bank_mask:0xc\n\t"
      "v_add_f32_dpp %1, %11, %11 row_ror:8 row_mask:0xf bank_mask:0xc\n\t"
      "v_add_f32_dpp %2, %12, %12 row_ror:8 row_mask:0xf bank_mask:0xc\n\t"
      "v_add_f32_dpp %3, %13, %13 row_ror:8 row_mask:0xf bank_mask:0xc\n\t"
      "v_add_f32_dpp %4, %0, %0 row_half_mirror row_mask:0xf bank_mask:0xf\n\t"
      "v_add_f32_dpp %5, %1, %1 row_half_mirror row_mask:0xf bank_mask:0xf\n\t"
      "v_add_f32_dpp %4, %2, %2 row_half_mirror row_mask:0xf bank_mask:0xa\n\t"
      "v_add_f32_dpp %5, %3, %3 row_half_mirror row_mask:0xf bank_mask:0xa\n\t"
      "s_nop 0\n\t"
      "v_add_f32_dpp %0, %4, %4 quad_perm:[1,0,3,2] row_mask:0xf bank_mask:0xf\n\t"
      "v_add_f32_dpp %1, %5, %5 quad_perm:[1,0,3,2] row_mask:0xf bank_mask:0xf\n\t"
      "s_nop 0\n\t"
      "v_add_f32_dpp %4, %0, %0 quad_perm:[2,3,0,1] row_mask:0xf bank_mask:0xf\n\t"
      "v_add_f32_dpp %5, %1, %1 quad_perm:[2,3,0,1] row_mask:0xf bank_mask:0xf"
      : "=&v"(w0), "=&v"(w1), "=&v"(w2), "=&v"(w3), "=&v"(out[0]), "=&v"(out[1])
      : "v"(v[0]), "v"(v[1]), "v"(v[2]), "v"(v[3]), "v"(v[4]), "v"(v[5]), "v"(v[6]), "v"(v[7]));
}

// A workgroup's sums of its waves' gradients of B (0) and C (1)
template <int CN> struct Board {
  float v[2][kTileTokens<CN>][4 * CN];
};

// What a lane reads of a token: its channel's step, dy, step times x and x, B and C
template <int CN> struct Token {
  f32x4_t of;
  float b[CN], c[CN];
  __device__ __forceinline__ void read(const Pass<CN>& pass, int t, const Stand& at, bool both) {
    of = pass.of_channel[t][at.j];
    if (both) read_lds(b, &pass.of_token[0][t][at.q * CN]);
    read_lds(c, &pass.of_token[1][t][at.q * CN]);
  }
};

// FOLD: only what a chunk hands back to the one in front of it
template <typename S, int CN, bool FOLD>
__global__ __launch_bounds__(64 * kScanWaves, FOLD ? 4 : 2) void selective_scan_bwd_kernel(SelScanArgs p) {
  constexpr int T = kTileTokens<CN>, R = T / 4, NP = 4 * CN;
  __shared__ __align__(16) Pass<CN> lds[kScanWaves];
  __shared__ __align__(16) Board<CN> boards[FOLD ? 1 : 2][FOLD ? 1 : kScanWaves];
  const Stand at(p);
  Pass<CN>& pass = lds[at.wave];
  const float bias = p.bias && at.has ? p.bias[at.c] : 0.f, skip = p.skip && at.has ? p.skip[at.c] : 0.f;
  float A[CN], back[CN];  // back: a dh of the token behind
  load_states(A, p.A, 0, p.D, p.N, p.N, at);
#pragma unroll
  for (int i = 0; i < CN; ++i) A[i] *= kLog2e;
  const size_t row = (size_t)at.b * p.chunks + at.chunk;
  const Kept<CN> states(at);
  if constexpr (FOLD) {
#pragma unroll
    for (int i = 0; i < CN; ++i) back[i] = 0.f;
  }
  const bool gated = p.z.at;
  float sum = 0.f, dskip = 0.f, dbias = 0.f, dA[CN];
#pragma unroll
  for (int i = 0; i < CN; ++i) dA[i] = 0.f;
  [[maybe_unused]] const Line<S> dx = dense_line<S>(p, p.dx, at), ddelta = dense_line<S>(p, p.ddelta, at), dz = dense_line<S>(p, p.dz, at);
  const int tiles = (p.L + T - 1) / T, last = at.first + (at.end - 1 - at.first) / T * T;
  Channels<S, T> x, delta, z, d_o;
  [[maybe_unused]] float kept[CN];
  Shared<S, CN> B, C;
  delta.stand(p, p.delta, at), d_o.stand(p, p.d_o, at), C.stand(p, p.C, at), z.stand(p, p.z, at);
  if constexpr (!FOLD) x.stand(p, p.x, at), B.stand(p, p.B, at);
  auto load = [&](int first) {
    const Tile<T> tile(p, first, at.end);
    delta.load(tile), d_o.load(tile), C.load(tile);
    if (gated) z.load(tile);
    if constexpr (!FOLD) x.load(tile), B.load(tile);
    if constexpr (!FOLD && CN <= 4) states.load(kept, p.kept, (size_t)at.b * tiles + first / T, p.D);  // (more of them have no room)
  };
  load(last);
  if constexpr (!FOLD) {  // (behind the first rows' loads, which are on their way meanwhile)
    if (p.chunks > kFewChunks) {
      states.load(back, p.ends, row, p.D);
    } else {
      load_states(back, p.dhT, at.b, p.D, p.N, p.N, at);
      entering<true>(back, A, p, at);
    }
  }
  for (int first = last, turn = 0; first >= at.first; first -= T, turn ^= 1) {
    [[maybe_unused]] const Tile<T> tile(p, first, at.end);
    float by_raw[R], by_y[R], steps[R];  // what makes gradients of raw steps of those of steps, and dz of y
#pragma unroll
    for (int m = 0; m < R; ++m) {
      const float raw = delta[m] + bias;
      steps[m] = step_of(raw, p.softplus), by_raw[m] = dstep_of(raw, p.softplus);
    }
    // (a token that is not there has no share in the bias's gradient either)
    if (tile.rows < T) leave_out<R>(steps, tile.rows, at), leave_out<R>(by_raw, tile.rows, at);
#pragma unroll
    for (int m = 0; m < R; ++m) {
      const float step = steps[m];
      float dy = d_o[m], xs = 0.f;
      if constexpr (!FOLD) xs = x[m];
      if (gated) {
        const float zs = z[m], s = sigmoidf_(zs), g = zs * s;
        by_y[m] = dy * fmaf(g, 1.f - s, s);
        dy *= g;
      }
      pass.of_channel[4 * m + at.q][at.j] = f32x4_t{step, dy, step * xs, xs};
      if constexpr (FOLD) sum += step;
    }
    if constexpr (!FOLD) B.pass(pass.of_token[0], at);
    C.pass(pass.of_token[1], at);
    passed();
    // a token's numbers are on their way while the one in front is worked on; the fences keep the compiler from reading further ahead, for which there are no registers
    constexpr int kAhead = CN <= 4 ? 2 : 1;
    Token<CN> ahead[kAhead];
    if constexpr (FOLD) {
      if (first > at.first) load(first - T);
      if (kAhead > 1) ahead[(T - 1) % kAhead].read(pass, T - 1, at, false);
#pragma unroll
      for (int t = T - 1; t >= 0; --t) {
        if (kAhead == 1) ahead[0].read(pass, t, at, false);
        else if (t > 0) ahead[(t - 1) % kAhead].read(pass, t - 1, at, false);
        if (t / 4 * 4 >= tile.rows) continue;  // (a last tile's tokens that are not there, by fours)
        const Token<CN>& now = ahead[t % kAhead];
#pragma unroll
        for (int i = 0; i < CN; ++i) back[i] = __builtin_amdgcn_exp2f(now.of[0] * A[i]) * fmaf(now.c[i], now.of[1], back[i]);
      }
      passed();
    } else {
      Board<CN>& board = boards[turn][at.wave];
      // eight values of tokens and states at a time: of 8 / CN tokens behind one another, or of a token's states by eights
      constexpr int TT = CN >= 8 ? 1 : 8 / CN, NN = CN >= 8 ? 8 : CN;
      auto shared = [&](const float (&v)[8], int which, int token, int state) {
        float s[2];
        of_channels(v, s);
        const int i = at.j & 1, e = i + 2 * (at.j >> 2 & 1) + 4 * (at.j >> 3);
        board.v[which][token + e / NN][at.q * CN + state + e % NN] = i ? s[1] : s[0];
      };
      // A last tile's tokens that are not there are left out by fours where a lane has eight states: the blocks that this makes need no spilled registers then (42 without).  A tile of sixteen
      // states is four tokens, one of which is there, so that nothing is ever left out; the branches part the code all the same, and leave 51 (bf16) and 54 (fp32) spilled registers of 134.
      // Up to four states the tokens are gone through with steps of 0: blocks cost 303 us for 278 there (128 x 196 x 768, 16 states, 13 tiles of which the last is a quarter; 2 spilled registers at
      // four states, none below).
      constexpr bool kSkip = CN >= 8;
      float h[CN], a[T][CN], ph[T][CN], few[8], of_four[4];
      if constexpr (CN > 4) states.load(kept, p.kept, (size_t)at.b * tiles + first / T, p.D);
#pragma unroll
      for (int i = 0; i < CN; ++i) h[i] = kept[i];
      // forward again
      if (kAhead > 1) ahead[0].read(pass, 0, at, true);
#pragma unroll
      for (int t = 0; t < T; ++t) {
        if (kSkip && t % 4 == 0 && t >= tile.rows) break;
        __builtin_amdgcn_sched_barrier(0);
        if (kAhead == 1) ahead[0].read(pass, t, at, true);
        else if (t + 1 < T) ahead[(t + 1) % kAhead].read(pass, t + 1, at, true);
        const Token<CN>& now = ahead[t % kAhead];
        of_four[t % 4] = 0.f;
#pragma unroll
        for (int i = 0; i < CN; ++i) {
          a[t][i] = __builtin_amdgcn_exp2f(now.of[0] * A[i]);
          ph[t][i] = a[t][i] * h[i];
          h[i] = fmaf(now.of[2], now.b[i], ph[t][i]);
          of_four[t % 4] = fmaf(now.c[i], h[i], of_four[t % 4]);
          few[t % TT * NN + i % 8] = now.of[1] * h[i];
          if (t % TT == TT - 1 && i % 8 == NN - 1) shared(few, 1, t - (TT - 1), i - (NN - 1));
        }
        if (t % 4 == 3 && gated) {
          const int m = t / 4;
          dz.store(tile, m, by_y[m] * fmaf(skip, pass.of_channel[4 * m + at.q][at.j][3], of_rows(of_four[0], of_four[1], of_four[2], of_four[3])));
        }
      }
      // and back
      float of_du[4];
      if (kAhead > 1) ahead[(T - 1) % kAhead].read(pass, T - 1, at, true);
#pragma unroll
      for (int t = T - 1; t >= 0; --t) {
        __builtin_amdgcn_sched_barrier(0);
        if (kAhead == 1) ahead[0].read(pass, t, at, true);
        else if (t > 0) ahead[(t - 1) % kAhead].read(pass, t - 1, at, true);
        if (kSkip && t / 4 * 4 >= tile.rows) {
          if (t == T - 4 && first > at.first) load(first - T);
          continue;
        }
        const Token<CN>& now = ahead[t % kAhead];
        of_du[t % 4] = of_four[t % 4] = 0.f;
#pragma unroll
        for (int i = 0; i < CN; ++i) {
          const float dh = fmaf(now.c[i], now.of[1], back[i]), e = dh * ph[t][i];
          of_du[t % 4] = fmaf(now.b[i], dh, of_du[t % 4]);
          of_four[t % 4] = fmaf(A[i], e, of_four[t % 4]);
          dA[i] = fmaf(now.of[0], e, dA[i]);
          back[i] = a[t][i] * dh;
          few[t % TT * NN + i % 8] = dh * now.of[2];
          if (t % TT == 0 && i % 8 == NN - 1) shared(few, 0, t, i - (NN - 1));
        }
        if (t % 4 == 0) {
          const int m = t / 4;
          const float du = of_rows(of_du[0], of_du[1], of_du[2], of_du[3]), dd = of_rows(of_four[0], of_four[1], of_four[2], of_four[3]);
          const f32x4_t own = pass.of_channel[4 * m + at.q][at.j];
          const float ds = fmaf(own[3], du, dd * kLn2) * by_raw[m];
          dx.store(tile, m, fmaf(own[0], du, skip * own[1]));
          ddelta.store(tile, m, ds);
          dbias += ds, dskip = fmaf(own[1], own[3], dskip);
          // (the next tile's rows, into registers that the last tokens' factors have left)
          if (m == R - 1 && first > at.first) load(first - T);
        }
      }
      // the workgroup's sums (the other turn's are read until the next barrier)
      __syncthreads();
      constexpr int kSums = 2 * T * NP, kThreads = 64 * kScanWaves;
      const size_t rows = (((size_t)at.b * p.G + at.g) * p.blocks + at.block) * p.L + tile.lowest;
      const rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(p.shared + rows * 2 * NP, 0, tile.rows * 2 * NP * (int)sizeof(float), 0x00020000);
#pragma unroll
      for (int k = 0; k < (kSums + kThreads - 1) / kThreads; ++k) {
        const int e = threadIdx.x + k * kThreads, n = e % NP, which = e / NP % 2, t = e / (2 * NP);
        float s = 0.f;
        if (kSums % kThreads == 0 || e < kSums) {
#pragma unroll
          for (int w = 0; w < kScanWaves; ++w) s += boards[turn][w].v[which][t][n];
        }
        // (tokens behind the end lie outside the descriptor; so do numbers behind the tile's)
        const unsigned to = (unsigned)(((tile.from + tile.step * t) * 2 + which) * NP + n) * sizeof(float);
        store1(r, kSums % kThreads == 0 || e < kSums ? to : kNowhere, s, 0.f);
      }
    }
  }
  if constexpr (FOLD) {
    states.store(p.ends, row, p.D, back);
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

// dB, dC [B, L, G, N]: the sums over a group's workgroups.  A thread takes four states of a token's dB or dC, four workgroups' on their way together.
template <typename S>
__global__ __launch_bounds__(256) void selective_shared_kernel(SelScanArgs p, int np) {
  constexpr int K = 4;
  const long long each = (long long)p.L * 2 * np, id = ((long long)blockIdx.x * 256 + threadIdx.x) * 4;  // of a group: token, which, state
  if (id >= each * p.batch * p.G) return;
  const long long bg = id / each, in = id - bg * each;
  const int n = (int)(in % np), which = (int)(in / np % 2);
  const long long t = in / (2 * np);
  if (n >= p.N) return;
  const float* from = p.shared + bg * p.blocks * each + in;
  f32x4_t s = {0.f, 0.f, 0.f, 0.f};
  for (int k0 = 0; k0 < p.blocks; k0 += K) {
    f32x4_t v[K];
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = k0 + k < p.blocks ? *reinterpret_cast<const f32x4_t*>(from + (k0 + k) * each) : f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < K; ++k) s += v[k];
  }
  const long long b = bg / p.G;
  S* const to = static_cast<S*>(which ? p.dC : p.dB) + ((b * p.L + t) * p.G + (bg - b * p.G)) * p.N + n;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (n + i < p.N) Elem<S>::store(to + i, s[i]);
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
  hipLaunchKernelGGL((selective_shared_kernel<S>), dim3((unsigned)shared_groups(p)), dim3(256), 0, stream, p, 4 * CN);
  if (hipGetLastError() != hipSuccess) return -5;
  vig_sum_jobs sums{};
  if (!put_off(sums, p.params, p.dparams, p.batch * p.chunks, (long long)p.D * (p.N + 2), false)) return -22;
  return launch_sum_jobs(sums, stream);
}

static size_t cut_workspace(SelScanArgs& p, void* workspace) {
  const int CN = scan_states(p.N);
  cut_chunks(p, true);
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
  return by_states(scan_states(p.N), [&](auto cn) { return io_dtype == VIG_BF16 ? run_backward<uint16_t, cn>(p, stream) : run_backward<float, cn>(p, stream); });
}
size_t selective_scan_bwd_workspace(int batch, int L, int D, int N, int G) {
  SelScanArgs p{};
  p.batch = batch, p.L = L, p.D = D, p.N = N, p.G = G;
  return cut_workspace(p, nullptr);
}

}  // namespace vig
