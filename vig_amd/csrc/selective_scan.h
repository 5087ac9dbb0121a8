// The selective scan's pieces that its forward and its backward share (selective_scan.hip, selective_scan_bwd.hip).
//
// A wave takes sixteen channels: lane = 16 q + j holds the states n = q CN .. q CN + CN - 1 of channel j, so that a row of sixteen lanes reads a row of a
// tensor.  Tokens come in tiles of T = 4 R: the lane loads, prepares (step, step times x, gate) and stores the tokens 4 m + q of its channel, m < R, each value once in the wave,
// and passes them on to the other three lanes of the channel through LDS that no other wave touches.  What a lane sums over its own states of the
// tokens 4 m .. 4 m + 3 is added up over q by swaps of lane rows that leave token 4 m + q with q (of_rows).
#pragma once
#include "common.h"
#include "launch.h"

#include <algorithm>
#include <type_traits>

namespace vig {

int launch_selective_join(const SelScanArgs& p, int np, bool back, hipStream_t stream);

namespace {

typedef __amdgpu_buffer_rsrc_t rsrc_t;
constexpr unsigned kNowhere = 0x40000000u;  // byte offset behind every descriptor here (sixteen rows of kScanRow elements at most)
constexpr int kScanWaves = 4;               // of a workgroup, on channels side by side
constexpr int kScanBlock = 16 * kScanWaves; // channels of a workgroup
constexpr int kScanUnits = 256;             // compute units that they fill

// tokens of a tile (the backward keeps two numbers a state and token in registers: 128 of them at most)
constexpr int scan_tile(int CN) { return CN <= 4 ? 16 : 64 / CN; }
template <int CN> constexpr int kTileTokens = scan_tile(CN);
// states of a lane: a quarter of N, as a power of two
inline int scan_states(int N) {
  int CN = 1;
  while (4 * CN < N) CN *= 2;
  return CN;
}
template <typename F> int by_states(int CN, F f) {
  switch (CN) {
    case 1: return f(std::integral_constant<int, 1>{});
    case 2: return f(std::integral_constant<int, 2>{});
    case 4: return f(std::integral_constant<int, 4>{});
    case 8: return f(std::integral_constant<int, 8>{});
    default: return f(std::integral_constant<int, 16>{});
  }
}
// Groups of channels from which on sequences go through whole.  Chunks cost a second walk without the outputs and whole tiles; what they give is four workgroups a compute unit, whose waves hide
// one another's waits, the more the fewer states a lane has to work on and the fewer waves there are else (the backward's).  Time of cut to whole sequences at 168, 192, 216, 252, 288, 336, 384
// groups:  196 tokens, 16 states, forward 1.05 1.03 1.27 1.28 1.08 1.27 1.31, with the backward .91 .90 1.08 1.15 1.00 1.13 1.21;   4 states .89 .89 1.05 1.04 .98 1.07 1.13, .83 .84 .97 1.02 .91 1.02 1.03.
// 1024 tokens, 4 states, forward .48 .54 .64 .65 .74 .79 .96;  16: .67 .76 .91 .91 .97 1.02 1.16;  64: .74 .88 1.07 1.07 1.04 1.05 1.21;  with the backward .54 .60 .70 .70 .77 .84 .94,
// .62 .70 .84 .86 .88 .94 1.09, .63 .72 .85 .88 .89 .91 1.14.  (320 to 4096 tokens: alike.)  64 tokens, 144 and 192 groups, 4, 16, 64 states: forward 1.10 1.10, 1.23 1.23, 1.39 1.44.
inline int whole_from(const SelScanArgs& p, bool back) {
  const int CN = scan_states(p.N);
  if (p.L < 256) return p.L < 128 ? 128 : 200;
  return back || CN <= 2 ? 352 : CN <= 4 ? 300 : 200;
}
// Chunks of tokens, 16 at least.  65536 x 1024, 16 states, fold and walk: four workgroups a unit 229 + 305 us, two 248 + 367, one 331 + 536.
inline void cut_chunks(SelScanArgs& p, bool back) {
  p.of_group = p.D / p.G, p.blocks = (p.of_group + kScanBlock - 1) / kScanBlock;
  const long long groups = (long long)p.batch * p.G * p.blocks;
  const long long want = groups >= whole_from(p, back) ? 1 : std::min<long long>(4 * kScanUnits / groups, (p.L + 15) / 16);
  const int T = scan_tile(scan_states(p.N));
  p.chunk = (int)(((p.L + want - 1) / want + T - 1) / T * T);
  p.chunks = (p.L + p.chunk - 1) / p.chunk;
}
// workgroups of the sum of dB and dC, of four numbers a thread
inline long long shared_groups(const SelScanArgs& p) { return ((long long)p.batch * p.G * p.L * 2 * scan_states(p.N) + 255) / 256; }
// Whether every launch stays below 2^32 threads: the walk's (and the folding's), and in training the sum of dB and dC over the workgroups.  (Chunks that take a launch to be joined, more than 32
// of them, are those of fewer than 32 workgroups' channels: 500 workgroups.)
inline bool scan_fits(const SelScanArgs& p, bool training) {
  const long long most = 0xffffffLL;
  return (long long)p.batch * p.G * p.blocks * p.chunks <= most && (!training || shared_groups(p) <= most);
}
// Few chunks are joined by those who come behind them (entering), many by a launch of their own: each reads all in front of it, 68 bytes a channel of 16 states.
constexpr int kFewChunks = 32;
inline unsigned scan_grid(const SelScanArgs& p) { return (unsigned)((long long)p.batch * p.G * p.blocks * p.chunks); }
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// An element as stored, and its value: rows that are loaded ahead stay as they came, since whatever is done to them there would wait for them
template <typename S> using Raw = std::conditional_t<sizeof(S) == 2, uint16_t, uint32_t>;
__device__ __forceinline__ uint32_t load1(rsrc_t r, unsigned off, float) { return __builtin_amdgcn_raw_buffer_load_b32(r, off, 0, 0); }
__device__ __forceinline__ uint16_t load1(rsrc_t r, unsigned off, uint16_t) { return __builtin_amdgcn_raw_buffer_load_b16(r, off, 0, 0); }
__device__ __forceinline__ float value(uint16_t raw) { return bf16_to_f32(raw); }
__device__ __forceinline__ float value(uint32_t raw) { return __uint_as_float(raw); }
__device__ __forceinline__ void store1(rsrc_t r, unsigned off, float v, float) { __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(v), r, off, 0, 0); }
__device__ __forceinline__ void store1(rsrc_t r, unsigned off, float v, uint16_t) { __builtin_amdgcn_raw_buffer_store_b16(f32_to_bf16(v), r, off, 0, 0); }

// Where a wave stands.
struct Stand {
  int b, g, block, chunk;
  int wave, q, j, c;  // c: channel
  bool has;
  int first, end;     // tokens of the chunk
  __device__ __forceinline__ Stand(const SelScanArgs& p) {
    // (workgroups go round the eight XCDs: each takes a stretch of neighbours, which share lines and the rows of B and C)
    const unsigned each = gridDim.x / 8;
    unsigned id = blockIdx.x;
    if (id < 8 * each) id = id % 8 * each + id / 8;
    block = (int)(id % (unsigned)p.blocks), id /= (unsigned)p.blocks;
    g = (int)(id % (unsigned)p.G), id /= (unsigned)p.G;
    chunk = (int)(id % (unsigned)p.chunks), b = (int)(id / (unsigned)p.chunks);
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), q = (threadIdx.x >> 4) & 3, j = threadIdx.x & 15;
    const int in = block * kScanBlock + wave * 16 + j;
    has = in < p.of_group;
    c = g * p.of_group + in;
    first = chunk * p.chunk, end = min(first + p.chunk, p.L);
  }
};

// A tile of tokens from token `first` of the walk on, as many of them as lie in front of `end` (one at least).  A tensor's descriptor begins at the lowest of their rows in memory and ends
// behind the highest, so that lanes without a token, whose offsets lie outside, read zeros and store nothing.
template <int T> struct Tile {
  int rows, from, step;  // the row of memory of token k lies from + step k rows behind the lowest
  long long lowest;
  __device__ __forceinline__ Tile(const SelScanArgs& p, int first, int end) {
    rows = min(end - first, T);
    lowest = p.reverse ? (long long)p.L - first - rows : first;
    from = p.reverse ? rows - 1 : 0, step = p.reverse ? -1 : 1;
  }
};
// A tensor's rows as a lane reads or writes them, one element each
template <typename S> struct Line {
  const char* at;
  unsigned pitch, offset;  // bytes; offset: the lane's, from its row of lanes' first token
  // column: the lane's element of a row, or none
  __device__ __forceinline__ void stand(const SelScanArgs& p, const void* base, long long before, long long l, int q, int column, bool has) {
    at = static_cast<const char*>(base) + before * (long long)sizeof(S);
    pitch = (unsigned)l * sizeof(S);
    offset = has ? column * sizeof(S) + (p.reverse ? 0u - q * pitch : q * pitch) : kNowhere;
  }
  template <int T> __device__ __forceinline__ rsrc_t of(const Tile<T>& t) const {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(at) + t.lowest * pitch, 0, (int)(t.rows * pitch), 0x00020000);
  }
  // token 4 m + q of the tile
  template <int T> __device__ __forceinline__ unsigned place(const Tile<T>& t, int m) const { return offset + (unsigned)(t.from + t.step * 4 * m) * pitch; }
  template <int T> __device__ __forceinline__ Raw<S> load(rsrc_t r, const Tile<T>& t, int m) const { return load1(r, place(t, m), S{}); }
  template <int T> __device__ __forceinline__ void store(const Tile<T>& t, int m, float v) const { store1(of(t), place(t, m), v, S{}); }
};

// log(1 + e), e in [0, 1]: the logarithm of the rounded sum, and what the sum has lost (whose factor 1 / (1 + e) is within a unit of the result).  Over all such floats 3.5 units of 2^-24
// of itself at most, in 6 instructions (a series in e / (2 + e): 13).
__device__ __forceinline__ float log1p_01(float e) {
  const float w = 1.f + e;
  return fmaf(__builtin_amdgcn_logf(w), kLn2, e - (w - 1.f));
}
// the step of a token from what its projection gives (with the bias), and its derivative
__device__ __forceinline__ float step_of(float raw, int softplus) {
  const float soft = fmaxf(raw, 0.f) + log1p_01(exp_fast(-fabsf(raw)));
  return softplus ? soft : raw;
}
__device__ __forceinline__ float dstep_of(float raw, int softplus) {
  const float e = exp_fast(-fabsf(raw)), soft = (raw >= 0.f ? 1.f : e) * __builtin_amdgcn_rcpf(1.f + e);
  return softplus ? soft : 1.f;
}

// sums over the four lane rows of four tokens' values: the row q is left with token q's
__device__ __forceinline__ float of_rows(float s0, float s1, float s2, float s3) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(s0), __float_as_uint(s2), false, false);
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(s1), __float_as_uint(s3), false, false);
  const float even = __uint_as_float(a[0]) + __uint_as_float(a[1]), odd = __uint_as_float(b[0]) + __uint_as_float(b[1]);
  const auto c = __builtin_amdgcn_permlane16_swap(__float_as_uint(even), __float_as_uint(odd), false, false);
  return __uint_as_float(c[0]) + __uint_as_float(c[1]);
}
// the sum over the four lane rows, in all of them
__device__ __forceinline__ float of_all_rows(float s) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(s), __float_as_uint(s), false, false);
  s = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(s), __float_as_uint(s), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// A wave's LDS: of a tile four numbers of each token and channel side by side, each token's B and C.
template <int CN> struct Pass {
  static constexpr int T = kTileTokens<CN>;
  f32x4_t of_channel[T][16];
  float of_token[2][T][4 * CN];
};
// what other lanes of the wave wrote is read behind this
__device__ __forceinline__ void passed() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}
template <int N> __device__ __forceinline__ void read_lds(float (&v)[N], const float* from) {
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const f32x4_t w = *reinterpret_cast<const f32x4_t*>(from + i);
      v[i] = w[0], v[i + 1] = w[1], v[i + 2] = w[2], v[i + 3] = w[3];
    }
  } else if constexpr (N == 2) {
    const f32x2_t w = *reinterpret_cast<const f32x2_t*>(from);
    v[0] = w[0], v[1] = w[1];
  } else {
    v[0] = *from;
  }
}

// A lane's states in memory, [.., D, stride] with `stride` numbers a channel of which `n` are there
template <int CN> __device__ __forceinline__ void load_states(float (&h)[CN], const float* base, size_t row, int D, int stride, int n, const Stand& at) {
#pragma unroll
  for (int i = 0; i < CN; ++i) h[i] = base && at.has && at.q * CN + i < n ? base[(row * D + at.c) * stride + at.q * CN + i] : 0.f;
}
template <int CN> __device__ __forceinline__ void store_states(float* base, const float (&h)[CN], size_t row, int D, int stride, int n, const Stand& at) {
  if (!at.has) return;
#pragma unroll
  for (int i = 0; i < CN; ++i)
    if (at.q * CN + i < n) base[(row * D + at.c) * stride + at.q * CN + i] = h[i];
}
// ... of rows of 4 CN numbers, all of them there, on 16-byte boundaries
template <int CN> struct Kept {
  unsigned offset;
  __device__ __forceinline__ explicit Kept(const Stand& at) : offset(at.has ? (at.c * 4 + at.q) * CN * (unsigned)sizeof(float) : kNowhere) {}
  static __device__ __forceinline__ rsrc_t of(const float* base, size_t row, int D) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(base) + row * (unsigned)(D * 4 * CN), 0, D * 4 * CN * (int)sizeof(float), 0x00020000);
  }
  __device__ __forceinline__ void store(float* base, size_t row, int D, const float (&h)[CN]) const {
    const rsrc_t r = of(base, row, D);
    if constexpr (CN >= 4) {
#pragma unroll
      for (int i = 0; i < CN; i += 4)
        __builtin_amdgcn_raw_buffer_store_b128(u32x4_t{__float_as_uint(h[i]), __float_as_uint(h[i + 1]), __float_as_uint(h[i + 2]), __float_as_uint(h[i + 3])}, r, offset + 4 * i, 0, 0);
    } else {
#pragma unroll
      for (int i = 0; i < CN; ++i) __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(h[i]), r, offset + 4 * i, 0, 0);
    }
  }
  __device__ __forceinline__ void load(float (&h)[CN], const float* base, size_t row, int D) const {
    const rsrc_t r = of(base, row, D);
    if constexpr (CN >= 4) {
#pragma unroll
      for (int i = 0; i < CN; i += 4) {
        const u32x4_t w = __builtin_amdgcn_raw_buffer_load_b128(r, offset + 4 * i, 0, 0);
#pragma unroll
        for (int k = 0; k < 4; ++k) h[i + k] = __uint_as_float(w[k]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < CN; ++i) h[i] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(r, offset + 4 * i, 0, 0));
    }
  }
};

// What enters a chunk from the chunks in front of it (BACK: behind it), whose ends and sums of steps a launch before has left: h, what enters the first of them, moved on
template <bool BACK, int CN> __device__ __forceinline__ void entering(float (&h)[CN], const float (&A)[CN], const SelScanArgs& p, const Stand& at) {
  constexpr int K = CN <= 4 ? 8 : 4;  // on their way together
  const Kept<CN> kept(at);
  if (!at.has) return;
  const int count = BACK ? p.chunks - 1 - at.chunk : at.chunk;
  for (int k0 = 0; k0 < count; k0 += K) {
    float leaves[K][CN], sum[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int i = min(k0 + k, count - 1);
      const size_t row = (size_t)at.b * p.chunks + (BACK ? p.chunks - 1 - i : i);
      kept.load(leaves[k], p.ends, row, p.D);
      sum[k] = p.sums[row * p.D + at.c];
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (k0 + k >= count) break;
#pragma unroll
      for (int i = 0; i < CN; ++i) h[i] = fmaf(__builtin_amdgcn_exp2f(A[i] * sum[k]), h[i], leaves[k][i]);
    }
  }
}

// Zeros for a last tile's tokens that are not there: steps of 0 leave the state as it is
template <int R> __device__ __forceinline__ void leave_out(float (&v)[R], int rows, const Stand& at) {
#pragma unroll
  for (int m = 0; m < R; ++m) v[m] = 4 * m + at.q < rows ? v[m] : 0.f;
}

// Numbers of B or C of a tile as loaded: token 4 m + q, states j, j + 16, ...
template <typename S, int CN> struct Shared {
  static constexpr int T = kTileTokens<CN>, R = T / 4, NP = 4 * CN, E = NP > 16 ? NP / 16 : 1;
  Line<S> line[E];
  Raw<S> v[R][E];
  __device__ __forceinline__ void stand(const SelScanArgs& p, const Rows& t, const Stand& at) {
#pragma unroll
    for (int e = 0; e < E; ++e) line[e].stand(p, t.at, at.b * t.b + at.g * t.g, t.l, at.q, at.j + 16 * e, at.j + 16 * e < p.N);
  }
  __device__ __forceinline__ void load(const Tile<T>& t) {
    const rsrc_t r = line[0].of(t);
#pragma unroll
    for (int m = 0; m < R; ++m)
#pragma unroll
      for (int e = 0; e < E; ++e) v[m][e] = line[e].load(r, t, m);
  }
  __device__ __forceinline__ void pass(float (&to)[T][NP], const Stand& at) const {
#pragma unroll
    for (int m = 0; m < R; ++m)
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (NP >= 16 || at.j < NP) to[4 * m + at.q][at.j + 16 * e] = value(v[m][e]);
  }
};
// Values of a tile's rows of channels as loaded: token 4 m + q of channel j
template <typename S, int T> struct Channels {
  Line<S> line;
  Raw<S> v[T / 4];
  __device__ __forceinline__ float operator[](int m) const { return value(v[m]); }
  __device__ __forceinline__ void stand(const SelScanArgs& p, const Rows& t, const Stand& at) { line.stand(p, t.at, at.b * t.b, t.l, at.q, at.c, at.has); }
  __device__ __forceinline__ void load(const Tile<T>& t) {
    const rsrc_t r = line.of(t);
#pragma unroll
    for (int m = 0; m < T / 4; ++m) v[m] = line.load(r, t, m);
  }
};
// a dense tensor's
template <typename S> __device__ __forceinline__ Line<S> dense_line(const SelScanArgs& p, void* base, const Stand& at) {
  Line<S> line;
  line.stand(p, base, (long long)at.b * p.L * p.D, p.D, at.q, at.c, at.has);
  return line;
}

}  // namespace
}  // namespace vig
