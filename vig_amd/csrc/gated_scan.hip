// The gated linear recurrence of a vector state, forward and backward, and its step for one token.
//
//   h_t = e^{g_t} h_{t-1} + x_t,      o_t = h_t                        (causal; h_{-1} = initial state or 0)
//   o_t = s (h_t + h'_t),  h'_t = e^{g'_t} h'_{t+1} + x_t              (both directions)
//
// What a run of tokens does to the state that enters it is an affine map per channel, h -> A h + S, and maps compose in any grouping:
//   (A, S) then (A', S')  =  (A A', A' S + S').
// A thread folds the eight tokens that it holds in registers, a wave its four threads of a channel by swaps of lane rows, a workgroup its waves through
// LDS; then every thread knows the state that enters its tokens and walks them once more, which costs one fused multiply-add a value.  Memory is what
// bounds it: rows and gates are read once.  Sequences that one workgroup does not hold are cut in chunks: a first launch folds the chunks
// (reads everything once, writes 8 bytes a chunk and channel), the second folds the chunks in front of its own and walks.
//
// Backward: dh_t = do_t + e^{g_{t+1}} dh_{t+1}; with D_t = e^{g_t} dh_t, what token t hands back, the walk against the direction is D -> e^{g_t} (do_t + D), an
// affine map again, and dx_t = dh_t, dg_t = dh_t u_t with u_t = e^{g_t} h_{t-1} from the walk along it, recomputed in 32 bits from x and g (the stored
// output is rounded, and for both directions holds their sum).
//
// Measured, bf16 (a large copy: 5.3 TB/s of reads and writes).  One workgroup a sequence, 128 x 196 x 384: both directions 14.8 us, 5.2 TB/s, with the last calls' tensors in the
// 256 MB cache, 21.7 and 3.6 past it, causal 13.5 past it, 4.3, gradients of both 33 to 36, 4.3 to 4.7, where the arithmetic of four maps begins to count.  Chunks, 65536 x 1024: folding 63 us, 4.2 TB/s (loads alone in this pattern of 64-byte rows 53, in rows of 128
// bytes 48; with the next rows on their way during the arithmetic no less, and more registers a thread, 143 to 158 us for both launches), walking 82, 4.9; fp32, 4 x 2305 x 333: 7 and 10,
// gradients 10 and 15, of 420 workgroups each.
#include "common.h"
#include "launch.h"
#include <algorithm>
#include <type_traits>

namespace vig {
namespace {

typedef __amdgpu_buffer_rsrc_t rsrc_t;
constexpr unsigned kBeyond = 0x40000000u;  // byte offset that no descriptor here covers (kScanRow)
constexpr int kTokens = 8;                 // of a thread, where a comment does not say otherwise
constexpr int kLanes = 16;                 // that take a token's channels
constexpr int kRuns = 64 / kLanes;         // of tokens in a wave
constexpr int kMaxWaves = 16;
constexpr unsigned kMostThreads = 0xffffff00u;  // of a launch

// N consecutive channels of one token as stored
template <typename T, int N> struct Piece;
template <> struct Piece<uint16_t, 2> {
  uint32_t v;
  __device__ __forceinline__ void load(rsrc_t r, unsigned off) { v = __builtin_amdgcn_raw_buffer_load_b32(r, off, 0, 0); }
  __device__ __forceinline__ float get(int i) const { return i ? bf16hi_to_f32(v) : bf16lo_to_f32(v); }
  static __device__ __forceinline__ void store(rsrc_t r, unsigned off, const float (&x)[2]) { __builtin_amdgcn_raw_buffer_store_b32(pack_bf16x2(x[0], x[1]), r, off, 0, 0); }
};
template <> struct Piece<float, 2> {
  u32x2_t v;
  __device__ __forceinline__ void load(rsrc_t r, unsigned off) { v = __builtin_amdgcn_raw_buffer_load_b64(r, off, 0, 0); }
  __device__ __forceinline__ float get(int i) const { return __uint_as_float(v[i]); }
  static __device__ __forceinline__ void store(rsrc_t r, unsigned off, const float (&x)[2]) {
    __builtin_amdgcn_raw_buffer_store_b64(u32x2_t{__float_as_uint(x[0]), __float_as_uint(x[1])}, r, off, 0, 0);
  }
};
template <> struct Piece<uint16_t, 1> {
  uint16_t v;
  __device__ __forceinline__ void load(rsrc_t r, unsigned off) { v = __builtin_amdgcn_raw_buffer_load_b16(r, off, 0, 0); }
  __device__ __forceinline__ float get(int) const { return bf16_to_f32(v); }
  static __device__ __forceinline__ void store(rsrc_t r, unsigned off, const float (&x)[1]) {
    __builtin_amdgcn_raw_buffer_store_b16(f32_to_bf16(x[0]), r, off, 0, 0);
  }
};
template <> struct Piece<float, 1> {
  uint32_t v;
  __device__ __forceinline__ void load(rsrc_t r, unsigned off) { v = __builtin_amdgcn_raw_buffer_load_b32(r, off, 0, 0); }
  __device__ __forceinline__ float get(int) const { return __uint_as_float(v); }
  static __device__ __forceinline__ void store(rsrc_t r, unsigned off, const float (&x)[1]) {
    __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(x[0]), r, off, 0, 0);
  }
};

// h -> a h + s for each of a thread's channels
template <int N> struct Map {
  float a[N], s[N];
  __device__ __forceinline__ void identity() {
#pragma unroll
    for (int i = 0; i < N; ++i) a[i] = 1.f, s[i] = 0.f;
  }
  // this one behind `first`
  __device__ __forceinline__ void behind(const Map& first) {
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] = fmaf(a[i], first.s[i], s[i]), a[i] *= first.a[i];
  }
  __device__ __forceinline__ void apply(float (&h)[N]) const {
#pragma unroll
    for (int i = 0; i < N; ++i) h[i] = fmaf(a[i], h[i], s[i]);
  }
};

// Where a thread stands: sixteen lanes side by side take a token's channels, the wave's four rows of lanes four runs of tokens behind one another.
struct Place {
  int wave, waves, lane, run, lc;  // lc: lane of the token's channels
  __device__ __forceinline__ Place()
      : wave(__builtin_amdgcn_readfirstlane(threadIdx.x >> 6)), waves(blockDim.x >> 6), lane(threadIdx.x & 63), run((threadIdx.x & 63) / kLanes), lc(threadIdx.x % kLanes) {}
};

// LDS of one direction: each wave's map of a channel; `waves` of them, as many as the workgroup has
template <int N> struct Board {
  float (*v)[kLanes][2 * N];
  static constexpr size_t kBytes = sizeof(float) * kLanes * 2 * N;  // of a wave
};

template <int N, int DIRS> struct Boards {
  char* at;
  int waves;
  __device__ __forceinline__ Boards(char* at, int waves) : at(at), waves(waves) {}
  __device__ __forceinline__ Board<N> operator[](int dir) const { return {reinterpret_cast<float (*)[kLanes][2 * N]>(at + dir * waves * Board<N>::kBytes)}; }
};

// A map's values in the lower and the upper of each two rows of lanes (HALVES: of the wave's halves), in both of them
template <bool HALVES, int N>
__device__ __forceinline__ void both_of(const Map<N>& m, Map<N>& low, Map<N>& high) {
  auto swap = [](float x, float& l, float& h) {
    const unsigned v = __float_as_uint(x);
    const auto r = HALVES ? __builtin_amdgcn_permlane32_swap(v, v, false, false) : __builtin_amdgcn_permlane16_swap(v, v, false, false);
    l = __uint_as_float(r[0]), h = __uint_as_float(r[1]);
  };
#pragma unroll
  for (int i = 0; i < N; ++i) swap(m.a[i], low.a[i], high.a[i]), swap(m.s[i], low.s[i], high.s[i]);
}

// Folds the threads' maps along a wave.  UP: tokens in their order; else against it.  Leaves in `m` the map of what lies in front of this
// thread in its wave, and the whole wave's on the board.
template <bool UP, int N>
__device__ __forceinline__ void fold_wave(Map<N>& m, const Place& at, const Board<N>& board) {
  Map<N> low, high, first, second;
  both_of<false>(m, low, high);
  const bool behind = UP ? at.run & 1 : !(at.run & 1), last = UP ? at.run >= 2 : at.run < 2;
#pragma unroll
  for (int i = 0; i < N; ++i) m.a[i] = behind ? (UP ? low : high).a[i] : 1.f, m.s[i] = behind ? (UP ? low : high).s[i] : 0.f;
  if (UP) high.behind(low);
  else low.behind(high);
  both_of<true>(UP ? high : low, first, second);  // (the halves' maps)
  if (!UP) {
    const Map<N> t = first;
    first = second, second = t;
  }
  if (last) m.behind(first);
  second.behind(first);
  if (at.lane < kLanes) {
    float* to = board.v[at.wave][at.lc];
#pragma unroll
    for (int i = 0; i < N; ++i) to[2 * i] = second.a[i], to[2 * i + 1] = second.s[i];
  }
}
// (behind the barrier) h: state that enters the workgroup -> the one that enters this thread's tokens
template <bool UP, int N>
__device__ __forceinline__ void enter(float (&h)[N], const Map<N>& m, const Place& at, const Board<N>& board) {
  for (int w = UP ? 0 : at.waves - 1; w != at.wave; w += UP ? 1 : -1) {
    const float* from = board.v[w][at.lc];
#pragma unroll
    for (int i = 0; i < N; ++i) h[i] = fmaf(from[2 * i], h[i], from[2 * i + 1]);
  }
  m.apply(h);
}
// (behind the barrier) the map of the whole workgroup
template <bool UP, int N>
__device__ __forceinline__ Map<N> whole(const Place& at, const Board<N>& board) {
  Map<N> t;
  t.identity();
  for (int k = 0; k < at.waves; ++k) {
    const float* from = board.v[UP ? k : at.waves - 1 - k][at.lc];
#pragma unroll
    for (int i = 0; i < N; ++i) t.s[i] = fmaf(from[2 * i], t.s[i], from[2 * i + 1]), t.a[i] *= from[2 * i];
  }
  return t;
}

struct ScanArgs {
  const void *x, *g[2], *d_o;  // d_o: dense, like the outputs
  void *o, *dx, *dg[2];
  const float *h0, *dhT;
  float *hT, *dh0;
  float* maps;  // [B, directions, chunks, D, 2]; directions: gates 0 along, gates 0 against (backward), gates 1 against, gates 1 along (backward)
  long long xb, xl, gb, gl;  // strides of batch element and token, in elements
  int L, D, groups, chunks, chunk;
  float scale;
};

// The workgroup's piece of the tensors.  Workgroups go round the eight XCDs: each of them takes a stretch of neighbouring pieces, so that the halves of a
// 128-byte line are met in one L2.
struct Tile {
  int b, ch, cg, t0, rows;
  __device__ __forceinline__ Tile(const ScanArgs& p, bool fold) {
    const unsigned each = gridDim.x / 8;
    unsigned id = blockIdx.x;
    if (id < 8 * each) id = id % 8 * each + id / 8;
    if (!fold && p.chunks > 1) id = gridDim.x - 1 - id;
    const unsigned q = id / (unsigned)p.groups;
    cg = (int)(id - q * p.groups);
    b = (int)(q / (unsigned)p.chunks);
    ch = (int)(q - (unsigned)b * p.chunks);
    t0 = ch * p.chunk;
    rows = min(p.chunk, p.L - t0);
  }
  template <typename T>
  __device__ __forceinline__ rsrc_t rows_of(const void* base, long long sb, long long sl) const {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(static_cast<const T*>(base)) + b * sb + t0 * sl, 0, (int)(rows * sl * (long long)sizeof(T)), 0x00020000);
  }
};

// gates as the factors they stand for; tokens behind the sequence read as gates of 0 and rows of 0, the map that changes nothing
template <typename T, int N, int TOKENS>
__device__ __forceinline__ void factors(const Piece<T, N> (&raw)[TOKENS], float (&a)[TOKENS][N]) {
#pragma unroll
  for (int t = 0; t < TOKENS; ++t)
#pragma unroll
    for (int i = 0; i < N; ++i) a[t][i] = exp_fast(raw[t].get(i));
}
template <typename T, int N, int TOKENS>
__device__ __forceinline__ void load_run(Piece<T, N> (&raw)[TOKENS], rsrc_t r, unsigned first, unsigned pitch) {
#pragma unroll
  for (int t = 0; t < TOKENS; ++t) raw[t].load(r, first + t * pitch);
}

// A thread's map along its tokens, h -> a h + x
template <bool UP, typename T, int N, int TOKENS>
__device__ __forceinline__ Map<N> fold_run(const float (&a)[TOKENS][N], const Piece<T, N> (&x)[TOKENS]) {
  Map<N> m;
  m.identity();
#pragma unroll
  for (int k = 0; k < TOKENS; ++k) {
    const int t = UP ? k : TOKENS - 1 - k;
#pragma unroll
    for (int i = 0; i < N; ++i) m.s[i] = fmaf(a[t][i], m.s[i], x[t].get(i)), m.a[i] *= a[t][i];
  }
  return m;
}
// ... and the gradient's against them, h -> a (h + scale y), whose factor is the same
template <bool UP, typename T, int N, int TOKENS>
__device__ __forceinline__ Map<N> fold_back(const float (&a)[TOKENS][N], const Piece<T, N> (&y)[TOKENS], float scale, const Map<N>& along) {
  Map<N> m;
#pragma unroll
  for (int i = 0; i < N; ++i) m.a[i] = along.a[i], m.s[i] = 0.f;
#pragma unroll
  for (int k = 0; k < TOKENS; ++k) {
    const int t = UP ? k : TOKENS - 1 - k;
#pragma unroll
    for (int i = 0; i < N; ++i) m.s[i] = a[t][i] * fmaf(scale, y[t].get(i), m.s[i]);
  }
  return m;
}

// The state that enters this workgroup's chunk from the chunks in front of it: each of the workgroup's runs folds a
// stretch of them, and the runs fold as tokens do.
template <bool UP, int N>
__device__ __forceinline__ Map<N> fold_chunks(const ScanArgs& p, const Tile& tile, const Place& at, int dir, int dirs, int c, bool has) {
  const int n = UP ? tile.ch : p.chunks - 1 - tile.ch;  // chunks in front
  const int runs = at.waves * kRuns, each = (n + runs - 1) / runs;
  const int slot = at.wave * kRuns + at.run;
  // (runs in the order of the tokens; against it the last run comes first)
  const int first = UP ? slot * each : tile.ch + 1 + slot * each, end = min(first + each, UP ? n : p.chunks);
  const float* from = p.maps + (((size_t)tile.b * dirs + dir) * p.chunks) * p.D * 2;
  Map<N> m;
  m.identity();
  for (int k = 0; k < each; ++k) {
    const int j = UP ? first + k : end - 1 - k;
    if (j < first || j >= end || !has) continue;
    const float* v = from + ((size_t)j * p.D + c) * 2;
    if constexpr (N == 2) {
      const f32x4_t w = *reinterpret_cast<const f32x4_t*>(v);
#pragma unroll
      for (int i = 0; i < N; ++i) m.s[i] = fmaf(w[2 * i], m.s[i], w[2 * i + 1]), m.a[i] *= w[2 * i];
    } else {
      m.s[0] = fmaf(v[0], m.s[0], v[1]), m.a[0] *= v[0];
    }
  }
  return m;
}
template <int N>
__device__ __forceinline__ void store_map(const ScanArgs& p, const Tile& tile, int dir, int dirs, int c, const Map<N>& m) {
  float* v = p.maps + ((((size_t)tile.b * dirs + dir) * p.chunks + tile.ch) * p.D + c) * 2;
#pragma unroll
  for (int i = 0; i < N; ++i) v[2 * i] = m.a[i], v[2 * i + 1] = m.s[i];
}
template <int N>
__device__ __forceinline__ void load_state(float (&h)[N], const float* from, const ScanArgs& p, int b, int c, bool has) {
#pragma unroll
  for (int i = 0; i < N; ++i) h[i] = from && has ? from[(size_t)b * p.D + c + i] : 0.f;
}
template <int N>
__device__ __forceinline__ void store_state(float* to, const float (&h)[N], const ScanArgs& p, int b, int c) {
#pragma unroll
  for (int i = 0; i < N; ++i) to[(size_t)b * p.D + c + i] = h[i];
}

// ---- forward.  FOLD: only the chunks' maps

template <typename TX, typename TG, bool BOTH, bool FOLD, int N, int TOKENS>
__global__ __launch_bounds__(64 * kMaxWaves) void gated_scan_kernel(ScanArgs p) {
  constexpr int dirs = BOTH ? 2 : 1;
  extern __shared__ __align__(16) char lds[];
  const Place at;
  const Boards<N, dirs> board(lds, at.waves), front(lds + dirs * at.waves * Board<N>::kBytes, at.waves);
  const Tile tile(p, FOLD);
  const int c = (tile.cg * kLanes + at.lc) * N;
  const bool has = c < p.D;
  const int first = (at.wave * kRuns + at.run) * TOKENS;
  auto offset = [&](long long sl, int size) { return has ? (unsigned)((first * sl + c) * size) : kBeyond; };
  Piece<TX, N> x[TOKENS];
  Piece<TG, N> raw[TOKENS];
  float a[TOKENS][N], a2[BOTH ? TOKENS : 1][N];
  load_run(raw, tile.rows_of<TG>(p.g[0], p.gb, p.gl), offset(p.gl, sizeof(TG)), (unsigned)(p.gl * sizeof(TG)));
  load_run(x, tile.rows_of<TX>(p.x, p.xb, p.xl), offset(p.xl, sizeof(TX)), (unsigned)(p.xl * sizeof(TX)));
  [[maybe_unused]] Piece<TG, N> raw2[BOTH ? TOKENS : 1];
  if constexpr (BOTH) load_run(raw2, tile.rows_of<TG>(p.g[1], p.gb, p.gl), offset(p.gl, sizeof(TG)), (unsigned)(p.gl * sizeof(TG)));
  [[maybe_unused]] Map<N> before, after;
  if constexpr (!FOLD) {
    if (p.chunks > 1) {
      before = fold_chunks<true, N>(p, tile, at, 0, dirs, c, has);
      fold_wave<true, N>(before, at, front[0]);
      if constexpr (BOTH) {
        after = fold_chunks<false, N>(p, tile, at, 1, dirs, c, has);
        fold_wave<false, N>(after, at, front[1]);
      }
    }
  }
  factors(raw, a);
  Map<N> m = fold_run<true>(a, x), m2;
  fold_wave<true, N>(m, at, board[0]);
  if constexpr (BOTH) {
    factors(raw2, a2);
    m2 = fold_run<false>(a2, x);
    fold_wave<false, N>(m2, at, board[1]);
  }
  __syncthreads();
  if constexpr (FOLD) {
    if (at.wave == 0 && at.run == 0 && has) {
      store_map(p, tile, 0, dirs, c, whole<true, N>(at, board[0]));
      if constexpr (BOTH) store_map(p, tile, 1, dirs, c, whole<false, N>(at, board[1]));
    }
    return;
  }
  float h[N], y[TOKENS][N];
  load_state(h, p.h0, p, tile.b, c, has);
  if (p.chunks > 1) whole<true, N>(at, front[0]).apply(h);
  enter<true, N>(h, m, at, board[0]);
#pragma unroll
  for (int t = 0; t < TOKENS; ++t)
#pragma unroll
    for (int i = 0; i < N; ++i) y[t][i] = h[i] = fmaf(a[t][i], h[i], x[t].get(i));
  // (tokens behind the sequence change nothing: the last run ends with the state behind its last token)
  if (p.hT && tile.ch == p.chunks - 1 && at.wave == at.waves - 1 && at.run == kRuns - 1 && has) store_state(p.hT, h, p, tile.b, c);
  if constexpr (BOTH) {
    float r[N];
#pragma unroll
    for (int i = 0; i < N; ++i) r[i] = 0.f;
    if (p.chunks > 1) whole<false, N>(at, front[1]).apply(r);
    enter<false, N>(r, m2, at, board[1]);
#pragma unroll
    for (int t = TOKENS - 1; t >= 0; --t)
#pragma unroll
      for (int i = 0; i < N; ++i) r[i] = fmaf(a2[t][i], r[i], x[t].get(i)), y[t][i] += r[i];
  }
  const rsrc_t out = tile.rows_of<TX>(p.o, (long long)p.L * p.D, p.D);
  const unsigned to = offset(p.D, sizeof(TX));
#pragma unroll
  for (int t = 0; t < TOKENS; ++t) {
#pragma unroll
    for (int i = 0; i < N; ++i) y[t][i] *= p.scale;
    Piece<TX, N>::store(out, to + t * (unsigned)(p.D * sizeof(TX)), y[t]);
  }
}

// ---- backward

template <typename TX, typename TG, bool BOTH, bool FOLD, int N, int TOKENS>
__global__ __launch_bounds__(64 * kMaxWaves) void gated_scan_bwd_kernel(ScanArgs p) {
  constexpr int dirs = BOTH ? 4 : 2;
  extern __shared__ __align__(16) char lds[];
  const Place at;
  const Boards<N, dirs> board(lds, at.waves), front(lds + dirs * at.waves * Board<N>::kBytes, at.waves);
  const Tile tile(p, FOLD);
  const int c = (tile.cg * kLanes + at.lc) * N;
  const bool has = c < p.D;
  const int first = (at.wave * kRuns + at.run) * TOKENS;
  auto offset = [&](long long sl, int size) { return has ? (unsigned)((first * sl + c) * size) : kBeyond; };
  const long long dense = (long long)p.L * p.D;
  Piece<TX, N> x[TOKENS], dy[TOKENS];
  load_run(x, tile.rows_of<TX>(p.x, p.xb, p.xl), offset(p.xl, sizeof(TX)), (unsigned)(p.xl * sizeof(TX)));
  load_run(dy, tile.rows_of<TX>(p.d_o, dense, p.D), offset(p.D, sizeof(TX)), (unsigned)(p.D * sizeof(TX)));
  Piece<TG, N> raw[BOTH ? 2 : 1][TOKENS];
#pragma unroll
  for (int w = 0; w < (BOTH ? 2 : 1); ++w)
    load_run(raw[w], tile.rows_of<TG>(p.g[w], p.gb, p.gl), offset(p.gl, sizeof(TG)), (unsigned)(p.gl * sizeof(TG)));
  float a[BOTH ? 2 : 1][TOKENS][N];
  Map<N> along[BOTH ? 2 : 1], against[BOTH ? 2 : 1];
  if constexpr (!FOLD) {
    if (p.chunks > 1) {
      // (only the boards are wanted)
#pragma unroll
      for (int w = 0; w < (BOTH ? 2 : 1); ++w) {
        Map<N> f = w ? fold_chunks<false, N>(p, tile, at, 2, dirs, c, has) : fold_chunks<true, N>(p, tile, at, 0, dirs, c, has);
        if (w) fold_wave<false, N>(f, at, front[2]);
        else fold_wave<true, N>(f, at, front[0]);
        f = w ? fold_chunks<true, N>(p, tile, at, 3, dirs, c, has) : fold_chunks<false, N>(p, tile, at, 1, dirs, c, has);
        if (w) fold_wave<true, N>(f, at, front[3]);
        else fold_wave<false, N>(f, at, front[1]);
      }
    }
  }
#pragma unroll
  for (int w = 0; w < (BOTH ? 2 : 1); ++w) {
    factors(raw[w], a[w]);
    if (w == 0) {
      along[w] = fold_run<true>(a[w], x);
      against[w] = fold_back<false>(a[w], dy, p.scale, along[w]);
      fold_wave<true>(along[w], at, board[0]);
      fold_wave<false>(against[w], at, board[1]);
    } else {
      along[w] = fold_run<false>(a[w], x);
      against[w] = fold_back<true>(a[w], dy, p.scale, along[w]);
      fold_wave<false>(along[w], at, board[2]);
      fold_wave<true>(against[w], at, board[3]);
    }
  }
  __syncthreads();
  if constexpr (FOLD) {
    if (at.wave == 0 && at.run == 0 && has) {
      store_map(p, tile, 0, dirs, c, whole<true, N>(at, board[0]));
      store_map(p, tile, 1, dirs, c, whole<false, N>(at, board[1]));
      if constexpr (BOTH) {
        store_map(p, tile, 2, dirs, c, whole<false, N>(at, board[2]));
        store_map(p, tile, 3, dirs, c, whole<true, N>(at, board[3]));
      }
    }
    return;
  }
  float dx[TOKENS][N];
#pragma unroll
  for (int w = 0; w < (BOTH ? 2 : 1); ++w) {
    float h[N], d[N], u[TOKENS][N];
    load_state(h, w ? nullptr : p.h0, p, tile.b, c, has);
    load_state(d, w ? nullptr : p.dhT, p, tile.b, c, has);
    if (w == 0) {
      if (p.chunks > 1) whole<true, N>(at, front[0]).apply(h), whole<false, N>(at, front[1]).apply(d);
      enter<true, N>(h, along[w], at, board[0]);
      enter<false, N>(d, against[w], at, board[1]);
    } else {
      if (p.chunks > 1) whole<false, N>(at, front[2]).apply(h), whole<true, N>(at, front[3]).apply(d);
      enter<false, N>(h, along[w], at, board[2]);
      enter<true, N>(d, against[w], at, board[3]);
    }
#pragma unroll
    for (int k = 0; k < TOKENS; ++k) {
      const int t = w == 0 ? k : TOKENS - 1 - k;
#pragma unroll
      for (int i = 0; i < N; ++i) u[t][i] = a[w][t][i] * h[i], h[i] = u[t][i] + x[t].get(i);
    }
    const rsrc_t out = tile.rows_of<TG>(p.dg[w], dense, p.D);
    const unsigned to = offset(p.D, sizeof(TG));
#pragma unroll
    for (int k = 0; k < TOKENS; ++k) {
      const int t = w == 0 ? TOKENS - 1 - k : k;
      float dg[N];
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float dh = fmaf(p.scale, dy[t].get(i), d[i]);
        dx[t][i] = w == 0 ? dh : dx[t][i] + dh;
        dg[i] = dh * u[t][i];
        d[i] = a[w][t][i] * dh;
      }
      Piece<TG, N>::store(out, to + t * (unsigned)(p.D * sizeof(TG)), dg);
    }
    if (w == 0 && p.dh0 && tile.ch == 0 && at.wave == 0 && at.run == 0 && has) store_state(p.dh0, d, p, tile.b, c);
  }
  const rsrc_t out = tile.rows_of<TX>(p.dx, dense, p.D);
  const unsigned to = offset(p.D, sizeof(TX));
#pragma unroll
  for (int t = 0; t < TOKENS; ++t) Piece<TX, N>::store(out, to + t * (unsigned)(p.D * sizeof(TX)), dx[t]);
}

// ---- bf16 sequences of at most 256 tokens whose rows keep 16-byte boundaries: everything moves 16 bytes a lane and by whole lines
//
// Loads of four bytes a lane keep the address units busy four times as long as ones of sixteen, and lines whose halves two workgroups write go to memory by halves: a
// copy of three tensors into one in the pattern of the kernels above takes 20.5 us at 128 x 196 x 384, one of 16 bytes a lane and 128-byte rows 14.3.  Here a wave has
// 16 tokens of 64 channels; its rows go straight to its own part of LDS, from where each lane takes its channels, and back the same way, past the caches; the waves' maps
// lie where the gates were.  128 x 196 x 384: causal 15.9 -> 13.5 us, its gradients 26.8 -> 25.9, those of both directions 41.6 -> 35.6, of 1024 x 20 x 384 26.6 -> 23.7.  (The
// forward of both directions needs more registers than two workgroups a compute unit leave: 21.7 -> 23.3; a persistent form with the next rows on their way 20.7.)

typedef Piece<uint16_t, 2> Pair;
constexpr int kHalf = 32;                        // lanes that take a token's channels: two runs of eight tokens a wave
constexpr int kStep = 2 * kTokens;               // tokens of a wave
constexpr int kRow = 4 * kHalf;                  // bytes of a token's row
constexpr int kRows = kStep * kRow;              // of a wave's rows of one tensor, two loads of a kilobyte
constexpr int kHalfBoard = kHalf * 4 * (int)sizeof(float);  // of a wave's maps in one direction
constexpr int kRowsTokens = kMaxWaves * kStep;
static_assert(kRows == 2048 && 2 * kHalfBoard <= kRows, "two boards take a tensor's place");

struct HalfPlace {
  int wave, waves, lane, run, lc;
  __device__ __forceinline__ HalfPlace()
      : wave(__builtin_amdgcn_readfirstlane(threadIdx.x >> 6)), waves(blockDim.x >> 6), lane(threadIdx.x & 63), run((threadIdx.x & 63) / kHalf), lc(threadIdx.x % kHalf) {}
};

// Token t of the second run lies beside token t of the first, so that a read of both meets every bank once.
__device__ __forceinline__ int token_of_row(int row) { return (row >> 1) + kTokens * (row & 1); }
// a wave's rows into LDS; tokens and pieces of a row that the tensor does not have are read from its last ones
__device__ __forceinline__ void fetch_rows(const uint16_t* base, long long pitch, int first, int rows, int width, int lane, uint32_t lds) {
  const int piece = min(lane % 8, width / 8 - 1);
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int t = min(first + token_of_row(k * 8 + lane / 8), rows - 1);
    load_to_lds16(base, (unsigned)t * (unsigned)(2 * pitch) + piece * 16u, lds + k * 1024);
  }
}
__device__ __forceinline__ void take_rows(const char* lds, const HalfPlace& at, Pair (&x)[kTokens]) {
#pragma unroll
  for (int t = 0; t < kTokens; ++t) x[t].v = *reinterpret_cast<const uint32_t*>(lds + (2 * t + at.run) * kRow + 4 * at.lc);
}
// tokens behind the sequence: nothing
__device__ __forceinline__ void cut_rows(int left, Pair (&x)[kTokens]) {
#pragma unroll
  for (int t = 0; t < kTokens; ++t) x[t].v = t < left ? x[t].v : 0u;
}
// the thread's values of its token t into the wave's rows ...
__device__ __forceinline__ void put_row(char* lds, const HalfPlace& at, int t, const float (&y)[2]) {
  *reinterpret_cast<uint32_t*>(lds + (2 * t + at.run) * kRow + 4 * at.lc) = pack_bf16x2(y[0], y[1]);
}
// ... and the rows to memory
__device__ __forceinline__ void send_rows(const char* lds, void* base, const ScanArgs& p, int b, int first, int c0, int width, int lane) {
  const rsrc_t out = __builtin_amdgcn_make_buffer_rsrc(static_cast<uint16_t*>(base) + (long long)b * p.L * p.D, 0, p.L * p.D * 2, 0x00020000);
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int t = first + token_of_row(k * 8 + lane / 8);
    const u32x4_t v = *reinterpret_cast<const u32x4_t*>(lds + k * 1024 + lane * 16);
    const unsigned to = lane % 8 * 8 < width ? (unsigned)(t * p.D + c0) * 2u + lane % 8 * 16u : kBeyond;
    __builtin_amdgcn_raw_buffer_store_b128(v, out, to, 0, 2);  // (non-temporal)
  }
}
__device__ __forceinline__ void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// As fold_wave: what lies in front of this thread in its wave stays in `m`, the wave's map goes to its board.
template <bool UP>
__device__ __forceinline__ void fold_halves(Map<2>& m, const HalfPlace& at, char* board) {
  Map<2> low, high;
  both_of<true>(m, low, high);
  const bool behind = UP ? at.run == 1 : at.run == 0;
#pragma unroll
  for (int i = 0; i < 2; ++i) m.a[i] = behind ? (UP ? low : high).a[i] : 1.f, m.s[i] = behind ? (UP ? low : high).s[i] : 0.f;
  if (UP) high.behind(low);
  else low.behind(high);
  const Map<2>& t = UP ? high : low;
  if (at.run == 0) reinterpret_cast<f32x4_t*>(board)[at.lc] = f32x4_t{t.a[0], t.s[0], t.a[1], t.s[1]};
}
// (behind the barrier) the state that enters this thread's tokens, four waves' maps at a time; boards lie `pitch` bytes apart
template <bool UP>
__device__ __forceinline__ void enter_halves(float (&h)[2], const Map<2>& m, const HalfPlace& at, const char* boards, int pitch) {
  const int n = UP ? at.wave : at.waves - 1 - at.wave;
  for (int k = 0; k < n; k += 4) {
    f32x4_t v[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) v[q] = reinterpret_cast<const f32x4_t*>(boards + (UP ? min(k + q, at.waves - 1) : max(at.waves - 1 - k - q, 0)) * pitch)[at.lc];
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (k + q < n) h[0] = fmaf(v[q][0], h[0], v[q][1]), h[1] = fmaf(v[q][2], h[1], v[q][3]);
  }
  m.apply(h);
}

__global__ __launch_bounds__(64 * kMaxWaves) __attribute__((amdgpu_waves_per_eu(7))) void gated_scan_rows_kernel(ScanArgs p) {
  constexpr int kWave = 2 * kRows;  // of LDS: x, gates
  extern __shared__ __align__(16) char lds[];
  const HalfPlace at;
  char *const xs = lds + at.wave * kWave, *const gs = xs + kRows;
  const int first = at.wave * kStep, mine = first + at.run * kTokens;
  const Tile tile(p, true);
  const int b = tile.b, c0 = tile.cg * 2 * kHalf, width = min(2 * kHalf, p.D - c0), c = c0 + 2 * at.lc;
  const bool has = c < p.D;
  const uint32_t to = __builtin_amdgcn_readfirstlane(lds_offset(xs));
  fetch_rows(static_cast<const uint16_t*>(p.g[0]) + b * p.gb + c0, p.gl, first, p.L, width, at.lane, to + kRows);
  fetch_rows(static_cast<const uint16_t*>(p.x) + b * p.xb + c0, p.xl, first, p.L, width, at.lane, to);
  float h[2], a[kTokens][2];
  load_state(h, p.h0, p, b, c, has);
  Pair x[kTokens], raw[kTokens];
  wait_vmem<0>();
  take_rows(gs, at, raw), take_rows(xs, at, x);
  if (first + kStep > p.L) cut_rows(p.L - mine, raw), cut_rows(p.L - mine, x);  // (the last wave)
  factors(raw, a);
  wait_lds();  // (before a map takes the gates' place)
  Map<2> m = fold_run<true>(a, x);
  fold_halves<true>(m, at, gs);
  __syncthreads();
  enter_halves<true>(h, m, at, lds + kRows, kWave);
#pragma unroll
  for (int t = 0; t < kTokens; ++t) {
    float y[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) h[i] = fmaf(a[t][i], h[i], x[t].get(i)), y[i] = p.scale * h[i];
    put_row(xs, at, t, y);
  }
  if (p.hT && at.wave == at.waves - 1 && at.run == 1 && has) store_state(p.hT, h, p, b, c);
  wait_lds();
  send_rows(xs, p.o, p, b, first, c0, width, at.lane);
}

template <bool BOTH>
__global__ __launch_bounds__(64 * kMaxWaves) void gated_scan_rows_bwd_kernel(ScanArgs p) {
  constexpr int ways = BOTH ? 2 : 1, kWave = (2 + ways) * kRows;  // of LDS: x, the output's gradient, gates
  extern __shared__ __align__(16) char lds[];
  const HalfPlace at;
  char *const xs = lds + at.wave * kWave, *const ds = xs + kRows, *const gs = ds + kRows;
  const int first = at.wave * kStep, mine = first + at.run * kTokens;
  const Tile tile(p, true);
  const int b = tile.b, c0 = tile.cg * 2 * kHalf, width = min(2 * kHalf, p.D - c0), c = c0 + 2 * at.lc;
  const bool has = c < p.D;
  const uint32_t to = __builtin_amdgcn_readfirstlane(lds_offset(xs));
#pragma unroll
  for (int w = 0; w < ways; ++w) fetch_rows(static_cast<const uint16_t*>(p.g[w]) + b * p.gb + c0, p.gl, first, p.L, width, at.lane, to + (2 + w) * kRows);
  fetch_rows(static_cast<const uint16_t*>(p.x) + b * p.xb + c0, p.xl, first, p.L, width, at.lane, to);
  fetch_rows(static_cast<const uint16_t*>(p.d_o) + (long long)b * p.L * p.D + c0, p.D, first, p.L, width, at.lane, to + kRows);
  Pair x[kTokens], dy[kTokens];
  float a[ways][kTokens][2];
  wait_vmem<0>();
  {
    Pair raw[ways][kTokens];
#pragma unroll
    for (int w = 0; w < ways; ++w) take_rows(gs + w * kRows, at, raw[w]);
    take_rows(xs, at, x), take_rows(ds, at, dy);
    if (first + kStep > p.L) {  // (the last wave)
#pragma unroll
      for (int w = 0; w < ways; ++w) cut_rows(p.L - mine, raw[w]);
      cut_rows(p.L - mine, x), cut_rows(p.L - mine, dy);
    }
#pragma unroll
    for (int w = 0; w < ways; ++w) factors(raw[w], a[w]);
  }
  wait_lds();  // (before maps take the gates' place)
  Map<2> along[ways], against[ways];
#pragma unroll
  for (int w = 0; w < ways; ++w) {
    char* const board = gs + w * kRows;
    along[w] = w ? fold_run<false>(a[w], x) : fold_run<true>(a[w], x);
    against[w] = w ? fold_back<true>(a[w], dy, p.scale, along[w]) : fold_back<false>(a[w], dy, p.scale, along[w]);
    if (w) fold_halves<false>(along[w], at, board), fold_halves<true>(against[w], at, board + kHalfBoard);
    else fold_halves<true>(along[w], at, board), fold_halves<false>(against[w], at, board + kHalfBoard);
  }
  __syncthreads();
  float dx[kTokens][2];
#pragma unroll
  for (int w = 0; w < ways; ++w) {
    const char* const board = lds + (2 + w) * kRows;
    float h[2], d[2], u[kTokens][2];
    load_state(h, w ? nullptr : p.h0, p, b, c, has);
    load_state(d, w ? nullptr : p.dhT, p, b, c, has);
    if (w) enter_halves<false>(h, along[w], at, board, kWave), enter_halves<true>(d, against[w], at, board + kHalfBoard, kWave);
    else enter_halves<true>(h, along[w], at, board, kWave), enter_halves<false>(d, against[w], at, board + kHalfBoard, kWave);
#pragma unroll
    for (int k = 0; k < kTokens; ++k) {
      const int t = w == 0 ? k : kTokens - 1 - k;
#pragma unroll
      for (int i = 0; i < 2; ++i) u[t][i] = a[w][t][i] * h[i], h[i] = u[t][i] + x[t].get(i);
    }
#pragma unroll
    for (int k = 0; k < kTokens; ++k) {
      const int t = w == 0 ? kTokens - 1 - k : k;
      float dg[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float dh = fmaf(p.scale, dy[t].get(i), d[i]);
        dx[t][i] = w == 0 ? dh : dx[t][i] + dh;
        dg[i] = dh * u[t][i];
        d[i] = a[w][t][i] * dh;
      }
      put_row(xs, at, t, dg);
    }
    if (w == 0 && p.dh0 && at.wave == 0 && at.run == 0 && has) store_state(p.dh0, d, p, b, c);
    wait_lds();
    send_rows(xs, p.dg[w], p, b, first, c0, width, at.lane);
    wait_lds();  // (before the next rows take these rows' place)
  }
#pragma unroll
  for (int t = 0; t < kTokens; ++t) put_row(xs, at, t, dx[t]);
  wait_lds();
  send_rows(xs, p.dx, p, b, first, c0, width, at.lane);
}

// ---- one token

template <typename T>
__device__ __forceinline__ void load_some(const T* p, float (&x)[1]) { x[0] = Elem<T>::load(p); }
__device__ __forceinline__ void load_some(const float* p, float (&x)[4]) {
  const f32x4_t v = *reinterpret_cast<const f32x4_t*>(p);
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = v[i];
}
__device__ __forceinline__ void load_some(const uint16_t* p, float (&x)[4]) {
  const u32x2_t v = *reinterpret_cast<const u32x2_t*>(p);
  x[0] = bf16lo_to_f32(v[0]), x[1] = bf16hi_to_f32(v[0]), x[2] = bf16lo_to_f32(v[1]), x[3] = bf16hi_to_f32(v[1]);
}
template <typename T>
__device__ __forceinline__ void store_some(T* p, const float (&x)[1]) { Elem<T>::store(p, x[0]); }
__device__ __forceinline__ void store_some(float* p, const float (&x)[4]) { *reinterpret_cast<f32x4_t*>(p) = f32x4_t{x[0], x[1], x[2], x[3]}; }
__device__ __forceinline__ void store_some(uint16_t* p, const float (&x)[4]) {
  *reinterpret_cast<u32x2_t*>(p) = u32x2_t{pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3])};
}

// 14 bytes a channel in bf16, and nothing to wait for but memory: 2048 x 1024 5.8 us, 5.0 TB/s; one sequence of 384 channels 1.4 us, less than its launch.
template <typename TX, typename TG, int N>
__global__ __launch_bounds__(256) void gated_scan_step_kernel(const TX* x, const TG* g, float* h, TX* o, unsigned n, unsigned per_row, long long xl, long long gl, int D) {
  const unsigned id = blockIdx.x * 256u + threadIdx.x;
  if (id >= n) return;
  const unsigned b = id / per_row, c = (id - b * per_row) * N;
  const TX* xr = x + b * xl + c;
  const TG* gr = g + b * gl + c;
  const size_t at = (size_t)b * D + c;
  float a[N], v[N], s[N];
  load_some(gr, a), load_some(xr, v), load_some(h + at, s);
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = fmaf(exp_fast(a[i]), s[i], v[i]);
  store_some(h + at, v), store_some(o + at, v);
}

static_assert(16LL * kRuns * kMaxWaves * kScanRow * 4 <= kBeyond, "byte offsets of a workgroup's rows");

// ---- host side

struct Cut {
  bool pairs;
  int tokens, waves, chunks, chunk, groups;
};
// Whether N channels move at once: whole ones of them in every row, on boundaries of their size (a null pointer stands on any)
inline bool whole(int n, int D, long long a, long long b, long long c, long long d) { return D % n == 0 && (a | b | c | d) % n == 0; }
template <typename... P>
bool on(int n, int dtype, P... p) {
  const uintptr_t size = n * (dtype == VIG_BF16 ? 2 : 4);
  return ((reinterpret_cast<uintptr_t>(p) % size == 0) && ...);
}

inline Cut cut(int L, int D, bool pairs, int tokens) {
  Cut k{pairs, tokens};
  const int tile = kLanes * (pairs ? 2 : 1), run = kRuns * tokens;  // channels of a workgroup, tokens of a wave
  k.groups = (D + tile - 1) / tile;
  const int waves = (L + run - 1) / run;
  k.chunks = (waves + kMaxWaves - 1) / kMaxWaves;
  k.waves = (waves + k.chunks - 1) / k.chunks;
  k.chunk = k.waves * run;
  k.chunks = (L + k.chunk - 1) / k.chunk;
  return k;
}

// Sequences of 513 to 1024 tokens are one workgroup's with 16 tokens a thread, where 8 make two chunks of them and read everything twice; for both directions with
// one channel a lane, which leaves the registers for it.  us, 64 x 1024 x 384: causal 51.8 -> 35.4, its gradients 104 -> 60, both 94 -> 68, gradients 154 -> 109.  Many
// chunks of a causal gradient gain too (65536 x 1024: 278 -> 252; 4 x 2305 x 384, fewer workgroups than fill the chip: 19.0 -> 21.8).
inline Cut cut_for(int B, int L, int D, bool pairs, bool both, bool bwd) {
  const Cut few = cut(L, D, pairs, kTokens);
  if (few.chunks == 1) return few;
  if (L <= 16 * kRuns * kMaxWaves) return cut(L, D, pairs && !both, 16);
  const Cut wide = cut(L, D, pairs, 16);
  return bwd && !both && (long long)B * wide.groups * wide.chunks >= 1024 ? wide : few;
}

template <typename TX, typename TG, bool BOTH, int N, int TOKENS>
void start(const ScanArgs& p, bool bwd, bool fold, dim3 grid, dim3 block, hipStream_t stream) {
  const size_t lds = block.x / 64 * Board<N>::kBytes * (BOTH ? 2 : 1) * (bwd ? 2 : 1) * (!fold && p.chunks > 1 ? 2 : 1);  // (at most 64 KB)
  if (bwd) {
    if (fold) hipLaunchKernelGGL((gated_scan_bwd_kernel<TX, TG, BOTH, true, N, TOKENS>), grid, block, lds, stream, p);
    else hipLaunchKernelGGL((gated_scan_bwd_kernel<TX, TG, BOTH, false, N, TOKENS>), grid, block, lds, stream, p);
  } else {
    if (fold) hipLaunchKernelGGL((gated_scan_kernel<TX, TG, BOTH, true, N, TOKENS>), grid, block, lds, stream, p);
    else hipLaunchKernelGGL((gated_scan_kernel<TX, TG, BOTH, false, N, TOKENS>), grid, block, lds, stream, p);
  }
}
template <typename TX, typename TG>
void start(const ScanArgs& p, bool bwd, bool fold, const Cut& k, dim3 grid, dim3 block, hipStream_t stream) {
  if (p.g[1]) {
    if (k.tokens == 16) start<TX, TG, true, 1, 16>(p, bwd, fold, grid, block, stream);
    else if (k.pairs) start<TX, TG, true, 2, 8>(p, bwd, fold, grid, block, stream);
    else start<TX, TG, true, 1, 8>(p, bwd, fold, grid, block, stream);
  } else if (k.tokens == 8) {
    if (k.pairs) start<TX, TG, false, 2, 8>(p, bwd, fold, grid, block, stream);
    else start<TX, TG, false, 1, 8>(p, bwd, fold, grid, block, stream);
  } else {
    if (k.pairs) start<TX, TG, false, 2, 16>(p, bwd, fold, grid, block, stream);
    else start<TX, TG, false, 1, 16>(p, bwd, fold, grid, block, stream);
  }
}
// Whether and how bf16 sequences go by whole rows: 0, or launched
inline int start_rows(ScanArgs p, bool bwd, int B, hipStream_t stream) {
  const bool lies = p.L <= kRowsTokens && whole(8, p.D, p.xb, p.xl, p.gb, p.gl) && on(8, VIG_BF16, p.x, p.g[0], p.g[1], p.d_o, p.o, p.dx, p.dg[0], p.dg[1]);
  if (!lies || (!bwd && p.g[1])) return 0;
  p.groups = (p.D + 2 * kHalf - 1) / (2 * kHalf), p.chunks = 1, p.chunk = p.L;
  const long long groups = (long long)B * p.groups;
  // Few workgroups finish sooner as the smaller ones of the other kernels (4 x 196 x 192, gradients of both directions 5.6 us for 7.6), and lanes behind
  // the last channel work for nothing (500 x 100 x 200: 38 for 52).
  if (groups < 256 || groups * (64 * kMaxWaves) > kMostThreads || p.groups * 2 * kHalf * 8 > p.D * 9) return 0;
  const int waves = (p.L + kStep - 1) / kStep;
  const size_t lds = (size_t)waves * kRows * (bwd ? p.g[1] ? 4 : 3 : 2);
  static bool allowed[3][64];
  const void* const kernel = !bwd ? (const void*)gated_scan_rows_kernel : p.g[1] ? (const void*)gated_scan_rows_bwd_kernel<true> : (const void*)gated_scan_rows_bwd_kernel<false>;
  if (!allow_lds(kernel, kMaxWaves * kRows * (bwd ? p.g[1] ? 4 : 3 : 2), allowed[!bwd ? 0 : p.g[1] ? 2 : 1])) return 0;
  const dim3 grid((unsigned)groups), block(64 * waves);
  if (!bwd) hipLaunchKernelGGL(gated_scan_rows_kernel, grid, block, lds, stream, p);
  else if (p.g[1]) hipLaunchKernelGGL(gated_scan_rows_bwd_kernel<true>, grid, block, lds, stream, p);
  else hipLaunchKernelGGL(gated_scan_rows_bwd_kernel<false>, grid, block, lds, stream, p);
  return 1;
}

int run_some(ScanArgs& p, bool bwd, int B, const Cut& k, int io_dtype, int gate_dtype, hipStream_t stream) {
  const dim3 grid((unsigned)B * (unsigned)(k.groups * k.chunks)), block(64 * k.waves);
  for (int fold = k.chunks > 1; fold >= 0; --fold) {
    if (io_dtype == VIG_BF16) {
      if (gate_dtype == VIG_BF16) start<uint16_t, uint16_t>(p, bwd, fold, k, grid, block, stream);
      else start<uint16_t, float>(p, bwd, fold, k, grid, block, stream);
    } else {
      if (gate_dtype == VIG_BF16) start<float, uint16_t>(p, bwd, fold, k, grid, block, stream);
      else start<float, float>(p, bwd, fold, k, grid, block, stream);
    }
    if (hipGetLastError() != hipSuccess) return VIG_ELAUNCH;
  }
  return VIG_OK;
}

int run(ScanArgs& p, bool bwd, int B, int io_dtype, int gate_dtype, hipStream_t stream) {
  if (io_dtype == VIG_BF16 && gate_dtype == VIG_BF16 && start_rows(p, bwd, B, stream)) return hipGetLastError() == hipSuccess ? VIG_OK : VIG_ELAUNCH;
  const bool pairs = whole(2, p.D, p.xb, p.xl, p.gb, p.gl) && on(2, io_dtype, p.x, p.d_o, p.o, p.dx) && on(2, gate_dtype, p.g[0], p.g[1], p.dg[0], p.dg[1]);
  const Cut k = cut_for(B, p.L, p.D, pairs, p.g[1] != nullptr, bwd);
  p.groups = k.groups, p.chunks = k.chunks, p.chunk = k.chunk;
  // a launch takes 2^32 threads at most: more batch elements go by several (each element's chunks alone have to fit)
  const long long most = (long long)kMostThreads / (64 * k.waves) / ((long long)k.groups * k.chunks);
  if (most < 1) return VIG_ENOTSUP;
  const size_t sx = io_dtype == VIG_BF16 ? 2 : 4, sg = gate_dtype == VIG_BF16 ? 2 : 4;
  const size_t dense = (size_t)p.L * p.D, maps = (size_t)(p.g[1] ? 2 : 1) * (bwd ? 2 : 1) * k.chunks * p.D * 2;
  for (long long b = 0; b < B; b += most) {
    ScanArgs q = p;
    auto at = [](auto& t, size_t bytes) { t = t ? (std::remove_reference_t<decltype(t)>)((uintptr_t)t + bytes) : t; };
    at(q.x, b * p.xb * sx), at(q.g[0], b * p.gb * sg), at(q.g[1], b * p.gb * sg), at(q.d_o, b * dense * sx), at(q.o, b * dense * sx), at(q.dx, b * dense * sx);
    at(q.dg[0], b * dense * sg), at(q.dg[1], b * dense * sg), at(q.maps, k.chunks > 1 ? b * maps * sizeof(float) : 0);
    for (auto* t : {&q.h0, &q.dhT}) at(*t, b * p.D * sizeof(float));
    for (auto* t : {&q.hT, &q.dh0}) at(*t, b * p.D * sizeof(float));
    const int rc = run_some(q, bwd, (int)std::min(most, B - b), k, io_dtype, gate_dtype, stream);
    if (rc != VIG_OK) return rc;
  }
  return VIG_OK;
}

}  // namespace

// Bytes for the chunks' maps, whichever way the rows lie.
size_t gated_scan_workspace(int B, int L, int D, bool both, bool bwd) {
  const int chunks = std::max(cut_for(B, L, D, false, both, bwd).chunks, cut_for(B, L, D, true, both, bwd).chunks);
  return chunks > 1 ? (size_t)B * (both ? 2 : 1) * (bwd ? 2 : 1) * chunks * D * 2 * sizeof(float) : 0;
}

int launch_gated_scan(const GatedScan& s, hipStream_t stream) {
  ScanArgs p{};
  p.x = s.x, p.g[0] = s.g_fwd, p.g[1] = s.g_bwd, p.o = s.o, p.h0 = s.initial, p.hT = s.final, p.maps = static_cast<float*>(s.workspace);
  p.xb = s.x_strides[0], p.xl = s.x_strides[1], p.gb = s.g_strides[0], p.gl = s.g_strides[1];
  p.L = s.L, p.D = s.D, p.scale = s.out_scale;
  p.d_o = s.d_o, p.dx = s.dx, p.dg[0] = s.dg_fwd, p.dg[1] = s.dg_bwd, p.dhT = s.d_final, p.dh0 = s.d_initial;
  return run(p, s.d_o != nullptr, s.B, s.io_dtype, s.gate_dtype, stream);
}

template <typename TX, typename TG>
static void start_step(const GatedScanStep& s, bool vector, hipStream_t stream) {
  const unsigned per_row = vector ? s.D / 4 : s.D, n = (unsigned)s.B * per_row;
  const dim3 grid((n + 255) / 256), block(256);
  if (vector)
    hipLaunchKernelGGL((gated_scan_step_kernel<TX, TG, 4>), grid, block, 0, stream, (const TX*)s.x, (const TG*)s.g, s.state, (TX*)s.o, n, per_row, s.x_stride,
                       s.g_stride, s.D);
  else
    hipLaunchKernelGGL((gated_scan_step_kernel<TX, TG, 1>), grid, block, 0, stream, (const TX*)s.x, (const TG*)s.g, s.state, (TX*)s.o, n, per_row, s.x_stride,
                       s.g_stride, s.D);
}

int launch_gated_scan_step(const GatedScanStep& s, hipStream_t stream) {
  if ((long long)s.B * s.D > 0x7fffff00LL) return VIG_ENOTSUP;
  const bool vector = whole(4, s.D, s.x_stride, s.g_stride, 0, 0) && on(4, s.io_dtype, s.x, s.o) && on(4, s.gate_dtype, s.g) && on(4, VIG_F32, s.state);
  if (s.io_dtype == VIG_BF16) {
    if (s.gate_dtype == VIG_BF16) start_step<uint16_t, uint16_t>(s, vector, stream);
    else start_step<uint16_t, float>(s, vector, stream);
  } else {
    if (s.gate_dtype == VIG_BF16) start_step<float, uint16_t>(s, vector, stream);
    else start_step<float, float>(s, vector, stream);
  }
  return hipGetLastError() == hipSuccess ? VIG_OK : VIG_ELAUNCH;
}

}  // namespace vig
