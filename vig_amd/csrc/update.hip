// What a training step does to a list of tensors: the norm of all gradients, and AdamW with its moments in 32 or in 8 bits.
//
//   norm = sqrt(sum g^2),  factor = min(1, max_norm / (norm + 1e-6))
//   g' = factor g;  m <- b1 m + (1 - b1) g';  v <- b2 v + (1 - b2) g'^2
//   p <- p (1 - lr decay) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// Both are bound by memory: every tensor is read once, what changes is written once, 16 bytes a lane.  A launch takes a table of tensors in its
// arguments (nothing is copied to the device, so that a captured launch holds all it needs); a workgroup takes one piece of 2048 elements
// (norm: 8192) and finds its tensor by comparing its number with the tensors' last pieces, one a lane.  Measured (us, TB/s; a large copy by torch: 5.3): fp32, 89 M parameters 417,
// 6.0; in 8 bits beside fp32 282, 5.1, beside bf16 165 to 187, 4.8 to 5.4, where the arithmetic (75 instructions an element) comes near the memory's time; norm of 89 M bf16 32, 5.5.
//
// 8 bits: blocks of 256 elements, counted from each tensor's first, hold m and r = sqrt(v) as e4m3 values times a scale of max / 448.  (The root: v spans
// twice the octaves that e4m3 has.)  Rounding is stochastic: by the nearest value a moment would stand still, as a step of e4m3 is 6 to 12 % and b2 moves v
// by 0.1 %.  Parameters in bf16 are rounded the same way, for the same reason.  A positive r never becomes 0, which would divide by eps alone.
#include "common.h"
#include "launch.h"
#include <type_traits>

namespace vig {
namespace {

// Elements of a workgroup.  us with half / as many / twice as many: AdamW in fp32 over the 180 parameters of a ViG-T 33 / 33 / 36, of a ViG-B 417 / 417 / 420, in 8 bits
// and bf16 27 / 27 / 32 and 187 / 188 / 187; the norm of the latter's gradients 57 / 32 / 31, of a ViG-T's 9.7 / 9.7 / 11.5.
constexpr int kPiece = 2048;
constexpr int kNormPiece = 8192;
constexpr int kNormJobs = 192;
constexpr unsigned kMostPieces = 0xffffffu;  // of a launch: it takes 2^32 threads at most

// A launch's table: at most 4 KB of arguments in all.
template <bool BITS8> struct UpdateJobs;
template <> struct UpdateJobs<false> {
  static constexpr int kMost = 90;
  void* p[kMost];
  const void* g[kMost];
  void* m[kMost];
  void* v[kMost];
  unsigned n[kMost];      // elements
  unsigned upto[kMost];   // pieces up to and with this tensor's
  unsigned first[kMost];  // number of the tensor's first element, from the launch's on
};
template <> struct UpdateJobs<true> {
  static constexpr int kMost = 64;
  void* p[kMost];
  const void* g[kMost];
  void* m[kMost];
  void* v[kMost];
  float* ms[kMost];
  float* vs[kMost];
  unsigned n[kMost], upto[kMost], first[kMost];
};

struct UpdateScalars {
  float keep, step, rs2, b1, c1, b2, c2, eps;  // keep = 1 - lr decay, step = lr / (1 - b1^t), rs2 = 1 / sqrt(1 - b2^t), c = 1 - b
};
struct UpdateOnDevice {  // where the step's number or the learning rate lies on the device
  const long long* step;
  const float* lr;
  double b1, b2;
  float lr_host, decay;
  long long step_host;
};
static_assert(sizeof(UpdateJobs<false>) + sizeof(UpdateScalars) + sizeof(UpdateOnDevice) + 32 <= 4096 &&
                  sizeof(UpdateJobs<true>) + sizeof(UpdateScalars) + sizeof(UpdateOnDevice) + 32 <= 4096,
              "a launch's arguments");

typedef u32x4_t u32x4_any __attribute__((aligned(2)));  // pieces of tensors that begin anywhere
typedef u32x2_t u32x2_any __attribute__((aligned(1)));

// one 32-bit word from another, each bit of x deciding about every bit of it: multiplications by the fractional parts of two roots
__device__ __host__ inline uint32_t mix(uint32_t x) {
  x = (x ^ (x >> 16)) * 0x6A09E667u;
  x = (x ^ (x >> 15)) * 0xBB67AE85u;
  return x ^ (x >> 16);
}
constexpr uint32_t kGolden = 0x9E3779B9u;
__device__ __host__ inline uint32_t key_of(unsigned long long seed, long long step) {
  return mix(mix(mix((uint32_t)seed) + (uint32_t)(seed >> 32)) + (uint32_t)step);
}

// E consecutive elements of a tensor, of which `left` exist.  Nothing of a list is read again before its next step, and a list is larger than the caches as a rule:
// non-temporal (89 M parameters in fp32: 475 -> 420 us).
template <bool STREAM, typename V>
__device__ __forceinline__ V piece(const V* p) {
  if constexpr (STREAM) return __builtin_nontemporal_load(p);
  else return *p;
}
template <typename T> struct Some;
template <> struct Some<float> {
  template <int E, bool STREAM = true>
  static __device__ __forceinline__ void load(const void* p, size_t i, int left, float (&x)[E]) {
    const float* at = static_cast<const float*>(p) + i;
    if (left >= E) {
#pragma unroll
      for (int q = 0; q < E / 4; ++q) {
        const u32x4_t v = piece<STREAM>(reinterpret_cast<const u32x4_any*>(at + 4 * q));
#pragma unroll
        for (int k = 0; k < 4; ++k) x[4 * q + k] = __uint_as_float(v[k]);
      }
    } else {
#pragma unroll
      for (int k = 0; k < E; ++k) x[k] = k < left ? at[k] : 0.f;
    }
  }
  template <int E>
  static __device__ __forceinline__ void store(void* p, size_t i, int left, const float (&x)[E], const uint32_t (&)[E]) {
    float* at = static_cast<float*>(p) + i;
    if (left >= E) {
#pragma unroll
      for (int q = 0; q < E / 4; ++q)
        __builtin_nontemporal_store(u32x4_t{__float_as_uint(x[4 * q]), __float_as_uint(x[4 * q + 1]), __float_as_uint(x[4 * q + 2]), __float_as_uint(x[4 * q + 3])},
                                    reinterpret_cast<u32x4_any*>(at + 4 * q));
    } else {
#pragma unroll
      for (int k = 0; k < E; ++k)
        if (k < left) at[k] = x[k];
    }
  }
};
template <> struct Some<uint16_t> {
  template <int E, bool STREAM = true>
  static __device__ __forceinline__ void load(const void* p, size_t i, int left, float (&x)[E]) {
    const uint16_t* at = static_cast<const uint16_t*>(p) + i;
    if (left >= E) {
      uint32_t v[E / 2];
      if constexpr (E == 8) {
        const u32x4_t w = piece<STREAM>(reinterpret_cast<const u32x4_any*>(at));
        v[0] = w[0], v[1] = w[1], v[2] = w[2], v[3] = w[3];
      } else {
        const u32x2_t w = piece<STREAM>(reinterpret_cast<const u32x2_any*>(at));
        v[0] = w[0], v[1] = w[1];
      }
#pragma unroll
      for (int q = 0; q < E / 2; ++q) x[2 * q] = bf16lo_to_f32(v[q]), x[2 * q + 1] = bf16hi_to_f32(v[q]);
    } else {
#pragma unroll
      for (int k = 0; k < E; ++k) x[k] = k < left ? bf16_to_f32(at[k]) : 0.f;
    }
  }
  // the upper half of x plus 16 random bits at its lower half: up with the probability that the cut part is of a step (NaN stays one)
  template <int E>
  static __device__ __forceinline__ void store(void* p, size_t i, int left, const float (&x)[E], const uint32_t (&word)[E]) {
    uint16_t* at = static_cast<uint16_t*>(p) + i;
    uint32_t y[E];
#pragma unroll
    for (int k = 0; k < E; ++k) y[k] = x[k] == x[k] ? __float_as_uint(x[k]) + ((word[k] * kGolden) >> 16) : 0x7fc00000u;
    if (left >= E) {
      uint32_t v[E / 2];
#pragma unroll
      for (int q = 0; q < E / 2; ++q) v[q] = __builtin_amdgcn_perm(y[2 * q + 1], y[2 * q], 0x07060302u);
      if constexpr (E == 8) __builtin_nontemporal_store(u32x4_t{v[0], v[1], v[2], v[3]}, reinterpret_cast<u32x4_any*>(at));
      else __builtin_nontemporal_store(u32x2_t{v[0], v[1]}, reinterpret_cast<u32x2_any*>(at));
    } else {
#pragma unroll
      for (int k = 0; k < E; ++k)
        if (k < left) at[k] = (uint16_t)(y[k] >> 16);
    }
  }
};

// ---- states in 8 bits: eight elements a lane, a block of 256 half a wave's

__device__ __forceinline__ void load_codes(const void* p, size_t i, int left, float scale, float (&x)[8]) {
  const uint8_t* at = static_cast<const uint8_t*>(p) + i;
  u32x2_t w = {0u, 0u};
  if (left >= 8) {
    w = __builtin_nontemporal_load(reinterpret_cast<const u32x2_any*>(at));
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k < left) w[k / 4] |= (uint32_t)at[k] << (8 * (k % 4));
  }
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const f32x2_t lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[q], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[q], true);
    x[4 * q] = lo[0] * scale, x[4 * q + 1] = lo[1] * scale, x[4 * q + 2] = hi[0] * scale, x[4 * q + 3] = hi[1] * scale;
  }
}
// the largest of a lane's words in its half of the wave, in every lane of it
__device__ __forceinline__ uint32_t half_max(uint32_t x) {
  auto with = [&](uint32_t y) { x = max(x, y); };
  with(__builtin_amdgcn_update_dpp(0u, x, 0x111, 0xf, 0xf, true));  // the lane 1, 2, 4, 8 in front in its row of 16
  with(__builtin_amdgcn_update_dpp(0u, x, 0x112, 0xf, 0xf, true));
  with(__builtin_amdgcn_update_dpp(0u, x, 0x114, 0xf, 0xf, true));
  with(__builtin_amdgcn_update_dpp(0u, x, 0x118, 0xf, 0xf, true));
  const uint32_t a = max(__builtin_amdgcn_readlane(x, 15), __builtin_amdgcn_readlane(x, 31)), b = max(__builtin_amdgcn_readlane(x, 47), __builtin_amdgcn_readlane(x, 63));
  return (threadIdx.x & 32) ? b : a;
}
// The block's scale, and the codes of a lane's values.  y = |x| / scale <= 448 (1 + 2^-22), whose step is 2^-20 of the power of two below it, 2^-9 under
// 2^-6: the conversion adds the random bits to the top of the cut part (a test of all exponents holds it to that).  Magnitudes compare as their bits do, a NaN
// above all: a value that is not finite makes the scale so, and the block NaN.
__device__ __forceinline__ float store_codes(void* p, size_t i, int left, const float (&x)[8], const uint32_t (&bits)[8], bool root) {
  uint32_t most = 0u;
#pragma unroll
  for (int k = 0; k < 8; ++k) most = max(most, __float_as_uint(x[k]) & 0x7fffffffu);
  most = half_max(most);
  const bool fine = most < 0x7f800000u;
  const float scale = most ? fmaxf(__uint_as_float(most) * (1.f / 448.f), 0x1p-126f) : 0.f;
  const float inv = most ? __builtin_amdgcn_rcpf(scale) : 0.f;
  u32x2_t w = {0u, 0u};
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    // (a division's bits: the remainder of the quotient by the reciprocal, times it)
    const float near = x[k] * inv;
    float y = fmaf(fmaf(-near, scale, x[k]), inv, near);
    if (root) y = x[k] > 0.f ? fmaxf(y, 0x1p-9f) : 0.f;
    switch (k % 4) {
      case 0: w[k / 4] = __builtin_amdgcn_cvt_sr_fp8_f32(y, bits[k], w[k / 4], 0); break;
      case 1: w[k / 4] = __builtin_amdgcn_cvt_sr_fp8_f32(y, bits[k], w[k / 4], 1); break;
      case 2: w[k / 4] = __builtin_amdgcn_cvt_sr_fp8_f32(y, bits[k], w[k / 4], 2); break;
      default: w[k / 4] = __builtin_amdgcn_cvt_sr_fp8_f32(y, bits[k], w[k / 4], 3);
    }
  }
  w = fine ? w : u32x2_t{0x7f7f7f7fu, 0x7f7f7f7fu};
  uint8_t* at = static_cast<uint8_t*>(p) + i;
  if (left >= 8) {
    __builtin_nontemporal_store(w, reinterpret_cast<u32x2_any*>(at));
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k < left) at[k] = (uint8_t)(w[k / 4] >> (8 * (k % 4)));
  }
  return scale;
}

// (the table is read through the kernel's argument pointer: an index into a by-value argument would copy it to scratch)
template <typename T>
__device__ __forceinline__ const T* arguments() {
  return (const T*)(const void*)__builtin_amdgcn_kernarg_segment_ptr();
}
// the tensor of a piece: the first whose last piece lies behind it
template <int MOST>
__device__ __forceinline__ int tensor_of(const unsigned* upto, unsigned count, unsigned piece, unsigned mask = ~0u) {
  const unsigned lane = threadIdx.x & 63;
  int j = 0;
#pragma unroll
  for (unsigned first = 0; first < (unsigned)MOST; first += 64) j += __popcll(__ballot(first + lane < count && (upto[first + lane] & mask) <= piece));
  return __builtin_amdgcn_readfirstlane(j);
}

template <typename TP, typename TG, bool BITS8>
__global__ __launch_bounds__(256) void adamw_kernel(UpdateJobs<BITS8> by_value, UpdateScalars s, const float* grad_scale, unsigned count, uint32_t key, unsigned long long seed,
                                                    unsigned long long from, UpdateOnDevice dev) {
  constexpr int E = BITS8 ? 8 : 4, kTurns = kPiece / (256 * E);
  const UpdateJobs<BITS8>* jobs = arguments<UpdateJobs<BITS8>>();
  const unsigned piece = blockIdx.x;
  const int j = tensor_of<UpdateJobs<BITS8>::kMost>(jobs->upto, count, piece);
  const float clip = grad_scale ? *grad_scale : 1.f;
  if (clip != clip) return;  // the norm was not finite: everything stays as it is
  const unsigned first = (piece - (j ? jobs->upto[j - 1] : 0u)) * kPiece, n = jobs->n[j];
  void *const p = jobs->p[j], *const m = jobs->m[j], *const v = jobs->v[j];
  const void* const g = jobs->g[j];
  const unsigned long long number0 = from + jobs->first[j];
  float P[kTurns][E], G[kTurns][E], M[kTurns][E], V[kTurns][E];
  auto load = [&](auto full) {
    constexpr bool FULL = decltype(full)::value;
#pragma unroll
    for (int k = 0; k < kTurns; ++k) {
      const unsigned i = first + (k * 256 + threadIdx.x) * E;
      const int left = FULL ? E : i < n ? (int)min(n - i, (unsigned)E) : 0;
      Some<TP>::load(p, i, left, P[k]);
      Some<TG>::load(g, i, left, G[k]);
      if constexpr (BITS8) {
        const unsigned b = i >> 8;
        load_codes(m, i, left, left ? jobs->ms[j][b] : 0.f, M[k]);
        load_codes(v, i, left, left ? jobs->vs[j][b] : 0.f, V[k]);
#pragma unroll
        for (int e = 0; e < E; ++e) V[k][e] *= V[k][e];
      } else {
        Some<float>::load(m, i, left, M[k]);
        Some<float>::load(v, i, left, V[k]);
      }
    }
  };
  const bool whole = first + kPiece <= n;  // (of a piece that its tensor fills nothing is asked again)
  if (whole) load(std::true_type{});
  else load(std::false_type{});
  if (dev.step || dev.lr) {
    __shared__ float sc[4];
    if (threadIdx.x == 0) {
      const double lr = dev.lr ? (double)*dev.lr : (double)dev.lr_host, t = (double)(dev.step ? *dev.step : dev.step_host);
      sc[0] = (float)(1.0 - lr * (double)dev.decay);
      sc[1] = (float)(lr / -expm1(t * log(dev.b1)));
      sc[2] = (float)(1.0 / sqrt(-expm1(t * log(dev.b2))));
      sc[3] = __uint_as_float(key_of(seed, dev.step ? *dev.step : dev.step_host));
    }
    __syncthreads();
    s.keep = sc[0], s.step = sc[1], s.rs2 = sc[2], key = __float_as_uint(sc[3]);
  }
  auto finish = [&](auto full) {
    constexpr bool FULL = decltype(full)::value;
#pragma unroll
    for (int k = 0; k < kTurns; ++k) {
      const unsigned i = first + (k * 256 + threadIdx.x) * E;
      const int left = FULL ? E : i < n ? (int)min(n - i, (unsigned)E) : 0;
      float root[E];
      uint32_t word[E];
      if constexpr (BITS8 || sizeof(TP) == 2) {
        // (numbers of elements pass 32 bits: the upper ones go into the key)
        const unsigned long long number = number0 + i;
        const uint32_t low32 = (uint32_t)number, k2 = key + (uint32_t)(number >> 32) * kGolden;
#pragma unroll
        for (int e = 0; e < E; ++e) word[e] = mix((low32 + e) ^ k2);
        if (low32 > ~0u - (E - 1)) {
#pragma unroll
          for (int e = 0; e < E; ++e)
            if (low32 + e < low32) word[e] = mix((low32 + e) ^ (k2 + kGolden));
        }
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e) word[e] = 0u;
      }
#pragma unroll
      for (int e = 0; e < E; ++e) {
        // (products and sums rounded one by one: a last bit can turn a code over, and so the moments' bits are those of their formula)
#pragma clang fp contract(off)
        const float x = G[k][e] * clip;
        M[k][e] = s.b1 * M[k][e] + s.c1 * x;
        V[k][e] = s.b2 * V[k][e] + s.c2 * x * x;
        if constexpr (BITS8) {
          // a square root's bits from its reciprocal and one remainder (from the least normal value on; below, between 0 and the root)
          const float r = __builtin_amdgcn_rsqf(fmaxf(V[k][e], 0x1p-126f)), q = V[k][e] * r;
          root[e] = fmaf(fmaf(-q, q, V[k][e]), 0.5f * r, q);
          P[k][e] = fmaf(P[k][e], s.keep, -(s.step * M[k][e] * __builtin_amdgcn_rcpf(fmaf(root[e], s.rs2, s.eps))));
        } else {
          P[k][e] = fmaf(P[k][e], s.keep, -(s.step * M[k][e] / fmaf(sqrtf(V[k][e]), s.rs2, s.eps)));
        }
      }
      if constexpr (BITS8) {
        uint32_t low[E], high[E];
#pragma unroll
        for (int e = 0; e < E; ++e) low[e] = word[e] << 16, high[e] = word[e] & 0xffff0000u;
        if (left < E) {  // (what is not there has no part in its block's scale)
#pragma unroll
          for (int e = 0; e < E; ++e)
            if (e >= left) M[k][e] = root[e] = 0.f;
        }
        const float ms = store_codes(m, i, left, M[k], low, false), vs = store_codes(v, i, left, root, high, true);
        if ((threadIdx.x & 31) == 0 && left) jobs->ms[j][i >> 8] = ms, jobs->vs[j][i >> 8] = vs;
      } else {
        Some<float>::store(m, i, left, M[k], word);
        Some<float>::store(v, i, left, V[k], word);
      }
      Some<TP>::store(p, i, left, P[k], word);
    }
  };
  if (whole) finish(std::true_type{});
  else finish(std::false_type{});
}

// ---- norm

struct NormJobs {
  const void* g[kNormJobs];
  unsigned n[kNormJobs];
  unsigned upto[kNormJobs];  // its upper bit: bf16
};

// Squares are added up in 64 bits: their rate is a fraction of memory's here, no gradient that fp32 holds overflows, and nothing is lost to the length.
__global__ __launch_bounds__(256) void square_sums_kernel(NormJobs by_value, unsigned count, double* partial) {
  const NormJobs* jobs = arguments<NormJobs>();
  const unsigned lane = threadIdx.x & 63, piece = blockIdx.x;
  const int j = tensor_of<kNormJobs>(jobs->upto, count, piece, 0x7fffffffu);
  const unsigned first = (piece - (j ? jobs->upto[j - 1] & 0x7fffffffu : 0u)) * kNormPiece, n = jobs->n[j];
  const void* g = jobs->g[j];
  double sums[4] = {0.0, 0.0, 0.0, 0.0};
  auto add = [&](auto type, auto full) {
    typedef decltype(type) T;
    constexpr int E = 16 / (int)sizeof(T), kLoads = kNormPiece / (256 * E);
#pragma unroll
    for (int k = 0; k < kLoads; k += 4) {
      float x[4][E];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const unsigned i = first + ((k + q) * 256 + threadIdx.x) * E;
        Some<T>::template load<E, false>(g, i, decltype(full)::value ? E : i < n ? (int)min(n - i, (unsigned)E) : 0, x[q]);
      }
#pragma unroll
      for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int e = 0; e < E; ++e) sums[q] = fma((double)x[q][e], (double)x[q][e], sums[q]);
    }
  };
  const bool bf16 = jobs->upto[j] >> 31;
  if (first + kNormPiece <= n) {
    if (bf16) add(uint16_t{}, std::true_type{});
    else add(float{}, std::true_type{});
  } else {
    if (bf16) add(uint16_t{}, std::false_type{});
    else add(float{}, std::false_type{});
  }
  double sum = (sums[0] + sums[1]) + (sums[2] + sums[3]);
#pragma unroll
  for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
  __shared__ double part[4];
  if (lane == 0) part[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x == 0) partial[piece] = (part[0] + part[1]) + (part[2] + part[3]);
}

__global__ __launch_bounds__(1024) void norm_kernel(const double* partial, unsigned pieces, float max_norm, float* norm, float* scale) {
  double sum = 0.0;
  for (unsigned i = threadIdx.x; i < pieces; i += 1024) sum += partial[i];
#pragma unroll
  for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
  __shared__ double part[16];
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int k = 1; k < 16; ++k) sum += part[k];
    const float r = (float)sqrt(sum);
    *norm = r;
    if (scale) *scale = r < __builtin_inff() ? fminf(1.f, max_norm / (r + 1e-6f)) : __builtin_nanf("");
  }
}

}  // namespace

size_t grad_norm_workspace(const long long* n, int count) {
  size_t pieces = 0;
  for (int j = 0; j < count; ++j) pieces += (size_t)((n[j] + kNormPiece - 1) / kNormPiece);
  return (pieces ? pieces : 1) * sizeof(double);
}

int launch_grad_norm(const void* const* g, const long long* n, const int* dtype, int count, float max_norm, float* norm, float* scale, void* workspace,
                     hipStream_t stream) {
  double* partial = static_cast<double*>(workspace);
  size_t done = 0;
  NormJobs jobs;
  unsigned used = 0, pieces = 0;
  auto flush = [&]() {
    if (!used) return true;
    hipLaunchKernelGGL(square_sums_kernel, dim3(pieces), dim3(256), 0, stream, jobs, used, partial + done);
    done += pieces, used = pieces = 0;
    return hipGetLastError() == hipSuccess;
  };
  constexpr long long kMost = 1LL << 30;  // elements of one entry: larger tensors take several
  for (int j = 0; j < count; ++j) {
    const size_t size = dtype[j] == VIG_BF16 ? 2 : 4;
    for (long long at = 0; at < n[j]; at += kMost) {
      const unsigned part = (unsigned)(n[j] - at < kMost ? n[j] - at : kMost);
      const unsigned more = (part + kNormPiece - 1) / kNormPiece;
      if (used == kNormJobs || pieces + more > kMostPieces) {
        if (!flush()) return VIG_ELAUNCH;
      }
      pieces += more;
      jobs.g[used] = static_cast<const char*>(g[j]) + at * size, jobs.n[used] = part;
      jobs.upto[used++] = pieces | (dtype[j] == VIG_BF16 ? 0x80000000u : 0u);
    }
  }
  if (!flush()) return VIG_ELAUNCH;
  hipLaunchKernelGGL(norm_kernel, dim3(1), dim3(1024), 0, stream, partial, (unsigned)done, max_norm, norm, scale);
  return hipGetLastError() == hipSuccess ? VIG_OK : VIG_ELAUNCH;
}

template <bool BITS8>
static int launch_adamw_of(const AdamW& a, hipStream_t stream) {
  const double t = (double)a.step;
  UpdateScalars s;
  s.keep = (float)(1.0 - a.lr * a.weight_decay), s.step = (float)(a.lr / (1.0 - pow(a.beta1, t))), s.rs2 = (float)(1.0 / sqrt(1.0 - pow(a.beta2, t)));
  s.b1 = (float)a.beta1, s.c1 = (float)(1.0 - a.beta1), s.b2 = (float)a.beta2, s.c2 = (float)(1.0 - a.beta2), s.eps = (float)a.eps;
  const UpdateOnDevice dev{a.step_on_device, a.lr_on_device, a.beta1, a.beta2, (float)a.lr, (float)a.weight_decay, a.step};
  const uint32_t key = key_of(a.seed, a.step);
  constexpr long long kMost = 1LL << 30;
  // one launch takes tensors of one pair of types
  for (int types = 0; types < 4; ++types) {
    UpdateJobs<BITS8> jobs;
    unsigned used = 0, pieces = 0;
    unsigned long long from = 0;  // number of the launch's first element
    auto flush = [&]() {
      if (!used) return true;
      auto start = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(pieces), dim3(256), 0, stream, jobs, s, a.grad_scale, used, key, a.seed, from, dev); };
      if (types == 0) start(adamw_kernel<float, float, BITS8>);
      else if (types == 1) start(adamw_kernel<float, uint16_t, BITS8>);
      else if (types == 2) start(adamw_kernel<uint16_t, float, BITS8>);
      else start(adamw_kernel<uint16_t, uint16_t, BITS8>);
      used = pieces = 0;
      return hipGetLastError() == hipSuccess;
    };
    unsigned long long block = 0;
    for (int j = 0; j < a.count; ++j) {
      const bool mine = (a.param_dtype[j] == VIG_BF16) * 2 + (a.grad_dtype[j] == VIG_BF16) == types;
      const size_t sp = a.param_dtype[j] == VIG_BF16 ? 2 : 4, sg = a.grad_dtype[j] == VIG_BF16 ? 2 : 4, sm = BITS8 ? 1 : 4;
      for (long long at = 0; mine && at < a.n[j]; at += kMost) {
        const unsigned part = (unsigned)(a.n[j] - at < kMost ? a.n[j] - at : kMost);
        const unsigned long long number = (a.first ? (unsigned long long)a.first[j] : 256 * block) + at;
        const unsigned more = (part + kPiece - 1) / kPiece;
        if (used == UpdateJobs<BITS8>::kMost || pieces + more > kMostPieces || (used && (number < from || number - from > 0xffffffffULL))) {
          if (!flush()) return VIG_ELAUNCH;
        }
        pieces += more;
        jobs.p[used] = static_cast<char*>(a.param[j]) + at * sp, jobs.g[used] = static_cast<const char*>(a.grad[j]) + at * sg;
        jobs.m[used] = static_cast<char*>(a.exp_avg[j]) + at * sm, jobs.v[used] = static_cast<char*>(a.exp_avg_sq[j]) + at * sm;
        if constexpr (BITS8) jobs.ms[used] = a.avg_scale[j] + at / 256, jobs.vs[used] = a.sq_scale[j] + at / 256;
        if (!used) from = number;
        jobs.n[used] = part, jobs.upto[used] = pieces, jobs.first[used++] = (unsigned)(number - from);
      }
      block += (unsigned long long)(a.n[j] + 255) / 256;
    }
    if (!flush()) return VIG_ELAUNCH;
  }
  return VIG_OK;
}

int launch_adamw(const AdamW& a, hipStream_t stream) { return a.state_bits == 8 ? launch_adamw_of<true>(a, stream) : launch_adamw_of<false>(a, stream); }

}  // namespace vig
