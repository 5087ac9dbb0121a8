// What a training step does to a list of tensors: the norm of all gradients, and AdamW with its moments in 32 or in 8 bits.
//
//   norm = sqrt(sum g^2),  factor = min(1, max_norm / (norm + 1e-6))
//   g' = factor g;  m <- b1 m + (1 - b1) g';  v <- b2 v + (1 - b2) g'^2
//   p <- p (1 - lr decay) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// Both are bound by memory: every tensor is read once, what changes is written once, 16 bytes a lane.  A launch takes a table of tensors in its
// arguments (nothing is copied to the device, so that a captured launch holds all it needs); a workgroup takes one piece of 4096 elements
// (norm: 16384) and finds its tensor by comparing its number with the tensors' last pieces, one a lane.
//
// 8 bits: blocks of 256 elements, counted from each tensor's first, hold m and r = sqrt(v) as e4m3 values times a scale of max / 448.  (The root: v spans
// twice the octaves that e4m3 has.)  Rounding is stochastic: by the nearest value a moment would stand still, as a step of e4m3 is 6 to 12 % and b2 moves v
// by 0.1 %.  Parameters in bf16 are rounded the same way, for the same reason.  A positive r never becomes 0, which would divide by eps alone.
#include "common.h"
#include "launch.h"

namespace vig {
namespace {

constexpr int kPiece = 4096;       // elements of a workgroup: four a lane, four times
constexpr int kNormPiece = 16384;
constexpr int kUpdateJobs = 64;    // tensors of a launch: one a lane; the table stays under 4 KB
constexpr int kNormJobs = 192;

struct UpdateJobs {
  void* p[kUpdateJobs];
  const void* g[kUpdateJobs];
  void* m[kUpdateJobs];
  void* v[kUpdateJobs];
  float* ms[kUpdateJobs];
  float* vs[kUpdateJobs];
  unsigned n[kUpdateJobs];      // elements
  unsigned upto[kUpdateJobs];   // pieces up to and with this tensor's
  unsigned block[kUpdateJobs];  // number of the tensor's first block of 256 in the whole list
};
static_assert(sizeof(UpdateJobs) <= 3904, "a launch's arguments take 4 KB");

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

typedef u32x4_t u32x4_any __attribute__((aligned(4)));  // quads of tensors that begin anywhere
typedef u32x2_t u32x2_any __attribute__((aligned(2)));
typedef uint32_t u32_any __attribute__((aligned(1)));

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

template <typename T> struct Quad;
template <> struct Quad<float> {
  static __device__ __forceinline__ void load(const void* p, size_t i, int left, float (&x)[4]) {
    const float* at = static_cast<const float*>(p) + i;
    if (left >= 4) {
      const u32x4_t v = *reinterpret_cast<const u32x4_any*>(at);
#pragma unroll
      for (int k = 0; k < 4; ++k) x[k] = __uint_as_float(v[k]);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) x[k] = k < left ? at[k] : 0.f;
    }
  }
  static __device__ __forceinline__ void store(void* p, size_t i, int left, const float (&x)[4], const uint32_t (&)[4]) {
    float* at = static_cast<float*>(p) + i;
    if (left >= 4) {
      *reinterpret_cast<u32x4_any*>(at) = u32x4_t{__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3])};
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (k < left) at[k] = x[k];
    }
  }
};
template <> struct Quad<uint16_t> {
  static __device__ __forceinline__ void load(const void* p, size_t i, int left, float (&x)[4]) {
    const uint16_t* at = static_cast<const uint16_t*>(p) + i;
    if (left >= 4) {
      const u32x2_t v = *reinterpret_cast<const u32x2_any*>(at);
      x[0] = bf16lo_to_f32(v[0]), x[1] = bf16hi_to_f32(v[0]), x[2] = bf16lo_to_f32(v[1]), x[3] = bf16hi_to_f32(v[1]);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) x[k] = k < left ? bf16_to_f32(at[k]) : 0.f;
    }
  }
  // the upper half of x plus 16 random bits at its lower half: up with the probability that the cut part is of a step (NaN stays one)
  static __device__ __forceinline__ void store(void* p, size_t i, int left, const float (&x)[4], const uint32_t (&word)[4]) {
    uint16_t* at = static_cast<uint16_t*>(p) + i;
    uint32_t y[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) y[k] = x[k] == x[k] ? (__float_as_uint(x[k]) + ((word[k] * kGolden) >> 16)) >> 16 : 0x7fc0u;
    if (left >= 4) {
      *reinterpret_cast<u32x2_any*>(at) = u32x2_t{y[0] | y[1] << 16, y[2] | y[3] << 16};
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (k < left) at[k] = (uint16_t)y[k];
    }
  }
};

__device__ __forceinline__ void load_codes(const void* p, size_t i, int left, float scale, float (&x)[4]) {
  const uint8_t* at = static_cast<const uint8_t*>(p) + i;
  uint32_t w = 0;
  if (left >= 4) {
    w = *reinterpret_cast<const u32_any*>(at);
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (k < left) w |= (uint32_t)at[k] << (8 * k);
  }
  const f32x2_t lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  x[0] = lo[0] * scale, x[1] = lo[1] * scale, x[2] = hi[0] * scale, x[3] = hi[1] * scale;
}
__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
  for (int d = 32; d; d >>= 1) x = fmaxf(x, __shfl_xor(x, d));
  return x;
}
// The block's scale, and the codes of a lane's four values.  y = |x| / scale <= 448 (1 + 2^-22), whose step is 2^-20 of the power of two below it, 2^-9 under
// 2^-6: 16 random bits at the top of the cut part carry into the code.  A value that is not finite makes the scale so, and the block with it.
__device__ __forceinline__ float store_codes(void* p, size_t i, int left, const float (&x)[4], const uint32_t (&bits)[4], bool least) {
  float most = fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3])));
  // (the maximum drops a NaN: infinity stands for it)
#pragma unroll
  for (int k = 0; k < 4; ++k) most = x[k] == x[k] ? most : __builtin_inff();
  most = wave_max(most);
  float scale = most * (1.f / 448.f);
  scale = most > 0.f ? fmaxf(scale, 0x1p-126f) : 0.f;
  const float inv = most > 0.f ? 1.f / scale : 0.f;
  const bool fine = most < __builtin_inff();
  uint32_t code[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    // (a division's bits: the remainder of the quotient by the reciprocal, times it)
    const float near = fabsf(x[k]) * inv, y = fmaf(fmaf(-near, scale, fabsf(x[k])), inv, near);
    const uint32_t normal = ((__float_as_uint(y) + (bits[k] << 4)) >> 20) - (120u << 3);
    const uint32_t below = (uint32_t)floorf(fmaf(y, 512.f, (float)bits[k] * 0x1p-16f));
    uint32_t q = y >= 0x1p-6f ? normal : below;
    if (least && q == 0 && x[k] > 0.f) q = 1;
    code[k] = fine ? q | (__float_as_uint(x[k]) >> 31) << 7 : 0x7fu;
  }
  uint8_t* at = static_cast<uint8_t*>(p) + i;
  if (left >= 4) {
    *reinterpret_cast<u32_any*>(at) = code[0] | code[1] << 8 | code[2] << 16 | code[3] << 24;
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (k < left) at[k] = (uint8_t)code[k];
  }
  return scale;
}

// (the table is read through the kernel's argument pointer: an index into a by-value argument would copy it to scratch)
template <typename T>
__device__ __forceinline__ const T* arguments() {
  return (const T*)(const void*)__builtin_amdgcn_kernarg_segment_ptr();
}

template <typename TP, typename TG, bool BITS8>
__global__ __launch_bounds__(256) void adamw_kernel(UpdateJobs by_value, UpdateScalars s, const float* grad_scale, unsigned count, uint32_t key, unsigned long long seed,
                                                    UpdateOnDevice dev) {
  const UpdateJobs* jobs = arguments<UpdateJobs>();
  const unsigned lane = threadIdx.x & 63, piece = blockIdx.x;
  const int j = __builtin_amdgcn_readfirstlane(__popcll(__ballot(lane < count && jobs->upto[lane] <= piece)));
  const float clip = grad_scale ? *grad_scale : 1.f;
  if (clip != clip) return;  // the norm was not finite: everything stays as it is
  const unsigned first = (piece - (j ? jobs->upto[j - 1] : 0u)) * kPiece, n = jobs->n[j];
  void *const p = jobs->p[j], *const m = jobs->m[j], *const v = jobs->v[j];
  const void* const g = jobs->g[j];
  const unsigned block0 = jobs->block[j];
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
  float P[4][4], G[4][4], M[4][4], V[4][4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const unsigned i = first + k * 1024 + threadIdx.x * 4;
    const int left = i < n ? (int)min(n - i, 4u) : 0;
    Quad<TP>::load(p, i, left, P[k]);
    Quad<TG>::load(g, i, left, G[k]);
    if constexpr (BITS8) {
      const unsigned b = __builtin_amdgcn_readfirstlane(i >> 8);
      const bool some = b * 256u < n;
      const float ms = some ? jobs->ms[j][b] : 0.f, vs = some ? jobs->vs[j][b] : 0.f;
      load_codes(m, i, left, ms, M[k]);
      load_codes(v, i, left, vs, V[k]);
#pragma unroll
      for (int e = 0; e < 4; ++e) V[k][e] *= V[k][e];
    } else {
      Quad<float>::load(m, i, left, M[k]);
      Quad<float>::load(v, i, left, V[k]);
    }
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const unsigned i = first + k * 1024 + threadIdx.x * 4;
    const int left = i < n ? (int)min(n - i, 4u) : 0;
    float root[4];
    uint32_t word[4] = {0u, 0u, 0u, 0u};
    if constexpr (BITS8 || sizeof(TP) == 2) {
      // (numbers of elements in the whole list pass 32 bits: the upper ones go into the key)
      const unsigned long long number = (unsigned long long)block0 * 256u + i;
      const uint32_t k2 = key + (uint32_t)(number >> 32) * kGolden;
#pragma unroll
      for (int e = 0; e < 4; ++e) word[e] = mix(((uint32_t)number + e) ^ k2);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      // (products and sums rounded one by one: a last bit can turn a code over, and so the moments' bits are those of their formula)
#pragma clang fp contract(off)
      const float x = G[k][e] * clip;
      M[k][e] = s.b1 * M[k][e] + s.c1 * x;
      V[k][e] = s.b2 * V[k][e] + s.c2 * x * x;
      root[e] = sqrtf(V[k][e]);
      P[k][e] = fmaf(P[k][e], s.keep, -(s.step * M[k][e] / fmaf(root[e], s.rs2, s.eps)));
    }
    if constexpr (BITS8) {
      const unsigned b = __builtin_amdgcn_readfirstlane(i >> 8);
      uint32_t low[4], high[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        low[e] = word[e] & 0xffffu, high[e] = word[e] >> 16;
        if (e >= left) M[k][e] = root[e] = 0.f;
      }
      const float ms = store_codes(m, i, left, M[k], low, false), vs = store_codes(v, i, left, root, high, true);
      if (lane == 0 && b * 256u < n) jobs->ms[j][b] = ms, jobs->vs[j][b] = vs;
    } else {
      Quad<float>::store(m, i, left, M[k], word);
      Quad<float>::store(v, i, left, V[k], word);
    }
    Quad<TP>::store(p, i, left, P[k], word);
  }
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
  int j = 0;
  for (unsigned first = 0; first < count; first += 64) j += __popcll(__ballot(first + lane < count && (jobs->upto[first + lane] & 0x7fffffffu) <= piece));
  j = __builtin_amdgcn_readfirstlane(j);
  const unsigned first = (piece - (j ? jobs->upto[j - 1] & 0x7fffffffu : 0u)) * kNormPiece, n = jobs->n[j];
  const bool bf16 = jobs->upto[j] >> 31;
  const void* g = jobs->g[j];
  double sum = 0.0;
#pragma unroll 1
  for (int k = 0; k < kNormPiece / 4096; ++k) {
    float x[4][4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const unsigned i = first + k * 4096 + q * 1024 + threadIdx.x * 4;
      const int left = i < n ? (int)min(n - i, 4u) : 0;
      if (bf16) Quad<uint16_t>::load(g, i, left, x[q]);
      else Quad<float>::load(g, i, left, x[q]);
    }
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
      for (int e = 0; e < 4; ++e) sum = fma((double)x[q][e], (double)x[q][e], sum);
  }
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
      if (used == kNormJobs || pieces >= 0x10000000u) {
        if (!flush()) return VIG_ELAUNCH;
      }
      pieces += (part + kNormPiece - 1) / kNormPiece;
      jobs.g[used] = static_cast<const char*>(g[j]) + at * size, jobs.n[used] = part;
      jobs.upto[used++] = pieces | (dtype[j] == VIG_BF16 ? 0x80000000u : 0u);
    }
  }
  if (!flush()) return VIG_ELAUNCH;
  hipLaunchKernelGGL(norm_kernel, dim3(1), dim3(1024), 0, stream, partial, (unsigned)done, max_norm, norm, scale);
  return hipGetLastError() == hipSuccess ? VIG_OK : VIG_ELAUNCH;
}

template <typename TP, typename TG>
static void start(bool bits8, const UpdateJobs& jobs, unsigned pieces, unsigned used, const UpdateScalars& s, const AdamW& a, uint32_t key, const UpdateOnDevice& dev,
                  hipStream_t stream) {
  if (bits8) hipLaunchKernelGGL((adamw_kernel<TP, TG, true>), dim3(pieces), dim3(256), 0, stream, jobs, s, a.grad_scale, used, key, a.seed, dev);
  else hipLaunchKernelGGL((adamw_kernel<TP, TG, false>), dim3(pieces), dim3(256), 0, stream, jobs, s, a.grad_scale, used, key, a.seed, dev);
}

int launch_adamw(const AdamW& a, hipStream_t stream) {
  const bool bits8 = a.state_bits == 8;
  const double t = (double)a.step;
  UpdateScalars s;
  s.keep = (float)(1.0 - a.lr * a.weight_decay), s.step = (float)(a.lr / (1.0 - pow(a.beta1, t))), s.rs2 = (float)(1.0 / sqrt(1.0 - pow(a.beta2, t)));
  s.b1 = (float)a.beta1, s.c1 = (float)(1.0 - a.beta1), s.b2 = (float)a.beta2, s.c2 = (float)(1.0 - a.beta2), s.eps = (float)a.eps;
  const UpdateOnDevice dev{a.step_on_device, a.lr_on_device, a.beta1, a.beta2, (float)a.lr, (float)a.weight_decay, a.step};
  const uint32_t key = key_of(a.seed, a.step);
  constexpr long long kMost = 1LL << 30;
  // one launch takes tensors of one pair of types
  for (int types = 0; types < 4; ++types) {
    UpdateJobs jobs;
    unsigned used = 0, pieces = 0;
    auto flush = [&]() {
      if (!used) return true;
      if (types == 0) start<float, float>(bits8, jobs, pieces, used, s, a, key, dev, stream);
      else if (types == 1) start<float, uint16_t>(bits8, jobs, pieces, used, s, a, key, dev, stream);
      else if (types == 2) start<uint16_t, float>(bits8, jobs, pieces, used, s, a, key, dev, stream);
      else start<uint16_t, uint16_t>(bits8, jobs, pieces, used, s, a, key, dev, stream);
      used = pieces = 0;
      return hipGetLastError() == hipSuccess;
    };
    unsigned long long block = 0;
    for (int j = 0; j < a.count; ++j) {
      const bool mine = (a.param_dtype[j] == VIG_BF16) * 2 + (a.grad_dtype[j] == VIG_BF16) == types;
      const size_t sp = a.param_dtype[j] == VIG_BF16 ? 2 : 4, sg = a.grad_dtype[j] == VIG_BF16 ? 2 : 4, sm = bits8 ? 1 : 4;
      for (long long at = 0; mine && at < a.n[j]; at += kMost) {
        const unsigned part = (unsigned)(a.n[j] - at < kMost ? a.n[j] - at : kMost);
        if (used == kUpdateJobs || pieces >= 0x10000000u) {
          if (!flush()) return VIG_ELAUNCH;
        }
        pieces += (part + kPiece - 1) / kPiece;
        jobs.p[used] = static_cast<char*>(a.param[j]) + at * sp, jobs.g[used] = static_cast<const char*>(a.grad[j]) + at * sg;
        jobs.m[used] = static_cast<char*>(a.exp_avg[j]) + at * sm, jobs.v[used] = static_cast<char*>(a.exp_avg_sq[j]) + at * sm;
        jobs.ms[used] = bits8 ? a.avg_scale[j] + at / 256 : nullptr, jobs.vs[used] = bits8 ? a.sq_scale[j] + at / 256 : nullptr;
        jobs.n[used] = part, jobs.upto[used] = pieces, jobs.block[used++] = (unsigned)(block + at / 256);
      }
      block += (unsigned long long)(a.n[j] + 255) / 256;
    }
    if (!flush()) return VIG_ELAUNCH;
  }
  return VIG_OK;
}

}  // namespace vig
