// act_quant.cu -- activation rows in 8 bits with a scale each: residual
// addition + RMSNorm (ec_op_add_rmsnorm_quant) and SwiGLU
// (ec_op_silu_mul_quant), the inputs of ec_op_gemm_w8a8.
//
//   h = x + r (rounded to the row's type);  y = h / sqrt(sum h^2 / n + eps) * w
//   y = g / (1 + exp(-g)) * u
//   amax = max |y|;  q = rint(y * (127 / amax));  scale = amax / 127
//
// Bytes bound both (3 or 4 passes over a row's memory for two operations a
// byte), so a row is read once and held on chip until its scale is known:
// one CTA per row, kF values a thread in registers (rows_kernel), 16 bytes a
// load, several rows' CTAs on an SM to cover one another's reductions.
// Rows past 1024 threads' registers stay in shared memory instead
// (wide_kernel).
#include "typed.cuh"

namespace ec {
namespace {

constexpr int kMaxN = 57344;       // wide_kernel: f32 row, 224 KB of shared memory
constexpr int kMaxThr = 1024;
constexpr int kWideThr = 1024;

struct NormArgs {
  const void* x;
  const void* r;
  void* h;
  long ldx, ldr, ldh;
  const uint16_t* w;
  float eps;
  int n;
  int8_t* q;
  long ldq;
  float* scale;
};

struct SiluArgs {
  const void* g;
  const void* u;
  long ld;
  int n;
  int8_t* q;
  long ldq;
  float* scale;
};

// ------------------------------------------------------------ the 8-bit rule --

// The row's 8-bit factor and scale from amax' bits: as unsigned integers
// the bit patterns of |y| order like the values, infinities and NaN above
// all finite ones, so neither is lost in the maximum.
__device__ __forceinline__ float quant_factor(unsigned amax_bits, float* scale) {
  const float amax = __uint_as_float(amax_bits);
  if (amax_bits >= 0x7f800000u) {
    *scale = __uint_as_float(0x7fc00000u);
    return 0.0f;
  }
  if (amax < 0x1p-100f) {
    *scale = 1.0f;
    return 0.0f;
  }
  *scale = __fdiv_rn(amax, 127.0f);
  return __fdiv_rn(127.0f, amax);
}

// y * f rounded to the nearest integer, ties to even, in the low byte: the
// one rounding of the sum with 1.5 * 2^23, whose unit is 1 (|y * f| <= 127
// and a rounding of it).  f = 0 marks a row of zeros, whatever y holds.
__device__ __forceinline__ unsigned quant_byte(float y, float f) {
  return __float_as_uint(__fmaf_rn(y, f, 12582912.0f)) & 0xffu;
}
__device__ __forceinline__ unsigned quant4(const float* y, float f) {
  const unsigned a = __float_as_uint(__fmaf_rn(y[0], f, 12582912.0f));
  const unsigned b = __float_as_uint(__fmaf_rn(y[1], f, 12582912.0f));
  const unsigned c = __float_as_uint(__fmaf_rn(y[2], f, 12582912.0f));
  const unsigned d = __float_as_uint(__fmaf_rn(y[3], f, 12582912.0f));
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

__device__ __forceinline__ unsigned abs_bits(float y) { return __float_as_uint(y) & 0x7fffffffu; }

// ---------------------------------------------------------------- row sources --

// the statistics of a block: one barrier, then every warp joins the warps'
// values in the same tree
__device__ __forceinline__ float block_sum(float v, float* red) {
  const int lane = threadIdx.x & 31, warps = (blockDim.x + 31) >> 5;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = __fadd_rn(v, __shfl_xor_sync(0xffffffffu, v, o));
  if (lane == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = lane < warps ? red[lane] : 0.0f;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = __fadd_rn(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

__device__ __forceinline__ unsigned block_max(unsigned v, unsigned* red) {
  const int lane = threadIdx.x & 31, warps = (blockDim.x + 31) >> 5;
  v = __reduce_max_sync(0xffffffffu, v);
  if (lane == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  return __reduce_max_sync(0xffffffffu, lane < warps ? red[lane] : 0u);
}

// 1 / sqrt(sum / n + eps).  A sum past f32's range gives NaN, not a silent row
// of zeros.
__device__ __forceinline__ float norm_factor(float ss, int n, float eps) {
  const float inv = __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(__fdiv_rn(ss, (float)n), eps)));
  return ss == INFINITY ? __uint_as_float(0x7fc00000u) : inv;
}

// g * u / (1 + exp(-g)): the exponential and the reciprocal are the
// hardware's approximations (2 units each of f32 rounding), the argument's
// rounding adds |g| units of it
__device__ __forceinline__ float silu_mul(float g, float u) {
  float e, s;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(__fmul_rn(g, -1.44269504f)));
  asm("rcp.approx.f32 %0, %1;" : "=f"(s) : "f"(__fadd_rn(1.0f, e)));
  return __fmul_rn(__fmul_rn(g, s), u);
}

// N elements of T from 16 aligned bytes (N * sizeof(T) = 16) or 8, as f32
template <typename T, int N>
__device__ __forceinline__ void unpack(const void* p, float* v) {
  static_assert(N * sizeof(T) == 16 || N * sizeof(T) == 8, "one load");
  if constexpr (N * sizeof(T) == 16) {
    // a plain load: the row may be written in place (sum_out = x)
    const uint4 raw = *static_cast<const uint4*>(p);
    const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = to_f32(e[i]);
  } else {
    const uint2 raw = *static_cast<const uint2*>(p);
    const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = to_f32(e[i]);
  }
}

// A thread's part of a row: kF values.  VEC: runs of one 16-byte load (kPer
// elements), every kPer * blockDim.x apart; else single elements, blockDim.x
// apart, so that a warp's accesses are contiguous at any alignment.
template <typename T, int F, bool VEC>
struct Part {
  static constexpr int kPer = VEC ? 16 / (int)sizeof(T) : 1;
  static constexpr int kRuns = F / kPer;
  static __device__ __forceinline__ int at(int run) {
    return (run * (int)blockDim.x + (int)threadIdx.x) * kPer;
  }
  static __device__ __forceinline__ void load(const T* row, int i, float* v) {
    if constexpr (VEC)
      unpack<T, kPer>(row + i, v);
    else
      v[0] = to_f32(row[i]);
  }
  static __device__ __forceinline__ void store(T* row, int i, const float* v) {
    if constexpr (VEC) {
      uint4 raw;
      T* e = reinterpret_cast<T*>(&raw);
#pragma unroll
      for (int k = 0; k < kPer; k++) e[k] = from_f32<T>(v[k]);
      *reinterpret_cast<uint4*>(row + i) = raw;
    } else {
      row[i] = from_f32<T>(v[0]);
    }
  }
  // y (F values) -> 8 bits
  static __device__ __forceinline__ void quantise(const float* y, int n, unsigned amax_bits,
                                                  int8_t* q, float* scale) {
    float sc;
    const float f = quant_factor(amax_bits, &sc);
    if (threadIdx.x == 0) *scale = sc;
#pragma unroll
    for (int run = 0; run < kRuns; run++) {
      const int i = at(run);
      if (i < n) {
        const float* v = y + run * kPer;
        if constexpr (!VEC) {
          q[i] = f != 0.0f ? (int8_t)quant_byte(v[0], f) : (int8_t)0;
        } else if constexpr (kPer == 8) {
          *reinterpret_cast<uint2*>(q + i) =
              f != 0.0f ? make_uint2(quant4(v, f), quant4(v + 4, f)) : make_uint2(0, 0);
        } else {
          *reinterpret_cast<unsigned*>(q + i) = f != 0.0f ? quant4(v, f) : 0u;
        }
      }
    }
  }
};

// --------------------------------------------------------------- the kernels --

template <typename T, int F, bool VEC>
__global__ void __launch_bounds__(kMaxThr) norm_rows_kernel(NormArgs a) {
  using P = Part<T, F, VEC>;
  __shared__ float red[32];
  __shared__ unsigned redu[32];
  pdl_wait();
  pdl_launch_dependents();
  const long row = blockIdx.x;
  const T* x = static_cast<const T*>(a.x) + row * a.ldx;
  const T* r = a.r ? static_cast<const T*>(a.r) + row * a.ldr : nullptr;
  T* h = a.h ? static_cast<T*>(a.h) + row * a.ldh : nullptr;
  float v[F];
#pragma unroll
  for (int run = 0; run < P::kRuns; run++) {
    const int i = P::at(run);
#pragma unroll
    for (int k = 0; k < P::kPer; k++) v[run * P::kPer + k] = 0.0f;
    if (i < a.n) P::load(x, i, v + run * P::kPer);
  }
  if (r) {
#pragma unroll
    for (int run = 0; run < P::kRuns; run++) {
      const int i = P::at(run);
      if (i < a.n) {
        float b[P::kPer];
        P::load(r, i, b);
#pragma unroll
        for (int k = 0; k < P::kPer; k++)
          v[run * P::kPer + k] = to_f32(from_f32<T>(__fadd_rn(v[run * P::kPer + k], b[k])));
      }
    }
  }
  float ss = 0.0f;
#pragma unroll
  for (int k = 0; k < F; k++) ss = __fmaf_rn(v[k], v[k], ss);
  if (h) {
#pragma unroll
    for (int run = 0; run < P::kRuns; run++) {
      const int i = P::at(run);
      if (i < a.n) P::store(h, i, v + run * P::kPer);
    }
  }
  const float inv = norm_factor(block_sum(ss, red), a.n, a.eps);
  unsigned m = 0;
#pragma unroll
  for (int run = 0; run < P::kRuns; run++) {
    const int i = P::at(run);
    if (i < a.n) {
      float w[P::kPer];
#pragma unroll
      for (int k = 0; k < P::kPer; k++) w[k] = 1.0f;
      if (a.w) {
        if constexpr (VEC)
          unpack<__nv_bfloat16, P::kPer>(a.w + i, w);
        else
          w[0] = bf16_to_f32(a.w[i]);
      }
#pragma unroll
      for (int k = 0; k < P::kPer; k++) {
        float& y = v[run * P::kPer + k];
        y = __fmul_rn(__fmul_rn(y, inv), w[k]);
        m = max(m, abs_bits(y));
      }
    }
  }
  P::quantise(v, a.n, block_max(m, redu), a.q + row * a.ldq, a.scale + row);
}

template <typename T, int F, bool VEC>
__global__ void __launch_bounds__(kMaxThr) silu_rows_kernel(SiluArgs a) {
  using P = Part<T, F, VEC>;
  __shared__ unsigned redu[32];
  pdl_wait();
  pdl_launch_dependents();
  const long row = blockIdx.x;
  const T* g = static_cast<const T*>(a.g) + row * a.ld;
  const T* u = static_cast<const T*>(a.u) + row * a.ld;
  float v[F];
  unsigned m = 0;
#pragma unroll
  for (int run = 0; run < P::kRuns; run++) {
    const int i = P::at(run);
#pragma unroll
    for (int k = 0; k < P::kPer; k++) v[run * P::kPer + k] = 0.0f;
    if (i < a.n) {
      float gv[P::kPer], uv[P::kPer];
      P::load(g, i, gv);
      P::load(u, i, uv);
#pragma unroll
      for (int k = 0; k < P::kPer; k++) {
        const float y = silu_mul(gv[k], uv[k]);
        v[run * P::kPer + k] = y;
        m = max(m, abs_bits(y));
      }
    }
  }
  P::quantise(v, a.n, block_max(m, redu), a.q + row * a.ldq, a.scale + row);
}

// Rows of more than 32 x 1024 values: f32 in shared memory.
__device__ void quantise_wide(const float* ys, int n, unsigned amax_bits, int8_t* q,
                              float* scale) {
  float sc;
  const float f = quant_factor(amax_bits, &sc);
  for (int i = threadIdx.x; i < n; i += kWideThr)
    q[i] = f != 0.0f ? (int8_t)quant_byte(ys[i], f) : (int8_t)0;
  if (threadIdx.x == 0) *scale = sc;
}

template <typename T>
__global__ void __launch_bounds__(kWideThr) norm_wide_kernel(NormArgs a) {
  extern __shared__ __align__(16) float ys[];
  __shared__ float red[32];
  __shared__ unsigned redu[32];
  pdl_wait();
  pdl_launch_dependents();
  const long row = blockIdx.x;
  const T* x = static_cast<const T*>(a.x) + row * a.ldx;
  const T* r = a.r ? static_cast<const T*>(a.r) + row * a.ldr : nullptr;
  T* h = a.h ? static_cast<T*>(a.h) + row * a.ldh : nullptr;
  float ss = 0.0f;
  for (int i = threadIdx.x; i < a.n; i += kWideThr) {
    T v = x[i];
    if (r) v = from_f32<T>(__fadd_rn(to_f32(v), to_f32(r[i])));
    if (h) h[i] = v;
    const float f = to_f32(v);
    ys[i] = f;
    ss = __fmaf_rn(f, f, ss);
  }
  const float inv = norm_factor(block_sum(ss, red), a.n, a.eps);
  unsigned m = 0;
  for (int i = threadIdx.x; i < a.n; i += kWideThr) {  // the elements it stored itself
    float y = __fmul_rn(ys[i], inv);
    if (a.w) y = __fmul_rn(y, bf16_to_f32(a.w[i]));
    ys[i] = y;
    m = max(m, abs_bits(y));
  }
  quantise_wide(ys, a.n, block_max(m, redu), a.q + row * a.ldq, a.scale + row);
}

template <typename T>
__global__ void __launch_bounds__(kWideThr) silu_wide_kernel(SiluArgs a) {
  extern __shared__ __align__(16) float ys[];
  __shared__ unsigned redu[32];
  pdl_wait();
  pdl_launch_dependents();
  const long row = blockIdx.x;
  const T* g = static_cast<const T*>(a.g) + row * a.ld;
  const T* u = static_cast<const T*>(a.u) + row * a.ld;
  unsigned m = 0;
  for (int i = threadIdx.x; i < a.n; i += kWideThr) {
    const float y = silu_mul(to_f32(g[i]), to_f32(u[i]));
    ys[i] = y;
    m = max(m, abs_bits(y));
  }
  quantise_wide(ys, a.n, block_max(m, redu), a.q + row * a.ldq, a.scale + row);
}

// ------------------------------------------------------------------- launches --

template <typename Args>
int launch(void (*kern)(Args), const Args& a, int rows, int threads, size_t smem,
           cudaStream_t st) {
  if (smem > 48 * 1024)
    EC_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(rows);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  EC_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, a));
  return EC_OK;
}

// Values a thread holds: 8 while the rows are few (more threads a row hide the
// latency), else 16 or 32.
inline int values_per_thread(int rows, int n) {
  int f = rows < 148 * 2 ? 8 : 16;
  while (f < 32 && n > f * kMaxThr) f *= 2;
  return f;
}
inline int threads_for(int n, int f) { return ((n + f - 1) / f + 31) / 32 * 32; }

inline bool aligned(const void* p, long ld, size_t esize, size_t to) {
  return (reinterpret_cast<uintptr_t>(p) % to) == 0 && ((size_t)ld * esize) % to == 0;
}

template <typename T>
int norm_rows(const NormArgs& a, int rows, cudaStream_t st) {
  constexpr int per = 16 / (int)sizeof(T);
  const int f = values_per_thread(rows, a.n);
  if (a.n > f * kMaxThr) return launch(norm_wide_kernel<T>, a, rows, kWideThr, (size_t)a.n * 4, st);
  const bool vec = a.n % per == 0 && aligned(a.x, a.ldx, sizeof(T), 16) &&
                   (!a.r || aligned(a.r, a.ldr, sizeof(T), 16)) &&
                   (!a.h || aligned(a.h, a.ldh, sizeof(T), 16)) &&
                   (!a.w || aligned(a.w, 0, 2, 2 * per)) && aligned(a.q, a.ldq, 1, per);
  void (*kern)(NormArgs) =
      vec ? (f == 8 ? norm_rows_kernel<T, 8, true>
                    : f == 16 ? norm_rows_kernel<T, 16, true> : norm_rows_kernel<T, 32, true>)
          : (f == 8 ? norm_rows_kernel<T, 8, false>
                    : f == 16 ? norm_rows_kernel<T, 16, false> : norm_rows_kernel<T, 32, false>);
  return launch(kern, a, rows, threads_for(a.n, f), 0, st);
}

template <typename T>
int silu_rows(const SiluArgs& a, int rows, cudaStream_t st) {
  constexpr int per = 16 / (int)sizeof(T);
  const int f = values_per_thread(rows, a.n);
  if (a.n > f * kMaxThr) return launch(silu_wide_kernel<T>, a, rows, kWideThr, (size_t)a.n * 4, st);
  const bool vec = a.n % per == 0 && aligned(a.g, a.ld, sizeof(T), 16) &&
                   aligned(a.u, a.ld, sizeof(T), 16) && aligned(a.q, a.ldq, 1, per);
  void (*kern)(SiluArgs) =
      vec ? (f == 8 ? silu_rows_kernel<T, 8, true>
                    : f == 16 ? silu_rows_kernel<T, 16, true> : silu_rows_kernel<T, 32, true>)
          : (f == 8 ? silu_rows_kernel<T, 8, false>
                    : f == 16 ? silu_rows_kernel<T, 16, false> : silu_rows_kernel<T, 32, false>);
  return launch(kern, a, rows, threads_for(a.n, f), 0, st);
}

}  // namespace
}  // namespace ec

extern "C" int ec_op_add_rmsnorm_quant(int type, const void* x, int64_t ldx, const void* residual,
                                       int64_t ldr, void* sum_out, int64_t lds, const uint16_t* w,
                                       float eps, int rows, int n, int8_t* q, int64_t ldq,
                                       float* scales, void* stream) {
  if (!ec::known_type(type)) return ec::arg_error("ec_op_add_rmsnorm_quant: unknown type");
  if (!x || !q || !scales || rows <= 0 || n <= 0 || !(eps >= 0.0f))
    return ec::arg_error("ec_op_add_rmsnorm_quant: null pointer, empty shape or negative eps");
  if (ldx < n || ldq < n || (residual && ldr < n) || (sum_out && lds < n))
    return ec::arg_error("ec_op_add_rmsnorm_quant: a row stride is shorter than the row");
  if (n > ec::kMaxN) return ec::unsupported("ec_op_add_rmsnorm_quant: n > 57344");
  const ec::NormArgs a{x, residual, sum_out, (long)ldx, (long)ldr, (long)lds, w, eps, n,
                       q, (long)ldq, scales};
  return ec::with_type(type, [&](auto t) {
    return ec::norm_rows<decltype(t)>(a, rows, static_cast<cudaStream_t>(stream));
  });
}

extern "C" int ec_op_silu_mul_quant(int type, const void* gate, const void* up, int64_t ld,
                                    int rows, int n, int8_t* q, int64_t ldq, float* scales,
                                    void* stream) {
  if (!ec::known_type(type)) return ec::arg_error("ec_op_silu_mul_quant: unknown type");
  if (!gate || !up || !q || !scales || rows <= 0 || n <= 0)
    return ec::arg_error("ec_op_silu_mul_quant: null pointer or empty shape");
  if (ld < n || ldq < n)
    return ec::arg_error("ec_op_silu_mul_quant: a row stride is shorter than the row");
  if (n > ec::kMaxN) return ec::unsupported("ec_op_silu_mul_quant: n > 57344");
  const ec::SiluArgs a{gate, up, (long)ld, n, q, (long)ldq, scales};
  return ec::with_type(type, [&](auto t) {
    return ec::silu_rows<decltype(t)>(a, rows, static_cast<cudaStream_t>(stream));
  });
}
