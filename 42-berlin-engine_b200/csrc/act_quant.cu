// act_quant.cu -- activation rows in 8 bits with a scale each: residual
// addition + RMSNorm (ec_op_add_rmsnorm_quant) and SwiGLU
// (ec_op_silu_mul_quant), the inputs of ec_op_gemm_w8a8.
//
//   h = x + r (rounded to the row's type);  y = h / sqrt(sum h^2 / n + eps) * w
//   y = g / (1 + exp(-g)) * u
//   amax = max |y|;  q = rint(y * (127 / amax));  scale = amax / 127
//
// One CTA per row; the row stays in shared memory as f32 between the passes.
#include "typed.cuh"

namespace ec {
namespace {

constexpr int kThr = 256;
constexpr int kMaxN = 57344;  // f32 row: 224 KB of shared memory

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

template <typename T, typename Op>
__device__ T block_all(T v, T* red, Op op) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  T t = red[0];
  for (int i = 1; i < kThr / 32; i++) t = op(t, red[i]);
  return t;
}

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

// the row ys in shared memory -> 8 bits (factor 0: all zero, whatever ys holds)
__device__ void store_row(const float* ys, int n, unsigned amax_bits, int8_t* q, float* scale) {
  float sc;
  const float f = quant_factor(amax_bits, &sc);
  for (int i = threadIdx.x; i < n; i += kThr)
    q[i] = f != 0.0f ? (int8_t)__float2int_rn(__fmul_rn(ys[i], f)) : (int8_t)0;
  if (threadIdx.x == 0) *scale = sc;
}

template <typename T>
__global__ void __launch_bounds__(kThr) add_rmsnorm_quant_kernel(NormArgs a) {
  extern __shared__ __align__(16) float ys[];
  __shared__ float red[kThr / 32];
  __shared__ unsigned redu[kThr / 32];
  const long row = blockIdx.x;
  const T* x = static_cast<const T*>(a.x) + row * a.ldx;
  const T* r = a.r ? static_cast<const T*>(a.r) + row * a.ldr : nullptr;
  T* h = a.h ? static_cast<T*>(a.h) + row * a.ldh : nullptr;
  float ss = 0.0f;
  for (int i = threadIdx.x; i < a.n; i += kThr) {
    T v = x[i];
    if (r) v = from_f32<T>(__fadd_rn(to_f32(v), to_f32(r[i])));
    if (h) h[i] = v;
    const float f = to_f32(v);
    ys[i] = f;
    ss = __fmaf_rn(f, f, ss);
  }
  ss = block_all(ss, red, [](float p, float q) { return __fadd_rn(p, q); });
  float inv = __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(__fdiv_rn(ss, (float)a.n), a.eps)));
  if (ss == INFINITY) inv = __uint_as_float(0x7fc00000u);  // not a silent row of zeros
  unsigned m = 0;
  for (int i = threadIdx.x; i < a.n; i += kThr) {
    float y = __fmul_rn(ys[i], inv);
    if (a.w) y = __fmul_rn(y, bf16_to_f32(a.w[i]));
    ys[i] = y;
    m = max(m, __float_as_uint(fabsf(y)));
  }
  m = block_all(m, redu, [](unsigned p, unsigned q) { return max(p, q); });
  store_row(ys, a.n, m, a.q + row * a.ldq, a.scale + row);
}

template <typename T>
__global__ void __launch_bounds__(kThr) silu_mul_quant_kernel(SiluArgs a) {
  extern __shared__ __align__(16) float ys[];
  __shared__ unsigned redu[kThr / 32];
  const long row = blockIdx.x;
  const T* g = static_cast<const T*>(a.g) + row * a.ld;
  const T* u = static_cast<const T*>(a.u) + row * a.ld;
  unsigned m = 0;
  for (int i = threadIdx.x; i < a.n; i += kThr) {
    const float gv = to_f32(g[i]);
    const float y = __fmul_rn(__fdiv_rn(gv, __fadd_rn(1.0f, expf(-gv))), to_f32(u[i]));
    ys[i] = y;
    m = max(m, __float_as_uint(fabsf(y)));
  }
  m = block_all(m, redu, [](unsigned p, unsigned q) { return max(p, q); });
  store_row(ys, a.n, m, a.q + row * a.ldq, a.scale + row);
}

template <typename Kern, typename Args>
int launch_rows(Kern kern, const Args& a, int rows, cudaStream_t st) {
  const size_t smem = (size_t)a.n * 4;
  EC_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  kern<<<rows, kThr, smem, st>>>(a);
  EC_CUDA_TRY(cudaGetLastError());
  return EC_OK;
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
    return ec::launch_rows(ec::add_rmsnorm_quant_kernel<decltype(t)>, a, rows,
                           static_cast<cudaStream_t>(stream));
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
    return ec::launch_rows(ec::silu_mul_quant_kernel<decltype(t)>, a, rows,
                           static_cast<cudaStream_t>(stream));
  });
}
