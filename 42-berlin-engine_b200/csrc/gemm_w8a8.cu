// gemm_w8a8.cu -- INT8 activation rows times INT8 weights, a scale for each
// token and each channel (ec_op_gemm_w8a8).
//
//   y[t][c] = (x_scale[t] * sum_k x[t][k] w[c][k]) * w_scale[c]
//
// A 64 x 64 tile per CTA from shared memory, four byte products an instruction.
#include "typed.cuh"

namespace ec {
namespace {

constexpr int kMaxK = 131071;  // 128 * 128 * k < 2^31

struct W8A8Args {
  const int8_t* x;
  const int8_t* w;
  const float* sx;
  const float* sw;
  void* y;
  long ldx, ldw, ldy;
  int m, k, nb;
  int* status;
};

__device__ __forceinline__ int load4(const int8_t* row, int k0, int k) {
  if (k0 + 4 <= k) return *reinterpret_cast<const int*>(row + k0);
  unsigned v = 0;
  for (int i = 0; i < 4; i++)
    if (k0 + i < k) v |= (unsigned)(uint8_t)row[k0 + i] << (8 * i);
  return (int)v;
}

template <typename T>
__global__ void __launch_bounds__(256) gemm_w8a8_kernel(W8A8Args a) {
  __shared__ int xs[64][17], ws[64][17];
  const int c0 = blockIdx.x * 64, t0 = blockIdx.y * 64;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  int acc[4][4] = {};
  for (int k0 = 0; k0 < a.k; k0 += 64) {
    __syncthreads();
    for (int i = threadIdx.x; i < 64 * 16; i += 256) {
      const int r = i >> 4, kk = (i & 15) * 4;
      xs[r][i & 15] = t0 + r < a.nb ? load4(a.x + (t0 + r) * a.ldx, k0 + kk, a.k) : 0;
      ws[r][i & 15] = c0 + r < a.m ? load4(a.w + (c0 + r) * a.ldw, k0 + kk, a.k) : 0;
    }
    __syncthreads();
    for (int kk = 0; kk < 16; kk++)
#pragma unroll
      for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++)
          acc[i][j] = __dp4a(xs[ty + 16 * i][kk], ws[tx + 16 * j][kk], acc[i][j]);
  }
  for (int i = 0; i < 4; i++)
    for (int j = 0; j < 4; j++) {
      const int t = t0 + ty + 16 * i, c = c0 + tx + 16 * j;
      if (t < a.nb && c < a.m)
        static_cast<T*>(a.y)[t * a.ldy + c] =
            from_f32<T>(__fmul_rn(__fmul_rn((float)acc[i][j], a.sx[t]), a.sw[c]));
    }
}

}  // namespace
}  // namespace ec

extern "C" int ec_op_gemm_w8a8(const int8_t* x, int64_t ldx, const float* x_scale, const int8_t* w,
                               int64_t ldw, const float* w_scale, int type, void* y, int64_t ldy,
                               int m, int k, int nb, int* status, void* stream) {
  if (!ec::known_type(type)) return ec::arg_error("ec_op_gemm_w8a8: unknown type");
  if (!x || !x_scale || !w || !w_scale || !y || m <= 0 || k <= 0 || nb <= 0)
    return ec::arg_error("ec_op_gemm_w8a8: null pointer or empty shape");
  if (ldx < k || ldw < k || ldy < m)
    return ec::arg_error("ec_op_gemm_w8a8: a row stride is shorter than the row");
  if ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(w) | (uintptr_t)ldx |
       (uintptr_t)ldw) & 15)
    return ec::arg_error("ec_op_gemm_w8a8: x, w, ldx and ldw must be multiples of 16 bytes");
  if (k > ec::kMaxK) return ec::unsupported("ec_op_gemm_w8a8: k > 131071");
  const ec::W8A8Args a{x, w, x_scale, w_scale, y, (long)ldx, (long)ldw, (long)ldy, m, k, nb, status};
  const dim3 grid((m + 63) / 64, (nb + 63) / 64);
  if (grid.y > 65535) return ec::unsupported("ec_op_gemm_w8a8: too many rows");
  return ec::with_type(type, [&](auto t) {
    ec::gemm_w8a8_kernel<decltype(t)>
        <<<grid, 256, 0, static_cast<cudaStream_t>(stream)>>>(a);
    EC_CUDA_TRY(cudaGetLastError());
    return EC_OK;
  });
}
