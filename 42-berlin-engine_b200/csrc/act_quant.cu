// act_quant.cu -- activation rows in 8 bits with a scale each: residual
// addition + RMSNorm (ec_op_add_rmsnorm_quant) and SwiGLU
// (ec_op_silu_mul_quant), the inputs of ec_op_gemm_w8a8.
//
//   h = x + r (rounded to the row's type);  y = h / sqrt(sum h^2 / n + eps) * w
//   y = g / (1 + exp(-g)) * u
//   amax = max |y|;  q = rint(y * (127 / amax));  scale = amax / 127
//
// Bytes bound both (a few operations a byte), so a row is read once and held
// in registers, F values a thread, until its scale is known (rows_kernel).
// CTAs walk over rows; the next row is copied into shared memory while this
// one is reduced and stored, so loads stay under way through the reductions.
// Aligned rows: every thread copies and reads back its own 16-byte pieces, and
// needs no barrier for them.  Others: the 16-byte pieces inside the row at
// their own alignment, the ends one by one, read back one element a lane.
// Rows past 1024 threads' registers stay in shared memory as f32 (wide_kernel).
#include <type_traits>

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
  int rows, n;
  int8_t* q;
  long ldq;
  float* scale;
};

struct SiluArgs {
  const void* g;
  const void* u;
  long ld;
  int rows, n;
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
__device__ __forceinline__ uint64_t both(float v) {
  return pack2(__float_as_uint(v), __float_as_uint(v));
}
__device__ __forceinline__ uint64_t quant_pair(uint64_t y, uint64_t f) {
  uint64_t t = both(12582912.0f);
  fma2(t, y, f);
  return t;
}
__device__ __forceinline__ unsigned quant4(uint64_t y01, uint64_t y23, uint64_t f) {
  const uint64_t a = quant_pair(y01, f), b = quant_pair(y23, f);
  return __byte_perm(__byte_perm((unsigned)a, (unsigned)(a >> 32), 0x0040),
                     __byte_perm((unsigned)b, (unsigned)(b >> 32), 0x0040), 0x5410);
}

__device__ __forceinline__ unsigned abs_bits(float y) { return __float_as_uint(y) & 0x7fffffffu; }
// max(m, |a|, |b|), NaN if any is
__device__ __forceinline__ float max_abs(float m, uint64_t y) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(m), "f"(fabsf(lo_f(y))), "f"(fabsf(hi_f(y))));
  return r;
}

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
// rounding adds |g| units of it.  Gates below -87 give 0.
__device__ __forceinline__ uint64_t silu_mul(uint64_t g, uint64_t u) {
  const uint64_t x = mul2(g, both(-1.44269504f));
  float e0, e1, s0, s1;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e0) : "f"(lo_f(x)));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e1) : "f"(hi_f(x)));
  const uint64_t d = add2(pack2(__float_as_uint(e0), __float_as_uint(e1)), both(1.0f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s0) : "f"(lo_f(d)));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s1) : "f"(hi_f(d)));
  return mul2(mul2(g, pack2(__float_as_uint(s0), __float_as_uint(s1))), u);
}

// two elements of T in a word (f32: in two) <-> a pair of f32
template <typename T>
__device__ __forceinline__ uint64_t widen(uint32_t w) {
  if constexpr (sizeof(T) == 2) {
    const T* e = reinterpret_cast<const T*>(&w);
    if constexpr (std::is_same<T, __nv_bfloat16>::value) return pack2(w << 16, w & 0xffff0000u);
    return pack2(__float_as_uint(to_f32(e[0])), __float_as_uint(to_f32(e[1])));
  }
  return 0;
}
template <typename T>
__device__ __forceinline__ uint32_t narrow(uint64_t v) {  // to the nearest, ties to even
  uint32_t w;
  if constexpr (std::is_same<T, __nv_bfloat16>::value)
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(hi_f(v)), "f"(lo_f(v)));
  else
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(hi_f(v)), "f"(lo_f(v)));
  return w;
}
// a pair rounded to T
template <typename T>
__device__ __forceinline__ uint64_t rounded(uint64_t v) {
  if constexpr (sizeof(T) == 4)
    return v;
  else
    return widen<T>(narrow<T>(v));
}

// A thread's part of a row: F values in pairs.  VEC: runs of one 16-byte piece
// (kPer elements), every kPer * blockDim.x apart; else a run is one element,
// blockDim.x apart, so that a warp's accesses are contiguous at any alignment,
// and a pair two runs.
template <typename T, int F, bool VEC>
struct Part {
  static constexpr int kPiece = 16 / (int)sizeof(T);
  static constexpr int kPer = VEC ? kPiece : 1;
  static constexpr int kRuns = F / kPer;
  static __device__ __forceinline__ int at(int run) {
    return (run * (int)blockDim.x + (int)threadIdx.x) * kPer;
  }
  // where the row starts in its buffer: at its own place within 16 bytes
  static __device__ __forceinline__ int offset(const T* row) {
    return VEC ? 0 : (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
  }
  // starts the copy of a row into buf (16-byte aligned, n + kPiece elements)
  static __device__ __forceinline__ void stage(T* buf, const T* row, int n) {
    if constexpr (VEC) {
#pragma unroll
      for (int run = 0; run < kRuns; run++) {
        const int i = at(run);
        if (i < n) cp_async16(buf + i, row + i);
      }
    } else {
      const int mis = offset(row), head = min(n, mis ? kPiece - mis : 0);
      const int pieces = (n - head) / kPiece, tail = n - head - pieces * kPiece;
      T* dst = buf + mis;
      for (int i = threadIdx.x; i < pieces; i += blockDim.x)
        cp_async16(dst + head + i * kPiece, row + head + i * kPiece);
      const int t = threadIdx.x;
      if (t < head) dst[t] = row[t];
      if (t >= 16 && t - 16 < tail) dst[n - 1 - (t - 16)] = row[n - 1 - (t - 16)];
    }
  }
  static constexpr int kStep = VEC ? 1 : 2;         // runs handled together
  static constexpr int kPairs = VEC ? kPer / 2 : 1;  // pairs of them
  // the runs from `run` on -> pairs; elements behind n are `none`
  static __device__ __forceinline__ void load(const T* row, int run, int n, uint64_t* v,
                                              float none) {
    const int i = at(run);
#pragma unroll
    for (int k = 0; k < kPairs; k++) v[k] = both(none);
    if constexpr (VEC) {
      if (i < n) {
        const uint4 raw = *reinterpret_cast<const uint4*>(row + i);
        if constexpr (sizeof(T) == 4) {
          v[0] = pack2(raw.x, raw.y);
          v[1] = pack2(raw.z, raw.w);
        } else {
          v[0] = widen<T>(raw.x);
          v[1] = widen<T>(raw.y);
          v[2] = widen<T>(raw.z);
          v[3] = widen<T>(raw.w);
        }
      }
    } else {
      const float a = i < n ? to_f32(row[i]) : none;
      const float b = at(run + 1) < n ? to_f32(row[at(run + 1)]) : none;
      v[0] = pack2(__float_as_uint(a), __float_as_uint(b));
    }
  }
  // the norm's weights, bf16
  static __device__ __forceinline__ void load_w(const uint16_t* w, int run, int n, uint64_t* v) {
    const int i = at(run);
#pragma unroll
    for (int k = 0; k < kPairs; k++) v[k] = both(1.0f);
    if constexpr (VEC) {
      if (i < n) {
        uint32_t raw[kPairs];
        if constexpr (kPairs == 4)
          *reinterpret_cast<uint4*>(raw) = *reinterpret_cast<const uint4*>(w + i);
        else
          *reinterpret_cast<uint2*>(raw) = *reinterpret_cast<const uint2*>(w + i);
#pragma unroll
        for (int k = 0; k < kPairs; k++) v[k] = widen<__nv_bfloat16>(raw[k]);
      }
    } else {
      const float a = i < n ? bf16_to_f32(w[i]) : 1.0f;
      const float b = at(run + 1) < n ? bf16_to_f32(w[at(run + 1)]) : 1.0f;
      v[0] = pack2(__float_as_uint(a), __float_as_uint(b));
    }
  }
  static __device__ __forceinline__ void store(T* row, int run, int n, const uint64_t* v) {
    const int i = at(run);
    if constexpr (VEC) {
      uint4 raw;
      if constexpr (sizeof(T) == 4)
        raw = make_uint4((uint32_t)v[0], (uint32_t)(v[0] >> 32), (uint32_t)v[1],
                         (uint32_t)(v[1] >> 32));
      else
        raw = make_uint4(narrow<T>(v[0]), narrow<T>(v[1]), narrow<T>(v[2]), narrow<T>(v[3]));
      if (i < n) *reinterpret_cast<uint4*>(row + i) = raw;
    } else {
      if (i < n) row[i] = from_f32<T>(lo_f(v[0]));
      if (at(run + 1) < n) row[at(run + 1)] = from_f32<T>(hi_f(v[0]));
    }
  }
  // y (F values) -> 8 bits
  static __device__ __forceinline__ void quantise(const uint64_t* y, int n, unsigned amax_bits,
                                                  int8_t* q, float* scale) {
    float sc;
    const float f = quant_factor(amax_bits, &sc);
    if (threadIdx.x == 0) *scale = sc;
    const uint64_t f2 = both(f);
#pragma unroll
    for (int run = 0; run < kRuns; run += kStep) {
      const int i = at(run);
      const uint64_t* v = y + run / kStep * kPairs;
      if constexpr (!VEC) {
        const uint64_t t = f != 0.0f ? quant_pair(v[0], f2) : 0;
        if (i < n) q[i] = (int8_t)(uint8_t)t;
        if (at(run + 1) < n) q[at(run + 1)] = (int8_t)(uint8_t)(t >> 32);
      } else if (i < n) {
        if constexpr (kPer == 8)
          *reinterpret_cast<uint2*>(q + i) =
              f != 0.0f ? make_uint2(quant4(v[0], v[1], f2), quant4(v[2], v[3], f2))
                        : make_uint2(0, 0);
        else
          *reinterpret_cast<unsigned*>(q + i) = f != 0.0f ? quant4(v[0], v[1], f2) : 0u;
      }
    }
  }
};

__device__ __forceinline__ void copies_commit() {
  asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int N>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// A CTA's walk over its rows with two operands a row (the second may be
// missing): the next row is under way while f works on this one.
//   VEC: one buffer an operand.  A thread's pieces are its own, so it starts
//     the next row's as soon as f has taken this row's into registers.
//   else: two buffers, a barrier before a row is read (all threads' copies of it
//     have landed, and all have read the buffer that is filled next).
// f(row, a, b, next): a, b the staged row; calls next() once they are read.
template <typename T, int F, bool VEC, typename Body>
__device__ __forceinline__ void walk_rows(uint8_t* smem, const T* a, long lda, const T* b, long ldb,
                                          int n, int rows, Body f) {
  using P = Part<T, F, VEC>;
  const int room = ((n + P::kPiece - 1) / P::kPiece + (VEC ? 0 : 1)) * P::kPiece;
  T* buf = reinterpret_cast<T*>(smem);
  const int step = gridDim.x;
  int row = blockIdx.x, at = 0;
  auto stage = [&](int r, int which) {
    if (r < rows) {
      T* to = buf + (long)which * 2 * room;
      P::stage(to, a + r * lda, n);
      if (b) P::stage(to + room, b + r * ldb, n);
    }
    copies_commit();
  };
  stage(row, 0);
  for (; row < rows; row += step) {
    const T* pa = a + row * lda;
    const T* pb = b ? b + row * ldb : nullptr;
    if constexpr (VEC) {
      copies_wait<0>();
      f(row, buf, buf + room, [&] { stage(row + step, 0); });
    } else {
      copies_wait<0>();
      __syncthreads();
      stage(row + step, at ^ 1);
      const T* from = buf + (long)at * 2 * room;
      f(row, from + P::offset(pa), from + room + (pb ? P::offset(pb) : 0), [] {});
      at ^= 1;
    }
  }
}

// --------------------------------------------------------------- the kernels --

template <typename T, int F, bool VEC>
__global__ void __launch_bounds__(kMaxThr) norm_rows_kernel(NormArgs a) {
  using P = Part<T, F, VEC>;
  extern __shared__ __align__(16) uint8_t stage_mem[];
  __shared__ float red[32];
  __shared__ unsigned redu[32];
  pdl_wait();
  pdl_launch_dependents();
  walk_rows<T, F, VEC>(
      stage_mem, static_cast<const T*>(a.x), a.ldx, static_cast<const T*>(a.r), a.ldr, a.n, a.rows,
      [&](long row, const T* x, const T* r, auto next) {
        uint64_t v[F / 2];
#pragma unroll
        for (int run = 0; run < P::kRuns; run += P::kStep) {
          uint64_t* vr = v + run / P::kStep * P::kPairs;
          P::load(x, run, a.n, vr, 0.0f);
          if (a.r) {
            uint64_t b[P::kPairs];
            P::load(r, run, a.n, b, 0.0f);
#pragma unroll
            for (int k = 0; k < P::kPairs; k++) vr[k] = rounded<T>(add2(vr[k], b[k]));
          }
        }
        next();
        uint64_t ss = 0;
#pragma unroll
        for (int k = 0; k < F / 2; k++) fma2(ss, v[k], v[k]);
        if (a.h) {
          T* h = static_cast<T*>(a.h) + row * a.ldh;
#pragma unroll
          for (int run = 0; run < P::kRuns; run += P::kStep)
            P::store(h, run, a.n, v + run / P::kStep * P::kPairs);
        }
        const float inv =
            norm_factor(block_sum(__fadd_rn(lo_f(ss), hi_f(ss)), red), a.n, a.eps);
        float m = 0.0f;
#pragma unroll
        for (int run = 0; run < P::kRuns; run += P::kStep) {
          uint64_t* vr = v + run / P::kStep * P::kPairs;
          uint64_t w[P::kPairs];
          if (a.w) P::load_w(a.w, run, a.n, w);
#pragma unroll
          for (int k = 0; k < P::kPairs; k++) {
            vr[k] = mul2(vr[k], both(inv));
            if (a.w) vr[k] = mul2(vr[k], w[k]);
            m = max_abs(m, vr[k]);
          }
        }
        // red and redu: the other's barrier lies between a row's reads and the
        // next row's writes
        P::quantise(v, a.n, block_max(abs_bits(m), redu), a.q + row * a.ldq, a.scale + row);
      });
}

template <typename T, int F, bool VEC>
__global__ void __launch_bounds__(kMaxThr) silu_rows_kernel(SiluArgs a) {
  using P = Part<T, F, VEC>;
  extern __shared__ __align__(16) uint8_t stage_mem[];
  __shared__ unsigned redu[2][32];  // by the row's parity: one barrier a row
  int parity = 0;
  pdl_wait();
  pdl_launch_dependents();
  walk_rows<T, F, VEC>(
      stage_mem, static_cast<const T*>(a.g), a.ld, static_cast<const T*>(a.u), a.ld, a.n, a.rows,
      [&](long row, const T* g, const T* u, auto next) {
        uint64_t v[F / 2];
        float m = 0.0f;
#pragma unroll
        for (int run = 0; run < P::kRuns; run += P::kStep) {
          uint64_t* vr = v + run / P::kStep * P::kPairs;
          uint64_t gv[P::kPairs], uv[P::kPairs];
          P::load(g, run, a.n, gv, 0.0f);
          P::load(u, run, a.n, uv, 0.0f);
#pragma unroll
          for (int k = 0; k < P::kPairs; k++) {
            vr[k] = silu_mul(gv[k], uv[k]);
            m = max_abs(m, vr[k]);
          }
        }
        next();
        P::quantise(v, a.n, block_max(abs_bits(m), redu[parity]), a.q + row * a.ldq, a.scale + row);
        parity ^= 1;
      });
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
    const float y = lo_f(silu_mul(both(to_f32(g[i])), both(to_f32(u[i]))));
    ys[i] = y;
    m = max(m, abs_bits(y));
  }
  quantise_wide(ys, a.n, block_max(m, redu), a.q + row * a.ldq, a.scale + row);
}

// ------------------------------------------------------------------- launches --

template <typename Args>
int launch(void (*kern)(Args), const Args& a, int grid, int threads, size_t smem,
           cudaStream_t st) {
  if (smem > 48 * 1024)
    EC_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
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

constexpr size_t kStageMax = 224 * 1024;  // an SM's shared memory, less the reductions'

// Launches the kernel of the row's alignment and size; `wide` where a row does
// not fit the registers, or two unaligned ones the shared memory.
template <typename T, typename Args, typename Pick>
int rows_launch(const Args& a, bool vec, void (*wide)(Args), Pick pick,
                cudaStream_t st) {
  constexpr int per = 16 / (int)sizeof(T);
  const int f = values_per_thread(a.rows, a.n);
  const int room = ((a.n + per - 1) / per + (vec ? 0 : 1)) * per;
  const size_t smem = (size_t)room * sizeof(T) * 2 * (vec ? 1 : 2);
  if (a.n > f * kMaxThr || smem > kStageMax)
    return launch(wide, a, a.rows, kWideThr, (size_t)a.n * 4, st);
  const int threads = threads_for(a.n, f);
  // CTAs that an SM holds: by threads (64 registers each) and shared memory
  int per_sm = kMaxThr / threads;
  const int by_smem = (int)(kStageMax / (smem + 1024));
  if (per_sm > by_smem) per_sm = by_smem;
  if (per_sm > 16) per_sm = 16;
  if (per_sm < 1) per_sm = 1;
  const long at_once = 148L * per_sm;
  return launch(pick(f, vec), a, a.rows < at_once ? a.rows : (int)at_once, threads, smem, st);
}

template <typename T>
int norm_rows(const NormArgs& a, cudaStream_t st) {
  constexpr int per = 16 / (int)sizeof(T);
  const bool vec = a.n % per == 0 && aligned(a.x, a.ldx, sizeof(T), 16) &&
                   (!a.r || aligned(a.r, a.ldr, sizeof(T), 16)) &&
                   (!a.h || aligned(a.h, a.ldh, sizeof(T), 16)) &&
                   (!a.w || aligned(a.w, 0, 2, 2 * per)) && aligned(a.q, a.ldq, 1, per);
  return rows_launch<T>(a, vec, norm_wide_kernel<T>, [](int f, bool v) {
    return v ? (f == 8 ? norm_rows_kernel<T, 8, true>
                       : f == 16 ? norm_rows_kernel<T, 16, true> : norm_rows_kernel<T, 32, true>)
             : (f == 8 ? norm_rows_kernel<T, 8, false>
                       : f == 16 ? norm_rows_kernel<T, 16, false> : norm_rows_kernel<T, 32, false>);
  }, st);
}

template <typename T>
int silu_rows(const SiluArgs& a, cudaStream_t st) {
  constexpr int per = 16 / (int)sizeof(T);
  const bool vec = a.n % per == 0 && aligned(a.g, a.ld, sizeof(T), 16) &&
                   aligned(a.u, a.ld, sizeof(T), 16) && aligned(a.q, a.ldq, 1, per);
  return rows_launch<T>(a, vec, silu_wide_kernel<T>, [](int f, bool v) {
    return v ? (f == 8 ? silu_rows_kernel<T, 8, true>
                       : f == 16 ? silu_rows_kernel<T, 16, true> : silu_rows_kernel<T, 32, true>)
             : (f == 8 ? silu_rows_kernel<T, 8, false>
                       : f == 16 ? silu_rows_kernel<T, 16, false> : silu_rows_kernel<T, 32, false>);
  }, st);
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
  const ec::NormArgs a{x, residual, sum_out, (long)ldx, (long)ldr, (long)lds, w, eps, rows, n,
                       q, (long)ldq, scales};
  return ec::with_type(type, [&](auto t) {
    return ec::norm_rows<decltype(t)>(a, static_cast<cudaStream_t>(stream));
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
  const ec::SiluArgs a{gate, up, (long)ld, rows, n, q, (long)ldq, scales};
  return ec::with_type(type, [&](auto t) {
    return ec::silu_rows<decltype(t)>(a, static_cast<cudaStream_t>(stream));
  });
}
