// logprobs.cu -- log probabilities of given tokens, entropy and the top
// alternatives of logit rows (ec_op_token_logprobs).
//
//   z = l / T;  m = max z;  S = sum exp(z - m);  W = sum exp(z - m) (z - m)
//   logprob(i) = (z_i - m) - log S;  H = log S - W / S
//
// One CTA per row: a pass for the maximum, one for the sums, one for each
// alternative (the largest key below the last one's).
#include "typed.cuh"

namespace ec {
namespace {

constexpr int kThr = 256;
constexpr int kMaxTop = 32;

typedef unsigned long long u64;

struct LogprobArgs {
  const void* l;
  long ld;
  int n;
  const int* tokens;
  float inv_t;
  int top;
  float* logprob;
  float* entropy;
  int* ids;
  float* top_lp;
};

// Larger logit first, then smaller index, in one unsigned integer: the float's
// bits made monotonic (-0 as +0, NaN below -inf), then the inverted index.
__device__ __forceinline__ u64 order_key(float v, int i) {
  unsigned b = __float_as_uint(v == 0.0f ? 0.0f : v);
  b = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
  if (v != v) b = 0;
  return ((u64)b << 32) | (unsigned)~i;
}

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

// log probability from the logit, the row's maximum and log S
__device__ __forceinline__ float logprob_of(float v, float m, float inv_t, float logs) {
  if (m == -INFINITY) return v == v ? -INFINITY : v;  // every token barred
  return __fsub_rn(__fmul_rn(__fsub_rn(v, m), inv_t), logs);
}

template <typename T>
__global__ void __launch_bounds__(kThr) token_logprobs_kernel(LogprobArgs a) {
  __shared__ float red[kThr / 32];
  __shared__ u64 redk[kThr / 32];
  const long row = blockIdx.x;
  const T* l = static_cast<const T*>(a.l) + row * a.ld;
  float m = -INFINITY;
  for (int i = threadIdx.x; i < a.n; i += kThr) {
    const float v = to_f32(l[i]);
    m = (v > m || v != v) ? v : m;  // a NaN stays
    if (m != m) break;
  }
  m = block_all(m, red, [](float p, float q) { return (p != p || p > q) ? p : q; });
  float s = 0.0f, w = 0.0f;
  if (m != -INFINITY) {
    for (int i = threadIdx.x; i < a.n; i += kThr) {
      const float d = __fmul_rn(__fsub_rn(to_f32(l[i]), m), a.inv_t);
      const float e = expf(d);
      s = __fadd_rn(s, e);
      if (e != 0.0f) w = __fmaf_rn(e, d, w);
    }
  }
  auto add = [](float p, float q) { return __fadd_rn(p, q); };
  s = block_all(s, red, add);
  w = block_all(w, red, add);
  const float logs = logf(s);
  if (threadIdx.x == 0) {
    if (a.entropy) a.entropy[row] = m == -INFINITY ? 0.0f : __fsub_rn(logs, __fdiv_rn(w, s));
    if (a.logprob) {
      const int t = a.tokens[row];
      float lp = t == -1 ? 0.0f : __uint_as_float(0x7fc00000u);
      if (t >= 0 && t < a.n) lp = logprob_of(to_f32(l[t]), m, a.inv_t, logs);
      a.logprob[row] = lp;
    }
  }
  u64 last = ~0ull;
  for (int j = 0; j < a.top; j++) {
    u64 best = 0;
    for (int i = threadIdx.x; i < a.n; i += kThr) {
      const u64 k = order_key(to_f32(l[i]), i);
      if (k < last && k > best) best = k;
    }
    last = block_all(best, redk, [](u64 p, u64 q) { return p > q ? p : q; });
    if (threadIdx.x == 0) {
      const int i = (int)~(unsigned)last;
      a.ids[row * a.top + j] = i;
      a.top_lp[row * a.top + j] = logprob_of(to_f32(l[i]), m, a.inv_t, logs);
    }
  }
}

}  // namespace
}  // namespace ec

extern "C" int ec_op_token_logprobs(int type, const void* logits, int64_t ld, int n, int rows,
                                    const int* tokens, float temperature, int top_k,
                                    float* logprob, float* entropy, int* top_ids,
                                    float* top_logprobs, void* stream) {
  if (!ec::known_type(type)) return ec::arg_error("ec_op_token_logprobs: unknown type");
  if (!logits || rows <= 0 || n <= 0 || ld < n || !(temperature >= 0x1p-100f) ||
      !(temperature <= 0x1p100f))
    return ec::arg_error("ec_op_token_logprobs: null logits, empty shape, ld < n, or temperature");
  if (!tokens != !logprob || top_k < 0 || top_k > n || (top_k > 0 && (!top_ids || !top_logprobs)))
    return ec::arg_error("ec_op_token_logprobs: tokens and logprob go together; top_k 0..n with "
                         "both outputs");
  if (top_k > ec::kMaxTop) return ec::unsupported("ec_op_token_logprobs: top_k > 32");
  const ec::LogprobArgs a{logits, (long)ld, n, tokens, 1.0f / temperature, top_k, logprob, entropy,
                          top_ids, top_logprobs};
  return ec::with_type(type, [&](auto t) {
    ec::token_logprobs_kernel<decltype(t)>
        <<<rows, ec::kThr, 0, static_cast<cudaStream_t>(stream)>>>(a);
    EC_CUDA_TRY(cudaGetLastError());
    return EC_OK;
  });
}
