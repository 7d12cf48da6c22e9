// Log probabilities of logits rows: given token, rank, entropy, top alternatives.
//
// For a row x of V logits, m = max x and s = sum_j exp(x_j - m):
//   log p_j = (x_j - m) - ln s
//   rank of t = 1 + #{j : x_j > x_t}
//   entropy = -sum_j p_j log p_j = ln s - (1/s) sum_j exp(x_j - m) (x_j - m)
// so one pass over the row gives everything.  A running (m, s, w) triple, with
// w the last sum, takes a new maximum m' by
//   s' = s exp(m - m'),  w' = exp(m - m') (w + s (m - m')),
// and two triples join the same way.  Exponents are base 2 internally
// (t = (x - m) log2 e), sums are fp32.
//
// The simple form: one CTA per row, the alternatives by repeated arg-max.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "neb_common.cuh"

namespace neb {

constexpr int kLpThreads = 256;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct LogprobParams {
  const void* logits;
  long long row_stride;
  int vocab, num_rows, num_top;
  const int32_t* token_ids;
  float* logprobs;
  int32_t* ranks;
  float* entropy;
  int32_t* top_ids;
  float* top_logprobs;
  unsigned int* error_bits;
};

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }

// An unsigned order of fp32 values: NaN highest, -0 == +0.
__device__ __forceinline__ unsigned int order_f32(float x) {
  if (x != x) return 0xffffffffu;
  const unsigned int b = __float_as_uint(x + 0.f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float value_of_order(unsigned int o) {
  return __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o);
}
__device__ __forceinline__ unsigned long long logit_key(float x, int idx) {
  return ((unsigned long long)order_f32(x) << 32) | (unsigned int)~(unsigned int)idx;
}

// Keeps a NaN, unlike fmaxf.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

struct Sums {
  float m, s, w;  // reference value, sum of e = 2^t, sum of e t with t = (x - m) log2 e
};

// Moves the reference value up to m2 (finite deltas only: an empty sum has
// s = w = 0 and stays so).
__device__ __forceinline__ void raise_to(Sums& a, float m2) {
  const float dt = fmaxf((a.m - m2) * kLog2e, -1000.f);
  const float f = fast_exp2(dt);
  a.w = f * (a.w + a.s * dt);
  a.s *= f;
  a.m = m2;
}
__device__ __forceinline__ Sums join(Sums a, Sums b) {
  const float m = fmaxf(a.m, b.m);
  raise_to(a, m);
  raise_to(b, m);
  return Sums{m, a.s + b.s, a.w + b.w};
}

template <typename T>
__global__ void __launch_bounds__(kLpThreads) token_logprobs_kernel(const LogprobParams p) {
  __shared__ Sums red[kLpThreads / 32];
  __shared__ int red_count[kLpThreads / 32];
  __shared__ unsigned long long red_key[kLpThreads / 32], best_key;
  const int row = blockIdx.x, tid = threadIdx.x;
  const T* x = static_cast<const T*>(p.logits) + (long long)row * p.row_stride;
  int tok = p.token_ids ? p.token_ids[row] : -1;
  if (tok < -1 || tok >= p.vocab) {
    if (tid == 0 && p.error_bits) atomicOr(p.error_bits, kErrTokenId);
    tok = -1;
  }
  const float given = tok >= 0 ? to_f32(x[tok]) : 0.f;
  const unsigned int given_ord = tok >= 0 ? order_f32(given) : 0xffffffffu;
  // The lowest finite value as the empty reference: differences from it stay
  // defined, and a row of that value still sums to its length.
  Sums a{-3.402823466e38f, 0.f, 0.f};
  int above = 0;
  for (int j = tid; j < p.vocab; j += kLpThreads) {
    const float v = to_f32(x[j]);
    if (v > a.m) raise_to(a, v);
    const float t = max_nan((v - a.m) * kLog2e, -200.f);
    const float e = fast_exp2(t);
    a.s += e;
    a.w = fmaf(e, t, a.w);
    above += order_f32(v) > given_ord;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    Sums b{__shfl_xor_sync(~0u, a.m, o), __shfl_xor_sync(~0u, a.s, o), __shfl_xor_sync(~0u, a.w, o)};
    a = join(a, b);
    above += __shfl_xor_sync(~0u, above, o);
  }
  if ((tid & 31) == 0) {
    red[tid >> 5] = a;
    red_count[tid >> 5] = above;
  }
  __syncthreads();
  a = red[0];
  above = red_count[0];
  for (int i = 1; i < kLpThreads / 32; ++i) {
    a = join(a, red[i]);
    above += red_count[i];
  }
  const float nan = __int_as_float(0x7fffffff);
  const bool empty = a.s == 0.f;
  const float ln_s = empty ? nan : logf(a.s);
  if (tid == 0) {
    if (p.logprobs) p.logprobs[row] = tok >= 0 ? (given - a.m) - ln_s : nan;
    if (p.ranks) p.ranks[row] = tok >= 0 ? 1 + above : 0;
    if (p.entropy) p.entropy[row] = ln_s - kLn2 * (a.w / a.s);
  }
  unsigned long long limit = ~0ull;
  for (int k = 0; k < p.num_top; ++k) {
    unsigned long long best = 0;
    for (int j = tid; j < p.vocab; j += kLpThreads) {
      const unsigned long long key = logit_key(to_f32(x[j]), j);
      if (key < limit && key > best) best = key;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const unsigned long long n = __shfl_xor_sync(~0u, best, o);
      best = n > best ? n : best;
    }
    if ((tid & 31) == 0) red_key[tid >> 5] = best;
    __syncthreads();
    if (tid == 0) {
      for (int i = 1; i < kLpThreads / 32; ++i) best = red_key[i] > best ? red_key[i] : best;
      best_key = best;
      const float v = value_of_order((unsigned int)(best >> 32));
      p.top_ids[(long long)row * p.num_top + k] = (int)~(unsigned int)best;
      p.top_logprobs[(long long)row * p.num_top + k] = (v - a.m) - ln_s;
    }
    __syncthreads();
    limit = best_key;
  }
}

}  // namespace neb

using namespace neb;

extern "C" int neb_token_logprobs(const void* logits, int32_t dtype, int64_t row_stride, int32_t vocab,
                                  int32_t num_rows, const int32_t* token_ids, int32_t num_top, float* logprobs,
                                  int32_t* ranks, float* entropy, int32_t* top_ids, float* top_logprobs,
                                  uint32_t* error_bits, void* stream) {
  NEB_REQUIRE(dtype == NEB_DTYPE_F16 || dtype == NEB_DTYPE_BF16 || dtype == NEB_DTYPE_F32, NEB_ERR_INVALID,
              "unknown logits dtype %d", dtype);
  NEB_REQUIRE(num_rows >= 0 && vocab > 0 && row_stride >= 0, NEB_ERR_INVALID, "invalid sizes");
  NEB_REQUIRE(num_top >= 0 && num_top <= vocab && num_top <= NEB_MAX_TOP_LOGPROBS, NEB_ERR_INVALID,
              "num_top %d outside [0, min(vocab, %d)]", num_top, NEB_MAX_TOP_LOGPROBS);
  if (num_rows == 0) return NEB_OK;
  NEB_REQUIRE(logits, NEB_ERR_INVALID, "logits are null");
  NEB_REQUIRE((token_ids != nullptr) == (logprobs != nullptr) && (token_ids != nullptr) == (ranks != nullptr),
              NEB_ERR_INVALID, "token_ids, logprobs and ranks go together");
  NEB_REQUIRE(num_top == 0 || (top_ids && top_logprobs), NEB_ERR_INVALID, "top outputs are null");
  const size_t item = dtype == NEB_DTYPE_F32 ? 4 : 2;
  NEB_REQUIRE(reinterpret_cast<uintptr_t>(logits) % item == 0, NEB_ERR_INVALID, "logits are misaligned");
  LogprobParams p;
  p.logits = logits;
  p.row_stride = row_stride;
  p.vocab = vocab;
  p.num_rows = num_rows;
  p.num_top = num_top;
  p.token_ids = token_ids;
  p.logprobs = logprobs;
  p.ranks = ranks;
  p.entropy = entropy;
  p.top_ids = top_ids;
  p.top_logprobs = top_logprobs;
  p.error_bits = error_bits;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == NEB_DTYPE_F16) token_logprobs_kernel<__half><<<num_rows, kLpThreads, 0, s>>>(p);
  else if (dtype == NEB_DTYPE_BF16) token_logprobs_kernel<__nv_bfloat16><<<num_rows, kLpThreads, 0, s>>>(p);
  else token_logprobs_kernel<float><<<num_rows, kLpThreads, 0, s>>>(p);
  NEB_CUDA(cudaGetLastError());
  return NEB_OK;
}
