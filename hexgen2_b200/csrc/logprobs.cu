// Log probabilities of given tokens, the entropy of their distribution and its most likely tokens:
// for a row x of logits (f32 arithmetic whatever their type), m = max x, Z = sum exp(x - m),
//   logprob[t] = x_t - m - log Z,   entropy = log Z - (sum exp(x - m) (x - m)) / Z.
// As torch.log_softmax: a masked logit of -inf has probability 0 (and adds nothing to the entropy), a
// row with a NaN or +inf, or of -inf alone, gives NaN. The top list orders by value (NaN first, as
// hx_argmax), equal values by the lower index.
#include "common.cuh"

namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxTop = 32;

// Unique 64-bit key of (value, index): larger value first, NaN above all, -0 equal to +0, then the
// lower index. Never 0.
HX_DEVICE unsigned long long order_key(float x, uint32_t index) {
  uint32_t bits = __float_as_uint(x + 0.f);
  bits = isnan(x) ? 0xffffffffu : (bits & 0x80000000u) ? ~bits : bits | 0x80000000u;
  return ((unsigned long long)bits << 32) | (0xffffffffu - index);
}

HX_DEVICE float block_max(float v, float* sm) {
  v = warp_max(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = v;
  __syncthreads();
  v = sm[0];
  for (int w = 1; w < kWarps; ++w) v = fmaxf(v, sm[w]);
  return v;
}

HX_DEVICE float block_sum(float v, float* sm) {
  v = warp_sum(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.f;
  for (int w = 0; w < kWarps; ++w) v += sm[w];
  return v;
}

// One CTA per row: maximum, then the sums, then top_k rounds of "largest key below the last".
template <typename T>
__global__ void __launch_bounds__(kThreads) logprobs_kernel(
    const T* __restrict__ logits, int64_t cols, int64_t ld, const int64_t* __restrict__ tokens,
    int top_k, float* __restrict__ logprobs, float* __restrict__ entropy,
    float* __restrict__ top_logprobs, int64_t* __restrict__ top_tokens) {
  __shared__ float sm[kWarps];
  __shared__ unsigned long long sm_key[kWarps];
  pdl_wait();
  pdl_trigger();
  const int64_t r = blockIdx.x;
  const T* row = logits + r * ld;
  float m = -INFINITY;
  for (int64_t i = threadIdx.x; i < cols; i += kThreads) m = fmaxf(m, DT<T>::to_f(row[i]));
  m = block_max(m, sm);
  float z = 0.f, s = 0.f;
  for (int64_t i = threadIdx.x; i < cols; i += kThreads) {
    const float d = DT<T>::to_f(row[i]) - m, e = expf(d);
    z += e;
    s += e > 0.f ? e * d : (e == 0.f ? 0.f : e);
  }
  z = block_sum(z, sm);
  s = block_sum(s, sm);
  const float log_z = logf(z);
  if (threadIdx.x == 0) {
    if (logprobs) {
      const int64_t t = tokens[r];
      logprobs[r] = t >= 0 && t < cols ? DT<T>::to_f(row[t]) - m - log_z : NAN;
    }
    if (entropy) entropy[r] = log_z - s / z;
  }
  unsigned long long last = ~0ull;
  for (int j = 0; j < top_k; ++j) {
    unsigned long long best = 0;
    for (int64_t i = threadIdx.x; i < cols; i += kThreads) {
      const unsigned long long key = order_key(DT<T>::to_f(row[i]), (uint32_t)i);
      if (key < last && key > best) best = key;
    }
    for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sm_key[threadIdx.x >> 5] = best;
    __syncthreads();
    for (int w = 0; w < kWarps; ++w) best = max(best, sm_key[w]);
    last = best;
    if (threadIdx.x == 0) {
      const int64_t i = 0xffffffffu - (uint32_t)best;
      top_tokens[r * top_k + j] = i;
      top_logprobs[r * top_k + j] = DT<T>::to_f(row[i]) - m - log_z;
    }
  }
}

}  // namespace

extern "C" int hx_token_logprobs(const void* logits, int64_t rows, int64_t cols, int64_t ld,
                                 const int64_t* tokens, int64_t top_k, float* logprobs,
                                 float* entropy, float* top_logprobs, int64_t* top_tokens,
                                 int dtype, void* stream) {
  HX_REQUIRE(logits && (!logprobs || tokens), "hx_token_logprobs: null pointer");
  HX_REQUIRE(rows >= 0 && rows < (int64_t(1) << 31) && cols > 0 && cols < (int64_t(1) << 31) &&
                 ld >= cols,
             "hx_token_logprobs: bad sizes");
  HX_REQUIRE(top_k >= 0 && top_k <= kMaxTop && top_k <= cols,
             "hx_token_logprobs: top_k %lld out of range (at most %d and the vocabulary)",
             (long long)top_k, kMaxTop);
  HX_REQUIRE(top_k == 0 || (top_logprobs && top_tokens), "hx_token_logprobs: no room for the top list");
  if (rows == 0) return HX_OK;
  HX_DISPATCH_DTYPE(dtype, T, {
    const int s = hx::cuda_status(
        launch_ex(logprobs_kernel<T>, dim3((unsigned)rows), dim3(kThreads), 0, (cudaStream_t)stream,
                  1, (const T*)logits, cols, ld, tokens, (int)top_k, logprobs, entropy,
                  top_logprobs, top_tokens),
        "logprobs_kernel launch");
    if (s) return s;
  });
  HX_LAUNCH_CHECK("logprobs_kernel");
  return HX_OK;
}
