// Log probabilities of given tokens, the entropy of their distribution and its most likely tokens:
// for a row x of logits (f32 arithmetic whatever their type), m = max x, Z = sum exp(x - m),
//   logprob[t] = x_t - m - log Z,   entropy = log Z - (sum exp(x - m) (x - m)) / Z.
// As torch.log_softmax: a masked logit of -inf has probability 0 (and adds nothing to the entropy), a
// row with a NaN or +inf, or of -inf alone, gives NaN. The top list orders by value (NaN first, as
// hx_argmax), equal values by the lower index.
//
// One pass over the row: every thread keeps its maximum so far, the sums relative to it, and where it
// was first seen. A row is one CTA, or a cluster of up to eight where there are few rows (one SM would
// read a long row while the others wait); the CTAs' sums meet through distributed shared memory, in
// rank order.
//
// The top list needs no second pass over the row. T, the top_k-th largest of the best keys of 64 groups
// of threads, is no larger than the row's top_k-th largest key, since top_k groups have an element at or
// above it. Only threads whose best is at least T can own listed elements; they read their own elements
// again and collect those >= T, in practice few more than top_k. A candidate's place in the list is
// the number of larger candidates. Rows whose candidates do not fit, and rows with NaN, take top_k
// rounds of "largest key below the last" instead.
#include "common.cuh"

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kGroups = 64;       // of kThreads / kGroups adjacent threads
constexpr int kMaxTop = 32;
constexpr int kCandidates = 2048;

using Key = unsigned long long;

// Unique 64-bit key of (value, index): larger value first, NaN above all, -0 equal to +0, then the
// lower index. Never 0.
HX_DEVICE Key order_key(float x, uint32_t index) {
  uint32_t bits = __float_as_uint(x + 0.f);
  bits = isnan(x) ? 0xffffffffu : (bits & 0x80000000u) ? ~bits : bits | 0x80000000u;
  return ((Key)bits << 32) | (0xffffffffu - index);
}
HX_DEVICE float key_value(Key k) {
  const uint32_t bits = (uint32_t)(k >> 32);
  return __uint_as_float((bits & 0x80000000u) ? bits ^ 0x80000000u : ~bits);
}
HX_DEVICE int64_t key_index(Key k) { return 0xffffffffu - (uint32_t)k; }

HX_DEVICE uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
HX_DEVICE void cluster_sync() {
  asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}
HX_DEVICE uint32_t cluster_addr(const void* p, uint32_t rank) {
  uint32_t remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(smem_u32(p)), "r"(rank));
  return remote;
}
// *p in CTA `rank` of the cluster (this CTA's own without one).
HX_DEVICE float peek(const float* p, int rank, int C) {
  if (C == 1) return *p;
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(cluster_addr(p, rank)) : "memory");
  return v;
}
HX_DEVICE int peek(const int* p, int rank, int C) {
  if (C == 1) return *p;
  int v;
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(cluster_addr(p, rank)) : "memory");
  return v;
}
HX_DEVICE Key peek(const Key* p, int rank, int C) {
  if (C == 1) return *p;
  Key v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(cluster_addr(p, rank)) : "memory");
  return v;
}

// exp(d) for d <= 0: the SFU's exp2, 2 ulp, of a product whose rounding moves a term of size exp(d) by
// |d| 2^-24 of itself.
HX_DEVICE float exp_neg(float d) { return ex2_approx(d * 1.4426950408889634f); }

// The calling thread's elements of row[begin, end), in rising order: single elements up to a 16-byte
// boundary, vectors with four loads in flight, single elements again. f(x, index) takes an array.
template <typename T, typename F>
HX_DEVICE void for_each(const T* row, int64_t begin, int64_t end, F&& f) {
  constexpr int V = 16 / sizeof(T);
  const int64_t first = min(begin + (int64_t)((16 - ((uintptr_t)(row + begin) & 15)) & 15) / (int64_t)sizeof(T), end);
  const int64_t nvec = (end - first) / V, tail = first + nvec * V;
  if (begin + threadIdx.x < first) {
    float x[1] = {DT<T>::to_f(row[begin + threadIdx.x])};
    f(x, begin + threadIdx.x);
  }
  const uint4* v = reinterpret_cast<const uint4*>(row + first);
  for (int64_t base = threadIdx.x; base < nvec; base += 4 * kThreads) {
    uint4 raw[4];
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (base + u * kThreads < nvec) raw[u] = __ldg(v + base + u * kThreads);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (base + u * kThreads >= nvec) break;
      const T* e = reinterpret_cast<const T*>(&raw[u]);
      float x[V];
#pragma unroll
      for (int j = 0; j < V; ++j) x[j] = DT<T>::to_f(e[j]);
      f(x, first + (base + u * kThreads) * V);
    }
  }
  if (tail + threadIdx.x < end) {
    float x[1] = {DT<T>::to_f(row[tail + threadIdx.x])};
    f(x, tail + threadIdx.x);
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 4) logprobs_kernel(
    const T* __restrict__ logits, int64_t cols, int64_t ld, const int64_t* __restrict__ tokens, int C,
    int top_k, float* __restrict__ logprobs, float* __restrict__ entropy,
    float* __restrict__ top_logprobs, int64_t* __restrict__ top_tokens) {
  __shared__ float sm_max[kWarps], sm_z[kWarps], sm_s[kWarps], sm_total[3];
  __shared__ Key sm_group[kGroups], sm_list[kMaxTop], sm_limit;
  __shared__ Key sm_cand[kCandidates];
  __shared__ int sm_count;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  pdl_wait();
  pdl_trigger();
  const int64_t r = blockIdx.x / C;
  const int rank = C > 1 ? (int)cluster_rank() : 0;
  const T* row = logits + r * ld;
  const int64_t begin = cols * rank / C, end = cols * (rank + 1) / C;

  float m = -INFINITY, z = 0.f, s = 0.f;
  int64_t where = -1;  // of the first element equal to m
  for_each(row, begin, end, [&](auto& x, int64_t at) {
    constexpr int n = sizeof(x) / sizeof(float);
    float top = x[0];
#pragma unroll
    for (int j = 1; j < n; ++j) top = fmaxf(top, x[j]);
    if (where < 0) where = at;
    if (top > m) {
      const float d = m - top, f = exp_neg(d);  // 0 and nothing to scale while m is -inf
      if (m != -INFINITY) s = fmaf(d, z, s) * f, z *= f;
      m = top;
      int j = 0;
#pragma unroll
      for (int i = n - 1; i >= 0; --i) j = x[i] == top ? i : j;
      where = at + j;
    }
    const float ref = m == -INFINITY ? 0.f : m;  // masked logits alone so far: exp(-inf) = 0
#pragma unroll
    for (int j = 0; j < n; ++j) {
      const float d = x[j] - ref, e = exp_neg(d);
      z += e;
      s = fmaf(e, fmaxf(d, -1000.f), s);  // 0 where d is -inf; a NaN stays in z
    }
  });

  // The row's maximum, then the sums relative to it.
  const float own = m;
  float top = warp_max(m);
  if (lane == 0) sm_max[warp] = top;
  __syncthreads();
  top = sm_max[0];
#pragma unroll
  for (int w = 1; w < kWarps; ++w) top = fmaxf(top, sm_max[w]);
  if (m != -INFINITY) {
    const float d = m - top, f = exp_neg(d);
    s = fmaf(d, z, s) * f;
    z *= f;
  }
  z = warp_sum(z);
  s = warp_sum(s);
  if (lane == 0) sm_z[warp] = z, sm_s[warp] = s;
  // The best keys of the thread groups, for the top list.
  const Key best = where >= 0 ? order_key(own, (uint32_t)where) : 0;
  if (top_k > 0) {
    Key k = best;
#pragma unroll
    for (int o = kThreads / kGroups / 2; o > 0; o >>= 1) {
      const Key other = __shfl_xor_sync(0xffffffffu, k, o);
      k = k > other ? k : other;
    }
    if (tid % (kThreads / kGroups) == 0) sm_group[tid / (kThreads / kGroups)] = k;
    if (tid < kMaxTop) sm_list[tid] = 0;
    if (tid == 0) sm_limit = 0, sm_count = 0;
  }
  __syncthreads();
  if (tid == 0) {
    z = s = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) z += sm_z[w], s += sm_s[w];
    sm_total[0] = top, sm_total[1] = z, sm_total[2] = s;
  }
  if (top_k > 0 && tid < kGroups) {  // this CTA's largest group keys, falling
    const Key mine = sm_group[tid];
    int place = 0;
#pragma unroll 8
    for (int i = 0; i < kGroups; ++i) place += sm_group[i] > mine;
    if (mine && place < top_k) sm_list[place] = mine;
  }
  if (C > 1) cluster_sync(); else __syncthreads();
  top = -INFINITY;
  for (int c = 0; c < C; ++c) top = fmaxf(top, peek(&sm_total[0], c, C));
  z = s = 0.f;
  for (int c = 0; c < C; ++c) {
    const float mc = peek(&sm_total[0], c, C), zc = peek(&sm_total[1], c, C), sc = peek(&sm_total[2], c, C);
    const float d = mc - top, f = mc == -INFINITY ? 1.f : exp_neg(d);  // without a maximum: 0, or NaN to keep
    z += zc * f;
    s += (mc == -INFINITY ? sc : fmaf(d, zc, sc)) * f;
  }
  if (top == -INFINITY) z = NAN;
  const float log_z = logf(z);
  if (rank == 0 && tid == 0) {
    if (logprobs) {
      const int64_t t = tokens[r];
      logprobs[r] = t >= 0 && t < cols ? DT<T>::to_f(row[t]) - top - log_z : NAN;
    }
    if (entropy) entropy[r] = log_z - s / z;
  }
  if (top_k == 0) {
    if (C > 1) cluster_sync();  // no CTA leaves while others read its sums
    return;
  }
  auto put = [&](int place, Key k) {
    top_tokens[r * top_k + place] = key_index(k);
    top_logprobs[r * top_k + place] = key_value(k) - top - log_z;
  };
  bool rounds = isnan(z);
  if (!rounds) {
    // T: the top_k-th largest of the CTAs' group keys (0, everything, where there are not as many).
    for (int i = tid; i < C * top_k; i += kThreads) {
      const Key mine = peek(&sm_list[i % top_k], i / top_k, C);
      int place = 0;
      for (int c = 0; c < C; ++c)
        for (int j = 0; j < top_k; ++j) place += peek(&sm_list[j], c, C) > mine;
      if (mine && place == top_k - 1) sm_limit = mine;
    }
    __syncthreads();
    const Key limit = sm_limit;
    if (top_k == 1) {
      if (rank == 0 && tid == 0) put(0, limit);
    } else {
      if (best >= limit && best)
        for_each(row, begin, end, [&](auto& x, int64_t at) {
          constexpr int n = sizeof(x) / sizeof(float);
#pragma unroll
          for (int j = 0; j < n; ++j) {
            const Key k = order_key(x[j], (uint32_t)(at + j));
            if (k >= limit) {
              const int i = atomicAdd(&sm_count, 1);
              if (i < kCandidates) sm_cand[i] = k;
            }
          }
        });
      if (C > 1) cluster_sync(); else __syncthreads();
      for (int c = 0; c < C; ++c) rounds |= peek(&sm_count, c, C) > kCandidates;
      if (!rounds)
        for (int i = tid; i < sm_count; i += kThreads) {
          const Key mine = sm_cand[i];
          int place = 0;
          for (int c = 0; c < C && place < top_k; ++c) {
            const int n = peek(&sm_count, c, C);
            for (int j = 0; j < n; ++j) place += peek(&sm_cand[j], c, C) > mine;
          }
          if (place < top_k) put(place, mine);
        }
    }
  }
  if (rounds && rank == 0) {
    Key last = ~0ull;
    for (int j = 0; j < top_k; ++j) {
      Key k = 0;
      for (int64_t i = tid; i < cols; i += kThreads) {
        const Key here = order_key(DT<T>::to_f(row[i]), (uint32_t)i);
        if (here < last && here > k) k = here;
      }
      for (int o = 16; o > 0; o >>= 1) {
        const Key other = __shfl_xor_sync(0xffffffffu, k, o);
        k = k > other ? k : other;
      }
      __syncthreads();
      if (lane == 0) sm_group[warp] = k;
      __syncthreads();
      for (int w = 0; w < kWarps; ++w) k = k > sm_group[w] ? k : sm_group[w];
      last = k;
      if (tid == 0) put(j, k);
    }
  }
  if (C > 1) cluster_sync();  // no CTA leaves while others read its lists
}

}  // namespace

extern "C" int hx_token_logprobs(const void* logits, int64_t rows, int64_t cols, int64_t ld,
                                 const int64_t* tokens, int64_t top_k, float* logprobs,
                                 float* entropy, float* top_logprobs, int64_t* top_tokens,
                                 int dtype, void* stream) {
  HX_REQUIRE(logits && (!logprobs || tokens), "hx_token_logprobs: null pointer");
  HX_REQUIRE(rows >= 0 && rows < (int64_t(1) << 28) && cols > 0 && cols < (int64_t(1) << 31) &&
                 ld >= cols,
             "hx_token_logprobs: bad sizes");
  HX_REQUIRE(top_k >= 0 && top_k <= kMaxTop && top_k <= cols,
             "hx_token_logprobs: top_k %lld out of range (at most %d and the vocabulary)",
             (long long)top_k, kMaxTop);
  HX_REQUIRE(top_k == 0 || (top_logprobs && top_tokens), "hx_token_logprobs: no room for the top list");
  if (rows == 0) return HX_OK;
  // CTAs per row: while all of them find room at once (four to an SM) and each keeps a thread's four
  // loads in flight busy.
  int C = 1;
  while (C < 8 && rows * C * 2 <= 148 * 4 && cols / (C * 2) >= 4096) C *= 2;
  HX_DISPATCH_DTYPE(dtype, T, {
    const int s = hx::cuda_status(
        launch_ex(logprobs_kernel<T>, dim3((unsigned)(rows * C)), dim3(kThreads), 0, (cudaStream_t)stream,
                  C, (const T*)logits, cols, ld, tokens, C, (int)top_k, logprobs, entropy,
                  top_logprobs, top_tokens),
        "logprobs_kernel launch");
    if (s) return s;
  });
  HX_LAUNCH_CHECK("logprobs_kernel");
  return HX_OK;
}
