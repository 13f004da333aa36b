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
// The top list needs no second pass over the row. A thread knows its maximum and the 16 bytes that hold
// it first, so its best key lies between (maximum, last index there) and (maximum, first index there).
// T, the top_k-th largest of the lower ends of 64 groups of threads, is no larger than the row's
// top_k-th largest key, since top_k groups have an element at or above it. Only threads whose upper end is
// at least T can own listed elements; they read their own elements again and collect those >= T, in
// practice few more than top_k. A candidate's place in the list is
// the number of larger candidates. Rows whose candidates do not fit, and rows with NaN, take top_k
// rounds of "largest key below the last" instead.
//
// Measured: 4096 rows x 32000 bf16 with the top token 63 us (4.2 TB/s, 0.64 of the measured copy rate; 55
// without the list), 1 row 7.8 us, 32 x 128007 f32 with twenty 16 us. Many rows are bound by instructions
// (99 per eight logits a lane and warp in all, 73 % of the issue slots and half of the SFU's), few by the chain of
// barriers behind the row.
#include "common.cuh"

namespace {

constexpr int kThreads = 128;  // few, so that rows overlap: a row's last steps keep one or two warps busy
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

// z = sum exp(x - m) and s = sum exp(x - m) (x - m) move to a larger maximum, d = m - maximum <= 0. Logits
// masked with a type's lowest value make d as low as -3.4e38, and d z would overflow; below -1000 exp(d) is 0
// already, so d stops there. A NaN (from infinities) stays in z.
HX_DEVICE void rebase(float d, float& z, float& s) {
  const float f = exp_neg(d);
  s = fmaf(fmaxf(d, -1000.f), z, s) * f;
  z *= f;
}

// row[begin, end) as thread `tid` of kThreads sees it: an element up to a 16-byte boundary, vectors tid, tid +
// kThreads, ... of 16 bytes, an element behind them.
template <typename T>
struct Slice {
  static constexpr int V = 16 / sizeof(T);
  const T* row;
  int64_t begin, end, first, nvec;
  HX_DEVICE Slice(const T* row, int64_t begin, int64_t end) : row(row), begin(begin), end(end) {
    first = min(begin + (int64_t)((16 - ((uintptr_t)(row + begin) & 15)) & 15) / (int64_t)sizeof(T), end);
    nvec = (end - first) / V;
  }
  HX_DEVICE int64_t tail() const { return first + nvec * V; }
  HX_DEVICE uint4 load(int64_t v) const { return __ldg(reinterpret_cast<const uint4*>(row + first) + v); }
  static HX_DEVICE void convert(uint4 raw, float (&x)[V]) {
#pragma unroll
    for (int j = 0; j < V; ++j) x[j] = DT<T>::to_f(reinterpret_cast<const T*>(&raw)[j]);
  }
  // Thread tid's elements in rising order, four loads in flight. f(x, index) takes one or four runs of
  // neighbouring elements, run u beginning at index + u * kThreads * (its length).
  template <typename F>
  HX_DEVICE void walk(F&& f) const {
    const int tid = threadIdx.x;
    if (begin + tid < first) {
      float x[1][1] = {{DT<T>::to_f(row[begin + tid])}};
      f(x, begin + tid);
    }
    int64_t v = tid;
    for (; v + 3 * kThreads < nvec; v += 4 * kThreads) {
      uint4 raw[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) raw[u] = load(v + u * kThreads);
      float x[4][V];
#pragma unroll
      for (int u = 0; u < 4; ++u) convert(raw[u], x[u]);
      f(x, first + v * V);
    }
    uint4 raw[3];
#pragma unroll
    for (int u = 0; u < 3; ++u)
      if (v + u * kThreads < nvec) raw[u] = load(v + u * kThreads);
#pragma unroll
    for (int u = 0; u < 3; ++u)
      if (v + u * kThreads < nvec) {
        float x[1][V];
        convert(raw[u], x[0]);
        f(x, first + (v + u * kThreads) * V);
      }
    if (tail() + tid < end) {
      float x[1][1] = {{DT<T>::to_f(row[tail() + tid])}};
      f(x, tail() + tid);
    }
  }
  // The elements of thread `owner`, shared out over the calling warp. f(x, index), one at a time.
  template <typename F>
  HX_DEVICE void walk_together(int owner, F&& f) const {
    const int lane = threadIdx.x & 31;
    if (lane == 0 && begin + owner < first) f(DT<T>::to_f(row[begin + owner]), begin + owner);
    for (int64_t v = owner + (int64_t)lane * kThreads; v < nvec; v += 32 * kThreads) {
      float x[V];
      convert(load(v), x);
#pragma unroll
      for (int j = 0; j < V; ++j) f(x[j], first + v * V + j);
    }
    if (lane == 0 && tail() + owner < end) f(DT<T>::to_f(row[tail() + owner]), tail() + owner);
  }
};

template <typename T>
__global__ void __launch_bounds__(kThreads, 8) logprobs_kernel(
    const T* __restrict__ logits, int64_t cols, int64_t ld, const int64_t* __restrict__ tokens, int log_c,
    int top_k, float* __restrict__ logprobs, float* __restrict__ entropy,
    float* __restrict__ top_logprobs, int64_t* __restrict__ top_tokens) {
  __shared__ float sm_max[kWarps], sm_z[kWarps], sm_s[kWarps], sm_total[3];
  __shared__ Key sm_group[kGroups], sm_list[kMaxTop], sm_limit;
  __shared__ Key sm_cand[kCandidates];
  __shared__ int sm_count;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  pdl_wait();
  pdl_trigger();
  const int C = 1 << log_c;
  const int64_t r = blockIdx.x >> log_c;
  const int rank = C > 1 ? (int)cluster_rank() : 0;
  const T* row = logits + r * ld;
  const Slice<T> slice(row, (cols * rank) >> log_c, (cols * (rank + 1)) >> log_c);

  // The given token's logit, asked for ahead of the row.
  float given = NAN;
  if (logprobs && rank == 0 && tid == 0) {
    const int64_t at = tokens[r];
    if (at >= 0 && at < cols) given = DT<T>::to_f(row[at]);
  }

  float m = -INFINITY, z = 0.f, s = 0.f;
  int64_t where = -1;  // first index of the run that holds m first
  int width = 0;       // and its length
  slice.walk([&](auto& x, int64_t at) {
    constexpr int U = sizeof(x) / sizeof(x[0]), V = sizeof(x[0]) / sizeof(float);
    float tops[U], top = -INFINITY;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      tops[u] = x[u][0];
#pragma unroll
      for (int j = 1; j < V; ++j) tops[u] = fmaxf(tops[u], x[u][j]);
      top = fmaxf(top, tops[u]);
    }
    if (where < 0) where = at, width = V;
    if (top > m) {
      if (m != -INFINITY) rebase(m - top, z, s);
      m = top;
      int at_u = 0;
#pragma unroll
      for (int u = U - 1; u >= 0; --u) at_u = tops[u] == top ? u : at_u;
      where = at + at_u * kThreads * V;
      width = V;
    }
    const float ref = m == -INFINITY ? 0.f : m;  // masked logits alone so far: exp(-inf) = 0
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float d = x[u][j] - ref, e = exp_neg(d);
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
  if (m != -INFINITY) rebase(m - top, z, s);
  z = warp_sum(z);
  s = warp_sum(s);
  if (lane == 0) sm_z[warp] = z, sm_s[warp] = s;
  // The best keys of the thread groups, for the top list.
  const Key most = where >= 0 ? order_key(own, (uint32_t)where) : 0;
  if (top_k > 0) {
    Key k = where >= 0 ? order_key(own, (uint32_t)(where + width - 1)) : 0;
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
#pragma unroll 16
    for (int i = 0; i < kGroups; ++i) place += sm_group[i] > mine;
    if (mine && place < top_k) sm_list[place] = mine;
  }
  if (C > 1) cluster_sync(); else __syncthreads();
  // The cluster's totals: lane c of every warp reads CTA c's.
  {
    const bool some = lane < C;
    const float mc = some ? peek(&sm_total[0], lane, C) : -INFINITY;
    float zc = some ? peek(&sm_total[1], lane, C) : 0.f, sc = some ? peek(&sm_total[2], lane, C) : 0.f;
    top = warp_max(mc);
    if (mc != -INFINITY) rebase(mc - top, zc, sc);  // without a maximum: 0, or NaN to keep
    z = warp_sum(zc);
    s = warp_sum(sc);
  }
  if (top == -INFINITY) z = NAN;
  const float log_z = logf(z);
  if (rank == 0 && tid == 0) {
    if (logprobs) logprobs[r] = given - top - log_z;
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
    Key limit = sm_list[top_k - 1];
    if (C > 1) {
      const int n = C * top_k;
      for (int i = tid; i < n; i += kThreads) sm_cand[i] = peek(&sm_list[i % top_k], i / top_k, C);
      __syncthreads();
      for (int i = tid; i < n; i += kThreads) {
        const Key mine = sm_cand[i];
        int place = 0;
#pragma unroll 8
        for (int j = 0; j < n; ++j) place += sm_cand[j] > mine;
        if (mine && place == top_k - 1) sm_limit = mine;
      }
      __syncthreads();  // sm_cand is free again
      limit = sm_limit;
    }
    const float least = limit ? key_value(limit) : -INFINITY;
    // A warp walks the elements of its owning lanes together.
    uint32_t owners = __ballot_sync(0xffffffffu, most >= limit && most);
    while (owners) {
      const int owner = (tid & ~31) + __ffs(owners) - 1;
      owners &= owners - 1;
      slice.walk_together(owner, [&](float x, int64_t at) {
        if (x >= least) {
          const Key k = order_key(x, (uint32_t)at);
          const int i = k >= limit ? atomicAdd(&sm_count, 1) : kCandidates;
          if (i < kCandidates) sm_cand[i] = k;
        }
      });
    }
    if (C > 1) cluster_sync(); else __syncthreads();
    if (rank == 0) {  // the candidates of all CTAs, behind this one's
      int n = sm_count;
      if (C > 1) {
        const int theirs = lane < C ? peek(&sm_count, lane, C) : 0;
        for (int c = 1; c < C; ++c) {
          const int k = __shfl_sync(0xffffffffu, theirs, c);
          if (n <= kCandidates && n + k <= kCandidates)
            for (int i = tid; i < k; i += kThreads) sm_cand[n + i] = peek(&sm_cand[i], c, C);
          n += k;
        }
        __syncthreads();
      }
      rounds = n > kCandidates;
      if (!rounds)
        for (int i = tid; i < n; i += kThreads) {
          const Key here = sm_cand[i];
          int place = 0;
#pragma unroll 8
          for (int j = 0; j < n; ++j) place += sm_cand[j] > here;
          if (place < top_k) put(place, here);
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
  // CTAs per row: while each keeps a thread's four loads in flight busy, as long as all find room at once.
  int log_c = 0;
  while (log_c < 3 && rows << (log_c + 1) <= 148 * 8 && cols >> (log_c + 1) >= 2048) ++log_c;
  HX_DISPATCH_DTYPE(dtype, T, {
    const int s = hx::cuda_status(
        launch_ex(logprobs_kernel<T>, dim3((unsigned)(rows << log_c)), dim3(kThreads), 0, (cudaStream_t)stream,
                  1 << log_c, (const T*)logits, cols, ld, tokens, log_c, (int)top_k, logprobs, entropy,
                  top_logprobs, top_tokens),
        "logprobs_kernel launch");
    if (s) return s;
  });
  HX_LAUNCH_CHECK("logprobs_kernel");
  return HX_OK;
}
