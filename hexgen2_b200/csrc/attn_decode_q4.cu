// Single-query decode attention over a KV cache held in 4-bit records (kv_q4.cu has the format).
//
// For query head h of KV head h / G and the live positions t of its sequence, with a key standing
// for k_t = kmin_t + ks_t * ck_t (ck_t the integer codes) and a value for v_t = vmin_t + vs_t * cv_t:
//   s_t = scale * (ks_t * (q . ck_t) + kmin_t * sum(q))
//   out = (sum_t (p_t vs_t) cv_t + sum_t p_t vmin_t) / sum_t p_t,   p_t = exp(s_t - max s)
// so the products run on the small integers and the scales are applied once per position, in f32.
// The softmax is online (base 2, f32 maximum and sum). A sequence of length 0 gives zeros.
#include "common.cuh"

namespace {

constexpr int kThreads = 128;
constexpr int kWarps = kThreads / 32;
constexpr int NQ = 8;  // query heads of one KV head that a CTA serves from one read of the records

// Live length of sequence b, inside what the caller promised; a broken promise is reported.
HX_DEVICE int live_length(const int32_t* seqlens, int b, int64_t max_len) {
  const int64_t len = seqlens[b];
  if (len < 0 || len > max_len) {
    if (threadIdx.x == 0) record_device_error(HX_DEVERR_BAD_ARGUMENT);
    return len < 0 ? 0 : (int)max_len;
  }
  return (int)len;
}

struct Args {
  const void* q;
  const uint8_t* q4;
  const int32_t* seqlens;
  void* out;
  float* ws_o;   // [batch, n_heads, splits, D]
  float* ws_ml;  // [batch, n_heads, splits, 2]
  int64_t qbs, qhs, q_stride, max_len;
  int n_heads, group, q_chunks, chunk, splits;
  float scale_log2;
};

// CUDA-core kernel: f32 products for every type. One CTA per (key split, KV head and eight of its
// query heads, sequence); a warp takes 32 keys at a time, one per lane for the scores, all lanes
// across D for the values.
template <typename T, int D>
__global__ void __launch_bounds__(kThreads) decode_q4_kernel(const Args a) {
  constexpr int EPL = D / 32;  // output elements per lane
  __shared__ float sm_q[NQ][D];
  __shared__ float sm_sum[NQ];
  __shared__ float sm_o[kWarps][NQ][D];
  __shared__ float sm_m[kWarps][NQ], sm_l[kWarps][NQ], sm_z[kWarps][NQ];
  pdl_wait();
  pdl_trigger();
  const int split = blockIdx.x, b = blockIdx.z;
  const int hk = blockIdx.y / a.q_chunks, h0 = hk * a.group + (blockIdx.y % a.q_chunks) * NQ;
  const int nq = min(NQ, (hk + 1) * a.group - h0);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int len = live_length(a.seqlens, b, a.max_len);
  const int start = split * a.chunk, end = min(start + a.chunk, len);
  T* out = (T*)a.out + ((int64_t)b * a.n_heads + h0) * D;
  if (start >= end) {
    if (a.splits == 1)
      for (int i = tid; i < nq * D; i += kThreads) out[i] = DT<T>::from_f(0.f);
    return;  // the merge counts the splits that hold keys
  }
  const T* q = (const T*)a.q + (int64_t)b * a.q_stride + (int64_t)h0 * D;
  for (int i = tid; i < NQ * D; i += kThreads)
    sm_q[i / D][i % D] = i < nq * D ? DT<T>::to_f(q[i]) : 0.f;
  __syncthreads();
  for (int g = warp; g < NQ; g += kWarps) {
    float s = 0.f;
    for (int e = lane; e < D; e += 32) s += sm_q[g][e];
    s = warp_sum(s);
    if (lane == 0) sm_sum[g] = s;
  }
  __syncthreads();

  const uint8_t* recs = a.q4 + (int64_t)b * a.qbs + (int64_t)hk * a.qhs;
  float m[NQ], l[NQ], z[NQ], o[NQ][EPL];
#pragma unroll
  for (int g = 0; g < NQ; ++g) {
    m[g] = -INFINITY;
    l[g] = z[g] = 0.f;
#pragma unroll
    for (int e = 0; e < EPL; ++e) o[g][e] = 0.f;
  }
  for (int base = start + warp * 32; base < end; base += kThreads) {
    const int n = min(32, end - base);
    const bool valid = lane < n;
    const uint8_t* rec = recs + (int64_t)(base + (valid ? lane : 0)) * (D + 16);
    const float4 meta = *reinterpret_cast<const float4*>(rec + D);
    float s[NQ];
#pragma unroll
    for (int g = 0; g < NQ; ++g) s[g] = 0.f;
#pragma unroll 1
    for (int c = 0; c < D / 8; ++c) {
      const uint32_t w = *reinterpret_cast<const uint32_t*>(rec + c * 4);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float code = (float)((w >> (4 * i)) & 15u);
#pragma unroll
        for (int g = 0; g < NQ; ++g) s[g] = fmaf(sm_q[g][c * 8 + i], code, s[g]);
      }
    }
    float pv[NQ];
#pragma unroll
    for (int g = 0; g < NQ; ++g) {
      const float score = a.scale_log2 * (meta.x * s[g] + meta.y * sm_sum[g]);
      const float top = fmaxf(m[g], warp_max(valid ? score : -INFINITY));
      const float alpha = exp2f(m[g] - top);
      const float p = valid ? exp2f(score - top) : 0.f;
      m[g] = top;
      l[g] = l[g] * alpha + p;  // this lane's share; lanes are added up at the end
      z[g] = z[g] * alpha + (valid ? p * meta.w : 0.f);
      pv[g] = valid ? p * meta.z : 0.f;
#pragma unroll
      for (int e = 0; e < EPL; ++e) o[g][e] *= alpha;
    }
    const uint8_t* vrow = recs + (int64_t)base * (D + 16) + D / 2;
    for (int j = 0; j < n; ++j, vrow += D + 16) {
      float code[EPL];
      if constexpr (EPL == 1) {
        code[0] = (float)((vrow[lane >> 1] >> (4 * (lane & 1))) & 15);
      } else if constexpr (EPL == 2) {
        const uint32_t w = vrow[lane];
        code[0] = (float)(w & 15u), code[1] = (float)(w >> 4);
      } else {
        const uint32_t w = *reinterpret_cast<const uint16_t*>(vrow + 2 * lane);
#pragma unroll
        for (int e = 0; e < EPL; ++e) code[e] = (float)((w >> (4 * e)) & 15u);
      }
#pragma unroll
      for (int g = 0; g < NQ; ++g) {
        const float w = __shfl_sync(0xffffffffu, pv[g], j);
#pragma unroll
        for (int e = 0; e < EPL; ++e) o[g][e] = fmaf(w, code[e], o[g][e]);
      }
    }
  }
#pragma unroll
  for (int g = 0; g < NQ; ++g) {
    l[g] = warp_sum(l[g]);
    z[g] = warp_sum(z[g]);
    if (lane == 0) sm_m[warp][g] = m[g], sm_l[warp][g] = l[g], sm_z[warp][g] = z[g];
#pragma unroll
    for (int e = 0; e < EPL; ++e) sm_o[warp][g][lane * EPL + e] = o[g][e];
  }
  __syncthreads();
  for (int i = tid; i < nq * D; i += kThreads) {
    const int g = i / D, e = i % D;
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) M = fmaxf(M, sm_m[w][g]);
    float L = 0.f, O = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (start + w * 32 >= end) continue;  // this warp had no keys
      const float f = exp2f(sm_m[w][g] - M);
      L += f * sm_l[w][g];
      O += f * (sm_o[w][g][e] + sm_z[w][g]);
    }
    if (a.splits == 1) {
      out[i] = DT<T>::from_f(O / L);
    } else {
      const int64_t slot = ((int64_t)b * a.n_heads + h0 + g) * a.splits + split;
      a.ws_o[slot * D + e] = O;
      if (e == 0) a.ws_ml[2 * slot] = M, a.ws_ml[2 * slot + 1] = L;
    }
  }
}

// out = sum_s 2^(m_s - M) o_s / sum_s 2^(m_s - M) l_s over the splits that hold keys: one CTA per
// (sequence, query head), one thread per output element.
template <typename T, int D>
__global__ void __launch_bounds__(D) decode_q4_merge_kernel(const Args a) {
  pdl_wait();
  pdl_trigger();
  const int64_t bh = blockIdx.x;
  const int len = live_length(a.seqlens, (int)(bh / a.n_heads), a.max_len);
  const int n = (len + a.chunk - 1) / a.chunk;
  const float* ml = a.ws_ml + bh * a.splits * 2;
  const float* o = a.ws_o + bh * a.splits * D + threadIdx.x;
  float M = -INFINITY, L = 0.f, O = 0.f;
  for (int s = 0; s < n; ++s) M = fmaxf(M, ml[2 * s]);
  for (int s = 0; s < n; ++s) {
    const float f = exp2f(ml[2 * s] - M);
    L += f * ml[2 * s + 1];
    O += f * o[(int64_t)s * D];
  }
  ((T*)a.out)[bh * D + threadIdx.x] = DT<T>::from_f(n ? O / L : 0.f);
}

struct Plan {
  int chunk, splits;
};

// Key splits: whole 128-key steps, about four CTAs per SM, at most 65535 splits.
Plan plan(int64_t batch, int64_t n_heads, int64_t n_heads_kv, int64_t max_len) {
  const int64_t group = n_heads / n_heads_kv;
  const int64_t units = std::max<int64_t>(1, batch * n_heads_kv * ((group + NQ - 1) / NQ));
  const int64_t steps = std::max<int64_t>(1, (max_len + 127) / 128);
  const int64_t want = std::min<int64_t>(steps, std::max<int64_t>(1, (148 * 4 + units - 1) / units));
  const int64_t per = (steps + want - 1) / want;
  return {(int)(per * 128), (int)((steps + per - 1) / per)};
}

template <typename T, int D>
int launch(Args a, int64_t batch, int64_t n_heads_kv, cudaStream_t stream) {
  const dim3 grid((unsigned)a.splits, (unsigned)(n_heads_kv * a.q_chunks), (unsigned)batch);
  int s = hx::cuda_status(launch_ex(decode_q4_kernel<T, D>, grid, dim3(kThreads), 0, stream, 1, a),
                          "decode_q4_kernel launch");
  if (s || a.splits == 1) return s;
  return hx::cuda_status(launch_ex(decode_q4_merge_kernel<T, D>, dim3((unsigned)(batch * a.n_heads)),
                                   dim3(D), 0, stream, 1, a),
                         "decode_q4_merge_kernel launch");
}

}  // namespace

extern "C" {

size_t hx_decode_attention_q4_workspace(int64_t batch, int64_t n_heads, int64_t n_heads_kv,
                                        int64_t head_dim, int64_t max_seqlen_k) {
  if (batch <= 0 || n_heads <= 0 || n_heads_kv <= 0 || head_dim <= 0 || max_seqlen_k <= 0) return 0;
  const int splits = plan(batch, n_heads, n_heads_kv, max_seqlen_k).splits;
  return splits == 1 ? 0 : (size_t)batch * n_heads * splits * (head_dim + 2) * sizeof(float);
}

int hx_decode_attention_q4(const void* q, int64_t q_batch_stride, const void* cache_q4,
                           int64_t q4_batch_stride, int64_t q4_head_stride,
                           const int32_t* seqlens_k, int64_t batch, int64_t n_heads,
                           int64_t n_heads_kv, int64_t head_dim, int64_t max_seqlen_k,
                           float softmax_scale, void* out, void* workspace,
                           size_t workspace_bytes, int dtype, void* stream) {
  HX_REQUIRE(q && cache_q4 && seqlens_k && out, "hx_decode_attention_q4: null pointer");
  HX_REQUIRE(n_heads_kv > 0 && n_heads > 0 && n_heads % n_heads_kv == 0,
             "hx_decode_attention_q4: unsupported head grouping %lld/%lld", (long long)n_heads,
             (long long)n_heads_kv);
  HX_REQUIRE(head_dim == 32 || head_dim == 64 || head_dim == 128,
             "hx_decode_attention_q4: head_dim %lld unsupported (32, 64 or 128)",
             (long long)head_dim);
  HX_REQUIRE(max_seqlen_k >= 0 && max_seqlen_k < (int64_t(1) << 30) && batch >= 0 && batch < 65536,
             "hx_decode_attention_q4: bad sizes");
  const int esz = dtype == HX_F32 ? 4 : 2;
  HX_REQUIRE((uintptr_t)cache_q4 % 16 == 0 && q4_batch_stride % 16 == 0 && q4_head_stride % 16 == 0 &&
                 q4_head_stride >= max_seqlen_k * (head_dim + 16),
             "hx_decode_attention_q4: the 4-bit cache must be 16-byte aligned with contiguous records");
  HX_REQUIRE((uintptr_t)q % 16 == 0 && (q_batch_stride * esz) % 16 == 0 && (uintptr_t)out % 16 == 0,
             "hx_decode_attention_q4: q and out must be 16-byte aligned");
  if (batch == 0) return HX_OK;
  const Plan p = plan(batch, n_heads, n_heads_kv, max_seqlen_k);
  Args a;
  a.q = q;
  a.q4 = (const uint8_t*)cache_q4;
  a.seqlens = seqlens_k;
  a.out = out;
  a.qbs = q4_batch_stride;
  a.qhs = q4_head_stride;
  a.q_stride = q_batch_stride;
  a.max_len = max_seqlen_k;
  a.n_heads = (int)n_heads;
  a.group = (int)(n_heads / n_heads_kv);
  a.q_chunks = (a.group + NQ - 1) / NQ;
  HX_REQUIRE(n_heads_kv * a.q_chunks < 65536, "hx_decode_attention_q4: too many heads");
  a.chunk = p.chunk;
  a.splits = p.splits;
  a.scale_log2 = softmax_scale * 1.4426950408889634f;
  const size_t need = hx_decode_attention_q4_workspace(batch, n_heads, n_heads_kv, head_dim, max_seqlen_k);
  HX_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && (uintptr_t)workspace % 16 == 0),
             "hx_decode_attention_q4: workspace too small (%zu < %zu) or misaligned",
             workspace_bytes, need);
  a.ws_o = (float*)workspace;
  a.ws_ml = need ? a.ws_o + (size_t)batch * n_heads * p.splits * head_dim : nullptr;
  cudaStream_t s = (cudaStream_t)stream;
  HX_DISPATCH_DTYPE(dtype, T, {
    if (head_dim == 32) return launch<T, 32>(a, batch, n_heads_kv, s);
    if (head_dim == 64) return launch<T, 64>(a, batch, n_heads_kv, s);
    return launch<T, 128>(a, batch, n_heads_kv, s);
  });
  return HX_OK;
}

}  // extern "C"
