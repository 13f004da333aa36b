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
// across D for the values. Codes are taken about the code of zero (the nearest, where a row has no zero), so that
// sums of products are of the values' size, not of the codes', and lose no more than plain f32 sums do.
HX_DEVICE float code_of_zero(float scale, float low) { return scale > 0.f ? fminf(fmaxf(-low / scale, 0.f), 15.f) : 0.f; }

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
    const float k_zero = code_of_zero(meta.x, meta.y), k_base = fmaf(meta.x, k_zero, meta.y);
    const float v_zero = code_of_zero(meta.z, meta.w), v_base = fmaf(meta.z, v_zero, meta.w);
    float s[NQ];
#pragma unroll
    for (int g = 0; g < NQ; ++g) s[g] = 0.f;
#pragma unroll 1
    for (int c = 0; c < D / 8; ++c) {
      const uint32_t w = *reinterpret_cast<const uint32_t*>(rec + c * 4);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float code = (float)((w >> (4 * i)) & 15u) - k_zero;
#pragma unroll
        for (int g = 0; g < NQ; ++g) s[g] = fmaf(sm_q[g][c * 8 + i], code, s[g]);
      }
    }
    float pv[NQ];
#pragma unroll
    for (int g = 0; g < NQ; ++g) {
      const float score = a.scale_log2 * (meta.x * s[g] + k_base * sm_sum[g]);
      const float top = fmaxf(m[g], warp_max(valid ? score : -INFINITY));
      const float alpha = exp2f(m[g] - top);
      const float p = valid ? exp2f(score - top) : 0.f;
      m[g] = top;
      l[g] = l[g] * alpha + p;  // this lane's share; lanes are added up at the end
      z[g] = z[g] * alpha + (valid ? p * v_base : 0.f);
      pv[g] = valid ? p * meta.z : 0.f;
#pragma unroll
      for (int e = 0; e < EPL; ++e) o[g][e] *= alpha;
    }
    const uint8_t* vrow = recs + (int64_t)base * (D + 16) + D / 2;
    for (int j = 0; j < n; ++j, vrow += D + 16) {
      const float zero = __shfl_sync(0xffffffffu, v_zero, j);
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
      for (int e = 0; e < EPL; ++e) code[e] -= zero;
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

// ------------------------------------------------------------------------------------------
// Tensor-core kernel (f16/bf16): S = K codes . q^T and O^T = V codes^T . P'^T with P' = p * v_scale, on
// mma.m16n8k16 with f16 operands and f32 sums; the 16 rows of A are positions (S) or output elements
// (O), its 8 columns query heads.
//   - The bits of a code are an f16 as they stand: below 2^11 an f16's value is its bits times 2^-24
//     (subnormals and the first binade). A masked word is an operand register: w & 0x000f000f
//     holds codes * 2^-24, w & 0x00f000f0 codes * 2^-20; no bias, no conversion, nothing rounded.
//     The tensor core takes subnormals as they are.
//   - q goes in as f16 times a power of two of its own per head (max |q| in [2^9, 2^10), times 16
//     where the codes are not): bf16 and f16 values down to 2^-24 of the head's largest are exact.
//   - The order of the D elements in S and of the output elements in O is free, so each lane takes
//     the words it can read with one wide load: for S 1/4 of a position's K codes, for O 1/8 of
//     a position's V codes (bytes of two positions joined with one permute).
//   - P' enters as f16, relative to the largest P' seen (the running reference r follows
//     s + log2 v_scale, not s, down to v_scale = 2^-80): at most 2^-11 of each value off, and
//     2^-25 * 2^-7 of the largest. For f16 outputs, whose half step is no coarser, P' is the sum of two f16 (2^-22).
//   - Where values average out, sums of codes are many times the output, and so would be what they lose: the
//     rounding of P', and what the tensor core cuts off its sums, always towards zero (of 20000 positions 2e-4
//     of the output). So codes are taken about 7.5: the sum of 7.5 P' that goes off is the tensor core's own,
//     rounded and cut alike (the mean of eight rows of codes 6 to 9), and a row's middle v_min + 7.5 v_scale
//     comes in with p itself, in f32.
//   - As measured, products are cut at about 2^-24 of the largest with a subnormal operand counted as 2^-14, so
//     a code in the lowest bits keeps 14. For f16 outputs, even elements move to bit 4 and up as well (bf16 rounds
//     eight times as much off and does without, 5 % of its time).
//   - S comes out position-major; movmatrix turns it into the B operand of O.
// Each warp streams 32-position tiles through a ring of its own (bulk copies by its lane 0, one
// mbarrier per stage): no block barrier until the warps' partials are added up at the end.
// NT tiles of eight columns; NJ = 1 puts at most four heads into the even columns, which halves the
// softmax work per position.
// Measured (bf16, D = 128): 32 sequences of up to 2478 positions, 32 heads, 190 MB of records, 46.5 us
// (4.1 TB/s, 0.62 of the measured copy rate; f16 53.6 us); 4 documents of up to 65536, 64 heads on 8, 205 MB,
// 50 us (4.1 TB/s, 0.63; f16 55.7 us). What bounds it: instructions per position (225 per warp and 16
// positions, of which 88 unpack codes on the half-rate ALU pipe) at twelve warps an SM, and uneven CTAs at ragged
// lengths. An equal split over persistent CTAs was slower (59 and 50 us): many short runs leave some
// CTAs with a run's fixed cost twenty times over.
// ------------------------------------------------------------------------------------------
constexpr int kTile = 32;    // positions per stage
constexpr int kStages = 4;

// Transpose of the 8x8 16-bit matrix that a warp holds one row pair per lane.
HX_DEVICE uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

HX_DEVICE float lg2_approx(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <int D, int NT>
struct McSmem {
  static constexpr int kRing = kWarps * kStages * kTile * (D + 16);
  static constexpr int kMerge = kWarps * NT * 8 * D * 4;
  static constexpr int kBytes = (kRing > kMerge ? kRing : kMerge);
};

// State of one warp's online softmax. Per lane, for columns 2t + j of each tile of eight: the
// reference r (the same in all lanes of equal t), this lane's shares of sum p and of the sum of p times the rows'
// middles (z), the output elements of its rows times 2^-20 (bf16: even elements times 2^-24), and c, the
// outputs of rows of codes 6, 6, 7, 7, 8, 8, 9, 9 as the even and the odd elements hold them (f16: one for both).
template <int D, int NT, int NJ>
struct Softmax {
  float r[NT][NJ], l[NT][NJ], z[NT][NJ], o[NT][D / 16][4], c[NT][4];
};

// What the reference follows of a row's values is log2 of v_scale, or of 2^-24 |v_min| where that is more (flat rows,
// so that p v_min stays finite), but no less than this (rows of zeros): p then stays below 2^95, a sum of 2^30
// of them in f32, and a P' of the smallest v_scale that records have (2^-104) is still 2^-17 or more at the top.
constexpr float kFloor = -80.f;

// Sums move to a reference that is 2^(2 log2 half) higher. A row of zeros may be 2^200 away from one of large values:
// the factor is 0 in f32 then, as it may be for o and z, but not for l.
HX_DEVICE float scale_l(float l, float half) { return l * half * half; }

// One tile of n positions (kFull: n = kTile) in shared memory.
template <typename T, int D, int NT, int NJ, bool kFull>
HX_DEVICE void attend_tile(const uint8_t* tile, int n, float scale_log2, const uint32_t (&qf)[NT][D / 16][2],
                           const float (&qscale)[NT][NJ], const float (&qsum)[NT][NJ],
                           Softmax<D, NT, NJ>& st) {
  constexpr int kRec = D + 16, W = D / 32, OT = D / 16;
  constexpr bool kTwo = std::is_same<T, __half>::value;  // P' as the sum of two f16
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  float s[2][NT][4];
  float4 meta[2][2];
#pragma unroll
  for (int sub = 0; sub < 2; ++sub) {
    const uint8_t* r0 = tile + (sub * 16 + g) * kRec;
    const uint8_t* r1 = r0 + 8 * kRec;
    uint32_t k0[W], k1[W];
    if constexpr (W == 4) {
      const uint4 x = *reinterpret_cast<const uint4*>(r0 + 16 * t), y = *reinterpret_cast<const uint4*>(r1 + 16 * t);
      k0[0] = x.x, k0[1] = x.y, k0[2] = x.z, k0[3] = x.w;
      k1[0] = y.x, k1[1] = y.y, k1[2] = y.z, k1[3] = y.w;
    } else if constexpr (W == 2) {
      const uint2 x = *reinterpret_cast<const uint2*>(r0 + 8 * t), y = *reinterpret_cast<const uint2*>(r1 + 8 * t);
      k0[0] = x.x, k0[1] = x.y, k1[0] = y.x, k1[1] = y.y;
    } else {
      k0[0] = *reinterpret_cast<const uint32_t*>(r0 + 4 * t);
      k1[0] = *reinterpret_cast<const uint32_t*>(r1 + 4 * t);
    }
    meta[sub][0] = *reinterpret_cast<const float4*>(r0 + D);
    meta[sub][1] = *reinterpret_cast<const float4*>(r1 + D);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < 4; ++j) s[sub][nt][j] = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w)
#pragma unroll
      for (int h = 0; h < 2; ++h) {  // elements (0,4), (1,5), then (2,6), (3,7) of the word
        const uint32_t x = k0[w] >> (8 * h), y = k1[w] >> (8 * h);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
          mma_f16(s[sub][nt], x & 0x000f000fu, y & 0x000f000fu, x & 0x00f000f0u, y & 0x00f000f0u,
                  qf[nt][2 * w + h][0], qf[nt][2 * w + h][1]);
      }
  }
  // Scores in base 2, and the tile's largest score + log2 v_scale per head.
  float top[NT][NJ];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int j = 0; j < NJ; ++j) top[nt][j] = -INFINITY;
#pragma unroll
  for (int sub = 0; sub < 2; ++sub)
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const float ks = meta[sub][r].x * scale_log2, km = meta[sub][r].y * scale_log2;
      const float lv = fmaxf(lg2_approx(fmaxf(meta[sub][r].z, fabsf(meta[sub][r].w) * 0x1p-24f)), kFloor);
      const bool live = kFull || sub * 16 + r * 8 + g < n;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          float& x = s[sub][nt][2 * r + j];
          x = fmaf(ks, x * qscale[nt][j], km * qsum[nt][j]);
          if (!live) x = -INFINITY;
          top[nt][j] = fmaxf(top[nt][j], x + lv);
        }
    }
  bool grows = false;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
#pragma unroll
      for (int x = 4; x < 32; x <<= 1)
        top[nt][j] = fmaxf(top[nt][j], __shfl_xor_sync(0xffffffffu, top[nt][j], x));
      grows |= top[nt][j] > st.r[nt][j] + 15.f;
    }
  // The reference keeps P' below 2^15; it moves only when a tile would leave that range.
  if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const float next = fmaxf(st.r[nt][j], top[nt][j] - 7.f);
        const float half = ex2_approx(0.5f * (st.r[nt][j] - next));
        st.r[nt][j] = next;
        const float f = half * half;
        st.l[nt][j] = scale_l(st.l[nt][j], half);
        st.z[nt][j] *= f;
#pragma unroll
        for (int i = 0; i < OT; ++i) st.o[nt][i][j] *= f, st.o[nt][i][2 + j] *= f;
        st.c[nt][j] *= f;
        if (!kTwo) st.c[nt][2 + j] *= f;
      }
  }
#pragma unroll
  for (int sub = 0; sub < 2; ++sub) {
    uint32_t bh[NT][2], bl[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const bool live = kFull || sub * 16 + r * 8 + g < n;  // stale scales may be NaN
        const float middle = fmaf(7.5f, meta[sub][r].z, meta[sub][r].w);
        float pv[2] = {0.f, 0.f};
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          const float p = ex2_approx(s[sub][nt][2 * r + j] - st.r[nt][j]);
          if (live) {
            st.l[nt][j] += p;
            st.z[nt][j] = fmaf(p, middle, st.z[nt][j]);
            pv[j] = p * meta[sub][r].z;
          }
        }
        const uint32_t hi = pack2<__half>(pv[0], pv[1]);
        bh[nt][r] = transpose8x8(hi);
        if constexpr (kTwo) {
          const float2 back = __half22float2(*reinterpret_cast<const __half2*>(&hi));
          bl[nt][r] = transpose8x8(pack2<__half>(pv[0] - back.x, pv[1] - back.y));
        }
      }
    const uint32_t odd = (6 + g / 2) * 0x00100010u, even = kTwo ? odd : odd >> 4;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      mma_f16(st.c[nt], even, odd, even, odd, bh[nt][0], bh[nt][1]);
      if (kTwo) mma_f16(st.c[nt], even, odd, even, odd, bl[nt][0], bl[nt][1]);
    }
    // V codes of positions 2t, 2t + 1, 2t + 8, 2t + 9: lane (g, t) takes bytes [D/16 g, D/16 (g + 1)).
    const uint8_t* v = tile + (sub * 16 + 2 * t) * kRec + D / 2 + (D / 16) * g;
    constexpr int VW = D >= 64 ? D / 64 : 1;
    uint32_t vw[4][VW];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint8_t* at = v + ((i & 1) + 8 * (i >> 1)) * kRec;
      if constexpr (D == 128) {
        const uint2 x = *reinterpret_cast<const uint2*>(at);
        vw[i][0] = x.x, vw[i][1] = x.y;
      } else if constexpr (D == 64) {
        vw[i][0] = *reinterpret_cast<const uint32_t*>(at);
      } else {
        vw[i][0] = *reinterpret_cast<const uint16_t*>(at);
      }
    }
#pragma unroll
    for (int i = 0; i < OT; ++i) {
      const uint32_t sel = (i % 4) * 0x0011u + (4 + i % 4) * 0x1100u;
      const uint32_t x = __byte_perm(vw[0][i / 4], vw[1][i / 4], sel);
      const uint32_t y = __byte_perm(vw[2][i / 4], vw[3][i / 4], sel);
      const uint32_t x0 = kTwo ? (x * 16u) & 0x00f000f0u : x & 0x000f000fu, x1 = x & 0x00f000f0u;
      const uint32_t y0 = kTwo ? (y * 16u) & 0x00f000f0u : y & 0x000f000fu, y1 = y & 0x00f000f0u;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        mma_f16(st.o[nt][i], x0, x1, y0, y1, bh[nt][0], bh[nt][1]);
        if (kTwo) mma_f16(st.o[nt][i], x0, x1, y0, y1, bl[nt][0], bl[nt][1]);
      }
    }
  }
}

template <typename T, int D, int NT, int NJ>
__global__ void __launch_bounds__(kThreads) decode_q4_mma_kernel(const Args a) {
  constexpr int kRec = D + 16, W = D / 32, OT = D / 16;
  constexpr int kHeads = NT * 4 * NJ;  // head h sits in column h (NJ = 2) or 2h (NJ = 1)
  constexpr bool kTwo = std::is_same<T, __half>::value;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint64_t full[kWarps][kStages];
  __shared__ float sm_m[kWarps][kHeads], sm_l[kWarps][kHeads];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  if (lane == 0) {
    for (int s = 0; s < kStages; ++s) mbar_init(&full[warp][s], 1);
    fence_mbar_init();
  }
  __syncwarp();
  pdl_wait();
  pdl_trigger();
  const int split = blockIdx.x, b = blockIdx.z;
  const int hk = blockIdx.y / a.q_chunks, h0 = hk * a.group + (blockIdx.y % a.q_chunks) * kHeads;
  const int nq = min(kHeads, (hk + 1) * a.group - h0);
  const int len = live_length(a.seqlens, b, a.max_len);
  const int start = split * a.chunk, end = min(start + a.chunk, len);
  T* out = (T*)a.out + ((int64_t)b * a.n_heads + h0) * D;
  if (start >= end) {
    if (a.splits == 1)
      for (int i = tid; i < nq * D; i += kThreads) out[i] = DT<T>::from_f(0.f);
    return;
  }
  const uint8_t* recs = a.q4 + (int64_t)b * a.qbs + (int64_t)hk * a.qhs;
  uint8_t* ring = smem + warp * (kStages * kTile * kRec);
  const int first = start + warp * kTile;
  const int n_tiles = first < end ? (end - first + kWarps * kTile - 1) / (kWarps * kTile) : 0;
  // Lane 0: tile i (positions first + 128 i ...) into stage i % kStages; never past the live end.
  auto load = [&](int i) {
    const int at = first + i * (kWarps * kTile);
    const uint32_t bytes = (uint32_t)min(kTile, end - at) * kRec;
    uint64_t* bar = &full[warp][i % kStages];
    mbar_arrive_expect_tx(bar, bytes);
    bulk_load(ring + (i % kStages) * (kTile * kRec), recs + (int64_t)at * kRec, bytes, bar);
  };
  if (lane == 0)
    for (int i = 0; i < min(n_tiles, kStages); ++i) load(i);

  // q as B operands: lane (g, t) holds column g's elements of K words [W t, W t + W).
  uint32_t qf[NT][2 * W][2];
  float qscale[NT][NJ], qsum[NT][NJ];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int h = NJ == 2 ? nt * 8 + g : (g & 1) ? nq : nt * 4 + g / 2;
    uint4 raw[W];
    float sum = 0.f, big = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      raw[w] = make_uint4(0, 0, 0, 0);
      if (h < nq)
        raw[w] = *reinterpret_cast<const uint4*>((const T*)a.q + (int64_t)b * a.q_stride +
                                                 (int64_t)(h0 + h) * D + (t * W + w) * 8);
      const T* e = reinterpret_cast<const T*>(&raw[w]);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float x = DT<T>::to_f(e[i]);
        sum += x;
        big = fmaxf(big, fabsf(x));
      }
    }
#pragma unroll
    for (int x = 1; x < 4; x <<= 1) {
      sum += __shfl_xor_sync(0xffffffffu, sum, x);
      big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, x));
    }
    // 2^e brings the largest element into [2^9, 2^10); e stays inside f32's exponents.
    const int e = min(max((int)((__float_as_uint(big) >> 23) & 0xff) - 127, -100), 100);
    const float f = __uint_as_float((uint32_t)(127 + 9 - e) << 23);
    const float back = __uint_as_float((uint32_t)(127 - 9 + e) << 23) * 1048576.f;  // * 2^20
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const T* q = reinterpret_cast<const T*>(&raw[w]);
      auto at = [&](int i) { return DT<T>::to_f(q[i]) * f; };
      qf[nt][2 * w][0] = pack2<__half>(at(0) * 16.f, at(4) * 16.f);
      qf[nt][2 * w][1] = pack2<__half>(at(1), at(5));
      qf[nt][2 * w + 1][0] = pack2<__half>(at(2) * 16.f, at(6) * 16.f);
      qf[nt][2 * w + 1][1] = pack2<__half>(at(3), at(7));
    }
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      qsum[nt][j] = __shfl_sync(0xffffffffu, sum, 8 * t + 4 * j);
      qscale[nt][j] = __shfl_sync(0xffffffffu, back, 8 * t + 4 * j);
    }
  }

  Softmax<D, NT, NJ> st;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      st.r[nt][j] = -INFINITY;
      st.l[nt][j] = st.z[nt][j] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < OT; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) st.o[nt][i][j] = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) st.c[nt][j] = 0.f;
  }

  int done = 0;
  for (; done < n_tiles; ++done) {
    const int stage = done % kStages;
    if (!mbar_wait_warp_timed(&full[warp][stage], (done / kStages) & 1)) break;
    const uint8_t* tile = ring + stage * (kTile * kRec);
    const int n = end - (first + done * (kWarps * kTile));
    if (n >= kTile)
      attend_tile<T, D, NT, NJ, true>(tile, kTile, a.scale_log2, qf, qscale, qsum, st);
    else
      attend_tile<T, D, NT, NJ, false>(tile, n, a.scale_log2, qf, qscale, qsum, st);
    __syncwarp();
    if (lane == 0 && done + kStages < n_tiles) load(done + kStages);
  }
  if (done < n_tiles) {  // a wait gave up: let the copies in flight land before the ring is reused
    for (int i = done; i < min(n_tiles, done + kStages); ++i)
      mbar_wait_drain(&full[warp][i % kStages], (i / kStages) & 1);
  }
  // Lane shares to warp sums, then the warps' partials through shared memory (the rings are idle).
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) {
        st.l[nt][j] += __shfl_xor_sync(0xffffffffu, st.l[nt][j], x);
        st.z[nt][j] += __shfl_xor_sync(0xffffffffu, st.z[nt][j], x);
        st.c[nt][j] += __shfl_xor_sync(0xffffffffu, st.c[nt][j], x);
        if (!kTwo) st.c[nt][2 + j] += __shfl_xor_sync(0xffffffffu, st.c[nt][2 + j], x);
      }
      const int h = (nt * 4 + t) * NJ + j;
      if (g == 0) sm_m[warp][h] = st.r[nt][j], sm_l[warp][h] = st.l[nt][j];
    }
  __syncthreads();
  float* sm_o = reinterpret_cast<float*>(smem);  // [kWarps][kHeads][D]
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int i = 0; i < OT; ++i)
#pragma unroll
      for (int j = 0; j < NJ; ++j)
        *reinterpret_cast<float2*>(sm_o + (warp * kHeads + (nt * 4 + t) * NJ + j) * D + (D / 8) * g + 2 * i) =
            make_float2(fmaf(st.o[nt][i][j] - 0.125f * st.c[nt][j], kTwo ? 1048576.f : 16777216.f, st.z[nt][j]),
                        fmaf(st.o[nt][i][2 + j] - 0.125f * st.c[nt][kTwo ? j : 2 + j], 1048576.f, st.z[nt][j]));
  __syncthreads();
  for (int i = tid; i < nq * D; i += kThreads) {
    const int q = i / D;
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) M = fmaxf(M, sm_m[w][q]);
    float L = 0.f, O = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (start + w * kTile >= end) continue;  // this warp had no positions
      const float half = exp2f(0.5f * (sm_m[w][q] - M));
      L += scale_l(sm_l[w][q], half);
      O += half * half * sm_o[w * kHeads * D + i];
    }
    if (a.splits == 1) {
      out[i] = DT<T>::from_f(O / L);
    } else {
      const int64_t slot = ((int64_t)b * a.n_heads + h0 + q) * a.splits + split;
      a.ws_o[slot * D + i % D] = O;
      if (i % D == 0) a.ws_ml[2 * slot] = M, a.ws_ml[2 * slot + 1] = L;
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
    const float half = exp2f(0.5f * (ml[2 * s] - M));
    L += scale_l(ml[2 * s + 1], half);
    O += half * half * o[(int64_t)s * D];
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

template <typename T, int D, int NT, int NJ>
int launch_mma(Args& a, int64_t batch, int64_t n_heads_kv, cudaStream_t stream) {
  a.q_chunks = ceil_div(a.group, NT * 4 * NJ);
  constexpr int smem = McSmem<D, NT>::kBytes;
  auto kern = decode_q4_mma_kernel<T, D, NT, NJ>;
  static std::atomic<uint64_t> allowed{0};  // devices where the kernel may use that much shared memory
  if (const int s = allow_shared(reinterpret_cast<const void*>(kern), smem, allowed)) return s;
  const dim3 grid((unsigned)a.splits, (unsigned)(n_heads_kv * a.q_chunks), (unsigned)batch);
  return hx::cuda_status(launch_ex(kern, grid, dim3(kThreads), smem, stream, 1, a),
                         "decode_q4_mma_kernel launch");
}

template <typename T, int D>
int launch(Args a, int64_t batch, int64_t n_heads_kv, cudaStream_t stream) {
  int s;
  if constexpr (sizeof(T) == 2) {
    s = a.group > 8   ? launch_mma<T, D, 2, 2>(a, batch, n_heads_kv, stream)
        : a.group > 4 ? launch_mma<T, D, 1, 2>(a, batch, n_heads_kv, stream)
                      : launch_mma<T, D, 1, 1>(a, batch, n_heads_kv, stream);
  } else {
    const dim3 grid((unsigned)a.splits, (unsigned)(n_heads_kv * a.q_chunks), (unsigned)batch);
    s = hx::cuda_status(launch_ex(decode_q4_kernel<T, D>, grid, dim3(kThreads), 0, stream, 1, a),
                        "decode_q4_kernel launch");
  }
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
