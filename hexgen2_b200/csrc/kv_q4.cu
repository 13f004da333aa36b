// The KV cache held in 4 bits: writing records (from 16-bit cache rows, or from the packed qkv of a
// decode step with rotary) and reading them back.
//
// A record is one position of one KV head, D + 16 bytes: D/2 bytes of K codes (element 2j in the
// low nibble of byte j, 2j + 1 in the high one), D/2 bytes of V codes, then k_scale, k_min,
// v_scale, v_min in f32. For a row x of D values (in f32):
//   lo = min x,  R = max x - lo
//   R not finite (or a NaN in x): scale = min = NaN, codes 0 -- the row reads back as NaN
//   R < 2^-100:  scale = 0, codes 0 (a flat row reads back as its minimum)
//   else         scale = R / 15, code = min(15, rint((x - lo) * (15 / R)))
// every operation one IEEE f32 operation in that order (no contraction), so the codes are the same
// wherever they are computed. A value reads back as lo + scale * code, at most half a step
// (R / 30) plus rounding away from x. Scale and minimum stay in f32: one format for every
// activation type, and 16 bytes of them bring a record to a multiple of 16 bytes (144 at D = 128),
// which bulk copies and the gather-pack of the handoff need.
//
// cache_q4 is [B, n_heads_kv, S, D + 16]: a head's positions are contiguous, so decode attention
// streams them with plain bulk copies and the live part of a head is one run of bytes.
#include "common.cuh"

namespace {

constexpr int kThreads = 256;
constexpr int E = 8;  // row elements per thread: 16 bytes of 16-bit input, one 32-bit word of codes

template <typename T> HX_DEVICE void load8(const T* p, float (&x)[E]) {
  if constexpr (sizeof(T) == 2) {
    const uint4 raw = *reinterpret_cast<const uint4*>(p);
    const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
    for (int i = 0; i < E; ++i) x[i] = DT<T>::to_f(e[i]);
  } else {
#pragma unroll
    for (int i = 0; i < E; i += 4) {
      const float4 v = *reinterpret_cast<const float4*>(p + i);
      x[i] = v.x, x[i + 1] = v.y, x[i + 2] = v.z, x[i + 3] = v.w;
    }
  }
}

template <typename T> HX_DEVICE void store8(T* p, const float (&x)[E]) {
  if constexpr (sizeof(T) == 2) {
    uint4 raw;
    raw.x = pack2<T>(x[0], x[1]);
    raw.y = pack2<T>(x[2], x[3]);
    raw.z = pack2<T>(x[4], x[5]);
    raw.w = pack2<T>(x[6], x[7]);
    *reinterpret_cast<uint4*>(p) = raw;
  } else {
    *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
  }
}

// Encodes a row held by U adjacent lanes (E elements each; U a power of two, all lanes of the warp
// call it) into its record: `half` 0 = K, 1 = V, `lane` the lane's place in the row.
template <int U> HX_DEVICE void encode_row(const float (&x)[E], int lane, int half, bool live,
                                          uint8_t* rec) {
  constexpr int D = U * E;
  float lo = x[0], hi = x[0], sum = 0.f;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    lo = fminf(lo, x[i]);
    hi = fmaxf(hi, x[i]);
    sum += x[i] - x[i];  // NaN as soon as one element is not finite (fminf / fmaxf drop NaN)
  }
#pragma unroll
  for (int o = U / 2; o > 0; o >>= 1) {
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    sum += __shfl_xor_sync(0xffffffffu, sum, o);
  }
  if (!live) return;
  const float span = __fsub_rn(hi, lo);
  uint32_t word = 0;
  float scale = 0.f;
  if (!(sum == 0.f) || isinf(span)) {
    scale = lo = __int_as_float(0x7fffffff);
  } else if (span >= 7.888609052210118e-31f) {  // 2^-100
    scale = __fdiv_rn(span, 15.f);
    const float rate = __fdiv_rn(15.f, span);
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const int code = __float2int_rn(__fmul_rn(__fsub_rn(x[i], lo), rate));
      word |= (uint32_t)min(code, 15) << (4 * i);
    }
  }
  *reinterpret_cast<uint32_t*>(rec + half * (D / 2) + lane * 4) = word;
  if (lane == 0) *reinterpret_cast<float2*>(rec + D + half * 8) = make_float2(scale, lo);
}

// Rows [0, counts[b]) of cache[b] -> records of cache_q4[b0 + b] at positions starts[b] + i.
// U lanes per (row, K or V, head); heads fastest, so a warp reads consecutive bytes of one row.
template <typename T, int U>
__global__ void __launch_bounds__(kThreads) quantize_kernel(
    const T* __restrict__ cache, int64_t cbs, int64_t css, int64_t max_rows,
    const int32_t* __restrict__ starts, const int32_t* __restrict__ counts, int n_heads_kv,
    uint8_t* __restrict__ q4, int64_t qbs, int64_t qhs, int64_t b0, int64_t max_seq) {
  constexpr int D = U * E, kUnits = kThreads / U;
  pdl_wait();
  pdl_trigger();
  const int b = blockIdx.y;
  const int64_t start = starts ? starts[b] : 0, want = counts[b];
  // Rows the buffers do not hold are not touched; the caller learns of them.
  const int64_t n = min(want, min(max_rows, max_seq - start));
  if (want < 0 || start < 0 || n < want) {
    if (blockIdx.x == 0 && threadIdx.x == 0) record_device_error(HX_DEVERR_BAD_ARGUMENT);
    if (start < 0) return;
  }
  const int lane = threadIdx.x % U;
  const int64_t units = n * 2 * n_heads_kv;
  for (int64_t base = (int64_t)blockIdx.x * kUnits; base < units; base += (int64_t)gridDim.x * kUnits) {
    const int64_t unit = base + threadIdx.x / U;
    const bool live = unit < units;
    const int64_t row = live ? unit / (2 * n_heads_kv) : 0;
    const int slot = live ? (int)(unit - row * (2 * n_heads_kv)) : 0;
    const int half = slot >= n_heads_kv, head = slot - half * n_heads_kv;
    float x[E];
    load8(cache + b * cbs + row * css + (int64_t)slot * D + lane * E, x);
    encode_row<U>(x, lane, half, live,
                  q4 + (b0 + b) * qbs + head * qhs + (start + row) * (D + 16));
  }
}

// Records of cache_q4[b0 + b] at positions starts[b] + i -> rows [0, counts[b]) of cache[b].
template <typename T, int U>
__global__ void __launch_bounds__(kThreads) dequantize_kernel(
    const uint8_t* __restrict__ q4, int64_t qbs, int64_t qhs, int64_t b0, int64_t max_seq,
    const int32_t* __restrict__ starts, const int32_t* __restrict__ counts, int n_heads_kv,
    T* __restrict__ cache, int64_t cbs, int64_t css, int64_t max_rows) {
  constexpr int D = U * E, kUnits = kThreads / U;
  pdl_wait();
  pdl_trigger();
  const int b = blockIdx.y;
  const int64_t start = starts ? starts[b] : 0, want = counts[b];
  const int64_t n = min(want, min(max_rows, max_seq - start));
  if (want < 0 || start < 0 || n < want) {
    if (blockIdx.x == 0 && threadIdx.x == 0) record_device_error(HX_DEVERR_BAD_ARGUMENT);
    if (start < 0) return;
  }
  const int lane = threadIdx.x % U;
  const int64_t units = n * 2 * n_heads_kv;
  for (int64_t unit = (int64_t)blockIdx.x * kUnits + threadIdx.x / U; unit < units;
       unit += (int64_t)gridDim.x * kUnits) {
    const int64_t row = unit / (2 * n_heads_kv);
    const int slot = (int)(unit - row * (2 * n_heads_kv));
    const int half = slot >= n_heads_kv, head = slot - half * n_heads_kv;
    const uint8_t* rec = q4 + (b0 + b) * qbs + head * qhs + (start + row) * (D + 16);
    const uint32_t word = *reinterpret_cast<const uint32_t*>(rec + half * (D / 2) + lane * 4);
    const float2 meta = *reinterpret_cast<const float2*>(rec + D + half * 8);
    float x[E];
#pragma unroll
    for (int i = 0; i < E; ++i) x[i] = fmaf(meta.x, (float)((word >> (4 * i)) & 15u), meta.y);
    store8(cache + b * cbs + row * css + (int64_t)slot * D + lane * E, x);
  }
}

// Rotary on q and k of the packed qkv, q to q_out, k and v as records at pos_start[b] + s. U lanes
// per head of q, k or v. The rotation is hx_rotary_cache_write's (f32, rounded to T); the record is
// taken from the rounded row, so it equals the one made from a 16-bit cache row of the same token.
template <typename T, int U, bool kInterleaved>
__global__ void __launch_bounds__(kThreads) rotary_q4_kernel(
    const T* __restrict__ qkv, int64_t seqlen, int n_heads, int n_heads_kv,
    const int32_t* __restrict__ pos_start, const T* __restrict__ cos_t, const T* __restrict__ sin_t,
    int64_t table_rows, T* __restrict__ q_out, uint8_t* __restrict__ q4, int64_t qbs, int64_t qhs,
    int64_t b0, int64_t max_seq) {
  constexpr int D = U * E;
  pdl_wait();
  pdl_trigger();
  const int64_t token = blockIdx.x, b = token / seqlen;
  const int64_t pos = (int64_t)pos_start[b] + (token - b * seqlen);
  if (pos < 0 || pos >= max_seq || pos >= table_rows) {
    if (threadIdx.x == 0 && blockIdx.y == 0) record_device_error(HX_DEVERR_BAD_ARGUMENT);
    return;
  }
  const int units = n_heads + 2 * n_heads_kv;
  const int at = blockIdx.y * (kThreads / U) + threadIdx.x / U, lane = threadIdx.x % U;
  const bool live = at < units;
  const int unit = live ? at : units - 1;
  const T* src = qkv + token * units * D + (int64_t)unit * D;
  float x[E];
  load8(src + lane * E, x);
  if (unit < n_heads + n_heads_kv) {
    const T* cs = cos_t + pos * (D / 2);
    const T* sn = sin_t + pos * (D / 2);
    if (kInterleaved) {
#pragma unroll
      for (int p = 0; p < E / 2; ++p) {
        const float c = DT<T>::to_f(cs[lane * (E / 2) + p]), s = DT<T>::to_f(sn[lane * (E / 2) + p]);
        const float x0 = x[2 * p], x1 = x[2 * p + 1];
        x[2 * p] = round_to<T>(__fsub_rn(__fmul_rn(x0, c), __fmul_rn(x1, s)));
        x[2 * p + 1] = round_to<T>(__fadd_rn(__fmul_rn(x0, s), __fmul_rn(x1, c)));
      }
    } else {  // pairs (i, i + D/2): the partner chunk is U/2 lanes away
      const bool low = lane < U / 2;
      float y[E];
      load8(src + (low ? lane + U / 2 : lane - U / 2) * E, y);
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const int f = (low ? lane : lane - U / 2) * E + i;
        const float c = DT<T>::to_f(cs[f]), s = DT<T>::to_f(sn[f]);
        x[i] = round_to<T>(low ? __fsub_rn(__fmul_rn(x[i], c), __fmul_rn(y[i], s))
                               : __fadd_rn(__fmul_rn(y[i], s), __fmul_rn(x[i], c)));
      }
    }
  }
  if (live && unit < n_heads) store8(q_out + (token * n_heads + unit) * D + lane * E, x);
  const int half = unit >= n_heads + n_heads_kv;
  const int head = unit - n_heads - half * n_heads_kv;
  encode_row<U>(x, lane, half, live && unit >= n_heads,
                q4 + (b0 + b) * qbs + head * qhs + pos * (D + 16));
}

int check_q4(const char* who, const void* q4, int64_t qbs, int64_t qhs, int64_t max_seq,
             int64_t n_heads_kv, int64_t head_dim) {
  HX_REQUIRE(head_dim == 32 || head_dim == 64 || head_dim == 128,
             "%s: head_dim %lld unsupported (32, 64 or 128)", who, (long long)head_dim);
  HX_REQUIRE(n_heads_kv > 0 && max_seq > 0, "%s: bad sizes", who);
  HX_REQUIRE((uintptr_t)q4 % 16 == 0 && qbs % 16 == 0 && qhs % 16 == 0 &&
                 qhs >= max_seq * (head_dim + 16),
             "%s: the 4-bit cache must be 16-byte aligned with contiguous records", who);
  return HX_OK;
}

int check_rows(const char* who, const void* cache, int64_t cbs, int64_t css, int64_t n_heads_kv,
               int64_t head_dim, int dtype) {
  const int esz = dtype == HX_F32 ? 4 : 2;
  HX_REQUIRE((uintptr_t)cache % 16 == 0 && (cbs * esz) % 16 == 0 && (css * esz) % 16 == 0 &&
                 css >= 2 * n_heads_kv * head_dim,
             "%s: cache rows must be 16-byte aligned", who);
  return HX_OK;
}

// CTAs per sequence: enough for every row the buffers can hold, at most a few waves in all (the
// kernels stride over the live rows, which only the device knows).
unsigned row_blocks(int64_t rows, int64_t batch, int64_t n_heads_kv, int U) {
  const int64_t want = (rows * 2 * n_heads_kv * U + kThreads - 1) / kThreads;
  const int64_t cap = std::max<int64_t>(1, (int64_t)device_sm_count() * 32 / std::max<int64_t>(batch, 1));
  return (unsigned)std::max<int64_t>(1, std::min(want, cap));
}

}  // namespace

#define HX_Q4_DIM(head_dim, U, ...)                 \
  switch (head_dim) {                               \
    case 32: { constexpr int U = 4; __VA_ARGS__; break; }  \
    case 64: { constexpr int U = 8; __VA_ARGS__; break; }  \
    default: { constexpr int U = 16; __VA_ARGS__; break; } \
  }

extern "C" {

int hx_quantize_cache_q4(const void* cache, int64_t cache_batch_stride, int64_t cache_seq_stride,
                         int64_t cache_rows, const int32_t* starts, const int32_t* counts,
                         int64_t batch, int64_t n_heads_kv, int64_t head_dim, void* cache_q4,
                         int64_t q4_batch_stride, int64_t q4_head_stride, int64_t q4_batch_offset,
                         int64_t q4_max_seq, int dtype, void* stream) {
  HX_REQUIRE(cache && counts && cache_q4, "hx_quantize_cache_q4: null pointer");
  if (int s = check_q4("hx_quantize_cache_q4", cache_q4, q4_batch_stride, q4_head_stride,
                       q4_max_seq, n_heads_kv, head_dim))
    return s;
  if (int s = check_rows("hx_quantize_cache_q4", cache, cache_batch_stride, cache_seq_stride,
                         n_heads_kv, head_dim, dtype))
    return s;
  HX_REQUIRE(batch >= 0 && batch < 65536 && cache_rows >= 0, "hx_quantize_cache_q4: bad sizes");
  if (batch == 0 || cache_rows == 0) return HX_OK;
  HX_DISPATCH_DTYPE(dtype, T, HX_Q4_DIM(head_dim, U, {
    const int s = hx::cuda_status(
        launch_ex(quantize_kernel<T, U>,
                  dim3(row_blocks(cache_rows, batch, n_heads_kv, U), (unsigned)batch),
                  dim3(kThreads), 0, (cudaStream_t)stream, 1, (const T*)cache, cache_batch_stride,
                  cache_seq_stride, cache_rows, starts, counts, (int)n_heads_kv,
                  (uint8_t*)cache_q4, q4_batch_stride, q4_head_stride, q4_batch_offset, q4_max_seq),
        "quantize_kernel launch");
    if (s) return s;
  }));
  HX_LAUNCH_CHECK("quantize_kernel");
  return HX_OK;
}

int hx_dequantize_cache_q4(const void* cache_q4, int64_t q4_batch_stride, int64_t q4_head_stride,
                           int64_t q4_batch_offset, int64_t q4_max_seq, const int32_t* starts,
                           const int32_t* counts, int64_t batch, int64_t n_heads_kv,
                           int64_t head_dim, void* cache, int64_t cache_batch_stride,
                           int64_t cache_seq_stride, int64_t cache_rows, int dtype, void* stream) {
  HX_REQUIRE(cache && counts && cache_q4, "hx_dequantize_cache_q4: null pointer");
  if (int s = check_q4("hx_dequantize_cache_q4", cache_q4, q4_batch_stride, q4_head_stride,
                       q4_max_seq, n_heads_kv, head_dim))
    return s;
  if (int s = check_rows("hx_dequantize_cache_q4", cache, cache_batch_stride, cache_seq_stride,
                         n_heads_kv, head_dim, dtype))
    return s;
  HX_REQUIRE(batch >= 0 && batch < 65536 && cache_rows >= 0, "hx_dequantize_cache_q4: bad sizes");
  if (batch == 0 || cache_rows == 0) return HX_OK;
  HX_DISPATCH_DTYPE(dtype, T, HX_Q4_DIM(head_dim, U, {
    const int s = hx::cuda_status(
        launch_ex(dequantize_kernel<T, U>,
                  dim3(row_blocks(cache_rows, batch, n_heads_kv, U), (unsigned)batch),
                  dim3(kThreads), 0, (cudaStream_t)stream, 1, (const uint8_t*)cache_q4,
                  q4_batch_stride, q4_head_stride, q4_batch_offset, q4_max_seq, starts, counts,
                  (int)n_heads_kv, (T*)cache, cache_batch_stride, cache_seq_stride, cache_rows),
        "dequantize_kernel launch");
    if (s) return s;
  }));
  HX_LAUNCH_CHECK("dequantize_kernel");
  return HX_OK;
}

int hx_rotary_cache_write_q4(const void* qkv, int64_t batch, int64_t seqlen, int64_t n_heads,
                             int64_t n_heads_kv, int64_t head_dim, const int32_t* pos_start,
                             const void* cos_table, const void* sin_table, int64_t table_rows,
                             int interleaved, void* q_out, void* cache_q4, int64_t q4_batch_stride,
                             int64_t q4_head_stride, int64_t q4_batch_offset, int64_t q4_max_seq,
                             int dtype, void* stream) {
  HX_REQUIRE(qkv && pos_start && cos_table && sin_table && q_out && cache_q4,
             "hx_rotary_cache_write_q4: null pointer");
  if (int s = check_q4("hx_rotary_cache_write_q4", cache_q4, q4_batch_stride, q4_head_stride,
                       q4_max_seq, n_heads_kv, head_dim))
    return s;
  HX_REQUIRE(n_heads > 0 && n_heads % n_heads_kv == 0 && n_heads < 65536 && batch >= 0 &&
                 seqlen >= 0 && batch * seqlen < (int64_t(1) << 31),
             "hx_rotary_cache_write_q4: bad sizes");
  HX_REQUIRE((uintptr_t)qkv % 16 == 0 && (uintptr_t)q_out % 16 == 0,
             "hx_rotary_cache_write_q4: qkv and q_out must be 16-byte aligned");
  if (batch == 0 || seqlen == 0) return HX_OK;
  HX_DISPATCH_DTYPE(dtype, T, HX_Q4_DIM(head_dim, U, {
    const unsigned y = (unsigned)ceil_div((n_heads + 2 * n_heads_kv) * U, kThreads);
    auto kern = interleaved ? rotary_q4_kernel<T, U, true> : rotary_q4_kernel<T, U, false>;
    const int s = hx::cuda_status(
        launch_ex(kern, dim3((unsigned)(batch * seqlen), y), dim3(kThreads), 0,
                  (cudaStream_t)stream, 1, (const T*)qkv, seqlen, (int)n_heads, (int)n_heads_kv,
                  pos_start, (const T*)cos_table, (const T*)sin_table, table_rows, (T*)q_out,
                  (uint8_t*)cache_q4, q4_batch_stride, q4_head_stride, q4_batch_offset, q4_max_seq),
        "rotary_q4_kernel launch");
    if (s) return s;
  }));
  HX_LAUNCH_CHECK("rotary_q4_kernel");
  return HX_OK;
}

}  // extern "C"
