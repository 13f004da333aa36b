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
//
// Bytes bound these kernels: 16 sequences of up to 2048 rows, 32 heads of 128, bf16 take 104 us into records
// and 61 us back (387 MB each at 3.7 and 6.3 TB/s). Writing is held back by the arithmetic of the codes
// (158 instructions per warp for eight elements a lane in all, 78 % of the issue slots; a 64-bit
// division per row had made it 170 us).
#include "common.cuh"

namespace {

constexpr int kThreads = 256;
constexpr int E = 8;  // row elements per thread: 16 bytes of 16-bit input, one 32-bit word of codes

// Eight row elements as they lie in memory.
template <typename T> struct Raw {
  uint4 v[sizeof(T) / 2];
  HX_DEVICE void load(const T* p) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) v[i] = *(reinterpret_cast<const uint4*>(p) + i);
  }
  HX_DEVICE void to_f(float (&x)[E]) const {
#pragma unroll
    for (int i = 0; i < E; ++i) x[i] = DT<T>::to_f(reinterpret_cast<const T*>(v)[i]);
  }
};

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

HX_DEVICE float min_nan(float a, float b) {
  float y;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

// Minimum and maximum of a row held by U adjacent lanes, NaN in both if there is one. 16-bit rows go as
// packed pairs, the maximum as the negated minimum of the negated row (both exact), one shuffle a step.
template <typename T, int U> HX_DEVICE void row_range(const Raw<T>& raw, float& lo, float& hi) {
  if constexpr (sizeof(T) == 2) {
    using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    const T2* e = reinterpret_cast<const T2*>(raw.v);
    const T2 least = __hmin2_nan(__hmin2_nan(e[0], e[1]), __hmin2_nan(e[2], e[3]));
    const T2 most = __hmax2_nan(__hmax2_nan(e[0], e[1]), __hmax2_nan(e[2], e[3]));
    T2 p;
    p.x = __hmin_nan(least.x, least.y);
    p.y = __hneg(__hmax_nan(most.x, most.y));
#pragma unroll
    for (int o = U / 2; o > 0; o >>= 1) {
      const uint32_t other = __shfl_xor_sync(0xffffffffu, *reinterpret_cast<const uint32_t*>(&p), o);
      p = __hmin2_nan(p, *reinterpret_cast<const T2*>(&other));
    }
    lo = DT<T>::to_f(p.x);
    hi = -DT<T>::to_f(p.y);
  } else {
    const float* e = reinterpret_cast<const float*>(raw.v);
    float top = -e[0];
    lo = e[0];
#pragma unroll
    for (int i = 1; i < E; ++i) lo = min_nan(lo, e[i]), top = min_nan(top, -e[i]);
#pragma unroll
    for (int o = U / 2; o > 0; o >>= 1) {
      lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
      top = min_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
    }
    hi = -top;
  }
}

// Encodes a row held by U adjacent lanes (E elements each; U a power of two, all lanes of the warp
// call it) into its record: `half` 0 = K, 1 = V, `lane` the lane's place in the row.
template <typename T, int U> HX_DEVICE void encode_row(const Raw<T>& raw, int lane, int half, bool live,
                                                      uint8_t* rec) {
  constexpr int D = U * E;
  float lo, hi;
  row_range<T, U>(raw, lo, hi);
  const float span = __fsub_rn(hi, lo);
  uint32_t word = 0;
  float scale = 0.f;
  if (!(span < INFINITY)) {
    scale = lo = __int_as_float(0x7fffffff);
  } else if (span >= 7.888609052210118e-31f) {  // 2^-100
    scale = __fdiv_rn(span, 15.f);
    const float rate = __fdiv_rn(15.f, span);
    float x[E];
    raw.to_f(x);
#pragma unroll
    for (int i = 0; i < E; ++i) {
      // Adding 1.5 * 2^23 leaves the nearest integer (ties to even) in the low bits; it is at most 15,
      // span * rate being 15 up to two roundings.
      const float y = __fadd_rn(__fmul_rn(__fsub_rn(x[i], lo), rate), 12582912.f);
      word |= (__float_as_uint(y) & 15u) << (4 * i);
    }
  }
  if (!live) return;
  *reinterpret_cast<uint32_t*>(rec + half * (D / 2) + lane * 4) = word;
  if (lane == 0) *reinterpret_cast<float2*>(rec + D + half * 8) = make_float2(scale, lo);
}

// Rows of a cache and positions of a 4-bit cache that belong together.
struct Rows {
  int64_t cbs, css;            // cache: elements per sequence and row
  int64_t qbs, qhs, b0;        // 4-bit cache: bytes per sequence and head, first sequence
  int64_t max_rows, max_seq;
  const int32_t *starts, *counts;
  int n_heads_kv, row_step;    // rows from one step of a unit to its next
};

// The range of sequence b: rows [0, n) and positions from `start`. Rows the buffers do not hold are not
// touched; the caller learns of them.
HX_DEVICE int64_t live_rows(const Rows& p, int b, int64_t& start) {
  start = p.starts ? p.starts[b] : 0;
  const int64_t want = p.counts[b], n = start < 0 ? 0 : min(want, min(p.max_rows, p.max_seq - start));
  if ((want < 0 || start < 0 || n < want) && blockIdx.x == 0 && threadIdx.x == 0)
    record_device_error(HX_DEVERR_BAD_ARGUMENT);
  return n;
}

// cache -> records. A unit is U lanes on one (K or V, head), heads fastest, so a warp reads consecutive
// bytes of a row; the grid is a whole number of rows, so a unit keeps its head from step to step.
template <typename T, int U>
__global__ void __launch_bounds__(kThreads) quantize_kernel(const T* __restrict__ cache, uint8_t* __restrict__ q4,
                                                           const Rows p) {
  constexpr int D = U * E, kRec = D + 16;
  pdl_wait();
  pdl_trigger();
  const int b = blockIdx.y, lane = threadIdx.x % U, slots = 2 * p.n_heads_kv;
  int64_t start;
  const int64_t n = live_rows(p, b, start);
  const unsigned unit = blockIdx.x * (kThreads / U) + threadIdx.x / U;
  int64_t row = unit / (unsigned)slots;
  const int slot = (int)(unit - (unsigned)row * slots), half = slot >= p.n_heads_kv, head = slot - half * p.n_heads_kv;
  const T* from = cache + b * p.cbs + row * p.css + slot * D + lane * E;
  uint8_t* to = q4 + (p.b0 + b) * p.qbs + head * p.qhs + (start + row) * kRec;
  const int64_t from_step = p.row_step * p.css;
  // Lanes of a warp may be on different rows: it stays until all are done. Two loads in flight.
  while (__any_sync(0xffffffffu, row < n)) {
    Raw<T> raw[2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (row + i * p.row_step < n) raw[i].load(from + i * from_step);
#pragma unroll
    for (int i = 0; i < 2; ++i)
      encode_row<T, U>(raw[i], lane, half, row + i * p.row_step < n, to + (int64_t)i * p.row_step * kRec);
    row += 2 * p.row_step;
    from += 2 * from_step;
    to += (int64_t)2 * p.row_step * kRec;
  }
}

// records -> cache, by the same units.
template <typename T, int U>
__global__ void __launch_bounds__(kThreads) dequantize_kernel(const uint8_t* __restrict__ q4, T* __restrict__ cache,
                                                             const Rows p) {
  constexpr int D = U * E, kRec = D + 16;
  pdl_wait();
  pdl_trigger();
  const int b = blockIdx.y, lane = threadIdx.x % U, slots = 2 * p.n_heads_kv;
  int64_t start;
  const int64_t n = live_rows(p, b, start);
  const unsigned unit = blockIdx.x * (kThreads / U) + threadIdx.x / U;
  int64_t row = unit / (unsigned)slots;
  const int slot = (int)(unit - (unsigned)row * slots), half = slot >= p.n_heads_kv, head = slot - half * p.n_heads_kv;
  const uint8_t* from = q4 + (p.b0 + b) * p.qbs + head * p.qhs + (start + row) * kRec + half * (D / 2) + lane * 4;
  const int to_meta = D + half * 8 - half * (D / 2) - lane * 4;
  T* to = cache + b * p.cbs + row * p.css + slot * D + lane * E;
  const int64_t to_step = p.row_step * p.css, from_step = (int64_t)p.row_step * kRec;
  for (; row < n; row += 2 * p.row_step, from += 2 * from_step, to += 2 * to_step) {
    uint32_t word[2] = {};
    float2 meta[2] = {};
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (row + i * p.row_step < n) {
        word[i] = __ldg(reinterpret_cast<const uint32_t*>(from + i * from_step));
        meta[i] = __ldg(reinterpret_cast<const float2*>(from + i * from_step + to_meta));
      }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (row + i * p.row_step >= n) break;
      float x[E];
#pragma unroll
      for (int j = 0; j < E; ++j) {
        const float code = __uint_as_float(((word[i] >> (4 * j)) & 15u) | 0x4b000000u) - 8388608.f;
        x[j] = fmaf(meta[i].x, code, meta[i].y);
      }
      store8(to + i * to_step, x);
    }
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
  Raw<T> raw;
  raw.load(src + lane * E);
  if (unit < n_heads + n_heads_kv) {
    float x[E];
    raw.to_f(x);
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
      Raw<T> partner;
      partner.load(src + (low ? lane + U / 2 : lane - U / 2) * E);
      float y[E];
      partner.to_f(y);
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const int f = (low ? lane : lane - U / 2) * E + i;
        const float c = DT<T>::to_f(cs[f]), s = DT<T>::to_f(sn[f]);
        x[i] = round_to<T>(low ? __fsub_rn(__fmul_rn(x[i], c), __fmul_rn(y[i], s))
                               : __fadd_rn(__fmul_rn(y[i], s), __fmul_rn(x[i], c)));
      }
    }
    if (live && unit < n_heads) store8(q_out + (token * n_heads + unit) * D + lane * E, x);
    store8(reinterpret_cast<T*>(raw.v), x);
  }
  const int half = unit >= n_heads + n_heads_kv;
  const int head = unit - n_heads - half * n_heads_kv;
  encode_row<T, U>(raw, lane, half, live && unit >= n_heads,
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

// CTAs per sequence: enough for two steps on every row the buffers can hold, at most a few waves in all
// (the kernels stride over the live rows, which only the device knows), a whole number of rows.
unsigned row_blocks(Rows& p, int64_t rows, int64_t batch, int U) {
  const int64_t slots = 2 * p.n_heads_kv, units = kThreads / U;
  int64_t whole = slots, rest = units;  // CTAs that make whole rows: slots / gcd(slots, units)
  while (rest) std::swap(whole, rest), rest %= whole;
  whole = slots / whole;
  const int64_t want = (rows * slots + 2 * units - 1) / (2 * units);
  const int64_t cap = std::max<int64_t>(1, (int64_t)device_sm_count() * 32 / std::max<int64_t>(batch, 1));
  const int64_t blocks = (std::max<int64_t>(1, std::min(want, cap)) + whole - 1) / whole * whole;
  p.row_step = (int)(blocks * units / slots);
  return (unsigned)blocks;
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
  HX_REQUIRE(batch >= 0 && batch < 65536 && cache_rows >= 0 && n_heads_kv < 32768, "hx_quantize_cache_q4: bad sizes");
  if (batch == 0 || cache_rows == 0) return HX_OK;
  Rows p{cache_batch_stride, cache_seq_stride, q4_batch_stride, q4_head_stride, q4_batch_offset,
         cache_rows, q4_max_seq, starts, counts, (int)n_heads_kv, 0};
  HX_DISPATCH_DTYPE(dtype, T, HX_Q4_DIM(head_dim, U, {
    const unsigned blocks = row_blocks(p, cache_rows, batch, U);
    const int s = hx::cuda_status(
        launch_ex(quantize_kernel<T, U>, dim3(blocks, (unsigned)batch), dim3(kThreads), 0,
                  (cudaStream_t)stream, 1, (const T*)cache, (uint8_t*)cache_q4, p),
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
  HX_REQUIRE(batch >= 0 && batch < 65536 && cache_rows >= 0 && n_heads_kv < 32768, "hx_dequantize_cache_q4: bad sizes");
  if (batch == 0 || cache_rows == 0) return HX_OK;
  Rows p{cache_batch_stride, cache_seq_stride, q4_batch_stride, q4_head_stride, q4_batch_offset,
         cache_rows, q4_max_seq, starts, counts, (int)n_heads_kv, 0};
  HX_DISPATCH_DTYPE(dtype, T, HX_Q4_DIM(head_dim, U, {
    const unsigned blocks = row_blocks(p, cache_rows, batch, U);
    const int s = hx::cuda_status(
        launch_ex(dequantize_kernel<T, U>, dim3(blocks, (unsigned)batch), dim3(kThreads), 0,
                  (cudaStream_t)stream, 1, (const uint8_t*)cache_q4, (T*)cache, p),
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
