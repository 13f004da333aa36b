// Products with 4-bit weights and group scales for decode batches:
//   c[m, n] = sum_g s[n, g] * sum_{k in group g} a[m, k] * (code[n, k] - 8)
// w [N, K / 2] bytes (element 2j in the low nibble of byte j, 2j + 1 in the high one), scales
// [N, K / group] in the activation type, groups of 32, 64 or 128 along K. The epilogues are
// hx_gemm's (none, + residual, SwiGLU over rows interleaved in blocks of 16), evaluated in f32 and
// rounded once.
#include "common.cuh"

namespace {

constexpr int kThreads = 128;
constexpr int MB = 8;  // activation rows per pass over the weights

struct Args {
  const void* a;
  const uint8_t* w;
  const void* scales;
  const void* residual;
  void* out;
  int64_t lda, ldr, ldo;
  int M, N, K, group;
};

HX_DEVICE float silu_f(float g) { return g / (1.0f + expf(-g)); }

// CUDA-core kernel: one warp per weight row (SwiGLU: per up/gate pair of rows) and MB rows of a.
template <typename T, int EPI>
__global__ void __launch_bounds__(kThreads) gemm_q4_kernel(const Args p) {
  pdl_wait();
  pdl_trigger();
  constexpr int R = EPI == HX_EPI_SWIGLU ? 2 : 1;
  const int lane = threadIdx.x & 31;
  const int64_t col = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
  const int64_t cols = EPI == HX_EPI_SWIGLU ? p.N / 2 : p.N;
  if (col >= cols) return;
  const int64_t row = EPI == HX_EPI_SWIGLU ? (col / 16) * 32 + col % 16 : col;  // + 16: gate
  const int m0 = blockIdx.y * MB, nm = min(MB, p.M - m0);
  float acc[R][MB];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int m = 0; m < MB; ++m) acc[r][m] = 0.f;
  const int groups = p.K / p.group;
  for (int k = lane * 8; k < p.K; k += 256) {
    float w[R][8];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t n = row + 16 * r;
      const uint32_t bits = *reinterpret_cast<const uint32_t*>(p.w + n * (p.K / 2) + k / 2);
      const float s = DT<T>::to_f(((const T*)p.scales)[n * groups + k / p.group]);
#pragma unroll
      for (int i = 0; i < 8; ++i) w[r][i] = s * (float)((int)((bits >> (4 * i)) & 15u) - 8);
    }
#pragma unroll
    for (int m = 0; m < MB; ++m) {
      if (m >= nm) break;
      const T* a = (const T*)p.a + (int64_t)(m0 + m) * p.lda + k;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float x = DT<T>::to_f(a[i]);
#pragma unroll
        for (int r = 0; r < R; ++r) acc[r][m] = fmaf(x, w[r][i], acc[r][m]);
      }
    }
  }
#pragma unroll
  for (int m = 0; m < MB; ++m) {
    float v = warp_sum(acc[0][m]);
    if constexpr (EPI == HX_EPI_SWIGLU) v *= silu_f(warp_sum(acc[R - 1][m]));
    if (m < nm && lane == 0) {
      if (EPI == HX_EPI_RESIDUAL)
        v += DT<T>::to_f(((const T*)p.residual)[(int64_t)(m0 + m) * p.ldr + col]);
      ((T*)p.out)[(int64_t)(m0 + m) * p.ldo + col] = DT<T>::from_f(v);
    }
  }
}

template <typename T>
int launch(const Args& p, int epilogue, cudaStream_t stream) {
  const int64_t cols = epilogue == HX_EPI_SWIGLU ? p.N / 2 : p.N;
  const dim3 grid((unsigned)ceil_div(cols, kThreads / 32), (unsigned)ceil_div(p.M, MB));
  auto kern = epilogue == HX_EPI_SWIGLU     ? gemm_q4_kernel<T, HX_EPI_SWIGLU>
              : epilogue == HX_EPI_RESIDUAL ? gemm_q4_kernel<T, HX_EPI_RESIDUAL>
                                            : gemm_q4_kernel<T, HX_EPI_NONE>;
  return hx::cuda_status(launch_ex(kern, grid, dim3(kThreads), 0, stream, 1, p),
                         "gemm_q4_kernel launch");
}

}  // namespace

extern "C" int hx_gemm_q4(const void* a, const void* w, const void* scales, void* c, int64_t m,
                          int64_t n, int64_t k, int64_t group, int64_t lda, int64_t ldc,
                          int epilogue, const void* residual, int64_t ld_residual, int dtype,
                          void* stream) {
  HX_REQUIRE(a && w && scales && c, "hx_gemm_q4: null pointer");
  HX_REQUIRE(group == 32 || group == 64 || group == 128,
             "hx_gemm_q4: group %lld unsupported (32, 64 or 128)", (long long)group);
  HX_REQUIRE(m >= 0 && m <= 64 && n > 0 && n < (int64_t(1) << 30) && k > 0 && k % group == 0 &&
                 k < (int64_t(1) << 30),
             "hx_gemm_q4: bad sizes (at most 64 rows, k a multiple of the group)");
  HX_REQUIRE(epilogue >= HX_EPI_NONE && epilogue <= HX_EPI_SWIGLU, "hx_gemm_q4: bad epilogue");
  HX_REQUIRE(epilogue != HX_EPI_SWIGLU || n % 32 == 0,
             "hx_gemm_q4: SwiGLU needs n (interleaved up/gate rows) to be a multiple of 32");
  HX_REQUIRE(epilogue != HX_EPI_RESIDUAL || residual, "hx_gemm_q4: residual is null");
  const int64_t cols = epilogue == HX_EPI_SWIGLU ? n / 2 : n;
  const int esz = dtype == HX_F32 ? 4 : 2;
  HX_REQUIRE(lda >= k && (lda * esz) % 16 == 0 && (uintptr_t)a % 16 == 0 && (uintptr_t)w % 16 == 0,
             "hx_gemm_q4: a and w must be 16-byte aligned, rows of a too");
  HX_REQUIRE(ldc >= cols && (epilogue != HX_EPI_RESIDUAL || ld_residual >= cols),
             "hx_gemm_q4: bad output or residual stride");
  if (m == 0) return HX_OK;
  const Args p{a, (const uint8_t*)w, scales, residual, c, lda, ld_residual, ldc,
               (int)m, (int)n, (int)k, (int)group};
  HX_DISPATCH_DTYPE(dtype, T, return launch<T>(p, epilogue, (cudaStream_t)stream));
  return HX_OK;
}
