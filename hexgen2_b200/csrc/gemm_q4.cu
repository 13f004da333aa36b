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

// ------------------------------------------------------------------------------------------
// Tensor-core kernel (f16/bf16) on mma.m16n8k16 with f32 sums: the 16 rows of A are weight rows, its 8
// columns rows of a. A code goes in as an exact 16-bit float: bf16 128 + code (OR into the mantissa),
// f16 code * 2^-24 (its bits are the subnormal); the constant's share, and that of the 8 that codes
// are offset by, is kOffset * sum of a's group, subtracted with the group's scale in f32.
//   - A unit is 16 weight rows x 128 k. Nibbles 16 bits apart make one operand register, and the
//     order of k inside a group is free, so a lane reads whole words of its two rows straight from
//     global memory (16 bytes at groups of 128), four units ahead.
//   - a is staged in shared memory in the order of the B operands (one 16-byte load per two
//     mma), with its group sums.
//   - A CTA holds 128 weight rows, eight warps of 16. K is split over the S CTAs of a cluster; each
//     leaves f32 partials in its shared memory and CTA s adds up rows s, s + S, ... of the batch in rank
//     order, applies the epilogue and stores 128 neighbouring outputs at a time.
// ------------------------------------------------------------------------------------------
constexpr int kMmaThreads = 256;
constexpr int kRows = 128;   // weight rows per CTA
constexpr int kUnitK = 128;
constexpr int kPitch = kRows + 4;

template <typename T> struct Codes;
template <> struct Codes<__nv_bfloat16> {
  static constexpr float kOffset = 136.f, kScale = 1.f;
  static HX_DEVICE uint32_t pair(uint32_t w, int e) { return ((w >> (4 * e)) & 0x000f000fu) | 0x43004300u; }
  static HX_DEVICE void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};
template <> struct Codes<__half> {
  static constexpr float kOffset = 8.f / 16777216.f, kScale = 16777216.f;
  static HX_DEVICE uint32_t pair(uint32_t w, int e) { return (w >> (4 * e)) & 0x000f000fu; }
  static HX_DEVICE void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};

HX_DEVICE uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
HX_DEVICE void cluster_sync() {
  asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}
HX_DEVICE float ld_cluster_f32(uint32_t addr, uint32_t rank) {
  uint32_t remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(addr), "r"(rank));
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(remote) : "memory");
  return v;
}
HX_DEVICE uint4 ld_stream(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

// One unit of a lane: the words of rows g and g + 8 and their groups' scales.
template <typename T, int G>
struct Unit {
  uint32_t w[2][4];
  T s[2][kUnitK / G];
};

// Byte offset, in a's staged chunk of NT tiles of 8 rows, of elements [8 c, 8 c + 8) of batch row m.
template <int G, int NT>
HX_DEVICE int staged(int m, int c) {
  const int u = c >> 4, in = (c & 15) * 8;
  const int j = in / G, rest = in % G, t = rest / (G / 4), w = j * (G / 32) + rest % (G / 4) / 8;
  return (((u * NT + (m >> 3)) * 4 + w) * 32 + (m & 7) * 4 + t) * 16;
}

template <typename T, int G, int NT, int EPI>
__global__ void __launch_bounds__(kMmaThreads, NT == 8 ? 1 : 2) gemm_q4_mma_kernel(const Args p, int S, int chunk_units) {
  constexpr int kAhead = 4;       // units in flight per warp
  constexpr int GU = kUnitK / G;  // groups per unit
  extern __shared__ __align__(128) uint8_t smem[];
  uint8_t* sm_a = smem;                                                     // chunk_units * NT * 2 KB
  float* sm_sum = reinterpret_cast<float*>(smem + chunk_units * NT * 2048);  // [groups][NT * 8]
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  pdl_wait();
  pdl_trigger();
  const int rank = S > 1 ? (int)cluster_rank() : 0;
  const int n0 = (blockIdx.x / S) * kRows;
  const int units = (p.K + kUnitK - 1) / kUnitK;
  const int begin = (int)((int64_t)units * rank / S), end = (int)((int64_t)units * (rank + 1) / S);
  const int groups = p.K / G;
  const int row = n0 + warp * 16 + g;
  const bool in[2] = {row < p.N, row + 8 < p.N};
  const uint8_t* wp = p.w + (int64_t)row * (p.K / 2);
  const T* sp = (const T*)p.scales + (int64_t)row * groups;
  using U = Unit<T, G>;
  auto fetch = [&](U& x, int u) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const uint8_t* base = wp + (int64_t)r * 8 * (p.K / 2) + (int64_t)u * (kUnitK / 2);
#pragma unroll
      for (int j = 0; j < GU; ++j) {
        const int grp = u * GU + j;
        const bool some = in[r] && u < end && grp < groups;
        if constexpr (G == 128) {
          const uint4 v = some ? ld_stream(base + 16 * t) : make_uint4(0, 0, 0, 0);
          x.w[r][0] = v.x, x.w[r][1] = v.y, x.w[r][2] = v.z, x.w[r][3] = v.w;
        } else if constexpr (G == 64) {
          const uint2 v = some ? __ldg(reinterpret_cast<const uint2*>(base + 32 * j + 8 * t)) : make_uint2(0, 0);
          x.w[r][2 * j] = v.x, x.w[r][2 * j + 1] = v.y;
        } else {
          x.w[r][j] = some ? __ldg(reinterpret_cast<const uint32_t*>(base + 16 * j + 4 * t)) : 0u;
        }
        x.s[r][j] = some ? __ldg(sp + (int64_t)r * 8 * groups + grp) : DT<T>::from_f(0.f);
      }
    }
  };
  U buf[kAhead];
#pragma unroll
  for (int i = 0; i < kAhead; ++i) fetch(buf[i], begin + i);

  float tot[NT][4];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int j = 0; j < 4; ++j) tot[nt][j] = 0.f;

  for (int c0 = begin; c0 < end; c0 += chunk_units) {
    const int nu = min(chunk_units, end - c0);
    // Stage a's chunk: 16 bytes a thread, neighbouring threads along k, group sums over G / 8 lanes.
    if (c0 != begin) __syncthreads();
    const int per_row = nu * 16, items = p.M * per_row;
    for (int i0 = 0; i0 < items; i0 += kMmaThreads) {
      const int i = i0 + tid;
      const int m = min(i / per_row, p.M - 1), c = i - i / per_row * per_row;
      const int64_t k = (int64_t)c0 * kUnitK + c * 8;
      uint4 raw = make_uint4(0, 0, 0, 0);
      if (i < items && k < p.K) raw = *reinterpret_cast<const uint4*>((const T*)p.a + (int64_t)m * p.lda + k);
      const T* e = reinterpret_cast<const T*>(&raw);
      float sum = 0.f;
#pragma unroll
      for (int x = 0; x < 8; ++x) sum += DT<T>::to_f(e[x]);
#pragma unroll
      for (int o = 1; o < G / 8; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (i < items) {
        *reinterpret_cast<uint4*>(sm_a + staged<G, NT>(m, c)) =
            make_uint4(__byte_perm(raw.x, raw.z, 0x5410), __byte_perm(raw.x, raw.z, 0x7632),
                       __byte_perm(raw.y, raw.w, 0x5410), __byte_perm(raw.y, raw.w, 0x7632));
        if (c % (G / 8) == 0) sm_sum[(c / (G / 8)) * (NT * 8) + m] = sum;
      }
    }
    __syncthreads();
    for (int u = 0; u < nu; u += kAhead) {
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        if (u + i >= nu) break;
        const U x = buf[i];
        const uint8_t* b = sm_a + (u + i) * (NT * 2048) + lane * 16;
#pragma unroll
        for (int j = 0; j < GU; ++j) {
          float acc[NT][4];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int y = 0; y < 4; ++y) acc[nt][y] = 0.f;
#pragma unroll
          for (int w = j * (G / 32); w < (j + 1) * (G / 32); ++w) {
            const uint32_t lo[4] = {Codes<T>::pair(x.w[0][w], 0), Codes<T>::pair(x.w[1][w], 0),
                                    Codes<T>::pair(x.w[0][w], 1), Codes<T>::pair(x.w[1][w], 1)};
            const uint32_t hi[4] = {Codes<T>::pair(x.w[0][w], 2), Codes<T>::pair(x.w[1][w], 2),
                                    Codes<T>::pair(x.w[0][w], 3), Codes<T>::pair(x.w[1][w], 3)};
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              const uint4 v = *reinterpret_cast<const uint4*>(b + (nt * 4 + w) * 512);
              Codes<T>::mma(acc[nt], lo, v.x, v.y);
              Codes<T>::mma(acc[nt], hi, v.z, v.w);
            }
          }
          const float s0 = DT<T>::to_f(x.s[0][j]) * Codes<T>::kScale, s1 = DT<T>::to_f(x.s[1][j]) * Codes<T>::kScale;
          const float* sums = sm_sum + ((u + i) * GU + j) * (NT * 8) + 2 * t;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const float2 sum = *reinterpret_cast<const float2*>(sums + nt * 8);
            tot[nt][0] = fmaf(s0, fmaf(-Codes<T>::kOffset, sum.x, acc[nt][0]), tot[nt][0]);
            tot[nt][1] = fmaf(s0, fmaf(-Codes<T>::kOffset, sum.y, acc[nt][1]), tot[nt][1]);
            tot[nt][2] = fmaf(s1, fmaf(-Codes<T>::kOffset, sum.x, acc[nt][2]), tot[nt][2]);
            tot[nt][3] = fmaf(s1, fmaf(-Codes<T>::kOffset, sum.y, acc[nt][3]), tot[nt][3]);
          }
        }
        fetch(buf[i], c0 + u + i + kAhead);
      }
    }
  }

  // Partials [batch row][weight row] in shared memory, added up over the cluster.
  __syncthreads();
  float* part = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      part[(nt * 8 + 2 * t + (j & 1)) * kPitch + warp * 16 + g + 8 * (j >> 1)] = tot[nt][j];
  if (S > 1) cluster_sync(); else __syncthreads();
  constexpr int kCols = EPI == HX_EPI_SWIGLU ? kRows / 2 : kRows;
  const int cols = EPI == HX_EPI_SWIGLU ? p.N / 2 : p.N, col0 = EPI == HX_EPI_SWIGLU ? n0 / 2 : n0;
  auto total = [&](int m, int r) {
    const float* at = part + m * kPitch + r;
    if (S == 1) return *at;
    float v = 0.f;
    for (int s = 0; s < S; ++s) v += ld_cluster_f32(smem_u32(at), s);
    return v;
  };
  const int c = tid % kCols;
  for (int m = rank + S * (tid / kCols); m < p.M; m += S * (kMmaThreads / kCols)) {
    if (col0 + c >= cols) break;
    float v;
    if constexpr (EPI == HX_EPI_SWIGLU) {
      const int r = (c / 16) * 32 + c % 16;
      v = total(m, r) * silu_f(total(m, r + 16));
    } else {
      v = total(m, c);
      if (EPI == HX_EPI_RESIDUAL) v += DT<T>::to_f(((const T*)p.residual)[(int64_t)m * p.ldr + col0 + c]);
    }
    ((T*)p.out)[(int64_t)m * p.ldo + col0 + c] = DT<T>::from_f(v);
  }
  if (S > 1) cluster_sync();  // no CTA leaves while others read its partials
}

template <typename T, int G, int NT, int EPI>
int launch_mma(const Args& p, cudaStream_t stream) {
  const int blocks = ceil_div(p.N, kRows), units = ceil_div(p.K, kUnitK);
  const int S = std::max(1, std::min({8, 2 * 148 / blocks, units / 2}));
  const int chunk = std::min(32 / NT, ceil_div(units, S));
  const size_t stage = (size_t)chunk * NT * 2048 + (size_t)chunk * (kUnitK / G) * NT * 8 * sizeof(float);
  const size_t smem = std::max(stage, (size_t)NT * 8 * kPitch * sizeof(float));
  auto kern = gemm_q4_mma_kernel<T, G, NT, EPI>;
  if (smem > 48 * 1024) cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 72 * 1024);
  return hx::cuda_status(launch_ex(kern, dim3((unsigned)(blocks * S)), dim3(kMmaThreads), smem, stream, S, p, S, chunk),
                         "gemm_q4_mma_kernel launch");
}

template <typename T, int G, int NT>
int launch_epilogue(const Args& p, int epilogue, cudaStream_t stream) {
  return epilogue == HX_EPI_SWIGLU     ? launch_mma<T, G, NT, HX_EPI_SWIGLU>(p, stream)
         : epilogue == HX_EPI_RESIDUAL ? launch_mma<T, G, NT, HX_EPI_RESIDUAL>(p, stream)
                                       : launch_mma<T, G, NT, HX_EPI_NONE>(p, stream);
}

template <typename T, int G>
int launch_rows(const Args& p, int epilogue, cudaStream_t stream) {
  return p.M <= 8    ? launch_epilogue<T, G, 1>(p, epilogue, stream)
         : p.M <= 16 ? launch_epilogue<T, G, 2>(p, epilogue, stream)
         : p.M <= 32 ? launch_epilogue<T, G, 4>(p, epilogue, stream)
                     : launch_epilogue<T, G, 8>(p, epilogue, stream);
}

template <typename T>
int launch(const Args& p, int epilogue, cudaStream_t stream) {
  if constexpr (sizeof(T) == 2) {
    return p.group == 128  ? launch_rows<T, 128>(p, epilogue, stream)
           : p.group == 64 ? launch_rows<T, 64>(p, epilogue, stream)
                           : launch_rows<T, 32>(p, epilogue, stream);
  } else {
    const int64_t cols = epilogue == HX_EPI_SWIGLU ? p.N / 2 : p.N;
    const dim3 grid((unsigned)ceil_div(cols, kThreads / 32), (unsigned)ceil_div(p.M, MB));
    auto kern = epilogue == HX_EPI_SWIGLU     ? gemm_q4_kernel<T, HX_EPI_SWIGLU>
                : epilogue == HX_EPI_RESIDUAL ? gemm_q4_kernel<T, HX_EPI_RESIDUAL>
                                              : gemm_q4_kernel<T, HX_EPI_NONE>;
    return hx::cuda_status(launch_ex(kern, grid, dim3(kThreads), 0, stream, 1, p),
                           "gemm_q4_kernel launch");
  }
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
