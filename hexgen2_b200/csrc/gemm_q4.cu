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
// Tensor-core kernel (f16/bf16) on mma.m16n8k16 with f16 operands and f32 sums: the 16 rows of A are
// weight rows, its 8 columns rows of a.
//   - The bits of a code are an f16 as they stand: below 2^11 an f16's value is its bits times 2^-24
//     (subnormals and the first binade). A masked word is an operand register: w & 0x000f000f
//     holds codes * 2^-24, w & 0x00f000f0 codes * 2^-20; nothing is converted or rounded, and the
//     8 that codes are offset by comes off with the group's sum of a, in f32.
//   - a goes in as f16 times a power of two of its own per (row, 128 k): max |a| in [2^9, 2^10), times 16
//     where the codes are not, so bf16 and f16 values down to 2^-24 of the unit's largest are exact
//     (smaller ones to 2^-35 of it). The factor comes off with the group's scale.
//   - A unit is 16 weight rows x 128 k. Nibbles 16 bits apart make one operand register, and the order of
//     k inside a group is free, so a lane reads whole words of its two rows straight from global
//   - a is staged in the order of the B operands (one 16-byte load feeds two mma) with its group
//     sums and factors: by every CTA for its own slice up to eight rows; above, once by
//     stage_kernel, and warp 0 keeps a ring of its blocks filled.
//   - A CTA has `warps` warps of 16 weight rows. K is split over the S CTAs of a cluster; each leaves
//     f32 partials in its shared memory and CTA s adds up rows s, s + S, ... of the batch in rank
//     order, applies the epilogue and stores neighbouring outputs together.
// ------------------------------------------------------------------------------------------
constexpr int kMaxWarps = 8;
constexpr int kUnitK = 128;
constexpr int kPair = 2;     // units per stage of a warp's ring of weights
constexpr int kStageBytes = 16 * 128;
constexpr int kChunk = 16;   // units of a staged at a time up to eight rows

// One unit of a: operands [NT][4 words][8 rows][4 lanes] x 16 bytes, then [groups][NT * 8] (offset, factor).
template <int G, int NT>
struct Block {
  static constexpr int kGroups = kUnitK / G;
  static constexpr int kOperands = NT * 2048;
  static constexpr int kBytes = kOperands + kGroups * NT * 8 * 8;
  static constexpr int kPerStage = NT == 2 ? 2 : 1;  // units per stage of the ring of a
  static constexpr int kStages = NT == 8 ? 3 : 4;
  static constexpr int kWeightStages = NT == 8 ? 3 : 4;
  static constexpr int kWarpBytes = kWeightStages * kStageBytes;
};

HX_DEVICE void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
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
HX_DEVICE void bulk_load(void* smem_dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
          smem_u32(smem_dst)),
      "l"(src), "r"(bytes), "r"(smem_u32(bar))
      : "memory");
}

// Elements [8 c, 8 c + 8) of a unit of batch row m (`raw`, zeros where a has none) into its block.
// Called by whole warps, the 16 lanes of a unit side by side; `live` lanes store.
template <typename T, int G, int NT>
HX_DEVICE void stage(uint8_t* block, int m, int c, uint4 raw, bool live) {
  const T* e = reinterpret_cast<const T*>(&raw);
  float x[8], sum = 0.f, big = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    x[i] = DT<T>::to_f(e[i]);
    sum += x[i];
    big = fmaxf(big, fabsf(x[i]));
  }
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) {
    if (o < G / 8) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, o));
  }
  if (!live) return;
  const int ex = max((int)((__float_as_uint(big) >> 23) & 0xff) - 127, -100);
  const float f = __uint_as_float((uint32_t)(127 + 9 - ex) << 23);
  const int at = 8 * c, j = at / G, rest = at % G, t = rest / (G / 4), w = j * (G / 32) + rest % (G / 4) / 8;
  *reinterpret_cast<uint4*>(block + (((m >> 3) * 4 + w) * 32 + (m & 7) * 4 + t) * 16) =
      make_uint4(pack2<__half>(x[0] * f * 16.f, x[4] * f * 16.f), pack2<__half>(x[1] * f, x[5] * f),
                 pack2<__half>(x[2] * f * 16.f, x[6] * f * 16.f), pack2<__half>(x[3] * f, x[7] * f));
  if (rest == 0)  // (offset, factor) of acc * factor + offset, both times 2^-20
    *reinterpret_cast<float2*>(block + Block<G, NT>::kOperands + (j * NT * 8 + m) * 8) =
        make_float2(sum * (-8.f / 1048576.f), __uint_as_float((uint32_t)(127 - 9 + ex) << 23));
}

template <typename T, int G, int NT>
__global__ void __launch_bounds__(256) stage_kernel(const Args p, uint8_t* __restrict__ blocks) {
  pdl_wait();
  pdl_trigger();
  const int u = blockIdx.x, c = threadIdx.x & 15;
  const int64_t k = (int64_t)u * kUnitK + c * 8;
#pragma unroll
  for (int m0 = 0; m0 < NT * 8; m0 += 16) {
    const int m = m0 + (threadIdx.x >> 4);
    uint4 raw = make_uint4(0, 0, 0, 0);
    if (m < p.M && k < p.K) raw = *reinterpret_cast<const uint4*>((const T*)p.a + (int64_t)m * p.lda + k);
    stage<T, G, NT>(blocks + (int64_t)u * Block<G, NT>::kBytes, m, c, raw, true);
  }
}

// Adds one unit of a pair to the totals: w the warp's stage of weights (16 rows of 128 bytes, the 16-byte
// chunks of row r permuted by r % 8), scales in the lane's s (groups 4 q + t of the pair in s[row][q],
// handed round by shuffles).
template <typename T, int G, int NT>
HX_DEVICE void multiply(const uint8_t* w, int unit, const float (&s)[2][kPair * (kUnitK / G) > 4 ? 2 : 1],
                        const uint8_t* block, float (&tot)[NT][4]) {
  constexpr int GU = kUnitK / G;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  uint32_t x[2][4];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const uint8_t* row = w + (g + 8 * r) * 128;
    auto chunk = [&](int c) { return row + ((4 * unit + c) ^ g) * 16; };
    if constexpr (G == 128) {
      const uint4 v = *reinterpret_cast<const uint4*>(chunk(t));
      x[r][0] = v.x, x[r][1] = v.y, x[r][2] = v.z, x[r][3] = v.w;
    } else if constexpr (G == 64) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const uint2 v = *reinterpret_cast<const uint2*>(chunk(2 * j + (t >> 1)) + (t & 1) * 8);
        x[r][2 * j] = v.x, x[r][2 * j + 1] = v.y;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) x[r][j] = *reinterpret_cast<const uint32_t*>(chunk(j) + 4 * t);
    }
  }
#pragma unroll
  for (int j = 0; j < GU; ++j) {
    float acc[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int y = 0; y < 4; ++y) acc[nt][y] = 0.f;
#pragma unroll
    for (int i = j * (G / 32); i < (j + 1) * (G / 32); ++i) {
      const uint32_t x0 = x[0][i], y0 = x[1][i], x1 = x0 >> 8, y1 = y0 >> 8;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const uint4 v = *reinterpret_cast<const uint4*>(block + (nt * 4 + i) * 512 + lane * 16);
        mma_f16(acc[nt], x0 & 0x000f000fu, y0 & 0x000f000fu, x0 & 0x00f000f0u, y0 & 0x00f000f0u, v.x, v.y);
        mma_f16(acc[nt], x1 & 0x000f000fu, y1 & 0x000f000fu, x1 & 0x00f000f0u, y1 & 0x00f000f0u, v.z, v.w);
      }
    }
    const int grp = unit * GU + j, from = (lane & ~3) | (grp & 3);
    const float s0 = __shfl_sync(0xffffffffu, s[0][grp >> 2], from), s1 = __shfl_sync(0xffffffffu, s[1][grp >> 2], from);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const float4 f = *reinterpret_cast<const float4*>(block + Block<G, NT>::kOperands +
                                                        (j * NT * 8 + nt * 8 + 2 * t) * 8);
      tot[nt][0] = fmaf(s0, fmaf(acc[nt][0], f.y, f.x), tot[nt][0]);
      tot[nt][1] = fmaf(s0, fmaf(acc[nt][1], f.w, f.z), tot[nt][1]);
      tot[nt][2] = fmaf(s1, fmaf(acc[nt][2], f.y, f.x), tot[nt][2]);
      tot[nt][3] = fmaf(s1, fmaf(acc[nt][3], f.w, f.z), tot[nt][3]);
    }
  }
}

template <typename T, int G, int NT, int EPI>
__global__ void __launch_bounds__(kMaxWarps * 32, 2) gemm_q4_mma_kernel(
    const Args p, const __grid_constant__ CUtensorMap w_map, const uint8_t* __restrict__ blocks, int S,
    int warps) {
  using B = Block<G, NT>;
  constexpr bool kRing = NT > 1;
  constexpr int kPerStage = B::kPerStage, kStages = B::kStages, kW = B::kWeightStages;
  constexpr int kPairGroups = kPair * B::kGroups, kScales = kPairGroups > 4 ? 2 : 1;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  __shared__ uint64_t full[kStages], empty[kStages], w_full[kMaxWarps][kW];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  uint8_t* ring = smem + warp * B::kWarpBytes;
  uint8_t* sm_a = smem + warps * B::kWarpBytes;
  if (lane == 0) {
    for (int i = 0; i < kW; ++i) mbar_init(&w_full[warp][i], 1);
    if (kRing && warp == 0)
      for (int i = 0; i < kStages; ++i) mbar_init(&full[i], 1), mbar_init(&empty[i], warps);
    fence_mbar_init();
  }
  __syncthreads();
  pdl_wait();
  pdl_trigger();
  const int rank = S > 1 ? (int)cluster_rank() : 0;
  const int rows = warps * 16, n0 = (int)(blockIdx.x / S) * rows;
  const int units = (p.K + kUnitK - 1) / kUnitK, groups = p.K / G;
  const int begin = (int)((int64_t)units * rank / S), end = (int)((int64_t)units * (rank + 1) / S);
  const int pairs = (end - begin + kPair - 1) / kPair;
  bool ok = true;

  // Weights, 16 rows of two units: TMA fills rows past N and bytes past K with zeros.
  const int w_at = begin * (kUnitK / 4), w_rows = n0 + warp * 16;  // in 16-bit elements
  auto ask_weights = [&](int pair, int st) {
    if (lane == 0) {
      mbar_arrive_expect_tx(&w_full[warp][st], kStageBytes);
      tma_load_2d(ring + st * kStageBytes, &w_map, &w_full[warp][st], w_at + pair * (kPair * kUnitK / 4), w_rows);
    }
  };
  for (int i = 0; i < min(pairs, kW); ++i) ask_weights(i, i);

  // Scales of rows g and g + 8: lane t holds groups t and t + 4 of a pair, times 2^20.
  const T* s_row[2] = {(const T*)p.scales + (int64_t)min(n0 + warp * 16 + g, p.N - 1) * groups,
                       (const T*)p.scales + (int64_t)min(n0 + warp * 16 + g + 8, p.N - 1) * groups};
  T next[2][kScales];
  auto ask_scales = [&](int pair) {
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int q = 0; q < kScales; ++q)
        next[r][q] = __ldg(s_row[r] + min((begin + pair * kPair) * B::kGroups + 4 * q + (t & (kPairGroups - 1)), groups - 1));
  };
  ask_scales(0);

  // Warp 0's lane 0: the next stage of a's blocks, once every warp has left the stage it replaces.
  int asked = 0;
  auto ask = [&]() {
    const int u = begin + asked * kPerStage, st = asked % kStages;
    if (u >= end || !ok) return;
    if (asked >= kStages && !(ok = mbar_wait(&empty[st], (asked / kStages - 1) & 1))) return;
    const uint32_t bytes = (uint32_t)min(kPerStage, end - u) * B::kBytes;
    mbar_arrive_expect_tx(&full[st], bytes);
    bulk_load(sm_a + st * (kPerStage * B::kBytes), blocks + (int64_t)u * B::kBytes, bytes, &full[st]);
    ++asked;
  };
  if (kRing && tid == 0)
    for (int i = 0; i < kStages - 1; ++i) ask();

  float tot[NT][4];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int j = 0; j < 4; ++j) tot[nt][j] = 0.f;
  int st = 0, phase = 0, w_st = 0, w_phase = 0, done = 0;
  for (; done < pairs; ++done) {
    const int u0 = begin + done * kPair;
    if (!kRing && done % (kChunk / kPair) == 0) {  // stage a's slice: 16 bytes a thread, neighbours along k
      __syncthreads();
      const int per_row = min(kChunk, end - u0) * 16, items = p.M * per_row;
      for (int i0 = 0; i0 < items; i0 += warps * 32) {
        const int i = i0 + tid, m = min(i / per_row, p.M - 1), c = i - i / per_row * per_row;
        const int64_t k = (int64_t)u0 * kUnitK + c * 8;
        uint4 raw = make_uint4(0, 0, 0, 0);
        if (i < items && k < p.K) raw = *reinterpret_cast<const uint4*>((const T*)p.a + (int64_t)m * p.lda + k);
        stage<T, G, NT>(sm_a + (c >> 4) * B::kBytes, m, c & 15, raw, i < items);
      }
      __syncthreads();
    }
    float s[2][kScales];
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int q = 0; q < kScales; ++q) s[r][q] = DT<T>::to_f(next[r][q]) * 1048576.f;
    if (done + 1 < pairs) ask_scales(done + 1);
    if (ok) ok = mbar_wait_warp(&w_full[warp][w_st], w_phase);
#pragma unroll
    for (int i = 0; i < kPair; ++i) {
      if (u0 + i >= end || !ok) break;
      if (kRing && i % kPerStage == 0) {
        if (tid == 0) ask();
        ok = mbar_wait_warp(&full[st], phase) && __all_sync(0xffffffffu, ok);
        if (!ok) break;
      }
      const uint8_t* block = kRing ? sm_a + (st * kPerStage + i % kPerStage) * B::kBytes
                                   : sm_a + ((done % (kChunk / kPair)) * kPair + i) * B::kBytes;
      multiply<T, G, NT>(ring + w_st * kStageBytes, i, s, block, tot);
      if (kRing && (i % kPerStage == kPerStage - 1 || u0 + i + 1 == end)) {
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[st]);
        if (++st == kStages) st = 0, phase ^= 1;
      }
    }
    if (!ok && kRing) break;  // up to eight rows the block's barriers go on
    __syncwarp();
    if (ok && done + kW < pairs) ask_weights(done + kW, w_st);
    if (ok && ++w_st == kW) w_st = 0, w_phase ^= 1;
  }
  if (!ok) {  // a wait gave up: let the copies in flight land
    for (int i = 0; i < kW; ++i) mbar_wait_drain(&w_full[warp][i], i < w_st ? w_phase ^ 1 : w_phase);
    if (kRing && tid == 0)
      for (int i = max(0, asked - kStages); i < asked; ++i) mbar_wait_drain(&full[i % kStages], (i / kStages) & 1);
  }

  // Partials [batch row][weight row] in shared memory, added up over the cluster.
  __syncthreads();
  float* part = reinterpret_cast<float*>(smem);
  const int pitch = rows + 4;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      part[(nt * 8 + 2 * t + (j & 1)) * pitch + warp * 16 + g + 8 * (j >> 1)] = tot[nt][j];
  if (S > 1) cluster_sync(); else __syncthreads();
  const int width = EPI == HX_EPI_SWIGLU ? rows / 2 : rows;  // outputs of one batch row in this CTA
  const int cols = EPI == HX_EPI_SWIGLU ? p.N / 2 : p.N, col0 = EPI == HX_EPI_SWIGLU ? n0 / 2 : n0;
  auto total = [&](int m, int r) {
    const float* at = part + m * pitch + r;
    if (S == 1) return *at;
    float v = 0.f;
    for (int s = 0; s < S; ++s) v += ld_cluster_f32(smem_u32(at), s);
    return v;
  };
  const int mine = (p.M - rank + S - 1) / S * width;  // rows rank, rank + S, ...
  for (int i = tid; i < mine; i += blockDim.x) {
    const int m = rank + S * (i / width), c = i % width;
    if (col0 + c >= cols) continue;
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

int tiles_of(int64_t m) { return m <= 8 ? 1 : m <= 16 ? 2 : m <= 32 ? 4 : 8; }

// Warps per CTA and CTAs per cluster: the pair whose fullest SM has the least to do, a CTA counting
// its 16-row tiles times its units of K plus what it takes to start and to store (about 16 of those).
struct Plan {
  int warps, S;
};
Plan plan(int64_t n, int64_t k, bool pairs) {
  const int tiles = ceil_div(n, 16), units = ceil_div(k, kUnitK);
  Plan best{kMaxWarps, 1};
  int64_t least = INT64_MAX;
  for (int warps = kMaxWarps; warps >= 4; warps -= pairs ? 2 : 1)
    for (int S = 1; S <= 8 && (S == 1 || 2 * S <= units); ++S) {
      const int64_t ctas = (int64_t)ceil_div(tiles, warps) * S;
      const int64_t cost = ceil_div(ctas, 148) * ((int64_t)warps * ceil_div(units, S) + 16);
      if (cost < least) least = cost, best = {warps, S};
    }
  return best;
}

template <typename T, int G, int NT, int EPI>
int launch_mma(const Args& p, uint8_t* blocks, cudaStream_t stream) {
  using B = Block<G, NT>;
  const Plan pl = plan(p.N, p.K, EPI == HX_EPI_SWIGLU);
  const int units = ceil_div(p.K, kUnitK);
  if (NT > 1) {
    const int s = hx::cuda_status(launch_ex(stage_kernel<T, G, NT>, dim3((unsigned)units), dim3(256), 0, stream, 1, p, blocks),
                                  "gemm_q4 stage_kernel launch");
    if (s) return s;
  }
  const size_t staged = (size_t)pl.warps * B::kWarpBytes +
                        (size_t)(NT > 1 ? B::kStages * B::kPerStage : std::min(kChunk, ceil_div(units, pl.S))) * B::kBytes;
  const size_t smem = std::max(staged, (size_t)NT * 8 * (pl.warps * 16 + 4) * sizeof(float)) + 1024;  // + alignment
  CUtensorMap w_map;  // [N, K / 2] bytes as 16-bit elements
  const uint64_t dims[2] = {(uint64_t)p.K / 4, (uint64_t)p.N}, strides[1] = {(uint64_t)p.K / 2};
  const uint32_t box[2] = {kPair * kUnitK / 4, 16};
  if (const int s = make_tensor_map(&w_map, p.w, 2, dims, strides, box, HX_BF16)) return s;
  auto kern = gemm_q4_mma_kernel<T, G, NT, EPI>;
  if (smem > 48 * 1024) cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 114 * 1024);
  return hx::cuda_status(
      launch_ex(kern, dim3((unsigned)(ceil_div(p.N, pl.warps * 16) * pl.S)),
                dim3((unsigned)(pl.warps * 32)), smem, stream, pl.S, p, w_map,
                (const uint8_t*)blocks, pl.S, pl.warps),
      "gemm_q4_mma_kernel launch");
}

template <typename T, int G, int NT>
int launch_epilogue(const Args& p, int epilogue, uint8_t* blocks, cudaStream_t stream) {
  return epilogue == HX_EPI_SWIGLU     ? launch_mma<T, G, NT, HX_EPI_SWIGLU>(p, blocks, stream)
         : epilogue == HX_EPI_RESIDUAL ? launch_mma<T, G, NT, HX_EPI_RESIDUAL>(p, blocks, stream)
                                       : launch_mma<T, G, NT, HX_EPI_NONE>(p, blocks, stream);
}

template <typename T, int G>
int launch_rows(const Args& p, int epilogue, uint8_t* blocks, cudaStream_t stream) {
  switch (tiles_of(p.M)) {
    case 1: return launch_epilogue<T, G, 1>(p, epilogue, blocks, stream);
    case 2: return launch_epilogue<T, G, 2>(p, epilogue, blocks, stream);
    case 4: return launch_epilogue<T, G, 4>(p, epilogue, blocks, stream);
    default: return launch_epilogue<T, G, 8>(p, epilogue, blocks, stream);
  }
}

template <typename T>
int launch(const Args& p, int epilogue, uint8_t* blocks, cudaStream_t stream) {
  if constexpr (sizeof(T) == 2) {
    return p.group == 128  ? launch_rows<T, 128>(p, epilogue, blocks, stream)
           : p.group == 64 ? launch_rows<T, 64>(p, epilogue, blocks, stream)
                           : launch_rows<T, 32>(p, epilogue, blocks, stream);
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

extern "C" size_t hx_gemm_q4_workspace(int64_t m, int64_t k, int64_t group, int dtype) {
  if (m <= 8 || m > 64 || k <= 0 || group < 32 || group > kUnitK || dtype == HX_F32) return 0;
  const size_t nt = (size_t)tiles_of(m);
  return (size_t)ceil_div(k, kUnitK) * nt * (2048 + (size_t)(kUnitK / group) * 64);
}

extern "C" int hx_gemm_q4(const void* a, const void* w, const void* scales, void* c, int64_t m,
                          int64_t n, int64_t k, int64_t group, int64_t lda, int64_t ldc,
                          int epilogue, const void* residual, int64_t ld_residual, void* workspace,
                          size_t workspace_bytes, int dtype, void* stream) {
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
  const size_t need = hx_gemm_q4_workspace(m, k, group, dtype);
  HX_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && (uintptr_t)workspace % 16 == 0),
             "hx_gemm_q4: workspace too small (%zu < %zu) or misaligned", workspace_bytes, need);
  const Args p{a, (const uint8_t*)w, scales, residual, c, lda, ld_residual, ldc,
               (int)m, (int)n, (int)k, (int)group};
  HX_DISPATCH_DTYPE(dtype, T, return launch<T>(p, epilogue, (uint8_t*)workspace, (cudaStream_t)stream));
  return HX_OK;
}
