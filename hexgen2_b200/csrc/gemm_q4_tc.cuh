// gemm_q4 on tcgen05: large weights times 17 to 64 rows of a. A part of gemm_q4.cu, which has the operator, its
// other kernels and the arguments and conversions that both use, and includes this once.
//
// D[128 weight rows, NT rows of a] = A B^T by tcgen05.mma kind::f16, M = 128. A, the codes, is made in tensor
// memory: the bits of a code are an f16 as they stand (codes * 2^-24, or 2^-20 one nibble up), so a
// lane, which is a weight row, masks its words and stores them with tcgen05.st, 64 columns for 128 k. B, the
// rows of a in the matching order of k, is staged once by stage_kernel (f16 times a power of two per row
// and 128 k, as in gemm_q4.cu) as the swizzled image the MMA reads. Every group of k has an accumulator
// of its own; its scale, its offset (8 codes' worth of a's sum) and a's factor come in when it is read.
//
// A CTA per SM takes an equal range of the list of (128-row block, 256 k) items, block by block. Warps:
//   0      producer: 16 KB of weights by TMA and the block of a by a bulk copy per item
//   1      issues the MMAs
//   2-9    unpack: four warps for either unit (128 k) of an item, shared memory -> registers -> tensor memory
//   10-17  accumulate: tensor memory -> registers, four warps (a lane per weight row) for either half of
//          a's rows; at the end of a block's part they write it to the workspace
// join_kernel adds the parts of a block up in CTA order and applies the epilogue.
//
// What bounds it: the issue of the MMAs. 32 x 22016 x 4096 (SwiGLU, groups of 128) takes 32 us for 7.3 us of
// bytes: 8 us for the three launches, then 18.6 items of 2300 cycles per SM, of which the one thread
// that issues spends 1000 on its 16 MMAs (62 cycles each at 32 rows, the tensor pipe needs 16), 250 on
// commits and the rest waiting.
#pragma once

namespace tc {

constexpr int kThreads = 18 * 32;
constexpr int kRows = 128;
constexpr int kWeightBytes = kRows * 128;  // of an item: 256 k
constexpr int kAccs = 2;                   // pairs of accumulators in flight

// An item of a: two units of swizzled operands ([2 halves of 64 k][NT rows][128 bytes]), then (offset, factor)
// [2 units][groups][NT].
template <int G, int NT>
struct Item {
  static constexpr int kGroups = 128 / G;  // per unit
  static constexpr int kUnit = NT * 256;
  static constexpr int kStats = 2 * kGroups * NT * 8;
  static constexpr int kBytes = 2 * kUnit + kStats;
  static constexpr int kPitch = (kWeightBytes + kBytes + 1023) / 1024 * 1024;  // of the ring
  static constexpr int kStages = NT == 64 ? 4 : 6;
  // Items whose operands (2 x 64 columns) are in tensor memory at a time; the accumulators behind them. (With
  // one its way round, unpack - MMA - free, took 3000 cycles.)
  static constexpr int kPer = NT == 64 ? 2 : 3;
  static constexpr uint32_t kAccColumn = kPer * 2 * 64;
  static constexpr int kShared = kStages * kPitch + 1024;
};

// Equal ranges of the list of items: the first `extra` CTAs take one more than the others.
struct Ranges {
  unsigned each, extra;
  __host__ HX_DEVICE Ranges(int total, int grid) : each((unsigned)total / grid), extra((unsigned)total % grid) {}
  HX_DEVICE int begin(int c) const { return (int)(c * each + min((unsigned)c, extra)); }
  HX_DEVICE int holder(int x) const {
    const unsigned wide = extra * (each + 1);
    return (int)((unsigned)x < wide ? x / (each + 1) : extra + (x - wide) / each);
  }
};

template <typename T, int G, int NT>
__global__ void __launch_bounds__(256) stage_kernel(const Args p, uint8_t* __restrict__ blocks) {
  using I = Item<G, NT>;
  pdl_wait();
  pdl_trigger();
  const int u = blockIdx.x, c = threadIdx.x & 15;
  uint8_t* item = blocks + (int64_t)(u >> 1) * I::kBytes;
  const int64_t k = (int64_t)u * 128 + c * 8;
#pragma unroll
  for (int m0 = 0; m0 < NT; m0 += 16) {
    const int m = m0 + (threadIdx.x >> 4);
    uint4 raw = make_uint4(0, 0, 0, 0);
    if (m < p.M && k < p.K) raw = *reinterpret_cast<const uint4*>((const T*)p.a + (int64_t)m * p.lda + k);
    float sum, factor;
    const uint4 op = operands<T, G>(raw, sum, factor);
    *reinterpret_cast<uint4*>(item + (u & 1) * I::kUnit + (c >> 3) * (NT * 128) + m * 128 + (((c & 7) ^ (m & 7)) * 16)) = op;
    if (c * 8 % G == 0)
      *reinterpret_cast<float2*>(item + 2 * I::kUnit + (((u & 1) * I::kGroups + c * 8 / G) * NT + m) * 8) =
          make_float2(sum * (-8.f / 1048576.f), factor);
  }
}

HX_DEVICE bool wait(uint64_t* bar, uint32_t parity) { return mbar_wait_warp_timed(bar, parity); }

// D(tmem) (+)= A(tmem) * B(smem desc)^T, f16 operands, f32 sums.
HX_DEVICE void mma_tmem(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
HX_DEVICE void tmem_ld(uint32_t addr, uint32_t (&r)[32]) { tmem_ld_32x32b_x32(addr, r); }
HX_DEVICE void tmem_ld(uint32_t addr, uint32_t (&r)[16]) { tmem_ld_32x32b_x16(addr, r); }

template <typename T, int G, int NT>
__global__ void __launch_bounds__(kThreads, 1) gemm_q4_tc_kernel(
    const Args p, const __grid_constant__ CUtensorMap w_map, const uint8_t* __restrict__ blocks,
    float* __restrict__ parts, int items_per_block, int total) {
  using I = Item<G, NT>;
  constexpr int kStages = I::kStages, kHalf = NT / 2, kPer = I::kPer;
  constexpr uint32_t kAccColumn = I::kAccColumn;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  __shared__ uint64_t full[kStages], empty[kStages], a_full[kPer], a_empty[kPer], d_full[kAccs], d_empty[kAccs];
  __shared__ uint32_t tmem_at;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int i = 0; i < kStages; ++i) mbar_init(&full[i], 1), mbar_init(&empty[i], 17);
    for (int i = 0; i < kPer; ++i) mbar_init(&a_full[i], 8), mbar_init(&a_empty[i], 1);
    for (int i = 0; i < kAccs; ++i) mbar_init(&d_full[i], 1), mbar_init(&d_empty[i], 8);
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(&tmem_at, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // All 512 columns begin at address 0. Known at compile time, the addresses of the MMAs stay in uniform
  // registers; read back from shared memory they cost 80 cycles of moves per MMA.
  constexpr uint32_t tmem = 0;
  pdl_wait();
  pdl_trigger();
  const Ranges ranges(total, gridDim.x);
  const int begin = ranges.begin(blockIdx.x), end = ranges.begin(blockIdx.x + 1);
  bool ok = tmem_at == tmem;
  if (!ok) record_device_error(HX_DEVERR_BAD_ARGUMENT);

  if (warp == 0) {
    int n = 0;
    for (int x = begin; x < end && ok; ++x, ++n) {
      const int st = n % kStages;
      if (n >= kStages && !(ok = wait(&empty[st], (n / kStages - 1) & 1))) break;
      if (lane == 0) {
        const int block = x / items_per_block, item = x - block * items_per_block;
        uint8_t* at = smem + st * I::kPitch;
        mbar_arrive_expect_tx(&full[st], kWeightBytes + I::kBytes);
        tma_load_2d(at, &w_map, &full[st], item * 64, block * kRows);  // 16-bit elements; zeros past N and K
        bulk_load(at + kWeightBytes, blocks + (int64_t)item * I::kBytes, I::kBytes, &full[st]);
      }
      __syncwarp();
    }
    if (!ok)  // let the copies in flight land
      for (int i = max(0, n - kStages); i < n; ++i) mbar_wait_drain(&full[i % kStages], (i / kStages) & 1);
  } else if (warp == 1) {
    constexpr uint32_t idesc = make_idesc_f16<__half>(128, NT);
    const uint64_t desc = sw128_kmajor_desc(smem_u32(smem + kWeightBytes));
    int acc = 0, acc_phase = 0, st = 0, st_phase = 0, per = 0, per_phase = 0;
    for (int n = 0; n < end - begin && ok; ++n) {
      if (!(ok = wait(&full[st], st_phase) && wait(&a_full[per], per_phase))) break;
#pragma unroll
      for (int j = 0; j < I::kGroups; ++j) {
        if (!(ok = wait(&d_empty[acc], acc_phase ^ 1))) break;
        tc_fence_after();
        if (lane == 0) {
          const uint64_t b = desc + ((st * I::kPitch) >> 4);
          const uint32_t d = tmem + kAccColumn + acc * 2 * NT, from = tmem + per * 128;
#pragma unroll
          for (int i = 0; i < G / 16; ++i)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              const int k = j * (G / 16) + i;  // 16 k at a time: 8 columns of A, 32 bytes of a row of B
              mma_tmem(d + u * NT, from + u * 64 + k * 8,
                       b + ((u * I::kUnit + (k >> 2) * (NT * 128) + (k & 3) * 32) >> 4), idesc, i > 0);
            }
          tc_commit(&d_full[acc]);
          if (j == I::kGroups - 1) {
            tc_commit(&a_empty[per]);
            tc_commit(&empty[st]);
          }
        }
        __syncwarp();
        if (++acc == kAccs) acc = 0, acc_phase ^= 1;
      }
      if (++st == kStages) st = 0, st_phase ^= 1;
      if (++per == kPer) per = 0, per_phase ^= 1;
    }
  } else if (warp < 10) {
    const int u = (warp - 2) >> 2, quadrant = warp & 3, row = quadrant * 32 + lane;
    const uint32_t lanes = tmem + ((uint32_t)(quadrant * 32) << 16);
    int per = 0, per_phase = 1;
    for (int n = 0; n < end - begin && ok; ++n) {
      const int st = n % kStages;
      if (!(ok = wait(&full[st], (n / kStages) & 1))) break;
      const uint8_t* w = smem + st * I::kPitch + row * 128;
      uint4 v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = *reinterpret_cast<const uint4*>(w + ((4 * u + i) ^ (row & 7)) * 16);
      if (!(ok = wait(&a_empty[per], per_phase))) break;  // at once on its first round
      tc_fence_after();
      const uint32_t to = lanes + per * 128 + u * 64;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t r[32];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint4 q = v[2 * h + i / 4];
          const uint32_t x = i % 4 == 0 ? q.x : i % 4 == 1 ? q.y : i % 4 == 2 ? q.z : q.w, y = x >> 8;
          r[4 * i] = x & 0x000f000fu;
          r[4 * i + 1] = x & 0x00f000f0u;
          r[4 * i + 2] = y & 0x000f000fu;
          r[4 * i + 3] = y & 0x00f000f0u;
        }
        tmem_st_32x32b_x32(to + h * 32, r);
      }
      tc_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&a_full[per]);
        mbar_arrive(&empty[st]);
      }
      if (++per == kPer) per = 0, per_phase ^= 1;
    }
  } else {
    const int half = (warp - 10) >> 2, quadrant = warp & 3, row = quadrant * 32 + lane;
    const uint32_t from = tmem + ((uint32_t)(quadrant * 32) << 16) + kAccColumn + half * kHalf;
    const int groups = p.K / G;
    float tot[kHalf];
#pragma unroll
    for (int i = 0; i < kHalf; ++i) tot[i] = 0.f;
    int acc = 0, acc_phase = 0, block = begin / items_per_block, item = begin - block * items_per_block;
    // Scales times 2^20; rows past N and groups past K read the last ones and meet zeros.
    T next[2 * I::kGroups];
    auto ask_scales = [&](int block, int item) {
      const T* s = (const T*)p.scales + (int64_t)min(block * kRows + row, p.N - 1) * groups;
#pragma unroll
      for (int i = 0; i < 2 * I::kGroups; ++i) next[i] = __ldg(s + min(item * 2 * I::kGroups + i, groups - 1));
    };
    if (begin < end) ask_scales(block, item);
    for (int n = 0; n < end - begin && ok; ++n) {
      const int st = n % kStages;
      float s[2 * I::kGroups];
#pragma unroll
      for (int i = 0; i < 2 * I::kGroups; ++i) s[i] = DT<T>::to_f(next[i]) * 1048576.f;
      const bool last = item + 1 == items_per_block;
      if (n + 1 < end - begin) ask_scales(last ? block + 1 : block, last ? 0 : item + 1);
      if (!(ok = wait(&full[st], (n / kStages) & 1))) break;
      const uint8_t* stats = smem + st * I::kPitch + kWeightBytes + 2 * I::kUnit + half * kHalf * 8;
#pragma unroll
      for (int j = 0; j < I::kGroups; ++j) {
        if (!(ok = wait(&d_full[acc], acc_phase))) break;
        tc_fence_after();
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int i = u * I::kGroups + j;
          uint32_t d[kHalf];
          tmem_ld(from + (acc * 2 + u) * NT, d);
          tc_wait_ld();
          if (u == 1) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&d_empty[acc]);
          }
#pragma unroll
          for (int m = 0; m < kHalf; m += 2) {
            const float4 f = *reinterpret_cast<const float4*>(stats + (i * NT + m) * 8);
            tot[m] = fmaf(s[i], fmaf(__uint_as_float(d[m]), f.y, f.x), tot[m]);
            tot[m + 1] = fmaf(s[i], fmaf(__uint_as_float(d[m + 1]), f.w, f.z), tot[m + 1]);
          }
        }
        if (++acc == kAccs) acc = 0, acc_phase ^= 1;
      }
      if (!ok) break;
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[st]);
      if (last || n + 1 == end - begin) {  // this CTA's part of the block: part blockIdx.x + block of the list
        float* out = parts + ((int64_t)(blockIdx.x + block) * p.M + half * kHalf) * kRows + row;
#pragma unroll
        for (int m = 0; m < kHalf; ++m) {
          if (half * kHalf + m < p.M) out[m * kRows] = tot[m];
          tot[m] = 0.f;
        }
      }
      if (last) item = 0, ++block;
      else ++item;
    }
  }
  if (!ok && warp == 1) {  // whatever was issued ends before tensor memory goes: a commit behind it, waited for
    __shared__ uint64_t drained;
    if (lane == 0) {
      mbar_init(&drained, 1);
      fence_mbar_init();
      tc_commit(&drained);
      mbar_wait_drain(&drained, 0);
    }
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_at, 512);
  }
}

// The parts of a block, added up in CTA order, and the epilogue: a CTA per (block, kJoin rows of a).
constexpr int kJoin = 4;
template <typename T, int EPI>
__global__ void __launch_bounds__(128) join_kernel(const Args p, const float* __restrict__ parts, int items_per_block,
                                                  int total, int grid) {
  pdl_wait();
  pdl_trigger();
  const int block = blockIdx.x, t = threadIdx.x;
  const Ranges ranges(total, grid);
  const int c0 = ranges.holder(block * items_per_block), c1 = ranges.holder((block + 1) * items_per_block - 1);
  constexpr bool kGated = EPI == HX_EPI_SWIGLU;
  constexpr int kCols = kGated ? 64 : 128;  // outputs of a block per row of a
  const int cols = kGated ? p.N / 2 : p.N, col = block * kCols + t % kCols;
  const int row = kGated ? (t % 64 / 16) * 32 + t % 16 : t;
  if (col >= cols) return;
  for (int m = blockIdx.y * kJoin + t / kCols; m < min(p.M, (int)(blockIdx.y + 1) * kJoin); m += 128 / kCols) {
    const float* from = parts + ((int64_t)(c0 + block) * p.M + m) * kRows + row;
    float v = 0.f, gate = 0.f, add = 0.f;
    if (EPI == HX_EPI_RESIDUAL) add = DT<T>::to_f(((const T*)p.residual)[(int64_t)m * p.ldr + col]);
#pragma unroll 4
    for (int c = c0; c <= c1; ++c, from += (int64_t)p.M * kRows) {
      v += from[0];
      if (kGated) gate += from[16];
    }
    if (kGated) v *= silu_f(gate);
    ((T*)p.out)[(int64_t)m * p.ldo + col] = DT<T>::from_f(v + add);
  }
}

inline int items(int64_t k) { return ceil_div(k, 256); }
inline int rows_of_a(int64_t m) { return m <= 32 ? 32 : 64; }

// Workspace: the staged rows of a, then the parts.
inline size_t staged_bytes(int64_t m, int64_t k, int64_t group) {
  const size_t nt = rows_of_a(m);
  return (size_t)items(k) * (nt * 512 + 2 * (128 / group) * nt * 8);
}
inline size_t workspace(int64_t m, int64_t n, int64_t k, int64_t group) {
  return staged_bytes(m, k, group) + (size_t)(148 + ceil_div(n, kRows)) * m * kRows * sizeof(float);
}

template <typename T, int G, int NT>
int launch(const Args& p, int epilogue, void* ws, cudaStream_t stream) {
  using I = Item<G, NT>;
  uint8_t* blocks = (uint8_t*)ws;
  float* parts = reinterpret_cast<float*>(blocks + staged_bytes(p.M, p.K, G));
  const int per_block = items(p.K), n_blocks = ceil_div(p.N, kRows), total = per_block * n_blocks;
  const int grid = std::min(148, total);
  CUtensorMap w_map;  // [N, K / 2] bytes as 16-bit elements
  const uint64_t dims[2] = {(uint64_t)p.K / 4, (uint64_t)p.N}, strides[1] = {(uint64_t)p.K / 2};
  const uint32_t box[2] = {64, kRows};
  if (const int s = make_tensor_map(&w_map, p.w, 2, dims, strides, box, HX_BF16)) return s;
  auto kern = gemm_q4_tc_kernel<T, G, NT>;
  static std::atomic<uint64_t> allowed{0};
  if (const int s = allow_shared(reinterpret_cast<const void*>(kern), I::kShared, allowed)) return s;
  int s = hx::cuda_status(launch_ex(stage_kernel<T, G, NT>, dim3((unsigned)(2 * per_block)), dim3(256), 0, stream, 1, p, blocks),
                          "gemm_q4 stage_kernel launch");
  if (s) return s;
  s = hx::cuda_status(launch_ex(kern, dim3((unsigned)grid), dim3(kThreads), I::kShared, stream, 1, p, w_map,
                                (const uint8_t*)blocks, parts, per_block, total),
                      "gemm_q4_tc_kernel launch");
  if (s) return s;
  auto join = epilogue == HX_EPI_SWIGLU     ? join_kernel<T, HX_EPI_SWIGLU>
              : epilogue == HX_EPI_RESIDUAL ? join_kernel<T, HX_EPI_RESIDUAL>
                                            : join_kernel<T, HX_EPI_NONE>;
  return hx::cuda_status(launch_ex(join, dim3((unsigned)n_blocks, (unsigned)ceil_div(p.M, kJoin)), dim3(128), 0, stream, 1,
                                   p, (const float*)parts, per_block, total, grid),
                         "gemm_q4 join_kernel launch");
}

template <typename T, int G>
int launch_rows(const Args& p, int epilogue, void* ws, cudaStream_t stream) {
  return p.M <= 32 ? launch<T, G, 32>(p, epilogue, ws, stream) : launch<T, G, 64>(p, epilogue, ws, stream);
}

}  // namespace tc
