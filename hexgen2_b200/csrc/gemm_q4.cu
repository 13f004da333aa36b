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
//     (smaller ones to 2^-35 of it). The factor comes off with the group's scale. Products are cut, towards zero,
//     at about 2^-14 of the largest times 1 (codes in the lowest bits): beside the rounding of an f16 output nothing,
//     but for rows of one sign with outliers, 1.19 times its error at 300 times the rest and 16384 k.
//   - A unit is 16 weight rows x 128 k. Nibbles 16 bits apart make one operand register, and the order of
//     k inside a group is free, so a lane takes whole words of its two rows (16 bytes at groups of 128).
//   - The weights are what has to move, so a stays: a CTA keeps up to 16 rows of a over up to 4096 k (8
//     rows: 8192 k) in shared memory in operand order, and the weight rows stream past it. Its 16 warps
//     are R row tiles x KW slices of k; each streams its slice of one tile after another, two units at
//     a time, through a ring of its own by TMA, and the KW partials of a tile are added up in slice order
//     through shared memory. More rows of a are more CTAs on the same weights (passes side by side,
//     so that a tile comes from HBM once and from L2 for the others), more k further rounds, whose
//     running sums wait in an f32 workspace.
//   Against this, with a streamed through shared memory and K split over clusters: clusters of 2 and 3
//   left SMs idle (the fullest had 1.6 times the average), and staging a in every CTA of 128 rows cost a
//   third of the instructions. Weights by plain loads, eight rows to an instruction, kept L1's tags 75 %
//   busy at a quarter of the memory's bandwidth; bulk copies of 128 bytes took about 20 cycles each.
//   Measured (device time): 1x4096x4096 6 us, 1x12288x4096 12.3 us (2.1 TB/s), 5x32000x4096 (f16, groups of 64)
//   25.5 us (2.7 TB/s, 0.42 of the measured copy rate); without the products the same loads take 4.4, 7.5
//   and 16 us. Instructions bound it: 325 per pair of units and warp in all, 130 to 160 of them unpacking,
//   loading and multiplying, at 45 % of the issue slots.
// ------------------------------------------------------------------------------------------
constexpr int kWarps = 16;
constexpr int kMmaThreads = kWarps * 32;
constexpr int kUnitK = 128;
constexpr int kPair = 2;                     // units per stage of a warp's ring: 16 rows of 128 bytes
constexpr int kStageBytes = 16 * 128;
constexpr int kSmem = 226 * 1024;  // dynamic; the barriers are static

// One unit of a: operands [NT][4 words][8 rows][4 lanes] x 16 bytes, then [groups][NT * 8] (offset, factor).
template <int G, int NT>
struct Block {
  static constexpr int kGroups = kUnitK / G;
  static constexpr int kOperands = NT * 2048;
  static constexpr int kBytes = kOperands + kGroups * NT * 8 * 8;
  static constexpr int kMaxUnits = 64 / NT;             // of a in shared memory at a time
  static constexpr int kPartial = kWarps * NT * 8 * 16;  // floats
};

// Largest |x| of eight 16-bit floats, as its bits (NaN above infinity above the rest).
HX_DEVICE uint32_t largest_bits(uint4 v) {
  const uint32_t m = 0x7fff7fffu;
  const uint32_t a = __vmaxu2(__vmaxu2(v.x & m, v.y & m), __vmaxu2(v.z & m, v.w & m));
  return max(a & 0xffffu, a >> 16);
}

// Eight elements of a row of a (`raw`; the 16 lanes of a unit of 128 k side by side, whole warps) as operands:
// times the unit's power of two, in the order of the codes' pairs (0,4), (1,5), (2,6), (3,7), the even pairs
// times 16. sum: of the group's elements (f32); factor: what brings a sum of products back, times 2^-20.
template <typename T, int G>
HX_DEVICE uint4 operands(uint4 raw, float& sum, float& factor) {
  const T* e = reinterpret_cast<const T*>(&raw);
  float x[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = DT<T>::to_f(e[i]);
  sum = ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
  uint32_t bits = largest_bits(raw);
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) {
    if (o < G / 8) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, o));
  }
  const float big = DT<T>::to_f(__builtin_bit_cast(T, (unsigned short)bits));
  const int ex = max((int)(__float_as_uint(big) >> 23), 27);  // biased; at least 2^-100
  const float f = __uint_as_float((uint32_t)(263 - ex) << 23), f16 = f * 16.f;
  factor = __uint_as_float((uint32_t)(ex - 9) << 23);
  return make_uint4(pack2<__half>(x[0] * f16, x[4] * f16), pack2<__half>(x[1] * f, x[5] * f),
                    pack2<__half>(x[2] * f16, x[6] * f16), pack2<__half>(x[3] * f, x[7] * f));
}

// Elements [8 c, 8 c + 8) of a unit of row m of a (zeros where a has none) into its block; `live` lanes store.
template <typename T, int G, int NT>
HX_DEVICE void stage(uint8_t* block, int m, int c, uint4 raw, bool live) {
  float sum, factor;
  const uint4 op = operands<T, G>(raw, sum, factor);
  const int at = 8 * c, j = at / G, rest = at % G, t = rest / (G / 4), w = j * (G / 32) + rest % (G / 4) / 8;
  if (!live) return;
  *reinterpret_cast<uint4*>(block + (((m >> 3) * 4 + w) * 32 + (m & 7) * 4 + t) * 16) = op;
  if (rest == 0)  // (offset, factor) of acc * factor + offset, both times 2^-20
    *reinterpret_cast<float2*>(block + Block<G, NT>::kOperands + (j * NT * 8 + m) * 8) =
        make_float2(sum * (-8.f / 1048576.f), factor);
}

// Adds a pair of units to the totals: w the warp's stage of weights (16 rows of 128 bytes, the 16-byte
// chunks of row r permuted by r % 8), scales in the lane's s (groups 4 q + t of the pair in s[row][q],
// handed round by shuffles), block the two units of a. The units' sums run side by side: one chain of mma
// would wait for itself.
template <typename T, int G, int NT>
HX_DEVICE void multiply(const uint8_t* w, const float (&s)[2][kPair * (kUnitK / G) > 4 ? 2 : 1],
                        const uint8_t* block, float (&tot)[NT][4]) {
  using B = Block<G, NT>;
  constexpr int GU = kUnitK / G;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  uint32_t x[kPair][2][4];
#pragma unroll
  for (int u = 0; u < kPair; ++u)
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const uint8_t* row = w + (g + 8 * r) * 128;
      auto chunk = [&](int c) { return row + ((4 * u + c) ^ g) * 16; };
      if constexpr (G == 128) {
        const uint4 v = *reinterpret_cast<const uint4*>(chunk(t));
        x[u][r][0] = v.x, x[u][r][1] = v.y, x[u][r][2] = v.z, x[u][r][3] = v.w;
      } else if constexpr (G == 64) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const uint2 v = *reinterpret_cast<const uint2*>(chunk(2 * j + (t >> 1)) + (t & 1) * 8);
          x[u][r][2 * j] = v.x, x[u][r][2 * j + 1] = v.y;
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) x[u][r][j] = *reinterpret_cast<const uint32_t*>(chunk(j) + 4 * t);
      }
    }
#pragma unroll
  for (int j = 0; j < GU; ++j) {
    float acc[kPair][NT][4];
#pragma unroll
    for (int u = 0; u < kPair; ++u)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int y = 0; y < 4; ++y) acc[u][nt][y] = 0.f;
#pragma unroll
    for (int i = j * (G / 32); i < (j + 1) * (G / 32); ++i)
#pragma unroll
      for (int u = 0; u < kPair; ++u) {
        const uint32_t x0 = x[u][0][i], y0 = x[u][1][i], x1 = x0 >> 8, y1 = y0 >> 8;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const uint4 v = *reinterpret_cast<const uint4*>(block + u * B::kBytes + (nt * 4 + i) * 512 + lane * 16);
          mma_f16(acc[u][nt], x0 & 0x000f000fu, y0 & 0x000f000fu, x0 & 0x00f000f0u, y0 & 0x00f000f0u, v.x, v.y);
          mma_f16(acc[u][nt], x1 & 0x000f000fu, y1 & 0x000f000fu, x1 & 0x00f000f0u, y1 & 0x00f000f0u, v.z, v.w);
        }
      }
#pragma unroll
    for (int u = 0; u < kPair; ++u) {
      const int grp = u * GU + j, from = (lane & ~3) | (grp & 3);
      const float s0 = __shfl_sync(0xffffffffu, s[0][grp >> 2], from), s1 = __shfl_sync(0xffffffffu, s[1][grp >> 2], from);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float4 f = *reinterpret_cast<const float4*>(block + u * B::kBytes + B::kOperands +
                                                          (j * NT * 8 + nt * 8 + 2 * t) * 8);
        tot[nt][0] = fmaf(s0, fmaf(acc[u][nt][0], f.y, f.x), tot[nt][0]);
        tot[nt][1] = fmaf(s0, fmaf(acc[u][nt][1], f.w, f.z), tot[nt][1]);
        tot[nt][2] = fmaf(s1, fmaf(acc[u][nt][2], f.y, f.x), tot[nt][2]);
        tot[nt][3] = fmaf(s1, fmaf(acc[u][nt][3], f.w, f.z), tot[nt][3]);
      }
    }
  }
}

#include "gemm_q4_tc.cuh"

struct Plan {
  int log_kw;  // of the slices of k
  int passes;  // CTAs that share a tile, each with NT * 8 rows of a
  int ctas;    // per pass
  int rounds;  // over k, of `units` units each (the last may have fewer)
  int units;
  int stages;  // of a warp's ring
  int buffers;  // of partials, one or two
};

template <typename T, int G, int NT, int EPI>
__global__ void __launch_bounds__(kMmaThreads, 1) gemm_q4_mma_kernel(
    const Args p, const __grid_constant__ CUtensorMap w_map, const Plan pl, float* __restrict__ running) {
  using B = Block<G, NT>;
  constexpr int kPairGroups = kPair * B::kGroups, kScales = kPairGroups > 4 ? 2 : 1, kMaxStages = 4;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  __shared__ uint64_t full[kWarps][kMaxStages];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  uint8_t* ring = smem + warp * pl.stages * kStageBytes;
  float* part = reinterpret_cast<float*>(smem + kWarps * pl.stages * kStageBytes);  // [kWarps][NT * 8][16]
  uint8_t* sm_a = reinterpret_cast<uint8_t*>(part + pl.buffers * B::kPartial);
  if (lane == 0) {
    for (int i = 0; i < pl.stages; ++i) mbar_init(&full[warp][i], 1);
    fence_mbar_init();
  }
  __syncwarp();
  pdl_wait();
  pdl_trigger();
  const int log_r = 4 - pl.log_kw, R = 1 << log_r, r = warp >> pl.log_kw, kw = warp & ((1 << pl.log_kw) - 1);
  const int pass = blockIdx.x % pl.passes, first = blockIdx.x / pl.passes;
  const int m0 = pass * NT * 8, M = min(NT * 8, p.M - m0);
  const int tiles = (p.N + 15) / 16, steps_all = (tiles + R - 1) >> log_r;  // of R tiles
  const int steps = first < steps_all ? (steps_all - first + pl.ctas - 1) / pl.ctas : 0;
  const int all_units = (p.K + kUnitK - 1) / kUnitK, groups = p.K / G;
  bool ok = true;
  int st = 0, phase = 0;

  for (int round = 0; round < pl.rounds; ++round) {
    const int u0 = round * pl.units, pairs = (min(pl.units, all_units - u0) + 1) / 2;
    // This warp's pairs: kw, kw + KW, ...: the KW warps of a tile read neighbouring bytes of its rows at a time.
    const int mine = (pairs - kw + (1 << pl.log_kw) - 1) >> pl.log_kw;
    // The warp's stages in order: pair after pair of its slice, tile after tile; the next one goes where the
    // last was read. TMA fills rows past N and bytes past K with zeros; a tile past the last is all zeros.
    const int x_step = (kPair * kUnitK / 4) << pl.log_kw;
    const int x_first = (u0 / kPair + kw) * (kPair * kUnitK / 4), x_last = x_first + (mine - 1) * x_step;
    int left = ok ? steps * mine : 0, x = x_first, y = (first * R + r) * 16;
    auto ask = [&](int slot) {
      if (left <= 0) return;
      --left;
      if (lane == 0) {
        mbar_arrive_expect_tx(&full[warp][slot], kStageBytes);
        tma_load_2d(ring + slot * kStageBytes, &w_map, &full[warp][slot], x, y);
      }
      const bool wrap = x == x_last;
      x = wrap ? x_first : x + x_step;
      y += wrap ? pl.ctas * R * 16 : 0;
    };
    for (int i = 0, slot = st; i < pl.stages; ++i, slot = slot + 1 == pl.stages ? 0 : slot + 1) ask(slot);

    // This round's a, whole pairs: a half warp per unit and row, 16 bytes a lane.
    const int units = pairs * kPair, log_units = 32 - __clz(units - 1), c = lane & 15;
    for (int i0 = warp * 2 + (lane >> 4); i0 < M << log_units; i0 += kWarps * 2 * 4) {
      uint4 raw[4];  // four loads in flight
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i = i0 + j * kWarps * 2, u = i & ((1 << log_units) - 1), m = i >> log_units;
        const int64_t k = (int64_t)(u0 + u) * kUnitK + c * 8;
        raw[j] = make_uint4(0, 0, 0, 0);
        if (m < M && u < units && k < p.K)
          raw[j] = *reinterpret_cast<const uint4*>((const T*)p.a + (int64_t)(m0 + m) * p.lda + k);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i = i0 + j * kWarps * 2, u = i & ((1 << log_units) - 1), m = i >> log_units;
        stage<T, G, NT>(sm_a + u * B::kBytes, m, c, raw[j], m < M && u < units);
      }
    }
    __syncthreads();

    // Scales of rows g and g + 8 of a tile: lane t holds groups t and t + 4 of a pair, times 2^20. Rows past
    // N and groups past K read the last ones and meet zeros.
    const T* s_row[2];
    T next[2][kScales];
    const int grp0 = (u0 + kw * kPair) * B::kGroups + (t & (kPairGroups - 1));
    auto ask_scales = [&](int step, int pair) {
      if (pair == 0) {
        const int row = ((first + step * pl.ctas) * R + r) * 16 + g;
        s_row[0] = (const T*)p.scales + (int64_t)min(row, p.N - 1) * groups;
        s_row[1] = (const T*)p.scales + (int64_t)min(row + 8, p.N - 1) * groups;
      }
#pragma unroll
      for (int q = 0; q < kScales; ++q) {
        const int grp = min(grp0 + ((pair * kPairGroups) << pl.log_kw) + 4 * q, groups - 1);
        next[0][q] = __ldg(s_row[0] + grp);
        next[1][q] = __ldg(s_row[1] + grp);
      }
    };
    if (mine > 0) ask_scales(0, 0);

    for (int step = 0; step < steps; ++step) {
      float tot[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < 4; ++j) tot[nt][j] = 0.f;
#pragma unroll 1
      for (int pair = 0; pair < mine; ++pair) {
        float s[2][kScales];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int q = 0; q < kScales; ++q) s[h][q] = DT<T>::to_f(next[h][q]) * 1048576.f;
        if (pair + 1 < mine) ask_scales(step, pair + 1);
        else if (step + 1 < steps) ask_scales(step + 1, 0);
        if (ok) ok = mbar_wait_warp_timed(&full[warp][st], phase);
        if (!ok) break;
        multiply<T, G, NT>(ring + st * kStageBytes, s, sm_a + (kw + (pair << pl.log_kw)) * (kPair * B::kBytes), tot);
        __syncwarp();
        ask(st);
        if (++st == pl.stages) st = 0, phase ^= 1;
      }
      // Partials [slice][row of a][weight row], added up in slice order. With two buffers the threads that
      // add up (others at every step) do so while the rest go on.
      float* buffer = part + (step & (pl.buffers - 1)) * B::kPartial;
      float* mine_at = buffer + warp * (NT * 8 * 16);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < 4; ++j) mine_at[(nt * 8 + 2 * t + (j & 1)) * 16 + g + 8 * (j >> 1)] = tot[nt][j];
      __syncthreads();
      const int n0 = (first + step * pl.ctas) * R * 16;
      auto total_of = [&](int m, int row) {
        const float* at = buffer + ((row >> 4) << pl.log_kw) * (NT * 8 * 16) + m * 16 + (row & 15);
        float v = 0.f;
#pragma unroll 4
        for (int i = 0; i < 1 << pl.log_kw; ++i) v += at[i * (NT * 8 * 16)];
        if (pl.rounds > 1) {
          float* keep = running + (int64_t)(m0 + m) * p.N + n0 + row;
          if (round > 0) v += *keep;
          if (round + 1 < pl.rounds) *keep = v;
        }
        return v;
      };
      const bool last = round + 1 == pl.rounds;
      constexpr bool kGated = EPI == HX_EPI_SWIGLU;
      const int log_width = log_r + (kGated ? 3 : 4), col0 = kGated ? n0 / 2 : n0, cols = kGated ? p.N / 2 : p.N;
      const int turn = pl.buffers == 2 ? step * (kMmaThreads / 4) : 0;
      for (int i = (tid + turn) & (kMmaThreads - 1); i < M << log_width; i += kMmaThreads) {
        const int m = i >> log_width, c = i & ((1 << log_width) - 1);
        if (col0 + c >= cols) continue;
        float v, add = 0.f;
        if (EPI == HX_EPI_RESIDUAL && last) add = DT<T>::to_f(((const T*)p.residual)[(int64_t)(m0 + m) * p.ldr + col0 + c]);
        if constexpr (kGated) {
          const int row = (c / 16) * 32 + c % 16;
          const float up = total_of(m, row), gate = total_of(m, row + 16);
          v = up * silu_f(gate);
        } else {
          v = total_of(m, c) + add;
        }
        if (last) ((T*)p.out)[(int64_t)(m0 + m) * p.ldo + col0 + c] = DT<T>::from_f(v);
      }
      if (pl.buffers == 1) __syncthreads();
    }
    __syncthreads();  // every sum is read before the next round
    if (!ok)  // a wait gave up: let the copies in flight land
      for (int i = 0; i < pl.stages; ++i) mbar_wait_drain(&full[warp][i], i < st ? phase ^ 1 : phase);
  }
}

// The slices of k that leave the fullest CTA the least to do: a step costs its pairs per warp, and about
// 0.6 of a pair for adding up and storing.
template <int G, int NT>
Plan plan(int64_t m, int64_t n, int64_t k, bool gated) {
  using B = Block<G, NT>;
  Plan pl;
  const int units = ceil_div(k, kUnitK), tiles = ceil_div(n, 16);
  pl.rounds = ceil_div(units, B::kMaxUnits);
  pl.units = ceil_div(units, pl.rounds);
  pl.units += pl.units & 1;  // rounds begin at whole pairs
  pl.rounds = ceil_div(units, pl.units);
  pl.passes = ceil_div(m, NT * 8);
  const int ctas = 148 / pl.passes, pairs = (pl.units + 1) / 2;
  double least = 1e30;
  for (int log_kw = gated ? 3 : 4; log_kw >= 0; --log_kw) {
    const int kw = 1 << log_kw;
    if (kw > pairs && kw > 1) continue;
    const double cost = ceil_div(ceil_div(tiles, kWarps / kw), ctas) * (ceil_div(pairs, kw) + 0.6);
    if (cost < least) least = cost, pl.log_kw = log_kw;
  }
  pl.ctas = std::min(ctas, ceil_div(tiles, kWarps >> pl.log_kw));
  // What a leaves of shared memory: a second buffer of partials where two stages stay, then up to four stages.
  const int64_t rest = kSmem - 1024 - (int64_t)pl.units * B::kBytes, buffer = B::kPartial * sizeof(float);
  pl.buffers = rest - 2 * buffer >= 2 * kWarps * kStageBytes ? 2 : 1;
  pl.stages = (int)std::min<int64_t>(4, (rest - pl.buffers * buffer) / (kWarps * kStageBytes));
  return pl;
}

// Whether the tcgen05 kernel takes a product: its three launches cost about 8 us whatever the size, its items
// less than the passes that 17 and more rows take here. Measured, us here / there (bf16, groups of 128,
// m x n x k): 24x4096x4096 15.3 / 15.8, 64x4096x4096 20.8 / 18.4, 32x22016x4096 42.6 / 32.4,
// 64x22016x4096 69 / 38.5, 64x1024x1024 6.0 / 9.6; in one pass 16x12288x4096 20.4 / 22.0.
bool use_tc(int64_t m, int64_t n, int64_t k) { return m > 16 && m * n * k >= int64_t(1) << 29; }

template <typename T, int G, int NT, int EPI>
int launch_mma(const Args& p, float* running, cudaStream_t stream) {
  using B = Block<G, NT>;
  const Plan pl = plan<G, NT>(p.M, p.N, p.K, EPI == HX_EPI_SWIGLU);
  const size_t smem = 1024 + (size_t)kWarps * pl.stages * kStageBytes + pl.buffers * B::kPartial * sizeof(float) +
                      (size_t)pl.units * B::kBytes;
  CUtensorMap w_map;  // [N, K / 2] bytes as 16-bit elements
  const uint64_t dims[2] = {(uint64_t)p.K / 4, (uint64_t)p.N}, strides[1] = {(uint64_t)p.K / 2};
  const uint32_t box[2] = {kPair * kUnitK / 4, 16};
  if (const int s = make_tensor_map(&w_map, p.w, 2, dims, strides, box, HX_BF16)) return s;
  auto kern = gemm_q4_mma_kernel<T, G, NT, EPI>;
  static std::atomic<uint64_t> allowed{0};  // devices where the kernel may use that much shared memory
  if (const int s = allow_shared(reinterpret_cast<const void*>(kern), kSmem, allowed)) return s;
  return hx::cuda_status(launch_ex(kern, dim3((unsigned)(pl.passes * pl.ctas)), dim3(kMmaThreads), smem, stream, 1, p,
                                   w_map, pl, running),
                         "gemm_q4_mma_kernel launch");
}

template <typename T, int G, int NT>
int launch_epilogue(const Args& p, int epilogue, float* running, cudaStream_t stream) {
  return epilogue == HX_EPI_SWIGLU     ? launch_mma<T, G, NT, HX_EPI_SWIGLU>(p, running, stream)
         : epilogue == HX_EPI_RESIDUAL ? launch_mma<T, G, NT, HX_EPI_RESIDUAL>(p, running, stream)
                                       : launch_mma<T, G, NT, HX_EPI_NONE>(p, running, stream);
}

template <typename T, int G>
int launch_rows(const Args& p, int epilogue, float* running, cudaStream_t stream) {
  return p.M <= 8 ? launch_epilogue<T, G, 1>(p, epilogue, running, stream)
                  : launch_epilogue<T, G, 2>(p, epilogue, running, stream);
}

template <typename T>
int launch(const Args& p, int epilogue, float* running, cudaStream_t stream) {
  if constexpr (sizeof(T) == 2) {
    if (use_tc(p.M, p.N, p.K))
      return p.group == 128  ? tc::launch_rows<T, 128>(p, epilogue, running, stream)
             : p.group == 64 ? tc::launch_rows<T, 64>(p, epilogue, running, stream)
                             : tc::launch_rows<T, 32>(p, epilogue, running, stream);
    return p.group == 128  ? launch_rows<T, 128>(p, epilogue, running, stream)
           : p.group == 64 ? launch_rows<T, 64>(p, epilogue, running, stream)
                           : launch_rows<T, 32>(p, epilogue, running, stream);
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

extern "C" size_t hx_gemm_q4_workspace(int64_t m, int64_t n, int64_t k, int64_t group, int dtype) {
  if (m <= 0 || m > 64 || n <= 0 || k <= 0 || group < 32 || group > kUnitK || dtype == HX_F32) return 0;
  if (use_tc(m, n, k)) return tc::workspace(m, n, k, group);
  return k <= (m <= 8 ? 64 : 32) * kUnitK ? 0 : (size_t)m * n * sizeof(float);
}

extern "C" int hx_gemm_q4_launches(int64_t m, int64_t n, int64_t k, int dtype) {
  if (m <= 0) return 0;
  return dtype != HX_F32 && use_tc(m, n, k) ? 3 : 1;
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
  const size_t need = hx_gemm_q4_workspace(m, n, k, group, dtype);
  HX_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && (uintptr_t)workspace % 16 == 0),
             "hx_gemm_q4: workspace too small (%zu < %zu) or misaligned", workspace_bytes, need);
  const Args p{a, (const uint8_t*)w, scales, residual, c, lda, ld_residual, ldc,
               (int)m, (int)n, (int)k, (int)group};
  HX_DISPATCH_DTYPE(dtype, T, return launch<T>(p, epilogue, (float*)workspace, (cudaStream_t)stream));
  return HX_OK;
}
