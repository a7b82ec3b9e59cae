// W4A16 matrix-vector products: Y[M, N] = X[M, K] * W[K, N] for the 1 to 16 rows of a token
// step, W from AWQ tensors in the kernel layout (qweight_mes i32 [K/8, N]).
//
// The weights are read once and everything else is small, so the bound is their K * N / 2 bytes
// (and latency below a few megabytes).  One row would leave 46 fp32 FMAs a clock and SM at the
// full memory rate, eight rows 368, more than an SM has, so the products run on the tensor cores
// in the transposed form Y^T = W^T X^T: 16 features by 8 rows by 16 k a step, which costs the
// same for 1 row as for 8.
//
// A block is some warps that share 32 or 64 features and deal the steps of K (128 k each) among
// themselves.  Each warp has its own ring of TMA tiles, 16 words of 32 features each (2 KB) and
// the rows of X that go with them, so that many loads are in flight without a register.  A lane
// (g, c) = (lane / 4, lane % 4) reads the words of features 4g..4g+3 for one block of eight k,
// 16 bytes; the order of k within a product is free as long as both operands agree, so each word
// feeds the A fragment of its own lane without a shuffle, and 16 bytes of X row g feed the B
// fragment.
//
// Arithmetic: sum_k (q - z) x = sum_k q x - z sum_k x over one group of k, both sums from the tensor
// cores in fp32, then scaled in fp32: the weights themselves are never rounded.  What costs time is
// taking the codes out of their words, so they are used where they lie: masked out of a word, a
// code at bits 0-3 or 4-7 of a half is the bf16 number q 2^-133 or q 2^-129 (bf16 is linear from
// zero up to 2^-125), so one shift and four masks make eight operands.  X is multiplied by 2^60 or
// 2^56 to meet them, which is exact for |x| < 2^67, and the result by 2^73.  A sum is then a multiple of
// 2^-76, fp32's least number times 2^73: values of x below 2^-53 lose bits, which norms' and activations' rows
// have next to none of.
//
// Measured: 8 rows of 4096 x 24576 with silu 16.2 us (52 MB, 3.2 TB/s, half of the copy rate: the
// integer pipe that masks the codes is 45% busy, and 384 blocks share 148 SMs unevenly), 16 rows 24.2; 1 row of
// 2048 x 1024 3.4 us, a launch and one round of loads.
#include "common.cuh"

namespace {

__device__ int g_err_awq_gemv = 0;

constexpr int kFeatures = 32;        // output features of a weight tile
constexpr int kStep = 128;           // k of a step
constexpr int kRedStride = 36;       // floats between rows of the partial sums (bank spread)
constexpr int kMaxWarps = 16;
constexpr int kWBytes = kStep / 8 * kFeatures * 4;                     // 2 KB of weights
constexpr int stage_bytes(int cols, int tiles) { return cols * kWBytes + tiles * 8 * kStep * 2; }

constexpr float kUp = 9444732965739290427392.f;      // 2^73

// Two bf16 values times 2^60 or 2^56 (the power as its bf16 pair).
__device__ __forceinline__ uint32_t scale_x(uint32_t x, uint32_t power) {
  __nv_bfloat162 r = __hmul2(*reinterpret_cast<__nv_bfloat162*>(&x), *reinterpret_cast<__nv_bfloat162*>(&power));
  return *reinterpret_cast<uint32_t*>(&r);
}
constexpr uint32_t kPow60 = 0x5d805d80u, kPow56 = 0x5b805b80u;

// The first product of a sum (`add` false) has nothing to add to.
__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1, bool add) {
  if (add) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  } else {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%10, %10, %10, %10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
  }
}

// Zero points of features 4g..4g+3 from their packed word: nibbles 0, 4, 1, 5 of its half for those
// features, read as 2^23 + z.
__device__ __forceinline__ void zero_points(uint32_t word, int g, float (&z)[4]) {
  const uint32_t w = word >> (8 * (g & 1));
  const uint32_t n[4] = {w & 15u, (w >> 16) & 15u, (w >> 4) & 15u, (w >> 20) & 15u};
#pragma unroll
  for (int i = 0; i < 4; ++i) z[i] = __uint_as_float(0x4b000000u | n[i]) - 8388608.f;
}

// kGroup: k per scale.  kCols: tiles of 32 features (1 or 2).  kTiles: 8-row tiles of X (1 or 2).  kEpi: 0 bf16 (+ bias), 1 fp32 +=
// (+ bias), 2 silu(gate) * up.  The warps' sums meet in shared memory, added in warp order, so a
// call repeats bit for bit.
template <int kGroup, int kCols, int kTiles, int kEpi>
__global__ void __launch_bounds__(32 * kMaxWarps)
awq_gemv_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x,
                const uint32_t* __restrict__ qz, const __half* __restrict__ scales,
                const __nv_bfloat16* __restrict__ bias, void* Y, int64_t ldy, int M, int N, int K,
                int stages) {
  extern __shared__ __align__(1024) uint8_t smem[];   // [warps][stages]: weights, X; then the barriers
  constexpr int kStage = stage_bytes(kCols, kTiles), kX = kCols * kWBytes, kGroups = kStep / kGroup;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const int g = lane >> 2, c = lane & 3;
  const int n0 = blockIdx.x * kCols * kFeatures, steps = K / kStep;
  uint8_t* ring = smem + warp * stages * kStage;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + warps * stages * kStage) + warp * stages;
  int& abort_flag = *reinterpret_cast<int*>(smem + warps * stages * (kStage + 8));
  if (threadIdx.x == 0) abort_flag = 0;
  if (lane == 0) {
    for (int i = 0; i < stages; ++i) mes::mbar_init(full + i, 1);
    mes::fence_barrier_init();
  }
  const uint32_t x_bytes = (uint32_t)M * kStep * 2;
  auto load = [&](int step, int stage) {     // one lane
    uint8_t* at = ring + stage * kStage;
    mes::mbar_arrive_expect_tx(full + stage, kX + x_bytes);
#pragma unroll
    for (int i = 0; i < kCols; ++i)      // columns past the end arrive as zeros
      mes::tma_load_2d(at + i * kWBytes, &map_w, full + stage, n0 + i * kFeatures, step * (kStep / 8));
    mes::tma_load_2d(at + kX, &map_x, full + stage, step * kStep, 0);
    mes::tma_load_2d(at + kX + kTiles * 1024, &map_x, full + stage, step * kStep + 64, 0);
  };
  if (lane == 0)
    for (int i = 0; i < stages && warp + i * warps < steps; ++i) load(warp + i * warps, i);
  __syncthreads();

  // This lane's four features of each tile; past the end the last ones stand in, whose results
  // are not stored.
  int f0[kCols];
#pragma unroll
  for (int i = 0; i < kCols; ++i) f0[i] = min(n0 + i * kFeatures + 4 * g, N - 4);
  const __half* sp = scales + (int64_t)warp * kGroups * N;
  const uint32_t* zp = qz + (int64_t)warp * kGroups * (N / 8);
  uint2 sc[kGroups][kCols];
  uint32_t zw[kGroups][kCols];
  auto fetch = [&] {        // scales and zero points of the step the pointers are at
#pragma unroll
    for (int i = 0; i < kGroups; ++i)
#pragma unroll
      for (int j = 0; j < kCols; ++j) {
        sc[i][j] = __ldg(reinterpret_cast<const uint2*>(sp + (int64_t)i * N + f0[j]));
        zw[i][j] = __ldg(zp + (int64_t)i * (N / 8) + f0[j] / 8);
      }
    sp += (int64_t)warps * kGroups * N;
    zp += (int64_t)warps * kGroups * (N / 8);
  };
  // Block of eight k of product i: lane c's four are two apart where the groups allow it, so that
  // the 16-byte reads of eight lanes, two rows of X or four of words, meet every bank once.
  auto block8 = [&](int i) { return kGroup == 32 ? 4 * i + c : 8 * (i >> 1) + 2 * c + (i & 1); };

  float acc[kTiles][kCols][2][4] = {};
  bool ok = true;
  int stage = 0;
  uint32_t parity = 0;
  if (warp < steps) fetch();
  for (int step = warp; step < steps; step += warps) {
    ok = mes::mbar_wait_warp(full + stage, parity, &abort_flag, &g_err_awq_gemv, MES_ERR_TIMEOUT) && ok;
    const uint8_t* ws = ring + stage * kStage;
    const uint8_t* xs = ws + kX;
    uint2 s_now[kGroups][kCols];
    uint32_t z_now[kGroups][kCols];
#pragma unroll
    for (int i = 0; i < kGroups; ++i)
#pragma unroll
      for (int j = 0; j < kCols; ++j) {
        s_now[i][j] = sc[i][j];
        z_now[i][j] = zw[i][j];
      }
    if (step + warps < steps) fetch();
#pragma unroll
    for (int gi = 0; gi < kGroups; ++gi) {
      float part[kTiles][kCols][2][4], xsum[kTiles][4];
#pragma unroll
      for (int i = gi * (4 / kGroups); i < (gi + 1) * (4 / kGroups); ++i) {
        const int kb = block8(i);
        uint4 x[kTiles];
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {    // 64 k a box
          x[t] = *reinterpret_cast<const uint4*>(xs + (kb >> 3) * kTiles * 1024 + (8 * t + g) * 128 + (((kb & 7) ^ g) << 4));
          x[t].x = scale_x(x[t].x, kPow60);
          x[t].y = scale_x(x[t].y, kPow56);
          x[t].z = scale_x(x[t].z, kPow60);
          x[t].w = scale_x(x[t].w, kPow56);
        }
        uint4 w[kCols];
#pragma unroll
        for (int n = 0; n < kCols; ++n)
          w[n] = *reinterpret_cast<const uint4*>(ws + n * kWBytes + kb * 128 + ((g ^ (kb & 7)) << 4));
        // Products of one sum are kept apart: each waits for the one before it.
#pragma unroll
        for (int half = 0; half < 2; ++half) {
#pragma unroll
          for (int n = 0; n < kCols; ++n)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const uint32_t w0 = (j ? w[n].z : w[n].x) >> (8 * half), w1 = (j ? w[n].w : w[n].y) >> (8 * half);
#pragma unroll
              for (int t = 0; t < kTiles; ++t)
                mma_bf16(part[t][n][j], w0 & 0x000F000Fu, w1 & 0x000F000Fu, w0 & 0x00F000F0u, w1 & 0x00F000F0u,
                         half ? x[t].z : x[t].x, half ? x[t].w : x[t].y, half || i % (4 / kGroups));
            }
          // The sum of x, as if every code were 1.
#pragma unroll
          for (int t = 0; t < kTiles; ++t)
            mma_bf16(xsum[t], 0x00010001u, 0x00010001u, 0x00100010u, 0x00100010u, half ? x[t].z : x[t].x,
                     half ? x[t].w : x[t].y, half || i % (4 / kGroups));
        }
      }
#pragma unroll
      for (int n = 0; n < kCols; ++n) {
        float z[4];
        zero_points(z_now[gi][n], g, z);
        const float2 s01 = __half22float2(*reinterpret_cast<const __half2*>(&s_now[gi][n].x));
        const float2 s23 = __half22float2(*reinterpret_cast<const __half2*>(&s_now[gi][n].y));
        const float sf[4] = {s01.x, s01.y, s23.x, s23.y};
#pragma unroll
        for (int t = 0; t < kTiles; ++t)
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int f = 2 * j + (e >> 1);
              acc[t][n][j][e] = fmaf(fmaf(-z[f], xsum[t][e], part[t][n][j][e]), sf[f], acc[t][n][j][e]);
            }
      }
    }
    __syncwarp();           // the stage has been read by every lane
    const int ahead = step + stages * warps;
    if (lane == 0 && ahead < steps) load(ahead, stage);
    if (++stage == stages) {
      stage = 0;
      parity ^= 1;
    }
  }
  if (!ok) {
    // A wait ran out: no block leaves while copies into its memory may be in flight.
    int mine = 0;
    for (int i = 0; i < stages; ++i) {
      mes::mbar_wait_limit(full + i, 0, &mine, &g_err_awq_gemv, MES_ERR_TIMEOUT, mes::kWaitLimitNs);
      mes::mbar_wait_limit(full + i, 1, &mine, &g_err_awq_gemv, MES_ERR_TIMEOUT, mes::kWaitLimitNs);
    }
  }

  // Row 8t + 2c + e of features 4g..4g+3: one 16-byte store.  The rings are idle by now.
  __syncthreads();
  float* red = reinterpret_cast<float*>(smem);   // [warps][kCols][8 kTiles][kRedStride]
#pragma unroll
  for (int t = 0; t < kTiles; ++t)
#pragma unroll
    for (int n = 0; n < kCols; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e)
        *reinterpret_cast<float4*>(&red[((warp * kCols + n) * 8 * kTiles + 8 * t + 2 * c + e) * kRedStride + 4 * g]) =
            make_float4(acc[t][n][0][e], acc[t][n][0][2 + e], acc[t][n][1][e], acc[t][n][1][2 + e]);
  __syncthreads();
  for (int i = warp; i < M * kCols; i += warps) {
    const int m = i / kCols, col = i - m * kCols, n = n0 + col * kFeatures + lane;
    float y = 0.f;
#pragma unroll 4
    for (int w = 0; w < warps; ++w) y += red[((w * kCols + col) * 8 * kTiles + m) * kRedStride + lane];
    y *= kUp;
    if (kEpi == 2) {
      const float up = __shfl_xor_sync(0xffffffffu, y, 16);
      if (lane < 16 && n < N)
        static_cast<__nv_bfloat16*>(Y)[m * ldy + (n0 + col * kFeatures) / 2 + lane] =
            __float2bfloat16_rn(y / (1.0f + expf(-y)) * up);
    } else if (n < N) {
      const float b = bias ? __bfloat162float(bias[n]) : 0.f;
      if (kEpi == 1) {
        float* r = static_cast<float*>(Y) + m * ldy + n;
        *r = *r + (y + b);
      } else {
        static_cast<__nv_bfloat16*>(Y)[m * ldy + n] = __float2bfloat16_rn(y + b);
      }
    }
  }
}

bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

// How a product is cut: a power of two of warps a block (4 to 16, up to 16 an SM; other numbers
// measured 10 to 25% slower, and more warps or stages an SM than let the whole grid be resident at
// once up to 50%), and stages of a ring.
struct Shape {
  int warps, stages;
  int smem;
};
Shape shape_for(int64_t tiles, int64_t K, int cols, int row_tiles) {
  const int64_t steps = K / kStep, sms = mes_host::sm_count(), stage = stage_bytes(cols, row_tiles) + 8;
  int64_t w = 4;
  while (w < kMaxWarps && w < steps && 2 * w * tiles <= 16 * sms) w *= 2;
  const int64_t s = steps > w ? 2 : 1;
  const int64_t ring = stage * w * s + 16, red = 4 * cols * w * 8 * row_tiles * kRedStride;
  return {(int)w, (int)s, (int)(ring > red ? ring : red)};
}

template <int kGroup, int kCols, int kTiles, int kEpi>
int launch(const CUtensorMap& map_w, const CUtensorMap& map_x, const int32_t* qz, const void* scales,
           const void* bias, void* Y, int64_t ldy, int64_t M, int64_t N, int64_t K, void* stream) {
  auto kernel = awq_gemv_kernel<kGroup, kCols, kTiles, kEpi>;
  constexpr int kMost = 2 * kMaxWarps * (stage_bytes(kCols, kTiles) + 8) + 16;
  static std::atomic<uint64_t> configured{0};
  int st = mes_host::once_per_device(configured, [&] {
    return mes_host::from_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMost));
  });
  if (st != MES_OK) return st;
  const int64_t tiles = (N + kCols * kFeatures - 1) / (kCols * kFeatures);
  const Shape s = shape_for(tiles, K, kCols, kTiles);
  kernel<<<(unsigned)tiles, 32 * s.warps, s.smem, (cudaStream_t)stream>>>(
      map_w, map_x, (const uint32_t*)qz, (const __half*)scales, (const __nv_bfloat16*)bias, Y, ldy, (int)M, (int)N,
      (int)K, s.stages);
  return mes_host::from_cuda(cudaGetLastError());
}

template <int kGroup, int kCols, int kTiles, typename... A>
int launch_epi(int epilogue, const A&... a) {
  return epilogue == 0 ? launch<kGroup, kCols, kTiles, 0>(a...)
                       : epilogue == 1 ? launch<kGroup, kCols, kTiles, 1>(a...) : launch<kGroup, kCols, kTiles, 2>(a...);
}
template <int kGroup, typename... A>
int launch_tiles(bool wide, bool two_tiles, int epilogue, const A&... a) {
  if (two_tiles) return launch_epi<kGroup, 1, 2>(epilogue, a...);
  return wide ? launch_epi<kGroup, 2, 1>(epilogue, a...) : launch_epi<kGroup, 1, 1>(epilogue, a...);
}
template <typename... A>
int launch_any(int group, const A&... a) {
  switch (group) {
    case 32: return launch_tiles<32>(a...);
    case 64: return launch_tiles<64>(a...);
    default: return launch_tiles<128>(a...);
  }
}

}  // namespace

extern "C" int mes_awq_gemv_take_error(int* code) {
  int v = 0, zero = 0;
  cudaError_t e = cudaMemcpyFromSymbol(&v, g_err_awq_gemv, sizeof(int));
  if (e != cudaSuccess) return MES_ERR_CUDA;
  e = cudaMemcpyToSymbol(g_err_awq_gemv, &zero, sizeof(int));
  *code = v;
  return mes_host::from_cuda(e);
}

extern "C" int mes_awq_gemv(int epilogue, const void* X, int64_t ldx, const int32_t* qweight_mes,
                            const int32_t* qzeros, const void* scales, const void* bias, void* Y,
                            int64_t ldy, int64_t M, int64_t N, int64_t K, int group_size,
                            void* stream) {
  if (epilogue < 0 || epilogue > 2 || M < 0 || M > 16 || N <= 0 || K <= 0) return MES_ERR_INVALID;
  if (group_size != 32 && group_size != 64 && group_size != 128) return MES_ERR_INVALID;
  if (K % kStep || N % 8 || (epilogue == 2 && N % 32) || (epilogue == 2 && bias)) return MES_ERR_INVALID;
  if (N > 0x7fffffffll - kFeatures || K > 0x7fffffffll) return MES_ERR_INVALID;
  if (ldx < K || ldx % 8 || ldy < (epilogue == 2 ? N / 2 : N)) return MES_ERR_INVALID;
  if (M == 0) return MES_OK;
  if (!X || !qweight_mes || !qzeros || !scales || !Y) return MES_ERR_INVALID;
  if (!aligned(X, 16) || !aligned(qweight_mes, 16) || !aligned(qzeros, 4) || !aligned(scales, 8) ||
      !aligned(bias, 2) || !aligned(Y, epilogue == 1 ? 4 : 2))
    return MES_ERR_ALIGN;
  CUtensorMap map_w, map_x;
  if (!mes_host::make_map_2d(&map_w, qweight_mes, CU_TENSOR_MAP_DATA_TYPE_INT32, 4, K / 8, N, N, kStep / 8,
                             kFeatures, CU_TENSOR_MAP_SWIZZLE_128B) ||
      !mes_host::make_map_2d(&map_x, X, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, M, K, ldx, (uint32_t)M, 64,
                             CU_TENSOR_MAP_SWIZZLE_128B))
    return MES_ERR_CUDA;
  // Two tiles of features share the work on X where that leaves two blocks an SM (8 rows of
  // 4096 x 24576: 16.2 us against 19.6 with one).
  const bool wide = N >= 4 * (int64_t)mes_host::sm_count() * kFeatures;
  return launch_any(group_size, wide, M > 8, epilogue, map_w, map_x, qzeros, scales, bias, Y, ldy, M, N, K, stream);
}
