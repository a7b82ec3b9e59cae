// W4A16 matrix-vector products: Y[M, N] = X[M, K] * W[K, N] for the 1 to 16 rows of a token
// step, W from AWQ tensors in the kernel layout (qweight_mes i32 [K/8, N]).
//
// The weights are read once and everything else is small, so the kernel is bound by their
// K * N / 2 bytes (and by latency below a few megabytes).  One row would leave 46 fp32 FMAs a
// clock and SM at the full memory rate, eight rows 368, more than an SM has, so the products run
// on the tensor cores in the transposed form Y^T = W^T X^T: 16 features by 8 rows by 16 k a step,
// which costs the same for 1 row as for 8.
//
// A warp's 16-byte loads cover 32 features by 32 k: lane (g, c) = (lane / 4, lane % 4) holds the
// words of features 4g..4g+3 and k 8c..8c+7.  The order of k within a product is free as long as
// both operands agree, so each word feeds the A fragment of its own lane without a shuffle, and
// 16 bytes of X row g feed the B fragment.
//
// Arithmetic: (q - z) is exact in bf16 (128 + q by one LOP3, minus 128 + z), the products with
// bf16 x are exact and summed in fp32 over one group of k, and the group's sum is scaled in fp32:
// the weights themselves are never rounded.
#include "common.cuh"

namespace {

constexpr int kFeatures = 32;        // output features of a block
constexpr int kStep = 128;           // k of one step of a warp: four 16-byte loads a lane
constexpr int kRedStride = 36;       // floats between rows of the partial sums (bank spread)
// Most warps of a block: two row tiles take more registers.
constexpr int max_warps(int tiles) { return tiles == 1 ? 32 : 16; }

__device__ __forceinline__ uint4 ld_stream(const uint32_t* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.L2::256B.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

__device__ __forceinline__ uint32_t sub_bf16x2(uint32_t a, uint32_t b) {
  __nv_bfloat162 r = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&a),
                             *reinterpret_cast<__nv_bfloat162*>(&b));
  return *reinterpret_cast<uint32_t*>(&r);
}

// Codes (2j, 2j + 1) of a word as bf16 128 + q.
template <int j>
__device__ __forceinline__ uint32_t codes_pair(uint32_t w) {
  return ((w >> (4 * j)) & 0x000F000Fu) | 0x43004300u;
}

__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Zero points of features 4g..4g+3 from their packed word, as bf16x2 (128 + z, 128 + z).
__device__ __forceinline__ void zero_pairs(uint32_t word, int g, uint32_t (&z)[4]) {
  const uint32_t w = word >> (8 * (g & 1));       // columns 0..3 or 4..7: nibbles 0, 4, 1, 5
  const uint32_t n[4] = {w & 15u, (w >> 16) & 15u, (w >> 4) & 15u, (w >> 20) & 15u};
#pragma unroll
  for (int i = 0; i < 4; ++i) z[i] = (n[i] * 0x00010001u) | 0x43004300u;
}

// kGroup: k per scale.  kTiles: 8-row tiles of X (1 or 2).  kEpi: 0 bf16 (+ bias), 1 fp32 +=
// (+ bias), 2 silu(gate) * up.  Block: `warps` warps share 32 features and deal the steps of K
// among themselves; their sums meet in shared memory, added in warp order, so a call repeats bit
// for bit.
template <int kGroup, int kTiles, int kEpi>
__global__ void __launch_bounds__(32 * max_warps(kTiles))
awq_gemv_kernel(const __nv_bfloat16* __restrict__ X, int64_t ldx, const uint32_t* __restrict__ qw,
                const uint32_t* __restrict__ qz, const __half* __restrict__ scales,
                const __nv_bfloat16* __restrict__ bias, void* Y, int64_t ldy, int M, int N, int K) {
  extern __shared__ float red[];   // [warps][8 kTiles][kRedStride]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const int g = lane >> 2, c = lane & 3;
  const int n0 = blockIdx.x * kFeatures;
  const int f0 = n0 + 4 * g;              // this lane's four features
  const bool live = f0 < N;
  const int fl = live ? f0 : 0;

  float acc[kTiles][2][4] = {};
  for (int step = warp; step < K / kStep; step += warps) {
    const int k0 = step * kStep;
    uint4 w[4], x[kTiles][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[i] = live ? ld_stream(qw + (int64_t)(k0 / 8 + 4 * i + c) * N + fl) : make_uint4(0, 0, 0, 0);
    constexpr int kGroups = kStep / kGroup;
    uint2 sc[kGroups];
    uint32_t zw[kGroups];
#pragma unroll
    for (int i = 0; i < kGroups; ++i) {
      const int64_t gr = k0 / kGroup + i;
      sc[i] = live ? __ldg(reinterpret_cast<const uint2*>(scales + gr * N + fl)) : make_uint2(0, 0);
      zw[i] = live ? __ldg(qz + gr * (N / 8) + fl / 8) : 0u;
    }
#pragma unroll
    for (int t = 0; t < kTiles; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        x[t][i] = 8 * t + g < M
                      ? __ldg(reinterpret_cast<const uint4*>(X + (8 * t + g) * ldx + k0 + 32 * i + 8 * c))
                      : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int gi = 0; gi < kGroups; ++gi) {
      uint32_t z[4];
      zero_pairs(zw[gi], g, z);
      float part[kTiles][2][4] = {};
#pragma unroll
      for (int i = gi * (4 / kGroups); i < (gi + 1) * (4 / kGroups); ++i) {
        const uint32_t wf[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
        uint32_t a[4][4];   // [feature][pair]
#pragma unroll
        for (int f = 0; f < 4; ++f) {
          a[f][0] = sub_bf16x2(codes_pair<0>(wf[f]), z[f]);
          a[f][1] = sub_bf16x2(codes_pair<1>(wf[f]), z[f]);
          a[f][2] = sub_bf16x2(codes_pair<2>(wf[f]), z[f]);
          a[f][3] = sub_bf16x2(codes_pair<3>(wf[f]), z[f]);
        }
#pragma unroll
        for (int t = 0; t < kTiles; ++t)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            mma_bf16(part[t][j], a[2 * j][0], a[2 * j + 1][0], a[2 * j][1], a[2 * j + 1][1],
                     x[t][i].x, x[t][i].y);
            mma_bf16(part[t][j], a[2 * j][2], a[2 * j + 1][2], a[2 * j][3], a[2 * j + 1][3],
                     x[t][i].z, x[t][i].w);
          }
      }
      const float2 s01 = __half22float2(*reinterpret_cast<__half2*>(&sc[gi].x));
      const float2 s23 = __half22float2(*reinterpret_cast<__half2*>(&sc[gi].y));
      const float s[4] = {s01.x, s01.y, s23.x, s23.y};
#pragma unroll
      for (int t = 0; t < kTiles; ++t)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[t][j][e] = fmaf(part[t][j][e], s[2 * j + (e >> 1)], acc[t][j][e]);
    }
  }

  // Row 8t + 2c + e of features 4g..4g+3: one 16-byte store.
#pragma unroll
  for (int t = 0; t < kTiles; ++t)
#pragma unroll
    for (int e = 0; e < 2; ++e)
      *reinterpret_cast<float4*>(&red[(warp * 8 * kTiles + 8 * t + 2 * c + e) * kRedStride + 4 * g]) =
          make_float4(acc[t][0][e], acc[t][0][2 + e], acc[t][1][e], acc[t][1][2 + e]);
  __syncthreads();
  const int n = n0 + lane;
  const float b = bias && n < N ? __bfloat162float(bias[n]) : 0.f;
  for (int m = warp; m < M; m += warps) {
    float y = 0.f;
    for (int w = 0; w < warps; ++w) y += red[(w * 8 * kTiles + m) * kRedStride + lane];
    if (kEpi == 2) {
      const float up = __shfl_xor_sync(0xffffffffu, y, 16);
      if (lane < 16 && n < N)
        static_cast<__nv_bfloat16*>(Y)[m * ldy + n0 / 2 + lane] =
            __float2bfloat16_rn(y / (1.0f + expf(-y)) * up);
    } else if (n < N) {
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

// Warps of a block: enough that the whole grid holds about 24 warps an SM, at most one for each
// step of K.
int warps_for(int64_t N, int64_t K, int most) {
  const int64_t blocks = (N + kFeatures - 1) / kFeatures, steps = K / kStep;
  int w = 4;
  while (w < most && w < steps && blocks * w < 24ll * mes_host::sm_count()) w *= 2;
  return w;
}

template <int kGroup, int kTiles, int kEpi>
int launch(const void* X, int64_t ldx, const int32_t* qw, const int32_t* qz, const void* scales,
           const void* bias, void* Y, int64_t ldy, int64_t M, int64_t N, int64_t K, void* stream) {
  const int warps = warps_for(N, K, max_warps(kTiles));
  const size_t smem = sizeof(float) * warps * 8 * kTiles * kRedStride;
  awq_gemv_kernel<kGroup, kTiles, kEpi>
      <<<(unsigned)((N + kFeatures - 1) / kFeatures), 32 * warps, smem, (cudaStream_t)stream>>>(
          (const __nv_bfloat16*)X, ldx, (const uint32_t*)qw, (const uint32_t*)qz, (const __half*)scales,
          (const __nv_bfloat16*)bias, Y, ldy, (int)M, (int)N, (int)K);
  return mes_host::from_cuda(cudaGetLastError());
}

template <int kGroup, int kTiles, typename... A>
int launch_epi(int epilogue, A... a) {
  return epilogue == 0 ? launch<kGroup, kTiles, 0>(a...)
                       : epilogue == 1 ? launch<kGroup, kTiles, 1>(a...) : launch<kGroup, kTiles, 2>(a...);
}
template <typename... A>
int launch_any(int group, bool two_tiles, int epilogue, A... a) {
  switch (group) {
    case 32: return two_tiles ? launch_epi<32, 2>(epilogue, a...) : launch_epi<32, 1>(epilogue, a...);
    case 64: return two_tiles ? launch_epi<64, 2>(epilogue, a...) : launch_epi<64, 1>(epilogue, a...);
    default: return two_tiles ? launch_epi<128, 2>(epilogue, a...) : launch_epi<128, 1>(epilogue, a...);
  }
}

}  // namespace

extern "C" int mes_awq_gemv(int epilogue, const void* X, int64_t ldx, const int32_t* qweight_mes,
                            const int32_t* qzeros, const void* scales, const void* bias, void* Y,
                            int64_t ldy, int64_t M, int64_t N, int64_t K, int group_size,
                            void* stream) {
  if (epilogue < 0 || epilogue > 2 || M < 0 || M > 16 || N <= 0 || K <= 0) return MES_ERR_INVALID;
  if (group_size != 32 && group_size != 64 && group_size != 128) return MES_ERR_INVALID;
  if (K % kStep || N % 8 || (epilogue == 2 && N % 32) || (epilogue == 2 && bias)) return MES_ERR_INVALID;
  if (N > 0x7fffffffll - kFeatures || K > 0x7fffffffll || K / 8 > 0x7fffffffffffffffll / N) return MES_ERR_INVALID;
  if (ldx < K || ldx % 8 || ldy < (epilogue == 2 ? N / 2 : N)) return MES_ERR_INVALID;
  if (M == 0) return MES_OK;
  if (!X || !qweight_mes || !qzeros || !scales || !Y) return MES_ERR_INVALID;
  if (!aligned(X, 16) || !aligned(qweight_mes, 16) || !aligned(qzeros, 4) || !aligned(scales, 8) ||
      !aligned(bias, 2) || !aligned(Y, epilogue == 1 ? 4 : 2))
    return MES_ERR_ALIGN;
  return launch_any(group_size, M > 8, epilogue, X, ldx, qweight_mes, qzeros, scales, bias, Y, ldy, M,
                    N, K, stream);
}
