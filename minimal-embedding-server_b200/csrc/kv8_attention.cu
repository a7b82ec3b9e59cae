// Attention of new tokens over the 8-bit paged KV cache (layout: kv8.cuh):
//   o_i = sum_t w_it v_t,  w_it = softmax_t(q_i . k_t * scale),  t <= position of query i,
// for the G = Hq / Hkv query heads that share a kv head.  Optionally sums[t] += sum_i w_it.
//
// Bound: with a few query rows for each kv head the 256 bytes of a cached token feed 512 G
// multiply-adds, far below what the tensor cores need, so the kernel is built to keep the cache
// streaming: about 23 bytes a clock and SM at the full memory rate.
//
// Work: a (sequence, kv head, row tile) is an item, 128 keys of it a unit.  The units of all items
// form one line that is cut evenly among the blocks, whatever the lengths are, so no block waits
// for a long sequence.  An item cut between blocks leaves at most two partial results a block (its
// first and its last segment), joined by a second kernel.  The lengths stay on the device.
//
// A block is four warps.  Each takes 32 keys of a unit for itself: its own ring of TMA tiles
// (128-byte swizzle, so the 16-byte reads below meet no bank conflict), its own running maximum
// and sum.  Codes become f16 in registers (exact for both types) and feed mma.sync with the query
// rows as the 16-row operand; with so few rows a tcgen05 tile of 128 rows would be mostly empty
// and its operands would have to be converted and written back to shared memory first.
//
// The order of the contracted index is free, so a lane's 16-byte chunk of a K row is its B fragment
// for four steps, and four lanes' V rows are transposed with byte permutes.
//
// Scales: a page's K scale multiplies its logits.  Its V scale vs goes into the exponent,
// p' = exp2(s + log2(vs) - m), with m the running maximum of s + log2(vs): p' stays within f16
// whatever the scales are, and the softmax sum adds p' / vs.
#include "kv8.cuh"

namespace {

__device__ int g_err_kv8_attention = 0;

constexpr int kWarps = 4, kThreads = 32 * kWarps, kTile = 32, kUnit = kWarps * kTile;
constexpr int kStages = 2;
constexpr int kMaxSeqs = 1024;
constexpr int kHalfBytes = kTile * kv8::kD;                 // one side of a stage
constexpr int kStageBytes = 2 * kHalfBytes;
constexpr int kORow = 144;        // floats of an output row in shared memory (bank spread)
constexpr float kShift = 10.f;    // p' is held times 2^10: f16 keeps weights down to 2^-24 of the largest
// Blocks of an SM that shared memory holds.
constexpr int blocks_per_sm(int R) { return R == 1 ? 2 : 1; }

template <int R>
struct Smem {
  uint8_t ring[kWarps][kStages][kStageBytes];   // 1024-byte aligned
  float o[kWarps][16 * R][kORow];
  uint4 q[R][8][32];                            // A fragments
  float m[kWarps][16 * R], l[kWarps][16 * R];
  float qscale[16 * R];                         // logit factor of a row, in the exp2 domain
  int last[16 * R];                             // last visible key of a row
  float4 sc[kWarps][kStages];                   // K and V scale factors of a tile's two halves
  uint64_t full[kWarps][kStages];
  int prefix[kMaxSeqs + 1];
  int warp_sum[kWarps];
  int abort;
};

struct Params {
  const __nv_bfloat16* q;
  int64_t ldq;
  const float* scales;
  const int32_t* table;
  int64_t width;
  const int32_t* cu;
  const int32_t* ctx;
  int B, T, Hq, Hkv, G, P, page_shift;
  int64_t num_pages;
  float scale;
  __nv_bfloat16* out;
  int* prefix_out;      // [B + 1] for the join
  float* part_o;        // [blocks][2][16 R][128]
  float2* part_ml;      // [blocks][2][16 R]
  float* lse;           // [T * Hq] with sums, else null
  float* logits;        // [T * Hq][max_ctx] with sums, else null
  int64_t max_ctx;
};

// Row p of a tile's 8-key group that lane group n (or column n) holds: rows n and n ^ 1 differ in
// bit 2, and for a fixed parity the rows of n / 2 = 0..3 differ in bits 1 and 2, which is what the
// swizzled K and V reads need to touch every bank once.
__device__ __forceinline__ int key_of(int n) {
  return ((n >> 1) & 1) | (((n >> 2) & 1) << 1) | (((n ^ (n >> 1)) & 1) << 2);
}

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint4& a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two codes of a 32-bit word as f16x2.  int8: bytes (0, 2) and (1, 3); the byte, with its sign bit
// flipped, is the low mantissa of 1024, and 1024 + 128 is taken off again.  e4m3: bytes (0, 1) and
// (2, 3) by the conversion instruction.
__device__ __forceinline__ uint32_t int8_pair(uint32_t w) {
  const uint32_t v = (w & 0x00ff00ffu) ^ 0x64806480u;
  const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&v), __half2half2(__ushort_as_half(0x6480)));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t e4m3_pair(uint32_t w) {
  uint32_t r;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(r) : "r"(w));
  return r;
}
template <int kKind>
__device__ __forceinline__ void convert(uint32_t w, uint32_t& a, uint32_t& b) {
  a = kKind == kv8::kInt8 ? int8_pair(w) : e4m3_pair(w);
  b = kKind == kv8::kInt8 ? int8_pair(w >> 8) : e4m3_pair(w >> 16);
}

// Units of a sequence's items and their number.  A sequence with query rows has at least one unit
// an item, so that rows that see nothing are written too.
__device__ __forceinline__ int units_of(int len) { return len > 0 ? (len + kUnit - 1) / kUnit : 1; }
template <int R>
__device__ __forceinline__ int row_tiles(int n, int G) { return (n * G + 16 * R - 1) / (16 * R); }

struct Seq {
  int r0, n, len;
};
// Lengths of a sequence, made safe: rows within [0, T), tokens within the table.
__device__ __forceinline__ Seq sequence(const Params& p, int b) {
  Seq s;
  s.r0 = p.cu[b];
  s.n = p.cu[b + 1] - s.r0;
  s.len = p.ctx[b];
  if (s.r0 < 0 || s.n < 0 || (int64_t)s.r0 + s.n > p.T || s.len < 0 || s.len > p.width * p.P) {
    atomicCAS(&g_err_kv8_attention, 0, MES_ERR_INVALID);
    s.r0 = s.n = s.len = 0;
  }
  return s;
}

// First unit of block i's share.
__device__ __forceinline__ int share(int64_t units, int i, int blocks) { return (int)(units * i / blocks); }

template <int kKind, int R, bool kSums>
__global__ void __launch_bounds__(kThreads, blocks_per_sm(R))
kv8_attention_kernel(const __grid_constant__ CUtensorMap map, const Params p) {
  extern __shared__ uint8_t raw[];
  Smem<R>& sh = *reinterpret_cast<Smem<R>*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  constexpr int kRows = 16 * R;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;

  if (tid == 0) {
    sh.abort = 0;
    for (int w = 0; w < kWarps; ++w)
      for (int s = 0; s < kStages; ++s) mes::mbar_init(&sh.full[w][s], 1);
    mes::fence_barrier_init();
    mes::tma_prefetch_desc(&map);
  }
  // Units before each sequence.
  int total = 0;
  for (int b0 = 0; b0 < p.B; b0 += kThreads) {
    const int b = b0 + tid;
    int x = 0;
    if (b < p.B) {
      const Seq s = sequence(p, b);
      x = s.n > 0 ? units_of(s.len) * p.Hkv * row_tiles<R>(s.n, p.G) : 0;
    }
    const int mine = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 31) sh.warp_sum[warp] = x;
    __syncthreads();
    int before = total;
    for (int w = 0; w < warp; ++w) before += sh.warp_sum[w];
    if (b < p.B) sh.prefix[b] = before + x - mine;
    for (int w = 0; w < kWarps; ++w) total += sh.warp_sum[w];
  }
  if (tid == 0) sh.prefix[p.B] = total;
  __syncthreads();
  if (blockIdx.x == 0)
    for (int b = tid; b <= p.B; b += kThreads) p.prefix_out[b] = sh.prefix[b];
  const int blocks = min((int)gridDim.x, total);
  if ((int)blockIdx.x >= blocks) return;
  const int first = share(total, blockIdx.x, blocks), end = share(total, blockIdx.x + 1, blocks);

  auto find = [&](int u) {      // sequence of unit u: the last b with prefix[b] <= u that has units
    int lo = 0, hi = p.B;       // prefix[lo] <= u < prefix[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (sh.prefix[mid] <= u) lo = mid; else hi = mid;
    }
    return lo;
  };

  // ---- the warp's tiles: unit first + i is its tile i ----
  // Lane j holds what tiles 32 i + j need: the cache rows of its halves and its scales.
  int t_row0 = 0, t_row1 = 0, t_halves = 0;
  float4 t_sc = make_float4(0.f, 0.f, 0.f, 0.f);
  auto look_up = [&](int i0) {
    const int u = first + i0 + lane;
    t_halves = 0;
    if (u >= end) return;
    const int b = find(u);
    const Seq s = sequence(p, b);
    const int units = units_of(s.len), rest = u - sh.prefix[b], item = rest / units;
    const int t0 = (rest - item * units) * kUnit + warp * kTile;
    const int h = item / row_tiles<R>(s.n, p.G);
    float ks[2] = {0.f, 0.f}, vs[2] = {1.f, 1.f};
    int row[2] = {0, 0};
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int t = t0 + 16 * half;
      if (t >= s.len) continue;
      int64_t page = p.table[(int64_t)b * p.width + (t >> p.page_shift)];
      if (page < 0 || page >= p.num_pages) {
        atomicCAS(&g_err_kv8_attention, 0, MES_ERR_INVALID);
        page = 0;
      }
      const int64_t run = page * 2 * p.Hkv + h;
      row[half] = (int)(run * p.P + (t & (p.P - 1)));
      ks[half] = p.scales[run];
      vs[half] = p.scales[run + p.Hkv];
      if (vs[half] == 0.f) vs[half] = -1.f;      // marks V values that are all 0
      ++t_halves;
    }
    t_row0 = row[0];
    t_row1 = row[1];
    t_sc = make_float4(ks[0], ks[1], vs[0], vs[1]);
  };
  auto issue = [&](int i) {      // the whole warp; tile i into stage i % kStages
    if (first + i >= end) return;
    if ((i & 31) == 0) look_up(i);
    const int src = i & 31, stage = i % kStages;
    const int halves = __shfl_sync(0xffffffffu, t_halves, src);
    const int row0 = __shfl_sync(0xffffffffu, t_row0, src), row1 = __shfl_sync(0xffffffffu, t_row1, src);
    if (lane == src) sh.sc[warp][stage] = t_sc;
    if (halves == 0 || lane != 0) return;
    uint64_t* bar = &sh.full[warp][stage];
    uint8_t* k = sh.ring[warp][stage];
    const int vrow = p.Hkv << p.page_shift;
    if (p.P >= kTile) {       // one box of 32 rows a side
      mes::mbar_arrive_expect_tx(bar, kStageBytes);
      mes::tma_load_2d(k, &map, bar, 0, row0);
      mes::tma_load_2d(k + kHalfBytes, &map, bar, 0, row0 + vrow);
    } else {                  // pages of 16: a box for each half that holds tokens
      mes::mbar_arrive_expect_tx(bar, halves * (kStageBytes / 2));
      mes::tma_load_2d(k, &map, bar, 0, row0);
      mes::tma_load_2d(k + kHalfBytes, &map, bar, 0, row0 + vrow);
      if (halves == 2) {
        mes::tma_load_2d(k + kHalfBytes / 2, &map, bar, 0, row1);
        mes::tma_load_2d(k + kHalfBytes + kHalfBytes / 2, &map, bar, 0, row1 + vrow);
      }
    }
  };
  for (int i = 0; i < kStages; ++i) issue(i);

  uint32_t phase = 0;           // bit s: parity of stage s's next load
  bool ok = true;
  for (int u = first; u < end;) {
    // ---- segment: units [u, stop) of one item ----
    const int b = find(u);
    const Seq s = sequence(p, b);
    const int units = units_of(s.len), tiles = row_tiles<R>(s.n, p.G);
    const int rest = u - sh.prefix[b], item = rest / units, unit0 = rest - item * units;
    const int h = item / tiles, tile = item - h * tiles;
    const int item0 = u - unit0, stop = min(end, item0 + units);
    const int row_base = tile * kRows, rows = min(kRows, s.n * p.G - row_base);
    const int start = s.len - s.n;
    __syncthreads();            // the previous segment's readers of q / o are done
    // Query rows: f16 times a power of two that brings the row's largest value near 2^8.
    for (int e = tid; e < kRows * 8; e += kThreads) {
      const int r = e >> 3, part = e & 7, row = row_base + r;
      float f[16];
      float amax = 0.f;
      if (r < rows) {
        const int i = row / p.G, head = h * p.G + row - i * p.G;
        const uint4* src = reinterpret_cast<const uint4*>(p.q + (int64_t)(s.r0 + i) * p.ldq + head * kv8::kD + part * 16);
        const uint4 v[2] = {__ldg(src), __ldg(src + 1)};
        const __nv_bfloat162* hv = reinterpret_cast<const __nv_bfloat162*>(v);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float2 t = __bfloat1622float2(hv[j]);
          f[2 * j] = t.x;
          f[2 * j + 1] = t.y;
          amax = fmaxf(amax, fmaxf(fabsf(t.x), fabsf(t.y)));
        }
        if (part == 0) sh.last[r] = start + i;
      } else {
#pragma unroll
        for (int j = 0; j < 16; ++j) f[j] = 0.f;
        if (part == 0) sh.last[r] = 0x7fffffff;
      }
#pragma unroll
      for (int o = 4; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
      // 2^e just below the row's maximum, within what both powers of two can be.
      const int ex = min(max((int)((__float_as_uint(amax) >> 23) & 255) - 127, -110), 120);
      const float down = __uint_as_float((uint32_t)(127 + 8 - ex) << 23), up = __uint_as_float((uint32_t)(127 - 8 + ex) << 23);
      if (part == 0) sh.qscale[r] = p.scale * 1.4426950408889634f * up;
      const int cc = part & 3, u0 = (part >> 2) * 4, fl = (r & 7) * 4 + cc, hi = (r >> 3) & 1;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float e0 = f[4 * w] * down, e1 = f[4 * w + 1] * down, e2 = f[4 * w + 2] * down, e3 = f[4 * w + 3] * down;
        const __half2 lo2 = kKind == kv8::kInt8 ? __floats2half2_rn(e0, e2) : __floats2half2_rn(e0, e1);
        const __half2 hi2 = kKind == kv8::kInt8 ? __floats2half2_rn(e1, e3) : __floats2half2_rn(e2, e3);
        uint32_t* frag = reinterpret_cast<uint32_t*>(&sh.q[r >> 4][u0 + w][fl]);
        frag[hi] = *reinterpret_cast<const uint32_t*>(&lo2);
        frag[2 + hi] = *reinterpret_cast<const uint32_t*>(&hi2);
      }
    }
    __syncthreads();
    float qs[R][2];
    int last[R][2];
    int first_last = 0x7fffffff;      // keys every row of this lane sees
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        qs[r][e] = sh.qscale[16 * r + 8 * e + g];
        last[r][e] = min(sh.last[16 * r + 8 * e + g], s.len - 1);
        first_last = min(first_last, last[r][e]);
      }
    first_last = __reduce_min_sync(0xffffffffu, first_last);

    float O[R][16][4], m[R][2], l[R][2];
#pragma unroll
    for (int r = 0; r < R; ++r) {
#pragma unroll
      for (int t = 0; t < 16; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) O[r][t][e] = 0.f;
      m[r][0] = m[r][1] = -INFINITY;
      l[r][0] = l[r][1] = 0.f;
    }

    for (; u < stop; ++u) {
      const int i = u - first, stage = i % kStages;
      const int t0 = (u - item0) * kUnit + warp * kTile;
      if (t0 < s.len) {
        ok = mes::mbar_wait_warp(&sh.full[warp][stage], (phase >> stage) & 1, &sh.abort,
                                 &g_err_kv8_attention, MES_ERR_TIMEOUT) && ok;
        phase ^= 1u << stage;
        const uint8_t* kt = sh.ring[warp][stage];
        const uint8_t* vt = kt + kHalfBytes;
        float4 sc = sh.sc[warp][stage];
        // V codes of scale 0 count as 0 (their factor is then free, here 1); so do slots past the
        // end, which hold anything, NaN codes too, and 0 * NaN is NaN.
        const int v_end[2] = {sc.z < 0.f ? 0 : s.len, sc.w < 0.f ? 0 : s.len};
        const bool tail = t0 + kTile > min(v_end[0], v_end[1]);
        sc.z = fabsf(sc.z);
        sc.w = fabsf(sc.w);
        // ---- S = Q K^T ----
        float S[R][4][4];
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int nt = 0; nt < 4; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) S[r][nt][e] = 0.f;
        uint4 kw[4][2];
        const int kg = key_of(g);
#pragma unroll
        for (int nt = 0; nt < 4; ++nt)
#pragma unroll
          for (int half = 0; half < 2; ++half)
            kw[nt][half] = *reinterpret_cast<const uint4*>(kt + (8 * nt + kg) * kv8::kD + (((c + 4 * half) ^ kg) << 4));
#pragma unroll
        for (int st = 0; st < 8; ++st) {
          uint4 a[R];
#pragma unroll
          for (int r = 0; r < R; ++r) a[r] = sh.q[r][st][lane];
#pragma unroll
          for (int nt = 0; nt < 4; ++nt) {
            const uint4& v = kw[nt][st >> 2];
            const uint32_t w = (st & 3) == 0 ? v.x : (st & 3) == 1 ? v.y : (st & 3) == 2 ? v.z : v.w;
            uint32_t b0, b1;
            convert<kKind>(w, b0, b1);
#pragma unroll
            for (int r = 0; r < R; ++r) mma_f16(S[r][nt], a[r], b0, b1);
          }
        }
        // ---- logits, running maximum ----
        const float lv[2] = {__log2f(sc.z), __log2f(sc.w)};
        const bool masked = t0 + kTile - 1 > first_last;
        uint4 P[R][2];
#pragma unroll
        for (int r = 0; r < R; ++r) {
          float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
          for (int nt = 0; nt < 4; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float ks = nt < 2 ? sc.x : sc.y;
              float x = S[r][nt][e] * (ks * qs[r][e >> 1]);
              if (masked) x = t0 + 8 * nt + key_of(2 * c + (e & 1)) > last[r][e >> 1] ? -INFINITY : x;
              if (kSums) {
                const int row = 16 * r + 8 * (e >> 1) + g, t = t0 + 8 * nt + key_of(2 * c + (e & 1));
                if (row < rows && t < s.len) {
                  const int q = row_base + row, qi = q / p.G;
                  p.logits[((int64_t)(s.r0 + qi) * p.Hq + h * p.G + q - qi * p.G) * p.max_ctx + t] = x;
                }
              }
              x += lv[nt >> 1];
              S[r][nt][e] = x;
              mx[e >> 1] = fmaxf(mx[e >> 1], x);
            }
          bool grew = false;
          float alpha[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 1));
            mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 2));
            const float now = fmaxf(m[r][e], mx[e]);
            grew |= now > m[r][e];
            alpha[e] = now == -INFINITY ? 1.f : ex2(m[r][e] - now);
            m[r][e] = now;
          }
          if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
            for (int t = 0; t < 16; ++t)
#pragma unroll
              for (int e = 0; e < 4; ++e) O[r][t][e] *= alpha[e >> 1];
            l[r][0] *= alpha[0];
            l[r][1] *= alpha[1];
          }
          float off[2], add[2][2] = {};
#pragma unroll
          for (int e = 0; e < 2; ++e) off[e] = m[r][e] == -INFINITY ? 0.f : m[r][e] - kShift;
          uint32_t pw[4][2];
#pragma unroll
          for (int nt = 0; nt < 4; ++nt) {
            float x[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              x[e] = ex2(S[r][nt][e] - off[e >> 1]);
              add[nt >> 1][e >> 1] += x[e];
            }
            const __half2 p0 = __floats2half2_rn(x[0], x[1]), p1 = __floats2half2_rn(x[2], x[3]);
            pw[nt][0] = *reinterpret_cast<const uint32_t*>(&p0);
            pw[nt][1] = *reinterpret_cast<const uint32_t*>(&p1);
          }
          const float iv[2] = {__fdividef(1.f, sc.z), __fdividef(1.f, sc.w)};
#pragma unroll
          for (int e = 0; e < 2; ++e) l[r][e] += add[0][e] * iv[0] + add[1][e] * iv[1];
#pragma unroll
          for (int j = 0; j < 2; ++j)
            P[r][j] = make_uint4(pw[2 * j][0], pw[2 * j][1], pw[2 * j + 1][0], pw[2 * j + 1][1]);
        }
        // ---- O += P V ----
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          uint4 v[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int key = 8 * (2 * j + (e >> 1)) + key_of(2 * c + (e & 1));
            v[e] = *reinterpret_cast<const uint4*>(vt + key * kv8::kD + ((g ^ (key & 7)) << 4));
            if (tail && t0 + key >= v_end[j]) v[e] = make_uint4(0, 0, 0, 0);
          }
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const uint32_t w[4] = {q == 0 ? v[0].x : q == 1 ? v[0].y : q == 2 ? v[0].z : v[0].w,
                                   q == 0 ? v[1].x : q == 1 ? v[1].y : q == 2 ? v[1].z : v[1].w,
                                   q == 0 ? v[2].x : q == 1 ? v[2].y : q == 2 ? v[2].z : v[2].w,
                                   q == 0 ? v[3].x : q == 1 ? v[3].y : q == 2 ? v[3].z : v[3].w};
#pragma unroll
            for (int half = 0; half < 2; ++half) {    // values 2 half and 2 half + 1 of the four
              // Bytes of the two keys side by side as `convert` pairs them.
              constexpr uint32_t kSel[2][2] = {{0x5410, 0x7632}, {0x5140, 0x7362}};
              const uint32_t x = __byte_perm(w[0], w[1], kSel[kKind][half]);
              const uint32_t y = __byte_perm(w[2], w[3], kSel[kKind][half]);
              uint32_t x0, x1, y0, y1;
              convert<kKind>(x, x0, x1);
              convert<kKind>(y, y0, y1);
#pragma unroll
              for (int r = 0; r < R; ++r) {
                mma_f16(O[r][4 * q + 2 * half], P[r][j], x0, y0);
                mma_f16(O[r][4 * q + 2 * half + 1], P[r][j], x1, y1);
              }
            }
          }
        }
      }
      __syncwarp();               // the stage has been read by every lane
      issue(i + kStages);
    }

    // ---- join the four warps ----
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        l[r][e] += __shfl_xor_sync(0xffffffffu, l[r][e], 1);
        l[r][e] += __shfl_xor_sync(0xffffffffu, l[r][e], 2);
        const int row = 16 * r + 8 * e + g;
        if (c == 0) {
          sh.m[warp][row] = m[r][e];
          sh.l[warp][row] = l[r][e];
        }
        // Lane (g, c) holds values 32 c .. 32 c + 31 of its rows.
        float4* dst = reinterpret_cast<float4*>(&sh.o[warp][row][36 * c]);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          dst[q] = make_float4(O[r][4 * q][2 * e], O[r][4 * q + 1][2 * e], O[r][4 * q + 2][2 * e], O[r][4 * q + 3][2 * e]);
          dst[4 + q] = make_float4(O[r][4 * q][2 * e + 1], O[r][4 * q + 1][2 * e + 1], O[r][4 * q + 2][2 * e + 1],
                                   O[r][4 * q + 3][2 * e + 1]);
        }
      }
    __syncthreads();
    const bool whole = unit0 == 0 && stop == item0 + units;
    const int slot = 2 * blockIdx.x + (item0 + unit0 == first ? 0 : 1);
    for (int e = tid; e < rows * 32; e += kThreads) {
      const int row = e >> 5, d4 = e & 31;          // four values a thread
      float mx = -INFINITY;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) mx = fmaxf(mx, sh.m[w][row]);
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
      float sum = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float f = mx == -INFINITY ? 0.f : ex2(sh.m[w][row] - mx);
        const float4 x = *reinterpret_cast<const float4*>(&sh.o[w][row][4 * d4 + 4 * (d4 >> 3)]);
        o.x += f * x.x;
        o.y += f * x.y;
        o.z += f * x.z;
        o.w += f * x.w;
        sum += f * sh.l[w][row];
      }
      if (whole) {
        const int q = row_base + row, qi = q / p.G;
        const int64_t at = (int64_t)(s.r0 + qi) * p.Hq + h * p.G + q - qi * p.G;
        const float inv = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;      // NaN stays NaN
        *reinterpret_cast<uint2*>(p.out + at * kv8::kD + 4 * d4) =
            make_uint2(mes::pack_bf16x2(o.x * inv, o.y * inv), mes::pack_bf16x2(o.z * inv, o.w * inv));
        if (kSums && d4 == 0) p.lse[at] = mx - kShift + log2f(sum);
      } else {
        *reinterpret_cast<float4*>(p.part_o + ((int64_t)slot * kRows + row) * kv8::kD + 4 * d4) = o;
        if (d4 == 0) p.part_ml[(int64_t)slot * kRows + row] = make_float2(mx, sum);
      }
    }
  }
  if (!ok) {
    // A wait ran out: no block leaves while copies into its memory may be in flight.
    int mine = 0;
    for (int s = 0; s < kStages; ++s)
      mes::mbar_wait_limit(&sh.full[warp][s], ((phase >> s) & 1) ^ 1, &mine, &g_err_kv8_attention,
                           MES_ERR_TIMEOUT, mes::kWaitLimitNs);
  }
}

// ---- join the partial results of items cut between blocks: a warp for each (token, query head) ----
template <int R, bool kSums>
__global__ void __launch_bounds__(128)
kv8_join_kernel(const Params p, int grid) {
  constexpr int kRows = 16 * R;
  const int lane = threadIdx.x & 31;
  const int64_t at = blockIdx.x * 4ll + (threadIdx.x >> 5);
  if (at >= (int64_t)p.T * p.Hq) return;
  const int token = (int)(at / p.Hq), head = (int)(at - (int64_t)token * p.Hq), h = head / p.G;
  int lo = 0, hi = p.B;                       // cu[lo] <= token < cu[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (p.cu[mid] <= token) lo = mid; else hi = mid;
  }
  const Seq s = sequence(p, lo);
  if (s.n <= 0 || token < s.r0 || token >= s.r0 + s.n) return;
  const int total = p.prefix_out[p.B], blocks = min(grid, total);
  const int row = (token - s.r0) * p.G + head - h * p.G, tile = row / kRows;
  const int units = units_of(s.len);
  const int u0 = p.prefix_out[lo] + (h * row_tiles<R>(s.n, p.G) + tile) * units, u1 = u0 + units;
  // The blocks whose shares meet [u0, u1).
  int from = (int)((int64_t)u0 * blocks / total);
  while (from + 1 < blocks && share(total, from + 1, blocks) <= u0) ++from;
  while (from > 0 && share(total, from, blocks) > u0) --from;
  if (share(total, from + 1, blocks) >= u1) return;         // not cut
  float mx = -INFINITY, sum = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i = from; i < blocks; ++i) {
    const int begin = share(total, i, blocks);
    if (begin >= u1) break;
    const int64_t slot = ((int64_t)2 * i + (begin < u0 ? 1 : 0)) * kRows + row - tile * kRows;
    const float2 ml = p.part_ml[slot];
    const float4 x = *reinterpret_cast<const float4*>(p.part_o + slot * kv8::kD + 4 * lane);
    const float now = fmaxf(mx, ml.x);
    if (now == -INFINITY) continue;
    const float a = ex2(mx - now), f = ex2(ml.x - now);
    o.x = o.x * a + x.x * f;
    o.y = o.y * a + x.y * f;
    o.z = o.z * a + x.z * f;
    o.w = o.w * a + x.w * f;
    sum = sum * a + ml.y * f;
    mx = now;
  }
  const float inv = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;
  *reinterpret_cast<uint2*>(p.out + at * kv8::kD + 4 * lane) =
      make_uint2(mes::pack_bf16x2(o.x * inv, o.y * inv), mes::pack_bf16x2(o.z * inv, o.w * inv));
  if (kSums && lane == 0) p.lse[at] = mx - kShift + log2f(sum);
}

// ---- sums[t] += sum over the rows of a kv head of exp2(logit - lse): a thread for each key ----
__global__ void __launch_bounds__(256)
kv8_sums_kernel(const Params p, float* sums) {
  const int64_t b = blockIdx.y / p.Hkv;
  const int h = (int)(blockIdx.y - b * p.Hkv);
  const Seq s = sequence(p, (int)b);
  const int t = blockIdx.x * 256 + threadIdx.x;
  if (t >= s.len || s.n == 0) return;
  float add = 0.f;
  for (int i = 0; i < s.n; ++i) {
    const int64_t at = (int64_t)(s.r0 + i) * p.Hq + h * p.G;
    for (int q = 0; q < p.G; ++q) {
      const float x = p.logits[(at + q) * p.max_ctx + t];
      add += x == -INFINITY ? 0.f : ex2(x - p.lse[at + q]);
    }
  }
  const int64_t page = p.table[b * p.width + (t >> p.page_shift)];
  if (page < 0 || page >= p.num_pages) return;              // recorded by the attention kernel
  float* at = sums + (page * p.Hkv + h) * p.P + (t & (p.P - 1));
  *at += add;
}

// Row tiles of 32 are for calls whose kv heads have more than 16 query rows: the converted keys
// then feed twice the products.
int row_tile_factor(int64_t max_new, int G) { return max_new * G > 16 ? 2 : 1; }
int max_blocks(int R) { return mes_host::sm_count() * blocks_per_sm(R); }

constexpr int64_t up256(int64_t x) { return (x + 255) / 256 * 256; }
struct Layout {
  int64_t prefix, part_o, part_ml, lse, logits, bytes;
};
Layout layout(int64_t T, int64_t B, int Hq, int R, int64_t max_ctx) {
  Layout w;
  const int64_t slots = 2ll * max_blocks(R) * 16 * R;
  w.prefix = 0;
  w.part_o = up256(4 * (B + 1));
  w.part_ml = w.part_o + slots * kv8::kD * 4;
  w.lse = up256(w.part_ml + slots * 8);
  w.logits = up256(w.lse + (max_ctx > 0 ? 4 * T * Hq : 0));
  w.bytes = w.logits + 4 * T * Hq * max_ctx;
  return w;
}
bool valid_sizes(int64_t T, int64_t B, int Hq, int Hkv, int64_t max_new, int64_t max_ctx) {
  return T >= 0 && B >= 0 && B <= kMaxSeqs && Hkv > 0 && Hkv <= 1024 && Hq > 0 && Hq % Hkv == 0 && Hq <= 8192 &&
         max_new >= 0 && max_new <= T && T <= 0x7fffffffll / Hq && max_ctx >= 0 && max_ctx <= 0x7fffffffll;
}

template <int kKind, int R, bool kSums>
int launch(const CUtensorMap& map, const Params& p, float* sums, void* stream) {
  auto kernel = kv8_attention_kernel<kKind, R, kSums>;
  const size_t smem = sizeof(Smem<R>) + 1024;
  static std::atomic<uint64_t> configured{0};
  int st = mes_host::once_per_device(configured, [&] {
    return mes_host::from_cuda(
        cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  });
  if (st != MES_OK) return st;
  const int grid = mes_host::persistent_ctas() * blocks_per_sm(R);
  kernel<<<grid, kThreads, smem, (cudaStream_t)stream>>>(map, p);
  const int64_t rows = (int64_t)p.T * p.Hq;
  kv8_join_kernel<R, kSums><<<(unsigned)((rows + 3) / 4), 128, 0, (cudaStream_t)stream>>>(p, grid);
  if (kSums)
    kv8_sums_kernel<<<dim3((unsigned)((p.max_ctx + 255) / 256), (unsigned)(p.B * p.Hkv)), 256, 0, (cudaStream_t)stream>>>(p, sums);
  return mes_host::from_cuda(cudaGetLastError());
}

}  // namespace

extern "C" int mes_kv8_attention_take_error(int* code) {
  int v = 0, zero = 0;
  cudaError_t e = cudaMemcpyFromSymbol(&v, g_err_kv8_attention, sizeof(int));
  if (e != cudaSuccess) return MES_ERR_CUDA;
  e = cudaMemcpyToSymbol(g_err_kv8_attention, &zero, sizeof(int));
  *code = v;
  return mes_host::from_cuda(e);
}

extern "C" int64_t mes_kv8_attention_workspace_size(int64_t T, int64_t B, int Hq, int Hkv, int64_t max_new,
                                                    int64_t max_context) {
  if (!valid_sizes(T, B, Hq, Hkv, max_new, max_context)) return -1;
  return layout(T, B, Hq, row_tile_factor(max_new, Hq / Hkv), max_context).bytes;
}

extern "C" int mes_kv8_attention(int dtype, const void* q, int64_t ldq, const void* codes, const float* scales,
                                 float* sums, const int32_t* block_table, int64_t table_width,
                                 const int32_t* cu_new, const int32_t* context_lens, int64_t B, int64_t T,
                                 int64_t max_new, int Hq, int Hkv, int D, int page_size, int64_t num_pages,
                                 float scale, void* out, void* workspace, int64_t workspace_bytes, void* stream) {
  if (!kv8::valid_cache(dtype, num_pages, Hkv, D, page_size)) return MES_ERR_INVALID;
  if (table_width <= 0 || table_width > 0x7fffffffll / page_size) return MES_ERR_INVALID;
  const int64_t max_ctx = sums ? table_width * page_size : 0;
  if (!valid_sizes(T, B, Hq, Hkv, max_new, max_ctx)) return MES_ERR_INVALID;
  if (ldq < (int64_t)Hq * D || ldq % 8) return MES_ERR_INVALID;
  if (B == 0 || T == 0 || max_new == 0) return MES_OK;
  if (!q || !codes || !scales || !block_table || !cu_new || !context_lens || !out || !workspace) return MES_ERR_INVALID;
  if (!kv8::aligned(q, 16) || !kv8::aligned(codes, 16) || !kv8::aligned(scales, 4) || !kv8::aligned(sums, 4) ||
      !kv8::aligned(block_table, 4) || !kv8::aligned(cu_new, 4) || !kv8::aligned(context_lens, 4) ||
      !kv8::aligned(out, 16) || !kv8::aligned(workspace, 256))
    return MES_ERR_ALIGN;
  const int G = Hq / Hkv, R = row_tile_factor(max_new, G);
  const Layout w = layout(T, B, Hq, R, max_ctx);
  if (workspace_bytes < w.bytes) return MES_ERR_INVALID;
  // Units are counted in 32 bits.
  const int64_t tiles = (max_new * G + 16 * R - 1) / (16 * R);
  if (((table_width * page_size + kUnit - 1) / kUnit) * Hkv > 0x7fffffffll / (B * tiles)) return MES_ERR_INVALID;
  if (sums && B * Hkv > 65535) return MES_ERR_INVALID;
  CUtensorMap map;
  const int box = page_size < kTile ? page_size : kTile;
  if (!mes_host::make_map_2d(&map, codes, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, (uint64_t)num_pages * 2 * Hkv * page_size,
                             kv8::kD, kv8::kD, box, kv8::kD, CU_TENSOR_MAP_SWIZZLE_128B))
    return MES_ERR_CUDA;
  char* ws = static_cast<char*>(workspace);
  Params p;
  p.q = (const __nv_bfloat16*)q;
  p.ldq = ldq;
  p.scales = scales;
  p.table = block_table;
  p.width = table_width;
  p.cu = cu_new;
  p.ctx = context_lens;
  p.B = (int)B;
  p.T = (int)T;
  p.Hq = Hq;
  p.Hkv = Hkv;
  p.G = G;
  p.P = page_size;
  p.page_shift = __builtin_ctz((unsigned)page_size);
  p.num_pages = num_pages;
  p.scale = scale;
  p.out = (__nv_bfloat16*)out;
  p.prefix_out = (int*)(ws + w.prefix);
  p.part_o = (float*)(ws + w.part_o);
  p.part_ml = (float2*)(ws + w.part_ml);
  p.lse = sums ? (float*)(ws + w.lse) : nullptr;
  p.logits = sums ? (float*)(ws + w.logits) : nullptr;
  p.max_ctx = max_ctx;
  const bool i8 = dtype == kv8::kInt8;
  if (R == 1) {
    if (sums) return i8 ? launch<kv8::kInt8, 1, true>(map, p, sums, stream) : launch<kv8::kE4m3, 1, true>(map, p, sums, stream);
    return i8 ? launch<kv8::kInt8, 1, false>(map, p, sums, stream) : launch<kv8::kE4m3, 1, false>(map, p, sums, stream);
  }
  if (sums) return i8 ? launch<kv8::kInt8, 2, true>(map, p, sums, stream) : launch<kv8::kE4m3, 2, true>(map, p, sums, stream);
  return i8 ? launch<kv8::kInt8, 2, false>(map, p, sums, stream) : launch<kv8::kE4m3, 2, false>(map, p, sums, stream);
}
