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
// for a long sequence; beginning an item counts as a few units.  An item cut between blocks leaves
// at most two partial results a block (its first and its last segment), joined by a second kernel.
// The lengths stay on the device.  Where no sequence can be long (the table has room for four units
// at most), items are dealt whole and there is no second kernel: 256 sequences of 100 to 500 tokens
// take 58 instead of 63 us.  One of 500 alone takes 10.1 instead of 8.8, but its call, which the
// host bounds, 12.3 instead of 15.6.
//
// A block is four warps.  Each takes 32 keys of a unit for itself: its own ring of TMA tiles
// (128-byte swizzle, so the 16-byte reads below meet no bank conflict), its own running maximum
// and sum.  Codes become f16 in registers (exact for both types) and feed mma.sync in the
// transposed form, S^T = K Q^T and O^T = V^T P^T: keys, then head dimensions, are the 16-row
// operand and 8 query rows the columns, so that a token step's 1 to 8 rows fill a product.  A
// tcgen05 tile would have the converted codes written back to shared memory first.
//
// The order of the contracted index is free, so a lane's 16-byte chunk of a K row is its A fragment
// for four steps, and four lanes' V rows are transposed with byte permutes.
//
// Scales: a page's K scale multiplies its logits.  Its V scale vs goes into the exponent,
// p' = exp2(s + log2(vs) - m), with m a running reference near the maximum of s + log2(vs), so that p'
// stays within f16.  The softmax sum needs exp2(s) alone: it adds p' 2^b / vs, which is exp2(s - (m - b)).
// The base 2^b is 1 while scales are ordinary (2^-40 to 2^40) and otherwise a power of two near the largest
// that the warp has seen, so that neither exponent leaves its range whatever the scales are.  V of scale 0, or
// of less than 2^-60 of the base, counts as 0: its codes are cleared, and its scale is taken as one that
// does not lift m above what the others need.  When partial results meet, outputs are joined by m and sums
// by m - b, and the output is multiplied by 2^b at the end.
//
// Measured: two sequences of 131072 tokens, 8 kv heads, one query each 94 us (537 MB, 5.7 TB/s, 0.87 of
// the copy rate); 64 of 100 to 8192 tokens 101 us (0.85).  With 138 query rows for each kv head it
// comes to 178 TFLOP/s (8 sequences of 16384 tokens, 104 us): two warps a scheduler, which is what the
// registers leave, do not hide one another's latencies.
#include "kv8.cuh"

namespace {

__device__ int g_err_kv8_attention = 0;

constexpr int kWarps = 4, kThreads = 32 * kWarps, kTile = 32, kUnit = kWarps * kTile;
constexpr int kStages = 2;
constexpr int kMaxSeqs = 1024;
constexpr int kMaxPrefix = 48;      // what the room for three blocks an SM leaves
constexpr int kWholeUnits = 4;      // most units of an item that is dealt whole
constexpr int kHalfBytes = kTile * kv8::kD;                 // one side of a stage
constexpr int kStageBytes = 2 * kHalfBytes;
// p' is 2^kShift for a tile's largest value when its reference is set, and may grow to 2^kMost: f16
// keeps weights down to 2^-24 of that largest one and ends at 2^16.
constexpr float kShift = 10.f, kMost = 15.f;
// Blocks of an SM: registers and shared memory hold three with 8 query rows, two with more.
constexpr int blocks_per_sm(int N) { return N == 1 ? 3 : 2; }
// Log2 of the scales around 1 that leave the base there; how far the base may be below a scale otherwise; and
// how far a scale below the base, before its V counts as 0 (f16 keeps weights down to 2^-35 of the largest).
constexpr float kOrdinary = 40.f, kBaseStep = 16.f, kBaseRange = 60.f;
// What beginning an item costs a block, in units of work.  Against 0: 64 ragged sequences of up to
// 8192 tokens take 100 instead of 105 us.
constexpr int kSegmentCost = 2;

// N: 8-row tiles of query rows.
template <int N>
struct Smem {
  uint8_t ring[kWarps][kStages][kStageBytes];   // 1024-byte aligned
  union {
    float4 o[kWarps][4 * N][32];                // halves of the warps' results on their way to others
    uint2 q[N][8][32];                          // Q fragments
  };
  uint4 raw[8 * N][16];                         // the next segment's query rows
  float2 ml[kWarps][8 * N];                     // reference and sum of the warps' rows
  float qscale[8 * N];                          // logit factor of a row, in the exp2 domain
  int last[8 * N];                              // last visible key of a row
  float2 sc[kWarps][kStages][3];                // factors of a tile's two halves: K scale, log2 and
                                                // reciprocal of the V scale (negative: not an ordinary one)
  float base[kWarps];                           // the warps' bases, -inf where all V counted as 0
  uint64_t full[kWarps][kStages];
  int2 warp_sum[kWarps];
  int abort;
  int2 prefix[kMaxPrefix + 1];                  // units and items before every `coarse`-th sequence, and all
};

struct Params {
  const __nv_bfloat16* q;
  int64_t ldq;
  const float* scales;
  const int32_t* table;
  int64_t width;
  const int32_t* cu;
  const int32_t* ctx;
  int B, T, max_new, Hq, Hkv, G, P, page_shift;
  int64_t num_pages;
  float scale;
  __nv_bfloat16* out;
  float* part_o;        // [blocks][2][8 N][128]
  float4* part_ml;      // [blocks][2][8 N]: reference of the outputs, that of the sum, the sum
  float* lse;           // [T * Hq] with sums, else null
  float* logits;        // [T * Hq][max_ctx] with sums, else null
  int64_t max_ctx;
  int whole;            // units of every item where items are dealt whole, else 0
};

// Key of an 8-key group that is row n of a product: keys of n and n ^ 1 differ in bit 2, and for a
// fixed parity the keys of n / 2 = 0..3 differ in bits 1 and 2, which is what the swizzled K and V
// reads need to touch every bank once.
__device__ __forceinline__ int key_of(int n) {
  return ((n >> 1) & 1) | (((n >> 2) & 1) << 1) | (((n ^ (n >> 1)) & 1) << 2);
}

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                        uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Transposes an 8 x 8 matrix of 16-bit values: lane (g, c) gives row g, columns 2c and 2c + 1.
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ void copy16_async(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(mes::smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ uint32_t word_of(const uint4& v, int i) {
  return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w;
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
  uint32_t v;      // (w & 0x00ff00ff) ^ 0x64806480
  asm("lop3.b32 %0, %1, %2, %3, 0x6a;" : "=r"(v) : "r"(w), "r"(0x00ff00ffu), "r"(0x64806480u));
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

// Units of an item of a sequence: at least one, so that rows that see nothing are written too; the
// same for all where items are dealt whole.
__device__ __forceinline__ int units_of(const Params& p, int len) {
  return p.whole > 0 ? p.whole : len > 0 ? (len + kUnit - 1) / kUnit : 1;
}
template <int kRows>
__device__ __forceinline__ int row_tiles(int n, int G) { return (n * G + kRows - 1) / kRows; }

struct Seq {
  int r0, n, len;
};
// Lengths of a sequence, made safe: rows within [0, T), at most max_new, tokens within the table.
__device__ __forceinline__ Seq sequence(const Params& p, int b) {
  Seq s;
  s.r0 = p.cu[b];
  s.n = p.cu[b + 1] - s.r0;
  s.len = p.ctx[b];
  if (s.r0 < 0 || s.n < 0 || (int64_t)s.r0 + s.n > p.T || s.n > p.max_new || s.len < 0 || s.len > p.width * p.P) {
    atomicCAS(&g_err_kv8_attention, 0, MES_ERR_INVALID);
    s.r0 = s.n = s.len = 0;
  }
  return s;
}

// First unit of block i's share.
// It is floor(units i / blocks) without a 64-bit division.
struct Shares {
  int blocks, whole, rest;
  __device__ __forceinline__ Shares(int units, int blocks) : blocks(blocks), whole(units / blocks), rest(units - whole * blocks) {}
  __device__ __forceinline__ int at(int i) const { return whole * i + (int)((uint32_t)(rest * i) / (uint32_t)blocks); }
};

// A block's share of the line of units, with row tiles of kRows query rows.
struct Found {
  int b, base, items;   // a sequence, the units and the items before it
  Seq s;
};
struct Segment {        // the units of one item that a block has
  int h, row_base, rows, item0, units, stop;
  Seq s;
};
struct Tile {           // 32 keys: the pages and the rows of its halves (of the page, then of the cache), how
  int page[2], row[2];  // many of them exist, the kv head, their scales
  int halves, h;
  float2 ks, vs;
};

// The line of units; for the shares, each item has kSegmentCost units of nothing before its own.
struct Count {
  int units, items;
  __device__ __forceinline__ int with(int c) const { return units + c * items; }
};
template <int kRows>
__device__ __forceinline__ Count count_of(const Params& p, const Seq& s) {
  const int items = s.n > 0 ? p.Hkv * row_tiles<kRows>(s.n, p.G) : 0;
  return {items > 0 ? items * units_of(p, s.len) : 0, items};
}
// Units of nothing before an item's own: none where items are dealt whole or each unit has a block.
template <int kRows>
__device__ __forceinline__ int cost_of(const Params& p, int units, int grid) {
  return p.whole > 0 || units <= grid ? 0 : kSegmentCost;
}

template <int kRows>
struct Line {
  const Params& p;
  int2* prefix;         // units and items before every `coarse`-th sequence, and all
  int coarse, marks, first, end;

  // The whole block; returns false where it has no share.
  __device__ bool set_up(int2* warp_sum) {
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    coarse = (p.B + kMaxPrefix - 1) / kMaxPrefix;
    marks = (p.B + coarse - 1) / coarse;
    Count total = {0, 0};
    for (int b0 = 0; b0 < p.B; b0 += kThreads) {
      const int b = b0 + tid;
      const Count mine = b < p.B ? count_of<kRows>(p, sequence(p, b)) : Count{0, 0};
      int x = mine.units, y = mine.items;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int px = __shfl_up_sync(0xffffffffu, x, o), py = __shfl_up_sync(0xffffffffu, y, o);
        if (lane >= o) {
          x += px;
          y += py;
        }
      }
      if (b0 > 0) __syncthreads();
      if (lane == 31) warp_sum[warp] = make_int2(x, y);
      __syncthreads();
      Count before = total;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const int2 sum = warp_sum[w];
        if (w < warp) {
          before.units += sum.x;
          before.items += sum.y;
        }
        total.units += sum.x;
        total.items += sum.y;
      }
      if (b < p.B && b % coarse == 0)
        prefix[b / coarse] = make_int2(before.units + x - mine.units, before.items + y - mine.items);
    }
    if (tid == 0) prefix[marks] = make_int2(total.units, total.items);
    __syncthreads();
    const int cost = cost_of<kRows>(p, total.units, gridDim.x);
    const int grain = p.whole > 0 ? p.whole : 1;     // a multiple of this many units for each block
    const int all = total.with(cost) / grain, blocks = min((int)gridDim.x, all);
    if ((int)blockIdx.x >= blocks) return false;
    const Shares shares(all, blocks);
    first = shares.at(blockIdx.x) * grain;
    end = shares.at(blockIdx.x + 1) * grain;
    if (cost > 0) {             // both at once, in odd and even lanes
      const int x = units_before(lane & 1 ? end : first, cost);
      first = __shfl_sync(0xffffffffu, x, 0);
      end = __shfl_sync(0xffffffffu, x, 1);
    }
    return first < end;
  }
  // The sequence that place x of the line is in: `cost` 0, its units alone.
  __device__ __forceinline__ Found find(int x, int cost = 0) const {
    int lo = 0, hi = marks;     // prefix[lo] <= x < prefix[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      const int2 at = prefix[mid];
      if (at.x + cost * at.y <= x) lo = mid; else hi = mid;
    }
    const int2 at = prefix[lo];
    Found f = {lo * coarse, at.x, at.y, sequence(p, lo * coarse)};
    // Past sequences that end before x (those without query rows have no units).
    while (true) {
      const Count mine = count_of<kRows>(p, f.s);
      if (f.base + mine.units + cost * (f.items + mine.items) > x || f.b + 1 >= p.B) return f;
      f.base += mine.units;
      f.items += mine.items;
      f.s = sequence(p, ++f.b);
    }
  }
  __device__ __forceinline__ int units_before(int x, int cost) const {
    const Found at = find(x, cost);
    const int units = units_of(p, at.s.len), rest = x - at.base - cost * at.items, item = rest / (units + cost);
    return at.base + item * units + max(rest - item * (units + cost) - cost, 0);
  }
  __device__ __forceinline__ Segment segment(int u) const {
    Segment g;
    const Found at = find(u);
    g.s = at.s;
    g.units = units_of(p, g.s.len);
    const int tiles = row_tiles<kRows>(g.s.n, p.G), rest = u - at.base, item = rest / g.units;
    g.h = item / tiles;
    g.row_base = (item - g.h * tiles) * kRows;
    g.rows = min(kRows, g.s.n * p.G - g.row_base);
    g.item0 = u - (rest - item * g.units);
    g.stop = min(end, g.item0 + g.units);
    return g;
  }
  // Tile `sub` of unit u, in two steps with a load each: its pages, then their scales.
  __device__ __forceinline__ Tile tile(int u, int sub) const {
    Tile t = {{0, 0}, {0, 0}, 0, 0, make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
    if (u >= end) return t;
    const Found at = find(u);
    const Seq s = at.s;
    const int units = units_of(p, s.len), rest = u - at.base, item = rest / units;
    const int t0 = (rest - item * units) * kUnit + sub * kTile;
    t.h = item / row_tiles<kRows>(s.n, p.G);
#pragma unroll
    for (int half = 0; half < 2; ++half)
      if (t0 + 16 * half < s.len) {
        t.page[half] = p.table[(int64_t)at.b * p.width + ((t0 + 16 * half) >> p.page_shift)];
        t.row[half] = (t0 + 16 * half) & (p.P - 1);
        ++t.halves;
      }
    return t;
  }
  __device__ __forceinline__ void resolve(Tile& t) const {
    int64_t run[2];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      if (t.page[half] < 0 || t.page[half] >= p.num_pages) {
        atomicCAS(&g_err_kv8_attention, 0, MES_ERR_INVALID);
        t.page[half] = 0;
      }
      run[half] = (int64_t)t.page[half] * 2 * p.Hkv + t.h;       // that of K; that of V is Hkv further
      t.row[half] += (int)(run[half] * p.P);
    }
    if (t.halves > 0) {
      t.ks.x = p.scales[run[0]];
      t.vs.x = p.scales[run[0] + p.Hkv];
    }
    if (t.halves > 1) {
      t.ks.y = p.scales[run[1]];
      t.vs.y = p.scales[run[1] + p.Hkv];
    }
  }
  // Sixteen values of a query row of a segment: task e is part e % 8 of row e / 8.
  __device__ __forceinline__ const __nv_bfloat16* q_source(const Segment& g, int e) const {
    const int q = g.row_base + (e >> 3), i = q / p.G;
    return p.q + (int64_t)(g.s.r0 + i) * p.ldq + (g.h * p.G + q - i * p.G) * kv8::kD + (e & 7) * 16;
  }
};

// One lane: a tile's copies into a stage.
__device__ __forceinline__ void load_tile(const Params& p, const CUtensorMap& map, const Tile& t, uint8_t* k, uint64_t* bar) {
  const int vrow = p.Hkv << p.page_shift;
  if (p.P >= kTile) {       // one box of 32 rows a side
    mes::mbar_arrive_expect_tx(bar, kStageBytes);
    mes::tma_load_2d(k, &map, bar, 0, t.row[0]);
    mes::tma_load_2d(k + kHalfBytes, &map, bar, 0, t.row[0] + vrow);
  } else {                  // pages of 16: a box for each half that holds tokens
    mes::mbar_arrive_expect_tx(bar, t.halves * (kStageBytes / 2));
    mes::tma_load_2d(k, &map, bar, 0, t.row[0]);
    mes::tma_load_2d(k + kHalfBytes, &map, bar, 0, t.row[0] + vrow);
    if (t.halves == 2) {
      mes::tma_load_2d(k + kHalfBytes / 2, &map, bar, 0, t.row[1]);
      mes::tma_load_2d(k + kHalfBytes + kHalfBytes / 2, &map, bar, 0, t.row[1] + vrow);
    }
  }
}
// Log2 of a V scale and its reciprocal, negative where the scale is not an ordinary one.
__device__ __forceinline__ float2 v_factors(float vs) {
  const float lv = log2f(vs);
  return make_float2(lv, fabsf(lv) <= kOrdinary ? ex2(-lv) : -1.f);
}
// Part `part` of a query row: f16 times a power of two that brings the row's largest value near
// 2^8, as the B fragments of its four steps; returns the logit factor of the row.  The eight lanes
// of a row call it together.
template <int kKind>
__device__ __forceinline__ float q_fragments(const uint4 (&v)[2], bool real, float scale, uint2 (&frag)[4]) {
  const __nv_bfloat162* hv = reinterpret_cast<const __nv_bfloat162*>(v);
  float f[16], amax = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float2 t = real ? __bfloat1622float2(hv[j]) : make_float2(0.f, 0.f);
    f[2 * j] = t.x;
    f[2 * j + 1] = t.y;
    amax = fmaxf(amax, fmaxf(fabsf(t.x), fabsf(t.y)));
  }
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  // 2^e just below the row's maximum, within what both powers of two can be.
  const int ex = min(max((int)((__float_as_uint(amax) >> 23) & 255) - 127, -110), 120);
  const float down = __uint_as_float((uint32_t)(127 + 8 - ex) << 23), up = __uint_as_float((uint32_t)(127 - 8 + ex) << 23);
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const float e0 = f[4 * w] * down, e1 = f[4 * w + 1] * down, e2 = f[4 * w + 2] * down, e3 = f[4 * w + 3] * down;
    const __half2 lo2 = kKind == kv8::kInt8 ? __floats2half2_rn(e0, e2) : __floats2half2_rn(e0, e1);
    const __half2 hi2 = kKind == kv8::kInt8 ? __floats2half2_rn(e1, e3) : __floats2half2_rn(e2, e3);
    frag[w] = make_uint2(*reinterpret_cast<const uint32_t*>(&lo2), *reinterpret_cast<const uint32_t*>(&hi2));
  }
  return scale * 1.4426950408889634f * up;
}

// From the logits of a tile to the B fragments of P: S holds products of query rows and codes on
// entry, logits (in the exp2 domain) after.  Value e of S[t][mt] is key t0 + 16 mt + 8 (e / 2) +
// key_of(g), row 8 t + 2 c + e % 2.  p' = exp2(s + log2(vs) - m): m is a reference that need not be
// the maximum, only near it: it moves when a value passes 2^kMost, where f16 would end, so most
// tiles neither reduce over lanes nor touch O.
template <int N, bool kSums>
__device__ __forceinline__ void weights(const Params& p, float (&S)[N][2][4], float (&O)[N][8][4], float (&m)[N][2],
                                        float (&l)[N][2], uint2 (&P)[N][2], const float (&qs)[N][2], const int (&last)[N][2],
                                        const int64_t (&logit_row)[N][2], float2 ks, float2 lv, float2 iv, int t0, int len,
                                        bool masked, int kg) {
#pragma unroll
  for (int t = 0; t < N; ++t) {
    float x[2][4], mx = -INFINITY;
#pragma unroll
    for (int mt = 0; mt < 2; ++mt)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        S[t][mt][e] *= (mt == 0 ? ks.x : ks.y) * qs[t][e & 1];
        x[mt][e] = S[t][mt][e] + ((mt == 0 ? lv.x : lv.y) - m[t][e & 1]);
      }
    if (kSums) {
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int key = t0 + 16 * mt + 8 * (e >> 1) + kg;
          if (logit_row[t][e & 1] >= 0 && key < len)
            p.logits[logit_row[t][e & 1] + key] = key > last[t][e & 1] ? -INFINITY : S[t][mt][e];
        }
    }
    if (masked) {
      __syncwarp();       // keeps this a branch: as selects it would cost every tile
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (t0 + 16 * mt + 8 * (e >> 1) + kg > last[t][e & 1]) x[mt][e] = -INFINITY;
    }
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) mx = fmaxf(mx, fmaxf(fmaxf(x[mt][0], x[mt][1]), fmaxf(x[mt][2], x[mt][3])));
    if (__any_sync(0xffffffffu, mx > kMost)) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        // The row's largest value of this tile, without the old reference.
        float top = -INFINITY;
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
          for (int i2 = e; i2 < 4; i2 += 2)
            if (x[mt][i2] != -INFINITY) top = fmaxf(top, S[t][mt][i2] + (mt == 0 ? lv.x : lv.y));
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        const float now = fmaxf(m[t][e], top - kShift);
        if (now > m[t][e]) {
          const float alpha = ex2(m[t][e] - now);
          l[t][e] *= alpha;
#pragma unroll
          for (int d = 0; d < 8; ++d) {
            O[t][d][e] *= alpha;
            O[t][d][2 + e] *= alpha;
          }
          m[t][e] = now;
#pragma unroll
          for (int mt = 0; mt < 2; ++mt)
#pragma unroll
            for (int i2 = e; i2 < 4; i2 += 2)
              if (x[mt][i2] != -INFINITY) x[mt][i2] = S[t][mt][i2] + ((mt == 0 ? lv.x : lv.y) - now);
        }
      }
    }
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
      for (int e = 0; e < 4; ++e) x[mt][e] = ex2(x[mt][e]);
      const float inv = mt == 0 ? iv.x : iv.y;
      l[t][0] = fmaf(x[mt][0] + x[mt][2], inv, l[t][0]);
      l[t][1] = fmaf(x[mt][1] + x[mt][3], inv, l[t][1]);
      const __half2 p0 = __floats2half2_rn(x[mt][0], x[mt][1]), p1 = __floats2half2_rn(x[mt][2], x[mt][3]);
      P[t][mt] = make_uint2(transpose8(*reinterpret_cast<const uint32_t*>(&p0)),
                            transpose8(*reinterpret_cast<const uint32_t*>(&p1)));
    }
  }
}

template <int kKind, int N, bool kSums>
__global__ void __launch_bounds__(kThreads, blocks_per_sm(N))
kv8_attention_kernel(const __grid_constant__ CUtensorMap map, const Params p) {
  extern __shared__ __align__(1024) uint8_t raw[];
  Smem<N>& sh = *reinterpret_cast<Smem<N>*>(raw);
  constexpr int kRows = 8 * N;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;

  if (mes::smem_u32(raw) & 1023) {      // the swizzle goes by the address
    if (tid == 0) atomicCAS(&g_err_kv8_attention, 0, MES_ERR_ALIGN);
    return;
  }
  if (tid == 0) {
    sh.abort = 0;
    for (int w = 0; w < kWarps; ++w)
      for (int s = 0; s < kStages; ++s) mes::mbar_init(&sh.full[w][s], 1);
    mes::fence_barrier_init();
    mes::tma_prefetch_desc(&map);
  }
  // The join may be launched as soon as every block of this grid runs (it waits for their end).
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  Line<kRows> line{p, sh.prefix};
  if (!line.set_up(sh.warp_sum)) return;
  const int first = line.first, end = line.end;

  // The warp's tiles: tile `warp` of unit first + i is its i-th.  Lane j holds tile 32 i + j.
  Tile t_tile;
  float2 t_lv, t_iv;
  auto copy = [&](int i) {       // the whole warp: tile i into stage i % kStages
    if (first + i >= end) return;
    if ((i & 31) == 0) {
      if (i > 0) t_tile = line.tile(first + i + lane, warp);
      line.resolve(t_tile);
    }
    if (lane == (i & 31) && t_tile.halves > 0)
      load_tile(p, map, t_tile, sh.ring[warp][i % kStages], &sh.full[warp][i % kStages]);
  };
  auto factors = [&](int i) {    // and what goes with it: apart, since the scales arrive later
    if (first + i >= end) return;
    if ((i & 31) == 0) {
      const float2 x = v_factors(t_tile.vs.x), y = v_factors(t_tile.vs.y);
      t_lv = make_float2(x.x, y.x);
      t_iv = make_float2(x.y, y.y);
    }
    if (lane == (i & 31)) {
      sh.sc[warp][i % kStages][0] = t_tile.ks;
      sh.sc[warp][i % kStages][1] = t_lv;
      sh.sc[warp][i % kStages][2] = t_iv;
    }
  };
  // Copies the rows of a segment in, while the one before is worked on.
  auto q_ahead = [&](const Segment& g) {
    for (int e = tid; e < kRows * 8; e += kThreads)
      if ((e >> 3) < g.rows) {
        uint4* dst = sh.raw[e >> 3] + 2 * (e & 7);
        const __nv_bfloat16* src = line.q_source(g, e);
        copy16_async(dst, src);
        copy16_async(dst + 1, src + 8);
      }
  };
  // What is loaded arrives while the next is worked out: pages, query rows, tiles, scales.
  t_tile = line.tile(first + lane, warp);
  Segment seg = line.segment(first);
  q_ahead(seg);
  for (int i = 0; i < kStages; ++i) copy(i);

  uint32_t phase = 0;           // bit s: parity of stage s's next load
  bool ok = true;
  for (int u = first; u < end;) {
    const Seq s = seg.s;
    const int h = seg.h, row_base = seg.row_base, rows = seg.rows, item0 = seg.item0, units = seg.units, stop = seg.stop;
    const int unit0 = u - item0, start = s.len - s.n;
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();            // the previous segment's readers of q / o are done
    for (int e = tid; e < kRows * 8; e += kThreads) {
      const int r = e >> 3, part = e & 7;
      uint4 v[2] = {};
      if (r < rows) {
        v[0] = sh.raw[r][2 * part];
        v[1] = sh.raw[r][2 * part + 1];
      }
      uint2 frag[4];
      const float qs = q_fragments<kKind>(v, r < rows, p.scale, frag);
      if (part == 0) {
        sh.qscale[r] = qs;
        sh.last[r] = r < rows ? start + (row_base + r) / p.G : 0x7fffffff;
      }
#pragma unroll
      for (int w = 0; w < 4; ++w)
        sh.q[r >> 3][(part >> 2) * 4 + w][(r & 7) * 4 + (part & 3)] = frag[w];
    }
    if (u == first)         // the first tiles' scales have arrived by now
      for (int i = 0; i < kStages; ++i) factors(i);
    __syncthreads();
    if (stop < end) {
      seg = line.segment(stop);
      q_ahead(seg);
    }
    // This lane's rows are 8 t + 2 c + e of tile t.
    float qs[N][2];
    int last[N][2];
    int first_last = 0x7fffffff;      // keys that every row sees
#pragma unroll
    for (int t = 0; t < N; ++t)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        qs[t][e] = sh.qscale[8 * t + 2 * c + e];
        last[t][e] = min(sh.last[8 * t + 2 * c + e], s.len - 1);
        first_last = min(first_last, last[t][e]);
      }
    first_last = __reduce_min_sync(0xffffffffu, first_last);
    int64_t logit_row[N][2];          // where this lane's rows' logits go, with sums
    if (kSums) {
#pragma unroll
      for (int t = 0; t < N; ++t)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int row = 8 * t + 2 * c + e, q = row_base + row, qi = q / p.G;
          logit_row[t][e] = row < rows ? ((int64_t)(s.r0 + qi) * p.Hq + h * p.G + q - qi * p.G) * p.max_ctx : -1;
        }
    }
    uint2 q1[8];
    if (N == 1) {
#pragma unroll
      for (int st = 0; st < 8; ++st) q1[st] = sh.q[0][st][lane];
    }

    float O[N][8][4], m[N][2], l[N][2];
#pragma unroll
    for (int t = 0; t < N; ++t) {
#pragma unroll
      for (int d = 0; d < 8; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e) O[t][d][e] = 0.f;
      m[t][0] = m[t][1] = -INFINITY;
      l[t][0] = l[t][1] = 0.f;
    }
    float base = 0.f;             // log2 of the base
    bool any = false;             // any V that does not count as 0; O is 0 until then
    int plain_len = s.len;        // tiles that end by it and have ordinary scales need nothing else; -1 with another base
    auto move_base = [&](float to) {
      const float d = to - base, alpha = any ? ex2(-d) : 1.f;
#pragma unroll
      for (int t = 0; t < N; ++t) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) O[t][i][e] *= alpha;
        m[t][0] += d;
        m[t][1] += d;
      }
      base = to;
    };

    for (; u < stop; ++u) {
      const int i = u - first, stage = i % kStages;
      const int t0 = (u - item0) * kUnit + warp * kTile;
      if (t0 < s.len) {
        ok = mes::mbar_wait_warp(&sh.full[warp][stage], (phase >> stage) & 1, &sh.abort,
                                 &g_err_kv8_attention, MES_ERR_TIMEOUT) && ok;
        phase ^= 1u << stage;
        const uint8_t* kt = sh.ring[warp][stage];
        const uint8_t* vt = kt + kHalfBytes;
        const float2 ks = sh.sc[warp][stage][0];
        float2 lv = sh.sc[warp][stage][1], iv = sh.sc[warp][stage][2];
        if (t0 + kTile > plain_len || iv.x < 0.f || iv.y < 0.f) {
          const float top = fmaxf(lv.x, lv.y);
          if (top > -INFINITY) {
            const float to = fabsf(top) <= kOrdinary ? 0.f : floorf(top);
            if (any ? top > (base == 0.f ? kOrdinary : base + kBaseStep) : to != base) move_base(to);
            any = true;
            plain_len = base == 0.f ? s.len : -1;
          }
          // V slots past the end hold anything, NaN codes too, and 0 * NaN is NaN; codes of no scale
          // count as 0.  Lane = slot.
          const bool none0 = lv.x < base - kBaseRange, none1 = lv.y < base - kBaseRange;
          if (t0 + lane >= s.len || (lane < 16 ? none0 : none1)) {
            uint4* row = reinterpret_cast<uint4*>(const_cast<uint8_t*>(vt) + lane * kv8::kD);
#pragma unroll
            for (int j = 0; j < 8; ++j) row[j] = make_uint4(0, 0, 0, 0);
          }
          mes::fence_proxy_async_smem();      // before the stage is loaded again
          __syncwarp();
          const float none = base == 0.f ? -kOrdinary : base;
          lv = make_float2(none0 ? none : lv.x, none1 ? none : lv.y);
          iv = make_float2(ex2(base - lv.x), ex2(base - lv.y));
        } else {
          any = true;
        }
        // ---- S^T = K Q^T: keys 16 mt + key_of(g) and 8 more by rows 2 c and 2 c + 1 ----
        float S[N][2][4];
#pragma unroll
        for (int t = 0; t < N; ++t)
#pragma unroll
          for (int mt = 0; mt < 2; ++mt)
#pragma unroll
            for (int e = 0; e < 4; ++e) S[t][mt][e] = 0.f;
        const int kg = key_of(g);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          uint4 kw[4];
#pragma unroll
          for (int nt = 0; nt < 4; ++nt)
            kw[nt] = *reinterpret_cast<const uint4*>(kt + (8 * nt + kg) * kv8::kD + (((c + 4 * half) ^ kg) << 4));
#pragma unroll
          for (int st = 0; st < 4; ++st) {
            uint2 b[N];
#pragma unroll
            for (int t = 0; t < N; ++t) b[t] = N == 1 ? q1[4 * half + st] : sh.q[t][4 * half + st][lane];
#pragma unroll
            for (int mt = 0; mt < 2; ++mt) {
              uint32_t a0, a1, a2, a3;
              convert<kKind>(word_of(kw[2 * mt], st), a0, a2);
              convert<kKind>(word_of(kw[2 * mt + 1], st), a1, a3);
#pragma unroll
              for (int t = 0; t < N; ++t) mma_f16(S[t][mt], a0, a1, a2, a3, b[t].x, b[t].y);
            }
          }
        }
        uint2 P[N][2];      // B fragments of the two 16-key steps
        weights<N, kSums>(p, S, O, m, l, P, qs, last, logit_row, ks, lv, iv, t0, s.len, t0 + kTile - 1 > first_last, kg);
        // ---- O^T += V^T P^T: tile d of O is values 16 g + 2 d and one more of the head ----
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          uint4 v[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int key = 8 * (2 * j + (e >> 1)) + key_of(2 * c + (e & 1));
            v[e] = *reinterpret_cast<const uint4*>(vt + key * kv8::kD + ((g ^ (key & 7)) << 4));
          }
#pragma unroll
          for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int half = 0; half < 2; ++half) {    // values 2 half and 2 half + 1 of the four
              // Bytes of two keys side by side as `convert` pairs them.
              constexpr uint32_t kSel[2][2] = {{0x5410, 0x7632}, {0x5140, 0x7362}};
              const uint32_t x = __byte_perm(word_of(v[0], q), word_of(v[1], q), kSel[kKind][half]);
              const uint32_t y = __byte_perm(word_of(v[2], q), word_of(v[3], q), kSel[kKind][half]);
              uint32_t a0, a1, a2, a3;
              convert<kKind>(x, a0, a1);
              convert<kKind>(y, a2, a3);
#pragma unroll
              for (int t = 0; t < N; ++t) mma_f16(O[t][2 * q + half], a0, a1, a2, a3, P[t][j].x, P[t][j].y);
            }
        }
      }
      __syncwarp();               // the stage has been read by every lane
      copy(i + kStages);
      factors(i + kStages);
    }

    // ---- join the four warps: they trade halves of their sums two apart, then halves of those with
    // their neighbours, so that warp w ends with the w-th quarter of all ----
#pragma unroll
    for (int t = 0; t < N; ++t)
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) l[t][e] += __shfl_xor_sync(0xffffffffu, l[t][e], o);
    // Element i: tile i / 8, values 2 (i % 8) and one more of its 16.
    float4 part[4 * N];
    float mine[N][2], theirs[N][2];
    auto give_rows = [&] {
      if (g == 0)
#pragma unroll
        for (int t = 0; t < N; ++t)
#pragma unroll
          for (int e = 0; e < 2; ++e) sh.ml[warp][8 * t + 2 * c + e] = make_float2(m[t][e], l[t][e]);
    };
    auto take_rows = [&](int from) {     // joins another warp's references and sums
#pragma unroll
      for (int t = 0; t < N; ++t)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float2 ml = sh.ml[from][8 * t + 2 * c + e];
          const float now = fmaxf(m[t][e], ml.x);
          mine[t][e] = m[t][e] == -INFINITY ? 0.f : ex2(m[t][e] - now);
          theirs[t][e] = ml.x == -INFINITY ? 0.f : ex2(ml.x - now);
          m[t][e] = now;
          l[t][e] = l[t][e] * mine[t][e] + ml.y * theirs[t][e];
        }
    };
    auto join = [&](float4& a, const float4& x, const float (&fm)[2], const float (&ft)[2]) {
      a.x = a.x * fm[0] + x.x * ft[0];
      a.y = a.y * fm[1] + x.y * ft[1];
      a.z = a.z * fm[0] + x.z * ft[0];
      a.w = a.w * fm[1] + x.w * ft[1];
    };
    const bool upper = warp >= 2, odd = warp & 1;
    if (lane == 0) sh.base[warp] = any ? base : -INFINITY;
    __syncthreads();
    const float most = fmaxf(fmaxf(sh.base[0], sh.base[1]), fmaxf(sh.base[2], sh.base[3]));
    if (most != -INFINITY && most != base) move_base(most);      // one base for the four
#pragma unroll
    for (int i = 0; i < 4 * N; ++i) {
      const int j = i + 4 * N;
      const float4 a = make_float4(O[i / 8][i % 8][0], O[i / 8][i % 8][1], O[i / 8][i % 8][2], O[i / 8][i % 8][3]);
      const float4 z = make_float4(O[j / 8][j % 8][0], O[j / 8][j % 8][1], O[j / 8][j % 8][2], O[j / 8][j % 8][3]);
      part[i] = upper ? z : a;
      sh.o[warp][i][lane] = upper ? a : z;
    }
    give_rows();
    __syncthreads();
    take_rows(warp ^ 2);
#pragma unroll
    for (int i = 0; i < 4 * N; ++i) {
      const int t0 = i / 8, t1 = (i + 4 * N) / 8;
      const float fm[2] = {upper ? mine[t1][0] : mine[t0][0], upper ? mine[t1][1] : mine[t0][1]};
      const float ft[2] = {upper ? theirs[t1][0] : theirs[t0][0], upper ? theirs[t1][1] : theirs[t0][1]};
      join(part[i], sh.o[warp ^ 2][i][lane], fm, ft);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2 * N; ++i) {
      sh.o[warp][i][lane] = odd ? part[i] : part[i + 2 * N];
      part[i] = odd ? part[i + 2 * N] : part[i];
    }
    give_rows();
    __syncthreads();
    take_rows(warp ^ 1);
    // This warp's tile and the place of its 4 N values in a lane's 16.
    const int tile = N == 1 ? 0 : warp >> 1, at16 = N == 1 ? 4 * warp : 8 * (warp & 1);
    float fm[2] = {0.f, 0.f}, ft[2] = {0.f, 0.f}, row_m[2] = {0.f, 0.f}, row_l[2] = {0.f, 0.f};
#pragma unroll
    for (int t = 0; t < N; ++t)
      if (t == tile)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          fm[e] = mine[t][e];
          ft[e] = theirs[t][e];
          row_m[e] = m[t][e];
          row_l[e] = l[t][e];
        }
#pragma unroll
    for (int i = 0; i < 2 * N; ++i) join(part[i], sh.o[warp ^ 1][i][lane], fm, ft);

    const bool whole = unit0 == 0 && stop == item0 + units;
    const int slot = 2 * blockIdx.x + (item0 + unit0 == first ? 0 : 1);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int row = 8 * tile + 2 * c + e;
      if (row >= rows) continue;
      if (whole) {
        const int q = row_base + row, qi = q / p.G;
        const int64_t at = (int64_t)(s.r0 + qi) * p.Hq + h * p.G + q - qi * p.G;
        const float half = ex2(0.5f * base);      // 2^base in two steps, either of which may be
        const float inv = half * (row_l[e] > 0.f ? 1.f / row_l[e] : row_l[e] == 0.f ? 0.f : row_l[e]);     // NaN stays NaN
        uint32_t w[2 * N];
#pragma unroll
        for (int i = 0; i < 2 * N; ++i)
          w[i] = mes::pack_bf16x2((e ? part[i].y : part[i].x) * inv * half, (e ? part[i].w : part[i].z) * inv * half);
        uint2* dst = reinterpret_cast<uint2*>(p.out + at * kv8::kD + 16 * g + at16);
#pragma unroll
        for (int i = 0; i < N; ++i) dst[i] = make_uint2(w[2 * i], w[2 * i + 1]);
        if (kSums && g == 0 && at16 == 0) p.lse[at] = row_m[e] - base + log2f(row_l[e]);
      } else {
        float4* dst = reinterpret_cast<float4*>(p.part_o + ((int64_t)slot * kRows + row) * kv8::kD + 16 * g + at16);
#pragma unroll
        for (int i = 0; i < N; ++i)
          dst[i] = e ? make_float4(part[2 * i].y, part[2 * i].w, part[2 * i + 1].y, part[2 * i + 1].w)
                     : make_float4(part[2 * i].x, part[2 * i].z, part[2 * i + 1].x, part[2 * i + 1].z);
        if (g == 0 && at16 == 0)
          p.part_ml[(int64_t)slot * kRows + row] =
              make_float4(most == -INFINITY ? most : row_m[e], row_m[e] - base, row_l[e], 0.f);
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

// ---- join the partial results of items cut between blocks: W warps for each (token, query head) ----
template <int N, int W, bool kSums>
__global__ void __launch_bounds__(kThreads)
kv8_join_kernel(const Params p, int grid) {
  constexpr int kRows = 8 * N;
  __shared__ float4 part[kWarps][32];
  __shared__ float3 part_ml[kWarps];
  if (kSums) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  // Every block waits for the attention kernel's end before it ends itself, whether it has work or
  // not: what follows this kernel may rely on that one.
  auto wait = [] { asm volatile("griddepcontrol.wait;" ::: "memory"); };
  const int64_t at = blockIdx.x * (int64_t)(kWarps / W) + warp / W;
  if (at >= (int64_t)p.T * p.Hq) return wait();
  const int token = (int)(at / p.Hq), head = (int)(at - (int64_t)token * p.Hq), h = head / p.G;
  // The token's sequence and what is before it and in all, from the lengths alone: this part runs
  // while the attention kernel does.
  Seq s = {0, 0, 0};
  Count total = {0, 0}, before = {0, 0};
  for (int b0 = 0; b0 < p.B; b0 += 32) {
    Seq x = {0, 0, 0};
    if (b0 + lane < p.B) x = sequence(p, b0 + lane);
    const Count mine = count_of<kRows>(p, x);
    const bool is_before = x.r0 + x.n <= token;
    total.units += __reduce_add_sync(0xffffffffu, mine.units);
    total.items += __reduce_add_sync(0xffffffffu, mine.items);
    before.units += __reduce_add_sync(0xffffffffu, is_before ? mine.units : 0);
    before.items += __reduce_add_sync(0xffffffffu, is_before ? mine.items : 0);
    const uint32_t found = __ballot_sync(0xffffffffu, x.n > 0 && token >= x.r0 && token < x.r0 + x.n);
    if (found) {
      const int src = __ffs(found) - 1;
      s.r0 = __shfl_sync(0xffffffffu, x.r0, src);
      s.n = __shfl_sync(0xffffffffu, x.n, src);
      s.len = __shfl_sync(0xffffffffu, x.len, src);
    }
  }
  if (s.n <= 0) return wait();
  const int cost = cost_of<kRows>(p, total.units, grid), all = total.with(cost), blocks = min(grid, all);
  const int row = (token - s.r0) * p.G + head - h * p.G, tile = row / kRows;
  const int units = units_of(p, s.len), item = h * row_tiles<kRows>(s.n, p.G) + tile;
  // The item begins at u_item of the line, its units are [u0, u1).
  const int u_item = before.with(cost) + item * (units + cost), u0 = u_item + cost, u1 = u0 + units;
  // The blocks whose shares meet [u0, u1).
  const Shares shares(all, blocks);
  const float each = (float)blocks / (float)all;             // near enough to begin with
  int from = min((int)(u0 * each), blocks - 1);
  while (from + 1 < blocks && shares.at(from + 1) <= u0) ++from;
  while (from > 0 && shares.at(from) > u0) --from;
  if (shares.at(from + 1) >= u1) return wait();              // not cut
  const int to = [&] {                                     // one past the last of them
    int i = min((int)((u1 - 1) * each), blocks - 1);
    while (i + 1 < blocks && shares.at(i + 1) < u1) ++i;
    while (shares.at(i) >= u1) --i;
    return i + 1;
  }();
  const int local = row - tile * kRows;
  const bool cut = shares.at(from) < u_item;
  // Only the item's first block can have it as its second segment: where it has units before it.
  auto slot = [&](int i) { return ((int64_t)2 * i + (i == from && cut ? 1 : 0)) * kRows + local; };
  wait();                                                  // the partial results are there
  // Each of the W warps takes every W-th partial result; its loads do not wait for one another.  Outputs
  // go by the reference `mx`, sums by `ms`: they differ by the blocks' bases.
  float mx = -INFINITY, ms = -INFINITY, sum = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  auto factor = [](float from, float to) { return from == -INFINITY ? 0.f : ex2(from - to); };
  for (int i0 = from + warp % W; i0 < to; i0 += 8 * W) {
    float4 ml[8], x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      ml[j] = make_float4(-INFINITY, -INFINITY, 0.f, 0.f);
      x[j] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (i0 + j * W < to) {
        ml[j] = p.part_ml[slot(i0 + j * W)];
        x[j] = *reinterpret_cast<const float4*>(p.part_o + slot(i0 + j * W) * kv8::kD + 4 * lane);
      }
    }
    float now = mx, now_s = ms;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      now = fmaxf(now, ml[j].x);
      now_s = fmaxf(now_s, ml[j].y);
    }
    const float keep = factor(mx, now);
    sum *= factor(ms, now_s);
    o = make_float4(o.x * keep, o.y * keep, o.z * keep, o.w * keep);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float f = factor(ml[j].x, now);
      sum += factor(ml[j].y, now_s) * ml[j].z;
      o.x += f * x[j].x;
      o.y += f * x[j].y;
      o.z += f * x[j].z;
      o.w += f * x[j].w;
    }
    mx = now;
    ms = now_s;
  }
  if (W > 1) {
    part[warp][lane] = o;
    if (lane == 0) part_ml[warp] = make_float3(mx, ms, sum);
    __syncthreads();                // W == kWarps: the block's warps have all come here
    if (warp != 0) return;
    mx = ms = -INFINITY;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      mx = fmaxf(mx, part_ml[w].x);
      ms = fmaxf(ms, part_ml[w].y);
    }
    sum = 0.f;
    o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float3 ml = part_ml[w];
      const float4 x = part[w][lane];
      const float f = factor(ml.x, mx);
      sum += factor(ml.y, ms) * ml.z;
      o.x += f * x.x;
      o.y += f * x.y;
      o.z += f * x.z;
      o.w += f * x.w;
    }
  }
  const float half = mx == -INFINITY ? 1.f : ex2(0.5f * (mx - ms));      // 2^base in two steps; no reference: o is 0
  const float inv = half * (sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum);
  *reinterpret_cast<uint2*>(p.out + at * kv8::kD + 4 * lane) =
      make_uint2(mes::pack_bf16x2(o.x * inv * half, o.y * inv * half), mes::pack_bf16x2(o.z * inv * half, o.w * inv * half));
  if (kSums && lane == 0) p.lse[at] = ms + log2f(sum);
}

// ---- sums[t] += sum over the rows of a kv head of exp2(logit - lse): a thread for four keys, which
// are in one page, in the order of the rows ----
__global__ void __launch_bounds__(256)
kv8_sums_kernel(const Params p, float* sums) {
  const int64_t b = blockIdx.y / p.Hkv;
  const int h = (int)(blockIdx.y - b * p.Hkv);
  const Seq s = sequence(p, (int)b);
  const int t = 4 * (blockIdx.x * 256 + threadIdx.x);
  const bool any = t < s.len && s.n > 0;
  // What no kernel before this one writes is read while they run.
  const int64_t page = any ? p.table[b * p.width + (t >> p.page_shift)] : -1;
  const bool valid = page >= 0 && page < p.num_pages;        // else recorded by the attention kernel
  float* at = sums + (valid ? (page * p.Hkv + h) * p.P + (t & (p.P - 1)) : 0);
  float old[4], add[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int j = 0; j < 4; ++j) old[j] = valid && t + j < s.len ? at[j] : 0.f;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (!valid) return;
  const float* logits = p.logits + ((int64_t)s.r0 * p.Hq + h * p.G) * p.max_ctx + t;
  const float* lse = p.lse + (int64_t)s.r0 * p.Hq + h * p.G;
  for (int i = 0; i < s.n; ++i, logits += p.Hq * p.max_ctx, lse += p.Hq) {
    for (int q0 = 0; q0 < p.G; q0 += 4) {
      float4 x[4];
      float norm[4];
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (q0 + q < p.G) {
          x[q] = *reinterpret_cast<const float4*>(logits + (q0 + q) * p.max_ctx);
          norm[q] = lse[q0 + q];
        }
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (q0 + q < p.G) {
          const float v[4] = {x[q].x, x[q].y, x[q].z, x[q].w};
#pragma unroll
          for (int j = 0; j < 4; ++j) add[j] += v[j] == -INFINITY ? 0.f : ex2(v[j] - norm[q]);
        }
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (t + j < s.len) at[j] = old[j] + add[j];
}

// Row tiles of 8 or 16 rows: 16 sequences of 8192 tokens and 8 rows take 33.2 us in tiles of 8 and 34.6 in
// tiles of 16.  Tiles of 32 share a converted key among more products, but their registers spill and leave
// less room for loads in flight: 30 rows after 2048 tokens 17.5 instead of 14.5 us, 138 rows 34.1 instead of 29.8.
int row_factor(int64_t max_new, int G) { return max_new * G <= 8 ? 1 : 2; }
int max_blocks(int N) { return mes_host::sm_count() * blocks_per_sm(N); }

constexpr int64_t up256(int64_t x) { return (x + 255) / 256 * 256; }
struct Layout {
  int64_t part_o, part_ml, lse, logits, bytes;
};
Layout layout(int64_t T, int Hq, int N, int64_t max_ctx) {
  Layout w;
  const int64_t slots = 2ll * max_blocks(N) * 8 * N;
  w.part_o = 0;
  w.part_ml = w.part_o + slots * kv8::kD * 4;
  w.lse = up256(w.part_ml + slots * 16);
  w.logits = up256(w.lse + (max_ctx > 0 ? 4 * T * Hq : 0));
  w.bytes = w.logits + 4 * T * Hq * max_ctx;
  return w;
}
bool valid_sizes(int64_t T, int64_t B, int Hq, int Hkv, int64_t max_new, int64_t max_ctx) {
  return T >= 0 && B >= 0 && B <= kMaxSeqs && Hkv > 0 && Hkv <= 1024 && Hq > 0 && Hq % Hkv == 0 && Hq <= 8192 &&
         max_new >= 0 && max_new <= T && T <= 0x7fffffffll / Hq && max_ctx >= 0 && max_ctx <= 0x7fffffffll &&
         T * Hq <= (1ll << 58) / (max_ctx + 1);
}

template <int kKind, int N, bool kSums>
int launch(const CUtensorMap& map, const Params& p, float* sums, void* stream) {
  auto kernel = kv8_attention_kernel<kKind, N, kSums>;
  static std::atomic<uint64_t> configured{0};
  int st = mes_host::once_per_device(configured, [&] {
    return mes_host::from_cuda(
        cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(Smem<N>)));
  });
  if (st != MES_OK) return st;
  static_assert((sizeof(Smem<N>) + 1024) * blocks_per_sm(N) <= 233472, "1 KB of a block is the system's");
  const int grid = mes_host::persistent_ctas() * blocks_per_sm(N);
  kernel<<<grid, kThreads, sizeof(Smem<N>), (cudaStream_t)stream>>>(map, p);
  if (cudaGetLastError() != cudaSuccess) return MES_ERR_CUDA;
  // The kernels that follow start while the one before them ends (programmatic launch).  What they read
  // ahead of that end is older than the attention kernel, which is launched in plain order.
  cudaLaunchAttribute attr = {};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.stream = (cudaStream_t)stream;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  // Few items leave many partial results each: four warps then share a row's (100000 tokens and a query, 43.4
  // instead of 50.4 us).  More items than that leave one block of the join little to do.
  const int64_t items = (int64_t)p.Hkv * max(p.B, (p.T * p.G + 8 * N - 1) / (8 * N));
  const bool wide = items * 8 <= grid;
  const int per_block = wide ? 1 : kWarps;
  cfg.gridDim = dim3((unsigned)(((int64_t)p.T * p.Hq + per_block - 1) / per_block));
  cfg.blockDim = dim3(kThreads);
  if (p.whole == 0 && cudaLaunchKernelEx(&cfg, wide ? kv8_join_kernel<N, kWarps, kSums> : kv8_join_kernel<N, 1, kSums>, p, grid) != cudaSuccess)
    return MES_ERR_CUDA;
  if (kSums) {
    cfg.gridDim = dim3((unsigned)((p.max_ctx + 1023) / 1024), (unsigned)(p.B * p.Hkv));
    cfg.blockDim = dim3(256);
    if (cudaLaunchKernelEx(&cfg, kv8_sums_kernel, p, sums) != cudaSuccess) return MES_ERR_CUDA;
  }
  return MES_OK;
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
  return layout(T, Hq, row_factor(max_new, Hq / Hkv), max_context).bytes;
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
  if (!q || !codes || !scales || !block_table || !cu_new || !context_lens || !out) return MES_ERR_INVALID;
  if (!kv8::aligned(q, 16) || !kv8::aligned(codes, 16) || !kv8::aligned(scales, 4) || !kv8::aligned(sums, 4) ||
      !kv8::aligned(block_table, 4) || !kv8::aligned(cu_new, 4) || !kv8::aligned(context_lens, 4) ||
      !kv8::aligned(out, 16) || !kv8::aligned(workspace, 256))
    return MES_ERR_ALIGN;
  const int G = Hq / Hkv, N = row_factor(max_new, G);
  const Layout w = layout(T, Hq, N, max_ctx);
  // Whole items without sums leave nothing to keep.
  const int64_t most = (table_width * page_size + kUnit - 1) / kUnit;
  const int whole = most <= kWholeUnits ? (int)most : 0;
  if ((whole == 0 || sums) && (!workspace || workspace_bytes < w.bytes)) return MES_ERR_INVALID;
  // Places of the line are counted in 32 bits.
  const int64_t tiles = (max_new * G + 8 * N - 1) / (8 * N);
  if (((table_width * page_size + kUnit - 1) / kUnit + kSegmentCost) * Hkv > 0x7fffffffll / (B * tiles)) return MES_ERR_INVALID;
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
  p.max_new = (int)max_new;
  p.Hq = Hq;
  p.Hkv = Hkv;
  p.G = G;
  p.P = page_size;
  p.page_shift = __builtin_ctz((unsigned)page_size);
  p.num_pages = num_pages;
  p.scale = scale;
  p.out = (__nv_bfloat16*)out;
  p.part_o = (float*)(ws + w.part_o);
  p.part_ml = (float4*)(ws + w.part_ml);
  p.lse = sums ? (float*)(ws + w.lse) : nullptr;
  p.logits = sums ? (float*)(ws + w.logits) : nullptr;
  p.max_ctx = max_ctx;
  p.whole = whole;
  auto go = [&](auto n) {
    constexpr int kN = decltype(n)::value;
    if (dtype == kv8::kInt8)
      return sums ? launch<kv8::kInt8, kN, true>(map, p, sums, stream) : launch<kv8::kInt8, kN, false>(map, p, sums, stream);
    return sums ? launch<kv8::kE4m3, kN, true>(map, p, sums, stream) : launch<kv8::kE4m3, kN, false>(map, p, sums, stream);
  };
  return N == 1 ? go(std::integral_constant<int, 1>()) : go(std::integral_constant<int, 2>());
}
