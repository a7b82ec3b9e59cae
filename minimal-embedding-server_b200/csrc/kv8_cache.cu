// Writing, reading back and compacting the 8-bit paged KV cache (layout: kv8.cuh).  All three
// move bytes: their bound is what they read and write.
#include "kv8.cuh"

namespace {

__device__ int g_err_kv8_cache = 0;

__device__ __forceinline__ void record(int code) { atomicCAS(&g_err_kv8_cache, 0, code); }

__device__ __forceinline__ void unpack8(const uint4& v, float (&f)[8]) {
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 t = __bfloat1622float2(h[i]);
    f[2 * i] = t.x;
    f[2 * i + 1] = t.y;
  }
}

// Eight values -> codes, as `encode(f / scale)` gives them.  The quotients are correctly rounded
// (Markstein's theorem: with y = RN(1 / b), q within one unit of a / b and r = RN(a - b q), RN(q + r y)
// is a / b rounded, where nothing underflows; a y may be two units off, a first step brings it
// within one), which takes five products instead of a division: ties are common among 16-bit
// values (half of a run's largest value is one), so near is not enough.  `direct`: the scale or
// the values are outside the range in which that holds.
struct Divisor {
  float scale, inv;
  bool direct;
};
__device__ __forceinline__ Divisor divisor(float scale, bool direct) {
  return {scale, 1.f / scale, direct || !(scale >= 8.6736174e-19f && scale <= 1.2676506e30f)};   // 2^-60, 2^100
}
template <int kKind>
__device__ __forceinline__ uint2 quantise8(const float (&f)[8], const Divisor& by) {
  uint32_t o[2] = {0, 0};
  if (by.direct) {
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e >> 2] |= kv8::encode<kKind>(f[e] / by.scale) << (8 * (e & 3));
    return make_uint2(o[0], o[1]);
  }
  float q[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    q[e] = f[e] * by.inv;
    q[e] = fmaf(fmaf(-q[e], by.scale, f[e]), by.inv, q[e]);
    q[e] = fmaf(fmaf(-q[e], by.scale, f[e]), by.inv, q[e]);
    if (kKind == kv8::kE4m3) q[e] = copysignf(q[e], f[e]);      // the steps turn -0 into 0
  }
  // No quotient passes the largest code by more than its rounding.
#pragma unroll
  for (int i = 0; i < 2; ++i)
    if (kKind == kv8::kInt8) {
      uint32_t t[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) t[e] = __float_as_uint(q[4 * i + e] + 12582912.f);    // 1.5 2^23: rounds to an integer
      o[i] = __byte_perm(__byte_perm(t[0], t[1], 0x0040), __byte_perm(t[2], t[3], 0x0040), 0x5410);
    } else {
      o[i] = __nv_cvt_float2_to_fp8x2(make_float2(q[4 * i], q[4 * i + 1]), __NV_SATFINITE, __NV_E4M3) |
             (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(q[4 * i + 2], q[4 * i + 3]), __NV_SATFINITE, __NV_E4M3) << 16;
    }
  return make_uint2(o[0], o[1]);
}

// Eight codes of scale `was` -> codes of by.scale, as quantise8 gives them for fl(code * was).  A code
// times the ratio, a little less and a little more than it, encloses the quotient, and rounding is
// monotone: where both give one code, that is it.  (Ties are rare here, the ratio being arbitrary.)
template <int kKind>
__device__ __forceinline__ uint2 requantise8(uint2 c, float was, const Divisor& by) {
  float f[8];
  kv8::decode4<kKind>(c.x, f);
  kv8::decode4<kKind>(c.y, f + 4);
  const float ratio = was * by.inv, lo = ratio * (1.f - 4.76837158e-7f), hi = ratio * (1.f + 4.76837158e-7f);
  uint32_t o[2], differ = by.direct || !(was >= 8.6736174e-19f);
  if (kKind == kv8::kInt8) {
    uint32_t t[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      t[e] = __float_as_uint(fmaf(f[e], lo, 12582912.f));
      differ |= t[e] ^ __float_as_uint(fmaf(f[e], hi, 12582912.f));
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
      o[i] = __byte_perm(__byte_perm(t[4 * i], t[4 * i + 1], 0x0040), __byte_perm(t[4 * i + 2], t[4 * i + 3], 0x0040), 0x5410);
  } else {
    auto pack = [&](int i, float r) {
      return __nv_cvt_float2_to_fp8x2(make_float2(f[4 * i] * r, f[4 * i + 1] * r), __NV_SATFINITE, __NV_E4M3) |
             (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(f[4 * i + 2] * r, f[4 * i + 3] * r), __NV_SATFINITE, __NV_E4M3) << 16;
    };
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      o[i] = pack(i, lo);
      differ |= o[i] ^ pack(i, hi);
    }
  }
  if (differ == 0) return make_uint2(o[0], o[1]);
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] *= was;
  return quantise8<kKind>(f, by);
}

// Eight values -> codes in the ordinary case (not by.direct); false where `quantise8` has to decide.
// int8: as there.  e4m3, whose ties are rare (448 = 7 * 2^6: a value has to be some sevenths of the
// scale's largest): products with a little less and a little more than 1 / scale enclose the quotient.
template <int kKind>
__device__ __forceinline__ bool quantise8_fast(const float (&f)[8], const Divisor& by, uint2& o) {
  if (kKind == kv8::kInt8) {
    o = quantise8<kKind>(f, {by.scale, by.inv, false});
    return true;
  }
  auto pack = [&](int i, float r) {
    return __nv_cvt_float2_to_fp8x2(make_float2(f[i] * r, f[i + 1] * r), __NV_SATFINITE, __NV_E4M3) |
           (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(f[i + 2] * r, f[i + 3] * r), __NV_SATFINITE, __NV_E4M3) << 16;
  };
  const float lo = by.inv * (1.f - 4.76837158e-7f), hi = by.inv * (1.f + 4.76837158e-7f);
  o = make_uint2(pack(0, lo), pack(4, lo));
  return ((o.x ^ pack(0, hi)) | (o.y ^ pack(4, hi))) == 0;
}

// Rows of one run handled by a warp, and the block shape that follows: a run of P tokens takes
// P / kRows warps, and a block holds at least four warps, so small pages share a block.  With 8 rows
// 20 x 1000 tokens take 53 instead of 49 us to write and read back: what a warp does once counts twice.
constexpr int kRows = 16;
template <int P>
struct Shape {
  static constexpr int kRunWarps = P / kRows;
  static constexpr int kRuns = kRunWarps < 4 ? 4 / kRunWarps : 1;   // runs of a block
  static constexpr int kThreads = 32 * kRunWarps * kRuns;
};

// Largest value over the warps of a run; every thread of the block calls it.
template <int kRunWarps>
__device__ __forceinline__ float run_max(float v, float* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  if (kRunWarps == 1) return v;
  const int warp = threadIdx.x >> 5, first = warp / kRunWarps * kRunWarps;
  if ((threadIdx.x & 31) == 0) red[warp] = v;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kRunWarps; ++i) v = fmaxf(v, red[first + i]);
  return v;
}

// ----------------------------------------- append --------------------------------------
// Run (sequence b, touched page j, side, head): s = max(s_old, amax|new| / Q), old tokens of the
// run re-rounded when s grew, new tokens rounded once.  s_old counts only where the run already
// held tokens.  Non-finite inputs do not set the scale: an infinity saturates, NaN becomes 0.
// Each new value is read once and kept in registers between the maximum and the rounding.
// Measured: 20 x 1000 tokens of 8 heads 26.3 us by itself, 28.3 with the read-back between (123 MB, 4.3 to 4.7 TB/s,
// 0.66 to 0.71 of the copy rate, with 73% of the issue slots taken); one token for each of 32 sequences 2.8 us.
template <int kKind, int P>
__global__ void __launch_bounds__(Shape<P>::kThreads)
kv8_append_kernel(const __nv_bfloat16* __restrict__ Kn, int64_t ldk, const __nv_bfloat16* __restrict__ Vn,
                  int64_t ldv, uint8_t* codes, float* scales, float* sums,
                  const int32_t* __restrict__ table, int64_t width, const int32_t* __restrict__ cu,
                  const int32_t* __restrict__ ctx, int64_t T, int max_new, int max_pages, int Hkv,
                  int64_t num_pages) {
  using Run = Shape<P>;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  __shared__ float red[8];
  constexpr float kQ = kv8::code_max<kKind>();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int b = blockIdx.x / max_pages, j = blockIdx.x - b * max_pages;
  const int run = blockIdx.y * Run::kRuns + warp / Run::kRunWarps;
  const int side = run >= Hkv, h = run - side * Hkv;
  const int r0 = cu[b], n = cu[b + 1] - r0, len = ctx[b], start = len - n;
  // A sequence with more new tokens than max_new is not written at all, as the attention skips it.
  const bool sane = r0 >= 0 && n >= 0 && n <= max_new && start >= 0 && r0 + (int64_t)n <= T && (int64_t)len <= width * P;
  const int p = sane ? start / P + j : 0;
  bool ok = run < 2 * Hkv && n > 0 && sane && (int64_t)p * P < len;
  if (!sane && threadIdx.x == 0 && blockIdx.y == 0) record(MES_ERR_INVALID);
  // The page's slots [old, end) are new; this lane has the even or odd rows of the warp's.
  const int old = max(start - p * P, 0), end = ok ? min(len - p * P, P) : 0;
  const int slot0 = warp % Run::kRunWarps * kRows + (lane >> 4), col = (lane & 15) * 8;
  const int64_t ld = side ? ldv : ldk;
  const __nv_bfloat16* src = (side ? Vn : Kn) + (int64_t)(r0 + p * P + slot0 - start) * ld + h * kv8::kD + col;
  uint4 x[kRows / 2];
#pragma unroll
  for (int i = 0; i < kRows / 2; ++i) {
    const int slot = slot0 + 2 * i;
    x[i] = slot >= old && slot < end ? __ldg(reinterpret_cast<const uint4*>(src)) : make_uint4(0, 0, 0, 0);
    src += 2 * ld;
  }
  auto again = [&](int i, float (&f)[8]) {      // row i of them once more, for the paths that few values take
    unpack8(__ldg(reinterpret_cast<const uint4*>(src - (kRows - 2 * i) * ld)), f);
  };
  int64_t page = ok ? table[(int64_t)b * width + p] : 0;
  if (page < 0 || page >= num_pages) {
    ok = false;
    page = 0;
    record(MES_ERR_INVALID);
  }
  const int64_t si = (page * 2 + side) * Hkv + h;
  const float was = ok && old > 0 ? scales[si] : 0.f;
  // |x| in 16 bits orders as integers do; from 0x7f80 on it is no finite number.
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < kRows / 2; ++i)
    top = __vmaxu2(__vmaxu2(top, __vmaxu2(x[i].x & 0x7fff7fffu, x[i].y & 0x7fff7fffu)),
                   __vmaxu2(x[i].z & 0x7fff7fffu, x[i].w & 0x7fff7fffu));
  top = max(top & 0xffffu, top >> 16);
  const bool odd = top >= 0x7f80u;
  float amax = __uint_as_float(top << 16);
  if (odd) {
    amax = 0.f;
#pragma unroll 1
    for (int i = 0; i < kRows / 2; ++i) {
      if (slot0 + 2 * i < old || slot0 + 2 * i >= end) continue;
      float f[8];
      again(i, f);
#pragma unroll
      for (int e = 0; e < 8; ++e) amax = fabsf(f[e]) <= 3.4028235e38f ? fmaxf(amax, fabsf(f[e])) : amax;
    }
  }
  amax = run_max<Run::kRunWarps>(amax, red);
  __syncthreads();                      // every warp of the run has read the old scale
  if (!ok) return;
  const float now = fmaxf(was, amax / kQ);
  const Divisor by = divisor(now > 0.f ? now : 1.f, odd);
  uint8_t* dst = codes + (si * P + slot0) * kv8::kD + col;
  uint32_t rest = 0;                    // rows for quantise8
#pragma unroll
  for (int i = 0; i < kRows / 2; ++i) {
    const int slot = slot0 + 2 * i;
    if (slot >= old && slot < end) {
      float f[8];
      uint2 o;
      unpack8(x[i], f);
      if (by.direct || !quantise8_fast<kKind>(f, by, o))
        rest |= 1u << i;
      else
        *reinterpret_cast<uint2*>(dst + 2 * i * kv8::kD) = o;
    }
  }
  for (; rest; rest &= rest - 1) {
    const int i = __ffs(rest) - 1;
    float f[8];
    again(i, f);
    *reinterpret_cast<uint2*>(dst + 2 * i * kv8::kD) = quantise8<kKind>(f, by);
  }
  if (old > 0 && now > was) {
    for (int slot = slot0; slot < min(old, slot0 + kRows); slot += 2) {
      uint2* at = reinterpret_cast<uint2*>(dst + (slot - slot0) * kv8::kD);
      *at = requantise8<kKind>(*at, was, by);
    }
  }
  if (sums && side == 0 && col == 0)
    for (int slot = slot0; slot < slot0 + kRows; slot += 2)
      if (slot >= old && slot < end) sums[(page * Hkv + h) * P + slot] = 0.f;
  if (lane == 0 && warp % Run::kRunWarps == 0) scales[si] = now;
}

// ------------------------------------------ read ---------------------------------------
// out[i] = code * scale of pages[i], rounded to bf16: a lane turns 8 codes into one 16-byte store, so
// that a warp's stores cover whole lines; a block does a piece of a page, a thread eight times.
// Measured: 20000 tokens of 8 heads 18 us (123 MB, 6.8 TB/s: part of the codes is still in L2).
constexpr int kReadChunks = 8;
template <int kKind>
__global__ void __launch_bounds__(256)
kv8_read_kernel(const uint8_t* __restrict__ codes, const float* __restrict__ scales,
                const int32_t* __restrict__ pages, int page_chunks, int run_shift, int64_t num_pages,
                uint4* __restrict__ out) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int64_t n = blockIdx.x, page = __ldg(pages + n);
  const bool ok = page >= 0 && page < num_pages;
  if (!ok && threadIdx.x == 0) record(MES_ERR_INVALID);
  const int first = blockIdx.y * kReadChunks * 256 + threadIdx.x;
  const uint2* src = reinterpret_cast<const uint2*>(codes) + (ok ? page * page_chunks : 0) + first;
  const float* sc = scales + (ok ? page * (page_chunks >> run_shift) : 0);
  uint4* dst = out + n * page_chunks + first;
  uint2 v[kReadChunks];
  float s[kReadChunks];
#pragma unroll
  for (int i = 0; i < kReadChunks; ++i) {
    const bool in = ok && first + 256 * i < page_chunks;
    v[i] = in ? __ldg(src + 256 * i) : make_uint2(0, 0);
    s[i] = in ? __ldg(sc + ((first + 256 * i) >> run_shift)) : 0.f;
  }
#pragma unroll
  for (int i = 0; i < kReadChunks; ++i) {
    if (first + 256 * i >= page_chunks) return;
    float f[8];
    kv8::decode4<kKind>(v[i].x, f);
    kv8::decode4<kKind>(v[i].y, f + 4);
    dst[256 * i] = make_uint4(mes::pack_bf16x2(f[0] * s[i], f[1] * s[i]), mes::pack_bf16x2(f[2] * s[i], f[3] * s[i]),
                              mes::pack_bf16x2(f[4] * s[i], f[5] * s[i]), mes::pack_bf16x2(f[6] * s[i], f[7] * s[i]));
  }
}

// ------------------------------------------ evict --------------------------------------
// Selection: a cluster for each (sequence, head).  The candidates (all but the last `recent`
// tokens) are cut into one contiguous slice a block, whose sums are turned into ordered integers
// once, in shared memory where they fit.  The k-th largest follows from three histograms of 11,
// 11 and 10 bits, added over the cluster through distributed shared memory; then each warp walks
// its part of the slice in token order, so the kept indices come out sorted and a tie goes to
// the lower index.
// Measured: 8 heads of 100003 tokens 24.5 us, 64 of 4096 10.3 us.  Latency bounds it: lengths, pages and
// sums are loaded one after the other (5 us), and each pass has two barriers of the cluster (5 us).
constexpr int kSelThreads = 1024, kBins = 2048, kSelWarps = kSelThreads / 32;

// Larger float -> larger integer; -0 equals +0 and NaN is lowest.
__device__ __forceinline__ uint32_t order_key(float f) {
  if (!(f == f)) return 0u;
  const uint32_t u = __float_as_uint(f + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

struct SelShared {
  alignas(8) uint32_t hist[kBins];
  uint32_t warp_sum[2][kSelWarps];
  uint32_t digit, above;       // this pass's bin and how many keys lie above it
  alignas(8) uint32_t greater;
  uint32_t equal;              // this block's counts against the threshold
};

__device__ __forceinline__ uint2 ld_dsmem_u32x2(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared::cluster.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr) : "memory");
  return v;
}
__global__ void __launch_bounds__(kSelThreads, 1)
kv8_select_kernel(const float* __restrict__ sums, const int32_t* __restrict__ table, int64_t width,
                  const int32_t* __restrict__ ctx, int Hkv, int page_shift, int64_t num_pages, int keep,
                  int recent, int cap, int ranks, bool vectors, int32_t* __restrict__ kept,
                  int32_t* __restrict__ new_lens) {
  extern __shared__ __align__(16) uint32_t cached[];
  __shared__ SelShared sh;
  // The compaction may be launched as soon as every block of this grid runs (it waits for their end).
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = ranks > 1 ? static_cast<int>(mes::cluster_ctarank()) : 0;
  const int item = blockIdx.x / ranks, b = item / Hkv, h = item - b * Hkv;
  const int64_t room = width << page_shift;
  int len = ctx[b];
  if (len < 0 || len > room) {
    if (tid == 0) record(MES_ERR_INVALID);
    len = 0;
  }
  int32_t* out = kept + (int64_t)item * keep;
  const int left = min(len, keep);
  if (h == 0 && rank == 0 && tid == 0) new_lens[b] = left;
  if (len <= keep) {   // nothing to evict (uniform over the cluster)
    for (int i = rank * kSelThreads + tid; i < keep; i += ranks * kSelThreads) out[i] = i < len ? i : -1;
    return;
  }
  const int n = len - recent;                       // candidates; recent <= keep < len
  const uint32_t k = static_cast<uint32_t>(keep - recent);
  for (int i = rank * kSelThreads + tid; i < recent; i += ranks * kSelThreads) out[k + i] = n + i;
  if (k == 0) return;
  // Slices are multiples of 32 tokens, so four tokens at a multiple of 4 lie in one page; what a
  // last four reads past `count` is memory of its page and is not used.
  const int slice = ((n + ranks - 1) / ranks + 31) / 32 * 32;
  const int lo = min(rank * slice, n), count = min(lo + slice, n) - lo;
  bool bad = false;
  auto page_of = [&](int i) { return table[b * width + ((lo + i) >> page_shift)]; };
  auto place = [&](int i, int64_t page) {
    if (page < 0 || page >= num_pages) {
      bad = true;
      page = 0;
    }
    return sums + ((page * Hkv + h) << page_shift) + ((lo + i) & ((1 << page_shift) - 1));
  };
  const int in_smem = min(count, cap);
  for (int i0 = 4 * tid; i0 < in_smem; i0 += 16 * kSelThreads) {      // four pages, then four loads in flight
    int page[4];
    float4 v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = i0 + 4 * kSelThreads * j;
      page[j] = i < in_smem ? page_of(i) : 0;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = i0 + 4 * kSelThreads * j;
      if (i >= in_smem) continue;
      const float* at = place(i, page[j]);
      v[j] = vectors ? *reinterpret_cast<const float4*>(at) : make_float4(at[0], at[1], at[2], at[3]);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = i0 + 4 * kSelThreads * j;
      if (i < in_smem)
        *reinterpret_cast<uint4*>(cached + i) =
            make_uint4(order_key(v[j].x), order_key(v[j].y), order_key(v[j].z), order_key(v[j].w));
    }
  }
  auto load = [&](int i) { return order_key(*place(i, page_of(i))); };
  auto key = [&](int i) { return i < cap ? cached[i] : load(i); };

  uint32_t prefix = 0, want = k;      // the threshold's high bits; its place among the keys that share them
  const int shifts[3] = {21, 10, 0}, bits[3] = {11, 11, 10};
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = shifts[pass];
    const uint32_t mask = (1u << bits[pass]) - 1, high = pass == 0 ? 0u : ~((1u << shifts[pass - 1]) - 1);
    for (int i = tid; i < kBins; i += kSelThreads) sh.hist[i] = 0;
    __syncthreads();
#pragma unroll 4
    for (int i = tid; i < count; i += kSelThreads) {
      const uint32_t x = key(i);
      if ((x & high) == prefix) atomicAdd(&sh.hist[(x >> shift) & mask], 1u);
    }
    if (ranks > 1) mes::cluster_sync(); else __syncthreads();
    // Bins from the top: thread t owns the pair of bins 2047 - 2t and 2046 - 2t.
    const int top = kBins - 1 - 2 * tid;
    uint32_t hi = 0, lo2 = 0;
    if (ranks > 1) {
      const uint32_t at = mes::smem_u32(&sh.hist[top - 1]);
#pragma unroll
      for (int r = 0; r < 8; ++r)
        if (r < ranks) {
          const uint2 v = ld_dsmem_u32x2(mes::mapa_shared(at, r));
          lo2 += v.x;
          hi += v.y;
        }
    } else {
      hi = sh.hist[top];
      lo2 = sh.hist[top - 1];
    }
    uint32_t x = hi + lo2;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) sh.warp_sum[0][warp] = x;
    __syncthreads();
    // Keys in bins above this thread's.
    const uint32_t before = __reduce_add_sync(0xffffffffu, lane < warp ? sh.warp_sum[0][lane] : 0u) + x - hi - lo2;
    if (before < want && before + hi >= want) {
      sh.digit = top;
      sh.above = before;
    } else if (before + hi < want && before + hi + lo2 >= want) {
      sh.digit = top - 1;
      sh.above = before + hi;
    }
    if (ranks > 1) mes::cluster_sync(); else __syncthreads();   // also: the histograms may be reused
    prefix |= sh.digit << shift;
    want -= sh.above;
  }
  // Keep every key above `prefix` and the first `want` equal to it.
  const int per_warp = (slice / 32 + kSelWarps - 1) / kSelWarps * 32;
  const int w0 = min(warp * per_warp, count), w1 = min(w0 + per_warp, count);
  uint32_t gt = 0, eq = 0;
#pragma unroll 4
  for (int i = w0 + lane; i < w1; i += 32) {
    const uint32_t x = key(i);
    gt += x > prefix;
    eq += x == prefix;
  }
  gt = __reduce_add_sync(0xffffffffu, gt);
  eq = __reduce_add_sync(0xffffffffu, eq);
  if (lane == 0) {
    sh.warp_sum[0][warp] = gt;
    sh.warp_sum[1][warp] = eq;
  }
  __syncthreads();
  if (warp == 0) {
    const uint32_t a = __reduce_add_sync(0xffffffffu, sh.warp_sum[0][lane]);
    const uint32_t e = __reduce_add_sync(0xffffffffu, sh.warp_sum[1][lane]);
    if (lane == 0) {
      sh.greater = a;
      sh.equal = e;
    }
  }
  if (ranks > 1) mes::cluster_sync(); else __syncthreads();
  uint2 others = make_uint2(0, 0);      // lane r: what block r < rank keeps
  if (lane < rank) others = ld_dsmem_u32x2(mes::mapa_shared(mes::smem_u32(&sh.greater), lane));
  uint32_t gt_before = __reduce_add_sync(0xffffffffu, others.x + (lane < warp ? sh.warp_sum[0][lane] : 0u));
  uint32_t eq_before = __reduce_add_sync(0xffffffffu, others.y + (lane < warp ? sh.warp_sum[1][lane] : 0u));
  // No block leaves while another reads its counts: this warp has read them.
  if (ranks > 1) asm volatile("barrier.cluster.arrive.aligned;" ::: "memory");
#pragma unroll 4
  for (int i0 = w0; i0 < w1; i0 += 32) {
    const int i = i0 + lane;
    const uint32_t x = i < w1 ? key(i) : 0u;
    const uint32_t is_gt = __ballot_sync(0xffffffffu, i < w1 && x > prefix);
    const uint32_t is_eq = __ballot_sync(0xffffffffu, i < w1 && x == prefix);
    const uint32_t below = (1u << lane) - 1;
    const uint32_t g = gt_before + __popc(is_gt & below), e = eq_before + __popc(is_eq & below);
    if (i < w1 && (x > prefix || (x == prefix && e < want))) out[g + min(e, want)] = lo + i;
    gt_before += __popc(is_gt);
    eq_before += __popc(is_eq);
  }
  if (bad) record(MES_ERR_INVALID);
  __syncwarp();
  if (ranks > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
}

// Compaction: run (sequence, new page, side, head) gathers its tokens in kept order.  The run's
// scale is the largest of its sources' scales, so tokens from the source that has it move
// unchanged and the others are re-rounded once.
// Measured: 16384 tokens of 8 heads 16 us after the selection (67 MB, 4.2 TB/s; a chain of four loads,
// index, page, scale and codes, for each run).
template <int kKind, int P>
__global__ void __launch_bounds__(Shape<P>::kThreads)
kv8_compact_kernel(uint8_t* codes, float* scales, float* sums, const int32_t* __restrict__ table,
                   int64_t width, const int32_t* __restrict__ new_table, int new_width,
                   const int32_t* __restrict__ kept, int keep, int Hkv, int64_t num_pages) {
  using Run = Shape<P>;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  __shared__ float red[8];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int b = blockIdx.x / new_width, j = blockIdx.x - b * new_width;
  const int run = blockIdx.y * Run::kRuns + warp / Run::kRunWarps;
  const int side = run >= Hkv, h = run - side * Hkv;
  bool ok = run < 2 * Hkv;
  int64_t to = 0;
  if (ok) {
    to = new_table[blockIdx.x];
    if (to < 0 || to >= num_pages) {
      ok = false;
      record(MES_ERR_INVALID);
    }
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");      // the kept tokens are there; every block waits
  // Lane l looks up token l of the warp's rows (the upper lanes once more).
  const int slot0 = warp % Run::kRunWarps * kRows;
  const int place = j * P + slot0 + (lane & (kRows - 1));
  const int t = ok && place < keep ? kept[((int64_t)b * Hkv + h) * keep + place] : -1;
  int64_t row = -1;
  float s = 0.f, sum = 0.f;
  if (t >= 0) {
    const int64_t page = table[(int64_t)b * width + t / P];
    if (page < 0 || page >= num_pages) {
      record(MES_ERR_INVALID);
    } else {
      const int64_t si = (page * 2 + side) * Hkv + h;
      row = si * P + t % P;
      s = scales[si];
      if (side == 0) sum = sums[(page * Hkv + h) * P + t % P];
    }
  }
  uint4 v[kRows / 4];
#pragma unroll
  for (int i = 0; i < kRows / 4; ++i) {
    const int64_t r = __shfl_sync(0xffffffffu, row, 4 * i + (lane >> 3));
    v[i] = r >= 0 ? *reinterpret_cast<const uint4*>(codes + r * kv8::kD + (lane & 7) * 16)
                  : make_uint4(0, 0, 0, 0);
  }
  const float now = run_max<Run::kRunWarps>(s, red);
  const Divisor by = divisor(now > 0.f ? now : 1.f, false);
  const int64_t di = (to * 2 + side) * Hkv + h;
#pragma unroll
  for (int i = 0; i < kRows / 4; ++i) {
    const float was = __shfl_sync(0xffffffffu, s, 4 * i + (lane >> 3));
    if (was != now) {
      const uint2 o[2] = {requantise8<kKind>(make_uint2(v[i].x, v[i].y), was, by),
                          requantise8<kKind>(make_uint2(v[i].z, v[i].w), was, by)};
      v[i] = make_uint4(o[0].x, o[0].y, o[1].x, o[1].y);
    }
    if (ok)
      *reinterpret_cast<uint4*>(codes + (di * P + slot0 + 4 * i + (lane >> 3)) * kv8::kD + (lane & 7) * 16) = v[i];
  }
  if (!ok) return;
  if (side == 0 && lane < kRows) sums[(to * Hkv + h) * P + slot0 + lane] = sum;
  if (lane == 0 && warp % Run::kRunWarps == 0) scales[di] = now;
}

template <typename F>
int by_page(int page, F f) {
  switch (page) {
    case 16: return f(std::integral_constant<int, 16>());
    case 32: return f(std::integral_constant<int, 32>());
    case 64: return f(std::integral_constant<int, 64>());
    default: return f(std::integral_constant<int, 128>());
  }
}

unsigned run_blocks(int Hkv, int runs) { return (unsigned)((2 * Hkv + runs - 1) / runs); }

}  // namespace

extern "C" int mes_kv8_cache_take_error(int* code) {
  int v = 0, zero = 0;
  cudaError_t e = cudaMemcpyFromSymbol(&v, g_err_kv8_cache, sizeof(int));
  if (e != cudaSuccess) return MES_ERR_CUDA;
  e = cudaMemcpyToSymbol(g_err_kv8_cache, &zero, sizeof(int));
  *code = v;
  return mes_host::from_cuda(e);
}

extern "C" int mes_kv8_append(int dtype, const void* K, int64_t ldk, const void* V, int64_t ldv,
                              void* codes, float* scales, float* sums, const int32_t* block_table,
                              int64_t table_width, const int32_t* cu_new, const int32_t* context_lens,
                              int64_t B, int64_t T, int64_t max_new, int Hkv, int D, int page_size,
                              int64_t num_pages, void* stream) {
  if (!kv8::valid_cache(dtype, num_pages, Hkv, D, page_size)) return MES_ERR_INVALID;
  if (B < 0 || T < 0 || max_new < 0 || max_new > T || table_width <= 0) return MES_ERR_INVALID;
  if (table_width > 0x7fffffffll / page_size || T > 0x7fffffffll) return MES_ERR_INVALID;
  if (ldk < (int64_t)Hkv * D || ldv < (int64_t)Hkv * D || ldk % 8 || ldv % 8) return MES_ERR_INVALID;
  if (B == 0 || T == 0 || max_new == 0) return MES_OK;
  if (!K || !V || !codes || !scales || !block_table || !cu_new || !context_lens) return MES_ERR_INVALID;
  if (!kv8::aligned(K, 16) || !kv8::aligned(V, 16) || !kv8::aligned(codes, 16) || !kv8::aligned(scales, 4) ||
      !kv8::aligned(sums, 4) || !kv8::aligned(block_table, 4) || !kv8::aligned(cu_new, 4) ||
      !kv8::aligned(context_lens, 4))
    return MES_ERR_ALIGN;
  // Pages that max_new tokens can touch, starting anywhere in one.
  const int64_t pages = (max_new + page_size - 2) / page_size + 1;
  if (B * pages > 0x7fffffffll) return MES_ERR_INVALID;
  return by_page(page_size, [&](auto p) {
    constexpr int P = decltype(p)::value;
    using Run = Shape<P>;
    const dim3 grid((unsigned)(B * pages), run_blocks(Hkv, Run::kRuns));
    auto kernel = dtype == kv8::kInt8 ? kv8_append_kernel<kv8::kInt8, P> : kv8_append_kernel<kv8::kE4m3, P>;
    kernel<<<grid, Run::kThreads, 0, (cudaStream_t)stream>>>(
        (const __nv_bfloat16*)K, ldk, (const __nv_bfloat16*)V, ldv, (uint8_t*)codes, scales, sums,
        block_table, table_width, cu_new, context_lens, T, (int)max_new, (int)pages, Hkv, num_pages);
    return mes_host::from_cuda(cudaGetLastError());
  });
}

extern "C" int mes_kv8_read(int dtype, const void* codes, const float* scales, const int32_t* pages,
                            int64_t n, int Hkv, int D, int page_size, int64_t num_pages, void* out,
                            void* stream) {
  if (!kv8::valid_cache(dtype, num_pages, Hkv, D, page_size) || n < 0) return MES_ERR_INVALID;
  if (n == 0) return MES_OK;
  if (!codes || !scales || !pages || !out) return MES_ERR_INVALID;
  if (!kv8::aligned(codes, 16) || !kv8::aligned(out, 16) || !kv8::aligned(scales, 4) || !kv8::aligned(pages, 4))
    return MES_ERR_ALIGN;
  const int run_shift = __builtin_ctz((unsigned)page_size * D / 8);
  const int page_chunks = (2 * Hkv) << run_shift;
  if (n > 0x7fffffffll || n > 0x7fffffffffffffffll / ((int64_t)page_chunks * 32)) return MES_ERR_INVALID;
  const dim3 grid((unsigned)n, (unsigned)((page_chunks + 256 * kReadChunks - 1) / (256 * kReadChunks)));
  auto kernel = dtype == kv8::kInt8 ? kv8_read_kernel<kv8::kInt8> : kv8_read_kernel<kv8::kE4m3>;
  cudaLaunchAttribute early = {};
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(256);
  cfg.stream = (cudaStream_t)stream;
  cfg.attrs = &early;
  cfg.numAttrs = 1;
  return mes_host::from_cuda(cudaLaunchKernelEx(&cfg, kernel, (const uint8_t*)codes, scales, pages, page_chunks, run_shift,
                                                num_pages, (uint4*)out));
}

extern "C" int mes_kv8_evict(int dtype, void* codes, float* scales, float* sums,
                             const int32_t* block_table, int64_t table_width,
                             const int32_t* context_lens, int64_t B, const int32_t* new_table,
                             int64_t new_width, int64_t keep, int64_t recent, int Hkv, int D,
                             int page_size, int64_t num_pages, int32_t* kept, int32_t* new_lens,
                             void* stream) {
  if (!kv8::valid_cache(dtype, num_pages, Hkv, D, page_size)) return MES_ERR_INVALID;
  if (B < 0 || table_width <= 0 || keep <= 0 || recent < 0 || recent > keep) return MES_ERR_INVALID;
  if (table_width > 0x7fffffffll / page_size || keep > 0x7fffffffll - 128) return MES_ERR_INVALID;
  if (new_width != (keep + page_size - 1) / page_size) return MES_ERR_INVALID;
  if (B == 0) return MES_OK;
  if (!codes || !scales || !sums || !block_table || !context_lens || !new_table || !kept || !new_lens)
    return MES_ERR_INVALID;
  if (!kv8::aligned(codes, 16) || !kv8::aligned(scales, 4) || !kv8::aligned(sums, 4) ||
      !kv8::aligned(block_table, 4) || !kv8::aligned(context_lens, 4) || !kv8::aligned(new_table, 4) ||
      !kv8::aligned(kept, 4) || !kv8::aligned(new_lens, 4))
    return MES_ERR_ALIGN;
  // Blocks of a cluster, at most 8 (the portable limit): one for each 8192 possible tokens while all of the
  // grid is resident (a block fills an SM), and as many as keep the keys in shared memory.  One block against
  // the most: 8 heads of 4096 tokens 17 and 24 us (with the compaction), 100003 206 and 58; 256 heads of 9000
  // 94 and 344.
  constexpr int kKeys = 49152;
  const int64_t most = table_width * page_size;
  int ranks = 1;
  while (ranks < 8 && (ranks * (int64_t)kKeys < most ||
                       (ranks * 8192ll < most && B * Hkv * ranks * 2 <= mes_host::sm_count())))
    ranks *= 2;
  if (B * Hkv > 0x7fffffffll / ranks || B * new_width > 0x7fffffffll) return MES_ERR_INVALID;
  // Keys kept in shared memory (up to 192 KB); a longer slice's rest is read again in each pass.
  const int64_t slice = (most + ranks - 1) / ranks + 32;
  const int cap = (int)(slice < kKeys ? slice : kKeys);
  static std::atomic<uint64_t> configured{0};
  int st = mes_host::once_per_device(configured, [] {
    return mes_host::from_cuda(cudaFuncSetAttribute(
        kv8_select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kKeys * 4));
  });
  if (st != MES_OK) return st;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(B * Hkv * ranks));
  cfg.blockDim = dim3(kSelThreads);
  cfg.dynamicSmemBytes = (size_t)cap * 4;
  cfg.stream = (cudaStream_t)stream;
  cudaLaunchAttribute attr = {};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = ranks;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kv8_select_kernel, (const float*)sums, block_table, table_width,
                                     context_lens, Hkv, __builtin_ctz((unsigned)page_size), num_pages, (int)keep, (int)recent,
                                     cap, ranks, kv8::aligned(sums, 16), kept, new_lens);
  if (e != cudaSuccess) return MES_ERR_CUDA;
  return by_page(page_size, [&](auto p) {
    constexpr int P = decltype(p)::value;
    using Run = Shape<P>;
    const dim3 grid((unsigned)(B * new_width), run_blocks(Hkv, Run::kRuns));
    auto kernel = dtype == kv8::kInt8 ? kv8_compact_kernel<kv8::kInt8, P> : kv8_compact_kernel<kv8::kE4m3, P>;
    cudaLaunchAttribute early = {};
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t next = {};
    next.gridDim = grid;
    next.blockDim = dim3(Run::kThreads);
    next.stream = (cudaStream_t)stream;
    next.attrs = &early;
    next.numAttrs = 1;
    return mes_host::from_cuda(cudaLaunchKernelEx(
        &next, kernel, (uint8_t*)codes, scales, sums, block_table, table_width, new_table, (int)new_width,
        (const int32_t*)kept, (int)keep, Hkv, num_pages));
  });
}
