// The 4-bit paged cache outside attention, for sm_100a: tokens written into it
// and read back, and its pages reserved, forked, freed, compacted and copied.
//
// The page operations work on device arrays alone (no count goes through the
// host), so a decode loop that uses them can be captured in a graph: `table`
// [slots, width] int32 names the pages of each slot, `lens` [slots] its tokens,
// `refs` [pages] how many slots hold a page. A page with refs <= 0 is free, and
// free pages are always given out from the lowest number up, so that the result
// depends on the inputs alone, not on the history or on the order of threads.
#include <cooperative_groups.h>

#include "felix_internal.h"
#include "kv4_layout.cuh"
#include "sm100_ptx.cuh"

namespace felix_impl {
namespace kv4_cache {

using namespace felix_kv4;

// ------------------------------------------------------------ tokens in and out
struct TokenParams {
  CacheView c;
  const int32_t* counts;  // new tokens of each slot, or nullptr: rows
  uint32_t rows;
  uint32_t blocks;             // append: blocks that the rows of a slot can lie in
  bool vec;                    // append: every row is 16-byte aligned
  const void *k, *v;           // append: sources
  int64_t ks[3], vs[3];        // element strides: slot, head, row
  __half *ko, *vo;             // read: [slots, kv_heads, rows, D]
};

template <typename T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }

// A head vector is held by kLanes = 8 neighbouring lanes, D/8 dimensions each: that
// is a V code's group g, so that a lane's codes of two tokens are one vector of the
// layout, and a warp has four tokens under way with three shuffles to a minimum.
constexpr int kLanes = 8;

// Two fp32 numbers in a register pair.
__device__ __forceinline__ unsigned long long f2(float a, float b) {
  unsigned long long r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 un2(unsigned long long a) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a));
  return r;
}
__device__ __forceinline__ unsigned long long add2(unsigned long long a, unsigned long long b) {
  unsigned long long r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ unsigned long long mul2(unsigned long long a, unsigned long long b) {
  unsigned long long r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ unsigned long long fma2(unsigned long long a, unsigned long long b,
                                                   unsigned long long c) {
  unsigned long long r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
// Minimum and maximum that hand NaN on.
__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// (scale, base) and codes of a head vector, N values a lane:
//   scale = fp16((max - min) / 15), base = fp16(min + 8 scale),
//   code = clamp(rint((x - base) / scale) + 8, 0, 15).
// Values past fp16's range count as its largest; a vector with an infinity or a
// NaN has scale and base NaN. scale = 0 (all equal): the value is base alone.
//
// Long prompts are bound by these instructions (about 9 a value, 30 before these
// forms: 40 us for 8 x 2047 x 8 x 128 x 2 values), so: quotients of two values at a
// time, correctly rounded by Markstein's correction (1990: r = RN(1 / s), q = RN(d r)
// is within a unit in the last place, its remainder exact in a fused operation);
// rint by adding 1.5 * 2^23, which leaves the code in the low bits; and codes joined
// by a multiply-add of those bits, whose upper parts are a constant.
template <int N>
__device__ __forceinline__ uint32_t quantise(float (&x)[N], uint32_t (&words)[N / 8]) {
  float lo = x[0], hi = x[0];
#pragma unroll
  for (int i = 1; i < N; ++i) lo = min_nan(lo, x[i]), hi = max_nan(hi, x[i]);
#pragma unroll
  for (int d = kLanes / 2; d; d /= 2) {
    lo = min_nan(lo, __shfl_xor_sync(~0u, lo, d));
    hi = max_nan(hi, __shfl_xor_sync(~0u, hi, d));
  }
  const bool bad = !(lo > -INFINITY && hi < INFINITY);
  if (!(lo >= -65504.f && hi <= 65504.f)) {
    lo = fmaxf(lo, -65504.f), hi = fminf(hi, 65504.f);
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = fminf(fmaxf(x[i], -65504.f), 65504.f);
  }
  const __half sh = __float2half_rn(__fdiv_rn(hi - lo, 15.f));
  const float s = __half2float(sh);
  const __half bh = __float2half_rn(__fadd_rn(lo, 8.f * s));
  const float b = __half2float(bh), r = s > 0.f ? __frcp_rn(s) : 0.f;  // 0: all codes 8
  constexpr float kRound = 12582912.f;  // 1.5 * 2^23
  const auto nb = f2(-b, -b), rr = f2(r, r), ns = f2(-s, -s), up = f2(kRound + 8.f, kRound + 8.f);
#pragma unroll
  for (int w = 0; w < N / 8; ++w) {
    uint32_t sum = 0;
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      const auto d = add2(f2(x[8 * w + i], x[8 * w + i + 1]), nb);
      const auto q = mul2(d, rr);
      // adding an even 8 with the rounding constant keeps ties to even
      const float2 c = un2(add2(fma2(fma2(q, ns, d), rr, q), up));
      const float c0 = fminf(fmaxf(c.x, kRound), kRound + 15.f);
      const float c1 = fminf(fmaxf(c.y, kRound), kRound + 15.f);
      sum += __float_as_uint(c0) * (1u << (4 * i)) + __float_as_uint(c1) * (1u << (4 * i + 4));
    }
    words[w] = sum - 0x4b400000u * 0x11111111u;  // the bits of kRound, eight times
  }
  const uint32_t par = uint32_t(__half_as_ushort(sh)) | (uint32_t(__half_as_ushort(bh)) << 16);
  return bad ? 0x7e007e00u : par;
}

// One warp per (slot, head, block of the cache that has new tokens), four tokens at
// a time. Bytes of other tokens are not touched.
template <typename T, int D>
__global__ void __launch_bounds__(256) kv4_append_kernel(const TokenParams P) {
  constexpr int N = D / kLanes;
  const int lane = threadIdx.x & 31, part = lane % kLanes;
  const uint32_t head = blockIdx.y, nth = blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32;
  for (uint32_t slot = blockIdx.z; slot < P.c.slots; slot += gridDim.z) {
    const int len = slot_length(P.c, slot);
    const int count = P.counts ? min(P.counts[slot], int(P.rows)) : int(P.rows);
    const int start = len - count;  // token of row 0; tokens before 0 have no place
    const int from = max(start, 0), t0 = (from / int(kBlock) + int(nth)) * int(kBlock);
    if (t0 >= len || count <= 0) continue;
    unsigned char* blk = block_of(P.c, slot, t0, head, D);
    if (!blk) continue;
    const int i1 = (min(len - t0, int(kBlock)) + 3) / 4;
    for (int i = max(from - t0, 0) / 4; i < i1; ++i) {
      const uint32_t r = 4 * i + lane / kLanes;
      const int token = t0 + int(r), row = token - start;
      const bool mine = token >= from && token < len;
      float both_x[2][N];
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        const int64_t* st = which ? P.vs : P.ks;
        const T* src = static_cast<const T*>(which ? P.v : P.k) + int64_t(slot) * st[0] +
                       int64_t(head) * st[1] + int64_t(row) * st[2] + part * N;
        float (&x)[N] = both_x[which];
        if (mine && P.vec) {
#pragma unroll
          for (int j = 0; j < N / 8; ++j) {
            const uint4 w = __ldg(reinterpret_cast<const uint4*>(src) + j);
            const T* e = reinterpret_cast<const T*>(&w);
#pragma unroll
            for (int y = 0; y < 8; ++y) x[8 * j + y] = to_f<T>(e[y]);
          }
        } else {
#pragma unroll
          for (int y = 0; y < N; ++y) x[y] = mine ? to_f<T>(src[y]) : 0.f;
        }
      }
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        float (&x)[N] = both_x[which];
        uint32_t w[N / 8];
        const uint32_t par = quantise<N>(x, w);
        if (which == 0) {
          if (mine) {
            if constexpr (N == 16)
              *reinterpret_cast<uint2*>(blk + r * (D / 2) + part * 8) = make_uint2(w[0], w[1]);
            else
              *reinterpret_cast<uint32_t*>(blk + r * (D / 2) + part * 4) = w[0];
          }
        } else {
          // four codes of this token and of the pair's other one make a word
          unsigned char* dst = blk + v_codes_at(D) + (r / 8) * 4 * D + part * (D / 2) +
                               (r % 8 / 2) * (D / 8);
          const bool both = __shfl_xor_sync(~0u, int(mine), kLanes) && mine;
          uint32_t o[N / 8], pair[N / 4];
#pragma unroll
          for (int j = 0; j < N / 8; ++j) {
            o[j] = __shfl_xor_sync(~0u, w[j], kLanes);
            pair[2 * j] = (w[j] & 0xffffu) | (o[j] << 16);
            pair[2 * j + 1] = (w[j] >> 16) | (o[j] & 0xffff0000u);
          }
          if (both && !(r & 1)) {
            if constexpr (N == 16)
              *reinterpret_cast<uint4*>(dst) = make_uint4(pair[0], pair[1], pair[2], pair[3]);
            else
              *reinterpret_cast<uint2*>(dst) = make_uint2(pair[0], pair[1]);
          } else if (mine && !both) {
#pragma unroll
            for (int j = 0; j < N / 4; ++j)
              *reinterpret_cast<uint16_t*>(dst + 4 * j + 2 * (r & 1)) =
                  uint16_t(w[j / 2] >> (16 * (j % 2)));
          }
        }
        if (mine && part == 0)
          reinterpret_cast<uint32_t*>(blk + (which ? v_params_at(D) : k_params_at(D)))[r] = par;
      }
    }
  }
}

// kLanes lanes per (slot, head, row).
template <int D>
__global__ void __launch_bounds__(256) kv4_read_kernel(const TokenParams P) {
  constexpr int N = D / kLanes;
  const int part = threadIdx.x % kLanes;
  const uint32_t head = blockIdx.y, row = (blockIdx.x * blockDim.x + threadIdx.x) / kLanes;
  if (row >= P.rows) return;
  for (uint32_t slot = blockIdx.z; slot < P.c.slots; slot += gridDim.z) {
    const uint64_t item = (uint64_t(slot) * P.c.kv_heads + head) * P.rows + row;
    const int len = slot_length(P.c, slot);
    const int count = P.counts ? min(P.counts[slot], int(P.rows)) : int(P.rows);
    const int token = len - count + int(row);
    const unsigned char* blk = (int(row) < count && token >= 0)
                                   ? block_of(P.c, slot, token, head, D) : nullptr;
    const uint32_t r = uint32_t(token) % kBlock;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      uint32_t w[N / 8] = {};
      float2 sb = make_float2(0.f, 0.f);
      if (blk) {
        if (which == 0) {
#pragma unroll
          for (int j = 0; j < N / 8; ++j)
            w[j] = __ldg(reinterpret_cast<const uint32_t*>(blk + r * (D / 2) + part * (N / 2)) + j);
        } else {
          const uint16_t* src = reinterpret_cast<const uint16_t*>(
              blk + v_codes_at(D) + (r / 8) * 4 * D + part * (D / 2) + (r % 8 / 2) * (D / 8) +
              2 * (r & 1));
#pragma unroll
          for (int j = 0; j < N / 4; ++j)
            w[j / 2] |= uint32_t(__ldg(src + 2 * j)) << (16 * (j % 2));
        }
        const uint32_t par = __ldg(
            reinterpret_cast<const uint32_t*>(blk + (which ? v_params_at(D) : k_params_at(D))) + r);
        sb = __half22float2(*reinterpret_cast<const __half2*>(&par));
      }
      // 2^23 + code by its bits, less 2^23 + 8; scale times that is exact
      alignas(16) __half2 out[N / 2];
      const auto less = f2(-8388616.f, -8388616.f), scale = f2(sb.x, sb.x), base = f2(sb.y, sb.y);
#pragma unroll
      for (int i = 0; i < N; i += 2) {
        const uint32_t v = w[i / 8] >> (4 * (i % 8));
        const auto c = add2(f2(__uint_as_float((v & 15u) | 0x4b000000u),
                               __uint_as_float((v >> 4 & 15u) | 0x4b000000u)), less);
        const float2 y = un2(fma2(scale, c, base));
        out[i / 2] = __floats2half2_rn(y.x, y.y);
      }
      uint4* dst = reinterpret_cast<uint4*>((which ? P.vo : P.ko) + item * D + part * N);
#pragma unroll
      for (int j = 0; j < N / 8; ++j) dst[j] = reinterpret_cast<const uint4*>(out)[j];
    }
  }
}

// ---------------------------------------------------------------------- copies
// Pages src[i] of one pool to dst[i] of another (or the same), `count` of them
// (known on the device). Work is cut in chunks of 16 KB. 515 pages of 35 KB take 5.4 us
// in a graph (floor 5.5 at the card's copy rate; part of it stays in the L2), the 776
// moved by a compaction of 6007 pages of 70 KB 19 us (16.5).
constexpr uint32_t kChunk = 16384;

__global__ void __launch_bounds__(256) kv4_copy_kernel(
    const unsigned char* from, uint64_t from_pages, unsigned char* to, uint64_t to_pages,
    size_t page_bytes, const int32_t* src, const int32_t* dst, const uint32_t* count_dev,
    uint32_t count_host) {
  const uint64_t count = count_dev ? *count_dev : count_host;
  const uint32_t chunks = uint32_t((page_bytes + kChunk - 1) / kChunk);
  for (uint64_t i = blockIdx.x; i < count * chunks; i += gridDim.x) {
    const int s = src[i / chunks], d = dst[i / chunks];
    if (s < 0 || d < 0 || uint64_t(s) >= from_pages || uint64_t(d) >= to_pages) continue;
    const size_t at = size_t(i % chunks) * kChunk;
    const uint32_t n = uint32_t(min(size_t(kChunk), page_bytes - at)) / 16;
    const uint4* a = reinterpret_cast<const uint4*>(from + size_t(s) * page_bytes + at);
    uint4* b = reinterpret_cast<uint4*>(to + size_t(d) * page_bytes + at);
    for (uint32_t j = threadIdx.x; j < n; j += 256) b[j] = a[j];
  }
}

// ------------------------------------------------------------- page operations
// One cluster of kCtas CTAs does each: scans over refs and slots run in the
// CTAs, their totals are exchanged through distributed shared memory, and the
// cluster barrier orders global reads and writes between the steps. Barriers and
// dependent loads bound them: in a graph free, fork (with its copies) and reserve
// take 20 us together for 16 slots and 1024 pages, 42 us for 512 slots and 65536.
constexpr int kCtas = 8;
constexpr int kMeta = 1024;

struct MetaParams {
  const int32_t *table, *lens, *refs;
  int32_t *table_out, *lens_out, *refs_out;  // each may be its input
  int32_t* status;                           // [2]: pages missing, entries skipped
  const int32_t *a, *b;                      // counts; parents, children; slots to free
  uint32_t slots, width, pages, page_shift, n;
  // scratch
  int32_t *fresh;           // [pages] free pages in ascending order; compact: page map
  int32_t *start;           // [slots or n] first fresh page of each
  int32_t *owner;           // [slots]
  int32_t *src, *dst;       // copies to make
  uint32_t* moves;          // their number
};

struct MetaShared {
  uint32_t warp[32];
  uint32_t total[2];  // this CTA's totals, read by the others
};

// Cluster barrier after code in which a warp's threads may have gone apart.
__device__ __forceinline__ void csync() {
  __syncwarp();
  felix_sm100::cluster_sync();
}

// Exclusive prefix of v over the CTA; *sum the total.
__device__ __forceinline__ uint32_t scan(uint32_t v, MetaShared& sh, uint32_t* sum) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t x = v;
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const uint32_t y = __shfl_up_sync(~0u, x, d);
    if (lane >= d) x += y;
  }
  __syncthreads();  // sh.warp of an earlier scan has been read
  if (lane == 31) sh.warp[warp] = x;
  __syncthreads();
  uint32_t w = sh.warp[lane];
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const uint32_t y = __shfl_up_sync(~0u, w, d);
    if (lane >= d) w += y;
  }
  const uint32_t before = __shfl_sync(~0u, w, warp == 0 ? 0 : warp - 1);
  *sum = __shfl_sync(~0u, w, 31);
  return x - v + (warp ? before : 0);
}

__device__ __forceinline__ uint32_t total_of(MetaShared& sh, int which, uint32_t rank) {
  uint32_t v;
  const uint32_t a = felix_sm100::mapa_shared(felix_sm100::smem_u32(&sh.total[which]), rank);
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}

// A CTA's pages are neighbouring, and so are the kRun of a thread in a pass: 65536
// pages are one pass, one scan.
constexpr uint32_t kRun = 8, kPass = kRun * kMeta;
struct Range {
  uint32_t lo, hi;
};
__device__ __forceinline__ Range pages_of_cta(uint32_t pages, uint32_t rank) {
  const uint32_t run = ((pages + kCtas - 1) / kCtas + kRun - 1) & ~(kRun - 1);
  const uint32_t lo = min(rank * run, pages);
  return {lo, min(lo + run, pages)};
}
// refs of pages p0 .. p0 + kRun - 1, `none` past the range.
__device__ __forceinline__ void load_run(const int32_t* refs, uint32_t p0, uint32_t hi, int none,
                                         int (&v)[kRun]) {
  if (p0 + kRun <= hi && (reinterpret_cast<uintptr_t>(refs) & 15) == 0) {
    const int4 a = *reinterpret_cast<const int4*>(refs + p0);
    const int4 b = *reinterpret_cast<const int4*>(refs + p0 + 4);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
    v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  } else {
#pragma unroll
    for (uint32_t e = 0; e < kRun; ++e) v[e] = p0 + e < hi ? refs[p0 + e] : none;
  }
}

// Counts the CTA's pages for which f holds, two predicates at once.
template <class F, class G>
__device__ __forceinline__ void count_pages(const int32_t* refs, Range r, MetaShared& sh, F f,
                                            G g) {
  uint32_t nf = 0, ng = 0, sum;
  for (uint32_t p0 = r.lo + threadIdx.x * kRun; p0 < r.hi; p0 += kPass) {
    int v[kRun];
    load_run(refs, p0, r.hi, 0, v);
#pragma unroll
    for (uint32_t e = 0; e < kRun; ++e)
      if (p0 + e < r.hi) nf += f(p0 + e, v[e]), ng += g(p0 + e, v[e]);
  }
  scan(nf, sh, &sum);
  if (threadIdx.x == 0) sh.total[0] = sum;
  scan(ng, sh, &sum);
  if (threadIdx.x == 0) sh.total[1] = sum;
}

// Tokens of a slot after `count` more (lengths stop short of 2^31).
__device__ __forceinline__ int grown(int len, int count) {
  return int(min((long long)max(len, 0) + max(count, 0), 0x7fffffffll - kMaxPageSize));
}
__device__ __forceinline__ int pages_for(int len, uint32_t shift) {
  return len <= 0 ? 0 : int((uint32_t(len) + (1u << shift) - 1) >> shift);
}

// Free pages: their number, then the first `want` of them into P.fresh, refs
// copied to refs_out with those pages at 1. Call with fits = want <= number.
__device__ uint32_t count_free(const MetaParams& P, MetaShared& sh, Range r, uint32_t rank,
                               uint32_t* before) {
  count_pages(P.refs, r, sh, [](uint32_t, int v) { return uint32_t(v <= 0); },
              [](uint32_t, int) { return 0u; });
  csync();
  uint32_t all = 0;
  *before = 0;
  for (uint32_t k = 0; k < kCtas; ++k) {
    const uint32_t v = total_of(sh, 0, k);
    if (k < rank) *before += v;
    all += v;
  }
  return all;
}
__device__ void take_free(const MetaParams& P, MetaShared& sh, Range r, uint32_t before,
                          uint32_t want) {
  for (uint32_t q = r.lo; q < r.hi; q += kPass) {
    const uint32_t p0 = q + threadIdx.x * kRun;
    int v[kRun];
    load_run(P.refs, p0, r.hi, 1, v);
    uint32_t mine = 0, sum;
#pragma unroll
    for (uint32_t e = 0; e < kRun; ++e) mine += v[e] <= 0;
    uint32_t at = before + scan(mine, sh, &sum);
#pragma unroll
    for (uint32_t e = 0; e < kRun; ++e) {
      if (p0 + e >= r.hi) break;
      const bool is_free = v[e] <= 0, take = is_free && at < want;
      if (take) P.fresh[at] = int32_t(p0 + e);
      P.refs_out[p0 + e] = take ? 1 : v[e];
      at += is_free;
    }
    before += sum;
  }
}

__global__ void __cluster_dims__(kCtas, 1, 1) __launch_bounds__(kMeta, 1)
    kv4_reserve_kernel(const MetaParams P) {
  __shared__ MetaShared sh;
  const uint32_t rank = felix_sm100::cluster_ctarank();
  const Range r = pages_of_cta(P.pages, rank);
  // pages that each slot needs (every CTA counts them all; CTA 0 notes the starts)
  uint32_t want = 0, over = 0;
  for (uint32_t s0 = 0; s0 < P.slots; s0 += kMeta) {
    const uint32_t s = s0 + threadIdx.x;
    uint32_t need = 0, past = 0;
    if (s < P.slots) {
      const int len = max(P.lens[s], 0);
      const int now = pages_for(len, P.page_shift);
      const int then = pages_for(grown(len, P.a[s]), P.page_shift);
      past = max(then - max(now, int(P.width)), 0);
      need = uint32_t(then - now) - past;
    }
    uint32_t sum, sum2;
    const uint32_t at = want + scan(need, sh, &sum);
    scan(past, sh, &sum2);
    if (rank == 0 && s < P.slots) P.start[s] = int32_t(at);
    want += sum;
    over += sum2;
  }
  uint32_t before;
  const uint32_t room = count_free(P, sh, r, rank, &before);
  const bool fits = want <= room && over == 0;
  take_free(P, sh, r, before, fits ? want : 0);
  if (rank == 0 && threadIdx.x == 0) {
    P.status[0] = int32_t((want > room ? want - room : 0) + over);
    P.status[1] = 0;
  }
  csync();
  for (uint32_t s = rank * 32 + threadIdx.x / 32; s < P.slots; s += kCtas * 32) {
    const int len = max(P.lens[s], 0), more = grown(len, P.a[s]);
    const int now = pages_for(len, P.page_shift);
    const int then = fits ? pages_for(more, P.page_shift) : now;
    const int32_t* in = P.table + size_t(s) * P.width;
    int32_t* out = P.table_out + size_t(s) * P.width;
    const bool inplace = P.table == P.table_out;
    const int lo = inplace ? now : 0, hi = inplace ? then : int(P.width);
#pragma unroll 4
    for (int j = lo + int(threadIdx.x & 31); j < min(hi, int(P.width)); j += 32)
      out[j] = j >= now && j < then ? P.fresh[P.start[s] + j - now] : in[j];
    __syncwarp();
    if ((threadIdx.x & 31) == 0) P.lens_out[s] = fits ? more : P.lens[s];
  }
}

__global__ void __cluster_dims__(kCtas, 1, 1) __launch_bounds__(kMeta, 1)
    kv4_fork_kernel(const MetaParams P) {
  __shared__ MetaShared sh;
  const uint32_t rank = felix_sm100::cluster_ctarank();
  const Range r = pages_of_cta(P.pages, rank);
  const uint32_t all = kCtas * kMeta, me = rank * kMeta + threadIdx.x;
  const int32_t none = int32_t(P.n);
  for (uint32_t s = me; s < P.slots; s += all) P.owner[s] = none;
  csync();
  // the first pair that names a child has it
  for (uint32_t i = me; i < P.n; i += all) {
    const int c = P.b[i];
    if (c >= 0 && uint32_t(c) < P.slots) atomicMin(&P.owner[c], int32_t(i));
  }
  uint32_t before;
  const uint32_t room = count_free(P, sh, r, rank, &before);  // has a cluster barrier
  uint32_t want = 0, skipped = 0;
  for (uint32_t i0 = 0; i0 < P.n; i0 += kMeta) {
    const uint32_t i = i0 + threadIdx.x;
    bool valid = false, need = false;
    int len = 0;
    if (i < P.n) {
      const int p = P.a[i], c = P.b[i];
      valid = p >= 0 && c >= 0 && uint32_t(p) < P.slots && uint32_t(c) < P.slots && p != c &&
              P.owner[c] == int32_t(i) && P.lens[c] <= 0;
      if (valid) len = max(P.lens[p], 0);
      const uint32_t whole = uint32_t(len) >> P.page_shift;
      need = valid && (uint32_t(len) & ((1u << P.page_shift) - 1)) != 0 && whole < P.width;
      // a last page that is not in the pool is missing in the copy too: a fresh one
      // would show what its tokens held for an earlier slot
      if (need) {
        const int last = P.table[size_t(p) * P.width + whole];
        need = last >= 0 && uint32_t(last) < P.pages;
      }
    }
    uint32_t sum, sum2;
    const uint32_t at = want + scan(need, sh, &sum);
    scan(i < P.n && !valid, sh, &sum2);
    if (rank == 0 && i < P.n) {
      P.start[2 * i] = need ? int32_t(at) : -1;
      P.start[2 * i + 1] = valid ? len : -1;  // -1: the pair is skipped
    }
    want += sum;
    skipped += sum2;
  }
  const bool fits = want <= room;
  take_free(P, sh, r, before, fits ? want : 0);
  if (rank == 0 && threadIdx.x == 0) {
    P.status[0] = fits ? 0 : int32_t(want - room);
    P.status[1] = int32_t(skipped);
    *P.moves = fits ? want : 0;
  }
  csync();
  const int lane = threadIdx.x & 31;
  for (uint32_t s = rank * 32 + threadIdx.x / 32; s < P.slots; s += kCtas * 32) {
    const int i = P.owner[s];
    const int len = i != none && fits ? P.start[2 * i + 1] : -1;
    const bool child = len >= 0;
    if (!child && P.table == P.table_out) {
      if (lane == 0) P.lens_out[s] = P.lens[s];
      continue;
    }
    const int32_t* in = P.table + size_t(child ? uint32_t(P.a[i]) : s) * P.width;
    int32_t* out = P.table_out + size_t(s) * P.width;
    const int whole = child ? len >> P.page_shift : 0, at = child ? P.start[2 * i] : -1;
#pragma unroll 4
    for (int j = lane; j < int(P.width); j += 32) {
      int v = in[j];
      if (child) {
        if (j < whole) {
          if (v >= 0 && uint32_t(v) < P.pages) atomicAdd(&P.refs_out[v], 1);
        } else if (j == whole && at >= 0) {
          P.src[at] = v;
          v = P.dst[at] = P.fresh[at];
        } else {
          v = -1;
        }
      }
      out[j] = v;
    }
    if (lane == 0) P.lens_out[s] = child ? len : P.lens[s];
  }
}

__global__ void __cluster_dims__(kCtas, 1, 1) __launch_bounds__(kMeta, 1)
    kv4_free_kernel(const MetaParams P) {
  const uint32_t rank = felix_sm100::cluster_ctarank();
  const uint32_t all = kCtas * kMeta, me = rank * kMeta + threadIdx.x;
  for (uint32_t s = me; s < P.slots; s += all) P.owner[s] = 0;
  if (P.refs != P.refs_out)
    for (uint32_t p = me; p < P.pages; p += all) P.refs_out[p] = P.refs[p];
  csync();
  for (uint32_t i = me; i < P.n; i += all) {
    const int s = P.a[i];
    if (s >= 0 && uint32_t(s) < P.slots) P.owner[s] = 1;  // twice named, once freed
  }
  csync();
  const int lane = threadIdx.x & 31;
  for (uint32_t s = rank * 32 + threadIdx.x / 32; s < P.slots; s += kCtas * 32) {
    const bool gone = P.owner[s] != 0;
    const int len = P.lens[s];
    const int held = min(pages_for(len, P.page_shift), int(P.width));
    if (gone || P.table != P.table_out) {
      const int32_t* in = P.table + size_t(s) * P.width;
      int32_t* out = P.table_out + size_t(s) * P.width;
#pragma unroll 4
      for (int j = lane; j < int(P.width); j += 32) {
        const int v = in[j];
        if (gone && j < held && v >= 0 && uint32_t(v) < P.pages) atomicSub(&P.refs_out[v], 1);
        out[j] = gone ? -1 : v;
      }
    }
    __syncwarp();
    if (lane == 0) P.lens_out[s] = gone ? 0 : len;
  }
}

__global__ void __cluster_dims__(kCtas, 1, 1) __launch_bounds__(kMeta, 1)
    kv4_compact_kernel(const MetaParams P) {
  __shared__ MetaShared sh;
  const uint32_t rank = felix_sm100::cluster_ctarank();
  const Range r = pages_of_cta(P.pages, rank);
  const uint32_t all = kCtas * kMeta, me = rank * kMeta + threadIdx.x;
  uint32_t before;
  const uint32_t live = P.pages - count_free(P, sh, r, rank, &before);
  csync();  // the totals have been read
  // live pages from `live` on move into the free ones below it, both in order
  count_pages(P.refs, r, sh, [&](uint32_t p, int v) { return uint32_t(v > 0 && p >= live); },
              [&](uint32_t p, int v) { return uint32_t(v <= 0 && p < live); });
  csync();
  uint32_t s_at = 0, d_at = 0, moves = 0;
  for (uint32_t k = 0; k < kCtas; ++k) {
    const uint32_t v = total_of(sh, 0, k), w = total_of(sh, 1, k);
    if (k < rank) s_at += v, d_at += w;
    moves += v;
  }
  for (uint32_t q = r.lo; q < r.hi; q += kPass) {
    const uint32_t p0 = q + threadIdx.x * kRun;
    int v[kRun];
    load_run(P.refs, p0, r.hi, 0, v);
    uint32_t nf = 0, ni = 0, sum, sum2;
#pragma unroll
    for (uint32_t e = 0; e < kRun; ++e) {
      const uint32_t p = p0 + e;
      nf += p < r.hi && v[e] > 0 && p >= live;
      ni += p < r.hi && v[e] <= 0 && p < live;
    }
    uint32_t a = s_at + scan(nf, sh, &sum), b = d_at + scan(ni, sh, &sum2);
#pragma unroll
    for (uint32_t e = 0; e < kRun; ++e) {
      const uint32_t p = p0 + e;
      if (p >= r.hi) break;
      if (v[e] > 0 && p >= live) {
        P.src[a++] = int32_t(p);
      } else {
        P.fresh[p] = int32_t(p);
        if (v[e] <= 0 && p < live) P.dst[b++] = int32_t(p);
        else P.refs_out[p] = v[e] > 0 ? v[e] : 0;
      }
    }
    s_at += sum;
    d_at += sum2;
  }
  if (me == 0) *P.moves = moves;
  csync();
  for (uint32_t i = me; i < moves; i += all) {
    const int s = P.src[i], d = P.dst[i];
    P.fresh[s] = d;
    P.refs_out[d] = P.refs[s];
    P.refs_out[s] = 0;
  }
  csync();
  const uint64_t entries = uint64_t(P.slots) * P.width;
#pragma unroll 4
  for (uint64_t i = me; i < entries; i += all) {
    const int v = P.table[i];
    P.table_out[i] = v >= 0 && uint32_t(v) < P.pages ? P.fresh[v] : -1;
  }
}

FelixCode done(const char* what) {
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return launch_error(e, what);
  return FelixCode{FELIX_SUCCESS, cudaSuccess};
}

FelixCode copy(DeviceInfo* dev, const void* from, uint64_t from_pages, void* to, uint64_t to_pages,
               size_t page_bytes, const int32_t* src, const int32_t* dst, const uint32_t* count_dev,
               uint32_t count, uint32_t most, cudaStream_t stream) {
  if (most == 0) return FelixCode{FELIX_SUCCESS, cudaSuccess};
  const uint64_t chunks = (page_bytes + kChunk - 1) / kChunk * uint64_t(most);
  const uint32_t grid = uint32_t(chunks < uint64_t(dev->num_sms) * 8 ? chunks : dev->num_sms * 8);
  kv4_copy_kernel<<<grid, 256, 0, stream>>>(
      static_cast<const unsigned char*>(from), from_pages, static_cast<unsigned char*>(to),
      to_pages, page_bytes, src, dst, count_dev, count);
  return done("kv4: page copies");
}

// Scratch of a page operation: the number of copies, then int32 arrays.
size_t scratch_bytes(uint32_t pages, uint32_t slots, uint32_t n) {
  return kWsCounterBytes + 256 +
         sizeof(int32_t) * (size_t(pages) * 3 + size_t(slots) * 2 + size_t(n) * 4);
}

FelixCode scratch(DeviceInfo* dev, MetaParams& P, cudaStream_t stream, Workspace* ws) {
  *ws = library_workspace(dev, stream, scratch_bytes(P.pages, P.slots, P.n));
  if (!ws->ptr) return launch_error(cudaErrorMemoryAllocation, "kv4: workspace");
  char* p = static_cast<char*>(ws->ptr) + kWsCounterBytes;
  P.moves = reinterpret_cast<uint32_t*>(p);
  P.fresh = reinterpret_cast<int32_t*>(p + 256);
  P.src = P.fresh + P.pages;
  P.dst = P.src + P.pages;
  P.owner = P.dst + P.pages;
  P.start = P.owner + P.slots;
  return FelixCode{FELIX_SUCCESS, cudaSuccess};
}

}  // namespace kv4_cache

FelixCode kv4_append_launch(const felix_kv4::CacheView& c, uint32_t head_dim, const void* key,
                            const void* value, bool bf16, uint32_t rows, const int64_t* ks,
                            const int64_t* vs, const int32_t* counts, cudaStream_t stream) {
  kv4_cache::TokenParams P{};
  P.c = c;
  P.counts = counts;
  P.rows = rows;
  P.k = key;
  P.v = value;
  for (int i = 0; i < 3; ++i) P.ks[i] = ks[i], P.vs[i] = vs[i];
  uintptr_t bits = reinterpret_cast<uintptr_t>(key) | reinterpret_cast<uintptr_t>(value);
  for (int i = 0; i < 3; ++i) bits |= uintptr_t(ks[i] * 2) | uintptr_t(vs[i] * 2);
  P.vec = (bits & 15) == 0;
  // rows can start anywhere in a block
  P.blocks = rows == 1 ? 1 : (rows + 14) / felix_kv4::kBlock + 1;
  const dim3 grid((P.blocks + 7) / 8, c.kv_heads, c.slots < 65535u ? c.slots : 65535u);
  if (grid.z == 0 || rows == 0) return FelixCode{FELIX_SUCCESS, cudaSuccess};
  const int threads = P.blocks < 8 ? int(P.blocks) * 32 : 256;
  if (bf16) {
    if (head_dim == 128)
      kv4_cache::kv4_append_kernel<__nv_bfloat16, 128><<<grid, threads, 0, stream>>>(P);
    else kv4_cache::kv4_append_kernel<__nv_bfloat16, 64><<<grid, threads, 0, stream>>>(P);
  } else {
    if (head_dim == 128) kv4_cache::kv4_append_kernel<__half, 128><<<grid, threads, 0, stream>>>(P);
    else kv4_cache::kv4_append_kernel<__half, 64><<<grid, threads, 0, stream>>>(P);
  }
  return kv4_cache::done("kv4_append");
}

FelixCode kv4_read_launch(const felix_kv4::CacheView& c, uint32_t head_dim, uint32_t rows,
                          const int32_t* counts, __half* key, __half* value, cudaStream_t stream) {
  kv4_cache::TokenParams P{};
  P.c = c;
  P.counts = counts;
  P.rows = rows;
  P.ko = key;
  P.vo = value;
  const dim3 grid((rows + 31) / 32, c.kv_heads, c.slots < 65535u ? c.slots : 65535u);
  if (grid.z == 0 || rows == 0) return FelixCode{FELIX_SUCCESS, cudaSuccess};
  if (head_dim == 128) kv4_cache::kv4_read_kernel<128><<<grid, 256, 0, stream>>>(P);
  else kv4_cache::kv4_read_kernel<64><<<grid, 256, 0, stream>>>(P);
  return kv4_cache::done("kv4_read");
}

FelixCode kv4_copy_launch(const void* from, uint64_t from_pages, void* to, uint64_t to_pages,
                          size_t page_bytes, const int32_t* src, const int32_t* dst, uint32_t count,
                          cudaStream_t stream) {
  DeviceInfo* dev = current_device_info();
  if (!dev) return launch_error(cudaGetLastError(), "kv4_copy_pages: no device");
  return kv4_cache::copy(dev, from, from_pages, to, to_pages, page_bytes, src, dst, nullptr, count,
                         count, stream);
}

FelixCode kv4_pages_launch(const Kv4PagesOp& o, cudaStream_t stream) {
  DeviceInfo* dev = current_device_info();
  if (!dev) return launch_error(cudaGetLastError(), "kv4: no device");
  kv4_cache::MetaParams P{};
  P.table = o.table, P.lens = o.lens, P.refs = o.refs;
  P.table_out = o.table_out, P.lens_out = o.lens_out, P.refs_out = o.refs_out;
  P.status = o.status;
  P.a = o.a, P.b = o.b;
  P.slots = o.slots, P.width = o.width, P.pages = o.num_pages;
  P.page_shift = o.page_shift, P.n = o.n;
  Workspace ws;  // until the copies, which take their list from the plan, are launched
  FelixCode rc = kv4_cache::scratch(dev, P, stream, &ws);
  if (rc.type != FELIX_SUCCESS) return rc;
  using namespace kv4_cache;
  switch (o.kind) {
    case Kv4PagesOp::kReserve: kv4_reserve_kernel<<<kCtas, kMeta, 0, stream>>>(P); break;
    case Kv4PagesOp::kFork: kv4_fork_kernel<<<kCtas, kMeta, 0, stream>>>(P); break;
    case Kv4PagesOp::kFree: kv4_free_kernel<<<kCtas, kMeta, 0, stream>>>(P); break;
    case Kv4PagesOp::kCompact: kv4_compact_kernel<<<kCtas, kMeta, 0, stream>>>(P); break;
  }
  rc = done("kv4: page operation");
  if (rc.type != FELIX_SUCCESS) return rc;
  const uint32_t most = o.kind == Kv4PagesOp::kFork ? o.n
                        : o.kind == Kv4PagesOp::kCompact ? o.num_pages / 2 + 1 : 0;
  return kv4_cache::copy(dev, o.pages, o.num_pages, o.pages, o.num_pages, o.page_bytes, P.src, P.dst,
                   P.moves, 0, most, stream);
}

}  // namespace felix_impl
