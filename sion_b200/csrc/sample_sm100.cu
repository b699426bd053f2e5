// Sampling of one token per row of logits from a given uniform number, with
// temperature, top-k, top-p and min-p, for sm_100a.
//
// Definition (x the row, NaN counting as -inf; m its maximum, T > 0):
//   w_i = exp((x_i - m) / T),  mass_i = round(w_i * 2^31), an integer
//   order: larger x first, ties by lower index
//   top-k keeps the first k; top-p those with less than p of the mass of the
//   kept ones before them; min-p those with w_i >= min_p; the first one always
//   stays. The token is the first, by index, at which the running sum of the
//   kept masses exceeds floor(u * their total).
// T <= 0 takes the first of the largest. A row with nothing above -inf gives -1.
//
// Probabilities are summed as integers: the sums, and so every comparison, do
// not depend on the order or on how the row is split, and the same row and
// number give the same token in every batch. 2^-31 of the largest probability
// is the resolution (a running sum in fp32 would have 2^-24 of the total).
// All three filters keep a prefix of the order, so together they are a threshold
// on the value and a number of ties to keep.
#include "felix_internal.h"
#include "sm100_ptx.cuh"

#include <cuda_bf16.h>

namespace felix_impl {
namespace smp {

constexpr int kThreads = 1024;

template <typename T>
__device__ __forceinline__ float value(const T* p, uint32_t i);
template <>
__device__ __forceinline__ float value(const float* p, uint32_t i) { return p[i]; }
template <>
__device__ __forceinline__ float value(const __half* p, uint32_t i) { return __half2float(p[i]); }
template <>
__device__ __forceinline__ float value(const __nv_bfloat16* p, uint32_t i) {
  return __bfloat162float(p[i]);
}

// Unsigned key in the order of the values; NaN as -inf, -0 as +0.
__device__ __forceinline__ uint32_t key_of(float x) {
  if (x != x) x = -INFINITY;
  x += 0.f;
  const uint32_t b = __float_as_uint(x);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
__device__ __forceinline__ float scaled(float x, float top, float temp) {
  return x == top ? 0.f : __fdiv_rn(x - top, temp);
}
__device__ __forceinline__ uint32_t mass_of(float w) { return __float2uint_rn(w * 2147483648.f); }

struct Shared {
  unsigned long long sum[32];
  uint32_t count[256];
  unsigned long long mass[256];
  unsigned long long before;  // mass or count above the digits chosen so far
  uint32_t prefix, ties;
  int found;
};

__device__ __forceinline__ unsigned long long warp_sum(unsigned long long v) {
#pragma unroll
  for (int d = 16; d; d /= 2) v += __shfl_xor_sync(~0u, v, d);
  return v;
}
// Exclusive prefix over the block; *total its sum.
__device__ unsigned long long block_scan(unsigned long long v, Shared& sh, unsigned long long* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  unsigned long long x = v;
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const unsigned long long y = __shfl_up_sync(~0u, x, d);
    if (lane >= d) x += y;
  }
  __syncthreads();
  if (lane == 31) sh.sum[warp] = x;
  __syncthreads();
  unsigned long long w = sh.sum[lane];
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const unsigned long long y = __shfl_up_sync(~0u, w, d);
    if (lane >= d) w += y;
  }
  const unsigned long long before = __shfl_sync(~0u, w, warp ? warp - 1 : 0);
  *total = __shfl_sync(~0u, w, 31);
  return x - v + (warp ? before : 0);
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 1) sample_kernel(const SampleArgs A) {
  __shared__ Shared sh;
  const uint32_t row = blockIdx.x, V = A.vocab, tid = threadIdx.x;
  const T* x = static_cast<const T*>(A.logits) + int64_t(row) * A.stride;
  const float temp = A.temperature ? A.temperature[row] : 1.f;

  // the largest value and its first index: (key, ~index) as one number
  unsigned long long best = 0;
  for (uint32_t i = tid; i < V; i += kThreads) {
    const unsigned long long k = (unsigned long long)key_of(value<T>(x, i)) << 32 | ~i;
    best = k > best ? k : best;
  }
#pragma unroll
  for (int d = 16; d; d /= 2) {
    const unsigned long long o = __shfl_xor_sync(~0u, best, d);
    best = o > best ? o : best;
  }
  if ((tid & 31) == 0) sh.sum[tid >> 5] = best;
  __syncthreads();
  best = sh.sum[tid & 31];
#pragma unroll
  for (int d = 16; d; d /= 2) {
    const unsigned long long o = __shfl_xor_sync(~0u, best, d);
    best = o > best ? o : best;
  }
  const uint32_t top_key = uint32_t(best >> 32), first = ~uint32_t(best);
  const float top = value_of(top_key);
  if (top == -INFINITY || !(temp > 0.f)) {
    if (tid == 0) {
      A.tokens[row] = top == -INFINITY ? -1 : int32_t(first);
      A.logprobs[row] = top == -INFINITY ? -INFINITY : 0.f;
    }
    return;
  }

  // threshold (key, ties): keys above it are kept, and `ties` of those equal to it
  uint32_t key = 0, ties = 0xffffffffu;
  const int k = A.top_k ? A.top_k[row] : 0;
  const float p = A.top_p ? A.top_p[row] : 1.f, mp = A.min_p ? A.min_p[row] : 0.f;
  const bool only_first = (A.top_p && !(p > 0.f)) || (A.min_p && !(mp <= 1.f));
  for (int pass = 0; pass < 2 && !only_first; ++pass) {
    const bool by_mass = pass == 1;
    if (by_mass ? !(A.top_p && p < 1.f) : !(k > 0 && uint32_t(k) < V)) continue;
    double want = double(k);
    if (by_mass) {
      unsigned long long mine = 0, total, tie_mass = 0;
      uint32_t n_ties = 0;
      for (uint32_t i = tid; i < V; i += kThreads) {
        const uint32_t kk = key_of(value<T>(x, i));
        if (kk > key) mine += mass_of(expf(scaled(value_of(kk), top, temp)));
        n_ties += kk == key;
      }
      block_scan(mine, sh, &total);
      if (ties == 0xffffffffu) {
        block_scan(n_ties, sh, &tie_mass);
      } else {
        tie_mass = ties;
      }
      total += tie_mass * mass_of(expf(scaled(value_of(key), top, temp)));
      want = double(p) * double(total);
    }
    if (tid == 0) sh.before = 0, sh.prefix = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
      if (tid < 256) sh.count[tid] = 0, sh.mass[tid] = 0;
      __syncthreads();
      const uint32_t prefix = sh.prefix;
      for (uint32_t i = tid; i < V; i += kThreads) {
        const uint32_t kk = key_of(value<T>(x, i));
        if (kk < key || (shift < 24 && (kk ^ prefix) >> (shift + 8))) continue;
        const uint32_t d = (kk >> shift) & 255u;
        atomicAdd(&sh.count[d], 1u);
        if (by_mass)
          atomicAdd(&sh.mass[d], (unsigned long long)mass_of(expf(scaled(value_of(kk), top, temp))));
      }
      __syncthreads();
      if (tid == 0) {
        // the last digit, from the top, that something before `want` falls in
        unsigned long long acc = sh.before, at = acc;
        int last = -1;
        for (int d = 255; d >= 0; --d) {
          if (!sh.count[d]) continue;
          if (last >= 0 && !(double(acc) < want)) break;
          last = d;
          at = acc;
          acc += by_mass ? sh.mass[d] : sh.count[d];
        }
        sh.before = at;
        sh.prefix = prefix | uint32_t(last) << shift;
        sh.ties = sh.count[last];
      }
      __syncthreads();
    }
    // of the equal ones, those with less than `want` before them
    const uint32_t found = sh.prefix;
    const unsigned long long each =
        by_mass ? mass_of(expf(scaled(value_of(found), top, temp))) : 1ull;
    uint32_t n = min(sh.ties, found == key ? ties : 0xffffffffu);
    if (each) {
      uint32_t lo = 1, hi = n;  // the largest n with before + (n - 1) each < want
      while (lo < hi) {
        const uint32_t mid = lo + (hi - lo + 1) / 2;
        if (double(sh.before + (unsigned long long)(mid - 1) * each) < want) lo = mid;
        else hi = mid - 1;
      }
      n = lo;
    }
    key = found;
    ties = n;
    __syncthreads();
  }
  if (only_first) key = top_key, ties = 1;

  // total of the kept masses, then the token
  auto walk = [&](unsigned long long target, bool find) -> unsigned long long {
    unsigned long long sum = 0;
    uint32_t seen = 0;
    for (uint32_t i0 = 0; i0 < V; i0 += kThreads) {
      const uint32_t i = i0 + tid;
      const uint32_t kk = i < V ? key_of(value<T>(x, i)) : 0;
      unsigned long long tot;
      const bool tie = i < V && kk == key;
      uint32_t rank = 0;
      if (ties != 0xffffffffu) {
        rank = seen + uint32_t(block_scan(tie, sh, &tot));
        seen += uint32_t(tot);
      }
      const float w = i < V ? expf(scaled(value_of(kk), top, temp)) : 0.f;
      const bool keep = i < V && (kk > key || (tie && rank < ties)) && (kk == top_key || !(w < mp));
      const unsigned long long mass = keep ? mass_of(w) : 0;
      const unsigned long long at = sum + block_scan(mass, sh, &tot);
      sum += tot;
      if (find && at <= target && target < at + mass) sh.found = int(i);
      if (find && sum > target) break;
    }
    return sum;
  };
  const unsigned long long total = walk(0, false);
  const double at = double(A.uniform[row]) * double(total);
  unsigned long long target = at > 0. ? (unsigned long long)at : 0;
  if (target >= total) target = total - 1;
  walk(target, true);
  __syncthreads();
  if (tid == 0) {
    const float z = scaled(value_of(key_of(value<T>(x, uint32_t(sh.found)))), top, temp);
    A.tokens[row] = sh.found;
    A.logprobs[row] = z - logf(__ull2float_rn(total) * 4.656612873077393e-10f);
  }
}

}  // namespace smp

FelixCode sample_launch(const SampleArgs& a, cudaStream_t stream) {
  if (a.rows == 0) return FelixCode{FELIX_SUCCESS, cudaSuccess};
  switch (a.dtype) {
    case FELIX_F16: smp::sample_kernel<__half><<<a.rows, smp::kThreads, 0, stream>>>(a); break;
    case FELIX_BF16:
      smp::sample_kernel<__nv_bfloat16><<<a.rows, smp::kThreads, 0, stream>>>(a);
      break;
    default: smp::sample_kernel<float><<<a.rows, smp::kThreads, 0, stream>>>(a); break;
  }
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return launch_error(e, "sample");
  return FelixCode{FELIX_SUCCESS, cudaSuccess};
}

}  // namespace felix_impl
