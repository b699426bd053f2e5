// Products of few tokens (9 to 64) with a layer's weights, y = x W^T, same epilogues as
// ffn_product_sm100.cu. Bound by reading W once.
//
// Roles are swapped: the tensor core's 128 rows are 128 rows of W (gated: 64 of the gate's and
// the same 64 of the up projection's), its columns 32 or 64 tokens, so that nearly all of a
// stage is what has to be read. Where there are fewer tiles than SMs, their depth is cut into
// parts over clusters; where there are more, two CTAs with smaller rings share an SM and hide
// each other's ends. Each CTA leaves its fp32 part in its own shared memory as
// [token][feature]; after a cluster barrier each takes a share of the tile, adds the parts
// in their order and finishes it (ffn_finish.cuh). Measured: 24 tokens x 4096 x 16384 26.9 us
// (5 TB/s), 61 through a block of 4096 x 11264 58.5 to 61 us (4.7 TB/s, two launches).
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "ffn_finish.cuh"
#include "ffn_internal.h"
#include "sm100_ptx.cuh"

namespace felix_ffn {
namespace narrow {

using namespace felix_sm100;

constexpr uint32_t kRows = 128, kDepth = 128, kWarps = 6, kThreads = 32 * kWarps;

template <int BN>
struct Shape {
  static constexpr uint32_t kABytes = kRows * kDepth * 2, kBBytes = BN * kDepth * 2;
  static constexpr uint32_t kStageBytes = kABytes + kBBytes;
  // of a CTA that shares its SM with another, or has it for itself
  static constexpr uint32_t kShared = 98304 / kStageBytes, kAlone = 196608 / kStageBytes;
  static constexpr uint32_t bytes(uint32_t stages) { return stages * kStageBytes + 1024 + 256; }
  static_assert(2 * kRows * BN * 4 <= kShared * kStageBytes, "two parts fit the ring");
  static_assert((2 * kAlone + 4) * 8 <= 256, "barriers");
};

struct alignas(64) Params {
  CUtensorMap w[2], x;
  uint32_t tokens, features;
  uint32_t parts, kb, stages;
  uint32_t whole;  // two blocks of 64 k in one request
  Finish fin;
  unsigned* status;
};

template <class T, int EPI, int BN>
__global__ void __launch_bounds__(kThreads, 2) ffn_narrow_kernel(const __grid_constant__ Params p) {
  using S = Shape<BN>;
  constexpr uint32_t kWide = EPI == kGated ? 64 : 128;  // features of a tile
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  const uint32_t stages = p.stages;
  uint64_t* full = reinterpret_cast<uint64_t*>(ring + stages * S::kStageBytes);
  uint64_t* empty = full + stages;
  uint64_t* done = empty + stages;
  uint64_t* received = done + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(received + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const uint32_t rank = p.parts > 1 ? cluster_ctarank() : 0u, tile = blockIdx.x / p.parts;
  const uint32_t f0 = tile * kWide;
  const uint32_t kb0 = p.kb * rank / p.parts, kb1 = p.kb * (rank + 1) / p.parts;

  if (threadIdx.x == 0) {
    tma_prefetch_desc(&p.w[0]);
    tma_prefetch_desc(&p.x);
    for (uint32_t s = 0; s < stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(done, 1);
    mbar_init(received, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, BN);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  wait_for_earlier_launches();

  if (warp == 0) {
    if (elect_one()) {
      // rows of 128 k as two blocks of [rows][64]
      auto load = [&](uint8_t* dst, const CUtensorMap* map, uint64_t* bar, uint32_t row, uint32_t kb,
                      uint32_t block) {
        if (p.whole && block) {
          tma_load_3d(dst, map, bar, 0, int(row), int(kb * 2));
        } else {
          // (gated: the blocks of the two weights alternate)
          const uint32_t step = block ? block : kRows * 128;
          tma_load_2d(dst, map, bar, int(kb * kDepth), int(row));
          tma_load_2d(dst + step, map, bar, int(kb * kDepth + 64), int(row));
        }
      };
      uint32_t stage = 0, phase = 0;
      for (uint32_t kb = kb0; kb < kb1; ++kb) {
        if (!mbar_sleep_wait(&empty[stage], phase ^ 1u, abort_flag, p.status, kWdProducerEmpty))
          break;
        uint8_t* sa = ring + stage * S::kStageBytes;
        mbar_arrive_expect_tx(&full[stage], S::kStageBytes);
        if constexpr (EPI == kGated) {
          load(sa, &p.w[0], &full[stage], f0, kb, 0);
          load(sa + 64 * 128, &p.w[1], &full[stage], f0, kb, 0);
        } else {
          load(sa, &p.w[0], &full[stage], f0, kb, kRows * 128);
        }
        load(sa + S::kABytes, &p.x, &full[stage], 0, kb, BN * 128);
        if (++stage == stages) stage = 0, phase ^= 1u;
      }
    }
  } else if (warp == 1) {
    const uint32_t idesc = make_idesc_f16_f32(kRows, BN, false, false) |
                           (Pair<T>::kBf16 ? (1u << 7 | 1u << 10) : 0u);
    uint32_t stage = 0, phase = 0;
    bool ok = true;
    for (uint32_t kb = kb0; kb < kb1; ++kb) {
      ok = __all_sync(~0u, mbar_sleep_wait(&full[stage], phase, abort_flag, p.status, kWdMmaFull));
      if (!ok) break;
      tc_fence_after();
      if (elect_one()) {
        const uint32_t a0 = smem_u32(ring + stage * S::kStageBytes);
        const uint64_t ad = make_sdesc_sw128(a0, 16, 1024);
        const uint64_t bd = make_sdesc_sw128(a0 + S::kABytes, 16, 1024);
#pragma unroll
        for (uint32_t k = 0; k < kDepth / 16; ++k)
          umma_f16_ss(tmem, ad + ((k >> 2) * (kRows * 128) + (k & 3) * 32 >> 4),
                      bd + ((k >> 2) * (BN * 128) + (k & 3) * 32 >> 4), idesc, kb > kb0 || k > 0);
        umma_commit(&empty[stage]);
        if (kb + 1 == kb1) umma_commit(done);
      }
      __syncwarp();
      if (++stage == stages) stage = 0, phase ^= 1u;
    }
    if (!ok) {
      // gave up: what was issued completes, and copies under way land, before the memory
      // goes away
      if (elect_one()) umma_commit(done);
      __syncwarp();
      int none = 0;
      for (uint32_t s = 0; s < stages; ++s)
        mbar_wait(&full[(stage + s) % stages], phase ^ uint32_t(stage + s >= stages), &none,
                  p.status, kWdDrain, 100000000ull);
    }
  } else {
    // the accumulator to shared memory, as [token][feature]
    const bool ok = __all_sync(~0u, mbar_sleep_wait(done, 0, abort_flag, p.status,
                                                    kWdEpilogueTmemFull)) != 0;
    if (ok) {
      tc_fence_after();
      const uint32_t row = (warp & 3) * 32 + lane;
      float* part = reinterpret_cast<float*>(ring);
#pragma unroll 1
      for (uint32_t c = 0; c < BN; c += 32) {
        uint32_t r[32];
        tmem_ld_32x32b_x32(tmem + ((warp & 3) * 32u << 16) + c, r);
        tmem_ld_wait();
#pragma unroll
        for (uint32_t j = 0; j < 32; ++j)
          part[((c + j) * 32 + ((row / 4) ^ ((c + j) & 7))) * 4 + row % 4] = __uint_as_float(r[j]);
      }
      fence_proxy_async_smem();  // it will be sent from there
    } else {
      int none = 0;
      mbar_wait(done, 0, &none, p.status, kWdDrain, 200000000ull);
    }
    tc_fence_before();
  }

  const TilePlace place{0, 0, f0, p.tokens, min(kWide, p.features - f0)};  // all tokens
  finish_tile<T, EPI, 128, BN, 8>(p.fin, place, ring, p.parts, rank, 0, 1, kThreads, received,
                                  p.status);
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, BN);
  }
}

template <class T, int EPI, int BN>
FelixCode launch(DeviceInfo* dev, Params& p, uint32_t tiles, cudaStream_t stream) {
  p.stages = tiles * p.parts <= uint32_t(dev->num_sms) ? Shape<BN>::kAlone : Shape<BN>::kShared;
  const auto kernel = ffn_narrow_kernel<T, EPI, BN>;
  static felix_impl::PerDeviceOnce once;
  const int rc = once.run(dev->ordinal, [&] {
    return int(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    Shape<BN>::bytes(Shape<BN>::kAlone)));
  });
  if (rc) return felix_impl::launch_error(cudaError_t(rc), "feed-forward product: attributes");
  const cudaError_t e = launch_behind(kernel, tiles * p.parts, 1, kThreads,
                                      Shape<BN>::bytes(p.stages), p.parts, stream, p);
  if (e != cudaSuccess) return felix_impl::launch_error(e, "feed-forward product: launch failed");
  return FelixCode{FELIX_SUCCESS, cudaSuccess};
}

template <class T>
FelixCode launch(DeviceInfo* dev, Params& p, uint32_t tiles, bool gated, uint32_t bn,
                 cudaStream_t stream) {
  if (gated)
    return bn == 32 ? launch<T, kGated, 32>(dev, p, tiles, stream)
                    : launch<T, kGated, 64>(dev, p, tiles, stream);
  return bn == 32 ? launch<T, kLinear, 32>(dev, p, tiles, stream)
                  : launch<T, kLinear, 64>(dev, p, tiles, stream);
}

// Rows of whole 64-wide blocks as a third dimension, or as they are.
int encode(CUtensorMap* map, const Mat& m, bool whole, uint32_t rows, uint32_t k, uint32_t box) {
  const uint64_t pitch = rows > 1 ? uint64_t(m.ld) * 2 : (uint64_t(k) * 2 + 15) / 16 * 16;
  if (whole)
    return felix_impl::encode_tmap_3d_f16(map, m.p, 64, rows, k / 64, pitch, 128, 64, box, 2);
  return felix_impl::encode_tmap_2d_f16(map, m.p, k, rows, pitch, 64, box);
}

}  // namespace narrow

using namespace narrow;

FelixCode narrow_launch(DeviceInfo* dev, const Product& x, cudaStream_t stream) {
  const bool gated = x.epilogue == kGated;
  const uint32_t bn = x.m[0] > 32 ? 64 : 32, wide = gated ? 64 : 128;
  Params p{};
  p.tokens = x.m[0];
  p.features = x.n[0];
  const uint32_t tiles = (p.features + wide - 1) / wide;
  p.kb = (x.k[0] + kDepth - 1) / kDepth;
  // Parts of 256 k at least, one CTA per SM at most. Measured, tokens x depth x features in 1,
  // 2, 4, 8 parts, us: 24 x 4096 x 4096 17.0, 12.2, 10.6, 11.1; 40 x 8192 x 1024 31.4, 19.2,
  // 12.8, 9.8; 64 x 8192 x 8192 33.6, 28.1, 27.3, 33.6; 24 x 4096 x 16384 26.2, 26.2, 29.9, 35.4;
  // gated 40 x 2048 x 5632 12.9, 14.8, 17.7, 22.9.
  p.parts = 1;
  while (p.parts < 8 && tiles * p.parts * 2 <= uint32_t(dev->num_sms) && p.kb >= 4 * p.parts)
    p.parts *= 2;
  p.whole = x.k[0] % 64 == 0;
  int rc = 0;
  for (int i = 0; i < (gated ? 2 : 1); ++i)
    rc |= encode(&p.w[i], x.b[i], p.whole && !gated, p.features, x.k[0], wide);
  rc |= encode(&p.x, x.a[0], p.whole, p.tokens, x.k[0], bn);
  if (rc) return felix_impl::api_error("feed-forward product: cuTensorMapEncodeTiled failed");
  p.fin = finish_of(x);
  p.status = dev->status_word;
  return x.bf16 ? launch<__nv_bfloat16>(dev, p, tiles, gated, bn, stream)
                : launch<__half>(dev, p, tiles, gated, bn, stream);
}

}  // namespace felix_ffn
