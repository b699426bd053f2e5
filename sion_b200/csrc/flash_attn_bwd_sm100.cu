// Flash-attention backward for sm_100a, fp16 in/out, fp32 accumulation:
//   given Q, K, V, O, dO and the forward's natural-log LSE, computes
//   dQ, dK, dV of O = softmax(Q K^T * scale) V (optionally causal).
// No reference counterpart (the reference has a forward kernel only); the
// backward of its operator is listed as the next attention feature.
//
// Math (per (b, h)): P = exp(scale * Q K^T - LSE), dV = P^T dO,
// dP = dO V^T, Delta = rowsum(dO * O), dS = P * (dP - Delta),
// dK = scale * dS^T Q, dQ = scale * dS K.
//
// Kernel layout: one CTA per (b, h) and 128-key block j (TMEM lanes = its
// keys), looping over 128-query blocks i (from the diagonal block when
// causal); every MMA is N >= 64 wide and 128 queries deep (narrower MMAs cost
// as much per instruction on this tensor core). See the pipe namespace below.
#include <cuda.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <cstdint>

#include "felix_internal.h"
#include "sm100_ptx.cuh"

// Timing experiments only (results are wrong when set): skip the dQ
// reductions.
#ifndef FELIX_FA_BWD_EXP_NO_DQRED
#define FELIX_FA_BWD_EXP_NO_DQRED 0
#endif
// bit mask of MMA groups left out: 1 S^T, 2 dP^T, 4 dV, 8 dK, 16 dQ (their
// commits stay, so the barrier protocol is unchanged)
#ifndef FELIX_FA_BWD_EXP_SKIP
#define FELIX_FA_BWD_EXP_SKIP 0
#endif

// Timing experiments only: per-role cycle counters around the waits of the
// kernel, summed over all CTAs (read with felix_debug_bwd_trace, which
// exists only in such builds).
#ifndef FELIX_FA_BWD_TRACE
#define FELIX_FA_BWD_TRACE 0
#endif
#if FELIX_FA_BWD_TRACE
__device__ unsigned long long g_bwd_trace[16];
#define BWD_TR_BEGIN(v) const long long v = clock64()
#define BWD_TR_ACC(acc, v) acc += clock64() - v
#define BWD_TR_FLUSH(slot, acc) atomicAdd(&g_bwd_trace[slot], (unsigned long long)(acc))
#else
#define BWD_TR_BEGIN(v)
#define BWD_TR_ACC(acc, v)
#define BWD_TR_FLUSH(slot, acc)
#endif

namespace felix_sm100 {
namespace attn_bwd {

constexpr int kBlk = 128;  // keys per CTA, queries per loop step

struct Params {
  const float* lse;     // [BH, S] natural log (forward output)
  const float* delta;   // [BH, S] rowsum(dO * O)
  __half* dK;
  __half* dV;
  uint32_t S, n_blk;
  float scale, scale_log2;
  uint32_t causal;
  unsigned* status;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// TMEM column (relative to the S^T / dP^T region) of packed fp16 query
// column q: queries [64h, 64h + 64) are packed into columns [64h, 64h + 32).
__device__ __forceinline__ uint32_t packed_col(int q) {
  return uint32_t(q & ~63) + uint32_t(q & 63) / 2;
}

template <int ROWS>
__device__ __forceinline__ uint64_t kmajor(uint32_t tile, int k) {
  return make_sdesc_sw128(tile + (uint32_t(k) >> 2) * (ROWS * 128) + (uint32_t(k) & 3u) * 32, 16,
                          1024);
}
// MN-major operand made of 64-column chunks of 128 rows (16 KB each), K step k.
__device__ __forceinline__ uint64_t mnmajor(uint32_t tile, int k) {
  return make_sdesc_sw128(tile + uint32_t(k) * 2048, kBlk * 128, 1024);
}
// The same descriptors from step 0's: the start-address field (address / 16)
// advances by the byte offset / 16 and never carries for shared memory.
template <int ROWS>
__device__ __forceinline__ uint64_t kmajor_step(uint64_t d0, int k) {
  return d0 + uint64_t(((k >> 2) * (ROWS * 128) + (k & 3) * 32) >> 4);
}
__device__ __forceinline__ uint64_t mnmajor_step(uint64_t d0, int k) {
  return d0 + uint64_t(k * (2048 >> 4));
}

// ---------------------------------------------------------------------------
// The kernel (D = 64 or 128): 128-query steps with the work of neighbouring
// steps interleaved.
//
// TMEM (512 columns, lanes = the CTA's 128 keys unless noted):
//   [0, 128)   S^T(i) fp32; P^T(i) fp16 packed into the first 32 columns of
//              each 64-query half (TS operand of dV)
//   [128, 256) dP^T(i) fp32; dS^T(i) fp16 packed the same way (TS operand of
//              dK); then dQ(i) = dS K (lanes = queries, columns = d)
//   [256, 256 + D) dV, [384, 384 + D) dK
// MMA issue order per step i:
//   dV(i) | S^T(i + 1) | dP^T(i) | dK(i) dQ(i)
// with the waits: P^T(i) ready; Q(i + 1) loaded; dQ(i - 1) read out; dS(i)
// ready. The element-wise warps run, per step:
//   dS(i) (needs dP^T(i) and P(i), kept in registers as fp16 pairs) |
//   P(i + 1) (needs S^T(i + 1)) | read-out of dQ(i) into the fp32 accumulator,
// so the exponentials of step i + 1 and the dQ read-out overlap dK(i), dQ(i)
// and dV(i + 1), S^T(i + 2).
// Warps: 0 TMA loader, 1 MMA issuer, 4-11 element-wise: two warpgroups, each
// one half of the queries (S/P/dS) and one half of d (dQ, dK, dV).
namespace pipe {

constexpr int kB = 128;  // keys per CTA, queries per step
constexpr int kThreads = 384;
constexpr int kEwWarps = 8;

template <int D>
struct PCfg {
  static constexpr int kTile = kB * D * 2;  // 32 KB at D = 128
  static constexpr int kKOff = 0;
  static constexpr int kVOff = kKOff + kTile;
  static constexpr int kQOff = kVOff + kTile;        // [2]
  static constexpr int kDOOff = kQOff + 2 * kTile;   // [2]
  // dS (rows = keys, 64-query 128-byte chunks); after the dQ MMA has read it,
  // each element-wise warp's 4 KB of it is that warp's dQ staging box
  static constexpr int kDSOff = kDOOff + 2 * kTile;
  static constexpr int kVecOff = kDSOff + kB * kB * 2;  // [2] x (lse2[128], delta[128])
  static constexpr int kBarOff = kVecOff + 2 * 2 * kB * 4;
  static constexpr int kSmemBytes = kBarOff + 256;  // no alignment slack: checked in the kernel
  static_assert(kSmemBytes <= 232448, "shared memory");
};

template <int D>
__global__ void __launch_bounds__(kThreads, 1)
    flash_attn_bwd_pipe_kernel(const __grid_constant__ CUtensorMap tmQ,
                               const __grid_constant__ CUtensorMap tmK,
                               const __grid_constant__ CUtensorMap tmV,
                               const __grid_constant__ CUtensorMap tmDO,
                               const __grid_constant__ CUtensorMap tmDQ, const Params p) {
  constexpr int kD = D;
  constexpr int kTile = PCfg<D>::kTile;
  constexpr int kKOff = PCfg<D>::kKOff, kVOff = PCfg<D>::kVOff, kQOff = PCfg<D>::kQOff;
  constexpr int kDOOff = PCfg<D>::kDOOff, kDSOff = PCfg<D>::kDSOff;
  constexpr int kVecOff = PCfg<D>::kVecOff, kBarOff = PCfg<D>::kBarOff;
  extern __shared__ __align__(1024) uint8_t smem[];
  if (smem_u32(smem) & 1023u) {  // uniform over the CTA: nobody touches a barrier
    if (threadIdx.x == 0) atomicCAS(p.status, 0u, unsigned(kWdSmemAlign));
    return;
  }
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kBarOff);
  uint64_t* kv_full = bars;         // K_j, V_j landed
  uint64_t* qdo_full = bars + 1;    // [2] Q_i, dO_i landed in stage i % 2
  uint64_t* qdo_empty = bars + 3;   // [2] MMAs of step i done with stage i % 2
  uint64_t* s_full = bars + 5;      // S^T(i) in TMEM
  uint64_t* p_ready = bars + 6;     // P^T(i) in TMEM (8 warp arrivals)
  uint64_t* dp_full = bars + 7;     // dP^T(i) in TMEM
  uint64_t* ds_ready = bars + 8;    // dS^T(i) in TMEM, dS(i) in smem (8 warp arrivals)
  uint64_t* dq_full = bars + 9;     // dQ(i) in TMEM
  uint64_t* dq_free = bars + 10;    // dQ(i) read out of TMEM (8 warp arrivals)
  uint64_t* done = bars + 11;       // every MMA complete
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 12);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  float* s_vec = reinterpret_cast<float*>(smem + kVecOff);

  const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const uint32_t bh = blockIdx.x / p.n_blk;
  const uint32_t j = blockIdx.x % p.n_blk;  // key block
  const uint32_t i0 = p.causal ? j : 0;     // first query block
  const uint32_t n = p.n_blk - i0;

  if (threadIdx.x == 0) {
    for (int b = 0; b < 12; ++b)
      mbar_init(&bars[b], (b == 6 || b == 8 || b == 10) ? kEwWarps : 1);
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
    tma_prefetch_desc(&tmDO);
    tma_prefetch_desc(&tmDQ);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  constexpr uint32_t kColS = 0, kColDP = 128, kColDV = 256, kColDK = 384;

  if (warp == 0) {
    // ---------------------------------------------------------------- loader
    if (elect_one()) {
      mbar_arrive_expect_tx(kv_full, 2 * kTile);
#pragma unroll
      for (int c = 0; c < kD / 64; ++c) {
        tma_load_3d(smem + kKOff + c * (kB * 128), &tmK, kv_full, 64 * c, int(j * kB), int(bh));
        tma_load_3d(smem + kVOff + c * (kB * 128), &tmV, kv_full, 64 * c, int(j * kB), int(bh));
      }
      uint32_t filled = 0;
      for (uint32_t s = 0; s < n; ++s) {
        const uint32_t st = s & 1u, use = s >> 1;
        if (!mbar_wait(qdo_empty + st, (use & 1u) ^ 1u, abort_flag, p.status, kWdAttnLoad)) break;
        mbar_arrive_expect_tx(qdo_full + st, 2 * kTile);
#pragma unroll
        for (int c = 0; c < kD / 64; ++c) {
          tma_load_3d(smem + kQOff + st * kTile + c * (kB * 128), &tmQ, qdo_full + st, 64 * c,
                      int((i0 + s) * kB), int(bh));
          tma_load_3d(smem + kDOOff + st * kTile + c * (kB * 128), &tmDO, qdo_full + st, 64 * c,
                      int((i0 + s) * kB), int(bh));
        }
        ++filled;
      }
      // drain: the last load of each stage has landed
      int dummy = 0;
      mbar_wait(kv_full, 0, &dummy, p.status, kWdDrain, 100000000ull);
      for (uint32_t s = filled > 2 ? filled - 2 : 0; s < filled; ++s)
        mbar_wait(qdo_full + (s & 1u), (s >> 1) & 1u, &dummy, p.status, kWdDrain, 100000000ull);
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------------- MMA issuer
    // The whole warp runs the loop converged (every lane waits, the lanes
    // agree on the outcome); one elected lane issues the MMAs and commits.
    {
      auto wait_all = [&](uint64_t* bar, uint32_t parity) {
        return __all_sync(0xffffffffu,
                          mbar_wait(bar, parity, abort_flag, p.status, kWdAttnMma)) != 0;
      };
      const uint32_t id_st = make_idesc_f16_f32(kB, kB, false, false);  // S^T, dP^T
      const uint32_t id_acc = make_idesc_f16_f32(kB, kD, false, true);  // dV, dK
      const uint32_t id_dq = make_idesc_f16_f32(kB, kD, true, true);    // dQ
      const uint32_t sK = smem_u32(smem + kKOff), sV = smem_u32(smem + kVOff);
      const uint32_t sDS = smem_u32(smem + kDSOff);
      long long tr_qdo = 0, tr_dqf = 0, tr_pr = 0;
      (void)tr_qdo; (void)tr_dqf; (void)tr_pr;
      BWD_TR_BEGIN(tr_total);
      auto sq = [&](uint32_t s) { return smem_u32(smem + kQOff + (s & 1u) * kTile); };
      auto sdo = [&](uint32_t s) { return smem_u32(smem + kDOOff + (s & 1u) * kTile); };
      auto issue_s = [&](uint32_t s) -> bool {
        BWD_TR_BEGIN(t0);
        if (!wait_all(qdo_full + (s & 1u), (s >> 1) & 1u)) return false;
        BWD_TR_ACC(tr_qdo, t0);
        tc_fence_after();
        if (elect_one()) {
          const uint64_t a0 = kmajor<kB>(sK, 0), b0 = kmajor<kB>(sq(s), 0);
#pragma unroll
          for (int k = 0; k < kD / 16; ++k)
            if (!(FELIX_FA_BWD_EXP_SKIP & 1))
              umma_f16_ss(tmem + kColS, kmajor_step<kB>(a0, k), kmajor_step<kB>(b0, k), id_st,
                          k > 0 ? 1u : 0u);
          umma_commit(s_full);
        }
        __syncwarp();
        return true;
      };
      bool ok = wait_all(kv_full, 0) && issue_s(0);
      for (uint32_t i = 0; ok && i < n; ++i) {
        BWD_TR_BEGIN(t1);
        if (!(ok = wait_all(p_ready, i & 1u))) break;
        BWD_TR_ACC(tr_pr, t1);
        tc_fence_after();
        if (elect_one()) {
          const uint64_t b0 = mnmajor(sdo(i), 0);
#pragma unroll
          for (int k = 0; k < kB / 16; ++k)
            if (!(FELIX_FA_BWD_EXP_SKIP & 4))
              umma_f16_ts(tmem + kColDV, tmem + kColS + packed_col(16 * k), mnmajor_step(b0, k),
                          id_acc, (i > 0 || k > 0) ? 1u : 0u);
        }
        __syncwarp();
        if (i + 1 < n && !(ok = issue_s(i + 1))) break;
        // dQ(i - 1) sits in the dP^T columns until it has been read out
        BWD_TR_BEGIN(t2);
        if (i > 0 && !(ok = wait_all(dq_free, (i - 1) & 1u))) break;
        BWD_TR_ACC(tr_dqf, t2);
        tc_fence_after();
        if (elect_one()) {
          const uint64_t a0 = kmajor<kB>(sV, 0), b0 = kmajor<kB>(sdo(i), 0);
#pragma unroll
          for (int k = 0; k < kD / 16; ++k)
            if (!(FELIX_FA_BWD_EXP_SKIP & 2))
              umma_f16_ss(tmem + kColDP, kmajor_step<kB>(a0, k), kmajor_step<kB>(b0, k), id_st,
                          k > 0 ? 1u : 0u);
          umma_commit(dp_full);
        }
        __syncwarp();
        BWD_TR_BEGIN(t3);
        if (!(ok = wait_all(ds_ready, i & 1u))) break;
        BWD_TR_ACC(tr_pr, t3);
        tc_fence_after();
        if (elect_one()) {
          const uint64_t b0 = mnmajor(sq(i), 0);
#pragma unroll
          for (int k = 0; k < kB / 16; ++k)
            if (!(FELIX_FA_BWD_EXP_SKIP & 8))
              umma_f16_ts(tmem + kColDK, tmem + kColDP + packed_col(16 * k), mnmajor_step(b0, k),
                          id_acc, (i > 0 || k > 0) ? 1u : 0u);
          const uint64_t a1 = mnmajor(sDS, 0), b1 = mnmajor(sK, 0);
#pragma unroll
          for (int k = 0; k < kB / 16; ++k)
            if (!(FELIX_FA_BWD_EXP_SKIP & 16))
              umma_f16_ss(tmem + kColDP, mnmajor_step(a1, k), mnmajor_step(b1, k), id_dq,
                          k > 0 ? 1u : 0u);
          umma_commit(qdo_empty + (i & 1u));
          umma_commit(dq_full);
        }
        __syncwarp();
      }
      if (elect_one()) umma_commit(done);
      __syncwarp();
      int dummy = 0;
      mbar_wait(done, 0, &dummy, p.status, kWdDrain, 100000000ull);
      long long tr_all = 0;
      (void)tr_all;
      BWD_TR_ACC(tr_all, tr_total);
      if (lane == 0) {
        BWD_TR_FLUSH(0, tr_qdo);
        BWD_TR_FLUSH(1, tr_dqf);
        BWD_TR_FLUSH(2, tr_pr);
        BWD_TR_FLUSH(3, tr_all);
        BWD_TR_FLUSH(15, 1);
      }
    }
  } else if (warp >= 4) {
    // ---------------------------------------------------------------- element-wise
    const uint32_t q4 = warp & 3u;        // TMEM lane quadrant
    const uint32_t g = (warp - 4) >> 2;   // queries [64g, 64g + 64); d [64g, 64g + 64)
    const uint32_t r = q4 * 32 + lane;    // key row (S/P/dS) or query row (dQ)
    const uint32_t key = j * kB + r;
    const uint32_t la = (q4 * 32u) << 16;
    const uint32_t tid = threadIdx.x - 128;
    const bool key_ok = key < p.S;
    const float sl2 = p.scale_log2;
    uint8_t* sDS = smem + kDSOff;
    uint8_t* stg = sDS + (g * 4 + q4) * 4096;  // this warp's 4 KB of dS = dQ staging box
    const int c0 = int(g) * 64;        // this warpgroup's 64 queries of a step
    const int dc0 = int(g) * (kD / 2);  // its half of d (dQ read-out, dK, dV)
    // threads 0..127 fetch lse * log2(e), 128..255 Delta, one step ahead
    auto fetch_vec = [&](uint32_t s) -> float {
      const uint32_t q = (i0 + s) * kB + (tid & (kB - 1));
      if (tid < kB)
        return q < p.S ? __ldg(p.lse + size_t(bh) * p.S + q) * 1.4426950408889634f : INFINITY;
      return q < p.S ? __ldg(p.delta + size_t(bh) * p.S + q) : 0.f;
    };
    float vec_next = fetch_vec(0);
    uint32_t pk[32];  // P(i) of this thread's key row and 64 queries, fp16 pairs
    bool ok = true;
    long long tr_bar = 0, tr_st = 0, tr_ld = 0, tr_math = 0, tr_tst = 0, tr_sts = 0;
    (void)tr_bar; (void)tr_st; (void)tr_ld; (void)tr_math; (void)tr_tst; (void)tr_sts;
    BWD_TR_BEGIN(tr_total);

    // P(s) = exp2(S^T * scale * log2 e - lse2): registers and TMEM (P^T operand)
    auto p_phase = [&](uint32_t s) -> bool {
      const uint32_t qb = (i0 + s) * kB;
      float* s_lse2 = s_vec + (s & 1u) * (2 * kB);
      BWD_TR_BEGIN(t0);
      s_lse2[tid] = vec_next;  // Delta follows lse2 in the same buffer
      if (s + 1 < n) vec_next = fetch_vec(s + 1);
      named_barrier_sync(1, kEwWarps * 32);
      BWD_TR_ACC(tr_bar, t0);
      BWD_TR_BEGIN(t1);
      if (!mbar_wait(s_full, s & 1u, abort_flag, p.status, kWdAttnSoftmax)) return false;
      BWD_TR_ACC(tr_st, t1);
      tc_fence_after();
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int c = c0 + 32 * h;
        uint32_t sr[32];
        tmem_ld_32x32b_x32(tmem + la + kColS + c, sr);
        tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < 32; e += 4) {
          const float4 l4 = *reinterpret_cast<const float4*>(s_lse2 + c + e);
          const float lv[4] = {l4.x, l4.y, l4.z, l4.w};
          float pv[4];
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            float pr = ex2(fmaf(__uint_as_float(sr[e + x]), sl2, -lv[x]));
            if (!key_ok || (p.causal && qb + uint32_t(c + e + x) < key)) pr = 0.f;
            pv[x] = pr;
          }
          pk[16 * h + e / 2] = pack_half2(pv[0], pv[1]);
          pk[16 * h + e / 2 + 1] = pack_half2(pv[2], pv[3]);
        }
      }
      // packed P^T: this warpgroup's 64 queries into its first 32 columns
      // (columns it has already read)
      tmem_st_32x32b_x16(tmem + la + kColS + packed_col(c0), *reinterpret_cast<uint32_t(*)[16]>(pk));
      tmem_st_32x32b_x16(tmem + la + kColS + packed_col(c0) + 16,
                         *reinterpret_cast<uint32_t(*)[16]>(pk + 16));
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(p_ready);
      return true;
    };

    ok = p_phase(0);
    for (uint32_t i = 0; ok && i < n; ++i) {
      // ---- dS(i) = P(i) * (dP^T(i) - Delta)
      const float* s_delta = s_vec + (i & 1u) * (2 * kB) + kB;
      BWD_TR_BEGIN(t1);
      if (!(ok = mbar_wait(dp_full, i & 1u, abort_flag, p.status, kWdAttnSoftmax))) break;
      BWD_TR_ACC(tr_st, t1);
      tc_fence_after();
      // the dS writes reuse the staging box: its reductions must have read it
      if (lane == 0) bulk_wait_group_read<0>();
      __syncwarp();
      BWD_TR_BEGIN(t2);
      uint32_t dk[32];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int c = c0 + 32 * h;
        uint32_t dr[32];
        tmem_ld_32x32b_x32(tmem + la + kColDP + c, dr);
        tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < 32; e += 4) {
          const float4 d4 = *reinterpret_cast<const float4*>(s_delta + c + e);
          const float2 p01 = __half22float2(*reinterpret_cast<const __half2*>(&pk[16 * h + e / 2]));
          const float2 p23 =
              __half22float2(*reinterpret_cast<const __half2*>(&pk[16 * h + e / 2 + 1]));
          dk[16 * h + e / 2] = pack_half2(p01.x * (__uint_as_float(dr[e]) - d4.x),
                                          p01.y * (__uint_as_float(dr[e + 1]) - d4.y));
          dk[16 * h + e / 2 + 1] = pack_half2(p23.x * (__uint_as_float(dr[e + 2]) - d4.z),
                                              p23.y * (__uint_as_float(dr[e + 3]) - d4.w));
        }
      }
      BWD_TR_ACC(tr_math, t2);
      BWD_TR_BEGIN(t3);
      tmem_st_32x32b_x16(tmem + la + kColDP + packed_col(c0), *reinterpret_cast<uint32_t(*)[16]>(dk));
      tmem_st_32x32b_x16(tmem + la + kColDP + packed_col(c0) + 16,
                         *reinterpret_cast<uint32_t(*)[16]>(dk + 16));
      // dS (queries x keys) as an MN-major A tile: query chunk g, row = key r,
      // 16-byte units swizzled with the row (128-byte swizzle)
      uint8_t* row = sDS + g * (kB * 128) + r * 128;
#pragma unroll
      for (int u = 0; u < 8; ++u)
        *reinterpret_cast<uint4*>(row + ((uint32_t(u) ^ (r & 7u)) * 16)) =
            make_uint4(dk[4 * u], dk[4 * u + 1], dk[4 * u + 2], dk[4 * u + 3]);
      tmem_st_wait();
      fence_proxy_async_smem();
      tc_fence_before();
      __syncwarp();
      BWD_TR_ACC(tr_tst, t3);
      if (lane == 0) mbar_arrive(ds_ready);
      // ---- P(i + 1)
      if (i + 1 < n && !(ok = p_phase(i + 1))) break;
      // ---- dQ(i) (lane = query, columns d [64g, 64g + 64)) -> staged 32 x 32
      // boxes -> TMA reduction into the fp32 accumulator
      BWD_TR_BEGIN(t4);
      if (!(ok = mbar_wait(dq_full, i & 1u, abort_flag, p.status, kWdAttnSoftmax))) break;
      BWD_TR_ACC(tr_sts, t4);
      tc_fence_after();
      constexpr int kBoxes = kD / 64;  // 32-column boxes per warpgroup
      uint32_t v0[32], v1[32];
      tmem_ld_32x32b_x32(tmem + la + kColDP + dc0, v0);
      if constexpr (kBoxes > 1) tmem_ld_32x32b_x32(tmem + la + kColDP + dc0 + 32, v1);
      tmem_ld_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(dq_free);
      const uint32_t q0 = (i0 + i) * kB + q4 * 32;
#pragma unroll
      for (int bx = 0; bx < kBoxes; ++bx) {
        const uint32_t(&v)[32] = bx ? v1 : v0;
        if (bx) {
          if (lane == 0) bulk_wait_group_read<0>();
          __syncwarp();
        }
#pragma unroll
        for (int u = 0; u < 8; ++u)
          *reinterpret_cast<uint4*>(stg + lane * 128 + ((uint32_t(u) ^ (lane & 7u)) * 16)) =
              make_uint4(v[4 * u], v[4 * u + 1], v[4 * u + 2], v[4 * u + 3]);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          if (q0 < p.S && !FELIX_FA_BWD_EXP_NO_DQRED)
            tma_reduce_add_3d(&tmDQ, stg, dc0 + 32 * bx, int(q0), int(bh));
          bulk_commit_group();
        }
      }
    }
    if (lane == 0 && warp == 4) {
      long long tr_all = 0;
      (void)tr_all;
      BWD_TR_ACC(tr_all, tr_total);
      BWD_TR_FLUSH(4, tr_bar);
      BWD_TR_FLUSH(5, tr_st);
      BWD_TR_FLUSH(6, tr_all);
      BWD_TR_FLUSH(11, tr_math);
      BWD_TR_FLUSH(12, tr_tst);
      BWD_TR_FLUSH(13, tr_sts);
    }
    // dK_j, dV_j (lane = key) -> fp16, columns [64g, 64g + 64)
    if (ok && mbar_wait(done, 0, abort_flag, p.status, kWdAttnSoftmax)) {
      tc_fence_after();
#pragma unroll 1
      for (int which = 0; which < 2; ++which) {
        const uint32_t col = which ? kColDK : kColDV;
        const float mul = which ? p.scale : 1.f;
        __half* out = (which ? p.dK : p.dV) + (size_t(bh) * p.S + key) * kD;
#pragma unroll 1
        for (int c = dc0; c < dc0 + kD / 2; c += 32) {
          uint32_t v[32];
          tmem_ld_32x32b_x32(tmem + la + col + c, v);
          tmem_ld_wait();
          if (key_ok) {
            uint4 o4[4];
            uint32_t* o = reinterpret_cast<uint32_t*>(o4);
#pragma unroll
            for (int e = 0; e < 16; ++e)
              o[e] = pack_half2(__uint_as_float(v[2 * e]) * mul, __uint_as_float(v[2 * e + 1]) * mul);
#pragma unroll
            for (int e = 0; e < 4; ++e) reinterpret_cast<uint4*>(out + c)[e] = o4[e];
          }
        }
      }
    }
    // every staged reduction complete before the shared memory goes away
    if (lane == 0) bulk_wait_group<0>();
    __syncwarp();
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace pipe

// Delta[row] = sum_d dO[row, d] * O[row, d] (fp32), one warp per row.
__global__ void delta_kernel(const __half* __restrict__ O, const __half* __restrict__ dO,
                             float* __restrict__ delta, uint64_t rows, uint32_t D) {
  const uint64_t row = (uint64_t(blockIdx.x) * blockDim.x + threadIdx.x) / 32;
  const uint32_t lane = threadIdx.x % 32;
  if (row >= rows) return;
  const __half2* o = reinterpret_cast<const __half2*>(O + row * D);
  const __half2* g = reinterpret_cast<const __half2*>(dO + row * D);
  float acc = 0.f;
  for (uint32_t k = lane; k < D / 2; k += 32) {
    const float2 a = __half22float2(o[k]), b = __half22float2(g[k]);
    acc = fmaf(a.x, b.x, fmaf(a.y, b.y, acc));
  }
#pragma unroll
  for (int off = 16; off; off >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, off);
  if (lane == 0) delta[row] = acc;
}

__global__ void dq_convert_kernel(const float* __restrict__ acc, __half* __restrict__ dQ, size_t n,
                                  float scale) {
  for (size_t i = (blockIdx.x * size_t(blockDim.x) + threadIdx.x) * 4; i < n;
       i += size_t(gridDim.x) * blockDim.x * 4) {
    const float4 v = *reinterpret_cast<const float4*>(acc + i);
    reinterpret_cast<__half2*>(dQ + i)[0] = __floats2half2_rn(v.x * scale, v.y * scale);
    reinterpret_cast<__half2*>(dQ + i)[1] = __floats2half2_rn(v.z * scale, v.w * scale);
  }
}

}  // namespace attn_bwd
}  // namespace felix_sm100

namespace felix_impl {

using namespace felix_sm100::attn_bwd;

namespace {
template <int D>
int configure_bwd_pipe(int device) {
  static PerDeviceOnce once;
  return once.run(device, [] {
    return int(cudaFuncSetAttribute(pipe::flash_attn_bwd_pipe_kernel<D>,
                                    cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    pipe::PCfg<D>::kSmemBytes));
  });
}

}  // namespace

size_t flash_attn_bwd_workspace_bytes(uint32_t heads, uint32_t batch, uint32_t seqlen,
                                      uint32_t head_dim) {
  const size_t rows = size_t(heads) * batch * seqlen;
  return kWsCounterBytes + rows * 4 + 16 + rows * head_dim * 4;
}

FelixCode flash_attn_bwd_launch(const __half* Q, const __half* K, const __half* V,
                                const __half* O, const __half* dO, const float* lse, __half* dQ,
                                __half* dK, __half* dV, uint32_t heads, uint32_t batch,
                                uint32_t seqlen, uint32_t head_dim, float scale, bool causal,
                                void* workspace, size_t ws_bytes, cudaStream_t stream) {
  if (head_dim != 64 && head_dim != 128)
    return api_error("flash_attn_bwd: head_dim must be 64 or 128");
  if (heads == 0 || batch == 0 || seqlen == 0) return FelixCode{FELIX_SUCCESS, cudaSuccess};
  if (!Q || !K || !V || !O || !dO || !lse || !dQ || !dK || !dV)
    return api_error("flash_attn_bwd: null pointer");
  if ((reinterpret_cast<uintptr_t>(Q) | reinterpret_cast<uintptr_t>(K) |
       reinterpret_cast<uintptr_t>(V) | reinterpret_cast<uintptr_t>(O) |
       reinterpret_cast<uintptr_t>(dO) | reinterpret_cast<uintptr_t>(dQ) |
       reinterpret_cast<uintptr_t>(dK) | reinterpret_cast<uintptr_t>(dV)) & 15u)
    return api_error("flash_attn_bwd: tensors must be 16-byte aligned");
  const uint64_t bh = uint64_t(heads) * batch;
  if (bh > (1u << 31) || seqlen > (1u << 30)) return api_error("flash_attn_bwd: too large");
  DeviceInfo* dev = current_device_info();
  if (!dev) return launch_error(cudaGetLastError(), "flash_attn_bwd: no CUDA device");

  const size_t rows = size_t(bh) * seqlen;
  const size_t need = flash_attn_bwd_workspace_bytes(heads, batch, seqlen, head_dim);
  Workspace scratch;  // until the last launch
  if (!workspace) {
    scratch = library_workspace(dev, stream, need);
    workspace = scratch.ptr;
    if (!workspace) return launch_error(cudaErrorMemoryAllocation, "flash_attn_bwd: workspace");
  } else if (ws_bytes < need) {
    return api_error("flash_attn_bwd: workspace too small");
  }
  float* delta = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + kWsCounterBytes);
  float* dq_acc = delta + rows;  // 16-byte aligned: rows * 4 bytes after a 16 KiB block
  if ((reinterpret_cast<uintptr_t>(dq_acc) & 15u) != 0) {
    dq_acc = reinterpret_cast<float*>((reinterpret_cast<uintptr_t>(dq_acc) + 15) & ~uintptr_t(15));
  }

  CUtensorMap tq, tk, tv, tdo, tdq;
  auto enc = [&](CUtensorMap* m, const void* base, uint32_t rows) {
    return encode_tmap_3d_f16(m, base, head_dim, seqlen, bh, uint64_t(head_dim) * 2,
                              uint64_t(seqlen) * head_dim * 2, 64, rows, 1);
  };
  if (enc(&tq, Q, kBlk) || enc(&tk, K, kBlk) || enc(&tv, V, kBlk) || enc(&tdo, dO, kBlk) ||
      encode_tmap_3d_f32(&tdq, dq_acc, head_dim, seqlen, bh, uint64_t(head_dim) * 4,
                         uint64_t(seqlen) * head_dim * 4, 32, 32, 1))
    return api_error("flash_attn_bwd: cuTensorMapEncodeTiled failed");

  cudaError_t e = cudaMemsetAsync(dq_acc, 0, rows * head_dim * 4, stream);
  if (e != cudaSuccess) return launch_error(e, "flash_attn_bwd: clearing dQ accumulator");
  delta_kernel<<<unsigned((rows * 32 + 255) / 256), 256, 0, stream>>>(O, dO, delta, rows,
                                                                     head_dim);

  Params p{};
  p.lse = lse;
  p.delta = delta;
  p.dK = dK;
  p.dV = dV;
  p.S = seqlen;
  p.n_blk = (seqlen + kBlk - 1) / kBlk;
  p.scale = scale > 0.f ? scale : 1.0f / sqrtf(float(head_dim));
  p.scale_log2 = p.scale * 1.4426950408889634f;
  p.causal = causal ? 1u : 0u;
  p.status = dev->status_word;
  const uint64_t grid = bh * p.n_blk;
  if (grid > 0x7fffffffull) return api_error("flash_attn_bwd: grid too large");
  int rc;
  if (head_dim == 128) {
    if ((rc = configure_bwd_pipe<128>(dev->ordinal)))
      return FelixCode{FELIX_API_ERROR, cudaError_t(rc)};
    pipe::flash_attn_bwd_pipe_kernel<128><<<unsigned(grid), pipe::kThreads,
                                            pipe::PCfg<128>::kSmemBytes, stream>>>(tq, tk, tv,
                                                                                   tdo, tdq, p);
  } else {
    if ((rc = configure_bwd_pipe<64>(dev->ordinal)))
      return FelixCode{FELIX_API_ERROR, cudaError_t(rc)};
    pipe::flash_attn_bwd_pipe_kernel<64><<<unsigned(grid), pipe::kThreads,
                                           pipe::PCfg<64>::kSmemBytes, stream>>>(tq, tk, tv, tdo,
                                                                                 tdq, p);
  }
  dq_convert_kernel<<<592, 256, 0, stream>>>(dq_acc, dQ, rows * head_dim, p.scale);
  e = cudaGetLastError();
  if (e != cudaSuccess) return launch_error(e, "flash_attn_bwd: launch failed");
  return FelixCode{FELIX_SUCCESS, cudaSuccess};
}

}  // namespace felix_impl

#if FELIX_FA_BWD_TRACE
extern "C" int felix_debug_bwd_trace(unsigned long long* out16, int clear) {
  if (cudaMemcpyFromSymbol(out16, g_bwd_trace,
                           sizeof(unsigned long long) * 16) != cudaSuccess)
    return 1;
  if (clear) {
    unsigned long long z[16] = {0};
    cudaMemcpyToSymbol(g_bwd_trace, z, sizeof(z));
  }
  return 0;
}
#endif
