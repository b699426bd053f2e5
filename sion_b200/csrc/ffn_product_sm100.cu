// Products of the feed-forward operators on tcgen05, fp16 or bf16 in, fp32 accumulators
// in TMEM, everything that follows a product done on them before they are rounded once:
//   kLinear  act(x W^T + bias) + residual, and the value in front of the activation
//   kGated   both projections of a gated block: gate and up accumulate side by side in
//            TMEM, so that one thread holds both of an element: act(g) u
//   kDGated  dh = dy Wd never leaves the SM: dg, du and h are written from it
//
// Tiles. CG = 2: a CTA pair (cta_group::2) computes 256 x 256, each CTA loading 128
// rows of A and 128 of B per stage and holding 128 rows of the tile in its TMEM; for
// kGated one CTA's 128 rows of B are the gate's and the other's the up projection's.
// CG = 1: 128 x 128, for products of few tiles. A stage is 128 deep: 32 KB per operand
// (one request where the tensor map can say it, two of 16 KB where a size is no multiple
// of 64), three stages. Two accumulators, so that the epilogue of a tile overlaps the
// next tile's products. An operand may be stored with k or with m / n contiguous: the
// three products of a training step need x W^T, dz W and dz^T x, without a transpose.
//
// Warps: 0 TMA, 1 MMA, 2-9 epilogue (two per quarter of the TMEM lanes, each with half
// the columns: activations cost 10 to 50 instructions a value).
//
// Schedule: persistent; the tiles of an incomplete last wave are cut along k in equal
// parts, first of all, and finished by the last contributor in the order of the parts
// (repeatable); from four waves on whole tiles are handed out at run time (tile_queue.cuh).
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "activation.cuh"
#include "ffn_internal.h"
#include "sm100_ptx.cuh"
#include "tile_queue.cuh"

namespace felix_ffn {
namespace product {

using namespace felix_sm100;

constexpr uint32_t kRows = 128;               // rows of A, and of B, of one CTA's stage
constexpr uint32_t kDepth = 128;              // k of a stage
constexpr uint32_t kOpBytes = kRows * kDepth * 2;
constexpr uint32_t kStageBytes = 2 * kOpBytes;
constexpr uint32_t kStages = 3;
constexpr uint32_t kEpiWarps = 8;
constexpr uint32_t kThreads = 64 + 32 * kEpiWarps;
constexpr uint32_t kBoxBytes = 32 * 64;       // 32 rows x 32 columns
constexpr uint32_t kStagingBytes = kEpiWarps * 2 * kBoxBytes;
constexpr uint32_t kBarBytes = 512;
constexpr uint32_t kSmemBytes = kStages * kStageBytes + kStagingBytes + kBarBytes + 1024;

struct Problem {
  uint32_t m, n, tiles_m, tiles_n, tile0;
};

struct alignas(64) Params {
  CUtensorMap a[3], b[3], out[3];
  Problem prob[3];
  uint32_t problems, tiles;
  uint32_t kb_seg, kb;         // 128-deep blocks of a segment, of a tile
  uint32_t a_mn, b_mn;         // operands stored with m / n contiguous
  uint32_t a_3d, b_3d;         // one request per operand and stage
  uint32_t group_m;
  uint32_t split_tiles, parts; // the first tiles, cut into `parts` along k
  uint32_t dyn;                // whole tiles come from the queue
  void* out_ptr[3];
  int64_t out_ld[3];
  uint32_t out_tma, out_want;  // bit per output
  const void* in_ptr[2];
  int64_t in_ld[2];
  uint32_t in_vec;             // bit per input: rows of whole 16-byte vectors
  const void* bias;
  int act;
  unsigned* counters;          // [split tiles x CG], zero between launches
  unsigned* dyn_counter;       // [0] next whole tile, [1] CTAs that are done
  float* partials;             // [unit][CG][128 x 128 CG]
  unsigned* status;
};

struct Unit {
  uint32_t tile, kb0, kb1;
  bool split;
};

// The walk of every role of a CTA: its part of a split tile, then whole tiles.
struct Walk {
  uint32_t unit, units, next_tile;
  bool first;
  __device__ __forceinline__ void init(const Params& p, uint32_t cg) {
    unit = blockIdx.x / cg;
    units = gridDim.x / cg;
    first = unit < p.split_tiles * p.parts;
    next_tile = p.split_tiles + unit;
  }
  __device__ __forceinline__ static void whole(const Params& p, Unit& u, uint32_t tile) {
    u = {tile, 0, p.kb, false};
  }
  __device__ __forceinline__ bool next(const Params& p, Unit& u) {
    if (first) {
      first = false;
      const uint32_t part = unit % p.parts;
      u = {unit / p.parts, p.kb * part / p.parts, p.kb * (part + 1) / p.parts, true};
      return true;
    }
    if (p.dyn || next_tile >= p.tiles) return false;
    whole(p, u, next_tile);
    next_tile += units;
    return true;
  }
};

struct Place {
  uint32_t prob, tm, tn;
};
// Grouped raster: runs of group_m tiles along m sweep across n, so that CTAs that run
// together share panels of A and B in the L2.
__device__ __forceinline__ Place place_of(const Params& p, uint32_t tile) {
  Place r{0, 0, 0};
  while (r.prob + 1 < p.problems && tile >= p.prob[r.prob + 1].tile0) ++r.prob;
  const Problem& q = p.prob[r.prob];
  const uint32_t t = tile - q.tile0, per_group = p.group_m * q.tiles_n, g = t / per_group;
  const uint32_t m0 = g * p.group_m, gm = min(p.group_m, q.tiles_m - m0), i = t - g * per_group;
  r.tm = m0 + i % gm;
  r.tn = i / gm;
  return r;
}

// float4 of (32-column chunk c, float4 j of it, row r) of a partial tile: a warp's rows
// touch 512 contiguous bytes.
__device__ __forceinline__ uint32_t partial_index(uint32_t c, uint32_t j, uint32_t r) {
  return (c * 8 + j) * kRows + r;
}

// 32 columns of one row of an input, as 16 packed pairs; what lies outside reads as 0.
// Rows that are no whole vectors go through the warp's staging, 64 bytes a row.
template <class T>
__device__ __forceinline__ void load_chunk(const Params& p, int which, uint32_t row0, uint32_t col,
                                           uint32_t M, uint32_t N, uint8_t* stg, uint32_t lane,
                                           uint32_t (&raw)[16]) {
  const uint16_t* base = static_cast<const uint16_t*>(p.in_ptr[which]);
  const int64_t ld = p.in_ld[which];
  if (p.in_vec >> which & 1) {
    const uint32_t row = row0 + lane;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint4 v = make_uint4(0, 0, 0, 0);
      if (row < M && col + 8 * j < N)
        v = *reinterpret_cast<const uint4*>(base + int64_t(row) * ld + col + 8 * j);
      raw[4 * j] = v.x, raw[4 * j + 1] = v.y, raw[4 * j + 2] = v.z, raw[4 * j + 3] = v.w;
    }
    return;
  }
  if (lane == 0) bulk_wait_group_read<0>();
  __syncwarp();
  uint16_t* s = reinterpret_cast<uint16_t*>(stg);
  const uint32_t rows = min(32u, M - row0);
#pragma unroll 8
  for (uint32_t r = 0; r < rows; ++r)
    s[r * 32 + lane] = col + lane < N ? base[int64_t(row0 + r) * ld + col + lane] : uint16_t(0);
  __syncwarp();
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint4 v = reinterpret_cast<const uint4*>(stg + lane * 64)[j];
    raw[4 * j] = v.x, raw[4 * j + 1] = v.y, raw[4 * j + 2] = v.z, raw[4 * j + 3] = v.w;
  }
  __syncwarp();
}

// Rounds 32 columns of each of the warp's rows and writes them: through a 64-byte
// swizzled box and TMA, which clips the ragged edge, or, where rows are not 16-byte
// multiples, row by row. `turn` alternates between the warp's two boxes.
template <class T>
__device__ __forceinline__ void store_chunk(const Params& p, int which, uint32_t row0, uint32_t col,
                                            uint32_t M, uint32_t N, uint8_t* stg, uint32_t& turn,
                                            uint32_t lane, const float (&v)[32]) {
  uint8_t* box = stg + (turn++ & 1) * kBoxBytes;
  if (lane == 0) bulk_wait_group_read<1>();
  __syncwarp();
#pragma unroll
  for (uint32_t j = 0; j < 4; ++j) {
    uint4 w;
    w.x = Pair<T>::pack(v[8 * j], v[8 * j + 1]);
    w.y = Pair<T>::pack(v[8 * j + 2], v[8 * j + 3]);
    w.z = Pair<T>::pack(v[8 * j + 4], v[8 * j + 5]);
    w.w = Pair<T>::pack(v[8 * j + 6], v[8 * j + 7]);
    *reinterpret_cast<uint4*>(box + lane * 64 + ((j ^ ((lane >> 1) & 3)) * 16)) = w;
  }
  if (p.out_tma >> which & 1) {
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) {
      tma_store_2d(&p.out[which], box, int(col), int(row0));
      bulk_commit_group();
    }
  } else {
    __syncwarp();
    uint16_t* base = static_cast<uint16_t*>(p.out_ptr[which]);
    const int64_t ld = p.out_ld[which];
    const uint32_t rows = min(32u, M - row0);
    if (col + lane < N) {
#pragma unroll 8
      for (uint32_t r = 0; r < rows; ++r)
        base[int64_t(row0 + r) * ld + col + lane] = *reinterpret_cast<const uint16_t*>(
            box + r * 64 + (((lane >> 3) ^ ((r >> 1) & 3)) * 16) + (lane & 7) * 2);
    }
    if (lane == 0) bulk_commit_group();  // an empty one: the boxes' turns are counted in groups
  }
}

// Bias of 32 columns (the same for every row: one broadcast load each).
template <class T>
__device__ __forceinline__ void add_bias(const Params& p, uint32_t col, uint32_t N, float (&v)[32]) {
  const uint16_t* b = static_cast<const uint16_t*>(p.bias) + col;
  if (col + 32 <= N && (reinterpret_cast<uintptr_t>(b) & 15) == 0) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint4 w = __ldg(reinterpret_cast<const uint4*>(b) + j);
      const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = Pair<T>::unpack(x[i]);
        v[8 * j + 2 * i] += f.x;
        v[8 * j + 2 * i + 1] += f.y;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (col + i < N) v[i] += Pair<T>::to_float(__ldg(b + i));
  }
}

template <class T, int EPI, int CG>
__global__ void __launch_bounds__(kThreads, 1)
    ffn_product_kernel(const __grid_constant__ Params p) {
  constexpr uint32_t BN = kRows * CG;   // columns of a tile's accumulator
  constexpr uint32_t kTmemCols = 2 * BN;
  const uint32_t rank = CG == 2 ? cluster_ctarank() : 0u;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  uint8_t* staging = ring + kStages * kStageBytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(staging + kStagingBytes);
  uint64_t* full = bars;
  uint64_t* empty = full + kStages;
  uint64_t* tfull = empty + kStages;
  uint64_t* tempty = tfull + 2;
  uint64_t* drain = tempty + 2;
  uint64_t* tq_full = drain + 1;
  uint64_t* tq_empty = tq_full + kTq;
  uint32_t* words = reinterpret_cast<uint32_t*>(tq_empty + kTq);
  static_assert((2 * kStages + 5 + 2 * kTq) * 8 + (kTq + 3) * 4 <= kBarBytes, "barrier block");
  TileQueue tq{words, tq_full, tq_empty, 0};
  uint32_t* tmem_slot = words + kTq;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(words + kTq + 1);
  uint32_t* bcast = words + kTq + 2;

  const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  if (threadIdx.x == 0) {
    for (uint32_t i = 0; i < kStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&tfull[i], 1);
      mbar_init(&tempty[i], kEpiWarps * CG);  // a pair's leader counts both CTAs' warps
    }
    mbar_init(drain, 1);
    for (uint32_t i = 0; i < kTq; ++i) {
      mbar_init(&tq_full[i], 1);
      // the MMA warp and the epilogue warps; of the peer its producer and epilogue warps
      mbar_init(&tq_empty[i], CG * (kEpiWarps + 1));
    }
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&p.a[0]);
    tma_prefetch_desc(&p.b[0]);
  }
  if (CG == 2) cluster_sync();  // the peer uses this CTA's barriers
  if (warp == 1) {
    if constexpr (CG == 2) {
      tmem_alloc_pair(tmem_slot, kTmemCols);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(tmem_slot, kTmemCols);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    if (elect_one()) {
      Walk walk;
      walk.init(p, CG);
      Unit u;
      uint32_t stage = 0, phase = 0, filled = 0;
      bool ok = true;
      // loads of a pair's CTAs complete on the leader's barrier
      auto load2 = [&](uint8_t* dst, const CUtensorMap* map, uint64_t* bar, uint32_t x, uint32_t y) {
        if constexpr (CG == 2)
          tma_load_2d_pair(dst, map, mapa_shared(smem_u32(bar), 0), int(x), int(y));
        else
          tma_load_2d(dst, map, bar, int(x), int(y));
      };
      auto load3 = [&](uint8_t* dst, const CUtensorMap* map, uint64_t* bar, uint32_t y, uint32_t z) {
        if constexpr (CG == 2)
          tma_load_3d_pair(dst, map, mapa_shared(smem_u32(bar), 0), 0, int(y), int(z));
        else
          tma_load_3d(dst, map, bar, 0, int(y), int(z));
      };
      // 128 rows (of m or n, from mn0) of 128-deep block kb: two blocks of 64 k, or of 64
      // m / n, 16 KB each
      auto load = [&](uint8_t* dst, const CUtensorMap* map, uint64_t* bar, bool mn, bool whole,
                      uint32_t mn0, uint32_t kb) {
        if (whole) {
          if (mn)
            load3(dst, map, bar, kb * kDepth, mn0 / 64);
          else
            load3(dst, map, bar, mn0, kb * 2);
        } else {
#pragma unroll
          for (uint32_t j = 0; j < 2; ++j) {
            if (mn)
              load2(dst + j * (kOpBytes / 2), map, bar, mn0 + 64 * j, kb * kDepth);
            else
              load2(dst + j * (kOpBytes / 2), map, bar, kb * kDepth + 64 * j, mn0);
          }
        }
      };
      uint32_t ahead = 0;
      bool have_ahead = false;
      auto next_unit = [&](Unit& uu) -> bool {
        if (walk.next(p, uu)) return true;
        if (!p.dyn) return false;
        uint32_t t;
        if (rank == 0) {
          if (!have_ahead) ahead = p.split_tiles + atomicAdd(p.dyn_counter, 1u);
          t = ahead;
          if (!tq_push(tq, t, CG == 2, abort_flag, p.status)) return ok = false;
          have_ahead = t < p.tiles;
          if (have_ahead) ahead = p.split_tiles + atomicAdd(p.dyn_counter, 1u);
        } else {
          uint32_t slot;
          if (!tq_pop(tq, t, slot, abort_flag, p.status)) return ok = false;
          tq_release(tq, slot, rank);
        }
        if (t >= p.tiles) return false;
        Walk::whole(p, uu, t);
        return true;
      };
      while (ok && next_unit(u)) {
        const Place at = place_of(p, u.tile);
        const uint32_t m0 = (at.tm * CG + rank) * kRows;
        const uint32_t n0 = EPI == kGated ? at.tn * (BN / 2) : (at.tn * CG + rank) * kRows;
        for (uint32_t kb = u.kb0; kb < u.kb1; ++kb) {
          if (!mbar_wait(&empty[stage], phase ^ 1u, abort_flag, p.status, kWdProducerEmpty)) {
            ok = false;
            break;
          }
          uint8_t* sa = ring + stage * kStageBytes;
          uint8_t* sb = sa + kOpBytes;
          if (rank == 0) mbar_arrive_expect_tx(&full[stage], CG * kStageBytes);
          const uint32_t seg = kb / p.kb_seg, k = kb - seg * p.kb_seg, op = at.prob + seg;
          load(sa, &p.a[op], &full[stage], p.a_mn, p.a_3d, m0, k);
          if constexpr (EPI == kGated && CG == 1) {
            // 64 rows of the gate's weights, then 64 of the up projection's
#pragma unroll
            for (uint32_t h = 0; h < 2; ++h)
#pragma unroll
              for (uint32_t j = 0; j < 2; ++j)
                load2(sb + j * (kOpBytes / 2) + h * (kOpBytes / 4), &p.b[h], &full[stage],
                      k * kDepth + 64 * j, n0);
          } else {
            load(sb, &p.b[EPI == kGated ? rank : op], &full[stage], p.b_mn, p.b_3d, n0, k);
          }
          ++filled;
          if (++stage == kStages) stage = 0, phase ^= 1u;
        }
      }
      // No copy may be in flight when the CTA exits: wait for the last fill of every
      // stage (a pair's leader counts both CTAs' bytes, the final barrier holds the peer).
      const uint32_t n = rank == 0 ? min(filled, kStages) : 0u;
      for (uint32_t i = 0; i < n; ++i) {
        const uint32_t f = filled - 1 - i;
        int none = 0;
        mbar_wait(&full[f % kStages], (f / kStages) & 1u, &none, p.status, kWdDrain, 100000000ull);
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA
    if (rank == 0) {
      auto wait_all = [&](uint64_t* bar, uint32_t parity, unsigned site) {
        return __all_sync(~0u, mbar_wait(bar, parity, abort_flag, p.status, site)) != 0;
      };
      // bits 7 and 10: bf16 operands
      const uint32_t idesc = make_idesc_f16_f32(kRows * CG, BN, p.a_mn != 0, p.b_mn != 0) |
                             (Pair<T>::kBf16 ? (1u << 7 | 1u << 10) : 0u);
      auto commit_all = [&](uint64_t* bar) {
        if constexpr (CG == 2) {
          const uint32_t a = smem_u32(bar);
          umma_commit_pair(a);
          umma_commit_pair(mapa_shared(a, 1));
        } else {
          umma_commit(bar);
        }
      };
      // per 16 k: K-major 32 bytes within the 128-byte rows of a 64-deep block, m / n
      // contiguous 16 rows of 128 bytes
      const uint32_t lbo_a = p.a_mn ? kOpBytes / 2 : 16, lbo_b = p.b_mn ? kOpBytes / 2 : 16;
      const uint32_t a_step = p.a_mn ? 2048 : 32, a_half = p.a_mn ? 4 * 2048 : kOpBytes / 2;
      const uint32_t b_step = p.b_mn ? 2048 : 32, b_half = p.b_mn ? 4 * 2048 : kOpBytes / 2;
      Walk walk;
      walk.init(p, CG);
      Unit u;
      uint32_t stage = 0, phase = 0, i = 0;
      bool ok = true;
      auto next_unit = [&](Unit& uu) -> bool {
        if (walk.next(p, uu)) return true;
        if (!p.dyn) return false;
        uint32_t t, slot;
        const bool got = tq_pop(tq, t, slot, abort_flag, p.status);
        if (__all_sync(~0u, got) == 0) return ok = false;
        if (lane == 0) tq_release(tq, slot, 0);
        if (t >= p.tiles) return false;
        Walk::whole(p, uu, t);
        return true;
      };
      while (ok && next_unit(u)) {
        const uint32_t buf = i & 1u;
        if (!wait_all(&tempty[buf], ((i >> 1) & 1u) ^ 1u, kWdMmaTmemEmpty)) break;
        tc_fence_after();
        const uint32_t d = tmem_base + buf * BN;
        for (uint32_t kb = u.kb0; kb < u.kb1; ++kb) {
          if (!wait_all(&full[stage], phase, kWdMmaFull)) {
            ok = false;
            break;
          }
          tc_fence_after();
          if (elect_one()) {
            const uint32_t a0 = smem_u32(ring + stage * kStageBytes);
            const uint64_t ad0 = make_sdesc_sw128(a0, lbo_a, 1024);
            const uint64_t bd0 = make_sdesc_sw128(a0 + kOpBytes, lbo_b, 1024);
#pragma unroll
            for (uint32_t k = 0; k < kDepth / 16; ++k) {
              const uint64_t ad = ad0 + (((k >> 2) * a_half + (k & 3) * a_step) >> 4);
              const uint64_t bd = bd0 + (((k >> 2) * b_half + (k & 3) * b_step) >> 4);
              const uint32_t add = kb > u.kb0 || k > 0;
              if constexpr (CG == 2)
                umma_f16_ss_pair(d, ad, bd, idesc, add);
              else
                umma_f16_ss(d, ad, bd, idesc, add);
            }
            commit_all(&empty[stage]);
          }
          __syncwarp();
          if (++stage == kStages) stage = 0, phase ^= 1u;
        }
        if (!ok) break;
        if (elect_one()) commit_all(&tfull[buf]);
        __syncwarp();
        ++i;
      }
      // every product that was issued completes (bounded) before the memory goes away
      if (elect_one()) {
        if constexpr (CG == 2)
          umma_commit_pair(smem_u32(drain));
        else
          umma_commit(drain);
      }
      __syncwarp();
      int none = 0;
      mbar_wait(drain, 0, &none, p.status, kWdDrain, 100000000ull);
    }
  } else {
    // ------------------------------------------------------------ epilogue
    const uint32_t e = warp - 2, q = warp & 3u, half = e >> 2;
    const uint32_t row_in_tile = q * 32 + lane;
    uint8_t* stg = staging + e * 2 * kBoxBytes;
    auto wait_all = [&](uint64_t* bar, uint32_t parity, unsigned site) {
      return __all_sync(~0u, mbar_wait(bar, parity, abort_flag, p.status, site)) != 0;
    };
    Walk walk;
    walk.init(p, CG);
    Unit u;
    uint32_t i = 0, turn = 0;
    auto next_unit = [&](Unit& uu) -> bool {
      if (walk.next(p, uu)) return true;
      if (!p.dyn) return false;
      uint32_t t, slot;
      const bool got = tq_pop(tq, t, slot, abort_flag, p.status);
      if (__all_sync(~0u, got) == 0) return false;
      if (lane == 0) tq_release(tq, slot, rank);
      if (t >= p.tiles) return false;
      Walk::whole(p, uu, t);
      return true;
    };
    while (next_unit(u)) {
      const uint32_t buf = i & 1u;
      if (!wait_all(&tfull[buf], (i >> 1) & 1u, kWdEpilogueTmemFull)) break;
      tc_fence_after();
      const uint32_t taddr = tmem_base + ((q * 32u) << 16) + buf * BN;
      bool mine = true;  // whether this CTA finishes the tile
      const float4* parts = nullptr;
      if (u.split) {
        // publish the fp32 part, take a ticket; the last one finishes the tile
        float4* slot = reinterpret_cast<float4*>(p.partials) +
                       (size_t(walk.unit) * CG + rank) * (kRows * BN / 4);
#pragma unroll 1
        for (uint32_t c = half * (BN / 64); c < (half + 1) * (BN / 64); ++c) {
          uint32_t r[32];
          tmem_ld_32x32b_x32(taddr + c * 32, r);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 8; ++j)
            __stcg(slot + partial_index(c, j, row_in_tile),
                   make_float4(__uint_as_float(r[4 * j]), __uint_as_float(r[4 * j + 1]),
                               __uint_as_float(r[4 * j + 2]), __uint_as_float(r[4 * j + 3])));
        }
        __threadfence();
        named_barrier_sync(1, 32 * kEpiWarps);
        if (e == 0 && lane == 0) {
          unsigned* counter = &p.counters[u.tile * CG + rank];
          const bool last = atomicAdd(counter, 1u) == p.parts - 1;
          if (last) atomicExch(counter, 0u);
          *bcast = last;
        }
        named_barrier_sync(1, 32 * kEpiWarps);
        mine = *reinterpret_cast<volatile uint32_t*>(bcast) != 0;
        if (mine) {
          __threadfence();
          parts = reinterpret_cast<const float4*>(p.partials) +
                  (size_t(u.tile) * p.parts * CG + rank) * (kRows * BN / 4);
        }
        named_barrier_sync(1, 32 * kEpiWarps);  // the word is read before it is written again
      }
      // columns 32 c .. of the tile's sums, from TMEM or from all parts in their order
      auto sums = [&](uint32_t c, float (&v)[32]) {
        if (!parts) {
          uint32_t r[32];
          tmem_ld_32x32b_x32(taddr + c * 32, r);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(r[j]);
          return;
        }
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] = 0.f;
#pragma unroll 2
        for (uint32_t s = 0; s < p.parts; ++s) {
          const float4* src = parts + size_t(s) * CG * (kRows * BN / 4);
          float4 x[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) x[j] = __ldcg(src + partial_index(c, j, row_in_tile));
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            v[4 * j] += x[j].x;
            v[4 * j + 1] += x[j].y;
            v[4 * j + 2] += x[j].z;
            v[4 * j + 3] += x[j].w;
          }
        }
      };
      if (mine) {
        const Place at = place_of(p, u.tile);
        const uint32_t M = p.prob[at.prob].m, N = p.prob[at.prob].n;
        const uint32_t row0 = (at.tm * CG + rank) * kRows + q * 32;
        constexpr uint32_t kWide = EPI == kGated ? BN / 2 : BN;  // output columns of a tile
        constexpr uint32_t kChunks = kWide / 64;                 // 32-column chunks of this warp
#pragma unroll 1
        for (uint32_t cc = 0; cc < kChunks; ++cc) {
          const uint32_t c = half * kChunks + cc, col = at.tn * kWide + c * 32;
          if (row0 >= M || col >= N) break;  // this and the following chunks lie outside
          float v[32];
          if constexpr (EPI == kLinear) {
            uint32_t res[16];
            if (p.in_ptr[0]) load_chunk<T>(p, 0, row0, col, M, N, stg, lane, res);
            sums(c, v);
            if (p.bias) add_bias<T>(p, col, N, v);
            if (p.out_want >> 1 & 1)
              store_chunk<T>(p, 1, row0, col, M, N, stg, turn, lane, v);
            with_activation(p.act, [&]<int ACT>() {
#pragma unroll
              for (int j = 0; j < 32; ++j) v[j] = activate<ACT>(v[j]);
            });
            if (p.in_ptr[0]) {
#pragma unroll
              for (int j = 0; j < 16; ++j) {
                const float2 f = Pair<T>::unpack(res[j]);
                v[2 * j] += f.x;
                v[2 * j + 1] += f.y;
              }
            }
            store_chunk<T>(p, int(at.prob), row0, col, M, N, stg, turn, lane, v);
          } else if constexpr (EPI == kGated) {
            float up[32];
            sums(c, v);
            sums(c + BN / 64, up);
            if (p.out_want >> 1 & 1) store_chunk<T>(p, 1, row0, col, M, N, stg, turn, lane, v);
            if (p.out_want >> 2 & 1) store_chunk<T>(p, 2, row0, col, M, N, stg, turn, lane, up);
            with_activation(p.act, [&]<int ACT>() {
#pragma unroll
              for (int j = 0; j < 32; ++j) v[j] = activate<ACT>(v[j]) * up[j];
            });
            store_chunk<T>(p, 0, row0, col, M, N, stg, turn, lane, v);
          } else {
            uint32_t graw[16], uraw[16];
            load_chunk<T>(p, 0, row0, col, M, N, stg, lane, graw);
            load_chunk<T>(p, 1, row0, col, M, N, stg, lane, uraw);
            sums(c, v);
            float du[32], h[32];
            with_activation(p.act, [&]<int ACT>() {
#pragma unroll
              for (int j = 0; j < 16; ++j) {
                const float2 g = Pair<T>::unpack(graw[j]), up = Pair<T>::unpack(uraw[j]);
                float a, d;
                activate_both<ACT>(g.x, a, d);
                du[2 * j] = v[2 * j] * a;
                h[2 * j] = a * up.x;
                v[2 * j] *= up.x * d;
                activate_both<ACT>(g.y, a, d);
                du[2 * j + 1] = v[2 * j + 1] * a;
                h[2 * j + 1] = a * up.y;
                v[2 * j + 1] *= up.y * d;
              }
            });
            store_chunk<T>(p, 0, row0, col, M, N, stg, turn, lane, v);
            store_chunk<T>(p, 1, row0, col, M, N, stg, turn, lane, du);
            store_chunk<T>(p, 2, row0, col, M, N, stg, turn, lane, h);
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (CG == 2 && rank == 1)
          mbar_arrive_cluster(mapa_shared(smem_u32(&tempty[buf]), 0));  // the leader's MMA waits
        else
          mbar_arrive(&tempty[buf]);
      }
      ++i;
    }
    if (lane == 0) bulk_wait_group<0>();  // the boxes stay until they have been written out
    __syncwarp();
  }

  tc_fence_before();
  if (CG == 2)
    cluster_sync();  // no CTA exits while its peer may still use its memory
  else
    __syncthreads();
  if (p.dyn && rank == 0 && threadIdx.x == 0) {
    // every leader has taken its final tile id: the last one puts the counter back
    __threadfence();
    if (atomicAdd(p.dyn_counter + 1, 1u) == gridDim.x / CG - 1) {
      atomicExch(p.dyn_counter, 0u);
      atomicExch(p.dyn_counter + 1, 0u);
    }
  }
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    if constexpr (CG == 2)
      tmem_dealloc_pair(tmem_base, kTmemCols);
    else
      tmem_dealloc(tmem_base, kTmemCols);
  }
}

struct Plan {
  int cg;
  uint32_t tiles, kb, units, split_tiles, parts;
  bool dyn;
};

uint64_t count_tiles(const Product& p, int cg) {
  const uint64_t bm = kRows * cg, bn = kRows * cg / (p.epilogue == kGated ? 2 : 1);
  uint64_t tiles = 0;
  for (uint32_t i = 0; i < p.problems; ++i)
    tiles += ((p.m[i] + bm - 1) / bm) * ((p.n[i] + bn - 1) / bn);
  return tiles;
}

Plan plan_for(const Product& p, int cg, int num_sms) {
  Plan r{};
  r.cg = cg;
  r.tiles = uint32_t(count_tiles(p, cg));
  r.kb = (p.k + kDepth - 1) / kDepth * p.segments;
  const uint32_t units = std::max(1u, uint32_t(num_sms) / cg);
  const uint32_t rem = r.tiles % units, waves = (r.tiles + units - 1) / units;
  // The last wave's tiles are cut along k where that fills at least twice as many units
  // and whole waves would leave more than 5 % of them idle; a part is at least 2 blocks.
  r.parts = 1;
  if (rem && uint64_t(r.tiles) * 100 < uint64_t(waves) * units * 95)
    r.parts = std::max(1u, std::min({units / rem, r.kb / 2, 8u}));
  r.split_tiles = r.parts > 1 ? rem : 0;
  r.units = std::min(units, r.tiles - r.split_tiles + r.split_tiles * r.parts);
  r.dyn = r.tiles - r.split_tiles >= 4 * r.units;
  return r;
}

// Time of a plan in units of one 128-deep block of a CTA pair's 256 x 256 tile. A single
// CTA's 128 x 128 tile does half a CTA's share of that at about 0.7 of the rate (it reads
// twice the bytes per product from the L2).
double cost_of(const Plan& r, int num_sms) {
  const double units = std::max(1, num_sms / r.cg);
  const double block = r.cg == 2 ? 1.0 : 0.72;
  const double whole = double((r.tiles - r.split_tiles + uint32_t(units) - 1) / uint32_t(units));
  const double split = r.split_tiles ? 1.0 / r.parts : 0.0;
  return block * (r.kb * (whole + split) + 6 * (whole + (r.split_tiles ? 2 : 0)));
}

Plan make_plan(const Product& p, int num_sms) {
  const Plan one = plan_for(p, 1, num_sms), two = plan_for(p, 2, num_sms);
  return cost_of(two, num_sms) <= cost_of(one, num_sms) ? two : one;
}

size_t workspace_need(const Plan& r) {
  size_t n = felix_impl::kWsCounterBytes;
  if (r.split_tiles)
    n += size_t(r.split_tiles) * r.parts * r.cg * kRows * (kRows * r.cg) * sizeof(float);
  return n;
}

// Tensor map of an operand: whole 64-wide blocks as a third dimension where its
// contiguous extent is a multiple of 64, two dimensions otherwise.
int encode_operand(CUtensorMap* map, const Mat& x, bool mn, bool whole, uint32_t rows, uint32_t k,
                   uint32_t box_rows) {
  const uint64_t inner = mn ? rows : k, outer = mn ? k : rows;
  // a single row's distance to the next one is never used, but has to be encodable
  const uint64_t pitch = outer > 1 ? uint64_t(x.ld) * 2 : (inner * 2 + 15) / 16 * 16;
  if (whole)
    return felix_impl::encode_tmap_3d_f16(map, x.p, 64, outer, inner / 64, pitch, 128, 64,
                                          mn ? kDepth : box_rows, 2);
  return felix_impl::encode_tmap_2d_f16(map, x.p, inner, outer, pitch, 64, mn ? kDepth : box_rows);
}

template <class T, int EPI, int CG>
FelixCode launch(DeviceInfo* dev, const Params& p, uint32_t units, cudaStream_t stream) {
  static felix_impl::PerDeviceOnce once;
  const int rc = once.run(dev->ordinal, [] {
    return int(cudaFuncSetAttribute(ffn_product_kernel<T, EPI, CG>,
                                    cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes));
  });
  if (rc) return felix_impl::launch_error(cudaError_t(rc), "feed-forward product: attributes");
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(units * CG);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kSmemBytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {CG, 1, 1};
  cfg.attrs = attr;
  cfg.numAttrs = CG > 1 ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, ffn_product_kernel<T, EPI, CG>, p);
  if (e != cudaSuccess) return felix_impl::launch_error(e, "feed-forward product: launch failed");
  return FelixCode{FELIX_SUCCESS, cudaSuccess};
}

template <class T, int EPI>
FelixCode launch(DeviceInfo* dev, const Params& p, const Plan& r, cudaStream_t stream) {
  return r.cg == 2 ? launch<T, EPI, 2>(dev, p, r.units, stream)
                   : launch<T, EPI, 1>(dev, p, r.units, stream);
}

template <class T>
FelixCode launch(DeviceInfo* dev, const Params& p, const Plan& r, int epilogue,
                 cudaStream_t stream) {
  switch (epilogue) {
    case kGated: return launch<T, kGated>(dev, p, r, stream);
    case kDGated: return launch<T, kDGated>(dev, p, r, stream);
    default: return launch<T, kLinear>(dev, p, r, stream);
  }
}

}  // namespace product

using namespace product;

size_t product_workspace_bytes(const Product& p, int num_sms) {
  return workspace_need(make_plan(p, num_sms));
}

FelixCode product_launch(DeviceInfo* dev, const Product& x, void* workspace, cudaStream_t stream) {
  if (count_tiles(x, 1) > 0x3fffffffu)
    return felix_impl::api_error("feed-forward product: too many tiles");
  const Plan r = make_plan(x, dev->num_sms);
  if (r.split_tiles * r.cg > felix_impl::kWsMaxCounters - 2)
    return felix_impl::api_error("feed-forward product: too many split tiles");
  Params p{};
  const uint32_t bm = kRows * r.cg, bn = kRows * r.cg / (x.epilogue == kGated ? 2 : 1);
  const uint32_t operands = std::max(x.segments, x.problems);
  const bool gated = x.epilogue == kGated;
  uint32_t tile = 0;
  p.a_3d = p.b_3d = 1;
  for (uint32_t i = 0; i < x.problems; ++i) {
    p.prob[i] = {x.m[i], x.n[i], (x.m[i] + bm - 1) / bm, (x.n[i] + bn - 1) / bn, tile};
    tile += p.prob[i].tiles_m * p.prob[i].tiles_n;
    if ((x.a_mn ? x.m[i] : x.k) % 64) p.a_3d = 0;
    if ((x.b_mn ? x.n[i] : x.k) % 64) p.b_3d = 0;
  }
  if (gated && r.cg == 1) p.b_3d = 0;  // boxes of 64 rows, side by side in a stage
  for (uint32_t i = 0; i < std::max(operands, gated ? 2u : 1u); ++i) {
    const uint32_t prob = std::min(i, x.problems - 1);
    if (i < operands &&
        encode_operand(&p.a[i], x.a[i], x.a_mn, p.a_3d, x.m[prob], x.k, kRows))
      return felix_impl::api_error("feed-forward product: cuTensorMapEncodeTiled failed");
    if (encode_operand(&p.b[i], x.b[i], x.b_mn, p.b_3d, x.n[prob], x.k,
                       gated && r.cg == 1 ? 64 : kRows))
      return felix_impl::api_error("feed-forward product: cuTensorMapEncodeTiled failed");
  }
  for (uint32_t i = 0; i < 3; ++i) {
    if (!x.out[i].p) continue;
    const uint32_t prob = std::min(i, x.problems - 1), m = x.m[prob], n = x.n[prob];
    p.out_ptr[i] = x.out[i].p;
    p.out_ld[i] = x.out[i].ld;
    p.out_want |= 1u << i;
    if (!tma_ok(x.out[i].p, x.out[i].ld, m, n)) continue;
    const uint64_t pitch = m > 1 ? uint64_t(x.out[i].ld) * 2 : (uint64_t(n) * 2 + 15) / 16 * 16;
    if (felix_impl::encode_tmap_2d_f16_swizzle(&p.out[i], x.out[i].p, n, m, pitch, 32, 32, 64))
      return felix_impl::api_error("feed-forward product: cuTensorMapEncodeTiled failed");
    p.out_tma |= 1u << i;
  }
  if (x.problems > 1) p.out_want &= 1;  // there out[] are the problems' results
  for (uint32_t i = 0; i < 2; ++i) {
    if (!x.in[i].p) continue;
    p.in_ptr[i] = x.in[i].p;
    p.in_ld[i] = x.in[i].ld;
    const bool vec = (reinterpret_cast<uintptr_t>(x.in[i].p) & 15) == 0 && x.n[0] % 8 == 0 &&
                     (x.m[0] <= 1 || x.in[i].ld % 8 == 0);
    p.in_vec |= uint32_t(vec) << i;
  }
  p.problems = x.problems;
  p.tiles = r.tiles;
  p.kb = r.kb;
  p.kb_seg = r.kb / x.segments;
  p.a_mn = x.a_mn;
  p.b_mn = x.b_mn;
  p.group_m = r.cg == 2 ? 8 : 16;
  p.split_tiles = r.split_tiles;
  p.parts = r.parts;
  p.dyn = r.dyn;
  p.bias = x.bias;
  p.act = x.act;
  p.counters = static_cast<unsigned*>(workspace);
  p.dyn_counter = p.counters + (felix_impl::kWsMaxCounters - 2);
  p.partials = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) +
                                        felix_impl::kWsCounterBytes);
  p.status = dev->status_word;
  return x.bf16 ? launch<__nv_bfloat16>(dev, p, r, x.epilogue, stream)
                : launch<__half>(dev, p, r, x.epilogue, stream);
}

}  // namespace felix_ffn
