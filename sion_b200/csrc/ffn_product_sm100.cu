// Products of the feed-forward operators on tcgen05, fp16 or bf16 in, fp32 accumulators
// in TMEM, everything that follows a product done on them before they are rounded once:
//   kLinear  act(x W^T + bias) + residual, and the value in front of the activation
//   kGated   both projections of a gated block: gate and up accumulate side by side in
//            TMEM, so that one thread holds both of an element: act(g) u
//   kDGated  dh = dy Wd never leaves the SM: dg, du and h are written from it
//
// Tiles. CG = 2: a CTA pair (cta_group::2) computes 256 rows x BN columns, each CTA loading
// its 128 rows of A and BN / 2 of B per stage and holding its rows of the tile in its TMEM;
// for kGated one CTA's rows of B are the gate's and the other's the up projection's. CG = 1:
// 128 x 128. Two accumulators, so that the epilogue of a tile overlaps the next tile's
// products. HALVES = 2: two accumulators of one tile of 256 x 512; its epilogue has to be short.
// What bounds a tile is the L2's 64 bytes a cycle and SM: per 128 k a pair's CTA needs 1024
// cycles for 64 KB at BN = 256, as long as its products take, 768 for 48 KB at BN = 128
// (products 512), 768 a half at 512 columns; so few tiles are cut along k rather than made
// small. An operand may be stored with k or with m / n contiguous: a training step's x W^T,
// dz W and dz^T x need no transpose. One launch may do several products (a backward pass does
// all of its own), deepest tiles first. Measured: 8192 x 4096 x 16384 843 us in a loop under
// the power cap (1.3 PFLOP/s); 500 x 4096 x 11264 49 us, with two projections 92, which are
// 176 tiles for 74 pairs: three waves for 2.4.
//
// Warps: 0 TMA, 1 MMA, 8 of the epilogue (two per quarter of the TMEM lanes, which take every
// other 32 columns: activations cost 10 to 50 instructions a value).
//
// Schedule: persistent, tiles from a queue (tile_queue.cuh) where there are several per CTA;
// or, where tiles are few, each tile in parts of its depth over a cluster (ffn_finish.cuh).
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "activation.cuh"
#include "ffn_finish.cuh"
#include "ffn_internal.h"
#include "sm100_ptx.cuh"
#include "tile_queue.cuh"

namespace felix_ffn {
namespace product {

using namespace felix_sm100;

constexpr uint32_t kRows = 128;               // rows of A, and of a tile, in one CTA
constexpr uint32_t kEpiWarps = 8;
constexpr uint32_t kBoxBytes = 32 * 64;       // 32 rows x 32 columns
constexpr uint32_t kStagingBytes = kEpiWarps * kBoxBytes;
constexpr uint32_t kBarBytes = 512;
constexpr uint32_t kRingBytes = 192 * 1024;
constexpr uint32_t kSmemBytes = kRingBytes + kStagingBytes + kBarBytes + 1024;

// CG CTAs per tile, HALVES accumulators of BN columns side by side in a tile. Stages of 128 k:
// with stages of 64 k and requests of 16 KB a pair's 256 x 256 tiles ran 2 % faster alone
// (8192 x 4096 x 16384: 730 -> 711 us), but 3 % slower under the power cap (843 -> 871).
template <int CG, int BN, int HALVES>
struct Shape {
  static constexpr uint32_t kDepth = HALVES == 2 ? 64 : 128;
  static constexpr uint32_t kBRows = BN / CG;
  static constexpr uint32_t kABytes = kRows * kDepth * 2, kBBytes = kBRows * kDepth * 2;
  static constexpr uint32_t kStageBytes = kABytes + HALVES * kBBytes;
  static constexpr uint32_t kStages = kRingBytes / kStageBytes;
  // a tile's parts: a CTA's own and what it receives of the others' lie in the ring
  static constexpr uint32_t kMaxParts = BN == 256 ? 2 : 8;
  static_assert(kRows * BN * 4 + (kMaxParts - 1) * (kRows / kMaxParts) * BN * 4 <= kRingBytes);
  static constexpr uint32_t kFirstEpi = HALVES == 2 ? 4 : 2;  // first epilogue warp
  static constexpr uint32_t kThreads = 32 * (kFirstEpi + kEpiWarps);
};
// Wide tiles: the epilogue's two warpgroups hold 128 results a thread and take registers from
// the first one (TMA, MMA and two idle warps): 128 x 80 + 256 x 208 <= 384 x 168, which the
// host checks before the first launch.
constexpr int kRegsLaunch = 168, kRegsFirst = 80, kRegsEpi = 208;
static_assert(128 * kRegsFirst + 256 * kRegsEpi <= 384 * kRegsLaunch, "registers at launch");
// Stages that a pair works through for one half of a wide tile before the other.
constexpr uint32_t kSkew = 2;

struct Problem {
  uint32_t m, n, tiles_m, tiles_n, tile0;
  uint32_t kb, kb_seg;      // blocks of kDepth of a tile, of a segment
  uint32_t map;             // its first operands in a[], b[]
  uint32_t a_mn, b_mn;      // operands stored with m / n contiguous
  uint32_t a_3d, b_3d;      // one request per operand and stage
};

struct alignas(64) Params {
  CUtensorMap a[kMaxOperands], b[kMaxOperands];
  Problem prob[kMaxProblems];
  uint32_t problems, tiles, group_m;
  uint32_t parts;              // of each tile's depth, a cluster's CTAs or pairs
  uint32_t dyn;                // tiles come from the queue
  Finish fin;
  // bit per output and input: rows of whole 16-byte vectors, of whole 32-byte sectors
  uint32_t out_vec, out_sectors, in_vec, in_sectors;
  unsigned* dyn_counter;       // [0] next tile, [1] CTAs that are done; zero between launches
  unsigned* status;
};

struct Unit {
  uint32_t prob, tm, tn, kb0, kb1;
};

// Where a tile stands. Grouped raster: runs of group_m tiles along m sweep across n, so that
// CTAs that run together share panels of A and B in the L2.
__device__ __forceinline__ Unit unit_of(const Params& p, uint32_t tile) {
  Unit u{};
  while (u.prob + 1 < p.problems && tile >= p.prob[u.prob + 1].tile0) ++u.prob;
  const Problem& q = p.prob[u.prob];
  const uint32_t t = tile - q.tile0, per_group = p.group_m * q.tiles_n, g = t / per_group;
  const uint32_t m0 = g * p.group_m, gm = min(p.group_m, q.tiles_m - m0), i = t - g * per_group;
  u.tm = m0 + i % gm;
  u.tn = i / gm;
  u.kb1 = q.kb;
  return u;
}

// The walk of every role of a CTA: a part of one tile, or whole tiles. Every other wave runs
// backwards: who had one of the first, deepest tiles comes last.
struct Walk {
  uint32_t unit, units, wave;
  __device__ __forceinline__ void init(uint32_t cg) {
    unit = blockIdx.x / cg;
    units = gridDim.x / cg;
    wave = 0;
  }
  __device__ __forceinline__ bool next(const Params& p, Unit& u) {
    if (p.parts > 1) {
      if (wave++) return false;
      const uint32_t part = unit % p.parts;
      u = unit_of(p, unit / p.parts);
      u.kb0 = u.kb1 * part / p.parts;
      u.kb1 = u.kb1 * (part + 1) / p.parts;
      return true;
    }
    const uint32_t tile = wave * units + (wave & 1 ? units - 1 - unit : unit);
    ++wave;
    if (p.dyn || tile >= p.tiles) return false;
    u = unit_of(p, tile);
    return true;
  }
};

// A warp's box in shared memory: 32 rows of 64 bytes (32 columns), the 16-byte pieces of a
// row swizzled so that neither 8 lanes of a row each nor 8 rows of 4 lanes conflict.
__device__ __forceinline__ uint32_t box_offset(uint32_t row, uint32_t piece) {
  return row * 64 + ((piece ^ ((row >> 1) & 3)) * 16);
}

// 32 bytes of global memory at once (32-byte aligned), or as two vectors of 16.
__device__ __forceinline__ void load32(const void* p, uint32_t* v) {
  asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]),
                 "=r"(v[7])
               : "l"(p)
               : "memory");
}
__device__ __forceinline__ void store32(void* p, const uint32_t* v) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(v[0]),
               "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}

// 32 columns of this lane's row of an input, packed; what lies outside reads as 0. Rows
// that are no whole vectors are read 64 bytes of a row at a time through the box.
__device__ __forceinline__ void load_chunk(const Params& p, int which, uint32_t row0, uint32_t col,
                                           uint32_t M, uint32_t N, uint8_t* box, uint32_t lane,
                                           uint32_t (&raw)[16]) {
  const uint16_t* base = static_cast<const uint16_t*>(p.fin.in[which]);
  const int64_t ld = p.fin.in_ld[which];
  if (p.in_vec >> which & 1) {
    const uint32_t row = row0 + lane;
    const bool sectors = p.in_sectors >> which & 1;
#pragma unroll
    for (uint32_t j = 0; j < 2; ++j) {
      const uint16_t* at = base + int64_t(row) * ld + col + 16 * j;
      if (sectors && row < M && col + 16 * j < N) {
        load32(at, raw + 8 * j);
      } else {
#pragma unroll
        for (uint32_t i = 0; i < 2; ++i) {
          uint4 v = make_uint4(0, 0, 0, 0);
          if (row < M && col + 16 * j + 8 * i < N) v = *reinterpret_cast<const uint4*>(at + 8 * i);
          raw[8 * j + 4 * i] = v.x, raw[8 * j + 4 * i + 1] = v.y;
          raw[8 * j + 4 * i + 2] = v.z, raw[8 * j + 4 * i + 3] = v.w;
        }
      }
    }
    return;
  }
  const uint32_t rows = M - row0;
  const uint16_t* at = base + int64_t(row0) * ld + col + lane;
  uint16_t v[32];  // all 32 rows under way together
#pragma unroll
  for (uint32_t r = 0; r < 32; ++r)
    v[r] = r < rows && col + lane < N ? at[int64_t(r) * ld] : uint16_t(0);
  __syncwarp();
#pragma unroll
  for (uint32_t r = 0; r < 32; ++r)
    *reinterpret_cast<uint16_t*>(box + box_offset(r, lane / 8) + lane % 8 * 2) = v[r];
  __syncwarp();
#pragma unroll
  for (uint32_t j = 0; j < 4; ++j) {
    const uint4 v = *reinterpret_cast<const uint4*>(box + box_offset(lane, j));
    raw[4 * j] = v.x, raw[4 * j + 1] = v.y, raw[4 * j + 2] = v.z, raw[4 * j + 3] = v.w;
  }
}

// Writes 32 columns of each of the warp's rows: a lane its row, two sectors, straight from
// registers (rows that are no whole vectors: through the box, 64 bytes of a row at a
// time). Shared memory is busy with the operands.
__device__ __forceinline__ void store_packed(const Params& p, int which, uint32_t row0,
                                             uint32_t col, uint32_t M, uint32_t N, uint8_t* box,
                                             uint32_t lane, const uint32_t (&w)[16]) {
  uint16_t* base = static_cast<uint16_t*>(p.fin.out[which]);
  const int64_t ld = p.fin.out_ld[which];
  if (p.out_vec >> which & 1) {
    const uint32_t row = row0 + lane;
    if (row >= M) return;
    uint16_t* at = base + int64_t(row) * ld + col;
    if (p.out_sectors >> which & 1) {
#pragma unroll
      for (uint32_t j = 0; j < 2; ++j)
        if (col + 16 * j < N) store32(at + 16 * j, w + 8 * j);
    } else {
#pragma unroll
      for (uint32_t j = 0; j < 4; ++j)
        if (col + 8 * j < N)
          *reinterpret_cast<uint4*>(at + 8 * j) =
              make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
    }
    return;
  }
  __syncwarp();
#pragma unroll
  for (uint32_t j = 0; j < 4; ++j)
    *reinterpret_cast<uint4*>(box + box_offset(lane, j)) =
        make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
  __syncwarp();
  if (col + lane < N) {
    const uint32_t rows = M - row0;
    uint16_t* at = base + int64_t(row0) * ld + col + lane;
#pragma unroll
    for (uint32_t r = 0; r < 32; ++r)
      if (r < rows)
        at[int64_t(r) * ld] =
            *reinterpret_cast<const uint16_t*>(box + box_offset(r, lane / 8) + lane % 8 * 2);
  }
}
template <class T>
__device__ __forceinline__ void store_chunk(const Params& p, int which, uint32_t row0, uint32_t col,
                                            uint32_t M, uint32_t N, uint8_t* box, uint32_t lane,
                                            const float (&v)[32]) {
  uint32_t w[16];
#pragma unroll
  for (int j = 0; j < 16; ++j) w[j] = Pair<T>::pack(v[2 * j], v[2 * j + 1]);
  store_packed(p, which, row0, col, M, N, box, lane, w);
}

// Bias of 32 columns (the same for every row: one broadcast load each).
template <class T>
__device__ __forceinline__ void add_bias(const Params& p, uint32_t col, uint32_t N, float (&v)[32]) {
  const uint16_t* b = static_cast<const uint16_t*>(p.fin.bias) + col;
  if (col + 32 <= N && (reinterpret_cast<uintptr_t>(b) & 15) == 0) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint4 w = reinterpret_cast<const uint4*>(b)[j];
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
      if (col + i < N) v[i] += Pair<T>::to_float(b[i]);
  }
}

template <class T, int EPI, int CG, int BN, int HALVES>
__global__ void __launch_bounds__((Shape<CG, BN, HALVES>::kThreads), 1)
    ffn_product_kernel(const __grid_constant__ Params p) {
  using S = Shape<CG, BN, HALVES>;
  constexpr uint32_t kDepth = S::kDepth, kABytes = S::kABytes, kBBytes = S::kBBytes;
  constexpr uint32_t kBRows = S::kBRows, kStages = S::kStages, kStageBytes = S::kStageBytes;
  const uint32_t cta = CG == 2 || p.parts > 1 ? cluster_ctarank() : 0u;  // in the cluster
  const uint32_t rank = CG == 2 ? cta & 1u : 0u;                         // in the pair
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  uint8_t* staging = ring + kRingBytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(staging + kStagingBytes);
  uint64_t* full = bars;
  uint64_t* empty = full + kStages;
  uint64_t* tfull = empty + kStages;
  uint64_t* tempty = tfull + 2;
  uint64_t* drain = tempty + 2;
  uint64_t* received = drain + 1;
  uint64_t* tq_full = received + 1;
  uint64_t* tq_empty = tq_full + kTq;
  uint32_t* words = reinterpret_cast<uint32_t*>(tq_empty + kTq);
  static_assert((2 * kStages + 6 + 2 * kTq) * 8 + (kTq + 2) * 4 <= kBarBytes, "barrier block");
  TileQueue tq{words, tq_full, tq_empty, 0};
  uint32_t* tmem_slot = words + kTq;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(words + kTq + 1);

  const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  if (threadIdx.x == 0) {
    tma_prefetch_desc(&p.a[0]);
    tma_prefetch_desc(&p.b[0]);
    for (uint32_t i = 0; i < kStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&tfull[i], 1);
      mbar_init(&tempty[i], kEpiWarps * CG);  // a pair's leader counts both CTAs' warps
    }
    mbar_init(drain, 1);
    mbar_init(received, 1);
    for (uint32_t i = 0; i < kTq; ++i) {
      mbar_init(&tq_full[i], 1);
      // the MMA warp and the epilogue warps; of the peer its producer and epilogue warps
      mbar_init(&tq_empty[i], CG * (kEpiWarps + 1));
    }
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (CG == 2) cluster_sync();  // the peer uses this CTA's barriers
  if (warp == 1) {
    if constexpr (CG == 2) {
      tmem_alloc_pair(tmem_slot, 2 * BN);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(tmem_slot, 2 * BN);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  wait_for_earlier_launches();

  // A warp's next unit from the queue (MMA and epilogue warps); false at the end, or where a
  // wait gave up.
  auto pop_unit = [&](Unit& u, uint32_t who) -> bool {
    if (!p.dyn) return false;
    uint32_t t, slot;
    const bool got = tq_pop(tq, t, slot, abort_flag, p.status);
    if (__all_sync(~0u, got) == 0) return false;
    if (lane == 0) tq_release(tq, slot, who);
    if (t >= p.tiles) return false;
    u = unit_of(p, t);
    return true;
  };

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    if constexpr (HALVES == 2) setmaxnreg_dec<kRegsFirst>();
    if (elect_one()) {
      Walk walk;
      walk.init(CG);
      Unit u;
      uint32_t stage = 0, phase = 0, filled = 0;
      bool ok = true;
      // loads of a pair's CTAs complete on the leader's barrier
      auto load2 = [&](uint8_t* dst, const CUtensorMap* map, uint64_t* bar, uint32_t x, uint32_t y) {
        if constexpr (CG == 2)
          tma_load_2d_pair(dst, map, mapa_shared(smem_u32(bar), cta & ~1u), int(x), int(y));
        else
          tma_load_2d(dst, map, bar, int(x), int(y));
      };
      auto load3 = [&](uint8_t* dst, const CUtensorMap* map, uint64_t* bar, uint32_t y, uint32_t z) {
        if constexpr (CG == 2)
          tma_load_3d_pair(dst, map, mapa_shared(smem_u32(bar), cta & ~1u), 0, int(y), int(z));
        else
          tma_load_3d(dst, map, bar, 0, int(y), int(z));
      };
      // `rows` (of m or n, from mn0) of k block kb: blocks of 64 k of all rows, or of 64
      // m / n of all k
      auto load = [&](uint8_t* dst, const CUtensorMap* map, uint64_t* bar, bool mn, bool whole,
                      uint32_t rows, uint32_t mn0, uint32_t kb) {
        if (mn) {
          if (whole) {
            load3(dst, map, bar, kb * kDepth, mn0 / 64);
          } else {
            for (uint32_t j = 0; j < rows / 64; ++j)
              load2(dst + j * (kDepth * 128), map, bar, mn0 + 64 * j, kb * kDepth);
          }
        } else if (whole && kDepth == 128) {
          load3(dst, map, bar, mn0, kb * 2);
        } else {
#pragma unroll
          for (uint32_t j = 0; j < kDepth / 64; ++j)
            load2(dst + j * (rows * 128), map, bar, kb * kDepth + 64 * j, mn0);
        }
      };
      uint32_t ahead = 0;
      bool have_ahead = false;
      auto next_unit = [&](Unit& uu) -> bool {
        if (walk.next(p, uu)) return true;
        if (!p.dyn) return false;
        uint32_t t;
        if (rank == 0) {
          if (!have_ahead) ahead = atomicAdd(p.dyn_counter, 1u);
          t = ahead;
          if (!tq_push(tq, t, CG == 2, abort_flag, p.status)) return ok = false;
          have_ahead = t < p.tiles;
          if (have_ahead) ahead = atomicAdd(p.dyn_counter, 1u);
        } else {
          uint32_t slot;
          if (!tq_pop(tq, t, slot, abort_flag, p.status)) return ok = false;
          tq_release(tq, slot, rank);
        }
        if (t >= p.tiles) return false;
        uu = unit_of(p, t);
        return true;
      };
      while (ok && next_unit(u)) {
        const Problem& q = p.prob[u.prob];
        const uint32_t m0 = (u.tm * CG + rank) * kRows;
        const uint32_t n0 =
            EPI == kGated ? u.tn * (BN / 2) : u.tn * (BN * HALVES) + rank * kBRows;
        for (uint32_t kb = u.kb0; kb < u.kb1; ++kb) {
          if (!mbar_sleep_wait(&empty[stage], phase ^ 1u, abort_flag, p.status,
                               kWdProducerEmpty)) {
            ok = false;
            break;
          }
          uint8_t* sa = ring + stage * kStageBytes;
          uint8_t* sb = sa + kABytes;
          if (rank == 0) mbar_arrive_expect_tx(&full[stage], CG * kStageBytes);
          const uint32_t seg = kb / q.kb_seg, k = kb - seg * q.kb_seg, op = q.map + seg;
          load(sa, &p.a[op], &full[stage], q.a_mn, q.a_3d, kRows, m0, k);
          if constexpr (EPI == kGated && CG == 1) {
            // half the rows of B are the gate's, then the up projection's
#pragma unroll
            for (uint32_t h = 0; h < 2; ++h)
#pragma unroll
              for (uint32_t j = 0; j < kDepth / 64; ++j)
                load2(sb + (j * 2 + h) * (kBRows / 2 * 128), &p.b[h], &full[stage],
                      k * kDepth + 64 * j, n0);
          } else {
#pragma unroll
            for (uint32_t h = 0; h < HALVES; ++h)
              load(sb + h * kBBytes, &p.b[EPI == kGated ? rank : op], &full[stage], q.b_mn, q.b_3d,
                   kBRows, n0 + h * BN, k);
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
    if constexpr (HALVES == 2) setmaxnreg_dec<kRegsFirst>();
    if (rank == 0) {
      auto wait_all = [&](uint64_t* bar, uint32_t parity, unsigned site) {
        return __all_sync(~0u, mbar_sleep_wait(bar, parity, abort_flag, p.status, site)) != 0;
      };
      auto commit_all = [&](uint64_t* bar) {
        if constexpr (CG == 2) {
          const uint32_t a = smem_u32(bar);
          umma_commit_pair(a);
          umma_commit_pair(mapa_shared(a, cta | 1u));
        } else {
          umma_commit(bar);
        }
      };
      // Operands of a unit's problem. Per 16 k: K-major 32 bytes within the 128-byte rows of
      // a 64-deep block, m / n contiguous 16 rows of 128 bytes.
      uint32_t idesc = 0, lbo_a = 0, lbo_b = 0, a_step = 0, b_step = 0, a_block = 0, b_block = 0;
      auto use_problem = [&](const Problem& q) {
        constexpr uint32_t kChunk = kDepth * 128;  // from 64 m or n to the next
        // bits 7 and 10: bf16 operands
        idesc = make_idesc_f16_f32(kRows * CG, BN, q.a_mn != 0, q.b_mn != 0) |
                (Pair<T>::kBf16 ? (1u << 7 | 1u << 10) : 0u);
        lbo_a = q.a_mn ? kChunk : 16;
        lbo_b = q.b_mn ? kChunk : 16;
        a_step = q.a_mn ? 2048 : 32;
        b_step = q.b_mn ? 2048 : 32;
        a_block = q.a_mn ? 4 * 2048 : kRows * 128;
        b_block = q.b_mn ? 4 * 2048 : kBRows * 128;
      };
      // One stage's products into both halves' accumulators: rows of A that the first half's
      // instruction has fetched stay for the second's.
      auto issue_both = [&](uint32_t stage) {
        const uint32_t a0 = smem_u32(ring + stage * kStageBytes);
        const uint64_t ad0 = make_sdesc_sw128(a0, lbo_a, 1024);
        const uint64_t bd0 = make_sdesc_sw128(a0 + kABytes, lbo_b, 1024);
#pragma unroll
        for (uint32_t k = 0; k < kDepth / 16; ++k) {
          const uint64_t ad = ad0 + (((k >> 2) * a_block + (k & 3) * a_step) >> 4);
          const uint64_t bd = bd0 + (((k >> 2) * b_block + (k & 3) * b_step) >> 4);
          umma_f16_ss_pair_keep_a(tmem_base, ad, bd, idesc);
          umma_f16_ss_pair_use_a(tmem_base + BN, ad, bd + (kBBytes >> 4), idesc);
        }
      };
      // one stage's products into the accumulator of half h
      auto issue = [&](uint32_t stage, uint32_t d, uint32_t h, bool add0) {
        const uint32_t a0 = smem_u32(ring + stage * kStageBytes);
        const uint64_t ad0 = make_sdesc_sw128(a0, lbo_a, 1024);
        const uint64_t bd0 = make_sdesc_sw128(a0 + kABytes + h * kBBytes, lbo_b, 1024);
#pragma unroll
        for (uint32_t k = 0; k < kDepth / 16; ++k) {
          const uint64_t ad = ad0 + (((k >> 2) * a_block + (k & 3) * a_step) >> 4);
          const uint64_t bd = bd0 + (((k >> 2) * b_block + (k & 3) * b_step) >> 4);
          const uint32_t add = add0 || k > 0;
          if constexpr (CG == 2)
            umma_f16_ss_pair(d, ad, bd, idesc, add);
          else
            umma_f16_ss(d, ad, bd, idesc, add);
        }
      };
      Walk walk;
      walk.init(CG);
      Unit u;
      uint32_t stage = 0, phase = 0, i = 0;
      bool ok = true;
      auto advance = [&](uint32_t& st, uint32_t& ph) {
        if (++st == kStages) st = 0, ph ^= 1u;
      };
      while (ok && (walk.next(p, u) || pop_unit(u, 0))) {
        use_problem(p.prob[u.prob]);
        if constexpr (HALVES == 1) {
          const uint32_t buf = i & 1u;
          if (!wait_all(&tempty[buf], ((i >> 1) & 1u) ^ 1u, kWdMmaTmemEmpty)) break;
          tc_fence_after();
          for (uint32_t kb = u.kb0; kb < u.kb1; ++kb) {
            if (!wait_all(&full[stage], phase, kWdMmaFull)) {
              ok = false;
              break;
            }
            tc_fence_after();
            if (elect_one()) {
              issue(stage, tmem_base + buf * BN, 0, kb > u.kb0);
              commit_all(&empty[stage]);
            }
            __syncwarp();
            advance(stage, phase);
          }
          if (!ok) break;
          if (elect_one()) commit_all(&tfull[buf]);
          __syncwarp();
        } else {
          // The first and the last kSkew kStages go through one half's accumulator, then
          // through the other's: while the epilogue reads the first half, products of the
          // second are still under way, and the next tile begins with the first.
          for (uint32_t kb = u.kb0; ok && kb < u.kb1;) {
            const bool first = kb == u.kb0;
            const uint32_t left = u.kb1 - kb;
            uint32_t n = 1;
            if (first || left <= kSkew) n = min(kSkew, left);
            const bool last = n == left;
            if (!first && !last) {
              if (!wait_all(&full[stage], phase, kWdMmaFull)) {
                ok = false;
                break;
              }
              tc_fence_after();
              if (elect_one()) {
                issue_both(stage);
                commit_all(&empty[stage]);
              }
              __syncwarp();
              advance(stage, phase);
              ++kb;
              continue;
            }
#pragma unroll 1
            for (uint32_t h = 0; ok && h < 2; ++h) {
              if (first && !wait_all(&tempty[h], (i & 1u) ^ 1u, kWdMmaTmemEmpty)) {
                ok = false;
                break;
              }
              uint32_t st = stage, ph = phase;
              for (uint32_t j = 0; j < n; ++j) {
                if (h == 0 && !wait_all(&full[st], ph, kWdMmaFull)) {
                  ok = false;
                  break;
                }
                tc_fence_after();
                if (elect_one()) {
                  issue(st, tmem_base + h * BN, h, !first || j > 0);
                  if (h == 1) commit_all(&empty[st]);
                  if (last && j + 1 == n) commit_all(&tfull[h]);
                }
                __syncwarp();
                advance(st, ph);
              }
              if (h == 1) stage = st, phase = ph;
            }
            kb += n;
          }
          if (!ok) break;
        }
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
  } else if (warp >= S::kFirstEpi) {
    // ------------------------------------------------------------ epilogue
    if constexpr (HALVES == 2) setmaxnreg_inc<kRegsEpi>();
    const uint32_t e = warp - S::kFirstEpi, q = warp & 3u, half = e >> 2;
    const uint32_t row_in_tile = q * 32 + lane;
    uint8_t* box = staging + e * kBoxBytes;
    auto wait_all = [&](uint64_t* bar, uint32_t parity, unsigned site) {
      return __all_sync(~0u, mbar_sleep_wait(bar, parity, abort_flag, p.status, site)) != 0;
    };
    Walk walk;
    walk.init(CG);
    Unit u;
    uint32_t i = 0;
    bool ok = true;
    while (ok && (walk.next(p, u) || pop_unit(u, rank))) {
      // Accumulator h of a tile: the tiles alternate between two, or each has both.
      auto accumulator = [&](uint32_t h) { return HALVES == 2 ? h : i & 1u; };
      auto wait_full = [&](uint32_t h) -> bool {
        if (!wait_all(&tfull[accumulator(h)], (HALVES == 2 ? i : i >> 1) & 1u, kWdEpilogueTmemFull))
          return ok = false;
        tc_fence_after();
        return true;
      };
      auto set_empty = [&](uint32_t h) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          uint64_t* bar = &tempty[accumulator(h)];
          if (CG == 2 && rank == 1)
            mbar_arrive_cluster(mapa_shared(smem_u32(bar), cta & ~1u));  // the leader's MMA warp waits
          else
            mbar_arrive(bar);
        }
      };
      auto taddr = [&](uint32_t h) {
        return tmem_base + ((q * 32u) << 16) + accumulator(h) * BN;
      };
      if constexpr (HALVES == 1) {
        if (p.parts > 1) {
          // a part: its sums to shared memory (the ring is idle once they are complete)
          if (!wait_full(0)) break;
          float4* part = reinterpret_cast<float4*>(ring);
#pragma unroll 1
          for (uint32_t c = half; c < BN / 32; c += 2) {
            uint32_t r[32];
            tmem_ld_32x32b_x32(taddr(0) + c * 32, r);
            tmem_ld_wait();
#pragma unroll
            for (uint32_t j = 0; j < 8; ++j)
              part[row_in_tile * (BN / 4) + ((c * 8 + j) ^ (row_in_tile & 7))] =
                  make_float4(__uint_as_float(r[4 * j]), __uint_as_float(r[4 * j + 1]),
                              __uint_as_float(r[4 * j + 2]), __uint_as_float(r[4 * j + 3]));
          }
          fence_proxy_async_smem();  // it will be sent from there
          ++i;
          continue;
        }
      }
      const uint32_t M = p.prob[u.prob].m;
      const uint32_t row0 = (u.tm * CG + rank) * kRows + q * 32;
      if constexpr (HALVES == 2) {
        // Wide tiles: bias, relu, residual. Both halves are read, finished and rounded before
        // anything is written: the next tile's products wait for the reads alone. (All CTAs
        // write at about the same time, 64 KB each at 9 bytes a cycle; written in between,
        // that took 7000 cycles a half.)
        constexpr uint32_t kChunks = BN / 64;  // 32-column chunks of this warp in a half
        const uint32_t N = p.prob[u.prob].n;
        const uint32_t col0 = u.tn * 2 * BN + half * 32;
        uint32_t hold[2][kChunks][16];  // the residual, then the results
        if (p.fin.in[0]) {
#pragma unroll
          for (uint32_t h = 0; h < 2; ++h)
#pragma unroll
            for (uint32_t c = 0; c < kChunks; ++c)
              if (row0 < M && col0 + h * BN + c * 64 < N)
                load_chunk(p, 0, row0, col0 + h * BN + c * 64, M, N, box, lane, hold[h][c]);
        }
#pragma unroll
        for (uint32_t h = 0; h < 2; ++h) {
          if (!wait_full(h)) break;
#pragma unroll
          for (uint32_t c = 0; c < kChunks; ++c) {
            uint32_t r[32];
            tmem_ld_32x32b_x32(taddr(h) + (half + 2 * c) * 32, r);
            tmem_ld_wait();
            float v[32];
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(r[j]);
            if (p.fin.bias) add_bias<T>(p, col0 + h * BN + c * 64, N, v);
            if (p.fin.act == FELIX_ACT_RELU) {
#pragma unroll
              for (int j = 0; j < 32; ++j) v[j] = activate<FELIX_ACT_RELU>(v[j]);
            }
            if (p.fin.in[0]) {
#pragma unroll
              for (int j = 0; j < 16; ++j) {
                const float2 f = Pair<T>::unpack(hold[h][c][j]);
                v[2 * j] += f.x;
                v[2 * j + 1] += f.y;
              }
            }
#pragma unroll
            for (int j = 0; j < 16; ++j) hold[h][c][j] = Pair<T>::pack(v[2 * j], v[2 * j + 1]);
          }
          set_empty(h);
        }
        if (ok) {
#pragma unroll
          for (uint32_t h = 0; h < 2; ++h)
#pragma unroll
            for (uint32_t c = 0; c < kChunks; ++c)
              if (row0 < M && col0 + h * BN + c * 64 < N)
                store_packed(p, int(u.prob), row0, col0 + h * BN + c * 64, M, N, box, lane,
                             hold[h][c]);
        }
      } else {
        if (!wait_full(0)) break;
        // columns 32 c .. of the accumulator's sums
        auto sums = [&](uint32_t column, float (&v)[32]) {
          uint32_t r[32];
          tmem_ld_32x32b_x32(taddr(0) + column, r);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(r[j]);
        };
        constexpr uint32_t wide = EPI == kGated ? BN / 2 : BN;  // output columns of the tile
        const uint32_t first = u.tn * wide;
        const uint32_t N = min(p.prob[u.prob].n, first + wide);
        // chunks of 32 columns that lie inside, every other one this warp's
        const uint32_t chunks = row0 < M ? (N - first + 31) / 32 : 0u;
        if (chunks <= half) set_empty(0);
#pragma unroll 1
        for (uint32_t c = half; c < chunks; c += 2) {
          const uint32_t col = first + c * 32;
          // the accumulator is free for the next products once the last chunk is read
          const bool done = c + 2 >= chunks;
          float v[32];
          if constexpr (EPI == kLinear) {
            uint32_t res[16];
            if (p.fin.in[0]) load_chunk(p, 0, row0, col, M, N, box, lane, res);
            sums(c * 32, v);
            if (done) set_empty(0);
            if (p.fin.bias) add_bias<T>(p, col, N, v);
            if (p.fin.extra >> 1 & 1) store_chunk<T>(p, 1, row0, col, M, N, box, lane, v);
            with_activation(p.fin.act, [&]<int ACT>() {
#pragma unroll
              for (int j = 0; j < 32; ++j) v[j] = activate<ACT>(v[j]);
            });
            if (p.fin.in[0]) {
#pragma unroll
              for (int j = 0; j < 16; ++j) {
                const float2 f = Pair<T>::unpack(res[j]);
                v[2 * j] += f.x;
                v[2 * j + 1] += f.y;
              }
            }
            store_chunk<T>(p, int(u.prob), row0, col, M, N, box, lane, v);
          } else if constexpr (EPI == kGated) {
            float up[32];
            sums(c * 32, v);
            sums(wide + c * 32, up);
            if (done) set_empty(0);
            if (p.fin.extra >> 1 & 1) store_chunk<T>(p, 1, row0, col, M, N, box, lane, v);
            if (p.fin.extra >> 2 & 1) store_chunk<T>(p, 2, row0, col, M, N, box, lane, up);
            with_activation(p.fin.act, [&]<int ACT>() {
#pragma unroll
              for (int j = 0; j < 32; ++j) v[j] = activate<ACT>(v[j]) * up[j];
            });
            store_chunk<T>(p, 0, row0, col, M, N, box, lane, v);
          } else {
            uint32_t graw[16], uraw[16];
            load_chunk(p, 0, row0, col, M, N, box, lane, graw);
            load_chunk(p, 1, row0, col, M, N, box, lane, uraw);
            sums(c * 32, v);
            if (done) set_empty(0);
            float du[32], h[32];
            with_activation(p.fin.act, [&]<int ACT>() {
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
            store_chunk<T>(p, 0, row0, col, M, N, box, lane, v);
            store_chunk<T>(p, 1, row0, col, M, N, box, lane, du);
            if (p.fin.extra >> 2 & 1) store_chunk<T>(p, 2, row0, col, M, N, box, lane, h);
          }
        }
      }
      ++i;
    }
  } else {
    if constexpr (HALVES == 2) setmaxnreg_dec<kRegsFirst>();
  }

  tc_fence_before();
  if (p.parts > 1) {
    if constexpr (HALVES == 1) {
      const Unit u = unit_of(p, blockIdx.x / (CG * p.parts));
      const Problem& q = p.prob[u.prob];
      constexpr uint32_t wide = EPI == kGated ? BN / 2 : BN;
      TilePlace at{u.prob, (u.tm * CG + rank) * kRows, u.tn * wide, 0, 0};
      at.tokens = at.t0 < q.m ? min(kRows, q.m - at.t0) : 0u;
      at.features = min(wide, q.n - at.f0);
      finish_tile<T, EPI, BN, kRows, S::kMaxParts>(p.fin, at, ring, p.parts, cta / CG, rank, CG,
                                                   S::kThreads, received, p.status);
    }
  } else if (CG == 2) {
    cluster_sync();  // no CTA exits while its peer may still use its memory
  } else {
    __syncthreads();
  }
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
      tmem_dealloc_pair(tmem_base, 2 * BN);
    else
      tmem_dealloc(tmem_base, 2 * BN);
  }
}

// ------------------------------------------------------------------------------ host
uint64_t over(uint64_t a, uint64_t b) { return (a + b - 1) / b; }

struct Plan {
  int cg, halves;
  uint32_t bn, parts, units, tiles;
  double cost;
  uint32_t bm() const { return kRows * cg; }
  uint32_t wide(const Product& p) const {
    return bn * halves / (p.epilogue == kGated ? 2 : 1);
  }
  uint32_t max_parts() const {
    return bn == 256 ? Shape<2, 256, 1>::kMaxParts : Shape<1, 128, 1>::kMaxParts;
  }
  uint32_t depth() const { return halves == 2 ? 64 : 128; }
};

// Clusters of 1, 2, 4 and 8 CTAs that run at the same time, one CTA per SM.
struct Clusters {
  uint32_t n[4];
};
const Clusters* clusters_of(DeviceInfo* dev) {
  static Clusters all[64];
  static felix_impl::PerDeviceOnce once;
  const int rc = once.run(dev->ordinal, [&] {
    const auto kernel = ffn_product_kernel<__half, kLinear, 1, 128, 1>;
    int rc = int(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      kSmemBytes));
    for (uint32_t i = 0; i < 4 && !rc; ++i) {
      cudaLaunchConfig_t cfg{};
      cfg.gridDim = dim3(uint32_t(dev->num_sms) << i);
      cfg.blockDim = dim3(Shape<1, 128, 1>::kThreads);
      cfg.dynamicSmemBytes = kSmemBytes;
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim = {1u << i, 1, 1};
      cfg.attrs = attr;
      cfg.numAttrs = 1;
      int n = 0;
      rc = int(cudaOccupancyMaxActiveClusters(&n, kernel, &cfg));
      all[dev->ordinal].n[i] = uint32_t(n);
      if (!rc && n == 0) rc = int(cudaErrorInvalidConfiguration);
    }
    return rc;
  });
  return rc ? nullptr : &all[dev->ordinal];
}

// When the last of `units` is done that take tiles off one queue, problem after problem, each
// for `block` us per block of its depth (more by `ragged` where operands' rows are) and some
// more, `least` us at any rate.
double makespan(const Product& p, const Plan& r, uint32_t units, double block, double least,
                double ragged) {
  struct Group {
    double free;     // when these units are
    uint64_t units;
  };
  Group groups[16] = {{0.0, units}};  // by time; at most two more per problem are open at once
  uint32_t n = 1;
  for (uint32_t i = 0; i < p.problems; ++i) {
    uint64_t tiles = over(p.m[i], r.bm()) * over(p.n[i], r.wide(p));
    // rows of no whole 128-byte lines: two requests for one, each row in two lines
    const bool ragged_a = (p.a_mn[i] ? p.m[i] : p.k[i]) % 64, ragged_b = (p.b_mn[i] ? p.n[i] : p.k[i]) % 64;
    const double rows = 1 + ragged / 2 * (int(ragged_a) + int(ragged_b));
    const double length = std::max(
        rows * block * double(over(over(p.k[i], r.depth()) * p.segments[i], r.parts)) + 0.3 * least,
        least);
    while (tiles) {
      // many waves of units that are level keep their distances: all but the last few at once
      if (tiles > 8 * uint64_t(units) && groups[n - 1].free - groups[0].free <= 2 * length) {
        const uint64_t waves = tiles / units - 4;
        for (uint32_t j = 0; j < n; ++j) groups[j].free += double(waves) * length;
        tiles -= waves * units;
      }
      const uint64_t take = std::min(tiles, groups[0].units);
      const double until = groups[0].free + length;
      tiles -= take;
      groups[0].units -= take;
      if (!groups[0].units) std::copy(groups + 1, groups + n--, groups);
      uint32_t at = n;
      while (at && groups[at - 1].free > until) --at;
      if (at && groups[at - 1].free == until) {
        groups[at - 1].units += take;
      } else if (n < 16) {
        std::copy_backward(groups + at, groups + n, groups + n + 1);
        groups[at] = {until, take};
        ++n;
      } else {
        groups[at ? at - 1 : 0].units += take;
      }
    }
  }
  return groups[n - 1].free;
}

// Tiles of one shape, each in `parts` parts of its depth, with an estimate of the time in us:
// waves of 128-deep blocks at the rate that the shape reaches with all SMs at work (one CTA's
// and narrow pairs' tiles are bound by their operands from the L2, 120 GB/s an SM; 256 wide
// and more by the tensor cores), the start and the last epilogue, and for parts the cluster's
// barrier, the exchange and the sums. Measured, tokens x depth x features, us, one CTA |
// pair 128 | 256 | two halves wide: 500 x 4096 x 4096 23.2 | 20.8 | 29.0 | 47.8,
// 500 x 11264 x 4096 54 | 45 | 66 | 111, 2000 x 4096 x 4096 75 | 59 | 51 | 51, 777 x 1024 x
// 5008 13.7 | 16.9 | 17.6 | 19.7; one CTA's tiles of 128 x 4096 x 4096 in 1, 2, 4 parts 22.7,
// 17.5, 14.5; pairs' of 500 x 11264 x 4096 in 2 42.
Plan plan_for(const Product& p, int cg, uint32_t bn, int halves, uint32_t parts, uint32_t units) {
  Plan r{};
  r.cg = cg;
  r.bn = bn;
  r.halves = halves;
  r.parts = parts;
  uint64_t tiles = 0;
  for (uint32_t i = 0; i < p.problems; ++i) tiles += over(p.m[i], r.bm()) * over(p.n[i], r.wide(p));
  r.tiles = uint32_t(std::min<uint64_t>(tiles, 0x7fffffff));
  r.units = std::min(units, r.tiles);
  double block = cg == 1 ? 0.555 : halves == 2 ? 1.16 : bn == 256 ? 0.63 : 0.44;
  if (p.epilogue != kLinear) block *= bn == 256 ? 1.06 : 1.15;  // two values a result
  block *= r.depth() / 128.0;
  // a tile's own: its turn in the queue, its epilogue where that is longer than its products
  const double least = cg == 1 ? 1.9 : halves == 2 ? 9.0 : bn == 256 ? 5.8 : 3.9;
  const double ends = cg == 1 ? 4.8 : halves == 2 ? 7.8 : bn == 256 ? 6.2 : 5.5;
  // 2000 x 4104 x 4096 against 4096 deep: 106, 85, 61, 53 us for 74, 59, 50, 51
  const double ragged = bn == 128 ? 0.42 : halves == 2 ? 0.05 : 0.2;
  r.cost = ends + makespan(p, r, units, block, least, ragged);
  if (parts > 1) r.cost += bn == 256 ? 4.5 : 2.5 + 0.3 * parts;
  return r;
}

Plan make_plan(const Product& p, const Clusters& clusters) {
  Plan best = plan_for(p, 2, 256, 1, 1, clusters.n[1]);
  auto consider = [&](const Plan& r) {
    if (r.cost < best.cost) best = r;
  };
  consider(plan_for(p, 2, 128, 1, 1, clusters.n[1]));
  consider(plan_for(p, 1, 128, 1, 1, clusters.n[0]));
  if (p.epilogue == kLinear && p.act <= FELIX_ACT_RELU && (p.problems > 1 || !p.out[1].p))
    consider(plan_for(p, 2, 256, 2, 1, clusters.n[1]));
  // in parts: one wave of clusters of 2, 4 or 8 CTAs, parts of 256 at least
  uint32_t least = ~0u;
  for (uint32_t i = 0; i < p.problems; ++i)
    least = std::min<uint32_t>(least, uint32_t(over(p.k[i], 128)) * p.segments[i]);
  for (int i = 1; i < 4; ++i) {
    auto split = [&](int cg, uint32_t bn) {
      const Plan r = plan_for(p, cg, bn, 1, (1u << i) / cg, clusters.n[i]);
      if (r.parts > 1 && r.parts <= r.max_parts() && r.tiles <= clusters.n[i] &&
          least >= 2 * r.parts)
        consider(r);
    };
    split(1, 128);
    split(2, 128);
    split(2, 256);
  }
  return best;
}

// Problems [from, to) of a product of several.
Product some_of(const Product& x, uint32_t from, uint32_t to) {
  Product y;
  y.bf16 = x.bf16;
  y.problems = to - from;
  uint32_t first = 0, operand = 0;
  for (uint32_t i = 0; i < from; ++i) first += x.segments[i];
  for (uint32_t i = from; i < to; ++i) {
    const uint32_t j = i - from;
    y.m[j] = x.m[i];
    y.n[j] = x.n[i];
    y.k[j] = x.k[i];
    y.segments[j] = x.segments[i];
    y.a_mn[j] = x.a_mn[i];
    y.b_mn[j] = x.b_mn[i];
    y.out[j] = x.out[i];
    for (uint32_t s = 0; s < x.segments[i]; ++s, ++operand) {
      y.a[operand] = x.a[first + operand];
      y.b[operand] = x.b[first + operand];
    }
  }
  return y;
}

// How many of a product's problems, which come deepest first, make the first of two launches;
// 0: one launch is best. Problems of very different depth have no parts in common: 479 x 128
// x 10880 backward, dx 21760 deep and the weights' gradients 479, takes 101 us in one launch
// and 59 in two. Only for a clear gain: one launch reads weights while it writes gradients
// (20 x 4096 x 11264 63 us against 68 in two).
uint32_t two_launches(const Product& x, const Clusters& clusters, double one) {
  auto depth = [&](uint32_t i) { return over(x.k[i], 128) * x.segments[i]; };
  uint32_t best = 0;
  one *= 0.9;
  for (uint32_t s = 1; s < x.problems; ++s) {
    if (depth(s - 1) < 4 * depth(s)) continue;
    const double two = make_plan(some_of(x, 0, s), clusters).cost +
                       make_plan(some_of(x, s, x.problems), clusters).cost;
    if (two < one) {
      one = two;
      best = s;
    }
  }
  return best;
}

// Tensor map of an operand: whole 64-wide blocks as a third dimension where its
// contiguous extent is a multiple of 64, two dimensions otherwise.
int encode_operand(CUtensorMap* map, const Mat& x, bool mn, bool whole, uint32_t rows, uint32_t k,
                   uint32_t box_rows, uint32_t depth) {
  const uint64_t inner = mn ? rows : k, outer = mn ? k : rows;
  // a single row's distance to the next one is never used, but has to be encodable
  const uint64_t pitch = outer > 1 ? uint64_t(x.ld) * 2 : (inner * 2 + 15) / 16 * 16;
  if (whole)
    return felix_impl::encode_tmap_3d_f16(map, x.p, 64, outer, inner / 64, pitch, 128, 64,
                                          mn ? depth : box_rows, mn ? box_rows / 64 : depth / 64);
  return felix_impl::encode_tmap_2d_f16(map, x.p, inner, outer, pitch, 64, mn ? depth : box_rows);
}

template <class T, int EPI, int CG, int BN, int HALVES>
FelixCode launch_shape(DeviceInfo* dev, const Params& p, const Plan& r, cudaStream_t stream) {
  const auto kernel = ffn_product_kernel<T, EPI, CG, BN, HALVES>;
  static felix_impl::PerDeviceOnce once;
  const int rc = once.run(dev->ordinal, [&] {
    if (HALVES == 2) {
      cudaFuncAttributes attr;
      const cudaError_t e = cudaFuncGetAttributes(&attr, kernel);
      if (e != cudaSuccess) return int(e);
      if (attr.numRegs != kRegsLaunch) return -1;
    }
    return int(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    kSmemBytes));
  });
  if (rc == -1)
    return felix_impl::api_error("feed-forward product: built with another register count than "
                                 "its register split assumes");
  if (rc) return felix_impl::launch_error(cudaError_t(rc), "feed-forward product: attributes");
  const cudaError_t e =
      launch_behind(kernel, r.units * r.parts * CG, 1, Shape<CG, BN, HALVES>::kThreads, kSmemBytes,
                    CG * r.parts, stream, p);
  if (e != cudaSuccess) return felix_impl::launch_error(e, "feed-forward product: launch failed");
  return FelixCode{FELIX_SUCCESS, cudaSuccess};
}

template <class T, int EPI>
FelixCode launch(DeviceInfo* dev, const Params& p, const Plan& r, cudaStream_t stream) {
  if constexpr (EPI == kLinear)
    if (r.halves == 2) return launch_shape<T, EPI, 2, 256, 2>(dev, p, r, stream);
  return r.cg == 1     ? launch_shape<T, EPI, 1, 128, 1>(dev, p, r, stream)
         : r.bn == 256 ? launch_shape<T, EPI, 2, 256, 1>(dev, p, r, stream)
                       : launch_shape<T, EPI, 2, 128, 1>(dev, p, r, stream);
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

// Whether rows consist of whole vectors of n elements.
bool whole(uint32_t n, const void* p, int64_t ld, uint32_t rows, uint32_t cols) {
  return reinterpret_cast<uintptr_t>(p) % (2 * n) == 0 && cols % n == 0 && (rows <= 1 || ld % n == 0);
}

}  // namespace product

using namespace product;

FelixCode product_launch(DeviceInfo* dev, const Product& x, void* workspace, cudaStream_t stream) {
  const Clusters* clusters = clusters_of(dev);
  if (!clusters) return felix_impl::launch_error(cudaGetLastError(), "feed-forward product: device");
  const Plan r = make_plan(x, *clusters);
  if (r.tiles > 0x3fffffffu)
    return felix_impl::api_error("feed-forward product: too many tiles");
  if (const uint32_t first = two_launches(x, *clusters, r.cost)) {
    const FelixCode code = product_launch(dev, some_of(x, 0, first), workspace, stream);
    if (code.type != FELIX_SUCCESS) return code;
    return product_launch(dev, some_of(x, first, x.problems), workspace, stream);
  }
  const bool gated = x.epilogue == kGated;
  Params p{};
  p.fin = finish_of(x);
  p.problems = x.problems;
  p.tiles = r.tiles;
  p.parts = r.parts;
  p.group_m = r.halves == 2 ? 12 : r.cg == 2 ? 8 : 16;
  p.dyn = r.parts == 1 && r.tiles >= 4 * r.units;
  const uint32_t depth = r.depth(), wide = r.wide(x), b_rows = r.bn / r.cg;
  uint32_t tile = 0, map = 0;
  for (uint32_t i = 0; i < x.problems; ++i) {
    Problem& q = p.prob[i];
    q.m = x.m[i];
    q.n = x.n[i];
    q.tiles_m = uint32_t(over(q.m, r.bm()));
    q.tiles_n = uint32_t(over(q.n, wide));
    q.tile0 = tile;
    tile += q.tiles_m * q.tiles_n;
    q.kb_seg = uint32_t(over(x.k[i], depth));
    q.kb = q.kb_seg * x.segments[i];
    q.map = map;
    q.a_mn = x.a_mn[i];
    q.b_mn = x.b_mn[i];
    // whole 64-wide blocks (a stage of 64 k is one block of K-major rows; a gated CTA's two
    // boxes lie side by side)
    q.a_3d = q.a_mn ? q.m % 64 == 0 : x.k[i] % 64 == 0 && depth == 128;
    q.b_3d = q.b_mn ? q.n % 64 == 0
                    : x.k[i] % 64 == 0 && depth == 128 && !(gated && r.cg == 1);
    const uint32_t operands = gated ? 2 : x.segments[i];
    for (uint32_t s = 0; s < operands; ++s, ++map) {
      if (s < x.segments[i] &&
          encode_operand(&p.a[map], x.a[map], q.a_mn, q.a_3d, q.m, x.k[i], kRows, depth))
        return felix_impl::api_error("feed-forward product: cuTensorMapEncodeTiled failed");
      if (encode_operand(&p.b[map], x.b[map], q.b_mn, q.b_3d, q.n, x.k[i],
                         gated && r.cg == 1 ? b_rows / 2 : b_rows, depth))
        return felix_impl::api_error("feed-forward product: cuTensorMapEncodeTiled failed");
    }
  }
  for (uint32_t i = 0; i < kMaxProblems; ++i) {
    if (!x.out[i].p) continue;
    const uint32_t prob = std::min(i, x.problems - 1), m = x.m[prob], n = x.n[prob];
    p.out_vec |= uint32_t(whole(8, x.out[i].p, x.out[i].ld, m, n)) << i;
    p.out_sectors |= uint32_t(whole(16, x.out[i].p, x.out[i].ld, m, n)) << i;
  }
  for (uint32_t i = 0; i < 2; ++i) {
    if (!x.in[i].p) continue;
    p.in_vec |= uint32_t(whole(8, x.in[i].p, x.in[i].ld, x.m[0], x.n[0])) << i;
    p.in_sectors |= uint32_t(whole(16, x.in[i].p, x.in[i].ld, x.m[0], x.n[0])) << i;
  }
  p.dyn_counter = static_cast<unsigned*>(workspace) + (felix_impl::kWsMaxCounters - 2);
  p.status = dev->status_word;
  return x.bf16 ? launch<__nv_bfloat16>(dev, p, r, x.epilogue, stream)
                : launch<__half>(dev, p, r, x.epilogue, stream);
}

}  // namespace felix_ffn
