// Tiles handed out at run time to persistent CTAs or CTA pairs, passed to every role
// of the CTA (and of its peer) through a small queue in shared memory.
#pragma once
#include <cstdint>

#include "sm100_ptx.cuh"

namespace felix_sm100 {

// Dynamic whole-tile schedule of the persistent products. With a static stride the
// persistent CTAs drift apart over many waves (16384^3: 55 waves), so the CTAs
// running at the same time stop sharing A and B panels in L2: measured 18.9 GB
// of DRAM reads for 1.07 GB of operands. Instead the leader CTA's producer
// takes each next whole tile from a global counter (one atomicAdd per tile,
// fetched one tile ahead) and hands it to every role of its CTA, and of the
// peer CTA of a pair, through a kTq-slot queue in shared memory: tq[slot],
// tq_full[slot] (completed by the producer's arrival; the peer's copy by a
// remote arrival after a remote store) and the leader's tq_empty[slot] (one
// arrival per consuming warp role, remote ones from the peer). Tiles then run
// in the order the CTAs become free: neighbours in the grouped raster run
// together. Each tile is still computed by one CTA (pair) in a fixed k order,
// so results do not depend on the assignment. A tile id >= tiles ends the walk.
constexpr uint32_t kTq = 4;
struct TileQueue {
  uint32_t* tq;
  uint64_t* full;
  uint64_t* empty;
  uint32_t n;  // queue entries used so far
};

__device__ __forceinline__ bool tq_push(TileQueue& q, uint32_t t, bool pair,
                                        volatile int* abort_flag, unsigned* status) {
  const uint32_t slot = q.n % kTq, par = (q.n / kTq) & 1u;
  if (!mbar_wait_cluster(&q.empty[slot], par ^ 1u, abort_flag, status, kWdTileQueue))
    return false;
  q.tq[slot] = t;
  if (pair) {
    st_shared_cluster_u32(mapa_shared(smem_u32(&q.tq[slot]), 1), t);
    mbar_arrive_cluster(mapa_shared(smem_u32(&q.full[slot]), 1));
  }
  mbar_arrive(&q.full[slot]);
  ++q.n;
  return true;
}

// Waits for the next queue entry and reads it (every calling thread); the
// caller then releases the slot once per warp with tq_release.
__device__ __forceinline__ bool tq_pop(TileQueue& q, uint32_t& t, uint32_t& slot,
                                       volatile int* abort_flag, unsigned* status) {
  slot = q.n % kTq;
  const uint32_t par = (q.n / kTq) & 1u;
  if (!mbar_wait_cluster(&q.full[slot], par, abort_flag, status, kWdTileQueue)) return false;
  t = reinterpret_cast<volatile uint32_t*>(q.tq)[slot];
  ++q.n;
  return true;
}

__device__ __forceinline__ void tq_release(TileQueue& q, uint32_t slot, uint32_t rank) {
  if (rank == 0)
    mbar_arrive(&q.empty[slot]);
  else
    mbar_arrive_cluster(mapa_shared(smem_u32(&q.empty[slot]), 0));
}

}  // namespace felix_sm100
