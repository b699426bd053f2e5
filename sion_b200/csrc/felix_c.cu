// C-ABI layer and host runtime of libfelix_b200.so: per-device state, tensor-map
// encoding, library-owned scratch, error reporting, the device watchdog word,
// and the extern "C" entry points declared in include/felix_c.h.
#include <cuda.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdio>
#include <cstring>
#include <exception>
#include <initializer_list>
#include <map>
#include <mutex>
#include <thread>
#include <tuple>
#include <utility>
#include <vector>

#include "felix_internal.h"
#include "sm100_ptx.cuh"

// Watchdog word, one per device (each device holds its own copy of a __device__
// variable). Its device address is looked up once per device.
__device__ unsigned g_felix_watchdog_word;

namespace felix_impl {

namespace {
thread_local int t_last_cuda = 0;
// Memory of its own: errors are recorded, out of entry points that may not throw, where
// there may be none left. Longer texts are cut off.
thread_local char t_last_msg[512] = "";

std::mutex g_mu;
DeviceInfo g_dev[64];
bool g_dev_ready[64] = {false};

struct Buffer {
  void* ptr = nullptr;
  size_t bytes = 0;
};
struct WsEntry {
  std::mutex mu;  // held by a call from here to its last launch
  Buffer own;
  Buffer captured;                 // of the capture with this id, which owns it
  unsigned long long capture = 0;
};
// Device, stream, and the host thread where the handle stands for each thread's own
// stream. Entries stay: a map's elements do not move.
using WsKey = std::tuple<int, cudaStream_t, std::thread::id>;
std::map<WsKey, WsEntry> g_ws;

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                   const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                   const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                   CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn g_encode = nullptr;
std::once_flag g_encode_once;

void load_encode() {
  void* fn = nullptr;
  cudaDriverEntryPointQueryResult q;
  if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q) ==
          cudaSuccess &&
      q == cudaDriverEntryPointSuccess)
    g_encode = reinterpret_cast<EncodeTiledFn>(fn);
}
}  // namespace

FelixCode api_error(const char* msg, cudaError_t e) {
  t_last_cuda = int(e);
  std::snprintf(t_last_msg, sizeof(t_last_msg), "%s", msg ? msg : "");
  return FelixCode{FELIX_API_ERROR, e};
}

FelixCode launch_error(cudaError_t e, const char* msg) {
  t_last_cuda = int(e);
  std::snprintf(t_last_msg, sizeof(t_last_msg), "%s: %s", msg ? msg : "", cudaGetErrorString(e));
  return FelixCode{FELIX_KERNEL_LAUNCH_FAILED, e};
}

DeviceInfo* current_device_info() {
  int d = -1;
  if (cudaGetDevice(&d) != cudaSuccess || d < 0 || d >= 64) return nullptr;
  // A host thread that has made no call of the runtime has no context yet, and
  // encoding a tensor map, which is a call of the driver, would be refused there. The
  // look-up gives it the device's (and leaves one that the caller has set as it is).
  static thread_local int t_bound = -1;
  if (t_bound != d) {
    void* addr = nullptr;
    if (cudaGetSymbolAddress(&addr, g_felix_watchdog_word) != cudaSuccess) return nullptr;
    t_bound = d;
  }
  std::lock_guard<std::mutex> lk(g_mu);
  if (!g_dev_ready[d]) {
    DeviceInfo& di = g_dev[d];
    di.ordinal = d;
    if (cudaDeviceGetAttribute(&di.num_sms, cudaDevAttrMultiProcessorCount, d) != cudaSuccess)
      return nullptr;
    cudaDeviceGetAttribute(&di.max_smem_optin, cudaDevAttrMaxSharedMemoryPerBlockOptin, d);
    void* addr = nullptr;
    if (cudaGetSymbolAddress(&addr, g_felix_watchdog_word) != cudaSuccess) return nullptr;
    di.status_word = static_cast<unsigned*>(addr);
    g_dev_ready[d] = true;
  }
  return &g_dev[d];
}

static WsEntry& workspace_entry(int device, cudaStream_t stream) {
  const auto thread =
      stream == cudaStreamPerThread ? std::this_thread::get_id() : std::thread::id();
  std::lock_guard<std::mutex> lk(g_mu);
  return g_ws[WsKey(device, stream, thread)];
}

// Allocations are no part of a capture, of this thread or another.
struct NotCaptured {
  cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
  NotCaptured() { cudaThreadExchangeStreamCaptureMode(&mode); }
  ~NotCaptured() { cudaThreadExchangeStreamCaptureMode(&mode); }
};

constexpr size_t kWsLeast = size_t(1) << 20;

// Buffers whose graphs are gone, for the next captures. They outlive the process's
// static objects: graphs may be destroyed after those.
struct Spare {
  std::mutex mu;
  std::vector<Buffer> free[64];
};
static Spare& spare() {
  static Spare* s = new Spare;
  return *s;
}
struct GraphBuffer {
  int device;
  Buffer b;
};
// Called when the last graph that holds the buffer is gone and has run to its end; may
// not call CUDA.
static void graph_gone(void* p) {
  GraphBuffer* g = static_cast<GraphBuffer*>(p);
  Spare& s = spare();
  try {
    std::lock_guard<std::mutex> lk(s.mu);
    s.free[g->device].push_back(g->b);
  } catch (...) {  // no memory for the list: the buffer is lost
  }
  delete g;
}

// A zeroed buffer that belongs to the graph. It cannot be zeroed on the stream, whose
// work is being recorded.
static Buffer graph_buffer(int device, cudaGraph_t graph, size_t bytes) {
  NotCaptured outside;
  Buffer b;
  Spare& s = spare();
  {
    std::lock_guard<std::mutex> lk(s.mu);
    auto& f = s.free[device];
    auto best = f.end();
    for (auto i = f.begin(); i != f.end(); ++i)
      if (i->bytes >= bytes && (best == f.end() || i->bytes < best->bytes)) best = i;
    if (best != f.end()) {
      b = *best;
      f.erase(best);
    }
  }
  if (!b.ptr) {
    b.bytes = bytes < kWsLeast ? kWsLeast : bytes;
    if (cudaMalloc(&b.ptr, b.bytes) != cudaSuccess) return {};
  }
  auto* g = new GraphBuffer{device, b};
  cudaStream_t side = nullptr;
  cudaUserObject_t object = nullptr;
  bool ok = cudaStreamCreateWithFlags(&side, cudaStreamNonBlocking) == cudaSuccess;
  ok = ok && cudaMemsetAsync(b.ptr, 0, b.bytes, side) == cudaSuccess &&
       cudaStreamSynchronize(side) == cudaSuccess;
  if (side) cudaStreamDestroy(side);
  ok = ok && cudaUserObjectCreate(&object, g, graph_gone, 1, cudaUserObjectNoDestructorSync) ==
                 cudaSuccess;
  if (!ok) {
    graph_gone(g);
    return {};
  }
  if (cudaGraphRetainUserObject(graph, object, 1, cudaGraphUserObjectMove) != cudaSuccess) {
    cudaUserObjectRelease(object, 1);  // back to the spare ones
    return {};
  }
  return b;
}

Workspace library_workspace(DeviceInfo* dev, cudaStream_t stream, size_t bytes) {
  WsEntry& w = workspace_entry(dev->ordinal, stream);
  std::unique_lock<std::mutex> lk(w.mu);
  cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
  unsigned long long id = 0;
  cudaGraph_t graph = nullptr;
  if (cudaStreamGetCaptureInfo(stream, &status, &id, &graph) != cudaSuccess) {
    cudaGetLastError();  // the launch will say so
    status = cudaStreamCaptureStatusNone;
  }
  if (status == cudaStreamCaptureStatusActive) {
    if (w.capture != id || w.captured.bytes < bytes) {
      w.captured = graph_buffer(dev->ordinal, graph, bytes);  // a smaller one stays the graph's
      w.capture = id;
    }
    return {w.captured.ptr, std::move(lk)};
  }
  if (w.own.bytes >= bytes) return {w.own.ptr, std::move(lk)};
  NotCaptured outside;
  if (w.own.ptr) {
    // The old buffer may still be in use by work queued on this stream.
    cudaStreamSynchronize(stream);
    cudaFree(w.own.ptr);
    w.own = {};
  }
  const size_t sz = bytes < kWsLeast ? kWsLeast : bytes;
  if (cudaMalloc(&w.own.ptr, sz) != cudaSuccess) {
    w.own.ptr = nullptr;
    return {};
  }
  if (cudaMemsetAsync(w.own.ptr, 0, sz, stream) != cudaSuccess) return {};
  w.own.bytes = sz;
  return {w.own.ptr, std::move(lk)};
}

static int encode_2d(CUtensorMap* map, const void* base, uint64_t inner, uint64_t outer,
                     uint64_t pitch, uint32_t bi, uint32_t bo, CUtensorMapSwizzle sw) {
  std::call_once(g_encode_once, load_encode);
  if (!g_encode) return -1;
  cuuint64_t dims[2] = {inner, outer};
  cuuint64_t strides[1] = {pitch};
  cuuint32_t box[2] = {bi, bo};
  cuuint32_t estr[2] = {1, 1};
  CUresult r = g_encode(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<void*>(base), dims,
                        strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, sw,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : int(r);
}

int encode_tmap_2d_f16(CUtensorMap* map, const void* base, uint64_t inner, uint64_t outer,
                       uint64_t pitch, uint32_t bi, uint32_t bo) {
  return encode_2d(map, base, inner, outer, pitch, bi, bo, CU_TENSOR_MAP_SWIZZLE_128B);
}
int encode_tmap_2d_f16_swizzle(CUtensorMap* map, const void* base, uint64_t inner,
                               uint64_t outer, uint64_t pitch, uint32_t bi, uint32_t bo,
                               int swizzle_bytes) {
  CUtensorMapSwizzle sw = CU_TENSOR_MAP_SWIZZLE_NONE;
  if (swizzle_bytes == 32) sw = CU_TENSOR_MAP_SWIZZLE_32B;
  else if (swizzle_bytes == 64) sw = CU_TENSOR_MAP_SWIZZLE_64B;
  else if (swizzle_bytes == 128) sw = CU_TENSOR_MAP_SWIZZLE_128B;
  return encode_2d(map, base, inner, outer, pitch, bi, bo, sw);
}

int encode_tmap_3d_f16(CUtensorMap* map, const void* base, uint64_t inner, uint64_t outer1,
                       uint64_t outer2, uint64_t pitch1, uint64_t pitch2, uint32_t bi,
                       uint32_t bo1, uint32_t bo2) {
  std::call_once(g_encode_once, load_encode);
  if (!g_encode) return -1;
  cuuint64_t dims[3] = {inner, outer1, outer2};
  cuuint64_t strides[2] = {pitch1, pitch2};
  cuuint32_t box[3] = {bi, bo1, bo2};
  cuuint32_t estr[3] = {1, 1, 1};
  CUresult r = g_encode(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(base), dims,
                        strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : int(r);
}

int encode_tmap_3d_f32(CUtensorMap* map, const void* base, uint64_t inner, uint64_t outer1,
                       uint64_t outer2, uint64_t pitch1, uint64_t pitch2, uint32_t bi,
                       uint32_t bo1, uint32_t bo2) {
  std::call_once(g_encode_once, load_encode);
  if (!g_encode) return -1;
  cuuint64_t dims[3] = {inner, outer1, outer2};
  cuuint64_t strides[2] = {pitch1, pitch2};
  cuuint32_t box[3] = {bi, bo1, bo2};
  cuuint32_t estr[3] = {1, 1, 1};
  CUresult r = g_encode(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 3, const_cast<void*>(base), dims,
                        strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : int(r);
}

int encode_tmap_2d_f32(CUtensorMap* map, const void* base, uint64_t inner, uint64_t outer,
                       uint64_t pitch, uint32_t bi, uint32_t bo, bool swizzle128) {
  std::call_once(g_encode_once, load_encode);
  if (!g_encode) return -1;
  cuuint64_t dims[2] = {inner, outer};
  cuuint64_t strides[1] = {pitch};
  cuuint32_t box[2] = {bi, bo};
  cuuint32_t estr[2] = {1, 1};
  CUresult r = g_encode(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 2, const_cast<void*>(base), dims,
                        strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        swizzle128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : int(r);
}

int encode_tmap_2d_f16_noswizzle(CUtensorMap* map, const void* base, uint64_t inner,
                                 uint64_t outer, uint64_t pitch, uint32_t bi, uint32_t bo) {
  return encode_2d(map, base, inner, outer, pitch, bi, bo, CU_TENSOR_MAP_SWIZZLE_NONE);
}

__global__ void scale_half_kernel(__half* c, size_t n, float beta) {
  for (size_t i = blockIdx.x * size_t(blockDim.x) + threadIdx.x; i < n;
       i += size_t(gridDim.x) * blockDim.x)
    c[i] = beta == 0.f ? __float2half_rn(0.f) : __float2half_rn(beta * __half2float(c[i]));
}
__global__ void scale_float_kernel(float* c, size_t n, float beta) {
  for (size_t i = blockIdx.x * size_t(blockDim.x) + threadIdx.x; i < n;
       i += size_t(gridDim.x) * blockDim.x)
    c[i] = beta == 0.f ? 0.f : beta * c[i];
}

FelixCode scale_half_matrix(__half* C, size_t n, float beta, cudaStream_t stream) {
  if (n == 0) return FelixCode{FELIX_SUCCESS, cudaSuccess};
  scale_half_kernel<<<592, 256, 0, stream>>>(C, n, beta);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return launch_error(e, "scale");
  return FelixCode{FELIX_SUCCESS, cudaSuccess};
}
FelixCode scale_float_matrix(float* C, size_t n, float beta, cudaStream_t stream) {
  if (n == 0) return FelixCode{FELIX_SUCCESS, cudaSuccess};
  scale_float_kernel<<<592, 256, 0, stream>>>(C, n, beta);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return launch_error(e, "scale");
  return FelixCode{FELIX_SUCCESS, cudaSuccess};
}

// One CTA waits on an mbarrier that nothing arrives on; the bounded wait gives
// up after limit_ns, records kWdProbe in the watchdog word and the kernel
// returns. Exercises the same wait routine the GEMM/attention kernels use.
__global__ void watchdog_probe_kernel(unsigned* status, unsigned long long limit_ns) {
  __shared__ uint64_t bar;
  __shared__ int abort_flag;
  if (threadIdx.x == 0) {
    felix_sm100::mbar_init(&bar, 1);
    abort_flag = 0;
    felix_sm100::fence_mbar_init();
  }
  __syncthreads();
  if (threadIdx.x == 0)
    felix_sm100::mbar_wait(&bar, 0, &abort_flag, status, felix_sm100::kWdProbe, limit_ns);
  __syncthreads();
}

FelixCode watchdog_probe_launch(uint32_t limit_us, cudaStream_t stream) {
  if (limit_us == 0 || limit_us > 1000000) return api_error("watchdog_probe: limit_us in 1..1e6");
  DeviceInfo* dev = current_device_info();
  if (!dev) return launch_error(cudaGetLastError(), "watchdog_probe: no device");
  watchdog_probe_kernel<<<1, 32, 0, stream>>>(dev->status_word,
                                              (unsigned long long)limit_us * 1000ull);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return launch_error(e, "watchdog_probe");
  return FelixCode{FELIX_SUCCESS, cudaSuccess};
}

int finish(FelixCode c) {
  if (c.type == FELIX_SUCCESS) {
    t_last_cuda = 0;
    t_last_msg[0] = 0;
  }
  return c.type;
}

}  // namespace felix_impl

using namespace felix_impl;

// The entry points below may not throw (scratch is kept in a std::map).
template <class F>
static int guarded(F&& f) {
  try {
    return finish(f());
  } catch (const std::exception& e) {
    return api_error(e.what(), cudaErrorMemoryAllocation).type;
  } catch (...) {
    return api_error("unknown C++ exception", cudaErrorUnknown).type;
  }
}

// Whether a caller's pointers are multiples of n (a power of two). Kernels read and
// write vectors there: what is not aligned is refused, it would fault the device.
static bool aligned(size_t n, std::initializer_list<const void*> pointers) {
  for (const void* p : pointers)
    if (reinterpret_cast<uintptr_t>(p) & (n - 1)) return false;
  return true;
}
constexpr char kWorkspaceAlignment[] = "workspace must be 16-byte aligned";

// log2 of a page size, or -1 where it is none.
static int page_shift_of(uint32_t page_size) {
  if (page_size < felix_kv4::kBlock || page_size > felix_kv4::kMaxPageSize ||
      (page_size & (page_size - 1)))
    return -1;
  return __builtin_ctz(page_size);
}

static FelixCode view_of(const felix_kv4_cache* c, felix_kv4::CacheView* v) {
  // arrays without elements may be null
  if (!c || !c->pages || (!c->table && c->slots && c->width) || (!c->lens && c->slots))
    return api_error("kv4: null cache or array");
  if (c->head_dim != 64 && c->head_dim != 128) return api_error("kv4: head_dim must be 64 or 128");
  const int shift = page_shift_of(c->page_size);
  if (shift < 0) return api_error("kv4: page_size must be a power of two, 16..4096");
  if (c->kv_heads == 0 || c->kv_heads > 65535) return api_error("kv4: kv_heads must be 1..65535");
  if (c->num_pages == 0 || c->num_pages > 0x7fffffffull)
    return api_error("kv4: num_pages must be 1..2^31-1");
  if (c->slots > (1u << 24) || c->width > 0x7fffffffu / c->page_size)
    return api_error("kv4: too many slots or pages of a slot");
  if (reinterpret_cast<uintptr_t>(c->pages) & 15) return api_error("kv4: pages must be 16-byte aligned");
  v->pages = static_cast<unsigned char*>(c->pages);
  v->table = c->table;
  v->lens = c->lens;
  v->num_pages = c->num_pages;
  v->page_bytes = size_t(c->page_size) * c->kv_heads * (c->head_dim + 8);
  v->slots = c->slots;
  v->width = c->width;
  v->kv_heads = c->kv_heads;
  v->page_shift = uint32_t(shift);
  return FelixCode{FELIX_SUCCESS, cudaSuccess};
}

static FelixCode pages_op(const Kv4PagesOp& o, uint32_t page_size, void* stream) {
  if (!o.refs || !o.refs_out || ((!o.table || !o.table_out) && o.slots && o.width))
    return api_error("kv4: null array");
  if (o.num_pages == 0 || o.num_pages > 0x7fffffffu)
    return api_error("kv4: num_pages must be 1..2^31-1");
  if (o.slots > (1u << 24) || o.n > (1u << 24) || o.width > 0x7fffffffu / page_size)
    return api_error("kv4: too many slots, pages of a slot or list entries");
  if (o.pages && ((reinterpret_cast<uintptr_t>(o.pages) & 15) || o.page_bytes == 0 ||
                  o.page_bytes % 16))
    return api_error("kv4: pages must be 16-byte aligned and their size a multiple of 16");
  return kv4_pages_launch(o, static_cast<cudaStream_t>(stream));
}

extern "C" {

int felix_last_cuda_error(void) { return t_last_cuda; }
const char* felix_last_error_message(void) { return t_last_msg; }
const char* felix_version(void) { return "sion-b200 0.1 (sm_100a)"; }

int felix_num_sms(int* count) {
  DeviceInfo* d = current_device_info();
  if (!d) return launch_error(cudaGetLastError(), "no device").type;
  if (count) *count = d->num_sms;
  return FELIX_SUCCESS;
}

int felix_sgemm(uint32_t M, uint32_t N, uint32_t K, float alpha, const float* A, const float* B,
                float beta, float* C, void* stream) {
  SgemmOptions o;
  return finish(sgemm_launch(M, N, K, alpha, A, B, beta, C, o, nullptr, 0,
                             static_cast<cudaStream_t>(stream)));
}

int felix_sgemm_ex(uint32_t M, uint32_t N, uint32_t K, float alpha, const float* A,
                   const float* B, float beta, float* C, int split_k, void* workspace,
                   size_t workspace_bytes, void* stream) {
  if (split_k < 0) return api_error("sgemm: split_k must be >= 0").type;
  if (!aligned(16, {workspace})) return api_error(kWorkspaceAlignment).type;
  SgemmOptions o;
  o.split_k = split_k;
  return finish(sgemm_launch(M, N, K, alpha, A, B, beta, C, o, workspace, workspace_bytes,
                             static_cast<cudaStream_t>(stream)));
}

int felix_sgemm_noalloc(uint32_t M, uint32_t N, uint32_t K, float alpha, const float* A,
                        const float* B, float beta, float* C, int split_k, void* stream) {
  return finish(sgemm_noalloc_launch(M, N, K, alpha, A, B, beta, C, split_k,
                                     static_cast<cudaStream_t>(stream)));
}

int felix_sgemm_workspace_size(uint32_t M, uint32_t N, uint32_t K, int split_k, size_t* bytes) {
  DeviceInfo* d = current_device_info();
  if (!d) return launch_error(cudaGetLastError(), "no device").type;
  SgemmOptions o;
  o.split_k = split_k;
  if (bytes) *bytes = sgemm_workspace_bytes(M, N, K, o, d->num_sms);
  return FELIX_SUCCESS;
}

int felix_hgemm(uint32_t M, uint32_t N, uint32_t K, float alpha, const void* A, const void* B,
                float beta, void* C, int b_layout, void* stream) {
  if (b_layout != FELIX_B_KN && b_layout != FELIX_B_NK)
    return api_error("hgemm: b_layout must be FELIX_B_KN or FELIX_B_NK").type;
  HgemmOptions o;
  return finish(hgemm_launch(M, N, K, alpha, static_cast<const __half*>(A),
                             static_cast<const __half*>(B), beta, static_cast<__half*>(C),
                             b_layout == FELIX_B_KN, o, nullptr, 0,
                             static_cast<cudaStream_t>(stream)));
}

int felix_hgemm_ex(uint32_t M, uint32_t N, uint32_t K, float alpha, const void* A, const void* B,
                   float beta, void* C, int b_layout, int block_n, int stream_k, int max_ctas,
                   void* workspace, size_t workspace_bytes, void* stream) {
  if (b_layout != FELIX_B_KN && b_layout != FELIX_B_NK)
    return api_error("hgemm: b_layout must be FELIX_B_KN or FELIX_B_NK").type;
  if (stream_k < 0 || stream_k > 2) return api_error("hgemm: stream_k must be 0, 1 or 2").type;
  if (max_ctas < 0) return api_error("hgemm: max_ctas must be >= 0").type;
  if (!aligned(16, {workspace})) return api_error(kWorkspaceAlignment).type;
  HgemmOptions o;
  o.block_n = block_n;
  o.stream_k = stream_k;
  o.max_ctas = max_ctas;
  return finish(hgemm_launch(M, N, K, alpha, static_cast<const __half*>(A),
                             static_cast<const __half*>(B), beta, static_cast<__half*>(C),
                             b_layout == FELIX_B_KN, o, workspace, workspace_bytes,
                             static_cast<cudaStream_t>(stream)));
}

int felix_hgemm_ex2(uint32_t M, uint32_t N, uint32_t K, float alpha, const void* A, const void* B,
                    float beta, void* C, int b_layout, int block_n, int stream_k, int max_ctas,
                    int cta_pair, void* workspace, size_t workspace_bytes, void* stream) {
  if (b_layout != FELIX_B_KN && b_layout != FELIX_B_NK)
    return api_error("hgemm: b_layout must be FELIX_B_KN or FELIX_B_NK").type;
  if (stream_k < 0 || stream_k > 2) return api_error("hgemm: stream_k must be 0, 1 or 2").type;
  if (max_ctas < 0) return api_error("hgemm: max_ctas must be >= 0").type;
  if (!aligned(16, {workspace})) return api_error(kWorkspaceAlignment).type;
  if (cta_pair < 0 || cta_pair > 2) return api_error("hgemm: cta_pair must be 0, 1 or 2").type;
  if (cta_pair == 2 && block_n != 0 && block_n != 256)
    return api_error("hgemm: CTA pairs use 256-wide tiles (block_n 0 or 256)").type;
  HgemmOptions o;
  o.block_n = block_n;
  o.stream_k = stream_k;
  o.max_ctas = max_ctas;
  o.cta_pair = cta_pair;
  return finish(hgemm_launch(M, N, K, alpha, static_cast<const __half*>(A),
                             static_cast<const __half*>(B), beta, static_cast<__half*>(C),
                             b_layout == FELIX_B_KN, o, workspace, workspace_bytes,
                             static_cast<cudaStream_t>(stream)));
}

int felix_hgemm_workspace_size2(uint32_t M, uint32_t N, uint32_t K, int block_n, int stream_k,
                                int max_ctas, int cta_pair, size_t* bytes) {
  DeviceInfo* d = current_device_info();
  if (!d) return launch_error(cudaGetLastError(), "no device").type;
  HgemmOptions o;
  o.block_n = block_n;
  o.stream_k = stream_k;
  o.max_ctas = max_ctas;
  o.cta_pair = cta_pair;
  if (bytes) *bytes = hgemm_workspace_bytes(M, N, K, o, d->num_sms);
  return FELIX_SUCCESS;
}

int felix_hgemm_workspace_size(uint32_t M, uint32_t N, uint32_t K, int block_n, int stream_k,
                               int max_ctas, size_t* bytes) {
  DeviceInfo* d = current_device_info();
  if (!d) return launch_error(cudaGetLastError(), "no device").type;
  HgemmOptions o;
  o.block_n = block_n;
  o.stream_k = stream_k;
  o.max_ctas = max_ctas;
  if (bytes) *bytes = hgemm_workspace_bytes(M, N, K, o, d->num_sms);
  return FELIX_SUCCESS;
}

int felix_flash_attn_fwd(const void* Q, const void* K, const void* V, void* O, float* lse,
                         uint32_t heads, uint32_t batch, uint32_t seqlen, uint32_t head_dim,
                         float scale, void* stream) {
  return finish(flash_attn_launch(static_cast<const __half*>(Q), static_cast<const __half*>(K),
                                  static_cast<const __half*>(V), static_cast<__half*>(O), lse,
                                  heads, batch, seqlen, head_dim, scale, false,
                                  static_cast<cudaStream_t>(stream)));
}

int felix_flash_attn_fwd_ex(const void* Q, const void* K, const void* V, void* O, float* lse,
                            uint32_t heads, uint32_t batch, uint32_t seqlen, uint32_t head_dim,
                            float scale, int causal, void* stream) {
  return finish(flash_attn_launch(static_cast<const __half*>(Q), static_cast<const __half*>(K),
                                  static_cast<const __half*>(V), static_cast<__half*>(O), lse,
                                  heads, batch, seqlen, head_dim, scale, causal != 0,
                                  static_cast<cudaStream_t>(stream)));
}

int felix_flash_attn_bwd(const void* Q, const void* K, const void* V, const void* O,
                         const void* dO, const float* lse, void* dQ, void* dK, void* dV,
                         uint32_t heads, uint32_t batch, uint32_t seqlen, uint32_t head_dim,
                         float scale, int causal, void* workspace, size_t workspace_bytes,
                         void* stream) {
  return finish(flash_attn_bwd_launch(
      static_cast<const __half*>(Q), static_cast<const __half*>(K), static_cast<const __half*>(V),
      static_cast<const __half*>(O), static_cast<const __half*>(dO), lse,
      static_cast<__half*>(dQ), static_cast<__half*>(dK), static_cast<__half*>(dV), heads, batch,
      seqlen, head_dim, scale, causal != 0, workspace, workspace_bytes,
      static_cast<cudaStream_t>(stream)));
}

int felix_flash_attn_bwd_workspace_size(uint32_t heads, uint32_t batch, uint32_t seqlen,
                                        uint32_t head_dim, size_t* bytes) {
  if (bytes) *bytes = flash_attn_bwd_workspace_bytes(heads, batch, seqlen, head_dim);
  return FELIX_SUCCESS;
}

int felix_topk_select(const float* data, float* out, uint32_t num_slices, uint32_t slice_size,
                      uint32_t k, int largest, void* stream) {
  return finish(topk_select_launch(data, out, num_slices, slice_size, k, largest != 0,
                                   static_cast<cudaStream_t>(stream)));
}

int felix_kv4_page_bytes(uint32_t kv_heads, uint32_t head_dim, uint32_t page_size, size_t* bytes) {
  if (head_dim != 64 && head_dim != 128) return api_error("kv4: head_dim must be 64 or 128").type;
  if (page_shift_of(page_size) < 0)
    return api_error("kv4: page_size must be a power of two, 16..4096").type;
  if (kv_heads == 0 || kv_heads > 65535)
    return api_error("kv4: kv_heads must be 1..65535").type;
  if (bytes) *bytes = size_t(page_size) * kv_heads * (head_dim + 8);
  return FELIX_SUCCESS;
}

int felix_kv4_append(const felix_kv4_cache* cache, const void* key, const void* value, int dtype,
                     uint32_t rows, const int64_t* key_strides, const int64_t* value_strides,
                     const int32_t* counts, void* stream) {
  return guarded([&]() -> FelixCode {
    felix_kv4::CacheView v;
    const FelixCode rc = view_of(cache, &v);
    if (rc.type != FELIX_SUCCESS) return rc;
    if (dtype != FELIX_F16 && dtype != FELIX_BF16)
      return api_error("kv4_append: key and value must be fp16 or bf16");
    if (rows > 0x7fffffffu) return api_error("kv4_append: at most 2^31-1 rows");
    if (rows == 0 || v.slots == 0) return FelixCode{FELIX_SUCCESS, cudaSuccess};
    if (!key || !value || !key_strides || !value_strides) return api_error("kv4_append: null pointer");
    if (!aligned(2, {key, value})) return api_error("kv4_append: key and value must be 2-byte aligned");
    return kv4_append_launch(v, cache->head_dim, key, value, dtype == FELIX_BF16, rows, key_strides,
                             value_strides, counts, static_cast<cudaStream_t>(stream));
  });
}

int felix_kv4_read(const felix_kv4_cache* cache, uint32_t rows, const int32_t* counts, void* key,
                   void* value, void* stream) {
  return guarded([&]() -> FelixCode {
    felix_kv4::CacheView v;
    const FelixCode rc = view_of(cache, &v);
    if (rc.type != FELIX_SUCCESS) return rc;
    if (rows > 0x7fffffffu) return api_error("kv4_read: at most 2^31-1 rows");
    if (rows == 0 || v.slots == 0) return FelixCode{FELIX_SUCCESS, cudaSuccess};
    if (!key || !value) return api_error("kv4_read: null pointer");
    if ((reinterpret_cast<uintptr_t>(key) | reinterpret_cast<uintptr_t>(value)) & 15)
      return api_error("kv4_read: outputs must be 16-byte aligned");
    return kv4_read_launch(v, cache->head_dim, rows, counts, static_cast<__half*>(key),
                           static_cast<__half*>(value), static_cast<cudaStream_t>(stream));
  });
}

int felix_kv4_attention(const felix_kv4_cache* cache, const void* q, int dtype, uint32_t heads,
                        uint32_t rows, const int64_t* q_strides, const int32_t* counts,
                        float scale, void* out, float* lse, void* workspace,
                        size_t workspace_bytes, void* stream) {
  return guarded([&]() -> FelixCode {
    felix_kv4::CacheView v;
    const FelixCode rc = view_of(cache, &v);
    if (rc.type != FELIX_SUCCESS) return rc;
    if (dtype != FELIX_F16 && dtype != FELIX_BF16)
      return api_error("kv4_attention: q must be fp16 or bf16");
    if (rows == 0 || v.slots == 0) return FelixCode{FELIX_SUCCESS, cudaSuccess};
    if (!q || !q_strides || !out) return api_error("kv4_attention: null pointer");
    if (heads == 0 || heads > 65535 || heads % v.kv_heads)
      return api_error("kv4_attention: heads must be a multiple of kv_heads, at most 65535");
    if (rows > 65535) return api_error("kv4_attention: at most 65535 rows");
    if (!aligned(2, {q}) || !aligned(8, {out}))
      return api_error("kv4_attention: q must be 2-byte and out 8-byte aligned");
    if (!aligned(16, {workspace})) return api_error(kWorkspaceAlignment);
    return kv4_attention_launch(v, cache->head_dim, q, dtype == FELIX_BF16, heads, rows, q_strides,
                                counts, scale, out, lse, workspace, workspace_bytes,
                                static_cast<cudaStream_t>(stream));
  });
}

int felix_kv4_attention_workspace_size(uint32_t head_dim, size_t* bytes) {
  if (head_dim != 64 && head_dim != 128) return api_error("kv4: head_dim must be 64 or 128").type;
  DeviceInfo* d = current_device_info();
  if (!d) return launch_error(cudaGetLastError(), "no device").type;
  if (bytes) *bytes = kv4_attention_workspace_bytes(head_dim, d->num_sms);
  return FELIX_SUCCESS;
}

int felix_kv4_reserve(const int32_t* table, const int32_t* lens, const int32_t* refs,
                      const int32_t* counts, uint32_t slots, uint32_t width, uint32_t num_pages,
                      uint32_t page_size, int32_t* table_out, int32_t* lens_out,
                      int32_t* refs_out, int32_t* status, void* stream) {
  return guarded([&]() -> FelixCode {
    const int shift = page_shift_of(page_size);
    if (shift < 0) return api_error("kv4: page_size must be a power of two, 16..4096");
    if (!status || ((!lens || !counts || !lens_out) && slots)) return api_error("kv4_reserve: null array");
    return pages_op({Kv4PagesOp::kReserve, table, lens, refs, table_out, lens_out, refs_out, status,
                     counts, nullptr, slots, width, num_pages, uint32_t(shift), 0, nullptr, 0},
                    page_size, stream);
  });
}

int felix_kv4_fork(void* pages, size_t page_bytes, const int32_t* table, const int32_t* lens,
                   const int32_t* refs, const int32_t* parents, const int32_t* children,
                   uint32_t n, uint32_t slots, uint32_t width, uint32_t num_pages,
                   uint32_t page_size, int32_t* table_out, int32_t* lens_out, int32_t* refs_out,
                   int32_t* status, void* stream) {
  return guarded([&]() -> FelixCode {
    const int shift = page_shift_of(page_size);
    if (shift < 0) return api_error("kv4: page_size must be a power of two, 16..4096");
    if (!pages || !status || ((!lens || !lens_out) && slots) || ((!parents || !children) && n))
      return api_error("kv4_fork: null array");
    return pages_op({Kv4PagesOp::kFork, table, lens, refs, table_out, lens_out, refs_out, status,
                     parents, children, slots, width, num_pages, uint32_t(shift), n, pages,
                     page_bytes},
                    page_size, stream);
  });
}

int felix_kv4_free(const int32_t* table, const int32_t* lens, const int32_t* refs,
                   const int32_t* list, uint32_t n, uint32_t slots, uint32_t width,
                   uint32_t num_pages, uint32_t page_size, int32_t* table_out, int32_t* lens_out,
                   int32_t* refs_out, void* stream) {
  return guarded([&]() -> FelixCode {
    const int shift = page_shift_of(page_size);
    if (shift < 0) return api_error("kv4: page_size must be a power of two, 16..4096");
    if (((!lens || !lens_out) && slots) || (!list && n)) return api_error("kv4_free: null array");
    return pages_op({Kv4PagesOp::kFree, table, lens, refs, table_out, lens_out, refs_out, nullptr,
                     list, nullptr, slots, width, num_pages, uint32_t(shift), n, nullptr, 0},
                    page_size, stream);
  });
}

int felix_kv4_compact(void* pages, size_t page_bytes, const int32_t* table, const int32_t* refs,
                      uint32_t slots, uint32_t width, uint32_t num_pages, int32_t* table_out,
                      int32_t* refs_out, void* stream) {
  return guarded([&]() -> FelixCode {
    if (!pages) return api_error("kv4_compact: null array");
    return pages_op({Kv4PagesOp::kCompact, table, nullptr, refs, table_out, nullptr, refs_out,
                     nullptr, nullptr, nullptr, slots, width, num_pages, 4, 0, pages, page_bytes},
                    16, stream);
  });
}

int felix_kv4_copy_pages(const void* from, uint64_t from_pages, void* to, uint64_t to_pages,
                         size_t page_bytes, const int32_t* src, const int32_t* dst, uint32_t n,
                         void* stream) {
  return guarded([&]() -> FelixCode {
    if (n == 0) return FelixCode{FELIX_SUCCESS, cudaSuccess};
    if (!from || !to || !src || !dst) return api_error("kv4_copy_pages: null pointer");
    if (((reinterpret_cast<uintptr_t>(from) | reinterpret_cast<uintptr_t>(to)) & 15) ||
        page_bytes == 0 || page_bytes % 16)
      return api_error("kv4_copy_pages: pools must be 16-byte aligned, pages a multiple of 16 bytes");
    return kv4_copy_launch(from, from_pages, to, to_pages, page_bytes, src, dst, n,
                           static_cast<cudaStream_t>(stream));
  });
}

int felix_sample(const void* logits, int dtype, uint32_t rows, uint32_t vocab, int64_t stride,
                 const float* uniform, const float* temperature, const int32_t* top_k,
                 const float* top_p, const float* min_p, int32_t* tokens, float* logprobs,
                 void* stream) {
  return guarded([&]() -> FelixCode {
    if (dtype != FELIX_F16 && dtype != FELIX_BF16 && dtype != FELIX_F32)
      return api_error("sample: logits must be fp16, bf16 or fp32");
    if (rows == 0) return FelixCode{FELIX_SUCCESS, cudaSuccess};
    if (!logits || !uniform || !tokens || !logprobs) return api_error("sample: null pointer");
    if (vocab == 0 || vocab > 524288u) return api_error("sample: vocab must be 1..524288");
    if (rows > (1u << 27)) return api_error("sample: at most 2^27 rows");
    if (stride < 0) return api_error("sample: stride must not be negative");
    if (!aligned(dtype == FELIX_F32 ? 4 : 2, {logits}))
      return api_error("sample: logits must be aligned to their type");
    return sample_launch({logits, dtype, rows, vocab, stride, uniform, temperature, top_k, top_p,
                          min_p, tokens, logprobs},
                         static_cast<cudaStream_t>(stream));
  });
}

int felix_watchdog_status(unsigned* code, int clear) {
  DeviceInfo* d = current_device_info();
  if (!d) return launch_error(cudaGetLastError(), "no device").type;
  cudaError_t e = cudaDeviceSynchronize();
  if (e != cudaSuccess) return launch_error(e, "watchdog_status: device sync").type;
  unsigned v = 0;
  e = cudaMemcpy(&v, d->status_word, sizeof(v), cudaMemcpyDeviceToHost);
  if (e != cudaSuccess) return launch_error(e, "watchdog_status: read").type;
  if (clear) {
    unsigned z = 0;
    e = cudaMemcpy(d->status_word, &z, sizeof(z), cudaMemcpyHostToDevice);
    if (e != cudaSuccess) return launch_error(e, "watchdog_status: clear").type;
  }
  if (code) *code = v;
  if (v != 0) {
    t_last_cuda = 0;
    std::snprintf(t_last_msg, sizeof(t_last_msg),
                  "device watchdog: a bounded wait gave up (site %u)", v);
    return FELIX_KERNEL_RUNTIME_ERROR;
  }
  return finish(FelixCode{FELIX_SUCCESS, cudaSuccess});
}

int felix_watchdog_probe(uint32_t limit_us, void* stream) {
  return finish(watchdog_probe_launch(limit_us, static_cast<cudaStream_t>(stream)));
}

}  // extern "C"
