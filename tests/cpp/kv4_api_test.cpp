// C++ check of the decode operators in libfelix_b200.so (felix/felix.hpp): page
// sizes and refusals without a device; with the argument "gpu" one token per slot
// is appended, attended to and read back, a slot is forked and freed, pages are
// compacted and a token is sampled. Exit code 0 = pass.
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <felix/felix.hpp>

#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <vector>

static int failures = 0;
#define CHECK(cond)                                        \
  do {                                                     \
    if (!(cond)) {                                         \
      std::printf("FAILED line %d: %s\n", __LINE__, #cond); \
      ++failures;                                          \
    }                                                      \
  } while (0)

template <class T>
T* to_device(const std::vector<T>& v) {
  T* p = nullptr;
  cudaMalloc(&p, v.size() * sizeof(T));
  cudaMemcpy(p, v.data(), v.size() * sizeof(T), cudaMemcpyHostToDevice);
  return p;
}
template <class T>
std::vector<T> to_host(const T* p, size_t n) {
  std::vector<T> v(n);
  cudaMemcpy(v.data(), p, n * sizeof(T), cudaMemcpyDeviceToHost);
  return v;
}

static void without_device() {
  CHECK(felix::kv4_page_bytes(8, 128, 64) == 64u * 8 * 136);
  CHECK(felix::kv4_page_bytes(8, 96, 64) == 0);
  CHECK(felix::kv4_page_bytes(8, 128, 63) == 0);
  felix::Kv4Cache c{};
  const int64_t st[3] = {0, 0, 0};
  const auto s = felix::kv4_attention_launch(c, nullptr, felix::ElementType::F16, 8, 1, st, nullptr,
                                             0.f, nullptr, nullptr, nullptr);
  CHECK(!s.ok() && s.type == felix::FelixStatus::Type::API_ERROR);
  CHECK(s.str().find("kv4") != std::string::npos);
  CHECK(!felix::sample_launch(nullptr, felix::ElementType::F32, 1, 5, 5, nullptr, nullptr, nullptr,
                              nullptr, nullptr, nullptr, nullptr, nullptr)
             .ok());
}

static void with_device() {
  constexpr uint32_t kSlots = 3, kWidth = 2, kPages = 6, kPage = 16, kD = 64;
  const size_t bytes = felix::kv4_page_bytes(1, kD, kPage);
  unsigned char* pool = nullptr;
  cudaMalloc(&pool, kPages * bytes);
  int32_t* table = to_device(std::vector<int32_t>(kSlots * kWidth, -1));
  int32_t* lens = to_device(std::vector<int32_t>(kSlots, 0));
  int32_t* refs = to_device(std::vector<int32_t>{1, 0, 0, 0, 0, 0});  // page 0 is taken
  int32_t* status = to_device(std::vector<int32_t>(2, -7));
  const felix::Kv4Pages state{table, lens, refs};
  int32_t* counts = to_device(std::vector<int32_t>{1, 1, 0});
  CHECK(felix::kv4_reserve_launch(state, counts, kSlots, kWidth, kPages, kPage, state, status,
                                  nullptr).ok());
  CHECK(to_host(status, 2) == (std::vector<int32_t>{0, 0}));
  CHECK(to_host(table, 6) == (std::vector<int32_t>{1, -1, 2, -1, -1, -1}));

  // one token per slot: attention gives its value back
  std::vector<half> kv(kSlots * kD);
  for (uint32_t i = 0; i < kv.size(); ++i) kv[i] = __float2half(float(i % kD) - 30.f + float(i / kD));
  half* k = to_device(kv);
  const int64_t st[3] = {kD, kD, kD};
  const felix::Kv4Cache cache{pool, kPages, kPage, 1, kD, table, lens, kSlots, kWidth};
  CHECK(felix::kv4_append_launch(cache, k, k, felix::ElementType::F16, 1, st, st, counts, nullptr).ok());
  half *out = to_device(kv), *rk = to_device(kv), *rv = to_device(kv);
  float* lse = to_device(std::vector<float>(kSlots, 0.f));
  CHECK(felix::kv4_attention_launch(cache, k, felix::ElementType::F16, 1, 1, st, counts, 0.01f, out,
                                    lse, nullptr).ok());
  CHECK(felix::kv4_read_launch(cache, 1, counts, rk, rv, nullptr).ok());
  CHECK(cudaDeviceSynchronize() == cudaSuccess);
  const auto o = to_host(out, kv.size()), r = to_host(rv, kv.size());
  for (uint32_t i = 0; i < kv.size(); ++i) {
    const float want = i / kD == 2 ? 0.f : __half2float(r[i]);
    CHECK(std::fabs(__half2float(o[i]) - want) <= 1e-3f * std::fabs(want));
    if (i / kD < 2) CHECK(std::fabs(__half2float(r[i]) - __half2float(kv[i])) <= 63.f / 15 / 2 + 0.02f);
  }
  CHECK(std::isinf(to_host(lse, 3)[2]));

  // slot 2 becomes a copy of slot 0 (its page is not full: copied), slot 0 leaves
  int32_t *zero = to_device(std::vector<int32_t>{0}), *two = to_device(std::vector<int32_t>{2});
  CHECK(felix::kv4_fork_launch(pool, bytes, state, zero, two, 1, kSlots, kWidth, kPages, kPage, state,
                               status, nullptr).ok());
  CHECK(felix::kv4_free_launch(state, zero, 1, kSlots, kWidth, kPages, kPage, state, nullptr).ok());
  CHECK(to_host(refs, 6) == (std::vector<int32_t>{1, 0, 1, 1, 0, 0}));
  CHECK(felix::kv4_compact_launch(pool, bytes, state, kSlots, kWidth, kPages, state, nullptr).ok());
  CHECK(to_host(table, 6) == (std::vector<int32_t>{-1, -1, 2, -1, 1, -1}));
  CHECK(felix::kv4_attention_launch(cache, k, felix::ElementType::F16, 1, 1, st, nullptr, 0.01f, out,
                                    nullptr, nullptr).ok());
  const auto o2 = to_host(out, kv.size());
  CHECK(std::memcmp(&o2[2 * kD], &o[0], kD * sizeof(half)) == 0);
  CHECK(felix::kv4_copy_pages_launch(pool, kPages, pool, kPages, bytes, two, zero, 1, nullptr).ok());

  std::vector<float> logits(100, 0.f);
  logits[42] = 50.f;
  float *x = to_device(logits), *u = to_device(std::vector<float>{0.3f}), *lp = to_device(std::vector<float>{1.f});
  int32_t* token = to_device(std::vector<int32_t>{-5});
  CHECK(felix::sample_launch(x, felix::ElementType::F32, 1, 100, 100, u, nullptr, nullptr, nullptr,
                             nullptr, token, lp, nullptr).ok());
  CHECK(to_host(token, 1)[0] == 42 && to_host(lp, 1)[0] == 0.f);
  CHECK(felix::check_watchdog().ok());
}

int main(int argc, char** argv) {
  without_device();
  if (argc > 1 && std::strcmp(argv[1], "gpu") == 0) with_device();
  if (failures == 0) std::printf("all checks passed\n");
  return failures != 0;
}
