// C++ check of the feed-forward operators in libfelix_b200.so (felix/felix.hpp): refusals
// without a device; with the argument "gpu" a linear layer and a gated block, forward and
// backward, against sums in double on the host. Exit code 0 = pass.
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <felix/felix.hpp>

#include <cmath>
#include <cstdint>
#include <cstdio>
#include <vector>

static int failures = 0;
#define CHECK(cond)                                        \
  do {                                                     \
    if (!(cond)) {                                         \
      std::printf("FAILED line %d: %s\n", __LINE__, #cond); \
      ++failures;                                          \
    }                                                      \
  } while (0)

// Rows x cols of small multiples of 1/8: products and short sums of them are exact in fp16.
struct Host {
  uint32_t rows, cols;
  std::vector<double> v;
  Host(uint32_t r, uint32_t c, int seed) : rows(r), cols(c), v(size_t(r) * c) {
    uint32_t s = uint32_t(seed) * 2654435761u + 12345u;
    for (double& x : v) {
      s = s * 1664525u + 1013904223u;
      x = (int(s >> 24) % 5 - 2) * 0.125;
    }
  }
  double at(uint32_t r, uint32_t c) const { return v[size_t(r) * cols + c]; }
};
struct Device {
  half* p = nullptr;
  uint32_t rows, cols;
  Device(uint32_t r, uint32_t c) : rows(r), cols(c) {
    cudaMalloc(&p, size_t(r) * c * sizeof(half));
    cudaMemset(p, 0xff, size_t(r) * c * sizeof(half));
  }
  explicit Device(const Host& h) : Device(h.rows, h.cols) {
    std::vector<half> t(h.v.size());
    for (size_t i = 0; i < t.size(); ++i) t[i] = __float2half(float(h.v[i]));
    cudaMemcpy(p, t.data(), t.size() * sizeof(half), cudaMemcpyHostToDevice);
  }
  ~Device() { cudaFree(p); }
  felix::Matrix m() const { return {p, int64_t(cols)}; }
  double at(uint32_t r, uint32_t c) const {
    half h;
    cudaMemcpy(&h, p + size_t(r) * cols + c, sizeof(half), cudaMemcpyDeviceToHost);
    return __half2float(h);
  }
};

static void without_device() {
  felix::LinearArgs a;
  auto s = felix::linear_launch(a, nullptr);
  CHECK(!s.ok() && s.type == felix::FelixStatus::Type::API_ERROR);
  CHECK(s.str().find("features") != std::string::npos);
  a.tokens = a.in_features = a.out_features = 4;
  CHECK(felix::linear_launch(a, nullptr).str().find("null") != std::string::npos);
  a.type = felix::ElementType::F32;
  CHECK(!felix::linear_bwd_launch(a, nullptr).ok());
  felix::GatedArgs g;
  CHECK(!felix::gated_linear_launch(g, nullptr).ok() && !felix::gated_ffn_launch(g, nullptr).ok());
  CHECK(!felix::gated_linear_bwd_launch(g, nullptr).ok() && !felix::gated_ffn_bwd_launch(g, nullptr).ok());
  size_t n = 0;
  CHECK(!felix::linear_workspace_size(a, true, &n).ok() && !felix::gated_workspace_size(g, true, false, &n).ok());
}

static double relu(double v) { return v > 0 ? v : 0; }

static void with_device(uint32_t T) {
  const uint32_t K = 48, N = 72;
  const Host x(T, K, 1), w(N, K, 2), b(1, N, 3), r(T, N, 4), dy(T, N, 5);
  const Device dx_(x), dw_(w), db_(b), dr(r), ddy(dy), y(T, N), pre(T, N), gx(T, K), gw(N, K), gb(1, N);
  felix::LinearArgs a;
  a.tokens = T;
  a.in_features = K;
  a.out_features = N;
  a.activation = felix::Activation::Relu;
  a.x = dx_.m();
  a.weight = dw_.m();
  a.bias = db_.p;
  a.residual = dr.m();
  a.out = y.m();
  a.pre = pre.m();
  CHECK(felix::linear_launch(a, nullptr).ok());
  a.grad = ddy.m();
  a.dx = gx.m();
  a.dweight = gw.m();
  a.dbias = gb.p;
  size_t need = 0;
  CHECK(felix::linear_workspace_size(a, true, &need).ok());
  void* ws = nullptr;
  if (need) cudaMalloc(&ws, need);
  CHECK(felix::linear_bwd_launch(a, nullptr, ws, need).ok());
  CHECK(cudaDeviceSynchronize() == cudaSuccess);
  cudaFree(ws);
  auto z = [&](uint32_t t, uint32_t n) {
    double s = b.at(0, n);
    for (uint32_t k = 0; k < K; ++k) s += x.at(t, k) * w.at(n, k);
    return s;
  };
  auto dz = [&](uint32_t t, uint32_t n) { return z(t, n) > 0 ? dy.at(t, n) : 0.0; };
  for (uint32_t t : {0u, T / 2, T - 1})
    for (uint32_t n : {0u, 31u, N - 1}) {
      CHECK(pre.at(t, n) == z(t, n));
      CHECK(y.at(t, n) == relu(z(t, n)) + r.at(t, n));
    }
  for (uint32_t n : {0u, N - 1}) {
    double s = 0;
    for (uint32_t t = 0; t < T; ++t) s += dz(t, n);
    CHECK(std::fabs(gb.at(0, n) - s) <= std::fabs(s) / 2048);
    for (uint32_t k : {0u, K - 1}) {
      s = 0;
      for (uint32_t t = 0; t < T; ++t) s += dz(t, n) * x.at(t, k);
      CHECK(std::fabs(gw.at(n, k) - s) <= std::fabs(s) / 2048);
    }
  }
  for (uint32_t k : {0u, K - 1}) {
    double s = 0;
    for (uint32_t n = 0; n < N; ++n) s += dz(T - 1, n) * w.at(n, k);
    CHECK(gx.at(T - 1, k) == s);
  }

  // a gated block without an activation: (x Wg^T) (x Wu^T) Wd^T
  const Host wu(N, K, 6), wd(K, N, 7);
  const Device du(wu), dd(wd), h(T, N), gate(T, N), up(T, N), out(T, K);
  felix::GatedArgs g;
  g.tokens = T;
  g.features = K;
  g.hidden = N;
  g.activation = felix::Activation::None;
  g.x = dx_.m();
  g.w_gate = dw_.m();
  g.w_up = du.m();
  g.gate = gate.m();
  g.up = up.m();
  g.out = h.m();
  CHECK(felix::gated_linear_launch(g, nullptr).ok());
  g.w_down = dd.m();
  g.out = out.m();
  CHECK(felix::gated_ffn_launch(g, nullptr).ok());
  const Device hx(T, K), hg(N, K), hu(N, K), hd(K, N);
  g.grad = dx_.m();
  g.dx = hx.m();
  g.dw_gate = hg.m();
  g.dw_up = hu.m();
  g.dw_down = hd.m();
  CHECK(felix::gated_ffn_bwd_launch(g, nullptr).ok());
  CHECK(cudaDeviceSynchronize() == cudaSuccess);
  auto gv = [&](uint32_t t, uint32_t n) { return z(t, n) - b.at(0, n); };
  auto uv = [&](uint32_t t, uint32_t n) {
    double s = 0;
    for (uint32_t k = 0; k < K; ++k) s += x.at(t, k) * wu.at(n, k);
    return s;
  };
  for (uint32_t t : {0u, T - 1})
    for (uint32_t n : {0u, N - 1}) {
      CHECK(gate.at(t, n) == gv(t, n) && up.at(t, n) == uv(t, n));
      CHECK(std::fabs(h.at(t, n) - gv(t, n) * uv(t, n)) <= std::fabs(gv(t, n) * uv(t, n)) / 2048);
    }
  double s = 0, magnitude = 0;
  for (uint32_t n = 0; n < N; ++n) {
    s += gv(T - 1, n) * uv(T - 1, n) * wd.at(3, n);
    magnitude += std::fabs(gv(T - 1, n) * uv(T - 1, n) * wd.at(3, n));
  }
  CHECK(std::fabs(out.at(T - 1, 3) - s) <= (magnitude + std::fabs(s)) / 2048);
  s = magnitude = 0;
  for (uint32_t t = 0; t < T; ++t) {
    s += x.at(t, 3) * gv(t, 5) * uv(t, 5);
    magnitude += std::fabs(x.at(t, 3) * gv(t, 5) * uv(t, 5));
  }
  CHECK(std::fabs(hd.at(3, 5) - s) <= (magnitude + std::fabs(s)) / 2048);
  CHECK(felix::check_watchdog().ok());
}

int main(int argc, char**) {
  without_device();
  if (argc > 1)
    for (uint32_t T : {1u, 20u, 300u}) with_device(T);
  std::printf(failures ? "%d checks failed\n" : "all checks passed\n", failures);
  return failures != 0;
}
