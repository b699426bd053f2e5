// Refused calls of the C ABI while the host has no memory left (operator new throws): each
// returns its error, with a message, and none lets an exception out. No device is touched.
// Exit code 0 = pass.
#include <felix_c.h>

#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <new>

static bool none_left = false;
void* operator new(std::size_t n) {
  if (void* p = none_left ? nullptr : std::malloc(n ? n : 1)) return p;
  throw std::bad_alloc();
}
void operator delete(void* p) noexcept { std::free(p); }
void operator delete(void* p, std::size_t) noexcept { std::free(p); }

static int failures = 0;
static void expect(const char* what, int rc, const char* text) {
  none_left = false;
  if (rc != FELIX_API_ERROR || !std::strstr(felix_last_error_message(), text)) {
    std::printf("FAILED %s: %d \"%s\"\n", what, rc, felix_last_error_message());
    ++failures;
  }
}
#define REFUSED(call, text)       \
  do {                            \
    none_left = true;             \
    const int rc_ = call;         \
    expect(#call, rc_, text);     \
  } while (0)

int main() {
  felix_linear_args l{};
  felix_gated_args g{};
  l.dtype = g.dtype = 9;
  size_t n = 0;
  REFUSED(felix_linear(nullptr, nullptr, 0, nullptr), "null pointer");
  REFUSED(felix_linear(&l, nullptr, 0, nullptr), "must be fp16 or bf16");
  REFUSED(felix_linear_bwd(&l, nullptr, 0, nullptr), "must be fp16 or bf16");
  REFUSED(felix_gated_linear(&g, nullptr, 0, nullptr), "must be fp16 or bf16");
  REFUSED(felix_gated_linear_bwd(&g, nullptr, 0, nullptr), "must be fp16 or bf16");
  REFUSED(felix_gated_ffn(&g, nullptr, 0, nullptr), "must be fp16 or bf16");
  REFUSED(felix_gated_ffn_bwd(&g, nullptr, 0, nullptr), "must be fp16 or bf16");
  REFUSED(felix_linear_workspace_size(&l, 0, &n), "must be fp16 or bf16");
  REFUSED(felix_gated_workspace_size(&g, 1, 1, &n), "must be fp16 or bf16");
  REFUSED(felix_hgemm(8, 8, 8, 1.f, nullptr, nullptr, 0.f, nullptr, 9, nullptr),
          "b_layout must be FELIX_B_KN or FELIX_B_NK");
  REFUSED(felix_sample(nullptr, 9, 1, 1, 1, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr,
                       nullptr, nullptr),
          "sample");
  if (!failures) std::puts("all checks passed");
  return failures != 0;
}
