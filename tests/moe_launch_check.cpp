// The launches of the mixture layer, recorded instead of run.
// argv: bf16 failing hidden inner group tokens experts top_k, the last three 0: every count of a sweep.  Fails (status 1)
// where a launch has no workgroups, more than a grid takes or 2^32 threads; `failing` >= 0: where that launch of a call
// fails and the call queues another behind it or does not return its error.
#include <stdio.h>
#include <stdlib.h>

#include "../oct_amd/csrc/reactor_internal.h"

#define hipGetLastError no_last_error  // its own, below
#include "recorded_launches.h"
#undef hipGetLastError

#include "../oct_amd/csrc/moe_w4.hip"

namespace {
int g_launches = 0, g_failing = -1;
bool g_wrong = false;
hipError_t g_error = hipSuccess;
}  // namespace

extern "C" hipError_t hipGetLastError(void) {
  const hipError_t e = g_error;
  g_error = hipSuccess;
  return e;
}

hipError_t recorded_launch(const std::string& kernel, dim3 grid, dim3 block, void**) {
  if (grid.x == 0 || grid.y == 0 || grid.z == 0 || grid.y > 65535u || grid.z > 65535u ||
      (uint64_t)grid.x * block.x >= 1ull << 32) {
    printf("%s: %u %u %u\n", kernel.c_str(), grid.x, grid.y, grid.z);
    g_wrong = true;
  }
  if (g_launches++ == g_failing) g_error = hipErrorInvalidConfiguration;
  return g_error;
}

int main(int argc, char** argv) {
  if (argc < 9) return 2;
  long v[8];
  for (int i = 0; i < 8; ++i) v[i] = strtol(argv[i + 1], nullptr, 10);
  const bool bf16 = v[0] != 0;
  const uint32_t hidden = (uint32_t)v[2], inner = (uint32_t)v[3], group = (uint32_t)v[4];
  void* const somewhere = reinterpret_cast<void*>(1ull << 40);
  const auto call = [&](int tokens, int experts, int top_k) {
    if (top_k > experts || tokens * top_k > prom::kMoeMaxPairs) return;
    prom::W4MoeArgs a{};
    a.gate = a.up = prom::w4_view(somewhere, inner, hidden, group, (uint32_t)experts);
    a.down = prom::w4_view(somewhere, hidden, inner, group, (uint32_t)experts);
    a.x = a.out = somewhere;
    a.x_stride = a.out_stride = hidden;
    a.tokens = tokens;
    a.experts = experts;
    a.top_k = top_k;
    prom::moe_w4_workspace(a, somewhere);
    for (g_failing = (int)v[1] < 0 ? -1 : 0; g_failing < 4; ++g_failing) {
      g_launches = 0;
      const hipError_t e = prom::launch_moe_w4(a, bf16, nullptr);
      if (g_failing < 0) {
        if (e != hipSuccess || g_launches != (a.joins ? 3 : 4)) g_wrong = true;
      } else if (g_launches > g_failing && (e != hipErrorInvalidConfiguration || g_launches != g_failing + 1)) {
        g_wrong = true;
      }
      if (g_wrong) {
        printf("%d tokens, %d of %d experts, failing %d: %d launches, error %d\n", tokens, top_k, experts, g_failing,
               g_launches, (int)e);
        exit(1);
      }
      if (g_failing < 0) break;
    }
  };
  if (v[5] != 0) {
    call((int)v[5], (int)v[6], (int)v[7]);
    return 0;
  }
  for (int experts : {1, 2, 3, 8, 63, 64, 65, 128, 131, 132, 256, 257, 300, 513, 1023, 1024})
    for (int top_k : {1, 2, 3, 5, 8, 64})
      for (int tokens = 1; tokens <= 520; ++tokens) call(tokens, experts, top_k);
  for (int tokens : {1000, 1024, 8192, 65535, 65536}) call(tokens, 1024, 1), call(tokens, 5, 1), call(tokens, 64, 8);
  return 0;
}
