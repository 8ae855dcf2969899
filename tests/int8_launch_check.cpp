// The launches of the int8 product, recorded instead of run.  argv: m n k.
// Fails (status 1) where the product of contiguous, aligned operands is refused, a launch has 2^32
// threads or more, which HIP refuses, or the launches do not take the columns one after the other,
// each once.
#include <stdio.h>
#include <stdlib.h>

#include "recorded_launches.h"

#include "../oct_amd/csrc/gemm_int8.hip"

namespace {
int8_t* const kW = reinterpret_cast<int8_t*>(1ull << 40);
float* const kScale = reinterpret_cast<float*>(1ull << 42);
float* const kOut = reinterpret_cast<float*>(1ull << 43);
uint64_t g_next = 0, g_n = 0, g_k = 0;
bool g_wrong = false;
}  // namespace

hipError_t recorded_launch(const std::string& kernel, dim3 grid, dim3 block, void** args) {
  const uint64_t threads = (uint64_t)grid.x * block.x;
  printf("%s: %llu threads of %u\n", kernel.c_str(), (unsigned long long)threads, block.x);
  if (threads >= 1ull << 32 || grid.y > 65535u) g_wrong = true;
  const bool few = kernel.find("gemm_int8_rows_kernel") != std::string::npos;
  if (!few && kernel.find("gemm_int8_tile_kernel") == std::string::npos) return hipSuccess;
  const prom::Int8Args& g = *static_cast<prom::Int8Args*>(args[0]);
  const uint64_t columns = (uint64_t)g.n;
  if (few && (g.w != kW + g_next * g_k || (uint64_t)grid.x * 16 < columns)) g_wrong = true;
  if (g.w_scale != kScale + g_next || g.c != kOut + g_next || (uint64_t)g.ldc != g_n) g_wrong = true;
  g_next += columns;
  return hipSuccess;
}

int main(int argc, char** argv) {
  if (argc < 4) return 2;
  const uint32_t m = (uint32_t)strtoul(argv[1], nullptr, 10), n = (uint32_t)strtoul(argv[2], nullptr, 10),
                 k = (uint32_t)strtoul(argv[3], nullptr, 10);
  g_n = n;
  g_k = k;
  const hipError_t e = prom::launch_gemm_int8(kW, kW, kScale, kScale, kOut, false, m, n, k, nullptr);
  return e != hipSuccess || g_wrong || g_next != n;
}
