// The plan of an attention call over the 4-bit cache.  argv: bf16 head_dim kv_heads group sequences
// rows max_rows max_length window.  Prints the splits, whether prompts and few rows go their own ways, the
// sums that a thread of the join adds and the pages of a split.
#include <stdio.h>
#include <stdlib.h>

#include "recorded_launches.h"

#include "../oct_amd/csrc/attention_kv4.hip"

hipError_t recorded_launch(const std::string&, dim3, dim3, void**) { return hipErrorInvalidDeviceFunction; }

int main(int argc, char** argv) {
  if (argc < 10) return 2;
  uint32_t v[9];
  for (int i = 0; i < 9; ++i) v[i] = (uint32_t)strtoul(argv[i + 1], nullptr, 10);
  prom::Kv4AttentionArgs a{};
  a.c.kv_heads = (int)v[2];
  a.group = (int)v[3];
  a.q_heads = a.c.kv_heads * a.group;
  a.c.sequences = (int)v[4];
  a.rows = v[5];
  a.max_rows = v[6];
  a.max_length = v[7];
  a.window = v[8];
  const prom::Plan p = prom::plan(a, (int)v[1], v[0] != 0);
  const int parts = v[1] == 64 ? prom::kJoinParts<64> : v[1] == 128 ? prom::kJoinParts<128> : prom::kJoinParts<256>;
  printf("%d %d %d %d %d\n", p.splits, p.prompts ? 1 : 0, p.few ? 1 : 0,
         p.splits <= parts ? 1 : prom::kMaxSplits / parts, 1 << p.shift);
}
