// The mixture layer's arguments and workspace (moe_w4.hip; filled in by the entry points).
#pragma once

#include "w4_tiles.h"

namespace prom {

constexpr int kMoeMaxExperts = 1024, kMoeMaxTopK = 64, kMoeMaxPairs = 65536;
constexpr int kMoeFewTokens = 64;  // a token a lane

struct MoeExpert {
  int expert, start, count;  // its pairs: pairs[start] ..
  int unused;                // sixteen bytes: one load
};

struct W4MoeArgs {
  W4View gate, up, down;  // [inner, hidden] twice, [hidden, inner]; a matrix an expert
  const float* router;    // [experts, hidden]
  const void* x;
  void* out;
  int32_t* out_chosen;  // may be null
  float* out_weights;   // may be null
  uint32_t x_stride, out_stride, activation;
  int tokens, experts, top_k;
  bool renormalise;
  // workspace
  double* logits;   // [tokens][experts]
  int32_t* chosen;  // [pairs], pairs = tokens * top_k
  float* weights;   // [pairs]
  uint8_t* places;  // [tokens][experts]: 1 + an expert's place among the token's, 0 where it is none (few tokens)
  int32_t* pairs;   // by expert (more tokens)
  MoeExpert* reached;  // min(experts, pairs), those behind the last with count 0 (more tokens)
  uint16_t* hidden;    // terms of [pairs][hidden_stride], hidden_plane elements apart
  size_t hidden_plane;
  uint32_t hidden_stride;  // whole tiles of 128
  float* part;             // [column group][pairs][parts][columns of a group]
  int out_tiles, split;    // of the second product
  int parts;               // of K that leave sums of their own: split or 1
  int blocks;              // of sixteen pairs of an expert, taken at once
  bool joins;              // the second product's last workgroups join the sums
};

// Bytes of the workspace; sets the pointers into `base`.
size_t moe_w4_workspace(W4MoeArgs& a, void* base);
hipError_t launch_moe_w4(const W4MoeArgs& a, bool bf16, hipStream_t stream);

}  // namespace prom
