// Expert layer with MXFP4 weights: parameter blocks and host entries (internal).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "exf_kernels.h"

namespace exf {

struct MxRoutes {               // moe_align's result
  const int32_t* num_post_pad;
  const int32_t* expert_ids;    // [blocks]
  const int32_t* sorted_ids;    // [capacity]
};

struct MxLayerParams {
  MxRoutes routes;
  int experts;
  int numel;                    // routes = tokens * top_k
  int hidden;
  int inter;
  int m_blocks;                 // route blocks of the capacity
  int* status;                  // set to 1 if a pipeline wait timed out (may be null)
  const uint8_t* w13;           // weights and their scales (see MxArgs)
  const uint8_t* s13;
  const uint8_t* w2;
  const uint8_t* s2;
  const uint8_t* xs;            // scales of the split token rows
  uint8_t* hq;                  // GEMM-1 output in the same form
  uint8_t* hs;
  const float* route_w;
  float* out;                   // GEMM-2 output [numel][hidden]; prefill: 16-bit multiples of
  uint8_t* out_scale;           // the powers in [numel][hidden / 32]
  int32_t* sync;                // [0] next tile; [1 + b] GEMM-1 epilogue warps done with block b
};

struct MxArgs {
  const void* x;                // bf16 [tokens][hidden]
  const float* topk_w;          // [tokens][top_k]
  const int32_t* topk_ids;
  int64_t tokens;
  int top_k;
  const uint8_t* w13;           // codes [experts][2 * inter][hidden / 2]
  const uint8_t* s13;           // scales [experts][2 * inter / 128][hidden / 128][512]
  const uint8_t* w2;            // codes [experts][hidden][inter / 2]
  const uint8_t* s2;            // scales [experts][hidden / 128][inter / 128][512]
  int experts;
  int hidden;
  int inter;
  void* y;                      // bf16 [tokens][hidden]
  int* status;
};

struct MxWorkspace {
  int block;                    // routes of a block (with few routes there is only out: h fp32)
  int64_t capacity;
  int32_t* sorted_ids;
  int32_t* expert_ids;
  int32_t* num_post_pad;
  void* align_ws;
  int32_t* slots;               // slot of each route (more routes than one align launch takes)
  uint8_t* xq;                  // two-term token rows [blocks][2 * block][hidden] (exf_mx.cuh)
  uint8_t* xs;                  // their scales [blocks][tables][hidden / 128][512]
  uint8_t* hq;
  uint8_t* hs;
  float* out;
  uint8_t* out_scale;
  int32_t* sync;
  int sync_ints;
  int64_t bytes;
};

// Carves the workspace at `base` (null: sizes only).
MxWorkspace mx_workspace(int64_t tokens, int top_k, int experts, int hidden, int inter, void* base);
// Layers of few routes (mx_few): h [tokens * top_k][inter] is scratch.
bool mx_few(int64_t routes, int hidden, int inter);
cudaError_t launch_mx_few(const MxArgs& a, float* h, cudaStream_t s);
cudaError_t launch_mx_experts(const MxArgs& a, const MxWorkspace& w, cudaStream_t s);

}  // namespace exf
