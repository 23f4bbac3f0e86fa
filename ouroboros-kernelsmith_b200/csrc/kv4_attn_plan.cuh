// What the 4-bit cache attention's entry point and its instances share: the
// arguments, and how a call is cut for the GPU.
#pragma once

#include "kv4.cuh"

namespace b2k {

int kv4_check(const char* what, const void* data, int64_t pages, int64_t Hk, int64_t P, int64_t D,
              int64_t g);

constexpr int kAttnWarps = 4;  // of a block

struct Kv4AttnArgs {
  Kv4 c;
  FastDiv dG, dRT, dP, dHk;
  const void* q;
  void* o;
  float* lse;
  const int32_t *table, *lens;
  int64_t B, Sq, H, width;
  int64_t qb, qs, qh;  // strides of q in elements (batch, token, head)
  float scale;
  int causal, bf16, q_aligned;
  int warps;  // of the launch
  int G, RT;  // query heads per cache head; row tiles per (sequence, head)
  float* part;      // [2 * warps][rows][D] outputs, then [2 * warps][rows][2] (m, l)
  int2* spans;      // [segments] first and last warp
};

// rows of a row tile
__host__ __device__ constexpr int attn_rows(int NT) { return 8 * NT; }
// resident blocks per SM: registers (NT D / 4 for the output) and shared memory.
// Three leave 168 registers, which D 128 with groups of 32, D 64 with 16 rows and D
// 256 exceed by 4 to 10 (spilled); two leave 255, which D 256 with 16 rows exceeds
// by 9 to 22.  One block more spilled far more and was slower.
__host__ __device__ constexpr int attn_cps(int D, int NT) { return NT * D >= 256 && NT > 1 ? 2 : 3; }

struct AttnPlan {
  int nt, blocks, warps;
  int64_t rt, segs, part_bytes, bytes;
};

int attn_d64(const Kv4AttnArgs& a, const AttnPlan& p, cudaStream_t st);
int attn_d128(const Kv4AttnArgs& a, const AttnPlan& p, cudaStream_t st);
int attn_d256(const Kv4AttnArgs& a, const AttnPlan& p, cudaStream_t st);

}  // namespace b2k
