// The 4-bit paged key/value cache: layout and quantisation.
//
// Pool: [pages, Hk, page / 16, micro], one contiguous micro block per 16
// tokens of one head, so that a reader fetches keys, values and parameters of
// those tokens with one bulk copy:
//
//   16 key rows    D / 2 bytes each
//   16 key (s, lo)   D / g pairs of float16 each
//   16 value rows
//   16 value (s, lo)
//
// A row is D / 8 words of 32 bits, eight dimensions each (dimension i of a
// word in bits 4i .. 4i+3).  Value words are in order.  Key words are stored
// transposed, word (c, j) = dimensions 32 j + 8 c .. + 7 at c * (D / 32) + j:
// a lane that loads quarter c then holds, in its j-th word, dimensions of the
// j-th 32, the order in which an MMA's lanes take one group after another.
//
// A group of g dimensions holds n = clamp(rint((x - lo) / s), 0, 15) for
// s = f16((max - min) / 15) and lo = f16(min), and stands for lo + n s.
// Inputs are clamped to +-65408 first, the largest magnitude at which
// lo + 15 s stays finite in float16 whatever way s was rounded; a NaN makes
// its group NaN.
#pragma once

#include "common.cuh"

namespace b2k {

constexpr float kKv4Limit = 65408.0f;

// n / d for 0 <= n < 2^31 by a multiplication (d is known on the host):
// with s = ceil(log2 d) and m = floor(2^32 (2^s - d) / d) + 1,
// floor(n / d) = (hi32(m n) + n) >> s.
struct FastDiv {
  uint32_t d, m, s;
  __device__ __forceinline__ int div(int n) const {
    return (int)((__umulhi((uint32_t)n, m) + (uint32_t)n) >> s);
  }
};
inline FastDiv fast_div(int64_t d) {
  FastDiv f;
  f.d = (uint32_t)d;
  f.s = 0;
  while ((1ll << f.s) < d) ++f.s;
  f.m = (uint32_t)(((1ull << 32) * ((1ull << f.s) - (uint64_t)d)) / (uint64_t)d + 1);
  return f;
}

struct Kv4 {
  unsigned char* data;
  int64_t pages;
  int Hk, P, D, g;

  __host__ __device__ int micro_bytes() const { return 16 * (D + 8 * (D / g)); }
  __host__ __device__ int row_bytes() const { return D / 2; }
  __host__ __device__ int par_bytes() const { return 4 * (D / g); }
  __host__ __device__ int64_t slots() const { return pages * P; }
  // micro block of `token` (0 .. P-1) of a page, for one head
  __device__ __forceinline__ unsigned char* micro(int64_t page, int head, int token) const {
    return data + ((page * Hk + head) * (P >> 4) + (token >> 4)) * (int64_t)micro_bytes();
  }
};

// index of the stored word that holds dimensions 8 t .. 8 t + 7
__device__ __forceinline__ int kv4_key_word(int t, int D) { return (t & 3) * (D >> 5) + (t >> 2); }

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

}  // namespace b2k
