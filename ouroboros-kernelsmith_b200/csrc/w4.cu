// 4-bit weights with group scales: b2k_w4_pack (lay out given integers),
// b2k_w4_quantize (from floating weights) and b2k_w4_matmul.
//
//   W[n, k] = s[n, k / g] (w[n, k] - z[n, k / g]),  w in 0..15, z = 8 without zeros
//   y[m, n] = sum_k x[m, k] W[n, k]                 (x of 8 bits: times its scales)
//
// Layout (kernel's own, made once): tiles of 16 rows x 128 columns, 1 KB
// each, [ceil(N/16), ceil(K/128), 16 rows, 4 quarters, 4 words]: word j of
// quarter c holds columns 32 j + 8 c .. + 7 of the tile (column i of a word in
// bits 4i .. 4i+3).  Scales and zeros: [ceil(N/16), ceil(K/128), 128/g, 16].
// Rows and columns past N and K hold zeros with scale zero.
#include <cuda_fp8.h>

#include "rowio.cuh"
#include "tma.cuh"

namespace b2k {

struct W4 {
  const unsigned char* tiles;
  const void *scales, *zeros;
  int64_t N, K;
  int g;
  __host__ __device__ int64_t ntiles() const { return (N + 15) / 16; }
  __host__ __device__ int64_t ktiles() const { return (K + 127) / 128; }
};

// -------------------------------------------------------------- laying out
// one thread per stored word; `get(n, k)` is the integer of row n, column k
struct W4PackArgs {
  const uint8_t* q;
  int64_t ldq;
  const void *scales, *zeros;  // [N, ceil(K / g)] of T
  int64_t lds;
  unsigned char* tiles;
  void *oscales, *ozeros;
  int64_t N, K;
  int g;
};

__global__ void __launch_bounds__(256) w4_pack_words_kernel(W4PackArgs a) {
  const int64_t kt = (a.K + 127) / 128, nt = (a.N + 15) / 16;
  const int64_t total = nt * kt * 256;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total;
       i += (int64_t)gridDim.x * 256) {
    const int64_t tile = i >> 8;
    const int r = (int)(i >> 4) & 15, c = (int)(i >> 2) & 3, j = (int)i & 3;
    const int64_t n = tile / kt * 16 + r, k = tile % kt * 128 + 32 * j + 8 * c;
    uint32_t w = 0;
    if (n < a.N)
      for (int e = 0; e < 8 && k + e < a.K; ++e)
        w |= (uint32_t)(a.q[n * a.ldq + k + e] & 15u) << (4 * e);
    reinterpret_cast<uint32_t*>(a.tiles)[i] = w;
  }
}

__global__ void __launch_bounds__(256) w4_pack_scales_kernel(W4PackArgs a) {
  const int64_t kt = (a.K + 127) / 128, nt = (a.N + 15) / 16;
  const int gs = 128 / a.g;
  const int64_t total = nt * kt * gs * 16;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total;
       i += (int64_t)gridDim.x * 256) {
    const int64_t tile = i / (16 * gs);
    const int64_t n = tile / kt * 16 + (i & 15);
    const int64_t grp = tile % kt * gs + (i >> 4) % gs;
    const bool in = n < a.N && grp * a.g < a.K;
    static_cast<uint16_t*>(a.oscales)[i] =
        in ? static_cast<const uint16_t*>(a.scales)[n * a.lds + grp] : (uint16_t)0;
    if (a.zeros)
      static_cast<uint16_t*>(a.ozeros)[i] =
          in ? static_cast<const uint16_t*>(a.zeros)[n * a.lds + grp] : (uint16_t)0;
  }
}

// One thread per group of one row: scale (and zero) and integers of floating
// weights.  Without zeros s = max|w| / 7 rounded to S and n = round(w / s) + 8
// within 1..15; with zeros the group's range, widened to hold 0, is divided
// into 15 steps and z is the whole number that stands for 0.
template <typename T, typename S>
__global__ void __launch_bounds__(256) w4_quantize_kernel(const T* w, int64_t ldw, int64_t N,
                                                          int64_t K, int g, unsigned char* tiles,
                                                          S* scales, S* zeros) {
  const int64_t kt = (K + 127) / 128, nt = (N + 15) / 16;
  const int gs = 128 / g;
  const int64_t total = nt * kt * gs * 16;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total;
       i += (int64_t)gridDim.x * 256) {
    const int r = (int)(i & 15), sub = (int)(i >> 4) % gs;
    const int64_t tile = i / (16 * gs);
    const int64_t n = tile / kt * 16 + r, k0 = tile % kt * 128 + sub * g;
    const int64_t cnt = n < N ? min((int64_t)g, K - k0) : 0;
    const T* row = w + n * ldw + k0;
    float lo = 0.0f, hi = 0.0f;
    for (int64_t e = 0; e < cnt; ++e) {
      const float v = ld1(row + e);
      lo = v < lo || v != v ? v : lo;
      hi = v > hi || v != v ? v : hi;
    }
    const float s = to_f<S>(from_f<S>(zeros ? (hi - lo) / 15.0f : fmaxf(hi, -lo) / 7.0f));
    const float z = zeros ? (s > 0.0f ? fminf(fmaxf(rintf(-lo / s), 0.0f), 15.0f) : 0.0f) : 8.0f;
    scales[i] = from_f<S>(cnt > 0 ? s : 0.0f);
    if (zeros) zeros[i] = from_f<S>(cnt > 0 ? z : 0.0f);
    uint32_t* words = reinterpret_cast<uint32_t*>(tiles) + tile * 256 + r * 16;
    for (int t = 0; t < g / 8; ++t) {
      uint32_t bits = 0;
      for (int e = 0; e < 8; ++e) {
        float q = 0.0f;
        if (8 * t + e < cnt) {
          q = s > 0.0f ? rintf(ld1(row + 8 * t + e) / s) + z : z;
          q = fminf(fmaxf(q, zeros ? 0.0f : 1.0f), 15.0f);
        }
        bits |= (uint32_t)q << (4 * e);
      }
      const int word = sub * (g / 8) + t;  // columns 8 word .. + 7 of the tile
      words[(word & 3) * 4 + (word >> 2)] = bits;
    }
  }
}

// -------------------------------------------------------------- the product
struct W4Args {
  W4 w;
  const void* x;
  int64_t ldx;
  const float* xs;  // scales of 8-bit x, [M, K / xgroup] (xgroup 0: one per row)
  int64_t ldxs;
  int xgroup;
  void* y;
  int64_t ldy, M;
  int xtype, ytype, stype;
};

__device__ __forceinline__ float w4_x(const W4Args& a, int64_t m, int64_t k) {
  const int64_t i = m * a.ldx + k;
  float v;
  switch (a.xtype) {
    case B2K_F32: return static_cast<const float*>(a.x)[i];
    case B2K_F16: return to_f(static_cast<const __half*>(a.x)[i]);
    case B2K_BF16: return to_f(static_cast<const __nv_bfloat16*>(a.x)[i]);
    case B2K_I8: v = (float)static_cast<const int8_t*>(a.x)[i]; break;
    default: v = (float)static_cast<const __nv_fp8_e4m3*>(a.x)[i]; break;
  }
  return v * a.xs[m * a.ldxs + (a.xgroup ? k / a.xgroup : 0)];
}

__device__ __forceinline__ float w4_s(const void* p, int type, int64_t i) {
  return type == B2K_F16 ? to_f(static_cast<const __half*>(p)[i])
                         : to_f(static_cast<const __nv_bfloat16*>(p)[i]);
}

// one warp per output
__global__ void __launch_bounds__(128) w4_simple_kernel(W4Args a) {
  griddep_launch_dependents();
  griddep_wait();
  const int lane = threadIdx.x & 31;
  const int64_t id = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (id >= a.M * a.w.N) return;
  const int64_t m = id / a.w.N, n = id % a.w.N;
  const int64_t kt = a.w.ktiles();
  const int gs = 128 / a.w.g;
  float acc = 0.0f;
  for (int64_t k = lane; k < a.w.K; k += 32) {
    const int64_t tile = n / 16 * kt + k / 128;
    const int col = (int)(k & 127), word = col >> 3;
    const uint32_t w = reinterpret_cast<const uint32_t*>(a.w.tiles)[tile * 256 + (n & 15) * 16 +
                                                                   (word & 3) * 4 + (word >> 2)];
    const int64_t si = (tile * gs + col / a.w.g) * 16 + (n & 15);
    const float z = a.w.zeros ? w4_s(a.w.zeros, a.stype, si) : 8.0f;
    const float v = ((float)((w >> (4 * (col & 7))) & 15u) - z) * w4_s(a.w.scales, a.stype, si);
    const float xv = w4_x(a, m, k);
    acc = fmaf(isfinite(xv) ? xv : __int_as_float(0x7fc00000), v, acc);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
  if (lane == 0) {
    const int64_t i = m * a.ldy + n;
    if (a.ytype == B2K_F32) static_cast<float*>(a.y)[i] = acc;
    else if (a.ytype == B2K_F16) static_cast<__half*>(a.y)[i] = from_f<__half>(acc);
    else static_cast<__nv_bfloat16*>(a.y)[i] = from_f<__nv_bfloat16>(acc);
  }
}

static int w4_check(const char* what, int64_t N, int64_t K, int group, int stype) {
  B2K_REQUIRE(N >= 0 && K >= 0, "%s: negative shape N=%lld K=%lld", what, (long long)N, (long long)K);
  B2K_REQUIRE(group == 32 || group == 64 || group == 128, "%s: group %d is not 32, 64 or 128", what,
              group);
  B2K_REQUIRE(stype == B2K_F16 || stype == B2K_BF16, "%s: scales of dtype %d are not 16-bit", what,
              stype);
  B2K_REQUIRE(N <= ((int64_t)1 << 31) && K <= ((int64_t)1 << 31) &&
                  ((N + 15) / 16) * ((K + 127) / 128) <= ((int64_t)1 << 38),
              "%s: shape too large", what);
  return B2K_OK;
}

static unsigned w4_blocks(int64_t items) {
  const int64_t b = (items + 255) / 256;
  return (unsigned)(b < 65536 ? (b < 1 ? 1 : b) : 65536);
}

}  // namespace b2k

using namespace b2k;

extern "C" int b2k_w4_pack(const uint8_t* q, int64_t ldq, const void* scales, const void* zeros,
                           int64_t lds, int64_t N, int64_t K, int group, int stype, void* tiles,
                           void* tile_scales, void* tile_zeros, void* stream) {
  if (int st = w4_check("b2k_w4_pack", N, K, group, stype)) return st;
  if (N == 0 || K == 0) return B2K_OK;
  B2K_REQUIRE(q && scales && tiles && tile_scales && (!zeros == !tile_zeros),
              "b2k_w4_pack: null operand");
  W4PackArgs a = {q, ldq, scales, zeros, lds, static_cast<unsigned char*>(tiles), tile_scales,
                  tile_zeros, N, K, group};
  const int64_t nk = ((N + 15) / 16) * ((K + 127) / 128);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  w4_pack_words_kernel<<<w4_blocks(nk * 256), 256, 0, st>>>(a);
  w4_pack_scales_kernel<<<w4_blocks(nk * (128 / group) * 16), 256, 0, st>>>(a);
  return check_launch("b2k_w4_pack");
}

extern "C" int b2k_w4_quantize(const void* w, int64_t ldw, int64_t N, int64_t K, int dtype,
                               int group, int stype, void* tiles, void* tile_scales,
                               void* tile_zeros, void* stream) {
  if (int st = w4_check("b2k_w4_quantize", N, K, group, stype)) return st;
  if (N == 0 || K == 0) return B2K_OK;
  B2K_REQUIRE(w && tiles && tile_scales, "b2k_w4_quantize: null operand");
  const int64_t items = ((N + 15) / 16) * ((K + 127) / 128) * (128 / group) * 16;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  B2K_DISPATCH_FLOAT(dtype, {
    if (stype == B2K_F16)
      w4_quantize_kernel<T, __half><<<w4_blocks(items), 256, 0, st>>>(
          static_cast<const T*>(w), ldw, N, K, group, static_cast<unsigned char*>(tiles),
          static_cast<__half*>(tile_scales), static_cast<__half*>(tile_zeros));
    else
      w4_quantize_kernel<T, __nv_bfloat16><<<w4_blocks(items), 256, 0, st>>>(
          static_cast<const T*>(w), ldw, N, K, group, static_cast<unsigned char*>(tiles),
          static_cast<__nv_bfloat16*>(tile_scales), static_cast<__nv_bfloat16*>(tile_zeros));
  });
  return check_launch("b2k_w4_quantize");
}

extern "C" int b2k_w4_matmul(const void* x, int64_t ldx, int xtype, const float* xs, int64_t ldxs,
                             int xgroup, const void* tiles, const void* tile_scales,
                             const void* tile_zeros, int stype, int group, int64_t M, int64_t N,
                             int64_t K, void* y, int64_t ldy, int ytype, void* stream) {
  if (int st = w4_check("b2k_w4_matmul", N, K, group, stype)) return st;
  const bool x8 = xtype == B2K_I8 || xtype == B2K_E4M3;
  B2K_REQUIRE(x8 || (xtype >= B2K_F32 && xtype <= B2K_BF16), "b2k_w4_matmul: bad x dtype %d", xtype);
  B2K_REQUIRE(ytype >= B2K_F32 && ytype <= B2K_BF16, "b2k_w4_matmul: bad y dtype %d", ytype);
  B2K_REQUIRE(x8 == (xs != nullptr) || M == 0 || N == 0 || K == 0,
              "b2k_w4_matmul: scales go with x of 8 bits, and only with it");
  B2K_REQUIRE(xgroup == 0 || (x8 && xgroup % group == 0 && 128 % xgroup == 0),
              "b2k_w4_matmul: x's group %d is no multiple of the weight's %d up to 128", xgroup,
              group);
  B2K_REQUIRE(M >= 0 && M <= 0x7fffffffLL, "b2k_w4_matmul: bad number of rows %lld", (long long)M);
  if (M == 0 || N == 0) return B2K_OK;
  B2K_REQUIRE(y && (K == 0 || (x && tiles && tile_scales)), "b2k_w4_matmul: null operand");
  B2K_REQUIRE(M <= 1 || (ldx >= K && ldy >= N), "b2k_w4_matmul: row stride smaller than the row");
  W4Args a = {};
  a.w = W4{static_cast<const unsigned char*>(tiles), tile_scales, tile_zeros, N, K, group};
  a.x = x; a.ldx = ldx; a.xs = xs; a.ldxs = ldxs; a.xgroup = xgroup;
  a.y = y; a.ldy = ldy; a.M = M;
  a.xtype = xtype; a.ytype = ytype; a.stype = stype;
  launch_pdl(w4_simple_kernel, dim3((unsigned)((M * N + 3) / 4)), dim3(128), 0,
             static_cast<cudaStream_t>(stream), a);
  return check_launch("b2k_w4_matmul");
}
