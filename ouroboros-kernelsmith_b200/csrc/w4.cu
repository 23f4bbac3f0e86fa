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
#include "rowpipe.cuh"

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
//
// Bound by reading the weights, N K / 2 bytes, while M is small.  A warp takes
// 16 weight rows (or twice that) as the 16 rows of mma.m16n8k16, the rows of
// x as its columns: the words of a tile are unpacked straight into A operands
// (`word & 0x000f000f` is a pair of float16 subnormals n 2^-24, exact; `&
// 0x00f000f0` 16 times that, against x / 16) and meet x from shared memory.
// Per group
//
//   y += s xs (sum x' n  -  z sum x'),    x = x' xs
//
// in fp32: x' is x in float16 after a power of two xs that brings the largest
// of the group's columns to [2^14, 2^15), so 16-bit x is exact unless it is
// 2^-25 of its group's maximum; float32 x takes two columns, x' = hi + 2^-11 lo
// (22 bits).  8-bit x is exact as it is and xs is its scale.
//
// Blocks are persistent and hold all of x (their slice of K) in shared memory,
// prepared once.  KW warps share a row tile, each with every KW-th block of 128
// columns; loads of the next ones are always in flight, across tiles too.
constexpr int kW4Smem = 200 << 10;  // shared memory of an SM that x may take

struct W4Args {
  W4 w;
  const void* x;
  int64_t ldx;
  const float* xs;  // scales of 8-bit x, [M, K / xgroup] (xgroup 0: one per row)
  int64_t ldxs;
  int xgroup;
  void* y;
  int64_t ldy, M;
  int xtype, ytype, stype, x_aligned;
  int KW;          // warps that share a row tile
  int kslice;      // blocks of 128 columns per grid.z
  int rows;        // rows of x per grid.y
  float* part;     // [grid.z][M][N] partial sums when K is split over blocks
};

// eight columns k .. k + 7 of row m as floats, zeros past K
__device__ __forceinline__ void w4_x8(const W4Args& a, int64_t m, int64_t k, float* v) {
  const bool whole = a.x_aligned && k + 8 <= a.w.K;
  const int64_t at = m * a.ldx + k;
  auto each = [&](auto get) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = k + e < a.w.K ? get(at + e) : 0.0f;
  };
  if (a.xtype == B2K_BF16) {
    const __nv_bfloat16* p = static_cast<const __nv_bfloat16*>(a.x);
    if (whole) unpack<__nv_bfloat16>(ld_keep(p + at), v);
    else each([&](int64_t i) { return to_f(p[i]); });
  } else if (a.xtype == B2K_F16) {
    const __half* p = static_cast<const __half*>(a.x);
    if (whole) unpack<__half>(ld_keep(p + at), v);
    else each([&](int64_t i) { return to_f(p[i]); });
  } else if (a.xtype == B2K_F32) {
    const float* p = static_cast<const float*>(a.x);
    if (whole) {
      unpack<float>(ld_keep(p + at), v);
      unpack<float>(ld_keep(p + at + 4), v + 4);
    } else {
      each([&](int64_t i) { return p[i]; });
    }
  } else {
    uint8_t b[8];
    const uint8_t* p = static_cast<const uint8_t*>(a.x);
    if (whole) {
      *reinterpret_cast<uint2*>(b) = __ldg(reinterpret_cast<const uint2*>(p + at));
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) b[e] = k + e < a.w.K ? p[at + e] : (uint8_t)0;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (a.xtype == B2K_I8) v[e] = (float)(int8_t)b[e];
      else v[e] = __half2float(__half(__nv_cvt_fp8_to_halfraw(b[e], __NV_E4M3)));
    }
  }
}

__device__ __forceinline__ uint32_t h2_bits(__half a, __half b) {
  const __half2 h = __halves2half2(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ void w4_mma(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                       uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// row tiles of 16 per warp, and blocks of 128 columns in flight
__host__ __device__ constexpr int w4_rt(int NT) { return NT == 1 ? 1 : 2; }
__host__ __device__ constexpr int w4_ring(int NT) { return NT == 1 ? 4 : 2; }

// bytes of x, its groups' sums and scales, and the warps' partial results
__host__ __device__ inline int64_t w4_x_bytes(int64_t kslice, int cols) { return kslice * 256 * cols; }
__host__ __device__ inline int64_t w4_g_bytes(int64_t kslice, int gs, int NT) {
  return kslice * gs * 64 * NT;
}
__host__ __device__ constexpr int w4_red_bytes(int NT) { return w4_rt(NT) * 16 * 8 * NT * 4; }

// GS = groups per 128 columns, 8 NT = columns (rows of x; two each for float32)
template <int NT, int GS> __global__ void __launch_bounds__(512, 1) w4_kernel(
    const __grid_constant__ W4Args a) {
  constexpr int RT = w4_rt(NT), UK = w4_ring(NT), G = 128 / GS;
  extern __shared__ __align__(128) unsigned char smem[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, r = lane >> 2, c = lane & 3;
  const int nwarps = blockDim.x >> 5;
  const int64_t KT = a.w.ktiles(), tiles = a.w.ntiles();
  const int64_t kb0 = (int64_t)blockIdx.z * a.kslice;
  const int kn = (int)min((int64_t)a.kslice, KT - kb0);  // blocks of this slice
  const int64_t m0 = (int64_t)blockIdx.y * a.rows;
  const int rows = (int)min((int64_t)a.rows, a.M - m0);
  const bool f32 = a.xtype == B2K_F32;
  const int C = f32 ? 2 * rows : rows;
  unsigned char* xsm = smem;
  float2* gsm = reinterpret_cast<float2*>(smem + w4_x_bytes(a.kslice, f32 ? 2 * a.rows : a.rows));
  float* red = reinterpret_cast<float*>(reinterpret_cast<unsigned char*>(gsm) +
                                        w4_g_bytes(a.kslice, GS, NT));

  // ---- this warp's stream of weights ---------------------------------------
  const int KW = a.KW, kw = warp % KW, grp = warp / KW, groups = nwarps / KW;
  const int64_t items = (tiles + RT - 1) / RT, step = (int64_t)gridDim.x * groups;
  const int64_t first = (int64_t)blockIdx.x * groups + grp;
  uint4 wa[UK][RT], wb[UK][RT];
  uint32_t ws[UK][RT], wz[UK][RT];
  int64_t pit = first;  // next to load
  int pk = kw;
  auto load = [&](int u) {
    if (pit < items && pk < kn) {
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        const int64_t tile = min(pit * RT + t, tiles - 1);
        const int64_t at = tile * KT + kb0 + pk;
        const uint4* p = reinterpret_cast<const uint4*>(a.w.tiles) + at * 64 + lane;
        wa[u][t] = __ldcs(p);
        wb[u][t] = __ldcs(p + 32);
        const int64_t si = (at * GS + c % GS) * 16 + r;
        const uint16_t* sp = static_cast<const uint16_t*>(a.w.scales) + si;
        ws[u][t] = (uint32_t)__ldcs(sp) | ((uint32_t)__ldcs(sp + 8) << 16);
        if (a.w.zeros) {
          const uint16_t* zp = static_cast<const uint16_t*>(a.w.zeros) + si;
          wz[u][t] = (uint32_t)__ldcs(zp) | ((uint32_t)__ldcs(zp + 8) << 16);
        }
      }
      pk += KW;
      if (pk >= kn) {
        pk = kw;
        pit += step;
      }
    }
  };
  griddep_launch_dependents();
  griddep_wait();
  if (kw < kn) {
#pragma unroll
    for (int u = 0; u < UK; ++u) load(u);
  }

  // ---- x into shared memory -------------------------------------------------
  // [32 columns][C][quarter c] of 16 bytes: columns (0,4) (2,6) and, / 16,
  // (1,5) (3,7) of the quarter's eight, the order of the unpacked words
  {
    const int per_row = kn * 16;  // eights of columns
    const int total = rows * per_row;
    for (int i = tid; i < kn * GS * 8 * NT; i += blockDim.x) gsm[i] = f2(0.0f, 0.0f);
    __syncthreads();
    for (int base = warp * 32; base < total; base += blockDim.x) {
      const int i = base + lane;
      const bool live = i < total;
      const int m = live ? i / per_row : 0, v8 = live ? i - m * per_row : 0;
      const int64_t k = kb0 * 128 + v8 * 8;
      float v[8];
      if (live) {
        w4_x8(a, m0 + m, k, v);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = 0.0f;
      }
      float f = 1.0f, xs;
      if (a.xs) {
        const int64_t g = a.xgroup ? k / a.xgroup : 0;
        xs = live && k < a.w.K ? a.xs[(m0 + m) * a.ldxs + g] * 16384.0f : 0.0f;
        // a group of 8-bit values that are not finite, or of such a scale, is NaN
        bool odd = false;
#pragma unroll
        for (int e = 0; e < 8; ++e) odd |= !isfinite(v[e]);
        if (odd) xs = __int_as_float(0x7fc00000);
#pragma unroll
        for (int o = 1; o < G / 8; o <<= 1) {
          const float t = __shfl_xor_sync(0xffffffffu, xs, o);
          if (t != t || k >= a.w.K) xs = t;
        }
      } else {
        uint32_t top = 0;  // magnitudes as integers: a NaN stays on top
#pragma unroll
        for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(v[e]) & 0x7fffffffu);
#pragma unroll
        for (int o = 1; o < G / 8; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
        const int ex = (int)(top >> 23);
        if (ex == 255) {
          xs = __int_as_float(0x7fc00000);
        } else {
          const int fb = min(268 - ex, 254);
          f = __uint_as_float((uint32_t)fb << 23);
          xs = __uint_as_float((uint32_t)(268 - fb) << 23);
        }
      }
      for (int part = 0; part < (f32 ? 2 : 1); ++part) {
        const int col = f32 ? 2 * m + part : m;
        __half h[8], h16[8];
        float sum = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float t = part == 0 ? v[e] * f : v[e];
          h[e] = __float2half_rn(t);
          const float back = __half2float(h[e]);
          sum += back;
          h16[e] = __float2half_rn(back * 0.0625f);
          v[e] = (t - back) * 2048.0f;
        }
#pragma unroll
        for (int o = 1; o < G / 8; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (live) {
          *reinterpret_cast<uint4*>(xsm + ((int64_t)(v8 >> 2) * C + col) * 64 + (v8 & 3) * 16) =
              make_uint4(h2_bits(h[0], h[4]), h2_bits(h[2], h[6]), h2_bits(h16[1], h16[5]),
                         h2_bits(h16[3], h16[7]));
          // the sum in units of the products, 2^-24
          if (v8 % (G / 8) == 0)
            gsm[(v8 / (G / 8)) * 8 * NT + col] = f2(sum * 5.9604644775390625e-8f, xs);
        }
      }
    }
    __syncthreads();
  }

  // ---- the group's warps add up a tile; its rows are columns of y ------------
  auto join = [&](int64_t it, float (&y)[RT][NT][4]) {
    constexpr int PER = RT * 16 * 8 * NT;
    if (KW > 1) named_bar_sync(1 + grp, 32 * KW);  // the last tile's sums are read
    float* mine = red + (int64_t)warp * PER;       // [column][RT * 16 rows]
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          mine[(nt * 8 + 2 * c + (e & 1)) * RT * 16 + t * 16 + r + 8 * (e >> 1)] = y[t][nt][e];
    if (KW > 1) named_bar_sync(1 + grp, 32 * KW);
    else __syncwarp();
    const float* from = red + (int64_t)(grp * KW) * PER;
    for (int i = kw * 32 + lane; i < rows * RT * 16; i += 32 * KW) {
      const int m = i / (RT * 16), n16 = i - m * (RT * 16);
      const int64_t n = it * (RT * 16) + n16;
      if (n >= a.w.N) continue;
      float v = 0.0f;
      if (f32) {
        float lo = 0.0f;
        for (int w = 0; w < KW; ++w) {
          v += from[w * PER + (2 * m) * RT * 16 + n16];
          lo += from[w * PER + (2 * m + 1) * RT * 16 + n16];
        }
        v = fmaf(lo, 0.00048828125f, v);
      } else {
        for (int w = 0; w < KW; ++w) v += from[w * PER + i];
      }
      if (a.part) {
        a.part[((int64_t)blockIdx.z * a.M + m0 + m) * a.w.N + n] = v;
        continue;
      }
      const int64_t at = (m0 + m) * a.ldy + n;
      if (a.ytype == B2K_F32) static_cast<float*>(a.y)[at] = v;
      else if (a.ytype == B2K_F16) static_cast<__half*>(a.y)[at] = from_f<__half>(v);
      else static_cast<__nv_bfloat16*>(a.y)[at] = from_f<__nv_bfloat16>(v);
    }
    if (KW == 1) __syncwarp();
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) y[t][nt][e] = 0.0f;
  };

  // ---- tiles, as one stream of blocks whose ring slots are taken in turn ----
  float y[RT][NT][4];
#pragma unroll
  for (int t = 0; t < RT; ++t)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) y[t][nt][e] = 0.0f;
  int k = kw;
  for (int64_t it = first; it < items;) {
#pragma unroll
    for (int u = 0; u < UK; ++u) {
      if (it < items) {
        if (k < kn) {
          float acc[RT][NT][4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (j * 32 % G == 0) {
#pragma unroll
              for (int t = 0; t < RT; ++t)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                  for (int e = 0; e < 4; ++e) acc[t][nt][e] = 0.0f;
            }
            const unsigned char* xp = xsm + (int64_t)(4 * k + j) * C * 64 + r * 64 + c * 16;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              uint4 b = zero4();
              if (nt * 8 + r < C) b = *reinterpret_cast<const uint4*>(xp + nt * 512);
#pragma unroll
              for (int t = 0; t < RT; ++t) {
                const uint32_t w0 = j == 0 ? wa[u][t].x : j == 1 ? wa[u][t].y : j == 2 ? wa[u][t].z : wa[u][t].w;
                const uint32_t w1 = j == 0 ? wb[u][t].x : j == 1 ? wb[u][t].y : j == 2 ? wb[u][t].z : wb[u][t].w;
                const uint32_t v0 = w0 >> 8, v1 = w1 >> 8;
                w4_mma(acc[t][nt], w0 & 0x000f000fu, w1 & 0x000f000fu, v0 & 0x000f000fu,
                       v1 & 0x000f000fu, b.x, b.y);
                w4_mma(acc[t][nt], w0 & 0x00f000f0u, w1 & 0x00f000f0u, v0 & 0x00f000f0u,
                       v1 & 0x00f000f0u, b.z, b.w);
              }
            }
            if ((j + 1) * 32 % G == 0) {
              const int gi = j * 32 / G;
              const float4* gp = reinterpret_cast<const float4*>(gsm + (k * GS + gi) * 8 * NT + 2 * c);
              float4 g4[NT];  // (sum, scale) of columns 2c, 2c + 1
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) g4[nt] = gp[nt * 4];
#pragma unroll
              for (int t = 0; t < RT; ++t) {
                const int src = (lane & ~3) | gi;
                const uint32_t sb = GS == 1 ? ws[u][t] : __shfl_sync(0xffffffffu, ws[u][t], src);
                float s0, s1, z0 = 8.0f, z1 = 8.0f;
                if (a.stype == B2K_F16) {
                  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&sb));
                  s0 = f.x; s1 = f.y;
                } else {
                  s0 = __uint_as_float(sb << 16); s1 = __uint_as_float(sb & 0xffff0000u);
                }
                if (a.w.zeros) {
                  const uint32_t zb = GS == 1 ? wz[u][t] : __shfl_sync(0xffffffffu, wz[u][t], src);
                  if (a.stype == B2K_F16) {
                    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&zb));
                    z0 = f.x; z1 = f.y;
                  } else {
                    z0 = __uint_as_float(zb << 16); z1 = __uint_as_float(zb & 0xffff0000u);
                  }
                }
                s0 *= 1024.0f;  // 2^24 of the integers' unit, 2^-14 of x's
                s1 *= 1024.0f;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                  float* q = acc[t][nt];
                  const float4 g = g4[nt];
                  y[t][nt][0] = fmaf(fmaf(-z0, g.x, q[0]) * s0, g.y, y[t][nt][0]);
                  y[t][nt][1] = fmaf(fmaf(-z0, g.z, q[1]) * s0, g.w, y[t][nt][1]);
                  y[t][nt][2] = fmaf(fmaf(-z1, g.x, q[2]) * s1, g.y, y[t][nt][2]);
                  y[t][nt][3] = fmaf(fmaf(-z1, g.z, q[3]) * s1, g.w, y[t][nt][3]);
                }
              }
            }
          }
          load(u);
        }
        k += KW;
        if (k >= kn) {
          join(it, y);
          k = kw;
          it += step;
        }
      }
    }
  }
}

// y = the sum of K's slices, in order
template <typename T> __global__ void __launch_bounds__(256) w4_sum_kernel(const float* part, int slices,
                                                                          T* y, int64_t ldy,
                                                                          int64_t M, int64_t N) {
  griddep_launch_dependents();
  griddep_wait();
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < M * N; i += (int64_t)gridDim.x * 256) {
    float v = 0.0f;
    for (int s = 0; s < slices; ++s) v += part[(int64_t)s * M * N + i];
    const int64_t m = i / N;
    st1(y + m * ldy + (i - m * N), v);
  }
}

// How a product is split.  Blocks are of 8 warps, two per SM, while x fits half
// an SM's shared memory, else of 16; K is split over blocks only when x does
// not fit at all.  KW is the number of warps per tile that leaves the longest
// warp the least to do, counting a tile's join as two blocks of 128 columns.
struct W4Plan {
  int nt, rows, warps, cps, kslice, slices, kw, grid_x, grid_y;
  int64_t smem, bytes;
};

static W4Plan w4_plan(int64_t M, int64_t N, int64_t K, int group, bool f32) {
  W4Plan p;
  const int per = f32 ? 2 : 1;
  const int64_t cols = M * per, KT = (K + 127) / 128, tiles = (N + 15) / 16;
  p.nt = cols <= 8 ? 1 : cols <= 16 ? 2 : 4;
  p.rows = (int)(M < 8 * p.nt / per ? M : 8 * p.nt / per);
  p.grid_y = (int)((M + p.rows - 1) / p.rows);
  const int gs = 128 / group;
  auto need = [&](int64_t kslice, int warps) {
    return w4_x_bytes(kslice, p.rows * per) + w4_g_bytes(kslice, gs, p.nt) +
           (int64_t)warps * w4_red_bytes(p.nt);
  };
  p.slices = 1;
  p.kslice = (int)(KT > 0 ? KT : 1);
  p.warps = 8;
  p.cps = 2;
  if (need(p.kslice, 8) > kW4Smem / 2) {
    p.warps = 16;
    p.cps = 1;
    while (need(p.kslice, 16) > kW4Smem) {
      ++p.slices;
      p.kslice = (int)((KT + p.slices - 1) / p.slices);
    }
    p.slices = (int)((KT + p.kslice - 1) / p.kslice);
  }
  p.smem = need(p.kslice, p.warps);
  const int64_t items = (tiles + w4_rt(p.nt) - 1) / w4_rt(p.nt);
  int64_t slots = (int64_t)sm_count() * p.cps / (p.slices * p.grid_y);
  if (slots < 1) slots = 1;
  int64_t best = -1;
  for (int kw = 1; kw <= p.warps; kw <<= 1) {
    const int64_t rounds = (items * kw + slots * p.warps - 1) / (slots * p.warps);
    const int64_t cost = rounds * ((p.kslice + kw - 1) / kw + (kw > 1 ? 2 : 1));
    if (best < 0 || cost < best) {
      best = cost;
      p.kw = kw;
    }
  }
  const int64_t blocks = (items * p.kw + p.warps - 1) / p.warps;
  p.grid_x = (int)(blocks < slots ? (blocks > 0 ? blocks : 1) : slots);
  p.bytes = p.slices > 1 ? (int64_t)p.slices * M * N * 4 : 0;
  return p;
}

template <int NT, int GS> static void w4_launch(const W4Args& a, const W4Plan& p, cudaStream_t st) {
  auto kern = w4_kernel<NT, GS>;
  allow_max_dynamic_smem(kern);
  launch_pdl(kern, dim3(p.grid_x, p.grid_y, p.slices), dim3(32 * p.warps), (size_t)p.smem, st, a);
}

template <int NT> static void w4_dispatch(const W4Args& a, const W4Plan& p, cudaStream_t st) {
  switch (a.w.g) {
    case 32: w4_launch<NT, 4>(a, p, st); break;
    case 64: w4_launch<NT, 2>(a, p, st); break;
    default: w4_launch<NT, 1>(a, p, st); break;
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

extern "C" int64_t b2k_w4_matmul_workspace(int64_t M, int64_t N, int64_t K, int group, int xtype) {
  if (M < 0 || N < 0 || K < 0 || M > 0x7fffffffLL || (group != 32 && group != 64 && group != 128))
    return -1;
  if (M == 0 || N == 0) return 0;
  return w4_plan(M, N, K, group, xtype == B2K_F32).bytes;
}

extern "C" int b2k_w4_matmul(const void* x, int64_t ldx, int xtype, const float* xs, int64_t ldxs,
                             int xgroup, const void* tiles, const void* tile_scales,
                             const void* tile_zeros, int stype, int group, int64_t M, int64_t N,
                             int64_t K, void* y, int64_t ldy, int ytype, void* workspace,
                             int64_t workspace_bytes, void* stream) {
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
  const W4Plan p = w4_plan(M, N, K, group, xtype == B2K_F32);
  B2K_REQUIRE(p.grid_y <= 65535 && p.slices <= 65535, "b2k_w4_matmul: shape too large");
  B2K_REQUIRE(p.bytes == 0 || (workspace && workspace_bytes >= p.bytes &&
                               (reinterpret_cast<uintptr_t>(workspace) & 3u) == 0),
              "b2k_w4_matmul: the workspace needs %lld bytes, got %lld", (long long)p.bytes,
              (long long)workspace_bytes);
  const int xsize = dtype_size(xtype);
  // eight columns are read as 16-byte vectors (8 bytes for 8-bit x)
  a.x_aligned = reinterpret_cast<uintptr_t>(x) % (xsize == 1 ? 8 : 16) == 0 &&
                ldx * xsize % (xsize == 1 ? 8 : 16) == 0;
  a.KW = p.kw; a.kslice = p.kslice; a.rows = p.rows;
  a.part = p.bytes ? static_cast<float*>(workspace) : nullptr;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (p.nt == 1) w4_dispatch<1>(a, p, st);
  else if (p.nt == 2) w4_dispatch<2>(a, p, st);
  else w4_dispatch<4>(a, p, st);
  if (a.part) {
    const unsigned grid = w4_blocks(M * N);
    B2K_DISPATCH_FLOAT(ytype, {
      launch_pdl(w4_sum_kernel<T>, dim3(grid), dim3(256), 0, st, static_cast<const float*>(a.part),
                 p.slices, static_cast<T*>(y), ldy, M, N);
    });
  }
  return check_launch("b2k_w4_matmul");
}
