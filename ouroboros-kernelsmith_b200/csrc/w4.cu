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
#include <limits.h>

#include "ring.cuh"
#include "rowio.cuh"
#include "rowpipe.cuh"

B2K_DEFINE_TIMEOUT_COUNTER()

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
// 16 weight rows as the 16 rows of mma.m16n8k16, the rows of
// x as its columns: the words of a tile are unpacked straight into A operands
// (`word & 0x000f000f` is a pair of float16 subnormals n 2^-24, exact; `&
// 0x00f000f0` 16 times that, against x / 16) and meet x from shared memory.
// Per group
//
//   y += s xs (sum x' n  -  z sum x'),    x = x' xs
//
// in fp32: x' is x in float16 after a power of two xs that brings the largest
// of the group's columns to [2^14, 2^15), so 16-bit x is exact unless it is
// 2^-25 of its group's maximum; float32 x takes three columns, x' = hi + 2^-11
// mid + 2^-22 lo.  Of these hi and mid are multiples of 16, up to 2^15 and 2^14:
// their products with the integers, and the sums of 128, are multiples of 16 below
// 2^26, so nothing of them is lost beside a column that is much larger than the
// others.  (The matrix instruction drops what lies 24 bits below its largest term:
// two columns of 11 leading bits each were off by 2^-17 of the result in such
// rows, and took 21.1 us instead of 29.8 at 4 x 4096 x 28672, 45.7 instead of 88
// with 16 rows.)  A row takes four columns, the last empty.  8-bit x is exact (x'
// = 128 x) and xs goes by its scale.
//
// Blocks are persistent, one per SM, and hold all of x (their slice of K) in
// shared memory, prepared once.  A block takes an equal share of the row tiles
// and its warps equal runs of their blocks of 128 columns, whatever tile these
// lie in; a tile that spans warps is added up at the end.  Every warp has its
// own ring of bulk copies, which runs ahead across tiles.
constexpr int kW4F32 = 4;  // columns of a row of float32
constexpr int kW4Stages = 4, kW4Smem = 226 << 10;  // stages at most; of an SM's memory

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
  int kslice;      // blocks of 128 columns per grid.z
  int rows;        // rows of x per grid.y
  int64_t each, more;  // items of a block; one more in the first `more`
  int stages;      // of a warp's ring
  unsigned char* xw;  // x prepared by w4_x_kernel (null: each block prepares its own)
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

// the same on zero sums
__device__ __forceinline__ void w4_mma_first(float* c, uint32_t a0, uint32_t a1, uint32_t a2,
                                             uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%10,%10,%10,%10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}

constexpr int kW4Warps = 16;  // of a block
constexpr int kW4Blocks = 2;  // of 128 columns in a stage of a warp's ring
// stage: 2 KB of weights, then the scales and the zeros of their groups
__host__ __device__ constexpr int w4_stage(int gs) { return 2048 + 128 * gs; }
// bytes of x, and of its groups' sums and scales, for kslice blocks of columns;
// and of both for all of K in the workspace
__host__ __device__ inline int64_t w4_x_bytes(int64_t kslice, int cols) { return kslice * 256 * cols; }
__host__ __device__ inline int64_t w4_g_bytes(int64_t kslice, int gs, int NT) {
  return kslice * gs * 64 * NT;
}
__host__ __device__ inline int64_t w4_image_bytes(int64_t KT, int cols, int gs, int NT) {
  return w4_x_bytes(KT, cols) + w4_g_bytes(KT, gs, NT);
}

// Eight columns of one row of x (column 128 kb0 + 8 v8) into the form that the
// products read, by all lanes of a warp (`live`: this lane has any):
//   xo  [32 columns][C][quarter] of 16 bytes: columns (0,4) (2,6) and, / 16,
//       (1,5) (3,7) of the quarter's eight, the order of the unpacked words
//   go  [group][pitch] of (sum, scale)
template <int GS>
__device__ __forceinline__ void w4_stage_eight(const W4Args& a, int64_t row, int64_t kb0, int v8,
                                               bool live, int m, int C, unsigned char* xo,
                                               float2* go, int pitch) {
  constexpr int G = 128 / GS;
  const bool f32 = a.xtype == B2K_F32;
  const int64_t k = kb0 * 128 + (int64_t)v8 * 8;
  float v[8];
  if (live) {
    w4_x8(a, row, k, v);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = 0.0f;
  }
  float f = 1.0f, xs;
  if (a.xs) {
    const int64_t g = a.xgroup ? k / a.xgroup : 0;
    // half of the units' 2^14 in the values, where it is exact (448 * 128 fits
    // float16), so that the scales of the largest fp32 rows stay finite
    f = 128.0f;
    xs = live && k < a.w.K ? a.xs[row * a.ldxs + g] * 128.0f : 0.0f;
    // a group of 8-bit values that are not finite, or of such a scale, is NaN
    bool odd = false;
#pragma unroll
    for (int e = 0; e < 8; ++e) odd |= !isfinite(v[e]);
    if (odd || !isfinite(xs)) xs = __int_as_float(0x7fc00000);
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
  for (int part = 0; part < (f32 ? 3 : 1); ++part) {
    const int col = f32 ? kW4F32 * m + part : m;
    __half h[8], h16[8];
    float sum = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float t = part == 0 ? v[e] * f : v[e];
      const float all = t;
      // float32: multiples of 16, first of x' and then of 2^11 times the rest
      if (f32 && part < 2) t = rintf(t * 0.0625f) * 16.0f;
      h[e] = __float2half_rn(t);
      const float back = __half2float(h[e]);
      sum += back;
      h16[e] = __float2half_rn(back * 0.0625f);
      v[e] = (all - back) * 2048.0f;
    }
#pragma unroll
    for (int o = 1; o < G / 8; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (live) {
      *reinterpret_cast<uint4*>(xo + ((int64_t)(v8 >> 2) * C + col) * 64 + (v8 & 3) * 16) =
          make_uint4(h2_bits(h[0], h[4]), h2_bits(h[2], h[6]), h2_bits(h16[1], h16[5]),
                     h2_bits(h16[3], h16[7]));
      // the sum in units of the products, 2^-24
      if (v8 % (G / 8) == 0) {
        float2* to = go + (int64_t)(v8 / (G / 8)) * pitch + col;
        to[0] = f2(sum * 5.9604644775390625e-8f, xs);
        if (f32 && part == 2) to[1] = f2(0.0f, 0.0f);  // the row's fourth column
      }
    }
  }
}

// The whole of x, once, in the form of the blocks' shared memory: for every
// grid.y of the product its rows' image and their groups (zeros for columns
// past the rows).  A warp takes 32 eights of a row.
template <int GS>
__global__ void __launch_bounds__(256) w4_x_kernel(const __grid_constant__ W4Args a, int nt) {
  griddep_wait();
  // Only now: the product starts on its weights before it waits for this grid,
  // and what came before this grid may have written them.
  griddep_launch_dependents();
  const int64_t KT = a.w.ktiles(), per_row = KT * 16;
  const int per = a.xtype == B2K_F32 ? kW4F32 : 1, cols = a.rows * per;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t y = blockIdx.y, m0 = y * a.rows;
  const int rows = (int)min((int64_t)a.rows, a.M - m0);
  const bool live = i < rows * per_row;
  const int m = live ? (int)(i / per_row) : 0;
  const int v8 = live ? (int)(i - m * per_row) : 0;
  unsigned char* xo = a.xw + y * w4_image_bytes(KT, cols, GS, nt);
  float2* go = reinterpret_cast<float2*>(xo + KT * 256 * cols);
  w4_stage_eight<GS>(a, m0 + m, 0, v8, live, m, rows * per, xo, go, 8 * nt);
  if (live && m == 0 && v8 % (16 / GS) == 0)
    for (int col = rows * per; col < 8 * nt; ++col)
      go[(int64_t)(v8 / (16 / GS)) * 8 * nt + col] = f2(0.0f, 0.0f);
}

// GS = groups per 128 columns, 8 NT = columns (rows of x; four each for
// float32, F32), BF: scales and zeros are bfloat16
template <int NT, int GS, bool BF, bool F32>
__global__ void __launch_bounds__(32 * kW4Warps, 1) w4_kernel(const __grid_constant__ W4Args a) {
  constexpr int G = 128 / GS, STAGE = w4_stage(GS);
  constexpr int SBK = kW4Blocks, W = kW4Warps;
  const int S = a.stages;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ uint64_t full[16][kW4Stages], xbar;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, r = lane >> 2, c = lane & 3;
  const int64_t KT = a.w.ktiles(), tiles = a.w.ntiles();
  const int64_t kb0 = (int64_t)blockIdx.z * a.kslice;
  const int kn = (int)min((int64_t)a.kslice, KT - kb0);  // blocks of this slice
  const int64_t m0 = (int64_t)blockIdx.y * a.rows;
  const int rows = (int)min((int64_t)a.rows, a.M - m0);
  const bool zeros = a.w.zeros != nullptr;
  constexpr int per = F32 ? kW4F32 : 1;
  const int C = per * rows;
  unsigned char* ring = smem + warp * (S * STAGE);
  unsigned char* xsm = smem + W * (S * STAGE);
  float2* gsm = reinterpret_cast<float2*>(xsm + w4_x_bytes(a.kslice, per * a.rows));
  // 16 zero bytes, what lanes past the last column read
  const uint32_t nothing = (uint32_t)(reinterpret_cast<unsigned char*>(gsm) - smem) +
                           (uint32_t)w4_g_bytes(a.kslice, GS, NT);

  // ---- this warp's run of blocks --------------------------------------------
  // The block's items, its row tiles, laid end to end, kn blocks of columns
  // apiece, and divided into equal runs.  A run's whole items are taken first,
  // then the end of the run that begins another item (its tail), last its head,
  // the end of an item that an earlier warp begins.
  const int64_t b = blockIdx.x;
  const int64_t i0 = b * a.each + min(b, a.more);        // its items: the first
  const int n_items = (int)(a.each + (b < a.more));      // and their number
  const int64_t units = (int64_t)n_items * kn;
  auto run_at = [&](int w) { return (int)(w * units / W); };
  const int u0 = run_at(warp), u1 = run_at(warp + 1);
  // whole items before the run's first item boundary, and where that lies
  const int before = kn > 0 ? (int)((uint32_t)(u0 + kn - 1) / (uint32_t)kn) : 0;
  const int body = min(u1, before * kn);

  // a walk over the run: blocks [k, end) of item i0 + item
  struct Walk {
    int item, k, end, at;  // at: the units up to here, past u1 after the head
  };
  // the next item of the walk; false after the last
  auto next_item = [&](Walk& w) {
    if (w.at < u1 && w.at >= body) {
      w.k = 0;
      w.end = min(kn, u1 - w.at);
      w.at += w.end;
      return true;
    }
    if (w.at == u1 && u0 < body) {  // from the body to the head
      w.item = before - 1;
      w.k = u0 - w.item * kn;
      w.end = w.k + body - u0;
      w.at = INT_MAX;
      return true;
    }
    return false;
  };
  const Walk begin = {before, 0, 0, body};
  Walk get = begin;
  int get_stage = 0;
  uint32_t issued = 0;
  RingUse taken;
  auto arrived = [&](int stage, uint32_t phase) { return mbar_wait_warp(&full[warp][stage], phase); };
  int64_t get_at = 0;  // block of the item's (first) tile in the layout
  int get_left = 0;    // blocks of it to come
  bool getting = false;
  auto open = [&]() {
    getting = u0 < u1 && next_item(get);
    get_at = (i0 + get.item) * KT + kb0 + get.k;
    get_left = get.end - get.k;
  };
  auto issue = [&]() {
    if (lane == 0) {
      const int n = min(SBK, get_left);
      uint64_t* bar = &full[warp][get_stage];
      unsigned char* dst = ring + get_stage * STAGE;
      const uint32_t wb = n * 1024, sb = n * GS * 32;
      fence_proxy_async();
      mbar_arrive_expect_tx(bar, wb + (zeros ? 2 : 1) * sb);
      bulk_g2s(dst, a.w.tiles + get_at * 1024, wb, bar);
      bulk_g2s(dst + 2048, static_cast<const unsigned char*>(a.w.scales) + get_at * GS * 32,
               sb, bar);
      if (zeros)
        bulk_g2s(dst + 2048 + SBK * GS * 32,
                 static_cast<const unsigned char*>(a.w.zeros) + get_at * GS * 32, sb, bar);
    }
    if (++get_stage == S) get_stage = 0;
    ++issued;
    get_at += SBK;
    get_left -= SBK;
    if (get_left <= 0) {
      ++get.item;
      open();
    }
  };
  griddep_launch_dependents();
  if (lane < S) mbar_init(&full[warp][lane], 1);
  if (tid == 0) *reinterpret_cast<uint4*>(smem + nothing) = zero4();
  fence_barrier_init();
  __syncwarp();
  // With x prepared by the kernel before, the weights need not wait for it.
  if (!a.xw) griddep_wait();
  open();
  for (int s = 0; s < S && getting; ++s) issue();
  if (a.xw) griddep_wait();

  // ---- x into shared memory -------------------------------------------------
  if (a.xw) {  // prepared by w4_x_kernel
    if (tid == 0) {
      mbar_init(&xbar, 1);
      fence_barrier_init();
    }
    __syncthreads();
    if (tid == 0) {
      const unsigned char* xw = a.xw + (int64_t)blockIdx.y * w4_image_bytes(KT, per * a.rows, GS, NT);
      const uint32_t xb = kn * 256 * C, gb = kn * GS * 64 * NT;
      fence_proxy_async();
      mbar_arrive_expect_tx(&xbar, xb + gb);
      for (uint32_t o = 0; o < xb; o += 32768)
        bulk_g2s(xsm + o, xw + kb0 * 256 * C + o, min(xb - o, 32768u), &xbar);
      bulk_g2s(gsm, xw + KT * 256 * (per * a.rows) + kb0 * GS * 64 * NT, gb, &xbar);
    }
    taken.dead = !mbar_wait_warp(&xbar, 0);  // then nothing is taken from the ring
  } else {
    for (int i = tid; i < kn * GS * 8 * NT; i += blockDim.x) gsm[i] = f2(0.0f, 0.0f);
    __syncthreads();
    const int per_row = kn * 16, total = rows * per_row;  // eights of columns
    for (int base = warp * 32; base < total; base += blockDim.x) {
      const int i = base + lane, m = min(i, total - 1) / per_row;
      w4_stage_eight<GS>(a, m0 + m, kb0, i - m * per_row, i < total, m, C, xsm, gsm, 8 * NT);
    }
    __syncthreads();
  }

  // ---- results ----------------------------------------------------------------
  const int odd = r & 1, row_a = 2 * r + odd, row_b = 2 * r + 1 - odd;  // rows r, r + 8 of the products
  // column n of row m of y (of the partial sums when K is split)
  auto store = [&](int m, int64_t n, float v) {
    if (n >= a.w.N) return;
    if (a.part) {
      a.part[((int64_t)blockIdx.z * a.M + m0 + m) * a.w.N + n] = v;
      return;
    }
    const int64_t at = (m0 + m) * a.ldy + n;
    if (a.ytype == B2K_F32) static_cast<float*>(a.y)[at] = v;
    else if (a.ytype == B2K_F16) static_cast<__half*>(a.y)[at] = from_f<__half>(v);
    else static_cast<__nv_bfloat16*>(a.y)[at] = from_f<__nv_bfloat16>(v);
  };
  constexpr float kLow = 0.00048828125f;  // 2^-11, from a column of float32 to the next

  float y[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) y[nt][e] = 0.0f;
  const uint32_t swap = odd ? 0x1032u : 0x3210u;
  // this lane's fragments of x: where, and from one 32 columns to the next
  uint32_t xat[NT], xstep[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const bool in = nt * 8 + r < C && !(F32 && (r & 3) == 3);
    xat[nt] = in ? (uint32_t)(xsm - smem) + (nt * 8 + r) * 64 + c * 16 : nothing;
    xstep[nt] = in ? C * 64 : 0;
  }
  float tail[NT][4];  // of the item that the run begins and does not end
  int tail_item = -1;
  Walk use = begin;
  while (u0 < u1 && next_item(use)) {
    for (int k = use.k; k < use.end; k += SBK) {
      const int stage = taken.take(S, arrived);
      if (stage < 0) break;
      const unsigned char* st = ring + stage * STAGE;
#pragma unroll
      for (int i = 0; i < SBK; ++i) {
        if (k + i >= use.end) break;
        const uint4 wa = *reinterpret_cast<const uint4*>(st + i * 1024 + row_a * 64 + c * 16);
        const uint4 wb = *reinterpret_cast<const uint4*>(st + i * 1024 + row_b * 64 + c * 16);
        // two sums for 8 columns (even and odd nibbles), so that half as many
        // products wait for one another
        constexpr int CH = NT == 1 ? 2 : 1;
        float acc[CH][NT][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t w0 = j == 0 ? wa.x : j == 1 ? wa.y : j == 2 ? wa.z : wa.w;
          const uint32_t w1 = j == 0 ? wb.x : j == 1 ? wb.y : j == 2 ? wb.z : wb.w;
          const uint32_t v0 = w0 >> 8, v1 = w1 >> 8;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const uint4 b = *reinterpret_cast<const uint4*>(smem + xat[nt] + (4 * (k + i) + j) * xstep[nt]);
            if (j * 32 % G == 0)
              w4_mma_first(acc[0][nt], w0 & 0x000f000fu, w1 & 0x000f000fu, v0 & 0x000f000fu,
                           v1 & 0x000f000fu, b.x, b.y);
            else
              w4_mma(acc[0][nt], w0 & 0x000f000fu, w1 & 0x000f000fu, v0 & 0x000f000fu,
                     v1 & 0x000f000fu, b.x, b.y);
            if (CH == 2 && j * 32 % G == 0)
              w4_mma_first(acc[CH - 1][nt], w0 & 0x00f000f0u, w1 & 0x00f000f0u, v0 & 0x00f000f0u,
                           v1 & 0x00f000f0u, b.z, b.w);
            else
              w4_mma(acc[CH - 1][nt], w0 & 0x00f000f0u, w1 & 0x00f000f0u, v0 & 0x00f000f0u,
                     v1 & 0x00f000f0u, b.z, b.w);
          }
          if ((j + 1) * 32 % G == 0) {
            const int gi = j * 32 / G;
            // (sum, scale) of columns 2c, 2c + 1 of x; scales and zeros of rows 2r, 2r + 1
            const float4* gp = reinterpret_cast<const float4*>(gsm + ((k + i) * GS + gi) * (8 * NT) + 2 * c);
            const uint32_t* sp = reinterpret_cast<const uint32_t*>(st + 2048 + (i * GS + gi) * 32) + r;
            auto two = [&](uint32_t bits) {
              bits = __byte_perm(bits, 0, swap);
              if constexpr (!BF) return __half22float2(*reinterpret_cast<const __half2*>(&bits));
              else return f2(__uint_as_float(bits << 16), __uint_as_float(bits & 0xffff0000u));
            };
            const float2 z = zeros ? two(sp[SBK * GS * 8]) : f2s(8.0f);
            // 2^10: 2^24 of the integers' unit, 2^-14 of x's
            const float2 s = mul2(two(*sp), f2s(1024.0f));
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              float q[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) q[e] = CH == 2 ? acc[0][nt][e] + acc[CH - 1][nt][e] : acc[0][nt][e];
              const float4 g = gp[nt * 4];
              y[nt][0] = fmaf(fmaf(-z.x, g.x, q[0]) * s.x, g.y, y[nt][0]);
              y[nt][1] = fmaf(fmaf(-z.x, g.z, q[1]) * s.x, g.w, y[nt][1]);
              y[nt][2] = fmaf(fmaf(-z.y, g.x, q[2]) * s.y, g.y, y[nt][2]);
              y[nt][3] = fmaf(fmaf(-z.y, g.z, q[3]) * s.y, g.w, y[nt][3]);
            }
          }
        }
      }
      __syncwarp();
      if (getting) issue();
    }
    if (taken.dead) break;
    if (use.at == INT_MAX) break;  // the head stays in y
    const bool ends = use.end == kn;
    const int64_t item = i0 + use.item;
    ++use.item;
    if (!ends) {
      tail_item = use.item - 1;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) tail[nt][e] = y[nt][e];
    } else {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int64_t n = item * 16 + (h ? row_b : row_a);
            const float v0 = y[nt][2 * h], v1 = y[nt][2 * h + 1];
            const int col = nt * 8 + 2 * c;
            if (F32) {
              const float v2 = __shfl_down_sync(0xffffffffu, v0, 1);  // columns 2c + 2
              if (!(c & 1) && col < C) store(col / kW4F32, n, fmaf(v2, kLow * kLow, fmaf(v1, kLow, v0)));
            } else {
              if (col < C) store(col, n, v0);
              if (col + 1 < C) store(col + 1, n, v1);
            }
          }
    }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) y[nt][e] = 0.0f;
  }
  if (taken.dead) {  // a wait ran out: nothing may land where the parts go, or later
    taken.drain(issued, S, arrived);
    if (a.xw) mbar_wait_warp(&xbar, 0);
    if (lane == 0) atomicAdd(&b2k_tu_timeouts, 1u);
    // the item at hand and those to come are NaN
    while (u0 < u1 && use.at != INT_MAX) {
      if (use.end != kn) {
        tail_item = use.item;
      } else {
        for (int i = lane; i < rows * 16; i += 32)
          store(i >> 4, (i0 + use.item) * 16 + (i & 15), __int_as_float(0x7fc00000));
      }
      ++use.item;
      if (!next_item(use)) break;
    }
  }

  // ---- items that span warps: their parts, in the warps' drained rings ----------
  if (kn == 0) {  // no columns at all
    for (int64_t i = tid; i < (int64_t)n_items * 16 * rows; i += blockDim.x)
      store((int)(i % rows), i0 * 16 + i / rows, 0.0f);
    return;
  }
  constexpr int PER = 16 * 8 * NT;
  const bool has_tail = tail_item >= 0;
  __syncwarp();
  float* mine = reinterpret_cast<float*>(ring);  // [head, tail][column][16 rows]
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int at = (nt * 8 + 2 * c + (e & 1)) * 16 + (e >> 1 ? row_b : row_a);
        // zeros where there is no head
        mine[at] = taken.dead ? __int_as_float(0x7fc00000) : y[nt][e];
        if (has_tail) mine[PER + at] = taken.dead ? __int_as_float(0x7fc00000) : tail[nt][e];
      }
  __syncthreads();
  // this warp's tail, and the heads of the next warps whose runs lie in that item
  if (!has_tail) return;
  const int past = (tail_item + 1) * kn;
  int last = warp;
#pragma unroll
  for (int w = 1; w < W; ++w) last += w > warp && run_at(w) < past;
  for (int i = lane; i < rows * 16; i += 32) {
    const int m = i >> 4, n16 = i & 15;
    const int c0 = per * m * 16 + n16;
    const float* from = reinterpret_cast<const float*>(smem);
    float v = 0.0f;
    for (int part = F32 ? 2 : 0; part >= 0; --part) {
      const int at = c0 + part * 16;
      float t = mine[PER + at];
#pragma unroll 4
      for (int w = warp + 1; w <= last; ++w) t += from[w * (S * STAGE / 4) + at];
      v = fmaf(v, kLow, t);
    }
    store(m, (i0 + tail_item) * 16 + n16, v);
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

// How a product is split.  One block per SM, its warps' rings as deep as shared
// memory allows beside x (2 to kW4Stages stages); K is split over blocks where
// x does not fit beside that.  x is prepared once by a kernel of its own where
// every block's own preparation would take it more than kW4Own eights of
// columns per thread (own preparation against the kernel: 1 x 4096 x 4096 5.6
// and 6.2 us, 1 x 14336 x 4096 16.2 and 15.4, 8 x 11008 x 4096 23.0 and 15.2, 16 x 4096 x 128256 95 and 83).
constexpr int kW4Own = 2;
struct W4Plan {
  int nt, rows, stages, kslice, slices, grid_x, grid_y;
  bool prepare;
  int64_t smem, image, bytes, each, more;
};

static W4Plan w4_plan(int64_t M, int64_t N, int64_t K, int group, bool f32) {
  W4Plan p;
  const int per = f32 ? kW4F32 : 1, gs = 128 / group;
  const int64_t cols = M * per, KT = (K + 127) / 128, tiles = (N + 15) / 16;
  p.nt = cols <= 8 ? 1 : cols <= 16 ? 2 : 4;
  p.rows = (int)(M < 8 * p.nt / per ? M : 8 * p.nt / per);
  p.grid_y = (int)((M + p.rows - 1) / p.rows);
  auto need = [&](int64_t kslice, int stages) {
    return w4_x_bytes(kslice, p.rows * per) + w4_g_bytes(kslice, gs, p.nt) +
           (int64_t)kW4Warps * stages * w4_stage(gs) + 16;
  };
  p.slices = 1;
  p.kslice = (int)(KT > 0 ? KT : 1);
  while (need(p.kslice, 2) > kW4Smem) {
    ++p.slices;
    p.kslice = (int)((KT + p.slices - 1) / p.slices);
  }
  p.slices = KT > 0 ? (int)((KT + p.kslice - 1) / p.kslice) : 1;
  p.stages = kW4Stages;
  while (need(p.kslice, p.stages) > kW4Smem) --p.stages;
  p.prepare = (int64_t)p.rows * p.kslice * 16 > kW4Own * 32 * kW4Warps;
  p.smem = need(p.kslice, p.stages);
  int64_t slots = (int64_t)sm_count() / (p.slices * p.grid_y);
  if (slots < 1) slots = 1;
  p.grid_x = (int)(tiles < slots ? tiles : slots);
  p.each = tiles / p.grid_x;
  p.more = tiles % p.grid_x;
  p.image = p.prepare ? p.grid_y * w4_image_bytes(KT, p.rows * per, gs, p.nt) : 0;
  p.bytes = p.image + (p.slices > 1 ? (int64_t)p.slices * M * N * 4 : 0);
  return p;
}

// rows of x in one launch: 65535 blocks of 32 columns
static int64_t w4_most_rows(bool f32) { return (int64_t)65535 * 32 / (f32 ? kW4F32 : 1); }

template <int NT, int GS, bool BF> static void w4_launch(const W4Args& a, const W4Plan& p, cudaStream_t st) {
  if (p.prepare) {
    const int64_t eights = (int64_t)p.rows * a.w.ktiles() * 16;
    launch_pdl(w4_x_kernel<GS>, dim3((unsigned)((eights + 255) / 256), p.grid_y), dim3(256), 0, st, a, NT);
  }
  auto kern = a.xtype == B2K_F32 ? w4_kernel<NT, GS, BF, true> : w4_kernel<NT, GS, BF, false>;
  allow_max_dynamic_smem(kern);
  launch_pdl(kern, dim3(p.grid_x, p.grid_y, p.slices), dim3(32 * kW4Warps), (size_t)p.smem, st, a);
}

template <int NT, bool BF> static void w4_dispatch(const W4Args& a, const W4Plan& p, cudaStream_t st) {
  switch (a.w.g) {
    case 32: w4_launch<NT, 4, BF>(a, p, st); break;
    case 64: w4_launch<NT, 2, BF>(a, p, st); break;
    default: w4_launch<NT, 1, BF>(a, p, st); break;
  }
}

template <bool BF> static void w4_columns(const W4Args& a, const W4Plan& p, cudaStream_t st) {
  if (p.nt == 1) w4_dispatch<1, BF>(a, p, st);
  else if (p.nt == 2) w4_dispatch<2, BF>(a, p, st);
  else w4_dispatch<4, BF>(a, p, st);
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

// the product copies all three in bulk
static int w4_check_aligned(const char* what, const void* tiles, const void* scales, const void* zeros) {
  B2K_REQUIRE(aligned16(tiles) && aligned16(scales) && aligned16(zeros),
              "%s: the tiles, their scales and zeros must be 16-byte aligned", what);
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
  if (int st = w4_check_aligned("b2k_w4_pack", tiles, tile_scales, tile_zeros)) return st;
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
  if (int st = w4_check_aligned("b2k_w4_quantize", tiles, tile_scales, tile_zeros)) return st;
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
  // the chunks that the product takes its rows in use it one after another
  const int64_t most = w4_most_rows(xtype == B2K_F32);
  int64_t bytes = 0;
  for (int64_t m : {M < most ? M : most, M % most})
    if (m > 0) {
      const int64_t b = w4_plan(m, N, K, group, xtype == B2K_F32).bytes;
      bytes = b > bytes ? b : bytes;
    }
  return bytes;
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
  if (K > 0)
    if (int st = w4_check_aligned("b2k_w4_matmul", tiles, tile_scales, tile_zeros)) return st;
  B2K_REQUIRE(M <= 1 || (ldx >= K && ldy >= N), "b2k_w4_matmul: row stride smaller than the row");
  const int64_t most = w4_most_rows(xtype == B2K_F32);
  if (M > most) {
    const char* xb = static_cast<const char*>(x);
    char* yb = static_cast<char*>(y);
    for (int64_t m = 0; m < M; m += most)
      if (int st = b2k_w4_matmul(xb + m * ldx * dtype_size(xtype), ldx, xtype, xs ? xs + m * ldxs : xs,
                                 ldxs, xgroup, tiles, tile_scales, tile_zeros, stype, group,
                                 M - m < most ? M - m : most, N, K, yb + m * ldy * dtype_size(ytype), ldy,
                                 ytype, workspace, workspace_bytes, stream))
        return st;
    return B2K_OK;
  }
  W4Args a = {};
  a.w = W4{static_cast<const unsigned char*>(tiles), tile_scales, tile_zeros, N, K, group};
  a.x = x; a.ldx = ldx; a.xs = xs; a.ldxs = ldxs; a.xgroup = xgroup;
  a.y = y; a.ldy = ldy; a.M = M;
  a.xtype = xtype; a.ytype = ytype; a.stype = stype;
  const W4Plan p = w4_plan(M, N, K, group, xtype == B2K_F32);
  B2K_REQUIRE(p.slices <= 65535, "b2k_w4_matmul: shape too large");
  B2K_REQUIRE(p.bytes == 0 || (workspace && workspace_bytes >= p.bytes && aligned16(workspace)),
              "b2k_w4_matmul: the workspace needs %lld bytes, got %lld", (long long)p.bytes,
              (long long)workspace_bytes);
  const int xsize = dtype_size(xtype);
  // eight columns are read as 16-byte vectors (8 bytes for 8-bit x)
  a.x_aligned = reinterpret_cast<uintptr_t>(x) % (xsize == 1 ? 8 : 16) == 0 &&
                ldx * xsize % (xsize == 1 ? 8 : 16) == 0;
  a.kslice = p.kslice; a.rows = p.rows;
  a.stages = p.stages; a.each = p.each; a.more = p.more;
  a.xw = p.prepare ? static_cast<unsigned char*>(workspace) : nullptr;
  a.part = p.slices > 1 ? reinterpret_cast<float*>(static_cast<unsigned char*>(workspace) + p.image)
                        : nullptr;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (stype == B2K_F16) w4_columns<false>(a, p, st);
  else w4_columns<true>(a, p, st);
  if (a.part) {
    const unsigned grid = w4_blocks(M * N);
    B2K_DISPATCH_FLOAT(ytype, {
      launch_pdl(w4_sum_kernel<T>, dim3(grid), dim3(256), 0, st, static_cast<const float*>(a.part),
                 p.slices, static_cast<T*>(y), ldy, M, N);
    });
  }
  return check_launch("b2k_w4_matmul");
}
