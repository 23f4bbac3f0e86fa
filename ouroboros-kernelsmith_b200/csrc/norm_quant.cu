// b2k_norm_quant: [residual addition] -> RMS norm -> *w -> 8-bit values with
// fp32 scales, one scale per row or per group of 32 / 64 / 128 columns.
//
//   h = T(x + r)                      (the residual stream, written when asked)
//   y = (h w) rs,   rs = rsqrt(mean(h^2) + eps)
//   a = max |y| over the row / group;  scale = a / Q;  q = round(y Q / a)
//   (Q = 127 for int8, 448 for e4m3; a < 1e-30: scale 0 and q 0)
//
// y is quantised from fp32, as h w times Q / max |h w|: rs drops out of q.
// Multiplying by rs > 0 and rounding are monotone, so max |y| is exactly
// rs * max |h w|: the sum of squares and the row's maximum come out of ONE
// block reduction, and the row is read once.  Bound by HBM: 2 reads and one
// write of T and one byte per element.
#include <cuda_fp8.h>

#include "rowio.cuh"
#include "rowpipe.cuh"

B2K_DEFINE_TIMEOUT_COUNTER()

namespace b2k {

constexpr float kQuantTiny = 1e-30f;

struct NormQuantArgs {
  const void *x, *r, *w;
  void *h, *q;
  float* scale;
  int64_t ldx, ldr, ldh, ldq, lds, M, N;
  int group;  // 0 = one scale per row
  float eps;
  int aligned;
};

// NaN-propagating maximum of magnitudes (fmaxf would drop a NaN).  Between
// lanes and warps it travels as its bit pattern: as an unsigned integer a NaN
// is above infinity, so an integer maximum keeps it as well.
__device__ __forceinline__ float max_mag(float m, float v) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(m), "f"(fabsf(v)));
  return r;
}

// Scale, and multiplier of h w, of a row or group whose largest |h w| is `m`:
// q = round(y Q / a) is round(h w Q / m), without the norm's own rounding (h w
// is exact for 16-bit h and w, which leaves two roundings before the last).
template <bool I8>
__device__ __forceinline__ void quant_scale(float m, float rs, float& scale, float& mul) {
  constexpr float Q = I8 ? 127.0f : 448.0f;
  const float a = m * rs;
  if (a < kQuantTiny) {
    scale = 0.0f;
    mul = 0.0f;
  } else {  // a NaN goes on into scale and values
    scale = __fdiv_rn(a, Q);
    mul = a == a ? __fdiv_rn(Q, m) : a;
  }
}

// E values -> E bytes.  The saturating conversions round to nearest even;
// |v| <= Q up to the roundings of v = h w Q / m.
template <bool I8, int E> __device__ __forceinline__ void quant_pack(const float* v, uint32_t* out) {
#pragma unroll
  for (int k = 0; k < E / 4; ++k) {
    if constexpr (I8) {
      uint32_t b[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        int t;
        asm("cvt.rni.sat.s8.f32 %0, %1;" : "=r"(t) : "f"(v[4 * k + e]));
        b[e] = (uint32_t)t;
      }
      out[k] = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
    } else {
      const uint32_t lo = __nv_cvt_float2_to_fp8x2(f2(v[4 * k], v[4 * k + 1]), __NV_SATFINITE,
                                                   __NV_E4M3);
      const uint32_t hi = __nv_cvt_float2_to_fp8x2(f2(v[4 * k + 2], v[4 * k + 3]), __NV_SATFINITE,
                                                   __NV_E4M3);
      out[k] = lo | (hi << 16);
    }
  }
}

template <bool I8, int E>
__device__ __forceinline__ void quant_store(uint8_t* row, int64_t c, int64_t N, bool aligned,
                                            const float* v) {
  uint32_t b[E / 4];
  quant_pack<I8, E>(v, b);
  if (aligned) {
    if (c < N) {
      if constexpr (E == 8) __stcs(reinterpret_cast<uint2*>(row + c), make_uint2(b[0], b[1]));
      else __stcs(reinterpret_cast<uint32_t*>(row + c), b[0]);
    }
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (c + e < N) row[c + e] = (uint8_t)(b[e >> 2] >> (8 * (e & 3)));
  }
}

// sum of `ss` and maximum of `mx` over the row's thread group, in every
// thread; one round through shared memory for both.  red: 1024 words.
__device__ __forceinline__ void group_sum_max(float& ss, uint32_t& mx, const Group& g, float* red) {
  const int width = g.G < 32 ? g.G : 32;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    if (o < width) {
      ss += __shfl_xor_sync(0xffffffffu, ss, o);
      mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    }
  if (g.G > 32) {
    const int nw = g.G >> 5, w = g.tx >> 5, lane = g.tx & 31;
    float* rs = red + g.ty * 32;
    uint32_t* rm = reinterpret_cast<uint32_t*>(red) + 512 + g.ty * 32;
    if (lane == 0) {
      rs[w] = ss;
      rm[w] = mx;
    }
    __syncthreads();
    ss = lane < nw ? rs[lane] : 0.0f;
    mx = lane < nw ? rm[lane] : 0u;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      ss += __shfl_xor_sync(0xffffffffu, ss, o);
      mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    }
  }
}

// quantises and stores the E values v = h w at column c (vector slot `vec` of
// the row); every lane of the warp calls it.  `width` lanes share a group.
template <bool I8, int E>
__device__ __forceinline__ void quant_slot(const NormQuantArgs& a, int64_t row, int64_t c, float* v,
                                           float rs, float row_mul, int width) {
  float mul = row_mul;
  if (a.group) {
    float mf = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) mf = max_mag(mf, v[e]);
    uint32_t m = __float_as_uint(mf);
    for (int o = width >> 1; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    float scale;
    quant_scale<I8>(__uint_as_float(m), rs, scale, mul);
    if (c < a.N && c % a.group == 0) a.scale[row * a.lds + c / a.group] = scale;
  }
#pragma unroll
  for (int e = 0; e < E; ++e) v[e] *= mul;
  quant_store<I8, E>(static_cast<uint8_t*>(a.q) + row * a.ldq, c, a.N, a.aligned != 0, v);
}

// One thread group per row, the row in registers between its two uses.
template <typename T, bool I8, int V>
__global__ void __launch_bounds__(1024) norm_quant_rows_kernel(NormQuantArgs a) {
  constexpr int E = Traits<T>::E;
  __shared__ float red[1024];
  const Group g;
  const int64_t row0 = (int64_t)blockIdx.x * blockDim.y;
  const int64_t nrows = a.M - row0 < (int64_t)blockDim.y ? a.M - row0 : (int64_t)blockDim.y;
  pdl_rows_prologue(static_cast<const T*>(a.x), a.ldx * (int64_t)sizeof(T), a.r,
                    a.ldr * (int64_t)sizeof(T), row0, nrows, (uint32_t)(a.N * sizeof(T)),
                    a.aligned != 0);
  const int64_t row = row0 + g.ty;
  const bool live = row < a.M;
  const bool al = a.aligned != 0;
  const T* xr = static_cast<const T*>(a.x) + row * a.ldx;
  const T* rr = static_cast<const T*>(a.r) + row * a.ldr;
  T* hr = static_cast<T*>(a.h) + row * a.ldh;
  float v[V][E];
  float ss = 0.0f;
  float top = 0.0f;
#pragma unroll
  for (int k = 0; k < V; ++k) {
    const int64_t c = ((int64_t)k * g.G + g.tx) * E;
    if (live) load_vec<T, true>(v[k], xr, c, a.N, al);
    else
#pragma unroll
      for (int e = 0; e < E; ++e) v[k][e] = 0.0f;
    if (a.r && live) {
      float r[E];
      load_vec<T, true>(r, rr, c, a.N, al);
#pragma unroll
      for (int e = 0; e < E; ++e) v[k][e] = round_to<T>(v[k][e] + r[e]);
      if (a.h) store_vec<T>(hr, c, a.N, al, v[k]);
    }
    float w[E];
    load_vec<T, false>(w, static_cast<const T*>(a.w), c, a.N, al);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      ss = fmaf(v[k][e], v[k][e], ss);
      v[k][e] *= w[e];
      top = max_mag(top, v[k][e]);
    }
  }
  uint32_t mx = __float_as_uint(top);
  group_sum_max(ss, mx, g, red);
  const float rs = rsqrtf(ss / (float)a.N + a.eps);
  float mul = 0.0f;
  if (!a.group) {
    float scale;
    quant_scale<I8>(__uint_as_float(mx), rs, scale, mul);
    if (live && g.tx == 0) a.scale[row * a.lds] = scale;
  }
  const int lanes = a.group / E;
  const int width = lanes < g.G ? lanes : g.G;
#pragma unroll
  for (int k = 0; k < V; ++k) {
    const int64_t c = ((int64_t)k * g.G + g.tx) * E;
    quant_slot<I8, E>(a, row, live ? c : a.N, v[k], rs, mul, width);
  }
}

// Rows beyond the register budget: one block per row, the row read twice
// (the second time through L2).
template <typename T, bool I8>
__global__ void __launch_bounds__(1024) norm_quant_stream_kernel(NormQuantArgs a) {
  constexpr int E = Traits<T>::E;
  __shared__ float red[1024];
  const Group g;
  griddep_launch_dependents();
  griddep_wait();
  const int64_t row = blockIdx.x;
  const bool al = a.aligned != 0;
  const T* xr = static_cast<const T*>(a.x) + row * a.ldx;
  const T* rr = static_cast<const T*>(a.r) + row * a.ldr;
  const T* wr = static_cast<const T*>(a.w);
  T* hr = static_cast<T*>(a.h) + row * a.ldh;
  float ss = 0.0f, top = 0.0f;
  auto load = [&](float* v, int64_t c, bool first) {
    load_vec<T, false>(v, xr, c, a.N, al);
    if (a.r) {
      float r[E];
      load_vec<T, false>(r, rr, c, a.N, al);
#pragma unroll
      for (int e = 0; e < E; ++e) v[e] = round_to<T>(v[e] + r[e]);
      if (first && a.h) store_vec<T>(hr, c, a.N, al, v);
    }
  };
  for (int64_t c = (int64_t)g.tx * E; c < a.N; c += (int64_t)g.G * E) {
    float v[E], w[E];
    load(v, c, true);
    load_vec<T, false>(w, wr, c, a.N, al);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      ss = fmaf(v[e], v[e], ss);
      top = max_mag(top, v[e] * w[e]);
    }
  }
  uint32_t mx = __float_as_uint(top);
  group_sum_max(ss, mx, g, red);
  const float rs = rsqrtf(ss / (float)a.N + a.eps);
  float mul = 0.0f;
  if (!a.group) {
    float scale;
    quant_scale<I8>(__uint_as_float(mx), rs, scale, mul);
    if (g.tx == 0) a.scale[row * a.lds] = scale;
  }
  // whole warps stay in the loop: a group's lanes reduce together
  const int64_t end = (a.N + 32 * E - 1) / (32 * E) * (32 * E);
  for (int64_t c = (int64_t)g.tx * E; c < end; c += (int64_t)g.G * E) {
    float v[E], w[E];
    load(v, c, false);
    load_vec<T, false>(w, wr, c, a.N, al);
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] *= w[e];
    quant_slot<I8, E>(a, row, c, v, rs, mul, a.group / E);
  }
}

// Many aligned rows: persistent blocks on the bulk-copy row pipeline, the
// weights in registers for all of a block's rows.  One block barrier per row:
// the warps' partial results alternate between two buffers, and every thread
// sums them itself.
template <typename T, bool I8, bool RESID, bool GROUPED, int V, int THREADS>
__global__ void __launch_bounds__(THREADS) norm_quant_pipe_kernel(const __grid_constant__ NormQuantArgs a,
                                                              const int S) {
  constexpr int E = Traits<T>::E, H = E / 2, NIN = RESID ? 2 : 1;
  extern __shared__ __align__(128) unsigned char dsm[];
  __shared__ float2 part[2][THREADS / 32];
  __shared__ volatile int abort_flag;
  const int tx = threadIdx.x, G = blockDim.x, N = (int)a.N, lane = tx & 31, nw = G >> 5;
  if (tx == 0) abort_flag = 0;
  griddep_launch_dependents();
  const void* srcs[2] = {a.x, a.r};
  const int64_t lds[2] = {a.ldx, a.ldr};
  RowPipe<NIN>::prefetch_l2(srcs, lds, (int)sizeof(T), (uint32_t)N * (uint32_t)sizeof(T), a.M, 1);
  griddep_wait();
  RowPipe<NIN> pipe;
  pipe.init(dsm, S, a.M, (uint32_t)N * (uint32_t)sizeof(T), srcs, lds, (int)sizeof(T));
  uint4 wraw[V];
#pragma unroll
  for (int k = 0; k < V; ++k) {
    const int c = (k * G + tx) * E;
    wraw[k] = c < N ? ld_keep(static_cast<const T*>(a.w) + c) : zero4();
  }
  const int width = a.group / E, gshift = a.group ? __ffs(a.group) - 1 : 0;
  int64_t n = 0;
  for (; n < pipe.nrows; ++n) {
    bool ok;
    const T* xs = reinterpret_cast<const T*>(pipe.wait_next(ok));
    if (!ok) {
      abort_flag = 1;  // every thread leaves after the reduction
      atomicAdd(&b2k_tu_timeouts, 1u);
    }
    const int64_t row = pipe.row_of(n);
    T* hrow = static_cast<T*>(a.h) + row * a.ldh;
    float2 v[V][H], ss2 = f2s(0.0f);
    float top = 0.0f;
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const int c = (k * G + tx) * E;
      if (c < N) {
        unpack2<T>(*reinterpret_cast<const uint4*>(xs + c), v[k]);
        if constexpr (RESID) {
          float2 t[H];
          unpack2<T>(*reinterpret_cast<const uint4*>(xs + N + c), t);
#pragma unroll
          for (int j = 0; j < H; ++j) v[k][j] = add2(v[k][j], t[j]);
          const uint4 h = pack2<T>(v[k]);
          st_stream(hrow + c, h);
          unpack2<T>(h, v[k]);  // the stream as it is stored
        }
        float2 w[H];
        unpack2<T>(wraw[k], w);
#pragma unroll
        for (int j = 0; j < H; ++j) {
          ss2 = fma2(v[k][j], v[k][j], ss2);
          v[k][j] = mul2(v[k][j], w[j]);
          if constexpr (!GROUPED) top = max_mag(max_mag(top, v[k][j].x), v[k][j].y);
        }
      } else {
#pragma unroll
        for (int j = 0; j < H; ++j) v[k][j] = f2s(0.0f);
      }
    }
    float ss = ss2.x + ss2.y;
    uint32_t mx = __float_as_uint(top);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      ss += __shfl_xor_sync(0xffffffffu, ss, o);
      if constexpr (!GROUPED) mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    }
    if (lane == 0) part[n & 1][tx >> 5] = make_float2(ss, __uint_as_float(mx));
    __syncthreads();  // also: every thread has read the stage
    if (abort_flag) break;
    pipe.refill();
    ss = 0.0f;
    mx = 0;
    for (int w = 0; w < nw; ++w) {
      const float2 t = part[n & 1][w];
      ss += t.x;
      if constexpr (!GROUPED) mx = max(mx, __float_as_uint(t.y));
    }
    const float rs = rsqrtf(ss / (float)N + a.eps);
    float mul = 0.0f, scale;
    if constexpr (!GROUPED) {
      quant_scale<I8>(__uint_as_float(mx), rs, scale, mul);
      if (tx == 0) a.scale[row * a.lds] = scale;
    }
    uint8_t* qrow = static_cast<uint8_t*>(a.q) + row * a.ldq;
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const int c = (k * G + tx) * E;
      if constexpr (GROUPED) {
        float m = 0.0f;
#pragma unroll
        for (int j = 0; j < H; ++j) m = max_mag(max_mag(m, v[k][j].x), v[k][j].y);
        uint32_t mb = __float_as_uint(m);
        for (int o = width >> 1; o > 0; o >>= 1) mb = max(mb, __shfl_xor_sync(0xffffffffu, mb, o));
        quant_scale<I8>(__uint_as_float(mb), rs, scale, mul);
        if (c < N && (c & (a.group - 1)) == 0) a.scale[row * a.lds + (c >> gshift)] = scale;
      }
      const float2 f = f2s(mul);
#pragma unroll
      for (int j = 0; j < H; ++j) v[k][j] = mul2(v[k][j], f);
      quant_store<I8, E>(qrow, c, N, true, reinterpret_cast<const float*>(v[k]));
    }
  }
  pipe.drain(n);
}

template <typename T, bool I8, bool RESID, bool GROUPED>
static bool norm_quant_try_pipe(const NormQuantArgs& a, cudaStream_t st) {
  constexpr int E = Traits<T>::E, NIN = RESID ? 2 : 1;
  const int64_t nvec = a.N / E, row_bytes = a.N * (int64_t)sizeof(T);
  if (!a.aligned || (RESID && !a.h) || nvec < 256 || a.M < sm_count()) return false;
  // Two vectors per thread up to 256 threads, then four (16381 x 8192 bf16:
  // 199 us with two, 148 with four; 8192 x 4096 fp16 with its reading back: 61
  // and 62).  Compiled for 768 threads a kernel has at most 80 registers: more
  // resident blocks (16000 x 4096 bf16 79 against 84 us, 4000 x 8192 fp32 73
  // against 81), but four 16-bit vectors spill (16381 x 8192 179 us), so those
  // are compiled for 512 where that is enough.
  const int V = nvec <= 512 ? 2 : 4, G = (int)((nvec + 32 * V - 1) / (32 * V)) * 32;
  if (G > 768) return false;
  auto kern = V == 2                ? norm_quant_pipe_kernel<T, I8, RESID, GROUPED, 2, 768>
              : E == 8 && G <= 512 ? norm_quant_pipe_kernel<T, I8, RESID, GROUPED, 4, E == 8 ? 512 : 768>
                                   : norm_quant_pipe_kernel<T, I8, RESID, GROUPED, 4, 768>;
  PipeShape ps;
  if (!choose_pipe_shape(kern, G, NIN * row_bytes, 0, 2, &ps)) return false;
  int64_t grid = (int64_t)sm_count() * ps.cps;
  if (a.M < grid) return false;  // a row per block at most: no pipeline to keep
  launch_pdl(kern, dim3((unsigned)grid), dim3(G), RowPipe<NIN>::smem_bytes(ps.S, row_bytes), st, a, ps.S);
  return true;
}

template <typename T, bool I8> static int norm_quant_launch(const NormQuantArgs& a, cudaStream_t st) {
  constexpr int E = Traits<T>::E;
  const bool piped = a.r ? (a.group ? norm_quant_try_pipe<T, I8, true, true>(a, st)
                                    : norm_quant_try_pipe<T, I8, true, false>(a, st))
                         : (a.group ? norm_quant_try_pipe<T, I8, false, true>(a, st)
                                    : norm_quant_try_pipe<T, I8, false, false>(a, st));
  if (piped) return check_launch("b2k_norm_quant");
  RowCfg cfg;
  // few rows: as many threads as a row has vectors, for the latency (300 x 4096
  // bf16 4.4 us with 512 threads a row, 6.5 with 128; 4 rows to int8 and back 4.6
  // and 7.4)
  if (!choose_row_cfg(a.N, E, a.M < 8 * sm_count() ? 512 : 128, &cfg, 4, 512)) {
    launch_pdl(norm_quant_stream_kernel<T, I8>, dim3((unsigned)a.M), dim3(1024), 0, st, a);
    return check_launch("b2k_norm_quant");
  }
  const dim3 block(cfg.G, cfg.R);
  const dim3 grid((unsigned)((a.M + cfg.R - 1) / cfg.R));
  switch (cfg.V) {
    case 1: launch_pdl(norm_quant_rows_kernel<T, I8, 1>, grid, block, 0, st, a); break;
    case 2: launch_pdl(norm_quant_rows_kernel<T, I8, 2>, grid, block, 0, st, a); break;
    default: launch_pdl(norm_quant_rows_kernel<T, I8, 4>, grid, block, 0, st, a); break;
  }
  return check_launch("b2k_norm_quant");
}

}  // namespace b2k

using namespace b2k;

extern "C" int b2k_norm_quant(const void* x, int64_t ldx, const void* r, int64_t ldr, const void* w,
                              void* h, int64_t ldh, void* q, int64_t ldq, float* scale, int64_t lds,
                              int64_t M, int64_t N, int dtype, int qtype, int group, float eps,
                              void* stream) {
  B2K_REQUIRE(M >= 0 && N >= 0, "b2k_norm_quant: negative shape M=%lld N=%lld", (long long)M,
              (long long)N);
  B2K_REQUIRE(qtype == B2K_I8 || qtype == B2K_E4M3, "b2k_norm_quant: bad qtype %d", qtype);
  B2K_REQUIRE(group == 0 || group == 32 || group == 64 || group == 128,
              "b2k_norm_quant: group %d is not 0, 32, 64 or 128", group);
  B2K_REQUIRE(dtype_size(dtype) >= 2 && dtype_size(dtype) <= 4, "b2k_norm_quant: bad dtype %d", dtype);
  const int64_t nscales = group ? (N + group - 1) / group : 1;
  B2K_REQUIRE(M == 0 || N == 0 || (x && w && q && scale), "b2k_norm_quant: null x, w, q or scale");
  B2K_REQUIRE(!h || r, "b2k_norm_quant: h is the sum with a residual, which is missing");
  B2K_REQUIRE(M <= 1 || (ldx >= N && ldq >= N && lds >= nscales && (!r || ldr >= N) &&
                         (!h || ldh >= N)),
              "b2k_norm_quant: row stride smaller than the row");
  B2K_REQUIRE(N <= ((int64_t)1 << 30) && M <= 0x7fffffffLL, "b2k_norm_quant: shape too large");
  if (M == 0 || N == 0) return B2K_OK;
  NormQuantArgs a;
  a.x = x; a.r = r; a.w = w; a.h = h; a.q = q; a.scale = scale;
  a.ldx = ldx; a.ldr = ldr; a.ldh = ldh; a.ldq = ldq; a.lds = lds;
  a.M = M; a.N = N; a.group = group; a.eps = eps;
  const int es = dtype_size(dtype), E = 16 / es;
  bool al = N % E == 0 && aligned16(x) && aligned16(w) && (ldx * es) % 16 == 0 &&
            reinterpret_cast<uintptr_t>(q) % E == 0 && ldq % E == 0;
  if (r) al = al && aligned16(r) && (ldr * es) % 16 == 0;
  if (h) al = al && aligned16(h) && (ldh * es) % 16 == 0;
  a.aligned = al ? 1 : 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  B2K_DISPATCH_FLOAT(dtype, {
    return qtype == B2K_I8 ? norm_quant_launch<T, true>(a, st) : norm_quant_launch<T, false>(a, st);
  });
  return B2K_OK;
}
