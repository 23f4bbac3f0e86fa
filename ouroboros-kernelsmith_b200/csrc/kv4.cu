// b2k_kv4_write / b2k_kv4_read: keys and values into and out of the 4-bit
// paged cache (kv4.cuh), any set of slots in any order.
//
// One thread holds 8 dimensions of a row (16 bytes on one side, one 32-bit
// word of nibbles on the other); g / 8 neighbouring lanes reduce their group's
// minimum and maximum with shuffles.  A block takes 16 tokens and kKvHeads
// heads of both keys and values, so every thread has four loads in flight and
// a prefill's writes fill whole micro blocks.  Both are bound by HBM: 2 D Hk
// values of T on one side, Hk (D + 8 D / g) bytes on the other.
#include "kv4.cuh"
#include "rowio.cuh"
#include "tma.cuh"

namespace b2k {

constexpr int kKvHeads = 2;

struct Kv4IoArgs {
  Kv4 c;
  const void *k, *v;      // write: inputs
  void *ko, *vo;          // read: outputs
  const int64_t* slots;
  int64_t T;
  int64_t ldk, hdk, ldv, hdv;  // token and head strides in elements
  int aligned;
};

// where a token's slot lies: micro block of head 0 and row within it
struct Kv4Place {
  unsigned char* micro;
  int row;
  bool in, padding;
};
__device__ __forceinline__ Kv4Place kv4_place(const Kv4IoArgs& a, int64_t slot) {
  Kv4Place p;
  p.padding = slot < 0;
  p.in = slot >= 0 && slot < a.c.slots();
  const int64_t s = p.in ? slot : 0;
  // pools below 2^32 slots (a TB and more) divide in 32 bits
  const int64_t page = (s >> 32) == 0 ? (int64_t)((uint32_t)s / (uint32_t)a.c.P) : s / a.c.P;
  const int tok = (int)(s - page * a.c.P);
  p.micro = a.c.micro(page, 0, tok);
  p.row = tok & 15;
  return p;
}

// d / s rounded to the nearest whole number, ties to even, and clamped to 0 ..
// 15, for s > 0 a float16 and r near 1 / s.  The product d r is off by a few
// 2^-23 of itself, so its nearest whole number n is the quotient's except
// where that is (almost) halfway.  d - n s is exact there (n s has 15 bits)
// and tells: beyond s / 2, or equal to it with n odd, the neighbour is meant.
__device__ __forceinline__ uint32_t kv4_round(float d, float s, float r, float half) {
  constexpr float kShift = 12582912.0f;  // 1.5 * 2^23: adding it rounds to an integer
  const float n = fminf(fmaxf(__fadd_rn(__fadd_rn(d * r, kShift), -kShift), 0.0f), 15.0f);
  const float rest = fmaf(-n, s, d);
  uint32_t q = __float_as_uint(n + 8388608.0f) & 15u;
  if (fabsf(rest) >= half) {
    // at the ends of the range there is no neighbour
    const bool move = fabsf(rest) > half || (q & 1u);
    if (move && rest > 0.0f && q < 15u) ++q;
    if (move && rest < 0.0f && q > 0u) --q;
  }
  return q;
}

template <typename T, int D>
__global__ void __launch_bounds__(2 * D) kv4_write_kernel(const __grid_constant__ Kv4IoArgs a) {
  constexpr int W = D / 8;
  griddep_launch_dependents();
  griddep_wait();
  const int word = threadIdx.x % W;
  const int64_t token = (int64_t)blockIdx.x * 16 + threadIdx.x / W;
  const bool live = token < a.T;
  const int64_t slot = live ? a.slots[token] : -1;
  const int h0 = blockIdx.y * kKvHeads;
  float x[kKvHeads][2][8];
#pragma unroll
  for (int h = 0; h < kKvHeads; ++h)
#pragma unroll
    for (int v = 0; v < 2; ++v) {
      if (live && h0 + h < a.c.Hk) {
        const T* src = v ? static_cast<const T*>(a.v) + token * a.ldv + (h0 + h) * a.hdv
                         : static_cast<const T*>(a.k) + token * a.ldk + (h0 + h) * a.hdk;
        load_vec<T, true>(x[h][v], src, word * 8, D, a.aligned != 0);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[h][v][e] = 0.0f;
      }
    }
  const Kv4Place p = kv4_place(a, slot);
  const int lanes = a.c.g >> 3, rows = 8 * D, half_micro = rows + 16 * a.c.par_bytes();
  const int64_t head_bytes = (int64_t)(a.c.P >> 4) * a.c.micro_bytes();
#pragma unroll
  for (int h = 0; h < kKvHeads; ++h)
#pragma unroll
    for (int v = 0; v < 2; ++v) {
      float* y = x[h][v];
      float lo = INFINITY, hi = -INFINITY;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        y[e] = min_nan(max_nan(y[e], -kKv4Limit), kKv4Limit);
        lo = min_nan(lo, y[e]);
        hi = max_nan(hi, y[e]);
      }
      for (int o = lanes >> 1; o > 0; o >>= 1) {
        lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
      }
      const __half sh = __float2half_rn(__fdiv_rn(hi - lo, 15.0f)), lh = __float2half_rn(lo);
      const float s = __half2float(sh), l = __half2float(lh);
      uint32_t bits = 0;
      if (s > 0.0f) {  // not for a constant group (n = 0), nor a NaN one
        const float r = __frcp_rn(s), half = 0.5f * s;
#pragma unroll
        for (int e = 0; e < 8; ++e) bits |= kv4_round(y[e] - l, s, r, half) << (4 * e);
      }
      // a slot outside the pool (negative: padding) is not written
      if (!p.in || h0 + h >= a.c.Hk) continue;
      unsigned char* m = p.micro + (h0 + h) * head_bytes + v * half_micro;
      reinterpret_cast<uint32_t*>(m + p.row * (D / 2))[v ? word : kv4_key_word(word, D)] = bits;
      if ((word & (lanes - 1)) == 0)
        reinterpret_cast<__half2*>(m + rows + p.row * a.c.par_bytes())[word / lanes] =
            __halves2half2(sh, lh);
    }
}

template <typename T, int D>
__global__ void __launch_bounds__(2 * D) kv4_read_kernel(const __grid_constant__ Kv4IoArgs a) {
  constexpr int W = D / 8;
  static_assert(Traits<T>::E == 8, "16-bit outputs");
  griddep_launch_dependents();
  griddep_wait();
  const int word = threadIdx.x % W;
  const int64_t token = (int64_t)blockIdx.x * 16 + threadIdx.x / W;
  if (token >= a.T) return;
  const Kv4Place p = kv4_place(a, a.slots[token]);
  const int lanes = a.c.g >> 3, rows = 8 * D, half_micro = rows + 16 * a.c.par_bytes();
  const int64_t head_bytes = (int64_t)(a.c.P >> 4) * a.c.micro_bytes();
  const int h0 = blockIdx.y * kKvHeads;
  uint32_t bits[kKvHeads][2];
  __half2 par[kKvHeads][2];
#pragma unroll
  for (int h = 0; h < kKvHeads; ++h)
#pragma unroll
    for (int v = 0; v < 2; ++v)
      if (p.in && h0 + h < a.c.Hk) {
        const unsigned char* m = p.micro + (h0 + h) * head_bytes + v * half_micro;
        bits[h][v] = __ldcs(reinterpret_cast<const uint32_t*>(m + p.row * (D / 2)) +
                            (v ? word : kv4_key_word(word, D)));
        par[h][v] = __ldcs(reinterpret_cast<const __half2*>(m + rows + p.row * a.c.par_bytes()) +
                           word / lanes);
      }
#pragma unroll
  for (int h = 0; h < kKvHeads; ++h)
#pragma unroll
    for (int v = 0; v < 2; ++v) {
      if (h0 + h >= a.c.Hk) continue;
      float x[8];
      if (p.in) {
        // 2^23 + n as a float; (2^23 + n) s - 2^23 s is n s exactly, fused
        const float2 f = __half22float2(par[h][v]);
        const float back = -8388608.0f * f.x;
#pragma unroll
        for (int e = 0; e < 8; ++e)
          x[e] = fmaf(__uint_as_float(((bits[h][v] >> (4 * e)) & 15u) | 0x4b000000u), f.x, back) + f.y;
      } else {
        // padding reads zeros; a slot past the pool is an error and reads NaN
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = p.padding ? 0.0f : __int_as_float(0x7fc00000);
      }
      T* dst = static_cast<T*>(v ? a.vo : a.ko) + (token * a.c.Hk + h0 + h) * D;
      store_vec<T>(dst, word * 8, D, true, x);
    }
}

}  // namespace b2k

using namespace b2k;

namespace b2k {

// geometry shared by the cache's entry points; 0 when it is valid
int kv4_check(const char* what, const void* data, int64_t pages, int64_t Hk, int64_t P, int64_t D,
              int64_t g) {
  B2K_REQUIRE(D == 64 || D == 128 || D == 256, "%s: head dimension %lld is not 64, 128 or 256",
              what, (long long)D);
  B2K_REQUIRE((g == 32 || g == 64 || g == 128) && g <= D,
              "%s: group %lld is not 32, 64 or 128, or above the head dimension", what, (long long)g);
  B2K_REQUIRE(P >= 16 && P % 16 == 0 && P <= 65536, "%s: page size %lld is not a multiple of 16",
              what, (long long)P);
  B2K_REQUIRE(Hk >= 1 && Hk <= 65536, "%s: bad number of heads %lld", what, (long long)Hk);
  B2K_REQUIRE(pages >= 0 && pages <= 0x7fffffffLL, "%s: bad number of pages %lld", what,
              (long long)pages);
  B2K_REQUIRE(pages == 0 || (data && aligned16(data)), "%s: the pool is null or not 16-byte aligned",
              what);
  return B2K_OK;
}

template <typename T> static void kv4_launch(const Kv4IoArgs& a, bool write, cudaStream_t st) {
  const dim3 grid((unsigned)((a.T + 15) / 16), (a.c.Hk + kKvHeads - 1) / kKvHeads);
  auto go = [&](auto w, auto r, int D) { launch_pdl(write ? w : r, grid, dim3(2 * D), 0, st, a); };
  if (a.c.D == 64) go(kv4_write_kernel<T, 64>, kv4_read_kernel<T, 64>, 64);
  else if (a.c.D == 128) go(kv4_write_kernel<T, 128>, kv4_read_kernel<T, 128>, 128);
  else go(kv4_write_kernel<T, 256>, kv4_read_kernel<T, 256>, 256);
}

}  // namespace b2k

extern "C" int b2k_kv4_write(const void* k, int64_t ldk, int64_t hdk, const void* v, int64_t ldv,
                             int64_t hdv, const int64_t* slots, int64_t T, void* data,
                             int64_t pages, int64_t Hk, int64_t P, int64_t D, int64_t group,
                             int dtype, void* stream) {
  if (int st = kv4_check("b2k_kv4_write", data, pages, Hk, P, D, group)) return st;
  B2K_REQUIRE(T >= 0 && T <= (1ll << 34), "b2k_kv4_write: bad number of tokens %lld", (long long)T);
  B2K_REQUIRE(dtype == B2K_F16 || dtype == B2K_BF16, "b2k_kv4_write: dtype %d is not 16-bit", dtype);
  B2K_REQUIRE(T == 0 || (k && v && slots), "b2k_kv4_write: null k, v or slots");
  if (T == 0 || pages == 0) return B2K_OK;
  Kv4IoArgs a = {};
  a.c = Kv4{static_cast<unsigned char*>(data), pages, (int)Hk, (int)P, (int)D, (int)group};
  a.k = k; a.v = v; a.slots = slots; a.T = T;
  a.ldk = ldk; a.hdk = hdk; a.ldv = ldv; a.hdv = hdv;
  a.aligned = aligned16(k) && aligned16(v) && ldk % 8 == 0 && hdk % 8 == 0 && ldv % 8 == 0 &&
              hdv % 8 == 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == B2K_F16) kv4_launch<__half>(a, true, st);
  else kv4_launch<__nv_bfloat16>(a, true, st);
  return check_launch("b2k_kv4_write");
}

extern "C" int b2k_kv4_read(const void* data, int64_t pages, int64_t Hk, int64_t P, int64_t D,
                            int64_t group, const int64_t* slots, int64_t T, void* k, void* v,
                            int dtype, void* stream) {
  if (int st = kv4_check("b2k_kv4_read", data, pages, Hk, P, D, group)) return st;
  B2K_REQUIRE(T >= 0 && T <= (1ll << 34), "b2k_kv4_read: bad number of tokens %lld", (long long)T);
  B2K_REQUIRE(dtype == B2K_F16 || dtype == B2K_BF16, "b2k_kv4_read: dtype %d is not 16-bit", dtype);
  B2K_REQUIRE(T == 0 || (k && v && slots && aligned16(k) && aligned16(v)),
              "b2k_kv4_read: null slots, or k or v null or not 16-byte aligned");
  if (T == 0) return B2K_OK;
  Kv4IoArgs a = {};
  a.c = Kv4{static_cast<unsigned char*>(const_cast<void*>(data)), pages, (int)Hk, (int)P, (int)D,
            (int)group};
  a.ko = k; a.vo = v; a.slots = slots; a.T = T;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == B2K_F16) kv4_launch<__half>(a, false, st);
  else kv4_launch<__nv_bfloat16>(a, false, st);
  return check_launch("b2k_kv4_read");
}
