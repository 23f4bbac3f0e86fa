// b2k_kv4_write / b2k_kv4_read: keys and values into and out of the 4-bit
// paged cache (kv4.cuh), any set of slots in any order.
//
// One thread holds 8 dimensions of a row (16 bytes on one side, one 32-bit
// word of nibbles on the other) of several heads in turn; g / 8 neighbouring
// lanes reduce their group's minimum and maximum with shuffles.  A block takes
// a few tokens, keys and values.  Both are bound by HBM: 2 D Hk values of T on
// one side, Hk (D + 8 D / g) bytes on the other.  Close to that the
// instructions per element count too, hence the packed 16-bit and fp32
// arithmetic below: 30011 tokens of 8 heads of 128 (fp16, g 32) take 76 us to
// write and to read back (30 us of it the reading), whose bytes take 49 us at
// the copy bandwidth; the write issues in 77 % of its cycles.
#include "kv4.cuh"
#include "rowio.cuh"
#include "tma.cuh"

namespace b2k {

// Heads of a thread.  A read has all of its in flight at once; a write takes
// kAhead at a time, as its arithmetic wants the registers.
constexpr int kReadHeads = 4, kAhead = 2;
constexpr int kTokens = 4;  // of a block (30011 tokens written and read back: 76 us, 78 with 8)

struct Kv4IoArgs {
  Kv4 c;
  FastDiv dP;
  const void *k, *v;      // write: inputs
  void *ko, *vo;          // read: outputs
  const int64_t* slots;
  int64_t T;
  int64_t ldk, hdk, ldv, hdv;  // token and head strides in elements
  int aligned;
  int heads;  // of a block
};

// this thread's row: its token, keys or values, and where the token's slot
// lies in the pool
struct Kv4Row {
  int64_t token;
  int word, is_v, head;  // first of its heads
  bool live, in, padding;
  unsigned char *bits, *par;  // of head 0: the row's words, its parameters
};
template <int D> __device__ __forceinline__ Kv4Row kv4_row(const Kv4IoArgs& a, int heads) {
  constexpr int W = D / 8;
  Kv4Row p;
  p.word = threadIdx.x % W;
  p.token = (int64_t)blockIdx.x * kTokens + threadIdx.x / W;
  p.is_v = threadIdx.y;
  p.head = blockIdx.y * heads;
  p.live = p.token < a.T;
  const int64_t slot = p.live ? a.slots[p.token] : -1;
  p.padding = slot < 0;
  p.in = slot >= 0 && slot < a.c.slots();
  const int64_t s = p.in ? slot : 0;
  const int64_t page = a.c.slots() < (1ll << 31) ? (int64_t)a.dP.div((int)s) : s / a.c.P;
  const int tok = (int)(s - page * a.c.P), row = tok & 15, pars = a.c.par_bytes();
  unsigned char* m = a.c.micro(page, p.head, tok) + p.is_v * (8 * D + 16 * pars);
  p.bits = m + row * (D / 2) + 4 * (p.is_v ? p.word : kv4_key_word(p.word, D));
  p.par = m + 8 * D + row * pars + 4 * (p.word / (a.c.g >> 3));
  return p;
}

template <typename T> struct Pair16;
template <> struct Pair16<__half> {
  using type = __half2;
  static __device__ __forceinline__ float2 f(__half2 v) { return __half22float2(v); }
  static __device__ __forceinline__ __half low(__half2 v) { return __low2half(v); }
  static __device__ __forceinline__ __half high(__half2 v) { return __high2half(v); }
  static __device__ __forceinline__ __half2 pair(__half a, __half b) { return __halves2half2(a, b); }
};
template <> struct Pair16<__nv_bfloat16> {
  using type = __nv_bfloat162;
  static __device__ __forceinline__ float2 f(__nv_bfloat162 v) { return __bfloat1622float2(v); }
  static __device__ __forceinline__ __nv_bfloat16 low(__nv_bfloat162 v) { return __low2bfloat16(v); }
  static __device__ __forceinline__ __nv_bfloat16 high(__nv_bfloat162 v) { return __high2bfloat16(v); }
  static __device__ __forceinline__ __nv_bfloat162 pair(__nv_bfloat16 a, __nv_bfloat16 b) {
    return __halves2bfloat162(a, b);
  }
};

// n = clamp(rint(d / s), 0, 15) of eight values, as nibbles, for s > 0 a
// float16.  The product with 1 / s and its rounding give n exactly except
// where the quotient is (almost) halfway between two integers (the product is
// off by 2^-22 of itself, 3e-6 at most) or outside the range (where lo was
// rounded by more than s / 2).  d - n s, whose terms fit fp32 (n s has 15
// bits), tells whether any of the eight is that near; then its comparison with
// s / 2 decides, ties to even.
__device__ __forceinline__ uint32_t kv4_round8(const float2* x, float lo, float s) {
  constexpr float kShift = 12582912.0f;      // 1.5 * 2^23: adding it rounds to an integer
  constexpr uint32_t kBits = 0x4b400000u;    // its bits; the integer lies in the low ones
  const float r = rcp_approx(s), half = 0.5f * s, safe = half * (1.0f - 1e-5f);
  uint32_t bits = 0, all = 0;
  bool near = false;
#pragma unroll
  for (int e = 3; e >= 0; --e) {
    const float2 d = add2(x[e], f2s(-lo));
    const float2 t = fma2(d, f2s(r), f2s(kShift));
    const float2 rest = fma2(sub2(f2s(kShift), t), f2s(s), d);
    near |= fabsf(rest.x) >= safe;
    near |= fabsf(rest.y) >= safe;
    const uint32_t a = __float_as_uint(t.x), b = __float_as_uint(t.y);
    bits = bits * 256u + b * 16u + a;
    all |= (a ^ kBits) | (b ^ kBits);
  }
  bits -= kBits * 0x11111111u;
  if (near || all > 15u) {
    bits = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float d = (e & 1 ? x[e >> 1].y : x[e >> 1].x) - lo;
      const float n = fminf(fmaxf(rintf(d * r), 0.0f), 15.0f), rest = fmaf(-n, s, d);
      uint32_t q = (uint32_t)n;
      if (fabsf(rest) > half || (fabsf(rest) == half && (q & 1u)))
        q = rest > 0.0f ? min(q + 1u, 15u) : q - (q > 0u ? 1u : 0u);
      bits |= q << (4 * e);
    }
  }
  return bits;
}

// f16(d / 15) with the division rounded to fp32 first.  The product with 1 / 15
// is within 2 units of the quotient's last place, which float16 drops with 12
// others: only near a tie of that rounding, or among subnormals, does the
// division have to be made.
__device__ __forceinline__ __half kv4_step(float d) {
  float t = d * (1.0f / 15.0f);
  const uint32_t low = __float_as_uint(t) & 0x1fffu;
  if (low - 0xffcu <= 8u || !(t >= 1.2207031e-4f)) t = __fdiv_rn(d, 15.0f);
  return __float2half_rn(t);
}

template <typename T, int D, int LANES>
__global__ void __launch_bounds__(kTokens * D / 4, 5 * 1024 / (kTokens * D)) kv4_write_kernel(const __grid_constant__ Kv4IoArgs a) {
  using P = Pair16<T>;
  griddep_launch_dependents();
  griddep_wait();
  Kv4Row p = kv4_row<D>(a, a.heads);
  const int heads = min(a.heads, a.c.Hk - p.head);  // of this block
  const int64_t hd = p.is_v ? a.hdv : a.hdk;
  const T* src = (p.is_v ? static_cast<const T*>(a.v) + p.token * a.ldv
                         : static_cast<const T*>(a.k) + p.token * a.ldk) + p.head * hd + p.word * 8;
  const int64_t head_bytes = (int64_t)(a.c.P >> 4) * a.c.micro_bytes();
  auto load = [&](int h) {
    if (!p.live || h >= heads) return zero4();
    const T* from = src + h * hd;
    if (a.aligned) return ld_stream(from);
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = ld1(from + e);
    return pack<T>(x);
  };
  uint4 raw[kAhead];
#pragma unroll
  for (int i = 0; i < kAhead; ++i) raw[i] = load(i);
  auto one = [&](const uint4& row) {
    // minimum and minus maximum of the group, as a pair
    const typename P::type* w = reinterpret_cast<const typename P::type*>(&row);
    const typename P::type mn = __hmin2_nan(__hmin2_nan(w[0], w[1]), __hmin2_nan(w[2], w[3]));
    const typename P::type mx = __hmax2_nan(__hmax2_nan(w[0], w[1]), __hmax2_nan(w[2], w[3]));
    typename P::type ends = P::pair(__hmin_nan(P::low(mn), P::high(mn)),
                                    __hneg(__hmax_nan(P::low(mx), P::high(mx))));
#pragma unroll
    for (int o = LANES >> 1; o > 0; o >>= 1) {
      uint32_t t = __shfl_xor_sync(0xffffffffu, *reinterpret_cast<uint32_t*>(&ends), o);
      ends = __hmin2_nan(ends, *reinterpret_cast<typename P::type*>(&t));
    }
    const float2 f = P::f(ends);
    float lo = f.x, hi = -f.y;
    float2 x[4];
    unpack2<T>(row, x);
    if (!(lo >= -kKv4Limit && hi <= kKv4Limit)) {  // beyond the range, or a NaN
      lo = min_nan(max_nan(lo, -kKv4Limit), kKv4Limit);
      hi = min_nan(max_nan(hi, -kKv4Limit), kKv4Limit);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[e].x = min_nan(max_nan(x[e].x, -kKv4Limit), kKv4Limit);
        x[e].y = min_nan(max_nan(x[e].y, -kKv4Limit), kKv4Limit);
      }
    }
    const __half sh = kv4_step(hi - lo), lh = __float2half_rn(lo);
    const float s = __half2float(sh);
    // a constant group has n = 0, and so has a NaN one
    const uint32_t bits = s > 0.0f ? kv4_round8(x, __half2float(lh), s) : 0u;
    // a slot outside the pool (negative: padding) is not written
    if (p.in) {
      *reinterpret_cast<uint32_t*>(p.bits) = bits;
      if ((p.word & (LANES - 1)) == 0) *reinterpret_cast<__half2*>(p.par) = __halves2half2(sh, lh);
    }
    p.bits += head_bytes;
    p.par += head_bytes;
  };
  for (int h = 0; h < heads; h += kAhead)
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
      if (h + i < heads) {
        const uint4 row = raw[i];
        raw[i] = load(h + i + kAhead);
        one(row);
      }
}

template <typename T, int D>
__global__ void __launch_bounds__(kTokens * D / 4) kv4_read_kernel(const __grid_constant__ Kv4IoArgs a) {
  static_assert(Traits<T>::E == 8, "16-bit outputs");
  griddep_launch_dependents();
  griddep_wait();
  const Kv4Row p = kv4_row<D>(a, kReadHeads);
  if (!p.live) return;
  const int64_t head_bytes = (int64_t)(a.c.P >> 4) * a.c.micro_bytes();
  uint32_t bits[kReadHeads];
  __half2 par[kReadHeads];
#pragma unroll
  for (int h = 0; h < kReadHeads; ++h)
    if (p.in && p.head + h < a.c.Hk) {
      bits[h] = __ldcs(reinterpret_cast<const uint32_t*>(p.bits + h * head_bytes));
      par[h] = __ldcs(reinterpret_cast<const __half2*>(p.par + h * head_bytes));
    }
  T* dst = static_cast<T*>(p.is_v ? a.vo : a.ko) + (p.token * a.c.Hk + p.head) * D + p.word * 8;
#pragma unroll
  for (int h = 0; h < kReadHeads; ++h) {
    if (p.head + h >= a.c.Hk) continue;
    uint4 out;
    uint32_t* w = &out.x;
    if (p.in) {
      // pairs (i, i + 4) as 1024 + n, the integers exactly after that is taken
      const uint32_t b = bits[h], magic = 0x64006400u;
      const __half2 m1024 = __float2half2_rn(-1024.0f), m64 = __float2half2_rn(-64.0f),
                    sixteenth = __float2half2_rn(0.0625f);
      auto h2 = [](uint32_t v) { return *reinterpret_cast<__half2*>(&v); };
      __half2 n[4] = {__hadd2(h2((b & 0x000f000fu) | magic), m1024),
                      __hfma2(h2((b & 0x00f000f0u) | magic), sixteenth, m64),
                      __hadd2(h2(((b >> 8) & 0x000f000fu) | magic), m1024),
                      __hfma2(h2(((b >> 8) & 0x00f000f0u) | magic), sixteenth, m64)};
      if constexpr (std::is_same<T, __half>::value) {
        // lo + n s with one rounding, then back into order
        const __half2 s = __low2half2(par[h]), l = __high2half2(par[h]);
        uint32_t v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const __half2 t = __hfma2(n[e], s, l);
          v[e] = *reinterpret_cast<const uint32_t*>(&t);
        }
        w[0] = __byte_perm(v[0], v[1], 0x5410);
        w[1] = __byte_perm(v[2], v[3], 0x5410);
        w[2] = __byte_perm(v[0], v[1], 0x7632);
        w[3] = __byte_perm(v[2], v[3], 0x7632);
      } else {
        const float2 f = __half22float2(par[h]);
        float x[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 t = __half22float2(n[e]);
          x[e] = fmaf(t.x, f.x, f.y);
          x[e + 4] = fmaf(t.y, f.x, f.y);
        }
        out = pack<T>(x);
      }
    } else {
      // padding reads zeros; a slot past the pool is an error and reads NaN
      const uint32_t fill = p.padding ? 0u : std::is_same<T, __half>::value ? 0x7e007e00u : 0x7fc07fc0u;
      out = make_uint4(fill, fill, fill, fill);
    }
    st_stream(dst + h * D, out);
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

template <typename T, int D> static void kv4_launch_d(Kv4IoArgs a, bool write, cudaStream_t st) {
  const int64_t chunks = (a.T + kTokens - 1) / kTokens;
  a.heads = kReadHeads;
  if (write) {
    // a thread's own costs (its slot, its place) are those of several heads: as
    // many of them as leave six blocks per SM (30011 tokens written and read
    // back: 89 us with two heads a thread, 78 with all eight; 64 tokens take
    // two)
    for (a.heads = a.c.Hk; a.heads > 2 && chunks * ((a.c.Hk + a.heads - 1) / a.heads) < 6 * sm_count();)
      a.heads = (a.heads + 1) / 2;
  }
  const dim3 grid((unsigned)chunks, (a.c.Hk + a.heads - 1) / a.heads), block(kTokens * D / 8, 2);
  if (!write) launch_pdl(kv4_read_kernel<T, D>, grid, block, 0, st, a);
  else if (a.c.g == 32) launch_pdl(kv4_write_kernel<T, D, 4>, grid, block, 0, st, a);
  else if (a.c.g == 64) launch_pdl(kv4_write_kernel<T, D, 8>, grid, block, 0, st, a);
  else if constexpr (D >= 128) launch_pdl(kv4_write_kernel<T, D, 16>, grid, block, 0, st, a);
}
template <typename T> static void kv4_launch(const Kv4IoArgs& a, bool write, cudaStream_t st) {
  if (a.c.D == 64) kv4_launch_d<T, 64>(a, write, st);
  else if (a.c.D == 128) kv4_launch_d<T, 128>(a, write, st);
  else kv4_launch_d<T, 256>(a, write, st);
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
  a.dP = fast_div(P);
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
  a.dP = fast_div(P);
  a.ko = k; a.vo = v; a.slots = slots; a.T = T;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == B2K_F16) kv4_launch<__half>(a, false, st);
  else kv4_launch<__nv_bfloat16>(a, false, st);
  return check_launch("b2k_kv4_read");
}
