// b2k_kv4_write / b2k_kv4_read: keys and values into and out of the 4-bit
// paged cache (kv4.cuh), any set of slots in any order.
//
// One thread holds 8 dimensions of one row (16 bytes in, one 32-bit word of
// nibbles out), g / 8 neighbouring lanes reduce their group's minimum and
// maximum with shuffles.  Rows are taken 16 tokens of one head at a time, so
// that a prefill's writes fill whole micro blocks.  Both are bound by HBM:
// 2 D Hk values of T on one side, Hk (D + 8 D / g) bytes on the other.
#include "kv4.cuh"
#include "rowio.cuh"
#include "tma.cuh"

namespace b2k {

constexpr int kKvThreads = 256;

struct Kv4IoArgs {
  Kv4 c;
  const void *k, *v;      // write: inputs
  void *ko, *vo;          // read: outputs
  const int64_t* slots;
  int64_t T;
  int64_t ldk, hdk, ldv, hdv;  // token and head strides in elements
  int aligned;
};

// unit (16 tokens x one head x keys or values) -> this thread's row and word
struct Kv4Item {
  int64_t token;
  int head, word, is_v;
  bool live;
};

__device__ __forceinline__ Kv4Item kv4_item(const Kv4IoArgs& a) {
  const int W = a.c.D >> 3;  // words per row: 8, 16 or 32
  const int64_t id = (int64_t)blockIdx.x * kKvThreads + threadIdx.x;
  const int64_t row = id / W;
  const int64_t unit = row >> 4;
  Kv4Item it;
  it.word = (int)(id - row * W);
  it.is_v = (int)(unit & 1);
  const int64_t u = unit >> 1;
  const int64_t chunk = u / a.c.Hk;
  it.head = (int)(u - chunk * a.c.Hk);
  it.token = chunk * 16 + (row & 15);
  it.live = it.token < a.T;
  return it;
}

template <typename T> __global__ void __launch_bounds__(kKvThreads) kv4_write_kernel(Kv4IoArgs a) {
  griddep_launch_dependents();
  griddep_wait();
  const Kv4Item it = kv4_item(a);
  const int64_t slot = it.live ? a.slots[it.token] : -1;
  float x[8];
  float lo = INFINITY, hi = -INFINITY;
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = 0.0f;
  if (it.live) {
    const T* src = it.is_v
                       ? static_cast<const T*>(a.v) + it.token * a.ldv + it.head * a.hdv
                       : static_cast<const T*>(a.k) + it.token * a.ldk + it.head * a.hdk;
    load_vec<T, true>(x, src, it.word * 8, a.c.D, a.aligned != 0);
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    x[e] = min_nan(max_nan(x[e], -kKv4Limit), kKv4Limit);
    lo = min_nan(lo, x[e]);
    hi = max_nan(hi, x[e]);
  }
  const int lanes = a.c.g >> 3;
  for (int o = lanes >> 1; o > 0; o >>= 1) {
    lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
  }
  const __half sh = __float2half_rn(__fdiv_rn(hi - lo, 15.0f)), lh = __float2half_rn(lo);
  const float s = __half2float(sh), l = __half2float(lh);
  uint32_t bits = 0;
  if (s > 0.0f) {  // not for a constant group (n = 0), nor a NaN one
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float n = fminf(fmaxf(rintf(__fdiv_rn(x[e] - l, s)), 0.0f), 15.0f);
      bits |= (uint32_t)n << (4 * e);
    }
  }
  // a slot outside the pool (negative: padding) is not written
  if (slot < 0 || slot >= a.c.slots()) return;
  const int64_t page = slot / a.c.P;
  const int tok = (int)(slot - page * a.c.P);
  unsigned char* m = a.c.micro(page, it.head, tok);
  const int rows = 16 * a.c.row_bytes(), pars = 16 * a.c.par_bytes();
  if (it.is_v) m += rows + pars;
  const int w = it.is_v ? it.word : kv4_key_word(it.word, a.c.D);
  reinterpret_cast<uint32_t*>(m + (tok & 15) * a.c.row_bytes())[w] = bits;
  if ((it.word & (lanes - 1)) == 0)
    reinterpret_cast<__half2*>(m + rows + (tok & 15) * a.c.par_bytes())[it.word / lanes] =
        __halves2half2(sh, lh);
}

template <typename T> __global__ void __launch_bounds__(kKvThreads) kv4_read_kernel(Kv4IoArgs a) {
  griddep_launch_dependents();
  griddep_wait();
  const Kv4Item it = kv4_item(a);
  if (!it.live) return;
  const int64_t slot = a.slots[it.token];
  float x[8];
  if (slot < 0 || slot >= a.c.slots()) {
    // padding reads zeros; a slot past the pool is an error and reads NaN
    const float fill = slot < 0 ? 0.0f : __int_as_float(0x7fc00000);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = fill;
  } else {
    const int64_t page = slot / a.c.P;
    const int tok = (int)(slot - page * a.c.P);
    const unsigned char* m = a.c.micro(page, it.head, tok);
    const int rows = 16 * a.c.row_bytes(), pars = 16 * a.c.par_bytes();
    if (it.is_v) m += rows + pars;
    const int w = it.is_v ? it.word : kv4_key_word(it.word, a.c.D);
    const uint32_t bits = reinterpret_cast<const uint32_t*>(m + (tok & 15) * a.c.row_bytes())[w];
    const float2 p = __half22float2(reinterpret_cast<const __half2*>(
        m + rows + (tok & 15) * a.c.par_bytes())[it.word / (a.c.g >> 3)]);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = fmaf((float)((bits >> (4 * e)) & 15u), p.x, p.y);
  }
  T* dst = static_cast<T*>(it.is_v ? a.vo : a.ko) + (it.token * a.c.Hk + it.head) * a.c.D;
  constexpr int E = Traits<T>::E;
  static_assert(E == 8, "16-bit outputs");
  store_vec<T>(dst, it.word * 8, a.c.D, true, x);
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

static int kv4_grid(const Kv4IoArgs& a, const char* what, unsigned* grid) {
  const int64_t rows = (a.T + 15) / 16 * 16 * a.c.Hk * 2;
  const int64_t blocks = (rows * (a.c.D >> 3) + kKvThreads - 1) / kKvThreads;
  B2K_REQUIRE(blocks <= 0x7fffffffLL, "%s: too many tokens (%lld)", what, (long long)a.T);
  *grid = (unsigned)blocks;
  return B2K_OK;
}

}  // namespace b2k

extern "C" int b2k_kv4_write(const void* k, int64_t ldk, int64_t hdk, const void* v, int64_t ldv,
                             int64_t hdv, const int64_t* slots, int64_t T, void* data,
                             int64_t pages, int64_t Hk, int64_t P, int64_t D, int64_t group,
                             int dtype, void* stream) {
  if (int st = kv4_check("b2k_kv4_write", data, pages, Hk, P, D, group)) return st;
  B2K_REQUIRE(T >= 0, "b2k_kv4_write: negative number of tokens");
  B2K_REQUIRE(dtype == B2K_F16 || dtype == B2K_BF16, "b2k_kv4_write: dtype %d is not 16-bit", dtype);
  B2K_REQUIRE(T == 0 || (k && v && slots), "b2k_kv4_write: null k, v or slots");
  if (T == 0 || pages == 0) return B2K_OK;
  Kv4IoArgs a = {};
  a.c = Kv4{static_cast<unsigned char*>(data), pages, (int)Hk, (int)P, (int)D, (int)group};
  a.k = k; a.v = v; a.slots = slots; a.T = T;
  a.ldk = ldk; a.hdk = hdk; a.ldv = ldv; a.hdv = hdv;
  a.aligned = aligned16(k) && aligned16(v) && ldk % 8 == 0 && hdk % 8 == 0 && ldv % 8 == 0 &&
              hdv % 8 == 0;
  unsigned grid;
  if (int st = kv4_grid(a, "b2k_kv4_write", &grid)) return st;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == B2K_F16) launch_pdl(kv4_write_kernel<__half>, dim3(grid), dim3(kKvThreads), 0, st, a);
  else launch_pdl(kv4_write_kernel<__nv_bfloat16>, dim3(grid), dim3(kKvThreads), 0, st, a);
  return check_launch("b2k_kv4_write");
}

extern "C" int b2k_kv4_read(const void* data, int64_t pages, int64_t Hk, int64_t P, int64_t D,
                            int64_t group, const int64_t* slots, int64_t T, void* k, void* v,
                            int dtype, void* stream) {
  if (int st = kv4_check("b2k_kv4_read", data, pages, Hk, P, D, group)) return st;
  B2K_REQUIRE(T >= 0, "b2k_kv4_read: negative number of tokens");
  B2K_REQUIRE(dtype == B2K_F16 || dtype == B2K_BF16, "b2k_kv4_read: dtype %d is not 16-bit", dtype);
  B2K_REQUIRE(T == 0 || (k && v && slots && aligned16(k) && aligned16(v)),
              "b2k_kv4_read: null slots, or k or v null or not 16-byte aligned");
  if (T == 0) return B2K_OK;
  Kv4IoArgs a = {};
  a.c = Kv4{static_cast<unsigned char*>(const_cast<void*>(data)), pages, (int)Hk, (int)P, (int)D,
            (int)group};
  a.ko = k; a.vo = v; a.slots = slots; a.T = T;
  unsigned grid;
  if (int st = kv4_grid(a, "b2k_kv4_read", &grid)) return st;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == B2K_F16) launch_pdl(kv4_read_kernel<__half>, dim3(grid), dim3(kKvThreads), 0, st, a);
  else launch_pdl(kv4_read_kernel<__nv_bfloat16>, dim3(grid), dim3(kKvThreads), 0, st, a);
  return check_launch("b2k_kv4_read");
}
