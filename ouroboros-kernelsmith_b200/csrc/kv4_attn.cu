// b2k_kv4_attention: attention of new queries over the 4-bit paged cache
// (kv4.cuh).
//
//   o_i = sum_j p_ij v_j / sum_j p_ij,   p_ij = exp(scale q_i . k_j - m_i)
//   over j <= len - Sq + i (causal) or j < len; a row that sees nothing is 0.
//
// One warp per query row; each lane holds D / 32 dimensions of the query and
// of the output; the running maximum and sum of the softmax, and the output,
// are fp32.
#include "kv4.cuh"
#include "rowio.cuh"
#include "tma.cuh"

namespace b2k {

struct Kv4AttnArgs {
  Kv4 c;
  const void* q;
  void* o;
  float* lse;
  const int32_t *table, *lens;
  int64_t B, Sq, H, width;
  int64_t qb, qs, qh;  // strides of q in elements (batch, token, head)
  float scale;
  int causal;
};

template <typename T, int D> __global__ void __launch_bounds__(128) kv4_attn_simple(Kv4AttnArgs a) {
  constexpr int N = D / 32;  // dimensions per lane: lane + 32 n
  griddep_launch_dependents();
  griddep_wait();
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (row >= a.B * a.Sq * a.H) return;
  const int64_t b = row / (a.Sq * a.H), i = row / a.H % a.Sq, h = row % a.H;
  const int hk = (int)(h / (a.H / a.c.Hk));
  const int64_t cap = a.width * a.c.P;
  const int64_t given = a.lens[b];
  const int64_t len = min(max(given, (int64_t)0), cap);
  const int64_t end = a.causal ? len - a.Sq + i + 1 : len;
  const T* qr = static_cast<const T*>(a.q) + b * a.qb + i * a.qs + h * a.qh;
  float q[N], acc[N];
#pragma unroll
  for (int n = 0; n < N; ++n) {
    q[n] = ld1(qr + lane + 32 * n) * a.scale;
    acc[n] = 0.0f;
  }
  float m = -INFINITY, l = 0.0f;
  bool bad = given > cap;
  const int rows = 16 * a.c.row_bytes(), pars = 16 * a.c.par_bytes();
  for (int64_t j = 0; j < end; ++j) {
    const int page = a.table[b * a.width + j / a.c.P];
    if (page < 0 || page >= a.c.pages) {
      bad = true;
      break;
    }
    const int t = (int)(j % a.c.P);
    const unsigned char* mb = a.c.micro(page, hk, t);
    float dot = 0.0f, val[N];
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int d = lane + 32 * n;
      const uint32_t* kr = reinterpret_cast<const uint32_t*>(mb + (t & 15) * a.c.row_bytes());
      const uint32_t* vr = reinterpret_cast<const uint32_t*>(mb + rows + pars + (t & 15) * a.c.row_bytes());
      const float2 kp = __half22float2(reinterpret_cast<const __half2*>(
          mb + rows + (t & 15) * a.c.par_bytes())[d / a.c.g]);
      const float2 vp = __half22float2(reinterpret_cast<const __half2*>(
          mb + 2 * rows + pars + (t & 15) * a.c.par_bytes())[d / a.c.g]);
      const float kn = (float)((kr[kv4_key_word(d >> 3, D)] >> (4 * (d & 7))) & 15u);
      const float vn = (float)((vr[d >> 3] >> (4 * (d & 7))) & 15u);
      dot = fmaf(q[n], fmaf(kn, kp.x, kp.y), dot);
      val[n] = fmaf(vn, vp.x, vp.y);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
    const float mn = fmaxf(m, dot);
    const float f = expf(m - mn), p = expf(dot - mn);
    l = l * f + p;
#pragma unroll
    for (int n = 0; n < N; ++n) acc[n] = fmaf(p, val[n], acc[n] * f);
    m = mn;
  }
  const float nan = __int_as_float(0x7fc00000);
  const float inv = bad ? nan : l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : nan);
  T* orow = static_cast<T*>(a.o) + row * D;
#pragma unroll
  for (int n = 0; n < N; ++n) st1(orow + lane + 32 * n, acc[n] * inv);
  if (a.lse && lane == 0)
    a.lse[(b * a.H + h) * a.Sq + i] = bad ? nan : l > 0.0f ? m + logf(l) : (l == 0.0f ? -INFINITY : nan);
}

template <typename T> static int kv4_attn_launch(const Kv4AttnArgs& a, cudaStream_t st) {
  const unsigned grid = (unsigned)((a.B * a.Sq * a.H + 3) / 4);
  switch (a.c.D) {
    case 64: launch_pdl(kv4_attn_simple<T, 64>, dim3(grid), dim3(128), 0, st, a); break;
    case 128: launch_pdl(kv4_attn_simple<T, 128>, dim3(grid), dim3(128), 0, st, a); break;
    default: launch_pdl(kv4_attn_simple<T, 256>, dim3(grid), dim3(128), 0, st, a); break;
  }
  return check_launch("b2k_kv4_attention");
}

int kv4_check(const char* what, const void* data, int64_t pages, int64_t Hk, int64_t P, int64_t D,
              int64_t g);

}  // namespace b2k

using namespace b2k;

extern "C" int64_t b2k_kv4_attention_workspace(int64_t B, int64_t Sq, int64_t H, int64_t Hk,
                                               int64_t D) {
  return B >= 0 && Sq >= 0 && H >= 0 && Hk >= 1 && D >= 0 ? 0 : -1;
}

extern "C" int b2k_kv4_attention(const void* q, int64_t qb, int64_t qs, int64_t qh, void* o,
                                 float* lse, const void* data, int64_t pages, int64_t Hk, int64_t P,
                                 int64_t D, int64_t group, const int32_t* table, int64_t width,
                                 const int32_t* lens, int64_t B, int64_t Sq, int64_t H, float scale,
                                 int causal, int dtype, void* workspace, int64_t workspace_bytes,
                                 void* stream) {
  (void)workspace; (void)workspace_bytes;
  if (int st = kv4_check("b2k_kv4_attention", data, pages, Hk, P, D, group)) return st;
  B2K_REQUIRE(B >= 0 && Sq >= 0 && H >= 0 && width >= 0, "b2k_kv4_attention: negative shape");
  B2K_REQUIRE(H % Hk == 0, "b2k_kv4_attention: %lld heads are no multiple of the cache's %lld",
              (long long)H, (long long)Hk);
  B2K_REQUIRE(dtype == B2K_F16 || dtype == B2K_BF16, "b2k_kv4_attention: dtype %d is not 16-bit",
              dtype);
  if (B == 0 || Sq == 0 || H == 0) return B2K_OK;
  B2K_REQUIRE(B * Sq <= 0x7fffffffLL / H, "b2k_kv4_attention: too many query rows");
  B2K_REQUIRE(q && o && lens && (table || width == 0), "b2k_kv4_attention: null operand");
  Kv4AttnArgs a = {};
  a.c = Kv4{static_cast<unsigned char*>(const_cast<void*>(data)), pages, (int)Hk, (int)P, (int)D,
            (int)group};
  a.q = q; a.o = o; a.lse = lse; a.table = table; a.lens = lens;
  a.B = B; a.Sq = Sq; a.H = H; a.width = width;
  a.qb = qb; a.qs = qs; a.qh = qh;
  a.scale = scale; a.causal = causal != 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == B2K_F16 ? kv4_attn_launch<__half>(a, st) : kv4_attn_launch<__nv_bfloat16>(a, st);
}
