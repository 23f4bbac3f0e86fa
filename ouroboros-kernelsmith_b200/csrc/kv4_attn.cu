// b2k_kv4_attention: argument checks and dispatch to the instances
// (kv4_attn_impl.cuh, kv4_attn_d*.cu).
#include "kv4_attn_plan.cuh"

namespace b2k {

// Columns of the products, in eights: the fewest that hold the rows, two at
// most.  One and two at 4 rows a head: 32 x 8192 tokens 82 and 104 us.  Four
// were slower: their registers cost more than reading the cache again from L2
// (D 128, two and four: 16 x 8192 tokens with 32 rows 107 and 129 us, 8 x 8192
// with 256 rows 374 and 422; D 64: 2 x 3000 with 32 rows 15.0 and 17.8, 16 x
// 8192 with 20 rows 77 and 68, the one case that lost).
static int attn_nt(int64_t rows) { return rows <= 8 ? 1 : 2; }

static AttnPlan attn_plan(int64_t B, int64_t Sq, int64_t H, int64_t Hk, int64_t D) {
  AttnPlan p;
  const int64_t rows = Sq * (H / Hk);
  p.nt = attn_nt(rows);
  p.rt = (rows + 8 * p.nt - 1) / (8 * p.nt);
  p.blocks = sm_count() * attn_cps((int)D, p.nt);
  p.warps = p.blocks * kAttnWarps;
  p.segs = B * p.rt * Hk;
  p.part_bytes = (int64_t)2 * p.warps * 8 * p.nt * (D + 2) * 4;
  p.bytes = p.part_bytes + p.segs * (int64_t)sizeof(int2);
  return p;
}

}  // namespace b2k

using namespace b2k;

extern "C" int64_t b2k_kv4_attention_workspace(int64_t B, int64_t Sq, int64_t H, int64_t Hk,
                                               int64_t D) {
  if (B < 0 || Sq < 0 || H < 0 || Hk < 1 || H % Hk || (D != 64 && D != 128 && D != 256)) return -1;
  if (B == 0 || Sq == 0 || H == 0) return 0;
  return attn_plan(B, Sq, H, Hk, D).bytes;
}

extern "C" int b2k_kv4_attention(const void* q, int64_t qb, int64_t qs, int64_t qh, void* o,
                                 float* lse, const void* data, int64_t pages, int64_t Hk, int64_t P,
                                 int64_t D, int64_t group, const int32_t* table, int64_t width,
                                 const int32_t* lens, int64_t B, int64_t Sq, int64_t H, float scale,
                                 int causal, int dtype, void* workspace, int64_t workspace_bytes,
                                 void* stream) {
  if (int st = kv4_check("b2k_kv4_attention", data, pages, Hk, P, D, group)) return st;
  B2K_REQUIRE(B >= 0 && Sq >= 0 && H >= 0 && width >= 0, "b2k_kv4_attention: negative shape");
  B2K_REQUIRE(H % Hk == 0, "b2k_kv4_attention: %lld heads are no multiple of the cache's %lld",
              (long long)H, (long long)Hk);
  B2K_REQUIRE(dtype == B2K_F16 || dtype == B2K_BF16, "b2k_kv4_attention: dtype %d is not 16-bit",
              dtype);
  if (B == 0 || Sq == 0 || H == 0) return B2K_OK;
  B2K_REQUIRE(B <= 0x7fffffffLL && Sq <= 0x7fffffffLL && H <= 0x7fffffffLL &&
                  B * Sq <= 0x7fffffffLL / H,
              "b2k_kv4_attention: too many query rows");
  B2K_REQUIRE(width <= (0x7fffffffLL - 64) / P, "b2k_kv4_attention: a table of %lld pages is too wide",
              (long long)width);
  B2K_REQUIRE(q && o && lens && (table || width == 0), "b2k_kv4_attention: null operand");
  B2K_REQUIRE(aligned16(o), "b2k_kv4_attention: o is not 16-byte aligned");
  const AttnPlan p = attn_plan(B, Sq, H, Hk, D);
  B2K_REQUIRE(workspace && aligned16(workspace) && workspace_bytes >= p.bytes,
              "b2k_kv4_attention: the workspace needs %lld aligned bytes, got %lld",
              (long long)p.bytes, (long long)workspace_bytes);
  Kv4AttnArgs a = {};
  a.c = Kv4{static_cast<unsigned char*>(const_cast<void*>(data)), pages, (int)Hk, (int)P, (int)D,
            (int)group};
  a.q = q; a.o = o; a.lse = lse; a.table = table; a.lens = lens;
  a.B = B; a.Sq = Sq; a.H = H; a.width = width;
  a.qb = qb; a.qs = qs; a.qh = qh;
  a.scale = scale; a.causal = causal != 0; a.bf16 = dtype == B2K_BF16;
  a.q_aligned = aligned16(q) && qb % 8 == 0 && qs % 8 == 0 && qh % 8 == 0;
  a.G = (int)(H / Hk);
  a.RT = (int)p.rt;
  a.warps = p.warps;
  a.dG = fast_div(a.G);
  a.dRT = fast_div(a.RT);
  a.dP = fast_div(P);
  a.dHk = fast_div(Hk);
  a.part = static_cast<float*>(workspace);
  a.spans = reinterpret_cast<int2*>(static_cast<unsigned char*>(workspace) + p.part_bytes);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (D == 64) return attn_d64(a, p, st);
  return D == 128 ? attn_d128(a, p, st) : attn_d256(a, p, st);
}
