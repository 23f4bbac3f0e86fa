// b2k_kv4_attention: attention of new queries over the 4-bit paged cache
// (kv4.cuh).
//
//   o_i = sum_j p_ij v_j / sum_j p_ij,   p_ij = exp(scale q_i . k_j - m_i)
//   over j <= len - Sq + i (causal) or j < len; a row that sees nothing is 0.
//
// With k_j = lo_g + s_g n over each group g of dimensions,
//   q . k = sum_g s_g (sum_{d in g} q_d n_d) + lo_g (sum_{d in g} q_d),
// so the products run on the stored integers and the parameters meet fp32
// sums.  What has to be read is the cache, D + 8 D / g bytes per token and
// head; the G = H / Hk query heads of a cache head share that reading.  Each
// element is unpacked once for all of them and meets them in matrix
// instructions: rows of the queries (G per new token) are the 8 NT columns
// of mma.m16n8k16, tokens (scores) and dimensions (output) its 16 rows, so a
// lane unpacks straight into the A operand.  For a few rows per head the
// kernel is bound by the reading and by unpacking, not by the products.
//
//   * Keys: `word & 0x000f000f` is a pair of float16 subnormals n * 2^-24,
//     exact in the product, without a conversion (`& 0x00f000f0`: 16 times
//     that, against queries held / 16).  Queries are scaled by a power of two
//     to a row maximum in [2^9, 2^10), which keeps bfloat16's range.
//   * Values: tokens are the contracted index, so their parameters cannot
//     wait for the sum: lo + s n is formed in float16 (one rounding, 2^-11) and
//     meets probabilities in float16 (2^-11), sums in fp32.  Probabilities are
//     held times 2^10, which keeps small ones out of the subnormals.
//   * The running maximum and sum are fp32, per lane for its own tokens; the
//     output is rescaled only when a maximum moves.
//
// Work is split by tiles of tokens, not by sequences: all (sequence, row
// tile, head) segments are laid end to end and every block takes an equal
// run of tiles, found on the device from the lengths (which the host does not
// know), so ragged batches and single long sequences fill the GPU alike.  A
// segment that spans blocks leaves partial (m, l, O) in the workspace, merged
// in block order by a second kernel (the same bits whatever ran first).
// Within a block the warps take tiles in turn, each with its own ring of bulk
// copies; they meet once per segment.
#include "kv4.cuh"
#include "rowio.cuh"
#include "tma.cuh"

B2K_DEFINE_TIMEOUT_COUNTER()

namespace b2k {

int kv4_check(const char* what, const void* data, int64_t pages, int64_t Hk, int64_t P, int64_t D,
              int64_t g);

constexpr int kAttnWarps = 4;
constexpr int kAttnStages = 3;
constexpr float kPScale = 10.0f;  // probabilities are held times 2^10

struct Kv4AttnArgs {
  Kv4 c;
  const void* q;
  void* o;
  float* lse;
  const int32_t *table, *lens;
  int64_t B, Sq, H, width;
  int64_t qb, qs, qh;  // strides of q in elements (batch, token, head)
  float scale;
  int causal, bf16, q_aligned;
  int G, RT;  // query heads per cache head; row tiles per (sequence, head)
  float* part;      // [2 * blocks][rows][D] outputs, then [2 * blocks][rows][2] (m, l)
  int2* spans;      // [segments] first and last block
};

// tokens of a tile: about the same bytes for every D, and registers for its
// scores (NT T / 8 per thread) beside the output's
__host__ __device__ constexpr int attn_tile(int D, int NT) { return D == 256 || NT * D > 256 ? 16 : 32; }
__host__ __device__ constexpr int attn_rows(int NT) { return 8 * NT; }
// resident blocks per SM: registers (NT D / 4 for the output) and shared memory
__host__ __device__ constexpr int attn_cps(int D, int NT) { return NT * D > 256 ? 2 : 3; }

// Token counts fit 32 bits (the host refuses wider tables), runs of tiles over
// all segments do not.
__device__ __forceinline__ int attn_len(const Kv4AttnArgs& a, int b, bool& bad) {
  const int given = a.lens[b], cap = (int)(a.width * a.c.P);
  bad = given > cap;
  return min(max(given, 0), cap);
}
// first token that no row of the row tile sees
template <int D, int NT>
__device__ __forceinline__ int attn_end(const Kv4AttnArgs& a, int len, int rt) {
  const int last_row = (int)min((int64_t)(rt + 1) * attn_rows(NT), a.Sq * a.G) - 1;
  return max(a.causal ? len - (int)a.Sq + last_row / a.G + 1 : len, 0);
}
// tiles of each of its segments (one at least: somebody writes the zeros)
template <int D, int NT> __device__ __forceinline__ int attn_tiles(const Kv4AttnArgs& a, int entry) {
  bool bad;
  const int b = entry / a.RT, end = attn_end<D, NT>(a, attn_len(a, b, bad), entry - b * a.RT);
  return max((end + attn_tile(D, NT) - 1) / attn_tile(D, NT), 1);
}

__device__ __forceinline__ void mma16816(float* c, uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
__device__ __forceinline__ uint32_t as_u32(__half2 v) { return *reinterpret_cast<uint32_t*>(&v); }
__device__ __forceinline__ __half2 as_h2(uint32_t v) { return *reinterpret_cast<__half2*>(&v); }

template <int BYTES> __device__ __forceinline__ void load_words(uint32_t* w, const unsigned char* p) {
  if constexpr (BYTES >= 16) {
#pragma unroll
    for (int i = 0; i < BYTES / 16; ++i) {
      const uint4 v = reinterpret_cast<const uint4*>(p)[i];
      w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
    }
  } else if constexpr (BYTES == 8) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x; w[1] = v.y;
  } else {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  }
}

// four nibbles of each half of x (the halves: two tokens) -> (lo + s n) pairs
__device__ __forceinline__ void value_pairs(uint32_t x, __half2 s, __half2 lo, uint32_t* out) {
  const __half2 k1024 = __float2half2_rn(1024.0f), k16 = __float2half2_rn(0.0625f),
                km64 = __float2half2_rn(-64.0f);
  const uint32_t y = x >> 8;
  // 0x6400 | n is 1024 + n; the upper nibble of a byte is 1024 + 16 n
  const __half2 n0 = __hsub2(as_h2((x & 0x000f000fu) | 0x64006400u), k1024);
  const __half2 n1 = __hfma2(as_h2((x & 0x00f000f0u) | 0x64006400u), k16, km64);
  const __half2 n2 = __hsub2(as_h2((y & 0x000f000fu) | 0x64006400u), k1024);
  const __half2 n3 = __hfma2(as_h2((y & 0x00f000f0u) | 0x64006400u), k16, km64);
  out[0] = as_u32(__hfma2(n0, s, lo));
  out[1] = as_u32(__hfma2(n1, s, lo));
  out[2] = as_u32(__hfma2(n2, s, lo));
  out[3] = as_u32(__hfma2(n3, s, lo));
}

template <int D, int GRP, int NT> struct AttnShape {
  static constexpr int T = attn_tile(D, NT), U = T / 16, J = D / 32, NG = D / GRP, ROWS = attn_rows(NT);
  static constexpr int MB = 16 * (D + 8 * NG);           // bytes of a micro block
  static constexpr int KP = 8 * D, VR = KP + 64 * NG, VP = VR + 8 * D;  // its fields
  static constexpr int STAGE = U * MB;
  static constexpr int RING = kAttnWarps * kAttnStages * STAGE;
  static constexpr int MERGE = kAttnWarps * ROWS * D * 4;
  // query fragments, and the groups' sums, in shared memory instead of registers
  static constexpr bool QS = NT * D > 128, GS = NT * NG > 4;
  static constexpr int QB = (QS ? NT * J * 512 : 0) + (GS ? NT * NG * 32 : 0);
  static constexpr int SMEM = (RING > MERGE ? RING : MERGE) + QB;
};

template <int D, int GRP, int NT>
__global__ void __launch_bounds__(32 * kAttnWarps, attn_cps(D, NT))
kv4_attn_kernel(const __grid_constant__ Kv4AttnArgs a) {
  using X = AttnShape<D, GRP, NT>;
  constexpr int T = X::T, U = X::U, J = X::J, NG = X::NG, MB = X::MB, S = kAttnStages;
  constexpr int VW = D / 64;  // words of a lane's D / 8 value dimensions
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ uint64_t full[kAttnWarps][S];
  __shared__ int64_t scan[kAttnWarps + 1];
  __shared__ int start_entry;
  __shared__ int64_t start_rest;
  __shared__ float mrg[kAttnWarps][X::ROWS][2];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, r = lane >> 2, c = lane & 3;
  unsigned char* ring = smem + warp * (S * X::STAGE);
  uint32_t* qsm = reinterpret_cast<uint32_t*>(smem + X::SMEM - X::QB);
  float* gsm = reinterpret_cast<float*>(smem + X::SMEM - (X::GS ? NT * NG * 32 : 0));

  griddep_launch_dependents();
  if (lane < S) mbar_init(&full[warp][lane], 1);
  fence_barrier_init();
  griddep_wait();

  // ---- this block's run of tiles -----------------------------------------
  const int entries = (int)(a.B * a.RT);  // (sequence, row tile), Hk segments each
  const int chunk = (entries + (int)blockDim.x - 1) / (int)blockDim.x;
  const int e0 = min(entries, tid * chunk), e1 = min(entries, e0 + chunk);
  int64_t mine = 0;
  for (int e = e0; e < e1; ++e) mine += attn_tiles<D, NT>(a, e);
  int64_t incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t t = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += t;
  }
  if (lane == 31) scan[warp] = incl;
  __syncthreads();
  int64_t before = incl - mine, total = 0;
#pragma unroll
  for (int w = 0; w < kAttnWarps; ++w) {
    if (w < warp) before += scan[w];
    total += scan[w];
  }
  before *= a.c.Hk;
  total *= a.c.Hk;
  // a block has at least one tile per warp
  const int64_t blocks = min((int64_t)gridDim.x, (total + kAttnWarps - 1) / kAttnWarps);
  const int64_t me = blockIdx.x;
  if (me >= blocks) return;
  const int64_t u0 = me * total / blocks, u1 = (me + 1) * total / blocks;
  if (u0 >= before && u0 < before + mine * a.c.Hk) {
    int64_t at = before;
    int e = e0;
    for (;; ++e) {
      const int64_t n = (int64_t)attn_tiles<D, NT>(a, e) * a.c.Hk;
      if (u0 < at + n) break;
      at += n;
    }
    start_entry = e;
    start_rest = u0 - at;
  }
  __syncthreads();

  int entry = start_entry;
  int64_t unit = u0;
  int n_seg = attn_tiles<D, NT>(a, entry);
  int head = (int)(start_rest / n_seg);
  int t0 = (int)(start_rest - (int64_t)head * n_seg);  // first tile of this part
  uint32_t issued = 0, used = 0;                       // stages, over the whole block
  bool timeout = false;

  while (unit < u1 && !timeout) {
    const int b = entry / a.RT, rt = entry - b * a.RT;
    bool bad;
    const int len = attn_len(a, b, bad);
    const int end = attn_end<D, NT>(a, len, rt);
    const int t1 = (int)min((int64_t)n_seg, t0 + (u1 - unit));  // one past its last tile
    const int R = (int)(a.Sq * a.G);
    const int row0 = rt * X::ROWS;
    // last token that a row of the tile sees
    auto last_of = [&](int row) {
      return a.causal ? len - (int)a.Sq + min(row0 + row, R - 1) / a.G : len - 1;
    };

    // ---- the ring: tile t of this warp into stage `issued` ----------------
    const int32_t* pages = a.table + b * a.width;
    auto issue = [&](int t) {
      const int s = issued % S;
      const int tok = t * T + (lane < U ? 16 * lane : 0);
      bool have = false;
      int page = 0;
      if (lane < U && tok < end) {
        page = pages[tok / a.c.P];
        have = page >= 0 && page < a.c.pages;
        if (!have) bad = true;
      }
      const uint32_t n = __popc(__ballot_sync(0xffffffffu, have));
      fence_proxy_async();
      if (lane == 0) mbar_arrive_expect_tx(&full[warp][s], n * MB);
      __syncwarp();
      if (have)
        bulk_g2s(ring + s * X::STAGE + lane * MB, a.c.micro(page, head, tok % a.c.P), MB,
                 &full[warp][s]);
      ++issued;
    };
    int next = t0 + warp;  // tile of the next issue
    for (int k = 0; k < S && next < t1; ++k, next += kAttnWarps) issue(next);

    // ---- query rows -> B fragments -----------------------------------------
    // lane (r, c) holds row r of each 8, dimensions 32 j + 8 c .. + 7
    uint32_t qf[X::QS ? 1 : NT][X::QS ? 1 : J][4];
    float qsum[X::GS ? 1 : NT][X::GS ? 1 : NG][2], cmul[NT][2];
    if (X::QS || X::GS) __syncthreads();
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int row = row0 + nt * 8 + r;
      float v[J][8];
#pragma unroll
      for (int j = 0; j < J; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) v[j][e] = 0.0f;
      if (row < R) {
        const int i = row / a.G, hq = head * a.G + (row - i * a.G);
        const int64_t off = b * a.qb + i * a.qs + hq * a.qh;
#pragma unroll
        for (int j = 0; j < J; ++j) {
          const int d = 32 * j + 8 * c;
          if (a.bf16)
            load_vec<__nv_bfloat16, false>(v[j], static_cast<const __nv_bfloat16*>(a.q) + off, d, D,
                                           a.q_aligned != 0);
          else
            load_vec<__half, false>(v[j], static_cast<const __half*>(a.q) + off, d, D,
                                    a.q_aligned != 0);
        }
      }
      float top = 0.0f;
#pragma unroll
      for (int j = 0; j < J; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(v[j][e]));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // 2^(9 - floor(log2 top)); 1 for a row of zeros or one that is not finite
      const int ex = (int)(__float_as_uint(top) >> 23);
      const float f = top > 0.0f && ex < 255
                          ? __uint_as_float((uint32_t)min(263 - ex, 254) << 23) : 1.0f;
      float part[NG];
#pragma unroll
      for (int g = 0; g < NG; ++g) part[g] = 0.0f;
#pragma unroll
      for (int j = 0; j < J; ++j) {
        __half h[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          h[e] = __float2half_rn(v[j][e] * f);
          part[j * 32 / GRP] += __half2float(h[e]);
          // odd nibbles are unpacked as 16 n
          if (e & 1) h[e] = __float2half_rn(v[j][e] * (f * 0.0625f));
        }
        uint32_t w[4] = {as_u32(__halves2half2(h[0], h[4])), as_u32(__halves2half2(h[2], h[6])),
                         as_u32(__halves2half2(h[1], h[5])), as_u32(__halves2half2(h[3], h[7]))};
        if constexpr (X::QS) {
          if ((nt * J + j) % kAttnWarps == warp)
            reinterpret_cast<uint4*>(qsm)[(nt * J + j) * 32 + lane] =
                make_uint4(w[0], w[1], w[2], w[3]);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) qf[nt][j][e] = w[e];
        }
      }
      const float cm = a.scale * kLog2e * (16777216.0f / f);
#pragma unroll
      for (int p = 0; p < 2; ++p) {  // what this lane's columns 2c, 2c + 1 need
        const int src = (2 * c + p) * 4;
        cmul[nt][p] = __shfl_sync(0xffffffffu, cm, src);
      }
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        float t = part[g];
        t += __shfl_xor_sync(0xffffffffu, t, 1);
        t += __shfl_xor_sync(0xffffffffu, t, 2);
        t *= 5.9604644775390625e-8f;  // 2^-24, the unit of the integers' products
        if constexpr (X::GS) {
          if (nt % kAttnWarps == warp && c == 0) gsm[(nt * NG + g) * 8 + r] = t;
        } else {
          qsum[nt][g][0] = __shfl_sync(0xffffffffu, t, 8 * c);
          qsum[nt][g][1] = __shfl_sync(0xffffffffu, t, 8 * c + 4);
        }
      }
    }
    if (X::QS || X::GS) __syncthreads();
    const int all_see = last_of(0);  // tokens up to here are seen by every row

    float o[D / 16][NT][4];
    float m[NT][2], l[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int i = 0; i < D / 16; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][nt][e] = 0.0f;
      m[nt][0] = m[nt][1] = -INFINITY;
      l[nt][0] = l[nt][1] = 0.0f;
    }

    for (int t = t0 + warp; t < t1; t += kAttnWarps) {
      const int s = used % S;
      if (!mbar_wait(&full[warp][s], (used / S) & 1)) {
        timeout = true;
        break;
      }
      ++used;
      unsigned char* st = ring + s * X::STAGE;
      const int tok0 = t * T;
      const bool masked = tok0 + T - 1 > all_see;
      if (masked) {
        // What lies past the length is garbage, and a value some row does not
        // see must not reach it as 0 * NaN: such parameters become zero, and
        // rows that do see a value that is not finite become NaN.
        bool nan = false;
        const int tok = tok0 + lane;
        if (lane < T && tok > all_see) {
          uint32_t* p = reinterpret_cast<uint32_t*>(st + (lane >> 4) * MB + X::VP) + (lane & 15) * NG;
#pragma unroll
          for (int g = 0; g < NG; ++g) {
            const uint32_t w = p[g];
            const bool odd = (w & 0x7c00u) == 0x7c00u || (w & 0x7c000000u) == 0x7c000000u;
            if (tok >= end) p[g] = 0;
            else if (odd) {
              p[g] = 0;
              nan = true;
            }
          }
        }
        uint32_t some = __ballot_sync(0xffffffffu, nan);
        for (; some; some &= some - 1) {
          const int at = tok0 + __ffs(some) - 1;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int p = 0; p < 2; ++p)
              if (last_of(nt * 8 + 2 * c + p) >= at) l[nt][p] = __int_as_float(0x7fc00000);
        }
        __syncwarp();
      }

      // ---- scores: [tokens] x [rows] ---------------------------------------
      float z[U][NT][4];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const unsigned char* mb = st + u * MB;
        uint32_t wa[J], wb[J], pa[NG], pb[NG];
        load_words<D / 8>(wa, mb + r * (D / 2) + c * (D / 8));
        load_words<D / 8>(wb, mb + (r + 8) * (D / 2) + c * (D / 8));
        load_words<4 * NG>(pa, mb + X::KP + r * 4 * NG);
        load_words<4 * NG>(pb, mb + X::KP + (r + 8) * 4 * NG);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) z[u][nt][e] = 0.0f;
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          float acc[NT][4];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[nt][e] = 0.0f;
#pragma unroll
          for (int j = g * (GRP / 32); j < (g + 1) * (GRP / 32); ++j) {
            const uint32_t ya = wa[j] >> 8, yb = wb[j] >> 8;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              uint32_t q4[4];
              if constexpr (X::QS) {
                const uint4 v = reinterpret_cast<const uint4*>(qsm)[(nt * J + j) * 32 + lane];
                q4[0] = v.x; q4[1] = v.y; q4[2] = v.z; q4[3] = v.w;
              } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) q4[e] = qf[nt][j][e];
              }
              mma16816(acc[nt], wa[j] & 0x000f000fu, wb[j] & 0x000f000fu, ya & 0x000f000fu,
                       yb & 0x000f000fu, q4[0], q4[1]);
              mma16816(acc[nt], wa[j] & 0x00f000f0u, wb[j] & 0x00f000f0u, ya & 0x00f000f0u,
                       yb & 0x00f000f0u, q4[2], q4[3]);
            }
          }
          const float2 fa = __half22float2(as_h2(pa[g])), fb = __half22float2(as_h2(pb[g]));
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            float2 qs;
            if constexpr (X::GS) qs = reinterpret_cast<const float2*>(gsm)[(nt * NG + g) * 4 + c];
            else qs = f2(qsum[nt][g][0], qsum[nt][g][1]);
            z[u][nt][0] = fmaf(fa.x, acc[nt][0], fmaf(fa.y, qs.x, z[u][nt][0]));
            z[u][nt][1] = fmaf(fa.x, acc[nt][1], fmaf(fa.y, qs.y, z[u][nt][1]));
            z[u][nt][2] = fmaf(fb.x, acc[nt][2], fmaf(fb.y, qs.x, z[u][nt][2]));
            z[u][nt][3] = fmaf(fb.x, acc[nt][3], fmaf(fb.y, qs.y, z[u][nt][3]));
          }
        }
      }

      // ---- softmax: columns 2c, 2c + 1 are this lane's rows of queries -------
      float top[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        top[nt][0] = top[nt][1] = -INFINITY;
        int last[2] = {0, 0};
        if (masked) {
          last[0] = last_of(nt * 8 + 2 * c);
          last[1] = last_of(nt * 8 + 2 * c + 1);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float v = z[u][nt][e] * cmul[nt][e & 1];
            if (masked && tok0 + 16 * u + r + 8 * (e >> 1) > last[e & 1]) v = -INFINITY;
            z[u][nt][e] = v;
            top[nt][e & 1] = fmaxf(top[nt][e & 1], v);
          }
      }
      bool moved = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          float v = top[nt][p];
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, x));
          top[nt][p] = fmaxf(v, m[nt][p]);
          moved |= top[nt][p] > m[nt][p];
        }
      if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float f[2];
#pragma unroll
          for (int p = 0; p < 2; ++p) {
            // from -inf: nothing was summed yet (0 * 0 whatever the new one is)
            f[p] = m[nt][p] == -INFINITY ? 0.0f : ex2_approx(m[nt][p] - top[nt][p]);
            l[nt][p] *= f[p];
            m[nt][p] = top[nt][p];
          }
#pragma unroll
          for (int i = 0; i < D / 16; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[i][nt][e] *= f[e & 1];
        }
      }
      uint32_t pf[U][NT][2];  // probabilities as B fragments: [tokens] x [rows]
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float off[2];
#pragma unroll
        for (int p = 0; p < 2; ++p) off[p] = m[nt][p] == -INFINITY ? 0.0f : m[nt][p] - kPScale;
#pragma unroll
        for (int u = 0; u < U; ++u) {
          float p[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            p[e] = ex2_approx(z[u][nt][e] - off[e & 1]);
            l[nt][e & 1] += p[e];
          }
          pf[u][nt][0] = transpose8x8(as_u32(__floats2half2_rn(p[0], p[1])));
          pf[u][nt][1] = transpose8x8(as_u32(__floats2half2_rn(p[2], p[3])));
        }
      }

      // ---- output: [dimensions] x [rows] -----------------------------------
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const unsigned char* mb = st + u * MB;
        uint32_t v[4][VW], par[4];  // tokens 2c, 2c + 1, 2c + 8, 2c + 9
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int tk = 2 * c + (k & 1) + 8 * (k >> 1);
          load_words<4 * VW>(v[k], mb + X::VR + tk * (D / 2) + r * (D / 16));
          par[k] = reinterpret_cast<const uint32_t*>(mb + X::VP)[tk * NG + r * (D / 8) / GRP];
        }
        const __half2 s0 = as_h2(__byte_perm(par[0], par[1], 0x5410));
        const __half2 o0 = as_h2(__byte_perm(par[0], par[1], 0x7632));
        const __half2 s1 = as_h2(__byte_perm(par[2], par[3], 0x5410));
        const __half2 o1 = as_h2(__byte_perm(par[2], par[3], 0x7632));
#pragma unroll
        for (int w = 0; w < VW; ++w)
#pragma unroll
          for (int hi = 0; hi < 2; ++hi) {
            const uint32_t sel = hi ? 0x7632 : 0x5410;
            uint32_t x0[4], x1[4];
            value_pairs(__byte_perm(v[0][w], v[1][w], sel), s0, o0, x0);
            value_pairs(__byte_perm(v[2][w], v[3][w], sel), s1, o1, x1);
#pragma unroll
            for (int q = 0; q < 2; ++q)
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
                mma16816(o[w * 4 + hi * 2 + q][nt], x0[2 * q], x0[2 * q + 1], x1[2 * q],
                         x1[2 * q + 1], pf[u][nt][0], pf[u][nt][1]);
          }
      }
      __syncwarp();
      if (next < t1) {
        issue(next);
        next += kAttnWarps;
      }
    }
    if (timeout)  // nothing may land after the block has gone
      for (; used < issued; ++used) mbar_wait(&full[warp][used % S], (used / S) & 1);
    timeout = __syncthreads_or(timeout) != 0;
    bad = __syncthreads_or(bad || timeout) != 0;
    if (timeout && tid == 0) atomicAdd(&b2k_tu_timeouts, 1u);

    // ---- the warps' parts meet (the rings are drained) ----------------------
    float* mo = reinterpret_cast<float*>(smem);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        float v = l[nt][p];
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) v += __shfl_xor_sync(0xffffffffu, v, x);
        if (r == 0) {
          mrg[warp][nt * 8 + 2 * c + p][0] = m[nt][p];
          mrg[warp][nt * 8 + 2 * c + p][1] = v;
        }
#pragma unroll
        for (int i = 0; i < D / 16; ++i)
          *reinterpret_cast<float2*>(mo + (size_t)(warp * X::ROWS + nt * 8 + 2 * c + p) * D +
                                     r * (D / 8) + 2 * i) = f2(o[i][nt][p], o[i][nt][2 + p]);
      }
    }
    __syncthreads();
    const bool whole = t0 == 0 && t1 == n_seg;
    const int slot = (int)(2 * me + (t0 == 0 ? 1 : 0));
    const int64_t seg = (int64_t)entry * a.c.Hk + head;
    if (tid == 0 && t0 == 0) {
      // blocks that hold the segment's first and last tile
      const int64_t lastu = unit + n_seg - 1;
      a.spans[seg] = make_int2((int)me, whole ? (int)me : (int)(((lastu + 1) * blocks - 1) / total));
    }
    for (int x = tid; x < X::ROWS * (D / 4); x += blockDim.x) {
      const int row = x / (D / 4), d = (x - row * (D / 4)) * 4;
      if (row0 + row >= R) continue;
      float M = -INFINITY;
#pragma unroll
      for (int w = 0; w < kAttnWarps; ++w) M = fmaxf(M, mrg[w][row][0]);
      float L = 0.0f;
      float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int w = 0; w < kAttnWarps; ++w) {
        const float mw = mrg[w][row][0];
        const float f = mw == -INFINITY ? (mrg[w][row][1] == 0.0f ? 0.0f : 1.0f) : ex2_approx(mw - M);
        const float4 t = *reinterpret_cast<const float4*>(mo + (size_t)(w * X::ROWS + row) * D + d);
        L = fmaf(mrg[w][row][1], f, L);
        v.x = fmaf(t.x, f, v.x); v.y = fmaf(t.y, f, v.y);
        v.z = fmaf(t.z, f, v.z); v.w = fmaf(t.w, f, v.w);
      }
      if (bad) L = __int_as_float(0x7fc00000);
      if (!whole) {
        *reinterpret_cast<float4*>(a.part + ((size_t)slot * X::ROWS + row) * D + d) = v;
        if (d == 0) {
          float* ml = a.part + (size_t)2 * gridDim.x * X::ROWS * D + ((size_t)slot * X::ROWS + row) * 2;
          ml[0] = M;
          ml[1] = L;
        }
        continue;
      }
      const int i = (row0 + row) / a.G, hq = head * a.G + (row0 + row - i * a.G);
      const float inv = L == 0.0f ? 0.0f : 1.0f / L;
      const float y[4] = {v.x * inv, v.y * inv, v.z * inv, v.w * inv};
      const int64_t at = (((int64_t)b * a.Sq + i) * a.H + hq) * D + d;
      uint2 w2;
      if (a.bf16) {
        __nv_bfloat162 p0 = __floats2bfloat162_rn(y[0], y[1]), p1 = __floats2bfloat162_rn(y[2], y[3]);
        w2 = make_uint2(*reinterpret_cast<uint32_t*>(&p0), *reinterpret_cast<uint32_t*>(&p1));
      } else {
        w2 = make_uint2(as_u32(__floats2half2_rn(y[0], y[1])), as_u32(__floats2half2_rn(y[2], y[3])));
      }
      *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.o) + at) = w2;
      if (a.lse && d == 0)
        a.lse[((int64_t)b * a.H + hq) * a.Sq + i] =
            L == 0.0f ? -INFINITY : (M - kPScale) * kLn2 + logf(L);
    }
    __syncthreads();

    unit += t1 - t0;
    t0 = 0;
    if (++head == a.c.Hk) {
      head = 0;
      ++entry;
      if (unit < u1) n_seg = attn_tiles<D, NT>(a, entry);
    }
  }
}

// Merges the partial (m, l, O) of segments that span blocks, in block order.
// One block per row of a segment: D / 4 threads hold four dimensions each.
template <int D, int NT>
__global__ void __launch_bounds__(D / 4) kv4_attn_merge_kernel(const __grid_constant__ Kv4AttnArgs a,
                                                                int blocks) {
  constexpr int ROWS = attn_rows(NT);
  griddep_launch_dependents();
  griddep_wait();
  const int64_t seg = blockIdx.x;
  const int row = blockIdx.y, d = threadIdx.x * 4;
  const int2 span = a.spans[seg];
  if (span.x == span.y) return;
  const int64_t entry = seg / a.c.Hk, b = entry / a.RT;
  const int head = (int)(seg - entry * a.c.Hk);
  const int64_t rr = (entry - b * a.RT) * ROWS + row;
  if (rr >= a.Sq * a.G) return;
  const float* ml = a.part + (size_t)2 * blocks * ROWS * D;
  float M = -INFINITY, L = 0.0f;
  float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (int i = span.x; i <= span.y; ++i) {
    const size_t slot = (size_t)(2 * i + (i == span.x ? 1 : 0)) * ROWS + row;
    const float2 p = *reinterpret_cast<const float2*>(ml + 2 * slot);
    const float4 t = *reinterpret_cast<const float4*>(a.part + slot * D + d);
    const float Mn = fmaxf(M, p.x);
    const float f0 = M == -INFINITY ? (L == 0.0f ? 0.0f : 1.0f) : ex2_approx(M - Mn);
    const float f1 = p.x == -INFINITY ? (p.y == 0.0f ? 0.0f : 1.0f) : ex2_approx(p.x - Mn);
    L = L * f0 + p.y * f1;
    v.x = v.x * f0 + t.x * f1; v.y = v.y * f0 + t.y * f1;
    v.z = v.z * f0 + t.z * f1; v.w = v.w * f0 + t.w * f1;
    M = Mn;
  }
  const int64_t i = rr / a.G, hq = head * a.G + (rr - i * a.G);
  const float inv = L == 0.0f ? 0.0f : 1.0f / L;
  const int64_t at = ((b * a.Sq + i) * a.H + hq) * D + d;
  uint2 w2;
  if (a.bf16) {
    __nv_bfloat162 p0 = __floats2bfloat162_rn(v.x * inv, v.y * inv);
    __nv_bfloat162 p1 = __floats2bfloat162_rn(v.z * inv, v.w * inv);
    w2 = make_uint2(*reinterpret_cast<uint32_t*>(&p0), *reinterpret_cast<uint32_t*>(&p1));
  } else {
    w2 = make_uint2(as_u32(__floats2half2_rn(v.x * inv, v.y * inv)),
                    as_u32(__floats2half2_rn(v.z * inv, v.w * inv)));
  }
  *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.o) + at) = w2;
  if (a.lse && d == 0)
    a.lse[(b * a.H + hq) * a.Sq + i] = L == 0.0f ? -INFINITY : (M - kPScale) * kLn2 + logf(L);
}

// columns of the products, in eights: the fewest that hold the rows, up to
// what the output's registers (NT D / 4 per thread) allow
static int attn_nt(int64_t rows, int64_t D) {
  if (rows <= 8) return 1;
  if (rows <= 16 || D == 256) return 2;
  return 4;
}

struct AttnPlan {
  int nt, blocks;
  int64_t rt, segs, part_bytes, bytes;
};

static AttnPlan attn_plan(int64_t B, int64_t Sq, int64_t H, int64_t Hk, int64_t D) {
  AttnPlan p;
  const int64_t rows = Sq * (H / Hk);
  p.nt = attn_nt(rows, D);
  p.rt = (rows + 8 * p.nt - 1) / (8 * p.nt);
  p.blocks = sm_count() * attn_cps((int)D, p.nt);
  p.segs = B * p.rt * Hk;
  p.part_bytes = (int64_t)2 * p.blocks * 8 * p.nt * (D + 2) * 4;
  p.bytes = p.part_bytes + p.segs * (int64_t)sizeof(int2);
  return p;
}

template <int D, int GRP, int NT>
static int attn_launch(const Kv4AttnArgs& a, const AttnPlan& p, cudaStream_t st) {
  auto kern = kv4_attn_kernel<D, GRP, NT>;
  static bool done[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !done[dev]) {
    cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                         AttnShape<D, GRP, NT>::SMEM);
    if (dev >= 0 && dev < 64) done[dev] = true;
  }
  launch_pdl(kern, dim3(p.blocks), dim3(32 * kAttnWarps), AttnShape<D, GRP, NT>::SMEM, st, a);
  launch_pdl(kv4_attn_merge_kernel<D, NT>, dim3((unsigned)p.segs, 8 * NT), dim3(D / 4), 0, st, a,
             p.blocks);
  return check_launch("b2k_kv4_attention");
}

template <int D, int GRP>
static int attn_dispatch(const Kv4AttnArgs& a, const AttnPlan& p, cudaStream_t st) {
  switch (p.nt) {
    case 1: return attn_launch<D, GRP, 1>(a, p, st);
    case 2: return attn_launch<D, GRP, 2>(a, p, st);
    default:
      if constexpr (D < 256) return attn_launch<D, GRP, 4>(a, p, st);
      return B2K_EUNSUPPORTED;
  }
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
  B2K_REQUIRE((reinterpret_cast<uintptr_t>(o) & 7u) == 0, "b2k_kv4_attention: o is not 8-byte aligned");
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
  a.part = static_cast<float*>(workspace);
  a.spans = reinterpret_cast<int2*>(static_cast<unsigned char*>(workspace) + p.part_bytes);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (D * 1000 + group) {
    case 64032: return attn_dispatch<64, 32>(a, p, st);
    case 64064: return attn_dispatch<64, 64>(a, p, st);
    case 128032: return attn_dispatch<128, 32>(a, p, st);
    case 128064: return attn_dispatch<128, 64>(a, p, st);
    case 128128: return attn_dispatch<128, 128>(a, p, st);
    case 256032: return attn_dispatch<256, 32>(a, p, st);
    case 256064: return attn_dispatch<256, 64>(a, p, st);
    default: return attn_dispatch<256, 128>(a, p, st);
  }
}
