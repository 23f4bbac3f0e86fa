// b2k_kv4_attention (kernels; one unit per head dimension): attention of new queries over the 4-bit paged cache
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
//     With one group for the whole head (g = D) the parameters can go with the
//     tokens after all: sum_t p_t (lo_t + s_t n_t) = sum_t (p_t s_t) (n_t - 8) +
//     sum_t p_t (lo_t + 8 s_t), the integers again as they are, p s formed in
//     fp32 and rounded once, the second sum one fp32 number per row.  The -8, the
//     same for every dimension, is summed apart and settled every four tiles: left
//     to the end, the sums would exceed the output by the square root of the tokens.
//     The running maximum is that of p s, so that these products use float16's
//     range whatever the values' magnitude.  (8 x 65536 tokens, D 128, g 128: 119
//     us instead of 135.)
//     For float16 queries the probabilities take two products, p (or p s)
//     rounded and what that left: their rounding would show beside float16's own
//     (errors 1.4 to 1.6 times those of fp32 products; 32 x 8192 tokens, g 32: 90
//     us instead of 83).
//   * The running maximum and sum are fp32, per lane for its own tokens; the
//     output is rescaled only when a row's maximum has moved by 2^4.
//
// Work is split by tiles of tokens, not by sequences: all (sequence, row
// tile, head) segments are laid end to end and every warp takes an equal run
// of tiles (a segment counts some more for its own costs), found on the
// device from the lengths, which the host does not know; so ragged batches and
// single long sequences fill the GPU alike.  Warps are independent: each has
// its own ring of bulk copies, which runs ahead across segments, and writes
// the segments that it holds whole.  A segment that spans warps leaves partial
// (m, l, O) in the workspace, merged in order by a second kernel (the same
// bits whatever ran first); where all of a block's runs lie in one segment,
// the long sequences, the block's warps merge theirs first.
#pragma once

#include "kv4_attn_plan.cuh"
#include "kv4_span.cuh"
#include "rowio.cuh"
#include "rowpipe.cuh"

namespace b2k {

constexpr int kAttnStages = 3;
constexpr float kPScale = 10.0f;  // probabilities are held times 2^10
constexpr float kPSlack = 4.0f;   // ... and below 2^(10 + 4) until the maximum is moved

// 64-bit division that takes the short way for what fits 32 bits
__device__ __forceinline__ int64_t wide_div(int64_t n, int64_t d) {
  if (((n | d) >> 32) == 0) return (uint32_t)n / (uint32_t)d;
  return n / d;
}



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
  const int last_row = min((rt + 1) * attn_rows(NT), (int)a.Sq * a.G) - 1;
  return max(a.causal ? len - (int)a.Sq + a.dG.div(last_row) + 1 : len, 0);
}
// tiles of each of its segments (one at least: somebody writes the zeros)
template <int D, int NT, int T> __device__ __forceinline__ int attn_tiles(const Kv4AttnArgs& a, int entry) {
  bool bad;
  const int b = a.dRT.div(entry), end = attn_end<D, NT>(a, attn_len(a, b, bad), entry - b * a.RT);
  return max((end + T - 1) / T, 1);
}

__device__ __forceinline__ void mma16816(float* c, uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// the same on zero sums
__device__ __forceinline__ void mma16816_first(float* c, uint32_t a0, uint32_t a1, uint32_t a2,
                                               uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%10,%10,%10,%10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
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

// A constant that stays in its register (the compiler would otherwise build it
// anew before most uses).
__device__ __forceinline__ uint32_t held(uint32_t v) {
  uint32_t r;
  asm volatile("mov.b32 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
struct ValueConsts {
  uint32_t magic;        // 0x6400 in both halves: 0x6400 | n is 1024 + n
  __half2 sixteenth, m64;
};

// four nibbles of each half of x (the halves: two tokens) -> (lo + s n) pairs
__device__ __forceinline__ void value_pairs(uint32_t x, __half2 s, __half2 lo, const ValueConsts& k,
                                            uint32_t* out) {
  const __half2 m1024 = __float2half2_rn(-1024.0f);
  const uint32_t y = x >> 8;
  // the upper nibble of a byte comes as 1024 + 16 n
  const __half2 n0 = __hadd2(as_h2((x & 0x000f000fu) | k.magic), m1024);
  const __half2 n1 = __hfma2(as_h2((x & 0x00f000f0u) | k.magic), k.sixteenth, k.m64);
  const __half2 n2 = __hadd2(as_h2((y & 0x000f000fu) | k.magic), m1024);
  const __half2 n3 = __hfma2(as_h2((y & 0x00f000f0u) | k.magic), k.sixteenth, k.m64);
  out[0] = as_u32(__hfma2(n0, s, lo));
  out[1] = as_u32(__hfma2(n1, s, lo));
  out[2] = as_u32(__hfma2(n2, s, lo));
  out[3] = as_u32(__hfma2(n3, s, lo));
}

template <int D, int GRP, int NT, int T> struct AttnShape {
  static constexpr int U = T / 16, J = D / 32, NG = D / GRP, ROWS = attn_rows(NT);
  static constexpr int MB = 16 * (D + 8 * NG);           // bytes of a micro block
  static constexpr bool FOLD = NG == 1;                  // values' parameters with the tokens
  static constexpr int KP = 8 * D, VR = KP + 64 * NG, VP = VR + 8 * D;  // its fields
  static constexpr int STAGE = U * MB;
  static constexpr int MERGE = kAttnWarps * ROWS * D * 4;
  // each warp's shared memory: its ring, the fragments of its queries and their
  // sums over each group
  static constexpr int QB = NT * J * 512, WARP = kAttnStages * STAGE + QB + NT * NG * 32;
  static constexpr int SMEM = kAttnWarps * WARP > MERGE ? kAttnWarps * WARP : MERGE;
};

// Four output values of 16 bits
__device__ __forceinline__ uint2 attn_pack4(const float4& v, float f, int bf16) {
  if (bf16) {
    const __nv_bfloat162 p0 = __floats2bfloat162_rn(v.x * f, v.y * f);
    const __nv_bfloat162 p1 = __floats2bfloat162_rn(v.z * f, v.w * f);
    return make_uint2(*reinterpret_cast<const uint32_t*>(&p0), *reinterpret_cast<const uint32_t*>(&p1));
  }
  return make_uint2(as_u32(__floats2half2_rn(v.x * f, v.y * f)),
                    as_u32(__floats2half2_rn(v.z * f, v.w * f)));
}
// 0 for a row that sees nothing; a NaN stays one
__device__ __forceinline__ float attn_inverse(float l) { return l == 0.0f ? 0.0f : 1.0f / l; }
__device__ __forceinline__ float attn_lse(float m, float l) {
  return l == 0.0f ? -INFINITY : (m - kPScale) * kLn2 + logf(l);
}
// factor of a part with maximum m and sum l in a merge to the maximum M; a
// part that saw nothing counts 0, one made NaN before it saw anything NaN
__device__ __forceinline__ float attn_weight(float m, float l, float M) {
  return m == -INFINITY ? (l == 0.0f ? 0.0f : 1.0f) : ex2_approx(m - M);
}

// (m, l) of a row of a partial slot, after the outputs of all slots
__device__ __forceinline__ float2* attn_ml(const Kv4AttnArgs& a, int64_t slot_row, int slot_floats) {
  return reinterpret_cast<float2*>(a.part + (int64_t)2 * a.warps * slot_floats) + slot_row;
}

// A walk over the parts of segments in a warp's run: tiles [t, t1) of segment
// (entry, head), which has n.
struct AttnWalk {
  int entry, head, n, pos, left;  // pos: units of the segment already taken
  int lead;                       // a segment's fixed costs, in units of a tile
  int t, t1;
};
// on to the next part that has tiles
template <int D, int NT, int T>
__device__ __forceinline__ bool attn_next(const Kv4AttnArgs& a, AttnWalk& k) {
  while (k.left > 0) {
    if (k.n == 0) k.n = attn_tiles<D, NT, T>(a, k.entry);
    const int take = min(k.left, k.n + k.lead - k.pos);
    k.t = max(k.pos - k.lead, 0);
    k.t1 = max(k.pos + take - k.lead, 0);
    k.left -= take;
    k.pos += take;
    if (k.t1 > k.t) return true;
    // only the lead of a segment that goes on in the next warp's run
  }
  return false;
}
// past a finished part
__device__ __forceinline__ void attn_step(const Kv4AttnArgs& a, AttnWalk& k) {
  if (k.pos < k.n + k.lead) return;  // the run ends within the segment
  k.pos = 0;
  if (++k.head == a.c.Hk) {
    k.head = 0;
    k.n = 0;
    ++k.entry;
  }
}

// A run in which a wait ran out, from the part at hand on: its parts are NaN,
// and accounted for like others, as the merges go by what the workspace says.
// Not inline: the kernel's registers are for the way that is taken.
template <int D, int NT, int T>
__device__ __noinline__ void attn_give_up(const Kv4AttnArgs& a, AttnWalk use, int run, int64_t u1,
                                          int64_t each, int64_t more) {
  constexpr int ROWS = attn_rows(NT);
  const int lane = threadIdx.x & 31;
  const float nan = __int_as_float(0x7fc00000);
  do {
    const bool whole = use.t == 0 && use.t1 == use.n;
    if (use.t == 0 && lane == 0) {
      const int64_t last = u1 - use.left - use.pos + use.n + use.lead - 1;  // unit
      const int64_t to = last < more * (each + 1) ? last / (each + 1) : more + (last - more * (each + 1)) / each;
      a.spans[(int64_t)use.entry * a.c.Hk + use.head] = make_int2(run, whole ? run : (int)to);
    }
    const int b = a.dRT.div(use.entry), row0 = (use.entry - b * a.RT) * ROWS;
    const int64_t slot = 2 * (int64_t)run + (use.t == 0 ? 1 : 0);
    for (int row = 0; row < ROWS && row0 + row < (int)(a.Sq * a.G); ++row) {
      if (!whole) {
        if (lane == 0) *attn_ml(a, slot * ROWS + row, ROWS * D) = make_float2(-INFINITY, nan);
        continue;
      }
      const int i = a.dG.div(row0 + row), hq = use.head * a.G + (row0 + row - i * a.G);
      uint16_t* dst = static_cast<uint16_t*>(a.o) + (((int64_t)b * a.Sq + i) * a.H + hq) * D;
      for (int d = lane; d < D; d += 32) dst[d] = 0x7fff;  // NaN in both types
      if (a.lse && lane == 0) a.lse[((int64_t)b * a.H + hq) * a.Sq + i] = nan;
    }
    attn_step(a, use);
  } while (attn_next<D, NT, T>(a, use));
}

template <int D, int GRP, int NT, int T, bool SPLIT, bool FINE>
__global__ void __launch_bounds__(32 * kAttnWarps, attn_cps(D, NT))
kv4_attn_kernel(const __grid_constant__ Kv4AttnArgs a) {
  using X = AttnShape<D, GRP, NT, T>;
  constexpr int U = X::U, J = X::J, NG = X::NG, MB = X::MB, S = kAttnStages;
  constexpr int VW = D / 64;  // words of a lane's D / 8 value dimensions
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ uint64_t full[kAttnWarps][S];
  __shared__ int ends[kAttnWarps], first_segment[2];
  __shared__ float mrg[kAttnWarps][X::ROWS][2];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, r = lane >> 2, c = lane & 3;
  unsigned char* ring = smem + warp * X::WARP;
  uint32_t* qsm = reinterpret_cast<uint32_t*>(ring + S * X::STAGE);
  float* gsm = reinterpret_cast<float*>(ring + S * X::STAGE + X::QB);

  griddep_launch_dependents();
  if (lane < S) mbar_init(&full[warp][lane], 1);
  fence_barrier_init();
  griddep_wait();

  // ---- this warp's run: each lane sums the segments of some entries ----------
  const int entries = (int)(a.B * a.RT);  // (sequence, row tile), Hk segments each
  const int chunk = (entries + 31) / 32;
  const int e0 = min(entries, lane * chunk), e1 = min(entries, e0 + chunk);
  int64_t mine = 0;
  for (int e = e0; e < e1; ++e) mine += attn_tiles<D, NT, T>(a, e);
  int64_t before = mine;
#pragma unroll
  for (int x = 1; x < 32; x <<= 1) {
    const int64_t t = __shfl_up_sync(0xffffffffu, before, x);
    if (lane >= x) before += t;
  }
  const int64_t tiles = __shfl_sync(0xffffffffu, before, 31) * a.c.Hk, warps = (int64_t)gridDim.x * kAttnWarps;
  // What a segment costs beside its tiles (its queries, its results) and the
  // least units of a run: with many tiles per warp 4 and with few 2 measured
  // best (64 ragged sequences 50.5 against 54.5 us, 16 x 5 tokens 19.7 against
  // 17.6, 1 x 1021 13.1 against 11.1).
  const int lead = tiles >= 8 * warps ? 4 : 2, least = lead + 1;
  before = (before - mine + (int64_t)e0 * lead) * a.c.Hk;
  mine = (mine + (int64_t)(e1 - e0) * lead) * a.c.Hk;
  const int64_t total = tiles + (int64_t)entries * a.c.Hk * lead;
  // the first `more` runs are one unit longer than `each`
  const int64_t runs = min(warps, wide_div(total + least - 1, least));
  const int64_t each = wide_div(total, runs), more = total - each * runs;
  auto run_at = [&](int64_t i) { return i * each + min(i, more); };
  auto run_of = [&](int64_t u) {
    return u < more * (each + 1) ? wide_div(u, each + 1) : more + wide_div(u - more * (each + 1), each);
  };
  const int64_t run0 = (int64_t)blockIdx.x * kAttnWarps, run = run0 + warp;
  if (run0 >= runs) return;
  AttnWalk use = {};
  use.lead = lead;
  bool one_segment = false;  // of all the block's runs
  const int64_t u1 = run_at(min(run + 1, runs));
  if (run < runs) {
    const int64_t u0 = run_at(run);
    int64_t at = u0 - before;
    const bool here = at >= 0 && at < mine;
    int e = e0, n = 0;
    if (here)
      for (;; ++e) {
        n = attn_tiles<D, NT, T>(a, e);
        const int64_t all = (int64_t)(n + lead) * a.c.Hk;
        if (at < all) break;
        at -= all;
      }
    const int src = __ffs(__ballot_sync(0xffffffffu, here)) - 1;
    use.entry = __shfl_sync(0xffffffffu, e, src);
    use.n = __shfl_sync(0xffffffffu, n, src);
    at = __shfl_sync(0xffffffffu, at, src);
    use.head = (int)wide_div(at, use.n + lead);
    use.pos = (int)(at - (int64_t)use.head * (use.n + lead));
    use.left = (int)(u1 - u0);
    const int64_t base = u0 - use.pos;  // of the segment
    one_segment = base <= run_at(run0) &&
                  run_at(min(run0 + kAttnWarps, runs)) <= base + use.n + lead;
  }
  // the warps past the last run join the merge of the others
  one_segment = __syncthreads_or(one_segment) != 0;
  AttnWalk get = use;
  uint32_t issued = 0, used = 0, use_phase = 0;  // tiles
  int use_stage = 0;
  bool timeout = false;

  // ---- the ring: the walk `get` runs ahead of `use` by up to S tiles ---------
  // Where pages hold tiles whole, get_src is a tile's bytes for as long as the
  // page (or the part) lasts, up to tile get_stop; a page is looked up one call
  // before it is needed.  Else (SPLIT) lanes 0 and 1 look up and copy 16 tokens
  // each (two copies by one lane: 75 against 56 us at 32 x 8192, D 64, P 16).
  int get_stop = 0, get_end = 0, get_pid = 0, get_at = 0, get_stage = 0;
  const int32_t* get_page = nullptr;
  const unsigned char* get_src = nullptr;
  bool getting = false, get_fresh = false, get_ok = false;
  bool bad = false, my_first = false, my_last = false;
  uint32_t bad_stages = 0;  // stages of tokens whose page is outside the pool
  const int64_t head_bytes = (int64_t)(a.c.P >> 4) * MB;
  auto look_up = [&](int tok) {
    const int pi = a.dP.div(tok);
    get_at = tok - pi * a.c.P;
    get_pid = tok < get_end ? get_page[pi] : -1;
  };
  auto open = [&]() {  // the next part's first tile
    getting = attn_next<D, NT, T>(a, get);
    if (getting) {
      const int b = a.dRT.div(get.entry), tok = get.t * T;
      bool over;
      get_end = attn_end<D, NT>(a, attn_len(a, b, over), get.entry - b * a.RT);
      get_page = a.table + b * a.width;
      if constexpr (SPLIT) {
        look_up(tok + 16 * (lane & 1));
        get_stop = get.t1;
      } else {
        const int pi = a.dP.div(tok);
        get_page += pi;
        get_pid = get_end > 0 ? *get_page : -1;
        get_at = tok - pi * a.c.P;
        get_stop = min(get.t1, get.t + (a.c.P - get_at) / T);
        get_fresh = true;
      }
    }
  };
  auto micro = [&](int pid, int at) {
    return a.c.data + ((int64_t)pid * a.c.Hk + get.head) * head_bytes + (at >> 4) * MB;
  };
  auto issue = [&]() {
    uint64_t* bar = &full[warp][get_stage];
    unsigned char* dst = ring + get_stage * X::STAGE;
    bool miss;
    if constexpr (SPLIT) {
      const bool want = lane < 2 && get.t * T + 16 * lane < get_end;
      const bool ok = want && (uint32_t)get_pid < (uint32_t)a.c.pages;
      const uint32_t n = __popc(__ballot_sync(0xffffffffu, ok));
      miss = __any_sync(0xffffffffu, want && !ok);
      fence_proxy_async();
      if (lane == 0) mbar_arrive_expect_tx(bar, n * MB);
      __syncwarp();
      if (ok) bulk_g2s(dst + lane * MB, micro(get_pid, get_at), MB, bar);
    } else {
      if (get_fresh) {
        get_fresh = false;
        get_ok = (uint32_t)get_pid < (uint32_t)a.c.pages;
        get_src = micro(get_pid, get_at);
      }
      miss = !get_ok && get_end > 0;
      if (lane == 0) {
        fence_proxy_async();
        mbar_arrive_expect_tx(bar, get_ok ? X::STAGE : 0);
        if (get_ok) bulk_g2s(dst, get_src, X::STAGE, bar);
      }
      get_src += X::STAGE;
    }
    if (miss || bad_stages) bad_stages = (bad_stages & ~(1u << get_stage)) | ((uint32_t)miss << get_stage);
    if (++get_stage == S) get_stage = 0;
    ++issued;
    if (++get.t == get_stop) {
      if (SPLIT || get.t == get.t1) {
        attn_step(a, get);
        open();
      } else {
        get_pid = *++get_page;
        get_at = 0;
        get_stop = min(get.t1, get_stop + a.c.P / T);
        get_fresh = true;
      }
    } else if constexpr (SPLIT) {
      look_up(get.t * T + 16 * (lane & 1));
    }
  };
  open();
  for (int k = 0; k < S && getting; ++k) issue();

  const ValueConsts vk = {held(0x64006400u), as_h2(held(0x2c002c00u)), as_h2(held(0xd400d400u))};
  // per row: maximum, sum, score that moves the maximum, exponent's offset
  float o[D / 16][NT][4];
  float m[NT][2], l[NT][2], lim[NT][2], off[NT][2], olo[X::FOLD ? NT : 1][2];
  float eight[X::FOLD ? NT : 1][4];  // FOLD: what the integers' -8 still owes the output
  auto settle = [&]() {
    if constexpr (X::FOLD) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
#pragma unroll
          for (int i = 0; i < D / 16; ++i) o[i][nt][e] += eight[nt][e];
          eight[nt][e] = 0.0f;
        }
    }
  };
  auto clear = [&]() {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int i = 0; i < D / 16; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][nt][e] = 0.0f;
      m[nt][0] = m[nt][1] = -INFINITY;
      l[nt][0] = l[nt][1] = off[nt][0] = off[nt][1] = 0.0f;
      lim[nt][0] = lim[nt][1] = -INFINITY;
      if constexpr (X::FOLD) {
        olo[nt][0] = olo[nt][1] = 0.0f;
#pragma unroll
        for (int e = 0; e < 4; ++e) eight[nt][e] = 0.0f;
      }
    }
  };
  clear();

  while (!timeout && attn_next<D, NT, T>(a, use)) {
    const int b = a.dRT.div(use.entry), rt = use.entry - b * a.RT, head = use.head;
    const int t0 = use.t, t1 = use.t1;
    const int len = attn_len(a, b, bad);
    const int end = attn_end<D, NT>(a, len, rt);
    const int R = (int)(a.Sq * a.G);
    const int row0 = rt * X::ROWS;
    // last token that a row of the tile sees
    auto last_of = [&](int row) {
      return a.causal ? len - (int)a.Sq + a.dG.div(min(row0 + row, R - 1)) : len - 1;
    };

    // ---- query rows -> B fragments -----------------------------------------
    // lane (r, c) holds row r of each 8, dimensions 32 j + 8 c .. + 7
    float cmul[NT][2];
    __syncwarp();
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int row = row0 + nt * 8 + r;
      float v[J][8];
#pragma unroll
      for (int j = 0; j < J; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) v[j][e] = 0.0f;
      if (row < R) {
        const int i = a.dG.div(row), hq = head * a.G + (row - i * a.G);
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
      const int me = top > 0.0f && ex < 255 ? min(263 - ex, 254) : 127;
      const float mag = __uint_as_float((uint32_t)me << 23);
      // scores are multiplied by |scale|; a scale of NaN goes in with the queries,
      // so that what a row does not see stays at -inf
      const float f = a.scale < 0.0f ? -mag : a.scale == a.scale ? mag : a.scale;
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
        reinterpret_cast<uint4*>(qsm)[(nt * J + j) * 32 + lane] = make_uint4(w[0], w[1], w[2], w[3]);
      }
      // |scale| log2(e) 2^24 / mag; the power of two alone may be past fp32's
      // range (bfloat16 queries of 2^113 on).  At least a number that leaves
      // scale = 0 a factor of its own: 0 * -inf is NaN
      const float cm = fmaxf(scalbnf(fabsf(a.scale) * kLog2e, 24 + 127 - me), 1e-37f);
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
        if (c == 0) gsm[(nt * NG + g) * 8 + r] = t;
      }
    }
    __syncwarp();
    const int all_see = last_of(0);  // tokens up to here are seen by every row
    const int mask_from = max(all_see + 1, 0) / T;  // and the tiles before this one

    clear();

    for (int t = t0; t < t1; ++t) {
      const int s = use_stage;
      if (!mbar_wait_warp(&full[warp][s], use_phase)) {
        timeout = true;
        break;
      }
      ++used;
      if (++use_stage == S) {
        use_stage = 0;
        use_phase ^= 1;
      }
      if (bad_stages) bad |= (bad_stages >> s) & 1;
      unsigned char* st = ring + s * X::STAGE;
      const int tok0 = t * T;
      const bool masked = t >= mask_from;
      if (masked) {
        // What lies past the length is garbage, and a value some row does not
        // see must not reach it as 0 * NaN: such parameters become zero, and
        // rows that do see a value that is not finite become NaN in the
        // dimensions of its group, as they do where every row sees it.
        uint32_t odd = 0;  // the groups of lane's token
        const int tok = tok0 + lane;
        if (lane < T && tok > all_see) {
          uint32_t* p = reinterpret_cast<uint32_t*>(st + (lane >> 4) * MB + X::VP) + (lane & 15) * NG;
#pragma unroll
          for (int g = 0; g < NG; ++g) {
            const uint32_t w = p[g];
            const bool bits = (w & 0x7c00u) == 0x7c00u || (w & 0x7c000000u) == 0x7c000000u;
            if (tok >= end) {
              p[g] = 0;
            } else if (bits) {
              p[g] = 0;
              odd |= 1u << g;
            }
          }
        }
        uint32_t some = __ballot_sync(0xffffffffu, odd != 0);
        for (; some; some &= some - 1) {
          const int from = __ffs(some) - 1;
          const bool mine = __shfl_sync(0xffffffffu, odd, from) >> (r * (D / 8) / GRP) & 1u;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int p = 0; p < 2; ++p)
              if (mine && last_of(nt * 8 + 2 * c + p) >= tok0 + from) {
#pragma unroll
                for (int i = 0; i < D / 16; ++i)
                  o[i][nt][p] = o[i][nt][2 + p] = __int_as_float(0x7fc00000);
              }
        }
        __syncwarp();
      }

      // ---- scores: [tokens] x [rows] ---------------------------------------
      float z[U][NT][4];
      uint32_t kw[U][2][J], kp[U][2][NG];  // rows r and r + 8
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const unsigned char* mb = st + (u) * MB;
          load_words<D / 8>(kw[u][h], mb + (r + 8 * h) * (D / 2) + c * (D / 8));
          load_words<4 * NG>(kp[u][h], mb + X::KP + (r + 8 * h) * 4 * NG);
        }
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        float acc[U][NT][4];
#pragma unroll
        for (int j = g * (GRP / 32); j < (g + 1) * (GRP / 32); ++j) {
          uint32_t qv[NT][4];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const uint4 v = reinterpret_cast<const uint4*>(qsm)[(nt * J + j) * 32 + lane];
            qv[nt][0] = v.x; qv[nt][1] = v.y; qv[nt][2] = v.z; qv[nt][3] = v.w;
          }
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const uint32_t x0 = kw[u][0][j], x1 = kw[u][1][j], y0 = x0 >> 8, y1 = x1 >> 8;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              if (j == g * (GRP / 32))
                mma16816_first(acc[u][nt], x0 & 0x000f000fu, x1 & 0x000f000fu, y0 & 0x000f000fu,
                               y1 & 0x000f000fu, qv[nt][0], qv[nt][1]);
              else
                mma16816(acc[u][nt], x0 & 0x000f000fu, x1 & 0x000f000fu, y0 & 0x000f000fu,
                         y1 & 0x000f000fu, qv[nt][0], qv[nt][1]);
              mma16816(acc[u][nt], x0 & 0x00f000f0u, x1 & 0x00f000f0u, y0 & 0x00f000f0u,
                       y1 & 0x00f000f0u, qv[nt][2], qv[nt][3]);
            }
          }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const float2 fa = __half22float2(as_h2(kp[u][0][g])), fb = __half22float2(as_h2(kp[u][1][g]));
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const float2 qs = reinterpret_cast<const float2*>(gsm)[(nt * NG + g) * 4 + c];
            float* zz = z[u][nt];
            zz[0] = fmaf(fa.x, acc[u][nt][0], fmaf(fa.y, qs.x, g ? zz[0] : 0.0f));
            zz[1] = fmaf(fa.x, acc[u][nt][1], fmaf(fa.y, qs.y, g ? zz[1] : 0.0f));
            zz[2] = fmaf(fb.x, acc[u][nt][2], fmaf(fb.y, qs.x, g ? zz[2] : 0.0f));
            zz[3] = fmaf(fb.x, acc[u][nt][3], fmaf(fb.y, qs.y, g ? zz[3] : 0.0f));
          }
        }
      }

      // ---- softmax: columns 2c, 2c + 1 are this lane's rows of queries -------
      // m is the maximum of the scores as they are (FOLD: in powers of two, and
      // with the value's scale); a tile moves it only when one is beyond it by
      // more than the slack, which each lane checks for its own
      float vs[U][2], vlo[U][2], vls[U][2];  // FOLD: s, lo + 8 s, log2(s) of tokens r, r + 8
      if constexpr (X::FOLD) {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float2 f = __half22float2(
                as_h2(reinterpret_cast<const uint32_t*>(st + u * MB + X::VP)[r + 8 * h]));
            vs[u][h] = f.x;
            vlo[u][h] = fmaf(8.0f, f.x, f.y);
            vls[u][h] = lg2_approx(fmaxf(f.x, 5.9604644775390625e-8f));
          }
      }
      bool moved = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        if (masked) {
          const int last[2] = {last_of(nt * 8 + 2 * c), last_of(nt * 8 + 2 * c + 1)};
#pragma unroll
          for (int u = 0; u < U; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (tok0 + 16 * u + r + 8 * (e >> 1) > last[e & 1]) z[u][nt][e] = -INFINITY;
        }
      }
      // what the maximum is taken of
      auto rank = [&](int u, int nt, int e) {
        return X::FOLD ? fmaf(z[u][nt][e], cmul[nt][e & 1], vls[u][e >> 1]) : z[u][nt][e];
      };
      float top[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          float v = fmaxf(rank(0, nt, p), rank(0, nt, 2 + p));
#pragma unroll
          for (int u = 1; u < U; ++u) v = fmaxf(v, fmaxf(rank(u, nt, p), rank(u, nt, 2 + p)));
          top[nt][p] = v;
          moved |= v > lim[nt][p];
        }
      if (__any_sync(0xffffffffu, moved)) {
        settle();
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float f[2];
#pragma unroll
          for (int p = 0; p < 2; ++p) {
            const float unit = X::FOLD ? 1.0f : cmul[nt][p];
            float v = fmaxf(m[nt][p], top[nt][p]);
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, x));
            // from -inf: nothing was summed yet (0 * 0 whatever the new one is)
            f[p] = m[nt][p] == -INFINITY ? 0.0f : ex2_approx((m[nt][p] - v) * unit);
            l[nt][p] *= f[p];
            if constexpr (X::FOLD) olo[nt][p] *= f[p];
            m[nt][p] = v;
            lim[nt][p] = v + kPSlack / unit;
            off[nt][p] = v == -INFINITY ? 0.0f : kPScale - v * unit;
          }
#pragma unroll
          for (int i = 0; i < D / 16; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[i][nt][e] *= f[e & 1];
        }
      }
      // probabilities as B fragments, [tokens] x [rows]; FINE: and their remainders
      uint32_t pf[U][NT][2], pr[FINE ? U : 1][FINE ? NT : 1][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int u = 0; u < U; ++u) {
          float p[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            p[e] = ex2_approx(fmaf(z[u][nt][e], cmul[nt][e & 1], off[nt][e & 1]));
            l[nt][e & 1] += p[e];
            if constexpr (X::FOLD) {
              olo[nt][e & 1] = fmaf(p[e], vlo[u][e >> 1], olo[nt][e & 1]);
              p[e] *= vs[u][e >> 1];
            }
          }
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const __half2 r2 = __floats2half2_rn(p[2 * h], p[2 * h + 1]);
            pf[u][nt][h] = transpose8x8(as_u32(r2));
            if constexpr (FINE) {
              const float2 back = __half22float2(r2);
              pr[u][nt][h] =
                  transpose8x8(as_u32(__floats2half2_rn(p[2 * h] - back.x, p[2 * h + 1] - back.y)));
            }
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
          if constexpr (!X::FOLD)
            par[k] = reinterpret_cast<const uint32_t*>(mb + X::VP)[tk * NG + r * (D / 8) / GRP];
          else par[k] = 0;
        }
        if constexpr (X::FOLD) {  // -8 for every dimension, in the units of the two rows
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            mma16816(eight[nt], 0x80088008u, 0x80808080u, 0x80088008u, 0x80808080u, pf[u][nt][0],
                     pf[u][nt][1]);
            if constexpr (FINE)
              mma16816(eight[nt], 0x80088008u, 0x80808080u, 0x80088008u, 0x80808080u, pr[u][nt][0],
                       pr[u][nt][1]);
          }
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
            const uint32_t b0 = __byte_perm(v[0][w], v[1][w], sel), b1 = __byte_perm(v[2][w], v[3][w], sel);
            uint32_t x0[4], x1[4];
            if constexpr (X::FOLD) {
              // n 2^-24, and 16 times that in the second rows
              x0[0] = b0 & 0x000f000fu; x0[1] = b0 & 0x00f000f0u;
              x1[0] = b1 & 0x000f000fu; x1[1] = b1 & 0x00f000f0u;
              x0[2] = (b0 >> 8) & 0x000f000fu; x0[3] = (b0 >> 8) & 0x00f000f0u;
              x1[2] = (b1 >> 8) & 0x000f000fu; x1[3] = (b1 >> 8) & 0x00f000f0u;
            } else {
              value_pairs(b0, s0, o0, vk, x0);
              value_pairs(b1, s1, o1, vk, x1);
            }
#pragma unroll
            for (int q = 0; q < 2; ++q)
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                float* sum = o[w * 4 + hi * 2 + q][nt];
                mma16816(sum, x0[2 * q], x0[2 * q + 1], x1[2 * q], x1[2 * q + 1], pf[u][nt][0],
                         pf[u][nt][1]);
                if constexpr (FINE)
                  mma16816(sum, x0[2 * q], x0[2 * q + 1], x1[2 * q], x1[2 * q + 1], pr[u][nt][0],
                           pr[u][nt][1]);
              }
          }
      }
      if (X::FOLD && (t & 3) == 3) settle();
      __syncwarp();
      if (getting) issue();
    }
    if (timeout) break;
    settle();
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int p = 0; p < 2; ++p) {
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) l[nt][p] += __shfl_xor_sync(0xffffffffu, l[nt][p], x);
        if (bad) l[nt][p] = __int_as_float(0x7fc00000);
        if constexpr (X::FOLD) {
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) olo[nt][p] += __shfl_xor_sync(0xffffffffu, olo[nt][p], x);
#pragma unroll
          for (int i = 0; i < D / 16; ++i) {
            o[i][nt][p] = fmaf(o[i][nt][p], 16777216.0f, olo[nt][p]);
            o[i][nt][2 + p] = fmaf(o[i][nt][2 + p], 1048576.0f, olo[nt][p]);
          }
        } else {
          m[nt][p] *= cmul[nt][p];  // in powers of two from here on
        }
      }
    const bool whole = t0 == 0 && t1 == use.n;
    const int64_t seg = (int64_t)use.entry * a.c.Hk + head;
    if (t0 == 0 && lane == 0) {
      // runs that hold the segment's first and last tile
      const int64_t past = u1 - use.left - use.pos + use.n + lead;
      a.spans[seg] = make_int2((int)run, whole ? (int)run : (int)run_of(past - 1));
    }
    if (one_segment) {  // the only part: the block's warps meet below
      my_first = t0 == 0;
      if (lane == 0) {
        first_segment[0] = use.entry;  // the same from every warp
        first_segment[1] = head;
      }
      my_last = t1 == use.n;
      break;
    }
    const int64_t slot = 2 * run + (t0 == 0 ? 1 : 0);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const int row = nt * 8 + 2 * c + p;
        if (row0 + row >= R) continue;
        if (whole) {
          const int i = a.dG.div(row0 + row), hq = head * a.G + (row0 + row - i * a.G);
          const float inv = attn_inverse(l[nt][p]);
          uint16_t* dst = static_cast<uint16_t*>(a.o) +
                          (((int64_t)b * a.Sq + i) * a.H + hq) * D + r * (D / 8);
#pragma unroll
          for (int k = 0; k < D / 64; ++k) {
            const uint2 x = attn_pack4(make_float4(o[4 * k][nt][p], o[4 * k][nt][2 + p],
                                                   o[4 * k + 1][nt][p], o[4 * k + 1][nt][2 + p]),
                                       inv, a.bf16);
            const uint2 y = attn_pack4(make_float4(o[4 * k + 2][nt][p], o[4 * k + 2][nt][2 + p],
                                                   o[4 * k + 3][nt][p], o[4 * k + 3][nt][2 + p]),
                                       inv, a.bf16);
            *reinterpret_cast<uint4*>(dst + 8 * k) = make_uint4(x.x, x.y, y.x, y.y);
          }
          if (a.lse && r == 0)
            a.lse[((int64_t)b * a.H + hq) * a.Sq + i] = attn_lse(m[nt][p], l[nt][p]);
        } else {
          float* dst = a.part + (slot * X::ROWS + row) * D + r * (D / 8);
#pragma unroll
          for (int k = 0; k < D / 32; ++k)
            *reinterpret_cast<float4*>(dst + 4 * k) =
                make_float4(o[2 * k][nt][p], o[2 * k][nt][2 + p], o[2 * k + 1][nt][p],
                            o[2 * k + 1][nt][2 + p]);
          if (r == 0) *attn_ml(a, slot * X::ROWS + row, X::ROWS * D) = make_float2(m[nt][p], l[nt][p]);
        }
      }
    attn_step(a, use);
  }
  if (timeout) {
    // nothing may land after the block has gone
    for (; used < issued; ++used) mbar_wait_warp(&full[warp][used % S], (used / S) & 1);
    if (lane == 0) {
      atomicAdd(&b2k_tu_timeouts, 1u);
      first_segment[0] = use.entry;
      first_segment[1] = use.head;
    }
    my_first = use.t == 0;
    my_last = use.t1 == use.n;
    attn_give_up<D, NT, T>(a, use, (int)run, u1, each, more);
  }
  if (!one_segment) return;

  // ---- the block's warps merge their parts of one segment ---------------------
  if (lane == 0) ends[warp] = (my_first ? 1 : 0) | (my_last ? 2 : 0);
  __syncthreads();  // the rings are drained: their memory holds the parts now
  float* mo = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const int row = nt * 8 + 2 * c + p;
      if (r == 0) {
        mrg[warp][row][0] = m[nt][p];
        mrg[warp][row][1] = timeout ? __int_as_float(0x7fc00000) : l[nt][p];
      }
#pragma unroll
      for (int i = 0; i < D / 16; ++i)
        *reinterpret_cast<float2*>(mo + (warp * X::ROWS + row) * D + r * (D / 8) + 2 * i) =
            f2(o[i][nt][p], o[i][nt][2 + p]);
    }
  __syncthreads();
  int first = -1, both = 0;  // the warp with the segment's first tile
#pragma unroll
  for (int w = 0; w < kAttnWarps; ++w) {
    if (ends[w] & 1) first = w;
    both |= ends[w];
  }
  const int entry = first_segment[0], head = first_segment[1];
  const int b = a.dRT.div(entry), row0 = (entry - b * a.RT) * X::ROWS, R = (int)(a.Sq * a.G);
  const int64_t slot = 2 * (run0 + max(first, 0)) + (first >= 0 ? 1 : 0);
  if (both != 3 && tid < X::ROWS * kAttnWarps) {
    // the other warps' slots, which the merge passes, hold nothing
    const int w = tid / X::ROWS, row = tid - w * X::ROWS;
    if (w > max(first, 0)) *attn_ml(a, 2 * (run0 + w) * X::ROWS + row, X::ROWS * D) = make_float2(-INFINITY, 0.0f);
  }
  for (int x = tid; x < X::ROWS * (D / 4); x += blockDim.x) {
    const int row = x / (D / 4), d = (x - row * (D / 4)) * 4;
    if (row0 + row >= R) continue;
    float M = -INFINITY, L = 0.0f;
#pragma unroll
    for (int w = 0; w < kAttnWarps; ++w) M = fmaxf(M, mrg[w][row][0]);
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int w = 0; w < kAttnWarps; ++w) {
      const float f = attn_weight(mrg[w][row][0], mrg[w][row][1], M);
      const float4 t = *reinterpret_cast<const float4*>(mo + (w * X::ROWS + row) * D + d);
      L = fmaf(mrg[w][row][1], f, L);
      v.x = fmaf(t.x, f, v.x); v.y = fmaf(t.y, f, v.y);
      v.z = fmaf(t.z, f, v.z); v.w = fmaf(t.w, f, v.w);
    }
    if (both == 3) {
      const int i = a.dG.div(row0 + row), hq = head * a.G + (row0 + row - i * a.G);
      *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.o) +
                                (((int64_t)b * a.Sq + i) * a.H + hq) * D + d) =
          attn_pack4(v, attn_inverse(L), a.bf16);
      if (a.lse && d == 0) a.lse[((int64_t)b * a.H + hq) * a.Sq + i] = attn_lse(M, L);
    } else {
      *reinterpret_cast<float4*>(a.part + (slot * X::ROWS + row) * D + d) = v;
      if (d == 0) *attn_ml(a, slot * X::ROWS + row, X::ROWS * D) = make_float2(M, L);
    }
  }
  if (both == 3 && tid == 0) a.spans[(int64_t)entry * a.c.Hk + head] = make_int2(0, 0);
}

// Merges the partial (m, l, O) of segments that span runs.  One block per row
// of a segment: all threads read the parts' (m, l) at once and leave their
// weights in shared memory, then D / 4 threads hold four dimensions each and
// kMergeSlices such slices take every kMergeSlices-th part, their loads
// independent of one another.  Fixed order of sums.
constexpr int kMergeSlices = 8, kMergeChunk = 1024;
template <int D, int NT>
__global__ void __launch_bounds__(D / 4 * kMergeSlices) kv4_attn_merge_kernel(
    const __grid_constant__ Kv4AttnArgs a) {
  constexpr int ROWS = attn_rows(NT), THREADS = D / 4 * kMergeSlices;
  __shared__ float4 sv[kMergeSlices][D / 4];
  __shared__ float weight[kMergeChunk], red[2][THREADS / 32];
  griddep_launch_dependents();
  griddep_wait();
  const int64_t seg = blockIdx.x;
  const int row = blockIdx.y, tid = threadIdx.x, slice = tid / (D / 4), d4 = tid - slice * (D / 4);
  const int2 span = a.spans[seg];
  const int parts = attn_parts(span.x, span.y, a.warps);
  if (parts == 0) return;
  const int entry = a.dHk.div((int)seg), b = a.dRT.div(entry), head = (int)seg - entry * a.c.Hk;
  const int rr = (entry - b * a.RT) * ROWS + row;
  if (rr >= (int)(a.Sq * a.G)) return;
  auto slot = [&](int i) { return (2 * (int64_t)(span.x + i) + (i == 0 ? 1 : 0)) * ROWS + row; };
  float M = -INFINITY;
  for (int i = tid; i < parts; i += THREADS) M = fmaxf(M, attn_ml(a, slot(i), ROWS * D)->x);
  M = warp_allmax(M);
  if ((tid & 31) == 0) red[0][tid >> 5] = M;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) M = fmaxf(M, red[0][w]);
  float L = 0.0f;
  float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (int base = 0; base < parts; base += kMergeChunk) {
    const int n = min(parts - base, kMergeChunk);
    __syncthreads();
    for (int i = tid; i < n; i += THREADS) {
      const float2 p = *attn_ml(a, slot(base + i), ROWS * D);
      const float f = attn_weight(p.x, p.y, M);
      // -1: holds nothing; a part that weighs 0 is read, its output may be NaN
      weight[i] = p.x == -INFINITY && p.y == 0.0f ? -1.0f : f;
      L = fmaf(p.y, f, L);
    }
    __syncthreads();
    for (int i = slice; i < n; i += 8 * kMergeSlices) {
      // eight loads together; a part that holds nothing has no output either
      float4 t[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int k = i + j * kMergeSlices;
        t[j] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (k < n && weight[k] != -1.0f)
          t[j] = *reinterpret_cast<const float4*>(a.part + slot(base + k) * D + 4 * d4);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int k = i + j * kMergeSlices;
        const float f = k < n && weight[k] != -1.0f ? weight[k] : 0.0f;
        v.x = fmaf(t[j].x, f, v.x); v.y = fmaf(t[j].y, f, v.y);
        v.z = fmaf(t[j].z, f, v.z); v.w = fmaf(t[j].w, f, v.w);
      }
    }
  }
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) L += __shfl_xor_sync(0xffffffffu, L, x);
  if ((tid & 31) == 0) red[1][tid >> 5] = L;
  sv[slice][d4] = v;
  __syncthreads();
  if (slice) return;
  L = 0.0f;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) L += red[1][w];
#pragma unroll
  for (int s = 1; s < kMergeSlices; ++s) {
    const float4 t = sv[s][d4];
    v.x += t.x; v.y += t.y; v.z += t.z; v.w += t.w;
  }
  const int i = a.dG.div(rr), hq = head * a.G + (rr - i * a.G);
  *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.o) + (((int64_t)b * a.Sq + i) * a.H + hq) * D +
                            4 * d4) = attn_pack4(v, attn_inverse(L), a.bf16);
  if (a.lse && d4 == 0) a.lse[((int64_t)b * a.H + hq) * a.Sq + i] = attn_lse(M, L);
}

// The same for many segments, of few parts each: every thread merges four
// dimensions of one row by itself, a block holds 1024 / D rows.
template <int D, int NT>
__global__ void __launch_bounds__(256) kv4_attn_merge_few_kernel(const __grid_constant__ Kv4AttnArgs a) {
  constexpr int ROWS = attn_rows(NT);
  griddep_launch_dependents();
  griddep_wait();
  const int seg = blockIdx.x, row = blockIdx.y * (1024 / D) + threadIdx.x / (D / 4);
  const int d = threadIdx.x % (D / 4) * 4;
  const int2 span = a.spans[seg];
  const int parts = attn_parts(span.x, span.y, a.warps);
  if (parts == 0) return;
  const int entry = a.dHk.div(seg), b = a.dRT.div(entry), head = seg - entry * a.c.Hk;
  const int rr = (entry - b * a.RT) * ROWS + row;
  if (row >= ROWS || rr >= (int)(a.Sq * a.G)) return;
  auto slot = [&](int i) { return (2 * (int64_t)(span.x + i) + (i == 0 ? 1 : 0)) * ROWS + row; };
  float M = -INFINITY, L = 0.0f;
  float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (int base = 0; base < parts; base += 4) {
    // four parts' loads together, the sums so far moved to their maximum
    float2 p[4];
    float4 t[4];
    float Mn = M;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      p[j] = base + j < parts ? *attn_ml(a, slot(base + j), ROWS * D) : make_float2(-INFINITY, 0.0f);
      Mn = fmaxf(Mn, p[j].x);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      // a part that holds nothing has no output either
      t[j] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (!(p[j].x == -INFINITY && p[j].y == 0.0f))
        t[j] = *reinterpret_cast<const float4*>(a.part + slot(base + j) * D + d);
    }
    const float f0 = attn_weight(M, L, Mn);
    L *= f0;
    v.x *= f0; v.y *= f0; v.z *= f0; v.w *= f0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float f = attn_weight(p[j].x, p[j].y, Mn);
      L = fmaf(p[j].y, f, L);
      v.x = fmaf(t[j].x, f, v.x); v.y = fmaf(t[j].y, f, v.y);
      v.z = fmaf(t[j].z, f, v.z); v.w = fmaf(t[j].w, f, v.w);
    }
    M = Mn;
  }
  const int i = a.dG.div(rr), hq = head * a.G + (rr - i * a.G);
  *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.o) + (((int64_t)b * a.Sq + i) * a.H + hq) * D + d) =
      attn_pack4(v, attn_inverse(L), a.bf16);
  if (a.lse && d == 0) a.lse[((int64_t)b * a.H + hq) * a.Sq + i] = attn_lse(M, L);
}

template <int D, int GRP, int NT, int T, bool SPLIT>
static int attn_launch(const Kv4AttnArgs& a, const AttnPlan& p, cudaStream_t st) {
  auto kern = a.bf16 ? kv4_attn_kernel<D, GRP, NT, T, SPLIT, false>
                     : kv4_attn_kernel<D, GRP, NT, T, SPLIT, true>;
  allow_max_dynamic_smem(kern);
  launch_pdl(kern, dim3(p.blocks), dim3(32 * kAttnWarps), AttnShape<D, GRP, NT, T>::SMEM, st, a);
  // A segment has about warps / segments parts; up to 16 a thread merges by
  // itself (few against one block per row: 64 ragged sequences 54.3 and 59.2 us,
  // 32 x 8192 tokens, 7 parts, 82.0 and 84.3; 8 x 65536, 28 parts, 122.7 and
  // 117.3; 1 x 100000, 222 parts, 78 and 44).
  const unsigned rows = (unsigned)(a.Sq * a.G < 8 * NT ? a.Sq * a.G : 8 * NT);
  if (p.segs * 16 >= p.warps)
    launch_pdl(kv4_attn_merge_few_kernel<D, NT>, dim3((unsigned)p.segs, (rows + 1024 / D - 1) / (1024 / D)),
               dim3(256), 0, st, a);
  else
    launch_pdl(kv4_attn_merge_kernel<D, NT>, dim3((unsigned)p.segs, rows), dim3(D / 4 * kMergeSlices), 0,
               st, a);
  return check_launch("b2k_kv4_attention");
}

// Tiles of 32 tokens where registers hold their scores (NT T / 8 per thread
// beside the output's NT D / 4), up to D 128, else of 16: 83 against 94 us at 16
// sequences of 16384 tokens, D 128.  Pages that are no multiple of 32 tokens
// take two copies per tile.
template <int D, int GRP, int NT>
static int attn_tokens(const Kv4AttnArgs& a, const AttnPlan& p, cudaStream_t st) {
  if constexpr (D < 256) {
    if (a.c.P % 32 == 0) return attn_launch<D, GRP, NT, 32, false>(a, p, st);
    return attn_launch<D, GRP, NT, 32, true>(a, p, st);
  } else {
    return attn_launch<D, GRP, NT, 16, false>(a, p, st);
  }
}

template <int D, int GRP>
static int attn_dispatch(const Kv4AttnArgs& a, const AttnPlan& p, cudaStream_t st) {
  return p.nt == 1 ? attn_tokens<D, GRP, 1>(a, p, st) : attn_tokens<D, GRP, 2>(a, p, st);
}

}  // namespace b2k
