// Instances of the 4-bit cache attention for head dimension 256.
#include "tma.cuh"

B2K_DEFINE_TIMEOUT_COUNTER()

#include "kv4_attn_impl.cuh"

namespace b2k {

int attn_d256(const Kv4AttnArgs& a, const AttnPlan& p, cudaStream_t st) {
  switch (a.c.g) {
    case 32: return attn_dispatch<256, 32>(a, p, st);
    case 64: return attn_dispatch<256, 64>(a, p, st);
    default: return attn_dispatch<256, 128>(a, p, st);
  }
}

}  // namespace b2k
