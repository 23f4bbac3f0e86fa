// Instances of the 4-bit cache attention for head dimension 64.
#include "tma.cuh"

B2K_DEFINE_TIMEOUT_COUNTER()

#include "kv4_attn_impl.cuh"

namespace b2k {

int attn_d64(const Kv4AttnArgs& a, const AttnPlan& p, cudaStream_t st) {
  switch (a.c.g) {
    case 32: return attn_dispatch<64, 32>(a, p, st);
    default: return attn_dispatch<64, 64>(a, p, st);
  }
}

}  // namespace b2k
