// Which parts of a segment a merge of the 4-bit cache attention reads.  Plain
// C++, so that a test can compile it by itself.
#pragma once

#include "host_device.cuh"

namespace b2k {

// Parts in the runs first .. last of `warps`; 0 where one run held the segment
// whole.  The pair comes from the workspace: what is no such range (the kernel
// that writes it did not run) has no parts either.
B2K_HOST_DEVICE int attn_parts(int first, int last, int warps) {
  return first >= 0 && first < last && last < warps ? last - first + 1 : 0;
}

}  // namespace b2k
