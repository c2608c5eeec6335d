// Arguments of the tree attention kernels (tree.cu).
#pragma once

#include <stdint.h>

namespace mb {

struct TreeAttnArgs {
  const uint16_t *q, *k, *v, *kd, *vd;
  uint16_t* out;
  const int32_t* lens;
  const uint64_t* masks;
  int64_t mask_stride;
  // element strides: q / out / drafts (trace, node, head), caches (trace, head, row)
  int64_t qs[3], ks[3], vs[3], kds[3], vds[3], os[3];
  int T, m, H, Hkv, Lmax, d;
  float scale_log2;  // scale * log2(e)
  const float* scores;  // [T, Hkv, Lmax] or null
  float* scores_out;    // [T, Hkv, Lmax] or null
  float* draft_scores;  // [T, Hkv, m] or null
};

}  // namespace mb
